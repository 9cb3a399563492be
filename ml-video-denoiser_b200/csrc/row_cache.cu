// The 8/4-bit row cache: rows are quantised as they are written to scattered
// or consecutive cache rows, and read back through row numbers or page tables
// (include/denoiser_b200_quant.h has the definition, quant.cuh the arithmetic).
//
// Both directions are bound by HBM. A sub-warp of SG lanes takes one group of a
// row, a lane 8 columns (a 16-byte load of FP16), so each byte moves once, the
// group's maximum is log2(SG) shuffles and nothing passes through shared memory;
// every lane has the loads of several groups in flight before it uses the first.
// Rows that begin anywhere (odd column counts, strides and addresses) move
// between their own boundaries and the vectors' in registers. Groups of more than
// 2048 columns take a CTA each (their warps' maxima meet in shared memory), and
// what is left (cache rows without the vectors' alignment, groups that are wide
// and odd) a warp per group with scalar accesses; both read what their registers
// do not hold twice.
//
// Measured: 2088960 x 32 FP16 written in 41.5 us and read back in 36 (209 MB each;
// in turn 79 to 82, out of L2 in part); five frames of 522240 x 64 read in 91 to 93
// (512 MB).
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <string>

#include "denoiser_b200_quant.h"
#include "launch.cuh"
#include "quant.cuh"
#include "row_cache.h"
#include "status.h"

namespace dnb {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr uint32_t kSiteWrite = 0x60, kSiteRead = 0x61;

// Rows of one scattered write may name the same slot; the last one counts.
//   up to kScanRows rows: every group looks through the later slots (64 x 1024:
//   2.5 us, 3.7 with marks; 1024 x 1024: 8.0 and 4.6);
//   more: the slot's scale words, which are about to be overwritten, first
//   hold the largest row index that names the slot (two small kernels). An
//   index below 2^23 is never the bit pattern of a scale (scales are >= 2^-126,
//   0x00800000, or NaN), so a group that finds another value has lost.
constexpr int64_t kScanRows = 256;
constexpr int64_t kMarkRows = 1 << 23;
enum : int { kOrderNone = 0, kOrderScan = 1, kOrderMark = 2 };

struct WriteArgs {
    CacheWrite p;
    int ngroups;
    int order;
};

// A launch has fewer than 2^30 groups, so rows and groups are counted in 32
// bits; addresses in 64.
__device__ __forceinline__ int64_t slot_of(const WriteArgs& a, int row) {
    return a.p.slots ? a.p.slots[row] : a.p.row0 + row;
}

// Whether group g of `row` is written; reports a slot behind the cache.
// Warp-wide call; the SG lanes of a sub-warp pass the same row.
template <int SG>
__device__ __forceinline__ bool wins(const WriteArgs& a, int row, int g, int64_t slot, bool live) {
    if (!a.p.slots) return live;
    if (live && slot >= a.p.capacity) report_error(a.p.err, kSiteWrite, kErrBadShape);
    live = live && slot >= 0 && slot < a.p.capacity;
    if (a.order == kOrderScan) {
        const int lane = threadIdx.x & 31;
        bool later = false;
        for (int j = lane % SG; j < static_cast<int>(a.p.rows); j += SG) later = later || (j > row && a.p.slots[j] == slot);
        const uint32_t hit = __ballot_sync(0xffffffffu, later);
        const uint32_t mine = SG == 32 ? 0xffffffffu : ((1u << (SG & 31)) - 1u) << (lane / SG * SG);
        live = live && !(hit & mine);
    } else if (a.order == kOrderMark && live) {
        live = __ldcg(reinterpret_cast<const int*>(a.p.scales + slot * a.ngroups + g)) == row;
    }
    __syncwarp();  // every lane has read the mark before one of them writes the scale over it
    return live;
}

__global__ void __launch_bounds__(kThreads) mark_kernel(const WriteArgs a, int phase) {
    pdl_trigger();
    pdl_wait();
    const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
    const int64_t row = i / a.ngroups;
    if (row >= a.p.rows) return;
    const int64_t slot = a.p.slots[row];
    if (slot < 0 || slot >= a.p.capacity) return;
    int* m = reinterpret_cast<int*>(a.p.scales + slot * a.ngroups + (i - row * a.ngroups));
    if (phase == 0)
        *m = -1;
    else
        atomicMax(m, static_cast<int>(row));
}

// 8 values from a 16-byte boundary `at` on, those outside [0, n) as zeros; the
// first of the row is value `first` of the 8. What a row's neighbours lie in is
// read with it, but nothing before the first row or behind the last one.
template <typename T>
__device__ __forceinline__ typename QuantOf<T>::Vec load_span(const T* at, int first, int n, const T* begin, const T* end) {
    using Q = QuantOf<T>;
    const int lo = max(first, 0), hi = min(first + n, 8);
    if (lo >= hi) return Q::zero();
    if (at >= begin && at + 8 <= end) {
        const typename Q::Vec v = Q::load(at);
        return lo > 0 || hi < 8 ? Q::only(v, lo, hi) : v;
    }
    T x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = i >= lo && i < hi ? at[i] : T(0.f);
    return Q::load_local(x);
}

// SHIFT: rows that begin anywhere. A lane's 8 values begin at the 16-byte
// boundary at or before its place in the row, so that they are one load; the
// codes move to their own boundary in registers, with the next lane's (1000000
// x 25: 182 us a value at a time, 36 this way).
template <typename T, int BITS, int SG, int V, int U, bool SHIFT>
__global__ void __launch_bounds__(kThreads) write_vec_kernel(const WriteArgs a) {
    using Q = QuantOf<T>;
    pdl_trigger();
    pdl_wait();
    constexpr int kPer = 32 / SG;  // groups of a warp at a time
    constexpr float qmax = BITS == 8 ? 127.f : 7.f;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int sub = lane / SG, l = lane % SG;
    const int nv = a.p.group / 8;
    const int units = static_cast<int>(a.p.rows) * a.ngroups;
    const int u0 = (blockIdx.x * kWarps + warp) * (kPer * U);
    if (u0 >= units) return;
    const T* x = static_cast<const T*>(a.p.x);
    const T* x_end = x + (a.p.rows - 1) * a.p.ldx + static_cast<int64_t>(a.ngroups) * a.p.group;
    typename Q::Vec v[U][V];
    int row[U], grp[U], off[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const int u = u0 + i * kPer + sub;
        row[i] = a.ngroups == 1 ? u : static_cast<int>(static_cast<uint32_t>(u) / static_cast<uint32_t>(a.ngroups));
        grp[i] = a.ngroups == 1 ? 0 : u - row[i] * a.ngroups;
        const T* src = x + row[i] * a.p.ldx + grp[i] * a.p.group;
        if constexpr (SHIFT) {
            off[i] = static_cast<int>(reinterpret_cast<uintptr_t>(src) / sizeof(T) % (16 / sizeof(T)));
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const int c = l + k * SG;
                v[i][k] = u < units ? load_span<T>(src - off[i] + c * 8, off[i] - c * 8, a.p.group, x, x_end) : Q::zero();
            }
        } else {
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const int c = l + k * SG;
                v[i][k] = (u < units && c < nv) ? Q::load(src + c * 8) : Q::zero();
            }
        }
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const bool there = u0 + i * kPer + sub < units;
        uint32_t mag = Q::mag(v[i][0]);
#pragma unroll
        for (int k = 1; k < V; ++k) mag = max(mag, Q::mag(v[i][k]));
#pragma unroll
        for (int d = SG / 2; d > 0; d >>= 1) mag = max(mag, __shfl_xor_sync(0xffffffffu, mag, d));
        const GroupScale g = group_scale<T>(mag, qmax);
        const bool rare = __any_sync(0xffffffffu, g.rare);
        const int64_t slot = there ? slot_of(a, row[i]) : -1;
        uint2 q[V];
        if constexpr (SHIFT) {
#pragma unroll
            for (int k = 0; k < V; ++k) {
                q[k] = codes8<T>(v[i][k], g, rare);
                if (BITS == 4) q[k].x = pack_nibbles(q[k]);
            }
#pragma unroll
            for (int k = 0; k < V; ++k) {
                // The next lane's, the last lane's next being the first one's next vector.
                uint2 b = l == 0 ? (k + 1 < V ? q[k + 1 < V ? k + 1 : k] : make_uint2(0, 0)) : q[k];
                if (SG == 1) {
                    // (a lane's own next vector)
                } else {
                    const int from = (lane & ~(SG - 1)) | ((l + 1) & (SG - 1));
                    b.x = __shfl_sync(0xffffffffu, b.x, from);
                    if (BITS == 8) b.y = __shfl_sync(0xffffffffu, b.y, from);
                }
                if (BITS == 4) {
                    q[k].x = __funnelshift_r(q[k].x, b.x, 4 * off[i]);
                } else {
                    const bool far = off[i] >= 4;
                    const uint32_t w0 = far ? q[k].y : q[k].x, w1 = far ? b.x : q[k].y, w2 = far ? b.y : b.x;
                    q[k] = make_uint2(__funnelshift_r(w0, w1, 8 * (off[i] & 3)), __funnelshift_r(w1, w2, 8 * (off[i] & 3)));
                }
            }
        }
        if (!wins<SG>(a, row[i], grp[i], slot, there)) continue;
        uint8_t* dst = a.p.codes + slot * a.p.ldc + static_cast<int64_t>(grp[i]) * (a.p.group * BITS / 8);
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const int c = l + k * SG;
            if constexpr (SHIFT) {
                const int left = a.p.group - c * 8;
                if (left >= 8) {
                    if (BITS == 8)
                        *reinterpret_cast<uint2*>(dst + c * 8) = q[k];
                    else
                        *reinterpret_cast<uint32_t*>(dst + c * 4) = q[k].x;
                } else {  // the row's last bytes
#pragma unroll
                    for (int b = 0; b < BITS; ++b)
                        if (b * 8 < left * BITS)
                            dst[c * BITS + b] = static_cast<uint8_t>((b < 4 ? q[k].x : q[k].y) >> (8 * (b & 3)));
                }
            } else if (c < nv) {
                const uint2 w = codes8<T>(v[i][k], g, rare);
                if (BITS == 8)
                    *reinterpret_cast<uint2*>(dst + c * 8) = w;
                else
                    *reinterpret_cast<uint32_t*>(dst + c * 4) = pack_nibbles(w);
            }
        }
        if (l == 0) a.p.scales[slot * a.ngroups + grp[i]] = g.s;
    }
}

// Groups of more than 2048 columns: a CTA per group, V vectors a thread in
// registers; what a group has beyond them is read twice.
template <typename T, int BITS, int V>
__global__ void __launch_bounds__(kThreads) write_wide_kernel(const WriteArgs a) {
    using Q = QuantOf<T>;
    __shared__ uint32_t s_mag;
    pdl_trigger();
    if (threadIdx.x == 0) s_mag = 0;
    __syncthreads();
    pdl_wait();
    constexpr float qmax = BITS == 8 ? 127.f : 7.f;
    const int u = blockIdx.x;
    const int row = static_cast<int>(static_cast<uint32_t>(u) / static_cast<uint32_t>(a.ngroups)), grp = u - row * a.ngroups;
    const int nv = a.p.group / 8;
    const T* src = static_cast<const T*>(a.p.x) + row * a.p.ldx + static_cast<int64_t>(grp) * a.p.group;
    typename Q::Vec v[V];
    uint32_t mag = 0;
#pragma unroll
    for (int k = 0; k < V; ++k) {
        const int c = threadIdx.x + k * kThreads;
        v[k] = c < nv ? Q::load(src + c * 8) : Q::zero();
    }
#pragma unroll
    for (int k = 0; k < V; ++k) mag = max(mag, Q::mag(v[k]));
    for (int c = threadIdx.x + V * kThreads; c < nv; c += kThreads) mag = max(mag, Q::mag(Q::load(src + c * 8)));
    mag = __reduce_max_sync(0xffffffffu, mag);
    if ((threadIdx.x & 31) == 0) atomicMax(&s_mag, mag);
    __syncthreads();
    const GroupScale g = group_scale<T>(s_mag, qmax);
    const int64_t slot = slot_of(a, row);
    const bool won = wins<32>(a, row, grp, slot, true);
    __syncthreads();  // every warp has read the mark before one thread writes the scale over it
    if (!won) return;
    uint8_t* dst = a.p.codes + slot * a.p.ldc + static_cast<int64_t>(grp) * a.p.group * BITS / 8;
    auto put = [&](int c, const typename Q::Vec& x) {
        const uint2 w = codes8<T>(x, g, g.rare);
        if (BITS == 8)
            *reinterpret_cast<uint2*>(dst + static_cast<int64_t>(c) * 8) = w;
        else
            *reinterpret_cast<uint32_t*>(dst + static_cast<int64_t>(c) * 4) = pack_nibbles(w);
    };
#pragma unroll
    for (int k = 0; k < V; ++k)
        if (static_cast<int>(threadIdx.x) + k * kThreads < nv) put(threadIdx.x + k * kThreads, v[k]);
    for (int c = threadIdx.x + V * kThreads; c < nv; c += kThreads) put(c, Q::load(src + c * 8));
    if (threadIdx.x == 0) a.p.scales[slot * a.ngroups + grp] = g.s;
}

// Any size and alignment: a warp takes U groups, lanes along the columns (a
// pair of them each, so that a byte of 4-bit codes is one lane's). KEEP pairs a
// lane stay in registers; what a group has more is read twice.
template <typename T, int KEEP, int U>
__global__ void __launch_bounds__(kThreads) write_any_kernel(const WriteArgs a) {
    using Q = QuantOf<T>;
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const int units = static_cast<int>(a.p.rows) * a.ngroups;
    const int u0 = (blockIdx.x * kWarps + (threadIdx.x >> 5)) * U;
    const int n = a.p.group;
    const float qmax = a.p.bits == 8 ? 127.f : 7.f;
    T keep[U][KEEP][2];
    auto place = [&](int u, int& row, int& grp) {
        row = static_cast<int>(static_cast<uint32_t>(u) / static_cast<uint32_t>(a.ngroups));
        grp = u - row * a.ngroups;
        return static_cast<const T*>(a.p.x) + row * a.p.ldx + static_cast<int64_t>(grp) * n;
    };
#pragma unroll
    for (int j = 0; j < U; ++j) {
        int row, grp;
        const T* src = place(min(u0 + j, units - 1), row, grp);
#pragma unroll
        for (int i = 0; i < KEEP; ++i) {
            const int c = lane * 2 + 64 * i;
            keep[j][i][0] = c < n ? src[c] : T(0.f);
            keep[j][i][1] = c + 1 < n ? src[c + 1] : T(0.f);
        }
    }
#pragma unroll
    for (int j = 0; j < U; ++j) {
        if (u0 + j >= units) break;
        int row, grp;
        const T* src = place(u0 + j, row, grp);
        uint32_t mag = 0;
#pragma unroll
        for (int i = 0; i < KEEP; ++i) mag = max(mag, max(Q::mag1(keep[j][i][0]), Q::mag1(keep[j][i][1])));
        for (int c = lane * 2 + 64 * KEEP; c < n; c += 64) {
            mag = max(mag, Q::mag1(src[c]));
            if (c + 1 < n) mag = max(mag, Q::mag1(src[c + 1]));
        }
        mag = __reduce_max_sync(0xffffffffu, mag);
        const GroupScale g = group_scale<T>(mag, qmax);
        const int64_t slot = slot_of(a, row);
        if (!wins<32>(a, row, grp, slot, true)) continue;
        uint8_t* dst = a.p.codes + slot * a.p.ldc + static_cast<int64_t>(grp) * n * a.p.bits / 8;
        auto put = [&](int c, T x0, T x1) {
            const uint32_t q0 = code1<T>(x0, g), q1 = code1<T>(x1, g);
            if (a.p.bits == 4) {
                dst[c / 2] = static_cast<uint8_t>((q0 & 15u) | (q1 << 4));
            } else {
                dst[c] = static_cast<uint8_t>(q0);
                if (c + 1 < n) dst[c + 1] = static_cast<uint8_t>(q1);
            }
        };
#pragma unroll
        for (int i = 0; i < KEEP; ++i)
            if (lane * 2 + 64 * i < n) put(lane * 2 + 64 * i, keep[j][i][0], keep[j][i][1]);
        for (int c = lane * 2 + 64 * KEEP; c < n; c += 64) put(c, src[c], c + 1 < n ? src[c + 1] : T(0.f));
        if (lane == 0) a.p.scales[slot * a.ngroups + grp] = g.s;
    }
}

// ---------------------------------------------------------------------------
// Reading
// ---------------------------------------------------------------------------

struct ReadArgs {
    const uint8_t* codes;
    int64_t ldc;
    const float* scales;
    int64_t capacity;
    int cols, bits, group, ngroups;
    const int64_t* slots;  // read_rows: slots or row0
    int64_t row0;
    const int32_t* table;  // read_pages (else null)
    int64_t table_ld;
    uint32_t page_rows, page_mul, page_shift;  // i / page_rows = (umulhi(i, page_mul) + i) >> page_shift for i < 2^31
    const int32_t* lengths;
    int64_t rows;          // rows of out a sequence may fill
    void* out;
    int64_t out_batch, ldo;
    uint32_t* err;
};

// Cache row of out row i of sequence b, or -1. i < 2^31.
__device__ __forceinline__ int64_t source_row(const ReadArgs& a, int b, int64_t i64, int64_t n) {
    if (i64 >= n) return -1;
    const uint32_t i = static_cast<uint32_t>(i64);
    int64_t r;
    if (a.table) {
        const uint32_t q = (__umulhi(i, a.page_mul) + i) >> a.page_shift;
        const int32_t page = __ldg(a.table + b * a.table_ld + q);
        if (page < 0) return -1;
        r = static_cast<int64_t>(page) * a.page_rows + (i - q * a.page_rows);
    } else {
        r = a.slots ? a.slots[i] : a.row0 + i;
        if (r < 0) return -1;
    }
    if (r >= a.capacity) {
        report_error(a.err, kSiteRead, kErrBadShape);
        return -1;
    }
    return r;
}

__device__ __forceinline__ int64_t sequence_rows(const ReadArgs& a, int b) {
    if (!a.lengths) return a.rows;
    const int64_t n = a.lengths[b];
    return n < 0 ? 0 : (n < a.rows ? n : a.rows);
}

__device__ __forceinline__ void store8(__half* p, const float2 (&f)[4]) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_half2(f[0].x, f[0].y), pack_half2(f[1].x, f[1].y),
                                              pack_half2(f[2].x, f[2].y), pack_half2(f[3].x, f[3].y));
}
__device__ __forceinline__ void store8(float* p, const float2 (&f)[4]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(f[0].x, f[0].y, f[1].x, f[1].y);
    reinterpret_cast<float4*>(p)[1] = make_float4(f[2].x, f[2].y, f[3].x, f[3].y);
}
__device__ __forceinline__ void store1(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }

// SG lanes per row, a lane W = 8 or 16 columns at a time (of one group), U rows
// of each sub-warp in flight.
template <typename T, int BITS, int SG, int U, int W>
__global__ void __launch_bounds__(kThreads) read_vec_kernel(const ReadArgs a) {
    pdl_trigger();
    pdl_wait();
    constexpr int kPer = 32 / SG;
    constexpr int kWords = W * BITS / 32;
    const int lane = threadIdx.x & 31;
    const int sub = lane / SG, l = lane % SG;
    const int b = blockIdx.y;
    const int64_t n = sequence_rows(a, b);
    const int64_t i0 = (static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5)) * (kPer * U) + sub;
    if (i0 - sub >= n) return;
    const int nv = a.cols / W;
    int64_t src[U];
#pragma unroll
    for (int k = 0; k < U; ++k) src[k] = source_row(a, b, i0 + k * kPer, n);
    T* out = static_cast<T*>(a.out) + b * a.out_batch + i0 * a.ldo;
    for (int c = l; c < nv; c += SG) {
        uint32_t w[U][kWords];
        float s[U];
        const int g = a.ngroups == 1 ? 0 : c * W / a.group;
#pragma unroll
        for (int k = 0; k < U; ++k) {
            if (src[k] < 0) continue;
            const uint8_t* p = a.codes + src[k] * a.ldc + c * (W * BITS / 8);
            if constexpr (kWords == 4) {
                const uint4 v = *reinterpret_cast<const uint4*>(p);
                w[k][0] = v.x, w[k][1] = v.y, w[k][2] = v.z, w[k][3] = v.w;
            } else if constexpr (kWords == 2) {
                const uint2 v = *reinterpret_cast<const uint2*>(p);
                w[k][0] = v.x, w[k][1] = v.y;
            } else {
                w[k][0] = *reinterpret_cast<const uint32_t*>(p);
            }
            s[k] = a.scales[src[k] * a.ngroups + g];
        }
#pragma unroll
        for (int k = 0; k < U; ++k) {
            if (src[k] < 0) continue;
            const float2 s2 = make_float2(s[k], s[k]), zero2 = make_float2(0.f, 0.f);
            T* o = out + k * kPer * a.ldo + c * W;
#pragma unroll
            for (int h = 0; h < W / 8; ++h) {
                float2 f[4];
                if constexpr (BITS == 8) {
                    float2 lo[2], hi[2];
                    bytes_to_f(w[k][2 * h], lo);
                    bytes_to_f(w[k][2 * h + 1], hi);
                    f[0] = lo[0], f[1] = lo[1], f[2] = hi[0], f[3] = hi[1];
                } else {
                    nibbles_to_f(w[k][h], f);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) f[i] = ffma2(f[i], s2, zero2);
                store8(o + h * 8, f);
            }
        }
    }
}

// Rows of out that begin anywhere: a lane's 8 columns begin at the 16-byte
// boundary at or before its place in the row, so that all but a row's ends are
// 16-byte stores; their codes are cut from the words they lie in (1000000 x 25:
// 121 us a value at a time, 38 this way). One scale a row.
template <typename T, int BITS, int SG>
__global__ void __launch_bounds__(kThreads) read_shift_kernel(const ReadArgs a) {
    pdl_trigger();
    pdl_wait();
    constexpr int kPer = 32 / SG;
    const int lane = threadIdx.x & 31;
    const int b = blockIdx.y;
    const int64_t n = sequence_rows(a, b);
    const int64_t i = (static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5)) * kPer + lane / SG;
    const int64_t src = source_row(a, b, i, n);
    if (src < 0) return;
    T* out = static_cast<T*>(a.out) + b * a.out_batch + i * a.ldo;
    const int off = static_cast<int>(reinterpret_cast<uintptr_t>(out) / sizeof(T) % (16 / sizeof(T)));
    const uint32_t* w = reinterpret_cast<const uint32_t*>(a.codes + src * a.ldc);
    const int words = (a.cols * BITS + 31) / 32;
    const float s = a.scales[src];
    const float2 s2 = make_float2(s, s), zero2 = make_float2(0.f, 0.f);
    for (int c = lane % SG * 8 - off; c < a.cols; c += SG * 8) {
        constexpr int kIn = 32 / BITS;  // codes of a word
        const int first = c >= 0 ? c / kIn : -((kIn - 1 - c) / kIn);
        const int shift = (c - first * kIn) * BITS;
        auto word = [&](int k) { return first + k >= 0 && first + k < words ? __ldg(w + first + k) : 0u; };
        float2 f[4];
        if constexpr (BITS == 8) {
            const uint32_t w0 = word(0), w1 = word(1), w2 = shift ? word(2) : 0u;
            float2 lo[2], hi[2];
            bytes_to_f(__funnelshift_r(w0, w1, shift), lo);
            bytes_to_f(__funnelshift_r(w1, w2, shift), hi);
            f[0] = lo[0], f[1] = lo[1], f[2] = hi[0], f[3] = hi[1];
        } else {
            const uint32_t w0 = word(0), w1 = shift ? word(1) : 0u;
            nibbles_to_f(__funnelshift_r(w0, w1, shift), f);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) f[k] = ffma2(f[k], s2, zero2);
        if (c >= 0 && c + 8 <= a.cols) {
            store8(out + c, f);
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (c + k >= 0 && c + k < a.cols) store1(out + c + k, k & 1 ? f[k >> 1].y : f[k >> 1].x);
        }
    }
}

// Any size and alignment: a warp takes U rows, lanes along the columns.
template <typename T, int BITS, int U>
__global__ void __launch_bounds__(kThreads) read_any_kernel(const ReadArgs a) {
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const int b = blockIdx.y;
    const int64_t n = sequence_rows(a, b);
    const int64_t i0 = (static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5)) * U;
    if (i0 >= n) return;
    int64_t src[U];
#pragma unroll
    for (int k = 0; k < U; ++k) src[k] = source_row(a, b, i0 + k, n);
    T* out = static_cast<T*>(a.out) + b * a.out_batch + i0 * a.ldo;
    for (int c = lane; c < a.cols; c += 32) {
        const int g = a.ngroups == 1 ? 0 : c / a.group;
        int q[U];
        float s[U];
#pragma unroll
        for (int k = 0; k < U; ++k) {
            if (src[k] < 0) continue;
            const uint8_t* p = a.codes + src[k] * a.ldc;
            q[k] = BITS == 8 ? static_cast<int>(static_cast<int8_t>(p[c])) : static_cast<int>(p[c >> 1]);
            s[k] = a.scales[src[k] * a.ngroups + g];
        }
#pragma unroll
        for (int k = 0; k < U; ++k) {
            if (src[k] < 0) continue;
            if (BITS == 4) q[k] = static_cast<int>(static_cast<uint32_t>(q[k]) << (c & 1 ? 24 : 28)) >> 28;  // the signed nibble
            store1(out + k * a.ldo + c, static_cast<float>(q[k]) * s[k]);
        }
    }
}

bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

int pow2_lanes(int nv) {
    int s = 1;
    while (s < nv && s < 32) s <<= 1;
    return s;
}

template <typename T, int BITS, bool SHIFT, int SG, int V, int U>
cudaError_t write_run(const WriteArgs& a, cudaStream_t s) {
    const int64_t per = static_cast<int64_t>(kWarps) * (32 / SG) * U;
    const int64_t units = a.p.rows * a.ngroups;
    return launch_pdl(write_vec_kernel<T, BITS, SG, V, U, SHIFT>, dim3(static_cast<unsigned>((units + per - 1) / per)),
                      dim3(kThreads), 0, s, a);
}

// Two groups in flight per sub-warp for long FP16 writes, where that still gives
// every SM four CTAs (522240 x 64: 21.6 us, 22.6 with one; 1000 x 256: 1.9 and
// 1.5). FP32 values are twice the bytes a lane: one (522240 x 64: 29.5, 31.0
// with two).
template <typename T, int BITS, bool SHIFT, int SG>
cudaError_t write_groups(const WriteArgs& a, cudaStream_t s) {
    const bool two = sizeof(T) == 2 && a.p.rows * a.ngroups >= 4 * 148 * kWarps * (32 / SG) * 2;
    return two ? write_run<T, BITS, SHIFT, SG, 1, 2>(a, s) : write_run<T, BITS, SHIFT, SG, 1, 1>(a, s);
}

template <typename T, int KEEP, int U>
cudaError_t write_any(const WriteArgs& a, cudaStream_t s) {
    const int64_t units = a.p.rows * a.ngroups, per = static_cast<int64_t>(kWarps) * U;
    return launch_pdl(write_any_kernel<T, KEEP, U>, dim3(static_cast<unsigned>((units + per - 1) / per)), dim3(kThreads), 0,
                      s, a);
}

// Vectors that 8-value pieces of a group may touch: SHIFT begins up to a vector early.
template <typename T, bool SHIFT>
int group_vecs(const WriteArgs& a) {
    return (a.p.group + 7 + (SHIFT ? static_cast<int>(16 / sizeof(T)) - 1 : 0)) / 8;
}

template <typename T, int BITS, bool SHIFT>
cudaError_t write_bits(const WriteArgs& a, cudaStream_t s) {
    const int nv = group_vecs<T, SHIFT>(a);
    switch (pow2_lanes(nv)) {
        case 1: return write_groups<T, BITS, SHIFT, 1>(a, s);
        case 2: return write_groups<T, BITS, SHIFT, 2>(a, s);
        case 4: return write_groups<T, BITS, SHIFT, 4>(a, s);
        case 8: return write_groups<T, BITS, SHIFT, 8>(a, s);
        case 16: return write_groups<T, BITS, SHIFT, 16>(a, s);
        default: break;
    }
    if (nv <= 32) return write_groups<T, BITS, SHIFT, 32>(a, s);
    if (nv <= 64) return write_run<T, BITS, SHIFT, 32, 2, 1>(a, s);
    if (nv <= 128) return write_run<T, BITS, SHIFT, 32, 4, 1>(a, s);
    if (SHIFT || nv <= 256) return write_run<T, BITS, SHIFT, 32, 8, 1>(a, s);
    const dim3 grid(static_cast<unsigned>(a.p.rows * a.ngroups));
    if (nv <= 2 * kThreads) return launch_pdl(write_wide_kernel<T, BITS, 2>, grid, dim3(kThreads), 0, s, a);
    return launch_pdl(write_wide_kernel<T, BITS, 4>, grid, dim3(kThreads), 0, s, a);
}

template <typename T>
cudaError_t write_type(const WriteArgs& a, cudaStream_t s) {
    const CacheWrite& p = a.p;
    // A vector of 8 codes has `bits` bytes.
    const bool codes = aligned(p.codes, p.bits) && p.ldc % p.bits == 0;
    const bool rows = p.group % 8 == 0 && aligned(p.x, 16) && p.ldx * sizeof(T) % 16 == 0;
    if (codes && rows) return p.bits == 8 ? write_bits<T, 8, false>(a, s) : write_bits<T, 4, false>(a, s);
    if (codes && group_vecs<T, true>(a) <= 256) return p.bits == 8 ? write_bits<T, 8, true>(a, s) : write_bits<T, 4, true>(a, s);
    // 8 pairs a lane in registers: groups of one row, or pieces of several.
    if (p.group <= 64) return write_any<T, 1, 8>(a, s);
    if (p.group <= 256) return write_any<T, 4, 2>(a, s);
    return write_any<T, 8, 1>(a, s);
}

template <typename T, int BITS, int SG, int U, int W>
cudaError_t read_run(const ReadArgs& a, int batch, cudaStream_t s) {
    const int64_t per = static_cast<int64_t>(kWarps) * (32 / SG) * U;
    return launch_pdl(read_vec_kernel<T, BITS, SG, U, W>, dim3(static_cast<unsigned>((a.rows + per - 1) / per), batch),
                      dim3(kThreads), 0, s, a);
}

template <typename T, int BITS, int SG, int W>
cudaError_t read_rows(const ReadArgs& a, int batch, cudaStream_t s) {
    // One row in flight per sub-warp: more CTAs hide more than more loads of one
    // (five frames of 522240 x 64 to FP16: 93 us, 102 with four rows). Lanes of 8
    // FP16 columns take two in long reads (1000000 x 24: 16.4, 18.5 with one).
    const bool two = W == 8 && sizeof(T) == 2 && a.rows * batch >= 4 * 148 * kWarps * (32 / SG) * 2;
    return two ? read_run<T, BITS, SG, 2, W>(a, batch, s) : read_run<T, BITS, SG, 1, W>(a, batch, s);
}

template <typename T, int BITS, int W>
cudaError_t read_width(const ReadArgs& a, int batch, cudaStream_t s) {
    switch (pow2_lanes(a.cols / W)) {
        case 1: return read_rows<T, BITS, 1, W>(a, batch, s);
        case 2: return read_rows<T, BITS, 2, W>(a, batch, s);
        case 4: return read_rows<T, BITS, 4, W>(a, batch, s);
        case 8: return read_rows<T, BITS, 8, W>(a, batch, s);
        case 16: return read_rows<T, BITS, 16, W>(a, batch, s);
        default: return read_rows<T, BITS, 32, W>(a, batch, s);
    }
}

// 16 columns a lane halve the work per FP16 row (five frames of 522240 x 64: 93
// us, 96 with 8). FP32 rows take 8, so that a lane's stores stay closer (522240 x
// 64: 37 us, 41 with 16; 168000 x 512 from 4 bits: 76 and 91).
template <typename T, int BITS>
cudaError_t read_bits(const ReadArgs& a, int batch, cudaStream_t s) {
    if constexpr (sizeof(T) == 4) return read_width<T, BITS, 8>(a, batch, s);
    const bool wide = a.cols % 16 == 0 && a.group % 16 == 0 && aligned(a.codes, 2 * BITS) && a.ldc % (2 * BITS) == 0;
    return wide ? read_width<T, BITS, 16>(a, batch, s) : read_width<T, BITS, 8>(a, batch, s);
}

template <typename T, int BITS>
cudaError_t read_shift(const ReadArgs& a, int batch, cudaStream_t s) {
    auto run = [&](auto kernel, int sg) {
        const int64_t per = static_cast<int64_t>(kWarps) * (32 / sg);
        return launch_pdl(kernel, dim3(static_cast<unsigned>((a.rows + per - 1) / per), batch), dim3(kThreads), 0, s, a);
    };
    switch (pow2_lanes((a.cols + 6 + static_cast<int>(16 / sizeof(T))) / 8)) {
        case 1: return run(read_shift_kernel<T, BITS, 1>, 1);
        case 2: return run(read_shift_kernel<T, BITS, 2>, 2);
        case 4: return run(read_shift_kernel<T, BITS, 4>, 4);
        case 8: return run(read_shift_kernel<T, BITS, 8>, 8);
        case 16: return run(read_shift_kernel<T, BITS, 16>, 16);
        default: return run(read_shift_kernel<T, BITS, 32>, 32);
    }
}

template <typename T>
cudaError_t read_type(const ReadArgs& a, int batch, cudaStream_t s) {
    const bool vec = a.cols % 8 == 0 && a.group % 8 == 0 && aligned(a.codes, a.bits) && a.ldc % a.bits == 0 &&
                     aligned(a.out, 16) && a.ldo * sizeof(T) % 16 == 0 && a.out_batch * sizeof(T) % 16 == 0;
    if (!vec && a.ngroups == 1 && aligned(a.codes, 4) && a.ldc % 4 == 0)
        return a.bits == 8 ? read_shift<T, 8>(a, batch, s) : read_shift<T, 4>(a, batch, s);
    if (!vec) {
        constexpr int kU = 2;
        const dim3 grid(static_cast<unsigned>((a.rows + kWarps * kU - 1) / (kWarps * kU)), batch);
        return a.bits == 8 ? launch_pdl(read_any_kernel<T, 8, kU>, grid, dim3(kThreads), 0, s, a)
                           : launch_pdl(read_any_kernel<T, 4, kU>, grid, dim3(kThreads), 0, s, a);
    }
    return a.bits == 8 ? read_bits<T, 8>(a, batch, s) : read_bits<T, 4>(a, batch, s);
}

int run_read(const ReadArgs& a, int batch, int dtype, cudaStream_t s, const char* name) {
    const cudaError_t e = dtype == 1 ? read_type<__half>(a, batch, s) : read_type<float>(a, batch, s);
    return e == cudaSuccess ? DN_OK : dn_cuda_fail(e, name);
}

// The kernels read row numbers, page tables and lengths as the words that they are.
int check_words(const void* slots, const void* table, const void* lengths, const void* err, const std::string& name) {
    if (!aligned(slots, 8)) return dn_fail_str(DN_ERR_INVALID_ARG, name + ": slots must be 8-byte aligned");
    if (!aligned(table, 4) || !aligned(lengths, 4))
        return dn_fail_str(DN_ERR_INVALID_ARG, name + ": page table and lengths must be 4-byte aligned");
    if (!aligned(err, 4)) return dn_fail_str(DN_ERR_INVALID_ARG, name + ": the error word must be 4-byte aligned");
    return DN_OK;
}

// The shape of a cache: DN_OK, or the status of what is wrong with it.
int check_cache(const void* codes, int64_t ldc, const float* scales, int64_t capacity, int cols, int bits, int& group,
                int dtype, const std::string& name) {
    if (dtype != 0 && dtype != 1) return dn_fail_str(DN_ERR_DTYPE, name + ": dtype must be 0 (FP32) or 1 (FP16)");
    if (bits != 8 && bits != 4) return dn_fail_str(DN_ERR_INVALID_ARG, name + ": bits must be 8 or 4");
    if (cols <= 0 || cols > (1 << 24)) return dn_fail_str(DN_ERR_INVALID_ARG, name + ": cols outside [1, 2^24]");
    if (group == 0) group = cols;
    if (group < 0 || cols % group != 0) return dn_fail_str(DN_ERR_INVALID_ARG, name + ": group does not divide cols");
    if (group != cols && group % 8 != 0)
        return dn_fail_str(DN_ERR_INVALID_ARG, name + ": a group smaller than a row must be a multiple of 8");
    if (capacity < 0 || capacity >= (1LL << 31))
        return dn_fail_str(DN_ERR_INVALID_ARG, name + ": capacity outside [0, 2^31)");
    if (ldc < (static_cast<int64_t>(cols) * bits + 7) / 8)
        return dn_fail_str(DN_ERR_INVALID_ARG, name + ": ld_codes is less than a row");
    if (capacity > 0 && (!codes || !scales)) return dn_fail_str(DN_ERR_INVALID_ARG, name + ": null cache");
    if (!aligned(scales, 4)) return dn_fail_str(DN_ERR_INVALID_ARG, name + ": scales must be 4-byte aligned");
    return DN_OK;
}

// Rows of a caller's matrix: aligned to their type, strides that hold a row.
int check_rows(const void* x, int dtype, int64_t rows, int64_t ld, int cols, const std::string& name) {
    if (rows < 0 || rows >= (1LL << 31)) return dn_fail_str(DN_ERR_INVALID_ARG, name + ": rows outside [0, 2^31)");
    if (rows == 0) return DN_OK;
    if (!x) return dn_fail_str(DN_ERR_INVALID_ARG, name + ": null pointer");
    if (!aligned(x, dtype == 1 ? 2 : 4)) return dn_fail_str(DN_ERR_INVALID_ARG, name + ": misaligned pointer");
    if (ld < cols && rows > 1) return dn_fail_str(DN_ERR_INVALID_ARG, name + ": row stride is less than a row");
    return DN_OK;
}

}  // namespace

int launch_cache_write(const CacheWrite& p0, cudaStream_t s) {
    const int ngroups = p0.cols / p0.group;
    // A launch takes up to 2^23 rows (marks) and 2^30 groups.
    const int64_t most = std::max<int64_t>(1, std::min<int64_t>(p0.slots ? kMarkRows : (1LL << 30), (1LL << 30) / ngroups));
    for (int64_t r = 0; r < p0.rows; r += most) {
        WriteArgs a{p0, ngroups, kOrderNone};
        a.p.rows = std::min(most, p0.rows - r);
        a.p.x = static_cast<const char*>(p0.x) + r * p0.ldx * (p0.dtype == 1 ? 2 : 4);
        a.p.row0 = p0.row0 + r;
        if (p0.slots) {
            a.p.slots = p0.slots + r;
            a.order = a.p.rows == 1 ? kOrderNone : a.p.rows <= kScanRows ? kOrderScan : kOrderMark;
        }
        if (a.order == kOrderMark) {
            const unsigned blocks = static_cast<unsigned>((a.p.rows * ngroups + kThreads - 1) / kThreads);
            for (int phase = 0; phase < 2; ++phase) {
                const cudaError_t e = launch_pdl(mark_kernel, dim3(blocks), dim3(kThreads), 0, s, a, phase);
                if (e != cudaSuccess) return dn_cuda_fail(e, "cache write: mark launch");
            }
        }
        const cudaError_t e = p0.dtype == 1 ? write_type<__half>(a, s) : write_type<float>(a, s);
        if (e != cudaSuccess) return dn_cuda_fail(e, "cache write: launch");
    }
    return DN_OK;
}

}  // namespace dnb

using namespace dnb;

extern "C" {

int dn_launch_cache_write(const void* x, int dtype, int64_t ldx, int64_t rows, int cols, const int64_t* slots,
                          int64_t row0, void* codes, int64_t ld_codes, float* scales, int64_t capacity, int bits,
                          int group, uint32_t* err_dev, void* stream) {
    const char* name = "dn_launch_cache_write";
    DN_TRY(check_cache(codes, ld_codes, scales, capacity, cols, bits, group, dtype, name));
    DN_TRY(check_rows(x, dtype, rows, ldx, cols, name));
    DN_TRY(check_words(slots, nullptr, nullptr, err_dev, name));
    if (!slots && (row0 < 0 || row0 > capacity - rows))
        return dn_fail(DN_ERR_INVALID_ARG, "dn_launch_cache_write: rows outside the cache");
    if (rows == 0) return DN_OK;
    return launch_cache_write(CacheWrite{x, dtype, ldx, rows, cols, slots, row0, static_cast<uint8_t*>(codes), ld_codes,
                                         scales, capacity, bits, group, err_dev},
                              static_cast<cudaStream_t>(stream));
}

int dn_launch_cache_read_rows(const void* codes, int64_t ld_codes, const float* scales, int64_t capacity, int cols,
                              int bits, int group, const int64_t* slots, int64_t row0, int64_t rows, void* out,
                              int dtype, int64_t ldo, uint32_t* err_dev, void* stream) {
    const char* name = "dn_launch_cache_read_rows";
    DN_TRY(check_cache(codes, ld_codes, scales, capacity, cols, bits, group, dtype, name));
    DN_TRY(check_rows(out, dtype, rows, ldo, cols, name));
    DN_TRY(check_words(slots, nullptr, nullptr, err_dev, name));
    if (!slots && (row0 < 0 || row0 > capacity - rows))
        return dn_fail(DN_ERR_INVALID_ARG, "dn_launch_cache_read_rows: rows outside the cache");
    if (rows == 0) return DN_OK;
    ReadArgs a{};
    a.codes = static_cast<const uint8_t*>(codes);
    a.ldc = ld_codes;
    a.scales = scales;
    a.capacity = capacity;
    a.cols = cols;
    a.bits = bits;
    a.group = group;
    a.ngroups = cols / group;
    a.slots = slots;
    a.row0 = row0;
    a.rows = rows;
    a.out = out;
    a.ldo = ldo;
    a.err = err_dev;
    return run_read(a, 1, dtype, static_cast<cudaStream_t>(stream), name);
}

int dn_launch_cache_read_pages(const void* codes, int64_t ld_codes, const float* scales, int64_t capacity, int cols,
                               int bits, int group, int64_t page_rows, const int32_t* table, int64_t table_ld,
                               int64_t table_cols, const int32_t* lengths, int batch, int64_t max_rows, void* out,
                               int dtype, int64_t out_batch, int64_t ldo, uint32_t* err_dev, void* stream) {
    const char* name = "dn_launch_cache_read_pages";
    DN_TRY(check_cache(codes, ld_codes, scales, capacity, cols, bits, group, dtype, name));
    if (page_rows <= 0 || page_rows >= (1LL << 31))
        return dn_fail(DN_ERR_INVALID_ARG, "dn_launch_cache_read_pages: page_rows outside [1, 2^31)");
    if (batch < 0 || batch > 65535) return dn_fail(DN_ERR_INVALID_ARG, "dn_launch_cache_read_pages: batch outside [0, 65535]");
    if (table_cols < 0 || table_cols >= (1LL << 31) || (batch > 1 && table_ld < table_cols))
        return dn_fail(DN_ERR_INVALID_ARG, "dn_launch_cache_read_pages: bad page table");
    DN_TRY(check_rows(out, dtype, max_rows, ldo, cols, name));
    DN_TRY(check_words(nullptr, table, lengths, err_dev, name));
    const int64_t rows = std::min(max_rows, table_cols * page_rows);
    if (rows == 0 || batch == 0) return DN_OK;
    if (!table) return dn_fail(DN_ERR_INVALID_ARG, "dn_launch_cache_read_pages: null page table");
    if (batch > 1 && out_batch < (max_rows - 1) * ldo + cols)
        return dn_fail(DN_ERR_INVALID_ARG, "dn_launch_cache_read_pages: out_batch is less than a sequence");
    ReadArgs a{};
    a.codes = static_cast<const uint8_t*>(codes);
    a.ldc = ld_codes;
    a.scales = scales;
    a.capacity = capacity;
    a.cols = cols;
    a.bits = bits;
    a.group = group;
    a.ngroups = cols / group;
    a.table = table;
    a.table_ld = table_ld;
    a.page_rows = static_cast<uint32_t>(page_rows);
    while ((1LL << a.page_shift) < page_rows) ++a.page_shift;
    a.page_mul = static_cast<uint32_t>((((1ULL << a.page_shift) - static_cast<uint64_t>(page_rows)) << 32) /
                                           static_cast<uint64_t>(page_rows) + 1);
    a.lengths = lengths;
    a.rows = rows;
    a.out = out;
    a.out_batch = batch > 1 ? out_batch : 0;
    a.ldo = ldo;
    a.err = err_dev;
    return run_read(a, batch, dtype, static_cast<cudaStream_t>(stream), name);
}

}  // extern "C"
