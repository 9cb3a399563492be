// The 8-bit product of narrow layers (Cin <= 256 for token rows, <= 128 for
// planes, Cout <= 256) in one pass: the tokens are quantised on their way from
// global to shared memory, so that they are read once and no codes go through
// memory. What bounds such a layer is HBM: rows * (2 Cin + 2 Cout) bytes.
//
// A CTA keeps the whole weight in shared memory and takes tiles of 128 tokens:
//   1. the tile, loaded into registers during the previous tile's epilogue, is
//      quantised and written as a swizzled K-major operand (token rows: SG
//      lanes share a row and its maximum is log2(SG) shuffles; planes: a lane
//      is a pixel and holds all its channels);
//   2. one thread issues the MMAs (M = 128, N = NT, K = 32; int32 in TMEM);
//   3. the next tile's loads are issued;
//   4. epilogue: a lane is a token; scales, bias, SimpleGate in FP32, a staging
//      tile per warp and a TMA store (or direct stores, see linear8_tc.cu).
// Two to four CTAs per SM overlap each other's phases; there is one CTA-wide
// barrier per tile. 522240 x 64 -> 128 takes 43 us on the device (4.7 TB/s; its
// writes alone would take 35 at the rate of a plain fill).
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <string>

#include "denoiser_b200.h"
#include "launch.cuh"
#include "linear8.cuh"
#include "linear8.h"
#include "quant.cuh"
#include "status.h"

namespace dnb {
namespace {

constexpr int kRows = 128;

struct FusedArgs {
    ProductArgs p;
    const __half* x;
    int64_t ldx;     // row stride (token rows)
    int m_tiles;
    int vec_in;      // token rows: 16-byte loads of x are aligned
    int tma_out;
    int pairs;       // direct stores: pairs of outputs are 4-byte aligned
    int unit;        // columns of a staging tile (tma_out)
};

// Shapes of one instantiation: SG lanes per token row, i.e. up to 8 SG input
// channels.
template <bool PLANES, int SG, int NT>
struct Shape {
    // Planes: a lane per pixel. Token rows: as many warps as keep 8 vectors a
    // lane in registers (130560 x 256 -> 256: 36 us with 16 warps, 57 with 8;
    // 522240 x 64 -> 128: 42 us with 4, 45 with 8), and 8 where TMEM leaves
    // room for two CTAs only (130560 x 128 -> 256: 29 us, 49 with 4).
    static constexpr int kWarps = PLANES ? 4 : SG == 32 ? 16 : SG == 16 || NT == 256 ? 8 : 4;
    static constexpr int kGroups = kWarps / 4;                              // warps that share a TMEM quadrant
    static constexpr int kThreads = kWarps * 32;
    static constexpr int kVecs = PLANES ? SG : (kRows / kWarps) * SG / 32;  // 8-value vectors of a lane
    static constexpr int kBytesK = SG <= 4 ? 32 : SG * 8;                   // bytes of an operand row
    static constexpr int kSpan = kBytesK < 128 ? kBytesK : 128;             // its swizzle span
    static constexpr int kA = kRows * kBytesK, kB = NT * kBytesK;
    static constexpr int kStg = kWarps * 32 * 128;
    // The tile's tokens as they came, where they are loaded as one run, come
    // behind that; up to kRunK channels, so that a CTA stays below 223 KB.
    static constexpr int kSmem = 1024 + kA + kB + kStg;
    static constexpr int kRoomK = (228352 - kSmem) / (kRows * 2);
    static constexpr int kRunK = PLANES ? 0 : kRoomK < 8 * SG ? kRoomK : 8 * SG;
    static constexpr int smem(int run_k) { return kSmem + kRows * 2 * run_k; }
};

// RUN: token rows one behind the other that are no multiple of 16 bytes, loaded
// as one run.
template <typename T, bool PLANES, int SG, int NT, bool RUN>
__global__ void __launch_bounds__(Shape<PLANES, SG, NT>::kThreads) product_fused_kernel(
    const __grid_constant__ FusedArgs g, const __grid_constant__ CUtensorMap out_map) {
    using S = Shape<PLANES, SG, NT>;
    using Q = QuantOf<__half>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    __shared__ uint64_t bar, bar_end;
    __shared__ uint32_t tslot;
    __shared__ volatile int s_abort;
    __shared__ float s_x[2][kRows];       // the tokens' scales, of this and the previous tile
    __shared__ __align__(16) float2 s_par[NT];  // scale and bias of each weight row, read two at a time
    const ProductArgs& p = g.p;
    const int tid = threadIdx.x, warp = warp_index(), lane = tid & 31;
    uint8_t* sa = smem;
    uint8_t* sb = smem + S::kA;
    uint8_t* stg = smem + S::kA + S::kB + warp * 32 * 128;
    const int half = NT / 2;
    const int K = p.seg_c;

    constexpr uint32_t kCols = NT < 32 ? 32 : NT;
    if (warp == 0) {
        tmem_alloc(&tslot, kCols);
        tmem_relinquish();
    }
    if (tid == 0) {
        mbar_init(&bar, 1);
        mbar_init(&bar_end, 1);
        s_abort = 0;
        fence_mbar_init();
        if (g.tma_out) prefetch_tmap(&out_map);
    }
    // The weight, as rows of the second operand (gated layers: the first
    // factors' rows in the lower half of the tile, the second ones' above).
    auto weight_row = [&](int r) { return !p.gate ? (r < p.cout ? r : -1)
                                                  : (r < half ? (r < p.n_out ? r : -1)
                                                              : (r - half < p.n_out ? p.n_out + r - half : -1)); };
    for (int i = tid; i < NT * (S::kBytesK / 16); i += S::kThreads) {
        const int r = i / (S::kBytesK / 16), j = i % (S::kBytesK / 16);
        const int c = weight_row(r);
        const uint4 v = c >= 0 && j * 16 < p.ldw ? *reinterpret_cast<const uint4*>(p.w + c * p.ldw + j * 16)
                                                 : make_uint4(0, 0, 0, 0);
        constexpr int kPer = S::kSpan / 16;
        *reinterpret_cast<uint4*>(sb + (j / kPer) * (NT * S::kSpan) + sw_offset(r, j % kPer, S::kSpan)) = v;
    }
    for (int r = tid; r < NT; r += S::kThreads) s_par[r] = __ldg(p.par + (p.gate && r >= half ? p.npad + r - half : r));
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tslot;
    pdl_trigger();
    pdl_wait();

    typename Q::Vec v[S::kVecs];
    const int sub = lane / SG, l = lane % SG;
    constexpr int kPer = 32 / SG;             // token rows a warp loads at a time
    constexpr int kWarpRows = kRows / S::kWarps;
    auto load = [&](int tile) {
        if (PLANES) {
            const int64_t m = static_cast<int64_t>(tile) * kRows + warp * 32 + lane;
            const bool in = m < p.rows;
            const int64_t img = in ? m / p.ldo : 0;
            const __half* src = g.x + img * K * p.ldo + (in ? m - img * p.ldo : 0);
#pragma unroll
            for (int i = 0; i < S::kVecs; ++i) {
                uint32_t w[4];
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    const int k = i * 8 + h * 2;
                    const uint32_t lo = in && k < K ? __half_as_ushort(__ldg(src + k * p.ldo)) : 0u;
                    const uint32_t hi = in && k + 1 < K ? __half_as_ushort(__ldg(src + (k + 1) * p.ldo)) : 0u;
                    w[h] = lo | (hi << 16);
                }
                v[i].v = make_uint4(w[0], w[1], w[2], w[3]);
            }
        } else if (RUN) {
            // This warp's rows are one run of kWarpRows K values from a 16-byte boundary on.
            const int64_t first = (static_cast<int64_t>(tile) * kRows + warp * kWarpRows) * K;
            const int64_t end = p.rows * K;
#pragma unroll
            for (int i = 0; i < S::kVecs; ++i) {
                const int f = (lane + 32 * i) * 8;
                const int64_t at = first + f;
                v[i] = f >= kWarpRows * K || at >= end ? Q::zero()
                       : at + 8 <= end                 ? Q::load(g.x + at)
                                                       : Q::load_some(g.x + at, static_cast<int>(end - at));
            }
        } else {
            const int64_t m0 = static_cast<int64_t>(tile) * kRows + warp * kWarpRows + sub;
            const bool in = l * 8 < K;
#pragma unroll
            for (int i = 0; i < S::kVecs; ++i) {
                const int64_t m = m0 + i * kPer;
                const __half* src = g.x + m * g.ldx + l * 8;
                v[i] = !in || m >= p.rows ? Q::zero() : g.vec_in ? Q::load(src) : Q::load_some(src, min(8, K - l * 8));
            }
        }
    };
    // Code bytes of 16 channels of tile row r in the A operand.
    auto a_chunk = [&](int r, int j) {
        constexpr int kPerSpan = S::kSpan / 16;
        return sa + (j / kPerSpan) * (kRows * S::kSpan) + sw_offset(r, j % kPerSpan, S::kSpan);
    };

    const uint64_t ad0 = sdesc_kmajor_sw(smem_u32(sa), S::kSpan), bd0 = sdesc_kmajor_sw(smem_u32(sb), S::kSpan);
    const int steps = (K + 31) / 32;
    const int out_cols = p.gate ? half : NT;
    T* out = static_cast<T*>(p.out);
    int n = 0;
    if (static_cast<int>(blockIdx.x) < g.m_tiles) load(blockIdx.x);
    for (int tile = blockIdx.x; tile < g.m_tiles; tile += gridDim.x, ++n) {
        float* sx = s_x[n & 1];
        if (PLANES) {
            uint32_t mag = Q::mag(v[0]);
#pragma unroll
            for (int i = 1; i < S::kVecs; ++i) mag = max(mag, Q::mag(v[i]));
            const GroupScale q = group_scale<__half>(mag, 127.f);
            const bool rare = __any_sync(0xffffffffu, q.rare);
            const int r = warp * 32 + lane;
#pragma unroll
            for (int i = 0; i < S::kVecs; i += 2) {
                const uint2 lo = codes8<__half>(v[i], q, rare), hi = codes8<__half>(v[i + 1], q, rare);
                *reinterpret_cast<uint4*>(a_chunk(r, i / 2)) = make_uint4(lo.x, lo.y, hi.x, hi.y);
            }
            sx[r] = q.s;
        } else {
            if (RUN) {  // from the run to a lane's vectors of its rows
                uint8_t* raw = smem + S::kA + S::kB + S::kStg + warp * kWarpRows * K * 2;
                __syncwarp();
#pragma unroll
                for (int i = 0; i < S::kVecs; ++i)
                    if ((lane + 32 * i) * 8 < kWarpRows * K) *reinterpret_cast<uint4*>(raw + (lane + 32 * i) * 16) = v[i].v;
                __syncwarp();
#pragma unroll
                for (int i = 0; i < S::kVecs; ++i)
                    v[i] = l * 8 < K ? Q::load_some(reinterpret_cast<const __half*>(raw) + (i * kPer + sub) * K + l * 8,
                                                    min(8, K - l * 8))
                                     : Q::zero();
            }
            auto scale_of = [&](int i) {
                uint32_t mag = Q::mag(v[i]);
#pragma unroll
                for (int d = SG / 2; d > 0; d >>= 1) mag = max(mag, __shfl_xor_sync(0xffffffffu, mag, d));
                return group_scale<__half>(mag, 127.f);
            };
            auto code_at = [&](int i) {
                return reinterpret_cast<uint2*>(a_chunk(warp * kWarpRows + i * kPer + sub, l / 2) + (l & 1) * 8);
            };
            // One vote for the warp's rows (a fifth of 32 rows has a rare one).
            float r[S::kVecs];
            bool rare = false;
#pragma unroll
            for (int i = 0; i < S::kVecs; ++i) {
                const GroupScale q = scale_of(i);
                r[i] = q.r;
                rare = rare || q.rare;
                if (l == 0) sx[warp * kWarpRows + i * kPer + sub] = q.s;
            }
            if (!__any_sync(0xffffffffu, rare)) {
#pragma unroll
                for (int i = 0; i < S::kVecs; ++i) *code_at(i) = codes8_fast(v[i], r[i]);
            } else {
#pragma unroll
                for (int i = 0; i < S::kVecs; ++i) *code_at(i) = codes8_rare<__half>(v[i], scale_of(i));
            }
        }
        fence_async_smem();
        tc_fence_before();
        __syncthreads();  // the operand is complete, and every warp is done with the previous accumulator
        if (warp == 0) {
            tc_fence_after();
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < S::kBytesK / 32; ++k)
                    if (k < steps) {
                        const uint32_t span_steps = S::kSpan / 32;
                        const uint32_t s = k / span_steps, o = 2 * (k % span_steps);
                        mma_s8(tmem, ad0 + s * ((kRows * S::kSpan) >> 4) + o, bd0 + s * ((NT * S::kSpan) >> 4) + o,
                               idesc_s8(kRows, NT), k > 0 ? 1u : 0u);
                    }
                mma_commit(&bar);
            }
            __syncwarp();
        }
        if (tile + static_cast<int>(gridDim.x) < g.m_tiles) load(tile + gridDim.x);
        // A wait that runs out marks the launch as failed and lets the CTA finish.
        wait_or_abort(&bar, n & 1, &s_abort, p.err, 0x74);
        __syncwarp();
        tc_fence_after();

        const int quad = warp & 3, group = warp >> 2;
        const int64_t m0 = static_cast<int64_t>(tile) * kRows + quad * 32;
        const int64_t row = m0 + lane;
        const bool live = row < p.rows;
        const int64_t img = PLANES && live ? row / p.ldo : 0;
        const float s = sx[quad * 32 + lane];
        const uint32_t acc = tmem + (static_cast<uint32_t>(quad * 32) << 16);
        // 32 columns from c on, scaled.
        auto scaled = [&](int c, float (&y)[32]) {
            int a[32];
            tmem_ld32(acc + c, a);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
                const float4 w = *reinterpret_cast<const float4*>(&s_par[c + i]);  // two rows' (scale, bias)
                const float2 t = ffma2(make_float2(static_cast<float>(a[i]), static_cast<float>(a[i + 1])), make_float2(s, s),
                                       make_float2(0.f, 0.f));
                const float2 z = ffma2(t, make_float2(w.x, w.z), make_float2(w.y, w.w));
                y[i] = z.x;
                y[i + 1] = z.y;
            }
        };
        const int unit = !PLANES && g.tma_out ? g.unit : 32;
        for (int c0 = 0, u = 0; c0 < out_cols && c0 < p.n_out; c0 += unit, ++u) {
            if (u % S::kGroups != group) continue;
            if (!PLANES && g.tma_out) {
                if (lane == 0) bulk_wait_read0();
                __syncwarp();
            }
            for (int c = c0; c < c0 + unit; c += 32) {
                float y[32];
                scaled(c, y);
                if (p.gate) {
                    float z[32];
                    scaled(half + c, z);
#pragma unroll
                    for (int i = 0; i < 32; ++i) y[i] *= z[i];
                }
                if (PLANES) {
                    if (live) store_planes32(out + (img * p.n_out + c) * p.ldo + (row - img * p.ldo), p.ldo, y, c, p.n_out);
                } else if (g.tma_out) {
                    constexpr int kVec = 16 / sizeof(T);
                    const uint32_t span = g.unit * sizeof(T);
#pragma unroll
                    for (int i = 0; i < 32; i += kVec)
                        *reinterpret_cast<uint4*>(stg + sw_offset(lane, (c - c0 + i) / kVec, span)) =
                            pack16(y + i, static_cast<T*>(nullptr));
                } else {
                    store_block32(stg, y, out, p.ldo, m0, p.rows, c, p.n_out, g.pairs);
                }
            }
            if (!PLANES && g.tma_out) {
                fence_async_smem();
                __syncwarp();
                if (lane == 0 && m0 < p.rows) {
                    tma_store_2d(&out_map, c0, static_cast<int>(m0), stg);
                    bulk_commit();
                }
            }
        }
    }
    if (!PLANES && g.tma_out && lane == 0) bulk_wait_read0();
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        if (s_abort) drain_mmas(&bar_end);
        tmem_dealloc(tmem, kCols);
    }
}

template <typename T, bool PLANES, int SG, int NT, bool RUN>
int run(FusedArgs& g, int sms, cudaStream_t s) {
    using S = Shape<PLANES, SG, NT>;
    const ProductArgs& p = g.p;
    const int out_cols = p.gate ? NT / 2 : NT;
    g.tma_out = !PLANES && tma_rows(p.out, sizeof(T), p.n_out, p.ldo);
    g.pairs = reinterpret_cast<uintptr_t>(p.out) % 4 == 0 && p.ldo % 2 == 0;
    // Staging rows of 128 bytes, or shorter ones so that every group of four
    // warps has columns to finish.
    g.unit = std::max(32, std::min<int>(128 / sizeof(T), out_cols / S::kGroups));
    CUtensorMap map{};
    if (g.tma_out)
        DN_TRY(linear8_map(&map, sizeof(T) == 2 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32,
                           sizeof(T), p.out, p.n_out, p.rows, p.ldo, g.unit, 32));
    static int resident[64] = {};
    int per_sm = 0;
    auto kernel = product_fused_kernel<T, PLANES, SG, NT, RUN>;
    const int smem = S::smem(RUN ? p.seg_c : 0);
    int fresh[64] = {};  // a run's buffer depends on Cin
    cudaError_t e = tmem_kernel_ctas(kernel, S::kThreads, smem, S::smem(RUN ? S::kRunK : 0), NT, RUN ? fresh : resident, &per_sm);
    if (e == cudaSuccess)
        e = launch_pdl(kernel, dim3(static_cast<unsigned>(std::min(g.m_tiles, per_sm * sms))), dim3(S::kThreads), smem, s, g,
                       map);
    return e == cudaSuccess ? DN_OK : dn_cuda_fail(e, "linear8: fused launch");
}

template <typename T, bool PLANES, int SG, int NT>
int run_kind(FusedArgs& g, const void* x, int sms, cudaStream_t s) {
    const bool contiguous = !g.vec_in && g.ldx == g.p.seg_c && reinterpret_cast<uintptr_t>(x) % 16 == 0;
    if constexpr (!PLANES)
        if (contiguous && g.p.seg_c <= Shape<PLANES, SG, NT>::kRunK) return run<T, PLANES, SG, NT, true>(g, sms, s);
    return run<T, PLANES, SG, NT, false>(g, sms, s);
}

template <typename T, bool PLANES, int SG>
int run_nt(FusedArgs& g, const void* x, int sms, cudaStream_t s) {
    const int need = fused_width(g.p);
    if (need <= 32) return run_kind<T, PLANES, SG, 32>(g, x, sms, s);
    if (need <= 64) return run_kind<T, PLANES, SG, 64>(g, x, sms, s);
    if (need <= 128) return run_kind<T, PLANES, SG, 128>(g, x, sms, s);
    return run_kind<T, PLANES, SG, 256>(g, x, sms, s);
}

template <typename T, bool PLANES>
int run_k(FusedArgs& g, const void* x, int sms, cudaStream_t s) {
    const int K = g.p.seg_c;
    if (K <= 16) return run_nt<T, PLANES, 2>(g, x, sms, s);
    if (K <= 32) return run_nt<T, PLANES, 4>(g, x, sms, s);
    if (K <= 64) return run_nt<T, PLANES, 8>(g, x, sms, s);
    if constexpr (!PLANES)
        if (K > 128) return run_nt<T, PLANES, 32>(g, x, sms, s);
    return run_nt<T, PLANES, 16>(g, x, sms, s);
}

}  // namespace

bool product_fused_takes(const ProductArgs& a) {
    return fused_width(a) <= 256 && a.segs == 1 && a.seg_c <= (a.planes ? 128 : 256);
}

int launch_product_fused(const ProductArgs& a, const void* x, int64_t ldx, int out_dtype, int sms, cudaStream_t s) {
    FusedArgs g{};
    g.p = a;
    g.x = static_cast<const __half*>(x);
    g.ldx = ldx;
    g.vec_in = a.seg_c % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0 && ldx % 8 == 0;
    g.m_tiles = static_cast<int>((a.rows + kRows - 1) / kRows);
    if (a.planes) return run_k<__half, true>(g, x, sms, s);
    return out_dtype == 1 ? run_k<__half, false>(g, x, sms, s) : run_k<float, false>(g, x, sms, s);
}

}  // namespace dnb
