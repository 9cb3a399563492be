// The 8-bit product on the tensor cores (tcgen05 kind::i8, int32 in TMEM):
//
//   y[m, n] = s_w[n] sum_t s_x[t, m] (sum_c q_x[t, m, c] q_w[n, t, c]) + bias[n]
//
// A persistent, warp-specialised kernel (352 threads, one CTA per SM) over
// tiles of 128 tokens x NT channels:
//   warp 8      TMA loads of the token codes: boxes of 128 rows x KC bytes,
//               swizzled by KC = 128 / 64 / 32 (the least that holds a
//               segment); bytes behind a segment read as zeros;
//   warp 9      TMA loads of the weight rows (gated layers: the two halves'
//               rows, so that a tile has both factors of its outputs);
//   warp 10     one thread issues the MMAs (M = 128, N = NT, K = 32), a TMEM
//               accumulator of NT columns per segment, a ring of them, so that
//               epilogues overlap the next products;
//   warps 0-7   epilogue: a lane is a token; scales, bias, SimpleGate in FP32,
//               then through a swizzled staging tile per warp and a TMA store
//               (rows and planes whose address or stride does not allow it
//               are stored by the lanes).
// A segment's int32 sum is exact; it is scaled once, in FP32: layers with
// segments keep their columns' running sums in registers (NT <= 128: 64 a
// lane). Every wait is bounded.
//
// Measured on the device: 8192 x 4096 -> 4096 116 us with its quantisation (2.37
// POP/s; the product alone 98 us, tensor pipe 75% busy; copies into shared memory,
// 48 KB a chunk, and the power limit bind), the fusion of 5 cached frames of
// 522240 x 64 -> 64 61 us (4.0 TB/s; no pipe is full: issue slots 47%, DRAM 40%,
// so latency binds, of the epilogue's chain of accumulator load, wait and sums
// in two warps a scheduler).
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <string>
#include <type_traits>

#include "denoiser_b200.h"
#include "launch.cuh"
#include "linear8.cuh"
#include "linear8.h"
#include "sm100.cuh"
#include "status.h"

namespace dnb {

PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder();  // gemm_tc.cu

namespace {

constexpr int kRows = 128;
constexpr int kThreads = 352;
constexpr int kEpiWarps = 8;
constexpr int kStageA = kRows * 128;
constexpr int kStgWarp = 32 * 128;  // staging tile of an epilogue warp: 32 rows x 128 bytes

// Shared memory: the ring of operand stages (at most kStages), the resident
// weight if there is one, the epilogue's staging tiles.
template <int NT>
struct Plan {
    static constexpr int kStage = kStageA + NT * 128;
    static constexpr int kStages = NT == 256 ? 4 : NT == 128 ? 5 : 8;
    static constexpr int kRing = NT == 256 ? 4 * kStage : NT == 128 ? 5 * kStage : 6 * (kStageA + 64 * 128);
    static constexpr int kBytes = 1024 + kRing + kEpiWarps * kStgWarp;
};

struct Maps {
    CUtensorMap a, b, out;
};

struct TcArgs {
    ProductArgs p;
    int kc, chunks;      // bytes of a K chunk, chunks of a segment
    int m_tiles, n_tiles;
    int box_rows;        // token rows of a load: 128, or fewer of a single tile
    int tma_out;         // 1: staged TMA stores
    int unit;            // columns of a staging tile
    int resident;        // the whole weight stays in shared memory (one column tile)
    int stage, stages;   // bytes and number of the ring's stages
    int units;           // K chunks of a stage: 1, or (resident weight) all of a tile's
    int seg_full;        // accumulators are handed over one by one, not a tile's together
    int pairs;           // direct stores of FP16 rows: pairs are 4-byte aligned
    int tma_planes;      // planes by TMA: boxes of 32 channels x 32 pixels of one image
};

// 32 columns from c on, (scale, bias) from par.
__device__ __forceinline__ void finish32(const float2* par, float (&y)[32]) {
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
        const float4 w = __ldg(reinterpret_cast<const float4*>(par + i));
        const float2 z = ffma2(make_float2(y[i], y[i + 1]), make_float2(w.x, w.z), make_float2(w.y, w.w));
        y[i] = z.x, y[i + 1] = z.y;
    }
}

// 32 columns of tokens some of which have a large scale (see kLargeScale).
__device__ __forceinline__ void finish32_large(const float2* par, const int (&a)[32], float s, float (&y)[32]) {
    const bool large = s >= kLargeScale;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        const float2 w = __ldg(par + i);
        y[i] = fmaf(static_cast<float>(a[i]) * (large ? w.x : s), large ? s : w.x, w.y);
    }
}

template <typename T, int NT, bool SEG>
__global__ void __launch_bounds__(kThreads, 1) product_tc_kernel(const __grid_constant__ TcArgs g,
                                                                 const __grid_constant__ Maps maps) {
    using P = Plan<NT>;
    const int kSt = g.stages;  // stages of the ring
    constexpr int kVec = 16 / sizeof(T);      // values of 16 bytes
    constexpr int kAcc = SEG ? 512 / NT : NT == 256 ? 2 : 4;  // accumulators of the ring
    constexpr uint32_t kCols = kAcc * NT;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    __shared__ uint64_t bar_full[P::kStages], bar_empty[P::kStages], bar_b, bar_acc_full[kAcc], bar_acc_empty[kAcc], bar_tile[8],
        bar_end;
    // A tile's scales, [segment][token] per epilogue warp.
    __shared__ float s_scale[SEG ? kEpiWarps : 1][SEG ? kMaxSegments : 1][32];
    __shared__ uint32_t tslot;
    __shared__ volatile int s_abort;
    const ProductArgs& p = g.p;
    const int tid = threadIdx.x, warp = warp_index(), lane = tid & 31;
    const int tiles = g.m_tiles * g.n_tiles;

    if (warp == 10) {
        tmem_alloc(&tslot, kCols);
        tmem_relinquish();
    }
    if (tid == 0) {
        for (int s = 0; s < kSt; ++s) {
            mbar_init(&bar_full[s], g.resident ? 1 : 2);
            mbar_init(&bar_empty[s], 1);
        }
        mbar_init(&bar_b, 1);
        mbar_init(&bar_end, 1);
        // The ring holds at most four tiles of two segments, so that a tile's
        // barrier is waited for before it comes round again.
        for (int b = 0; b < 8; ++b) mbar_init(&bar_tile[b], 1);
        for (int b = 0; b < kAcc; ++b) {
            mbar_init(&bar_acc_full[b], 1);
            mbar_init(&bar_acc_empty[b], kEpiWarps);
        }
        s_abort = 0;
        fence_mbar_init();
        prefetch_tmap(&maps.a);
        prefetch_tmap(&maps.b);
        if (g.tma_out || g.tma_planes) prefetch_tmap(&maps.out);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tslot;
    pdl_trigger();
    if (warp != 9) pdl_wait();  // the weights (warp 9) were there before; codes, scales and `out` belong to earlier kernels

    constexpr int half = NT / 2;
    const int out_cols = p.gate ? half : NT;  // output columns of a tile

    // Whole warps run the loops of warps 8 to 10 and elect a lane in them, which
    // every lane has to reach. Where a wait ends at another role's timeout the
    // lanes' answers (ok) may differ, so a lane that has given up goes through
    // the rest of the tile, waiting and loading no more (what it multiplies then
    // is wasted), and the warp leaves together. (A vote at every wait: 5 x 2088960 x
    // 32 -> 32 218.4 us, 215 this way.)
    auto leaves = [](bool ok) { return !__all_sync(0xffffffffu, ok); };
    uint8_t* b_res = smem + kSt * g.stage;  // resident weight: its chunks one behind the other
    const int seg_c = p.seg_c, segs = p.segs, chunks = g.chunks, kc = g.kc, units = g.units, stage = g.stage;
    if (warp == 9 && g.resident) {
        if (elect_one()) {
            mbar_arrive_expect_tx(&bar_b, static_cast<uint32_t>(segs * chunks * NT * kc));
            for (int i = 0; i < segs * chunks; ++i) {
                uint8_t* sb = b_res + i * (NT * kc);
                const int k = (i / chunks) * p.seg_p + (i % chunks) * kc;
                tma_load_2d(sb, &maps.b, k, 0, &bar_b);
                if (p.gate) tma_load_2d(sb + half * kc, &maps.b, k, p.n_out, &bar_b);
            }
            // It has landed before this CTA leaves, whatever became of the others
            // (another role's timeout ends the first wait at once).
            if (!wait_or_abort(&bar_b, 0, &s_abort, p.err, 0x77)) mbar_wait(&bar_b, 0, 100000000ull);
        }
    } else if (warp == 8) {
        const uint32_t bytes = static_cast<uint32_t>(g.box_rows * kc * units);
        int filled = 0, left = 0, s = 0;  // stages begun, chunks that the current one still takes
        uint32_t ph = 1;
        bool ok = true;
        for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
            const int m0 = (tile / g.n_tiles) * kRows;
            for (int t = 0; t < segs; ++t) {
                const int row = static_cast<int>(p.arow[t]) + m0;
                for (int j = 0; j < chunks; ++j) {
                    if (left == 0) {
                        ok = ok && wait_or_abort(&bar_empty[s], ph, &s_abort, p.err, 0x70);
                        if (elect_one() && ok) mbar_arrive_expect_tx(&bar_full[s], bytes);
                        left = units;
                        if (ok) ++filled;
                    }
                    uint8_t* sa = smem + s * stage + (units - left) * (kRows * kc);
                    if (elect_one() && ok) tma_load_2d(sa, &maps.a, j * kc, row, &bar_full[s]);
                    if (--left == 0 && ++s == kSt) s = 0, ph ^= 1;
                }
            }
            if (leaves(ok)) break;
        }
        // After a wait that ran out: the copies in flight land before the CTA leaves.
        if (!ok)
            for (int k = max(0, filled - kSt); k < filled; ++k) mbar_wait(&bar_full[k % kSt], (k / kSt) & 1, 100000000ull);
    } else if (warp == 9) {
        const uint32_t bytes = static_cast<uint32_t>(NT * kc);
        int filled = 0, s = 0;
        uint32_t ph = 1;
        bool ok = true;
        for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
            const int n0 = (tile % g.n_tiles) * out_cols;
            for (int t = 0; t < segs; ++t)
                for (int j = 0; j < chunks; ++j) {
                    // The ring filled up once ahead of the earlier kernels; what
                    // empties it waits for them, however long they take.
                    if (filled == kSt) pdl_wait();
                    ok = ok && wait_or_abort(&bar_empty[s], ph, &s_abort, p.err, 0x70);
                    uint8_t* sb = smem + s * stage + kStageA;
                    const int k = t * p.seg_p + j * kc;
                    if (elect_one() && ok) {
                        mbar_arrive_expect_tx(&bar_full[s], bytes);
                        tma_load_2d(sb, &maps.b, k, n0, &bar_full[s]);
                        if (p.gate) tma_load_2d(sb + half * kc, &maps.b, k, p.n_out + n0, &bar_full[s]);
                    }
                    if (ok) ++filled;
                    if (++s == kSt) s = 0, ph ^= 1;
                }
            if (leaves(ok)) break;
        }
        if (!ok)
            for (int k = max(0, filled - kSt); k < filled; ++k) mbar_wait(&bar_full[k % kSt], (k / kSt) & 1, 100000000ull);
    } else if (warp == 10) {
        constexpr uint32_t idesc = idesc_s8(kRows, NT);
        const uint32_t sm0 = smem_u32(smem);
        const uint64_t ad0 = sdesc_kmajor_sw(sm0, kc);
        const uint64_t bd0 = sdesc_kmajor_sw(g.resident ? smem_u32(b_res) : sm0 + kStageA, kc);
        const uint32_t a_unit = (kRows * kc) >> 4;                         // from chunk to chunk of a stage
        const uint32_t b_unit = g.resident ? (NT * kc) >> 4 : 0;           // of the resident weight
        const uint32_t b_stage = g.resident ? 0 : stage >> 4;              // from stage to stage
        int s = 0, b = 0, n = 0, left = 0;
        uint32_t ph = 0, acc_ph = 1;
        uint64_t ad = ad0;
        bool ok = !g.resident || wait_or_abort(&bar_b, 0, &s_abort, p.err, 0x78);
        for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, ++n) {
            uint64_t bd = bd0;  // of the chunk, but for the stage
            for (int t = 0; t < segs; ++t) {
                ok = ok && wait_or_abort(&bar_acc_empty[b], acc_ph, &s_abort, p.err, 0x71);
                tc_fence_after();
                const uint32_t acc = tmem + b * NT;
                int steps_left = (seg_c + 31) / 32;
                for (int j = 0; j < chunks; ++j) {
                    if (left == 0) {
                        ok = ok && wait_or_abort(&bar_full[s], ph, &s_abort, p.err, 0x72);
                        tc_fence_after();
                        left = units;
                        ad = ad0 + static_cast<uint32_t>(s * (stage >> 4));
                    }
                    const uint64_t bs = bd + s * b_stage;
                    if (elect_one()) {
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (k < steps_left && k * 32 < kc)
                                mma_s8(acc, ad + 2 * k, bs + 2 * k, idesc, (j > 0 || k > 0) ? 1u : 0u);
                        if (left == 1) mma_commit(&bar_empty[s]);
                        if (j == chunks - 1) {
                            if (g.seg_full)
                                mma_commit(&bar_acc_full[b]);
                            else if (t == segs - 1)
                                mma_commit(&bar_tile[n & 7]);
                        }
                    }
                    __syncwarp();
                    steps_left -= kc / 32;
                    ad += a_unit;
                    bd += b_unit;
                    if (--left == 0 && ++s == kSt) s = 0, ph ^= 1;
                }
                if (++b == kAcc) b = 0, acc_ph ^= 1;
            }
            if (leaves(ok)) break;
        }
        if (leaves(ok)) drain_mmas(&bar_end);
    } else {
        const int quad = warp & 3, group = warp >> 2;
        uint8_t* stg = smem + P::kRing + warp * kStgWarp;
        const uint32_t lane_base = tmem + (static_cast<uint32_t>(quad * 32) << 16);
        T* out = static_cast<T*>(p.out);
        // 32 finished values of a lane's row, tile columns c .. c + 31; in a
        // staging tile that starts at column c0.
        auto stage32 = [&](const float (&y)[32], int c, int c0) {
            const uint32_t span = g.unit * sizeof(T);
#pragma unroll
            for (int i = 0; i < 32; i += kVec)
                *reinterpret_cast<uint4*>(stg + sw_offset(lane, (c - c0 + i) / kVec, span)) =
                    pack16(y + i, static_cast<T*>(nullptr));
        };
        auto store32 = [&](const float (&y)[32], int c, int64_t row, int64_t img) {
            if (!p.planes)
                store_block32(stg, y, out, p.ldo, row - lane, p.rows, c, p.n_out, g.pairs);
            else if (row < p.rows)
                store_planes32(out + (img * p.n_out + c) * p.ldo + (row - img * p.ldo), p.ldo, y, c, p.n_out);
        };
        auto stage_free = [&]() {
            if (lane == 0) bulk_wait_read0();
            __syncwarp();
        };
        auto stage_out = [&](int c, int64_t m0) {
            fence_async_smem();
            __syncwarp();
            if (lane == 0 && m0 < p.rows) {
                tma_store_2d(&maps.out, c, static_cast<int>(m0), stg);
                bulk_commit();
            }
        };
        auto full_wait = [&](uint64_t* bar, int use) {
            const bool ok = lane == 0 ? wait_or_abort(bar, use & 1, &s_abort, p.err, 0x73) : true;
            const bool all = __shfl_sync(0xffffffffu, ok, 0);
            tc_fence_after();
            return all;
        };
        auto acc_done = [&](int q) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar_acc_empty[q % kAcc]);
        };
        // The scales of a lane's token, loaded a tile ahead: their latency would
        // otherwise show in every tile.
        constexpr int kScales = SEG ? kMaxSegments : 1;
        float next[kScales];
        auto load_scales = [&](int tile) {
            const int64_t row = static_cast<int64_t>(tile / g.n_tiles) * kRows + quad * 32 + lane;
#pragma unroll
            for (int t = 0; t < kScales; ++t)
                next[t] = t < p.segs && tile < tiles && row < p.rows ? __ldg(p.as + p.arow[t] + row) : 0.f;
        };
        int q = 0, n = 0;
        uint32_t boxes = 0;
        load_scales(blockIdx.x);
        for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, ++n) {
            const float s = next[0];
            [[maybe_unused]] bool large = false;
            if constexpr (SEG) {
#pragma unroll
                for (int t = 0; t < kScales; ++t) s_scale[warp][t][lane] = next[t];  // read by this lane alone
#pragma unroll
                for (int t = 0; t < kScales; ++t) large = large || next[t] >= kLargeScale;
            }
            load_scales(tile + gridDim.x);
            const int64_t m0 = static_cast<int64_t>(tile / g.n_tiles) * kRows + quad * 32;
            const int n0 = (tile % g.n_tiles) * out_cols;
            const int64_t row = m0 + lane;
            const int64_t img = p.planes && row < p.rows ? row / p.ldo : 0;
            if constexpr (SEG) {
                // A warp takes 32-column blocks: NT/2 columns of its group of
                // warps, or (gated, NT = 128) 32 of each factor.
                constexpr int kBlocks = NT / 64;
                float y[kBlocks][32];
                int col[kBlocks];
#pragma unroll
                for (int k = 0; k < kBlocks; ++k) col[k] = p.gate ? k * half + group * 32 : group * half + k * 32;
                auto par_of = [&](int k) { return p.par + (p.gate ? k * p.npad + n0 + group * 32 : n0 + col[k]); };
                bool ok = g.seg_full || full_wait(&bar_tile[n & 7], n >> 3);
                if (!ok) break;
#pragma unroll
                for (int k = 0; k < kBlocks; ++k)
#pragma unroll
                    for (int i = 0; i < 32; ++i) y[k][i] = 0.f;
                // The sums of the segments, scaled; any_large: a token of the warp
                // has a large scale in one of them.
                auto add_segments = [&](auto any_large) {
#pragma unroll 1
                    for (int t = 0; t < p.segs; ++t) {
                        const float st = s_scale[warp][t][lane];
                        if (g.seg_full && !(ok = full_wait(&bar_acc_full[q % kAcc], q / kAcc))) break;
#pragma unroll
                        for (int k = 0; k < kBlocks; ++k) {
                            int a[32];
                            tmem_ld32(lane_base + (q % kAcc) * NT + col[k], a);
                            tmem_ld_wait();
                            const float2 st2 = make_float2(st, st);
#pragma unroll
                            for (int i = 0; i < 32; i += 2) {
                                float2 v = make_float2(static_cast<float>(a[i]), static_cast<float>(a[i + 1]));
                                if constexpr (any_large) {
                                    const float2* par = par_of(k) + i;
                                    if (large) v.x *= __ldg(par).x, v.y *= __ldg(par + 1).x;
                                }
                                const float2 z = ffma2(v, st2, make_float2(y[k][i], y[k][i + 1]));
                                y[k][i] = z.x, y[k][i + 1] = z.y;
                            }
                        }
                        acc_done(q);
                        ++q;
                    }
                };
                const bool any_large = __any_sync(0xffffffffu, large);
                if (any_large)
                    add_segments(std::true_type{});
                else
                    add_segments(std::false_type{});
                if (!ok) break;
#pragma unroll
                for (int k = 0; k < kBlocks; ++k) {
                    if (any_large) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            const float2 w = __ldg(par_of(k) + i);
                            y[k][i] = fmaf(y[k][i], large ? 1.f : w.x, w.y);
                        }
                    } else {
                        finish32(par_of(k), y[k]);
                    }
                }
                if (p.gate) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) y[0][i] *= y[kBlocks - 1][i];
                }
#pragma unroll
                for (int k = 0; k < kBlocks; ++k) {
                    const int c = n0 + (p.gate ? group * 32 : col[k]);
                    if ((k > 0 && p.gate) || c >= p.n_out) continue;
                    if (g.tma_out) {
                        stage_free();
                        stage32(y[k], c, c);
                        stage_out(c, m0);
                    } else {
                        store32(y[k], c, row, img);
                    }
                }
            } else {
                if (!full_wait(&bar_acc_full[q % kAcc], q / kAcc)) break;
                const uint32_t acc = lane_base + (q % kAcc) * NT;
                const bool large = __any_sync(0xffffffffu, s >= kLargeScale);
                auto scaled = [&](int c, const float2* par, float (&y)[32]) {
                    int a[32];
                    tmem_ld32(acc + c, a);
                    tmem_ld_wait();
                    if (large) {
                        finish32_large(par, a, s, y);
                        return;
                    }
#pragma unroll
                    for (int i = 0; i < 32; ++i) y[i] = static_cast<float>(a[i]) * s;
                    finish32(par, y);
                };
                if constexpr (sizeof(T) == 2) {
                    if (g.tma_planes) {
                        // As in linear8_planes.cu: lane t has, of pixels 8 i + t / 4,
                        // channels 8 k + 2 (t % 4) and the next.
                        const int j4 = lane & 3, px = lane >> 2;
                        float sp[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) sp[i] = __shfl_sync(0xffffffffu, s, 8 * i + px);
                        auto block = [&](int c, const float2* par, float2 (&y)[4][4]) {
                            int a[2][16];
                            tmem_ld_16x32(acc + c, a[0]);
                            tmem_ld_16x32(acc + (16u << 16) + c, a[1]);
                            tmem_ld_wait();
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                const float4 w = __ldg(reinterpret_cast<const float4*>(par + 8 * k + 2 * j4));
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    const int* v = &a[i >> 1][4 * k + 2 * (i & 1)];
                                    const float2 t = ffma2(make_float2(static_cast<float>(v[0]), static_cast<float>(v[1])),
                                                           make_float2(sp[i], sp[i]), make_float2(0.f, 0.f));
                                    y[k][i] = ffma2(t, make_float2(w.x, w.z), make_float2(w.y, w.w));
                                }
                            }
                        };
                        const int64_t image = m0 / p.ldo;
                        for (int c = 0, u = n & 1; c < out_cols; c += 32, ++u) {
                            if ((u & 1) != group || n0 + c >= p.n_out) continue;
                            float2 y[4][4];
                            block(c, p.par + n0 + c, y);
                            if (p.gate) {
                                float2 z[4][4];
                                block(half + c, p.par + p.npad + n0 + c, z);
#pragma unroll
                                for (int k = 0; k < 4; ++k)
#pragma unroll
                                    for (int i = 0; i < 4; ++i) y[k][i].x *= z[k][i].x, y[k][i].y *= z[k][i].y;
                            }
                            // Two boxes take turns in the staging tile.
                            uint8_t* box = stg + (boxes++ & 1) * (32 * 64);
                            if (lane == 0) bulk_wait_read1();
                            __syncwarp();
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                stmatrix4_trans(smem_u32(box) + sw_offset(8 * k + (lane & 7), lane >> 3, 64),
                                                pack_half2(y[k][0].x, y[k][0].y), pack_half2(y[k][1].x, y[k][1].y),
                                                pack_half2(y[k][2].x, y[k][2].y), pack_half2(y[k][3].x, y[k][3].y));
                            fence_async_smem();
                            __syncwarp();
                            if (lane == 0) {
                                if (m0 < p.rows)
                                    tma_store_3d(&maps.out, static_cast<int>(m0 - image * p.ldo), n0 + c,
                                                 static_cast<int>(image), box);
                                bulk_commit();
                            }
                        }
                        acc_done(q);
                        ++q;
                        continue;
                    }
                }
                // The two groups of four warps take the tile's runs of `unit`
                // columns in turn.
                for (int c0 = 0, u = n & 1; c0 < out_cols; c0 += g.unit, ++u) {
                    if ((u & 1) != group || n0 + c0 >= p.n_out) continue;
                    if (g.tma_out) stage_free();
                    for (int c = c0; c < c0 + g.unit; c += 32) {
                        float y[32];
                        scaled(c, p.par + n0 + c, y);
                        if (p.gate) {
                            float z[32];
                            scaled(half + c, p.par + p.npad + n0 + c, z);
#pragma unroll
                            for (int i = 0; i < 32; ++i) y[i] *= z[i];
                        }
                        if (g.tma_out)
                            stage32(y, c, c0);
                        else
                            store32(y, n0 + c, row, img);
                    }
                    if (g.tma_out) stage_out(n0 + c0, m0);
                }
                acc_done(q);
                ++q;
            }
        }
        if ((g.tma_out || g.tma_planes) && lane == 0) bulk_wait_read0();
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 10) tmem_dealloc(tmem, kCols);
}

template <typename T, int NT, bool SEG>
int run(TcArgs& g, int sms, cudaStream_t s) {
    const ProductArgs& p = g.p;
    const int out_cols = p.gate ? NT / 2 : NT;
    g.kc = p.seg_c > 64 ? 128 : p.seg_c > 32 ? 64 : 32;
    g.chunks = (p.seg_c + g.kc - 1) / g.kc;
    g.m_tiles = static_cast<int>((p.rows + kRows - 1) / kRows);
    g.n_tiles = (p.n_out + out_cols - 1) / out_cols;
    g.tma_out = !p.planes && tma_rows(p.out, sizeof(T), p.n_out, p.ldo);
    g.pairs = reinterpret_cast<uintptr_t>(p.out) % 4 == 0 && p.ldo % 2 == 0;
    // A weight of one column tile that leaves room for four stages of codes
    // stays in shared memory (5 x 522240 x 64 -> 64: 63 us, 66.5 without; 5 x
    // 2088960 x 32 -> 32: 216 and 237).
    const int64_t b_bytes = static_cast<int64_t>(p.segs) * g.chunks * NT * g.kc;
    g.resident = g.n_tiles == 1 && b_bytes <= Plan<NT>::kRing - 4 * kStageA;
    g.stage = g.resident ? kRows * g.kc : Plan<NT>::kStage;
    const int ring = Plan<NT>::kRing - static_cast<int>(g.resident ? b_bytes : 0);
    // With a resident weight all of a tile's chunks make one stage where three
    // fit: fewer waits and commits (the same layers: 66 and 237 us without).
    const int tile_bytes = p.segs * g.chunks * g.stage;
    g.units = g.resident && 3 * tile_bytes <= ring ? p.segs * g.chunks : 1;
    g.stage *= g.units;
    g.stages = std::min<int>(Plan<NT>::kStages, ring / g.stage);
    // A tile's accumulators together where the ring holds them all.
    g.seg_full = !SEG || p.segs > 512 / NT;
    // Staging tiles of 128-byte rows; 32 columns with segments (a warp's
    // blocks), and for direct stores.
    g.unit = SEG || !g.tma_out ? 32 : std::min<int>(128 / sizeof(T), out_cols);
    Maps maps{};
    // TMA takes about as long for a row that does not exist as for one that does;
    // of a single short tile only the rows that it has are loaded. The operand's
    // other rows hold what was there, and their sums are not stored.
    g.box_rows = p.rows < kRows ? static_cast<int>((p.rows + 7) / 8 * 8) : kRows;
    DN_TRY(linear8_map(&maps.a, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.a, p.seg_c, p.a_rows, p.lda, g.kc, g.box_rows));
    DN_TRY(linear8_map(&maps.b, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.w, p.ldw, p.cout, p.ldw, g.kc, p.gate ? NT / 2 : NT));
    if (g.tma_out)
        DN_TRY(linear8_map(&maps.out, sizeof(T) == 2 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32,
                           sizeof(T), p.out, p.n_out, p.rows, p.ldo, g.unit, 32));
    // A warp's 32 pixels are of one image, and the planes are what TMA can address.
    g.tma_planes = p.planes && sizeof(T) == 2 && !SEG && reinterpret_cast<uintptr_t>(p.out) % 16 == 0 && p.ldo % 8 == 0 &&
                   (p.ldo % 32 == 0 || p.rows == p.ldo);
    if (g.tma_planes) DN_TRY(linear8_planes_map(&maps.out, p.out, p.ldo, p.n_out, p.rows / p.ldo, 32, 32));
    const int64_t tiles = static_cast<int64_t>(g.m_tiles) * g.n_tiles;
    if (tiles >= (1LL << 30)) return dn_fail(DN_ERR_UNSUPPORTED, "linear8: the product has 2^30 tiles or more");
    static bool configured[64] = {};  // per device
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e == cudaSuccess && (device >= 64 || !configured[device])) {
        e = cudaFuncSetAttribute(product_tc_kernel<T, NT, SEG>, cudaFuncAttributeMaxDynamicSharedMemorySize, Plan<NT>::kBytes);
        if (e == cudaSuccess && device < 64) configured[device] = true;
    }
    if (e == cudaSuccess)
        e = launch_pdl(product_tc_kernel<T, NT, SEG>, dim3(static_cast<unsigned>(std::min<int64_t>(tiles, sms))),
                       dim3(kThreads), Plan<NT>::kBytes, s, g, maps);
    return e == cudaSuccess ? DN_OK : dn_cuda_fail(e, "linear8: product launch");
}

// The tile width that moves the least into the busiest SM's shared memory: a
// tile's operands are 128 + NT rows of every K chunk. On the device, the widths
// 32 / 64 / 128 / 256: 1000 x 1024 -> 1024 10.8 / 9.3 / 8.6 / 10.5 us, 2040 x 512
// -> 1024 12.0 / 10.2 / 9.4 / 9.8, 20000 x 300 -> 300 26.9 / 25.3 / 27.1 / 35.5,
// 1000 x 4096 -> 4096 60 / 39 / 25 / 19 (taken: 64, 128, 128, 256).
int tile_width(const ProductArgs& p, int sms, int widest) {
    const int64_t m_tiles = (p.rows + kRows - 1) / kRows;
    int best = widest;
    int64_t least = INT64_MAX;
    for (int nt = widest; nt >= (p.gate ? 64 : 32); nt >>= 1) {
        const int oc = p.gate ? nt / 2 : nt;
        const int64_t tiles = m_tiles * ((p.n_out + oc - 1) / oc), cost = (tiles + sms - 1) / sms * (kRows + nt);
        if (cost < least) least = cost, best = nt;
    }
    return best;
}

template <typename T>
int run_type(TcArgs& g, int sms, cudaStream_t s) {
    if (g.p.segs > 1) {
        // Running sums of 64 columns a lane are the most that stay in
        // registers; a gated tile needs 32 columns of each factor for both
        // groups of warps.
        return g.p.gate || tile_width(g.p, sms, 128) == 128 ? run<T, 128, true>(g, sms, s) : run<T, 64, true>(g, sms, s);
    }
    switch (tile_width(g.p, sms, 256)) {
        case 32: return run<T, 32, false>(g, sms, s);
        case 64: return run<T, 64, false>(g, sms, s);
        case 128: return run<T, 128, false>(g, sms, s);
        default: return run<T, 256, false>(g, sms, s);
    }
}

}  // namespace

int linear8_map(CUtensorMap* m, CUtensorMapDataType type, int esz, const void* base, int64_t cols, int64_t rows,
                int64_t ld, int box_cols, int box_rows) {
    auto fn = tensor_map_encoder();
    if (!fn) return dn_fail(DN_ERR_CUDA, "linear8: cuTensorMapEncodeTiled unavailable");
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld) * esz};
    const cuuint32_t box[2] = {static_cast<cuuint32_t>(box_cols), static_cast<cuuint32_t>(box_rows)};
    const cuuint32_t estr[2] = {1, 1};
    const int span = box_cols * esz;
    const CUtensorMapSwizzle swz = span == 128  ? CU_TENSOR_MAP_SWIZZLE_128B
                                   : span == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                                                : CU_TENSOR_MAP_SWIZZLE_32B;
    const CUresult r = fn(m, type, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          swz, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return dn_fail_str(DN_ERR_CUDA, "linear8: cuTensorMapEncodeTiled failed (" + std::to_string(r) + ")");
    return DN_OK;
}

int linear8_planes_map(CUtensorMap* m, const void* base, int64_t pixels, int64_t channels, int64_t images, int box_px,
                       int box_ch) {
    auto fn = tensor_map_encoder();
    if (!fn) return dn_fail(DN_ERR_CUDA, "linear8: cuTensorMapEncodeTiled unavailable");
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(pixels), static_cast<cuuint64_t>(channels),
                                static_cast<cuuint64_t>(images)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(pixels) * 2, static_cast<cuuint64_t>(pixels * channels) * 2};
    const cuuint32_t box[3] = {static_cast<cuuint32_t>(box_px), static_cast<cuuint32_t>(box_ch), 1};
    const cuuint32_t estr[3] = {1, 1, 1};
    const CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base), dims, strides, box, estr,
                          CU_TENSOR_MAP_INTERLEAVE_NONE,
                          box_px == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return dn_fail_str(DN_ERR_CUDA, "linear8: cuTensorMapEncodeTiled failed (" + std::to_string(r) + ")");
    return DN_OK;
}

int launch_product_tc(const ProductArgs& a, int out_dtype, int sms, cudaStream_t s) {
    TcArgs g{};
    g.p = a;
    return out_dtype == 1 ? run_type<__half>(g, sms, s) : run_type<float>(g, sms, s);
}

}  // namespace dnb
