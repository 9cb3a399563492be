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
//               (rows whose address or stride does not allow it, and planes,
//               are stored directly).
// A segment's int32 sum is exact; it is scaled once, in FP32: layers with
// segments keep their columns' running sums in registers (NT <= 128: 64 a
// lane). Every wait is bounded.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <string>

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

template <int NT>
struct Plan {
    static constexpr int kStage = kStageA + NT * 128;
    static constexpr int kStages = NT == 256 ? 4 : NT == 128 ? 5 : 6;
    static constexpr int kBytes = 1024 + kStages * kStage + kEpiWarps * kStgWarp;
};

struct Maps {
    CUtensorMap a, b, out;
};

struct TcArgs {
    ProductArgs p;
    int kc, chunks;      // bytes of a K chunk, chunks of a segment
    int m_tiles, n_tiles;
    int tma_out;         // 1: staged TMA stores
    int unit;            // columns of a staging tile
    int vec_out;         // direct stores: 16-byte vectors of a row are aligned
};

// 32 columns from c on, (scale, bias) from par.
__device__ __forceinline__ void finish32(const float2* par, float (&y)[32]) {
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
        const float4 w = __ldg(reinterpret_cast<const float4*>(par + i));
        y[i] = fmaf(y[i], w.x, w.y);
        y[i + 1] = fmaf(y[i + 1], w.z, w.w);
    }
}

template <typename T, int NT, bool SEG>
__global__ void __launch_bounds__(kThreads, 1) product_tc_kernel(const __grid_constant__ TcArgs g,
                                                                 const __grid_constant__ Maps maps) {
    using P = Plan<NT>;
    constexpr int kSt = P::kStages;
    constexpr int kVec = 16 / sizeof(T);      // values of 16 bytes
    constexpr int kAcc = NT == 256 ? 2 : 4;   // accumulators of the ring
    constexpr uint32_t kCols = kAcc * NT;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    __shared__ uint64_t bar_full[kSt], bar_empty[kSt], bar_acc_full[kAcc], bar_acc_empty[kAcc];
    __shared__ uint32_t tslot;
    __shared__ volatile int s_abort;
    const ProductArgs& p = g.p;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int tiles = g.m_tiles * g.n_tiles;

    if (warp == 10) {
        tmem_alloc(&tslot, kCols);
        tmem_relinquish();
    }
    if (tid == 0) {
        for (int s = 0; s < kSt; ++s) {
            mbar_init(&bar_full[s], 2);
            mbar_init(&bar_empty[s], 1);
        }
        for (int b = 0; b < kAcc; ++b) {
            mbar_init(&bar_acc_full[b], 1);
            mbar_init(&bar_acc_empty[b], kEpiWarps);
        }
        s_abort = 0;
        fence_mbar_init();
        prefetch_tmap(&maps.a);
        prefetch_tmap(&maps.b);
        if (g.tma_out) prefetch_tmap(&maps.out);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tslot;
    pdl_trigger();
    if (warp != 9) pdl_wait();  // the weights (warp 9) were there before; codes, scales and `out` belong to earlier kernels

    constexpr int half = NT / 2;
    const int out_cols = p.gate ? half : NT;  // output columns of a tile

    if (warp == 8 || warp == 9) {
        if (lane == 0) {
            const uint32_t bytes = static_cast<uint32_t>(warp == 8 ? kRows : NT) * g.kc;
            int it = 0;
            bool ok = true;
            for (int tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x) {
                const int m0 = (tile / g.n_tiles) * kRows, n0 = (tile % g.n_tiles) * out_cols;
                for (int t = 0; ok && t < p.segs; ++t)
                    for (int j = 0; j < g.chunks; ++j, ++it) {
                        const int s = it % kSt;
                        ok = wait_or_abort(&bar_empty[s], ((it / kSt) & 1) ^ 1, &s_abort, p.err, 0x70);
                        if (!ok) break;
                        uint8_t* sa = smem + s * P::kStage;
                        mbar_arrive_expect_tx(&bar_full[s], bytes);
                        if (warp == 8) {
                            tma_load_2d(sa, &maps.a, j * g.kc, static_cast<int>(p.arow[t]) + m0, &bar_full[s]);
                        } else {
                            uint8_t* sb = sa + kStageA;
                            const int k = t * p.seg_p + j * g.kc;
                            tma_load_2d(sb, &maps.b, k, n0, &bar_full[s]);
                            if (p.gate) tma_load_2d(sb + half * g.kc, &maps.b, k, p.n_out + n0, &bar_full[s]);
                        }
                    }
            }
            // After a wait that ran out: the copies in flight land before the CTA leaves.
            if (!ok)
                for (int k = max(0, it - kSt); k < it; ++k) mbar_wait(&bar_full[k % kSt], (k / kSt) & 1, 100000000ull);
        }
    } else if (warp == 10) {
        if (lane == 0) {
            constexpr uint32_t idesc = idesc_s8(kRows, NT);
            const uint32_t sm0 = smem_u32(smem);
            const uint64_t ad0 = sdesc_kmajor_sw(sm0, g.kc), bd0 = sdesc_kmajor_sw(sm0 + kStageA, g.kc);
            int it = 0, q = 0;
            bool ok = true;
            for (int tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x) {
                for (int t = 0; ok && t < p.segs; ++t, ++q) {
                    const int b = q % kAcc;
                    ok = wait_or_abort(&bar_acc_empty[b], ((q / kAcc) & 1) ^ 1, &s_abort, p.err, 0x71);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t acc = tmem + b * NT;
                    for (int j = 0; j < g.chunks; ++j, ++it) {
                        const int s = it % kSt;
                        ok = wait_or_abort(&bar_full[s], (it / kSt) & 1, &s_abort, p.err, 0x72);
                        if (!ok) break;
                        tc_fence_after();
                        const uint64_t so = static_cast<uint64_t>(s) * (P::kStage >> 4);
                        const int steps = min(g.kc, p.seg_c - j * g.kc + 31) / 32;
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (k < steps) mma_s8(acc, ad0 + so + 2 * k, bd0 + so + 2 * k, idesc, (j > 0 || k > 0) ? 1u : 0u);
                        mma_commit(&bar_empty[s]);
                    }
                    if (ok) mma_commit(&bar_acc_full[b]);
                }
            }
        }
    } else {
        const int quad = warp & 3, group = warp >> 2;
        uint8_t* stg = smem + kSt * P::kStage + warp * kStgWarp;
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
            if (row >= p.rows) return;
            if (p.planes)
                store_planes32(out + (img * p.n_out + c) * p.ldo + (row - img * p.ldo), p.ldo, y, c, p.n_out);
            else
                store_row32(out + row * p.ldo + c, y, c, p.n_out, g.vec_out);
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
        auto acc_wait = [&](int q) {
            const bool ok =
                lane == 0 ? wait_or_abort(&bar_acc_full[q % kAcc], (q / kAcc) & 1, &s_abort, p.err, 0x73) : true;
            const bool all = __shfl_sync(0xffffffffu, ok, 0);
            tc_fence_after();
            return all;
        };
        auto acc_done = [&](int q) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar_acc_empty[q % kAcc]);
        };
        int q = 0, n = 0;
        for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, ++n) {
            const int64_t m0 = static_cast<int64_t>(tile / g.n_tiles) * kRows + quad * 32;
            const int n0 = (tile % g.n_tiles) * out_cols;
            const int64_t row = m0 + lane;
            const int64_t img = p.planes && row < p.rows ? row / p.ldo : 0;
            if constexpr (SEG) {
                // A warp takes 32-column blocks: NT/2 columns of its group of
                // warps, or (gated, NT = 128) 32 of each factor.
                constexpr int kBlocks = NT / 64;
                float s[kMaxSegments];
#pragma unroll
                for (int t = 0; t < kMaxSegments; ++t)
                    s[t] = t < p.segs && row < p.rows ? __ldg(p.as + p.arow[t] + row) : 0.f;
                float y[kBlocks][32];
                int col[kBlocks];
#pragma unroll
                for (int k = 0; k < kBlocks; ++k) col[k] = p.gate ? k * half + group * 32 : group * half + k * 32;
                bool ok = true;
#pragma unroll
                for (int t = 0; t < kMaxSegments; ++t) {
                    if (t >= p.segs) break;
                    ok = acc_wait(q);
                    if (!ok) break;
#pragma unroll
                    for (int k = 0; k < kBlocks; ++k) {
                        int a[32];
                        tmem_ld32(lane_base + (q % kAcc) * NT + col[k], a);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            y[k][i] = t == 0 ? static_cast<float>(a[i]) * s[0] : fmaf(static_cast<float>(a[i]), s[t], y[k][i]);
                    }
                    acc_done(q);
                    ++q;
                }
                if (!ok) break;
#pragma unroll
                for (int k = 0; k < kBlocks; ++k)
                    finish32(p.par + (p.gate ? k * p.npad + n0 + group * 32 : n0 + col[k]), y[k]);
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
                const float s = row < p.rows ? __ldg(p.as + p.arow[0] + row) : 0.f;
                if (!acc_wait(q)) break;
                const uint32_t acc = lane_base + (q % kAcc) * NT;
                auto scaled = [&](int c, const float2* par, float (&y)[32]) {
                    int a[32];
                    tmem_ld32(acc + c, a);
                    tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 32; ++i) y[i] = static_cast<float>(a[i]) * s;
                    finish32(par, y);
                };
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
        if (g.tma_out && lane == 0) bulk_wait_read0();
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
    const bool al16 = reinterpret_cast<uintptr_t>(p.out) % 16 == 0 && p.ldo * sizeof(T) % 16 == 0 && p.ldo >= p.n_out;
    g.tma_out = g.vec_out = !p.planes && al16;
    // Staging tiles of 128-byte rows; 32 columns with segments (a warp's
    // blocks), and for direct stores.
    g.unit = SEG || !g.tma_out ? 32 : std::min<int>(128 / sizeof(T), out_cols);
    Maps maps{};
    DN_TRY(linear8_map(&maps.a, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.a, p.seg_c, p.a_rows, p.lda, g.kc, kRows));
    DN_TRY(linear8_map(&maps.b, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.w, p.ldw, p.cout, p.ldw, g.kc, p.gate ? NT / 2 : NT));
    if (g.tma_out)
        DN_TRY(linear8_map(&maps.out, sizeof(T) == 2 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32,
                           sizeof(T), p.out, p.n_out, p.rows, p.ldo, g.unit, 32));
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

// The widest tile that still gives every SM one (not wider than the layer).
int tile_width(const ProductArgs& p, int sms, int widest) {
    const int64_t m_tiles = (p.rows + kRows - 1) / kRows;
    const int least = p.gate ? 64 : 32;
    int nt = widest;
    while (nt > least) {
        const int oc = p.gate ? nt / 2 : nt;
        if (oc / 2 >= p.n_out || m_tiles * ((p.n_out + oc - 1) / oc) < sms)
            nt >>= 1;
        else
            break;
    }
    return nt;
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

PFN_cuTensorMapEncodeTiled_v12000 linear8_encoder() { return tensor_map_encoder(); }

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

int launch_product_tc(const ProductArgs& a, int out_dtype, int sms, cudaStream_t s) {
    TcArgs g{};
    g.p = a;
    return out_dtype == 1 ? run_type<__half>(g, sms, s) : run_type<float>(g, sms, s);
}

}  // namespace dnb
