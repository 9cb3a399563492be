// The 8-bit product over NCHW planes of narrow layers (Cin <= 128, Cout <= 256)
// whose planes TMA can address (H * W a multiple of 8, 32 or more; 16-byte aligned): one
// pass, bound by HBM (2 Cin + 2 Cout bytes a pixel).
//
// Planes are channel-major and the operand of the MMA is pixel-major. The
// transposes cost one instruction per 8 x 32 values each way:
//   in    TMA brings [KP channels][64 pixels] boxes (128-byte swizzle);
//         ldmatrix.trans hands lane t of a warp, for pixel t / 4, the channels
//         8 m + 2 (t % 4) + {0, 1} of four 8-channel groups m. A lane quantises
//         these 8 values (the pixel's maximum is two shuffles) and writes them
//         as 8 adjacent bytes: the K order of the operand is a permutation of
//         the channels within each 32, and the weight is laid out in the same
//         one, so the sums are those of the definition;
//   out   tcgen05.ld 16x256b returns the accumulator in the layout whose
//         packed pairs stmatrix.trans stores channel-major; TMA stores boxes
//         of all channels x 64 pixels, each filled by two warps.
// A CTA of four warps takes tiles of 128 pixels of one image, keeps the weight
// in shared memory and two tiles' loads in flight; several CTAs per SM overlap
// each other's phases. 32 -> 64 over 1088x1920 takes 92 us (4.3 TB/s); the same
// bytes in 16 images of 272x480 take 77: planes that lie megabytes apart cost
// something (address translations, it seems; no counter was read), and there are
// two CTA-wide barriers a tile.
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
constexpr int kThreads = 128;

struct PlanesArgs {
    ProductArgs p;
    int tiles_per_image, tiles;
};

template <int KP, int NT>
struct Shape {
    static constexpr int kBox = KP * 128;            // 64 pixels of KP channels
    static constexpr int kIn = 2 * kBox;             // a tile
    static constexpr int kA = kRows * KP, kB = NT * KP;
    // The output tile, two boxes of 64 pixels: a gated layer uses half of it.
    static int smem(bool gate) { return 1024 + 2 * kIn + kA + kB + (gate ? NT / 2 : NT) * 256; }
};

template <int KP, int NT>
__global__ void __launch_bounds__(kThreads) product_planes_kernel(const __grid_constant__ PlanesArgs g,
                                                                  const __grid_constant__ CUtensorMap in_map,
                                                                  const __grid_constant__ CUtensorMap out_map) {
    using S = Shape<KP, NT>;
    using Q = QuantOf<__half>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    __shared__ uint64_t bar, bar_in[2], bar_end;
    __shared__ uint32_t tslot;
    __shared__ volatile int s_abort;
    __shared__ float s_x[2][kRows];
    __shared__ __align__(16) float2 s_par[NT];
    const ProductArgs& p = g.p;
    const int tid = threadIdx.x, warp = warp_index(), lane = tid & 31;
    uint8_t* s_in = smem;
    uint8_t* sa = smem + 2 * S::kIn;
    uint8_t* sb = sa + S::kA;
    constexpr int half = NT / 2;
    const int out_cols = p.gate ? half : NT;
    uint8_t* stg = sb + S::kB + (warp >> 1) * (out_cols * 128);  // this warp's 64-pixel box of the output tile
    constexpr uint32_t kCols = NT < 32 ? 32 : NT;

    if (warp == 0) {
        tmem_alloc(&tslot, kCols);
        tmem_relinquish();
    }
    if (tid == 0) {
        mbar_init(&bar, 1);
        mbar_init(&bar_end, 1);
        mbar_init(&bar_in[0], 1);
        mbar_init(&bar_in[1], 1);
        s_abort = 0;
        fence_mbar_init();
        prefetch_tmap(&in_map);
        prefetch_tmap(&out_map);
    }
    // The weight, its channels in the operand's order: byte position 32 v +
    // 8 j + 2 m + e holds channel 32 v + 8 m + 2 j + e.
    for (int i = tid; i < NT * (KP / 16); i += kThreads) {
        const int r = i / (KP / 16), q = i % (KP / 16);
        int c;
        if (!p.gate)
            c = r < p.cout ? r : -1;
        else
            c = r < half ? (r < p.n_out ? r : -1) : (r - half < p.n_out ? p.n_out + r - half : -1);
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int h = 0; h < 8; ++h) {  // pairs of adjacent channels
            const int pos = q * 16 + 2 * h;
            const int ch = (pos & ~31) + ((pos & 7) >> 1) * 8 + ((pos >> 3) & 3) * 2;
            if (c >= 0 && ch < p.ldw)
                w[h >> 1] |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(p.w + c * p.ldw + ch)) << ((h & 1) * 16);
        }
        *reinterpret_cast<uint4*>(sb + sw_offset(r, q, KP)) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    for (int r = tid; r < NT; r += kThreads) s_par[r] = __ldg(p.par + (p.gate && r >= half ? p.npad + r - half : r));
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tslot;
    pdl_trigger();
    pdl_wait();

    auto load = [&](int tile, int b) {
        const int img = tile / g.tiles_per_image, x0 = (tile - img * g.tiles_per_image) * kRows;
        mbar_arrive_expect_tx(&bar_in[b], S::kIn);
        tma_load_3d(s_in + b * S::kIn, &in_map, x0, 0, img, &bar_in[b]);
        tma_load_3d(s_in + b * S::kIn + S::kBox, &in_map, x0 + 64, 0, img, &bar_in[b]);
    };
    if (tid == 0) {
        if (static_cast<int>(blockIdx.x) < g.tiles) load(blockIdx.x, 0);
        if (static_cast<int>(blockIdx.x + gridDim.x) < g.tiles) load(blockIdx.x + gridDim.x, 1);
    }
    int issued = static_cast<int>(blockIdx.x + gridDim.x) < g.tiles ? 2 : 1;  // loads, for the lane that issues them
    const uint64_t ad0 = sdesc_kmajor_sw(smem_u32(sa), KP), bd0 = sdesc_kmajor_sw(smem_u32(sb), KP);
    const int steps = (p.seg_c + 31) / 32;
    const int j4 = lane & 3, px = lane >> 2;  // a lane's channel pair and pixel of 8
    int n = 0;
    // The tile's image and place in it, stepped along with the tile.
    const int step_img = gridDim.x / g.tiles_per_image, step_x = gridDim.x - step_img * g.tiles_per_image;
    int img = blockIdx.x / g.tiles_per_image, xt = blockIdx.x - img * g.tiles_per_image;
    const bool issues = tid == 32;  // this thread stores the output tiles
    for (int tile = blockIdx.x; tile < g.tiles; tile += gridDim.x, ++n) {
        const int b = n & 1;
        float* sx = s_x[b];
        wait_or_abort(&bar_in[b], (n >> 1) & 1, &s_abort, p.err, 0x75);
        __syncwarp();
        // This warp's 32 pixels: half of a 64-pixel box, four groups of 8.
        const uint32_t box = smem_u32(s_in + b * S::kIn + (warp >> 1) * S::kBox);
        typename Q::Vec v[4][KP / 32];
        GroupScale q[4];
        bool rare = false;
#pragma unroll
        for (int pg = 0; pg < 4; ++pg) {
            const uint32_t chunk = (warp & 1) * 4 + pg;
            uint32_t mag = 0;
#pragma unroll
            for (int k = 0; k < KP / 32; ++k) {
                uint32_t r[4];
                ldmatrix4_trans(r, box + (k * 32 + lane) * 128 + ((chunk ^ (lane & 7)) << 4));
                v[pg][k].v = make_uint4(r[0], r[1], r[2], r[3]);
                mag = max(mag, Q::mag(v[pg][k]));
            }
            mag = max(mag, __shfl_xor_sync(0xffffffffu, mag, 1));
            mag = max(mag, __shfl_xor_sync(0xffffffffu, mag, 2));
            q[pg] = group_scale<__half>(mag, 127.f);
            rare = rare || q[pg].rare;
            if (j4 == 0) sx[warp * 32 + pg * 8 + px] = q[pg].s;
        }
        auto code_at = [&](int pg, int k) {
            return reinterpret_cast<uint2*>(sa + sw_offset(warp * 32 + pg * 8 + px, k * 2 + (j4 >> 1), KP) + (j4 & 1) * 8);
        };
        // One vote for the warp's 32 pixels (a fifth of the warps has a rare one).
        if (!__any_sync(0xffffffffu, rare)) {
#pragma unroll
            for (int pg = 0; pg < 4; ++pg)
#pragma unroll
                for (int k = 0; k < KP / 32; ++k) *code_at(pg, k) = codes8_fast(v[pg][k], q[pg].r);
        } else {
#pragma unroll
            for (int pg = 0; pg < 4; ++pg)
#pragma unroll
                for (int k = 0; k < KP / 32; ++k) *code_at(pg, k) = codes8_rare<__half>(v[pg][k], q[pg]);
        }
        fence_async_smem();
        tc_fence_before();
        if (issues) bulk_wait_read0();
        __syncthreads();  // the operand is complete; this input buffer, the accumulator and the output tile are free
        if (warp == 0) {
            tc_fence_after();
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < KP / 32; ++k)
                    if (k < steps) mma_s8(tmem, ad0 + 2 * k, bd0 + 2 * k, idesc_s8(kRows, NT), k > 0 ? 1u : 0u);
                mma_commit(&bar);
                const int64_t next = static_cast<int64_t>(tile) + 2 * static_cast<int64_t>(gridDim.x);
                if (next < g.tiles && !s_abort) {
                    load(static_cast<int>(next), b);
                    ++issued;
                }
            }
            __syncwarp();
        }
        wait_or_abort(&bar, n & 1, &s_abort, p.err, 0x76);
        __syncwarp();
        tc_fence_after();

        const uint32_t acc = tmem + (static_cast<uint32_t>(warp * 32) << 16);
        float s[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] = sx[warp * 32 + i * 8 + px];
        // y[k][pg]: tile columns c + 8 k + 2 j4 and the next of pixel 8 pg + px.
        auto scaled = [&](int c, float2 (&y)[4][4]) {
            int a[2][16];
            tmem_ld_16x32(acc + c, a[0]);
            tmem_ld_16x32(acc + (16u << 16) + c, a[1]);
            tmem_ld_wait();
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float4 w = *reinterpret_cast<const float4*>(&s_par[c + 8 * k + 2 * j4]);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int* v = &a[i >> 1][4 * k + 2 * (i & 1)];
                    const float2 t = ffma2(make_float2(static_cast<float>(v[0]), static_cast<float>(v[1])),
                                           make_float2(s[i], s[i]), make_float2(0.f, 0.f));
                    y[k][i] = ffma2(t, make_float2(w.x, w.z), make_float2(w.y, w.w));
                }
            }
        };
        for (int c = 0; c < out_cols && c < p.n_out; c += 32) {
            float2 y[4][4];
            scaled(c, y);
            if (p.gate) {
                float2 z[4][4];
                scaled(half + c, z);
#pragma unroll
                for (int k = 0; k < 4; ++k)
#pragma unroll
                    for (int i = 0; i < 4; ++i) y[k][i].x *= z[k][i].x, y[k][i].y *= z[k][i].y;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)
                stmatrix4_trans(smem_u32(stg) + sw_offset(c + 8 * k + (lane & 7), (warp & 1) * 4 + (lane >> 3), 128),
                                pack_half2(y[k][0].x, y[k][0].y), pack_half2(y[k][1].x, y[k][1].y),
                                pack_half2(y[k][2].x, y[k][2].y), pack_half2(y[k][3].x, y[k][3].y));
        }
        fence_async_smem();
        __syncthreads();
        if (issues) {
            const int x0 = xt * kRows;
            tma_store_3d(&out_map, x0, 0, img, stg);
            if (x0 + 64 < p.ldo) tma_store_3d(&out_map, x0 + 64, 0, img, stg + out_cols * 128);
            bulk_commit();
        }
        img += step_img;
        xt += step_x;
        if (xt >= g.tiles_per_image) {
            xt -= g.tiles_per_image;
            ++img;
        }
    }
    if (issues) bulk_wait_read0();
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        // After a wait that ran out: the loads and MMAs in flight end before the CTA leaves.
        if (s_abort) {
            if (elect_one())
                for (int k = max(0, issued - 2); k < issued; ++k) mbar_wait(&bar_in[k & 1], (k >> 1) & 1, 100000000ull);
            __syncwarp();
            drain_mmas(&bar_end);
        }
        tmem_dealloc(tmem, kCols);
    }
}

template <int KP, int NT>
int run(PlanesArgs& g, const void* x, int sms, cudaStream_t s) {
    using S = Shape<KP, NT>;
    const ProductArgs& p = g.p;
    const int64_t images = p.rows / p.ldo;
    CUtensorMap in{}, out{};
    DN_TRY(linear8_planes_map(&in, x, p.ldo, p.seg_c, images, 64, KP));
    // (Output boxes of 32 pixels, one per warp, cost 157 us instead of 93 at 32 ->
    // 64 channels, 1088x1920: half lines, and twice the address translations
    // where the planes are megabytes apart.)
    DN_TRY(linear8_planes_map(&out, p.out, p.ldo, p.n_out, images, 64, p.gate ? NT / 2 : NT));
    static int resident[2][64] = {};
    const int smem = S::smem(p.gate);
    int per_sm = 0;
    cudaError_t e = tmem_kernel_ctas(product_planes_kernel<KP, NT>, kThreads, smem, S::smem(false), NT,
                                     resident[p.gate ? 1 : 0], &per_sm);
    if (e == cudaSuccess)
        e = launch_pdl(product_planes_kernel<KP, NT>, dim3(static_cast<unsigned>(std::min(g.tiles, per_sm * sms))),
                       dim3(kThreads), smem, s, g, in, out);
    return e == cudaSuccess ? DN_OK : dn_cuda_fail(e, "linear8: planes launch");
}

template <int KP>
int run_nt(PlanesArgs& g, const void* x, int sms, cudaStream_t s) {
    const int need = fused_width(g.p);
    if (need <= 32) return run<KP, 32>(g, x, sms, s);
    if (need <= 64) return run<KP, 64>(g, x, sms, s);
    if (need <= 128) return run<KP, 128>(g, x, sms, s);
    return run<KP, 256>(g, x, sms, s);
}

}  // namespace

bool product_planes_takes(const ProductArgs& a, const void* x) {
    // A tile is of one image, so planes of a few pixels fill it badly (522240
    // pixels, 64 -> 64: 166 us in planes of 16 and 86 of 32; tiles across images
    // take 112 us of any).
    return a.planes && fused_width(a) <= 256 && a.segs == 1 && a.seg_c <= 128 && a.ldo % 8 == 0 && a.ldo >= 32 &&
           reinterpret_cast<uintptr_t>(x) % 16 == 0 && reinterpret_cast<uintptr_t>(a.out) % 16 == 0;
}

int launch_product_planes(const ProductArgs& a, const void* x, int sms, cudaStream_t s) {
    PlanesArgs g{};
    g.p = a;
    g.tiles_per_image = static_cast<int>((a.ldo + kRows - 1) / kRows);
    g.tiles = static_cast<int>(g.tiles_per_image * (a.rows / a.ldo));
    if (a.seg_c <= 32) return run_nt<32>(g, x, sms, s);
    if (a.seg_c <= 64) return run_nt<64>(g, x, sms, s);
    return run_nt<128>(g, x, sms, s);
}

}  // namespace dnb
