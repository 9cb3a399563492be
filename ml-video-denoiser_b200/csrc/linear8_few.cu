// The 8-bit product of a few tokens (serving one or some tokens at a time): one launch
// that quantises the tokens and streams the weight once. Bound by the weight's
// bytes (Cout * Cin) where it is large, by latency where it is small.
//
// Every CTA quantises all tokens into shared memory itself (a few KB out of
// L2), behind the loads of its first weight bytes; a warp then takes CPW
// weight rows at a time, a lane 16 bytes of each, and R tokens with dp4a:
// each weight byte is used R times from registers, and the int32 sums meet in
// one warp-wide reduction per (token, channel). One token, on the device (calls
// behind each other in a graph): 512 -> 1024 2.0 us (5.2 by the tensor cores),
// 4096 -> 4096 5.3 us (12.3), 4096 -> 16384 8.9 us (14.2; 67 MB of weight out of
// L2).
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "denoiser_b200.h"
#include "launch.cuh"
#include "linear8.cuh"
#include "linear8.h"
#include "quant.cuh"
#include "status.h"

namespace dnb {
namespace {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxTokens = 16;
// Codes of all tokens in shared memory. Every CTA makes them all, which costs
// more than the tensor-core path from there on (8 x 4096 -> 4096: 16.1 us against
// 12.3, -> 512: 12.4 against 12.2; 4 x 4096 -> 4096: 10.2 against 12.2).
constexpr int kMaxBytes = 16 * 1024;
// Nine to sixteen tokens: one launch and no workspace are worth five
// microseconds of the host, where no SM has more than two CTAs (13 x 1000 ->
// 520, FP32: 10.3 us a call, 14 by the tensor cores, but replayed 9.1 and 7.3; 13
// x 1024 -> 16384 replayed: 21.7 and 8.0).
constexpr int kManyTokens = 8, kManyChannels = 2 * 148 * 8;

struct FewArgs {
    ProductArgs p;
    const void* x;
    int64_t ldx;
    int vec_in;   // 16-byte loads of x are aligned
    int out_f32;
};

template <typename T, int R, int CPW>
__global__ void __launch_bounds__(kThreads) product_few_kernel(const __grid_constant__ FewArgs g) {
    using Q = QuantOf<T>;
    const ProductArgs& p = g.p;
    extern __shared__ __align__(16) uint8_t s_codes[];  // [R][ldw]
    __shared__ uint32_t s_mag[R];
    __shared__ float s_scale[R];
    const int tid = threadIdx.x, lane = tid & 31;
    const int K = p.seg_c, vecs = static_cast<int>(p.ldw / 16);
    // The warp's weight rows: slots 0 .. CPW-1 are channels c0 ..; of a gated
    // layer slot 2 i and 2 i + 1 are the two factors of output c0 + i.
    const int outs = p.gate ? CPW / 2 : CPW;
    const int c0 = (blockIdx.x * kWarps + (tid >> 5)) * outs;
    const int8_t* w[CPW];
#pragma unroll
    for (int j = 0; j < CPW; ++j) {
        const int c = p.gate ? c0 + j / 2 : c0 + j;
        // Slots behind the last channel repeat it; their sums are not stored.
        w[j] = p.w + static_cast<int64_t>(min(c, p.n_out - 1) + (p.gate && (j & 1) ? p.n_out : 0)) * p.ldw;
    }
    uint4 wv[CPW];
#pragma unroll
    for (int j = 0; j < CPW; ++j)
        wv[j] = lane < vecs ? __ldg(reinterpret_cast<const uint4*>(w[j]) + lane) : make_uint4(0, 0, 0, 0);
    if (R < kWarps) {
        if (tid < R) s_mag[tid] = 0;
        __syncthreads();
    }
    pdl_trigger();
    pdl_wait();

    const T* x = static_cast<const T*>(g.x);
    const int rows = static_cast<int>(p.rows);
    const int groups = (K + 7) / 8;
    auto load = [&](int r, int k) {
        const T* src = x + r * g.ldx + k * 8;
        return g.vec_in ? Q::load(src) : Q::load_some(src, min(8, K - k * 8));
    };
    auto code_at = [&](int r, int k) { return reinterpret_cast<uint2*>(s_codes + r * p.ldw + k * 8); };
    if constexpr (R >= kWarps) {
        // A warp per token, the next one's first kKeep vectors a lane on their way;
        // those stay in registers, what a token has more is read twice.
        constexpr int kKeep = 4, kEach = R / kWarps;
        typename Q::Vec v[kEach > 1 ? 2 : 1][kKeep];
        auto fetch = [&](int r, typename Q::Vec (&t)[kKeep]) {
#pragma unroll
            for (int i = 0; i < kKeep; ++i) t[i] = r < rows && lane + 32 * i < groups ? load(r, lane + 32 * i) : Q::zero();
        };
        fetch(tid >> 5, v[0]);
#pragma unroll
        for (int t = 0; t < kEach; ++t) {
            const int r = (tid >> 5) + t * kWarps;
            if (t + 1 < kEach) fetch(r + kWarps, v[(t + 1) % 2]);
            typename Q::Vec(&cur)[kKeep] = v[t % 2];
            uint32_t mag = 0;
#pragma unroll
            for (int i = 0; i < kKeep; ++i) mag = max(mag, Q::mag(cur[i]));
            if (r < rows)
#pragma unroll 4
                for (int k = lane + 32 * kKeep; k < groups; k += 32) mag = max(mag, Q::mag(load(r, k)));
            mag = __reduce_max_sync(0xffffffffu, mag);
            const GroupScale q = group_scale<T>(mag, 127.f);
            if (lane == 0) s_scale[r] = q.s;
#pragma unroll
            for (int i = 0; i < kKeep; ++i)
                if (lane + 32 * i < vecs * 2) *code_at(r, lane + 32 * i) = codes8<T>(cur[i], q, q.rare);
#pragma unroll 4
            for (int k = lane + 32 * kKeep; k < vecs * 2; k += 32)
                *code_at(r, k) = codes8<T>(r < rows && k < groups ? load(r, k) : Q::zero(), q, q.rare);
        }
    } else {
        // All warps on one or two tokens.
        for (int r = 0; r < rows; ++r) {
            uint32_t mag = 0;
            for (int k = tid; k < groups; k += kThreads) mag = max(mag, Q::mag(load(r, k)));
            mag = __reduce_max_sync(0xffffffffu, mag);
            if (lane == 0) atomicMax(&s_mag[r], mag);
        }
        __syncthreads();
        for (int r = 0; r < R; ++r) {
            const GroupScale q = group_scale<T>(r < rows ? s_mag[r] : 0u, 127.f);
            if (tid == 0) s_scale[r] = q.s;
            for (int k = tid; k < vecs * 2; k += kThreads)
                *code_at(r, k) = codes8<T>(r < rows && k < groups ? load(r, k) : Q::zero(), q, q.rare);
        }
    }
    __syncthreads();

    int acc[R][CPW];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int j = 0; j < CPW; ++j) acc[r][j] = 0;
    for (int v = lane; v < vecs; v += 32) {
        uint4 cur[CPW];
#pragma unroll
        for (int j = 0; j < CPW; ++j) {
            cur[j] = wv[j];
            if (v + 32 < vecs) wv[j] = __ldg(reinterpret_cast<const uint4*>(w[j]) + v + 32);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const uint4 a = *reinterpret_cast<const uint4*>(s_codes + r * p.ldw + v * 16);
#pragma unroll
            for (int j = 0; j < CPW; ++j) {
                int s = __dp4a(static_cast<int>(a.x), static_cast<int>(cur[j].x), acc[r][j]);
                s = __dp4a(static_cast<int>(a.y), static_cast<int>(cur[j].y), s);
                s = __dp4a(static_cast<int>(a.z), static_cast<int>(cur[j].z), s);
                acc[r][j] = __dp4a(static_cast<int>(a.w), static_cast<int>(cur[j].w), s);
            }
        }
    }
    // Sums over the warp; lane r * CPW + j keeps that of token r, slot j.
    int mine = 0;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int j = 0; j < CPW; ++j) {
            const int s = __reduce_add_sync(0xffffffffu, acc[r][j]);
            if (lane == r * CPW + j) mine = s;
        }
    const int r = lane / CPW, j = lane % CPW;
    const int o = p.gate ? c0 + j / 2 : c0 + j;
    const bool in = r < R && o < p.n_out;
    float y = 0.f;
    if (in) {
        const float2 wb = __ldg(p.par + o + (p.gate && (j & 1) ? p.npad : 0));
        const float s = s_scale[r];
        const bool large = s >= kLargeScale;
        y = fmaf(static_cast<float>(mine) * (large ? wb.x : s), large ? s : wb.x, wb.y);
    }
    if (p.gate) y *= __shfl_down_sync(0xffffffffu, y, 1);
    if (in && r < rows && !(p.gate && (j & 1))) {
        if (g.out_f32)
            static_cast<float*>(p.out)[r * p.ldo + o] = y;
        else
            static_cast<__half*>(p.out)[r * p.ldo + o] = __float2half_rn(y);
    }
}

template <typename T, int R, int CPW>
cudaError_t run(const FewArgs& g, cudaStream_t s) {
    const int per = kWarps * (g.p.gate ? CPW / 2 : CPW);
    const size_t smem = static_cast<size_t>(R) * g.p.ldw;
    return launch_pdl(product_few_kernel<T, R, CPW>, dim3((g.p.n_out + per - 1) / per), dim3(kThreads), smem, s, g);
}

template <typename T, int R>
cudaError_t run_cpw(const FewArgs& g, int sms, cudaStream_t s) {
    // Four weight rows a warp where that still gives every SM a CTA (one token,
    // 4096 -> 16384: 8.9 us, 10.6 with two rows; 8 x 512 -> 1024: 3.0 and 2.9).
    return g.p.cout >= sms * kWarps * 4 ? run<T, R, 4>(g, s) : run<T, R, 2>(g, s);
}

template <typename T>
cudaError_t run_rows(const FewArgs& g, int sms, cudaStream_t s) {
    if (g.p.rows == 1) return run_cpw<T, 1>(g, sms, s);
    if (g.p.rows == 2) return run_cpw<T, 2>(g, sms, s);
    if (g.p.rows <= 4) return run_cpw<T, 4>(g, sms, s);
    if (g.p.rows <= 8) return run_cpw<T, 8>(g, sms, s);
    return run<T, 16, 2>(g, s);  // a lane for each of 32 sums
}

}  // namespace

bool product_few_takes(const ProductArgs& a) {
    const int64_t r = a.rows <= 2 ? a.rows : a.rows <= 4 ? 4 : a.rows <= 8 ? 8 : 16;
    return a.rows <= kMaxTokens && !a.planes && a.segs == 1 && r * a.ldw <= kMaxBytes &&
           (a.rows <= kManyTokens || a.cout <= kManyChannels);
}

int launch_product_few(const ProductArgs& a, const void* x, int dtype, int64_t ldx, int out_dtype, int sms,
                       cudaStream_t s) {
    FewArgs g{};
    g.p = a;
    g.x = x;
    g.ldx = ldx;
    g.out_f32 = out_dtype == 0;
    g.vec_in = a.seg_c % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0 && ldx * (dtype == 1 ? 2 : 4) % 16 == 0;
    const cudaError_t e = dtype == 1 ? run_rows<__half>(g, sms, s) : run_rows<float>(g, sms, s);
    return e == cudaSuccess ? DN_OK : dn_cuda_fail(e, "linear8: launch over a few tokens");
}

}  // namespace dnb
