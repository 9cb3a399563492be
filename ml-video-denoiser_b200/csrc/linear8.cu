// Linear8: y[m, n] = s_x[m] s_w[n] sum_k q_x[m, k] q_w[n, k] + bias[n] in 8-bit
// integers (include/denoiser_b200_quant.h has the definition).
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <memory>
#include <new>
#include <string>
#include <vector>

#include "capi_internal.h"
#include "denoiser_b200_quant.h"
#include "launch.cuh"
#include "linear8.h"
#include "quant.cuh"
#include "row_cache.h"
#include "status.h"

namespace dnb {
namespace {

constexpr int kMaxK = 131072;  // 127 * 127 * 131072 < 2^31

// Codes and scales of the pixels of NCHW planes (layers too wide for one pass):
// a CTA of eight warps takes 32 PX pixels, a lane PX adjacent ones of them
// (two where pairs are 4-byte aligned) and a warp 32 channels at a time, so
// that the loads of 32 channels are in flight and a lane's codes are a whole
// 32-byte sector. Between the two passes a warp's first run of channels stays in
// registers; with pixel pairs the next `kept` ones stay in shared memory (each
// lane its own vectors), what a very wide layer has beyond them is read again.
// Single pixels read all of them again: there the occupancy is worth more (2
// images of 36867 pixels, 1296 -> 26 gated: 151 us, 274 with 96 KB kept; pairs of
// 36868: 111 us, 120 without).
template <int PX>
__global__ void __launch_bounds__(256) quantise_planes_kernel(const __half* __restrict__ x, int64_t rows, int K, int64_t hw,
                                                              uint8_t* __restrict__ codes, int64_t ldc,
                                                              float* __restrict__ scales, int kept) {
    using Q = QuantOf<__half>;
    extern __shared__ __align__(16) uint4 s_keep[];  // [run][warp][pixel][4][lane]
    __shared__ uint32_t s_mag[32 * PX];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x < 32 * PX) s_mag[threadIdx.x] = 0;
    __syncthreads();
    pdl_trigger();
    pdl_wait();
    const int64_t m = (static_cast<int64_t>(blockIdx.x) * 32 + lane) * PX;
    const bool live = m < rows;  // PX == 2: the planes' pixels are even in number
    const int64_t img = live ? m / hw : 0;
    const __half* src = x + img * K * hw + (live ? m - img * hw : 0);
    auto load = [&](int k0, Q::Vec (&v)[PX][4]) {
        uint32_t w[PX][16];
        const __half* p = src + k0 * hw;
#pragma unroll
        for (int i = 0; i < 32; i += 2, p += 2 * hw) {
            if constexpr (PX == 2) {
                const uint32_t a = live && k0 + i < K ? __ldg(reinterpret_cast<const uint32_t*>(p)) : 0u;
                const uint32_t b = live && k0 + i + 1 < K ? __ldg(reinterpret_cast<const uint32_t*>(p + hw)) : 0u;
                w[0][i >> 1] = __byte_perm(a, b, 0x5410);
                w[1][i >> 1] = __byte_perm(a, b, 0x7632);
            } else {
                const uint32_t a = live && k0 + i < K ? __half_as_ushort(__ldg(p)) : 0u;
                const uint32_t b = live && k0 + i + 1 < K ? __half_as_ushort(__ldg(p + hw)) : 0u;
                w[0][i >> 1] = a | (b << 16);
            }
        }
#pragma unroll
        for (int q = 0; q < PX; ++q)
#pragma unroll
            for (int i = 0; i < 4; ++i) v[q][i].v = make_uint4(w[q][4 * i], w[q][4 * i + 1], w[q][4 * i + 2], w[q][4 * i + 3]);
    };
    uint32_t mag[PX] = {};
    auto largest = [&](const Q::Vec (&v)[PX][4]) {
#pragma unroll
        for (int q = 0; q < PX; ++q)
#pragma unroll
            for (int i = 0; i < 4; ++i) mag[q] = max(mag[q], Q::mag(v[q][i]));
    };
    Q::Vec keep[PX][4];
    load(warp * 32, keep);
    largest(keep);
    auto kept_at = [&](int j, int q, int i) { return &s_keep[(((j * 8 + warp) * PX + q) * 4 + i) * 32 + lane]; };
    for (int k0 = warp * 32 + 256, j = 0; k0 < K; k0 += 256, ++j) {
        Q::Vec v[PX][4];
        load(k0, v);
        largest(v);
        if constexpr (PX == 2)
            if (j < kept)
#pragma unroll
                for (int q = 0; q < PX; ++q)
#pragma unroll
                    for (int i = 0; i < 4; ++i) *kept_at(j, q, i) = v[q][i].v;
    }
#pragma unroll
    for (int q = 0; q < PX; ++q) atomicMax(&s_mag[lane * PX + q], mag[q]);
    __syncthreads();
    GroupScale g[PX];
    bool rare = false;
#pragma unroll
    for (int q = 0; q < PX; ++q) {
        g[q] = group_scale<__half>(s_mag[lane * PX + q], 127.f);
        rare = rare || g[q].rare;
    }
    rare = __any_sync(0xffffffffu, rare);
    auto store = [&](int k0, const Q::Vec (&v)[PX][4]) {
#pragma unroll
        for (int q = 0; q < PX; ++q) {
            uint8_t* dst = codes + (m + q) * ldc + k0;
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                const uint2 lo = codes8<__half>(v[q][i], g[q], rare), hi = codes8<__half>(v[q][i + 1], g[q], rare);
                if (live && k0 + i * 8 < ldc) *reinterpret_cast<uint4*>(dst + i * 8) = make_uint4(lo.x, lo.y, hi.x, hi.y);
            }
        }
    };
    store(warp * 32, keep);
    for (int k0 = warp * 32 + 256, j = 0; k0 < K; k0 += 256, ++j) {
        Q::Vec v[PX][4];
        if (PX == 2 && j < kept) {
#pragma unroll
            for (int q = 0; q < PX; ++q)
#pragma unroll
                for (int i = 0; i < 4; ++i) v[q][i].v = *kept_at(j, q, i);
        } else {
            load(k0, v);
        }
        store(k0, v);
    }
    if (warp == 0 && live)
#pragma unroll
        for (int q = 0; q < PX; ++q) scales[m + q] = g[q].s;
}

template <int PX>
cudaError_t quantise_planes(const void* x, int64_t rows, int K, int64_t hw, uint8_t* codes, int64_t ldc, float* scales,
                            cudaStream_t s) {
    constexpr int kRun = 8 * PX * 4 * 32 * 16;  // one run of all warps
    constexpr int kMost = PX == 2 ? 96 * 1024 / kRun : 0;  // two CTAs per SM
    const int kept = std::min((K - 1) / 256, kMost);
    static bool configured[64] = {};
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e == cudaSuccess && (device >= 64 || !configured[device])) {
        e = cudaFuncSetAttribute(quantise_planes_kernel<PX>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost * kRun);
        if (e == cudaSuccess && device < 64) configured[device] = true;
    }
    if (e != cudaSuccess) return e;
    return launch_pdl(quantise_planes_kernel<PX>, dim3(static_cast<unsigned>((rows + 32 * PX - 1) / (32 * PX))),
                      dim3(256), static_cast<size_t>(kept) * kRun, s, static_cast<const __half*>(x), rows, K, hw, codes, ldc,
                      scales, kept);
}

// par of ProductArgs from the weight rows' scales and the bias (may be null).
__global__ void params_kernel(const float* ws, const void* b, int dtype, float2* par, int cout, int n_out, int npad) {
    const int c = blockIdx.x * blockDim.x + threadIdx.x;
    if (c >= cout) return;
    const float v = !b ? 0.f : dtype == 1 ? __half2float(static_cast<const __half*>(b)[c]) : static_cast<const float*>(b)[c];
    par[c < n_out ? c : npad + c - n_out] = make_float2(ws[c], v);
}

struct DeviceScope {
    int prev = -1;
    explicit DeviceScope(int d) {
        cudaGetDevice(&prev);
        if (prev != d) cudaSetDevice(d);
    }
    ~DeviceScope() {
        int cur = -1;
        cudaGetDevice(&cur);
        if (prev >= 0 && cur != prev) cudaSetDevice(prev);
    }
};

int64_t round16(int64_t v) { return (v + 15) / 16 * 16; }

}  // namespace
}  // namespace dnb

using namespace dnb;

struct dn_linear8 {
    int device = 0;
    int cout = 0, cin = 0, gate = 0, segs = 1, seg_c = 0, seg_p = 0;
    int64_t ldw = 0;
    int sms = 148;
    uint8_t* arena = nullptr;  // weight codes, channel parameters, error word
    int8_t* w = nullptr;
    float2* par = nullptr;
    uint32_t* err = nullptr;
    int n_out() const { return gate ? cout / 2 : cout; }
    int npad() const { return (n_out() + 255) / 256 * 256; }
};

namespace {

int check_shape(int64_t cout, int64_t cin, int gate, int segments) {
    if (cout <= 0 || cin <= 0) return dn_fail(DN_ERR_INVALID_ARG, "dn_linear8_create: empty weight");
    if (cin > kMaxK) return dn_fail(DN_ERR_UNSUPPORTED, "dn_linear8_create: more than 131072 input channels");
    if (cout > (1 << 20)) return dn_fail(DN_ERR_UNSUPPORTED, "dn_linear8_create: more than 2^20 output channels");
    if (gate && cout % 2) return dn_fail(DN_ERR_INVALID_ARG, "dn_linear8_create: the gate needs an even number of channels");
    if (segments < 1 || cin % segments)
        return dn_fail(DN_ERR_INVALID_ARG, "dn_linear8_create: segments does not divide the input channels");
    if (segments > kMaxSegments) return dn_fail(DN_ERR_UNSUPPORTED, "dn_linear8_create: more than 8 segments");
    return DN_OK;
}

int check_device(int device) {
    int count = 0;
    const cudaError_t e = cudaGetDeviceCount(&count);
    if (e != cudaSuccess) return dn_cuda_fail(e, "dn_linear8_create: cudaGetDeviceCount");
    if (device < 0 || device >= count)
        return dn_fail_str(DN_ERR_INVALID_ARG, "dn_linear8_create: CUDA device " + std::to_string(device) +
                                                   " not available (" + std::to_string(count) + " devices found)");
    return DN_OK;
}

// The layer's own copy of the weight, quantised; the current device is the layer's.
cudaError_t lay_out(dn_linear8* L, const void* weight, int dtype, int64_t ldw, const void* bias, cudaStream_t s, int& rc) {
    const int64_t codes = round16(L->cout * L->ldw);
    const size_t pars = static_cast<size_t>(L->npad()) * (L->gate ? 2 : 1) * sizeof(float2);
    const size_t total = static_cast<size_t>(codes) + pars + 16;
    cudaError_t e = cudaMalloc(&L->arena, total);
    if (e != cudaSuccess) return e;
    L->w = reinterpret_cast<int8_t*>(L->arena);
    L->par = reinterpret_cast<float2*>(L->arena + codes);
    L->err = reinterpret_cast<uint32_t*>(L->arena + codes + pars);
    if ((e = cudaMemsetAsync(L->arena, 0, total, s)) != cudaSuccess) return e;
    // Segments that are padded one by one are quantised apart and copied.
    const bool apart = L->segs > 1 && L->seg_p != L->seg_c;
    const size_t dense_bytes = apart ? static_cast<size_t>(L->cout) * L->cin : 0;
    uint8_t* tmp = nullptr;
    if ((e = cudaMalloc(&tmp, static_cast<size_t>(L->cout) * sizeof(float) + dense_bytes)) != cudaSuccess) return e;
    float* ws = reinterpret_cast<float*>(tmp);
    uint8_t* dense = apart ? tmp + static_cast<size_t>(L->cout) * sizeof(float) : L->arena;
    rc = launch_cache_write(CacheWrite{weight, dtype, ldw, L->cout, L->cin, nullptr, 0, dense, apart ? L->cin : L->ldw, ws,
                                       L->cout, 8, L->cin, nullptr},
                            s);
    for (int t = 0; apart && rc == DN_OK && e == cudaSuccess && t < L->segs; ++t)
        e = cudaMemcpy2DAsync(L->w + t * L->seg_p, L->ldw, dense + t * L->seg_c, L->cin, L->seg_c, L->cout,
                              cudaMemcpyDeviceToDevice, s);
    if (rc == DN_OK && e == cudaSuccess) {
        params_kernel<<<(L->cout + 255) / 256, 256, 0, s>>>(ws, bias, dtype, L->par, L->cout, L->n_out(), L->npad());
        e = cudaGetLastError();
    }
    const cudaError_t e2 = cudaStreamSynchronize(s);
    cudaFree(tmp);
    return e != cudaSuccess ? e : e2;
}

int create(const void* weight, int dtype, int64_t ldw, const void* bias, int cout, int cin, int gate, int segments,
           int device, cudaStream_t s, dn_linear8** out) {
    std::unique_ptr<dn_linear8> L(new (std::nothrow) dn_linear8);
    if (!L) return dn_fail(DN_ERR_INVALID_ARG, "dn_linear8_create: out of host memory");
    L->device = device;
    L->cout = cout;
    L->cin = cin;
    L->gate = gate ? 1 : 0;
    L->segs = segments;
    L->seg_c = cin / segments;
    L->seg_p = static_cast<int>(round16(L->seg_c));
    L->ldw = static_cast<int64_t>(L->seg_p) * segments;
    int rc = DN_OK;
    cudaDeviceGetAttribute(&L->sms, cudaDevAttrMultiProcessorCount, device);
    const cudaError_t e = lay_out(L.get(), weight, dtype, ldw, bias, s, rc);
    if (e != cudaSuccess || rc != DN_OK) {
        cudaFree(L->arena);
        return rc != DN_OK ? rc : dn_cuda_fail(e, "dn_linear8_create: upload");
    }
    *out = L.release();
    return DN_OK;
}

ProductArgs product_args(const dn_linear8* L) {
    ProductArgs a{};
    a.segs = L->segs;
    a.seg_c = L->seg_c;
    a.seg_p = L->seg_p;
    a.w = L->w;
    a.ldw = L->ldw;
    a.par = L->par;
    a.npad = L->npad();
    a.cout = L->cout;
    a.n_out = L->n_out();
    a.gate = L->gate;
    a.err = L->err;
    return a;
}

bool aligned_to(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

int check_matrix(const void* p, int dtype, int64_t rows, int64_t ld, int64_t cols, const std::string& what) {
    if (dtype != 0 && dtype != 1) return dn_fail_str(DN_ERR_DTYPE, what + ": dtype must be 0 (FP32) or 1 (FP16)");
    if (rows < 0 || rows >= (1LL << 31)) return dn_fail_str(DN_ERR_INVALID_ARG, what + ": rows outside [0, 2^31)");
    if (rows == 0) return DN_OK;
    if (!p) return dn_fail_str(DN_ERR_INVALID_ARG, what + ": null pointer");
    if (!aligned_to(p, dtype == 1 ? 2 : 4)) return dn_fail_str(DN_ERR_INVALID_ARG, what + ": misaligned pointer");
    if (ld < cols && rows > 1) return dn_fail_str(DN_ERR_INVALID_ARG, what + ": row stride is less than a row");
    return DN_OK;
}

// Whether rows of x (xb bytes, stride xs) and of out (ob bytes, stride os) share
// bytes: tokens are read while others' outputs are written. Columns side by
// side of one buffer (one stride) do not; of rows that lie among each other with
// two strides it is taken that they do.
bool share_bytes(const void* x, int64_t xs, int64_t xb, const void* out, int64_t os, int64_t ob, int64_t rows) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(x), b = reinterpret_cast<uintptr_t>(out);
    if (a + (rows - 1) * xs + xb <= b || b + (rows - 1) * os + ob <= a) return false;
    if (rows == 1 || xs != os) return true;
    const int64_t d = (static_cast<int64_t>(b - a) % xs + xs) % xs;
    return d < xb || d + ob > xs;
}

// How the product of `rows` tokens runs. One pass where the tokens are few or
// the layer is narrow; otherwise the tokens are quantised into the workspace
// and the product reads their codes. (Narrow layers in one pass and in two:
// 522240 x 64 -> 128 43 and 75 us, 130560 x 256 -> 256 33 and 53, 2000 x 64 ->
// 128 5.2 and 6.2, planes 32 -> 64 of 1088x1920 92 and 456.)
enum class Path { kFew, kFused, kTwoPass };

Path path_of(const ProductArgs& a, int dtype) {
    if (product_few_takes(a)) return Path::kFew;
    return dtype == 1 && product_fused_takes(a) ? Path::kFused : Path::kTwoPass;
}

int64_t workspace_bytes_of(const ProductArgs& a, int dtype) {
    return path_of(a, dtype) == Path::kTwoPass ? a.rows * (round16(a.seg_c) + 4) : 0;
}

int check_workspace(int64_t need, const void* ws, int64_t bytes, const char* what) {
    if (need == 0) return DN_OK;
    if (!ws || bytes < need)
        return dn_fail_str(DN_ERR_INVALID_ARG, std::string(what) + ": the workspace holds " + std::to_string(ws ? bytes : 0) +
                                                   " bytes, " + std::to_string(need) + " are needed");
    if (!aligned_to(ws, 16)) return dn_fail_str(DN_ERR_INVALID_ARG, std::string(what) + ": misaligned workspace");
    return DN_OK;
}

}  // namespace

extern "C" {

int dn_linear8_create(const dn_weights* store, const char* weight_name, const char* bias_name, int gate, int segments,
                      int device, dn_linear8** out) {
    if (!store || !weight_name || !out) return dn_fail(DN_ERR_INVALID_ARG, "dn_linear8_create: null argument");
    *out = nullptr;
    try {
        const HostWeights& hw = *store->hw;
        if (!hw.contains(weight_name)) return dn_fail_str(DN_ERR_NOT_FOUND, std::string("weight not found: ") + weight_name);
        if (bias_name && !hw.contains(bias_name))
            return dn_fail_str(DN_ERR_NOT_FOUND, std::string("weight not found: ") + bias_name);
        const auto& sh = hw.entry(weight_name).shape;
        if (!(sh.size() == 2 || (sh.size() == 4 && sh[2] == 1 && sh[3] == 1)))
            return dn_fail(DN_ERR_FORMAT, "dn_linear8_create: weight must be (Cout, Cin) or (Cout, Cin, 1, 1)");
        DN_TRY(check_shape(sh[0], sh[1], gate, segments));
        const int cout = static_cast<int>(sh[0]), cin = static_cast<int>(sh[1]);
        const std::vector<float> w = hw.to_f32(weight_name);
        std::vector<float> b;
        if (bias_name) {
            b = hw.to_f32(bias_name);
            if (static_cast<int64_t>(b.size()) != cout) return dn_fail(DN_ERR_FORMAT, "dn_linear8_create: bias size");
        }
        DN_TRY(check_device(device));
        DeviceScope scope(device);
        float* dev = nullptr;
        const size_t nw = w.size() * 4, nb = b.size() * 4;
        cudaError_t e = cudaMalloc(&dev, nw + nb);
        if (e == cudaSuccess) e = cudaMemcpy(dev, w.data(), nw, cudaMemcpyHostToDevice);
        if (e == cudaSuccess && nb) e = cudaMemcpy(dev + w.size(), b.data(), nb, cudaMemcpyHostToDevice);
        int rc = e == cudaSuccess ? create(dev, 0, cin, nb ? dev + w.size() : nullptr, cout, cin, gate, segments, device,
                                           nullptr, out)
                                  : dn_cuda_fail(e, "dn_linear8_create: upload");
        cudaFree(dev);
        return rc;
    } catch (const std::exception& ex) {
        return dn_fail_str(DN_ERR_FORMAT, ex.what());
    }
}

int dn_linear8_create_device(const void* weight, int dtype, int64_t ldw, const void* bias, int cout, int cin, int gate,
                             int segments, int device, void* stream, dn_linear8** out) {
    if (!out) return dn_fail(DN_ERR_INVALID_ARG, "dn_linear8_create_device: null argument");
    *out = nullptr;
    DN_TRY(check_shape(cout, cin, gate, segments));
    DN_TRY(check_matrix(weight, dtype, cout, ldw, cin, "dn_linear8_create_device"));
    if (!aligned_to(bias, dtype == 1 ? 2 : 4))
        return dn_fail(DN_ERR_INVALID_ARG, "dn_linear8_create_device: misaligned bias");
    DN_TRY(check_device(device));
    DeviceScope scope(device);
    return create(weight, dtype, ldw, bias, cout, cin, gate, segments, device, static_cast<cudaStream_t>(stream), out);
}

int dn_linear8_destroy(dn_linear8* L) {
    if (!L) return DN_OK;
    DeviceScope scope(L->device);
    cudaFree(L->arena);
    delete L;
    return DN_OK;
}

int dn_linear8_info(const dn_linear8* L, int* out_channels, int* in_channels, int* gate, int* segments) {
    if (!L) return dn_fail(DN_ERR_INVALID_ARG, "dn_linear8_info: null layer");
    if (out_channels) *out_channels = L->n_out();
    if (in_channels) *in_channels = L->cin;
    if (gate) *gate = L->gate;
    if (segments) *segments = L->segs;
    return DN_OK;
}

int dn_linear8_workspace(const dn_linear8* L, int64_t rows, int dtype, int nchw, int64_t* bytes) {
    if (!L || !bytes) return dn_fail(DN_ERR_INVALID_ARG, "dn_linear8_workspace: null argument");
    if (rows < 0 || rows >= (1LL << 31)) return dn_fail(DN_ERR_INVALID_ARG, "dn_linear8_workspace: rows outside [0, 2^31)");
    if (dtype != 0 && dtype != 1) return dn_fail(DN_ERR_DTYPE, "dn_linear8_workspace: dtype must be 0 (FP32) or 1 (FP16)");
    ProductArgs a = product_args(L);
    a.rows = rows;
    a.planes = nchw ? 1 : 0;
    *bytes = workspace_bytes_of(a, dtype);
    return DN_OK;
}

int dn_linear8_forward(dn_linear8* L, const void* x, int dtype, int64_t ldx, int64_t rows, void* out, int out_dtype,
                       int64_t ldo, void* workspace, int64_t workspace_bytes, void* stream) {
    const char* name = "dn_linear8_forward";
    if (!L) return dn_fail(DN_ERR_INVALID_ARG, "dn_linear8_forward: null layer");
    if (L->segs != 1) return dn_fail(DN_ERR_INVALID_ARG, "dn_linear8_forward: a layer with segments reads cached rows");
    DN_TRY(check_matrix(x, dtype, rows, ldx, L->cin, name));
    DN_TRY(check_matrix(out, out_dtype, rows, ldo, L->n_out(), name));
    if (rows == 0) return DN_OK;
    const int xe = dtype == 1 ? 2 : 4, oe = out_dtype == 1 ? 2 : 4;
    if (share_bytes(x, ldx * xe, static_cast<int64_t>(L->cin) * xe, out, ldo * oe, static_cast<int64_t>(L->n_out()) * oe, rows))
        return dn_fail(DN_ERR_INVALID_ARG, "dn_linear8_forward: input and output overlap");
    ProductArgs a = product_args(L);
    a.rows = rows;
    a.out = out;
    a.ldo = ldo;
    DN_TRY(check_workspace(workspace_bytes_of(a, dtype), workspace, workspace_bytes, name));
    DeviceScope scope(L->device);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const Path path = path_of(a, dtype);
    if (path == Path::kFew) return launch_product_few(a, x, dtype, ldx, out_dtype, L->sms, s);
    if (path == Path::kFused) return launch_product_fused(a, x, ldx, out_dtype, L->sms, s);
    a.lda = round16(L->cin);
    auto* codes = static_cast<uint8_t*>(workspace);
    auto* scales = reinterpret_cast<float*>(codes + rows * a.lda);
    DN_TRY(launch_cache_write(CacheWrite{x, dtype, ldx, rows, L->cin, nullptr, 0, codes, a.lda, scales, rows, 8, L->cin,
                                         nullptr},
                              s));
    a.a = reinterpret_cast<const int8_t*>(codes);
    a.as = scales;
    a.a_rows = rows;
    return launch_product_tc(a, out_dtype, L->sms, s);
}

int dn_linear8_forward_nchw(dn_linear8* L, const void* input, int N, int H, int W, void* output, void* workspace,
                            int64_t workspace_bytes, void* stream) {
    const char* name = "dn_linear8_forward_nchw";
    if (!L) return dn_fail(DN_ERR_INVALID_ARG, "dn_linear8_forward_nchw: null layer");
    if (L->segs != 1) return dn_fail(DN_ERR_INVALID_ARG, "dn_linear8_forward_nchw: a layer with segments reads cached rows");
    if (N < 0 || H < 0 || W < 0) return dn_fail(DN_ERR_INVALID_ARG, "dn_linear8_forward_nchw: negative size");
    const int64_t hw = static_cast<int64_t>(H) * W;
    if (hw >= (1LL << 31)) return dn_fail(DN_ERR_INVALID_ARG, "dn_linear8_forward_nchw: rows outside [0, 2^31)");
    const int64_t rows = hw * N;
    DN_TRY(check_matrix(input, 1, rows, L->cin, L->cin, name));
    DN_TRY(check_matrix(output, 1, rows, L->n_out(), L->n_out(), name));
    if (rows == 0) return DN_OK;
    if (share_bytes(input, 0, rows * L->cin * 2, output, 0, rows * L->n_out() * 2, 1))
        return dn_fail(DN_ERR_INVALID_ARG, "dn_linear8_forward_nchw: input and output overlap");
    ProductArgs a = product_args(L);
    a.rows = rows;
    a.out = output;
    a.ldo = hw;
    a.planes = 1;
    DN_TRY(check_workspace(workspace_bytes_of(a, 1), workspace, workspace_bytes, name));
    DeviceScope scope(L->device);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (path_of(a, 1) == Path::kFused)
        return product_planes_takes(a, input) ? launch_product_planes(a, input, L->sms, s)
                                              : launch_product_fused(a, input, 0, 1, L->sms, s);
    a.lda = round16(L->cin);
    auto* codes = static_cast<uint8_t*>(workspace);
    auto* scales = reinterpret_cast<float*>(codes + rows * a.lda);
    const bool pairs = hw % 2 == 0 && aligned_to(input, 4);
    const cudaError_t e = pairs ? quantise_planes<2>(input, rows, L->cin, hw, codes, a.lda, scales, s)
                                : quantise_planes<1>(input, rows, L->cin, hw, codes, a.lda, scales, s);
    if (e != cudaSuccess) return dn_cuda_fail(e, "dn_linear8_forward_nchw: quantise launch");
    a.a = reinterpret_cast<const int8_t*>(codes);
    a.as = scales;
    a.a_rows = rows;
    return launch_product_tc(a, 1, L->sms, s);
}

int dn_linear8_forward_cached(dn_linear8* L, const void* codes, int64_t ld_codes, const float* scales, int64_t capacity,
                              int64_t page_rows, const int64_t* pages, int n_pages, int64_t rows, void* out,
                              int out_dtype, int64_t ldo, void* stream) {
    const char* name = "dn_linear8_forward_cached";
    if (!L || !pages) return dn_fail(DN_ERR_INVALID_ARG, "dn_linear8_forward_cached: null argument");
    if (n_pages != L->segs)
        return dn_fail_str(DN_ERR_INVALID_ARG, std::string(name) + ": " + std::to_string(n_pages) +
                                                   " pages for a layer of " + std::to_string(L->segs) + " segments");
    if (capacity < 0 || capacity >= (1LL << 31) || page_rows <= 0 || page_rows >= (1LL << 31) || rows > page_rows)
        return dn_fail(DN_ERR_INVALID_ARG, "dn_linear8_forward_cached: bad cache or page size");
    if (ld_codes < L->seg_c || ld_codes % 16 || !aligned_to(codes, 16) || !aligned_to(scales, 4))
        return dn_fail(DN_ERR_INVALID_ARG, "dn_linear8_forward_cached: codes rows must be 16-byte aligned and hold a segment");
    DN_TRY(check_matrix(out, out_dtype, rows, ldo, L->n_out(), name));
    ProductArgs a = product_args(L);
    for (int t = 0; t < n_pages; ++t) {
        if (pages[t] < 0 || pages[t] > (capacity - page_rows) / page_rows || capacity < page_rows)
            return dn_fail(DN_ERR_INVALID_ARG, "dn_linear8_forward_cached: page outside the cache");
        a.arow[t] = pages[t] * page_rows;
    }
    if (rows == 0) return DN_OK;
    if (!codes || !scales) return dn_fail(DN_ERR_INVALID_ARG, "dn_linear8_forward_cached: null cache");
    DeviceScope scope(L->device);
    a.a = static_cast<const int8_t*>(codes);
    a.lda = ld_codes;
    a.as = scales;
    a.a_rows = capacity;
    a.rows = rows;
    a.out = out;
    a.ldo = ldo;
    return launch_product_tc(a, out_dtype, L->sms, static_cast<cudaStream_t>(stream));
}

int dn_linear8_sync(dn_linear8* L, void* stream) {
    if (!L) return dn_fail(DN_ERR_INVALID_ARG, "dn_linear8_sync: null layer");
    DeviceScope scope(L->device);
    cudaError_t e = cudaStreamSynchronize(static_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) return dn_cuda_fail(e, "dn_linear8_sync");
    uint32_t word = 0;
    e = cudaMemcpy(&word, L->err, 4, cudaMemcpyDeviceToHost);
    if (e != cudaSuccess) return dn_cuda_fail(e, "dn_linear8_sync: error word");
    if (word) {
        cudaMemset(L->err, 0, 4);
        return dn_fail_str(DN_ERR_DEVICE, "linear8 kernel reported device error word " + std::to_string(word));
    }
    return DN_OK;
}

}  // extern "C"
