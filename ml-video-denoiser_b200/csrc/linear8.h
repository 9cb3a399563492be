// Internal interface of the 8-bit product: what a launch needs, shared by the
// layer (linear8.cu) and its kernels (linear8_tc.cu, linear8_fused.cu,
// linear8_planes.cu, linear8_few.cu).
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace dnb {

constexpr int kMaxSegments = 8;

struct ProductArgs {
    const int8_t* a;             // codes of the tokens, rows of lda bytes (a multiple of 16)
    int64_t lda, a_rows;         // a_rows: rows that `a` has
    const float* as;             // a scale per code row
    int64_t arow[kMaxSegments];  // first code row of each segment
    int segs, seg_c, seg_p;      // segments, their channels, their bytes in a weight row (a multiple of 16)
    const int8_t* w;             // [cout][ldw]
    int64_t ldw;
    // (scale, bias) of the channels: of output c at par[c], of a gated layer's
    // second factor at par[npad + c]; npad = n_out rounded up to 256, zeros
    // behind n_out, so that a tile's columns need no check.
    const float2* par;
    int npad;
    int cout, n_out, gate;
    int64_t rows;
    void* out;
    int64_t ldo;                 // row stride of out; planes: pixels of a plane
    int planes;                  // out[(m / ldo) * n_out + c][m % ldo] instead of out[m][c]
    uint32_t* err;
};

// The product on the tensor cores; out_dtype 0 FP32, 1 FP16; `sms` of the
// current device.
int launch_product_tc(const ProductArgs& a, int out_dtype, int sms, cudaStream_t s);

// One pass over FP16 tokens (rows with stride ldx, or planes) of a narrow
// layer; a.a, a.lda and a.as are not used. `takes` goes by sizes alone.
bool product_fused_takes(const ProductArgs& a);
int launch_product_fused(const ProductArgs& a, const void* x, int64_t ldx, int out_dtype, int sms, cudaStream_t s);

// Tile columns that hold all channels of a layer (gated ones need whole
// 32-column runs of each factor); the one-pass kernels take up to 256.
inline int fused_width(const ProductArgs& a) { return a.gate ? 2 * ((a.n_out + 31) / 32 * 32) : a.cout; }

// One pass over planes that TMA can address.
bool product_planes_takes(const ProductArgs& a, const void* x);
int launch_product_planes(const ProductArgs& a, const void* x, int sms, cudaStream_t s);

// One pass over a few token rows.
bool product_few_takes(const ProductArgs& a);
int launch_product_few(const ProductArgs& a, const void* x, int dtype, int64_t ldx, int out_dtype, int sms,
                       cudaStream_t s);

}  // namespace dnb
