/*
 * denoiser_b200_quant.h — C-ABI of the 8-bit serving operators: a row cache
 * that is quantised as it is written (8 or 4 bits), and Linear8, the product
 * of tokens with a weight matrix in 8-bit integers. The reference has no
 * counterpart; they stand beside the layers of denoiser_b200_layers.h (a 1x1
 * Conv2dLayer is this product over the pixels of its planes) and the frame
 * caches of the temporal models.
 *
 * Quantisation of a group x_0 .. x_{g-1} of a row to b bits, qmax = 127 (8)
 * or 7 (4):
 *   s   = max(fl32(max |x_k| * fl32(1 / qmax)), 2^-126)
 *   q_k = the whole number nearest to x_k / s, halves to the even one
 * (x_k and s taken exactly), and q_k s stands for x_k. A group that holds a
 * NaN or an infinity has s = NaN and codes 0, so everything computed from it
 * is NaN.
 *
 * Tensors are device pointers; dtype is that of dn_weights_info (0 FP32,
 * 1 FP16); `stream` is a cudaStream_t (NULL = legacy default stream), and the
 * calls are asynchronous on it, allocate nothing and may be captured into a
 * graph, but for the create functions. Every function returns DN_OK or a
 * negative DN_ERR_* code (denoiser_b200.h); dn_last_error() has the message.
 */
#ifndef DENOISER_B200_QUANT_H
#define DENOISER_B200_QUANT_H

#include "denoiser_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ------------------------------------------------------------------------
 * Row cache. `capacity` rows of `cols` values: codes, row r at codes + r *
 * ld_codes bytes (8 bits: one code a byte; 4 bits: two, the even column in
 * the low half), and scales [capacity][cols / group]. `group` divides cols;
 * 0 = cols (one scale a row). Rows are counted in 64 bits, so a cache may
 * exceed 2^32 bytes; capacity < 2^31. All `capacity` rows have their ld_codes
 * bytes; those behind a row's codes are not written. Any alignment of `codes`
 * and ld_codes is right; multiples of 16 are fastest. Everything else is
 * aligned to its type (DN_ERR_INVALID_ARG otherwise).
 *
 * The launchers run on the current device, which `stream` and the tensors
 * belong to. Calls that may overlap must not write what another one reads or
 * writes.
 *
 * A row number outside [0, capacity): negative ones are skipped in silence
 * (padding); others are skipped too and set *err_dev (a device word, may be
 * NULL) to a non-zero value.
 * ------------------------------------------------------------------------ */

/* Quantise `rows` rows of x (row stride ldx elements, unit column stride)
 * into the cache rows slots[i] (device int64), or row0 + i where slots is
 * NULL (which must then fit). A slot that occurs twice holds the last of its
 * rows. The source must not overlap the cache. */
int dn_launch_cache_write(const void* x, int dtype, int64_t ldx, int64_t rows, int cols, const int64_t* slots,
                          int64_t row0, void* codes, int64_t ld_codes, float* scales, int64_t capacity, int bits,
                          int group, uint32_t* err_dev, void* stream);

/* Read back rows: out row i (row stride ldo elements) = cache row slots[i],
 * or row0 + i where slots is NULL. Rows of skipped slots stay as they were, and
 * so does what lies between rows. `out` must not overlap the cache. */
int dn_launch_cache_read_rows(const void* codes, int64_t ld_codes, const float* scales, int64_t capacity, int cols,
                              int bits, int group, const int64_t* slots, int64_t row0, int64_t rows, void* out,
                              int dtype, int64_t ldo, uint32_t* err_dev, void* stream);

/* Read back sequences through page tables. Page p is the cache rows
 * [p * page_rows, (p + 1) * page_rows); position i of sequence b is row
 * i % page_rows of page table[b * table_ld + i / page_rows] (device int32).
 * out[b * out_batch + i * ldo ..] = that row for i < min(lengths[b],
 * max_rows, table_cols * page_rows) (lengths: device int32, NULL = max_rows;
 * negative = 0). Rows behind a sequence's length and rows of negative pages
 * stay as they were. A page may occur more than once. */
int dn_launch_cache_read_pages(const void* codes, int64_t ld_codes, const float* scales, int64_t capacity, int cols,
                               int bits, int group, int64_t page_rows, const int32_t* table, int64_t table_ld,
                               int64_t table_cols, const int32_t* lengths, int batch, int64_t max_rows, void* out,
                               int dtype, int64_t out_batch, int64_t ldo, uint32_t* err_dev, void* stream);

/* ------------------------------------------------------------------------
 * Linear8: y[m, n] = s_x[m] s_w[n] sum_k q_x[m, k] q_w[n, k] + bias[n], the
 * tokens quantised to 8 bits with a scale each, the weights with a scale for
 * each output channel; the sum is exact in int32, the rest FP32, rounded once
 * to the output type; what lies between overflows only where the product (with
 * segments: a segment's part of it) does, whatever the scales. With `gate` (SimpleGate) the output has half the
 * channels: out[m, c] = y[m, c] * y[m, c + Cout / 2].
 *
 * segments > 1: the input channels are `segments` equal runs, each with a
 * scale of its own per token: the layer of dn_linear8_forward_cached.
 * ------------------------------------------------------------------------ */
typedef struct dn_linear8 dn_linear8;

/* Weight (Cout, Cin) or (Cout, Cin, 1, 1) and optional bias (Cout) from the
 * store, quantised onto `device`. DN_ERR_NOT_FOUND for a missing key,
 * DN_ERR_FORMAT for another shape, DN_ERR_INVALID_ARG for an odd Cout with
 * gate, a Cin that segments does not divide or a device that is not there,
 * DN_ERR_UNSUPPORTED for Cin > 131072 (the int32 sum) or segments > 8. */
int dn_linear8_create(const dn_weights* store, const char* weight_name, const char* bias_name, int gate, int segments,
                      int device, dn_linear8** out);
/* The same from device memory of `device`: weight [cout][cin] with row stride
 * ldw elements, bias [cout] of the same dtype or NULL, read after the work
 * queued on `stream`; returns once the layer holds its copy. */
int dn_linear8_create_device(const void* weight, int dtype, int64_t ldw, const void* bias, int cout, int cin, int gate,
                             int segments, int device, void* stream, dn_linear8** out);
int dn_linear8_destroy(dn_linear8* layer);
/* Channels of the input and of the output (half of Cout with gate). */
int dn_linear8_info(const dn_linear8* layer, int* out_channels, int* in_channels, int* gate, int* segments);
/* Bytes of device workspace that dn_linear8_forward over `rows` tokens of
 * `dtype` needs, or with nchw dn_linear8_forward_nchw over N * H * W = `rows`
 * pixels (16-byte aligned; 0 = none). Calls that may overlap need a workspace each; the layer
 * itself may be shared by any number of calls. */
int dn_linear8_workspace(const dn_linear8* layer, int64_t rows, int dtype, int nchw, int64_t* bytes);
/* Token rows: x [rows][Cin] (row stride ldx) -> out [rows][out_channels] (row
 * stride ldo), unit column strides, the two apart from each other (columns
 * side by side of one buffer are; DN_ERR_INVALID_ARG otherwise). Segments must
 * be 1. */
int dn_linear8_forward(dn_linear8* layer, const void* x, int dtype, int64_t ldx, int64_t rows, void* out, int out_dtype,
                       int64_t ldo, void* workspace, int64_t workspace_bytes, void* stream);
/* A 1x1 convolution over NCHW planes: input (N, Cin, H, W) -> output
 * (N, out_channels, H, W), both FP16 and contiguous, apart from each other; a
 * pixel is a token. */
int dn_linear8_forward_nchw(dn_linear8* layer, const void* input, int N, int H, int W, void* output, void* workspace,
                            int64_t workspace_bytes, void* stream);
/* Straight from an 8-bit row cache with one scale a row and
 * cols = Cin / segments: out row i = the product over cache rows
 * pages[t] * page_rows + i, t < segments, side by side (the temporal fusion
 * of T cached frames), i < rows <= page_rows. `pages` is a host array; every
 * page must lie in the cache. No workspace. ld_codes a multiple of 16, codes
 * 16-byte aligned. */
int dn_linear8_forward_cached(dn_linear8* layer, const void* codes, int64_t ld_codes, const float* scales,
                              int64_t capacity, int64_t page_rows, const int64_t* pages, int n_pages, int64_t rows,
                              void* out, int out_dtype, int64_t ldo, void* stream);
/* Synchronise `stream` and report a device-side error of the layer's kernels. */
int dn_linear8_sync(dn_linear8* layer, void* stream);

#ifdef __cplusplus
} /* extern "C" */
#endif

#endif /* DENOISER_B200_QUANT_H */
