// The quantising row writer of row_cache.cu, also the first pass of the
// 8-bit product over tokens.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace dnb {

struct CacheWrite {
    const void* x;         // rows of `cols` values, stride ldx elements
    int dtype;             // 0 FP32, 1 FP16
    int64_t ldx, rows;
    int cols;
    const int64_t* slots;  // cache row of row i, or null: row0 + i
    int64_t row0;
    uint8_t* codes;
    int64_t ldc;           // bytes
    float* scales;         // [capacity][cols / group]
    int64_t capacity;
    int bits, group;
    uint32_t* err;
};

// Validated by the caller: 0 < cols, group divides cols, rows >= 0.
int launch_cache_write(const CacheWrite& p, cudaStream_t s);

}  // namespace dnb
