// Device pieces shared by the kernels of the 8-bit product (linear8_tc.cu,
// linear8_fused.cu, linear8_planes.cu, linear8_few.cu), and the tensor maps they
// use.
#pragma once

#include <cuda.h>
#include <cuda_fp16.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <cstdint>

#include "sm100.cuh"

namespace dnb {

// A tensor map over a [rows][cols] matrix of `esz`-byte elements, row stride
// ld elements, boxes of box_rows x box_cols swizzled by their width (32, 64 or
// 128 bytes). Base and row stride are multiples of 16 bytes; a load reads what
// lies behind a row up to the next multiple of 16 bytes, and zeros from there on.
int linear8_map(CUtensorMap* m, CUtensorMapDataType type, int esz, const void* base, int64_t cols, int64_t rows,
                int64_t ld, int box_cols, int box_rows);

// Whether TMA may store rows of n elements: it cuts what lies behind a row only
// to 16 bytes, so that a row that is no multiple of them would run over what is
// beside it.
inline bool tma_rows(const void* out, int esz, int64_t n, int64_t ld) {
    return reinterpret_cast<uintptr_t>(out) % 16 == 0 && ld * esz % 16 == 0 && n * esz % 16 == 0 && ld >= n;
}

// The same over FP16 planes [images][channels][pixels], boxes of box_ch x
// box_px pixels of one image (64 or 32, swizzled by their 128 or 64 bytes).
int linear8_planes_map(CUtensorMap* m, const void* base, int64_t pixels, int64_t channels, int64_t images, int box_px,
                       int box_ch);

// CTAs per SM of a kernel that allocates tmem_cols TMEM columns: by registers
// (allocated in eights a thread), shared memory (228 KB, 1 KB a CTA reserved)
// and TMEM (512 columns). The occupancy query answers 1 for kernels that use
// TMEM. `cache` (per device) keeps the answer; sets the kernel's shared-memory
// limit, smem_limit, on the first call.
template <typename Kernel>
cudaError_t tmem_kernel_ctas(Kernel kernel, int threads, int smem, int smem_limit, int tmem_cols, int (&cache)[64],
                             int* per_sm) {
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    *per_sm = e == cudaSuccess && device < 64 ? cache[device] : 0;
    if (e != cudaSuccess || *per_sm > 0) return e;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_limit);
    cudaFuncAttributes at{};
    if (e == cudaSuccess) e = cudaFuncGetAttributes(&at, kernel);
    if (e != cudaSuccess) return e;
    const int by_regs = 65536 / (std::max(1, (at.numRegs + 7) / 8 * 8) * threads);
    const int by_smem = 233472 / (smem + static_cast<int>(at.sharedSizeBytes) + 1024);
    *per_sm = std::max(1, std::min({by_regs, by_smem, 512 / tmem_cols}));
    if (device < 64) cache[device] = *per_sm;
    return e;
}

__host__ __device__ constexpr uint32_t idesc_s8(int M, int N) {
    return (2u << 4)                                 // D: s32
           | (1u << 7) | (1u << 10)                  // A, B: s8
           | (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}

__device__ __forceinline__ void mma_s8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                       uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, int (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,"
        "%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}

// An output is (sum s) w + b, s its token's scale, w and b its channel's: a sum
// is below 2^31 (all segments of a token together), so that sum * s stays below
// 2^128 as long as s is below this. Tokens with a larger scale (FP32 values of
// 2^103 or more; FP16 ones never have one) take (sum w) s + b: there sum * w
// overflows only where the output does.
constexpr float kLargeScale = 7.9228163e28f;  // 2^96

__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void stmatrix4_trans(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a), "r"(b), "r"(c),
                 "r"(d)
                 : "memory");
}
// 16 lanes x 32 columns: r[4 k + i] is (lane t / 4 + 8 (i / 2), column 8 k + 2 (t % 4) + i % 2).
__device__ __forceinline__ void tmem_ld_16x32(uint32_t taddr, int (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}

// One lane of a converged warp, always the same one. Roles of a single thread
// run their loops with the whole warp and elect a lane around each MMA, commit
// or copy only: the loop stays warp-uniform, so that descriptors, coordinates
// and barrier addresses live in uniform registers. Under `if (lane == 0)` every
// operand of an MMA was moved there one by one, and a loop of two MMAs took
// 1100 cycles.
__device__ __forceinline__ bool elect_one() {
    uint32_t e;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(e));
    return e != 0;
}

// After a wait that ran out: the MMAs that the elected lane of this warp has
// issued end before the CTA gives back its TMEM and shared memory. `bar`: a
// barrier of one arrival, not used otherwise. Warp-wide.
__device__ __forceinline__ void drain_mmas(uint64_t* bar) {
    if (elect_one()) {
        mma_commit(bar);
        mbar_wait(bar, 0, 100000000ull);
    }
    __syncwarp();
}

// The warp's index as a value that the compiler knows to be warp-uniform.
__device__ __forceinline__ int warp_index() { return __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x) >> 5, 0); }

__device__ __forceinline__ void put(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }

// 16 bytes of a row from 8 (FP16) or 4 (FP32) values.
__device__ __forceinline__ uint4 pack16(const float* y, __half*) {
    return make_uint4(pack_half2(y[0], y[1]), pack_half2(y[2], y[3]), pack_half2(y[4], y[5]), pack_half2(y[6], y[7]));
}
__device__ __forceinline__ uint4 pack16(const float* y, float*) {
    return make_uint4(__float_as_uint(y[0]), __float_as_uint(y[1]), __float_as_uint(y[2]), __float_as_uint(y[3]));
}

// Rows that TMA cannot store (address, stride or length no multiple of 16 bytes): a
// warp's block of 32 rows x 32 columns (a lane holds a row's columns c .. c +
// 31) goes through its 4 KB staging tile and leaves row by row, lanes along the
// columns. (Stored by each lane along its own row, 2 bytes at a time, 522240 x
// 60 outputs took 300 us more than the product.) `pairs`: rows are 4-byte
// aligned. Warp-wide.
__device__ __forceinline__ void store_block32(uint8_t* stg, const float (&y)[32], __half* out, int64_t ldo, int64_t row0,
                                              int64_t rows, int c, int n_out, bool pairs) {
    const int lane = threadIdx.x & 31;
    uint32_t* w = reinterpret_cast<uint32_t*>(stg);  // word i of row r at r * 16 + (i ^ (r / 2)): no bank conflicts
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 16; ++i) w[lane * 16 + (i ^ (lane >> 1))] = pack_half2(y[2 * i], y[2 * i + 1]);
    __syncwarp();
    const int live = static_cast<int>(rows - row0 < 32 ? rows - row0 : 32);
    // Whole blocks with all their loads before the first store: one by one, a
    // block took 1450 cycles (pairs) or 1200.
    if (live == 32 && c + 32 <= n_out) {
        if (pairs) {
            uint32_t v[16];
            __half* o = out + (row0 + (lane >> 4)) * ldo + c + 2 * (lane & 15);
#pragma unroll
            for (int k = 0; k < 16; ++k) v[k] = w[(2 * k + (lane >> 4)) * 16 + ((lane & 15) ^ k)];
#pragma unroll
            for (int k = 0; k < 16; ++k, o += 2 * ldo) *reinterpret_cast<uint32_t*>(o) = v[k];
        } else {
            uint32_t v[32];
            __half* o = out + row0 * ldo + c + lane;
#pragma unroll
            for (int r = 0; r < 32; ++r) v[r] = w[r * 16 + ((lane >> 1) ^ (r >> 1))];
#pragma unroll
            for (int r = 0; r < 32; ++r, o += ldo)
                *o = __ushort_as_half(static_cast<unsigned short>(lane & 1 ? v[r] >> 16 : v[r]));
        }
    } else if (pairs) {
        const int i = lane & 15, col = c + 2 * i;
        for (int r = lane >> 4; r < live; r += 2) {
            const uint32_t v = w[r * 16 + (i ^ (r >> 1))];
            __half* o = out + (row0 + r) * ldo + col;
            if (col + 1 < n_out)
                *reinterpret_cast<uint32_t*>(o) = v;
            else if (col < n_out)
                *o = __ushort_as_half(static_cast<unsigned short>(v));
        }
    } else if (c + lane < n_out) {
        for (int r = 0; r < live; ++r) {
            const uint32_t v = w[r * 16 + ((lane >> 1) ^ (r >> 1))];
            out[(row0 + r) * ldo + c + lane] = __ushort_as_half(static_cast<unsigned short>(lane & 1 ? v >> 16 : v));
        }
    }
}
__device__ __forceinline__ void store_block32(uint8_t* stg, const float (&y)[32], float* out, int64_t ldo, int64_t row0,
                                              int64_t rows, int c, int n_out, bool) {
    const int lane = threadIdx.x & 31;
    float* w = reinterpret_cast<float*>(stg);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 32; ++i) w[lane * 32 + (i ^ lane)] = y[i];
    __syncwarp();
    const int live = static_cast<int>(rows - row0 < 32 ? rows - row0 : 32);
    if (live == 32 && c + 32 <= n_out) {
        float v[32];
        float* o = out + row0 * ldo + c + lane;
#pragma unroll
        for (int r = 0; r < 32; ++r) v[r] = w[r * 32 + (lane ^ r)];
#pragma unroll
        for (int r = 0; r < 32; ++r, o += ldo) *o = v[r];
    } else if (c + lane < n_out)
        for (int r = 0; r < live; ++r) out[(row0 + r) * ldo + c + lane] = w[r * 32 + (lane ^ r)];
}

// 32 channels of a pixel into planes of `plane` pixels; o: channel c's value.
template <typename T>
__device__ __forceinline__ void store_planes32(T* o, int64_t plane, const float (&y)[32], int c, int n_out) {
#pragma unroll
    for (int i = 0; i < 32; ++i)
        if (c + i < n_out) put(o + i * plane, y[i]);
}

}  // namespace dnb
