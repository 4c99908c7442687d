// Shared pieces of the operators for blocks of language models (kernels_w4.hip, kernels_grouped.hip, norm_res.h).
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <atomic>

#include "qcnn_internal.h"

namespace qcnn {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
// 16 bytes at any address: global loads and stores of gfx950 take any, and 16 bytes that cross a cache line cost one line more.
typedef u32x4 u32x4_any __attribute__((aligned(1)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

struct bf16_t {
    uint16_t bits;
};
typedef _Float16 f16_t;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(f16_t v) { return (float)v; }
__device__ __forceinline__ float to_f32(bf16_t v) { return __uint_as_float((unsigned)v.bits << 16); }

__device__ __forceinline__ void from_f32(float v, float &o) { o = v; }
__device__ __forceinline__ void from_f32(float v, f16_t &o) { o = (f16_t)v; }
__device__ __forceinline__ void from_f32(float v, bf16_t &o)  // round to nearest even, v_cvt_pk_bf16_f32
{
    const __bf16 r = (__bf16)v;
    __builtin_memcpy(&o, &r, 2);
}

// One value into an output whose type is known at run time (uniform over the launch).
__device__ __forceinline__ void store_typed(void *p, size_t i, int type, float v)
{
    if (type == QCNN_F32) {
        ((float *)p)[i] = v;
    } else if (type == QCNN_F16) {
        ((f16_t *)p)[i] = (f16_t)v;
    } else {
        bf16_t b;
        from_f32(v, b);
        ((bf16_t *)p)[i] = b;
    }
}

// 16 x 16 outputs, 32 k: lane l holds k 8 (l >> 4) .. 8 (l >> 4) + 7 of row l & 15 of either operand.
__device__ __forceinline__ f32x4 mma(f16_t, u32x4 a, u32x4 b, f32x4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(bf16_t, u32x4 a, u32x4 b, f32x4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Waits until at most min(runs, MOST) runs' loads, and nothing else, are on their way.
template <int MOST, int LOADS>
__device__ __forceinline__ void wait_for_all_but(int runs)
{
    if constexpr (MOST <= 0) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    } else {
        if (runs >= MOST)
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(LOADS * MOST) : "memory");
        else
            wait_for_all_but<MOST - 1, LOADS>(runs);
    }
}

__device__ __forceinline__ float sigmoid(float v) { return 1.f / (1.f + __expf(-v)); }

// ReLU as the library's layers have it, with NaN kept; SiLU v * sigmoid(v), -0 where e^-v overflows.
__device__ __forceinline__ float block_act(float v, int act)
{
    if (act == QCNN_ACT_RELU) return v < 0.f ? 0.f : v;
    if (act == QCNN_ACT_SILU) return v / (1.f + __expf(-v));
    return v;
}

// Workgroups of a launch whose kernel finds its work by itself, counted along x and y: a grid's width times the workgroup's threads
// has to stay below 2^32, so more than 2^21 workgroups stand in rows of 2^21; those too many in the last row find nothing.
constexpr unsigned GRID_ROW = 1u << 21;
__device__ __forceinline__ unsigned workgroup() { return blockIdx.y * GRID_ROW + blockIdx.x; }
inline hipError_t grid_of(unsigned long long groups, dim3 &grid)
{
    const unsigned long long rows = (groups + GRID_ROW - 1) / GRID_ROW;
    if (rows > 2047) return hipErrorNotSupported;  // workgroup() has 32 bits
    grid = rows > 1 ? dim3(GRID_ROW, (unsigned)rows) : dim3((unsigned)groups);
    return hipSuccess;
}

// Lets kernel `fn` have `bytes` of LDS beyond the 64 KB that need no asking; `asked` holds a bit for each device on which that has
// been done (asking again at every launch is 0.5 us of the caller's time).
inline hipError_t allow_lds(const void *fn, int bytes, std::atomic<unsigned long long> &asked)
{
    if (bytes <= 65536) return hipSuccess;
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return e;
    const unsigned long long bit = 1ull << (dev & 63);
    if (dev < 64 && (asked.load(std::memory_order_relaxed) & bit)) return hipSuccess;
    e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == hipSuccess && dev < 64) asked.fetch_or(bit, std::memory_order_relaxed);
    return e;
}

hipError_t launch_matvec_w4(const qcnn_matvec_w4_t &a, hipStream_t s);
hipError_t launch_grouped_matmul(const qcnn_grouped_matmul_t &a, hipStream_t s);
template <typename T>
hipError_t norm_res_of(const qcnn_norm_res_t &a, hipStream_t s);
inline hipError_t launch_norm_res(const qcnn_norm_res_t &a, hipStream_t s)
{
    if (a.type == QCNN_F32) return norm_res_of<float>(a, s);
    if (a.type == QCNN_F16) return norm_res_of<f16_t>(a, s);
    return norm_res_of<bf16_t>(a, s);
}

}  // namespace qcnn
