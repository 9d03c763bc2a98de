// Helpers of the kernels that work on the rows of a matrix in fp32, bf16 or fp16 (layer norm, policy loss,
// Newton-Schulz): element types, 16-byte packs, and reductions over the threads that share a row.
#pragma once
#include "common.h"

namespace step {

typedef _Float16 f16;
typedef __bf16 bf16;

template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
    T v[N];
};

// element e of an array whose type is known at run time only (weights: read once per block)
static __device__ __forceinline__ float load_as(const void* p, size_t e, int dtype) {
    if (dtype == STEP_BF16) return (float)((const bf16*)p)[e];
    if (dtype == STEP_F16) return (float)((const f16*)p)[e];
    return ((const float*)p)[e];
}
static __device__ __forceinline__ void store_as(void* p, size_t e, int dtype, float v) {
    if (dtype == STEP_BF16) ((bf16*)p)[e] = (bf16)v;
    else if (dtype == STEP_F16) ((f16*)p)[e] = (f16)v;
    else ((float*)p)[e] = v;
}

static inline int elem_bytes(int dtype) { return dtype == STEP_F32 ? 4 : dtype == STEP_BF16 || dtype == STEP_F16 ? 2 : 0; }

// G threads share a row; GW = how many of them are in one wave
template <int G, typename F>
static __device__ __forceinline__ float group_wave_reduce(float v, F f) {
#pragma unroll
    for (int o = (G < 64 ? G : 64) / 2; o > 0; o >>= 1) v = f(v, __shfl_xor(v, o, 64));
    return v;
}

}  // namespace step
