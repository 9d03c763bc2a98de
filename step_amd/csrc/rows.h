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

// 16 bytes (or fewer) at any element: the hardware takes unaligned vector accesses
template <typename T, int N>
static __device__ __forceinline__ Pack<T, N> load_pack(const T* p) {
    Pack<T, N> q;
    __builtin_memcpy(&q, p, sizeof(q));
    return q;
}
template <typename T, int N>
static __device__ __forceinline__ void store_pack(T* p, const Pack<T, N>& q) {
    __builtin_memcpy(p, &q, sizeof(q));
}

// Who has which columns of a row of (NV - LAST) G N < cols <= NV G N, cols >= N elements: thread `lane` of G has NV packs of N, pack i
// at column (i G + lane) N.  Only the last LAST packs may not fit: one that would end behind the row lies at the row's end instead,
// and its first dup(i) elements, which belong to the pack before, are not its own; one that would begin behind the row owns
// nothing (dup(i) >= N).  So nothing outside the row is touched and no load waits for a branch.
template <int N, int NV, int G, int LAST = 1>
struct Columns {
    int cols, lane;
    __device__ __forceinline__ int at(int i) const {
        const int c = (i * G + lane) * N;
        return i + LAST < NV || c < cols - N ? c : cols - N;
    }
    __device__ __forceinline__ int dup(int i) const { return (i * G + lane) * N - at(i); }
    __device__ __forceinline__ bool mine(int i, int e) const { return i + LAST < NV || e >= dup(i); }
    template <typename T>
    __device__ __forceinline__ void load(Pack<T, N>* v, const T* row) const {
#pragma unroll
        for (int i = 0; i < NV; ++i) v[i] = load_pack<T, N>(row + at(i));
    }
    // what is not the thread's own becomes `x`
    template <typename T>
    __device__ __forceinline__ void fill(Pack<T, N>* v, T x) const {
#pragma unroll
        for (int i = NV > LAST ? NV - LAST : 0; i < NV; ++i) {
            const int d = dup(i);
#pragma unroll
            for (int e = 0; e < N; ++e) v[i].v[e] = e >= d ? v[i].v[e] : x;
        }
    }
    template <typename T>
    __device__ __forceinline__ void store(T* row, int i, const Pack<T, N>& v) const {
        const int d = i + LAST < NV ? 0 : dup(i);
        if (d == 0) store_pack<T, N>(row + at(i), v);
        else if (d < N)
#pragma unroll
            for (int e = 1; e < N; ++e)
                if (e >= d) row[cols - N + e] = v.v[e];
    }
    template <typename T>
    __device__ __forceinline__ void store(T* row, const Pack<T, N>* v) const {
#pragma unroll
        for (int i = 0; i < NV; ++i) store(row, i, v[i]);
    }
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

// a neighbour's value: quad_perm, row_half_mirror, row_mirror (data-parallel primitives: no LDS)
template <int CTRL>
static __device__ __forceinline__ float dpp(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
// f over the four values that the rows of 16 threads hold, the same in all threads
template <typename F>
static __device__ __forceinline__ float rows16(float v, F f) {
    const int x = __builtin_bit_cast(int, v);
    const float p = __builtin_bit_cast(float, __builtin_amdgcn_readlane(x, 0)), q = __builtin_bit_cast(float, __builtin_amdgcn_readlane(x, 16)),
                r = __builtin_bit_cast(float, __builtin_amdgcn_readlane(x, 32)), t = __builtin_bit_cast(float, __builtin_amdgcn_readlane(x, 48));
    return f(f(p, q), f(r, t));
}
// f over the 8, 16 or 64 threads of a wave that share a row, the same bits in all of them (f commutes)
template <int G, typename F>
static __device__ __forceinline__ float wave_reduce(float v, F f) {
    v = f(v, dpp<0xb1>(v));
    v = f(v, dpp<0x4e>(v));
    v = f(v, dpp<0x141>(v));
    if constexpr (G >= 16) v = f(v, dpp<0x140>(v));
    if constexpr (G >= 64) v = rows16(v, f);
    return v;
}

}  // namespace step
