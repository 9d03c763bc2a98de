// Layer norm over the rows of a (rows, cols) matrix, forward and backward, fp32 / bf16 / fp16 tensors.
//
//   mu = mean x,  var = mean (x - mu)^2,  r = 1 / sqrt(var + eps),  xhat = (x - mu) r,  y = xhat w + b
//   t = dy w:  dx = r (t - mean t - xhat mean(t xhat)),  dw = SUM_rows dy xhat,  db = SUM_rows dy
//
// Memory-bound both ways: forward 2 and backward 3 elements moved per element.  A row stays in the registers of the G
// threads that share it between the statistics and the result, so each tensor is moved once.  G is the smallest of
// 8 / 64 / 256 / 1024 whose threads hold the row in at most two 16-byte packs each (plan() below): short rows share a
// wave, long ones have a block.  The statistics are combined pairwise from (count, mean, sum of squared deviations),
// which loses nothing to a mean far from zero and takes one reduction instead of two.
// dw and db: a block keeps its columns' sums in fp32 registers over all its rows, writes one line of partial sums, and a
// second launch adds the lines in a fixed order - the same bits every time, no atomics.
#include "rows.h"

namespace {
using namespace step;

struct Stat {
    float n, mean, m2;
};
// pairwise combination of two sets of values; the same result whichever half a thread is in is not needed: the first
// thread's value is broadcast
__device__ __forceinline__ Stat combine(const Stat a, const Stat b) {
    const float n = a.n + b.n;
    const float f = n > 0.f ? b.n / n : 0.f;
    const float d = b.mean - a.mean;
    return Stat{n, a.mean + d * f, a.m2 + b.m2 + d * d * (a.n * f)};
}

template <int G>
__device__ __forceinline__ Stat group_stat(Stat s, Stat* sm) {
#pragma unroll
    for (int o = 1; o < (G < 64 ? G : 64); o <<= 1) {
        const Stat t{__shfl_xor(s.n, o, 64), __shfl_xor(s.mean, o, 64), __shfl_xor(s.m2, o, 64)};
        s = combine(s, t);
    }
    if constexpr (G <= 64) {
        const int src = (threadIdx.x & 63) & ~(G - 1);
        return Stat{s.n, __shfl(s.mean, src, 64), __shfl(s.m2, src, 64)};
    } else {
        __syncthreads();                       // the last row's readers are done with sm
        if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = s;
        __syncthreads();
        Stat r = sm[0];
#pragma unroll
        for (int i = 1; i < G / 64; ++i) r = combine(r, sm[i]);
        return r;
    }
}

template <int G>
__device__ __forceinline__ void group_sum2(float& a, float& b, float* sm) {
#pragma unroll
    for (int o = 1; o < (G < 64 ? G : 64); o <<= 1) {
        a += __shfl_xor(a, o, 64);
        b += __shfl_xor(b, o, 64);
    }
    if constexpr (G > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) {
            sm[2 * (threadIdx.x >> 6)] = a;
            sm[2 * (threadIdx.x >> 6) + 1] = b;
        }
        __syncthreads();
        a = sm[0];
        b = sm[1];
#pragma unroll
        for (int i = 1; i < G / 64; ++i) {
            a += sm[2 * i];
            b += sm[2 * i + 1];
        }
    }
}

template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T* p, float* v) {
    const Pack<T, VEC> q = *(const Pack<T, VEC>*)p;
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = (float)q.v[e];
}
template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const float* v) {
    Pack<T, VEC> q;
#pragma unroll
    for (int e = 0; e < VEC; ++e) q.v[e] = (T)v[e];          // the result's only rounding
    *(Pack<T, VEC>*)p = q;
}

template <typename T, int VEC, int NV, int G>
__global__ __launch_bounds__(G < 256 ? 256 : G) void ln_fwd_kernel(const T* __restrict__ x, const void* __restrict__ w,
                                                                   const void* __restrict__ b, T* __restrict__ y,
                                                                   float* __restrict__ mean, float* __restrict__ rstd,
                                                                   long long rows, int cols, int wdtype, float eps) {
    constexpr int BLOCK = G < 256 ? 256 : G, RPB = BLOCK / G;
    __shared__ Stat sm[G > 64 ? G / 64 : 1];
    const int lane = threadIdx.x % G;
    float wv[NV][VEC], bv[NV][VEC];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const int c = (i * G + lane) * VEC + e;
            wv[i][e] = w && c < cols ? load_as(w, c, wdtype) : 1.f;
            bv[i][e] = b && c < cols ? load_as(b, c, wdtype) : 0.f;
        }
    for (long long r0 = (long long)blockIdx.x * RPB; r0 < rows; r0 += (long long)gridDim.x * RPB) {
        const long long row = r0 + threadIdx.x / G;
        const bool live = row < rows;
        const T* xr = x + (size_t)row * cols;
        float v[NV][VEC];
        float s = 0.f;
        int n = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * G + lane) * VEC;
            if (live && c < cols) {
                load_vec<T, VEC>(xr + c, v[i]);
                n += VEC;
#pragma unroll
                for (int e = 0; e < VEC; ++e) s += v[i][e];
            }
        }
        Stat st{(float)n, n ? s / (float)n : 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (live && (i * G + lane) * VEC < cols)
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float d = v[i][e] - st.mean;
                    st.m2 += d * d;
                }
        st = group_stat<G>(st, sm);
        const float inv = 1.f / sqrtf(st.m2 / (float)cols + eps);
        if (!live) continue;
        if (lane == 0 && mean) {
            mean[row] = st.mean;
            rstd[row] = inv;
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * G + lane) * VEC;
            if (c < cols) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[i][e] = (v[i][e] - st.mean) * inv * wv[i][e] + bv[i][e];
                store_vec<T, VEC>(y + (size_t)row * cols + c, v[i]);
            }
        }
    }
}

template <typename T, int VEC, int NV, int G>
__global__ __launch_bounds__(G < 256 ? 256 : G) void ln_bwd_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                                                                   const void* __restrict__ w,
                                                                   const float* __restrict__ mean,
                                                                   const float* __restrict__ rstd, T* __restrict__ dx,
                                                                   float* __restrict__ part, long long rows, int cols,
                                                                   int wdtype) {
    constexpr int BLOCK = G < 256 ? 256 : G, RPB = BLOCK / G;
    __shared__ float sm[G > 64 ? 2 * G / 64 : 1];
    __shared__ float acc[RPB > 1 ? BLOCK * NV * VEC : 1];
    const int lane = threadIdx.x % G, group = threadIdx.x / G;
    float wv[NV][VEC], dw[NV][VEC], db[NV][VEC];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const int c = (i * G + lane) * VEC + e;
            wv[i][e] = w && c < cols ? load_as(w, c, wdtype) : 1.f;
            dw[i][e] = db[i][e] = 0.f;
        }
    const float inv_c = 1.f / (float)cols;
    for (long long r0 = (long long)blockIdx.x * RPB; r0 < rows; r0 += (long long)gridDim.x * RPB) {
        const long long row = r0 + group;
        const bool live = row < rows;
        const size_t at = (size_t)row * cols;
        const float mu = live ? mean[row] : 0.f, inv = live ? rstd[row] : 0.f;
        float g[NV][VEC], xh[NV][VEC];
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * G + lane) * VEC;
            if (live && c < cols) {
                load_vec<T, VEC>(dy + at + c, g[i]);
                load_vec<T, VEC>(x + at + c, xh[i]);
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    xh[i][e] = (xh[i][e] - mu) * inv;
                    dw[i][e] += g[i][e] * xh[i][e];
                    db[i][e] += g[i][e];
                    g[i][e] *= wv[i][e];
                    s1 += g[i][e];
                    s2 += g[i][e] * xh[i][e];
                }
            }
        }
        if (dx) {
            group_sum2<G>(s1, s2, sm);
            s1 *= inv_c;
            s2 *= inv_c;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (i * G + lane) * VEC;
                if (live && c < cols) {
#pragma unroll
                    for (int e = 0; e < VEC; ++e) g[i][e] = inv * (g[i][e] - s1 - xh[i][e] * s2);
                    store_vec<T, VEC>(dx + at + c, g[i]);
                }
            }
        }
    }
    if (!part) return;
    float* line = part + (size_t)blockIdx.x * 2 * cols;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        if constexpr (RPB > 1) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int e = 0; e < VEC; ++e)
                    acc[group * G * NV * VEC + (i * G + lane) * VEC + e] = which ? db[i][e] : dw[i][e];
            __syncthreads();
            for (int c = threadIdx.x; c < cols; c += BLOCK) {
                float s = 0.f;
                for (int r = 0; r < RPB; ++r) s += acc[r * G * NV * VEC + c];
                line[which * cols + c] = s;
            }
        } else {
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const int c = (i * G + lane) * VEC + e;
                    if (c < cols) line[which * cols + c] = which ? db[i][e] : dw[i][e];
                }
        }
    }
}

// the lines of partial sums [lines][2 cols] -> dw, db: 32 columns a block, 32 threads share a column's lines
__global__ __launch_bounds__(1024) void ln_join_kernel(const float* __restrict__ part, void* __restrict__ dw,
                                                       void* __restrict__ db, int lines, int cols, int wdtype) {
    __shared__ float sm[32][33];
    const int j = threadIdx.x & 31, k = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + j;
    float s = 0.f;
    if (c < 2 * cols)
        for (int l = k; l < lines; l += 32) s += part[(size_t)l * 2 * cols + c];
    sm[k][j] = s;
    __syncthreads();
    if (k == 0 && c < 2 * cols) {
        for (int i = 1; i < 32; ++i) s += sm[i][j];
        if (c < cols) {
            if (dw) store_as(dw, c, wdtype, s);
        } else if (db) {
            store_as(db, c - cols, wdtype, s);
        }
    }
}

// Rows longer than 1024 threads hold: the row is read again for the result, the columns' sums are a pass of their own.
template <typename T>
__global__ __launch_bounds__(1024) void ln_fwd_long_kernel(const T* __restrict__ x, const void* __restrict__ w,
                                                           const void* __restrict__ b, T* __restrict__ y,
                                                           float* __restrict__ mean, float* __restrict__ rstd,
                                                           long long rows, int cols, int wdtype, float eps) {
    __shared__ Stat sm[16];
    for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
        const T* xr = x + (size_t)row * cols;
        Stat st{0.f, 0.f, 0.f};
        for (int c0 = 0; c0 < cols; c0 += 8192) {                // eight values a thread, then one combination
            float v[8];
            float s = 0.f, n = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int c = c0 + e * 1024 + threadIdx.x;
                if (c < cols) {
                    v[e] = (float)xr[c];
                    s += v[e];
                    n += 1.f;
                }
            }
            Stat t{n, n > 0.f ? s / n : 0.f, 0.f};
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (c0 + e * 1024 + (int)threadIdx.x < cols) t.m2 += (v[e] - t.mean) * (v[e] - t.mean);
            st = combine(st, t);
        }
        st = group_stat<1024>(st, sm);
        const float inv = 1.f / sqrtf(st.m2 / (float)cols + eps);
        if (threadIdx.x == 0 && mean) {
            mean[row] = st.mean;
            rstd[row] = inv;
        }
        for (int c = threadIdx.x; c < cols; c += 1024)
            y[(size_t)row * cols + c] = (T)(((float)xr[c] - st.mean) * inv * (w ? load_as(w, c, wdtype) : 1.f) +
                                            (b ? load_as(b, c, wdtype) : 0.f));
    }
}

template <typename T>
__global__ __launch_bounds__(1024) void ln_bwd_long_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                                                           const void* __restrict__ w, const float* __restrict__ mean,
                                                           const float* __restrict__ rstd, T* __restrict__ dx,
                                                           long long rows, int cols, int wdtype) {
    __shared__ float sm[32];
    for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
        const size_t at = (size_t)row * cols;
        const float mu = mean[row], inv = rstd[row];
        float s1 = 0.f, s2 = 0.f;
        for (int c = threadIdx.x; c < cols; c += 1024) {
            const float t = (float)dy[at + c] * (w ? load_as(w, c, wdtype) : 1.f);
            s1 += t;
            s2 += t * (((float)x[at + c] - mu) * inv);
        }
        group_sum2<1024>(s1, s2, sm);
        s1 /= (float)cols;
        s2 /= (float)cols;
        for (int c = threadIdx.x; c < cols; c += 1024) {
            const float t = (float)dy[at + c] * (w ? load_as(w, c, wdtype) : 1.f);
            dx[at + c] = (T)(inv * (t - s1 - ((float)x[at + c] - mu) * inv * s2));
        }
    }
}

template <typename T>
__global__ __launch_bounds__(1024) void ln_cols_long_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                                                            const float* __restrict__ mean,
                                                            const float* __restrict__ rstd, float* __restrict__ part,
                                                            long long rows, int cols) {
    __shared__ float sm[16][2][64];
    const int j = threadIdx.x & 63, k = threadIdx.x >> 6;
    const int c = blockIdx.x * 64 + j;
    float s1 = 0.f, s2 = 0.f;
    if (c < cols)
        for (long long row = (long long)blockIdx.y * 16 + k; row < rows; row += (long long)gridDim.y * 16) {
            const float g = (float)dy[(size_t)row * cols + c];
            s1 += g * (((float)x[(size_t)row * cols + c] - mean[row]) * rstd[row]);
            s2 += g;
        }
    sm[k][0][j] = s1;
    sm[k][1][j] = s2;
    __syncthreads();
    if (k < 2 && c < cols) {
        float s = 0.f;
        for (int i = 0; i < 16; ++i) s += sm[i][k][j];
        part[(size_t)blockIdx.y * 2 * cols + k * cols + c] = s;
    }
}

struct Plan {
    int g, nv, vec;                 // g 0: a row is too long for the registers of 1024 threads
};
// Threads per row and packs per thread.  16-byte packs where every row starts at a multiple of 16 bytes; single elements
// otherwise (their columns must be the same for all rows: a thread keeps its columns' gradient sums).
Plan plan(int cols, int dtype, bool aligned) {
    const int vec = 16 / elem_bytes(dtype);
    if (aligned && cols % vec == 0) {
        for (int g : {8, 64, 256, 1024})
            for (int nv : {1, 2})
                if (cols <= g * nv * vec) return Plan{g, nv, vec};
    } else {
        for (int g : {8, 64, 256, 1024})
            for (int nv : {2, 8})
                if (cols <= g * nv) return Plan{g, nv, 1};
        if (cols <= 16384) return Plan{1024, 16, 1};
    }
    return Plan{0, 0, 0};
}
int lines_of(long long rows, const Plan& p) {
    if (!p.g) return (int)(rows < 16 * 64 ? (rows + 15) / 16 : 64);
    const int rpb = p.g < 256 ? 256 / p.g : 1, cap = p.g == 1024 ? 256 : 512;
    const long long blocks = (rows + rpb - 1) / rpb;
    return (int)(blocks < cap ? blocks : cap);
}

bool aligned16(const void* a, const void* b, const void* c) {
    return (((uintptr_t)a | (uintptr_t)b | (uintptr_t)c) & 15) == 0;
}

template <typename F>
int with_type(int dtype, F f) {
    if (dtype == STEP_F32) return f(float());
    if (dtype == STEP_BF16) return f(bf16());
    return f(f16());
}

// calls f(integral constants VEC, NV, G) for a plan of element type T
template <int V>
using Int = std::integral_constant<int, V>;
template <typename T, typename F>
void with_plan(const Plan& p, F f) {
    constexpr int VEC = 16 / (int)sizeof(T);
    auto groups = [&](auto vec, auto nv) {
        if (p.g == 8) f(vec, nv, Int<8>());
        else if (p.g == 64) f(vec, nv, Int<64>());
        else if (p.g == 256) f(vec, nv, Int<256>());
        else f(vec, nv, Int<1024>());
    };
    if (p.vec > 1) {
        if (p.nv == 1) groups(Int<VEC>(), Int<1>());
        else groups(Int<VEC>(), Int<2>());
    } else if (p.nv == 2) groups(Int<1>(), Int<2>());
    else if (p.nv == 8) groups(Int<1>(), Int<8>());
    else f(Int<1>(), Int<16>(), Int<1024>());
}

}  // namespace

extern "C" size_t step_layernorm_bwd_ws_bytes(long long rows, int cols) {
    if (rows <= 0 || cols <= 0) return 0;
    // the same for every type and alignment: 512 lines at most
    const long long lines = rows < 512 ? rows : 512;
    return (size_t)lines * 2 * cols * sizeof(float);
}

extern "C" int step_layernorm_fwd(const void* x, const void* w, const void* b, void* y, float* mean, float* rstd,
                                  long long rows, int cols, int dtype, int wdtype, float eps, void* stream) {
    STEP_REQUIRE(x && y, "step_layernorm_fwd: null pointer");
    STEP_REQUIRE(rows >= 1 && cols >= 1, "step_layernorm_fwd: bad shape rows=%lld cols=%d", rows, cols);
    STEP_REQUIRE(elem_bytes(dtype) && elem_bytes(wdtype), "step_layernorm_fwd: unknown type %d / %d", dtype, wdtype);
    STEP_REQUIRE((mean == nullptr) == (rstd == nullptr), "step_layernorm_fwd: mean and rstd come together");
    hipStream_t st = (hipStream_t)stream;
    const Plan p = plan(cols, dtype, aligned16(x, y, nullptr));
    with_type(dtype, [&](auto t) {
        using T = decltype(t);
        if (!p.g) {
            const long long blocks = rows < 1024 ? rows : 1024;
            hipLaunchKernelGGL(ln_fwd_long_kernel<T>, dim3((unsigned)blocks), dim3(1024), 0, st, (const T*)x, w, b, (T*)y, mean,
                               rstd, rows, cols, wdtype, eps);
            return 0;
        }
        with_plan<T>(p, [&](auto vec, auto nv, auto g) {
            constexpr int G = decltype(g)::value, BLOCK = G < 256 ? 256 : G, RPB = BLOCK / G;
            const long long need = (rows + RPB - 1) / RPB, cap = 4096;
            hipLaunchKernelGGL((ln_fwd_kernel<T, decltype(vec)::value, decltype(nv)::value, G>),
                               dim3((unsigned)(need < cap ? need : cap)), dim3(BLOCK), 0, st, (const T*)x, w, b, (T*)y, mean,
                               rstd, rows, cols, wdtype, eps);
        });
        return 0;
    });
    return step::check_launch("step_layernorm_fwd");
}

extern "C" int step_layernorm_bwd(const void* dy, const void* x, const void* w, const float* mean, const float* rstd,
                                  void* dx, void* dw, void* db, long long rows, int cols, int dtype, int wdtype, void* ws,
                                  size_t ws_bytes, void* stream) {
    STEP_REQUIRE(dy && x && mean && rstd, "step_layernorm_bwd: null pointer");
    STEP_REQUIRE(rows >= 1 && cols >= 1, "step_layernorm_bwd: bad shape rows=%lld cols=%d", rows, cols);
    STEP_REQUIRE(elem_bytes(dtype) && elem_bytes(wdtype), "step_layernorm_bwd: unknown type %d / %d", dtype, wdtype);
    const bool sums = dw || db;
    STEP_REQUIRE(!sums || ws, "step_layernorm_bwd: null workspace");
    if (sums && ws_bytes < step_layernorm_bwd_ws_bytes(rows, cols)) {
        step::set_error("step_layernorm_bwd: workspace %zu < %zu bytes", ws_bytes, step_layernorm_bwd_ws_bytes(rows, cols));
        return STEP_ERR_WORKSPACE;
    }
    if (!dx && !sums) return STEP_OK;
    hipStream_t st = (hipStream_t)stream;
    const Plan p = plan(cols, dtype, aligned16(dy, x, dx));
    const int lines = lines_of(rows, p);
    float* part = sums ? (float*)ws : nullptr;
    with_type(dtype, [&](auto t) {
        using T = decltype(t);
        if (!p.g) {
            const long long blocks = rows < 1024 ? rows : 1024;
            if (dx)
                hipLaunchKernelGGL(ln_bwd_long_kernel<T>, dim3((unsigned)blocks), dim3(1024), 0, st, (const T*)dy, (const T*)x,
                                   w, mean, rstd, (T*)dx, rows, cols, wdtype);
            if (sums)
                hipLaunchKernelGGL(ln_cols_long_kernel<T>, dim3(step::ceil_div(cols, 64), lines), dim3(1024), 0, st,
                                   (const T*)dy, (const T*)x, mean, rstd, part, rows, cols);
            return 0;
        }
        with_plan<T>(p, [&](auto vec, auto nv, auto g) {
            constexpr int G = decltype(g)::value, BLOCK = G < 256 ? 256 : G;
            hipLaunchKernelGGL((ln_bwd_kernel<T, decltype(vec)::value, decltype(nv)::value, G>), dim3(lines), dim3(BLOCK), 0,
                               st, (const T*)dy, (const T*)x, w, mean, rstd, (T*)dx, part, rows, cols, wdtype);
        });
        return 0;
    });
    if (sums)
        hipLaunchKernelGGL(ln_join_kernel, dim3((2 * (unsigned)cols + 31) / 32), dim3(1024), 0, st, part, dw, db, lines, cols, wdtype);
    return step::check_launch("step_layernorm_bwd");
}
