// Layer norm over the rows of a (rows, cols) matrix, forward and backward, fp32 / bf16 / fp16 tensors.
//
//   mu = mean x,  var = mean (x - mu)^2,  r = 1 / sqrt(var + eps),  xhat = (x - mu) r,  y = xhat w + b
//   t = dy w:  dx = r (t - mean t - xhat mean(t xhat)),  dw = SUM_rows dy xhat,  db = SUM_rows dy
//
// Memory-bound both ways: forward 2 and backward 3 elements moved per element (16384 x 4096 bf16: 47 us, 5.7 TB/s, and 80 us,
// 5.0 TB/s; a copy of that size 4.9 to 5.2).  A row stays in the registers of the G
// threads that share it between the statistics and the result, so each tensor is moved once.  G is 8, 64, 256 or 1024, the
// smallest whose threads hold the row (plan() below): up to 4096 16-bit columns a wave has a row to itself and needs no
// barrier; sums over a wave are data-parallel-primitive adds (no LDS).  Two sums in the forward, the mean's
// and that of the squared deviations from it, the second with the rest of the mean: nothing is lost to a mean far from zero.
// dw and db: a thread keeps its columns' sums in fp32 registers over all its rows; a block adds its waves' in order and
// writes one line of partial sums, and a second launch adds the lines in a fixed order - the same bits every time, no
// atomics.
#include "rows.h"

namespace {
using namespace step;

// sums of a and b over the 8 or 64 threads that share a row, the same bits in all of them
template <int G>
__device__ __forceinline__ void wave_sum2(float& a, float& b) {
    a += dpp<0xb1>(a);             // quad_perm 1 0 3 2
    b += dpp<0xb1>(b);
    a += dpp<0x4e>(a);             // quad_perm 2 3 0 1
    b += dpp<0x4e>(b);
    a += dpp<0x141>(a);            // row_half_mirror
    b += dpp<0x141>(b);
    if constexpr (G >= 64) {
        a += dpp<0x140>(a);        // row_mirror: sums of 16
        b += dpp<0x140>(b);
        a = rows16(a, [](float x, float y) { return x + y; });
        b = rows16(b, [](float x, float y) { return x + y; });
    }
}
// the same over G threads that may be several waves (then the whole block comes here): `sm` the group's 2 G / 64 floats, which the
// next call does not use
template <int G>
__device__ __forceinline__ void group_sum2(float& a, float& b, float* sm) {
    wave_sum2<G>(a, b);
    if constexpr (G > 64) {
        const int wave = (threadIdx.x % G) >> 6;
        if ((threadIdx.x & 63) == 0) {
            sm[2 * wave] = a;
            sm[2 * wave + 1] = b;
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

// a block: 256 threads, or one row's 1024
template <typename T, typename W, int VEC, int NV, int G>
__global__ __launch_bounds__(G > 256 ? G : 256) void ln_fwd_kernel(const T* __restrict__ x, const W* __restrict__ w,
                                                                   const W* __restrict__ b, T* __restrict__ y,
                                                                   float* __restrict__ mean, float* __restrict__ rstd,
                                                                   long long rows, int cols, float eps) {
    constexpr int BLOCK = G > 256 ? G : 256, RPB = BLOCK / G;
    constexpr int SUMS = G > 64 ? 2 * BLOCK / 64 : 1;
    __shared__ float sm[2 * SUMS];
    float* const mine = sm + (G > 64 ? threadIdx.x / G * (2 * G / 64) : 0);
    const int lane = threadIdx.x % G;
    const float inv_c = 1.f / (float)cols;
    Pack<W, VEC> wv[NV], bv[NV];
    const Columns<VEC, NV, G> own{cols, lane};
    if (w) own.load(wv, w);
    if (b) own.load(bv, b);
    for (long long r0 = (long long)blockIdx.x * RPB; r0 < rows; r0 += (long long)gridDim.x * RPB) {
        const long long row = r0 + threadIdx.x / G;
        const bool live = row < rows;
        Pack<T, VEC> v[NV];
        own.load(v, x + (size_t)(live ? row : rows - 1) * cols);
        own.fill(v, (T)0.f);
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < VEC; e += 2) {               // two chains
                s1 += (float)v[i].v[e];
                if (e + 1 < VEC) s2 += (float)v[i].v[e + 1];
            }
        s1 += s2;
        s2 = 0.f;
        group_sum2<G>(s1, s2, mine);
        float mu = s1 * inv_c;
        s1 = s2 = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float d = own.mine(i, e) ? (float)v[i].v[e] - mu : 0.f;
                s1 += d;
                s2 += d * d;
            }
        group_sum2<G>(s1, s2, mine + SUMS);
        s1 *= inv_c;                                         // the rest of the mean
        const float inv = 1.f / sqrtf(fmaxf(s2 * inv_c - s1 * s1, 0.f) + eps);
        mu += s1;
        if (!live) continue;
        if (lane == 0 && mean) {
            mean[row] = mu;
            rstd[row] = inv;
        }
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                float o = ((float)v[i].v[e] - mu) * inv;
                if (w) o *= (float)wv[i].v[e];
                if (b) o += (float)bv[i].v[e];
                v[i].v[e] = (T)o;                            // the result's only rounding
            }
        own.store(y + (size_t)row * cols, v);
    }
}

// a block: 512 threads, or one row's 1024
template <typename T, typename W, int VEC, int NV, int G>
__global__ __launch_bounds__(G > 512 ? G : 512) void ln_bwd_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                                                                   const W* __restrict__ w, const float* __restrict__ mean,
                                                                   const float* __restrict__ rstd, T* __restrict__ dx,
                                                                   float* __restrict__ part, long long rows, int cols) {
    constexpr int BLOCK = G > 512 ? G : 512, RPB = BLOCK / G, SUMS = G > 64 ? 2 * BLOCK / 64 : 1;
    __shared__ float sm[2 * SUMS];
    __shared__ float acc[RPB > 1 ? G * NV * VEC : 1];
    const int lane = threadIdx.x % G, group = threadIdx.x / G;
    Pack<W, VEC> wv[NV];
    const Columns<VEC, NV, G> own{cols, lane};
    if (w) own.load(wv, w);
    float dw[NV][VEC], db[NV][VEC];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) dw[i][e] = db[i][e] = 0.f;
    const float inv_c = 1.f / (float)cols;
    int turn = 0;
    for (long long r0 = (long long)blockIdx.x * RPB; r0 < rows; r0 += (long long)gridDim.x * RPB) {
        const long long row = r0 + group;
        const bool live = row < rows;
        const size_t at = (size_t)(live ? row : rows - 1) * cols;
        const float mu = mean[live ? row : rows - 1], inv = rstd[live ? row : rows - 1];
        Pack<T, VEC> g[NV], v[NV];
        own.load(g, dy + at);
        own.load(v, x + at);
        own.fill(g, (T)0.f);
        if (!live)
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int e = 0; e < VEC; ++e) g[i].v[e] = (T)0.f;
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {                  // (dy is 0 where the column is not its own)
                const float d = (float)g[i].v[e], xh = ((float)v[i].v[e] - mu) * inv, t = w ? d * (float)wv[i].v[e] : d;
                dw[i][e] += d * xh;
                db[i][e] += d;
                s1 += t;
                s2 += t * xh;
            }
        if (dx) {
            group_sum2<G>(s1, s2, sm + (G > 64 ? turn * SUMS + group * (2 * G / 64) : 0));
            turn ^= 1;
            s1 *= inv_c;
            s2 *= inv_c;
            if (live) {
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        const float d = (float)g[i].v[e], xh = ((float)v[i].v[e] - mu) * inv, t = w ? d * (float)wv[i].v[e] : d;
                        g[i].v[e] = (T)(inv * (t - s1 - xh * s2));
                    }
                own.store(dx + at, g);
            }
        }
    }
    if (!part) return;
    float* line = part + (size_t)blockIdx.x * 2 * cols;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        if constexpr (RPB > 1) {
            if constexpr (G < 64)                            // a wave's rows first
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int e = 0; e < VEC; ++e)
#pragma unroll
                        for (int o = G; o < 64; o <<= 1) {
                            if (which) db[i][e] += __shfl_xor(db[i][e], o, 64);
                            else dw[i][e] += __shfl_xor(dw[i][e], o, 64);
                        }
            constexpr int GROUP = G < 64 ? 64 : G;
            for (int k = 0; k < BLOCK / GROUP; ++k) {        // then the block's, in order
                if ((int)threadIdx.x / GROUP == k && threadIdx.x % GROUP < G)
#pragma unroll
                    for (int i = 0; i < NV; ++i)
#pragma unroll
                        for (int e = 0; e < VEC; ++e)
                            if (own.mine(i, e)) {
                                const int c = own.at(i) + e;
                                const float t = which ? db[i][e] : dw[i][e];
                                acc[c] = k ? acc[c] + t : t;
                            }
                __syncthreads();
            }
            for (int c = threadIdx.x; c < cols; c += BLOCK) line[which * cols + c] = acc[c];
            __syncthreads();
        } else {
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int e = 0; e < VEC; ++e)
                    if (own.mine(i, e)) line[which * cols + own.at(i) + e] = which ? db[i][e] : dw[i][e];
        }
    }
}

// the lines of partial sums [lines][2 cols] -> dw, db: 32 columns a block, 32 threads share a column's lines
__global__ __launch_bounds__(1024) void ln_join_kernel(const float* __restrict__ part, void* __restrict__ dw,
                                                       void* __restrict__ db, int lines, int cols, int wdtype) {
    __shared__ float sm[32][33];
    const int j = threadIdx.x & 31, k = threadIdx.x >> 5;
    for (int c0 = blockIdx.x * 32; c0 < 2 * cols; c0 += gridDim.x * 32) {
        const int c = c0 + j;
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
        __syncthreads();
    }
}

// Rows longer than 1024 threads hold: the row is read again for each sum and the result, the columns' sums are a pass of their
// own.
template <typename T>
__global__ __launch_bounds__(1024) void ln_fwd_long_kernel(const T* __restrict__ x, const void* __restrict__ w,
                                                           const void* __restrict__ b, T* __restrict__ y,
                                                           float* __restrict__ mean, float* __restrict__ rstd,
                                                           long long rows, int cols, int wdtype, float eps) {
    __shared__ float sm[64];
    for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
        const T* xr = x + (size_t)row * cols;
        float s1 = 0.f, s2 = 0.f;
        for (int c = threadIdx.x; c < cols; c += 1024) s1 += (float)xr[c];
        group_sum2<1024>(s1, s2, sm);
        float mu = s1 / (float)cols;
        s1 = s2 = 0.f;
        for (int c = threadIdx.x; c < cols; c += 1024) {
            const float d = (float)xr[c] - mu;
            s1 += d;
            s2 += d * d;
        }
        group_sum2<1024>(s1, s2, sm + 32);
        s1 /= (float)cols;
        const float inv = 1.f / sqrtf(fmaxf(s2 / (float)cols - s1 * s1, 0.f) + eps);
        mu += s1;
        if (threadIdx.x == 0 && mean) {
            mean[row] = mu;
            rstd[row] = inv;
        }
        for (int c = threadIdx.x; c < cols; c += 1024)
            y[(size_t)row * cols + c] = (T)(((float)xr[c] - mu) * inv * (w ? load_as(w, c, wdtype) : 1.f) +
                                            (b ? load_as(b, c, wdtype) : 0.f));
        __syncthreads();
    }
}

template <typename T>
__global__ __launch_bounds__(1024) void ln_bwd_long_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                                                           const void* __restrict__ w, const float* __restrict__ mean,
                                                           const float* __restrict__ rstd, T* __restrict__ dx,
                                                           long long rows, int cols, int wdtype) {
    __shared__ float sm[64];
    int turn = 0;
    for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
        const size_t at = (size_t)row * cols;
        const float mu = mean[row], inv = rstd[row];
        float s1 = 0.f, s2 = 0.f;
        for (int c = threadIdx.x; c < cols; c += 1024) {
            const float t = (float)dy[at + c] * (w ? load_as(w, c, wdtype) : 1.f);
            s1 += t;
            s2 += t * (((float)x[at + c] - mu) * inv);
        }
        group_sum2<1024>(s1, s2, sm + 32 * turn);
        turn ^= 1;
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
    for (int c0 = blockIdx.x * 64; c0 < cols; c0 += gridDim.x * 64) {
        const int c = c0 + j;
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
        __syncthreads();
    }
}

constexpr int MAX_LINES = 512;
// blocks over the columns, which go on to further ones: a launch has fewer than 2^32 threads, and rows up to 2^28 columns
constexpr int MAX_COLUMN_BLOCKS = 1 << 16;
int column_blocks(long long cols, int per) {
    const long long blocks = (cols + per - 1) / per;
    return (int)(blocks < MAX_COLUMN_BLOCKS ? blocks : MAX_COLUMN_BLOCKS);
}

struct Plan {
    int g, nv, vec;                 // threads per row, packs per thread, elements of a pack; g 0: too long for the registers of 1024 threads
};
// The fewest threads whose registers hold the row.  The forward keeps a row's elements as they are, and the weights: 8 packs a
// thread (16384 x 4096 bf16 on a wave a row: 47 us, 5.7 TB/s; on a block of 256 threads 48).  The backward also keeps two sums
// per column, 32 elements a thread are the most without spills (8192 x 8192 bf16: 84 us at 256 threads x 32, 100 at 1024 x 8).
// Rows shorter than a pack are read by elements.
constexpr int NV_FWD = 8, NV_1024 = 4;              // (1024 threads have half the registers)
constexpr int nv_bwd(int vec) { return 32 / vec; }
Plan plan(int cols, int dtype, bool fwd) {
    const int vec = 16 / elem_bytes(dtype);
    if (cols < vec) return Plan{8, 1, 1};
    if (cols <= 8 * vec) return Plan{8, 1, vec};
    const int most = fwd ? NV_FWD : nv_bwd(vec);
    for (int g : {64, 256})
        if (cols <= (long long)g * most * vec) return Plan{g, step::ceil_div(cols, g * vec), vec};
    if (fwd && cols <= 1024 * NV_1024 * vec) return Plan{1024, step::ceil_div(cols, 1024 * vec), vec};
    if (!fwd && cols <= 512 * most * vec) return Plan{512, step::ceil_div(cols, 512 * vec), vec};
    return Plan{0, 0, 0};
}
int lines_of(long long rows, const Plan& p) {
    if (!p.g) return (int)(rows < 16 * 64 ? (rows + 15) / 16 : 64);
    // a block a CU where a thread has many elements (the rows in flight are enough and the lines of sums are fewer), two
    // otherwise; as many rows a group as leave 128 blocks, up to four, or adding the lines takes longer than the rows
    const int rpb = p.g < 512 ? 512 / p.g : 1, cap = p.nv * p.vec > 16 ? MAX_LINES / 2 : MAX_LINES;
    const long long one = (rows + rpb - 1) / rpb, blocks = one / 4 > 128 ? one / 4 : one < 128 ? one : 128;
    return (int)(blocks < cap ? blocks : cap);
}

// calls f(integral constants VEC, NV, G) for a plan
template <int V>
using Int = std::integral_constant<int, V>;
template <int VEC, int G, int FROM, int MOST, typename F>
void with_nv(int nv, F f) {
    if (nv == FROM) f(Int<VEC>(), Int<FROM>(), Int<G>());
    else if constexpr (FROM < MOST) with_nv<VEC, G, FROM + 1, MOST>(nv, f);
}
template <typename T, bool FWD, typename F>
void with_plan(const Plan& p, F f) {
    constexpr int VEC = 16 / (int)sizeof(T), MOST = FWD ? NV_FWD : nv_bwd(VEC);
    if (p.vec == 1) with_nv<1, 8, 1, 1>(p.nv, f);
    else if (p.g == 8) with_nv<VEC, 8, 1, 1>(p.nv, f);
    else if (p.g == 64) with_nv<VEC, 64, 1, MOST>(p.nv, f);
    else if (p.g == 256) with_nv<VEC, 256, MOST / 4 + 1, MOST>(p.nv, f);      // fewer fit in 64 threads
    else if constexpr (FWD) with_nv<VEC, 1024, MOST / 4 + 1, NV_1024>(p.nv, f);
    else with_nv<VEC, 512, MOST / 2 + 1, MOST>(p.nv, f);
}
// calls f(T(), W()) for the rows' and the weights' types: the same, or fp32 weights
template <typename F>
int with_types(int dtype, int wdtype, F f) {
    if (dtype == STEP_F32) return f(float(), float());
    if (dtype == STEP_BF16) return wdtype == STEP_F32 ? f(bf16(), float()) : f(bf16(), bf16());
    return wdtype == STEP_F32 ? f(f16(), float()) : f(f16(), f16());
}

}  // namespace

extern "C" size_t step_layernorm_bwd_ws_bytes(long long rows, int cols) {
    if (rows <= 0 || cols <= 0) return 0;
    // the same for every type and alignment
    const long long lines = rows < MAX_LINES ? rows : MAX_LINES;
    return (size_t)lines * 2 * cols * sizeof(float);
}

extern "C" int step_layernorm_fwd(const void* x, const void* w, const void* b, void* y, float* mean, float* rstd,
                                  long long rows, int cols, int dtype, int wdtype, float eps, void* stream) {
    STEP_REQUIRE(x && y, "step_layernorm_fwd: null pointer");
    STEP_REQUIRE(rows >= 1 && cols >= 1 && cols <= 1 << 28, "step_layernorm_fwd: bad shape rows=%lld cols=%d", rows, cols);
    STEP_REQUIRE(elem_bytes(dtype) && elem_bytes(wdtype), "step_layernorm_fwd: unknown type %d / %d", dtype, wdtype);
    STEP_REQUIRE(wdtype == STEP_F32 || wdtype == dtype, "step_layernorm_fwd: weights of type %d beside rows of type %d", wdtype, dtype);
    STEP_REQUIRE((mean == nullptr) == (rstd == nullptr), "step_layernorm_fwd: mean and rstd come together");
    hipStream_t st = (hipStream_t)stream;
    const Plan p = plan(cols, dtype, true);
    with_types(dtype, wdtype, [&](auto t, auto u) {
        using T = decltype(t);
        using W = decltype(u);
        if (!p.g) {
            const long long blocks = rows < 1024 ? rows : 1024;
            hipLaunchKernelGGL(ln_fwd_long_kernel<T>, dim3((unsigned)blocks), dim3(1024), 0, st, (const T*)x, w, b, (T*)y, mean,
                               rstd, rows, cols, wdtype, eps);
            return 0;
        }
        auto go = [&](auto vec, auto nv, auto g) {
            constexpr int G = decltype(g)::value, BLOCK = G > 256 ? G : 256, RPB = BLOCK / G;
            // four rows a thread group or more, once every CU has two blocks: the weights are read once for them
            const long long need = (rows + RPB - 1) / RPB, cap = need / 4 < 512 ? 512 : need / 4 < 2048 ? need / 4 : 2048;
            hipLaunchKernelGGL((ln_fwd_kernel<T, W, decltype(vec)::value, decltype(nv)::value, G>),
                               dim3((unsigned)(need < cap ? need : cap)), dim3(BLOCK), 0, st, (const T*)x, (const W*)w,
                               (const W*)b, (T*)y, mean, rstd, rows, cols, eps);
        };
        with_plan<T, true>(p, go);
        return 0;
    });
    return step::check_launch("step_layernorm_fwd");
}

extern "C" int step_layernorm_bwd(const void* dy, const void* x, const void* w, const float* mean, const float* rstd,
                                  void* dx, void* dw, void* db, long long rows, int cols, int dtype, int wdtype, void* ws,
                                  size_t ws_bytes, void* stream) {
    STEP_REQUIRE(dy && x && mean && rstd, "step_layernorm_bwd: null pointer");
    STEP_REQUIRE(rows >= 1 && cols >= 1 && cols <= 1 << 28, "step_layernorm_bwd: bad shape rows=%lld cols=%d", rows, cols);
    STEP_REQUIRE(elem_bytes(dtype) && elem_bytes(wdtype), "step_layernorm_bwd: unknown type %d / %d", dtype, wdtype);
    STEP_REQUIRE(wdtype == STEP_F32 || wdtype == dtype, "step_layernorm_bwd: weights of type %d beside rows of type %d", wdtype, dtype);
    const bool sums = dw || db;
    STEP_REQUIRE(!sums || ws, "step_layernorm_bwd: null workspace");
    if (sums && ws_bytes < step_layernorm_bwd_ws_bytes(rows, cols)) {
        step::set_error("step_layernorm_bwd: workspace %zu < %zu bytes", ws_bytes, step_layernorm_bwd_ws_bytes(rows, cols));
        return STEP_ERR_WORKSPACE;
    }
    if (!dx && !sums) return STEP_OK;
    hipStream_t st = (hipStream_t)stream;
    const Plan p = plan(cols, dtype, false);
    const int lines = lines_of(rows, p);
    float* part = sums ? (float*)ws : nullptr;
    with_types(dtype, wdtype, [&](auto t, auto u) {
        using T = decltype(t);
        using W = decltype(u);
        if (!p.g) {
            const long long blocks = rows < 1024 ? rows : 1024;
            if (dx)
                hipLaunchKernelGGL(ln_bwd_long_kernel<T>, dim3((unsigned)blocks), dim3(1024), 0, st, (const T*)dy, (const T*)x,
                                   w, mean, rstd, (T*)dx, rows, cols, wdtype);
            if (sums)
                hipLaunchKernelGGL(ln_cols_long_kernel<T>, dim3(column_blocks(cols, 64), lines), dim3(1024), 0, st,
                                   (const T*)dy, (const T*)x, mean, rstd, part, rows, cols);
            return 0;
        }
        auto go = [&](auto vec, auto nv, auto g) {
            constexpr int G = decltype(g)::value, BLOCK = G > 512 ? G : 512;
            hipLaunchKernelGGL((ln_bwd_kernel<T, W, decltype(vec)::value, decltype(nv)::value, G>), dim3(lines), dim3(BLOCK), 0,
                               st, (const T*)dy, (const T*)x, (const W*)w, mean, rstd, (T*)dx, part, rows, cols);
        };
        with_plan<T, false>(p, go);
        return 0;
    });
    if (sums)
        hipLaunchKernelGGL(ln_join_kernel, dim3(column_blocks(2LL * cols, 32)), dim3(1024), 0, st, part, dw, db, lines, cols, wdtype);
    return step::check_launch("step_layernorm_bwd");
}
