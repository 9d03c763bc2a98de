// Orthogonalised updates by Newton-Schulz products (Muon), for lists of matrices of any shape.
//
//   X_0 = G / (|G|_F + eps),   A = X X^T,  B = b A + c A^2,  X <- a X + B X   (a, b, c) = (3.4445, -4.7750, 2.0315)
//
// on the side with the fewer rows: r = min(m, n), l = max(m, n), X is r x l (G or its transpose).  With q(t) = a + b t + c t^2
// every step is X <- q(A) X.  Two forms:
//
// r <= 64, all in fp64: X_k = P_k X_0 with P_k and A_k polynomials of A_0, so the long side is read twice only - once for
//   G G^T and once for P G: A <- q(A) A q(A), P <- q(A) P, r x r products on the fp64 matrix cores.  The recursion on A
//   multiplies a small eigenvalue's error by up to a^2 in every step, which fp32 does not bear and fp64 does.
//   The trace of G G^T is the squared norm.  Three launches for a whole list of matrices: bound by the latency of a chain of
//   16 x 16 x 4 fp64 products (64 cycles each) on one CU a matrix.  The matrices of a classifier of widths 32, 64, 64 with 75
//   taps (14 MB with momentum and update): 14 + 47 + 16 us; 7.6 us of the second launch a step at r = 64.
//
// r > 64, every product on the f16 matrix cores: a value v, scaled by a power of two, is hi = f16(v) plus lo = f16(v - hi)
//   (together 22 bits and the sign of lo: the 24 bits of an fp32 value to half a unit or so), a product takes three terms
//   hi hi + hi lo + lo hi with fp32 accumulation.  The dropped lo lo is 2^-24 of a product.  The singular values stay
//   under 1.21 (q's maximum on [0, 1.46]) and so do all elements, so the scales are constants.  Matrices lie packed, 32
//   hi and 32 lo of a row in 128 bytes, X also transposed, so that every product has both its operands along the
//   contraction.  A and q(A) are symmetric: only the tiles on and over the diagonal are computed.  Bound by the matrix cores where
//   the products fill the card (4096 x 4096: X's update 355 us, 1.16 PFLOP/s of f16 products, the cores busy in 65 % of the
//   cycles at the 1.8 GHz that their power leaves; a plain f16 product of 8192^3 reaches 1.02), by the chain of r x r products
//   otherwise (256 x 19200: 11 of them, 6 us each, of 187).  An element's error is 2^-23 of it, or 2^-39 where it is under 2^-17
//   (f16's subnormals hold its lo): of the matrix's size, since X is lifted by a power of two as long as |G| is far below eps
//   and X with it (lift() below).
#include <vector>
#include "rows.h"

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef double f64x4 __attribute__((ext_vector_type(4)));

namespace {
using namespace step;

constexpr double QA = 3.4445, QB = -4.7750, QC = 2.0315;

// how a matrix comes in and how its result leaves
struct Io {
    const void* g;
    void* out;                   // orthogonalised matrix (plain form), or
    float* momentum;             // the optimizer's form: momentum <- mu momentum + g,  u = g + mu momentum (nesterov),
    float* param;                //   param <- param (1 - lr decay) - lr scale o
    float mu, keep, step;        // keep = 1 - lr decay, step = lr scale
    int nesterov;
};
template <typename T>
__device__ __forceinline__ float read_u(const Io& io, size_t at, bool update) {
    const float g = (float)((const T*)io.g)[at];
    if (!io.momentum) return g;
    float m = io.momentum[at];
    if (update) {
        m = io.mu * m + g;
        io.momentum[at] = m;
    }
    return io.nesterov ? g + io.mu * m : m;
}
template <typename T>
__device__ __forceinline__ void write_o(const Io& io, size_t at, float o) {
    if (io.param) io.param[at] = io.param[at] * io.keep - io.step * o;
    else ((T*)io.out)[at] = (T)o;                            // the result's only rounding to fewer bits
}

// ---------------------------------------------------------------------------------------------- r <= 64
constexpr int S_ITEMS = 24;                       // matrices' descriptions that fit a launch's arguments
constexpr int S_P = 66;                           // row pitch of a 64 x 64 fp64 matrix in LDS: 16 rows begin 4 banks apart

struct SmallItem {
    Io io;
    int m, n, chunks, width;                      // chunks of `width` columns of the long side
    size_t slab, p;                               // offsets in the workspace, in doubles
};
struct SmallArgs {
    int first[S_ITEMS];                           // first matrix of each item; behind the items more than all
    SmallItem item[S_ITEMS];
    int steps, max_chunks, max_parts;             // (parts: 64 columns each, of ns_apply_kernel)
    float eps;
    double* ws;
};
// item and element offset of matrix z
__device__ __forceinline__ const SmallItem& find(const SmallArgs& p, int z, int& local) {
    int i = 0, first = 0;
#pragma unroll
    for (int k = 1; k < S_ITEMS; ++k)             // (all read at once, and not one after the other)
        if (p.first[k] <= z) {
            i = k;
            first = p.first[k];
        }
    local = z - first;
    return p.item[i];
}
__device__ __host__ __forceinline__ Io shifted(Io io, size_t by, int bytes) {
    io.g = (const char*)io.g + by * bytes;
    if (io.out) io.out = (char*)io.out + by * bytes;
    if (io.momentum) io.momentum += by;
    if (io.param) io.param += by;
    return io;
}

constexpr int GRAM_WAVES = 12;
// sixteen columns c0 .. c0 + 15 of the short side's rows 16 t + i16: element (t, s) is column c0 + 4 q + s
template <typename T, bool UPDATE>
__device__ __forceinline__ void read_columns(float (&u)[4][4], const Io& io, int m, int n, int r, int c0, int c1, int i16, int q) {
    const bool tall = m > n;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const int row = 16 * t + i16, col = c0 + 4 * q;
        if (!tall && row < r && col + 4 <= c1) {             // four neighbours
            const size_t at = (size_t)row * n + col;
            const Pack<T, 4> g = load_pack<T, 4>((const T*)io.g + at);
            Pack<float, 4> v{{(float)g.v[0], (float)g.v[1], (float)g.v[2], (float)g.v[3]}};
            if (io.momentum) {
                Pack<float, 4> w = load_pack<float, 4>(io.momentum + at);
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    if (UPDATE) w.v[s] = io.mu * w.v[s] + v.v[s];
                    v.v[s] = io.nesterov ? v.v[s] + io.mu * w.v[s] : w.v[s];
                }
                if (UPDATE) store_pack<float, 4>(io.momentum + at, w);
            }
#pragma unroll
            for (int s = 0; s < 4; ++s) u[t][s] = v.v[s];
        } else {
#pragma unroll
            for (int s = 0; s < 4; ++s)
                u[t][s] = row < r && col + s < c1 ? read_u<T>(io, tall ? (size_t)(col + s) * n + row : (size_t)row * n + col + s, UPDATE) : 0.f;
        }
    }
}

// one chunk of columns: its part of G G^T, upper 16 x 16 tiles, [10][256] doubles; 16 columns a wave at a time
template <typename T>
__global__ __launch_bounds__(64 * GRAM_WAVES) void ns_gram_kernel(const SmallArgs p) {
    __shared__ double sm[4][2560];
    const int z = blockIdx.x / p.max_chunks, chunk = blockIdx.x % p.max_chunks;
    int local;
    const SmallItem& it = find(p, z, local);
    if (chunk >= it.chunks) return;
    const int r = min(it.m, it.n), l = max(it.m, it.n);
    const Io io = shifted(it.io, (size_t)local * it.m * it.n, sizeof(T));
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i16 = lane & 15, q = lane >> 4;
    f64x4 acc[10];
#pragma unroll
    for (int t = 0; t < 10; ++t) acc[t] = f64x4{0, 0, 0, 0};
    const int c1 = min(l, (chunk + 1) * it.width);
    for (int c0 = chunk * it.width + 16 * wave; c0 < c1; c0 += 16 * GRAM_WAVES) {
        float u[4][4];                                       // step s takes the columns 4 q + s: the order of a contraction is free
        read_columns<T, true>(u, io, it.m, it.n, r, c0, c1, i16, q);
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            int k = 0;
#pragma unroll
            for (int a = 0; a < 4; ++a)
#pragma unroll
                for (int b = a; b < 4; ++b, ++k)
                    if (16 * b < r)
                        acc[k] = __builtin_amdgcn_mfma_f64_16x16x4f64((double)u[a][s], (double)u[b][s], acc[k], 0, 0, 0);
        }
    }
    // the waves' sums in four columns of three, in order
    for (int w = 0; w < GRAM_WAVES / 4; ++w) {
        if (wave / 4 == w)
#pragma unroll
            for (int t = 0; t < 10; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    double& d = sm[wave & 3][t * 256 + i * 64 + lane];
                    d = w ? d + acc[t][i] : acc[t][i];
                }
        __syncthreads();
    }
    double* slab = p.ws + it.slab + ((size_t)local * it.chunks + chunk) * 2560;
    for (int e = threadIdx.x; e < 2560; e += 64 * GRAM_WAVES) slab[e] = (sm[0][e] + sm[1][e]) + (sm[2][e] + sm[3][e]);
}

// Products X Y of commuting symmetric matrices of 16 NT rows in LDS, by 16 x 16 tiles on or over the diagonal, a wave each.
constexpr int SMALL_THREADS = 1024;
template <int NT>
constexpr int tri_of() {
    return NT * (NT + 1) / 2;
}
template <int NT>
__device__ __forceinline__ void tile_at(int t, int& a, int& b) {   // row a of the triangle has NT - a tiles
    a = 0;
    b = t;
    while (b >= NT) b -= NT - ++a;
}
template <int NT>
__device__ __forceinline__ f64x4 sym_tile(const double* X, const double* Y, int tile) {
    const int lane = threadIdx.x & 63, i16 = lane & 15, q = lane >> 4;
    int a, b;
    tile_at<NT>(tile, a, b);
    const double* x = X + (16 * a + i16) * S_P + q;
    const double* y = Y + (16 * b + i16) * S_P + q;
    f64x4 c{0, 0, 0, 0}, d{0, 0, 0, 0};
#pragma unroll
    for (int s = 0; s < 4 * NT; s += 2) {
        c = __builtin_amdgcn_mfma_f64_16x16x4f64(x[4 * s], y[4 * s], c, 0, 0, 0);
        d = __builtin_amdgcn_mfma_f64_16x16x4f64(x[4 * s + 4], y[4 * s + 4], d, 0, 0, 0);
    }
    return c + d;
}
// a tile and its mirror image: f(i, j, value) stores, one value for both places, bit for bit
template <int NT, typename F>
__device__ __forceinline__ void mirrored(const f64x4& v, int tile, F f) {
    const int lane = threadIdx.x & 63, i16 = lane & 15, q = lane >> 4;
    int a, b;
    tile_at<NT>(tile, a, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = 16 * a + 4 * i + q, col = 16 * b + i16;
        if (a != b || row <= col) {
            f(row, col, v[i]);
            if (row != col) f(col, row, v[i]);
        }
    }
}

// A in LDS -> P with O = P G.  A step is three rounds of products: Q = q(A) from A^2; Q P and Q A, whose tiles (20 at r = 64) are
// five for each SIMD; (Q A) Q.  Results take their operand's place once all waves have read it.
template <int NT>
__device__ __forceinline__ void small_steps(double* A, double* Q, double* P, double inv, int steps) {
    constexpr int T = tri_of<NT>(), WAVES = SMALL_THREADS / 64;
    const int wave = threadIdx.x >> 6;
    auto into = [](double* M) { return [M](int i, int j, double v) { M[i * S_P + j] = v; }; };
    for (int step = 0; step < steps; ++step) {
        if (wave < T)
            mirrored<NT>(sym_tile<NT>(A, A, wave), wave, [&](int i, int j, double v) {
                const double w = QB * A[i * S_P + j] + QC * v + (i == j ? QA : 0.0);
                Q[i * S_P + j] = w;
                if (step == 0) P[i * S_P + j] = w * inv;
            });
        __syncthreads();
        // tiles [0, T) of Q P (not in the first step), [T, 2 T) of Q A (not in the last)
        const int from = step ? 0 : T, to = step + 1 < steps ? 2 * T : T;
        const int u0 = from + wave, u1 = u0 + WAVES;
        f64x4 v0, v1;
        if (u0 < to) v0 = sym_tile<NT>(Q, u0 < T ? P : A, u0 < T ? u0 : u0 - T);
        if (u1 < to) v1 = sym_tile<NT>(Q, u1 < T ? P : A, u1 < T ? u1 : u1 - T);
        __syncthreads();
        if (u0 < to) mirrored<NT>(v0, u0 < T ? u0 : u0 - T, into(u0 < T ? P : A));
        if (u1 < to) mirrored<NT>(v1, u1 < T ? u1 : u1 - T, into(u1 < T ? P : A));
        __syncthreads();
        if (step + 1 < steps) {
            if (wave < T) v0 = sym_tile<NT>(A, Q, wave);
            __syncthreads();
            if (wave < T) mirrored<NT>(v0, wave, into(A));
            __syncthreads();
        }
    }
}

__global__ __launch_bounds__(SMALL_THREADS) void ns_small_kernel(const SmallArgs p) {
    extern __shared__ __attribute__((aligned(16))) double lds[];
    __shared__ double norm_s;
    int local;
    const SmallItem& it = find(p, blockIdx.x, local);
    const int r = min(it.m, it.n), nt = (r + 15) / 16, R = 16 * nt, tid = threadIdx.x;
    double *A = lds, *Q = lds + 64 * S_P, *P = lds + 2 * 64 * S_P;
    const double* slab = p.ws + it.slab + (size_t)local * it.chunks * 2560;
    // join the chunks in order: element e of tile t is row 16 a + 4 (e / 64) + (e % 64) / 16, column 16 b + e % 16
    constexpr int NJ = (2560 + SMALL_THREADS - 1) / SMALL_THREADS;
    double v[NJ] = {};
#pragma unroll 8
    for (int c = 0; c < it.chunks; ++c)
#pragma unroll
        for (int j = 0; j < NJ; ++j) v[j] += slab[(size_t)c * 2560 + min(tid + SMALL_THREADS * j, 2559)];
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
        const int e = tid + SMALL_THREADS * j;
        if (e >= 2560) continue;
        const int t = e >> 8, a = t < 4 ? 0 : t < 7 ? 1 : t < 9 ? 2 : 3, b = t < 4 ? t : t < 7 ? t - 3 : t < 9 ? t - 5 : 3;
        const int row = 16 * a + 4 * ((e & 255) >> 6) + ((e & 63) >> 4), col = 16 * b + (e & 15);
        if (b >= nt || (a == b && row > col)) continue;
        A[row * S_P + col] = v[j];
        A[col * S_P + row] = v[j];
    }
    __syncthreads();
    if (tid < 64) {                                          // the trace is the squared norm
        double tr = tid < R ? A[tid * S_P + tid] : 0.0;
        for (int o = 1; o < 64; o <<= 1) tr += __shfl_xor(tr, o, 64);
        if (tid == 0) norm_s = tr == 0.0 ? 0.0 : 1.0 / (sqrt(tr) + (double)p.eps);      // (a zero matrix stays zero)
    }
    __syncthreads();
    const double inv = norm_s;
    for (int e = tid; e < 64 * R; e += SMALL_THREADS) A[(e >> 6) * S_P + (e & 63)] *= inv * inv;
    __syncthreads();
    if (nt == 1) small_steps<1>(A, Q, P, inv, p.steps);
    else if (nt == 2) small_steps<2>(A, Q, P, inv, p.steps);
    else if (nt == 3) small_steps<3>(A, Q, P, inv, p.steps);
    else small_steps<4>(A, Q, P, inv, p.steps);
    double* out = p.ws + it.p + (size_t)local * 4096;
    for (int e = tid; e < 64 * R; e += SMALL_THREADS)
        if ((e & 63) < R) out[e] = P[(e >> 6) * S_P + (e & 63)];
}

// O = P U: 16 columns of the long side a wave
template <typename T>
__global__ __launch_bounds__(256) void ns_apply_kernel(const SmallArgs p) {
    __shared__ double P[64 * S_P];
    const int z = blockIdx.x / p.max_parts, part = blockIdx.x % p.max_parts;
    int local;
    const SmallItem& it = find(p, z, local);
    const bool tall = it.m > it.n;
    const int r = tall ? it.n : it.m, l = tall ? it.m : it.n, nt = (r + 15) / 16;
    if (part * 64 >= l) return;
    const Io io = shifted(it.io, (size_t)local * it.m * it.n, sizeof(T));
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i16 = lane & 15, q = lane >> 4;
    const double* src = p.ws + it.p + (size_t)local * 4096;
    const int c0 = part * 64 + 16 * wave, col = c0 + i16;
    // the column's elements j = 16 t + 4 q + s for step (t, s), and what the result is added to
    float u[4][4], old[4][4];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int j = 16 * t + 4 * q + s;
            u[t][s] = j < r && col < l ? read_u<T>(io, tall ? (size_t)col * it.n + j : (size_t)j * it.n + col, false) : 0.f;
        }
    // element (a, i) of the result: rows are the short side, or the long one where it is the matrix's rows
    auto place = [&](int a, int i, size_t& at) {
        const int rr = 4 * i + q, srt = 16 * a + (tall ? i16 : rr), lng = c0 + (tall ? rr : i16);
        at = tall ? (size_t)lng * it.n + srt : (size_t)srt * it.n + lng;
        return srt < r && lng < l;
    };
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            size_t at;
            old[a][i] = place(a, i, at) && io.param ? io.param[at] : 0.f;
        }
    double pv[16];                                           // all 64 x 64, of which 16 nt rows and columns are looked at
#pragma unroll
    for (int k = 0; k < 16; ++k) pv[k] = src[threadIdx.x + 256 * k];
#pragma unroll
    for (int k = 0; k < 16; ++k) P[(4 * k + (threadIdx.x >> 6)) * S_P + (threadIdx.x & 63)] = pv[k];
    __syncthreads();
    if (c0 >= l) return;
#pragma unroll
    for (int a = 0; a < 4; ++a) {
        if (a >= nt) break;
        f64x4 acc{0, 0, 0, 0};
#pragma unroll
        for (int t = 0; t < 4; ++t)
            if (t < nt)
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    const double pv = P[(16 * a + i16) * S_P + 16 * t + 4 * q + s];
                    acc = tall ? __builtin_amdgcn_mfma_f64_16x16x4f64((double)u[t][s], pv, acc, 0, 0, 0)
                               : __builtin_amdgcn_mfma_f64_16x16x4f64(pv, (double)u[t][s], acc, 0, 0, 0);
                }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            size_t at;
            if (!place(a, i, at)) continue;
            if (io.param) io.param[at] = old[a][i] * io.keep - io.step * (float)acc[i];
            else ((T*)io.out)[at] = (T)(float)acc[i];        // the result's only rounding to fewer bits
        }
    }
}

// ---------------------------------------------------------------------------------------------- r > 64
constexpr int KS = 32;                            // contraction per stage
constexpr int ROWB = 128;                         // bytes of a row's stage: 32 hi, 32 lo
// scales of X, of A and q(A) A, and of products of one, two and three q(A): elements under 1.21, 1.47, 3.45, 11.9 and 41
constexpr float SX = 16384.f, SA = 16384.f, SQ[3] = {8192.f, 4096.f, 1024.f};
constexpr int CUS = 256;
constexpr int NORM_BLOCKS = 1024;
constexpr int BATCH = 1024;                       // matrices of a stack at a time, at most

struct Big {
    Io io;
    int m, n, r, l, R, L, RA;                     // R, L: r and l rounded up to whole tiles; RA: rows that X and A have
    float eps;
    double* part;                                 // [batch][NORM_BLOCKS] sums of squares, and before them [BATCH] -log2 |X_0| in floats
    char *x, *xt, *xt2;                           // packed matrices, one after the other for the batch
    const char *s1, *s2;                          // R x R (RA rows) operands of a product, and its result
    char* s3;
    float scale;                                  // result's scale over the operands'
    int from : 16, by : 16;                       // the step whose lift a product's operands have, and how many steps further its result is
    float* slab;                                  // shares of split tiles
};

// |X_k| <= q(0)^k |X_0|, and |X_0| = |G| / (|G| + eps) may be anything below 1: X_k is held times 2^lift(k), the largest power with
// which that bound stays at 1 or below (0 once the bound reaches 1/2, as from the start where |G| is over eps), A_k times its square.
__device__ __forceinline__ float* heads(const Big& p) { return (float*)p.part - BATCH; }
__device__ __forceinline__ int lift(float head, int k) {
    constexpr float GROWTH = 1.78429458f;         // log2 QA
    return (int)fmaxf(floorf(head - (float)k * GROWTH), 0.f);
}

// sums of squares in fp64; with the momentum's update in the optimizer's form (4096 x 4096 fp32: 17 us, 4.0 TB/s, once per call)
template <typename T>
__global__ __launch_bounds__(256) void ns_norm_kernel(const Big p) {
    __shared__ double red[4];
    const size_t e = (size_t)p.m * p.n;
    const Io io = shifted(p.io, e * blockIdx.y, sizeof(T));
    double s = 0.0;
    constexpr int N = 16 / (int)sizeof(T);
    if (!io.momentum) {
        const size_t packs = e / N;
        double part[4] = {0.0, 0.0, 0.0, 0.0};               // four chains
#pragma unroll 2
        for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < packs; i += (size_t)gridDim.x * 256) {
            const Pack<T, N> q = load_pack<T, N>((const T*)io.g + i * N);
#pragma unroll
            for (int k = 0; k < N; ++k) part[k & 3] += (double)(float)q.v[k] * (double)(float)q.v[k];
        }
        s = (part[0] + part[1]) + (part[2] + part[3]);
        if (blockIdx.x == 0 && threadIdx.x < (unsigned)(e - packs * N)) {
            const double v = (double)(float)((const T*)io.g)[packs * N + threadIdx.x];
            s += v * v;
        }
    } else {
        for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < e; i += (size_t)gridDim.x * 256) {
            const double v = (double)read_u<T>(io, i, true);
            s += v * v;
        }
    }
    for (int o = 1; o < 64; o <<= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) p.part[(size_t)blockIdx.y * NORM_BLOCKS + blockIdx.x] = red[0] + red[1] + red[2] + red[3];
}

__device__ __forceinline__ void split8(const float* v, f16x8& hi, f16x8& lo) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        hi[e] = (f16)v[e];
        lo[e] = (f16)(v[e] - (float)hi[e]);
    }
}
// eight neighbours k .. k + 7 of a packed row (k a multiple of 8)
__device__ __forceinline__ char* packed(char* base, size_t row, int k, int K) {
    return base + (row * (K / KS) + k / KS) * ROWB + (k % KS) * 2;
}
__device__ __forceinline__ void put8(char* to, const float* v) {
    f16x8 hi, lo;
    split8(v, hi, lo);
    *(f16x8*)to = hi;
    *(f16x8*)(to + 64) = lo;
}

// X_0 scaled and packed, both ways: one 64 x 64 tile a block.  Memory-bound: 4 bytes read, 8 written (4096 x 4096 fp32: 39 us, 5.2 TB/s).  (Rows behind R, which X and the R x R matrices have up to RA, are
// read by the products whose results are not written: they stay as they are.)
template <typename T>
__global__ __launch_bounds__(256) void ns_pack_kernel(const Big p) {
    __shared__ float sm[64][65];
    __shared__ double red[4];
    const int tid = threadIdx.x, z = blockIdx.z;
    const Io io = shifted(p.io, (size_t)p.m * p.n * z, sizeof(T));
    const bool tall = p.m > p.n;
    const int i0 = blockIdx.y * 64, k0 = blockIdx.x * 64;                    // rows of the short side, columns of the long
    float in[16];                                            // on their way while the norm is added up
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        const int a = 4 * j + (tid >> 6), b = tid & 63, i = i0 + (tall ? b : a), k = k0 + (tall ? a : b);
        in[j] = i < p.r && k < p.l ? read_u<T>(io, tall ? (size_t)k * p.n + i : (size_t)i * p.n + k, false) : 0.f;
    }
    double s = 0.0;
    for (int i = tid; i < NORM_BLOCKS; i += 256) s += p.part[(size_t)z * NORM_BLOCKS + i];
    for (int o = 1; o < 64; o <<= 1) s += __shfl_xor(s, o, 64);
    if ((tid & 63) == 0) red[tid >> 6] = s;
    __syncthreads();
    const double norm = sqrt(red[0] + red[1] + red[2] + red[3]), over = norm + (double)p.eps, size = norm / over;
    // (head: 0 of 0 / 0, and where there are NaN or infinities)
    const float head = size > 0.0 ? -((float)__builtin_amdgcn_frexp_exp(size) + __builtin_amdgcn_logf((float)__builtin_amdgcn_frexp_mant(size))) : 0.f;
    if (blockIdx.x == 0 && blockIdx.y == 0 && tid == 0) heads(p)[z] = head;
    // 2^lift SX / (norm + eps) in two factors, for either may be beyond fp32; a zero matrix stays zero
    const double scale = norm == 0.0 ? 0.0 : (double)SX / over;
    const int power = __builtin_amdgcn_frexp_exp(scale) + lift(head, 0);
    const float factor = (float)__builtin_amdgcn_frexp_mant(scale);
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        const int a = 4 * j + (tid >> 6), b = tid & 63;
        sm[tall ? b : a][tall ? a : b] = __builtin_ldexpf(in[j], power) * factor;
    }
    __syncthreads();
    char* x = p.x + (size_t)z * p.RA * p.L * 4;
    char* xt = p.xt + (size_t)z * p.R * p.L * 4;
    for (int u = tid; u < 512; u += 256) {
        float v[8];
        const int a = u >> 3, b = (u & 7) * 8;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = sm[a][b + e];
        put8(packed(x, i0 + a, k0 + b, p.L), v);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = sm[b + e][a];
        put8(packed(xt, k0 + a, i0 + b, p.R), v);
    }
}

// Tiles: 64 MT x 64 NT, a wave's share 32 MT x 32 NT.  The variants V: 0 is 256 x 128, 1 and 2 128 x 128, 3 128 x 64 and 4 64 x 64,
// for products too small to fill the CUs with larger ones.  Of 2, 3 and 4 two lie in a CU, and one tile's beginning and end pass
// beside the other's products; 1 has the CU to itself and twice the stages in flight.
constexpr int VARIANTS = 5;
constexpr int mt_of(int v) { return v == 0 ? 4 : v == 4 ? 1 : 2; }
constexpr int nt_of(int v) { return v < 3 ? 2 : 1; }
constexpr int per_cu(int v) { return v < 2 ? 1 : 2; }
// The products of the hi parts, and the two small terms in sums of their own, so that the large sum is rounded once per product
// and not three times.
template <int V>
struct Acc {
    f32x16 v[mt_of(V)][nt_of(V)], w[mt_of(V)][nt_of(V)];
};
template <int V>
struct Frag {
    f16x8 ah[mt_of(V)], al[mt_of(V)], bh[nt_of(V)], bl[nt_of(V)];
};
template <int V>
__device__ __forceinline__ void multiply(Acc<V>& acc, const Frag<V>& f) {
    constexpr int MT = mt_of(V), NT = nt_of(V);
#pragma unroll
    for (int a = 0; a < MT; ++a)
#pragma unroll
        for (int b = 0; b < NT; ++b) acc.w[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.al[a], f.bh[b], acc.w[a][b], 0, 0, 0);
#pragma unroll
    for (int a = 0; a < MT; ++a)
#pragma unroll
        for (int b = 0; b < NT; ++b) acc.v[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.ah[a], f.bh[b], acc.v[a][b], 0, 0, 0);
#pragma unroll
    for (int a = 0; a < MT; ++a)
#pragma unroll
        for (int b = 0; b < NT; ++b) acc.w[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.ah[a], f.bl[b], acc.w[a][b], 0, 0, 0);
}

template <int V>
constexpr int stages_of() {
    return V == 0 || V == 3 ? 3 : V == 2 ? 2 : 4;
}
// acc += rows [i0, i0 + 64 MT) of A times rows [j0, j0 + 64 NT) of B over the stages [s0, s1): operands packed alike, K along both.
// A stage lies in LDS as rows of 128 bytes whose eight 16-byte pieces are in the order piece ^ order(row): 16 neighbouring rows
// are read from different banks (64 banks hold two rows).  Three or four stages in LDS, copied there directly, all but one in
// flight.  A wave reads the operands of the next half stage among the products of the present one; one barrier a stage, in the
// middle: before it a wave has its reads of the stage behind it and its copies of the next one, after it the stage's place is
// filled again.  A wave's 128 x 64 reads 192 rows for three products of 128 x 64: 94 of the 128 bytes that LDS gives a cycle; with
// 64 x 64 it is 125, with less LDS bounds.  The smaller two variants' stages leave room for a second tile in a CU.
template <int V>
__device__ __forceinline__ void main_loop(Acc<V>& acc, const char* A, const char* B, int K, int i0, int j0, int s0, int s1, char* lds) {
    constexpr int MT = mt_of(V), NT = nt_of(V), TM = 64 * MT, TN = 64 * NT, STAGE = (TM + TN) * ROWB, NST = stages_of<V>();
    constexpr int NA = TM / 32, NB = TN / 32, NL = NA + NB;                  // a wave's copies, of 8 rows each
    constexpr int GROUPS = V == 0 ? 12 : V < 3 ? 4 : V == 3 ? 3 : 1;        // reads are issued in so many parts, a product between two
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l31 = lane & 31, q = lane >> 5;
    const size_t pitch = (size_t)(K / KS) * ROWB;
    const int lrow = lane >> 3, piece = (lane & 7) ^ lrow, order = (l31 & 7) ^ ((l31 >> 3) & 1);
    // a copy's address: the panel's descriptor, this lane's place in it, and a scalar offset
    const __amdgpu_buffer_rsrc_t pa = __builtin_amdgcn_make_buffer_rsrc((void*)(A + (size_t)i0 * pitch), 0, 0xffffffff, 0x00020000);
    const __amdgpu_buffer_rsrc_t pb = __builtin_amdgcn_make_buffer_rsrc((void*)(B + (size_t)j0 * pitch), 0, 0xffffffff, 0x00020000);
    const unsigned va = (unsigned)((wave * (TM / 4) + lrow) * pitch), vb = (unsigned)((wave * (TN / 4) + lrow) * pitch);
    const unsigned at8[2] = {piece * 16u, (piece ^ 1) * 16u};                // rows 0 .. 7 and 8 .. 15 of each 16
    const unsigned row8 = (unsigned)(8 * pitch);
    char* da = lds + wave * (TM / 4) * ROWB;
    char* db = lds + TM * ROWB + wave * (TN / 4) * ROWB;
    auto copy = [](__amdgpu_buffer_rsrc_t from, unsigned lane_at, unsigned at, char* to) {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (__attribute__((address_space(3))) void*)to, 16, (int)lane_at, (int)at, 0, 0);
    };
    auto issue = [&](int s, int buf) {
        const unsigned at = (unsigned)(s < s1 ? s : s1 - 1) * ROWB;          // behind the end: any stage, never used
#pragma unroll
        for (int i = 0; i < NA; ++i) copy(pa, va + at8[i & 1], at + i * row8, da + buf * STAGE + i * 1024);
#pragma unroll
        for (int i = 0; i < NB; ++i) copy(pb, vb + at8[i & 1], at + i * row8, db + buf * STAGE + i * 1024);
    };
    const char* ra = lds + ((wave >> 1) * (TM / 2) + l31) * ROWB;
    const char* rb = lds + (TM + (wave & 1) * (TN / 2) + l31) * ROWB;
    auto read = [&](Frag<V>& f, int buf, int kk) {
        const int hi = buf * STAGE + (((kk * 2 + q) ^ order) * 16), lo = buf * STAGE + (((4 + kk * 2 + q) ^ order) * 16);
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            f.al[t] = *(const f16x8*)(ra + lo + t * 32 * ROWB);
            f.ah[t] = *(const f16x8*)(ra + hi + t * 32 * ROWB);
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            f.bh[t] = *(const f16x8*)(rb + hi + t * 32 * ROWB);
            f.bl[t] = *(const f16x8*)(rb + lo + t * 32 * ROWB);
        }
    };
#pragma unroll
    for (int i = 0; i < NST; ++i) issue(s0 + i, i);
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NST - 1) * NL) : "memory");
    __builtin_amdgcn_s_barrier();
    Frag<V> f0, f1;
    read(f0, 0, 0);
    int buf = 0;
    for (int s = s0; s < s1; ++s) {
        const int next = buf == NST - 1 ? 0 : buf + 1;
        __builtin_amdgcn_s_waitcnt(0xc07f);       // lgkmcnt(0): f0, read half a stage ago.  (The builtin, which the compiler counts
        __builtin_amdgcn_sched_barrier(0);        // too: else it waits for f1 as well before f0 is used.)
        read(f1, buf, 1);
        multiply(acc, f0);
        // the reads among the first half of the products: the rest of them covers the last read's way
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x100, 2 * (MT + NT) / GROUPS, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("" ::: "memory");
        constexpr int FLY = (NST - 2) * NL;       // lgkmcnt(0), vmcnt(FLY): f1, and this wave's copies of the next stage
        __builtin_amdgcn_s_waitcnt(0x0070 | (FLY & 15) | FLY >> 4 << 14);
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        read(f0, next, 0);
        issue(s + NST, buf);
        multiply(acc, f1);
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x100, 2 * (MT + NT) / GROUPS, 1);
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 1);
        }
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x010, 1, 1);
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 1);
        }
        __builtin_amdgcn_sched_barrier(0);
        buf = next;
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");              // the copies behind the end
    __syncthreads();
}

// f(row, column, value) for the wave's share of a tile
template <int V, typename F>
__device__ __forceinline__ void each(const Acc<V>& acc, F f) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l31 = lane & 31, q = lane >> 5;
    constexpr int MT = mt_of(V), NT = nt_of(V);
    const int wi = (wave >> 1) * 32 * MT, wj = (wave & 1) * 32 * NT;
#pragma unroll
    for (int a = 0; a < MT; ++a)
#pragma unroll
        for (int b = 0; b < NT; ++b)
#pragma unroll
            for (int e = 0; e < 16; ++e)
                f(wi + 32 * a + 8 * (e >> 2) + 4 * q + (e & 3), wj + 32 * b + l31, acc.v[a][b][e] + acc.w[a][b][e]);
}

// The products: what they multiply, and what becomes of `rows` rows of a tile [rows][EP] in LDS that begins at (i0, j0).
enum Product { XXT, POLY, SYM, UPDATE, RESULT };                             // X X^T; q(s1); s1 s2, commuting; s2 X; s2 X as the result

// tiles that hold the diagonal of an R x R matrix and what is over it, in blocks of 8 tiles' columns squared (which share their
// operands in an XCD's L2): block column after block column
__device__ __host__ __forceinline__ int tri_count(int cols, int per) {       // tiles of the first `cols` columns of a block on the diagonal
    int n = 0;
    for (int j = 0; j < cols; ++j) n += j / per + 1;
    return n;
}
template <int V>
__device__ __forceinline__ void tri_tile(int t, int cols, int& ti, int& tj) {
    constexpr int PER = mt_of(V) / nt_of(V), H = 8 / PER;   // columns of tiles per row of tiles; rows of tiles in a block
    int J = 0;
    for (;; ++J) {
        const int w = cols - 8 * J < 8 ? cols - 8 * J : 8;
        const int n = J * H * w + tri_count(w, PER);
        if (t < n) {
            if (t < J * H * w) {
                const int blk = t / (H * w), in = t % (H * w);
                ti = blk * H + in / w;
                tj = 8 * J + in % w;
            } else {
                t -= J * H * w;
                int j = 0;
                while (t >= j / PER + 1) t -= j++ / PER + 1;
                ti = J * H + t;
                tj = 8 * J + j;
            }
            return;
        }
        t -= n;
    }
}
int tri_tiles(int cols, int per) {
    const int h = 8 / per;
    int n = 0;
    for (int J = 0; 8 * J < cols; ++J) {
        const int w = cols - 8 * J < 8 ? cols - 8 * J : 8;
        n += J * h * w + tri_count(w, per);
    }
    return n;
}

template <int PROD, int V>
__device__ __forceinline__ void locate(const Big& p, int tile, int& z, int& i0, int& j0, int tiles) {
    constexpr int MT = mt_of(V), TN = 64 * nt_of(V);
    z = tile / tiles;
    int t = tile - z * tiles, ti, tj;
    if constexpr (PROD <= SYM) {
        tri_tile<V>(t, (p.r + TN - 1) / TN, ti, tj);
    } else {                                       // eight columns of tiles at a time
        const int rows = (p.l + 64 * MT - 1) / (64 * MT), cols = (p.r + TN - 1) / TN, g = t / (8 * rows), w = cols - 8 * g < 8 ? cols - 8 * g : 8, in = t - g * 8 * rows;
        ti = in / w;
        tj = 8 * g + in % w;
    }
    i0 = ti * 64 * MT;
    j0 = tj * TN;
}
// pitch of a tile in LDS at the end: rows of 16-byte pieces, or columns in different banks where the result is written by columns
template <int PROD, int TN>
constexpr int pitch_of() {
    return PROD == RESULT ? TN + 1 : TN + 4;
}
// columns of ROWS rows in LDS as rows of a packed matrix: four neighbouring threads write 64 bytes of a row, and a wave reads at
// most two values from a bank
template <int ROWS, int TN, int EP, typename F>
__device__ __forceinline__ void transposed(const float* sm, F to) {
#pragma unroll 4
    for (int u = threadIdx.x; u < ROWS * TN / 8; u += 256) {
        const int j = ROWS == 8 ? u : (u >> 2) & (TN - 1), i = ROWS == 8 ? 0 : (u / (4 * TN) * 4 + (u & 3)) * 8;
        char* d = to(i, j);
        if (!d) continue;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = sm[(i + e) * EP + j];
        put8(d, v);
    }
}

template <int PROD, int ROWS, int TN, typename T>
__device__ __forceinline__ void finish(const Big& p, float* sm, int z, int i0, int j0, float head) {
    constexpr int EP = pitch_of<PROD, TN>(), STEP = 256 / (TN / 8);           // rows that the threads' packs of eight neighbours cover
    constexpr int N = ROWS < STEP ? 1 : ROWS / STEP, M = N < 8 ? N : 8;      // N times, M of them at a time
    const int row = threadIdx.x / (TN / 8), col = threadIdx.x % (TN / 8) * 8;
    if constexpr (PROD <= SYM) {
        char* to = p.s3 + (size_t)z * p.RA * p.R * 4;
        const char* a = p.s1 + (size_t)z * p.RA * p.R * 4;
        const int cb = j0 / TN;
        const float qb = PROD == POLY ? __builtin_ldexpf((float)QB * (SQ[0] / SA), -2 * lift(head, p.from)) : 0.f;
        for (int u = 0; u < N; u += M) {
            f16x8 hi[M], lo[M];
            if constexpr (PROD == POLY) {
#pragma unroll
                for (int k = 0; k < M; ++k) {
                    const int i = row + STEP * (u + k);
                    if (i >= ROWS || (i0 + i) / TN > cb) continue;
                    const char* s = packed((char*)a, i0 + i, j0 + col, p.R);
                    hi[k] = *(const f16x8*)s;
                    lo[k] = *(const f16x8*)(s + 64);
                }
            }
#pragma unroll
            for (int k = 0; k < M; ++k) {
                const int i = row + STEP * (u + k);
                if (i >= ROWS || (i0 + i) / TN > cb) continue;
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    v[e] = sm[i * EP + col + e];
                    if constexpr (PROD == POLY) {
                        v[e] += qb * ((float)hi[k][e] + (float)lo[k][e]);
                        if (i0 + i == j0 + col + e) v[e] += (float)QA * SQ[0];
                        sm[i * EP + col + e] = v[e];
                    }
                }
                put8(packed(to, i0 + i, j0 + col, p.R), v);
            }
        }
        if constexpr (PROD == POLY) __syncthreads();
        transposed<ROWS, TN, EP>(sm, [&](int i, int j) { return (i0 + i) / TN >= cb ? nullptr : packed(to, j0 + j, i0 + i, p.R); });
    } else if constexpr (PROD == UPDATE) {                                   // rows: the long side
        char* xt = p.xt2 + (size_t)z * p.R * p.L * 4;
        char* x = p.x + (size_t)z * p.RA * p.L * 4;
#pragma unroll 4
        for (int i = row; i < ROWS; i += STEP) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = sm[i * EP + col + e];
            put8(packed(xt, i0 + i, j0 + col, p.R), v);
        }
        transposed<ROWS, TN, EP>(sm, [&](int i, int j) { return packed(x, j0 + j, i0 + i, p.L); });
    } else {
        // packs along the matrix's rows: of the tile's columns where the long side is the matrix's rows, of its rows otherwise
        const Io io = shifted(p.io, (size_t)p.m * p.n * z, sizeof(T));
        const bool tall = p.m > p.n;
        constexpr int V = 16 / (int)sizeof(T), RP = ROWS / V;
#pragma unroll 2
        for (int u = threadIdx.x; u < ROWS * TN / V; u += 256) {
            const int i = tall ? u / (TN / V) : u % RP * V, j = tall ? u % (TN / V) * V : u / RP;
            const int left = tall ? (i0 + i < p.l ? p.r - (j0 + j) : 0) : (j0 + j < p.r ? p.l - (i0 + i) : 0);
            if (left <= 0) continue;
            const size_t at = tall ? (size_t)(i0 + i) * p.n + j0 + j : (size_t)(j0 + j) * p.n + i0 + i;
            float v[V];
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = tall ? sm[i * EP + j + e] : sm[(i + e) * EP + j];
            if (left >= V && !io.param) {
                Pack<T, V> o;
#pragma unroll
                for (int e = 0; e < V; ++e) o.v[e] = (T)v[e];                // the result's only rounding to fewer bits
                store_pack<T, V>((T*)io.out + at, o);
            } else if (left >= V) {
                Pack<float, V> o = load_pack<float, V>(io.param + at);
#pragma unroll
                for (int e = 0; e < V; ++e) o.v[e] = o.v[e] * io.keep - io.step * v[e];
                store_pack<float, V>(io.param + at, o);
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e)
                    if (e < left) write_o<T>(io, at + e, v[e]);
            }
        }
    }
}

// Blocks [0, full): a tile each, the card's CUs filled `full / 256` times.  The tiles that are left share the card: `splits`
// blocks a tile, each with a part of the contraction, whose sums ns_join_kernel adds up.
template <int PROD, int V, typename T>
__global__ __launch_bounds__(256, per_cu(V)) void ns_product_kernel(const Big p, int tiles, int full, int splits) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    // blocks go to the eight XCDs in turn: each gets neighbouring tiles, whose operands its L2 then holds
    auto neighbours = [](int b, int n) { return (b & 7) * (n >> 3) + min(b & 7, n & 7) + (b >> 3); };
    int tile, split = 0;
    if ((int)blockIdx.x < full) tile = neighbours(blockIdx.x, full);
    else {
        const int rest = ((int)gridDim.x - full) / splits, u = neighbours((int)blockIdx.x - full, (int)gridDim.x - full);
        split = u / rest;
        tile = full + u % rest;
    }
    const bool whole = (int)blockIdx.x < full || splits == 1;
    int z, i0, j0;
    locate<PROD, V>(p, tile, z, i0, j0, tiles);
    const float head = PROD == XXT ? 0.f : heads(p)[z];      // (read here, it has come before it is looked at)
    const char *A, *B;
    int K;
    if constexpr (PROD == XXT) {
        A = B = p.x + (size_t)z * p.RA * p.L * 4;
        K = p.L;
    } else if constexpr (PROD <= SYM) {
        A = p.s1 + (size_t)z * p.RA * p.R * 4;
        B = PROD == POLY ? A : p.s2 + (size_t)z * p.RA * p.R * 4;
        K = p.R;
    } else {
        A = p.xt + (size_t)z * p.R * p.L * 4;
        B = p.s2 + (size_t)z * p.RA * p.R * 4;
        K = p.R;
    }
    const int stages = ((PROD == XXT ? p.l : p.r) + KS - 1) / KS;            // (behind them is nothing but zeros)
    const int s0 = whole ? 0 : (int)((long long)stages * split / splits), s1 = whole ? stages : (int)((long long)stages * (split + 1) / splits);
    constexpr int MT = mt_of(V), TN = 64 * nt_of(V);
    Acc<V> acc;
#pragma unroll
    for (int a = 0; a < MT; ++a)
#pragma unroll
        for (int b = 0; b < nt_of(V); ++b)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc.v[a][b][e] = acc.w[a][b][e] = 0.f;
    main_loop(acc, A, B, K, i0, j0, s0, s1, smem);
    // the operands' lift off, the result's on (the last result's power is not one with the factor: it may be beyond fp32)
    int power = 0;
    if constexpr (PROD == POLY) power = -4 * lift(head, p.from);
    else if constexpr (PROD == SYM || PROD == UPDATE) power = (PROD == SYM ? 2 : 1) * (lift(head, p.from + p.by) - lift(head, p.from));
    else if constexpr (PROD == RESULT) power = -lift(head, p.from);
    const float f = PROD == RESULT ? p.scale : __builtin_ldexpf(p.scale, power);
    auto scaled = [=](float v) { return PROD == RESULT ? __builtin_ldexpf(v * f, power) : v * f; };
    if (whole) {
        float* sm = (float*)smem;
        each(acc, [&](int i, int j, float v) { sm[i * pitch_of<PROD, TN>() + j] = scaled(v); });
        __syncthreads();
        finish<PROD, 64 * MT, TN, T>(p, sm, z, i0, j0, head);
    } else {
        float* slab = p.slab + ((size_t)(tile - full) * splits + split) * (64 * MT * TN);
        each(acc, [&](int i, int j, float v) { slab[i * TN + j] = scaled(v); });
    }
}
// eight rows of a split tile, its shares added in order (16 tiles of 16 shares: 6 us)
template <int PROD, int V, typename T>
__global__ __launch_bounds__(256) void ns_join_kernel(const Big p, int tiles, int full, int splits) {
    constexpr int MT = mt_of(V), TN = 64 * nt_of(V), EP = pitch_of<PROD, TN>();
    __shared__ __attribute__((aligned(16))) float sm[8 * EP];
    int z, i0, j0;
    locate<PROD, V>(p, full + blockIdx.x, z, i0, j0, tiles);
    const float head = PROD == POLY ? heads(p)[z] : 0.f;
    const int i = threadIdx.x / (TN / 4), j = threadIdx.x % (TN / 4) * 4;
    if (i < 8) {
        const float* slab = p.slab + (size_t)blockIdx.x * splits * (64 * MT * TN) + (blockIdx.y * 8 + i) * TN + j;
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
        for (int s = 0; s < splits; ++s) v += *(const f32x4*)(slab + (size_t)s * 64 * MT * TN);
#pragma unroll
        for (int e = 0; e < 4; ++e) sm[i * EP + j + e] = v[e];
    }
    __syncthreads();
    finish<PROD, 8, TN, T>(p, sm, z, i0 + blockIdx.y * 8, j0, head);
}

// ---------------------------------------------------------------------------------------------- host
// How a product's tiles are shared out: variant v; whole rounds over the CUs, and the rest in `splits` parts
struct Share {
    int v, tiles, full, rest, splits;
};
// The variant that takes the least time by this count, in cycles at the 1.8 GHz of a full card: a stage 2290 at 256 x 128 a tile (1536
// of them on the matrix cores), 1150 and 1180 at 128 x 128, 690 at 128 x 64, 480 at 64 x 64; a tile's beginning and end, half of
// which two tiles in a CU share; writing the parts of split tiles and joining them.  All five steps in us:
//                             as chosen   tiles never split   one 128 x 128 a CU only   128 columns only   256 x 128 only
//   4096 x 4096 fp32                3660                4178                      3787               3652             3792
//   3 x 4101 x 1030 bf16             637                 638                       668                764              890
//   256 x 19200 fp32                 185                 497                       192                276              370
//   1024 x 4096 fp32                 319                 337                       318                401              503
//   512 x 512 fp32                   132                 132                       131                194              241
Share share(int v, long long tiles, long long total) {
    Share s{v, (int)tiles, (int)(total / CUS * CUS), (int)(total % CUS), 1};
    return s;
}
double cycles(const Share& s, int stages) {
    static const double stage[VARIANTS] = {2290, 1150, 1180, 690, 480}, end[VARIANTS] = {18000, 11000, 10000, 14000, 7000};
    const double one = stage[s.v], ends = end[s.v], more = per_cu(s.v) == 1 ? 1.0 : 0.5;
    const int rounds = s.full / CUS;
    double c = rounds * stages * one + (rounds ? 1 + (rounds - 1) * more : 0) * ends;
    if (s.rest) c += (s.splits > 1 ? (stages + s.splits - 1) / s.splits * one + ends + 12000 + 150 * s.rest : stages * one + (rounds ? more : 1) * ends);
    return c;
}
Share best(const Share& a, const Share& b, int stages) { return cycles(b, stages) < cycles(a, stages) ? b : a; }
Share fastest(int v, long long tiles, int nb, int stages) {
    Share s = share(v, tiles, tiles * nb), t = s;
    if (s.rest) {
        t.splits = CUS / s.rest;
        if (t.splits > stages / 4) t.splits = stages / 4;
        if (t.splits > 48) t.splits = 48;
        if (t.splits < 2) t.splits = 1;
    }
    return best(s, t, stages);
}
struct Layout {
    size_t part, x, xt, xt2, r[4], slab, total;
    int sub, R, L, RA;
    bool group;                                   // steps are taken together
    Share xxt, sym, update;
};
Layout layout_of(int nb, int r, int l) {
    Layout o{};
    o.R = step::round_up(r, 128);
    o.L = step::round_up(l, 256);
    o.RA = step::round_up(r, 256);
    const int sx = step::ceil_div(l, KS), sr = step::ceil_div(r, KS);
    auto of = [&](bool tri, int stages) {
        Share s{};
        for (int v = 0; v < VARIANTS; ++v) {
            const int mt = mt_of(v), nt = nt_of(v), cols = step::ceil_div(r, 64 * nt);
            const long long tiles = tri ? tri_tiles(cols, mt / nt) : (long long)step::ceil_div(l, 64 * mt) * cols;
            if (v == 2 && tiles * nb <= CUS) continue;       // one tile a CU: two stages are too few
            const Share t = fastest(v, tiles, nb, stages);
            s = v == 0 ? t : best(s, t, stages);
        }
        return s;
    };
    o.xxt = of(true, sx);
    o.sym = of(true, sr);
    o.update = of(false, sr);
    return o;
}
// workspace of a stack of `batch` matrices with r > 64, `sub` of them at a time
Layout layout(int batch, int m, int n) {
    const int r = m < n ? m : n, l = m < n ? n : m;
    const size_t most = (size_t)1 << 28;                           // elements of X at a time
    const size_t fit = most / ((size_t)step::round_up(r, 256) * step::round_up(l, 256));
    int sub = (int)(fit < (size_t)batch ? fit : (size_t)batch);
    sub = sub < 1 ? 1 : sub > BATCH ? BATCH : sub;
    Layout o = layout_of(sub, r, l);
    o.sub = sub;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    const size_t R = o.R, L = o.L, RA = o.RA;
    o.part = take(BATCH * sizeof(float) + (size_t)sub * NORM_BLOCKS * sizeof(double)) + BATCH * sizeof(float);
    o.x = take(sub * RA * L * 4);
    o.xt = take(sub * R * L * 4);
    o.xt2 = take(sub * R * L * 4);
    // Steps taken together: k steps at once are one X X^T and one P X, P = q(A_k) .. q(A_1), with A_i+1 = q(A_i) A_i q(A_i) from
    // products of r x r matrices, of which each further step takes three more: where the two passes over X cost more than those
    // (3 x 4101 x 1030 bf16: 637 us together, 933 step by step; 400 x 900, taken step by step, 139, and 150 together; 3.8 passes' worth is
    // where they are even: 1690 x 71 111, step by step).  together() says how many.
    const double passes = cycles(o.xxt, step::ceil_div(l, KS)) + cycles(o.update, step::ceil_div(r, KS));
    o.group = l >= 2 * r && passes > 3.8 * cycles(o.sym, step::ceil_div(r, KS));
    for (int i = 0; i < (o.group ? 4 : 2); ++i) o.r[i] = take(sub * RA * R * 4);
    // shares of split tiles: fewer than one a CU, of 256 x 128 at most.  A last part of the batch that is smaller is shared out anew.
    const bool any = sub < batch || o.xxt.splits > 1 || o.sym.splits > 1 || o.update.splits > 1;
    o.slab = take(any ? (size_t)CUS * 256 * 128 * 4 : 0);
    o.total = at;
    return o;
}
bool small(int m, int n) { return (m < n ? m : n) <= 64; }

// matrices [from, from + count) of an item
struct Piece {
    int item, from, count, first;          // first: number of its first matrix in the group
    SmallItem s;
};
struct Group {
    std::vector<Piece> pieces;
    int total, max_chunks, max_parts;
    size_t doubles;
};
// Matrices of a group: 218 MB of workspace (the sums of one chunk and P, 52 KB a matrix), and sixteen times what the CUs hold at a time.
// A launch has fewer than 2^32 threads: ns_apply_kernel's bound is the first to be met, 256 threads for each part of each matrix.
constexpr int GROUP_MATRICES = 4096;
constexpr int GROUP_PARTS = (1 << 24) - 1;
// small items in groups of one launch of each kernel; the workspace is used again by every group
std::vector<Group> small_groups(const step_ns_item* items, int count) {
    std::vector<Group> groups;
    auto parts_of = [&](int i) { return step::ceil_div(items[i].m > items[i].n ? items[i].m : items[i].n, 64); };
    auto room = [&](int parts) { return GROUP_PARTS / parts < GROUP_MATRICES ? GROUP_PARTS / parts : GROUP_MATRICES; };
    // `of`: the matrices that share the card, for the count of chunks (all of a stack, so that its matrices are added up alike)
    auto add = [&](std::vector<Piece>& pieces, int of) {
        Group g{};
        g.max_chunks = g.max_parts = 1;
        const int share = of < 1024 ? 1024 / of : 1;
        for (Piece& p : pieces) {
            const step_ns_item& it = items[p.item];
            const int l = it.m > it.n ? it.m : it.n;
            int chunks = step::ceil_div(l, 16 * GRAM_WAVES);
            if (chunks > share) chunks = share;
            if (chunks > 32) chunks = 32;
            p.s.m = it.m;
            p.s.n = it.n;
            p.s.width = step::round_up(step::ceil_div(l, chunks), 16);
            p.s.chunks = step::ceil_div(l, p.s.width);
            p.s.slab = g.doubles;
            g.doubles += (size_t)p.count * p.s.chunks * 2560;
            p.s.p = g.doubles;
            g.doubles += (size_t)p.count * 4096;
            p.first = g.total;
            g.total += p.count;
            if (p.s.chunks > g.max_chunks) g.max_chunks = p.s.chunks;
            if (parts_of(p.item) > g.max_parts) g.max_parts = parts_of(p.item);
        }
        g.pieces.swap(pieces);
        groups.push_back(std::move(g));
        pieces.clear();
    };
    std::vector<Piece> open;
    int total = 0, parts = 1;
    for (int i = 0; i < count; ++i) {
        if (!small(items[i].m, items[i].n)) continue;
        const int mine = parts_of(i), most = mine > parts ? mine : parts, batch = items[i].batch;
        if (!open.empty() && ((int)open.size() == S_ITEMS || batch > room(most) - total)) {
            add(open, total);
            total = 0;
            parts = 1;
        }
        if (batch > room(mine)) {                            // a stack of several groups, by itself
            for (int from = 0; from < batch; from += room(mine)) {
                std::vector<Piece> one{Piece{i, from, batch - from < room(mine) ? batch - from : room(mine), 0, SmallItem{}}};
                add(one, batch);
            }
            continue;
        }
        open.push_back(Piece{i, 0, batch, 0, SmallItem{}});
        total += batch;
        if (mine > parts) parts = mine;
    }
    if (!open.empty()) add(open, total);
    return groups;
}

int check(const step_ns_item* items, int count) {
    STEP_REQUIRE(items && count >= 1, "step_newton_schulz: no matrices");
    long long total = 0;
    for (int i = 0; i < count; ++i) {
        const step_ns_item& it = items[i];
        STEP_REQUIRE(it.batch >= 1 && it.m >= 1 && it.n >= 1, "step_newton_schulz: item %d: bad shape %d x %d x %d", i, it.batch, it.m, it.n);
        STEP_REQUIRE(it.m <= (1 << 21) && it.n <= (1 << 21), "step_newton_schulz: item %d: %d x %d is over 2^21 a side", i, it.m, it.n);
        STEP_REQUIRE((it.m < it.n ? it.m : it.n) <= 32768, "step_newton_schulz: item %d: %d x %d is over 32768 on both sides", i, it.m, it.n);
        total += it.batch;
        STEP_REQUIRE((long long)it.batch * step::ceil_div(it.m > it.n ? it.m : it.n, 64) < 1LL << 31, "step_newton_schulz: item %d: %d matrices of %d x %d", i,
                     it.batch, it.m, it.n);
    }
    STEP_REQUIRE(total <= 1 << 24, "step_newton_schulz: %lld matrices", total);
    return STEP_OK;
}

template <int PROD, int V, typename T>
int product_of(const Big& p, const Share& s, hipStream_t st) {
    auto kern = ns_product_kernel<PROD, V, T>;
    constexpr size_t loop = stages_of<V>() * 64 * (mt_of(V) + nt_of(V)) * ROWB, end = 64 * mt_of(V) * pitch_of<PROD, 64 * nt_of(V)>() * sizeof(float);
    constexpr size_t lds = loop > end ? loop : end;
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) {
        step::set_error("step_newton_schulz: hipFuncSetAttribute(%zu): %s", lds, hipGetErrorString(e));
        return STEP_ERR_LAUNCH;
    }
    hipLaunchKernelGGL(kern, dim3(s.full + s.rest * s.splits), dim3(256), lds, st, p, s.tiles, s.full, s.splits);
    if (s.splits > 1) hipLaunchKernelGGL((ns_join_kernel<PROD, V, T>), dim3(s.rest, 8 * mt_of(V)), dim3(256), 0, st, p, s.tiles, s.full, s.splits);
    return STEP_OK;
}
template <int PROD, typename T>
int product(const Big& p, const Share& s, hipStream_t st) {
    switch (s.v) {
        case 0: return product_of<PROD, 0, T>(p, s, st);
        case 1: return product_of<PROD, 1, T>(p, s, st);
        case 2: return product_of<PROD, 2, T>(p, s, st);
        case 3: return product_of<PROD, 3, T>(p, s, st);
        default: return product_of<PROD, 4, T>(p, s, st);
    }
}
// Steps taken together: the first `first` alone, then `most` at a time, where layout() finds that this pays.  An error of A grows by
// a^2 = 12 in each step of a group for the smallest eigenvalues, so that three at a time are for results of 16 bits, rounded far above
// it.  fp32 takes the first step, before which the smallest are smallest, by itself and then two at a time.  Its error over that of
// fp32 products (the library's), the worst of six kinds of matrices (low rank and noise, Gaussian, singular values over a range of 30
// and of 1000, ...), step by step / one and two / three at a time: 160 x 6000 1.08 / 1.12 / 1.67, 192 x 14000 1.05 / 1.08 / 1.40,
// 256 x 9000 1.04 / 1.07 / 1.3, 340 x 6000 1.04 / 1.09 / 1.36, 1000 x 3000 0.93 / 1.05 / 0.96, 1400 x 6000 0.92 / 1.08 / 0.96; not
// taken together: 130 x 6000 1.13 / 1.17 / 1.52, 1400 x 4000 0.94 / 1.40 / 1.32.  Times: 256 x 19200 218 / 183 / 167 us, 1000 x 6000
// 450 / 368 / 334, 192 x 7000 152 / 136 / 130.
struct Together {
    int first, most;
};
template <typename T>
Together together(int r, int l) {
    if (sizeof(T) < 4) return Together{3, 3};
    return r >= 160 && l >= 4 * r ? Together{1, 2} : Together{1, 1};
}
template <typename T>
int run_big(const step_ns_item& it, const Io& io, int steps, float eps, char* base, hipStream_t st) {
    const Layout all = layout(it.batch, it.m, it.n);
    Big p{};
    p.m = it.m;
    p.n = it.n;
    p.r = it.m < it.n ? it.m : it.n;
    p.l = it.m < it.n ? it.n : it.m;
    p.R = all.R;
    p.L = all.L;
    p.RA = all.RA;
    p.eps = eps;
    p.part = (double*)(base + all.part);
    p.slab = (float*)(base + all.slab);
    p.x = base + all.x;
    const Together group = all.group ? together<T>(p.r, p.l) : Together{1, 1};
    char* r[4];
    for (int i = 0; i < 4; ++i) r[i] = base + all.r[i];
    for (int b0 = 0; b0 < it.batch; b0 += all.sub) {
        const int nb = it.batch - b0 < all.sub ? it.batch - b0 : all.sub;
        const Layout o = layout_of(nb, p.r, p.l);
        const size_t by = (size_t)b0 * it.m * it.n;
        p.io = io;
        p.io.g = (const T*)io.g + by;
        if (io.out) p.io.out = (T*)io.out + by;
        if (io.momentum) p.io.momentum = io.momentum + by;
        if (io.param) p.io.param = io.param + by;
        p.xt = base + all.xt;
        p.xt2 = base + all.xt2;
        hipLaunchKernelGGL(ns_norm_kernel<T>, dim3(NORM_BLOCKS, nb), dim3(256), 0, st, p);
        hipLaunchKernelGGL(ns_pack_kernel<T>, dim3(p.L / 64, p.R / 64, nb), dim3(256), 0, st, p);
        int rc = STEP_OK;
        // s3 <- s1 s2, scales f1, f2 -> f3; from A_k to A_k + 1 where it is that
        auto sym = [&](const char* s1, float f1, const char* s2, float f2, char* s3, float f3, int k = -1) {
            p.from = k;
            p.by = k < 0 ? 0 : 1;
            p.s1 = s1;
            p.s2 = s2;
            p.s3 = s3;
            p.scale = f3 / (f1 * f2);
            if (rc == STEP_OK) rc = product<SYM, float>(p, o.sym, st);
        };
        auto poly = [&](const char* a, char* to, int k) {
            p.from = k;
            p.s1 = a;
            p.s3 = to;
            p.scale = (float)QC * SQ[0] / (SA * SA);
            if (rc == STEP_OK) rc = product<POLY, float>(p, o.sym, st);
        };
        for (int s = 0; s < steps && rc == STEP_OK;) {
            const int want = s ? group.most : group.first, g = steps - s < want ? steps - s : want;
            char *A = r[0], *P = r[1], *Q = r[1], *W = r[2], *F = r[3];      // F: free
            p.s3 = A;
            p.scale = SA / (SX * SX);
            rc = product<XXT, float>(p, o.xxt, st);
            poly(A, Q, s);
            for (int k = 1; k < g; ++k) {
                sym(Q, SQ[0], A, SA, W, SA);                                 // A <- q(A) A q(A)
                sym(W, SA, Q, SQ[0], A, SA, s + k - 1);
                if (k > 1) {                                                 // (the last q(A) is no longer needed, P is)
                    F = Q;
                }
                poly(A, F, s + k);
                Q = F;
                sym(Q, SQ[0], P, SQ[k - 1], W, SQ[k]);
                F = P;
                P = W;
                W = F;
            }
            p.s2 = P;
            p.from = s;
            p.by = g;
            s += g;
            p.scale = s < steps ? SX / (SQ[g - 1] * SX) : 1.f / (SQ[g - 1] * SX);
            if (rc == STEP_OK) rc = s < steps ? product<UPDATE, float>(p, o.update, st) : product<RESULT, T>(p, o.update, st);
            char* t = p.xt;
            p.xt = p.xt2;
            p.xt2 = t;
        }
        if (rc != STEP_OK) return rc;
    }
    return STEP_OK;
}

template <typename T>
int run(const step_ns_item* items, int count, int steps, float eps, float mu, int nesterov, float lr, float decay, void* ws, hipStream_t st) {
    auto io_of = [&](const step_ns_item& it) {
        return Io{it.g, it.out, it.momentum, it.param, mu, 1.f - lr * decay, lr * it.scale, nesterov};
    };
    const std::vector<Group> groups = small_groups(items, count);
    if (!groups.empty()) {
        constexpr size_t lds = 3 * 64 * S_P * sizeof(double);
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(ns_small_kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) {
            step::set_error("step_newton_schulz: hipFuncSetAttribute(%zu): %s", lds, hipGetErrorString(e));
            return STEP_ERR_LAUNCH;
        }
    }
    for (const Group& g : groups) {
        constexpr size_t lds = 3 * 64 * S_P * sizeof(double);
        SmallArgs a{};
        const int n = (int)g.pieces.size();
        a.steps = steps;
        a.max_chunks = g.max_chunks;
        a.max_parts = g.max_parts;
        a.eps = eps;
        a.ws = (double*)ws;
        for (int i = 0; i < S_ITEMS; ++i) a.first[i] = i < n ? g.pieces[i].first : 0x7fffffff;
        for (int i = 0; i < n; ++i) {
            const Piece& p = g.pieces[i];
            const step_ns_item& it = items[p.item];
            a.item[i] = p.s;
            a.item[i].io = shifted(io_of(it), (size_t)p.from * it.m * it.n, sizeof(T));
        }
        hipLaunchKernelGGL(ns_gram_kernel<T>, dim3((unsigned)g.total * g.max_chunks), dim3(64 * GRAM_WAVES), 0, st, a);
        hipLaunchKernelGGL(ns_small_kernel, dim3((unsigned)g.total), dim3(SMALL_THREADS), lds, st, a);
        hipLaunchKernelGGL(ns_apply_kernel<T>, dim3((unsigned)g.total * g.max_parts), dim3(256), 0, st, a);
    }
    for (int i = 0; i < count; ++i) {
        if (small(items[i].m, items[i].n)) continue;
        const int rc = run_big<T>(items[i], io_of(items[i]), steps, eps, (char*)ws, st);
        if (rc != STEP_OK) return rc;
    }
    return step::check_launch("step_newton_schulz");
}

}  // namespace

extern "C" size_t step_newton_schulz_ws_bytes(const step_ns_item* items, int count) {
    if (check(items, count) != STEP_OK) return 0;
    try {
        size_t most = 256;
        for (int i = 0; i < count; ++i) {
            if (small(items[i].m, items[i].n)) continue;
            const size_t b = layout(items[i].batch, items[i].m, items[i].n).total;
            if (b > most) most = b;
        }
        for (const Group& g : small_groups(items, count))
            if (g.doubles * sizeof(double) > most) most = g.doubles * sizeof(double);
        return most;
    } catch (...) {
        step::set_error("step_newton_schulz_ws_bytes: out of host memory");
        return 0;
    }
}

extern "C" int step_newton_schulz(const step_ns_item* items, int count, int dtype, int steps, float eps, float momentum, int nesterov, float lr,
                                  float decay, void* ws, size_t ws_bytes, void* stream) {
    const int rc = check(items, count);
    if (rc != STEP_OK) return rc;
    STEP_REQUIRE(elem_bytes(dtype), "step_newton_schulz: unknown type %d", dtype);
    STEP_REQUIRE(steps >= 1 && steps <= 100, "step_newton_schulz: steps=%d", steps);
    STEP_REQUIRE(ws, "step_newton_schulz: null workspace");
    for (int i = 0; i < count; ++i) {
        STEP_REQUIRE(items[i].g && (items[i].out || items[i].param), "step_newton_schulz: item %d: null pointer", i);
        STEP_REQUIRE(!(items[i].momentum || items[i].param) || dtype == STEP_F32, "step_newton_schulz: item %d: the optimizer's form takes fp32", i);
    }
    const size_t need = step_newton_schulz_ws_bytes(items, count);
    if (!need || ws_bytes < need) {
        if (need) step::set_error("step_newton_schulz: workspace %zu < %zu bytes", ws_bytes, need);
        return STEP_ERR_WORKSPACE;
    }
    try {
        hipStream_t st = (hipStream_t)stream;
        if (dtype == STEP_F32) return run<float>(items, count, steps, eps, momentum, nesterov, lr, decay, ws, st);
        if (dtype == STEP_BF16) return run<bf16>(items, count, steps, eps, momentum, nesterov, lr, decay, ws, st);
        return run<f16>(items, count, steps, eps, momentum, nesterov, lr, decay, ws, st);
    } catch (...) {
        step::set_error("step_newton_schulz: out of host memory");
        return STEP_ERR_LAUNCH;
    }
}
