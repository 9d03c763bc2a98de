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
//   The trace of G G^T is the squared norm.  Three launches for a whole list of matrices: bound by latency.
//
// r > 64, every product on the f16 matrix cores: a value v, scaled by a power of two, is hi = f16(v) plus lo = f16(v - hi)
//   (together 22 bits and the sign of lo: the 24 bits of an fp32 value to half a unit or so), a product takes three terms
//   hi hi + hi lo + lo hi with fp32 accumulation.  The dropped lo lo is 2^-24 of a product.  The singular values stay
//   under 1.21 (q's maximum on [0, 1.46]) and so do all elements, so the scales are constants.  Matrices lie packed, 32
//   hi and 32 lo of a row in 128 bytes, X also transposed, so that every product has both its operands along the
//   contraction.  A and q(A) are symmetric: only the tiles on and over the diagonal are computed.
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
constexpr int S_P = 68;                           // row pitch of a 64 x 64 fp64 matrix in LDS: 8 rows in different banks

struct SmallItem {
    Io io;
    int m, n, first, chunks, width;               // first matrix of the item; chunks of `width` columns of the long side
    size_t slab, p;                               // offsets in the workspace, in doubles
};
struct SmallArgs {
    SmallItem item[S_ITEMS];
    int items, total, steps, max_chunks;
    float eps;
    double* ws;
};
// item and element offset of matrix z
__device__ __forceinline__ const SmallItem& find(const SmallArgs& p, int z, int& local) {
    int i = 0;
    while (i + 1 < p.items && p.item[i + 1].first <= z) ++i;
    local = z - p.item[i].first;
    return p.item[i];
}
__device__ __forceinline__ Io shifted(Io io, size_t by, int bytes) {
    io.g = (const char*)io.g + by * bytes;
    if (io.out) io.out = (char*)io.out + by * bytes;
    if (io.momentum) io.momentum += by;
    if (io.param) io.param += by;
    return io;
}

// one chunk of columns: its part of G G^T, upper 16 x 16 tiles, [10][256] doubles
template <typename T>
__global__ __launch_bounds__(256) void ns_gram_kernel(const SmallArgs p) {
    __shared__ double sm[10 * 256];
    const int z = blockIdx.x / p.max_chunks, chunk = blockIdx.x % p.max_chunks;
    int local;
    const SmallItem& it = find(p, z, local);
    if (chunk >= it.chunks) return;
    const bool tall = it.m > it.n;
    const int r = tall ? it.n : it.m, l = tall ? it.m : it.n;
    const Io io = shifted(it.io, (size_t)local * it.m * it.n, sizeof(T));
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i16 = lane & 15, q = lane >> 4;
    f64x4 acc[10];
#pragma unroll
    for (int t = 0; t < 10; ++t) acc[t] = f64x4{0, 0, 0, 0};
    const int c1 = min(l, (chunk + 1) * it.width);
    for (int c0 = chunk * it.width + 16 * wave; c0 < c1; c0 += 64) {
        // 16 columns; step s takes the columns 4 q + s (the order of a contraction is free)
        float u[4][4];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const int row = 16 * t + i16, col = c0 + 4 * q + s;
                u[t][s] = row < r && col < c1
                              ? read_u<T>(io, tall ? (size_t)col * it.n + row : (size_t)row * it.n + col, true)
                              : 0.f;
            }
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
    // the four waves' sums, in order
    for (int w = 0; w < 4; ++w) {
        if (wave == w)
#pragma unroll
            for (int t = 0; t < 10; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int at = t * 256 + i * 64 + lane;
                    sm[at] = w ? sm[at] + acc[t][i] : acc[t][i];
                }
        __syncthreads();
    }
    double* slab = p.ws + it.slab + ((size_t)local * it.chunks + chunk) * 2560;
    for (int e = threadIdx.x; e < 2560; e += 256) slab[e] = sm[e];
}

// C = X Y for commuting symmetric X, Y in LDS: tiles on and over the diagonal, mirrored; f(i, j, value) stores
template <typename F>
__device__ __forceinline__ void sym_product(const double* X, const double* Y, int nt, F f) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i16 = lane & 15, q = lane >> 4;
    int k = 0;
    for (int a = 0; a < nt; ++a)
        for (int b = a; b < nt; ++b, ++k) {
            if (k % 8 != wave) continue;
            f64x4 c{0, 0, 0, 0}, d{0, 0, 0, 0};
            for (int s = 0; s < 4 * nt; s += 2) {
                c = __builtin_amdgcn_mfma_f64_16x16x4f64(X[(16 * a + i16) * S_P + 4 * s + q], Y[(16 * b + i16) * S_P + 4 * s + q], c, 0, 0, 0);
                d = __builtin_amdgcn_mfma_f64_16x16x4f64(X[(16 * a + i16) * S_P + 4 * s + 4 + q], Y[(16 * b + i16) * S_P + 4 * s + 4 + q], d, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = 16 * a + 4 * i + q, col = 16 * b + i16;
                const double v = c[i] + d[i];
                if (a != b || row <= col) {                  // one value for both places, bit for bit
                    f(row, col, v);
                    if (row != col) f(col, row, v);
                }
            }
        }
}

__global__ __launch_bounds__(512) void ns_small_kernel(const SmallArgs p) {
    extern __shared__ __attribute__((aligned(16))) double lds[];
    __shared__ double norm_s;
    int local;
    const SmallItem& it = find(p, blockIdx.x, local);
    const int r = min(it.m, it.n), nt = (r + 15) / 16, R = 16 * nt, tid = threadIdx.x;
    double *A = lds, *Q = lds + 64 * S_P, *P = lds + 2 * 64 * S_P, *W = lds + 3 * 64 * S_P;
    const double* slab = p.ws + it.slab + (size_t)local * it.chunks * 2560;
    // join the chunks in order: element e of tile t is row 16 a + 4 (e / 64) + (e % 64) / 16, column 16 b + e % 16
    for (int e = tid; e < 2560; e += 512) {
        const int t = e >> 8, a = t < 4 ? 0 : t < 7 ? 1 : t < 9 ? 2 : 3, b = t < 4 ? t : t < 7 ? t - 3 : t < 9 ? t - 5 : 3;
        const int row = 16 * a + 4 * ((e & 255) >> 6) + ((e & 63) >> 4), col = 16 * b + (e & 15);
        if (b >= nt || (a == b && row > col)) continue;
        double v = 0.0;
        for (int c = 0; c < it.chunks; ++c) v += slab[(size_t)c * 2560 + e];
        A[row * S_P + col] = v;
        A[col * S_P + row] = v;
    }
    __syncthreads();
    if (tid == 0) {
        double tr = 0.0;
        for (int i = 0; i < r; ++i) tr += A[i * S_P + i];
        norm_s = 1.0 / (sqrt(tr) + (double)p.eps);
    }
    __syncthreads();
    const double inv = norm_s;
    for (int e = tid; e < R * R; e += 512) A[e / R * S_P + e % R] *= inv * inv;
    __syncthreads();
    if (!p.steps)
        for (int e = tid; e < R * R; e += 512) P[e / R * S_P + e % R] = e / R == e % R ? inv : 0.0;
    for (int step = 0; step < p.steps; ++step) {
        sym_product(A, A, nt, [&](int i, int j, double v) {
            const double w = QB * A[i * S_P + j] + QC * v + (i == j ? QA : 0.0);
            Q[i * S_P + j] = w;
            if (step == 0) P[i * S_P + j] = w * inv;
        });
        __syncthreads();
        const bool last = step + 1 == p.steps;
        if (step) {
            sym_product(Q, P, nt, [&](int i, int j, double v) { W[i * S_P + j] = v; });
            __syncthreads();
            double* t = P;
            P = W;
            W = t;
        }
        if (!last) {
            sym_product(Q, A, nt, [&](int i, int j, double v) { W[i * S_P + j] = v; });
            __syncthreads();
            sym_product(W, Q, nt, [&](int i, int j, double v) { A[i * S_P + j] = v; });
            __syncthreads();
        }
    }
    __syncthreads();
    double* out = p.ws + it.p + (size_t)local * 4096;
    for (int e = tid; e < R * R; e += 512) out[(e / R) * 64 + e % R] = P[e / R * S_P + e % R];
}

// O = P U: 16 columns of the long side a wave
template <typename T>
__global__ __launch_bounds__(256) void ns_apply_kernel(const SmallArgs p) {
    __shared__ double P[64 * S_P];
    const int z = blockIdx.x / p.max_chunks, chunk = blockIdx.x % p.max_chunks;
    int local;
    const SmallItem& it = find(p, z, local);
    if (chunk >= it.chunks) return;
    const bool tall = it.m > it.n;
    const int r = tall ? it.n : it.m, l = tall ? it.m : it.n, nt = (r + 15) / 16, R = 16 * nt;
    const Io io = shifted(it.io, (size_t)local * it.m * it.n, sizeof(T));
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i16 = lane & 15, q = lane >> 4;
    const double* src = p.ws + it.p + (size_t)local * 4096;
    for (int e = threadIdx.x; e < R * R; e += 256) P[e / R * S_P + e % R] = src[(e / R) * 64 + e % R];
    __syncthreads();
    const int c1 = min(l, (chunk + 1) * it.width);
    for (int c0 = chunk * it.width + 16 * wave; c0 < c1; c0 += 64) {
        const int col = c0 + i16;
        // the column's elements j = 16 t + 4 q + s for step (t, s)
        double u[4][4];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const int j = 16 * t + 4 * q + s;
                u[t][s] = j < r && col < c1
                              ? (double)read_u<T>(io, tall ? (size_t)col * it.n + j : (size_t)j * it.n + col, false)
                              : 0.0;
            }
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
                        // rows of the result: the short side, or the long one where it is the matrix's rows
                        acc = tall ? __builtin_amdgcn_mfma_f64_16x16x4f64(u[t][s], pv, acc, 0, 0, 0)
                                   : __builtin_amdgcn_mfma_f64_16x16x4f64(pv, u[t][s], acc, 0, 0, 0);
                    }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int rr = 4 * i + q;
                const int srt = 16 * a + (tall ? i16 : rr), lng = c0 + (tall ? rr : i16);
                if (srt < r && lng < c1)
                    write_o<T>(io, tall ? (size_t)lng * it.n + srt : (size_t)srt * it.n + lng, (float)acc[i]);
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------- r > 64
constexpr int TILE = 128, KS = 32;                // output tile, contraction per stage
constexpr int ROWB = 128;                         // bytes of a row's stage: 32 hi, 32 lo
constexpr int EP = TILE + 4;                      // pitch of the tile in LDS at the end
constexpr float SX = 16384.f, SA = 16384.f, SB = 8192.f;   // scales of X, A and q(A): elements under 1.21, 1.47, 3.45

struct Big {
    Io io;
    int m, n, r, l, R, L;                         // R, L: r and l rounded up to whole tiles
    int bytes;                                    // of an element
    float eps;
    double* part;                                 // [batch][NORM_BLOCKS] sums of squares
    char *x, *xt, *xt2, *a, *b;                   // packed matrices, one after the other for the batch
    float* slab;                                  // [batch][tiles][splits] partial tiles
    int splits;
};
constexpr int NORM_BLOCKS = 256;

template <typename T>
__global__ __launch_bounds__(256) void ns_norm_kernel(const Big p) {
    __shared__ double red[4];
    const size_t e = (size_t)p.m * p.n;
    const Io io = shifted(p.io, e * blockIdx.y, sizeof(T));
    double s = 0.0;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < e; i += (size_t)gridDim.x * 256) {
        const double v = (double)read_u<T>(io, i, true);
        s += v * v;
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

// X_0 scaled and packed, both ways: one 64 x 64 tile a block
template <typename T>
__global__ __launch_bounds__(256) void ns_pack_kernel(const Big p) {
    __shared__ float sm[64][65];
    __shared__ double red[4];
    const int tid = threadIdx.x, z = blockIdx.z;
    double s = p.part[(size_t)z * NORM_BLOCKS + tid];
    for (int o = 1; o < 64; o <<= 1) s += __shfl_xor(s, o, 64);
    if ((tid & 63) == 0) red[tid >> 6] = s;
    __syncthreads();
    const float scale = (float)((double)SX / (sqrt(red[0] + red[1] + red[2] + red[3]) + (double)p.eps));
    const Io io = shifted(p.io, (size_t)p.m * p.n * z, sizeof(T));
    const bool tall = p.m > p.n;
    const int i0 = blockIdx.y * 64, k0 = blockIdx.x * 64;                    // rows of the short side, columns of the long
    for (int e = tid; e < 4096; e += 256) {
        const int a = e >> 6, b = e & 63;
        const int i = i0 + (tall ? b : a), k = k0 + (tall ? a : b);
        const float v = i < p.r && k < p.l ? read_u<T>(io, tall ? (size_t)k * p.n + i : (size_t)i * p.n + k, false) * scale : 0.f;
        sm[i - i0][k - k0] = v;
    }
    __syncthreads();
    char* x = p.x + (size_t)z * p.R * p.L * 4;
    char* xt = p.xt + (size_t)z * p.R * p.L * 4;
    for (int u = tid; u < 512; u += 256) {
        float v[8];
        f16x8 hi, lo;
        const int a = u >> 3, b = (u & 7) * 8;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = sm[a][b + e];
        split8(v, hi, lo);
        char* d = packed(x, i0 + a, k0 + b, p.L);
        *(f16x8*)d = hi;
        *(f16x8*)(d + 64) = lo;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = sm[b + e][a];
        split8(v, hi, lo);
        d = packed(xt, k0 + a, i0 + b, p.R);
        *(f16x8*)d = hi;
        *(f16x8*)(d + 64) = lo;
    }
}

// a wave's 64 x 64 share of a tile: the products of the hi parts, and the two small terms in sums of their own, so that the
// large sum is rounded once per product and not three times
struct Acc {
    f32x16 v[2][2], w[2][2];
};

// acc += rows [i0, i0 + 128) of A times rows [j0, j0 + 128) of B over the stages [s0, s1): operands packed alike, K along
// both.  128 rows of a stage are 16 KiB, two stages in LDS; a row's eight 16-byte pieces lie in the order piece ^ (row & 7),
// so that eight neighbouring rows are read from different banks.
__device__ __forceinline__ void main_loop(Acc& acc, const char* A, const char* B, int K, int i0, int j0, int s0, int s1, char* lds) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l31 = lane & 31, q = lane >> 5;
    const int wi = (wave >> 1) * 64, wj = (wave & 1) * 64;
    const size_t pitch = (size_t)(K / KS) * ROWB;
    // a wave's load: 8 rows x 128 bytes; lane -> row lane / 8, piece (lane % 8) ^ row
    const int lrow = lane >> 3, piece = (lane & 7) ^ lrow;
    const char* src = (wave < 2 ? A + (size_t)(i0 + (wave & 1) * 64 + lrow) * pitch : B + (size_t)(j0 + (wave & 1) * 64 + lrow) * pitch) + piece * 16;
    auto issue = [&](int s, int buf) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(src + (size_t)s * ROWB + i * 8 * pitch),
                                             (__attribute__((address_space(3))) void*)(lds + buf * 32768 + wave * 8192 + i * 1024), 16, 0, 0);
    };
    issue(s0, 0);
    for (int s = s0; s < s1; ++s) {
        const int buf = (s - s0) & 1;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // this wave's share of the stage has arrived
        __syncthreads();                          // everybody's has, and the other stage is read
        if (s + 1 < s1) issue(s + 1, buf ^ 1);
        const char* la = lds + buf * 32768;
        const char* lb = la + 16384;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            f16x8 ah[2], al[2], bh[2], bl[2];
            const int ph = kk * 2 + q, pl = 4 + ph;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int ra = wi + 32 * t + l31, rb = wj + 32 * t + l31;
                ah[t] = *(const f16x8*)(la + ra * ROWB + ((ph ^ (ra & 7)) * 16));
                al[t] = *(const f16x8*)(la + ra * ROWB + ((pl ^ (ra & 7)) * 16));
                bh[t] = *(const f16x8*)(lb + rb * ROWB + ((ph ^ (rb & 7)) * 16));
                bl[t] = *(const f16x8*)(lb + rb * ROWB + ((pl ^ (rb & 7)) * 16));
            }
#pragma unroll
            for (int a = 0; a < 2; ++a)
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    acc.w[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(al[a], bh[b], acc.w[a][b], 0, 0, 0);
                    acc.v[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah[a], bh[b], acc.v[a][b], 0, 0, 0);
                    acc.w[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah[a], bl[b], acc.w[a][b], 0, 0, 0);
                }
        }
    }
    __syncthreads();
}

// the tile to LDS, times f
__device__ __forceinline__ void stage_tile(const Acc& acc, float f, float* sm) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l31 = lane & 31, q = lane >> 5;
    const int wi = (wave >> 1) * 64, wj = (wave & 1) * 64;
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int e = 0; e < 16; ++e)
                sm[(wi + 32 * a + 8 * (e >> 2) + 4 * q + (e & 3)) * EP + wj + 32 * b + l31] = (acc.v[a][b][e] + acc.w[a][b][e]) * f;
    __syncthreads();
}
// the tile in LDS packed to rows [i0, +128), columns [j0, +128) of `to` (K columns in all)
__device__ __forceinline__ void put_rows(const float* sm, char* to, int K, int i0, int j0) {
    for (int u = threadIdx.x; u < 2048; u += 256) {
        const int i = u >> 4, j = (u & 15) * 8;
        float v[8];
        f16x8 hi, lo;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = sm[i * EP + j + e];
        split8(v, hi, lo);
        char* d = packed(to, i0 + i, j0 + j, K);
        *(f16x8*)d = hi;
        *(f16x8*)(d + 64) = lo;
    }
}
// its transpose, rows [j0, +128), columns [i0, +128)
__device__ __forceinline__ void put_cols(const float* sm, char* to, int K, int i0, int j0) {
    for (int u = threadIdx.x; u < 2048; u += 256) {
        const int j = u >> 4, i = (u & 15) * 8;
        float v[8];
        f16x8 hi, lo;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = sm[(i + e) * EP + j];
        split8(v, hi, lo);
        char* d = packed(to, j0 + j, i0 + i, K);
        *(f16x8*)d = hi;
        *(f16x8*)(d + 64) = lo;
    }
}

// tile t of the upper triangle, counted column by column
__device__ __forceinline__ void tri(int t, int& i, int& j) {
    j = (int)((sqrtf(8.f * (float)t + 1.f) - 1.f) * 0.5f);
    while ((j + 1) * (j + 2) / 2 <= t) ++j;
    while (j * (j + 1) / 2 > t) --j;
    i = t - j * (j + 1) / 2;
}

__device__ __forceinline__ void gram_end(const Big& p, const Acc& acc, int i0, int j0, int z, float* sm) {
    char* a = p.a + (size_t)z * p.R * p.R * 4;
    stage_tile(acc, SA / (SX * SX), sm);
    put_rows(sm, a, p.R, i0, j0);
    if (i0 != j0) put_cols(sm, a, p.R, i0, j0);
}

__device__ __forceinline__ void zero(Acc& acc) {
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc.v[a][b][e] = acc.w[a][b][e] = 0.f;
}

// A = X X^T; with splits > 1 a share of the contraction, left in the slab
__global__ __launch_bounds__(256) void ns_xxt_kernel(const Big p) {
    __shared__ __attribute__((aligned(16))) float sm[TILE * EP];
    int ti, tj;
    tri(blockIdx.x, ti, tj);
    const int z = blockIdx.z, stages = p.L / KS, split = blockIdx.y;
    const int s0 = (int)((long long)stages * split / p.splits), s1 = (int)((long long)stages * (split + 1) / p.splits);
    const char* x = p.x + (size_t)z * p.R * p.L * 4;
    Acc acc;
    zero(acc);
    main_loop(acc, x, x, p.L, ti * TILE, tj * TILE, s0, s1, (char*)sm);
    if (p.splits == 1) {
        gram_end(p, acc, ti * TILE, tj * TILE, z, sm);
        return;
    }
    float* slab = p.slab + (((size_t)z * gridDim.x + blockIdx.x) * p.splits + split) * (TILE * TILE);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l31 = lane & 31, q = lane >> 5;
    const int wi = (wave >> 1) * 64, wj = (wave & 1) * 64;
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int e = 0; e < 16; ++e)
                slab[(wi + 32 * a + 8 * (e >> 2) + 4 * q + (e & 3)) * TILE + wj + 32 * b + l31] = acc.v[a][b][e] + acc.w[a][b][e];
}
// the shares of 16 rows of a tile, added in order
__global__ __launch_bounds__(256) void ns_join_kernel(const Big p) {
    __shared__ float sm[16][EP];
    int ti, tj;
    tri(blockIdx.x, ti, tj);
    const int z = blockIdx.z, row = threadIdx.x >> 4, col = (threadIdx.x & 15) * 8;
    const int i0 = ti * TILE + blockIdx.y * 16, j0 = tj * TILE;
    const float* slab = p.slab + ((size_t)z * gridDim.x + blockIdx.x) * p.splits * (TILE * TILE) + (blockIdx.y * 16 + row) * TILE + col;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < p.splits; ++s) {
        const Pack<float, 4> u = *(const Pack<float, 4>*)(slab + (size_t)s * TILE * TILE);
        const Pack<float, 4> w = *(const Pack<float, 4>*)(slab + (size_t)s * TILE * TILE + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[e] += u.v[e];
            v[4 + e] += w.v[e];
        }
    }
    char* a = p.a + (size_t)z * p.R * p.R * 4;
    f16x8 hi, lo;
#pragma unroll
    for (int e = 0; e < 8; ++e) sm[row][col + e] = v[e] *= SA / (SX * SX);
    split8(v, hi, lo);
    char* d = packed(a, i0 + row, j0 + col, p.R);
    *(f16x8*)d = hi;
    *(f16x8*)(d + 64) = lo;
    if (ti == tj) return;
    __syncthreads();
    const int c = threadIdx.x >> 1, k = (threadIdx.x & 1) * 8;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = sm[k + e][c];
    split8(v, hi, lo);
    d = packed(a, j0 + c, i0 + k, p.R);
    *(f16x8*)d = hi;
    *(f16x8*)(d + 64) = lo;
}

// q(A) = a I + b A + c A A
__global__ __launch_bounds__(256) void ns_poly_kernel(const Big p) {
    __shared__ __attribute__((aligned(16))) float sm[TILE * EP];
    int ti, tj;
    tri(blockIdx.x, ti, tj);
    const int z = blockIdx.z, i0 = ti * TILE, j0 = tj * TILE;
    char* a = p.a + (size_t)z * p.R * p.R * 4;
    char* b = p.b + (size_t)z * p.R * p.R * 4;
    Acc acc;
    zero(acc);
    main_loop(acc, a, a, p.R, i0, j0, 0, p.R / KS, (char*)sm);
    stage_tile(acc, (float)QC * SB / (SA * SA), sm);
    for (int u = threadIdx.x; u < 2048; u += 256) {
        const int i = u >> 4, j = (u & 15) * 8;
        const char* s = packed(a, i0 + i, j0 + j, p.R);
        const f16x8 hi = *(const f16x8*)s, lo = *(const f16x8*)(s + 64);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float v = sm[i * EP + j + e] + (float)QB * (SB / SA) * ((float)hi[e] + (float)lo[e]);
            if (i0 + i == j0 + j + e) v += (float)QA * SB;
            sm[i * EP + j + e] = v;
        }
    }
    __syncthreads();
    put_rows(sm, b, p.R, i0, j0);
    if (i0 != j0) put_cols(sm, b, p.R, i0, j0);
}

// X <- q(A) X: packed both ways, or the result
template <typename T>
__global__ __launch_bounds__(256) void ns_update_kernel(const Big p, int last) {
    __shared__ __attribute__((aligned(16))) float sm[TILE * EP];
    const int z = blockIdx.z, i0 = blockIdx.x * TILE, j0 = blockIdx.y * TILE;
    Acc acc;
    zero(acc);
    main_loop(acc, p.b + (size_t)z * p.R * p.R * 4, p.xt + (size_t)z * p.R * p.L * 4, p.R, i0, j0, 0, p.R / KS, (char*)sm);
    if (!last) {
        stage_tile(acc, SX / (SB * SX), sm);
        put_rows(sm, p.x + (size_t)z * p.R * p.L * 4, p.L, i0, j0);
        put_cols(sm, p.xt2 + (size_t)z * p.R * p.L * 4, p.R, i0, j0);
        return;
    }
    stage_tile(acc, 1.f / (SB * SX), sm);
    const Io io = shifted(p.io, (size_t)p.m * p.n * z, sizeof(T));
    const bool tall = p.m > p.n;
    for (int u = threadIdx.x; u < TILE * TILE; u += 256) {
        const int a = u >> 7, b = u & 127;
        const int i = tall ? b : a, j = tall ? a : b;
        if (i0 + i < p.r && j0 + j < p.l)
            write_o<T>(io, tall ? (size_t)(j0 + j) * p.n + i0 + i : (size_t)(i0 + i) * p.n + j0 + j, sm[i * EP + j]);
    }
}

// ---------------------------------------------------------------------------------------------- host
struct Layout {
    size_t part, x, xt, xt2, a, b, slab, total;
    int sub, splits;
};
int tiles_of(int R) { return R / TILE * (R / TILE + 1) / 2; }
// workspace of a stack of `batch` matrices with r > 64, `sub` of them at a time
Layout layout(int batch, int m, int n) {
    const int r = m < n ? m : n, l = m < n ? n : m;
    const size_t R = step::round_up(r, TILE), L = step::round_up(l, TILE);
    Layout o;
    const size_t most = (size_t)1 << 28;                           // elements of X at a time
    const size_t fit = most / (R * L) ? most / (R * L) : 1;
    o.sub = (int)(fit < (size_t)batch ? fit : (size_t)batch);
    if (o.sub > 1024) o.sub = 1024;
    // the contraction of X X^T is split where its tiles do not fill the card twice over, into parts of 8 stages at least
    const int tiles = tiles_of((int)R) * o.sub, stages = (int)(L / KS);
    o.splits = 512 / tiles;
    if (o.splits > stages / 8) o.splits = stages / 8;
    if (o.splits > 48) o.splits = 48;
    if (o.splits < 1) o.splits = 1;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    o.part = take((size_t)o.sub * NORM_BLOCKS * sizeof(double));
    o.x = take(o.sub * R * L * 4);
    o.xt = take(o.sub * R * L * 4);
    o.xt2 = take(o.sub * R * L * 4);
    o.a = take(o.sub * R * R * 4);
    o.b = take(o.sub * R * R * 4);
    o.slab = take(o.splits > 1 ? (size_t)tiles * o.splits * TILE * TILE * 4 : 0);
    o.total = at;
    return o;
}
bool small(int m, int n) { return (m < n ? m : n) <= 64; }

struct Group {
    int begin, end;                        // items (indices into the list of small ones)
    int total, max_chunks;
    size_t doubles;
};
// small items in groups of one launch each; the workspace is used again by every group
int small_groups(const step_ns_item* items, const std::vector<int>& idx, std::vector<Group>& groups, std::vector<SmallItem>& out) {
    for (size_t i = 0; i < idx.size();) {
        Group g{(int)i, (int)i, 0, 1, 0};
        int total = 0;
        size_t end = i;
        while (end < idx.size() && end - i < (size_t)S_ITEMS) total += items[idx[end++]].batch;
        const int share = total < 1024 ? 1024 / total : 1;
        int first = 0;
        size_t at = 0;
        for (; i < end; ++i) {
            const step_ns_item& it = items[idx[i]];
            const int l = it.m > it.n ? it.m : it.n;
            int chunks = step::ceil_div(l, 64);
            if (chunks > share) chunks = share;
            if (chunks > 32) chunks = 32;
            SmallItem s{};
            s.m = it.m;
            s.n = it.n;
            s.first = first;
            s.width = step::round_up(step::ceil_div(l, chunks), 64);
            s.chunks = step::ceil_div(l, s.width);
            s.slab = at;
            at += (size_t)it.batch * s.chunks * 2560;
            s.p = at;
            at += (size_t)it.batch * 4096;
            first += it.batch;
            if (s.chunks > g.max_chunks) g.max_chunks = s.chunks;
            out.push_back(s);
        }
        g.end = (int)end;
        g.total = first;
        g.doubles = at;
        groups.push_back(g);
    }
    return 0;
}

int check(const step_ns_item* items, int count) {
    STEP_REQUIRE(items && count >= 1, "step_newton_schulz: no matrices");
    long long total = 0;
    for (int i = 0; i < count; ++i) {
        const step_ns_item& it = items[i];
        STEP_REQUIRE(it.batch >= 1 && it.m >= 1 && it.n >= 1, "step_newton_schulz: item %d: bad shape %d x %d x %d", i, it.batch, it.m, it.n);
        STEP_REQUIRE(it.m <= (1 << 22) && it.n <= (1 << 22), "step_newton_schulz: item %d: %d x %d is over 2^22 a side", i, it.m, it.n);
        STEP_REQUIRE((it.m < it.n ? it.m : it.n) <= 32768, "step_newton_schulz: item %d: %d x %d is over 32768 on both sides", i, it.m, it.n);
        total += it.batch;
    }
    STEP_REQUIRE(total <= 1 << 24, "step_newton_schulz: %lld matrices", total);
    return STEP_OK;
}

template <typename T>
int run(const step_ns_item* items, int count, int steps, float eps, float mu, int nesterov, float lr, float decay, void* ws, hipStream_t st) {
    std::vector<int> idx;
    auto io_of = [&](const step_ns_item& it) {
        return Io{it.g, it.out, it.momentum, it.param, mu, 1.f - lr * decay, lr * it.scale, nesterov};
    };
    for (int i = 0; i < count; ++i)
        if (small(items[i].m, items[i].n)) idx.push_back(i);
    if (!idx.empty()) {
        std::vector<Group> groups;
        std::vector<SmallItem> sm;
        small_groups(items, idx, groups, sm);
        constexpr size_t lds = 4 * 64 * S_P * sizeof(double);
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(ns_small_kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) {
            step::set_error("step_newton_schulz: hipFuncSetAttribute(%zu): %s", lds, hipGetErrorString(e));
            return STEP_ERR_LAUNCH;
        }
        for (const Group& g : groups) {
            SmallArgs a{};
            a.items = g.end - g.begin;
            a.total = g.total;
            a.steps = steps;
            a.max_chunks = g.max_chunks;
            a.eps = eps;
            a.ws = (double*)ws;
            for (int i = 0; i < a.items; ++i) {
                a.item[i] = sm[g.begin + i];
                a.item[i].io = io_of(items[idx[g.begin + i]]);
            }
            hipLaunchKernelGGL(ns_gram_kernel<T>, dim3((unsigned)g.total * g.max_chunks), dim3(256), 0, st, a);
            hipLaunchKernelGGL(ns_small_kernel, dim3((unsigned)g.total), dim3(512), lds, st, a);
            hipLaunchKernelGGL(ns_apply_kernel<T>, dim3((unsigned)g.total * g.max_chunks), dim3(256), 0, st, a);
        }
    }
    for (int i = 0; i < count; ++i) {
        const step_ns_item& it = items[i];
        if (small(it.m, it.n)) continue;
        const Layout o = layout(it.batch, it.m, it.n);
        Big p{};
        p.m = it.m;
        p.n = it.n;
        p.r = it.m < it.n ? it.m : it.n;
        p.l = it.m < it.n ? it.n : it.m;
        p.R = step::round_up(p.r, TILE);
        p.L = step::round_up(p.l, TILE);
        p.eps = eps;
        p.splits = o.splits;
        char* base = (char*)ws;
        p.part = (double*)(base + o.part);
        p.slab = (float*)(base + o.slab);
        const int tiles = tiles_of(p.R);
        for (int b0 = 0; b0 < it.batch; b0 += o.sub) {
            const unsigned nb = (unsigned)(it.batch - b0 < o.sub ? it.batch - b0 : o.sub);
            const size_t by = (size_t)b0 * it.m * it.n;
            p.io = io_of(it);
            p.io.g = (const T*)p.io.g + by;
            if (p.io.out) p.io.out = (T*)p.io.out + by;
            if (p.io.momentum) p.io.momentum += by;
            if (p.io.param) p.io.param += by;
            p.x = base + o.x;
            p.xt = base + o.xt;
            p.xt2 = base + o.xt2;
            p.a = base + o.a;
            p.b = base + o.b;
            hipLaunchKernelGGL(ns_norm_kernel<T>, dim3(NORM_BLOCKS, nb), dim3(256), 0, st, p);
            hipLaunchKernelGGL(ns_pack_kernel<T>, dim3(p.L / 64, p.R / 64, nb), dim3(256), 0, st, p);
            for (int s = 0; s < steps; ++s) {
                hipLaunchKernelGGL(ns_xxt_kernel, dim3(tiles, p.splits, nb), dim3(256), 0, st, p);
                if (p.splits > 1) hipLaunchKernelGGL(ns_join_kernel, dim3(tiles, TILE / 16, nb), dim3(256), 0, st, p);
                hipLaunchKernelGGL(ns_poly_kernel, dim3(tiles, 1, nb), dim3(256), 0, st, p);
                hipLaunchKernelGGL(ns_update_kernel<T>, dim3(p.R / TILE, p.L / TILE, nb), dim3(256), 0, st, p, (int)(s + 1 == steps));
                char* t = p.xt;
                p.xt = p.xt2;
                p.xt2 = t;
            }
        }
    }
    return step::check_launch("step_newton_schulz");
}

}  // namespace

extern "C" size_t step_newton_schulz_ws_bytes(const step_ns_item* items, int count) {
    if (check(items, count) != STEP_OK) return 0;
    try {
        std::vector<int> idx;
        size_t most = 256;
        for (int i = 0; i < count; ++i) {
            if (small(items[i].m, items[i].n)) {
                idx.push_back(i);
                continue;
            }
            const size_t b = layout(items[i].batch, items[i].m, items[i].n).total;
            if (b > most) most = b;
        }
        std::vector<Group> groups;
        std::vector<SmallItem> sm;
        small_groups(items, idx, groups, sm);
        for (const Group& g : groups)
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
