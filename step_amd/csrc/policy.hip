// Clipped policy loss with a KL term, value and gradient in one pass over the logits (rows, classes).
//
//   lp = z[a] - log SUM exp z,  rho = exp(lp - old),  o1 = rho A,  o2 = min(max(rho, 1 - cl), 1 + ch) A
//   L = -min(o1, o2),  kl = exp(ref - lp) - (ref - lp) - 1 >= 0
//   loss = SUM_live (L + beta kl) / max(#live, 1)
//   dL/dlp = [o1 <= o2] (-o1) + beta (1 - exp(ref - lp)),  dz = dL/dlp / max(#live, 1) * (onehot(a) - softmax z)
//
// Memory-bound: the least is one read of the live rows' logits and one write of the gradient.  A row stays in the
// registers of the G threads that share it between its softmax sums and its gradient (up to 128 K classes in 16 bits,
// 64 K in fp32; 8192 x 32000 bf16 with 0.8 of the rows live: 200 us, 4.7 TB/s; 16384 x 8000 fp32: 209 us, 5.0 TB/s); longer
// rows are read twice.  The number of live rows, which every row's gradient is divided by, is
// counted by a launch before.  A row's few scalars are taken in fp64: its ratio may lie next to the border of the
// clipping.  Per-block fp64 sums are added in block order by the last launch: the same bits every time, no atomics.
// A masked row is not read at all (its logits, and its action, may be anything): log probability 0, gradient 0.
#include "rows.h"

namespace {
using namespace step;

constexpr float L2E = 1.4426950408889634f, L2E_REST = 1.92596299e-8f;
constexpr double LN2 = 0.69314718055994530942;
constexpr float LN2_HI = 0.6931471824645996f;            // ln 2 in fp32, and what is left
constexpr double LN2_LO = -1.904654299957768e-09;
constexpr int MAX_BLOCKS = 2048;


struct Args {
    const void* logits;
    const long long* actions;
    const float *old_logp, *adv, *ref;
    const unsigned char* mask;
    void* dlogits;
    float* logp;
    const double* count;           // device: number of live rows (NULL: all of them)
    double* part;                  // [blocks][3]
    const float* upstream;         // NULL: the loss itself; else only dlogits, times *upstream
    int skip_one;                  // with upstream: nothing to do where it is exactly 1, and count and a long row's sums are there
    long long rows;
    int classes;
    double clip_low, clip_high, beta;   // a clipped ratio's 1.2 in fp32 is off by 4e-8, the same way in every row
};

// maximum and sum of exponentials about it, joined over the G threads of a row.  The maximum is taken off before the multiplication
// by log2 e: the type's lowest values, as masks write them, times log2 e would overflow.
struct Soft {
    float m, s;
};
// the same of many threads: what the rounding of one addition costs them all is not averaged out, so it takes fp64
struct Row {
    float m;
    double s;
};
// e^(x - m) scale, an element of the gradient.  fp32: the product with log2 e is rounded at its own size, 2^-19 for a probability of
// e^-23, and what that is off by, d - y ln 2, is put right in the first order.  16 bits, whose rounding is far above that, do without.
template <typename T>
__device__ __forceinline__ float exp_scaled(T x, float m, float scale) {
    if constexpr (sizeof(T) < 4) return __builtin_amdgcn_exp2f(((float)x - m) * L2E) * scale;
    const float d = fmaxf(x - m, -1000.f), y = d * L2E;      // (no -inf + inf; a row with a NaN has a NaN as its scale)
    const float g = __builtin_amdgcn_exp2f(y) * scale;
    return __builtin_fmaf(g, __builtin_fmaf(y, -LN2_HI, d), g);
}
// for the sum, whose logarithm the loss hangs on: the product with log2 e to 48 bits, rounded once (fp32's log2 e alone is off by
// 1.3e-8, the same way for all elements: log probabilities 3.5e-8 too low on average over 613 classes)
__device__ __forceinline__ float exp_for_sum(float x, float m) {
    const float d = x - m;
    return __builtin_amdgcn_exp2f(__builtin_fmaf(d, L2E, d * L2E_REST));
}
__device__ __forceinline__ float finite_or_0(float m) { return m == -__builtin_inff() ? 0.f : m; }   // no -inf - -inf

template <int CTRL>
__device__ __forceinline__ double dpp64(double v) {
    const u32x2 q = __builtin_bit_cast(u32x2, v);
    u32x2 r;
    r[0] = (unsigned)__builtin_amdgcn_mov_dpp((int)q[0], CTRL, 0xf, 0xf, true);
    r[1] = (unsigned)__builtin_amdgcn_mov_dpp((int)q[1], CTRL, 0xf, 0xf, true);
    return __builtin_bit_cast(double, r);
}
__device__ __forceinline__ double lane64(double v, int lane) {
    const u32x2 q = __builtin_bit_cast(u32x2, v);
    u32x2 r;
    r[0] = (unsigned)__builtin_amdgcn_readlane((int)q[0], lane);
    r[1] = (unsigned)__builtin_amdgcn_readlane((int)q[1], lane);
    return __builtin_bit_cast(double, r);
}
template <int G>
__device__ __forceinline__ double wave_sum64(double v) {       // (wave_reduce's steps)
    v += dpp64<0xb1>(v);
    v += dpp64<0x4e>(v);
    v += dpp64<0x141>(v);
    if constexpr (G >= 16) v += dpp64<0x140>(v);
    if constexpr (G >= 64) v = (lane64(v, 0) + lane64(v, 16)) + (lane64(v, 32) + lane64(v, 48));
    return v;
}
// over the G threads that have the maximum and sum of their elements, the same bits in all of them
template <int G>
__device__ __forceinline__ Row reduce(float m, double s, Row* sm) {
    constexpr int W = G < 64 ? G : 64;
    Row w;
    w.m = wave_reduce<W>(m, [](float a, float b) { return fmaxf(a, b); });
    w.s = wave_sum64<W>(s * exp_for_sum(m, finite_or_0(w.m)));
    if constexpr (G > 64) {
        if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = w;
        __syncthreads();
        w = sm[0];
#pragma unroll
        for (int i = 1; i < G / 64; ++i) w.m = fmaxf(w.m, sm[i].m);
        const float m0 = finite_or_0(w.m);
        w.s = 0.0;
#pragma unroll
        for (int i = 0; i < G / 64; ++i) w.s += sm[i].s * exp_for_sum(sm[i].m, m0);
    }
    return w;
}

// exp and log2 in fp64 for a row's scalars, from their series: a third of the registers and of the time that the general
// functions take, which one thread of a block spends while the others wait.
// log2 s = e + log2 m, s = m 2^e with m in [sqrt 1/2, sqrt 2): log m = 2 atanh t, t = (m - 1) / (m + 1), |t| <= 0.172, to t^13:
// the rest is under 2 t^15 / 15 = 5e-13.  (s is 1 or more, or NaN, or comes from a row that allows nothing, where m is -inf.)
__device__ __forceinline__ double log2_of(double s) {
    int e = __builtin_amdgcn_frexp_exp(s);
    double m = __builtin_amdgcn_frexp_mant(s);
    if (m < 0.70710678) {
        m *= 2.0;
        --e;
    }
    const double d = m + 1.0;
    double r = __builtin_amdgcn_rcp(d);
    r = r * (2.0 - d * r);
    r = r * (2.0 - d * r);
    const double t = (m - 1.0) * r, u = t * t;
    const double a = 1.0 + u * (1.0 / 3 + u * (1.0 / 5 + u * (1.0 / 7 + u * (1.0 / 9 + u * (1.0 / 11 + u * (1.0 / 13))))));
    return (double)e + (2.0 / LN2) * (t * a);
}
// e^x = 2^n e^r, |r| <= ln 2 / 2, to r^10: the rest is under 0.347^11 / 11! = 3e-13; beyond e^+-700 infinity and 0, NaN stays
__device__ __forceinline__ double exp_of64(double x) {
    if (!(x < 700.0)) return x == x ? (double)__builtin_inff() : x;
    if (x < -700.0) return 0.0;
    const double n = __builtin_rint(x * (1.0 / LN2));
    const double r = __builtin_fma(n, -(LN2_LO), __builtin_fma(n, -(double)LN2_HI, x));   // n LN2_HI is exact
    double p = 1.0 / 3628800;
    p = p * r + 1.0 / 362880;
    p = p * r + 1.0 / 40320;
    p = p * r + 1.0 / 5040;
    p = p * r + 1.0 / 720;
    p = p * r + 1.0 / 120;
    p = p * r + 1.0 / 24;
    p = p * r + 1.0 / 6;
    p = p * r + 0.5;
    p = p * r + 1.0;
    p = p * r + 1.0;
    return __builtin_ldexp(p, (int)n);
}

// the row's scalars: returns dL/dlp / count (times the upstream gradient), adds the row to the block's sums
__device__ __forceinline__ float row_scalars(const Args& p, long long row, const Row& f, float za, bool valid, double count,
                                             double* sums, bool write = true) {
    const double lp = valid ? (double)za - (double)f.m - log2_of(f.s) * LN2 : (double)__builtin_nanf("");
    const double a = p.adv[row], ratio = exp_of64(lp - (double)p.old_logp[row]);
    const double lo = 1.0 - p.clip_low, hi = 1.0 + p.clip_high;
    const double o1 = ratio * a, o2 = (ratio > hi ? hi : ratio < lo ? lo : ratio) * a;   // a NaN stays one
    const bool clipped = o1 > o2;
    double slope = clipped ? 0.0 : -o1, kl = 0.0;
    if (p.ref) {
        const double d = (double)p.ref[row] - lp, e = exp_of64(d);
        kl = e - d - 1.0;
        slope += p.beta * (1.0 - e);
    }
    sums[0] += clipped ? -o2 : -o1;
    sums[1] += kl;
    sums[2] += clipped ? 1.0 : 0.0;
    if (p.upstream) slope *= (double)*p.upstream;
    else if (write) p.logp[row] = (float)lp;
    return (float)(slope / count);
}

// -coef softmax(z) for the elements of a pack; the drawn action's + coef comes afterwards
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> gradient_of(const Pack<T, N>& z, float m, float scale) {
    Pack<T, N> g;
#pragma unroll
    for (int e = 0; e < N; ++e) g.v[e] = (T)exp_scaled(z.v[e], m, scale);       // the gradient's only rounding to fewer bits
    return g;
}
// adds N elements to a thread's maximum and sum: their largest first, so that nothing overflows
template <typename T, int N>
__device__ __forceinline__ void add_to(Soft& f, const Pack<T, N>* q, int packs) {
    float m = -__builtin_inff();
#pragma unroll
    for (int k = 0; k < packs; ++k)
#pragma unroll
        for (int e = 0; e < N; ++e) m = fmaxf(m, (float)q[k].v[e]);
    m = fmaxf(f.m, m);
    const float m0 = finite_or_0(m);
    float s0 = f.s * exp_for_sum(f.m, m0), s1 = 0.f;             // two chains
#pragma unroll
    for (int k = 0; k < packs; ++k)
#pragma unroll
        for (int e = 0; e < N; e += 2) {
            s0 += exp_for_sum((float)q[k].v[e], m0);
            if (e + 1 < N) s1 += exp_for_sum((float)q[k].v[e + 1], m0);
        }
    f.s = s0 + s1;
    f.m = m;
}

// sums of one block -> part[block]; the threads that hold none pass zeros
template <int BLOCK>
__device__ __forceinline__ void block_sums(double* part, double* sums) {
    __shared__ double red[3][BLOCK / 64];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        double v = sums[k];
        for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o, 64);
        if ((threadIdx.x & 63) == 0) red[k][threadIdx.x >> 6] = v;
    }
    __syncthreads();
    if (threadIdx.x < 3) {
        double v = 0.0;
        for (int i = 0; i < BLOCK / 64; ++i) v += red[threadIdx.x][i];
        part[3 * blockIdx.x + threadIdx.x] = v;
    }
}

// what was computed from a pack is computed again behind this: a row's elements stay in registers as they are, and not as
// floats beside
template <typename T, int N>
__device__ __forceinline__ void forget(Pack<T, N>& v) {
    if constexpr (sizeof(T) < 4 && sizeof(v) == 16) {
        u32x4 q = __builtin_bit_cast(u32x4, v);
        asm volatile("" : "+v"(q));
        v = __builtin_bit_cast(Pack<T, N>, q);
    }
}

template <typename T, int N, int NV>
__device__ __forceinline__ void add_packs(Soft& f, Pack<T, N>* v) {
    constexpr int U = N == 4 && NV % 2 == 0 ? 2 : 1;         // eight elements at a time
#pragma unroll
    for (int i = 0; i < NV; i += U) {
        add_to<T, N>(f, v + i, U);
#pragma unroll
        for (int k = 0; k < U; ++k) forget(v[i + k]);
    }
}
// G threads a row, NV packs of N elements a thread (the last LAST of them may not fit)
template <typename T, int N, int NV, int LAST, int G>
__global__ __launch_bounds__(G < 256 ? 256 : G, G == 1024 ? 4 : 3) void policy_kernel(const Args p) {
    constexpr int BLOCK = G < 256 ? 256 : G, RPB = BLOCK / G;
    __shared__ Row sm[2][G > 64 ? G / 64 : 1];
    __shared__ float coef_s;
    if (p.upstream && p.skip_one && *p.upstream == 1.f) return;
    const int lane = threadIdx.x % G;
    const Columns<N, NV, G, LAST> own{p.classes, lane};
    const double live_rows = p.count ? *p.count : (double)p.rows, count = live_rows > 1.0 ? live_rows : 1.0;
    double sums[3] = {0.0, 0.0, 0.0};
    int turn = 0;
    for (long long r0 = (long long)blockIdx.x * RPB; r0 < p.rows; r0 += (long long)gridDim.x * RPB) {
        const long long row = r0 + threadIdx.x / G;
        if (G <= 64 && row >= p.rows) continue;              // (whole blocks share a row otherwise)
        const T* z = (const T*)p.logits + (size_t)row * p.classes;
        T* g = p.dlogits ? (T*)p.dlogits + (size_t)row * p.classes : nullptr;
        if (p.mask && !p.mask[row]) {
            if (lane == 0 && !p.upstream) p.logp[row] = 0.f;
            if (g) {
                Pack<T, N> zero;
#pragma unroll
                for (int e = 0; e < N; ++e) zero.v[e] = (T)0.f;
                for (int c = lane * N; c < p.classes; c += G * N) store_pack<T, N>(g + (c < p.classes - N ? c : p.classes - N), zero);
            }
            continue;
        }
        const long long a64 = p.actions[row];
        const bool valid = a64 >= 0 && a64 < p.classes;
        const int action = valid ? (int)a64 : -1;
        Pack<T, N> v[NV];
        Soft f{-__builtin_inff(), 0.f};
        own.load(v, z);
        const float za = lane == 0 && valid ? (float)z[action] : 0.f;
        own.fill(v, (T)-__builtin_inff());
        add_packs<T, N, NV>(f, v);
        const Row w = reduce<G>(f.m, (double)f.s, sm[turn]);
        turn ^= 1;
        float coef;
        if constexpr (G <= 64) {
            double add[3] = {0.0, 0.0, 0.0};
            coef = row_scalars(p, row, w, __shfl(za, (threadIdx.x & 63) & ~(G - 1), 64), valid, count, add);
            if (lane == 0)
                for (int k = 0; k < 3; ++k) sums[k] += add[k];
        } else {
            if (threadIdx.x == 0) coef_s = row_scalars(p, row, w, za, valid, count, sums);
            __syncthreads();
            coef = coef_s;
        }
        if (!g) continue;
        const float scale = -coef / (float)w.s;
#pragma unroll
        for (int i = 0; i < NV; ++i) own.store(g, i, gradient_of<T, N>(v[i], w.m, scale));
        // the thread that wrote the action's element writes it once more
        if (valid && lane == action / N % G) g[action] = (T)(exp_scaled(z[action], w.m, scale) + coef);
    }
    if (!p.upstream) block_sums<BLOCK>(p.part, sums);
}

// Rows too long for the registers of 1024 threads, in parts of at most PART_PACKS packs a thread: first each part's maximum and
// sum, then, from the row's parts together, its scalars and the part's gradient - the row is read twice.  The parts fill the
// card where there are few rows (640 x 140001 bf16: 120 us, 145 with a block of 1024 threads a row;
// 2000 x 100000 fp32: 465 us, 5.2 TB/s of what it reads and writes; 4 or 16 packs: within 4 % either way).
constexpr int PART_PACKS = 8;
template <typename T, int N, bool GRAD>
__global__ __launch_bounds__(256) void policy_parts_kernel(const Args p, Row* soft, int parts, int span) {
    __shared__ Row sm[2][4];
    __shared__ float coef_s[2];
    if (p.upstream && p.skip_one && *p.upstream == 1.f) return;
    const int tid = threadIdx.x;
    const double live_rows = p.count ? *p.count : (double)p.rows, count = live_rows > 1.0 ? live_rows : 1.0;
    double sums[3] = {0.0, 0.0, 0.0};
    int turn = 0;
    for (long long item = blockIdx.x; item < p.rows * parts; item += gridDim.x) {
        const long long row = item / parts;
        const int part = (int)(item - row * parts), c0 = part * span;
        const Columns<N, PART_PACKS, 256, PART_PACKS> own{span < p.classes - c0 ? span : p.classes - c0, tid};
        const T* z = (const T*)p.logits + (size_t)row * p.classes;
        T* g = GRAD && p.dlogits ? (T*)p.dlogits + (size_t)row * p.classes : nullptr;
        if (GRAD && !g && part) continue;                    // only the row's scalars are asked for
        if (p.mask && !p.mask[row]) {
            if (GRAD && part == 0 && tid == 0 && !p.upstream) p.logp[row] = 0.f;
            if (g) {
                Pack<T, N> zero;
#pragma unroll
                for (int e = 0; e < N; ++e) zero.v[e] = (T)0.f;
#pragma unroll
                for (int i = 0; i < PART_PACKS; ++i) own.store(g + c0, i, zero);
            }
            continue;
        }
        Pack<T, N> v[PART_PACKS];
        if (!GRAD || g) own.load(v, z + c0);                 // (a pack at the end of a short last part lies in the part before)
        if constexpr (!GRAD) {
            Soft t{-__builtin_inff(), 0.f};
            own.fill(v, (T)-__builtin_inff());
            add_packs<T, N, PART_PACKS>(t, v);
            const Row f = reduce<256>(t.m, (double)t.s, sm[turn]);
            turn ^= 1;
            if (tid == 0) soft[item] = f;
        } else {
            const long long a64 = p.actions[row];
            const bool valid = a64 >= 0 && a64 < p.classes;
            const float za = tid == 0 && valid ? (float)z[a64] : 0.f;
            Row f{-__builtin_inff(), 0.0};
            for (int i = tid; i < parts; i += 256) {
                const Row o = soft[row * parts + i];
                const float m = fmaxf(f.m, o.m), m0 = finite_or_0(m);
                f.s = f.s * exp_for_sum(f.m, m0) + o.s * exp_for_sum(o.m, m0);
                f.m = m;
            }
            f = reduce<256>(f.m, f.s, sm[turn]);
            if (tid == 0) {
                double add[3] = {0.0, 0.0, 0.0};
                coef_s[turn] = row_scalars(p, row, f, za, valid, count, add, part == 0);
                if (part == 0)
                    for (int k = 0; k < 3; ++k) sums[k] += add[k];
            }
            __syncthreads();
            const float coef = coef_s[turn];
            turn ^= 1;
            if (!g) continue;
            const float scale = -coef / (float)f.s;
#pragma unroll
            for (int i = 0; i < PART_PACKS; ++i) own.store(g + c0, i, gradient_of<T, N>(v[i], f.m, scale));
            // the thread that wrote the action's element writes it once more
            const long long at = a64 - c0;
            if (valid && at >= 0 && at < own.cols && tid == (int)at / N % 256) g[a64] = (T)(exp_scaled(z[a64], f.m, scale) + coef);
        }
    }
    if (GRAD && !p.upstream) block_sums<256>(p.part, sums);
}

__global__ __launch_bounds__(1024) void policy_count_kernel(const unsigned char* __restrict__ mask, double* count,
                                                            long long rows) {
    __shared__ long long red[16];
    long long n = 0;
    const long long head = ((16 - ((uintptr_t)mask & 15)) & 15) < (unsigned long long)rows ? (16 - ((uintptr_t)mask & 15)) & 15 : rows;
    const long long packs = (rows - head) / 16;
    for (long long i = threadIdx.x; i < packs; i += 1024) {
        const Pack<unsigned char, 16> q = *(const Pack<unsigned char, 16>*)(mask + head + 16 * i);
#pragma unroll
        for (int e = 0; e < 16; ++e) n += q.v[e] != 0;
    }
    if (threadIdx.x < head) n += mask[threadIdx.x] != 0;
    for (long long i = head + 16 * packs + threadIdx.x; i < rows; i += 1024) n += mask[i] != 0;
    for (int o = 1; o < 64; o <<= 1) n += __shfl_xor(n, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = n;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < 16; ++i) n += red[i];
        *count = (double)n;
    }
}

__global__ __launch_bounds__(256) void policy_finish_kernel(const double* __restrict__ part, const double* count,
                                                            double rows, int blocks, double beta, float* loss,
                                                            float* stats) {
    __shared__ double red[3][4];
    double s[3] = {0.0, 0.0, 0.0};
    for (int b = threadIdx.x; b < blocks; b += 256)
        for (int k = 0; k < 3; ++k) s[k] += part[3 * b + k];
    for (int k = 0; k < 3; ++k) {
        for (int o = 1; o < 64; o <<= 1) s[k] += __shfl_xor(s[k], o, 64);
        if ((threadIdx.x & 63) == 0) red[k][threadIdx.x >> 6] = s[k];
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        double n = count ? *count : rows;
        n = n > 1.0 ? n : 1.0;
        double mean[3];
        for (int k = 0; k < 3; ++k) {
            mean[k] = (red[k][0] + red[k][1] + red[k][2] + red[k][3]) / n;
            stats[k] = (float)mean[k];
        }
        *loss = (float)(mean[0] + beta * mean[1]);
    }
}

struct Plan {
    int g, nv, vec;                                          // g 0: too long for the registers of 1024 threads
};
// The fewest threads whose registers hold the row: few waves wait for each other, more rows are in a CU at a time, and the rows
// of a wave share the time of their scalars (65536 x 1000 bf16: 53 us with 16 threads a row, 71 with a wave).  Rows shorter than a pack are read by
// elements.
Plan plan(int classes, int dtype) {
    const int n = 16 / elem_bytes(dtype);
    if (classes < n) return Plan{8, 1, 1};
    const int packs = (classes - 1) / n + 1;
    for (int g : {8, 16, 64, 256, 512, 1024})
        if (packs <= (g < 64 ? 8 : 16) * g) {
            const int nv = (packs + g - 1) / g;
            return Plan{g, nv <= 4 ? nv : (nv + 1) / 2 * 2, n};
        }
    return Plan{0, 0, n};
}
// parts of a long row, and columns of a part (whole packs)
int parts_of(int classes, int vec, int& span) {
    const int packs = (classes - 1) / vec + 1, parts = (packs - 1) / (256 * PART_PACKS) + 1;
    span = ((packs - 1) / parts + 1) * vec;
    return (classes - 1) / span + 1;
}
int blocks_of(long long rows, const Plan& p) {
    const int rpb = p.g < 256 ? 256 / p.g : 1, cap = p.g == 1024 ? 512 : p.g == 512 ? 1024 : MAX_BLOCKS;
    const long long need = (rows + rpb - 1) / rpb;
    return (int)(need < cap ? need : cap);
}

template <typename T, int N, int G, int NV, int MOST>
void launch_nv(int nv, int blocks, const Args& a, hipStream_t st) {
    if (nv == NV) hipLaunchKernelGGL((policy_kernel<T, N, NV, NV <= 4 ? 1 : 2, G>), dim3(blocks), dim3(G < 256 ? 256 : G), 0, st, a);
    else if constexpr (NV < MOST) launch_nv<T, N, G, NV < 4 ? NV + 1 : NV + 2, MOST>(nv, blocks, a, st);
}
template <typename T>
void launch(const Plan& pl, int blocks, const Args& a, hipStream_t st) {
    constexpr int N = 16 / (int)sizeof(T);
    if (pl.vec == 1) launch_nv<T, 1, 8, 1, 1>(1, blocks, a, st);
    else if (pl.g == 8) launch_nv<T, N, 8, 1, 8>(pl.nv, blocks, a, st);
    else if (pl.g == 16) launch_nv<T, N, 16, 6, 8>(pl.nv, blocks, a, st);      // fewer fit in 8 threads, and so on
    else if (pl.g == 64) launch_nv<T, N, 64, 3, 16>(pl.nv, blocks, a, st);
    else if (pl.g == 256) launch_nv<T, N, 256, 6, 16>(pl.nv, blocks, a, st);
    else if (pl.g == 512) launch_nv<T, N, 512, 10, 16>(pl.nv, blocks, a, st);
    else launch_nv<T, N, 1024, 10, 16>(pl.nv, blocks, a, st);
}
template <typename T>
void launch_parts(int parts, int span, int blocks, const Args& a, Row* soft, hipStream_t st) {
    constexpr int N = 16 / (int)sizeof(T);
    if (!a.skip_one) hipLaunchKernelGGL((policy_parts_kernel<T, N, false>), dim3(blocks), dim3(256), 0, st, a, soft, parts, span);
    hipLaunchKernelGGL((policy_parts_kernel<T, N, true>), dim3(blocks), dim3(256), 0, st, a, soft, parts, span);
}

}  // namespace

extern "C" size_t step_policy_loss_ws_bytes(long long rows, int classes) {
    if (rows <= 0 || classes <= 0 || classes > 1 << 30) return 0;
    int span;                                                // (fp32's parts: a 16-bit type has fewer)
    const size_t soft = plan(classes, STEP_F32).g ? 0 : (size_t)rows * parts_of(classes, 4, span) * sizeof(Row);
    return (1 + 3 * (size_t)MAX_BLOCKS) * sizeof(double) + soft;
}

extern "C" int step_policy_loss(const void* logits, const long long* actions, const float* old_logp,
                                const float* advantages, const float* ref_logp, const unsigned char* mask,
                                double clip_low, double clip_high, double beta, const float* upstream, int skip_one,
                                float* loss, float* stats, float* logp, void* dlogits, long long rows, int classes,
                                int dtype, void* ws, size_t ws_bytes, void* stream) {
    STEP_REQUIRE(logits && actions && old_logp && advantages && ws, "step_policy_loss: null pointer");
    STEP_REQUIRE(rows >= 1 && classes >= 1 && classes <= 1 << 30, "step_policy_loss: bad shape rows=%lld classes=%d", rows, classes);
    STEP_REQUIRE(elem_bytes(dtype), "step_policy_loss: unknown type %d", dtype);
    STEP_REQUIRE(upstream ? dlogits != nullptr : loss && stats && logp, "step_policy_loss: null output");
    STEP_REQUIRE((((uintptr_t)logits | (uintptr_t)dlogits) & (elem_bytes(dtype) - 1)) == 0, "step_policy_loss: logits or dlogits lie across elements");
    if (ws_bytes < step_policy_loss_ws_bytes(rows, classes)) {
        step::set_error("step_policy_loss: workspace %zu < %zu bytes", ws_bytes, step_policy_loss_ws_bytes(rows, classes));
        return STEP_ERR_WORKSPACE;
    }
    hipStream_t st = (hipStream_t)stream;
    double* count = (double*)ws;
    double* part = count + 1;
    const Plan pl = plan(classes, dtype);
    int blocks, parts = 0, span = 0;
    if (pl.g) {
        blocks = blocks_of(rows, pl);
    } else {
        parts = parts_of(classes, pl.vec, span);
        blocks = rows * parts < MAX_BLOCKS ? (int)(rows * parts) : MAX_BLOCKS;
    }
    if (!upstream) skip_one = 0;
    if (mask && !skip_one) hipLaunchKernelGGL(policy_count_kernel, dim3(1), dim3(1024), 0, st, mask, count, rows);
    const Args a{logits, actions, old_logp, advantages, ref_logp, mask, dlogits, logp, mask ? count : nullptr, part,
                 upstream, skip_one, rows, classes, clip_low, clip_high, beta};
    auto go = [&](auto t) {
        using T = decltype(t);
        if (pl.g) launch<T>(pl, blocks, a, st);
        else launch_parts<T>(parts, span, blocks, a, (Row*)(part + 3 * MAX_BLOCKS), st);
    };
    if (dtype == STEP_F32) go(float());
    else if (dtype == STEP_BF16) go(bf16());
    else go(f16());
    if (!upstream)
        hipLaunchKernelGGL(policy_finish_kernel, dim3(1), dim3(256), 0, st, part, mask ? count : nullptr, (double)rows,
                           blocks, beta, loss, stats);
    return step::check_launch("step_policy_loss");
}
