// Clipped policy loss with a KL term, value and gradient in one pass over the logits (rows, classes).
//
//   lp = z[a] - log SUM exp z,  rho = exp(lp - old),  o1 = rho A,  o2 = min(max(rho, 1 - cl), 1 + ch) A
//   L = -min(o1, o2),  kl = exp(ref - lp) - (ref - lp) - 1 >= 0
//   loss = SUM_live (L + beta kl) / max(#live, 1)
//   dL/dlp = [o1 <= o2] (-o1) + beta (1 - exp(ref - lp)),  dz = dL/dlp / max(#live, 1) * (onehot(a) - softmax z)
//
// Memory-bound: the least is one read of the live rows' logits and one write of the gradient.  A row stays in the
// registers of the G threads that share it between its softmax sums and its gradient (up to 128 K classes in 16 bits,
// 64 K in fp32); longer rows are read twice.  The number of live rows, which every row's gradient is divided by, is
// counted by a launch before.  A row's few scalars are taken in fp64: its ratio may lie next to the border of the
// clipping.  Per-block fp64 sums are added in block order by the last launch: the same bits every time, no atomics.
// A masked row is not read at all (its logits, and its action, may be anything): log probability 0, gradient 0.
#include "rows.h"

namespace {
using namespace step;

constexpr float L2E = 1.4426950408889634f, L2E_REST = 1.92596299e-8f;
constexpr double LN2 = 0.69314718055994530942;
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
    int skip_one;                  // with upstream: nothing to do where it is exactly 1
    long long rows;
    int classes;
    double clip_low, clip_high, beta;   // a clipped ratio's 1.2 in fp32 is off by 4e-8, the same way in every row
};

// 16 bytes of a row, -inf outside it; a pack that the row fills only in part is read by elements, so nothing outside the
// row is touched
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load_pack(const T* row, int e0, int classes) {
    if (e0 >= 0 && e0 + N <= classes) return *(const Pack<T, N>*)(row + e0);
    Pack<T, N> q;
#pragma unroll
    for (int e = 0; e < N; ++e) q.v[e] = e0 + e >= 0 && e0 + e < classes ? row[e0 + e] : (T)(-__builtin_inff());
    return q;
}
template <typename T, int N>
__device__ __forceinline__ void store_pack(T* row, int e0, int classes, const Pack<T, N> q) {
    if (e0 >= 0 && e0 + N <= classes) {
        *(Pack<T, N>*)(row + e0) = q;
        return;
    }
#pragma unroll
    for (int e = 0; e < N; ++e)
        if (e0 + e >= 0 && e0 + e < classes) row[e0 + e] = q.v[e];
}

// maximum and sum of exponentials about it, joined over the G threads of a row, in base 2: m is the row's largest logit
// times log2 e, rounded once and from there on exact, an element's exponent x log2 e - m is one fused operation
struct Soft {
    float m, s;
};
__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float exp_of(float x, float m) { return __builtin_amdgcn_exp2f(__builtin_fmaf(x, L2E, -m)); }
// for the sum, whose logarithm the loss hangs on: with the rest of log2 e too (fp32's log2 e alone is off by 1.3e-8, the same
// way for all elements)
__device__ __forceinline__ float exp_for_sum(float x, float m) {
    return __builtin_amdgcn_exp2f(__builtin_fmaf(x, L2E_REST, __builtin_fmaf(x, L2E, -m)));
}
__device__ __forceinline__ float finite_or_0(float m) { return m == -__builtin_inff() ? 0.f : m; }   // no -inf - -inf

template <int G>
__device__ __forceinline__ Soft join(const Soft w, Soft* sm) {
    if constexpr (G <= 64) {
        return w;
    } else {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = w;
        __syncthreads();
        Soft r = sm[0];
#pragma unroll
        for (int i = 1; i < G / 64; ++i) r.m = fmaxf(r.m, sm[i].m);
        const float m0 = finite_or_0(r.m);
        r.s = 0.f;
#pragma unroll
        for (int i = 0; i < G / 64; ++i) r.s += sm[i].s * exp_of(sm[i].m - m0);
        return r;
    }
}

// the row's scalars: returns dL/dlp / count (times the upstream gradient), adds the row to the block's sums
__device__ __forceinline__ float row_scalars(const Args& p, long long row, Soft f, float za, bool valid, double count,
                                             double* sums) {
    const double lp = valid ? (double)za - ((double)f.m + log2((double)f.s)) * LN2 : (double)__builtin_nanf("");
    const double a = p.adv[row], ratio = exp(lp - (double)p.old_logp[row]);
    const double lo = 1.0 - p.clip_low, hi = 1.0 + p.clip_high;
    const double o1 = ratio * a, o2 = (ratio > hi ? hi : ratio < lo ? lo : ratio) * a;   // a NaN stays one
    const bool clipped = o1 > o2;
    double slope = clipped ? 0.0 : -o1, kl = 0.0;
    if (p.ref) {
        const double d = (double)p.ref[row] - lp, e = exp(d);
        kl = e - d - 1.0;
        slope += p.beta * (1.0 - e);
    }
    sums[0] += clipped ? -o2 : -o1;
    sums[1] += kl;
    sums[2] += clipped ? 1.0 : 0.0;
    if (!p.upstream) p.logp[row] = (float)lp;
    else slope *= (double)*p.upstream;
    return (float)(slope / count);
}

template <typename T, int N>
__device__ __forceinline__ Pack<T, N> gradient_of(const Pack<T, N> z, int e0, long long action, float m, float inv_s,
                                                  float coef) {
    Pack<T, N> g;
#pragma unroll
    for (int e = 0; e < N; ++e) {
        float v = -coef * (exp_of((float)z.v[e], m) * inv_s);
        if (e0 + e == action) v += coef;
        g.v[e] = (T)v;                                       // the gradient's only rounding
    }
    return g;
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

// NV packs of 16 bytes a thread; NV = 0: the row is read twice
template <typename T, int G, int NV>
__global__ __launch_bounds__(G < 256 ? 256 : G) void policy_kernel(const Args p) {
    constexpr int BLOCK = G < 256 ? 256 : G, RPB = BLOCK / G, N = 16 / (int)sizeof(T), KEEP = NV ? NV : 1;
    __shared__ Soft sm[G > 64 ? G / 64 : 1];
    __shared__ float coef_s;
    if (p.upstream && p.skip_one && *p.upstream == 1.f) return;
    const int lane = threadIdx.x % G;
    const double live_rows = p.count ? *p.count : (double)p.rows, count = live_rows > 1.0 ? live_rows : 1.0;
    double sums[3] = {0.0, 0.0, 0.0};
    for (long long r0 = (long long)blockIdx.x * RPB; r0 < p.rows; r0 += (long long)gridDim.x * RPB) {
        const long long row = r0 + threadIdx.x / G;
        if (G <= 64 && row >= p.rows) continue;              // (whole blocks share a row otherwise)
        const T* z = (const T*)p.logits + (size_t)row * p.classes;
        T* g = p.dlogits ? (T*)p.dlogits + (size_t)row * p.classes : nullptr;
        const int shift = (int)(((uintptr_t)z & 15) / sizeof(T));
        const int packs = (shift + p.classes + N - 1) / N;
        if (p.mask && !p.mask[row]) {
            if (lane == 0 && !p.upstream) p.logp[row] = 0.f;
            if (g) {
                Pack<T, N> zero;
#pragma unroll
                for (int e = 0; e < N; ++e) zero.v[e] = (T)0.f;
                for (int i = lane; i < packs; i += G) store_pack<T, N>(g, i * N - shift, p.classes, zero);
            }
            continue;
        }
        const long long action = p.actions[row];
        const bool valid = action >= 0 && action < p.classes;
        const float za = lane == 0 && valid ? (float)z[action] : 0.f;
        Pack<T, N> v[KEEP];
        Soft f{-__builtin_inff(), 0.f};
        if constexpr (NV > 0) {
#pragma unroll
            for (int i = 0; i < NV; ++i) v[i] = load_pack<T, N>(z, (i * G + lane) * N - shift, p.classes);
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int e = 0; e < N; ++e) f.m = fmaxf(f.m, (float)v[i].v[e]);
            f.m = group_wave_reduce<G>(f.m, [](float a, float b) { return fmaxf(a, b); }) * L2E;
            const float m0 = finite_or_0(f.m);
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int e = 0; e < N; ++e) f.s += exp_for_sum((float)v[i].v[e], m0);
        } else {
            for (int i = lane; i < packs; i += G) {
                const Pack<T, N> q = load_pack<T, N>(z, i * N - shift, p.classes);
                float m = -__builtin_inff();
#pragma unroll
                for (int e = 0; e < N; ++e) m = fmaxf(m, (float)q.v[e]);
                m = fmaxf(f.m, m * L2E);
                const float m0 = finite_or_0(m);
                f.s *= exp_of(f.m - m0);
#pragma unroll
                for (int e = 0; e < N; ++e) f.s += exp_for_sum((float)q.v[e], m0);
                f.m = m;
            }
            const float m = group_wave_reduce<G>(f.m, [](float a, float b) { return fmaxf(a, b); });
            f.s *= exp_of(f.m - finite_or_0(m));
            f.m = m;
        }
        f.s = group_wave_reduce<G>(f.s, [](float a, float b) { return a + b; });
        f = join<G>(f, sm);
        float coef;
        if constexpr (G <= 64) {
            double add[3] = {0.0, 0.0, 0.0};
            coef = row_scalars(p, row, f, __shfl(za, (threadIdx.x & 63) & ~(G - 1), 64), valid, count, add);
            if (lane == 0)
                for (int k = 0; k < 3; ++k) sums[k] += add[k];
        } else {
            if (threadIdx.x == 0) coef_s = row_scalars(p, row, f, za, valid, count, sums);
            __syncthreads();
            coef = coef_s;
        }
        if (!g) continue;
        const float inv_s = 1.f / f.s;
        if constexpr (NV > 0) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int e0 = (i * G + lane) * N - shift;
                if (e0 < p.classes) store_pack<T, N>(g, e0, p.classes, gradient_of<T, N>(v[i], e0, action, f.m, inv_s, coef));
            }
        } else {
            for (int i = lane; i < packs; i += G) {
                const int e0 = i * N - shift;
                const Pack<T, N> q = load_pack<T, N>(z, e0, p.classes);
                store_pack<T, N>(g, e0, p.classes, gradient_of<T, N>(q, e0, action, f.m, inv_s, coef));
            }
        }
    }
    if (!p.upstream) block_sums<BLOCK>(p.part, sums);
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
    int g, nv;
};
Plan plan(int classes, int dtype, bool aligned) {
    const int n = 16 / elem_bytes(dtype);
    // packs that the row touches at most, whatever 16-byte boundary it starts behind
    const long long packs = aligned && classes % n == 0 ? classes / n : ((long long)classes + 2 * n - 2) / n;
    const Plan all[] = {{8, 1}, {64, 1}, {64, 4}, {256, 4}, {1024, 2}, {1024, 4}, {1024, 8}, {1024, 16}};
    for (const Plan& p : all)
        if (packs <= (long long)p.g * p.nv) return p;
    return Plan{1024, 0};
}
int blocks_of(long long rows, const Plan& p) {
    const int rpb = p.g < 256 ? 256 / p.g : 1, cap = p.g == 1024 ? 512 : MAX_BLOCKS;
    const long long need = (rows + rpb - 1) / rpb;
    return (int)(need < cap ? need : cap);
}

template <typename T>
void launch(const Plan& pl, int blocks, const Args& a, hipStream_t st) {
#define STEP_POLICY(G, NV)                                                                                     \
    if (pl.g == G && pl.nv == NV) {                                                                            \
        hipLaunchKernelGGL((policy_kernel<T, G, NV>), dim3(blocks), dim3(G < 256 ? 256 : G), 0, st, a);        \
        return;                                                                                                \
    }
    STEP_POLICY(8, 1)
    STEP_POLICY(64, 1)
    STEP_POLICY(64, 4)
    STEP_POLICY(256, 4)
    STEP_POLICY(1024, 2)
    STEP_POLICY(1024, 4)
    STEP_POLICY(1024, 8)
    STEP_POLICY(1024, 16)
    STEP_POLICY(1024, 0)
#undef STEP_POLICY
}

}  // namespace

extern "C" size_t step_policy_loss_ws_bytes(long long rows) {
    return rows > 0 ? (1 + 3 * (size_t)MAX_BLOCKS) * sizeof(double) : 0;
}

extern "C" int step_policy_loss(const void* logits, const long long* actions, const float* old_logp,
                                const float* advantages, const float* ref_logp, const unsigned char* mask,
                                double clip_low, double clip_high, double beta, const float* upstream, int skip_one,
                                float* loss, float* stats, float* logp, void* dlogits, long long rows, int classes,
                                int dtype, void* ws, size_t ws_bytes, void* stream) {
    STEP_REQUIRE(logits && actions && old_logp && advantages && ws, "step_policy_loss: null pointer");
    STEP_REQUIRE(rows >= 1 && classes >= 1 && classes <= 0x7fffff00, "step_policy_loss: bad shape rows=%lld classes=%d", rows, classes);
    STEP_REQUIRE(elem_bytes(dtype), "step_policy_loss: unknown type %d", dtype);
    STEP_REQUIRE(upstream ? dlogits != nullptr : loss && stats && logp, "step_policy_loss: null output");
    STEP_REQUIRE(!dlogits || (((uintptr_t)logits ^ (uintptr_t)dlogits) & 15) == 0,
                 "step_policy_loss: logits and dlogits lie differently to 16 bytes");
    STEP_REQUIRE(((uintptr_t)logits & (elem_bytes(dtype) - 1)) == 0, "step_policy_loss: logits lie across elements");
    if (ws_bytes < step_policy_loss_ws_bytes(rows)) {
        step::set_error("step_policy_loss: workspace %zu < %zu bytes", ws_bytes, step_policy_loss_ws_bytes(rows));
        return STEP_ERR_WORKSPACE;
    }
    hipStream_t st = (hipStream_t)stream;
    double* count = (double*)ws;
    double* part = count + 1;
    const Plan pl = plan(classes, dtype, ((uintptr_t)logits & 15) == 0);
    const int blocks = blocks_of(rows, pl);
    if (mask && !upstream) hipLaunchKernelGGL(policy_count_kernel, dim3(1), dim3(1024), 0, st, mask, count, rows);
    const Args a{logits, actions, old_logp, advantages, ref_logp, mask, dlogits, logp, mask ? count : nullptr, part,
                 upstream, skip_one, rows, classes, clip_low, clip_high, beta};
    if (dtype == STEP_F32) launch<float>(pl, blocks, a, st);
    else if (dtype == STEP_BF16) launch<bf16>(pl, blocks, a, st);
    else launch<f16>(pl, blocks, a, st);
    if (!upstream)
        hipLaunchKernelGGL(policy_finish_kernel, dim3(1), dim3(256), 0, st, part, mask ? count : nullptr, (double)rows,
                           blocks, beta, loss, stats);
    return step::check_launch("step_policy_loss");
}
