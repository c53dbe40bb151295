// Log probabilities of given tokens from logits, with the entropy of each distribution and its
// most likely tokens, and the gradient of both with respect to the logits.
//
//   lse = m + log sum_j e^(x_j - m),  log_prob = x_t - lse,
//   entropy = -sum_j p_j log p_j = log s - u / s,  s = sum_j e^(x_j - m),  u = sum_j (x_j - m) e^(x_j - m)
//
// s and u are kept together with the running maximum m: when m grows by d, s and u become
// s e^-d and (u - d s) e^-d, so one pass over the row gives all three.  A logit of -inf (a
// masked token) adds nothing; a row of nothing else has lse = log_prob = -inf and entropy 0.
// The alternatives are ordered by logit, ties by the lower token id, NaN after every number.
//
//   d_logits_j = d_log_prob (1[j = t] - p_j) - d_entropy p_j (log p_j + entropy)
#pragma once
#include "dt_common.cuh"

namespace dt {
namespace logprobs {

constexpr int kThreads = 512;
constexpr int kMaxTop = 32;

struct Params {
    const void* x;       // [N, V], rows ld apart
    long long ld;
    int N, V;
    const void* targets; // int32 or int64 [N], or null
    int targets64;
    int top;
    float* log_prob;     // [N] or null
    float* entropy;      // [N] or null
    float* lse;          // [N] or null
    int* top_ids;        // [N, top]
    float* top_log_probs;
};

struct GradParams {
    const void* x;
    long long ld;
    int N, V;
    const void* targets;
    int targets64;
    const float* lse;
    const float* entropy;
    const float* d_log_prob;  // or null
    const float* d_entropy;   // or null
    void* dx;                 // [N, V], rows dx_ld apart
    long long dx_ld;
};

template <bool kF32>
__device__ __forceinline__ float logit(const void* x, long long i) {
    return kF32 ? __ldg(static_cast<const float*>(x) + i)
                : __bfloat162float(__ldg(static_cast<const __nv_bfloat16*>(x) + i));
}

__device__ __forceinline__ long long target_of(const void* t, int is64, int row) {
    if (!t) return -1;
    return is64 ? __ldg(static_cast<const long long*>(t) + row) : (long long)__ldg(static_cast<const int*>(t) + row);
}

// Larger key = earlier alternative: the logit's bits in an order that integers share, NaN
// lowest, then the token id downwards.
__device__ __forceinline__ unsigned long long order_key(float x, int id) {
    uint32_t u = __float_as_uint(x);
    u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
    if (x != x) u = 0u;
    if (x == 0.f) u = 0x80000000u;  // -0 and 0 are equal
    return ((unsigned long long)u << 32) | (uint32_t)(0x7fffffff - id);
}

__device__ __forceinline__ void merge(float& m, float& s, float& u, float m2, float s2, float u2) {
    const float mn = fmaxf(m, m2);
    if (mn == -INFINITY) return;
    const float d1 = m - mn, d2 = m2 - mn;  // 0 or negative; -inf for an empty side
    const float e1 = expf(d1), e2 = expf(d2);
    // (a term whose weight underflows is dropped before d * s can overflow)
    u = (e1 == 0.f ? 0.f : (u + d1 * s) * e1) + (e2 == 0.f ? 0.f : (u2 + d2 * s2) * e2);
    s = s * e1 + s2 * e2;
    m = mn;
}

// One CTA per row; one pass for the sums, then one pass per alternative.
template <bool kF32>
__global__ void __launch_bounds__(kThreads) row_kernel(const Params p) {
    pdl_enter();
    __shared__ float sm[kThreads / 32], ss[kThreads / 32], su[kThreads / 32];
    __shared__ unsigned long long sk[kThreads / 32];
    const int row = blockIdx.x;
    const long long base = (long long)row * p.ld;
    float m = -INFINITY, s = 0.f, u = 0.f;
    bool bad = false;
    for (int j = threadIdx.x; j < p.V; j += kThreads) {
        const float x = logit<kF32>(p.x, base + j);
        bad |= x != x;
        if (x > -INFINITY) merge(m, s, u, x, 1.f, 0.f);
    }
    if (bad) s = u = NAN;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o),
                    u2 = __shfl_xor_sync(0xffffffffu, u, o);
        const bool nan = s != s || s2 != s2;
        merge(m, s, u, m2, s2, u2);
        if (nan) s = u = NAN;
    }
    if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = m, ss[threadIdx.x >> 5] = s, su[threadIdx.x >> 5] = u;
    __syncthreads();
    m = sm[0], s = ss[0], u = su[0];
    for (int w = 1; w < kThreads / 32; ++w) {
        const bool nan = s != s || ss[w] != ss[w];
        merge(m, s, u, sm[w], ss[w], su[w]);
        if (nan) s = u = NAN;
    }
    const bool empty = s == 0.f;
    const float ls = logf(s);
    const float lse = empty ? -INFINITY : m + ls;
    if (threadIdx.x == 0) {
        const long long t = target_of(p.targets, p.targets64, row);
        float lp = 0.f;
        if (t >= 0 && t < p.V) lp = empty ? -INFINITY : (logit<kF32>(p.x, base + t) - m) - ls;
        if (p.log_prob) p.log_prob[row] = lp;
        if (p.entropy) p.entropy[row] = empty ? 0.f : ls - u / s;
        if (p.lse) p.lse[row] = lse;
    }
    unsigned long long last = ~0ull;
    for (int k = 0; k < p.top; ++k) {
        unsigned long long best = 0;
        for (int j = threadIdx.x; j < p.V; j += kThreads) {
            const unsigned long long key = order_key(logit<kF32>(p.x, base + j), j);
            if (key < last && key > best) best = key;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
            best = other > best ? other : best;
        }
        __syncthreads();
        if ((threadIdx.x & 31) == 0) sk[threadIdx.x >> 5] = best;
        __syncthreads();
        for (int w = 0; w < kThreads / 32; ++w) best = sk[w] > best ? sk[w] : best;
        last = best;
        if (threadIdx.x == 0) {
            const int id = 0x7fffffff - (int)(uint32_t)best;
            p.top_ids[(long long)row * p.top + k] = id;
            p.top_log_probs[(long long)row * p.top + k] = empty ? -INFINITY : (logit<kF32>(p.x, base + id) - m) - ls;
        }
    }
}

template <bool kF32>
__global__ void __launch_bounds__(kThreads) grad_kernel(const GradParams p) {
    pdl_enter();
    const int row = blockIdx.x;
    const long long base = (long long)row * p.ld, dbase = (long long)row * p.dx_ld;
    const long long t = target_of(p.targets, p.targets64, row);
    const bool has = t >= 0 && t < p.V;
    const float g = has && p.d_log_prob ? p.d_log_prob[row] : 0.f;
    const float h = p.d_entropy ? p.d_entropy[row] : 0.f;
    const float lse = p.lse[row], ent = p.entropy ? p.entropy[row] : 0.f;
    for (int j = threadIdx.x; j < p.V; j += kThreads) {
        const float x = logit<kF32>(p.x, base + j);
        float d = 0.f;
        if (lse != -INFINITY) {
            const float lp = x - lse;
            if (x != -INFINITY) d = -expf(lp) * (g + h * (lp + ent));
            if (j == t) d += g;
        }
        if (kF32) static_cast<float*>(p.dx)[dbase + j] = d;
        else static_cast<__nv_bfloat16*>(p.dx)[dbase + j] = __float2bfloat16_rn(d);
    }
}

}  // namespace logprobs
}  // namespace dt
