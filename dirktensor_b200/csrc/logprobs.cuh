// Log probabilities of given tokens from logits, with the entropy of each distribution and its
// most likely tokens, and the gradient of both with respect to the logits.
//
//   lse = m + log sum_j e^(x_j - m),  log_prob = x_t - lse,
//   entropy = -sum_j p_j log p_j = log s - u / s,  s = sum_j e^(x_j - m),  u = sum_j (x_j - m) e^(x_j - m)
//
// s and u are kept together with the running maximum m: when m grows by d, s and u become
// s e^-d and (u - d s) e^-d, so one pass over the row gives all three.  A logit of -inf (a
// masked token) adds nothing; a row of nothing else has lse = log_prob = -inf and entropy 0.
// Differences below -200 weigh nothing in fp32 and are cut there, which keeps infinities (and masks of the
// type's lowest value) out of products with zero.  The alternatives are ordered by logit, ties by
// the lower token id, NaN after every number.
//
//   d_logits_j = d_log_prob (1[j = t] - p_j) - d_entropy p_j (log p_j + entropy)
#pragma once
#include <cooperative_groups.h>

#include "dt_common.cuh"

namespace dt {
namespace logprobs {

constexpr int kThreads = 256;
constexpr int ctas_per_sm(bool f32) { return f32 ? 4 : 5; }  // (64 and 48 registers a thread)
constexpr int kWarps = kThreads / 32;
constexpr int kMaxTop = 32;
constexpr int kMaxCluster = 16;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLowest = -3.402823466e38f;
constexpr float kFar = -200.f;  // e^-200 is 0 in fp32: no difference below it counts

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
    int split;           // CTAs (a cluster) per row
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
    int chunks;               // CTAs per row
};

template <bool kF32>
__device__ __forceinline__ float logit(const void* x, long long i) {
    return kF32 ? static_cast<const float*>(x)[i] : __bfloat162float(static_cast<const __nv_bfloat16*>(x)[i]);
}

__device__ __forceinline__ long long target_of(const void* t, int is64, int row) {
    if (!t) return -1;
    return is64 ? __ldg(static_cast<const long long*>(t) + row) : (long long)__ldg(static_cast<const int*>(t) + row);
}

// The larger of two, a NaN if either is one.
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// The logit's bits in an order that unsigned numbers share, NaN lowest; -0 and 0 alike.
__device__ __forceinline__ uint32_t order_bits(float x) {
    const uint32_t u = __float_as_uint(x + 0.f);
    return x != x ? 0u : (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float from_order_bits(uint32_t u) {
    return u == 0u ? __uint_as_float(0x7fffffffu) : __uint_as_float((u & 0x80000000u) ? (u & 0x7fffffffu) : ~u);
}
// Larger key = earlier alternative: by logit, then by the lower id.  No logit has the key 0.
__device__ __forceinline__ unsigned long long order_key(float x, int id) {
    return ((unsigned long long)order_bits(x) << 32) | (uint32_t)(0x7fffffff - id);
}

// Lists of 32 numbers, one per lane, largest first.
template <typename K>
__device__ __forceinline__ K keep_larger(K x, int distance, bool larger) {
    const K y = __shfl_xor_sync(0xffffffffu, x, distance);
    return larger == (y > x) ? y : x;
}
template <typename K>
__device__ __forceinline__ K sorted(K x) {  // bitonic
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int d = size >> 1; d > 0; d >>= 1) x = keep_larger(x, d, ((lane & d) == 0) == ((lane & size) == 0 || size == 32));
    return x;
}
// The 32 largest of two lists.
template <typename K>
__device__ __forceinline__ K merged(K a, K b) {
    const int lane = threadIdx.x & 31;
    b = __shfl_sync(0xffffffffu, b, 31 - lane);
    a = b > a ? b : a;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) a = keep_larger(a, d, (lane & d) == 0);
    return a;
}
// The 32 largest of the lists of the CTA's first `n` warps (a power of two), in warp 0.
template <typename K>
__device__ __forceinline__ K merged_over_warps(K x, int n, K (*scratch)[32]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int half = n >> 1; half > 0; half >>= 1) {
        __syncthreads();
        if (warp >= half && warp < 2 * half) scratch[warp][lane] = x;
        __syncthreads();
        if (warp < half) x = merged(x, scratch[warp + half][lane]);
    }
    return x;
}

// s = sum e^(x - m), u = sum (x - m) e^(x - m), relative to m.
struct Sums {
    float m, s, u;
    static __device__ __forceinline__ Sums none() { return {kLowest, 0.f, 0.f}; }
    __device__ __forceinline__ void move_to(float mn) {  // mn >= m
        const float d = max_nan(m - mn, kFar);
        const float e = ex2_approx(d * kLog2e);
        u = (u + d * s) * e;
        s *= e;
        m = mn;
    }
    __device__ __forceinline__ void add(Sums o) {
        const float mn = max_nan(m, o.m);
        move_to(mn);
        o.move_to(mn);
        s += o.s;
        u += o.u;
    }
};

// 16 bytes of a row as fp32.
template <bool kF32>
struct Vec {
    static constexpr int kN = kF32 ? 4 : 8;
    float x[kN];
};

// One row, or one CTA's share of it, as vectors of 16 aligned bytes; the first and the last may lie
// partly outside the row, and then only what is inside is read.
template <bool kF32>
struct Row {
    static constexpr int kN = Vec<kF32>::kN;
    const char* base;  // of vector 0
    int skip;          // elements of vector 0 before the row
    int V;
    __device__ __forceinline__ Row(const void* x, long long first, int V_) : V(V_) {
        const char* p = static_cast<const char*>(x) + first * (kF32 ? 4 : 2);
        const int off = (int)(reinterpret_cast<uintptr_t>(p) & 15);
        skip = off / (kF32 ? 4 : 2);
        base = p - off;
    }
    __device__ __forceinline__ int vectors() const { return (V + skip + kN - 1) / kN; }
    __device__ __forceinline__ int id(int v, int e) const { return v * kN + e - skip; }
    __device__ __forceinline__ bool inside(int v) const { return id(v, 0) >= 0 && id(v, kN - 1) < V; }
    __device__ __forceinline__ uint4 load(int v) const { return __ldg(reinterpret_cast<const uint4*>(base) + v); }
    __device__ __forceinline__ static Vec<kF32> unpack(uint4 y) {
        Vec<kF32> r;
        const uint32_t w[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (kF32) r.x[i] = __uint_as_float(w[i]);
            else r.x[2 * (i & 3) % kN] = __uint_as_float(w[i] << 16), r.x[(2 * (i & 3) + 1) % kN] = __uint_as_float(w[i] & 0xffff0000u);
        }
        return r;
    }
    // a vector at either end, -inf where it is outside
    __device__ __forceinline__ Vec<kF32> edge(int v) const {
        Vec<kF32> r;
#pragma unroll
        for (int e = 0; e < kN; ++e) r.x[e] = id(v, e) >= 0 && id(v, e) < V ? logit<kF32>(base, (long long)v * kN + e) : -INFINITY;
        return r;
    }
};

constexpr int kGroups = kThreads / 8;     // of threads, whose largest logits bound the k-th
static_assert(kGroups >= kMaxTop, "a bound for every k");
constexpr int kCandidates = 512;

struct Smem {
    unsigned long long list[kWarps][32];
    unsigned long long found[kCandidates];  // logits that reach the threshold
    unsigned long long best[32];            // the CTA's alternatives
    Sums sums[kWarps];
    Sums total;                             // of the CTA, for the cluster
    float groups[kGroups];
    float threshold;
    int count;
};

// A cluster of `split` CTAs per row (one, unless the rows are too few to fill the GPU).  One pass gives the
// sums and every thread's largest logit.  The k-th largest of 32 groups' largest logits is no larger than
// the row's k-th largest logit, so the alternatives all lie with threads whose largest logit reaches it: about k
// of 256.  Each of these reads the 16 logits around its largest again, or, where another of its batches
// reaches the threshold too, its warp reads all of its logits.  What reaches the threshold is collected
// and sorted by one warp; rows with more than 512 such logits (ties) are sorted by all warps instead.
// Bound by the read: 2048 rows of 100352 fp32 logits take 123 us (6.7 TB/s) without alternatives, 132 with
// 5 and 143 with 20; bf16, whose 2 bytes a logit leave half the time for the same arithmetic, 85 us (4.9 TB/s).
// (512 threads, two or three CTAs per SM: 144 to 160 us with 5.)
template <bool kF32>
__global__ void __launch_bounds__(kThreads, ctas_per_sm(kF32)) row_kernel(const Params p) {
    pdl_enter();
    __shared__ Smem sm;
    constexpr int kN = Vec<kF32>::kN;
    constexpr int kBatch = 16 / kN;  // vectors at a time
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int row = p.split == 1 ? (int)blockIdx.x : (int)(blockIdx.x / (unsigned)p.split), rank = (int)blockIdx.x - row * p.split;
    const Row<kF32> r(p.x, (long long)row * p.ld, p.V);
    const int vectors = r.vectors();
    const int begin = (int)((long long)vectors * rank / p.split), end = (int)((long long)vectors * (rank + 1) / p.split);
    // whole vectors; the first and the last may cross the row's ends
    const int lo = begin + (r.inside(begin) ? 0 : 1), hi = end - (end > begin && r.inside(end - 1) ? 0 : 1);
    // thread 0 takes the share's first vector and thread 1 its last, where they do
    const int edge = threadIdx.x == 0 && lo > begin ? begin : threadIdx.x == 1 && hi < end && hi >= lo ? hi : -1;

    Sums a = Sums::none();
    float most = -INFINITY, next = -INFINITY;  // this thread's largest logit, and that of its other batches
    int where = 0;                             // first vector of the batch that has it
    bool odd = false;                          // it saw a NaN
    auto take = [&](const uint4 (&y)[kBatch], int v) {
        uint64_t x[8];  // pairs
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const uint32_t w[4] = {y[i].x, y[i].y, y[i].z, y[i].w};
#pragma unroll
            for (int e = 0; e < kN / 2; ++e)
                x[i * (kN / 2) + e] = kF32 ? f2_pack(__uint_as_float(w[2 * e % 4]), __uint_as_float(w[(2 * e + 1) % 4]))
                                           : f2_pack(__uint_as_float(w[e % 4] << 16), __uint_as_float(w[e % 4] & 0xffff0000u));
        }
        float t = -INFINITY;
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            float x0, x1, x2, x3;
            f2_unpack(x[i], x0, x1);
            f2_unpack(x[i + 1], x2, x3);
            t = max_nan(t, max_nan(max3_nan(x0, x1, x2), x3));
        }
        odd |= t != t;
        const bool larger = t > most;
        next = fmaxf(next, larger ? most : t);
        where = larger ? v : where;
        most = larger ? t : most;
        if (!(t <= a.m)) a.move_to(max_nan(a.m, t));  // (a NaN too)
        const uint64_t minus = f2_pack(-a.m, -a.m);
        uint64_t s = f2_pack(0.f, 0.f), u = f2_pack(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float d0, d1;
            f2_unpack(f2_add(x[i], minus), d0, d1);
            d0 = max_nan(d0, kFar), d1 = max_nan(d1, kFar);
            const uint64_t e = f2_pack(ex2_approx(d0 * kLog2e), ex2_approx(d1 * kLog2e));
            s = f2_add(s, e);
            u = f2_fma(f2_pack(d0, d1), e, u);
        }
        float s0, s1, u0, u1;
        f2_unpack(s, s0, s1);
        f2_unpack(u, u0, u1);
        a.s += s0 + s1;
        a.u += u0 + u1;
    };
    const uint32_t none = kF32 ? 0xff800000u : 0xff80ff80u;  // -inf
    auto fetch = [&](uint4 (&y)[kBatch], int v) {
#pragma unroll
        for (int i = 0; i < kBatch; ++i) y[i] = v + i * kThreads < hi ? r.load(v + i * kThreads) : make_uint4(none, none, none, none);
    };
    {  // the next batch is on its way while this one is added up
        uint4 y[kBatch], z[kBatch];
        fetch(y, lo + threadIdx.x);
        for (int v = lo + threadIdx.x; v < hi; v += 2 * kBatch * kThreads) {
            fetch(z, v + kBatch * kThreads);
            take(y, v);
            fetch(y, v + 2 * kBatch * kThreads);
            if (v + kBatch * kThreads < hi) take(z, v + kBatch * kThreads);
        }
    }
    if (edge >= 0) {
        const Vec<kF32> z = r.edge(edge);
        uint4 y[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) y[i] = make_uint4(none, none, none, none);
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            w[e] = kF32 ? __float_as_uint(z.x[e % kN]) : (__float_as_uint(z.x[2 * e % kN]) >> 16) | __float_as_uint(z.x[(2 * e + 1) % kN]);
        y[0] = make_uint4(w[0], w[1], w[2], w[3]);
        take(y, edge);
        next = most;  // (its batch is not as the others': all of its logits are read again)
    }

    if (p.top > 0) {
        // a logit that the row's k-th largest reaches
        float top = most;
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        if ((lane & 7) == 0) sm.groups[threadIdx.x >> 3] = top;
        if (threadIdx.x == 0) sm.count = 0;
        __syncthreads();
        if (threadIdx.x < kGroups) {
            const float mine = sm.groups[threadIdx.x];
            int above = 0;
#pragma unroll 8
            for (int j = 0; j < kGroups; ++j) {
                const float x = sm.groups[j];
                above += x > mine || (x == mine && j < (int)threadIdx.x);
            }
            if (above == p.top - 1) sm.threshold = mine;
        }
        __syncthreads();
        const float threshold = sm.threshold;
        // (at -inf everything counts, NaNs too)
        auto reaches = [&](float x, int id) { return id >= 0 && id < p.V && (x >= threshold || threshold == -INFINITY); };
        auto collect = [&](float x, int id) {
            if (reaches(x, id)) {
                const int at = atomicAdd(&sm.count, 1);
                if (at < kCandidates) sm.found[at] = order_key(x, id);
            }
        };
        // reads all vectors of thread `who` again, a lane each, and calls each(element, key of this lane or 0)
        auto again = [&](int who, auto each) {
            const int extra = who == 0 && lo > begin ? begin : who == 1 && hi < end && hi >= lo ? hi : -1;
            const int n = (hi - lo - who + kThreads - 1) / kThreads + (extra >= 0 ? 1 : 0);
#pragma unroll 1
            for (int i0 = 0; i0 < n; i0 += 32) {
                const int i = i0 + lane;
                const int mine = i >= n ? -1 : extra >= 0 && i == n - 1 ? extra : lo + who + i * kThreads;
                Vec<kF32> z;
#pragma unroll
                for (int e = 0; e < kN; ++e) z.x[e] = -INFINITY;
                if (mine >= 0) z = mine == extra ? r.edge(mine) : Row<kF32>::unpack(r.load(mine));
#pragma unroll
                for (int e = 0; e < kN; ++e) each(z.x[e], mine >= 0 ? r.id(mine, e) : -1);
            }
        };
        const bool flagged = odd || most >= threshold;
        const bool all = odd || next >= threshold;
        if (flagged && !all) {
            uint4 y[kBatch];
            fetch(y, where);
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                const Vec<kF32> z = Row<kF32>::unpack(y[i]);
#pragma unroll
                for (int e = 0; e < kN; ++e) collect(z.x[e], where + i * kThreads < hi ? r.id(where + i * kThreads, e) : -1);
            }
        }
        for (uint32_t todo = __ballot_sync(0xffffffffu, flagged && all); todo; todo &= todo - 1)
            again(warp * 32 + __ffs(todo) - 1, collect);
        __syncthreads();
        const int count = sm.count;
        unsigned long long list = 0;
        if (count <= kCandidates) {
            if (warp == 0)
                for (int i = 0; i < count; i += 32) list = merged(list, sorted(i + lane < count ? sm.found[i + lane] : 0ull));
        } else {
            unsigned long long least = 0;  // this warp's k-th
            for (uint32_t todo = __ballot_sync(0xffffffffu, flagged); todo; todo &= todo - 1)
                again(warp * 32 + __ffs(todo) - 1, [&](float x, int id) {
                    const unsigned long long key = reaches(x, id) ? order_key(x, id) : 0ull;
                    if (__any_sync(0xffffffffu, key > least)) {
                        list = merged(list, sorted(key));
                        least = __shfl_sync(0xffffffffu, list, p.top - 1);
                    }
                });
            list = merged_over_warps(list, kWarps, sm.list);
        }
        if (warp == 0) sm.best[lane] = list;
    }

    // join the threads' sums, the warps', the cluster's
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        Sums b;
        b.m = __shfl_xor_sync(0xffffffffu, a.m, o);
        b.s = __shfl_xor_sync(0xffffffffu, a.s, o);
        b.u = __shfl_xor_sync(0xffffffffu, a.u, o);
        a.add(b);
    }
    if (lane == 0) sm.sums[warp] = a;
    __syncthreads();
    if (warp == 0) {
        a = lane < kWarps ? sm.sums[lane] : Sums::none();
#pragma unroll
        for (int o = kWarps / 2; o > 0; o >>= 1) {
            Sums b;
            b.m = __shfl_xor_sync(0xffffffffu, a.m, o);
            b.s = __shfl_xor_sync(0xffffffffu, a.s, o);
            b.u = __shfl_xor_sync(0xffffffffu, a.u, o);
            a.add(b);
        }
        if (lane == 0) sm.total = a;
    }
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    if (p.split > 1) cluster.sync();
    unsigned long long list = 0;
    if (rank == 0 && p.top > 0) {
        list = p.split == 1 ? sm.best[lane] : 0ull;
        if (p.split > 1) {  // a warp takes the lists of two CTAs
            static_assert(2 * kWarps >= kMaxCluster, "two lists per warp");
            if (warp < p.split) list = cluster.map_shared_rank(&sm, warp)->best[lane];
            if (warp + kWarps < p.split) list = merged(list, cluster.map_shared_rank(&sm, warp + kWarps)->best[lane]);
            list = merged_over_warps(list, kWarps, sm.list);
        }
    }
    if (rank == 0 && warp == 0) {
        if (p.split > 1) {  // a lane per CTA
            a = lane < p.split ? cluster.map_shared_rank(&sm, lane)->total : Sums::none();
#pragma unroll
            for (int o = kMaxCluster / 2; o > 0; o >>= 1) {
                Sums b;
                b.m = __shfl_xor_sync(0xffffffffu, a.m, o);
                b.s = __shfl_xor_sync(0xffffffffu, a.s, o);
                b.u = __shfl_xor_sync(0xffffffffu, a.u, o);
                a.add(b);
            }
        }
        a.m = __shfl_sync(0xffffffffu, a.m, 0), a.s = __shfl_sync(0xffffffffu, a.s, 0), a.u = __shfl_sync(0xffffffffu, a.u, 0);
        const bool empty = a.s == 0.f;  // every logit is -inf
        const float ls = logf(a.s);
        if (lane == 0) {
            const long long t = target_of(p.targets, p.targets64, row);
            float lp = 0.f;
            if (t >= 0 && t < p.V) lp = empty ? -INFINITY : (logit<kF32>(p.x, (long long)row * p.ld + t) - a.m) - ls;
            if (p.log_prob) p.log_prob[row] = lp;
            if (p.entropy) p.entropy[row] = empty ? 0.f : ls - a.u / a.s;
            if (p.lse) p.lse[row] = empty ? -INFINITY : a.m + ls;
        }
        if (p.top > 0) {
            if (lane < p.top) {
                const float x = from_order_bits((uint32_t)(list >> 32));
                p.top_ids[(long long)row * p.top + lane] = 0x7fffffff - (int)(uint32_t)list;
                p.top_log_probs[(long long)row * p.top + lane] = empty ? -INFINITY : (x - a.m) - ls;
            }
        }
    }
    if (p.split > 1) cluster.sync();  // no CTA leaves while its shared memory is read
}

constexpr int kGradThreads = 256;
constexpr int kGradVectors = 4;  // 16-byte vectors per thread
// lse in fp32 is off by up to |lse| 2^-24, and so is each p = e^(x - lse), relatively: 2^-12 at this size
constexpr float kFarLse = 4096.f;

// One pass: a CTA takes a stretch of a row.  kAligned: the rows of both arrays start equally far from a
// 16-byte boundary, so vectors of one are vectors of the other; else element by element.
// Where lse is far from zero (at the worst in a row masked whole with the type's lowest value, where it has no digit left
// for log V) the row's first CTA takes all of it, adds up e^(x - lse) before it writes, and divides by that sum: alone,
// since the gradient may go where the logits are.  (One such row of 100352 fp32 logits takes 69 us a call, where one near
// zero takes 16; 1023 of them 297 against 119.)
template <bool kF32, bool kAligned>
__global__ void __launch_bounds__(kGradThreads) grad_kernel(const GradParams p) {
    pdl_enter();
    const int row = (int)(blockIdx.x / (unsigned)p.chunks), chunk = (int)(blockIdx.x % (unsigned)p.chunks);
    const long long base = (long long)row * p.ld, dbase = (long long)row * p.dx_ld;
    const long long t = target_of(p.targets, p.targets64, row);
    const bool has = t >= 0 && t < p.V;
    const float g = has && p.d_log_prob ? p.d_log_prob[row] : 0.f;
    const float h = p.d_entropy ? p.d_entropy[row] : 0.f;
    const float lse = p.lse[row], ent = p.entropy ? p.entropy[row] : 0.f;
    const bool empty = lse == -INFINITY;
    auto grad = [&](float x, int j, float rest) {  // rest: the log of the sum of e^(x - lse), 0 to lse's digits
        const float lp = max_nan((x - lse) - rest, kFar);  // (at -inf too: no weight, and no inf * 0)
        float d = -ex2_approx(lp * kLog2e) * fmaf(h, lp + ent, g);
        if (j == t) d += g;
        return empty ? 0.f : d;
    };
    auto put = [&](int j, float d) {
        if (kF32) static_cast<float*>(p.dx)[dbase + j] = d;
        else static_cast<__nv_bfloat16*>(p.dx)[dbase + j] = __float2bfloat16_rn(d);
    };
    constexpr int kN = Vec<kF32>::kN;
    constexpr int kPer = kGradThreads * kGradVectors;  // vectors per CTA
    const Row<kF32> r(p.x, base, p.V);
    const int vectors = r.vectors();
    uint4 y[kGradVectors];
    if (kAligned) {  // (asked for before anything waits for lse)
#pragma unroll
        for (int i = 0; i < kGradVectors; ++i) {
            const int v = chunk * kPer + i * kGradThreads + threadIdx.x;
            // (not __ldg: the gradient may go where the logits are)
            if (v < vectors && r.inside(v)) y[i] = *(reinterpret_cast<const uint4*>(r.base) + v);
        }
    }
    if (fabsf(lse) > kFarLse && !isinf(lse)) {
        if (chunk != 0) return;
        __shared__ float sums[kGradThreads / 32];
        float s = 0.f;
#pragma unroll 4
        for (int j = threadIdx.x; j < p.V; j += kGradThreads)
            s += ex2_approx(max_nan(logit<kF32>(p.x, base + j) - lse, kFar) * kLog2e);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = s;
        __syncthreads();
        s = 0.f;
        for (int w = 0; w < kGradThreads / 32; ++w) s += sums[w];
        const float rest = s > 0.f ? logf(s) : 0.f;  // (0: an lse that is not of these logits)
        for (int j0 = threadIdx.x; j0 < p.V; j0 += 4 * kGradThreads) {
            float x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = j0 + i * kGradThreads < p.V ? logit<kF32>(p.x, base + j0 + i * kGradThreads) : 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (j0 + i * kGradThreads < p.V) put(j0 + i * kGradThreads, grad(x[i], j0 + i * kGradThreads, rest));
        }
        return;
    }
    if (!kAligned) {
        const int j0 = chunk * kPer * kN, j1 = min(p.V, j0 + kPer * kN);
        for (int j = j0 + threadIdx.x; j < j1; j += kGradThreads) put(j, grad(logit<kF32>(p.x, base + j), j, 0.f));
        return;
    }
    char* out = static_cast<char*>(p.dx) + (dbase - r.skip) * (kF32 ? 4 : 2);
#pragma unroll
    for (int i = 0; i < kGradVectors; ++i) {
        const int v = chunk * kPer + i * kGradThreads + threadIdx.x;
        if (v >= vectors) continue;
        if (r.inside(v)) {
            const Vec<kF32> z = Row<kF32>::unpack(y[i]);
            float d[kN];
#pragma unroll
            for (int e = 0; e < kN; ++e) d[e] = grad(z.x[e], r.id(v, e), 0.f);
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = kF32 ? __float_as_uint(d[e % kN]) : pack_bf16x2(d[2 * e % kN], d[(2 * e + 1) % kN]);
            reinterpret_cast<uint4*>(out)[v] = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
            for (int e = 0; e < kN; ++e) {
                const int j = r.id(v, e);
                if (j >= 0 && j < p.V) put(j, grad(logit<kF32>(p.x, base + j), j, 0.f));
            }
        }
    }
}

}  // namespace logprobs
}  // namespace dt
