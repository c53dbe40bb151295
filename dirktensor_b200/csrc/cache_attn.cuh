// Attention of new tokens over the quantised K/V cache.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale * q . k_j - m),  m = max_j scale * q . k_j
//
// over the keys j < seq_len - q_len + t + 1 that query t of a sequence sees (its own token is
// the cache's last but q_len - t - 1), after all `prefix_len` keys of a prefix that every
// sequence shares.  Rows with no key, and padding rows t >= q_len, are written as zeros with
// m = l = 0.
#pragma once
#include <cooperative_groups.h>

#include "kv_cache.cuh"

namespace dt {
namespace cache_attn {

constexpr int kD = 128;

struct Params {
    kv::Cache c;
    const void* q;
    long long q_batch, q_token;  // strides in elements; heads are 128 apart
    void* o;                     // [B, T, heads, 128], q's type
    float* m_out;                // [B, T, heads] or null
    float* l_out;
    const int* table;            // [B, max_pages]
    long long table_stride;
    int max_pages;
    const int* seq_lens;         // [B] keys of each sequence in the cache
    const int* q_lens;           // [B] queries of each sequence (null: T)
    const int* prefix_pages;     // shared prefix, or null
    int prefix_len;
    int B, T, heads, group;      // heads = kv heads * group
    float scale;
    int split;                   // CTAs per work item: a cluster, or, with `parts`, on their own
    // Partial results in the workspace (null: none), one per query row and CTA of its item:
    // o relative to 2^m, and (m, l, largest score), for the join kernel.
    float* part_o;               // [n_parts][B * T * heads][128]
    float4* part_s;              // [n_parts][B * T * heads]
    int n_parts;                 // of them, `split` are this kernel's, from first_part on
    int first_part;
};

// One warp per query row, lane l holding dims 4l .. 4l + 3, keys one after another.
template <int kFmt, bool kF32>
__global__ void __launch_bounds__(128) row_kernel(const Params p) {
    pdl_enter();
    const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (row >= (long long)p.B * p.T * p.heads) return;
    const int lane = threadIdx.x & 31;
    const int h = (int)(row % p.heads);
    const int t = (int)(row / p.heads % p.T);
    const int b = (int)(row / p.heads / p.T);
    const int hk = h / p.group;
    const int q_len = p.q_lens ? min(p.q_lens[b], p.T) : p.T;
    const long long cap = (long long)p.max_pages << p.c.page_shift;
    const long long seen = p.max_pages > 0 ? (long long)p.seq_lens[b] - q_len + t + 1 : 0;  // (lengths may be null then)
    const int own = t < q_len ? (int)max(0ll, min(seen, cap)) : 0;
    const int shared = t < q_len ? p.prefix_len : 0;
    float q[4] = {0.f, 0.f, 0.f, 0.f};
    const long long at = (long long)b * p.q_batch + (long long)t * p.q_token + h * kD + 4 * lane;
    if (kF32) {
        const float4 x = *reinterpret_cast<const float4*>(static_cast<const float*>(p.q) + at);
        q[0] = x.x, q[1] = x.y, q[2] = x.z, q[3] = x.w;
    } else {
        const uint2 x = *reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(p.q) + at);
        q[0] = __uint_as_float(x.x << 16), q[1] = __uint_as_float(x.x & 0xffff0000u);
        q[2] = __uint_as_float(x.y << 16), q[3] = __uint_as_float(x.y & 0xffff0000u);
    }
    float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int j = 0; j < shared + own; ++j) {
        const bool pre = j < shared;
        const int pos = pre ? j : j - shared;
        const int* table = pre ? p.prefix_pages : p.table + (long long)b * p.table_stride;
        const int page = table[pos >> p.c.page_shift];
        if (page < 0 || page >= p.c.pages) continue;
        const long long r = kv::row_of(p.c, page, hk, pos);
        float k[4], v[4];
        kv::decode4<kFmt>(reinterpret_cast<const uint32_t*>(p.c.k + r * kD)[lane], k);
        float s = q[0] * k[0] + q[1] * k[1] + q[2] * k[2] + q[3] * k[3];
#pragma unroll
        for (int w = 16; w > 0; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
        s *= p.c.ks[r] * p.scale;
        const float mn = fmaxf(m, s);
        const float a = expf(m - mn), e = expf(s - mn);
        kv::decode4<kFmt>(reinterpret_cast<const uint32_t*>(p.c.v + r * kD)[lane], v);
        const float ev = e * p.c.vs[r];
        l = l * a + e;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = o[i] * a + ev * v[i];
        m = mn;
    }
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
    if (kF32) {
        reinterpret_cast<float4*>(static_cast<float*>(p.o) + row * kD)[lane] =
            make_float4(o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
    } else {
        reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.o) + row * kD)[lane] =
            make_uint2(pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv));
    }
    if (lane == 0) {
        const bool any = l > 0.f || l != l;
        if (p.m_out) p.m_out[row] = any ? m : 0.f;
        if (p.l_out) p.l_out[row] = any ? l : 0.f;
    }
}

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kSub = 16;      // keys of an MMA step: the smallest page, so these share a page
constexpr int kTile = 32;     // keys per warp and step
constexpr int kStages = 2;    // tiles of a warp: one in use, one in flight
constexpr int kMaxCluster = 8;
constexpr float kGrow = 8.f;  // the running maximum moves when a score passes it by this much (log2)
constexpr float kLog2e = 1.4426950408889634f;

// One tile of one warp.  Every lane copies the 16-byte pieces that it will read itself, at
// [piece][lane], so that reads have no bank conflicts and K and V need no exchange; the scales
// are read by all lanes.
struct Stage {
    uint4 k[8][32];
    uint4 v[8][32];
    float4 scales[16];  // K's of the tile's keys, four by four, then V's
};

struct Smem {
    Stage ring[kWarps][kStages];  // afterwards each warp's rows, [rows][kD] fp32, at its first stage
    float m[kWarps][16];          // running maxima that the warps' sums refer to (log2 units)
    float l[kWarps][16];
    float mx[kWarps][16];         // largest score
    float om[16], ol[16], omx[16];  // the CTA's own, for the cluster; its rows are at ring[0][1]
};
static_assert(sizeof(Stage) >= 16 * kD * 4, "16 rows fit into a stage");
static_assert(3 * (sizeof(Smem) + 1024) <= 227 * 1024, "three CTAs per SM");

__device__ __forceinline__ void cp16(void* dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// D (16 x 8, fp32) += A (16 x 16, fp16) B (16 x 8, fp16)
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) { return __byte_perm(a, b, sel); }

// Codes as fp16 pairs, exactly: (bytes 0, 1) and (bytes 2, 3) of a word.  int8: with the sign
// bit flipped a byte bb is the code plus 128, and 0x64bb is 1024 + bb in fp16.
template <int kFmt>
__device__ __forceinline__ void pairs_of_word(uint32_t w, uint32_t& lo, uint32_t& hi) {
    if (kFmt == kv::kInt8) {
        const uint32_t x = w ^ 0x80808080u;
        const __half2 bias = __half2half2(__ushort_as_half(0x6480));
        const uint32_t a = prmt(x, 0x64646464u, 0x4140), b = prmt(x, 0x64646464u, 0x4342);
        const __half2 ra = __hsub2(*reinterpret_cast<const __half2*>(&a), bias);
        const __half2 rb = __hsub2(*reinterpret_cast<const __half2*>(&b), bias);
        lo = *reinterpret_cast<const uint32_t*>(&ra);
        hi = *reinterpret_cast<const uint32_t*>(&rb);
    } else {
        asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
            : "=r"(lo), "=r"(hi)
            : "r"(w));
    }
}

// The pairs (byte d of x, byte d of y) for d = 2i and 2i + 1.
template <int kFmt>
__device__ __forceinline__ void pairs_across(uint32_t x, uint32_t y, int i, uint32_t& even, uint32_t& odd) {
    pairs_of_word<kFmt>(prmt(x, y, i == 0 ? 0x5140 : 0x7362), even, odd);
}

__device__ __forceinline__ uint32_t half_pair(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float2 half_values(uint32_t h) { return __half22float2(*reinterpret_cast<const __half2*>(&h)); }
// The pair and what its rounding left, again as a pair.
__device__ __forceinline__ void split_pair(float a, float b, uint32_t& hi, uint32_t& lo) {
    hi = half_pair(a, b);
    const float2 f = half_values(hi);
    lo = half_pair(a - f.x, b - f.y);
}

__device__ __forceinline__ float quad_max(float x) {
    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
    return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
}
__device__ __forceinline__ float quad_sum(float x) {
    x += __shfl_xor_sync(0xffffffffu, x, 1);
    return x + __shfl_xor_sync(0xffffffffu, x, 2);
}

// 2^e for e in [-126, 127]
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }
// floor(log2 |x|) of a normal number
__device__ __forceinline__ int exponent(float x) { return ((__float_as_int(x) >> 23) & 0xff) - 127; }

// Sums of p and of p * v over parts that each refer to a maximum of their own.
struct Joined {
    float l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    // a part with sums (pl, po) relative to 2^pm, best the largest of all pm
    __device__ __forceinline__ void add(float pm, float pl, float best, float4 po) {
        if (pm == -INFINITY && pl == pl) return;                 // it saw no key
        const float a = pl != pl ? pl : ex2_approx(pm - best);  // (scores that are all NaN leave pm at -inf)
        l += pl * a;
        o.x += po.x * a, o.y += po.y * a, o.z += po.z * a, o.w += po.w * a;
    }
};

// Four dims of an output row, and from lane 0 its statistics.
template <bool kF32>
__device__ __forceinline__ void store_row(const Params& p, long long row, int lane, const Joined& y, float best, float big) {
    const bool any = y.l > 0.f || y.l != y.l;
    const float inv = any ? 1.f / y.l : 0.f;
    if (kF32)
        reinterpret_cast<float4*>(static_cast<float*>(p.o) + row * kD)[lane] =
            make_float4(y.o.x * inv, y.o.y * inv, y.o.z * inv, y.o.w * inv);
    else
        reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.o) + row * kD)[lane] =
            make_uint2(pack_bf16x2(y.o.x * inv, y.o.y * inv), pack_bf16x2(y.o.z * inv, y.o.w * inv));
    if (lane == 0) {
        if (p.m_out) p.m_out[row] = any ? big / kLog2e : 0.f;
        if (p.l_out) p.l_out[row] = any ? y.l * ex2_approx(best - big) : 0.f;
    }
}

// Split attention over the cache.  `split` CTAs take 8 or 16 query rows of one sequence and K/V
// head; their warps take the sequence's 32-key tiles in turn, keep their own running softmax, and
// are joined in shared memory, then over the CTAs' cluster or, where more CTAs than a cluster
// holds share few rows, through the workspace by join_kernel.
//
// Both products run on the tensor cores as m16n8k16 with the queries as the 16 rows.  8 rows:
// MMA rows 0-7 are fp16(q), rows 8-15 the rest q - fp16(q), so that fp32 queries lose nothing (bf16
// queries fit the first part; each row is scaled by a power of two into fp16's range first), and
// the weights p * v_scale are split the same way for the second product.  16 rows (kWide: bf16
// queries, more than 8 of them per K/V head, whose keys would be read twice otherwise): the weights
// are rounded to fp16 once, at 2^-11 well below the bf16 result's own 2^-8.  Codes are exact in fp16.
//
// The k and n indices of an MMA may be permuted freely if both operands agree, which saves every
// exchange.  Lane 4g + t holds, of each 16-key half of a tile,
//   K: keys 4 (g / 2) + 2 i + g % 2 (i = 0, 1: column g of 8-key block i), dims 16 (4 hf + t) ..+15;
//   S: query g, keys 4t .. 4t + 3 (columns 2t, 2t + 1 of block 0, then of block 1);
//   V: keys 4t .. 4t + 3, dims 16 g ..+15.
template <int kFmt, bool kF32, bool kWide>
__global__ void __launch_bounds__(kThreads, 3) split_kernel(const Params p) {
    static_assert(!(kF32 && kWide), "fp32 queries take both halves of the MMA rows");
    pdl_enter();
    constexpr int kSets = kWide ? 2 : 1;  // query rows per lane: g, and g + 8
    constexpr int kRows = 8 * kSets;
    extern __shared__ __align__(16) uint8_t smem_raw[];
    Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    const int rank = (int)(blockIdx.x % (unsigned)p.split);
    const int item = (int)(blockIdx.x / (unsigned)p.split);
    const int per_head = (p.T * p.group + kRows - 1) / kRows;
    const int hk = item / per_head % p.c.heads;
    const int b = item / per_head / p.c.heads;
    const int row0 = item % per_head * kRows;

    // this lane's query rows, and how many keys they and the CTA's rows see
    const int q_len = p.q_lens ? min(p.q_lens[b], p.T) : p.T;
    const long long cap = (long long)p.max_pages << p.c.page_shift;
    const long long base = p.max_pages > 0 ? (long long)p.seq_lens[b] - q_len + 1 : 0;  // (lengths may be null then)
    int lim[kSets], keys = 0;
#pragma unroll
    for (int z = 0; z < kSets; ++z) {
        const int r = row0 + g + 8 * z;
        const int tq = r / p.group;
        lim[z] = tq < q_len && p.max_pages > 0 ? (int)max(0ll, min(base + tq, cap)) : 0;
        if (r >= p.T * p.group) lim[z] = 0x7fffffff;  // (an MMA row that no query fills: nothing to mask, and never stored)
        else keys = max(keys, lim[z]);
    }
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) keys = max(keys, __shfl_xor_sync(0xffffffffu, keys, o));
    const int tiles = (keys + kTile - 1) / kTile;
    const int step = p.split * kWarps;
    const int first = rank * kWarps + warp;

    // Pages of a tile's two halves (-1 where there is none), looked up a step ahead.
    const int* table = p.table + (long long)b * p.table_stride;
    const int shift = p.c.page_shift;
    auto page_at = [&](int tile, int half) {
        const int key = tile * kTile + half * kSub;
        return tile < tiles && key < keys ? __ldg(table + (key >> shift)) : -1;
    };
    Stage* ring = sm.ring[warp];
    const int in_page = (1 << shift) - 1;
    const uint8_t* k_lane = p.c.k + (4 * (g >> 1) + (g & 1)) * kD + t * 16;
    const uint8_t* v_lane = p.c.v + (4 * t) * kD + g * 16;
    // (lanes 0-7 copy K's scales, 8-15 V's: four keys each, the first half of the tile first)
    const float* s_lane = (lane < 8 ? p.c.ks : p.c.vs) + 4 * (lane & 3);
    // Starts the copies of a tile's halves whose pages exist; returns which.
    auto issue = [&](int tile, int page0, int page1, int slot) {
        Stage& st = ring[slot];
        uint32_t ok = 0;
#pragma unroll
        for (int a = 0; a < 2; ++a) {
            const int page = a ? page1 : page0;
            if (page >= 0 && page < p.c.pages) {
                ok |= 1u << a;
                const int off = (tile * kTile + a * kSub) & in_page;
                const long long row = (((long long)page * p.c.heads + hk) << shift) + off;
                const uint8_t* k = k_lane + row * kD;
                const uint8_t* v = v_lane + row * kD;
#pragma unroll
                for (int i = 0; i < 4; ++i) cp16(&st.k[4 * a + i][lane], k + (i >> 1) * 2 * kD + (i & 1) * 64);
#pragma unroll
                for (int i = 0; i < 4; ++i) cp16(&st.v[4 * a + i][lane], v + i * kD);
                if (lane < 16 && ((lane >> 2) & 1) == a) cp16(&st.scales[lane], s_lane + row);
            }
        }
        cp_commit();
        return ok;
    };

    int pages[2] = {page_at(first, 0), page_at(first, 1)};
    int ahead[2] = {page_at(first + step, 0), page_at(first + step, 1)};
    uint32_t have = issue(first, pages[0], pages[1], 0);

    // the query rows, scaled by a power of two to at most 2^14, as fp16 (and what that leaves)
    uint32_t qa[2][16];     // MMA rows g and g + 8
    float factor[kSets];    // back from the scaled products to scores in log2 units
#pragma unroll
    for (int z = 0; z < kSets; ++z) {
        const int r = row0 + g + 8 * z;
        const bool in = r < p.T * p.group;
        const int tq = in ? r / p.group : 0;
        const int h = hk * p.group + (in ? r % p.group : 0);
        const long long at = (long long)b * p.q_batch + (long long)tq * p.q_token + (long long)h * kD;
        float x[32];
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
            const int d0 = 16 * (4 * hf + t);
            if (kF32) {
                const float4* src = reinterpret_cast<const float4*>(static_cast<const float*>(p.q) + at + d0);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float4 y = in ? src[i] : make_float4(0.f, 0.f, 0.f, 0.f);
                    x[16 * hf + 4 * i] = y.x, x[16 * hf + 4 * i + 1] = y.y, x[16 * hf + 4 * i + 2] = y.z, x[16 * hf + 4 * i + 3] = y.w;
                }
            } else {
                const uint4* src = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.q) + at + d0);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint4 y = in ? src[i] : make_uint4(0, 0, 0, 0);
                    const uint32_t w[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        x[16 * hf + 8 * i + 2 * e] = __uint_as_float(w[e] << 16);
                        x[16 * hf + 8 * i + 2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
                    }
                }
            }
        }
        // largest magnitude as an integer: infinities and NaNs order above every finite value
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 32; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const bool finite = top < 0x7f800000u;
        const int e = finite ? max(exponent(__uint_as_float(top)), -100) : 0;
        const float mul = finite ? pow2(13 - e) : 0.f;
        factor[z] = finite ? pow2(e - 13) * p.scale * kLog2e : __uint_as_float(0x7fffffffu);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float a = finite ? x[2 * i] * mul : 0.f, c = finite ? x[2 * i + 1] * mul : 0.f;
            if (kF32) split_pair(a, c, qa[0][i], qa[1][i]);
            else qa[z][i] = half_pair(a, c);
            if (!kF32 && !kWide) qa[1][i] = 0u;
        }
    }

    float acc[16][4];
#pragma unroll
    for (int j = 0; j < 16; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[j][e] = 0.f;
    float m[kSets], l[kSets], mx[kSets];
    float f[kSets];  // acc holds sums of p * v_scale * f: f keeps them in fp16's range
#pragma unroll
    for (int z = 0; z < kSets; ++z) m[z] = mx[z] = -INFINITY, l[z] = 0.f, f[z] = pow2(100);
    auto rescale = [&](int z, float a) {
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            acc[j][2 * z] *= a, acc[j][2 * z + 1] *= a;
            if (!kWide) acc[j][2] *= a, acc[j][3] *= a;
        }
    };

    uint32_t slot = 0;
    for (int tile = first; tile < tiles; tile += step) {
        const uint32_t now = have;
        __syncwarp();  // every lane is done with the other slot's scales
        have = issue(tile + step, ahead[0], ahead[1], slot ^ 1);
        ahead[0] = page_at(tile + 2 * step, 0);
        ahead[1] = page_at(tile + 2 * step, 1);
        cp_wait<1>();
        __syncwarp();
        const Stage& st = ring[slot];
        slot ^= 1;

        // scores: keys 4t .. 4t + 3 of either half (four chains of products side by side)
        float s[kSets][8], vv[8];
        {
            float d[4][4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) d[i][e] = 0.f;
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                uint32_t w[4][4];
#pragma unroll
                for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(w[i]) = st.k[2 * i + hf][lane];
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t b0, b1;
                        pairs_of_word<kFmt>(w[i][e], b0, b1);
                        const int q = 8 * hf + 2 * e;
                        mma_f16(d[i], qa[0][q], qa[1][q], qa[0][q + 1], qa[1][q + 1], b0, b1);
                    }
            }
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                const float4 ks = st.scales[4 * a + t], vs = st.scales[8 + 4 * a + t];
                const float kk[4] = {ks.x, ks.y, ks.z, ks.w};
                vv[4 * a] = vs.x, vv[4 * a + 1] = vs.y, vv[4 * a + 2] = vs.z, vv[4 * a + 3] = vs.w;
#pragma unroll
                for (int z = 0; z < kSets; ++z)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float* dd = d[2 * a + (i >> 1)];
                        const float y = kWide ? dd[2 * z + (i & 1)] : (kF32 ? dd[i & 1] + dd[2 + (i & 1)] : dd[i & 1]);
                        s[z][4 * a + i] = y * (kk[i] * factor[z]);
                    }
            }
        }
        const int key0 = tile * kTile + 4 * t;
        bool whole = now == 3u;
#pragma unroll
        for (int z = 0; z < kSets; ++z) whole &= tile * kTile + kTile <= lim[z];
        whole = __all_sync(0xffffffffu, whole);
        if (!whole) {  // hidden keys: past a row's last one, or on a page that does not exist
#pragma unroll
            for (int z = 0; z < kSets; ++z)
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (key0 + (i >> 2) * kSub + (i & 3) >= lim[z] || !((now >> (i >> 2)) & 1u)) s[z][i] = -INFINITY;
        }
        float top[kSets];
        bool grows = false;
#pragma unroll
        for (int z = 0; z < kSets; ++z) {
            const float* x = s[z];
            top[z] = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
            mx[z] = fmaxf(mx[z], top[z]);
            grows |= top[z] > m[z] + kGrow;
        }
        if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
            for (int z = 0; z < kSets; ++z) {
                const float best = quad_max(top[z]);
                if (best > m[z] + kGrow) {
                    const float a = m[z] == -INFINITY ? 0.f : ex2_approx(m[z] - best);
                    m[z] = best;
                    l[z] *= a;
                    rescale(z, a);
                }
            }
        }
        // weights p and p * v_scale; a hidden key weighs nothing, whatever its scale is
        float u[kSets][8], utop[kSets];
        grows = false;
#pragma unroll
        for (int z = 0; z < kSets; ++z) {
            const float m_safe = m[z] == -INFINITY ? 0.f : m[z];  // (no key seen yet: every weight is 2^-inf)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float w = ex2_approx(s[z][i] - m_safe);
                l[z] += w;
                u[z][i] = w * vv[i];
            }
            if (!whole) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (s[z][i] == -INFINITY) u[z][i] = 0.f;
            }
            const float* x = u[z];
            utop[z] = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
            grows |= utop[z] * f[z] > 32768.f;
        }
        if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
            for (int z = 0; z < kSets; ++z) {
                const float best = quad_max(utop[z]);
                if (best * f[z] > 32768.f) {
                    const float fn = pow2(min(max(8 - exponent(best), -120), 100));
                    rescale(z, fn / f[z]);  // a power of two
                    f[z] = fn;
                }
            }
        }
#pragma unroll
        for (int a = 0; a < 2; ++a) {
            uint32_t a0, a1, a2, a3;
            if (kWide) {
                constexpr int y = kSets - 1;
                a0 = half_pair(u[0][4 * a] * f[0], u[0][4 * a + 1] * f[0]);
                a1 = half_pair(u[y][4 * a] * f[y], u[y][4 * a + 1] * f[y]);
                a2 = half_pair(u[0][4 * a + 2] * f[0], u[0][4 * a + 3] * f[0]);
                a3 = half_pair(u[y][4 * a + 2] * f[y], u[y][4 * a + 3] * f[y]);
            } else {
                split_pair(u[0][4 * a] * f[0], u[0][4 * a + 1] * f[0], a0, a1);
                split_pair(u[0][4 * a + 2] * f[0], u[0][4 * a + 3] * f[0], a2, a3);
            }
            uint4 v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = st.v[4 * a + i][lane];
            if (!whole) {  // codes of hidden keys may be anything, a NaN too
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (key0 + a * kSub + i >= keys || !((now >> a) & 1u)) v[i] = make_uint4(0, 0, 0, 0);
            }
            const uint32_t v0[4] = {v[0].x, v[0].y, v[0].z, v[0].w}, v1[4] = {v[1].x, v[1].y, v[1].z, v[1].w};
            const uint32_t v2[4] = {v[2].x, v[2].y, v[2].z, v[2].w}, v3[4] = {v[3].x, v[3].y, v[3].z, v[3].w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    uint32_t b0e, b0o, b1e, b1o;
                    pairs_across<kFmt>(v0[e], v1[e], i, b0e, b0o);
                    pairs_across<kFmt>(v2[e], v3[e], i, b1e, b1o);
                    mma_f16(acc[4 * e + 2 * i], a0, a1, a2, a3, b0e, b1e);
                    mma_f16(acc[4 * e + 2 * i + 1], a0, a1, a2, a3, b0o, b1o);
                }
        }
    }
    cp_wait<0>();
    __syncwarp();

    // join the warps: every warp's rows in units of 2^-m
#pragma unroll
    for (int z = 0; z < kSets; ++z) {
        const int row = g + 8 * z;
        const float lq = quad_sum(l[z]), mq = quad_max(mx[z]);
        const float inv = 1.f / f[z];
        // (the 16-byte pieces of a 128-byte span are exchanged by 2t + row: no bank conflicts)
        float* o = reinterpret_cast<float*>(ring) + row * kD;
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int j = 0; j < 16; j += 4) {
                const int piece = 8 * t + ((4 * c + (j >> 2)) ^ ((2 * t + g) & 7));
                float y[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = (kWide ? acc[j + e][2 * z + c] : acc[j + e][c] + acc[j + e][c + 2]) * inv;
                *reinterpret_cast<float4*>(o + 4 * piece) = make_float4(y[0], y[1], y[2], y[3]);
            }
        if (t == 0) sm.m[warp][row] = m[z], sm.l[warp][row] = lq, sm.mx[warp][row] = mq;
    }
    __syncthreads();
    const int rows = min(kRows, p.T * p.group - row0);
    float* mine = reinterpret_cast<float*>(&sm.ring[0][1]);
    for (int row = warp; row < rows; row += kWarps) {  // a warp per row, four dims a lane
        const int piece = (lane & 24) + ((lane & 7) ^ ((2 * (lane >> 3) + row) & 7));
        float best = -INFINITY, big = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) best = fmaxf(best, sm.m[w][row]), big = fmaxf(big, sm.mx[w][row]);
        Joined y;
#pragma unroll
        for (int w = 0; w < kWarps; ++w)
            y.add(sm.m[w][row], sm.l[w][row], best,
                  *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(sm.ring[w]) + row * kD + 4 * piece));
        if (p.part_o) {
            const int rr = row0 + row;
            const long long out = ((long long)b * p.T + rr / p.group) * p.heads + hk * p.group + rr % p.group;
            const long long at = (long long)(p.first_part + rank) * p.B * p.T * p.heads + out;
            reinterpret_cast<float4*>(p.part_o + at * kD)[lane] = y.o;
            if (lane == 0) p.part_s[at] = make_float4(best, y.l, big, 0.f);
        } else {
            reinterpret_cast<float4*>(mine + row * kD)[lane] = y.o;
            if (lane == 0) sm.om[row] = best, sm.ol[row] = y.l, sm.omx[row] = big;
        }
    }
    if (p.part_o) return;
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    if (p.split > 1) cluster.sync();
    else __syncthreads();

    // join the cluster: its CTAs share the rows' elements
    for (int i = rank * kThreads + threadIdx.x; i < rows * (kD / 4); i += p.split * kThreads) {
        const int row = i >> 5;
        const int rr = row0 + row;
        float best = -INFINITY, big = -INFINITY;
        for (int c = 0; c < p.split; ++c) {
            const Smem* other = p.split > 1 ? cluster.map_shared_rank(&sm, c) : &sm;
            best = fmaxf(best, other->om[row]), big = fmaxf(big, other->omx[row]);
        }
        Joined y;
        for (int c = 0; c < p.split; ++c) {
            const Smem* other = p.split > 1 ? cluster.map_shared_rank(&sm, c) : &sm;
            y.add(other->om[row], other->ol[row], best,
                  reinterpret_cast<const float4*>(reinterpret_cast<const float*>(&other->ring[0][1]) + row * kD)[lane]);
        }
        store_row<kF32>(p, ((long long)b * p.T + rr / p.group) * p.heads + hk * p.group + rr % p.group, lane, y, best, big);
    }
    if (p.split > 1) cluster.sync();  // no CTA leaves while another reads its shared memory
}

// Joins the parts of each query row: a warp per row, four dims a lane.
template <bool kF32>
__global__ void __launch_bounds__(128) join_kernel(const Params p) {
    pdl_enter();
    const long long rows = (long long)p.B * p.T * p.heads;
    const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (row >= rows) return;
    float best = -INFINITY, big = -INFINITY;
    for (int i = lane; i < p.n_parts; i += 32) {
        const float4 s = p.part_s[i * rows + row];
        best = fmaxf(best, s.x), big = fmaxf(big, s.z);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
    }
    Joined y;
#pragma unroll 8
    for (int i = 0; i < p.n_parts; ++i) {
        const float4 s = p.part_s[i * rows + row];
        y.add(s.x, s.y, best, reinterpret_cast<const float4*>(p.part_o + (i * rows + row) * kD)[lane]);
    }
    store_row<kF32>(p, row, lane, y, best, big);
}

}  // namespace cache_attn
}  // namespace dt
