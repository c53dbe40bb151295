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
    int split;                   // CTAs (one cluster) per work item
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

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kRows = 8;      // query rows (of one K/V head) that a CTA takes
constexpr int kTile = 16;     // keys per warp and step: the smallest page, so a tile has one page
constexpr int kStages = 3;    // tiles of a warp in flight or in use
constexpr int kMaxSplit = 16;
constexpr float kGrow = 8.f;  // the running maximum moves when a score passes it by this much (log2)
constexpr float kLog2e = 1.4426950408889634f;

// One tile of one warp.  Every lane copies the 16-byte pieces that it will read itself, at
// [piece][lane], so that reads have no bank conflicts and K and V need no exchange; the scales
// are read by all lanes.
struct Stage {
    uint4 k[4][32];
    uint4 v[4][32];
    float4 ks[4];
    float4 vs[4];
};

struct Smem {
    Stage ring[kWarps][kStages];  // afterwards each warp's rows, [kRows][kD] fp32, at its first stage
    float m[kWarps][kRows];       // running maxima that the warps' sums refer to (log2 units)
    float l[kWarps][kRows];
    float mx[kWarps][kRows];      // largest score
    float om[kRows], ol[kRows], omx[kRows];  // the CTA's own, for the cluster
    float o[kRows][kD];
};
static_assert(sizeof(Stage) >= kRows * kD * 4, "a warp's rows fit into its first stage");

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
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) { return __byte_perm(a, b, sel); }

// fp16 pairs from codes: (bytes 0, 1) and (bytes 2, 3) of a word.  int8: 0x64bb is 1024 + bb in
// fp16, so with the sign bit flipped the byte is a number plus 1152, exactly.
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

// fp16 pairs (byte 2i of x, byte 2i of y) and (byte 2i + 1 of x, byte 2i + 1 of y).
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

// Split attention over the cache.  A cluster of `split` CTAs takes kRows query rows of one
// sequence and K/V head; its warps take the sequence's 16-key tiles in turn, keep their own
// running softmax, and are joined in shared memory, then over the cluster.
//
// Both products run on the tensor cores as m16n8k16 with the queries as the 16 rows: rows 0-7
// are fp16(q), rows 8-15 the rest q - fp16(q), so that fp32 queries lose nothing (bf16 queries fit the
// first part; each row is scaled by a power of two into fp16's range first).  The weights
// p * v_scale are split the same way for the second product.  Codes are exact in fp16.
//
// The k and n indices of an MMA may be permuted freely if both operands agree, which saves every
// exchange.  Lane 4g + t holds, of a 16-key tile,
//   K: keys 4 (g / 2) + 2 i + g % 2 (i = 0, 1: column g of 8-key block i), dims 16 (4 hf + t) ..+15;
//   S: query g, keys 4t .. 4t + 3 (columns 2t, 2t + 1 of block 0, then of block 1);
//   V: keys 4t .. 4t + 3, dims 16 g ..+15.
template <int kFmt, bool kF32>
__global__ void __launch_bounds__(kThreads, 2) split_kernel(const Params p) {
    pdl_enter();
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

    // this lane's query row, and how many keys it and the CTA's rows see
    const int r = row0 + g;
    const bool row_in = r < p.T * p.group;
    const int tq = row_in ? r / p.group : 0;
    const int h = hk * p.group + (row_in ? r % p.group : 0);
    const int q_len = p.q_lens ? min(p.q_lens[b], p.T) : p.T;
    const long long cap = (long long)p.max_pages << p.c.page_shift;
    const long long base = p.max_pages > 0 ? (long long)p.seq_lens[b] - q_len + 1 : 0;  // (lengths may be null then)
    const int lim = row_in && tq < q_len && p.max_pages > 0 ? (int)max(0ll, min(base + tq, cap)) : 0;
    int keys = lim;
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) keys = max(keys, __shfl_xor_sync(0xffffffffu, keys, o));
    const int tiles = (keys + kTile - 1) / kTile;
    const int step = p.split * kWarps;
    const int first = rank * kWarps + warp;
    const int* table = p.table + (long long)b * p.table_stride;

    Stage* ring = sm.ring[warp];
    const int tiles_per_page_shift = p.c.page_shift - 4;
    auto page_at = [&](int tile) { return tile < tiles ? __ldg(table + (tile >> tiles_per_page_shift)) : -1; };
    // starts the copies of a tile; false (and nothing copied) where its page does not exist
    auto issue = [&](int tile, int page, int slot) {
        const bool ok = tile < tiles && page >= 0 && page < p.c.pages;
        if (ok) {
            Stage& s = ring[slot];
            const long long row = kv::row_of(p.c, page, hk, tile * kTile);
            const uint8_t* k = p.c.k + row * kD + (4 * (g >> 1) + (g & 1)) * kD + t * 16;
            const uint8_t* v = p.c.v + row * kD + (4 * t) * kD + g * 16;
#pragma unroll
            for (int i = 0; i < 4; ++i) cp16(&s.k[i][lane], k + (i >> 1) * 2 * kD + (i & 1) * 64);
#pragma unroll
            for (int i = 0; i < 4; ++i) cp16(&s.v[i][lane], v + i * kD);
            if (lane < 4) cp16(&s.ks[lane], p.c.ks + row + 4 * lane);
            else if (lane < 8) cp16(&s.vs[lane - 4], p.c.vs + row + 4 * (lane - 4));
        }
        cp_commit();
        return ok;
    };

    int page = page_at(first);
    uint32_t live = 0;  // bit s: slot s holds a tile
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) {
        const int next = page_at(first + (s + 1) * step);
        live |= (uint32_t)issue(first + s * step, page, s) << s;
        page = next;
    }

    // the query row, scaled by a power of two to at most 2^14, as fp16 and what is left
    uint32_t qh[16], ql[kF32 ? 16 : 1];
    float factor;  // back from the scaled products to scores in log2 units
    {
        float amax = 0.f;
        bool finite = true;
        const long long at = (long long)b * p.q_batch + (long long)tq * p.q_token + (long long)h * kD;
        float x[32];
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
            const int d0 = 16 * (4 * hf + t);
            if (kF32) {
                const float4* src = reinterpret_cast<const float4*>(static_cast<const float*>(p.q) + at + d0);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float4 y = row_in ? src[i] : make_float4(0.f, 0.f, 0.f, 0.f);
                    x[16 * hf + 4 * i] = y.x, x[16 * hf + 4 * i + 1] = y.y, x[16 * hf + 4 * i + 2] = y.z, x[16 * hf + 4 * i + 3] = y.w;
                }
            } else {
                const uint4* src = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.q) + at + d0);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint4 y = row_in ? src[i] : make_uint4(0, 0, 0, 0);
                    const uint32_t w[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        x[16 * hf + 8 * i + 2 * e] = __uint_as_float(w[e] << 16);
                        x[16 * hf + 8 * i + 2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
                    }
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            amax = fmaxf(amax, fabsf(x[i]));
            finite &= fabsf(x[i]) <= 3.402823466e38f;
        }
        amax = quad_max(amax);
        finite = quad_sum(finite ? 0.f : 1.f) == 0.f;
        const int e = finite ? min(max(exponent(amax), -100), 126) : 0;
        const float mul = finite ? pow2(13 - e) : 0.f;
        factor = finite ? pow2(e - 13) * p.scale * kLog2e : __uint_as_float(0x7fffffffu);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float a = finite ? x[2 * i] * mul : 0.f, c = finite ? x[2 * i + 1] * mul : 0.f;
            if (kF32) split_pair(a, c, qh[i], ql[i]);
            else qh[i] = half_pair(a, c);
        }
    }

    float acc[16][4];
#pragma unroll
    for (int j = 0; j < 16; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[j][e] = 0.f;
    float m = -INFINITY, l = 0.f, mx = -INFINITY;
    float f = pow2(100);  // acc holds sums of p * v_scale * f: f keeps them in fp16's range

    int slot = 0;
    for (int tile = first; tile < tiles; tile += step) {
        {
            const int ahead = tile + (kStages - 1) * step;
            const int into = slot == 0 ? kStages - 1 : slot - 1;
            const int next = page_at(ahead + step);
            __syncwarp();  // every lane is done with that slot's scales
            const bool ok = issue(ahead, page, into);
            live = (live & ~(1u << into)) | ((uint32_t)ok << into);
            page = next;
        }
        cp_wait<kStages - 1>();
        __syncwarp();
        const Stage& st = ring[slot];
        const bool have = (live >> slot) & 1u;
        slot = slot + 1 == kStages ? 0 : slot + 1;
        if (!have) continue;  // a page that does not exist: none of its keys is seen

        // scores of keys 4t .. 4t + 3 for query g
        float s[4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                const uint4 w = st.k[2 * i + hf][lane];
                const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint32_t b0, b1;
                    pairs_of_word<kFmt>(ww[e], b0, b1);
                    const int q = 8 * hf + 2 * e;
                    mma_f16(d, qh[q], kF32 ? ql[kF32 ? q : 0] : 0u, qh[q + 1], kF32 ? ql[kF32 ? q + 1 : 0] : 0u, b0, b1);
                }
            }
            s[2 * i] = d[0] + d[2];
            s[2 * i + 1] = d[1] + d[3];
        }
        const float4 ks = st.ks[t], vs = st.vs[t];
        const float kk[4] = {ks.x, ks.y, ks.z, ks.w}, vv[4] = {vs.x, vs.y, vs.z, vs.w};
        const int key0 = tile * kTile + 4 * t;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            s[i] = s[i] * kk[i] * factor;
            if (key0 + i >= lim) s[i] = -INFINITY;
        }
        const float top = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
        mx = fmaxf(mx, top);
        if (__any_sync(0xffffffffu, top > m + kGrow)) {
            const float best = quad_max(top);
            if (best > m + kGrow) {
                const float a = m == -INFINITY ? 0.f : ex2_approx(m - best);
                m = best;
                l *= a;
#pragma unroll
                for (int j = 0; j < 16; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[j][e] *= a;
            }
        }
        float u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool out = s[i] == -INFINITY;  // (not a NaN: that has to come through)
            const float w = out ? 0.f : ex2_approx(s[i] - m);
            l += w;
            u[i] = out ? 0.f : w * vv[i];
        }
        const float utop = fmaxf(fmaxf(u[0], u[1]), fmaxf(u[2], u[3]));
        if (__any_sync(0xffffffffu, utop * f > 32768.f)) {
            const float best = quad_max(utop);
            if (best * f > 32768.f) {
                const float fn = pow2(min(max(8 - exponent(best), -120), 100));
                const float a = fn / f;  // a power of two
                f = fn;
#pragma unroll
                for (int j = 0; j < 16; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[j][e] *= a;
            }
        }
        uint32_t a0, a1, a2, a3;
        split_pair(u[0] * f, u[1] * f, a0, a1);
        split_pair(u[2] * f, u[3] * f, a2, a3);
        uint4 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = st.v[i][lane];
        if (tile * kTile + kTile > keys) {  // codes past the last key may be anything, a NaN too
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (key0 + i >= keys) v[i] = make_uint4(0, 0, 0, 0);
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
    cp_wait<0>();
    __syncwarp();

    // join the warps: every warp's rows in units of 2^-m
    {
        l = quad_sum(l);
        mx = quad_max(mx);
        const float inv = 1.f / f;
        float* o = reinterpret_cast<float*>(ring) + g * kD;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            o[32 * t + j] = (acc[j][0] + acc[j][2]) * inv;
            o[32 * t + 16 + j] = (acc[j][1] + acc[j][3]) * inv;
        }
        if (t == 0) sm.m[warp][g] = m, sm.l[warp][g] = l, sm.mx[warp][g] = mx;
    }
    __syncthreads();
    {
        const int row = warp;  // a warp per row, four dims a lane
        float best = -INFINITY, big = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) best = fmaxf(best, sm.m[w][row]), big = fmaxf(big, sm.mx[w][row]);
        float ls = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float mw = sm.m[w][row];
            const float a = mw == -INFINITY ? 0.f : ex2_approx(mw - best);
            const float4 y = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(sm.ring[w]) + row * kD + 4 * lane);
            const float lw = sm.l[w][row];
            if (mw != -INFINITY || lw != lw) {  // (scores that are all NaN leave the maximum at -inf)
                const float aw = lw != lw ? lw : a;
                ls += lw * aw;
                o.x += y.x * aw, o.y += y.y * aw, o.z += y.z * aw, o.w += y.w * aw;
            }
        }
        *reinterpret_cast<float4*>(&sm.o[row][4 * lane]) = o;
        if (lane == 0) sm.om[row] = best, sm.ol[row] = ls, sm.omx[row] = big;
    }
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    if (p.split > 1) cluster.sync();
    else __syncthreads();

    // join the cluster: its CTAs share the rows' elements
    for (int i = rank * kThreads + threadIdx.x; i < kRows * kD / 4; i += p.split * kThreads) {
        const int row = i / (kD / 4), d = 4 * (i % (kD / 4));
        const int rr = row0 + row;
        if (rr >= p.T * p.group) continue;
        float best = -INFINITY, big = -INFINITY;
        for (int c = 0; c < p.split; ++c) {
            const Smem* other = p.split > 1 ? cluster.map_shared_rank(&sm, c) : &sm;
            best = fmaxf(best, other->om[row]), big = fmaxf(big, other->omx[row]);
        }
        float ls = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int c = 0; c < p.split; ++c) {
            const Smem* other = p.split > 1 ? cluster.map_shared_rank(&sm, c) : &sm;
            const float mc = other->om[row], lc = other->ol[row];
            if (mc == -INFINITY && lc == lc) continue;
            const float a = lc != lc ? lc : ex2_approx(mc - best);
            const float4 y = *reinterpret_cast<const float4*>(&other->o[row][d]);
            ls += lc * a;
            o.x += y.x * a, o.y += y.y * a, o.z += y.z * a, o.w += y.w * a;
        }
        const bool any = ls > 0.f || ls != ls;
        const float inv = any ? 1.f / ls : 0.f;
        const int tt = rr / p.group, hh = hk * p.group + rr % p.group;
        const long long out = ((long long)b * p.T + tt) * p.heads + hh;
        if (kF32) {
            *reinterpret_cast<float4*>(static_cast<float*>(p.o) + out * kD + d) =
                make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
        } else {
            *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.o) + out * kD + d) =
                make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
        }
        if (d == 0) {
            if (p.m_out) p.m_out[out] = any ? big / kLog2e : 0.f;
            if (p.l_out) p.l_out[out] = any ? ls * ex2_approx(best - big) : 0.f;
        }
    }
    if (p.split > 1) cluster.sync();  // no CTA leaves while another reads its shared memory
}

}  // namespace cache_attn
}  // namespace dt
