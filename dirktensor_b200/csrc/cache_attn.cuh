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

// Query row r of a K/V head is query head r % group of token r / group.  (A group of one, the model's own case,
// spares the division, which takes some 30 instructions that are run for a few tiles only.)
__device__ __forceinline__ int token_of(int r, int group) { return group == 1 ? r : (int)((unsigned)r / (unsigned)group); }

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
    int split;                   // CTAs of a cluster per work item (split_kernel)
    int by_length;               // split_kernel takes the longest sequences first
    // Workspace of stream_kernel and join_kernel: partial sums of the CTAs and, of the prefix
    // kernel, of the shared keys.  Sums are relative to 2^m; statistics are (m, l, largest score, -).
    int shares;                  // CTAs that stream_kernel shares out (0: not launched, no keys but the prefix's)
    int* starts;                 // [B + 1] first CTA of each sequence, were each of one item
    float* part_o;               // [shares + items][rows of an item][128]
    float4* part_s;              // [shares + items][rows of an item]
    int n_shared;                // parts of the prefix
    float* shared_o;             // [n_shared][B * T * heads][128]
    float4* shared_s;            // [n_shared][B * T * heads]
};

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kSub = 16;       // keys of an MMA step: the smallest page, so these share a page
constexpr int kTile = 32;      // keys per warp and step
constexpr int kStages = 3;     // pieces (K or V of a tile) of a warp: one in use, two in flight
constexpr int kMaxCluster = 8;
constexpr float kGrow = 8.f;   // the running maximum moves when a score passes it by this much (log2)
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kFirstFactor = 118;  // log2 of the weights' factor before any: rows of 2^-100, the smallest kept, then weigh 2^8 or more

// K or V of one tile of one warp.  Every lane copies the 16-byte pieces that it will read itself,
// at [piece][lane], so that reads have no bank conflicts and need no exchange; the scales are read
// by all lanes.
struct Stage {
    uint4 d[8][32];
    float scale[kTile];
};

struct Smem {
    Stage ring[kWarps][kStages];    // afterwards each warp's rows, [rows][kD] fp32, from its start
    float m[kWarps][16];            // running maxima that the warps' sums refer to (log2 units)
    float l[kWarps][16];
    float mx[kWarps][16];           // largest score
    float om[16], ol[16], omx[16];  // the CTA's own, for the cluster
    // and its rows, behind the warps': eight at the end of each of the first two rings
    __device__ __forceinline__ float* joined(int row) {
        return reinterpret_cast<float*>(&ring[row >> 3][0]) + 16 * kD + (row & 7) * kD;
    }
};
static_assert(kStages * sizeof(Stage) >= 24 * kD * 4, "16 rows of a warp and 8 of the CTA fit into a ring");
static_assert(4 * (sizeof(Smem) + 1024) <= 227 * 1024, "four CTAs per SM");

// Query rows that a warp takes.  An MMA has eight columns for them; each lane has the scores of
// columns 2t and 2t + 1, so up to four queries sit in the even columns, at half the softmax work.
enum : int { kFew = 0, kEight = 1, kWide = 2 };  // 4, 8, or 16 in two sets of columns
constexpr int rows_of(int form) { return form == kFew ? 4 : form == kEight ? 8 : 16; }

// CTAs per SM: four where 128 registers a thread suffice; 16 rows spill at three (28 us instead of 26 for 16 x 2047 keys).
constexpr int ctas_per_sm(bool f32, int form) { return form == kWide ? 2 : f32 && form != kFew ? 3 : 4; }

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

// The transpose of an 8 x 8 matrix of 16-bit values, row g's columns 2t, 2t + 1 in lane 4g + t.
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// Over the eight lanes of one t.
__device__ __forceinline__ float column_max(float x) {
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
    return x;
}
__device__ __forceinline__ float column_sum(float x) {
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}

__device__ __forceinline__ float warp_max(float x) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
    return x;
}

// 2^e for e in [-126, 127]
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }
// 2^e for e <= 127, 0 where that is below the normal numbers
__device__ __forceinline__ float pow2_or_0(int e) { return e < -126 ? 0.f : pow2(e); }
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
    __device__ __forceinline__ void scale(float a) {
        l *= a;
        o.x *= a, o.y *= a, o.z *= a, o.w *= a;
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

// A warp's attention of 8 or 16 query rows of one sequence and K/V head over 32-key tiles
// tile0, tile0 + step, ... below tile1, with its own running softmax.
//
// Both products run on the tensor cores as m16n8k16 with the queries as the 8 columns:
//   S^T (16 keys x 8 queries) = K (16 keys x 16 dims) Q^T,  O^T (16 dims x 8 queries) = V^T (16 dims x 16 keys) P^T
// so that no row of an MMA is idle however few queries there are.  Codes are exact in fp16.  Queries
// are scaled row by row by a power of two into fp16's range, where bf16 values are exact; fp32 ones
// go in as fp16(q) and q - fp16(q), and so do their weights p * v_scale: in two columns, where there are
// four queries at most, else in two MMAs.  The weights of bf16 queries
// are rounded to fp16 once, at 2^-11 well below the result's own 2^-8.  More than 8 bf16 queries of
// a K/V head take two sets of columns (kWide), so that the keys are read and converted once.
//
// The k indices of an MMA may be permuted freely if both operands agree, and its rows if the result is
// read accordingly, which saves every exchange but the transpose of P.  Lane 4g + t holds, of
// each 16-key half of a tile,
//   K: keys g and g + 8, dims 16 (4 hf + t) ..+15;      S, P: keys g and g + 8, queries 2t and 2t + 1;
//   V: keys 2t, 2t + 1, 2t + 8, 2t + 9, dims 16 g ..+15;  O: dims 16 g ..+15, queries 2t and 2t + 1.
//
// Bound by the codes' read (256 bytes a key and head against 8 to 16 tensor products a query) and, next, by the
// latency of its own chain: a 32-key tile takes a warp some 650 instructions, 230 of them conversions.  64 sequences
// of 1024 to 4096 keys and 16 heads, 692 MB, take 132 us (5.25 TB/s, 0.82 of the measured copy); 512 keys
// of one sequence 6.1 us.  Keys as MMA columns and queries as rows, the first form, left half of each MMA idle and
// needed twice the accumulators (159 us); register-resident tiles without the ring were slower still (207 us).
template <int kForm>
struct State {
    static constexpr int kSets = kForm == kWide ? 2 : 1, kCols = kForm == kFew ? 1 : 2;
    float acc[kSets][8][4];  // of step j: dims 16g + 2j (0, 1) and 16g + 2j + 1 (2, 3), queries 2t (0, 2) and 2t + 1 (1, 3)
    float m[kSets][kCols];       // running maxima that the sums refer to (log2 units, whole numbers; -inf: no key seen)
    float l[kSets][kCols];       // this lane's share of the sums of p
    float mx[kSets][kCols];      // this lane's largest scores
    float f[kSets][kCols];       // acc holds sums of p * v_scale * f, f = 2^e: the largest so far lies in 2^8..2^15 (fp16)
    // dim 16g + d of query 2t + c (kFew: of query t, the sum of its two columns)
    __device__ __forceinline__ float sum(int z, int c, int d) const {
        const float* a = acc[z][d >> 1] + 2 * (d & 1);
        return kForm == kFew ? a[0] + a[1] : a[c];
    }
    __device__ __forceinline__ void rescale(int z, int c, float a) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            acc[z][j][c] *= a, acc[z][j][2 + c] *= a;
            if (kForm == kFew) acc[z][j][1] *= a, acc[z][j][3] *= a;
        }
    }
};

template <int kFmt, bool kF32, int kForm>
__device__ __forceinline__ void attend(const Params& p, Stage* ring, int b, int hk, int row0, int tile0, int tile1, int step,
                                       State<kForm>& st) {
    static_assert(!(kF32 && kForm == kWide), "fp32 queries have no wide form: twice the registers");
    constexpr int kSets = kForm == kWide ? 2 : 1, kCols = kForm == kFew ? 1 : 2;
    constexpr bool kBeside = kF32 && kForm == kFew;  // the rest of an fp32 query in the column beside it
    constexpr int kParts = kF32 && !kBeside ? 2 : 1;  // or in an MMA of its own
    const int lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;

    // the query of column g of each set, asked for first, since nothing else is needed to
    uint4 raw[kSets][kF32 ? 8 : 4];
#pragma unroll
    for (int z = 0; z < kSets; ++z) {
        const int r = row0 + (kCols == 1 ? g >> 1 : g) + 8 * z;
        const bool in = r < p.T * p.group && (kCols == 2 || kBeside || !(g & 1));
        const int tq = in ? token_of(r, p.group) : 0;
        const int h = hk * p.group + (in ? r - tq * p.group : 0);
        const long long at = (long long)b * p.q_batch + (long long)tq * p.q_token + (long long)h * kD + 16 * t;
        const uint4* src = kF32 ? reinterpret_cast<const uint4*>(static_cast<const float*>(p.q) + at)
                                : reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.q) + at);
        constexpr int kPieces = kF32 ? 4 : 2;  // of 16 dims
#pragma unroll
        for (int hf = 0; hf < 2; ++hf)
#pragma unroll
            for (int i = 0; i < kPieces; ++i)
                raw[z][kPieces * hf + i] = in ? __ldg(src + hf * 4 * kPieces + i) : make_uint4(0, 0, 0, 0);
    }
    // Pages of a tile's two halves (-1 past the table), looked up ahead: entries past the
    // sequence's keys may be anything, and are not followed.  From 32 tokens a page on, one serves both.
    const long long cap = (long long)p.max_pages << p.c.page_shift;
    const int* table = p.table + (long long)b * p.table_stride;
    const int shift = p.c.page_shift;
    auto page_at = [&](int tile, int (&page)[2]) {
        const int key = tile * kTile;
        page[0] = key < cap ? __ldg(table + (key >> shift)) : -1;
        page[1] = page[0];
        if (shift < 5) page[1] = key + kSub < cap ? __ldg(table + (key >> shift) + 1) : -1;
    };
    int pages[3][2];  // of the next tile, the one after it, and the one after that
#pragma unroll
    for (int i = 0; i < 3; ++i) page_at(tile0 + i * step, pages[i]);

    // how many keys this lane's queries 2t and 2t + 1, and all of the warp's, see
    const int q_len = p.q_lens ? min(p.q_lens[b], p.T) : p.T;
    const long long base = (long long)p.seq_lens[b] - q_len + 1;
    int lim[kSets][kCols], keys = 0, least = 0x7fffffff;
#pragma unroll
    for (int z = 0; z < kSets; ++z)
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
            const int r = row0 + kCols * t + c + 8 * z;
            const int tq = token_of(r, p.group);
            lim[z][c] = tq < q_len ? (int)max(0ll, min(base + tq, cap)) : 0;
            if (r >= p.T * p.group) lim[z][c] = 0x7fffffff;  // (a column that no query fills: nothing to mask, and never stored)
            else keys = max(keys, lim[z][c]);
            least = min(least, lim[z][c]);
        }
    keys = max(keys, __shfl_xor_sync(0xffffffffu, keys, 1));
    keys = max(keys, __shfl_xor_sync(0xffffffffu, keys, 2));
    least = min(least, __shfl_xor_sync(0xffffffffu, least, 1));
    least = min(least, __shfl_xor_sync(0xffffffffu, least, 2));
    tile1 = min(tile1, (int)(((long long)keys + kTile - 1) / kTile));

    // Which halves of a tile there are to read.
    auto halves = [&](int tile, const int (&page)[2]) {
        uint32_t ok = 0;
#pragma unroll
        for (int a = 0; a < 2; ++a)
            if (page[a] >= 0 && page[a] < p.c.pages && tile < tile1 && tile * kTile + a * kSub < keys) ok |= 1u << a;
        return ok;
    };
    const int in_page = (1 << shift) - 1;
    const uint8_t* k_lane = p.c.k + g * kD + t * 16;
    const uint8_t* v_lane = p.c.v + 2 * t * kD + g * 16;
    const float* ks_lane = p.c.ks + 4 * (lane & 3);
    const float* vs_lane = p.c.vs + 4 * (lane & 3);
    // Starts the copies of K or V of a tile's halves.  (A cache has fewer than 2^31 rows.)
    auto issue = [&](bool v, int tile, const int (&page)[2], uint32_t ok, int slot) {
        Stage& into = ring[slot];
        if (ok) {
            uint32_t row0 = ((uint32_t)(page[0] * p.c.heads + hk) << shift) + ((tile * kTile) & in_page);
            uint32_t row1 = ((uint32_t)(page[1] * p.c.heads + hk) << shift) + ((tile * kTile + kSub) & in_page);
            if (ok == 1u) row1 = row0;  // (the other half again, and hidden)
            if (ok == 2u) row0 = row1;
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                const uint8_t* src = (v ? v_lane : k_lane) + (size_t)(a ? row1 : row0) * kD;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    cp16(&into.d[4 * a + i][lane], src + (i >> 1) * 8 * kD + (i & 1) * (v ? kD : 64));
            }
            if (lane < 8) cp16(&into.scale[4 * lane], (v ? vs_lane : ks_lane) + (lane < 4 ? row0 : row1));
        }
        cp_commit();
    };
    uint32_t have = halves(tile0, pages[0]), next = halves(tile0 + step, pages[1]);
    issue(false, tile0, pages[0], have, 0);
    issue(true, tile0, pages[0], have, 1);
    issue(false, tile0 + step, pages[1], next, 2);

    // the queries, scaled by a power of two to at most 2^14, as fp16 (and what that leaves)
    uint32_t qb[kSets][kParts][16];
    float factor[kSets][kCols];  // back from the scaled products to scores in log2 units, of queries 2t, 2t + 1
#pragma unroll
    for (int z = 0; z < kSets; ++z) {
        float x[32];
#pragma unroll
        for (int i = 0; i < (kF32 ? 8 : 4); ++i) {
            const uint32_t w[4] = {raw[z][i].x, raw[z][i].y, raw[z][i].z, raw[z][i].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (kF32) x[4 * i + e] = __uint_as_float(w[e]);
                else x[8 * (i & 3) + 2 * e] = __uint_as_float(w[e] << 16), x[8 * (i & 3) + 2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
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
        const float back = finite ? pow2(e - 13) * p.scale * kLog2e : __uint_as_float(0x7fffffffu);
        factor[z][0] = __shfl_sync(0xffffffffu, back, 8 * t);
        if (kCols == 2) factor[z][kCols - 1] = __shfl_sync(0xffffffffu, back, 8 * t + 4);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float a = finite ? x[2 * i] * mul : 0.f, c = finite ? x[2 * i + 1] * mul : 0.f;
            if (kBeside) {
                uint32_t hi, lo;
                split_pair(a, c, hi, lo);
                qb[z][0][i] = g & 1 ? lo : hi;
            } else if (kF32) {
                split_pair(a, c, qb[z][0][i], qb[z][kParts - 1][i]);
            } else {
                qb[z][0][i] = half_pair(a, c);
            }
        }
    }

#pragma unroll
    for (int z = 0; z < kSets; ++z) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) st.acc[z][j][e] = 0.f;
#pragma unroll
        for (int c = 0; c < kCols; ++c) st.m[z][c] = st.mx[z][c] = -INFINITY, st.l[z][c] = 0.f, st.f[z][c] = pow2(kFirstFactor);
    }

    int slot = 0;
    for (int tile = tile0; tile < tile1; tile += step) {
        const uint32_t now = have;
        // the pages of three tiles ahead are asked for here and first used in the next step
        int far[2];
        page_at(tile + 3 * step, far);
        cp_wait<kStages - 1>();
        __syncwarp();

        // scores [half][key g, key g + 8][query column 2t, 2t + 1]
        float s[kSets][2][2][kCols];
        {
            const Stage& k = ring[slot];
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                float d[kSets][2][4];  // (two chains of products each)
#pragma unroll
                for (int z = 0; z < kSets; ++z)
#pragma unroll
                    for (int e = 0; e < 4; ++e) d[z][0][e] = d[z][1][e] = 0.f;
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    uint32_t w0[4], w1[4];  // rows g and g + 8
                    *reinterpret_cast<uint4*>(w0) = k.d[4 * a + hf][lane];
                    *reinterpret_cast<uint4*>(w1) = k.d[4 * a + 2 + hf][lane];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        uint32_t a0, a1, a2, a3;
                        pairs_of_word<kFmt>(w0[e], a0, a2);
                        pairs_of_word<kFmt>(w1[e], a1, a3);
#pragma unroll
                        for (int z = 0; z < kSets; ++z)
#pragma unroll
                            for (int c = 0; c < kParts; ++c)
                                mma_f16(d[z][e & 1], a0, a1, a2, a3, qb[z][c][8 * hf + 2 * e], qb[z][c][8 * hf + 2 * e + 1]);
                    }
                }
                const float ks0 = k.scale[kSub * a + g], ks1 = k.scale[kSub * a + g + 8];
#pragma unroll
                for (int z = 0; z < kSets; ++z)
#pragma unroll
                    for (int c = 0; c < kCols; ++c) {
                        float s0 = d[z][0][c] + d[z][1][c], s1 = d[z][0][2 + c] + d[z][1][2 + c];
                        if (kBeside) s0 += d[z][0][1] + d[z][1][1], s1 += d[z][0][3] + d[z][1][3];
                        s[z][a][0][c] = s0 * (ks0 * factor[z][c]);
                        s[z][a][1][c] = s1 * (ks1 * factor[z][c]);
                    }
            }
        }
        __syncwarp();  // every lane is done with this piece
        issue(true, tile + step, pages[1], next, slot);
        slot = slot == kStages - 1 ? 0 : slot + 1;

        const int key0 = tile * kTile + g;
        const bool whole = now == 3u && tile * kTile + kTile <= least;
        if (!whole) {  // hidden keys: past a row's last one, or on a page that does not exist
#pragma unroll
            for (int z = 0; z < kSets; ++z)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int c = 0; c < kCols; ++c)
                        if (key0 + 8 * i >= lim[z][c] || !((now >> (i >> 1)) & 1u)) s[z][i >> 1][i & 1][c] = -INFINITY;
        }
        float top[kSets][kCols];
        bool grows = false;
#pragma unroll
        for (int z = 0; z < kSets; ++z)
#pragma unroll
            for (int c = 0; c < kCols; ++c) {
                top[z][c] = fmaxf(fmaxf(s[z][0][0][c], s[z][0][1][c]), fmaxf(s[z][1][0][c], s[z][1][1][c]));
                st.mx[z][c] = fmaxf(st.mx[z][c], top[z][c]);
                grows |= top[z][c] > st.m[z][c] + kGrow;
            }
        if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
            for (int z = 0; z < kSets; ++z)
#pragma unroll
                for (int c = 0; c < kCols; ++c) {
                    const float best = column_max(top[z][c]);
                    if (best > st.m[z][c] + kGrow) {
                        const float whole_best = ceilf(best);  // so that what it changes changes by powers of two
                        if (st.m[z][c] != -INFINITY || st.l[z][c] != 0.f) {  // (else there is nothing to scale yet)
                            const int d = (int)fminf(whole_best - st.m[z][c], 1000.f);
                            st.l[z][c] *= pow2_or_0(-d);
                            // f grows as p shrinks, up to its first value: the largest weights summed so far stay where they
                            // are in fp16's range, and so does acc.  (A factor that only fell would leave the weights behind
                            // a large row of V that has vanished among fp16's subnormals.)
                            const int was = exponent(st.f[z][c]), fe = min(was + d, kFirstFactor);
                            if (fe != was + d) st.rescale(z, c, pow2_or_0(fe - was - d));
                            st.f[z][c] = pow2(fe);
                        }
                        st.m[z][c] = whole_best;
                    }
                }
        }
        cp_wait<kStages - 1>();
        __syncwarp();
        const Stage& vp = ring[slot];
        // weights p and p * v_scale; a hidden key weighs nothing, whatever its scale is
        float u[kSets][2][2][kCols];
        grows = false;
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const float vs = vp.scale[kSub * a + 8 * k + g];
#pragma unroll
                for (int z = 0; z < kSets; ++z)
#pragma unroll
                    for (int c = 0; c < kCols; ++c) {
                        const float m_safe = st.m[z][c] == -INFINITY ? 0.f : st.m[z][c];  // (no key seen yet: every weight is 2^-inf)
                        const float w = ex2_approx(s[z][a][k][c] - m_safe);
                        st.l[z][c] += w;
                        u[z][a][k][c] = w * vs;
                        if (!whole && s[z][a][k][c] == -INFINITY) u[z][a][k][c] = 0.f;
                    }
            }
#pragma unroll
        for (int z = 0; z < kSets; ++z)
#pragma unroll
            for (int c = 0; c < kCols; ++c) {
                // (scales of a caller's own codes may be below zero)
                top[z][c] = fmaxf(fmaxf(fabsf(u[z][0][0][c]), fabsf(u[z][0][1][c])), fmaxf(fabsf(u[z][1][0][c]), fabsf(u[z][1][1][c])));
                grows |= top[z][c] * st.f[z][c] > 32768.f;
            }
        if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
            for (int z = 0; z < kSets; ++z)
#pragma unroll
                for (int c = 0; c < kCols; ++c) {
                    const float best = column_max(top[z][c]);
                    if (best * st.f[z][c] > 32768.f) {
                        const float fn = pow2(min(max(8 - exponent(best), -120), kFirstFactor));
                        // (a power of two, 0 below 2^-149; also from the first factor, with which small weights may have been summed)
                        st.rescale(z, c, fn / st.f[z][c]);
                        st.f[z][c] = fn;
                    }
                }
        }
#pragma unroll
        for (int a = 0; a < 2; ++a) {
            uint32_t pb[kSets][kParts][2];
#pragma unroll
            for (int z = 0; z < kSets; ++z)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const float x = u[z][a][k][0] * st.f[z][0], y = kCols == 2 ? u[z][a][k][kCols - 1] * st.f[z][kCols - 1] : 0.f;
                    if (kBeside) {
                        const uint32_t hi = half_pair(x, 0.f);
                        pb[z][0][k] = transposed(half_pair(x, x - half_values(hi).x));
                    } else if (kF32) {
                        uint32_t hi, lo;
                        split_pair(x, y, hi, lo);
                        pb[z][0][k] = transposed(hi);
                        pb[z][kParts - 1][k] = transposed(lo);
                    } else {
                        pb[z][0][k] = transposed(half_pair(x, y));
                    }
                }
            uint32_t v[4][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(v[i]) = vp.d[4 * a + i][lane];
            if (!whole) {  // codes of hidden keys may be anything, a NaN too
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (tile * kTile + kSub * a + 2 * t + (i & 1) + 8 * (i >> 1) >= keys || !((now >> a) & 1u))
                        v[i][0] = v[i][1] = v[i][2] = v[i][3] = 0u;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    uint32_t a0, a1, a2, a3;
                    pairs_across<kFmt>(v[0][e], v[1][e], i, a0, a1);
                    pairs_across<kFmt>(v[2][e], v[3][e], i, a2, a3);
#pragma unroll
                    for (int z = 0; z < kSets; ++z)
#pragma unroll
                        for (int c = 0; c < kParts; ++c) mma_f16(st.acc[z][2 * e + i], a0, a1, a2, a3, pb[z][c][0], pb[z][c][1]);
                }
        }
        __syncwarp();  // every lane is done with this piece
        have = next;
        next = halves(tile + 2 * step, pages[2]);
        issue(false, tile + 2 * step, pages[2], next, slot);
        slot = slot == kStages - 1 ? 0 : slot + 1;
#pragma unroll
        for (int i = 0; i < 2; ++i) pages[1][i] = pages[2][i], pages[2][i] = far[i];
    }
    cp_wait<0>();
    __syncwarp();
}

// Joins a CTA's warps: each puts its rows into its ring, then a warp takes a row, four dims a
// lane, and calls done(row, sums, maximum that they refer to, largest score).
template <int kForm, typename Done>
__device__ __forceinline__ void join_warps(Smem& sm, const State<kForm>& st, int rows, Done done) {
    constexpr int kSets = kForm == kWide ? 2 : 1, kCols = kForm == kFew ? 1 : 2;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int z = 0; z < kSets; ++z)
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
            const int row = 8 * z + kCols * t + c;
            const float l = column_sum(st.l[z][c]), mx = column_max(st.mx[z][c]);
            const float inv = 1.f / st.f[z][c];
            // (a row's 16-byte pieces are exchanged within 128-byte spans: fewer bank conflicts)
            float* o = reinterpret_cast<float*>(sm.ring[warp]) + row * kD;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<float4*>(o + 4 * ((4 * g + i) ^ (row & 7))) =
                    make_float4(st.sum(z, c, 4 * i) * inv, st.sum(z, c, 4 * i + 1) * inv, st.sum(z, c, 4 * i + 2) * inv,
                                st.sum(z, c, 4 * i + 3) * inv);
            if (g == 0) sm.m[warp][row] = st.m[z][c], sm.l[warp][row] = l, sm.mx[warp][row] = mx;
        }
    __syncthreads();
    for (int row = warp; row < rows; row += kWarps) {  // a warp per row, four dims a lane
        float best = -INFINITY, big = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) best = fmaxf(best, sm.m[w][row]), big = fmaxf(big, sm.mx[w][row]);
        Joined y;
#pragma unroll
        for (int w = 0; w < kWarps; ++w)
            y.add(sm.m[w][row], sm.l[w][row], best,
                  *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(sm.ring[w]) + row * kD + 4 * (lane ^ (row & 7))));
        done(row, y, best, big);
    }
}

// A cluster of `split` CTAs per work item (8 or 16 query rows of a sequence and K/V head): their
// warps take the sequence's tiles in turn and are joined in shared memory, then over the cluster.
// Where there are more CTAs than the GPU holds, those of the longest sequences come first, so
// that the last to start are the shortest.
template <int kFmt, bool kF32, int kForm>
__global__ void __launch_bounds__(kThreads, ctas_per_sm(kF32, kForm)) split_kernel(const Params p) {
    pdl_enter();
    constexpr int kRows = rows_of(kForm);
    extern __shared__ __align__(16) uint8_t smem_raw[];
    Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int item = p.split == 1 ? (int)blockIdx.x : (int)(blockIdx.x / (unsigned)p.split);
    const int rank = (int)blockIdx.x - item * p.split;
    const int per_head = (p.T * p.group + kRows - 1) / kRows;
    const int of_head = per_head == 1 ? item : (int)((unsigned)item / (unsigned)per_head);
    int b = (int)((unsigned)of_head / (unsigned)p.c.heads);
    const int hk = of_head - b * p.c.heads, row0 = (item - of_head * per_head) * kRows;
    if (p.by_length) {  // the b-th longest, ties by number: every thread ranks its sequences
        int* lens = reinterpret_cast<int*>(&sm.ring);
        for (int i = threadIdx.x; i < p.B; i += kThreads) lens[i] = p.seq_lens[i];
        __syncthreads();
        for (int i = threadIdx.x; i < p.B; i += kThreads) {
            const int mine = lens[i];
            int rank = 0;
#pragma unroll 8
            for (int j = 0; j < p.B; ++j) rank += lens[j] > mine || (lens[j] == mine && j < i);
            if (rank == b) sm.om[0] = __int_as_float(i);
        }
        __syncthreads();
        b = __float_as_int(sm.om[0]);
        __syncthreads();
    }

    State<kForm> st;
    attend<kFmt, kF32, kForm>(p, sm.ring[warp], b, hk, row0, rank * kWarps + warp, 0x7fffffff, p.split * kWarps, st);

    const int rows = min(kRows, p.T * p.group - row0);
    join_warps<kForm>(sm, st, rows, [&](int row, const Joined& y, float best, float big) {
        reinterpret_cast<float4*>(sm.joined(row))[lane] = y.o;
        if (lane == 0) sm.om[row] = best, sm.ol[row] = y.l, sm.omx[row] = big;
    });
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
            Smem* other = p.split > 1 ? cluster.map_shared_rank(&sm, c) : &sm;
            best = fmaxf(best, other->om[row]), big = fmaxf(big, other->omx[row]);
        }
        Joined y;
        for (int c = 0; c < p.split; ++c) {
            Smem* other = p.split > 1 ? cluster.map_shared_rank(&sm, c) : &sm;
            y.add(other->om[row], other->ol[row], best,
                  reinterpret_cast<const float4*>(other->joined(row))[lane]);
        }
        const int tq = token_of(rr, p.group);
        const long long out = ((long long)b * p.T + tq) * p.heads + hk * p.group + rr - tq * p.group;
        // the prefix's parts (at most 16: all of them on their way at once)
        const int q_len = p.q_lens ? min(p.q_lens[b], p.T) : p.T;
        const int shared = tq < q_len ? p.n_shared : 0;
        if (shared > 0) {
            const long long all = (long long)p.B * p.T * p.heads;
            float4 s = make_float4(-INFINITY, 0.f, -INFINITY, 0.f);
            if (lane < shared) s = p.shared_s[lane * all + out];
            const float own = best;
            best = fmaxf(best, warp_max(s.x)), big = fmaxf(big, warp_max(s.z));
            if (own != -INFINITY) y.scale(ex2_approx(own - best));
#pragma unroll 1
            for (int c0 = 0; c0 < shared; c0 += 8) {
                float4 o[8];
#pragma unroll
                for (int c = 0; c < 8; ++c)
                    o[c] = c0 + c < shared ? reinterpret_cast<const float4*>(p.shared_o + ((c0 + c) * all + out) * kD)[lane]
                                           : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int c = 0; c < 8; ++c)
                    y.add(__shfl_sync(0xffffffffu, s.x, c0 + c), __shfl_sync(0xffffffffu, s.y, c0 + c), best, o[c]);
            }
        }
        store_row<kF32>(p, out, lane, y, best, big);
    }
    if (p.split > 1) cluster.sync();  // no CTA leaves while another reads its shared memory
}

// Tiles of sequence b's keys (those of its last query).
__device__ __forceinline__ int tiles_of(const Params& p, int b) {
    const int q_len = p.q_lens ? min(p.q_lens[b], p.T) : p.T;
    const long long keys = min((long long)p.seq_lens[b], (long long)p.max_pages << p.c.page_shift);
    return q_len > 0 && keys > 0 ? (int)((keys + kTile - 1) / kTile) : 0;
}

// CTAs that take an item of sequence b: its share of the GPU by its tiles, one at least.  (`all`: tiles of all
// items.  All together that is at most p.shares + the number of items.)
__device__ __forceinline__ int shares_of(const Params& p, int tiles, long long all) {
    return tiles == 0 ? 0 : max(1, (int)((long long)p.shares * tiles / all));
}

// Few items of many keys: as many CTAs for each as its keys are of all keys, whose warps take its tiles in
// turn, so that all of them, and those of the other heads, read the same pages at about the same time.
// What a CTA has goes to the workspace, and join_kernel adds an item's parts up; an item of one CTA is written at once.
constexpr int kMaxBatch = 8192;  // the first CTAs of so many sequences fit into the ring's memory
template <int kFmt, bool kF32, int kForm>
__global__ void __launch_bounds__(kThreads, ctas_per_sm(kF32, kForm)) stream_kernel(const Params p) {
    pdl_enter();
    constexpr int kRows = rows_of(kForm);
    extern __shared__ __align__(16) uint8_t smem_raw[];
    Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
    static_assert(sizeof(sm.ring) >= (kMaxBatch + 1) * 4, "first CTAs of a batch");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int per_head = (p.T * p.group + kRows - 1) / kRows;
    const int items = p.c.heads * per_head;  // of one sequence

    // starts[b] = CTAs per item of the sequences before b; in the ring's memory until the first tile comes
    int* starts = reinterpret_cast<int*>(&sm.ring);
    {
        __shared__ int totals[kWarps];
        const int per = (p.B + kThreads - 1) / kThreads;
        const int b0 = min((int)threadIdx.x * per, p.B), b1 = min(b0 + per, p.B);
        // sum over the CTA's threads, and over those before this one
        auto scan = [&](int mine, int& before) {
            int upto = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += y;
            }
            __syncthreads();
            if (lane == 31) totals[warp] = upto;
            __syncthreads();
            int all = 0;
            before = upto - mine;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                if (w < warp) before += totals[w];
                all += totals[w];
            }
            return all;
        };
        int sum = 0, before;
        for (int b = b0; b < b1; ++b) sum += tiles_of(p, b);
        const long long all = (long long)scan(sum, before) * items;
        sum = 0;
        for (int b = b0; b < b1; ++b) sum += shares_of(p, tiles_of(p, b), all);
        scan(sum, before);
        for (int b = b0; b < b1; ++b) {
            starts[b] = before;
            if (blockIdx.x == 0) p.starts[b] = before;
            before += shares_of(p, tiles_of(p, b), all);
        }
        if (threadIdx.x == kThreads - 1) {
            starts[p.B] = before;
            if (blockIdx.x == 0) p.starts[p.B] = before;
        }
        __syncthreads();
    }
    const int w = blockIdx.x;
    if (w >= starts[p.B] * items) return;
    // the sequence of this CTA: the last one that starts at or before it
    int b = 0;
    for (int up = kMaxBatch / 2; up > 0; up >>= 1)
        if (b + up < p.B && starts[b + up] * items <= w) b += up;
    const int split = starts[b + 1] - starts[b];
    const int i = (w - starts[b] * items) / split, rank = (w - starts[b] * items) % split;
    __syncthreads();  // the ring's memory is free
    const int hk = i / per_head, row0 = i % per_head * kRows;
    State<kForm> st;
    attend<kFmt, kF32, kForm>(p, sm.ring[warp], b, hk, row0, rank * kWarps + warp, 0x7fffffff, split * kWarps, st);
    const bool whole = split == 1 && p.n_shared == 0;
    join_warps<kForm>(sm, st, min(kRows, p.T * p.group - row0), [&](int row, const Joined& y, float best, float big) {
        if (whole) {
            const int r = row0 + row;
            store_row<kF32>(p, ((long long)b * p.T + r / p.group) * p.heads + hk * p.group + r % p.group, lane, y, best, big);
        } else {
            const long long at = (long long)w * kRows + row;
            reinterpret_cast<float4*>(p.part_o + at * kD)[lane] = y.o;
            if (lane == 0) p.part_s[at] = make_float4(best, y.l, big, 0.f);
        }
    });
}

// Joins the parts of each query row: a CTA per row, of as many warps as there are eights of parts, up to 16; a
// warp takes eight parts at a time (so that eight rows of 512 bytes are on their way at once).
constexpr int kJoinWarps = 16;
template <bool kF32, int kForm>
__global__ void __launch_bounds__(kJoinWarps * 32) join_kernel(const Params p) {
    pdl_enter();
    constexpr int kRows = rows_of(kForm);
    const long long rows = (long long)p.B * p.T * p.heads;
    const long long row = blockIdx.x;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int h = (int)(row % p.heads), tq = (int)(row / p.heads % p.T), b = (int)(row / p.heads / p.T);
    const int r = tq * p.group + h % p.group;
    const int q_len = p.q_lens ? min(p.q_lens[b], p.T) : p.T;

    // the CTAs that had a part of this row's item
    int parts = 0;
    long long slot = 0;
    if (p.shares > 0) {
        const int per_head = (p.T * p.group + kRows - 1) / kRows;
        const int items = p.c.heads * per_head;
        const int i = h / p.group * per_head + r / kRows;
        const int start = p.starts[b];
        parts = p.starts[b + 1] - start;
        if (parts == 1 && p.n_shared == 0) return;  // written by stream_kernel
        slot = (long long)start * items + (long long)i * parts;
    }
    const int shared = tq < q_len ? p.n_shared : 0;
    const float4* own_s = p.part_s + slot * kRows + r % kRows;
    const float4* own_o = reinterpret_cast<const float4*>(p.part_o + (slot * kRows + r % kRows) * kD) + lane;
    const float4* shared_s = p.shared_s + row;
    const float4* shared_o = reinterpret_cast<const float4*>(p.shared_o + row * kD) + lane;
    float m = -INFINITY, big = -INFINITY;
    Joined y;
    for (int i0 = 8 * warp; i0 < parts + shared; i0 += 8 * warps) {
        float4 s = make_float4(-INFINITY, 0.f, -INFINITY, 0.f);
        const int mine = i0 + (lane & 7);
        if (mine < parts) s = own_s[(long long)mine * kRows];
        else if (mine < parts + shared) s = shared_s[(mine - parts) * rows];
        float4 o[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (i0 + i < parts) o[i] = own_o[(long long)(i0 + i) * kRows * (kD / 4)];
            else if (i0 + i < parts + shared) o[i] = shared_o[(i0 + i - parts) * rows * (kD / 4)];
        }
        float top = s.x;
#pragma unroll
        for (int w = 1; w < 8; w <<= 1) {
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
            s.z = fmaxf(s.z, __shfl_xor_sync(0xffffffffu, s.z, w));
        }
        big = fmaxf(big, s.z);
        if (top > m) {
            const float a = m == -INFINITY ? 1.f : ex2_approx(m - top);  // (at -inf there may be NaNs, which stay)
            m = top;
            y.scale(a);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
            y.add(__shfl_sync(0xffffffffu, s.x, i), __shfl_sync(0xffffffffu, s.y, i), m, o[i]);
    }
    __shared__ float4 so[kJoinWarps][32];
    __shared__ float sm[kJoinWarps], sl[kJoinWarps], sx[kJoinWarps];
    so[warp][lane] = y.o;
    if (lane == 0) sm[warp] = m, sl[warp] = y.l, sx[warp] = big;
    __syncthreads();
    if (warp != 0) return;
    float best = -INFINITY;
    big = -INFINITY;
    for (int w = 0; w < warps; ++w) best = fmaxf(best, sm[w]), big = fmaxf(big, sx[w]);
    Joined all;
    for (int w = 0; w < warps; ++w) all.add(sm[w], sl[w], best, so[w][lane]);
    store_row<kF32>(p, row, lane, all, best, big);
}

}  // namespace cache_attn
}  // namespace dt
