// The quantised K/V cache: rows of 128 values (one token, one head) are kept as 8-bit
// codes with one fp32 scale per row, in pages of `page` tokens:
//   codes  [pages][heads][page][128]   one byte per value (int8, or fp8 e4m3)
//   scales [pages][heads][page]
// so that one head's tokens of a page are contiguous: page * 128 bytes of codes.
//
// Writing:  amax = max |x|, scale = amax / Q, code = round(x * Q / amax) to the nearest
// code, ties to even, with Q = 127 (int8) or 448 (e4m3, its largest value).  The product
// x * Q is exact for bf16 values and the quotient is rounded once, so a value half-way
// between two codes is seen as such.  Rows with amax < 2^-100 are stored as zeros with
// scale 0 (Q / amax would overflow below 2^-119); a row that holds an infinity or a NaN
// gets the scale NaN and zero codes, so that it reads back as NaN and poisons only
// the queries that see it.
// Reading:  value = code * scale in fp32, rounded once to the output type.
//
// Both are bound by memory.  16384 tokens of 16 heads: writing from fp32 (268 MB in, 68 MB out) takes 65 us,
// 5.2 TB/s, where its 470 instructions per warp and four rows are the next bound; reading back as bf16 (68 MB
// in, 134 MB out) 36 us, 5.6 TB/s.
#pragma once
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "dt_common.cuh"

namespace dt {
namespace kv {

constexpr int kD = 128;
constexpr int kThreads = 256;
constexpr int kRowLanes = 8;                      // lanes per row of 128 values, 16 values each
constexpr int kRows = kThreads / kRowLanes;       // rows a CTA handles at once
constexpr int kEntries = 2048;                    // page entries of a launch that writes
constexpr float kTiny = 7.888609052210118e-31f;   // 2^-100
constexpr float kHuge = 1.2676506002282294e30f;   // 2^100

enum : int { kInt8 = 0, kE4m3 = 1 };

struct Cache {
    uint8_t* k;
    uint8_t* v;
    float* ks;
    float* vs;
    int pages;
    int page_shift;  // page = 1 << page_shift
    int heads;
};

struct Span {                 // which tokens of which sequences a call touches
    const int* table;         // [B, max_pages], rows table_stride apart
    long long table_stride;
    int max_pages;
    const int* start;         // [B] position of the first token (null: 0)
    const int* lens;          // [B] tokens of each sequence, at most T (null: T)
    int B, T;
    int first;                // tokens of each sequence before the T ones of this launch
};

// Tokens of sequence b among the launch's T (none: 0 or less).  kLater: the launch has tokens before its own; known at
// compile time, since the append kernel has no register to spare (4 x 4096 tokens of fp32, written and read back: 101 us, 107 with seven more).
template <bool kLater>
__device__ __forceinline__ int length_of(const Span& s, int b) {
    if (!s.lens) return s.T;
    return min(kLater ? max(s.lens[b], 0) - s.first : s.lens[b], s.T);
}

// Page of position pos of sequence b, or -1 where the table has none.
__device__ __forceinline__ int page_of(const Span& s, const Cache& c, int b, int pos) {
    if (pos < 0) return -1;
    const int j = pos >> c.page_shift;
    if (j >= s.max_pages) return -1;
    const int p = __ldg(s.table + (long long)b * s.table_stride + j);
    return (p >= 0 && p < c.pages) ? p : -1;
}

__device__ __forceinline__ long long row_of(const Cache& c, int page, int head, int pos) {
    return (((long long)page * c.heads + head) << c.page_shift) + (pos & ((1 << c.page_shift) - 1));
}

// Positions never pass 2^31 - 1: starts and lengths are ints and their sum is clamped.
__device__ __forceinline__ int position(int start, int t) {
    const long long p = (long long)start + t;
    return p > 0x7fffffffll ? -1 : (int)p;
}

// Where a page table gives one slot to several tokens of a call, the token of the highest
// (sequence, position) is kept: within a launch by looking through its page entries, and by the order of launches
// where a call has more than kEntries of them (each CTA looks through all that follow its own, so the time would
// grow with their square: 163 ms for 4 million tokens of one sequence in pages of 16, 2.9 in stretches).  True if one above (b, pos) writes page `page` at the same
// offset (pos >= 0), or any offset (pos < 0: above sequence b's page index j0).  The calling
// lanes share the entries: lane `part` of `parts`.
template <bool kLater>
__device__ __forceinline__ bool written_above(const Span& s, const Cache& c, int b, int j0, int pos, int page, int part,
                                              int parts) {
    const unsigned width = (unsigned)(s.T >> c.page_shift) + 2u;  // pages that one sequence's tokens can touch
    const unsigned n = (unsigned)(s.B - b) * width;  // (at most kEntries)
    const int off = pos & ((1 << c.page_shift) - 1);
    for (unsigned i = part; i < n; i += parts) {
        const unsigned skip = i / width;
        const int b2 = b + (int)skip;
        const int len = length_of<kLater>(s, b2);
        const long long first = (s.start ? s.start[b2] : 0) + (kLater ? (long long)s.first : 0ll), last = min(first + len - 1, 0x7fffffffll);
        if (len <= 0) continue;
        const long long j = (first >> c.page_shift) + (i - skip * width);
        if (j < 0 || j > (last >> c.page_shift) || j >= s.max_pages || (b2 == b && j <= j0)) continue;
        if (__ldg(s.table + (long long)b2 * s.table_stride + j) != page) continue;
        const long long at = (j << c.page_shift) + off;
        if (pos < 0 || (at >= first && at <= last)) return true;
    }
    return false;
}

// Codes of four values: round(x * mul / den), mul / den = Q / amax, inv = 1 / den.
// int8: x * mul * inv is within three units of fp32's last place of the rounded quotient, so its code is the
// quotient's unless a border between two codes is as near: then, for one value in some 10,000, the quotient
// itself is formed (25 us instead of 30 for 131072 rows).  e4m3's borders lie at many distances, and
// looking for them takes longer than the division (32 us instead of 28).
template <int kFmt>
__device__ __forceinline__ uint32_t encode4(const float (&x)[4], float mul, float den, float inv) {
    constexpr float kMagic = 12582912.f;  // 1.5 * 2^23: the sum's low byte is the rounded value
    float y[4];
    if constexpr (kFmt == kInt8) {
        bool near = false;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            y[i] = __fmul_rn(__fmul_rn(x[i], mul), inv);
            // |y| <= 127 and a bit: three units of its last place are below 2.3e-5
            const float whole = __fsub_rn(__fadd_rn(y[i], kMagic), kMagic);
            near |= fabsf(__fsub_rn(y[i], whole)) > 0.49995f;
        }
        if (near) {
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = __fdiv_rn(__fmul_rn(x[i], mul), den);
        }
        uint32_t c[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) c[i] = __float_as_uint(__fadd_rn(y[i], kMagic));
        return __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = __fdiv_rn(__fmul_rn(x[i], mul), den);
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(y[0], y[1]), __NV_SATFINITE, __NV_E4M3);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(y[2], y[3]), __NV_SATFINITE, __NV_E4M3);
        return lo | (hi << 16);
    }
}

// Four codes to fp32 (exact: both formats' values have at most 8 significant bits).
template <int kFmt>
__device__ __forceinline__ void decode4(uint32_t w, float (&x)[4]) {
    if (kFmt == kInt8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = (float)(int)(int8_t)(w >> (8 * i));
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> (16 * i)), __NV_E4M3);
            const float2 f = __half22float2(__half2(h));
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
    }
}

struct AppendParams {
    Cache c;
    Span s;
    const void* k;
    const void* v;
    long long k_batch, k_token, v_batch, v_token;  // strides in elements; heads are 128 apart
    int tile;                                      // tokens per CTA
    int tiles;                                     // CTAs per sequence
};

// Quantises and stores the new tokens.  A CTA takes `tile` tokens of one sequence, 8 lanes
// per row; lane l holds the row's 16-byte source chunks l, l + 8, ..., so that loads and
// stores of a row are contiguous over its lanes.
template <int kFmt, bool kF32, bool kLater>
__global__ void __launch_bounds__(kThreads) append_kernel(const AppendParams p) {
    pdl_enter();
    const int b = (int)(blockIdx.x / (unsigned)p.tiles);
    const int t0 = (int)(blockIdx.x % (unsigned)p.tiles) * p.tile;
    const int t1 = min(t0 + p.tile, length_of<kLater>(p.s, b));
    if (t0 >= t1) return;
    int start = p.s.start ? p.s.start[b] : 0;
    if (kLater) {
        const long long from = (long long)start + p.s.first;
        if (from > 0x7fffffffll) return;  // past the last position
        start = (int)from;
    }
    const int lane = threadIdx.x & (kRowLanes - 1);
    const int per_token = 2 * p.c.heads;
    const int rows = (t1 - t0) * per_token;
    // Does a later token of this call write one of this tile's pages?  (A tile is at most a
    // page long, so it touches two pages at most.)  Almost always not.  (Asked while the first
    // rows are on their way.)
    auto ask = [&] {
        const int first = position(start, t0), last = position(start, t1 - 1);
        const int pa = page_of(p.s, p.c, b, first), pb = page_of(p.s, p.c, b, last);
        const int ja = first >> p.c.page_shift, jb = last >> p.c.page_shift;
        bool contested = false;
        if (pa >= 0) contested = written_above<kLater>(p.s, p.c, b, ja, -1, pa, threadIdx.x, kThreads);
        if (pb >= 0 && jb != ja) contested |= written_above<kLater>(p.s, p.c, b, jb, -1, pb, threadIdx.x, kThreads);
        return __syncthreads_or(contested) != 0;
    };
    // A row of 8 lanes: K or V of head h of a token; the next one is 32 rows on.
    const int token_step = (int)((unsigned)kRows / (unsigned)per_token), rest_step = kRows - token_step * per_token;
    int r = threadIdx.x >> 3;
    int t = t0 + (int)((unsigned)r / (unsigned)per_token);
    int rest = r - (t - t0) * per_token;
    constexpr int kPieces = kF32 ? 4 : 2, kSize = kF32 ? 4 : 2;
    const char* k_src = static_cast<const char*>(p.k) + ((long long)b * p.k_batch * kSize + 16 * lane);
    const char* v_src = static_cast<const char*>(p.v) + ((long long)b * p.v_batch * kSize + 16 * lane);
    const int* table = p.s.table + (long long)b * p.s.table_stride;
    auto load = [&](uint4 (&raw)[kPieces]) {
        const bool is_v = rest >= p.c.heads;
        const char* src = is_v ? v_src : k_src;
        const long long at = (long long)t * (is_v ? p.v_token : p.k_token) + (is_v ? rest - p.c.heads : rest) * kD;
        const uint4* f = reinterpret_cast<const uint4*>(src + at * kSize);
#pragma unroll
        for (int i = 0; i < kPieces; ++i) raw[i] = r < rows ? __ldg(f + 8 * i) : make_uint4(0, 0, 0, 0);
    };
    uint4 ahead[kPieces];
    load(ahead);
    const bool contested = ask();
    for (int r0 = 0; r0 < rows; r0 += kRows) {
        const bool in = r < rows;
        const bool is_v = rest >= p.c.heads;
        const int h = is_v ? rest - p.c.heads : rest;
        const int pos = in ? position(start, t) : -1;
        int page = -1;
        if (pos >= 0 && (pos >> p.c.page_shift) < p.s.max_pages) {
            page = __ldg(table + (pos >> p.c.page_shift));
            if (page >= p.c.pages) page = -1;
        }
        uint4 raw[kPieces];
#pragma unroll
        for (int i = 0; i < kPieces; ++i) raw[i] = ahead[i];
        r += kRows, t += token_step, rest += rest_step;
        if (rest >= per_token) rest -= per_token, ++t;
        if (r0 + kRows < rows) load(ahead);  // the next rows are on their way while these are coded
        if (contested) {
            const bool lost = page >= 0 && written_above<kLater>(p.s, p.c, b, pos >> p.c.page_shift, pos, page, lane, kRowLanes);
            const uint32_t votes = __ballot_sync(0xffffffffu, lost);
            if ((votes >> (threadIdx.x & 24)) & 0xffu) page = -1;
        }
        float x[16];
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (kF32) x[4 * i + e] = __uint_as_float(w[e]);
                else x[8 * (i & 1) + 2 * e] = __uint_as_float(w[e] << 16), x[8 * (i & 1) + 2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
            }
        }
        // the largest magnitude, and 0 or, where a value is not finite, NaN
        float amax = 0.f, odd = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) amax = fmaxf(amax, fabsf(x[i])), odd = fmaf(x[i], 0.f, odd);
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) {
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
            odd += __shfl_xor_sync(0xffffffffu, odd, o);
        }
        if (page < 0) continue;  // (whole row groups: no lane of a live row leaves)
        const bool finite = odd == 0.f;
        const bool live = finite && amax >= kTiny;
        constexpr float kTop = kFmt == kInt8 ? 127.f : 448.f;
        // x * Q could overflow from 2^119 on: there both sides of the quotient lose a factor of 2^20, exactly
        const float pre = amax >= kHuge ? 9.5367431640625e-07f : 1.f;
        const float mul = kTop * pre, den = amax * pre, inv = live ? __fdiv_rn(1.f, den) : 0.f;
        // (a cache has fewer than 2^31 rows)
        const uint32_t row = ((uint32_t)(page * p.c.heads + h) << p.c.page_shift) + (pos & ((1 << p.c.page_shift) - 1));
        uint8_t* dst = (is_v ? p.c.v : p.c.k) + (size_t)row * kD;
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[i] = live ? encode4<kFmt>(*reinterpret_cast<const float(*)[4]>(x + 4 * i), mul, den, inv) : 0u;
        if (kF32) {
#pragma unroll
            for (int i = 0; i < 4; ++i) reinterpret_cast<uint32_t*>(dst)[8 * i + lane] = w[i];
        } else {
            reinterpret_cast<uint2*>(dst)[lane] = make_uint2(w[0], w[1]);
            reinterpret_cast<uint2*>(dst)[8 + lane] = make_uint2(w[2], w[3]);
        }
        if (lane == 0) {
            const float scale = live ? __fdiv_rn(amax, kTop) : finite ? 0.f : __uint_as_float(0x7fffffffu);
            (is_v ? p.c.vs : p.c.ks)[row] = scale;
        }
    }
}

struct ReadParams {
    Cache c;
    Span s;
    void* k;  // [B, T, heads, 128]
    void* v;
    long long rows;  // B * T * 2 * heads
};

// Reads rows back as fp32 or bf16; tokens at or past a sequence's length, and tokens whose
// page the table does not have, are written as zeros.  8 lanes per row, in the append
// kernel's interleaved order.
template <int kFmt, bool kF32>
__global__ void __launch_bounds__(kThreads) read_kernel(const ReadParams p) {
    pdl_enter();
    const int lane = threadIdx.x & (kRowLanes - 1);
    for (long long r = (long long)blockIdx.x * kRows + (threadIdx.x >> 3); r < p.rows;
         r += (long long)gridDim.x * kRows) {
        const int h2 = (int)(r % (2 * p.c.heads));
        const long long bt = r / (2 * p.c.heads);
        const int t = (int)(bt % p.s.T);
        const int b = (int)(bt / p.s.T);
        const bool is_v = h2 >= p.c.heads;
        const int h = is_v ? h2 - p.c.heads : h2;
        const int len = p.s.lens ? min(p.s.lens[b], p.s.T) : p.s.T;
        const int pos = position(p.s.start ? p.s.start[b] : 0, t);
        const int page = t < len ? page_of(p.s, p.c, b, pos) : -1;
        uint32_t w[4] = {0, 0, 0, 0};
        float scale = 0.f;
        if (page >= 0) {
            const long long row = row_of(p.c, page, h, pos);
            const uint8_t* src = (is_v ? p.c.v : p.c.k) + row * kD;
            scale = (is_v ? p.c.vs : p.c.ks)[row];
            if (kF32) {
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = reinterpret_cast<const uint32_t*>(src)[8 * i + lane];
            } else {
                const uint2 a = reinterpret_cast<const uint2*>(src)[lane], c = reinterpret_cast<const uint2*>(src)[8 + lane];
                w[0] = a.x, w[1] = a.y, w[2] = c.x, w[3] = c.y;
            }
        }
        const long long out = (bt * p.c.heads + h) * kD;
        float x[16];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            decode4<kFmt>(w[i], *reinterpret_cast<float(*)[4]>(x + 4 * i));
#pragma unroll
            for (int e = 0; e < 4; ++e) x[4 * i + e] *= scale;
        }
        if (kF32) {
            float4* dst = reinterpret_cast<float4*>(static_cast<float*>(is_v ? p.v : p.k) + out);
#pragma unroll
            for (int i = 0; i < 4; ++i) dst[8 * i + lane] = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
        } else {
            uint4* dst = reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(is_v ? p.v : p.k) + out);
#pragma unroll
            for (int i = 0; i < 2; ++i)
                dst[8 * i + lane] = make_uint4(pack_bf16x2(x[8 * i], x[8 * i + 1]), pack_bf16x2(x[8 * i + 2], x[8 * i + 3]),
                                               pack_bf16x2(x[8 * i + 4], x[8 * i + 5]), pack_bf16x2(x[8 * i + 6], x[8 * i + 7]));
        }
    }
}

}  // namespace kv
}  // namespace dt
