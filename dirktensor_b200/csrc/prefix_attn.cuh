// Attention of a whole batch's new tokens over the keys of a prefix that all its sequences share,
// read once: the queries of all sequences that read a K/V head (B * T * group rows) are one matrix, so
// both products are tensor-core matrix products (tcgen05, accumulators in TMEM), where the same
// keys read per sequence would be as many vector products.
//
// A CTA takes up to 256 (or 128) query rows of one K/V head and a stretch of the prefix's 128-key tiles:
//   warps 0-3, 4-7  softmax, one thread per row (TMEM lane).  With more than 128 rows the two
//                   warpgroups take 128 rows each and both see every tile; otherwise they take every
//                   other tile of the same rows, as two parts that are joined at the end;
//   warps 8-11      convert: codes from global memory, as fp16 into the 128-byte-swizzled tiles that
//                   the MMAs read (K and V, two buffers each), with the next tile's codes in registers;
//   warp 12         issues the MMAs (one thread) and owns TMEM.
// TMEM (512 columns): S0 S1 O0 O1 of 128 each; P_i, fp16 pairs, overwrites S_i and feeds the second product
// from there.  The issue order PV_i(t), S_i(next) keeps the tensor core on one warpgroup's
// tile while the other does its softmax.
//
// Codes are exact in fp16, and so are bf16 queries, each row scaled by a power of two into its
// range; fp32 queries go in as fp16(q) and the rest, as two products into one accumulator.  Scales stay out of
// the operands: S is multiplied by k_scale (and the row's factor) in fp32, and the weights p by v_scale before they
// are rounded to fp16 (once, at 2^-11 below a bf16 result's own 2^-8; for fp32 queries as two numbers
// again).  f, a power of two of each row, keeps p * v_scale * f below 2^15 and the largest of them so far at 1 or
// more, so that each is off by at most 2^-25 of that one: it falls where the row's largest weight asks for it and grows
// as the running maximum takes older weights away.  Only where both together change the unit of O is O rescaled.
//
// Bound by its chain of steps rather than by a unit: per tile and warpgroup about 5000 cycles of softmax (two
// passes over 128 TMEM columns; MUFU's share is 1024), 1400 of MMAs, and 10000 before the first tile is there (page
// numbers, then codes, each a first touch of its memory).  64 queries x 16 heads over 8192 keys: 30 us; 800 x 8 over
// 6143: 62 us, 330 TFLOP/s.  More converting warps, TMEM loads ahead of use and precomputed descriptors
// each changed that by under 5 %; fewer instructions before the first tile by 20 %.
#pragma once
#include "cache_attn.cuh"

namespace dt {
namespace prefix_attn {

using cache_attn::half_pair;
using cache_attn::kLog2e;
using cache_attn::pow2;
using cache_attn::exponent;

constexpr int kD = 128;
constexpr int kBM = 128;                   // rows of a Q tile
constexpr int kBN = 128;                   // keys of a tile
constexpr int kTileBytes = 128 * kD * 2;   // fp16
constexpr int kHalfBytes = kTileBytes / 2; // 64 dims: one swizzle span
constexpr int kConvWarps = 4;
constexpr int kMmaWarp = 8 + kConvWarps;
constexpr int kThreads = (kMmaWarp + 1) * 32;
constexpr float kGrow = 8.f;               // log2 units, as in flash_fwd.cuh
// log2 of the weights' factor before any: rows of 2^-100, the smallest kept, weigh 2 or more, and 128 weights of 2^8 stay finite
constexpr int kFirstFactor = 110;
constexpr int kLowered = 7;                // a lowered factor puts the tile's largest weight below 2^kLowered (11: 86 us for 800 x 8 rows over 6143 keys and their own, 84 at 7)
constexpr float kNear = 32.f;              // scales of a tile this near to each other need no look at its products: a bound is that near too

struct Params {
    cache_attn::Params a;
    int rows;     // B * T * group
    int blocks;   // of rows: blocks of 256, or of 128 with `pairs`
    int pairs;    // 1: one Q tile, the warpgroups take every other key tile; 0: two Q tiles
    int split;    // stretches of the prefix
    int tiles;    // of the prefix
};

struct __align__(1024) Smem {
    uint8_t q[2][kTileBytes];   // the two Q tiles; or fp16(q) of one and the rest
    uint8_t k[2][kTileBytes];
    uint8_t v[2][kTileBytes];
    float ks[4][kBN];           // of tile t: at t & 3
    float vs[4][kBN];
    float most[4][kConvWarps], least[4][kConvWarps];  // largest and smallest |v_scale| of the 32 keys of each converting warp
    uint32_t hidden[4][kConvWarps];  // keys past the prefix, or on a page that does not exist
    float factor[2][kBM];       // from S back to scores in log2 units (k_scale apart)
    float m[kBM], l[kBM], mx[kBM];  // of the second warpgroup, for the first (pairs)
    uint64_t q_full;
    uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2];
    uint64_t s_full[2], p_full[2], o_full[2];
    uint64_t mma_done;
    uint32_t tmem_base;
};

enum : unsigned { kSiteQ = 0x21, kSiteKFull, kSiteKEmpty, kSiteVFull, kSiteVEmpty, kSiteS, kSiteP, kSiteO, kSiteDone };

// tcgen05 instruction descriptor: fp16 A and B, fp32 accumulator.
constexpr uint32_t idesc_f16(int M, int N, int b_mn_major) {
    return (1u << 4) | ((uint32_t)b_mn_major << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

__device__ __forceinline__ void st_shared_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ uint64_t f2_mul(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// (f2_fma flushes subnormal numbers to zero, also a factor)
__device__ __forceinline__ uint64_t f2_fma_full(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Waits for this thread's TMEM loads; x is valid afterwards, and the compiler uses it no earlier.
__device__ __forceinline__ void wait_for(float (&x)[32]) {
    tmem_wait_ld();
#pragma unroll
    for (int e = 0; e < 32; ++e) asm volatile("" : "+f"(x[e]));
}

// A 16-byte piece of codes (16 dims of one key) as fp16: two 16-byte chunks of a swizzled tile.  The
// lanes of the second half of the dims store theirs in the other order (`swap`): no bank conflicts.
template <int kFmt>
__device__ __forceinline__ void put_piece(uint32_t first, uint32_t second, bool swap, uint4 c) {
    const uint32_t w[4] = {swap ? c.z : c.x, swap ? c.w : c.y, swap ? c.x : c.z, swap ? c.y : c.w};
    uint32_t h[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) cache_attn::pairs_of_word<kFmt>(w[i], h[2 * i], h[2 * i + 1]);
    st_shared_v4(first, h[0], h[1], h[2], h[3]);
    st_shared_v4(second, h[4], h[5], h[6], h[7]);
}

template <int kFmt, bool kF32>
__global__ void __launch_bounds__(kThreads, 1) prefix_kernel(const Params pp) {
    pdl_enter();
    const cache_attn::Params& p = pp.a;
    extern __shared__ uint8_t smem_raw[];
    Smem& sm = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    const int group = (int)(blockIdx.x / (unsigned)pp.split);
    const int part = (int)blockIdx.x - group * pp.split;
    const int hk = (int)((unsigned)group / (unsigned)pp.blocks), block = group - hk * pp.blocks;
    const int row0 = block * (pp.pairs ? kBM : 2 * kBM);
    // (tiles and parts are at most 2^24 and 148)
    const int t0 = (int)((unsigned)pp.tiles / (unsigned)pp.split) * part + min(part, (int)((unsigned)pp.tiles % (unsigned)pp.split));
    const int t1 = t0 + (int)((unsigned)pp.tiles / (unsigned)pp.split) + (part < (int)((unsigned)pp.tiles % (unsigned)pp.split) ? 1 : 0);
    const int n = t1 - t0;  // at least one: split <= tiles
    const bool second_rows = !pp.pairs && row0 + kBM < pp.rows;
    // steps of warpgroup i: its s-th one is tile s, or 2 s + i
    const int steps[2] = {pp.pairs ? (n + 1) / 2 : n, pp.pairs ? n / 2 : (second_rows ? n : 0)};

    if (threadIdx.x == 0) {
        mbar_init(&sm.q_full, 8);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sm.k_full[i], kConvWarps);
            mbar_init(&sm.v_full[i], kConvWarps);
            mbar_init(&sm.k_empty[i], 1);
            mbar_init(&sm.v_empty[i], 1);
            mbar_init(&sm.s_full[i], 1);
            mbar_init(&sm.p_full[i], 4);
            mbar_init(&sm.o_full[i], 1);
        }
        mbar_init(&sm.mma_done, 1);
        fence_mbar_init();
    }
    if (warp == kMmaWarp) {
        tmem_alloc(&sm.tmem_base, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sm.tmem_base;

    if (warp >= 8 && warp < kMmaWarp) {
        // ------------------------------ convert -----------------------------
        const int cw = warp - 8;
        const int shift = p.c.page_shift, in_page = (1 << shift) - 1;
        // this warp's 32 keys of a tile are two groups of 16, each on one page: lanes 0-15 and 16-31 look up one
        auto look_up = [&](int tile) {
            const int key = tile * kBN + cw * 32 + (lane & 16);
            const int page = key < p.prefix_len ? __ldg(p.prefix_pages + (key >> shift)) : -1;
            return page >= 0 && page < p.c.pages ? page : -1;
        };
        // lane: piece lane & 7 of rows 4 i + lane / 8
        const int rl = lane >> 3, piece = lane & 7;
        // row of the cache where group g of a tile starts
        auto row_at = [&](int tile, int page, int g) {
            return ((uint32_t)(page * p.c.heads + hk) << shift) + ((tile * kBN + cw * 32 + 16 * g) & in_page);
        };
        auto load = [&](const uint8_t* codes, int tile, int pages, uint4 (&x)[8]) {
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const int page = __shfl_sync(0xffffffffu, pages, 16 * g);
                // hidden keys: zeros
                const int left = page >= 0 ? p.prefix_len - (tile * kBN + cw * 32 + 16 * g) : 0;
                const uint4* src = reinterpret_cast<const uint4*>(codes + (size_t)row_at(tile, page, g) * kD) + rl * (kD / 16) + piece;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    x[4 * g + i] = 4 * i + rl < left ? __ldg(src + i * 4 * (kD / 16)) : make_uint4(0, 0, 0, 0);
            }
        };
        // offsets of a lane's chunks in a tile, of even and odd i (row & 7 is rl, or 4 + rl)
        const bool swap = piece >= 4;
        uint32_t off[2][2];
#pragma unroll
        for (int o = 0; o < 2; ++o)
#pragma unroll
            for (int c = 0; c < 2; ++c)
                off[o][c] = (uint32_t)(piece >> 2) * kHalfBytes + (uint32_t)(cw * 32 + 4 * o + rl) * 128 +
                            (((2 * (piece & 3) + ((c == 0) == swap ? 1 : 0)) ^ (4 * o + rl)) << 4);
        auto put = [&](uint8_t* tile, const uint4 (&x)[8]) {
            const uint32_t base = smem_u32(tile);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                put_piece<kFmt>(base + off[i & 1][0] + (i >> 1) * 1024, base + off[i & 1][1] + (i >> 1) * 1024, swap, x[i]);
        };
        // scales of a tile, one key a lane (a hidden key's score becomes -inf)
        auto load_scales = [&](int tile, int page, float& k, float& v, bool& see) {
            see = page >= 0 && tile * kBN + cw * 32 + lane < p.prefix_len;
            const uint32_t row = row_at(tile, page, lane >> 4) + (lane & 15);
            k = see ? __ldg(p.c.ks + row) : 1.f;
            v = see ? __ldg(p.c.vs + row) : 0.f;
        };
        // Pieces in the order K0, K1, V0, K2, V1, ...: a tile's codes are on their way while the tile before
        // is converted, and its page number for a tile longer.
        bool ok = true, see;
        uint4 xk[8], xv[8];
        float ks, vs;
        int page0 = look_up(t0), page1 = look_up(t0 + 1), page2;  // of tiles j, j + 1, j + 2
        load(p.c.k, t0, page0, xk);
        load_scales(t0, page0, ks, vs, see);
        load(p.c.v, t0, page0, xv);
        page2 = look_up(t0 + 2);
#pragma unroll 1
        for (int j = 0; j <= n; ++j) {
            const int s = j & 1;
            if (j < n) {  // K of tile j
                if (j >= 2) ok = __all_sync(0xffffffffu, mbar_wait_sleep(&sm.k_empty[s], ((j >> 1) - 1) & 1, kSiteKEmpty));
                if (!ok) break;
                sm.ks[j & 3][cw * 32 + lane] = ks;
                sm.vs[j & 3][cw * 32 + lane] = vs;
                // (sizes: their bits order as they do; a NaN is neither the largest nor the smallest)
                const uint32_t size = __float_as_uint(fabsf(vs));
                const uint32_t most = __reduce_max_sync(0xffffffffu, vs == vs ? size : 0u);
                const uint32_t least = __reduce_min_sync(0xffffffffu, see && vs == vs ? size : 0x7f800000u);
                const uint32_t seen = __ballot_sync(0xffffffffu, see);
                if (lane == 0) {
                    sm.most[j & 3][cw] = __uint_as_float(most), sm.least[j & 3][cw] = __uint_as_float(least);
                    sm.hidden[j & 3][cw] = ~seen;
                }
                put(sm.k[s], xk);
                fence_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.k_full[s]);
                if (j + 1 < n) {
                    load(p.c.k, t0 + j + 1, page1, xk);
                    load_scales(t0 + j + 1, page1, ks, vs, see);
                }
            }
            if (j >= 1) {  // V of tile j - 1
                const int i = j - 1;
                if (i >= 2) ok = __all_sync(0xffffffffu, mbar_wait_sleep(&sm.v_empty[i & 1], ((i >> 1) - 1) & 1, kSiteVEmpty));
                if (!ok) break;
                put(sm.v[i & 1], xv);
                fence_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.v_full[i & 1]);
                if (j < n) load(p.c.v, t0 + j, page0, xv);
            }
            page0 = page1, page1 = page2;
            page2 = look_up(t0 + j + 3);
        }
    } else if (warp == kMmaWarp) {
        // ------------------------------ MMA issue ---------------------------
        if (lane == 0) {
            constexpr uint32_t idesc_qk = idesc_f16(kBM, kBN, 0);
            constexpr uint32_t idesc_pv = idesc_f16(kBM, kD, 1);
            bool ok = mbar_wait_sleep(&sm.q_full, 0, kSiteQ);
            int k_seen = 0, v_seen = 0;  // tiles whose K and V have been waited for
            auto want_k = [&](int t) {
                for (; ok && k_seen <= t; ++k_seen) ok = mbar_wait_sleep(&sm.k_full[k_seen & 1], (k_seen >> 1) & 1, kSiteKFull);
            };
            auto want_v = [&](int t) {
                for (; ok && v_seen <= t; ++v_seen) ok = mbar_wait_sleep(&sm.v_full[v_seen & 1], (v_seen >> 1) & 1, kSiteVFull);
            };
            // descriptors of the tiles' starts; offsets add to their address fields (in 16 bytes)
            const uint64_t q_desc = umma_desc_sw128(smem_u32(sm.q[0]), 16, 1024);
            const uint64_t k_desc = umma_desc_sw128(smem_u32(sm.k[0]), 16, 1024);
            const uint64_t v_desc = umma_desc_sw128(smem_u32(sm.v[0]), kHalfBytes, 1024);
            constexpr uint64_t kTileStep = kTileBytes >> 4;
            auto issue_s = [&](int i, int t) {
                const uint64_t k = k_desc + (t & 1) * kTileStep, q = q_desc + (pp.pairs ? 0 : i * kTileStep);
#pragma unroll
                for (int half = 0; half < (kF32 ? 2 : 1); ++half)
#pragma unroll
                    for (int kk = 0; kk < kD / 16; ++kk) {
                        constexpr uint64_t kHalfStep = kHalfBytes >> 4;
                        const uint64_t off = (kk >> 2) * kHalfStep + (kk & 3) * 2;
                        umma_ss(tmem + i * 128, q + half * kTileStep + off, k + off, idesc_qk, kk > 0 || half > 0 ? 1u : 0u);
                    }
                umma_commit(&sm.s_full[i]);
            };
            auto issue_pv = [&](int i, int t, bool add) {
                const uint64_t v = v_desc + (t & 1) * kTileStep;
#pragma unroll
                for (int half = 0; half < (kF32 ? 2 : 1); ++half)
#pragma unroll
                    for (int kk = 0; kk < kBN / 16; ++kk)
                        umma_ts(tmem + 256 + i * 128, tmem + i * 128 + (kF32 ? (kk >> 1) * 32 + half * 16 + (kk & 1) * 8 : kk * 8),
                                v + kk * (2048 >> 4), idesc_pv, (add || kk > 0 || half > 0) ? 1u : 0u);
            };
            auto tile_of = [&](int i, int s) { return pp.pairs ? 2 * s + i : s; };
            for (int i = 0; i < 2; ++i)
                if (steps[i] > 0) {
                    want_k(tile_of(i, 0));
                    if (!ok) break;
                    tc_fence_after();
                    issue_s(i, tile_of(i, 0));
                    if (pp.pairs || i == 1 || steps[1] == 0) umma_commit(&sm.k_empty[tile_of(i, 0) & 1]);
                }
            for (int s = 0; ok && s < steps[0]; ++s) {
                for (int i = 0; ok && i < 2; ++i) {
                    if (s >= steps[i]) continue;
                    const int t = tile_of(i, s), tn = tile_of(i, s + 1);
                    want_v(t);
                    if (ok && s + 1 < steps[i]) want_k(tn);
                    if (ok) ok = mbar_wait_sleep(&sm.p_full[i], s & 1, kSiteP);
                    if (!ok) break;
                    tc_fence_after();
                    issue_pv(i, t, s > 0);
                    const bool last_use = pp.pairs || i == 1 || steps[1] == 0;
                    if (last_use) umma_commit(&sm.v_empty[t & 1]);
                    if (s + 1 < steps[i]) {
                        issue_s(i, tn);
                        if (last_use) umma_commit(&sm.k_empty[tn & 1]);
                    } else {
                        umma_commit(&sm.o_full[i]);
                    }
                }
            }
            // all issued work is complete before TMEM is released
            umma_commit(&sm.mma_done);
            mbar_wait_sleep(&sm.mma_done, 0, kSiteDone);
        }
        __syncwarp();
    } else {
        // ------------------------------ softmax -----------------------------
        const int i = warp >> 2;  // warpgroup
        // The Q rows: 16 of a Q tile per warp and round, two lanes a row, 64 dims each.  (Few instructions: they
        // run once, and are fetched for that.)
        {
#pragma unroll 1
            for (int z = 0; z < (pp.pairs ? 1 : 2); ++z) {
                const int r = warp * 16 + (lane >> 1);  // row of the tile
                const int half = lane & 1;
                const int row = row0 + z * kBM + r;
                const bool in = row < pp.rows;
                const int bt = cache_attn::token_of(row, p.group);
                const int b = cache_attn::token_of(bt, p.T);
                const long long at = (long long)b * p.q_batch + (long long)(bt - b * p.T) * p.q_token +
                                     ((long long)hk * p.group + (row - bt * p.group)) * kD + 64 * half;
                constexpr int kPieces = kF32 ? 16 : 8;
                const uint4* src = kF32 ? reinterpret_cast<const uint4*>(static_cast<const float*>(p.q) + at)
                                        : reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.q) + at);
                uint4 x[kPieces];
#pragma unroll
                for (int i = 0; i < kPieces; ++i) x[i] = in ? __ldg(src + i) : make_uint4(0, 0, 0, 0);
                // largest magnitude as an integer: infinities and NaNs order above every finite value
                uint32_t top = 0;
#pragma unroll
                for (int i = 0; i < kPieces; ++i) {
                    const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        top = max(top, w[e] & 0x7fffffffu);
                        if (!kF32) top = max(top, (w[e] << 16) & 0x7fffffffu);
                    }
                }
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                if (!kF32) top &= 0xffff0000u;  // (the lower value's bits below an upper one's)
                const bool finite = top < 0x7f800000u;
                const int ex = finite ? max(exponent(__uint_as_float(top)), -100) : 0;
                // (a negative scale changes the queries' sign, so that factor stays positive)
                const float mul = finite ? (p.scale < 0.f ? -pow2(13 - ex) : pow2(13 - ex)) : 0.f;
                if (half == 0) sm.factor[z][r] = finite ? pow2(ex - 13) * fabsf(p.scale) * kLog2e : __uint_as_float(0x7fffffffu);
                const uint32_t dst = smem_u32(sm.q[z]) + (uint32_t)half * kHalfBytes + (uint32_t)r * 128;
#pragma unroll
                for (int c = 0; c < 8; ++c) {  // 16-byte chunks of the tile: 8 dims
                    float y[8];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (kF32) {
                            const uint4 u = x[(2 * c + (e >> 1)) % kPieces];
                            y[2 * e] = __uint_as_float(e & 1 ? u.z : u.x), y[2 * e + 1] = __uint_as_float(e & 1 ? u.w : u.y);
                        } else {
                            const uint32_t w = e == 0 ? x[c].x : e == 1 ? x[c].y : e == 2 ? x[c].z : x[c].w;
                            y[2 * e] = __uint_as_float(w << 16), y[2 * e + 1] = __uint_as_float(w & 0xffff0000u);
                        }
                    }
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float y0 = finite ? y[2 * e] * mul : 0.f, y1 = finite ? y[2 * e + 1] * mul : 0.f;
                        if (kF32) cache_attn::split_pair(y0, y1, hi[e], lo[e]);
                        else hi[e] = half_pair(y0, y1);
                    }
                    const uint32_t to = dst + ((uint32_t)(c ^ (r & 7)) << 4);
                    st_shared_v4(to, hi[0], hi[1], hi[2], hi[3]);
                    if (kF32) st_shared_v4(to + kTileBytes, lo[0], lo[1], lo[2], lo[3]);
                }
            }
            fence_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.q_full);
            named_bar_sync(1, 256);  // factors of all rows
        }
        const int r = (warp & 3) * 32 + lane;
        const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t tS = tmem + lane_off + i * 128;
        const uint32_t tO = tmem + lane_off + 256 + i * 128;
        float factor = sm.factor[pp.pairs ? 0 : i][r];
        if (factor == 0.f) factor = __uint_as_float(1u);  // 2^-149: no 0 * -inf where a key is hidden; scores of 2^-22 at most weigh as 0 do
        // Weights are computed as p * f, and O holds sums with that factor.
        float m = -INFINITY, l = 0.f, mx = -INFINITY;
        int fe = kFirstFactor;  // f = 2^fe
        const bool idle = row0 + (pp.pairs ? 0 : i * kBM) + (warp & 3) * 32 >= pp.rows;  // no query in this warp's rows
        bool ok = true;
        for (int s = 0; s < steps[i]; ++s) {
            // warp-uniform, since the step synchronises the warp
            if (!__all_sync(0xffffffffu, mbar_wait_sleep(&sm.s_full[i], s & 1, kSiteS))) { ok = false; break; }
            if (idle) {  // (what stays in their P rows reaches only their O rows)
                if (lane == 0) mbar_arrive(&sm.p_full[i]);
                continue;
            }
            tc_fence_after();
            const int at = (pp.pairs ? 2 * s + i : s) & 3;
            const uint4 hidden = *reinterpret_cast<const uint4*>(sm.hidden[at]);
            const bool some = (hidden.x | hidden.y | hidden.z | hidden.w) != 0u;
            if (some) {  // the last tile, or a page that does not exist: hidden scores become -inf
#pragma unroll 1
                for (int cc = 0; cc < 8; ++cc) {
                    float x[16];
                    tmem_ld16(tS + cc * 16, x);
                    tmem_wait_ld();
                    const uint32_t bits = sm.hidden[at][cc >> 1] >> (16 * (cc & 1));
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if ((bits >> e) & 1u) x[e] = -INFINITY;
                    tmem_st16(tS + cc * 16, *reinterpret_cast<uint32_t(*)[16]>(x));
                }
                tmem_wait_st();
            }
            // first pass: the row's largest score (the next 32 columns are on their way while 32 are looked at)
            float top = -INFINITY;
            float xa[32], xb[32];
            auto largest = [&](const float(&x)[32], int cc) {
                float best[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int e = 0; e < 32; e += 4) {
                    const float4 k = *reinterpret_cast<const float4*>(&sm.ks[at][cc * 32 + e]);
                    float y[4];
                    f2_unpack(f2_mul(f2_pack(x[e], x[e + 1]), f2_pack(k.x, k.y)), y[0], y[1]);
                    f2_unpack(f2_mul(f2_pack(x[e + 2], x[e + 3]), f2_pack(k.z, k.w)), y[2], y[3]);
                    best[(e >> 2) & 3] = fmax3(best[(e >> 2) & 3], fmaxf(y[0], y[1]), fmaxf(y[2], y[3]));
                }
                top = fmax3(top, fmaxf(best[0], best[1]), fmaxf(best[2], best[3]));
            };
            tmem_ld32(tS, xa);
#pragma unroll 1
            for (int cc = 0; cc < 4; cc += 2) {
                wait_for(xa);
                tmem_ld32(tS + cc * 32 + 32, xb);
                largest(xa, cc);
                wait_for(xb);
                if (cc == 0) tmem_ld32(tS + 64, xa);
                largest(xb, cc + 1);
            }
            top *= factor;  // (-inf where every key is hidden; factor is not negative)
            if (top != top) top = -INFINITY;  // (a row whose query is not finite: no maximum)
            mx = fmaxf(mx, top);
            int d = 0;  // log2 of the maximum's change: whole maxima change the sums by powers of two
            if (top > m + kGrow) {
                const float whole = ceilf(top);
                if (m != -INFINITY) d = (int)fminf(whole - m, 1000.f);
                m = whole;
                l *= cache_attn::pow2_or_0(-d);
            }
            // The row's largest p * v_scale in this tile is below 2^eb.  By the largest score and the largest scale, where
            // scales are within a factor of kNear; else from the products themselves, since the key of the largest
            // score may have a row of V that is small, or zeros.
            const float4 most4 = *reinterpret_cast<const float4*>(sm.most[at]), least4 = *reinterpret_cast<const float4*>(sm.least[at]);
            const float most = fmaxf(fmaxf(most4.x, most4.y), fmaxf(most4.z, most4.w));
            const float least = fminf(fminf(least4.x, least4.y), fminf(least4.z, least4.w));
            int eb = (int)ceilf(fminf(fmaxf(top - m, -1000.f), 1000.f)) + exponent(most) + 1;
            if (most > kNear * least) {  // (the same for all rows)
                float z = -INFINITY;
#pragma unroll 1
                for (int cc = 0; cc < 8; ++cc) {
                    float x[16];
                    tmem_ld16(tS + cc * 16, x);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        z = fmaxf(z, fmaf(x[e] * sm.ks[at][cc * 16 + e], factor, __log2f(fabsf(sm.vs[at][cc * 16 + e]))));
                }
                eb = (int)ceilf(fminf(fmaxf(z - m, -1000.f), 1000.f)) + 1;
            }
            // f grows as p shrinks, up to its first value, so that the largest weights summed so far stay where they are in
            // fp16's range, and so does O; new ones at or above 2^15 lower it.
            int fn = min(fe + d, kFirstFactor);
            if (eb + fn > 15) fn = max(kLowered - eb, -120);
            const int change = fn - fe - d;  // <= 0
            fe = fn;
            if (s > 0 && __any_sync(0xffffffffu, change != 0)) {
                const float by = cache_attn::pow2_or_0(change);
#pragma unroll 1
                for (int cc = 0; cc < 8; ++cc) {
                    float o[16];
                    tmem_ld16(tO + cc * 16, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[e] *= by;
                    tmem_st16(tO + cc * 16, *reinterpret_cast<uint32_t(*)[16]>(o));
                }
            }
            // second pass: weights
            tmem_ld32(tS, xa);
            const float m_safe = (m == -INFINITY ? 0.f : m) - (float)fe;  // exponents are those of p * f
            const uint64_t c2 = f2_pack(factor, factor), nm2 = f2_pack(-m_safe, -m_safe);
            uint64_t sum2[2] = {f2_pack(0.f, 0.f), f2_pack(0.f, 0.f)};
            auto weigh = [&](const float(&x)[32], int cc) {
                uint32_t hi[16], lo[kF32 ? 16 : 1];
#pragma unroll
                for (int e = 0; e < 32; e += 4) {
                    const float4 k = *reinterpret_cast<const float4*>(&sm.ks[at][cc * 32 + e]);
                    const float4 v = *reinterpret_cast<const float4*>(&sm.vs[at][cc * 32 + e]);
                    float y[4];
                    f2_unpack(f2_fma_full(f2_mul(f2_pack(x[e], x[e + 1]), f2_pack(k.x, k.y)), c2, nm2), y[0], y[1]);
                    f2_unpack(f2_fma_full(f2_mul(f2_pack(x[e + 2], x[e + 3]), f2_pack(k.z, k.w)), c2, nm2), y[2], y[3]);
                    const uint64_t p0 = f2_pack(ex2_approx(y[0]), ex2_approx(y[1])), p1 = f2_pack(ex2_approx(y[2]), ex2_approx(y[3]));
                    sum2[0] = f2_add(sum2[0], p0);
                    sum2[1] = f2_add(sum2[1], p1);
                    float u[4];
                    f2_unpack(f2_mul(p0, f2_pack(v.x, v.y)), u[0], u[1]);
                    f2_unpack(f2_mul(p1, f2_pack(v.z, v.w)), u[2], u[3]);
                    if (kF32) {
                        cache_attn::split_pair(u[0], u[1], hi[e / 2], lo[kF32 ? e / 2 : 0]);
                        cache_attn::split_pair(u[2], u[3], hi[e / 2 + 1], lo[kF32 ? e / 2 + 1 : 0]);
                    } else {
                        hi[e / 2] = half_pair(u[0], u[1]);
                        hi[e / 2 + 1] = half_pair(u[2], u[3]);
                    }
                }
                // P takes the columns of scores that have been read: chunk cc's 16 (and the rests' 16 behind them)
                tmem_st16(tS + cc * (kF32 ? 32 : 16), hi);
                if (kF32) tmem_st16(tS + cc * 32 + 16, *reinterpret_cast<uint32_t(*)[16]>(lo));
            };
#pragma unroll 1
            for (int cc = 0; cc < 4; cc += 2) {
                wait_for(xa);
                tmem_ld32(tS + cc * 32 + 32, xb);
                weigh(xa, cc);
                wait_for(xb);
                if (cc == 0) tmem_ld32(tS + 64, xa);
                weigh(xb, cc + 1);
            }
            float s0, s1;
            f2_unpack(f2_add(sum2[0], sum2[1]), s0, s1);
            l = fmaf(s0 + s1, pow2(-fe), l);
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.p_full[i]);
        }
        // ---- the rows' sums, in units of 2^-m
        bool have = false;
        if (steps[i] > 0 && ok) have = mbar_wait_sleep(&sm.o_full[i], 0, kSiteO);
        have = __all_sync(0xffffffffu, have);
        if (have) tc_fence_after();
        const float inv = pow2(-fe);
        named_bar_sync(1, 256);  // both warpgroups' products are done: the K tiles are free
        if (pp.pairs) {
            // the second warpgroup's rows go through shared memory (64 KB: K's two tiles) to the first's
            float4* mine = reinterpret_cast<float4*>(sm.k[0]) + r * (kD / 4);
            if (i == 1) {
                if (have) {
#pragma unroll 1
                    for (int cc = 0; cc < 4; ++cc) {
                        float o[32];
                        tmem_ld32(tO + cc * 32, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            mine[(cc * 8 + e) ^ (r & 7)] = make_float4(o[4 * e] * inv, o[4 * e + 1] * inv, o[4 * e + 2] * inv, o[4 * e + 3] * inv);
                    }
                }
                sm.m[r] = have ? m : -INFINITY, sm.l[r] = have ? l : 0.f, sm.mx[r] = have ? mx : -INFINITY;
            }
            named_bar_sync(1, 256);
        }
        if (i == 0 || !pp.pairs) {
            const int row = row0 + (pp.pairs ? 0 : i * kBM) + r;
            const bool in = row < pp.rows && have;
            const int bt = in ? cache_attn::token_of(row, p.group) : 0;
            const long long rows = (long long)p.B * p.T * p.heads;
            const long long at = (long long)part * rows + (long long)bt * p.heads + (long long)hk * p.group + (in ? row - bt * p.group : 0);
            float a0 = inv, a1 = 0.f, best = m, sum = l, big = mx;
            const bool both = pp.pairs && steps[1] > 0;
            if (both) {
                const float m1 = sm.m[r], l1 = sm.l[r];
                best = fmaxf(m, m1);
                const float e0 = m == -INFINITY ? 1.f : ex2_approx(m - best), e1 = m1 == -INFINITY ? 1.f : ex2_approx(m1 - best);
                a0 = inv * e0;
                a1 = e1;
                sum = l * e0 + l1 * e1;
                big = fmaxf(mx, sm.mx[r]);
            }
            const float4* other = reinterpret_cast<const float4*>(sm.k[0]) + r * (kD / 4);
            float4* dst = reinterpret_cast<float4*>(p.shared_o + at * kD);
#pragma unroll 1
            for (int cc = 0; cc < 4; ++cc) {
                float o[32];
                if (have) {
                    tmem_ld32(tO + cc * 32, o);
                    tmem_wait_ld();
                }
                if (in) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        float4 y = make_float4(o[4 * e] * a0, o[4 * e + 1] * a0, o[4 * e + 2] * a0, o[4 * e + 3] * a0);
                        if (both) {
                            const float4 z = other[(cc * 8 + e) ^ (r & 7)];
                            y.x = fmaf(z.x, a1, y.x), y.y = fmaf(z.y, a1, y.y), y.z = fmaf(z.z, a1, y.z), y.w = fmaf(z.w, a1, y.w);
                        }
                        dst[cc * 8 + e] = y;
                    }
                }
            }
            if (in) p.shared_s[at] = make_float4(best, sum, big, 0.f);
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

}  // namespace prefix_attn
}  // namespace dt
