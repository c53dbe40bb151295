// Attention of new tokens over the quantised K/V cache.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale * q . k_j - m),  m = max_j scale * q . k_j
//
// over the keys j < seq_len - q_len + t + 1 that query t of a sequence sees (its own token is
// the cache's last but q_len - t - 1), after all `prefix_len` keys of a prefix that every
// sequence shares.  Rows with no key, and padding rows t >= q_len, are written as zeros with
// m = l = 0.
#pragma once
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

}  // namespace cache_attn
}  // namespace dt
