// extern "C" layer of the serving operators: the quantised K/V cache, the attention that
// reads it, and token log probabilities.  Included by capi.cu, whose error handling and
// launch helpers it uses.
#pragma once

namespace {

int check_cache(const dt_kv_cache* c, dt::kv::Cache* out) {
    if (!c) return fail(DT_ERR_INVALID_ARGUMENT, "null cache");
    if (c->format != DT_KV_INT8 && c->format != DT_KV_E4M3)
        return fail(DT_ERR_INVALID_ARGUMENT, "cache format must be DT_KV_INT8 or DT_KV_E4M3");
    if (c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1)))
        return fail(DT_ERR_INVALID_ARGUMENT, "page_size must be 16, 32, 64, 128 or 256");
    if (c->num_pages < 1 || c->kv_heads < 1 || c->kv_heads > 1024)
        return fail(DT_ERR_INVALID_ARGUMENT, "num_pages must be >= 1 and kv_heads 1..1024");
    if ((long long)c->num_pages * c->kv_heads * c->page_size > 0x7fffffffll)
        return fail(DT_ERR_INVALID_ARGUMENT, "num_pages * kv_heads * page_size must be below 2^31");
    if (!c->k || !c->v || !c->k_scale || !c->v_scale) return fail(DT_ERR_INVALID_ARGUMENT, "null cache array");
    if (!aligned16(c->k) || !aligned16(c->v) || !aligned16(c->k_scale) || !aligned16(c->v_scale))
        return fail(DT_ERR_INVALID_ARGUMENT, "cache arrays must be 16-byte aligned");
    out->k = static_cast<uint8_t*>(c->k);
    out->v = static_cast<uint8_t*>(c->v);
    out->ks = c->k_scale;
    out->vs = c->v_scale;
    out->pages = c->num_pages;
    out->heads = c->kv_heads;
    int shift = 4;
    while ((1 << shift) < c->page_size) ++shift;
    out->page_shift = shift;
    return DT_OK;
}

int check_table(const int* table, long long stride, int max_pages, int B) {
    if (max_pages < 0 || stride < max_pages)
        return fail(DT_ERR_INVALID_ARGUMENT, "page_table_stride must be >= max_pages >= 0");
    if (!table && max_pages > 0 && B > 0) return fail(DT_ERR_INVALID_ARGUMENT, "null page_table");
    return DT_OK;
}

// A row of values starts on a 16-byte boundary whatever its token and sequence.
int check_strides(const char* name, const void* p, long long batch, long long token, int elem_bytes) {
    const long long step = 16 / elem_bytes;
    if (!p || !aligned16(p)) return fail(DT_ERR_INVALID_ARGUMENT, "%s must be non-null and 16-byte aligned", name);
    if (batch % step || token % step || batch < 0 || token < 0)
        return fail(DT_ERR_INVALID_ARGUMENT, "%s strides must be non-negative multiples of 16 bytes", name);
    return DT_OK;
}

}  // namespace

extern "C" {

int dt_kv_cache_append(const dt_kv_cache* cache, const void* k, long long k_batch_stride, long long k_token_stride,
                       const void* v, long long v_batch_stride, long long v_token_stride, int src_f32,
                       const int* page_table, long long page_table_stride, int max_pages, const int* start,
                       const int* lens, int B, int T, void* stream) {
    t_last_error.clear();
    dt::kv::AppendParams p{};
    DT_TRY(check_cache(cache, &p.c));
    if (B < 0 || T < 0) return fail(DT_ERR_INVALID_ARGUMENT, "B and T must be >= 0");
    if (B == 0 || T == 0) return DT_OK;
    DT_TRY(check_table(page_table, page_table_stride, max_pages, B));
    const int elem = src_f32 ? 4 : 2;
    DT_TRY(check_strides("k", k, k_batch_stride, k_token_stride, elem));
    DT_TRY(check_strides("v", v, v_batch_stride, v_token_stride, elem));
    p.s = {page_table, page_table_stride, max_pages, start, lens, B, T};
    p.k = k;
    p.v = v;
    p.k_batch = k_batch_stride;
    p.k_token = k_token_stride;
    p.v_batch = v_batch_stride;
    p.v_token = v_token_stride;
    int dev;
    DT_TRY(prepare_device(&dev));
    p.tile = (long long)B * T > 148 * 8 ? 8 : 1;
    p.tiles = (T + p.tile - 1) / p.tile;
    if ((long long)p.tiles * B > 0x7fffffffll) return fail(DT_ERR_INVALID_ARGUMENT, "B * T is too large");
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const dim3 grid((unsigned)(p.tiles * B)), block(dt::kv::kThreads);
    if (cache->format == DT_KV_INT8)
        return src_f32 ? launch_pdl(dt::kv::append_kernel<0, true>, grid, block, 0, st, p)
                       : launch_pdl(dt::kv::append_kernel<0, false>, grid, block, 0, st, p);
    return src_f32 ? launch_pdl(dt::kv::append_kernel<1, true>, grid, block, 0, st, p)
                   : launch_pdl(dt::kv::append_kernel<1, false>, grid, block, 0, st, p);
}

int dt_kv_cache_read(const dt_kv_cache* cache, void* k, void* v, int dst_f32, const int* page_table,
                     long long page_table_stride, int max_pages, const int* start, const int* lens, int B, int T,
                     void* stream) {
    t_last_error.clear();
    dt::kv::ReadParams p{};
    DT_TRY(check_cache(cache, &p.c));
    if (B < 0 || T < 0) return fail(DT_ERR_INVALID_ARGUMENT, "B and T must be >= 0");
    if (B == 0 || T == 0) return DT_OK;
    DT_TRY(check_table(page_table, page_table_stride, max_pages, B));
    if (!k || !v || !aligned16(k) || !aligned16(v))
        return fail(DT_ERR_INVALID_ARGUMENT, "k and v must be non-null and 16-byte aligned");
    p.s = {page_table, page_table_stride, max_pages, start, lens, B, T};
    p.k = k;
    p.v = v;
    p.rows = (long long)B * T * 2 * p.c.heads;
    int dev;
    DT_TRY(prepare_device(&dev));
    const long long blocks = std::min<long long>((p.rows + dt::kv::kRows - 1) / dt::kv::kRows, 148 * 32);
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const dim3 grid((unsigned)blocks), block(dt::kv::kThreads);
    if (cache->format == DT_KV_INT8)
        return dst_f32 ? launch_pdl(dt::kv::read_kernel<0, true>, grid, block, 0, st, p)
                       : launch_pdl(dt::kv::read_kernel<0, false>, grid, block, 0, st, p);
    return dst_f32 ? launch_pdl(dt::kv::read_kernel<1, true>, grid, block, 0, st, p)
                   : launch_pdl(dt::kv::read_kernel<1, false>, grid, block, 0, st, p);
}

}  // extern "C"

namespace {

constexpr int kPlanSms = 148;  // B200; the plan is made without a device, for the workspace size

// How the split kernel's work is cut: see the rules at plan_split.
struct SplitPlan {
    bool wide;       // 16 query rows per CTA
    long long items; // (sequence, K/V head, rows) that a cluster or a group of CTAs takes
    int split;       // CTAs per item
    bool parts;      // joined through the workspace
};

#ifndef DT_ATTN_FORCE_SPLIT
#define DT_ATTN_FORCE_SPLIT 0
#endif
SplitPlan plan_split(int B, int T, int heads, int kv_heads, int q_f32, int page_size, int max_pages) {
    namespace ca = dt::cache_attn;
    SplitPlan s{};
    const int rows = T * (heads / kv_heads);
    s.wide = !q_f32 && rows > 8;
    s.items = (long long)B * kv_heads * ((rows + (s.wide ? 15 : 7)) / (s.wide ? 16 : 8));
    const long long tiles = ((long long)max_pages * page_size + ca::kTile - 1) / ca::kTile;
    const long long slots = 3 * kPlanSms;
    s.split = 1;
    while (s.split < ca::kMaxCluster && s.items * s.split * 2 <= slots && tiles > (long long)s.split * ca::kWarps) s.split *= 2;
    if (s.split == ca::kMaxCluster && s.items * s.split * 2 <= slots && tiles > 4ll * s.split * ca::kWarps) {
        s.parts = true;
        s.split = (int)std::min(slots / s.items, tiles / (2 * ca::kWarps));
    }
    if (DT_ATTN_FORCE_SPLIT) s.split = DT_ATTN_FORCE_SPLIT, s.parts = false;
    return s;
}

size_t parts_bytes(long long parts, int B, int T, int heads) {
    const size_t rows = (size_t)B * T * heads;
    return align256(parts * rows * 16) + align256(parts * rows * dt::cache_attn::kD * 4);
}

int launch_split(void (*kernel)(dt::cache_attn::Params), const dt::cache_attn::Params& p, long long items,
                 cudaStream_t st) {
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = DT_PDL;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = p.part_o ? 1u : (unsigned)p.split;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(items * p.split));
    cfg.blockDim = dim3(dt::cache_attn::kThreads);
    cfg.dynamicSmemBytes = sizeof(dt::cache_attn::Smem);
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    DT_CUDA(cudaLaunchKernelEx(&cfg, kernel, p));
    return DT_OK;
}

int launch_join(const dt::cache_attn::Params& p, int q_f32, cudaStream_t st) {
    const dim3 grid((unsigned)(((long long)p.B * p.T * p.heads + 3) / 4)), block(128);
    return q_f32 ? launch_pdl(dt::cache_attn::join_kernel<true>, grid, block, 0, st, p)
                 : launch_pdl(dt::cache_attn::join_kernel<false>, grid, block, 0, st, p);
}

template <int kFmt>
void (*split_kernel_of(bool f32, bool wide))(dt::cache_attn::Params) {
    namespace ca = dt::cache_attn;
    return f32 ? ca::split_kernel<kFmt, true, false> : wide ? ca::split_kernel<kFmt, false, true> : ca::split_kernel<kFmt, false, false>;
}

// Per-device attributes of the kernels below (called with g_mu held, from ensure_attrs).
int serving_attrs() {
    for (int i = 0; i < 6; ++i) {
        auto* k = i & 1 ? split_kernel_of<1>(i >= 4, i >= 2) : split_kernel_of<0>(i >= 4, i >= 2);
        DT_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(dt::cache_attn::Smem)));
    }
    return DT_OK;
}

void set_parts(dt::cache_attn::Params& p, int parts, void* workspace) {
    p.n_parts = parts;
    p.part_s = static_cast<float4*>(workspace);
    p.part_o = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + align256((size_t)parts * p.B * p.T * p.heads * 16));
}

int cache_attn(const dt_kv_cache* cache, const void* q, long long q_batch_stride, long long q_token_stride, int q_f32,
               void* o, float* m, float* l, const int* prefix_pages, int prefix_len, const int* page_table,
               long long page_table_stride, int max_pages, const int* seq_lens, const int* q_lens, int B, int T,
               int heads, float scale, void* workspace, size_t workspace_bytes, void* stream) {
    dt::cache_attn::Params p{};
    DT_TRY(check_cache(cache, &p.c));
    if (B < 0 || T < 0 || heads < 0) return fail(DT_ERR_INVALID_ARGUMENT, "B, T and heads must be >= 0");
    if (heads % cache->kv_heads)
        return fail(DT_ERR_INVALID_ARGUMENT, "heads (%d) must be a multiple of kv_heads (%d)", heads, cache->kv_heads);
    if (B == 0 || T == 0 || heads == 0) return DT_OK;
    DT_TRY(check_table(page_table, page_table_stride, max_pages, B));
    if (!seq_lens && max_pages > 0) return fail(DT_ERR_INVALID_ARGUMENT, "null seq_lens");
    DT_TRY(check_strides("q", q, q_batch_stride, q_token_stride, q_f32 ? 4 : 2));
    if (!o || !aligned16(o)) return fail(DT_ERR_INVALID_ARGUMENT, "o must be non-null and 16-byte aligned");
    if (prefix_len < 0 || (prefix_len > 0 && !prefix_pages))
        return fail(DT_ERR_INVALID_ARGUMENT, "prefix_len must be >= 0, with its pages");
    if ((long long)B * T * heads > 0x7fffffffll) return fail(DT_ERR_INVALID_ARGUMENT, "B * T * heads must be below 2^31");
    p.q = q;
    p.q_batch = q_batch_stride;
    p.q_token = q_token_stride;
    p.o = o;
    p.m_out = m;
    p.l_out = l;
    p.table = page_table;
    p.table_stride = page_table_stride;
    p.max_pages = max_pages;
    p.seq_lens = seq_lens;
    p.q_lens = q_lens;
    p.prefix_pages = prefix_pages;
    p.prefix_len = prefix_len;
    p.B = B;
    p.T = T;
    p.heads = heads;
    p.group = heads / cache->kv_heads;
    p.scale = scale;
    const size_t need = prefix_len > 0 ? dt_prefix_attn_workspace_bytes(B, T, heads, cache->kv_heads, prefix_len)
                                       : dt_cache_attn_workspace_bytes(B, T, heads, cache->kv_heads, q_f32,
                                                                       cache->page_size, max_pages);
    if (need > 0 && (!workspace || workspace_bytes < need || !aligned16(workspace)))
        return fail(DT_ERR_INVALID_ARGUMENT, "workspace must be >= %zu bytes and 16-byte aligned", need);
    int dev;
    DT_TRY(prepare_device(&dev));
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (prefix_len == 0) {
        const SplitPlan plan = plan_split(B, T, heads, cache->kv_heads, q_f32, cache->page_size, max_pages);
        if (plan.items * plan.split > 0x7fffffffll)
            return fail(DT_ERR_INVALID_ARGUMENT, "B * kv_heads * query rows is too large");
        p.split = plan.split;
        if (plan.parts) set_parts(p, plan.split, workspace);
        DT_TRY(launch_split(cache->format == DT_KV_INT8 ? split_kernel_of<0>(q_f32, plan.wide) : split_kernel_of<1>(q_f32, plan.wide),
                            p, plan.items, st));
        return plan.parts ? launch_join(p, q_f32, st) : DT_OK;
    }
    const dim3 grid((unsigned)(((long long)B * T * heads + 3) / 4)), block(128);
    if (cache->format == DT_KV_INT8)
        return q_f32 ? launch_pdl(dt::cache_attn::row_kernel<0, true>, grid, block, 0, st, p)
                     : launch_pdl(dt::cache_attn::row_kernel<0, false>, grid, block, 0, st, p);
    return q_f32 ? launch_pdl(dt::cache_attn::row_kernel<1, true>, grid, block, 0, st, p)
                 : launch_pdl(dt::cache_attn::row_kernel<1, false>, grid, block, 0, st, p);
}

}  // namespace

extern "C" {

int dt_cache_attn_fwd(const dt_kv_cache* cache, const void* q, long long q_batch_stride, long long q_token_stride,
                      int q_f32, void* o, float* softmax_m, float* softmax_l, const int* page_table,
                      long long page_table_stride, int max_pages, const int* seq_lens, const int* q_lens, int B, int T,
                      int heads, float scale, void* workspace, size_t workspace_bytes, void* stream) {
    t_last_error.clear();
    return cache_attn(cache, q, q_batch_stride, q_token_stride, q_f32, o, softmax_m, softmax_l, nullptr, 0, page_table,
                      page_table_stride, max_pages, seq_lens, q_lens, B, T, heads, scale, workspace, workspace_bytes,
                      stream);
}

size_t dt_cache_attn_workspace_bytes(int B, int T, int heads, int kv_heads, int q_f32, int page_size, int max_pages) {
    if (B <= 0 || T <= 0 || kv_heads <= 0 || heads < kv_heads || page_size <= 0 || max_pages <= 0) return 0;
    if ((long long)B * T * heads > 0x7fffffffll) return 0;
    const SplitPlan plan = plan_split(B, T, heads, kv_heads, q_f32, page_size, max_pages);
    return plan.parts ? parts_bytes(plan.split, B, T, heads) : 0;
}

size_t dt_prefix_attn_workspace_bytes(int B, int T, int heads, int kv_heads, int prefix_len) {
    if (B <= 0 || T <= 0 || heads <= 0 || kv_heads <= 0 || prefix_len <= 0) return 0;
    return 0;
}

int dt_prefix_attn_fwd(const dt_kv_cache* cache, const void* q, long long q_batch_stride, long long q_token_stride,
                       int q_f32, void* o, float* softmax_m, float* softmax_l, const int* prefix_pages, int prefix_len,
                       const int* page_table, long long page_table_stride, int max_pages, const int* seq_lens,
                       const int* q_lens, int B, int T, int heads, float scale, void* workspace, size_t workspace_bytes,
                       void* stream) {
    t_last_error.clear();
    return cache_attn(cache, q, q_batch_stride, q_token_stride, q_f32, o, softmax_m, softmax_l, prefix_pages,
                      prefix_len, page_table, page_table_stride, max_pages, seq_lens, q_lens, B, T, heads, scale,
                      workspace, workspace_bytes, stream);
}

int dt_token_log_probs(const void* logits, int logits_f32, long long ld, int N, int V, const void* targets,
                       int targets_int64, int top, float* log_prob, float* entropy, float* lse, int* top_ids,
                       float* top_log_probs, void* stream) {
    t_last_error.clear();
    if (N < 0 || V < 1) return fail(DT_ERR_INVALID_ARGUMENT, "N must be >= 0 and V >= 1");
    if (top < 0 || top > dt::logprobs::kMaxTop || top > V)
        return fail(DT_ERR_INVALID_ARGUMENT, "top must be 0..%d and at most V", dt::logprobs::kMaxTop);
    if (N == 0) return DT_OK;
    if (!logits || ld < V) return fail(DT_ERR_INVALID_ARGUMENT, "logits must be non-null with ld >= V");
    if (reinterpret_cast<uintptr_t>(logits) % (logits_f32 ? 4 : 2))
        return fail(DT_ERR_INVALID_ARGUMENT, "logits must be aligned to their type");
    if (top > 0 && (!top_ids || !top_log_probs)) return fail(DT_ERR_INVALID_ARGUMENT, "null top_ids/top_log_probs");
    if (log_prob && !targets) return fail(DT_ERR_INVALID_ARGUMENT, "log_prob needs targets");
    int dev;
    DT_TRY(prepare_device(&dev));
    dt::logprobs::Params p{logits, ld, N, V, targets, targets_int64 ? 1 : 0, top, log_prob, entropy, lse, top_ids,
                           top_log_probs};
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const dim3 grid((unsigned)N), block(dt::logprobs::kThreads);
    return logits_f32 ? launch_pdl(dt::logprobs::row_kernel<true>, grid, block, 0, st, p)
                      : launch_pdl(dt::logprobs::row_kernel<false>, grid, block, 0, st, p);
}

int dt_token_log_probs_bwd(const void* logits, int logits_f32, long long ld, int N, int V, const void* targets,
                           int targets_int64, const float* lse, const float* entropy, const float* d_log_prob,
                           const float* d_entropy, void* d_logits, long long d_ld, void* stream) {
    t_last_error.clear();
    if (N < 0 || V < 1) return fail(DT_ERR_INVALID_ARGUMENT, "N must be >= 0 and V >= 1");
    if (N == 0) return DT_OK;
    if (!logits || !d_logits || ld < V || d_ld < V)
        return fail(DT_ERR_INVALID_ARGUMENT, "logits and d_logits must be non-null with ld >= V");
    const uintptr_t mask = logits_f32 ? 3 : 1;
    if ((reinterpret_cast<uintptr_t>(logits) & mask) || (reinterpret_cast<uintptr_t>(d_logits) & mask))
        return fail(DT_ERR_INVALID_ARGUMENT, "logits and d_logits must be aligned to their type");
    if (!lse) return fail(DT_ERR_INVALID_ARGUMENT, "null lse");
    if (d_log_prob && !targets) return fail(DT_ERR_INVALID_ARGUMENT, "d_log_prob needs targets");
    if (d_entropy && !entropy) return fail(DT_ERR_INVALID_ARGUMENT, "d_entropy needs entropy");
    int dev;
    DT_TRY(prepare_device(&dev));
    dt::logprobs::GradParams p{logits, ld, N, V, targets, targets_int64 ? 1 : 0, lse, entropy, d_log_prob, d_entropy,
                               d_logits, d_ld};
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const dim3 grid((unsigned)N), block(dt::logprobs::kThreads);
    return logits_f32 ? launch_pdl(dt::logprobs::grad_kernel<true>, grid, block, 0, st, p)
                      : launch_pdl(dt::logprobs::grad_kernel<false>, grid, block, 0, st, p);
}

}  // extern "C"
