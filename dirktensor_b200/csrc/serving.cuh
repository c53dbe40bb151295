// extern "C" layer of the serving operators: the quantised K/V cache, the attention that
// reads it, and token log probabilities.  Included by capi.cu, whose error handling and
// launch helpers it uses.
#pragma once

namespace {

constexpr int kPlanSms = 148;  // B200; the plan is made without a device, for the workspace size

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

// Whether no two of a cache's arrays share memory.
bool arrays_apart(const dt_kv_cache* c) {
    const size_t rows = (size_t)c->num_pages * c->kv_heads * c->page_size;
    const struct { const void* at; size_t bytes; } a[4] = {
        {c->k, rows * dt::kv::kD}, {c->v, rows * dt::kv::kD}, {c->k_scale, rows * 4}, {c->v_scale, rows * 4}};
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < i; ++j) {
            const uintptr_t x = reinterpret_cast<uintptr_t>(a[i].at), y = reinterpret_cast<uintptr_t>(a[j].at);
            if (x < y ? y - x < a[i].bytes : x - y < a[j].bytes) return false;
        }
    return true;
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
    if (!arrays_apart(cache)) return fail(DT_ERR_INVALID_ARGUMENT, "cache arrays that are written must not overlap");
    p.k_batch = k_batch_stride;
    p.k_token = k_token_stride;
    p.v_batch = v_batch_stride;
    p.v_token = v_token_stride;
    // Page entries of a sequence's tokens, and how many sequences, and tokens of one, a launch takes: later ones write
    // after it, as the highest (b, position) is to.
    const int width = T / cache->page_size + 2;
    if ((long long)width * B > 0x7fffffffll) return fail(DT_ERR_INVALID_ARGUMENT, "B * T is too large");
    const int seqs = std::max(1, dt::kv::kEntries / width);
    const int tokens = width <= dt::kv::kEntries ? T : (dt::kv::kEntries - 2) * cache->page_size;
    // A CTA takes 32 rows at a time: as many tokens as that are, or up to four times so many where there are more CTAs than
    // the GPU holds (8 per SM); at most 16, the smallest page.
    const long long rows = 2ll * std::min(B, seqs) * std::min(T, tokens) * p.c.heads;
    const int once = std::max(1, dt::kv::kRows / (2 * p.c.heads));
    const int times = (int)std::min<long long>(4, std::max<long long>(1, rows / (dt::kv::kRows * 8ll * kPlanSms)));
    p.tile = std::min(16, once * times);
    int dev;
    DT_TRY(prepare_device(&dev));
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    typedef void (*AppendKernel)(dt::kv::AppendParams);
    const bool e4m3 = cache->format == DT_KV_E4M3;
    const AppendKernel from_first = e4m3 ? (src_f32 ? dt::kv::append_kernel<1, true, false> : dt::kv::append_kernel<1, false, false>)
                                         : (src_f32 ? dt::kv::append_kernel<0, true, false> : dt::kv::append_kernel<0, false, false>);
    const AppendKernel later = e4m3 ? (src_f32 ? dt::kv::append_kernel<1, true, true> : dt::kv::append_kernel<1, false, true>)
                                    : (src_f32 ? dt::kv::append_kernel<0, true, true> : dt::kv::append_kernel<0, false, true>);
    for (int b = 0; b < B; b += std::min(seqs, B - b))
        for (int t = 0; t < T; t += std::min(tokens, T - t)) {
            const int n = std::min(seqs, B - b), len = std::min(tokens, T - t);
            p.s = {page_table ? page_table + b * page_table_stride : nullptr, page_table_stride, max_pages,
                   start ? start + b : nullptr, lens ? lens + b : nullptr, n, len, t};
            p.k = static_cast<const char*>(k) + (b * k_batch_stride + t * k_token_stride) * elem;
            p.v = static_cast<const char*>(v) + (b * v_batch_stride + t * v_token_stride) * elem;
            p.tiles = (len + p.tile - 1) / p.tile;
            // (a launch has at most kEntries pages of at most 256 tokens)
            DT_TRY(launch_pdl(t > 0 ? later : from_first, dim3((unsigned)(p.tiles * n)), dim3(dt::kv::kThreads), 0, st, p));
        }
    return DT_OK;
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
    p.s = {page_table, page_table_stride, max_pages, start, lens, B, T, 0};
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


// How the prefix's part is cut: one CTA per SM, each with a block of query rows of a K/V head and an
// even stretch of the prefix.  Two Q tiles per CTA, so that keys are converted once for 256 rows,
// where there are more than 128 rows; fp32 queries take both tiles' memory for their two parts.
struct PrefixPlan {
    int rows, blocks, pairs, tiles, split;
};
PrefixPlan plan_prefix(int B, int T, int heads, int kv_heads, int q_f32, int prefix_len) {
    PrefixPlan s{};
    s.rows = B * T * (heads / kv_heads);
    s.pairs = q_f32 || s.rows <= 128;
    s.blocks = (s.rows - 1) / (s.pairs ? 128 : 256) + 1;
    s.tiles = (int)(((long long)prefix_len + 127) / 128);
    const long long groups = (long long)kv_heads * s.blocks;
    s.split = (int)std::max<long long>(1, std::min<long long>(s.tiles, kPlanSms / groups));
    return s;
}
// How the attention's work is cut.
struct AttnPlan {
    int form;         // query rows per item: rows_of(form)
    long long items;  // (sequence, K/V head, rows)
    int split;        // CTAs per item (split_kernel), or
    bool by_length;   // longest sequences first (split_kernel)
    int shares;       // CTAs that stream_kernel shares out, and one per item at least; join_kernel follows (0: split_kernel)
};

// split_kernel, with as many CTAs per item as the GPU holds at once, up to a cluster, and no more
// than there are tiles for; stream_kernel where that leaves most of the GPU idle: few items with
// many keys.  (8 x 131071 keys: 149 us in 8 clusters of 8, 70 shared out over 592 CTAs.  The rule knows the items and the
// table's width, not the lengths: of 128 items, 8 of 131071 keys and 120 of 200, split_kernel's even split takes 398 us.)
// Behind a prefix, split_kernel also joins its rows with the prefix's n_shared parts, if these are few.
AttnPlan plan_attn(int B, int T, int heads, int kv_heads, int q_f32, int page_size, int max_pages, int n_shared) {
    namespace ca = dt::cache_attn;
    AttnPlan s{};
    const int rows = T * (heads / kv_heads);
    s.form = rows <= 4 ? ca::kFew : q_f32 || rows <= 8 ? ca::kEight : ca::kWide;
    s.items = (long long)B * kv_heads * ((rows + ca::rows_of(s.form) - 1) / ca::rows_of(s.form));
    const long long tiles = ((long long)max_pages * page_size + ca::kTile - 1) / ca::kTile;
    const int slots = ca::ctas_per_sm(q_f32, s.form) * kPlanSms;
    const bool fits = B <= ca::kMaxBatch && tiles * B < 0x7fffffffll && s.items < 0x7fffffffll - slots;
    const bool few = s.items * ca::kMaxCluster * 2 < slots && tiles > 4ll * ca::kMaxCluster * ca::kWarps;
    if (max_pages == 0) return s;  // no keys of their own: join_kernel alone
    if (n_shared > 16 || (fits && few)) {
        s.shares = fits ? (int)std::min<long long>(slots, (s.items * tiles + ca::kWarps - 1) / ca::kWarps) : -1;
        return s;
    }
    s.split = 1;
    while (s.split < ca::kMaxCluster && s.items * (s.split + 1) <= slots && tiles > (long long)s.split * ca::kWarps) ++s.split;
    s.by_length = s.items > slots && B <= 256 && tiles >= 64;  // (ranking the lengths takes a microsecond)
    return s;
}

constexpr size_t kPrefixSmem = sizeof(dt::prefix_attn::Smem) + 1024;

// Workspace of a plan: the tile counts, the CTAs' parts, the prefix's parts.
struct AttnSpace {
    size_t starts, part_s, part_o, shared_s, shared_o, total;
};
AttnSpace attn_space(const AttnPlan& plan, int B, int T, int heads, int n_shared) {
    AttnSpace w{};
    const size_t parts = plan.shares > 0 ? ((size_t)plan.shares + plan.items) * dt::cache_attn::rows_of(plan.form) : 0;
    const size_t shared = (size_t)n_shared * B * T * heads;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += align256(bytes);
        return here;
    };
    w.starts = take(plan.shares > 0 ? ((size_t)B + 1) * 4 : 0);
    w.part_s = take(parts * 16);
    w.part_o = take(parts * dt::cache_attn::kD * 4);
    w.shared_s = take(shared * 16);
    w.shared_o = take(shared * dt::cache_attn::kD * 4);
    w.total = at;
    return w;
}

int launch_split(void (*kernel)(dt::cache_attn::Params), const dt::cache_attn::Params& p, long long items,
                 cudaStream_t st) {
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = DT_PDL;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)p.split;
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

typedef void (*AttnKernel)(dt::cache_attn::Params);
template <int kFmt, bool kF32, int kForm>
AttnKernel attn_kernel_of(bool stream) {
    return stream ? dt::cache_attn::stream_kernel<kFmt, kF32, kForm> : dt::cache_attn::split_kernel<kFmt, kF32, kForm>;
}
template <int kFmt>
AttnKernel attn_kernel_of(bool stream, bool f32, int form) {
    namespace ca = dt::cache_attn;
    if (f32) return form == ca::kFew ? attn_kernel_of<kFmt, true, ca::kFew>(stream) : attn_kernel_of<kFmt, true, ca::kEight>(stream);
    return form == ca::kFew     ? attn_kernel_of<kFmt, false, ca::kFew>(stream)
           : form == ca::kEight ? attn_kernel_of<kFmt, false, ca::kEight>(stream)
                                : attn_kernel_of<kFmt, false, ca::kWide>(stream);
}
AttnKernel attn_kernel_of(bool stream, int format, bool f32, int form) {
    return format == DT_KV_INT8 ? attn_kernel_of<0>(stream, f32, form) : attn_kernel_of<1>(stream, f32, form);
}

int launch_stream(const dt::cache_attn::Params& p, const AttnPlan& plan, int format, int q_f32, cudaStream_t st) {
    namespace ca = dt::cache_attn;
    if (plan.shares > 0)
        DT_TRY(launch_pdl(attn_kernel_of(true, format, q_f32, plan.form),
                          dim3((unsigned)(plan.shares + plan.items)), dim3(ca::kThreads), sizeof(ca::Smem), st, p));
    // (an item's CTAs are its share of all keys: of as many equal ones, about this many)
    const long long parts = (plan.items > 0 ? plan.shares / plan.items : 0) + p.n_shared;
    const int warps = (int)std::min<long long>(ca::kJoinWarps, std::max<long long>(1, (parts + 7) / 8));
    const dim3 grid((unsigned)((long long)p.B * p.T * p.heads)), block((unsigned)warps * 32);
    AttnKernel join = ca::join_kernel<false, ca::kWide>;
    if (plan.form == ca::kFew) join = q_f32 ? ca::join_kernel<true, ca::kFew> : ca::join_kernel<false, ca::kFew>;
    if (plan.form == ca::kEight) join = q_f32 ? ca::join_kernel<true, ca::kEight> : ca::join_kernel<false, ca::kEight>;
    return launch_pdl(join, grid, block, 0, st, p);
}

int launch_prefix(const dt::cache_attn::Params& p, const PrefixPlan& plan, int format, int q_f32, cudaStream_t st) {
    namespace pa = dt::prefix_attn;
    pa::Params pp{};
    pp.a = p;
    pp.rows = plan.rows;
    pp.blocks = plan.blocks;
    pp.pairs = plan.pairs;
    pp.split = plan.split;
    pp.tiles = plan.tiles;
    const long long ctas = (long long)p.c.heads * plan.blocks * plan.split;
    if (ctas > 0x7fffffffll) return fail(DT_ERR_INVALID_ARGUMENT, "B * T * heads is too large");
    auto* k = format == DT_KV_INT8 ? (q_f32 ? pa::prefix_kernel<0, true> : pa::prefix_kernel<0, false>)
                                   : (q_f32 ? pa::prefix_kernel<1, true> : pa::prefix_kernel<1, false>);
    return launch_pdl(k, dim3((unsigned)ctas), dim3(pa::kThreads), kPrefixSmem, st, pp);
}

// Per-device attributes of the kernels below (called with g_mu held, from ensure_attrs).
int serving_attrs() {
    for (int i = 0; i < 24; ++i)
        DT_CUDA(cudaFuncSetAttribute(attn_kernel_of(i & 1, (i >> 1) & 1, (i >> 2) & 1, i / 8),
                                     cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(dt::cache_attn::Smem)));
    for (auto* k : {dt::logprobs::row_kernel<false>, dt::logprobs::row_kernel<true>})
        DT_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    for (auto* k : {dt::prefix_attn::prefix_kernel<0, false>, dt::prefix_attn::prefix_kernel<0, true>,
                    dt::prefix_attn::prefix_kernel<1, false>, dt::prefix_attn::prefix_kernel<1, true>})
        DT_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kPrefixSmem));
    return DT_OK;
}

// Whether the dense output at o may be written while queries are read: it is q's own dense memory (whoever writes a row
// has read it), or no row of q lies in it.
bool output_apart(const void* q, long long batch, long long token, const void* o, int B, int T, int heads, int elem) {
    typedef unsigned __int128 Wide;
    const Wide x = reinterpret_cast<uintptr_t>(q), y = reinterpret_cast<uintptr_t>(o);
    const Wide row = (Wide)heads * dt::cache_attn::kD * elem, end = y + row * T * B;
    if (x == y && (T == 1 || (Wide)token * elem == row) && (B == 1 || (Wide)batch * elem == row * T)) return true;
    if (x >= end || x + ((Wide)(B - 1) * batch + (Wide)(T - 1) * token) * elem + row <= y) return true;
    for (int b = 0; b < B; ++b) {  // the first row of sequence b that ends behind o's start
        const Wide first = x + (Wide)b * batch * elem, step = (Wide)token * elem;
        const Wide t = first + row > y ? 0 : step == 0 ? (Wide)T : (y - first - row) / step + 1;
        if (t < (Wide)T && first + t * step < end) return false;
    }
    return true;
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
    if (((long long)max_pages << p.c.page_shift) > (1ll << 30))
        return fail(DT_ERR_INVALID_ARGUMENT, "max_pages * page_size must be at most 2^30");
    if (!seq_lens && max_pages > 0) return fail(DT_ERR_INVALID_ARGUMENT, "null seq_lens");
    DT_TRY(check_strides("q", q, q_batch_stride, q_token_stride, q_f32 ? 4 : 2));
    if (!o || !aligned16(o)) return fail(DT_ERR_INVALID_ARGUMENT, "o must be non-null and 16-byte aligned");
    if (prefix_len < 0 || (prefix_len > 0 && !prefix_pages))
        return fail(DT_ERR_INVALID_ARGUMENT, "prefix_len must be >= 0, with its pages");
    // (positions are 32-bit, and the kernel looks up pages a few tiles past the end)
    if (prefix_len > (1 << 30)) return fail(DT_ERR_INVALID_ARGUMENT, "prefix_len must be at most 2^30");
    if ((long long)B * T * heads > 0x7fffffffll) return fail(DT_ERR_INVALID_ARGUMENT, "B * T * heads must be below 2^31");
    if (!output_apart(q, q_batch_stride, q_token_stride, o, B, T, heads, q_f32 ? 4 : 2))
        return fail(DT_ERR_INVALID_ARGUMENT, "o may be q's own dense memory, and must not overlap it otherwise");
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
    const PrefixPlan prefix = prefix_len > 0 ? plan_prefix(B, T, heads, cache->kv_heads, q_f32, prefix_len) : PrefixPlan{};
    const AttnPlan plan = plan_attn(B, T, heads, cache->kv_heads, q_f32, cache->page_size, max_pages, prefix.split);
    // (so many parts of a prefix go with at most 8 blocks of 256 query rows, well below kMaxBatch sequences: what is left
    // is the batch's count of tiles)
    if (plan.shares < 0)
        return fail(DT_ERR_INVALID_ARGUMENT, "behind a prefix in more than 16 parts, B * max_pages * page_size must be below 2^36");
    if (plan.items * std::max(plan.split, 1) > 0x7fffffffll)
        return fail(DT_ERR_INVALID_ARGUMENT, "B * kv_heads * query rows is too large");
    const AttnSpace space = attn_space(plan, B, T, heads, prefix.split);
    if (space.total > 0 && (!workspace || workspace_bytes < space.total || !aligned16(workspace)))
        return fail(DT_ERR_INVALID_ARGUMENT, "workspace must be >= %zu bytes and 16-byte aligned", space.total);
    int dev;
    DT_TRY(prepare_device(&dev));
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    p.split = plan.split;
    p.by_length = plan.by_length;
    p.shares = plan.shares;
    p.n_shared = prefix.split;
    uint8_t* w = static_cast<uint8_t*>(workspace);
    p.starts = reinterpret_cast<int*>(w + space.starts);
    p.part_s = reinterpret_cast<float4*>(w + space.part_s);
    p.part_o = reinterpret_cast<float*>(w + space.part_o);
    p.shared_s = reinterpret_cast<float4*>(w + space.shared_s);
    p.shared_o = reinterpret_cast<float*>(w + space.shared_o);
    if (prefix_len > 0) DT_TRY(launch_prefix(p, prefix, cache->format, q_f32, st));
    if (plan.split > 0) return launch_split(attn_kernel_of(false, cache->format, q_f32, plan.form), p, plan.items, st);
    return launch_stream(p, plan, cache->format, q_f32, st);
}

// Whether N rows of V elements at b may be written while those at a are read, each thread reading what it
// writes before it does: the rows are the same, or none of one lies in one of the other.
bool writes_apart(const void* a, long long lda, const void* b, long long ldb, int N, int V, int elem) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    if (x == y) return lda == ldb || N == 1;
    const auto end = [&](uintptr_t at, long long ld) { return (unsigned __int128)at + ((unsigned __int128)(N - 1) * ld + V) * elem; };
    if (y >= end(x, lda) || x >= end(y, ldb)) return true;
    // rows between each other's: at an even distance, so that the first two show it
    const unsigned long long step = (unsigned long long)lda * elem, off = (x < y ? y - x : x - y) % step;
    const unsigned long long row = (unsigned long long)V * elem;
    return lda == ldb && off >= row && off <= step - row;
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
    return attn_space(plan_attn(B, T, heads, kv_heads, q_f32, page_size, max_pages, 0), B, T, heads, 0).total;
}

size_t dt_prefix_attn_workspace_bytes(int B, int T, int heads, int kv_heads, int q_f32, int page_size, int max_pages,
                                      int prefix_len) {
    if (prefix_len <= 0) return dt_cache_attn_workspace_bytes(B, T, heads, kv_heads, q_f32, page_size, max_pages);
    if (B <= 0 || T <= 0 || kv_heads <= 0 || heads < kv_heads || page_size <= 0 || max_pages < 0) return 0;
    if ((long long)B * T * heads > 0x7fffffffll) return 0;
    const int n_shared = plan_prefix(B, T, heads, kv_heads, q_f32, prefix_len).split;
    return attn_space(plan_attn(B, T, heads, kv_heads, q_f32, page_size, max_pages, n_shared), B, T, heads, n_shared).total;
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
    if (N < 0 || V < 1 || V > (1 << 30)) return fail(DT_ERR_INVALID_ARGUMENT, "N must be >= 0 and V 1..2^30");
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
                           top_log_probs, 1};
    // A cluster per row while all its CTAs fit on the GPU and every thread has a batch of its own.  (Four rows of
    // 100352: 9.5 us in clusters of 8, 8.6 in clusters of 16.)
    const int slots = dt::logprobs::ctas_per_sm(logits_f32) * kPlanSms;
    while (p.split < dt::logprobs::kMaxCluster && (long long)N * p.split * 2 <= slots &&
           V >= p.split * 2 * dt::logprobs::kThreads * 16)
        p.split *= 2;
    if ((long long)N * p.split > 0x7fffffffll) return fail(DT_ERR_INVALID_ARGUMENT, "N is too large");
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = DT_PDL;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)p.split;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(N * p.split));
    cfg.blockDim = dim3(dt::logprobs::kThreads);
    cfg.stream = reinterpret_cast<cudaStream_t>(stream);
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    DT_CUDA(cudaLaunchKernelEx(&cfg, logits_f32 ? dt::logprobs::row_kernel<true> : dt::logprobs::row_kernel<false>, p));
    return DT_OK;
}

int dt_token_log_probs_bwd(const void* logits, int logits_f32, long long ld, int N, int V, const void* targets,
                           int targets_int64, const float* lse, const float* entropy, const float* d_log_prob,
                           const float* d_entropy, void* d_logits, long long d_ld, void* stream) {
    t_last_error.clear();
    if (N < 0 || V < 1 || V > (1 << 30)) return fail(DT_ERR_INVALID_ARGUMENT, "N must be >= 0 and V 1..2^30");
    if (N == 0) return DT_OK;
    if (!logits || !d_logits || ld < V || d_ld < V)
        return fail(DT_ERR_INVALID_ARGUMENT, "logits and d_logits must be non-null with ld >= V");
    const uintptr_t mask = logits_f32 ? 3 : 1;
    if ((reinterpret_cast<uintptr_t>(logits) & mask) || (reinterpret_cast<uintptr_t>(d_logits) & mask))
        return fail(DT_ERR_INVALID_ARGUMENT, "logits and d_logits must be aligned to their type");
    if (!lse) return fail(DT_ERR_INVALID_ARGUMENT, "null lse");
    if (d_log_prob && !targets) return fail(DT_ERR_INVALID_ARGUMENT, "d_log_prob needs targets");
    if (d_entropy && !entropy) return fail(DT_ERR_INVALID_ARGUMENT, "d_entropy needs entropy");
    if (!writes_apart(logits, ld, d_logits, d_ld, N, V, logits_f32 ? 4 : 2))
        return fail(DT_ERR_INVALID_ARGUMENT, "d_logits may be the logits' own rows, and must not overlap them otherwise");
    namespace lp = dt::logprobs;
    dt::logprobs::GradParams p{logits, ld, N, V, targets, targets_int64 ? 1 : 0, lse, entropy, d_log_prob, d_entropy,
                               d_logits, d_ld, 1};
    const int elem = logits_f32 ? 4 : 2;
    // (one vector more than V has: a row may start inside one)
    const long long vectors = ((long long)V * elem + 15) / 16 + 1;
    p.chunks = (int)((vectors + lp::kGradThreads * lp::kGradVectors - 1) / (lp::kGradThreads * lp::kGradVectors));
    if ((long long)N * p.chunks > 0x7fffffffll) return fail(DT_ERR_INVALID_ARGUMENT, "N * V is too large");
    int dev;
    DT_TRY(prepare_device(&dev));
    const bool aligned = ((reinterpret_cast<uintptr_t>(logits) ^ reinterpret_cast<uintptr_t>(d_logits)) & 15) == 0 &&
                         ((ld - d_ld) * elem) % 16 == 0;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const dim3 grid((unsigned)(N * p.chunks)), block(lp::kGradThreads);
    if (logits_f32) return launch_pdl(aligned ? lp::grad_kernel<true, true> : lp::grad_kernel<true, false>, grid, block, 0, st, p);
    return launch_pdl(aligned ? lp::grad_kernel<false, true> : lp::grad_kernel<false, false>, grid, block, 0, st, p);
}

}  // extern "C"
