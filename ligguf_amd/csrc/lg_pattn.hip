/* lg_pattn.hip -- attention over caches in pages, the rows that a group of
 * sequences shares once for the whole group (the kernels: lg_cattn.h). */
#include "lg_cattn.h"

/* How a call is cut: the shared rows as a sequence of all the group's rows, the
 * others sequence by sequence, each as a call over contiguous caches would be;
 * their parts one behind the other. */
struct PaPlan {
    bool shared;
    CaPlan a, b;   /* shared rows, own rows */
    int parts;     /* 1: written out as they are */
    size_t ws;
};

static PaPlan pa_plan(int64_t nseq, int64_t ntok, int n_heads, int n_kv, int hd, int window, int sinks, int max_pos, bool kv4,
                      int group, int max_prefix)
{
    PaPlan p = {};
    p.shared = group > 1 && max_prefix > 0;
    if (p.shared) p.a = lg_ca_plan(nseq / group, ntok * group, n_heads, n_kv, hd, window, sinks, std::min(max_prefix - 1, max_pos), kv4);
    /* (the own rows' number lies in device memory: of the longest prompt's) */
    p.b = lg_ca_plan(nseq, ntok, n_heads, n_kv, hd, window, sinks, p.shared ? std::max(max_pos - max_prefix, 0) : max_pos, kv4);
    p.parts = p.b.nsplit + (p.shared ? p.a.nsplit : 0);
    if (p.parts > 1) p.ws = (size_t)p.parts * nseq * ntok * n_heads * (hd + 2) * sizeof(float);
    return p;
}

template <int HD, bool KV4>
static void pa_launch(const CAttnPaged& a, const CaPlan& p, int units, float* part, hipStream_t s)
{
    const int64_t n = (int64_t)units * a.c.n_kv * p.nsplit;
    if constexpr (HD <= 128)
        if (p.wide) {
            if (p.dec) k_cattn_dec<HD, KV4, 8, CAttnPaged><<<(unsigned)n, 512, 0, s>>>(a, p.nsplit, p.chunk, part);
            else k_cattn_tile<HD, KV4, 8, CAttnPaged><<<(unsigned)(n * p.ncb), 512, 0, s>>>(a, p.ncb, p.nsplit, part);
            return;
        }
    if (p.dec) k_cattn_dec<HD, KV4, 4, CAttnPaged><<<(unsigned)n, 256, 0, s>>>(a, p.nsplit, p.chunk, part);
    else k_cattn_tile<HD, KV4, 4, CAttnPaged><<<(unsigned)(n * p.ncb), 256, 0, s>>>(a, p.ncb, p.nsplit, part);
}

template <int HD>
static void pa_type(const CAttnPaged& a, const CaPlan& p, int units, float* part, hipStream_t s)
{
    if constexpr (HD != 48)
        if (a.c.type == LG_KV4) return pa_launch<HD, true>(a, p, units, part, s);
    pa_launch<HD, false>(a, p, units, part, s);
}

static void pa_phase(const CAttnPaged& a, const CaPlan& p, int units, float* part, hipStream_t s)
{
    switch (a.c.hd) {
    case 48: pa_type<48>(a, p, units, part, s); break;
    case 64: pa_type<64>(a, p, units, part, s); break;
    case 96: pa_type<96>(a, p, units, part, s); break;
    case 128: pa_type<128>(a, p, units, part, s); break;
    default: pa_type<256>(a, p, units, part, s); break;
    }
}

static bool pa_head_dim(int hd, int type)
{
    return hd == 64 || hd == 96 || hd == 128 || hd == 256 || (hd == 48 && type == LG_F16);
}

extern "C" size_t lg_attn_paged_workspace_size(const lg_kv_pages* cache, int nseq, int ntok, int n_heads, int window, int sinks,
                                               int max_pos, int group, int max_prefix)
{
    if (!cache || cache->pool.n_kv_heads <= 0 || cache->pool.head_dim <= 0 || nseq <= 0 || ntok <= 0 || n_heads <= 0 ||
        window < 0 || sinks < 0 || max_pos < 0 || group <= 0 || nseq % group || max_prefix < 0)
        return 0;
    return pa_plan(nseq, ntok, n_heads, cache->pool.n_kv_heads, cache->pool.head_dim, window, sinks, max_pos,
                   cache->pool.type == LG_KV4, group, max_prefix).ws;
}

extern "C" int lg_attn_paged(const float* q, int64_t q_stride, const lg_kv_pages* cache, const int* pos, int nseq, int ntok,
                             int n_heads, int window, int sinks, int max_pos, const int* prefix, int group, int max_prefix,
                             float* out, int64_t out_stride, void* workspace, size_t workspace_bytes, void* stream)
{
    const char* who = "lg_attn_paged";
    if (!cache || nseq < 0 || ntok < 0 || window < 0 || sinks < 0) {
        lg_set_error("%s: bad argument (%d sequences of %d tokens, window %d, sinks %d)", who, nseq, ntok, window, sinks);
        return LG_ERR_ARG;
    }
    CAttnPaged a = {};
    const int rc = lg_kv_pages_arg(cache, who, &a.c, &a.shift);
    if (rc) return rc;
    const int hd = a.c.hd;
    if (!pa_head_dim(hd, a.c.type)) {
        lg_set_error("%s: head_dim %d unsupported (48 in fp16, 64, 96, 128, 256)", who, hd);
        return LG_ERR_ARG;
    }
    if (n_heads <= 0 || n_heads > 65536 || n_heads % a.c.n_kv) {
        lg_set_error("%s: %d query heads over %d key heads", who, n_heads, a.c.n_kv);
        return LG_ERR_ARG;
    }
    if (max_pos < 0 || max_pos >= cache->max_pages * a.c.n_ctx) {
        lg_set_error("%s: positions up to %d in %d pages of %d rows", who, max_pos, cache->max_pages, a.c.n_ctx);
        return LG_ERR_ARG;
    }
    if (max_prefix < 0 || group <= 0 || nseq % group || (max_prefix && !prefix)) {
        lg_set_error("%s: groups of %d of %d sequences, %d rows shared", who, group, nseq, max_prefix);
        return LG_ERR_ARG;
    }
    const int64_t rows = (int64_t)nseq * ntok, width = (int64_t)n_heads * hd;
    if (!rows) return LG_OK;
    if (!pos || !q || !out || !lg_al16(q) || !lg_al16(out) || q_stride % 4 || out_stride % 4 || q_stride < width ||
        out_stride < width) {
        lg_set_error("%s: rows must be given, 16-byte aligned and as wide as their heads", who);
        return LG_ERR_ARG;
    }
    if (rows > INT32_MAX / n_heads) {
        lg_set_error("%s: %lld rows of %d heads are too many for one call", who, (long long)rows, n_heads);
        return LG_ERR_ARG;
    }
    a.q = q;
    a.out = out;
    a.pos = pos;
    a.qs = q_stride;
    a.os = out_stride;
    a.rows = (int)rows;
    a.n_heads = n_heads;
    a.nrep = n_heads / a.c.n_kv;
    a.window = window;
    a.sinks = sinks;
    a.max_pos = max_pos;
    a.scale2 = 1.44269504088896341f / sqrtf((float)hd);
    a.table = cache->table;
    a.tstride = cache->table_stride;
    a.n_pages = cache->n_pages;
    a.group = group;
    const PaPlan p = pa_plan(nseq, ntok, n_heads, a.c.n_kv, hd, window, sinks, max_pos, a.c.type == LG_KV4, group, max_prefix);
    a.max_prefix = max_prefix;
    a.prefix = p.shared ? prefix : nullptr;
    a.nparts = p.parts;
    const int64_t na = p.shared ? (int64_t)(nseq / group) * a.c.n_kv * p.a.nsplit * (p.a.dec ? 1 : p.a.ncb) : 0;
    const int64_t nb = (int64_t)nseq * a.c.n_kv * p.b.nsplit * (p.b.dec ? 1 : p.b.ncb);
    const bool by_group = p.parts > 8 || rows * n_heads <= 4096;   /* (as lg_attn_cache) */
    const int64_t joins = p.ws ? by_group ? rows * n_heads : (rows * n_heads * (hd / 4) + 255) / 256 : 0;
    if (!lg_grid_fits(na, 512) || !lg_grid_fits(nb, 512) || !lg_grid_fits(joins, 256)) {
        lg_set_error("%s: %lld rows of %d heads are too many for one call", who, (long long)rows, n_heads);
        return LG_ERR_ARG;
    }
    if (p.ws && (!workspace || !lg_al16(workspace) || workspace_bytes < p.ws)) {
        lg_set_error("%s: workspace of %zu bytes, 16-byte aligned, %zu needed", who, workspace_bytes, p.ws);
        return LG_ERR_ARG;
    }
    hipStream_t s = (hipStream_t)stream;
    float* const part = p.ws ? (float*)workspace : nullptr;
    if (p.shared) {
        a.ntok = ntok * group;
        a.tstep = group;
        a.share = 1;
        pa_phase(a, p.a, nseq / group, part, s);
        a.part0 = p.a.nsplit;
    }
    a.ntok = ntok;
    a.tstep = 1;
    a.share = 0;
    pa_phase(a, p.b, nseq, part, s);
    if (part) {
        if (by_group) k_cattn_merge_wide<CAttnPaged><<<(unsigned)joins, 256, 0, s>>>(a, p.parts, part);
        else k_cattn_merge<CAttnPaged><<<(unsigned)joins, 256, 0, s>>>(a, p.parts, part);
    }
    return lg_check_launch(who);
}
