/* lg_cattn.hip -- attention of many rows over contiguous caches that callers keep:
 * plan, launch and entry points (the kernels: lg_cattn.h). */
#include "lg_cattn.h"

CaPlan lg_ca_plan(int64_t nseq, int64_t ntok, int n_heads, int n_kv, int hd, int window, int sinks, int max_pos,
                  bool kv4)
{
    CaPlan p = {};
    const int64_t cols = ntok * (n_heads / n_kv);
    p.dec = cols <= 16;
    p.nsplit = 1;
    int64_t keys = (int64_t)max_pos + 1;
    if (window > 0) keys = std::min(keys, (int64_t)window + sinks + ntok - 1);
    if (!p.dec) {
        /* Blocks of columns by workgroups of eight waves or, at 128 dims and less,
         * of four where those fit the 256 CUs at once, and parts of the keys.
         * The unit of time is a tile of an eight-wave workgroup (2.9 us at 128
         * dims); a tile of four waves alone on their CU takes 0.95 of it, a
         * start and end 4.5 and 2.6; joined parts are a second launch and are
         * written and read once, about 19 MB in a unit.  Without a window the
         * last columns see all keys, the mean half a prompt less.  32 heads of
         * 128 over 8 key heads, us in (waves, parts) as chosen and others: 100
         * tokens of 100 keys (4, 1) 14.3, (8, 1) 15.7; 1000 keys (4, 8) 27.9,
         * (4, 1) 51, (8, 4) 33; 6000 keys (8, 16) 40, (8, 8) 56, (4, 8) 49; 700
         * of 700 (4, 1) 38, (8, 1) 45; of 9000 (8, 5) 198, (8, 2) 226, (8, 3)
         * 284, (8, 1) 419; 2000 of 2000 (8, 2) 92, (8, 1) 105. */
        const int kt = hd <= 128 ? 64 : 32;
        double best = 0.0;
        for (int nw = hd <= 128 ? 8 : 4; nw >= 4; nw /= 2) {
            const bool small = hd <= 128 && nw == 4;
            const int64_t width = 32 * nw, ncb = (cols + width - 1) / width, wgs = nseq * n_kv * ncb;
            if (small && cols <= 128) break;   /* (no more workgroups than of eight) */
            int64_t seen = (int64_t)max_pos + 1, mean = std::max<int64_t>(1, seen - ntok / 2);
            if (window > 0) seen = mean = std::min(seen, (int64_t)window + sinks + width * n_kv / n_heads);
            const double last = (double)((seen + kt - 1) / kt), tiles = (double)(mean + kt - 1) / kt;
            const double each = small ? 0.95 : 1.0, ends = small ? 2.6 : 4.5;
            for (int ns = 1; ns <= 64 && (ns == 1 || last / ns >= 1.5); ns++) {
                if (small && wgs * ns > 256) break;
                double cost = std::max(last / ns * each + ends,
                                       (double)((wgs * ns + 255) / 256) * (tiles / ns * each + ends));
                if (ns > 1) cost += 2.0 + 6e-6 / 14.0 * ns * (double)(nseq * ntok) * n_heads * hd;
                if (!p.ncb || cost < best) {
                    best = cost;
                    p.ncb = (int)ncb;
                    p.nsplit = ns;
                    p.wide = nw == 8;
                }
            }
        }
    } else {
        /* Short contexts: eight waves and no second launch.  32 heads of 128, 8
         * key heads, us of the GPU, one launch / parts and their join (which
         * cost an eager caller 4 more): fp16 256 keys 8.0 / 8.5, 512 11.3 / 8.6,
         * 768 14.7 / 8.9, but of 32 sequences 512 15 / 19, 1024 25 / 29; 4 bits
         * 512 8.4 / 9.4, 768 9.5 / 9.7, 1024 11.7 / 9.6, of 32 sequences 13.5
         * / 17 (both 0.3 to 0.9 less since the first loads go ahead).
         * Else two workgroups a CU, of 64 keys at least in fp16 (512 keys
         * 8.6 us, with 128 9.5, with 256 11.0) and 256 in 4 bits (6000 keys
         * 11.0 us, with 64 12.2); and chunks short enough to even out ragged
         * lengths: 24 sequences of up to 12000 fp16 rows 133 us with 1024 keys,
         * 148 with 2048, 186 with half a length; 40 of up to 8208 rows in 4
         * bits 148 with 512, 117 with 1024, 106 with 2048, 121 with 4096. */
        const int64_t groups = nseq * n_kv;
        const int kt = kv4 && hd <= 128 ? 64 : 32, least = kv4 ? 256 : 64;   /* (CaDec::KT) */
        p.wide = hd <= 128 && groups <= 256 && keys <= (groups >= 128 ? 1024 : kv4 ? 768 : 512);
        if (!p.wide) {
            p.nsplit = (int)std::max<int64_t>({1, std::min<int64_t>(512 / groups, (keys + least - 1) / least),
                                               std::min<int64_t>({keys / (kv4 ? 2048 : 1024), 16384 / groups, CA_PARTS})});
            p.chunk = (int)((keys + (int64_t)kt * p.nsplit - 1) / ((int64_t)kt * p.nsplit));
        }
    }
    if (p.nsplit > 1) p.ws = (size_t)p.nsplit * nseq * ntok * n_heads * (hd + 2) * sizeof(float);
    return p;
}

extern "C" size_t lg_attn_cache_workspace_size(const lg_kv_cache* cache, int nseq, int ntok, int n_heads, int window,
                                               int sinks, int max_pos)
{
    if (!cache || cache->n_kv_heads <= 0 || cache->head_dim <= 0 || nseq <= 0 || ntok <= 0 || n_heads <= 0 || window < 0 ||
        sinks < 0 || max_pos < 0)
        return 0;
    return lg_ca_plan(nseq, ntok, n_heads, cache->n_kv_heads, cache->head_dim, window, sinks, max_pos,
                   cache->type == LG_KV4).ws;
}

template <int HD, bool KV4>
static void ca_launch(const CAttn& a, const CaPlan& p, int nseq, float* part, hipStream_t s)
{
    const int64_t n = (int64_t)nseq * a.c.n_kv * p.nsplit;
    if constexpr (HD <= 128)
        if (p.wide) {
            if (p.dec) k_cattn_dec<HD, KV4, 8, CAttn><<<(unsigned)n, 512, 0, s>>>(a, p.nsplit, p.chunk, part);
            else k_cattn_tile<HD, KV4, 8, CAttn><<<(unsigned)(n * p.ncb), 512, 0, s>>>(a, p.ncb, p.nsplit, part);
            return;
        }
    if (p.dec)
        k_cattn_dec<HD, KV4, 4, CAttn><<<(unsigned)n, 256, 0, s>>>(a, p.nsplit, p.chunk, part);
    else
        k_cattn_tile<HD, KV4, 4, CAttn><<<(unsigned)(n * p.ncb), 256, 0, s>>>(a, p.ncb, p.nsplit, part);
}

template <int HD>
static void ca_type(const CAttn& a, const CaPlan& p, int nseq, float* part, hipStream_t s)
{
    if constexpr (HD != 48)
        if (a.c.type == LG_KV4) return ca_launch<HD, true>(a, p, nseq, part, s);
    ca_launch<HD, false>(a, p, nseq, part, s);
}

extern "C" int lg_attn_cache(const float* q, int64_t q_stride, const lg_kv_cache* cache, const int* pos, int nseq,
                             int ntok, int n_heads, int window, int sinks, int max_pos, float* out, int64_t out_stride,
                             void* workspace, size_t workspace_bytes, void* stream)
{
    const char* who = "lg_attn_cache";
    if (!cache || nseq < 0 || ntok < 0 || window < 0 || sinks < 0) {
        lg_set_error("%s: bad argument (%d sequences of %d tokens, window %d, sinks %d)", who, nseq, ntok, window, sinks);
        return LG_ERR_ARG;
    }
    CAttn a = {q, out, pos, q_stride, out_stride, 0, ntok, n_heads, 0, window, sinks, max_pos, 0.0f, {}};
    const int rc = lg_kv_arg(cache, nseq, who, &a.c);
    if (rc) return rc;
    const int hd = a.c.hd;
    if (!(hd == 64 || hd == 96 || hd == 128 || hd == 256 || (hd == 48 && a.c.type == LG_F16))) {
        lg_set_error("%s: head_dim %d unsupported (48 in fp16, 64, 96, 128, 256)", who, hd);
        return LG_ERR_ARG;
    }
    if (n_heads <= 0 || n_heads > 65536 || n_heads % a.c.n_kv) {
        lg_set_error("%s: %d query heads over %d key heads", who, n_heads, a.c.n_kv);
        return LG_ERR_ARG;
    }
    if (max_pos < 0 || max_pos >= a.c.n_ctx) {
        lg_set_error("%s: positions up to %d in a cache of %d rows", who, max_pos, a.c.n_ctx);
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
    a.rows = (int)rows;
    a.nrep = n_heads / a.c.n_kv;
    a.scale2 = 1.44269504088896341f / sqrtf((float)hd);
    const CaPlan p = lg_ca_plan(nseq, ntok, n_heads, a.c.n_kv, hd, window, sinks, max_pos, a.c.type == LG_KV4);
    /* workgroups of the kernel and, of a split call, of its join */
    const int64_t blocks = (int64_t)nseq * a.c.n_kv * p.nsplit * (p.dec ? 1 : p.ncb);
    const bool by_group = p.nsplit > 8 || rows * n_heads <= 4096;   /* 8 parts of 32 heads: 4.0 us against 8.5 */
    const int64_t joins = p.ws ? by_group ? rows * n_heads : (rows * n_heads * (hd / 4) + 255) / 256 : 0;
    if (!lg_grid_fits(blocks, p.wide ? 512 : 256) || !lg_grid_fits(joins, 256)) {
        lg_set_error("%s: %lld rows of %d heads are too many for one call", who, (long long)rows, n_heads);
        return LG_ERR_ARG;
    }
    if (p.ws && (!workspace || !lg_al16(workspace) || workspace_bytes < p.ws)) {
        lg_set_error("%s: workspace of %zu bytes, 16-byte aligned, %zu needed", who, workspace_bytes, p.ws);
        return LG_ERR_ARG;
    }
    hipStream_t s = (hipStream_t)stream;
    float* const part = p.ws ? (float*)workspace : nullptr;
    switch (hd) {
    case 48: ca_type<48>(a, p, nseq, part, s); break;
    case 64: ca_type<64>(a, p, nseq, part, s); break;
    case 96: ca_type<96>(a, p, nseq, part, s); break;
    case 128: ca_type<128>(a, p, nseq, part, s); break;
    default: ca_type<256>(a, p, nseq, part, s); break;
    }
    if (part) {
        if (by_group) k_cattn_merge_wide<CAttn><<<(unsigned)joins, 256, 0, s>>>(a, p.nsplit, part);
        else k_cattn_merge<CAttn><<<(unsigned)joins, 256, 0, s>>>(a, p.nsplit, part);
    }
    return lg_check_launch(who);
}
