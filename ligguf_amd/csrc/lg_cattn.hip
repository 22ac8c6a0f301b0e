/* lg_cattn.hip -- attention of many rows over contiguous caches that callers keep:
 * prompts, plan, launch and entry points (single tokens and joins: lg_cattn.h). */
#include "lg_cattn.h"

/* Prompts: 32 columns (query heads of a key head, tokens in order) a wave, NW
 * waves a workgroup, which share tiles of KT keys in LDS; both products on
 * 32 x 32 x 16 fp16 MFMA with the operands of k_cattn_dec: lane l feeds row /
 * column l % 32, k = 8 (l / 32) .. +7, register i of a result is row 8 (i / 4)
 * + 4 (l / 32) + i % 4 of column l % 32, so registers 8s .. 8s+7 of the scores
 * are the lane's k of step s of the second product: keys 16s + 4h .. and
 * 16s + 8 + 4h .. of lane half h.  The next tile is on its way while one
 * computes (two LDS stages, one barrier a tile).  Bound by the MFMA and VALU
 * work of a SIMD's two waves, 51 % and 44 % of the cycles, at 2.04 of 2.4 GHz
 * (keeping the waves half a tile apart, products and softmax interleaved by
 * hand, or V's fragments read a step ahead was no faster): 2000 tokens over
 * windows of 4096 rows 260 us, 520 TFLOP/s of the products asked for, 1040 issued
 * with the parts, 0.88 of what torch's fp16 product reaches on this card.  One
 * wave a SIMD does a tile in 0.9 of the time of two: two to a SIMD wherever
 * there are columns enough. */
template <int HD, bool KV4, int NW_>
struct CaTile {
    static constexpr int NW = NW_, NTH = 64 * NW, KT = HD <= 128 ? 64 : 32, NK = KT / 32;
    static constexpr int NJ = HD / 16, NT = (HD + 31) / 32;
    static constexpr int KST = HD + 8;                       /* halves per K row in LDS */
    static constexpr int VST = NT * 32 + 32;                 /* and per V row: rows 64 bytes on */
    static constexpr int PW = KV4 ? 16 : 8;                  /* values of a piece that a thread moves */
    static constexpr int PR = HD / PW, NP = (KT * PR + NTH - 1) / NTH;   /* pieces of a row; of a tile per thread */
    static constexpr int STAGE = KT * (KST + VST);           /* halves */
};

template <int HD, bool KV4, int NW>
struct CaPieces {
    using C = CaTile<HD, KV4, NW>;
    v4u h[KV4 ? 1 : C::NP];
    uint2 w[KV4 ? C::NP : 1];
    uint32_t dm[KV4 ? C::NP : 1];

    /* (the tile's address is the wave's, a thread's part of it fits 32 bits) */
    __device__ __forceinline__ void load(const CAttn& a, const uint8_t* base, int g, int kb)
    {
        const uint8_t* const p = base + (KV4 ? lg_kv4_codes(a.c, g, kb) : lg_kv16_at(a.c, g, kb));
        const uint8_t* const q = base + (KV4 ? lg_kv4_dm(a.c, g, kb) : 0);
        const int last = a.max_pos - kb;   /* (rows past it are never visible) */
#pragma unroll
        for (int u = 0; u < C::NP; u++) {
            const int i = min((int)threadIdx.x + u * C::NTH, C::KT * C::PR - 1);
            const uint32_t key = min(i / C::PR, last), x = i % C::PR;
            if constexpr (KV4) {
                w[u] = *(const uint2*)(p + (key * (HD / 2) + 8 * x));
                dm[u] = *(const uint32_t*)(q + (key * (HD / 8) + x / 2 * 4));
            } else
                h[u] = *(const v4u*)(p + (key * (uint32_t)(a.c.n_kv * HD * 2) + 16 * x));
        }
    }
    /* into rows of ST halves; with `bad`, infinities and NaN as 0 and their keys noted */
    template <int ST>
    __device__ __forceinline__ void store(_Float16* dst, uint32_t* bad) const
    {
#pragma unroll
        for (int u = 0; u < C::NP; u++) {
            const int i = threadIdx.x + u * C::NTH;
            if ((C::KT * C::PR) % C::NTH == 0 || i < C::KT * C::PR) {
                _Float16* const q = dst + i / C::PR * ST + i % C::PR * C::PW;
                v4u x[C::PW / 8];
                if constexpr (KV4) {
                    lg_kv4_values(w[u].x, dm[u], (lg_h2*)&x[0]);
                    lg_kv4_values(w[u].y, dm[u], (lg_h2*)&x[1]);
                } else
                    x[0] = h[u];
                if (bad) {
                    bool any = false;
#pragma unroll
                    for (int e = 0; e < C::PW / 8; e++) any |= ca_drop_bad(x[e]);
                    if (any) atomicOr(bad + i / C::PR / 32, 1u << (i / C::PR % 32));
                }
#pragma unroll
                for (int e = 0; e < C::PW / 8; e++) *(v4u*)(q + 8 * e) = x[e];
            }
        }
    }
};

/* (256 registers a lane, or 512 where those would not do) */
template <int HD, bool KV4, int NW>
__global__ __launch_bounds__(64 * NW, (NW == 8 || HD < 128 || (HD == 128 && KV4) ? 2 : 1)) void k_cattn_tile(
    CAttn a, int ncb, int nsplit, float* __restrict__ part)
{
    using C = CaTile<HD, KV4, NW>;
    constexpr int KT = C::KT, NK = C::NK, NJ = C::NJ, NT = C::NT;
    __shared__ __attribute__((aligned(16))) _Float16 s_kv[2 * C::STAGE];
    __shared__ int s_pos[2 * C::NW];
    __shared__ uint32_t s_bad[3][2];
    /* key head fastest; the last columns, which may see most, first */
    const int n_kv = a.c.n_kv, g = blockIdx.x % n_kv;
    const int seq = blockIdx.x / n_kv % (a.rows / a.ntok), rest = blockIdx.x / n_kv / (a.rows / a.ntok);
    const int sp = rest % nsplit, cb = ncb - 1 - rest / nsplit;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 31, h = lane >> 5;
    const int ncol = a.ntok * a.nrep, idx = cb * 32 * C::NW + 32 * wave + col;
    const int tok = min(idx, ncol - 1) / a.nrep, head = g * a.nrep + idx % a.nrep;
    const int64_t row = (int64_t)seq * a.ntok + tok;
    int p = a.pos[row];
    if (idx >= ncol || p > a.max_pos) p = -1;
    int wmin = p < 0 ? INT32_MAX : p, wmax = p;   /* of the wave */
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        wmin = min(wmin, __shfl_xor(wmin, o));
        wmax = max(wmax, __shfl_xor(wmax, o));
    }
    if (lane == 0) {
        s_pos[2 * wave] = wmin;
        s_pos[2 * wave + 1] = wmax;
    }
    if (threadIdx.x < 6) s_bad[threadIdx.x / 2][threadIdx.x % 2] = 0;
    __syncthreads();
    wmin = __builtin_amdgcn_readfirstlane(wmin);
    wmax = __builtin_amdgcn_readfirstlane(wmax);
    int pmin = INT32_MAX, pmax = -1;              /* of the workgroup */
#pragma unroll
    for (int w = 0; w < C::NW; w++) {
        pmin = min(pmin, s_pos[2 * w]);
        pmax = max(pmax, s_pos[2 * w + 1]);
    }
    pmin = __builtin_amdgcn_readfirstlane(pmin);
    pmax = __builtin_amdgcn_readfirstlane(pmax);

    typedef float v16f __attribute__((ext_vector_type(16)));
    v16f o[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) o[t] = (v16f){};
    float l = 0.0f, unit = -INFINITY;
    if (pmax >= 0) {
        const CaTiles tiles(a, pmin, pmax, KT);
        int t0, t1;
        tiles.chunk(sp, nsplit, 0, &t0, &t1);
        const uint8_t* const kc = a.c.k + (size_t)seq * a.c.seq;
        const uint8_t* const vc = a.c.v + (size_t)seq * a.c.seq;
        /* tiles with keys that some row of the workgroup (wave) does not see */
        auto partly = [&](int kb, int lo, int hi) {
            return kb + KT - 1 > lo || (a.window > 0 && kb <= hi - a.window && kb + KT > a.sinks);
        };
        CaPieces<HD, KV4, NW> P, V;
        v8h qh[NJ], ql[NJ];
        CaMax mx(0.0f);
        {
            /* queries, first keys and first values on their way together */
            v4f x[2 * NJ];
            const float* const q = a.q + row * a.qs + (size_t)head * HD + 8 * h;
#pragma unroll
            for (int j = 0; j < 2 * NJ; j++)
                x[j] = idx < ncol ? *(const v4f*)(q + 16 * (j / 2) + 4 * (j % 2)) : (v4f){};
            const int k0 = tiles.at(t0) * KT;
            if (t0 < t1) {
                P.load(a, kc, g, k0);
                V.load(a, vc, g, k0);
            }
            float big = 0.0f;
#pragma unroll
            for (int j = 0; j < 2 * NJ; j++)
                big = fmaxf(fmaxf(big, fmaxf(fabsf(x[j][0]), fabsf(x[j][1]))), fmaxf(fabsf(x[j][2]), fabsf(x[j][3])));
            big = fmaxf(big, lg_partner<5>(big));
            const int ex = __builtin_amdgcn_frexp_expf(big);
            mx = CaMax(ca_scale(a.scale2, ex));
#pragma unroll
            for (int j = 0; j < NJ; j++)
#pragma unroll
                for (int e = 0; e < 8; e += 2)
                    ca_query2(x[2 * j + e / 4][e % 4], x[2 * j + e / 4][e % 4 + 1], ex, qh[j], ql[j], e);
            if (t0 < t1) {
                P.template store<C::KST>(s_kv, nullptr);
                V.template store<C::VST>(s_kv + KT * C::KST, partly(k0, pmin, pmax) ? s_bad[0] : nullptr);
            }
        }
        __syncthreads();
        for (int it = t0; it < t1; it++) {
            const bool more = it + 1 < t1;
            const int kb = tiles.at(it) * KT, kn = more ? tiles.at(it + 1) * KT : 0;
            const int cur = (it - t0) & 1, nxt = cur ^ 1, slot = (it - t0) % 3;
            _Float16* const sK = s_kv + cur * C::STAGE;
            _Float16* const sV = sK + KT * C::KST;
            _Float16* const nK = s_kv + nxt * C::STAGE;
            const bool on = kb <= wmax && (a.window <= 0 || kb + KT - 1 > wmin - a.window || kb < a.sinks);
            if (more) {
                P.load(a, kc, g, kn);
                V.load(a, vc, g, kn);
            }
            v16f s[NK];
            if (on) {
                /* its products ahead of the other wave's softmax: 700 x 9000 251 -> 243 us */
                __builtin_amdgcn_s_setprio(1);
#pragma unroll
                for (int n = 0; n < NK; n++) s[n] = (v16f){};
#pragma unroll
                for (int j = 0; j < NJ; j++)
#pragma unroll
                    for (int n = 0; n < NK; n++) {
                        const v8h k = *(const v8h*)(sK + (32 * n + col) * C::KST + 16 * j + 8 * h);
                        s[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, qh[j], s[n], 0, 0, 0);
                        s[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, ql[j], s[n], 0, 0, 0);
                    }
            }
            __builtin_amdgcn_s_setprio(0);
            if (more) P.template store<C::KST>(nK, nullptr);
            if (threadIdx.x < 2) s_bad[(slot + 2) % 3][threadIdx.x] = 0;
            if (on) {
                if (partly(kb, wmin, wmax)) {
#pragma unroll
                    for (int n = 0; n < NK; n++)
#pragma unroll
                        for (int i = 0; i < 16; i++)
                            if (!ca_sees(a, p, kb + 32 * n + 8 * (i >> 2) + 4 * h + (i & 3))) s[n][i] = -INFINITY;
                }
                float mn = s[0][0];
#pragma unroll
                for (int n = 0; n < NK; n++)
#pragma unroll
                    for (int i = 0; i < 16; i++) mn = fmaxf(mn, s[n][i]);
                if (mx.due(mn)) {
                    mn = fmaxf(mn, lg_partner<5>(mn));
                    float off;
                    const float al = mx.raise(mn, &off);
                    l *= al;
#pragma unroll
                    for (int t = 0; t < NT; t++) o[t] *= al;
#pragma unroll
                    for (int n = 0; n < NK; n++) s[n] -= off;
                }
#pragma unroll
                for (int st = 0; st < 2 * NK; st++) {
                    float w[8];
                    v8h ph, pl;
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        w[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[st / 2][8 * (st & 1) + i], mx.sc, mx.cc));
                    l += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
#pragma unroll
                    for (int i = 0; i < 8; i += 2) ca_split2(w[i], w[i + 1], ph, pl, i);
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        const _Float16* const v =
                            sV + (16 * st + 4 * h + (lane & 15) / 4) * C::VST + 32 * t + (lane & 16) + 4 * (lane & 3);
                        const v4s x0 = ca_tr16(v), x1 = ca_tr16(v + 8 * C::VST);
                        const v8h x = __builtin_bit_cast(v8h, __builtin_shufflevector(x0, x1, 0, 1, 2, 3, 4, 5, 6, 7));
                        o[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, ph, o[t], 0, 0, 0);
                        o[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, pl, o[t], 0, 0, 0);
                    }
                }
                /* infinities and NaN of keys that only some rows see: added by
                 * itself to those that do, whatever the (positive) weight */
#pragma unroll
                for (int n = 0; n < NK; n++)
                    for (uint32_t keys = __builtin_amdgcn_readfirstlane(s_bad[slot][n]); keys; keys &= keys - 1) {
                        const int key = kb + 32 * n + __builtin_ctz(keys);
                        if (ca_sees(a, p, key))
#pragma unroll
                            for (int t = 0; t < NT; t++)
#pragma unroll
                                for (int i = 0; i < 16; i += 4) {
                                    const int d = 32 * t + 2 * i + 4 * h;
                                    if (HD % 32 != 0 && d >= HD) continue;
                                    const v4f x = ca_values<KV4>(a.c, vc, g, key, d);
#pragma unroll
                                    for (int e = 0; e < 4; e++) o[t][i + e] = ca_add_bad(o[t][i + e], x[e]);
                                }
                    }
            }
            if (more) V.template store<C::VST>(nK + KT * C::KST, partly(kn, pmin, pmax) ? s_bad[(slot + 1) % 3] : nullptr);
            __syncthreads();
        }
        l += lg_partner<5>(l);
        unit = mx.unit(l);
    }
    if (idx >= ncol) return;
    const int64_t at = ((int64_t)sp * a.rows + row) * a.n_heads + head;
    float* const dst = part ? part + at * HD : a.out + row * a.os + (size_t)head * HD;
    const float f = part ? 1.0f : 1.0f / l;   /* (0: every visible key is -infinity) */
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const int d = 32 * t + 2 * i + 4 * h;
            const v4f y = {o[t][i], o[t][i + 1], o[t][i + 2], o[t][i + 3]};
            if (HD % 32 == 0 || d < HD) *(v4f*)(dst + d) = p < 0 ? (v4f){} : y * f;
        }
    if (part && h == 0) ca_part_ml(a, nsplit, part, HD, at) = make_float2(unit, l);
}

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
            if (p.dec) k_cattn_dec<HD, KV4, 8><<<(unsigned)n, 512, 0, s>>>(a, p.nsplit, p.chunk, part);
            else k_cattn_tile<HD, KV4, 8><<<(unsigned)(n * p.ncb), 512, 0, s>>>(a, p.ncb, p.nsplit, part);
            return;
        }
    if (p.dec)
        k_cattn_dec<HD, KV4, 4><<<(unsigned)n, 256, 0, s>>>(a, p.nsplit, p.chunk, part);
    else
        k_cattn_tile<HD, KV4, 4><<<(unsigned)(n * p.ncb), 256, 0, s>>>(a, p.ncb, p.nsplit, part);
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
