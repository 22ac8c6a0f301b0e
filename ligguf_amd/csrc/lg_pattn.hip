/* lg_pattn.hip -- attention over caches in pages, the rows that a group of
 * sequences shares once for the whole group (the kernels: lg_cattn.h). */
#include "lg_cattn.h"

/* A phase of a call: the shared rows (units are groups) or the own ones
 * (sequences), and how it is cut. */
enum PaKind { PA_DEC, PA_COLS, PA_TILE };
struct PaPhase {
    CAttnPaged a;
    int kind, ncb, cw, nsplit, chunk;
};
/* Both phases in one launch, the first one's workgroups before the second's. */
struct PaArgs {
    PaPhase f[2];
    int na;
    float* part;
    __device__ __forceinline__ const PaPhase& of(int blk) const { return f[blk < na ? 0 : 1]; }
    __device__ __forceinline__ int in(int blk) const { return blk < na ? blk : blk - na; }
};

constexpr int PA_WAVES = 4;                                      /* of the other kernels' */
constexpr int pa_blocks(int hd) { return hd <= 128 ? 2 : 1; }    /* of 16 columns, of pa_cols' waves */
constexpr int pa_waves(int hd) { return hd <= 64 ? 16 : 12; }   /* of k_pattn_tile's workgroups */

/* ca_query2 in 11 operations for two values, not 19: lo is 0 only where hi is, which
 * is rounded to 0 below 2^-37 of the row's largest value (there an infinite key's
 * score is NaN, as at a query's 0). */
__device__ __forceinline__ void pa_query2(float x0, float x1, int ex, v8h& hi, v8h& lo, int i)
{
    typedef uint16_t u2 __attribute__((ext_vector_type(2)));
    const u2 sign = {0x8000, 0x8000}, least = {1, 1};
    const float y0 = ldexpf(x0, 14 - ex), y1 = ldexpf(x1, 14 - ex);
    const lg_h2 h = __builtin_bit_cast(lg_h2, __builtin_amdgcn_cvt_pkrtz(y0, y1));
    const lg_h2 l = __builtin_convertvector(((lg_f2){__builtin_fmaf(-(float)h[0], 1.0f, y0), __builtin_fmaf(-(float)h[1], 1.0f, y1)}), lg_h2);
    const u2 hb = __builtin_bit_cast(u2, h), lb = __builtin_bit_cast(u2, l), ha = hb & ~sign;
    const lg_h2 b = __builtin_bit_cast(lg_h2, __builtin_elementwise_max(lb & ~sign, __builtin_elementwise_min(ha, least)) | (hb & sign));
    hi[i] = h[0];
    hi[i + 1] = h[1];
    lo[i] = b[0];
    lo[i + 1] = b[1];
}

/* ca_split2, the difference in one operation for a value, not two (ten prompts of 160 tokens behind 2900 shared rows,
 * 32 heads of 64: 104 -> 102 us) */
__device__ __forceinline__ void pa_split2(float x0, float x1, v8h& hi, v8h& lo, int i)
{
    float one = -1.0f;
    asm("" : "+s"(one));   /* (a constant's product would become a conversion and a subtraction) */
    const lg_h2 h = __builtin_convertvector(((lg_f2){x0, x1}), lg_h2);
    const lg_h2 l = __builtin_convertvector(((lg_f2){__builtin_fmaf((float)h[0], one, x0), __builtin_fmaf((float)h[1], one, x1)}), lg_h2);
    hi[i] = h[0];
    hi[i + 1] = h[1];
    lo[i] = l[0];
    lo[i + 1] = l[1];
}

/* Many columns: 16 a wave, NW waves a workgroup, which share tiles of KT keys in
 * LDS; the products of k_cattn_dec, 32 keys at a time:
 *   S^T[key][col] = K Q^T      O^T[d][col] += V^T P^T
 * 16 columns take so few registers that a SIMD has three or four waves to fill
 * each other's waits with.  More columns a wave read LDS less often, and are
 * slower for want of waves: 192 columns over 20000 keys in 12 waves of 16 70 us
 * in all, 8 of 32 82, 4 of 48 94; heads of 64, ten prompts, 16 waves of 16 104,
 * 8 of 32 119, 4 of 64 175.  The next tile's rows are on their way while one
 * computes (two LDS stages, one barrier a tile), its table entries while the one
 * before does.  Maxima lag by up to 2^8, raised but once or twice: a weight is
 * off by up to 2^-25, fp16's least step, where the largest is 2^7 or more.
 * Bound by VALU and MFMA, which one SIMD hardly overlaps: 55 % and 38 % of the
 * cycles with heads of 64 (ten prompts, 320 TFLOP/s of the products asked for, 640
 * issued; 4 bits 110 us, 58 % and 36 %), 35 % and 33 % with 128 over 20000 keys, five
 * tiles a workgroup after 8 us of first loads. */
template <int HD, bool KV4, int NW_>
struct PaTile {
    static constexpr int NW = NW_, NTH = 64 * NW, KT = 128;
    static constexpr int NS = (HD + 31) / 32, NT = HD / 16;
    static constexpr int KST = HD + 16, VST = HD + 16;       /* halves per K and V row in LDS: 8 banks on, no conflicts (4 for K: 1 in 2) */
    static constexpr int PW = KV4 ? 16 : 8, PR = HD / PW;    /* values of a piece that a thread moves, pieces of a row */
    static constexpr int NP = (2 * KT * PR + NTH - 1) / NTH; /* of a tile's keys and values per thread */
    static constexpr int STAGE = KT * (KST + VST);           /* halves */
    static constexpr bool WHOLE = 64 % PR == 0 && 16 % (64 / PR) == 0;   /* a wave's piece is rows of one page */
};

/* what a thread holds of a tile: pieces of its keys, then of its values */
template <int HD, bool KV4, int NW>
struct PaPieces {
    using C = PaTile<HD, KV4, NW>;
    v4u h[KV4 ? 1 : C::NP];
    uint2 w[KV4 ? C::NP : 1];
    uint32_t dm[KV4 ? C::NP : 1];

    /* the wave's piece u: its first one, from 0 on in keys and values */
    static __device__ __forceinline__ int first(int u)
    {
        return __builtin_amdgcn_readfirstlane(threadIdx.x & ~63) + u * C::NTH;
    }
    __device__ __forceinline__ void load(const CAttnPaged& a, int g, int kb, const CaEntries& id)
    {
        const int mask = a.page_rows() - 1, lane = threadIdx.x & 63;
        const uint32_t rb = KV4 ? HD / 2 : (uint32_t)a.c.n_kv * (HD * 2);                       /* bytes from row to row */
        const uint32_t at0 = KV4 ? (uint32_t)g * a.c.n_ctx * (HD / 2) : (uint32_t)g * (HD * 2);   /* the head's in a page */
        const uint32_t dm0 = (uint32_t)a.c.n_ctx * ((uint32_t)a.c.n_kv * (HD / 2) + (uint32_t)g * (HD / 8));
#pragma unroll
        for (int u = 0; u < C::NP; u++) {
            int i = first(u);
            if (i >= 2 * C::KT * C::PR) break;
            const uint8_t* const base = i < C::KT * C::PR ? a.c.k : a.c.v;
            i = i < C::KT * C::PR ? i : i - C::KT * C::PR;
            size_t at;
            uint32_t row, sub, x;   /* the wave's row and the lane's beyond it */
            if constexpr (C::WHOLE) {
                const int k0 = i / C::PR;
                at = id.at(a, k0 / 16);
                row = ((kb + k0) & mask & ~15) + k0 % 16;
                sub = lane / C::PR;
                x = lane % C::PR;
            } else {
                const int key = (i + lane) / C::PR;
                at = id.at(a, 0);
#pragma unroll
                for (int j = 1; j < C::KT / 16; j++) at = key >= 16 * j ? id.at(a, j) : at;
                row = (kb + key) & mask;
                sub = 0;
                x = (i + lane) % C::PR;
            }
            /* (a page's bytes fit 32 bits) */
            const uint8_t* const b = base + at + (at0 + row * rb);
            if constexpr (KV4) {
                w[u] = *(const uint2*)(b + (sub * rb + 8 * x));
                dm[u] = *(const uint32_t*)(base + at + (dm0 + row * (HD / 8)) + (sub * (HD / 8) + x / 2 * 4));
            } else
                h[u] = *(const v4u*)(b + (sub * rb + 16 * x));
        }
    }
    /* into a stage; with `bad`, values' infinities and NaN as 0 and their keys noted */
    __device__ __forceinline__ void store(_Float16* stage, uint32_t* bad) const
    {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int u = 0; u < C::NP; u++) {
            const int i0 = first(u);
            if (i0 >= 2 * C::KT * C::PR) break;
            const bool key_row = i0 < C::KT * C::PR;
            const int i = (key_row ? i0 : i0 - C::KT * C::PR) + lane, r = i / C::PR;
            _Float16* const q = stage + (key_row ? r * C::KST : C::KT * C::KST + r * C::VST) + i % C::PR * C::PW;
            v4u x[C::PW / 8];
            if constexpr (KV4) {
                lg_kv4_values(w[u].x, dm[u], (lg_h2*)&x[0]);
                lg_kv4_values(w[u].y, dm[u], (lg_h2*)&x[1]);
            } else
                x[0] = h[u];
            if (bad && !key_row) {
                bool any = false;
#pragma unroll
                for (int e = 0; e < C::PW / 8; e++) any |= ca_drop_bad(x[e]);
                if (any) atomicOr(bad + r / 32, 1u << (r % 32));
            }
#pragma unroll
            for (int e = 0; e < C::PW / 8; e++) *(v4u*)(q + 8 * e) = x[e];
        }
    }
};

/* Whether some column of positions lo .. hi does not see some key of the tile at kb. */
struct PaPartly {
    int klo, last, wlo, sinks, kt;
    __device__ __forceinline__ PaPartly(const CAttnPaged& a, int lo, int hi, int klo_, int khi, int kt_)
        : klo(klo_), last(min(khi - 1, lo) - kt_ + 1), wlo(a.window > 0 ? hi - a.window : INT32_MIN), sinks(a.sinks), kt(kt_)
    {
    }
    __device__ __forceinline__ bool operator()(int kb, int none) const
    {
        return (kb < klo) | (kb > last) | (none != 0) | ((kb <= wlo) & (kb + kt > sinks));
    }
};

template <int HD, bool KV4, int NW>
__global__ __launch_bounds__(64 * NW, NW / 4) void k_pattn_tile(PaArgs args)
{
    using C = PaTile<HD, KV4, NW>;
    constexpr int KT = C::KT, NS = C::NS, NT = C::NT;
    const PaPhase& f = args.of(blockIdx.x);
    const CAttnPaged& a = f.a;
    const int ncb = f.ncb, nsplit = f.nsplit, chunk = f.chunk, blk = args.in(blockIdx.x);
    float* const part = args.part;
    __shared__ __attribute__((aligned(16))) _Float16 s_kv[2 * C::STAGE];
    __shared__ int s_pos[2 * NW];
    __shared__ uint32_t s_bad[3][KT / 32];
    /* key head fastest, then the units; the last columns, which may see most, first */
    const int n_kv = a.c.n_kv, g = blk % n_kv, units = a.rows / a.ntok;
    const int unit = blk / n_kv % units, rest = blk / n_kv / units;
    const int sp = rest % nsplit, cb = ncb - 1 - rest / nsplit;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, c = lane >> 4;
    const int ncol = a.ntok * a.nrep, idx = (cb * NW + wave) * 16 + col;
    const int tok = min(idx, ncol - 1) / a.nrep, head = g * a.nrep + idx % a.nrep;
    const int64_t row = (int64_t)unit * a.ntok + tok;
    const int* const trow = a.table + (int64_t)unit * a.tstep * a.tstride;
    /* Without a window and from row 0 on the first tile is known: its entries and
     * rows are on their way before the positions are (there is one, unless the
     * unit has fewer keys than the launch was cut for). */
    const bool early = a.window <= 0 && (a.share || !a.prefix);
    CaEntries id, id1;   /* of the next tile and the one after */
    PaPieces<HD, KV4, NW> P;
    if (early) {
        id.load(a, trow, sp * chunk * KT);
        id1.load(a, trow, (sp * chunk + 1) * KT);
    }
    int klo, khi;
    a.range(unit, &klo, &khi);
    int p = a.pos[row];
    /* the columns' queries on their way */
    v4f x[2 * NS];
    {
        const float* const q = a.q + row * a.qs + (size_t)head * HD + 8 * c;
#pragma unroll
        for (int j = 0; j < 2 * NS; j++) {
            const int d = 32 * (j / 2) + 4 * (j % 2);
            x[j] = idx < ncol && (HD % 32 == 0 || d + 8 * c < HD) ? *(const v4f*)(q + d) : (v4f){};
        }
    }
    if (early) P.load(a, g, sp * chunk * KT, id);
    if (idx >= ncol || p > a.max_pos) p = -1;
    int wmin = p < 0 ? INT32_MAX : p, wmax = p;   /* of the wave */
#pragma unroll
    for (int o = 1; o < 16; o *= 2) {
        wmin = min(wmin, __shfl_xor(wmin, o));
        wmax = max(wmax, __shfl_xor(wmax, o));
    }
    if (lane == 0) {
        s_pos[2 * wave] = wmin;
        s_pos[2 * wave + 1] = wmax;
    }
    if (threadIdx.x < 3 * KT / 32) s_bad[threadIdx.x / (KT / 32)][threadIdx.x % (KT / 32)] = 0;
    __syncthreads();
    wmin = __builtin_amdgcn_readfirstlane(wmin);
    wmax = __builtin_amdgcn_readfirstlane(wmax);
    int pmin = INT32_MAX, pmax = -1;              /* of the workgroup */
#pragma unroll
    for (int w = 0; w < NW; w++) {
        pmin = min(pmin, s_pos[2 * w]);
        pmax = max(pmax, s_pos[2 * w + 1]);
    }
    pmin = __builtin_amdgcn_readfirstlane(pmin);
    pmax = __builtin_amdgcn_readfirstlane(pmax);

    v4f o[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) o[t] = (v4f){};
    float l = 0.0f, unit2 = -INFINITY;
    const CaTiles tiles(a, pmin, pmax, KT, klo, khi);
    int t0, t1;
    tiles.chunk(sp, nsplit, chunk, &t0, &t1);
    if (t0 < t1) {   /* (workgroup-uniform) */
        /* tiles with keys that some row of the workgroup (wave) does not see */
        const PaPartly some(a, pmin, pmax, klo, khi, KT), mine(a, wmin, wmax, klo, khi, KT);
        const int wfirst = a.window > 0 ? wmin - a.window - KT + 1 : INT32_MIN;   /* tiles up to it are before the wave's windows */
        const CaSeen seen(a, p, klo, khi);
        int kb = tiles.at(t0) * KT, kn = tiles.at(min(t0 + 1, t1 - 1)) * KT;
        if (!early || kb != sp * chunk * KT) {
            id.load(a, trow, kb);
            id1.load(a, trow, kn);
            P.load(a, g, kb, id);
        }
        int none = id.none(a, KT / 16);   /* rows 16 j .. of the present tile have no page: bit j */
        v8h qh[NS], ql[NS];
        float big = 0.0f;
        CaMaxOf<7, 8> mx;
        if (wmax >= 0) {   /* (a wave without rows has but the tiles to move) */
#pragma unroll
        for (int j = 0; j < 2 * NS; j++)
            big = fmaxf(fmaxf(big, fmaxf(fabsf(x[j][0]), fabsf(x[j][1]))), fmaxf(fabsf(x[j][2]), fabsf(x[j][3])));
        big = fmaxf(big, lg_partner<4>(big));
        big = fmaxf(big, lg_partner<5>(big));
        const int ex = __builtin_amdgcn_frexp_expf(big);
        mx = CaMaxOf<7, 8>(ca_scale(a.scale2, ex));
#pragma unroll
        for (int j = 0; j < NS; j++)
#pragma unroll
            for (int e = 0; e < 8; e += 2) pa_query2(x[2 * j + e / 4][e % 4], x[2 * j + e / 4][e % 4 + 1], ex, qh[j], ql[j], e);
        }
        bool dropped = some(kb, none);   /* the present tile's infinities and NaN are zeros, their keys in s_bad */
        P.store(s_kv, dropped ? s_bad[0] : nullptr);
        __syncthreads();
        for (int it = t0; it < t1; it++) {
            const bool more = it + 1 < t1;
            const int cur = (it - t0) & 1, slot = (it - t0) % 3;
            const _Float16* const sK = s_kv + cur * C::STAGE;
            const _Float16* const sV = sK + KT * C::KST;
            const bool on = (kb <= wmax) & ((kb > wfirst) | (kb < a.sinks));
            const int k2 = tiles.at(min(it + 2, t1 - 1)) * KT;
            int none1 = 0;
            /* the next tile's rows: not at once, when all waves would work out addresses, but where they have drifted apart */
            auto next = [&]() __attribute__((always_inline)) {
                if (more) {
                    id = id1;
                    id1.load(a, trow, k2);
                    P.load(a, g, kn, id);
                    none1 = id.none(a, KT / 16);
                }
            };
            if (threadIdx.x < KT / 32) s_bad[(slot + 2) % 3][threadIdx.x] = 0;
            if (!on) next();
            else {
                const bool part_seen = mine(kb, none);
#pragma unroll
                for (int b = 0; b < KT / 32; b++) {
                    v4f s[2];
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        s[u] = (v4f){};
#pragma unroll
                        for (int j = 0; j < NS; j++) {
                            const v8h k = HD % 32 == 0 || 32 * j + 8 * c < HD ?
                                              *(const v8h*)(sK + (32 * b + 16 * u + col) * C::KST + 32 * j + 8 * c) : (v8h){};
                            s[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qh[j], s[u], 0, 0, 0);
                            s[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, ql[j], s[u], 0, 0, 0);
                        }
                    }
                    if (b == 0) next();
                    if (part_seen) {
#pragma unroll
                        for (int u = 0; u < 2; u++)
#pragma unroll
                            for (int i = 0; i < 4; i++)
                                s[u][i] = seen(kb + 32 * b + 16 * u + 4 * c + i, kb, none) ? s[u][i] : -INFINITY;
                    }
                    /* the weights; whether one outgrew its maximum, their sum tells */
                    float w[8], sum;
                    auto weigh = [&]() __attribute__((always_inline)) {
#pragma unroll
                        for (int i = 0; i < 8; i++) w[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i / 4][i % 4], mx.sc, mx.cc));
                        sum = ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
                    };
                    weigh();
                    if (mx.over(sum)) {
                        float mn = fmaxf(s[0][0], s[1][0]);
#pragma unroll
                        for (int i = 1; i < 4; i++) mn = fmaxf(mn, fmaxf(s[0][i], s[1][i]));
                        mn = fmaxf(mn, lg_partner<4>(mn));
                        mn = fmaxf(mn, lg_partner<5>(mn));
                        float off;
                        const float al = mx.raise(mn, &off);
                        l *= al;
#pragma unroll
                        for (int t = 0; t < NT; t++) o[t] *= al;
                        s[0] -= off;
                        s[1] -= off;
                        weigh();
                    }
                    l += sum;
                    v8h ph, pl;
#pragma unroll
                    for (int i = 0; i < 8; i += 2) pa_split2(w[i], w[i + 1], ph, pl, i);
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        const _Float16* const v = sV + (32 * b + 4 * c + col / 4) * C::VST + 16 * t + 4 * (col % 4);
                        const v4s x0 = ca_tr16(v), x1 = ca_tr16(v + 16 * C::VST);
                        const v8h y = __builtin_bit_cast(v8h, __builtin_shufflevector(x0, x1, 0, 1, 2, 3, 4, 5, 6, 7));
                        o[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(y, ph, o[t], 0, 0, 0);
                        o[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(y, pl, o[t], 0, 0, 0);
                    }
                }
                /* infinities and NaN of keys that only some rows of the workgroup see:
                 * added by itself to those that do, whatever the (positive) weight,
                 * in waves that see all of the tile too */
                if (dropped)
                    for (int w = 0; w < KT / 32; w++)
                        for (uint32_t keys = __builtin_amdgcn_readfirstlane(s_bad[slot][w]); keys; keys &= keys - 1) {
                            const int key = kb + 32 * w + __builtin_ctz(keys);
                            if (seen(key, kb, none))
#pragma unroll
                                for (int t = 0; t < NT; t++) {
                                    const v4f y = ca_values<KV4>(a, a.c.v, trow, g, key, 16 * t + 4 * c);
#pragma unroll
                                    for (int i = 0; i < 4; i++) o[t][i] = ca_add_bad(o[t][i], y[i]);
                                }
                        }
            }
            dropped = some(kn, none1);
            if (more) P.store(s_kv + (cur ^ 1) * C::STAGE, dropped ? s_bad[(slot + 1) % 3] : nullptr);
            none = none1;
            kb = kn;
            kn = k2;
            __syncthreads();
        }
        l += lg_partner<4>(l);
        l += lg_partner<5>(l);
        unit2 = mx.unit(l);
    }
    if (idx >= ncol) return;
    const int64_t at = ((int64_t)(a.part0 + sp) * a.rows + row) * a.n_heads + head;
    if (!part) {
        const float f = p < 0 || l == 0.0f ? 0.0f : 1.0f / l;
        float* const dst = a.out + row * a.os + (size_t)head * HD + 4 * c;
#pragma unroll
        for (int t = 0; t < NT; t++) *(v4f*)(dst + 16 * t) = f == 0.0f && (p < 0 || l == 0.0f) ? (v4f){} : o[t] * f;
        return;
    }
    if (l != 0.0f) {   /* (a part without keys is not read) */
#pragma unroll
        for (int t = 0; t < NT; t++) *(v4f*)(part + at * HD + 4 * c + 16 * t) = o[t];
    }
    if (c == 0) ca_part_ml(a, a.nparts, part, HD, at) = make_float2(unit2, l);
}

/* More than 16 columns (query heads of a key head, tokens in order): 16 NCB a wave,
 * the products of k_cattn_dec,
 *   S^T[key][col] = K Q^T      O^T[d][col] += V^T P^T
 * with each key's and value's fragment used for all of a wave's columns, 32 of them
 * or, with heads of 256, 16, which need no more registers than there are (48 sequences
 * behind 5000 rows, 16 heads 72 -> 64 us, a prompt of 300 tokens 74 -> 46).  Of a
 * workgroup's NW waves `cw` (1, 2 or all) have columns of their own and NW / cw
 * share those, each with tiles of KT keys of its own.  Waves with the same keys
 * read them through the first-level cache and wait for nothing but their own
 * loads: of few columns or keys tiles in LDS cost more in barriers and address
 * work, of which all waves then do the same at the same time, than their reads
 * took (both measured: pa_plan).  Maxima lag by up to 2^8, as above.  Bound by
 * first loads, then VALU: nine groups of 24 columns over up to 5000 keys of 4 bits
 * and 250 own 42 us, 47 % VALU, 12 % MFMA. */
template <int HD, bool KV4, int NW, int NCB>
__device__ __forceinline__ void pa_cols(const CAttnPaged& a, int blk, int ncb, int cw, int nsplit, int chunk, float* __restrict__ part,
                                        uint8_t* s_raw, float (*s_ml)[16][2])
{
    using C = CaDec<HD, KV4>;
    constexpr int KT = C::KT, NU = C::NU, NB = C::NB, NS = C::NS, NT = C::NT;
    /* key head fastest, then columns, which read the same keys; the last ones, which may see most, first */
    const int n_kv = a.c.n_kv, g = blk % n_kv, units = a.rows / a.ntok;
    const int cb = ncb - 1 - blk / n_kv % ncb, rest = blk / n_kv / ncb, unit = rest % units, sp = rest / units;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kg = wave / cw, nkg = NW / cw, cwave = wave - kg * cw;
    const int col = lane & 15, c = lane >> 4;
    const int ncol = a.ntok * a.nrep, idx0 = ((cb * cw + cwave) * NCB) * 16 + col;
    int klo, khi;
    a.range(unit, &klo, &khi);
    /* the first tile's entries and rows on their way before the positions are, where it is known (see ca_dec) */
    CaEntries id, id1, id2;   /* of the present tile, the next and the one after */
    CaRows<HD, KV4> K, V;
    const int* const trow = a.table + (int64_t)unit * a.tstep * a.tstride;
    int ahead = -1;
    if (a.window <= 0) {
        ahead = (klo / KT + sp * chunk + kg) * KT;
        if (ahead > a.max_pos) ahead = -1;
    }
    if (ahead >= 0) {
        id.load(a, trow, ahead);
        id1.load(a, trow, ahead + nkg * KT);
    }
    int p[NCB];
    v4f x[NCB][2 * NS];
    float big[NCB];
#pragma unroll
    for (int n = 0; n < NCB; n++) {
        const int idx = idx0 + 16 * n, tok = min(idx, ncol - 1) / a.nrep, head = g * a.nrep + idx % a.nrep;
        const int64_t row = (int64_t)unit * a.ntok + tok;
        p[n] = a.pos[row];
        const float* const q = a.q + row * a.qs + (size_t)head * HD;
#pragma unroll
        for (int s = 0; s < NS; s++) {
            const int d = C::dim(s, c);
            const bool in = idx < ncol && d < HD;
            x[n][2 * s] = in ? *(const v4f*)(q + d) : (v4f){};
            x[n][2 * s + 1] = in ? *(const v4f*)(q + d + 4) : (v4f){};
        }
    }
    if (ahead >= 0) {
        K.load(a, a.c.k, g, ahead, id, col, c);
        V.load(a, a.c.v, g, ahead, id, col, c);
    }
    int pmin = INT32_MAX, pmax = -1;   /* of the wave's columns */
#pragma unroll
    for (int n = 0; n < NCB; n++) {
        if (idx0 + 16 * n >= ncol || p[n] > a.max_pos) p[n] = -1;
        pmin = min(pmin, p[n] < 0 ? INT32_MAX : p[n]);
        pmax = max(pmax, p[n]);
    }
#pragma unroll
    for (int o = 1; o < 16; o *= 2) {
        pmin = min(pmin, __shfl_xor(pmin, o));
        pmax = max(pmax, __shfl_xor(pmax, o));
    }
    pmin = __builtin_amdgcn_readfirstlane(pmin);
    pmax = __builtin_amdgcn_readfirstlane(pmax);

    v4f o[NCB][NT];
    float l[NCB], unit2[NCB];
#pragma unroll
    for (int n = 0; n < NCB; n++) {
#pragma unroll
        for (int t = 0; t < NT; t++) o[n][t] = (v4f){};
        l[n] = 0.0f;
        unit2[n] = -INFINITY;
    }
    const CaTiles tiles(a, pmin, pmax, KT, klo, khi);
    int t0, t1;
    tiles.chunk(sp, nsplit, chunk, &t0, &t1);
    if (t0 + kg < t1) {       /* (the wave's) */
        _Float16* const sV = (_Float16*)(s_raw + wave * C::WAVE);
        int it = t0 + kg, kb = tiles.at(it) * KT;
        auto ids_of = [&](int i, CaEntries& to) __attribute__((always_inline)) { to.load(a, trow, tiles.at(min(i, t1 - 1)) * KT); };
        if (kb != ahead) {
            ids_of(it, id);
            ids_of(it + nkg, id1);
            K.load(a, a.c.k, g, kb, id, col, c);
            V.load(a, a.c.v, g, kb, id, col, c);
        }
        v8h qh[NCB][NS], ql[NCB][NS];
        int ex[NCB];
#pragma unroll
        for (int n = 0; n < NCB; n++) {
            big[n] = 0.0f;
#pragma unroll
            for (int i = 0; i < 2 * NS; i++)
                big[n] = fmaxf(fmaxf(big[n], fmaxf(fabsf(x[n][i][0]), fabsf(x[n][i][1]))), fmaxf(fabsf(x[n][i][2]), fabsf(x[n][i][3])));
            big[n] = fmaxf(big[n], lg_partner<4>(big[n]));
            big[n] = fmaxf(big[n], lg_partner<5>(big[n]));
            ex[n] = __builtin_amdgcn_frexp_expf(big[n]);   /* big < 2^ex */
#pragma unroll
            for (int j = 0; j < NS; j++)
#pragma unroll
                for (int e = 0; e < 8; e += 2)
                    pa_query2(x[n][2 * j + e / 4][e % 4], x[n][2 * j + e / 4][e % 4 + 1], ex[n], qh[n][j], ql[n][j], e);
        }
        CaMaxOf<7, 8> mx[NCB];
#pragma unroll
        for (int n = 0; n < NCB; n++) mx[n] = CaMaxOf<7, 8>(ca_scale(a.scale2, ex[n]));
        for (; it < t1; it += nkg) {
            v4f s[NU][NCB];
#pragma unroll
            for (int u = 0; u < NU; u++) {
#pragma unroll
                for (int n = 0; n < NCB; n++) s[u][n] = (v4f){};
#pragma unroll
                for (int j = 0; j < NS; j++) {
                    const v8h k = __builtin_bit_cast(v8h, K.get(u, j));
#pragma unroll
                    for (int n = 0; n < NCB; n++) s[u][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qh[n][j], s[u][n], 0, 0, 0);
#pragma unroll
                    for (int n = 0; n < NCB; n++) s[u][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, ql[n][j], s[u][n], 0, 0, 0);
                }
            }
            const int kn = it + nkg < t1 ? tiles.at(it + nkg) * KT : -1;
            ids_of(it + 2 * nkg, id2);
            if (kn >= 0) K.load(a, a.c.k, g, kn, id1, col, c);
            const int none = id.none(a, NU);
            /* whether some column does not see some of the keys */
            const bool part_seen = kb + KT > khi || kb < klo || none || kb + KT - 1 > pmin ||
                                   (a.window > 0 && kb <= pmax - a.window && kb + KT > a.sinks);
            if (part_seen) {
#pragma unroll
                for (int n = 0; n < NCB; n++) {
                    const CaSeen seen(a, p[n], klo, khi);
#pragma unroll
                    for (int u = 0; u < NU; u++)
#pragma unroll
                        for (int i = 0; i < 4; i++) s[u][n][i] = seen(kb + 16 * u + 4 * c + i, kb, none) ? s[u][n][i] : -INFINITY;
                }
            }
            uint64_t bad = 0;   /* keys of the tile */
#pragma unroll
            for (int b = 0; b < NB; b++) {
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int j = 0; j < NS; j++) {
                        v4u y = V.get(2 * b + u, j);
                        if (part_seen) bad |= ca_row16(__builtin_amdgcn_ballot_w64(ca_drop_bad(y))) << (32 * b + 16 * u);
                        if (HD % 32 == 0 || C::dim(j, c) < HD) *(v4u*)(sV + (16 * u + col) * C::VST + C::dim(j, c)) = y;
                    }
                if (b == NB - 1 && kn >= 0) V.load(a, a.c.v, g, kn, id1, col, c);
                v8h ph[NCB], pl[NCB];
#pragma unroll
                for (int n = 0; n < NCB; n++) {
                    /* the weights; whether one outgrew its maximum, their sum tells */
                    v4f &s0 = s[2 * b][n], &s1 = s[2 * b + 1][n];
                    float w[8], sum;
                    auto weigh = [&]() __attribute__((always_inline)) {
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            w[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s0[i], mx[n].sc, mx[n].cc));
                            w[4 + i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s1[i], mx[n].sc, mx[n].cc));
                        }
                        sum = ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
                    };
                    weigh();
                    if (mx[n].over(sum)) {
                        float mn = fmaxf(s0[0], s1[0]);
#pragma unroll
                        for (int i = 1; i < 4; i++) mn = fmaxf(mn, fmaxf(s0[i], s1[i]));
                        mn = fmaxf(mn, lg_partner<4>(mn));
                        mn = fmaxf(mn, lg_partner<5>(mn));
                        float off;
                        const float al = mx[n].raise(mn, &off);
                        l[n] *= al;
#pragma unroll
                        for (int t = 0; t < NT; t++) o[n][t] *= al;
                        s0 -= off;
                        s1 -= off;
                        weigh();
                    }
                    l[n] += sum;
#pragma unroll
                    for (int i = 0; i < 8; i += 2) pa_split2(w[i], w[i + 1], ph[n], pl[n], i);
                }
                ca_wave_sync();
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    const _Float16* const v = sV + (4 * c + col / 4) * C::VST + 16 * t + 4 * (col % 4);
                    const v4s x0 = ca_tr16(v), x1 = ca_tr16(v + 16 * C::VST);
                    const v8h y = __builtin_bit_cast(v8h, __builtin_shufflevector(x0, x1, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
                    for (int n = 0; n < NCB; n++) o[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(y, ph[n], o[n][t], 0, 0, 0);
#pragma unroll
                    for (int n = 0; n < NCB; n++) o[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(y, pl[n], o[n][t], 0, 0, 0);
                }
                ca_wave_sync();   /* (the reads before the next block's writes) */
            }
            /* infinities and NaN of keys that only some columns see: added by
             * itself to those that do, whatever the (positive) weight */
            for (; bad; bad &= bad - 1) {
                const int key = kb + __builtin_ctzll(bad);
#pragma unroll
                for (int n = 0; n < NCB; n++)
                    if (CaSeen(a, p[n], klo, khi)(key, kb, none))
#pragma unroll
                        for (int t = 0; t < NT; t++) {
                            const v4f y = ca_values<KV4>(a, a.c.v, trow, g, key, 16 * t + 4 * c);
#pragma unroll
                            for (int i = 0; i < 4; i++) o[n][t][i] = ca_add_bad(o[n][t][i], y[i]);
                        }
            }
            kb = kn;
            id = id1;
            id1 = id2;
        }
#pragma unroll
        for (int n = 0; n < NCB; n++) {
            l[n] += lg_partner<4>(l[n]);
            l[n] += lg_partner<5>(l[n]);
            unit2[n] = mx[n].unit(l[n]);
        }
    }
    /* a column's sums, by one lane for four dims of each t: as a part, or as they are */
    auto put = [&](int idx, int d, v4f y, float M, float L) __attribute__((always_inline)) {
        if (idx >= ncol) return;
        const int tok = idx / a.nrep, head = g * a.nrep + idx % a.nrep;
        const int64_t row = (int64_t)unit * a.ntok + tok;
        if (part) {
            const int64_t at = ((int64_t)(a.part0 + sp) * a.rows + row) * a.n_heads + head;
            if (L != 0.0f) *(v4f*)(part + at * HD + d) = y;
            if (d == 0) ca_part_ml(a, a.nparts, part, HD, at) = make_float2(M, L);
        } else {
            const int pk = a.pos[row];
            *(v4f*)(a.out + row * a.os + (size_t)head * HD + d) = pk < 0 || pk > a.max_pos || L == 0.0f ? (v4f){} : y * (1.0f / L);
        }
    };
    if (nkg == 1) {   /* (kg is 0) */
#pragma unroll
        for (int n = 0; n < NCB; n++)
#pragma unroll
            for (int t = 0; t < NT; t++) put(idx0 + 16 * n, 16 * t + 4 * c, o[n][t], unit2[n], l[n]);
        return;
    }
    /* the waves' parts of each column together, 16 columns of each at a time, by way of LDS */
#pragma unroll
    for (int n = 0; n < NCB; n++) {
        float* const sO = (float*)(s_raw + wave * C::WAVE);
        if (n) __syncthreads();
#pragma unroll
        for (int t = 0; t < NT; t++) *(v4f*)(sO + col * C::OST + 16 * t + 4 * c) = o[n][t];
        if (c == 0) {
            s_ml[wave][col][0] = unit2[n];
            s_ml[wave][col][1] = l[n];
        }
        __syncthreads();
        for (int i = threadIdx.x; i < cw * 16 * (HD / 4); i += 64 * NW) {
            const int w0 = i / (16 * (HD / 4)), k = i / (HD / 4) % 16, d = i % (HD / 4) * 4;
            float M = -INFINITY, L = 0.0f;
            for (int w = w0; w < NW; w += cw) M = fmaxf(M, s_ml[w][k][0]);
            v4f y = {};
            for (int w = w0; w < NW; w += cw) {
                /* (a wave without keys has l = 0 and all zeros) */
                const float lw = s_ml[w][k][1], f = lw == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(s_ml[w][k][0] - M);
                const v4f v = *(const v4f*)((const float*)(s_raw + w * C::WAVE) + k * C::OST + d);
                L = __builtin_fmaf(lw, f, L);
#pragma unroll
                for (int e = 0; e < 4; e++) y[e] = __builtin_fmaf(v[e], f, y[e]);
            }
            put(((cb * cw + w0) * NCB + n) * 16 + k, d, y, M, L);
        }
    }
}

template <int HD, bool KV4, int NW>
__global__ __launch_bounds__(64 * NW, (HD <= 128 ? 2 : 1)) void k_pattn_cols(PaArgs args)
{
    __shared__ __attribute__((aligned(16))) uint8_t s_raw[NW * CaDec<HD, KV4>::WAVE];
    __shared__ float s_ml[NW][16][2];
    const PaPhase& f = args.of(blockIdx.x);
    pa_cols<HD, KV4, NW, pa_blocks(HD)>(f.a, args.in(blockIdx.x), f.ncb, f.cw, f.nsplit, f.chunk, args.part, s_raw, s_ml);
}

template <int HD, bool KV4, int NW>
__global__ __launch_bounds__(64 * NW, (HD <= 128 ? 2 : 1)) void k_pattn_dec(PaArgs args)
{
    __shared__ __attribute__((aligned(16))) uint8_t s_raw[NW * CaDec<HD, KV4>::WAVE];
    __shared__ float s_ml[NW][16][2];
    const PaPhase& f = args.of(blockIdx.x);
    ca_dec<HD, KV4, NW>(f.a, args.in(blockIdx.x), f.nsplit, f.chunk, args.part, s_raw, s_ml);
}

/* shared rows by the one, own rows by the other */
template <int HD, bool KV4, int NW>
__global__ __launch_bounds__(64 * NW, (HD <= 128 ? 2 : 1)) void k_pattn_cols_dec(PaArgs args)
{
    __shared__ __attribute__((aligned(16))) uint8_t s_raw[NW * CaDec<HD, KV4>::WAVE];
    __shared__ float s_ml[NW][16][2];
    const PaPhase& f = args.of(blockIdx.x);
    if ((int)blockIdx.x < args.na)
        pa_cols<HD, KV4, NW, pa_blocks(HD)>(f.a, blockIdx.x, f.ncb, f.cw, f.nsplit, f.chunk, args.part, s_raw, s_ml);
    else ca_dec<HD, KV4, NW>(f.a, blockIdx.x - args.na, f.nsplit, f.chunk, args.part, s_raw, s_ml);
}

/* How a phase is cut. */
struct PaCut {
    int kind;
    int cw, ncb;         /* waves with columns of their own; blocks of columns */
    int nsplit, chunk;   /* parts of the keys, tiles in a part */
    int64_t blocks;
    double us;           /* about */
};

/* units of ntok rows each over `keys` keys by one kind of kernel.  Its time is counted in tiles: rounds of workgroups,
 * as many as fit the chip at once, each of a start worth some tiles and the tiles of its part; parts are written and
 * read once.  More of them fill the chip, until their starts and the join cost more: 192 columns over 20000 keys in 13
 * parts 95 us, in 32 (all CUs) 63; 24 columns of nine groups over 4000 keys, 4 bits, in 1 part 76 us, 4 41, 6 44, 13 56;
 * 2240 columns of two groups over 1500 keys in 1 part 89 us, 2 114, 6 151. */
static PaCut pa_cut(int kind, int64_t units, int64_t ntok, int n_heads, int n_kv, int hd, int64_t keys, bool kv4, bool lone)
{
    const int64_t cols = ntok * (n_heads / n_kv);
    PaCut p = {kind};
    int kt = kv4 && hd <= 128 ? 64 : 32;   /* (CaDec::KT) */
    p.cw = p.ncb = 1;
    double slots = hd <= 128 ? 512.0 : 256.0, start = 3.0, join = 1.5e-6;
    /* about: a tile's microseconds, starts and tiles of 4 bits (twice the keys) in those of fp16 */
    double tile_us = 0.3 + 0.0164 * hd, start_of = kv4 ? 0.6 : 1.0, tile_of = kv4 ? 2.0 : 1.0;
    int64_t wide = PA_WAVES;   /* tiles that a workgroup has at a time */
    if (kind == PA_TILE) {
        const int64_t width = 16 * pa_waves(hd);
        p.ncb = (int)((cols + width - 1) / width);
        kt = 128;   /* (PaTile::KT) */
        slots = 256.0;
        wide = 1;
        start = 1.5;
        join = 0.3e-6;
        /* (waves without columns leave the others more of their SIMD) */
        tile_us = (0.6 + 0.0234 * hd) * (0.5 + 0.5 * (double)cols / (double)(p.ncb * width));
        start_of = tile_of = 1.0;
    } else if (kind == PA_COLS) {
        const int64_t nb = (cols + 16 * pa_blocks(hd) - 1) / (16 * pa_blocks(hd));
        for (p.cw = PA_WAVES; p.cw > 1 && (nb + p.cw - 1) / p.cw * p.cw * 8 > nb * 9; p.cw /= 2) {}
        p.ncb = (int)((nb + p.cw - 1) / p.cw);
        wide = PA_WAVES / p.cw;
    }
    const double tiles = std::max(1.0, (double)((keys + kt - 1) / kt) / (double)wide);   /* one after the other */
    const int64_t wgs = units * n_kv * p.ncb;
    double best = 0.0;
    /* (those of both phases together: CA_PARTS at most) */
    for (int ns = 1; ns <= (lone ? CA_PARTS : CA_PARTS / 2) && (ns == 1 || tiles / ns >= 1.0); ns++) {
        const double rounds = ceil((double)(wgs * ns) / slots), parts = ns > 1 ? join * ns * (double)(units * ntok) * n_heads * hd : 0.0;
        const double cost = rounds * (start + tiles / ns) + (lone && ns > 1 ? 2.0 : 0.0) + parts;
        if (ns == 1 || cost < best) {
            best = cost;
            p.nsplit = ns;
            p.us = tile_us * (rounds * (start * start_of + tiles / ns * tile_of) + parts);
        }
    }
    p.chunk = (int)((keys + (int64_t)kt * p.nsplit - 1) / ((int64_t)kt * p.nsplit));
    p.blocks = wgs * p.nsplit;
    return p;
}

/* How a call is cut: the shared rows as a sequence of all the group's rows, the
 * others sequence by sequence; their parts one behind the other. */
struct PaPlan {
    bool shared;
    PaCut a, b;    /* shared rows, own rows */
    int parts;     /* 1: written out as they are */
    size_t ws;
};

static PaPlan pa_plan(int64_t nseq, int64_t ntok, int n_heads, int n_kv, int hd, int window, int sinks, int max_pos, bool kv4,
                      int group, int max_prefix)
{
    PaPlan p = {};
    p.shared = group > 1 && max_prefix > 0;
    auto cut = [&](int kind, bool shared, int top) {
        const int64_t n = shared ? ntok * group : ntok;
        int64_t keys = (int64_t)top + 1;
        if (window > 0) keys = std::min(keys, (int64_t)window + sinks + n - 1);
        return pa_cut(kind, shared ? nseq / group : nseq, n, n_heads, n_kv, hd, keys, kv4, !p.shared);
    };
    const int64_t rep = n_heads / n_kv, cols = ntok * rep;
    /* Own rows (their number lies in device memory: taken to be what max_pos leaves beyond max_prefix; four sequences of
     * 3000 behind 2000 shared rows 23 us, with max_prefix 5000, for one own row, 54).  Of many columns tiles in LDS: 2000 tokens
     * of 32 heads of 128 92 us against 179, 64 18 against 20.  Not where heads of 64 fill the chip with less than a tile
     * a workgroup: 64 tokens 15 against 13, 256 22 against 18, 512 27 and 26, 1024 39 against 47. */
    const int top = p.shared ? std::max(max_pos - max_prefix, 0) : max_pos;
    if (cols <= 16) p.b = cut(PA_DEC, false, top);
    else {
        if (hd <= 128 && cols > 64) p.b = cut(PA_TILE, false, top);
        if (hd > 128 || cols <= 64 || (hd <= 64 && p.b.blocks * p.b.chunk < 256)) p.b = cut(PA_COLS, false, top);
    }
    /* Shared rows: whichever takes less by the estimates.  Tiles in LDS are a launch of their own unless the own rows have
     * such too, which counts as 25 us; with that and the tiles' times the choice is 1 % from the faster one in the mean of
     * 222 calls of both types, always the one or the other 9 % and 12 %.  With single tokens' own rows, 32 heads of 128, 8
     * key heads: 192 columns over 700 keys 36 us against 26, over 5000 44 against 40, over 20000 61 against 80; 64 over
     * 3000 28 against 27, over 20000 37 against 44; twelve groups of 80 columns over 600 61 against 51.  Two groups of
     * prompts, 2240 columns over 1500 keys, 4 bits, 90 against 165. */
    if (p.shared) {
        const int last = std::min(max_prefix - 1, max_pos);
        if (cols * group <= 16) p.a = cut(PA_DEC, true, last);
        else {
            p.a = cut(PA_COLS, true, last);
            if (hd <= 128 && cols * group > 32) {
                const PaCut t = cut(PA_TILE, true, last);
                if (t.us + (p.b.kind == PA_TILE ? 0.0 : 25.0) < p.a.us) p.a = t;
            }
        }
    }
    p.parts = p.b.nsplit + (p.shared ? p.a.nsplit : 0);
    if (p.parts > 1) p.ws = (size_t)p.parts * nseq * ntok * n_heads * (hd + 2) * sizeof(float);
    return p;
}

template <int HD, bool KV4>
static void pa_launch(const PaArgs& x, int64_t nb, hipStream_t s)
{
    constexpr int NW = PA_WAVES;
    const int ka = x.na ? x.f[0].kind : x.f[1].kind, kb = x.f[1].kind;
    const unsigned n = (unsigned)(x.na + nb);
    auto one = [&](const PaArgs& y, int kind, unsigned blocks) {
        if (kind == PA_DEC) k_pattn_dec<HD, KV4, NW><<<blocks, 64 * NW, 0, s>>>(y);
        else if (kind == PA_COLS) k_pattn_cols<HD, KV4, NW><<<blocks, 64 * NW, 0, s>>>(y);
        else if constexpr (HD <= 128) k_pattn_tile<HD, KV4, pa_waves(HD)><<<blocks, 64 * pa_waves(HD), 0, s>>>(y);
    };
    if (ka == kb) one(x, ka, n);
    else if (ka == PA_COLS && kb == PA_DEC) k_pattn_cols_dec<HD, KV4, NW><<<n, 64 * NW, 0, s>>>(x);
    else {
        one(x, ka, (unsigned)x.na);
        PaArgs y = x;
        y.na = 0;
        one(y, kb, (unsigned)nb);
    }
}

template <int HD>
static void pa_type(const PaArgs& x, int64_t nb, hipStream_t s)
{
    if constexpr (HD != 48)
        if (x.f[1].a.c.type == LG_KV4) return pa_launch<HD, true>(x, nb, s);
    pa_launch<HD, false>(x, nb, s);
}

/* a window of all positions is none (and differences of positions and windows fit 32 bits) */
static int pa_window(int window, int max_pos) { return window > max_pos ? 0 : window; }

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
    return pa_plan(nseq, ntok, n_heads, cache->pool.n_kv_heads, cache->pool.head_dim, pa_window(window, max_pos), sinks, max_pos,
                   cache->pool.type == LG_KV4, group, std::min(max_prefix, max_pos + 1)).ws;
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
    window = pa_window(window, max_pos);
    max_prefix = std::min(max_prefix, max_pos + 1);   /* (rows behind are not seen) */
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
    const int64_t na = p.shared ? p.a.blocks : 0, nb = p.b.blocks;
    const bool by_group = p.parts > 8 || rows * n_heads <= 4096;   /* (as lg_attn_cache) */
    const int64_t joins = p.ws ? by_group ? rows * n_heads : (rows * n_heads * (hd / 4) + 255) / 256 : 0;
    if (!lg_grid_fits(na + nb, 1024) || !lg_grid_fits(joins, 256)) {
        lg_set_error("%s: %lld rows of %d heads are too many for one call", who, (long long)rows, n_heads);
        return LG_ERR_ARG;
    }
    if (p.ws && (!workspace || !lg_al16(workspace) || workspace_bytes < p.ws)) {
        lg_set_error("%s: workspace of %zu bytes, 16-byte aligned, %zu needed", who, workspace_bytes, p.ws);
        return LG_ERR_ARG;
    }
    hipStream_t s = (hipStream_t)stream;
    float* const part = p.ws ? (float*)workspace : nullptr;
    auto phase = [&](const PaCut& c, int units_of, int part0) {
        PaPhase f = {a, c.kind, c.ncb, c.cw, c.nsplit, c.chunk};
        f.a.ntok = ntok * units_of;
        f.a.tstep = units_of;
        f.a.part0 = part0;
        return f;
    };
    PaArgs x = {};
    x.na = (int)na;
    x.part = part;
    if (p.shared) {
        x.f[0] = phase(p.a, group, 0);
        x.f[0].a.share = 1;
    }
    x.f[1] = phase(p.b, 1, p.shared ? p.a.nsplit : 0);
    switch (hd) {
    case 48: pa_type<48>(x, nb, s); break;
    case 64: pa_type<64>(x, nb, s); break;
    case 96: pa_type<96>(x, nb, s); break;
    case 128: pa_type<128>(x, nb, s); break;
    default: pa_type<256>(x, nb, s); break;
    }
    a.ntok = ntok;
    if (part) {
        if (by_group) k_cattn_merge_wide<CAttnPaged><<<(unsigned)joins, 256, 0, s>>>(a, p.parts, part);
        else k_cattn_merge<CAttnPaged><<<(unsigned)joins, 256, 0, s>>>(a, p.parts, part);
    }
    return lg_check_launch(who);
}
