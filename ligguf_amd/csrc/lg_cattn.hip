/* lg_cattn.hip -- attention of many rows over the caches that callers keep:
 * fp16 or 4 bits, causal, with a sliding window and first positions that stay
 * visible. */
#include <float.h>
#include <math.h>

#include <algorithm>

#include "lg_kv.h"

struct CAttn {
    const float* q;
    float* out;
    const int* pos;
    int64_t qs, os;
    int rows, ntok, n_heads, nrep, window, sinks, max_pos;
    float scale2;   /* log2(e) / sqrt(head_dim): scores in units of a power of two */
    LgKv c;
};

__device__ __forceinline__ bool ca_sees(const CAttn& a, int p, int key)
{
    return key <= p && (a.window <= 0 || key > p - a.window || key < a.sinks);
}

typedef float lg_f2 __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));

/* fp32 x0, x1 as elements i, i + 1 of two fp16 parts: hi = fp16(x), lo =
 * fp16(x - hi); the products of both with fp16 values are exact in fp32 */
__device__ __forceinline__ void ca_split2(float x0, float x1, v8h& hi, v8h& lo, int i)
{
    const lg_h2 x = __builtin_convertvector(((lg_f2){x0, x1}), lg_h2);
    const lg_h2 y = __builtin_convertvector(((lg_f2){x0 - (float)x[0], x1 - (float)x[1]}), lg_h2);
    hi[i] = x[0];
    hi[i + 1] = x[1];
    lo[i] = y[0];
    lo[i + 1] = y[1];
}

/* A query's values x0, x1, times 2^(14 - ex), in two parts that have x's sign
 * and are 0 only if x is: both products with an infinity are then the one that
 * x's is (NaN where x is 0), and so is their sum.  hi is rounded towards 0, so
 * that lo has its sign, 22 bits in all; a part that would be 0 takes the least
 * fp16, at most 2^-37 of the row's largest value. */
__device__ __forceinline__ void ca_query2(float x0, float x1, int ex, v8h& hi, v8h& lo, int i)
{
    typedef uint16_t u2 __attribute__((ext_vector_type(2)));
    const float y0 = ldexpf(x0, 14 - ex), y1 = ldexpf(x1, 14 - ex);
    const u2 least = {(uint16_t)(x0 != 0.0f), (uint16_t)(x1 != 0.0f)}, sign = {0x8000, 0x8000};
    const lg_h2 h = __builtin_bit_cast(lg_h2, __builtin_amdgcn_cvt_pkrtz(y0, y1));
    const lg_h2 l = __builtin_convertvector(((lg_f2){y0 - (float)h[0], y1 - (float)h[1]}), lg_h2);
    const u2 hb = __builtin_bit_cast(u2, h), lb = __builtin_bit_cast(u2, l);
    const lg_h2 a = __builtin_bit_cast(lg_h2, __builtin_elementwise_max(hb & ~sign, least) | (hb & sign));
    const lg_h2 b = __builtin_bit_cast(lg_h2, __builtin_elementwise_max(lb & ~sign, least) | (hb & sign));
    hi[i] = a[0];
    hi[i + 1] = a[1];
    lo[i] = b[0];
    lo[i + 1] = b[1];
}

/* the wave's LDS writes before its other lanes' reads */
__device__ __forceinline__ void ca_wave_sync()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

/* four halves each of 4 x 16 (rows x columns) out of LDS, transposed: of 16
 * lanes, lane i points at row i / 4, columns 4 (i % 4) .. +3 and receives
 * column i of the four rows */
__device__ __forceinline__ v4s ca_tr16(const _Float16* p)
{
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s*)p);
}

/* the scale of scores whose queries are held times 2^(14 - ex): not 0, so that
 * it times -infinity is no NaN (queries of 1e-40: the scores differ by nothing) */
__device__ __forceinline__ float ca_scale(float scale2, int ex) { return fmaxf(ldexpf(scale2, ex - 14), FLT_MIN); }

/* A column's running maximum.  Its weights are 2^(s sc + cc), cc = 14 - m sc as
 * rounded: the rounding is the same for all of them, and goes along when the
 * sums are rescaled (by the difference of two cc) or joined (-cc).  Where that
 * is so far from 0 that its rounding would matter (scores of 10^6, or no key
 * seen yet), the maximum is taken off the scores first and cc is 14; a wave
 * with such a column raises at every tile.  cc belongs to m from the start: of
 * small queries -2^40 sc is near, and a first tile without a key of the column
 * would else raise from 14 by a factor that is infinite. */
struct CaMax {
    float sc, m, cc;
    bool any_far;                         /* of the wave */

    __device__ __forceinline__ explicit CaMax(float scale) : sc(scale), m(-0x1p40f), any_far(true)   /* (-2^40: below any score) */
    {
        const float c = __builtin_fmaf(-m, sc, 14.0f);
        cc = far(c) ? 14.0f : c;
    }
    __device__ __forceinline__ bool far(float c) const { return fabsf(c) > 0x1p22f; }
    __device__ __forceinline__ bool due(float mn) const { return __builtin_amdgcn_ballot_w64(mn > m) || any_far; }
    /* maximum mn of a tile's scores; returns what the sums so far are to be
     * multiplied by, and in *off what to take off the tile's scores */
    __device__ __forceinline__ float raise(float mn, float* off)
    {
        mn = fmaxf(mn, m);
        const float c = __builtin_fmaf(-mn, sc, 14.0f), cn = far(c) ? 14.0f : c;
        const bool was = far(__builtin_fmaf(-m, sc, 14.0f));
        const float al = __builtin_amdgcn_exp2f(far(c) || was ? (m - mn) * sc : cn - cc);
        m = mn;
        cc = cn;
        any_far = __builtin_amdgcn_ballot_w64(far(c)) != 0;
        *off = far(c) ? mn : 0.0f;
        return al;
    }
    /* the power of two that weights are multiples of, for sums to be joined; l: the sum of weights.  (Of far columns
     * as rounded: off by up to 2^-24 of itself, less than scores of that size are by their 22 bits.) */
    __device__ __forceinline__ float unit(float l) const
    {
        const float c = __builtin_fmaf(-m, sc, 14.0f);
        return l == 0.0f ? -INFINITY : -c;
    }
};

/* halves that are infinite or NaN to 0; whether there were any */
__device__ __forceinline__ bool ca_drop_bad(v4u& w)
{
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t b = ((w[i] & 0x7FFF7FFFu) + 0x04000400u) & 0x80008000u;   /* exponent 31: bit 15 of the half */
        w[i] &= ~((b >> 15) * 0xFFFFu);
        any |= b;
    }
    return any != 0;
}

/* a mask of lanes as one of their rows l % 16 */
__device__ __forceinline__ uint64_t ca_row16(uint64_t b) { return (b | b >> 16 | b >> 32 | b >> 48) & 0xFFFF; }

/* four values of a cached value row, from dim d (a multiple of 4) on */
template <bool KV4>
__device__ __forceinline__ v4f ca_values(const LgKv& c, const uint8_t* v, int g, int key, int d)
{
    lg_h2 x[4];
    if constexpr (!KV4) *(uint2*)x = *(const uint2*)(v + lg_kv16_at(c, g, key) + 2 * d);
    else {
        lg_kv4_values(*(const uint32_t*)(v + lg_kv4_codes(c, g, key) + d / 8 * 4),
                      *(const uint32_t*)(v + lg_kv4_dm(c, g, key) + d / 32 * 4), x);
        if (d & 4) {
            x[0] = x[2];
            x[1] = x[3];
        }
    }
    return (v4f){(float)x[0][0], (float)x[0][1], (float)x[1][0], (float)x[1][1]};
}

/* o plus those of x that are infinite or NaN */
__device__ __forceinline__ float ca_add_bad(float o, float x) { return fabsf(x) <= FLT_MAX ? o : o + x; }

/* The keys that rows of positions pmin .. pmax may see, in tiles of KT: those
 * that hold sinks, then those of the windows (one run where they meet). */
struct CaTiles {
    int first, lo, n;
    __device__ __forceinline__ CaTiles(const CAttn& a, int pmin, int pmax, int kt)
    {
        lo = a.window > 0 ? max(0, pmin - a.window + 1) / kt : 0;
        first = min((min(a.sinks, pmax + 1) + kt - 1) / kt, lo);
        n = pmax < 0 ? 0 : first + pmax / kt - lo + 1;
    }
    /* split sp's run of them: `chunk` tiles or, where that leaves some, equal parts */
    __device__ __forceinline__ void chunk(int sp, int nsplit, int chunk, int* t0, int* t1) const
    {
        const int64_t len = max(chunk, (n + nsplit - 1) / nsplit);
        *t0 = (int)min(sp * len, (int64_t)n);
        *t1 = (int)min(*t0 + len, (int64_t)n);
    }
    __device__ __forceinline__ int at(int i) const { return i < first ? i : lo + i - first; }
};

constexpr int CA_PARTS = 512;   /* at most */

/* Partials of a split call: [split][row][head] sums, then (maximum, sum of
 * weights) of each; a part without keys has weight 0 and no sums. */
__device__ __forceinline__ float2& ca_part_ml(const CAttn& a, int nsplit, float* part, int hd, int64_t at)
{
    return ((float2*)(part + (int64_t)nsplit * a.rows * a.n_heads * hd))[at];
}

/* One token's query heads of a key head, or a few tokens' (up to 16 columns):
 * split over the keys, every wave with tiles of KT keys of its own.
 *   S^T[key][col] = K Q^T      A = K rows as they lie, B = Q^T, 32 dims a step
 *   O^T[d][col]  += V^T P^T    A = V^T, B = P^T, 32 keys a step
 * on 16 x 16 x 32 fp16 MFMA: lane l feeds row / column l % 16, k = 8 (l / 16)
 * .. +7, and register i of a result is row 4 (l / 16) + i of column l % 16.  So
 * a lane's eight scores of two 16-key results are its eight k of the second
 * product -- keys 4c .. 4c+3 and 16 + 4c .. of quarter c -- and P never leaves
 * its registers.  V's rows go through the wave's own part of LDS and come back
 * transposed (ds_read_b64_tr_b16); K needs no LDS at all, its dims being
 * summed in whatever order both operands agree on: in 4 bits a quarter takes a
 * run of HD / 4 dims, one load for all steps and one (d, m) pair.
 *
 * q is held times a power of two that brings the row's largest value to
 * 2^13 .. 2^14 and p times 2^14, each in two fp16 parts, so 22 bits of both
 * survive whatever their size.  The loads of one tile run while the last one
 * computes.  fp16 is bound by the cache's bytes (32 heads of 128, 8 key heads:
 * 64 sequences of 2000 rows 100 us, 5.2 TB/s; 24 ragged ones of up to 12000
 * 131 to 143 us on several cards, 4.3 to 4.6 TB/s); 4 bits by bytes and by VALU work, 62 % of the cycles (64 of
 * 2000 rows 36 us, 4.5 TB/s; 40 ragged ones 104 us, 3.9 TB/s), most of it the 13
 * operations for eight values: of 16 columns four are used. */
template <int HD, bool KV4>
struct CaDec {
    static constexpr int KT = KV4 && HD <= 128 ? 64 : 32, NU = KT / 16, NB = KT / 32;
    static constexpr int NS = (HD + 31) / 32, NT = HD / 16;
    static constexpr bool RUN = KV4 && HD != 96;               /* a quarter's dims are one run */
    static constexpr int ND = !KV4 ? 1 : HD == 96 ? NS : HD > 128 ? HD / 128 : 1;   /* (d, m) pairs of a lane's key */
    static constexpr int VST = HD + 16;                        /* halves per V row in LDS: 8 banks on */
    static constexpr int OST = HD + 4;                         /* floats per column in LDS */
    static constexpr int WAVE = 32 * VST * 2 > 16 * OST * 4 ? 32 * VST * 2 : 16 * OST * 4;
    /* first dim of lane quarter c at step s */
    static __device__ __forceinline__ int dim(int s, int c) { return RUN ? c * (HD / 4) + 8 * s : 32 * s + 8 * c; }
};

/* what a lane holds of 16 NU key (or value) rows */
template <int HD, bool KV4>
struct CaRows {
    using C = CaDec<HD, KV4>;
    v4u h[KV4 ? 1 : C::NU][KV4 ? 1 : C::NS];
    uint32_t w[KV4 ? C::NU : 1][KV4 ? C::NS : 1], dm[KV4 ? C::NU : 1][C::ND];

    /* at: the lane's rows of the tile at kb.  The tile's address is the wave's, a lane's part of it fits 32 bits (rows of
     * at most 2^25 bytes). */
    __device__ __forceinline__ void load(const CAttn& a, const uint8_t* base, int g, int kb, const uint32_t at[C::NU],
                                         int c)
    {
        const uint8_t* const p0 = base + (KV4 ? lg_kv4_codes(a.c, g, kb) : lg_kv16_at(a.c, g, kb));
        const uint8_t* const q0 = base + (KV4 ? lg_kv4_dm(a.c, g, kb) : 0);
#pragma unroll
        for (int u = 0; u < C::NU; u++) {
            if constexpr (KV4) {
                const uint8_t* const p = p0 + at[u] * (uint32_t)(HD / 2) + (C::RUN ? c * (HD / 8) : 4 * c);
#pragma unroll
                for (int s = 0; s < C::NS; s++) w[u][s] = *(const uint32_t*)(p + s * (C::RUN ? 4 : 16));
                const uint8_t* const q = q0 + at[u] * (uint32_t)(HD / 8) +
                                         (HD == 96 ? 0 : HD == 64 ? c / 2 * 4 : c * C::ND * 4);
#pragma unroll
                for (int i = 0; i < C::ND; i++) dm[u][i] = *(const uint32_t*)(q + 4 * i);
            } else {
                const uint8_t* const p = p0 + at[u] * (uint32_t)(a.c.n_kv * HD * 2) + 16 * c;
#pragma unroll
                for (int s = 0; s < C::NS; s++)
                    h[u][s] = HD % 32 == 0 || 32 * s + 8 * c < HD ? *(const v4u*)(p + 64 * s) : (v4u){};
            }
        }
    }
    __device__ __forceinline__ v4u get(int u, int s) const
    {
        if constexpr (KV4) {
            lg_h2 x[4];
            lg_kv4_values(w[u][s], dm[u][HD == 96 ? s : HD == 64 ? 0 : s / 4], x);
            return (v4u){__builtin_bit_cast(uint32_t, x[0]), __builtin_bit_cast(uint32_t, x[1]),
                         __builtin_bit_cast(uint32_t, x[2]), __builtin_bit_cast(uint32_t, x[3])};
        } else
            return h[u][s];
    }
};

template <int HD, bool KV4, int NW>
__global__ __launch_bounds__(64 * NW, (HD <= 128 ? 2 : 1)) void k_cattn_dec(CAttn a, int nsplit, int chunk,
                                                                           float* __restrict__ part)
{
    using C = CaDec<HD, KV4>;
    constexpr int KT = C::KT, NU = C::NU, NB = C::NB, NS = C::NS, NT = C::NT;
    __shared__ __attribute__((aligned(16))) uint8_t s_raw[NW * C::WAVE];
    __shared__ float s_ml[NW][16][2];
    const int n_kv = a.c.n_kv, g = blockIdx.x % n_kv, sp = blockIdx.x / n_kv % nsplit, seq = blockIdx.x / n_kv / nsplit;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, c = lane >> 4;
    const int tok = col / a.nrep, ncol = a.ntok * a.nrep;
    const int64_t row = (int64_t)seq * a.ntok + min(tok, a.ntok - 1);
    const int head = g * a.nrep + col % a.nrep;
    int p = a.pos[row];
    /* the column's query, on its way before the first keys: loads come back in order */
    v4f x[2 * NS];
    {
        const float* const q = a.q + row * a.qs + (size_t)head * HD;
#pragma unroll
        for (int s = 0; s < NS; s++) {
            const int d = C::dim(s, c);
            const bool in = col < ncol && d < HD;
            x[2 * s] = in ? *(const v4f*)(q + d) : (v4f){};
            x[2 * s + 1] = in ? *(const v4f*)(q + d + 4) : (v4f){};
        }
    }
    /* Without a window a lone workgroup's waves know their first tiles before
     * the positions, and read them along (512 fp16 keys 10.7 -> 10.4 us, of 32
     * sequences 15.0 -> 14.3); not where a wave has but one (256 keys 7.3 -> 8.4,
     * the last being read twice) or in 4 bits (8.5 -> 9.1). */
    const uint8_t* const kc = a.c.k + (size_t)seq * a.c.seq;
    const uint8_t* const vc = a.c.v + (size_t)seq * a.c.seq;
    CaRows<HD, KV4> K, V;
    uint32_t at[NU];
    const int early = NW == 8 && !KV4 && a.window <= 0 && a.max_pos >= NW * KT ? wave * KT : -1;
    if (early >= 0) {
#pragma unroll
        for (int u = 0; u < NU; u++) at[u] = min(16 * u + col, a.max_pos - early);
        K.load(a, kc, g, early, at, c);
        V.load(a, vc, g, early, at, c);
    }
    if (col >= ncol || p > a.max_pos) p = -1;
    int pmin = p < 0 ? INT32_MAX : p, pmax = p;
#pragma unroll
    for (int o = 1; o < 16; o *= 2) {
        pmin = min(pmin, __shfl_xor(pmin, o));
        pmax = max(pmax, __shfl_xor(pmax, o));
    }
    pmin = __builtin_amdgcn_readfirstlane(pmin);
    pmax = __builtin_amdgcn_readfirstlane(pmax);

    const CaTiles tiles(a, pmin, pmax, KT);
    int t0, t1;
    tiles.chunk(sp, nsplit, chunk, &t0, &t1);
    if (part && t0 >= t1) {   /* (workgroup-uniform) */
        if ((int)threadIdx.x < ncol)
            ca_part_ml(a, nsplit, part, HD,
                       ((int64_t)sp * a.rows + (int64_t)seq * a.ntok + threadIdx.x / a.nrep) * a.n_heads + g * a.nrep +
                           threadIdx.x % a.nrep) = make_float2(-INFINITY, 0.0f);
        return;
    }
    v4f o[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) o[t] = (v4f){};
    float l = 0.0f, unit = -INFINITY;   /* sum of weights (this lane's keys) */
    if (t0 + wave < t1) {
        _Float16* const sV = (_Float16*)(s_raw + wave * C::WAVE);
        /* keys that some column does not see (wave-uniform) */
        auto partly = [&](int kb) {
            return kb + KT - 1 > pmin || (a.window > 0 && kb <= pmax - a.window && kb + KT > a.sinks);
        };
        /* the lane's rows of the tile at kb.  Those that none of the columns at
         * one position sees give way to one that they do, so that whatever
         * they hold takes no part; where positions differ, see `bad` below. */
        auto rows_of = [&](int kb) __attribute__((always_inline)) {
#pragma unroll
            for (int u = 0; u < NU; u++) at[u] = min(16 * u + col, a.max_pos - kb);
            if (pmin == pmax && partly(kb)) {
                const int some = kb < a.sinks || a.window <= 0 ? 0 : max(0, pmax - a.window + 1 - kb);
#pragma unroll
                for (int u = 0; u < NU; u++)
                    if (!ca_sees(a, pmax, kb + 16 * u + col)) at[u] = some;
            }
        };
        int it = t0 + wave, kb = tiles.at(it) * KT;
        if (kb != early || (pmin == pmax && partly(kb))) {
            rows_of(kb);
            K.load(a, kc, g, kb, at, c);
            V.load(a, vc, g, kb, at, c);
        }
        /* (all of these loads ahead of what waits for the query: 0.3 to 0.8 us) */
        __builtin_amdgcn_sched_barrier(0);
        /* the query in two parts, while the first keys come */
        v8h qh[NS], ql[NS];
        float big = 0.0f;
#pragma unroll
        for (int i = 0; i < 2 * NS; i++)
            big = fmaxf(fmaxf(big, fmaxf(fabsf(x[i][0]), fabsf(x[i][1]))), fmaxf(fabsf(x[i][2]), fabsf(x[i][3])));
        big = fmaxf(big, lg_partner<4>(big));
        big = fmaxf(big, lg_partner<5>(big));
        const int ex = __builtin_amdgcn_frexp_expf(big);   /* big < 2^ex */
        CaMax mx(ca_scale(a.scale2, ex));
#pragma unroll
        for (int j = 0; j < NS; j++)
#pragma unroll
            for (int e = 0; e < 8; e += 2)
                ca_query2(x[2 * j + e / 4][e % 4], x[2 * j + e / 4][e % 4 + 1], ex, qh[j], ql[j], e);
        for (; it < t1; it += NW) {
            v4f s[NU];
#pragma unroll
            for (int u = 0; u < NU; u++) {
                s[u] = (v4f){};
#pragma unroll
                for (int j = 0; j < NS; j++) {
                    const v8h k = __builtin_bit_cast(v8h, K.get(u, j));
                    s[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qh[j], s[u], 0, 0, 0);
                    s[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, ql[j], s[u], 0, 0, 0);
                }
            }
            const int kn = it + NW < t1 ? tiles.at(it + NW) * KT : -1;
            if (kn >= 0) {
                rows_of(kn);
                K.load(a, kc, g, kn, at, c);
            }
            const bool part_seen = partly(kb);
            if (part_seen) {
#pragma unroll
                for (int u = 0; u < NU; u++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (!ca_sees(a, p, kb + 16 * u + 4 * c + i)) s[u][i] = -INFINITY;
            }
            float mn = s[0][0];
#pragma unroll
            for (int u = 0; u < NU; u++)
#pragma unroll
                for (int i = 0; i < 4; i++) mn = fmaxf(mn, s[u][i]);
            if (mx.due(mn)) {
                mn = fmaxf(mn, lg_partner<4>(mn));
                mn = fmaxf(mn, lg_partner<5>(mn));
                float off;
                const float al = mx.raise(mn, &off);
                l *= al;
#pragma unroll
                for (int t = 0; t < NT; t++) o[t] *= al;
#pragma unroll
                for (int u = 0; u < NU; u++) s[u] -= off;
            }
            uint64_t bad = 0;   /* keys of the tile */
#pragma unroll
            for (int b = 0; b < NB; b++) {
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int j = 0; j < NS; j++) {
                        v4u y = V.get(2 * b + u, j);
                        if (part_seen && pmin != pmax)
                            bad |= ca_row16(__builtin_amdgcn_ballot_w64(ca_drop_bad(y))) << (32 * b + 16 * u);
                        if (HD % 32 == 0 || C::dim(j, c) < HD) *(v4u*)(sV + (16 * u + col) * C::VST + C::dim(j, c)) = y;
                    }
                if (b == NB - 1 && kn >= 0) V.load(a, vc, g, kn, at, c);
                v8h ph, pl;
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    float w[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) w[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * b + u][i], mx.sc, mx.cc));
                    l += (w[0] + w[1]) + (w[2] + w[3]);
                    ca_split2(w[0], w[1], ph, pl, 4 * u);
                    ca_split2(w[2], w[3], ph, pl, 4 * u + 2);
                }
                ca_wave_sync();
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    const _Float16* const v = sV + (4 * c + col / 4) * C::VST + 16 * t + 4 * (col % 4);
                    const v4s x0 = ca_tr16(v), x1 = ca_tr16(v + 16 * C::VST);
                    const v8h y = __builtin_bit_cast(v8h, __builtin_shufflevector(x0, x1, 0, 1, 2, 3, 4, 5, 6, 7));
                    o[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(y, ph, o[t], 0, 0, 0);
                    o[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(y, pl, o[t], 0, 0, 0);
                }
                ca_wave_sync();   /* (the reads before the next block's writes) */
            }
            /* infinities and NaN of keys that only some columns see: added by
             * itself to those that do, whatever the (positive) weight */
            for (; bad; bad &= bad - 1) {
                const int key = kb + __builtin_ctzll(bad);
                if (ca_sees(a, p, key))
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        const v4f y = ca_values<KV4>(a.c, vc, g, key, 16 * t + 4 * c);
#pragma unroll
                        for (int i = 0; i < 4; i++) o[t][i] = ca_add_bad(o[t][i], y[i]);
                    }
            }
            kb = kn;
        }
        l += lg_partner<4>(l);
        l += lg_partner<5>(l);
        unit = mx.unit(l);
    }
    /* the waves' parts of each column together, by way of LDS */
    float* const sO = (float*)(s_raw + wave * C::WAVE);
#pragma unroll
    for (int t = 0; t < NT; t++) *(v4f*)(sO + col * C::OST + 16 * t + 4 * c) = o[t];
    if (c == 0) {
        s_ml[wave][col][0] = unit;
        s_ml[wave][col][1] = l;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < ncol * (HD / 4); i += 64 * NW) {
        const int k = i / (HD / 4), d = i % (HD / 4) * 4;
        float M = s_ml[0][k][0];
#pragma unroll
        for (int w = 1; w < NW; w++) M = fmaxf(M, s_ml[w][k][0]);
        v4f y = {};
        float L = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; w++) {
            /* (a wave without keys has l = 0 and all zeros) */
            const float lw = s_ml[w][k][1], f = lw == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(s_ml[w][k][0] - M);
            const v4f x = *(const v4f*)((const float*)(s_raw + w * C::WAVE) + k * C::OST + d);
            L = __builtin_fmaf(lw, f, L);
#pragma unroll
            for (int e = 0; e < 4; e++) y[e] = __builtin_fmaf(x[e], f, y[e]);
        }
        const int64_t r = (int64_t)seq * a.ntok + k / a.nrep;
        const int hh = g * a.nrep + k % a.nrep;
        if (part) {
            const int64_t at = ((int64_t)sp * a.rows + r) * a.n_heads + hh;
            *(v4f*)(part + at * HD + d) = y;
            if (d == 0) ca_part_ml(a, nsplit, part, HD, at) = make_float2(M, L);
        } else {
            const float inv = 1.0f / L;   /* (0 times infinity where every visible key is -infinity) */
            const int pk = a.pos[r];
            *(v4f*)(a.out + r * a.os + (size_t)hh * HD + d) = pk < 0 || pk > a.max_pos ? (v4f){} : y * inv;
        }
    }
}

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

/* The parts of a row's head together: sum w_i o_i / sum w_i l_i, w_i = 2^(M_i - M).
 * Of many rows: a thread per four dims. */
__global__ __launch_bounds__(256) void k_cattn_merge(CAttn a, int nsplit, const float* __restrict__ part)
{
    const int hd = a.c.hd, dq = hd / 4;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, n = (int64_t)a.rows * a.n_heads;
    if (i >= n * dq) return;
    const int64_t at = i / dq, row = at / a.n_heads;
    const int d = (int)(i % dq) * 4, head = (int)(at % a.n_heads), p = a.pos[row];
    const float2* const ml = (const float2*)(part + nsplit * n * hd);
    v4f y = {};
    float L = 0.0f;
    if (p >= 0 && p <= a.max_pos) {
        float M = -INFINITY;
        for (int s = 0; s < nsplit; s++) M = fmaxf(M, ml[s * n + at].x);
        for (int s = 0; s < nsplit; s++) {
            const float2 x = ml[s * n + at];
            if (x.y == 0.0f) continue;   /* (no keys, no sums written) */
            const float f = __builtin_amdgcn_exp2f(x.x - M);
            const v4f v = *(const v4f*)(part + (s * n + at) * hd + d);
            L = __builtin_fmaf(x.y, f, L);
#pragma unroll
            for (int e = 0; e < 4; e++) y[e] = __builtin_fmaf(v[e], f, y[e]);
        }
    }
    *(v4f*)(a.out + row * a.os + (size_t)head * hd + d) = p < 0 || p > a.max_pos ? (v4f){} : y * (1.0f / L);
}

/* Many parts or few rows: a workgroup per row's head, the weights by one wave,
 * the sums by groups of hd / 4 threads -- a thread that walks over the parts
 * waits for one load after the other (64 parts of 32 heads: 34 us) */
__global__ __launch_bounds__(256) void k_cattn_merge_wide(CAttn a, int nsplit, const float* __restrict__ part)
{
    __shared__ float s_f[CA_PARTS], s_l;
    __shared__ v4f s_y[256];
    const int hd = a.c.hd, dq = hd / 4, grp = threadIdx.x / dq, ng = 256 / dq, d = threadIdx.x % dq * 4;
    const int64_t at = blockIdx.x, n = (int64_t)a.rows * a.n_heads, row = at / a.n_heads;
    const int head = (int)(at % a.n_heads), p = a.pos[row];
    const float2* const ml = (const float2*)(part + nsplit * n * hd);
    if (threadIdx.x < 64) {
        float2 x[CA_PARTS / 64];
        float M = -INFINITY, L = 0.0f;
#pragma unroll
        for (int k = 0; k < CA_PARTS / 64; k++) {
            const int s = threadIdx.x + 64 * k;
            x[k] = s < nsplit ? ml[s * n + at] : make_float2(-INFINITY, 0.0f);
            M = fmaxf(M, x[k].x);
        }
        M = lg_group_max<64>(M);
#pragma unroll
        for (int k = 0; k < CA_PARTS / 64; k++) {
            /* -1: no keys, no sums written (0 counts: it may meet an infinity) */
            const float f = x[k].y == 0.0f ? -1.0f : __builtin_amdgcn_exp2f(x[k].x - M);
            s_f[threadIdx.x + 64 * k] = f;
            L = __builtin_fmaf(x[k].y, f, L);
        }
        L = lg_group_sum<64>(L);
        if (threadIdx.x == 0) s_l = L;
    }
    __syncthreads();
    v4f y = {};
    if (grp < ng) {
#pragma unroll 4
        for (int s = grp; s < nsplit; s += ng) {
            const float f = s_f[s];
            const v4f v = f == -1.0f ? (v4f){} : *(const v4f*)(part + (s * n + at) * hd + d);
#pragma unroll
            for (int e = 0; e < 4; e++) y[e] = __builtin_fmaf(v[e], f, y[e]);
        }
        s_y[threadIdx.x] = y;
    }
    __syncthreads();
    if (grp) return;
    for (int k = 1; k < ng; k++) y += s_y[threadIdx.x + k * dq];
    const float L = s_l;
    *(v4f*)(a.out + row * a.os + (size_t)head * hd + d) = p < 0 || p > a.max_pos ? (v4f){} : y * (1.0f / L);
}

/* How a call is cut, from its sizes alone. */
struct CaPlan {
    bool dec;     /* up to 16 columns a key head */
    int ncb;      /* else: blocks of columns of a sequence's key head */
    bool wide;    /* eight waves a workgroup, else four */
    int nsplit, chunk;   /* parts of the keys, tiles in a part */
    size_t ws;
};

static CaPlan ca_plan(int64_t nseq, int64_t ntok, int n_heads, int n_kv, int hd, int window, int sinks, int max_pos,
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
    return ca_plan(nseq, ntok, n_heads, cache->n_kv_heads, cache->head_dim, window, sinks, max_pos,
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
    const CaPlan p = ca_plan(nseq, ntok, n_heads, a.c.n_kv, hd, window, sinks, max_pos, a.c.type == LG_KV4);
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
        if (by_group) k_cattn_merge_wide<<<(unsigned)joins, 256, 0, s>>>(a, p.nsplit, part);
        else k_cattn_merge<<<(unsigned)joins, 256, 0, s>>>(a, p.nsplit, part);
    }
    return lg_check_launch(who);
}
