/* lg_cattn.h -- attention of many rows over the caches that callers keep, causal,
 * with a sliding window and first positions that stay visible: what contiguous
 * caches (lg_cattn.hip) and pages (lg_pattn.hip) have in common, fp16 or 4 bits. */
#pragma once

#include <float.h>
#include <math.h>

#include <algorithm>

#include "lg_kv.h"

/* units of ntok rows each (a sequence's), one after the other */
struct CAttn {
    static constexpr bool paged = false;
    const float* q;
    float* out;
    const int* pos;
    int64_t qs, os;
    int rows, ntok, n_heads, nrep, window, sinks, max_pos;
    float scale2;   /* log2(e) / sqrt(head_dim): scores in units of a power of two */
    LgKv c;
};

/* The same over pages: a page is a sequence of c (n_ctx rows, a power of two from
 * 16 on).  Unit u has the table's row u * tstep; its keys are those below the
 * group's shared ones (`share`: the unit is a group) or from there on (a
 * sequence of `group`; without prefix all).  Its partials are parts part0 .. of nparts. */
struct CAttnPaged : CAttn {
    static constexpr bool paged = true;
    const int *table, *prefix;
    int64_t tstride;
    int n_pages, shift, tstep, group, share, max_prefix, part0, nparts;

    __device__ __forceinline__ int page_rows() const { return 1 << shift; }
    /* the keys of unit u: [lo, hi) */
    __device__ __forceinline__ void range(int u, int* lo, int* hi) const
    {
        const int n = prefix ? min(max(prefix[share ? u : u / group], 0), max_prefix) : 0;
        *lo = share ? 0 : n;
        *hi = share ? n : INT32_MAX;
    }
    __device__ __forceinline__ bool is_page(int id) const { return (uint32_t)id < (uint32_t)n_pages; }
    /* the table's entry for row `key` of table row t (rows past max_pos, which
     * nothing sees, take its) */
    __device__ __forceinline__ int entry(const int* t, int key) const { return t[min(key, max_pos) >> shift]; }
};

/* What a column at position p sees of the keys [lo, hi): none, bit by bit, are the
 * present tile's groups of 16 rows without a page.  Without branches: as a
 * chain of conditions around the write of -infinity (clang 22, gfx950) the
 * compiler dropped the write of the first score. */
struct CaSeen {
    int lo, hi, wlo, sinks;
    __device__ __forceinline__ CaSeen(const CAttnPaged& a, int p, int klo, int khi)
        : lo(klo), hi(min(p, khi - 1)), wlo(a.window > 0 ? p - a.window + 1 : INT32_MIN), sinks(a.sinks)
    {
    }
    __device__ __forceinline__ bool operator()(int key, int kb, int none) const
    {
        return (key >= lo) & (key <= hi) & ((key >= wlo) | (key < sinks)) & !(none >> ((key - kb) >> 4) & 1);
    }
};

/* A tile's table entries, that of its rows 16 j .. in lane j (mod 8): loaded ahead
 * like any other vector load, in the order of the keys and values, so that
 * nothing waits for them alone. */
struct CaEntries {
    int e;
    __device__ __forceinline__ void load(const CAttnPaged& a, const int* trow, int kb)
    {
        e = a.entry(trow, kb + 16 * (threadIdx.x & 7));
    }
    /* those of the tile's n groups of 16 rows that are no pages, bit by bit */
    __device__ __forceinline__ int none(const CAttnPaged& a, int n) const
    {
        return (int)__builtin_amdgcn_ballot_w64(!a.is_page(e)) & ((1 << n) - 1);
    }
    /* where group j's (the wave's j) page lies in a pool, page 0 in place of none */
    __device__ __forceinline__ size_t at(const CAttnPaged& a, int j) const
    {
        return (uint64_t)(uint32_t)__builtin_amdgcn_readlane(a.is_page(e) ? e : 0, j) * (uint32_t)a.c.seq;
    }
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
 * would else raise from 14 by a factor that is infinite.  With LAG the maximum
 * follows only scores that are 2^LAG times above it: weights are up to 2^(BASE +
 * LAG), which fp16 has to hold, and the sums are rescaled but once or twice. */
template <int BASE_, int LAG>
struct CaMaxOf {
    static constexpr float BASE = (float)BASE_;
    float sc, m, cc;
    bool any_far;                         /* of the wave */

    __device__ __forceinline__ explicit CaMaxOf(float scale = 0.0f) : sc(scale), m(-0x1p40f), any_far(true)   /* (-2^40: below any score) */
    {
        const float c = __builtin_fmaf(-m, sc, BASE);
        cc = far(c) ? BASE : c;
    }
    __device__ __forceinline__ bool far(float c) const { return fabsf(c) > 0x1p22f; }
    __device__ __forceinline__ bool due(float mn) const
    {
        static_assert(LAG == 0, "a maximum that lags goes by over()");
        return __builtin_amdgcn_ballot_w64(mn > m) || any_far;
    }
    /* whether some weights (sum: a lane's, which no one of them exceeds) are too far above the maximum */
    __device__ __forceinline__ bool over(float sum) const
    {
        constexpr float most = (float)(1 << (BASE_ + LAG));
        return __builtin_amdgcn_ballot_w64(sum > most) || any_far;
    }
    /* maximum mn of a tile's scores; returns what the sums so far are to be
     * multiplied by, and in *off what to take off the tile's scores */
    __device__ __forceinline__ float raise(float mn, float* off)
    {
        mn = fmaxf(mn, m);
        const float c = __builtin_fmaf(-mn, sc, BASE), cn = far(c) ? BASE : c;
        const bool was = far(__builtin_fmaf(-m, sc, BASE));
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
        const float c = __builtin_fmaf(-m, sc, BASE);
        return l == 0.0f ? -INFINITY : -c;
    }
};
using CaMax = CaMaxOf<14, 0>;

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

/* the same by the key's row in its page */
template <bool KV4>
__device__ __forceinline__ v4f ca_values(const CAttnPaged& a, const uint8_t* v, const int* t, int g, int key, int d)
{
    const int id = a.entry(t, key);   /* (of a key that is seen: a page) */
    return ca_values<KV4>(a.c, v + (size_t)(a.is_page(id) ? id : 0) * a.c.seq, g, key & (a.page_rows() - 1), d);
}

/* o plus those of x that are infinite or NaN */
__device__ __forceinline__ float ca_add_bad(float o, float x) { return fabsf(x) <= FLT_MAX ? o : o + x; }

/* The keys that rows of positions pmin .. pmax may see, in tiles of KT: those
 * that hold sinks, then those of the windows (one run where they meet). */
struct CaTiles {
    int first, lo, n;
    int s0 = 0;   /* (of keys lo .. hi - 1 alone: their first tile) */
    __device__ __forceinline__ CaTiles(const CAttn& a, int pmin, int pmax, int kt, int klo, int khi)
    {
        const int top = min(pmax, khi - 1);
        s0 = klo / kt;
        lo = a.window > 0 ? max(klo, pmin - a.window + 1) / kt : s0;
        first = min(max((min(a.sinks, top + 1) + kt - 1) / kt - s0, 0), lo - s0);
        n = top < klo ? 0 : max(first + top / kt - lo + 1, first);
    }
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
    __device__ __forceinline__ int at(int i) const { return i < first ? s0 + i : lo + i - first; }
};

__device__ __forceinline__ CaTiles ca_tiles(const CAttn& a, int pmin, int pmax, int kt, int, int)
{
    return CaTiles(a, pmin, pmax, kt);
}
__device__ __forceinline__ CaTiles ca_tiles(const CAttnPaged& a, int pmin, int pmax, int kt, int klo, int khi)
{
    return CaTiles(a, pmin, pmax, kt, klo, khi);
}

/* split sp of a launch as a part, and how many there are */
__device__ __forceinline__ int ca_part(const CAttn&, int sp) { return sp; }
__device__ __forceinline__ int ca_part(const CAttnPaged& a, int sp) { return a.part0 + sp; }
__device__ __forceinline__ int ca_nparts(const CAttn&, int nsplit) { return nsplit; }
__device__ __forceinline__ int ca_nparts(const CAttnPaged& a, int) { return a.nparts; }

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
    /* of pages: rows 16 u .. of the tile are 16 of one page, row c16 the lane's */
    __device__ __forceinline__ void load(const CAttnPaged& a, const uint8_t* base, int g, int kb, const CaEntries& id,
                                         int c16, int c)
    {
#pragma unroll
        for (int u = 0; u < C::NU; u++) {
            const int row = (kb + 16 * u) & (a.page_rows() - 1);
            const uint8_t* const b = base + id.at(a, u);
            if constexpr (KV4) {
                const uint8_t* const p = b + lg_kv4_codes(a.c, g, row) + (c16 * (uint32_t)(HD / 2) + (C::RUN ? c * (HD / 8) : 4 * c));
#pragma unroll
                for (int s = 0; s < C::NS; s++) w[u][s] = *(const uint32_t*)(p + s * (C::RUN ? 4 : 16));
                const uint8_t* const q = b + lg_kv4_dm(a.c, g, row) +
                                         (c16 * (uint32_t)(HD / 8) + (HD == 96 ? 0 : HD == 64 ? c / 2 * 4 : c * C::ND * 4));
#pragma unroll
                for (int i = 0; i < C::ND; i++) dm[u][i] = *(const uint32_t*)(q + 4 * i);
            } else {
                const uint8_t* const p = b + lg_kv16_at(a.c, g, row) + (c16 * (uint32_t)(a.c.n_kv * HD * 2) + 16 * c);
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

template <int HD, bool KV4, int NW, class A>
__device__ __forceinline__ void ca_dec(const A& a, int blk, int nsplit, int chunk, float* __restrict__ part, uint8_t* s_raw,
                                       float (*s_ml)[16][2])
{
    using C = CaDec<HD, KV4>;
    constexpr int KT = C::KT, NU = C::NU, NB = C::NB, NS = C::NS, NT = C::NT;
    const int n_kv = a.c.n_kv, g = blk % n_kv, sp = blk / n_kv % nsplit, seq = blk / n_kv / nsplit;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, c = lane >> 4;
    const int tok = col / a.nrep, ncol = a.ntok * a.nrep;
    const int64_t row = (int64_t)seq * a.ntok + min(tok, a.ntok - 1);
    const int head = g * a.nrep + col % a.nrep;
    int klo = 0, khi = INT32_MAX;
    if constexpr (A::paged) a.range(seq, &klo, &khi);
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
    const uint8_t* const kc = a.c.k + (A::paged ? 0 : (size_t)seq * a.c.seq);
    const uint8_t* const vc = a.c.v + (A::paged ? 0 : (size_t)seq * a.c.seq);
    CaRows<HD, KV4> K, V;
    uint32_t at[NU];
    const int early = !A::paged && NW == 8 && !KV4 && a.window <= 0 && a.max_pos >= NW * KT ? wave * KT : -1;
    if constexpr (!A::paged)
        if (early >= 0) {
#pragma unroll
            for (int u = 0; u < NU; u++) at[u] = min(16 * u + col, a.max_pos - early);
            K.load(a, kc, g, early, at, c);
            V.load(a, vc, g, early, at, c);
        }
    /* Of pages, likewise: the table's entries and their rows, while the positions
     * come.  (Which tile is the first is known: splits are of `chunk` tiles, unless
     * the launch was cut for fewer keys; then that is not this wave's, and is read again.) */
    CaEntries id, id1, id2;   /* of the present tile, the next and the one after */
    const int* trow = nullptr;
    int ahead = -1;
    if constexpr (A::paged) {
        trow = a.table + (int64_t)seq * a.tstep * a.tstride;
        if (a.window <= 0) {
            ahead = (klo / KT + sp * chunk + wave) * KT;
            if (ahead > a.max_pos) ahead = -1;
        }
        if (ahead >= 0) {
            id.load(a, trow, ahead);
            id1.load(a, trow, ahead + NW * KT);
            K.load(a, kc, g, ahead, id, col, c);
            V.load(a, vc, g, ahead, id, col, c);
        }
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

    const CaTiles tiles = ca_tiles(a, pmin, pmax, KT, klo, khi);
    int t0, t1;
    tiles.chunk(sp, nsplit, chunk, &t0, &t1);
    if (part && t0 >= t1) {   /* (workgroup-uniform) */
        if ((int)threadIdx.x < ncol)
            ca_part_ml(a, ca_nparts(a, nsplit), part, HD,
                       ((int64_t)ca_part(a, sp) * a.rows + (int64_t)seq * a.ntok + threadIdx.x / a.nrep) * a.n_heads +
                           g * a.nrep + threadIdx.x % a.nrep) = make_float2(-INFINITY, 0.0f);
        return;
    }
    v4f o[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) o[t] = (v4f){};
    float l = 0.0f, unit = -INFINITY;   /* sum of weights (this lane's keys) */
    if (t0 + wave < t1) {
        _Float16* const sV = (_Float16*)(s_raw + wave * C::WAVE);
        int none = 0;   /* rows 16 u .. of the present tile have no page: bit u */
        auto ids_of = [&](int i, CaEntries& to) __attribute__((always_inline)) {
            if constexpr (A::paged)
                if (i < t1) to.load(a, trow, tiles.at(i) * KT);
        };
        /* keys that some column does not see (wave-uniform) */
        auto partly = [&](int kb) {
            if constexpr (A::paged)
                if (kb + KT > khi || kb < klo || none) return true;
            return kb + KT - 1 > pmin || (a.window > 0 && kb <= pmax - a.window && kb + KT > a.sinks);
        };
        auto sees = [&](int kb, int key) __attribute__((always_inline)) {
            if constexpr (A::paged) return CaSeen(a, p, klo, khi)(key, kb, none);
            else return ca_sees(a, p, key);
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
        if constexpr (A::paged) {
            if (kb != ahead) {
                ids_of(it, id);
                ids_of(it + NW, id1);
                K.load(a, kc, g, kb, id, col, c);
                V.load(a, vc, g, kb, id, col, c);
            }
        } else if (kb != early || (pmin == pmax && partly(kb))) {
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
            if constexpr (A::paged) {
                ids_of(it + 2 * NW, id2);
                if (kn >= 0) K.load(a, kc, g, kn, id1, col, c);
                none = id.none(a, NU);
            } else if (kn >= 0) {
                rows_of(kn);
                K.load(a, kc, g, kn, at, c);
            }
            const bool part_seen = partly(kb);
            if (part_seen) {
#pragma unroll
                for (int u = 0; u < NU; u++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        if constexpr (A::paged) s[u][i] = sees(kb, kb + 16 * u + 4 * c + i) ? s[u][i] : -INFINITY;
                        else if (!sees(kb, kb + 16 * u + 4 * c + i)) s[u][i] = -INFINITY;
                    }
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
                        if (part_seen && (A::paged || pmin != pmax))
                            bad |= ca_row16(__builtin_amdgcn_ballot_w64(ca_drop_bad(y))) << (32 * b + 16 * u);
                        if (HD % 32 == 0 || C::dim(j, c) < HD) *(v4u*)(sV + (16 * u + col) * C::VST + C::dim(j, c)) = y;
                    }
                if (b == NB - 1 && kn >= 0) {
                    if constexpr (A::paged) V.load(a, vc, g, kn, id1, col, c);
                    else V.load(a, vc, g, kn, at, c);
                }
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
                if (sees(kb, key))
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        v4f y;
                        if constexpr (A::paged) y = ca_values<KV4>(a, vc, trow, g, key, 16 * t + 4 * c);
                        else y = ca_values<KV4>(a.c, vc, g, key, 16 * t + 4 * c);
#pragma unroll
                        for (int i = 0; i < 4; i++) o[t][i] = ca_add_bad(o[t][i], y[i]);
                    }
            }
            kb = kn;
            if constexpr (A::paged) {
                id = id1;
                id1 = id2;
            }
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
            const int64_t at = ((int64_t)ca_part(a, sp) * a.rows + r) * a.n_heads + hh;
            *(v4f*)(part + at * HD + d) = y;
            if (d == 0) ca_part_ml(a, ca_nparts(a, nsplit), part, HD, at) = make_float2(M, L);
        } else {
            const float inv = 1.0f / L;   /* (0 times infinity where every visible key is -infinity) */
            const int pk = a.pos[r];
            *(v4f*)(a.out + r * a.os + (size_t)hh * HD + d) = pk < 0 || pk > a.max_pos || (A::paged && L == 0.0f) ? (v4f){} : y * inv;
        }
    }
}

template <int HD, bool KV4, int NW>
__global__ __launch_bounds__(64 * NW, (HD <= 128 ? 2 : 1)) void k_cattn_dec(CAttn a, int nsplit, int chunk,
                                                                           float* __restrict__ part)
{
    __shared__ __attribute__((aligned(16))) uint8_t s_raw[NW * CaDec<HD, KV4>::WAVE];
    __shared__ float s_ml[NW][16][2];
    ca_dec<HD, KV4, NW>(a, blockIdx.x, nsplit, chunk, part, s_raw, s_ml);
}

/* The parts of a row's head together: sum w_i o_i / sum w_i l_i, w_i = 2^(M_i - M).
 * Of many rows: a thread per four dims. */
template <class A>
__global__ __launch_bounds__(256) void k_cattn_merge(A a, int nsplit, const float* __restrict__ part)
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
    *(v4f*)(a.out + row * a.os + (size_t)head * hd + d) = p < 0 || p > a.max_pos || (A::paged && L == 0.0f) ? (v4f){} : y * (1.0f / L);
}

/* Many parts or few rows: a workgroup per row's head, the weights by one wave,
 * the sums by groups of hd / 4 threads -- a thread that walks over the parts
 * waits for one load after the other (64 parts of 32 heads: 34 us) */
template <class A>
__global__ __launch_bounds__(256) void k_cattn_merge_wide(A a, int nsplit, const float* __restrict__ part)
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
    *(v4f*)(a.out + row * a.os + (size_t)head * hd + d) = p < 0 || p > a.max_pos || (A::paged && L == 0.0f) ? (v4f){} : y * (1.0f / L);
}

/* How a call is cut, from its sizes alone. */
struct CaPlan {
    bool dec;     /* up to 16 columns a key head */
    int ncb;      /* else: blocks of columns of a sequence's key head */
    bool wide;    /* eight waves a workgroup, else four */
    int nsplit, chunk;   /* parts of the keys, tiles in a part */
    size_t ws;
};
CaPlan lg_ca_plan(int64_t nseq, int64_t ntok, int n_heads, int n_kv, int hd, int window, int sinks, int max_pos, bool kv4);
