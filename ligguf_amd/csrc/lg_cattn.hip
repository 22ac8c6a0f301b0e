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

typedef float v4f __attribute__((ext_vector_type(4)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));

/* fp32 x0, x1 as elements i, i + 1 of two fp16 parts: hi = fp16(x), lo =
 * fp16(x - hi); the products of both with fp16 values are exact in fp32 */
__device__ __forceinline__ void ca_split2(float x0, float x1, v8h& hi, v8h& lo, int i)
{
    const lg_h2 x = {(_Float16)x0, (_Float16)x1};
    hi[i] = x[0];
    hi[i + 1] = x[1];
    lo[i] = (_Float16)(x0 - (float)x[0]);
    lo[i + 1] = (_Float16)(x1 - (float)x[1]);
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

/* one value of a cached value row */
__device__ __forceinline__ float ca_value(const LgKv& c, const uint8_t* v, int g, int key, int d)
{
    if (c.type == LG_F16) return lg_h2f(*(const uint16_t*)(v + lg_kv16_at(c, g, key) + 2 * d));
    lg_h2 x[4];
    lg_kv4_values(*(const uint32_t*)(v + lg_kv4_codes(c, g, key) + d / 8 * 4),
                  *(const uint32_t*)(v + lg_kv4_dm(c, g, key) + d / 32 * 4), x);
    const lg_h2 y = d & 4 ? (d & 2 ? x[3] : x[2]) : (d & 2 ? x[1] : x[0]);
    return (float)(d & 1 ? y[1] : y[0]);
}

/* The keys that rows of positions pmin .. pmax may see, in tiles of KT: those
 * that hold sinks, then those of the windows (one run where they meet). */
struct CaTiles {
    int first, lo, n;
    __device__ __forceinline__ CaTiles(const CAttn& a, int pmin, int pmax, int kt)
    {
        lo = a.window > 0 ? max(0, pmin - a.window + 1) / kt : 0;
        first = min((min(a.sinks, pmax + 1) + kt - 1) / kt, lo);
        n = first + pmax / kt - lo + 1;
    }
    __device__ __forceinline__ int at(int i) const { return i < first ? i : lo + i - first; }
};

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
 * survive whatever their size.  Bound by the cache's bytes: the loads of one
 * tile run while the last one computes. */
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

    __device__ __forceinline__ void load(const CAttn& a, const uint8_t* base, int g, int kb, int r, int c)
    {
#pragma unroll
        for (int u = 0; u < C::NU; u++) {
            const int key = min(kb + 16 * u + r, a.max_pos);   /* (rows past it are never visible) */
            if constexpr (KV4) {
                const uint8_t* const p = base + lg_kv4_codes(a.c, g, key) + (C::RUN ? c * (HD / 8) : 4 * c);
#pragma unroll
                for (int s = 0; s < C::NS; s++) w[u][s] = *(const uint32_t*)(p + s * (C::RUN ? 4 : 16));
                const uint8_t* const q = base + lg_kv4_dm(a.c, g, key) + (HD == 96 ? 0 : HD == 64 ? c / 2 * 4 : c * C::ND * 4);
#pragma unroll
                for (int i = 0; i < C::ND; i++) dm[u][i] = *(const uint32_t*)(q + 4 * i);
            } else {
                const uint8_t* const p = base + lg_kv16_at(a.c, g, key) + 16 * c;
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

template <int HD, bool KV4>
__global__ __launch_bounds__(256, HD <= 128 ? 2 : 1) void k_cattn_dec(CAttn a, int nsplit, float* __restrict__ part)
{
    using C = CaDec<HD, KV4>;
    constexpr int KT = C::KT, NU = C::NU, NB = C::NB, NS = C::NS, NT = C::NT;
    __shared__ __attribute__((aligned(16))) uint8_t s_raw[4 * C::WAVE];
    __shared__ float s_ml[4][16][2];
    const int n_kv = a.c.n_kv, g = blockIdx.x % n_kv, sp = blockIdx.x / n_kv % nsplit, seq = blockIdx.x / n_kv / nsplit;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, c = lane >> 4;
    const int tok = col / a.nrep, ncol = a.ntok * a.nrep;
    const int64_t row = (int64_t)seq * a.ntok + min(tok, a.ntok - 1);
    const int head = g * a.nrep + col % a.nrep;
    int p = a.pos[row];
    if (col >= ncol || p > a.max_pos) p = -1;
    int pmin = p < 0 ? INT32_MAX : p, pmax = p;
#pragma unroll
    for (int o = 1; o < 16; o *= 2) {
        pmin = min(pmin, __shfl_xor(pmin, o));
        pmax = max(pmax, __shfl_xor(pmax, o));
    }
    pmin = __builtin_amdgcn_readfirstlane(pmin);
    pmax = __builtin_amdgcn_readfirstlane(pmax);

    v4f o[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) o[t] = (v4f){};
    float l = 0.0f, mx = -INFINITY;   /* the column's maximum in units of a power of two; l over this lane's keys */
    if (pmax >= 0) {
        const CaTiles tiles(a, pmin, pmax, KT);
        const int t0 = (int)((int64_t)tiles.n * sp / nsplit), t1 = (int)((int64_t)tiles.n * (sp + 1) / nsplit);
        const uint8_t* const kc = a.c.k + (size_t)seq * a.c.seq;
        const uint8_t* const vc = a.c.v + (size_t)seq * a.c.seq;
        _Float16* const sV = (_Float16*)(s_raw + wave * C::WAVE);
        CaRows<HD, KV4> K, V;
        int it = t0 + wave;
        if (it < t1) {
            K.load(a, kc, g, tiles.at(it) * KT, col, c);
            V.load(a, vc, g, tiles.at(it) * KT, col, c);
        }
        /* the column's query in two parts */
        v8h qh[NS], ql[NS];
        float sc;
        {
            float x[NS][8], big = 0.0f;
            const float* const q = a.q + row * a.qs + (size_t)head * HD;
#pragma unroll
            for (int s = 0; s < NS; s++) {
                const int d = C::dim(s, c);
                const bool in = col < ncol && d < HD;
#pragma unroll
                for (int e = 0; e < 8; e += 4) {
                    const v4f y = in ? *(const v4f*)(q + d + e) : (v4f){};
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        x[s][e + i] = y[i];
                        big = fmaxf(big, fabsf(y[i]));
                    }
                }
            }
            big = fmaxf(big, lg_partner<4>(big));
            big = fmaxf(big, lg_partner<5>(big));
            const int ex = __builtin_amdgcn_frexp_expf(big);   /* big < 2^ex */
            sc = ldexpf(a.scale2, ex - 14);
#pragma unroll
            for (int s = 0; s < NS; s++)
#pragma unroll
                for (int e = 0; e < 8; e += 2) ca_split2(ldexpf(x[s][e], 14 - ex), ldexpf(x[s][e + 1], 14 - ex), qh[s], ql[s], e);
        }
        float m = -0x1p40f, cc = __builtin_fmaf(-m, sc, 14.0f);   /* below any score; cc: 14 less the maximum */
        for (; it < t1; it += 4) {
            const int kb = tiles.at(it) * KT;
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
            const int kn = it + 4 < t1 ? tiles.at(it + 4) * KT : -1;
            if (kn >= 0) K.load(a, kc, g, kn, col, c);
            /* keys that some column does not see (wave-uniform) */
            const bool part_seen = kb + KT - 1 > pmin || (a.window > 0 && kb <= pmax - a.window && kb + KT > a.sinks);
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
            if (__builtin_amdgcn_ballot_w64(mn > m)) {
                mn = fmaxf(mn, lg_partner<4>(mn));
                mn = fmaxf(mn, lg_partner<5>(mn));
                mn = fmaxf(mn, m);
                const float cn = __builtin_fmaf(-mn, sc, 14.0f), al = __builtin_amdgcn_exp2f(cn - cc);
                m = mn;
                cc = cn;
                l *= al;
#pragma unroll
                for (int t = 0; t < NT; t++) o[t] *= al;
            }
#pragma unroll
            for (int b = 0; b < NB; b++) {
                uint64_t bad[2] = {};
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int j = 0; j < NS; j++) {
                        v4u x = V.get(2 * b + u, j);
                        if (part_seen) bad[u] |= __builtin_amdgcn_ballot_w64(ca_drop_bad(x));
                        if (HD % 32 == 0 || C::dim(j, c) < HD) *(v4u*)(sV + (16 * u + col) * C::VST + C::dim(j, c)) = x;
                    }
                if (b == NB - 1 && kn >= 0) V.load(a, vc, g, kn, col, c);
                v8h ph, pl;
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    float w[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) w[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * b + u][i], sc, cc));
                    l += (w[0] + w[1]) + (w[2] + w[3]);
                    ca_split2(w[0], w[1], ph, pl, 4 * u);
                    ca_split2(w[2], w[3], ph, pl, 4 * u + 2);
                }
                ca_wave_sync();
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    const _Float16* const v = sV + (4 * c + col / 4) * C::VST + 16 * t + 4 * (col % 4);
                    const v4s x0 = ca_tr16(v), x1 = ca_tr16(v + 16 * C::VST);
                    const v8h x = __builtin_bit_cast(v8h, __builtin_shufflevector(x0, x1, 0, 1, 2, 3, 4, 5, 6, 7));
                    o[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, ph, o[t], 0, 0, 0);
                    o[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, pl, o[t], 0, 0, 0);
                }
                ca_wave_sync();   /* (the reads before the next block's writes) */
                /* infinities and NaN of keys that only some columns see: added
                 * by itself to those that do, whatever the (positive) weight */
#pragma unroll
                for (int u = 0; u < 2; u++)
                    for (uint32_t keys = (uint32_t)(bad[u] | bad[u] >> 16 | bad[u] >> 32 | bad[u] >> 48) & 0xFFFFu; keys;
                         keys &= keys - 1) {
                        const int key = kb + 32 * b + 16 * u + __builtin_ctz(keys);
                        if (ca_sees(a, p, key))
#pragma unroll
                            for (int t = 0; t < NT; t++)
#pragma unroll
                                for (int i = 0; i < 4; i++) {
                                    const float x = ca_value(a.c, vc, g, key, 16 * t + 4 * c + i);
                                    if (!(fabsf(x) <= FLT_MAX)) o[t][i] += x;
                                }
                    }
            }
        }
        l += lg_partner<4>(l);
        l += lg_partner<5>(l);
        mx = l == 0.0f ? -INFINITY : m * sc;
    }
    /* the four waves' parts of each column together, by way of LDS */
    float* const sO = (float*)(s_raw + wave * C::WAVE);
#pragma unroll
    for (int t = 0; t < NT; t++) *(v4f*)(sO + col * C::OST + 16 * t + 4 * c) = o[t];
    if (c == 0) {
        s_ml[wave][col][0] = mx;
        s_ml[wave][col][1] = l;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < ncol * (HD / 4); i += 256) {
        const int k = i / (HD / 4), d = i % (HD / 4) * 4;
        float M = s_ml[0][k][0];
#pragma unroll
        for (int w = 1; w < 4; w++) M = fmaxf(M, s_ml[w][k][0]);
        v4f y = {};
        float L = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; w++) {
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
            if (d == 0) *(float2*)(part + (int64_t)nsplit * a.rows * a.n_heads * HD + 2 * at) = make_float2(M, L);
        } else {
            const float inv = L == 0.0f ? 0.0f : 1.0f / L;
            const int pk = a.pos[r];
            *(v4f*)(a.out + r * a.os + (size_t)hh * HD + d) = pk < 0 || pk > a.max_pos ? (v4f){} : y * inv;
        }
    }
}

/* the splits' parts of a row's head: sum w_i o_i / sum w_i l_i, w_i = 2^(M_i - M);
 * a thread per four dims */
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
            const float f = x.y == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(x.x - M);
            const v4f v = *(const v4f*)(part + (s * n + at) * hd + d);
            L = __builtin_fmaf(x.y, f, L);
#pragma unroll
            for (int e = 0; e < 4; e++) y[e] = __builtin_fmaf(v[e], f, y[e]);
        }
    }
    *(v4f*)(a.out + row * a.os + (size_t)head * hd + d) = y * (L == 0.0f ? 0.0f : 1.0f / L);
}

/* How a call is cut, from its sizes alone. */
struct CaPlan {
    bool dec;     /* up to 16 columns a key head */
    int nsplit;
    size_t ws;
};

static CaPlan ca_plan(int64_t nseq, int64_t ntok, int n_heads, int n_kv, int hd, int window, int sinks, int max_pos)
{
    CaPlan p = {};
    const int64_t cols = ntok * (n_heads / n_kv);
    p.dec = cols <= 16;
    p.nsplit = 1;
    if (p.dec) {
        int64_t keys = (int64_t)max_pos + 1;
        if (window > 0) keys = std::min(keys, (int64_t)window + sinks + ntok - 1);
        /* two workgroups a CU, each with at least a tile for each wave */
        p.nsplit = (int)std::max<int64_t>(1, std::min(512 / (nseq * n_kv), (keys + 255) / 256));
    }
    if (p.nsplit > 1) p.ws = (size_t)p.nsplit * nseq * ntok * n_heads * (hd + 2) * sizeof(float);
    return p;
}

/* One wave per row and head: 64 keys a step, one a lane, their scores from
 * whole cache rows, a running maximum and sum, then each visible key's value
 * row times its weight with the dims over the lanes. */
__global__ __launch_bounds__(256) void k_cattn_row(CAttn a)
{
    __shared__ __attribute__((aligned(16))) float s_q[4][256];
    __shared__ float s_p[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, hd = a.c.hd;
    const int64_t item = (int64_t)blockIdx.x * 4 + wave;
    if (item >= (int64_t)a.rows * a.n_heads) return;
    const int row = (int)(item / a.n_heads), head = (int)(item % a.n_heads), g = head / a.nrep;
    const int p = a.pos[row];
    float o[4] = {0.0f, 0.0f, 0.0f, 0.0f}, m = -FLT_MAX, l = 0.0f;
    for (int d = lane; d < hd; d += 64) s_q[wave][d] = a.q[row * a.qs + head * hd + d] * a.scale2;
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    const size_t seq = (size_t)(row / a.ntok) * a.c.seq;
    if (p >= 0 && p <= a.max_pos) {
        const int lo = a.window > 0 ? max(0, p - a.window + 1) / 64 : 0;
        const int first = min((min(a.sinks, p + 1) + 63) / 64, lo);
        for (int i = 0; i < first + p / 64 - lo + 1; i++) {
            const int kb = 64 * (i < first ? i : lo + i - first), key = kb + lane;
            const bool vis = ca_sees(a, p, key);
            float s = -INFINITY;
            if (vis) {
                s = 0.0f;
                for (int d = 0; d < hd; d += 8) {
                    lg_h2 k[4];
                    if (a.c.type == LG_F16) *(uint4*)k = *(const uint4*)(a.c.k + seq + lg_kv16_at(a.c, g, key) + 2 * d);
                    else
                        lg_kv4_values(*(const uint32_t*)(a.c.k + seq + lg_kv4_codes(a.c, g, key) + d / 2),
                                      *(const uint32_t*)(a.c.k + seq + lg_kv4_dm(a.c, g, key) + d / 32 * 4), k);
                    for (int e = 0; e < 4; e++)
                        s = __builtin_fmaf(s_q[wave][d + 2 * e], (float)k[e][0], __builtin_fmaf(s_q[wave][d + 2 * e + 1], (float)k[e][1], s));
                }
            }
            const float mn = fmaxf(m, lg_group_max<64>(s)), w = vis ? exp2f(s - mn) : 0.0f, al = exp2f(m - mn);
            m = mn;
            l = __builtin_fmaf(l, al, lg_group_sum<64>(w));
            for (int e = 0; e < 4; e++) o[e] *= al;
            s_p[wave][lane] = w;
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            for (uint64_t bits = __builtin_amdgcn_ballot_w64(vis); bits; bits &= bits - 1) {
                const int j = __builtin_ctzll(bits);
                const float w1 = s_p[wave][j];
                for (int e = 0, d = lane; d < hd; e++, d += 64) {
                    float v;
                    if (a.c.type == LG_F16) v = lg_h2f(*(const uint16_t*)(a.c.v + seq + lg_kv16_at(a.c, g, kb + j) + 2 * d));
                    else {
                        lg_h2 x[4];
                        lg_kv4_values(*(const uint32_t*)(a.c.v + seq + lg_kv4_codes(a.c, g, kb + j) + d / 8 * 4),
                                      *(const uint32_t*)(a.c.v + seq + lg_kv4_dm(a.c, g, kb + j) + d / 32 * 4), x);
                        const lg_h2 y = d & 4 ? (d & 2 ? x[3] : x[2]) : (d & 2 ? x[1] : x[0]);
                        v = (float)(d & 1 ? y[1] : y[0]);
                    }
                    o[e] = __builtin_fmaf(w1, v, o[e]);
                }
            }
            __builtin_amdgcn_wave_barrier();
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;   /* (no visible key) */
    for (int e = 0, d = lane; d < hd; e++, d += 64) a.out[row * a.os + head * hd + d] = o[e] * inv;
}

extern "C" size_t lg_attn_cache_workspace_size(int nseq, int ntok, int n_heads, int n_kv_heads, int head_dim, int window,
                                               int sinks, int max_pos)
{
    if (nseq <= 0 || ntok <= 0 || n_heads <= 0 || n_kv_heads <= 0 || head_dim <= 0 || max_pos < 0) return 0;
    return ca_plan(nseq, ntok, n_heads, n_kv_heads, head_dim, window, sinks, max_pos).ws;
}

template <int HD>
static void ca_dec(const CAttn& a, const CaPlan& p, int nseq, float* part, hipStream_t s)
{
    const unsigned n = (unsigned)((int64_t)nseq * a.c.n_kv * p.nsplit);
    if constexpr (HD != 48)
        if (a.c.type == LG_KV4) {
            k_cattn_dec<HD, true><<<n, 256, 0, s>>>(a, p.nsplit, part);
            return;
        }
    k_cattn_dec<HD, false><<<n, 256, 0, s>>>(a, p.nsplit, part);
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
    if (!pos || !q || !out || !lg_al16(q) || !lg_al16(out) || q_stride % 4 || out_stride % 4 || q_stride < width || out_stride < width) {
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
    const CaPlan p = ca_plan(nseq, ntok, n_heads, a.c.n_kv, hd, window, sinks, max_pos);
    if (p.ws && (!workspace || !lg_al16(workspace) || workspace_bytes < p.ws)) {
        lg_set_error("%s: workspace of %zu bytes, 16-byte aligned, %zu needed", who, workspace_bytes, p.ws);
        return LG_ERR_ARG;
    }
    hipStream_t s = (hipStream_t)stream;
    float* const part = p.ws ? (float*)workspace : nullptr;
    if (p.dec) switch (hd) {
        case 48: ca_dec<48>(a, p, nseq, part, s); break;
        case 64: ca_dec<64>(a, p, nseq, part, s); break;
        case 96: ca_dec<96>(a, p, nseq, part, s); break;
        case 128: ca_dec<128>(a, p, nseq, part, s); break;
        default: ca_dec<256>(a, p, nseq, part, s); break;
        }
    else
        k_cattn_row<<<(unsigned)((rows * n_heads + 3) / 4), 256, 0, s>>>(a);
    if (part) k_cattn_merge<<<(unsigned)((rows * n_heads * (hd / 4) + 255) / 256), 256, 0, s>>>(a, p.nsplit, part);
    return lg_check_launch(who);
}
