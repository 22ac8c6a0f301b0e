/* lg_kvrope.hip -- norm and rotation of many tokens' query and key heads with
 * the cache write, rotary frequency tables, reading a 4-bit cache back. */
#include <math.h>

#include <algorithm>

#include "lg_kv.h"

extern "C" int64_t lg_kv_bytes(int type, int n_ctx, int n_kv_heads, int head_dim)
{
    if (n_ctx <= 0 || n_ctx > 1 << 30 || n_kv_heads <= 0 || head_dim <= 0 || head_dim > 256) return -1;
    const int64_t n = (int64_t)n_ctx * n_kv_heads;   /* < 2^62; times 512 checked below */
    if (n > ((int64_t)1 << 50)) return -1;
    if (type == LG_F16) return n * head_dim * 2;
    if (type == LG_KV4 && head_dim % 32 == 0) return n * (head_dim / 2 + head_dim / 8);
    return -1;
}

int lg_kv_arg(const lg_kv_cache* c, int nseq, const char* who, LgKv* out)
{
    if (c->type != LG_F16 && c->type != LG_KV4) {
        lg_set_error("%s: cache type %d (LG_F16, LG_KV4)", who, c->type);
        return LG_ERR_TYPE;
    }
    const int64_t need = lg_kv_bytes(c->type, c->n_ctx, c->n_kv_heads, c->head_dim);
    if (need < 0) {
        lg_set_error("%s: no cache of %d rows, %d heads of %d", who, c->n_ctx, c->n_kv_heads, c->head_dim);
        return LG_ERR_ARG;
    }
    if (!c->k || !c->v || !lg_al16(c->k) || !lg_al16(c->v)) {
        lg_set_error("%s: cache pointers must be 16-byte aligned", who);
        return LG_ERR_ARG;
    }
    if (nseq > 1 && (c->seq_bytes % 16 || c->seq_bytes < (size_t)need || c->seq_bytes > ((size_t)1 << 58) / nseq)) {
        lg_set_error("%s: sequences %zu bytes apart, %lld needed, in multiples of 16", who, c->seq_bytes,
                     (long long)need);
        return LG_ERR_ARG;
    }
    *out = {(uint8_t*)c->k, (uint8_t*)c->v, c->type, c->n_ctx, c->n_kv_heads, c->head_dim, nseq > 1 ? c->seq_bytes : 0};
    return LG_OK;
}

extern "C" int lg_rope_table(int scaling, int rope_dim, double base, double factor, int orig_ctx, double p0, double p1,
                             float* freq, float* mscale)
{
    const bool parts = scaling == LG_ROPE_YARN || scaling == LG_ROPE_BANDS;
    if (!freq || !mscale || rope_dim <= 0 || rope_dim % 2 || rope_dim > 256 || !(base > 1.0) || !std::isfinite(base)) {
        lg_set_error("lg_rope_table: bad argument");
        return LG_ERR_ARG;
    }
    if (scaling < LG_ROPE_PLAIN || scaling > LG_ROPE_BANDS) {
        lg_set_error("lg_rope_table: scaling %d unknown", scaling);
        return LG_ERR_ARG;
    }
    if (scaling != LG_ROPE_PLAIN && (!(factor >= 1.0) || !std::isfinite(factor))) {
        lg_set_error("lg_rope_table: factor %g below 1", factor);
        return LG_ERR_ARG;
    }
    if (parts && (orig_ctx <= 0 || !(p1 > 0.0) || !(p0 > p1) || !std::isfinite(p0))) {
        lg_set_error("lg_rope_table: needs a trained context and p0 > p1 > 0 (%d, %g, %g)", orig_ctx, p0, p1);
        return LG_ERR_ARG;
    }
    if (scaling == LG_ROPE_NTK && rope_dim == 2) {
        lg_set_error("lg_rope_table: no base to scale for one pair");
        return LG_ERR_ARG;
    }
    const double two_pi = 6.283185307179586476925;
    const double b = scaling == LG_ROPE_NTK ? base * pow(factor, rope_dim / (rope_dim - 2.0)) : base;
    double first = 0.0, last = 0.0;
    if (scaling == LG_ROPE_YARN) {
        /* the dim that turns n times over the trained context */
        auto dim = [&](double n) { return rope_dim * log(orig_ctx / (n * two_pi)) / (2.0 * log(base)); };
        first = std::max(floor(dim(p0)), 0.0);
        last = std::min(ceil(dim(p1)), rope_dim - 1.0);
    }
    for (int i = 0; i < rope_dim / 2; i++) {
        double f = pow(b, -2.0 * i / rope_dim);
        if (scaling == LG_ROPE_LINEAR) f /= factor;
        if (scaling == LG_ROPE_YARN) {
            const double r = std::min(std::max((i - first) / std::max(last - first, 1e-3), 0.0), 1.0);
            f = f * (1.0 - r) + f / factor * r;
        }
        if (scaling == LG_ROPE_BANDS) {
            const double turns = orig_ctx * f / two_pi;
            const double r = std::min(std::max((turns - p1) / (p0 - p1), 0.0), 1.0);
            f = f / factor * (1.0 - r) + f * r;
        }
        freq[i] = (float)f;
    }
    *mscale = scaling == LG_ROPE_YARN ? (float)(1.0 + 0.1 * log(factor)) : 1.0f;
    return LG_OK;
}

struct RopeArgs {
    const float *q, *k, *v, *qw, *kw, *freq;
    float *qo, *ko;
    const int* pos;
    int64_t qs, qos, ks, kos, vs;
    int n_heads, n_kv, hd, rope, ntok;
    float mscale, eps;
    LgKv c;   /* c.type 0: no cache */
};

/* cos, sin of pos * freq, times mscale, rounded once.  Far positions need the angle in
 * double: at 10^5 radians fp32 would leave 0.004 of it.  a / 2 pi with its low
 * half in a fused multiply-add, less the nearest whole number of turns. */
__device__ __forceinline__ float2 lg_turn(int pos, float freq, float mscale)
{
    const double inv = 0.15915494309189535, inv_lo = -9.839338337591243e-18;
    const double a = (double)pos * (double)freq, n = __builtin_rint(a * inv);
    const double r = __builtin_fma(a, inv, -n) + a * inv_lo;
    double s, c;
    sincospi(2.0 * r, &s, &c);
    return make_float2((float)(c * mscale), (float)(s * mscale));
}

typedef float v2f __attribute__((ext_vector_type(2), aligned(4)));
typedef float v4f __attribute__((ext_vector_type(4)));

/* A workgroup takes a token's heads from `blk * per` rounds on: queries, then
 * keys, then values; in a round each of its four waves takes 64 / G heads, G
 * lanes a head.  A lane holds N neighbouring pairs p = N i .. of its head (and
 * those 64 on, in the one-pair form): the two values that turn together, or
 * past rope_dim two neighbours that stay -- so a pair never leaves its lane in
 * either layout, and the norm's sum is the only exchange.  N = 2 needs the
 * pairs to come in twos (head_dim % 4 == 0, rope_dim % 4 == 0): 16 bytes a
 * lane.  N = 1 takes every other shape.  Bound by its bytes: 6000 tokens of
 * 32 + 8 heads of 128, 246 MB, 46 us, 5.3 TB/s (73 us with one pair a lane; 56
 * with two rounds loaded at a time, whose registers halve the waves).  Rows for the 4-bit cache
 * go through LDS to eight consecutive values a lane. */
template <bool HALF, int N, int G>
__global__ __launch_bounds__(256) void k_rope_tokens(RopeArgs a, int nblk, int per)
{
    constexpr int HPW = 64 / G, J = N == 2 ? 1 : 2;   /* heads of a wave, runs of pairs of a lane */
    __shared__ float2 s_cs[128];
    __shared__ __attribute__((aligned(16))) float s_row[4][256];
    const int row = blockIdx.x / nblk, blk = blockIdx.x % nblk;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, li = lane % G;
    const int pos = a.pos[row];
    const int np = a.rope / 2, hd = a.hd, seq = row / a.ntok;
    const int n_all = a.n_heads + a.n_kv * (a.c.type ? 2 : 1);
    const bool on = pos >= 0 && (!a.c.type || pos < a.c.n_ctx);   /* (workgroup-uniform) */

    struct Head {
        int kind, g;   /* 0 query, 1 key, 2 value, 3 none */
        float e[J][2 * N];
    };
    auto head_of = [&](int h, Head& x) {
        x.kind = h < a.n_heads ? 0 : h < a.n_heads + a.n_kv ? 1 : h < n_all ? 2 : 3;
        x.g = x.kind == 0 ? h : x.kind == 1 ? h - a.n_heads : h - a.n_heads - a.n_kv;
    };
    /* element e of the lane's run j: pair N (li + G j) + e / 2; HALF keeps the first
     * values of its pairs together, then the second ones */
    auto at = [&](int j, int e, bool value) {
        const int p = N * (li + G * j), half = HALF && !value && p < np;
        return half ? (e < N ? p + e : p + np + e - N) : 2 * p + e;
    };
    auto turns = [&](int j, bool value) { return !value && N * (li + G * j) < np; };
    auto in = [&](int j) { return N * (li + G * j) < hd / 2; };
    auto ld = [&](const float* p, int j, bool value, float* e) {
        if constexpr (N == 2) {
            if (HALF) {
                *(v2f*)e = *(const v2f*)(p + at(j, 0, value));
                *(v2f*)(e + 2) = *(const v2f*)(p + at(j, 2, value));
            } else
                *(v4f*)e = *(const v4f*)(p + at(j, 0, value));
        } else {
            e[0] = p[at(j, 0, value)];
            e[1] = p[at(j, 1, value)];
        }
    };
    auto st = [&](float* p, int j, bool value, const float* e) {
        if constexpr (N == 2) {
            if (HALF) {
                *(v2f*)(p + at(j, 0, value)) = *(const v2f*)e;
                *(v2f*)(p + at(j, 2, value)) = *(const v2f*)(e + 2);
            } else
                *(v4f*)(p + at(j, 0, value)) = *(const v4f*)e;
        } else {
            p[at(j, 0, value)] = e[0];
            p[at(j, 1, value)] = e[1];
        }
    };

    for (int i = 0; i < per; i++) {
        const int h0 = ((blk * per + i) * 4 + wave) * HPW;
        Head x;
        head_of(h0 + lane / G, x);
        const int kind = x.kind, g = x.g;
        {
            const float* const p = kind == 0 ? a.q + row * a.qs : kind == 1 ? a.k + row * a.ks : a.v + row * a.vs;
#pragma unroll
            for (int j = 0; j < J; j++) {
#pragma unroll
                for (int e = 0; e < 2 * N; e++) x.e[j][e] = 0.0f;
                if (on && kind < 3 && in(j)) ld(p + (size_t)g * hd, j, kind == 2, x.e[j]);
            }
        }
        if (i == 0) {   /* (the first loads are on their way) */
            if (on && (int)threadIdx.x < np) s_cs[threadIdx.x] = lg_turn(pos, a.freq[threadIdx.x], a.mscale);
            __syncthreads();
        }
        const bool value = kind == 2;
        const float* const w = kind == 0 ? a.qw : kind == 1 ? a.kw : nullptr;
        if (a.qw || a.kw) {   /* (all lanes take part in the sums) */
            float ss = 0.0f;
#pragma unroll
            for (int j = 0; j < J; j++)
#pragma unroll
                for (int e = 0; e < 2 * N; e++) ss = __builtin_fmaf(x.e[j][e], x.e[j][e], ss);
            const float sc = 1.0f / sqrtf(lg_group_sum<G>(ss) / (float)hd + a.eps);
#pragma unroll
            for (int j = 0; j < J; j++)
                if (w && in(j)) {
                    float f[2 * N];
                    ld(w, j, value, f);
#pragma unroll
                    for (int e = 0; e < 2 * N; e++) x.e[j][e] = on ? x.e[j][e] * sc * f[e] : 0.0f;
                }
        }
        float* const y = kind == 0 ? a.qo + row * a.qos : kind == 1 && a.ko ? a.ko + row * a.kos : nullptr;
#pragma unroll
        for (int j = 0; j < J; j++) {
            float* const e = x.e[j];
            if (on && turns(j, value)) {
#pragma unroll
                for (int k = 0; k < N; k++) {
                    const float2 t = s_cs[N * (li + G * j) + k];
                    float &v0 = e[HALF ? k : 2 * k], &v1 = e[HALF ? k + N : 2 * k + 1];
                    const float x0 = v0, x1 = v1;
                    v0 = lg_fma2(x0, t.x, -x1, t.y);
                    v1 = lg_fma2(x0, t.y, x1, t.x);
                }
            }
            if (kind < 2 && y && in(j)) st(y + (size_t)g * hd, j, value, e);
        }
        if (!a.c.type || !on) continue;
        if (a.c.type == LG_F16) {
            if (kind == 1 || kind == 2) {
                uint16_t* const r = (uint16_t*)((value ? a.c.v : a.c.k) + (size_t)seq * a.c.seq + lg_kv16_at(a.c, g, pos));
#pragma unroll
                for (int j = 0; j < J; j++)
                    if (in(j)) {
                        const float* const e = x.e[j];
                        if constexpr (N == 2) {
                            const uint32_t w0 = (uint32_t)lg_f2h(e[0]) | (uint32_t)lg_f2h(e[1]) << 16;
                            const uint32_t w1 = (uint32_t)lg_f2h(e[2]) | (uint32_t)lg_f2h(e[3]) << 16;
                            if (HALF) {
                                *(uint32_t*)(r + at(j, 0, value)) = w0;
                                *(uint32_t*)(r + at(j, 2, value)) = w1;
                            } else
                                *(uint2*)(r + at(j, 0, value)) = make_uint2(w0, w1);
                        } else {
                            r[at(j, 0, value)] = lg_f2h(e[0]);
                            r[at(j, 1, value)] = lg_f2h(e[1]);
                        }
                    }
            }
        } else if (__builtin_amdgcn_ballot_w64(kind == 1 || kind == 2)) {
            float* const s = s_row[wave];
#pragma unroll
            for (int j = 0; j < J; j++)
                if (in(j)) st(s + lane / G * hd, j, value, x.e[j]);
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            const int hw = hd / 8, k = lane / hw;   /* the wave's head that this lane has a word of, four lanes a group */
            Head z;
            head_of(h0 + k, z);
            float v[8] = {};
            if (k < HPW) {
                *(v4f*)v = *(const v4f*)(s + 8 * lane);
                *(v4f*)(v + 4) = *(const v4f*)(s + 8 * lane + 4);
            }
            uint32_t dm;
            const uint32_t code = lg_kv4_encode(v, &dm);
            if (k < HPW && (z.kind == 1 || z.kind == 2)) {
                uint8_t* const c = (z.kind == 2 ? a.c.v : a.c.k) + (size_t)seq * a.c.seq;
                const int wd = lane % hw;
                ((uint32_t*)(c + lg_kv4_codes(a.c, z.g, pos)))[wd] = code;
                if (wd % 4 == 0) ((uint32_t*)(c + lg_kv4_dm(a.c, z.g, pos)))[wd / 4] = dm;
            }
            __builtin_amdgcn_wave_barrier();   /* the row's reads before the next round's writes */
        }
    }
}

template <bool HALF, int N, int G>
static void rope_launch(const RopeArgs& a, int64_t rows, int all, hipStream_t s)
{
    /* rounds of four waves' heads.  Many rows: a workgroup takes all of a
     * token's, so that its angles (in double) are worked out once; few: one
     * round each, for more of them at a time */
    const int rounds = (all + 4 * (64 / G) - 1) / (4 * (64 / G));
    const int nblk = rows >= 512 || !lg_grid_fits(rows * rounds, 256) ? 1 : rounds;
    k_rope_tokens<HALF, N, G><<<(unsigned)(rows * nblk), 256, 0, s>>>(a, nblk, nblk == 1 ? rounds : 1);
}

template <bool HALF>
static void rope_shape(const RopeArgs& a, int64_t rows, int all, hipStream_t s)
{
    if (a.hd % 4 || a.rope % 4 || (a.qw && !lg_al16(a.qw)) || (a.kw && !lg_al16(a.kw)))
        rope_launch<HALF, 1, 64>(a, rows, all, s);
    else if (a.hd <= 64) rope_launch<HALF, 2, 16>(a, rows, all, s);
    else if (a.hd <= 128) rope_launch<HALF, 2, 32>(a, rows, all, s);
    else rope_launch<HALF, 2, 64>(a, rows, all, s);
}

static bool rows_bad(const void* p, int64_t stride, int64_t least)
{
    return !p || !lg_al16(p) || stride % 4 || stride < least;
}

extern "C" int lg_qk_norm_rope_tokens(const float* q, int64_t q_stride, float* q_out, int64_t q_out_stride,
                                      const float* k, int64_t k_stride, float* k_out, int64_t k_out_stride,
                                      const float* v, int64_t v_stride, const float* qw, const float* kw, int n_heads,
                                      int n_kv_heads, int head_dim, int rope_dim, int layout, const float* freq,
                                      float mscale, float eps, const int* pos, int nseq, int ntok,
                                      const lg_kv_cache* cache, void* stream)
{
    const char* who = "lg_qk_norm_rope_tokens";
    if (nseq < 0 || ntok < 0 || n_heads < 0 || n_kv_heads <= 0 || n_heads > 65536 || n_kv_heads > 65536) {
        lg_set_error("%s: bad sizes (%d sequences of %d tokens, %d / %d heads)", who, nseq, ntok, n_heads, n_kv_heads);
        return LG_ERR_ARG;
    }
    if (head_dim <= 0 || head_dim > 256 || head_dim % 2 || rope_dim < 0 || rope_dim % 2 || rope_dim > head_dim ||
        (layout != LG_ROPE_ADJACENT && layout != LG_ROPE_HALF)) {
        lg_set_error("%s: head_dim %d, rope_dim %d, layout %d", who, head_dim, rope_dim, layout);
        return LG_ERR_ARG;
    }
    const int64_t rows = (int64_t)nseq * ntok;
    if (!rows) return LG_OK;
    if (!(eps >= 0.0f) || !pos || (rope_dim && !freq)) {
        lg_set_error("%s: bad argument", who);
        return LG_ERR_ARG;
    }
    const int64_t nq = (int64_t)n_heads * head_dim, nk = (int64_t)n_kv_heads * head_dim;
    if ((n_heads && (rows_bad(q, q_stride, nq) || rows_bad(q_out, q_out_stride, nq))) || rows_bad(k, k_stride, nk) ||
        (k_out && rows_bad(k_out, k_out_stride, nk)) || (!k_out && !cache) || (cache && rows_bad(v, v_stride, nk))) {
        lg_set_error("%s: rows must be given, 16-byte aligned and as wide as their heads", who);
        return LG_ERR_ARG;
    }
    RopeArgs a = {q, k, v, qw, kw, freq, q_out, k_out, pos, q_stride, q_out_stride, k_stride, k_out_stride, v_stride,
                  n_heads, n_kv_heads, head_dim, rope_dim, ntok, mscale, eps, {}};
    if (cache) {
        const int rc = lg_kv_arg(cache, nseq, who, &a.c);
        if (rc) return rc;
        if (cache->n_kv_heads != n_kv_heads || cache->head_dim != head_dim) {
            lg_set_error("%s: the cache has %d heads of %d, the keys %d of %d", who, cache->n_kv_heads,
                         cache->head_dim, n_kv_heads, head_dim);
            return LG_ERR_ARG;
        }
    }
    const int waves = n_heads + n_kv_heads * (cache ? 2 : 1);
    if (rows > INT32_MAX / waves || !lg_grid_fits(rows, 256)) {
        lg_set_error("%s: %lld rows of %d heads are too many for one call", who, (long long)rows, waves);
        return LG_ERR_ARG;
    }
    if (layout == LG_ROPE_HALF) rope_shape<true>(a, rows, waves, (hipStream_t)stream);
    else rope_shape<false>(a, rows, waves, (hipStream_t)stream);
    return lg_check_launch(who);
}

/* One thread per word of eight codes; keys, then values.  Fewer than 2^32 words of
 * a sequence (64-bit divisions cost more than the reads). */
__global__ __launch_bounds__(256) void k_kv4_read(LgKv c, int pos0, int npos, uint16_t* __restrict__ ko,
                                                  uint16_t* __restrict__ vo)
{
    const uint32_t hw = c.hd / 8, i = blockIdx.x * 256 + threadIdx.x;   /* words of a head's row */
    if (i >= (uint32_t)npos * c.n_kv * hw) return;
    const uint32_t r = i / hw, n_kv = c.n_kv;
    const int wd = (int)(i - r * hw), p = (int)(r / n_kv), g = (int)(r - p * n_kv), seq = blockIdx.y;
    const uint8_t* const b = (blockIdx.z ? c.v : c.k) + (size_t)seq * c.seq;
    const uint32_t w = ((const uint32_t*)(b + lg_kv4_codes(c, g, pos0 + p)))[wd];
    const uint32_t dm = ((const uint32_t*)(b + lg_kv4_dm(c, g, pos0 + p)))[wd / 4];
    lg_h2 v[4];
    lg_kv4_values(w, dm, v);
    uint16_t* const o = (blockIdx.z ? vo : ko) + (size_t)seq * npos * c.n_kv * c.hd + 8 * (size_t)i;
    *(uint4*)o = *(const uint4*)v;
}

extern "C" int lg_kv4_read(const lg_kv_cache* cache, int nseq, int pos0, int npos, uint16_t* k_out, uint16_t* v_out,
                           void* stream)
{
    const char* who = "lg_kv4_read";
    if (!cache || nseq < 0 || nseq > 65535) {
        lg_set_error("%s: bad argument (%d sequences)", who, nseq);
        return LG_ERR_ARG;
    }
    LgKv c;
    const int rc = lg_kv_arg(cache, nseq, who, &c);
    if (rc) return rc;
    if (c.type != LG_KV4) {
        lg_set_error("%s: the cache is not in 4 bits", who);
        return LG_ERR_TYPE;
    }
    if (pos0 < 0 || npos < 0 || npos > c.n_ctx - pos0 || !k_out || !v_out || !lg_al16(k_out) || !lg_al16(v_out)) {
        lg_set_error("%s: rows %d .. %d of %d, or outputs not 16-byte aligned", who, pos0, pos0 + npos, c.n_ctx);
        return LG_ERR_ARG;
    }
    const int64_t n = ((int64_t)npos * c.n_kv * (c.hd / 8) + 255) / 256;
    if (!lg_grid_fits(n, 256)) {
        lg_set_error("%s: %d rows are too many for one call", who, npos);
        return LG_ERR_ARG;
    }
    if (!n || !nseq) return LG_OK;
    const dim3 grid((unsigned)n, nseq, 2);
    k_kv4_read<<<grid, 256, 0, (hipStream_t)stream>>>(c, pos0, npos, k_out, v_out);
    return lg_check_launch(who);
}
