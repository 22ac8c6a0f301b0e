/* lg_kv.h -- the caches that callers keep themselves (lg_kv_cache): where a
 * head's row lies, and the 4-bit form of 32 values. */
#pragma once

#include "lg_common.h"

typedef _Float16 lg_h2 __attribute__((ext_vector_type(2)));

/* pointers + shape as the kernels take them */
struct LgKv {
    uint8_t *k, *v;
    int type, n_ctx, n_kv, hd;
    size_t seq;   /* bytes from one sequence to the next */
};

/* LG_OK, or the refusal of a cache that a call names (nseq sequences) */
int lg_kv_arg(const lg_kv_cache* c, int nseq, const char* who, LgKv* out);

/* LG_OK, or the refusal of caches in pages; *out their pool, a page per sequence */
int lg_kv_pages_arg(const lg_kv_pages* c, const char* who, LgKv* out, int* shift);

static inline bool lg_al16(const void* p) { return ((uintptr_t)p & 15) == 0; }

/* byte offsets within one sequence: a head's fp16 row; its codes and its
 * (d, m) pairs in 4 bits */
__device__ __forceinline__ size_t lg_kv16_at(const LgKv& c, int g, int pos)
{
    return ((size_t)pos * c.n_kv + g) * c.hd * 2;
}
__device__ __forceinline__ size_t lg_kv4_codes(const LgKv& c, int g, int pos)
{
    return ((size_t)g * c.n_ctx + pos) * (c.hd / 2);
}
__device__ __forceinline__ size_t lg_kv4_dm(const LgKv& c, int g, int pos)
{
    return (size_t)c.n_kv * c.n_ctx * (c.hd / 2) + ((size_t)g * c.n_ctx + pos) * (c.hd / 8);
}

/* the eight fp16 values of a word of codes: 2j, 2j + 1 in v[j], by the published
 * method of products of fp16 by 4-bit weights.  A code under the exponent of 1024 is 1024 + c (in bits 0..3) or 1024 + 16 c (4..7); taking
 * the 1024 off, for the latter as x / 16 - 64, is exact.  c d + m is one fused
 * fp16 multiply-add, the one rounding that the format has.  The constants are
 * kept in registers: v_and_or_b32 takes no literal, and as literals they cost
 * two operations and a shift more per pair (19 a word instead of 13). */
__device__ __forceinline__ void lg_kv4_values(uint32_t w, uint32_t dm, lg_h2 v[4])
{
    uint32_t m0 = 0x000F000Fu, m1 = 0x00F000F0u, one = 0x64006400u;
    __asm__("" : "+v"(m0));
    __asm__("" : "+v"(m1));
    __asm__("" : "+s"(one));
    const lg_h2 x = __builtin_bit_cast(lg_h2, dm), d = {x[0], x[0]}, m = {x[1], x[1]};
    const lg_h2 off = {(_Float16)-1024.0f, (_Float16)-1024.0f}, six = {(_Float16)0.0625f, (_Float16)0.0625f};
    const lg_h2 off16 = {(_Float16)-64.0f, (_Float16)-64.0f};
    const uint32_t u = w >> 8;
    const lg_h2 c0 = __builtin_bit_cast(lg_h2, (w & m0) | one) + off;
    const lg_h2 c1 = __builtin_elementwise_fma(__builtin_bit_cast(lg_h2, (w & m1) | one), six, off16);
    const lg_h2 c2 = __builtin_bit_cast(lg_h2, (u & m0) | one) + off;
    const lg_h2 c3 = __builtin_elementwise_fma(__builtin_bit_cast(lg_h2, (u & m1) | one), six, off16);
    v[0] = __builtin_elementwise_fma(c0, d, m);
    v[1] = __builtin_elementwise_fma(c1, d, m);
    v[2] = __builtin_elementwise_fma(c2, d, m);
    v[3] = __builtin_elementwise_fma(c3, d, m);
}

/* the codes of eight values of a group of 32 that four neighbouring lanes
 * (a quad) hold; *dm the group's pair, in every lane.  The code is decided by
 * (x - m) / d in double: in fp32 the same number is off by at most 2^-24
 * relative in the difference and in the quotient, under 2e-6 for quotients up
 * to 16, so only those within 1e-4 of a half are worked out again in double
 * (about one in 5000).  Quotients that clamp need none: far outside 0..15 both
 * forms clamp alike. */
__device__ __forceinline__ uint32_t lg_kv4_encode(const float x[8], uint32_t* dm)
{
    float v[8], lo = INFINITY, hi = -INFINITY;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        nan |= x[i] != x[i];
        v[i] = fminf(fmaxf(x[i], -60000.0f), 60000.0f);
        lo = fminf(lo, v[i]);
        hi = fmaxf(hi, v[i]);
    }
    lo = fminf(lo, lg_partner<0>(lo));
    lo = fminf(lo, lg_partner<1>(lo));
    hi = fmaxf(hi, lg_partner<0>(hi));
    hi = fmaxf(hi, lg_partner<1>(hi));
    int bad = nan;
    bad |= lg_partner<0>(bad);
    bad |= lg_partner<1>(bad);
    if (bad) {
        *dm = 0x7E007E00u;
        return 0;
    }
    const _Float16 m16 = (_Float16)lo;
    const double m = (double)(float)m16;
    /* (m may round above the largest value: then there is nothing to step) */
    const _Float16 d16 = (_Float16)fmaxf((float)(((double)hi - m) / 15.0), 0.0f);
    *dm = (uint32_t)__builtin_bit_cast(uint16_t, d16) | ((uint32_t)__builtin_bit_cast(uint16_t, m16) << 16);
    const float d = (float)d16;
    uint32_t w = 0;
    if (d > 0.0f) {
        const float mf = (float)m16;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float t = (v[i] - mf) / d, r = t - floorf(t);
            float c = rintf(t);
            if (fabsf(r - 0.5f) < 1e-4f) c = (float)__builtin_rint(((double)v[i] - m) / (double)d);
            const uint32_t u = (uint32_t)fminf(fmaxf(c, 0.0f), 15.0f);
            w |= u << (4 * (i >> 1) + 16 * (i & 1));
        }
    }
    return w;
}
