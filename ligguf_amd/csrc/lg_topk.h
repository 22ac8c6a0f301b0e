/* lg_topk.h -- the highest entries of a row of logits, in order, by one workgroup:
 * log probabilities (lg_logp.hip) and beam search (lg_beam.hip). */
#pragma once

#include <float.h>
#include <math.h>

#include "lg_common.h"

/* (value descending, id ascending) as one unsigned number, larger first: the
 * value's bits in the order of the reals, NaN above all, -0 as +0 */
__device__ __forceinline__ uint64_t lp_key(float x, int id)
{
    const uint32_t b = __float_as_uint(x + 0.0f);
    const uint32_t u = x != x ? 0xFFFFFFFFu : b & 0x80000000u ? ~b : b | 0x80000000u;
    return (uint64_t)u << 32 | (uint32_t)~id;
}
__device__ __forceinline__ float lp_value(uint64_t key)
{
    const uint32_t u = (uint32_t)(key >> 32);
    return u == 0xFFFFFFFFu ? NAN : __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u);
}

constexpr int LP_CAP = 1024;    /* candidates that LDS holds */
constexpr int LP_COLS = 64;     /* threads whose values are looked through for them */
constexpr float LP_LOG2E = 1.44269504088896341f;

/* a row as quads of 16 aligned bytes: quad q holds ids 4q - sh .. +3, the
 * first and last may be cut */
struct LpRow {
    const float* x;
    int vocab, sh;
    __device__ __forceinline__ LpRow(const float* p, int n) : x(p), vocab(n), sh((int)((uintptr_t)p >> 2 & 3)) {}
    __device__ __forceinline__ int quads() const { return (vocab + sh + 3) / 4; }
    /* a quad's values, -infinity in the place of none */
    __device__ __forceinline__ float4 load(int q) const
    {
        const int i = 4 * q - sh;
        if (i >= 0 && i + 3 < vocab) return *(const float4*)(x + i);
        float4 v;
        v.x = i >= 0 && i < vocab ? x[i] : -INFINITY;
        v.y = i + 1 >= 0 && i + 1 < vocab ? x[i + 1] : -INFINITY;
        v.z = i + 2 >= 0 && i + 2 < vocab ? x[i + 2] : -INFINITY;
        v.w = i + 3 < vocab ? x[i + 3] : -INFINITY;
        return v;
    }
};

struct LpShared {
    uint64_t list[LP_CAP];
    float4 sums[16];            /* a wave's m, z, h and its largest value */
    __attribute__((aligned(16))) uint32_t top[256];
    uint32_t hist[256], bound;
    uint64_t prefix;
    int n, nsel, need, sel[LP_COLS];
};

/* a value's place among the reals as an unsigned number; lp_key's upper half */
__device__ __forceinline__ uint32_t lp_ord(float x) { return (uint32_t)(lp_key(x, 0) >> 32); }

/* f(value, id) for the values of quad q */
template <typename F>
__device__ __forceinline__ void lp_quad(const LpRow& r, int q, F f)
{
    const float4 v = r.load(q);
    const int i = 4 * q - r.sh;
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (i + e >= 0 && i + e < r.vocab) f(e == 0 ? v.x : e == 1 ? v.y : e == 2 ? v.z : v.w, i + e);
}

/* the `top` largest keys of s.list[0 .. n), in order, each by the number of
 * larger ones (keys are unique); n >= top */
template <int T, typename F>
__device__ __forceinline__ void lp_emit(const LpShared& s, int n, int top, F f)
{
    for (int i = threadIdx.x; i < n; i += T) {
        const uint64_t k = s.list[i];
        int rank = 0;
#pragma unroll 8
        for (int j = 0; j < n; j++) rank += s.list[j] > k ? 1 : 0;
        if (rank < top) f(rank, k);
    }
}

/* The keys of the row's nq quads that may be among the `top` largest into s.list;
 * returns how many (top at least).  The workgroup's 256 maxima in s.top, of
 * disjoint values, are published; mine: this thread's own, of its quads
 * off + threadIdx.x, + T, ...  A bound that `top` of the 256 reach is found by
 * halving over the upper 16 bits of their order -- a few values more than
 * asked reach it -- and all that do lie in the quads of the threads whose
 * maximum does, so only those are read again.  Where that says little (many
 * maxima reach the bound, fewer than `top` are above -infinity, NaN: `any`)
 * the top-th key is found digit by digit, a pass over the quads for each of
 * its eight bytes. */
template <int T>
__device__ __forceinline__ int lp_top(LpShared& s, const LpRow& r, int nq, int off, int top, uint32_t mine, bool any)
{
    const int t = threadIdx.x;
    if (t < 64) {
        const uint4 v = *(const uint4*)(s.top + 4 * t);
        uint32_t bound = 0;
#pragma unroll
        for (int b = 31; b >= 16; b--) {
            const uint32_t c = bound | 1u << b;
            const int n = __popcll(__builtin_amdgcn_ballot_w64(v.x >= c)) + __popcll(__builtin_amdgcn_ballot_w64(v.y >= c)) +
                          __popcll(__builtin_amdgcn_ballot_w64(v.z >= c)) + __popcll(__builtin_amdgcn_ballot_w64(v.w >= c));
            if (n >= top) bound = c;
        }
        if (t == 0) {
            s.bound = bound;
            s.n = 0;
            s.nsel = 0;
        }
    }
    __syncthreads();
    const uint32_t bound = s.bound;
    const bool use = !any && bound > 0x007FFFFFu;   /* (that of -infinity) */
    if (use && mine >= bound) {
        const int i = atomicAdd(&s.nsel, 1);   /* (in whatever order: the list is ranked) */
        if (i < LP_COLS) s.sel[i] = t;
    }
    __syncthreads();
    const int nsel = s.nsel, per = (nq + T - 1) / T;
    if (use && nsel <= LP_COLS) {
        auto add = [&](float x, int id) {
            const uint64_t k = lp_key(x, id);
            if ((uint32_t)(k >> 32) >= bound) {
                const int at = atomicAdd(&s.n, 1);
                if (at < LP_CAP) s.list[at] = k;
            }
        };
        for (int i = t; i < nsel * per; i += T) {
            const int q = off + s.sel[i / per] + i % per * T;
            if (q < nq) lp_quad(r, q, add);
        }
        if (off && t == T - 1) lp_quad(r, 0, add);
        __syncthreads();
        if (s.n <= LP_CAP) return s.n;
    }
    if (t == 0) {
        s.prefix = 0;
        s.need = top;
    }
    for (int d = 7; d >= 0; d--) {
        if (t < 256) s.hist[t] = 0;
        __syncthreads();
        const uint64_t prefix = s.prefix;
        for (int q = t; q < nq; q += T)
            lp_quad(r, q, [&](float x, int id) {
                const uint64_t k = lp_key(x, id);
                if (d == 7 || k >> (8 * d + 8) == prefix) atomicAdd(&s.hist[k >> (8 * d) & 255], 1u);
            });
        __syncthreads();
        if (t < 64) {   /* the digit in which the need-th largest key lies: lane t counts four, from the top */
            uint32_t c[4], sum = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) sum += c[e] = s.hist[255 - 4 * t - e];
            uint32_t before = sum;
#pragma unroll
            for (int o = 1; o < 64; o *= 2) {
                const uint32_t y = __shfl_up(before, o);
                if (t >= o) before += y;
            }
            before -= sum;
            const uint32_t need = (uint32_t)s.need;
            if (before < need && before + sum >= need) {
                int e = 0;
                while (before + c[e] < need) before += c[e++];   /* (ends: the four reach it) */
                s.prefix = prefix << 8 | (uint32_t)(255 - 4 * t - e);
                s.need = (int)(need - before);
            }
        }
        __syncthreads();
    }
    const uint64_t last = s.prefix;
    if (t == 0) s.n = 0;
    __syncthreads();
    for (int q = t; q < nq; q += T)
        lp_quad(r, q, [&](float x, int id) {
            const uint64_t k = lp_key(x, id);
            if (k >= last) s.list[atomicAdd(&s.n, 1)] = k;   /* exactly top of them */
        });
    __syncthreads();
    return s.n;
}
