/* lg_logp.hip -- log probabilities of given tokens, entropy and the top
 * alternatives of rows of logits. */
#include <float.h>
#include <math.h>

#include <algorithm>

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

struct LpArgs {
    const float* logits;
    int64_t stride;
    int vocab, top;
    const int* toks;
    float *logprob, *entropy, *top_logprob;
    int* top_id;
};

/* a row's scalars from its m, z = sum e^(x - m), h = sum e^(x - m) (x - m);
 * returns log z */
__device__ __forceinline__ float lp_scalars(const LpArgs& a, int row, float m, float z, float h)
{
    const float lz = z > 0.0f ? logf(z) : NAN;   /* (0: nothing above -infinity; NaN: a NaN or +infinity) */
    if (threadIdx.x == 0) {
        if (a.entropy) a.entropy[row] = lz - h / z;
        if (a.logprob) {
            const int t = a.toks[row];
            a.logprob[row] = t >= 0 && t < a.vocab ? a.logits[row * a.stride + t] - m - lz : NAN;
        }
    }
    return lz;
}

__device__ __forceinline__ float lp_first(float x) { return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(x))); }

/* (m, z, h) over the wave: the first lane's, since the compiler fuses a
 * product here into the first addition and the lanes' sums then differ in the
 * last bit -- and which thread writes an entry differs from run to run */
__device__ __forceinline__ void lp_wave(float& m, float& z, float& h)
{
    const float M = lg_group_max<64>(m), d = fmaxf(m - M, -1e30f), al = __builtin_amdgcn_exp2f(d * LP_LOG2E);
    h = lp_first(lg_group_sum<64>(al * __builtin_fmaf(z, d, h)));
    z = lp_first(lg_group_sum<64>(z * al));
    m = lp_first(M);
}

/* One read of the logits: a workgroup takes a row, a thread
 * 16 values at a time with a maximum, a sum and a weighted sum of its own.
 * e^x as 2^(x log2 e) with the maximum taken off before the product, so that
 * the largest term is 1 to the last bit and log z has no error of log2 e's
 * rounding times the maximum.  Bound by the logits' bytes: 600 x 151936, top 20,
 * 74 us, 4.9 TB/s (83 us without the next block's loads ahead); a row of 32000 by
 * the chain of its steps, 7 us. */
template <int T>
__global__ __launch_bounds__(T) void k_logp(LpArgs a)
{
    __shared__ LpShared s;
    const int row = blockIdx.x, t = threadIdx.x;
    const LpRow r(a.logits + row * a.stride, a.vocab);
    const int nq = r.quads();
    float m = -FLT_MAX, z = 0.0f, h = 0.0f, mine = -INFINITY;
    auto take = [&](const float4 (&v)[4]) __attribute__((always_inline)) {
        float x[16];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            x[4 * j] = v[j].x;
            x[4 * j + 1] = v[j].y;
            x[4 * j + 2] = v[j].z;
            x[4 * j + 3] = v[j].w;
        }
#pragma unroll
        for (int i = 0; i < 16; i++) mine = fmaxf(mine, x[i]);
        const float mn = fmaxf(m, mine), d0 = fmaxf(m - mn, -1e30f);
        const float al = __builtin_amdgcn_exp2f(d0 * LP_LOG2E);
        h = al * __builtin_fmaf(z, d0, h);
        z *= al;
        m = mn;
        float zs = 0.0f, hs = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const float d = x[i] - m, e = __builtin_amdgcn_exp2f(d * LP_LOG2E);
            zs += e;
            hs = __builtin_fmaf(e, fmaxf(d, -1e30f), hs);   /* (-infinity times 0 adds nothing) */
        }
        z += zs;
        h += hs;
    };
    /* whole blocks of 4 T quads, the next one on its way; what is left, quad by
     * quad; the first quad of a row that is not aligned, which no thread counts
     * among its own */
    const float4 none = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    const int off = r.sh ? 1 : 0, full = (a.vocab + r.sh) / 4;
    int q = off;
    float4 v[4];
    if (q + 4 * T <= full) {
        const float4* const p = (const float4*)(r.x - r.sh) + t;
        float4 w[4];
#pragma unroll
        for (int j = 0; j < 4; j++) w[j] = p[q + j * T];
        for (; q + 4 * T <= full; q += 4 * T) {
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] = w[j];
            if (q + 8 * T <= full)
#pragma unroll
                for (int j = 0; j < 4; j++) w[j] = p[q + (4 + j) * T];
            take(v);
        }
    }
    for (; q < nq; q += 4 * T) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int at = q + t + j * T;
            v[j] = at < nq ? r.load(at) : none;
        }
        take(v);
    }
    const uint32_t ord = lp_ord(mine);
    if (off) {
        v[0] = t == 0 ? r.load(0) : none;
        v[1] = v[2] = v[3] = none;
        take(v);
    }
    {   /* of T / 256 neighbours */
        uint32_t o = ord;
        if constexpr (T >= 512) o = max(o, (uint32_t)lg_partner<0>((int)o));
        if constexpr (T >= 1024) o = max(o, (uint32_t)lg_partner<1>((int)o));
        if (t % (T / 256) == 0) s.top[t / (T / 256)] = o;
    }
    lp_wave(m, z, h);
    if (t % 64 == 0) s.sums[t / 64] = make_float4(m, z, h, 0.0f);
    __syncthreads();
    {
        const float4 v = t % 64 < T / 64 ? s.sums[t % 64] : make_float4(-FLT_MAX, 0.0f, 0.0f, 0.0f);
        m = v.x;
        z = v.y;
        h = v.z;
        lp_wave(m, z, h);
    }
    const float lz = lp_scalars(a, row, m, z, h);
    if (!a.top) return;
    const int n = lp_top<T>(s, r, nq, off, a.top, ord, z != z);
    lp_emit<T>(s, n, a.top, [&](int rank, uint64_t k) {
        a.top_id[(int64_t)row * a.top + rank] = (int)~(uint32_t)k;
        a.top_logprob[(int64_t)row * a.top + rank] = lp_value(k) - m - lz;
    });
}

extern "C" int lg_logprobs(const float* logits, int64_t stride, int rows, int vocab, const int* toks, int top,
                           float* logprob, float* entropy, int* top_id, float* top_logprob, void* stream)
{
    const char* who = "lg_logprobs";
    if ((rows && !logits) || ((uintptr_t)logits & 3) || rows < 0 || vocab <= 0 || vocab > INT32_MAX - 16 || stride < vocab ||
        top < 0 || top > LG_LOGPROBS_TOP || top > vocab) {
        lg_set_error("%s: bad argument (%d rows of %d, %lld apart, top %d)", who, rows, vocab, (long long)stride, top);
        return LG_ERR_ARG;
    }
    if (!rows) return LG_OK;
    if (!toks != !logprob || !top_id != !top_logprob || !top != !top_id) {
        lg_set_error("%s: tokens and their log probabilities, ids and log probabilities of the top go together", who);
        return LG_ERR_ARG;
    }
    const LpArgs a = {logits, stride, vocab, top, toks, logprob, entropy, top_logprob, top_id};
    /* A workgroup has a row to itself.  1024 threads, and two of them a CU; of
     * many short rows more at a time, with 256 threads each: 700 rows of 4000,
     * top 20, 6 us against 14, of 32000 21 against 23, of 50000 32 against 30;
     * 256 of 16000 11 against 8.  Rows in parts of 4096 logits and a second
     * launch to join them were faster for one row of 151936 only (11 us against
     * 16, without the host's time for that launch; 32000 logits 9 against 8). */
    const bool narrow = rows > 512 && vocab <= 32768;
    if (!lg_grid_fits(rows, narrow ? 256 : 1024)) {
        lg_set_error("%s: %d rows are too many for one call", who, rows);
        return LG_ERR_ARG;
    }
    if (narrow) k_logp<256><<<rows, 256, 0, (hipStream_t)stream>>>(a);
    else k_logp<1024><<<rows, 1024, 0, (hipStream_t)stream>>>(a);
    return lg_check_launch(who);
}
