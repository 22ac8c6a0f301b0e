/* lg_logp.hip -- log probabilities of given tokens, entropy and the top
 * alternatives of rows of logits. */
#include <algorithm>

#include "lg_topk.h"

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
