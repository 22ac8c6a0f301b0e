/* lg_logp.hip -- log probabilities of given tokens, entropy and the top
 * alternatives of rows of logits. */
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


__global__ __launch_bounds__(1024) void k_logp_row(const float* __restrict__ logits, int64_t stride, int vocab,
                                                   const int* __restrict__ toks, int top, float* __restrict__ logprob,
                                                   float* __restrict__ entropy, int* __restrict__ top_id,
                                                   float* __restrict__ top_logprob)
{
    __shared__ float s_m[16], s_z[16], s_h[16];
    __shared__ uint64_t s_k[16];
    const int row = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const float* const x = logits + row * stride;
    float m = -FLT_MAX, bad = 0.0f;
    for (int i = threadIdx.x; i < vocab; i += 1024) {
        m = fmaxf(m, x[i]);
        bad += x[i] == INFINITY || x[i] != x[i] ? 1.0f : 0.0f;
    }
    m = lg_group_max<64>(m);
    if (lane == 0) s_m[wave] = m;
    __syncthreads();
    for (int i = 0; i < 16; i++) m = fmaxf(m, s_m[i]);
    float z = 0.0f, h = 0.0f;
    for (int i = threadIdx.x; i < vocab; i += 1024) {
        const float d = x[i] - m, e = expf(d);
        z += e;
        h += e > 0.0f ? e * d : 0.0f;
    }
    z = lg_block_sum(z, s_z);
    h = lg_block_sum(h, s_h);
    bad = lg_block_sum(bad, s_m);
    const float lz = bad > 0.0f || z == 0.0f ? NAN : logf(z);
    if (threadIdx.x == 0) {
        if (entropy) entropy[row] = lz - h / z;
        if (logprob) {
            const int t = toks[row];
            logprob[row] = t >= 0 && t < vocab ? x[t] - m - lz : NAN;
        }
    }
    uint64_t last = ~0ull;
    for (int r = 0; r < top; r++) {
        uint64_t best = 0;
        for (int i = threadIdx.x; i < vocab; i += 1024) {
            const uint64_t k = lp_key(x[i], i);
            if (k < last && k > best) best = k;
        }
        for (int o = 32; o; o >>= 1) {
            const uint64_t k = __shfl_xor(best, o);
            if (k > best) best = k;
        }
        __syncthreads();
        if (lane == 0) s_k[wave] = best;
        __syncthreads();
        for (int i = 0; i < 16; i++) best = s_k[i] > best ? s_k[i] : best;
        last = best;
        if (threadIdx.x == 0) {
            const int id = (int)~(uint32_t)best;
            top_id[(int64_t)row * top + r] = id;
            top_logprob[(int64_t)row * top + r] = x[id] - m - lz;
        }
    }
}

extern "C" size_t lg_logprobs_workspace_size(int rows, int vocab, int top)
{
    return 0;
}

extern "C" int lg_logprobs(const float* logits, int64_t stride, int rows, int vocab, const int* toks, int top,
                           float* logprob, float* entropy, int* top_id, float* top_logprob, void* workspace,
                           size_t workspace_bytes, void* stream)
{
    const char* who = "lg_logprobs";
    if ((rows && !logits) || ((uintptr_t)logits & 3) || rows < 0 || vocab <= 0 || stride < vocab || top < 0 || top > LG_LOGPROBS_TOP ||
        top > vocab) {
        lg_set_error("%s: bad argument (%d rows of %d, %lld apart, top %d)", who, rows, vocab, (long long)stride, top);
        return LG_ERR_ARG;
    }
    if (!rows) return LG_OK;
    if (!toks != !logprob || !top_id != !top_logprob || !top != !top_id) {
        lg_set_error("%s: tokens and their log probabilities, ids and log probabilities of the top go together", who);
        return LG_ERR_ARG;
    }
    k_logp_row<<<rows, 1024, 0, (hipStream_t)stream>>>(logits, stride, vocab, toks, top, logprob, entropy, top_id, top_logprob);
    return lg_check_launch(who);
}
