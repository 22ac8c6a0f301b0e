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
    return 0;
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
    k_cattn_row<<<(unsigned)((rows * n_heads + 3) / 4), 256, 0, (hipStream_t)stream>>>(a);
    return lg_check_launch(who);
}
