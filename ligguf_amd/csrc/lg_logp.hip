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

constexpr int LP_T = 256;       /* threads */
constexpr int LP_CAP = 1024;    /* candidates that LDS holds */
constexpr int LP_COLS = 64;     /* lanes whose values are looked through for them */
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
    float red[8], top[LP_T];
    uint32_t hist[256];
    uint64_t prefix;
    int n, nsel, need, sel[LP_COLS];
};

/* f(value, id) for the values of quads q0 + lane column `col` of every LP_T */
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
template <typename F>
__device__ __forceinline__ void lp_emit(const LpShared& s, int n, int top, F f)
{
    for (int i = threadIdx.x; i < n; i += LP_T) {
        const uint64_t k = s.list[i];
        int rank = 0;
        for (int j = 0; j < n; j++) rank += s.list[j] > k ? 1 : 0;
        if (rank < top) f(rank, k);
    }
}

/* The top keys of quads [q0, q1) into s.list, returns how many (top or a few
 * more).  mine: the largest value of this thread's quads q0 + threadIdx.x,
 * + LP_T, ...  At least `top` values reach T, the top-th largest of the
 * threads' own maxima, and all that do lie in the quads of threads whose
 * maximum does: only those few threads' quads are read again.  Where that
 * says little -- many maxima equal to T, fewer maxima than `top`, NaN (any) --
 * the top-th key is found digit by digit, a pass over the quads for each of
 * its eight bytes. */
__device__ __forceinline__ int lp_top(LpShared& s, const LpRow& r, int q0, int q1, int top, float mine, bool any)
{
    const int t = threadIdx.x;
    s.top[t] = mine;
    if (t == 0) {
        s.n = 0;
        s.nsel = 0;
    }
    __syncthreads();
    int rank = 0;
    for (int j = 0; j < LP_T; j += 4) {
        const float4 v = *(const float4*)(s.top + j);
        rank += (v.x > mine || (v.x == mine && j < t)) + (v.y > mine || (v.y == mine && j + 1 < t)) +
                (v.z > mine || (v.z == mine && j + 2 < t)) + (v.w > mine || (v.w == mine && j + 3 < t));
    }
    if (rank == top - 1) s.red[0] = mine;
    __syncthreads();
    const float T = s.red[0];
    if (mine >= T && T > -INFINITY) {
        const int i = atomicAdd(&s.nsel, 1);   /* (in whatever order: the list is ranked) */
        if (i < LP_COLS) s.sel[i] = t;
    }
    __syncthreads();
    const int nsel = s.nsel, per = (q1 - q0 + LP_T - 1) / LP_T;
    if (!any && nsel && nsel <= LP_COLS) {
        for (int i = t; i < nsel * per; i += LP_T) {
            const int q = q0 + s.sel[i / per] + i % per * LP_T;
            if (q < q1)
                lp_quad(r, q, [&](float x, int id) {
                    if (x >= T) {
                        const int at = atomicAdd(&s.n, 1);
                        if (at < LP_CAP) s.list[at] = lp_key(x, id);
                    }
                });
        }
        __syncthreads();
        if (s.n <= LP_CAP) return s.n;
    }
    if (t == 0) {
        s.prefix = 0;
        s.need = top;
    }
    for (int d = 7; d >= 0; d--) {
        s.hist[t] = 0;
        __syncthreads();
        const uint64_t prefix = s.prefix;
        for (int q = q0 + t; q < q1; q += LP_T)
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
    for (int q = q0 + t; q < q1; q += LP_T)
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
    int rows, vocab, top, nsplit;
    const int* toks;
    float *logprob, *entropy, *top_logprob;
    int* top_id;
    float4* sums;     /* [rows][nsplit]: m, z, h */
    uint64_t* keys;   /* [rows][nsplit][top], descending */
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

__device__ __forceinline__ void lp_put(const LpArgs& a, int row, int rank, uint64_t key, float m, float lz)
{
    a.top_id[(int64_t)row * a.top + rank] = (int)~(uint32_t)key;
    a.top_logprob[(int64_t)row * a.top + rank] = lp_value(key) - m - lz;
}

/* One read of the logits: a workgroup takes a row or a part of one, a thread
 * 16 values at a time with a maximum, a sum and a weighted sum of its own.
 * e^x as 2^(x log2 e) with the maximum taken off before the product, so that
 * the largest term is 1 to the last bit and log z has no error of log2 e's
 * rounding times the maximum. */
__global__ __launch_bounds__(LP_T) void k_logp(LpArgs a)
{
    __shared__ LpShared s;
    const int row = blockIdx.x / a.nsplit, sp = blockIdx.x % a.nsplit;
    const LpRow r(a.logits + row * a.stride, a.vocab);
    const int64_t nq = r.quads();
    const int q0 = (int)(nq * sp / a.nsplit), q1 = (int)(nq * (sp + 1) / a.nsplit);
    float m = -FLT_MAX, z = 0.0f, h = 0.0f, mine = -INFINITY;
    for (int q = q0 + threadIdx.x; q < q1; q += 4 * LP_T) {
        float x[16];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int at = q + j * LP_T;
            const float4 v = at < q1 ? r.load(at) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            x[4 * j] = v.x;
            x[4 * j + 1] = v.y;
            x[4 * j + 2] = v.z;
            x[4 * j + 3] = v.w;
        }
#pragma unroll
        for (int i = 0; i < 16; i++) mine = fmaxf(mine, x[i]);
        const float mn = fmaxf(m, mine), d0 = fmaxf(m - mn, -1e30f), al = __builtin_amdgcn_exp2f(d0 * LP_LOG2E);
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
    }
    float M = lg_group_max<64>(m);
    if ((threadIdx.x & 63) == 0) s.red[threadIdx.x >> 6] = M;
    __syncthreads();
    M = fmaxf(fmaxf(s.red[0], s.red[1]), fmaxf(s.red[2], s.red[3]));
    const float d0 = fmaxf(m - M, -1e30f), al = __builtin_amdgcn_exp2f(d0 * LP_LOG2E);
    h = lg_block_sum(al * __builtin_fmaf(z, d0, h), s.red);
    z = lg_block_sum(z * al, s.red);
    __syncthreads();
    const bool whole = a.nsplit == 1;
    float lz = 0.0f;
    if (whole) lz = lp_scalars(a, row, M, z, h);
    else if (threadIdx.x == 0) a.sums[blockIdx.x] = make_float4(M, z, h, 0.0f);
    if (!a.top) return;
    const int n = lp_top(s, r, q0, q1, a.top, mine, z != z);
    lp_emit(s, n, a.top, [&](int rank, uint64_t k) {
        if (whole) lp_put(a, row, rank, k, M, lz);
        else a.keys[(int64_t)blockIdx.x * a.top + rank] = k;
    });
}

/* The parts of a row.  Every part has `top` keys in order, so at least `top` keys reach the largest of
 * the parts' last ones, and the least of the parts' (ceil(top / parts))-th
 * ones: the larger bound leaves few to rank. */
__global__ __launch_bounds__(LP_T) void k_logp_join(LpArgs a)
{
    __shared__ LpShared s;
    const int row = blockIdx.x, t = threadIdx.x, ns = a.nsplit, top = a.top;
    const float4* const p = a.sums + (int64_t)row * ns;
    float M = -FLT_MAX, z = 0.0f, h = 0.0f;
    for (int i = 0; i < ns; i++) M = fmaxf(M, p[i].x);
    for (int i = 0; i < ns; i++) {
        const float d0 = fmaxf(p[i].x - M, -1e30f), al = __builtin_amdgcn_exp2f(d0 * LP_LOG2E);
        h += al * __builtin_fmaf(p[i].y, d0, p[i].z);
        z = __builtin_fmaf(p[i].y, al, z);
    }
    const float lz = lp_scalars(a, row, M, z, h);
    if (!top) return;
    const uint64_t* const keys = a.keys + (int64_t)row * ns * top;
    const int deep = (top + ns - 1) / ns - 1;
    uint64_t b0 = 0, b1 = ~0ull;
    for (int i = 0; i < ns; i++) {
        const uint64_t x = keys[i * top + top - 1], y = keys[i * top + deep];
        b0 = x > b0 ? x : b0;
        b1 = y < b1 ? y : b1;
    }
    const uint64_t bound = b0 > b1 ? b0 : b1;
    if (t == 0) s.n = 0;
    __syncthreads();
    for (int i = t; i < ns * top; i += LP_T)
        if (keys[i] >= bound) s.list[atomicAdd(&s.n, 1)] = keys[i];
    __syncthreads();
    lp_emit(s, s.n, top, [&](int rank, uint64_t k) { lp_put(a, row, rank, k, M, lz); });
}

/* parts of a row: some eight workgroups a CU in all, parts of at least 4096
 * logits, and no more keys than the join's list holds */
static int lp_split(int64_t rows, int vocab)
{
    return (int)std::max<int64_t>(1, std::min<int64_t>({2048 / rows, vocab / 4096, LP_CAP / LG_LOGPROBS_TOP}));
}

extern "C" size_t lg_logprobs_workspace_size(int rows, int vocab, int top)
{
    if (rows <= 0 || vocab <= 0 || top < 0) return 0;
    const int ns = lp_split(rows, vocab);
    return ns > 1 ? (size_t)rows * ns * (16 + 8 * (size_t)top) : 0;
}

extern "C" int lg_logprobs(const float* logits, int64_t stride, int rows, int vocab, const int* toks, int top,
                           float* logprob, float* entropy, int* top_id, float* top_logprob, void* workspace,
                           size_t workspace_bytes, void* stream)
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
    LpArgs a = {logits, stride, rows, vocab, top, lp_split(rows, vocab), toks, logprob, entropy, top_logprob, top_id,
                nullptr, nullptr};
    const size_t need = lg_logprobs_workspace_size(rows, vocab, top);
    if (need && (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < need)) {
        lg_set_error("%s: workspace of %zu bytes, 16-byte aligned, %zu needed", who, workspace_bytes, need);
        return LG_ERR_ARG;
    }
    if (need) {
        a.sums = (float4*)workspace;
        a.keys = (uint64_t*)(a.sums + (size_t)rows * a.nsplit);
    }
    k_logp<<<(unsigned)rows * a.nsplit, LP_T, 0, (hipStream_t)stream>>>(a);
    if (a.nsplit > 1) k_logp_join<<<rows, LP_T, 0, (hipStream_t)stream>>>(a);
    return lg_check_launch(who);
}
