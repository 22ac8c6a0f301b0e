/* lg_beam.hip -- the best continuations over beams and vocabulary, and the page
 * tables of the chosen ones. */
#include <algorithm>

#include "lg_kv.h"
#include "lg_topk.h"

struct BeamArgs {
    const float *logits, *scores;
    const int* done;
    int64_t stride;
    int end, beams, vocab, top, parts, part;   /* a row in `parts` of `part` logits (the last one fewer) */
    float2* mz;       /* of each row's parts: maximum, sum of e^(x - m) */
    uint64_t* keys;   /* and its highest entries (lp_key), `top` places each */
    float* score;
    int *parent, *token;
};

/* whether a row's logits are read: an unfinished beam that has a score */
__device__ __forceinline__ bool bm_live(const BeamArgs& a, int64_t row)
{
    return fabsf(a.scores[row]) <= FLT_MAX && !(a.done && a.done[row]);
}

/* A part of a row: its maximum, the sum of e^(x - m) and its `top` highest
 * entries in order.  16 values of a thread at a time, the next ones on their way
 * (as k_logp).  Bound by the logits' bytes, read once: 320 rows of 151936, a fifth of
 * them finished, 38 us, 4.1 TB/s (a copy's 4.9; 32 values at a time spill, 55; parts
 * and 256 or 512 threads 44 to 50); of few rows by its chain: 4 of 32000 6.5 us. */
constexpr int BM_ROW_THREADS = 1024;
__global__ __launch_bounds__(BM_ROW_THREADS) void k_beam_rows(BeamArgs a)
{
    constexpr int T = BM_ROW_THREADS;
    __shared__ LpShared s;
    const int64_t row = blockIdx.x / a.parts;
    const int part = blockIdx.x % a.parts, t = threadIdx.x;
    if (!bm_live(a, row)) return;
    const int first = part * a.part, n = min(a.part, a.vocab - first);
    const LpRow r(a.logits + row * a.stride + first, n);
    const int nq = r.quads();
    float m = -FLT_MAX, z = 0.0f, mine = -INFINITY;
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
        const float mn = fmaxf(m, mine);
        z *= __builtin_amdgcn_exp2f((m - mn) * LP_LOG2E);
        m = mn;
        float zs[4] = {};
#pragma unroll
        for (int i = 0; i < 16; i++) zs[i % 4] += __builtin_amdgcn_exp2f((x[i] - m) * LP_LOG2E);
        z += (zs[0] + zs[1]) + (zs[2] + zs[3]);
    };
    const float4 none = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    const int off = r.sh ? 1 : 0, full = (n + r.sh) / 4;
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
    if (off) {   /* the cut quad of a row that is not aligned, which no thread counts among its own */
        v[0] = t == 0 ? r.load(0) : none;
        v[1] = v[2] = v[3] = none;
        take(v);
    }
    {   /* of T / 256 = 4 neighbours */
        uint32_t o = max(ord, (uint32_t)lg_partner<0>((int)ord));
        o = max(o, (uint32_t)lg_partner<1>((int)o));
        if (t % 4 == 0) s.top[t / 4] = o;
    }
    auto join = [&]() {   /* m, z over the wave */
        const float M = lg_group_max<64>(m);
        z = lg_group_sum<64>(z * __builtin_amdgcn_exp2f(fmaxf(m - M, -1e30f) * LP_LOG2E));
        m = M;
    };
    join();
    if (t % 64 == 0) s.sums[t / 64] = make_float4(m, z, 0.0f, 0.0f);
    __syncthreads();
    {
        const float4 y = t % 64 < T / 64 ? s.sums[t % 64] : make_float4(-FLT_MAX, 0.0f, 0.0f, 0.0f);
        m = y.x;
        z = y.y;
        join();
    }
    const int64_t at = row * a.parts + part;
    if (t == 0) a.mz[at] = make_float2(m, z);
    const int top = min(a.top, n);
    const int c = lp_top<T>(s, r, nq, off, top, ord, z != z);
    lp_emit<T>(s, c, top, [&](int rank, uint64_t k) { a.keys[at * a.top + rank] = k - (uint32_t)first; });   /* (~id - first = ~(id + first)) */
}

constexpr int BM_HELD = 4096;    /* entries of a group's parts that its workgroup holds, as doubles and keys */
constexpr int BM_LISTS = 1024;   /* and parts */
constexpr int BM_VALS = 256;     /* candidates whose values lie side by side */

/* A group: log sums of its beams' parts, then every part's entries as scores in
 * double.  The first few entries of each part, `top` together at least, have a
 * top-th highest of their own, and only entries that are no lower than it are
 * compared with each other: places by counting, first a hundred or so, then
 * hardly more than `top`.  Bound by its chain: loads, an exponential and a
 * logarithm in double, six barriers: 5 to 8 us. */
constexpr int BM_GROUP_THREADS = 256;
__global__ __launch_bounds__(BM_GROUP_THREADS) void k_beam_group(BeamArgs a)
{
    constexpr int T = BM_GROUP_THREADS;
    extern __shared__ double s_score[];   /* [beams][parts][top] and, behind, their keys */
    __shared__ double s_off[LG_BEAMS_MAX], s_lse[LG_BEAMS_MAX], s_val[BM_VALS], s_least;
    union Lists {
        float2 mz[BM_LISTS];
        double z[BM_LISTS];
        uint16_t list[BM_HELD];
    };
    __shared__ Lists s;
    __shared__ int s_kind[LG_BEAMS_MAX], s_n;   /* 0: no candidates, 1: logits, 2: finished */
    const int64_t row0 = (int64_t)blockIdx.x * a.beams, key0 = row0 * a.parts * a.top;
    const int t = threadIdx.x, lists = a.beams * a.parts, n = lists * a.top, run = a.parts * a.top;
    uint64_t* const s_key = (uint64_t*)(s_score + n);
    if (t < a.beams) {
        const float sc = a.scores[row0 + t];
        s_kind[t] = !(fabsf(sc) <= FLT_MAX) ? 0 : a.done && a.done[row0 + t] ? 2 : 1;
        s_off[t] = (double)sc;
    }
    /* (what beams without logits left there is not used) */
    for (int l = t; l < lists; l += T) s.mz[l] = a.mz[row0 * a.parts + l];
    for (int i = t; i < n; i += T) {
        const uint64_t k = a.keys[key0 + i];
        s_score[i] = (double)lp_value(k);
        s_key[i] = k;
    }
    if (t == 0) {
        s_n = 0;
        s_least = -INFINITY;
    }
    __syncthreads();
    /* the parts' sums over their beam's maximum, an exponential a thread */
    auto top_of = [&](int b) {
        float M = -FLT_MAX;
        for (int p = 0; p < a.parts; p++) M = fmaxf(M, s.mz[b * a.parts + p].x);
        return M;
    };
    double z[BM_LISTS / T];
#pragma unroll
    for (int k = 0; k < BM_LISTS / T; k++) {
        const int l = t + k * T;
        z[k] = l < lists ? s.mz[l].y * (a.parts > 1 ? exp((double)s.mz[l].x - (double)top_of(l / a.parts)) : 1.0) : 0.0;
    }
    const float M = t < a.beams ? top_of(t) : 0.0f;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < BM_LISTS / T; k++)
        if (t + k * T < lists) s.z[t + k * T] = z[k];
    __syncthreads();
    if (t < a.beams) {
        double sum = 0.0;
        for (int p = 0; p < a.parts; p++) sum += s.z[t * a.parts + p];
        const double lse = (double)M + log(sum);
        s_lse[t] = lse;
        if (s_kind[t] == 1 && !(fabs(lse) <= (double)FLT_MAX)) s_kind[t] = 0;   /* (NaN, infinities) */
    }
    __syncthreads();
    for (int i = t; i < n; i += T) {
        const int b = i / run, in = i - b * run, part = in / a.top, at = in - part * a.top;
        const int held = min(a.top, min(a.part, a.vocab - part * a.part));
        double v = -INFINITY;
        if (s_kind[b] == 1 && at < held) v = s_off[b] + (s_score[i] - s_lse[b]);
        if (s_kind[b] == 2 && in == 0) {
            v = s_off[b];
            s_key[i] = ~(uint32_t)a.end;
        }
        s_score[i] = v;
    }
    /* place of entry i, value v, among the c entries of s.list: those that are higher, or equal and of a lower beam or,
     * of the same one, of a higher key (logit, then token), whatever parts they come from.  Eight values at a time, no
     * branches (16 entries of 8 beams: 12 us with them), whatever lies behind the c-th being -infinity; equal values are
     * rare and looked at again. */
    auto place = [&](int c, int i, double v) __attribute__((always_inline)) {
        int rank = 0, same = 0;
        const int fast = min(c, BM_VALS);
        for (int o = 0; o < fast; o += 8)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const double w = s_val[o + e];
                rank += w > v ? 1 : 0;
                same += w == v ? 1 : 0;
            }
        for (int o = fast; o < c; o++) {
            const double w = s_score[s.list[o]];
            rank += w > v ? 1 : 0;
            same += w == v ? 1 : 0;
        }
        if (same > 1) {
            const int first = i / run * run;   /* the beam's entries */
            const uint64_t key = s_key[i];
#pragma unroll 4
            for (int o = 0; o < c; o++) {
                const int j = s.list[o];
                const double w = s_score[j];
                const uint64_t k = s_key[j];
                rank += (w == v) & ((j < first) | ((j < first + run) & (k > key))) ? 1 : 0;
            }
        }
        return rank;
    };
    auto gather = [&](int c) {
        for (int k = t; k < BM_VALS; k += T) s_val[k] = k < c ? s_score[s.list[k]] : -INFINITY;
    };
    const int each = (a.top + lists - 1) / lists, heads = each * lists;   /* (fewer than top + lists) */
    __syncthreads();
    for (int k = t; k < heads; k += T) s.list[k] = (uint16_t)(k / each * a.top + k % each);
    __syncthreads();
    gather(heads);
    __syncthreads();
    for (int k = t; k < heads; k += T) {
        const int i = s.list[k];
        const double v = s_score[i];
        if (v > -INFINITY && place(heads, i, v) == a.top - 1) s_least = v;
    }
    __syncthreads();
    const double least = s_least;   /* (-infinity: fewer than `top` of them are any) */
    for (int i = t; i < n; i += T) {
        const double v = s_score[i];
        if (v > -INFINITY && v >= least) s.list[atomicAdd(&s_n, 1)] = (uint16_t)i;   /* (in whatever order: ranked below) */
    }
    __syncthreads();
    const int cand = s_n;
    gather(cand);
    __syncthreads();
    for (int k = t; k < cand; k += T) {
        const int i = s.list[k];
        const double v = s_score[i];
        const int rank = place(cand, i, v);
        if (rank < a.top) {
            const int64_t at = (int64_t)blockIdx.x * a.top + rank;
            a.score[at] = (float)v;
            a.parent[at] = i / run;
            a.token[at] = (int)~(uint32_t)s_key[i];
        }
    }
    if (t >= cand && t < a.top) {
        const int64_t at = (int64_t)blockIdx.x * a.top + t;
        a.score[at] = -INFINITY;
        a.parent[at] = -1;
        a.token[at] = -1;
    }
}

/* Parts of a row: enough of them for the 256 CUs, of 16384 logits at least (4 rows of
 * 151936 whole 17.4 us, in parts of 4096 16.5, of 16384 12.4; 35 of 50257 13.8,
 * 16.4, 12.6; 240 of 32000 13.9, 15.8, 13.7); and the entries of a group's parts,
 * which a workgroup holds with their keys, at most 4096 (more where one part a beam
 * has them). */
static int bm_parts(int64_t rows, int beams, int vocab, int top)
{
    const int64_t want = std::max<int64_t>(1, 512 / std::max<int64_t>(rows, 1));
    return (int)std::max<int64_t>(1, std::min({want, (int64_t)vocab / 16384, (int64_t)BM_HELD / ((int64_t)beams * top),
                                                  (int64_t)BM_LISTS / beams}));
}

static bool bm_sizes(int ngroups, int beams, int vocab, int top)
{
    return ngroups >= 0 && beams > 0 && beams <= LG_BEAMS_MAX && top > 0 && top <= LG_BEAMS_MAX && vocab > 0 &&
           vocab <= INT32_MAX - 16;
}

extern "C" size_t lg_beam_select_workspace_size(int ngroups, int beams, int vocab, int top)
{
    if (!bm_sizes(ngroups, beams, vocab, top)) return 0;
    const int64_t rows = (int64_t)ngroups * beams;
    return (size_t)rows * bm_parts(rows, beams, vocab, top) * (sizeof(float2) + 8 * (size_t)top);
}

extern "C" int lg_beam_select(const float* logits, int64_t stride, const float* scores, const int* done, int end, int ngroups,
                              int beams, int vocab, int top, float* score, int* parent, int* token, void* workspace,
                              size_t workspace_bytes, void* stream)
{
    const char* who = "lg_beam_select";
    if (!bm_sizes(ngroups, beams, vocab, top) || stride < vocab) {
        lg_set_error("%s: bad sizes (%d groups of %d beams, rows of %d, %lld apart, top %d)", who, ngroups, beams, vocab,
                     (long long)stride, top);
        return LG_ERR_ARG;
    }
    if (!ngroups) return LG_OK;
    if (!logits || ((uintptr_t)logits & 3) || !scores || !score || !parent || !token) {
        lg_set_error("%s: logits, scores and outputs must be given", who);
        return LG_ERR_ARG;
    }
    const int64_t rows = (int64_t)ngroups * beams;
    BeamArgs a = {logits, scores, done, stride, end, beams, vocab, top, bm_parts(rows, beams, vocab, top), 0, nullptr, nullptr,
                  score, parent, token};
    /* (parts begin 16 bytes apart, so that all are as aligned as the row; up to 512 of 16384 at least: none is empty) */
    a.part = (vocab / a.parts + 4) & ~3;
    if (!lg_grid_fits(rows * a.parts, BM_ROW_THREADS)) {
        lg_set_error("%s: %lld rows are too many for one call", who, (long long)rows);
        return LG_ERR_ARG;
    }
    const size_t need = lg_beam_select_workspace_size(ngroups, beams, vocab, top);
    if (!workspace || !lg_al16(workspace) || workspace_bytes < need) {
        lg_set_error("%s: workspace of %zu bytes, 16-byte aligned, %zu needed", who, workspace_bytes, need);
        return LG_ERR_ARG;
    }
    a.mz = (float2*)workspace;
    a.keys = (uint64_t*)(a.mz + rows * a.parts);
    hipStream_t s = (hipStream_t)stream;
    const int lists = beams * a.parts * top;
    k_beam_rows<<<(unsigned)(rows * a.parts), BM_ROW_THREADS, 0, s>>>(a);
    k_beam_group<<<ngroups, BM_GROUP_THREADS, lists * (sizeof(double) + sizeof(uint64_t)), s>>>(a);
    return lg_check_launch(who);
}

/* ---- the tables of chosen beams ---- */

struct ReorderArgs {
    int* table;
    int64_t tstride;
    const int *parent, *length;
    int beams, max_pages, n_pages, shift;
    int4* jobs;   /* of each sequence: copy rows 0 .. z - 1 of page x to page y */
};

constexpr int BM_ENTRIES = 64;   /* table entries of a group's beams that LDS holds at a time */

/* A group: who takes which part-filled page, then the full pages' entries.  Bound by its dependent loads, 2.5 to 5 us. */
__global__ __launch_bounds__(256) void k_beam_tables(ReorderArgs a)
{
    __shared__ int s_par[LG_BEAMS_MAX], s_page[LG_BEAMS_MAX], s_spare[LG_BEAMS_MAX], s_tab[LG_BEAMS_MAX][BM_ENTRIES];
    const int g = blockIdx.x, t = threadIdx.x, len = a.length[g];
    int* const table = a.table + (int64_t)g * a.beams * a.tstride;
    const bool on = len >= 0 && len <= a.max_pages << a.shift;
    const int n = on ? len >> a.shift : 0, rows = on ? len & ((1 << a.shift) - 1) : 0;
    if (t < a.beams) {
        const int p = a.parent[g * a.beams + t];
        s_par[t] = (uint32_t)p < (uint32_t)a.beams ? p : t;
        s_page[t] = rows ? table[t * a.tstride + n] : 0;
    }
    __syncthreads();
    if (t < 64) {   /* a lane a beam */
        const int par = t < a.beams ? s_par[t] : -1;
        bool first = true, none = true;
        for (int i = 0; i < a.beams; i++) {
            if (i < t && s_par[i] == par) first = false;
            if (s_par[i] == t) none = false;
        }
        const uint64_t below = ((uint64_t)1 << t) - 1;
        const uint64_t others = __builtin_amdgcn_ballot_w64(t < a.beams && !first);
        const uint64_t spare = __builtin_amdgcn_ballot_w64(t < a.beams && none);
        if (t < a.beams && none) s_spare[__builtin_popcountll(spare & below)] = s_page[t];
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        if (t < a.beams) {
            const int src = s_page[par], dst = first ? src : s_spare[__builtin_popcountll(others & below)];
            if (rows) table[t * a.tstride + n] = dst;
            const bool copy = rows && !first && (uint32_t)src < (uint32_t)a.n_pages && (uint32_t)dst < (uint32_t)a.n_pages && src != dst;
            a.jobs[g * a.beams + t] = make_int4(src, dst, copy ? rows : 0, 0);
        }
    }
    for (int e0 = 0; e0 < n; e0 += BM_ENTRIES) {
        const int w = min(BM_ENTRIES, n - e0);
        for (int i = t; i < a.beams * BM_ENTRIES; i += 256) {
            const int b = i / BM_ENTRIES, e = i % BM_ENTRIES;
            if (e < w) s_tab[b][e] = table[b * a.tstride + e0 + e];
        }
        __syncthreads();
        for (int i = t; i < a.beams * BM_ENTRIES; i += 256) {
            const int b = i / BM_ENTRIES, e = i % BM_ENTRIES, p = s_par[b];
            if (e < w && p != b) table[b * a.tstride + e0 + e] = s_tab[p][e];
        }
        __syncthreads();
    }
}

constexpr int BM_POOLS = 64;         /* layers a launch */
constexpr int BM_SLICE = 65536;      /* bytes that a workgroup moves at most (or 16 rows) */

struct CopyArgs {
    uint8_t* pool[BM_POOLS][2];
    const int4* jobs;
    LgKv c;
    int slice;   /* rows a workgroup */
};

/* rows of a page: [rows][n_kv][hd] fp16 are one run, 4-bit ones a run of codes and
 * one of pairs for each head.  Bound by scattered runs of a few KB, read and written:
 * 40 groups of 8 beams, 24 layers, 16 rows of 2 KB each on average, 335 MB in 88 us, 3.8
 * TB/s (a copy's 4.9); runs of 32 KB at most a workgroup, twice the loads ahead or
 * stores past the caches 95 to 99 us in all against 96.  Of 4 bits by the heads' short
 * runs one after the other, a fraction of the threads each: the same rows, 119 MB,
 * 46 us, 2.6 TB/s. */
__global__ __launch_bounds__(256) void k_beam_copy(CopyArgs a)
{
    const int4 j = a.jobs[blockIdx.x];
    const int r0 = blockIdx.z / 2 * a.slice, n = min(j.z - r0, a.slice);
    if (n <= 0) return;
    uint8_t* const p = a.pool[blockIdx.y][blockIdx.z % 2];
    const uint8_t* const src = p + (size_t)j.x * a.c.seq;
    uint8_t* const dst = p + (size_t)j.y * a.c.seq;
    auto run = [&](size_t at, int bytes) {   /* multiples of 4 from 16-byte addresses on */
        const int n = bytes / 16;
        const uint4* const x = (const uint4*)(src + at);
        uint4* const y = (uint4*)(dst + at);
        int i = threadIdx.x;
        for (; i + 3 * 256 < n; i += 4 * 256) {
            const uint4 v0 = x[i], v1 = x[i + 256], v2 = x[i + 512], v3 = x[i + 768];
            y[i] = v0;
            y[i + 256] = v1;
            y[i + 512] = v2;
            y[i + 768] = v3;
        }
        for (; i < n; i += 256) y[i] = x[i];
        i = 4 * n + threadIdx.x;
        if (i < bytes / 4) ((uint32_t*)y)[i] = ((const uint32_t*)x)[i];
    };
    if (a.c.type == LG_F16) run(lg_kv16_at(a.c, 0, r0), n * a.c.n_kv * a.c.hd * 2);
    else
        for (int g = 0; g < a.c.n_kv; g++) {
            run(lg_kv4_codes(a.c, g, r0), n * (a.c.hd / 2));
            run(lg_kv4_dm(a.c, g, r0), n * (a.c.hd / 8));
        }
}

extern "C" int lg_beam_reorder(const lg_kv_cache* pools, int n_pools, int n_pages, int32_t* table, int64_t table_stride,
                               int max_pages, const int* parent, const int* length, int ngroups, int beams, void* workspace,
                               size_t workspace_bytes, void* stream)
{
    const char* who = "lg_beam_reorder";
    if (!pools || n_pools < 1 || ngroups < 0 || beams < 1 || beams > LG_BEAMS_MAX) {
        lg_set_error("%s: bad argument (%d layers, %d groups of %d beams)", who, n_pools, ngroups, beams);
        return LG_ERR_ARG;
    }
    ReorderArgs r = {table, table_stride, parent, length, beams, max_pages, n_pages, 0, (int4*)workspace};
    CopyArgs c = {};
    for (int i = 0; i < n_pools; i++) {
        const lg_kv_pages p = {pools[i], n_pages, max_pages, table, table_stride};
        const int rc = lg_kv_pages_arg(&p, who, &c.c, &r.shift);
        if (rc) return rc;
        if (pools[i].type != pools[0].type || pools[i].n_ctx != pools[0].n_ctx || pools[i].n_kv_heads != pools[0].n_kv_heads ||
            pools[i].head_dim != pools[0].head_dim || pools[i].seq_bytes != pools[0].seq_bytes) {
            lg_set_error("%s: layer %d has other pages than the first", who, i);
            return LG_ERR_ARG;
        }
    }
    if (c.c.type == LG_F16 && c.c.hd % 2) {
        lg_set_error("%s: heads of %d values", who, c.c.hd);
        return LG_ERR_ARG;
    }
    if ((int64_t)c.c.n_ctx * c.c.n_kv * c.c.hd * 2 > INT32_MAX - 1024) {
        lg_set_error("%s: pages of %d rows of %d heads are too large", who, c.c.n_ctx, c.c.n_kv);
        return LG_ERR_ARG;
    }
    if (!ngroups) return LG_OK;
    if (!parent || !length) {
        lg_set_error("%s: parents and lengths must be given", who);
        return LG_ERR_ARG;
    }
    const int64_t nseq = (int64_t)ngroups * beams;
    if (!lg_grid_fits(nseq, 256)) {
        lg_set_error("%s: %lld sequences are too many for one call", who, (long long)nseq);
        return LG_ERR_ARG;
    }
    if (!workspace || !lg_al16(workspace) || workspace_bytes < (size_t)nseq * sizeof(int4)) {
        lg_set_error("%s: workspace of %zu bytes, 16-byte aligned, %zu needed", who, workspace_bytes, (size_t)nseq * sizeof(int4));
        return LG_ERR_ARG;
    }
    hipStream_t s = (hipStream_t)stream;
    k_beam_tables<<<ngroups, 256, 0, s>>>(r);
    c.jobs = r.jobs;
    const int64_t row = (int64_t)c.c.n_kv * (c.c.type == LG_F16 ? 2 * c.c.hd : c.c.hd / 2 + c.c.hd / 8);
    c.slice = (int)std::min<int64_t>(std::max<int64_t>((BM_SLICE / row) & ~15, 16), c.c.n_ctx);
    const unsigned slices = (c.c.n_ctx + c.slice - 1) / c.slice;
    for (int l = 0; l < n_pools; l += BM_POOLS) {
        const int n = std::min(BM_POOLS, n_pools - l);
        for (int i = 0; i < n; i++) {
            c.pool[i][0] = (uint8_t*)pools[l + i].k;
            c.pool[i][1] = (uint8_t*)pools[l + i].v;
        }
        k_beam_copy<<<dim3((unsigned)nseq, n, 2 * slices), 256, 0, s>>>(c);
    }
    return lg_check_launch(who);
}
