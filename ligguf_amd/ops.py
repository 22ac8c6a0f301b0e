"""Per-op calls of the C-ABI on torch device tensors.

Names follow the reference's math layer (fast/lil_math.h:5-39).  torch only
supplies device memory and the stream: every call goes to libligguf_hip.so
and raises LgError on failure; there is no CPU path.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple

import torch

from . import lib as L
from .lib import BLOCK, F16, F32, KV4, Q8_0, Q8_K, LgError, check, load


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _p(t):
    if t is None:
        return None
    assert t.is_cuda and t.is_contiguous(), "device tensors must be contiguous CUDA tensors"
    return t.data_ptr()


def dequantize_row(t: int, x: torch.Tensor, n: int) -> torch.Tensor:
    y = torch.empty(n, dtype=torch.float32, device=x.device)
    check(load().lg_dequantize_row(t, _p(x), _p(y), n, _stream()))
    return y


def quantize_q8_0(x: torch.Tensor) -> torch.Tensor:
    n = x.numel()
    y = torch.empty(n // 32 * 34, dtype=torch.uint8, device=x.device)
    check(load().lg_quantize_q8_0(_p(x), n, _p(y), _stream()))
    return y


def quantize_q8_K(x: torch.Tensor) -> torch.Tensor:
    n = x.numel()
    y = torch.empty(n // 256 * 292, dtype=torch.uint8, device=x.device)
    check(load().lg_quantize_q8_K(_p(x), n, _p(y), _stream()))
    return y


def matvec(t: int, w: torch.Tensor, rsz: int, n: int, d: int, xq: torch.Tensor, out: torch.Tensor = None,
           accumulate: bool = False) -> torch.Tensor:
    if out is None:
        out = torch.empty(d, dtype=torch.float32, device=w.device)
    check(load().lg_matvec(t, _p(w), rsz, n, d, _p(xq), _p(out), 1 if accumulate else 0, _stream()))
    return out


def matmul_tokens(t: int, w: torch.Tensor, rsz: int, n: int, d: int, x: torch.Tensor) -> torch.Tensor:
    """lg_matmul_tokens: x [T, n] fp32 -> [T, d], each row quantized to the
    activation form of weight type t (Q8_K for the K-quants, else Q8_0)."""
    T = x.shape[0]
    out = torch.empty((T, d), dtype=torch.float32, device=w.device)
    check(load().lg_matmul_tokens(t, _p(w), rsz, n, d, _p(x), T, _p(out), _stream()))
    return out


def rmsnorm_quant(x: torch.Tensor, w: torch.Tensor, eps: float, qtype: int, want_float: bool = False):
    n = x.numel()
    if qtype == F32:
        q = None
        f = torch.empty(n, dtype=torch.float32, device=x.device)
        check(load().lg_rmsnorm_quant(_p(x), _p(w), n, eps, qtype, None, _p(f), _stream()))
        return f
    qk, bs = BLOCK[qtype]
    q = torch.empty((n + qk - 1) // qk * bs, dtype=torch.uint8, device=x.device)
    f = torch.empty(n, dtype=torch.float32, device=x.device) if want_float else None
    check(load().lg_rmsnorm_quant(_p(x), _p(w), n, eps, qtype, _p(q), _p(f), _stream()))
    return (q, f) if want_float else q


def qk_norm_rope_kv(q, k, v, qw, kw, n_heads, n_kv_heads, head_dim, rope_dim, pos, freq, eps, kc_row=None,
                    vc_row=None) -> None:
    check(load().lg_qk_norm_rope_kv(_p(q), _p(k), _p(v), _p(qw), _p(kw), n_heads, n_kv_heads, head_dim, rope_dim,
                                    pos, _p(freq), eps, _p(kc_row), _p(vc_row), _stream()))


def attention(q, k, v, kc, vc, n_heads, n_kv_heads, head_dim, pos, workspace: torch.Tensor = None) -> torch.Tensor:
    lib = load()
    need = lib.lg_attn_workspace_size(n_heads, head_dim, pos)
    if workspace is None:
        workspace = torch.empty(max(need, 16), dtype=torch.uint8, device=q.device)
    out = torch.empty(n_heads * head_dim, dtype=torch.float32, device=q.device)
    check(lib.lg_attn_decode(_p(q), _p(k), _p(v), _p(kc), _p(vc), n_heads, n_kv_heads, head_dim, pos, _p(out),
                             _p(workspace), workspace.numel(), _stream()))
    return out


def swiglu_quant(hb: torch.Tensor, hb2: torch.Tensor, qtype: int = Q8_K):
    n = hb.numel()
    if qtype == F32:
        check(load().lg_swiglu_quant(_p(hb), _p(hb2), n, qtype, None, _stream()))
        return None
    qk, bs = BLOCK[qtype]
    q = torch.empty((n + qk - 1) // qk * bs, dtype=torch.uint8, device=hb.device)
    check(load().lg_swiglu_quant(_p(hb), _p(hb2), n, qtype, _p(q), _stream()))
    return q


# --------------------------------------------------------------------------
# many tokens and long contexts
# --------------------------------------------------------------------------
# A serving loop makes these calls once per layer and token: each costs the host a few
# microseconds beside the launches themselves, so the checks below read a tensor's fields once.
_FP32, _INT32, _DENSE = torch.float32, torch.int32, torch.contiguous_format
_raw_stream = torch._C._cuda_getCurrentRawStream     # current_stream(i).cuda_stream without the Stream object


def _refuse(msg):
    raise LgError(f"LG_ERR_ARG: {msg}")


def _on(i, fn, *args):
    """fn(*args, stream) on device i and its current stream."""
    if i == torch.cuda.current_device():
        rc = fn(*args, _raw_stream(i))
    else:
        with torch.cuda.device(i):
            rc = fn(*args, _raw_stream(i))
    if rc:
        check(rc)


def _rows(t, i, nseq, ntok, width, name):
    """(pointer, floats from row to row) of fp32 rows [nseq, ntok, width] on
    device i; the last axis is dense and the first two are one run of rows."""
    if t.dtype is not _FP32 or t.get_device() != i or t.shape != (nseq, ntok, width):
        _refuse(f"{name}: fp32 [{nseq}, {ntok}, {width}] on GPU {i} wanted, {t.dtype} {tuple(t.shape)} on {t.device} given")
    s0, s1, s2 = t.stride()
    if not (nseq and ntok and width):
        return None, (width + 3) // 4 * 4
    row = s1 if ntok > 1 else s0 if nseq > 1 else (width + 3) // 4 * 4
    if (s2 != 1 and width > 1) or (nseq > 1 and s0 != row * ntok):
        _refuse(f"{name}: rows of strides {t.stride()} are not one run")
    return t.data_ptr(), row


def _fresh(like, rows, width):
    """A dense tensor like `like` (whose last axis is `width`; rows of a width that is no multiple of four are
    padded to one) and its (pointer, floats from row to row)."""
    wide = (width + 3) // 4 * 4
    if wide != width and rows > 1:
        t = like.new_empty((*like.shape[:-1], wide))[..., :width]
    else:
        t = torch.empty_like(like, memory_format=_DENSE)
    return t, (t.data_ptr(), wide)


def _pos(pos):
    if pos.dtype is not _INT32 or not pos.is_cuda or pos.dim() != 2 or not pos.is_contiguous():
        _refuse("pos: contiguous int32 [nseq, ntok] on the GPU wanted")
    return pos.data_ptr()


def _vec(t, n, i, name):
    if t is None:
        return None
    if t.dtype is not _FP32 or t.get_device() != i or not t.is_contiguous() or t.numel() < n:
        _refuse(f"{name}: {n} contiguous fp32 values on GPU {i} wanted")
    return t.data_ptr()


class KvCache:
    """One layer's keys and values of nseq sequences (lg_kv_cache): F16 tensors
    [nseq, n_ctx, n_kv_heads * head_dim] -- a context's own cache has that form
    -- or KV4 bytes [nseq, lg_kv_bytes or more, a multiple of 16 for several sequences]."""

    def __init__(self, k, v, n_kv_heads: int, head_dim: int, type: int = F16, n_ctx: int = None):
        if n_ctx is None:
            if type != F16 or k.dim() != 3:
                _refuse("n_ctx is needed for a cache that is not fp16 [nseq, n_ctx, kv_dim]")
            n_ctx = k.shape[1]
        need = load().lg_kv_bytes(type, n_ctx, n_kv_heads, head_dim)
        if need < 0:
            _refuse(f"no cache of type {type}, {n_ctx} rows, {n_kv_heads} heads of {head_dim}")
        want = torch.float16 if type == F16 else torch.uint8
        i, shape = k.get_device(), k.shape
        if (k.dtype is not want or v.dtype is not want or i < 0 or v.get_device() != i or v.shape != shape or not k.is_contiguous()
                or not v.is_contiguous()):
            _refuse(f"k and v: contiguous {want} tensors of one shape on one GPU wanted")
        nseq = shape[0] if len(shape) > 1 else 0
        size = k.nbytes // nseq if nseq else -1
        if size < need or (type == F16 and size != need):
            _refuse(f"k and v: {need} bytes a sequence wanted, shape {tuple(shape)} given")
        self.k, self.v, self.type, self.n_ctx, self.nseq = k, v, type, n_ctx, nseq
        self.n_kv_heads, self.head_dim, self.index = n_kv_heads, head_dim, i
        self.desc = L.LgKvCache(k.data_ptr(), v.data_ptr(), type, n_ctx, n_kv_heads, head_dim, size)

    @classmethod
    def empty(cls, type: int, n_ctx: int, n_kv_heads: int, head_dim: int, nseq: int = 1, device="cuda") -> "KvCache":
        """A cache of zeros."""
        need = load().lg_kv_bytes(type, n_ctx, n_kv_heads, head_dim)
        if need < 0 or nseq < 1:
            _refuse(f"no cache of type {type}, {nseq} x {n_ctx} rows, {n_kv_heads} heads of {head_dim}")
        shape, dt = ((nseq, n_ctx, n_kv_heads * head_dim), torch.float16) if type == F16 else ((nseq, (need + 15) // 16 * 16), torch.uint8)
        return cls(*(torch.zeros(shape, dtype=dt, device=device) for _ in range(2)), n_kv_heads, head_dim, type, n_ctx)


class PagedKvCache:
    """One layer's keys and values of many sequences in pages of `page` rows
    (lg_kv_pages): F16 pools [n_pages, page, n_kv_heads * head_dim] or KV4 bytes
    [n_pages, lg_kv_bytes of a page or more, a multiple of 16], and an int32
    table [nseq, max_pages] of page numbers (-1: no page), whose rows may be
    part of longer ones.  `pool` is the pages as a KvCache, a page per sequence."""

    def __init__(self, k, v, table, n_kv_heads: int, head_dim: int, type: int = F16, page: int = None):
        self.pool = p = KvCache(k, v, n_kv_heads, head_dim, type, page)
        if (table.dtype is not _INT32 or table.get_device() != p.index or table.dim() != 2 or not table.numel()
                or (table.shape[1] > 1 and table.stride(1) != 1)):
            _refuse(f"table: int32 [nseq, max_pages] with dense rows on GPU {p.index} wanted")
        self.k, self.v, self.table, self.type, self.page, self.n_pages = k, v, table, type, p.n_ctx, p.nseq
        self.nseq, self.max_pages = table.shape
        self.n_kv_heads, self.head_dim, self.index, self.n_ctx = n_kv_heads, head_dim, p.index, self.max_pages * p.n_ctx
        stride = table.stride(0) if self.nseq > 1 else self.max_pages
        self.desc = L.LgKvPages(p.desc, p.nseq, self.max_pages, table.data_ptr(), stride)

    @classmethod
    def empty(cls, type: int, n_pages: int, page: int, n_kv_heads: int, head_dim: int, table) -> "PagedKvCache":
        """Pages of zeros on the table's device."""
        c = KvCache.empty(type, page, n_kv_heads, head_dim, n_pages, table.device)
        return cls(c.k, c.v, table, n_kv_heads, head_dim, type, page)


class PagedLayers:
    """The caches of a model's layers that have one table: what beam_reorder moves."""

    def __init__(self, caches):
        c = caches[0] if caches else _refuse("no layers")
        for x in caches:
            if (not isinstance(x, PagedKvCache) or x.table.data_ptr() != c.table.data_ptr() or x.table.shape != c.table.shape or x.table.stride() != c.table.stride()
                    or (x.type, x.page, x.n_pages, x.n_kv_heads, x.head_dim) != (c.type, c.page, c.n_pages, c.n_kv_heads, c.head_dim)):
                _refuse("layers of one table and pages of one form wanted")
        self.caches, self.table, self.index, self.nseq = list(caches), c.table, c.index, c.nseq
        self.desc = (L.LgKvCache * len(caches))(*(x.pool.desc for x in caches))
        self.args = (self.desc, len(caches), c.n_pages, c.table.data_ptr(), c.desc.table_stride, c.max_pages)


def rope_table(rope_dim: int, base: float, scaling: int = L.ROPE_PLAIN, factor: float = 1.0, orig_ctx: int = 0, p0: float = 0.0,
               p1: float = 0.0):
    """lg_rope_table: (rope_dim / 2 frequencies as a CPU tensor, mscale)."""
    f = torch.empty(max(rope_dim, 0) // 2, dtype=torch.float32)
    m = C.c_float()
    check(load().lg_rope_table(scaling, rope_dim, base, factor, orig_ctx, p0, p1, f.data_ptr(), C.byref(m)))
    return f, m.value


def qk_norm_rope_tokens(q, k, v, pos, freq, head_dim: int, rope_dim: int = None, half: bool = False, qw=None, kw=None,
                        eps: float = 1e-6, mscale: float = 1.0, cache=None, want_k: bool = False, q_out=None, k_out=None):
    """lg_qk_norm_rope_tokens on q, k, v [nseq, ntok, heads * head_dim] (views of
    a fused q | k | v row are fine; q or, without a cache, v may be None) and pos
    [nseq, ntok]: the rotated queries and keys; keys only with want_k or k_out.
    cache: a KvCache, or a PagedKvCache (lg_qk_norm_rope_paged)."""
    rope_dim = head_dim if rope_dim is None else rope_dim
    p, i = _pos(pos), pos.get_device()
    nseq, ntok = pos.shape
    kd = k.shape[-1]
    qd = 0 if q is None else q.shape[-1]
    if head_dim < 1 or kd % head_dim or qd % head_dim:
        _refuse(f"rows of {qd} and {kd} values are no heads of {head_dim}")
    at = (i, nseq, ntok)
    if q is None:
        q_out, rq, rqo = None, (None, 0), (None, 0)
    else:
        rq = _rows(q, *at, qd, "q")
        q_out, rqo = _fresh(q, nseq * ntok, qd) if q_out is None else (q_out, _rows(q_out, *at, qd, "q_out"))
    rk = _rows(k, *at, kd, "k")
    if k_out is not None:
        rko = _rows(k_out, *at, kd, "k_out")
    elif want_k:
        k_out, rko = _fresh(k, nseq * ntok, kd)
    else:
        rko = (None, 0)
    if cache is None:
        rv, desc = (None, 0), None
    else:
        if cache.index != i or cache.nseq != nseq or v is None:
            _refuse(f"cache: values and {nseq} sequences on GPU {i} wanted")
        rv, desc = _rows(v, *at, kd, "v"), C.byref(cache.desc)
    lib = load()
    fn = lib.lg_qk_norm_rope_paged if isinstance(cache, PagedKvCache) else lib.lg_qk_norm_rope_tokens
    _on(i, fn, *rq, *rqo, *rk, *rko, *rv, _vec(qw, head_dim, i, "qw"), _vec(kw, head_dim, i, "kw"),
        qd // head_dim, kd // head_dim, head_dim, rope_dim, 1 if half else 0, _vec(freq, rope_dim // 2, i, "freq"), mscale, eps, p,
        nseq, ntok, desc)
    return q_out, k_out


def kv_values(cache: KvCache, pos0: int = 0, npos: int = None):
    """lg_kv4_read: the fp16 values [nseq, npos, kv_dim] that rows pos0 .. of a
    KV4 cache stand for, keys and values."""
    if isinstance(cache, PagedKvCache):
        _refuse("cache: a KvCache wanted (of pages: cache.pool)")
    npos = cache.n_ctx - pos0 if npos is None else npos
    if npos < 0:
        _refuse(f"{npos} rows")
    shape = (cache.nseq, npos, cache.n_kv_heads * cache.head_dim)
    k = cache.k.new_empty(shape, dtype=torch.float16)
    v = torch.empty_like(k)
    if npos:
        _on(cache.index, load().lg_kv4_read, C.byref(cache.desc), cache.nseq, pos0, npos, k.data_ptr(), v.data_ptr())
    return k, v


def _work(need, workspace, like):
    """The workspace of a call beside `like`, a new one unless given, and its (pointer, bytes)."""
    if workspace is None:
        if not need:
            return None, (None, 0)
        workspace = like.new_empty((need + 3) // 4)
    elif workspace.get_device() != like.get_device() or not workspace.is_contiguous():
        _refuse(f"workspace: contiguous memory on {like.device} wanted")
    return workspace, (workspace.data_ptr(), workspace.numel() * workspace.element_size())


def attention_cache(q, cache: KvCache, pos, window: int = 0, sinks: int = 0, max_pos: int = None, out=None, workspace=None):
    """lg_attn_cache: q [nseq, ntok, n_heads * head_dim] at pos [nseq, ntok] over
    the cache rows that each position sees.  max_pos, a bound of the positions
    (n_ctx - 1 by default), sizes the launch."""
    p, i = _pos(pos), pos.get_device()
    nseq, ntok = pos.shape
    if isinstance(cache, PagedKvCache) or cache.index != i or cache.nseq != nseq:
        _refuse(f"cache: a KvCache of {nseq} sequences on GPU {i} wanted")
    max_pos = cache.n_ctx - 1 if max_pos is None else max_pos
    width, hd = q.shape[-1], cache.head_dim
    heads = width // hd
    if heads * hd != width:
        _refuse(f"rows of {width} values are no heads of {hd}")
    rows = _rows(q, i, nseq, ntok, width, "q")
    out, ro = _fresh(q, nseq * ntok, width) if out is None else (out, _rows(out, i, nseq, ntok, width, "out"))
    lib, desc = load(), C.byref(cache.desc)
    workspace, ws = _work(lib.lg_attn_cache_workspace_size(desc, nseq, ntok, heads, window, sinks, max_pos), workspace, q)
    _on(i, lib.lg_attn_cache, *rows, desc, p, nseq, ntok, heads, window, sinks, max_pos, *ro, *ws)
    return out


def attention_paged(q, cache: PagedKvCache, pos, window: int = 0, sinks: int = 0, max_pos: int = None, prefix=None,
                    max_prefix: int = None, out=None, workspace=None):
    """lg_attn_paged: attention_cache over pages.  prefix, int32 [groups] on the GPU
    (nseq is a multiple of groups): the sequences of a group share so many first
    rows, which lie in the pages of its first one and are read once for all;
    max_prefix, a bound of them (max_pos + 1 by default), sizes the launch with max_pos: the own rows are cut for
    max_pos - max_prefix + 1, by default for one, so that many of them run in a single part.  Pass it where it is known
    (four sequences, 2000 shared and 3000 own rows: 23 us with it, 54 without)."""
    p, i = _pos(pos), pos.get_device()
    nseq, ntok = pos.shape
    if not isinstance(cache, PagedKvCache) or cache.index != i or cache.nseq != nseq:
        _refuse(f"cache: a PagedKvCache of {nseq} sequences on GPU {i} wanted")
    max_pos = cache.n_ctx - 1 if max_pos is None else max_pos
    group, pp = 1, None
    if prefix is None:
        max_prefix = 0
    else:
        groups = prefix.numel()
        if prefix.dtype is not _INT32 or prefix.get_device() != i or not prefix.is_contiguous() or not groups or nseq % groups:
            _refuse(f"prefix: contiguous int32 on GPU {i} wanted, one for each group of {nseq} sequences")
        group, pp = nseq // groups or 1, prefix.data_ptr()
        max_prefix = max_pos + 1 if max_prefix is None else max_prefix
    width, hd = q.shape[-1], cache.head_dim
    heads = width // hd
    if heads * hd != width:
        _refuse(f"rows of {width} values are no heads of {hd}")
    rows = _rows(q, i, nseq, ntok, width, "q")
    out, ro = _fresh(q, nseq * ntok, width) if out is None else (out, _rows(out, i, nseq, ntok, width, "out"))
    lib, desc = load(), C.byref(cache.desc)
    need = lib.lg_attn_paged_workspace_size(desc, nseq, ntok, heads, window, sinks, max_pos, group, max_prefix)
    workspace, ws = _work(need, workspace, q)
    _on(i, lib.lg_attn_paged, *rows, desc, p, nseq, ntok, heads, window, sinks, max_pos, pp, group, max_prefix, *ro, *ws)
    return out


class BeamChoice(NamedTuple):
    score: torch.Tensor          # fp32 [groups, top], the highest first
    parent: torch.Tensor         # int32: the beam that each goes on from, -1: none
    token: torch.Tensor          # int32


def beam_select(logits, scores, top: int, done=None, end: int = -1, workspace=None) -> BeamChoice:
    """lg_beam_select of logits [groups, beams, vocab] (dense rows, one run of
    them) and scores [groups, beams]: the `top` best continuations of each group.
    done, int32 [groups, beams]: beams that have ended (with the token `end`)."""
    if logits.dtype is not _FP32 or not logits.is_cuda or logits.dim() != 3:
        _refuse("logits: fp32 [groups, beams, vocab] on the GPU wanted")
    i, (groups, beams, vocab) = logits.get_device(), logits.shape
    s0, s1, s2 = logits.stride()
    row = s1 if beams > 1 else s0 if groups > 1 else vocab
    if (s2 != 1 and vocab > 1) or (groups > 1 and s0 != row * beams):
        _refuse(f"logits: rows of strides {logits.stride()} are not one run")
    for t, dt, name in ((scores, _FP32, "scores"), (done, _INT32, "done")):
        if t is None and name == "done":
            continue
        if t.dtype is not dt or t.get_device() != i or t.shape != (groups, beams) or not t.is_contiguous():
            _refuse(f"{name}: contiguous {dt} [{groups}, {beams}] on {logits.device} wanted")
    if top < 1:
        _refuse(f"top {top}")
    lib, new = load(), logits.new_empty
    score = new((groups, top))
    both = torch.empty((2, groups, top), dtype=_INT32, device=logits.device)
    parent, token = both.unbind()
    workspace, ws = _work(lib.lg_beam_select_workspace_size(groups, beams, vocab, top), workspace, logits)
    _on(i, lib.lg_beam_select, logits.data_ptr(), row, scores.data_ptr(), None if done is None else done.data_ptr(), end, groups, beams,
        vocab, top, score.data_ptr(), parent.data_ptr(), token.data_ptr(), *ws)
    return BeamChoice(score, parent, token)


def beam_reorder(layers: PagedLayers, parent, length, workspace=None) -> None:
    """lg_beam_reorder, in place: the sequences go on from `parent` (int32 [groups,
    beams], beams of their group) with length rows each (int32 [groups])."""
    i = layers.index
    for t, name in ((parent, "parent"), (length, "length")):
        if t.dtype is not _INT32 or t.get_device() != i or not t.is_contiguous():
            _refuse(f"{name}: contiguous int32 on GPU {i} wanted")
    if parent.dim() != 2 or length.shape != parent.shape[:1] or parent.numel() != layers.nseq:
        _refuse(f"parent {tuple(parent.shape)}, length {tuple(length.shape)}: {layers.nseq} sequences in groups wanted")
    workspace, ws = _work(16 * layers.nseq, workspace, parent)
    _on(i, load().lg_beam_reorder, *layers.args, parent.data_ptr(), length.data_ptr(), *parent.shape, *ws)


class Logprobs(NamedTuple):
    logprob: torch.Tensor        # [rows], None without tokens
    entropy: torch.Tensor        # [rows]
    top_id: torch.Tensor         # [rows, top], None for top 0
    top_logprob: torch.Tensor


def logprobs(logits, toks=None, top: int = 0) -> Logprobs:
    """lg_logprobs of logits [rows, vocab] (dense rows) and int32 toks [rows]."""
    if logits.dtype is not _FP32 or not logits.is_cuda or logits.dim() != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        _refuse("logits: dense fp32 rows on the GPU wanted")
    i, (rows, vocab) = logits.get_device(), logits.shape
    if toks is not None and (toks.dtype is not _INT32 or toks.get_device() != i or toks.shape != (rows,) or not toks.is_contiguous()):
        _refuse(f"toks: {rows} contiguous int32 on {logits.device} wanted")
    if top < 0:
        _refuse(f"top {top}")
    new = logits.new_empty
    entropy = new(rows)
    lp, pt, pl = (None, None, None) if toks is None else (t := new(rows), toks.data_ptr(), t.data_ptr())
    top_id = top_lp = None
    if top:
        top_lp = new((rows, top))
        top_id = torch.empty_like(top_lp, dtype=_INT32)
    _on(i, load().lg_logprobs, logits.data_ptr(), logits.stride(0) if rows > 1 else vocab, rows, vocab, pt, top, pl, entropy.data_ptr(),
        top_id.data_ptr() if top else None, top_lp.data_ptr() if top else None)
    return Logprobs(lp, entropy, top_id, top_lp)


__all__ = ["dequantize_row", "quantize_q8_0", "quantize_q8_K", "matvec", "rmsnorm_quant", "qk_norm_rope_kv",
           "attention", "swiglu_quant", "KvCache", "rope_table", "qk_norm_rope_tokens", "kv_values",
           "attention_cache", "PagedKvCache", "PagedLayers", "attention_paged", "BeamChoice", "beam_select", "beam_reorder", "Logprobs", "logprobs", "Q8_0", "Q8_K", "F32", "F16", "KV4"]
