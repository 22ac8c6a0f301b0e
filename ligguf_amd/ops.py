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


def rope_table(rope_dim: int, base: float, scaling: int = L.ROPE_PLAIN, factor: float = 1.0, orig_ctx: int = 0, p0: float = 0.0,
               p1: float = 0.0):
    """lg_rope_table: (rope_dim / 2 frequencies as a CPU tensor, mscale)."""
    f = torch.empty(max(rope_dim, 0) // 2, dtype=torch.float32)
    m = C.c_float()
    check(load().lg_rope_table(scaling, rope_dim, base, factor, orig_ctx, p0, p1, f.data_ptr(), C.byref(m)))
    return f, m.value


def qk_norm_rope_tokens(q, k, v, pos, freq, head_dim: int, rope_dim: int = None, half: bool = False, qw=None, kw=None,
                        eps: float = 1e-6, mscale: float = 1.0, cache: KvCache = None, want_k: bool = False, q_out=None,
                        k_out=None):
    """lg_qk_norm_rope_tokens on q, k, v [nseq, ntok, heads * head_dim] (views of
    a fused q | k | v row are fine; q or, without a cache, v may be None) and pos
    [nseq, ntok]: the rotated queries and keys; keys only with want_k or k_out."""
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
    _on(i, load().lg_qk_norm_rope_tokens, *rq, *rqo, *rk, *rko, *rv, _vec(qw, head_dim, i, "qw"), _vec(kw, head_dim, i, "kw"),
        qd // head_dim, kd // head_dim, head_dim, rope_dim, 1 if half else 0, _vec(freq, rope_dim // 2, i, "freq"), mscale, eps, p,
        nseq, ntok, desc)
    return q_out, k_out


def kv_values(cache: KvCache, pos0: int = 0, npos: int = None):
    """lg_kv4_read: the fp16 values [nseq, npos, kv_dim] that rows pos0 .. of a
    KV4 cache stand for, keys and values."""
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
    if cache.index != i or cache.nseq != nseq:
        _refuse(f"cache: {nseq} sequences on GPU {i} wanted")
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
           "attention_cache", "Logprobs", "logprobs", "Q8_0", "Q8_K", "F32", "F16", "KV4"]
