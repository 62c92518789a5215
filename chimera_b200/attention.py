"""Generation over cached keys and values: rotary positions, a paged
key-value cache that is quantised as it is written, and the attention of one
new token over it (include/chimera_b200.h, chm_rotary to chm_paged_attention).

A reader that answers from retrieved documents keeps their key and value
vectors in such a cache.  Its step for a batch of sequences:

    q, k = rotary(q, k, positions, freqs)
    cache_write(k, v, slots, k_pages, v_pages, k_scale, v_scale)
    out, lse = paged_attention(q, k_pages, v_pages, tables, lens, k_scale, v_scale)

Pages are tensors [num_pages, heads, page_size, dim] (any strides that are
multiples of 16 bytes, 1 along dim; k and v alike): fp16 or bf16, or int8 or
float8_e4m3fn with scales [num_pages, heads, page_size].  Token s of the cache,
its slot, is in page s // page_size at s % page_size.

Every call runs on `stream` (default: the current stream of its tensors'
device), allocates its outputs where none are given, never synchronises, and
can be captured into a CUDA graph.  Arguments that do not fit raise TypeError
or ValueError before anything is launched.
"""
from __future__ import annotations

import ctypes as C
import math

import torch

from . import capi

_FLOAT = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_HELD = {torch.float16: 1, torch.bfloat16: 2, torch.int8: 3, torch.float8_e4m3fn: 4}
_SCALED = (torch.int8, torch.float8_e4m3fn)
KINDS = {"plain": 0, "linear": 1, "base": 2, "parts": 3}


def _check(status, where):
    if status == capi.CHM_ERR_INVALID:
        raise ValueError(capi.lib().chm_last_error().decode() or where)
    capi.check(status, where)


def _on(device, x, name):
    if x.device != device:
        raise ValueError(f"{name} is on {x.device}, not on {device}")


class _Device:
    """The tensors' device made current for a call, where it is not yet."""

    def __init__(self, x, name, stream):
        if not isinstance(x, torch.Tensor) or not x.is_cuda:
            raise TypeError(f"{name} must be a CUDA tensor")
        self.device = x.device
        if stream is not None and stream.device != x.device:
            raise ValueError(f"the stream is on {stream.device}, not on {x.device}")
        self.stream = stream

    def __enter__(self):
        self.before = torch.cuda.current_device()
        if self.before != self.device.index:
            torch.cuda.set_device(self.device)
        return (self.stream or torch.cuda.current_stream()).cuda_stream

    def __exit__(self, *_):
        if self.before != self.device.index:
            torch.cuda.set_device(self.before)


def _heads(x, name, dims):
    """[batch, tokens, heads, dim], [tokens, heads, dim] or [batch, heads, dim]
    as a chm_heads (`dims`: what the axes before the last two are)."""
    if x.dim() != len(dims) + 2:
        raise ValueError(f"{name} must have {len(dims) + 2} axes")
    st = x.stride()
    if x.shape[-1] > 1 and st[-1] != 1 and x.numel():
        raise ValueError(f"the last axis of {name} must be contiguous")
    at = dict(zip(dims, st))
    return capi.ChmHeads(x.data_ptr(), x.shape[-2], at.get("batch", 0), at.get("token", 0), st[-2])


def _out_like(out, shape, dtype, device, name):
    if out is None:
        return torch.empty(shape, dtype=dtype, device=device)
    _on(device, out, name)
    if tuple(out.shape) != tuple(shape) or out.dtype != dtype:
        raise ValueError(f"{name} must be {dtype} of shape {tuple(shape)}")
    return out


def rotary_frequencies(rot_dim, base=10000.0, *, kind="plain", factor=1.0, original_len=4096, slow=1.0, fast=32.0,
                       device=None):
    """Rotation frequencies (float64 [rot_dim / 2], radians per position) for
    `rotary`, for contexts up to `factor` times longer than `original_len`:
    "plain" (unscaled), "linear" (all divided by the factor), "base" (a larger
    base) or "parts" (pairs that turn more than `fast` times over original_len
    as they are, fewer than `slow` times divided, a ramp between)."""
    if kind not in KINDS:
        raise ValueError(f"kind must be one of {sorted(KINDS)}")
    rot_dim = int(rot_dim)
    out = torch.empty(max(rot_dim, 0) // 2, dtype=torch.float64)
    _check(capi.lib().chm_rotary_frequencies(rot_dim, base, KINDS[kind], factor, original_len, slow, fast,
                                             out.data_ptr() or None), "rotary_frequencies")
    return out.to(device) if device is not None else out


def rotary(q, k, positions, freqs, *, interleaved=False, inverse=False, scale=1.0, q_out=None, k_out=None,
           stream=None):
    """Rotate the first 2 * len(freqs) elements of every vector of q
    [batch, tokens, q_heads, dim] and k [batch, tokens, k_heads, dim] (or both
    [tokens, heads, dim]; k may be None) by positions * freqs, in one launch.

    positions: int64 or int32 [batch, tokens], [tokens] (shared by the batch);
    freqs: float64, from rotary_frequencies; scale multiplies sine and cosine.
    Pairs are (i, i + n/2), or neighbours with `interleaved`.  `inverse` turns
    back: the gradient with respect to q and k of the outputs' gradients, with
    the same scale.  q_out / k_out may be q and k themselves.  Returns
    (q_out, k_out)."""
    dev = _Device(q, "q", stream)
    if q.dtype not in _FLOAT:
        raise TypeError("q must be float32, float16 or bfloat16")
    if q.dim() not in (3, 4):
        raise ValueError("q must be [batch, tokens, heads, dim] or [tokens, heads, dim]")
    dims = ("batch", "token")[4 - q.dim():]
    batch = q.shape[0] if q.dim() == 4 else 1
    tokens, dim = q.shape[-3], q.shape[-1]
    if k is not None:
        if k.dtype != q.dtype:
            raise TypeError("k must have q's type")
        _on(q.device, k, "k")
        if k.dim() != q.dim() or k.shape[:-2] != q.shape[:-2] or k.shape[-1] != dim:
            raise ValueError("k must agree with q but for its heads")
    elif k_out is not None:
        raise ValueError("k_out without k")
    if positions.dtype not in (torch.int64, torch.int32):
        raise TypeError("positions must be int64 or int32")
    _on(q.device, positions, "positions")
    if positions.shape == (batch, tokens) and positions.dim() == 2:
        pb, pt = positions.stride()
    elif positions.shape == (tokens,):
        pb, pt = 0, positions.stride(0)
    else:
        raise ValueError("positions must be [batch, tokens] or [tokens]")
    if freqs.dtype != torch.float64 or freqs.dim() != 1 or not freqs.is_contiguous():
        raise TypeError("freqs must be a contiguous float64 vector")
    _on(q.device, freqs, "freqs")
    q_out = _out_like(q_out, q.shape, q.dtype, q.device, "q_out")
    n = 1
    src, dst = (capi.ChmHeads * 2)(), (capi.ChmHeads * 2)()
    src[0], dst[0] = _heads(q, "q", dims), _heads(q_out, "q_out", dims)
    if k is not None:
        k_out = _out_like(k_out, k.shape, k.dtype, k.device, "k_out")
        src[1], dst[1], n = _heads(k, "k", dims), _heads(k_out, "k_out", dims), 2
    with dev as st:
        _check(capi.lib().chm_rotary(src, dst, n, _FLOAT[q.dtype], batch, tokens, dim, 2 * freqs.shape[0],
                                     positions.data_ptr(), positions.element_size(), pb, pt, freqs.data_ptr(),
                                     scale, (1 if interleaved else 0) | (2 if inverse else 0), st), "rotary")
    return q_out, k_out


def _cache(k_pages, v_pages, k_scale, v_scale):
    if k_pages.dtype not in _HELD:
        raise TypeError("pages must be float16, bfloat16, int8 or float8_e4m3fn")
    if k_pages.dim() != 4:
        raise ValueError("pages must be [num_pages, heads, page_size, dim]")
    st = k_pages.stride()
    if v_pages.dtype != k_pages.dtype or v_pages.shape != k_pages.shape or v_pages.stride() != st:
        raise ValueError("k_pages and v_pages must be alike in type, shape and strides")
    _on(k_pages.device, v_pages, "v_pages")
    n, heads, size, dim = k_pages.shape
    if st[3] != 1 and dim > 1:
        raise ValueError("the last axis of the pages must be contiguous")
    scales = [None, None]
    if k_pages.dtype in _SCALED:
        for i, s in enumerate((k_scale, v_scale)):
            if s is None:
                raise ValueError("an 8-bit cache needs k_scale and v_scale")
            _on(k_pages.device, s, "scales")
            if s.dtype != torch.float32 or s.shape != (n, heads, size) or not s.is_contiguous():
                raise ValueError("scales must be contiguous float32 [num_pages, heads, page_size]")
            scales[i] = s.data_ptr()
    elif k_scale is not None or v_scale is not None:
        raise ValueError("a 16-bit cache has no scales")
    return capi.ChmKvCache(k_pages.data_ptr(), v_pages.data_ptr(), scales[0], scales[1], n, st[0], st[1], st[2],
                           size, heads, dim, _HELD[k_pages.dtype])


def _slots(slots, device):
    if slots.dtype != torch.int64 or slots.dim() != 1 or not slots.is_contiguous():
        raise TypeError("slots must be a contiguous int64 vector")
    _on(device, slots, "slots")
    return slots


def cache_write(k, v, slots, k_pages, v_pages, k_scale=None, v_scale=None, *, stream=None):
    """Write tokens' keys and values (k, v: [tokens, heads, dim], float32,
    float16 or bfloat16) to slots [tokens] (int64) of the cache; int8 and
    float8_e4m3fn pages get codes and one scale per vector (chm_cache_write).
    A slot outside the cache is skipped.  No slot may stand twice."""
    dev = _Device(k, "k", stream)
    cache = _cache(k_pages, v_pages, k_scale, v_scale)
    _on(k.device, k_pages, "k_pages")
    _on(k.device, v, "v")
    if k.dtype not in _FLOAT or v.dtype != k.dtype:
        raise TypeError("k and v must be float32, float16 or bfloat16, and alike")
    n = _slots(slots, k.device).shape[0]
    if k.shape != (n, cache.heads, cache.dim) or v.shape != k.shape:
        raise ValueError(f"k and v must be [{n}, {cache.heads}, {cache.dim}]")
    kh, vh = _heads(k, "k", ("token",)), _heads(v, "v", ("token",))
    with dev as st:
        _check(capi.lib().chm_cache_write(C.byref(cache), C.byref(kh), C.byref(vh), _FLOAT[k.dtype], n,
                                          slots.data_ptr(), st), "cache_write")


def cache_read(slots, k_pages, v_pages, k_scale=None, v_scale=None, *, dtype=torch.bfloat16, k_out=None, v_out=None,
               stream=None):
    """Keys and values [tokens, heads, dim] of slots [tokens] (int64), as the
    values the cache holds, rounded to `dtype`.  A slot outside the cache
    reads as zeros.  Returns (k, v)."""
    dev = _Device(k_pages, "k_pages", stream)
    cache = _cache(k_pages, v_pages, k_scale, v_scale)
    if dtype not in _FLOAT:
        raise TypeError("dtype must be float32, float16 or bfloat16")
    shape = (_slots(slots, k_pages.device).shape[0], cache.heads, cache.dim)
    k_out = _out_like(k_out, shape, dtype, k_pages.device, "k_out")
    v_out = _out_like(v_out, shape, dtype, k_pages.device, "v_out")
    kh, vh = _heads(k_out, "k_out", ("token",)), _heads(v_out, "v_out", ("token",))
    with dev as st:
        _check(capi.lib().chm_cache_read(C.byref(cache), slots.data_ptr(), shape[0], C.byref(kh), C.byref(vh),
                                         _FLOAT[dtype], st), "cache_read")
    return k_out, v_out


def paged_attention(q, k_pages, v_pages, tables, lens, k_scale=None, v_scale=None, *, starts=None, scale=None,
                    out=None, lse=None, workspace=None, stream=None):
    """Attention of one new token per sequence, q [batch, q_heads, dim]
    (float16 or bfloat16, a 16-bit cache's own type), over tokens
    starts[b] <= j < lens[b] of its sequence (int32 [batch]; starts default to
    0), token j in page tables[b, j // page_size] (int32 [batch, width]).
    Query heads share key heads evenly.  scale defaults to dim ** -0.5.

    Returns (out like q, lse float32 [batch, q_heads]); a row with nothing to
    attend to gets zeros and -inf, one whose table or length does not fit the
    cache NaN (chm_paged_attention).  `workspace`: a uint8 tensor of
    paged_attention_workspace bytes for callers that keep one; calls that may
    overlap, captured graphs among them, each need their own."""
    dev = _Device(q, "q", stream)
    cache = _cache(k_pages, v_pages, k_scale, v_scale)
    device = q.device
    _on(device, k_pages, "k_pages")
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError("q must be float16 or bfloat16")
    if q.dim() != 3 or q.shape[2] != cache.dim:
        raise ValueError(f"q must be [batch, q_heads, {cache.dim}]")
    batch, heads = q.shape[0], q.shape[1]
    if tables.dtype != torch.int32 or tables.dim() != 2 or tables.shape[0] != batch or \
            (tables.shape[1] > 1 and tables.stride(1) != 1):
        raise ValueError("tables must be int32 [batch, width], contiguous along the width")
    _on(device, tables, "tables")
    for x, name in ((lens, "lens"), (starts, "starts")):
        if x is None and name == "starts":
            continue
        if x.dtype != torch.int32 or x.shape != (batch,) or not x.is_contiguous():
            raise ValueError(f"{name} must be contiguous int32 [batch]")
        _on(device, x, name)
    out = _out_like(out, q.shape, q.dtype, device, "out")
    lse = _out_like(lse, (batch, heads), torch.float32, device, "lse")
    if not lse.is_contiguous():
        raise ValueError("lse must be contiguous")
    L = capi.lib()
    width = tables.shape[1]
    qh, oh = _heads(q, "q", ("batch",)), _heads(out, "out", ("batch",))
    with dev as st:
        need = L.chm_paged_attention_workspace_bytes(C.byref(cache), batch, heads, width)
        if workspace is None:
            workspace = torch.empty(need, dtype=torch.uint8, device=device)
        else:
            _on(device, workspace, "workspace")
            if workspace.dtype != torch.uint8 or not workspace.is_contiguous() or workspace.numel() < need or \
                    workspace.data_ptr() % 256:
                raise ValueError(f"workspace must be contiguous uint8, 256-byte aligned, of {need} bytes or more")
        _check(L.chm_paged_attention(C.byref(cache), C.byref(qh), C.byref(oh), _HELD[q.dtype], batch,
                                     tables.data_ptr(), tables.stride(0), width, lens.data_ptr(),
                                     starts.data_ptr() if starts is not None else None,
                                     scale if scale is not None else 1.0 / math.sqrt(cache.dim), lse.data_ptr(),
                                     workspace.data_ptr(), workspace.numel(), st), "paged_attention")
        if stream is not None and stream != torch.cuda.current_stream():
            workspace.record_stream(stream)
    return out, lse


def paged_attention_workspace(k_pages, v_pages, batch, q_heads, table_width, k_scale=None, v_scale=None):
    """Bytes of the workspace paged_attention needs for these sizes."""
    cache = _cache(k_pages, v_pages, k_scale, v_scale)
    with _Device(k_pages, "k_pages", None):
        return capi.lib().chm_paged_attention_workspace_bytes(C.byref(cache), batch, q_heads, table_width)
