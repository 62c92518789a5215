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
its slot, is in page s // page_size at s % page_size.  dim is a multiple of 16,
at most 256.

Every call runs on `stream` (default: the current stream of its tensors'
device), allocates its outputs there where none are given, never synchronises,
and can be captured into a CUDA graph.  As with any work on a stream of one's
own, its order against the tensors' other uses is the caller's, and so is keeping
them until it is done (torch.Tensor.record_stream).  Arguments that do not fit raise
TypeError or ValueError before anything is launched; so do tensors that
require a gradient while gradients are recorded, and tensors with a
forward-mode tangent.  Tensors that a call writes (outputs given to it, pages,
scales) count as modified in place; one whose vectors share memory (an expanded
one), or that starts where another one does, is refused.  The calls are plain
functions, not registered operators: torch.compile breaks its graph at them, and
torch.export cannot hold them.
"""
from __future__ import annotations

import torch

from . import _generation as _g
from . import capi

KINDS = {"plain": 0, "linear": 1, "base": 2, "parts": 3}


def _run(stream, x, call, *args):
    """call(*args) on `stream` (its device is x's)."""
    if isinstance(x, torch.Tensor) and x.is_cuda and stream.device != x.device:
        raise ValueError(f"the stream is on {stream.device}, not on {x.device}")
    with torch.cuda.stream(stream):
        return call(*args)


def rotary_frequencies(rot_dim, base=10000.0, *, kind="plain", factor=1.0, original_len=4096, slow=1.0, fast=32.0,
                       device=None):
    """Rotation frequencies (float64 [rot_dim / 2], radians per position) for
    `rotary`, for contexts up to `factor` times longer than `original_len`:
    "plain" (unscaled), "linear" (all divided by the factor), "base" (a larger
    base) or "parts" (pairs that turn more than `fast` times over original_len
    as they are, fewer than `slow` times divided, between them a ramp that is
    linear in the number of turns, not in the pair's index)."""
    if kind not in KINDS:
        raise ValueError(f"kind must be one of {sorted(KINDS)}")
    rot_dim = int(rot_dim)
    out = torch.empty(max(rot_dim, 0) // 2, dtype=torch.float64)
    L = capi.lib()
    status = L.chm_rotary_frequencies(rot_dim, base, KINDS[kind], factor, original_len, slow, fast,
                                      out.data_ptr() or None)
    if status == capi.CHM_ERR_INVALID:
        raise ValueError(L.chm_last_error().decode())
    capi.check(status, "rotary_frequencies")
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
    the same scale.  q_out / k_out may be q and k themselves, but not overlap
    them in any other way.  Returns (q_out, k_out)."""
    if stream is None:
        return _g.rotary(q, k, positions, freqs, interleaved, inverse, scale, q_out, k_out)
    return _run(stream, q, _g.rotary, q, k, positions, freqs, interleaved, inverse, scale, q_out, k_out)


def cache_write(k, v, slots, k_pages, v_pages, k_scale=None, v_scale=None, *, stream=None):
    """Write tokens' keys and values (k, v: [tokens, heads, dim], float32,
    float16 or bfloat16) to slots [tokens] (int64) of the cache; int8 and
    float8_e4m3fn pages get codes and one scale per vector (chm_cache_write).
    A slot outside the cache is skipped.  No slot may stand twice."""
    if stream is None:
        return _g.cache_write(k, v, slots, k_pages, v_pages, k_scale, v_scale)
    return _run(stream, k, _g.cache_write, k, v, slots, k_pages, v_pages, k_scale, v_scale)


def cache_read(slots, k_pages, v_pages, k_scale=None, v_scale=None, *, dtype=torch.bfloat16, k_out=None, v_out=None,
               stream=None):
    """Keys and values [tokens, heads, dim] of slots [tokens] (int64), as the
    values the cache holds, rounded to `dtype`.  A slot outside the cache
    reads as zeros.  Returns (k, v)."""
    if stream is None:
        return _g.cache_read(slots, k_pages, v_pages, k_scale, v_scale, dtype, k_out, v_out)
    return _run(stream, k_pages, _g.cache_read, slots, k_pages, v_pages, k_scale, v_scale, dtype, k_out, v_out)


def paged_attention(q, k_pages, v_pages, tables, lens, k_scale=None, v_scale=None, *, starts=None, scale=None,
                    out=None, lse=None, workspace=None, stream=None):
    """Attention of one new token per sequence, q [batch, q_heads, dim]
    (float16 or bfloat16, a 16-bit cache's own type), over tokens
    starts[b] <= j < lens[b] of its sequence (int32 [batch]; starts default to
    0), token j in page tables[b, j // page_size] (int32 [batch, width]).
    Query heads share key heads evenly.  scale defaults to dim ** -0.5.  out may
    be q itself.

    Returns (out like q, lse float32 [batch, q_heads]); a row with nothing to
    attend to gets zeros and -inf, one whose table or length does not fit the
    cache NaN (chm_paged_attention).  `workspace`: a uint8 tensor of
    paged_attention_workspace bytes for callers that keep one; calls that may
    overlap, captured graphs among them, each need their own."""
    if stream is None:
        return _g.paged_attention(q, k_pages, v_pages, k_scale, v_scale, tables, lens, starts, scale, out, lse,
                                  workspace)
    return _run(stream, q, _g.paged_attention, q, k_pages, v_pages, k_scale, v_scale, tables, lens, starts, scale,
                out, lse, workspace)


def paged_attention_workspace(k_pages, v_pages, batch, q_heads, table_width, k_scale=None, v_scale=None):
    """Bytes of the workspace paged_attention needs for these sizes."""
    return _g.paged_attention_workspace(k_pages, v_pages, k_scale, v_scale, batch, q_heads, table_width)
