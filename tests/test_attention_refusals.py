"""The generation operators' refusals at the C ABI and their host-side parts,
on a machine without a GPU: a call that does not fit returns CHM_ERR_INVALID
with a reason and launches nothing, a call on nothing returns CHM_OK.  The
pointers are placeholders; no refused or empty call follows them."""
import ctypes as C
import math

import numpy as np
import pytest

from chimera_b200 import capi

torch = pytest.importorskip("torch")
from chimera_b200 import attention as A  # noqa: E402

P = 4096  # a placeholder address, 16-byte aligned
L = capi.lib()


def heads(**over):
    kw = dict(data=P, heads=8, batch_stride=1024, token_stride=1024, head_stride=128)
    kw.update(over)
    return capi.ChmHeads(**kw)


def cache(**over):
    kw = dict(k=P, v=P, k_scale=P, v_scale=P, num_pages=10, page_stride=8 * 16 * 128, head_stride=16 * 128,
              token_stride=128, page_size=16, heads=8, dim=128, type=3)
    kw.update(over)
    return capi.ChmKvCache(**kw)


def rotary(n=1, type=2, batch=0, tokens=0, dim=128, rot=128, pos=P, pos_bytes=8, freqs=P, flags=0, **h):
    one = (capi.ChmHeads * 2)(heads(**h), heads(**h))
    return L.chm_rotary(one, one, n, type, batch, tokens, dim, rot, pos, pos_bytes, 0, 1, freqs, 1.0, flags, None)


def refused(status, word):
    assert status == capi.CHM_ERR_INVALID
    assert word in L.chm_last_error().decode()


def test_rotary_on_nothing():
    assert rotary() == capi.CHM_OK
    assert rotary(batch=3) == capi.CHM_OK
    assert rotary(batch=3, tokens=5, heads=0) == capi.CHM_OK


@pytest.mark.parametrize("over,word", [
    (dict(n=0), "sets"), (dict(n=3), "sets"), (dict(type=3), "fp32"), (dict(type=-1), "fp32"),
    (dict(batch=-1), "negative"), (dict(tokens=-1), "negative"), (dict(rot=63), "even"), (dict(rot=0), "even"),
    (dict(rot=130), "even"), (dict(dim=4098, rot=64), "4096"), (dict(pos_bytes=2), "int32"),
    (dict(flags=4), "flag"), (dict(batch=1, tokens=1, data=None), "null"), (dict(batch=1, tokens=1, pos=None), "null"),
    (dict(batch=1, tokens=1, freqs=None), "null"), (dict(batch=1 << 20, tokens=1 << 11), "2^31"),
    (dict(batch=1, tokens=1, heads=-1), "heads"), (dict(batch=1, tokens=1, heads=65537), "heads"),
])
def test_rotary_refuses(over, word):
    refused(rotary(**over), word)


CACHE_FAULTS = [
    (dict(type=0), "fp16, bf16"), (dict(type=5), "fp16, bf16"), (dict(page_size=0), "page_size"),
    (dict(heads=0), "heads"), (dict(num_pages=-1), "page_size"), (dict(num_pages=1 << 62), "too many"),
    (dict(dim=8), "dim"), (dict(dim=120), "dim"), (dict(dim=272), "dim"), (dict(k=P + 8), "aligned"),
    (dict(v=P + 1), "aligned"), (dict(page_stride=8), "strides"), (dict(head_stride=24), "strides"),
    (dict(token_stride=129), "strides"), (dict(type=2, token_stride=132), "strides"), (dict(k=None), "null"),
    (dict(k_scale=None), "scales"), (dict(v_scale=None, type=4), "scales"),
]


@pytest.mark.parametrize("over,word", CACHE_FAULTS)
def test_every_cache_call_refuses_a_bad_cache(over, word):
    c, h = cache(**over), heads()
    refused(L.chm_cache_write(C.byref(c), C.byref(h), C.byref(h), 2, 1, P, None), word)
    refused(L.chm_cache_read(C.byref(c), P, 1, C.byref(h), C.byref(h), 2, None), word)
    refused(attend(c), word)


def test_cache_calls_on_nothing():
    c, h = cache(), heads(data=None)
    assert L.chm_cache_write(C.byref(c), C.byref(h), C.byref(h), 2, 0, None, None) == capi.CHM_OK
    assert L.chm_cache_read(C.byref(c), None, 0, C.byref(h), C.byref(h), 2, None) == capi.CHM_OK
    assert attend(c, batch=0) == capi.CHM_OK


@pytest.mark.parametrize("over,word", [
    (dict(type=3), "fp32"), (dict(tokens=-1), "negative"), (dict(slots=None), "null"), (dict(heads=4), "heads"),
    (dict(data=None), "null"), (dict(tokens=1 << 29), "2^31"),
])
def test_cache_calls_refuse(over, word):
    o = dict(type=2, tokens=1, slots=P)
    o.update({k: v for k, v in over.items() if k in o})
    c, h = cache(), heads(**{k: v for k, v in over.items() if k not in o})
    refused(L.chm_cache_write(C.byref(c), C.byref(h), C.byref(h), o["type"], o["tokens"], o["slots"], None), word)
    refused(L.chm_cache_read(C.byref(c), o["slots"], o["tokens"], C.byref(h), C.byref(h), o["type"], None), word)


def attend(c, type=2, batch=1, tables=P, width=4, lens=P, ws=P, ws_bytes=1 << 40, q_heads=32, out_heads=None,
           q_data=P):
    q = heads(heads=q_heads, data=q_data)
    o = heads(heads=q_heads if out_heads is None else out_heads)
    return L.chm_paged_attention(C.byref(c), C.byref(q), C.byref(o), type, batch, tables, width, width, lens, None,
                                 0.1, None, ws, ws_bytes, None)


@pytest.mark.parametrize("over,word", [
    (dict(type=0), "fp16 or bf16"), (dict(type=3), "fp16 or bf16"), (dict(batch=-1), "negative"),
    (dict(width=-1), "negative"), (dict(q_heads=12), "multiple"), (dict(q_heads=0), "multiple"),
    (dict(out_heads=8), "multiple"), (dict(batch=65536), "65535"), (dict(width=1 << 27), "2^30"),
    (dict(lens=None), "null"), (dict(tables=None), "null"), (dict(q_data=None), "null"),
])
def test_attention_refuses(over, word):
    refused(attend(cache(), **over), word)


def test_attention_refuses_another_type_than_a_16_bit_caches():
    refused(attend(cache(type=1), type=2), "type")
    refused(attend(cache(type=2), type=1), "type")


def test_attention_refuses_a_small_workspace():
    c = cache()
    need = L.chm_paged_attention_workspace_bytes(C.byref(c), 1, 32, 4)
    assert need > 0
    assert attend(c, ws_bytes=need - 1) == capi.CHM_ERR_CAPACITY
    assert attend(c, ws=None) == capi.CHM_ERR_CAPACITY


def test_null_arguments_are_refused():
    h, c = heads(), cache()
    assert L.chm_rotary(None, None, 1, 2, 1, 1, 128, 128, P, 8, 0, 1, P, 1.0, 0, None) == capi.CHM_ERR_INVALID
    assert L.chm_cache_write(None, C.byref(h), C.byref(h), 2, 1, P, None) == capi.CHM_ERR_INVALID
    assert L.chm_cache_write(C.byref(c), None, C.byref(h), 2, 1, P, None) == capi.CHM_ERR_INVALID
    assert L.chm_cache_read(C.byref(c), P, 1, C.byref(h), None, 2, None) == capi.CHM_ERR_INVALID
    assert L.chm_paged_attention(C.byref(c), None, None, 2, 1, P, 4, 4, P, None, 0.1, None, P, 1 << 40,
                                 None) == capi.CHM_ERR_INVALID


# ---- frequencies ---------------------------------------------------------------

def test_frequencies_plain_linear_base():
    i = np.arange(32)
    f = 10000.0 ** (-2.0 * i / 64)
    np.testing.assert_allclose(A.rotary_frequencies(64).numpy(), f, rtol=1e-14)
    np.testing.assert_allclose(A.rotary_frequencies(64, kind="linear", factor=8).numpy(), f / 8, rtol=1e-14)
    g = A.rotary_frequencies(64, kind="base", factor=8).numpy()
    assert g[0] == 1.0
    np.testing.assert_allclose(g[-1], f[-1] / 8, rtol=1e-12)  # the slowest is slowed by the factor
    assert np.all(np.diff(g / f) < 0)
    np.testing.assert_allclose(A.rotary_frequencies(2, 500000.0, kind="base", factor=4).numpy(), [1.0])


def test_frequencies_parts():
    f = A.rotary_frequencies(128).numpy()
    g = A.rotary_frequencies(128, kind="parts", factor=16, original_len=4096, slow=1, fast=32).numpy()
    turns = 4096 * f / (2 * math.pi)
    for a, b, r in zip(f, g, turns):
        share = min(max((r - 1) / 31, 0.0), 1.0)
        assert b == pytest.approx(a * share + a / 16 * (1 - share), rel=1e-13)
    assert g[0] == f[0] and g[-1] == pytest.approx(f[-1] / 16, rel=1e-14)


@pytest.mark.parametrize("kw", [
    dict(rot_dim=0), dict(rot_dim=-2), dict(rot_dim=7), dict(rot_dim=64, base=1.0), dict(rot_dim=64, base=math.nan),
    dict(rot_dim=64, kind="linear", factor=0.5), dict(rot_dim=64, kind="base", factor=math.inf),
    dict(rot_dim=64, kind="parts", factor=2, original_len=0), dict(rot_dim=64, kind="parts", factor=2, slow=0),
    dict(rot_dim=64, kind="parts", factor=2, slow=4, fast=4), dict(rot_dim=64, kind="other"),
])
def test_frequencies_refuse(kw):
    with pytest.raises(ValueError):
        A.rotary_frequencies(**kw)


def test_python_calls_want_cuda_tensors():
    x = torch.zeros(4, 8, 128)
    i = torch.zeros(4, dtype=torch.int64)
    pages = torch.zeros(2, 8, 16, 128)
    with pytest.raises(TypeError):
        A.rotary(x, None, i, A.rotary_frequencies(128))
    with pytest.raises(TypeError):
        A.cache_write(x, x, i, pages, pages)
    with pytest.raises(TypeError):
        A.cache_read(i, pages, pages)
    with pytest.raises(TypeError):
        A.paged_attention(x, pages, pages, i, i)


@pytest.mark.parametrize("batch,q_heads,width", [(1, 12, 4), (1, 0, 4), (-1, 32, 4), (65536, 32, 4), (1, 32, -1),
                                                 (1, 32, 1 << 27), (65535, 32, 1 << 26)])
def test_the_workspace_of_what_is_refused_is_nothing(batch, q_heads, width):
    """And the reason is the call's; the last has more work than one call takes."""
    c = cache()
    assert L.chm_paged_attention_workspace_bytes(C.byref(c), batch, q_heads, width) == 0
    reason = L.chm_last_error().decode()
    assert reason.startswith("paged_attention: ")
    assert attend(c, batch=batch, q_heads=q_heads, width=width, tables=P) == capi.CHM_ERR_INVALID
    assert L.chm_last_error().decode() == reason
