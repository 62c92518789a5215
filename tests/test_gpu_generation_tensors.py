"""The generation operators as calls on torch tensors, on the GPU: what autograd
sees of them, and which tensors are taken and refused."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from chimera_b200 import attention as A  # noqa: E402
from tests.test_gpu_attention import DEV, Case, make_pages  # noqa: E402


def versions(*xs):
    return [x._version for x in xs]


def test_what_is_written_counts_as_changed():
    """Tensors that a call writes have their version raised, those it reads not."""
    f = A.rotary_frequencies(64, device=DEV)
    pos = torch.arange(5, device=DEV)
    q, k, qo, ko = (torch.randn(5, 2, 64, device=DEV).bfloat16() for _ in range(4))
    before = versions(q, k, qo, ko)
    A.rotary(q, k, pos, f)
    assert versions(q, k, qo, ko) == before
    A.rotary(q, k, pos, f, q_out=qo, k_out=ko)
    after = versions(q, k, qo, ko)
    assert after[:2] == before[:2] and after[2] > before[2] and after[3] > before[3]
    A.rotary(q, None, pos, f, q_out=q)
    assert q._version > before[0] and k._version == before[1]

    for held in (torch.int8, torch.bfloat16):
        cache = make_pages(2, 2, 8, 64, held)
        there = [x for x in cache if x is not None]
        before = versions(k, *there)
        A.cache_write(k, k, pos, *cache)
        after = versions(k, *there)
        assert after[0] == before[0] and all(a > b for a, b in zip(after[1:], before[1:]))
        A.cache_read(pos, *cache, k_out=ko, v_out=qo)
        assert versions(k, *there) == after

    c = Case(lens=[40, 9], q_heads=4, k_heads=2, dim=64, page=16, held="int8", t="bf16")
    out, lse = c.run()
    there = [c.q, c.kp, c.vp, c.ks, c.vs, c.tables, c.l]
    before, seen = versions(*there), versions(out, lse)
    c.run(out=out, lse=lse)
    assert versions(*there) == before and all(a > b for a, b in zip(versions(out, lse), seen))


def test_a_saved_tensor_that_is_turned_in_place_is_noticed():
    f = A.rotary_frequencies(64, device=DEV)
    pos = torch.arange(5, device=DEV)
    w = torch.randn(5, 2, 64, device=DEV, requires_grad=True)
    x = torch.randn(5, 2, 64, device=DEV)
    y = (w * x).sum()     # saves x
    with torch.no_grad():
        A.rotary(x, None, pos, f, q_out=x)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_tensors_of_inference_mode_are_taken_everywhere():
    f = A.rotary_frequencies(64, device=DEV)
    pos = torch.arange(5, device=DEV)
    with torch.inference_mode():
        x = torch.randn(5, 2, 64, device=DEV)
        cache = make_pages(2, 2, 8, 64, torch.int8)
        A.rotary(x, None, pos, f, q_out=x)
        A.cache_write(x, x, pos, *cache)
    A.rotary(x, None, pos, f, q_out=x)
    A.cache_write(x, x, pos, *cache)
    k, v = A.cache_read(pos, *cache, dtype=torch.float32)
    assert torch.equal(k, v)


def test_tensors_with_tangents_are_refused():
    """A call that would drop a forward-mode tangent says so, under no_grad too."""
    import torch.autograd.forward_ad as ad
    f = A.rotary_frequencies(64, device=DEV)
    c = Case(lens=[40, 9], q_heads=4, k_heads=2, dim=64, page=16, held="bf16")
    pos = torch.arange(2, device=DEV)
    with ad.dual_level():
        q = ad.make_dual(c.q, torch.ones_like(c.q))
        k = q[:, :2]
        assert ad.unpack_dual(k).tangent is not None
        for call in (lambda: A.rotary(q, None, pos, f), lambda: A.rotary(c.q, k, pos, f),
                     lambda: A.cache_write(k, c.q[:, :2], pos, c.kp, c.vp),
                     lambda: A.cache_write(c.q[:, :2], k, pos, c.kp, c.vp),
                     lambda: A.paged_attention(q, c.kp, c.vp, c.tables, c.l)):
            with pytest.raises(ValueError, match="tangent"):
                call()
            with torch.no_grad(), pytest.raises(ValueError, match="tangent"):
                call()
        A.rotary(c.q, None, pos, f)     # tensors without one are taken
        c.run()
        A.rotary(ad.unpack_dual(q).primal, None, pos, f)


@pytest.mark.parametrize("held", ["bf16", "int8"])
def test_strides_of_axes_of_one_do_not_matter(held):
    """k and v pages of one page, one head or one token a page, as views with any stride along that axis."""
    for pages, heads, page in ((1, 2, 16), (5, 1, 16), (3, 2, 1), (1, 1, 1)):
        n = min(pages * page, 9)
        c = Case(lens=[n], q_heads=2 * heads, k_heads=heads, dim=64, page=page, held=held, t="bf16",
                 spare=pages - -(-n // page))
        want, wlse = c.run()

        def restrided(x, by):
            s = [by if x.shape[i] == 1 else x.stride(i) for i in range(3)] + [1]
            return x.as_strided(x.shape, s, x.storage_offset())
        c.vp = restrided(c.vp, 7)
        got, lse = c.run()
        assert torch.equal(got, want) and torch.equal(lse, wlse)
        c.kp = restrided(c.kp, 1 << 40)
        got, lse = c.run()
        assert torch.equal(got, want) and torch.equal(lse, wlse)
        slots = torch.arange(c.n * page, device=DEV)
        k, v = A.cache_read(slots, c.kp, c.vp, c.ks, c.vs)
        A.cache_write(k, v, slots, c.kp, c.vp, c.ks, c.vs)
        plain = make_pages(c.n, heads, page, 64, c.ht)
        A.cache_write(k, v, slots, *plain)
        for x, y in zip(A.cache_read(slots, c.kp, c.vp, c.ks, c.vs), A.cache_read(slots, *plain)):
            assert torch.equal(x, y)
    # where an axis has more than one, k and v still go alike
    c = Case(lens=[9], q_heads=4, k_heads=2, dim=64, page=16, held=held, t="bf16")
    with pytest.raises(ValueError):
        A.paged_attention(c.q, c.kp, c.vp.transpose(1, 2).contiguous().transpose(1, 2), c.tables, c.l, c.ks, c.vs)


def test_outputs_that_overlap_are_refused():
    f = A.rotary_frequencies(64, device=DEV)
    c = Case(lens=[40, 9], q_heads=4, k_heads=2, dim=64, page=16, held="int8", t="bf16")
    pos = torch.arange(2, device=DEV)
    kv = c.q[:, :2].contiguous()
    one = torch.zeros(1, 1, 64, dtype=torch.bfloat16, device=DEV)
    lines = torch.zeros(4 * 64, dtype=torch.bfloat16, device=DEV).as_strided((2, 2, 64), (64, 32, 1))
    wide = make_pages(1, 2, 16, 64, torch.int8)
    over = [x.expand(3, *x.shape[1:]) for x in wide[:2]]
    scales = [torch.zeros(3, 2, 16, device=DEV) for _ in range(2)]
    for call in (lambda: A.rotary(c.q, None, pos, f, q_out=one.expand(2, 4, 64)),
                 lambda: A.rotary(kv, kv, pos, f, k_out=one.expand(2, 2, 64)),
                 lambda: A.rotary(kv, None, pos, f, q_out=lines),
                 lambda: A.rotary(one.expand(2, 4, 64), None, pos, f, q_out=one.expand(2, 4, 64)),
                 lambda: A.cache_read(pos, c.kp, c.vp, c.ks, c.vs, k_out=one.expand(2, 2, 64)),
                 lambda: A.cache_read(pos, c.kp, c.vp, c.ks, c.vs, v_out=lines),
                 lambda: A.cache_write(kv, kv, pos, *over, *scales),
                 lambda: c.run(out=one.expand(2, 4, 64)),
                 lambda: A.rotary(kv, kv, pos, f, q_out=kv, k_out=kv),     # or one another
                 lambda: A.cache_read(pos, c.kp, c.vp, c.ks, c.vs, k_out=kv, v_out=kv),
                 lambda: A.cache_write(kv, kv, pos, c.kp, c.kp, c.ks, c.vs),
                 lambda: A.cache_write(kv, kv, pos, c.kp, c.vp, c.ks, c.ks)):
        with pytest.raises(ValueError, match="overlap"):
            call()
    # read, they may: a page that stands three times, keys that are the values too, heads that share one vector
    A.cache_read(pos, *over, *scales)
    A.cache_read(pos, c.kp, c.kp, c.ks, c.ks)
    A.paged_attention(c.q, c.kp, c.kp, c.tables, c.l, c.ks, c.ks)
    A.rotary(one.expand(2, 4, 64), None, pos, f)
    # axes of one, and outputs with their axes in another order, do not overlap
    A.rotary(one, None, pos[:1], f, q_out=torch.zeros(64, dtype=torch.bfloat16, device=DEV).as_strided((1, 1, 64), (0, 0, 1)))
    A.rotary(c.q, None, pos, f, q_out=torch.zeros(4, 2, 64, dtype=torch.bfloat16, device=DEV).transpose(0, 1))


def test_the_workspace_of_what_is_refused_is_refused():
    c = Case(lens=[40, 9], q_heads=4, k_heads=2, dim=64, page=16, held="int8", t="bf16")
    cache = c.kp, c.vp
    assert A.paged_attention_workspace(*cache, 2, 4, 3, c.ks, c.vs) > 0
    for batch, heads, width in ((2, 5, 3), (2, 0, 3), (65536, 4, 3), (2, 4, 1 << 27), (65535, 4, 1 << 26)):
        with pytest.raises(ValueError):
            A.paged_attention_workspace(*cache, batch, heads, width, c.ks, c.vs)
