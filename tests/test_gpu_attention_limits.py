"""Attention over the cache at the limits of its inputs, on the GPU.  Bounds and the
plain form in 64 bits are those of test_gpu_attention.py."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from chimera_b200 import attention as A  # noqa: E402
from tests.test_gpu_attention import DEV, Case, gen, within  # noqa: E402


I32 = torch.iinfo(torch.int32)


@pytest.mark.parametrize("held,t", [("bf16", None), ("int8", "bf16")])
@pytest.mark.parametrize("width", [8, 200])   # segments whole, and split and joined
@pytest.mark.parametrize("copies", [1, 40])   # with 40, 200 sequences: the join reads what the main kernel left
def test_the_smallest_lengths_with_positive_starts(copies, width, held, t):
    """lens - starts passes the ends of int32: nothing to attend to, and the others' bits as beside lengths of 0."""
    lens = [100, I32.min, 128, I32.min + 3, -1] * copies
    starts = [0, 5, 3, I32.max, I32.max] * copies
    c = Case(lens=lens, starts=starts, q_heads=6, k_heads=2, dim=64, page=16, held=held, t=t, width=width)
    got, lse = c.check()
    empty = torch.tensor(lens, device=DEV) < 0
    assert bool((got[empty] == 0).all() & (lse[empty] == -math.inf).all())
    c.l.clamp_(min=0)
    c.s[empty] = 0
    plain, plse = c.run()
    assert torch.equal(got, plain) and torch.equal(lse, plse)


@pytest.mark.parametrize("start", [1, 5, 1 << 30, I32.max])
@pytest.mark.parametrize("length", [I32.min, I32.min + 1, -(1 << 30) - 1, -1, 0])
def test_one_sequence_of_no_length_with_a_start(length, start):
    for width in (4, 4000):
        c = Case(lens=[length], starts=[start], q_heads=4, k_heads=2, dim=64, page=16, held="fp16", width=width)
        got, lse = c.run()
        assert bool((got == 0).all() & (lse == -math.inf).all())


def place(c, b, token):
    return int(c.tables[b, token // c.page]), token % c.page


@pytest.mark.parametrize("held", ["bf16", "fp16"])
@pytest.mark.parametrize("dim,group", [(64, 4), (64, 12), (128, 3), (128, 9), (256, 2), (80, 1)])
@pytest.mark.parametrize("n", [90, 9000])   # one block, and parts that are joined
def test_infinite_values(n, dim, group, held):
    """An element with infinite values of one sign among those attended to is that infinity, with both signs or a
    NaN it is NaN; all else keeps its bits.  Weights reach from the largest to far below what 16 bits hold."""
    c = Case(lens=[n, 70], q_heads=2 * group, k_heads=2, dim=dim, page=16, held=held, seed=dim + n)
    c.q *= 0.5
    k = c.values(c.kp, None)[c.tables[0].long()].transpose(0, 1).flatten(1, 2)[:, :n]
    s = torch.einsum("hd,hnd->hn", c.q[0].double(), k.repeat_interleave(group, 0)) * c.scale
    order = s[0].argsort().tolist()   # by the first row's weights
    near, far, last = order[-1], order[0], order[n // 2]
    p, w = place(c, 0, far)
    c.kp[p, 0, w] *= 16.0             # far below the others for that row, above them for some
    clean, clse = c.run()
    inf = math.inf
    #       element: (token, value), ...
    marks = {0: [(near, inf)], 1: [(near, -inf)], 2: [(far, inf)], 3: [(far, -inf)], 4: [(last, inf), (near, inf)],
             5: [(last, inf), (far, -inf)], 6: [(near, inf), (far, math.nan)], 7: [(0, inf)], 8: [(n - 1, -inf)],
             dim - 1: [(n // 3, inf), (n - 2, inf)], dim - 2: [(n // 3, inf), (n - 2, -inf)]}
    want = {0: inf, 1: -inf, 2: inf, 3: -inf, 4: inf, 5: math.nan, 6: math.nan, 7: inf, 8: -inf, dim - 1: inf,
            dim - 2: math.nan}
    for d, m in marks.items():
        for token, value in m:
            p, w = place(c, 0, token)
            c.vp[p, 0, w, d] = value
    got, lse = c.run()
    assert torch.equal(lse, clse)
    expected = clean.clone()
    for d, y in want.items():
        expected[0, :group, d] = y
    same = (got == expected) | (got.isnan() & expected.isnan())
    assert bool(same.all()), f"elements {sorted(set((~same).nonzero()[:, 2].tolist()))} differ"


@pytest.mark.parametrize("held", ["bf16", "fp16"])
def test_infinite_values_outside_the_range_change_nothing(held):
    c = Case(lens=[100, 3000], starts=[20, 1000], q_heads=8, k_heads=2, dim=64, page=16, held=held)
    clean = c.run()
    for b, tokens in ((0, (0, 19, 100)), (1, (0, 999, 3000))):
        for token in tokens:
            p, w = place(c, b, token)
            c.vp[p, :, w] = math.inf
    got = c.run()
    assert all(torch.equal(x, y) for x, y in zip(got, clean))


def test_a_value_past_fp16_is_an_infinity():
    """cache_write rounds fp32 values above 65,504 to infinities in an fp16 cache."""
    c = Case(lens=[300], q_heads=4, k_heads=2, dim=64, page=16, held="fp16")
    _, clse = c.run()
    slots = torch.tensor([int(c.tables[0, 8]) * 16 + 5], device=DEV)
    k, v = A.cache_read(slots, c.kp, c.vp, dtype=torch.float32)
    v[0, 1, 7], v[0, 1, 9] = 1e5, -1e5
    A.cache_write(k, v, slots, c.kp, c.vp)
    got, lse = c.run()
    assert torch.equal(lse, clse)
    assert bool((got[0, 2:, 7] == math.inf).all() & (got[0, 2:, 9] == -math.inf).all())
    got[0, 2:, 7] = got[0, 2:, 9] = 0
    assert bool(got.isfinite().all())


@pytest.mark.parametrize("held", ["int8", "e4m3"])
@pytest.mark.parametrize("n", [200, 9000])
def test_infinite_scales_of_values(n, held):
    """Values are code * scale: infinities by the codes' signs, NaN where a code is 0; lse does not see them."""
    c = Case(lens=[n, 70], q_heads=6, k_heads=2, dim=64, page=16, held=held, t="bf16", seed=n)
    clean, _ = c.run()
    _, sums, _, tol = c.expected()
    p, w = place(c, 0, n // 2)
    c.vp.view(torch.uint8)[p, 1, w, 5] = 0
    c.vs[p, 1, w] = math.inf
    code = c.vp[p, 1, w].float()
    got, lse = c.run()
    within(lse, sums, tol + 2 * n * 2.0 ** -24)
    want = clean.clone()
    want[0, 3:] = code * math.inf
    assert bool(((got == want) | (got.isnan() & want.isnan())).all())


@pytest.mark.parametrize("held", ["int8", "e4m3"])
@pytest.mark.parametrize("by", [2.0 ** 50, 2.0 ** 60, 2.0 ** 100])
@pytest.mark.parametrize("zero", [
    lambda j, n: j < n // 2,             # all of the first warps, steps, blocks
    lambda j, n: j >= n // 2,
    lambda j, n: j % 2 == 0,             # within every step
    lambda j, n: j // 32 % 2 == 0,       # warp by warp
    lambda j, n: j // 128 % 2 == 0,      # step by step
    lambda j, n: j != n - 1,             # one token has values, the last
    lambda j, n: j != 0,
])
@pytest.mark.parametrize("n", [64, 500, 9000])
def test_sums_beside_scales_far_apart(n, zero, by, held):
    """Vectors of zeros beside huge ones, scores alike or a few units apart: the sum of the probabilities keeps those
    of both, though the exponents that the weights are taken against differ by up to 180."""
    c = Case(lens=[n], q_heads=4, k_heads=2, dim=64, page=16, held=held, t="bf16", seed=n, spare=0)
    slots = c.tables[0].long().repeat_interleave(16) * 16 + torch.arange(16, device=DEV).repeat(c.tables.shape[1])
    k, v = A.cache_read(slots, c.kp, c.vp, c.ks, c.vs, dtype=torch.float32)
    v = torch.randn(v.shape, generator=gen(3), device=DEV).clamp(-3, 3) * by
    v[zero(torch.arange(len(slots), device=DEV), n)] = 0
    A.cache_write(k, v, slots, c.kp, c.vp, c.ks, c.vs)
    for spread in (0.0, 1.0):
        c.q.normal_(generator=gen(4)).mul_(spread)
        got, lse = c.run()
        held_vs, c.vs = c.vs, c.vs.double() / by
        out, want, tol, ltol = c.expected()
        c.vs = held_vs
        more = 2 * n * 2.0 ** -24
        within(lse, want, ltol + more)
        within(got.double() / by, out, tol + more * 3)


@pytest.mark.parametrize("held", ["int8", "e4m3"])
@pytest.mark.parametrize("up", [126, 100, 60, -60, -100, -116])
def test_queries_from_the_ends_of_bf16(held, up):
    """Whole numbers by 2^-up as queries, keys by 2^up: powers of two, exact in every place, so the scores and all
    that follows keep their bits."""
    c = Case(lens=[1000, 40], q_heads=6, k_heads=2, dim=64, page=16, held=held, t="bf16")
    c.q = torch.randint(-100, 101, c.q.shape, generator=gen(1), device=DEV).bfloat16()
    want, wlse = c.run(scale=0.004)
    c.q = c.q * 2.0 ** -up
    c.ks *= 2.0 ** up
    assert bool(c.ks.isfinite().all() & (c.ks >= 2.0 ** -126).logical_or(c.ks == 0).all())
    got, lse = c.run(scale=0.004)
    assert torch.equal(got, want) and torch.equal(lse, wlse)


@pytest.mark.parametrize("held,t", [("bf16", None), ("fp16", None), ("int8", "bf16")])
def test_weights_keep_what_fp32_holds(held, t):
    """Three tokens whose values cancel, for 256 weights w: 1 * 1 - w (c1 + c2) with c1 + c2 next to 1 / w, so that the
    output shows a weight's own error.  The exponents' difference is below 0.87 and off by at most 9 roundings of it
    (5.5 u of the weight), exp2 by 2^-22; three products of 3 terms are summed, each off by at most 2 u of the largest
    (18 u): together below 2^-19 of sum p |v|."""
    b = 256
    c = Case(lens=[3] * b, q_heads=1, k_heads=1, dim=64, page=3, held=held, t=t)
    x = torch.linspace(0.01, 0.99, b, device=DEV).to(c.t)
    w = torch.exp(0.6 * (x.double() - 1))
    k = torch.zeros(b, 3, 64, device=DEV)
    v = torch.zeros(b, 3, 64, device=DEV)
    k[:, 0, 0], k[:, 1, 0], k[:, 2, 0] = 1, x.float(), x.float()
    v[:, 0] = 1
    v[:, 1] = -(1 / w).to(c.t).float()[:, None]
    v[:, 2] = -(1 / w + v[:, 1, 0]).to(c.t).float()[:, None]
    slots = (c.tables[:, :1].long() * 3 + torch.arange(3, device=DEV)).flatten()
    A.cache_write(k.view(-1, 1, 64), v.view(-1, 1, 64), slots, c.kp, c.vp, c.ks, c.vs)
    c.q.zero_()
    c.q[:, 0, 0] = 1
    got, lse = c.run(scale=0.6)
    kk, vv = (c.values(p, s)[c.tables[:, 0].long(), 0] for p, s in ((c.kp, c.ks), (c.vp, c.vs)))
    p = torch.softmax(0.6 * kk[..., 0], -1)[..., None]
    want = (p * vv).sum(1)
    within(got[:, 0], want, 2.0 ** -19 * (p * vv.abs()).sum(1) + torch.finfo(c.t).eps / 2 * want.abs() + 2.0 ** -25)


@pytest.mark.parametrize("n", [90, 9000])
def test_infinite_values_beside_infinite_and_nan_keys(n):
    """A NaN key makes its rows NaN whatever the values; where all scores are -inf the row is zeros and -inf, the
    values infinite or not; the other heads of the same call have their infinities."""
    c = Case(lens=[n, 300, 300], q_heads=12, k_heads=2, dim=64, page=16, held="bf16", seed=n)
    clean, clse = c.run()
    c.vp[..., 5] = math.inf
    c.vp[c.tables[2, :19].long(), 1, :, 6] = -math.inf
    for j in range(300):
        p, w = place(c, 1, j)
        c.kp[p, 0, w] = 0
        c.kp[p, 0, w, 0] = -math.inf
    c.q[1, :, 0] = 1.0
    c.q[0, 3, 9] = math.nan
    got, lse = c.run()
    assert bool(got[0, 3].isnan().all() & lse[0, 3].isnan())
    assert bool((got[1, :6] == 0).all() & (lse[1, :6] == -math.inf).all())
    rows = [(0, h) for h in range(12) if h != 3] + [(1, h) for h in range(6, 12)] + [(2, h) for h in range(12)]
    for b, h in rows:
        assert float(got[b, h, 5]) == math.inf
        assert b != 2 or h < 6 or float(got[b, h, 6]) == -math.inf
        rest = [d for d in range(64) if d != 5 and not (b == 2 and h > 5 and d == 6)]
        assert bool(got[b, h, rest].isfinite().all()) and bool(lse[b, h].isfinite())
        if b != 1:
            assert torch.equal(got[b, h, rest], clean[b, h, rest]) and torch.equal(lse[b, h], clse[b, h])
