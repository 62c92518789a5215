"""The generation operators (chimera_b200.attention) on the GPU against plain
implementations in 64 bits.

Tolerances are bounds from the arithmetic, before any run; u = 2^-24 is the
relative rounding of fp32 and half_step the one of the output's type
(torch.finfo(t).eps / 2).

* rotary: the angle is off by at most 2 pi 2^-26 (fp32 rounding of at most half
  a turn) plus 1e-6 at positions up to 2^31 (stated by the header; tests use
  positions below 2^21, where it is below 1e-9), sine and cosine by 2 ulp more,
  two products, a scaling and a sum by one rounding each: together below 2^-21
  of |scale| (|x0| + |x1|); then one rounding to the type.
* codes and scales: equal.
* attention: a score's error, with dim products summed in fp32 (the tensor
  core's sums may truncate: 2 u per term), is at most
  d = (2 dim + 8) u max_j |scale| sum_d |q_d k_jd|.  A probability relative to
  the sum is then off by 2 d, by 2^-21 from each of two exp2, and by 2^-16 from
  being split into two bf16 terms (2^-9 2^-9, with margin); the sums over n
  tokens by 2 n u, of which runs of 16 and a tree over warps make far less:
  2^-14 covers both up to 2,048 tokens.  So |out - exact| <=
  (2 d + 2^-14) sum_j p_j |v_j| + half_step |out|, and
  |lse - exact| <= d + 2^-14 + 4 u |lse|.
"""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from chimera_b200 import attention as A  # noqa: E402

U = 2.0 ** -24
DEV = "cuda"
NAMES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16, "int8": torch.int8,
         "e4m3": torch.float8_e4m3fn}
TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def half_step(t):
    return torch.finfo(t).eps / 2


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def within(got, want, tol):
    got = got.double()
    same = (got == want) | (got.isnan() & want.isnan())
    off = torch.where(same, torch.zeros_like(want), (got - want).abs())
    assert not bool((off > tol).any() | (off.isnan() & ~same).any()), \
        f"off by {float((off - tol).nan_to_num(1e30).max())} past the tolerance"


# ---- rotary ----------------------------------------------------------------------

def rotary64(x, positions, freqs, interleaved, inverse, scale):
    a = positions.double()[..., None] * freqs
    if inverse:
        a = -a
    c, s = (scale * a.cos())[..., None, :], (scale * a.sin())[..., None, :]
    half = freqs.numel()
    y = x.double().clone()
    i0, i1 = ((slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else
              (slice(0, half), slice(half, 2 * half)))
    x0, x1 = x.double()[..., i0], x.double()[..., i1]
    y[..., i0], y[..., i1] = x0 * c - x1 * s, x0 * s + x1 * c
    room = torch.zeros_like(y)
    room[..., i0] = room[..., i1] = abs(scale) * (x0.abs() + x1.abs())
    return y, room * 2.0 ** -21 + half_step(x.dtype) * y.abs() + 2.0 ** -25


@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("t", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("dim,rot", [(128, 128), (96, 64), (64, 20), (128, 2), (6, 6), (80, 80), (7, 4), (256, 128),
                                     (130, 64), (1030, 1024)])
def test_rotary(dim, rot, t, interleaved, inverse):
    g = gen(dim * 7 + rot)
    dt = NAMES[t]
    freqs = A.rotary_frequencies(rot, device=DEV)
    for b, s, hq, hk in ((1, 1, 1, 1), (2, 7, 5, 3), (3, 33, 4, 1)):
        q = torch.randn(b, s, hq, dim, generator=g, device=DEV).to(dt)
        k = torch.randn(b, s, hk, dim, generator=g, device=DEV).to(dt)
        pos = torch.randint(0, 1 << 21, (b, s), generator=g, device=DEV)
        scale = 1.25
        q0, k0 = q.clone(), k.clone()
        qo, ko = A.rotary(q, k, pos, freqs, interleaved=interleaved, inverse=inverse, scale=scale)
        assert torch.equal(q, q0) and torch.equal(k, k0)
        for got, x in ((qo, q), (ko, k)):
            within(got, *rotary64(x, pos, freqs, interleaved, inverse, scale))
            assert torch.equal(got[..., rot:], x[..., rot:])
        # in place, int32 positions, q alone: the same bits
        got, none = A.rotary(q, None, pos.int(), freqs, interleaved=interleaved, inverse=inverse, scale=scale,
                             q_out=q)
        assert none is None and got is q and torch.equal(q, qo)
        # tokens without a batch, positions shared by a batch
        q3, _ = A.rotary(q0[0], None, pos[0], freqs, interleaved=interleaved, inverse=inverse, scale=scale)
        assert torch.equal(q3, qo[0])
        shared, _ = A.rotary(q0, None, pos[0], freqs, interleaved=interleaved, inverse=inverse, scale=scale)
        assert torch.equal(shared[0], qo[0])


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_strides_and_alignment(interleaved):
    """q and k as views of one projection, out into another layout, bases off a 16-byte boundary."""
    g = gen(5)
    freqs = A.rotary_frequencies(64, device=DEV)
    for t in (torch.bfloat16, torch.float32):
        for lead in (0, 1, 8):
            buf = torch.randn(2, 9, lead + (4 + 2 + 2) * 64, generator=g, device=DEV).to(t)
            qkv = buf[..., lead:].unflatten(-1, (8, 64))
            q, k = qkv[:, :, :4], qkv[:, :, 4:6]
            pos = torch.randint(0, 5000, (9, 2), generator=g, device=DEV).t()
            head_first = torch.empty(2, 4, 9, 64, dtype=t, device=DEV)
            before = buf.clone()
            qo, ko = A.rotary(q, k, pos, freqs, interleaved=interleaved, q_out=head_first.transpose(1, 2))
            assert torch.equal(buf, before)
            within(qo, *rotary64(q, pos, freqs, interleaved, False, 1.0))
            within(ko, *rotary64(k, pos, freqs, interleaved, False, 1.0))
            A.rotary(q, k, pos, freqs, interleaved=interleaved, q_out=q, k_out=k)  # in place inside the projection
            assert torch.equal(q, qo) and torch.equal(k, ko)
            assert torch.equal(qkv[:, :, 6:], before[..., lead:].unflatten(-1, (8, 64))[:, :, 6:])
            assert torch.equal(buf[..., :lead], before[..., :lead])


def test_rotary_far_and_negative_positions():
    freqs = A.rotary_frequencies(128, device=DEV)
    pos = torch.tensor([0, -1, -77, 1 << 20, (1 << 31) - 1, 1 << 31, 12345678901], device=DEV)
    x = torch.randn(7, 2, 128, generator=gen(1), device=DEV)
    got, _ = A.rotary(x, None, pos, freqs)
    want, tol = rotary64(x, pos, freqs, False, False, 1.0)
    far = 1e-6 * pos.abs().double().clamp(min=2.0 ** 31)[:, None, None] / 2.0 ** 31
    within(got, want, tol + far * (x.abs().max().double() * 2))
    assert torch.equal(got[0], x[0])


def test_rotary_inverse_is_the_gradient():
    """Against differences: for L = sum(w * rotary(x)), L is linear in x, so a difference quotient over a step h of
    fp32 values is the gradient up to the roundings of the two sums (2^-21 each, over the step)."""
    freqs = A.rotary_frequencies(32, kind="parts", factor=4, device=DEV)
    g = gen(3)
    for interleaved in (False, True):
        x = torch.randn(5, 2, 40, generator=g, device=DEV)
        w = torch.randn(5, 2, 40, generator=g, device=DEV)
        pos = torch.randint(0, 9000, (5,), generator=g, device=DEV)
        grad, _ = A.rotary(w, None, pos, freqs, interleaved=interleaved, inverse=True, scale=1.3)
        for i in range(0, x.numel(), 7):
            up, down = x.clone(), x.clone()
            up.view(-1)[i] += 0.5
            down.view(-1)[i] -= 0.5
            step = (up.view(-1)[i] - down.view(-1)[i]).double()
            y = [A.rotary(z, None, pos, freqs, interleaved=interleaved, scale=1.3)[0].double() for z in (up, down)]
            num = ((y[0] - y[1]) * w.double()).sum() / step
            # two elements of y differ, each off by 2^-21 1.3 (|x0| + |x1|), times w
            room = 4 * 2.0 ** -21 * 1.3 * 2 * (x.abs().max() + 0.5).double() * w.abs().max().double() / step
            assert abs(num - grad.view(-1)[i].double()) <= room + 1e-6
        back, _ = A.rotary(A.rotary(x, None, pos, freqs, interleaved=interleaved)[0], None, pos, freqs,
                           interleaved=interleaved, inverse=True)
        assert float((back - x).abs().max()) <= 2 * 2.0 ** -21 * 2 * 1.5 * float(x.abs().max())


def test_rotary_of_infinities_keeps_to_its_pair():
    x = torch.ones(1, 1, 16, device=DEV)
    x[0, 0, 3] = math.inf
    x[0, 0, 6] = math.nan
    got, _ = A.rotary(x, None, torch.tensor([3], device=DEV), A.rotary_frequencies(16, device=DEV))
    bad = ~got.isfinite().view(16)
    assert sorted(bad.nonzero().flatten().tolist()) == [3, 6, 11, 14]


def test_rotary_of_nothing():
    freqs = A.rotary_frequencies(64, device=DEV)
    for shape in ((0, 4, 2, 64), (4, 0, 2, 64), (2, 3, 0, 64)):
        q = torch.empty(shape, device=DEV)
        got, _ = A.rotary(q, None, torch.zeros(shape[:2], dtype=torch.int64, device=DEV), freqs)
        assert got.shape == q.shape


# ---- the cache -------------------------------------------------------------------

def make_pages(n, heads, page, dim, held, token_major=False, fill=None):
    shape = (n, page, heads, dim) if token_major else (n, heads, page, dim)
    out = []
    for _ in range(2):
        p = torch.zeros(shape, dtype=torch.float32, device=DEV)
        if fill is not None:
            p.fill_(fill)
        p = p.to(held)
        out.append(p.transpose(1, 2) if token_major else p)
    scales = [torch.full((n, heads, page), -1.0, device=DEV) for _ in range(2)] if held in TOP else [None, None]
    return out[0], out[1], scales[0], scales[1]


def quantised64(x, held):
    """(values of the codes, scales) of the rule the header states, in 64 bits."""
    top = x.double().abs().amax(-1)
    odd = ~x.isfinite().all(-1)
    scale = (top / torch.full_like(top, TOP[held])).float()  # 64-bit quotient, then fp32
    # the largest scale whose top code reads back finite
    most = torch.tensor(torch.finfo(torch.float32).max / TOP[held], dtype=torch.float64).float()
    most = most if most.double() * TOP[held] <= torch.finfo(torch.float32).max else torch.nextafter(most, most * 0)
    scale = torch.where(top < 2.0 ** -96, torch.zeros_like(scale), scale).minimum(most.to(scale.device))
    s = scale.double()[..., None]
    y = torch.where((s > 0) & ~odd[..., None], x.double() / s, torch.zeros_like(x, dtype=torch.float64))
    if held == torch.int8:
        code = y.round()
    else:
        e = torch.frexp(y.abs().clamp(min=2.0 ** -6))[1] - 1
        grid = torch.ldexp(torch.ones(y.shape, dtype=torch.float64), (e - 3).cpu()).to(y.device)
        code = (y / grid).round() * grid
    return code, torch.where(odd, torch.full_like(scale, math.nan), scale)


def rows(pages, slots, page):
    """The vectors at slots, as raw stored elements [n, heads, dim]."""
    at, w = slots // page, slots % page
    if pages.element_size() == 1:
        return pages.view(torch.uint8)[at, :, w].view(pages.dtype)
    return pages[at, :, w]


@pytest.mark.parametrize("token_major", [False, True])
@pytest.mark.parametrize("held", ["int8", "e4m3", "fp16", "bf16"])
@pytest.mark.parametrize("t", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("dim,heads,page", [(128, 8, 16), (64, 5, 48), (96, 3, 1), (16, 1, 7), (256, 2, 64),
                                            (208, 2, 5)])
def test_cache_write_and_read(dim, heads, page, t, held, token_major):
    g = gen(dim + page)
    dt, ht = NAMES[t], NAMES[held]
    n = 131
    pages = -(-n // page) + 4
    kp, vp, ks, vs = make_pages(pages, heads, page, dim, ht, token_major, fill=3.0)
    slots = torch.randperm(pages * page, generator=g, device=DEV)[:n]
    slots[5], slots[77], slots[-1] = -1, pages * page, -(1 << 62)  # skipped
    on = (slots >= 0) & (slots < pages * page)
    x = torch.randn(2, n, heads, dim, generator=g, device=DEV) * torch.exp2(
        torch.randint(-20, 12, (2, n, heads, 1), generator=g, device=DEV).float())
    x = x.to(dt)
    x[0, 0] = 0
    before = kp.float().clone()
    A.cache_write(x[0], x[1], slots, kp, vp, ks, vs)
    free = torch.ones(pages * page, dtype=torch.bool, device=DEV)
    free[slots[on]] = False
    left = free.nonzero().flatten()
    assert torch.equal(rows(kp, left, page).float(), rows(before, left, page))
    for xi, p, s in ((x[0], kp, ks), (x[1], vp, vs)):
        stored = rows(p, slots[on], page).double()
        if ht in TOP:
            code, scale = quantised64(xi[on], ht)
            got = s[slots[on] // page, :, slots[on] % page]
            assert torch.equal(got, scale)
            assert torch.equal(stored, code)
            assert bool((s[left // page, :, left % page] == -1).all())
        else:
            assert torch.equal(stored, xi[on].to(ht).double())
    for out in ("fp32", "fp16", "bf16"):
        ko, vo = A.cache_read(slots, kp, vp, ks, vs, dtype=NAMES[out])
        for xi, got, p, s in ((x[0], ko, kp, ks), (x[1], vo, vp, vs)):
            want = rows(p, slots[on], page).float()
            if ht in TOP:
                want = want * s[slots[on] // page, :, slots[on] % page][..., None]
            assert torch.equal(got[on], want.to(NAMES[out]))
            assert bool((got[~on] == 0).all())


@pytest.mark.parametrize("held", ["int8", "e4m3", "bf16"])
@pytest.mark.parametrize("t", ["fp32", "bf16"])
@pytest.mark.parametrize("tokens,heads", [(8191, 8), (8192, 8), (16383, 8), (16384, 8), (131073, 1), (43691, 3)])
def test_cache_of_many_vectors(tokens, heads, t, held):
    """Counts on both sides of where the kernels take several vectors per thread, and not multiples of them."""
    ht, dim, page = NAMES[held], 32, 16
    g = gen(tokens)
    n = -(-tokens // page)
    kp, vp, ks, vs = make_pages(n, heads, page, dim, ht)
    x = torch.randn(2, tokens, heads, dim, generator=g, device=DEV).to(NAMES[t])
    slots = torch.randperm(n * page, generator=g, device=DEV)[:tokens]
    slots[-3] = -1
    A.cache_write(x[0], x[1], slots, kp, vp, ks, vs)
    k, v = A.cache_read(slots, kp, vp, ks, vs, dtype=torch.float32)
    for xi, got in ((x[0], k), (x[1], v)):
        if ht in TOP:
            code, scale = quantised64(xi, ht)
            want = code.float() * scale[..., None]
        else:
            want = xi.to(ht).float()
        want[-3] = 0
        assert torch.equal(got, want)


@pytest.mark.parametrize("held", ["int8", "e4m3"])
def test_cache_codes_at_ties_and_neighbours(held):
    """Quotients on, just above and just below the middle between two codes: scale 1 and scales that are not
    powers of two, of both signs."""
    ht = NAMES[held]
    top = TOP[ht]
    if held == "int8":
        mids = torch.arange(-126, 127, dtype=torch.float64) + 0.5
    else:
        vals = torch.arange(0, 127, dtype=torch.int16).to(torch.uint8).view(torch.float8_e4m3fn).double()
        mids = torch.cat([(vals[1:] + vals[:-1]) / 2, -(vals[1:] + vals[:-1]) / 2])
    points = mids.float()
    points = torch.cat([points, torch.nextafter(points, points + 1), torch.nextafter(points, points - 1),
                        torch.nextafter(torch.zeros(1), torch.ones(1)), torch.zeros(1)])
    lot = points[torch.randperm(points.numel(), generator=torch.Generator().manual_seed(0))]
    lot = torch.cat([lot, torch.zeros(-lot.numel() % 120)]).view(-1, 120)
    x = torch.zeros(lot.shape[0], 1, 128)
    x[:, 0, :120] = lot
    x[:, 0, 127] = top
    for unit in (1.0, 2.0 ** -40, 3.0, 0.7, 1e-3, 2.0 ** 60, 1.1754944e-20):
        y = (x.double() * unit).float().to(DEV)
        n = y.shape[0]
        kp, vp, ks, vs = make_pages(n, 1, 1, 128, ht)
        slots = torch.arange(n, device=DEV)
        A.cache_write(y, y, slots, kp, vp, ks, vs)
        code, scale = quantised64(y, ht)
        assert torch.equal(ks[:, :, 0], scale)
        assert torch.equal(rows(kp, slots, 1).double(), code)
        assert torch.equal(rows(vp, slots, 1).double(), code)


@pytest.mark.parametrize("held", ["int8", "e4m3"])
@pytest.mark.parametrize("t", ["bf16", "fp16"])
def test_cache_codes_of_every_fraction(t, held):
    """Every fraction of a 16-bit type under every largest value's fraction, over the exponents that get codes: exact
    ties, scales rounded up, down and not at all."""
    ht, dt = NAMES[held], NAMES[t]
    bits = 8 if t == "bf16" else 11
    n = 1 << (bits - 1)
    part = torch.arange(n, 2 * n, device=DEV, dtype=torch.float64) / n    # 1 to 2
    for e in range(0, 20 if held == "e4m3" else 10):
        lot = torch.cat([part, torch.zeros(-n % 127, device=DEV, dtype=torch.float64)]).view(-1, 127) * 2.0 ** -e
        x = torch.zeros(n, lot.shape[0], 128, device=DEV, dtype=torch.float64)
        x[:, :, :127] = lot
        x[:, :, 127] = 2.0 if e == 0 else 1.0
        x[:, :, 127] *= part[:, None]
        x = x.view(-1, 1, 128)
        sign = torch.where(torch.arange(128, device=DEV) % 2 == 0, 1.0, -1.0)
        y = (x * sign).to(dt)
        kp, vp, ks, vs = make_pages(y.shape[0], 1, 1, 128, ht)
        A.cache_write(y, y, torch.arange(y.shape[0], device=DEV), kp, vp, ks, vs)
        code, scale = quantised64(y, ht)
        assert torch.equal(ks[:, :, 0], scale)
        assert torch.equal(kp.view(-1, 128).double(), code.view(-1, 128))


@pytest.mark.parametrize("held", ["int8", "e4m3"])
def test_cache_holds_odd_vectors(held):
    ht = NAMES[held]
    x = torch.ones(8, 2, 32, device=DEV)
    x[0, 0, 5] = math.inf
    x[1, 1, 31] = math.nan
    x[2, 0, 0] = -math.inf
    x[3] = 2.0 ** -97          # held as zeros
    x[4] = 2.0 ** -96          # the smallest that is held
    x[5] = torch.finfo(torch.float32).max
    x[6] = -0.0
    x[7, 0] = torch.finfo(torch.float32).tiny / 4
    kp, vp, ks, vs = make_pages(1, 2, 8, 32, ht)
    slots = torch.arange(8, device=DEV)
    A.cache_write(x, x.flip(0), slots, kp, vp, ks, vs)
    k, v = A.cache_read(slots, kp, vp, ks, vs, dtype=torch.float32)
    assert bool(k[0, 0].isnan().all() & k[1, 1].isnan().all() & k[2, 0].isnan().all())
    assert bool((k[0, 1] == 1).all() & (k[1, 0] == 1).all() & (k[2, 1] == 1).all())
    assert bool((k[3] == 0).all() & (k[6] == 0).all() & (k[7, 0] == 0).all() & (k[7, 1] == 1).all())
    assert torch.equal(ks[0, :, 3], torch.zeros(2, device=DEV))
    for i in (4, 5):
        assert float((k[i] / x[i] - 1).abs().max()) <= 2.0 ** -22  # code is the top one: the scale's two roundings
    assert torch.equal(v.nan_to_num(7), k.flip(0).nan_to_num(7))


@pytest.mark.parametrize("held", ["int8", "e4m3"])
def test_cache_reads_every_code(held):
    ht = NAMES[held]
    codes = torch.arange(256, device=DEV).to(torch.uint8).view(1, 1, 1, 256).view(ht)
    s = torch.full((1, 1, 1), 0.375, device=DEV)
    k, v = A.cache_read(torch.zeros(1, dtype=torch.int64, device=DEV), codes, codes.clone(), s, s.clone(),
                        dtype=torch.float32)
    want = codes.float().view(-1) * 0.375  # e4m3: 0x7f and 0xff are NaN
    assert torch.equal(k.view(-1).nan_to_num(7e9), want.nan_to_num(7e9))
    assert torch.equal(v.view(-1).nan_to_num(7e9), want.nan_to_num(7e9))


def test_cache_takes_views_off_a_boundary():
    g = gen(9)
    buf = torch.randn(21, 1 + 3 * 4 * 64, generator=g, device=DEV).bfloat16()
    for lead in (0, 1):
        qkv = buf[:, lead:lead + 768].unflatten(-1, (12, 64))
        k, v = qkv[:, 4:8], qkv[:, 8:]
        a, b = make_pages(3, 4, 8, 64, torch.int8), make_pages(3, 4, 8, 64, torch.int8)
        slots = torch.arange(21, device=DEV)
        A.cache_write(k, v, slots, *a)
        A.cache_write(k.contiguous(), v.contiguous(), slots, *b)
        assert all(torch.equal(x, y) for x, y in zip(a, b))
        out = torch.zeros(21, 1 + 2 * 4 * 64, dtype=torch.bfloat16, device=DEV)
        views = out[:, lead:lead + 512].unflatten(-1, (8, 64))
        A.cache_read(slots, *a, k_out=views[:, :4], v_out=views[:, 4:])
        ko, vo = A.cache_read(slots, *b)
        assert torch.equal(views[:, :4], ko) and torch.equal(views[:, 4:], vo)
        assert bool((out[:, :lead] == 0).all() & (out[:, lead + 512:] == 0).all())


# ---- attention -------------------------------------------------------------------

class Case:
    def __init__(self, *, lens, q_heads, k_heads, dim, page, held, t=None, token_major=False, starts=None, seed=0,
                 loud=1.0, spare=2, width=None):
        g = gen(seed)
        self.ht, self.t = NAMES[held], NAMES[t or held]
        self.page, self.lens, self.starts = page, lens, starts
        b = len(lens)
        need = [-(-max(n, 0) // page) for n in lens]
        self.n = sum(need) + spare
        shape = (self.n, k_heads, page, dim)
        kv = torch.randn(2, *shape, generator=g, device=DEV) * loud
        self.kp, self.vp, self.ks, self.vs = make_pages(self.n, k_heads, page, dim, self.ht, token_major)
        slots = torch.arange(self.n * page, device=DEV)
        flat = kv.transpose(2, 3).reshape(2, self.n * page, k_heads, dim).contiguous()
        A.cache_write(flat[0], flat[1], slots, self.kp, self.vp, self.ks, self.vs)
        self.q = (torch.randn(b, q_heads, dim, generator=g, device=DEV) * 1.5).to(self.t)
        order = torch.randperm(self.n, generator=g, device=DEV).int()
        width = width or max([1] + need)
        self.tables = torch.full((b, width), -7, dtype=torch.int32, device=DEV)
        at = 0
        for i, m in enumerate(need):
            self.tables[i, :m] = order[at:at + m]
            at += m
        self.l = torch.tensor(lens, dtype=torch.int32, device=DEV)
        self.s = torch.tensor(starts, dtype=torch.int32, device=DEV) if starts is not None else None
        self.scale = dim ** -0.5

    def cache(self):
        return self.kp, self.vp

    def run(self, **kw):
        return A.paged_attention(self.q, self.kp, self.vp, self.tables, self.l, self.ks, self.vs, starts=self.s, **kw)

    def values(self, p, s):
        x = p.float().double()
        return x if s is None else x * s.double()[..., None]

    def expected(self):
        k, v = self.values(self.kp, self.ks), self.values(self.vp, self.vs)
        b, hq, dim = self.q.shape
        group = hq // k.shape[1]
        out = torch.zeros(b, hq, dim, dtype=torch.float64, device=DEV)
        tol = torch.zeros_like(out)
        lse = torch.full((b, hq), -math.inf, dtype=torch.float64, device=DEV)
        ltol = torch.zeros_like(lse)
        for i, n in enumerate(self.lens):
            first = max(self.starts[i], 0) if self.starts is not None else 0
            if n <= first:
                continue
            pages = self.tables[i, :-(-n // self.page)].long()
            ki = k[pages].transpose(0, 1).flatten(1, 2)[:, first:n].repeat_interleave(group, 0)
            vi = v[pages].transpose(0, 1).flatten(1, 2)[:, first:n].repeat_interleave(group, 0)
            q = self.q[i].double()
            s = torch.einsum("hd,hnd->hn", q, ki) * self.scale
            d = (2 * dim + 8) * U * abs(self.scale) * torch.einsum("hd,hnd->hn", q.abs(), ki.abs()).amax(-1)
            p = torch.softmax(s, -1)
            out[i] = torch.einsum("hn,hnd->hd", p, vi)
            lse[i] = torch.logsumexp(s, -1)
            tol[i] = (2 * d[:, None] + 2.0 ** -14) * torch.einsum("hn,hnd->hd", p, vi.abs()) + \
                half_step(self.t) * out[i].abs() + 2.0 ** -25
            ltol[i] = d + 2.0 ** -14 + 4 * U * lse[i].abs()
        return out, lse, tol, ltol

    def check(self, **kw):
        got, lse = self.run(**kw)
        out, want, tol, ltol = self.expected()
        within(got, out, tol)
        within(lse, want, ltol)
        return got, lse


LENS = [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 255, 257, -3, 1000]


@pytest.mark.parametrize("held,t", [("bf16", None), ("fp16", None), ("int8", "bf16"), ("int8", "fp16"),
                                    ("e4m3", "bf16"), ("e4m3", "fp16")])
@pytest.mark.parametrize("dim", [16, 48, 64, 96, 128, 192, 256])
def test_attention_types_and_widths(dim, held, t):
    Case(lens=LENS, q_heads=8, k_heads=2, dim=dim, page=16, held=held, t=t, seed=dim).check()


@pytest.mark.parametrize("held,t", [("bf16", None), ("int8", "fp16"), ("e4m3", "bf16")])
@pytest.mark.parametrize("group,k_heads", [(1, 1), (1, 7), (3, 2), (7, 2), (8, 3), (9, 2), (16, 1), (17, 1), (40, 1)])
def test_attention_head_layouts(group, k_heads, held, t):
    for dim in (64, 128, 160):
        Case(lens=LENS, q_heads=group * k_heads, k_heads=k_heads, dim=dim, page=16, held=held, t=t,
             seed=group).check()


@pytest.mark.parametrize("token_major", [False, True])
@pytest.mark.parametrize("held,t", [("fp16", None), ("int8", "bf16")])
@pytest.mark.parametrize("page", [1, 5, 32, 257, 4096])
def test_attention_pages(page, held, t, token_major):
    Case(lens=LENS, q_heads=12, k_heads=3, dim=128, page=page, held=held, t=t, token_major=token_major,
         seed=page).check()


@pytest.mark.parametrize("held,t", [("bf16", None), ("e4m3", "fp16")])
def test_attention_starts(held, t):
    starts = [0, 0, 5, 3, 16, 0, -9, 1, 62, 64, 1, 128, 100, 128, 17, 250, 0, 900]
    Case(lens=LENS, starts=starts, q_heads=8, k_heads=2, dim=128, page=16, held=held, t=t).check()


@pytest.mark.parametrize("held,t", [("bf16", None), ("int8", "bf16"), ("e4m3", "fp16")])
@pytest.mark.parametrize("lens", [[2047], [2048, 1, 2000], [300] * 67, [0] * 5, [1] * 300, [0, 2048, 0]])
def test_attention_batches(lens, held, t):
    Case(lens=lens, q_heads=14, k_heads=2, dim=128, page=32, held=held, t=t, seed=len(lens)).check()


@pytest.mark.parametrize("held,t", [("bf16", None), ("fp16", None), ("int8", "bf16")])
def test_attention_of_peaked_and_flat_scores(held, t):
    """Scores in the thousands (one token takes all) and all alike (zero queries)."""
    c = Case(lens=[1500, 700], q_heads=8, k_heads=2, dim=128, page=16, held=held, t=t, loud=60.0)
    c.check()
    c.q.zero_()
    c.check()
    c.scale = 0.0
    c.check(scale=0.0)
    c.scale = -0.3
    c.q.normal_(generator=gen(2))
    c.check(scale=-0.3)


@pytest.mark.parametrize("held,t", [("bf16", None), ("fp16", None), ("int8", "bf16"), ("e4m3", "bf16")])
def test_attention_does_not_read_past_the_range(held, t):
    """Everything outside the attended range is NaN or an infinity, in the last page and in pages of no sequence."""
    lens, starts = [1, 17, 100, 130, 0, 40], [0, 3, 0, 127, 0, 40]
    c = Case(lens=lens, starts=starts, q_heads=8, k_heads=2, dim=64, page=24, held=held, t=t)
    want, wlse = c.run()
    used = torch.zeros(c.n, 24, dtype=torch.bool, device=DEV)
    for i, (n, f) in enumerate(zip(lens, starts)):
        for j in range(f, n):
            used[int(c.tables[i, j // 24]), j % 24] = True
    for bad in (math.nan, math.inf, -math.inf):
        for p, s in ((c.kp, c.ks), (c.vp, c.vs)):
            where = ~used[:, None, :].expand(c.n, 2, 24)
            if s is None:
                p[where] = bad
            else:
                s[where] = bad
        got, lse = c.run()
        assert torch.equal(got, want) and torch.equal(lse, wlse)
    assert bool((got[4] == 0).all() & (got[5] == 0).all() & (lse[4] == -math.inf).all() & (lse[5] == -math.inf).all())


@pytest.mark.parametrize("held", ["bf16", "int8"])
def test_attention_with_nan_and_infinite_tokens(held):
    c = Case(lens=[200, 200, 200, 90], q_heads=4, k_heads=2, dim=64, page=16, held=held, t="bf16")
    clean, clse = c.run()

    def poke(p, s, b, token, value, head=0):
        page = int(c.tables[b, token // 16])
        if s is None:
            p[page, head, token % 16, 3] = value
        else:
            s[page, head, token % 16] = math.nan
    poke(c.kp, c.ks, 0, 150, math.nan)          # a NaN key: the rows of its head
    poke(c.vp, c.vs, 1, 7, math.nan)            # a NaN value: its element (8 bits: its vector's scale)
    got, lse = c.run()
    assert bool(got[0, :2].isnan().all() & lse[0, :2].isnan().all())
    assert torch.equal(got[0, 2:], clean[0, 2:]) and torch.equal(lse[1:], clse[1:])
    if held == "bf16":
        assert bool(got[1, :2, 3].isnan().all()) and torch.equal(got[1, :2, 4:], clean[1, :2, 4:])
    else:
        assert bool(got[1, :2].isnan().all())
    assert torch.equal(got[1, 2:], clean[1, 2:]) and torch.equal(got[2:], clean[2:])


def test_attention_over_every_code():
    """Caches of arbitrary bytes: int8's -128, and e4m3's NaN codes, which make their own NaN and no other."""
    g = gen(6)
    for held in ("int8", "e4m3"):
        ht = NAMES[held]
        raw = torch.randint(0, 256, (2, 9, 2, 16, 128), generator=g, device=DEV).to(torch.uint8)
        if held == "e4m3":
            raw = torch.where((raw & 0x7F) == 0x7F, torch.zeros_like(raw), raw)
        c = Case(lens=[140], q_heads=4, k_heads=2, dim=128, page=16, held=held, t="bf16", spare=0)
        c.kp, c.vp = raw[0].clone().view(ht), raw[1].clone().view(ht)
        c.q = c.q * (0.02 if held == "int8" else 0.05)
        clean, clse = c.check()
        if held == "e4m3":
            c.vp.view(torch.uint8)[c.tables[0, 3], 1, 5, 77] = 0xFF
            got, lse = c.run()
            bad = got.isnan()
            assert bool(bad[0, 2:, 77].all()) and int(bad.sum()) == 2 and torch.equal(lse, clse)
            c.kp.view(torch.uint8)[c.tables[0, 8], 0, 2, 0] = 0x7F
            got, lse = c.run()
            assert bool(got[0, :2].isnan().all() & lse[0, :2].isnan().all()) and torch.equal(lse[0, 2:], clse[0, 2:])


@pytest.mark.parametrize("held", ["int8", "e4m3"])
@pytest.mark.parametrize("by", [0.0, 2.0 ** -94, 2.0 ** -60, 2.0 ** 100])
def test_attention_of_values_of_any_size(held, by):
    """Values that are all zero, near the smallest that are held, and huge: the weights carry their scale, lse does
    not.  Below 2^-80 a weight may be held by fp16's 11 bits alone: 2^-11 of sum p |v| more."""
    c = Case(lens=[3000, 40, 1], q_heads=6, k_heads=2, dim=64, page=16, held=held, t="bf16")
    flat = torch.randn(c.n * 16, 2, 64, generator=gen(7), device=DEV)
    slots = torch.arange(c.n * 16, device=DEV)
    k, _ = A.cache_read(slots, c.kp, c.vp, c.ks, c.vs, dtype=torch.float32)
    A.cache_write(k, flat * by, slots, c.kp, c.vp, c.ks, c.vs)
    got, lse = c.run()
    c.vs = c.vs.double() / (by or 1.0)     # the same values of ordinary size, in 64 bits
    out, want, tol, ltol = c.expected()
    within(lse, want, ltol)
    assert bool(lse.isfinite().all())
    room = tol + (2.0 ** -11 * 5 if by < 2.0 ** -80 else 0)
    within(got.double() / (by or 1.0), out, room)


@pytest.mark.parametrize("held,t", [("int8", "bf16"), ("e4m3", "bf16"), ("bf16", None)])
@pytest.mark.parametrize("up", [90, -90])
def test_attention_of_queries_and_keys_far_from_one(held, t, up):
    """Queries by 2^-up and keys by 2^up: powers of two, so the scores are the same."""
    c = Case(lens=[1000, 40], q_heads=6, k_heads=2, dim=64, page=16, held=held, t=t)
    want, wlse = c.run()
    c.q = c.q * 2.0 ** -up
    if c.ks is None:
        c.kp *= 2.0 ** up
    else:
        c.ks *= 2.0 ** up
    got, lse = c.run()
    assert torch.equal(got, want) and torch.equal(lse, wlse)


def test_attention_of_many_sequences():
    lens = [(i * 7) % 40 for i in range(5000)]
    c = Case(lens=lens, q_heads=4, k_heads=1, dim=16, page=16, held="fp16", width=64)
    got, lse = c.run()
    few = [0, 1, 2, 127, 128, 129, 2500, 4998, 4999]
    c.lens = [lens[i] for i in few]
    c.q, c.tables = c.q[few], c.tables[few]
    out, want, tol, ltol = c.expected()
    within(got[few], out, tol)
    within(lse[few], want, ltol)


def test_attention_where_every_score_is_minus_infinity():
    """Infinite keys: all scores -inf gives an empty row, some -inf leave the others."""
    c = Case(lens=[150, 150], q_heads=2, k_heads=1, dim=16, page=16, held="bf16")
    c.q.fill_(1.0)
    for j in range(150):
        c.kp[int(c.tables[0, j // 16]), 0, j % 16, 0] = -math.inf
        if j % 2:
            c.kp[int(c.tables[1, j // 16]), 0, j % 16, 0] = -math.inf
    got, lse = c.run()
    assert bool((got[0] == 0).all() & (lse[0] == -math.inf).all())
    out, want, tol, ltol = c.expected()
    ok = torch.isfinite(c.kp.float()).all(-1)[c.tables[1].long(), 0].flatten()[:150]
    k = c.values(c.kp, None)[c.tables[1].long(), 0].flatten(0, 1)[:150][ok]
    v = c.values(c.vp, None)[c.tables[1].long(), 0].flatten(0, 1)[:150][ok]
    s = c.q[1].double() @ k.t() * c.scale
    p = torch.softmax(s, -1)
    within(got[1], p @ v, 2.0 ** -7 * (p @ v.abs()))  # the output's half step and the bound above, with room
    within(lse[1], torch.logsumexp(s, -1), torch.full((2,), 2.0 ** -12, dtype=torch.float64, device=DEV))


def test_attention_marks_what_does_not_fit():
    c = Case(lens=[100, 100, 100, 100, 16, 40], q_heads=4, k_heads=2, dim=64, page=16, held="int8", t="bf16")
    want, wlse = c.run()
    c.tables[0, 3] = -1                       # needed
    c.tables[1, 6] = c.n                      # needed
    c.tables[2, 0] = torch.iinfo(torch.int32).max
    c.l[3] = c.tables.shape[1] * 16 + 1       # past the table
    c.tables[4, 1:] = -5                      # not needed
    got, lse = c.run()
    assert bool(got[:4].isnan().all() & lse[:4].isnan().all())
    assert torch.equal(got[4:], want[4:]) and torch.equal(lse[4:], wlse[4:])
    c.l.fill_(torch.iinfo(torch.int32).max)
    got, lse = c.run()
    assert bool(got.isnan().all() & lse.isnan().all())
    c.l.fill_(torch.iinfo(torch.int32).min)
    got, lse = c.run()
    assert bool((got == 0).all() & (lse == -math.inf).all())


def test_attention_start_does_not_need_the_pages_before_it():
    c = Case(lens=[100], starts=[70], q_heads=4, k_heads=2, dim=64, page=16, held="bf16")
    want, _ = c.run()
    c.tables[0, :4] = -1
    got, _ = c.run()
    assert torch.equal(got, want)


def test_attention_strides():
    c = Case(lens=[33, 70, 0], q_heads=6, k_heads=2, dim=48, page=16, held="bf16")
    want, wlse = c.run()
    wide = torch.zeros(3, 6, 51, dtype=torch.bfloat16, device=DEV)
    wide[..., 1:49] = c.q
    out = torch.full((6, 3, 50), 9.0, dtype=torch.bfloat16, device=DEV)
    tables = torch.full((3, 40), -1, dtype=torch.int32, device=DEV)
    tables[:, 3:3 + c.tables.shape[1]] = c.tables
    got, lse = A.paged_attention(wide[..., 1:49], c.kp, c.vp, tables[:, 3:], c.l, out=out.transpose(0, 1)[..., 1:49])
    # a wider table may split the sequences elsewhere: the same up to the bound, not bit for bit
    exact, elog, tol, ltol = c.expected()
    within(got, exact, tol)
    within(lse, elog, ltol)
    got, lse = A.paged_attention(wide[..., 1:49], c.kp, c.vp, tables[:, 3:3 + c.tables.shape[1]], c.l,
                                 out=out.transpose(0, 1)[..., 1:49])
    assert torch.equal(got, want) and torch.equal(lse, wlse)
    assert bool((out[..., 0] == 9).all() & (out[..., 49] == 9).all())


def test_attention_and_cache_past_32_bits():
    """Pages whose elements lie beyond 2^31 and 2^32 elements from the first."""
    page, heads, dim = 16, 2, 64
    stride = 1 << 24
    n = 300  # 2^24 * 300 > 2^32 elements
    k = torch.empty(stride * (n - 1) + page * heads * dim, dtype=torch.int8, device=DEV)
    v = torch.empty_like(k)
    shape, st = (n, heads, page, dim), (stride, page * dim, dim, 1)
    kp, vp = k.as_strided(shape, st), v.as_strided(shape, st)
    ks, vs = (torch.zeros(n, heads, page, device=DEV) for _ in range(2))
    g = gen(4)
    x = torch.randn(2, 40, heads, dim, generator=g, device=DEV)
    pages = torch.tensor([299, 128, 256], device=DEV)
    i = torch.arange(40, device=DEV)
    slots = pages[i // page] * page + i % page
    A.cache_write(x[0], x[1], slots, kp, vp, ks, vs)
    small = make_pages(3, heads, page, dim, torch.int8)
    A.cache_write(x[0], x[1], i, *small)
    far, near = A.cache_read(slots, kp, vp, ks, vs), A.cache_read(i, *small)
    assert torch.equal(far[0], near[0]) and torch.equal(far[1], near[1])
    q = torch.randn(1, 4, dim, generator=g, device=DEV).bfloat16()
    lens = torch.tensor([40], dtype=torch.int32, device=DEV)
    a = A.paged_attention(q, kp, vp, pages.int()[None], lens, ks, vs)
    b = A.paged_attention(q, small[0], small[1], torch.arange(3, dtype=torch.int32, device=DEV)[None], lens,
                          small[2], small[3])
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_attention_of_nothing():
    c = Case(lens=[5, 9], q_heads=4, k_heads=2, dim=64, page=16, held="bf16")
    out, lse = A.paged_attention(c.q[:0], c.kp, c.vp, c.tables[:0], c.l[:0])
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    empty = torch.empty(2, 0, dtype=torch.int32, device=DEV)
    out, lse = A.paged_attention(c.q, c.kp, c.vp, empty, torch.zeros_like(c.l))
    assert bool((out == 0).all() & (lse == -math.inf).all())
    out, lse = A.paged_attention(c.q, c.kp[:0], c.vp[:0], empty, torch.zeros_like(c.l))
    assert bool((out == 0).all())
    out, lse = A.paged_attention(c.q, c.kp, c.vp, empty, c.l)
    assert bool(out.isnan().all() & lse.isnan().all())


@pytest.mark.parametrize("held,t,group", [("bf16", None, 7), ("fp16", None, 12), ("int8", "bf16", 4), ("e4m3", "fp16", 1)])
@pytest.mark.parametrize("lens", [[20011], [1, 9000, 0, 5, 17000]])
def test_attention_split_over_its_length(lens, held, t, group):
    """Sequences cut into many parts.  The sums over n tokens add 2 n u of sum p |v| to the bound."""
    c = Case(lens=lens, q_heads=2 * group, k_heads=2, dim=128, page=16, held=held, t=t, seed=group)
    got, lse = c.run()
    out, want, tol, ltol = c.expected()
    more = 2 * max(lens) * U
    within(got, out, tol + more * c.values(c.vp, c.vs).abs().amax())
    within(lse, want, ltol + more)
    whole = c.tables.clone()
    worst = max(range(len(lens)), key=lambda i: lens[i])
    c.tables[worst, lens[worst] // 32] = c.n + 7   # a page in the middle that is not there
    got2, lse2 = c.run()
    assert bool(got2[worst].isnan().all() & lse2[worst].isnan().all())
    c.tables = whole
    rest = [i for i in range(len(lens)) if i != worst]
    assert all(torch.equal(got2[i], got[i]) and torch.equal(lse2[i], lse[i]) for i in rest)
    # one token left of the longest
    c.s = torch.zeros(len(lens), dtype=torch.int32, device=DEV)
    c.starts = [0] * len(lens)
    c.starts[worst] = lens[worst] - 1
    c.s[worst] = lens[worst] - 1
    c.check()


@pytest.mark.parametrize("held,t", [("bf16", None), ("int8", "bf16")])
@pytest.mark.parametrize("batch", [1, 63, 64])
@pytest.mark.parametrize("tokens", [128, 144, 256, 272, 512, 528, 1024, 1040])
def test_attention_where_segments_begin_to_split(tokens, batch, held, t):
    """Tables on both sides of the sizes up to which a sequence stays whole, with many heads and sequences and few."""
    g = torch.Generator().manual_seed(tokens + batch)
    lens = [tokens] + torch.randint(0, tokens + 1, (batch - 1,), generator=g).tolist()
    Case(lens=lens, q_heads=6, k_heads=2, dim=64, page=16, held=held, t=t, seed=batch, width=tokens // 16).check()


def test_attention_in_place_and_without_pages():
    c = Case(lens=[700, 3, 2000], q_heads=16, k_heads=2, dim=64, page=16, held="e4m3", t="bf16")
    want, _ = c.run()
    got, _ = c.run(out=c.q)
    assert got is c.q and torch.equal(got, want)
    none = c.kp[:0], c.vp[:0]
    out, lse = A.paged_attention(c.q, *none, c.tables, c.l, c.ks[:0], c.vs[:0])
    assert bool(out.isnan().all() & lse.isnan().all())


def test_graph_of_split_sequences():
    """Two calls captured back to back on one workspace, replayed as lengths and caches change."""
    c = Case(lens=[1, 9000, 0, 4000], q_heads=16, k_heads=2, dim=128, page=16, held="bf16")
    d = Case(lens=[6000, 70, 0, 0], q_heads=16, k_heads=2, dim=128, page=16, held="bf16", seed=1,
             width=c.tables.shape[1])
    ws = torch.empty(A.paged_attention_workspace(c.kp, c.vp, 4, 16, c.tables.shape[1]), dtype=torch.uint8, device=DEV)
    c.run(workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, b = c.run(workspace=ws), d.run(workspace=ws)
    for lens in ([1, 9000, 0, 4000], [0, 17, 0, 4000], [16, 8999, 3000, 1]):
        c.l.copy_(torch.tensor(lens, device=DEV))
        c.tables[2] = c.tables[1]   # two sequences may share pages
        d.q.normal_()
        ws.fill_(0xFF)
        graph.replay()
        got = [x.clone() for x in (*a, *b)]
        want = [*c.run(), *d.run()]
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_results_do_not_depend_on_the_run():
    c = Case(lens=[1900, 3, 700, 0, 64], q_heads=28, k_heads=4, dim=128, page=16, held="e4m3", t="bf16")
    a = c.run()
    for _ in range(10):
        b = c.run()
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_streams_and_workspaces():
    """Two calls in flight on streams of their own, with workspaces of their own and without."""
    c = Case(lens=[1500, 20, 800], q_heads=16, k_heads=2, dim=128, page=16, held="bf16")
    d = Case(lens=[90, 1990], q_heads=16, k_heads=2, dim=128, page=16, held="bf16", seed=5)
    want = c.run(), d.run()
    need = max(A.paged_attention_workspace(x.kp, x.vp, x.q.shape[0], 16, x.tables.shape[1]) for x in (c, d))
    ws = [torch.empty(need, dtype=torch.uint8, device=DEV) for _ in range(2)]
    s = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for k in range(8):
        for i, x in enumerate((c, d)):
            out = torch.zeros_like(x.q)
            lse = torch.zeros(x.q.shape[:2], device=DEV)
            s[i].wait_stream(torch.cuda.current_stream())
            x.run(stream=s[i], workspace=ws[i] if k % 2 else None, out=out, lse=lse)
            got.append((i, out, lse))
    torch.cuda.synchronize()
    for i, out, lse in got:
        assert torch.equal(out, want[i][0]) and torch.equal(lse, want[i][1])


def test_graphs():
    """A decoding step captured, then replayed over changing inputs; two graphs with workspaces of their own."""
    heads, dim, page = 2, 64, 16
    freqs = A.rotary_frequencies(dim, device=DEV)
    kp, vp, ks, vs = make_pages(8, heads, page, dim, torch.int8)
    q = torch.zeros(2, 6, dim, dtype=torch.bfloat16, device=DEV)
    k, v = (torch.zeros(2, heads, dim, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    pos = torch.zeros(2, dtype=torch.int64, device=DEV)
    slots = torch.zeros(2, dtype=torch.int64, device=DEV)
    lens = torch.zeros(2, dtype=torch.int32, device=DEV)
    tables = torch.arange(8, dtype=torch.int32, device=DEV).view(2, 4)

    def step():
        a, b = A.rotary(q, k, pos, freqs)
        A.cache_write(b, v, slots, kp, vp, ks, vs)
        return A.paged_attention(a, kp, vp, tables, lens, ks, vs)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    g = gen(8)
    for i in range(64):
        q.copy_(torch.randn(q.shape, generator=g, device=DEV))
        k.copy_(torch.randn(k.shape, generator=g, device=DEV))
        v.copy_(torch.randn(v.shape, generator=g, device=DEV))
        pos.fill_(i)
        slots.copy_(torch.tensor([i, 64 + i], device=DEV))
        lens.fill_(i + 1)
        graph, out = graphs[i % 2]
        graph.replay()
        got = out[0].clone(), out[1].clone()
        want = step()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("held", ["bf16", "int8", "e4m3"])
def test_generation_run(held):
    """The operators together as a reader uses them: two prompts read in, then tokens one by one; every step against
    a dense 64-bit softmax over the keys and values the cache reads back."""
    g = gen(11)
    ht = NAMES[held]
    hq, hk, dim, page = 12, 4, 128, 16
    freqs = A.rotary_frequencies(dim, kind="parts", factor=4, device=DEV)
    scale = 0.1 * math.log(4) + 1
    kp, vp, ks, vs = make_pages(40, hk, page, dim, ht)
    prompts = [70, 33]
    tables = torch.randperm(40, generator=g, device=DEV).int().view(2, 20)
    lens = torch.zeros(2, dtype=torch.int32, device=DEV)

    def slot(b, p):
        return tables[b].long()[p // page] * page + p % page

    for b, n in enumerate(prompts):
        p = torch.arange(n, device=DEV)
        q, k = (torch.randn(n, h, dim, generator=g, device=DEV).bfloat16() for h in (hq, hk))
        v = torch.randn(n, hk, dim, generator=g, device=DEV).bfloat16()
        _, k = A.rotary(q, k, p, freqs, scale=scale)
        A.cache_write(k, v, slot(b, p), kp, vp, ks, vs)
        lens[b] = n
    for _ in range(20):
        p = lens.long()
        q, k = (torch.randn(2, h, dim, generator=g, device=DEV).bfloat16() for h in (hq, hk))
        v = torch.randn(2, hk, dim, generator=g, device=DEV).bfloat16()
        q, k = A.rotary(q, k, p, freqs, scale=scale)
        slots = torch.stack([slot(b, p[b]) for b in range(2)])
        A.cache_write(k, v, slots, kp, vp, ks, vs)
        lens += 1
        out, lse = A.paged_attention(q, kp, vp, tables, lens, ks, vs)
        for b in range(2):
            n = int(lens[b])
            kk, vv = A.cache_read(slot(b, torch.arange(n, device=DEV)), kp, vp, ks, vs, dtype=torch.float32)
            kk = kk.double().transpose(0, 1).repeat_interleave(3, 0)
            vv = vv.double().transpose(0, 1).repeat_interleave(3, 0)
            s = torch.einsum("hd,hnd->hn", q[b].double(), kk) * dim ** -0.5
            d = (2 * dim + 8) * U * dim ** -0.5 * torch.einsum("hd,hnd->hn", q[b].double().abs(), kk.abs()).amax(-1)
            w = torch.softmax(s, -1)
            want = torch.einsum("hn,hnd->hd", w, vv)
            # 2^-23 more of each value: what reads back is rounded to fp32
            within(out[b], want, (2 * d[:, None] + 2.0 ** -13) * torch.einsum("hn,hnd->hd", w, vv.abs()) +
                   half_step(torch.bfloat16) * want.abs())
            within(lse[b], torch.logsumexp(s, -1), d + 2.0 ** -13)


# ---- refusals --------------------------------------------------------------------

def test_python_refusals():
    c = Case(lens=[40, 9], q_heads=4, k_heads=2, dim=64, page=16, held="int8", t="bf16")
    f = A.rotary_frequencies(64, device=DEV)
    pos = torch.zeros(2, dtype=torch.int64, device=DEV)
    q4 = c.q[:, None]
    args = (c.q, c.kp, c.vp, c.tables, c.l, c.ks, c.vs)

    def attention(i, x, **kw):
        a = list(args)
        a[i] = x
        return A.paged_attention(*a, **kw)

    bad = [
        (TypeError, lambda: A.rotary(c.q.int(), None, pos, f)),
        (TypeError, lambda: A.rotary(c.q, c.q.float(), pos, f)),
        (TypeError, lambda: A.rotary(c.q, None, pos.float(), f)),
        (TypeError, lambda: A.rotary(c.q, None, pos, f.float())),
        (ValueError, lambda: A.rotary(c.q[0], None, pos, f)),
        (ValueError, lambda: A.rotary(c.q, c.q[:1], pos, f)),
        (ValueError, lambda: A.rotary(c.q, None, pos[:1], f)),
        (ValueError, lambda: A.rotary(q4, None, pos, f)),
        (ValueError, lambda: A.rotary(c.q, None, pos.cpu(), f)),
        (ValueError, lambda: A.rotary(c.q, None, pos, f.cpu())),
        (ValueError, lambda: A.rotary(c.q, None, pos, f, k_out=c.q)),
        (ValueError, lambda: A.rotary(c.q, None, pos, f, q_out=c.q[:, :2])),
        (ValueError, lambda: A.rotary(c.q[..., ::2], None, pos, f[:16])),
        (ValueError, lambda: A.rotary(c.q[..., :32].contiguous(), None, pos, f)),   # rot_dim past dim
        (TypeError, lambda: attention(0, c.q.float())),
        (ValueError, lambda: attention(0, c.q[:1])),
        (ValueError, lambda: attention(0, c.q[..., :48])),
        (ValueError, lambda: attention(0, c.q[:, :3])),
        (TypeError, lambda: attention(1, c.kp.float())),
        (ValueError, lambda: attention(2, c.vp[:-1])),
        (ValueError, lambda: attention(2, c.vp.transpose(1, 2).contiguous().transpose(1, 2))),
        (ValueError, lambda: attention(3, c.tables.long())),
        (ValueError, lambda: attention(3, c.tables[:1])),
        (ValueError, lambda: attention(3, c.tables.cpu())),
        (ValueError, lambda: attention(4, c.l.long())),
        (ValueError, lambda: attention(4, c.l[:1])),
        (ValueError, lambda: attention(4, c.l.cpu())),
        (ValueError, lambda: attention(5, None)),
        (ValueError, lambda: attention(5, c.ks[..., :8])),
        (ValueError, lambda: attention(6, c.vs.double())),
        (ValueError, lambda: A.paged_attention(*args, starts=c.l.long())),
        (ValueError, lambda: A.paged_attention(*args, out=c.q.float())),
        (ValueError, lambda: A.paged_attention(*args, lse=torch.zeros(2, 3, device=DEV))),
        (ValueError, lambda: A.paged_attention(*args, workspace=torch.empty(1, dtype=torch.uint8, device=DEV))),
        (ValueError, lambda: A.paged_attention(c.q, c.kp.to(torch.float16), c.vp.to(torch.float16), c.tables, c.l)),
        (ValueError, lambda: A.paged_attention(c.q, c.kp.bfloat16(), c.vp.bfloat16(), c.tables, c.l, c.ks, c.vs)),
        (TypeError, lambda: A.cache_write(c.q.int(), c.q.int(), pos, c.kp, c.vp, c.ks, c.vs)),
        (TypeError, lambda: A.cache_write(c.q[:, :2], c.q[:, :2].float(), pos, c.kp, c.vp, c.ks, c.vs)),
        (TypeError, lambda: A.cache_write(c.q[:, :2], c.q[:, :2], pos.int(), c.kp, c.vp, c.ks, c.vs)),
        (ValueError, lambda: A.cache_write(c.q, c.q, pos, c.kp, c.vp, c.ks, c.vs)),
        (ValueError, lambda: A.cache_write(c.q[:, :2], c.q[:, :2], pos[:1], c.kp, c.vp, c.ks, c.vs)),
        (TypeError, lambda: A.cache_read(pos, c.kp, c.vp, c.ks, c.vs, dtype=torch.int8)),
        (ValueError, lambda: A.cache_read(pos, c.kp, c.vp, c.ks, c.vs, k_out=c.q)),
        (ValueError, lambda: A.cache_read(pos.cpu(), c.kp, c.vp, c.ks, c.vs)),
        (ValueError, lambda: A.cache_read(pos, c.kp, c.vp)),
    ]
    for i, (kind, call) in enumerate(bad):
        with pytest.raises(kind):
            call()
            pytest.fail(f"refusal {i} was taken")
    A.paged_attention(*args)
    torch.cuda.synchronize()
