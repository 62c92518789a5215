"""Attention over the cache in large batches whose sequences are cut over
several blocks and joined: fewer segments than blocks and more, the join's plan
worked out for itself (up to 128 sequences) and read from the main kernel's.
Bounds and the plain form in 64 bits are those of test_gpu_attention.py; the sums
over n tokens add 2 n u of sum p |v|."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from chimera_b200 import attention as A  # noqa: E402
from tests.test_gpu_attention import U, Case, within  # noqa: E402


def ragged(batch, longest, seed):
    """Lengths from nothing to the longest, which stands first, last and in places between."""
    g = torch.Generator().manual_seed(seed)
    lens = (torch.rand(batch, generator=g) ** 3 * longest).int().tolist()
    for i in {0, 31, 32, 63, 64, 95, 96, 127, 128, batch // 2, batch - 1}:
        if i < batch:
            lens[i] = longest - i
    for i in {1, 33, 65, 97, 129}:
        if i < batch - 1:
            lens[i] = 0
    return lens


@pytest.mark.parametrize("held,t,dim", [("bf16", None, 64), ("fp16", None, 128), ("int8", "bf16", 128),
                                        ("e4m3", "fp16", 64), ("bf16", None, 256)])
@pytest.mark.parametrize("k_heads", [1, 8])   # 65 to 300 segments, and 520 to 2,400
@pytest.mark.parametrize("batch", [65, 97, 128, 129, 300])
def test_joins_of_large_batches(batch, k_heads, held, t, dim):
    longest = 2500 if k_heads == 1 else 1300
    lens = ragged(batch, longest, batch)
    c = Case(lens=lens, q_heads=2 * k_heads, k_heads=k_heads, dim=dim, page=16, held=held, t=t, seed=batch, width=300)
    ws = torch.full((A.paged_attention_workspace(c.kp, c.vp, batch, 2 * k_heads, 300, c.ks, c.vs),), 0xFF,
                    dtype=torch.uint8, device="cuda")   # parts left unwritten would be NaN
    got, lse = c.run(workspace=ws)
    out, want, tol, ltol = c.expected()
    more = 2 * longest * U
    within(got, out, tol + more * c.values(c.vp, c.vs).abs().amax())
    within(lse, want, ltol + more)
    again, lagain = c.run()
    assert torch.equal(got, again) and torch.equal(lse, lagain)


@pytest.mark.parametrize("held,t", [("bf16", None), ("int8", "bf16")])
@pytest.mark.parametrize("batch", [128, 129])
def test_joins_with_starts_and_rows_that_do_not_fit(batch, held, t):
    """Windows of long sequences; a page that is not there and a length past the table mark their rows alone."""
    lens = ragged(batch, 2400, 5)
    starts = [max(0, n - 1100) if i % 3 == 0 else -4 if i % 3 == 1 else 0 for i, n in enumerate(lens)]
    c = Case(lens=lens, starts=starts, q_heads=6, k_heads=2, dim=64, page=16, held=held, t=t, width=200)
    got, lse = c.run()
    out, want, tol, ltol = c.expected()
    more = 2 * 2400 * U
    within(got, out, tol + more * c.values(c.vp, c.vs).abs().amax())
    within(lse, want, ltol + more)
    c.tables[64, 110] = c.n          # 64 is 2,336 long, its window starts at 0
    c.tables[96, 0] = -1             # 96 is 2,304 long, its window starts at 1,204: not needed
    got2, lse2 = c.run()
    rest = [i for i in range(batch) if i != 64]
    assert bool(got2[64].isnan().all() & lse2[64].isnan().all())
    assert torch.equal(got2[rest], got[rest]) and torch.equal(lse2[rest], lse[rest])
    c.l[127] = 200 * 16 + 1
    got2, lse2 = c.run()
    for i in (64, 127):
        assert bool(got2[i].isnan().all() & lse2[i].isnan().all())
    # the others are cut elsewhere now: within the bound, not bit for bit
    rest = [i for i in rest if i != 127]
    within(got2[rest], out[rest], (tol + more * c.values(c.vp, c.vs).abs().amax())[rest])
    within(lse2[rest], want[rest], (ltol + more)[rest])
