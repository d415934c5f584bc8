"""GPU: infinities in the heads of qk_norm_rope."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("d,rot", [(64, 32), (128, 64), (80, 40), (40, 20), (7, 4), (64, 0)])
@pytest.mark.parametrize("value", [float("inf"), -float("inf")])
def test_an_infinity_reaches_its_pair_only(sdb, t, inter, d, rot, value):
    """u = x / sqrt(mean(x^2)) is 0 for finite x beside an infinity and NaN for the infinity, and a
    rotation spreads that over its own pair, not over channels that are not rotated."""
    q = torch.randn(6, 2, d, device="cuda").to(t)
    hits = [(0, d - 1), (1, rot), (2, min(rot + 1, d - 1)), (3, 0), (4, max(rot - 1, 0))]
    for row, c in hits:
        q[row, 1, c] = value
    a = torch.arange(6, device="cuda", dtype=torch.float64)[:, None] * (0.3 + torch.arange(rot // 2, device="cuda"))[None]
    a = a.repeat_interleave(2, 1) if inter else torch.cat([a, a], 1)
    cos, sin = a.cos().float().contiguous(), a.sin().float().contiguous()
    got, _ = sdb.backend.qk_norm_rope(q, None, cos, sin, interleaved=inter, out_dtype=F32)
    sdb.backend.synchronize()
    want = torch.zeros(6, d, dtype=torch.bool, device="cuda")  # NaN
    for row, c in hits:
        want[row, c] = True
        if c < rot:
            want[row, c ^ 1 if inter else (c + rot // 2) % rot] = True
    assert torch.equal(got[:, 1].isnan(), want)
    assert (got[:5, 1][~want[:5]] == 0).all()
    assert got[5].isfinite().all() and got[:, 0].isfinite().all() and (got[5] != 0).any()
