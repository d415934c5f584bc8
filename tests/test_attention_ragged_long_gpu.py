"""GPU: positions of attention_ragged that are no fp32 numbers."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.mark.parametrize("more", [1, 2, 131])
@pytest.mark.parametrize("nq", [1, 20, 150])
def test_distances_in_a_cache_of_more_than_2_24_keys(sdb, nq, more):
    """Scores are 0 but for the distance bias, whose slope is 1: only the last hundred keys count, each
    with e^-|p - j|. Positions beyond 2^24 are not all fp32 numbers; distances here are."""
    n, d, slope = (1 << 24) + more, 8, 1.0
    q = torch.zeros(nq, 1, d, device="cuda", dtype=BF16)
    k = torch.zeros(n, 1, d, device="cuda", dtype=BF16)
    v = torch.zeros(n, 1, d, device="cuda", dtype=BF16)
    g = torch.Generator(device="cuda")
    g.manual_seed(more)
    near = nq + 200
    v[n - near:] = torch.randn((near, 1, d), generator=g, device="cuda").to(BF16)
    col = lambda x: torch.tensor([x], device="cuda", dtype=torch.int32)  # noqa: E731
    got = sdb.backend.attention_ragged(q, k, v, col(0), col(nq), col(0), col(n), nq, n,
                                       slopes=torch.full((1,), slope, device="cuda"))
    sdb.backend.synchronize()
    p = torch.arange(nq, device="cuda")[:, None] + near - nq
    w = torch.softmax(-slope * (p - torch.arange(near, device="cuda")[None]).abs().double(), -1)
    vv = v[n - near:, 0].double()
    want = w @ vv
    # A score below 200 rounds to 200 x 2^-23, the exponential to 2^-21, a probability to bf16, the output to bf16;
    # the hidden tail of the softmax is below 2^24 e^-200.
    rel = 2 * (4 * 200 * 2.0 ** -23 + 2.0 ** -21) + 2.0 ** -8 + 500 * 2.0 ** -23
    tol = 2 * rel * (w @ vv.abs()) * (1 + 2.0 ** -8) + 2.0 ** -8 * want.abs()
    assert ((got[:, 0].double() - want).abs() <= tol).all()
