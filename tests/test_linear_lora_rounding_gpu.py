"""GPU: how far linear_lora may be off where an adapter's term cancels the shared product, so that no
bound relative to the result holds.

Besides half a step of the output: fp32 sums on the tensor core, whose adds may drop up to 2^-23 each
(K of them for x W and for h, r per part of h for h B), and h rounded to bf16 for a bf16 output (2^-8 of
each term) or held in two parts for an fp32 output (2^-16)."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
HALF = {F32: 2.0 ** -24, BF16: 2.0 ** -8}
CASES = [  # T, N, K, r, adapters
    (1, 200, 256, 16, 3), (7, 130, 64, 4, 2), (48, 256, 512, 32, 32), (128, 200, 128, 64, 5), (300, 264, 256, 20, 40),
    (600, 256, 128, 256, 2), (1100, 300, 192, 16, 3), (1500, 512, 256, 48, 7), (4200, 2048, 128, 16, 6),
]


@pytest.mark.parametrize("to", [BF16, F32])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_an_adapter_that_cancels_the_shared_product(sdb, case, to):
    """W is minus the first adapter's product, rounded to bf16."""
    T, N, K, r, n = case
    g = torch.Generator(device="cuda")
    g.manual_seed(T + K)
    randn = lambda *s, scale=1.0: (torch.randn(s, generator=g, device="cuda") * scale).to(BF16)  # noqa: E731
    x, A, B = randn(T, K), randn(n, r, K, scale=K ** -0.5), randn(n, N, r, scale=r ** -0.5)
    scale = 0.5 + torch.rand(n, generator=g, device="cuda")
    W = (-scale[0].double() * (B[0].double() @ A[0].double())).to(BF16)
    rows = torch.randint(-1, n, (T,), generator=g, device="cuda", dtype=torch.int32)
    rows[0] = 0
    got = sdb.backend.linear_lora(x, W, A, B, rows, scale=scale, out_dtype=to)
    sdb.backend.synchronize()
    x, W, A, B = x.double(), W.double(), A.double(), B.double()
    part, parts = (2.0 ** -8, 1) if to == BF16 else (2.0 ** -16, 2)
    want = x @ W.t()
    slack = K * 2.0 ** -23 * (x.abs() @ W.abs().t())
    for a in range(n):
        t = (rows == a).nonzero().flatten()
        if t.numel():
            s = float(scale[a])
            h, ha = x[t] @ A[a].t(), x[t].abs() @ A[a].abs().t()
            want[t] += s * (h @ B[a].t())
            slack[t] += s * ((part + (parts * r + 2) * 2.0 ** -23) * (h.abs() @ B[a].abs().t())
                             + K * 2.0 ** -23 * (ha @ B[a].abs().t()))
    slack = slack + 2.0 ** -22 * want.abs()
    tol = slack * (1 + HALF[to]) + HALF[to] * want.abs()
    assert ((got.double() - want).abs() <= tol).all(), float(((got.double() - want).abs() - tol).max())


@pytest.mark.parametrize("T", [1, 100, 700, 1500])
def test_an_fp32_result_keeps_what_is_left(sdb, T):
    """h = 1 + 1.5 x 2^-9 beside a shared product of -1: an fp32 result is their difference, exactly."""
    x = torch.zeros(T, 64, device="cuda", dtype=BF16)
    x[:, 0], x[:, 1] = 1.0, 1.5 * 2.0 ** -9
    A = torch.zeros(1, 1, 64, device="cuda", dtype=BF16)
    A[0, 0, :2] = 1.0
    W = torch.zeros(96, 64, device="cuda", dtype=BF16)
    W[:, 0] = -1.0
    B = torch.ones(1, 96, 1, device="cuda", dtype=BF16)
    y = sdb.backend.linear_lora(x, W, A, B, torch.zeros(T, device="cuda", dtype=torch.int32), out_dtype=F32)
    sdb.backend.synchronize()
    assert (y == 1.5 * 2.0 ** -9).all()
