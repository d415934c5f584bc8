"""GPU: small probabilities of long caches in attention_ragged."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
HALF = {BF16: 2.0 ** -8, F16: 2.0 ** -11}


@pytest.mark.parametrize("small", [18.0, 20.5, 23.5, 26.0])
@pytest.mark.parametrize("t", [F16, BF16])
@pytest.mark.parametrize("nq,H", [(1, 4), (40, 1), (200, 2)])
def test_many_small_probabilities_count(sdb, nq, H, t, small):
    """One key has nearly all the weight and a value of 0, 60000 keys have 2^-small of it and a value
    of 1: the output is what they sum up to.

    A score is small ln 2 (one product, fp32 roundings: 16 x 2^-23 of it) and exp() adds 2^-21, so a
    probability is off by e = 2^-20 + 32 x 2^-23; the tensor core reads it in the operand's type, by
    half a step, or, in fp16, by 2^-36 of the row's largest (half the least fp16 number, the largest
    probability being held as 2^11); the sum of n terms adds n 2^-23 in the worst case of one that
    loses every bit below, here 469 tiles of 128 keys: 600 x 2^-23."""
    n, d = 60000, 16
    q, k, v = (torch.zeros(m, H, d, device="cuda", dtype=t) for m in (nq, n, n))
    q[:, :, 0] = 4.0
    k[0, :, 0] = small  # exact in both types
    v[1:] = 1.0
    scale = 0.25 * 0.6931471805599453
    col = lambda x: torch.tensor([x], device="cuda", dtype=torch.int32)  # noqa: E731
    got = sdb.backend.attention_ragged(q, k, v, col(0), col(nq), col(0), col(n), nq, n, scale=scale, out_dtype=t)
    sdb.backend.synchronize()
    p = 2.0 ** -small
    want = (n - 1) * p / (1 + (n - 1) * p)
    rel = 2 * (2.0 ** -20 + 32 * 2.0 ** -23) + 600 * 2.0 ** -23 + HALF[t]
    off = want * rel + ((n - 1) * 2.0 ** -36 if t == F16 else 0.0)
    tol = off + HALF[t] * (want + off) + (2.0 ** -25 if t == F16 else 0.0)
    assert ((got.double() - want).abs() <= tol).all(), (float(got.double().min()), float(got.double().max()), want, tol)
