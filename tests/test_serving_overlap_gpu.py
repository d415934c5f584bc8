"""GPU: attention_ragged refuses a workspace that shares bytes with its operands (its size depends on the
device), and takes out beside q, k and v in the rows of one buffer."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def call(sdb, q, k, v, out, cols, ws, need, slopes=None):
    L, d = sdb.lib(), q.shape[2]
    return L.sdb200_set_stream(torch.cuda.current_stream().cuda_stream) or L.sdb200_attention_ragged(
        q.data_ptr(), q.stride(0), k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), 1, out.data_ptr(), out.stride(0), 1,
        q.shape[0], k.shape[0], 1, *[c.data_ptr() for c in cols], 3, 400, q.shape[1], k.shape[1], d, d ** -0.5, 0.0,
        slopes.data_ptr() if slopes is not None else None, 0, None, ws, need)


def test_attention_ragged_workspace(sdb):
    H, d = 4, 64
    need = sdb.lib().sdb200_attention_ragged_workspace(1, 3, 400, H, 1, d)
    assert need > 0
    big = torch.zeros(need + (1 << 20), device="cuda", dtype=torch.uint8)  # the workspace in its middle, operands in its place
    inside = lambda shape, t, at: big[at:at + torch.Size(shape).numel() * t.itemsize].view(t).view(shape)  # noqa: E731
    ws = big[1024:].data_ptr()
    i32 = torch.int32
    base = dict(q=torch.zeros(3, H, d, device="cuda", dtype=BF16), k=torch.zeros(400, 1, d, device="cuda", dtype=BF16),
                v=torch.zeros(400, 1, d, device="cuda", dtype=BF16), out=torch.zeros(3, H, d, device="cuda", dtype=BF16),
                slopes=torch.zeros(H, device="cuda"))
    cols = [torch.tensor([x], device="cuda", dtype=i32) for x in (0, 3, 0, 400)]

    def refused(text, cols=cols, **kw):
        assert call(sdb, cols=cols, ws=ws, need=need, **{**base, **kw}) == sdb.ERR_INVALID_ARG
        assert text in sdb.lib().sdb200_last_error().decode()

    refused("out overlaps ws", out=inside((3, H, d), BF16, 1024))
    refused("ws overlaps q", q=inside((3, H, d), BF16, 512))
    refused("ws overlaps k", k=inside((400, 1, d), BF16, 4096))
    refused("ws overlaps v", v=inside((400, 1, d), BF16, 4096))
    refused("ws overlaps slopes", slopes=inside((H,), torch.float32, 1024))
    refused("ws overlaps kv_len", cols=cols[:3] + [inside((1,), i32, 1024)])
    assert call(sdb, cols=cols, ws=ws, need=need, **base) == sdb.OK
    sdb.backend.synchronize()


@pytest.mark.parametrize("n", [3, 300])
def test_attention_ragged_writes_beside_its_operands(sdb, n):
    g = torch.Generator(device="cuda")
    g.manual_seed(n)
    H, Hk, d = 4, 2, 64
    buf = torch.randn(n, (2 * H + 2 * Hk) * d, generator=g, device="cuda").to(BF16)
    part = lambda a, b: buf[:, a * d:b * d].unflatten(1, (b - a, d))  # noqa: E731
    q, k, v, out = part(0, H), part(H, H + Hk), part(H + Hk, H + 2 * Hk), part(H + 2 * Hk, 2 * H + 2 * Hk)
    keep = buf[:, :(H + 2 * Hk) * d].clone()
    one = torch.tensor([n], device="cuda", dtype=torch.int32)
    want = sdb.backend.attention_ragged(q, k, v, one * 0, one, one * 0, one, n, n, causal=True)
    sdb.backend.attention_ragged(q, k, v, one * 0, one, one * 0, one, n, n, causal=True, out=out)
    sdb.backend.synchronize()
    assert torch.equal(out, want) and torch.equal(buf[:, :(H + 2 * Hk) * d], keep)
