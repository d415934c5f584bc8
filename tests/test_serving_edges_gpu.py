"""GPU: calls of the operators for several requests that their documentation allows and that are easily
forgotten: nothing of one kind, orders and gaps of any kind, graphs whose lengths change between replays."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def randn(*s, t=BF16, seed=0, scale=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed + sum(s))
    return (torch.randn(s, generator=g, device="cuda") * scale).to(t)


def ints(v):
    return torch.tensor(v, device="cuda", dtype=torch.int32)


def attention(q, k, v, seqs, scale, causal=False, prefix=None, slopes=None):
    """64-bit result; rows of no sequence are 5."""
    out = torch.full(q.shape, 5.0, device="cuda", dtype=torch.float64)
    G = q.shape[1] // k.shape[1]
    for s, (q0, nq, k0, nk) in enumerate(seqs):
        if nq == 0:
            continue
        qq = q[q0:q0 + nq].double().transpose(0, 1)
        kk, vv = (x[k0:k0 + nk].double().transpose(0, 1).repeat_interleave(G, 0) for x in (k, v))
        z = qq @ kk.transpose(1, 2) * scale
        p, j = torch.arange(nq, device="cuda")[:, None] + nk - nq, torch.arange(nk, device="cuda")[None]
        if slopes is not None:
            z = z - slopes.double()[:, None, None] * (p - j).abs()
        if causal:
            hide = j > p
            if prefix is not None:
                hide = hide & (j >= prefix[s])
            z = z.masked_fill(hide, -float("inf"))
        w = torch.softmax(z, -1).nan_to_num(0.0) if nk else z
        out[q0:q0 + nq] = (w @ vv).transpose(0, 1)
    return out


def near(got, want):
    """bf16 probabilities (2^-8 of sums of values of up to 5, in the mean far less) and a bf16 result."""
    assert ((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 5 * 2.0 ** -8).all(), float((got.double() - want).abs().max())


def test_no_heads_of_one_kind(sdb):
    x, cos = randn(9, 3, 64), torch.ones(9, 64, device="cuda")
    q0, k0 = sdb.backend.qk_norm_rope(x, None, cos, cos * 0)
    none = torch.empty(9, 0, 64, device="cuda", dtype=BF16)
    q1, k1 = sdb.backend.qk_norm_rope(none, x, cos, cos * 0)
    q2, k2 = sdb.backend.qk_norm_rope(x, none, cos, cos * 0)
    sdb.backend.synchronize()
    assert k0 is None and q1.shape == (9, 0, 64) and k2.shape == (9, 0, 64)
    assert torch.equal(q0, k1) and torch.equal(q0, q2)


def test_no_rows(sdb):
    be, e = sdb.backend, torch.empty
    dev = dict(device="cuda", dtype=BF16)
    cos = torch.ones(4, 64, device="cuda")
    q, k = be.qk_norm_rope(e(0, 2, 64, **dev), e(0, 1, 64, **dev), cos, cos)
    assert q.shape == (0, 2, 64) and k.shape == (0, 1, 64)
    y = be.linear_lora(e(0, 32, **dev), randn(16, 32), randn(2, 4, 32), randn(2, 16, 4), ints([]))
    assert y.shape == (0, 16)
    y = be.linear_lora(randn(3, 32), e(0, 32, **dev), randn(2, 4, 32), e(2, 0, 4, **dev), ints([0, 1, -1]))
    assert y.shape == (3, 0)
    o = be.attention_ragged(e(0, 2, 64, **dev), randn(5, 1, 64), randn(5, 1, 64), *[ints([0])] * 4, 0, 5)
    assert o.shape == (0, 2, 64)
    o = be.attention_ragged(randn(5, 2, 64), randn(5, 1, 64), randn(5, 1, 64), *[ints([])] * 4, 5, 5)
    assert (o == 0).all()
    be.synchronize()


def test_no_keys_at_all(sdb):
    q, none = randn(5, 2, 64), torch.empty(0, 1, 64, device="cuda", dtype=BF16)
    out = torch.full_like(q, 5.0)
    sdb.backend.attention_ragged(q, none, none, ints([0, 3]), ints([2, 1]), ints([0, 0]), ints([0, 0]), 2, 0, out=out)
    sdb.backend.synchronize()
    assert (out[[0, 1, 3]] == 0).all() and (out[[2, 4]] == 5).all()


@pytest.mark.parametrize("T", [2, 40, 300, 2000])
def test_adapters_of_rank_zero(sdb, T):
    x, W, bias = randn(T, 64), randn(48, 64, scale=0.1), randn(48, t=F32)
    none = dict(device="cuda", dtype=BF16)
    rows = torch.arange(T, device="cuda", dtype=torch.int32) % 3 - 1
    y = sdb.backend.linear_lora(x, W, torch.empty(2, 0, 64, **none), torch.empty(2, 48, 0, **none), rows,
                                scale=torch.ones(2, device="cuda"), bias=bias)
    want = sdb.backend.linear_lora(x, W, torch.empty(0, 4, 64, **none), torch.empty(0, 48, 4, **none), rows, bias=bias)
    sdb.backend.synchronize()
    assert torch.equal(y, want)


@pytest.mark.parametrize("d", [64, 128, 72, 256, 33])
@pytest.mark.parametrize("ql,kl", [([3, 1, 4, 2], [30, 200, 4, 150]), ([70, 200, 1, 129], [70, 300, 140, 129])])
def test_sequences_in_any_order_with_gaps(sdb, ql, kl, d):
    order = [2, 0, 3, 1]
    qb, kb, at, bt = [0] * 4, [0] * 4, 3, 5
    for i in order:
        qb[i], kb[i], at, bt = at, bt, at + ql[i] + i, bt + kl[i] + 2 * i
    q, k, v = randn(at + 2, 4, d), randn(bt + 2, 2, d, seed=1), randn(bt + 2, 2, d, seed=2)
    out = torch.full_like(q, 5.0)
    pre = [-5, 1000000, 2, 40]
    sdb.backend.attention_ragged(q, k, v, ints(qb), ints(ql), ints(kb), ints(kl), max(ql), max(kl), causal=True, prefix=ints(pre),
                                 out=out)
    sdb.backend.synchronize()
    near(out, attention(q, k, v, list(zip(qb, ql, kb, kl)), d ** -0.5, True, pre))


@pytest.mark.parametrize("pitch", [1, 4, 8])
def test_rows_of_odd_pitches(sdb, pitch):
    """Row pitches that TMA cannot read, and one that it can."""
    H, Hk, d, n = 4, 2, 64, 150
    wide = lambda h, s: randn(n, h * d + pitch, seed=s)[:, :h * d].unflatten(1, (h, d))  # noqa: E731
    q, k, v = wide(H, 1), wide(Hk, 2), wide(Hk, 3)
    out = wide(H, 4)
    one = ints([n])
    sdb.backend.attention_ragged(q, k, v, one * 0, one, one * 0, one, n, n, causal=True, out=out)
    sdb.backend.synchronize()
    near(out, attention(q, k, v, [(0, n, 0, n)], d ** -0.5, True))


@pytest.mark.parametrize("max_q", [2, 60, 300])
def test_a_graph_whose_lengths_change(sdb, max_q):
    """Lengths, positions and adapters are read when the graph runs."""
    n, be = 6, sdb.backend
    T, Tk = n * max_q, n * 700
    q, k, v = randn(T, 4, 64), randn(Tk, 1, 64, seed=1), randn(Tk, 1, 64, seed=2)
    b, kb = ints([i * max_q for i in range(n)]), ints([i * 700 for i in range(n)])
    ql, kl = ints([1] * n), ints([1] * n)
    x, W, A, B = randn(T, 64), randn(72, 64, scale=0.1), randn(3, 8, 64, scale=0.1), randn(3, 72, 8, scale=0.3)
    rows, out = ints([0] * T), torch.empty_like(q)

    def step():
        out.fill_(5.0)
        be.attention_ragged(q, k, v, b, ql, kb, kl, max_q, 700, causal=True, out=out)
        return be.linear_lora(x, W, A, B, rows)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        y = step()
    for r in range(4):
        a = [(r * 7 + i * 5) % (max_q + 1) for i in range(n)]
        c = [max(m, (r * 131 + i * 97) % 701) for i, m in enumerate(a)]
        ql.copy_(ints(a))
        kl.copy_(ints(c))
        rows.copy_((torch.arange(T, device="cuda") * (r + 1) // 5 % 4 - 1).int())
        g.replay()
        torch.cuda.synchronize()
        near(out, attention(q, k, v, list(zip(b.tolist(), a, kb.tolist(), c)), 0.125, True))
        assert torch.equal(y, be.linear_lora(x, W, A, B, rows))
    be.synchronize()


def test_queries_before_the_first_key_with_a_distance_bias(sdb):
    q, k, v = randn(200, 2, 64), randn(30, 2, 64, seed=1), randn(30, 2, 64, seed=2)
    slopes = torch.tensor([0.05, 0.5], device="cuda")
    got = sdb.backend.attention_ragged(q, k, v, ints([0]), ints([200]), ints([0]), ints([30]), 200, 30, slopes=slopes)
    sdb.backend.synchronize()
    near(got, attention(q, k, v, [(0, 200, 0, 30)], 0.125, slopes=slopes))


def test_the_same_tensor_as_keys_and_values(sdb):
    q, k = randn(40, 4, 128), randn(90, 2, 128, seed=1)
    got = sdb.backend.attention_ragged(q, k, k, ints([0]), ints([40]), ints([0]), ints([90]), 40, 90, causal=True)
    got2 = sdb.backend.attention_ragged(k[:, :2], k, k, ints([0]), ints([90]), ints([0]), ints([90]), 90, 90)
    sdb.backend.synchronize()
    near(got, attention(q, k, k, [(0, 40, 0, 90)], 128 ** -0.5, True))
    near(got2, attention(k, k, k, [(0, 90, 0, 90)], 128 ** -0.5))
