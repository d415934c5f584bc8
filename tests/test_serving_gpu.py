"""GPU: the operators for several requests at once against their formulas in 64 bits.

Tolerances, per element, from the roundings that the formulas allow (eps(t) / 2 is half a
step of type t relative to the value, 2^-25 half a step of fp16's subnormals):

  qk_norm_rope      all in fp32: a sum of d squares, a reciprocal root, four products and a
                    sum, so (d + 16) 2^-24 of |u_i| + |u_j|, and one rounding to the output
  linear_lora       fp32 sums of K (and r) products on the tensor core, whose adds may drop
                    up to 2^-23 each: K 2^-23 sum|x w| and r 2^-23 sum|h B|; h is held in
                    bf16 (bf16 output: 2^-8 relative) or in two bf16 parts (fp32 output:
                    2^-16), and carries K 2^-23 of its own sum
  attention_ragged  a score is off by e = 2^-23 (d sum|q k| scale + 8 |z| + 4 slope |p - j|)
                    (8 roundings in scaling, capping and the bias) and exp() by 2^-21, so
                    a probability by that much relative, once in the numerator and once in the
                    denominator; the tensor core reads it in the input type (eps(in) / 2); sums
                    of n terms 2^-23 n; all of it times sum_j p_j |v_j|
"""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
HALF = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}
TINY = {F32: 0.0, BF16: 0.0, F16: 2.0 ** -25}


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def randn(g, *shape, dtype=F32, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def close(got, want, slack):
    """|got - want| <= half a step of got's type at want, plus slack; both finite together."""
    g, tol = got.double(), HALF[got.dtype] * want.abs() + TINY[got.dtype] + slack * (1 + HALF[got.dtype])
    bad = ~((g - want).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float(((g - want).abs() - tol).max()):.3g}"


# ------------------------------------------------------------------------ qk_norm_rope
def tables(n_pos, rot, inter):
    a = torch.arange(n_pos, device="cuda", dtype=torch.float64)[:, None] * (
        10000.0 ** (-torch.arange(0, max(rot, 2), 2, device="cuda", dtype=torch.float64) / max(rot, 2)))[None]
    a = (a.repeat_interleave(2, 1) if inter else torch.cat([a, a], 1))[:, :rot]
    return a.cos().float().contiguous(), a.sin().float().contiguous()


def qk_want(x, gamma, cos, sin, at, inter, eps):
    """(value, |u_i| + |u_j|) in 64 bits."""
    u = x.double()
    u = u / (u.square().mean(-1, keepdim=True) + eps).sqrt()
    if gamma is not None:
        u = u * gamma.double()
    rot = cos.shape[1]
    y, mag = u.clone(), u.abs()
    if rot:
        i = torch.arange(0, rot, 2, device="cuda") if inter else torch.arange(rot // 2, device="cuda")
        j = i + (1 if inter else rot // 2)
        c, s = cos.double()[at][:, None], sin.double()[at][:, None]
        y[..., i] = u[..., i] * c[..., i] - u[..., j] * s[..., i]
        y[..., j] = u[..., j] * c[..., j] + u[..., i] * s[..., j]
        mag[..., i] = mag[..., j] = u[..., i].abs() + u[..., j].abs()
    return y, mag


QK = [  # T, heads, kv, d, rot, in, out, interleaved, fused, positions, gamma
    (1, 1, 1, 128, 128, BF16, BF16, False, False, True, True),
    (37, 32, 8, 128, 128, BF16, BF16, False, True, True, True),
    (300, 30, 30, 128, 128, F32, F16, True, False, False, True),
    (65, 4, 2, 64, 64, F16, F16, True, True, True, True),
    (33, 12, 4, 80, 40, F32, F32, False, False, True, True),
    (19, 3, 1, 40, 40, F16, BF16, False, True, True, False),
    (8, 2, 2, 96, 48, BF16, F16, True, False, True, True),
    (7, 5, 3, 256, 256, BF16, F32, False, True, False, True),
    (5, 2, 1, 6, 2, F32, F32, False, False, True, True),
    (4, 3, 2, 7, 6, F32, BF16, True, True, True, True),
    (3, 1, 1, 1, 0, F32, F32, False, False, False, True),
    (9, 2, 1, 1024, 512, F32, F16, True, False, True, True),
    (11, 4, 4, 128, 0, BF16, BF16, False, False, False, True),
    (50, 8, 0, 128, 128, F32, F32, True, False, True, True),
    (23, 6, 2, 120, 60, F16, F16, False, True, True, True),
    (1000, 7, 1, 128, 64, F32, BF16, False, True, True, False),
]


@pytest.mark.parametrize("case", QK, ids=lambda c: "-".join(str(v).replace("torch.", "") for v in c))
def test_qk_norm_rope(sdb, case):
    T, H, Hk, d, rot, ti, to, inter, fused, by_pos, gamma = case
    g = gen(T * 131 + d)
    if fused:
        y = randn(g, T, (H + 2 * Hk) * d + 3, dtype=ti, scale=2.0)
        q = y[:, : H * d].unflatten(1, (H, d))
        k = y[:, H * d: (H + Hk) * d].unflatten(1, (Hk, d))
    else:
        q, k = randn(g, T, H, d, dtype=ti), (randn(g, T, Hk, d, dtype=ti) if Hk else None)
    P = 50 if by_pos else max(1, T // 3)
    cos, sin = tables(P, rot, inter)
    pos = torch.randint(0, P, (T,), generator=g, device="cuda", dtype=torch.int32) if by_pos else None
    gq, gk = (1 + randn(g, d, scale=0.3), 1 + randn(g, d, scale=0.3)) if gamma else (None, None)
    gq0, gk0 = sdb.backend.qk_norm_rope(q, k, cos, sin, gq, gk, eps=1e-5, pos=pos, interleaved=inter, out_dtype=to)
    sdb.backend.synchronize()
    at = pos.long() if by_pos else torch.arange(T, device="cuda") % P
    for x, gam, got in ((q, gq, gq0), (k, gk, gk0)):
        if x is None:
            assert got is None
            continue
        want, mag = qk_want(x, gam, cos, sin, at, inter, 1e-5)
        assert got.dtype == to
        close(got, want, (d + 16) * 2.0 ** -24 * mag)


@pytest.mark.parametrize("ti,to", [(F32, F32), (BF16, BF16), (F16, BF16), (F32, F16)])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("d,rot", [(40, 20), (4, 4), (124, 60), (100, 0)])
def test_qk_norm_rope_of_pairs_of_channels(sdb, ti, to, inter, d, rot):
    """Heads and rotated parts that only chunks of two channels divide."""
    test_qk_norm_rope(sdb, (61, 5, 3, d, rot, ti, to, inter, False, True, True))


def test_qk_norm_rope_in_place_of_a_fused_buffer(sdb):
    g = gen(5)
    y = randn(g, 41, 10 * 128, dtype=BF16)
    q, k, v = y[:, :512].unflatten(1, (4, 128)), y[:, 512:1024].unflatten(1, (4, 128)), y[:, 1024:].clone()
    cos, sin = tables(64, 128, False)
    pos = torch.arange(41, device="cuda", dtype=torch.int32) + 20
    a, b = sdb.backend.qk_norm_rope(q.clone(), k.clone(), cos, sin, pos=pos)
    sdb.backend.qk_norm_rope(q, k, cos, sin, pos=pos, q_out=q, k_out=k)
    assert torch.equal(a, q) and torch.equal(b, k) and torch.equal(y[:, 1024:], v)


def test_qk_norm_rope_leaves_rows_of_bad_positions(sdb):
    g = gen(6)
    q = randn(g, 6, 2, 64, dtype=F16)
    cos, sin = tables(10, 64, True)
    pos = torch.tensor([0, 10, 9, -1, 2147483647, 3], device="cuda", dtype=torch.int32)
    out = torch.full_like(q, 7.0)
    sdb.backend.qk_norm_rope(q, None, cos, sin, pos=pos, interleaved=True, q_out=out)
    with pytest.raises(sdb.SdbError, match="out of range") as e:
        sdb.backend.synchronize()
    assert e.value.code == sdb.ERR_INVALID_ARG
    sdb.backend.synchronize()  # reported once
    bad = torch.tensor([1, 3, 4], device="cuda")
    assert (out[bad] == 7.0).all()
    good = torch.tensor([0, 2, 5], device="cuda")
    want, mag = qk_want(q[good], None, cos, sin, pos[good].long(), True, 1e-6)
    close(out[good], want, 80 * 2.0 ** -24 * mag)


def test_qk_norm_rope_keeps_nan_and_zero_rows_apart(sdb):
    g = gen(7)
    q = randn(g, 5, 3, 128, dtype=F32)
    q[1, 1, 5] = float("nan")
    q[2, 0] = 0.0
    cos, sin = tables(5, 128, False)
    got, _ = sdb.backend.qk_norm_rope(q, None, cos, sin)
    assert got[1, 1].isnan().all()
    assert (got[2, 0] == 0).all()
    keep = torch.ones(5, 3, dtype=torch.bool, device="cuda")
    keep[1, 1] = False
    want, mag = qk_want(q, None, cos, sin, torch.arange(5, device="cuda"), False, 1e-6)
    close(got[keep], want[keep], 144 * 2.0 ** -24 * mag[keep])


# ------------------------------------------------------------------------- linear_lora
def lora_inputs(g, T, N, K, r, n, x_type=BF16):
    return (randn(g, T, K, dtype=x_type), randn(g, N, K, dtype=BF16, scale=K ** -0.5),
            randn(g, n, r, K, dtype=BF16, scale=K ** -0.5), randn(g, n, N, r, dtype=BF16, scale=max(r, 1) ** -0.5),
            0.5 + torch.rand(n, generator=g, device="cuda"), randn(g, N))


def lora_close(got, x, W, A, B, rows, scale, bias):
    x, W, A, B = x.to(BF16).double(), W.double(), A.double(), B.double()
    K, r = W.shape[1], A.shape[1]
    want = x @ W.t()
    slack = K * 2.0 ** -23 * (x.abs() @ W.abs().t())
    if bias is not None:
        want = want + bias.double()
        slack = slack + 2.0 ** -23 * bias.abs()
    part = 2.0 ** -8 if got.dtype == BF16 else 2.0 ** -16
    for a in range(A.shape[0]):
        t = (rows == a).nonzero().flatten()
        if t.numel() and r:
            s = 1.0 if scale is None else float(scale[a])
            h, ha = x[t] @ A[a].t(), x[t].abs() @ A[a].abs().t()
            want[t] += s * (h @ B[a].t())
            slack[t] += s * ((part + (r + 2) * 2.0 ** -23) * (h.abs() @ B[a].abs().t())
                             + K * 2.0 ** -23 * (ha @ B[a].abs().t()))
    slack = slack + 2.0 ** -22 * want.abs()
    close(got, want, slack)


LORA = [  # T, N, K, r, adapters, rows: each | runs | random | one | none, in, out, scale, bias
    (1, 64, 64, 8, 1, "one", BF16, BF16, True, False),
    (1, 2560, 2560, 16, 4, "random", BF16, BF16, True, True),
    (3, 129, 72, 4, 5, "each", BF16, F32, False, True),
    (16, 256, 512, 16, 16, "each", BF16, BF16, True, False),
    (17, 300, 200, 12, 3, "random", F32, BF16, True, True),
    (48, 1000, 640, 32, 32, "each", BF16, BF16, True, False),
    (64, 512, 1024, 64, 7, "random", BF16, F32, True, True),
    (65, 260, 136, 16, 40, "random", BF16, BF16, True, False),
    (127, 128, 256, 8, 127, "each", BF16, BF16, True, True),
    (128, 256, 256, 128, 2, "runs", BF16, BF16, True, False),
    (129, 96, 64, 256, 3, "runs", BF16, F32, True, True),
    (333, 777, 331, 20, 6, "random", BF16, BF16, True, True),
    (500, 512, 512, 16, 4, "none", BF16, F32, True, True),
    (640, 768, 1000, 24, 9, "runs", F32, F32, True, False),
    (1500, 1024, 520, 48, 11, "runs", BF16, BF16, False, True),
    (2100, 640, 384, 16, 64, "random", BF16, BF16, True, False),
    (31, 40, 3, 1, 2, "random", BF16, F32, True, True),
    (200, 8, 24, 2, 3, "random", BF16, BF16, True, True),
    (257, 2048, 2048, 16, 2, "runs", BF16, BF16, True, False),
    (4300, 2056, 128, 16, 6, "runs", BF16, BF16, True, True),          # tiles of pairs of processors
    (4100, 2048, 192, 40, 5, "random", BF16, F32, True, False),
]


def lora_rows(g, kind, T, n):
    if kind == "each":
        return torch.arange(T, device="cuda", dtype=torch.int32) % n
    if kind == "none":
        return torch.full((T,), -1, device="cuda", dtype=torch.int32)
    if kind == "one":
        return torch.full((T,), n - 1, device="cuda", dtype=torch.int32)
    if kind == "runs":  # requests of unequal lengths one after another, the last without an adapter
        return (torch.arange(T, device="cuda", dtype=torch.int32) * (n + 1) // T + 1) % (n + 1) - 1
    return torch.randint(-1, n, (T,), generator=g, device="cuda", dtype=torch.int32)


@pytest.mark.parametrize("case", LORA, ids=lambda c: "-".join(str(v).replace("torch.", "") for v in c))
def test_linear_lora(sdb, case):
    T, N, K, r, n, kind, ti, to, scaled, biased = case
    g = gen(T + 7 * K)
    x, W, A, B, scale, bias = lora_inputs(g, T, N, K, r, n, ti)
    rows = lora_rows(g, kind, T, n)
    scale, bias = scale if scaled else None, bias if biased else None
    got = sdb.backend.linear_lora(x, W, A, B, rows, scale=scale, bias=bias, out_dtype=to)
    sdb.backend.synchronize()
    lora_close(got, x, W, A, B, rows, scale, bias)


@pytest.mark.parametrize("case", [
    (1025, 8, 24, 2, 3, "random", BF16, BF16, True, True),
    (1030, 96, 64, 256, 3, "runs", BF16, F32, True, True),
    (1100, 777, 331, 20, 6, "random", BF16, BF16, True, True),
    (1153, 300, 72, 33, 200, "each", BF16, F32, True, False),
    (1281, 512, 512, 16, 4, "none", BF16, F32, True, True),
    (1536, 130, 1000, 64, 1, "one", F32, BF16, False, True),
    (1023, 72, 136, 16, 300, "each", BF16, F32, True, True),           # eight blocks of 128 rows
], ids=lambda c: "-".join(str(v).replace("torch.", "") for v in c))
def test_linear_lora_of_many_rows(sdb, case):
    test_linear_lora(sdb, case)


@pytest.mark.parametrize("T", [1100, 1500])
@pytest.mark.parametrize("to", [BF16, F32])
def test_linear_lora_of_many_rows_keeps_requests_apart(sdb, T, to):
    test_linear_lora_strided_operands(sdb, T)
    test_linear_lora_keeps_requests_apart(sdb, T, 320, to)


@pytest.mark.parametrize("T", [5, 40, 200, 600])
def test_linear_lora_strided_operands(sdb, T):
    """Row pitches and bases that TMA cannot read, outputs with gaps left as they were."""
    g = gen(T)
    N, K, r, n = 200, 264, 16, 3
    x, W, A, B, scale, bias = lora_inputs(g, T, N, K, r, n)
    xs, Ws = randn(g, T, K + 5, dtype=BF16), randn(g, N, K + 3, dtype=BF16)
    As, Bs = randn(g, n, r, K + 1, dtype=BF16), randn(g, n, N, r + 3, dtype=BF16)
    xs[:, 1:K + 1], Ws[:, :K], As[:, :, :K], Bs[:, :, :r] = x, W, A, B
    rows = lora_rows(g, "random", T, n)
    out = torch.full((T, N + 7), 3.0, device="cuda", dtype=BF16)
    sdb.backend.linear_lora(xs[:, 1:K + 1], Ws[:, :K], As[:, :, :K], Bs[:, :, :r], rows, scale=scale, bias=bias,
                            out=out[:, 2:N + 2])
    sdb.backend.synchronize()
    lora_close(out[:, 2:N + 2], x, W, A, B, rows, scale, bias)
    assert (out[:, :2] == 3.0).all() and (out[:, N + 2:] == 3.0).all()


@pytest.mark.parametrize("T,N", [(4, 320), (30, 320), (130, 320), (400, 320), (4200, 2048)])
@pytest.mark.parametrize("to", [BF16, F32])
def test_linear_lora_keeps_requests_apart(sdb, T, N, to):
    """NaN and infinities of one adapter or of one row stay in the rows that use them."""
    g = gen(11 * T)
    K, r, n = 256, 16, 4
    x, W, A, B, scale, bias = lora_inputs(g, T, N, K, r, n)
    rows = torch.arange(T, device="cuda", dtype=torch.int32) % (n + 1) - 1
    clean = (rows != 1) & (rows != 2)
    clean[3] = False
    xb, Ab, Bb, sb = x.clone(), A.clone(), B.clone(), scale.clone()
    xb[3, 7] = float("inf")
    Ab[1, 3, 9] = float("nan")
    Bb[2, 100] = float("inf")
    Bb[2, 101, 5] = float("nan")
    got = sdb.backend.linear_lora(xb, W, Ab, Bb, rows, scale=sb, bias=bias, out_dtype=to)
    sdb.backend.synchronize()
    lora_close(got[clean], x[clean], W, A, B, rows[clean], scale, bias)
    assert not got[3].isfinite().any()
    assert got[(rows == 1) & (torch.arange(T, device="cuda") != 3)].isnan().all()
    assert not got[rows == 2][:, 100:102].isfinite().any()


@pytest.mark.parametrize("T", [9, 150])
def test_linear_lora_reports_bad_adapters(sdb, T):
    g = gen(3)
    x, W, A, B, scale, bias = lora_inputs(g, T, 64, 64, 8, 2)
    rows = torch.zeros(T, device="cuda", dtype=torch.int32)
    rows[4], rows[6] = 2, 2147483647
    got = sdb.backend.linear_lora(x, W, A, B, rows, scale=scale, bias=bias, out_dtype=F32)
    with pytest.raises(sdb.SdbError, match="out of range"):
        sdb.backend.synchronize()
    lora_close(got, x, W, A, B, torch.where(rows < 2, rows, -1), scale, bias)


@pytest.mark.parametrize("T", [6, 140])
def test_linear_lora_without_adapters(sdb, T):
    g = gen(4)
    x, W, A, B, _, bias = lora_inputs(g, T, 96, 80, 8, 0)
    got = sdb.backend.linear_lora(x, W, A, B, torch.full((T,), -1, device="cuda", dtype=torch.int32), bias=bias)
    lora_close(got, x, W, A, B, torch.full((T,), -1, device="cuda"), None, bias)


# -------------------------------------------------------------------- attention_ragged
def begins(lens, gap):
    out, at = [], 0
    for v in lens:
        out.append(at)
        at += v + gap
    return out, max(at, 1)


def attn_want(q, k, v, seqs, scale, causal, prefix, cap, slopes, in_type):
    """64-bit result, the slack of each element, and the rows that belong to a sequence."""
    Tq, H, d = q.shape
    G = H // k.shape[1]
    want, slack = torch.zeros(Tq, H, d, device="cuda", dtype=torch.float64), torch.zeros(Tq, H, d, device="cuda", dtype=torch.float64)
    live = torch.zeros(Tq, dtype=torch.bool, device="cuda")
    for s, (q0, nq, k0, nk) in enumerate(seqs):
        live[q0:q0 + nq] = True
        if nq == 0 or nk == 0:
            continue
        qq = q[q0:q0 + nq].double().transpose(0, 1)
        kk = k[k0:k0 + nk].double().transpose(0, 1).repeat_interleave(G, 0)
        vv = v[k0:k0 + nk].double().transpose(0, 1).repeat_interleave(G, 0)
        z = qq @ kk.transpose(1, 2) * scale
        off = d * (qq.abs() @ kk.abs().transpose(1, 2)) * scale + 8 * z.abs()
        if cap:
            z = cap * torch.tanh(z / cap)
            off = off + 8 * cap  # tanh as 1 - 2 / (1 + e^2x): roundings relative to 1, times cap
        p = torch.arange(nq, device="cuda")[:, None] + nk - nq
        j = torch.arange(nk, device="cuda")[None]
        if slopes is not None:
            z = z - slopes.double()[:, None, None] * (p - j).abs()
            off = off + 4 * slopes.double().abs()[:, None, None] * (p - j).abs()
        if causal:
            hide = j > p
            if prefix is not None:
                hide = hide & (j >= int(prefix[s]))
            z = z.masked_fill(hide, -math.inf)
        w = torch.softmax(z, -1).nan_to_num(0.0)
        want[q0:q0 + nq] = (w @ vv).transpose(0, 1)
        rel = 2 * (2.0 ** -23 * off + 2.0 ** -21) + HALF[in_type] + 2.0 ** -23 * nk
        wv = w * rel
        # the denominator's error is the probabilities' weighted mean error
        slack[q0:q0 + nq] = (wv @ vv.abs() + wv.sum(-1, keepdim=True) * (w @ vv.abs())).transpose(0, 1)
    return want, slack, live


def run_attn(sdb, q_lens, kv_lens, H, Hk, d, t, to=None, causal=False, prefix=None, cap=0.0, bias=False, gap=0, seed=1,
             spread=1.0, max_q=None, max_kv=None):
    g = gen(seed)
    qb, Tq = begins(q_lens, gap)
    kb, Tk = begins(kv_lens, gap)
    q, k, v = randn(g, Tq, H, d, dtype=t, scale=spread), randn(g, Tk, Hk, d, dtype=t), randn(g, Tk, Hk, d, dtype=t)
    seqs = list(zip(qb, q_lens, kb, kv_lens))
    if gap:  # rows of no sequence hold what must not be used
        for x, b0, lens in ((q, qb, q_lens), (k, kb, kv_lens), (v, kb, kv_lens)):
            for b, n in zip(b0, lens):
                x[b + n:b + n + gap] = float("nan")
    i32 = dict(device="cuda", dtype=torch.int32)
    slopes = 2.0 ** (-8.0 * torch.arange(1, H + 1, device="cuda") / H) if bias else None
    pre = torch.tensor(prefix, **i32) if prefix is not None else None
    out = torch.full((Tq, H, d), 5.0, device="cuda", dtype=to or t)
    sdb.backend.attention_ragged(q, k, v, torch.tensor(qb, **i32), torch.tensor(q_lens, **i32), torch.tensor(kb, **i32),
                                 torch.tensor(kv_lens, **i32), max_q or max(q_lens), max_kv or max(kv_lens), causal=causal,
                                 prefix=pre, cap=cap, slopes=slopes, out=out)
    sdb.backend.synchronize()
    want, slack, live = attn_want(q, k, v, seqs, d ** -0.5, causal, prefix, cap, slopes, t)
    close(out[live], want[live], slack[live])
    assert (out[~live] == 5.0).all()
    return out


ATTN = [  # q lengths, kv lengths, heads, kv heads, d, type, options
    ([1], [1], 1, 1, 64, F16, {}),
    ([1, 1, 1], [129, 64, 3000], 8, 2, 128, BF16, dict(causal=True)),
    ([1] * 16, [1 + 173 * i for i in range(16)], 32, 8, 128, BF16, dict(causal=True, bias=True)),
    ([1, 1], [40000, 17], 4, 4, 64, F16, dict(causal=True)),
    ([4, 2, 1, 3], [700, 2, 256, 130], 12, 4, 128, F16, dict(causal=True, cap=20.0)),
    ([77, 5, 31, 64, 1], [77, 5, 31, 64, 1], 12, 12, 64, F16, dict(causal=True)),
    ([127, 128, 129, 255, 256, 257], [127, 128, 129, 255, 256, 257], 2, 2, 128, F16, dict(causal=True)),
    ([127, 128, 129, 255, 256, 257], [127, 128, 129, 255, 256, 257], 4, 1, 128, BF16, {}),
    ([600, 33], [600, 33], 8, 2, 128, BF16, dict(causal=True, prefix=[100, 33])),
    ([600, 33], [700, 533], 8, 2, 64, BF16, dict(causal=True, prefix=[0, 533], cap=30.0)),
    ([513, 1024], [513, 1024], 4, 4, 128, BF16, dict(cap=50.0)),
    ([513, 300], [1025, 300], 6, 2, 128, F16, dict(causal=True, bias=True)),
    ([300, 40], [300, 40], 6, 6, 64, BF16, dict(bias=True)),
    ([400, 90], [400, 190], 5, 1, 80, F16, dict(causal=True, bias=True, cap=10.0)),
    ([130, 60], [130, 60], 8, 8, 40, F16, dict(causal=True)),
    ([150], [150], 14, 2, 96, BF16, dict(causal=True)),
    ([50, 20], [80, 20], 3, 3, 256, BF16, dict(causal=True, cap=20.0, bias=True)),
    ([20, 9], [30, 9], 6, 2, 33, F16, dict(causal=True, prefix=[25, 9])),
    ([1, 1], [5000, 31], 16, 1, 64, F16, dict(bias=True, cap=15.0)),
    ([2000], [2000], 2, 2, 128, F16, dict(causal=True)),
    ([1500, 700], [1500, 700], 3, 3, 64, F16, {}),
    ([10, 3], [4, 1], 4, 2, 64, F16, dict(causal=True)),                # queries before the first key see none
    ([300, 5], [200, 0], 4, 4, 128, BF16, dict(causal=True)),
    ([0, 7, 0], [5, 0, 0], 2, 1, 128, F16, {}),
    ([300, 5], [200, 3], 4, 4, 128, BF16, dict(causal=True, prefix=[40, 1])),
    ([40] * 40, [40] * 40, 4, 4, 64, BF16, dict(causal=True)),
    ([128, 64], [128, 64], 128, 1, 64, F16, dict(causal=True)),
    ([3, 200], [3, 200], 21, 3, 128, F16, dict(causal=True)),           # groups of 7 heads
]


@pytest.mark.parametrize("case", ATTN, ids=lambda c: "-".join(str(v).replace("torch.", "").replace(" ", "")[:40] for v in c))
@pytest.mark.parametrize("gap", [0, 3])
def test_attention_ragged(sdb, case, gap):
    ql, kl, H, Hk, d, t, opt = case
    run_attn(sdb, ql, kl, H, Hk, d, t, gap=gap, seed=sum(ql) + d, **opt)


@pytest.mark.parametrize("t,to", [(F16, BF16), (BF16, F16)])
@pytest.mark.parametrize("lens", [([1, 1], [300, 5]), ([290, 40], [290, 40])])
def test_attention_ragged_output_type(sdb, t, to, lens):
    run_attn(sdb, *lens, 4, 2, 128, t, to=to, causal=True)


@pytest.mark.parametrize("lens", [([1, 1, 2], [900, 64, 130]), ([260, 40], [260, 140])])
def test_attention_ragged_peaked_scores(sdb, lens):
    """Scores in the hundreds: one key takes the whole row, and the running maximum moves."""
    run_attn(sdb, *lens, 4, 2, 128, F16, causal=True, spread=100.0)
    run_attn(sdb, *lens, 4, 2, 64, BF16, causal=True, spread=60.0, cap=40.0)


@pytest.mark.parametrize("lens", [[300, 40, 129, 1], [260, 257, 3], [1, 130, 77]])
@pytest.mark.parametrize("H,Hk,d", [(4, 1, 128), (6, 6, 64)])
def test_attention_ragged_of_a_padded_batch(sdb, lens, H, Hk, d):
    """[N, S] rows with lengths of their own: the padding is not read and not written."""
    g = gen(sum(lens))
    N, S = len(lens), max(lens)
    q, k, v = (randn(g, N * S, h, d, dtype=BF16) for h in (H, Hk, Hk))
    for i, n in enumerate(lens):
        for x in (q, k, v):
            x[i * S + n:(i + 1) * S] = float("nan")
    b = torch.arange(N, device="cuda", dtype=torch.int32) * S
    n = torch.tensor(lens, device="cuda", dtype=torch.int32)
    out = torch.full_like(q, 5.0)
    sdb.backend.attention_ragged(q, k, v, b, n, b, n, S, S, causal=True, out=out)
    sdb.backend.synchronize()
    want, slack, live = attn_want(q, k, v, [(i * S, m, i * S, m) for i, m in enumerate(lens)], d ** -0.5, True, None, 0.0,
                                  None, BF16)
    close(out[live], want[live], slack[live])
    assert (out[~live] == 5.0).all()


@pytest.mark.parametrize("n", [700, 1030])
def test_attention_ragged_of_many_sequences(sdb, n):
    """More sequences than one step list holds, some of several tiles, some of none."""
    g = gen(n)
    ql = [(i * 7) % 5 + (200 if i % 300 == 3 else 0) for i in range(n)]
    kl = [q + (i * 13) % 140 for i, q in enumerate(ql)]
    run_attn(sdb, ql, kl, 4, 2, 64, F16, causal=True, seed=n)
    run_attn(sdb, [1] * n, [1 + (i * 31) % 300 for i in range(n)], 4, 1, 128, BF16, causal=True, seed=n)


def test_attention_ragged_loose_maxima(sdb):
    run_attn(sdb, [5, 60], [90, 60], 4, 2, 128, F16, causal=True, max_q=4000, max_kv=100000)
    run_attn(sdb, [1, 1], [90, 600], 4, 2, 128, BF16, causal=True, max_q=1, max_kv=1 << 40)


@pytest.mark.parametrize("max_q,max_kv", [(50, 700), (4000, 700), (1 << 40, 1 << 40), (50, 1 << 40)])
def test_attention_ragged_c_call_with_loose_maxima(sdb, max_q, max_kv):
    """The workspace that the C function names is enough for the same maxima, however loose."""
    g, d = gen(17), 64
    q, k, v = randn(g, 50, 2, d, dtype=F16), randn(g, 700, 1, d, dtype=F16), randn(g, 700, 1, d, dtype=F16)
    out = torch.empty_like(q)
    cols = [torch.tensor([x], device="cuda", dtype=torch.int32) for x in (0, 50, 0, 700)]
    L = sdb.lib()
    need = L.sdb200_attention_ragged_workspace(1, max_q, max_kv, 2, 1, d)
    assert need >= 0
    ws = torch.empty(max(need, 256), device="cuda", dtype=torch.uint8)
    torch.cuda.synchronize()
    rc = L.sdb200_set_stream(torch.cuda.current_stream().cuda_stream) or L.sdb200_attention_ragged(
        q.data_ptr(), 2 * d, k.data_ptr(), d, v.data_ptr(), d, 2, out.data_ptr(), 2 * d, 2, 50, 700, 1,
        *[c.data_ptr() for c in cols], max_q, max_kv, 2, 1, d, d ** -0.5, 0.0, None, 0, None, ws.data_ptr(), need)
    assert rc == 0
    sdb.backend.synchronize()
    want, slack, _ = attn_want(q, k, v, [(0, 50, 0, 700)], d ** -0.5, False, None, 0.0, None, F16)
    close(out, want, slack)


def test_attention_ragged_strided_rows_and_shared_keys(sdb):
    """q, k, v as views of one fused projection; two sequences that read the same keys."""
    g = gen(9)
    H, Hk, d, T = 8, 2, 128, 500
    y = randn(g, T, (H + 2 * Hk) * d, dtype=BF16)
    q = y[:, :H * d].unflatten(1, (H, d))
    k = y[:, H * d:(H + Hk) * d].unflatten(1, (Hk, d))
    v = y[:, (H + Hk) * d:].unflatten(1, (Hk, d))
    seqs = [(0, 200, 0, 300), (200, 150, 0, 300), (350, 150, 300, 200)]
    cols = [torch.tensor(c, device="cuda", dtype=torch.int32) for c in zip(*seqs)]
    big = torch.full((T, H, 2 * d), 2.0, device="cuda", dtype=BF16).view(T, 2 * H * d)
    out = big[:, 8:8 + H * d].unflatten(1, (H, d))
    sdb.backend.attention_ragged(q, k, v, *cols, 200, 300, causal=True, out=out)
    want, slack, _ = attn_want(q, k, v, seqs, d ** -0.5, True, None, 0.0, None, BF16)
    close(out, want, slack)
    assert (big[:, :8] == 2.0).all() and (big[:, 8 + H * d:] == 2.0).all()


@pytest.mark.parametrize("lens", [([1, 1], [200, 300]), ([300, 60], [300, 160])])
def test_attention_ragged_masked_values_do_not_count(sdb, lens):
    """NaN and infinities in keys and values reach only the rows that may see them."""
    (ql, kl), g = lens, gen(12)
    H, Hk, d = 4, 2, 128
    qb, Tq = begins(ql, 0)
    kb, Tk = begins(kl, 0)
    q, k, v = randn(g, Tq, H, d, dtype=BF16), randn(g, Tk, Hk, d, dtype=BF16), randn(g, Tk, Hk, d, dtype=BF16)
    seqs = list(zip(qb, ql, kb, kl))
    vb, kk = v.clone(), k.clone()
    hit = kb[1] + kl[1] - 20
    vb[hit, 0, 3], vb[hit, 1, 7], kk[hit, 1, 5] = float("nan"), float("inf"), float("nan")
    cols = [torch.tensor(c, device="cuda", dtype=torch.int32) for c in zip(*seqs)]
    got = sdb.backend.attention_ragged(q, kk, vb, *cols, max(ql), max(kl), causal=True)
    want, slack, _ = attn_want(q, k, v, seqs, d ** -0.5, True, None, 0.0, None, BF16)
    pos = torch.cat([torch.arange(n, device="cuda") + m - n for n, m in zip(ql, kl)])
    second = torch.arange(Tq, device="cuda") >= qb[1]
    sees = second & (pos >= kl[1] - 20)
    close(got[~sees], want[~sees], slack[~sees])
    assert got[sees][:, :2, 3].isnan().all()                    # heads of key head 0: only that channel
    assert got[sees][:, :2, :3].isfinite().all() and got[sees][:, :2, 4:].isfinite().all()
    assert got[sees][:, 2:].isnan().all()                       # a NaN key spoils the rows that score it
    keep = torch.ones(d, dtype=torch.bool, device="cuda")
    keep[3] = False
    close(got[:, :2][:, :, keep], want[:, :2][:, :, keep], slack[:, :2][:, :, keep])


LONG = [  # sequences of several tiles of queries and many of keys
    ([700, 1, 300], [1500, 1, 900], 6, 2, 64, F16, dict(causal=True)),
    ([1030], [1030], 2, 1, 128, BF16, {}),
    ([130, 900], [2600, 900], 3, 3, 128, F16, dict(causal=True, prefix=[2000, 5], cap=30.0, bias=True)),
    ([257, 0, 40, 600], [640, 5, 2000, 0], 4, 4, 40, BF16, {}),
    ([300], [5000], 16, 2, 80, BF16, dict(bias=True)),
    ([50] * 20 + [1200], [50] * 20 + [1333], 8, 8, 64, F16, dict(causal=True, cap=20.0)),
    ([900], [700], 4, 1, 128, F16, dict(causal=True)),
    ([400], [513], 64, 1, 8, BF16, {}),
]


@pytest.mark.parametrize("gap", [0, 7])
@pytest.mark.parametrize("case", LONG, ids=lambda c: f"{len(c[0])}x{max(c[0])}-{c[2]}-{c[3]}-{c[4]}")
def test_attention_ragged_of_long_sequences(sdb, case, gap):
    test_attention_ragged(sdb, case, gap)


def test_attention_ragged_of_long_sequences_isolates_and_reports(sdb):
    test_attention_ragged_masked_values_do_not_count(sdb, ([900, 700], [900, 1800]))
    test_attention_ragged_skips_bad_sequences(sdb, ([900, 60, 700], [900, 160, 1300]))


@pytest.mark.parametrize("n", [300, 700])
def test_attention_ragged_reports_shared_query_rows(sdb, n):
    """Eight sequences of the same query rows: more tiles than rows of their own could make."""
    g = gen(n)
    q, k, v = (randn(g, n, 1, 64, dtype=F16) for _ in range(3))
    cols = [torch.full((8,), x, device="cuda", dtype=torch.int32) for x in (0, n, 0, n)]
    sdb.backend.attention_ragged(q, k, v, *cols, n, n)
    with pytest.raises(sdb.SdbError, match="out of range"):
        sdb.backend.synchronize()


@pytest.mark.parametrize("lens", [([1, 1, 1], [200, 300, 9]), ([300, 60, 9], [300, 160, 9])])
def test_attention_ragged_skips_bad_sequences(sdb, lens):
    ql, kl = lens
    g = gen(13)
    Tq, Tk = sum(ql), sum(kl)
    q, k, v = randn(g, Tq, 4, 128, dtype=F16), randn(g, Tk, 2, 128, dtype=F16), randn(g, Tk, 2, 128, dtype=F16)
    seqs = list(zip(begins(ql, 0)[0], ql, begins(kl, 0)[0], kl))
    for column, value in ((0, Tq), (0, -1), (1, -5), (1, Tq + 1), (2, Tk), (2, -7), (3, Tk + 1), (3, -1)):
        broken = [list(s) for s in seqs]
        broken[1][column] = value
        cols = [torch.tensor(c, device="cuda", dtype=torch.int32) for c in zip(*broken)]
        out = torch.full_like(q, 5.0)
        sdb.backend.attention_ragged(q, k, v, *cols, max(ql), max(kl), causal=True, out=out)
        with pytest.raises(sdb.SdbError, match="out of range"):
            sdb.backend.synchronize()
        want, slack, live = attn_want(q, k, v, [seqs[0], seqs[2]], 128 ** -0.5, True, None, 0.0, None, F16)
        close(out[live], want[live], slack[live])
        assert (out[~live] == 5.0).all()


def test_attention_ragged_equals_attention_on_one_length(sdb):
    """The same tokens through attention() (fp32 operands) of the framework."""
    g = gen(14)
    N, S, H, Hk, d = 2, 300, 8, 2, 128
    q, k, v = (randn(g, N * S, h, d, dtype=F16) for h in (H, Hk, Hk))
    b = torch.arange(N, device="cuda", dtype=torch.int32) * S
    n = torch.full((N,), S, device="cuda", dtype=torch.int32)
    got = sdb.backend.attention_ragged(q, k, v, b, n, b, n, S, S, causal=True)
    ref = sdb.backend.attention(q.float().view(N, S, -1), k.float().view(N, S, -1), v.float().view(N, S, -1), H, True, Hk)
    want, slack, _ = attn_want(q, k, v, [(0, S, 0, S), (S, S, S, S)], d ** -0.5, True, None, 0.0, None, F16)
    close(got, want, slack)
    # both within their own roundings of the exact value: fp16 probabilities in each
    assert ((got.double() - ref.double().view(N * S, H, d)).abs() <= 2 * slack + 2.0 ** -11 * want.abs() + 2.0 ** -25).all()


# ------------------------------------------------------------------------------ together
def layer(sdb, x, W, A, B, rows, scale, gq, gk, cos, sin, pos, cols, ql, kl, W2, A2, B2):
    """Projection with adapters, norms and rotation, attention, output projection with adapters."""
    be = sdb.backend
    H, Hk, d = 8, 2, 128
    y = be.linear_lora(x, W, A, B, rows, scale=scale, out_dtype=BF16)
    q, k, v = (y[:, a * d:b * d].unflatten(1, (b - a, d)) for a, b in ((0, H), (H, H + Hk), (H + Hk, H + 2 * Hk)))
    be.qk_norm_rope(q, k, cos, sin, gq, gk, pos=pos, q_out=q, k_out=k)
    o = be.attention_ragged(q, k, v, *cols, ql, kl, causal=True)
    return be.linear_lora(o.view(-1, H * d), W2, A2, B2, rows, scale=scale, out_dtype=BF16)


def layer_inputs(lens, seed):
    g = gen(seed)
    T, D = sum(lens), 1024
    W, A, B = randn(g, 12 * 128, D, dtype=BF16, scale=D ** -0.5), randn(g, 3, 16, D, dtype=BF16, scale=D ** -0.5), randn(
        g, 3, 12 * 128, 16, dtype=BF16, scale=0.1)
    W2, A2, B2 = randn(g, D, 1024, dtype=BF16, scale=2.0 ** -5), randn(g, 3, 16, 1024, dtype=BF16, scale=2.0 ** -5), randn(
        g, 3, D, 16, dtype=BF16, scale=0.1)
    b = torch.tensor(begins(lens, 0)[0], device="cuda", dtype=torch.int32)
    n = torch.tensor(lens, device="cuda", dtype=torch.int32)
    rows = torch.cat([torch.full((m,), i % 4 - 1, device="cuda", dtype=torch.int32) for i, m in enumerate(lens)])
    pos = torch.cat([torch.arange(m, device="cuda", dtype=torch.int32) for m in lens])
    cos, sin = tables(max(lens), 128, False)
    gq, gk = 1 + randn(g, 128, scale=0.2), 1 + randn(g, 128, scale=0.2)
    return dict(x=randn(g, T, D, dtype=BF16), W=W, A=A, B=B, rows=rows, scale=0.5 + torch.rand(3, generator=g, device="cuda"),
                gq=gq, gk=gk, cos=cos, sin=sin, pos=pos, cols=(b, n, b, n), ql=max(lens), kl=max(lens), W2=W2, A2=A2, B2=B2)


def layer_want(s):
    f = torch.float64
    onehot = (s["rows"][:, None] == torch.arange(3, device="cuda")).to(f) * s["scale"].to(f)

    def proj(x, W, A, B):
        h = torch.einsum("tk,ark->tar", x, A.to(f)) * onehot[..., None]
        return x @ W.to(f).t() + torch.einsum("tar,anr->tn", h, B.to(f))

    y = proj(s["x"].to(f), s["W"], s["A"], s["B"])
    q, k, v = (y[:, a * 128:b * 128].unflatten(1, (b - a, 128)) for a, b in ((0, 8), (8, 10), (10, 12)))
    q = qk_want(q, s["gq"], s["cos"], s["sin"], s["pos"].long(), False, 1e-6)[0]
    k = qk_want(k, s["gk"], s["cos"], s["sin"], s["pos"].long(), False, 1e-6)[0]
    seqs = list(zip(*(c.tolist() for c in s["cols"])))
    o = attn_want(q, k, v, seqs, 128 ** -0.5, True, None, 0.0, None, BF16)[0]
    return proj(o.reshape(-1, 1024), s["W2"], s["A2"], s["B2"])


@pytest.mark.parametrize("lens", [[1, 1, 1, 1, 1], [200, 3, 77, 129], [1, 700, 30, 2, 512, 9]])
def test_a_layer_of_the_three(sdb, lens):
    s = layer_inputs(lens, sum(lens))
    got, want = layer(sdb, **s), layer_want(s)
    sdb.backend.synchronize()
    # Five tensors are rounded to bf16 on the way (y, q and k, probabilities, o, result), each by at
    # most 2^-8 relative; a score q.k of normed heads (|q||k| / sqrt(d) <= about 12) moves by
    # 2 x 2^-8 x 12 / sqrt(128) in the mean square sense, so the whole is within 8 x 2^-8 of the norm.
    assert float((got.double() - want).norm() / want.norm()) <= 8 * 2.0 ** -8


def test_the_three_on_their_own_stream_and_in_graphs(sdb):
    """A captured layer replays on new inputs, beside another captured layer of other sizes and beside eager calls."""
    one, two = layer_inputs([200, 3, 77, 129], 1), layer_inputs([1, 1, 900, 1], 2)
    eager = [layer(sdb, **one).clone(), layer(sdb, **two).clone()]
    stream = torch.cuda.Stream()
    graphs, outs = [], []
    for s in (one, two):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            layer(sdb, **s)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            outs.append(layer(sdb, **s))
        graphs.append(g)
    for _ in range(3):
        for g in graphs:
            g.replay()
        layer(sdb, **two)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], eager[0]) and torch.equal(outs[1], eager[1])
    x2 = layer_inputs([200, 3, 77, 129], 77)["x"]
    one["x"].copy_(x2)
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], layer(sdb, **one))
    sdb.backend.synchronize()


@pytest.mark.parametrize("to", [BF16, F32])
@pytest.mark.parametrize("T,n,r", [(9000, 64, 128), (20000, 40, 256), (3000, 200, 20)])
def test_linear_lora_of_many_adapters_and_rows(sdb, T, n, r, to):
    """H of all rows at once would pass its share of the workspace, so that blocks of rows go one after another."""
    test_linear_lora(sdb, (T, 40, 64, r, n, "random", BF16, to, True, True))


def test_linear_lora_on_two_streams_at_once(sdb):
    """Calls whose processors wait for one another's h, on streams of different priorities."""
    g = gen(23)
    calls, streams = [], [torch.cuda.Stream(), torch.cuda.Stream(priority=-1)]
    for T, N, K, r, n in ((3000, 2048, 512, 32, 5), (5000, 1024, 640, 16, 3)):
        x, W, A, B, scale, bias = lora_inputs(g, T, N, K, r, n)
        calls.append((x, W, A, B, lora_rows(g, "runs", T, n), scale, bias))
    want = [sdb.backend.linear_lora(*c) for c in calls]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(sdb.backend.linear_lora(*calls[i]))
    torch.cuda.synchronize()
    sdb.backend.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])


@pytest.mark.parametrize("T", [7, 300, 1100])
def test_linear_lora_beside_its_input(sdb, T):
    """x and out are columns of one buffer."""
    g = gen(T)
    x, W, A, B, scale, bias = lora_inputs(g, T, 128, 64, 16, 3)
    rows = lora_rows(g, "random", T, 3)
    buf = torch.cat([x, torch.zeros(T, 128, device="cuda", dtype=BF16)], 1)
    sdb.backend.linear_lora(buf[:, :64], W, A, B, rows, scale=scale, bias=bias, out=buf[:, 64:])
    sdb.backend.synchronize()
    assert torch.equal(buf[:, :64], x)
    lora_close(buf[:, 64:], x, W, A, B, rows, scale, bias)


def test_wrappers_name_what_does_not_fit(sdb):
    be, g = sdb.backend, gen(31)
    q, cos = randn(g, 4, 2, 8, dtype=BF16), randn(g, 4, 8)
    pos = torch.zeros(4, device="cuda", dtype=torch.int32)

    def refused(text, kind, f, *a, **kw):
        with pytest.raises(kind, match=text):
            f(*a, **kw)

    for kw, text, kind in (
            (dict(cos=cos.half()), "cos must be", TypeError), (dict(sin=cos[:3]), "sin must be", ValueError),
            (dict(cos=cos.cpu()), "cos is on", ValueError), (dict(gq=cos[0, :7]), "gq must be", ValueError),
            (dict(pos=pos.long()), "pos must be", TypeError), (dict(pos=pos[:3]), "pos must be", ValueError),
            (dict(k=q.float()), "k must be", TypeError), (dict(k=q[:3]), "k must be", ValueError),
            (dict(q=q[..., ::2]), "heads of q must be dense", ValueError), (dict(out_dtype=torch.int8), "output type", TypeError),
            (dict(q_out=q.float()[:, :1].to(BF16)), "shape of q", ValueError), (dict(q_out=q.cpu()), "q_out is on", ValueError),
            (dict(cos=cos[:, :7].contiguous(), sin=cos[:, :7].contiguous()), "rot must be even", sdb.SdbError),
            (dict(eps="x"), "not of its kind", TypeError)):
        a = dict(q=q, k=q, cos=cos, sin=cos)
        a.update(kw)
        if "q" in kw:
            a.update(k=None, cos=cos[:, :4].contiguous(), sin=cos[:, :4].contiguous())
        refused(text, kind, be.qk_norm_rope, **a)
    x, W, A, B = randn(g, 4, 16, dtype=BF16), randn(g, 8, 16, dtype=BF16), randn(g, 2, 4, 16, dtype=BF16), randn(g, 2, 8, 4, dtype=BF16)
    for kw, text, kind in (
            (dict(W=W.float()), "W must be", TypeError), (dict(W=W[:, :15]), "shapes", ValueError),
            (dict(rows=pos[:2]), "rows must be", ValueError), (dict(rows=pos.cpu()), "rows is on", ValueError),
            (dict(bias=cos[0, :7]), "bias must be", ValueError), (dict(scale=cos[0]), "scale must be", ValueError),
            (dict(out_dtype=F16), "output type", TypeError), (dict(out=cos[:, :7]), "out must be", ValueError),
            (dict(x=randn(g, 16, 4, dtype=BF16).t()), "rows of x must be dense", ValueError),
            (dict(A=randn(g, 4, 2, 16, dtype=BF16).transpose(0, 1)), "adapters of A", ValueError)):
        a = dict(x=x, W=W, A=A, B=B, rows=pos)
        a.update(kw)
        refused(text, kind, be.linear_lora, **a)
    one = torch.ones(1, device="cuda", dtype=torch.int32)
    for kw, text, kind in (
            (dict(k=q.half()), "k must be", TypeError), (dict(v=q[:, :1]), "shapes", ValueError),
            (dict(q_len=one.long()), "q_len must be", TypeError), (dict(kv_len=pos), "kv_len must be", ValueError),
            (dict(prefix=one), "prefix needs", sdb.SdbError), (dict(slopes=cos[0]), "slopes must be", ValueError),
            (dict(out=q[:3]), "shape of q", ValueError), (dict(out_dtype=F32), "output type", TypeError),
            (dict(out=q), "out overlaps", sdb.SdbError), (dict(max_q=-1), "bad shape", sdb.SdbError),
            (dict(scale=0.0), "scale must be", sdb.SdbError)):
        a = dict(q=q, k=q, v=q, q_begin=one * 0, q_len=one * 4, kv_begin=one * 0, kv_len=one * 4, max_q=4, max_kv=4)
        a.update(kw)
        refused(text, kind, be.attention_ragged, **a)
    sdb.backend.synchronize()


def test_calls_of_two_threads_go_to_their_own_streams(sdb):
    """A thread's call runs on its current stream, also while another thread calls."""
    import threading

    inputs = [layer_inputs([200, 3, 77], 11), layer_inputs([1, 1, 400], 12)]
    want = [layer(sdb, **s).clone() for s in inputs]
    torch.cuda.synchronize()
    got, wrong = [[], []], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(30):
                    got[i].append(layer(sdb, **inputs[i]))
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001 - shown below
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong
    sdb.backend.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])


def test_the_three_repeat_exactly(sdb):
    s = layer_inputs([333, 1, 64], 5)
    a = layer(sdb, **s)
    for _ in range(3):
        assert torch.equal(a, layer(sdb, **s))
