"""GPU: a row of attention_ragged depends, to the last bit, on what it may see alone: not on
finite keys and values that its mask hides, on other sequences, or on what the processor ran
before. Two ways to compute tanh (scores within the cap, and beyond it) differ by roundings, so a
choice between them that looked at hidden scores would show here."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16

SHAPES = [  # q lengths, kv lengths, heads, kv heads, d
    ([1, 1], [70, 300], 4, 1, 128),            # one token of four heads: rows 4 to 15 of the tile are nobody's
    ([1, 1, 1], [333, 5, 129], 8, 1, 64),
    ([3, 2], [200, 131], 12, 4, 64),
    ([40, 30, 9], [40, 30, 9], 6, 6, 64),      # one tile each
    ([31, 20], [131, 20], 4, 1, 128),
    ([42, 11], [42, 400], 3, 1, 128),          # groups of three: 126 rows of 128
    ([300, 200, 77], [300, 200, 177], 4, 2, 128),
    ([257, 130], [257, 1130], 3, 1, 64),
]


def inputs(shape, t, seed):
    ql, kl, H, Hk, d = shape
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    q, k, v = (torch.randn((n, h, d), generator=g, device="cuda").to(t) for n, h in
               ((sum(ql), H), (sum(kl), Hk), (sum(kl), Hk)))
    begin = lambda lens: [sum(lens[:i]) for i in range(len(lens))]  # noqa: E731
    return q, k, v, begin(ql), begin(kl)


def attend(sdb, shape, q, k, v, qb, kb, **kw):
    ql, kl = shape[:2]
    cols = [torch.tensor(c, device="cuda", dtype=torch.int32) for c in (qb, ql, kb, kl)]
    out = sdb.backend.attention_ragged(q, k, v, *cols, max(ql), max(kl), **kw)
    sdb.backend.synchronize()
    return out


def options(bias, H):
    return dict(slopes=2.0 ** (-8.0 * torch.arange(1, H + 1, device="cuda") / H)) if bias else {}


@pytest.mark.parametrize("cap", [0.0, 5.0, 50.0])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("t", [F16, BF16])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_later_keys_do_not_touch_a_row(sdb, shape, t, cap, bias):
    """Keys and values after the middle of the first sequence's queries, made forty times larger, change no row before."""
    q, k, v, qb, kb = inputs(shape, t, 1)
    (ql, kl), kw = shape[:2], options(bias, shape[2])
    a = attend(sdb, shape, q, k, v, qb, kb, causal=True, cap=cap, **kw)
    rows = ql[0] // 2  # these rows see the keys below first
    first = kb[0] + kl[0] - ql[0] + rows
    k2, v2 = k.clone(), v.clone()
    k2[first:] *= 40.0
    v2[first:] *= 40.0
    b = attend(sdb, shape, q, k2, v2, qb, kb, causal=True, cap=cap, **kw)
    assert torch.equal(a[:rows], b[:rows])
    assert not torch.equal(a[rows:], b[rows:])


@pytest.mark.parametrize("mask", ["full", "causal", "prefix"])
@pytest.mark.parametrize("cap", [0.0, 5.0, 50.0])
@pytest.mark.parametrize("t", [F16, BF16])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_other_sequences_do_not_touch_a_row(sdb, shape, t, cap, mask):
    q, k, v, qb, kb = inputs(shape, t, 2)
    ql, kl = shape[:2]
    kw = dict(cap=cap, causal=mask != "full")
    if mask == "prefix":
        kw["prefix"] = torch.tensor([n // 2 for n in kl], device="cuda", dtype=torch.int32)
    a = attend(sdb, shape, q, k, v, qb, kb, **kw)
    for s in range(len(ql)):
        rows, keys = slice(qb[s], qb[s] + ql[s]), slice(kb[s], kb[s] + kl[s])
        q2, k2, v2 = q * 40.0, k * 40.0, v * 40.0
        q2[rows], k2[keys], v2[keys] = q[rows], k[keys], v[keys]
        b = attend(sdb, shape, q2, k2, v2, qb, kb, **kw)
        assert torch.equal(a[rows], b[rows])


@pytest.mark.parametrize("cap", [5.0, 50.0])
@pytest.mark.parametrize("t", [F16, BF16])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_what_ran_before_does_not_touch_a_row(sdb, shape, t, cap):
    """Memory of the processors that holds large or small operands of an earlier call."""
    args = inputs(shape, t, 3)
    a = attend(sdb, shape, *args, causal=True, cap=cap)
    for scale in (1000.0, 1e-3):
        before = ([500] * 8, [500] * 8, shape[2], shape[3], shape[4])
        q, k, v, qb, kb = inputs(before, t, 4)
        attend(sdb, before, q * scale, k, v, qb, kb, causal=True, cap=cap)
        tokens = ([1] * 300, [200] * 300, shape[2], shape[3], shape[4])
        q, k, v, qb, kb = inputs(tokens, t, 5)
        attend(sdb, tokens, q * scale, k, v, qb, kb, causal=True, cap=cap)
        assert torch.equal(a, attend(sdb, shape, *args, causal=True, cap=cap))
