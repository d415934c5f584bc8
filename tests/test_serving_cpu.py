"""CPU: the operators for several requests at once (qk_norm_rope, linear_lora,
attention_ragged) refuse bad arguments on the host, before any device work, and their torch
wrappers refuse tensors that do not fit. Pointers here are made-up aligned numbers that a
refused call never reads."""
import pytest

from sdb200 import ERR_INVALID_ARG, OK, lib

P, P2 = 4096, 1 << 30  # two addresses far apart
BF16, F16, F32 = 1, 2, 0


def refused(rc, text):
    assert rc == ERR_INVALID_ARG
    assert text in lib().sdb200_last_error().decode(), lib().sdb200_last_error()


def qk(**kw):
    a = dict(T=4, q=P, ldq=256, heads=4, k=P + 512, ldk=256, kv=2, in_type=F32, d=32, rot=32, gq=None, gk=None, eps=1e-6,
             cos=P2, sin=P2, n_pos=8, pos=None, inter=0, q_out=P2, ldqo=128, k_out=2 * P2, ldko=64, out_type=F32)
    a.update(kw)
    return lib().sdb200_qk_norm_rope(*a.values())


@pytest.mark.parametrize("kw,text", [
    (dict(in_type=3), "element type"), (dict(out_type=-1), "element type"), (dict(T=-1), "bad shape"),
    (dict(heads=0, kv=0), "bad shape"), (dict(d=0, rot=0), "head width"), (dict(d=1025), "head width"),
    (dict(rot=31), "rot must"), (dict(rot=34), "rot must"), (dict(rot=-2), "rot must"),
    (dict(ldq=127), "pitch of q"), (dict(ldqo=127), "pitch of q"), (dict(ldk=63), "pitch of k"),
    (dict(q=None), "null pointer q"), (dict(q=P + 2), "misaligned pointer q"), (dict(k=None), "null pointer k"),
    (dict(cos=None), "null pointer cos"), (dict(sin=None), "null pointer sin"), (dict(n_pos=0), "n_pos"),
    (dict(pos=P + 1), "misaligned pointer pos"), (dict(gq=P + 2), "misaligned pointer gq"),
    (dict(q_out=P + 64, ldqo=256), "overlaps"), (dict(q_out=P, ldqo=128), "overlaps"),
    (dict(q_out=P, ldqo=256, out_type=BF16), "overlaps"),
    (dict(in_type=F16, out_type=BF16, q_out=P, ldqo=256), "one type"),
])
def test_qk_norm_rope_refusals(kw, text):
    refused(qk(**kw), text)


def test_empty_calls_are_no_ops():
    assert qk(T=0, q=None, k=None, q_out=None, k_out=None) == OK
    assert lora(T=0, X=None, Y=None) == OK
    assert lora(N=0, W=None, Y=None) == OK
    assert attn(n_seq=0, q_begin=None) == OK
    assert attn(Tq=0, q=None, out=None) == OK


def lora(**kw):
    a = dict(T=4, N=64, K=32, X=P, ldx=32, x_bf16=1, W=P, ldw=32, bias=None, rows=P, n=2, r=8, A=P, lda=32, B=P, ldb=8,
             scale=None, Y=P2, ldy=64, y_bf16=1, ws=None, ws_bytes=0)
    a.update(kw)
    return lib().sdb200_linear_lora(*a.values())


@pytest.mark.parametrize("kw,text", [
    (dict(T=-1), "bad shape"), (dict(K=0), "bad shape"), (dict(r=-1), "bad shape"), (dict(r=257), "rank"),
    (dict(N=1 << 31), "2^31"), (dict(ldx=31), "leading dimension"), (dict(ldw=31), "leading dimension"),
    (dict(ldy=63), "leading dimension"), (dict(X=None), "null pointer X"), (dict(x_bf16=0, X=P + 2), "misaligned pointer X"),
    (dict(W=None), "null pointer W"), (dict(bias=P + 2), "misaligned pointer bias"), (dict(rows=None), "row_adapter"),
    (dict(A=None), "null pointer A"), (dict(B=None), "null pointer B"), (dict(lda=31), "adapter leading"),
    (dict(ldb=7), "adapter leading"), (dict(scale=P + 1), "misaligned pointer scale"), (dict(Y=None), "null pointer Y"),
    (dict(Y=P2 + 2, y_bf16=0), "misaligned pointer Y"), (dict(ws_bytes=0), "workspace of"),
    (dict(ws=None, ws_bytes=1 << 40), "null pointer ws"), (dict(ws=P + 16, ws_bytes=1 << 40), "misaligned pointer ws"),
])
def test_linear_lora_refusals(kw, text):
    refused(lora(**kw), text)


@pytest.mark.parametrize("kw,text", [
    (dict(Y=P), "Y overlaps X"), (dict(Y=P + 128, X=P2 + (1 << 20), ldw=64), "Y overlaps W"),
    (dict(X=P2 + (1 << 20), W=P2 + (1 << 20), Y=P), "Y overlaps A"), (dict(T=(1 << 31) - 512), "2^31"),
    (dict(Y=P2, X=P2 + 100, ldx=64), "Y overlaps X"),
])
def test_linear_lora_refuses_shared_buffers_and_huge_ones(kw, text):
    refused(lora(**kw), text)


@pytest.mark.parametrize("kw", [dict(K=0), dict(r=300), dict(n=-1), dict(T=1 << 40), dict(N=1 << 31)])
def test_linear_lora_workspace_of_bad_shapes(kw):
    a = dict(T=4, N=64, K=32, X=P, ldx=32, x_bf16=1, W=P, ldw=32, n=2, r=8, A=P, lda=32, B=P, ldb=8)
    a.update(kw)
    assert lib().sdb200_linear_lora_workspace(*a.values()) == -1


def test_linear_lora_takes_columns_side_by_side():
    """X and Y may be columns of the same rows: only the missing workspace is refused here."""
    refused(lora(X=P2, ldx=96, Y=P2 + 64, ldy=96), "workspace of")
    refused(lora(X=P2 + 128, ldx=96, Y=P2, ldy=96), "workspace of")


def attn(**kw):
    a = dict(q=P, ldq=128, k=P, ldk=64, v=P, ldv=64, in_type=BF16, out=P2, ldo=128, out_type=BF16, Tq=4, Tkv=9, n_seq=2,
             q_begin=P, q_len=P, kv_begin=P, kv_len=P, max_q=4, max_kv=9, heads=4, kv_heads=2, d=32, scale=0.1, cap=0.0,
             slopes=None, causal=1, prefix=None, ws=None, ws_bytes=1 << 40)
    a.update(kw)
    return lib().sdb200_attention_ragged(*a.values())


@pytest.mark.parametrize("kw,text", [
    (dict(in_type=F32), "operands must"), (dict(out_type=F32), "output must"), (dict(n_seq=-1), "n_seq"),
    (dict(n_seq=65536), "n_seq"), (dict(max_q=-1), "bad shape"), (dict(Tkv=-1), "bad shape"),
    (dict(heads=3), "multiple of kv_heads"), (dict(heads=0), "multiple of kv_heads"), (dict(d=0), "head width"),
    (dict(d=257, ldq=4000, ldk=4000, ldv=4000, ldo=4000), "head width"), (dict(heads=258, kv_heads=2), "too many heads"),
    (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(cap=-1.0), "cap"), (dict(cap=float("inf")), "cap"), (dict(cap=float("nan")), "cap"),
    (dict(causal=0, prefix=P), "prefix needs"), (dict(q_begin=None), "q_begin"), (dict(kv_len=P + 2), "kv_len"),
    (dict(ldq=127), "row pitch"), (dict(ldo=127), "row pitch"), (dict(ldk=63), "row pitch"), (dict(q=None), "null pointer q"),
    (dict(k=None), "null pointer k"), (dict(v=P + 1), "misaligned pointer v"), (dict(out=None), "null pointer out"),
    (dict(out=P + 64), "out overlaps"), (dict(slopes=P + 2), "slopes"), (dict(prefix=P + 2), "prefix"),
])
def test_attention_ragged_refusals(kw, text):
    refused(attn(**kw), text)


@pytest.mark.parametrize("kw", [dict(Tq=(1 << 31) - 256), dict(Tkv=(1 << 31) - 256)])
def test_attention_ragged_refuses_huge_tensors(kw):
    refused(attn(**kw), "2^31")


def test_wrappers_refuse_host_tensors():
    import torch

    from sdb200 import backend as be

    f, b = torch.zeros(4, 2, 8), torch.zeros(4, 2, 8, dtype=torch.bfloat16)
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="current CUDA device"):
        be.qk_norm_rope(f, f, torch.zeros(4, 8), torch.zeros(4, 8))
    with pytest.raises(ValueError, match="current CUDA device"):
        be.linear_lora(b[:, 0], b[:, 0], b[:1], torch.zeros(1, 4, 2, dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int32))
    with pytest.raises(ValueError, match="current CUDA device"):
        be.attention_ragged(b, b, b, i, i, i, i, 4, 4)
    with pytest.raises(TypeError):
        be.attention_ragged(f, f, f, i, i, i, i, 4, 4)
    with pytest.raises(TypeError):
        be.qk_norm_rope(f.long(), f, torch.zeros(4, 8), torch.zeros(4, 8))
    with pytest.raises(ValueError):
        be.linear_lora(b[:, 0], b[:, 0, :4], b[:1], b[:1], i)
