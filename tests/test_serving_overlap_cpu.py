"""CPU: outputs of the operators for several requests that share bytes with anything a call reads, or
with its workspace, are refused; columns of one buffer side by side are not. Pointers are made-up
aligned numbers that a refused call never reads."""
import pytest

from sdb200 import ERR_INVALID_ARG, lib

MB = 1 << 20
BF16, F32 = 1, 0


def refused(rc, text):
    assert rc == ERR_INVALID_ARG
    assert text in lib().sdb200_last_error().decode(), lib().sdb200_last_error()


def qk(**kw):  # rows of 4 heads of q and 4 of k, 32 channels, fp32
    a = dict(T=4, q=MB, ldq=128, heads=4, k=2 * MB, ldk=128, kv=4, in_type=F32, d=32, rot=32, gq=3 * MB, gk=4 * MB, eps=1e-6,
             cos=5 * MB, sin=6 * MB, n_pos=8, pos=7 * MB, inter=0, q_out=8 * MB, ldqo=128, k_out=9 * MB, ldko=128, out_type=F32)
    a.update(kw)
    return lib().sdb200_qk_norm_rope(*a.values())


@pytest.mark.parametrize("kw,text", [
    (dict(q_out=2 * MB), "q_out overlaps k"), (dict(q_out=2 * MB + 512), "q_out overlaps k"),
    (dict(k_out=MB), "k_out overlaps q"), (dict(k_out=MB + 1536), "k_out overlaps q"),
    (dict(k_out=8 * MB), "k_out overlaps q_out"), (dict(q_out=MB, k_out=MB), "k_out overlaps q"),
    (dict(q_out=2 * MB, k_out=MB), "overlaps"),
    (dict(q=MB, ldq=256, k=MB + 512, ldk=256, q_out=MB, ldqo=256, k_out=MB + 256, ldko=256), "k_out overlaps"),
    (dict(q_out=5 * MB), "q_out overlaps cos"), (dict(k_out=6 * MB + 512), "k_out overlaps sin"),
    (dict(q_out=3 * MB), "q_out overlaps gq"), (dict(q_out=4 * MB + 64), "q_out overlaps gk"), (dict(k_out=7 * MB), "k_out overlaps pos"),
])
def test_qk_norm_rope(kw, text):
    refused(qk(**kw), text)


def test_qk_norm_rope_side_by_side():
    """q and k written in place of a fused buffer, and into other columns of it: all that is refused here is
    an array that overlaps on purpose, which is looked at last."""
    fused = dict(ldq=512, k=MB + 512, ldk=512, ldqo=512, ldko=512)
    refused(qk(q_out=MB, k_out=MB + 512, pos=MB, **fused), "q_out overlaps pos")
    refused(qk(q_out=MB + 1024, k_out=MB + 1536, pos=MB + 1024, **fused), "q_out overlaps pos")


def lora(**kw):
    a = dict(T=4, N=64, K=32, X=MB, ldx=32, x_bf16=1, W=2 * MB, ldw=32, bias=3 * MB, rows=4 * MB, n=2, r=8, A=5 * MB, lda=32,
             B=6 * MB, ldb=8, scale=7 * MB, Y=8 * MB, ldy=64, y_bf16=1, ws=16 * MB, ws_bytes=1 << 22)
    a.update(kw)
    return lib().sdb200_linear_lora(*a.values())


@pytest.mark.parametrize("kw,text", [
    (dict(Y=3 * MB), "Y overlaps bias"), (dict(Y=3 * MB + 128), "Y overlaps bias"), (dict(Y=4 * MB), "Y overlaps row_adapter"),
    (dict(Y=7 * MB), "Y overlaps scale"), (dict(Y=16 * MB), "Y overlaps ws"), (dict(Y=16 * MB + 1024), "Y overlaps ws"),
    (dict(X=16 * MB), "ws overlaps X"), (dict(W=16 * MB), "ws overlaps W"), (dict(A=16 * MB), "ws overlaps A"),
    (dict(B=16 * MB), "ws overlaps B"), (dict(bias=16 * MB), "ws overlaps bias"), (dict(rows=16 * MB), "ws overlaps row_adapter"),
    (dict(scale=16 * MB), "ws overlaps scale"), (dict(X=16 * MB - 64), "ws overlaps X"),
])
def test_linear_lora(kw, text):
    refused(lora(**kw), text)


def attn(**kw):
    a = dict(q=MB, ldq=128, k=2 * MB, ldk=64, v=3 * MB, ldv=64, in_type=BF16, out=4 * MB, ldo=128, out_type=BF16, Tq=4, Tkv=9, n_seq=2,
             q_begin=5 * MB, q_len=6 * MB, kv_begin=7 * MB, kv_len=8 * MB, max_q=4, max_kv=9, heads=4, kv_heads=2, d=32, scale=0.1,
             cap=0.0, slopes=9 * MB, causal=1, prefix=10 * MB, ws=None, ws_bytes=0)
    a.update(kw)
    return lib().sdb200_attention_ragged(*a.values())


@pytest.mark.parametrize("kw,text", [
    (dict(out=5 * MB), "out overlaps q_begin"), (dict(out=6 * MB), "out overlaps q_len"), (dict(out=7 * MB), "out overlaps kv_begin"),
    (dict(out=8 * MB - 512), "out overlaps kv_len"), (dict(out=9 * MB), "out overlaps slopes"), (dict(out=10 * MB), "out overlaps prefix"),
])
def test_attention_ragged(kw, text):
    refused(attn(**kw), text)
