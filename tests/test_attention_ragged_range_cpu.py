"""CPU: attention_ragged refuses scales and caps that leave no fp32 number for a factor it multiplies scores
with (scale log2(e), scale / cap, cap / scale, cap log2(e) and its least polynomial coefficient): 0 times an
infinite one would make a score of 0 NaN, and subnormal ones have lost their digits."""
import pytest

from sdb200 import ERR_INVALID_ARG, lib

MB = 1 << 20


def attn(scale, cap):  # out lies over the index arrays, which is looked at later
    rc = lib().sdb200_attention_ragged(MB, 128, 2 * MB, 64, 3 * MB, 64, 1, 5 * MB, 128, 1, 4, 9, 2, 5 * MB, 5 * MB, 5 * MB, 5 * MB, 4,
                                       9, 4, 2, 32, scale, cap, None, 1, None, 4 * MB, 0)
    return rc, lib().sdb200_last_error().decode()


@pytest.mark.parametrize("scale,cap", [
    (3e38, 0.0), (1e-40, 0.0), (1e-45, 0.0), (1.0, 1e-45), (1.0, 1e-40), (1.0, 5e-39), (1.0, 3e38), (0.125, 3.3e38),
    (1e30, 1e-20), (1e-30, 1e20), (1e20, 1e-30), (1.0, 1e38 * 2.5), (1e-20, 1e30),
    (1.0, 1e-37),  # 0.0041 of it, the least coefficient, is subnormal
])
def test_refused(scale, cap):
    rc, text = attn(scale, cap)
    assert rc == ERR_INVALID_ARG and "scale and cap" in text, (rc, text)


@pytest.mark.parametrize("scale,cap", [(1.0, 1e-30), (1.0, 1e30), (1e-10, 0.0), (1e10, 0.0), (1e-10, 1e-10), (0.0884, 50.0), (1.0, 2e-35)])
def test_taken(scale, cap):
    rc, text = attn(scale, cap)
    assert rc == ERR_INVALID_ARG and "out overlaps q_begin" in text, (rc, text)
