"""Refusals of the attention of any lengths that need an operand's whole extent: every call here is refused on the host, before anything is launched."""
import pytest

from didi_amd import _lib
from didi_amd._lib import lib
from test_long_attention_cpu import args

OVERLAP = _lib.ERR_OVERLAP
MB = 1 << 20
W, WK = 256, 128  # widths of args(): B = 2, 10 queries, 20 keys, bf16
APART = dict(Q=MB, K=2 * MB, V=3 * MB, O=4 * MB, O_lo=5 * MB, lse=6 * MB, dO=7 * MB, dQ=8 * MB, dK=9 * MB, dV=10 * MB, key_mask=11 * MB, key_count=12 * MB,
             table=13 * MB, buckets=14 * MB, num_buckets=32, max_distance=128, workspace=1 << 30)


@pytest.mark.parametrize("kw", [
    dict(O=MB), dict(O=MB + 16), dict(O=MB + 2 * (2 * 10 * W) - 16), dict(O=2 * MB + 16), dict(O=3 * MB - 2 * (2 * 10 * W) + 16), dict(O=11 * MB), dict(O=12 * MB),
    dict(O=13 * MB), dict(O=14 * MB), dict(O=6 * MB), dict(O_lo=4 * MB), dict(O_lo=2 * MB), dict(lse=MB), dict(lse=4 * MB + 2 * (2 * 10 * W) - 4),
    # a column of the neighbour's third, rows that meet another dialog's, the other order of dialogs and rows
    dict(Q=MB, ldq=3 * W, q_batch=30 * W, O=MB + 2 * W - 16, ldo=3 * W, o_batch=30 * W),
    dict(Q=MB, ldq=W, q_batch=11 * W, O=MB + 2 * 2 * W, ldo=W, o_batch=11 * W),
    dict(Q=MB, ldq=2 * W, q_batch=W, O=MB + 2 * 4 * W, ldo=2 * W, o_batch=W),
    dict(Q=MB, ldq=2 * W, q_batch=W, O=MB + 2 * 3 * W, ldo=W, o_batch=10 * W)])
def test_forward_refuses_results_over_operands(kw):
    assert lib.didi_long_attention_forward(args(**{**APART, **kw}), None) == OVERLAP


@pytest.mark.parametrize("kw", [
    dict(dQ=MB), dict(dQ=2 * MB + 16), dict(dK=2 * MB), dict(dV=3 * MB), dict(dQ=4 * MB), dict(dQ=5 * MB), dict(dQ=6 * MB), dict(dQ=7 * MB), dict(dK=11 * MB), dict(dV=12 * MB),
    dict(dK=8 * MB), dict(dV=9 * MB), dict(dV=9 * MB + 16), dict(dtable=13 * MB), dict(dtable=10 * MB + 512), dict(dtable=14 * MB), dict(workspace=MB), dict(workspace=10 * MB),
    dict(workspace=6 * MB), dict(dK=9 * MB, lddk=2 * WK, dk_batch=40 * WK, dV=9 * MB + 2 * WK - 16, lddv=2 * WK, dv_batch=40 * WK)])
def test_backward_refuses_results_over_operands_and_each_other(kw):
    assert lib.didi_long_attention_backward(args(**{**APART, **kw}), None) == OVERLAP


def test_the_refusal_has_a_text():
    assert b"operand" in lib.didi_error_string(OVERLAP)


@pytest.mark.parametrize("kw", [dict(o_batch=W - 8, ldo=2 * W), dict(o_batch=W, ldo=2 * W - 8), dict(o_batch=0, ldo=2 * W), dict(o_batch=10 * W - 8, ldo=W)])
def test_dialogs_of_a_result_over_each_other_are_refused(kw):
    assert lib.didi_long_attention_forward(args(**{**APART, **kw}), None) == -1


def test_rows_too_wide_for_a_tile_are_refused():
    wide = dict(heads=1 << 16, kv_heads=1 << 16, Sq=1, Sk=1, D=64, B=1, ldq=0, ldk=0, ldv=0, ldo=0)
    assert lib.didi_long_attention_forward(args(**{**APART, **wide}), None) == -2


@pytest.mark.parametrize("scale", [1e-40, 2.0 ** -149, 3e38, -1.0, float("nan")])
def test_a_scale_that_fp32_cannot_hold_is_refused(scale):
    assert lib.didi_long_attention_forward(args(**{**APART, "scale": scale}), None) == -1


def test_a_bias_larger_than_any_memory_is_refused():
    for Sq, Sk in ((1 << 30, 1 << 30), (1 << 21, 1 << 20)):
        assert lib.didi_relative_bias(MB, MB, 0, 4, 32, 128, Sq, Sk, 0, MB, None) == -2
        assert lib.didi_relative_bias_backward(MB, MB, 0, 1, 4, 32, 128, Sq, Sk, 0, MB, MB, None) == -2
