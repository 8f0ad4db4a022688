"""Refusals of the attention of any lengths and of the relative bias: every one is decided on the host, before anything is launched."""
import ctypes as C

import pytest
import torch

from didi_amd import _lib, ops
from didi_amd._lib import lib

BAD, UNSUPPORTED, WORKSPACE = -1, -2, -4
P = 1 << 20  # an aligned address that nothing reads: every call here is refused, or has nothing to do


def args(**kw):
    a = _lib.LongAttnArgs(2, 4, 2, 10, 20, 64, _lib.DT_BF16, 0, 0, 0.0)
    W, Wk = 256, 128
    base = dict(Q=P, K=P, V=P, O=P, q_batch=10 * W, k_batch=20 * Wk, v_batch=20 * Wk, o_batch=10 * W, ldq=W, ldk=Wk, ldv=Wk, ldo=W, lse=P, dO=P, do_batch=10 * W,
                lddo=W, dQ=P, dK=P, dV=P, dq_batch=10 * W, dk_batch=20 * Wk, dv_batch=20 * Wk, lddq=W, lddk=Wk, lddv=Wk, workspace=P, workspace_bytes=1 << 40)
    for k, v in {**base, **kw}.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("rc,kw", [
    (BAD, dict(B=-1)), (BAD, dict(heads=3)), (BAD, dict(kv_heads=0)), (BAD, dict(Sq=-1)), (BAD, dict(D=0)), (BAD, dict(dtype=3)), (BAD, dict(q_start=-1)),
    (BAD, dict(scale=-1.0)), (BAD, dict(scale=float("nan"))), (BAD, dict(scale=float("inf"))), (BAD, dict(drop_p=1.0)), (BAD, dict(drop_p=-0.1)),
    (BAD, dict(Q=None)), (BAD, dict(K=None)), (BAD, dict(O=None)), (BAD, dict(Q=P + 2)), (BAD, dict(V=P + 8)), (BAD, dict(ldq=255)), (BAD, dict(ldk=132)),
    (BAD, dict(ldk=64)), (BAD, dict(k_batch=2561)), (BAD, dict(k_batch=-128)), (BAD, dict(o_batch=2048)), (BAD, dict(table=P)),
    (BAD, dict(table=P, buckets=P, num_buckets=0, max_distance=8)), (BAD, dict(dtable=P)), (BAD, dict(workspace=P + 4)),
    (UNSUPPORTED, dict(D=136)), (UNSUPPORTED, dict(D=60)), (UNSUPPORTED, dict(table=P, buckets=P, num_buckets=8, max_distance=513)),
    (UNSUPPORTED, dict(table=P, buckets=P, num_buckets=1025, max_distance=8)), (UNSUPPORTED, dict(Sk=(1 << 30) + 1)), (UNSUPPORTED, dict(q_start=1 << 30)),
    (UNSUPPORTED, dict(B=1 << 19)),
])
def test_forward_refuses(rc, kw):
    assert lib.didi_long_attention_forward(args(**kw), None) == rc
    if "workspace" not in kw:
        assert lib.didi_long_attention_workspace_bytes(args(**kw), 0) == 0


@pytest.mark.parametrize("rc,kw", [(BAD, dict(dO=None)), (BAD, dict(dK=None)), (BAD, dict(lse=None)), (BAD, dict(dk_batch=0)), (BAD, dict(dv_batch=128)),
                                   (BAD, dict(lddq=8)), (WORKSPACE, dict(workspace_bytes=16)), (WORKSPACE, dict(workspace=None))])
def test_backward_refuses(rc, kw):
    assert lib.didi_long_attention_backward(args(**kw), None) == rc


def test_forward_wants_its_workspace():
    assert lib.didi_long_attention_workspace_bytes(args(Sk=4096, k_batch=4096 * 128, v_batch=4096 * 128), 0) > 0
    assert lib.didi_long_attention_forward(args(Sk=4096, k_batch=4096 * 128, v_batch=4096 * 128, workspace_bytes=8), None) == WORKSPACE


def test_nothing_to_do_is_no_error():
    assert lib.didi_long_attention_forward(args(B=0, Q=None, K=None, V=None, O=None), None) == 0
    assert lib.didi_long_attention_forward(args(Sq=0, Q=None, O=None), None) == 0


@pytest.mark.parametrize("rc,kw", [(BAD, dict(buckets=None)), (BAD, dict(heads=0)), (BAD, dict(q_start=-1)), (BAD, dict(dtype=9)), (BAD, dict(table=None)), (BAD, dict(out=P + 4)),
                                   (UNSUPPORTED, dict(max_distance=600)), (UNSUPPORTED, dict(num_buckets=5000)), (UNSUPPORTED, dict(heads=70000))])
def test_bias_refuses(rc, kw):
    a = dict(table=P, buckets=P, dtype=0, heads=4, num_buckets=32, max_distance=128, Sq=8, Sk=8, q_start=0, out=P)
    a.update(kw)
    assert lib.didi_relative_bias(*a.values(), None) == rc
    if "table" in kw or "out" in kw:
        return
    assert lib.didi_relative_bias_backward(P, a["buckets"], a["dtype"], 1, *[a[x] for x in ("heads", "num_buckets", "max_distance", "Sq", "Sk", "q_start")], P, P, None) == rc


def test_python_checks_name_the_operand():
    q, k = torch.zeros(2, 4, 64), torch.zeros(2, 6, 64)
    with pytest.raises(ValueError, match="on the GPU"):
        ops.cross_attention(q, k, k, 2)
    for kw in (dict(num_buckets=31), dict(num_buckets=2), dict(max_distance=8)):
        with pytest.raises(ValueError, match="num_buckets"):
            ops.relative_buckets(device="cpu", **kw)
    with pytest.raises(ValueError, match="buckets must be"):
        ops.relative_bias(torch.zeros(32, 2), torch.zeros(256, dtype=torch.int32), 4, 4)
    with pytest.raises(ValueError, match="table must be"):
        ops.relative_bias(torch.zeros(32, 2, dtype=torch.float64), torch.zeros(257, dtype=torch.int32), 4, 4)
    with pytest.raises(ValueError, match="dbias must be"):
        ops.relative_bias_backward(torch.zeros(4, 4), torch.zeros(257, dtype=torch.int32), 32)


def test_buckets_by_hand():
    b = ops.relative_buckets(8, 16, device="cpu").tolist()
    # two sides of four: distances 0 and 1 by themselves, then from 2 and from ceil(2 sqrt(8)) = 6 on
    assert b[16:] == [0, 5, 6, 6, 6, 6] + [7] * 11 and b[16::-1] == [0, 1, 2, 2, 2, 2] + [3] * 11
    one = ops.relative_buckets(4, 16, bidirectional=False, device="cpu").tolist()
    assert one[16:] == [0] * 17 and one[16::-1] == [0, 1, 2, 2, 2, 2] + [3] * 11
    assert C.sizeof(_lib.LongAttnArgs) % 8 == 0
