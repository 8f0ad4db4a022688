"""Attention of any lengths and the learned relative bias where they are easy to get wrong: long biases of odd widths, operands that hold
infinities and NaN, the ends of the types' ranges, dialogs whose mask leaves nothing."""
import math

import pytest
import torch

from test_gpu_long_attention import DT, SUB, U, bucket_of, compare, make, masks, ops, reference, run  # noqa: F401

pytestmark = pytest.mark.gpu


# Sizes at which a thread of the dense bias takes several chunks; all but the last two have heads whose block starts inside a 16-byte chunk, the narrow
# ones so that a step of 256 chunks stays among the distances that the table tells apart.
@pytest.mark.parametrize("dtype,H,Sq,Sk,q_start", [
    ("fp32", 32, 1023, 1023, 0), ("fp32", 12, 1023, 1023, 0), ("bf16", 32, 2047, 2047, 0), ("fp16", 12, 2045, 2045, 0), ("fp32", 32, 511, 511, 0),
    ("fp16", 9, 1025, 1023, 300), ("bf16", 8, 400001, 5, 0), ("fp16", 8, 300001, 7, 0), ("fp32", 9, 800001, 3, 0), ("bf16", 9, 1500001, 4, 0),
    ("bf16", 9, 3000001, 2, 0), ("fp32", 9, 3000001, 1, 0), ("fp32", 32, 1024, 1024, 0), ("bf16", 32, 2048, 2047, 7)])
def test_long_dense_bias_is_the_gathered_table(ops, dtype, H, Sq, Sk, q_start):  # noqa: F811
    buckets = (torch.arange(1025, dtype=torch.int32) * 7 % 1024).cuda()  # every distance another bucket, but for the ends'
    table = torch.randn(1024, H, generator=torch.Generator().manual_seed(Sq)).to(DT[dtype]).cuda()
    got = ops.relative_bias(table, buckets, Sq, Sk, q_start=q_start)
    bucket = bucket_of(buckets, Sq, Sk, q_start)
    for h in range(H):
        assert torch.equal(got[h], table[:, h][bucket]), h


def keep_of(B, H, Sq, Sk, p, seed, offset=0):
    """1 / (1 - p) where the documented stream keeps a probability, 0 where it drops it: [B, H, Sq, Sk]."""
    import numpy as np

    from oracle.philox import philox4x32_10

    G4 = (Sk + 3) // 4
    ctr = np.arange(B * H * Sq * G4, dtype=np.uint64) + np.uint64(offset)
    ctr = np.stack([ctr & np.uint64(0xFFFFFFFF), ctr >> np.uint64(32), ctr * 0, ctr * 0], 1).astype(np.uint32)
    words = philox4x32_10(ctr, np.array([seed & 0xFFFFFFFF, seed >> 32], np.uint32))
    words = torch.from_numpy(words.astype(np.int64)).reshape(B, H, Sq, G4 * 4)[..., :Sk]
    return (words >= int(np.float32(p) * np.float32(2.0 ** 32))).double().cuda() / float(np.float32(1) - np.float32(p))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("Sq", [1, 200])
def test_high_dropout_over_scores_that_grow(ops, dtype, Sq):  # noqa: F811
    """Scores that grow along the keys by just under 8 powers of two, which the running maximum lags behind, and a kept probability's factor of 1000: their
    product lies beyond fp16."""
    B, H, Sk, D, p, seed = 2, 3, 640, 32, 0.999, 77
    q, k, v, do = make(B, H, H, Sq, Sk, D, dtype, seed=11)
    q.fill_(0.5)
    k.mul_(2.0 ** -6)
    k[:, Sk // 2:] += 7.8 * math.log(2.0) / (0.5 * math.sqrt(D))
    do.mul_(2.0 ** -8)
    got, _ = run(ops, q, k, v, do, H, H, drop_p=p, seed=seed)
    val, tol = reference(q, k, v, do, H, H, dtype, keep=keep_of(B, H, Sq, Sk, p, seed))
    assert (val["o"] != 0).any()
    compare(got, val, tol)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_the_highest_dropout_over_one_key(ops, dtype):  # noqa: F811
    """One key: every probability is 1, a kept one counts 100000 times."""
    B, H, Sq, D, p, seed = 1, 4, 1 << 16, 32, 0.99999, 5
    q, k, v, do = make(B, H, H, Sq, 1, D, dtype, seed=12)
    v.mul_(2.0 ** -8)
    do.mul_(2.0 ** -8)
    o, saved = ops.cross_attention(q, k, v, H, need_grad=True, drop_p=p, seed=seed)
    dv = ops.cross_attention_backward(q, k, v, o, saved, do, H, drop_p=p, seed=seed)[2]
    keep = keep_of(B, H, Sq, 1, p, seed)[0, :, :, 0].t().repeat_interleave(D, 1)  # [Sq, H D]
    want_o, want_dv = keep * v.double()[0], (keep * do.double()[0]).sum(0)
    assert 0 < int((keep > 0).sum()) and (keep[0] == 0).all()
    n24 = 64 * 2.0 ** -24
    assert ((o.double()[0] - want_o).abs() <= (U[dtype] + n24) * want_o.abs() + SUB[dtype]).all()
    assert ((dv.double()[0, 0] - want_dv).abs() <= U[dtype] * want_dv.abs() + n24 * (keep * do.double()[0].abs()).sum(0) + SUB[dtype]).all()
