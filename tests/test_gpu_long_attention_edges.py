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
