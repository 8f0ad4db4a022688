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


@pytest.mark.parametrize("drop_p", [0.0, 0.5, 0.9])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("B,H,Hk,Sq,Sk,D,bias", [(2, 2, 2, 70, 8, 128, False), (1, 4, 2, 130, 40, 64, False), (2, 3, 1, 1, 5, 96, False), (1, 2, 2, 400, 5, 128, False),
                                                 (1, 4, 2, 130, 40, 64, True), (2, 2, 2, 70, 300, 32, True), (24, 16, 16, 130, 6, 64, False)])
def test_large_values_and_gradients_along_them(ops, dtype, B, H, Hk, Sq, Sk, D, bias, drop_p):  # noqa: F811
    """Value rows of norm 1000 to 4000 and do along one of them: score gradients that overflow fp16 unless they are scaled by their own size."""
    q, k, v, do = make(B, H, Hk, Sq, Sk, D, dtype, seed=Sq + Sk, scale_q=2.0 ** -4)
    v.mul_(200 if D > 64 else 400)
    along = v.reshape(B, Sk, Hk, D)[:, torch.arange(Sq, device="cuda") % Sk] / 400  # [B, Sq, Hk, D]
    do.copy_(along.repeat_interleave(H // Hk, 2).reshape(B, Sq, H * D))
    kw = dict(drop_p=drop_p, seed=3)
    keep = keep_of(B, H, Sq, Sk, drop_p, 3) if drop_p else None
    ref = {}
    if bias:
        table = torch.randn(32, H, generator=torch.Generator().manual_seed(3)).to(DT[dtype]).cuda()
        ref["rel_bias"] = kw["rel_bias"] = (table, ops.relative_buckets())
    got, _ = run(ops, q, k, v, do, H, Hk, **kw)
    val, tol = reference(q, k, v, do, H, Hk, dtype, keep=keep, **ref)
    assert all(float(x.abs().max()) < 60000 for n, x in val.items() if n != "lse")
    compare(got, val, tol)


@pytest.mark.parametrize("Sq,Sk,D", [(1, 1, 64), (200, 3, 64), (300, 70, 128), (40, 300, 32)])
def test_fp16_results_beyond_the_range_are_infinite(ops, Sq, Sk, D):  # noqa: F811
    """What overflows fp16 is infinite -- what a loss scaler looks for -- and the rest is right."""
    B, H = 2, 3
    q, k, v, do = make(B, H, H, Sq, Sk, D, "fp16", seed=8)
    do.mul_(14000)
    k.mul_(2.0)
    v.mul_(2.0)
    kw = dict(drop_p=0.5, seed=9)
    keep = keep_of(B, H, Sq, Sk, 0.5, 9)
    got, _ = run(ops, q, k, v, do, H, H, **kw)
    val, tol = reference(q, k, v, do, H, H, "fp16", keep=keep)
    beyond = 0
    for n, x in got.items():
        out, within = val[n].abs() - tol[n] > 65520, val[n].abs() + tol[n] < 65504
        beyond += int(out.sum())
        assert torch.equal(x.double()[out], torch.where(val[n] > 0, math.inf, -math.inf)[out]), n
        assert ((x.double() - val[n]).abs() <= tol[n])[within].all(), n
    assert beyond or Sk == 1 and Sq == 1
    v.fill_(40000.0)
    o = ops.cross_attention(q, k, v, H, **kw)  # half of the probabilities count twice
    want = (torch.softmax((q.double().reshape(B, Sq, H, D).transpose(1, 2) @ k.double().reshape(B, Sk, H, D).permute(0, 2, 3, 1)) / math.sqrt(D), -1) * keep).sum(-1) * 40000
    want = want.transpose(1, 2)[..., None].expand(B, Sq, H, D).reshape(B, Sq, H * D)
    assert torch.isinf(o[want > 65520 * 1.001]).all() and torch.isfinite(o[want < 65504 / 1.001]).all()


@pytest.mark.parametrize("Sq,Sk", [(1, 300), (1, 5000), (40, 300), (300, 1000), (200, 3)])
def test_fp16_values_at_the_largest_number(ops, Sq, Sk):  # noqa: F811
    """A mean of the largest number is that number: the 16-bit probabilities' roundings do not carry it over."""
    q, k, v, _ = make(2, 3, 3, Sq, Sk, 64, "fp16", seed=2)
    for sign in (1.0, -1.0):
        o = ops.cross_attention(q, k, torch.full_like(v, sign * 65504.0), 3)
        # probabilities rounded once, and fp32's rest of Sk terms
        assert ((o.double() - sign * 65504.0).abs() <= 65504.0 * (2 * 2.0 ** -11 + Sk * 2.0 ** -24)).all()


def cuts(Sq):
    """Sizes at which the launches are cut differently: 4 / 2 / 1 row blocks a workgroup, one and several splits of the keys."""
    return {1: [(3, 4, 2, 300, 64), (1, 2, 2, 5000, 128)], 40: [(3, 4, 2, 300, 64), (1, 1, 1, 3000, 96)], 200: [(3, 4, 2, 300, 64), (24, 12, 12, 130, 32)],
            300: [(24, 8, 8, 130, 64)]}[Sq]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("Sq,size", [(s, c) for s in (1, 40, 200, 300) for c in cuts(s)])
def test_nan_and_infinity_at_visible_places_reach_the_result(ops, dtype, Sq, size):  # noqa: F811
    """A query or a visible key that holds NaN gives rows of NaN and gradients of NaN, +inf scores do, whatever the launch's cut, and the other rows,
    heads and dialogs keep their bits."""
    B, H, Hk, Sk, D = size
    q, k, v, do = make(B, H, Hk, Sq, Sk, D, dtype, seed=Sq)
    G, b, row, key, kh = H // Hk, B // 2, Sq // 2, Sk * 2 // 3, Hk - 1
    count = torch.full((B,), Sk, dtype=torch.int32, device="cuda")
    count[0] = key + 1
    cut = lambda x, n: x.reshape(x.shape[0], x.shape[1], n, D)  # noqa: E731
    clean, clean_lse = run(ops, q, k, v, do, H, Hk, key_count=count)
    same = torch.ones(B, Sq, H, dtype=torch.bool, device="cuda")

    def check(hit, got, lse):
        o = cut(got["o"], H)
        assert torch.isnan(o[hit]).all() and torch.isnan(lse.transpose(1, 2)[hit]).all()
        assert torch.equal(o[same & ~hit], cut(clean["o"], H)[same & ~hit]) and torch.equal(lse.transpose(1, 2)[same & ~hit], clean_lse.transpose(1, 2)[same & ~hit])
        assert torch.isnan(cut(got["dq"], H)[hit]).all()
        visible = torch.arange(Sk, device="cuda")[None, :] < count[:, None]
        dead = hit.any(1).reshape(B, Hk, G).any(2)[:, None, :] & visible[:, :, None]  # every visible key of a head gets a part of each row
        for n in ("dk", "dv"):
            assert torch.isnan(cut(got[n], Hk)[dead]).all(), n

    x = q.clone()
    cut(x, H)[b, row, H - 1, 5] = math.nan
    hit = torch.zeros_like(same)
    hit[b, row, H - 1] = True
    check(hit, *run(ops, x, k, v, do, H, Hk, key_count=count))
    for bad in (math.nan, math.inf):
        x = k.clone()
        cut(x, Hk)[b, key, kh, 3] = bad
        hit = torch.zeros_like(same)
        up = cut(q, H)[b, :, kh * G:, 3] > 0  # -inf scores otherwise: a key of no weight
        hit[b, :, kh * G:] = True if math.isnan(bad) else up
        same = torch.ones_like(same)
        same[b, :, kh * G:] = False
        check(hit, *run(ops, q, x, v, do, H, Hk, key_count=count))
        x = v.clone()
        cut(x, Hk)[b, key, kh, 3] = bad
        got = cut(ops.cross_attention(q, k, x, H, kv_heads=Hk, key_count=count, need_grad=True)[0], H)
        assert not torch.isfinite(got[b, :, kh * G:, 3]).any()
        got[b, :, kh * G:, 3] = cut(clean["o"], H)[b, :, kh * G:, 3]
        assert torch.equal(got, cut(clean["o"], H))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("Sq", [1, 40, 200])
def test_a_bucket_outside_the_table_is_nan_in_the_attention(ops, dtype, Sq):  # noqa: F811
    B, H, Sk, D = 2, 3, 300, 64
    q, k, v, do = make(B, H, H, Sq, Sk, D, dtype, seed=1)
    table = torch.randn(32, H, generator=torch.Generator().manual_seed(3)).to(DT[dtype]).cuda()
    for at, value in ((20, 32), (-17, -1), (128, 1 << 30), (-128, 32)):
        buckets = ops.relative_buckets(32, 128)
        buckets[128 + at] = value
        rel = (torch.arange(Sk)[None] - torch.arange(Sq)[:, None] - 100).clamp(-128, 128)
        hit = (rel == at).any(1).cuda()
        o = ops.cross_attention(q, k, v, H, scale=0.125, q_start=100, rel_bias=(table, buckets))
        assert torch.isnan(o[:, hit]).all() and torch.isfinite(o[:, ~hit]).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("Sq,q_start,Sk,D,bias", [(1, 0, 40, 64, False), (7, 20, 60, 32, False), (40, 10, 300, 64, True), (200, 0, 230, 128, False), (33, 3, 37, 64, False),
                                                  (130, 6, 140, 96, True)])
def test_keys_behind_the_last_query_are_never_used(ops, dtype, Sq, q_start, Sk, D, bias):  # noqa: F811
    """Causal: a key past position q_start + Sq - 1 is visible to no row."""
    B, H, Hk = 2, 4, 2
    q, k, v, do = make(B, H, Hk, Sq, Sk, D, dtype, seed=6)
    kw = dict(causal=True, q_start=q_start)
    if bias:
        kw["rel_bias"] = (torch.randn(32, H, generator=torch.Generator().manual_seed(3)).to(DT[dtype]).cuda(), ops.relative_buckets(bidirectional=False))
    for mask in ({}, masks("count", B, Sk), masks("mask", B, Sk)):
        clean = run(ops, q, k, v, do, H, Hk, **kw, **mask)
        for bad in (math.nan, math.inf, -math.inf, torch.finfo(DT[dtype]).max):
            x, y = k.clone(), v.clone()
            x[:, q_start + Sq:] = bad
            y[:, q_start + Sq:] = bad
            got = run(ops, q, x, y, do, H, Hk, **kw, **mask)
            for n in clean[0]:
                assert torch.equal(clean[0][n], got[0][n]), (n, bad)
            assert (got[0]["dk"][:, q_start + Sq:] == 0).all() and (got[0]["dv"][:, q_start + Sq:] == 0).all()


def without(x, hit):
    return torch.where(hit.reshape(hit.shape + (1,) * (x.dim() - hit.dim())), torch.zeros((), dtype=x.dtype, device=x.device), x)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("B,H,Hk,Sq,Sk,D,q_start,bias", [(3, 4, 2, 70, 100, 64, 30, False), (3, 2, 2, 260, 260, 32, 0, False), (3, 3, 3, 40, 200, 96, 100, True),
                                                         (24, 8, 8, 130, 130, 64, 0, False), (3, 2, 1, 150, 150, 128, 0, True), (3, 6, 2, 9, 40, 40, 3, False)])
def test_rows_that_see_nothing_pass_nothing_on(ops, dtype, B, H, Hk, Sq, Sk, D, q_start, bias):  # noqa: F811
    """Left padding under a causal limit: the padded rows see no key.  Whatever their queries and their gradients hold, their results are zeros and
    everything else keeps its bits; an empty dialog likewise."""
    q, k, v, do = make(B, H, Hk, Sq, Sk, D, dtype, seed=13)
    pad = torch.arange(B) * 37 % (Sq * 3 // 4) + q_start  # first visible key
    pad[0], pad[B - 1] = Sk // 3, Sk
    mask = (torch.arange(Sk)[None] >= pad[:, None]).to(torch.int32).cuda()
    blind = (torch.arange(Sq)[None] + q_start < pad[:, None]).cuda()  # [B, Sq]
    kw = dict(causal=True, q_start=q_start, key_mask=mask)
    if bias:
        kw["rel_bias"] = (torch.randn(32, H, generator=torch.Generator().manual_seed(3)).to(DT[dtype]).cuda(), ops.relative_buckets(bidirectional=False))
    clean, lse = run(ops, without(q, blind), k, v, without(do, blind), H, Hk, **kw)
    assert (lse.transpose(1, 2)[blind] == -math.inf).all()
    compare(clean, *reference(without(q, blind), k, v, without(do, blind), H, Hk, dtype, **kw))
    for bad in (math.nan, math.inf, torch.finfo(DT[dtype]).max):
        x, g = q.clone(), do.clone()
        x[blind] = bad
        g[blind] = bad
        got, again = run(ops, x, k, v, g, H, Hk, **kw)
        assert torch.equal(lse, again)
        for n in clean:
            assert torch.equal(clean[n], got[n]), (n, bad)
        assert (got["o"][blind] == 0).all() and (got["dq"][blind] == 0).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("B,H,Hk,Sq,Sk,D", [(3, 2, 2, 1, 300, 64), (3, 4, 2, 70, 130, 64), (24, 12, 12, 130, 150, 64), (3, 2, 1, 300, 40, 128)])
def test_keys_that_nobody_sees_receive_nothing(ops, dtype, B, H, Hk, Sq, Sk, D):  # noqa: F811
    """A query or a gradient that is not a number belongs to the visible keys; the others' gradients are zeros all the same."""
    q, k, v, do = make(B, H, Hk, Sq, Sk, D, dtype, seed=14)
    kw = masks("mask", B, Sk)
    hidden = kw["key_mask"] == 0
    for name in ("q", "do"):
        for bad in (math.nan, math.inf):
            x = {"q": q.clone(), "do": do.clone()}
            x[name][:, Sq // 2, 3::D] = bad
            got, _ = run(ops, x["q"], k, v, x["do"], H, Hk, **kw)
            for n in ("dk", "dv"):
                assert (got[n][hidden] == 0).all(), (n, name, bad)
            if name == "do":
                assert not torch.isfinite(got["dv"].reshape(B, Sk, Hk, D)[..., 3][~hidden]).any()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("Sq", [1, 40, 200])
def test_minus_infinity_in_the_table_hides(ops, dtype, Sq):  # noqa: F811
    """Distances whose bias is -inf, or the lowest number of bf16 and fp32: rows that are left with nothing are rows that see nothing, the others as if
    those keys were masked."""
    B, H, Sk, D = 2, 3, 300, 64
    q, k, v, do = make(B, H, H, Sq, Sk, D, dtype, seed=1)
    table = torch.randn(32, H, generator=torch.Generator().manual_seed(3)).to(DT[dtype]).cuda()
    table[15] = table[31] = -math.inf  # the far distances of both sides
    buckets = ops.relative_buckets(32, 128)
    kw = dict(scale=0.125, q_start=350, rel_bias=(table, buckets), key_count=torch.tensor([300, 200], dtype=torch.int32, device="cuda"))
    got, lse = run(ops, q, k, v, do, H, H, **kw)
    val, tol = reference(q, k, v, do, H, H, dtype, **kw)
    blind = torch.isinf(val["lse"][:, 0])
    assert blind.any() and torch.equal(torch.isinf(lse), torch.isinf(val["lse"]))
    zero = {n: torch.nan_to_num(val[n]) for n in val}
    # the element-wise bound holds the largest |score|, infinite here; instead: probabilities, score gradients and results rounded once each, of o and dq
    # of size 1 (|v|, |k| of a few against probabilities that sum to 1), and fp32's rest of 300 terms
    for n in ("o", "dq"):
        assert (got[n][blind] == 0).all() and torch.isfinite(got[n]).all(), n
        assert (got[n].double() - zero[n]).abs().max() <= 8 * U[dtype] * (1 + zero[n].abs().max()) + 300 * 2.0 ** -22, n
    assert all(torch.isfinite(got[n]).all() for n in got)
    if dtype != "fp16":  # fp16's lowest is an ordinary number to the scores
        table[15] = table[31] = torch.finfo(DT[dtype]).min
        low, low_lse = run(ops, q, k, v, do, H, H, **kw)
        assert torch.equal(lse, low_lse) and all(torch.equal(got[n], low[n]) for n in got)


def test_results_that_share_elements_are_refused(ops):  # noqa: F811
    B, S, H, D = 2, 40, 2, 32
    W = H * D
    buf = torch.randn(B, S, 4 * W, generator=torch.Generator().manual_seed(4)).bfloat16().cuda()
    q, k, v = buf[:, :, :W], buf[:, :, W:2 * W], buf[:, :, 2 * W:3 * W]
    do = torch.randn(B, S, W, device="cuda").bfloat16()
    flat = buf.view(-1)
    for out in (buf[:, :, W - 8:2 * W - 8], buf[:, :, 2 * W + 8:3 * W + 8], flat[W // 2:][:B * S * W].view(B, S, W), k, buf[:, :, 3 * W - 8:4 * W - 8], q,
                flat.as_strided((B, S, W), (W, B * W, 1))):
        with pytest.raises(ValueError, match="operand"):
            ops.cross_attention(q, k, v, H, out=out)
    o, saved = ops.cross_attention(q, k, v, H, need_grad=True)
    a, b, c = (torch.empty_like(do) for _ in range(3))
    two = torch.empty(B, S, 2 * W, dtype=do.dtype, device="cuda")
    for out in ((a, b, b), (a, a, c), (a, b, a), (a, two[:, :, :W], two[:, :, W - 8:2 * W - 8]), (buf[:, :, W // 2:W + W // 2], b, c), (a, saved[1], c), (o, b, c), (a, do, c)):
        with pytest.raises(ValueError, match="operand"):
            ops.cross_attention_backward(q, k, v, o, saved, do, H, out=out)


def test_results_between_the_operands_are_written(ops):  # noqa: F811
    """Columns, rows, dialogs and ranges of the operands' own buffer that hold none of their elements."""
    B, S, H, D = 3, 35, 2, 32
    W = H * D
    g = torch.Generator().manual_seed(4)
    plain = [torch.randn(B, S, W, generator=g).bfloat16().cuda() for _ in range(4)]
    want, saved = ops.cross_attention(*plain[:3], H, need_grad=True)
    grads = ops.cross_attention_backward(*plain[:3], want, saved, plain[3], H)
    layouts = [lambda t, n: t.view(B, S, 8, W)[:, :, n],  # columns of a fused projection
               lambda t, n: t.view(B, 8, S, W)[:, n],  # ranges of a dialog's buffer
               lambda t, n: t.view(8, B, S, W)[n],
               lambda t, n: t.view(S, B, 8, W)[:, :, n].transpose(0, 1),  # rows of the dialogs in turn
               lambda t, n: t.view(8, S, B, W)[n].transpose(0, 1),
               lambda t, n: t.as_strided((B, S, W), ((8 * S + 1) * W, 8 * W, 1), n * W)]  # every eighth row, dialogs an odd number of rows apart
    for at in layouts:
        buf = torch.zeros(8 * B * S * W + B * W, dtype=torch.bfloat16, device="cuda")
        view = [at(buf if at is layouts[-1] else buf[:8 * B * S * W], n) for n in range(8)]
        for x, y in zip(view, plain):
            x.copy_(y)
        o, saved = ops.cross_attention(*view[:3], H, need_grad=True, out=view[4])
        assert torch.equal(o, want)
        got = ops.cross_attention_backward(*view[:3], o, saved, view[3], H, out=view[5:8])
        assert all(torch.equal(x, y) for x, y in zip(got, grads))
        assert all(torch.equal(x, y) for x, y in zip(view, plain))  # the operands are as they were


@pytest.mark.parametrize("ld", [0, 8, -64, 4096])
@pytest.mark.parametrize("Sq,Sk", [(1, 1), (1, 70), (70, 1)])
def test_the_row_stride_of_an_only_row_does_not_count(ops, Sq, Sk, ld):  # noqa: F811
    """C callers: an operand of one row with any row stride."""
    import ctypes as C

    from didi_amd import _lib

    B, H, Hk, D = 2, 4, 2, 64
    q, k, v, do = make(B, H, Hk, Sq, Sk, D, "bf16", seed=3)
    o, saved = ops.cross_attention(q, k, v, H, kv_heads=Hk, need_grad=True)
    want = (o, *ops.cross_attention_backward(q, k, v, o, saved, do, H, kv_heads=Hk))
    W, WK = H * D, Hk * D
    lq, lk = ld if Sq == 1 else W, ld if Sk == 1 else WK
    got = [torch.zeros_like(x) for x in want]
    lse, lo = torch.empty_like(saved[0]), torch.empty_like(o)
    a = _lib.LongAttnArgs(B, H, Hk, Sq, Sk, D, _lib.DT_BF16, 0, 0, 0.0)
    for name, x in dict(Q=q, K=k, V=v, O=got[0], O_lo=lo, lse=lse, dO=do, dQ=got[1], dK=got[2], dV=got[3]).items():
        setattr(a, name, x.data_ptr())
    a.q_batch = a.o_batch = a.do_batch = a.dq_batch = Sq * W
    a.k_batch = a.v_batch = a.dk_batch = a.dv_batch = Sk * WK
    a.ldq = a.ldo = a.lddo = a.lddq = lq
    a.ldk = a.ldv = a.lddk = a.lddv = lk
    ws = torch.empty(1 << 22, dtype=torch.uint8, device="cuda")
    assert max(_lib.lib.didi_long_attention_workspace_bytes(C.byref(a), n) for n in (0, 1)) <= ws.numel()
    a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
    _lib.check(_lib.lib.didi_long_attention_forward(C.byref(a), _lib.current_stream()))
    _lib.check(_lib.lib.didi_long_attention_backward(C.byref(a), _lib.current_stream()))
    assert all(torch.equal(x, y) for x, y in zip(got, want)) and torch.equal(lse, saved[0])


def test_the_ends_of_the_scale(ops):  # noqa: F811
    """A scale that rounds to zero in fp32 meant the default."""
    q, k, v, _ = make(1, 2, 2, 5, 9, 32, "fp32")
    for scale in (1e-50, 1e-40, 0.0, -1.0, 3e38, 1e39, math.inf, math.nan):
        with pytest.raises(ValueError, match="scale"):
            ops.cross_attention(q, k, v, 2, scale=scale)
    o = ops.cross_attention(q, k, v, 2, scale=2.0 ** -126)  # scores of zero: the mean of the values
    # a sum of nine terms, divided once: 12 roundings of fp32
    assert ((o.double() - v.double().mean(1, keepdim=True)).abs() <= 12 * 2.0 ** -24 * v.double().abs().mean(1, keepdim=True)).all()
    q.zero_()
    top = ops.cross_attention(q, k, v, 2, scale=2.0 ** 127)
    assert ((top.double() - v.double().mean(1, keepdim=True)).abs() <= 12 * 2.0 ** -24 * v.double().abs().mean(1, keepdim=True)).all()


@pytest.mark.parametrize("seed,offset", [(-5, 0), (2 ** 64 - 5, 3), (7, -(2 ** 40)), (2 ** 64 + 3, 2 ** 64 - 1), (torch.tensor(11), torch.tensor(1 << 34))])
def test_seeds_are_taken_as_the_training_attention_takes_them(ops, seed, offset):  # noqa: F811
    B, H, S, D = 2, 2, 20, 32
    q, k, v, _ = make(B, H, H, S, S, D, "fp32", seed=15)
    v.copy_((torch.arange(S * H * D).reshape(S, H * D) % S == torch.arange(S)[:, None]).float().cuda()[None])  # ones and zeros: o sums probabilities
    kw = dict(drop_p=0.5, seed=seed, offset=offset)
    a, b = ops.cross_attention(q, k, v, H, **kw), ops.attention_train(q, k, v, H, **kw)
    # probabilities to fp32's 32 + 8 roundings of scores of size 8 in both; another mask would differ by a probability, 0.05
    assert (a - b).abs().max() < 1e-4 and (a != ops.cross_attention(q, k, v, H)).any()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("H,Hk,Sq,Sk,D,bias,causal", [(4, 2, 1, 300, 64, False, False), (3, 3, 40, 130, 96, True, False), (4, 4, 130, 97, 64, False, False),
                                                      (2, 1, 70, 5000, 32, False, False), (24, 24, 260, 130, 64, True, False), (2, 2, 50, 60, 128, False, True)])
def test_a_negative_count_averages_the_values(ops, dtype, H, Hk, Sq, Sk, D, bias, causal):  # noqa: F811
    """A dialog whose key count is negative has scores of 0 at all its keys, and the gradients of scores that a mask has been added to."""
    B, G = 3, H // Hk
    q, k, v, do = make(B, H, Hk, Sq, Sk, D, dtype, seed=16)
    mask = (torch.rand(B, Sk, generator=torch.Generator().manual_seed(5)) < 0.7).int().cuda()
    mask[1] = 0
    count = torch.tensor([Sk, -1, (Sk + 1) // 2], dtype=torch.int32, device="cuda")
    kw = dict(key_mask=mask, key_count=count, causal=causal, q_start=5 if causal else 0)
    if bias:
        table = torch.randn(32, H, generator=torch.Generator().manual_seed(3)).to(DT[dtype]).cuda()
        kw["rel_bias"] = (table, ops.relative_buckets())
    got, lse = run(ops, q, k, v, do, H, Hk, **kw)
    # the other dialogs as ever
    rest = {**kw, "key_mask": mask[::2].contiguous(), "key_count": count[::2].contiguous()}
    val_rest, tol_rest = reference(*(x[::2].contiguous() for x in (q, k, v, do)), H, Hk, dtype, **rest)
    for n in ("o", "dq", "dk", "dv"):
        assert ((got[n][::2].double() - val_rest[n]).abs() <= tol_rest[n]).all(), n
    # the dialog itself: scores of zero, by a scale of zero in the definition; dq and dk are then those of scale 1, times the scale
    val, tol = reference(q[1:2] * 0, k[1:2], v[1:2], do[1:2], H, Hk, dtype, causal=causal, q_start=kw["q_start"])
    assert ((got["o"][1:2].double() - val["o"]).abs() <= tol["o"]).all() and ((got["dv"][1:2].double() - val["dv"]).abs() <= tol["dv"]).all()
    assert ((got["dq"][1:2].double() - val["dq"]).abs() <= tol["dq"]).all()
    seen = torch.arange(Sk, device="cuda")[None] <= torch.arange(Sq, device="cuda")[:, None] + 5 if causal else torch.ones(Sq, Sk, dtype=torch.bool, device="cuda")
    p = seen.double() / seen.sum(1, keepdim=True)
    heads = lambda x, n: x[1].double().reshape(-1, n, D).transpose(0, 1)  # noqa: E731
    dO, V, Q = heads(do, H), heads(v, Hk).repeat_interleave(G, 0), heads(q, H)
    dp = dO @ V.transpose(-1, -2)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    by_head = lambda x: x.reshape(Hk, G, Sk, D).sum(1).transpose(0, 1).reshape(Sk, Hk * D)  # noqa: E731
    dk = by_head(ds.transpose(-1, -2) @ Q) / math.sqrt(D)
    # ds: rounded once, D = do . o to the remainder's or fp32's bits; then a sum over rows and heads, rounded once
    u, lo = U[dtype], U[dtype] if dtype == "fp32" else U[dtype] ** 2
    err = ds.abs() * (0 if dtype == "fp32" else u) + p * (dO.abs() @ V.abs().transpose(-1, -2) + (dO.abs() * (p @ V.abs())).sum(-1, keepdim=True)) * (
        (0 if dtype == "fp32" else u) + lo + (D + Sk + 8) * 2.0 ** -24) + SUB[dtype] * 2.0 ** -6 * dO.norm(dim=-1).amax()
    bound = by_head(err.transpose(-1, -2) @ Q.abs() + (G * Sq + 4) * 2.0 ** -24 * (ds.abs().transpose(-1, -2) @ Q.abs())) / math.sqrt(D) + u * dk.abs() + SUB[dtype]
    assert ((got["dk"][1].double() - dk).abs() <= bound).all()
    want = torch.log(seen.sum(1).double())
    assert ((lse[1].double() - want).abs() <= 1e-5 * (1 + want)).all()
    if bias:
        hot = torch.nn.functional.one_hot(bucket_of(kw["rel_bias"][1], Sq, Sk, 0), 32).double().reshape(Sq * Sk, 32)
        by = lambda x: (x.reshape(H, Sq * Sk) @ hot).t()  # noqa: E731
        total = val_rest["dtable"] + by(ds)
        slack = tol_rest["dtable"] + by(err + ds.abs() * (B * Sq + 4) * 2.0 ** -24) + u * total.abs() + SUB[dtype]
        assert ((got["dtable"].double() - total).abs() <= slack).all()


# Sizes at which a workgroup of the gradient takes 64 rows (16 a wave, two at a time, over and again), a row has more chunks than a wave reads at a
# time (2048 columns of 16 bits, 1024 of fp32), or none: narrower than a chunk, or beyond the table's distances throughout
@pytest.mark.parametrize("dtype,B,H,Sq,Sk,q_start,bidirectional", [
    ("bf16", 1, 32, 4100, 2111, 7, True), ("fp16", 2, 32, 2100, 2053, 0, False), ("fp32", 1, 64, 2049, 1027, 5, True), ("bf16", 2, 33, 2000, 2603, 300, True),
    ("fp32", 1, 32, 4200, 9, 0, True), ("fp16", 1, 32, 4200, 5, 0, True), ("bf16", 3, 16, 3001, 1, 0, False), ("fp16", 1, 64, 2050, 601, 4000, True),
    ("fp32", 1, 1, 65, 300001, 0, True), ("bf16", 1, 2, 7, 200003, 100, True)])
def test_long_gradient_of_the_bias(ops, dtype, B, H, Sq, Sk, q_start, bidirectional):  # noqa: F811
    buckets = ops.relative_buckets(32, 128, bidirectional)
    d = torch.randn(B, H, Sq, Sk, generator=torch.Generator(device="cuda").manual_seed(Sq), device="cuda").to(DT[dtype])
    got = ops.relative_bias_backward(d, buckets, 32, q_start=q_start)
    bucket = bucket_of(buckets, Sq, Sk, q_start)
    other = [bucket != t for t in range(32)]
    assert torch.equal(got, ops.relative_bias_backward(d, buckets, 32, q_start=q_start))
    for h in range(H):
        by = lambda x: torch.stack([x.masked_fill(other[t], 0.0).sum() for t in range(32)])  # noqa: E731
        x = d[:, h].double()
        want, size = by(x), by(x.abs())
        # fp32 sums: a lane takes 64 rows of at most Sk / 64 elements, then partial sums of B Sq / 64 workgroups
        assert ((got[:, h].double() - want).abs() <= size * (B * Sq + Sk + 16) * 2.0 ** -24 + U[dtype] * want.abs() + SUB[dtype]).all(), h


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_what_was_saved_is_checked(ops, dtype):  # noqa: F811
    q, k, v, do = make(2, 2, 2, 9, 12, 32, dtype)
    o, (lse, lo) = ops.cross_attention(q, k, v, 2, need_grad=True)
    bad = [(lse.cpu(), lo), (lse.double(), lo), (lse[:1], lo), (lse.transpose(1, 2), lo), (lse, torch.empty(2, 9, 64, dtype=DT[dtype])),
           (lse, torch.empty(2, 9, 64, dtype=torch.float16, device="cuda")), (lse, torch.empty(2, 9, 128, dtype=DT[dtype], device="cuda")[:, :, :64])]
    for saved in bad:
        with pytest.raises(ValueError):
            ops.cross_attention_backward(q, k, v, o, saved, do, 2)
    # one dialog or one row: strides that do not count may differ
    for x in ((q[:1], k[:1], v[:1], do[:1]), (q[:, :1], k, v, do[:, :1])):
        x = [t.contiguous() for t in x]
        o, saved = ops.cross_attention(*x[:3], 2, need_grad=True)
        want = ops.cross_attention_backward(*x[:3], o, saved, x[3], 2)
        B, S, W = o.shape
        view = o.as_strided((B, S, W), (S * W if B > 1 else 8, W if S > 1 else 8, 1))
        got = ops.cross_attention_backward(*x[:3], view, saved, x[3], 2)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_keys_past_four_gibibytes(ops):  # noqa: F811
    """Rows, outputs and gradients whose offsets pass 32 bits: a few visible keys of a long cache, the last one among them, against the same keys alone."""
    H, D, Sk = 16, 128, (1 << 20) + 4097  # 4 KiB a row
    W = H * D
    g = torch.Generator().manual_seed(17)
    at = torch.tensor([0, 5, (1 << 19) - 1, 1 << 19, (1 << 20) - 1, 1 << 20, (1 << 20) + 1, (1 << 20) + 64, Sk - 2, Sk - 1]).cuda()
    k, v = (torch.full((1, Sk, W), math.nan, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    few = [torch.randn(1, at.numel(), W, generator=g).bfloat16().cuda() for _ in range(2)]
    k[:, at], v[:, at] = few
    mask = torch.zeros(1, Sk, dtype=torch.int32, device="cuda")
    mask[:, at] = 1
    for Sq in (1, 65):
        q, do = (torch.randn(1, Sq, W, generator=g).bfloat16().cuda() for _ in range(2))
        val, tol = reference(q, few[0], few[1], do, H, H, "bf16")
        o, saved = ops.cross_attention(q, k, v, H, key_mask=mask, need_grad=True)
        dq, dk, dv = ops.cross_attention_backward(q, k, v, o, saved, do, H, key_mask=mask)
        compare({"o": o, "dq": dq, "dk": dk[:, at], "dv": dv[:, at]}, val, tol)
        for x in (dk, dv):
            x[:, at] = 0
            assert not x.any()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("H,Sq,Sk", [(3, 7, 9), (1, 77, 301), (5, 133, 1023)])
def test_gradient_of_the_bias_from_one_dialog_of_many(ops, dtype, H, Sq, Sk):  # noqa: F811
    """A contiguous dialog whose first element lies anywhere in memory."""
    buckets = ops.relative_buckets(32, 128)
    d = torch.randn(3, H, Sq, Sk, generator=torch.Generator().manual_seed(Sk)).to(DT[dtype]).cuda()
    for b in range(3):
        assert torch.equal(ops.relative_bias_backward(d[b], buckets, 32), ops.relative_bias_backward(d[b].clone(), buckets, 32))
