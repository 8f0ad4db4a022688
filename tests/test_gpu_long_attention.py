"""Attention of any lengths and the learned relative position bias against their definition in 64 bits.

Element-wise bounds, from the roundings alone (u = half a step of the type: bf16 2^-8, fp16 2^-11, fp32 2^-24):
  scores      |t' - t| <= e_i = scale max_j sum_d |q||k| (D + 4) 2^-24 + 2^-21 (1 + |t|max): a relative error of 2 e_i in every probability
              (its own and the sum's) next to fp32's few 2^-24
  o           probabilities rounded once (u), the output once (u): u (A + |o|) + 2 e A,  A = sum_j p |v|
  ds          D = do . o from the rounded output: p u sum_d |do||o|; + |ds| (u + 2 e) + p sum |do||v| (D + 4) 2^-24
  dq, dk, dv, dtable: the sums of those over keys, rows or a bucket, plus u of the result
in fp32 the stored values are not rounded again (u counts the output alone) and the sums over n terms add n 2^-24 of their absolute sum.
fp16 adds 2^-24 absolute (its subnormal step) to every 16-bit rounding of a probability and of an output.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
U = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11, "fp32": 2.0 ** -24}
SUB = {"bf16": 0.0, "fp16": 2.0 ** -24, "fp32": 0.0}


@pytest.fixture(scope="module")
def ops():
    from didi_amd import ops as o

    return o


def make(B, H, Hk, Sq, Sk, D, dtype, seed=0, scale_q=1.0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).to(DT[dtype]).cuda()  # noqa: E731
    return (torch.randn(B, Sq, H * D, generator=g) * scale_q).to(DT[dtype]).cuda(), r(B, Sk, Hk * D), r(B, Sk, Hk * D), r(B, Sq, H * D)


def bucket_of(buckets, Sq, Sk, q_start):
    md = buckets.numel() // 2
    rel = torch.arange(Sk)[None] - torch.arange(Sq)[:, None] - q_start
    return buckets.cpu()[rel.clamp(-md, md) + md].long().cuda()


def split_heads(x, n):
    return x.reshape(x.shape[0], x.shape[1], n, -1).transpose(1, 2)


def reference(q, k, v, do, H, Hk, dtype, scale=None, causal=False, q_start=0, key_mask=None, key_count=None, rel_bias=None, keep=None):
    """Everything in 64 bits on the operands as they are -> ({name: value}, {name: element-wise bound})."""
    B, Sq, HD = q.shape
    Sk, D, G = k.shape[1], HD // H, H // Hk
    u, sub = U[dtype], SUB[dtype]
    up = 0.0 if dtype == "fp32" else u  # rounding of probabilities and score gradients
    scale = 1 / math.sqrt(D) if scale is None else scale
    see = torch.ones(B, 1, Sq, Sk, dtype=torch.bool, device=q.device)
    j = torch.arange(Sk, device=q.device)
    if key_count is not None:
        see = see & (j[None] < key_count[:, None].long())[:, None, None]
    if key_mask is not None:
        see = see & (key_mask != 0)[:, None, None]
    if causal:
        see = see & (j[None] <= torch.arange(Sq, device=q.device)[:, None] + q_start)[None, None]
    seen = see.any(2)[:, 0]  # keys that any row may use: the others' contents do not exist
    k, v = (torch.where(seen[..., None], x.double(), 0.0) for x in (k, v))
    Q, dO = split_heads(q.double(), H), split_heads(do.double(), H)
    K, V = (split_heads(x, Hk).repeat_interleave(G, 1) for x in (k, v))
    t = Q @ K.transpose(-1, -2) * scale
    if rel_bias is not None:
        bucket = bucket_of(rel_bias[1], Sq, Sk, q_start)
        t = t + rel_bias[0].double()[bucket].permute(2, 0, 1)[None]
    t = torch.where(see, t, -math.inf)
    p = torch.nan_to_num(torch.softmax(t, -1), nan=0.0) if Sk else t
    lse = torch.logsumexp(t, -1)
    drop = torch.ones_like(p) if keep is None else keep.double()
    pd = p * drop
    o = pd @ V
    mag = Q.abs() @ K.abs().transpose(-1, -2) * scale
    tm = torch.where(see, t.abs(), 0.0)
    amax = lambda x: x.amax(-1, keepdim=True) if Sk else x.sum(-1, keepdim=True)  # noqa: E731
    e = amax(torch.where(see, mag, 0.0)) * (D + 4) * 2.0 ** -24 + 2.0 ** -21 * (1 + amax(tm))
    n24 = lambda n: (n + 4) * 2.0 ** -24  # noqa: E731
    A = pd @ V.abs()
    val, tol = {}, {}
    rows = lambda x: x.transpose(1, 2).reshape(B, x.shape[2], -1)  # noqa: E731
    keys = lambda x: rows(x.reshape(B, Hk, G, *x.shape[2:]).sum(2))  # noqa: E731
    val["o"], tol["o"] = rows(o), rows(A * (up + 2 * e + n24(Sk)) + u * o.abs() + sub * (1 + see.double() @ V.abs()))
    dp = (dO @ V.transpose(-1, -2)) * drop
    delta = (dO * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    dpm = (dO.abs() @ V.abs().transpose(-1, -2)) * drop
    lo = u if dtype == "fp32" else u * u  # 16 bits: with the remainder plane
    dd = (dO.abs() * o.abs()).sum(-1, keepdim=True) * (lo + n24(D)) + (dO.abs() * (A * (up + 2 * e + n24(Sk)))).sum(-1, keepdim=True)
    err = p * dd + ds.abs() * (2 * e + 2.0 ** -21) + p * dpm * n24(D)
    # fp16 score gradients are scaled by powers of two before their rounding: no subnormals in range; saturation-free
    r16 = err + up * ds.abs() + (2.0 ** -30 * dO.norm(dim=-1).amax() if dtype == "fp16" else 0.0) * (p > 0)
    val["dv"], tol["dv"] = keys(pd.transpose(-1, -2) @ dO), None
    tol["dv"] = keys((pd * (up + 2 * e + n24(G * Sq)) + sub * see).transpose(-1, -2) @ dO.abs()) + u * val["dv"].abs() + sub
    val["dq"] = rows(ds @ K) * scale
    tol["dq"] = rows((r16 + ds.abs() * n24(Sk)) @ K.abs()) * scale + u * val["dq"].abs() + sub
    val["dk"] = keys(ds.transpose(-1, -2) @ Q) * scale
    tol["dk"] = keys((r16 + ds.abs() * n24(G * Sq)).transpose(-1, -2) @ Q.abs()) * scale + u * val["dk"].abs() + sub
    if rel_bias is not None:
        nb = rel_bias[0].shape[0]
        hot = torch.nn.functional.one_hot(bucket, nb).double().reshape(Sq * Sk, nb)
        by = lambda x: (x.sum(0).reshape(H, Sq * Sk) @ hot).t()  # noqa: E731
        val["dtable"] = by(ds)
        tol["dtable"] = by(err + ds.abs() * n24(B * Sq)) + u * val["dtable"].abs() + sub
    val["lse"] = lse
    return val, tol


def run(ops, q, k, v, do, H, Hk, **kw):
    o, saved = ops.cross_attention(q, k, v, H, kv_heads=Hk, need_grad=True, **kw)
    g = ops.cross_attention_backward(q, k, v, o, saved, do, H, kv_heads=Hk, **kw)
    got = dict(zip(("dq", "dk", "dv", "dtable"), g), o=o)
    again = ops.cross_attention_backward(q, k, v, o, saved, do, H, kv_heads=Hk, **kw)
    for a, b in zip(g, again):  # deterministic (bytes: NaN compares too)
        assert torch.equal(a.view(torch.uint8) if a.numel() else a, b.view(torch.uint8) if b.numel() else b)
    return got, saved[0]


def compare(got, val, tol):
    for n, x in got.items():
        d = (x.double() - val[n]).abs()
        bad = ~(d <= tol[n])
        assert not bad.any(), f"{n}: {int(bad.sum())} of {d.numel()} beyond the bound, worst {float((d / tol[n].clamp_min(1e-300)).max()):.3g} x"


CASES = [
    # B, H, Hk, Sq, Sk, D, mask, causal, q_start, bias
    (1, 2, 2, 1, 1, 64, "none", False, 0, False),
    (1, 3, 3, 1, 64, 64, "none", False, 0, False),
    (2, 4, 4, 63, 97, 64, "none", False, 0, False),
    (3, 4, 2, 33, 130, 64, "count", False, 0, False),
    (3, 2, 1, 129, 200, 80, "mask", False, 0, False),
    (2, 2, 2, 100, 100, 40, "none", True, 0, False),
    (2, 4, 1, 5, 300, 128, "mask", True, 295, False),
    (2, 2, 2, 40, 20, 96, "count", True, 3, False),
    (2, 3, 3, 150, 170, 64, "count", False, 0, True),
    (2, 2, 1, 97, 300, 32, "mask", True, 203, True),
    (1, 8, 8, 1, 1000, 64, "none", False, 999, True),
    (1, 2, 2, 700, 9, 16, "none", False, 0, True),
    (4, 6, 6, 256, 512, 64, "count", False, 0, True),
    (1, 1, 1, 40, 2000, 128, "mask", False, 0, False),
    (5, 8, 2, 2, 65, 8, "mask", False, 0, False),
    (3, 2, 1, 2, 12501, 64, "mask", False, 0, False),  # more keys than the ring of mask words holds, split and
    (1, 2, 2, 130, 9003, 32, "mask", True, 8873, False),  # in one piece
]


def masks(mask, B, Sk, seed=1):
    g = torch.Generator().manual_seed(seed)
    if mask == "none":
        return {}
    n = torch.randint(0, Sk + 1, (B,), generator=g, dtype=torch.int32)
    n[0] = Sk
    if B > 2:
        n[-1] = 0
    if mask == "count":
        return {"key_count": n.cuda()}
    keep = (torch.rand(B, Sk, generator=g) < 0.7) & (torch.arange(Sk)[None] < n[:, None])
    return {"key_mask": keep.to(torch.int32).cuda()}


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_forward_and_backward(ops, case, dtype):
    B, H, Hk, Sq, Sk, D, mask, causal, q_start, bias = case
    kw = dict(masks(mask, B, Sk), causal=causal, q_start=q_start)
    q, k, v, do = make(B, H, Hk, Sq, Sk, D, dtype, seed=Sq + Sk, scale_q=D ** -0.5 if bias else 1.0)
    if bias:
        kw["scale"] = 1.0
        table = (torch.randn(32, H, generator=torch.Generator().manual_seed(3)) * 0.7).to(DT[dtype]).cuda()
        kw["rel_bias"] = (table, ops.relative_buckets(32, 128, bidirectional=not causal))
    got, lse = run(ops, q, k, v, do, H, Hk, **kw)
    val, tol = reference(q, k, v, do, H, Hk, dtype, **kw)
    compare(got, val, tol)
    want = val["lse"]
    assert torch.equal(torch.isinf(want), torch.isinf(lse))
    fin = torch.isfinite(want)
    assert (lse.double()[fin] - want[fin]).abs().le(1e-4 * (1 + want[fin].abs())).all()
    # rows without a key: exact zeros
    gone = ~fin.transpose(1, 2)  # [B, Sq, H]
    assert (got["o"].reshape(B, Sq, H, D)[gone] == 0).all() and (got["dq"].reshape(B, Sq, H, D)[gone] == 0).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("B,H,Hk,Sq,Sk,D", [(2, 2, 2, 70, 1300, 128), (1, 4, 2, 1200, 65, 64), (2, 2, 1, 33, 40, 96)])
def test_the_widest_bias(ops, dtype, B, H, Hk, Sq, Sk, D):
    q, k, v, do = make(B, H, Hk, Sq, Sk, D, dtype, seed=Sq, scale_q=D ** -0.5)
    buckets = (torch.arange(1025, dtype=torch.int32) * 7 % 1024).cuda()  # every distance another bucket, but for the ends'
    table = (torch.randn(1024, H, generator=torch.Generator().manual_seed(5)) * 0.7).to(DT[dtype]).cuda()
    kw = dict(masks("count", B, Sk), scale=1.0, rel_bias=(table, buckets))
    got, _ = run(ops, q, k, v, do, H, Hk, **kw)
    val, tol = reference(q, k, v, do, H, Hk, dtype, **kw)
    compare(got, val, tol)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("Sq", [1, 40, 200])
def test_what_lies_at_invisible_keys_is_never_used(ops, dtype, Sq):
    B, H, Sk, D = 3, 2, 300, 64
    q, k, v, do = make(B, H, H, Sq, Sk, D, dtype, seed=5)
    count = torch.tensor([300, 77, 0], dtype=torch.int32).cuda()
    mask = torch.ones(B, Sk, dtype=torch.int32).cuda()
    mask[:, 10:20] = 0
    clean = run(ops, q, k, v, do, H, H, key_mask=mask, key_count=count)
    hidden = (mask == 0) | (torch.arange(Sk).cuda()[None] >= count[:, None])
    for x, bad in ((k, float("nan")), (v, float("inf")), (k, -float("inf")), (v, torch.finfo(DT[dtype]).min), (k, torch.finfo(DT[dtype]).max)):
        x[hidden] = bad
        got = run(ops, q, k, v, do, H, H, key_mask=mask, key_count=count)
        for n in clean[0]:
            assert torch.equal(clean[0][n], got[0][n]), (n, bad)
        assert torch.equal(clean[1], got[1])
        assert (got[0]["dk"][hidden] == 0).all() and (got[0]["dv"][hidden] == 0).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_views_of_fused_projections(ops, dtype):
    B, H, Sq, Sk, D = 2, 3, 70, 110, 64
    g = torch.Generator().manual_seed(2)
    W = H * D
    qkv = torch.randn(B, Sq, 3 * W, generator=g).to(DT[dtype]).cuda()
    kv = torch.randn(B, Sk + 7, 2 * W + 64, generator=g).to(DT[dtype]).cuda()[:, 3: 3 + Sk]
    do = torch.randn(Sq, B, W, generator=g).to(DT[dtype]).cuda().transpose(0, 1)  # rows of the dialogs interleaved
    q, k, v = qkv[:, :, W: 2 * W], kv[:, :, :W], kv[:, :, W + 64:]
    plain, _ = run(ops, q.contiguous(), k.contiguous(), v.contiguous(), do.contiguous(), H, H)
    got, saved = run(ops, q, k, v, do, H, H)
    for n in plain:
        assert torch.equal(plain[n], got[n])
    o, saved = ops.cross_attention(q, k, v, H, need_grad=True, out=torch.empty_like(qkv)[:, :, :W])
    dq3, dkv = torch.full_like(qkv, 7.0), torch.full((B, Sk, 2 * W), 7.0, dtype=DT[dtype], device="cuda")
    ops.cross_attention_backward(q, k, v, o, saved, do, H, out=(dq3[:, :, :W], dkv[:, :, :W], dkv[:, :, W:]))
    assert torch.equal(dq3[:, :, :W], plain["dq"]) and torch.equal(dkv, torch.cat([plain["dk"], plain["dv"]], 2)) and (dq3[:, :, W:] == 7).all()
    # one encoder state shared by the whole batch: a broadcast view
    one = ops.cross_attention(q, k[:1].expand(B, Sk, W), v[:1].expand(B, Sk, W), H)
    assert torch.equal(one, ops.cross_attention(q, k[:1].repeat(B, 1, 1), v[:1].repeat(B, 1, 1), H))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("Sq,Sk,Hk,bias", [(65, 130, 2, False), (1, 300, 4, False), (50, 99, 4, True)])
def test_dropout_is_the_training_attentions_mask(ops, dtype, Sq, Sk, Hk, bias):
    from oracle.philox import philox4x32_10

    import numpy as np

    B, H, D, p, seed, offset = 2, 4, 32, 0.3, 1234567, 5 << 34
    q, k, v, do = make(B, H, Hk, Sq, Sk, D, dtype, seed=9)
    G4 = (Sk + 3) // 4
    ctr = np.arange(B * H * Sq * G4, dtype=np.uint64) + np.uint64(offset)
    ctr = np.stack([ctr & np.uint64(0xFFFFFFFF), ctr >> np.uint64(32), ctr * 0, ctr * 0], 1).astype(np.uint32)
    words = philox4x32_10(ctr, np.array([seed & 0xFFFFFFFF, seed >> 32], np.uint32))
    words = torch.from_numpy(words.astype(np.int64)).reshape(B, H, Sq, G4 * 4)[..., :Sk]
    keep = (words >= int(np.float32(p) * np.float32(2.0 ** 32))).double().cuda() / (1 - float(np.float32(p)))
    kw = dict(drop_p=p, seed=seed, offset=offset)
    ref = {}
    if bias:
        table = torch.randn(32, H, generator=torch.Generator().manual_seed(3)).to(DT[dtype]).cuda()
        ref["rel_bias"] = kw["rel_bias"] = (table, ops.relative_buckets())
    got, _ = run(ops, q, k, v, do, H, Hk, **kw)
    val, tol = reference(q, k, v, do, H, Hk, dtype, keep=keep, **ref)
    compare(got, val, tol)


def test_gradients_against_differences(ops):
    """Central differences of sum(o w) in fp64 arithmetic of the forward's fp32 outputs: step 2^-7 along random directions."""
    B, H, Sq, Sk, D = 2, 2, 30, 45, 32
    q, k, v, w = make(B, H, H, Sq, Sk, D, "fp32", seed=21)
    table = (torch.randn(16, H, generator=torch.Generator().manual_seed(4)) * 0.5).cuda()
    buckets = ops.relative_buckets(16, 24)
    f = lambda q, k, v, t: float((ops.cross_attention(q, k, v, H, rel_bias=(t, buckets)).double() * w.double()).sum())  # noqa: E731
    o, saved = ops.cross_attention(q, k, v, H, rel_bias=(table, buckets), need_grad=True)
    grads = ops.cross_attention_backward(q, k, v, o, saved, w, H, rel_bias=(table, buckets))
    h = 2.0 ** -7
    for n, (x, g) in enumerate(zip((q, k, v, table), grads)):
        d = torch.randn(x.shape, generator=torch.Generator().manual_seed(n)).cuda()
        d = d / d.norm()
        at = lambda s: f(*[(y + s * h * d) if m == n else y for m, y in enumerate((q, k, v, table))])  # noqa: E731
        # third-order rest of a five-point rule, fp32 outputs: |w|_1 2^-22 / h
        num = (8 * (at(1) - at(-1)) - (at(2) - at(-2))) / (12 * h)
        assert abs(num - float((g.double() * d.double()).sum())) < float(w.abs().sum()) * 2.0 ** -22 / h * 2, n


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("B,H,Hk,Sq,Sk,D,causal", [(4, 16, 4, 495, 29, 80, False), (53, 12, 12, 19, 329, 32, True), (13, 6, 6, 31, 31, 64, True), (4, 8, 8, 57, 5, 40, False),
                                                   (16, 32, 16, 470, 380, 16, False)])
def test_query_and_key_gradients_lose_two_roundings(ops, dtype, B, H, Hk, Sq, Sk, D, causal):
    """The score gradients are rounded once and so are the results, independently and alike: sqrt(2) of the error that rounding the exact
    gradients makes, 1.5 with room for D = do . o."""
    q, k, v, do = make(B, H, Hk, Sq, Sk, D, dtype, seed=Sk)
    got, _ = run(ops, q, k, v, do, H, Hk, causal=causal)
    val, _ = reference(q, k, v, do, H, Hk, dtype, causal=causal)
    for name in ("dq", "dk"):
        want = val[name]
        once = (want.to(DT[dtype]).double() - want).norm()
        assert float((got[name].double() - want).norm() / once) <= 1.5, name


def test_bucket_rule_matches_the_encoder(ops):
    for nb, md in ((32, 128), (64, 256), (16, 64)):
        rel = torch.arange(-md - 40, md + 41)
        side, exact = nb // 2, nb // 4
        rp = rel.abs()
        large = exact + (torch.log(rp.float() / exact) / math.log(md / exact) * (side - exact)).to(torch.long)
        large = torch.min(large, torch.full_like(large, side - 1))
        want = (rel > 0).long() * side + torch.where(rp < exact, rp, large)
        got = ops.relative_buckets(nb, md).cpu().long()[rel.clamp(-md, md) + md]
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("B,H,Sq,Sk,q_start,bidirectional", [(1, 12, 64, 64, 0, True), (1, 1, 1, 1, 0, True), (2, 3, 77, 301, 0, False), (1, 2, 1, 1000, 999, False),
                                                             (3, 2, 500, 33, 7, True), (1, 5, 130, 7, 0, True), (1, 3, 64, 448, 7, True), (1, 3, 65, 64, 0, False), (1, 4, 400, 5, 3, False), (1, 2, 300, 1023, 723, True)])
def test_dense_bias_and_its_gradient(ops, dtype, B, H, Sq, Sk, q_start, bidirectional):
    g = torch.Generator().manual_seed(Sq)
    table = torch.randn(32, H, generator=g).to(DT[dtype]).cuda()
    buckets = ops.relative_buckets(32, 128, bidirectional)
    bucket = bucket_of(buckets, Sq, Sk, q_start)
    assert torch.equal(ops.relative_bias(table, buckets, Sq, Sk, q_start=q_start), table[bucket].permute(2, 0, 1))
    d = torch.randn(B, H, Sq, Sk, generator=g).to(DT[dtype]).cuda()
    hot = torch.nn.functional.one_hot(bucket, 32).double().reshape(Sq * Sk, 32)
    by = lambda x: (x.double().sum(0).reshape(H, Sq * Sk) @ hot).t()  # noqa: E731
    got = ops.relative_bias_backward(d if B > 1 else d[0], buckets, 32, q_start=q_start)
    tol = by(d.abs()) * (B * Sq + 16) * 2.0 ** -24 + U[dtype] * by(d).abs() + SUB[dtype]
    assert ((got.double() - by(d)).abs() <= tol).all()
    assert torch.equal(got, ops.relative_bias_backward(d if B > 1 else d[0], buckets, 32, q_start=q_start))


def test_a_bucket_outside_the_table_is_nan_and_collects_nothing(ops):
    table = torch.randn(8, 2, device="cuda")
    buckets = ops.relative_buckets(8, 16)
    buckets[16 + 3], buckets[16 - 2] = 8, -1
    bias = ops.relative_bias(table, buckets, 20, 20)
    rel = torch.arange(20)[None] - torch.arange(20)[:, None]
    assert torch.equal(torch.isnan(bias).any(0).cpu(), (rel == 3) | (rel == -2))
    d = torch.ones(2, 20, 20, device="cuda")
    got = ops.relative_bias_backward(d, buckets, 8)
    assert float(got.sum()) == 2 * (400 - 17 - 18)


def test_results_over_operands_are_refused(ops):
    q, k, v, do = make(1, 2, 2, 8, 8, 32, "bf16")
    with pytest.raises(ValueError):
        ops.cross_attention(q, k, v, 2, out=q)
    o, saved = ops.cross_attention(q, k, v, 2, need_grad=True)
    fresh = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    for x in (q, k, v, o, do):
        for n in range(3):
            with pytest.raises(ValueError):
                ops.cross_attention_backward(q, k, v, o, saved, do, 2, out=fresh[:n] + (x,) + fresh[n + 1:])


def test_lengths_of_zero(ops):
    q, k, v, do = make(2, 2, 2, 5, 9, 32, "bf16")
    none = torch.zeros(2, 0, 64, dtype=torch.bfloat16, device="cuda")
    o, saved = ops.cross_attention(q, none, none, 2, need_grad=True)
    assert (o == 0).all() and torch.isinf(saved[0]).all()
    dq, dk, dv = ops.cross_attention_backward(q, none, none, o, saved, do, 2)
    assert (dq == 0).all() and dk.shape == dv.shape == (2, 0, 64)
    rel = (torch.randn(32, 2, device="cuda").bfloat16(), ops.relative_buckets())
    o, saved = ops.cross_attention(none, k, v, 2, need_grad=True, rel_bias=rel)
    dq, dk, dv, dt = ops.cross_attention_backward(none, k, v, o, saved, none, 2, rel_bias=rel)
    assert o.shape == dq.shape == (2, 0, 64) and (dk == 0).all() and (dv == 0).all() and (dt == 0).all()
    assert ops.cross_attention(q[:0], k[:0], v[:0], 2).shape == (0, 5, 64)
    assert ops.relative_bias(rel[0], rel[1], 0, 5).shape == (2, 0, 5)
    assert (ops.relative_bias_backward(torch.zeros(2, 0, 5, device="cuda"), rel[1], 32) == 0).all()


def test_other_streams_and_graphs(ops):
    """Two calls on two streams at once, and a captured forward + backward replayed on new inputs between eager calls."""
    B, H, Sq, Sk, D = 2, 4, 90, 700, 64
    rel = (torch.randn(32, H, device="cuda").half(), ops.relative_buckets())
    count = torch.tensor([700, 311], dtype=torch.int32, device="cuda")
    sets = [make(B, H, H, Sq, Sk, D, "fp16", seed=s) for s in range(4)]
    kw = dict(rel_bias=rel, key_count=count)
    eager = [run(ops, *x, H, H, **kw)[0] for x in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for n in range(8):
        with torch.cuda.stream(streams[n % 2]):
            got.append(run(ops, *sets[n % 4], H, H, **kw)[0])
    torch.cuda.synchronize()
    for n, x in enumerate(got):
        for name in x:
            assert torch.equal(x[name], eager[n % 4][name])
    static = [t.clone() for t in sets[0]]
    graphs = []
    for _ in range(2):  # two graphs, replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o, saved = ops.cross_attention(*static[:3], H, need_grad=True, **kw)
            res = ops.cross_attention_backward(*static[:3], o, saved, static[3], H, **kw)
        graphs.append((g, dict(zip(("dq", "dk", "dv", "dtable"), res), o=o)))
    for n in range(6):
        for a, b in zip(static, sets[n % 4]):
            a.copy_(b)
        g, out = graphs[n % 2]
        g.replay()
        ops.cross_attention(*sets[3][:3], H)  # the program's own work between the replays
        torch.cuda.synchronize()
        for name in out:
            assert torch.equal(out[name], eager[n % 4][name]), (n, name)
