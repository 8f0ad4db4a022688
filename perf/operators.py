"""Cases of the attention to an encoder's states of another length and of the learned relative position bias.

Three kinds of pass:
  "attend"  the forward attention as serving calls it: queries [B, Sq, heads D] over an encoder's states [B, Sk, kv_heads D] of
            another length, with right padding ("count"), an arbitrary key mask ("mask"), a causal limit, or a bucketed relative bias;
  "train"   the same forward and its backward: the output and the gradients of queries, keys, values (and of the bias table);
  "bias"    the dense relative position bias of a bucket table [buckets, heads] and the table's gradient from a dense gradient.

``own`` False: ``run`` is the plain form (elementary torch operations in 32 bits, sums that are long in 64); True: the calls a user
makes of ``didi_amd.ops``.  ``exact`` is the definition in 64 bits.
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _attend(name, kind, dtype, B, heads, kv_heads, D, Sq, Sk, mask="none", causal=False, q_start=0, bias=False, buckets=32, max_distance=128,
            bidirectional=True):
    c = {"kind": kind, "dtype": dtype, "B": B, "heads": heads, "kv_heads": kv_heads, "D": D, "Sq": Sq, "Sk": Sk, "mask": mask, "causal": causal,
         "q_start": q_start, "bias": bias, "buckets": buckets, "max_distance": max_distance, "bidirectional": bidirectional}
    return dict(c, name=name) if name else c


def _bias(name, dtype, heads, Sq, Sk, buckets, max_distance, bidirectional, q_start=0):
    c = {"kind": "bias", "dtype": dtype, "heads": heads, "Sq": Sq, "Sk": Sk, "buckets": buckets, "max_distance": max_distance,
         "bidirectional": bidirectional, "q_start": q_start}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one reply position against one short context: the smallest call, all latency
        _attend("attend one token short", "attend", "bf16", 1, 12, 12, 64, 1, 64),
        # a served batch of single positions over long contexts of different lengths, one row of the batch padded away entirely
        _attend("attend one token ragged", "attend", "fp16", 32, 12, 12, 64, 1, 4096, mask="count"),
        # few rows over a very long context, keys and values shared by four heads: work has to be split over the keys
        _attend("attend one token long", "attend", "bf16", 4, 32, 8, 128, 1, 33001),
        # a denoiser call: 63 reply positions of each dialog against contexts of up to 512 tokens
        _attend("attend replies", "attend", "fp16", 64, 12, 12, 64, 63, 512, mask="count"),
        # the context encoder's own attention in 32 bits, 1280 wide with 32 heads, masked
        _attend("attend encoder fp32", "attend", "fp32", 16, 32, 32, 40, 127, 127, mask="mask"),
        # an encoder layer with the learned relative bias on the scores (its scale is folded into the weights)
        _attend("attend encoder bias", "attend", "bf16", 16, 12, 12, 64, 512, 512, mask="count", bias=True),
        # training, odd lengths, 80-wide heads, keys and values shared by two heads, holes in the mask
        _attend("train odd", "train", "fp16", 3, 10, 5, 80, 251, 777, mask="mask"),
        # training in the trainer's own type, causal with a bias that looks back only
        _attend("train causal fp32", "train", "fp32", 8, 12, 12, 64, 128, 128, causal=True, bias=True, bidirectional=False),
        # an encoder layer's training step with the bias table's gradient
        _attend("train encoder bias", "train", "bf16", 8, 12, 12, 64, 512, 512, mask="count", bias=True),
        # the largest: long replies against long documents
        _attend("train long", "train", "bf16", 2, 16, 16, 128, 2048, 8192, mask="count"),
        # the dense bias of a 64-token context, and its gradient
        _bias("bias short", "fp32", 12, 64, 64, 32, 128, True),
        # the dense bias of long sequences in 16 bits, looking back only, an odd width
        _bias("bias long", "bf16", 32, 2048, 2047, 64, 256, False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


MOST_PAIRS = 2 * 16 * 2048 * 8192  # score elements of the largest listed case
MOST_KEYS = 4 * 33001 * 8 * 128    # key elements of the longest listed one


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "train", "train", "bias"])
    dtype = rng.choice(["bf16", "fp16", "fp32"])
    buckets, max_distance = rng.choice([(32, 128), (32, 128), (64, 256), (16, 64)])
    bidirectional = rng.random() < 0.6
    if kind == "bias":
        heads = rng.choice([1, 4, 6, 12, 16, 32])
        Sq, Sk = _log(rng, 1, 2048), _log(rng, 1, 2048)
        return _bias(None, dtype, heads, Sq, Sk, buckets, max_distance, bidirectional, rng.choice([0, 0, Sk - 1 if Sq == 1 else 0]))
    kv_heads = rng.choice([1, 2, 4, 6, 8, 12, 16])
    group = rng.choice([1, 1, 1, 2, 4])
    D = rng.choice([16, 32, 40, 64, 64, 64, 80, 96, 128])
    if kind == "attend" and rng.random() < 0.5:
        Sq, Sk = rng.choice([1, 1, 1, 2, 4, 7]), _log(rng, 1, 33001)
    elif kind == "attend":
        Sq, Sk = _log(rng, 1, 2048), _log(rng, 1, 8192)
    else:  # with a key or two the gradients of the scores cancel to nothing: there is no value to compare
        Sq, Sk = _log(rng, 16, 2048), _log(rng, 16, 8192)
    causal = rng.random() < 0.25
    q_start = 0
    if causal:
        Sk = max(Sq, Sk)
        q_start = rng.choice([0, Sk - Sq])
    B = _log(rng, 1, 64)
    heads = kv_heads * group
    pairs = MOST_PAIRS // (4 if kind == "train" and dtype == "fp32" else 1)
    while B > 1 and (B * heads * Sq * Sk > pairs or B * kv_heads * Sk * D > MOST_KEYS or B * heads * Sq * D > MOST_KEYS):
        B //= 2
    while heads * Sq * Sk > pairs:
        Sq = (Sq + 1) // 2
    mask = rng.choice(["none", "count", "mask"])
    bias = heads <= 32 and rng.random() < 0.3
    return _attend(None, kind, dtype, B, heads, kv_heads, D, Sq, Sk, mask, causal, q_start, bias, buckets, max_distance, bidirectional)


def _edges(case):
    """Smallest distance of every logarithmic bucket after the exact ones, by whole-number arithmetic: bucket exact + k starts where
    distance ** n * exact ** k >= exact ** n * max_distance ** k, n = number of logarithmic buckets."""
    nb = case["buckets"] // 2 if case["bidirectional"] else case["buckets"]
    exact_ = nb // 2
    n, d, edges = nb - exact_, exact_, []
    while len(edges) < n - 1:
        k = len(edges) + 1
        while d ** n * exact_ ** k < exact_ ** n * case["max_distance"] ** k:
            d += 1
        edges.append(d)
    return nb, exact_, edges


def _plan(case):
    """int32 [2 max_distance + 1]: the bucket of every distance key - query from -max_distance to max_distance; farther ones share
    the buckets at its ends.  A model keeps it beside the table."""
    nb, exact_, edges = _edges(case)
    distance = torch.arange(-case["max_distance"], case["max_distance"] + 1)
    far = distance.abs() if case["bidirectional"] else (-distance).clamp_min(0)
    b = torch.where(far < exact_, far, exact_ + torch.bucketize(far, torch.tensor(edges), right=True))
    return (b + (distance > 0) * nb if case["bidirectional"] else b).to(torch.int32)


def _lengths(case):
    """Visible keys of each dialog under the padding of "count" and "mask": spread over the range by the case alone, the last row
    of a batch of three and more with none at all."""
    B, Sk = case["B"], case["Sk"]
    if case["mask"] == "none":
        return [Sk] * B
    got = [max(1, Sk - (b * 7919) % B * Sk // (B + 1)) for b in range(B)]
    if B >= 3:
        got[-1] = 0
    return got


def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = TYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device=dev) * scale).to(dt)

    s = {"case": case}
    if case["kind"] == "bias" or case["bias"]:
        s["table"] = normal(case["buckets"], case["heads"], scale=0.5)
        s["plan"] = _plan(case).to(dev)
    if case["kind"] == "bias":
        s["dbias"] = normal(case["heads"], case["Sq"], case["Sk"])
        return s
    B, Sq, Sk, D = case["B"], case["Sq"], case["Sk"], case["D"]
    # with the bias the scores are not scaled again: such a model's query weights are initialised D^-1/2 smaller
    s["q"] = normal(B, Sq, case["heads"] * D, scale=D ** -0.5 if case["bias"] else 1.0)
    s["k"], s["v"] = normal(B, Sk, case["kv_heads"] * D), normal(B, Sk, case["kv_heads"] * D)
    if case["kind"] == "train":
        s["do"] = normal(B, Sq, case["heads"] * D)
    s["count"] = s["mask"] = None
    if case["mask"] != "none":
        count = torch.tensor(_lengths(case), dtype=torch.int32, device=dev)
        if case["mask"] == "count":
            s["count"] = count
        else:
            keep = torch.rand(B, Sk, generator=g, device=dev) < 0.9
            keep[:, 0] = True
            s["mask"] = (keep & (torch.arange(Sk, device=dev)[None] < count[:, None])).to(torch.int32)
    return s


def _scale(case):
    return 1.0 if case["bias"] else 1.0 / math.sqrt(case["D"])


# ------------------------------------------------------------------ the plain form
def _bucket(case, s, distance):
    """Bucket of every key position minus query position."""
    return s["plan"][distance.clamp(-case["max_distance"], case["max_distance"]) + case["max_distance"]].long()


def _dense_bias(case, s, table):
    i = torch.arange(case["Sq"], device=table.device)[:, None] + case["q_start"]
    j = torch.arange(case["Sk"], device=table.device)[None]
    return table[_bucket(case, s, j - i)].permute(2, 0, 1)


def _table_gradient(case, s, d):
    """d fp32 [heads, Sq, Sk] -> [buckets, heads]: sums along the diagonals (rows shifted against each other by one), then by bucket."""
    H, Sq, Sk = d.shape
    W = Sk + Sq
    x = torch.nn.functional.pad(d.flip(1), (0, Sq)).reshape(H, Sq * W)[:, : Sq * (W - 1)].reshape(H, Sq, W - 1)
    diagonal = x.sum(1, dtype=torch.float64)
    distance = torch.arange(Sq + Sk - 1, device=d.device) - (Sq - 1) - case["q_start"]
    hot = torch.nn.functional.one_hot(_bucket(case, s, distance), case["buckets"]).to(torch.float64)
    return (diagonal @ hot).t()


def _visible(case, s):
    B, Sq, Sk = case["B"], case["Sq"], case["Sk"]
    dev = s["q"].device
    j = torch.arange(Sk, device=dev)
    see = torch.ones(B, 1, 1, 1, Sk, dtype=torch.bool, device=dev)
    if s["count"] is not None:
        see = see & (j < s["count"][:, None])[:, None, None, None]
    if s["mask"] is not None:
        see = see & (s["mask"] != 0)[:, None, None, None]
    if case["causal"]:
        i = torch.arange(Sq, device=dev)[:, None] + case["q_start"]
        see = see & (j[None] <= i)[None, None, None]
    return see


def _heads(x, n, D):
    """[B, S, n D] -> fp32 [B, n, S, D]"""
    return x.float().reshape(x.shape[0], x.shape[1], n, D).transpose(1, 2)


def _rows(x, like):
    """[B, kv, group, S, D] or [B, kv, S, D] -> [B, S, heads D] in the inputs' type"""
    B, S, D = x.shape[0], x.shape[-2], x.shape[-1]
    return x.reshape(B, -1, S, D).transpose(1, 2).reshape(B, S, -1).to(like.dtype)


def _plain_forward(case, s):
    B, Sq, Sk, D, Hk = case["B"], case["Sq"], case["Sk"], case["D"], case["kv_heads"]
    G = case["heads"] // Hk
    q = _heads(s["q"], case["heads"], D).reshape(B, Hk, G * Sq, D)
    k, v = _heads(s["k"], Hk, D).contiguous(), _heads(s["v"], Hk, D).contiguous()
    x = (torch.matmul(q, k.transpose(-1, -2)) * _scale(case)).reshape(B, Hk, G, Sq, Sk)
    if case["bias"]:
        x += _dense_bias(case, s, s["table"].float()).reshape(1, Hk, G, Sq, Sk)
    x = x.masked_fill_(~_visible(case, s), -math.inf)
    top = x.amax(-1, keepdim=True)
    x = torch.exp(x.sub_(torch.where(top == -math.inf, 0.0, top)))
    p = x / x.sum(-1, keepdim=True).clamp_min(1e-30)  # a row that sees no key: zeros
    o = torch.matmul(p.reshape(B, Hk, G * Sq, Sk), v)
    return q, k, v, p, o


def _plain(case, s):
    if case["kind"] == "bias":
        return {"bias": _dense_bias(case, s, s["table"]).contiguous(), "dtable": _table_gradient(case, s, s["dbias"].float()).to(s["dbias"].dtype)}
    B, Sq, Sk, D, Hk = case["B"], case["Sq"], case["Sk"], case["D"], case["kv_heads"]
    G = case["heads"] // Hk
    q, k, v, p, o = _plain_forward(case, s)
    out = {"o": _rows(o.reshape(B, Hk, G, Sq, D), s["q"])}
    if case["kind"] == "attend":
        return out
    p = p.reshape(B, Hk, G * Sq, Sk)
    do = _heads(s["do"], case["heads"], D).reshape(B, Hk, G * Sq, D)
    out["dv"] = _rows(torch.matmul(p.transpose(-1, -2), do), s["v"])
    ds = torch.matmul(do, v.transpose(-1, -2)).sub_((do * o).sum(-1, keepdim=True)).mul_(p)
    if case["bias"]:
        out["dtable"] = _table_gradient(case, s, ds.reshape(B, Hk * G, Sq, Sk).sum(0)).to(s["table"].dtype)
    out["dq"] = _rows((torch.matmul(ds, k) * _scale(case)).reshape(B, Hk, G, Sq, D), s["q"])
    out["dk"] = _rows(torch.matmul(ds.transpose(-1, -2), q) * _scale(case), s["k"])
    return out


# ------------------------------------------------------------------ the framework's calls
def _own(case, s):
    from didi_amd import ops

    if case["kind"] == "bias":
        return {"bias": ops.relative_bias(s["table"], s["plan"], case["Sq"], case["Sk"], q_start=case["q_start"]),
                "dtable": ops.relative_bias_backward(s["dbias"], s["plan"], case["buckets"], q_start=case["q_start"])}
    how = dict(kv_heads=case["kv_heads"], causal=case["causal"], q_start=case["q_start"], key_mask=s["mask"], key_count=s["count"],
               scale=_scale(case), rel_bias=(s["table"], s["plan"]) if case["bias"] else None)
    if case["kind"] == "attend":
        return {"o": ops.cross_attention(s["q"], s["k"], s["v"], case["heads"], **how)}
    o, saved = ops.cross_attention(s["q"], s["k"], s["v"], case["heads"], need_grad=True, **how)
    grads = ops.cross_attention_backward(s["q"], s["k"], s["v"], o, saved, s["do"], case["heads"], **how)
    return {"o": o, "dq": grads[0], "dk": grads[1], "dv": grads[2], **({"dtable": grads[3]} if case["bias"] else {})}


def run(state):
    return _own(state["case"], state) if own else _plain(state["case"], state)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "bias":
        n, t = case["heads"] * case["Sq"] * case["Sk"], case["buckets"] * case["heads"]
        return {"bytes": 2 * e * (n + t), "flops": n}
    B, H, Hk, D, Sq, Sk = case["B"], case["heads"], case["kv_heads"], case["D"], case["Sq"], case["Sk"]
    pairs = 0
    for n in _lengths(case):
        if case["causal"]:  # query i sees min(n, q_start + i + 1) keys
            full = max(0, min(Sq, n - case["q_start"] - 1))
            pairs += full * (case["q_start"] + 1) + full * (full - 1) // 2 + (Sq - full) * n
        else:
            pairs += Sq * n
    keys = sum(_lengths(case))
    rows = B * Sq * H * D * e
    fwd = 2 * rows + 2 * keys * Hk * D * e + (4 * B * Sk if case["mask"] == "mask" else 0)
    if case["kind"] == "attend":
        return {"bytes": fwd, "flops": 4 * pairs * H * D}
    return {"bytes": fwd + 2 * rows + 2 * B * Sk * Hk * D * e, "flops": 14 * pairs * H * D}


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    Sq, Sk = case["Sq"], case["Sk"]
    dev = "cuda"
    relative = torch.arange(Sk, device=dev)[None] - (torch.arange(Sq, device=dev)[:, None] + case["q_start"])
    nb, exact_, edges = _edges(case)
    if "table" in s:
        near = relative.abs() if case["bidirectional"] else torch.where(relative < 0, -relative, 0)
        bucket = near.clamp_max(exact_)
        for e in edges:
            bucket = bucket + (near >= e)
        if case["bidirectional"]:
            bucket = bucket + nb * (relative > 0)
        table = s["table"].double()

    def by_bucket(d):
        return torch.stack([d.masked_fill(bucket != b, 0.0).sum((-1, -2)) for b in range(case["buckets"])])

    if case["kind"] == "bias":
        return {"bias": torch.stack([table[:, h][bucket] for h in range(case["heads"])]),
                "dtable": torch.cat([by_bucket(s["dbias"][h: h + 1].double()) for h in range(case["heads"])], 1)}
    D, G = case["D"], case["heads"] // case["kv_heads"]
    train = case["kind"] == "train"
    out = {n: torch.zeros(s[m].shape, dtype=torch.float64, device=dev) for n, m in
           ([("o", "q")] + ([("dq", "q"), ("dk", "k"), ("dv", "v")] if train else []))}
    if train and case["bias"]:
        out["dtable"] = torch.zeros(case["buckets"], case["heads"], dtype=torch.float64, device=dev)
    if case["B"] * case["heads"] > 4096:
        return None
    for b in range(case["B"]):
        see = torch.ones(Sq, Sk, dtype=torch.bool, device=dev)
        if s["count"] is not None:
            see[:, int(s["count"][b]):] = False
        if s["mask"] is not None:
            see &= s["mask"][b][None] != 0
        if case["causal"]:
            see &= relative <= 0
        for h in range(case["heads"]):
            a, c = slice(h * D, (h + 1) * D), slice(h // G * D, (h // G + 1) * D)
            q, k, v = s["q"][b, :, a].double(), s["k"][b, :, c].double(), s["v"][b, :, c].double()
            x = q @ k.t() * _scale(case)
            if case["bias"]:
                x = x + table[:, h][bucket]
            x = torch.where(see, x, -math.inf)
            p = torch.nan_to_num(torch.softmax(x, -1), nan=0.0)  # no key to see: zeros
            out["o"][b, :, a] = p @ v
            if train:
                do = s["do"][b, :, a].double()
                dp = do @ v.t()
                ds = p * (dp - (p * dp).sum(-1, keepdim=True))
                out["dv"][b, :, c] += p.t() @ do
                out["dq"][b, :, a] = ds @ k * _scale(case)
                out["dk"][b, :, c] += ds.t() @ q * _scale(case)
                if case["bias"]:
                    out["dtable"][:, h] += by_bucket(ds)
    return out
