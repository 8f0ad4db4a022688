"""Dialogs past 96 tokens (heads of 128: past 84): the context encoders and the whole training step run their attention at any length.

Ground truth: the fp32 CPU oracle on the weights of the golden cases.  Bars as for the short cases of the same paths: context rel-L2 <= 1e-4,
x_0_hat 3e-5, gradients 2e-4 (bf16x3 products, fp32 attention)."""
import pytest
import torch

from golden_util import load_case, spec_to_config, weights_of

pytestmark = pytest.mark.gpu


def rel_l2(a, b):
    a, b = a.double().cpu(), b.double().cpu()
    return ((a - b).norm() / b.norm().clamp_min(1e-30)).item()


def _oracle_config(spec):
    from oracle.model import OracleConfig

    return OracleConfig(vocab=spec["vocab"], dec_dim=spec["dec_dim"], dec_layers=spec["dec_layers"], dec_heads=spec["dec_heads"], enc_kind=spec["enc_kind"],
                        enc_dim=spec["enc_dim"], enc_layers=spec["enc_layers"], enc_heads=spec["enc_heads"], diffusion_steps=spec["T"],
                        schedule=spec["schedule"], enc_ln_eps={"bert": 1e-12, "t5": 1e-6}.get(spec["enc_kind"], 1e-5))


def _dialogs(lens, width, vocab, seed):
    g = torch.Generator().manual_seed(seed)
    mask = (torch.arange(width)[None, :] < torch.tensor(lens)[:, None]).long()
    return torch.randint(3, vocab, (len(lens), width), generator=g) * mask, mask


@pytest.mark.parametrize("name,width", [("tiny_weights", 97), ("tiny_weights", 128), ("tiny_bbd80_ddpm_f2", 111), ("tiny_bertenc_ddpm_f2", 333),
                                        ("tiny_t5enc_ddpm_f2", 97), ("tiny_t5enc_ddpm_f2", 401), ("tiny_t5gated_euler_f3", 200), ("tiny_t5d128_ddpm_f2", 259),
                                        ("tiny_t5d128_ddpm_f2", 85), ("tiny_t5d128_ddpm_f2", 84)])
def test_context_encoder_past_96_tokens(name, width):
    from didi_amd.model import DiDiSampler
    from oracle.model import OracleDiDi

    t, meta = load_case(name)
    w, spec = weights_of(t), meta["spec"]
    model = DiDiSampler(w, spec_to_config(spec), device="cuda", precision="bf16x3")
    ids, mask = _dialogs([width, 1, width - 3, min(width, 96), 40], width, spec["vocab"], width)
    want = OracleDiDi(w, _oracle_config(spec)).encode_context(ids, mask)
    got = model._encode_context(ids.cuda(), mask.cuda())
    seen = mask.bool()  # padded positions are attended to by nobody
    assert rel_l2(got[seen.cuda()], want[seen]) <= 1e-4


@pytest.mark.parametrize("name", ["tiny_weights", "tiny_bertenc_ddpm_f2"])
def test_a_context_past_the_position_table_is_refused(name):
    from didi_amd.model import DiDiSampler

    t, meta = load_case(name)
    cfg = spec_to_config(meta["spec"])
    model = DiDiSampler(weights_of(t), cfg, device="cuda", precision="bf16x3")
    n = 1 + (128 if name == "tiny_weights" else 512)
    with pytest.raises(ValueError):
        model._encode_context(torch.ones((1, n), dtype=torch.int64, device="cuda"), torch.ones((1, n), dtype=torch.int64, device="cuda"))


def test_short_position_bias_is_the_gathered_table():
    from didi_amd.model import DiDiSampler
    from oracle.transformer import t5_position_bias

    t, meta = load_case("tiny_t5enc_ddpm_f2")
    w = weights_of(t)
    model = DiDiSampler(w, spec_to_config(meta["spec"]), device="cuda", precision="bf16x3")
    table = next(v for k, v in w.items() if k.endswith("relative_attention_bias.weight")).float()
    for c in (1, 2, 23, 96):
        assert torch.equal(model._t5_position_bias(c).cpu().view(-1, c, c), t5_position_bias(table, c, c).reshape(-1, c, c))


def _step(name, S, width, anchor=False, **kw):
    from didi_amd.synthetic import RawContext
    from didi_amd.trainer import DiDiTrainer

    t, meta = load_case(name)
    w, spec = weights_of(t), meta["spec"]
    B = 3
    cids, cmask = _dialogs([width, width // 2, 2], width, spec["vocab"], S)
    ids, tmask = _dialogs([S, S - 5, 3], S, spec["vocab"], width)
    g = torch.Generator().manual_seed(S * width)
    draws = [torch.randn((B, S, spec["dec_dim"]), generator=g) for _ in range(3)]
    steps = torch.tensor([[1], [spec["T"] // 2], [spec["T"]]])
    kw.setdefault("hidden_dropout", 0.0)
    kw.setdefault("attention_dropout", 0.0)
    tr = DiDiTrainer(w, spec_to_config(spec), device="cuda", precision="bf16x3", anchor_loss=anchor, **kw)
    return w, spec, tr, RawContext(cids, cmask), RawContext(ids, tmask), draws, steps


@pytest.mark.parametrize("name,S,width", [("tiny_weights", 101, 113), ("tiny_weights", 160, 40), ("tiny_weights", 24, 128), ("tiny_t5enc_ddpm_f2", 130, 203)])
def test_training_step_past_96_tokens_vs_oracle_autograd(name, S, width):
    from oracle.training import training_step_with_grads

    w, spec, tr, ctx, tgt, draws, t = _step(name, S, width)
    ref, want = training_step_with_grads(w, _oracle_config(spec), ctx, tgt, draws, t)
    out = tr.forward_backward(ctx.to("cuda"), tgt.to("cuda"), draws=draws, t=t, keep=True)
    assert rel_l2(out["x_0_hat"], ref["x_0_hat"].detach()) <= 3e-5
    for k in ("mse", "ce", "t_T", "loss"):
        assert abs(float(out[k]) - float(ref[k].detach())) <= 1e-4 * max(abs(float(ref[k].detach())), 1e-9), k
    for k, v in want.items():
        got = out["grads"][k]
        if k.endswith(".key.bias"):  # analytically zero: rounding alone, measured against the query bias
            assert float(got.norm()) <= 1e-4 * float(want[k.replace(".key.", ".query.")].norm()), k
        else:
            assert rel_l2(got, v) <= 2e-4, (k, rel_l2(got, v))


def test_training_step_with_dropout_past_96_tokens():
    """One dropout seed: the same bits twice (but for the embedding table's, whose rows are summed by float atomics), and the loss's slope along the gradient is the gradient's norm (1 %; a mask of the backward that is
    not the forward's would be off by 10 %)."""
    _, _, tr, ctx, tgt, draws, t = _step("tiny_weights", 111, 125, hidden_dropout=0.1, attention_dropout=0.1)
    ctx, tgt = ctx.to("cuda"), tgt.to("cuda")
    kw = dict(draws=draws, t=t, dropout_seed=1234)
    a, b = tr.forward_backward(ctx, tgt, **kw), tr.forward_backward(ctx, tgt, **kw)
    other = [k for k in a["grads"] if not torch.equal(a["grads"][k], b["grads"][k])]
    assert float(a["loss"]) == float(b["loss"]) and not [k for k in other if k != "emb.weight"], other
    flat = tr.flatten_gradients(a["grads"])[: tr._n_flat]
    norm = float(flat.norm())
    theta, losses, eps = tr._flat_p.clone(), [], 0.02
    for sign in (1.0, -1.0):
        tr._flat_p.copy_(theta + sign * eps * flat / norm)
        tr.refresh_planes()
        losses.append(float(tr.forward_backward(ctx, tgt, **kw)["loss"].double()))
    assert abs((losses[0] - losses[1]) / (2 * eps) - norm) <= 0.01 * norm
