"""Dialogs whose context mask is all zeros: the reference's additive masks then average over all positions, in the encoders and in the decoder's cross
attention, whatever the width.  Ground truth and bars as for the other dialogs of the same paths."""
import pytest

from golden_util import load_case, spec_to_config, weights_of
from test_gpu_long_dialogs import _dialogs, _oracle_config, _step, rel_l2

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name,width", [("tiny_weights", 90), ("tiny_weights", 97), ("tiny_bbd80_ddpm_f2", 111), ("tiny_bertenc_ddpm_f2", 333), ("tiny_t5enc_ddpm_f2", 90),
                                        ("tiny_t5enc_ddpm_f2", 203), ("tiny_t5d128_ddpm_f2", 90)])
def test_context_of_an_empty_dialog(name, width):
    from didi_amd.model import DiDiSampler
    from oracle.model import OracleDiDi

    t, meta = load_case(name)
    w, spec = weights_of(t), meta["spec"]
    model = DiDiSampler(w, spec_to_config(spec), device="cuda", precision="bf16x3")
    ids, mask = _dialogs([width, 0, width - 3], width, spec["vocab"], width)
    want = OracleDiDi(w, _oracle_config(spec)).encode_context(ids, mask)
    got = model._encode_context(ids.cuda(), mask.cuda())
    for b in range(3):
        seen = slice(None) if b == 1 else mask[b].bool()  # the empty dialog's positions are all averaged over by the decoder
        assert rel_l2(got[b].cpu()[seen], want[b][seen]) <= 1e-4, b


@pytest.mark.parametrize("name,S,width", [("tiny_weights", 30, 40), ("tiny_weights", 101, 113), ("tiny_weights", 24, 128), ("tiny_t5enc_ddpm_f2", 40, 130)])
def test_training_step_with_an_empty_context(name, S, width):
    from oracle.training import training_step_with_grads

    w, spec, tr, ctx, tgt, draws, t = _step(name, S, width)
    ctx.attention_mask[1] = 0
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
