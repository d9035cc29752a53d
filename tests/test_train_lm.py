"""The operators around the layer, run together: a small MoE language model trains."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def build(tokens, vocab, seed=0):
    from streamep_b200.models import ExpertAdamW, MoELM, make_buffer
    buf = make_buffer(None, tokens, 128, 2, 4, layers_in_flight=2)
    model = MoELM(vocab, 128, 64, 4, 2, 2, buf, device=DEV, seed=seed)
    return model, ExpertAdamW(model.replicated_parameters(), model.expert_parameters(), lr=1e-2)


def test_loss_falls_and_tokens_can_be_scored(native):
    from streamep_b200.stream_moe.train_lm import batch, train
    vocab, tokens = 500, 1000
    model, opt = build(tokens, vocab)
    losses = train(model, opt, 40, tokens, vocab, DEV, seed=1)
    assert abs(losses[0] - math.log(vocab)) < 0.5 and losses[-1] < 0.5 * losses[0] and all(math.isfinite(v) for v in losses)
    model.buffer.check_status()
    x, y = batch(torch.Generator(device=DEV).manual_seed(9), vocab, tokens, DEV)
    lp = model.log_probs(x, y)
    one = model.log_probs(x[:1], y[:1])
    assert lp.shape == y.shape and (lp <= 0).all()
    # the layer adds its experts' rows in bf16, in an order of its own: hidden states may differ in their last places
    assert abs(float(one[0] - lp[0])) < 0.1


def test_step_against_torch(native):
    """One step's gradients through torch's clipping and AdamW on the master copies."""
    from streamep_b200.stream_moe.train_lm import batch
    model, opt = build(300, 700)
    x, y = batch(torch.Generator(device=DEV).manual_seed(2), 700, 300, DEV)
    model(x, y).backward()
    masters = [m.clone().requires_grad_(True) for m in opt.masters]
    for m, p in zip(masters, opt.params):
        m.grad = p.grad.float()
    ref = torch.optim.AdamW(masters, lr=opt.lr, betas=opt.betas, eps=opt.eps, weight_decay=opt.weight_decay)
    want = torch.nn.utils.clip_grad_norm_(masters, opt.max_norm)
    ref.step()
    norm = opt.step()
    assert abs(float(norm) - float(want)) <= 1e-5 * float(want)
    for got, w, p in zip(opt.masters, masters, opt.params):
        torch.testing.assert_close(got, w.detach(), rtol=1e-5, atol=2e-5 * opt.lr)
        assert torch.equal(p.detach(), got.to(torch.bfloat16))


def test_state_round_trip_and_skipped_step(native):
    from streamep_b200.stream_moe.train_lm import batch
    model, opt = build(300, 700)
    x, y = batch(torch.Generator(device=DEV).manual_seed(2), 700, 300, DEV)
    model(x, y).backward()
    opt.step()
    other_model, other = build(300, 700, seed=5)
    other.load_state_dict(opt.state_dict())
    assert all(torch.equal(a, b) for a, b in zip(model.parameters(), other_model.parameters()) if a.requires_grad)
    before = [p.detach().clone() for p in opt.params]
    opt.params[0].grad.fill_(float("inf"))
    assert math.isinf(float(opt.step()))
    assert all(torch.equal(a, b) for a, b in zip(opt.params, before))
