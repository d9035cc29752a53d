"""The block around the experts where its own tests do not reach: the training command with its switches, decoding without a choice between experts."""
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from streamep_b200.models.moe_layer import make_buffer
from streamep_b200.models.moe_lm import ExpertAdamW, MoELM

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("switches", [["--mixer", "--train-router"], ["--mixer"], ["--train-router"]])
def test_the_training_command(native, switches):
    out = subprocess.run([sys.executable, "-m", "streamep_b200.stream_moe.train_lm", "--steps", "4", "--every", "2", "--tokens", "512", "--hidden", "128",
                          "--ffn", "64", "--vocab", "500", *switches], capture_output=True, text=True, timeout=300, cwd=Path(__file__).resolve().parent.parent)
    assert "Traceback" not in out.stderr, out.stderr[-2000:]
    assert "step 0: loss" in out.stdout and "train_lm: world=1 tokens/rank=512 vocab=500" in out.stdout and "nan" not in out.stdout


@pytest.mark.parametrize("tokens", [384, 200])
def test_a_run_with_sequences_of_128_or_one(native, tokens):
    from streamep_b200.stream_moe.train_lm import train
    buf = make_buffer(None, tokens, 128, 2, 8, layers_in_flight=1, world_size=1)
    model = MoELM(300, 128, 64, 8, 2, 1, buf, device=DEV, mixer=True, train_router=True)
    opt = ExpertAdamW(model.replicated_parameters(), model.expert_parameters(), lr=1e-3)
    losses = train(model, opt, 3, tokens, 300, DEV, seed=2)
    buf.check_status()
    assert len(losses) == 3 and all(v == v and v < float("inf") for v in losses)
    assert all(p.grad is not None and bool(p.grad.isfinite().all()) for p in opt.params)


def test_every_token_is_decoded_where_all_experts_are_chosen(native):
    """No token can be routed otherwise, so rounding is all that decoding and the whole sequence differ by: a logit is a sum of 128 products of a normalised
    row and weights of 0.02 (0.23 of standard deviation), behind a chain of about 25 roundings of up to 2^-8 of values of size one: 25 2^-8 0.23 = 0.022 if all go one
    way for an entry of one deviation, 0.1 for one of four."""
    buf = make_buffer(None, 256, 128, 4, 4, layers_in_flight=2, world_size=1)
    model = MoELM(500, 128, 64, 4, 4, 2, buf, device=DEV, mixer=True, train_router=True)
    g = torch.Generator(device=DEV).manual_seed(0)
    tokens = torch.randint(0, 500, (3, 60), generator=g, device=DEV)
    with torch.no_grad():
        whole = (model.hidden_states(tokens) @ model.head.t()).view(3, 60, -1).float()
    states = model.states(3)
    rows = torch.stack([model.step(tokens[:, t], states) for t in range(60)], 1).float()
    buf.check_status()
    assert float((rows - whole).abs().max()) <= 0.1


def test_steps_are_refused_without_mixers(native):
    buf = make_buffer(None, 64, 128, 2, 4, layers_in_flight=1, world_size=1)
    model = MoELM(100, 128, 64, 4, 2, 1, buf, device=DEV)
    with pytest.raises(RuntimeError, match="mixers"):
        model.step(torch.zeros(3, dtype=torch.int64, device=DEV), model.states(3))


@pytest.mark.parametrize("before", ["differentiated", "not differentiated", "taken"])
def test_a_step_is_captured_behind_forwards_whose_losses_nobody_took(native, before):
    """A sum or per-token losses leave the routers' losses to the program; what they hold of the graph must not meet the captured one."""
    buf = make_buffer(None, 256, 128, 2, 8, layers_in_flight=2, world_size=1)
    model = MoELM(500, 128, 64, 8, 2, 2, buf, device=DEV, mixer=True, train_router=True)
    g = torch.Generator(device=DEV).manual_seed(0)
    x, y = (torch.randint(0, 500, (2, 128), generator=g, device=DEV) for _ in range(2))
    for _ in range(2):
        loss = model(x, y, reduction="sum")
        if before != "not differentiated":
            (loss + model.router_losses() if before == "taken" else loss).backward()
        model.zero_grad(set_to_none=True)
        del loss
    want = model(x, y)
    want.backward()
    eager = [want.detach()] + [p.grad for p in model.parameters()]
    model.zero_grad(set_to_none=True)
    del want
    model(x, y, reduction="sum")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = model(x, y)
        loss.backward()
    graph.replay()
    buf.check_status()
    # (the layer adds its experts' rows in bf16, in an order of its own)
    torch.testing.assert_close(loss.detach(), eager[0], rtol=0.01, atol=0.0)
    for (n, p), e in zip(model.named_parameters(), eager[1:]):
        a, b = p.grad.float(), e.float()
        assert float((a - b).norm()) <= 0.05 * float(b.norm()) + 1e-7, n
