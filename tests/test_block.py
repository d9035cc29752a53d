"""The block around the experts as a model runs it: norms with the residual stream, the recurrence, the trained router, the experts, the loss,
the optimizer; its gradients against the same arithmetic in plain PyTorch, decoding against the whole sequence, packed against dense."""
import pytest
import torch

from streamep_b200.models.moe_layer import make_buffer
from streamep_b200.models.moe_lm import ExpertAdamW, MoELM

pytestmark = pytest.mark.gpu
DEV = "cuda"


def build(tokens=256, layers=2, **kw):
    buf = make_buffer(None, tokens, 128, 2, 8, layers_in_flight=layers, world_size=1)
    return MoELM(500, 128, 64, 8, 2, layers, buf, device=DEV, mixer=True, train_router=True, **kw), buf


def batch(B, T, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randint(0, 500, (B, T), generator=g, device=DEV), torch.randint(0, 500, (B, T), generator=g, device=DEV)


class Plain:
    """The model's forward in 32-bit PyTorch operations, on the same weights, with the experts chosen by the model itself."""

    def __init__(self, model):
        self.model = model
        self.p = {n: t.detach().float().requires_grad_(True) for n, t in model.named_parameters()}

    def norm(self, x, w=None, b=None):
        return torch.nn.functional.layer_norm(x, x.shape[-1:], w, b, 1e-5)

    def experts(self, i, y, idx):
        p, layer = self.p, self.model.layers[i]
        z = y @ p[f"layers.{i}.w_gate"].t()
        prob = torch.softmax(z, 1)
        w = prob.gather(1, idx)
        w = w / w.sum(1, keepdim=True)
        E = z.shape[1]
        counts = torch.bincount(idx.reshape(-1), minlength=E)
        balance = E * (counts / idx.numel() * prob.mean(0)).sum()
        zl = torch.logsumexp(z, 1).square().mean()
        out = torch.zeros_like(y)
        for e in range(E):
            t, k = (idx == e).nonzero(as_tuple=True)
            a = y[t] @ p[f"layers.{i}.w1"][e].t()
            h = torch.nn.functional.silu(a[:, 0::2]) * a[:, 1::2]
            out = out.index_add(0, t, w[t, k, None] * (h @ p[f"layers.{i}.w2"][e].t()))
        return out, balance, zl

    def loss(self, tokens, targets, routes):
        p, m = self.p, self.model
        B, T = tokens.shape
        x, aux = p["embedding"][tokens.reshape(-1)], 0.0
        for i in range(len(m.layers)):
            q = lambda n: p[f"mixers.{i}.{n}"]
            y = self.norm(x, q("norm_weight"), q("norm_bias"))
            v, g = (y @ q("w_in").t()).chunk(2, -1)
            keep = torch.sigmoid(g + q("gate_bias")).view(B, T, -1)
            v, h, rows = v.view(B, T, -1), 0.0, []
            for t in range(T):
                h = keep[:, t] * h + (1 - keep[:, t]) * v[:, t]
                rows.append(h)
            x = x + torch.stack(rows, 1).reshape(B * T, -1) @ q("w_out").t()
            out, balance, zl = self.experts(i, self.norm(x, q("expert_norm_weight"), q("expert_norm_bias")), routes[i])
            x = x + out
            aux = aux + m.balance_coef * balance + m.z_coef * zl
        logits = self.norm(x) @ p["head"].t()
        return torch.nn.functional.cross_entropy(logits, targets.reshape(-1)) + aux / len(m.layers)


def test_gradients_of_a_model(native):
    """bf16 activations against 32-bit ones: a chain of about 25 roundings (2^-9 each, rms, of values of size one) leads to each gradient, 25 2^-9 = 0.05 of
    its norm where they do not cancel; wrong terms show as errors of the order of one."""
    torch.manual_seed(0)
    model, buf = build()
    tokens, targets = batch(4, 64)
    loss = model(tokens, targets)
    loss.backward()
    buf.check_status()
    plain = Plain(model)
    want = plain.loss(tokens, targets, [layer.last_route.topk_idx for layer in model.layers])
    want.backward()
    assert abs(float(loss) - float(want)) < 0.02 * float(want)
    for n, p in model.named_parameters():
        assert p.grad is not None and p.grad.dtype == p.dtype, n
        a, b = p.grad.float(), plain.p[n].grad
        assert float((a - b).norm()) <= 0.08 * float(b.norm()) + 1e-7, (n, float((a - b).norm() / b.norm()))


def test_steps_of_a_run(native):
    model, buf = build(balance_coef=0.02)
    opt = ExpertAdamW(model.replicated_parameters(), model.expert_parameters(), lr=1e-3)
    assert len(opt.params) == len(list(model.parameters()))
    before = [p.detach().clone() for p in opt.params]
    for i in range(3):
        tokens, targets = batch(2, 128, seed=i)
        opt.zero_grad()
        model(tokens, targets).backward()
        norm = opt.step()
    buf.check_status()
    assert bool(torch.isfinite(norm)) and all(bool(p.isfinite().all()) for p in opt.params)
    assert all(not torch.equal(a, p) for a, p in zip(before, opt.params))
    for layer in model.layers:
        assert int(layer.last_route.expert_counts.sum()) == 2 * 256
        assert not layer.last_route.balance_loss.requires_grad and not layer.last_route.topk_weights.requires_grad      # no graph is kept
        with pytest.raises(RuntimeError, match="one forward"):
            layer.router_losses()
    with torch.no_grad():
        model(*batch(2, 128))
    assert all(layer.last_route is None for layer in model.layers)


def test_packed_is_dense(native):
    model, buf = build()
    tokens, targets = batch(2, 100)
    dense = model.log_probs(tokens, targets)
    flat, want = tokens.reshape(-1), dense.reshape(-1)
    cut = torch.tensor([0, 100, 200], dtype=torch.int32, device=DEV)
    packed = model.log_probs(flat, targets.reshape(-1), offsets=cut)
    # the recurrence alone may split time elsewhere: 2^-8 of activations of size one, a few times over, in logits of size one
    torch.testing.assert_close(packed, want, rtol=0.0, atol=0.1)
    # another cut is another model input: the second half of each sequence forgets the first
    other = model.log_probs(flat, targets.reshape(-1), offsets=torch.tensor([0, 50, 100, 150, 200], dtype=torch.int32, device=DEV))
    torch.testing.assert_close(other.view(2, 100)[:, :50], dense[:, :50], rtol=0.0, atol=0.1)
    assert float((other.view(2, 100)[:, 50:] - dense[:, 50:]).abs().max()) > 0.1
    buf.check_status()


def test_padding_of_a_packed_batch_is_not_counted(native):
    """Rows in front of the first sequence and behind the last one: counts are whole numbers, the losses those of the batch without them but for
    activations that the recurrence rounds elsewhere (2^-8 of values of size one, a few times over)."""
    model, buf = build()
    tokens, targets = batch(1, 150)
    tokens, targets = tokens.reshape(-1), targets.reshape(-1)
    model(tokens, targets, offsets=torch.tensor([0, 60, 150], device=DEV))
    routes = [layer.last_route for layer in model.layers]
    pad = lambda t, n, m, fill: torch.cat([t.new_full((n,), fill), t, t.new_full((m,), fill)])
    model(pad(tokens, 7, 43, 3), pad(targets, 7, 43, -100), offsets=torch.tensor([7, 67, 157], device=DEV))
    for layer, want in zip(model.layers, routes):
        got = layer.last_route
        assert int(got.expert_counts.sum()) == 150 * layer.top_k
        torch.testing.assert_close(got.z_loss, want.z_loss, rtol=0.02, atol=0.0)
        torch.testing.assert_close(got.balance_loss, want.balance_loss, rtol=0.02, atol=0.0)
    buf.check_status()


def test_decoding_continues(native):
    model, buf = build()
    tokens, _ = batch(3, 40)
    with torch.no_grad():
        whole = (model.hidden_states(tokens) @ model.head.t()).view(3, 40, -1).float()
    states = model.states(3)
    rows = torch.stack([model.step(tokens[:, t], states) for t in range(40)], 1).float()
    # a token whose two best experts are nearly alike may be routed otherwise where its activations differ by a rounding: few are
    off = (rows - whole).abs().amax(-1)
    assert float((off > 0.1).float().mean()) < 0.05
    buf.check_status()


def test_without_the_block_nothing_changes(native):
    buf = make_buffer(None, 256, 128, 2, 8, layers_in_flight=1, world_size=1)
    model = MoELM(500, 128, 64, 8, 2, 1, buf, device=DEV)
    assert not model.layers[0].w_gate.requires_grad and len(model.mixers) == 0
    tokens, targets = batch(1, 256)
    model(tokens, targets).backward()
    assert model.layers[0].w_gate.grad is None and model.layers[0].last_route is None
    assert {id(p) for p in model.replicated_parameters()} == {id(model.embedding), id(model.head)}


def test_a_run_of_the_operators_in_a_graph(native):
    """Forward and backward of the three operators together, captured: replays give what the eager calls give."""
    from streamep_b200.ops import balanced_router, gated_scan, layer_norm
    g = torch.Generator(device=DEV).manual_seed(3)
    x, r = (torch.randn(512, 128, generator=g, device=DEV).to(torch.bfloat16).requires_grad_(True) for _ in range(2))
    w = torch.ones(128, device=DEV, requires_grad=True)
    gate_w = torch.randn(16, 128, generator=g, device=DEV).to(torch.bfloat16).requires_grad_(True)
    up = torch.randn(512, 2, generator=g, device=DEV)

    def run():
        y, s = layer_norm(x, w, residual=r)
        h = gated_scan(y.view(4, 128, 128), s.view(4, 128, 128)).view(512, 128)
        route = balanced_router(h, gate_w, 2)
        return [h.detach(), route.balance_loss.detach()] + list(torch.autograd.grad([route.topk_weights, route.balance_loss], [x, r, w, gate_w], [up, torch.ones((), device=DEV)]))
    want = run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    for v in held:
        v.fill_(float("nan"))
    for _ in range(2):
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(held, want))
