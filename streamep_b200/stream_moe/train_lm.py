"""A short training run of a small MoE language model on synthetic data: every step is embedding, MoE layers, the loss over the
vocabulary, backward, norm, clipping and update (``streamep_b200.models.moe_lm``).

    python -m streamep_b200.stream_moe.train_lm --steps 50
    python -m torch.distributed.run --nnodes=1 --nproc-per-node 2 --master-addr 127.0.0.1 \
        --master-port 29552 -m streamep_b200.stream_moe.train_lm

The next token is a fixed function of the present one in seven of eight cases and random otherwise, so the loss can fall from
ln(vocabulary) to about ``ln(vocabulary) / 8 + 0.38``.  Prints the loss, the gradients' norm and the time of a step.
"""
from __future__ import annotations

import argparse
import sys

import torch

from ..models.moe_layer import make_buffer
from ..models.moe_lm import ExpertAdamW, MoELM
from ._harness_common import init_distributed, rank_zero_print


def batch(gen, vocab: int, tokens: int, device):
    x = torch.randint(0, vocab, (tokens,), generator=gen, device=device)
    follow = (x * 31 + 7) % vocab
    noise = torch.rand(tokens, generator=gen, device=device) < 0.125
    return x, torch.where(noise, torch.randint(0, vocab, (tokens,), generator=gen, device=device), follow)


def train(model, optimizer, steps: int, tokens: int, vocab: int, device, seed: int, report=None):
    """Returns the losses of all steps (one host read at the end)."""
    gen = torch.Generator(device=device).manual_seed(seed)
    losses = []
    for i in range(steps):
        x, y = batch(gen, vocab, tokens, device)
        optimizer.zero_grad()
        loss = model(x, y)
        loss.backward()
        norm = optimizer.step()
        losses.append(loss.detach())
        if report is not None:
            report(i, loss.detach(), norm)
    return torch.stack(losses).tolist()


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--tokens", type=int, default=4096, help="per rank")
    ap.add_argument("--hidden", type=int, default=512)
    ap.add_argument("--ffn", type=int, default=256)
    ap.add_argument("--experts", type=int, default=8, help="per rank")
    ap.add_argument("--topk", type=int, default=2)
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--vocab", type=int, default=8192)
    ap.add_argument("--steps", type=int, default=50)
    ap.add_argument("--lr", type=float, default=3e-3)
    ap.add_argument("--every", type=int, default=10, help="print every so many steps")
    args = ap.parse_args()
    rank, world, local, dev, group = init_distributed()
    experts = args.experts * world
    buf = make_buffer(group, args.tokens, args.hidden, args.topk, experts, layers_in_flight=args.layers, world_size=world)
    model = MoELM(args.vocab, args.hidden, args.ffn, experts, args.topk, args.layers, buf, device=dev)
    opt = ExpertAdamW(model.replicated_parameters(), model.expert_parameters(), lr=args.lr, group=group)
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)

    def report(i, loss, norm):
        if i % args.every == 0 or i == args.steps - 1:
            rank_zero_print(rank, f"step {i}: loss {float(loss):.4f}, norm {float(norm):.4f}")

    train(model, opt, 2, args.tokens, args.vocab, dev, seed=1000 + rank)        # warm-up
    start.record()
    losses = train(model, opt, args.steps, args.tokens, args.vocab, dev, seed=rank, report=report)
    end.record()
    torch.cuda.synchronize()
    buf.check_status()
    rank_zero_print(rank, f"train_lm: world={world} tokens/rank={args.tokens} vocab={args.vocab}: loss {losses[0]:.3f} -> {losses[-1]:.3f}, "
                          f"{start.elapsed_time(end) / args.steps:.3f} ms/step (includes the reads for printing)")
    if world > 1:
        torch.distributed.destroy_process_group()
    return 0 if losses[-1] < losses[0] else 1


if __name__ == "__main__":
    sys.exit(main())
