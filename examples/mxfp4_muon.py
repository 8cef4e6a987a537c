"""A small language model that trains and answers in 4-bit floating point.

    python -m examples.mxfp4_muon [--steps 400] [--width 512] [--tokens 4096]

The model predicts a token from the two before it: embeddings, residual blocks of two MXFP4 linear layers behind a norm that takes the
residual's addition along, an output matrix whose logits training never writes to memory.  The
blocks' matrices are stepped by FlashMuon (8-bit momentum, orthogonalised updates), everything else by FlashAdamW; the text
comes from a random second-order chain, so the best possible loss is known.  Afterwards the blocks' weights are kept in
MXFP4 alone (17/32 bytes each), the norms hand over MXFP4 too, and sequences are continued one token at a time.
"""

from __future__ import annotations

import argparse
import time
from typing import Optional

import torch
import torch.nn as nn
import torch.nn.functional as F

import flashoptim_amd as fo

VOCABULARY = 64
CHOICES = 4       # tokens that may follow a pair


class Block(nn.Module):
    def __init__(self, width: int):
        super().__init__()
        self.norm = fo.FlashRMSNorm(width)
        self.up = fo.MXFP4Linear(width, 4 * width, bias=False)
        self.down = fo.MXFP4Linear(4 * width, width, bias=False)

    def forward(self, branch: torch.Tensor, stream: Optional[torch.Tensor]) -> tuple[torch.Tensor, torch.Tensor]:
        """What the block adds to the stream, and the stream with what the block before added."""
        y, stream = (self.norm(branch), branch) if stream is None else self.norm(branch, stream)
        return self.down(F.gelu(self.up(y))), stream


class Model(nn.Module):
    def __init__(self, width: int, blocks: int):
        super().__init__()
        self.embed = fo.FlashEmbedding(VOCABULARY, width // 2)
        self.blocks = nn.ModuleList(Block(width) for _ in range(blocks))
        self.norm = fo.FlashRMSNorm(width)
        self.head = nn.Linear(width, VOCABULARY, bias=False)

    def forward(self, pairs: torch.Tensor, target: torch.Tensor) -> torch.Tensor:
        """The loss."""
        branch, stream = self.embed(pairs).flatten(1), None
        for block in self.blocks:
            branch, stream = block(branch, stream)
        y, _ = self.norm(branch, stream)
        return fo.linear_cross_entropy(y, self.head.weight, target)


class Served:
    """The trained model with its blocks' weights in MXFP4."""

    def __init__(self, model: Model):
        self.model = model
        self.weights = [(fo.mxfp4_quantize(b.up.weight), fo.mxfp4_quantize(b.down.weight)) for b in model.blocks]

    @torch.no_grad()
    def __call__(self, pairs: torch.Tensor) -> torch.Tensor:
        """The next token's logits."""
        branch, stream = self.model.embed(pairs).flatten(1), None
        for block, (up, down) in zip(self.model.blocks, self.weights):
            q = fo.rms_norm_mxfp4(branch, block.norm.weight, stream, eps=block.norm.eps)
            q, stream = (q, branch) if stream is None else q
            branch = fo.mxfp4_linear(F.gelu(fo.mxfp4_matmul(q, up)), down)
        y, _ = self.model.norm(branch, stream)
        return self.model.head(y)


class Chain:
    """Which tokens follow a pair of tokens, each of CHOICES with its probability."""

    def __init__(self, device: str):
        g = torch.Generator(device=device).manual_seed(7)
        weights = torch.rand(VOCABULARY, VOCABULARY, VOCABULARY, generator=g, device=device)
        kept = weights.topk(CHOICES, dim=2)
        self.next = torch.zeros_like(weights).scatter_(2, kept.indices, torch.softmax(8.0 * kept.values, 2))
        self.next /= self.next.sum(2, keepdim=True)
        self.entropy = -(self.next * self.next.clamp(min=1e-30).log()).sum(2).mean().item()
        self.g = g

    def draw(self, n: int):
        pairs = torch.randint(0, VOCABULARY, (n, 2), generator=self.g, device=self.next.device)
        return pairs, torch.multinomial(self.next[pairs[:, 0], pairs[:, 1]], 1, generator=self.g).squeeze(1)


def train(model: Model, chain: Chain, steps: int, tokens: int) -> list:
    hidden = [p for b in model.blocks for p in (b.up.weight, b.down.weight)]
    rest = [p for p in model.parameters() if not any(p is h for h in hidden)]
    optimizers = [fo.FlashMuon(hidden, lr=0.02, weight_decay=0.01), fo.FlashAdamW(rest, lr=3e-3, weight_decay=0.0)]
    losses = []
    for step in range(steps):
        for opt in optimizers:
            opt.param_groups[0]["lr"] = opt.defaults["lr"] * (1.0 - step / steps)
            opt.zero_grad()
        pairs, target = chain.draw(tokens)
        loss = model(pairs, target)
        loss.backward()
        for opt in optimizers:
            opt.step()
        losses.append(loss.detach())
    return torch.stack(losses).tolist()


@torch.no_grad()
def generate(served: Served, pairs: torch.Tensor, length: int) -> torch.Tensor:
    """Every pair continued by its likeliest tokens, one at a time."""
    out = [pairs[:, 0], pairs[:, 1]]
    for _ in range(length):
        out.append(served(torch.stack(out[-2:], 1)).argmax(1))
    return torch.stack(out, 1)


def main(argv=None) -> dict:
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--steps", type=int, default=400)
    parser.add_argument("--width", type=int, default=512)
    parser.add_argument("--blocks", type=int, default=2)
    parser.add_argument("--tokens", type=int, default=4096)
    parser.add_argument("--sequences", type=int, default=16)
    args = parser.parse_args(argv)
    device = "cuda:0"
    torch.manual_seed(0)
    model = Model(args.width, args.blocks).to(device).to(torch.bfloat16)
    chain = Chain(device)
    torch.cuda.synchronize()
    start = time.perf_counter()
    losses = train(model, chain, args.steps, args.tokens)
    took = time.perf_counter() - start
    served = Served(model)
    pairs, _ = chain.draw(args.sequences)
    text = generate(served, pairs, 32)
    allowed = (chain.next[text[:, :-2], text[:, 1:-1]].gather(2, text[:, 2:].unsqueeze(2)) > 0).float().mean().item()
    tail = sum(losses[-10:]) / len(losses[-10:])
    print(f"loss {losses[0]:.3f} -> {tail:.3f} (the chain's own entropy is {chain.entropy:.3f}), {args.steps / took:.0f} steps/s")
    print(f"{args.sequences} sequences continued in MXFP4: {100 * allowed:.1f} % of the tokens are ones that the chain allows "
          f"({100 * CHOICES / VOCABULARY:.1f} % by chance)")
    return dict(first=losses[0], last=tail, entropy=chain.entropy, allowed=allowed)


if __name__ == "__main__":
    main()
