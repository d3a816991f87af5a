"""Train a small student against a teacher's top logits, every step on one MI355X.

The whole step runs on this package's kernels: products of the blocks in 8-bit floating
point (``fp8_linear``), the norms, gate and residual scale around each block
(``block_norms``), the loss and its gradient in one pass, written over the logits
(``distill_topk_with_grad``), and the Muon update of the matrices.  The few vectors take a
plain gradient step.

    python examples/distill_step.py [--steps 40] [--width 512] [--layers 2] [--seed 0]
"""

from __future__ import annotations

import argparse
import math
import time

import torch

from muon_fusion_ascend950_amd import Muon
from muon_fusion_ascend950_amd.train import block_norms, distill_topk_with_grad, fp8_linear

VOCAB, TOP, SEQUENCES, LENGTH, TEMPERATURE = 4099, 16, 8, 128, 1.5


class Student(torch.nn.Module):
    """Embedding, ``layers`` MLP blocks between norms, and a head."""

    def __init__(self, width: int, layers: int, gen: torch.Generator):
        super().__init__()

        def matrix(n, k):
            return torch.nn.Parameter(torch.randn(n, k, generator=gen) / math.sqrt(k))

        self.embed = torch.nn.Parameter(torch.randn(VOCAB, width, generator=gen))
        self.up = torch.nn.ParameterList(matrix(4 * width, width) for _ in range(layers))
        self.down = torch.nn.ParameterList(matrix(width, 4 * width) for _ in range(layers))
        self.head = matrix(VOCAB, width)
        ones = [torch.nn.Parameter(torch.ones(width)) for _ in range(3 * layers)]
        self.post, self.pre, self.gate = (torch.nn.ParameterList(ones[i::3]) for i in range(3))
        self.scale = torch.nn.ParameterList(
            torch.nn.Parameter(torch.ones(1)) for _ in range(layers))

    def forward(self, tokens):
        x = torch.nn.functional.embedding(tokens, self.embed)  # the residual stream, float32
        h = torch.nn.functional.rms_norm(x, x.shape[-1:]).to(torch.bfloat16)
        for up, down, post, pre, gate, scale in zip(self.up, self.down, self.post, self.pre,
                                                    self.gate, self.scale):
            y = fp8_linear(torch.nn.functional.gelu(fp8_linear(h, up)), down)
            x, h = block_norms(y, x, post_weight=post, gate=gate, residual_scale=scale,
                               pre_weight=pre)
        return fp8_linear(h, self.head)

    def matrices(self):
        return [*self.up, *self.down]

    def vectors(self):
        chosen = {id(p) for p in self.matrices()}
        return [p for p in self.parameters() if id(p) not in chosen]


def train(steps: int, width: int = 512, layers: int = 2, seed: int = 0):
    """Losses of ``steps`` training steps and the microseconds of the last ones."""
    gen = torch.Generator().manual_seed(seed)  # seeded on the host: the same run every time
    student = Student(width, layers, gen).cuda()
    tokens = torch.randint(0, VOCAB, (SEQUENCES, LENGTH), generator=gen).cuda()
    # a stored teacher: the top logits of each token, fewer for some
    logits = 3.0 * torch.randn(SEQUENCES, LENGTH, VOCAB, generator=gen).cuda()
    teacher, index = torch.topk(logits, TOP, dim=-1)
    index = index.to(torch.int32)
    index[:, ::5, TOP // 2:] = -1
    counted = torch.ones(SEQUENCES, LENGTH, device="cuda")
    counted[:, :8] = 0.0  # prompt tokens
    weight = counted / counted.sum()

    muon = Muon(student.matrices(), lr=0.02)
    others = torch.optim.SGD(student.vectors(), lr=0.5)
    losses, began = [], 0.0
    for step in range(steps):
        if step == steps // 2:
            torch.cuda.synchronize()
            began = time.perf_counter()
        out = student(tokens)
        # nothing keeps the logits for the backward pass: the gradient takes their place
        z = out.detach()
        loss, grad = distill_topk_with_grad(z, teacher, index, grad_loss=weight,
                                            temperature=TEMPERATURE, out=z)
        out.backward(grad)
        muon.step()
        others.step()
        muon.zero_grad()
        others.zero_grad()
        losses.append((loss * weight).sum())
    torch.cuda.synchronize()
    us = (time.perf_counter() - began) / max(1, steps - steps // 2) * 1e6
    return [float(v) for v in losses], us


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=40)
    ap.add_argument("--width", type=int, default=512)
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--seed", type=int, default=0)
    args = ap.parse_args()
    losses, us = train(args.steps, args.width, args.layers, args.seed)
    print(f"{SEQUENCES * LENGTH} tokens, vocabulary {VOCAB}, {args.layers} blocks of width {args.width}")
    print(f"loss {losses[0]:.4f} -> {losses[-1]:.4f} in {args.steps} steps, {us:.0f} us a step")


if __name__ == "__main__":
    main()
