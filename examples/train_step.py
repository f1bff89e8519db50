"""A training step from the embedding to the optimizer with this package's operators.

A small residual model: every block has a norm before it and one behind it with a learned gate
(``residual_norm`` takes a block's output to the next block's input), the head's loss is the cross
entropy plus the divergence from a teacher's top logits (``linear_cross_entropy``,
``linear_distillation``; the logits are never held), and ``Muon`` updates the matrices.

    python examples/train_step.py [--steps 20]
"""
from __future__ import annotations

import argparse
import os
import sys

import torch
from torch import nn

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import dmuon_amd as dmuon  # noqa: E402


class Model(nn.Module):
    def __init__(self, vocab: int, dim: int, blocks: int, dtype: torch.dtype) -> None:
        super().__init__()
        def matrix(rows, cols):
            return nn.Parameter((torch.randn(rows, cols) / cols ** 0.5).to(dtype))
        self.embed = nn.Parameter(torch.randn(vocab, dim).to(dtype))
        self.head = matrix(vocab, dim)
        self.up = nn.ParameterList(matrix(2 * dim, dim) for _ in range(blocks))
        self.down = nn.ParameterList(matrix(dim, 2 * dim) for _ in range(blocks))
        # norm weights before each block and before the head, norms and gates behind each block
        self.pre = nn.ParameterList(nn.Parameter(torch.ones(dim)) for _ in range(blocks + 1))
        self.post = nn.ParameterList(nn.Parameter(torch.ones(dim)) for _ in range(blocks))
        self.gate = nn.ParameterList(nn.Parameter(torch.full((dim,), 0.5)) for _ in range(blocks))

    def forward(self, tokens: torch.Tensor) -> torch.Tensor:
        """The head's input, normed."""
        x, h = dmuon.residual_norm(self.embed[tokens], None, self.pre[0])
        for up, down, pre, post, gate in zip(self.up, self.down, self.pre[1:], self.post, self.gate):
            y = torch.relu(h @ up.t()).square() @ down.t()
            x, h = dmuon.residual_norm(x, y, pre, post_weight=post, gate=gate)
        return h


def main(steps: int = 20, batch: int = 8, length: int = 128, vocab: int = 5003, dim: int = 512,
         blocks: int = 2, teacher_k: int = 16, verbose: bool = True) -> list:
    torch.manual_seed(0)
    dev = torch.device("cuda")
    model = Model(vocab, dim, blocks, torch.bfloat16).to(dev)
    # the teacher of a stationary language: the next token depends on the last one alone
    follow = torch.randint(0, vocab, (vocab, teacher_k), device=dev)
    rank = torch.log_softmax(-0.5 * torch.arange(teacher_k, device=dev, dtype=torch.float32), 0)

    dmuon.dedicate_params(model, None, lambda name, p: p.dim() == 2 and p.shape[0] != vocab)
    dmuon.replicate(model)
    opt = dmuon.Muon(model, lr=0.02, momentum=0.95, weight_decay=0.0, adamw_lr=3e-3)
    losses = []
    for step in range(steps):
        tokens = torch.randint(0, vocab, (batch, length), device=dev)
        ids = follow[tokens]
        picked = torch.multinomial(rank.exp(), batch * length, replacement=True).view(batch, length, 1)
        target = ids.gather(2, picked)[..., 0]
        target[:, 0] = -100                               # nothing to predict the first one from
        h = model(tokens)
        hard = dmuon.linear_cross_entropy(h, model.head, target)
        soft = dmuon.linear_distillation(h, model.head, ids, rank.expand(ids.shape))
        (hard + soft).backward()
        opt.clip_grad_norm_(1.0)
        opt.step()
        opt.zero_grad()
        hard, soft = hard.detach(), soft.detach()
        losses.append((hard, soft))
        if verbose:
            print(f"step {step:3d}  cross entropy {float(hard):.4f}  distillation {float(soft):.4f}",
                  flush=True)
    return [(float(a), float(b)) for a, b in losses]


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=20)
    main(ap.parse_args().steps)
