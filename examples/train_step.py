"""A training step from the embedding to the optimizer with this package's operators.

A small residual model: tokens are looked up (``embedding``); every block has attention, whose
queries and keys are normed and rotated head by head (``rotary_heads``, ``attention``), and a
feed-forward part, each with a norm before it and one behind it with a learned gate
(``residual_norm`` takes one's output to the next one's input). The head's loss is the cross entropy
plus the divergence from a teacher's top logits (``linear_cross_entropy``, ``linear_distillation``;
the logits are never held), and ``Muon`` updates the matrices.

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
        self.head_dim, self.heads, self.kv_heads = 32, dim // 32, dim // 64
        self.embed = nn.Parameter(torch.randn(vocab, dim).to(dtype))
        self.head = matrix(vocab, dim)
        # one product for queries, keys and values; the norms of a head's queries and keys
        self.qkv = nn.ParameterList(matrix((self.heads + 2 * self.kv_heads) * self.head_dim, dim)
                                    for _ in range(blocks))
        self.out = nn.ParameterList(matrix(dim, dim) for _ in range(blocks))
        self.q_norm = nn.ParameterList(nn.Parameter(torch.ones(self.head_dim)) for _ in range(blocks))
        self.k_norm = nn.ParameterList(nn.Parameter(torch.ones(self.head_dim)) for _ in range(blocks))
        self.up = nn.ParameterList(matrix(2 * dim, dim) for _ in range(blocks))
        self.down = nn.ParameterList(matrix(dim, 2 * dim) for _ in range(blocks))
        # norm weights before each half block and before the head, norms and gates behind each half
        self.pre = nn.ParameterList(nn.Parameter(torch.ones(dim)) for _ in range(2 * blocks + 1))
        self.post = nn.ParameterList(nn.Parameter(torch.ones(dim)) for _ in range(2 * blocks))
        self.gate = nn.ParameterList(nn.Parameter(torch.full((dim,), 0.5)) for _ in range(2 * blocks))
        self.register_buffer("inv_freq", 10000.0 ** (-torch.arange(0, 1, 2 / self.head_dim)))

    def attend(self, h: torch.Tensor, block: int) -> torch.Tensor:
        d = self.head_dim
        heads = (h @ self.qkv[block].t()).unflatten(-1, (-1, d))
        q, k, v = heads.split([self.heads, self.kv_heads, self.kv_heads], -2)
        positions = torch.arange(h.shape[1], device=h.device)
        q, k = dmuon.rotary_heads(q, k, positions, self.inv_freq, q_weight=self.q_norm[block],
                                  k_weight=self.k_norm[block])
        return dmuon.attention(q, k, v).flatten(-2) @ self.out[block].t()

    def forward(self, tokens: torch.Tensor) -> torch.Tensor:
        """The head's input, normed."""
        x, h = dmuon.residual_norm(dmuon.embedding(tokens, self.embed), None, self.pre[0])
        half = 0
        for block, (up, down) in enumerate(zip(self.up, self.down)):
            for part in (lambda t: self.attend(t, block),
                         lambda t: torch.relu(t @ up.t()).square() @ down.t()):
                x, h = dmuon.residual_norm(x, part(h), self.pre[half + 1], post_weight=self.post[half],
                                           gate=self.gate[half])
                half += 1
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
