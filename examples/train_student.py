"""Trains a small mixture-of-experts transformer by distillation, with the package's
training-step operators and the ``Muon`` optimizer together:

    python examples/train_student.py [--steps 60]

Queries and keys are turned by ``rotary`` and tokens look back by ``attention``;
every block ends in ``residual_norm`` (the post-norm, gate and residual add of
this block and the pre-norm of the next in one pass), tokens go to experts by
``route_experts`` with a balancing bias, the loss and its gradient in the logits
come from ``distill_topk_grad``, ``clip_grad_norm`` holds the gradients to a norm,
and ``Muon`` updates the matrices, the experts' [experts, in, out] batches among
them.  The teacher is a table of logits for
each token, of which the student sees the top 16.
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch
import torch.nn.functional as F
from torch import nn

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from muon_fusion_ascend950_b200 import (  # noqa: E402
    Muon,
    attention,
    clip_grad_norm,
    distill_topk,
    distill_topk_grad,
    residual_norm,
    rotary,
    rotary_frequencies,
    route_experts,
)


def matrix(*shape):
    return nn.Parameter(torch.randn(*shape) * shape[-2] ** -0.5)


class Tail(nn.Module):
    """End of one residual block and norm before the next."""

    def __init__(self, width):
        super().__init__()
        self.post = nn.Parameter(torch.ones(width))
        self.pre = nn.Parameter(torch.ones(width))
        self.gate = nn.Parameter(torch.full((width,), 0.5))
        self.scale = nn.Parameter(torch.ones(1))

    def forward(self, block_out, hidden):
        return residual_norm(block_out, hidden, self.post, self.pre, gate=self.gate,
                             residual_scale=self.scale)


class Attention(nn.Module):
    """Causal attention of query heads that share key heads, at rotary positions."""

    def __init__(self, width, heads=4, kv_heads=2, dim=32):
        super().__init__()
        self.heads, self.dim = [heads, kv_heads, kv_heads], dim
        self.into, self.out = matrix(width, sum(self.heads) * dim), matrix(heads * dim, width)
        self.register_buffer("frequencies", rotary_frequencies(dim, device="cpu")[0])

    def forward(self, normed):
        heads = (normed @ self.into.to(normed.dtype)).unflatten(-1, (-1, self.dim))
        query, key, value = heads.split(self.heads, dim=-2)
        positions = torch.arange(normed.shape[1], device=normed.device)
        query, key = rotary(query, key, positions, self.frequencies)
        return attention(query, key, value, causal=True).flatten(-2) @ self.out.to(normed.dtype)


class Block(nn.Module):
    """Attention, a dense layer, then experts, each with its tail."""

    def __init__(self, width, inner, experts, k):
        super().__init__()
        self.k = k
        self.attention, self.attention_tail = Attention(width), Tail(width)
        self.dense_in, self.dense_out = matrix(width, inner), matrix(inner, width)
        self.router = matrix(width, experts)
        self.experts_in, self.experts_out = matrix(experts, width, inner), matrix(experts, inner, width)
        self.dense_tail, self.expert_tail = Tail(width), Tail(width)
        self.register_buffer("bias", torch.zeros(experts))

    def forward(self, hidden, normed):
        hidden, normed = self.attention_tail(self.attention(normed), hidden)
        out = F.silu(normed @ self.dense_in.to(normed.dtype)) @ self.dense_out.to(normed.dtype)
        hidden, normed = self.dense_tail(out, hidden)
        weights, indices, counts = route_experts(normed.float() @ self.router, self.k, score="sigmoid",
                                                 bias=self.bias, groups=2, top_groups=1)
        with torch.no_grad():  # an expert with few tokens is chosen more readily
            self.bias += 1e-2 * torch.sign(counts.float().mean() - counts)
        share = torch.zeros(*indices.shape[:-1], self.router.shape[1], device=weights.device)
        share = share.scatter(-1, indices, weights).to(normed.dtype)
        each = torch.einsum("btd,edh->bteh", normed, self.experts_in.to(normed.dtype))
        each = torch.einsum("bteh,ehd->bted", F.silu(each), self.experts_out.to(normed.dtype))
        return self.expert_tail(torch.einsum("bte,bted->btd", share, each), hidden)


class Student(nn.Module):
    def __init__(self, vocab=1000, width=128, inner=256, experts=8, k=2, blocks=2):
        super().__init__()
        self.embedding = matrix(vocab, width)
        self.first = nn.Parameter(torch.ones(width))
        self.blocks = nn.ModuleList(Block(width, inner, experts, k) for _ in range(blocks))
        self.head = matrix(width, vocab)

    def forward(self, tokens):
        hidden = (self.embedding[tokens] * self.embedding.shape[0] ** 0.5).to(torch.bfloat16)
        normed = F.rms_norm(hidden, (hidden.shape[-1],), self.first.to(hidden.dtype))
        for block in self.blocks:
            hidden, normed = block(hidden, normed)
        return normed @ self.head.to(normed.dtype)


def train(steps=60, batch=8, length=64, top=16, max_norm=1.0, seed=0, log=None):
    """Returns the mean loss a token of each step and of a last evaluation."""
    torch.manual_seed(seed)
    student = Student().cuda()
    vocab = student.embedding.shape[0]
    teacher = torch.randn(vocab, vocab, device="cuda") * 2.0
    matrices = [p for p in student.parameters() if p.ndim >= 2]
    vectors = [p for p in student.parameters() if p.ndim < 2]
    optimizers = [Muon(matrices, lr=0.02, momentum=0.9), torch.optim.AdamW(vectors, lr=1e-3)]
    losses = []

    def batch_of_tokens():
        tokens = torch.randint(0, vocab, (batch, length), device="cuda")
        values, indices = teacher[tokens].topk(top, dim=-1)
        indices[:, :4] = -1  # the prompt has no teacher: its rows do not count
        return tokens, values, indices

    for step in range(steps):
        tokens, values, indices = batch_of_tokens()
        counted = (indices[..., 0] >= 0).float()
        logits = student(tokens)
        loss, grad = distill_topk_grad(logits, values, indices, counted / counted.sum())
        logits.backward(grad)
        clip_grad_norm(student.parameters(), max_norm)
        for optimizer in optimizers:
            optimizer.step()
            optimizer.zero_grad(set_to_none=True)
        losses.append((loss * counted).sum() / counted.sum())
        if log is not None and step % 10 == 0:
            log(f"step {step:4d}  loss {losses[-1].item():.4f}")
    with torch.no_grad():
        tokens, values, indices = batch_of_tokens()
        loss = distill_topk(student(tokens), values, indices)
        losses.append(loss.sum() / (indices[..., 0] >= 0).sum())
    return [value.item() for value in losses]


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    parser.add_argument("--steps", type=int, default=60)
    losses = train(parser.parse_args().steps, log=print)
    print(f"evaluation loss {losses[-1]:.4f} (first step {losses[0]:.4f})")
