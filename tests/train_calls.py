"""Calls of the training-step operators that are taken or refused, for the tests
of the native operators and of their FakeTensor kernels alike."""
from __future__ import annotations

import math

import torch

import muon_fusion_ascend950_b200 as pkg

F64, F32, BF16, INT = torch.float64, torch.float32, torch.bfloat16, torch.int64


def make(*shape, dtype=F32):
    return torch.zeros(shape, dtype=dtype, device="cuda")


def distill(name, **kw):
    """One call with [4, 16] logits and lists of two, but for what kw says."""
    a = dict(z=make(4, 16), t=make(4, 2), i=make(4, 2, dtype=INT), lse=None, row_scale=None, temperature=1.0)
    a.update(kw)
    if name == "distill_topk_grad":
        return pkg.distill_topk_grad(a["z"], a["t"], a["i"], a["row_scale"], temperature=a["temperature"],
                                     teacher_lse=a["lse"])
    return pkg.distill_topk(a["z"], a["t"], a["i"], temperature=a["temperature"], teacher_lse=a["lse"])


def lists(top, dtype=F32):
    return dict(t=make(4, top, dtype=dtype), i=make(4, top, dtype=INT))


def norm(**kw):
    a = dict(y=make(4, 16), x=make(4, 16), post_weight=make(16), pre_weight=make(16))
    a.update(kw)
    return pkg.residual_norm(a.pop("y"), a.pop("x"), **a)


def route(experts=16, k=2, **kw):
    return pkg.route_experts(make(4, experts), k, **kw)


# name -> (call, the error it raises or None)
CALLS = {}
for op in ("distill_topk", "distill_topk_grad"):
    for what, kw, error in (
            ("plain", lambda: {}, None), ("longest list", lambda: lists(1024), None),
            ("list too long", lambda: lists(1025), ValueError), ("empty list", lambda: lists(0), ValueError),
            ("lists of integers", lambda: lists(2, INT), TypeError), ("lists of fp64", lambda: lists(2, F64), TypeError),
            ("logits of fp64", lambda: dict(z=make(4, 16, dtype=F64)), TypeError),
            ("indices of fp32", lambda: dict(i=make(4, 2)), TypeError),
            ("infinite temperature", lambda: dict(temperature=math.inf), ValueError),
            ("temperature beyond fp32", lambda: dict(temperature=1e39), ValueError),
            ("temperature below fp32", lambda: dict(temperature=1e-50), ValueError),
            ("least temperature", lambda: dict(temperature=2.0 ** -126), None),
            ("subnormal temperature", lambda: dict(temperature=2.0 ** -127), ValueError),
            ("no temperature", lambda: dict(temperature=math.nan), ValueError),
            ("normaliser of fp64", lambda: dict(lse=make(4, dtype=F64)), None),
            ("normaliser of bf16", lambda: dict(lse=make(4, dtype=BF16)), None),
            ("normaliser of integers", lambda: dict(lse=make(4, dtype=INT)), TypeError),
            ("normaliser of another shape", lambda: dict(lse=make(3)), ValueError)):
        CALLS[f"{op}: {what}"] = (lambda op=op, kw=kw: distill(op, **kw()), error)
CALLS["distill_topk_grad: weights of fp64"] = (
    lambda: distill("distill_topk_grad", row_scale=make(4, dtype=F64)), None)
CALLS["distill_topk_grad: weights of integers"] = (
    lambda: distill("distill_topk_grad", row_scale=make(4, dtype=INT)), TypeError)
for what, kw, error in (
        ("plain", lambda: {}, None), ("infinite eps", lambda: dict(eps=math.inf), ValueError),
        ("no eps", lambda: dict(eps=math.nan), ValueError), ("negative eps", lambda: dict(eps=-1.0), ValueError),
        ("eps of 0", lambda: dict(eps=0.0), None), ("weight of fp64", lambda: dict(pre_weight=make(16, dtype=F64)), TypeError),
        ("scale of fp64", lambda: dict(residual_scale=make(1, dtype=F64)), TypeError),
        ("scale of one element", lambda: dict(residual_scale=make(1, 1)), None),
        ("gate of another width", lambda: dict(gate=make(4, 1)), ValueError)):
    CALLS[f"residual_norm: {what}"] = (lambda kw=kw: norm(**kw()), error)
for what, kw, error in (
        ("plain", lambda: {}, None), ("most experts", lambda: dict(experts=1024, k=64), None),
        ("too many experts", lambda: dict(experts=2000, k=100), ValueError),
        ("too many choices", lambda: dict(experts=100, k=65), ValueError),
        ("no choice", lambda: dict(k=0), ValueError), ("more choices than experts", lambda: dict(k=17), ValueError),
        ("three best of a group", lambda: dict(groups=4, group_top=3), ValueError),
        ("none of a group", lambda: dict(groups=4, group_top=0), ValueError),
        ("two best of one", lambda: dict(groups=16, top_groups=4, group_top=2), ValueError),
        ("two best of the row", lambda: dict(group_top=2), None),
        ("groups of different sizes", lambda: dict(groups=3), ValueError),
        ("more groups than there are", lambda: dict(groups=4, top_groups=5), ValueError),
        ("infinite scale", lambda: dict(scale=math.inf), ValueError),
        ("an unknown score", lambda: dict(score="tanh"), ValueError),
        ("bias of fp64", lambda: dict(bias=make(16, dtype=F64)), None),
        ("bias of integers", lambda: dict(bias=make(16, dtype=INT)), TypeError),
        ("bias of another shape", lambda: dict(bias=make(15)), ValueError)):
    CALLS[f"route_experts: {what}"] = (lambda kw=kw: route(**kw()), error)
