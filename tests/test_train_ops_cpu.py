"""CPU tests of the training-step operators: argument checks of the Python
entry points and of the C ABI, the binding's coverage of the header, the
FakeTensor kernels, and the measured cases' own formulas."""
from __future__ import annotations

import ctypes
import importlib.util
import random
import re
from pathlib import Path

import pytest
import torch

import muon_fusion_ascend950_b200 as pkg
from muon_fusion_ascend950_b200 import capi as capi_module
from muon_fusion_ascend950_b200.capi import (
    CAPI,
    TRAIN_SIGNATURES,
    DistillArgs,
    NormArgs,
    NormGrads,
    RouteArgs,
)

from train_calls import CALLS

REPO = Path(__file__).resolve().parent.parent
HEADER = REPO / "include" / "muon_train_sm100.h"


@pytest.fixture(scope="module")
def lib():
    return CAPI().lib


def test_binding_covers_the_header(lib):
    names = set(re.findall(r"^\w[\w\s\*]*?\b(muon_train_\w+)\s*\(", HEADER.read_text(), re.M))
    assert names == set(TRAIN_SIGNATURES)
    for name in names:
        assert hasattr(lib, name), name


@pytest.mark.parametrize("struct, cname", [(DistillArgs, "distill_args"), (NormArgs, "norm_args"),
                                           (NormGrads, "norm_grads"), (RouteArgs, "route_args")])
def test_structs_have_the_headers_fields(struct, cname):
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    body = re.search(r"typedef struct \{([^}]*)\} muon_train_%s;" % cname, text).group(1)
    fields = []
    for line in body.split(";"):
        if line.strip():
            head, *rest = line.split(",")
            fields += [head.split()[-1].lstrip("*")] + [r.strip().lstrip("*") for r in rest]
    assert fields == [name for name, _ in struct._fields_]


def _distill(**kw):
    base = dict(logits=16, rows=2, vocab=8, ld=8, teacher_logits=16, teacher_indices=16, loss=16,
                top=2, temperature=1.0, dtype=1, teacher_dtype=0, index_bytes=8)
    return DistillArgs(**{**base, **kw})


@pytest.mark.parametrize("bad", [
    dict(rows=-1), dict(vocab=0), dict(ld=7), dict(top=0), dict(top=1025), dict(temperature=0.0),
    dict(temperature=float("nan")), dict(dtype=3), dict(teacher_dtype=-1), dict(index_bytes=2),
    dict(logits=None), dict(teacher_logits=None), dict(teacher_indices=None), dict(loss=None),
    dict(grad=16, ld_grad=8, stats=16), dict(grad=32, ld_grad=7, stats=16), dict(grad=32, ld_grad=8)])
def test_distill_refuses(lib, bad):
    args = _distill(**bad)
    assert lib.muon_train_distill_sm100(ctypes.byref(args), None) == -1


def test_distill_refuses_a_temperature_without_a_reciprocal(lib):
    assert lib.muon_train_distill_sm100(ctypes.byref(_distill(rows=0, temperature=2.0 ** -127)), None) == -1
    assert lib.muon_train_distill_sm100(ctypes.byref(_distill(rows=0, temperature=2.0 ** -126)), None) == 0


def test_wait_limit_refuses_null(lib):
    assert lib.muon_train_wait_limit_ns(None) == -1


def test_distill_refuses_null_and_backward_needs_stats(lib):
    assert lib.muon_train_distill_sm100(None, None) == -1
    args = _distill(grad=32, ld_grad=8)
    assert lib.muon_train_distill_backward_sm100(ctypes.byref(args), None) == -1
    args = _distill(stats=16)
    assert lib.muon_train_distill_backward_sm100(ctypes.byref(args), None) == -1
    assert lib.muon_train_distill_sm100(ctypes.byref(_distill(rows=0)), None) == 0


def _norm(**kw):
    base = dict(block_out=16, residual=16, post_weight=16, pre_weight=16, hidden=16, normed=16,
                rstd_post=16, rstd_pre=16, rows=6, width=8, eps=1e-6, dtype=1)
    return NormArgs(**{**base, **kw})


@pytest.mark.parametrize("bad", [
    dict(rows=-1), dict(width=0), dict(eps=-1.0), dict(eps=float("nan")), dict(dtype=5),
    dict(post_dtype=3), dict(pre_dtype=-1), dict(gate=16, gate_rows=4), dict(gate=16, gate_rows=0),
    dict(gate=16, gate_rows=1, gate_dtype=9), dict(residual_scale=16, scale_count=3),
    dict(residual_scale=16, scale_count=1, scale_dtype=7), dict(block_out=None),
    dict(residual=None), dict(hidden=None), dict(normed=None)])
def test_norm_refuses(lib, bad):
    args = _norm(**bad)
    assert lib.muon_train_residual_norm_sm100(ctypes.byref(args), None) == -1


def test_norm_backward_refuses(lib):
    call = lib.muon_train_residual_norm_backward_sm100
    ok = dict(grad_hidden=16, grad_normed=16, workspace=16, workspace_bytes=1 << 20)
    ref = ctypes.byref
    assert call(ref(_norm()), None, None) == -1
    assert call(ref(_norm()), ref(NormGrads(workspace=16, workspace_bytes=1 << 20)), None) == -1
    assert call(ref(_norm(rstd_post=None)), ref(NormGrads(**ok)), None) == -1
    assert call(ref(_norm(rstd_pre=None)), ref(NormGrads(**ok)), None) == -1
    assert call(ref(_norm(pre_weight=None)), ref(NormGrads(**ok)), None) == -1
    assert call(ref(_norm(rows=0)), ref(NormGrads()), None) == 0


def _route(**kw):
    base = dict(logits=16, weights=16, indices=16, tokens=3, experts=8, ld=8, dtype=0, score=0, k=2,
                groups=1, top_groups=1, group_top=1, scale=1.0)
    return RouteArgs(**{**base, **kw})


@pytest.mark.parametrize("bad", [
    dict(tokens=-1), dict(experts=0), dict(experts=1025, ld=1025), dict(k=0), dict(k=9), dict(k=65),
    dict(groups=0), dict(groups=3), dict(groups=2, top_groups=3), dict(groups=4, top_groups=1, k=3),
    dict(group_top=3), dict(groups=8, top_groups=8, group_top=2), dict(score=2), dict(dtype=4),
    dict(ld=7), dict(logits=None), dict(indices=None), dict(weights=None)])
def test_route_refuses(lib, bad):
    args = _route(**bad)
    assert lib.muon_train_route_sm100(ctypes.byref(args), None) == -1


def test_route_backward_refuses(lib):
    call = lib.muon_train_route_backward_sm100
    assert call(ctypes.byref(_route()), None, 16, None) == -1
    assert call(ctypes.byref(_route()), 16, None, None) == -1
    assert call(ctypes.byref(_route(tokens=0)), None, None, None) == 0


# ------------------------------------------------------- Python entry points
def test_entry_points_refuse_cpu_tensors_and_wrong_types():
    z, t, i = torch.zeros(2, 8), torch.zeros(2, 3), torch.zeros(2, 3, dtype=torch.int64)
    for call in (pkg.distill_topk, pkg.distill_topk_grad):
        with pytest.raises(ValueError):
            call(z, t, i)
        with pytest.raises(TypeError):
            call([[0.0]], t, i)
    with pytest.raises(ValueError):
        pkg.residual_norm(z, z)
    with pytest.raises(TypeError):
        pkg.residual_norm(z.tolist(), z)
    with pytest.raises(ValueError):
        pkg.route_experts(z, 2)
    with pytest.raises(TypeError):
        pkg.route_experts(None, 2)


@pytest.mark.parametrize("kw", [dict(), dict(groups=2), dict(groups=2, score="sigmoid")])
def test_route_refuses_what_is_no_tensor(kw):
    for logits in ([[0.0] * 4], None, 3):
        with pytest.raises(TypeError, match="logits must be a torch.Tensor"):
            pkg.route_experts(logits, 2, **kw)
    with _fake(), pytest.raises(ValueError):
        pkg.route_experts(_cuda(), 1, **kw)


def _fake():
    from torch._subclasses.fake_tensor import FakeTensorMode

    return FakeTensorMode()


def _cuda(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="cuda")


def test_entry_points_check_shapes_and_types():
    """The Python checks need no device: fake CUDA tensors reach them all."""
    with _fake():
        z, t = _cuda(2, 8), _cuda(2, 3)
        i = _cuda(2, 3, dtype=torch.int64)
        loss, grad = pkg.distill_topk_grad(z, t, i)
        assert loss.shape == (2,) and loss.dtype == torch.float32
        assert grad.shape == z.shape and grad.dtype == z.dtype
        assert pkg.distill_topk(z.view(2, 1, 8), t.view(2, 1, 3), i.view(2, 1, 3)).shape == (2, 1)
        for wrong in ((z, t, i[:, :2]), (z, t[:1], i[:1]), (z, t, _cuda(2, 3, dtype=torch.float32)),
                      (z.double(), t, i), (z, t.to(torch.int64), i)):
            with pytest.raises((TypeError, ValueError)):
                pkg.distill_topk(*wrong)
        with pytest.raises(ValueError):
            pkg.distill_topk(z, t, i, teacher_lse=_cuda(3, dtype=torch.float32))
        with pytest.raises(ValueError):
            pkg.distill_topk_grad(z, t, i, _cuda(2, 1, dtype=torch.float32))

        x, w = _cuda(2, 3, 16), _cuda(16)
        hidden, normed = pkg.residual_norm(x, x, w, w, gate=_cuda(2, 1, 16))
        assert hidden.shape == normed.shape == x.shape
        assert pkg.residual_norm(x, x, w)[1] is None
        for kw in (dict(gate=_cuda(3, 16)), dict(gate=_cuda(1, 3, 16)), dict(gate=_cuda(2, 3, 8)),
                   dict(gate=_cuda(2, 3, 1)), dict(residual_scale=_cuda(2)),
                   dict(pre_weight=_cuda(15)), dict(post_weight=_cuda(1, 16))):
            with pytest.raises(ValueError):
                pkg.residual_norm(x, x, **kw)
        with pytest.raises(ValueError):
            pkg.residual_norm(x, x[:1])
        with pytest.raises(TypeError):
            pkg.residual_norm(x, x.float())
        with pytest.raises(TypeError):
            pkg.residual_norm(x, x, w.double())

        weights, indices, counts = pkg.route_experts(_cuda(2, 5, 12), 3)
        assert weights.shape == indices.shape == (2, 5, 3) and counts.shape == (12,)
        assert weights.dtype == torch.float32 and indices.dtype == counts.dtype == torch.int64
        with pytest.raises(ValueError):
            pkg.route_experts(_cuda(2, 12), 3, score="tanh")
        with pytest.raises(ValueError):
            pkg.route_experts(_cuda(2, 12), 3, bias=_cuda(11))


def _calls(z):
    """Every operator as a function of its floating inputs, and these."""
    t, i = _cuda(2, 3), _cuda(2, 3, dtype=torch.int64)
    rows, w = _cuda(2, dtype=torch.float32), _cuda(8)
    return {
        "distill_topk": (lambda z, t, n: pkg.distill_topk(z, t, i, teacher_lse=n), (z, t, rows)),
        "distill_topk_grad": (lambda z, t, r, n: pkg.distill_topk_grad(z, t, i, r, teacher_lse=n),
                              (z, t, rows, rows.clone())),
        "residual_norm": (lambda y, x, p, q, g, s: pkg.residual_norm(y, x, p, q, gate=g, residual_scale=s),
                          (z, z.clone(), w, w.clone(), w.clone(), w.clone())),
        "route_experts": (lambda l, b: pkg.route_experts(l, 2, bias=b)[0], (z, w.float())),
    }


@pytest.mark.parametrize("name", ["distill_topk", "distill_topk_grad", "residual_norm", "route_experts"])
def test_forward_mode_is_refused(name):
    """A tangent in any input, whether gradients are recorded or not."""
    from torch.autograd import forward_ad

    with _fake():
        call, inputs = _calls(_cuda(2, 8))[name]
        for at in range(len(inputs)):
            with pytest.raises(NotImplementedError):
                torch.func.jvp(lambda v: call(*inputs[:at], v, *inputs[at + 1:]), (inputs[at],),
                               (torch.ones_like(inputs[at]),))
            with forward_ad.dual_level(), torch.no_grad(), pytest.raises(NotImplementedError):
                dual = forward_ad.make_dual(inputs[at], torch.ones_like(inputs[at]))
                call(*inputs[:at], dual, *inputs[at + 1:])


@pytest.mark.parametrize("name", CALLS)
def test_traced_calls_are_taken_and_refused(name):
    """As test_gpu_train_ops.py asks of the native operators."""
    call, error = CALLS[name]
    with _fake():
        if error is None:
            call()
        else:
            with pytest.raises(error):
                call()


def test_limits_are_the_headers():
    from muon_fusion_ascend950_b200 import training

    for name, value in (("TOP", training.MAX_TOP), ("EXPERTS", training.MAX_EXPERTS), ("ROUTES", training.MAX_ROUTES)):
        assert int(re.search(rf"#define MUON_TRAIN_MAX_{name} (\d+)", HEADER.read_text()).group(1)) == value


def test_gate_rows_of_every_shape():
    from muon_fusion_ascend950_b200.training import gate_rows

    shape = torch.Size((2, 3, 4, 8))
    for lead, rows in (((), 1), ((1,), 1), ((1, 1, 1), 1), ((2, 1, 1), 2), ((2, 3, 1), 6),
                       ((2, 3, 4), 24)):
        assert gate_rows(torch.empty(*lead, 8), shape) == rows
    for lead in ((3,), (1, 3, 1), (2, 1, 4), (2, 3, 4, 1)):
        with pytest.raises(ValueError):
            gate_rows(torch.empty(*lead, 8), shape)


def test_fake_backward_kernels():
    with _fake():
        ops = torch.ops.muon_ascend950
        z, t = _cuda(2, 8), _cuda(2, 3)
        i = _cuda(2, 3, dtype=torch.int64)
        loss, stats = ops.distill_topk(z, t, i, None, 1.0)
        assert stats.shape == (2, 2)
        assert ops.distill_topk_backward(loss, z, t, i, None, stats, 1.0).shape == z.shape
        x, w = _cuda(6, 16), _cuda(16, dtype=torch.float32)
        h, n, r = ops.residual_norm(x, x, w, None, None, None, 1e-6)
        assert n.shape == (0,) and r.shape == (2, 6)
        grads = ops.residual_norm_backward(h, None, x, x, w, None, None, None, r, 1e-6,
                                           [True, False, True, True, False, False])
        assert [g.shape[0] for g in grads] == [6, 0, 16, 0, 0, 0] and grads[2].dtype == torch.float32
        l = _cuda(4, 8)
        weights, indices, _ = ops.route_experts(l, None, 2, 0, 1, 1, 1, True, 1.0)
        assert ops.route_experts_backward(weights, l, indices, 0, True, 1.0).shape == l.shape


def test_fake_gradient_of_padded_logits_keeps_their_layout():
    with _fake():
        i = _cuda(2, 3, dtype=torch.int64)
        for pad, stride in ((8, 8), (10, 10), (16, 16), (17, 8)):
            z = _cuda(2, pad)[:, :8]
            assert pkg.distill_topk_grad(z, _cuda(2, 3), i)[1].stride() == (stride, 1)
        z = _cuda(2, 1, 10)[..., :8]
        grad = pkg.distill_topk_grad(z, _cuda(2, 1, 3), i.view(2, 1, 3))[1]
        assert grad.shape == z.shape and grad.stride(0) == 10


def test_measured_cases_stay_in_their_ranges():
    spec = importlib.util.spec_from_file_location("perf_operators", REPO / "perf" / "operators.py")
    cases = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(cases)
    assert not cases.own
    largest = max(cases.work(c)["bytes"] for c in cases.listed())
    for seed in range(200):
        c = cases.draw(random.Random(seed))
        assert cases.work(c)["bytes"] <= 1.02 * largest
        if c["op"] == "route":
            assert c["k"] <= c["top_groups"] * (c["experts"] // c["groups"])
    assert capi_module.TRAIN_SIGNATURES
