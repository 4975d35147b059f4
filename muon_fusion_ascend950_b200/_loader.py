"""Loads the native operator library and registers its FakeTensor kernel.

Mirrors muon_ascend950/_loader.py of the reference (lines 10-49): the
``MUON_ASCEND950_LIBRARY`` override, otherwise the first ``_C*.so`` next to
this file, loaded with ``torch.ops.load_library``; then
``register_fake("muon_ascend950::polar_step")`` returning
``empty_like(x, memory_format=contiguous)``, tolerating an existing
registration.  The reference imports torch_npu here; this build needs only
torch with CUDA.
"""
from __future__ import annotations

import os
from pathlib import Path

_LOADED = False


def _library_path() -> Path:
    configured = os.environ.get("MUON_ASCEND950_LIBRARY")
    if configured:
        path = Path(configured).expanduser().resolve()
        if not path.is_file():
            raise RuntimeError(f"MUON_ASCEND950_LIBRARY does not exist: {path}")
        return path

    package_dir = Path(__file__).resolve().parent
    candidates = sorted(package_dir.glob("_C*.so"))
    if not candidates:
        raise RuntimeError(
            "muon_ascend950 native library is missing. Build it with "
            "`python -m muon_fusion_ascend950_b200.build` (or "
            "`python -c 'import __graft_entry__ as g; g.build()'`)."
        )
    return candidates[0]


def load_library() -> None:
    global _LOADED
    if _LOADED:
        return

    try:
        import torch
    except ImportError as exc:  # pragma: no cover - torch is a hard requirement
        raise RuntimeError("muon_ascend950 requires torch") from exc

    torch.ops.load_library(str(_library_path()))

    def fake_polar_step(x, a: float, b: float, c: float):
        return torch.empty_like(x, memory_format=torch.contiguous_format)

    def fake_polar_express(x, coefficients, normalize=True):
        return torch.empty_like(x, dtype=torch.bfloat16, memory_format=torch.contiguous_format)

    def fake_muon_update(param, grad, momentum_buffer, lr, momentum, nesterov, weight_decay,
                         scale, coefficients):
        return None

    # The fake kernels of the training-step operators check their arguments as
    # the native ones do, so that a traced call is refused where a real one is.
    def fake_distill_topk(student, values, indices, lse, temperature):
        from .training import check_distill

        check_distill(student, values, indices, temperature, teacher_lse=lse)
        lead = student.shape[:-1]
        return (student.new_empty(lead, dtype=torch.float32),
                student.new_empty((lead.numel(), 2), dtype=torch.float32))

    def grad_like(student):
        """The gradient has the logits' layout where their rows are padded by
        no more than a row's length, else it is contiguous."""
        vocab = student.shape[-1]
        rows = student.reshape(-1, vocab)
        if rows.shape[0] > 1 and rows.stride(1) == 1 and vocab < rows.stride(0) <= 2 * vocab:
            return student.new_empty_strided(rows.shape, rows.stride()).view(student.shape)
        return student.new_empty(student.shape)

    def fake_distill_topk_backward(grad_loss, student, values, indices, lse, stats, temperature):
        return grad_like(student)

    def fake_distill_topk_grad(student, values, indices, row_scale, lse, temperature):
        from .training import check_distill

        check_distill(student, values, indices, temperature, row_scale=row_scale, teacher_lse=lse)
        return student.new_empty(student.shape[:-1], dtype=torch.float32), grad_like(student)

    def fake_residual_norm(block_out, residual, post, pre, gate, scale, eps):
        from .training import check_norm

        check_norm(block_out, residual, post, pre, gate, scale, eps)
        rows = block_out.shape[:-1].numel()
        return (block_out.new_empty(block_out.shape),
                block_out.new_empty(block_out.shape if pre is not None else (0,)),
                block_out.new_empty((2, rows), dtype=torch.float32))

    def fake_residual_norm_backward(grad_hidden, grad_normed, block_out, residual, post, pre, gate,
                                    scale, rstd, eps, wanted):
        inputs = (block_out, residual, post, pre, gate, scale)
        return tuple(t.new_empty(t.shape) if want and t is not None else block_out.new_empty((0,))
                     for t, want in zip(inputs, wanted))

    def fake_route_experts(logits, bias, k, score, groups, top_groups, group_top, renormalize, scale):
        from .training import check_route

        check_route(logits, bias, k, score, groups, top_groups, group_top, scale)
        shape = (*logits.shape[:-1], k)
        return (logits.new_empty(shape, dtype=torch.float32),
                logits.new_empty(shape, dtype=torch.int64),
                logits.new_empty((logits.shape[-1],), dtype=torch.int64))

    def fake_route_experts_backward(grad_weights, logits, indices, score, renormalize, scale):
        return logits.new_empty(logits.shape)

    # Extensions of this build: polar_step_t (the step of x^T in x's layout)
    # has polar_step's output contract; polar_express returns bf16 of x's
    # shape; muon_update_ mutates its arguments and returns nothing.  The
    # training-step operators (training.py) return fresh tensors.
    fakes = (("muon_ascend950::polar_step", fake_polar_step),
             ("muon_ascend950::polar_step_t", fake_polar_step),
             ("muon_ascend950::polar_express", fake_polar_express),
             ("muon_ascend950::muon_update_", fake_muon_update),
             ("muon_ascend950::distill_topk", fake_distill_topk),
             ("muon_ascend950::distill_topk_backward", fake_distill_topk_backward),
             ("muon_ascend950::distill_topk_grad", fake_distill_topk_grad),
             ("muon_ascend950::residual_norm", fake_residual_norm),
             ("muon_ascend950::residual_norm_backward", fake_residual_norm_backward),
             ("muon_ascend950::route_experts", fake_route_experts),
             ("muon_ascend950::route_experts_backward", fake_route_experts_backward))
    for name, fn in fakes:
        try:
            torch.library.register_fake(name)(fn)
        except RuntimeError as exc:
            if "already has" not in str(exc):
                raise
    _LOADED = True
