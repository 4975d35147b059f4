"""Operators of the training step around the Muon update, on the B200 kernels.

``Muon`` updates the matrices of a language model; these are the parts of the
step beside them that are bound by memory, each with its gradient:

* ``distill_topk`` / ``distill_topk_grad`` -- the distillation loss over a
  teacher's top logits, and the loss with its gradient in one call;
* ``residual_norm`` -- the norms before and after a residual block, fused with
  its gate and residual scale;
* ``route_experts`` -- the routing of tokens to the experts whose batched
  matrices ``Muon`` updates.

They are the operators ``torch.ops.muon_ascend950.*`` of the same names, which
check their arguments (ValueError, TypeError), run on the current stream and
take part in autograd (gradients of gradients and forward mode are refused).
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple

import torch

_FLOATS = (torch.float32, torch.bfloat16, torch.float16)
# muon_train_sm100.h: MUON_TRAIN_MAX_TOP, _MAX_EXPERTS, _MAX_ROUTES
MAX_TOP, MAX_EXPERTS, MAX_ROUTES = 1024, 1024, 64
_SCORES = {"softmax": 0, "sigmoid": 1}
_OPTIONAL = frozenset(("teacher_lse", "row_scale", "post_weight", "pre_weight", "gate", "residual_scale",
                       "bias"))
_distill_topk = torch.ops.muon_ascend950.distill_topk.default
_distill_topk_grad = torch.ops.muon_ascend950.distill_topk_grad.default
_residual_norm = torch.ops.muon_ascend950.residual_norm.default
_route_experts = torch.ops.muon_ascend950.route_experts.default


def _check(name: str, t, like: Optional[torch.Tensor] = None, *, floats: bool = True) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.device.type != "cuda":
        raise ValueError(f"{name} must be on a CUDA device, got {t.device}")
    if like is not None and t.device != like.device:
        raise ValueError(f"{name} must be on {like.device}, got {t.device}")
    if floats and t.dtype not in _FLOATS:
        raise TypeError(f"{name} must use torch.float32, bfloat16 or float16, got {t.dtype}")


def _check_values(name: str, t, like: torch.Tensor, shape) -> None:
    """Values that are converted to fp32: of any floating type."""
    _check(name, t, like, floats=False)
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if not t.is_floating_point():
        raise TypeError(f"{name} must be a floating tensor, got {t.dtype}")


def _float32(value: float) -> float:
    """`value` rounded to fp32, infinite beyond it."""
    return ctypes.c_float(value).value


# The native operators check their arguments themselves.  Only when a call has
# failed is it looked at here, so that what the dispatcher refuses before the
# operator sees it (no tensor, no CUDA tensor) gets the package's own error:
# small calls are bound by the host.
def _explain(**named) -> None:
    for name, t in named.items():
        if t is None and name in _OPTIONAL:
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
        if not t.is_cuda:
            raise ValueError(f"{name} must be on a CUDA device, got {t.device}")


# ------------------------------------------------- checks of traced calls
def check_distill(student_logits, teacher_logits, teacher_indices, temperature, **rows) -> None:
    _check("student_logits", student_logits)
    _check("teacher_logits", teacher_logits, student_logits)
    _check("teacher_indices", teacher_indices, student_logits, floats=False)
    if teacher_indices.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"teacher_indices must use torch.int64 or int32, got {teacher_indices.dtype}")
    if student_logits.ndim < 1 or student_logits.shape[-1] < 1:
        raise ValueError(f"student_logits must have shape [..., vocab], got {tuple(student_logits.shape)}")
    lead = student_logits.shape[:-1]
    if teacher_logits.shape != teacher_indices.shape or teacher_logits.ndim < 1 or (
            teacher_logits.shape[:-1] != lead):
        raise ValueError("teacher_logits and teacher_indices must both have shape "
                         f"{tuple(lead) + ('top',)}, got {tuple(teacher_logits.shape)} and "
                         f"{tuple(teacher_indices.shape)}")
    if not 1 <= teacher_logits.shape[-1] <= MAX_TOP:
        raise ValueError(f"a list must have 1 to {MAX_TOP} entries, got {teacher_logits.shape[-1]}")
    tau = _float32(temperature)
    if not (tau >= 2.0 ** -126 and math.isfinite(tau)):
        raise ValueError(f"temperature must be positive (2^-126 or more) and finite, got {temperature}")
    for name, t in rows.items():
        if t is not None:
            _check_values(name, t, student_logits, lead)


def gate_rows(gate: torch.Tensor, shape: torch.Size) -> int:
    """Rows of a gate whose leading sizes are ``shape``'s up to some axis and 1
    from there on, or which is one row."""
    if gate.ndim >= 1 and gate.shape[-1] == shape[-1]:
        lead = tuple(gate.shape[:-1])
        if all(n == 1 for n in lead):
            return 1
        if len(lead) == len(shape) - 1:
            same = 0
            while same < len(lead) and lead[same] == shape[same]:
                same += 1
            if all(n == 1 for n in lead[same:]):
                return gate.shape[:-1].numel()
    raise ValueError(f"gate must have shape [{shape[-1]}] or {tuple(shape)} with trailing leading sizes "
                     f"of 1, got {tuple(gate.shape)}")


def check_norm(block_out, residual, post_weight, pre_weight, gate, residual_scale, eps) -> None:
    _check("block_out", block_out)
    _check("residual", residual, block_out)
    if residual.dtype != block_out.dtype:
        raise TypeError(f"residual must use block_out's {block_out.dtype}, got {residual.dtype}")
    shape = block_out.shape
    if block_out.ndim < 1 or shape[-1] < 1:
        raise ValueError(f"block_out must have shape [..., width], got {tuple(shape)}")
    if residual.shape != shape:
        raise ValueError(f"residual must have block_out's shape {tuple(shape)}, got {tuple(residual.shape)}")
    width = shape[-1]
    for name, w in (("post_weight", post_weight), ("pre_weight", pre_weight)):
        if w is not None:
            _check(name, w, block_out)
            if w.shape != (width,):
                raise ValueError(f"{name} must have shape ({width},), got {tuple(w.shape)}")
    if gate is not None:
        _check("gate", gate, block_out)
        gate_rows(gate, shape)
    if residual_scale is not None:
        _check("residual_scale", residual_scale, block_out)
        if residual_scale.numel() != 1 and residual_scale.shape != (width,):
            raise ValueError(f"residual_scale must have one element or shape ({width},), "
                             f"got {tuple(residual_scale.shape)}")
    if not (eps >= 0.0 and math.isfinite(eps)):
        raise ValueError(f"eps must be finite and not negative, got {eps}")


def check_route(logits, bias, k, score, groups, top_groups, group_top, scale) -> None:
    _check("logits", logits)
    if logits.ndim < 1 or logits.shape[-1] < 1:
        raise ValueError(f"logits must have shape [..., experts], got {tuple(logits.shape)}")
    experts = logits.shape[-1]
    if experts > MAX_EXPERTS:
        raise ValueError(f"1 to {MAX_EXPERTS} experts are supported, got {experts}")
    if score not in (0, 1):
        raise ValueError("score must be 0 (softmax) or 1 (sigmoid)")
    if bias is not None:
        _check_values("bias", bias, logits, (experts,))
    if groups < 1 or experts % groups or not 1 <= top_groups <= groups:
        raise ValueError(f"groups must divide the {experts} experts and top_groups be 1 to groups, "
                         f"got {groups} and {top_groups}")
    if group_top != 1 and (group_top != 2 or (groups > 1 and experts // groups < 2)):
        raise ValueError(f"group_top must be 1, or 2 with groups of two experts or more, got {group_top}")
    if not 1 <= k <= min(MAX_ROUTES, top_groups * (experts // groups)):
        raise ValueError(f"k must be 1 to {MAX_ROUTES} and at most the experts of the chosen groups, got {k}")
    if not math.isfinite(scale):
        raise ValueError(f"scale must be finite, got {scale}")


# -------------------------------------------------------------- entry points
def distill_topk(student_logits: torch.Tensor, teacher_logits: torch.Tensor,
                 teacher_indices: torch.Tensor, *, temperature: float = 1.0,
                 teacher_lse: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Kullback-Leibler divergence of the student from the teacher's top
    logits, one fp32 value for each row.

    ``student_logits``: ``[..., vocab]``; ``teacher_logits`` and
    ``teacher_indices`` (int64 or int32): ``[..., top]``, up to 1024 entries of
    the same rows.  With ``tau = temperature`` the teacher's probabilities are
    the softmax of ``teacher_logits / tau`` over the row's entries, or, with
    ``teacher_lse`` (``[...]``: the log-sum-exp of the teacher's whole
    vocabulary at ``tau``), ``exp(teacher_logits / tau - teacher_lse)``, whose
    sum stays below one.  The loss is ``sum q (log q - log p)`` with ``p`` the
    softmax of ``student_logits / tau`` over the vocabulary.

    An entry whose index is outside the vocabulary (-1 pads a short list) or
    whose logit is -inf is left out; a row without entries has loss 0 and
    gradient 0.  Differentiable in ``student_logits``; the teacher's tensors
    are constants.
    """
    try:
        return _distill_topk(student_logits, teacher_logits, teacher_indices, teacher_lse, temperature)[0]
    except Exception:
        _explain(student_logits=student_logits, teacher_logits=teacher_logits,
                 teacher_indices=teacher_indices, teacher_lse=teacher_lse)
        raise


def distill_topk_grad(student_logits: torch.Tensor, teacher_logits: torch.Tensor,
                      teacher_indices: torch.Tensor, row_scale: Optional[torch.Tensor] = None, *,
                      temperature: float = 1.0, teacher_lse: Optional[torch.Tensor] = None
                      ) -> Tuple[torch.Tensor, torch.Tensor]:
    """``distill_topk`` and the gradient of ``sum(row_scale * loss)`` in
    ``student_logits`` in one launch.  The logits come from memory once: rows
    stay in registers, or in L2 until they are read again.

    ``row_scale`` (``[...]``, default 1) is what the rows weigh in the total,
    e.g. one over the number of tokens, or 0 for tokens that do not count.
    Returns ``(loss, grad)``, the gradient with the logits' shape and type; use
    it as ``student_logits.backward(grad)``.  Not recorded by autograd.
    """
    try:
        return _distill_topk_grad(student_logits, teacher_logits, teacher_indices, row_scale, teacher_lse,
                                  temperature)
    except Exception:
        _explain(student_logits=student_logits, teacher_logits=teacher_logits,
                 teacher_indices=teacher_indices, row_scale=row_scale, teacher_lse=teacher_lse)
        raise


def residual_norm(block_out: torch.Tensor, residual: torch.Tensor,
                  post_weight: Optional[torch.Tensor] = None,
                  pre_weight: Optional[torch.Tensor] = None, *,
                  gate: Optional[torch.Tensor] = None,
                  residual_scale: Optional[torch.Tensor] = None, eps: float = 1e-6
                  ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """The end of a residual block and the beginning of the next, in one pass:

        hidden = residual_scale * residual + gate * rms_norm(block_out, post_weight)
        normed = rms_norm(hidden, pre_weight)

    ``block_out``, ``residual``: ``[..., width]`` of one type (fp32, bf16 or
    fp16).  ``post_weight``, ``pre_weight``: ``[width]``; without
    ``post_weight`` the block's output is not normed, without ``pre_weight``
    ``normed`` is None.  ``gate``: ``[width]``, or the inputs' shape with 1 in
    place of trailing leading sizes (``[batch, 1, width]``: one row for each
    sequence).  ``residual_scale``: one element or ``[width]``.  Parameters may
    be of any of the three types.

    Statistics and sums are fp32, ``normed`` is computed from ``hidden`` before
    it is rounded, and each output is rounded once.  Differentiable in all
    tensor arguments; parameter gradients are summed in a fixed order.
    """
    try:
        hidden, normed, _ = _residual_norm(block_out, residual, post_weight, pre_weight, gate, residual_scale,
                                           eps)
    except Exception:
        _explain(block_out=block_out, residual=residual, post_weight=post_weight, pre_weight=pre_weight,
                 gate=gate, residual_scale=residual_scale)
        raise
    return hidden, normed if pre_weight is not None else None


def route_experts(logits: torch.Tensor, k: int, *, score: str = "softmax",
                  bias: Optional[torch.Tensor] = None, groups: int = 1, top_groups: int = 1,
                  group_top: Optional[int] = None, renormalize: bool = True, scale: float = 1.0
                  ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Choose ``k`` experts for each token.

    ``logits``: ``[..., experts]``, up to 1024 experts.  The scores are the
    softmax or the sigmoid of the logits.  ``bias`` (``[experts]``) is added to
    the scores for the choice only; balancing the experts is moving it.  With
    ``groups`` equal runs of experts, only the ``top_groups`` groups with the
    largest sum of their ``group_top`` best biased scores take part
    (``group_top``: 1 or 2, by default 1 for softmax and 2 for sigmoid).  The
    ``k`` best are returned in descending order; equal ones go to the lowest
    index.  Their weights are ``scale`` times their scores (without the bias),
    divided by the sum of the chosen scores when ``renormalize``.

    Returns ``(weights, indices, counts)``: fp32 and int64 ``[..., k]``, and
    int64 ``[experts]``, how many tokens each expert got.  Differentiable in
    ``logits`` through the weights.
    """
    try:
        if group_top is None:
            pairs = groups > 1 and score == "sigmoid" and logits.ndim > 0 and groups < logits.shape[-1]
            group_top = 2 if pairs else 1
        return _route_experts(logits, bias, k, _SCORES[score], groups, top_groups, group_top, renormalize, scale)
    except Exception:
        if score not in _SCORES:
            raise ValueError(f"score must be 'softmax' or 'sigmoid', got {score!r}") from None
        _explain(logits=logits, bias=bias)
        raise
