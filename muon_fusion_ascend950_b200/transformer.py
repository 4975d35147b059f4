"""Operators of a transformer block's training step, and of the clipping before
the update, on the B200 kernels:

* ``attention`` -- softmax attention with its backward pass, which computes the
  probabilities again instead of keeping them;
* ``rotary`` -- rotary positions of queries and keys in one launch, with
  ``rotary_frequencies`` for the usual frequencies and their stretched forms;
* ``clip_grad_norm`` / ``clip_gradients`` -- the global norm of many gradients,
  and the gradients scaled to a limit, before ``Muon`` and its companions step.

They are the operators ``torch.ops.muon_ascend950.*`` (``attention``,
``rotary``, ``clip_gradients_``, ``clip_gradients``), which check their arguments
(ValueError, TypeError), run on the current stream and, but for the clipping,
take part in autograd (gradients of gradients and forward mode are refused).
"""
from __future__ import annotations

import ctypes
import math
from typing import Iterable, Optional, Sequence, Tuple, Union

import torch

from ._loader import _library_path
from .training import _check, _explain, _float32

# muon_train_sm100.h: MUON_TRAIN_MAX_HEAD_DIM, _MAX_ROTARY_DIM
MAX_HEAD_DIM, MAX_ROTARY_DIM = 128, 4096
_MOST_TOKENS = 1 << 30
_attention = torch.ops.muon_ascend950.attention.default
_rotary = torch.ops.muon_ascend950.rotary.default
_clip_in_place = torch.ops.muon_ascend950.clip_gradients_.default
_clip_out = torch.ops.muon_ascend950.clip_gradients.default


def _list_entry(library):
    """The same on Python's own lists (clip_list.cpp), for long ones: the call
    itself takes longer.  None where the library is without it (one set by
    MUON_ASCEND950_LIBRARY) or does not find the tensors in this torch's objects."""
    entry, reads = (getattr(library, "muon_ascend950_clip_" + name, None) for name in ("list", "reads"))
    if entry is None or reads is None:
        return None
    reads.argtypes, reads.restype = [ctypes.py_object], ctypes.c_size_t
    probes = (torch.empty(shape, device="cpu") for shape in ((), (3, 2)))
    if any(reads(t) != t._cdata for t in probes):
        return None
    entry.argtypes = [ctypes.py_object, ctypes.c_void_p, ctypes.py_object, ctypes.c_double, ctypes.c_int]
    library.muon_ascend950_clip_message.restype = ctypes.c_char_p
    return entry


_library = ctypes.PyDLL(str(_library_path()))
_clip_list = _list_entry(_library)
_CLIP_ERRORS = {1: ValueError, 2: TypeError, 3: NotImplementedError, 4: RuntimeError}
_LONG_LIST = 32
_PLAIN = {torch.Tensor}


def _clip_lists(gradients: list, out: Optional[list], max_norm: float, largest: bool) -> Optional[torch.Tensor]:
    """The norm; None if the call has to go through the operator."""
    if set(map(type, gradients)) != _PLAIN or (out is not None and set(map(type, out)) != _PLAIN):
        return None
    if not gradients[0].is_cuda:
        return None
    norm = torch.empty((), dtype=torch.float32, device=gradients[0].device)
    status = _clip_list(gradients, None if out is None else id(out), norm, max_norm, largest)
    if status in _CLIP_ERRORS:
        raise _CLIP_ERRORS[status](_library.muon_ascend950_clip_message().decode(errors="replace"))
    return norm if status == 0 else None


# ------------------------------------------------- checks of traced calls
def _check_counts(name: str, t, like: torch.Tensor) -> None:
    _check(name, t, like, floats=False)
    if t.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name} must use torch.int32 or int64, got {t.dtype}")


def check_attention(query, key, value, offsets, lengths, window, scale) -> None:
    _check("query", query)
    _check("key", key, query)
    _check("value", value, query)
    n = 3 if offsets is not None else 4
    if query.ndim != n or key.ndim != n or value.ndim != n:
        raise ValueError("query, key and value must have shape "
                         f"{'[tokens, heads, dim]' if n == 3 else '[batch, length, heads, dim]'}, got "
                         f"{tuple(query.shape)}, {tuple(key.shape)} and {tuple(value.shape)}")
    if key.shape != value.shape or key.shape[-1] != query.shape[-1] or key.shape[0] != query.shape[0]:
        raise ValueError("key and value must have one shape, with query's first size and dim, got "
                         f"{tuple(query.shape)}, {tuple(key.shape)} and {tuple(value.shape)}")
    dim, heads, kv_heads = query.shape[-1], query.shape[-2], key.shape[-2]
    if not 8 <= dim <= MAX_HEAD_DIM or dim % 8:
        raise ValueError(f"dim must be 8 to {MAX_HEAD_DIM} in steps of 8, got {dim}")
    if heads < 1 or kv_heads < 1 or heads % kv_heads or heads > 65535:
        raise ValueError(f"the key heads must divide the query heads, got {kv_heads} and {heads}")
    if query.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"query must use torch.bfloat16 or float16, got {query.dtype}")
    if key.dtype != query.dtype or value.dtype != query.dtype:
        raise TypeError(f"key and value must use query's {query.dtype}, got {key.dtype} and {value.dtype}")
    if window < 0:
        raise ValueError(f"window must be positive, got {window}")
    s = _float32(scale)
    if not (s > 0.0 and math.isfinite(s)):
        raise ValueError(f"scale must be positive and finite, got {scale}")
    batch = 1 if n == 3 else query.shape[0]
    length, keys = query.shape[-3], key.shape[-3]
    if batch > 65535 or batch * length > _MOST_TOKENS or batch * keys > _MOST_TOKENS:
        raise ValueError("at most 65535 sequences and 2^30 tokens are supported")
    if offsets is not None:
        if lengths is not None:
            raise ValueError("offsets and lengths exclude each other")
        if offsets.ndim != 1 or offsets.shape[0] < 1:
            raise ValueError(f"offsets must have shape [sequences + 1], got {tuple(offsets.shape)}")
        _check_counts("offsets", offsets, query)
    if lengths is not None:
        if keys != length:
            raise ValueError(f"lengths need as many keys as queries, got {keys} and {length}")
        if lengths.shape != (batch,):
            raise ValueError(f"lengths must have shape ({batch},), got {tuple(lengths.shape)}")
        _check_counts("lengths", lengths, query)


def check_rotary(query, key, positions, frequencies, scale) -> None:
    _check("query", query)
    if query.ndim < 2:
        raise ValueError(f"query must have shape [..., heads, dim], got {tuple(query.shape)}")
    if key is not None:
        _check("key", key, query)
        if key.ndim != query.ndim or key.shape[-1] != query.shape[-1] or key.shape[:-2] != query.shape[:-2]:
            raise ValueError("key must have query's shape but for the heads, got "
                             f"{tuple(key.shape)} and {tuple(query.shape)}")
        if key.dtype != query.dtype:
            raise TypeError(f"key must use query's {query.dtype}, got {key.dtype}")
    _check_counts("positions", positions, query)
    _check("frequencies", frequencies, query, floats=False)
    if frequencies.dtype not in (torch.float32, torch.float64):
        raise TypeError(f"frequencies must use torch.float32 or float64, got {frequencies.dtype}")
    lead, dim = query.shape[:-2], query.shape[-1]
    if positions.shape != lead and not (len(lead) > 1 and positions.shape == lead[-1:]):
        raise ValueError(f"positions must have shape {tuple(lead)} or its last size, got {tuple(positions.shape)}")
    if not 1 <= dim <= MAX_ROTARY_DIM:
        raise ValueError(f"dim must be 1 to {MAX_ROTARY_DIM}, got {dim}")
    if frequencies.ndim != 1 or 2 * frequencies.shape[0] > dim:
        raise ValueError(f"frequencies must have shape [pairs] of at most dim / 2 = {dim // 2} pairs, "
                         f"got {tuple(frequencies.shape)}")
    if not math.isfinite(_float32(scale)):
        raise ValueError(f"scale must be finite, got {scale}")


def check_clip(gradients, out, max_norm) -> None:
    if len(gradients) == 0:
        raise ValueError("no gradients")
    if out is not None and len(out) != len(gradients):
        raise ValueError(f"out must have a tensor for each gradient, got {len(out)} and {len(gradients)}")
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must not be negative, got {max_norm}")
    for g, o in zip(gradients, gradients if out is None else out):
        _check("every gradient", g, gradients[0])
        _check("out", o, g)
        if g.requires_grad or o.requires_grad:
            raise ValueError("parameters and recorded tensors are not clipped (pass their gradients, detached)")
        if o.shape != g.shape:
            raise ValueError(f"out must have its gradient's shape, got {tuple(o.shape)} for {tuple(g.shape)}")


# -------------------------------------------------------------- entry points
def attention(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, *, causal: bool = False,
              window: Optional[int] = None, scale: Optional[float] = None,
              offsets: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None
              ) -> torch.Tensor:
    """Softmax attention of each query over the keys it sees.

    ``query``: ``[batch, length, heads, dim]``, ``key`` and ``value``: ``[batch,
    keys, kv_heads, dim]`` of one type (bf16 or fp16); ``dim`` is 8 to 128 in
    steps of 8, and ``kv_heads`` divides ``heads``: neighbouring query heads
    share a key head.  Slices of one projection are read in place.  ``scale``
    multiplies the products (by default ``dim ** -0.5``).

    Queries and keys are counted from the end: query ``i`` stands where key ``i +
    keys - length`` does.  With ``causal`` it sees the keys up to its own place,
    with ``window`` those less than ``window`` places away (on both sides, or
    behind it with ``causal``).  A query that sees no key has output 0 and
    gradient 0.

    ``lengths`` (``[batch]``, int32 or int64): only the first tokens of each
    sequence count; the output and the gradients of the others are 0.  With
    ``offsets`` (``[sequences + 1]``, int32 or int64, not descending) the tensors
    are ``[tokens, heads, dim]``: sequences one after another, of which sequence
    ``s`` is the tokens ``offsets[s]`` to ``offsets[s + 1]``; tokens outside of
    all have output and gradients 0.  Lengths and offsets stay on the device;
    those beyond the tensors are taken as their ends.  Tokens that do not count
    may hold anything.

    Returns the output with the query's shape.  Products are summed, and the
    softmax is taken, in fp32; probabilities are rounded to the inputs' type
    before they multiply the values, and so are the gradients of the scores
    before they multiply queries and keys.  Differentiable in the three tensors;
    all sums run in a fixed order.  The backward pass computes all three gradients,
    also where one of them is wanted.
    """
    try:
        if scale is None:
            scale = max(1, query.shape[-1]) ** -0.5
        if window is not None and window < 1:
            raise ValueError(f"window must be positive, got {window}")
        return _attention(query, key, value, offsets, lengths, causal, window or 0, scale, False)[0]
    except Exception:
        _explain(query=query, key=key, value=value)
        _explain(**{n: t for n, t in (("offsets", offsets), ("lengths", lengths)) if t is not None})
        raise


def rotary(query: torch.Tensor, key: Optional[torch.Tensor], positions: torch.Tensor,
           frequencies: torch.Tensor, *, interleaved: bool = False, scale: float = 1.0
           ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Rotary positions of queries and keys, in one launch.

    ``query``: ``[..., length, heads, dim]``; ``key`` the same but for the
    heads, or None.  ``positions`` (int32 or int64): ``[..., length]``, or
    ``[length]`` for all sequences alike.  ``frequencies`` (fp32 or fp64):
    ``[pairs]`` with ``2 * pairs <= dim``, radians a position.  Pair ``i``, the
    elements ``i`` and ``i + pairs`` of a head (``2 i`` and ``2 i + 1`` when
    ``interleaved``), is turned by ``position * frequencies[i]`` and multiplied
    by ``scale``; elements from ``2 * pairs`` on are copied.  Angles are taken in
    64 bits, their cosines and sines, the scaling and the products in fp32, and
    each output is rounded once.

    Returns the two turned tensors, contiguous (None without ``key``).
    Differentiable in ``query`` and ``key``; frequencies that require a gradient
    are refused (NotImplementedError).
    """
    try:
        turned, turned_key = _rotary(query, key, positions, frequencies, interleaved, scale)
    except Exception:
        _explain(query=query, positions=positions, frequencies=frequencies)
        if key is not None:
            _explain(key=key)
        raise
    return turned, turned_key if key is not None else None


def rotary_frequencies(dim: int, base: float = 10000.0, *, stretch: str = "none", factor: float = 1.0,
                       trained_length: Optional[int] = None, fast_turns: float = 32.0,
                       slow_turns: float = 1.0, device="cuda") -> Tuple[torch.Tensor, float]:
    """``(frequencies, scale)`` for ``rotary``: fp64 ``[dim // 2]`` radians a
    position, ``base ** (-2 i / dim)``, and 1.0; with ``stretch`` for contexts
    ``factor`` times longer than the trained ones:

    * ``"linear"``: every frequency is divided by ``factor`` (positions are
      interpolated);
    * ``"base"``: the base grows by ``factor ** (dim / (dim - 2))``, so that the
      slowest pair turns ``factor`` times slower and the fastest stays;
    * ``"ramp"``: pairs that turn ``fast_turns`` times or more within
      ``trained_length`` stay, those with ``slow_turns`` or fewer are divided by
      ``factor``; between them the share that stays grows linearly with the
      pair's number of turns.  (Models trained with a ramp that is linear in the
      pair's index need frequencies of their own.)  ``scale`` is ``0.1
      log(factor) + 1``.
    """
    if dim < 2 or dim % 2:
        raise ValueError(f"dim must be even and positive, got {dim}")
    if not (base > 0.0 and math.isfinite(base)) or not (factor > 0.0 and math.isfinite(factor)):
        raise ValueError(f"base and factor must be positive and finite, got {base} and {factor}")
    exponent = -torch.arange(dim // 2, dtype=torch.float64) * (2.0 / dim)
    scale = 1.0
    if stretch == "base":
        if dim < 4:
            raise ValueError("stretch='base' needs two pairs or more")
        base = base * factor ** (dim / (dim - 2))
    elif stretch not in ("none", "linear", "ramp"):
        raise ValueError(f"stretch must be 'none', 'linear', 'base' or 'ramp', got {stretch!r}")
    frequencies = base ** exponent
    if stretch == "linear":
        frequencies = frequencies / factor
    elif stretch == "ramp":
        if trained_length is None or trained_length < 1:
            raise ValueError("stretch='ramp' needs the trained length")
        if not fast_turns > slow_turns:
            raise ValueError(f"fast_turns must be above slow_turns, got {fast_turns} and {slow_turns}")
        turns = trained_length * frequencies / (2.0 * math.pi)
        keep = ((turns - slow_turns) / (fast_turns - slow_turns)).clamp(0.0, 1.0)
        frequencies = frequencies * (keep + (1.0 - keep) / factor)
        scale = 0.1 * math.log(factor) + 1.0 if factor > 1.0 else 1.0
    return frequencies.to(device), scale


def clip_gradients(gradients: Sequence[torch.Tensor], max_norm: float, *, norm_type: float = 2.0,
                   out: Optional[Sequence[torch.Tensor]] = None) -> torch.Tensor:
    """Scales gradients by ``min(1, max_norm / (norm + 1e-6))``, where ``norm`` is
    the norm of all their elements together, and returns ``norm`` (fp32, one
    element, on the device; nothing waits for it).

    ``gradients``: dense tensors on one device, each fp32, bf16 or fp16; in
    place, or into the tensors of ``out``, of the same shapes and any of the
    three types (gradients accumulated in fp32 go to the parameters' type in
    the same pass).  ``norm_type`` is 2 or infinity (the largest magnitude).
    ``max_norm=math.inf`` only takes the norm (and converts, with ``out``),
    whatever it is.  Squares are summed in fp32 over the elements of one load
    and in fp64 from there on, in a fixed order, products are fp32, and each
    output is rounded once.  With a finite limit a NaN makes the norm and all
    results NaN, and an infinite element makes them 0, its own NaN.
    """
    gradients = list(gradients)
    if not gradients:
        raise ValueError("no gradients")
    if norm_type not in (2, math.inf):
        raise ValueError(f"norm_type must be 2 or infinity, got {norm_type}")
    try:
        out = None if out is None else list(out)
        long = len(gradients) + (len(out) if out is not None else 0) > _LONG_LIST
        if long and _clip_list is not None and not torch.compiler.is_compiling():
            norm = _clip_lists(gradients, out, max_norm, norm_type != 2)
            if norm is not None:
                return norm
        if out is None:
            return _clip_in_place(gradients, max_norm, norm_type != 2)
        return _clip_out(gradients, out, max_norm, norm_type != 2)
    except Exception:
        for t in gradients:
            _explain(gradients=t)
        for t in out if out is not None else ():
            _explain(out=t)
        raise


def clip_grad_norm(parameters: Union[torch.Tensor, Iterable[torch.Tensor]], max_norm: float, *,
                   norm_type: float = 2.0) -> torch.Tensor:
    """``clip_gradients`` of the parameters' ``.grad``, in place, before the
    optimizers step.  Parameters without a gradient are left out, one listed
    twice counts once; without any gradient the norm is 0."""
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    grads = {}
    device = None
    for p in parameters:
        if not isinstance(p, torch.Tensor):
            raise TypeError("parameters must be torch.Tensors")
        device = device or p.device
        if p.grad is not None:
            grads[id(p)] = p.grad
    if not grads:
        if not max_norm >= 0.0:
            raise ValueError(f"max_norm must not be negative, got {max_norm}")
        return torch.zeros((), device=device)
    return clip_gradients(list(grads.values()), max_norm, norm_type=norm_type)
