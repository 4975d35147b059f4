"""CPU tests of attention, rotary positions and clipping: the C ABI's structures
and refusals, the entry points' checks and FakeTensor kernels, frequencies."""
from __future__ import annotations

import ctypes
import importlib.util
import math
import random
import re
from pathlib import Path

import pytest
import torch

import muon_fusion_ascend950_b200 as pkg
from muon_fusion_ascend950_b200 import transformer
from muon_fusion_ascend950_b200.capi import (
    AttentionArgs,
    AttentionGrads,
    ClipTensor,
    RotaryArgs,
    Strides,
    capi,
)

REPO = Path(__file__).resolve().parent.parent
HEADER = REPO / "include" / "muon_train_sm100.h"
BF16, F16, F32, F64, I32, I64 = (torch.bfloat16, torch.float16, torch.float32, torch.float64, torch.int32, torch.int64)


@pytest.fixture(scope="module")
def lib():
    return capi().lib


@pytest.mark.parametrize("cname,struct", [("strides", Strides), ("attention_args", AttentionArgs),
                                          ("attention_grads", AttentionGrads), ("rotary_args", RotaryArgs),
                                          ("clip_tensor", ClipTensor)])
def test_structures_are_the_headers(cname, struct):
    body = re.search(r"typedef struct \{([^}]*)\} muon_train_%s;" % cname, HEADER.read_text()).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    names = []
    for declaration in body.split(";"):
        for part in declaration.split(","):
            found = re.search(r"(\w+)(\[\d+\])?\s*$", part.strip())
            if found:
                names.append(found.group(1))
    assert names == [n for n, _ in struct._fields_]


def test_limits_are_the_headers():
    for name, value in (("HEAD", transformer.MAX_HEAD_DIM), ("ROTARY", transformer.MAX_ROTARY_DIM)):
        assert int(re.search(rf"#define MUON_TRAIN_MAX_{name}_DIM (\d+)", HEADER.read_text()).group(1)) == value


# ------------------------------------------------------------------ C ABI
BUFFER = ctypes.create_string_buffer(256)
HERE = (ctypes.addressof(BUFFER) + 63) // 64 * 64  # an aligned address that no refused call reads


def attention_args(**kw):
    row = Strides(1024, 128, 64)
    a = dict(q=HERE, k=HERE, v=HERE, out=HERE, lse=HERE, q_stride=row, k_stride=row, v_stride=row, batch=1, length=8,
             keys=8, heads=2, kv_heads=1, dim=64, scale=1.0, dtype=1)
    a.update(kw)
    return AttentionArgs(**a)


@pytest.mark.parametrize("kw,rc", [
    (dict(dim=60), -1), (dict(dim=136), -1), (dict(dim=0), -1), (dict(heads=3, kv_heads=2), -1), (dict(kv_heads=0), -1),
    (dict(dtype=0), -1), (dict(dtype=3), -1), (dict(scale=0.0), -1), (dict(scale=math.inf), -1), (dict(scale=math.nan), -1),
    (dict(window=-1), -1), (dict(batch=-1), -1), (dict(length=-1), -1), (dict(keys=1 << 31), -1), (dict(heads=65536), -1),
    (dict(lengths=HERE, keys=9), -1), (dict(offsets=HERE, batch=2), -1), (dict(offsets=HERE, lengths=HERE), -1),
    (dict(offsets=HERE, sequences=-1), -1), (dict(out=None), -1), (dict(lse=None), -1),
    (dict(q=None), -3), (dict(k=HERE + 2), -3), (dict(q_stride=Strides(1024, 130, 64)), -3),
    (dict(v_stride=Strides(1024, 0, 64)), -3), (dict(batch=0), 0), (dict(length=0, q=None, out=None, lse=None), 0)])
def test_attention_refuses_bad_arguments(lib, kw, rc):
    assert lib.muon_train_attention_sm100(ctypes.byref(attention_args(**kw)), None) == rc


def test_attention_backward_refuses_bad_arguments(lib):
    row, a = Strides(1024, 128, 64), attention_args()
    size = lib.muon_train_attention_workspace_bytes(ctypes.byref(a))
    assert size >= 2 * 8 * 4
    assert lib.muon_train_attention_workspace_bytes(ctypes.byref(attention_args(dim=7))) == 0
    assert lib.muon_train_attention_workspace_bytes(None) == 0
    good = dict(grad_out=HERE, grad_out_stride=row, grad_q=HERE, grad_k=HERE, grad_v=HERE, workspace=HERE,
                workspace_bytes=size)
    call = lib.muon_train_attention_backward_sm100
    for kw, rc in ((dict(grad_out=None), -3), (dict(grad_q=None), -1), (dict(grad_k=None), -1), (dict(grad_v=HERE + 4), -1),
                   (dict(workspace=None), -5), (dict(workspace_bytes=size - 1), -5),
                   (dict(grad_out_stride=Strides(1024, 100, 64)), -3)):
        assert call(ctypes.byref(a), ctypes.byref(AttentionGrads(**{**good, **kw})), None) == rc, kw
    assert call(ctypes.byref(a), None, None) == -1
    assert call(None, ctypes.byref(AttentionGrads(**good)), None) == -1
    assert call(ctypes.byref(attention_args(batch=0)), ctypes.byref(AttentionGrads()), None) == 0


def rotary_args(**kw):
    a = dict(positions=HERE, frequencies=HERE, batch=1, length=4, dim=8, pairs=4, position_rows=1, position_bytes=8,
             frequency_bytes=8, scale=1.0, dtype=1)
    a.update(kw)
    args = RotaryArgs(**{k: v for k, v in a.items() if k not in ("x", "y", "heads")})
    for i in range(2):
        args.x[i], args.y[i] = a.get("x", (HERE, HERE))[i], a.get("y", (HERE, HERE))[i]
        args.x_row[i], args.x_head[i], args.heads[i] = 16, 8, a.get("heads", (2, 1))[i]
    return args


@pytest.mark.parametrize("kw,rc", [
    (dict(dim=0), -1), (dict(dim=5000), -1), (dict(pairs=5), -1), (dict(pairs=-1), -1), (dict(dtype=3), -1),
    (dict(position_bytes=2), -1), (dict(frequency_bytes=2), -1), (dict(position_rows=3), -1), (dict(positions=None), -1),
    (dict(frequencies=None), -1), (dict(x=(None, HERE)), -1), (dict(y=(HERE, None)), -1), (dict(heads=(-1, 1)), -1),
    (dict(length=1 << 31), -1), (dict(heads=(1 << 22, 0)), -1), (dict(length=0), 0), (dict(heads=(0, 0)), 0)])
def test_rotary_refuses_bad_arguments(lib, kw, rc):
    assert lib.muon_train_rotary_sm100(ctypes.byref(rotary_args(**kw)), None) == rc
    assert lib.muon_train_rotary_sm100(None, None) == -1


@pytest.mark.parametrize("kw,norm,limit,rc", [
    (dict(count=-1), 2, 1.0, -1), (dict(dtype=3), 2, 1.0, -1), (dict(out_dtype=-1), 2, 1.0, -1), (dict(grad=None), 2, 1.0, -1),
    (dict(out=None), 2, 1.0, -1), (dict(out_dtype=1), 2, 1.0, -1), (dict(), 1, 1.0, -1), (dict(), 2, -1.0, -1),
    (dict(), 2, math.nan, -1), (dict(grad=HERE + 2, out=HERE), 2, 1.0, -3), (dict(out=HERE + 1, out_dtype=1), 2, 1.0, -3),
    (dict(count=1 << 50), 2, 1.0, -1), (dict(), 2, 1.0, -5)])
def test_clip_refuses_bad_arguments(lib, kw, norm, limit, rc):
    t = ClipTensor(**{**dict(grad=HERE, out=HERE, count=4), **kw})
    assert lib.muon_train_clip_sm100(ctypes.byref(t), 1, limit, norm, HERE, None, 0, None) == rc
    assert lib.muon_train_clip_sm100(ctypes.byref(t), 1, limit, norm, None, None, 0, None) == -1
    assert lib.muon_train_clip_sm100(None, 1, 1.0, 2, HERE, None, 0, None) == -1
    assert lib.muon_train_clip_sm100(None, -1, 1.0, 2, HERE, None, 0, None) == -1
    assert lib.muon_train_clip_workspace_bytes(-1) == 0


# ----------------------------------------------------------- entry points
def _fake():
    from torch._subclasses.fake_tensor import FakeTensorMode

    return FakeTensorMode()


def _cuda(*shape, dtype=BF16):
    return torch.empty(shape, dtype=dtype, device="cuda")


def test_entry_points_refuse_what_is_no_cuda_tensor():
    q = torch.zeros(1, 4, 2, 8, dtype=BF16)
    f, at = torch.ones(4, dtype=F64), torch.zeros(1, 4, dtype=I64)
    for wrong, error in ((q, ValueError), ([[0.0]], TypeError), (None, TypeError)):
        with pytest.raises(error):
            pkg.attention(wrong, q, q, scale=1.0)
        with pytest.raises(error):
            pkg.rotary(wrong, None, at, f)
        with pytest.raises(error):
            pkg.clip_gradients([wrong], 1.0)
    with pytest.raises(ValueError):
        pkg.clip_gradients([], 1.0)
    with pytest.raises(ValueError):
        pkg.clip_gradients([q], 1.0, norm_type=3.0)
    with pytest.raises(TypeError):
        pkg.clip_grad_norm([None], 1.0)
    with pytest.raises(ValueError):
        pkg.clip_grad_norm([torch.nn.Parameter(torch.zeros(3))], -1.0)
    assert pkg.clip_grad_norm([torch.nn.Parameter(torch.zeros(3))], 1.0) == 0.0


def attention(q=(2, 6, 4, 64), k=(2, 6, 2, 64), v=None, dtype=BF16, kv_dtype=None, offsets=None, lengths=None,
              index=I32, **kw):
    counts = {n: None if s is None else _cuda(*s, dtype=index) for n, s in (("offsets", offsets), ("lengths", lengths))}
    return pkg.attention(_cuda(*q, dtype=dtype), _cuda(*k, dtype=kv_dtype or dtype), _cuda(*(v or k), dtype=kv_dtype or dtype),
                         **counts, **kw)


@pytest.mark.parametrize("kw,error", [
    (dict(), None), (dict(dtype=F16, causal=True, window=3), None), (dict(k=(2, 9, 2, 64)), None),
    (dict(k=(2, 0, 2, 64)), None), (dict(lengths=(2,)), None), (dict(lengths=(2,), index=I64), None),
    (dict(q=(6, 4, 64), k=(6, 2, 64), offsets=(3,)), None), (dict(q=(6, 4, 64), k=(6, 2, 64), offsets=(1,)), None),
    (dict(dtype=F32), TypeError), (dict(kv_dtype=F16), TypeError), (dict(lengths=(2,), index=F32), TypeError),
    (dict(q=(2, 6, 4, 60), k=(2, 6, 2, 60)), ValueError), (dict(q=(2, 6, 4, 136), k=(2, 6, 2, 136)), ValueError),
    (dict(k=(2, 6, 3, 64)), ValueError), (dict(k=(3, 6, 2, 64)), ValueError), (dict(k=(2, 6, 2, 32)), ValueError),
    (dict(v=(2, 6, 2, 32)), ValueError), (dict(q=(6, 4, 64), k=(6, 2, 64)), ValueError),
    (dict(q=(6, 4, 64), k=(5, 2, 64), offsets=(3,)), ValueError), (dict(offsets=(3,)), ValueError),
    (dict(q=(6, 4, 64), k=(6, 2, 64), offsets=(0,)), ValueError), (dict(q=(6, 4, 64), k=(6, 2, 64), offsets=(3, 1)), ValueError),
    (dict(q=(6, 4, 64), k=(6, 2, 64), offsets=(3,), lengths=(1,)), ValueError), (dict(lengths=(3,)), ValueError),
    (dict(k=(2, 9, 2, 64), lengths=(2,)), ValueError), (dict(window=0), ValueError), (dict(window=-1), ValueError),
    (dict(scale=0.0), ValueError), (dict(scale=-1.0), ValueError), (dict(scale=math.inf), ValueError),
    (dict(scale=math.nan), ValueError), (dict(scale=1e-60), ValueError)], ids=str)
def test_attention_is_checked(kw, error):
    with _fake():
        if error is None:
            out = attention(**kw)
            assert out.shape == kw.get("q", (2, 6, 4, 64)) and out.dtype == kw.get("dtype", BF16)
        else:
            with pytest.raises(error):
                attention(**kw)


def test_attention_refuses_heads_without_elements():
    with _fake(), pytest.raises(ValueError):
        attention(q=(2, 6, 4, 0), k=(2, 6, 2, 0))


@pytest.mark.parametrize("q,k,at,f,kw,error", [
    ((2, 6, 4, 64), (2, 6, 1, 64), (2, 6), 32, {}, None), ((2, 6, 4, 64), None, (6,), 16, dict(interleaved=True), None),
    ((6, 4, 64), None, (6,), 0, {}, None), ((4, 64), (2, 64), (), 1, {}, None), ((2, 3, 6, 1, 7), None, (2, 3, 6), 3, {}, None),
    ((64,), None, (), 1, {}, ValueError), ((2, 6, 4, 64), (2, 5, 1, 64), (2, 6), 32, {}, ValueError),
    ((2, 6, 4, 64), (2, 6, 1, 32), (2, 6), 32, {}, ValueError), ((2, 6, 4, 64), None, (2,), 32, {}, ValueError),
    ((2, 6, 4, 64), None, (2, 1), 32, {}, ValueError), ((2, 6, 4, 64), None, (6,), 33, {}, ValueError),
    ((2, 6, 4, 64), None, (6,), 32, dict(scale=math.inf), ValueError), ((6, 1, 4098), None, (6,), 4, {}, ValueError)], ids=str)
def test_rotary_is_checked(q, k, at, f, kw, error):
    with _fake():
        def call(dtype=F32, key=None, index=I64, frequency=F64):
            return pkg.rotary(_cuda(*q, dtype=dtype), None if k is None else _cuda(*k, dtype=key or dtype),
                              _cuda(*at, dtype=index), _cuda(f, dtype=frequency), **kw)

        if error is not None:
            with pytest.raises(error):
                call()
            return
        turned, turned_key = call()
        assert turned.shape == q and (turned_key is None if k is None else turned_key.shape == k)
        call(F16, None, I32, F32)
        for wrong in (dict(dtype=F64), dict(index=F32), dict(frequency=BF16), *([dict(key=BF16)] if k else [])):
            with pytest.raises(TypeError):
                call(**wrong)


def test_clip_is_checked():
    with _fake():
        g = [_cuda(3, 4, dtype=F32), _cuda(5, dtype=F16)]
        assert pkg.clip_gradients(g, 1.0).shape == ()
        assert pkg.clip_gradients(g, math.inf, norm_type=math.inf, out=[_cuda(3, 4), _cuda(5)]).dtype == F32
        for grads, limit, out in ((g, -1.0, None), (g, math.nan, None), (g, 1.0, g[:1]), (g, 1.0, [g[1], g[0]]), ([], 1.0, None)):
            with pytest.raises(ValueError):
                pkg.clip_gradients(grads, limit, out=out)
        with pytest.raises(TypeError):
            pkg.clip_gradients([_cuda(3, dtype=I64)], 1.0)


def test_lists_are_read_only_where_tensors_are_as_expected():
    """A library that does not find the tensor in torch's objects, or cannot tell,
    is not given lists: calls go through the operator."""
    reads = transformer._library.muon_ascend950_clip_reads
    for t in (torch.zeros(3), torch.zeros(2, 2)[0], torch.nn.Parameter(torch.zeros(1))):
        assert reads(t) == t._cdata
    assert transformer._clip_list is not None and reads(object()) == 0  # too small to hold a tensor

    class Library:
        muon_ascend950_clip_list = muon_ascend950_clip_message = transformer._clip_list

        def __init__(self, reads=None):
            if reads is not None:
                self.muon_ascend950_clip_reads = reads

    class Entry:
        def __init__(self, answer):
            self.answer = answer

        def __call__(self, t):
            return self.answer(t)

    for library in (object(), Library(), Library(Entry(lambda t: 0)), Library(Entry(lambda t: t._cdata + 8))):
        assert transformer._list_entry(library) is None
    assert transformer._list_entry(Library(Entry(lambda t: t._cdata))) is transformer._clip_list


def test_forward_mode_is_refused():
    from torch.autograd import forward_ad

    with _fake():
        q, f, at = _cuda(1, 4, 2, 64), _cuda(32, dtype=F64), _cuda(4, dtype=I64)
        for call in (lambda t: pkg.attention(t, q, q), lambda t: pkg.attention(q, t, q), lambda t: pkg.attention(q, q, t),
                     lambda t: pkg.rotary(t, q, at, f)[0], lambda t: pkg.rotary(q, t, at, f)[1]):
            with pytest.raises(NotImplementedError):
                torch.func.jvp(call, (q.clone(),), (torch.ones_like(q),))
            with forward_ad.dual_level(), torch.no_grad(), pytest.raises(NotImplementedError):
                call(forward_ad.make_dual(q.clone(), torch.ones_like(q)))


def test_rotary_refuses_frequencies_that_want_a_gradient():
    with _fake():
        q, at = _cuda(4, 2, 64, dtype=F32), _cuda(4, dtype=I64)
        f = torch.empty(32, dtype=F64, device="cuda", requires_grad=True)
        for leaf in (q, q.clone().requires_grad_(True)):
            for key in (None, leaf):
                with pytest.raises(NotImplementedError):
                    pkg.rotary(leaf, key, at, f)
                assert pkg.rotary(leaf, key, at, f.detach())[0].requires_grad == leaf.requires_grad
        with torch.no_grad():
            pkg.rotary(q, None, at, f)


def test_fake_backward_kernels():
    with _fake():
        ops = torch.ops.muon_ascend950
        q, k = _cuda(2, 6, 4, 64), _cuda(2, 7, 2, 64)
        out, lse, rest = ops.attention(q, k, k, None, None, True, 0, 1.0, False)
        assert rest.shape == (0,) and ops.attention(q, k, k, None, None, True, 0, 1.0, True)[2].shape == q.shape
        assert lse.shape == (4, 12) and lse.dtype == F32
        grads = ops.attention_backward(out, q, k, k, out, lse, rest, None, None, True, 0, 1.0)
        assert [g.shape for g in grads] == [q.shape, k.shape, k.shape]
        f, at = _cuda(32, dtype=F64), _cuda(6, dtype=I64)
        assert ops.rotary_backward(q, None, at, f, False, 1.0, True)[0].shape == q.shape


def test_rotary_frequencies():
    f, scale = pkg.rotary_frequencies(8, 100.0, device="cpu")
    assert f.dtype == F64 and scale == 1.0
    assert torch.allclose(f, torch.tensor([1.0, 100.0 ** -0.25, 0.1, 100.0 ** -0.75], dtype=F64), rtol=1e-14)
    linear, scale = pkg.rotary_frequencies(8, 100.0, stretch="linear", factor=4.0, device="cpu")
    assert torch.equal(linear, f / 4) and scale == 1.0
    based, scale = pkg.rotary_frequencies(8, 100.0, stretch="base", factor=4.0, device="cpu")
    assert scale == 1.0 and based[0] == 1.0 and abs(float(based[-1] / f[-1]) - 0.25) < 1e-12
    ramp, scale = pkg.rotary_frequencies(64, stretch="ramp", factor=8.0, trained_length=4096, device="cpu")
    plain, _ = pkg.rotary_frequencies(64, device="cpu")
    turns = 4096 * plain / (2 * math.pi)
    assert torch.equal(ramp[turns >= 32], plain[turns >= 32])
    assert torch.allclose(ramp[turns <= 1], plain[turns <= 1] / 8, rtol=1e-14)
    between = (ramp / plain)[(turns > 1) & (turns < 32)]
    assert ((between > 1 / 8) & (between < 1)).all() and (between.diff() < 0).all()
    assert scale == 0.1 * math.log(8.0) + 1.0
    for kw in (dict(dim=7), dict(dim=0), dict(base=0.0), dict(factor=0.0), dict(stretch="other"), dict(stretch="ramp"),
               dict(dim=2, stretch="base", factor=2.0), dict(stretch="ramp", trained_length=10, fast_turns=1.0)):
        with pytest.raises(ValueError):
            pkg.rotary_frequencies(**{**dict(dim=8, device="cpu"), **kw})


def test_measured_cases_stay_in_their_ranges():
    spec = importlib.util.spec_from_file_location("perf_more_operators", REPO / "perf" / "more_operators.py")
    cases = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(cases)
    assert not cases.own
    largest = {op: max(cases.work(c)[what] for c in cases.listed() if c["op"] == op)
               for op, what in (("attention", "flops"), ("rotary", "bytes"), ("clip", "bytes"))}
    for seed in range(150):
        c = cases.draw(random.Random(seed))
        assert cases.work(c)["flops" if c["op"] == "attention" else "bytes"] <= 1.02 * largest[c["op"]]
