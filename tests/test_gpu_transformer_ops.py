"""GPU tests of attention, rotary positions and gradient clipping against their
definitions in 64 bits (on the same device), at the sizes, strides and masks
where they can go wrong.

Tolerances are bounds on rounding, formed in 64 bits from the magnitudes of the
terms: a rounding to a type is off by at most half a step, U = eps / 2, relative
to the value (half of a subnormal where the type has them), and a sum of n fp32
products by (n + a few) * 2^-24 times the sum of their magnitudes.
"""
from __future__ import annotations

import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

F64, F32, BF16, F16 = torch.float64, torch.float32, torch.bfloat16, torch.float16
U = {t: torch.finfo(t).eps / 2 for t in (F32, BF16, F16)}
TINY = {F32: 0.0, BF16: 0.0, F16: 2.0 ** -25}
E32 = 2.0 ** -24
LEAST = 2.0 ** -126


@pytest.fixture(scope="module")
def pkg(cuda_device):
    import muon_fusion_ascend950_b200 as pkg

    return pkg


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(*shape, seed, dtype=F32, std=1.0):
    return torch.randn(*shape, generator=gen(seed), device="cuda").mul_(std).to(dtype)


def near(actual, expected, bound, what=""):
    actual, expected = actual.double(), expected.double()
    assert actual.shape == expected.shape
    assert torch.equal(actual.isnan(), expected.isnan()), what
    over = ((actual - expected).abs() > bound) & ~expected.isnan()
    assert not over.any(), (what, int(over.sum()), over.numel(), over.nonzero()[:4].tolist(), actual[over][:4].tolist(),
                            expected[over][:4].tolist(),
                            torch.as_tensor(bound, device=over.device).expand_as(expected)[over][:4].tolist())


# ================================================================ attention
def sees(length, keys, causal, window):
    """[length, keys]: whether query i sees key j, both counted from the end."""
    behind = torch.arange(length, device="cuda")[:, None] + (keys - length) - torch.arange(keys, device="cuda")
    see = torch.ones_like(behind, dtype=torch.bool)
    if causal:
        see &= behind >= 0
    if window:
        see &= behind.abs() < window
    return see


def one_head(q, k, v, go, see, scale, dtype):
    """(value, bound) of out, dq, dk, dv of one head's sequence, in 64 bits."""
    q, k, v, go = (t.double() for t in (q, k, v, go))
    dim, u, tiny = q.shape[-1], U[dtype], TINY[dtype]
    some = see.any(1, keepdim=True)
    s = torch.where(see, scale * q @ k.T, -math.inf)
    p = torch.where(some, torch.softmax(torch.where(some, s, 0.0), -1), 0.0)
    out = p @ v
    # p's relative error: of s in the exponent (its fp32 sum, its scaling and the row's maximum, and the same of lse),
    # the exponential's own 2 ulp, the sum's; twice, above and below the fraction
    dots = scale * (q.abs() @ k.abs().T)
    big = torch.where(see, dots, 0.0).amax(1, keepdim=True) if k.shape[0] else dots.sum(1, keepdim=True)
    e = 2 * ((dim + 8) * E32 * big + (see.shape[1] / 64 + 64) * E32)
    # p is rounded to the type before it multiplies v: its half step, or half of a subnormal of a p up to 1; below
    # 2^-126 p is no normal fp32 number, and may be taken as 0
    seen = see.double()
    small = (tiny + LEAST) * (seen @ v.abs())
    out_bound = u * out.abs() + tiny + (u + e + 2 * E32) * (p @ v.abs()) + small
    # the gradients: delta comes from the rounded output
    dp = go @ v.T
    delta = (go * out).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    off = (go.abs() * out_bound).sum(-1, keepdim=True) + (2 * dim + 8) * E32 * (go.abs() @ v.abs().T
                                                                               + (go * out).abs().sum(-1, keepdim=True))
    ds_off = p * off + (u + 2 * e) * ds.abs() + LEAST * seen * ((dp - delta).abs() + 1)
    n = max(see.shape)
    grow = (n / 8 + 64) * E32  # sums over keys or queries, in runs of 16 terms at least
    dq, dk, dv = scale * ds @ k, scale * ds.T @ q, p.T @ go
    # u of the operand's rounding, the others' errors, the sum's, and the result's own rounding
    dq_bound = scale * (ds_off + grow * ds.abs()) @ k.abs() + u * dq.abs() + tiny
    dk_bound = scale * (ds_off + grow * ds.abs()).T @ q.abs()
    dv_bound = ((u + 2 * e + grow) * p).T @ go.abs() + (tiny + LEAST) * seen.T @ go.abs()
    return (out, out_bound), (dq, dq_bound), (dk, dk_bound), (dv, dv_bound)


def attention_reference(q, k, v, go, *, causal, window, scale, sequences):
    """Values and bounds of out, dq, dk and dv; `sequences`: (index of the rows
    of q, index of the rows of k) of each sequence."""
    group = q.shape[-2] // k.shape[-2]
    made = [[torch.zeros(t.shape, dtype=F64, device="cuda") for _ in range(2)] for t in (q, q, k, v)]
    for rows, keys in sequences:
        for h in range(q.shape[-2]):
            a = q[rows][:, h], k[keys][:, h // group], v[keys][:, h // group], go[rows][:, h]
            see = sees(a[0].shape[0], a[1].shape[0], causal, window)
            if see.numel() == 0:
                continue
            parts = one_head(*a, see, scale, q.dtype)
            for (value, bound), at, head, part in zip(made, (rows, rows, keys, keys), (h, h, h // group, h // group), parts):
                value[at][:, head] += part[0]
                bound[at][:, head] += part[1]
    for value, bound in made[2:]:
        bound += U[q.dtype] * value.abs() + TINY[q.dtype]
    return made


def attention_inputs(batch, length, keys, heads, kv_heads, dim, dtype, seed, *, fused=False, std=1.0):
    if fused:
        x = randn(batch, length, heads + 2 * kv_heads, dim, seed=seed, dtype=dtype, std=std)
        q, k, v = x.split([heads, kv_heads, kv_heads], dim=2)
    else:
        q = randn(batch, length, heads, dim, seed=seed, dtype=dtype, std=std)
        k = randn(batch, keys, kv_heads, dim, seed=seed + 1, dtype=dtype, std=std)
        v = randn(batch, keys, kv_heads, dim, seed=seed + 2, dtype=dtype)
    return q, k, v, randn(batch, length, heads, dim, seed=seed + 3, dtype=dtype, std=0.1)


def check_attention(pkg, q, k, v, go, *, sequences, causal=False, window=None, scale=None, **kw):
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = pkg.attention(*leaves, causal=causal, window=window, scale=scale, **kw)
    got = [out.detach(), *torch.autograd.grad(out, leaves, go)]
    made = attention_reference(q, k, v, go, causal=causal, window=window, scale=scale or q.shape[-1] ** -0.5,
                               sequences=sequences)
    for name, a, (value, bound) in zip(("out", "dq", "dk", "dv"), got, made):
        assert a.dtype == q.dtype and a.is_contiguous()
        near(a, value, bound, name)
    return got


def whole(batch):
    return [((b,), (b,)) for b in range(batch)]


SHAPES = [  # batch, length, keys, heads, kv_heads, dim
    (1, 1, 1, 1, 1, 64), (2, 33, 33, 4, 4, 64), (1, 128, 128, 2, 1, 128), (3, 129, 129, 3, 1, 128),
    (1, 257, 257, 2, 2, 64), (2, 7, 300, 4, 2, 128), (2, 300, 7, 4, 2, 64), (1, 640, 512, 2, 1, 128),
    (1, 255, 385, 6, 2, 72), (2, 100, 100, 2, 2, 8), (1, 1000, 1000, 2, 1, 120), (1, 1, 777, 8, 1, 128),
    (1, 700, 1, 2, 2, 128)]


@pytest.mark.parametrize("dtype", [BF16, F16], ids=str)
@pytest.mark.parametrize("mask", [(False, None), (True, None), (True, 100), (False, 50), (True, 1)], ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_attention_of_dense_sequences(pkg, shape, mask, dtype):
    """With fewer keys than queries and a causal mask, rows are left empty."""
    q, k, v, go = attention_inputs(*shape, dtype, seed=sum(shape))
    check_attention(pkg, q, k, v, go, sequences=whole(shape[0]), causal=mask[0], window=mask[1])


@pytest.mark.parametrize("dim", [64, 128])
def test_attention_of_long_sequences(pkg, dim):
    q, k, v, go = attention_inputs(1, 4500, 4500, 2, 1, dim, BF16, seed=5, fused=True)
    check_attention(pkg, q, k, v, go, sequences=whole(1), causal=True)
    check_attention(pkg, q, k, v, go, sequences=whole(1), causal=True, window=1000)
    check_attention(pkg, q, k, v, go, sequences=whole(1))


@pytest.mark.parametrize("causal", [False, True])
def test_attention_of_many_tiles(pkg, causal):
    """Many rounds of every ring and barrier, over and over: each run gives the
    same bits, and no wait runs out."""
    from muon_fusion_ascend950_b200.capi import capi

    q, k, v, go = attention_inputs(1, 8200, 8200, 4, 2, 128, BF16, seed=8, fused=True)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    first = None
    for _ in range(12):
        out = pkg.attention(*leaves, causal=causal)
        got = [out.detach(), *torch.autograd.grad(out, leaves, go)]
        first = first or got
        for a, b in zip(got, first):
            assert torch.equal(a, b)
    assert capi().train_device_status(torch.cuda.current_device()) == 0


@pytest.mark.parametrize("dtype", [BF16, F16], ids=str)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("index", [torch.int32, torch.int64], ids=str)
def test_attention_of_padded_sequences(pkg, dtype, causal, index):
    """What padding holds reaches nothing, and its own results are 0."""
    q, k, v, go = attention_inputs(5, 300, 300, 4, 2, 64, dtype, seed=11)
    counts = [300, 0, 1, 129, 256]
    sequences = [((b, slice(0, n)), (b, slice(0, n))) for b, n in enumerate(counts)]
    for b, n in enumerate(counts):
        q[b, n:], k[b, n:], v[b, n:] = math.nan, math.inf, math.nan
        go[b, n:] = math.nan
    lengths = torch.tensor(counts, device="cuda", dtype=index)
    clean = [torch.where(torch.arange(300, device="cuda")[None, :, None, None] < lengths[:, None, None, None], t, 0)
             for t in (q, k, v, go)]
    got = check_attention(pkg, *clean, sequences=sequences, causal=causal, lengths=lengths)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = pkg.attention(*leaves, causal=causal, lengths=lengths)
    for a, b in zip(got, [out.detach(), *torch.autograd.grad(out, leaves, go)]):
        assert torch.equal(a, b)
        for i, n in enumerate(counts):
            assert not b[i, n:].any()
    # lengths beyond the tensors are taken as their ends
    far = torch.tensor([1 << 20, -5, 1, 129, 256], device="cuda", dtype=index)
    assert torch.equal(pkg.attention(*clean[:3], causal=causal, lengths=far), got[0])


@pytest.mark.parametrize("dim,dtype", [(64, F16), (128, BF16), (40, BF16)], ids=str)
@pytest.mark.parametrize("causal,window", [(True, None), (False, None), (True, 64), (False, 3)])
def test_attention_of_packed_sequences(pkg, dim, dtype, causal, window):
    """Sequences of many lengths, empty ones among them, and tokens outside of
    all of them, which may hold anything."""
    ends = [3, 3, 4, 131, 131, 259, 600, 601, 900]
    total = 917
    q, k, v, go = attention_inputs(1, total, total, 4, 2, dim, dtype, seed=21, fused=True)
    for t in (q, k, v, go):
        t[:, :3], t[:, 900:] = 0, 0
    sequences = [((slice(a, b),), (slice(a, b),)) for a, b in zip(ends, ends[1:])]
    offsets = torch.tensor(ends, dtype=torch.int32, device="cuda")
    got = check_attention(pkg, q[0], k[0], v[0], go[0], sequences=sequences, causal=causal, window=window, offsets=offsets)
    for t in (q, k, v, go):
        t[:, :3], t[:, 900:] = math.nan, math.inf
    leaves = [t[0].detach().requires_grad_(True) for t in (q, k, v)]
    out = pkg.attention(*leaves, causal=causal, window=window, offsets=offsets.long())
    for a, b in zip(got, [out.detach(), *torch.autograd.grad(out, leaves, go[0])]):
        assert torch.equal(a, b) and not b[:3].any() and not b[900:].any()


def test_attention_of_many_short_sequences(pkg):
    rng = random.Random(4)
    ends = [0]
    while len(ends) < 700:
        ends.append(ends[-1] + rng.choice([0, 1, 2, 5, 17, 40]))
    total = ends[-1] + 5
    q, k, v, go = attention_inputs(1, total, total, 2, 1, 64, BF16, seed=22)
    go[:, ends[-1]:] = 0
    offsets = torch.tensor(ends, dtype=torch.int32, device="cuda")
    sequences = [((slice(a, b),), (slice(a, b),)) for a, b in zip(ends, ends[1:]) if b > a]
    check_attention(pkg, q[0], k[0], v[0], go[0], sequences=sequences, causal=True, offsets=offsets)


@pytest.mark.parametrize("kv_heads", [1, 2])
@pytest.mark.parametrize("shortest,longest", [(0, 3), (100, 300), (0, 600)])
def test_attention_of_more_sequences_than_a_warp_looks_at(pkg, shortest, longest, kv_heads):
    """1200 sequences, empty ones and ones of more than a tile among them: each
    token's results are those of its sequence among few others."""
    rng = random.Random(5)
    ends = [7]
    while len(ends) < 1201:
        ends.append(ends[-1] + rng.randint(shortest, longest))
    total = ends[-1] + 200
    q, k, v, go = attention_inputs(1, total, total, 2, kv_heads, 64, BF16, seed=24)

    def step(first, last):
        rows = slice(ends[first], ends[last])
        leaves = [t[0, rows].detach().requires_grad_(True) for t in (q, k, v)]
        out = pkg.attention(*leaves, causal=True, offsets=torch.tensor(ends[first:last + 1], device="cuda") - ends[first])
        return [out.detach(), *torch.autograd.grad(out, leaves, go[0, rows])]

    leaves = [t[0].detach().requires_grad_(True) for t in (q, k, v)]
    out = pkg.attention(*leaves, causal=True, offsets=torch.tensor(ends, device="cuda"))
    got = [out.detach(), *torch.autograd.grad(out, leaves, go[0])]
    for t in got:
        assert not t[:7].any() and not t[ends[-1]:].any()
    for first in range(0, 1200, 20):
        for a, b in zip(got, step(first, first + 20)):
            assert torch.equal(a[ends[first]:ends[first + 20]], b)


def test_counts_beyond_32_bits_are_the_tensors_ends(pkg):
    q, k, v, _ = attention_inputs(2, 300, 300, 2, 1, 64, BF16, seed=25)
    most = torch.iinfo(torch.int64).max
    for far in (most, (1 << 32) + 5, 1 << 31):
        lengths = torch.tensor([far, 200], device="cuda")
        clear = torch.tensor([300, 200], device="cuda")
        assert torch.equal(pkg.attention(q, k, v, lengths=lengths), pkg.attention(q, k, v, lengths=clear))
        offsets = torch.tensor([-far, 100, far], device="cuda")
        clear = torch.tensor([0, 100, 300], device="cuda")
        assert torch.equal(pkg.attention(q[0], k[0], v[0], offsets=offsets),
                           pkg.attention(q[0], k[0], v[0], offsets=clear))


def test_attention_takes_any_offsets(pkg):
    """Offsets are not looked at on the host: ends outside of the tensor are
    taken as its ends, descending ones make results void, but no access leaves
    the tensors."""
    q, k, v, go = attention_inputs(1, 300, 300, 2, 1, 64, BF16, seed=23)
    whole_row = pkg.attention(q[0], k[0], v[0], causal=True, offsets=torch.tensor([0, 300], device="cuda"))
    far = pkg.attention(q[0], k[0], v[0], causal=True, offsets=torch.tensor([-7, 1 << 20], device="cuda"))
    assert torch.equal(whole_row, far)
    for bad in ([300, 0], [50, 20, 290, 100], [-100, -50], [400, 500, 600], [0, 1 << 30, 3]):
        leaves = [t[0].detach().requires_grad_(True) for t in (q, k, v)]
        out = pkg.attention(*leaves, causal=True, offsets=torch.tensor(bad, device="cuda", dtype=torch.int32))
        torch.autograd.grad(out, leaves, go[0])
    torch.cuda.synchronize()
    none = pkg.attention(q[0], k[0], v[0], offsets=torch.tensor([0], device="cuda"))
    assert not none.any()


def test_attention_of_nothing(pkg):
    for batch, length, keys in ((0, 5, 5), (2, 0, 7), (2, 7, 0), (1, 0, 0)):
        q, k, v, go = attention_inputs(batch, length, keys, 2, 1, 64, BF16, seed=24)
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        out = pkg.attention(*leaves)
        grads = torch.autograd.grad(out, leaves, go)
        assert out.shape == q.shape and not out.any()
        assert all(g.shape == t.shape and not g.any() for g, t in zip(grads, leaves))


def test_attention_reads_slices_and_other_layouts(pkg):
    """Slices in place, what TMA cannot read (odd strides, transposed heads,
    expanded gradients) through a copy: the same bits."""
    q, k, v, go = attention_inputs(2, 150, 150, 4, 2, 64, BF16, seed=25)
    def grads(q, k, v, go):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        out = pkg.attention(*leaves, causal=True)
        return [out.detach(), *torch.autograd.grad(out, leaves, go)]

    want = grads(q, k, v, go)
    def wide(t):
        return torch.cat([t, t], -1)[..., :t.shape[-1]]

    def turned(t):  # [batch, heads, length, dim] in memory
        return t.transpose(1, 2).contiguous().transpose(1, 2)

    def odd(t):  # elements from an odd address on
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:]
        return flat.view(t.shape).copy_(t)

    def inner(t):  # the head's elements apart
        return t.transpose(-1, -2).contiguous().transpose(-1, -2)

    for change in (wide, turned, odd, inner):
        for a, b in zip(grads(*(change(t) for t in (q, k, v, go))), want):
            assert torch.equal(a, b)
    ones = torch.ones((), dtype=BF16, device="cuda")
    for a, b in zip(grads(q, k, v, ones.expand(q.shape)), grads(q, k, v, torch.ones_like(q))):
        assert torch.equal(a, b)
    shared = k[:, :1].expand(k.shape)  # the same keys again and again
    for a, b in zip(grads(q, shared, v, go), grads(q, shared.contiguous(), v, go)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype,std", [(F16, 1e-4), (F16, 30.0), (BF16, 1e-20), (BF16, 1e15)], ids=str)
def test_attention_gradients_of_any_size(pkg, dtype, std):
    """Small gradients are not lost below fp16's range, large ones not above it."""
    q, k, v, go = attention_inputs(1, 400, 400, 2, 1, 64, dtype, seed=26)
    go = (go.float() * 10 * std).to(dtype)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    got = torch.autograd.grad(pkg.attention(*leaves, causal=True), leaves, go)
    made = attention_reference(q, k, v, go, causal=True, window=None, scale=0.125, sequences=whole(1))
    for a, (value, bound) in zip(got, made[1:]):
        near(a, value, bound)


def test_attention_of_extreme_scores(pkg):
    """Scores of hundreds, rows that look at one key only, and the type's
    largest values where the mask hides them."""
    q, k, v, go = attention_inputs(1, 260, 260, 2, 2, 64, BF16, seed=27, std=6.0)
    check_attention(pkg, q, k, v, go, sequences=whole(1), causal=True, scale=1.0)
    low = torch.finfo(BF16).min
    k[:, 200:] = low
    out = pkg.attention(q, k, v, causal=True)
    want = pkg.attention(q[:, :200], k[:, :200], v[:, :200], causal=True)
    assert torch.equal(out[:, :200], want)


def test_attention_keeps_nan_where_it_is_seen(pkg):
    q, k, v, go = attention_inputs(2, 200, 200, 2, 1, 64, BF16, seed=28)
    q[0, 5, 1] = math.nan
    out = pkg.attention(q, k, v, causal=True)
    bad = torch.zeros(2, 200, 2, dtype=torch.bool, device="cuda")
    bad[0, 5, 1] = True
    assert torch.equal(out.isnan().all(-1), bad) and torch.equal(out.isnan().any(-1), bad)


def test_attention_against_differences(pkg):
    """The gradient along a direction against the difference of the formula's
    loss: of order h^2 apart, and by the gradient's own rounding."""
    q, k, v, go = attention_inputs(1, 70, 70, 2, 1, 64, F16, seed=29)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(pkg.attention(*leaves, causal=True), leaves, go)
    see = sees(70, 70, True, None)

    def loss(q, k, v):
        s = torch.einsum("blhd,bkhd->bhlk", q, k.repeat_interleave(2, 2)) / 8
        p = torch.softmax(s.masked_fill(~see, -math.inf), -1)
        return (torch.einsum("bhlk,bkhd->blhd", p, v.repeat_interleave(2, 2)) * go.double()).sum()

    made = attention_reference(q, k, v, go, causal=True, window=None, scale=0.125, sequences=whole(1))
    h = 1e-4
    for i in range(3):
        d = randn(*leaves[i].shape, seed=40 + i, dtype=F64)
        ends = []
        for sign in (1, -1):
            moved = [t.double() for t in (q, k, v)]
            moved[i] = moved[i] + sign * h * d
            ends.append(loss(*moved))
        slope = float((ends[0] - ends[1]) / (2 * h))
        bound = float((made[i + 1][1] * d.abs()).sum()) + 1e-4 * abs(slope) + 1e-5
        assert abs(float((grads[i].double() * d).sum()) - slope) <= bound


def test_attention_gives_gradients_where_asked(pkg):
    q, k, v, go = attention_inputs(1, 140, 140, 2, 1, 64, BF16, seed=30)
    every = check_attention(pkg, q, k, v, go, sequences=whole(1))[1:]
    for i in range(3):
        leaves = [t.detach().requires_grad_(j == i) for j, t in enumerate((q, k, v))]
        out = pkg.attention(*leaves)
        assert torch.equal(torch.autograd.grad(out, leaves[i], go)[0], every[i])
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = pkg.attention(*leaves)
    with pytest.raises(NotImplementedError):
        torch.autograd.grad(out, leaves, go, create_graph=True)
    out = pkg.attention(*leaves)
    out.backward(go, retain_graph=True)
    out.backward(go)
    for t, g in zip(leaves, every):
        assert torch.equal(t.grad, g + g)
    with pytest.raises(RuntimeError):
        out.backward(go)


@pytest.mark.parametrize("dtype", [BF16, F16], ids=str)
@pytest.mark.parametrize("length,keys,causal,window", [(300, 200, True, None), (300, 7, True, 3), (513, 300, False, 20),
                                                       (700, 1, True, None), (256, 128, True, None)])
def test_rows_that_see_nothing_reach_no_gradient(pkg, length, keys, causal, window, dtype):
    """Queries before the first key's place: whatever they and their gradients hold."""
    q, k, v, go = attention_inputs(2, length, keys, 4, 2, 64, dtype, seed=34)
    blind = ~sees(length, keys, causal, window).any(1)
    assert blind.any() and not blind.all()
    q[:, blind], go[:, blind] = 0, 0
    sequences = whole(2)
    got = check_attention(pkg, q, k, v, go, sequences=sequences, causal=causal, window=window)
    for bad in (math.nan, math.inf):
        q[:, blind], go[:, blind] = bad, -bad
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        out = pkg.attention(*leaves, causal=causal, window=window)
        for a, b in zip(got, [out.detach(), *torch.autograd.grad(out, leaves, go)]):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype,largest", [(F16, 65504.0), (BF16, 3e38)], ids=str)
@pytest.mark.parametrize("packed", [False, True])
def test_attention_gradients_whatever_finite_values_padding_holds(pkg, dtype, largest, packed):
    """The same bits with zeros and with the type's largest values in tokens that
    do not count."""
    counts = [300, 0, 1, 129, 256]
    q, k, v, go = attention_inputs(5, 300, 300, 4, 2, 64, dtype, seed=31)
    counted = torch.arange(300, device="cuda") < torch.tensor(counts, device="cuda")[:, None]
    kw = {"lengths": torch.tensor(counts, device="cuda")}
    if packed:  # the tokens of one sequence, between those of none
        q, k, v, go = (t.flatten(0, 1) for t in (q, k, v, go))
        counted = torch.arange(1500, device="cuda")
        counted = (counted >= 3) & (counted < 1300)
        kw = {"offsets": torch.tensor([3, 260, 260, 700, 1300], device="cuda")}
    results = []
    for fill in (0.0, largest, -largest):
        held = [torch.where(counted[..., None, None], t, fill).to(dtype) for t in (q, k, v, go)]
        leaves = [t.requires_grad_(True) for t in held[:3]]
        out = pkg.attention(*leaves, causal=True, **kw)
        results.append([out.detach(), *torch.autograd.grad(out, leaves, held[3])])
    for other in results[1:]:
        for a, b in zip(other, results[0]):
            assert torch.equal(a, b)


def check_fp16_gradients(pkg, q, k, v, go, sequences, causal, **kw):
    """ds is held in fp16 under powers of two that bring a bound B on a row's
    (dq) or a key's (dk) elements to 2^14 at least; an element below fp16's
    normal range is then off by half a subnormal, 2^-25, which is 2^-39 of B.
    For dq B is |dout_i| max_j |v_j| + |delta_i|, for dk max_i |dout_i| |v_j| +
    max_i |delta_i|, over the sequence and the heads that share the key head."""
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = pkg.attention(*leaves, causal=causal, **kw)
    got = torch.autograd.grad(out, leaves, go)
    scale, group = q.shape[-1] ** -0.5, q.shape[-2] // k.shape[-2]
    made = attention_reference(q, k, v, go, causal=causal, window=None, scale=scale, sequences=sequences)
    # the reference's bound is linear in what a product's terms are off by: add theirs
    for rows, keys in sequences:
        for h in range(k.shape[-2]):
            vn = v[keys][:, h].double().norm(dim=-1)
            heads = range(h * group, (h + 1) * group)
            gn = [go[rows][:, i].double().norm(dim=-1) for i in heads]
            delta = [(go[rows][:, i].double() * made[0][0][rows][:, i]).sum(-1).abs() for i in heads]
            most, most_delta = max(g.max() for g in gn), max(d.max() for d in delta)
            see = sees(len(gn[0]), len(vn), causal, None).double()
            for i, g, d in zip(heads, gn, delta):
                made[1][1][rows][:, i] += 2.0 ** -39 * scale * (g * vn.max() + d)[:, None] * (see @ k[keys][:, h].abs().double())
                made[2][1][keys][:, h] += 2.0 ** -39 * scale * (most * vn + most_delta)[:, None] * (
                    see.T @ q[rows][:, i].abs().double())
    for name, a, (value, bound) in zip(("dq", "dk", "dv"), got, made[1:]):
        near(a, value, bound, name)


@pytest.mark.parametrize("causal", [False, True])
def test_fp16_gradients_of_sequences_and_heads_of_different_sizes(pkg, causal):
    """Values and gradients that differ by 10^3 to 10^5 between sequences and
    heads: none is lost in the others' range."""
    q, k, v, go = attention_inputs(4, 1500, 1500, 4, 2, 64, F16, seed=32)
    v[0, :, 1] *= 2000.0
    v[3, :, 1] *= 2000.0
    go *= 0.2
    go[1] *= 1e4
    go[:, :, 2] *= 0.01
    v[2] *= 0.01
    check_fp16_gradients(pkg, q, k, v, go, whole(4), causal)
    offsets = torch.tensor([0, 1500, 1700, 4500, 6000], device="cuda")
    parts = [((slice(a, b),), (slice(a, b),)) for a, b in zip(offsets.tolist(), offsets.tolist()[1:])]
    check_fp16_gradients(pkg, *(t.flatten(0, 1) for t in (q, k, v, go)), parts, causal, offsets=offsets)


@pytest.mark.parametrize("kv_heads", [1, 2])
def test_fp16_gradients_of_more_sequences_than_a_warp_looks_at(pkg, kv_heads):
    """Each token's results are those of its sequence among few others, which
    are larger or smaller; offsets that descend leave no tensor."""
    rng = random.Random(6)
    ends = [7]
    while len(ends) < 401:
        ends.append(ends[-1] + rng.choice([0, 1, rng.randint(100, 300)]))
    total = ends[-1] + 200
    q, k, v, go = attention_inputs(1, total, total, 4, kv_heads, 64, F16, seed=36)
    for a, b in zip(ends, ends[1:]):
        v[0, a:b] *= rng.choice([1e-2, 1.0, 1e3])
        go[0, a:b] *= rng.choice([1e-2, 1.0, 10.0])

    def step(first, last):
        rows = slice(ends[first], ends[last])
        leaves = [t[0, rows].detach().requires_grad_(True) for t in (q, k, v)]
        out = pkg.attention(*leaves, causal=True, window=200,
                            offsets=torch.tensor(ends[first:last + 1], device="cuda") - ends[first])
        return [out.detach(), *torch.autograd.grad(out, leaves, go[0, rows])]

    leaves = [t[0].detach().requires_grad_(True) for t in (q, k, v)]
    out = pkg.attention(*leaves, causal=True, window=200, offsets=torch.tensor(ends, device="cuda"))
    got = [out.detach(), *torch.autograd.grad(out, leaves, go[0])]
    for t in got:
        assert not t[:7].any() and not t[ends[-1]:].any()
    for first in range(0, 400, 10):
        for a, b in zip(got, step(first, first + 10)):
            assert torch.equal(a[ends[first]:ends[first + 10]], b)
    for bad in ([300, 0], [50, 20, 290, 100], [-100, -50], [total, total + 100], [0, 1 << 30, 3]):
        out = pkg.attention(*leaves, causal=True, offsets=torch.tensor(bad, device="cuda"))
        torch.autograd.grad(out, leaves, go[0])
    torch.cuda.synchronize()


def test_fp16_gradients_beside_single_large_rows(pkg):
    """One token of a sequence with large values, another with a large gradient."""
    q, k, v, go = attention_inputs(2, 1200, 1200, 4, 2, 128, F16, seed=33)
    go *= 0.5
    v[0, 700] *= 1000.0
    go[1, 300] *= 1000.0
    check_fp16_gradients(pkg, q, k, v, go, whole(2), True)
    lengths = torch.tensor([701, 1111], device="cuda")
    go[0, 701:], go[1, 1111:] = 0, 0
    check_fp16_gradients(pkg, q, k, v, go, [((b, slice(0, n)), (b, slice(0, n))) for b, n in enumerate(lengths.tolist())],
                         False, lengths=lengths)


# =================================================================== rotary
def rotary_reference(x, positions, frequencies, interleaved, scale, sign=1.0):
    """(value, bound) in 64 bits."""
    r, dtype = 2 * frequencies.shape[0], x.dtype
    angle = positions.double()[..., None, None] * frequencies.double()
    c, s = scale * torch.cos(angle), sign * scale * torch.sin(angle)
    t = x.double()
    a, b = (t[..., 0:r:2], t[..., 1:r:2]) if interleaved else (t[..., :r // 2], t[..., r // 2:r])
    value, bound = t.clone(), torch.zeros_like(t)
    # cosine and sine within 2^-21 of their largest (the rounded angle, the function's 2 ulp, the scaling), two products
    off = abs(scale) * 2.0 ** -21 * (a.abs() + b.abs())
    for part, v in (((slice(0, r, 2) if interleaved else slice(0, r // 2)), a * c - b * s),
                    ((slice(1, r, 2) if interleaved else slice(r // 2, r)), b * c + a * s)):
        value[..., part] = v
        bound[..., part] = off + U[dtype] * v.abs() + TINY[dtype]
    return value, bound


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("lead,heads,kv_heads,dim,rotated", [
    ((1,), 1, 1, 64, 64), ((4, 1), 16, 4, 128, 128), ((2, 37), 3, 1, 80, 48), ((3, 5, 7), 2, 2, 64, 2), ((611,), 5, 5, 6, 4),
    ((2, 9), 3, 1, 7, 6), ((2, 100), 8, 2, 100, 50), ((130,), 2, 1, 256, 256), ((1, 33), 1, 1, 2048, 2048), ((4,), 2, 1, 64, 0),
    ((2, 513), 12, 12, 72, 24)], ids=str)
def test_rotary(pkg, lead, heads, kv_heads, dim, rotated, interleaved, dtype):
    q, k = randn(*lead, heads, dim, seed=1, dtype=dtype), randn(*lead, kv_heads, dim, seed=2, dtype=dtype)
    positions = torch.randint(0, 10_000_000, lead, generator=gen(3), device="cuda")
    frequencies = 10000.0 ** -(torch.arange(rotated // 2, dtype=F64, device="cuda") / max(1, rotated // 2))
    grads = [randn(*t.shape, seed=4 + i, dtype=dtype) for i, t in enumerate((q, k))]
    leaves = [t.detach().requires_grad_(True) for t in (q, k)]
    out = pkg.rotary(*leaves, positions, frequencies, interleaved=interleaved, scale=1.25)
    back = torch.autograd.grad(out, leaves, grads)
    for t, g, o, d in zip((q, k), grads, out, back):
        near(o, *rotary_reference(t, positions, frequencies, interleaved, 1.25))
        near(d, *rotary_reference(g, positions, frequencies, interleaved, 1.25, -1.0))
        assert torch.equal(o[..., rotated:], t[..., rotated:]) and o.is_contiguous()
    # a tensor alone, in other layouts: the same bits
    wide = torch.cat([q, q], -1)[..., :dim]
    odd = torch.empty(q.numel() + 1, dtype=dtype, device="cuda")[1:].view(q.shape).copy_(q)
    inner = q.transpose(-1, -2).contiguous().transpose(-1, -2)
    for x in (q, wide, odd, inner):
        alone, none = pkg.rotary(x, None, positions.int(), frequencies, interleaved=interleaved, scale=1.25)
        assert none is None
        near(alone, *rotary_reference(q, positions, frequencies, interleaved, 1.25))
        assert torch.equal(alone, out[0])


def test_rotary_of_shared_positions_and_slices(pkg):
    x = randn(3, 40, 12, 64, seed=6, dtype=BF16)
    q, k, _ = x.split([8, 2, 2], dim=2)
    f, scale = pkg.rotary_frequencies(64)
    at = torch.arange(40, device="cuda")
    a = pkg.rotary(q, k, at, f)
    b = pkg.rotary(q.contiguous(), k.contiguous(), at.expand(3, 40), f.float())
    for i in range(2):
        near(a[i], *rotary_reference((q, k)[i], at.expand(3, 40), f, False, 1.0))
        near(b[i], *rotary_reference((q, k)[i], at.expand(3, 40), f.float(), False, 1.0))
    assert scale == 1.0
    # gradients of one of the two
    for i in range(2):
        leaves = [t.detach().requires_grad_(j == i) for j, t in enumerate((q, k))]
        g = randn(*leaves[i].shape, seed=7, dtype=BF16)
        near(torch.autograd.grad(pkg.rotary(*leaves, at, f)[i], leaves[i], g)[0],
             *rotary_reference(g, at.expand(3, 40), f, False, 1.0, -1.0))


def test_rotary_turns_back(pkg):
    """A turn and its gradient's turn give the input again; scores depend on
    the distance of positions only."""
    q = randn(1, 50, 2, 64, seed=8)
    f, _ = pkg.rotary_frequencies(64)
    at = torch.arange(50, device="cuda") + 5_000_000
    leaf = q.detach().requires_grad_(True)
    out, _ = pkg.rotary(leaf, None, at, f)
    back = torch.autograd.grad(out, leaf, out.detach())[0]
    near(back, q, 2.0 ** -19 * (q.abs() + q.roll(32, -1).abs()))
    first, far = (torch.einsum("blhd,bmhd->bhlm", o.double(), o.double())
                  for o in (pkg.rotary(q, None, at - 5_000_000, f)[0], out.detach()))
    # both factors within 2^-21 of their pair's magnitude, in 64 products
    off = 4 * 2.0 ** -21 * torch.einsum("blhd,bmhd->bhlm", *[q.double().abs() + q.double().roll(32, -1).abs()] * 2)
    near(far, first, off)


def test_rotary_of_nothing(pkg):
    f = torch.ones(4, dtype=F64, device="cuda")
    for shape in ((0, 5, 2, 8), (2, 0, 2, 8), (2, 3, 0, 8)):
        x = torch.zeros(shape, device="cuda", dtype=BF16)
        out, _ = pkg.rotary(x, None, torch.zeros(shape[:2], dtype=torch.int64, device="cuda"), f)
        assert out.shape == x.shape


# ================================================================= clipping
def clip_reference(grads, max_norm, norm_type):
    flat = torch.cat([g.detach().double().flatten() for g in grads]) if grads else torch.zeros(0)
    norm = flat.norm(norm_type) if flat.numel() else torch.zeros((), dtype=F64, device="cuda")
    c = (max_norm / (norm + 1e-6)).clamp(max=1.0)
    return norm, [g.double() * c for g in grads]


def check_clip(pkg, grads, max_norm, *, norm_type=2.0, out_dtype=None):
    norm, want = clip_reference(grads, max_norm, norm_type)
    out = None if out_dtype is None else [torch.full_like(g, 7.0, dtype=out_dtype) for g in grads]
    kept = [g.clone() for g in grads]
    got = pkg.clip_gradients(grads, max_norm, norm_type=norm_type, out=out)
    assert got.shape == () and got.dtype == F32
    # up to eight squares are added up in fp32 (an error of each square and of each addition on the way: 8 * 2^-24 of the
    # sum at most, half of it in the root), the rest in 64 bits, and the root is rounded once
    near(got, norm, (5 + 1e-6) * E32 * norm.abs() + 2.0 ** -150)
    for g, k, o, w in zip(grads, kept, out or grads, want):
        # the factor is rounded to fp32, so is the product, then the result
        near(o, w, (U[o.dtype] + 2.1 * E32) * w.abs() + TINY[o.dtype] + 2.0 ** -149)
        if out is not None:
            assert torch.equal(g, k)
    return got


def some_grads(sizes, dtypes, seed, std=1e-2, shift=0):
    grads = []
    for i, n in enumerate(sizes):
        dtype = dtypes[i % len(dtypes)]
        grads.append(randn(n + shift, seed=seed + i, dtype=dtype, std=std)[shift:])
    return grads


@pytest.mark.parametrize("norm_type", [2.0, math.inf])
@pytest.mark.parametrize("out_dtype", [None, F32, BF16, F16], ids=str)
@pytest.mark.parametrize("shift", [0, 1, 3])
@pytest.mark.parametrize("sizes", [[1], [1000], [0, 5, 0], [8191, 64, 1, 100003], [3] * 70, [257] * 300,
                                   [3_000_001, 17, 2_000_000]], ids=lambda s: f"{len(s)}x{s[0]}")
def test_clip(pkg, sizes, shift, out_dtype, norm_type):
    for dtypes in ([F32], [BF16, F32, F16]):
        for limit in (1e-3, 1e6):
            check_clip(pkg, some_grads(sizes, dtypes, seed=50, shift=shift), limit, norm_type=norm_type, out_dtype=out_dtype)


@pytest.mark.parametrize("norm_type", [2.0, math.inf])
def test_clip_of_more_tensors_than_a_launch_takes(pkg, norm_type):
    for sizes in ([65, 0] * 600, [2] * 2500, [300] * 1025):
        grads = some_grads(sizes, [F32, BF16], seed=50)
        check_clip(pkg, grads, 1e-3, norm_type=norm_type, out_dtype=BF16)
        check_clip(pkg, grads, 1e-3, norm_type=norm_type)


@pytest.mark.parametrize("elements", [1, 2 ** 18 - 3, 2 ** 18, 2 ** 18 + 1, 2 ** 18 + 70000])
def test_clip_in_one_launch_or_two(pkg, elements):
    for parts in (1, 3, 64, 65):
        if elements >= parts:
            sizes = [elements // parts] * (parts - 1) + [elements - elements // parts * (parts - 1)]
            check_clip(pkg, some_grads(sizes, [BF16], seed=51), 1e-3)


def test_clip_of_shapes_and_layouts(pkg):
    x = randn(40, 30, seed=60)
    grads = [x, randn(30, 50, seed=61).T, randn(2, 3, 4, 5, seed=62).to(memory_format=torch.channels_last), randn(1, seed=63)[0]]
    check_clip(pkg, [g.clone(memory_format=torch.preserve_format) for g in grads], 0.5)
    check_clip(pkg, grads, 0.5, out_dtype=BF16)
    assert not pkg.clip_gradients([torch.zeros(5, device="cuda")], 1.0).any()


def test_clip_of_values_of_any_size(pkg):
    """Squares beyond fp32's range on both sides; what is no number stays none."""
    for std in (1e30, 1e-30):
        check_clip(pkg, some_grads([5000, 17], [F32, BF16], seed=64, std=std), 1.0)
    for dtype in (F32, BF16, F16):
        g = randn(10000, seed=65, dtype=dtype)
        g[7777] = math.nan
        for norm_type in (2.0, math.inf):
            h = g.clone()
            assert pkg.clip_gradients([h], 1.0, norm_type=norm_type).isnan() and h.isnan().all()
        g[7777] = -math.inf
        for norm_type in (2.0, math.inf):
            h = g.clone()
            assert pkg.clip_gradients([h], 1.0, norm_type=norm_type) == math.inf
            assert h[7777].isnan() and not h.nan_to_num(0.0).any()
    g = randn(1000, seed=66)
    kept = g.clone()
    norm = pkg.clip_gradients([g], math.inf)
    assert torch.equal(g, kept) and norm > 0
    pkg.clip_gradients([g], 0.0)
    assert not g.any()


@pytest.mark.parametrize("norm_type", [2.0, math.inf])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("sizes", [[1000, 7], [2 ** 18, 1001], [50] * 40, [300] * 1100], ids=lambda s: f"{len(s)}x{s[0]}")
def test_without_a_limit_clipping_only_takes_the_norm(pkg, sizes, bad, norm_type):
    """Whatever the norm is: one launch and two, short lists and long ones."""
    grads = some_grads(sizes, [F32, BF16, F16], seed=73)
    grads[-1][5] = bad
    kept = [g.clone() for g in grads]
    norms = [pkg.clip_gradients(grads, math.inf, norm_type=norm_type)]
    for out_dtype in (F32, BF16):
        out = [torch.full_like(g, 7.0, dtype=out_dtype) for g in grads]
        norms.append(pkg.clip_gradients(grads, math.inf, norm_type=norm_type, out=out))
        for o, k in zip(out, kept):
            assert torch.equal(o.nan_to_num(nan=-3.0), k.to(out_dtype).nan_to_num(nan=-3.0))
    for g, k in zip(grads, kept):
        assert torch.equal(g.nan_to_num(nan=-3.0), k.nan_to_num(nan=-3.0))
    for norm in norms:
        assert norm.isnan() if math.isnan(bad) else norm == math.inf


def test_clip_of_parameters(pkg):
    a, b, c = (torch.nn.Parameter(torch.zeros(50, 20, device="cuda")) for _ in range(3))
    a.grad, b.grad = randn(50, 20, seed=67), randn(50, 20, seed=68)
    norm, want = clip_reference([a.grad, b.grad], 1.0, 2.0)
    version = a.grad._version
    got = pkg.clip_grad_norm([a, b, c, a], 1.0)
    near(got, norm, E32 * norm * 1.01)
    for p, w in zip((a, b), want):
        near(p.grad, w, 2.1 * E32 * w.abs() + E32 * w.abs())
    assert c.grad is None and a.grad._version > version
    assert pkg.clip_grad_norm([c], 1.0) == 0.0 and pkg.clip_grad_norm(a, math.inf) > 0


def test_clip_goes_through_the_operator_where_something_listens(pkg):
    """Python's lists are read directly; dispatch modes, compilation and other
    tensor types see the operator, with the same results."""
    from torch.utils._python_dispatch import TorchDispatchMode

    seen = []

    class Listen(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(func)
            return func(*args, **(kwargs or {}))

    g = some_grads([1000, 17] * 20, [BF16, F32], seed=72)
    direct, listened, compiled = ([t.clone() for t in g] for _ in range(3))
    norms = [pkg.clip_gradients(direct, 0.1)]
    assert not seen
    with Listen():
        norms.append(pkg.clip_gradients(listened, 0.1))
    assert torch.ops.muon_ascend950.clip_gradients_.default in seen
    norms.append(torch.compile(lambda *t: pkg.clip_gradients(list(t), 0.1), backend="aot_eager", fullgraph=True)(*compiled))
    for a, b, c in zip(direct, listened, compiled):
        assert torch.equal(a, b) and torch.equal(a, c)
    assert norms[0] == norms[1] == norms[2]
    buffers = [torch.nn.Buffer(t.clone()) for t in g]  # not of the type torch.Tensor itself
    assert pkg.clip_gradients(buffers, 0.1) == norms[0] and torch.equal(buffers[0], direct[0])
    out = [torch.empty_like(t) for t in g]
    assert pkg.clip_gradients(tuple(g), 0.1, out=tuple(out)) == norms[0] and torch.equal(out[1], direct[1])
    for wrong, error in ((g[0].cpu(), ValueError), (g[0].long(), TypeError), (3, TypeError), (None, TypeError),
                         (g[1], ValueError), (g[0].clone().requires_grad_(True), ValueError)):
        for grads in ([wrong] + g, g + [wrong], [g[1], wrong]):
            with pytest.raises(error):
                pkg.clip_gradients(grads, 1.0)
    for out in ([], g[:39], g[:-1] + [g[0]], [torch.empty_like(t)[:5] for t in g]):
        with pytest.raises(ValueError):
            pkg.clip_gradients(g, 1.0, out=out)
    with pytest.raises(ValueError):
        pkg.clip_gradients(g, -1.0)


@pytest.mark.parametrize("count", [1, 40])
def test_clipping_in_place_leaves_lazy_clones_alone(pkg, count):
    """A clone that shares its memory until one of the two is written."""
    base = [randn(500, seed=74 + i) for i in range(count)]
    kept = [t.clone() for t in base]
    clones = [torch._lazy_clone(t) for t in base]
    norm, want = clip_reference(kept, 0.5, 2.0)
    near(pkg.clip_gradients(base, 0.5), norm, 6 * E32 * norm)
    for t, clone, k, w in zip(base, clones, kept, want):
        near(t, w, 3.2 * E32 * w.abs())
        assert torch.equal(clone, k)
    # parts of one buffer, and outputs that are the gradients themselves
    flat = randn(1000, seed=75)
    kept, clone = flat.clone(), torch._lazy_clone(flat)
    parts = list(flat.split(1000 // (2 * count)))
    norm, want = clip_reference([kept], 0.5, 2.0)
    pkg.clip_gradients(parts, 0.5, out=parts)
    near(flat, want[0], 3.2 * E32 * want[0].abs())
    assert torch.equal(clone, kept)


def test_clip_refuses_memory_that_would_be_scaled_twice(pkg):
    g = randn(100, seed=69)
    for grads, out in (([g, g], None), ([g[:60], g[40:]], None), ([g, randn(100, seed=70)], [g, g]),
                       ([g, randn(100, seed=70)], [torch.empty_like(g), g]), ([g[:50]], [g[1:51]])):
        kept = g.clone()
        with pytest.raises(ValueError):
            pkg.clip_gradients(grads, 1.0, out=out)
        assert torch.equal(g, kept)
    h = g.clone()
    pkg.clip_gradients([g[:50], g[50:]], 1.0)
    pkg.clip_gradients([h[50:], h[:50]], 1.0, out=[h[50:], h[:50]])
    near(g, h.double(), 4 * E32 * h.double().abs())
    with pytest.raises(ValueError):
        pkg.clip_gradients([g.requires_grad_(True)], 1.0)
    with pytest.raises(ValueError):
        pkg.clip_gradients([torch.zeros(10, 10, device="cuda")[:, :5]], 1.0)


# ================================================================= together
def block(pkg, x, projection, positions, f, offsets=None):
    """A rotated attention over one projection: [..., tokens, (4 + 2 + 2) * 64]."""
    q, k, v = (x @ projection).unflatten(-1, (8, 64)).split([4, 2, 2], dim=-2)
    q, k = pkg.rotary(q, k, positions, f)
    return pkg.attention(q, k, v, causal=True, offsets=offsets).flatten(-2)


def training_step(pkg, x, weight, positions, f, go):
    out = block(pkg, x, weight, positions, f)
    grad = torch.autograd.grad(out, weight, go)[0]
    clipped = [grad, torch.full((33,), 0.1, device="cuda")]
    norm = pkg.clip_gradients(clipped, 0.1)
    return [out.detach(), norm, *clipped]


def step_inputs(pkg, seed=71):
    x = randn(2, 200, 96, seed=seed, dtype=BF16)
    weight = randn(96, 512, seed=seed + 1, dtype=BF16, std=0.1).requires_grad_(True)
    return x, weight, torch.arange(200, device="cuda"), pkg.rotary_frequencies(64)[0], randn(2, 200, 256, seed=seed + 2, dtype=BF16)


def test_operators_together(pkg):
    """The same values from packed and from batched sequences, against 64 bits."""
    x, weight, at, f, go = step_inputs(pkg)
    out = block(pkg, x, weight, at, f)
    offsets = torch.tensor([0, 200, 400], device="cuda")
    packed = block(pkg, x.flatten(0, 1), weight, at.repeat(2), f, offsets)
    assert torch.equal(packed, out.flatten(0, 1))
    w = weight.detach().double().requires_grad_(True)
    q, k, v = (x.double() @ w).unflatten(-1, (8, 64)).split([4, 2, 2], dim=-2)

    def turn(t):
        angle = at.double()[:, None, None] * f
        a, b = t.chunk(2, -1)
        return torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()], -1)

    s = torch.einsum("blhd,bmhd->bhlm", turn(q), turn(k).repeat_interleave(2, 2)) / 8
    p = s.masked_fill(~sees(200, 200, True, None), -math.inf).softmax(-1)
    want = torch.einsum("bhlm,bmhd->blhd", p, v.repeat_interleave(2, 2)).flatten(-2)
    # six roundings to bf16 along the way (projection, turned keys and queries twice in the scores, probabilities,
    # values, output), relative to the largest value or, in the exponent, to scores of up to 8
    near(out, want, 2.0 ** -8 * (6 + 2 * 8) * want.abs().max())
    got, ref = torch.autograd.grad(out, weight, go)[0], torch.autograd.grad(want, w, go.double())[0]
    assert float((got.double() - ref).norm()) <= 22 * 2.0 ** -8 * float(ref.norm())


def test_repeated_steps_give_the_same_bits_on_any_stream(pkg):
    inputs = step_inputs(pkg)
    first = training_step(pkg, *inputs)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = training_step(pkg, *inputs)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, second):
        assert torch.equal(a, b)


def test_steps_on_two_streams_at_once(pkg):
    inputs = [step_inputs(pkg, seed) for seed in (71, 81)]
    want = [training_step(pkg, *i) for i in inputs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for n, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[n].append(training_step(pkg, *inputs[n]))
    torch.cuda.synchronize()
    for n in range(2):
        for one in got[n]:
            for a, b in zip(one, want[n]):
                assert torch.equal(a, b)


def test_steps_in_cuda_graphs(pkg):
    """Forward, backward and clipping captured; two graphs with a pool each,
    replayed in turn, with new inputs in the captured tensors."""
    inputs = [step_inputs(pkg, seed) for seed in (91, 101)]
    want = [[t.clone() for t in training_step(pkg, *i)] for i in inputs]
    torch.cuda.synchronize()
    graphs, got = [], []
    for i in inputs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got.append(training_step(pkg, *i))
        graphs.append(graph)
    for _ in range(3):
        for t in got[0] + got[1]:
            t.zero_()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got[0] + got[1], want[0] + want[1]):
            assert torch.equal(a, b)
    with torch.no_grad():  # other values in the captured tensors
        for to, t in zip(inputs[0], inputs[1]):
            to.copy_(t)
    graphs[0].replay()
    torch.cuda.synchronize()
    for a, b in zip(got[0], want[1]):
        assert torch.equal(a, b)


def test_fp16_attention_in_a_graph(pkg):
    """Its gradients' scale is found on the device, in every replay anew."""
    q, k, v, go = attention_inputs(2, 200, 200, 2, 1, 64, F16, seed=111)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]

    def grads():
        return torch.autograd.grad(pkg.attention(*leaves, causal=True), leaves, go)

    grads()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = grads()
    for size in (1.0, 1e-3, 500.0):
        go.mul_(size)
        want = grads()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_compiled_block(pkg):
    x, weight, at, f, go = step_inputs(pkg)
    want = torch.autograd.grad(block(pkg, x, weight, at, f), weight, go)[0]
    traced = torch.compile(lambda w: block(pkg, x, w, at, f), backend="aot_eager", fullgraph=True)
    assert torch.equal(torch.autograd.grad(traced(weight), weight, go)[0], want)


def test_kernels_are_launched_and_end(pkg):
    from muon_fusion_ascend950_b200.capi import capi

    api = capi()
    before = api.train_launch_count()
    training_step(pkg, *step_inputs(pkg))
    assert api.train_launch_count() >= before + 7
    assert api.train_device_status(torch.cuda.current_device()) == 0


def test_debug_sync_waits_for_every_call(pkg, monkeypatch):
    x, weight, at, f, go = step_inputs(pkg)
    q = randn(1, 64, 2, 64, seed=3, dtype=BF16)
    ops = torch.ops.muon_ascend950
    out, lse, rest = ops.attention(q, q, q, None, None, True, 0, 0.125, True)
    calls = [lambda: ops.attention(q, q, q, None, None, True, 0, 0.125, False),
             lambda: ops.attention_backward(q, q, q, q, out, lse, rest, None, None, True, 0, 0.125),
             lambda: ops.rotary(q, None, at[:64], f, False, 1.0),
             lambda: ops.clip_gradients_([q.clone()], 1.0, False)]
    for sync in (False, True):
        if sync:
            monkeypatch.setenv("MUON_POLAR_DEBUG_SYNC", "1")
        for call in calls:
            call()
            torch.cuda.synchronize()
            torch.cuda._sleep(100_000_000)
            call()
            assert torch.cuda.current_stream().query() == sync


def test_a_lower_wait_limit_reaches_every_kernel(pkg):
    """The limit read back is the largest of the kernels' copies: one that was
    left behind shows when the limit is lowered."""
    from muon_fusion_ascend950_b200.capi import capi

    api = capi()
    before = api.train_wait_limit_ns()
    previous = api.set_wait_limit_ns(before // 2)
    try:
        assert previous == before and api.train_wait_limit_ns() == before // 2
    finally:
        api.set_wait_limit_ns(previous)
    assert api.train_wait_limit_ns() == before
