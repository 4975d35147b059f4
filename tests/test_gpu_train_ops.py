"""GPU tests of the training-step operators against their definitions in 64
bits (on the same device), at the sizes, strides and masks where they can go
wrong.

Tolerances are bounds on rounding: every output is rounded once to its type
(unit roundoff `U`), and before that each value is a sum of products in fp32,
whose error is at most (number of sequential additions + a few operations) *
2^-24 times the sum of the terms' magnitudes, which the tests form in 64 bits.
"""
from __future__ import annotations

import math

import pytest
import torch

from train_calls import CALLS

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}  # half of a subnormal
E32 = 2.0 ** -24
F64 = torch.float64
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
NEG = -math.inf


@pytest.fixture(scope="module")
def pkg(cuda_device):
    import muon_fusion_ascend950_b200 as pkg

    return pkg


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def near(actual, expected, bound):
    """|actual - expected| <= bound wherever expected is finite; infinities
    and NaN in the same places."""
    actual, expected = actual.double(), expected.double()
    finite = expected.isfinite()
    assert torch.equal(actual[~finite].nan_to_num(7.0), expected[~finite].nan_to_num(7.0))
    assert torch.equal(actual.isnan(), expected.isnan())
    bound = torch.as_tensor(bound, dtype=F64, device=actual.device).expand_as(expected)
    over = ((actual - expected).abs() > bound) & finite
    assert not over.any(), (
        int(over.sum()), actual[over][:4].tolist(), expected[over][:4].tolist(), bound[over][:4].tolist())


def rounded(value, dtype):
    """Bound on the one rounding of `value` to dtype."""
    return U[dtype] * value.abs() + TINY[dtype]


# =========================================================== distillation
def distill_reference(z, t, i, g, tau, lse=None):
    """(loss, grad) in 64 bits, grad of sum(g * loss), by the formula."""
    z, t, g = z.double() / tau, t.double(), g.double()
    counted = (i >= 0) & (i < z.shape[1]) & (t > NEG)
    t = torch.where(counted, t, NEG) / tau
    some = counted.any(-1, keepdim=True)
    if lse is None:
        log_q = torch.where(some, t, 0.0).log_softmax(-1)  # relative to the largest, as below
    else:
        log_q = t - lse.double()[:, None]
    q = torch.where(counted, log_q.exp(), 0.0)
    at = torch.where(counted, i, 0).long()
    log_p = z.log_softmax(-1)  # relative to the row's largest: exact for the type's lowest value
    loss = torch.where(q == 0, 0.0, q * (log_q - log_p.gather(1, at))).sum(-1)
    total = q.sum(-1, keepdim=True)
    grad = log_p.exp() * total
    grad = grad.scatter_add(1, at, -q) * (g / tau)[:, None]
    none = (total == 0) | (g[:, None] == 0)
    return torch.where(total[:, 0] == 0, 0.0, loss), torch.where(none, 0.0, grad)


def distill_bounds(z, t, i, g, tau, lse, dtype):
    """Bounds on the errors of (loss, grad).  The row's sum of exponentials is
    taken by 32-lane warps of at least 256 threads, so vocab / 256 additions in
    a row and a few more cover it; an exponent x carries |x| 2^-22."""
    steps = (z.shape[1] / 256 + 64) * E32
    zs = torch.where(z.isfinite(), z.double(), 0.0) / tau
    log_z = zs.logsumexp(-1)
    counted = (i >= 0) & (i < z.shape[1]) & (t > NEG)
    ts = torch.where(counted, t.double(), 0.0) / tau
    span = zs.abs().amax(-1) + ts.abs().amax(-1) + log_z.abs()
    if lse is not None:
        span = span + lse.double().abs()
    at = torch.where(counted, i, 0).long()
    loss = (steps + t.shape[1] * E32) * (1 + 4 * span)
    ref = distill_reference(z, t, i, g, tau, lse)[1]
    p = (zs - log_z[:, None]).exp()
    # (z - max) / tau only: what underflows is no error of this size
    rel = steps + 8 * E32 * (zs.amax(-1, keepdim=True) - zs)
    q = torch.zeros_like(p).scatter_add(1, at, counted.double())
    scale = (g.double().abs() / tau)[:, None]
    grad = scale * (p * rel + q * (steps + 8 * E32 * span[:, None])) * 2 + rounded(
        torch.where(ref.isfinite(), ref, 0.0), dtype) + 2.0 ** -126
    return loss, grad


def distill_inputs(rows, vocab, top, dtype, index=torch.int64, seed=0):
    g = gen(seed)
    z = (torch.randn(rows, vocab, generator=g, device="cuda") * 3).to(dtype)
    order = torch.rand(rows, vocab, generator=g, device="cuda").topk(min(top, vocab), -1).indices
    i = order.to(index)
    t = (torch.randn(i.shape, generator=g, device="cuda") * 2 + 4).to(dtype)
    w = torch.rand(rows, generator=g, device="cuda") - 0.3
    return z, t, i, w


def check_distill(pkg, z, t, i, w, tau=1.0, lse=None):
    """All three forms of the operator against the definition."""
    ref_loss, ref_grad = distill_reference(z, t, i, w, tau, lse)
    b_loss, b_grad = distill_bounds(z, t, i, w, tau, lse, z.dtype)
    loss, grad = pkg.distill_topk_grad(z, t, i, w, temperature=tau, teacher_lse=lse)
    assert loss.dtype == torch.float32 and grad.dtype == z.dtype and grad.shape == z.shape
    near(loss, ref_loss, b_loss)
    near(grad, ref_grad, b_grad)
    assert torch.equal(loss, pkg.distill_topk_grad(z, t, i, temperature=tau, teacher_lse=lse)[0]
                       ) or bool(ref_loss.isnan().any())
    leaf = z.detach().requires_grad_(True)
    loss = pkg.distill_topk(leaf, t, i, temperature=tau, teacher_lse=lse)
    near(loss, ref_loss, b_loss)
    (grad,) = torch.autograd.grad(loss, leaf, w)
    assert grad.dtype == z.dtype and grad.shape == z.shape
    near(grad, ref_grad, b_grad)
    with torch.no_grad():
        near(pkg.distill_topk(z, t, i, temperature=tau, teacher_lse=lse), ref_loss, b_loss)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, vocab, top", [
    (1, 1, 1), (3, 7, 2), (5, 129, 129), (2, 1000, 1), (7, 4099, 33), (150, 2050, 8),
    (2, 32768, 64), (3, 32769, 16), (2, 50001, 32), (1, 131072, 128), (4, 131075, 100)])
def test_distill_sizes(pkg, rows, vocab, top, dtype):
    check_distill(pkg, *distill_inputs(rows, vocab, top, dtype, seed=vocab))


@pytest.mark.parametrize("rows, vocab", [(2, 262144), (2, 262149), (1, 400003), (1, 1100000)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_distill_largest_vocabularies(pkg, rows, vocab, dtype):
    check_distill(pkg, *distill_inputs(rows, vocab, 50, dtype, seed=3))


@pytest.mark.parametrize("rows, vocab, dtype, top", [
    (700, 24000, torch.bfloat16, 33), (300, 60001, torch.float16, 129), (900, 50001, torch.bfloat16, 7),
    (620, 131072, torch.bfloat16, 20), (89, 111553, torch.float32, 18), (310, 32771, torch.float32, 300),
    (75, 150001, torch.float32, 1024), (38, 260003, torch.bfloat16, 5)])
def test_distill_many_long_rows(pkg, rows, vocab, dtype, top):
    """Several rows for each block and cluster, so that stages, lists and slots
    come round again, at every alignment of the rows."""
    check_distill(pkg, *distill_inputs(rows, vocab, top, dtype, torch.int32, seed=rows))


@pytest.mark.parametrize("rows", [1, 16, 147, 148, 149, 300, 1200])
@pytest.mark.parametrize("vocab", [264, 8192, 33000])
def test_distill_row_counts(pkg, rows, vocab):
    check_distill(pkg, *distill_inputs(rows, vocab, 9, torch.bfloat16, torch.int32, seed=rows))


@pytest.mark.parametrize("tau", [0.5, 0.7, 2.0, 10.0])
@pytest.mark.parametrize("normalizer", [False, True])
def test_distill_temperature_and_normalizer(pkg, tau, normalizer):
    z, t, i, w = distill_inputs(9, 5001, 20, torch.float32, torch.int32, seed=4)
    lse = (t.double() / tau).logsumexp(-1).float() + 0.25 if normalizer else None
    check_distill(pkg, z, t, i, w, tau, lse)


@pytest.mark.parametrize("teacher", DTYPES)
def test_distill_teacher_types_and_longest_list(pkg, teacher):
    z, t, i, w = distill_inputs(3, 9000, 1024, torch.bfloat16, seed=5)
    check_distill(pkg, z, t.to(teacher), i, w)


@pytest.mark.parametrize("offset", [0, 1, 3, 5])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_distill_strides_and_alignment(pkg, offset, dtype):
    """Slices of padded logits at every alignment, a transposed matrix, and
    rows that are views of one row."""
    z, t, i, w = distill_inputs(6, 1203, 11, dtype, seed=6)
    padded = torch.full((6, 1300), math.nan, dtype=dtype, device="cuda")
    padded[:, offset:offset + 1203] = z
    check_distill(pkg, padded[:, offset:offset + 1203], t, i, w)
    wide = torch.full((6, 5000), math.nan, dtype=dtype, device="cuda")
    wide[:, offset:offset + 1203] = z
    check_distill(pkg, wide[:, offset:offset + 1203], t, i, w)
    check_distill(pkg, z.t().contiguous().t(), t.t().contiguous().t(), i.t().contiguous().t(), w)
    check_distill(pkg, z[2:3].expand(6, 1203), t, i, w)
    assert padded[:, :offset].isnan().all() and padded[:, offset + 1203:].isnan().all()


def test_distill_gradient_stays_inside_its_rows(pkg):
    """The gradient of a slice keeps the slice's layout; what lies between its
    rows is not written."""
    z, t, i, w = distill_inputs(5, 1203, 11, torch.bfloat16, seed=7)
    padded = torch.zeros(5, 1210, dtype=torch.bfloat16, device="cuda")
    padded[:, 3:1206] = z
    _, grad = pkg.distill_topk_grad(padded[:, 3:1206], t, i, w)
    torch.testing.assert_close(grad, pkg.distill_topk_grad(z, t, i, w)[1], rtol=2 ** -7, atol=1e-8)


def test_distill_leading_sizes(pkg):
    z, t, i, w = distill_inputs(12, 300, 5, torch.bfloat16, seed=8)
    loss, grad = pkg.distill_topk_grad(z, t, i, w)
    loss3, grad3 = pkg.distill_topk_grad(z.view(3, 4, 300), t.view(3, 4, 5), i.view(3, 4, 5), w.view(3, 4))
    assert torch.equal(loss3, loss.view(3, 4)) and torch.equal(grad3, grad.view(3, 4, 300))
    one, _ = pkg.distill_topk_grad(z[0], t[0], i[0], w[0])
    assert one.shape == () and torch.equal(one, loss[0])


@pytest.mark.parametrize("vocab", [700, 40000, 300000])
def test_distill_masks(pkg, vocab):
    """Left-out entries, empty rows over any logits, masked vocabulary."""
    z, t, i, w = distill_inputs(12, vocab, 16, torch.float32, seed=9)
    i[0, 3:] = -1
    i[1] = -1                                   # empty by index
    t[2] = NEG                                  # empty by logit
    z[3], i[3] = math.nan, -1                   # empty over NaN logits
    i[4, 2], i[4, 5] = vocab, 2 ** 40           # beyond the vocabulary
    i[5, :8] = i[5, 0].clone()                  # one index many times
    z[6, i[6, 0]] = NEG                         # the teacher's token is masked: infinite
    masked = torch.ones(vocab, dtype=torch.bool, device="cuda")
    masked[i[7]] = False
    z[7, masked] = NEG                          # only the list's tokens are left
    z[8] = torch.finfo(torch.float32).min       # a row of the type's lowest value
    t[9] = torch.finfo(torch.float32).min
    t[10, 1:] = torch.finfo(torch.float32).min
    t[11, 4] = math.nan                         # not above -inf: left out
    for tau in (1.0, 0.7):
        check_distill_masked(pkg, z, t, i, w, tau)


def check_distill_masked(pkg, z, t, i, w, tau):
    """As check_distill; rows with the type's lowest value are compared apart,
    as their bounds in terms of |z| say nothing."""
    ref_loss, ref_grad = distill_reference(z, t, i, w, tau)
    plain = [0, 1, 2, 3, 4, 5, 7, 11]
    near_rows = lambda x: x[plain]  # noqa: E731
    b_loss, b_grad = distill_bounds(z, t, i, w, tau, None, z.dtype)
    leaf = z.clone().requires_grad_(True)
    auto = pkg.distill_topk(leaf, t, i, temperature=tau)
    for loss, grad in (pkg.distill_topk_grad(z, t, i, w, temperature=tau),
                       (auto.detach(), torch.autograd.grad(auto, leaf, w)[0])):
        near(near_rows(loss), near_rows(ref_loss), near_rows(b_loss))
        near(near_rows(grad), near_rows(ref_grad), near_rows(b_grad).nan_to_num(0.0))
        for r in (1, 2, 3):
            assert loss[r] == 0 and bool((grad[r] == 0).all())
        assert loss[6] == math.inf and grad[6].isfinite().all()
        # a uniform row: p = 1 / vocab, whatever the value
        near(loss[8], ref_loss[8], 2.0 ** -14)
        near(grad[8], ref_grad[8], w[8].abs().double() / tau * 64 * E32)
        # lists of lowest values: uniform over 16; all on the first entry
        for r in (9, 10):
            near(grad[r], ref_grad[r], w[r].abs().double() / tau * 2 ** -14)
            near(loss[r], ref_loss[r], 2.0 ** -14 * (1 + ref_loss[r].abs()))


def test_distill_rows_without_a_finite_logit_are_nan(pkg):
    """As a softmax over nothing: NaN, and only in that row."""
    z, t, i, w = distill_inputs(3, 500, 4, torch.float32, seed=10)
    z[1] = NEG
    loss, grad = pkg.distill_topk_grad(z, t, i, w)
    assert loss[1].isnan() and grad[1].isnan().all()
    assert loss[[0, 2]].isfinite().all() and grad[[0, 2]].isfinite().all()
    z[1] = 0.0
    z[1, 77] = math.nan
    loss, grad = pkg.distill_topk_grad(z, t, i, w)
    assert loss[1].isnan() and grad[1].isnan().all() and grad[[0, 2]].isfinite().all()


def test_distill_zero_scale_gives_zero_gradient(pkg):
    z, t, i, w = distill_inputs(4, 1000, 4, torch.bfloat16, seed=11)
    z[1] = math.nan
    w[1] = 0.0
    _, grad = pkg.distill_topk_grad(z, t, i, w)
    assert bool((grad[1] == 0).all()) and grad.isfinite().all()
    leaf = z.clone().requires_grad_(True)
    (grad,) = torch.autograd.grad(pkg.distill_topk(leaf, t, i), leaf, w)
    assert bool((grad[1] == 0).all()) and grad.isfinite().all()


def test_distill_least_temperature(pkg):
    """All probability on the largest logit and entry: the loss of a row whose
    largest entry is its largest logit is 0, and no value is NaN."""
    z, t, i, w = distill_inputs(5, 700, 6, torch.float32, seed=48)
    z[:3] = z[:3].scatter(1, i[:3].gather(1, t[:3].argmax(-1, keepdim=True)), 100.0)
    tau = 2.0 ** -126
    loss, grad = pkg.distill_topk_grad(z, t, i, torch.zeros_like(w).fill_(tau), temperature=tau)
    assert bool((loss[:3] == 0).all()) and bool((loss[3:] == math.inf).all())
    assert int(grad[:3].count_nonzero()) == 0 and grad.isfinite().all()


def test_distill_no_rows(pkg):
    z = torch.empty(0, 100, device="cuda", requires_grad=True)
    t, i = torch.empty(0, 4, device="cuda"), torch.empty(0, 4, dtype=torch.int64, device="cuda")
    loss = pkg.distill_topk(z, t, i)
    assert loss.shape == (0,)
    loss.sum().backward()
    assert z.grad.shape == (0, 100)
    assert pkg.distill_topk_grad(z, t, i)[1].shape == (0, 100)


def test_distill_gradient_against_differences(pkg):
    """The gradient along random directions against central differences of the
    definition in 64 bits, and of the operator's own loss.  With |d| <= 1 and
    h = 2^-4 the differences are off by h^2 / 6 times the third derivative,
    which is at most 2 in a softmax's directions; the operator's loss of about
    10 is exact to 2^-19."""
    z, t, i, w = distill_inputs(6, 800, 12, torch.float32, seed=12)
    _, grad = pkg.distill_topk_grad(z, t, i, torch.ones_like(w))
    for seed in range(4):
        d = torch.rand(z.shape, generator=gen(seed), device="cuda") * 2 - 1
        along = (grad.double() * d.double()).sum(-1)
        one = torch.ones_like(w)
        h = 1e-4
        up, down = (distill_reference(z.double() + s * h * d.double(), t, i, one, 1.0)[0] for s in (1, -1))
        near(along, (up - down) / (2 * h), 1e-6)
        h = 2.0 ** -4
        up, down = (pkg.distill_topk(z + s * h * d, t, i).double() for s in (1, -1))
        near(along, (up - down) / (2 * h), h * h / 3 + 2.0 ** -18 / h)


def test_distill_past_32_bit_offsets(pkg):
    """More than 2^31 logits: the last rows are those of a small call."""
    rows, vocab = 16500, 131072
    z = torch.zeros(rows, vocab, dtype=torch.bfloat16, device="cuda")
    small, t, i, w = distill_inputs(3, vocab, 8, torch.bfloat16, seed=13)
    z[-3:] = small
    values = torch.zeros(rows, 8, dtype=torch.bfloat16, device="cuda")
    index = torch.full((rows, 8), -1, device="cuda")
    scale = torch.zeros(rows, device="cuda")
    values[-3:], index[-3:], scale[-3:] = t, i, w
    loss, grad = pkg.distill_topk_grad(z, values, index, scale)
    want_loss, want_grad = distill_reference(small, t, i, w, 1.0)
    b_loss, b_grad = distill_bounds(small, t, i, w, 1.0, None, torch.bfloat16)
    near(loss[-3:], want_loss, b_loss)
    near(grad[-3:], want_grad, b_grad)
    assert int(grad[:-3].count_nonzero()) == 0 and int(loss[:-3].count_nonzero()) == 0


# =========================================================== residual norm
NAMES = ("block_out", "residual", "post_weight", "pre_weight", "gate", "residual_scale")


def norm_reference(v, gate_rows, dh, dn, eps=1e-6):
    """(outputs, gradients, magnitudes of the gradients' terms) in 64 bits."""
    v = {n: t.double() for n, t in v.items() if t is not None}
    y, x = v["block_out"], v["residual"]
    rows, width = y.shape
    zero = torch.zeros_like(y)
    dh = zero if dh is None else dh.double()
    w = v.get("post_weight", torch.ones(width, dtype=F64, device="cuda"))
    gate = v["gate"].repeat_interleave(rows // gate_rows, 0) if "gate" in v else torch.ones_like(y)
    s = v.get("residual_scale", torch.ones(1, dtype=F64, device="cuda"))
    r = (y.square().mean(-1, keepdim=True) + eps).rsqrt() if "post_weight" in v else torch.ones_like(y[:, :1])
    u = y * r * w
    h = s * x + gate * u
    size = (s * x).abs() + (gate * u).abs()
    out, mag = {"hidden": h}, {"hidden": size}
    d, dmag = dh, dh.abs()
    grads = {}
    if "pre_weight" in v:
        p = v["pre_weight"]
        R = (h.square().mean(-1, keepdim=True) + eps).rsqrt()
        out["normed"], mag["normed"] = h * R * p, size * R * p.abs() + (h * R * p).abs()
        if dn is not None:
            dn = dn.double()
            a = dn * p
            k = R ** 3 / width
            d = dh + R * a - h * k * (a * h).sum(-1, keepdim=True)
            dmag = dmag + R * a.abs() + size * k * (a.abs() * size).sum(-1, keepdim=True)
            grads["pre_weight"] = (dn * h * R).sum(0)
            mag["pre_weight"] = (dn.abs() * size * R).sum(0)
        else:
            grads["pre_weight"] = torch.zeros_like(p)
            mag["pre_weight"] = grads["pre_weight"]
    b, bmag = d * gate * w, dmag * (gate * w).abs()
    if "post_weight" in v:
        k = r ** 3 / width
        grads["block_out"] = r * b - y * k * (b * y).sum(-1, keepdim=True)
        mag["block_out"] = r * bmag + y.abs() * k * (bmag * y.abs()).sum(-1, keepdim=True)
        grads["post_weight"] = (d * gate * y * r).sum(0)
        mag["post_weight"] = (dmag * (gate * y).abs() * r).sum(0)
    else:
        grads["block_out"], mag["block_out"] = b, bmag
    grads["residual"], mag["residual"] = d * s, dmag * s.abs()
    if "gate" in v:
        grads["gate"] = (d * u).unflatten(0, (gate_rows, -1)).sum(1)
        mag["gate"] = (dmag * u.abs()).unflatten(0, (gate_rows, -1)).sum(1)
    if "residual_scale" in v:
        full, fmag = (d * x).sum(0), (dmag * x.abs()).sum(0)
        one = s.numel() == 1
        grads["residual_scale"] = full.sum(0, keepdim=True) if one else full
        mag["residual_scale"] = fmag.sum(0, keepdim=True) if one else fmag
    return out, grads, mag


def norm_inputs(shape, dtype, params, gate, scale, post=True, pre=True, seed=0):
    g = gen(seed)
    width = shape[-1]

    def rand(*s, like=dtype, mean=0.0, std=1.0):
        return (torch.randn(*s, generator=g, device="cuda") * std + mean).to(like)

    v = {"block_out": rand(*shape, std=3.0), "residual": rand(*shape),
         "post_weight": rand(width, like=params, mean=0.5, std=0.3) if post else None,
         "pre_weight": rand(width, like=params, mean=1.0, std=0.3) if pre else None,
         "gate": None, "residual_scale": None}
    if gate is not None:
        v["gate"] = rand(*gate, width, like=params, std=1.0)
    if scale:
        v["residual_scale"] = rand(scale, like=params, mean=0.8, std=0.2)
    return v, rand(*shape, std=0.1), rand(*shape, std=0.1)


def check_norm(pkg, v, dh, dn, gate_rows=1, eps=1e-6, normed_used=True, hidden_used=True):
    shape, dtype = v["block_out"].shape, v["block_out"].dtype
    rows, width = v["block_out"].numel() // shape[-1], shape[-1]
    flat = {n: (t if t is None or n in ("post_weight", "pre_weight", "residual_scale")
                else t.reshape(-1, width)) for n, t in v.items()}
    use_dn = dn is not None and v["pre_weight"] is not None and normed_used
    out, grads, mag = norm_reference(flat, gate_rows, dh.reshape(rows, width) if hidden_used else None,
                                     dn.reshape(rows, width) if use_dn else None, eps)
    # a block's threads add width / 32 elements in a row at most, a row's
    # statistics carry their own error into every element twice
    steps = (width / 16 + 96) * E32
    leaves = {n: t.detach().requires_grad_(True) for n, t in v.items() if t is not None}
    hidden, normed = pkg.residual_norm(
        leaves["block_out"], leaves["residual"], leaves.get("post_weight"), leaves.get("pre_weight"),
        gate=leaves.get("gate"), residual_scale=leaves.get("residual_scale"), eps=eps)
    assert hidden.shape == shape and hidden.dtype == dtype
    near(hidden.reshape(rows, width), out["hidden"], rounded(out["hidden"], dtype) + steps * mag["hidden"])
    if v["pre_weight"] is None:
        assert normed is None
    else:
        assert normed.shape == shape and normed.dtype == dtype
        near(normed.reshape(rows, width), out["normed"], rounded(out["normed"], dtype) + steps * mag["normed"])
    ends, ups = ([hidden], [dh]) if hidden_used else ([], [])
    if use_dn:
        ends, ups = ends + [normed], ups + [dn]
    got = torch.autograd.grad(ends, list(leaves.values()), ups, allow_unused=True)
    for (name, leaf), grad in zip(leaves.items(), got):
        want = grads[name].reshape(-1)
        if grad is None:
            assert int(want.count_nonzero()) == 0
            continue
        assert grad.shape == leaf.shape and grad.dtype == leaf.dtype
        summed = 0 if name in ("block_out", "residual") else rows * (width if leaf.numel() == 1 else 1)
        bound = (steps * 2 + (summed + 64) * E32) * mag[name].reshape(-1)
        near(grad.reshape(-1), want, rounded(want, leaf.dtype) + bound)
    again = pkg.residual_norm(v["block_out"], v["residual"], v["post_weight"], v["pre_weight"],
                              gate=v["gate"], residual_scale=v["residual_scale"], eps=eps)
    assert torch.equal(again[0].nan_to_num(), hidden.nan_to_num())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, width", [
    (1, 1), (1, 8), (3, 7), (2, 129), (5, 264), (300, 64), (4, 512), (7, 1000), (150, 2050), (3, 2048),
    (33, 4096), (2, 4100), (5, 8192), (2, 8200), (2, 11008), (1, 16384), (2, 16400), (1, 65536), (1, 65537)])
def test_norm_sizes(pkg, rows, width, dtype):
    check_norm(pkg, *norm_inputs((rows, width), dtype, torch.float32, (), width, seed=width))


@pytest.mark.parametrize("rows, width, dtype, scale", [
    (700, 4104, torch.bfloat16, 1), (700, 8192, torch.float16, -1), (320, 12000, torch.bfloat16, -1),
    (500, 4100, torch.float32, -1), (320, 7684, torch.float32, 1), (320, 15360, torch.float32, -1),
    (500, 4098, torch.bfloat16, -1), (320, 9001, torch.float16, 1), (320, 15365, torch.float32, 1)])
def test_norm_many_wide_rows(pkg, rows, width, dtype, scale):
    """Several rows for each block and cluster of every wide layout."""
    check_norm(pkg, *norm_inputs((rows, width), dtype, torch.float32, (), width if scale < 0 else scale, seed=rows))


@pytest.mark.parametrize("width", [96, 130, 512, 4096])
@pytest.mark.parametrize("rows", [1, 2, 147, 148, 149, 295, 296, 297, 1000, 3001])
def test_norm_row_counts(pkg, rows, width):
    check_norm(pkg, *norm_inputs((rows, width), torch.bfloat16, torch.bfloat16, (), 1, seed=rows))


@pytest.mark.parametrize("width", [264, 258, 2048])
@pytest.mark.parametrize("post", [True, False])
@pytest.mark.parametrize("pre", [True, False])
@pytest.mark.parametrize("gate", [None, (), (4, 1), (4, 6)])
@pytest.mark.parametrize("scale", [0, 1, -1])
def test_norm_forms(pkg, width, post, pre, gate, scale):
    v, dh, dn = norm_inputs((4, 6, width), torch.bfloat16, torch.float32, gate, width if scale < 0 else scale,
                            post, pre, seed=14)
    rows = 1 if not gate else 4 if gate[-1] == 1 else 24
    check_norm(pkg, v, dh, dn, rows)


@pytest.mark.parametrize("params", DTYPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_norm_types(pkg, dtype, params):
    check_norm(pkg, *norm_inputs((37, 1024), dtype, params, (), 1024, seed=15))
    check_norm(pkg, *norm_inputs((37, 1021), dtype, params, (37,), 1, seed=15), gate_rows=37)


@pytest.mark.parametrize("groups, length", [(2, 1000), (7, 50), (100, 3), (700, 2), (1, 600), (900, 1), (5000, 2)])
@pytest.mark.parametrize("width", [256, 130])
def test_norm_gate_groups(pkg, groups, length, width):
    """More gate rows than blocks, one row each, fewer, and more than a grid's
    second axis has blocks for."""
    v, dh, dn = norm_inputs((groups, length, width), torch.bfloat16, torch.float32, (groups, 1), 1, seed=16)
    check_norm(pkg, v, dh, dn, groups)


@pytest.mark.parametrize("hidden_used, normed_used", [(True, False), (False, True)])
@pytest.mark.parametrize("width", [512, 130])
def test_norm_one_output_used(pkg, hidden_used, normed_used, width):
    v, dh, dn = norm_inputs((40, width), torch.bfloat16, torch.float32, (), width, seed=17)
    check_norm(pkg, v, dh, dn, hidden_used=hidden_used, normed_used=normed_used)


def test_norm_strides_and_alignment(pkg):
    """Transposed inputs, slices, and contiguous tensors that begin off a
    16-byte boundary."""
    for width in (512, 260):
        v, dh, dn = norm_inputs((24, width), torch.bfloat16, torch.bfloat16, (), width, seed=18)
        w = dict(v, block_out=v["block_out"].t().contiguous().t(), residual=v["residual"].repeat(1, 2)[:, :width])
        check_norm(pkg, w, dh.t().contiguous().t(), dn)
        check_norm(pkg, dict(v, residual=v["residual"][:1].expand(24, width)), dh, dn[:1].expand(24, width))
        for name in NAMES:
            t = v[name]
            moved = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape)
            moved.copy_(t)
            assert moved.data_ptr() % 16 == 2
            check_norm(pkg, dict(v, **{name: moved}), dh, dn)
        moved = torch.empty(dh.numel() + 1, dtype=dh.dtype, device="cuda")[1:].view(dh.shape).copy_(dh)
        check_norm(pkg, v, moved, dn)


def test_norm_special_rows(pkg):
    """Rows of zeros, a row whose hidden is zero, rows of NaN and infinity:
    each stays in its row."""
    v, dh, dn = norm_inputs((8, 264), torch.float32, torch.float32, None, 0, seed=19)
    v["block_out"][1] = 0.0
    v["block_out"][2] = v["residual"][2] = 0.0
    v["block_out"][3, 5] = math.nan
    v["block_out"][4, 7] = math.inf
    v["residual"][5] = math.nan
    leaves = {n: t.clone().requires_grad_(True) for n, t in v.items() if t is not None}
    hidden, normed = pkg.residual_norm(leaves["block_out"], leaves["residual"], leaves["post_weight"],
                                       leaves["pre_weight"])
    good = [0, 1, 2, 6, 7]
    assert hidden[good].isfinite().all() and normed[good].isfinite().all()
    assert int(normed[2].count_nonzero()) == 0
    assert hidden[3].isnan().all() and hidden[5].isnan().all() and hidden[4, 7].isnan()
    dy, dx = torch.autograd.grad([hidden, normed], [leaves["block_out"], leaves["residual"]], [dh, dn])
    assert dy[good].isfinite().all() and dx[good].isfinite().all() and dx[5].isnan().all()
    keep = dict(v, block_out=v["block_out"][good], residual=v["residual"][good])
    check_norm(pkg, keep, dh[good], dn[good])


@pytest.mark.parametrize("pre", [True, False])
@pytest.mark.parametrize("rows, width, dtype", [
    (5000, 64, torch.bfloat16), (1000, 130, torch.bfloat16), (3001, 512, torch.float16), (1000, 4096, torch.float32),
    (700, 4104, torch.bfloat16), (500, 4098, torch.bfloat16), (700, 8192, torch.bfloat16), (320, 9001, torch.float16),
    (320, 12000, torch.bfloat16), (320, 15360, torch.float32), (320, 15365, torch.float32), (50, 20000, torch.bfloat16)])
def test_norm_residual_scale_gradient_is_every_term_once(pkg, rows, width, dtype, pre):
    """With whole numbers and no gradient of normed, the terms dh x and every
    sum of them are exact, as all stay below 2^24 (a thread's and a column's) or
    2^53 (all): so must the gradient be, rounded once, whether the terms have one
    sign or cancel.  A row, block or cluster part left out or taken twice shows."""
    g = gen(49)

    def whole(low, high, *shape):
        return torch.randint(low, high + 1, shape, generator=g, device="cuda").to(dtype)

    w = torch.rand(width, generator=g, device="cuda")
    for low in (1, -3):
        x, dh = whole(low, 3, rows, width), whole(max(low, -2), 2, rows, width)
        y = torch.randn(rows, width, generator=g, device="cuda").to(dtype)
        terms = x.double() * dh.double()
        for scale in (torch.full((1,), 0.75, device="cuda"), torch.rand(width, generator=g, device="cuda")):
            scale.requires_grad_(True)
            hidden, _ = pkg.residual_norm(y, x, w, w if pre else None, residual_scale=scale)
            (grad,) = torch.autograd.grad(hidden, scale, dh)
            want = terms.sum().view(1) if scale.numel() == 1 else terms.sum(0)
            assert torch.equal(grad, want.float())


@pytest.mark.parametrize("size, eps", [(1e15, 1e-6), (1e-14, 0.0)])
@pytest.mark.parametrize("post", [True, False])
@pytest.mark.parametrize("rows, width, dtype", [
    (40, 64, torch.float32), (40, 200, torch.bfloat16), (300, 512, torch.float32), (300, 2048, torch.bfloat16),
    (20, 2050, torch.bfloat16), (20, 1021, torch.float32), (20, 8192, torch.bfloat16), (20, 12000, torch.float32),
    (20, 4098, torch.bfloat16), (5, 20000, torch.float32)])
def test_norm_gradients_of_large_and_small_rows(pkg, rows, width, dtype, size, eps, post):
    """Rows whose reciprocal roots are in fp32's range and whose cubes are not,
    in every layout; with the gradient of normed alone, whose projections are
    then as large as the rest."""
    v, dh, dn = norm_inputs((rows, width), dtype, torch.float32, (), 1, post=post, seed=42)
    for name in ("block_out", "residual"):
        v[name] = (v[name].float() * size).to(dtype)
    check_norm(pkg, v, dh, dn, eps=eps)
    check_norm(pkg, v, dh, dn, eps=eps, hidden_used=False)


@pytest.mark.parametrize("rows, width", [(300, 64), (300, 130), (700, 512), (400, 4096), (30, 8192), (20, 12000), (5, 20000)])
@pytest.mark.parametrize("post", [True, False])
@pytest.mark.parametrize("pre", [True, False])
def test_norm_statistics_are_written_in_every_form(pkg, rows, width, post, pre):
    """The operator's third output has no value that was there before."""
    v, _, _ = norm_inputs((rows, width), torch.bfloat16, torch.float32, None, 0, post, pre, seed=50)
    torch.full((2, rows), math.nan, device="cuda")  # what the allocator gives out next
    hidden, _, rstd = torch.ops.muon_ascend950.residual_norm(*(v[n] for n in NAMES), 1e-6)
    out, _, _ = norm_reference(v, 1, None, None)
    y, h = v["block_out"].double(), out["hidden"]
    steps = (width / 16 + 96) * E32
    for got, of, there, without in ((rstd[0], y, post, 1.0), (rstd[1], h, pre, 0.0)):
        want = (of.square().mean(-1) + 1e-6).rsqrt() if there else torch.full((rows,), without, device="cuda")
        near(got, want, steps * want.double() if there else 0.0)


def test_norm_no_rows(pkg):
    x = torch.empty(0, 64, device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda", requires_grad=True)
    hidden, normed = pkg.residual_norm(x, x, w, w, gate=w, residual_scale=w)
    assert hidden.shape == normed.shape == (0, 64)
    (hidden.sum() + normed.sum()).backward()
    assert x.grad.shape == (0, 64) and int(w.grad.count_nonzero()) == 0


def test_norm_gradient_against_differences(pkg):
    """Along random directions in all inputs at once, against central
    differences of the definition in 64 bits (off by about h^2 = 1e-8)."""
    v, dh, dn = norm_inputs((6, 264), torch.float32, torch.float32, (6,), 264, seed=20)
    leaves = {n: t.clone().requires_grad_(True) for n, t in v.items()}
    hidden, normed = pkg.residual_norm(*(leaves[n] for n in NAMES[:4]), gate=leaves["gate"],
                                       residual_scale=leaves["residual_scale"])
    grads = torch.autograd.grad([hidden, normed], list(leaves.values()), [dh, dn])

    def total(shift, d):
        out = norm_reference({n: t.double() + shift * d[n] for n, t in v.items()}, 6, None, None)[0]
        return (out["hidden"] * dh.double()).sum() + (out["normed"] * dn.double()).sum()

    for seed in range(4):
        g = gen(seed)
        d = {n: torch.randn(t.shape, generator=g, device="cuda").double() for n, t in v.items()}
        along = sum((a.double() * d[n]).sum() for n, a in zip(leaves, grads))
        size = sum((a.double() * d[n]).abs().sum() for n, a in zip(leaves, grads))
        h = 1e-4
        near(along, (total(h, d) - total(-h, d)) / (2 * h), size * 1e-5 + 1e-5)


def test_norm_past_32_bit_offsets(pkg):
    """More than 2^31 elements: the last rows, and the parameter gradients,
    are those of a small call when all other rows are zero."""
    rows, width = 530000, 4096
    v, dh, dn = norm_inputs((5, width), torch.bfloat16, torch.float32, (), width, seed=39)

    def grads(y, x, gh, gn):
        y, x = y.requires_grad_(True), x.requires_grad_(True)
        p = [v[n].detach().requires_grad_(True) for n in NAMES[2:]]
        ends = pkg.residual_norm(y, x, p[0], p[1], gate=p[2], residual_scale=p[3])
        return [e.detach()[-5:] for e in ends] + [
            g[-5:] if g.ndim == 2 else g for g in torch.autograd.grad(ends, [y, x, *p], [gh, gn])]

    def last(t):
        return torch.cat([torch.zeros(rows - 5, width, dtype=t.dtype, device="cuda"), t])

    small = grads(v["block_out"].clone(), v["residual"].clone(), dh, dn)
    large = grads(last(v["block_out"]), last(v["residual"]), last(dh), last(dn))
    for a, b in zip(small[:4], large[:4]):
        assert torch.equal(a, b)
    for a, b in zip(small[4:], large[4:]):  # the same five rows, added up in another order
        torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-6)


# =========================================================== routing
def route_scores(x, score):
    return x.double().softmax(-1) if score == "softmax" else x.double().sigmoid()


def check_route(pkg, x, k, score="softmax", bias=None, groups=1, top_groups=1, group_top=None,
                renormalize=True, scale=1.0, seed=0):
    tokens, experts = x.shape
    leaf = x.detach().requires_grad_(True)
    kw = dict(score=score, bias=bias, groups=groups, top_groups=top_groups, group_top=group_top,
              renormalize=renormalize, scale=scale)
    weights, indices, counts = pkg.route_experts(leaf, k, **kw)
    assert weights.dtype == torch.float32 and weights.shape == indices.shape == (tokens, k)
    assert indices.dtype == counts.dtype == torch.int64 and counts.shape == (experts,)
    assert bool(((indices >= 0) & (indices < experts)).all())
    assert torch.equal(counts, torch.bincount(indices.reshape(-1), minlength=experts))
    ordered = indices.sort(-1).values
    assert bool((ordered[:, 1:] > ordered[:, :-1]).all())  # no expert twice
    # the choice: keys in 64 bits, to the 2^-21 that an fp32 key may be off
    s = route_scores(x, score)
    key = s if bias is None else s + bias.double()
    slack = 2.0 ** -21 * (1 + (0 if bias is None else bias.double().abs().max()))
    if groups > 1:
        top = group_top or (2 if score == "sigmoid" and experts // groups > 1 else 1)
        parts = key.unflatten(-1, (groups, -1))
        group_key = parts.topk(top, -1).values.sum(-1)
        cut = group_key.topk(top_groups, -1).values[:, -1:]
        used = indices // (experts // groups)
        assert bool((group_key.gather(1, used) >= cut - 2 * slack).all())
        # ties of groups aside, the experts are the best of the allowed groups
        allowed = (group_key >= cut).repeat_interleave(experts // groups, 1)
        clear = (group_key >= cut - 2 * slack).sum(-1) == top_groups
        want = key.masked_fill(~allowed, NEG).topk(k, -1).values
        got = key.gather(1, indices)
        near(got[clear], want[clear], slack)
    else:
        near(key.gather(1, indices), key.topk(k, -1).values, slack)
    # weights and their gradient for that choice
    chosen = s.gather(1, indices)
    total = chosen.sum(-1, keepdim=True) + 1e-20 if renormalize else torch.ones_like(chosen[:, :1])
    want = scale * chosen / total
    # an exponent of x carries |x| 2^-23
    steps = (96 + 8 * float(torch.where(x.isfinite(), x, 0).abs().max()) + k) * E32
    near(weights, want, steps * want.abs() + 2.0 ** -126 * scale)
    up = torch.randn(tokens, k, generator=gen(seed), device="cuda")
    (grad,) = torch.autograd.grad(weights, leaf, up)
    assert grad.dtype == x.dtype and grad.shape == x.shape
    d = up.double() * scale
    size = d.abs()
    if renormalize:
        size = (size + (size * chosen / total).sum(-1, keepdim=True)) / total
        d = (d - (d * chosen / total).sum(-1, keepdim=True)) / total
    d = torch.zeros_like(s).scatter(1, indices, d)
    size = torch.zeros_like(s).scatter(1, indices, size)
    if score == "softmax":
        ref = s * (d - (d * s).sum(-1, keepdim=True))
        size = s * (size + (size * s).sum(-1, keepdim=True))
    else:
        ref, size = d * s * (1 - s), size * s
    near(grad, ref, rounded(ref, x.dtype) + 4 * steps * size + 2.0 ** -126)
    return weights, indices, counts


def logits(tokens, experts, dtype=torch.float32, seed=0, std=1.5):
    return (torch.randn(tokens, experts, generator=gen(seed), device="cuda") * std).to(dtype)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens, experts, k", [
    (1, 1, 1), (1, 2, 2), (3, 7, 3), (5, 31, 31), (1, 32, 8), (9, 33, 4), (64, 60, 4), (65, 64, 6), (7, 100, 10),
    (1000, 128, 8), (33, 129, 64), (40, 256, 8), (257, 257, 5), (5, 384, 12), (3, 511, 16), (4, 512, 64), (6, 1000, 7), (5, 1024, 64)])
def test_route_sizes(pkg, tokens, experts, k, dtype, score):
    x = logits(tokens, experts, dtype, seed=experts)
    check_route(pkg, x, k, score)
    check_route(pkg, x, k, score, renormalize=False, scale=2.5)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("tokens", [1, 2, 31, 63, 64, 65, 129, 2053, 20000])
def test_route_token_counts(pkg, tokens, score):
    bias = torch.randn(64, generator=gen(1), device="cuda") * 0.05
    check_route(pkg, logits(tokens, 64, seed=tokens), 6, score, bias=bias, scale=1.5)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("group_top", [None, 1, 2])
@pytest.mark.parametrize("experts, groups, top_groups, k", [
    (256, 8, 4, 8), (64, 8, 1, 8), (64, 2, 2, 40), (60, 4, 3, 5), (96, 32, 5, 6), (300, 100, 40, 64), (12, 3, 1, 4),
    (1024, 64, 8, 16), (1000, 8, 3, 9), (34, 17, 9, 2)])
@pytest.mark.parametrize("biased", [False, True])
def test_route_groups(pkg, experts, groups, top_groups, k, score, group_top, biased):
    bias = torch.randn(experts, generator=gen(2), device="cuda") * 0.1 if biased else None
    check_route(pkg, logits(150, experts, seed=21), k, score, bias, groups, top_groups, group_top)


def test_route_groups_of_one_expert(pkg):
    check_route(pkg, logits(20, 16, seed=22), 3, "softmax", None, 16, 5, 1)
    check_route(pkg, logits(20, 16, seed=22), 3, "sigmoid", None, 16, 5)


@pytest.mark.parametrize("experts", [8, 40, 64, 256, 1000])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_ties_go_to_the_lowest_index(pkg, experts, score):
    """Logits of few values: the choice is that of a stable sort."""
    k = min(8, experts)
    x = torch.randint(-2, 3, (300, experts), generator=gen(23), device="cuda").float()
    _, indices, _ = pkg.route_experts(x, k, score=score)
    assert torch.equal(indices, x.sort(dim=-1, descending=True, stable=True).indices[:, :k])
    bias = torch.randint(0, 2, (experts,), generator=gen(24), device="cuda").float() * 4
    _, indices, _ = pkg.route_experts(x, k, score=score, bias=bias)
    s = torch.sigmoid(x.double()) if score == "sigmoid" else x.double().softmax(-1)
    key = (s + bias).round(decimals=9)
    assert torch.equal(indices, key.sort(dim=-1, descending=True, stable=True).indices[:, :k])
    # equal groups: the lowest
    _, indices, _ = pkg.route_experts(torch.zeros(4, experts, device="cuda"), 2, score=score, groups=4, top_groups=1)
    assert torch.equal(indices, torch.tensor([[0, 1]] * 4, device="cuda"))
    # -0 and +0 are one key
    x = torch.zeros(3, experts, device="cuda")
    x[:, ::2] = -0.0
    _, indices, _ = pkg.route_experts(x, 4, score=score)
    assert torch.equal(indices, torch.arange(4, device="cuda").expand(3, 4))


@pytest.mark.parametrize("experts", [48, 64, 100, 128, 256, 300, 512, 1000])
@pytest.mark.parametrize("k", [3, 4, 8, 15, 16, 17])
def test_route_choice_is_that_of_a_stable_sort(pkg, experts, k):
    """Logits with some equal ones, the best spread over the row, side by side,
    few above a floor, or in falling or rising order."""
    x = torch.randn(400, experts, generator=gen(41), device="cuda")
    x[100:200] = (x[100:200] * 8).round() / 8
    x[200:300] = (x[200:300] * 2).round() / 2
    x[::5] = x[::5].sort(dim=-1, descending=True).values
    x[1::5] = x[1::5].sort(-1).values
    x[2::10] = x[2::10].clamp(min=x[2::10].topk(max(1, k // 2), -1).values[:, -1:])
    for start in (0, 7, experts - 20):
        x[300 + start % 50::50, start:start + 20] += 8
    x[399, 5:] = NEG
    want = x.sort(dim=-1, descending=True, stable=True).indices[:, :k]
    weights, indices, counts = pkg.route_experts(x, k)
    assert torch.equal(indices, want)
    assert torch.equal(counts, torch.bincount(want.reshape(-1), minlength=experts))
    near(weights, x.double().gather(1, want).softmax(-1), 1e-6)
    # in four groups, the two with the largest logit
    lead = x.view(400, 4, -1).amax(-1).sort(dim=-1, descending=True, stable=True).indices[:, :2]
    stays = torch.zeros(400, 4, dtype=torch.bool, device="cuda").scatter_(1, lead, True)
    stays = stays.repeat_interleave(experts // 4, 1)
    order = x.sort(dim=-1, descending=True, stable=True).indices
    rank = torch.where(stays.gather(1, order), torch.arange(experts, device="cuda"), experts)
    want = order.gather(1, rank.sort(-1).indices[:, :k])
    _, indices, _ = pkg.route_experts(x, k, groups=4, top_groups=2, group_top=1)
    assert torch.equal(indices, want)


@pytest.mark.parametrize("experts", [16, 300])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_masks(pkg, experts, score):
    """Masked experts, rows without any, the type's lowest value, NaN."""
    x = logits(8, experts, seed=25)
    x[1, 5:] = NEG                              # fewer than k are left
    x[2] = NEG                                  # none is left
    x[3, 3] = math.nan
    x[4] = torch.finfo(torch.float32).min
    x[5, 1:] = torch.finfo(torch.float32).min
    x[6] = math.nan
    leaf = x.clone().requires_grad_(True)
    weights, indices, counts = pkg.route_experts(leaf, 8, score=score)
    assert bool(((indices >= 0) & (indices < experts)).all()) and int(counts.sum()) == 64
    best = x[1, :5].sort(dim=-1, descending=True, stable=True).indices
    assert torch.equal(indices[1], torch.cat([best, torch.arange(5, 8, device="cuda")]))
    assert int(weights[1, 5:].count_nonzero()) == 0 and float(weights[1].detach().sum()) == pytest.approx(1.0, abs=1e-6)
    assert torch.equal(indices[2], torch.arange(8, device="cuda")) and int(weights[2].count_nonzero()) == 0
    assert not bool((indices[3] == 3).any()) and (score == "softmax") == bool(weights[3].isnan().all())
    assert torch.equal(indices[4], torch.arange(8, device="cuda"))
    near(weights[4], torch.full((8,), 0.125 if score == "softmax" else 0.0, device="cuda"), 1e-6)
    assert indices[5, 0] == 0 and float(weights[5, 0].detach()) == 1.0
    assert torch.equal(indices[6], torch.arange(8, device="cuda")) and weights[6].isnan().all()
    (grad,) = torch.autograd.grad(weights, leaf, torch.ones_like(weights))
    good = [0, 1, 2, 4, 5, 7]
    assert grad[good].isfinite().all() and int(grad[2].count_nonzero()) == 0


def test_route_strides_and_shapes(pkg):
    x = logits(30, 70, torch.bfloat16, seed=26)
    base = pkg.route_experts(x, 5)
    wide = torch.full((30, 100), math.inf, dtype=torch.bfloat16, device="cuda")
    wide[:, 7:77] = x
    for view in (wide[:, 7:77], x.t().contiguous().t()):
        for a, b in zip(pkg.route_experts(view, 5), base):
            assert torch.equal(a, b)
        check_route(pkg, view, 5, "sigmoid")
    weights, indices, counts = pkg.route_experts(x.view(5, 6, 70), 5)
    assert torch.equal(weights, base[0].view(5, 6, 5)) and torch.equal(indices, base[1].view(5, 6, 5))
    assert torch.equal(counts, base[2])
    one = pkg.route_experts(x[3], 5)
    assert one[0].shape == (5,) and torch.equal(one[1], base[1][3])
    check_route(pkg, x[:1].expand(30, 70), 5)


def test_route_past_32_bit_offsets(pkg):
    tokens = 2 ** 31 // 256 + 100
    small = logits(60, 256, torch.bfloat16, seed=40)
    x = torch.zeros(tokens, 256, dtype=torch.bfloat16, device="cuda")
    x[-60:] = small
    up = torch.randn(60, 4, generator=gen(41), device="cuda")
    grads = []
    for z, g in ((small.clone(), up), (x, torch.cat([torch.zeros(tokens - 60, 4, device="cuda"), up]))):
        z.requires_grad_(True)
        weights, indices, counts = pkg.route_experts(z, 4)
        grads.append([weights.detach()[-60:], indices[-60:], torch.autograd.grad(weights, z, g)[0][-60:]])
        assert int(counts.sum()) == 4 * z.shape[0]
    for a, b in zip(*grads):
        assert torch.equal(a, b)


def test_route_no_tokens(pkg):
    x = torch.empty(0, 16, device="cuda", requires_grad=True)
    weights, indices, counts = pkg.route_experts(x, 4)
    assert weights.shape == indices.shape == (0, 4) and int(counts.count_nonzero()) == 0
    weights.sum().backward()
    assert x.grad.shape == (0, 16)


def test_route_gradient_against_differences(pkg):
    """Central differences in 64 bits with the choice held."""
    for score in ("softmax", "sigmoid"):
        for renormalize in (True, False):
            x = logits(20, 48, seed=27).requires_grad_(True)
            weights, indices, _ = pkg.route_experts(x, 6, score=score, renormalize=renormalize, scale=1.5)
            up = torch.randn(weights.shape, generator=gen(28), device="cuda")
            (grad,) = torch.autograd.grad(weights, x, up)
            d = torch.randn(x.shape, generator=gen(29), device="cuda").double()

            def total(shift):
                s = route_scores(x.detach().double() + shift * d, score).gather(1, indices)
                return (1.5 * (s / s.sum(-1, keepdim=True) if renormalize else s) * up.double()).sum(-1)

            near((grad.double() * d).sum(-1), (total(1e-4) - total(-1e-4)) / 2e-4, 1e-5)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("experts, k", [(32, 4), (60, 6), (128, 40), (256, 8), (300, 5), (1024, 64)])
@pytest.mark.parametrize("spread", [0, 30, 45, 60, 90, 120])
def test_route_bias_for_vanishing_scores(pkg, experts, k, dtype, spread):
    """A bias that chooses the k experts `spread` below the others: their weights and
    gradients are those of s / (sum + 1e-20).  An fp32 score is off by a relative `steps`
    (an exponent of x carries |x| 2^-23) and, where it is subnormal, by 2^-147: `tiny` after
    the division by the sum."""
    x = logits(50, experts, seed=43)
    bias = torch.zeros(experts, device="cuda")
    bias[::experts // k][:k] = 4.0
    x[:, bias > 0] -= spread
    x = x.to(dtype)
    leaf = x.clone().requires_grad_(True)
    weights, indices, _ = pkg.route_experts(leaf, k, bias=bias, scale=1.5)
    assert torch.equal(indices.sort(-1).values, bias.nonzero().view(1, k).expand(50, k))
    up = torch.randn(50, k, generator=gen(44), device="cuda")
    (grad,) = torch.autograd.grad(weights, leaf, up)
    z = x.double().requires_grad_(True)
    s = z.softmax(-1)
    chosen = s.gather(1, indices)
    total = chosen.sum(-1, keepdim=True) + 1e-20
    want = 1.5 * chosen / total
    (ref,) = torch.autograd.grad(want, z, up.double(), retain_graph=True)
    s, chosen, total, want = (t.detach() for t in (s, chosen, total, want))
    steps = (96 + 8 * float(x.abs().max()) + k) * E32
    tiny = 1.5 * 2.0 ** -147 / total
    near(weights, want, steps * want + tiny)
    size = up.double().abs()
    mean = (size * chosen / total).sum(-1, keepdim=True)
    bound = torch.zeros_like(s).scatter(1, indices, 4 * steps * want * (size + mean) + (2 + k) * tiny * size.amax())
    # the others' part, and the cancellation of the 64-bit sum that it is compared with
    bound += s * 1.5 * mean * (4 * steps * 1e-20 / total + 2.0 ** -48) + s * k * tiny * size.amax() * 1e-20 / total
    near(grad, ref, bound + rounded(ref, dtype) + 2.0 ** -126)


def test_route_nan_reaches_the_whole_gradient(pkg):
    """A NaN logit makes a softmax of its row NaN, though it is not chosen."""
    for renormalize in (True, False):
        x = logits(6, 40, seed=45)
        x[2, 7] = math.nan
        x.requires_grad_(True)
        weights, indices, _ = pkg.route_experts(x, 4, renormalize=renormalize)
        assert not bool((indices[2] == 7).any()) and weights[2].isnan().all()
        (grad,) = torch.autograd.grad(weights, x, torch.ones_like(weights))
        assert grad[2].isnan().all() and grad[[0, 1, 3, 4, 5]].isfinite().all()


@pytest.mark.parametrize("seed", range(8))
def test_route_choice_is_the_plain_forms(pkg, seed):
    """Of the measured cases' ranges: a choice does not depend on how the scores
    were computed, so that indices and counts equal those of torch operations."""
    import importlib.util
    import random
    from pathlib import Path

    path = Path(__file__).resolve().parent.parent / "perf" / "operators.py"
    spec = importlib.util.spec_from_file_location("perf_operators", path)
    cases = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(cases)
    rng, done = random.Random(seed), 0
    while done < 25:
        case = cases.draw(rng)
        if case["op"] != "route":
            continue
        done += 1
        state = cases.prepare(case, seed)
        cases.own = False
        plain = cases.run(state)
        cases.own = True
        own = cases.run(state)
        assert torch.equal(own["indices"], plain["indices"]) and torch.equal(own["counts"], plain["counts"]), case


# =========================================================== all of them
def test_refusals_on_the_device(pkg):
    x = torch.zeros(4, 16, device="cuda")
    i = torch.zeros(4, 2, dtype=torch.int64, device="cuda")
    for tau in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError):
            pkg.distill_topk(x, x[:, :2], i, temperature=tau)
    with pytest.raises(ValueError):
        pkg.distill_topk(x, x[:, :0], i[:, :0])
    with pytest.raises(ValueError):
        pkg.distill_topk(x, torch.zeros(4, 1025, device="cuda"), torch.zeros(4, 1025, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError):
        pkg.residual_norm(x, x, eps=-1.0)
    for kw in (dict(k=0), dict(k=17), dict(k=2, groups=3), dict(k=2, groups=4, top_groups=5),
               dict(k=5, groups=4, top_groups=1), dict(k=2, groups=4, group_top=3), dict(k=2, scale=math.nan),
               dict(k=2, groups=16, top_groups=4, group_top=2)):
        with pytest.raises(ValueError):
            pkg.route_experts(x, **kw)
    with pytest.raises(ValueError):
        pkg.route_experts(torch.zeros(1, 1025, device="cuda"), 1)


@pytest.mark.parametrize("name", CALLS)
def test_calls_are_taken_and_refused(pkg, name):
    call, error = CALLS[name]
    if error is None:
        call()
    else:
        with pytest.raises(error):
            call()


def test_gradients_of_gradients_are_refused(pkg):
    x = torch.randn(4, 16, device="cuda", requires_grad=True)
    i = torch.zeros(4, 1, dtype=torch.int64, device="cuda")
    w = torch.ones(16, device="cuda")
    for value in (pkg.distill_topk(x, torch.zeros(4, 1, device="cuda"), i).sum(),
                  pkg.residual_norm(x, x, w, w)[1].sum(), pkg.route_experts(x, 2)[0].sum()):
        with pytest.raises(NotImplementedError):
            torch.autograd.grad(value, x, create_graph=True)


def test_tangents_of_gradients_are_refused(pkg):
    """Forward over reverse: a tangent in what flows back."""
    from torch.autograd import forward_ad

    x = torch.randn(4, 16, device="cuda", requires_grad=True)
    i = torch.zeros(4, 1, dtype=torch.int64, device="cuda")
    w = torch.ones(16, device="cuda")
    for out in (pkg.distill_topk(x, torch.zeros(4, 1, device="cuda"), i), pkg.residual_norm(x, x, w, w)[1],
                pkg.route_experts(x, 2)[0]):
        with forward_ad.dual_level(), pytest.raises(NotImplementedError):
            torch.autograd.grad(out, x, forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out)))


def test_same_bits_twice_and_on_another_stream(pkg):
    """Every output is deterministic, and follows its own stream's order."""
    def everything():
        out = []
        z, t, i, w = distill_inputs(64, 9001, 12, torch.bfloat16, seed=30)
        out += pkg.distill_topk_grad(z, t, i, w)
        leaf = z.requires_grad_(True)
        out += torch.autograd.grad(pkg.distill_topk(leaf, t, i), leaf, w)
        v, dh, dn = norm_inputs((3, 333, 520), torch.bfloat16, torch.float32, (3, 1), 520, seed=31)
        leaves = [t.requires_grad_(True) for t in v.values()]
        ends = pkg.residual_norm(*leaves[:4], gate=leaves[4], residual_scale=leaves[5])
        out += [*ends, *torch.autograd.grad(ends, leaves, [dh, dn])]
        x = logits(3000, 96, seed=32).requires_grad_(True)
        routed = pkg.route_experts(x, 8, score="sigmoid", groups=8, top_groups=3)
        out += [*routed, *torch.autograd.grad(routed[0], x, torch.ones_like(routed[0]))]
        return [o.detach() for o in out]

    first = everything()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = everything()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, second):
        assert torch.equal(a, b)


def test_in_a_cuda_graph(pkg):
    """The forward and fused calls allocate through torch only, so a graph
    captures them."""
    z, t, i, w = distill_inputs(32, 5000, 8, torch.bfloat16, seed=33)
    x = logits(200, 64, seed=34)
    v, _, _ = norm_inputs((40, 512), torch.bfloat16, torch.bfloat16, (), 1, seed=35)

    def calls():
        return [*pkg.distill_topk_grad(z, t, i, w), *pkg.route_experts(x, 4),
                *pkg.residual_norm(*list(v.values())[:4], gate=v["gate"], residual_scale=v["residual_scale"])]

    want = [o.clone() for o in calls()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = calls()
    for o in got:
        o.zero_()
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_compiled_training_step(pkg):
    """The operators and their gradients trace through AOT autograd."""
    v, dh, dn = norm_inputs((40, 264), torch.bfloat16, torch.float32, (), 1, seed=36)
    z, t, i, w = distill_inputs(40, 264, 8, torch.bfloat16, seed=37)

    def step(y, x, post, pre, gate, scale):
        hidden, normed = pkg.residual_norm(y, x, post, pre, gate=gate, residual_scale=scale)
        weights, _, _ = pkg.route_experts(normed[:, :64], 4)
        return (pkg.distill_topk(normed, t, i) * w).sum() + weights[:, 0].sum() + (hidden * dh).float().sum()

    grads = []
    for run in (step, torch.compile(step, backend="aot_eager", fullgraph=True)):
        leaves = [a.clone().requires_grad_(True) for a in v.values()]
        grads.append(torch.autograd.grad(run(*leaves), leaves))
    for a, b in zip(*grads):
        assert torch.equal(a, b)


def test_gradients_only_where_they_are_asked_for(pkg):
    """Inputs without a gradient get none, and the others the same as ever."""
    v, dh, dn = norm_inputs((50, 520), torch.bfloat16, torch.float32, (), 520, seed=38)

    def grads(wanted):
        leaves = {n: t.detach().requires_grad_(n in wanted) for n, t in v.items()}
        ends = pkg.residual_norm(*(leaves[n] for n in NAMES[:4]), gate=leaves["gate"],
                                 residual_scale=leaves["residual_scale"])
        return torch.autograd.grad(ends, [leaves[n] for n in wanted], [dh, dn])

    everything = dict(zip(NAMES, grads(NAMES)))
    for name in NAMES:
        assert torch.equal(grads([name])[0], everything[name])
    # saved for one backward pass, or as many as are kept
    x = torch.randn(4, 16, device="cuda", requires_grad=True)
    loss = pkg.route_experts(x, 2)[0][:, 0].sum()
    first = torch.autograd.grad(loss, x, retain_graph=True)[0]
    assert torch.equal(first, torch.autograd.grad(loss, x)[0])
    with pytest.raises(RuntimeError):
        torch.autograd.grad(loss, x)
    # a saved input that was changed since is noticed
    x = torch.randn(4, 16, device="cuda", requires_grad=True)
    y = x * 1
    out = pkg.route_experts(y, 2)[0]
    y.add_(1)
    with pytest.raises(RuntimeError):
        out.sum().backward()


def test_the_wait_limit_reaches_the_training_kernels(pkg):
    """The library's one setter holds for every kernel of the library."""
    from muon_fusion_ascend950_b200.capi import capi

    api = capi()
    before = api.train_wait_limit_ns()
    previous = api.set_wait_limit_ns(3_000_000_000)
    try:
        assert previous == before and api.train_wait_limit_ns() == 3_000_000_000
    finally:
        api.set_wait_limit_ns(previous)
    assert api.train_wait_limit_ns() == before


def test_debug_sync_waits_for_every_call(pkg, monkeypatch):
    """With MUON_POLAR_DEBUG_SYNC set each call, forward and backward, returns
    only when its kernels have ended and their status word has been read."""
    z, t, i, w = distill_inputs(4, 64, 3, torch.bfloat16, seed=47)
    v, dh, dn = norm_inputs((4, 64), torch.bfloat16, torch.float32, (), 1, seed=47)
    y, up = [v[n] for n in NAMES], torch.ones(4, 2, device="cuda")
    ops = torch.ops.muon_ascend950
    stats, rstd = ops.distill_topk(z, t, i, None, 1.0)[1], ops.residual_norm(*y, 1e-6)[2]
    chosen = ops.route_experts(z, None, 2, 0, 1, 1, 1, True, 1.0)[1]
    calls = [lambda: ops.distill_topk(z, t, i, None, 1.0), lambda: ops.distill_topk_grad(z, t, i, w, None, 1.0),
             lambda: ops.distill_topk_backward(w, z, t, i, None, stats, 1.0), lambda: ops.residual_norm(*y, 1e-6),
             lambda: ops.residual_norm_backward(dh, dn, *y, rstd, 1e-6, [True] * 6),
             lambda: ops.route_experts(z, None, 2, 0, 1, 1, 1, True, 1.0),
             lambda: ops.route_experts_backward(up, z, chosen, 0, True, 1.0)]
    for sync in (False, True):
        if sync:
            monkeypatch.setenv("MUON_POLAR_DEBUG_SYNC", "1")
        for call in calls:
            call()
            torch.cuda.synchronize()
            torch.cuda._sleep(100_000_000)  # some 50 ms before the call's kernels
            call()
            assert torch.cuda.current_stream().query() == sync


def test_kernels_are_launched_and_end(pkg):
    from muon_fusion_ascend950_b200.capi import capi

    api = capi()
    before = api.train_launch_count()
    pkg.route_experts(logits(4, 8), 2)
    assert api.train_launch_count() == before + 1
    assert api.train_device_status(torch.cuda.current_device()) == 0  # no wait has run out so far
