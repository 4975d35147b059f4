"""Measured cases of the training-step operators: the distillation loss over a
teacher's top logits, the norms around a residual block, and expert routing.

`listed()` and `draw()` give cases, `prepare()` makes a case's inputs on the
GPU, `run()` makes one pass: with `own` false in plain fp32 torch operations,
with `own` true through the package's entry points.  `exact()` is the same
result from the definitions in 64 bits, `work()` the bytes and operations a
pass cannot do without.
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
TINY = 1e-20  # added to the sum that renormalises the routing weights


# ------------------------------------------------------------------- cases
def listed():
    return [
        # the loss alone on a short validation snippet, small vocabulary: latency
        {"name": "distill_loss_short", "op": "distill", "mode": "loss", "rows": 16, "vocab": 8192, "top": 8,
         "dtype": "bf16", "index": "int64", "temperature": 1.0, "normalizer": False},
        # a training step through autograd, odd vocabulary (rows at every alignment), teacher's
        # lists read back from disk (int32), softened
        {"name": "distill_train_odd", "op": "distill", "mode": "train", "rows": 509, "vocab": 50001, "top": 32,
         "dtype": "bf16", "index": "int32", "temperature": 2.0, "normalizer": False},
        # fp32 logits of a smaller student, the teacher's own normaliser kept with its lists
        {"name": "distill_train_f32", "op": "distill", "mode": "train", "rows": 1024, "vocab": 32768, "top": 16,
         "dtype": "f32", "index": "int64", "temperature": 1.0, "normalizer": True},
        # the loss and its gradient in one call, a full batch over a large vocabulary
        {"name": "distill_grad_long", "op": "distill", "mode": "grad", "rows": 4096, "vocab": 131072, "top": 64,
         "dtype": "bf16", "index": "int64", "temperature": 1.0, "normalizer": False},
        # single tokens of four sequences, as in generation: latency
        {"name": "norm_tokens", "op": "norm", "mode": "forward", "batch": 4, "length": 1, "width": 2048,
         "dtype": "bf16", "params": "bf16", "gate": "none", "scale": "scalar"},
        # a ragged prompt, a learned gate for each channel
        {"name": "norm_prompt", "op": "norm", "mode": "forward", "batch": 3, "length": 683, "width": 4096,
         "dtype": "bf16", "params": "bf16", "gate": "channel", "scale": "none"},
        # an odd width, conditioned: one gate row for each sequence; forward and backward
        {"name": "norm_train_odd", "op": "norm", "mode": "train", "batch": 5, "length": 411, "width": 2050,
         "dtype": "bf16", "params": "f32", "gate": "sequence", "scale": "channel"},
        # a training batch, forward and backward, parameters kept in fp32
        {"name": "norm_train", "op": "norm", "mode": "train", "batch": 4, "length": 4096, "width": 4096,
         "dtype": "bf16", "params": "f32", "gate": "channel", "scale": "scalar"},
        # single tokens through a small router: latency
        {"name": "route_tokens", "op": "route", "mode": "forward", "tokens": 4, "experts": 64, "k": 6, "dtype": "bf16",
         "score": "softmax", "bias": False, "groups": 1, "top_groups": 1, "renormalize": True},
        # a prompt through a wide router with groups and the bias for balance
        {"name": "route_prompt", "op": "route", "mode": "forward", "tokens": 2053, "experts": 256, "k": 8, "dtype": "f32",
         "score": "sigmoid", "bias": True, "groups": 8, "top_groups": 4, "renormalize": True},
        # an odd number of experts in training, forward and backward
        {"name": "route_train_odd", "op": "route", "mode": "train", "tokens": 8191, "experts": 60, "k": 4, "dtype": "bf16",
         "score": "softmax", "bias": False, "groups": 1, "top_groups": 1, "renormalize": False},
        # a training batch through the wide router, forward and backward
        {"name": "route_train", "op": "route", "mode": "train", "tokens": 32768, "experts": 256, "k": 8, "dtype": "f32",
         "score": "sigmoid", "bias": True, "groups": 8, "top_groups": 4, "renormalize": True},
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["distill", "norm", "route"])
    if op == "distill":
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        vocab = _log_int(rng, 1000, 131072)
        rows = _log_int(rng, 1, min(4096, (1 << 30) // (vocab * SIZE[dtype])))
        return {"op": op, "mode": rng.choice(["loss", "train", "grad"]), "rows": rows, "vocab": vocab,
                "top": _log_int(rng, 1, 128), "dtype": dtype, "index": rng.choice(["int64", "int32"]),
                "temperature": rng.choice([1.0, 0.7, 2.0]), "normalizer": rng.random() < 0.3}
    if op == "norm":
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        batch = rng.randint(1, 8)
        length = _log_int(rng, 1, 16384 // batch)
        width = _log_int(rng, 64, min(8192, (1 << 27) // (batch * length * SIZE[dtype])))
        if rng.random() < 0.6:  # most widths keep rows on 16-byte boundaries
            width = max(80, width // 80 * 80)
        return {"op": op, "mode": rng.choice(["forward", "train", "train"]), "batch": batch, "length": length,
                "width": width, "dtype": dtype,
                "params": rng.choice(["own", "f32"]), "gate": rng.choice(["none", "channel", "sequence", "token"]),
                "scale": rng.choice(["none", "scalar", "channel"])}
    score = rng.choice(["softmax", "sigmoid"])
    groups = rng.choice([1, 1, 2, 4, 8])
    size = rng.randint(4, 384 // groups)
    top_groups = rng.randint(1, groups)
    return {"op": op, "mode": rng.choice(["forward", "train"]), "tokens": _log_int(rng, 1, 32768),
            "experts": groups * size, "k": rng.randint(1, min(16, top_groups * size)),
            "dtype": rng.choice(["bf16", "f32"]), "score": score, "bias": score == "sigmoid" and rng.random() < 0.7,
            "groups": groups, "top_groups": top_groups, "renormalize": rng.random() < 0.7}


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {"distill": _prepare_distill, "norm": _prepare_norm, "route": _prepare_route}[case["op"]](case, g)


def _prepare_distill(case, g):
    rows, vocab, tau = case["rows"], case["vocab"], case["temperature"]
    top = min(case["top"], vocab)
    dtype = TYPES[case["dtype"]]
    student = torch.empty(rows, vocab, dtype=dtype, device="cuda")
    values = torch.empty(rows, top, dtype=dtype, device="cuda")
    indices = torch.empty(rows, top, dtype=torch.int64, device="cuda")
    normalizer = torch.empty(rows, device="cuda")
    step = max(1, (1 << 26) // vocab)
    for r in range(0, rows, step):  # a teacher that the student follows in part
        teacher = torch.randn(min(step, rows - r), vocab, generator=g, device="cuda").mul_(2.5)
        student[r:r + step] = torch.randn(teacher.shape, generator=g, device="cuda").mul_(1.5).add_(teacher, alpha=0.8)
        v, i = teacher.topk(top, dim=-1)
        values[r:r + step], indices[r:r + step] = v, i
        normalizer[r:r + step] = teacher.div_(tau).logsumexp(-1)
    # prompt tokens have no list (but the first row has one), some rows a shorter one
    empty = torch.rand(rows, 1, generator=g, device="cuda") < 1 / 16
    empty[0] = False
    short = torch.rand(rows, 1, generator=g, device="cuda") < 1 / 8
    last = torch.arange(top, device="cuda") >= max(1, top - top // 4)
    indices.masked_fill_(empty | (short & last), -1)
    scale = (~empty).float().squeeze(1)
    return {"case": case, "student": student.requires_grad_(case["mode"] == "train"), "values": values,
            "indices": indices.to(torch.int32) if case["index"] == "int32" else indices,
            "normalizer": normalizer if case["normalizer"] else None, "row_scale": scale / scale.sum()}


def _prepare_norm(case, g):
    b, s, d = case["batch"], case["length"], case["width"]
    dtype = TYPES[case["dtype"]]
    params = dtype if case["params"] == "own" else TYPES[case["params"]]
    train = case["mode"] == "train"

    def rand(*shape, like, mean=0.0, std=1.0, grad=train):
        return torch.randn(*shape, generator=g, device="cuda").mul_(std).add_(mean).to(like).requires_grad_(grad)

    gates = {"channel": ((d,), params), "sequence": ((b, 1, d), dtype), "token": ((b, s, d), dtype)}
    scales = {"scalar": (1,), "channel": (d,)}
    state = {"case": case, "block_out": rand(b, s, d, like=dtype, std=3.0), "residual": rand(b, s, d, like=dtype),
             "post_weight": rand(d, like=params, mean=0.5, std=0.1), "pre_weight": rand(d, like=params, mean=1.0, std=0.1),
             "gate": None, "residual_scale": None}
    if case["gate"] != "none":
        shape, like = gates[case["gate"]]
        state["gate"] = rand(*shape, like=like, mean=0.7, std=0.3)
    if case["scale"] != "none":
        state["residual_scale"] = rand(*scales[case["scale"]], like=params, mean=0.9, std=0.05)
    if train:
        state["grads"] = [rand(b, s, d, like=dtype, std=1e-3, grad=False) for _ in range(2)]
    return state


def _prepare_route(case, g):
    t, e = case["tokens"], case["experts"]
    logits = torch.randn(t, e, generator=g, device="cuda").mul_(1.5).to(TYPES[case["dtype"]])
    bias = torch.randn(e, generator=g, device="cuda").mul_(0.05) if case["bias"] else None
    train = case["mode"] == "train"
    return {"case": case, "logits": logits.requires_grad_(train), "bias": bias,
            "scale": 2.5 if case["score"] == "sigmoid" else 1.0,
            "grad": torch.randn(t, case["k"], generator=g, device="cuda").mul_(1e-2) if train else None}


# -------------------------------------------------------------------- runs
def run(state):
    op = state["case"]["op"]
    if own:
        return {"distill": _own_distill, "norm": _own_norm, "route": _own_route}[op](state)
    with torch.no_grad():
        return {"distill": _plain_distill, "norm": _plain_norm, "route": _plain_route}[op](state)


def _own_distill(s):
    import muon_fusion_ascend950_b200 as m

    case = s["case"]
    if case["mode"] == "grad":
        loss, grad = m.distill_topk_grad(s["student"], s["values"], s["indices"], s["row_scale"],
                                         temperature=case["temperature"], teacher_lse=s["normalizer"])
        return {"loss": loss, "grad": grad}
    loss = m.distill_topk(s["student"], s["values"], s["indices"], temperature=case["temperature"],
                          teacher_lse=s["normalizer"])
    if case["mode"] == "loss":
        return {"loss": loss}
    (grad,) = torch.autograd.grad(loss, s["student"], s["row_scale"])
    return {"loss": loss, "grad": grad}


def _plain_distill(s):
    case, tau, index = s["case"], s["case"]["temperature"], s["indices"].long()
    z = s["student"].float() / tau
    top = z.amax(-1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(-1, keepdim=True)
    lse = (top + torch.log(total)).squeeze(1)
    t = s["values"].float() / tau
    valid = (index >= 0) & (index < z.shape[1]) & (t > -math.inf)
    if s["normalizer"] is None:
        t = torch.where(valid, t, torch.full_like(t, -math.inf))
        best = t.amax(-1, keepdim=True)
        best = torch.where(best > -math.inf, best, torch.zeros_like(best))
        sums = torch.exp(t - best).sum(-1, keepdim=True)
        log_q = t - best - torch.log(torch.where(sums > 0, sums, torch.ones_like(sums)))
    else:
        log_q = t - s["normalizer"][:, None]
    q = torch.where(valid, torch.exp(log_q), torch.zeros_like(t))
    index = torch.where(valid, index, torch.zeros_like(index))
    terms = q * (log_q - z.gather(1, index) + lse[:, None])
    loss = torch.where(valid & (q > 0), terms, torch.zeros_like(terms)).sum(-1)
    if case["mode"] == "loss":
        return {"loss": loss}
    grad = e.mul_(q.sum(-1, keepdim=True) / total).scatter_add_(1, index, -q)
    grad = grad.mul_((s["row_scale"] / tau)[:, None])
    return {"loss": loss, "grad": grad.to(s["student"].dtype)}


NORM_INPUTS = ("block_out", "residual", "post_weight", "pre_weight", "gate", "residual_scale")


def _own_norm(s):
    import muon_fusion_ascend950_b200 as m

    hidden, normed = m.residual_norm(s["block_out"], s["residual"], s["post_weight"], s["pre_weight"], gate=s["gate"],
                                     residual_scale=s["residual_scale"])
    out = {"hidden": hidden, "normed": normed}
    if s["case"]["mode"] == "train":
        names = [n for n in NORM_INPUTS if s[n] is not None]
        for n, v in zip(names, torch.autograd.grad([hidden, normed], [s[n] for n in names], s["grads"])):
            out["grad_" + n] = v
    return out


def _plain_norm(s, eps=1e-6):
    case, dtype = s["case"], s["block_out"].dtype
    y, x, w, p = (s[n].float() for n in NORM_INPUTS[:4])
    r = torch.rsqrt((y * y).mean(-1, keepdim=True) + eps)
    unit = y * r
    gate = 1.0 if s["gate"] is None else s["gate"].float()
    scale = 1.0 if s["residual_scale"] is None else s["residual_scale"].float()
    h = x * scale + unit * w * gate
    rh = torch.rsqrt((h * h).mean(-1, keepdim=True) + eps)
    hn = h * rh
    out = {"hidden": h.to(dtype), "normed": (hn * p).to(dtype)}
    if case["mode"] != "train":
        return out
    dh, dn = (v.float() for v in s["grads"])
    a = dn * p
    d = dh + rh * (a - hn * (a * hn).mean(-1, keepdim=True))
    b = d * gate * w
    out["grad_block_out"] = (r * (b - unit * (b * unit).mean(-1, keepdim=True))).to(dtype)
    out["grad_residual"] = (d * scale).to(dtype)
    out["grad_post_weight"] = (d * gate * unit).sum((0, 1)).to(s["post_weight"].dtype)
    out["grad_pre_weight"] = (dn * hn).sum((0, 1)).to(s["pre_weight"].dtype)
    if s["gate"] is not None:
        full = d * unit * w
        over = {"channel": full.sum((0, 1)), "sequence": full.sum(1, keepdim=True), "token": full}
        out["grad_gate"] = over[case["gate"]].to(s["gate"].dtype)
    if s["residual_scale"] is not None:
        full = (d * x).sum((0, 1))
        out["grad_residual_scale"] = (full.sum(0, keepdim=True) if case["scale"] == "scalar" else full).to(
            s["residual_scale"].dtype)
    return out


def _own_route(s):
    import muon_fusion_ascend950_b200 as m

    case = s["case"]
    weights, indices, counts = m.route_experts(
        s["logits"], case["k"], score=case["score"], bias=s["bias"], groups=case["groups"],
        top_groups=case["top_groups"], renormalize=case["renormalize"], scale=s["scale"])
    out = {"weights": weights, "indices": indices, "counts": counts}
    if case["mode"] == "train":
        (out["grad"],) = torch.autograd.grad(weights, s["logits"], s["grad"])
    return out


def _plain_route(s):
    case, x = s["case"], s["logits"].float()
    t, e, k = case["tokens"], case["experts"], case["k"]
    if case["score"] == "softmax":
        ex = torch.exp(x - x.amax(-1, keepdim=True))
        score, key = ex / ex.sum(-1, keepdim=True), x  # the softmax keeps the logits' order
    else:
        score = key = 1.0 / (1.0 + torch.exp(-x))
    if s["bias"] is not None:
        key = score + s["bias"]
    if case["groups"] > 1:
        size = e // case["groups"]
        # ties go to the lowest index: a stable sort, and not topk
        grouped = key.view(t, case["groups"], size).sort(dim=-1, descending=True, stable=True).values
        group_key = grouped[..., 0] + grouped[..., 1] if case["score"] == "sigmoid" else grouped[..., 0]
        best = group_key.sort(dim=-1, descending=True, stable=True).indices[:, :case["top_groups"]]
        keep = torch.zeros(t, case["groups"], dtype=torch.bool, device=x.device).scatter_(1, best, True)
        key = torch.where(keep.repeat_interleave(size, 1), key, torch.full_like(key, -math.inf))
    indices = key.sort(dim=-1, descending=True, stable=True).indices[:, :k]
    chosen = score.gather(1, indices)
    total = chosen.sum(-1, keepdim=True) + TINY if case["renormalize"] else torch.ones_like(chosen[:, :1])
    share = chosen / total
    counts = torch.zeros(e, dtype=torch.int64, device=x.device)
    counts.scatter_add_(0, indices.reshape(-1), torch.ones_like(indices.reshape(-1)))
    out = {"weights": share * s["scale"], "indices": indices.contiguous(), "counts": counts}
    if case["mode"] == "train":
        d = s["grad"] * s["scale"]
        if case["renormalize"]:
            d = (d - (d * share).sum(-1, keepdim=True)) / total
        d = torch.zeros_like(x).scatter_(1, indices, d)
        if case["score"] == "softmax":
            d = score * (d - (d * score).sum(-1, keepdim=True))
        else:
            d = d * score * (1.0 - score)
        out["grad"] = d.to(s["logits"].dtype)
    return out


# ------------------------------------------------------------------- exact
def exact(case, seed):
    state = prepare(case, seed)
    return {"distill": _exact_distill, "norm": _exact_norm, "route": _exact_route}[case["op"]](state)


def _exact_distill(s):
    case, tau, vocab = s["case"], s["case"]["temperature"], s["case"]["vocab"]
    losses, grads = [], []
    step = max(1, (1 << 26) // vocab)
    for r in range(0, case["rows"], step):
        z = s["student"][r:r + step].detach().double().requires_grad_(True)
        t, i = s["values"][r:r + step].double() / tau, s["indices"][r:r + step].long()
        inside = (i >= 0) & (i < vocab)
        if s["normalizer"] is None:
            log_q = torch.log_softmax(t.masked_fill(~inside, -math.inf), -1)
        else:
            log_q = t - s["normalizer"][r:r + step, None].double()
        q = torch.where(inside, log_q.exp(), 0.0)
        log_p = torch.log_softmax(z / tau, -1).gather(1, i.clamp(0, vocab - 1))
        loss = torch.where(inside, q * (log_q - log_p), 0.0).sum(-1)
        losses.append(loss.detach())
        if case["mode"] != "loss":
            grads.append(torch.autograd.grad(loss, z, s["row_scale"][r:r + step].double())[0])
    out = {"loss": torch.cat(losses)}
    if grads:
        out["grad"] = torch.cat(grads)
    return out


def _exact_norm(s, eps=1e-6):
    names = [n for n in NORM_INPUTS if s[n] is not None]
    v = {n: s[n].detach().double().requires_grad_(True) for n in names}

    def rms(a):
        return a / (a.pow(2).mean(-1, keepdim=True) + eps).sqrt()

    hidden = rms(v["block_out"]) * v["post_weight"] * v.get("gate", 1.0) + v.get("residual_scale", 1.0) * v["residual"]
    normed = rms(hidden) * v["pre_weight"]
    out = {"hidden": hidden.detach(), "normed": normed.detach()}
    if s["case"]["mode"] == "train":
        grads = torch.autograd.grad([hidden, normed], [v[n] for n in names], [g.double() for g in s["grads"]])
        out.update({"grad_" + n: g for n, g in zip(names, grads)})
    return out


def _exact_route(s):
    case = s["case"]
    x = s["logits"].detach().double().requires_grad_(True)
    score = x.softmax(-1) if case["score"] == "softmax" else x.sigmoid()
    key = score.detach() if s["bias"] is None else score.detach() + s["bias"].double()
    if case["groups"] > 1:
        parts = key.unflatten(-1, (case["groups"], -1))
        group_key = parts.topk(2, -1).values.sum(-1) if case["score"] == "sigmoid" else parts.amax(-1)
        cut = group_key.topk(case["top_groups"], -1).values[:, -1:]
        key = parts.masked_fill((group_key < cut)[..., None], -math.inf).flatten(-2)
    chosen = score.gather(1, key.sort(dim=-1, descending=True, stable=True).indices[:, :case["k"]])
    weights = s["scale"] * (chosen / (chosen.sum(-1, keepdim=True) + TINY) if case["renormalize"] else chosen)
    out = {"weights": weights.detach(), "indices": None, "counts": None}
    if case["mode"] == "train":
        out["grad"] = torch.autograd.grad(weights, x, s["grad"].double())[0]
    return out


# -------------------------------------------------------------------- work
def work(case):
    if case["op"] == "distill":
        n, grad = case["rows"] * case["vocab"], case["mode"] != "loss"
        lists = case["rows"] * case["top"] * (SIZE[case["dtype"]] + (4 if case["index"] == "int32" else 8))
        per_row = 4 + (4 if grad else 0) + (4 if case["normalizer"] else 0)
        return {"bytes": n * SIZE[case["dtype"]] * (2 if grad else 1) + lists + case["rows"] * per_row,
                "flops": n * (7 if grad else 4)}
    if case["op"] == "norm":
        n, d = case["batch"] * case["length"] * case["width"], case["width"]
        train, size = case["mode"] == "train", SIZE[case["dtype"]]
        psize = size if case["params"] == "own" else SIZE[case["params"]]
        small = 2 * d * psize + {"none": 0, "scalar": 1, "channel": d}[case["scale"]] * psize
        small += {"none": 0, "channel": d * psize, "sequence": case["batch"] * d * size, "token": n * size}[case["gate"]]
        return {"bytes": n * size * (8 if train else 4) + small * (2 if train else 1), "flops": n * (36 if train else 11)}
    n, pairs, train = case["tokens"] * case["experts"], case["tokens"] * case["k"], case["mode"] == "train"
    size = SIZE[case["dtype"]]
    small = case["experts"] * (12 if case["bias"] else 8) + pairs * (16 if train else 12)
    return {"bytes": n * size * (2 if train else 1) + small, "flops": n * (10 if train else 5)}
