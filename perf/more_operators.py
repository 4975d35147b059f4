"""Measured cases of the operators of a transformer's training step: attention
with its backward pass, rotary positions, and the global gradient norm with
clipping.

`listed()` and `draw()` give cases, `prepare()` makes a case's inputs on the
GPU, `run()` makes one pass: with `own` false in plain fp32 torch operations,
with `own` true through the package's entry points.  `exact()` is the same
result from the definitions in 64 bits, `work()` the bytes and operations a
pass cannot do without.
"""
import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}


# ------------------------------------------------------------------- cases
def listed():
    return [
        # two short snippets scored together, a small model: latency
        {"name": "attention_snippets", "op": "attention", "mode": "forward", "kind": "dense", "batch": 2, "length": 33,
         "keys": 33, "heads": 4, "kv_heads": 4, "dim": 64, "dtype": "bf16", "causal": True, "window": 0, "fused": False},
        # a held-out text of odd length, query heads that share key heads, slices of one projection
        {"name": "attention_prompt", "op": "attention", "mode": "forward", "kind": "dense", "batch": 1, "length": 4097,
         "keys": 4097, "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bf16", "causal": True, "window": 0, "fused": True},
        # documents of many lengths packed one after another, a sliding window, fp16: forward and backward
        {"name": "attention_train_packed", "op": "attention", "mode": "train", "kind": "packed", "batch": 11, "length": 8191,
         "keys": 8191, "heads": 16, "kv_heads": 16, "dim": 64, "dtype": "f16", "causal": True, "window": 512, "fused": True},
        # a training batch, forward and backward
        {"name": "attention_train", "op": "attention", "mode": "train", "kind": "dense", "batch": 4, "length": 4096,
         "keys": 4096, "heads": 16, "kv_heads": 4, "dim": 128, "dtype": "bf16", "causal": True, "window": 0, "fused": True},
        # both directions over long padded texts, forward and backward
        {"name": "attention_train_both", "op": "attention", "mode": "train", "kind": "padded", "batch": 2, "length": 8192,
         "keys": 8192, "heads": 16, "kv_heads": 16, "dim": 128, "dtype": "bf16", "causal": False, "window": 0, "fused": False},
        # single tokens of four sequences, as in generation: latency
        {"name": "rotary_tokens", "op": "rotary", "mode": "forward", "batch": 4, "length": 1, "heads": 16, "kv_heads": 4,
         "dim": 128, "rotated": 128, "dtype": "bf16", "interleaved": False, "first": 4095, "factor": 1.0, "fused": True},
        # part of the head in neighbouring pairs, fp32, positions stretched far beyond the trained length
        {"name": "rotary_train_far", "op": "rotary", "mode": "train", "batch": 3, "length": 1367, "heads": 12, "kv_heads": 12,
         "dim": 80, "rotated": 48, "dtype": "f32", "interleaved": True, "first": 1000000, "factor": 32.0, "fused": False},
        # a training batch, forward and backward
        {"name": "rotary_train", "op": "rotary", "mode": "train", "batch": 4, "length": 4096, "heads": 32, "kv_heads": 8,
         "dim": 128, "rotated": 128, "dtype": "bf16", "interleaved": False, "first": 0, "factor": 1.0, "fused": True},
        # a small model whose gradients are within the limit, in place: latency
        {"name": "clip_small", "op": "clip", "tensors": 24, "total": 200000, "dtype": "f32", "out": "none", "norm": 2,
         "over": False, "packed": False},
        # matrices in bf16 and vectors in fp32 that lie at any offset, clipped into fp32
        {"name": "clip_mixed", "op": "clip", "tensors": 157, "total": 20000003, "dtype": "mixed", "out": "f32", "norm": 2,
         "over": True, "packed": True},
        # gradients accumulated in fp32 over micro-batches, clipped into the parameters' type
        {"name": "clip_accumulated", "op": "clip", "tensors": 291, "total": 160000000, "dtype": "f32", "out": "bf16",
         "norm": 2, "over": True, "packed": False},
        # a larger model in bf16, a step within the limit, in place
        {"name": "clip_large", "op": "clip", "tensors": 435, "total": 640000000, "dtype": "bf16", "out": "none", "norm": 2,
         "over": False, "packed": False},
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "rotary", "clip"])
    if op == "attention":
        mode = rng.choice(["forward", "train", "train"])
        kind = rng.choice(["dense", "dense", "padded", "packed"])
        batch = rng.randint(1, 16 if kind == "packed" else 8)
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 3, 4, 8])
        dim = rng.choice([64, 128, 128, 8 * rng.randint(4, 16)])
        rows = 3 if kind == "packed" else batch
        most = int(min(8192, math.sqrt((1 << 31) / (rows * heads)), (1 << 25) / (rows * heads * dim)))
        # one token alone has nothing to learn: its gradients of queries and keys are 0
        least = 1 if mode == "forward" else 8 * batch if kind == "packed" else 16
        length = _log_int(rng, least, most)
        keys = _log_int(rng, least, most) if kind == "dense" and rng.random() < 0.3 else length
        return {"op": op, "mode": mode, "kind": kind, "batch": batch, "length": length,
                "keys": keys, "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": rng.choice(["bf16", "bf16", "f16"]),
                "causal": rng.random() < 0.7, "window": rng.choice([0, 0, _log_int(rng, 4, 2 * length)]),
                "fused": keys == length and rng.random() < 0.5}
    if op == "rotary":
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 3, 4, 8])
        dim = rng.choice([64, 128, 128, 2 * rng.randint(8, 128)])
        batch = rng.randint(1, 8)
        most = 80000000 // ((heads + kv_heads) * dim * batch) // (2 if dtype == "f32" else 1)
        return {"op": op, "mode": rng.choice(["forward", "train"]), "batch": batch, "length": _log_int(rng, 1, min(65536, most)),
                "heads": heads, "kv_heads": kv_heads, "dim": dim, "rotated": rng.choice([dim, dim, 2 * rng.randint(1, dim // 2)]),
                "dtype": dtype, "interleaved": rng.random() < 0.4, "first": rng.choice([0, 0, _log_int(rng, 1, 10000000)]),
                "factor": rng.choice([1.0, 1.0, 4.0, 32.0]), "fused": rng.random() < 0.5}
    dtype = rng.choice(["bf16", "f32", "f32", "f16", "mixed"])
    total = _log_int(rng, 1000, 160000000)
    out = rng.choice(["none", "bf16", "f32"])
    # in place only within the limit, so that the next pass meets the same gradients
    return {"op": op, "tensors": _log_int(rng, 1, min(700, total // 20)), "total": total, "dtype": dtype, "out": out,
            "norm": rng.choice([2, 2, 0]), "over": out != "none" and rng.random() < 0.7, "packed": rng.random() < 0.3}


def _sizes(case):
    """Lengths of a case's sequences, or sizes of its tensors: the same for every seed."""
    rng = random.Random("%s %s" % (case["op"], sorted((k, v) for k, v in case.items() if k != "name")))
    if case["op"] == "clip":
        # half of the tensors are vectors, the others matrices that share the rest
        count, total = case["tensors"], case["total"]
        small = [min(rng.choice([1, 64, 1000, 4096]), total // (2 * count)) for _ in range(count // 2)]
        weights = [rng.choice([1, 1, 2.7, 4]) for _ in range(count - len(small))]
        rest = total - sum(small)
        large = [int(rest * w / sum(weights)) for w in weights]
        large[0] += rest - sum(large)
        return small, large
    if case["kind"] == "packed":  # documents of many lengths, some empty, and tokens behind the last
        cuts = sorted(int(case["length"] * rng.random() ** 0.8) for _ in range(case["batch"] - 1))
        ends = cuts + [case["length"] - rng.randint(0, min(3, case["length"]))]
        return [max(0, b - a) for a, b in zip([0] + cuts, ends)]
    if case["kind"] == "padded":
        return [case["length"] if b == 0 else rng.randint(case["length"] // 2, case["length"]) for b in range(case["batch"])]
    return [case["length"]] * case["batch"]


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {"attention": _prepare_attention, "rotary": _prepare_rotary, "clip": _prepare_clip}[case["op"]](case, g)


def _randn(shape, g, dtype, std=1.0):
    return torch.randn(shape, generator=g, device="cuda").mul_(std).to(dtype)


def _heads(case, lead, keys, g):
    """Queries, keys (and values) apart, or as slices of one projection."""
    d, h, hk, dtype = case["dim"], case["heads"], case["kv_heads"], TYPES[case["dtype"]]
    sizes = [h, hk, hk] if case["op"] == "attention" else [h, hk]
    if case["fused"]:
        all_heads = _randn((*lead, sum(sizes), d), g, dtype)
        return list(all_heads.split(sizes, dim=-2))
    return [_randn((*(lead if i == 0 else keys), n, d), g, dtype) for i, n in enumerate(sizes)]


def _prepare_attention(case, g):
    packed, train, dtype = case["kind"] == "packed", case["mode"] == "train", TYPES[case["dtype"]]
    lead = (case["length"],) if packed else (case["batch"], case["length"])
    keys = (case["keys"],) if packed else (case["batch"], case["keys"])
    q, k, v = _heads(case, lead, keys, g)
    # some heads look almost evenly at all keys, others at few
    q.mul_(torch.linspace(0.5, 2.5, case["heads"], device="cuda").to(dtype)[:, None])
    lengths = _sizes(case)
    state = {"case": case, "q": q.requires_grad_(train), "k": k.requires_grad_(train), "v": v.requires_grad_(train),
             "longest": max(lengths + [1]), "offsets": None, "lengths": None}
    counts = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    if packed:
        state["offsets"] = torch.cat([counts.new_zeros(1), counts.cumsum(0, dtype=torch.int32)])
    elif case["kind"] == "padded":
        state["lengths"] = counts
    if train:
        state["grad"] = _randn((*lead, case["heads"], case["dim"]), g, dtype, 0.05)
    return state


def _frequencies(case):
    """Radians a position of each pair, and what cosine and sine are multiplied with: beyond the trained length, slow
    pairs turn `factor` times slower, with a ramp between them and the fast ones, which stay."""
    pairs = case["rotated"] // 2
    freq = 10000.0 ** (-torch.arange(pairs, dtype=torch.float64) / pairs)
    if case["factor"] == 1.0:
        return freq, 1.0
    turns = 4096 * freq / (2 * math.pi)
    keep = ((turns - 1) / 31).clamp(0, 1)
    return freq * (keep + (1 - keep) / case["factor"]), 0.1 * math.log(case["factor"]) + 1.0


def _prepare_rotary(case, g):
    train, lead = case["mode"] == "train", (case["batch"], case["length"])
    q, k = _heads(case, lead, lead, g)
    freq, scale = _frequencies(case)
    positions = case["first"] + torch.arange(case["length"], device="cuda").expand(lead)
    if case["batch"] > 1:  # every sequence stands somewhere else
        positions = positions + 17 * torch.randint(0, 64, (case["batch"], 1), generator=g, device="cuda")
    state = {"case": case, "q": q.requires_grad_(train), "k": k.requires_grad_(train), "positions": positions.contiguous(),
             "frequencies": freq.cuda(), "scale": scale}
    if train:
        state["grads"] = [_randn(t.shape, g, t.dtype, 0.05) for t in (q, k)]
    return state


def _prepare_clip(case, g):
    small, large = _sizes(case)
    kinds = {"f32": small, "bf16": large} if case["dtype"] == "mixed" else {case["dtype"]: small + large}
    state = {"case": case, "flat": [], "grads": [], "out_flat": [], "out": None}
    outs = []
    for kind, sizes in kinds.items():
        if not sizes:
            continue
        # one buffer a type; each tensor begins on 256 bytes, or right behind the one before
        step = 1 if case["packed"] else 128
        places = [0]
        for n in sizes:
            places.append(places[-1] + -(-n // step) * step)
        total = places[-1]
        flat = torch.zeros(total, dtype=TYPES[kind], device="cuda")
        out = torch.zeros(total, dtype=TYPES[case["out"]], device="cuda") if case["out"] != "none" else None
        for a in range(0, total, 1 << 27):
            part = flat[a:a + (1 << 27)]
            part.copy_(torch.randn(part.shape, generator=g, device="cuda").mul_(1e-3))
        if not case["packed"]:  # nothing stands between the tensors
            used = torch.zeros(total + 1, dtype=torch.int32, device="cuda")
            at = torch.tensor([(p, p + n) for p, n in zip(places, sizes) if n], device="cuda").T
            used.index_add_(0, at[0], torch.ones_like(at[0], dtype=torch.int32))
            used.index_add_(0, at[1], -torch.ones_like(at[1], dtype=torch.int32))
            flat.mul_(used[:-1].cumsum_(0)[:total].to(flat.dtype))
        state["flat"].append(flat)
        state["grads"] += [flat[p:p + n] for p, n in zip(places, sizes)]
        if out is not None:
            state["out_flat"].append(out)
            outs += [out[p:p + n] for p, n in zip(places, sizes)]
    state["out"] = outs or None
    # the norm to be expected, and a limit on one side of it
    expected = 1e-3 * math.sqrt(case["total"]) if case["norm"] == 2 else 3e-3
    state["max_norm"] = expected * (0.25 if case["over"] else 4.0)
    return state


# -------------------------------------------------------------------- runs
def run(state):
    op = state["case"]["op"]
    if own:
        return {"attention": _own_attention, "rotary": _own_rotary, "clip": _own_clip}[op](state)
    with torch.no_grad():
        return {"attention": _plain_attention, "rotary": _plain_rotary, "clip": _plain_clip}[op](state)


def _own_attention(s):
    import muon_fusion_ascend950_b200 as m

    case = s["case"]
    out = m.attention(s["q"], s["k"], s["v"], causal=case["causal"], window=case["window"] or None, offsets=s["offsets"],
                      lengths=s["lengths"])
    if case["mode"] == "forward":
        return {"out": out}
    grads = torch.autograd.grad(out, [s["q"], s["k"], s["v"]], s["grad"])
    return {"out": out, "grad_q": grads[0], "grad_k": grads[1], "grad_v": grads[2]}


def _plain_attention(s):
    case, dtype = s["case"], s["q"].dtype
    tensors = [s["q"], s["k"], s["v"]] + ([s["grad"]] if case["mode"] == "train" else [])
    if case["kind"] == "packed":  # each document as a row of a padded batch; absent tokens come from and go to a row behind
        total, longest = case["length"], s["longest"]
        first, last = s["offsets"][:-1].long(), s["offsets"][1:].long()
        rows = first[:, None] + torch.arange(longest, device=first.device)
        rows = torch.where(rows < last[:, None], rows, torch.full_like(rows, total))
        tensors = [torch.cat([t, torch.zeros_like(t[:1])])[rows] for t in tensors]
        counts = last - first
    else:
        counts = s["lengths"].long() if s["lengths"] is not None else None
    # [batch, kv heads, heads of the group, length, dim]; the keys' third size is 1
    q, k, v, *grad = (t.float().unflatten(2, (case["kv_heads"], -1)).permute(0, 2, 3, 1, 4) for t in tensors)
    length, keys = q.shape[3], k.shape[3]
    i = torch.arange(length, device=q.device)[:, None] + (keys - length)
    j = torch.arange(keys, device=q.device)
    see = torch.ones(1, 1, 1, length, keys, dtype=torch.bool, device=q.device)
    if case["causal"]:
        see = see & (j <= i)
    if case["window"]:
        see = see & (j > i - case["window"])
        if not case["causal"]:
            see = see & (j < i + case["window"])
    if counts is not None:
        here = torch.arange(length, device=q.device) < counts[:, None]
        see = see & (here[:, None, None, :, None] & here[:, None, None, None, :])
    scale = case["dim"] ** -0.5
    p = torch.matmul(q * scale, k.transpose(-1, -2))
    p = p.masked_fill_(~see, -math.inf)
    top = p.amax(-1, keepdim=True)
    p = p.sub_(torch.where(top > -math.inf, top, torch.zeros_like(top))).exp_()
    sums = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(sums > 0, sums, torch.ones_like(sums)))
    out = {"out": torch.matmul(p, v)}
    if case["mode"] == "train":
        out["grad_v"] = torch.matmul(p.transpose(-1, -2), grad[0]).sum(2, keepdim=True)
        ds = torch.matmul(grad[0], v.transpose(-1, -2))
        ds = ds.sub_((grad[0] * out["out"]).sum(-1, keepdim=True)).mul_(p)
        out["grad_q"] = torch.matmul(ds, k) * scale
        out["grad_k"] = torch.matmul(ds.transpose(-1, -2), q).sum(2, keepdim=True) * scale
    out = {n: t.permute(0, 3, 1, 2, 4).flatten(2, 3) for n, t in out.items()}
    if case["kind"] == "packed":
        out = {n: t.new_zeros((total + 1, *t.shape[2:])).index_copy_(0, rows.flatten(), t.flatten(0, 1))[:total]
               for n, t in out.items()}
    return {n: t.to(dtype) for n, t in out.items()}


def _own_rotary(s):
    import muon_fusion_ascend950_b200 as m

    case = s["case"]
    q, k = m.rotary(s["q"], s["k"], s["positions"], s["frequencies"], interleaved=case["interleaved"], scale=s["scale"])
    out = {"q": q, "k": k}
    if case["mode"] == "train":
        out["grad_q"], out["grad_k"] = torch.autograd.grad([q, k], [s["q"], s["k"]], s["grads"])
    return out


def _plain_rotary(s):
    case = s["case"]
    angle = s["positions"].double()[..., None, None] * s["frequencies"]
    cos, sin = ((f(angle) * s["scale"]).float() for f in (torch.cos, torch.sin))
    out = {"q": _turn(case, s["q"], cos, sin), "k": _turn(case, s["k"], cos, sin)}
    if case["mode"] == "train":
        out["grad_q"], out["grad_k"] = (_turn(case, t, cos, -sin) for t in s["grads"])
    return out


def _turn(case, t, cos, sin):
    r = case["rotated"]
    x = t[..., :r].float()
    a, b = (x[..., 0::2], x[..., 1::2]) if case["interleaved"] else (x[..., :r // 2], x[..., r // 2:])
    parts = [a * cos - b * sin, b * cos + a * sin]
    turned = torch.stack(parts, -1).flatten(-2) if case["interleaved"] else torch.cat(parts, -1)
    return torch.cat([turned.to(t.dtype), t[..., r:]], -1)


def _own_clip(s):
    import muon_fusion_ascend950_b200 as m

    case = s["case"]
    norm = m.clip_gradients(s["grads"], s["max_norm"], norm_type=2.0 if case["norm"] == 2 else math.inf, out=s["out"])
    return {"norm": norm, "out": s["out_flat"] if s["out"] is not None else s["flat"]}


def _plain_clip(s):
    if s["case"]["norm"] == 2:
        norm = torch.stack([f.float().square().sum(dtype=torch.float64) for f in s["flat"]]).sum().sqrt()
    else:
        norm = torch.stack([f.float().abs().amax() for f in s["flat"]]).amax().double()
    factor = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
    to = s["out_flat"] if s["out"] is not None else s["flat"]
    return {"norm": norm.float(), "out": [o.copy_(f.float() * factor) for o, f in zip(to, s["flat"])]}


# ------------------------------------------------------------------- exact
def exact(case, seed):
    state = prepare(case, seed)
    return {"attention": _exact_attention, "rotary": _exact_rotary, "clip": _exact_clip}[case["op"]](state)


def _exact_attention(s):
    case, train = s["case"], s["case"]["mode"] == "train"
    group = case["heads"] // case["kv_heads"]
    results = {"out": torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")}
    if train:
        results.update({"grad_" + n: torch.zeros(s[n].shape, dtype=torch.float64, device="cuda") for n in "qkv"})
    first = 0
    for b, n in enumerate(_sizes(case)):
        if case["kind"] == "packed":
            rows = keys = (slice(first, first + n),)
            first += n
        else:
            rows = (b, slice(0, n))
            keys = (b, slice(0, n if case["keys"] == case["length"] else case["keys"]))
        for h in range(case["heads"]):
            one = {"q": s["q"][rows][:, h], "k": s["k"][keys][:, h // group], "v": s["v"][keys][:, h // group]}
            one = {name: t.detach().double().requires_grad_(train) for name, t in one.items()}
            nq, nk = one["q"].shape[0], one["k"].shape[0]
            if nq == 0 or nk == 0:
                continue
            score = one["q"] @ one["k"].T / math.sqrt(case["dim"])
            # how far key j stands behind query i, both counted from the end (padding aside)
            shift = case["keys"] - case["length"]
            behind = torch.arange(nq, device="cuda")[:, None] + shift - torch.arange(nk, device="cuda")[None]
            hidden = torch.zeros_like(behind, dtype=torch.bool)
            if case["causal"]:
                hidden |= behind < 0
            if case["window"]:
                hidden |= behind.abs() >= case["window"]
            none = hidden.all(1, keepdim=True)
            p = torch.softmax(score.masked_fill(hidden & ~none, -math.inf), -1)
            out = p.masked_fill(none, 0.0) @ one["v"]
            results["out"][rows][:, h] = out.detach()
            if train:
                grads = torch.autograd.grad(out, [one["q"], one["k"], one["v"]], s["grad"][rows][:, h].double())
                results["grad_q"][rows][:, h] = grads[0]
                results["grad_k"][keys][:, h // group] += grads[1]
                results["grad_v"][keys][:, h // group] += grads[2]
    return results


def _exact_rotary(s):
    case = s["case"]
    pairs = case["rotated"] // 2
    # one complex number a pair, turned by a complex factor
    factor = s["scale"] * torch.exp(1j * (s["positions"].double()[..., None] * s["frequencies"]))[:, :, None, :]

    def turn(t, by):
        t = t.detach().double().clone()
        shape = (*t.shape[:-1], pairs, 2) if case["interleaved"] else (*t.shape[:-1], 2, pairs)
        x = t[..., :2 * pairs].reshape(shape)
        x = x if case["interleaved"] else x.transpose(-1, -2)
        y = torch.view_as_real(torch.view_as_complex(x.contiguous()) * by)
        y = y if case["interleaved"] else y.transpose(-1, -2)
        t[..., :2 * pairs] = y.flatten(-2)
        return t

    out = {"q": turn(s["q"], factor), "k": turn(s["k"], factor)}
    if case["mode"] == "train":
        out["grad_q"], out["grad_k"] = (turn(t, factor.conj()) for t in s["grads"])
    return out


def _exact_clip(s):
    grads = [f.double() for f in s["flat"]]
    if s["case"]["norm"] == 2:
        norm = math.sqrt(sum(float(torch.dot(f, f)) for f in grads))
    else:
        norm = max(float(f.abs().max()) for f in grads)
    factor = min(1.0, s["max_norm"] / (norm + 1e-6))
    return {"norm": torch.tensor(norm, dtype=torch.float64, device="cuda"), "out": [f * factor for f in grads]}


# -------------------------------------------------------------------- work
def _pairs(case):
    """Pairs of query and key that see each other, of one head."""
    pairs, shift = 0, case["keys"] - case["length"]
    for n in _sizes(case):
        keys = case["keys"] if case["kind"] == "dense" else n
        for i in range(n):
            low, high = 0, keys
            if case["causal"]:
                high = min(keys, i + shift + 1)
            if case["window"]:
                low = max(0, i + shift - case["window"] + 1)
                high = min(high, i + shift + case["window"])
            pairs += max(0, high - low)
    return pairs


def work(case):
    size = SIZE.get(case["dtype"], 2)
    if case["op"] == "attention":
        rows = 1 if case["kind"] == "packed" else case["batch"]
        query = rows * case["length"] * case["heads"] * case["dim"] * size
        key = rows * case["keys"] * case["kv_heads"] * case["dim"] * size
        train = case["mode"] == "train"
        # q, k, v and the output; with gradients the output's and those of q, k and v
        return {"bytes": (4 if train else 2) * query + (4 if train else 2) * key,
                "flops": _pairs(case) * case["heads"] * case["dim"] * (14 if train else 4)}
    if case["op"] == "rotary":
        n = case["batch"] * case["length"] * (case["heads"] + case["kv_heads"])
        both = 2 if case["mode"] == "train" else 1
        return {"bytes": both * (2 * n * case["dim"] * size + 8 * case["batch"] * case["length"]),
                "flops": both * 3 * n * case["rotated"]}
    small, large = (sum(part) for part in _sizes(case))
    read = (small * 4 if case["dtype"] == "mixed" else small * size) + large * size
    # in place, gradients within the limit stay as they are
    write = case["total"] * SIZE[case["out"]] if case["out"] != "none" else read if case["over"] else 0
    return {"bytes": read + write, "flops": case["total"] * (3 if write else 2)}
