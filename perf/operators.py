"""Timed cases of the mixture-of-experts operators and the 4-bit products.

Three families, as a sparse feed-forward layer uses them:

* ``route`` / ``exchange``: the router's top-k selection with its gradient, the
  grouping of the tokens by expert, and the movement of the rows there
  (dispatch) and back (weighted combine), each with its gradient
  (``tempname_dcu_b200.ops.moe``);
* ``linear``, ``linear_gelu``, ``data_grad``, ``weight_grad``: matrix products
  grouped by expert, group g holding the rows [offsets[g], offsets[g+1])
  (``tempname_dcu_b200.ops.grouped``);
* ``quantize4``, ``linear4``, ``grouped4``: microscaled 4-bit values (e2m1,
  one power-of-two scale per 32 values of a row) and products of two such
  operands (``tempname_dcu_b200.ops.mx4``).

With ``own`` false ``run`` computes the definitions with elementary torch
operations in 32 bits; with ``own`` true it calls the framework.
"""
import math

import numpy as np
import torch

own = False

DEVICE = "cuda"


def listed():
    return [
        # one token's choice among a few experts: launch latency only
        dict(name="route_one_token", kind="route", tokens=1, experts=8, top_k=2, normalize=True, dtype="float32"),
        # a full micro-batch of tokens over many fine-grained experts, forward and gradient
        dict(name="route_16k_tokens", kind="route", tokens=16384, experts=128, top_k=8, normalize=True,
             dtype="float32"),
        # a short odd batch: rows there and back, narrow model
        dict(name="exchange_odd", kind="exchange", tokens=77, experts=12, top_k=3, hidden=264),
        # a training micro-batch of two 2048-token sequences, two experts per token
        dict(name="exchange_train", kind="exchange", tokens=4096, experts=8, top_k=2, hidden=4096),
        # generating one token: two experts' first projection, weights read once
        dict(name="linear_one_token", kind="linear", rows=2, groups=8, active=2, n=16384, k=4096),
        # many small experts with uneven loads, some without a row, sizes off every tile
        dict(name="linear_gelu_ragged", kind="linear_gelu", rows=777, groups=60, active=41, n=1032, k=520),
        # the first projection of a training micro-batch (2048 tokens, two experts each)
        dict(name="linear_gelu_train", kind="linear_gelu", rows=4096, groups=8, active=8, n=16384, k=4096),
        # its backward: the gradient through the second projection and the GELU
        dict(name="data_grad_train", kind="data_grad", rows=4096, groups=8, active=8, n=4096, k=16384),
        # the experts' weight gradients of two such micro-batches' worth of rows
        dict(name="weight_grad_train", kind="weight_grad", rows=8192, groups=8, active=7, n=4096, k=4096),
        # activations of a feed-forward layer into 4 bits and back
        dict(name="quantize4_ffn", kind="quantize4", rows=4096, k=16384),
        # a feed-forward projection with 4-bit weights and activations, long prompt
        dict(name="linear4_prompt", kind="linear4", rows=4096, n=16384, k=4096),
        # a small batch of generated tokens over 16 experts held in 4 bits
        dict(name="grouped4_small_batch", kind="grouped4", rows=64, groups=16, active=15, n=4096, k=4096),
    ]


def _log(rng, lo, hi, multiple=1):
    """Log-uniform multiple of ``multiple`` in [lo, hi]."""
    value = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(value / multiple)) * multiple))


def draw(rng):
    kind = rng.choice(["route", "route", "exchange", "exchange", "linear", "linear", "linear_gelu", "data_grad",
                       "weight_grad", "quantize4", "linear4", "grouped4", "grouped4"])
    if kind == "route":
        experts = rng.choice([4, 8, 12, 16, 60, 64, 128, 160, 256])
        return dict(kind=kind, tokens=_log(rng, 1, 16384), experts=experts,
                    top_k=rng.randint(1, min(experts, 8)), normalize=rng.random() < 0.7,
                    dtype=rng.choice(["float32", "bfloat16"]))
    if kind == "exchange":
        experts = rng.choice([4, 8, 12, 16, 64, 128])
        top_k = rng.randint(1, min(experts, 6))
        return dict(kind=kind, tokens=_log(rng, 1, 8192 // top_k), experts=experts, top_k=top_k,
                    hidden=_log(rng, 64, 4096, 8))
    if kind == "quantize4":
        return dict(kind=kind, rows=_log(rng, 1, 8192), k=_log(rng, 32, 8192, 32))
    if kind == "linear4":
        return dict(kind=kind, rows=_log(rng, 1, 4096), n=_log(rng, 64, 8192, 8), k=_log(rng, 64, 8192, 32))
    groups = rng.choice([2, 4, 7, 8, 16, 32, 60, 64])
    rows = _log(rng, 1, 8192)
    active = max(1, min(rows, groups) - rng.choice([0, 0, 1, 3]))
    most = 8192 if groups <= 8 else 4096 if groups <= 16 else 2048
    step = 32 if kind == "grouped4" else 8
    return dict(kind=kind, rows=rows, groups=groups, active=active, n=_log(rng, 64, most, 8),
                k=_log(rng, 64, most, step))


# ------------------------------------------------------------------ inputs
def _generator(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(int(seed) * 1000003 + sum(ord(c) for c in case["kind"]))
    return gen


def _normal(gen, shape, std=1.0, dtype=torch.bfloat16):
    out = torch.empty(shape, dtype=dtype, device=DEVICE)
    return out.normal_(0.0, std, generator=gen)


def _bounds(case, seed):
    """Row bounds of the groups: ``active`` groups with at least one row each
    and uneven loads (a few experts take several times the mean)."""
    rng = np.random.default_rng([int(seed), case["rows"], case["groups"]])
    chosen = np.sort(rng.permutation(case["groups"])[:case["active"]])
    share = np.exp(0.7 * rng.standard_normal(case["active"]))
    counts = np.zeros(case["groups"], dtype=np.int64)
    counts[chosen] = 1 + rng.multinomial(case["rows"] - case["active"], share / share.sum())
    return [0] + [int(v) for v in np.cumsum(counts)]


def _chosen(gen, tokens, experts, top_k):
    """Distinct experts per token [tokens, top_k], as a router with a skewed preference picks them."""
    score = _normal(gen, (tokens, experts), 1.0, torch.float32) + _normal(gen, (experts,), 0.5, torch.float32)
    ids = []
    for _ in range(top_k):
        pick = score.max(dim=1).indices
        ids.append(pick)
        score.scatter_(1, pick[:, None], float("-inf"))
    return torch.stack(ids, 1).to(torch.int32)


def _outlying(x, gen):
    """Activations with a few strong columns, as feed-forward inputs have them."""
    strong = 1.0 + 15.0 * (torch.rand(x.shape[-1], device=DEVICE, generator=gen) < 0.01).float()
    return (x.float() * strong).to(torch.bfloat16)


def _inputs(case, seed):
    gen = _generator(case, seed)
    kind = case["kind"]
    s = dict(case=case)
    if kind == "route":
        logits = _normal(gen, (case["tokens"], case["experts"]), 1.5, torch.float32)
        s["logits"] = logits.to(getattr(torch, case["dtype"]))
        s["dweights"] = _normal(gen, (case["tokens"], case["top_k"]), 0.1, torch.float32)
        return s
    if kind == "exchange":
        tokens, top_k, hidden = case["tokens"], case["top_k"], case["hidden"]
        s["ids"] = _chosen(gen, tokens, case["experts"], top_k)
        weights = torch.rand((tokens, top_k), device=DEVICE, generator=gen) + 0.1
        s["weights"] = weights / weights.sum(1, keepdim=True)
        s["x"] = _normal(gen, (tokens, hidden))
        s["ys"] = _normal(gen, (tokens * top_k, hidden))
        s["dout"] = _normal(gen, (tokens, hidden), 0.05)
        s["dxs"] = _normal(gen, (tokens * top_k, hidden), 0.05)
        return s
    if kind == "quantize4":
        s["x"] = _outlying(_normal(gen, (case["rows"], case["k"])), gen)
        return s
    if kind == "linear4":
        s["x"] = _outlying(_normal(gen, (case["rows"], case["k"])), gen)
        s["w"] = _normal(gen, (case["n"], case["k"]), 0.02)
        s["bias"] = _normal(gen, (case["n"],), 0.02)
        return s
    rows, groups, n, k = case["rows"], case["groups"], case["n"], case["k"]
    s["bounds"] = _bounds(case, seed)
    s["offsets"] = torch.tensor(s["bounds"], dtype=torch.int32, device=DEVICE)
    if kind == "grouped4":
        s["x"] = _outlying(_normal(gen, (rows, k)), gen)
        s["w"] = _normal(gen, (groups, n, k), 0.02)
        s["bias"] = _normal(gen, (groups, n), 0.02)
    elif kind in ("linear", "linear_gelu"):
        s["x"] = _normal(gen, (rows, k))
        s["w"] = _normal(gen, (groups, n, k), 0.02)
        s["bias"] = _normal(gen, (groups, n), 0.02)
    elif kind == "data_grad":
        s["dy"] = _normal(gen, (rows, n), 0.05)
        s["w"] = _normal(gen, (groups, n, k), 0.02)
        s["pre"] = _normal(gen, (rows, k))
    else:
        s["dy"] = _normal(gen, (rows, n), 0.05)
        s["x"] = _normal(gen, (rows, k))
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    if kind in ("linear4", "grouped4"):
        # the weights are brought into 4 bits once, when they are loaded
        if own:
            from tempname_dcu_b200.ops import mx4
            s["qw"], s["sfw"] = mx4.quantize(s["w"])
        else:
            s["w4"] = _values4(s["w"])
        del s["w"]
    if kind == "exchange":
        # the routing that the router's call of this step returned
        experts = case["experts"]
        flat = s["ids"].reshape(-1).long()
        offsets, order, slots = _group(flat, experts)
        s["order"], s["slots"], s["offsets"] = order, slots, offsets
        if own:
            from tempname_dcu_b200.ops import moe
            s["routing"] = moe.Routing(ids=s["ids"], weights=s["weights"], offsets=offsets, order=order, slots=slots)
    if kind == "weight_grad":
        # the gradient buffer of the optimizer
        s["grad"] = torch.empty((case["groups"], case["n"], case["k"]), dtype=torch.float32, device=DEVICE)
    return s


# ------------------------------------------------------------------ plain forms
def _group(flat, experts):
    """Stable grouping by expert: (offsets [experts+1], order: slot -> choice, slots: choice -> slot)."""
    hot = (flat[:, None] == torch.arange(experts, device=flat.device)[None, :]).to(torch.int32)
    counts = hot.sum(0)
    offsets = torch.zeros(experts + 1, dtype=torch.int64, device=flat.device)
    offsets[1:] = counts.cumsum(0)
    rank = (hot.cumsum(0) * hot).sum(1) - 1
    slots = offsets[flat] + rank
    order = torch.empty_like(slots)
    order[slots] = torch.arange(flat.numel(), device=flat.device)
    return offsets.to(torch.int32), order.to(torch.int32), slots.to(torch.int32)


def _gelu(z):
    return 0.5 * z * (1.0 + torch.erf(z * (1.0 / math.sqrt(2.0))))


def _gelu_slope(z):
    cdf = 0.5 * (1.0 + torch.erf(z * (1.0 / math.sqrt(2.0))))
    return cdf + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))


def _values4(x):
    """The values that the 4-bit form of x stands for, in 32 bits."""
    blocks = x.float().reshape(*x.shape[:-1], -1, 32)
    top = blocks.abs().amax(-1, keepdim=True)
    mantissa, exponent = torch.frexp(top)  # top = mantissa * 2^exponent, mantissa in [0.5, 1)
    e = exponent - 3 + (mantissa > 0.75).to(exponent.dtype)  # the smallest with top / 2^e <= 6
    e = torch.where(top > 0, e, torch.full_like(e, -127)).clamp(-127, 127).float()
    v = blocks * torch.exp2(-e)
    size = v.abs()
    step = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0))
    v = torch.sign(v) * torch.round(size / step) * step
    return (v * torch.exp2(e)).reshape(x.shape)


def _plain(s):
    case, kind = s["case"], s["case"]["kind"]
    if kind == "route":
        score = s["logits"].float()
        work = score.clone()
        columns = torch.arange(case["experts"], device=score.device)
        ids = []
        for _ in range(case["top_k"]):
            best = work.amax(1, keepdim=True)
            pick = torch.where(work == best, columns, case["experts"]).amin(1)  # ties: the lowest index
            ids.append(pick)
            work.scatter_(1, pick[:, None], float("-inf"))
        ids = torch.stack(ids, 1)
        p = torch.exp(score - score.amax(1, keepdim=True))
        p = p / p.sum(1, keepdim=True)
        chosen = p.gather(1, ids)
        dw = s["dweights"]
        if case["normalize"]:
            weights = chosen / chosen.sum(1, keepdim=True)
            part = weights * (dw - (dw * weights).sum(1, keepdim=True))
            dlogits = torch.zeros_like(score).scatter(1, ids, part)
        else:
            weights = chosen
            full = torch.zeros_like(score).scatter(1, ids, dw)
            dlogits = p * (full - (dw * chosen).sum(1, keepdim=True))
        offsets, order, slots = _group(ids.reshape(-1), case["experts"])
        return [ids.to(torch.int32), weights, offsets, order, slots, dlogits.to(s["logits"].dtype)]
    if kind == "exchange":
        tokens, top_k, hidden = case["tokens"], case["top_k"], case["hidden"]
        token = torch.div(s["order"].long(), top_k, rounding_mode="floor")
        slots = s["slots"].long()
        xs = s["x"][token]
        y = s["ys"].float()[slots].reshape(tokens, top_k, hidden)
        out = (y * s["weights"][:, :, None]).sum(1)
        dout = s["dout"].float()
        dweights = (y * dout[:, None, :]).sum(2)
        dys = dout[token] * s["weights"].reshape(-1)[s["order"].long()][:, None]
        dx = s["dxs"].float()[slots].reshape(tokens, top_k, hidden).sum(1)
        return [xs, out.to(torch.bfloat16), dys.to(torch.bfloat16), dweights, dx.to(torch.bfloat16)]
    if kind == "quantize4":
        return _values4(s["x"]).to(torch.bfloat16)
    if kind == "linear4":
        return (_values4(s["x"]) @ s["w4"].t() + s["bias"].float()).to(torch.bfloat16)
    spans = [(g, a, b) for g, (a, b) in enumerate(zip(s["bounds"], s["bounds"][1:])) if b > a]
    if kind == "grouped4":
        x = _values4(s["x"])
        out = torch.empty((case["rows"], case["n"]), dtype=torch.bfloat16, device=x.device)
        for g, a, b in spans:
            out[a:b] = x[a:b] @ s["w4"][g].t() + s["bias"][g].float()
        return out
    if kind in ("linear", "linear_gelu"):
        x = s["x"].float()
        z = torch.empty((case["rows"], case["n"]), dtype=torch.float32, device=x.device)
        for g, a, b in spans:
            z[a:b] = x[a:b] @ s["w"][g].float().t() + s["bias"][g].float()
        if kind == "linear":
            return z.to(torch.bfloat16)
        return [_gelu(z).to(torch.bfloat16), z.to(torch.bfloat16)]
    if kind == "data_grad":
        dy = s["dy"].float()
        out = torch.empty((case["rows"], case["k"]), dtype=torch.float32, device=dy.device)
        for g, a, b in spans:
            out[a:b] = dy[a:b] @ s["w"][g].float()
        return (out * _gelu_slope(s["pre"].float())).to(torch.bfloat16)
    dy, x, grad = s["dy"].float(), s["x"].float(), s["grad"]
    dbias = torch.zeros((case["groups"], case["n"]), dtype=torch.float32, device=dy.device)
    grad.zero_()
    for g, a, b in spans:
        grad[g] = dy[a:b].t() @ x[a:b]
        dbias[g] = dy[a:b].sum(0)
    return [grad, dbias]


# ------------------------------------------------------------------ the framework's calls
def _own(s):
    case, kind = s["case"], s["case"]["kind"]
    if kind in ("route", "exchange"):
        from tempname_dcu_b200.ops import moe
        if kind == "route":
            r = moe.route(s["logits"], case["top_k"], normalize=case["normalize"])
            dlogits = moe.route_bwd(s["logits"], r, s["dweights"])
            return [r.ids, r.weights, r.offsets, r.order, r.slots, dlogits]
        r = s["routing"]
        xs = moe.dispatch(s["x"], r)
        out = moe.combine(s["ys"], r)
        dys, dweights = moe.combine_bwd(s["dout"], s["ys"], r)
        dx = moe.dispatch_bwd(s["dxs"], r)
        return [xs, out, dys, dweights, dx]
    if kind in ("quantize4", "linear4", "grouped4"):
        from tempname_dcu_b200.ops import mx4
        if kind == "quantize4":
            q, sf = mx4.quantize(s["x"])
            return mx4.dequantize(q, sf)
        if kind == "linear4":
            q, sf = mx4.quantize(s["x"])
            return mx4.linear(q, sf, s["qw"], s["sfw"], bias=s["bias"])
        q, sf = mx4.quantize(s["x"], offsets=s["offsets"])
        return mx4.grouped_linear(q, sf, s["qw"], s["sfw"], s["offsets"], bias=s["bias"])
    from tempname_dcu_b200.ops import grouped
    if kind == "linear":
        return grouped.linear(s["x"], s["w"], s["offsets"], s["bias"])
    if kind == "linear_gelu":
        return list(grouped.linear_gelu(s["x"], s["w"], s["offsets"], s["bias"]))
    if kind == "data_grad":
        return grouped.matmul_nt(s["dy"], s["w"], s["offsets"], gelu_pre=s["pre"])
    grouped.weight_grad(s["dy"], s["x"], s["offsets"], s["grad"], accumulate=False)
    dbias = grouped.bias_grad(s["dy"], s["offsets"])
    return [s["grad"], dbias]


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------ definitions in 64 bits
def _exact4(x):
    """4-bit values from their definition: the nearest point of the grid, ties to the even code."""
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=x.device)
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    flat, dest = x.reshape(-1, 32), out.view(-1, 32)
    for lo in range(0, flat.shape[0], 1 << 19):
        block = flat[lo:lo + (1 << 19)].double()
        top = block.abs().max(1, keepdim=True).values
        e = torch.ceil(torch.log2(top.clamp_min(1e-300) / 6.0))
        e = torch.where(top * torch.exp2(-e) > 6.0, e + 1, e)  # log2 rounded across a power of two
        e = torch.where(top * torch.exp2(1 - e) <= 6.0, e - 1, e)
        scale = torch.exp2(e.clamp(-127, 127))
        size = block.abs() / scale
        code = torch.zeros_like(size, dtype=torch.int64)
        for c in range(1, 8):
            middle = 0.5 * (grid[c - 1] + grid[c])
            code += (size >= middle if c % 2 == 0 else size > middle).long()
        dest[lo:lo + (1 << 19)] = torch.copysign(grid[code] * scale, block)
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    if kind == "route":
        z = s["logits"].double()
        experts, top_k = case["experts"], case["top_k"]
        ids = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :top_k]
        p = torch.softmax(z, 1)
        dw = s["dweights"].double()
        leaf = z.clone().requires_grad_(True)
        prob = torch.softmax(leaf, 1).gather(1, ids)
        weights = prob / prob.sum(1, keepdim=True) if case["normalize"] else prob
        (weights * dw).sum().backward()
        flat = ids.reshape(-1)
        order = torch.sort(flat, stable=True).indices
        slots = torch.empty_like(order)
        slots[order] = torch.arange(order.numel(), device=order.device)
        offsets = torch.zeros(experts + 1, dtype=torch.int64, device=order.device)
        offsets[1:] = torch.bincount(flat, minlength=experts).cumsum(0)
        del p
        return [ids, weights.detach(), offsets, order, slots, leaf.grad]
    if kind == "exchange":
        tokens, top_k, hidden = case["tokens"], case["top_k"], case["hidden"]
        order = torch.sort(s["ids"].reshape(-1), stable=True).indices
        slots = torch.empty_like(order)
        slots[order] = torch.arange(order.numel(), device=order.device)
        token = order // top_k
        w, dout = s["weights"].double(), s["dout"].double()
        ys, dxs = s["ys"].double(), s["dxs"].double()
        out = torch.zeros((tokens, hidden), dtype=torch.float64, device=DEVICE)
        dx = torch.zeros_like(out)
        dweights = torch.empty((tokens, top_k), dtype=torch.float64, device=DEVICE)
        for j in range(top_k):
            row = slots[j::top_k]
            out += w[:, j:j + 1] * ys[row]
            dx += dxs[row]
            dweights[:, j] = (dout * ys[row]).sum(1)
        dys = w.reshape(-1)[order][:, None] * dout[token]
        return [s["x"].double()[token], out, dys, dweights, dx]
    if kind == "quantize4":
        return _exact4(s["x"])
    if kind == "linear4":
        return _exact4(s["x"]) @ _exact4(s["w"]).t() + s["bias"].double()
    groups = range(case["groups"])
    bounds = s["bounds"]
    if kind in ("grouped4", "linear", "linear_gelu"):
        x = _exact4(s["x"]) if kind == "grouped4" else s["x"].double()
        z = torch.zeros((case["rows"], case["n"]), dtype=torch.float64, device=DEVICE)
        for g in groups:
            if bounds[g + 1] > bounds[g]:
                w = _exact4(s["w"][g]) if kind == "grouped4" else s["w"][g].double()
                z[bounds[g]:bounds[g + 1]] = torch.matmul(x[bounds[g]:bounds[g + 1]], w.t()) + s["bias"][g].double()
        if kind == "linear_gelu":
            return [0.5 * z * torch.erfc(-z / math.sqrt(2.0)), z]
        return z
    if kind == "data_grad":
        z = s["pre"].double()
        slope = 0.5 * torch.erfc(-z / math.sqrt(2.0)) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        out = torch.zeros_like(z)
        for g in groups:
            out[bounds[g]:bounds[g + 1]] = torch.matmul(s["dy"][bounds[g]:bounds[g + 1]].double(), s["w"][g].double())
        return out * slope
    grad = torch.zeros((case["groups"], case["n"], case["k"]), dtype=torch.float64, device=DEVICE)
    dbias = torch.zeros((case["groups"], case["n"]), dtype=torch.float64, device=DEVICE)
    for g in groups:
        part = s["dy"][bounds[g]:bounds[g + 1]].double()
        grad[g] = torch.matmul(part.t(), s["x"][bounds[g]:bounds[g + 1]].double())
        dbias[g] = part.sum(0)
    return [grad, dbias]


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    kind = case["kind"]
    if kind == "route":
        t, e, k = case["tokens"], case["experts"], case["top_k"]
        size = 4 if case["dtype"] == "float32" else 2
        # logits, weight gradients in; ids, weights, order, slots, offsets, logit gradients out
        return dict(bytes=2 * t * e * size + t * k * 20 + 4 * (e + 1), flops=t * e * 10)
    if kind == "exchange":
        t, k, h = case["tokens"], case["top_k"], case["hidden"]
        # x, ys, dout, dxs in; xs, out, dys, dx out; weights and their gradient, order and slots
        return dict(bytes=2 * h * (4 * t + 4 * t * k) + t * k * 16, flops=t * k * h * 6)
    if kind == "quantize4":
        # bf16 in, the values out (the packed form in between is written as well)
        n = case["rows"] * case["k"]
        return dict(bytes=2 * n + 2 * n + n // 2 + n // 32, flops=4 * n)
    if kind == "linear4":
        m, n, k = case["rows"], case["n"], case["k"]
        return dict(bytes=2 * m * k + n * k // 2 + n * k // 32 + 2 * n + 2 * m * n, flops=2 * m * n * k)
    rows, n, k, active = case["rows"], case["n"], case["k"], case["active"]
    flops = 2 * rows * n * k
    if kind == "grouped4":
        return dict(bytes=2 * rows * k + active * (n * k // 2 + n * k // 32 + 2 * n) + 2 * rows * n, flops=flops)
    if kind == "linear":
        return dict(bytes=2 * rows * k + active * (2 * n * k + 2 * n) + 2 * rows * n, flops=flops)
    if kind == "linear_gelu":
        return dict(bytes=2 * rows * k + active * (2 * n * k + 2 * n) + 4 * rows * n, flops=flops)
    if kind == "data_grad":
        return dict(bytes=2 * rows * n + active * 2 * n * k + 4 * rows * k, flops=flops)
    return dict(bytes=2 * rows * (n + k) + 4 * case["groups"] * n * (k + 1), flops=flops + rows * n)
