"""Cases for measuring the group-norm and AdamW operators.

Each case is one pass through one operator: a group norm over channels-last
activations (with its activation and residual, forward only or with its
backward pass), or one AdamW step over every tensor of a model (moments held
in 32 or in 8 bits). With ``own`` false a pass is computed in elementary torch
operations, with ``own`` true by the framework.
"""

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ALIGN = 64       # floats: every tensor of the flat space starts at a multiple
QBLOCK = 64      # values that share one exponent in the 8-bit moments


# --------------------------------------------------------------------------
# the cases
# --------------------------------------------------------------------------

def _gn(n, h, w, c, groups, act, residual, dtype, train):
    return {"op": "group_norm", "n": n, "h": h, "w": w, "c": c,
            "groups": groups, "act": act, "residual": residual,
            "dtype": dtype, "train": train}


def _adamw(model, count, smallest, largest, bits, beta2, decay_1d):
    return {"op": "adamw", "model": model, "count": count,
            "smallest": smallest, "largest": largest, "bits": bits,
            "beta2": beta2, "decay_1d": decay_1d}


def listed():
    return [
        # one image through the last stage of a ResNet: the smallest call of
        # an evaluation, where the launches are all of it
        {"name": "gn_fwd_one_image", **_gn(1, 4, 4, 512, 8, "relu", False, "bf16", False)},
        # the evaluation batch at a block's tail: norm, residual, ReLU
        {"name": "gn_fwd_eval_tail", **_gn(100, 32, 32, 64, 8, "relu", True, "bf16", False)},
        # one large map: few groups, each a long reduction
        {"name": "gn_fwd_one_map", **_gn(1, 512, 512, 128, 32, "silu", False, "bf16", False)},
        # ResNet-20's first stage at a small batch: launch-bound training
        {"name": "gn_train_narrow", **_gn(64, 32, 32, 16, 8, "relu", False, "bf16", True)},
        # the flagship's first stage at batch 256, block tail: the largest
        # activations of its training step
        {"name": "gn_train_stage1_tail", **_gn(256, 32, 32, 64, 8, "relu", True, "bf16", True)},
        # its last stage: many channels, 16 pixels
        {"name": "gn_train_stage4", **_gn(256, 4, 4, 512, 8, "relu", False, "bf16", True)},
        # wide maps, few samples, ten channels to a group
        {"name": "gn_train_wide_silu", **_gn(4, 128, 128, 320, 32, "silu", False, "bf16", True)},
        # odd everything, in 32 bits
        {"name": "gn_train_odd_fp32", **_gn(37, 15, 15, 30, 3, "silu", True, "fp32", True)},
        # the MNIST CNN: 8 tensors, 27,480 parameters, nothing but latency
        {"name": "adamw32_cnn2", **_adamw("cnn2", 0, 0, 0, 32, 0.999, True)},
        # the flagship: 86 tensors, 17.4 M parameters
        {"name": "adamw32_resnet18q", **_adamw("resnet18q", 0, 0, 0, 32, 0.999, True)},
        {"name": "adamw8_resnet18q", **_adamw("resnet18q", 0, 0, 0, 8, 0.999, False)},
        # the largest model of the zoo: 467 tensors, 58 M parameters
        {"name": "adamw8_resnet152", **_adamw("resnet152", 0, 0, 0, 8, 0.999, True)},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    if rng.random() < 0.6:
        groups = rng.choice([1, 2, 3, 4, 8, 16, 32])
        cpg = _log_int(rng, 1, 64)
        while groups * cpg > 2048:
            cpg = _log_int(rng, 1, 64)
        c = groups * cpg
        most = 16_000_000
        h, w = _log_int(rng, 1, 256), _log_int(rng, 1, 256)
        while h * w * c > most:
            h, w = max(1, h // 2), max(1, w // 2)
        while h * w * cpg < 16:  # fewer values have next to no statistics
            h, w = 2 * h, 2 * w
        n = _log_int(rng, 1, min(512, max(1, most // (h * w * c))))
        act = rng.choice(["none", "relu", "relu", "silu"])
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        if dtype == "fp32":  # the same bytes
            n = max(1, n // 2)
        return _gn(n, h, w, c, groups, act, rng.random() < 0.4, dtype, rng.random() < 0.7)
    largest = _log_int(rng, 64, 3_000_000)
    smallest = _log_int(rng, 1, min(largest, 2000))
    count = _log_int(rng, 1, max(1, min(400, 40_000_000 // largest)))
    return _adamw("", count, smallest, largest, rng.choice([8, 32]),
                  rng.choice([0.95, 0.99, 0.999]), rng.random() < 0.5)


# --------------------------------------------------------------------------
# what a model's parameters look like
# --------------------------------------------------------------------------

def _resnet(blocks, extra, bottleneck):
    """Shapes of a CIFAR ResNet's tensors, in order; `extra`: blocks beyond
    the count in each stage."""
    conv = lambda o, i, k: [(o, i, k, k), (o,), (o,)]  # noqa: E731
    shapes, ch = conv(64, 3, 3), 64
    for stage, count in enumerate(blocks):
        mid = 64 << stage
        out = 4 * mid if bottleneck else mid
        for b in range(count + extra):
            if bottleneck:
                shapes += conv(mid, ch, 1) + conv(mid, mid, 3) + conv(out, mid, 1)
            else:
                shapes += conv(mid, ch, 3) + conv(mid, mid, 3)
            if b == 0 and (stage or ch != out):
                shapes += conv(out, ch, 1)
            ch = out
    return shapes + [(10, ch), (10,)]


def _shapes(case):
    if case["model"] == "cnn2":
        return [(10, 1, 3, 3), (10,), (20, 10, 3, 3), (20,), (50, 500), (50,), (10, 50), (10,)]
    if case["model"] == "resnet18q":
        return _resnet((2, 2, 2, 2), 1, False)
    if case["model"] == "resnet152":
        return _resnet((3, 8, 36, 3), 0, True)
    # `count` tensors, their sizes spread geometrically; every other one flat,
    # as a bias or a norm's weight is
    low, high, k = case["smallest"], case["largest"], case["count"]
    sizes = [max(1, int(high * (low / high) ** (i / max(1, k - 1)))) for i in range(k)]
    return [(s,) if i % 2 else (s, 1) for i, s in enumerate(sizes)]


def _starts(shapes):
    at, starts = 0, []
    for s in shapes:
        starts.append(at)
        at += -(-math.prod(s) // ALIGN) * ALIGN
    return starts, at


HYPER = {"lr": 1e-3, "beta1": 0.9, "eps": 1e-8, "decay": 0.05, "seed": 17}


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------

def _inputs_gn(case, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    n, h, w, c = case["n"], case["h"], case["w"], case["c"]
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    dt = DTYPES[case["dtype"]]
    # a convolution's output: channels of their own mean and spread
    x = (rnd(n, h, w, c) * torch.exp(0.5 * rnd(c)) + 0.5 * rnd(c)).to(dt)
    gamma, beta = 1 + 0.2 * rnd(c), 0.2 * rnd(c)
    # what comes down the skip connection is a ReLU's output
    res = rnd(n, h, w, c).clamp_min(0).to(dt) if case["residual"] else None
    dy = rnd(n, h, w, c).to(dt) if case["train"] else None
    return x, gamma, beta, res, dy


def _inputs_adamw(case, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    shapes = _shapes(case)
    starts, total = _starts(shapes)
    sizes = [math.prod(s) for s in shapes]
    numels = torch.tensor(sizes, device=DEV)
    seg = torch.repeat_interleave(torch.arange(len(shapes), device=DEV),
                                  torch.tensor([e - s for s, e in zip(starts, starts[1:] + [total])], device=DEV))
    inside = torch.arange(total, device=DEV) - torch.tensor(starts, device=DEV)[seg] < numels[seg]
    # gradients of very different size from tensor to tensor, some of them
    # zero as behind a dead ReLU
    size = 10 ** (-4 + 3 * torch.rand(len(shapes), generator=g, device=DEV))
    grad = torch.randn(total, generator=g, device=DEV) * size[seg]
    grad *= inside & (torch.rand(total, generator=g, device=DEV) > 0.03)
    param = 0.05 * torch.randn(total, generator=g, device=DEV) * inside
    flat = torch.tensor([len(s) < 2 for s in shapes], device=DEV)
    decays = inside & (~flat[seg] | case["decay_1d"])
    ends = torch.tensor(starts, device=DEV) + numels
    return shapes, param, grad, decays, torch.tensor(starts, device=DEV), ends


def prepare(case, seed):
    if case["op"] == "group_norm":
        x, gamma, beta, res, dy = _inputs_gn(case, seed)
        if own and case["train"]:
            for t in (x, gamma, beta, res):
                if t is not None:
                    t.requires_grad_(True)
        return {"case": case, "x": x, "gamma": gamma, "beta": beta, "res": res, "dy": dy}
    shapes, param, grad, decays, starts, ends = _inputs_adamw(case, seed)
    if own:
        from eventgrad_amd.parallel import AdamW, FlatParamSpace
        model = torch.nn.ParameterList([torch.nn.Parameter(torch.empty(s, device=DEV)) for s in shapes])
        space = FlatParamSpace(model, torch.device(DEV, torch.cuda.current_device()))
        space.load_flat(param)
        space.grad.copy_(grad)
        opt = AdamW(space, lr=HYPER["lr"], betas=(HYPER["beta1"], case["beta2"]), eps=HYPER["eps"],
                    weight_decay=HYPER["decay"], decay_1d=case["decay_1d"], state_bits=case["bits"],
                    seed=HYPER["seed"])
        return {"case": case, "opt": opt, "space": space, "model": model}
    moments = torch.float32 if case["bits"] == 32 else torch.bfloat16
    return {"case": case, "param": param, "grad": grad, "decays": decays, "starts": starts, "ends": ends,
            "m": torch.zeros_like(param, dtype=moments), "v": torch.zeros_like(param, dtype=moments), "t": 0}


# --------------------------------------------------------------------------
# the plain forms
# --------------------------------------------------------------------------

def _plain_gn(s):
    case, x, gamma, beta, res, dy = (s[k] for k in ("case", "x", "gamma", "beta", "res", "dy"))
    n, h, w, c = x.shape
    groups = case["groups"]
    m = h * w * (c // groups)
    # the sums are long, and the sign of z decides a ReLU's gradient: 64 bits
    # up to z
    x5 = x.double().view(n, h * w, groups, c // groups)
    mean = x5.sum((1, 3), keepdim=True) / m
    off = x5 - mean
    rstd = ((off * off).sum((1, 3), keepdim=True) / m + 1e-5).rsqrt()
    xhat = (off * rstd).view(n, h, w, c)
    z = xhat * gamma.double() + beta.double()
    if res is not None:
        z = z + res.double()
    if case["act"] == "relu":
        gate = (z > 0).float()
        y = z.float() * gate
    elif case["act"] == "silu":
        z = z.float()
        sig = 1 / (1 + torch.exp(-z))
        y = z * sig
        gate = sig * (1 + z * (1 - sig))
    else:
        y, gate = z.float(), 1.0
    out = {"y": y.to(x.dtype)}
    if dy is None:
        return out
    xhat = xhat.float()
    dz = dy.float() * gate
    out["dgamma"] = (dz * xhat).sum((0, 1, 2))
    out["dbeta"] = dz.sum((0, 1, 2))
    if res is not None:
        out["dres"] = dz.to(x.dtype)
    d5 = (dz * gamma).view(n, h * w, groups, -1)
    h5 = xhat.view(n, h * w, groups, -1)
    s1 = d5.sum((1, 3), keepdim=True) / m
    s2 = (d5 * h5).sum((1, 3), keepdim=True) / m
    out["dx"] = (rstd.float() * (d5 - s1 - h5 * s2)).view(n, h, w, c).to(x.dtype)
    return out


def _mix(seed, index):
    """32 bits from a seed and an index, both below 2**32, in 64-bit integers."""
    low = 0xFFFFFFFF
    h = seed ^ (index * 0x9E3779B9 & low)
    h = (h ^ 61) ^ (h >> 16)
    h = h * 9 & low
    h = h ^ (h >> 4)
    h = h * 0x27D4EB2D & low
    return h ^ (h >> 15)


def _to_8_bits(x, random, exponent_bits, least):
    """x rounded to 8 bits a value: blocks of 64 share one power of two, and
    each value has `exponent_bits` more and 3 bits behind its leading one. It
    goes up with the probability of what lies below it; `random`: 16 bits a
    value. `least`: a value above zero stays above zero. Exact in 64 bits."""
    b = x.view(-1, QBLOCK)
    top = b.abs().amax(1, keepdim=True)
    # the power of two that leaves the largest value below 2 once rounded up
    floor = 2 + 2 ** exponent_bits
    shared = ((top.view(torch.int32) + 0xFFFFF) >> 23).clamp(floor, 254)
    y = b.abs().double() * torch.exp2((127 - shared).double())
    field = torch.floor(torch.log2(y.clamp_min(1e-300)))
    field = field - (torch.exp2(field) > y).double()      # log2 next to a power of two
    field = field + (torch.exp2(field + 1) <= y).double()
    step = torch.exp2(field.clamp_min(2 - 2 ** exponent_bits) - 3)
    q = torch.floor(y / step + random.view(-1, QBLOCK).double() / 65536)
    if least:
        q = torch.where(y > 0, q.clamp_min(1), q)
    y = (q * step).clamp_max(1.875)
    back = torch.where(b < 0, -y, y) * torch.exp2((shared - 127).double())
    back = torch.where(torch.isfinite(b).all(1, keepdim=True), back, math.nan)
    return back.to(torch.bfloat16).view(-1)


def _plain_adamw(s):
    case, p, g = s["case"], s["param"], s["grad"]
    lr, b1, b2, eps, decay = HYPER["lr"], HYPER["beta1"], case["beta2"], HYPER["eps"], HYPER["decay"]
    s["t"] += 1
    t = s["t"]
    m = s["m"].float() * b1 + g * (1 - b1)
    v = s["v"].float() * b2 + (g * g) * (1 - b2)
    p = torch.where(s["decays"], p * (1 - lr * decay), p)
    p = p - lr / (1 - b1 ** t) * m / (v.sqrt() / math.sqrt(1 - b2 ** t) + eps)
    if case["bits"] == 8:
        at = torch.arange(p.numel(), device=p.device)
        random = _mix(_mix(HYPER["seed"], t) + (at >> 32) & 0xFFFFFFFF, at & 0xFFFFFFFF)
        m = _to_8_bits(m, random & 0xFFFF, 4, False)
        v = _to_8_bits(v, random >> 16, 5, True)
    s["param"], s["m"], s["v"] = p, m, v
    sums = torch.nn.functional.pad((p.double() ** 2).cumsum(0), (1, 0))
    return {"param": p, "exp_avg": m, "exp_avg_sq": v, "sqnorms": (sums[s["ends"]] - sums[s["starts"]]).float()}


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------

def run(state):
    case = state["case"]
    if case["op"] == "adamw":
        if not own:
            return _plain_adamw(state)
        norms = state["opt"].step()
        m, v = state["opt"].moments()
        return {"param": state["space"].param, "exp_avg": m, "exp_avg_sq": v, "sqnorms": norms}
    if not own:
        return _plain_gn(state)
    from eventgrad_amd.ops import functional as O
    x, gamma, beta, res = (state[k] for k in ("x", "gamma", "beta", "res"))
    y = O.group_norm(x, gamma, beta, case["groups"], eps=1e-5, activation=case["act"], residual=res)
    if not case["train"]:
        return {"y": y}
    wrt = [x, gamma, beta] + ([res] if res is not None else [])
    d = torch.autograd.grad(y, wrt, state["dy"])
    out = {"y": y, "dx": d[0], "dgamma": d[1], "dbeta": d[2]}
    if res is not None:
        out["dres"] = d[3]
    return out


def work(case):
    if case["op"] == "group_norm":
        n = case["n"] * case["h"] * case["w"] * case["c"]
        size = 4 if case["dtype"] == "fp32" else 2
        # in: x, the residual, dy; out: y, dx, the residual's gradient
        tensors = 2 + case["residual"] + (2 + case["residual"] if case["train"] else 0)
        vectors = 2 * 4 * case["c"] * (2 if case["train"] else 1)
        return {"bytes": n * size * tensors + vectors, "flops": n * (30 if case["train"] else 10)}
    n = sum(math.prod(s) for s in _shapes(case))
    if case["bits"] == 32:  # param, grad, both moments in; param, both moments out
        return {"bytes": 28 * n, "flops": 16 * n}
    # param, grad, 2 codes in; param, 2 codes out; an exponent to 64 codes, in
    # and out; the values that the new codes stand for, 2 bytes each
    return {"bytes": 16 * n + 4 * n // QBLOCK + 4 * n, "flops": 60 * n}


# --------------------------------------------------------------------------
# in 64 bits
# --------------------------------------------------------------------------

def exact(case, seed):
    if case["op"] == "group_norm":
        # the gradients come from autograd
        x, gamma, beta, res, dy = (None if t is None else t.double() for t in _inputs_gn(case, seed))
        leaves = [x, gamma, beta] + ([res] if res is not None else [])
        for t in leaves:
            t.requires_grad_(case["train"])
        by_group = x.permute(0, 3, 1, 2).reshape(x.shape[0], case["groups"], -1)
        var, mean = torch.var_mean(by_group, dim=2, correction=0, keepdim=True)
        xhat = ((by_group - mean) / torch.sqrt(var + 1e-5)).view(x.shape[0], case["c"], case["h"], case["w"])
        z = xhat.permute(0, 2, 3, 1) * gamma + beta
        z = z if res is None else z + res
        y = {"none": lambda t: t, "relu": torch.relu, "silu": lambda t: t * torch.sigmoid(t)}[case["act"]](z)
        if not case["train"]:
            return {"y": y}
        d = torch.autograd.grad(y, leaves, dy)
        out = {"y": y, "dx": d[0], "dgamma": d[1], "dbeta": d[2]}
        return out if res is None else {**out, "dres": d[3]}
    shapes, param, grad, decays, starts, ends = _inputs_adamw(case, seed)
    p, g, b1, b2 = param.double(), grad.double(), HYPER["beta1"], case["beta2"]
    m, v = (1 - b1) * g, (1 - b2) * g.square()
    p = p - HYPER["lr"] * HYPER["decay"] * p * decays
    p = p - HYPER["lr"] * (m / (1 - b1)) / (torch.sqrt(v / (1 - b2)) + HYPER["eps"])
    norms = torch.stack([p[a:b].square().sum() for a, b in zip(starts.tolist(), ends.tolist())])
    # which of two neighbouring codes a value took is not the definition's
    whole = case["bits"] == 32
    return {"param": p, "exp_avg": m if whole else None, "exp_avg_sq": v if whole else None, "sqnorms": norms}
