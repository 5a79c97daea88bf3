"""Group norm with its activation and residual, against plain 64-bit math.

Tolerances. A value is rounded to its type once, off by at most half a step
(eps / 2 of itself). Before that it is computed in fp32, each operation off by
at most 2^-24 of its own size; the sums behind a group's statistics are added
in runs of a few dozen and then in pairs, and exp adds a few steps more. FP32
allows 128 such roundings of the terms' absolute sum, worst case on worst case.
"""

import pytest
import torch

from eventgrad_amd.models import GroupNorm2d, build_model
from eventgrad_amd.ops import functional as O

FP32 = 2.0 ** -17
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16,
         "fp32": torch.float32}


def inputs(n, h, w, c, dtype="fp32", residual=False, mean=0.0, seed=0):
    """NHWC x, gamma, beta, residual, dy on the CPU."""
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    dt = TYPES[dtype]
    x = (rnd(n, h, w, c) * torch.exp(0.5 * rnd(c)) + rnd(c) + mean).to(dt)
    res = rnd(n, h, w, c).to(dt) if residual else None
    return x, 1 + 0.5 * rnd(c), 0.5 * rnd(c), res, rnd(n, h, w, c).to(dt)


def oracle(x, gamma, beta, res, dy, groups, act, eps=1e-5):
    """Values in 64 bits, from the formulas; and for each, the absolute sum of
    the terms that make it."""
    n, h, w, c = x.shape
    cpg = c // groups
    m = h * w * cpg
    x, gamma, beta, dy = (t.double() for t in (x, gamma, beta, dy))
    r = torch.zeros_like(x) if res is None else res.double()
    split = lambda t: t.reshape(n, h * w, groups, cpg)  # noqa: E731
    back = lambda t: t.expand(n, h * w, groups, cpg).reshape(n, h, w, c)  # noqa: E731
    total = lambda t: back(split(t).sum((1, 3), keepdim=True) / m)  # noqa: E731
    mean = total(x)
    rstd = 1 / torch.sqrt(total((x - mean) ** 2) + eps)
    xh = (x - mean) * rstd
    z = gamma * xh + beta + r
    if act == "relu":
        y, slope = z.clamp_min(0), (z > 0).double()
    elif act == "silu":
        s = 1 / (1 + torch.exp(-z))
        y, slope = z * s, s * (1 + z * (1 - s))
    else:
        y, slope = z, torch.ones_like(z)
    dz = dy * slope
    d = gamma * dz
    dx = rstd * (d - total(d) - xh * total(d * xh))
    size_xh = rstd * (x.abs() + mean.abs())
    size_z = (gamma.abs() * size_xh + beta.abs() + r.abs()) * \
        (1 if act != "silu" else 2) + 1e-3
    # a smooth slope moves with z
    size_dz = dy.abs() * (1 + (size_z if act == "silu" else 0))
    size_d = gamma.abs() * size_dz
    size_dx = rstd * (size_d + total(size_d) + size_xh * total(d.abs()) +
                      xh.abs() * total(size_d * (xh.abs() + size_xh)))
    vals = {"y": y, "dx": dx, "dres": dz,
            "dgamma": (dz * xh).sum((0, 1, 2)), "dbeta": dz.sum((0, 1, 2))}
    sizes = {"y": size_z, "dx": size_dx, "dres": size_dz,
             "dgamma": (size_dz * xh.abs() + dz.abs() * size_xh).sum((0, 1, 2)),
             "dbeta": size_dz.sum((0, 1, 2))}
    return vals, sizes


def close(name, got, vals, sizes):
    got64, want = got.detach().cpu().double(), vals[name]
    tol = torch.finfo(got.dtype).eps / 2 * want.abs() + FP32 * sizes[name]
    if got.dtype == torch.float16:
        tol = tol + 2.0 ** -25     # half a step of its subnormals
    off = (got64 - want).abs()
    assert got64.shape == want.shape
    assert bool((off <= tol).all()), \
        (name, float((off / tol.clamp_min(1e-300)).max()))


def run_gpu(x, gamma, beta, res, dy, groups, act, eps=1e-5):
    x, gamma, beta = (t.to(DEV).requires_grad_(True)
                      for t in (x, gamma, beta))
    res = None if res is None else res.to(DEV).requires_grad_(True)
    y = O.group_norm(x, gamma, beta, groups, eps, act, res)
    y.backward(dy.to(DEV))
    out = {"y": y, "dx": x.grad, "dgamma": gamma.grad, "dbeta": beta.grad}
    if res is not None:
        out["dres"] = res.grad
    return out


# ---------------------------------------------------------------- on the CPU

@pytest.mark.parametrize("act", ["none", "relu", "silu"])
@pytest.mark.parametrize("shape,groups,residual", [
    ((3, 5, 7, 12), 3, False), ((2, 4, 4, 16), 8, True),
    ((2, 1, 1, 16), 1, True), ((5, 3, 2, 30), 30, False)])
def test_cpu_matches_formulas(shape, groups, residual, act):
    x, gamma, beta, res, dy = inputs(*shape, residual=residual)
    vals, sizes = oracle(x, gamma, beta, res, dy, groups, act)
    nchw = lambda t: t.permute(0, 3, 1, 2).contiguous()  # noqa: E731
    a = nchw(x).requires_grad_(True)
    r = nchw(res).requires_grad_(True) if residual else None
    gamma.requires_grad_(True)
    beta.requires_grad_(True)
    y = O.group_norm(a, gamma, beta, groups, 1e-5, act, r)
    y.backward(nchw(dy))
    nhwc = lambda t: t.permute(0, 2, 3, 1)  # noqa: E731
    close("y", nhwc(y), vals, sizes)
    close("dx", nhwc(a.grad), vals, sizes)
    close("dgamma", gamma.grad, vals, sizes)
    close("dbeta", beta.grad, vals, sizes)
    if residual:
        close("dres", nhwc(r.grad), vals, sizes)


@pytest.mark.parametrize("act", ["none", "silu"])
def test_oracle_gradients_match_differences(act):
    """The oracle's own formulas against differences of its values. In 64
    bits with a step of 1e-5 the difference is off by its second-order term,
    about 1e-10 of the third derivative, and by 1e-16 / 1e-5 of the loss."""
    x, gamma, beta, res, dy = (t if t is None else t.double() for t in
                               inputs(2, 3, 4, 6, residual=True))
    vals, _ = oracle(x, gamma, beta, res, dy, 3, act)
    g = torch.Generator().manual_seed(9)
    for name, at in (("dx", 0), ("dgamma", 1), ("dbeta", 2), ("dres", 3)):
        args = [x, gamma, beta, res]
        way = torch.randn(args[at].shape, generator=g, dtype=torch.float64)
        loss = []
        for h in (1e-5, -1e-5):
            moved = list(args)
            moved[at] = args[at] + h * way
            loss.append((oracle(*moved, dy, 3, act)[0]["y"] * dy).sum())
        diff = float(loss[0] - loss[1]) / 2e-5
        want = float((vals[name] * way).sum())
        assert abs(diff - want) <= 1e-7 * (1 + abs(want)), name


@pytest.mark.parametrize("call", [
    lambda x, v: O.group_norm(x, v, v, 3),                       # 8 / 3
    lambda x, v: O.group_norm(x, v, v, 0),
    lambda x, v: O.group_norm(x, v, v, 2.0),
    lambda x, v: O.group_norm(x, v, v, 2, eps=-1.0),
    lambda x, v: O.group_norm(x, v, v, 2, activation="gelu"),
    lambda x, v: O.group_norm(x[0], v, v, 2),
    lambda x, v: O.group_norm(x, v, v, 2, residual=x[:1]),
])
def test_refusals(call):
    with pytest.raises(ValueError):
        call(torch.randn(2, 8, 3, 3), torch.ones(8))


def test_module_and_models():
    with pytest.raises(ValueError):
        GroupNorm2d(12, 8)
    with pytest.raises(ValueError):
        build_model("resnet20", norm="layer")
    with pytest.raises(ValueError):
        build_model("cnn2", norm="group")
    with pytest.raises(ValueError):
        build_model("resnet20", norm="group", norm_groups=32)  # 16 channels
    batch, group = build_model("resnet18q"), build_model("resnet18q",
                                                         norm="group")
    # the same tensors under the same names, and nothing beside them
    assert [(k, p.shape) for k, p in batch.named_parameters()] == \
        [(k, p.shape) for k, p in group.named_parameters()]
    assert not list(group.named_buffers())


@pytest.mark.parametrize("name", ["resnet20", "resnet50"])
def test_model_cpu(name):
    torch.manual_seed(0)
    model = build_model(name, norm="group")
    x = torch.randn(2, 3, 32, 32)
    out = model(x)
    out.square().sum().backward()
    assert all(torch.isfinite(p.grad).all() for p in model.parameters())
    # a sample's output does not depend on the batch around it
    alone = model(x[:1])
    assert torch.allclose(alone, out[:1], atol=1e-4)


# ---------------------------------------------------------------- on the GPU

GPU_CASES = [
    # n, h, w, c, groups, act, residual, dtype
    (2, 4, 4, 64, 8, "relu", False, "bf16"),
    (3, 32, 32, 64, 8, "relu", True, "bf16"),      # a block's tail
    (2, 16, 16, 64, 32, "silu", False, "bf16"),    # 2 channels a group
    (5, 8, 8, 40, 4, "silu", True, "bf16"),        # 10: across vectors
    (300, 4, 4, 32, 4, "relu", False, "bf16"),     # many samples
    (1, 1, 1, 64, 1, "relu", True, "bf16"),        # one row
    (1, 1, 1, 16, 1, "none", False, "fp32"),
    (2, 1, 37, 512, 8, "none", True, "bf16"),
    (7, 3, 5, 30, 3, "silu", True, "fp32"),        # 4 does not divide 30
    (7, 3, 5, 30, 3, "relu", True, "bf16"),
    (2, 9, 7, 21, 7, "relu", False, "fp16"),       # odd channels
    (2, 5, 5, 20, 4, "silu", False, "fp16"),
    (2, 3, 3, 2047, 1, "relu", True, "bf16"),      # tiles of columns
    (2, 3, 3, 2048, 32, "silu", False, "fp32"),
    (1, 97, 101, 16, 2, "relu", False, "bf16"),    # one long map
    (1, 200, 200, 8, 1, "silu", True, "fp32"),
    (33, 6, 6, 128, 128, "relu", False, "bf16"),   # a channel a group
    (2, 64, 64, 320, 32, "silu", False, "bf16"),
    (130, 15, 15, 24, 3, "relu", True, "fp32"),
    (2, 129, 65, 48, 3, "none", True, "fp16"),
    (1, 40, 40, 1024, 8, "relu", True, "bf16"),
    (700, 1, 1, 256, 8, "silu", False, "bf16"),    # rows of tokens
    (20, 11, 13, 64, 4, "relu", True, "bf16"),
    (1, 1365, 1, 24, 1, "relu", False, "bf16"),    # rows just past a split
    (1, 70, 70, 4104, 8, "relu", True, "bf16"),    # groups of 513 channels
    (2, 7, 5, 8208, 2, "silu", True, "bf16"),      # of 4,104: slices of one
    (1, 33, 31, 5000, 1, "none", True, "fp16"),
    (1, 120, 120, 6, 3, "silu", True, "bf16"),
    (1, 300, 301, 10, 5, "relu", True, "fp32"),
    (3, 128, 128, 30, 2, "silu", False, "bf16"),
    (1, 9000, 1, 8, 8, "relu", False, "fp16"),     # a channel a group, long
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", GPU_CASES, ids=str)
def test_gpu_matches_formulas(case):
    n, h, w, c, groups, act, residual, dtype = case
    data = inputs(n, h, w, c, dtype, residual)
    vals, sizes = oracle(*data, groups, act)
    got = run_gpu(*data, groups, act)
    torch.cuda.synchronize()
    for name, t in got.items():
        assert t.dtype == (torch.float32 if name in ("dgamma", "dbeta")
                           else TYPES[dtype])
        close(name, t, vals, sizes)
    # without a gradient: the same values
    with torch.no_grad():
        x, gamma, beta, res, _ = (None if t is None else t.to(DEV)
                                  for t in data)
        y = O.group_norm(x, gamma, beta, groups, 1e-5, act, res)
    assert torch.equal(y, got["y"])


@pytest.mark.gpu
@pytest.mark.parametrize("shape,groups", [((2, 32, 32, 64), 8),
                                          ((1, 150, 150, 16), 2)])
def test_gpu_large_mean(shape, groups):
    """A mean of a thousand spreads. The mean itself is rounded to 24 bits,
    2^-25 of 1000 with the value's own distance from it exact: that is 3e-5
    of a spread; the tolerance is eight of them, and not the thousands of
    that a variance taken as E[x^2] - mean^2 would be off by."""
    x, _, _, _, dy = inputs(*shape, mean=0.0)
    x = (x / x.std() + 1000.0)
    one, zero = torch.ones(shape[3]), torch.zeros(shape[3])
    vals, _ = oracle(x, one, zero, None, dy, groups, "none")
    got = run_gpu(x, one, zero, None, dy, groups, "none")
    off = (got["y"].detach().cpu().double() - vals["y"]).abs()
    assert float(off.max()) <= 8 * 1000 * 2.0 ** -25 * (1 + float(
        vals["y"].abs().max()))


@pytest.mark.gpu
def test_gpu_same_every_time_and_leaves_inputs():
    data = inputs(64, 16, 16, 64, "bf16", True)
    first = run_gpu(*data, 8, "relu")
    for _ in range(3):
        again = run_gpu(*data, 8, "relu")
        for k in first:
            assert torch.equal(first[k], again[k]), k


@pytest.mark.gpu
def test_gpu_nonfinite_stays_in_its_group():
    x, gamma, beta, _, dy = inputs(3, 8, 8, 32, "bf16")
    clean = run_gpu(x, gamma, beta, None, dy, 4, "relu")["y"]
    for bad in (float("nan"), float("inf")):
        x2 = x.clone()
        x2[1, 3, 4, 9] = bad                       # sample 1, group 1
        y = run_gpu(x2, gamma, beta, None, dy, 4, "relu")["y"]
        assert torch.isnan(y[1, :, :, 8:16]).all()
        y, want = y.clone(), clean.clone()
        y[1, :, :, 8:16] = 0
        want[1, :, :, 8:16] = 0
        assert torch.equal(y, want)


@pytest.mark.gpu
def test_gpu_constant_groups():
    """No spread: xh is 0, and eps alone keeps rstd finite."""
    x = torch.full((2, 4, 4, 16), 3.0).bfloat16()
    gamma, beta = torch.ones(16), torch.linspace(-1, 1, 16)
    dy = torch.randn(2, 4, 4, 16,
                     generator=torch.Generator().manual_seed(0)).bfloat16()
    got = run_gpu(x, gamma, beta, None, dy, 4, "none")
    assert torch.equal(got["y"].float().cpu(),
                       beta.bfloat16().float().expand(2, 4, 4, 16))
    assert torch.isfinite(got["dx"]).all()
    assert torch.equal(got["dgamma"].cpu(), torch.zeros(16))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("shape,groups", [((2, 16, 16, 64), 8),
                                          ((1, 150, 150, 16), 2)])
def test_gpu_relu_gate_next_to_zero(shape, groups, dtype):
    """The residual is chosen as minus what the norm gives, rounded: many z
    are next to zero, where fp32 does not tell their sign. The gate is the
    sign in 64 bits, but for those within 2e-8 of the terms: the mean adds
    fp32 runs, each off by 2^-24 of itself, hundreds of them independent."""
    x, gamma, beta, _, dy = inputs(*shape, dtype)
    vals, _ = oracle(x, gamma, beta, None, dy, groups, "none")
    res = (-vals["y"]).to(TYPES[dtype])
    g = torch.Generator().manual_seed(1)
    wide = torch.randn(shape, generator=g).to(TYPES[dtype])
    res = torch.where(torch.rand(shape, generator=g) < 0.5, res, wide)
    z = vals["y"] + res.double()
    got = run_gpu(x, gamma, beta, res, dy, groups, "relu")["dres"].cpu()
    want = torch.where(z > 0, dy.double(), 0.0)
    sure = z.abs() > 2e-8 * (1 + res.double().abs())
    assert int((~sure).sum()) < z.numel() // (2 if dtype == "fp32" else 1000)
    assert torch.equal(got.double()[sure], want[sure])


@pytest.mark.gpu
def test_gpu_odd_alignment():
    """A view that starts in the middle of a 16-byte word."""
    n, h, w, c = 2, 5, 5, 16
    x, gamma, beta, res, dy = inputs(n, h, w, c, "bf16", True)
    vals, sizes = oracle(x, gamma, beta, res, dy, 4, "relu")

    def shifted(t, by):
        flat = torch.empty(t.numel() + 8, dtype=t.dtype, device=DEV)
        v = flat[by:by + t.numel()].view(t.shape)
        v.copy_(t)
        return v
    for by in (1, 2, 4):
        a, r = shifted(x, by), shifted(res, by)
        a.requires_grad_(True)
        y = O.group_norm(a, gamma.to(DEV), beta.to(DEV), 4, 1e-5, "relu", r)
        y.backward(shifted(dy, by))
        close("y", y, vals, sizes)
        close("dx", a.grad, vals, sizes)
    # and each of them alone
    for at in range(3):
        t = [x.to(DEV), res.to(DEV), dy.to(DEV)]
        t[at] = shifted(t[at], 1)
        a = t[0].requires_grad_(True)
        y = O.group_norm(a, gamma.to(DEV), beta.to(DEV), 4, 1e-5, "relu",
                         t[1])
        y.backward(t[2])
        close("y", y, vals, sizes)
        close("dx", a.grad, vals, sizes)


@pytest.mark.gpu
def test_gpu_empty():
    for shape in ((0, 4, 4, 16), (2, 0, 4, 16)):
        x = torch.zeros(shape, device=DEV, dtype=torch.bfloat16,
                        requires_grad=True)
        v = torch.ones(16, device=DEV, requires_grad=True)
        b = torch.ones(16, device=DEV, requires_grad=True)
        y = O.group_norm(x, v, b, 4, 1e-5, "relu")
        assert y.shape == x.shape
        y.sum().backward()
        assert x.grad.shape == x.shape
        assert not v.grad.any() and not b.grad.any()


@pytest.mark.gpu
def test_gpu_partial_gradients_and_views():
    """Only what is wanted is made, a dy of other strides is taken, and
    pre-allocated gradients are added to."""
    x, gamma, beta, res, dy = inputs(4, 6, 6, 32, "bf16", True)
    full = run_gpu(x, gamma, beta, res, dy, 4, "relu")
    x, gamma, beta, res, dy = (t.to(DEV) for t in (x, gamma, beta, res, dy))
    # parameters alone
    a, b = (t.clone().requires_grad_(True) for t in (gamma, beta))
    O.group_norm(x, a, b, 4, 1e-5, "relu", res).backward(dy)
    assert torch.equal(a.grad, full["dgamma"])
    # the residual alone
    r = res.clone().requires_grad_(True)
    O.group_norm(x, gamma, beta, 4, 1e-5, "relu", r).backward(dy)
    assert torch.equal(r.grad, full["dres"])
    # x alone, and a dy that is a transposed view
    t = x.clone().requires_grad_(True)
    turned = dy.transpose(1, 2).contiguous().transpose(1, 2)
    O.group_norm(t, gamma, beta, 4, 1e-5, "relu", res).backward(turned)
    assert torch.equal(t.grad, full["dx"])
    # one tensor as x and as residual: both gradients reach it
    t = x.clone().requires_grad_(True)
    O.group_norm(t, gamma, beta, 4, 1e-5, "none", t).backward(dy)
    u, v = (x.clone().requires_grad_(True) for _ in range(2))
    O.group_norm(u, gamma, beta, 4, 1e-5, "none", v).backward(dy)
    assert torch.equal(t.grad, u.grad + v.grad)
    # pre-allocated gradients are added to, twice with two uses
    a, b = (p.clone().requires_grad_(True) for p in (gamma, beta))
    a.grad, b.grad = torch.full_like(a, 2.0), torch.full_like(b, 3.0)
    view = a.grad
    O.group_norm(x, a, b, 4, 1e-5, "relu", res).backward(dy)
    assert a.grad is view
    assert torch.equal(a.grad, 2.0 + full["dgamma"])
    assert torch.equal(b.grad, 3.0 + full["dbeta"])
    O.group_norm(x, a, b, 4, 1e-5, "relu", res).backward(dy)
    assert torch.equal(a.grad, 2.0 + full["dgamma"] + full["dgamma"])


@pytest.mark.gpu
def test_gpu_refusals():
    x = torch.randn(2, 3, 3, 8, device=DEV).bfloat16()
    v = torch.ones(8, device=DEV)
    for bad in (
        lambda: O.group_norm(x.transpose(1, 2), v, v, 2),     # strides
        lambda: O.group_norm(x.double(), v, v, 2),
        lambda: O.group_norm(x, v.bfloat16(), v, 2),
        lambda: O.group_norm(x, v[:4], v, 2),
        lambda: O.group_norm(x, v.cpu(), v, 2),
        lambda: O.group_norm(x, v, v, 2, residual=x.float()),
        lambda: O.group_norm(x, v, v, 2, residual=x.cpu()),
    ):
        with pytest.raises(RuntimeError):
            bad()
    # a second derivative is refused, not made up
    t = x.clone().requires_grad_(True)
    y = O.group_norm(t, v, v, 2)
    (d,) = torch.autograd.grad(y.float().square().sum(), t, create_graph=True)
    with pytest.raises(RuntimeError):
        d.float().sum().backward()


@pytest.mark.gpu
def test_gpu_gradient_matches_differences():
    """<dx, way> against a difference of the kernel's own fp32 forward. The
    difference's error is its second-order term, taken as twice its change
    when the step is halved, and the losses' rounding over the step."""
    x, gamma, beta, res, dy = inputs(2, 9, 9, 24, "fp32", True)
    way = torch.randn(x.shape, generator=torch.Generator().manual_seed(5))
    got = run_gpu(x, gamma, beta, res, dy, 3, "silu")
    _, sizes = oracle(x, gamma, beta, res, dy, 3, "silu")
    want = float((got["dx"].cpu().double() * way.double()).sum())

    def diff(h):
        loss = []
        for s in (h, -h):
            y = run_gpu(x + s * way, gamma, beta, res, dy, 3, "silu")["y"]
            loss.append(float((y.detach().cpu().double() *
                               dy.double()).sum()))
        return (loss[0] - loss[1]) / (2 * h)
    a, b = diff(0.02), diff(0.01)
    rounding = float((dy.double().abs() * sizes["y"]).sum()) * 2 ** -24 / 0.01
    assert abs(b - want) <= 2 * abs(a - b) + rounding + 1e-3 * abs(want)


@pytest.mark.gpu
def test_gpu_captured_replays():
    """Forward and backward in a graph: every replay equals the eager pass,
    with eager work between the replays."""
    data = inputs(8, 16, 16, 64, "bf16", True)
    x, gamma, beta, res, dy = (t.to(DEV) for t in data)
    gamma.requires_grad_(True)
    beta.requires_grad_(True)
    gamma.grad, beta.grad = torch.zeros_like(gamma), torch.zeros_like(beta)
    scale = torch.ones(1, device=DEV, dtype=torch.bfloat16)
    side = torch.cuda.Stream()

    def step():
        gamma.grad.zero_()
        beta.grad.zero_()
        y = O.group_norm(x * scale, gamma, beta, 8, 1e-5, "relu", res * scale)
        y.backward(dy)
        return y
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = step()
    for k in range(4):
        x.copy_(inputs(8, 16, 16, 64, "bf16", seed=k + 1)[0])
        g.replay()
        torch.cuda.synchronize()
        got = (y.clone(), gamma.grad.clone(), beta.grad.clone())
        want = step()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want)
        assert torch.equal(got[1], gamma.grad)
        assert torch.equal(got[2], beta.grad)


@pytest.mark.gpu
def test_gpu_capture_refuses_leaves():
    x = torch.randn(2, 4, 4, 16, device=DEV).bfloat16()
    v = torch.ones(16, device=DEV, requires_grad=True)
    b = torch.zeros(16, device=DEV)
    O.group_norm(x, v.detach(), b, 4)              # loads the kernels
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = x + 1
        with pytest.raises(RuntimeError, match="captured"):
            O.group_norm(x, v, b, 4)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, x + 1)


@pytest.mark.gpu
def test_gpu_two_streams():
    """Two passes at once on streams of their own share nothing."""
    sets = [inputs(16, 16, 16, 64, "bf16", True, seed=s) for s in (1, 2)]
    want = [run_gpu(*d, 8, "relu") for d in sets]
    data = [tuple(t.to(DEV) for t in d) for d in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        got = []
        for s, (x, gamma, beta, res, dy) in zip(streams, data):
            with torch.cuda.stream(s):
                t = [p.clone().requires_grad_(True)
                     for p in (x, gamma, beta, res)]
                y = O.group_norm(t[0], t[1], t[2], 8, 1e-5, "relu", t[3])
                y.backward(dy)
                got.append((y, t))
        torch.cuda.synchronize()
        for (y, t), w in zip(got, want):
            assert torch.equal(y, w["y"])
            assert torch.equal(t[0].grad, w["dx"])
            assert torch.equal(t[1].grad, w["dgamma"])


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["resnet20", "resnet18q", "resnet50"])
def test_gpu_model_matches_cpu(name):
    """A whole model against the CPU's fp32: bf16 activations through its
    depth, so the logits are held to a few per cent of their norm, as those
    of the batch-norm models are."""
    from eventgrad_amd.parallel import FlatParamSpace
    torch.manual_seed(0)
    cpu = build_model(name, norm="group").eval()
    gpu = build_model(name, norm="group").eval()
    gpu.load_state_dict(cpu.state_dict())
    gpu.to(DEV)
    FlatParamSpace(gpu, torch.device(DEV))
    x = torch.randn(4, 3, 32, 32)
    with torch.no_grad():
        a, b = cpu(x), gpu(x.to(DEV)).cpu()
    assert ((a - b).norm() / a.norm()).item() < 5e-2


@pytest.mark.gpu
def test_gpu_one_tensor_as_gamma_and_beta():
    """Its gradient is the sum of both, also where it is added in place."""
    x, gamma, _, _, dy = (t if t is None else t.to(DEV) for t in
                          inputs(3, 5, 5, 32, "bf16"))
    a, b, one, kept = (gamma.clone().requires_grad_(True) for _ in range(4))
    t = x.clone().requires_grad_(True)
    O.group_norm(t, a, b, 4, 1e-5, "silu").backward(dy)
    O.group_norm(t, one, one, 4, 1e-5, "silu").backward(dy)
    assert torch.equal(one.grad, a.grad + b.grad)
    kept.grad = torch.zeros_like(kept)
    O.group_norm(t, kept, kept, 4, 1e-5, "silu").backward(dy)
    assert torch.equal(kept.grad, a.grad + b.grad)


@pytest.mark.gpu
@pytest.mark.parametrize("x_grad", [False, True])
def test_gpu_gradients_changed_between_forward_and_backward(x_grad):
    """The gradient goes where .grad is when the backward pass runs."""
    x, gamma, beta, _, dy = (t if t is None else t.to(DEV) for t in
                             inputs(3, 5, 5, 32, "bf16"))

    def leaves():
        return [p.clone().requires_grad_(True) for p in (gamma, beta)]

    def run(a, b):
        return O.group_norm(x.clone().requires_grad_(x_grad), a, b, 4)

    want = leaves()
    run(*want).backward(dy)
    for case in ("cleared", "half", "replaced"):
        a, b = leaves()
        a.grad, b.grad = torch.ones_like(a), torch.ones_like(b)
        old = a.grad
        y = run(a, b)
        a.grad = None if case != "replaced" else torch.full_like(a, 2.0)
        b.grad = None if case == "cleared" else torch.full_like(b, 3.0)
        y.backward(dy)
        assert torch.equal(old, torch.ones_like(old)), case
        base = [2.0 if case == "replaced" else 0.0,
                0.0 if case == "cleared" else 3.0]
        for p, q, c in zip((a, b), want, base):
            assert torch.equal(p.grad, c + q.grad), case


@pytest.mark.gpu
def test_gpu_computed_parameters_pass_their_gradients_on():
    """gamma and beta that are no leaves, and keep a gradient themselves."""
    x, gamma, beta, _, dy = (t if t is None else t.to(DEV) for t in
                             inputs(3, 5, 5, 32, "bf16"))
    roots = [p.clone().requires_grad_(True) for p in (gamma, beta)]
    a, b = (p * 2.0 for p in roots)
    a.retain_grad(), b.retain_grad()
    t = x.clone().requires_grad_(True)
    O.group_norm(t, a, b, 4, 1e-5, "relu").backward(dy, retain_graph=True)
    first = [p.grad.clone() for p in roots]
    O.group_norm(t, a, b, 4, 1e-5, "relu").backward(dy)
    for p, f in zip(roots, first):
        assert f.any() and torch.equal(p.grad, f + f)


@pytest.mark.gpu
@pytest.mark.parametrize("shape,groups", [
    ((8, 32, 32, 64), 8), ((8, 32, 32, 64), 32), ((64, 8, 8, 36), 4),
    ((1, 256, 256, 32), 2), ((1, 256, 256, 36), 6), ((40, 7, 7, 30), 6)])
def test_gpu_relu_gate_hangs_on_exact_statistics(shape, groups):
    """x is of sixteenths, so that its sums and those of its squares are exact
    in fp32; the residual takes back all of z that fp32 holds. What is left is
    2^-25 of z and less, and its sign is that of 64 bits: with the statistics
    off by 2^-50 of themselves, wherever more is left than 2^-45."""
    n, h, w, c = shape
    g = torch.Generator().manual_seed(3)
    x = (torch.randint(-60, 61, shape, generator=g) / 16.0)
    gamma = 1 + 0.5 * torch.rand(c, generator=g)
    beta = torch.randn(c, generator=g)
    xd = x.double().reshape(n, h * w, groups, c // groups)
    var, mean = torch.var_mean(xd, (1, 3), correction=0, keepdim=True)
    z = ((xd - mean) / torch.sqrt(var + 1e-5)).reshape(shape) * \
        gamma.double() + beta.double()
    res = -z.float()
    left = z + res.double()
    r = res.to(DEV).requires_grad_(True)
    O.group_norm(x.to(DEV), gamma.to(DEV), beta.to(DEV), groups, 1e-5, "relu",
                 r).backward(torch.ones(shape, device=DEV))
    sure = left.abs() > 2.0 ** -45
    assert sure.double().mean() > 0.9
    assert torch.equal((r.grad.cpu() > 0)[sure], (left > 0)[sure])


def cancelled(shape, groups, dtype, seed):
    """Inputs under which z is what fp32 leaves of it at many places, and z in
    64 bits with the absolute sum of its terms.

    In fp32 the residual takes back all of z that fp32 holds. In 16 bits,
    where a residual has too few digits, beta does it for the value that a
    channel has at one of its places, and with it for every place of the
    channel with the same value. The values' sums are not exact in fp32."""
    n, h, w, c = shape
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x = (rnd(n, h, w, c) * torch.exp(0.5 * rnd(c)) + rnd(c)).to(TYPES[dtype])
    gamma, beta = 1 + 0.5 * torch.rand(c, generator=g), rnd(c)
    xd = x.double().reshape(n, h * w, groups, c // groups)
    mean = xd.mean((1, 3), keepdim=True)
    rstd = 1 / torch.sqrt(((xd - mean) ** 2).mean((1, 3), keepdim=True) + 1e-5)
    norm = ((xd - mean) * rstd).reshape(shape) * gamma.double()
    terms = ((xd.abs() + mean.abs()) * rstd).reshape(shape) * gamma.double()
    if dtype == "fp32":
        res = -(norm + beta.double()).float()
    else:
        at = torch.randint(0, h * w, (c,), generator=g)
        beta = -norm[0].reshape(h * w, c)[at, torch.arange(c)].float()
        res = torch.zeros_like(x)
    z = norm + beta.double() + res.double()
    return x, gamma, beta, res, z, terms + beta.double().abs() + res.double().abs()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("shape,groups", [
    ((1, 128, 128, 64), 8), ((1, 128, 128, 256), 2),   # long: whole vectors
    ((1, 128, 128, 320), 32), ((2, 150, 150, 30), 6),  # across them
    ((1, 40, 50, 8208), 2),                            # slices of one group
    ((4, 32, 32, 64), 8), ((4, 16, 16, 36), 4)])       # slabs
def test_gpu_relu_gate_with_sums_that_round(shape, groups, dtype):
    """z is at most 2^-24 of its terms at many places, and its bit there hangs
    on the mean and rstd to as many digits. All of their sums are in 64 bits:
    a chain of under 1,024 additions, each off by 2^-53 of the sum, twice over
    for the mean and the squares. 2^-40 of the terms is four times that."""
    x, gamma, beta, res, z, terms = cancelled(shape, groups, dtype, 7)
    r = res.to(DEV).requires_grad_(True)
    O.group_norm(x.to(DEV), gamma.to(DEV), beta.to(DEV), groups, 1e-5, "relu",
                 r).backward(torch.ones(shape, device=DEV, dtype=x.dtype))
    sure = z.abs() > 2.0 ** -40 * terms
    next_to = sure & (z.abs() <= 2.0 ** -24 * terms)
    assert int(next_to.sum()) >= 30 and sure.double().mean() > 0.999
    wrong = (r.grad.cpu() > 0) != (z > 0)
    assert not wrong[sure].any(), \
        f"{int(wrong[sure].sum())} of {int(next_to.sum())}"


def _dual_calls(device, call):
    """Each of the inputs in turn with a tangent, with frozen parameters,
    trained ones and those that have a gradient already, with and without
    recorded gradients: none may come out as if it had no derivative."""
    import torch.autograd.forward_ad as fw
    x = torch.randn(2, 3, 3, 8, device=device).bfloat16()
    for trained in (False, True):
        for at in range(4):
            v = [x, torch.ones(8, device=device), torch.ones(8, device=device),
                 x.clone()]
            for p in v[1:3]:
                p.requires_grad_(trained)
                p.grad = torch.zeros_like(p) if trained else None
            for grad in (True, False):
                with fw.dual_level(), torch.set_grad_enabled(grad):
                    args = list(v)
                    args[at] = fw.make_dual(v[at], torch.ones_like(v[at]))
                    with pytest.raises(NotImplementedError,
                                       match="forward-mode"):
                        call(*args)


def test_forward_mode_is_refused():
    """The check comes before the one for the device."""
    from eventgrad_amd.ops.backend import native, native_available
    if not native_available():
        pytest.skip("the extension is not built")
    _dual_calls("cpu", lambda x, a, b, r: native().group_norm(
        x, a, b, r, 2, 1e-5, 1))


@pytest.mark.gpu
def test_gpu_forward_mode_is_refused():
    _dual_calls(DEV, lambda x, a, b, r: O.group_norm(
        x, a, b, 2, 1e-5, "relu", r))


@pytest.mark.gpu
def test_gpu_capture_refuses_one_trained_parameter():
    """Gradients are added in place where gamma and beta both have one. With
    the other frozen, or computed, autograd would accumulate into the leaf."""
    x = torch.randn(2, 4, 4, 16, device=DEV).bfloat16()
    trained = torch.ones(16, device=DEV, requires_grad=True)
    trained.grad = torch.zeros_like(trained)
    frozen = torch.zeros(16, device=DEV)
    # frozen parameters are taken, and so are those that both have gradients
    other = frozen.clone().requires_grad_(True)
    other.grad = torch.zeros_like(other)
    O.group_norm(x, frozen, frozen, 4)             # loads the kernels
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for pair in ((trained, frozen), (frozen, trained)):
            with pytest.raises(RuntimeError, match="both of them"):
                O.group_norm(x, *pair, 4)
        y = O.group_norm(x, trained, other, 4)
        z = O.group_norm(x, frozen + 1, frozen, 4)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, z)
    assert torch.equal(z, O.group_norm(x, frozen + 1, frozen, 4))
    # and outside of one each keeps its gradient
    O.group_norm(x, trained, frozen, 4).float().square().sum().backward()
    assert trained.grad.any()


@pytest.mark.gpu
def test_gpu_captured_beside_a_living_eager_graph():
    """Parameters alone are trained, x is data, and an eager graph of the same
    parameters lives while the pass is captured."""
    x, gamma, beta, _, dy = (t if t is None else t.to(DEV) for t in
                             inputs(3, 5, 5, 32, "bf16"))
    leaves = [p.clone().requires_grad_(True) for p in (gamma, beta)]
    for p in leaves:
        p.grad = torch.zeros_like(p)
    living = O.group_norm(x, *leaves, 4, 1e-5, "relu")
    living.backward(dy, retain_graph=True)
    want = [p.grad.clone() for p in leaves]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for p in leaves:
            p.grad.zero_()
        O.group_norm(x, *leaves, 4, 1e-5, "relu").backward(dy)
    for _ in range(3):
        for p in leaves:
            p.grad.fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p.grad, w) for p, w in zip(leaves, want))
    living.backward(dy)
    assert all(torch.equal(p.grad, w + w) for p, w in zip(leaves, want))


@pytest.mark.gpu
@pytest.mark.parametrize("shape,groups", [
    ((2, 32, 32, 64), 8), ((3, 16, 16, 36), 4),         # slabs
    ((1, 150, 150, 16), 2), ((1, 150, 150, 36), 4)])    # long samples
def test_gpu_large_mean_costs_no_digits(shape, groups):
    """A mean of a thousand spreads under a ReLU, whose sums are in 64 bits:
    fp32 has neither the mean nor what x - mean is off by when it is rounded,
    3e-5 of a spread. x less a rounded mean is exact (both have one exponent),
    and what the mean was rounded by is at most 2^-14 of a spread; the rest
    rounds as for a mean of zero, 128 times at most, terms of these sizes."""
    n, h, w, c = shape
    g = torch.Generator().manual_seed(11)
    x = torch.randn(shape, generator=g) + 1000.0
    gamma, beta = 1 + torch.rand(c, generator=g), torch.zeros(c)
    dy = torch.randn(shape, generator=g) + 1.0
    vals, _ = oracle(x, gamma, beta, None, dy, groups, "relu")
    split = lambda t: t.double().reshape(n, h * w, groups, c // groups)  # noqa: E731
    total = lambda t: split(t).mean((1, 3), keepdim=True)  # noqa: E731
    rstd = 1 / torch.sqrt(total((split(x) - total(x)).reshape(shape) ** 2) + 1e-5)
    xh = ((split(x) - total(x)) * rstd).abs() + 2.0 ** -14
    d = split((gamma.double() * vals["dres"]).abs())
    size = {"y": xh.reshape(shape) * gamma.double(),
            "dbeta": vals["dres"].abs().sum((0, 1, 2)),
            "dgamma": (vals["dres"].abs() * xh.reshape(shape)).sum((0, 1, 2)),
            "dx": (rstd * (d + total(d.reshape(shape)) + xh * total(
                (d * xh).reshape(shape)))).reshape(shape)}
    got = run_gpu(x, gamma, beta, None, dy, groups, "relu")
    for name, t in got.items():
        close(name, t, vals, size)


@pytest.mark.gpu
@pytest.mark.parametrize("shape,groups", [
    ((2, 32, 32, 64), 8), ((3, 16, 16, 36), 4),         # slabs
    ((1, 150, 150, 16), 2), ((1, 150, 150, 36), 4)])    # long samples
def test_gpu_huge_mean_keeps_the_spread(shape, groups):
    """A mean of 2^20 spreads, x in sixteenths of one. Variances are added up
    from distances, so that 64 bits keep all the digits of a spread that 24
    have; as mean squares they would leave 53 - 40. What a mean is rounded by
    is up to 2^-5 of a spread, added to the sizes of the terms."""
    n, h, w, c = shape
    g = torch.Generator().manual_seed(12)
    x = torch.randn(shape, generator=g) + 2.0 ** 20
    gamma, beta = 1 + torch.rand(c, generator=g), torch.zeros(c)
    dy = torch.randn(shape, generator=g) + 1.0
    vals, _ = oracle(x, gamma, beta, None, dy, groups, "relu")
    split = lambda t: t.double().reshape(n, h * w, groups, c // groups)  # noqa: E731
    off = split(x) - split(x).mean((1, 3), keepdim=True)
    xh = (off / off.square().mean((1, 3), keepdim=True).sqrt()).abs()
    size = {"y": (xh + 2.0 ** -5).reshape(shape) * gamma.double(),
            "dgamma": (vals["dres"].abs() *
                       (xh + 2.0 ** -5).reshape(shape)).sum((0, 1, 2))}
    got = run_gpu(x, gamma, beta, None, dy, groups, "relu")
    for name in size:
        close(name, got[name], vals, size)
