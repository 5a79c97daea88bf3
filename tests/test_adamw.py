"""AdamW over the flat space, moments in 32 and in 8 bits."""

import math

import pytest
import torch

from eventgrad_amd.parallel import AdamW, FlatParamSpace
from eventgrad_amd.parallel import adamw as A

SHAPES = [(7,), (130, 3), (64,), (1,), (5000, 2), (65,), (4096,), (33, 1, 3)]


def space_of(shapes=SHAPES, device="cpu", seed=0):
    model = torch.nn.ParameterList(
        [torch.nn.Parameter(torch.empty(s)) for s in shapes]).to(device)
    space = FlatParamSpace(model, torch.device(device))
    g = torch.Generator().manual_seed(seed)
    for i in range(space.sz):
        space.seg(space.param, i).copy_(
            torch.randn(space.numels[i], generator=g) * 0.1)
    return space, model


def set_grads(space, seed):
    """Gradients of very different size, some of them zero."""
    g = torch.Generator().manual_seed(1000 + seed)
    for i in range(space.sz):
        v = torch.randn(space.numels[i], generator=g) * 10.0 ** -(i % 5)
        v *= torch.rand(space.numels[i], generator=g) > 0.1
        space.seg(space.grad, i).copy_(v)


def oracle(shapes, steps, lr, betas, eps, wd, decay_1d):
    """param, m, v in 64 bits, from the definition, tensor by tensor."""
    space, _ = space_of(shapes)
    b1, b2 = betas
    p = space.param.double().clone()
    m, v = torch.zeros_like(p), torch.zeros_like(p)
    for t in range(1, steps + 1):
        set_grads(space, t)
        g = space.grad.double()
        m = b1 * m + (1 - b1) * g
        v = b2 * v + (1 - b2) * g * g
        for i, s in enumerate(shapes):
            w = wd if decay_1d or len(s) > 1 else 0.0
            q, mm, vv = (space.seg(t_, i) for t_ in (p, m, v))
            q.copy_(q - lr * w * q - lr * (mm / (1 - b1 ** t)) /
                    (torch.sqrt(vv / (1 - b2 ** t)) + eps))
    return p, m, v


def devices():
    return ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


HYPER = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)


@pytest.mark.parametrize("device", devices())
@pytest.mark.parametrize("decay_1d", [True, False])
def test_32_bits_match_definition(device, decay_1d):
    """Six steps. Each rounds a handful of times, off by 2^-24 of the value or
    of an update of lr, and beta rounded to fp32 is off by 2^-24 too: 64
    roundings in all are allowed. A moment may have passed close to zero, so
    it is held against the sizes that it was made of."""
    steps = 6
    space, _model = space_of(device=device)
    opt = AdamW(space, decay_1d=decay_1d, **HYPER)
    for t in range(1, steps + 1):
        set_grads(space, t)
        norms = opt.step()
    p, m, v = oracle(SHAPES, steps, HYPER["lr"], HYPER["betas"],
                     HYPER["eps"], HYPER["weight_decay"], decay_1d)
    unit = 64 * 2.0 ** -24
    got = [t.cpu().double() for t in (space.param, *opt.moments())]
    assert float((got[0] - p).abs().max()) <= unit * (
        float(p.abs().max()) + steps * HYPER["lr"] * 4)
    for i in range(space.sz):
        for a, b in ((got[1], m), (got[2], v)):
            a, b = space.seg(a, i), space.seg(b, i)
            assert float((a - b).abs().max()) <= unit * 4 * float(
                b.abs().max())
        want = float(space.seg(p, i).square().sum())
        # and a sum of up to 10,000 squares, in runs and pairs
        assert abs(float(norms[i]) - want) <= 4 * unit * want
    assert opt.steps == steps
    # the gaps between tensors stay zero
    gaps = torch.ones(space.total, dtype=torch.bool)
    for s, n in zip(space.starts, space.numels):
        gaps[s:s + n] = False
    assert not space.param.cpu()[gaps].any()


def test_matches_torch_optimizer():
    torch.manual_seed(0)
    space, model = space_of()
    mine = AdamW(space, lr=1e-2, weight_decay=0.1)
    other = [torch.nn.Parameter(p.detach().clone()) for p in model]
    ref = torch.optim.AdamW(other, lr=1e-2, weight_decay=0.1)
    for t in range(5):
        set_grads(space, t)
        for p, q in zip(model, other):
            q.grad = p.grad.clone()
        mine.step()
        ref.step()
        for p, q in zip(model, other):
            assert torch.allclose(p, q, rtol=1e-5, atol=1e-7)


# ---------------------------------------------------------------- the 8 bits

def _round_trip(x, exp_bits, random):
    q, e = A._encode(x, random, exp_bits)
    return q, e, A._decode(q, e, exp_bits)


@pytest.mark.parametrize("exp_bits", [4, 5])
def test_grid_values_survive(exp_bits):
    """Every byte stands for a value that comes back as itself, whatever the
    random bits, when the block's largest is in it."""
    q = torch.arange(8 << exp_bits)
    q = torch.cat([q, q.new_zeros(-len(q) % A.QBLOCK)])
    for e in (40, 127, 200):
        x = A._decode(q, torch.full((len(q) // A.QBLOCK,), e), exp_bits)
        rows = x.view(-1, A.QBLOCK)
        rows[:, 0] = 1.875 * 2.0 ** (e - 127)
        for r in (0, 1, 65535):
            got, ge, back = _round_trip(x, exp_bits, torch.full(x.shape, r))
            assert torch.equal(back, x)
            assert bool((ge == e).all())


@pytest.mark.parametrize("exp_bits", [4, 5])
def test_rounding_is_to_a_neighbour_and_unbiased(exp_bits):
    """A value goes to one of its two neighbours on the grid, and up for as
    many of the 65,536 random values as its place between them says: the mean
    over all of them is the value, to the 16 bits that it is cut at."""
    g = torch.Generator().manual_seed(3)
    x = torch.rand(A.QBLOCK, generator=g) * 2.0 ** -torch.arange(
        A.QBLOCK).div(4, rounding_mode="floor").float()
    x[0] = 1.9
    _, e = A._encode(x, torch.zeros_like(x, dtype=torch.int64), exp_bits)
    total = torch.zeros(A.QBLOCK, dtype=torch.float64)
    low = torch.full((A.QBLOCK,), math.inf, dtype=torch.float64)
    high = -low
    for r in range(0, 65536, 16):
        _, _, back = _round_trip(x, exp_bits, torch.full(x.shape, r))
        total += back.double()
        low = torch.minimum(low, back.double())
        high = torch.maximum(high, back.double())
    step = high - low
    # 8 steps an octave; below the smallest normal the step stays
    scale = 2.0 ** (float(e[0]) - 127)
    least = scale * 2.0 ** -(1 + (1 << exp_bits))
    assert bool((step <= torch.maximum(x.double() / 8,
                                       torch.tensor(least))).all())
    assert bool(((low <= x) & (x <= high)).all())
    # 4,096 of the 65,536 values, evenly: a step's 4,096th
    off = (total / 4096 - x.double()).abs()
    assert bool((off <= step / 4096 + 1e-12 * scale).all())


def test_moment_follows_where_nearest_would_stick():
    """A constant gradient, larger than before: v creeps by 0.1 % a step, an
    eighth of a step of the grid's at most, and gets there. 1,024 values with
    random bits of their own: each is off by at most a step (1/8), and their
    mean by a fraction of it; 10 % is allowed."""
    space, _ = space_of([(1024,)])
    opt = AdamW(space, lr=0.0, betas=(0.9, 0.999), state_bits=8,
                weight_decay=0.0)
    space.grad.fill_(1.0)
    for _ in range(1000):
        opt.step()
    m, v = (t.float() for t in opt.moments())
    want = 1 - 0.999 ** 1000
    assert abs(float(v.mean()) / want - 1) < 0.1
    assert abs(float(m.mean()) - 1) < 0.1


def test_small_second_moment_never_zero():
    """Beside a gradient of 1 one of 1e-9: v is below the grid, and would be
    zero; the step must stay a step."""
    space, _ = space_of([(64,)])
    before = space.param.clone()
    opt = AdamW(space, lr=1e-3, weight_decay=0.0, state_bits=8, eps=1e-12)
    space.grad.fill_(1e-9)
    space.grad[0] = 1.0
    for _ in range(20):
        opt.step()
    _, v = opt.moments()
    assert bool((v > 0).all())
    assert float((space.param - before).abs().max()) <= 20 * 1e-3 * 4


@pytest.mark.parametrize("device", devices())
def test_nonfinite_block(device):
    space, _ = space_of([(64,), (200,)], device)
    opt = AdamW(space, state_bits=8)
    set_grads(space, 1)
    space.grad[70] = float("inf")
    opt.step()
    m, v = (t.float().cpu() for t in opt.moments())
    assert torch.isnan(m[64:128]).all() and torch.isnan(v[64:128]).all()
    keep = torch.cat([torch.arange(64), torch.arange(128, space.total)])
    assert torch.isfinite(m[keep]).all() and torch.isfinite(v[keep]).all()


@pytest.mark.parametrize("device", devices())
def test_extreme_sizes(device):
    """Gradients whose squares leave fp32's range, at both ends."""
    space, _ = space_of([(64,), (64,), (64,)], device)
    opt = AdamW(space, lr=1e-3, state_bits=8)
    space.seg(space.grad, 0).fill_(1e-25)       # g^2 = 0 in fp32
    space.seg(space.grad, 1).fill_(1e15)
    space.seg(space.grad, 2).fill_(0.0)
    for _ in range(3):
        opt.step()
    m, v = (t.float().cpu() for t in opt.moments())
    assert torch.isfinite(space.param).all()
    assert torch.isfinite(m).all() and torch.isfinite(v).all()
    assert not m[128:].any() and not v[128:].any()
    assert float(m[64]) > 0 and float(v[64]) > 0


@pytest.mark.gpu
@pytest.mark.parametrize("shapes", [SHAPES, [(1,)], [(3, 3)] * 300,
                                    [(70000,), (4097, 5)],
                                    [(255 * 1024, 1), (5,)],   # 256 chunks
                                    [(256 * 1024,), (5, 7)],   # 257
                                    [(3, 1000)] * 400],
                         ids=lambda s: f"{len(s)}x{s[0]}")
def test_gpu_8_bits_equal_cpu(shapes):
    """The codes are the CPU's to the bit, step after step: what decides them
    is rounded after each operation on both sides. The weights are off by the
    rounding of a division and a root, 2^-23 of each update and of
    themselves; 16 are allowed for each step."""
    sides = []
    for device in ("cpu", "cuda"):
        space, model = space_of(shapes, device)
        sides.append((space, AdamW(space, state_bits=8, decay_1d=False,
                                   seed=7, **HYPER), model))
    for t in range(1, 6):
        norms = []
        for space, opt, _ in sides:
            set_grads(space, t)
            norms.append(opt.step().cpu())
        (sa, a, _), (sb, b, _) = sides
        assert torch.equal(a.codes, b.codes.cpu())
        assert torch.equal(a.exponents, b.exponents.cpu())
        off = (sa.param - sb.param.cpu()).abs()
        assert float(off.max()) <= 16 * t * 2.0 ** -23 * (
            float(sa.param.abs().max()) + HYPER["lr"] * 10)
        assert torch.allclose(norms[0], norms[1], rtol=1e-5)
        assert all(torch.equal(x, y.cpu())
                   for x, y in zip(a.moments(), b.moments()))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_gpu_same_every_time(bits):
    outs = []
    for _ in range(3):
        space, model = space_of(device="cuda")
        opt = AdamW(space, state_bits=bits, **HYPER)
        for t in range(3):
            set_grads(space, t)
            norms = opt.step()
        outs.append((space.param.clone(), norms, *opt.moments()))
    for other in outs[1:]:
        assert all(torch.equal(x, y) for x, y in zip(outs[0], other))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_gpu_captured_step_counts_on(bits):
    """A captured step replayed, with eager work and a change of the learning
    rate between the replays, is the same step taken eagerly."""
    pair = []
    for _ in range(2):
        space, model = space_of(device="cuda")
        pair.append((space, AdamW(space, state_bits=bits, seed=3, **HYPER),
                     model))
    (sa, a, _), (sb, b, _) = pair
    set_grads(sa, 0)
    set_grads(sb, 0)
    a.step()
    b.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norms = a.step()
    for t in range(1, 5):
        for s in (sa, sb):
            set_grads(s, t)
        if t == 3:
            a.lr = b.lr = 1e-2
        graph.replay()
        want = b.step()
        torch.cuda.synchronize()
        assert torch.equal(norms, want)
        assert torch.equal(sa.param, sb.param)
        assert all(torch.equal(x, y) for x, y in zip(a.moments(),
                                                     b.moments()))
    assert a.steps == b.steps == 5


@pytest.mark.gpu
def test_gpu_two_streams():
    sides = []
    for k in range(2):
        space, model = space_of(device="cuda", seed=k)
        set_grads(space, k)
        sides.append((space, AdamW(space, state_bits=8, seed=k), model))
    want = []
    for k in range(2):
        space, model = space_of(device="cuda", seed=k)
        set_grads(space, k)
        opt = AdamW(space, state_bits=8, seed=k)
        for _ in range(10):
            opt.step()
        want.append((space.param, *opt.moments()))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sides]
    for _ in range(10):
        for s, (_, opt, _) in zip(streams, sides):
            with torch.cuda.stream(s):
                opt.step()
    torch.cuda.synchronize()
    for (space, opt, _), w in zip(sides, want):
        assert all(torch.equal(x, y)
                   for x, y in zip((space.param, *opt.moments()), w))


# ---------------------------------------------------------------- state

@pytest.mark.parametrize("device", devices())
@pytest.mark.parametrize("bits", [8, 32])
def test_state_resumes_to_the_bit(device, bits):
    space, _m = space_of(device=device)
    opt = AdamW(space, state_bits=bits, seed=11, **HYPER)
    for t in range(3):
        set_grads(space, t)
        opt.step()
    saved, params = opt.state_dict(), space.param.clone()
    other, _m2 = space_of(device=device, seed=5)
    resumed = AdamW(other, state_bits=bits, **HYPER)
    resumed.load_state_dict(saved)
    other.load_flat(params)
    for t in range(3, 6):
        for s, o in ((space, opt), (other, resumed)):
            set_grads(s, t)
            o.step()
    assert torch.equal(space.param, other.param)
    assert all(torch.equal(x, y)
               for x, y in zip(opt.moments(), resumed.moments()))


@pytest.mark.parametrize("device", devices())
def test_state_carries_the_corrections(device):
    """b^t is a product on the GPU, and a resumed run goes on with the same
    one; with other betas it is the new ones' power."""
    space, _m = space_of(device=device)
    opt = AdamW(space, **HYPER)
    set_grads(space, 0)
    for _ in range(60):
        opt.step()
    saved = opt.state_dict()
    resumed = AdamW(space, **HYPER)
    resumed.load_state_dict(saved)
    assert resumed._powers.tolist() == opt._powers.tolist()
    assert resumed._coef.tolist() == opt._coef.tolist()
    other = AdamW(space, **{**HYPER, "betas": (0.5, 0.75)})
    other.load_state_dict(saved)
    assert other._powers.tolist() == [0.5 ** 61, 0.75 ** 61]


def test_state_refusals():
    space, _ = space_of()
    opt = AdamW(space, state_bits=8)
    with pytest.raises(ValueError):
        opt.load_state_dict(AdamW(space).state_dict())
    with pytest.raises(ValueError):
        opt.load_state_dict({"kind": "sgd"})
    small, _ = space_of([(3,)])
    with pytest.raises(ValueError):
        opt.load_state_dict(AdamW(small, state_bits=8).state_dict())


@pytest.mark.parametrize("kw", [
    dict(lr=-1.0), dict(lr=math.nan), dict(betas=(1.0, 0.9)),
    dict(betas=(0.9, -0.1)), dict(eps=0.0), dict(eps=-1e-8), dict(eps=1e-13),
    dict(weight_decay=-1.0), dict(state_bits=16)])
def test_refusals(kw):
    space, _ = space_of([(3,)])
    with pytest.raises(ValueError):
        AdamW(space, **kw)


@pytest.mark.gpu
def test_gpu_refusals():
    space, _model = space_of(device="cuda")
    opt = AdamW(space, state_bits=8)
    good = space.grad
    for bad in (good.double(), good[:-64], good.cpu(), good[1:]):
        space.grad = bad
        with pytest.raises(RuntimeError):
            opt.step()
    space.grad = good
    opt.step()
    assert opt.steps == 1


def test_memory_of_8_bits():
    space, _ = space_of([(100000,)])
    opt = AdamW(space, state_bits=8)
    held = sum(t.numel() * t.element_size()
               for t in opt.state_dict().values()
               if isinstance(t, torch.Tensor))
    assert held == space.total * 2 + 2 * space.total // 64


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_gpu_captured_step_follows_weight_decay(bits):
    pair = []
    for _ in range(2):
        space, model = space_of(device="cuda")
        set_grads(space, 0)
        opt = AdamW(space, state_bits=bits, decay_1d=False, **HYPER)
        opt.step()
        pair.append((space, opt, model))
    (sa, a, _), (sb, b, _) = pair
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step()
    for wd in (0.1, 0.5, 0.0, 0.5):
        a.weight_decay = b.weight_decay = wd
        graph.replay()
        b.step()
        torch.cuda.synchronize()
        assert torch.equal(sa.param, sb.param), wd
