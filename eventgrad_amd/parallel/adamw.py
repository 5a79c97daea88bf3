"""AdamW over the flat parameter space, moments in 32 or in 8 bits.

    m <- b1 m + (1 - b1) g
    v <- b2 v + (1 - b2) g^2
    p <- p - lr wd p - lr (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps)

One step takes every tensor of the space and returns each one's squared L2
norm, which is what the event trigger reads, like the SGD step beside it. On
the GPU it is csrc/adamw.hip; the CPU computes the same, to the bit in the
8-bit moments, and is its oracle.

8-bit moments take 2 1/32 bytes a parameter in the place of 8. Each block of
64 values shares a power of two, 2^(E - 127) with E in a byte, that leaves the
largest below 2 once it is rounded up; on top of it a value of m has a sign, 4
bits of exponent and 3 behind the leading one (2^-17 to 1.875), a value of v
has no sign and 5 bits of exponent (2^-33 to 1.875). Rounding is stochastic,
from 16 hashed bits of (seed, step, place): a step moves v by about 1 - b2 of
itself, far below the grid, and rounding to nearest would never move it. A v
above zero never becomes zero. A block with a value that is not finite has
E = 255 and reads as NaN.
"""

from __future__ import annotations

import math

import torch

from ..ops.backend import native
from .flat import ALIGN, FlatParamSpace

QBLOCK = 64       # values that share an exponent; divides ALIGN
# Values of one kernel block, a multiple of QBLOCK: four a thread, none of
# which then waits behind another. The 8-bit step of 17.4 M weights took 56 us
# with 1,024, 62 us with 4,096 and 68 us with 16,384.
CHUNK = 1024

assert ALIGN % QBLOCK == 0 and CHUNK % QBLOCK == 0


# --------------------------------------------------------------------------
# the 8-bit grid, in torch (the kernel's oracle)
# --------------------------------------------------------------------------

_U32 = 0xFFFFFFFF


def _hash_u32(seed, index):
    """csrc/common.h hash_u32 on int64 tensors that hold 32-bit values."""
    h = seed ^ (index * 0x9E3779B9 & _U32)
    h = (h ^ 61) ^ (h >> 16)
    h = h * 9 & _U32
    h = h ^ (h >> 4)
    h = h * 0x27D4EB2D & _U32
    return h ^ (h >> 15)


def _random_bits(seed: int, step: int, n: int, device) -> torch.Tensor:
    place = torch.arange(n, dtype=torch.int64, device=device)
    key = _hash_u32(torch.tensor(seed & _U32, device=device),
                    torch.tensor(step & _U32, device=device))
    return _hash_u32((key + (place >> 32)) & _U32, place & _U32)


def _encode(x, random, exp_bits):
    """The magnitudes' bytes [n] and the blocks' exponents [n / QBLOCK]."""
    bias = (1 << exp_bits) - 1
    bits = x.view(torch.int32).to(torch.int64) & 0x7FFFFFFF
    top = bits.view(-1, QBLOCK).amax(1)
    e = ((top + 0xFFFFF) >> 23).clamp(2 + (1 << exp_bits), 254)
    lift = (127 - e).repeat_interleave(QBLOCK)
    y = torch.ldexp(x.abs().double(), lift)
    y = torch.where(torch.isfinite(y), y, 0.0)
    mantissa = y.float().view(torch.int32).to(torch.int64)
    normal = ((mantissa + (random << 4)) >> 20) - ((127 - bias) << 3)
    low = (torch.floor(y * 2.0 ** (bias + 18)).to(torch.int64) + random) >> 16
    q = torch.where(y < 2.0 ** (1 - bias), low, normal)
    q = q.clamp_max((8 << exp_bits) - 1)
    return q, torch.where(top >= 0x7F800000, 255, e)


def _decode(q, e, exp_bits):
    bias = (1 << exp_bits) - 1
    field, last = q >> 3, (q & 7).double()
    y = torch.where(field > 0,
                    torch.ldexp(8.0 + last, field - bias - 3),
                    last * 2.0 ** (-2 - bias))
    e = e.repeat_interleave(QBLOCK)
    return torch.where(e == 255, math.nan, torch.ldexp(y, e - 127)).float()


def _split(codes, exps):
    """(m's bytes, v's bytes, m's exponents, v's exponents), as int64."""
    c = codes.view(-1, 2, 4).to(torch.int64)
    e = exps.view(-1, 2).to(torch.int64)
    return (c[:, 0].reshape(-1), c[:, 1].reshape(-1), e[:, 0], e[:, 1])


def _unpack(codes, exps):
    m, v, em, ev = _split(codes, exps)
    mv = _decode(m & 127, em, 4)
    return torch.where(m >= 128, -mv, mv), _decode(v, ev, 5)


def _pack(m, v, random, codes, exps):
    qm, em = _encode(m, random & 0xFFFF, 4)
    qv, ev = _encode(v, random >> 16, 5)
    qm = qm | (torch.signbit(m).to(torch.int64) << 7)
    qv = torch.where((qv == 0) & (v > 0), 1, qv)
    codes.view(-1, 2, 4).copy_(
        torch.stack([qm.view(-1, 4), qv.view(-1, 4)], 1).to(torch.uint8))
    exps.view(-1, 2).copy_(torch.stack([em, ev], 1).to(torch.uint8))


# --------------------------------------------------------------------------
# the optimizer
# --------------------------------------------------------------------------

class AdamW:
    """AdamW on a FlatParamSpace.

    state_bits: 32, or 8 for moments in 8 bits. decay_1d: whether weight decay
    reaches the tensors with fewer than two dimensions (biases, norm
    weights). seed: of the 8-bit moments' rounding.

    step() takes space.grad as it is, updates space.param and the moments,
    and returns the tensors' squared norms [sz]; it does not refresh the bf16
    weight shadows (space.refresh_shadows does). The learning rate, the
    decays, the step count and the bias corrections live on the space's
    device, so a step that was captured into a graph counts on and follows a
    new `lr` or `weight_decay` when it is replayed.
    """

    def __init__(self, space: FlatParamSpace, lr: float = 1e-3,
                 betas=(0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 0.01, decay_1d: bool = True,
                 state_bits: int = 32, seed: int = 0):
        b1, b2 = (float(b) for b in betas)
        if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
            raise ValueError(f"betas must be in [0, 1), got {betas}")
        if not 1e-12 <= eps < math.inf:
            raise ValueError(f"eps must be at least 1e-12, got {eps}")
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits}")
        self.space = space
        self.betas, self.eps = (b1, b2), float(eps)
        self.decay_1d = bool(decay_1d)
        self.state_bits, self.seed = state_bits, int(seed)
        dev, n = space.param.device, space.total
        f32 = dict(dtype=torch.float32, device=dev)
        i64 = dict(dtype=torch.int64, device=dev)
        u8 = dict(dtype=torch.uint8, device=dev)
        if state_bits == 32:
            self.exp_avg = torch.zeros(n, **f32)
            self.exp_avg_sq = torch.zeros(n, **f32)
            self.codes = torch.empty(0, **u8)
            self.exponents = torch.empty(0, **u8)
        else:
            self.exp_avg = self.exp_avg_sq = torch.empty(0, **f32)
            # for each 4 values 4 bytes of m, then 4 of v
            self.codes = torch.zeros(2 * n, **u8)
            # for each block of values m's exponent, then v's
            self.exponents = torch.tensor([18, 34], **u8).repeat(n // QBLOCK)
        # which tensors decay, and each one's decay
        self._decays = torch.tensor([bool(decay_1d or len(s) >= 2)
                                     for s in space.shapes], device=dev)
        self._decay = torch.zeros(space.sz, **f32)
        # the kernel's plan: no chunk crosses a tensor
        numels = torch.tensor(space.numels, dtype=torch.int64)
        counts = (numels + CHUNK - 1) // CHUNK
        first = torch.nn.functional.pad(counts.cumsum(0), (1, 0))
        tensor = torch.repeat_interleave(torch.arange(space.sz), counts)
        into = (torch.arange(len(tensor)) - first[tensor]) * CHUNK
        starts = torch.tensor(space.starts, dtype=torch.int64)
        self._chunks = torch.stack(
            [starts[tensor] + into,
             (numels[tensor] - into).clamp_max(CHUNK), tensor], 1).to(dev)
        self._first = first.to(dev)
        self._step = torch.zeros(1, **i64)
        # scratch of the norms, and behind it a counter that ends at zero
        self._part = torch.zeros(len(tensor) + 1, **f32)
        # of the next step: lr, 1 / (1 - b1^t), 1 / sqrt(1 - b2^t); b1^t, b2^t
        self._coef = torch.zeros(3, **f32)
        self._powers = torch.zeros(2, dtype=torch.float64, device=dev)
        self.lr = lr
        self.weight_decay = weight_decay
        self._set_corrections(1)

    # -- scalars -------------------------------------------------------------
    @property
    def lr(self) -> float:
        return self._lr

    @lr.setter
    def lr(self, value: float) -> None:
        if not 0.0 <= value < math.inf:
            raise ValueError(f"lr must not be negative, got {value}")
        self._lr = float(value)
        self._coef[0] = self._lr

    @property
    def weight_decay(self) -> float:
        return self._weight_decay

    @weight_decay.setter
    def weight_decay(self, value: float) -> None:
        if not 0.0 <= value < math.inf:
            raise ValueError(f"weight_decay must not be negative, "
                             f"got {value}")
        self._weight_decay = float(value)
        torch.mul(self._decays, self._weight_decay, out=self._decay)

    @property
    def steps(self) -> int:
        """Steps taken (waits for the device)."""
        return int(self._step.item())

    def _set_corrections(self, t: int) -> None:
        """Those of step t, which is the next."""
        p1, p2 = (b ** t for b in self.betas)
        self._powers.copy_(torch.tensor([p1, p2], dtype=torch.float64))
        self._coef[1:].copy_(torch.tensor(
            [1.0 / (1.0 - p1), 1.0 / math.sqrt(1.0 - p2)]))

    # -- the step ------------------------------------------------------------
    def step(self) -> torch.Tensor:
        sp = self.space
        if sp.param.is_cuda:
            return native().adamw_step_norm(
                sp.param, sp.grad, self.exp_avg, self.exp_avg_sq, self.codes,
                self.exponents, self._chunks, self._first, self._decay,
                self._coef, self._powers, self._step, self._part,
                self.betas[0], self.betas[1], self.eps, self.seed)
        return self._step_cpu()

    def _step_cpu(self) -> torch.Tensor:
        sp, (b1, b2) = self.space, self.betas
        t = self.steps + 1
        if self.state_bits == 32:
            m, v = self.exp_avg, self.exp_avg_sq
        else:
            m, v = _unpack(self.codes, self.exponents)
        g = sp.grad
        m.mul_(b1).add_(g * (1.0 - b1))
        v.mul_(b2).add_(g * g * (1.0 - b2))
        update = m / (v.sqrt() / math.sqrt(1.0 - b2 ** t) + self.eps)
        for i in range(sp.sz):
            d = float(self._decay[i])
            if d:
                sp.seg(sp.param, i).mul_(1.0 - self._lr * d)
        sp.param.add_(update, alpha=-self._lr / (1.0 - b1 ** t))
        if self.state_bits == 8:
            _pack(m, v, _random_bits(self.seed, t, sp.total, g.device),
                  self.codes, self.exponents)
        self._step += 1
        self._set_corrections(t + 1)
        return sp.sqnorms_cpu(sp.param) if sp.sz else sp.param.new_zeros(0)

    # -- state ---------------------------------------------------------------
    def moments(self):
        """(exp_avg, exp_avg_sq) over the flat space: the fp32 buffers
        themselves, or the values that the 8-bit ones stand for, in bfloat16,
        which holds them exactly."""
        if self.state_bits == 32:
            return self.exp_avg, self.exp_avg_sq
        if self.codes.is_cuda:
            m, v = native().adamw_moments(self.codes, self.exponents)
            return m, v
        m, v = _unpack(self.codes, self.exponents)
        return m.to(torch.bfloat16), v.to(torch.bfloat16)

    def _state(self) -> dict:
        if self.state_bits == 32:
            return {"exp_avg": self.exp_avg, "exp_avg_sq": self.exp_avg_sq}
        return {"codes": self.codes, "exponents": self.exponents}

    def state_dict(self) -> dict:
        """On the CPU; with the seed and the step it resumes to the bit."""
        return {"kind": "adamw", "state_bits": self.state_bits,
                "steps": self.steps, "seed": self.seed,
                "betas": list(self.betas), "powers": self._powers.tolist(),
                "corrections": self._coef[1:].tolist(),
                **{k: t.detach().cpu().clone()
                   for k, t in self._state().items()}}

    def load_state_dict(self, d: dict) -> None:
        if d.get("kind") != "adamw" or d["state_bits"] != self.state_bits:
            raise ValueError(
                f"the state is of {d.get('kind')!r} with "
                f"{d.get('state_bits')} bits, not of 'adamw' with "
                f"{self.state_bits}")
        mine = self._state()
        for k, t in mine.items():
            if d[k].shape != t.shape or d[k].dtype != t.dtype:
                raise ValueError(f"{k} does not fit this model")
        for k, t in mine.items():
            t.copy_(d[k])
        self.seed = int(d["seed"])
        self._step.fill_(int(d["steps"]))
        self._set_corrections(int(d["steps"]) + 1)
        if list(d["betas"]) == list(self.betas):
            # as the kernel's products left them, which ** only comes close to
            self._powers.copy_(torch.tensor(d["powers"], dtype=torch.float64))
            self._coef[1:].copy_(torch.tensor(d["corrections"]))
