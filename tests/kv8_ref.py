"""Plain 64-bit forms of the rotary, 8-bit-cache, attention and log-probability ops, on the CPU,
and a small paged cache to run them against (used by test_op_kv8.py and test_op_logprobs.py)."""
from __future__ import annotations

import numpy as np
import torch

PAGE = 16
TYPES = [torch.float32, torch.float16, torch.bfloat16]
INT8, E4M3 = 0, 1
CODE_MAX = (127.0, 448.0)


def type_id(t) -> int:
    return TYPES.index(t)


def half_step(t) -> float:
    """Largest relative error of one rounding to t."""
    return torch.finfo(t).eps / 2


def rope64(x, pos, freq, inter, mag=1.0, inverse=False):
    """x [rows][heads][dim] float64, pos [rows], freq [rot / 2] float64."""
    rot = 2 * len(freq)
    t = np.asarray(pos, np.float64)[:, None] * np.asarray(freq)[None]
    if inverse:
        t = -t
    c, s = np.cos(t)[:, None] * mag, np.sin(t)[:, None] * mag
    y = x.copy()
    ia = np.arange(0, rot, 2) if inter else np.arange(rot // 2)
    ib = ia + 1 if inter else ia + rot // 2
    y[..., ia] = x[..., ia] * c - x[..., ib] * s
    y[..., ib] = x[..., ib] * c + x[..., ia] * s
    return y


def freqs(rot, base=10000.0):
    return base ** (-2.0 * np.arange(rot // 2) / rot)


def steps_of(freq):
    """Whole 2^-64 turns a position, by exact integer arithmetic on the doubles."""
    from fractions import Fraction
    two_pi = 2 * Fraction(314159265358979323846264338327950288419716939937510, 10**50)
    return np.array([int(round(Fraction(float(f)) / two_pi * 2**64)) % 2**64 for f in freq], np.uint64)


def quantise32(x, fmt):
    """x [..., dim] float32 tensor -> (codes uint8, scales float32): the definition, in fp32."""
    x = x.float()
    top = x.abs().amax(-1)
    scale = top / CODE_MAX[fmt]
    bad = ~torch.isfinite(x).all(-1)
    zero = (scale < 2.0**-126) | bad
    y = torch.where(zero[..., None], torch.zeros(()), x) / torch.where(zero, torch.ones(()), scale)[..., None]
    codes = y.round().clamp(-127, 127).to(torch.int8) if fmt == INT8 else y.clamp(-448, 448).to(torch.float8_e4m3fn)
    scale = torch.where(bad, torch.full((), float("nan")), torch.where(zero, torch.zeros(()), scale))
    return codes.view(torch.uint8), scale


def values64(codes, fmt):
    return (codes.view(torch.int8) if fmt == INT8 else codes.view(torch.float8_e4m3fn).float()).double()


class Cache:
    """A paged pool on the CPU (torch tensors) whose cells hold garbage until something is put there:
    codes of any byte that the format allows, NaN scales."""

    def __init__(self, fmt, kvh, dim, slots, pages_per_slot, spare=3, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.fmt, self.kvh, self.dim, self.slots, self.pps = fmt, kvh, dim, slots, pages_per_slot
        self.pages = slots * pages_per_slot + spare
        c = torch.randint(0, 256, (self.pages, 2, kvh, PAGE, dim), generator=g).to(torch.uint8)
        if fmt == E4M3:  # NaN codes may lie in cells that nothing was written to
            self.codes = c
        else:
            self.codes = torch.where(c == 128, torch.zeros((), dtype=torch.uint8), c)
        self.scales = torch.full((self.pages, 2, kvh, PAGE), float("nan"))
        self.table = torch.randperm(self.pages, generator=g)[: slots * pages_per_slot].int().view(slots, pages_per_slot)

    def put(self, slot, pos, half, codes, scales):
        page = int(self.table[slot, pos // PAGE])
        self.codes[page, half, :, pos % PAGE] = codes
        self.scales[page, half, :, pos % PAGE] = scales

    def fill(self, slot, n, seed, spread=1.0):
        """Positions 0..n-1 of a slot hold random heads."""
        g = torch.Generator().manual_seed(seed)
        x = torch.randn(n, 2, self.kvh, self.dim, generator=g) * torch.exp(spread * torch.randn(n, 2, self.kvh, 1, generator=g) * 0.3)
        for half in (0, 1):
            codes, scales = quantise32(x[:, half], self.fmt)
            for p in range(n):
                self.put(slot, p, half, codes[p], scales[p])

    def heads(self, slot, n, half):
        """Positions 0..n-1 in 64 bits, [n][kvh][dim]."""
        if n == 0:
            return torch.zeros(0, self.kvh, self.dim, dtype=torch.float64)
        pos = torch.arange(n)
        page = self.table[slot].long()[pos // PAGE]
        return values64(self.codes[page, half, :, pos % PAGE], self.fmt) * self.scales[page, half, :, pos % PAGE].double()[..., None]

    def cuda(self):
        c = Cache.__new__(Cache)
        c.__dict__.update(self.__dict__)
        c.codes, c.scales, c.table = self.codes.cuda(), self.scales.cuda(), self.table.cuda()
        return c

    def struct(self, M):
        return M.KV8Cache(self.codes.data_ptr(), self.scales.data_ptr(), self.table.data_ptr(), self.pages, self.slots,
                          self.pps, self.kvh, self.dim, self.fmt)


def attend64(cache, q, starts, slots, ctx, scale, mask=None):
    """q [rows][heads][dim] float64 -> (out, spread): spread = sum_j p_j |V_j| and the largest |score| sum, which
    the tolerances of an output are made of."""
    rows, qh, dim = q.shape
    group = qh // cache.kvh
    out, mass, top = torch.zeros_like(q), torch.zeros_like(q), torch.zeros(rows, qh, dtype=torch.float64)
    for s in range(len(slots)):
        n = starts[s + 1] - starts[s]
        if n == 0:
            continue
        total = ctx[s] + n
        k, v = cache.heads(slots[s], total, 0), cache.heads(slots[s], total, 1)
        k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
        for i in range(n):
            r = starts[s] + i
            ok = torch.ones(total, dtype=torch.bool)
            for j in range(n):
                ok[ctx[s] + j] = j <= i if mask is None else (j < 32 * mask.shape[1] and bool(int(mask[r, j // 32]) >> (j % 32) & 1))
            if not ok.any():
                continue
            a = torch.einsum("hd,jhd->hj", q[r], k[ok]) * scale
            p = torch.softmax(a, -1)
            out[r] = torch.einsum("hj,jhd->hd", p, v[ok])
            mass[r] = torch.einsum("hj,jhd->hd", p, v[ok].abs())
            top[r] = (torch.einsum("hd,jhd->hj", q[r].abs(), k[ok].abs()) * abs(scale)).amax(-1)
    return out, mass, top


def attend_tolerance(mass, top, out, t):
    """Bound on |out - exact|.  Scores: both fp16 parts of q (2^-21 of |q||k| with their products' truncation),
    three fp32 roundings: 2^-20 of the largest sum |q||k|, which moves a weight by e^d - 1 ~ d, in numerator and
    denominator (2 d).  Weights: ex2.approx 2^-22, two products, the split 2^-21, sums 2^-19 in all; bf16 outputs
    round the weights to fp16 (2^-11).  Then the rounding to the output's type: half a step, which below the
    smallest normal number is that number's (fp16: 2^-25)."""
    w = 2.0**-19 + (2.0**-11 if t == torch.bfloat16 else 0.0)
    return mass * (2 * top[..., None] * 2.0**-20 + w) + out.abs().clamp(min=torch.finfo(t).tiny) * half_step(t)
