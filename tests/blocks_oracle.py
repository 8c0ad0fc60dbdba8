"""The 8-bit block cache by its definition, in 64 bits on the CPU."""
from __future__ import annotations

import math

import torch

TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
_E4M3 = torch.arange(0, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()


def nearest(x: torch.Tensor, store: torch.dtype) -> torch.Tensor:
    """Values of the 8-bit format nearest to x (float64), ties to the even code."""
    if store is torch.int8:
        return torch.round(x).clamp(-127, 127)
    a = x.abs().clamp(max=448.0)
    hi = torch.searchsorted(_E4M3, a).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    up, down = _E4M3[hi] - a, a - _E4M3[lo]
    i = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    return torch.copysign(_E4M3[i], x)


def f32_quotient(top: torch.Tensor, by: float) -> torch.Tensor:
    """fp32(top / by); below the smallest normal number it is 0."""
    s = (top.double() / by).float()
    return torch.where(s < 2.0 ** -126, torch.zeros_like(s), s)


class Cache:
    """Pages of one side: values of the codes (float64) and scales (float32)."""

    def __init__(self, codes: torch.Tensor, scale: torch.Tensor):
        self.store = codes.dtype
        self.codes = codes.cpu().float().double() if codes.dtype != torch.int8 else codes.cpu().double()
        self.scale = scale.cpu().clone()
        self.N = codes.shape[2]

    def append(self, table, end: int, x: torch.Tensor) -> None:
        """x [n, Hkv, dh] at positions end - n .. end - 1 of the sequence whose pages are `table`."""
        n, N = x.shape[0], self.N
        pos = end - n
        x = x.detach().cpu().float()
        while pos < end:
            page, lo = int(table[pos // N]), pos % N
            take = min(N - lo, end - pos)
            part = x[n - (end - pos):][:take].transpose(0, 1).double()     # [Hkv, take, dh]
            for h in range(x.shape[1]):
                top = part[h].abs().max().float() if not part[h].isnan().any() else torch.tensor(math.nan)
                s = f32_quotient(top, TOP[self.store]) if math.isfinite(top) else top
                old = self.scale[page, h].clone()
                if lo:
                    grown = bool(s.isnan() and not old.isnan()) or bool(s > old)
                    if not grown:
                        s = old
                    elif math.isfinite(s):
                        self.codes[page, h, :lo] = nearest(self.codes[page, h, :lo] * old.double() / s.double(), self.store)
                    else:
                        self.codes[page, h, :lo] = 0
                self.scale[page, h] = s
                dead = not math.isfinite(s) or s == 0
                self.codes[page, h, lo:lo + take] = 0 if dead else nearest(part[h] / s.double(), self.store)
            pos += take

    def rows(self, table, lo: int, hi: int) -> torch.Tensor:
        """float64 [hi - lo, Hkv, dh]"""
        t = torch.arange(lo, hi)
        page = torch.as_tensor([int(table[p // self.N]) for p in range(lo, hi)], dtype=torch.long)
        return self.codes[page, :, t % self.N] * self.scale[page].double()[..., None]


def attend(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, key0: int, pos, scale: float):
    """q [n, Hq, dh] at positions `pos`; k, v float64 [keys, Hkv, dh] at positions key0 ...  Returns out [n, Hq, dh], (max, sum)
    [n, Hq], the bound [n, Hq, dh] of what fp32 kernels may be off, sum p |v| [n, Hq, dh] and the bound [n, Hq] of a logit."""
    n, Hq, dh = q.shape
    group = Hq // k.shape[1]
    q = q.detach().cpu().double()
    out, off = torch.zeros(n, Hq, dh, dtype=torch.float64), torch.zeros(n, Hq, dh, dtype=torch.float64)
    sizes, errs = torch.zeros(n, Hq, dh, dtype=torch.float64), torch.zeros(n, Hq, dtype=torch.float64)
    top, total = torch.full((n, Hq), -math.inf, dtype=torch.float64), torch.zeros(n, Hq, dtype=torch.float64)
    at = torch.arange(key0, key0 + k.shape[0])
    for h in range(Hq):
        kh, vh = k[:, h // group], v[:, h // group]
        x = q[:, h] @ kh.T * scale
        # Bound of a logit: query elements and their scaling 2^-22, dh products summed in fp32 with cut-off additions (2^-23
        # each), factors of the scales 3 * 2^-24; the exponential adds 2^-21 (two ulp, and fp32 arguments).
        err = (q[:, h].abs() @ kh.abs().T * scale) * (2.0 ** -22 + dh * 2.0 ** -23 + 3 * 2.0 ** -24) + x.abs() * 2.0 ** -22 + 2.0 ** -21
        seen = at[None, :] <= torch.as_tensor(pos)[:, None]
        x = x.masked_fill(~seen, -math.inf)
        if k.shape[0] == 0:
            continue
        m = x.max(1).values
        some = m > -math.inf
        w = torch.exp(x - torch.where(some, m, torch.zeros_like(m))[:, None])
        s = w.sum(1)
        p = w / torch.where(s == 0, torch.ones_like(s), s)[:, None]
        out[:, h] = p @ vh
        top[:, h], total[:, h] = m, s
        # weights are off by err (relative) in the sum and the quotient; sums of 16 keys at a time in fp32
        size = p @ vh.abs()
        sizes[:, h], errs[:, h] = size, err.masked_fill(~seen, 0).amax(1)
        off[:, h] = (2 * errs[:, h, None] + (k.shape[0] / 16 + 64) * 2.0 ** -23) * size
    return out, top, total, off, sizes, errs
