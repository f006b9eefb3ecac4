"""The 8-bit paged cache restated in 64 bits with tensor operations on the host, page by page and row by row."""
import math

import torch

F8 = torch.float8_e4m3fn
LARGEST = 448.0 * 2.0 ** 50


def scale_for(amax: float) -> float:
    """The smallest 2^e, e >= -64, with amax <= 448 * 2^e."""
    e = -64
    if amax > 0:
        m, x = math.frexp(amax)                     # amax = m 2^x, 448 = 0.875 * 2^9
        e = max(e, x - 9 if m <= 0.875 else x - 8)
    return 2.0 ** e


def to_e4m3(x: torch.Tensor) -> torch.Tensor:
    """float64 rounded once to e4m3, ties to even, and back (|x| <= 448; NaN stays).  A float64 that lies on no tie of
    float32 keeps its side of every e4m3 tie when it goes through float32 first: ties of e4m3 are float32 numbers."""
    return x.to(torch.float32).to(F8).to(torch.float64)


def rotated(x: torch.Tensor, gain, eps, freq, factor, rotary_dim, adjacent, pos) -> torch.Tensor:
    """Norm and rotation of rows [n, heads, hd] in 64 bits (``freq`` None: no rotation, ``gain`` None: no norm)."""
    x = x.double()
    if gain is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * gain.double()
    if freq is None or rotary_dim == 0:
        return x
    half = rotary_dim // 2
    ang = pos.double()[:, None] * freq.double()[None, :]
    c, s = (torch.cos(ang) * factor)[:, None, :], (torch.sin(ang) * factor)[:, None, :]
    out = x.clone()
    i0 = torch.arange(half) * 2 if adjacent else torch.arange(half)
    i1 = i0 + 1 if adjacent else i0 + half
    a, b = x[..., i0], x[..., i1]
    out[..., i0], out[..., i1] = a * c - b * s, a * s + b * c
    return out


class PlainPages:
    """Numbers (float64) [n_pages, kv_heads, page, hd] and scales (float64) as the cache holds them; ``ideal`` are the values
    before the last rounding, ``slack`` what earlier roundings may have left (a page whose scale grew)."""

    def __init__(self, numbers: torch.Tensor, scales: torch.Tensor):
        self.n = numbers.detach().cpu().to(torch.float32).double()
        self.s = scales.detach().cpu().double()
        self.ideal = self.n * self.s.abs()[:, :, None, None]
        self.slack = torch.zeros_like(self.n)
        self.written = torch.zeros(self.n.shape[:1] + self.n.shape[2:3], dtype=torch.bool)

    def store(self, page: int, first: int, rows: torch.Tensor) -> None:
        """``rows`` [m, kv_heads, hd] at rows first.. of a page."""
        m = rows.shape[0]
        for h in range(self.n.shape[1]):
            x = rows[:, h].double()
            fine = x.abs() <= LARGEST
            amax = float(x[fine].abs().max()) if bool(fine.any()) else 0.0
            was = float(self.s[page, h]) if first else 0.0
            now = max(abs(was), scale_for(amax))
            if first and abs(was) < now:
                old = self.n[page, h, :first] * (abs(was) / now)
                # rounded again: exact unless the number falls below 2^-6, there off by up to 2^-10
                self.slack[page, h, :first] += 2.0 ** -10 * now
                self.n[page, h, :first] = to_e4m3(old)
            x = torch.where(fine, x, torch.full_like(x, math.nan))
            self.n[page, h, first:first + m] = to_e4m3(x / now)
            self.ideal[page, h, first:first + m] = x
            self.slack[page, h, first:first + m] = 0
            flagged = not bool(fine.all()) or (first and math.copysign(1, was) < 0)
            self.s[page, h] = -now if flagged else now
        self.written[page, first:first + m] = True


def attention(q, keys, values, scale, window, pos, page_scales=None):
    """softmax(scale q K^T) V of rows q [n, group, hd] at positions pos [n] over keys, values [L, hd] (position j in row j), all
    64-bit; also sum p |v| per entry, the largest sum |q||k| scale of a visible key per row and, with ``page_scales`` [L] (of
    the values), the number of visible keys times the largest p * page scale per row."""
    j = torch.arange(keys.shape[0])
    most = torch.zeros(q.shape, dtype=torch.float64)
    out, weight, spread = (torch.zeros(q.shape, dtype=torch.float64) for _ in range(3))
    for i in range(q.shape[0]):
        seen = (j <= pos[i]) & ((j > pos[i] - window) if window else (j >= 0))
        k, v = keys[seen], values[seen]
        s = (q[i] @ k.T) * scale
        p = torch.softmax(s, -1)
        out[i] = p @ v
        weight[i] = p @ v.abs()
        spread[i] = ((q[i].abs() @ k.abs().T) * scale).amax(-1, keepdim=True)
        if page_scales is not None:
            most[i] = (p.nan_to_num() * page_scales[seen]).amax(-1, keepdim=True) * int(seen.sum())
    return (out, weight, spread) if page_scales is None else (out, weight, spread, most)
