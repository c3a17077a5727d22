"""CPU statement of the 4-bit paged cache and of the operators over it, in 64 bits.

The format is stated in ``include/b200kv_kv4.h``; here it is written element by element (byte and nibble
addresses), without any packing trick, so that it can hold the kernels to it.  Test infrastructure only.
"""

from __future__ import annotations

import math
from typing import Optional

import torch

D, PS, GROUP, BLOCK = 128, 16, 32, 1152
MAX_SCALE = 9352.0


def _addresses():
    t = torch.arange(PS).view(-1, 1)
    d = torch.arange(D).view(1, -1)
    g, j, n = d // 32, d % 32 // 8, d % 8
    nibble = n // 2 + 4 * (n % 2)
    byte = 64 * t + 16 * (j ^ ((t // 2) % 4)) + 4 * g + nibble // 2
    return byte, (nibble % 2).expand(PS, D)


BYTE, HIGH = _addresses()          # [16, 128]: byte of each element, and whether it is the high nibble


def quantise(x: torch.Tensor):
    """fp16 ``[..., 128]`` -> (code - 8 in float64 ``[..., 128]``, fp16 scales ``[..., 4]``)."""
    assert x.dtype == torch.float16 and x.shape[-1] == D
    g = x.double().unflatten(-1, (D // GROUP, GROUP))
    amax = g.abs().amax(-1)
    scale = (amax / 7).to(torch.float16).clamp(max=MAX_SCALE)
    s = scale.double().unsqueeze(-1)
    c = torch.where(s > 0, torch.floor(g / s + 0.5), torch.zeros_like(g)).clamp(-8, 7)
    bad = ~torch.isfinite(amax)
    c = torch.where(bad.unsqueeze(-1), torch.zeros_like(c), c)
    scale = torch.where(bad, torch.full_like(scale, float("nan")), scale)
    return c.flatten(-2), scale


def append(rows: torch.Tensor, slots: torch.Tensor, pool: torch.Tensor) -> None:
    """Quantise ``rows`` fp16 [n, 2*kv_heads, 128] into ``pool`` uint8 [pages, 2*kv_heads, 1152], token by token."""
    codes, scales = quantise(rows)
    codes = (codes + 8).to(torch.uint8)
    scale_bytes = scales.contiguous().view(torch.uint8)                  # [n, rows, 8]
    for i, slot in enumerate(slots.tolist()):
        if not 0 <= slot < pool.shape[0] * PS:
            continue
        page, t = divmod(slot, PS)
        for high in (0, 1):
            pick = HIGH[t] == high
            at = BYTE[t][pick]
            old = pool[page][:, at]
            new = codes[i][:, pick]
            pool[page][:, at] = (old & 0x0F) | (new << 4) if high else (old & 0xF0) | new
        pool[page][:, 1024 + 8 * t: 1032 + 8 * t] = scale_bytes[i]


def rows_of(pool: torch.Tensor, slots: torch.Tensor) -> torch.Tensor:
    """What the slots stand for, unrounded: float64 [n, 2*kv_heads, 128]."""
    page, t = slots.long() // PS, slots.long() % PS
    blocks = pool[page]                                                  # [n, rows, 1152]
    n, r = blocks.shape[:2]
    raw = torch.gather(blocks, 2, BYTE[t].unsqueeze(1).expand(n, r, D))
    code = torch.where(HIGH[t].unsqueeze(1) == 1, raw >> 4, raw & 15).double() - 8
    sb = blocks[:, :, 1024:].contiguous().view(torch.float16).unflatten(-1, (PS, 4))
    scale = sb[torch.arange(n), :, t].double()
    return code * scale.repeat_interleave(GROUP, dim=-1)


def norm_rope(x: torch.Tensor, weight: Optional[torch.Tensor], eps: float, cos: torch.Tensor, sin: torch.Tensor,
              round_last: bool = True) -> torch.Tensor:
    """Head rows fp16 [n, heads, 128] normalised (two roundings to fp16, as the fp16 path defines it) and
    rotated, statistics in 64 bits; the last rounding to fp16 is optional."""
    y = x.double()
    if weight is not None:
        y = (y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps)).to(torch.float16).double()
        y = (y * weight.double()).to(torch.float16).double()
    h = D // 2
    c, s = cos[:, None, :h].double(), sin[:, None, :h].double()
    a, b = y[..., :h], y[..., h:]
    out = torch.cat((a * c - b * s, b * c + a * s), -1)
    return out.to(torch.float16) if round_last else out


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, first_pos: int, scale: float):
    """Query rows fp16 [m, heads, 128] at positions first_pos.. over keys float64 [n, kv_heads, 128]: row i sees
    keys 0 .. first_pos + i.  Returns (output, sum of p |v|, largest |scale q k| sum of a seen key), each
    float64; masked keys take no part whatever they hold; no visible key gives zeros."""
    m, heads, _ = q.shape
    n, kvh, _ = k.shape
    group = heads // kvh
    out = torch.zeros(m, heads, D, dtype=torch.float64)
    mag = torch.zeros(m, heads, D, dtype=torch.float64)
    dot = torch.zeros(m, heads, 1, dtype=torch.float64)
    for i in range(m):
        seen = min(n, first_pos + i + 1)
        if seen <= 0:
            continue
        for h in range(heads):
            kk, vv = k[:seen, h // group], v[:seen, h // group]
            qq = q[i, h].double()
            p = torch.softmax((kk @ qq) * scale, 0)
            out[i, h] = p @ vv
            mag[i, h] = p @ vv.abs()
            dot[i, h, 0] = ((kk.abs() @ qq.abs()) * abs(scale)).nan_to_num(0.0).max()
    return out, mag, dot
