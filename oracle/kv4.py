"""CPU restatement of the 4-bit paged K/V cache (fish_speech_amd/kv4.py, include/fishmi.h) in 64 bits: the number format,
the append's head norm and rotation, attention over the stored values.  The reference has no such cache; its norm,
rotation and attention are fish_speech/models/text2semantic/llama.py:862-864, 1004-1038, 928-934."""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

PAGE = 64
GRID = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)


def quantise(y: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(..., D) -> codes (..., D) 0..15 and scale bytes (..., D / 32): nearest representable value, ties to even codes."""
    b = y.double().unflatten(-1, (-1, 32))
    finite = torch.isfinite(b).all(-1)
    b = torch.where(finite[..., None], b, 0.0)
    top = b.abs().amax(-1)
    e = torch.full(top.shape, -100, dtype=torch.int64)
    for cand in range(-100, 125):                      # the smallest power with max <= 7 * 2^e, by trying them
        e = torch.where(top > 7 * 2.0 ** cand, cand + 1, e)
    a = b.abs() / torch.ldexp(torch.ones_like(top), e)[..., None]
    dist = (a[..., None] - GRID).abs()
    best = dist.amin(-1, keepdim=True)
    near = dist == best                                # one candidate, or two on a border: take the even one
    idx = torch.arange(8)
    first = torch.where(near, idx, 99).amin(-1)
    last = torch.where(near, idx, -1).amax(-1)
    code = torch.where(first % 2 == 0, first, last)
    code = torch.where(a > 6, 7, code)
    code = code + 8 * torch.signbit(b).long()
    code = torch.where(finite[..., None], code, 0)
    return code.to(torch.uint8).flatten(-2), torch.where(finite, e + 127, 255).to(torch.uint8)


def values(code: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    v = GRID[(code & 7).long()] * torch.where(code >= 8, -1.0, 1.0)
    s = torch.where(scale == 255, math.nan, torch.ldexp(torch.ones(scale.shape, dtype=torch.float64), scale.long() - 127))
    return (v.unflatten(-1, (-1, 32)) * s[..., None]).flatten(-2)


def stored(y: torch.Tensor) -> torch.Tensor:
    """What the cache gives back for y."""
    return values(*quantise(y))


def pack_block(code: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """One page block (64, D) -> its bytes: codes with the even dim in the low nibble, then the scales."""
    return torch.cat([(code[:, 0::2] | (code[:, 1::2] << 4)).flatten(), scale.flatten()])


def head_norm(x: torch.Tensor, w: Optional[torch.Tensor], eps: float) -> torch.Tensor:
    if w is None:
        return x
    rstd = (1.0 / (x.double().square().mean(-1, keepdim=True) + eps).sqrt()).float()
    return (x.float() * rstd * w.float()).to(torch.bfloat16)


def rotate(y: torch.Tensor, cs: Optional[torch.Tensor], half: bool) -> torch.Tensor:
    """y (rows, heads, D) bf16, cs (rows, rot / 2, 2) bf16.  The products of bf16 factors are exact in fp32."""
    if cs is None:
        return y
    h = cs.shape[1]
    out = y.clone()
    for i in range(h):
        a, b = (i, i + h) if half else (2 * i, 2 * i + 1)
        c, s = cs[:, None, i, 0].float(), cs[:, None, i, 1].float()
        x0, x1 = y[..., a].float(), y[..., b].float()
        out[..., a] = (x0 * c - x1 * s).to(torch.bfloat16)
        out[..., b] = (x1 * c + x0 * s).to(torch.bfloat16)
    return out


def attend(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, past: int, scale: float,
           seen: Optional[torch.Tensor] = None, weight: float = 2.0 ** -16) -> Tuple[torch.Tensor, torch.Tensor]:
    """One sequence: q (n, H, D) at positions past .. past + n - 1, k / v (keys, KVH, D) float64; `seen` (keys,) = keys that
    exist at all; `weight` = relative rounding of a softmax weight (bf16 high + low part 2^-16, fp16 2^-11).  -> output float64
    and, per output, a bound of the arithmetic's error before the last rounding."""
    n, H, D = q.shape
    G = H // k.shape[1]
    out = torch.zeros(n, H, D, dtype=torch.float64)
    bound = torch.zeros(n, H, D, dtype=torch.float64)
    for i in range(n):
        idx = torch.arange(max(0, min(past + i + 1, k.shape[0])))
        if seen is not None:
            idx = idx[seen[idx]]
        if idx.numel() == 0:
            continue
        for h in range(H):
            kk, vv, qq = k[idx, h // G], v[idx, h // G], q[i, h].double()
            s = kk @ qq * scale
            p = torch.exp(s - s.max())
            out[i, h] = p @ vv / p.sum()
            # fp32: a score is off by (D + 4) roundings of its absolute products, which moves every weight by that much;
            # weights carry their rounding and the fp32 exponential's 2^-16; sums of len(idx) terms add a rounding each, and a
            # weight below fp16's smallest step (2^-25 rounds to 0) loses no more than that
            ds = (D + 4) * 2.0 ** -24 * float((kk.abs() @ qq.abs()).max()) * abs(scale)
            bound[i, h] = (4 * ds + weight + 2.0 ** -16 + idx.numel() * 2.0 ** -24) * float(vv.abs().max())
    return out, bound
