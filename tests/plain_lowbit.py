"""The 4-bit cache's and the 8-bit products' formulas in plain float64, one function per rule, without the package's code."""
from __future__ import annotations

import math

import torch

F = torch.float64


def rounded4(x: torch.Tensor) -> torch.Tensor:
    """x [..., multiple of 32] as the 4-bit format holds it: per 32 features mn = bfloat16(min), sc = bfloat16((max - mn) / 15), code =
    rint((x - mn) * (1 / sc)) in 0 .. 15, float32 products as the format has them; a group that is not finite is NaN."""
    y = x.to(torch.float32).reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    lo, hi = y.amin(-1, keepdim=True), y.amax(-1, keepdim=True)
    mn = lo.bfloat16().float()
    sc = ((hi - mn).clamp(min=0) / torch.full_like(mn, 15.0)).bfloat16().float()
    inv = torch.where(sc > 1e-30, torch.ones_like(sc) / sc, torch.zeros_like(sc))
    code = torch.round((y - mn) * inv).clamp(0, 15)
    out = mn.to(F) + sc.to(F) * code.to(F)
    bad = ~torch.isfinite(y).all(-1, keepdim=True) | ~torch.isfinite(sc) | ~torch.isfinite(mn)
    return torch.where(bad, torch.full_like(out, math.nan), out).reshape(x.shape)


def step4(x: torch.Tensor) -> torch.Tensor:
    """What one code is worth in each feature's group."""
    y = x.to(F).reshape(*x.shape[:-1], -1, 32)
    return ((y.amax(-1, keepdim=True) - y.amin(-1, keepdim=True)) / 15).expand_as(y).reshape(x.shape)


def page_values(page: torch.Tensor, d: int):
    """Keys and values [64, d] of one page of one head (bytes), word by word as the format is written down."""
    b = page.cpu().to(torch.int64)
    word = lambda at: int(b[at] | b[at + 1] << 8 | b[at + 2] << 16 | b[at + 3] << 24)  # noqa: E731
    bf16 = lambda bits: float(torch.tensor([bits << 16], dtype=torch.int64).to(torch.int32).view(torch.float32)) if bits < 0x8000 else \
        float(torch.tensor([(bits << 16) - (1 << 32)], dtype=torch.int64).to(torch.int32).view(torch.float32))  # noqa: E731
    per, groups = 4096 // d, d // 32
    out = torch.zeros(2, 64, d, dtype=F)
    for slot in range(64):
        base, tok = slot // per * 5120, slot % per
        u = tok % 16
        for f in range(d):
            g, e = f // 32, f % 32
            kw = word(base + tok * (d // 2) + (e // 8 * groups + g) * 4)
            kn = kw >> 4 * ((e % 8) // 2 + 4 * (e % 2)) & 15
            vw = word(base + 2560 + ((((tok // 16) * (d // 64) + f // 64) * 8 + e // 4) * 4 + u % 8 // 2) * 16 + (u // 8 * 2 + u % 2) * 4)
            vn = vw >> 4 * (e % 4 + 4 * (f % 64 // 32)) & 15
            for i, (n, at) in enumerate(((kn, 2048), (vn, 4608))):
                w = word(base + at + (tok * groups + g) * 4)
                out[i, slot, f] = bf16(w & 0xFFFF) + bf16(w >> 16) * n
    return out[0], out[1]


def rotated(x: torch.Tensor, pos: torch.Tensor, theta: float = 10000.0) -> torch.Tensor:
    """x [T, heads, d] with pairs f, f + d / 2 turned by the angles of its position."""
    h = x.shape[-1] // 2
    a = pos.to(F)[:, None, None] * theta ** (-torch.arange(h, dtype=F, device=x.device) / h)
    u, v = x.to(F)[..., :h], x.to(F)[..., h:]
    return torch.cat([u * a.cos() - v * a.sin(), v * a.cos() + u * a.sin()], -1)


def attend(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, pos0: int, scale: float, window: int = 0, hidden_keys=()) -> torch.Tensor:
    """q [n, heads, d] at positions pos0 .., k and v [keys, kv heads, d]; a query that sees nothing gets zeros."""
    n, heads, d = q.shape
    g = heads // k.shape[1]
    out = torch.zeros(n, heads, v.shape[-1], dtype=F)
    for i in range(n):
        p = pos0 + i
        seen = [j for j in range(max(0, p - window + 1) if window else 0, min(p + 1, k.shape[0])) if j not in hidden_keys]
        if not seen:
            continue
        for h in range(heads):
            s = (k[seen, h // g].to(F) @ q[i, h].to(F)) * scale
            out[i, h] = torch.softmax(s, 0) @ v[seen, h // g].to(F)
    return out


def e4m3(x: torch.Tensor) -> torch.Tensor:
    """The nearest number of four exponent and three fraction bits, ties to even."""
    x = x.to(F)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return ((x / step).round() * step).clamp(-448, 448)


def rounded8(x: torch.Tensor):
    """Codes and scales of x [M, K], per row and 128 features, by the format's float32 products."""
    m, k = x.shape
    codes, scales = [], []
    for k0 in range(0, k, 128):
        y = x[:, k0:k0 + 128].float()
        a = y.abs().amax(1, keepdim=True).clamp(min=1e-30)
        codes.append(e4m3(y * (torch.full_like(a, 448.0) / a)))
        scales.append(a / torch.full_like(a, 448.0))
    return torch.cat(codes, 1), torch.cat(scales, 1).to(F)


def product8(x, w_codes, w_scales, bias=None, gated=False):
    """The product in float64 of x rounded per row and 128 features and w as its codes and scales stand."""
    cx, sx = rounded8(x)
    m, k = x.shape
    n = w_codes.shape[0]
    y = torch.zeros(m, n, dtype=F, device=x.device)
    for b, k0 in enumerate(range(0, k, 128)):
        part = cx[:, k0:k0 + 128] @ w_codes[:, k0:k0 + 128].float().to(F).T
        y += part * sx[:, b:b + 1] * w_scales[:, b].to(F).repeat_interleave(128)[:n]
    if bias is not None:
        y += bias.to(F)
    if gated:
        z = y.view(m, n // 16, 2, 8)
        y = (z[:, :, 0] * torch.sigmoid(z[:, :, 0]) * z[:, :, 1]).reshape(m, n // 2)
    return y
