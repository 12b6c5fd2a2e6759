"""Attention over shared and over chosen pages, bounds of pages and the choice by them, in float64 on the CPU, straight from the definitions."""
import math

import torch

F = torch.float64
PAGE = 64


class Paged:
    """Rows of ``(context, new)`` tokens in a paged cache on the CPU; ``share`` names, per row, its group and the pages it shares (or None).  Places that hold no
    row's token are NaN, pages are scrambled, and a few belong to nobody."""

    def __init__(self, rows, heads, kv_heads, d, share=None, seed=0, k_scale=1.0):
        gen = torch.Generator().manual_seed(seed)
        self.rows, self.h, self.g, self.d = rows, heads, kv_heads, d
        share = share or [None] * len(rows)
        common = {}
        order = None
        need = [-(-(c + n) // PAGE) for c, n in rows]
        sizes = {s[0]: s[1] for s in share if s}
        total = sum(sizes.values()) + sum(n - (s[1] if s else 0) for n, s in zip(need, share)) + 3
        order = torch.randperm(total, generator=gen).tolist()
        for name, n in sizes.items():
            common[name] = [order.pop() for _ in range(n)]
        width = max(need + [1])
        self.table = torch.full((len(rows), width), -1, dtype=torch.int32)
        for r, (n, s) in enumerate(zip(need, share)):
            mine = list(common[s[0]]) if s else []
            mine += [order.pop() for _ in range(n - len(mine))]
            self.table[r, :n] = torch.tensor(mine[:n], dtype=torch.int32)
        self.k = torch.full((total, kv_heads, PAGE, d), math.nan, dtype=torch.bfloat16)
        self.v = self.k.clone()
        for r, (c, n) in enumerate(rows):
            for p in range(need[r]):
                filled = min(PAGE, c + n - p * PAGE)
                page = int(self.table[r, p])
                if self.k[page, 0, 0, 0].isnan():                      # (shared pages once)
                    subject = 0.7 * torch.randn(kv_heads, 1, d, generator=gen)
                    self.k[page, :, :filled] = (k_scale * (torch.randn(kv_heads, filled, d, generator=gen) + subject)).bfloat16()
                    self.v[page, :, :filled] = torch.randn(kv_heads, filled, d, generator=gen).bfloat16()
        new = [n for _, n in rows]
        self.start = [sum(new[:i]) for i in range(len(new) + 1)]
        self.pos0 = [c for c, _ in rows]
        self.q = torch.randn(sum(new), heads * d, generator=gen).bfloat16()
        self.tok_pos = [c + i for c, n in rows for i in range(n)]
        self.tok_seq = [r for r, (_, n) in enumerate(rows) for _ in range(n)]
        self.max_new = max(new + [0])
        groups = []
        for r, s in enumerate(share):
            if s and groups and groups[-1][3] == s[0]:
                groups[-1][1] += 1
            elif s:
                groups.append([r, 1, s[1], s[0]])
        self.groups = [g[:3] for g in groups]

    def keys(self, row, upto):
        """Keys and values [kv heads, upto, d] in float64 of a row's first positions, and which of them are there (pages may be missing)."""
        n = -(-upto // PAGE)
        pages = [int(self.table[row, p]) if p < self.table.shape[1] else -1 for p in range(n)]
        pick = torch.tensor([max(p, 0) for p in pages], dtype=torch.long)
        there = torch.tensor([p >= 0 for p in pages], dtype=torch.bool).repeat_interleave(PAGE)[:upto]
        f = lambda x: x[pick].transpose(0, 1).reshape(self.g, n * PAGE, self.d)[:, :upto].to(F)  # noqa: E731
        return f(self.k), f(self.v), there


def attend(q, k, v, there, scale):
    """q [heads, d] of one kv head, keys and values [n, d]: the output, and sum of w |v| (which roundings of the weights scale with)."""
    if not bool(there.any()):
        z = torch.zeros(q.shape[0], v.shape[-1], dtype=F)
        return z, z
    k, v = k[there], v[there]
    w = torch.softmax((q.to(F) @ k.T) * scale, dim=-1)
    return w @ v, w @ v.abs()


def shared(case, scale):
    """[T, heads * d] of all tokens, and the weights' scale."""
    r = case.h // case.g
    out, size = torch.zeros(len(case.tok_pos), case.h, case.d, dtype=F), torch.zeros(len(case.tok_pos), case.h, case.d, dtype=F)
    for t, (pos, row) in enumerate(zip(case.tok_pos, case.tok_seq)):
        if pos < 0:
            continue
        k, v, there = case.keys(row, pos + 1)
        q = case.q[t].view(case.g, r, case.d)
        for g in range(case.g):
            out[t, g * r:(g + 1) * r], size[t, g * r:(g + 1) * r] = attend(q[g], k[g], v[g], there, scale)
    return out.flatten(1), size.flatten(1)


def listed(case, pages, scale):
    """The same over the pages of ``pages[t][g]``: the first min(count, pos // 64 + 1) entries, in any order, as often as they are listed."""
    r = case.h // case.g
    out, size = torch.zeros(len(case.tok_pos), case.h, case.d, dtype=F), torch.zeros(len(case.tok_pos), case.h, case.d, dtype=F)
    for t, (pos, row) in enumerate(zip(case.tok_pos, case.tok_seq)):
        if pos < 0:
            continue
        k, v, there = case.keys(row, pos + 1)
        q = case.q[t].view(case.g, r, case.d)
        for g in range(case.g):
            at = []
            for p in pages[t][g][:pos // PAGE + 1]:
                if 0 <= p <= pos // PAGE:
                    at += [i for i in range(p * PAGE, min((p + 1) * PAGE, pos + 1)) if bool(there[i])]
            at = torch.tensor(at, dtype=torch.long)
            out[t, g * r:(g + 1) * r], size[t, g * r:(g + 1) * r] = attend(q[g], k[g][at], v[g][at], torch.ones(len(at), dtype=torch.bool), scale)
    return out.flatten(1), size.flatten(1)


def off(got, want, size):
    """How far bfloat16 results are off, in units of what roundings may do.  Each probability is rounded to bfloat16 (2^-8 of it, so 2^-8 of sum w |v| together) and the
    result once (2^-8 of it).  The scores are float32 sums of at most 128 products and the exponentials good to 2^-21: with |score| up to 2^6 here an
    exponent is off by less than 2^-16, which 2^-12 of sum w |v| covers with the sums in float32."""
    err = (got.to(F).cpu() - want).abs()
    return float((err / (2.0 ** -8 * (want.abs() + size) + 2.0 ** -12 * size + 1e-30)).max())


def rounded(x, like):
    return torch.tensor(x, dtype=F).to(like).to(F)


def bounds(case, row, page, upto):
    """Codes [kv heads, 2, d] and scales [kv heads] of a row's page whose tokens below position ``upto`` are there: float32 steps restated in float64."""
    k = case.k[int(case.table[row, page]), :, :min(PAGE, upto - page * PAGE)].to(F)
    both = torch.stack([k.amin(1), k.amax(1)], dim=1)
    a = both.abs().amax((1, 2)).clamp(min=float(torch.tensor(1e-30)))
    inv = (127.0 / a).float().to(F)
    codes = (both * inv[:, None, None]).float().to(F).round().clamp(-127, 127)
    return codes, (a / 127.0).float()


def choose(case, codes, scales, t, count, first, last):
    """Pages [kv heads][count] for token t; codes and scales by physical page."""
    pos, row, r = case.tok_pos[t], case.tok_seq[t], case.h // case.g
    out = []
    n = pos // PAGE + 1 if pos >= 0 else 0
    for g in range(case.g):
        q = case.q[t].view(case.g, r, case.d)[g].to(F)
        a = q.abs().amax(-1, keepdim=True).clamp(min=float(torch.tensor(1e-30)))
        c = (q * (127.0 / a).float().to(F)).float().to(F).round().clamp(-127, 127)
        order = []
        for p in range(n):
            page = int(case.table[row, p])
            if page < 0:
                continue
            x = codes[page, g].to(F)
            whole = torch.maximum(c * x[0], c * x[1]).sum(-1).float()
            score = (whole * (a[:, 0] / 127.0).float()).max() * scales[page, g]
            rank = 2 if p < first or p >= n - last else 1 if math.isinf(float(scales[page, g])) else 0
            order.append((-rank, -float(score) if rank == 0 else 0.0, p))
        chosen = sorted(p for _, _, p in sorted(order)[:count])
        out.append(chosen + [-1] * (count - len(chosen)))
    return out
