"""The operators of a server whose contexts are long or shared, as cases that can be timed and compared.

The cache is the paged bfloat16 one: ``pool[page][key/value head][64 tokens][d]``, keys and values; a row's tokens lie on the pages that its row of the
block table lists.  Query head h reads key/value head ``h // (heads / kv_heads)``.  Three kinds of work:

``shared``  causal attention of a step's new tokens where the rows of a group have their first pages in common: ``softmax(q K^T * d^-0.5) V``.
``bounds``  a step's keys are in the cache; the pages that they went to get new bounds, the smallest and largest key of every feature in 8 bits:
            ``a = max |k|`` over the page's tokens so far, ``s = a / 127``, ``code = rint(x * (127 / a))`` in float32 (a at least 1e-30).  Output: the bounds
            of those pages as the values they stand for, ``code * s``.
``sparse``  attention of each token over ``count`` pages of its row, chosen for each key/value head: the first ``first`` and the last ``last`` ones and those of the
            highest scores (ties: the lower page; fewer where the row has fewer).  With ``a_h = max |q_h|`` and ``c_h = rint(q_h * (127 / a_h))`` for each query head
            the score of a page is ``max_h(n_h * (a_h / 127)) * s`` in float32, ``n_h = sum_i max(c_hi * low_i, c_hi * high_i)`` over the codes of
            its bounds, a whole number below 2^23.  Outputs: the pages in ascending order (-1 behind them) and the attention over their keys.

``exact`` restates them in float64.
"""
from __future__ import annotations

import math

import torch

own = False          # True: the library's kernels; False: the plain form
F64 = torch.float64
PAGE = 64            # tokens of a page


def listed():
    return [
        # two samples of one short prompt on the smallest model: latency
        dict(name="shared-samples", kind="shared", rows=2, groups=1, loose=0, pre_low=4, pre_high=4, own_low=17, own_high=40, new_low=1, new_high=1,
             heads=16, kv_heads=2, dim=64),
        # a full batch of requests behind one long system prompt, their own parts unequal
        dict(name="shared-system", kind="shared", rows=64, groups=1, loose=0, pre_low=64, pre_high=64, own_low=30, own_high=2000, new_low=1, new_high=1,
             heads=32, kv_heads=8, dim=128),
        # samples of one document, every head with keys of its own
        dict(name="shared-mha", kind="shared", rows=32, groups=1, loose=0, pre_low=130, pre_high=130, own_low=1, own_high=300, new_low=1, new_high=1,
             heads=36, kv_heads=36, dim=64),
        # several documents at once, rows that share nothing among them, drafts of one to four tokens
        dict(name="shared-groups", kind="shared", rows=48, groups=5, loose=7, pre_low=8, pre_high=95, own_low=0, own_high=700, new_low=1, new_high=4,
             heads=24, kv_heads=8, dim=64),
        # a book and sixteen answers, sixteen query heads a key/value head
        dict(name="shared-long", kind="shared", rows=16, groups=1, loose=0, pre_low=2048, pre_high=2048, own_low=1, own_high=500, new_low=1, new_high=1,
             heads=32, kv_heads=2, dim=128),
        # questions that come in behind a document, as prompts
        dict(name="shared-questions", kind="shared", rows=24, groups=1, loose=0, pre_low=94, pre_high=94, own_low=0, own_high=0, new_low=16, new_high=120,
             heads=32, kv_heads=8, dim=128),
        # a decoding step's pages: one token a row
        dict(name="bounds-step", kind="bounds", rows=64, own_low=200, own_high=4000, new_low=1, new_high=1, heads=32, kv_heads=8, dim=128),
        # a long prompt's pages, every head with keys of its own
        dict(name="bounds-prompt", kind="bounds", rows=1, own_low=0, own_high=0, new_low=8192, new_high=8192, heads=36, kv_heads=36, dim=64),
        # one user on the smallest model: latency
        dict(name="sparse-short", kind="sparse", rows=1, own_low=4000, own_high=4000, new_low=1, new_high=1, heads=16, kv_heads=2, dim=64, count=16,
             first=1, last=2),
        # a full batch of unequal contexts
        dict(name="sparse-ragged", kind="sparse", rows=64, own_low=1000, own_high=30000, new_low=1, new_high=1, heads=32, kv_heads=8, dim=128, count=64,
             first=1, last=2),
        # a few long contexts with drafts, every head with keys of its own
        dict(name="sparse-drafts", kind="sparse", rows=6, own_low=9000, own_high=17000, new_low=1, new_high=3, heads=36, kv_heads=36, dim=64, count=48,
             first=1, last=2),
        # one very long context
        dict(name="sparse-long", kind="sparse", rows=1, own_low=131070, own_high=131070, new_low=1, new_high=1, heads=32, kv_heads=8, dim=128, count=256,
             first=2, last=4),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_HEADS = ((16, 2, 64), (36, 36, 64), (32, 8, 128), (32, 2, 128), (8, 8, 128), (24, 8, 64), (7, 1, 128), (12, 12, 128), (20, 4, 64), (32, 1, 128))


def draw(rng):
    kind = rng.choice(["shared", "shared", "shared", "bounds", "sparse", "sparse"])
    most = {k: max(work(c)[k] for c in listed() if c["kind"] == kind) for k in ("bytes", "flops")}
    while True:
        h, g, d = rng.choice(_HEADS)
        rows = _log_int(rng, 1, 64)
        if kind == "shared":
            shape = rng.choice(["step", "step", "few", "prompt"])
            new = 1 if shape == "step" else _log_int(rng, 2, 12) if shape == "few" else _log_int(rng, 13, 300)
            pre, low = _log_int(rng, 1, 2048), _log_int(rng, 1, 3000)
            groups = min(rows, _log_int(rng, 1, 7))
            case = dict(kind=kind, rows=rows, groups=groups, loose=rng.randint(0, rows - groups) if rng.random() < 0.4 else 0,
                        pre_low=max(1, int(pre * rng.uniform(0.1, 1.0))), pre_high=pre, own_low=int(low * rng.uniform(0.0, 1.0)), own_high=low,
                        new_low=max(1, int(new * rng.uniform(0.1, 1.0))), new_high=new, heads=h, kv_heads=g, dim=d)
            keys = pre * PAGE + low + new
            # what the plain form writes out: one score for every pair of a row's longest, and every row's keys and values
            if rows * h * new * keys > 8e8 or rows * g * d * keys > 7e8:
                continue
        elif kind == "bounds":
            new = 1 if rng.random() < 0.5 else _log_int(rng, 2, 8192)
            high = _log_int(rng, 1, 8000)
            case = dict(kind=kind, rows=rows, own_low=int(high * rng.uniform(0.0, 1.0)), own_high=high, new_low=max(1, int(new * rng.uniform(0.2, 1.0))),
                        new_high=new, heads=h, kv_heads=g, dim=d)
        else:
            new = 1 if rng.random() < 0.7 else rng.randint(2, 5)
            high = _log_int(rng, 1, 131072)
            first, last = rng.randint(0, 4), rng.randint(1, 4)
            case = dict(kind=kind, rows=rows, own_low=int(high * rng.uniform(0.0, 1.0)), own_high=high, new_low=1, new_high=new, heads=h, kv_heads=g, dim=d,
                        count=max(first + last, _log_int(rng, 4, 300)), first=first, last=last)
            if rows * new * g * d * case["count"] * PAGE > 4e8 or rows * g * d * high > 1.1e9:
                continue
        w = work(case)
        if all(w[k] <= most[k] for k in most):
            return case


def _spread(i, lo, hi, step):
    return lo + int(round((((i + 1) * step) % 1.0) * (hi - lo)))


def _rows(case):
    """(shared pages, tokens before the step behind them, new tokens, group or -1) of each row: spread over the case's ranges, the same for every seed."""
    n, loose, k = case["rows"], case.get("loose", 0), case.get("groups", 0)
    cuts = [(n - loose) * i // max(k, 1) for i in range(k + 1)]
    for i in range(1, k):                                  # groups of unequal sizes, one row at least
        cuts[i] = max(i, min(cuts[i] + (i * 7) % 5 - 2, n - loose - (k - i)))
    for i in range(1, k + 1):
        cuts[i] = max(cuts[i], cuts[i - 1] + 1)
    out = []
    for i in range(n):
        group = next((j for j in range(k) if cuts[j] <= i < cuts[j + 1]), -1)
        pre = _spread(group, case["pre_low"], case["pre_high"], 0.4142135623730951) if group >= 0 else 0
        out.append((pre, _spread(i, case["own_low"], case["own_high"], 0.6180339887498949), _spread(i, case["new_low"], case["new_high"], 0.7548776662466927), group))
    return out


def _groups(case):
    """(first row, rows, shared pages) of each group."""
    rows = _rows(case)
    out = []
    for j in range(case["groups"]):
        mine = [i for i, r in enumerate(rows) if r[3] == j]
        out.append((mine[0], len(mine), rows[mine[0]][0]))
    return out


def work(case):
    h, g, d, rows = case["heads"], case["kv_heads"], case["dim"], _rows(case)
    new = sum(r[2] for r in rows)
    token = g * d * 4.0                                    # bytes of a token's keys and values
    if case["kind"] == "bounds":
        touched = sum(-(-(c + n) // PAGE) - c // PAGE for _, c, n, _ in rows)
        keys = sum(c + n - c // PAGE * PAGE for _, c, n, _ in rows)
        return {"bytes": keys * token / 2 + touched * g * (2.0 * d + 4.0 + 8.0 * d), "flops": 2.0 * keys * g * d}
    if case["kind"] == "shared":
        keys = PAGE * sum(p for _, _, p in _groups(case)) + sum(c + n for _, c, n, _ in rows)
        pairs = sum(n * (p * PAGE + c) + n * (n + 1) // 2 for p, c, n, _ in rows)
        return {"bytes": keys * token + new * h * d * 4.0, "flops": 4.0 * h * d * pairs}
    scored = chosen = looked = 0
    for _, c, n, _ in rows:
        scored += -(-(c + n) // PAGE)
        for pos in range(c, c + n):
            pages = pos // PAGE + 1
            looked += pages
            chosen += (min(pages, case["count"]) - 1) * PAGE + pos % PAGE + 1
    return {"bytes": scored * g * (2.0 * d + 4.0) + chosen * token + new * (h * d * 4.0 + 4.0 * g * case["count"]), "flops": 4.0 * h * d * (chosen + looked)}


# ---- inputs ------------------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    randn = lambda *s: torch.randn(*s, device="cuda", generator=gen, dtype=torch.bfloat16)  # noqa: E731
    h, g, d, rows = case["heads"], case["kv_heads"], case["dim"], _rows(case)
    ctx, new = [p * PAGE + c for p, c, _, _ in rows], [n for _, _, n, _ in rows]
    own_pages = [-(-(c + n) // PAGE) for _, c, n, _ in rows]
    groups = _groups(case) if case["kind"] == "shared" else []
    n_pages = sum(own_pages) + sum(p for _, _, p in groups)
    order = torch.randperm(n_pages + 3, generator=torch.Generator().manual_seed(int(seed)))[:n_pages].tolist()
    at, pre = 0, []
    for _, _, p in groups:
        pre.append(order[at:at + p])
        at += p
    width = max(r[0] + o for r, o in zip(rows, own_pages))
    table, touched = [], []
    for (p, c, n, j), o in zip(rows, own_pages):
        mine = order[at:at + o]
        at += o
        touched += mine[c // PAGE:]
        mine = (pre[j] if j >= 0 else []) + mine
        table.append(mine + [-1] * (width - len(mine)))
    ints = lambda v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    total = sum(new)
    s = {"case": case, "table": ints(table), "row_start": ints([sum(new[:i]) for i in range(len(new) + 1)]), "row_pos0": ints(ctx),
         "tok_pos": ints([c + i for c, n in zip(ctx, new) for i in range(n)]), "tok_seq": ints([r for r, n in enumerate(new) for _ in range(n)]),
         "max_new": max(new)}
    # keys drift from page to page, as a text's subjects do; a few features are large in all of them
    s["k"] = randn(n_pages + 3, g, PAGE, d)
    s["k"] += 0.7 * randn(n_pages + 3, g, 1, d) + 3.0 * (torch.arange(d, device="cuda") % 37 == 5)
    if case["kind"] != "bounds":
        s["q"] = randn(total, h * d)
        s["v"] = randn(n_pages + 3, g, PAGE, d)
    if case["kind"] == "shared":
        s["groups"] = ints(groups).view(-1, 3)
        return s
    s["touched"] = ints(touched)
    s["filled"] = ints([min(PAGE, c + n - p * PAGE) for _, c, n, _ in rows for p in range(c // PAGE, -(-(c + n) // PAGE))])
    s["codes"], s["scales"] = _bounds(s["k"], torch.full((n_pages + 3,), PAGE, device="cuda"))
    if case["kind"] == "sparse":
        last = torch.tensor([(t[o - 1], (c + n - 1) % PAGE + 1) for t, o, (_, c, n, _) in zip(table, own_pages, rows)], device="cuda")
        s["codes"][last[:, 0]], s["scales"][last[:, 0]] = _bounds(s["k"][last[:, 0]], last[:, 1])
    return s


def _over(a, b):
    """a / b, rounded once: with a plain number on one side the tensor would be multiplied by a reciprocal that is rounded itself."""
    a, b = (torch.full_like(b, a), b) if isinstance(a, float) else (a, torch.full_like(a, b))
    return a / b


def _bounds(k, filled):
    """Codes int8 [pages, heads, 2, d] and scales float32 [pages, heads] of the first `filled` tokens of pages k [pages, heads, 64, d]."""
    codes, scales = [], []
    for i in range(0, k.shape[0], 8192):
        x = k[i:i + 8192].float()
        there = (torch.arange(PAGE, device=k.device) < filled[i:i + 8192, None])[:, None, :, None]
        both = torch.stack([x.masked_fill(~there, math.inf).amin(2), x.masked_fill(~there, -math.inf).amax(2)], dim=2)
        a = both.abs().amax((2, 3)).clamp(min=1e-30)
        codes.append(torch.round(both * _over(127.0, a)[..., None, None]).clamp(-127.0, 127.0).to(torch.int8))
        scales.append(_over(a, 127.0))
    return torch.cat(codes), torch.cat(scales)


# ---- the plain form ----------------------------------------------------------------------------------------------------------

def _plain_bounds(s):
    touched = s["touched"].long()
    codes, scales = _bounds(s["k"][touched], s["filled"])
    s["codes"][touched], s["scales"][touched] = codes, scales
    return tuple((codes.float() * scales[..., None, None]).unbind(2))


def _plain_shared(s):
    c = s["case"]
    h, g, d = c["heads"], c["kv_heads"], c["dim"]
    table, start, pos0 = s["table"].long(), s["row_start"].long(), s["row_pos0"].long()
    rows, total, new, keys = table.shape[0], s["q"].shape[0], s["max_new"], table.shape[1] * PAGE
    k, v = (x[table.clamp(min=0)].transpose(1, 2).reshape(rows, g, keys, d).float() for x in (s["k"], s["v"]))
    step = torch.arange(new, device=table.device)
    q = s["q"].float()[(start[:rows, None] + step).clamp(max=total - 1)]                          # [rows, new, h * d], short rows padded
    q = q.view(rows, new, g, h // g, d).transpose(1, 2).reshape(rows, g, new * (h // g), d)
    x = (q @ k.transpose(2, 3)).mul_(d ** -0.5).view(rows, g, new, h // g, keys)
    hidden = torch.arange(keys, device=table.device) > (pos0[:, None] + step)[:, None, :, None, None]
    x = x.masked_fill_(hidden, -math.inf)
    x = x.sub_(x.amax(-1, keepdim=True)).exp_()
    y = (x.view(rows, g, -1, keys) @ v).view(rows, g, new, h // g, d) / x.sum(-1, keepdim=True)
    seq = s["tok_seq"].long()
    return y.transpose(1, 2).reshape(rows, new, h * d)[seq, torch.arange(total, device=table.device) - start[seq]].bfloat16()


def _plain_sparse(s):
    c = s["case"]
    h, g, d, count = c["heads"], c["kv_heads"], c["dim"], c["count"]
    seq, pos, total = s["tok_seq"].long(), s["tok_pos"].long(), s["q"].shape[0]
    table = s["table"].long().clamp(min=0)
    q = s["q"].float().view(total, g, h // g, d)
    a = q.abs().amax(-1, keepdim=True).clamp(min=1e-30)
    codes = torch.round(q * _over(127.0, a)).clamp(-127.0, 127.0)
    both = torch.cat([codes.clamp(max=0.0), codes.clamp(min=0.0)], dim=-1)                        # against low and high
    width, score = table.shape[1], []
    for t in range(total):
        held = table[seq[t]]
        n = both[t] @ s["codes"][held].float().permute(1, 2, 3, 0).reshape(g, 2 * d, width)       # [g, h / g, pages]
        score.append((n * _over(a[t], 127.0)).amax(1) * s["scales"][held].T)
    score = torch.stack(score)                                                                    # [total, g, pages]
    p, last = torch.arange(width, device=pos.device), (pos // PAGE)[:, None, None]
    score = score.masked_fill((p < c["first"]) | (p > last - c["last"]), math.inf).masked_fill(p > last, -math.inf)
    best = score.sort(dim=-1, descending=True, stable=True).indices[..., :count]
    best = torch.where(best <= last, best, width).sort(-1).values
    if best.shape[-1] < count:
        best = torch.nn.functional.pad(best, (0, count - best.shape[-1]), value=width)
    there = best < width
    held = table[seq[:, None, None], best.clamp(max=width - 1)]
    head = torch.arange(g, device=pos.device)[None, :, None]
    hidden = (best[..., None] * PAGE + torch.arange(PAGE, device=pos.device) > pos[:, None, None, None]) | ~there[..., None]
    out = []
    for i in range(0, total, 16):                          # (in parts: the chosen pages of all tokens are many)
        at = slice(i, i + 16)
        k, v = (x[held[at], head].float().flatten(2, 3) for x in (s["k"], s["v"]))                # [tokens, g, count * 64, d]
        x = (q[at] @ k.transpose(2, 3)).mul_(d ** -0.5).masked_fill_(hidden[at].flatten(2)[:, :, None], -math.inf)
        x = x.sub_(x.amax(-1, keepdim=True)).exp_()
        out.append((x @ v) / x.sum(-1, keepdim=True))
    return torch.where(there, best, -1).int(), torch.cat(out).view(total, h * d).bfloat16()


def run(state):
    kind, c = state["case"]["kind"], state["case"]
    if not own:
        return _plain_bounds(state) if kind == "bounds" else _plain_shared(state) if kind == "shared" else _plain_sparse(state)
    from exl3_server_b200.ops import kernels as K
    h, g, d = c["heads"], c["kv_heads"], c["dim"]
    if kind == "bounds":
        K.page_bounds(state["k"], state["codes"], state["scales"], state["table"], state["row_start"], state["row_pos0"], state["max_new"])
        return K.page_bounds_load(state["codes"], state["scales"], state["touched"])
    if "workspace" not in state:
        from exl3_server_b200.engine.batch import Workspace
        state["workspace"] = Workspace(state["q"].device)
    if kind == "shared":
        return K.attn_shared(state["q"], state["k"], state["v"], state["table"], state["row_start"], state["row_pos0"], state["groups"],
                             state["max_new"], h, g, d, scale=d ** -0.5, workspace=state["workspace"])
    pages = K.page_select(state["q"], state["codes"], state["scales"], state["table"], state["tok_pos"], state["tok_seq"], c["count"], h, g, d,
                          first=c["first"], last=c["last"])
    return pages, K.attn_pages(state["q"], state["k"], state["v"], state["table"], state["tok_pos"], state["tok_seq"], pages, h, g, d,
                               scale=d ** -0.5, workspace=state["workspace"])


# ---- in 64 bits --------------------------------------------------------------------------------------------------------------

def _attention(q, k, v, upto):
    """q [n, d], the keys of positions below `upto` (a number for each query) of k and v [keys, d]."""
    z = (q.to(F64) @ k.to(F64).T) / math.sqrt(q.shape[1])
    z = torch.where(torch.arange(k.shape[0], device=k.device)[None] < upto[:, None], z, torch.tensor(-math.inf, dtype=F64, device=k.device))
    return torch.softmax(z, dim=-1) @ v.to(F64)


def exact(case, seed):
    s = prepare(case, seed)
    h, g, d = case["heads"], case["kv_heads"], case["dim"]
    table, start, ctx = s["table"].tolist(), s["row_start"].tolist(), s["row_pos0"].tolist()
    if case["kind"] == "bounds":
        low, high = [], []
        for r, c in enumerate(ctx):
            end = c + start[r + 1] - start[r]
            for p in range(c // PAGE, (end - 1) // PAGE + 1):
                k = s["k"][table[r][p], :, :min(PAGE, end - p * PAGE)].to(F64)
                mn, mx = k.min(1).values, k.max(1).values
                a = torch.maximum(mn.abs(), mx.abs()).max(1, keepdim=True).values.clamp(min=1e-30)
                inv = (127 / a).float().to(F64)                                                   # what the codes are rounded from is float32 by the definition
                for x, out in ((mn, low), (mx, high)):
                    out.append((x * inv).float().to(F64).round().clamp(-127, 127) * (a / 127))
        return torch.stack(low), torch.stack(high)
    out = torch.empty(start[-1], h, d, dtype=F64, device="cuda")
    pages = torch.full((start[-1], g, case.get("count", 1)), -1, dtype=torch.int32)
    for r, c in enumerate(ctx):
        n = start[r + 1] - start[r]
        upto = torch.arange(c + 1, c + n + 1, device="cuda")
        held = torch.tensor(table[r][:-(-(c + n) // PAGE)], device="cuda")
        if case["kind"] == "shared":
            k, v = (s[x][held].transpose(0, 1).reshape(g, -1, d) for x in ("k", "v"))
            for head in range(h):
                out[start[r]:start[r + 1], head] = _attention(s["q"][start[r]:start[r + 1], head * d:(head + 1) * d], k[head // (h // g)], v[head // (h // g)], upto)
            continue
        for t in range(start[r], start[r + 1]):
            pos = c + t - start[r]
            mine = held[:pos // PAGE + 1]
            q = s["q"][t].view(g, h // g, d)
            a = q.to(F64).abs().max(-1, keepdim=True).values.clamp(min=1e-30)
            code = (q.to(F64) * (127 / a).float().to(F64)).float().to(F64).round().clamp(-127, 127)
            bound = s["codes"][mine].to(F64)                                                      # [pages, g, 2, d]
            for kv in range(g):
                whole = torch.stack([torch.maximum(x * bound[:, kv, 0], x * bound[:, kv, 1]).sum(-1) for x in code[kv]])       # [h / g, pages]
                score = (whole.float() * (a[kv] / 127).float()).max(0).values * s["scales"][mine, kv]
                score = score.tolist()
                must = {p for p in range(len(score)) if p < case["first"] or p >= len(score) - case["last"]}
                rest = sorted((p for p in range(len(score)) if p not in must), key=lambda p: (-score[p], p))
                picked = sorted(sorted(must)[:case["count"]] + rest[:max(0, case["count"] - len(must))])
                pages[t, kv, :len(picked)] = torch.tensor(picked, dtype=torch.int32)
                at = mine[torch.tensor(picked, device="cuda")]
                k, v = (s[x][at, kv].reshape(-1, d) for x in ("k", "v"))
                last = torch.full((h // g,), (len(picked) - 1) * PAGE + (pos % PAGE + 1 if picked[-1] == pos // PAGE else PAGE), device="cuda")
                out[t, kv * (h // g):(kv + 1) * (h // g)] = _attention(q[kv], k, v, last)
    out = out.view(start[-1], h * d)
    return out if case["kind"] == "shared" else (pages.cuda(), out)
