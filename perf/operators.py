"""The operators of a decode step that keeps its cache in 4 bits and its weights in 8, as cases that can be timed and compared.

Three kinds of work:

``cache``   a step's queries and keys are rotated, its keys and values go to the pages of the 4-bit cache, and the pages that were
            touched are read back.  Outputs: the rotated queries, and the keys and values that the pages stand for.
``attend``  attention of a step's new tokens over the 4-bit cache: one token a sequence (decoding), a few, or whole prompts.
``linear``  ``y = x W^T`` (plain, with a bias, or ``silu(gate) * up``), x rounded to 8-bit floating point with a scale for each row and
            128 features (``a = max |x|``, scale ``a / 448``, ``code = e4m3(x * (448 / a))`` in float32), W held in 8 bits with a scale for
            each block of 128 x 128.

The 4-bit format.  Each group of 32 features of a token's head keeps ``mn = bfloat16(min)`` and ``sc = bfloat16((max - mn) / 15)``, and for
each feature ``code = clamp(rint((x - mn) * (1 / sc)), 0, 15)`` in float32 (0 where sc is not above 1e-30); it stands for ``mn + sc * code``.  A page of
64 tokens of one key/value head is ``d / 64`` tiles of 5,120 bytes, each of ``4096 / d`` tokens: 2,048 bytes of key codes, a word
``sc << 16 | mn`` per token and group, 2,048 bytes of value codes, and their words.  Key codes: per token the words (t, group), t =
0..3, with features ``32 group + 8 t + e`` in nibble ``e / 2 + 4 (e % 2)``.  Value codes: per 16 tokens, 64 features and g = 0..7 the words (t,
u), t, u = 0..3, of token ``8 (u / 2) + 2 t + u % 2`` with features ``4 g + n`` in nibble n and ``32 + 4 g + n`` in nibble 4 + n.

``exact`` restates the operators in float64.
"""
from __future__ import annotations

import math

import torch

own = False          # True: the library's kernels; False: the plain form
F64 = torch.float64
TILE = 5120          # bytes of a tile of the 4-bit cache
PAGE = 64            # tokens of a page


def listed():
    return [
        # decoding's cache write: a busy server, one token a sequence
        dict(name="cache-step-64", kind="cache", rows=64, ctx_low=200, ctx_high=4000, new_low=1, new_high=1, heads=32, kv_heads=8, dim=128),
        # a prompt's cache write, every head with keys of its own
        dict(name="cache-prompt-4096", kind="cache", rows=1, ctx_low=0, ctx_high=0, new_low=4096, new_high=4096, heads=36, kv_heads=36, dim=64),
        # one user's short context on the smallest model: latency
        dict(name="attend-short", kind="attend", rows=1, ctx_low=127, ctx_high=127, new_low=1, new_high=1, heads=16, kv_heads=2, dim=64, window=0),
        # eight sequences, every head with keys of its own: the benchmark's decode step
        dict(name="attend-b8-4096", kind="attend", rows=8, ctx_low=4095, ctx_high=4095, new_low=1, new_high=1, heads=36, kv_heads=36, dim=64, window=0),
        # a full batch of unequal contexts, four query heads a key/value head
        dict(name="attend-b64-ragged", kind="attend", rows=64, ctx_low=130, ctx_high=8000, new_low=1, new_high=1, heads=32, kv_heads=8, dim=128, window=0),
        # a few tokens a sequence (drafts that are checked) over a window, sixteen query heads a key/value head
        dict(name="attend-drafts", kind="attend", rows=5, ctx_low=900, ctx_high=5000, new_low=2, new_high=5, heads=32, kv_heads=2, dim=128, window=2048),
        # one very long context
        dict(name="attend-long", kind="attend", rows=1, ctx_low=131070, ctx_high=131070, new_low=1, new_high=1, heads=32, kv_heads=8, dim=128, window=0),
        # a long prompt behind a shared beginning
        dict(name="attend-prompt", kind="attend", rows=1, ctx_low=1200, ctx_high=1200, new_low=3900, new_high=3900, heads=32, kv_heads=8, dim=128, window=0),
        # one user's decoding: the feed-forward's second matrix
        dict(name="linear-b1", kind="linear", m=1, n=2304, k=5760, gated=False, bias=False),
        # a small batch on the larger model: gate and up projections
        dict(name="linear-b8-gated", kind="linear", m=8, n=32768, k=4096, gated=True, bias=False),
        # a full batch's q/k/v projection
        dict(name="linear-b64", kind="linear", m=64, n=6144, k=4096, gated=False, bias=True),
        # a prompt's gate and up projections
        dict(name="linear-prompt", kind="linear", m=2048, n=28672, k=4096, gated=True, bias=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_HEADS = ((16, 2, 64), (36, 36, 64), (32, 8, 128), (32, 2, 128), (8, 8, 128), (24, 8, 64), (7, 1, 128), (12, 12, 128))


def draw(rng):
    kind = rng.choice(["cache", "attend", "attend", "attend", "linear", "linear"])
    most = {k: max(work(c)[k] for c in listed() if c["kind"] == kind) for k in ("bytes", "flops")}
    while True:
        if kind == "linear":
            gated = rng.random() < 0.4
            case = dict(kind=kind, m=_log_int(rng, 1, 4096), n=16 * _log_int(rng, 16, 2048), k=16 * _log_int(rng, 16, 1024), gated=gated,
                        bias=not gated and rng.random() < 0.5)
        else:
            h, g, d = rng.choice(_HEADS)
            rows = _log_int(rng, 1, 64)
            shape = rng.choice(["step", "step", "few", "prompt"])
            new = 1 if shape == "step" else _log_int(rng, 2, 16) if shape == "few" else _log_int(rng, 17, 3000)
            high = _log_int(rng, 1, 30000 if kind == "attend" else 8000)
            low = max(0, int(high * rng.uniform(0.0, 1.0)) - 1)
            case = dict(kind=kind, rows=rows, ctx_low=low, ctx_high=high, new_low=max(1, int(new * rng.uniform(0.2, 1.0))), new_high=new,
                        heads=h, kv_heads=g, dim=d)
            if kind == "attend":
                case["window"] = _log_int(rng, 64, 4096) if rng.random() < 0.25 else 0
                # what the plain form writes out: one score for every pair of a row's longest
                if rows * h * new * (high + new) > 8e8:
                    continue
        w = work(case)
        if all(w[k] <= most[k] for k in most):
            return case


def _rows(case):
    """(tokens before the step, new tokens) of each row: spread over the case's range, the same for every seed."""
    out = []
    for i in range(case["rows"]):
        u, v = ((i + 1) * 0.6180339887498949) % 1.0, ((i + 1) * 0.7548776662466927) % 1.0
        out.append((case["ctx_low"] + int(round(u * (case["ctx_high"] - case["ctx_low"]))),
                    case["new_low"] + int(round(v * (case["new_high"] - case["new_low"])))))
    return out


def _visible(ctx, new, window):
    """(pairs of a query and a key it sees, keys that some query sees) of one row."""
    seen = [min(p + 1, window) if window else p + 1 for p in range(ctx, ctx + new)]
    return sum(seen), ctx + new - (max(0, ctx - window + 1) if window else 0)


def work(case):
    if case["kind"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        blocks = -(-n // 128) * -(-k // 128)
        return {"bytes": 2.0 * m * k + n * k + 4.0 * blocks + 2.0 * m * (n // 2 if case["gated"] else n) + (2.0 * n if case["bias"] else 0.0),
                "flops": 2.0 * m * n * k}
    h, g, d, rows = case["heads"], case["kv_heads"], case["dim"], _rows(case)
    new = sum(n for _, n in rows)
    held = g * d * 1.25                                    # bytes of a token's keys and values in the cache
    if case["kind"] == "cache":
        back = PAGE * sum(-(-(c + n) // PAGE) - c // PAGE for c, n in rows)
        return {"bytes": new * ((h + 2 * g) * d * 2.0 + h * d * 2.0 + held) + back * (held + g * d * 4.0), "flops": new * (h + 2 * g) * d * 8.0}
    pairs, keys = (sum(x) for x in zip(*(_visible(c, n, case["window"]) for c, n in rows)))
    return {"bytes": keys * held + new * h * d * 4.0, "flops": 4.0 * h * d * pairs}


# ---- inputs ------------------------------------------------------------------------------------------------------------------

def _rotary_table(dim, theta=10000.0):
    """Frequencies in two float32 rows: rounded, and what the rounding lost."""
    f = theta ** (-2.0 * torch.arange(dim // 2, dtype=F64) / dim)
    hi = f.float()
    return torch.stack([hi, (f - hi.double()).float()]).cuda()


def _random_pool(pages, g, d, gen):
    """Pages whose codes are uniform and whose groups have scales around 0.3 and minima around -7.5 scales."""
    tok = 4096 // d
    pool = torch.randint(0, 256, (pages, g, d // 64, TILE), dtype=torch.uint8, device="cuda", generator=gen)
    n = tok * (d // 32)
    sc = (0.3 * torch.exp(0.4 * torch.randn(pages, g, d // 64, 2, n, device="cuda", generator=gen))).bfloat16()
    mn = (-sc.float() * (7.5 + 1.5 * torch.randn(sc.shape, device="cuda", generator=gen))).bfloat16()
    words = torch.stack([mn, sc], dim=-1).contiguous().view(torch.uint8).view(pages, g, d // 64, 2, 512)
    pool[..., 2048:2560] = words[..., 0, :]
    pool[..., 4608:5120] = words[..., 1, :]
    return pool.view(pages, g, d // 64 * TILE)


def _quantize_weight(w):
    """8-bit codes of w and a scale for each block of 128 x 128."""
    n, k = w.shape
    nb, kb = -(-n // 128), -(-k // 128)
    x = torch.zeros(nb * 128, kb * 128, device=w.device)
    x[:n, :k] = w.float()
    x = x.view(nb, 128, kb, 128)
    amax = x.abs().amax(dim=(1, 3)).clamp(min=1e-30)
    codes = (x * (448.0 / amax)[:, None, :, None]).to(torch.float8_e4m3fn)
    return codes.view(nb * 128, kb * 128)[:n, :k].contiguous(), (amax / 448.0).contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    randn = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    if case["kind"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        x = randn(m, k) * torch.where(torch.rand(k, device="cuda", generator=gen) < 0.005, 12.0, 1.0)      # a few features stand out
        w, ws = _quantize_weight(randn(n, k) * 0.02)
        return {"case": case, "x": x.bfloat16(), "w": w, "ws": ws, "bias": (randn(n) * 0.1).bfloat16() if case["bias"] else None}
    h, g, d, rows = case["heads"], case["kv_heads"], case["dim"], _rows(case)
    ctx, new = [c for c, _ in rows], [n for _, n in rows]
    total, width = sum(new), max(-(-(c + n) // PAGE) for c, n in rows)
    n_pages = sum(-(-(c + n) // PAGE) for c, n in rows)
    order = torch.randperm(n_pages + 3, generator=torch.Generator().manual_seed(int(seed)))[:n_pages].tolist()
    table, touched, at = [], [], 0
    for c, n in rows:
        mine = order[at:at + -(-(c + n) // PAGE)]
        at += len(mine)
        table.append(mine + [-1] * (width - len(mine)))
        touched += mine[c // PAGE:]
    ints = lambda v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    start = [sum(new[:i]) for i in range(len(new) + 1)]
    s = {"case": case, "pool": _random_pool(n_pages + 3, g, d, gen), "table": ints(table), "row_start": ints(start), "row_pos0": ints(ctx),
         "tok_pos": ints([c + i for c, n in rows for i in range(n)]), "tok_seq": ints([r for r, n in enumerate(new) for _ in range(n)]),
         "max_new": max(new), "max_len": max(c + n for c, n in rows)}
    if case["kind"] == "cache":
        s["qkv"] = (randn(total, (h + 2 * g) * d) * torch.exp(0.5 * randn((h + 2 * g) * d))).bfloat16()
        s["rotary"] = _rotary_table(d)
        s["touched"] = ints(touched)
    else:
        s["q"] = (1.5 * randn(total, h * d)).bfloat16()
        tiles = sorted(((ctx[r] + min(a + 128, new[r]), r, a) for r in range(len(new)) for a in range(0, new[r], 128)), key=lambda t: -t[0])
        s["tiles"] = (ints([r for _, r, _ in tiles]), ints([a for _, _, a in tiles]), len(tiles))
    return s


# ---- the plain form ----------------------------------------------------------------------------------------------------------

def _values(pool, d):
    """What pages [..., TILE * d / 64] stand for: keys and values [..., 64, d] in float32."""
    lead, tok, n = pool.shape[:-1], 4096 // d, d // 64
    x = pool.reshape(-1, n, TILE)
    part = lambda a, b: x[..., a:b].contiguous().view(torch.int32)  # noqa: E731
    e = torch.arange(8, dtype=torch.int32, device=pool.device)
    kc = part(0, 2048).view(-1, n, tok, 4, d // 32, 1) >> (4 * (e // 2 + 4 * (e % 2))) & 15        # [page, tile, token, t, group, e]
    kc = kc.transpose(3, 4).reshape(-1, n, tok, d // 32, 32)
    vc = part(2560, 4608).view(-1, n, tok // 16, d // 64, 8, 4, 2, 2, 1) >> (4 * e) & 15           # [page, tile, 16s, 64s, g, t, u / 2, u % 2, nibble]
    vc = vc.view(-1, n, tok // 16, d // 64, 8, 4, 2, 2, 2, 4).permute(0, 1, 2, 6, 5, 7, 3, 8, 4, 9).reshape(-1, n, tok, d // 32, 32)
    out = []
    for codes, words in ((kc, part(2048, 2560)), (vc, part(4608, 5120))):
        words = words.view(-1, n, tok, d // 32, 1)
        sc, mn = (words & -65536).view(torch.float32), (words << 16).view(torch.float32)
        out.append((mn + sc * codes.float()).reshape(*lead, PAGE, d))
    return out


def _over(a, b):
    """a / b, rounded once: with a plain number on one side the tensor would be multiplied by a reciprocal that is rounded itself."""
    a, b = (torch.full_like(b, a), b) if isinstance(a, float) else (a, torch.full_like(a, b))
    return a / b


def _rounded(x):
    """x [..., d] in float32 as the 4-bit format holds it."""
    y = x.reshape(*x.shape[:-1], -1, 32)
    mn, mx = y.amin(-1, keepdim=True).bfloat16().float(), y.amax(-1, keepdim=True)
    sc = _over((mx - mn).clamp(min=0.0), 15.0).bfloat16().float()
    inv = torch.where(sc > 1e-30, _over(1.0, sc), torch.zeros_like(sc))
    return (mn + sc * torch.round((y - mn) * inv).clamp(0.0, 15.0)).view(x.shape)


def _angles(pos, table):
    """Cosines and sines [tokens, pairs] in float32.  A product with the frequency's leading eight bits is exact for positions below 65,536,
    so the angle keeps its accuracy; the rest of the frequency makes a small angle of its own."""
    lead = (table[0].view(torch.int32) & -65536).view(torch.float32)
    p = pos.float()[:, None]
    a, b = p * lead, p * ((table[0] - lead) + table[1])
    return a.cos() * b.cos() - a.sin() * b.sin(), a.sin() * b.cos() + a.cos() * b.sin()


def _turned(x, cos, sin):
    u, v = x.chunk(2, dim=-1)
    return torch.cat([u * cos[:, None] - v * sin[:, None], v * cos[:, None] + u * sin[:, None]], dim=-1)


def _plain_cache(s):
    c = s["case"]
    h, g, d = c["heads"], c["kv_heads"], c["dim"]
    q, k, v = s["qkv"].float().view(-1, h + 2 * g, d).split([h, g, g], dim=1)
    cos, sin = _angles(s["tok_pos"], s["rotary"])
    q, k = _turned(q, cos, sin), _turned(k, cos, sin)
    touched, pos = s["touched"].long(), s["tok_pos"].long()
    keys, values = _values(s["pool"][touched], d)                                                 # [pages, heads, 64, d]
    place = torch.zeros(s["pool"].shape[0], dtype=torch.long, device=touched.device)
    place[touched] = torch.arange(touched.numel(), device=touched.device)
    page = place[s["table"][s["tok_seq"].long(), pos // PAGE].long()]
    keys[page, :, pos % PAGE] = _rounded(k)
    values[page, :, pos % PAGE] = _rounded(v)
    return q.reshape(-1, h * d).bfloat16(), keys.bfloat16(), values.bfloat16()


def _plain_attend(s):
    c = s["case"]
    h, g, d, window = c["heads"], c["kv_heads"], c["dim"], c["window"]
    table, start, pos0 = s["table"].long(), s["row_start"].long(), s["row_pos0"].long()
    rows, total, new, keys = table.shape[0], s["q"].shape[0], s["max_new"], table.shape[1] * PAGE
    k, v = (x.transpose(1, 2).reshape(rows, g, keys, d) for x in _values(s["pool"][table.clamp(min=0)], d))
    step = torch.arange(new, device=table.device)
    q = s["q"].float()[(start[:rows, None] + step).clamp(max=total - 1)]                          # [rows, new, h * d], short rows padded
    q = q.view(rows, new, g, h // g, d).transpose(1, 2).reshape(rows, g, new * (h // g), d)
    x = (q @ k.transpose(2, 3)).mul_(d ** -0.5).view(rows, g, new, h // g, keys)
    pos, at = (pos0[:, None] + step)[:, None, :, None, None], torch.arange(keys, device=table.device)
    hidden = at > pos
    if window:
        hidden = hidden | (pos - at >= window)
    x = x.masked_fill_(hidden, -math.inf)
    x = x.sub_(x.amax(-1, keepdim=True)).exp_()
    y = (x.view(rows, g, -1, keys) @ v).view(rows, g, new, h // g, d) / x.sum(-1, keepdim=True)
    seq = s["tok_seq"].long()
    return y.transpose(1, 2).reshape(rows, new, h * d)[seq, torch.arange(total, device=table.device) - start[seq]].bfloat16()


def _plain_linear(s):
    (m, k), n = s["x"].shape, s["w"].shape[0]
    kb = -(-k // 128)
    x = torch.nn.functional.pad(s["x"].float(), (0, kb * 128 - k)).view(m, kb, 128)
    amax = x.abs().amax(-1, keepdim=True).clamp(min=1e-30)
    x = (x * _over(448.0, amax)).to(torch.float8_e4m3fn).float() * _over(amax, 448.0)
    w = s["w"].float() * s["ws"].repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    y = x.view(m, kb * 128)[:, :k] @ w.T
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if s["case"]["gated"]:
        gate, up = y.view(m, n // 16, 2, 8).unbind(2)
        y = (gate / (1.0 + torch.exp(-gate)) * up).reshape(m, n // 2)
    return y.bfloat16()


def run(state):
    kind, c = state["case"]["kind"], state["case"]
    if not own:
        return _plain_cache(state) if kind == "cache" else _plain_attend(state) if kind == "attend" else _plain_linear(state)
    from exl3_server_b200.ops import kernels as K
    if kind == "cache":
        q = K.kv4_store(state["qkv"], state["rotary"], state["tok_pos"], state["tok_seq"], state["table"], state["pool"],
                        c["heads"], c["kv_heads"], c["dim"])
        return (q, *K.kv4_load(state["pool"], state["touched"], c["dim"]))
    if kind == "attend":
        if "workspace" not in state:
            from exl3_server_b200.engine.batch import Workspace
            state["workspace"] = Workspace(state["q"].device)
        return K.kv4_attn(state["q"], state["pool"], state["table"], state["row_start"], state["row_pos0"], state["tiles"],
                          state["max_new"], state["max_len"], c["heads"], c["kv_heads"], c["dim"], scale=c["dim"] ** -0.5,
                          window=c["window"], workspace=state["workspace"])
    return K.fp8_linear(state["x"], state["w"], state["ws"], bias=state["bias"], gated=c["gated"])


# ---- in 64 bits --------------------------------------------------------------------------------------------------------------

def _read_group(page, key, tok, grp, d):
    """One tensor of the 32 values of group `grp` of every token in `tok` (a tensor) on `page` [..., bytes], by the format's words."""
    per = 4096 // d
    tile, t_in = tok // per, tok % per
    base = tile * TILE + (0 if key else 2560)
    word = lambda byte: sum(page[..., byte + i].long() << (8 * i) for i in range(4))  # noqa: E731
    pw = word(base + 2048 + (t_in * (d // 32) + grp) * 4)
    bf = lambda bits: ((bits << 16) & 0xFFFFFFFF).to(torch.int32).view(torch.float32).to(F64)  # noqa: E731
    sc, mn = bf(pw >> 16), bf(pw & 0xFFFF)
    vals = []
    for i in range(32):
        if key:
            w = word(base + t_in * (d // 2) + ((i // 8) * (d // 32) + grp) * 4)
            nib = (i % 8) // 2 + 4 * (i % 2)
        else:
            u = t_in % 16
            slot = 2 * (u // 8) + u % 2
            w = word(base + ((((t_in // 16) * (d // 64) + grp // 2) * 8 + i // 4) * 4 + (u % 8) // 2) * 16 + slot * 4)
            nib = i % 4 + 4 * (grp % 2)
        vals.append(mn + sc * ((w >> (4 * nib)) & 15).to(F64))
    return torch.stack(vals, dim=-1)


def _read_pages(pages, d):
    """Keys and values [..., 64, d] in float64 of pages [..., bytes]."""
    tok = torch.arange(PAGE, device=pages.device)
    return [torch.cat([_read_group(pages, key, tok, grp, d) for grp in range(d // 32)], dim=-1) for key in (True, False)]


def _exact_group(x):
    """A group of 32 in float64 as the format holds it; what the format rounds (a group's two bfloat16 numbers, the float32 reciprocal and product) is rounded."""
    y = x.unflatten(-1, (-1, 32))
    mn = y.min(-1, keepdim=True).values.bfloat16().to(F64)
    sc = ((y.max(-1, keepdim=True).values - mn).clamp(min=0) / 15).bfloat16().to(F64)
    inv = torch.where(sc > 1e-30, (1 / sc.clamp(min=1e-38)).float().to(F64), torch.zeros_like(sc))
    code = ((y - mn) * inv).float().to(F64).round().clamp(0, 15)
    return (mn + sc * code).flatten(-2)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "linear":
        return _exact_linear(case, s)
    h, g, d, rows = case["heads"], case["kv_heads"], case["dim"], _rows(case)
    start = s["row_start"].tolist()
    if case["kind"] == "cache":
        x = s["qkv"].to(F64).view(-1, h + 2 * g, d)
        f = s["rotary"].to(F64).sum(0)
        a = s["tok_pos"].to(F64)[:, None, None] * f
        turn = lambda y: torch.cat([y[..., :d // 2] * a.cos() - y[..., d // 2:] * a.sin(), y[..., d // 2:] * a.cos() + y[..., :d // 2] * a.sin()], -1)  # noqa: E731
        q, k, v = turn(x[:, :h]), _exact_group(turn(x[:, h:h + g])), _exact_group(x[:, h + g:])
        keys, values = _read_pages(s["pool"][s["touched"].long()], d)
        at = 0
        for r, (c, n) in enumerate(rows):
            first, last = c // PAGE, -(-(c + n) // PAGE)
            for out, new in ((keys, k), (values, v)):
                mine = out[at:at + last - first].transpose(1, 2).reshape(-1, g, d).clone()
                mine[c - first * PAGE:c - first * PAGE + n] = new[start[r]:start[r + 1]]
                out[at:at + last - first] = mine.view(last - first, PAGE, g, d).transpose(1, 2)
            at += last - first
        return q.reshape(-1, h * d), keys, values
    out = torch.empty(start[-1], h, d, dtype=F64, device="cuda")
    for r, (c, n) in enumerate(rows):
        pages = s["pool"][s["table"][r, :-(-(c + n) // PAGE)].long()]
        i = torch.arange(c, c + n, device="cuda")[:, None]
        j = torch.arange(c + n, device="cuda")[None]
        hidden = (j > i) | (i - j >= case["window"]) if case["window"] else j > i
        for kv in range(g):
            k, v = (x.reshape(-1, d)[:c + n] for x in _read_pages(pages[:, kv], d))
            for head in range(kv * (h // g), (kv + 1) * (h // g)):
                z = (s["q"][start[r]:start[r + 1], head * d:(head + 1) * d].to(F64) @ k.T) * d ** -0.5
                out[start[r]:start[r + 1], head] = torch.softmax(z.masked_fill(hidden, -math.inf), dim=-1) @ v
    return out.view(-1, h * d)


def _e4m3(x):
    """The nearest number of 4 exponent and 3 fraction bits (ties to even), in float64."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return ((x / step).round() * step).clamp(-448, 448)


def _exact_linear(case, s):
    m, k = s["x"].shape
    y = torch.zeros(m, case["n"], dtype=F64, device="cuda")
    for b, k0 in enumerate(range(0, k, 128)):
        x = s["x"][:, k0:k0 + 128].to(F64)
        amax = x.abs().amax(1, keepdim=True).clamp(min=1e-30)
        codes = _e4m3((x * (448 / amax).float().to(F64)).float().to(F64))         # of a float32 product, by the definition
        block = (codes * (amax / 448)) @ s["w"][:, k0:k0 + 128].to(torch.float32).to(F64).T
        y += block * s["ws"][:, b].to(F64).repeat_interleave(128)[:case["n"]]
    if s["bias"] is not None:
        y += s["bias"].to(F64)
    if case["gated"]:
        y = y.view(m, -1, 2, 8)
        y = (y[:, :, 0] * torch.sigmoid(y[:, :, 0]) * y[:, :, 1]).reshape(m, -1)
    return y
