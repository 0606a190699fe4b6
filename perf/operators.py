"""Operators of a paged step over a key / value cache held in 4 bits, in their plain form (elementary torch operations in 32 bits, 64 where a border
decides) and, where `own` is set, as calls of `nanoengine_b200.ops`: the step's tables built on the GPU, the rows between the qkv projection and
the attention (head norms, rotation by one position or by one per axis, 4-bit or bf16 rows into their pages), and the attention that reads them.

A 4-bit page holds, for every kv head, the codes of its tokens and then their scales: uint8 [blocks, kv heads, block_size * (D / 2 + D / 32)].
Groups of 32 neighbouring dims share a scale byte b = 8 e + m, which stands for (8 + m) 2^(e - 19); a code c stands for (c - 8) scale.  A
32-bit word holds 8 dims, those of even place in its low half, the others in its high half, lowest first.

The listed cases stand for

  one            a single user's decode step behind a thousand tokens: latency
  decode         Qwen3-235B attention of an ordinary decode step: 128 sequences at about 4K tokens
  long           two users behind 128K tokens each
  wide_heads     Qwen3.5 attention (heads of 256) of a decode step, odd lengths
  verify         a short portion of four tokens per sequence, 8 kv heads, ragged contexts
  prompt         ragged prompts behind cached prefixes: the largest call
  rows_decode    the rows of a decode step: 128 tokens, 4-bit
  rows_image     the rows of 4096 prompt tokens with images (time, height, width taking turns over the angles), 4-bit
  rows_video     the same by sections into bf16 rows, 32 / 8 heads
  tables_decode  the tables of a decode step of 128 sequences, padded to a captured batch of 144
  tables_prompt  the tables of ragged prompts of 16K tokens
  tables_one     the tables of one sequence behind 128K tokens

and `draw` takes the same over the whole range: single tokens to thousands, short and long contexts, windows, the head counts of whole and
tensor-parallel layers."""
import math

import numpy as np
import torch

own = False
PAGE = 64
GROUP = 32
EPS = 1e-6
BF16 = torch.bfloat16
F64 = torch.float64


def listed():
    return [
        {"name": "one", "kind": "attention", "batch": 1, "prefix": 1000, "new": 1, "hq": 32, "hkv": 8, "dim": 128, "window": 0},
        {"name": "decode", "kind": "attention", "batch": 128, "prefix": 4095, "new": 1, "hq": 64, "hkv": 4, "dim": 128, "window": 0},
        {"name": "long", "kind": "attention", "batch": 2, "prefix": 131071, "new": 1, "hq": 64, "hkv": 4, "dim": 128, "window": 0},
        {"name": "wide_heads", "kind": "attention", "batch": 60, "prefix": 2999, "new": 1, "hq": 16, "hkv": 2, "dim": 256, "window": 0},
        {"name": "verify", "kind": "attention", "batch": 33, "prefix": 2500, "new": 4, "hq": 32, "hkv": 8, "dim": 128, "window": 0},
        {"name": "prompt", "kind": "attention", "batch": 4, "prefix": 700, "new": 1500, "hq": 64, "hkv": 4, "dim": 128, "window": 0},
        {"name": "rows_decode", "kind": "rows", "tokens": 128, "hq": 64, "hkv": 4, "dim": 128, "cache": "int4", "axes": 1, "turns": False},
        {"name": "rows_image", "kind": "rows", "tokens": 4096, "hq": 64, "hkv": 4, "dim": 128, "cache": "int4", "axes": 3, "turns": True},
        {"name": "rows_video", "kind": "rows", "tokens": 4097, "hq": 32, "hkv": 8, "dim": 128, "cache": "bf16", "axes": 3, "turns": False},
        {"name": "tables_decode", "kind": "tables", "batch": 128, "prefix": 4095, "new": 1, "rows": 144},
        {"name": "tables_prompt", "kind": "tables", "batch": 13, "prefix": 900, "new": 1260, "rows": 13},
        {"name": "tables_one", "kind": "tables", "batch": 1, "prefix": 131071, "new": 1, "rows": 1},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(["decode", "decode", "decode", "verify", "prompt", "rows", "rows", "rows", "tables", "tables"])
    hq, hkv, dim = rng.choice([(64, 4, 128), (64, 4, 128), (8, 1, 128), (32, 8, 128), (16, 2, 256), (16, 4, 64), (24, 2, 128), (8, 8, 128)])
    if kind in ("decode", "verify"):
        new = 1 if kind == "decode" else rng.randrange(2, 7)
        batch = _log(rng, 1, 192)
        return {"kind": "attention", "batch": batch, "prefix": _log(rng, 1, min(100000, 400000 // (batch * hkv))), "new": new, "hq": hq, "hkv": hkv, "dim": dim,
                "window": rng.choice([0, 0, 0, rng.randrange(100, 2000)])}
    if kind == "prompt":
        batch = _log(rng, 1, 5)
        return {"kind": "attention", "batch": batch, "prefix": rng.choice([0, rng.randrange(1, 1200)]), "new": _log(rng, 20, 3000 // batch), "hq": hq, "hkv": hkv, "dim": dim,
                "window": rng.choice([0, 0, rng.randrange(100, 1000)])}
    if kind == "rows":
        axes = rng.choice([1, 3, 3])
        return {"kind": "rows", "tokens": _log(rng, 1, 4096), "hq": hq, "hkv": hkv, "dim": dim, "cache": rng.choice(["int4", "int4", "bf16"]) if axes == 3 else "int4", "axes": axes,
                "turns": axes == 3 and rng.random() < 0.5}
    batch = _log(rng, 1, 256)
    new = rng.choice([1, 1, _log(rng, 1, 16000 // batch)])
    return {"kind": "tables", "batch": batch, "prefix": _log(rng, 1, min(131072, 4000000 // batch)), "new": new, "rows": batch + rng.choice([0, rng.randrange(0, 17)])}


# ---- sizes --------------------------------------------------------------------------------------------------------------------
def _spread(n, mean, least):
    """n ragged lengths around `mean`, from half of it to one and a half, with the same sum whatever their order."""
    return [max(least, mean)] if n == 1 else [max(least, int(mean * (0.5 + i / (n - 1)))) for i in range(n)]


def _lengths(case, seed):
    """(new tokens, context with them) of every sequence, in an order made from the seed."""
    b = case["batch"]
    new = [case["new"]] * b if case["new"] <= 6 else _spread(b, case["new"], 1)
    ctx = [n + p for n, p in zip(new, _spread(b, case["prefix"], 0) if case["prefix"] else [0] * b)]
    order = np.random.RandomState(seed).permutation(b)
    return [new[i] for i in order], [ctx[i] for i in order]


def _sections(half):
    """Angles of time, height and width: a quarter to the first, the rest shared."""
    side = half * 3 // 8
    return [half - 2 * side, side, side]


def _seen(new, ctx, window):
    """Query-key pairs of a causal portion, with the last `window` keys only where there is a window."""
    lengths = np.arange(ctx - new + 1, ctx + 1, dtype=np.int64)
    return int((np.minimum(lengths, window) if window else lengths).sum())


def work(case):
    if case["kind"] == "attention":
        new, ctx = _lengths(case, 0)
        row = case["dim"] // 2 + case["dim"] // GROUP
        read = [min(c, case["window"] + n - 1) if case["window"] else c for n, c in zip(new, ctx)]
        tables = sum(-(-c // PAGE) for c in ctx) * 4
        return {"bytes": 2 * sum(read) * case["hkv"] * row + 2 * 2 * sum(new) * case["hq"] * case["dim"] + tables,
                "flops": 4 * case["hq"] * case["dim"] * sum(_seen(n, c, case["window"]) for n, c in zip(new, ctx))}
    if case["kind"] == "rows":
        t, d, hq, hkv = case["tokens"], case["dim"], case["hq"], case["hkv"]
        row = 2 * d if case["cache"] == "bf16" else d // 2 + d // GROUP
        # the projection read, the queries and rows written; then the 4-bit rows read back and handed out as values
        back = 0 if case["cache"] == "bf16" else 2 * t * hkv * (row + 2 * d)
        return {"bytes": t * (hq + 2 * hkv) * d * 2 + t * hq * d * 2 + 2 * t * hkv * row + t * 8 * (case["axes"] + 1) + back, "flops": t * (10 * hq + 16 * hkv) * d}
    new, ctx = _lengths(case, 0)
    pages, rows = [-(-c // PAGE) for c in ctx], case["rows"]
    return {"bytes": 4 * (sum(pages) + 3 * len(new) + 1) + 4 * rows * max(pages) + 4 * (3 * rows + 1) + 16 * (sum(new) + rows - len(new)), "flops": 0}


# ---- the 4-bit format -----------------------------------------------------------------------------------------------------------
PLACES = [0, 2, 4, 6, 1, 3, 5, 7]              # dim of a word's nibble p


def _codes_and_scales(x):
    """x [..., D] in 64 bits -> (signed codes, scale bytes [..., D / 32], scales): nearest scale of four significant bits to a 7th of the largest."""
    g = x.reshape(*x.shape[:-1], -1, GROUP)
    m, e = torch.frexp(g.abs().amax(-1) / 7)
    n = torch.round(m * 16)
    e = torch.where(n == 16, e + 1, e)
    n = torch.where(n == 16, torch.full_like(n, 8), n)
    b = (8 * (e.long() - 4 + 19) + n.long() - 8).clamp(0, 255)
    b = torch.where(m == 0, torch.zeros_like(b), b)
    s = torch.ldexp((8 + b % 8).to(x.dtype), b // 8 - 19)
    return torch.round(g / s[..., None]).clamp(-7, 7).reshape(x.shape), b, s


def _rows_of(x):
    """Packed rows of x [..., D]: codes uint8 [..., D / 2] and scale bytes uint8 [..., D / 32]."""
    q, b, _ = _codes_and_scales(x.to(F64))
    n = (q.long() + 8).view(*x.shape[:-1], -1, 8)[..., PLACES]
    return (n[..., 0::2] + 16 * n[..., 1::2]).to(torch.uint8).reshape(*x.shape[:-1], -1), b.to(torch.uint8)


def _values_of(pages, dim):
    """Values [..., 64, D] in 32 bits of pages [..., 64 * (D / 2 + D / 32)]."""
    codes = pages[..., : PAGE * dim // 2].reshape(*pages.shape[:-1], PAGE, dim // 8, 4)
    b = pages[..., PAGE * dim // 2:].reshape(*pages.shape[:-1], PAGE, dim // GROUP).int()
    n = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)                         # nibbles 0 .. 7
    n = n[..., [PLACES.index(i) for i in range(8)]].flatten(-2).float() - 8
    s = torch.ldexp((8 + (b & 7)).float(), (b >> 3) - 19)
    return n * s.repeat_interleave(GROUP, -1)


# ---- inputs ---------------------------------------------------------------------------------------------------------------------
def _pages(ctx, gen):
    """Block table over randomly placed pages (unused entries point at page 0), and the same as one ragged list."""
    nb = [-(-n // PAGE) for n in ctx]
    ids = torch.randperm(sum(nb), generator=gen, device="cuda").int()
    off = np.concatenate([[0], np.cumsum(nb)])
    at = torch.from_numpy(off[:-1]).cuda()[:, None] + torch.arange(max(nb), device="cuda")[None]
    used = torch.arange(max(nb), device="cuda")[None] < torch.tensor(nb, device="cuda")[:, None]
    return torch.where(used, ids[at.clamp(max=sum(nb) - 1)], 0).int(), ids, torch.from_numpy(off).int().cuda()


def _axes_positions(tokens, gen):
    """Positions [3, tokens] of a text with images in it: runs of text stand still on all axes alike, an image spans its grid."""
    parts, at, left = [], 0, tokens
    sizes = torch.randint(0, 1 << 20, (4 * (tokens // 64 + 4),), generator=gen, device="cuda").tolist()
    while left > 0:
        text = min(left, 1 + sizes.pop() % 60)
        parts.append((at + np.arange(text))[None].repeat(3, 0))
        at, left = at + text, left - text
        if left:
            h, w = 4 + sizes.pop() % 29, 4 + sizes.pop() % 29
            grid = np.stack([np.zeros(h * w, np.int64), np.arange(h * w) // w, np.arange(h * w) % w])[:, : left]
            parts.append(at + grid)
            at, left = at + max(h, w), left - grid.shape[1]
    return torch.from_numpy(np.concatenate(parts, 1).astype(np.int64)).cuda().contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 11)
    rnd = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")               # noqa: E731
    s = {"case": dict(case)}
    if case["kind"] == "rows":
        t, hq, hkv, d = case["tokens"], case["hq"], case["hkv"], case["dim"]
        s["qkv"] = rnd(t, (hq + 2 * hkv) * d).to(BF16)
        s["q_norm"], s["k_norm"] = (1 + 0.1 * rnd(d)).to(BF16), (1 + 0.1 * rnd(d)).to(BF16)
        top = 8192
        angles = torch.outer(torch.arange(top, dtype=F64), 1e6 ** (-torch.arange(0, d, 2, dtype=F64) / d))
        s["rope"] = torch.cat([angles.cos(), angles.sin()], -1).float().cuda()
        s["positions"] = _axes_positions(t, gen) if case["axes"] == 3 else torch.randint(0, top, (t,), generator=gen, device="cuda")
        blocks = t // PAGE + 3
        s["slots"] = torch.randperm(blocks * PAGE, generator=gen, device="cuda")[:t].contiguous()
        if case["cache"] == "bf16":
            s["k"], s["v"] = (torch.zeros(blocks, PAGE, hkv, d, dtype=BF16, device="cuda") for _ in range(2))
        else:
            s["k"], s["v"] = (torch.zeros(blocks, hkv, PAGE * (d // 2 + d // GROUP), dtype=torch.uint8, device="cuda") for _ in range(2))
        s["sections"] = _sections(d // 2) if case["axes"] == 3 else None
        return s
    new, ctx = _lengths(case, seed)
    if case["kind"] == "tables":
        _, s["ids"], s["offsets"] = _pages(ctx, gen)
        s["new"], s["ctx"] = torch.tensor(new, dtype=torch.int32, device="cuda"), torch.tensor(ctx, dtype=torch.int32, device="cuda")
        s["tokens"], s["width"] = sum(new) + case["rows"] - len(new), max(-(-c // PAGE) for c in ctx)
        s["scratch"] = int(s["ids"].numel())
        return s
    hq, hkv, d = case["hq"], case["hkv"], case["dim"]
    s["tables"], ids, _ = _pages(ctx, gen)
    for name in ("k", "v"):
        # keys as they leave a head norm, values a little smaller
        parts = [_rows_of((rnd(n, hkv, PAGE, d) * (1.0 if name == "k" else 0.7)).to(BF16)) for n in [512] * (ids.numel() // 512) + [ids.numel() % 512] if n]
        s[name] = torch.cat([torch.cat([c.flatten(-2), b.flatten(-2)], -1) for c, b in parts]).contiguous()
    s["q"] = rnd(sum(new), hq, d).to(BF16)
    s["cu"] = torch.from_numpy(np.concatenate([[0], np.cumsum(new)]).astype(np.int32)).cuda()
    s["ctx"] = torch.tensor(ctx, dtype=torch.int32, device="cuda")
    s["longest"], s["scale"] = max(new), d ** -0.5
    return s


# ---- one pass ---------------------------------------------------------------------------------------------------------------------
def _attention(s):
    hkv, d, w = s["case"]["hkv"], s["case"]["dim"], s["case"]["window"]
    q, cu, ctx = s["q"], s["cu"].long(), s["ctx"].long()
    b, g = ctx.numel(), q.shape[1] // hkv
    k, v = (_values_of(s[n][s["tables"].long()], d).transpose(1, 2).reshape(b, hkv, -1, d) for n in ("k", "v"))
    new = cu[1:] - cu[:-1]
    step = torch.arange(s["longest"], device=q.device)
    at = (cu[:-1, None] + step).clamp(max=q.shape[0] - 1)
    x = q[at].float().view(b, -1, hkv, g, d).permute(0, 2, 1, 3, 4).reshape(b, hkv, -1, d)       # rows (token, head of the group)
    scores = (x @ k.transpose(-1, -2) * s["scale"]).view(b, hkv, -1, g, k.shape[2])
    place = ((ctx - new)[:, None] + step)[:, None, :, None, None]
    key = torch.arange(k.shape[2], device=q.device)
    hidden = (key > place) | (key <= place - w) if w else key > place
    p = torch.softmax(scores.masked_fill_(hidden, float("-inf")), -1).view(b, hkv, -1, k.shape[2])
    o = (p @ v).view(b, hkv, -1, g, d).permute(0, 2, 1, 3, 4).reshape(b, -1, hkv * g, d)
    return o[step[None] < new[:, None]].to(BF16)


def _angle_axis(case, sections, device):
    """Which axis every angle follows: by sections, or height and width at every third place until theirs are used up."""
    i = torch.arange(case["dim"] // 2, device=device)
    if case["turns"]:
        return torch.where((i % 3 == 1) & (i < 3 * sections[1]), 1, torch.where((i % 3 == 2) & (i < 3 * sections[2]), 2, 0))
    return (i >= sections[0]).long() + (i >= sections[0] + sections[1]).long()


def _normed(x, w):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.to(x.dtype)


def _turned(x, cos, sin):
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _rows(s):
    c = s["case"]
    t, hq, hkv, d = c["tokens"], c["hq"], c["hkv"], c["dim"]
    q, k, v = s["qkv"].view(t, -1, d).split([hq, hkv, hkv], 1)
    if c["axes"] == 3:
        axis = _angle_axis(c, s["sections"], q.device)
        place = s["positions"].t()[:, axis]                                                # [T, D / 2]
        i = torch.arange(d // 2, device=q.device)
        cos, sin = s["rope"][place, i][:, None], s["rope"][place, i + d // 2][:, None]
    else:
        cos, sin = s["rope"][s["positions"]][:, None].chunk(2, -1)
    q = _turned(_normed(q.float(), s["q_norm"]), cos, sin).to(BF16)
    if c["cache"] == "bf16":
        k = _turned(_normed(k.float(), s["k_norm"]), cos, sin)
        for cache, x in ((s["k"], k), (s["v"], v)):
            cache.view(-1, hkv, d)[s["slots"]] = x.to(BF16)
        return q, s["k"], s["v"]
    k = _turned(_normed(k.to(F64), s["k_norm"]), cos.to(F64), sin.to(F64))
    page, at = s["slots"] // PAGE, s["slots"] % PAGE
    back = []
    for cache, x in ((s["k"], k), (s["v"], v)):
        codes, scales = _rows_of(x)
        cache[:, :, : PAGE * d // 2].view(-1, hkv, PAGE, d // 2)[page, :, at] = codes
        cache[:, :, PAGE * d // 2:].view(-1, hkv, PAGE, d // GROUP)[page, :, at] = scales
        back.append(_values_of(cache, d)[page, :, at].to(BF16))
    return q, back[0], back[1]


def _tables(s):
    rows, new, ctx, off = s["case"]["rows"], s["new"].long(), s["ctx"].long(), s["offsets"].long()
    b, more = new.numel(), rows - new.numel()
    dev = new.device
    q = torch.cat([new, torch.ones(more, dtype=torch.long, device=dev)])
    n = torch.cat([ctx, torch.ones(more, dtype=torch.long, device=dev)])
    cu = torch.cat([torch.zeros(1, dtype=torch.long, device=dev), q.cumsum(0)])
    col = torch.arange(s["width"], device=dev)
    mine = torch.where(col < (off[1:] - off[:-1])[:, None], s["ids"][(off[:-1, None] + col).clamp(max=s["ids"].numel() - 1)], 0)
    table = torch.cat([mine, torch.full((more, s["width"]), s["scratch"], dtype=mine.dtype, device=dev)]).int()
    t = torch.arange(s["tokens"], device=dev)
    seq = torch.searchsorted(cu, t, right=True) - 1
    place = n[seq] - q[seq] + t - cu[seq]
    slot = table[seq, place // PAGE].long() * PAGE + place % PAGE
    return cu.int(), n.int(), place, slot, table, (cu[1:] - 1).int()


def run(state):
    s, c = state, state["case"]
    if own:
        from nanoengine_b200 import ops
        if c["kind"] == "attention":
            return ops.gqa_attention_paged(s["q"], s["k"], s["v"], s["tables"], s["cu"], s["ctx"], s["scale"], c["window"])
        if c["kind"] == "rows":
            q = ops.gqa_qkv_prepare(s["qkv"], c["hq"], c["hkv"], c["dim"], s["q_norm"], s["k_norm"], EPS, False, s["positions"], s["rope"], s["k"], s["v"], s["slots"],
                                    s["sections"], c["turns"])
            return (q, s["k"], s["v"]) if c["cache"] == "bf16" else (q, *ops.gqa_kv_gather(s["k"], s["v"], s["slots"], c["dim"]))
        return tuple(ops.step_tables(s["new"], s["ctx"], s["ids"], s["offsets"], PAGE, s["tokens"], s["width"], c["rows"], 1, s["scratch"]))
    return {"attention": _attention, "rows": _rows, "tables": _tables}[c["kind"]](s)


# ---- from the definitions, in 64 bits ---------------------------------------------------------------------------------------------
def _level(b):
    return (8 + b % 8) * 2.0 ** (b // 8 - 19)


def _decoded(page, token, dim):
    """One token's row [..., D] of pages [..., bytes]: bit by bit as the format's description has it."""
    words = page[..., token * dim // 2: (token + 1) * dim // 2].to(torch.int64).unflatten(-1, (-1, 4))
    word = (words * torch.tensor([1, 1 << 8, 1 << 16, 1 << 24], device=page.device)).sum(-1)
    scale = torch.tensor([_level(b) for b in range(256)], dtype=F64, device=page.device)[page[..., PAGE * dim // 2 + token * dim // GROUP:][..., : dim // GROUP].long()]
    row = torch.empty(*page.shape[:-1], dim, dtype=F64, device=page.device)
    for i in range(8):
        row[..., i::8] = ((word >> (4 * (i // 2) + 16 * (i % 2))) & 15).to(F64) - 8
    return row * scale.repeat_interleave(GROUP, -1)


def _nearest(x, levels):
    """The quantised values of x [..., D] in 64 bits: of all 256 scales the one nearest to a 7th of the group's largest (the even one of two),
    then the nearest of its 15 multiples."""
    g = x.unflatten(-1, (-1, GROUP))
    want = g.abs().amax(-1) / 7
    hi = torch.searchsorted(levels, want).clamp(1, 255)
    lo = hi - 1
    up, down = levels[hi] - want, want - levels[lo]
    pick = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    s = levels[pick][..., None]
    return (torch.round(g / s).clamp(-7, 7) * s).flatten(-2)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "attention":
        new, ctx = _lengths(case, seed)
        hkv, d, w = case["hkv"], case["dim"], case["window"]
        g, out, at = case["hq"] // hkv, [], 0
        if sum(n * c for n, c in zip(new, ctx)) * case["hq"] * d > 6e12:
            return None
        for i, (n, c) in enumerate(zip(new, ctx)):
            pages = s["tables"][i, : -(-c // PAGE)].long()
            k, v = (torch.stack([_decoded(s[x][pages], t, d) for t in range(PAGE)], 1).flatten(0, 1)[:c] for x in ("k", "v"))     # [c, kv heads, D]
            place = torch.arange(c - n, c, device="cuda")[:, None]
            key = torch.arange(c, device="cuda")[None]
            off = key > place
            if w:
                off = off | (place - key >= w)
            o = torch.empty(n, case["hq"], d, dtype=F64, device="cuda")
            for h in range(case["hq"]):
                z = s["q"][at: at + n, h].to(F64) @ k[:, h // g].t() * s["scale"]
                z[off] = -math.inf
                z = torch.exp(z - z.amax(-1, keepdim=True))
                o[:, h] = z @ v[:, h // g] / z.sum(-1, keepdim=True)
            out.append(o)
            at += n
        return torch.cat(out)
    if case["kind"] == "rows":
        t, hq, hkv, d = case["tokens"], case["hq"], case["hkv"], case["dim"]
        rows = s["qkv"].to(F64).view(t, hq + 2 * hkv, d)
        place = s["positions"].view(case["axes"], t)
        cos, sin = torch.empty(t, d // 2, dtype=F64, device="cuda"), torch.empty(t, d // 2, dtype=F64, device="cuda")
        for i in range(d // 2):
            if case["axes"] == 1:
                a = 0
            elif case["turns"]:
                a = i % 3 if i % 3 and i < 3 * s["sections"][i % 3] else 0
            else:
                a = 0 if i < s["sections"][0] else 1 if i < s["sections"][0] + s["sections"][1] else 2
            cos[:, i], sin[:, i] = s["rope"][place[a], i].to(F64), s["rope"][place[a], d // 2 + i].to(F64)
        out = torch.empty(t, hq + hkv, d, dtype=F64, device="cuda")
        for h in range(hq + hkv):
            x = rows[:, h]
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / d + EPS) * (s["q_norm"] if h < hq else s["k_norm"]).to(F64)
            out[:, h, : d // 2] = x[:, : d // 2] * cos - x[:, d // 2:] * sin
            out[:, h, d // 2:] = x[:, d // 2:] * cos + x[:, : d // 2] * sin
        q, k, v = out[:, :hq], out[:, hq:], rows[:, hq + hkv:]
        if case["cache"] == "int4":
            levels = torch.tensor([_level(b) for b in range(256)], dtype=F64, device="cuda")
            return q, _nearest(k, levels), _nearest(v, levels)
        full = []
        for x in (k, v):
            c = torch.zeros(s["k"].shape[0] * PAGE, hkv, d, dtype=F64, device="cuda")
            c[s["slots"]] = x
            full.append(c.view(-1, PAGE, hkv, d))
        return q, full[0], full[1]
    new, ctx = _lengths(case, seed)
    ids, off = s["ids"].tolist(), s["offsets"].tolist()
    rows, width = case["rows"], s["width"]
    cu, place, slot, table = [0], [], [], []
    for i in range(rows):
        n, c, mine = (new[i], ctx[i], ids[off[i]: off[i + 1]]) if i < len(new) else (1, 1, [s["scratch"]] * width)
        cu.append(cu[-1] + n)
        place += range(c - n, c)
        slot += [mine[p // PAGE] * PAGE + p % PAGE for p in range(c - n, c)]
        table.append(mine + [0] * (width - len(mine)))
    i32, i64 = torch.int32, torch.int64
    return (torch.tensor(cu, dtype=i32), torch.tensor(ctx + [1] * (rows - len(new)), dtype=i32), torch.tensor(place, dtype=i64), torch.tensor(slot, dtype=i64),
            torch.tensor(table, dtype=i32), torch.tensor(cu[1:], dtype=i32) - 1)
