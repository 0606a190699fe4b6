"""Plain 64-bit statements and inputs shared by the tests of the 4-bit cache, of positions on several axes and of the step tables."""
import math

import numpy as np
import torch

F64 = torch.float64
BF16_HALF_STEP = 2.0 ** -8


def level(b: int) -> float:
    """What scale byte b stands for."""
    return (8 + b % 8) * 2.0 ** (b // 8 - 19)


LEVELS = torch.tensor([level(b) for b in range(256)], dtype=F64)


def decode_row(page: bytes, tok: int, dim: int, bs: int) -> list:
    """Values of one token of one head's page, read byte by byte."""
    out = []
    for d in range(dim):
        word, place = d // 8, d % 8
        nib = place // 2 + 4 * (place % 2)
        byte = page[tok * dim // 2 + 4 * word + nib // 2]
        out.append(((byte >> 4 * (nib % 2) & 15) - 8) * level(page[bs * dim // 2 + tok * dim // 32 + d // 32]))
    return out


def nearest(x: torch.Tensor) -> torch.Tensor:
    """x [..., D] as the format holds it, in 64 bits: the nearest of all 256 scales to a seventh of a group's largest magnitude (the even byte of two),
    then the nearest of its 15 multiples."""
    g = x.to(F64).unflatten(-1, (-1, 32))
    lv = LEVELS.to(x.device)
    want = g.abs().amax(-1) / 7
    hi = torch.searchsorted(lv, want).clamp(1, 255)
    up, down = lv[hi] - want, want - lv[hi - 1]
    s = lv[torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, hi - 1)][..., None]
    return (torch.round(g / s).clamp(-7, 7) * s).flatten(-2)


def random_cache(blocks: int, hkv: int, dim: int, bs: int, gen, device="cpu"):
    """Pages of random codes under scales between 2^-7 and 2, as uint8 [blocks, hkv, bs * (dim / 2 + dim / 32)]."""
    codes = torch.randint(0, 256, (blocks, hkv, bs * dim // 2), generator=gen, dtype=torch.uint8)
    scales = torch.randint(72, 136, (blocks, hkv, bs * dim // 32), generator=gen, dtype=torch.uint8)
    return torch.cat([codes, scales], -1).contiguous().to(device)


def cache_values(cache: torch.Tensor, dim: int) -> torch.Tensor:
    """[blocks, bs, hkv, dim] in 64 bits."""
    bs = cache.shape[2] // (dim // 2 + dim // 32)
    c = cache[..., : bs * dim // 2].long().view(*cache.shape[:2], bs, dim // 8, 4)
    word = (c * torch.tensor([1, 1 << 8, 1 << 16, 1 << 24], device=cache.device)).sum(-1)
    s = LEVELS.to(cache.device)[cache[..., bs * dim // 2:].long()].view(*cache.shape[:2], bs, dim // 32)
    out = torch.empty(*cache.shape[:2], bs, dim, dtype=F64, device=cache.device)
    for i in range(8):
        out[..., i::8] = ((word >> (4 * (i // 2) + 16 * (i % 2))) & 15).to(F64) - 8
    return (out * s.repeat_interleave(32, -1)).transpose(1, 2)


def dense_attention(q, kv, vv, tables, new, ctx, scale, window=0):
    """(result, sum of weights times |v - result|, sum of weights times |v|, largest |score|) in 64 bits; kv / vv [blocks, bs, hkv, D]."""
    q = q.to(F64)
    T, hq, d = q.shape
    hkv, bs = kv.shape[2], kv.shape[1]
    out, spread, mass, top = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(q), 0.0
    at = 0
    for i, (n, c) in enumerate(zip(new, ctx)):
        c = min(c, tables.shape[1] * bs)
        if c > 0 and n > 0:
            ids = tables[i, : -(-c // bs)].tolist()
            zero = torch.zeros_like(kv[0])
            k = torch.cat([kv[p] if 0 <= p < kv.shape[0] else zero for p in ids])[:c]
            v = torch.cat([vv[p] if 0 <= p < vv.shape[0] else zero for p in ids])[:c]
            for t in range(n):
                pos = c - n + t
                if pos < 0:
                    continue
                lo = max(0, pos - window + 1) if window else 0
                for h in range(hkv):
                    rows = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
                    z = q[at + t, rows] @ k[lo: pos + 1, h].t() * scale
                    top = max(top, float(z.abs().max()))
                    w = torch.softmax(z, -1)
                    vs = v[lo: pos + 1, h]
                    o = w @ vs
                    out[at + t, rows] = o
                    spread[at + t, rows] = torch.einsum("gn,gnd->gd", w, (vs[None] - o[:, None]).abs())
                    mass[at + t, rows] = w @ vs.abs()
        at += n
    return out, spread, mass, top


def attention_bound(out, spread, mass, top):
    """How far a result may be off.  Weights w_i (1 + d_i), |d_i| <= h (a half step of bf16), normalised by their own sum give sum w_i d_i (v_i - o) / (1 + sum w d),
    at most h (1 + 2 h) sum w |v - o|; the result is rounded once, h |o|.  32-bit scores of up to `top` with products of up to 256 terms are off
    by at most 2^-15 top, which moves a weight by that share; the exponential adds 2^-20."""
    h = BF16_HALF_STEP
    return h * out.abs() + h * (1 + 2 * h) * (1 + h) * spread + (2.0 ** -15 * top + 2.0 ** -18) * mass + 1e-30


def table_of(ctx, bs, blocks, gen, spare=0):
    """A block table over distinct random pages, and the ragged list with its offsets."""
    nb = [max(0, -(-c // bs)) for c in ctx]
    assert sum(nb) <= blocks
    perm = torch.randperm(blocks, generator=gen)[: sum(nb)].int()
    off = np.concatenate([[0], np.cumsum(nb)]).astype(np.int32)
    table = torch.zeros(len(ctx), max(nb + [1]) + spare, dtype=torch.int32)
    for i, n in enumerate(nb):
        table[i, :n] = perm[off[i]: off[i + 1]]
    return table, perm, torch.from_numpy(off)


def rope_table(dim: int, top: int, device="cpu"):
    a = torch.outer(torch.arange(top, dtype=F64), 1e4 ** (-torch.arange(0, dim, 2, dtype=F64) / dim))
    return torch.cat([a.cos(), a.sin()], -1).float().to(device)


def axis_of(i: int, sections, interleaved: bool) -> int:
    if interleaved:
        a = i % len(sections)
        return a if a and i < len(sections) * sections[a] else 0
    return next(a for a in range(len(sections)) if i < sum(sections[: a + 1]))


def rows_exact(x, w, eps, offset, positions, table, sections, interleaved):
    """x [T, heads, D] normed and rotated in 64 bits; positions [A, T]."""
    x = x.to(F64)
    d = x.shape[-1]
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * (w.to(F64) + offset)
    out = torch.empty_like(x)
    for i in range(d // 2):
        p = positions[axis_of(i, sections, interleaved)]
        c, s = table[p, i].to(F64)[:, None], table[p, d // 2 + i].to(F64)[:, None]
        out[..., i], out[..., i + d // 2] = x[..., i] * c - x[..., i + d // 2] * s, x[..., i + d // 2] * c + x[..., i] * s
    return out


def tables_exact(new, ctx, ids, off, bs, tokens, width, rows, pad, scratch):
    """The step's tables by plain loops over lists."""
    cu, place, slot, table, lens = [0], [], [], [], []
    for i in range(rows):
        real = i < len(new)
        q, n = (max(0, new[i]), ctx[i]) if real else (pad, pad)
        lo, hi = (min(max(off[i], 0), len(ids)), min(max(off[i + 1], 0), len(ids))) if real else (0, 0)
        mine = ids[lo:hi] if real else [scratch] * width
        cu.append(cu[-1] + q)
        lens.append(n)
        table.append((mine + [0] * width)[:width])
        for j in range(q):
            p = n - q + j
            place.append(max(p, 0))
            ok = p >= 0 and p // bs < len(mine) and mine[p // bs] >= 0
            slot.append(mine[p // bs] * bs + p % bs if ok else -1)
    place, slot = (place + [0] * tokens)[:tokens], (slot + [-1] * tokens)[:tokens]
    i32, i64 = torch.int32, torch.int64
    return [torch.tensor(cu, dtype=i32), torch.tensor(lens, dtype=i32), torch.tensor(place, dtype=i64), torch.tensor(slot, dtype=i64),
            torch.tensor(table, dtype=i32).view(rows, width), torch.tensor(cu[1:], dtype=i32) - 1]


def softmax_scale(dim: int) -> float:
    return 1 / math.sqrt(dim)
