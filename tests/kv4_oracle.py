"""The 4-bit paged cache in plain numpy, from the format's definition: what the
tests of the serving operators compare with.  Nothing here uses the package."""
import math

import numpy as np

F32 = np.float32


def block_bytes(hd, page, group):
    return page * (hd + 8 * (hd // group))


def quantise(x, group):
    """x fp32 [n, heads, hd] -> codes [n, heads, hd] (0 .. 15), scale and zero
    float16 [n, heads, groups], held bool [n, heads]."""
    n, heads, hd = x.shape
    g = x.astype(F32).reshape(n, heads, hd // group, group)
    finite = np.isfinite(g).all(axis=(2, 3))
    g = np.where(finite[..., None, None], g, F32(0))
    with np.errstate(over="ignore"):
        zero = g.min(-1).astype(np.float16)
    z = zero.astype(F32)
    with np.errstate(invalid="ignore", over="ignore"):
        r = np.maximum((g.max(-1) - z) / F32(15), F32(0))
    # seven significant bits, rounded up
    s = ((r.view(np.uint32) + np.uint32(0x1FFFF)) & np.uint32(0xFFFE0000)).view(F32)
    s = np.where(s < F32(2.0**-17), np.ceil(s * F32(2.0**24)) * F32(2.0**-24), s).astype(F32)
    held = finite & (np.isfinite(z) & (s <= 4032)).all(-1)
    safe = np.where(s > 0, s, F32(1))[..., None]
    with np.errstate(invalid="ignore", over="ignore"):
        q = np.where(s[..., None] > 0, np.rint((g - z[..., None]) / safe), F32(0))
        codes = np.where(held[..., None, None], np.clip(q, 0, 15), 0).astype(np.uint8).reshape(n, heads, hd)
        return codes, np.where(s <= 4032, s, 0).astype(np.float16), np.where(np.isfinite(z), zero, np.float16(0)), held


def pack(k, v, pages, page, hd, group):
    """The cache's bytes from (codes, scale, zero) of every slot, k and v: codes
    [pages * page, heads, hd], scale and zero [pages * page, heads, groups]."""
    heads, groups = k[0].shape[1], hd // group
    data = np.zeros((pages, heads, block_bytes(hd, page, group)), np.uint8)
    words = data.view(np.uint32)
    halves = data.view(np.float16)
    kc, vc, ks = 0, page * hd // 8, page * hd // 4           # first word of each part
    vs = ks + page * groups
    for p in range(pages):
        for tok in range(page):
            slot = p * page + tok
            for c in range(hd):
                s, t, e = c // 32, c // 8 % 4, c % 8
                words[p, :, kc + tok * hd // 8 + t * (hd // 32) + s] |= \
                    k[0][slot, :, c].astype(np.uint32) << np.uint32(4 * (e // 2 + 4 * (e % 2)))
                words[p, :, vc + (tok // 4 * (hd // 8) + c // 8) * 4 + tok % 4] |= \
                    v[0][slot, :, c].astype(np.uint32) << np.uint32(4 * (c % 8))
            for g in range(groups):
                at = 2 * (ks + tok * groups + g)
                halves[p, :, at], halves[p, :, at + 1] = k[1][slot, :, g], k[2][slot, :, g]
                at = 2 * vs + (tok // 4 * groups + g) * 8 + tok % 4
                halves[p, :, at], halves[p, :, at + 4] = v[1][slot, :, g], v[2][slot, :, g]
    return data


def bytes_of(slots, pages, page, heads, hd, group):
    """A mask, 0xFF in every byte that belongs to one of the slots."""
    ones = np.full((pages * page, heads, hd // group), 0, np.uint16)
    ones[slots] = 0xFFFF
    codes = np.zeros((pages * page, heads, hd), np.uint8)
    codes[slots] = 15
    part = (codes, ones.view(np.float16), ones.view(np.float16))
    return pack(part, part, pages, page, hd, group)


def values(parts, group):
    """float64 values of (codes, scale, zero)."""
    codes, scale, zero = parts
    return codes.astype(np.float64) * np.repeat(scale.astype(np.float64), group, -1) + \
        np.repeat(zero.astype(np.float64), group, -1)


def rope(x, cos, sin):
    """Rotate-half RoPE in fp32, every step rounded: x [n, heads, hd], cos / sin [n, hd]."""
    h = x.shape[-1] // 2
    c, s = cos[:, None].astype(F32), sin[:, None].astype(F32)
    other = np.concatenate((-x[..., h:], x[..., :h]), -1).astype(F32)
    return (x.astype(F32) * c).astype(F32) + (other * s).astype(F32)


def attend(q, k, v, lengths, starts, table, page, scale=None):
    """float64 attention: q [rows, heads, hd], k / v [slots, kv heads, hd]; rows of no
    request and rows before the first token are zero."""
    q = q.astype(np.float64)
    rows, heads, hd = q.shape
    each = heads // k.shape[1]
    scale = 1.0 / math.sqrt(hd) if scale is None else scale
    out = np.zeros_like(q)
    for b, n in enumerate(lengths):
        lo, hi = starts[b], starts[b + 1]
        slots = np.array([table[b][i // page] * page + i % page for i in range(n)], dtype=np.int64)
        for r in range(lo, hi):
            seen = slots[:max(0, n - (hi - lo) + (r - lo) + 1)]
            if seen.size == 0:
                continue
            for h in range(heads):
                s = k[seen, h // each] @ q[r, h] * scale
                p = np.exp(s - s.max())
                out[r, h] = p @ v[seen, h // each] / p.sum()
    return out
