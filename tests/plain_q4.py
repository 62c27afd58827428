"""The 4-bit cache and the attention over it, plainly: NumPy in 64 bits (with the roundings that the format itself has), code by code
from the layout's description."""
from __future__ import annotations

import numpy as np
import torch

PAGE, GROUP = 64, 32


def quantise(x):
    """float32 [..., D] -> (codes [..., D] int, d, m float16 [..., D / 32])."""
    x = np.asarray(x, dtype=np.float32)
    g = x.reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        g = np.clip(g, np.float32(-65504), np.float32(65504))       # (a NaN stays one)
        lo, hi = g.min(-1), g.max(-1)                               # (of a group with a NaN: NaN)
        d = ((hi - lo) * np.float32(1 / 15)).astype(np.float16)
        m = lo.astype(np.float16)
        d32, m32 = d.astype(np.float32), m.astype(np.float32)
        inv = np.where(d32 > 0, np.float32(1) / np.where(d32 > 0, d32, np.float32(1)), np.float32(0))
        c = np.rint((g - m32[..., None]) * inv[..., None])
    c = np.clip(np.nan_to_num(c, nan=0.0), 0, 15).astype(np.int64)
    return c.reshape(x.shape), d, m


def numbers(c, d, m):
    """float64 [..., D]: d c + m."""
    return c * np.repeat(d.astype(np.float64), GROUP, -1) + np.repeat(m.astype(np.float64), GROUP, -1)


def nibble_places(D: int, values: bool):
    """[64, D]: in which nibble of a page (from its first byte's lower one) the code of (position, lane) lies."""
    tok, lane = np.arange(PAGE)[:, None], np.arange(D)[None, :]
    NG, g, x = D // GROUP, lane // GROUP, lane % GROUP
    if values:
        word = ((tok // 8 * 8 + x // 4) * 4 + tok % 8 // 2) * NG + g
        return word * 8 + tok % 2 * 4 + x % 4
    return (tok * 4 * NG + x // 8 * NG + g) * 8 + x % 8


def empty_pages(n_pages: int, n_kv: int, D: int, fill: int = 0):
    return np.full((n_pages, n_kv, 40 * D), fill, dtype=np.uint8)


def put(pages, page: int, head: int, at: int, x, values: bool) -> None:
    """Writes the float32 vector x [D] to position ``at`` of a page."""
    D = len(x)
    c, d, m = quantise(x)
    where = nibble_places(D, values)[at]
    row = pages[page, head]
    for n, code in zip(where, c):
        b = row[n // 2]
        row[n // 2] = (b & 0xF0) | code if n % 2 == 0 else (b & 0x0F) | (code << 4)
    scales = row[32 * D:].view(np.float16).reshape(PAGE, D // GROUP, 2)
    scales[at, :, 0], scales[at, :, 1] = d, m


def page_numbers(page_row, D: int, values: bool):
    """uint8 [40 D] -> float64 [64, D]."""
    n = nibble_places(D, values)
    c = (page_row[n // 2] >> (4 * (n % 2))) & 15
    s = page_row[32 * D:].view(np.float16).reshape(PAGE, D // GROUP, 2)
    return numbers(c.astype(np.int64), s[..., 0], s[..., 1])


def filled_cache(lens, n_kv: int, D: int, seed: int, spare: int = 3, fill: int = 0xFF):
    """Random sequences of the given lengths in shuffled pages; what no sequence holds is ``fill`` (0xFF: codes of 15 and NaN for
    d and m).  Returns (k_pages, v_pages, table int32, ks, vs): ks[b], vs[b] float64 [len, n_kv, D], the numbers that the pages hold."""
    rng = np.random.default_rng(seed)
    per = [max(1, -(-n // PAGE)) for n in lens]
    n_pages = sum(per) + spare
    order = list(rng.permutation(n_pages))
    kp, vp = empty_pages(n_pages, n_kv, D, fill), empty_pages(n_pages, n_kv, D, fill)
    table = np.full((len(lens), max(per)), -1, dtype=np.int32)
    ks, vs = [], []
    places = [nibble_places(D, False), nibble_places(D, True)]
    for b, n in enumerate(lens):
        got = []
        ids = [order.pop() for _ in range(per[b])]
        table[b, :per[b]] = ids
        for pages, values in ((kp, False), (vp, True)):
            x = rng.standard_normal((n, n_kv, D)).astype(np.float32)
            x *= 1 + 3 * (rng.random((1, n_kv, D)) < 0.05)
            c, d, m = quantise(x)
            for j, page in enumerate(ids):
                rows = slice(j * PAGE, min(n, (j + 1) * PAGE))
                count = rows.stop - rows.start
                if count <= 0:
                    continue
                for h in range(n_kv):
                    row = pages[page, h]
                    nib = np.stack([row[:32 * D] & 15, row[:32 * D] >> 4], -1).reshape(-1)
                    nib[places[values][:count]] = c[rows, h]
                    row[:32 * D] = nib[0::2] | (nib[1::2] << 4)
                    s = row[32 * D:].view(np.float16).reshape(PAGE, D // GROUP, 2)
                    s[:count, :, 0], s[:count, :, 1] = d[rows, h], m[rows, h]
            got.append(numbers(c, d, m))
        ks.append(got[0])
        vs.append(got[1])
    return kp, vp, table, ks, vs


def visible(pos: int, n: int, window: int, keep: int):
    """Which of the keys 0..n-1 the query at ``pos`` sees: window > 0 the last so many, < 0 those of its own block of -window."""
    key = np.arange(n)
    first = max(0, pos + 1 - window) if window > 0 else pos // -window * -window if window < 0 else 0
    return (key <= pos) & ((key >= first) | (key < keep))


def attend(q, k, v, pos: int, scale: float, window: int = 0, keep: int = 0, slope_base: float = 0.0, sinks=None, cap: float = 0.0,
           gate=None):
    """One token: q [n_heads, D], k, v [n, n_kv, D] (float64).  Returns (out [n_heads, D], mass [n_heads, D] = sum of p |v|,
    reach [n_heads] = greatest scale * sum |q k| among the keys seen)."""
    q = np.asarray(q, dtype=np.float64)
    n_heads, n_kv = q.shape[0], k.shape[1]
    see = visible(pos, k.shape[0], window, keep)
    out, mass, reach = np.zeros_like(q), np.zeros_like(q), np.zeros(n_heads)
    for h in range(n_heads):
        kk, vv = k[see, h // (n_heads // n_kv)], v[see, h // (n_heads // n_kv)]
        if not len(kk):
            continue
        z = kk @ q[h] * scale
        reach[h] = (np.abs(kk) @ np.abs(q[h])).max() * abs(scale)
        if cap:
            z = cap * np.tanh(z / cap)
        if slope_base:
            z = z - 2.0 ** (-slope_base * (h + 1) / n_heads) * (pos - np.arange(k.shape[0])[see])
        m = z.max()
        e = np.exp(z - m)
        total = e.sum() + (np.exp(sinks[h] - m) if sinks is not None else 0.0)
        f = 1.0 if gate is None else 1.0 / (1.0 + np.exp(-gate[h]))
        out[h] = e @ vv / total * f
        mass[h] = e @ np.abs(vv) / total * f
    return out, mass, reach


def as_cuda(*arrays):
    return [torch.from_numpy(np.ascontiguousarray(a)).cuda() for a in arrays]
