"""A group's step is its span over 15, correctly rounded to 32 bits and then to float16: groups whose step another rounding of that
quotient moves by its last bit."""
import numpy as np
import pytest
import torch

import plain_q4 as Q
from nncpu_b200.kernels import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def odd_groups(n, seed):
    """float32 [n, 32]: groups from 0 or so to a span that a product with the rounded 1 / 15 takes to another step; the lanes between lie
    anywhere, and three of them next to a border of two codes."""
    rng = np.random.default_rng(seed)
    found = np.zeros((0, 2), dtype=np.float32)
    while len(found) < n:
        lo = (rng.standard_normal(1 << 20) * 0.5).astype(np.float32)
        hi = lo + rng.uniform(0.3, 9.0, 1 << 20).astype(np.float32)
        span = hi - lo
        differ = (span / np.float32(15)).astype(np.float16) != (span * np.float32(1 / 15)).astype(np.float16)
        found = np.concatenate([found, np.stack([lo, hi], -1)[differ]])
    lo, hi = found[:n, :1], found[:n, 1:]
    x = (lo + (hi - lo) * rng.random((n, 32), dtype=np.float32)).astype(np.float32)
    d = ((hi - lo) / np.float32(15)).astype(np.float16).astype(np.float32)
    for lane, border in ((5, 3.5), (17, 8.5), (30, 13.5)):
        x[:, lane] = (lo + d * np.float32(border))[:, 0]
    x = np.clip(x, lo, hi)
    x[:, 0], x[:, 31] = lo[:, 0], hi[:, 0]
    return x


def cut(x):
    """float32 [..., 32] -> (codes, d, m): the format, with its division."""
    lo, hi = x.min(-1), x.max(-1)
    d, m = ((hi - lo) / np.float32(15)).astype(np.float16), lo.astype(np.float16)
    d32, m32 = d.astype(np.float32)[..., None], m.astype(np.float32)[..., None]
    return np.clip(np.rint((x - m32) * (np.float32(1) / d32)), 0, 15).astype(np.int64), d, m


@pytest.mark.parametrize("D", [32, 64, 96, 128, 256])
def test_steps_are_the_spans_over_fifteen(D):
    """(Of 32, 64 and 128 lanes the append has a kernel of its own, the others take the general one.)"""
    n, NG = 40, D // 32
    k, v = (odd_groups(n * NG, seed).reshape(n, D) for seed in (1, 2))
    table = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    seq, pos = torch.zeros(n, dtype=torch.int32, device=DEV), torch.arange(n, dtype=torch.int32, device=DEV)
    kp = torch.zeros(1, 1, 40 * D, dtype=torch.uint8, device=DEV)
    vp = kp.clone()
    qkv = torch.from_numpy(np.concatenate([np.zeros_like(k), k, v], -1)).to(DEV)
    ops.qk_norm_rope_append_q4(qkv, None, None, 0.0, None, seq, pos, table, kp, vp, torch.empty(n, D, device=DEV), 1, 1, D)
    for pages, x, values in ((kp, k, False), (vp, v, True)):
        row = pages.cpu().numpy()[0, 0]
        c, d, m = cut(x.reshape(n, NG, 32))
        held = row[32 * D:].view(np.float16).reshape(64, NG, 2)[:n]
        assert np.array_equal(held[..., 0], d) and np.array_equal(held[..., 1], m)
        where = Q.nibble_places(D, values)[:n]
        assert np.array_equal((row[where // 2] >> (4 * (where % 2))) & 15, c.reshape(n, D))


def test_a_prompts_codes_are_those_of_the_division():
    """Some 10^4 groups of ordinary numbers, whose odd one has such a step."""
    n, kv, D = 700, 8, 128
    x = (torch.randn(n, 3 * kv * D, generator=torch.Generator().manual_seed(3)) * 2)
    assert (lambda s: ((s / np.float32(15)).astype(np.float16) != (s * np.float32(1 / 15)).astype(np.float16)).sum())(
        np.ptp(x.numpy()[:, kv * D:].reshape(-1, 32), axis=-1)) > 0
    table = torch.arange(11, dtype=torch.int32, device=DEV)[None]
    seq, pos = torch.zeros(n, dtype=torch.int32, device=DEV), torch.arange(n, dtype=torch.int32, device=DEV)
    kp = torch.zeros(11, kv, 40 * D, dtype=torch.uint8, device=DEV)
    vp = kp.clone()
    ops.qk_norm_rope_append_q4(x.to(DEV), None, None, 0.0, None, seq, pos, table, kp, vp, torch.empty(n, kv * D, device=DEV), kv, kv, D)
    k, v = torch.empty(n, kv * D, device=DEV), torch.empty(n, kv * D, device=DEV)
    ops.q4_read(kp, vp, table, seq, pos, k, v)
    for got, part in ((k, x[:, kv * D:2 * kv * D]), (v, x[:, 2 * kv * D:])):
        c, d, m = cut(part.numpy().reshape(n, -1, 32))
        want = c * d.astype(np.float64)[..., None] + m.astype(np.float64)[..., None]
        assert np.array_equal(got.cpu().numpy(), want.astype(np.float32).reshape(n, -1))
