"""A group's step is its span times 1 / 15, each rounded to 32 bits, then rounded to float16: what dividing a tensor on the device by the number 15
computes, too.  A division rounded once gives one group in 15 000 another last bit; these are such groups."""
import numpy as np
import pytest
import torch

import plain_q4 as Q
from nncpu_b200.kernels import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def odd_groups(n, seed):
    """float32 [n, 32]: groups whose span's product and quotient give different steps; the lanes between lie anywhere, three of them
    next to a border of two codes."""
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
    d = ((hi - lo) * np.float32(1 / 15)).astype(np.float16).astype(np.float32)
    for lane, border in ((5, 3.5), (17, 8.5), (30, 13.5)):
        x[:, lane] = (lo + d * np.float32(border))[:, 0]
    x = np.clip(x, lo, hi)
    x[:, 0], x[:, 31] = lo[:, 0], hi[:, 0]
    return x


@pytest.mark.parametrize("D", [32, 64, 96, 128, 256])
def test_steps_and_codes_of_odd_groups(D):
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
        c, d, m = Q.quantise(x)
        held = row[32 * D:].view(np.float16).reshape(64, NG, 2)[:n]
        assert np.array_equal(held[..., 0], d) and np.array_equal(held[..., 1], m)
        where = Q.nibble_places(D, values)[:n]
        assert np.array_equal((row[where // 2] >> (4 * (where % 2))) & 15, c)
        g = torch.from_numpy(x).to(DEV).view(n, NG, 32)
        assert np.array_equal((((g.amax(-1) - g.amin(-1)) / 15).half()).cpu().numpy(), d)
