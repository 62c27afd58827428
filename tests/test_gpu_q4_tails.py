"""Rows whose result is a tail's: one key far above the others, whose value is zero (as a sequence's first token often is)."""
import numpy as np
import pytest
import torch

import plain_q4 as Q
from nncpu_b200.kernels import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def one_high_key(n, kv, D, above, seed):
    """Pages of one sequence of n tokens, key 0 ``above`` over all others for queries of 8 in lane 0 and a scale of 1/8; its value is 0,
    the others' lie around 1.  (k_pages, v_pages, table, k, v as the pages hold them)."""
    rng = np.random.default_rng(seed)
    k, v = 0.05 * rng.standard_normal((n, kv, D)), 1 + 0.2 * rng.standard_normal((n, kv, D))
    k[:, :, :32] = 0.0
    k[0, :, 0], v[0] = above, 0.0
    k, v = k.astype(np.float32), v.astype(np.float32)
    pages = -(-n // 64)
    kp, vp = Q.empty_pages(pages, kv, D), Q.empty_pages(pages, kv, D)
    for t in range(n):
        for h in range(kv):
            Q.put(kp, t // 64, h, t % 64, k[t, h], False)
            Q.put(vp, t // 64, h, t % 64, v[t, h], True)
    held = [np.stack([np.concatenate([Q.page_numbers(p[i, h], D, values) for i in range(pages)])[:n] for h in range(kv)], 1)
            for p, values in ((kp, False), (vp, True))]
    return kp, vp, np.arange(pages, dtype=np.int32)[None], held[0], held[1]


@pytest.mark.parametrize("new", [260, 100, 24, 1])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("above", [8.0, 14.0, 17.5])
def test_a_tail_below_a_key_without_value(above, D, new):
    """The weights of the tail are e^-above of the greatest, 2^-25.2 at 17.5.  The greatest of a step is held between 2^8 and 2^11
    or more, so the tail's lie above 2^-17.2 and float16's spacing of 2^-24 there moves one by 2^-7.8 at most; a key's number is rounded to 11
    bits, which moves a score by 2^-11 of its size; the result is rounded to 8."""
    n, heads, kv = 260, 4, 2
    kp, vp, table, k, v = one_high_key(n, kv, D, above, 5)
    q = 0.1 * torch.randn(new, heads, D, generator=torch.Generator().manual_seed(6))
    q[:, :, 0] = 8.0
    q = q.reshape(new, heads * D).bfloat16()
    pos = np.arange(n - new, n, dtype=np.int32)
    kpc, vpc, bt, ts, tp, cu = Q.as_cuda(kp, vp, table, np.zeros(new, np.int32), pos, np.array([0, new], np.int32))
    out, status = torch.empty(new, heads * D, dtype=torch.bfloat16, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.attention_q4_prompt(q.to(DEV), kpc, vpc, bt, cu, ts, tp, out, 1, heads, kv, D, 0.125, n, status)
    assert int(status) == 0
    for t in range(new):
        want, mass, _ = Q.attend(q[t].double().numpy().reshape(heads, D), k, v, pos[t], 0.125)
        got = out[t].double().cpu().numpy().reshape(heads, D)
        tol = (2.0 ** -7.8 + 2 * (above + 1) * 2.0 ** -11 + 2.0 ** -10 + 2.0 ** -8) * mass
        assert (np.abs(got - want) <= tol).all(), (t, float((np.abs(got - want) / (mass + 1e-300)).max()))
        assert pos[t] == 0 or (want[:, :32] > 0).all()
