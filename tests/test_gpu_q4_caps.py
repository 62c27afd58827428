"""Score caps that are far beyond the scores, over a cache of 4 bits: the error may not grow with the cap."""
import numpy as np
import pytest
import torch

import plain_q4 as Q
from nncpu_b200.kernels import ops
pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32


def rand(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def check(out, q, ks, vs, seq, pos, dt, heads, scale, cap):
    """Every row against 64 bits.  A score is a sum of D products in 32 bits; its cap is a quotient, a tanh of two units in the last
    place and a product, 2^-21 of the score together, whatever the cap; a weight is the exponential of a difference of scores, an output a
    sum over n keys, all in 32 bits.  A bfloat16 result is rounded once."""
    for t in range(len(seq)):
        k, v = ks[seq[t]], vs[seq[t]]
        D = k.shape[-1]
        row, qt = out[t].double().cpu().numpy().reshape(heads, D), q[t].double().cpu().numpy().reshape(heads, D)
        want, mass, _ = Q.attend(qt, k, v, pos[t], scale, cap=cap)
        wide = np.abs(k[:pos[t] + 1]) + np.repeat(np.ptp(k[:pos[t] + 1].reshape(pos[t] + 1, -1, D // 32, 32), -1), 32, -1)
        reach = np.array([(wide[:, h // (heads // k.shape[1])] @ np.abs(qt[h])).max() * scale for h in range(heads)])[:, None]
        tol = mass * (2 * reach * ((D + 16) * 2.0 ** -24 + 2.0 ** -21) + 2 * (pos[t] + 65) * 2.0 ** -24)
        if dt == BF16:
            tol = tol + 2.0 ** -8 * np.abs(want)
        err = np.abs(row - want)
        assert np.isfinite(row).all() and (err <= tol + 1e-30).all(), (t, float((err / (tol + 1e-30)).max()))


CAPS = [4097.0, 65536.0, 1e6, 1e7]


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("cap", CAPS)
@pytest.mark.parametrize("heads,kv,D", [(8, 2, 128), (4, 4, 64), (3, 1, 160)])
def test_single_tokens(heads, kv, D, cap, dt):
    lens = [300, 1, 64, 900]
    kp, vp, table, ks, vs = Q.filled_cache(lens, kv, D, 1)
    seq, pos = np.arange(4, dtype=np.int32), np.array(lens, np.int32) - 1
    q = (3 * rand(4, heads * D)).to(dt).to(DEV)
    out = torch.empty_like(q)
    ops.attention_q4(q, *Q.as_cuda(kp, vp, table, seq, pos), out, heads, kv, D, D ** -0.5, cap=cap)
    check(out, q, ks, vs, seq, pos, dt, heads, D ** -0.5, cap)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("cap", CAPS)
@pytest.mark.parametrize("lens,new", [([300], [24]), ([300, 90], [130, 60]), ([200], [200])])
def test_prompts(lens, new, cap, dt):
    heads, kv, D = 8, 2, 128
    kp, vp, table, ks, vs = Q.filled_cache(lens, kv, D, 2)
    seq = np.repeat(np.arange(len(lens)), new).astype(np.int32)
    pos = np.concatenate([np.arange(n - m, n) for n, m in zip(lens, new)]).astype(np.int32)
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    q = 3 * rand(len(seq), heads * D, seed=1)
    q[5] *= cap            # (one token's scores pass the cap, beside others of its tile that are far below it)
    q = q.to(dt).to(DEV)
    out, status = torch.empty_like(q), torch.zeros(1, dtype=torch.int32, device=DEV)
    kpc, vpc, bt, ts, tp, cuc = Q.as_cuda(kp, vp, table, seq, pos, cu)
    ops.attention_q4_prompt(q, kpc, vpc, bt, cuc, ts, tp, out, len(lens), heads, kv, D, D ** -0.5, max(lens), status, cap=cap)
    assert int(status) == 0
    check(out, q, ks, vs, seq, pos, dt, heads, D ** -0.5, cap)


@pytest.mark.parametrize("dt", [F32, BF16])
def test_the_stated_scratch_is_enough(dt):
    heads, kv, D, n = 8, 2, 128, 60
    kp, vp, table, ks, vs = Q.filled_cache([900], kv, D, 3)
    seq, pos, cu = np.zeros(n, np.int32), np.arange(900 - n, 900, dtype=np.int32), np.array([0, n], np.int32)
    kpc, vpc, bt, ts, tp, cuc = Q.as_cuda(kp, vp, table, seq, pos, cu)
    q = rand(n, heads * D, seed=4).to(dt).to(DEV)
    out, status = torch.empty_like(q), torch.zeros(1, dtype=torch.int32, device=DEV)
    scratch = torch.empty(ops.attention_q4_prompt_scratch_bytes(n, 1, heads, kv, D, dt, 900, 0.0, 1e6), dtype=torch.uint8, device=DEV)
    ops.attention_q4_prompt(q, kpc, vpc, bt, cuc, ts, tp, out, 1, heads, kv, D, D ** -0.5, 900, status, cap=1e6, scratch=scratch)
    check(out, q, ks, vs, seq, pos, dt, heads, D ** -0.5, 1e6)
    one = torch.empty(max(1, ops.attention_q4_scratch_floats(n, heads, kv, D, dt, 900, cap=1e6)), device=DEV)
    ops.attention_q4(q, kpc, vpc, bt, ts, tp, out, heads, kv, D, D ** -0.5, cap=1e6, longest=900, scratch=one)
    check(out, q, ks, vs, seq, pos, dt, heads, D ** -0.5, 1e6)
