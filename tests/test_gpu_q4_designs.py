"""Designs other than grouped-query attention with a rotation of whole heads, over a cache of 4 bits: slopes by distance, query temperatures, layers
with a state beside layers with keys, blocks of keys, partial rotations, layers that run several times.  The plain
model attends to the numbers that the cache holds (see test_gpu_q4_model)."""
import numpy as np
import pytest
import torch

import plain_romepel
import plain_zevivik
import test_gpu_romepel as R
import test_gpu_zevivik as Z
from gpu_util import TOL, check
from nncpu_b200 import Engine, Model
from nncpu_b200.cache.cache import KVGroup

pytestmark = pytest.mark.gpu

DESIGNS = {
    "romepel": (R, plain_romepel, "biased_attention",
                {"architecture": "Romepel", "vocab": 310, "width": 192, "max_positions": 700, "norm": {"eps": 3e-6},
                 "layers": [R.att(4, 2, 64, 64, 0.125, window=100, q_temp=(0.4, 32), ff=256), R.gla(2, 64, 64, 12.0, 8, ff=128),
                            R.att(3, 1, 96, 96, 0.1, q_temp=(0.7, 5), ff=128), R.att(2, 1, 128, 128, 0.09, window=256, ff=128)]}),
    "zevivik": (Z, plain_zevivik, "masked_attention",
                {"architecture": "Zevivik", "vocab": 310, "width": 192, "norm": {"eps": 1e-5}, "embedding": {"scale": 3.0},
                 "loop": {"start": 0, "stop": 2, "times": 2},
                 "layers": [Z.att(4, 2, 64, 64, 0.125, size=100, rot=(1000000.0, 64), mlp=Z.dense(256)),
                            Z.att(2, 1, 128, 128, 0.09, size=256, rot=(10000.0, 64), mlp=Z.dense(128)),
                            Z.att(3, 3, 32, 32, 0.2, mlp=Z.dense(128))]}),
}


@pytest.mark.parametrize("dtype", R.DTYPES)
@pytest.mark.parametrize("name", DESIGNS)
def test_whole_in_portions_and_one_by_one(tmp_path, monkeypatch, name, dtype):
    tests, plain, attention, cfg_dict = DESIGNS[name]
    folder = tests.write_folder(tmp_path / name, cfg_dict, 5, R.STORE[dtype], sharpen=1.0)
    cfg, w = plain.load(folder)
    monkeypatch.setattr(KVGroup, "trim", lambda self, slot, length: None)     # (windows keep their pages, for the plain model to read)
    engine = Engine(Model.load(folder, dtype=dtype), max_tokens=64 * 16, kv_dtype="q4")
    users = [u for u in range(100) if u < len(engine.cache._entry_group) and engine.cache.group_of(u) is not None]
    own_attention = getattr(plain, attention)

    def expected(tokens, slot):
        user = iter(users)

        def attend(q, k, v, *rest):
            held = [t.double().cpu().numpy() for t in engine.cached(slot, next(user))]
            for own, h in zip((k, v), held):
                span = np.ptp(own.reshape(*own.shape[:-1], -1, 32), -1).repeat(32, -1)
                # half a step, what the group's two numbers lose to half precision, and the run's own rounding of the number
                assert (np.abs(h - own) <= span / 30 + (np.abs(own) + 2 * span) * 2.0 ** -11 + 2 * TOL[dtype] * np.abs(own).max()).all()
            return own_attention(q, *held, *rest)
        with monkeypatch.context() as m:
            m.setattr(plain, attention, attend)
            logits = plain.forward(cfg, w, tokens)
        assert next(user, None) is None          # (every layer's keys and values have been read)
        return logits
    toks = np.random.RandomState(1).randint(0, 310, size=330).tolist()
    a = engine.alloc_slot()
    whole = engine.step([a], [toks], [list(range(330))]).clone()
    check(whole, expected(toks, a), TOL[dtype], "whole")
    b = engine.alloc_slot()
    parts = [engine.step([b], [toks[i:j]], [list(range(j - i))]).clone() for i, j in ((0, 1), (1, 130), (130, 149), (149, 300))]
    parts += [engine.step([b], [[t]]).clone() for t in toks[300:]]
    check(torch.cat(parts), expected(toks, b), TOL[dtype], "in portions")
