"""An engine over a cache of 4 bits: what captured portions hold, and slots without tokens."""
import gc

import pytest
import torch

from gpu_util import TOL, check
from nncpu_b200 import Engine, Model
from nncpu_b200.kernels import ops
from test_gpu_q4_model import DTYPES, STORE, ids, plain  # noqa: F401
from tiny import make_folder

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    root = tmp_path_factory.mktemp("q4engine")
    return {d: make_folder(root / d, "G", seed=7, store_dtype=STORE[d]) for d in DTYPES}


@pytest.mark.parametrize("dtype", DTYPES)
def test_captured_portions_of_all_sizes_share_what_the_keys_are_taken_out_to(folders, plain, dtype):
    """Portions of one sequence of 33 to 64, 128 and 256 tokens are three graphs; the keys and values of the whole context, as
    numbers, lie in one place for all of them."""
    context = 16384
    engine = Engine(Model.load(folders[dtype], dtype=dtype), max_tokens=context, kv_dtype="q4", max_step_tokens=256)
    spec = engine.model.blocks[0].mixers()[0].spec
    taken_out = ops.attention_q4_prompt_scratch_bytes(256, 1, spec.n_heads, spec.n_kv_heads, spec.head_dim, STORE[dtype], context)
    assert taken_out >= 2 * context * spec.n_kv_heads * spec.head_dim * STORE[dtype].itemsize
    slot = engine.alloc_slot()
    used, rows, text = [], [], []
    for n in (60, 120, 250, 50, 90, 200, 20, 5):
        text += ids(n, n)
        rows.append(engine.step([slot], [text[-n:]])[0].cpu())
        gc.collect()
        torch.cuda.synchronize()
        used.append((len(text), torch.cuda.memory_allocated()))
    assert sorted(engine.graphs.prompts) == [16, 32, 64, 128, 256]
    want = plain(folders[dtype], text, engine, slot)[[n - 1 for n, _ in used]]
    check(torch.stack(rows), want, TOL[dtype], "portions")
    assert all(b[1] - a[1] < taken_out // 4 for a, b in zip(used, used[1:])), used


@pytest.mark.parametrize("kv_dtype", [None, "q4"])
def test_a_slot_without_tokens_holds_nothing(folders, kv_dtype):
    engine = Engine(Model.load(folders["bfloat16"]), max_tokens=256, kv_dtype=kv_dtype)
    k, v = engine.cached(engine.alloc_slot())
    assert k.shape == v.shape == (0, 2, 128) and k.dtype == v.dtype == torch.float32
