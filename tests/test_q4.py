"""The 4-bit cache without a GPU: the plain format against itself, and what the calls refuse before anything is launched."""
import numpy as np
import pytest
import torch

import plain_q4 as Q
from nncpu_b200.errors import ExtensionError, InvalidArgument
from nncpu_b200.kernels import ops


@pytest.mark.parametrize("D", [32, 96, 128, 256])
def test_a_page_has_a_place_for_every_code(D):
    for values in (False, True):
        assert sorted(Q.nibble_places(D, values).reshape(-1)) == list(range(64 * D))
    assert ops.q4_page_bytes(D) == 40 * D == Q.empty_pages(1, 1, D).shape[-1]


def test_numbers_are_off_by_half_a_step_at_most():
    x = np.random.default_rng(0).standard_normal((50, 128)).astype(np.float32) * 3
    c, d, m = Q.quantise(x)
    assert c.min() == 0 and c.max() == 15
    step = np.repeat(d.astype(np.float64), 32, -1)
    # half a step, and what the least number and (15 times) the step lose to float16
    slack = np.repeat((np.abs(m.astype(np.float64)) + 15 * d) * 2.0 ** -11, 32, -1)
    assert (np.abs(Q.numbers(c, d, m) - x) <= step / 2 + slack).all()


def test_groups_of_one_number_of_nan_and_beyond_the_range():
    x = np.zeros((4, 32), dtype=np.float32)
    x[0] = 1.5
    x[1, 3] = np.nan
    x[2, 0], x[2, 1] = np.inf, -np.inf
    x[3] = 1e-30
    got = Q.numbers(*Q.quantise(x))
    assert (got[0] == 1.5).all() and np.isnan(got[1]).all() and (got[3] == 0).all()
    assert abs(got[2, 0] - 65504) <= 64 and got[2, 1] == -65504 and np.isfinite(got[2]).all()


def test_put_and_read_back():
    x = np.random.default_rng(1).standard_normal((64, 64)).astype(np.float32)
    for values in (False, True):
        pages = Q.empty_pages(1, 1, 64, 0xFF)
        for at in np.random.default_rng(2).permutation(64):
            Q.put(pages, 0, 0, at, x[at], values)
        assert (Q.page_numbers(pages[0, 0], 64, values) == Q.numbers(*Q.quantise(x))).all()


def _args(n=3, heads=4, kv=2, D=64, n_pages=5):
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    return dict(q=torch.zeros(n, heads * D, dtype=torch.bfloat16), k_pages=torch.zeros(n_pages, kv, 40 * D, dtype=torch.uint8),
                v_pages=torch.zeros(n_pages, kv, 40 * D, dtype=torch.uint8), block_table=i(1, 2), tok_seq=i(n), tok_pos=i(n),
                out=torch.zeros(n, heads * D, dtype=torch.bfloat16), n_heads=heads, n_kv=kv, head_dim=D, scale=0.1)


@pytest.mark.parametrize("change", [
    dict(head_dim=48), dict(head_dim=288), dict(n_heads=3), dict(n_kv=0), dict(k_pages=torch.zeros(5, 2, 40 * 32, dtype=torch.uint8)),
    dict(v_pages=torch.zeros(4, 2, 40 * 64, dtype=torch.uint8)), dict(k_pages=torch.zeros(5, 2, 40 * 64)),
    dict(k_pages=torch.zeros(5, 2, 80 * 64, dtype=torch.uint8)[..., ::2]), dict(k_pages=torch.zeros(5 * 2 * 2560 + 1, dtype=torch.uint8)[1:].view(5, 2, 2560)),
    dict(block_table=torch.zeros(2, dtype=torch.int32)), dict(block_table=torch.zeros(1, 0, dtype=torch.int32)),
    dict(block_table=torch.zeros(1, 2, dtype=torch.int64)), dict(tok_pos=torch.zeros(2, dtype=torch.int32)), dict(tok_seq=torch.zeros(3)),
    dict(out=torch.zeros(3, 256)), dict(out=torch.zeros(3, 128, dtype=torch.bfloat16)), dict(q=torch.zeros(3, 255, dtype=torch.bfloat16)),
    dict(keep=4), dict(keep=-1, window=8), dict(cap=-1.0), dict(sinks=torch.zeros(3)), dict(sinks=torch.zeros(4, dtype=torch.float16))])
def test_attention_refuses(change):
    with pytest.raises(InvalidArgument, match="attention_q4"):
        ops.attention_q4(**{**_args(), **change})


def test_there_is_no_cpu_path():
    with pytest.raises((ExtensionError, InvalidArgument)):
        ops.attention_q4(**_args(), scratch=torch.zeros(1 << 16))


@pytest.mark.parametrize("change", [dict(n_seqs=0), dict(n_seqs=2), dict(longest=0), dict(status=torch.zeros(1)), dict(status=torch.zeros(0, dtype=torch.int32)),
                                    dict(block_table=torch.zeros(0, 2, dtype=torch.int32)), dict(cu_seqlens=torch.zeros(2)), dict(head_dim=40)])
def test_prompt_attention_refuses(change):
    a = dict(_args(), cu_seqlens=torch.zeros(2, dtype=torch.int32), n_seqs=1, longest=128, status=torch.zeros(1, dtype=torch.int32))
    with pytest.raises(InvalidArgument, match="attention_q4"):
        ops.attention_q4_prompt(**{**a, **change})


@pytest.mark.parametrize("change", [
    dict(qkv=torch.zeros(3, 511)), dict(qkv=torch.zeros(2, 512)), dict(q_out=torch.zeros(3, 128)), dict(head_dim=16), dict(q_gamma=torch.ones(32)),
    dict(k_gamma=torch.ones(64, dtype=torch.bfloat16)), dict(cos_sin=torch.zeros(3, 33, 2)), dict(cos_sin=torch.zeros(2, 32, 2)),
    dict(cos_sin=torch.zeros(3, 32, 2, dtype=torch.float64)), dict(tok_pos=torch.zeros(3)), dict(k_pages=torch.zeros(5, 1, 2560, dtype=torch.uint8)),
    dict(block_table=torch.zeros(1, 2, dtype=torch.int64)), dict(tok_seq=torch.zeros(2, dtype=torch.int32))])
def test_append_refuses(change):
    a = _args()
    args = dict(qkv=torch.zeros(3, 512), q_gamma=torch.ones(64), k_gamma=torch.ones(64), eps=1e-6, cos_sin=torch.zeros(3, 32, 2), tok_seq=a["tok_seq"],
                tok_pos=a["tok_pos"], block_table=a["block_table"], k_pages=a["k_pages"], v_pages=a["v_pages"], q_out=torch.zeros(3, 256), n_heads=4,
                n_kv=2, head_dim=64)
    with pytest.raises(InvalidArgument, match="qk_norm_rope_append_q4"):
        ops.qk_norm_rope_append_q4(**{**args, **change})


@pytest.mark.parametrize("change", [dict(k_out=torch.zeros(3, 64)), dict(v_out=torch.zeros(3, 128, dtype=torch.bfloat16)), dict(v_out=torch.zeros(4, 128)),
                                    dict(tok_pos=torch.zeros(2, dtype=torch.int32))])
def test_read_refuses(change):
    a = _args()
    args = dict(k_pages=a["k_pages"], v_pages=a["v_pages"], block_table=a["block_table"], tok_seq=a["tok_seq"], tok_pos=a["tok_pos"],
                k_out=torch.zeros(3, 128), v_out=torch.zeros(3, 128))
    with pytest.raises(InvalidArgument, match="q4_read"):
        ops.q4_read(**{**args, **change})


@pytest.mark.parametrize("change", [
    dict(logits=torch.zeros(10)), dict(logits=torch.zeros(2, 0)), dict(logits=torch.zeros(2, 10, dtype=torch.float16)), dict(targets=torch.zeros(2)),
    dict(targets=torch.zeros(3, dtype=torch.int32)), dict(logprobs=torch.zeros(2, dtype=torch.bfloat16)), dict(entropy=torch.zeros(1)),
    dict(top=None), dict(ids=None), dict(top=torch.zeros(2, 11), ids=torch.zeros(2, 11, dtype=torch.int32)),
    dict(top=torch.zeros(2, 0), ids=torch.zeros(2, 0, dtype=torch.int32)), dict(top=torch.zeros(2, 4)), dict(ids=torch.zeros(2, 3)),
    dict(logits=torch.zeros(2, 200), top=torch.zeros(2, 33), ids=torch.zeros(2, 33, dtype=torch.int32)), dict(entropy=torch.zeros(2, device="meta"))])
def test_logprobs_refuse(change):
    args = dict(logits=torch.zeros(2, 10), targets=torch.zeros(2, dtype=torch.int32), logprobs=torch.zeros(2), entropy=torch.zeros(2),
                top=torch.zeros(2, 3), ids=torch.zeros(2, 3, dtype=torch.int32))
    with pytest.raises((InvalidArgument, ExtensionError)):
        ops.token_logprobs(**{**args, **change})
