"""Tensors of another number of dimensions are refused like any other wrong size, before anything is launched (no GPU)."""
import pytest
import torch

from nncpu_b200.errors import InvalidArgument
from nncpu_b200.kernels import ops
from test_q4 import _args


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(128, dtype=torch.bfloat16)), dict(q=torch.zeros(3, 4, 64, dtype=torch.bfloat16)), dict(q=torch.zeros((), dtype=torch.bfloat16)),
    dict(out=torch.zeros(3, 4, 64, dtype=torch.bfloat16)), dict(k_pages=torch.zeros(2560, dtype=torch.uint8)), dict(v_pages=torch.zeros((), dtype=torch.uint8)),
    dict(block_table=torch.zeros((), dtype=torch.int32))])
def test_attention(change):
    with pytest.raises(InvalidArgument, match="attention_q4"):
        ops.attention_q4(**{**_args(), **change})
    a = dict(_args(), cu_seqlens=torch.zeros(2, dtype=torch.int32), n_seqs=1, longest=128, status=torch.zeros(1, dtype=torch.int32))
    with pytest.raises(InvalidArgument, match="attention_q4_prompt"):
        ops.attention_q4_prompt(**{**a, **change})


@pytest.mark.parametrize("change", [dict(cu_seqlens=torch.zeros((), dtype=torch.int32)), dict(cu_seqlens=torch.zeros(1, 2, dtype=torch.int32))])
def test_prompts(change):
    a = dict(_args(), cu_seqlens=torch.zeros(2, dtype=torch.int32), n_seqs=1, longest=128, status=torch.zeros(1, dtype=torch.int32))
    with pytest.raises(InvalidArgument, match="attention_q4_prompt"):
        ops.attention_q4_prompt(**{**a, **change})


@pytest.mark.parametrize("change", [
    dict(qkv=torch.zeros(512)), dict(qkv=torch.zeros(())), dict(q_out=torch.zeros(())), dict(q_out=torch.zeros(3, 4, 64)), dict(cos_sin=torch.zeros(192)),
    dict(cos_sin=torch.zeros(())), dict(k_pages=torch.zeros(2560, dtype=torch.uint8)), dict(k_pages=torch.zeros((), dtype=torch.uint8)),
    dict(block_table=torch.zeros((), dtype=torch.int32))])
def test_append(change):
    a = _args()
    args = dict(qkv=torch.zeros(3, 512), q_gamma=torch.ones(64), k_gamma=torch.ones(64), eps=1e-6, cos_sin=torch.zeros(3, 32, 2), tok_seq=a["tok_seq"],
                tok_pos=a["tok_pos"], block_table=a["block_table"], k_pages=a["k_pages"], v_pages=a["v_pages"], q_out=torch.zeros(3, 256), n_heads=4,
                n_kv=2, head_dim=64)
    with pytest.raises(InvalidArgument, match="qk_norm_rope_append_q4"):
        ops.qk_norm_rope_append_q4(**{**args, **change})


@pytest.mark.parametrize("change", [
    dict(k_out=torch.zeros(128)), dict(k_out=torch.zeros(())), dict(k_out=torch.zeros(3, 2, 64)), dict(v_out=torch.zeros(128)),
    dict(k_pages=torch.zeros(2560, dtype=torch.uint8)), dict(k_pages=torch.zeros((), dtype=torch.uint8)),
    dict(k_pages=torch.zeros(5, 0, 2560, dtype=torch.uint8), v_pages=torch.zeros(5, 0, 2560, dtype=torch.uint8)),
    dict(block_table=torch.zeros((), dtype=torch.int32))])
def test_read(change):
    a = _args()
    args = dict(k_pages=a["k_pages"], v_pages=a["v_pages"], block_table=a["block_table"], tok_seq=a["tok_seq"], tok_pos=a["tok_pos"],
                k_out=torch.zeros(3, 128), v_out=torch.zeros(3, 128))
    with pytest.raises(InvalidArgument, match="q4_read"):
        ops.q4_read(**{**args, **change})


@pytest.mark.parametrize("change", [dict(logits=torch.zeros(())), dict(logits=torch.zeros(2, 5, 2)), dict(top=torch.zeros(6)), dict(ids=torch.zeros((), dtype=torch.int32)),
                                    dict(targets=torch.zeros((), dtype=torch.int32)), dict(entropy=torch.zeros(()))])
def test_logprobs(change):
    args = dict(logits=torch.zeros(2, 10), targets=torch.zeros(2, dtype=torch.int32), logprobs=torch.zeros(2), entropy=torch.zeros(2),
                top=torch.zeros(2, 3), ids=torch.zeros(2, 3, dtype=torch.int32))
    with pytest.raises(InvalidArgument, match="token_logprobs"):
        ops.token_logprobs(**{**args, **change})
