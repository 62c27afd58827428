"""Log probabilities on the host: parameters, results, and which rows of which steps belong to a sequence (no GPU)."""
import math

import pytest

import nncpu_b200.engine.generate as loop
from nncpu_b200.cli import parse_options
from nncpu_b200.errors import InvalidArgument
from nncpu_b200.sampling import GenerateParams, SamplerParams, ScoreResult, TokenLogprob
from test_generate_loop import FakeEngine, Script


class Rows:
    """Stands in for the device's rows: row i of a step says (logits row, token)."""
    made = []

    def __init__(self, k, vocab_size):
        self.rows = []
        Rows.made.append(self)

    def add(self, logits, tokens):
        first = len(self.rows)
        self.rows += [TokenLogprob(t, -float(slot), float(length)) for (slot, length), t in zip(logits, tokens)]
        return first

    def read(self):
        return self.rows


@pytest.mark.parametrize("max_batch", [1, 2, 5])
def test_rows_go_to_their_sequences_when_others_leave(monkeypatch, max_batch):
    monkeypatch.setattr(loop, "Logprobs", Rows)
    engine = FakeEngine()
    engine.vocab_size = 1000
    prompts = [[1] * 3, [1] * 5, [1] * 2, [1] * 7, [1]]
    # sequence 1 ends at once, 3 after two tokens
    special = {(1, 5): 7, (3, 9): 7}
    res = loop.generate(engine, Script(special), prompts, GenerateParams(6, SamplerParams.greedy(), logprobs=0), [7], max_batch=max_batch)
    assert [len(r.tokens) for r in res] == [6, 0, 6, 2, 6]
    for p, r in zip(prompts, res):
        assert [t.token for t in r.logprobs] == r.tokens
        assert [int(t.entropy) for t in r.logprobs] == [len(p) + i for i in range(len(r.tokens))]       # the length at which it was chosen
        assert len({t.logprob for t in r.logprobs}) <= 1                                                # one slot
    res = loop.generate(engine, Script(), prompts, GenerateParams(2, SamplerParams.greedy()), [7])
    assert all(r.logprobs is None for r in res)


def test_parameters():
    GenerateParams(0, SamplerParams(), 32).check()
    for bad in (-1, 33, 1.5, "2"):
        with pytest.raises(InvalidArgument):
            GenerateParams(logprobs=bad).check()
    with pytest.raises(InvalidArgument):
        GenerateParams(max_tokens=-1).check()
    o = parse_options(["-m", "d", "--tokens", "1", "--kv-q4", "--logprobs", "3"])
    assert o.kv_q4 and o.generate_params().logprobs == 3
    assert parse_options(["--perplexity", "dir", "file", "-c", "9"]).args == ["dir", "file"]
    for bad in (["--logprobs", "-1"], ["--logprobs", "33"], ["--kv-q4", "--kv-f32"], ["--perplexity", "dir"], ["--logprobs"]):
        with pytest.raises(InvalidArgument):
            parse_options(bad)


def test_a_texts_perplexity():
    r = ScoreResult([TokenLogprob(1, -1.0, 0.0), TokenLogprob(2, -3.0, 0.0)])
    assert r.logprob == -4.0 and math.isclose(r.perplexity, math.exp(2.0))
    assert math.isnan(ScoreResult().perplexity) and ScoreResult().logprob == 0.0
    assert ScoreResult([TokenLogprob(1, -math.inf, 0.0)]).perplexity == math.inf
