"""What the command line says about log probabilities, and what it refuses (no GPU)."""
import io
import json
import math
import math
from types import SimpleNamespace

import pytest

import nncpu_b200
from nncpu_b200 import cli
from nncpu_b200.cli import Options, chat_loop, parse_options, run_gen, run_perplexity
from nncpu_b200.errors import InvalidArgument
from nncpu_b200.sampling import GenerateResult, ScoreResult, StopReason, TokenLogprob

FOUND = [TokenLogprob(5, -0.5, 1.25, ((5, -0.5), (9, -1.0))), TokenLogprob(6, -2.0, 0.75, ((7, -0.25), (6, -2.0)))]


def lines(text):
    return [json.loads(x) for x in text.splitlines() if x.startswith("{")]


class Chat:
    """Stands in for a session: every reply is FOUND's tokens."""
    n_ctx = 100

    def cancel_handle(self):
        return SimpleNamespace(cancel=lambda: None)

    def chat(self, message, params, on_text):
        on_text(SimpleNamespace(text="yes"))
        return GenerateResult(StopReason.END_OF_TURN, 3, 2, 0.1, 0.1, [5, 6], FOUND if params.logprobs is not None else None)


@pytest.mark.parametrize("asked", [True, False])
def test_a_chats_replies_come_with_their_log_probabilities(asked):
    o = parse_options(["chat", "-m", "d", *(["--logprobs", "2"] if asked else [])])
    out, err = io.StringIO(), io.StringIO()
    assert chat_loop(Chat(), o, iter(["a\n", "b\n", "/exit\n"]), out, err) == 0
    got = lines(err.getvalue())
    assert out.getvalue() == "yes\nyes\n" and err.getvalue().count("tok/s") == 2
    assert [t["token"] for t in got] == ([5, 6, 5, 6] if asked else [])
    if asked:
        assert got[1] == {"token": 6, "logprob": -2.0, "entropy": 0.75, "top": [[7, -0.25], [6, -2.0]]}


class Token:
    """Stands in for a session that generates or scores."""

    def __init__(self, model, params, tokenizer=None):
        self.n_ctx, self.params = params.n_ctx or 100, params

    def generate(self, prompts, params, on_piece=None):
        return [GenerateResult(StopReason.MAX_TOKENS, len(p), 2, 0.1, 0.1, [5, 6], FOUND if params.logprobs is not None else None) for p in prompts]


@pytest.fixture
def fake(monkeypatch):
    monkeypatch.setattr(nncpu_b200, "Model", SimpleNamespace(load=lambda folder, dtype: None))
    monkeypatch.setattr(nncpu_b200, "Session", Token)


@pytest.mark.parametrize("asked", [True, False])
def test_the_greedy_run_tells_them_too(fake, asked):
    out, err = io.StringIO(), io.StringIO()
    assert run_gen(parse_options(["--gen", "d", "1 2 3", "2", *(["--logprobs", "2"] if asked else [])]), out, err) == 0
    assert out.getvalue().startswith("5 6\nprefill: 3 tokens")
    assert [t["token"] for t in lines(err.getvalue())] == ([5, 6] if asked else [])


@pytest.mark.parametrize("value", [-math.inf, math.nan, math.inf])
def test_every_line_is_json_whatever_the_numbers(value):
    """JSON has no infinities and no NaN: such a number is null."""
    def refuse(name):
        raise AssertionError(f"{name} is not JSON")
    line = cli._logprob_line(TokenLogprob(3, value, value, ((3, -0.5), (4, value))))
    assert json.loads(line, parse_constant=refuse) == {"token": 3, "logprob": None, "entropy": None, "top": [[3, -0.5], [4, None]]}


def perplexity(tmp_path, monkeypatch, text, n_ctx, logprob=-1.0):
    """run_perplexity over a file of ``text``: what it prints, and the stretches that were scored."""
    scored = []

    def score(self, texts, k):
        scored.extend(texts)
        return [ScoreResult([TokenLogprob(x, logprob, 0.0) for x in t[1:]]) for t in texts]
    monkeypatch.setattr(Token, "score", score, raising=False)
    f = tmp_path / "text"
    f.write_text(text)
    out = io.StringIO()
    assert run_perplexity(parse_options(["--perplexity", "d", str(f), "-c", str(n_ctx)]), out, io.StringIO()) == 0
    return out.getvalue(), scored


def test_a_perplexity_needs_a_context_of_two(fake, tmp_path, monkeypatch):
    with pytest.raises(InvalidArgument, match="context"):
        perplexity(tmp_path, monkeypatch, "1 2 3", 1)
    out, scored = perplexity(tmp_path, monkeypatch, "1 2 3 4 5", 2)
    assert scored == [[1, 2], [3, 4], [5]] and out.startswith("2 predictions of 5 tokens: -1.000000 nats a token, perplexity 2.7183")


def test_a_perplexity_of_no_number_is_none(fake, tmp_path, monkeypatch):
    """Logits of +inf give NaN, of which the perplexity is not infinite."""
    assert math.isnan(ScoreResult([TokenLogprob(1, -1.0, 0.0), TokenLogprob(1, math.nan, 0.0)]).perplexity)
    assert "perplexity nan" in perplexity(tmp_path, monkeypatch, "1 2 3", 9, math.nan)[0]
    assert "perplexity inf" in perplexity(tmp_path, monkeypatch, "1 2 3", 9, -math.inf)[0]


@pytest.mark.parametrize("text", ["² ³", "1 ²"])
def test_a_text_of_other_digits_is_text(fake, tmp_path, monkeypatch, text):
    """(Superscripts are digits, and no numbers.)"""
    monkeypatch.setattr("nncpu_b200.text.load_tokenizer", lambda folder: SimpleNamespace(encode=lambda t: list(t.encode())))
    assert perplexity(tmp_path, monkeypatch, text, 99)[1] == [list(text.encode())]
