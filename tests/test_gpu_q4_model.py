"""Whole models over a cache of 4 bits, and what they say about their tokens.

A number that lies next to the border of two codes takes one or the other by its last bit, and at a sequence's start one code moves a
logit by a percent; so the plain model attends to the numbers that the device's cache holds, layer by layer, and its own keys and
values have to be within half a step of those."""
import io
import json

import numpy as np
import pytest
import torch

import plain_q4 as Q
import plain_torch
from gpu_util import TOL, check
from nncpu_b200 import Engine, GenerateParams, Model, SamplerParams, Session, SessionParams
from nncpu_b200.cache.cache import KVGroup
from nncpu_b200.cli import main, parse_options, run_generate, run_perplexity
from nncpu_b200.errors import ContextFull, InvalidArgument, UnsupportedModel
from tiny import make_folder

pytestmark = pytest.mark.gpu
DTYPES = ["float32", "bfloat16"]
STORE = {"float32": torch.float32, "bfloat16": torch.bfloat16}
NAMES = ["B", "D", "E", "G"]          # heads of 32, 64 and 128 lanes, with biases, windows, one key/value head


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    root = tmp_path_factory.mktemp("q4")
    return {(n, d): make_folder(root / f"{n}_{d}", n, seed=ord(n), store_dtype=STORE[d]) for n in NAMES for d in DTYPES}


@pytest.fixture
def plain(monkeypatch):
    """(folder, tokens, engine, slot) -> logits of the plain model whose attention reads what the slot's cache holds."""
    monkeypatch.setattr(KVGroup, "trim", lambda self, slot, length: None)     # (windows keep their pages, for this to read)
    whole = plain_torch.masked_attention

    def logits(folder, toks, engine, slot):
        tol = TOL[str(engine.model.rt.dtype).replace("torch.", "")]
        layer = iter(range(100))

        def attention(q, k, v, window):
            held = [t.double().cpu() for t in engine.cached(slot, next(layer))]
            for own, h in zip((k, v), held):
                # half a step, what the group's two numbers lose to half precision, and the run's own rounding of the number
                g = own.reshape(*own.shape[:-1], -1, 32)
                span = (g.amax(-1) - g.amin(-1)).repeat_interleave(32, -1)
                assert ((h[:len(own)] - own).abs() <= span / 30 + (own.abs() + 2 * span) * 2.0 ** -11 + 2 * tol * own.abs().max()).all()
            return whole(q, held[0][:len(k)], held[1][:len(v)], window)
        with monkeypatch.context() as m:
            m.setattr(plain_torch, "masked_attention", attention)
            return plain_torch.TorchQwen3(folder).logits(toks)
    return logits


def ids(n, seed, vocab=300):
    return np.random.RandomState(seed).randint(0, vocab, size=n).tolist()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", NAMES)
def test_whole_in_portions_and_one_by_one(folders, plain, name, dtype):
    model = Model.load(folders[name, dtype], dtype=dtype)
    engine = Engine(model, max_tokens=64 * 24, kv_dtype="q4")
    toks = ids(330, 1)
    s = engine.alloc_slot()
    whole = engine.step([s], [toks], [list(range(330))]).clone()
    check(whole, plain(folders[name, dtype], toks, engine, s), TOL[dtype], "whole")
    s2 = engine.alloc_slot()
    parts = [engine.step([s2], [toks[a:b]], [list(range(b - a))]).clone() for a, b in ((0, 1), (1, 130), (130, 149), (149, 290))]
    parts += [engine.step([s2], [[t]]).clone() for t in toks[290:]]
    check(torch.cat(parts), plain(folders[name, dtype], toks, engine, s2), TOL[dtype], "in portions")


@pytest.mark.parametrize("dtype", DTYPES)
def test_unequal_sequences_side_by_side_and_slots_used_again(folders, plain, dtype):
    model = Model.load(folders["D", dtype], dtype=dtype)
    engine = Engine(model, max_tokens=64 * 20, kv_dtype="q4")
    for round in range(2):
        texts = [ids(n, 10 * round + n) for n in (5, 200, 64, 65, 131)]
        slots = [engine.alloc_slot() for _ in texts]
        got = [engine.step(slots, [t[:-3] for t in texts]).clone()]
        for k in (3, 2, 1):
            got.append(engine.step(slots, [[t[-k]] for t in texts]).clone())
        for b, t in enumerate(texts):
            want = plain(folders["D", dtype], t, engine, slots[b])[-4:]
            check(torch.stack([g[b] for g in got]), want, TOL[dtype], f"sequence {b} of round {round}")
        for s in slots:
            engine.free_slot(s)
        engine.cache.check()


def test_the_first_layer_holds_what_a_float32_cache_would_cut(folders):
    model = Model.load(folders["G", "float32"], dtype="float32")
    toks = ids(150, 3)
    held = []
    for kv in (None, "q4"):
        engine = Engine(model, max_tokens=256, kv_dtype=kv)
        s = engine.alloc_slot()
        engine.step([s], [toks[:140]])
        for t in toks[140:]:
            engine.step([s], [[t]])
        held.append([t.cpu().numpy() for t in engine.cached(s)])
        assert engine.cache.bytes() == (4 if kv is None else 5 / 8) * 2 * 2 * engine.cache.n_pages * 64 * 2 * 128
    for full, cut in zip(*held):
        want = Q.numbers(*Q.quantise(full.reshape(-1, 128))).reshape(full.shape)
        # keys of a float32 run are rounded here, from sums of more bits there: the odd code may be the next one
        step = np.ptp(full.reshape(150, 2, 4, 32), axis=-1).repeat(32, -1).reshape(full.shape) / 15
        off = np.abs(cut - want)
        assert (off <= 1.01 * step + 1e-6).all() and (off > 0.01 * step).mean() < 1e-4


@pytest.mark.parametrize("dtype", DTYPES)
def test_windows_that_have_given_pages_back(folders, monkeypatch, dtype):
    model = Model.load(folders["E", dtype], dtype=dtype)
    toks, got = ids(400, 4), []
    for keeps in (False, True):
        if keeps:
            monkeypatch.setattr(KVGroup, "trim", lambda self, slot, length: None)
        engine = Engine(model, max_tokens=64 * 8, kv_dtype="q4")
        s = engine.alloc_slot()
        rows = [engine.step([s], [toks[:250]]).clone(), engine.step([s], [toks[250:280]]).clone()]
        got.append(torch.cat(rows + [engine.step([s], [[t]]).clone() for t in toks[280:]]))
        assert (engine.cached(s, 0)[0][0].abs().max() == 0) == (not keeps)
    assert torch.equal(*got)


@pytest.mark.parametrize("run_ahead", [True, False])
@pytest.mark.parametrize("sampler", [SamplerParams.greedy(), SamplerParams(1.0, 0, 1.0, 0.0), SamplerParams(), SamplerParams(0.8, 0, 0.9, 0.0)])
def test_generation_tells_its_tokens_logprobs(folders, sampler, run_ahead):
    model = Model.load(folders["D", "float32"], dtype="float32")
    session = Session(model, SessionParams(n_ctx=200, seed=5, max_batch=3, run_ahead=run_ahead, kv_q4=True))
    prompts = [ids(20, 1), ids(7, 2), ids(33, 3), ids(5, 4)]
    res = session.generate(prompts, GenerateParams(12, sampler, logprobs=4), stop_token_ids=list(range(0, 520, 40)))
    plain_res = Session(model, SessionParams(n_ctx=200, seed=5, max_batch=3, run_ahead=run_ahead, kv_q4=True)).generate(
        prompts, GenerateParams(12, sampler), stop_token_ids=list(range(0, 520, 40)))
    assert [r.tokens for r in res] == [r.tokens for r in plain_res] and all(r.logprobs is None for r in plain_res)
    for p, r in zip(prompts, res):
        assert [t.token for t in r.logprobs] == r.tokens
        engine = Engine(model, max_tokens=256, kv_dtype="q4")
        s = engine.alloc_slot()
        for k, a in enumerate(r.logprobs):
            # the same steps again, one sequence by itself (whose sums may round otherwise, which may move a code; see above: a percent
            # of a logit of 1 or so)
            z = engine.step([s], [p if k == 0 else [r.tokens[k - 1]]])[0].double().log_softmax(-1)
            assert abs(a.logprob - z[a.token].item()) < 2e-2 and abs(a.entropy + (z.exp() * z).sum().item()) < 2e-2
            assert len(a.top) == 4 and all(x[1] >= y[1] for x, y in zip(a.top, a.top[1:]))
            if sampler.is_greedy:
                assert a.top[0][0] == a.token and a.top[0][1] == a.logprob


@pytest.mark.parametrize("kv_q4", [False, True])
def test_score_against_the_plain_model(folders, plain, monkeypatch, kv_q4):
    folder = folders["G", "float32"]
    session = Session(Model.load(folder, dtype="float32"), SessionParams(n_ctx=1000, kv_q4=kv_q4, max_batch=1))
    texts = [ids(600, 7), ids(2, 8), ids(1, 9), ids(257, 10)]
    free = session.engine.cache.groups[0].pool.n_free
    found = []
    free_slot = session.engine.free_slot
    # (the plain model reads the cache before the slot is given back)
    monkeypatch.setattr(session.engine, "free_slot", lambda s: (found.append(
        plain(folder, texts[len(found)], session.engine, s) if kv_q4 else plain_torch.TorchQwen3(folder).logits(texts[len(found)])), free_slot(s)))
    for text, r, z in zip(texts, session.score(texts, 3), found):
        z = z.astype(np.float64)
        m = z.max(-1, keepdims=True)
        logp = z - m - np.log(np.exp(z - m).sum(-1, keepdims=True))
        want = logp[np.arange(len(text) - 1), text[1:]]
        assert [t.token for t in r.tokens] == text[1:]
        tol = TOL["float32"] * np.abs(z).max() * 2       # a logit's error, and that of the sum
        assert np.abs(np.array([t.logprob for t in r.tokens]) - want).max(initial=0) <= tol
        entropy = -(np.exp(logp) * logp).sum(-1)[:-1]
        assert np.abs(np.array([t.entropy for t in r.tokens]) - entropy).max(initial=0) <= tol * (1 + np.log(z.shape[1]))
        for t, row in zip(r.tokens, logp):
            assert len(t.top) == 3 and all(abs(p - row[i]) <= tol for i, p in t.top) and t.top[0][1] >= row.max() - tol
        assert np.isnan(r.perplexity) if len(text) == 1 else abs(r.perplexity - np.exp(-want.mean())) < 1e-2 * r.perplexity
    assert session.engine.cache.groups[0].pool.n_free == free
    monkeypatch.setattr(session.engine, "free_slot", free_slot)
    with pytest.raises(InvalidArgument):
        session.score([[]])
    with pytest.raises(InvalidArgument):
        session.score([[1, 2]], 33)
    with pytest.raises(ContextFull):
        session.score([ids(1001, 1)])
    with pytest.raises(InvalidArgument):
        session.score([[1, 5000]])
    assert session.engine.cache.groups[0].pool.n_free == free


def test_a_conversation_over_4_bits(folders, plain):
    """Turns (captured prompt steps) and replies on the session's own sequence."""
    folder = folders["G", "bfloat16"]
    session = Session(Model.load(folder), SessionParams(n_ctx=400, seed=1, max_batch=1, kv_q4=True))
    text = []
    for turn in range(3):
        new = ids(20 + turn, 20 + turn)
        r = session.extend(new, GenerateParams(10, SamplerParams.greedy()), stop_token_ids=[])
        text += new + r.tokens
    assert session.tokens() == text
    session.eval([])
    check(session.logits()[None], plain(folder, text, session.engine, session._own_slot)[-1:], TOL["bfloat16"], "after three turns")


def test_what_cannot_be_kept_in_4_bits_is_refused(tmp_path):
    for name in "AC":       # heads of 16 and of 48 lanes
        model = Model.load(make_folder(tmp_path / name, name), dtype="float32")
        with pytest.raises(UnsupportedModel, match="4 bits"):
            Engine(model, max_tokens=256, kv_dtype="q4")
        with pytest.raises(InvalidArgument):
            Engine(model, max_tokens=256, kv_dtype="q8")
        with pytest.raises(InvalidArgument):
            Session(model, SessionParams(kv_f32=True, kv_q4=True))


def test_command_line(folders, tmp_path):
    folder = str(folders["G", "bfloat16"])
    f = tmp_path / "text.txt"
    f.write_text(" ".join(map(str, ids(150, 3))))

    def run(call, argv):
        out, err = io.StringIO(), io.StringIO()
        assert call(parse_options(argv), out, err) == 0
        return out.getvalue(), [json.loads(line) for line in err.getvalue().splitlines() if line.startswith("{")]
    found = {}
    for flags in ([], ["--kv-q4"]):
        out, lines = run(run_perplexity, ["--perplexity", folder, str(f), "--logprobs", "2", "-c", "100", *flags])
        assert len(lines) == 148 and all(len(t["top"]) == 2 for t in lines) and "148 predictions of 150 tokens" in out
        found[bool(flags)] = float(out.split("perplexity ")[1].split()[0])
    assert abs(found[True] / found[False] - 1) < 0.2
    out, lines = run(run_generate, ["-m", folder, "--tokens", "5 6 7", "-n", "4", "--temp", "0", "--kv-q4", "--logprobs", "1"])
    assert [t["token"] for t in lines] == [int(t) for t in out.split()] and all(t["top"][0][0] == t["token"] for t in lines)
    f.write_text("7")
    assert main(["--perplexity", folder, str(f)]) == 1
    assert main(["--perplexity", folder, str(tmp_path / "none")]) == 1


@pytest.mark.parametrize("dtype", DTYPES)
def test_the_arena_is_sized_ahead_and_steps_take_nothing_from_the_allocator(folders, dtype):
    engine = Engine(Model.load(folders["D", dtype], dtype=dtype), max_tokens=64 * 24, kv_dtype="q4", max_step_tokens=256)
    assert engine.arena.peak > 0
    a, b = engine.alloc_slot(), engine.alloc_slot()

    def steps():
        engine.step([a, b], [ids(100, 1), ids(30, 2)])
        engine.step([a, b], [[5], [6]])
        engine.step([a], [ids(17, 3)])
    steps()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    steps()
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() == before and torch.cuda.max_memory_allocated() - before < 1 << 16     # (metadata and ids)
