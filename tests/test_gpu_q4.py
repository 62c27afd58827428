"""The 4-bit cache on the device: the append, what is read back, and the attention over it, against NumPy in 64 bits."""
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


def places(lens_new, pasts):
    """tok_seq, tok_pos, cu_seqlens (int32) of sequences that bring so many tokens after so many."""
    seq = np.repeat(np.arange(len(lens_new)), lens_new).astype(np.int32)
    pos = np.concatenate([np.arange(p, p + n) for n, p in zip(lens_new, pasts)] + [np.zeros(0)]).astype(np.int32)
    cu = np.concatenate([[0], np.cumsum(lens_new)]).astype(np.int32)
    return seq, pos, cu


# -- append ----------------------------------------------------------------------------------------------------------------


def plain_append(qkv, qg, kg, eps, cs, heads, kv, D, half):
    """float64 q [n, heads, D], bound of a 32-bit rounding error of it, and float32 k, v [n, kv, D]."""
    x = qkv.double().numpy().reshape(len(qkv), -1)[:, :(heads + 2 * kv) * D].reshape(len(qkv), heads + 2 * kv, D)
    y, size = x.copy(), np.abs(x)
    for part, g in ((slice(0, heads), qg), (slice(heads, heads + kv), kg)):
        if g is not None:
            y[:, part] = x[:, part] / np.sqrt((x[:, part] ** 2).mean(-1, keepdims=True) + eps) * g.double().numpy()
    size = np.abs(y)
    if half:
        c, s = cs[..., 0].double().numpy()[:, None], cs[..., 1].double().numpy()[:, None]
        a, b = y[:, :heads + kv, :half].copy(), y[:, :heads + kv, half:2 * half].copy()
        y[:, :heads + kv, :half], y[:, :heads + kv, half:2 * half] = a * c - b * s, b * c + a * s
        size[:, :heads + kv, :half] = np.abs(a * c) + np.abs(b * s)
        size[:, :heads + kv, half:2 * half] = np.abs(b * c) + np.abs(a * s)
    return y[:, :heads], size[:, :heads], y[:, heads:heads + kv].astype(np.float32), x[:, heads + kv:].astype(np.float32)


@pytest.mark.parametrize("new,past,heads,kv,D,norm,half,qkv_dt,q_dt", [
    ([1], [0], 4, 2, 64, True, 32, F32, BF16),
    ([1, 1, 1], [63, 64, 700], 32, 8, 128, True, 64, F32, BF16),
    ([70, 3], [10, 61], 8, 2, 128, True, 64, F32, BF16),
    ([130], [0], 5, 1, 96, True, 48, F32, F32),
    ([9, 2], [0, 5], 6, 3, 32, False, 16, F32, F32),
    ([17], [30], 4, 4, 256, True, 40, F32, BF16),
    ([17], [30], 4, 4, 160, True, 0, BF16, BF16),
    ([33], [1], 2, 1, 64, False, 0, F32, BF16),
    ([200], [57], 16, 8, 128, True, 64, F32, F32)])
def test_append_is_bit_for_bit_the_format(new, past, heads, kv, D, norm, half, qkv_dt, q_dt):
    seq, pos, _ = places(new, past)
    n = len(seq)
    qkv = (rand(n, (heads + 2 * kv) * D + 8, seed=1) * 2).to(qkv_dt)        # (rows longer than their heads)
    qg, kg = ((1 + 0.1 * rand(D, seed=2), 1 + 0.1 * rand(D, seed=3)) if norm else (None, None))
    angle = rand(n, max(half, 1), seed=4).double() * 3
    cs = torch.stack((angle.cos(), angle.sin()), -1).float() if half else None
    eps = 1e-6
    per = [-(-(p + m) // 64) for m, p in zip(new, past)]
    ids = np.random.default_rng(5).permutation(sum(per) + 2)
    table = np.full((len(new), max(per)), -1, dtype=np.int32)
    at = 0
    for b, c in enumerate(per):
        table[b, :c] = ids[at:at + c]
        at += c
    want_q, size, k, v = plain_append(qkv, qg, kg, eps, cs, heads, kv, D, half)
    want = [Q.empty_pages(sum(per) + 2, kv, D, 0xAB) for _ in range(2)]
    for t in range(n):
        for h in range(kv):
            for pages, x, values in ((want[0], k, False), (want[1], v, True)):
                Q.put(pages, table[seq[t], pos[t] // 64], h, pos[t] % 64, x[t, h], values)
    kp, vp = Q.as_cuda(*[Q.empty_pages(sum(per) + 2, kv, D, 0xAB) for _ in range(2)])
    q = torch.empty(n, heads * D, dtype=q_dt, device=DEV)
    d = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    ts, tp, bt = Q.as_cuda(seq, pos, table)
    ops.qk_norm_rope_append_q4(qkv.to(DEV), d(qg), d(kg), eps, d(cs), ts, tp, bt, kp, vp, q, heads, kv, D)
    assert np.array_equal(kp.cpu().numpy(), want[0]) and np.array_equal(vp.cpu().numpy(), want[1])
    # a sum of D squares over 32 threads (D / 32 + 5 additions), a root, a division, up to six more roundings
    tol = size * (D / 32 + 13) * 2.0 ** -24 + (np.abs(want_q) * 2.0 ** -8 if q_dt == BF16 else 0)
    assert (np.abs(q.double().cpu().numpy().reshape(want_q.shape) - want_q) <= tol + 1e-30).all()
    ko, vo = torch.empty(n, kv * D, device=DEV), torch.empty(n, kv * D, device=DEV)
    ops.q4_read(kp, vp, bt, ts, tp, ko, vo)
    for got, x in ((ko, k), (vo, v)):
        held = Q.numbers(*Q.quantise(x)).reshape(n, -1)
        assert np.array_equal(got.cpu().numpy(), held.astype(np.float32))       # d c is exact in 32 bits, one rounding for + m
    kb, vb = torch.empty(n, kv * D, device=DEV, dtype=BF16), torch.empty(n, kv * D, device=DEV, dtype=BF16)
    ops.q4_read(kp, vp, bt, ts, tp, kb, vb)
    assert torch.equal(kb, ko.bfloat16()) and torch.equal(vb, vo.bfloat16())


def test_append_skips_tokens_without_a_place_and_reads_zeros_for_them():
    heads, kv, D, n = 2, 1, 64, 6
    table = torch.tensor([[0, -1, 9], [2, 1, 0]], dtype=torch.int32)
    seq = torch.tensor([-1, 0, 0, 0, 1, 1], dtype=torch.int32)
    pos = torch.tensor([0, 3, 64, 130, 192, -1], dtype=torch.int32)     # padding; there; given back; no such page; beyond the table; before it
    kp = torch.full((3, kv, 40 * D), 0xAB, dtype=torch.uint8, device=DEV)
    vp = kp.clone()
    qkv = rand(n, 4 * D).to(DEV)
    q = torch.empty(n, heads * D, device=DEV)
    args = (seq.to(DEV), pos.to(DEV), table.to(DEV))
    ops.qk_norm_rope_append_q4(qkv, None, None, 0.0, None, *args, kp, vp, q, heads, kv, D)
    assert torch.equal(q, qkv[:, :2 * D])
    want = Q.empty_pages(3, kv, D, 0xAB)
    Q.put(want, 0, 0, 3, qkv[1, 2 * D:3 * D].cpu().numpy(), False)
    assert np.array_equal(kp.cpu().numpy(), want)
    ko, vo = torch.full((n, D), 7.0, device=DEV), torch.full((n, D), 7.0, device=DEV)
    ops.q4_read(kp, vp, args[2], args[0], args[1], ko, vo)
    others = [0, 2, 3, 4, 5]
    assert (ko[others] == 0).all() and (vo[others] == 0).all() and (ko[1] != 0).any()
    # queries alone, for a mixer that reads another's cache
    q2 = torch.empty_like(q)
    ops.qk_norm_rope_append_q4(qkv, None, None, 0.0, None, *args, None, None, q2, heads, 0, D)
    assert torch.equal(q2, q)


def test_append_of_numbers_beyond_the_range_and_nan():
    D = 64
    x = torch.zeros(3, 3 * D)
    x[0, D + 3], x[0, 2 * D:2 * D + 2] = float("nan"), torch.tensor([float("inf"), -float("inf")])
    x[1, D:D + 4] = torch.tensor([1e6, -2e5, 7.0, 65504.0])
    x[2, D:] = 3.25
    table = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    seq, pos = torch.zeros(3, dtype=torch.int32, device=DEV), torch.arange(3, dtype=torch.int32, device=DEV)
    kp = torch.zeros(1, 1, 40 * D, dtype=torch.uint8, device=DEV)
    vp = kp.clone()
    ops.qk_norm_rope_append_q4(x.to(DEV), None, None, 0.0, None, seq, pos, table, kp, vp, torch.empty(3, D, device=DEV), 1, 1, D)
    k, v = torch.empty(3, D, device=DEV), torch.empty(3, D, device=DEV)
    ops.q4_read(kp, vp, table, seq, pos, k, v)
    for got, part in ((k, x[:, D:2 * D]), (v, x[:, 2 * D:])):
        want = Q.numbers(*Q.quantise(part.numpy()))
        np.testing.assert_array_equal(got.cpu().numpy(), want.astype(np.float32))
    assert k[0, :32].isnan().all() and (k[0, 32:] == 0).all() and (v[0].abs() <= 65600).all() and (k[2] == 3.25).all()


def test_append_with_a_query_temperature():
    D, n = 32, 5
    qkv, pos = rand(n, 3 * D).to(DEV), torch.tensor([0, 9, 10, 99, 5000], dtype=torch.int32, device=DEV)
    seq, table = torch.full((n,), -1, dtype=torch.int32, device=DEV), torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    kp = torch.zeros(1, 1, 40 * D, dtype=torch.uint8, device=DEV)
    q = torch.empty(n, D, device=DEV)
    ops.qk_norm_rope_append_q4(qkv, None, None, 0.0, None, seq, pos, table, kp, kp.clone(), q, 1, 1, D, q_temp=(0.1, 10))
    t = 1 + 0.1 * torch.log(torch.floor((pos.double() + 1) / 10) + 1)
    assert torch.allclose(q.double(), qkv[:, :D].double() * t[:, None], rtol=2.0 ** -21, atol=0)
    assert (kp == 0).all()


# -- attention -------------------------------------------------------------------------------------------------------------


def check_rows(got, q, ks, vs, seq, pos, dt, heads, scale, **opt):
    """Every output row against 64 bits, number by number.  32-bit: a score is a sum of D products, a weight the exponential of
    a difference of scores, an output a sum over n keys; all relative to the sums of the magnitudes.  bfloat16: a
    weight (times its group's step) is rounded once and multiplies a code of at most 8 steps, a key's and a value's number may be
    rounded to half precision (2^-11), the output once."""
    gate = opt.pop("gate", None)
    for t in range(len(seq)):
        row = got[t].double().cpu().numpy().reshape(heads, -1)
        if seq[t] < 0:
            assert (row == 0).all()
            continue
        k, v = ks[seq[t]], vs[seq[t]]
        D = k.shape[-1]
        qt = q[t].double().cpu().numpy().reshape(heads, D)
        wide = lambda a: np.abs(a) + np.repeat(np.ptp(a.reshape(*a.shape[:-1], D // 32, 32), -1), 32, -1)  # noqa: E731
        g = None if gate is None else gate[t].double().cpu().numpy()
        want, mass, _ = Q.attend(qt, k, v, pos[t], scale, gate=g, **opt)
        see = Q.visible(pos[t], len(k), opt.get("window", 0), opt.get("keep", 0))
        group = heads // k.shape[1]
        reach = np.array([(wide(k[see, h // group]) @ np.abs(qt[h])).max() * abs(scale) if see.any() else 0.0 for h in range(heads)])[:, None]
        n = int(see.sum())
        extra = opt.get("cap", 0.0) * 2.0 ** -20 + (n * 2.0 ** -22 if opt.get("slope_base") else 0)
        if dt == F32:
            tol = mass * (2 * (reach * (D + 16) * 2.0 ** -24 + extra) + 2 * (n + 64) * 2.0 ** -24)
        else:
            # weights' mass over codes of at most 8 steps: at most 8/15 of the groups' ranges, beside the values' own
            wmass = Q.attend(qt, k, wide(v), pos[t], scale, gate=g, **opt)[0]
            tol = 2.0 ** -8 * (np.abs(want) + wmass) + 2 * (reach * 2.0 ** -11 + extra + 2.0 ** -11) * wmass
        err = np.abs(row - want)
        assert np.isfinite(row).all() and (err <= tol + 1e-30).all(), (t, float((err / (tol + 1e-30)).max()))


def run_attention(lens, heads, kv, D, dt, seq=None, pos=None, seed=0, prompt=None, fill=0xFF, **opt):
    kp, vp, table, ks, vs = Q.filled_cache(lens, kv, D, seed, fill=fill)
    if prompt is not None:
        seq, pos, cu = places(*prompt)
    elif seq is None:
        seq, pos = np.arange(len(lens), dtype=np.int32), np.array(lens, dtype=np.int32) - 1
    n, scale = len(seq), D ** -0.5
    q = rand(n, heads * D, seed=seed + 1).to(dt).to(DEV)
    out = torch.full((n, heads * D), float("nan"), dtype=dt, device=DEV)
    kpc, vpc, bt, ts, tp = Q.as_cuda(kp, vp, table, np.asarray(seq, np.int32), np.asarray(pos, np.int32))
    sinks = opt.pop("sinks", None)
    gate = opt.pop("gate", None)
    if sinks is not None:
        sinks = rand(heads, seed=seed + 2).to(DEV)
    head_gate = None
    if gate is not None:
        head_gate = (rand(n, heads + 3, seed=seed + 3).to(DEV), 2)
    kw = dict(sinks=sinks, head_gate=head_gate, **opt)
    if prompt is not None:
        status = torch.zeros(1, dtype=torch.int32, device=DEV)
        cuc, = Q.as_cuda(cu)
        ops.attention_q4_prompt(q, kpc, vpc, bt, cuc, ts, tp, out, len(cu) - 1, heads, kv, D, scale, int(max(lens)), status, **kw)
        assert int(status) == 0
    else:
        ops.attention_q4(q, kpc, vpc, bt, ts, tp, out, heads, kv, D, scale, **kw)
    check_rows(out, q, ks, vs, seq, pos, dt, heads, scale, gate=None if gate is None else head_gate[0][:, 2:2 + heads],
               sinks=None if sinks is None else sinks.double().cpu().numpy(), **opt)
    return out


SHAPES = [(4, 2, 64), (32, 8, 128), (5, 1, 96), (8, 8, 32), (24, 2, 128), (16, 1, 64), (3, 1, 160), (2, 2, 256), (34, 2, 128)]


@pytest.mark.parametrize("heads,kv,D", SHAPES)
@pytest.mark.parametrize("dt", [F32, BF16])
def test_attention_of_single_tokens(heads, kv, D, dt):
    run_attention([1, 64, 65, 130, 2, 63], heads, kv, D, dt)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("lens", [[1], [1500], [4097, 3], [700] * 9, [200, 1, 3000, 64, 900]])
def test_attention_of_long_and_unequal_sequences(lens, dt):
    run_attention(lens, 8, 2, 128, dt, seed=3)
    run_attention(lens, 8, 2, 64, dt, seed=4)


@pytest.mark.parametrize("heads,kv,D", [(8, 8, 64), (32, 8, 128), (24, 2, 128)])
def test_attention_of_many_sequences(heads, kv, D):
    # more tokens than a warp looks at once, short ones beside long ones, rows of no sequence among them
    lens = [1 + (37 * i * i) % 300 for i in range(70)] + [2500]
    seq = list(range(71))
    seq[5] = seq[40] = seq[69] = -1
    run_attention(lens, heads, kv, D, BF16, seq=seq, pos=[n - 1 for n in lens], seed=11)


@pytest.mark.parametrize("window,keep", [(0, 0), (9000, 70)])
def test_attention_of_one_very_long_sequence(window, keep):
    run_attention([20000], 4, 1, 64, BF16, seed=12, window=window, keep=keep)
    run_attention([9003], 6, 2, 128, BF16, seed=13, window=window and 4000, keep=keep)


OPTIONS = [dict(window=1), dict(window=64), dict(window=100, keep=3), dict(window=70, keep=130), dict(window=-48), dict(window=-64),
           dict(slope_base=8.0), dict(sinks=True), dict(cap=5.0), dict(gate=True), dict(cap=30.0, sinks=True, gate=True, window=90, keep=1),
           dict(slope_base=4.0, sinks=True, gate=True)]


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("opt", OPTIONS, ids=str)
def test_attention_options(opt, dt):
    for heads, kv, D in ((4, 2, 128), (8, 1, 64), (3, 1, 96)):
        run_attention([1, 129, 400, 64], heads, kv, D, dt, seed=5, **opt)


@pytest.mark.parametrize("dt", [F32, BF16])
def test_attention_of_any_tokens_in_any_order_and_of_padding(dt):
    # several tokens of one sequence, a token twice, rows of no sequence between them
    run_attention([300, 70], 8, 2, 128, dt, seq=[1, -1, 0, 0, 1, -1, 0, 0], pos=[69, 0, 299, 10, 0, 5, 299, 64], seed=6)
    out = run_attention([5], 8, 2, 64, dt, seq=[-1, -1], pos=[0, 3])
    assert (out == 0).all()


@pytest.mark.parametrize("dt", [F32, BF16])
def test_what_lies_behind_the_end_and_outside_the_pages_is_not_seen(dt):
    heads, kv, D = 8, 2, 128
    kp, vp, table, ks, vs = Q.filled_cache([150, 200], kv, D, 7)
    table[0, 1] = -1                   # sequence 0 has lost its middle page
    table[1, 2] = 99                   # sequence 1's third page is none
    see = [np.r_[0:64, 128:150], np.r_[0:128, 192:200]]
    q = rand(2, heads * D).to(dt).to(DEV)
    out = torch.empty(2, heads * D, dtype=dt, device=DEV)
    ops.attention_q4(q, *Q.as_cuda(kp, vp, table, np.arange(2, dtype=np.int32), np.array([149, 199], dtype=np.int32)), out, heads, kv, D, D ** -0.5)
    for b in range(2):
        check_rows(out[b:b + 1], q[b:b + 1], [ks[b][see[b]]], [vs[b][see[b]]], [0], [len(see[b]) - 1], dt, heads, D ** -0.5)


PROMPTS = [(([1],), ([0],)), (([2],), ([0],)), (([64],), ([64],)), (([200],), ([0],)), (([130, 1, 70],), ([0, 300, 59],)), (([24],), ([701],)),
           (([300],), ([33],)), (([33, 40, 35],), ([0, 5, 190],)), (([47],), ([0],)), (([5],), ([3000],))]


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("heads,kv,D", [(8, 2, 128), (4, 4, 64), (10, 2, 96), (6, 1, 32), (4, 1, 160)])
@pytest.mark.parametrize("new,past", [(a[0], b[0]) for a, b in PROMPTS])
def test_attention_of_prompts(new, past, heads, kv, D, dt):
    run_attention([n + p for n, p in zip(new, past)], heads, kv, D, dt, seed=8, prompt=(new, past))


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("opt", OPTIONS, ids=str)
def test_prompt_attention_options(opt, dt):
    for heads, kv, D in ((4, 2, 128), (8, 1, 64), (3, 1, 96)):
        run_attention([230, 77], heads, kv, D, dt, seed=9, prompt=([200, 60], [30, 17]), **opt)


@pytest.mark.parametrize("dt", [F32, BF16])
def test_on_another_stream_and_captured(dt):
    heads, kv, D, lens = 8, 2, 128, [700, 33, 64]
    kp, vp, table, ks, vs = Q.filled_cache(lens, kv, D, 10)
    kp, vp, table, seq, pos = Q.as_cuda(kp, vp, table, np.arange(3, dtype=np.int32), np.array(lens, dtype=np.int32) - 1)
    q = rand(3, heads * D).to(dt).to(DEV)
    want, out = torch.empty_like(q), torch.empty_like(q)
    ops.attention_q4(q, kp, vp, table, seq, pos, want, heads, kv, D, 0.1)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        ops.attention_q4(q, kp, vp, table, seq, pos, out, heads, kv, D, 0.1)
    stream.synchronize()
    assert torch.equal(out, want)
    graph = torch.cuda.CUDAGraph()
    out.zero_()
    with torch.cuda.graph(graph):
        ops.attention_q4(q, kp, vp, table, seq, pos, out, heads, kv, D, 0.1)
    # replayed on other data: shorter sequences, other queries
    pos.copy_(torch.tensor([100, 0, 63]))
    q.copy_(rand(3, heads * D, seed=5).to(dt))
    graph.replay()
    check_rows(out, q, ks, vs, [0, 1, 2], [100, 0, 63], dt, heads, 0.1)


def test_too_little_scratch_is_refused():
    kp = torch.zeros(70, 1, 40 * 64, dtype=torch.uint8, device=DEV)
    q, out = torch.zeros(1, 64, device=DEV), torch.zeros(1, 64, device=DEV)
    table = torch.arange(64, dtype=torch.int32, device=DEV)[None]
    one = torch.zeros(1, dtype=torch.int32, device=DEV)
    assert ops.attention_q4_scratch_floats(1, 1, 1, 64, F32, 4096) > 8
    with pytest.raises(Exception, match="scratch"):
        ops.attention_q4(q, kp, kp, table, one, one, out, 1, 1, 64, 1.0, scratch=torch.zeros(8, device=DEV))


# -- as a program calls them -----------------------------------------------------------------------------------------------


def prompt_call(dt, lens, new, heads=8, kv=2, D=128, seed=0, pad=0):
    """A call of attention_q4_prompt over sequences of ``lens`` keys that bring ``new`` tokens: (call(out), q, out, what check_rows needs).
    ``pad`` rows of no sequence stand behind the last."""
    kp, vp, table, ks, vs = Q.filled_cache(lens, kv, D, seed)
    seq, pos, cu = places(new, [n - m for n, m in zip(lens, new)])
    seq, pos = np.concatenate([seq, np.full(pad, -1, np.int32)]), np.concatenate([pos, np.full(pad, 0, np.int32)])
    kp, vp, table, ts, tp, cud = Q.as_cuda(kp, vp, table, seq, pos, cu)
    q = rand(len(seq), heads * D, seed=seed + 1).to(dt).to(DEV)
    out, status = torch.zeros_like(q), torch.zeros(1, dtype=torch.int32, device=DEV)

    def call(to=out):
        ops.attention_q4_prompt(q, kp, vp, table, cud, ts, tp, to, len(new), heads, kv, D, D ** -0.5, max(lens), status)
    return call, q, out, (ks, vs, seq, pos, dt, heads, D ** -0.5), tp


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("lens,new", [([700, 33, 400], [200, 33, 0]), ([500], [20]), ([128, 300], [128, 1])])
def test_prompts_with_padding_and_with_sequences_that_bring_nothing(lens, new, dt):
    call, q, out, (ks, vs, seq, pos, *rest), _ = prompt_call(dt, lens, new, pad=5)
    call()
    n = sum(new)
    check_rows(out[:n], q[:n], ks, vs, seq[:n], pos[:n], *rest)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("lens,new", [([700, 200], [200, 90]), ([500], [20])])
def test_prompts_captured_and_replayed_on_other_places(lens, new, dt):
    call, q, out, (ks, vs, seq, pos, *rest), tp = prompt_call(dt, lens, new)
    call()
    check_rows(out, q, ks, vs, seq, pos, *rest)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    out.zero_()
    tp -= 60        # the same tokens, each 60 positions earlier
    q.copy_(rand(*q.shape, seed=9).to(dt))
    graph.replay()
    check_rows(out, q, ks, vs, seq, pos - 60, *rest)


@pytest.mark.parametrize("dt", [F32, BF16])
def test_calls_on_two_streams_do_not_disturb_one_another(dt):
    a, _, out_a, _, _ = prompt_call(dt, [900, 300], [300, 200], seed=3)
    b, _, out_b, _, _ = prompt_call(dt, [500], [40], seed=4)
    a(), b()
    torch.cuda.synchronize()
    want_a, want_b = out_a.clone(), out_b.clone()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[torch.zeros_like(out_a) for _ in range(6)], [torch.zeros_like(out_b) for _ in range(6)]]
    torch.cuda.synchronize()
    for i in range(6):
        for call, to, stream in zip((a, b), got, streams):
            with torch.cuda.stream(stream):
                call(to[i])
    torch.cuda.synchronize()
    assert all(torch.equal(t, want_a) for t in got[0]) and all(torch.equal(t, want_b) for t in got[1])


@pytest.mark.parametrize("dt", [F32, BF16])
def test_the_same_bits_without_launches_that_overlap(dt):
    def run():
        kp, vp, table, _, _ = Q.filled_cache([200, 4097, 65], 2, 128, 6)
        kp, vp, table, seq, pos = Q.as_cuda(kp, vp, table, np.arange(3, dtype=np.int32), np.array([199, 4096, 64], np.int32))
        q, out = torch.empty(3, 1024, dtype=dt, device=DEV), torch.empty(3, 1024, dtype=dt, device=DEV)
        qkv = rand(3, 12 * 128, seed=2).to(DEV)
        ops.qk_norm_rope_append_q4(qkv, None, None, 1e-6, None, seq, pos, table, kp, vp, q, 8, 2, 128)
        ops.attention_q4(q, kp, vp, table, seq, pos, out, 8, 2, 128, 0.1)
        k = torch.empty(3, 256, device=DEV)
        ops.q4_read(kp, vp, table, seq, pos, k, torch.empty_like(k))
        call, _, prompt, _, _ = prompt_call(dt, [700, 200], [200, 90])
        call()
        torch.cuda.synchronize()
        return out, k, prompt
    want = run()
    ops.launch_overlap(False)
    try:
        got = run()
    finally:
        ops.launch_overlap(True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dt", [F32, BF16])
def test_no_tokens(dt):
    kp, vp, table, _, _ = Q.filled_cache([64], 1, 64, 0)
    before = kp.copy()
    kp, vp, table, none = Q.as_cuda(kp, vp, table, np.zeros(0, np.int32))
    cu, status = torch.zeros(2, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    q, kv = torch.empty(0, 64, dtype=dt, device=DEV), torch.empty(0, 64, device=DEV)
    ops.qk_norm_rope_append_q4(torch.empty(0, 192, device=DEV), None, None, 1e-6, None, none, none, table, kp, vp, q, 1, 1, 64)
    ops.q4_read(kp, vp, table, none, none, kv, kv.clone())
    ops.attention_q4(q, kp, vp, table, none, none, torch.empty_like(q), 1, 1, 64, 0.1)
    ops.attention_q4_prompt(q, kp, vp, table, cu, none, none, torch.empty_like(q), 1, 1, 1, 64, 0.1, 64, status)
    assert np.array_equal(kp.cpu().numpy(), before)


@pytest.mark.parametrize("dt", [F32, BF16])
def test_sequences_without_a_table(dt):
    """A token of a sequence behind the tables' last is nobody's: nothing is written, zeros are read, and it attends to nothing."""
    kp, vp, table, ks, vs = Q.filled_cache([100, 70], 2, 128, 0)
    before = kp.copy()
    seq = np.array([1, 2, 900, 0], np.int32)
    pos = np.array([69, 5, 0, 99], np.int32)
    kp, vp, table, ts, tp = Q.as_cuda(kp, vp, table, seq, pos)
    q = rand(4, 1024).to(dt).to(DEV)
    out = torch.full_like(q, 3.0)
    ops.attention_q4(q, kp, vp, table, ts, tp, out, 8, 2, 128, 0.1)
    check_rows(out, q, ks, vs, [1, -1, -1, 0], pos, dt, 8, 0.1)
    k, v = torch.ones(4, 256, device=DEV), torch.ones(4, 256, device=DEV)
    ops.q4_read(kp, vp, table, ts, tp, k, v)
    assert (k[1:3] == 0).all() and (v[1:3] == 0).all() and (k[0] != 0).any() and (k[3] != 0).any()
    ops.qk_norm_rope_append_q4(rand(2, 12 * 128).to(DEV), None, None, 1e-6, None, ts[1:3].clone(), tp[1:3].clone(), table, kp, vp, q[:2], 8, 2, 128)
    assert np.array_equal(kp.cpu().numpy(), before)


def test_scratch_that_starts_off_its_boundary_is_refused():
    lens, new = [700, 200], [200, 90]
    kp, vp, table, _, _ = Q.filled_cache(lens, 2, 128, 0)
    seq, pos, cu = places(new, [500, 110])
    kp, vp, table, ts, tp, cu = Q.as_cuda(kp, vp, table, seq, pos, cu)
    q = rand(290, 1024).bfloat16().to(DEV)
    need = ops.attention_q4_prompt_scratch_bytes(290, 2, 8, 2, 128, BF16, 700)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    for scratch in (torch.empty(need + 8, dtype=torch.uint8, device=DEV)[8:], torch.empty(need - 1, dtype=torch.uint8, device=DEV),
                    torch.empty(need, dtype=torch.int8, device=DEV)):
        with pytest.raises(Exception, match="scratch"):
            ops.attention_q4_prompt(q, kp, vp, table, cu, ts, tp, torch.empty_like(q), 2, 8, 2, 128, 0.1, 700, status, scratch=scratch)


@pytest.mark.parametrize("dt", [F32, BF16])
def test_pages_behind_four_gigabytes(dt):
    """The same pages at the end of a cache of more than 2^32 bytes: the same bits."""
    kv, D, lens = 8, 128, [300, 64, 1]
    kp, vp, table, _, _ = Q.filled_cache(lens, kv, D, 4)
    first = (1 << 32) // (kv * 40 * D) + 50
    small = Q.as_cuda(kp, vp, table)
    big = [torch.empty(first + len(kp), kv, 40 * D, dtype=torch.uint8, device=DEV) for _ in range(2)]
    for b, s in zip(big, small):
        b[first:] = s
    seq, pos, cu = places([200, 64, 1], [100, 0, 0])
    ts, tp, cud, every, last = Q.as_cuda(seq, pos, cu, np.arange(3, dtype=np.int32), np.array(lens, np.int32) - 1)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    qkv, q = rand(3, 48 * 128, seed=1).to(DEV), rand(len(seq), 32 * 128, seed=2).to(dt).to(DEV)

    def results(k, v, bt):
        token, prompt, held = torch.zeros(3, 32 * 128, dtype=dt, device=DEV), torch.zeros_like(q), torch.zeros(len(seq), kv * D, device=DEV)
        new_q = torch.empty_like(token)
        ops.qk_norm_rope_append_q4(qkv, None, None, 1e-6, None, every, last, bt, k, v, new_q, 32, kv, D)
        ops.attention_q4(new_q, k, v, bt, every, last, token, 32, kv, D, 0.1)
        ops.attention_q4_prompt(q, k, v, bt, cud, ts, tp, prompt, 3, 32, kv, D, 0.1, 300, status)
        ops.q4_read(k, v, bt, ts, tp, held, torch.empty_like(held))
        return token, prompt, held
    want = results(*small)
    got = results(*big, torch.where(small[2] < 0, small[2], small[2] + first))
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and (want[2] != 0).any()
