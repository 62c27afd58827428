"""A key/value cache of 4 bits and the log probabilities that tell what it costs, as cases that can be timed and checked.

Three operators of the library, each through its own call: the append to the cache (norm and rotation of the heads on the way, with
what the cache then holds read back), the attention that reads it (one token a sequence, and prompts or portions of them), and the
log probabilities of given tokens with the distribution's entropy and its best alternatives.

The cache's pages are built here in their documented layout, so that both forms read the same bytes.  A page holds 64
positions of one key/value head; a head's lanes lie in groups of 32, and a lane's value is d c + m with c in 0..15 and the group's
float16 numbers d (a step) and m (its least value):

* key page: 64 rows of D / 2 bytes, then 64 rows of D / 32 pairs (d, m).  A row is 32-bit words [4][D / 32]; the
  word (c, g) holds the codes of lanes 32 g + 8 c + i at its bits 4 i, i = 0..7.
* value page: words [8][8][4][D / 32], then 64 rows of D / 32 pairs (d, m).  The word (b, r, p, g) holds position
  8 b + 2 p in its lower half and 8 b + 2 p + 1 in its upper one, each the codes of lanes 32 g + 4 r + i at its bits 4 i, i = 0..3.

Head counts are those of the benchmark's models (32, 40 and 16 heads over 8, heads of 128 lanes) and of the tests' small ones;
the vocabulary is the benchmark's.
"""
from __future__ import annotations

import math

import torch

own = False

PAGE = 64
GROUP = 32
EPS = 1e-6
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
VOCAB = 151936


def listed():
    return [
        # one user's next token: the smallest append there is, all latency
        dict(name="append-1", kind="append", seqs=1, new=1, past=700, heads=32, kv=8, dim=128, norm=True, rotary=True, dtype="bfloat16"),
        # a full server's decode step: 64 sequences of unequal lengths, one token each
        dict(name="append-64", kind="append", seqs=64, new=1, past=1000, heads=32, kv=8, dim=128, norm=True, rotary=True,
             dtype="bfloat16"),
        # the benchmark's prompt, starting in the middle of a page (a conversation goes on)
        dict(name="append-prompt-2048", kind="append", seqs=1, new=2048, past=37, heads=32, kv=8, dim=128, norm=True, rotary=True,
             dtype="bfloat16"),
        # one user's reply in the middle of a context: few keys for a whole device
        dict(name="decode-1", kind="decode", seqs=1, length=2500, heads=32, kv=8, dim=128, window=0, dtype="bfloat16"),
        # a server's batch of conversations of very unequal lengths with 14B-sized layers
        dict(name="decode-16-unequal", kind="decode", seqs=16, length=4500, heads=40, kv=8, dim=128, window=0, dtype="bfloat16"),
        # many long contexts at once: the stream over the cache is all there is
        dict(name="decode-64-long", kind="decode", seqs=64, length=8000, heads=32, kv=8, dim=128, window=0, dtype="bfloat16"),
        # a check run in 32 bits over the same kind of cache, with the small models' heads
        dict(name="decode-float32", kind="decode", seqs=4, length=1000, heads=16, kv=4, dim=64, window=0, dtype="float32"),
        # a chat message of a few words after a conversation
        dict(name="turn-24", kind="prompt", seqs=1, new=24, past=3001, heads=32, kv=8, dim=128, window=0, dtype="bfloat16"),
        # the benchmark's prompt
        dict(name="prompt-2048", kind="prompt", seqs=1, new=2048, past=0, heads=32, kv=8, dim=128, window=0, dtype="bfloat16"),
        # a decode step whose caller asked for the chosen tokens' log probabilities and five alternatives
        dict(name="logprobs-8", kind="logprobs", rows=8, vocab=VOCAB, top=5, dtype="float32"),
        # a text of a thousand and one tokens scored in one go: how well a model predicts it
        dict(name="logprobs-text", kind="logprobs", rows=1001, vocab=VOCAB, top=0, dtype="float32"),
        # the same with alternatives for every token, over a vocabulary that no tile divides
        dict(name="logprobs-top-20", kind="logprobs", rows=300, vocab=50257, top=20, dtype="float32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "append", "decode", "decode", "decode", "prompt", "prompt", "logprobs", "logprobs"])
    heads, kv = rng.choice([(32, 8), (32, 8), (40, 8), (16, 8), (16, 4), (8, 2), (64, 8), (24, 2), (5, 1)])
    dim = rng.choice([128, 128, 128, 64, 64, 32, 96])
    dtype = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
    shape = dict(heads=heads, kv=kv, dim=dim)
    if kind == "append":
        seqs = _log(rng, 1, 64)
        new = 1 if rng.random() < 0.5 else _log(rng, 2, max(2, 2048 // seqs))
        return dict(kind=kind, seqs=seqs, new=new, past=rng.choice([0, _log(rng, 1, 2000)]), norm=rng.random() < 0.7,
                    rotary=rng.random() < 0.8, dtype=dtype, **shape)
    if kind == "decode":
        seqs = _log(rng, 1, 64)
        limit = 260_000 // seqs if dtype == "bfloat16" and dim in (64, 128) else 16_000 // seqs
        length = _log(rng, 1, max(2, min(8000, limit)))
        return dict(kind=kind, seqs=seqs, length=length, window=rng.choice([0, 0, _log(rng, 1, 2000)]), dtype=dtype, **shape)
    if kind == "prompt":
        seqs = rng.choice([1, 1, _log(rng, 2, 8)])
        new = _log(rng, 2, max(2, (2048 if dtype == "bfloat16" else 500) // seqs))
        past = rng.choice([0, _log(rng, 1, 3000)])
        past = min(past, max(0, 120_000_000 // (seqs * heads * new) - new))
        return dict(kind=kind, seqs=seqs, new=new, past=past, window=rng.choice([0, 0, 0, _log(rng, 1, 1000)]), dtype=dtype, **shape)
    vocab = rng.choice([VOCAB, VOCAB, _log(rng, 2, 200_000)])
    return dict(kind=kind, rows=_log(rng, 1, min(1000, 150_000_000 // vocab)), vocab=vocab, top=min(vocab, rng.choice([0, 1, 5, 20])),
                dtype=rng.choice(["float32", "float32", "bfloat16"]))


# -- sizes that follow from a case --------------------------------------------------------------------------------------


def _spread(most, n):
    """n numbers from 1 to ``most`` spread over the range, the first of them ``most`` (0: all 0)."""
    return [most if b == 0 or most == 0 else 1 + int((most - 1) * ((0.37 + 0.618034 * b) % 1.0)) for b in range(n)]


def _held(case):
    """(positions before the step, positions that it brings) of every sequence."""
    if case["kind"] == "decode":
        return [n - 1 for n in _spread(case["length"], case["seqs"])], [1] * case["seqs"]
    return _spread(case["past"], case["seqs"]), _spread(case["new"], case["seqs"])


def _seen(case, pos):
    """Keys that the query at position ``pos`` sees."""
    w = case.get("window", 0)
    return min(pos + 1, w) if w else pos + 1


def work(case):
    if case["kind"] == "logprobs":
        n, v, k = case["rows"], case["vocab"], case["top"]
        size = 4 if case["dtype"] == "float32" else 2
        return {"bytes": n * v * size + n * (4 + 8 + 8 * k), "flops": 6 * n * v}
    past, new = _held(case)
    n, heads, kv, dim = sum(new), case["heads"], case["kv"], case["dim"]
    size = 4 if case["dtype"] == "float32" else 2
    position = kv * 2 * dim * 5 // 8          # bytes of a position's keys and values in the cache
    if case["kind"] == "append":
        read = n * (heads + 2 * kv) * dim * 4 + (n * dim * 4 if case["rotary"] else 0) + 8 * n
        read_back = n * 2 * kv * dim * size
        return {"bytes": read + n * heads * dim * size + n * position + read_back, "flops": n * (heads + 2 * kv) * dim * 8}
    keys = sum(_seen(case, p + i) for p, q in zip(past, new) for i in range(q))
    # a sequence's keys are read once, from the first that its first query sees
    held = sum(p + q - (p + 1 - _seen(case, p)) for p, q in zip(past, new))
    return {"bytes": held * position + 2 * n * heads * dim * size, "flops": 4 * keys * heads * dim}


# -- the cache's numbers and pages ---------------------------------------------------------------------------------------


def _quantise(x):
    """float32 [..., D] -> codes [..., D / 32, 32] (as float32), d and m float16 [..., D / 32]."""
    g = x.reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    lo, hi = g.amin(-1), g.amax(-1)
    d = ((hi - lo) / 15).clamp(max=65504.0).half()
    m = lo.clamp(-65504.0, 65504.0).half()
    r = torch.where(d > 0, 1.0 / d.float(), torch.zeros_like(lo))
    c = ((g - m.float()[..., None]) * r[..., None]).round().clamp(0, 15)
    return c, d, m


def _values(c, d, m):
    return (c * d.float()[..., None] + m.float()[..., None]).flatten(-2)


def _words(nibbles):
    """The 32-bit words of codes [..., 8] (int64), the first in the lowest bits, as bytes [..., 4]."""
    w = (nibbles << (4 * torch.arange(8, device=nibbles.device))).sum(-1)
    return ((w[..., None] >> (8 * torch.arange(4, device=w.device))) & 255).to(torch.uint8)


def _pack(x, values):
    """float32 [pages, kv, 64, D] -> uint8 [pages, kv, 40 D], laid out as key pages or as value pages."""
    c, d, m = _quantise(x)
    p, kv, _, g, _ = c.shape
    c = c.long()
    if values:      # positions (b, pair, half), lanes (g, r, i) -> words (b, r, pair, g) of (half, i)
        c = c.view(p, kv, 8, 4, 2, g, 8, 4).permute(0, 1, 2, 6, 3, 5, 4, 7).reshape(p, kv, -1, 8)
    else:           # lanes (g, c, i) -> words (c, g) of i
        c = c.view(p, kv, 64, g, 4, 8).permute(0, 1, 2, 4, 3, 5).reshape(p, kv, -1, 8)
    pairs = torch.stack((d, m), -1).view(p, kv, -1).view(torch.uint8)
    return torch.cat((_words(c).flatten(2), pairs), -1).contiguous()


def _unpack(pages, dim, values):
    """uint8 [..., 40 D] -> float32 [..., 64, D]."""
    g = dim // GROUP
    lead = pages.shape[:-1]
    w = pages[..., :32 * dim].contiguous().view(torch.int32)
    c = (w[..., None] >> (4 * torch.arange(8, device=w.device, dtype=torch.int32))) & 15
    n = len(lead)
    if values:
        c = c.view(*lead, 8, 8, 4, g, 2, 4).permute(*range(n), n, n + 2, n + 4, n + 3, n + 1, n + 5)
    else:
        c = c.view(*lead, 64, 4, g, 8).permute(*range(n), n, n + 2, n + 1, n + 3)
    c = c.reshape(*lead, 64, g, GROUP).float()
    s = pages[..., 32 * dim:].contiguous().view(torch.float16).view(*lead, 64, g, 2)
    return _values(c, s[..., 0], s[..., 1])


# -- what a program has in hand --------------------------------------------------------------------------------------------


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    dt = DTYPES[case["dtype"]]
    if case["kind"] == "logprobs":
        n, vocab = case["rows"], case["vocab"]
        # rows between nearly even and nearly decided; the given tokens are drawn among the likely and the unlikely
        logits = (normal(n, vocab) * (0.5 + 2.5 * torch.rand(n, 1, device="cuda", generator=gen))).to(dt)
        targets = torch.randint(0, vocab, (n,), device="cuda", generator=gen, dtype=torch.int32)
        targets[::2] = logits[::2].argmax(-1).int()
        k = case["top"]
        return dict(case=case, logits=logits, targets=targets, logprobs=torch.empty(n, device="cuda"),
                    entropy=torch.empty(n, device="cuda"), top=torch.empty(n, k, device="cuda") if k else None,
                    ids=torch.empty(n, k, device="cuda", dtype=torch.int32) if k else None)
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    past, new = _held(case)
    n = sum(new)
    per = [(p + q + PAGE - 1) // PAGE for p, q in zip(past, new)]
    width, n_pages = max(per), sum(per) + 2
    order = torch.randperm(n_pages, generator=gen, device="cuda").int()
    table = torch.full((len(per), width), -1, dtype=torch.int32)
    rows = [b for b, c in enumerate(per) for _ in range(c)]
    cols = [j for c in per for j in range(c)]
    table = table.cuda()
    table[torch.tensor(rows, device="cuda"), torch.tensor(cols, device="cuda")] = order[:len(rows)]
    cu = torch.zeros(len(new) + 1, dtype=torch.int32)
    cu[1:] = torch.tensor(new).cumsum(0)
    q_len = torch.tensor(new)
    tok_seq = torch.repeat_interleave(torch.arange(len(new)), q_len).int()
    tok_pos = (torch.arange(n) - cu[tok_seq.long()] + torch.tensor(past)[tok_seq.long()]).int()
    state = dict(case=case, table=table, tok_seq=tok_seq.cuda(), tok_pos=tok_pos.cuda(), cu=cu.cuda(), n=n, longest=max(p + q for p, q in zip(past, new)),
                 status=torch.zeros(1, dtype=torch.int32, device="cuda"))
    if case["kind"] == "append":
        half = dim // 2
        state.update(qkv=normal(n, (heads + 2 * kv) * dim), k_pages=torch.zeros(n_pages, kv, 40 * dim, dtype=torch.uint8, device="cuda"),
                     v_pages=torch.zeros(n_pages, kv, 40 * dim, dtype=torch.uint8, device="cuda"), q=torch.empty(n, heads * dim, dtype=dt, device="cuda"),
                     k=torch.empty(n, kv * dim, dtype=dt, device="cuda"), v=torch.empty(n, kv * dim, dtype=dt, device="cuda"),
                     q_gamma=None, k_gamma=None, cos_sin=None)
        if case["norm"]:
            state.update(q_gamma=(1 + 0.1 * normal(dim)).to(dt), k_gamma=(1 + 0.1 * normal(dim)).to(dt))
        if case["rotary"]:
            angle = state["tok_pos"].double()[:, None] * 1e6 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
            state.update(cos_sin=torch.stack((angle.cos(), angle.sin()), -1).float().contiguous())
        return state
    # keys with a few strong lanes, as trained models have them; what lies behind a sequence's end is an earlier one's
    strong = 1 + 3 * (torch.rand(kv, 1, dim, device="cuda", generator=gen) < 0.05).float()
    parts = [_pack(x, values) for values, make in ((False, lambda m: normal(m, kv, PAGE, dim) * strong), (True, lambda m: normal(m, kv, PAGE, dim)))
             for x in [make(n_pages)]]
    state.update(k_pages=parts[0], v_pages=parts[1], q=normal(n, heads * dim).to(dt), out=torch.empty(n, heads * dim, dtype=dt, device="cuda"))
    if case["kind"] == "prompt":
        # where a flat token lies in the batch of equally long rows, for the plain form
        first = torch.arange(max(new))[None, :].expand(len(new), -1)
        state.update(grid=torch.where(first < q_len[:, None], cu[:-1, None] + first, 0).cuda(),
                     flat=(tok_seq.long() * max(new) + (torch.arange(n) - cu[tok_seq.long()])).cuda(),
                     grid_pos=(torch.tensor(past)[:, None] + first).cuda())
    return state


# -- the operators --------------------------------------------------------------------------------------------------------


def run(s):
    c = s["case"]
    if own:
        return _run_own(s, c)
    return {"append": _append, "decode": _attend, "prompt": _attend, "logprobs": _logprobs}[c["kind"]](s, c)


def _run_own(s, c):
    from nncpu_b200.kernels import ops
    if c["kind"] == "logprobs":
        ops.token_logprobs(s["logits"], s["targets"], s["logprobs"], s["entropy"], s["top"], s["ids"])
        return dict(logprobs=s["logprobs"], entropy=s["entropy"], top=s["top"], ids=s["ids"])
    heads, kv, dim = c["heads"], c["kv"], c["dim"]
    if c["kind"] == "append":
        ops.qk_norm_rope_append_q4(s["qkv"], s["q_gamma"], s["k_gamma"], EPS, s["cos_sin"], s["tok_seq"], s["tok_pos"], s["table"],
                                   s["k_pages"], s["v_pages"], s["q"], heads, kv, dim)
        ops.q4_read(s["k_pages"], s["v_pages"], s["table"], s["tok_seq"], s["tok_pos"], s["k"], s["v"])
        return dict(q=s["q"], k=s["k"], v=s["v"])
    if c["kind"] == "decode":
        ops.attention_q4(s["q"], s["k_pages"], s["v_pages"], s["table"], s["tok_seq"], s["tok_pos"], s["out"], heads, kv, dim,
                         dim ** -0.5, window=c["window"])
    else:
        ops.attention_q4_prompt(s["q"], s["k_pages"], s["v_pages"], s["table"], s["cu"], s["tok_seq"], s["tok_pos"], s["out"],
                                len(s["cu"]) - 1, heads, kv, dim, dim ** -0.5, s["longest"], s["status"], window=c["window"])
    return dict(out=s["out"])


def _norm_rotate(x, gamma, cos_sin):
    """x [n, heads, D] in its type; the rotation turns the pairs of lanes (i, i + D / 2)."""
    if gamma is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * gamma.to(x.dtype)
    if cos_sin is not None:
        cos, sin = cos_sin.to(x.dtype)[:, None].unbind(-1)
        a, b = x.chunk(2, -1)
        x = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return x


def _append(s, c):
    heads, kv, dim, n = c["heads"], c["kv"], c["dim"], s["n"]
    q, k, v = s["qkv"].view(n, heads + 2 * kv, dim).split((heads, kv, kv), 1)
    q = _norm_rotate(q, s["q_gamma"], s["cos_sin"])
    # in 64 bits: a code next to a border is decided by the key's last bit
    k = _norm_rotate(k.double(), s["k_gamma"], s["cos_sin"]).float()
    dt = s["q"].dtype
    return dict(q=q.reshape(n, -1).to(dt), k=_values(*_quantise(k)).reshape(n, -1).to(dt), v=_values(*_quantise(v)).reshape(n, -1).to(dt))


def _attend(s, c):
    heads, kv, dim = c["heads"], c["kv"], c["dim"]
    table = s["table"].clamp(min=0).long()
    seqs, width = table.shape
    k, v = (_unpack(p[table], dim, values).transpose(1, 2).reshape(seqs, kv, width * PAGE, dim)
            for p, values in ((s["k_pages"], False), (s["v_pages"], True)))
    if c["kind"] == "decode":
        q, pos = s["q"].view(seqs, 1, heads, dim), s["tok_pos"][:, None]
    else:
        q, pos = s["q"].view(-1, heads, dim)[s["grid"]], s["grid_pos"]
    t = q.shape[1]
    q = q.float().view(seqs, t, kv, heads // kv, dim).permute(0, 2, 3, 1, 4).reshape(seqs, kv, -1, dim)
    z = (q @ k.transpose(2, 3)).view(seqs, kv, -1, t, width * PAGE) * dim ** -0.5
    key = torch.arange(width * PAGE, device=z.device)
    seen = key <= pos[..., None]
    if c["window"]:
        seen &= key > pos[..., None] - c["window"]
    z = z.masked_fill(~seen[:, None, None], -math.inf)
    z = torch.exp(z - z.amax(-1, keepdim=True))
    o = (z / z.sum(-1, keepdim=True)).view(seqs, kv, -1, width * PAGE) @ v
    o = o.view(seqs, kv, -1, t, dim).permute(0, 3, 1, 2, 4).reshape(seqs * t, heads * dim)
    return dict(out=(o if c["kind"] == "decode" else o[s["flat"]]).to(s["out"].dtype))


def _logprobs(s, c):
    x = s["logits"].float()
    y = x - x.amax(-1, keepdim=True)
    e = torch.exp(y)
    total = e.sum(-1)
    logs = torch.log(total)
    given = y.gather(1, s["targets"].long()[:, None])[:, 0] - logs
    entropy = logs - (e * y).sum(-1) / total
    if not c["top"]:
        return dict(logprobs=given, entropy=entropy, top=None, ids=None)
    # the order of the logits, and of the lower index where two are equal, as that of whole numbers
    bits = (x + 0.0).view(torch.int32).long()
    rank = torch.where(bits >= 0, bits, -2147483648 - bits) * 4194304 + (4194303 - torch.arange(x.shape[1], device=x.device))
    ids = 4194303 - (rank.topk(c["top"], -1).values & 4194303)
    return dict(logprobs=given, entropy=entropy, top=y.gather(1, ids) - logs[:, None], ids=ids.int())


# -- the definitions in 64 bits ---------------------------------------------------------------------------------------------


def _groups64(x):
    """What the cache makes of the float32 numbers x (given as float64 [..., 32]), with the roundings of its definition."""
    lo, hi = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
    d = ((hi - lo).float() / 15).clamp(max=65504).half().double()
    m = lo.float().clamp(-65504, 65504).half().double()
    inverse = torch.where(d > 0, 1 / d, 0 * d).float().double()
    c = torch.round(((x - m).float().double() * inverse).float()).double().clamp(0, 15)
    return d * c + m


def _number64(pages, lanes, values):
    """The numbers of one head's pages uint8 [pages, 40 D], as float64 [pages * 64, D]: byte by byte."""
    dim = lanes
    g = dim // GROUP
    low, high = pages[:, :32 * dim] & 15, pages[:, :32 * dim] >> 4
    nib = torch.stack((low, high), -1).reshape(len(pages), -1)
    tok = torch.arange(64, device=pages.device)[:, None]
    lane = torch.arange(dim, device=pages.device)[None, :]
    if values:
        word = ((tok // 8 * 8 + lane % 32 // 4) * 4 + tok % 8 // 2) * g + lane // 32
        at = word * 8 + tok % 2 * 4 + lane % 4
    else:
        word = tok * (dim // 8) + lane % 32 // 8 * g + lane // 32
        at = word * 8 + lane % 8
    pair = pages[:, 32 * dim:].contiguous().view(torch.float16).double().view(len(pages), 64, g, 2)
    d, m = pair[..., 0].repeat_interleave(32, -1), pair[..., 1].repeat_interleave(32, -1)
    return (nib[:, at].double() * d + m).reshape(-1, dim)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "logprobs":
        given, entropy, top = [], [], []
        for r in range(0, case["rows"], 64):
            x = s["logits"][r:r + 64].double()
            p = x - x.logsumexp(-1, keepdim=True)
            given.append(p[torch.arange(len(p), device="cuda"), s["targets"][r:r + 64].long()])
            entropy.append(-torch.where(p > -math.inf, p.exp() * p, 0 * p.exp()).sum(-1))
            if case["top"]:
                top.append(p.sort(-1, descending=True).values[:, :case["top"]])
        return dict(logprobs=torch.cat(given), entropy=torch.cat(entropy), top=torch.cat(top) if top else None, ids=None)
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    if case["kind"] == "append":
        n = s["n"]
        x = s["qkv"].double().view(n, heads + 2 * kv, dim)
        made = []
        for h in range(heads + kv):
            gamma = s["q_gamma"] if h < heads else s["k_gamma"]
            y = x[:, h]
            if gamma is not None:
                y = y * gamma.double() * (y.square().sum(-1, keepdim=True) / dim + EPS).rsqrt()
            if s["cos_sin"] is not None:
                turn = torch.view_as_complex(s["cos_sin"].double())
                z = torch.complex(y[:, :dim // 2], y[:, dim // 2:]) * turn
                y = torch.cat((z.real, z.imag), -1)
            made.append(y)
        k = torch.stack(made[heads:], 1).float().double()
        v = x[:, heads + kv:]
        k, v = (_groups64(t.reshape(n, kv, dim // 32, 32)).reshape(n, -1) for t in (k, v))
        return dict(q=torch.cat(made[:heads], -1), k=k, v=v)
    past, new = _held(case)
    out, at = [], 0
    for b, (p, t) in enumerate(zip(past, new)):
        pages = s["table"][b, :(p + t + 63) // 64].long()
        q = s["q"][at:at + t].double().view(t, heads, dim)
        at += t
        key = torch.arange(p + t, device="cuda")
        pos = p + torch.arange(t, device="cuda")[:, None]
        hidden = (key > pos) | (key <= pos - (case["window"] or p + t))
        o = []
        for h in range(kv):
            k, v = (_number64(pg[pages, h], dim, values)[:p + t] for pg, values in ((s["k_pages"], False), (s["v_pages"], True)))
            for j in range(h * (heads // kv), (h + 1) * (heads // kv)):
                w = (q[:, j] @ k.T / math.sqrt(dim)).masked_fill(hidden, -math.inf)
                o.append(torch.softmax(w, -1) @ v)
        out.append(torch.stack(o, 1).reshape(t, -1))
    return dict(out=torch.cat(out))
