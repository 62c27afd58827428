"""Log probabilities of given tokens, entropies and best alternatives against 64 bits."""
import numpy as np
import pytest
import torch

from nncpu_b200.kernels import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def plain(x, targets, k):
    """x float64 [n, vocab] with NaN as -inf -> (logprobs, entropy, top, ids)."""
    x = np.where(np.isnan(x), -np.inf, x)
    n, vocab = x.shape
    lp, en, top, ids = np.zeros(n), np.zeros(n), np.zeros((n, k)), np.zeros((n, k), dtype=np.int64)
    for r in range(n):
        m = x[r].max()
        order = np.lexsort((np.arange(vocab), -x[r]))[:k]
        ids[r] = order
        if m == -np.inf:
            p = np.full(vocab, -np.inf)
        elif m == np.inf:
            p = np.full(vocab, np.nan)
            en[r] = np.nan
        else:
            with np.errstate(divide="ignore"):
                p = x[r] - m - np.log(np.exp(x[r] - m).sum())
            live = p > -np.inf
            en[r] = -(np.exp(p[live]) * p[live]).sum()
        lp[r] = p[targets[r]] if 0 <= targets[r] < vocab else np.nan
        top[r] = p[order]
    return lp, en, top, ids


def run(logits, targets, k):
    n = logits.shape[0]
    lp, en = torch.full((n,), 9.0, device=DEV), torch.full((n,), 9.0, device=DEV)
    top = torch.full((n, k), 9.0, device=DEV) if k else None
    ids = torch.full((n, k), -7, dtype=torch.int32, device=DEV) if k else None
    ops.token_logprobs(logits, targets, lp, en, top, ids)
    return lp, en, top, ids


def check(logits, targets, k):
    want = plain(logits.double().cpu().numpy(), targets.cpu().numpy(), k)
    got = run(logits, targets, k)
    vocab = logits.shape[1]
    for name, g, w in zip(("logprobs", "entropy", "top"), got, want):
        if g is None:
            continue
        g = g.double().cpu().numpy()
        assert np.array_equal(np.isnan(g), np.isnan(w)) and np.array_equal(np.isinf(g), np.isinf(w)), name
        fine = np.isfinite(w)
        # exponentials are within two units in the last place and sums of positive numbers within some 2^-20 (a thread adds some
        # hundred of them); a difference of two numbers as large as the logits' spread is rounded
        spread = np.abs(logits.double().cpu().numpy())
        size = np.where(np.isfinite(spread), spread, 0).max() if spread.size else 0.0
        tol = 2.0 ** -20 * (1 + np.log(vocab)) + 2.0 ** -22 * size
        assert (np.abs(g[fine] - w[fine]) <= tol).all(), (name, np.abs(g[fine] - w[fine]).max(), tol)
    if k:
        assert np.array_equal(got[3].cpu().numpy(), want[3])


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,vocab,k", [(1, 1, 1), (1, 2, 2), (3, 7, 0), (5, 384, 20), (2, 1025, 32), (3, 33, 33 - 1), (70, 4100, 31), (9, 4099, 5), (1, 151936, 20), (300, 257, 1),
                                       (3, 50257, 10), (8, 151936, 5), (2, 200003, 3), (40, 32768, 2), (2, 400001, 8)])
def test_rows(n, vocab, k, dt):
    g = torch.Generator().manual_seed(n * vocab)
    logits = (torch.randn(n, vocab, generator=g) * (0.2 + 4 * torch.rand(n, 1, generator=g))).to(dt).to(DEV)
    targets = torch.randint(0, vocab, (n,), generator=g, dtype=torch.int32).to(DEV)
    check(logits, targets, k)


@pytest.mark.parametrize("vocab", [5, 1000, 151936])
def test_ties_go_to_the_lowest_id(vocab):
    k = min(vocab, 7)
    x = torch.zeros(4, vocab, device=DEV)
    x[1] = -0.0
    x[1, ::2] = 0.0                        # zeros of both signs are equal
    x[2, vocab // 2:] = 3.0
    x[3] = -torch.inf
    check(x, torch.tensor([0, vocab - 1, vocab // 2, 2], dtype=torch.int32, device=DEV), k)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_rows_in_order_and_masked_rows(dt):
    # ascending logits pass every bar, descending ones none; a mask that leaves fewer tokens than are asked for
    vocab = 40001
    up = torch.linspace(-3, 3, vocab, device=DEV)
    x = torch.stack([up, up.flip(0), torch.full_like(up, -torch.inf), torch.full_like(up, 2.5), torch.full_like(up, -1e30)]).to(dt)
    x[2, torch.tensor([39999, 7, 20000], device=DEV)] = 1.0
    x[4, 17::5000] = torch.arange(8, device=DEV).to(dt)
    check(x, torch.tensor([vocab - 1, 0, 7, 3, 17], dtype=torch.int32, device=DEV), 20)


@pytest.mark.parametrize("vocab", [9, 3001, 151936])
def test_rows_of_nothing_of_infinities_and_nan(vocab):
    x = torch.randn(7, vocab, generator=torch.Generator().manual_seed(1)).to(DEV)
    x[0] = -torch.inf
    x[1] = torch.nan
    x[2, 1:] = -torch.inf                  # one token is left
    x[3, ::3] = torch.nan
    x[4, 4] = torch.inf
    x[5, 2] = 1e4                          # decided
    x[6] = torch.finfo(torch.float32).min  # a mask of the type's lowest value: even
    targets = torch.tensor([3, 0, 0, 3, 4, 2, vocab - 1], dtype=torch.int32, device=DEV)
    check(x, targets, 6)
    check(x, targets, 0)
    check(x, (targets + 1) % vocab, 1)


def test_targets_outside_the_vocabulary():
    x = torch.randn(4, 50, device=DEV)
    lp, en, _, _ = run(x, torch.tensor([-1, 50, 2 ** 31 - 1, 49], dtype=torch.int32, device=DEV), 0)
    assert lp[:3].isnan().all() and lp[3].isfinite() and en.isfinite().all()


def test_no_rows():
    run(torch.empty(0, 10, device=DEV), torch.empty(0, dtype=torch.int32, device=DEV), 2)


def test_a_nearly_decided_row_keeps_its_small_entropy():
    # p = 1 - 2e-7 and the rest on one token: the entropy is 3.3e-6, of which 32 bits around 1 would lose most
    x = torch.tensor([[0.0, -15.424948]], device=DEV)
    lp, en, _, _ = run(x, torch.zeros(1, dtype=torch.int32, device=DEV), 0)
    want = plain(x.double().cpu().numpy(), [0], 0)
    assert abs(float(en[0]) - want[1][0]) <= 2.0 ** -23 and abs(float(lp[0]) - want[0][0]) <= 2.0 ** -23


def test_captured_and_replayed_on_other_logits():
    x = torch.randn(3, 151936, device=DEV)
    t = torch.tensor([5, 77, 151935], dtype=torch.int32, device=DEV)
    lp, en = torch.empty(3, device=DEV), torch.empty(3, device=DEV)
    top, ids = torch.empty(3, 4, device=DEV), torch.empty(3, 4, dtype=torch.int32, device=DEV)
    ops.token_logprobs(x, t, lp, en, top, ids)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.token_logprobs(x, t, lp, en, top, ids)
    x.copy_(torch.randn(3, 151936, generator=torch.Generator().manual_seed(3)))
    for _ in range(2):
        graph.replay()
        want = run(x, t, 4)
        for a, b in zip((lp, en, top, ids), want):
            assert torch.equal(a, b)


def test_on_another_stream_and_twice_the_same_bits():
    x = torch.randn(5, 100003, device=DEV)
    t = torch.arange(5, dtype=torch.int32, device=DEV)
    want = run(x, t, 9)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = run(x, t, 9)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_rows_behind_two_to_the_31_logits():
    n, vocab = 32800, 65536
    logits = torch.zeros(n, vocab, dtype=torch.bfloat16, device=DEV)
    logits[-3:] = torch.randn(3, vocab, generator=torch.Generator().manual_seed(0)).to(DEV)
    targets = torch.arange(n, dtype=torch.int32, device=DEV)

    def ask(x, t):
        lp, entropy, top, ids = (torch.empty(len(x), *s, device=DEV, dtype=d) for s, d in (((), torch.float32), ((), torch.float32),
                                                                                           ((4,), torch.float32), ((4,), torch.int32)))
        ops.token_logprobs(x, t, lp, entropy, top, ids)
        return lp, entropy, top, ids
    got = ask(logits, targets)
    few = ask(logits[-3:].clone(), targets[-3:].clone())
    assert torch.equal(got[3][-3:], few[3]) and (got[3][:-3] == torch.arange(4, device=DEV)).all()
    for a, b in zip(got[:3], few[:3]):       # (the few rows are shared by clusters: another order of 32-bit sums of 65 536 terms)
        assert torch.allclose(a[-3:], b, rtol=0, atol=1e-5)
    assert torch.allclose(got[0][:-3].double(), torch.tensor(-np.log(vocab)).double().to(DEV), rtol=0, atol=1e-5)
