"""Verification of drafted trees (dsv4cu_verify_greedy, dsv4cu_verify_sample) against the plain form in 64 bits:
tokens, paths and slots are whole numbers and have to be equal."""
from __future__ import annotations

import random

import pytest

import canary
import servefix

pytestmark = pytest.mark.gpu


def _i(x):
    import torch
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _trees(rng, lens):
    cu, parent = [0], []
    for n in lens:
        parent += [rng.choice([-1, 0, 5]) if i == 0 else max(0, i - 1 - int(rng.random() ** 2 * i)) for i in range(n)]
        cu.append(cu[-1] + n)
    return cu, parent


def _inputs(rng, seed, lens, vocab, sharp, drafted, flat=False):
    import torch
    gen = torch.Generator().manual_seed(seed)
    cu, parent = _trees(rng, lens)
    t = cu[-1]
    logits = torch.randn(t, vocab, generator=gen) * sharp
    p = torch.softmax(logits, 1)
    q = torch.softmax(logits + torch.randn(t, vocab, generator=gen) * (0 if flat else 0.7), 1) if drafted else None
    tokens = []
    for b, n in enumerate(lens):
        for i in range(n):
            row = cu[b] + max(0, parent[cu[b] + i]) if i else cu[b]
            src = q if drafted else p
            tokens.append(int(torch.multinomial(src[row], 1, generator=gen)))
    u = torch.rand(t, generator=gen)
    slot = torch.randperm(t, generator=gen).tolist()
    return cu, parent, tokens, p, q, u, slot


def _sample(dev, cu, parent, tokens, p, q, u, slot, guard=True):
    import torch
    n, t = len(cu) - 1, len(tokens)
    make = canary.guarded_empty if guard else (lambda m, d: torch.empty(m, dtype=d, device="cuda"))
    out = [make(m, torch.int32) for m in (n, n, t, t)]
    dev.verify_sample(out[0], out[1], out[2], _i(tokens), _i(parent), _i(cu), p.cuda(), u.cuda(),
                      draft=None if q is None else q.cuda(), slot=_i(slot), slot_out=out[3])
    got = [x.tolist() for x in out]
    for x in out:
        canary.check(x)
    return got


@pytest.mark.parametrize("drafted", [False, True])
@pytest.mark.parametrize("lens,vocab", [([1], 2), ([1], 1), ([2], 7), ([5], 1000), ([3, 0, 1, 9], 333), ([16] * 9, 4099),
                                        ([64, 1, 128], 515), ([8] * 21, 32000), ([6, 2], 129280)])
def test_sampled(dev, lens, vocab, drafted):
    for seed in range(4):
        rng = random.Random(seed)
        x = _inputs(rng, seed + vocab, lens, vocab, sharp=rng.choice([0.3, 2.0, 4.0]), drafted=drafted)
        cu, parent, tokens, p, q, u, slot = x
        want = servefix.verify(tokens, parent, cu, probs=p, u=u, draft=q, slot=slot)
        got = _sample(dev, *x)
        for name, a, b in zip(("accepted", "next", "path", "slot"), got, want):
            assert a == b, (name, seed)


def test_drafts_of_the_target_are_always_accepted(dev):
    rng = random.Random(1)
    cu, parent, tokens, p, q, u, slot = _inputs(rng, 3, [7] * 5, 900, 2.0, True, flat=True)
    parent = [-1 if i % 7 == 0 else i % 7 - 1 for i in range(35)]              # chains, draft equal to the target
    tokens = [x if i % 7 == 0 else int(p[i - 1].argmax()) for i, x in enumerate(tokens)]
    got = _sample(dev, cu, parent, tokens, p, p, u, slot)
    assert got[0] == [6] * 5 and got[2] == list(range(7)) * 5


def test_edges_of_the_numbers(dev):
    """u of 0 and just below 1, an empty remainder, zero rows, NaN rows, tokens outside the vocabulary."""
    import torch
    v = 300
    p = torch.zeros(7, v)
    p[0, 5], p[0, 290] = 0.25, 0.75
    p[1, 7] = 1.0
    p[2] = 0.0
    p[3] = float("nan")
    p[4, 0] = p[4, v - 1] = 0.5
    p[5, 3] = 1.0
    p[6, 9] = 1.0
    top = 1 - 2.0 ** -24
    one = lambda parent, tokens, rows, u, q=None: _sample(  # noqa: E731
        dev, [0, len(rows)], parent, tokens, p[rows], q, torch.tensor(u), list(range(len(rows))))
    assert one([-1], [0], [0], [0.0])[1] == [5] and one([-1], [0], [0], [0.25])[1] == [290]
    assert one([-1], [0], [0], [top])[1] == [290] and one([-1], [0], [4], [top])[1] == [v - 1]
    assert one([-1], [0], [2], [0.5])[1] == [-1] and one([-1], [0], [3], [0.5])[1] == [-1]
    # a certain draft of the only token is refused never; its double afterwards not tested
    assert one([-1, 0, 0], [0, 7, 7], [1, 5, 6], [0.5, top, 0.0])[:3] == [[1], [3], [0, 1, -1]]
    # drafts outside the vocabulary are refused and leave the row as it was
    assert one([-1, 0, 0], [0, -1, v], [0, 1, 1], [0.3, 0.0, 0.0])[:2] == [[0], [290]]
    # the remainder is empty (draft equal to the target, token of no mass): the target's row itself
    q = p[[0, 1]].clone()
    assert one([-1, 0], [0, 8], [0, 1], [0.1, 0.0], q)[:2] == [[0], [5]]


def test_uniforms_cover_the_target(dev):
    """Over an even grid of numbers the drawn tokens have the target's frequencies: the counts of a single node."""
    import torch
    vocab, n = 37, 4000
    p = torch.softmax(torch.randn(1, vocab, generator=torch.Generator().manual_seed(2)), 1)
    u = (torch.arange(n, dtype=torch.float32) + 0.5) / n
    got = _sample(dev, list(range(n + 1)), [-1] * n, [0] * n, p.expand(n, vocab).contiguous(), None, u, list(range(n)))
    count = torch.bincount(torch.tensor(got[1]), minlength=vocab).double()
    # an interval of length p holds between p n - 1 and p n + 1 grid points; the fp32 sum of p is 1 to 1e-6
    assert bool(((count - p[0].double() * n).abs() <= 1 + n * 2e-6).all())


def test_acceptance_keeps_the_target(dev):
    """One drafted token of every value q draws from, tested at an even grid: accepted plus redrawn tokens have the
    target's frequencies, sum over x of q(x) [accept(x) at x + (1 - accept(x)) rest(.)] = p."""
    import torch
    vocab, n = 6, 2000
    gen = torch.Generator().manual_seed(9)
    p = torch.softmax(torch.randn(vocab, generator=gen), 0)
    q = torch.softmax(torch.randn(vocab, generator=gen), 0)
    total = torch.zeros(vocab, dtype=torch.float64)
    for x in range(vocab):
        tokens, parent, u, cu = [], [], [], [0]
        for i in range(n):
            tokens += [0, x]
            parent += [-1, 0]
            u += [((i * 617) % n + 0.5) / n, (i + 0.5) / n]
            cu.append(cu[-1] + 2)
        rows = p.expand(2 * n, vocab).contiguous()
        acc, nxt, _, _ = _sample(dev, cu, parent, tokens, rows, q.expand(2 * n, vocab).contiguous(), torch.tensor(u),
                                 list(range(2 * n)))
        first = torch.tensor([x if a else t for a, t in zip(acc, nxt)])
        total += float(q[x]) * torch.bincount(first, minlength=vocab).double() / n
    # refused cases draw from numbers spread evenly but not independent of the grid: a discrepancy of O(sqrt(n) / n)
    assert float((total - p.double()).abs().max()) < 3 / n ** 0.5


@pytest.mark.parametrize("lens", [[1], [2], [5, 0, 3], [128], [9] * 40, [64, 33, 1]])
def test_greedy(dev, lens):
    import torch
    for seed in range(3):
        rng = random.Random(seed)
        cu, parent = _trees(rng, lens)
        t = cu[-1]
        best = [rng.randrange(3) for _ in range(t)]
        tokens = [rng.randrange(3) for _ in range(t)]
        slot = rng.sample(range(t), t)
        n = len(lens)
        out = [canary.guarded_empty(m, torch.int32) for m in (n, n, t, t)]
        dev.verify_greedy(out[0], out[1], out[2], _i(tokens), _i(parent), _i(cu), _i(best), slot=_i(slot), slot_out=out[3])
        want = servefix.verify(tokens, parent, cu, best=best, slot=slot)
        for x, w in zip(out, want):
            assert x.tolist() == w
            canary.check(x)


def test_greedy_takes_argmax(dev):
    """verify_greedy behind dsv4cu_argmax: the path follows the logits' own picks."""
    import torch
    logits = torch.randn(6, 1000, generator=torch.Generator().manual_seed(4)).cuda()
    best = torch.empty(6, dtype=torch.int32, device="cuda")
    dev.argmax(best, logits, 1000, 6)
    b = best.tolist()
    tokens = [0, b[0], 999, b[1], b[3], 1]
    out = [torch.empty(m, dtype=torch.int32, device="cuda") for m in (1, 1, 6)]
    dev.verify_greedy(*out, _i(tokens), _i([-1, 0, 0, 1, 3, 4]), _i([0, 6]), best)
    acc = 3 + (b[4] == 1)
    assert out[0].tolist() == [acc] and out[1].tolist() == [b[4] if acc == 3 else b[5]]


def test_too_many_nodes_are_refused(dev):
    import torch
    n = 129 + 3
    out = [torch.full((m,), 77, dtype=torch.int32, device="cuda") for m in (2, 2, n, n)]
    zero = torch.zeros(n, dtype=torch.int32, device="cuda")
    cu = _i([0, 129, n])
    dev.verify_greedy(out[0], out[1], out[2], zero, zero, cu, zero, slot=zero, slot_out=out[3])
    assert dev.status_code() == 76
    assert out[0].tolist()[0] == 0 and out[1].tolist()[0] == -1 and out[2].tolist()[:129] == [-1] * 129
    p = torch.full((n, 8), 0.125, device="cuda")
    dev.verify_sample(out[0], out[1], out[2], zero, zero, cu, p, torch.zeros(n, device="cuda"), slot=zero, slot_out=out[3])
    assert dev.status_code() == 76
    assert out[1].tolist()[0] == -1 and out[1].tolist()[1] >= 0


def test_rows_with_strides_and_other_streams(dev):
    """Probabilities inside wider rows, on a stream of their own, captured and replayed on new numbers."""
    import torch
    rng = random.Random(3)
    cu, parent, tokens, p, q, u, slot = _inputs(rng, 8, [6, 4, 1, 7], 2001, 2.0, True)
    t, n = len(tokens), 4
    wide = torch.full((2, t, 2304), float("nan"), device="cuda")
    wide[0, :, :2001], wide[1, :, :2001] = p.cuda(), q.cuda()
    du = u.cuda()
    out = [torch.empty(m, dtype=torch.int32, device="cuda") for m in (n, n, t)]
    args = (out[0], out[1], out[2], _i(tokens), _i(parent), _i(cu), wide[0, :, :2001], du)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        dev.verify_sample(*args, draft=wide[1, :, :2001])
    s.synchronize()
    want = servefix.verify(tokens, parent, cu, probs=p, u=u, draft=q)
    assert [x.tolist() for x in out] == list(want[:3])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        dev.verify_sample(*args, draft=wide[1, :, :2001])
    for seed in range(5):
        u2 = torch.rand(t, generator=torch.Generator().manual_seed(seed))
        du.copy_(u2)
        g.replay()
        torch.cuda.synchronize()
        want = servefix.verify(tokens, parent, cu, probs=p, u=u2, draft=q)
        assert [x.tolist() for x in out] == list(want[:3])


@pytest.mark.parametrize("vocab,at", [(300, 0), (300, 299), (4099, 2048), (129280, 77777)])
def test_rows_without_a_finite_sum_give_no_token(dev, vocab, at):
    """An infinite probability is no distribution: next is -1, with and without drafts, refused or not, whatever u is.
    The walk itself goes on by its comparisons."""
    import torch
    p = torch.full((3, vocab), 1.0 / vocab)
    p[1, at] = float("inf")
    top = 1 - 2.0 ** -24
    one = lambda rows, parent, tokens, u, q=None: _sample(  # noqa: E731
        dev, [0, len(rows)], parent, tokens, p[rows], None if q is None else q[rows], torch.tensor(u),
        list(range(len(rows))))
    other = (at + 1) % vocab
    q = torch.full((3, vocab), 1.0 / vocab)
    q[:, other] = 0.5
    for u in (0.0, 0.5, top):
        assert one([1], [-1], [0], [u])[1] == [-1]                      # the root's row
        assert one([1], [-1], [0], [u], q)[1] == [-1]
        assert one([0, 1], [-1, 0], [0, 5], [u, 0.0])[:2] == [[1], [-1]]    # the row behind an accepted node
        # a refused draft leaves an infinite remainder of an infinite row
        assert one([1, 0], [-1, 0], [0, other], [u, 0.9])[:2] == [[0], [-1]]
        assert one([1, 0], [-1, 0], [0, other], [u, 0.9], q)[:2] == [[0], [-1]]
        # the infinite entry itself is taken, and the finite row behind it gives a token
        assert one([1, 2], [-1, 0], [0, at], [u, top])[0] == [1]
        assert 0 <= one([1, 2], [-1, 0], [0, at], [u, top])[1][0] < vocab
    # a finite row whose draft was refused: the first token that is left
    assert one([2, 0], [-1, 0], [0, other], [0.0, top])[1] == [0 if other else 1]
