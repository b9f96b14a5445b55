"""What fp32 queries over bf16 keys promise beyond a worst-case bound: queries and weights keep all 24 significand
bits, and sums over blocks of keys are rounded to nearest. Each is shown by inputs whose exact result hangs on it; the
same checks refuse a form on the CPU that drops it."""
from __future__ import annotations

import pytest

BLOCK = 32                                          # least keys of a block


# ------------------------------------------------------------------ inputs: q [n][heads][dim], k / v [n][1][dim]
def _bf16(x):
    import torch
    return x.to(torch.bfloat16)


def score_bits(n, dim, gen):
    """Two keys of scores near 100 whose difference is below 1: it hangs on the last bits of the queries. All other
    keys weigh e^-64 at most. Values +1 and -1: an output is tanh(difference / 2)."""
    import torch
    q, k, v = torch.zeros(n, 2, dim), torch.zeros(n, 1, dim), torch.zeros(n, 1, dim)
    a = 1.0 + 0.9 * torch.rand(n, 2, generator=gen)
    q[:, :, 0], q[:, :, 1] = a, a + (torch.rand(n, 2, generator=gen) - 0.5) * 2.0 ** -6
    k[0, 0, 0] = k[n // 2, 0, 1] = 512.0
    v[0], v[n // 2] = 1.0, -1.0
    return q, _bf16(k), _bf16(v)


# scale * 512 = 64: scores below 128, in log2 units below 256, rounded once to 24 bits: half a step is 2^-17 each, and an
# output moves by half of what the difference (in nats, x ln 2) moves: 2 x 2^-17 x 0.7 / 2 = 0.7 x 2^-17. The products
# with 512 and their sums are exact, the rounding of the scale is common to both scores, and exp2, sum and division add
# 6 x 2^-23 at most.
SCORE_TOL = 2.0 ** -17


def weight_bits(n, dim, gen):
    """A key of weight 1 and value 0, one of weight w in (0.37, 1) and value 1, others of weight e^-256: w / (1 + w)."""
    import torch
    q, k, v = torch.zeros(n, 2, dim), torch.zeros(n, 1, dim), torch.zeros(n, 1, dim)
    q[:, :, 0] = 0.1 + 7.9 * torch.rand(n, 2, generator=gen)
    q[:, :, 2] = 1.0
    k[:, 0, 2] = -2048.0
    k[0] = k[n // 2] = 0.0
    k[n // 2, 0, 0] = -1.0
    v[n // 2] = 1.0
    return q, _bf16(k), _bf16(v)


# A score of at most 1.45 in log2 units off by 3 x 2^-24 of itself, exp2 by 2^-22: w by 4.2e-7 of itself, w / (1 + w) by
# half of that; three roundings (sum, reciprocal, product) by 1.8e-7 of at most 1/2. 3.0e-7 in all.
WEIGHT_TOL = 2.0 ** -21


def block_sums(n, dim, gen):
    """Equal weights; values of 1 .. 2 in steps of 2^-7 and of 2^-12 .. 2^-11 in steps of 2^-16 in turn: a block's sum
    has 23 bits and is exact however it is taken, the running sum over the blocks is not."""
    import torch
    q, k = torch.zeros(n, 2, dim), torch.randn(n, 1, dim, generator=gen)
    v = 1.0 + torch.randint(128, (n, 1, dim), generator=gen) / 128
    v[1::2] = (1.0 + torch.randint(16, (n // 2, 1, dim), generator=gen) / 16) * 2.0 ** -12
    return q, _bf16(k), _bf16(v)


def sum_tol(n, block):
    """Root mean square over the columns, relative to the sum: n / block additions rounded to nearest, each off by at
    most 2^-24 of the sum and evenly spread (a third of that squared); reciprocal and product by 2^-24 each."""
    return ((n / block / 3) ** 0.5 + 2) * 2.0 ** -24


SCALE = 0.125


def exact(q, k, v, first):
    """Causal outputs of tokens first .. n - 1 in 64 bits."""
    import torch
    n = q.shape[0]
    s = torch.einsum("rhd,kd->rhk", q[first:].double(), k[:, 0].double()) * SCALE
    late = torch.arange(n, device=q.device)[None] > torch.arange(first, n, device=q.device)[:, None]
    w = torch.softmax(s.masked_fill(late[:, None], float("-inf")), -1)
    return torch.einsum("rhk,kd->rhd", w, v[:, 0].double())


def off(got, want):
    return float((got.double() - want).abs().max())


def off_sums(got, want):
    """Largest over the rows of the relative error's root mean square over the columns."""
    return float(((got.double() / want - 1) ** 2).mean(-1).sqrt().max())


# ------------------------------------------------------------------ a form on the CPU that can drop bits
def _terms(x, terms):
    """x cut to `terms` bf16 terms of 8 bits, in 64 bits."""
    import torch
    out = torch.zeros_like(x, dtype=torch.float64)
    rest = x.float()
    for _ in range(terms):
        t = (rest.view(torch.int32) & -65536).view(torch.float32)
        out += t.double()
        rest = rest - t
    return out


def _cut(x):
    """x cut to 24 significand bits, toward zero."""
    import torch
    m, e = torch.frexp(x)
    return torch.ldexp(torch.trunc(m * 2.0 ** 24), e - 24)


def form(q, k, v, first, terms_q=3, terms_w=3, chain=False, block=64):
    """The kernel's arithmetic for tokens first .. n - 1: terms, fp32 scores and weights, sums cut at every 16 keys
    inside a block and rounded to nearest over blocks (with chain, cut there too)."""
    import torch
    n = q.shape[0]
    s = (torch.einsum("rhd,kd->rhk", _terms(q[first:], terms_q), k[:, 0].double()).float() * (SCALE * 1.4426950408889634))
    late = torch.arange(n)[None] > torch.arange(first, n)[:, None]
    s = s.masked_fill(late[:, None], float("-inf"))
    w = torch.exp2(s - s.amax(-1, keepdim=True))
    wt, o = _terms(w, terms_w), torch.zeros(n - first, 2, v.shape[2], dtype=torch.float64)
    for b in range(0, n, block):
        part = o if chain else torch.zeros_like(o)
        for j in range(b, min(n, b + block), 16):
            part = _cut(part + torch.einsum("rhk,kd->rhd", wt[..., j:j + 16], v[j:j + 16, 0].double()))
        o = part if chain else (o + part).float().double()
    return (o / w.double().sum(-1, keepdim=True)).float()


def _gen(device="cpu"):
    import torch
    return torch.Generator(device=device).manual_seed(11)


def test_checks_refuse_lost_bits():
    """The whole form passes every check; without the third term of queries or weights, or with cut sums, it does not."""
    q, k, v = score_bits(300, 64, _gen())
    want = exact(q, k, v, 0)
    assert off(form(q, k, v, 0), want) <= SCORE_TOL and off(form(q, k, v, 0, terms_q=2), want) > 8 * SCORE_TOL
    q, k, v = weight_bits(300, 64, _gen())
    want = exact(q, k, v, 0)
    assert off(form(q, k, v, 0), want) <= WEIGHT_TOL and off(form(q, k, v, 0, terms_w=2), want) > 4 * WEIGHT_TOL
    q, k, v = block_sums(4096, 64, _gen())
    want = exact(q, k, v, 4093)
    for block in (32, 64):
        tol = sum_tol(4096, block)
        assert off_sums(form(q, k, v, 4093, block=block), want) <= tol
        assert off_sums(form(q, k, v, 4093, block=block, chain=True), want) > 4 * tol


# ------------------------------------------------------------------ the kernels
def _outputs(dev, q, k, v, nodes, page=64):
    """The same tokens as a prompt, and the last `nodes` of them as a chain over a paged cache of the others."""
    import torch
    n, heads, dim = q.shape
    q, k, v = q.cuda(), k.cuda(), None if v is None else v.cuda()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    o = torch.empty_like(q)
    dev.prompt_attn(o, q, k, v, i32([0, n]), SCALE)
    ctx = n - nodes
    pages = -(-ctx // page)
    caches = []
    for x in (k, v):
        if x is None:
            caches.append(None)
            continue
        c = torch.zeros(pages, page, 1, dim, dtype=x.dtype, device="cuda")
        c.view(-1, 1, dim)[:ctx] = x[:ctx]
        caches.append(c)
    t = torch.empty_like(q[ctx:])
    dev.tree_attn(t, q[ctx:], k[ctx:], None if v is None else v[ctx:], *caches, i32([list(range(pages))]), i32([ctx]),
                  i32([0, nodes]), i32(list(range(-1, nodes - 1))), SCALE, nodes, ctx)
    return o, t


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128, 256, 512])
@pytest.mark.parametrize("inputs,tol", [(score_bits, SCORE_TOL), (weight_bits, WEIGHT_TOL)])
def test_last_bits_count(dev, dim, inputs, tol):
    n, nodes = 2100, 40
    q, k, v = inputs(n, dim, _gen())
    o, t = _outputs(dev, q, k, v, nodes)
    want = exact(q.cuda(), k.cuda(), v.cuda(), 0)
    assert off(o, want) <= tol
    assert off(t, want[n - nodes:]) <= tol


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128, 256, 512])
@pytest.mark.parametrize("shared", [False, True])
def test_sums_over_blocks_are_rounded_to_nearest(dev, dim, shared):
    n, nodes = 4096, 20
    q, k, v = block_sums(n, dim, _gen())
    o, t = _outputs(dev, q, v if shared else k, None if shared else v, nodes)
    first = n - 200
    want = exact(q.cuda(), k.cuda(), v.cuda(), first)
    tol = sum_tol(n, BLOCK)
    assert off_sums(o[first:], want) <= tol
    assert off_sums(t, want[200 - nodes:]) <= tol
