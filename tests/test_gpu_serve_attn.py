"""Prompt attention and tree attention (dsv4cu_prompt_attn, dsv4cu_tree_attn) against the plain form in 64 bits, within
bounds derived from the formats (servefix.attend)."""
from __future__ import annotations

import random

import pytest

import servefix

pytestmark = pytest.mark.gpu

KINDS = [("bfloat16", "bfloat16"), ("float16", "float16"), ("float32", "bfloat16")]


def _i(x):
    import torch
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _rows(gen, n, heads, dim, dtype, std=1.0, wide=0):
    """Token rows, `wide` elements apart beyond their own length (rows inside a wider buffer)."""
    import torch
    x = (torch.randn(n, heads * dim + wide, generator=gen, device="cuda") * std).to(dtype)
    return x[:, :heads * dim].unflatten(1, (heads, dim))


def _out(n, heads, dim, dtype):
    import torch
    o = servefix.guarded((n, heads, dim), dtype)
    o.fill_(7.0)
    return o


def _prompt(dev, lens, heads, kv, dim, kind, window=0, sink=False, shared=False, wide=0, seed=0, tail=3, edit=None):
    """Runs packed prompts and checks every row; `tail` rows behind the last sequence must stay as they were."""
    import torch
    qt, ct = (getattr(torch, x) for x in kind)
    gen = torch.Generator(device="cuda").manual_seed(seed + sum(lens) + dim)
    n = sum(lens) + tail
    q = _rows(gen, n, heads, dim, qt, 1.5, wide)
    k = _rows(gen, n, kv, dim, ct, 1.25, 2 * wide)
    v = None if shared else _rows(gen, n, kv, dim, ct, 1.0, wide)
    s = torch.randn(heads, generator=gen, device="cuda") if sink else None
    if edit:
        edit(q, k, v)
    cu = [0]
    for x in lens:
        cu.append(cu[-1] + x)
    o = _out(n, heads, dim, qt)
    scale = dim ** -0.5
    dev.prompt_attn(o, q, k, v, _i(cu), scale, window=window, sink=s)
    servefix.check_guards(o, "o")
    for b, x in enumerate(lens):
        if x:
            at = slice(cu[b], cu[b + 1])
            want, bound = servefix.attend(q[at], k[at], (k if shared else v)[at], servefix.causal_seen(x, window).cuda(),
                                          scale, s)
            servefix.check_close(o[at], want, bound(qt, ct), f"sequence {b}")
    assert bool((o[cu[-1]:] == 7.0).all()), "rows behind the last sequence were written"
    return o


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 64), (6, 2, 128), (3, 3, 128), (4, 1, 256), (16, 1, 512), (2, 2, 512)])
@pytest.mark.parametrize("lens", [[1], [2, 1], [17, 0, 64, 1, 65], [130, 3, 257]])
def test_prompts(dev, kind, heads, kv, dim, lens):
    _prompt(dev, lens, heads, kv, dim, kind)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128, 512])
@pytest.mark.parametrize("window", [1, 2, 63, 64, 65, 200, 100000])
def test_prompt_windows(dev, kind, dim, window):
    _prompt(dev, [129, 70, 1, 300], 4, 2, dim, kind, window=window, sink=window % 2 == 0)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,heads", [(64, 64), (128, 7), (256, 3), (512, 64)])
def test_prompt_shared_values_and_sinks(dev, kind, dim, heads):
    _prompt(dev, [40, 1, 133], heads, 1, dim, kind, sink=True, shared=True, window=128)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_prompt_strided_rows(dev, kind, dim):
    _prompt(dev, [33, 190], 6, 3, dim, kind, wide=3 * dim)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,heads,kv", [(64, 4, 4), (128, 8, 2), (512, 8, 1)])
def test_prompt_long(dev, kind, dim, heads, kv):
    _prompt(dev, [1021, 2, 515], heads, kv, dim, kind)


@pytest.mark.parametrize("kind", KINDS[:2])
@pytest.mark.parametrize("dim", [64, 128])
def test_prompt_many_sequences(dev, kind, dim):
    rng = random.Random(dim)
    _prompt(dev, [rng.choice([0, 1, 2, 5, 31, 64, 127, 128, 129, 140, 256, 300]) for _ in range(70)], 4, 1, dim, kind)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128, 512])
@pytest.mark.parametrize("seqs,window", [(32, 0), (33, 1025), (120, 0), (128, 1024), (129, 0), (300, 0), (300, 40)])
def test_prompt_order_of_tiles(dev, kind, dim, seqs, window):
    """Every way to deal tiles out: few and many sequences, all heads together and one after the other, windows that
    make tiles equal."""
    rng = random.Random(seqs)
    lens = [rng.choice([0, 1, 7, 20, 60, 110]) for _ in range(seqs)]
    lens[rng.randrange(seqs)] = 400
    _prompt(dev, lens, 16, 2, dim, kind, window=window, seed=seqs)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128, 512])
def test_prompt_nonfinite_values_stay_behind_the_mask(dev, kind, dim):
    """NaN and infinite values and keys of later tokens and of other sequences reach only the rows that see them."""
    import torch

    def edit(q, k, v):
        v[20, 0, 5], v[20, 1, 9] = float("nan"), float("inf")
        v[140, 1, 3] = float("-inf")
        k[60, 0, 0] = float("nan")
        v[190:, :, :] = float("nan")                       # the last sequence and the rows behind it

    # values 20, 140: rows 20 .. and 140 .. of the first sequence see them; key 60 makes rows 60 .. of head group 0 NaN
    o = _prompt(dev, [190, 5], 4, 2, dim, kind, edit=edit)
    assert bool(torch.isfinite(o[:20]).all()) and bool(torch.isnan(o[25, 0, 5])) and bool(torch.isinf(o[25, 2, 9]))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_prompt_visible_infinities(dev, kind, dim):
    """A key of -inf where every query is positive weighs nothing; an infinite value behind a small weight stays one."""
    import torch

    def edit(q, k, v):
        q[:, :, 0] = 1.5                                   # one term: the others of fp32 queries are 0
        k[3, :, 0] = float("-inf")
        k[100, 1, 0] = float("-inf")
        k[70, :, 1:] = 0.0
        k[70, :, 0] = -25.0 * dim ** 0.5                   # score -37.5, weight about 2^-54
        v[70, 0, 5], v[70, 1, 9] = float("inf"), float("-inf")

    o = _prompt(dev, [170, 90], 4, 2, dim, kind, edit=edit)
    assert bool(torch.isinf(o[80, 0, 5])) and bool(torch.isfinite(o[80, 0, 6])) and bool(torch.isfinite(o[30]).all())


@pytest.mark.parametrize("kind", KINDS)
def test_prompt_large_scores(dev, kind):
    """Scores in the hundreds: the running maximum moves often, weights underflow to 0."""
    def edit(q, k, v):
        q.mul_(6)
        k.mul_(4)
        k[7].mul_(2)
    _prompt(dev, [200, 90], 4, 2, 128, kind, edit=edit, sink=True)


@pytest.mark.parametrize("kind", KINDS[:2])
@pytest.mark.parametrize("dim", [64, 128])
def test_prompt_rising_scores(dev, kind, dim):
    """Every later key scores higher by a step: the maximum rises through the whole pass, in small and large steps."""
    import torch

    def edit(q, k, v):
        q.zero_()
        k.zero_()
        q[:, :, 0] = 4.0
        k[:, :, 0] = torch.linspace(-60, 60, k.shape[0], device="cuda")[:, None].to(k.dtype)
    _prompt(dev, [700], 4, 2, dim, kind, edit=edit)

    def steps(q, k, v):
        edit(q, k, v)
        k[:, :, 0] = (torch.arange(k.shape[0], device="cuda") // 100 * 16.0)[:, None].to(k.dtype)
    _prompt(dev, [700], 4, 2, dim, kind, edit=steps)


def test_prompt_hostile_offsets(dev):
    """Offsets outside the rows are clamped: nothing outside the buffers is touched."""
    import torch
    gen = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (_rows(gen, 50, h, 64, torch.bfloat16) for h in (4, 2, 2))
    for cu in ([-7, 20, 90], [0, 60, 10], [50, 50, 50], [2 ** 31 - 1, 5, 2 ** 31 - 1]):
        o = _out(50, 4, 64, torch.bfloat16)
        dev.prompt_attn(o, q, k, v, _i(cu), 0.125)
        servefix.check_guards(o, "o")


# ------------------------------------------------------------------ trees
def _parents(rng, n, chain=False):
    return ([rng.choice([-1, 0, n])] + [i - 1 if chain else rng.randrange(i) for i in range(1, n)])[:n]


def _tree(dev, ctx, nodes, heads, kv, dim, kind, page=16, window=0, sink=False, shared=False, wide=0, seed=0, lost=(),
          edit=None, max_ctx=None, spare=3, max_nodes=None, stream=None):
    """Runs one tree per request over a paged cache in random pages; `lost` (request, page) entries are not in the pool."""
    import torch
    rng = random.Random(seed)
    qt, ct = (getattr(torch, x) for x in kind)
    gen = torch.Generator(device="cuda").manual_seed(seed + sum(ctx) + dim)
    n = sum(nodes)
    q = _rows(gen, n, heads, dim, qt, 1.5, wide)
    k = _rows(gen, n, kv, dim, ct, 1.25, wide)
    v = None if shared else _rows(gen, n, kv, dim, ct, 1.0, 2 * wide)
    need = [-(-c // page) for c in ctx]
    total, width = sum(need) + spare, max(need + [1]) + 2
    ids = list(range(total))
    rng.shuffle(ids)
    table, at = [], 0
    for x in need:
        table.append(ids[at:at + x] + [-1] * (width - x))
        at += x
    kc = _rows(gen, total * page, kv, dim, ct, 1.25).reshape(total, page, kv, dim).contiguous()
    vc = None if shared else _rows(gen, total * page, kv, dim, ct).reshape(total, page, kv, dim).contiguous()
    par = [p for x in nodes for p in _parents(rng, x, rng.random() < 0.3)]
    cu = [0]
    for x in nodes:
        cu.append(cu[-1] + x)
    # whatever no request may read is not a number: page tails, spare pages
    used = torch.zeros(total * page, dtype=torch.bool, device="cuda")
    where = []
    for b, c in enumerate(ctx):
        j = torch.arange(c)
        where.append((torch.tensor(table[b])[j // page] * page + j % page).cuda())
        used[where[b]] = True
    for cache in (kc, vc):
        if cache is not None:
            cache.view(-1, kv, dim)[~used] = float("nan")
    for b, x in lost:
        table[b][x] = rng.choice([-1, total, 2 ** 31 - 1])
    s = torch.randn(heads, generator=gen, device="cuda") if sink else None
    if edit:
        edit(q, k, v, kc, vc, where)
    o = _out(n, heads, dim, qt)
    scale = dim ** -0.5
    args = (o, q, k, v, kc, vc, _i(table), _i(ctx), _i(cu), _i(par), scale, max_nodes or max(nodes),
            max(ctx) if max_ctx is None else max_ctx)
    dev.tree_attn(*args, window=window, sink=s)
    servefix.check_guards(o, "o")
    for b, x in enumerate(nodes):
        if not x:
            continue
        rows = slice(cu[b], cu[b + 1])
        seen = servefix.tree_seen(ctx[b], par[cu[b]:cu[b + 1]], window).cuda()
        for lb, lp in lost:
            if lb == b:
                seen[:, lp * page:min(ctx[b], (lp + 1) * page)] = False
        kk = torch.cat([kc.view(-1, kv, dim)[where[b]], k[rows]])
        vv = kk if shared else torch.cat([vc.view(-1, kv, dim)[where[b]], v[rows]])
        want, bound = servefix.attend(q[rows], kk, vv, seen, scale, s)
        servefix.check_close(o[rows], want, bound(qt, ct), f"request {b}")
    return args, s


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 64), (8, 1, 128), (5, 5, 128), (6, 2, 256), (16, 1, 512)])
@pytest.mark.parametrize("ctx,nodes", [([0], [1]), ([1], [1]), ([63, 64, 65, 0], [1, 2, 3, 4]), ([517], [1]),
                                       ([200, 31], [33, 128]), ([1500, 9], [5, 0])])
def test_trees(dev, kind, heads, kv, dim, ctx, nodes):
    _tree(dev, ctx, nodes, heads, kv, dim, kind)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128, 512])
@pytest.mark.parametrize("page", [1, 5, 16, 48, 64, 256])
def test_tree_pages(dev, kind, dim, page):
    _tree(dev, [300, 77, 129], [3, 1, 20], 4, 2, dim, kind, page=page)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128, 512])
@pytest.mark.parametrize("window", [1, 2, 7, 64, 150, 100000])
def test_tree_windows(dev, kind, dim, window):
    _tree(dev, [300, 5, 130], [12, 70, 1], 4, 2, dim, kind, window=window, sink=window % 2 == 0)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,heads", [(64, 3), (128, 16), (512, 64)])
def test_tree_shared_values_and_sinks(dev, kind, dim, heads):
    _tree(dev, [700, 64], [4, 9], heads, 1, dim, kind, sink=True, shared=True, page=64)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 128), (32, 8, 128), (4, 4, 64), (64, 1, 512)])
def test_tree_long_and_split(dev, kind, heads, kv, dim):
    _tree(dev, [5003, 64, 0, 2500], [1, 2, 3, 8], heads, kv, dim, kind, page=64, wide=dim)
    _tree(dev, [5003], [1], heads, kv, dim, kind, page=16, seed=1, sink=True)


@pytest.mark.parametrize("kind", KINDS)
def test_tree_estimate_of_the_context_does_not_matter(dev, kind):
    for max_ctx in (0, 10, 700, 100000, 2 ** 31 - 1):
        _tree(dev, [900, 1, 333], [2, 1, 7], 4, 2, 128, kind, max_ctx=max_ctx, max_nodes=30)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128, 512])
def test_tree_pages_outside_the_pool_are_masked(dev, kind, dim):
    _tree(dev, [300, 64, 16], [3, 1, 2], 4, 2, dim, kind, lost=[(0, 0), (0, 7), (0, 18), (2, 0)])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128, 512])
def test_tree_nonfinite_values_stay_behind_the_mask(dev, kind, dim):
    """A node's value that is not a number reaches its descendants alone; a cached one reaches every node in the window."""
    def edit(q, k, v, kc, vc, where):
        v[2] = float("nan")
        v[6, 0, 1] = float("inf")
        vc.view(-1, *vc.shape[2:])[where[1][3], 0, 2] = float("nan")
    _tree(dev, [1200, 90], [9, 4], 4, 2, dim, kind, window=60, edit=edit)
    _tree(dev, [1200, 90], [9, 4], 4, 2, dim, kind, edit=edit)


def test_tree_with_too_many_nodes_is_left_out(dev):
    import torch
    gen = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (_rows(gen, 12, h, 64, torch.bfloat16) for h in (4, 2, 2))
    o = _out(12, 4, 64, torch.bfloat16)
    cache = torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16, device="cuda")
    table = torch.zeros(2, 1, dtype=torch.int32, device="cuda")
    dev.tree_attn(o, q, k, v, cache, cache, table, _i([4, 4]), _i([0, 9, 12]), _i([-1] * 12), 0.125, 8, 4)
    assert dev.status_code() == 75
    assert bool((o[:9] == 7.0).all()) and not bool((o[9:] == 7.0).any())
    servefix.check_guards(o)


def test_tree_hostile_lists(dev):
    """Offsets, contexts, parents and page ids outside their ranges: nothing outside the buffers is touched."""
    import torch
    gen = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (_rows(gen, 12, h, 128, torch.bfloat16) for h in (4, 2, 2))
    cache = torch.randn(3, 16, 2, 128, device="cuda").to(torch.bfloat16)
    for table, ctx, cu, parent in (([[0, 99], [-5, 2]], [3000, -4], [0, 5, 12], [7, -9, 99, 2 ** 31 - 1] * 3),
                                   ([[1, 1], [1, 1]], [32, 32], [-3, 5, 99], [0] * 12),
                                   ([[2, 0], [0, 1]], [2 ** 31 - 1, 17], [0, 6, 2], [3] * 12)):
        o = _out(12, 4, 128, torch.bfloat16)
        dev.tree_attn(o, q, k, v, cache, cache, _i(table), _i(ctx), _i(cu), _i(parent), 0.1, 12, 32, window=64)
        servefix.check_guards(o)
        dev.status_code()


def test_tree_on_another_stream_captured_and_replayed(dev):
    """A captured call replays with new lengths, nodes and queries; a split pass and its join in one graph."""
    import torch
    kind = KINDS[0]
    (o, q, k, v, kc, vc, table, ctx, cu, par, scale, mn, mc), _ = _tree(dev, [3000, 1700], [6, 4], 8, 2, 128, kind)
    dev.L.dsv4cu_ctx_reserve(dev.ctx, 1 << 26)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        dev.tree_attn(o, q, k, v, kc, vc, table, ctx, cu, par, scale, mn, mc)
    for new_ctx, new_cu in (([3000, 1700], [0, 6, 10]), ([100, 1601], [0, 1, 7]), ([0, 2999 - 1300], [0, 0, 5])):
        ctx.copy_(_i(new_ctx))
        cu.copy_(_i(new_cu))
        par.copy_(_i([-1 if i in new_cu else (i - max(c for c in new_cu if c <= i)) // 2 for i in range(10)]))
        q.copy_(torch.randn(q.shape, device="cuda"))
        o.fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        p = par.tolist()
        for b in range(2):
            rows = slice(new_cu[b], new_cu[b + 1])
            if new_cu[b] == new_cu[b + 1]:
                continue
            j = torch.arange(new_ctx[b])
            where = (table[b].cpu().long()[j // 16] * 16 + j % 16).cuda()
            kk, vv = (torch.cat([c.view(-1, 2, 128)[where], x[rows]]) for c, x in ((kc, k), (vc, v)))
            want, bound = servefix.attend(q[rows], kk, vv, servefix.tree_seen(new_ctx[b], p[rows], 0).cuda(), scale)
            servefix.check_close(o[rows], want, bound(torch.bfloat16, torch.bfloat16), f"request {b}")
        assert bool((o[new_cu[-1]:] == 7.0).all())


@pytest.mark.parametrize("dim,kv", [(128, 8), (512, 2)])
def test_tree_cache_past_32_bits(dev, dim, kv):
    """Cached rows whose element offsets pass 2^31."""
    import torch
    page, pages = 64, (2 ** 31 // (64 * kv * dim)) + 40
    gen = torch.Generator(device="cuda").manual_seed(3)
    kc = torch.zeros(pages, page, kv, dim, dtype=torch.bfloat16, device="cuda")
    vc = torch.zeros_like(kc)
    last = list(range(pages - 4, pages))
    for c in (kc, vc):
        c[last] = torch.randn(4, page, kv, dim, generator=gen, device="cuda").to(torch.bfloat16)
    q, k, v = (_rows(gen, 2, h, dim, torch.bfloat16) for h in (2 * kv, kv, kv))
    o = _out(2, 2 * kv, dim, torch.bfloat16)
    dev.tree_attn(o, q, k, v, kc, vc, _i([last]), _i([250]), _i([0, 2]), _i([-1, 0]), dim ** -0.5, 2, 250)
    kk, vv = (torch.cat([c[last].view(-1, kv, dim)[:250], x]) for c, x in ((kc, k), (vc, v)))
    want, bound = servefix.attend(q, kk, vv, servefix.tree_seen(250, [-1, 0], 0).cuda(), dim ** -0.5)
    servefix.check_close(o, want, bound(torch.bfloat16, torch.bfloat16))


def test_one_node_is_the_prompts_last_token(dev):
    """The tree's single-token form over a cached prompt gives the prompt pass's last row, within both bounds."""
    import torch
    gen = torch.Generator(device="cuda").manual_seed(6)
    n, heads, kv, dim = 193, 8, 2, 128
    q, k, v = (_rows(gen, n, h, dim, torch.bfloat16) for h in (heads, kv, kv))
    o = _out(n, heads, dim, torch.bfloat16)
    dev.prompt_attn(o, q, k, v, _i([0, n]), dim ** -0.5)
    kc, vc = (torch.zeros(4, 64, kv, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    dev.paged_write(kc, vc, k[:-1], v[:-1], torch.arange(n - 1, dtype=torch.int32, device="cuda"))
    one = _out(1, heads, dim, torch.bfloat16)
    dev.tree_attn(one, q[-1:], k[-1:], v[-1:], kc, vc, _i([[0, 1, 2, 3]]), _i([n - 1]), _i([0, 1]), _i([-1]),
                  dim ** -0.5, 1, n)
    want, bound = servefix.attend(q[-1:], k, v, torch.ones(1, n, dtype=torch.bool, device="cuda"), dim ** -0.5)
    for got in (one, o[-1:]):
        servefix.check_close(got, want, bound(torch.bfloat16, torch.bfloat16))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,kv", [(64, 2), (128, 2), (512, 1)])
def test_same_call_same_bits(dev, kind, dim, kv):
    """Splits that finish in any order are joined in one: repeated calls, and calls after others, agree bit for bit."""
    import torch
    args, s = _tree(dev, [4000, 900, 0, 2111], [6, 1, 3, 17], 4 * kv, kv, dim, kind, page=64, sink=True)
    o, q = args[0], args[1]
    first = o.clone()
    for i in range(6):
        o.fill_(7.0)
        dev.tree_attn(*args, sink=s)
        if i % 2:
            _prompt(dev, [100], 4, 2, dim, kind)
        assert torch.equal(o, first)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128, 512])
def test_two_contexts_on_two_streams(dev, kind, dim):
    """Calls that run at the same time on streams of their own, each with its own context, as one after the other."""
    import torch
    import dsv4cu
    other = dsv4cu.Device(dev.device)
    try:
        cases = [_tree(dev, [3000, 500], [4, 2], 8, 2, dim, kind, page=64, seed=i) for i in range(2)]
        want = [c[0][0].clone() for c in cases]
        streams = [torch.cuda.Stream() for _ in range(2)]
        graphs = []
        for d, st, (args, s) in zip((dev, other), streams, cases):
            d.L.dsv4cu_ctx_reserve(d.ctx, 1 << 27)
            args[0].fill_(7.0)
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=st):
                for _ in range(20):
                    d.tree_attn(*args, sink=s)
            graphs.append(g)
        for _ in range(3):
            for g, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    g.replay()
        torch.cuda.synchronize()
        for w, (args, _) in zip(want, cases):
            assert torch.equal(args[0], w)
        assert other.status_code() == 0
    finally:
        other.close()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128, 512])
def test_prompt_captured_and_replayed(dev, kind, dim):
    """A captured prompt pass of a padded batch follows the offsets it finds: rows behind the last sequence stay."""
    import torch
    qt, ct = (getattr(torch, x) for x in kind)
    gen = torch.Generator(device="cuda").manual_seed(5)
    n = 700
    q, k, v = (_rows(gen, n, h, dim, t) for h, t in ((4, qt), (2, ct), (2, ct)))
    o, cu = _out(n, 4, dim, qt), _i([0, 0, 0, 0])
    dev.prompt_attn(o, q, k, v, cu, 0.1)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        dev.prompt_attn(o, q, k, v, cu, 0.1)
    for at in ([0, 700, 700, 700], [0, 1, 130, 600], [5, 5, 300, 301]):
        cu.copy_(_i(at))
        o.fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        for b in range(3):
            r = slice(at[b], at[b + 1])
            if at[b] == at[b + 1]:
                continue
            want, bound = servefix.attend(q[r], k[r], v[r], servefix.causal_seen(at[b + 1] - at[b], 0).cuda(), 0.1)
            servefix.check_close(o[r], want, bound(qt, ct), f"{at} sequence {b}")
        assert bool((o[at[-1]:] == 7.0).all()) and bool((o[:at[0]] == 7.0).all())


@pytest.mark.parametrize("dim", [64, 128])
def test_prompt_windows_of_wide_tiles(dev, dim):
    """One query head per key head: a tile's strips start blocks apart, each in its own part of the window."""
    for window in (1, 30, 64, 127, 128, 129, 300):
        _prompt(dev, [900, 40], 2, 2, dim, KINDS[0], window=window)


@pytest.mark.parametrize("dim", [64, 128, 256, 512])
@pytest.mark.parametrize("shared", [False, True])
def test_largest_fp32_queries(dev, dim, shared):
    """Finite fp32 queries above the largest bf16: their products with small keys are finite, and so are the outputs."""
    import torch
    big = torch.finfo(torch.float32).max
    kind = KINDS[2]

    def edit(q, k, v, *cache):
        q[:, :, 0], q[:, :, 1] = big, -big
        for x in (k,) + cache[:1]:
            x[..., :2] *= 2.0 ** -127                      # products of at most about 10

    _prompt(dev, [90, 5], 4, 1, dim, kind, shared=shared, edit=edit)
    _tree(dev, [200, 70], [3, 9], 4, 1, dim, kind, shared=shared, edit=edit)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,sink", [(64, False), (128, True), (256, True), (512, False)])
def test_tree_nonfinite_in_one_split_of_many(dev, kind, dim, sink):
    """A cache read in many splits: what is no number in one of them is not lost when they are joined - a query, the one
    key of a split that a row sees, a value whose split weighs next to nothing."""
    import torch

    def query(q, k, v, kc, vc, where):
        q[2, 1, 3] = float("nan")

    def key(q, k, v, kc, vc, where):
        k[1, 0, 0] = float("nan")

    def value(q, k, v, kc, vc, where):
        q[:, :, 0] = 8.0
        keys, values = (c.view(-1, *c.shape[2:]) for c in (kc, vc))
        keys[where[0][10], :, 0] = 25.0 * dim ** 0.5       # score 200: every other split's factor is below 2^-126
        values[where[0][4000], 0, 5], values[where[0][4000], 0, 9] = float("nan"), float("inf")

    for edit in (query, key, value):
        (o, *_), _ = _tree(dev, [5003, 0], [4, 2], 4, 2, dim, kind, page=64, edit=edit, sink=sink)
    assert bool(torch.isnan(o[:4, :2, 5]).all()) and bool(torch.isposinf(o[:4, :2, 9]).all())
    assert bool(torch.isfinite(o[:4, :, 10:]).all())
    _tree(dev, [5000], [1], 4, 2, dim, kind, page=64, window=1, edit=lambda q, k, *x: k.fill_(float("nan")), sink=sink)
    _tree(dev, [5003, 900], [3, 2], 4, 2, dim, kind, page=64, edit=lambda q, *x: q.fill_(float("nan")), sink=sink)
