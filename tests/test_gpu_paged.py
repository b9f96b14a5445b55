"""Page plans and paged writes (dsv4cu_page_plan, dsv4cu_paged_write) against plain forms: exact."""
from __future__ import annotations

import random

import pytest

import canary
import servefix

pytestmark = pytest.mark.gpu


def _i(x, dtype=None):
    import torch
    return torch.tensor(x, dtype=dtype or torch.int32, device="cuda")


def _make(rng, n, page, seq_hi, new_hi, spare=3, extra=0):
    """Lengths, held pages, table and ring of n requests in a consistent state."""
    seq = [rng.randint(0, seq_hi) for _ in range(n)]
    new = [-1 if rng.random() < 0.15 else rng.randint(0, new_hi) for _ in range(n)]
    held = [-(-x // page) + rng.choice([0, 0, 1]) for x in seq]
    grow = [0 if c < 0 else max(0, -(-(x + c) // page) - h) for x, c, h in zip(seq, new, held)]
    total = max(1, sum(held) + max(0, sum(grow) + extra))
    width = max(1, max(h + g for h, g in zip(held, grow)) + spare)
    ids = list(range(total))
    rng.shuffle(ids)
    table, k = [], 0
    for h in held:
        table.append(ids[k:k + h] + [-1] * (width - h))
        k += h
    free = ids[k:]
    head = rng.randrange(3 * total)
    ring = [-1] * total
    for i, x in enumerate(free):
        ring[(head + i) % total] = x
    return seq, new, held, table, ring, [head, head + len(free)], total, width


def _run(dev, case, page, cap, alias):
    import torch
    seq, new, held, table, ring, rp, total, width = case
    n = len(seq)
    t = {"table": _i(table), "held": _i(held), "ring": _i(ring), "rp": _i(rp, torch.int64), "seq": _i(seq),
         "new": _i(new), "cu": canary.guarded_empty(n + 1, torch.int32), "slot": canary.guarded_empty(cap, torch.int32),
         "pos": canary.guarded_empty(cap, torch.int32), "req": canary.guarded_empty(cap, torch.int32)}
    t["held_out"] = t["held"] if alias else canary.guarded_empty(n, torch.int32)
    t["rp_out"] = t["rp"] if alias else torch.empty(2, dtype=torch.int64, device="cuda")
    call = lambda: dev.page_plan(t["table"], t["held"], t["ring"], t["rp"], t["seq"], t["new"], page, t["cu"],  # noqa: E731
                                 t["slot"], t["pos"], t["req"], t["held_out"], t["rp_out"])
    return t, call


def _check(t, want):
    for name, w in zip(("table", "held_out", "ring", "rp_out", "cu", "slot", "pos", "req"), want):
        assert t[name].cpu().tolist() == w, name
        if hasattr(t[name], "_canary"):
            canary.check(t[name], name)


@pytest.mark.parametrize("n,page,seq_hi,new_hi", [(1, 16, 0, 1), (1, 1, 5, 9), (2, 16, 40, 40), (33, 7, 100, 30),
                                                  (300, 16, 400, 5), (1024, 64, 90, 3), (1500, 16, 60, 2),
                                                  (40, 16, 300, 1500), (2300, 5, 30, 9), (3, 64, 9000, 30000)])
@pytest.mark.parametrize("alias", [False, True])
def test_plan(dev, n, page, seq_hi, new_hi, alias):
    rng = random.Random(n * 31 + page)
    case = _make(rng, n, page, seq_hi, new_hi, extra=rng.choice([0, 7]))
    seq, new, held, table, ring, rp, total, width = case
    cap = max(1, sum(max(0, c) for c in new) + rng.choice([0, 9]))
    want = servefix.plan(seq, new, held, table, ring, rp, page, cap, total, width)
    t, call = _run(dev, case, page, cap, alias)
    call()
    _check(t, want[:8])
    assert dev.status_code() == 0 and not want[8]
    if not alias:                      # the same inputs again write the same again
        call()
        _check(t, want[:8])


@pytest.mark.parametrize("cap,extra,spare,new_hi,code", [(4000, -5, 3, 60, 71), (5000, -9999, 3, 900, 71),
                                                         (50, 5, 3, 60, 72), (4500, 5, -2, 800, 73)])
def test_plan_shortages(dev, cap, extra, spare, new_hi, code):
    """The ring, the token rows or the table run out: what fits is granted in order, the status says so."""
    rng = random.Random(cap)
    case = list(_make(rng, 24, 16, 100, new_hi, 3, extra))
    if spare < 0:                      # a narrower table: every row still holds its pages
        width = max(max(case[2]), case[7] - 8)
        case[3], case[7] = [r[:width] for r in case[3]], width
    seq, new, held, table, ring, rp, total, width = case
    want = servefix.plan(seq, new, held, table, ring, rp, 16, cap, total, width)
    assert code in want[8]
    t, call = _run(dev, case, 16, cap, False)
    call()
    assert dev.status_code() in want[8]
    _check(t, want[:8])
    assert dev.status_code() == 0


def test_plan_without_requests(dev):
    import torch
    e = torch.empty(0, dtype=torch.int32, device="cuda")
    rp, out = _i([4, 9], torch.int64), torch.zeros(2, dtype=torch.int64, device="cuda")
    cu, slot = _i([7]), _i([5, 5, 5])
    dev.page_plan(torch.empty((0, 3), dtype=torch.int32, device="cuda"), e, _i([0] * 8), rp, e, e, 16, cu, slot,
                  held_out=e, ring_pos_out=out)
    assert cu.tolist() == [0] and slot.tolist() == [-1] * 3 and out.tolist() == [4, 9]


def test_plan_odd_lengths_stay_inside(dev):
    """Negative lengths and holdings count as none, positions past 32 bits have no slot."""
    import torch
    big = 2 ** 31 - 2
    case = ([-5, big, 3], [2, 4, 1], [-3, 0, 99], [[-1] * 4] * 3, list(range(8)), [0, 8], 8, 4)
    t, call = _run(dev, case, 16, 8, False)
    call()
    torch.cuda.synchronize()
    assert dev.status_code() == 73
    assert t["cu"].tolist() == [0, 2, 6, 7]
    assert t["slot"].tolist()[:2] == [0, 1] and t["slot"].tolist()[2:] == [-1] * 6
    assert t["pos"].tolist()[:3] == [0, 1, big] and max(t["pos"].tolist()) <= 2 ** 31 - 1


def test_plan_lives_a_batch(dev):
    """Many steps in place, captured once and replayed: pages are never shared and never lost."""
    import torch
    rng = random.Random(5)
    n, page, pages, width, cap = 6, 8, 40, 12, 64
    table = torch.full((n, width), -1, dtype=torch.int32, device="cuda")
    held, seq, new = (torch.zeros(n, dtype=torch.int32, device="cuda") for _ in range(3))
    ring = torch.arange(pages, dtype=torch.int32, device="cuda")
    rp = _i([0, pages], torch.int64)
    cu, slot = _i([0] * (n + 1)), _i([0] * cap)
    args = (table, held, ring, rp, seq, new, page, cu, slot)
    dev.page_plan(*args)
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        dev.page_plan(*args)
    host = [0] * n
    for _ in range(60):
        step = []
        for b in range(n):
            if host[b] and rng.random() < 0.2:
                step.append(-1)
            else:
                step.append(rng.randint(0, min(9, 48 - host[b])))
        new.copy_(_i(step))
        g.replay()
        torch.cuda.synchronize()
        h, r = held.tolist(), rp.tolist()
        out = [x for b in range(n) for x in table[b, :h[b]].tolist()]
        free = [ring.tolist()[i % pages] for i in range(*r)]
        assert sorted(out + free) == list(range(pages))
        slots = [x for x in slot.tolist() if x >= 0]
        assert len(set(slots)) == len(slots) == sum(max(0, c) for c in step)
        host = [0 if c < 0 else a + c for a, c in zip(host, step)]
        assert h == [-(-x // page) for x in host]
        seq.copy_(_i(host))
    assert dev.status_code() == 0


# ------------------------------------------------------------------ writes
@pytest.mark.parametrize("nt,kv,dim,values", [(1, 1, 8, False), (1, 8, 128, True), (7, 3, 64, True), (130, 2, 24, True),
                                              (513, 1, 512, False), (4099, 4, 128, True)])
@pytest.mark.parametrize("src,cache", [("bfloat16", "bfloat16"), ("float16", "float16"), ("float32", "bfloat16"),
                                       ("float32", "float16")])
def test_write(dev, nt, kv, dim, values, src, cache):
    import torch
    st, ct = getattr(torch, src), getattr(torch, cache)
    gen = torch.Generator(device="cuda").manual_seed(nt + dim)
    page = 16
    pages = -(-nt // page) + 2
    fused = torch.randn(nt, 2 * kv + 2, dim, generator=gen, device="cuda").to(st)       # rows inside a wider buffer
    k, v = fused[:, :kv], fused[:, kv + 1:2 * kv + 1] if values else None
    caches = [servefix.guarded((pages, page, kv, dim), ct) for _ in range(2 if values else 1)]
    for c in caches:
        c.copy_(torch.randn(c.shape, generator=gen, device="cuda"))
    slot = torch.randperm(pages * page, generator=gen, device="cuda")[:nt].to(torch.int32)
    slot[torch.rand(nt, generator=gen, device="cuda") < 0.2] = -1
    if nt > 4:
        slot[1], slot[2] = pages * page, 2 ** 31 - 1
    want = [c.clone().view(-1, kv, dim) for c in caches]
    keep = torch.nonzero((slot >= 0) & (slot < pages * page))[:, 0]
    for w, rows in zip(want, (k, v)):
        w[slot[keep].long()] = rows[keep].to(ct)
    dev.paged_write(caches[0], caches[1] if values else None, k, v, slot)
    for c, w in zip(caches, want):
        assert torch.equal(c.view(torch.int16), w.view(c.shape).view(torch.int16))
        servefix.check_guards(c, "cache")


def test_write_rounds_to_nearest_and_keeps_nan(dev):
    import torch
    x = torch.tensor([1.0 + 2.0 ** -8, 1.0 + 3 * 2.0 ** -8, float("nan"), float("inf"), -0.0, 65520.0, 1e-41, 3.3e38],
                     device="cuda").view(1, 1, 8)
    for ct in (torch.bfloat16, torch.float16):
        cache = torch.zeros(1, 1, 1, 8, dtype=ct, device="cuda")
        dev.paged_write(cache, None, x, None, torch.zeros(1, dtype=torch.int32, device="cuda"))
        want = x.to(ct).view(-1)
        assert torch.equal(torch.nan_to_num(cache.view(-1), nan=7.0), torch.nan_to_num(want, nan=7.0))


def test_write_offsets_past_32_bits(dev):
    """A cache of more than 2^31 elements: the last slots land at its end."""
    import torch
    pages, page, kv, dim = 33000, 16, 8, 512                                 # 2.16e9 elements
    cache = torch.zeros(pages, page, kv, dim, dtype=torch.bfloat16, device="cuda")
    rows = torch.randn(3, kv, dim, device="cuda").to(torch.bfloat16)
    n = pages * page
    dev.paged_write(cache, None, rows, None, torch.tensor([n - 1, 0, n // 2 + 1], dtype=torch.int32, device="cuda"))
    flat = cache.view(n, kv, dim)
    assert torch.equal(flat[n - 1], rows[0]) and torch.equal(flat[0], rows[1]) and torch.equal(flat[n // 2 + 1], rows[2])
    assert int((flat[[1, n // 2, n - 2]] != 0).sum()) == 0


def test_binding_refuses_wrong_tensors(dev):
    import torch
    import dsv4cu
    cache = torch.zeros(2, 4, 1, 8, dtype=torch.bfloat16, device="cuda")
    rows = torch.zeros(2, 1, 8, dtype=torch.bfloat16, device="cuda")
    slot = torch.zeros(2, dtype=torch.int32, device="cuda")
    for bad in (lambda: dev.paged_write(cache, None, rows, None, slot.long()),
                lambda: dev.paged_write(cache, None, rows, None, slot.cpu()),
                lambda: dev.paged_write(cache, None, rows, None, slot[:1]),
                lambda: dev.paged_write(cache, None, rows.cpu(), None, slot),
                lambda: dev.paged_write(cache, None, rows.transpose(1, 2), None, slot),
                lambda: dev.paged_write(cache, cache[:1], rows, rows, slot),
                lambda: dev.paged_write(cache, cache, rows, rows.float(), slot)):
        with pytest.raises(dsv4cu.DSV4CUError):
            bad()


def _leave_out_everything(dev):
    """One call of each kind that leaves work out."""
    import torch
    zero = torch.zeros(132, dtype=torch.int32, device="cuda")
    cu = _i([0, 129, 132])
    out = [torch.empty(m, dtype=torch.int32, device="cuda") for m in (2, 2, 132)]
    rp = _i([0, 1], torch.int64)
    # one free page for a request of 3 pages over a table of 2; 40 tokens for 8 rows
    dev.page_plan(_i([[-1, -1]]), _i([0]), _i([0, 0]), rp, _i([0]), _i([40]), 16, _i([0, 0]), _i([0] * 8))
    dev.verify_greedy(*out, zero, zero, cu, zero)
    rows = torch.zeros(132, 1, 64, dtype=torch.bfloat16, device="cuda")
    cache = torch.zeros(1, 16, 1, 64, dtype=torch.bfloat16, device="cuda")
    dev.tree_attn(torch.empty_like(rows), rows, rows, rows, cache, cache, _i([[0], [0]]), _i([4, 4]), cu, zero, 0.1, 8, 4)


def test_work_left_out_is_told_apart(dev):
    """Every kind is remembered, none as a timeout; the status call gives the lowest and clears all."""
    import dsv4cu
    assert dev.refused() == set()
    _leave_out_everything(dev)
    assert dev.refused() == {71, 72, 73, 75, 76}
    assert dev.refused() == set() and dev.status_code() == 0
    _leave_out_everything(dev)
    with pytest.raises(dsv4cu.DSV4CUError, match=r"status -8: .*free pages.*\(71\).*\(75\)"):
        dev.check_status()
    assert dev.status_code() == 0


@pytest.mark.parametrize("first", [False, True])
def test_work_left_out_and_a_timeout_do_not_hide_each_other(dev, first):
    """A wait that runs out (a stage withheld in a streamed GEMV) before or after work is left out: both are told."""
    import numpy as np
    import torch
    rows = cols = 7168                         # as many stages per CTA as the withheld one takes
    w = torch.zeros(rows, cols, dtype=torch.uint8, device="cuda")
    s = torch.full((rows // 128, cols // 128), 127, dtype=torch.uint8, device="cuda")
    m = dev.qmat(w, s, 2, rows, cols, 128, 128)
    x = torch.from_numpy(np.ones((1, cols), np.float32)).cuda()
    y = torch.empty((1, rows), dtype=torch.float32, device="cuda")
    if first:
        _leave_out_everything(dev)
    dev.inject(dev.INJECT_WITHHOLD_STAGE)
    dev.gemv(y, x, m, 1)
    if not first:
        _leave_out_everything(dev)
    assert 0 < dev.status_code() < 71          # the timeout, whichever came first
    assert dev.refused() == {71, 72, 73, 75, 76}
    dev.gemv(y, x, m, 1)
    assert dev.status_code() == 0 and not bool(y.any())
