"""The paged serving operators together, as an engine runs them: page plan -> prompt attention -> paged write, then steps
of page plan -> tree attention -> output head -> verification -> paged write of the accepted rows, for several requests
of a one-layer model with random weights. Every committed token is checked against the plain model in 64 bits on the
committed prefix: a greedy token's logit is the largest to within what the attention's rounding allows, and the cache
holds exactly the committed tokens' rows."""
from __future__ import annotations

import random

import pytest

import servefix

pytestmark = pytest.mark.gpu

HEADS, KV, DIM, VOCAB, PAGE = 8, 2, 64, 211, 16


class Toy:
    """Embedding -> q, k, v -> attention -> logits; bf16 rows, fp32 head."""

    def __init__(self, seed):
        import torch
        gen = torch.Generator(device="cuda").manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
        self.q, self.k, self.v = (r(VOCAB, h, DIM).to(torch.bfloat16) for h in (HEADS, KV, KV))
        self.head = r(HEADS * DIM, VOCAB)

    def plain(self, tokens):
        """Logits behind every token of a sequence in 64 bits, and how far bf16 attention may be off them."""
        import torch
        t = torch.tensor(tokens, device="cuda")
        o, bound = servefix.attend(self.q[t], self.k[t], self.v[t], servefix.causal_seen(len(tokens), 0).cuda(),
                                   DIM ** -0.5)
        w = self.head.double()
        off = bound(torch.bfloat16, torch.bfloat16).flatten(1)
        flat = o.flatten(1)
        # the fp32 head adds its own rounding, 2^-24 per product and sum
        slack = off @ w.abs() + 2.0 ** -23 * HEADS * DIM * (flat.abs() @ w.abs())
        return flat @ w, slack


@pytest.mark.parametrize("how", ["greedy", "certain", "sampled"])
def test_serving_loop(dev, how):
    import torch
    rng = random.Random(7)
    toy = Toy(3)
    lens = [37, 1, 64, 90]
    n, cap, pages, width = len(lens), 256, 64, 12
    i32 = lambda *s: torch.full(s, -7, dtype=torch.int32, device="cuda")  # noqa: E731
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    kc, vc = (torch.full((pages, PAGE, KV, DIM), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    table, held, ring = i32(n, width), ints([0] * n), torch.randperm(pages, device="cuda").to(torch.int32)
    ring_pos = torch.tensor([0, pages], dtype=torch.int64, device="cuda")
    cu, slot = i32(n + 1), i32(cap)
    hist = [[rng.randrange(VOCAB) for _ in range(x)] for x in lens]
    # ---- the prompts, all but their last token (the first root)
    flat = ints([t for h in hist for t in h[:-1]])
    dev.page_plan(table, held, ring, ring_pos, ints([0] * n), ints([x - 1 for x in lens]), PAGE, cu, slot)
    m = flat.numel()
    o = torch.empty(m, HEADS, DIM, dtype=torch.bfloat16, device="cuda")
    q, k, v = toy.q[flat.long()], toy.k[flat.long()], toy.v[flat.long()]
    dev.prompt_attn(o, q, k, v, cu, DIM ** -0.5)
    dev.paged_write(kc, vc, k, v, slot[:m])
    at = 0
    for h in hist:
        if len(h) > 1:
            want, slack = toy.plain(h[:-1])
            got = o[at:at + len(h) - 1].flatten(1).double() @ toy.head.double()
            assert bool(((got - want).abs() <= slack).all())
        at += len(h) - 1
    # ---- decoding with drafted trees
    for step in range(12):
        nodes = [rng.randint(1, 9) for _ in range(n)]
        tokens, parent, base = [], [], [0]
        for b, x in enumerate(nodes):
            guess = [hist[b][-1]]
            par = [-1]
            for i in range(1, x):
                par.append(rng.choice([i - 1, i - 1, rng.randrange(i)]))
                line, j = [], par[i]
                while j > 0:
                    line.append(guess[j])
                    j = par[j]
                if rng.random() < 0.7:              # the plain model's pick behind this node's parent
                    seq = hist[b] + line[::-1]
                    guess.append(int(toy.plain(seq)[0][-1].argmax()))
                else:
                    guess.append(rng.randrange(VOCAB))
            tokens += guess
            parent += par
            base.append(base[-1] + x)
        t = base[-1]
        done = [len(h) - 1 for h in hist]
        tok = ints(tokens)
        dev.page_plan(table, held, ring, ring_pos, ints(done), ints(nodes), PAGE, cu, slot)
        assert cu.tolist() == base
        q, k, v = toy.q[tok.long()], toy.k[tok.long()], toy.v[tok.long()]
        o = torch.empty(t, HEADS, DIM, dtype=torch.bfloat16, device="cuda")
        dev.tree_attn(o, q, k, v, kc, vc, table, ints(done), cu, ints(parent), DIM ** -0.5, max(nodes), 200)
        logits = o.flatten(1).float() @ toy.head
        accepted, nxt, path, keep = i32(n), i32(n), i32(t), i32(t)
        if how == "greedy":
            best = i32(t)
            dev.argmax(best, logits, VOCAB, t)
            dev.verify_greedy(accepted, nxt, path, tok, ints(parent), cu, best, slot=slot[:t], slot_out=keep)
        else:
            p = torch.softmax(logits, 1)
            u = torch.rand(t, device="cuda")
            draft = torch.softmax(logits * 0.9, 1) if how == "sampled" else None
            dev.verify_sample(accepted, nxt, path, tok, ints(parent), cu, p, u, draft=draft, slot=slot[:t], slot_out=keep)
            want = servefix.verify(tokens, parent, base, probs=p.cpu(), u=u.cpu(),
                                   draft=None if draft is None else draft.cpu(), slot=slot[:t].tolist())
            assert [x.tolist() for x in (accepted, nxt, path, keep)] == list(want)
        dev.paged_write(kc, vc, k, v, keep)
        got, go, line = accepted.tolist(), nxt.tolist(), path.tolist()
        for b in range(n):
            took = [tokens[base[b] + x] for x in line[base[b] + 1:base[b] + 1 + got[b]]]
            if how == "greedy":
                seq = hist[b] + took
                want, slack = toy.plain(seq)
                for i, x in enumerate(took + [go[b]]):
                    row = len(hist[b]) - 1 + i
                    top = want[row].max()
                    assert float(want[row, x]) >= float(top - slack[row, x] - slack[row].max())
            hist[b] += took + [go[b]]
    assert dev.status_code() == 0
    # ---- the cache holds the committed tokens but the last, and nothing else was written
    used = torch.zeros(pages * PAGE, dtype=torch.bool, device="cuda")
    for b, h in enumerate(hist):
        j = torch.arange(len(h) - 1)
        at = (table[b].cpu().long()[j // PAGE] * PAGE + j % PAGE).cuda()
        t = torch.tensor(h[:-1], device="cuda")
        assert torch.equal(kc.view(-1, KV, DIM)[at], toy.k[t]) and torch.equal(vc.view(-1, KV, DIM)[at], toy.v[t])
        assert not bool(used[at].any())
        used[at] = True
    assert bool(torch.isnan(kc.view(-1, KV, DIM)[~used]).all())


@pytest.mark.parametrize("how", ["bfloat16", "float16"])
def test_fp32_projections_reach_the_prompt_and_the_cache(dev, how):
    """The way from fp32 projections: rounded into packed 16-bit rows by a write with the slots 0 .. n - 1, attended
    there, and written from there into the cache - the same rows as by rounding them elsewhere."""
    import torch
    ct = getattr(torch, how)
    gen = torch.Generator(device="cuda").manual_seed(4)
    n, pages = 77, 8
    fused = torch.randn(n, HEADS + 2 * KV, DIM, generator=gen, device="cuda")      # one product's output
    q, k, v = fused[:, :HEADS].to(ct), fused[:, HEADS:HEADS + KV], fused[:, HEADS + KV:]
    k16, v16 = (torch.empty(n, KV, DIM, dtype=ct, device="cuda") for _ in range(2))
    iota = torch.arange(n, dtype=torch.int32, device="cuda")
    dev.paged_write(k16.view(1, n, KV, DIM), v16.view(1, n, KV, DIM), k, v, iota)
    assert torch.equal(k16, k.to(ct)) and torch.equal(v16, v.to(ct))
    cu = torch.tensor([0, 30, n], dtype=torch.int32, device="cuda")
    o = torch.empty(n, HEADS, DIM, dtype=ct, device="cuda")
    dev.prompt_attn(o, q, k16, v16, cu, DIM ** -0.5)
    for at in (slice(0, 30), slice(30, n)):
        want, bound = servefix.attend(q[at], k16[at], v16[at], servefix.causal_seen(at.stop - at.start, 0).cuda(),
                                      DIM ** -0.5)
        servefix.check_close(o[at], want, bound(ct, ct))
    kc, vc = (torch.zeros(pages, PAGE, KV, DIM, dtype=ct, device="cuda") for _ in range(2))
    slot = torch.randperm(pages * PAGE, generator=gen, device="cuda")[:n].to(torch.int32)
    dev.paged_write(kc, vc, k16, v16, slot)
    for c, x in ((kc, k16), (vc, v16)):
        assert torch.equal(c.view(-1, KV, DIM)[slot.long()], x)
