"""The paged serving operators as they are measured: page plans, cache writes, prompt attention, attention
for trees of drafted tokens, and the verification of drafted tokens.

A case is a dict of plain values; ``prepare`` makes its inputs on the GPU from a seed, ``run`` is one pass
(the plain form in elementary torch operations, or with ``own`` the library's entry points) and ``exact``
the same outputs from the definitions in 64 bits.
"""
from __future__ import annotations

import math
import os
import random
import sys

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # One decode step of a small batch: every request appends a tree of up to 8 drafted tokens.
        {"name": "plan_decode", "op": "plan", "req": 24, "page": 64, "ctx": 8192, "new": 8},
        # A batch of prompts admitted at once while old requests finish: long slot maps, many new pages.
        {"name": "plan_prompts", "op": "plan", "req": 300, "page": 16, "ctx": 400, "new": 1500},
        # Keys and values of one small decode batch into a grouped-head bf16 cache.
        {"name": "write_decode", "op": "write", "rows": 48, "kv": 8, "dim": 128, "src": "bf16", "cache": "bf16",
         "shared": False, "page": 64},
        # A prompt's fp32 latent rows (this library's projections give fp32) into the engine's one-head cache.
        {"name": "write_latent", "op": "write", "rows": 65111, "kv": 1, "dim": 512, "src": "f32", "cache": "bf16",
         "shared": True, "page": 64},
        # The engine's own heads on two short prompts: 64 heads of 512 over one latent row per token, sliding
        # window 128, sinks, fp32 queries.
        {"name": "prompt_latent", "op": "prompt", "seqs": 2, "total": 301, "heads": 64, "kv": 1, "dim": 512,
         "q": "f32", "cache": "bf16", "shared": True, "window": 128, "sink": True},
        # A packed batch of ragged prompts at a small model's heads.
        {"name": "prompt_ragged", "op": "prompt", "seqs": 29, "total": 16001, "heads": 16, "kv": 4, "dim": 64,
         "q": "f16", "cache": "f16", "shared": False, "window": 0, "sink": False},
        # One long prompt at a large model's heads.
        {"name": "prompt_long", "op": "prompt", "seqs": 1, "total": 32768, "heads": 64, "kv": 8, "dim": 128,
         "q": "bf16", "cache": "bf16", "shared": False, "window": 0, "sink": False},
        # Plain decoding of one request: a tree of the root alone.
        {"name": "tree_single", "op": "tree", "req": 1, "nodes": 1, "ctx": 4001, "heads": 32, "kv": 8, "dim": 128,
         "q": "bf16", "cache": "bf16", "shared": False, "page": 16, "window": 0, "sink": False},
        # A serving batch with drafted trees over long, ragged caches.
        {"name": "tree_batch", "op": "tree", "req": 32, "nodes": 16, "ctx": 32000, "heads": 64, "kv": 8, "dim": 128,
         "q": "bf16", "cache": "bf16", "shared": False, "page": 64, "window": 0, "sink": False},
        # The engine's heads with drafted tokens over its latent cache, fp32 queries.
        {"name": "tree_latent", "op": "tree", "req": 6, "nodes": 5, "ctx": 9000, "heads": 64, "kv": 1, "dim": 512,
         "q": "f32", "cache": "bf16", "shared": True, "page": 64, "window": 0, "sink": True},
        # One request, a short chain of certain drafts (no draft probabilities).
        {"name": "verify_chain", "op": "verify", "req": 1, "nodes": 5, "vocab": 32000, "how": "certain",
         "chain": True},
        # A batch of sampled trees over the engine's vocabulary.
        {"name": "verify_trees", "op": "verify", "req": 64, "nodes": 8, "vocab": 129280, "how": "sampled",
         "chain": False},
    ]


def _spread(rng, lo, hi):
    """A whole number of lo .. hi, even over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng):
    """Head layouts: grouped heads of 64 or 128 in 16 bits, or latent heads with fp32 queries."""
    if rng.random() < 0.3:
        return {"heads": rng.choice([16, 48, 64]), "kv": 1, "dim": 512, "q": rng.choice(["f32", "bf16"]),
                "cache": "bf16", "shared": True, "sink": rng.random() < 0.7}
    t = rng.choice(["bf16", "bf16", "f16"])
    kv = rng.choice([1, 2, 4, 8])
    return {"heads": kv * rng.choice([1, 2, 3, 4, 7, 8]), "kv": kv, "dim": rng.choice([64, 128]), "q": t, "cache": t,
            "shared": False, "sink": rng.random() < 0.25}


def draw(rng):
    op = rng.choice(["plan", "write", "prompt", "prompt", "tree", "tree", "verify"])
    if op == "plan":
        return {"op": op, "req": _spread(rng, 1, 500), "page": rng.choice([16, 32, 64, 128]),
                "ctx": _spread(rng, 1, 9000), "new": _spread(rng, 1, 1500)}
    if op == "write":
        latent = rng.random() < 0.4
        cache = "bf16" if latent else rng.choice(["bf16", "f16"])
        return {"op": op, "rows": _spread(rng, 1, 65111 if latent else 30000), "kv": 1 if latent else rng.choice([1, 2, 4, 8]),
                "dim": 512 if latent else rng.choice([64, 128]), "src": rng.choice(["f32", cache]), "cache": cache,
                "shared": latent, "page": rng.choice([16, 32, 64])}
    if op == "prompt":
        h = _heads(rng)
        big = 4000 if h["q"] == "f32" else 16000
        total = _spread(rng, 1, big)
        return {"op": op, "seqs": _spread(rng, 1, min(64, total)), "total": total, **h,
                "window": rng.choice([0, 0, 128, rng.randint(1, 2000)])}
    if op == "tree":
        h = _heads(rng)
        return {"op": op, "req": _spread(rng, 1, 48), "nodes": _spread(rng, 1, 64), "ctx": _spread(rng, 1, 32000), **h,
                "page": rng.choice([16, 32, 64, 128]), "window": rng.choice([0, 0, 0, 128, 4096])}
    return {"op": op, "req": _spread(rng, 1, 64), "nodes": _spread(rng, 1, 16),
            "vocab": rng.choice([32000, 50257, 129280, rng.randint(1000, 140000)]),
            "how": rng.choice(["certain", "sampled", "greedy"]), "chain": rng.random() < 0.4}


# ------------------------------------------------------------------ inputs
def _ragged(rng, n, total):
    """n lengths that add up to `total`, spread over a factor of about 20."""
    w = [math.exp(rng.uniform(0, 3)) for _ in range(n)]
    s = sum(w)
    out = [max(1, int(total * x / s)) for x in w]
    out[out.index(max(out))] += total - sum(out)
    return out if min(out) >= 0 else [1] * (n - 1) + [total - n + 1]


def _shape(case, rng):
    """The case's lengths, the same for every seed so that outputs keep their shapes, in the seed's order."""
    fix = random.Random(str(sorted((k, str(x)) for k, x in case.items() if k != "name")))
    op, n = case["op"], case.get("req", 0)
    if op == "plan":
        seq = [fix.randint(0, case["ctx"]) for _ in range(n)]
        new = [-1 if n > 2 and fix.random() < 0.1 else fix.randint(0, case["new"]) for _ in range(n)]  # -1: finished
        held = [-(-(x + fix.choice([0, 0, case["page"]])) // case["page"]) for x in seq]
        rows = list(zip(seq, new, held))
    elif op == "prompt":
        rows = [(x,) for x in _ragged(fix, case["seqs"], case["total"])]
    else:
        nodes = [case["nodes"] if i == 0 else fix.randint((case["nodes"] + 1) // 2, case["nodes"]) for i in range(n)]
        top = case.get("ctx", 0)
        ctx = [top if i == n // 2 else int(top * fix.uniform(0.3, 1.0)) for i in range(n)]
        rows = list(zip(nodes, ctx))
    rng.shuffle(rows)
    return [list(x) for x in zip(*rows)]


def _parents(rng, n, chain):
    """Parents of n nodes: -1 for the root, and below it a chain or a tree that prefers early nodes."""
    return [-1] + [i - 1 if chain else max(0, min(i - 1, int((i - 1) * rng.random() ** 0.7))) for i in range(1, n)]


def _cu(lens):
    return [0] + np.cumsum(lens).tolist()


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _attn_rows(gen, n, heads, kv, dim, qt, ct, shared):
    """Queries, keys and values of n tokens; scores come out with a spread of about 2, as trained heads give."""
    q = (torch.randn(n, heads, dim, generator=gen, device="cuda") * 1.5).to(qt)
    k = (torch.randn(n, kv, dim, generator=gen, device="cuda") * 1.25).to(ct)
    v = None if shared else torch.randn(n, kv, dim, generator=gen, device="cuda").to(ct)
    return q, k, v


def prepare(case, seed):
    rng = random.Random(seed * 7919 + 1)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed * 7919 + 2)
    s = {"case": case}
    op = case["op"]
    if op == "plan":
        n, page = case["req"], case["page"]
        seq, new, held = _shape(case, rng)
        grow = [0 if c < 0 else max(0, -(-(x + c) // page) - h) for x, c, h in zip(seq, new, held)]
        width = max(h + g for h, g in zip(held, grow)) + 3
        total = sum(held) + sum(grow) + 7
        order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
        free = total - sum(held)
        table = torch.full((n, width), -1, dtype=torch.int32, device="cuda")
        at = _ints(_cu(held), torch.int64)[:-1, None] + torch.arange(width, device="cuda")[None]
        has = torch.arange(width, device="cuda")[None] < _ints(held)[:, None]
        table[has] = order[free + at[has]]
        head = rng.randrange(10 * total)
        ring = torch.full((total,), -1, dtype=torch.int32, device="cuda")
        ring[(head + torch.arange(free, device="cuda")) % total] = order[:free]
        tokens = sum(max(0, c) for c in new)
        cap = max(1, tokens + 5)                                 # a padded batch: no tokens behind the last request
        i32 = lambda *shape: torch.empty(shape, dtype=torch.int32, device="cuda")  # noqa: E731
        s.update(seq=_ints(seq), new=_ints(new), held=_ints(held), table=table, ring=ring, cap=cap,
                 ring_pos=_ints([head, head + free], torch.int64), held_out=i32(n), cu=i32(n + 1),
                 ring_out=torch.empty(2, dtype=torch.int64, device="cuda"), slot=i32(cap),
                 pos=i32(cap), of=i32(cap))
    elif op == "write":
        n, kv, dim, page = case["rows"], case["kv"], case["dim"], case["page"]
        st, ct = TYPES[case["src"]], TYPES[case["cache"]]
        pages = -(-n // page) * 5 // 4 + 2
        make = lambda *shape: torch.randn(shape, generator=gen, device="cuda")  # noqa: E731
        slot = torch.randperm(pages * page // 4, generator=gen, device="cuda")[: -(-n // 4)]
        slot = (slot[:, None] * 4 + torch.arange(4, device="cuda")).reshape(-1)[:n].to(torch.int32)
        if n > 8:                                                # rejected drafts and padding are skipped
            slot[torch.randperm(n, generator=gen, device="cuda")[: n // 9]] = -1
        s.update(k=make(n, kv, dim).to(st), v=None if case["shared"] else make(n, kv, dim).to(st), slot=slot,
                 k_cache=make(pages, page, kv, dim).to(ct),
                 v_cache=None if case["shared"] else make(pages, page, kv, dim).to(ct))
    elif op == "prompt":
        lens = _shape(case, rng)[0]
        q, k, v = _attn_rows(gen, case["total"], case["heads"], case["kv"], case["dim"], TYPES[case["q"]],
                             TYPES[case["cache"]], case["shared"])
        s.update(q=q, k=k, v=v, cu=_ints(_cu(lens)), lens=lens, scale=case["dim"] ** -0.5, o=torch.empty_like(q),
                 sink=torch.randn(case["heads"], generator=gen, device="cuda") if case["sink"] else None)
    elif op == "tree":
        n, page = case["req"], case["page"]
        nodes, ctx = _shape(case, rng)
        par = [p for x in nodes for p in _parents(rng, x, rng.random() < 0.3)]
        q, k, v = _attn_rows(gen, sum(nodes), case["heads"], case["kv"], case["dim"], TYPES[case["q"]],
                             TYPES[case["cache"]], case["shared"])
        np_ = [-(-c // page) for c in ctx]
        total, width = sum(np_) + 5, max(np_) + 2
        order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
        table = torch.full((n, width), -1, dtype=torch.int32, device="cuda")
        has = torch.arange(width, device="cuda")[None] < _ints(np_)[:, None]
        table[has] = order[(_ints(_cu(np_), torch.int64)[:-1, None] + torch.arange(width, device="cuda")[None])[has]]
        ct = TYPES[case["cache"]]
        shape = (total, page, case["kv"], case["dim"])
        kc = torch.empty(shape, dtype=ct, device="cuda").normal_(0, 1.25, generator=gen)
        vc = None if case["shared"] else torch.empty(shape, dtype=ct, device="cuda").normal_(generator=gen)
        s.update(q=q, k=k, v=v, k_cache=kc, v_cache=vc, table=table, ctx=_ints(ctx), cu=_ints(_cu(nodes)),
                 parent=_ints(par), host_ctx=ctx, host_nodes=nodes, max_nodes=max(nodes), max_ctx=max(ctx),
                 scale=case["dim"] ** -0.5, o=torch.empty_like(q),
                 sink=torch.randn(case["heads"], generator=gen, device="cuda") if case["sink"] else None)
    else:
        n, vocab = case["req"], case["vocab"]
        nodes = _shape(case, rng)[0]
        cu, t = _cu(nodes), sum(nodes)
        par = [p for x in nodes for p in _parents(rng, x, case["chain"])]
        base = [cu[b] + max(0, p) for b, x in enumerate(nodes) for p in par[cu[b]:cu[b] + x]]
        logits = torch.randn(t, vocab, generator=gen, device="cuda").mul_(2.5)
        draft = torch.randn(t, vocab, generator=gen, device="cuda").mul_(0.8).add_(logits)
        p, q = torch.softmax(logits, 1), torch.softmax(draft, 1)
        best = logits.argmax(1).to(torch.int32)
        up = _ints(base, torch.int64)                            # each node is drafted from its parent's row
        if case["how"] == "sampled":
            tok = torch.multinomial(q[up], 1, generator=gen)[:, 0]
        else:
            tok = draft.argmax(1)[up]
            tok = torch.where(torch.rand(t, generator=gen, device="cuda") < 0.5, tok, best.long()[up])
        del logits, draft
        i32 = lambda m: torch.empty(m, dtype=torch.int32, device="cuda")  # noqa: E731
        s.update(p=p, draft=q if case["how"] == "sampled" else None, best=best, tokens=tok.to(torch.int32),
                 parent=_ints(par), cu=_ints(cu), u=torch.rand(t, generator=gen, device="cuda"),
                 slot=torch.randperm(t, generator=gen, device="cuda").to(torch.int32), max_nodes=max(nodes),
                 accepted=i32(n), next=i32(n), path=i32(t), slot_out=i32(t))
    return s


# ------------------------------------------------------------------ one pass
_device = None


def _dev():
    """The library on the current device, made once as a program would."""
    global _device
    if _device is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                        "deepseek-v4-in-c_b200"))
        import dsv4cu
        _device = dsv4cu.Device(torch.cuda.current_device())
    return _device


def run(s):
    op = s["case"]["op"]
    if own:
        return _own(s, op, _dev())
    return {"plan": _plan, "write": _write, "prompt": _prompt, "tree": _tree, "verify": _verify}[op](s)


def _own(s, op, dev):
    if op == "plan":
        dev.page_plan(s["table"], s["held"], s["ring"], s["ring_pos"], s["seq"], s["new"], s["case"]["page"], s["cu"],
                      s["slot"], s["pos"], s["of"], s["held_out"], s["ring_out"])
        return {"table": s["table"], "held": s["held_out"], "ring": s["ring"], "ring_pos": s["ring_out"],
                "cu": s["cu"], "slot": s["slot"], "pos": s["pos"], "of": s["of"]}
    if op == "write":
        dev.paged_write(s["k_cache"], s["v_cache"], s["k"], s["v"], s["slot"])
        return [s["k_cache"], s["v_cache"]]
    if op == "prompt":
        dev.prompt_attn(s["o"], s["q"], s["k"], s["v"], s["cu"], s["scale"], window=s["case"]["window"], sink=s["sink"])
        return s["o"]
    if op == "tree":
        dev.tree_attn(s["o"], s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["ctx"], s["cu"],
                      s["parent"], s["scale"], s["max_nodes"], s["max_ctx"], window=s["case"]["window"], sink=s["sink"])
        return s["o"]
    if s["case"]["how"] == "greedy":
        dev.verify_greedy(s["accepted"], s["next"], s["path"], s["tokens"], s["parent"], s["cu"], s["best"],
                          slot=s["slot"], slot_out=s["slot_out"])
    else:
        dev.verify_sample(s["accepted"], s["next"], s["path"], s["tokens"], s["parent"], s["cu"], s["p"], s["u"],
                          draft=s["draft"], slot=s["slot"], slot_out=s["slot_out"])
    return {"accepted": s["accepted"], "next": s["next"], "path": s["path"], "slot": s["slot_out"]}


def _plan(s):
    page, table, ring, held = s["case"]["page"], s["table"], s["ring"], s["held"].long()
    head, tail = s["ring_pos"][0], s["ring_pos"][1]
    n, width = table.shape
    gone = s["new"] < 0
    new = s["new"].long().clamp(min=0)
    need = ((s["seq"] + new + page - 1) // page).clamp(max=width)
    grow = torch.where(gone, 0, (need - held).clamp(min=0))
    first = grow.cumsum(0) - grow
    grant = torch.minimum(grow, (tail - head - first).clamp(min=0))
    col = torch.arange(width, device=table.device)
    take = (col >= held[:, None]) & (col < (held + grant)[:, None])
    fresh = ring[(head + first[:, None] + col - held[:, None]) % ring.numel()]
    table_out = torch.where(take, fresh, table)
    back = torch.where(gone, held, 0)
    at = tail + (back.cumsum(0) - back)[:, None] + col
    put = col < back[:, None]
    ring_out = ring.clone()
    ring_out[at[put] % ring.numel()] = table[put]
    held_out = torch.where(gone, 0, held + grant)
    cu = torch.cat([new.new_zeros(1), new.cumsum(0)])
    t = torch.arange(s["cap"], device=table.device)
    of = torch.searchsorted(cu, t, right=True) - 1
    live = of < n
    b = of.clamp(max=n - 1)
    pos = s["seq"][b] + t - cu[b]
    pg = pos // page
    there = live & (pg < held_out[b])
    entry = table_out[b, pg.clamp(max=width - 1)]
    slot = torch.where(there & (entry >= 0), entry * page + pos % page, -1)
    i32 = torch.int32
    return {"table": table_out, "held": held_out.to(i32), "ring": ring_out,
            "ring_pos": torch.stack([head + grant.sum(), tail + back.sum()]), "cu": cu.to(i32), "slot": slot.to(i32),
            "pos": torch.where(live, pos, -1).to(i32), "of": torch.where(live, of, -1).to(i32)}


def _write(s):
    there = s["slot"] >= 0
    at = s["slot"][there].long()
    for cache, rows in ((s["k_cache"], s["k"]), (s["v_cache"], s["v"])):
        if cache is not None:
            cache.view(-1, *rows.shape[1:])[at] = rows[there].to(cache.dtype)
    return [s["k_cache"], s["v_cache"]]


def _attend(x, k, v, seen, scale, sink):
    """x [rows, kv, group, dim], k and v [kv, keys, dim], seen [rows, keys], sink [kv, group] or None -> as x."""
    rows, kv, group, dim = x.shape
    x = x.permute(1, 2, 0, 3).reshape(kv, group * rows, dim)
    score = (torch.matmul(x, k.transpose(1, 2)) * scale).view(kv, group, rows, -1)
    score = score.masked_fill(~seen, float("-inf"))
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - top)
    z = e.sum(-1, keepdim=True)
    if sink is not None:
        z = z + torch.exp(sink[:, :, None, None] - top)
    y = torch.matmul(e.view(kv, group * rows, -1), v).view(kv, group, rows, dim)
    return (y / z).permute(2, 0, 1, 3)


def _prompt(s):
    c, q, o = s["case"], s["q"], s["o"]
    kv, dim, group, window = c["kv"], c["dim"], c["heads"] // c["kv"], c["window"]
    sink = None if s["sink"] is None else s["sink"].view(kv, group)
    begin = 0
    for n in s["lens"]:
        k = s["k"][begin:begin + n].float().transpose(0, 1)                      # [kv, n, dim]
        v = k if s["v"] is None else s["v"][begin:begin + n].float().transpose(0, 1)
        step = max(128, min(n, (1 << 28) // (c["heads"] * n)))
        for r in range(0, n, step):                                             # query rows r .. e - 1
            e = min(n, r + step)
            lo = max(0, r - window + 1) if window else 0
            x = q[begin + r:begin + e].float().view(e - r, kv, group, dim)
            i = torch.arange(r, e, device=q.device)[:, None]
            j = torch.arange(lo, e, device=q.device)[None]
            seen = (j <= i) & (i - j < window) if window else j <= i
            y = _attend(x, k[:, lo:e], v[:, lo:e], seen, s["scale"], sink)
            o[begin + r:begin + e] = y.reshape(e - r, c["heads"], dim).to(o.dtype)
        begin += n
    return o


def _reach(parent):
    """reach[i][a]: node a is node i or one of its ancestors; by squaring, at most 128 nodes."""
    n = parent.numel()
    r = torch.eye(n, device=parent.device)
    i = torch.arange(1, n, device=parent.device)
    r[i, parent[1:].long()] = 1.0
    for _ in range(max(1, n - 1).bit_length()):
        r = (torch.matmul(r, r) > 0).float()
    return r > 0


def _tree(s):
    c, q, o, page = s["case"], s["q"], s["o"], s["case"]["page"]
    kv, dim, group, window = c["kv"], c["dim"], c["heads"] // c["kv"], c["window"]
    sink = None if s["sink"] is None else s["sink"].view(kv, group)
    begin = 0
    for b, (n, ctx) in enumerate(zip(s["host_nodes"], s["host_ctx"])):
        pages = s["table"][b, :-(-ctx // page)].long()
        old = s["k_cache"][pages].reshape(-1, kv, dim)[:ctx]
        k = torch.cat([old, s["k"][begin:begin + n]]).float().transpose(0, 1)
        if s["v"] is None:
            v = k
        else:
            old = s["v_cache"][pages].reshape(-1, kv, dim)[:ctx]
            v = torch.cat([old, s["v"][begin:begin + n]]).float().transpose(0, 1)
        reach = _reach(s["parent"][begin:begin + n])
        depth = reach.sum(1) - 1
        seen = torch.cat([torch.ones(n, ctx, dtype=torch.bool, device=q.device), reach], 1)
        if window:
            at = torch.cat([torch.arange(ctx, device=q.device), ctx + depth])
            seen &= (ctx + depth)[:, None] - at[None] < window
        x = q[begin:begin + n].float().view(n, kv, group, dim)
        y = _attend(x, k, v, seen, s["scale"], sink)
        o[begin:begin + n] = y.reshape(n, c["heads"], dim).to(o.dtype)
        begin += n
    return o


def _verify(s):
    greedy, tokens, parent = s["case"]["how"] == "greedy", s["tokens"].long(), s["parent"]
    cu = s["cu"].long()
    begin, count = cu[:-1], cu[1:] - cu[:-1]
    n, t = count.numel(), tokens.numel()
    cur = torch.zeros_like(begin)
    accepted = torch.zeros_like(begin)
    path = torch.full((t,), -1, dtype=torch.int64, device=tokens.device)
    slot = torch.full((t,), -1, dtype=torch.int64, device=tokens.device)
    path[begin] = 0
    slot[begin] = s["slot"][begin].long()
    rows = torch.arange(n, device=tokens.device)
    if not greedy:
        rest = s["p"][begin].double()                            # what is left of the target's row at cur
        mass = torch.ones(n, dtype=torch.float64, device=tokens.device)
    for i in range(1, s["max_nodes"]):                           # children come behind their parents
        at = (begin + i).clamp(max=t - 1)
        due = (i < count) & (parent[at] == cur)
        x = tokens[at]
        if greedy:
            ok = due & (s["best"][begin + cur] == x)
        else:
            left = rest[rows, x]
            bar = s["u"][at].double() * mass
            if s["draft"] is not None:
                drafted = s["draft"][begin + cur].double()
                bar = bar * drafted[rows, x]
            ok = due & (bar < left)
            no = due & ~ok
            if s["draft"] is not None:
                less = (rest - mass[:, None] * drafted).clamp(min=0)
                rest = torch.where(no[:, None], less, rest)
                mass = torch.where(no, rest.sum(1), mass)
            else:
                rest[rows, x] = torch.where(no, 0.0, left)
                mass = torch.where(no, (mass - left).clamp(min=0), mass)
        accepted = accepted + ok
        cur = torch.where(ok, i, cur)
        step = (begin + accepted).clamp(max=t - 1)
        path[step] = torch.where(ok, i, path[step])
        slot[at] = torch.where(ok, s["slot"][step].long(), slot[at])
        if not greedy:
            rest = torch.where(ok[:, None], s["p"][begin + cur].double(), rest)
            mass = torch.where(ok, 1.0, mass)
    if greedy:
        token = s["best"][begin + cur]
    else:
        rest = torch.where((rest.sum(1) > 0)[:, None], rest, s["p"][begin + cur].double())
        sums = rest.cumsum(1)
        token = (sums <= s["u"][begin].double()[:, None] * sums[:, -1:]).sum(1)
    i32 = torch.int32
    return {"accepted": accepted.to(i32), "next": token.to(i32), "path": path.to(i32), "slot": slot.to(i32)}


# ------------------------------------------------------------------ what a pass cannot do without
def _size(name):
    return 4 if name == "f32" else 2


def work(case):
    """Inputs read once, outputs written once; the products of the pairs that the masks leave."""
    op, n = case["op"], case.get("req", 0)
    lens = None if op == "write" else _shape(case, random.Random(0))
    if op == "plan":
        page, width = case["page"], 4
        tokens = sum(max(0, x) for x in lens[1])
        pages = sum(x // page + 1 for x in lens[1] if x >= 0) + sum(h for x, h in zip(lens[1], lens[2]) if x < 0)
        return {"bytes": width * (3 * tokens + 2 * pages + 5 * n), "flops": 4 * tokens}
    if op == "write":
        one = case["rows"] * case["kv"] * case["dim"] * (1 if case["shared"] else 2)
        return {"bytes": one * (_size(case["src"]) + 2) + 4 * case["rows"], "flops": one}
    if op == "verify":
        nodes = 24.0 * sum(lens[0])
        rows = n * {"greedy": 0, "certain": 1, "sampled": 2}[case["how"]]   # the row sampled from, and its draft
        return {"bytes": 4.0 * rows * case["vocab"] + nodes, "flops": 2.0 * rows * case["vocab"] + nodes}
    w, key = case["window"], case["dim"] * case["kv"] * (2 if case["shared"] else 4)
    if op == "prompt":
        rows = case["total"]
        pairs = sum(x * (x + 1) / 2 if not w or x <= w else w * (w + 1) / 2 + (x - w) * w for x in lens[0])
        old = 0
    else:
        rows = sum(lens[0])
        seen = [min(c, w) if w else c for c in lens[1]]
        pairs, old = sum(a * c for a, c in zip(lens[0], seen)), sum(seen)
    return {"bytes": (rows + old) * key + 2 * rows * case["dim"] * case["heads"] * _size(case["q"]),
            "flops": 4.0 * pairs * case["dim"] * case["heads"] + rows}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    """Attention and cache writes in 64 bits; plans and verifications are whole numbers and have no such value."""
    op = case["op"]
    if op in ("plan", "verify"):
        return None
    s = prepare(case, seed)
    if op == "write":
        out = []
        for cache, rows in ((s["k_cache"], s["k"]), (s["v_cache"], s["v"])):
            if cache is None:
                out.append(None)
                continue
            want = cache.double().view(-1, *rows.shape[1:])
            keep = torch.nonzero(s["slot"] >= 0)[:, 0]
            want.index_copy_(0, s["slot"].long()[keep], rows.double().index_select(0, keep))
            out.append(want.view(cache.shape))
        return out
    heads, kv, dim, w = case["heads"], case["kv"], case["dim"], case["window"]
    k, v = s["k"].double(), (s["k"] if s["v"] is None else s["v"]).double()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    begin = 0
    lens = s["lens"] if op == "prompt" else s["host_nodes"]
    for b, n in enumerate(lens):
        kb, vb = k[begin:begin + n], v[begin:begin + n]
        if op == "tree":
            ctx, page = s["host_ctx"][b], case["page"]
            at = torch.arange(ctx, device="cuda")
            row = s["table"][b].long()[at // page] * page + at % page
            kb = torch.cat([s["k_cache"].view(-1, kv, dim)[row].double(), kb])
            vc = s["k_cache"] if s["v"] is None else s["v_cache"]
            vb = torch.cat([vc.view(-1, kv, dim)[row].double(), vb])
            par = s["parent"][begin:begin + n].tolist()
            depth = [0] * n
            lines = [{i} for i in range(n)]
            for i in range(1, n):
                depth[i] = depth[par[i]] + 1
                lines[i] |= lines[par[i]]
            where = torch.cat([at, ctx + _ints(depth, torch.int64)])
            allow = torch.zeros(n, ctx + n, dtype=torch.bool)
            allow[:, :ctx] = True
            for i in range(n):
                allow[i, [ctx + a for a in lines[i]]] = True
            allow = allow.cuda()
            mine = where[ctx:]
        else:
            where = mine = torch.arange(n, device="cuda")
            allow = None
        total = kb.shape[0]
        step = max(1, (1 << 27) // total)
        for h in range(heads):
            g = h // (heads // kv)
            for r in range(0, n, step):
                e = min(n, r + step)
                z = s["q"][begin + r:begin + e, h].double() @ kb[:, g].t() * s["scale"]
                gap = mine[r:e, None] - where[None]
                ok = allow[r:e] if allow is not None else gap >= 0
                if w:
                    ok = ok & (gap < w)
                z = torch.where(ok, z, float("-inf"))
                norm = torch.logsumexp(z, 1)
                if s["sink"] is not None:
                    norm = torch.logaddexp(norm, s["sink"][h].double())
                out[begin + r:begin + e, h] = torch.exp(z - norm[:, None]) @ vb[:, g]
        begin += n
    return out
