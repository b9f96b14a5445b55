"""Plain 64-bit forms of the paged serving operators, and bounds for their kernels' outputs."""
from __future__ import annotations

import math

import torch

import canary

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def guarded(shape, dtype):
    """canary.guarded_empty for elements of any width: guard bytes around the buffer's bytes."""
    raw = canary.guarded_empty(math.prod(shape) * torch.empty((), dtype=dtype).element_size(), torch.uint8)
    t = raw.view(dtype).view(shape)
    t._guarded = raw
    return t


def check_guards(t, what="output"):
    canary.check(t._guarded, what)


def attend(q, k, v, seen, scale, sink=None):
    """q [rows][heads][dim], k / v [keys][kv][dim], seen [rows][keys] -> (o, bound_of(q_dtype, kv_dtype)), 64 bits.

    The bound of an output: half a step of its type, half a step of the value type on every weight (none for fp32
    queries, whose weights keep 24 bits), and fp32 arithmetic: a score's error, in units of 2^-23, is at most dim
    + 2 roundings of sum |q||k| scale, the same again as the relative error of its weight, twice (numerator and
    denominator), with one rounding per key summed and 4 for exp2. Masked rows (no key seen) are 0."""
    heads, kv = q.shape[1], k.shape[1]
    qd, kd, vd = q.double(), k.double(), v.double()
    group = heads // kv
    kx, vx = kd.repeat_interleave(group, 1), vd.repeat_interleave(group, 1)
    s = torch.einsum("rhd,khd->hrk", qd, kx) * scale
    size = torch.einsum("rhd,khd->hrk", qd.abs(), torch.nan_to_num(kx.abs(), posinf=0.0)) * scale
    s = s.masked_fill(~seen[None], float("-inf"))
    top = s.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), 0.0, top)
    e = torch.exp(s - top)
    z = e.sum(-1)
    if sink is not None:
        z = z + torch.exp(sink.double()[:, None] - top[..., 0])
    clean = torch.where(seen.any(0)[:, None, None], vx, 0.0)
    # a value is used only where its key is seen: 0 x inf of a masked value is not part of the sum
    if torch.isfinite(clean).all():
        num = torch.einsum("hrk,khd->hrd", e, clean)
    else:
        num = torch.where(seen[None, ..., None], e[..., None] * clean.transpose(0, 1)[:, None], 0.0).sum(2)
    mag = torch.einsum("hrk,khd->hrd", e, torch.nan_to_num(clean).abs())
    o = torch.where(z[..., None] == 0, 0.0, num / z[..., None]).transpose(0, 1)
    mag = torch.where(z[..., None] > 0, mag / z[..., None], 0.0).transpose(0, 1)
    worst = torch.where(seen[None], size, 0.0).amax(-1).transpose(0, 1)[..., None]          # [rows][heads][1]
    keys, dim = k.shape[0], q.shape[2]
    many = torch.einsum("hrk,khd->hrd", seen[None].expand(heads, -1, -1).double(), torch.nan_to_num(clean).abs())
    many = torch.where(z[..., None] > 0, many / z[..., None], 0.0).transpose(0, 1)

    def bound(out_dtype, weights_dtype):
        h = HALF_STEP[out_dtype]
        w = 0.0 if out_dtype is torch.float32 else HALF_STEP[weights_dtype]
        f = 2.0 ** -23 * ((dim + 2) * worst + keys + 4)
        tiny = 2.0 ** -25 if out_dtype is torch.float16 else 0.0   # half a step of an f16 subnormal: weights, output
        return h * o.abs() * 1.01 + (w + 2 * f) * mag + 1e-30 + tiny * (1 + many)

    return o, bound


def ancestors(parent):
    """(reach [n][n], depth [n]) of one tree; a parent that does not come before its child counts as none."""
    n = len(parent)
    reach = torch.zeros(n, n, dtype=torch.bool)
    depth = [0] * n
    for i in range(n):
        x, d = i, 0
        while True:
            reach[i, x] = True
            p = parent[x]
            if p < 0 or p >= x:
                break
            x, d = p, d + 1
        depth[i] = d
    return reach, torch.tensor(depth)


def causal_seen(n, window):
    i, j = torch.arange(n)[:, None], torch.arange(n)[None]
    return (j <= i) & (i - j < window) if window else j <= i


def tree_seen(ctx, parent, window):
    reach, depth = ancestors(parent)
    n = len(parent)
    where = torch.cat([torch.arange(ctx), ctx + depth])
    seen = torch.cat([torch.ones(n, ctx, dtype=torch.bool), reach], 1)
    if window:
        seen &= (ctx + depth)[:, None] - where[None] < window
    return seen


def check_close(got, want, bound, what=""):
    """NaN and infinities in the same places, everything else within its bound."""
    got = got.double()
    bad = ~torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    assert torch.equal(got[bad & ~torch.isnan(want)], want[bad & ~torch.isnan(want)]), f"{what}: infinities differ"
    off = torch.where(bad, 0.0, (got - want).abs())
    limit = torch.where(bad, 1.0, bound)
    assert bool((off <= limit).all()), f"{what}: off by {float((off / limit).max()):.3g} of the bound"


def plan(seq, new, held, table, ring, ring_pos, page, cap, n_pages, max_pages):
    """dsv4cu_page_plan on Python lists: (table, held, ring, ring_pos, cu, slot, pos, req, statuses)."""
    table, ring, held = [list(r) for r in table], list(ring), list(held)
    head, tail = ring_pos
    live, codes = tail - head, set()
    take = lambda: ring_take.pop(0)  # noqa: E731
    ring_take = [ring[(head + i) % n_pages] for i in range(live)]
    used = 0
    out_held = list(held)
    for b, n in enumerate(new):
        if n < 0:
            continue
        want = -(-(seq[b] + n) // page)
        if want > max_pages:
            codes.add(73)
        for j in range(held[b], min(want, max_pages)):
            if ring_take:
                table[b][j] = take()
                out_held[b] += 1
                used += 1
            else:
                codes.add(71)
    back = []
    for b, n in enumerate(new):
        if n < 0:
            back += table[b][:held[b]]
            out_held[b] = 0
    for i, x in enumerate(back):
        ring[(tail + i) % n_pages] = x
    cu, slot, pos, req = [0], [], [], []
    for b, n in enumerate(new):
        for i in range(max(0, n)):
            p = seq[b] + i
            pg = p // page
            e = table[b][pg] if pg < out_held[b] else -1
            slot.append(e * page + p % page if 0 <= e < n_pages else -1)
            pos.append(p)
            req.append(b)
        cu.append(cu[-1] + max(0, n))
    if cu[-1] > cap:
        codes.add(72)
    fit = lambda x: (x + [-1] * cap)[:cap]  # noqa: E731
    return table, out_held, ring, [head + used, tail + len(back)], cu, fit(slot), fit(pos), fit(req), codes


def verify(tokens, parent, cu, probs=None, u=None, draft=None, best=None, slot=None):
    """dsv4cu_verify_* on CPU tensors / lists: (accepted, next, path, slot_out)."""
    t = len(tokens)
    path, slot_out, accepted, nxt = [-1] * t, [-1] * t, [], []
    for b in range(len(cu) - 1):
        lo, n = cu[b], cu[b + 1] - cu[b]
        if n == 0:
            accepted.append(0)
            nxt.append(-1)
            continue
        cur, line, rest, mass = 0, [0], None, 1.0
        if probs is not None:
            rest = probs[lo].double()
        for i in range(1, n):
            if parent[lo + i] != cur:
                continue
            x = tokens[lo + i]
            if best is not None:
                ok = best[lo + cur] == x
            else:
                inside = 0 <= x < probs.shape[1]
                left = float(rest[x]) if inside else 0.0
                q = 1.0 if draft is None else float(draft[lo + cur][x]) if inside else 0.0
                ok = inside and float(u[lo + i]) * mass * q < left
                if not ok and draft is not None:
                    rest = (rest - mass * draft[lo + cur].double()).clamp(min=0)
                    mass = float(rest.sum())
                elif not ok and inside:
                    rest[x] = 0.0
                    mass = max(0.0, mass - left)
            if ok:
                cur = i
                line.append(i)
                if best is None:
                    rest, mass = probs[lo + i].double(), 1.0
        accepted.append(len(line) - 1)
        for d, i in enumerate(line):
            path[lo + d] = i
            if slot is not None:
                slot_out[lo + i] = slot[lo + d]
        if best is not None:
            nxt.append(best[lo + cur])
            continue
        if not float(rest.sum()) > 0:
            rest = probs[lo + cur].double()
        sums = rest.cumsum(0)
        if not float(sums[-1]) > 0:
            nxt.append(-1)
            continue
        hit = torch.nonzero(sums > float(u[lo]) * sums[-1])
        nxt.append(int(hit[0]))
    return accepted, nxt, path, slot_out
