"""Argument checks of the paged serving operators at the C entry points, and the binding's structures. CPU only:
every call is refused (or has nothing to do) before anything reaches a device."""
from __future__ import annotations

import ctypes as C
import os
import subprocess

import pytest

from conftest import ROOT

P = 0x10000           # an aligned address that no refused call follows
ARG, UNSUPPORTED = -1, -2


@pytest.fixture(scope="module")
def L():
    import dsv4cu
    return dsv4cu.lib()


@pytest.fixture(scope="module")
def ctx():
    return C.create_string_buffer(256)


def test_structures_have_the_headers_sizes(tmp_path):
    import dsv4cu
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include "dsv4cu.h"\nint main(void) { printf("%zu %zu %zu", '
                   "sizeof(dsv4cu_page_plan_args), sizeof(dsv4cu_prompt_attn_args), sizeof(dsv4cu_tree_attn_args)); "
                   "return 0; }\n")
    exe = str(tmp_path / "s")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", exe], check=True)
    sizes = [int(x) for x in subprocess.run([exe], capture_output=True, check=True).stdout.split()]
    assert sizes == [C.sizeof(x) for x in (dsv4cu.PagePlanArgs, dsv4cu.PromptAttnArgs, dsv4cu.TreeAttnArgs)]


def _plan(**kw):
    import dsv4cu
    base = dict(n_req=2, page_size=16, n_pages=8, max_pages=4, nt_cap=8, **{n: P for n in (
        "seq_len", "new_len", "held", "held_out", "table", "ring", "ring_pos", "ring_pos_out", "cu", "slot")})
    base.update(kw)
    return dsv4cu.PagePlanArgs(**base)


@pytest.mark.parametrize("kw", [dict(n_req=-1), dict(nt_cap=-1), dict(page_size=0), dict(n_pages=0), dict(max_pages=0),
                                dict(n_pages=1 << 20, page_size=1 << 12), dict(cu=None), dict(ring=None),
                                dict(ring_pos=None), dict(ring_pos_out=None), dict(seq_len=None), dict(new_len=None),
                                dict(held=None), dict(held_out=None), dict(table=None), dict(slot=None)])
def test_page_plan_refuses(L, ctx, kw):
    a = _plan(**kw)
    assert L.dsv4cu_page_plan(ctx, C.byref(a), None) == ARG
    assert b"page_plan" in L.dsv4cu_last_error()


def test_null_contexts_are_refused(L):
    a = _plan()
    assert L.dsv4cu_page_plan(None, C.byref(a), None) == ARG
    assert L.dsv4cu_paged_write(None, P, P, 1, P, P, 1, 64, 64, P, 1, 16, 1, 64, None) == ARG
    assert L.dsv4cu_prompt_attn(None, C.byref(_prompt()), None) == ARG
    assert L.dsv4cu_tree_attn(None, C.byref(_tree()), None) == ARG
    assert L.dsv4cu_verify_greedy(None, P, P, P, P, P, P, P, None, None, 1, 1, None) == ARG
    assert L.dsv4cu_verify_sample(None, P, P, P, P, P, P, P, 8, None, 0, P, 8, None, None, 1, 1, None) == ARG


WRITE = dict(kc=P, vc=P, ct=1, k=P, v=P, st=1, ldk=128, ldv=128, slot=P, nt=4, slots=64, kv=2, dim=64)


@pytest.mark.parametrize("kw,code", [(dict(nt=-1), ARG), (dict(slots=0), ARG), (dict(kv=0), ARG), (dict(dim=0), ARG),
                                     (dict(ct=0), UNSUPPORTED), (dict(ct=3), UNSUPPORTED), (dict(st=2), UNSUPPORTED),
                                     (dict(dim=60), UNSUPPORTED), (dict(v=None), ARG), (dict(vc=None), ARG),
                                     (dict(kc=None), ARG), (dict(slot=None), ARG), (dict(ldk=127), ARG),
                                     (dict(ldk=132), ARG), (dict(ldv=64), ARG), (dict(k=P + 8), ARG),
                                     (dict(vc=P + 2), ARG)])
def test_paged_write_refuses(L, ctx, kw, code):
    w = {**WRITE, **kw}
    assert L.dsv4cu_paged_write(ctx, w["kc"], w["vc"], w["ct"], w["k"], w["v"], w["st"], w["ldk"], w["ldv"], w["slot"],
                                w["nt"], w["slots"], w["kv"], w["dim"], None) == code
    assert b"paged_write" in L.dsv4cu_last_error()


def _prompt(**kw):
    import dsv4cu
    base = dict(o=2 * P, q=P, k=P, v=P, ldo=512, ldq=512, ldk=128, ldv=128, q_type=1, kv_type=1, cu=P, n_req=1, nt=4,
                n_heads=8, n_kv=2, head_dim=64, window=0, scale=0.125, sink=None)
    base.update(kw)
    return dsv4cu.PromptAttnArgs(**base)


def _tree(**kw):
    import dsv4cu
    base = dict(o=2 * P, q=P, k=P, v=P, k_cache=P, v_cache=P, ldo=512, ldq=512, ldk=128, ldv=128, q_type=1, kv_type=1,
                table=P, ctx_len=P, cu=P, parent=P, n_req=1, nt=4, n_heads=8, n_kv=2, head_dim=64, page_size=16,
                n_pages=8, max_pages=4, max_nodes=4, max_ctx=64, window=0, scale=0.125, sink=None)
    base.update(kw)
    return dsv4cu.TreeAttnArgs(**base)


BOTH = [(dict(n_req=-1), ARG), (dict(nt=-1), ARG), (dict(n_heads=0), ARG), (dict(n_kv=0), ARG), (dict(n_kv=3), ARG),
        (dict(window=-1), ARG), (dict(scale=0.0), ARG), (dict(scale=-1.0), ARG), (dict(scale=float("inf")), ARG),
        (dict(scale=float("nan")), ARG),
        (dict(scale=3.0e38), ARG), (dict(o=P), ARG), (dict(kv_type=0, q_type=0), UNSUPPORTED), (dict(kv_type=2), UNSUPPORTED),
        (dict(q_type=0, kv_type=2), UNSUPPORTED), (dict(q_type=5), UNSUPPORTED), (dict(head_dim=96), UNSUPPORTED),
        (dict(head_dim=0), UNSUPPORTED), (dict(o=None), ARG), (dict(q=None), ARG), (dict(k=None), ARG),
        (dict(cu=None), ARG), (dict(ldq=511), ARG), (dict(ldo=448), ARG), (dict(ldk=64), ARG), (dict(ldv=64), ARG),
        (dict(ldq=516), ARG), (dict(q=P + 8), ARG), (dict(v=P + 4), ARG), (dict(nt=1 << 30), ARG)]


@pytest.mark.parametrize("kw,code", BOTH)
def test_prompt_attn_refuses(L, ctx, kw, code):
    a = _prompt(**kw)
    assert L.dsv4cu_prompt_attn(ctx, C.byref(a), None) == code
    assert b"prompt_attn" in L.dsv4cu_last_error()


@pytest.mark.parametrize("kw,code", BOTH + [
    (dict(page_size=0), ARG), (dict(n_pages=-1), ARG), (dict(max_pages=-1), ARG), (dict(max_ctx=-1), ARG),
    (dict(max_nodes=0), ARG), (dict(max_nodes=129), ARG), (dict(v=None), ARG), (dict(v_cache=None), ARG),
    (dict(parent=None), ARG), (dict(ctx_len=None), ARG), (dict(table=None), ARG), (dict(k_cache=None), ARG),
    (dict(k_cache=P + 8), ARG), (dict(n_req=70000), ARG)])
def test_tree_attn_refuses(L, ctx, kw, code):
    a = _tree(**kw)
    assert L.dsv4cu_tree_attn(ctx, C.byref(a), None) == code
    assert b"tree_attn" in L.dsv4cu_last_error()


def test_empty_calls_do_nothing(L, ctx):
    assert L.dsv4cu_paged_write(ctx, None, None, 1, None, None, 1, 0, 0, None, 0, 16, 1, 64, None) == 0
    assert L.dsv4cu_prompt_attn(ctx, C.byref(_prompt(n_req=0)), None) == 0
    assert L.dsv4cu_prompt_attn(ctx, C.byref(_prompt(nt=0, q=None, o=None, k=None, v=None)), None) == 0
    assert L.dsv4cu_tree_attn(ctx, C.byref(_tree(n_req=0)), None) == 0
    assert L.dsv4cu_verify_greedy(ctx, None, None, None, None, None, None, None, None, None, 0, 0, None) == 0


@pytest.mark.parametrize("at", [1, 2, 3, 4, 5, 6, 7])
def test_verify_greedy_refuses_null(L, ctx, at):
    args = [ctx, P, P, P, P, P, P, P, None, None, 1, 1, None]
    args[at] = None
    assert L.dsv4cu_verify_greedy(*args) == ARG


def test_verify_refuses_slots_and_shapes(L, ctx):
    g = lambda slot, out, n=1, t=1: L.dsv4cu_verify_greedy(ctx, P, P, P, P, P, P, P, slot, out, n, t, None)  # noqa: E731
    assert g(P, None) == g(None, P) == g(P, P) == g(None, None, -1) == g(None, None, 1, -1) == ARG
    s = lambda p=P, ldp=8, d=None, ldd=0, u=P, vocab=8: L.dsv4cu_verify_sample(  # noqa: E731
        ctx, P, P, P, P, P, P, p, ldp, d, ldd, u, vocab, None, None, 1, 1, None)
    assert s(p=None) == s(ldp=7) == s(d=P, ldd=7) == s(u=None) == s(vocab=0) == ARG


def test_row_numbers_and_vocabularies_past_32_bits_are_refused(L, ctx):
    a = _tree(n_heads=1 << 24, n_kv=1, nt=1, max_nodes=128, ldq=1 << 30, ldo=1 << 30)
    assert L.dsv4cu_tree_attn(ctx, C.byref(a), None) == ARG and b"128 nodes" in L.dsv4cu_last_error()
    assert L.dsv4cu_tree_attn_workspace(ctx, C.byref(a)) == 0
    v = (1 << 30) + 1
    assert L.dsv4cu_verify_sample(ctx, P, P, P, P, P, P, P, v, None, 0, P, v, None, None, 1, 1, None) == ARG


class _TwoThreads:
    """Stands in for the library: every call reads its arguments, lets the other thread make its call, reads again."""

    def __init__(self):
        import threading
        self.meet = threading.Barrier(2, timeout=20)
        self.torn = []

    def _call(self, ctx, args, stream):
        size = len(bytes(args))
        first = C.string_at(args, size)
        self.meet.wait()                       # both have packed their arguments and are inside the library
        if C.string_at(args, size) != first:
            self.torn.append(first)
        self.meet.wait()
        return 0

    dsv4cu_page_plan = dsv4cu_prompt_attn = dsv4cu_tree_attn = _call


@pytest.mark.parametrize("op", ["plan", "prompt", "tree"])
def test_calls_of_two_threads_keep_their_arguments(op):
    """A call's arguments are its own: a second thread's call on the same Device does not change them under the first."""
    import threading

    import torch

    import dsv4cu
    dev = object.__new__(dsv4cu.Device)
    dev.torch, dev.L, dev.device, dev.ctx = torch, _TwoThreads(), -1, None       # tensors of the CPU count as device -1
    dev._elem = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
    dev._raw_stream = lambda device: 0

    def call(n):
        i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
        row = lambda h: torch.zeros(n, h, 64, dtype=torch.bfloat16)  # noqa: E731
        cache = torch.zeros(2, 8, 2, 64, dtype=torch.bfloat16)
        if op == "plan":
            dev.page_plan(i32(n, 3), i32(n), i32(8), torch.zeros(2, dtype=torch.int64), i32(n), i32(n), 8, i32(n + 1),
                          i32(5))
        elif op == "prompt":
            dev.prompt_attn(row(4), row(4), row(2), row(2), i32(2), 0.125)
        else:
            dev.tree_attn(row(4), row(4), row(2), row(2), cache, cache, i32(n, 3), i32(n), i32(n + 1), i32(n), 0.125, 4,
                          16)

    start = threading.Barrier(2, timeout=20)
    failed = []

    def run(n):
        try:
            start.wait()
            for _ in range(20):
                call(n)
        except Exception as e:  # noqa: BLE001
            failed.append(e)
    threads = [threading.Thread(target=run, args=(n,)) for n in (1, 2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed and not dev.L.torn
