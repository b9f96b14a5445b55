"""The context's host calls (csrc/ctx.cu) against a fake CUDA runtime: what dsv4cu_ctx_status and dsv4cu_ctx_refused say
of the device words."""
from __future__ import annotations

import os
import shutil
import subprocess

import pytest

from conftest import PKG

FAKE = r"""
#include <stdio.h>
#include <stdlib.h>
#include <string.h>
#include "%(csrc)s/ctx.h"
#include <cuda_runtime_api.h>

static int current = 0;                     // the calling thread's device
namespace dsv4cu { const float *router_table_get() { static float x; return &x; } }
extern "C" {
cudaError_t cudaGetDevice(int *d) { *d = current; return cudaSuccess; }
cudaError_t cudaSetDevice(int d) { current = d; return cudaSuccess; }
#undef cudaGetDeviceProperties
cudaError_t cudaGetDeviceProperties(cudaDeviceProp *p, int) { memset(p, 0, sizeof *p); p->multiProcessorCount = 4; return cudaSuccess; }
cudaError_t cudaGetDeviceProperties_v2(cudaDeviceProp *p, int d) { return cudaGetDeviceProperties(p, d); }
cudaError_t cudaMalloc(void **p, size_t n) { fprintf(stderr, "malloc %%d\n", current); *p = calloc(1, n); return cudaSuccess; }
cudaError_t cudaFree(void *p) { fprintf(stderr, "free %%d\n", current); free(p); return cudaSuccess; }
cudaError_t cudaMemset(void *p, int v, size_t n) { fprintf(stderr, "memset %%d\n", current); memset(p, v, n); return cudaSuccess; }
cudaError_t cudaMemcpy(void *d, const void *s, size_t n, enum cudaMemcpyKind) { fprintf(stderr, "memcpy %%d\n", current); memcpy(d, s, n); return cudaSuccess; }
cudaError_t cudaDeviceSynchronize() { fprintf(stderr, "device %%d\n", current); return cudaSuccess; }
cudaError_t cudaStreamSynchronize(cudaStream_t) { fprintf(stderr, "stream %%d\n", current); return cudaSuccess; }
const char *cudaGetErrorString(cudaError_t) { return "fake"; }
cudaError_t cudaGetLastError() { return cudaSuccess; }
cudaError_t cudaFuncSetAttribute(const void *, enum cudaFuncAttribute, int) { return cudaSuccess; }
cudaError_t cudaDeviceGetAttribute(int *v, enum cudaDeviceAttr, int) { *v = 4; return cudaSuccess; }
// what the compiler's own start-up code calls
void **__cudaRegisterFatBinary(void *) { static void *h; return &h; }
void __cudaRegisterFatBinaryEnd(void **) {}
void __cudaUnregisterFatBinary(void **) {}
char __cudaInitModule(void **) { return 0; }
}

%(main)s
"""


def _run(tmp_path, main):
    """Builds ctx.cu over the fake runtime with `main` and returns its stdout words and stderr lines."""
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("no nvcc")
    csrc = os.path.join(PKG, "csrc")
    src, exe = tmp_path / "fake.cpp", str(tmp_path / "ctx")
    src.write_text(FAKE % {"csrc": csrc, "main": main})
    subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "--expt-relaxed-constexpr",
                    "-cudart", "none", os.path.join(csrc, "ctx.cu"), str(src), "-o", exe], check=True)
    p = subprocess.run([exe], capture_output=True, check=True, timeout=60, text=True)
    return p.stdout.splitlines(), p.stderr.splitlines()


def test_status_and_work_left_out(tmp_path):
    """A timeout comes first and hides nothing; work left out has its own return code, text and bits."""
    out, _ = _run(tmp_path, r"""
static void look(dsv4cu_ctx *c)
{
    int code = 99;
    const int r = dsv4cu_ctx_status(c, nullptr, &code);
    printf("%d %d %s\n", r, code, r ? dsv4cu_last_error() : "");
}
int main()
{
    dsv4cu_ctx *c;
    dsv4cu_ctx_create(&c, 0);
    look(c);
    c->status[0] = 81;                       // a wait that gave up, and two refusals
    c->status[1] = 1 << (DSV4CU_NO_ROWS - DSV4CU_NO_PAGES) | 1 << (DSV4CU_VERIFY_NODES - DSV4CU_NO_PAGES);
    c->counters[7] = 3;
    look(c);
    printf("%d\n", c->counters[7]);
    look(c);
    look(c);
    c->status[1] = 1;
    c->counters[7] = 3;
    look(c);
    printf("%d\n", c->counters[7]);          // a refusal leaves no counts behind, nor clears any
    unsigned bits = 99;
    c->status[0] = 5;
    c->status[1] = 1 | 1 << 4;
    printf("%d", dsv4cu_ctx_refused(c, nullptr, &bits));
    printf(" %u\n", bits);
    look(c);
    look(c);
    printf("%d %d\n", dsv4cu_ctx_refused(nullptr, nullptr, &bits), dsv4cu_ctx_refused(c, nullptr, nullptr));
    dsv4cu_ctx_destroy(c);
    return 0;
}
""")
    assert out[0] == "0 0 "
    assert out[1].startswith("-5 81 ") and "timed out" in out[1] and out[2] == "0"
    assert out[3].startswith("-8 72 ") and "timed out" not in out[3] and "(72)" in out[3] and "(76)" in out[3]
    assert out[4] == "0 0 "
    assert out[5].startswith("-8 71 ") and "pages" in out[5] and out[6] == "3"
    assert out[7] == "0 17" and out[8].startswith("-5 5 ") and out[9] == "0 0 " and out[10] == "-1 -1"


def test_context_calls_run_on_the_contexts_device(tmp_path):
    """Reserving, looking and growing work on the context's device whichever device is current, and leave that current."""
    out, calls = _run(tmp_path, r"""
int main()
{
    dsv4cu_ctx *c;
    dsv4cu_ctx_create(&c, 1);
    fprintf(stderr, "--\n");
    int code;
    unsigned bits;
    void *ws;
    dsv4cu_ctx_reserve(c, 1 << 20);
    printf("%d\n", current);
    dsv4cu_ws_get(c, 5 << 20, &ws);
    printf("%d\n", current);
    c->status[0] = 9;
    dsv4cu_ctx_status(c, nullptr, &code);
    printf("%d\n", current);
    c->status[1] = 2;
    dsv4cu_ctx_status(c, nullptr, &code);
    c->status[1] = 2;
    dsv4cu_ctx_refused(c, nullptr, &bits);
    printf("%d %u\n", current, bits);
    dsv4cu_ctx_destroy(c);
    printf("%d\n", current);
    return 0;
}
""")
    assert out == ["0", "0", "0", "0 2", "0"]
    calls = calls[calls.index("--") + 1:]
    assert {x.split()[0] for x in calls} >= {"malloc", "free", "memset", "memcpy", "stream", "device"}
    assert all(x.split()[1] == "1" for x in calls), calls
