// serve.h - host-side helpers shared by the paged serving operators.
#pragma once

#include "common.cuh"
#include "ctx.h"

namespace dsv4cu {

// The calling thread's current device for the length of a call: the call
// works on its context's device whichever device is current.
struct DeviceGuard {
    int prev = -1;
    bool moved = false;
    cudaError_t enter(int device)
    {
        cudaError_t e = cudaGetDevice(&prev);
        if (e == cudaSuccess && prev != device) {
            e = cudaSetDevice(device);
            moved = e == cudaSuccess;
        }
        return e;
    }
    ~DeviceGuard()
    {
        if (moved) cudaSetDevice(prev);
    }
};

// Work that a kernel leaves out: a bit beside the watchdog's word, so neither
// hides the other and no code hides another.
DSV4CU_DEV void serve_refuse(int *status, int code) { atomicOr(status + 1, 1 << (code - DSV4CU_NO_PAGES)); }

static inline int elem_bytes(int type) { return type == DSV4CU_F32 ? 4 : 2; }
static inline bool elem_known(int type) { return type == DSV4CU_F32 || type == DSV4CU_BF16 || type == DSV4CU_F16; }
static inline bool aligned16(const void *p) { return ((uintptr_t)p & 15u) == 0; }

}  // namespace dsv4cu
