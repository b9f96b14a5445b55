// serve_attn_bf16.cu - the paged serving attention's mma.sync kernels, bf16 queries and cache.
#include "serve_attn.cuh"

namespace dsv4cu {
int serve_attn_bf16(const SaArgs &a, int D, bool tree, cudaStream_t st)
{
    return tree ? serve_attn_pick<1, false, true>(a, D, st) : serve_attn_pick<1, false, false>(a, D, st);
}
}  // namespace dsv4cu
