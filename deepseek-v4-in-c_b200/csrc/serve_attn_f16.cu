// serve_attn_f16.cu - the paged serving attention's mma.sync kernels, f16 queries and cache.
#include "serve_attn.cuh"

namespace dsv4cu {
int serve_attn_f16(const SaArgs &a, int D, bool tree, cudaStream_t st)
{
    return tree ? serve_attn_pick<1, true, true>(a, D, st) : serve_attn_pick<1, true, false>(a, D, st);
}
}  // namespace dsv4cu
