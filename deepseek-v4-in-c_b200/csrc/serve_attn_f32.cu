// serve_attn_f32.cu - the paged serving attention's mma.sync kernels, fp32 queries over a bf16 cache.
#include "serve_attn.cuh"

namespace dsv4cu {
int serve_attn_f32(const SaArgs &a, int D, bool tree, cudaStream_t st)
{
    return tree ? serve_attn_pick<3, false, true>(a, D, st) : serve_attn_pick<3, false, false>(a, D, st);
}
}  // namespace dsv4cu
