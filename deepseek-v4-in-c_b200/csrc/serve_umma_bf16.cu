// serve_umma_bf16.cu - the tcgen05 serving attention, bf16.
#include "serve_umma.cuh"

namespace dsv4cu {
int serve_umma_bf16(const SaArgs &a, int D, bool tree, cudaStream_t st)
{
    return D == 64 ? serve_umma_launch<64, false>(a, tree, st) : serve_umma_launch<128, false>(a, tree, st);
}
}  // namespace dsv4cu
