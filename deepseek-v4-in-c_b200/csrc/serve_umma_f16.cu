// serve_umma_f16.cu - the tcgen05 serving attention, f16.
#include "serve_umma.cuh"

namespace dsv4cu {
int serve_umma_f16(const SaArgs &a, int D, bool tree, cudaStream_t st)
{
    return D == 64 ? serve_umma_launch<64, true>(a, tree, st) : serve_umma_launch<128, true>(a, tree, st);
}
}  // namespace dsv4cu
