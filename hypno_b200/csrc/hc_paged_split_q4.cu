// Split attention over a pool in 4 bits (hc_paged_split.cuh has the kernels).
#include "hc_paged_split.cuh"

namespace hc {

int launch_split_q4(SplitArgs& X, int q16, cudaStream_t s) {
    return q16 ? launch_split_hd<__half, q4x, false>(X, s) : launch_split_hd<float, q4x, false>(X, s);
}

}  // namespace hc
