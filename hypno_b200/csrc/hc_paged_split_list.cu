// Split attention over the pages of each row's list (hc_paged_split.cuh has the kernels).
#include "hc_paged_split.cuh"

namespace hc {

int launch_split_list(SplitArgs& X, int q16, int kv, cudaStream_t s) {
    if (kv == HC_KV_Q4) return q16 ? launch_split_hd<__half, q4x, true>(X, s) : launch_split_hd<float, q4x, true>(X, s);
    if (kv == HC_KV_FP16) return q16 ? launch_split_hd<__half, __half, true>(X, s) : launch_split_hd<float, __half, true>(X, s);
    return q16 ? launch_split_hd<__half, float, true>(X, s) : launch_split_hd<float, float, true>(X, s);
}

}  // namespace hc
