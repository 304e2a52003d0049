// Attention over a paged cache of f16.
#include "paged_attention_mma.cuh"
#include "paged_attention_simt.cuh"

namespace focr {

int launch_attention_f16(AttnArgs &a, cudaStream_t st) {
    return mma_takes<__half>(a) ? launch_mma_dim<__half>(a, st) : launch_simt_dim<__half>(a, st);
}

}  // namespace focr
