// Attention over a paged cache of bf16.
#include "paged_attention_mma.cuh"
#include "paged_attention_simt.cuh"

namespace focr {

int launch_attention_bf16(AttnArgs &a, cudaStream_t st) {
    return mma_takes<__nv_bfloat16>(a) ? launch_mma_dim<__nv_bfloat16>(a, st) : launch_simt_dim<__nv_bfloat16>(a, st);
}

}  // namespace focr
