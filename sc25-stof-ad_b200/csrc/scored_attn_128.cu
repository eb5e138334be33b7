// Attention by formula and rules for heads of 128 (scored_attn.cuh).
#include "scored_attn.cuh"

namespace stof {
template <>
int launch_scored<128>(const ScoredMaps& maps, const ScoredParams& p, int halves, bool bf16, int mode, long long blocks, size_t smem, cudaStream_t stream) {
    return launch_scored_impl<128>(maps, p, halves, bf16, mode, blocks, smem, stream);
}
}  // namespace stof
