// Attention by formula and rules for heads of 64 (scored_attn.cuh).
#include "scored_attn.cuh"

namespace stof {
template <>
int launch_scored<64>(const ScoredMaps& maps, const ScoredParams& p, int halves, bool bf16, int mode, long long blocks, size_t smem, cudaStream_t stream) {
    return launch_scored_impl<64>(maps, p, halves, bf16, mode, blocks, smem, stream);
}
}  // namespace stof
