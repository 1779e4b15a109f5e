// Attention of chunks of new tokens over a paged K/V cache: head dimension 64.
#include "paged_chunk.cuh"

namespace pa {
namespace paged {
int launch_chunk_d64(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                    const ChunkParams& C, bool bf16, const PlanView& pv, float* scratch, int sms,
                    cudaStream_t stream) {
  return launch_chunk_body<64>(tq, tk, tv, C, bf16, pv, scratch, sms, stream);
}
}  // namespace paged
}  // namespace pa
