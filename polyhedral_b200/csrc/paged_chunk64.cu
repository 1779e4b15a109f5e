// Attention of chunks of new tokens over a paged K/V cache: head dimension 64.
#include "paged_chunk.cuh"

namespace pa {
namespace paged {
int launch_chunk_d64(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                    const ChunkParams& C, bool bf16, const PlanView& pv, float* scratch, int sms,
                    cudaStream_t stream) {
  return bf16 ? launch_chunk_body<64, true>(tq, tk, tv, C, pv, scratch, sms, stream)
              : launch_chunk_body<64, false>(tq, tk, tv, C, pv, scratch, sms, stream);
}
}  // namespace paged
}  // namespace pa
