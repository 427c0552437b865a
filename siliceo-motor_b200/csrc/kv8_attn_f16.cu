// Attention over the 8-bit KV cache for F16 rows: few a sequence
// (kv8_attn.cuh) or many (kv8_chunk.cuh).
#include "kv8_chunk.cuh"

namespace sm {
cudaError_t launch_kv8_attn_f16(const Kv8AttnArgs& a, uint32_t sms, cudaStream_t st) {
  return chunk_takes(a) ? chunk_typed<__half>(a, sms, st) : attn_typed<__half>(a, sms, st);
}
}  // namespace sm
