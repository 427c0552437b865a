// Attention over the 8-bit KV cache for BF16 rows (kv8_attn.cuh).
#include "kv8_attn.cuh"

namespace sm {
cudaError_t launch_kv8_attn_bf16(const Kv8AttnArgs& a, uint32_t sms, cudaStream_t st) { return attn_typed<__nv_bfloat16>(a, sms, st); }
}  // namespace sm
