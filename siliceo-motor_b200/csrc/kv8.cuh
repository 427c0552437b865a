// The 8-bit paged KV cache of hosts that batch their own requests: types and
// launchers of its kernels (kv8.cu: page plan and append; kv8_attn.cuh and
// kv8_chunk.cuh: attention; draw.cu: the sampler that follows a step).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

namespace sm {

// A kernel's shared memory limit, raised once on each device.
struct SmemOnce {
  std::atomic<uint64_t> done{0};
  cudaError_t allow(const void* kern, int bytes) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || (dev < 64 && done.load(std::memory_order_relaxed) >> dev & 1)) return e;
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && dev < 64) done.fetch_or(1ull << dev, std::memory_order_relaxed);
    return e;
  }
};

// Positions of a page: the engine's own page size (device.cuh).
constexpr uint32_t KV8_PAGE = 32;
// Sequences one plan takes: their two prefix sums stay in shared memory.
constexpr uint32_t KV8_PLAN_MAX_SEQS = 16384;
// Exponent of the smallest scale append writes (rows of zeros get it).
constexpr int KV8_MIN_EXP = -100;

enum Kv8Format : uint32_t { KV8_E4M3 = 0, KV8_I8 = 1 };
enum ActType : uint32_t { ACT_F32 = 0, ACT_F16 = 1, ACT_BF16 = 30 };  // ggml type codes

// One layer's cache: codes [page][kv head][K, V][32][hd], scales [page][kv head][K, V].
struct Kv8 {
  uint8_t* codes;
  float* scales;
  uint32_t n_pages, heads, hd, fmt;
};

struct Kv8PlanArgs {
  const int32_t *lens, *add;
  int32_t* table;
  uint64_t table_ld;
  const int32_t *free_pages, *n_free;
  uint32_t n_seqs, n_rows;
  int32_t *lens_out, *first;
  int64_t* slots;
  int32_t *pos, *seq;  // may be null
  int32_t* status;
};

struct Kv8AttnArgs {
  Kv8 c;
  const void* q;
  void* out;
  uint64_t ld_q, ld_out;  // elements between rows
  const int32_t *lens, *first, *table;
  uint64_t table_ld;
  uint32_t n_seqs, n_rows, n_heads, group;  // group = n_heads / c.heads
  uint32_t window;                          // 0: none
  float scale;
  float* part;    // partial results, kv8_attn_part_floats()
  float* keep;    // a CTA's products so far, kv8_attn_keep_floats()
  uint32_t* cnt;  // arrival counters, zero between launches, kv8_attn_counters()
  uint32_t* err;  // set when a bounded wait gave up
};

struct DrawParams {
  float temperature;
  int32_t top_k;
  float top_p, min_p;
};
struct DrawArgs {
  const void* logits;
  const uint8_t* mask;  // may be null
  const DrawParams* params;
  const float* u;
  int32_t* tokens;
  float* logprobs;  // may be null
  uint64_t ld;
  uint32_t n_rows, vocab, type;
};

cudaError_t launch_kv8_plan(const Kv8PlanArgs& a, uint32_t sms, cudaStream_t st);
// ld_k, ld_v: elements between rows.
cudaError_t launch_kv8_append(const Kv8& c, const void* k, const void* v, uint32_t type, uint32_t n_rows, uint64_t ld_k,
                              uint64_t ld_v, const int64_t* slots, cudaStream_t st);
// Streaming attention (kv8_attn.cuh), one translation unit a row type.
constexpr uint32_t KV8_MAX_HD = 128;
constexpr uint32_t KV8_PART_FLOATS = 16 * (KV8_MAX_HD + 2);  // a partial result of up to 16 rows: o, then m and l
constexpr uint32_t KV8_CHUNK_PART_FLOATS = 128 * (KV8_MAX_HD + 2);  // the tensor-core form's (kv8_chunk.cuh, two CTAs an SM)
inline uint64_t kv8_attn_part_floats(uint32_t sms) { return (uint64_t)sms * 2 * 2 * KV8_CHUNK_PART_FLOATS; }
constexpr uint32_t KV8_KEEP_FLOATS = 16 * 68 * 32;  // of an SM: O and m of 16 warps' lanes, or O of two CTAs' 128 rows
inline uint64_t kv8_attn_keep_floats(uint32_t sms) { return (uint64_t)sms * KV8_KEEP_FLOATS; }
inline uint32_t kv8_attn_counters(uint32_t sms) { return sms * 2; }
cudaError_t launch_kv8_attn_f32(const Kv8AttnArgs& a, uint32_t sms, cudaStream_t st);
cudaError_t launch_kv8_attn_f16(const Kv8AttnArgs& a, uint32_t sms, cudaStream_t st);
cudaError_t launch_kv8_attn_bf16(const Kv8AttnArgs& a, uint32_t sms, cudaStream_t st);
inline cudaError_t launch_kv8_attn(const Kv8AttnArgs& a, uint32_t type, uint32_t sms, cudaStream_t st) {
  return type == ACT_F32   ? launch_kv8_attn_f32(a, sms, st)
         : type == ACT_F16 ? launch_kv8_attn_f16(a, sms, st)
                           : launch_kv8_attn_bf16(a, sms, st);
}
// Largest vocabulary launch_draw takes.
constexpr uint32_t DRAW_MAX_VOCAB = 1u << 19;
cudaError_t launch_draw(const DrawArgs& a, uint32_t sms, cudaStream_t st);

}  // namespace sm
