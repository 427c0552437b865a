// C entries of the 8-bit paged KV cache and of sm_draw: checks of arguments,
// workspaces, launches.
#include <cuda_runtime.h>
#include <math.h>

#include <exception>
#include <new>
#include <string>

#include "../../include/sm_engine.h"
#include "common.hpp"
#include "kv8.cuh"

using namespace sm;

struct sm_kv8_ws {
  int device = 0;
  uint32_t sms = 0;
  float* part = nullptr;  // partial results, then kept products
  float* keep() const { return part + kv8_attn_part_floats(sms); }
  uint32_t* cnt = nullptr;  // the counters, then the error word
  uint32_t* err() const { return cnt + kv8_attn_counters(sms); }
};

namespace {

int arg_error(const char* fn, const std::string& what) {
  set_error(std::string(fn) + ": " + what);
  return SM_ERR_ARG;
}
int cuda_error(const char* fn, cudaError_t e) {
  cudaGetLastError();
  set_error(std::string(fn) + ": " + cudaGetErrorString(e));
  return e == cudaErrorMemoryAllocation ? SM_ERR_OOM : SM_ERR_CUDA;
}

// The checks of one call, the first failure kept: conditions; null and
// misaligned pointers as they are named; outputs that share bytes with another
// argument (its CTAs read inputs after others have written); and in memory(),
// which needs a device, that each pointer is memory of the current one.
struct Check {
  const char* fn;
  int dev = -1, rc = SM_OK;
  struct { const char* name; const void* p; uint64_t bytes; bool out; } ptrs[13];
  uint32_t n_ptrs = 0;
  explicit Check(const char* f) : fn(f) {}
  void want(bool ok, const char* what) {
    if (!rc && !ok) rc = arg_error(fn, what);
  }
  // bytes 0: not compared with the others
  void ptr(const char* name, const void* p, size_t align, bool optional = false, uint64_t bytes = 0, bool out = false) {
    if (rc || (!p && optional)) return;
    if (!p) { rc = arg_error(fn, std::string(name) + " is null"); return; }
    if ((uintptr_t)p % align) { rc = arg_error(fn, std::string(name) + " must be " + std::to_string(align) + "-byte aligned"); return; }
    for (uint32_t i = 0; i < n_ptrs; i++)
      if (bytes && ptrs[i].bytes && (out || ptrs[i].out) && (uintptr_t)p < (uintptr_t)ptrs[i].p + ptrs[i].bytes &&
          (uintptr_t)ptrs[i].p < (uintptr_t)p + bytes) {
        rc = arg_error(fn, std::string(name) + " overlaps " + ptrs[i].name);
        return;
      }
    ptrs[n_ptrs++] = {name, p, bytes, out};
  }
  int memory() {
    if (rc) return rc;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return rc = cuda_error(fn, e);
    for (uint32_t i = 0; i < n_ptrs; i++) {
      cudaPointerAttributes at{};
      e = cudaPointerGetAttributes(&at, ptrs[i].p);
      if (e != cudaSuccess) return rc = cuda_error(fn, e);
      if (at.type != cudaMemoryTypeManaged && (at.type != cudaMemoryTypeDevice || at.device != dev))
        return rc = arg_error(fn, std::string(ptrs[i].name) + " is not memory of the current device");
    }
    return SM_OK;
  }
};

size_t type_size(uint32_t t) { return t == ACT_F32 ? 4 : t == ACT_F16 || t == ACT_BF16 ? 2 : 0; }

void check_cache(Check& ck, const sm_kv8* c) {
  ck.want(c, "null cache");
  if (ck.rc) return;
  ck.want(c->format == SM_KV8_E4M3 || c->format == SM_KV8_I8, "unknown cache format");
  ck.want(c->head_dim >= 16 && c->head_dim <= 128 && c->head_dim % 16 == 0, "head_dim must be a multiple of 16, 16..128");
  ck.want(c->n_kv_heads >= 1 && c->n_kv_heads <= 1024, "n_kv_heads must be 1..1024");
  ck.want(c->n_pages >= 1 && c->n_pages <= 0x7FFFFFFF, "n_pages must be 1..2^31 - 1");
}
void check_cache_memory(Check& ck, const sm_kv8* c, bool out) {
  const uint64_t parts = c->n_pages * c->n_kv_heads * 2;
  ck.ptr("codes_dev", c->codes_dev, 16, false, parts * KV8_PAGE * c->head_dim, out);
  ck.ptr("scales_dev", c->scales_dev, 8, false, parts * sizeof(float), out);
}

Kv8 cache_of(const sm_kv8* c) {
  return Kv8{(uint8_t*)c->codes_dev, c->scales_dev, (uint32_t)c->n_pages, c->n_kv_heads, c->head_dim, c->format};
}

template <typename F>
int guarded(const char* fn, F f) {
  try {
    return f();
  } catch (const std::bad_alloc&) {
    set_error("out of host memory");
    return SM_ERR_OOM;
  } catch (const std::exception& e) {
    set_error(std::string(fn) + ": " + e.what());
    return SM_ERR_STATE;
  }
}

}  // namespace

extern "C" {

int sm_kv_plan(uint64_t n_seqs, const int32_t* lens_dev, const int32_t* add_dev, int32_t* table_dev, uint64_t table_ld,
               const int32_t* free_dev, const int32_t* n_free_dev, uint64_t n_rows, int32_t* lens_out_dev,
               int32_t* first_dev, int64_t* slots_dev, int32_t* pos_dev, int32_t* seq_dev, int32_t* status_dev,
               void* stream) {
  return guarded("sm_kv_plan", [&]() -> int {
    Check ck("sm_kv_plan");
    ck.want(n_seqs <= KV8_PLAN_MAX_SEQS, "at most 16384 sequences");
    ck.want(n_rows <= 0x7FFFFFFF, "at most 2^31 - 1 rows");
    ck.want(table_ld <= 0x7FFFFFFF, "table_ld must be below 2^31");
    if (ck.rc) return ck.rc;
    ck.ptr("lens_dev", lens_dev, 4, !n_seqs, n_seqs * 4);
    ck.ptr("add_dev", add_dev, 4, !n_seqs, n_seqs * 4);
    ck.ptr("table_dev", table_dev, 4, !n_seqs || !table_ld, n_seqs * table_ld * 4, true);
    ck.ptr("free_dev", free_dev, 4, true, 4);  // its length lies on the device
    ck.ptr("n_free_dev", n_free_dev, 4, false, 4);
    ck.ptr("lens_out_dev", lens_out_dev, 4, !n_seqs, n_seqs * 4, true);
    ck.ptr("first_dev", first_dev, 4, false, (n_seqs + 1) * 4, true);
    ck.ptr("slots_dev", slots_dev, 8, !n_rows, n_rows * 8, true);
    ck.ptr("pos_dev", pos_dev, 4, true, n_rows * 4, true);
    ck.ptr("seq_dev", seq_dev, 4, true, n_rows * 4, true);
    ck.ptr("status_dev", status_dev, 4, false, 8, true);
    if (ck.memory()) return ck.rc;
    Kv8PlanArgs a{lens_dev, add_dev, table_dev, table_ld, free_dev, n_free_dev, (uint32_t)n_seqs, (uint32_t)n_rows,
                  lens_out_dev, first_dev, slots_dev, pos_dev, seq_dev, status_dev};
    int sms = 0;
    cudaError_t e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, ck.dev);
    if (e == cudaSuccess) e = launch_kv8_plan(a, (uint32_t)sms, (cudaStream_t)stream);
    return e == cudaSuccess ? SM_OK : cuda_error("sm_kv_plan", e);
  });
}

int sm_kv8_append(const sm_kv8* c, const void* k_dev, const void* v_dev, uint32_t type, uint64_t n_rows, uint64_t ld_k,
                  uint64_t ld_v, const int64_t* slots_dev, void* stream) {
  return guarded("sm_kv8_append", [&]() -> int {
    Check ck("sm_kv8_append");
    check_cache(ck, c);
    const size_t es = type_size(type);
    ck.want(es, "type must be F32, F16 or BF16");
    ck.want(n_rows <= 0x7FFFFFFF, "at most 2^31 - 1 rows");
    if (ck.rc || !n_rows) return ck.rc;
    const uint64_t width = (uint64_t)c->n_kv_heads * c->head_dim;
    if (!ld_k) ld_k = width;
    if (!ld_v) ld_v = width;
    ck.want(ld_k >= width && ld_v >= width && ld_k < (1ull << 32) && ld_v < (1ull << 32), "a row stride is below n_kv_heads x head_dim, or 2^32 and above");
    ck.want(ld_k * es % 16 == 0 && ld_v * es % 16 == 0, "row strides must be multiples of 16 bytes");
    check_cache_memory(ck, c, true);
    ck.ptr("k_dev", k_dev, 16, false, ((n_rows - 1) * ld_k + width) * es);
    ck.ptr("v_dev", v_dev, 16, false, ((n_rows - 1) * ld_v + width) * es);
    ck.ptr("slots_dev", slots_dev, 8, false, n_rows * 8);
    if (ck.memory()) return ck.rc;
    const cudaError_t e = launch_kv8_append(cache_of(c), k_dev, v_dev, type, (uint32_t)n_rows, ld_k, ld_v, slots_dev, (cudaStream_t)stream);
    return e == cudaSuccess ? SM_OK : cuda_error("sm_kv8_append", e);
  });
}

int sm_kv8_ws_new(sm_kv8_ws** out) {
  return guarded("sm_kv8_ws_new", [&]() -> int {
    if (!out) return arg_error("sm_kv8_ws_new", "null argument");
    *out = nullptr;
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return cuda_error("sm_kv8_ws_new", e);
    // One allocation, the counters and the error word behind the partial results and kept products. They are zeroed on a stream of
    // the call's own, so that no other work is waited for.
    const size_t part = (kv8_attn_part_floats((uint32_t)sms) + kv8_attn_keep_floats((uint32_t)sms)) * sizeof(float);
    const size_t cnt = (kv8_attn_counters((uint32_t)sms) + 1) * sizeof(uint32_t);
    auto* w = new sm_kv8_ws;
    w->device = dev;
    w->sms = (uint32_t)sms;
    cudaStream_t st = nullptr;
    e = cudaMalloc(&w->part, part + cnt);
    if (e == cudaSuccess) e = cudaStreamCreateWithFlags(&st, cudaStreamNonBlocking);
    if (e == cudaSuccess) {
      w->cnt = (uint32_t*)((char*)w->part + part);
      e = cudaMemsetAsync(w->cnt, 0, cnt, st);
      if (e == cudaSuccess) e = cudaStreamSynchronize(st);
      cudaStreamDestroy(st);
    }
    if (e != cudaSuccess) {
      cudaFree(w->part);
      delete w;
      return cuda_error("sm_kv8_ws_new", e);
    }
    *out = w;
    return SM_OK;
  });
}

int sm_kv8_ws_free(sm_kv8_ws* w) {
  if (!w) return SM_OK;
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev != w->device) cudaSetDevice(w->device);
  cudaFree(w->part);
  if (dev != w->device) cudaSetDevice(dev);
  delete w;
  return SM_OK;
}

int sm_kv8_ws_status(const sm_kv8_ws* w, void* stream) {
  return guarded("sm_kv8_ws_status", [&]() -> int {
    if (!w) return arg_error("sm_kv8_ws_status", "null workspace");
    uint32_t h = 0;
    cudaError_t e = cudaMemcpyAsync(&h, w->err(), sizeof(h), cudaMemcpyDeviceToHost, (cudaStream_t)stream);
    if (e == cudaSuccess) e = cudaStreamSynchronize((cudaStream_t)stream);
    if (e == cudaSuccess && h) e = cudaMemsetAsync(w->cnt, 0, (kv8_attn_counters(w->sms) + 1) * sizeof(uint32_t), (cudaStream_t)stream);
    if (e != cudaSuccess) return cuda_error("sm_kv8_ws_status", e);
    if (!h) return SM_OK;
    set_error("sm_kv8_attend: a bounded wait gave up");
    return SM_ERR_CUDA;
  });
}

int sm_kv8_attend(const sm_kv8* c, sm_kv8_ws* ws, const void* q_dev, void* out_dev, uint32_t type, uint64_t n_rows,
                  uint32_t n_heads, uint64_t ld_q, uint64_t ld_out, uint64_t n_seqs, const int32_t* lens_dev,
                  const int32_t* first_dev, const int32_t* table_dev, uint64_t table_ld, float scale, uint32_t window,
                  void* stream) {
  return guarded("sm_kv8_attend", [&]() -> int {
    Check ck("sm_kv8_attend");
    check_cache(ck, c);
    ck.want(ws, "null workspace");
    const size_t es = type_size(type);
    ck.want(es, "type must be F32, F16 or BF16");
    if (ck.rc) return ck.rc;
    ck.want(n_heads >= 1 && n_heads % c->n_kv_heads == 0, "n_heads must be a multiple of n_kv_heads");
    ck.want(n_rows <= 0x7FFFFFFF && n_rows * n_heads <= 0x7FFFFFFF, "n_rows x n_heads must be below 2^31");
    ck.want(n_seqs <= 0x7FFFFFFF, "at most 2^31 - 1 sequences");
    ck.want(table_ld <= 0x7FFFFFFF, "table_ld must be below 2^31");
    ck.want(isfinite(scale), "scale must be finite");
    if (ck.rc || !n_rows || !n_seqs) return ck.rc;
    const uint64_t width = (uint64_t)n_heads * c->head_dim;
    if (!ld_q) ld_q = width;
    if (!ld_out) ld_out = width;
    ck.want(ld_q >= width && ld_out >= width && ld_q < (1ull << 32) && ld_out < (1ull << 32), "a row stride is below n_heads x head_dim, or 2^32 and above");
    ck.want(ld_q * es % 16 == 0 && ld_out * es % 16 == 0, "row strides must be multiples of 16 bytes");
    check_cache_memory(ck, c, false);
    // Every row of q is read before it is written in out: they may be the same rows, or other columns of a matrix
    // that holds both, but must not overlap in another way.
    const uint64_t q0 = (uint64_t)(uintptr_t)q_dev, o0 = (uint64_t)(uintptr_t)out_dev, row = width * es;
    const uint64_t q1 = q0 + ((n_rows - 1) * ld_q + width) * es, o1 = o0 + ((n_rows - 1) * ld_out + width) * es;
    if (q0 < o1 && o0 < q1) {
      const uint64_t pitch = ld_q * es, apart = (o0 > q0 ? o0 - q0 : q0 - o0) % pitch;
      ck.want(ld_q == ld_out && (q0 == o0 || (apart >= row && apart <= pitch - row)), "out overlaps q other than row on row");
    }
    ck.ptr("q_dev", q_dev, 16);
    ck.ptr("out_dev", out_dev, 16, false, o1 - o0, true);
    ck.ptr("lens_dev", lens_dev, 4, false, n_seqs * 4);
    ck.ptr("first_dev", first_dev, 4, false, (n_seqs + 1) * 4);
    ck.ptr("table_dev", table_dev, 4, !table_ld, n_seqs * table_ld * 4);
    if (ck.memory()) return ck.rc;
    if (ws->device != ck.dev) return arg_error("sm_kv8_attend", "the workspace belongs to another device");
    Kv8AttnArgs a{};
    a.c = cache_of(c);
    a.q = q_dev, a.out = out_dev, a.ld_q = ld_q, a.ld_out = ld_out;
    a.lens = lens_dev, a.first = first_dev, a.table = table_dev, a.table_ld = table_ld;
    a.n_seqs = (uint32_t)n_seqs, a.n_rows = (uint32_t)n_rows, a.n_heads = n_heads, a.group = n_heads / c->n_kv_heads;
    a.window = window;
    a.scale = scale;
    a.part = ws->part, a.keep = ws->keep(), a.cnt = ws->cnt, a.err = ws->err();
    const cudaError_t e = launch_kv8_attn(a, type, ws->sms, (cudaStream_t)stream);
    return e == cudaSuccess ? SM_OK : cuda_error("sm_kv8_attend", e);
  });
}

int sm_draw(const void* logits_dev, uint32_t type, uint64_t n_rows, uint64_t ld, uint64_t vocab, const uint8_t* mask_dev,
            const sm_draw_params* params_dev, const float* u_dev, int32_t* tokens_dev, float* logprobs_dev, void* stream) {
  return guarded("sm_draw", [&]() -> int {
    Check ck("sm_draw");
    const size_t es = type_size(type);
    ck.want(es, "type must be F32, F16 or BF16");
    ck.want(vocab >= 1 && vocab <= DRAW_MAX_VOCAB, "vocab must be 1..524288");
    ck.want(!ld || (ld >= vocab && ld < (1ull << 32)), "ld is below vocab, or 2^32 and above");
    ck.want(n_rows <= 65536, "at most 65536 rows");
    if (ck.rc || !n_rows) return ck.rc;
    const uint64_t span = ld && n_rows > 1 ? (n_rows - 1) * ld + vocab : n_rows * vocab;
    ck.ptr("logits_dev", logits_dev, es, false, span * es);
    ck.ptr("mask_dev", mask_dev, 1, true, span);
    ck.ptr("params_dev", params_dev, 16, false, n_rows * sizeof(sm_draw_params));
    ck.ptr("u_dev", u_dev, 4, false, n_rows * 4);
    ck.ptr("tokens_dev", tokens_dev, 4, false, n_rows * 4, true);
    ck.ptr("logprobs_dev", logprobs_dev, 4, true, n_rows * 4, true);
    if (ck.memory()) return ck.rc;
    static_assert(sizeof(sm_draw_params) == sizeof(DrawParams) && sizeof(DrawParams) == 16, "16 bytes a row");
    DrawArgs a{logits_dev, mask_dev, (const DrawParams*)params_dev, u_dev, tokens_dev, logprobs_dev, ld ? ld : vocab,
               (uint32_t)n_rows, (uint32_t)vocab, type};
    int sms = 0;
    cudaError_t e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, ck.dev);
    if (e == cudaSuccess) e = launch_draw(a, (uint32_t)sms, (cudaStream_t)stream);
    return e == cudaSuccess ? SM_OK : cuda_error("sm_draw", e);
  });
}

}  // extern "C"
