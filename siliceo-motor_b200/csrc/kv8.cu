// Page plan and quantising append of the 8-bit paged KV cache.
#include "kv8.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>

namespace sm {
namespace {

// ------------------------------------------------------------------ plan ----
// With need_i = ceil((len_i + add_i) / 32) - ceil(len_i / 32) and the prefix
// sums R_i of add and P_i of need, every row's slot is closed-form: row t
// belongs to the i with R_i <= t < R_{i+1} and sits at position
// len_i + t - R_i; a page ceil(len_i / 32) + k of it is the (P_i + k)-th from
// the end of the free list. So every CTA makes both prefix sums of all the
// sequences itself (a few KB out of L2) and then works on rows of its own:
// one launch, no CTA waits for another. What it costs is latency (a dozen
// dependent steps), not bytes: 4.2 us a launch for 32 sequences, 5.6 us for
// 512 sequences with 33 thousand rows (0.55 MB).
constexpr uint32_t PLAN_THREADS = 512;
constexpr uint32_t PLAN_ROWS = 1024;  // rows a CTA takes at a time

// Exclusive prefix of v over the CTA; total gets the sum.
__device__ int64_t block_exclusive(int64_t v, int64_t* warp_sums, int64_t* total) {
  const uint32_t lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int64_t x = v;
  for (uint32_t o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(~0u, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // warp_sums may still be read from an earlier call
  if (lane == 31) warp_sums[w] = x;
  __syncthreads();
  int64_t before = 0, all = 0;
  for (uint32_t i = 0; i < PLAN_THREADS / 32; i++) {
    const int64_t s = warp_sums[i];
    before += i < w ? s : 0;
    all += s;
  }
  *total = all;
  return before + x - v;
}

__global__ void __launch_bounds__(PLAN_THREADS) kv8_plan_kernel(Kv8PlanArgs a) {
  extern __shared__ int32_t plan_smem[];
  __shared__ int64_t warp_sums[PLAN_THREADS / 32];
  const uint32_t n = a.n_seqs, tid = threadIdx.x;
  int32_t* end = plan_smem;          // R_{i+1}, clamped to int32
  int32_t* base = plan_smem + n;     // P_i, or -1: refused
  const uint32_t per = (n + PLAN_THREADS - 1) / PLAN_THREADS;
  const uint32_t i0 = min(n, tid * per), i1 = min(n, i0 + per);
  const int64_t cap = min((int64_t)min(a.table_ld, (uint64_t)INT32_MAX) * KV8_PAGE, (int64_t)INT32_MAX);

  int64_t mine = 0, total;
  for (uint32_t i = i0; i < i1; i++) {
    const int32_t l = a.lens[i], d = a.add[i];
    mine += l >= 0 && d >= 0 ? d : 0;
  }
  int64_t r = block_exclusive(mine, warp_sums, &total);
  int64_t need = 0;
  for (uint32_t i = i0; i < i1; i++) {
    const int32_t l = a.lens[i], d = a.add[i];
    const bool sane = l >= 0 && d >= 0;
    r += sane ? d : 0;
    end[i] = (int32_t)min(r, (int64_t)INT32_MAX);
    const bool fits = sane && (int64_t)l + d <= cap && r <= (int64_t)a.n_rows;
    const int32_t w = fits ? (int32_t)(((int64_t)l + d + KV8_PAGE - 1) / KV8_PAGE - ((int64_t)l + KV8_PAGE - 1) / KV8_PAGE) : -1;
    base[i] = w;
    need += max(w, 0);
  }
  const int64_t have = a.free_pages ? max(*a.n_free, 0) : 0;
  int64_t p = block_exclusive(need, warp_sums, &total);
  int64_t used = 0, refused = 0;
  for (uint32_t i = i0; i < i1; i++) {
    const int32_t w = base[i];
    p += max(w, 0);
    const bool ok = w == 0 || (w > 0 && p <= have);
    base[i] = ok ? (int32_t)min(p - w, (int64_t)INT32_MAX) : -1;
    used += ok ? w : 0;
    refused += !ok;
  }
  int64_t all_used, all_refused;
  block_exclusive(used, warp_sums, &all_used);
  block_exclusive(refused, warp_sums, &all_refused);
  __syncthreads();

  const uint32_t gtid = blockIdx.x * PLAN_THREADS + tid, gsize = gridDim.x * PLAN_THREADS;
  if (gtid == 0) {
    a.status[0] = (int32_t)(have - all_used);
    a.status[1] = (int32_t)all_refused;
    a.first[0] = 0;
  }
  for (uint32_t i = gtid; i < n; i += gsize) {
    a.first[i + 1] = end[i];
    a.lens_out[i] = base[i] >= 0 ? a.lens[i] + a.add[i] : -1;
  }
  for (uint64_t t0 = (uint64_t)blockIdx.x * PLAN_ROWS; t0 < a.n_rows; t0 += (uint64_t)gridDim.x * PLAN_ROWS) {
    for (uint32_t k = tid; k < PLAN_ROWS && t0 + k < a.n_rows; k += PLAN_THREADS) {
      const uint32_t t = (uint32_t)(t0 + k);
      uint32_t lo = 0, hi = n;  // the first sequence that ends behind row t
      while (lo < hi) {
        const uint32_t mid = (lo + hi) / 2;
        if ((uint32_t)end[mid] > t) hi = mid; else lo = mid + 1;
      }
      int64_t slot = -1;
      int32_t pos = -1;
      if (lo < n && base[lo] >= 0) {
        const int32_t len = a.lens[lo];
        pos = len + (int32_t)(t - (lo ? (uint32_t)end[lo - 1] : 0u));
        const int32_t pg = pos / (int32_t)KV8_PAGE, held = (int32_t)(((int64_t)len + KV8_PAGE - 1) / KV8_PAGE);
        int32_t* entry = a.table + lo * a.table_ld + pg;
        int32_t page;
        if (pg < held) {
          page = *entry;
        } else {
          page = a.free_pages[have - 1 - ((int64_t)base[lo] + pg - held)];
          if (pos % (int32_t)KV8_PAGE == 0) *entry = page;  // the new page's first row
        }
        slot = page < 0 ? -1 : (int64_t)page * KV8_PAGE + pos % (int32_t)KV8_PAGE;
      }
      a.slots[t] = slot;
      if (a.pos) a.pos[t] = pos;
      if (a.seq) a.seq[t] = lo < n ? (int32_t)lo : -1;
    }
  }
}

// ---------------------------------------------------------------- append ----
// A page's rows of one head share a scale 2^E, the smallest with
// max |x| <= M 2^E (M = 448 for e4m3, 127 for int8). A power of two makes
// x / 2^E exact, so a code is the correctly rounded one and does not depend on
// the order of arithmetic, and when later rows raise E the codes of the rows
// already there move by 2^-k: one more rounding, of the exact value.
//
// Rows of a page that one call writes are consecutive (a "run": slots rise by
// one inside a page). A CTA takes the runs that begin in its `chunk` rows, for
// one head's K or V: eight elements a thread and pass, the whole run in
// registers between its maximum and its encoding, so the rows are read once.
// Memory-bound for prompts: 24 prompts of up to 1999 f16 rows, 8 heads of 128,
// to e4m3 in 40 us (224 MB, 5.5 TB/s, 0.85 of the measured 6515 GB/s; 47 us
// while the magnitudes were compared one by one; f32 rows 39 us for 24000, 6.3
// TB/s). For one row a sequence it is
// the chain slots -> scale -> store: 2.5 us for 32 rows.
constexpr uint32_t APP_GROUP = 128;

template <typename T>
struct Vec8;
template <>
struct Vec8<float> {
  float4 a, b;
  __device__ uint32_t top(uint32_t t) const {  // the larger of t and the magnitudes, as bits of a float
    const float x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 8; i++) t = max(t, __float_as_uint(x[i]) & 0x7FFFFFFFu);
    return t;
  }
  static __device__ uint32_t wide(uint32_t t) { return t; }
  __device__ void get(float (&x)[8]) const {
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  }
};
template <>
struct Vec8<__half> {
  uint4 v;
  // the larger of t and the magnitudes, two at a time as 16-bit integers (NaN above infinity)
  __device__ uint32_t top(uint32_t t) const {
    t = __vmaxu2(t, v.x & 0x7FFF7FFFu), t = __vmaxu2(t, v.y & 0x7FFF7FFFu);
    return __vmaxu2(__vmaxu2(t, v.z & 0x7FFF7FFFu), v.w & 0x7FFF7FFFu);
  }
  static __device__ uint32_t wide(uint32_t t) {  // as bits of a float
    t = max(t >> 16, t & 0xFFFFu);
    return t >= 0x7C00u ? 0x7F800000u + (t > 0x7C00u) : __float_as_uint(__half2float(__ushort_as_half((unsigned short)t)));
  }
  __device__ void get(float (&x)[8]) const {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    for (int i = 0; i < 4; i++) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
  }
};
template <>
struct Vec8<__nv_bfloat16> {
  uint4 v;
  // the larger of t and the magnitudes, two at a time as 16-bit integers (NaN above infinity)
  __device__ uint32_t top(uint32_t t) const {
    t = __vmaxu2(t, v.x & 0x7FFF7FFFu), t = __vmaxu2(t, v.y & 0x7FFF7FFFu);
    return __vmaxu2(__vmaxu2(t, v.z & 0x7FFF7FFFu), v.w & 0x7FFF7FFFu);
  }
  static __device__ uint32_t wide(uint32_t t) { return max(t & 0xFFFF0000u, t << 16); }  // as bits of a float
  __device__ void get(float (&x)[8]) const {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    for (int i = 0; i < 4; i++) x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
};

// 2^E for a largest magnitude with the bits `top` (finite).
template <uint32_t FMT>
__device__ float page_scale(uint32_t top) {
  // M = 1.75 * 2^8 (e4m3) or 1.984375 * 2^6 (int8)
  constexpr uint32_t frac = FMT == KV8_E4M3 ? 0x600000u : 0x7E0000u;
  constexpr int shift = FMT == KV8_E4M3 ? 8 : 6;
  int e = (int)(top >> 23) - 127 - shift + ((top & 0x7FFFFFu) > frac ? 1 : 0);
  if (top < 0x00800000u) e = KV8_MIN_EXP;  // zero and subnormal
  return __uint_as_float((uint32_t)(max(e, KV8_MIN_EXP) + 127) << 23);
}

template <uint32_t FMT>
__device__ uint32_t encode4(const float* x) {
  if (FMT == KV8_E4M3) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x[0], x[1]), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(x[2], x[3]), __NV_SATFINITE, __NV_E4M3);
    return lo | hi << 16;
  }
  uint32_t r = 0;
  for (int i = 0; i < 4; i++) r |= (uint32_t)(__float2int_rn(fminf(fmaxf(x[i], -127.f), 127.f)) & 0xFF) << (8 * i);
  return r;
}

template <uint32_t FMT>
__device__ uint32_t rescale4(uint32_t c, float ratio) {
  float x[4];
  if (FMT == KV8_E4M3) {
    for (int i = 0; i < 2; i++) {
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(c >> (16 * i)), __NV_E4M3);
      const float2 f = __half22float2(__half2(h));
      x[2 * i] = f.x * ratio, x[2 * i + 1] = f.y * ratio;
    }
  } else {
    for (int i = 0; i < 4; i++) x[i] = (float)(int8_t)(c >> (8 * i)) * ratio;
  }
  return encode4<FMT>(x);
}

// EVEN: head_dim divides 1024, a thread's vectors share a column.
template <uint32_t FMT, typename T, bool EVEN>
__global__ void __launch_bounds__(APP_GROUP, sizeof(T) == 4 ? 8 : 10)
    kv8_append_kernel(Kv8 c, const T* k, const T* v, uint32_t n_rows, uint64_t ld_k, uint64_t ld_v, const int64_t* slots,
                      uint32_t chunk) {
  __shared__ uint32_t tops[2][4];
  const uint32_t lane = threadIdx.x & 31, tid = threadIdx.x, head = blockIdx.y >> 1, which = blockIdx.y & 1;
  const uint32_t base = blockIdx.x * chunk, cpr = c.hd / 8;
  const uint32_t row0 = tid / cpr, col0 = tid - row0 * cpr;
  const uint32_t inv_cpr = (65536 + cpr - 1) / cpr;  // x * inv_cpr >> 16 is x / cpr for the x here (below 512)
  const T* src = which ? v : k;
  const uint64_t ld = which ? ld_v : ld_k;
  const int64_t n_slots = (int64_t)c.n_pages * KV8_PAGE;
  // the chunk's slots and those of the 32 rows behind it, where its last run may end: lane l has rows l and 32 + l
  auto slot_of = [&](uint32_t t) { return t < n_rows ? slots[t] : -2; };
  const int64_t s_lo = slot_of(base + lane), s_hi = slot_of(base + 32 + lane), s_first = base ? slots[base - 1] : -2;
  const int64_t s_up = __shfl_up_sync(~0u, s_lo, 1), s_before = lane ? s_up : s_first;
  const bool begins = lane < chunk && s_lo >= 0 && s_lo < n_slots && (s_lo % KV8_PAGE == 0 || s_before != s_lo - 1);
  uint32_t todo = __ballot_sync(~0u, begins), buf = 0;
  for (; todo; todo &= todo - 1, buf ^= 1) {
    const uint32_t first = __ffs(todo) - 1, t0 = base + first;
    const int64_t s0 = __shfl_sync(~0u, s_lo, first);
    const uint32_t page = (uint32_t)(s0 / KV8_PAGE), off = (uint32_t)(s0 % KV8_PAGE);
    const int64_t a = __shfl_sync(~0u, s_lo, (first + lane) & 31), b = __shfl_sync(~0u, s_hi, (first + lane) & 31);
    const bool goes = off + lane < KV8_PAGE && (first + lane < 32 ? a : b) == s0 + lane;
    const uint32_t stop = ~__ballot_sync(~0u, goes), rows = stop ? __ffs(stop) - 1 : 32;
    float* scale_at = c.scales + ((uint64_t)page * c.heads + head) * 2 + which;
    uint8_t* codes = c.codes + (((uint64_t)page * c.heads + head) * 2 + which) * KV8_PAGE * c.hd;
    const float old = off ? *scale_at : 0.f;

    // Vector i of this thread: 8 elements at column 8 col of row row(i), 128 vectors behind vector i - 1.
    auto row = [&](uint32_t i) { return EVEN ? row0 + i * (APP_GROUP / cpr) : (tid + i * APP_GROUP) * inv_cpr >> 16; };
    auto col = [&](uint32_t i) { return EVEN ? col0 : tid + i * APP_GROUP - row(i) * cpr; };
    Vec8<T> raw[4];
    uint32_t top = 0;
    const T* from = src + (uint64_t)t0 * ld + head * c.hd;
#pragma unroll
    for (uint32_t i = 0; i < 4; i++)
      if (row(i) < rows) raw[i] = *reinterpret_cast<const Vec8<T>*>(from + (uint64_t)row(i) * ld + col(i) * 8);
#pragma unroll
    for (uint32_t i = 0; i < 4; i++)
      if (row(i) < rows) top = raw[i].top(top);
    top = __reduce_max_sync(~0u, Vec8<T>::wide(top));
    if (lane == 0) tops[buf][tid / 32] = top;
    __syncthreads();
    for (int i = 0; i < 4; i++) top = max(top, tops[buf][i]);

    uint8_t* to = codes + off * c.hd;
    // A row that is not finite makes the scale NaN: the page's values of this head are NaN from then on.
    if (top >= 0x7F800000u || old != old) {
      if (tid == 0) *scale_at = __uint_as_float(0x7FC00000u);
#pragma unroll
      for (uint32_t i = 0; i < 4; i++)
        if (row(i) < rows) *reinterpret_cast<uint2*>(to + row(i) * c.hd + col(i) * 8) = make_uint2(0, 0);
      continue;
    }
    const float s = fmaxf(old, page_scale<FMT>(top)), inv = 1.f / s;
    if (tid == 0) *scale_at = s;
    if (off && s > old) {
      const float ratio = old * inv;
      for (uint32_t at = tid * 8; at < off * c.hd; at += APP_GROUP * 8) {
        uint2* p = reinterpret_cast<uint2*>(codes + at);
        const uint2 w = *p;
        *p = make_uint2(rescale4<FMT>(w.x, ratio), rescale4<FMT>(w.y, ratio));
      }
    }
#pragma unroll
    for (uint32_t i = 0; i < 4; i++) {
      if (row(i) >= rows) continue;
      float x[8];
      raw[i].get(x);
#pragma unroll
      for (int j = 0; j < 8; j++) x[j] *= inv;
      *reinterpret_cast<uint2*>(to + row(i) * c.hd + col(i) * 8) = make_uint2(encode4<FMT>(x), encode4<FMT>(x + 4));
    }
  }
}

template <uint32_t FMT, typename T>
cudaError_t append_typed(const Kv8& c, const void* k, const void* v, uint32_t n_rows, uint64_t ld_k, uint64_t ld_v,
                         const int64_t* slots, cudaStream_t st) {
  // Rows a CTA looks at: 32 (about one run) for prompts; fewer while that would leave SMs without work.
  const uint32_t chunk = std::max(1u, std::min(32u, (uint32_t)((uint64_t)n_rows * c.heads / 1024)));
  const dim3 grid((n_rows + chunk - 1) / chunk, c.heads * 2);
  auto* kern = 1024 % c.hd ? kv8_append_kernel<FMT, T, false> : kv8_append_kernel<FMT, T, true>;
  kern<<<grid, APP_GROUP, 0, st>>>(c, (const T*)k, (const T*)v, n_rows, ld_k, ld_v, slots, chunk);
  return cudaGetLastError();
}

template <uint32_t FMT>
cudaError_t append_fmt(const Kv8& c, const void* k, const void* v, uint32_t type, uint32_t n_rows, uint64_t ld_k,
                       uint64_t ld_v, const int64_t* slots, cudaStream_t st) {
  switch (type) {
    case ACT_F32: return append_typed<FMT, float>(c, k, v, n_rows, ld_k, ld_v, slots, st);
    case ACT_F16: return append_typed<FMT, __half>(c, k, v, n_rows, ld_k, ld_v, slots, st);
    default: return append_typed<FMT, __nv_bfloat16>(c, k, v, n_rows, ld_k, ld_v, slots, st);
  }
}

}  // namespace

cudaError_t launch_kv8_plan(const Kv8PlanArgs& a, uint32_t sms, cudaStream_t st) {
  const size_t smem = (size_t)a.n_seqs * 8;
  if (smem > 40 * 1024) {
    static SmemOnce once;
    const cudaError_t e = once.allow((const void*)kv8_plan_kernel, KV8_PLAN_MAX_SEQS * 8);
    if (e != cudaSuccess) return e;
  }
  const uint32_t grid = std::max(1u, std::min(sms, (uint32_t)(((uint64_t)a.n_rows + PLAN_ROWS - 1) / PLAN_ROWS)));
  kv8_plan_kernel<<<grid, PLAN_THREADS, smem, st>>>(a);
  return cudaGetLastError();
}

cudaError_t launch_kv8_append(const Kv8& c, const void* k, const void* v, uint32_t type, uint32_t n_rows, uint64_t ld_k,
                              uint64_t ld_v, const int64_t* slots, cudaStream_t st) {
  if (!n_rows) return cudaSuccess;
  return c.fmt == KV8_E4M3 ? append_fmt<KV8_E4M3>(c, k, v, type, n_rows, ld_k, ld_v, slots, st)
                           : append_fmt<KV8_I8>(c, k, v, type, n_rows, ld_k, ld_v, slots, st);
}

}  // namespace sm
