// Drawing tokens from logits with given uniform numbers: temperature, top-k,
// top-p and min-p, one row a request.
//
//   w_i = exp((x_i - max x) / T), rows sorted by x descending (lower index first)
//   kept: the first top_k; of those, while the weights before it sum to less
//   than top_p of their sum; of those, w_i >= min_p (the first always)
//   token: the first kept index, in the vocabulary's order, at which the
//   running sum of w passes u times the kept sum
//
// Which token comes out is a comparison of sums of up to 2^19 weights, so
// weights are 64-bit fixed-point numbers (2^-43, from an f64 evaluation): their
// sums are exact, whatever the order, and atomics cannot change a draw.
//
// A cluster of CTAs holds a row in shared memory and reads it once. No row is
// sorted: a histogram (2048 bins over the distance from the maximum) gives the
// bin in which the k-th largest value, or the nucleus's border, lies, and only
// that bin's values are ordered. For top-p the histogram's counts times the
// weight at a bin's middle give a guess, which one pass over the exact weights
// confirms (or widens). Bins that hold more than CAP values (long ties) are
// split again over (value, index). With top_k up to about a thousand the few
// candidates go to one CTA, which finishes the row.
//
// Bound by latency for one row (passes over shared memory and cluster
// barriers), by the f64 pipe where every weight is needed (top-p, min-p and
// plain sampling: eleven operations a value). Measured on B200: one row of
// 152064 f32 logits with top-k and top-p 14 us, with top-p alone 28 us, without
// either 11 us; 64 rows of 128256 bf16 logits with settings of their own 57 us,
// all with top-p 76 us: the rows run at once, two CTAs an SM (64 registers, 160
// bytes of spill stores), and the slowest one's chain of passes and cluster
// barriers counts.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <float.h>

#include <algorithm>
#include <type_traits>

#include "kv8.cuh"

namespace cg = cooperative_groups;

namespace sm {
namespace {

constexpr uint32_t THREADS = 512, WARPS = THREADS / 32;
constexpr uint32_t BINS = 2048;
constexpr uint32_t CAP = 1024;            // values ordered at once
constexpr double UNIT = 8796093022208.0;  // 2^43
constexpr double RANGE = 24.0;                // the histogram's: e^-24 of the largest weight, the last bin what is below
constexpr uint32_t MAX_CLUSTER = 16;
constexpr uint32_t MAX_PART = 78 * 1024;     // bytes of a row a CTA keeps: two fit an SM

// Order-preserving integer of a float, and a value's place in a row's order:
// larger = earlier (larger value, then lower index).
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); }
__device__ __forceinline__ uint64_t place(float x, uint32_t i) { return (uint64_t)ordered(x) << 32 | (uint32_t)~i; }

__device__ __forceinline__ float load_logit(float x) { return x; }
__device__ __forceinline__ float load_logit(__half x) { return __half2float(x); }
__device__ __forceinline__ float load_logit(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void store_logit(float x, float& o) { o = x; }
__device__ __forceinline__ void store_logit(float x, __half& o) { o = __float2half_rn(x); }
__device__ __forceinline__ void store_logit(float x, __nv_bfloat16& o) { o = __float2bfloat16_rn(x); }
template <typename T>
__device__ __forceinline__ float value(T x) { return fminf(load_logit(x), FLT_MAX); }  // +inf: the largest float

// What the CTAs of a cluster see of one another.
struct alignas(16) Shared {
  uint32_t count[BINS];
  uint64_t cand[CAP], sorted[CAP];  // places gathered by rank 0, and in order
  uint64_t weight[CAP];             // of the sorted ones
  double exp2_of[16];               // 2^(43 + j / 16)
  uint64_t warp64[WARPS], warp64b[WARPS];
  uint64_t post[10];                // what this CTA tells the others; no slot is written again before all have read it
  uint64_t cut;                     // rank 0's answer
  uint64_t found_run;
  double anchor;
  uint32_t n_cand, found[2], n_here, n_left, at_zero;
};

static_assert(sizeof(Shared) % 16 == 0, "the values behind it are read as float4");

// Sum over the CTA, in every thread. `tmp` may be reused after the next barrier.
__device__ uint64_t block_sum(uint64_t v, uint64_t* tmp) {
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) tmp[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (uint32_t i = 0; i < WARPS; i++) v += tmp[i];
  return v;
}
__device__ uint64_t block_max(uint64_t v, uint64_t* tmp) {
  for (int o = 16; o; o >>= 1) v = max(v, __shfl_xor_sync(~0u, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) tmp[threadIdx.x >> 5] = v;
  __syncthreads();
#pragma unroll
  for (uint32_t i = 0; i < WARPS; i++) v = max(v, tmp[i]);
  return v;
}
// Exclusive prefix over the CTA's threads, and the sum.
template <typename N>
__device__ N block_before(N v, uint64_t* tmp64, N* total) {
  N* tmp = reinterpret_cast<N*>(tmp64);
  const uint32_t lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  N x = v;
#pragma unroll
  for (uint32_t o = 1; o < 32; o <<= 1) {
    const N y = __shfl_up_sync(~0u, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) tmp[w] = x;
  __syncthreads();
  N before = 0, all = 0;
#pragma unroll
  for (uint32_t i = 0; i < WARPS; i++) {
    before += i < w ? tmp[i] : (N)0;
    all += tmp[i];
  }
  *total = all;
  return before + (x - v);
}

// Weights of a row: 2^43 exp((x - top) / T) = 2^(43 + y), y = (x - top) c, as integers.
// y = k / 16 + r, |r| <= 1/32: 2^(k/16) from a table and the exponent, 2^r by
// its Taylor polynomial of degree 5 (relative error (ln2 / 32)^6 / 720 < 2^-42).
// Sixteen doubles lie in different banks: no lookup conflicts.
struct Weights {
  const double* table;  // 2^(43 + j / 16)
  double c, top;
  float floor;  // values below it weigh nothing
  // A float in f64, by its bits (zero and subnormals come out as values below 2^-126: no weight changes by it while
  // c is below 2^81).
  static __device__ double wide(float x) {
    const uint32_t b = __float_as_uint(x);
    return __hiloint2double((int)((b & 0x80000000u) | (((b & 0x7FFFFFFFu) >> 3) + 0x38000000u)), (int)(b << 29));
  }
  __device__ uint64_t of(float x) const {
    const double y = (wide(fmaxf(x, floor)) - top) * c;
    constexpr double magic = 6755399441055744.0 / 16;  // 1.5 2^52 / 16: adding it rounds to a multiple of 1/16
    const double t = y + magic;
    const int k = __double2loint(t);
    const double r = y - (t - magic);
    constexpr double L = 0.69314718055994530942;
    double p = fma(r, L * L * L * L * L / 120, L * L * L * L / 24);
    p = fma(p, r, L * L * L / 6);
    p = fma(p, r, L * L / 2);
    p = fma(p, r, L);
    p = fma(p, r, 1.0);
    const double f = table[k & 15];
    const double scaled = __hiloint2double(__double2hiint(f) + (k >> 4 << 20), __double2loint(f));
    // adding 2^52 rounds to a whole number and leaves it in the low bits
    const uint64_t w = (uint64_t)__double_as_longlong(fma(scaled, p, 4503599627370496.0)) & 0xFFFFFFFFFFFFFull;
    return x >= floor ? w : 0;
  }
};

template <typename T>
__global__ void __launch_bounds__(THREADS, 2) draw_kernel(const DrawArgs a, uint32_t chunk) {
  extern __shared__ float4 draw_smem4[];
  Shared& sh = *reinterpret_cast<Shared*>(draw_smem4);
  T* vals = reinterpret_cast<T*>(&sh + 1);  // as they came (16-bit ones take half the room), the masked ones -inf
  cg::cluster_group cl = cg::this_cluster();
  const uint32_t CL = cl.num_blocks(), rank = cl.block_rank(), row = blockIdx.x / CL, tid = threadIdx.x;
  const uint32_t lane = tid & 31, V = a.vocab;
  const uint32_t begin = min(V, rank * chunk), n = min(V, begin + chunk) - begin;  // this CTA's part of the row
  auto peer = [&](uint32_t i) { return cl.map_shared_rank(&sh, i); };

  // ---- the part, into shared memory; the largest value, the lowest index among equals ----
  float mine_x = -INFINITY;  // this thread's largest
  uint32_t mine_i = 0;
  {
    const T* src = (const T*)a.logits + (uint64_t)row * a.ld + begin;
    const uint8_t* mk = a.mask ? a.mask + (uint64_t)row * a.ld + begin : nullptr;
    auto take = [&](uint32_t i, float x) {
      x = x > -INFINITY && (!mk || mk[i]) ? x + 0.f : -INFINITY;  // NaN, masked; -0 is 0
      store_logit(x, vals[i]);
      x = fminf(x, FLT_MAX);  // as `value` reads it
      if (x > mine_x) mine_x = x, mine_i = i;
    };
    constexpr uint32_t PER = 16 / sizeof(T), AHEAD = 5;  // 16-byte loads, five in flight
    const uint32_t nv = (uintptr_t)src % 16 == 0 ? n / PER : 0;
    for (uint32_t i = tid; i < nv; i += THREADS * AHEAD) {
      uint4 raw[AHEAD];
#pragma unroll
      for (uint32_t k = 0; k < AHEAD; k++)
        if (i + k * THREADS < nv) raw[k] = __ldcs(reinterpret_cast<const uint4*>(src) + i + k * THREADS);
#pragma unroll
      for (uint32_t k = 0; k < AHEAD; k++)
        if (i + k * THREADS < nv) {
#pragma unroll
          for (uint32_t j = 0; j < PER; j++) take((i + k * THREADS) * PER + j, load_logit(reinterpret_cast<const T*>(&raw[k])[j]));
        }
    }
    for (uint32_t i = nv * PER + tid; i < n; i += THREADS) take(i, load_logit(src[i]));
  }
  uint64_t best = mine_x > -INFINITY ? place(mine_x, begin + mine_i) : 0;
  for (uint32_t b = tid; b < BINS; b += THREADS) sh.count[b] = 0;
  if (tid < 16) sh.exp2_of[tid] = exp2(43.0 + tid / 16.0);
  best = block_max(best, sh.warp64);
  if (tid == 0) sh.post[0] = best, sh.n_cand = 0;
  const DrawParams p = a.params[row];
  float u = a.u[row];
  cl.sync();
  best = lane < CL ? peer(lane)->post[0] : 0;  // lane i asks CTA i
  for (int o = 16; o; o >>= 1) best = max(best, __shfl_xor_sync(~0u, best, o));
  if (best == 0 || !(p.temperature > 0.f)) {  // nothing to draw from, or greedy
    if (rank == 0 && tid == 0) {
      a.tokens[row] = best ? (int32_t)(uint32_t)~best : -1;
      if (a.logprobs) a.logprobs[row] = best ? 0.f : -INFINITY;
    }
    cl.sync();  // the others read post
    return;
  }
  float top = unordered((uint32_t)(best >> 32));
  double inv_t = 1.0 / (double)p.temperature;
  // At temperatures below 2^-80 zeros and subnormals differ from one another: row and temperature times 2^80, where
  // the largest value is tiny itself. (Else only its equals weigh anything; and f16 holds nothing so small.)
  if (sizeof(T) == 4 || std::is_same<T, __nv_bfloat16>::value) {
    constexpr float up = 1.2089258e24f, far = -1.7014118e38f;  // 2^80, -2^127
    if (p.temperature < 1.f / up && fabsf(top) < 9.0949470e-13f) {  // 2^-40
      for (uint32_t i = tid; i < n; i += THREADS) {
        const float x = load_logit(vals[i]);
        if (x > -INFINITY) store_logit(fmaxf(x * up, far), vals[i]);
      }
      if (mine_x > -INFINITY) mine_x = fmaxf(mine_x * up, far);
      top *= up, inv_t /= up;
      best = (uint64_t)ordered(top) << 32 | (uint32_t)best;
      __syncthreads();
    }
  }
  Weights wt;
  wt.table = sh.exp2_of;
  wt.c = inv_t * 1.4426950408889634074;
  wt.top = Weights::wide(top);
  wt.floor = (float)fmax((double)top - 60.0 / wt.c, -(double)FLT_MAX);  // 2^-60 of the largest
  u = u > 0.f ? fminf(u, 0.99999994f) : 0.f;
  // kept: weights of at least this
  const double min_w = fmin(ceil(fmax((double)p.min_p, 0.0) * UNIT), 1e18);
  const uint64_t min_weight = (uint64_t)min_w;
  auto finish = [&](uint32_t index, float x, uint64_t total) {
    a.tokens[row] = (int32_t)index;
    if (a.logprobs) a.logprobs[row] = (float)(((double)x - (double)top) * inv_t - log((double)total / UNIT));
  };
  // Where order counts a thread has consecutive values, an odd number of them (no bank conflicts).
  const uint32_t run_len = (n + THREADS - 1) / THREADS | 1, i0 = min(n, tid * run_len), i1 = min(n, i0 + run_len);
  // f(x, index in this CTA's part) for this thread's share of the values, -inf among them
  auto each = [&](auto f) {
    const uint32_t n4 = n / 4;
#pragma unroll 2
    for (uint32_t i = tid; i < n4; i += THREADS) {
      struct alignas(4 * sizeof(T)) Four { T x[4]; };
      const Four v = reinterpret_cast<const Four*>(vals)[i];
#pragma unroll
      for (int j = 0; j < 4; j++) f(value(v.x[j]), 4 * i + j);
    }
    if (4 * n4 + tid < n) f(value(vals[4 * n4 + tid]), 4 * n4 + tid);
  };
  // This CTA's sh.n_here places go behind those that rank 0's sh.cand holds; more than CAP are counted only.
  auto push = [&](const uint64_t* from) {
    __syncthreads();
    const uint32_t here = sh.n_here;
    Shared* zero = peer(0);
    if (tid == 0) sh.at_zero = here ? atomicAdd(&zero->n_cand, here) : 0;
    __syncthreads();
    const uint32_t base = sh.at_zero;
    for (uint32_t i = tid; i < min(here, CAP) && base + i < CAP; i += THREADS) zero->cand[base + i] = from[i];
  };
  // Rank 0's sh.cand and sh.n_cand get the places of the values that `in` picks, in any order: collected here
  // first (in sh.sorted), so that a CTA reserves its room at rank 0 once.
  auto gather = [&](auto in) {
    if (tid == 0) sh.n_here = 0;
    __syncthreads();
    each([&](float x, uint32_t i) {
      if (in(x, i)) {
        const uint32_t at = atomicAdd(&sh.n_here, 1u);
        if (at < CAP) sh.sorted[at] = place(x, begin + i);
      }
    });
    push(sh.sorted);
  };
  // The cluster's bins added up: thread t has bins [4t, 4t + 4). A CTA adds up a slice (its threads share
  // out the CTAs and four bins each) and gives it to all (sh.sorted).
  auto all_counts = [&](uint32_t (&c)[4]) {
    static_assert(BINS == 4 * THREADS && BINS * 4 == CAP * 8, "four bins a thread");
    const uint32_t per = THREADS / CL, from = tid / per, q = tid % per;
    uint4* part = reinterpret_cast<uint4*>(sh.weight);
    part[tid] = reinterpret_cast<const uint4*>(peer(from)->count)[rank * per + q];
    __syncthreads();
    uint4 v = make_uint4(0, 0, 0, 0);
    for (uint32_t i = 0; i < CL; i++) {
      const uint4 x = part[i * per + q];
      v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
    }
    reinterpret_cast<uint4*>(peer(from)->sorted)[rank * per + q] = v;
    cl.sync();
    v = reinterpret_cast<const uint4*>(sh.sorted)[tid];
    c[0] = v.x, c[1] = v.y, c[2] = v.z, c[3] = v.w;
    __syncthreads();
  };
  // All CTAs' post[slot] added up (lane i asks CTA i); `before`: those of the CTAs before this one.
  auto add_up = [&](uint32_t slot, uint64_t& before) -> uint64_t {
    uint64_t v = lane < CL ? peer(lane)->post[slot] : 0;
    before = lane < rank ? v : 0;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      v += __shfl_xor_sync(~0u, v, o);
      before += __shfl_xor_sync(~0u, before, o);
    }
    return v;
  };
  // Orders the n values of sh.cand, largest first, into sh.sorted: by counting
  // the larger ones while that is less work than a bitonic network.
  auto order = [&](uint32_t count) {
    __syncthreads();
    if (count <= 256) {  // two threads a value
      const uint32_t i = tid >> 1;
      if (i < (count + 15) / 16 * 16) {
        const uint64_t c = i < count ? sh.cand[i] : 0;
        uint32_t before = 0;
#pragma unroll 8
        for (uint32_t j = tid & 1; j < count; j += 2) before += sh.cand[j] > c;
        before += __shfl_xor_sync(~0u, before, 1);
        if (i < count && !(tid & 1)) sh.sorted[before] = c;
      }
    } else {
      uint32_t size = 512;
      while (size < count) size *= 2;
      for (uint32_t i = tid; i < size; i += THREADS) sh.sorted[i] = i < count ? sh.cand[i] : 0;
      __syncthreads();
      for (uint32_t len = 2; len <= size; len *= 2)
        for (uint32_t step = len / 2; step; step /= 2) {
          for (uint32_t i = tid; i < size / 2; i += THREADS) {
            const uint32_t x = (i & ~(step - 1)) * 2 + (i & (step - 1)), y = x + step;
            const uint64_t vx = sh.sorted[x], vy = sh.sorted[y];
            if ((vx < vy) == ((x & len) == 0)) sh.sorted[x] = vy, sh.sorted[y] = vx;
          }
          // pairs up to 32 apart lie in the 64 values of one warp
          if (step > 32 || (step == 1 && len >= 64)) __syncthreads(); else __syncwarp();
        }
    }
    __syncthreads();
  };

  const bool by_k = p.top_k > 0 && (uint32_t)p.top_k < V, by_p = p.top_p < 1.f;
  const float bin_scale = (float)fmin(BINS * inv_t / RANGE, (double)FLT_MAX);
  // Rank 0: the nucleus, min-p and the draw among the first `kept` of sh.sorted, the row's top_k.
  auto draw_sorted = [&](uint32_t kept) {
    constexpr uint32_t PER = CAP / THREADS;
    uint64_t w[PER], mine = 0, sum;
#pragma unroll
    for (uint32_t j = 0; j < PER; j++) {
      const uint32_t at = tid * PER + j;
      w[j] = at < kept ? wt.of(unordered((uint32_t)(sh.sorted[at] >> 32))) : 0;
      mine += w[j];
    }
    const uint64_t run0 = block_before(mine, sh.warp64, &sum);
    uint64_t run = run0, in = 0;
#pragma unroll
    for (uint32_t j = 0; j < PER; j++) {
      const uint32_t at = tid * PER + j;
      const bool keep = at < kept && (at == 0 || ((!by_p || (double)run < (double)p.top_p * (double)sum) && w[j] >= min_weight));
      in += keep;
      run += w[j];
      sh.weight[at] = keep ? w[j] : 0;
    }
    kept = (uint32_t)block_sum(in, sh.warp64b);  // a prefix
    uint64_t sum_kept = 0;
#pragma unroll
    for (uint32_t j = 0; j < PER; j++) sum_kept += sh.weight[tid * PER + j];
    sum_kept = block_sum(sum_kept, sh.warp64);
    const double aim = (double)u * (double)sum_kept;
    // the kept ones again, in the order of their indices
    for (uint32_t i = tid; i < kept; i += THREADS) sh.cand[i] = (uint64_t)(uint32_t)sh.sorted[i] << 32 | i;
    uint64_t keys[PER];
#pragma unroll
    for (uint32_t j = 0; j < PER; j++) keys[j] = tid + j * THREADS < kept ? sh.sorted[tid + j * THREADS] >> 32 : 0;
    order(kept);
#pragma unroll
    for (uint32_t j = 0; j < PER; j++)  // cand: the values, as they were sorted
      if (tid + j * THREADS < kept) sh.cand[tid + j * THREADS] = keys[j];
    __syncthreads();
    mine = 0;
#pragma unroll
    for (uint32_t j = 0; j < PER; j++) {
      const uint32_t at = tid * PER + j;
      w[j] = at < kept ? sh.weight[(uint32_t)sh.sorted[at]] : 0;
      mine += w[j];
    }
    run = block_before(mine, sh.warp64, &sum);
#pragma unroll
    for (uint32_t j = 0; j < PER; j++) {
      const uint32_t at = tid * PER + j;
      if (at < kept && (double)run <= aim && (double)(run + w[j]) > aim)
        finish(~(uint32_t)(sh.sorted[at] >> 32), unordered((uint32_t)sh.cand[(uint32_t)sh.sorted[at]]), sum_kept);
      run += w[j];
    }
  };
  // The bin of a value, in every pass alike: what overflows (or is 0 times infinity) lies in the last one. Masked
  // values fall there too; who looks at the last bin leaves them out.
  auto fast_bin = [&](float x) { return fminf((top - x) * bin_scale, (float)(BINS - 1)); };
  // Rank 0: of the `count` places in sh.cand the last, in order, before which less than `goal` lies (`run` in
  // the places before all of them): weights, or numbers of places. Bins over the candidates' own range leave
  // few of them; those are put in order.
  auto border_among = [&](uint32_t count, bool mass, uint64_t run, double goal) -> uint64_t {
    auto amount = [&](uint64_t pl) -> uint64_t { return mass ? wt.of(unordered((uint32_t)(pl >> 32))) : 1; };
    uint64_t* bins = sh.sorted;  // and sh.weight behind it
    static_assert(BINS == 2 * CAP && CAP == 2 * THREADS, "two candidates and four bins a thread");
    while (count > 256) {
      uint64_t pl[2];
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 2; j++) pl[j] = tid + j * THREADS < count ? sh.cand[tid + j * THREADS] : 0;
      const uint64_t hi = block_max(max(pl[0], pl[1]), sh.warp64);
      const uint64_t lo = ~block_max(max(pl[0] ? ~pl[0] : 0, pl[1] ? ~pl[1] : 0), sh.warp64b);
      const int bits = max(0, 53 - __clzll(hi - lo));  // (hi - lo) >> bits is below BINS, its half or more if bits > 0
#pragma unroll
      for (int j = 0; j < 4; j++) bins[tid + j * THREADS] = 0;
      if (tid == 0) sh.found[0] = 0, sh.n_left = 0;
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 2; j++)
        if (pl[j]) atomicAdd(reinterpret_cast<unsigned long long*>(&bins[(hi - pl[j]) >> bits]), (unsigned long long)amount(pl[j]));
      __syncthreads();
      uint64_t m[4], sum = 0, all;
#pragma unroll
      for (int j = 0; j < 4; j++) m[j] = bins[4 * tid + j], sum += m[j];
      uint64_t at = run + block_before(sum, sh.warp64, &all);
#pragma unroll
      for (int j = 0; j < 4; j++) {
        if (m[j] && (at == 0 || (double)at < goal) && !((double)(at + m[j]) < goal)) sh.found[0] = 4 * tid + j, sh.found_run = at;
        at += m[j];
      }
      __syncthreads();
      const uint32_t bin = sh.found[0];
      run = sh.found_run;
#pragma unroll
      for (int j = 0; j < 2; j++)
        if (pl[j] && (uint32_t)((hi - pl[j]) >> bits) == bin) sh.cand[atomicAdd(&sh.n_left, 1u)] = pl[j];
      __syncthreads();
      count = sh.n_left;
    }
    order(count);
    const uint64_t own = tid < count ? amount(sh.sorted[tid]) : 0;
    uint64_t all;
    const uint64_t at = run + block_before(own, sh.warp64, &all);
    const uint64_t kept = block_sum(tid < count && (tid == 0 || (double)at < goal), sh.warp64b);  // a prefix
    return sh.sorted[kept - 1];
  };

  uint64_t cut = 0;  // places >= cut are kept
  // The nucleus's border lay in a range of at most CAP places, which each CTA has in `local` (the bins are
  // done with then), and `mine` is the mass of this thread's consecutive values before that range.
  bool direct = false;
  uint64_t mine = 0;
  uint64_t* local = reinterpret_cast<uint64_t*>(sh.count);
  if (by_k && p.top_k <= (int32_t)CAP / 2) {
    // At least top_k of the row's values reach the top_k-th largest of the threads' maxima, and few others
    // do: a histogram of the maxima alone gives the bin down to which all values are gathered.
    if (mine_x > -INFINITY) atomicAdd(&sh.count[(uint32_t)fast_bin(mine_x)], 1u);
    if (tid == 0) sh.found[0] = ~0u;
    cl.sync();
    uint32_t c[4] = {}, all;
    all_counts(c);
    uint32_t before = block_before(c[0] + c[1] + c[2] + c[3], sh.warp64, &all);
#pragma unroll
    for (int j = 0; j < 4; j++) {
      if (before < (uint32_t)p.top_k && before + c[j] >= (uint32_t)p.top_k) sh.found[0] = 4 * tid + j;
      before += c[j];
    }
    __syncthreads();
    const uint32_t bin = sh.found[0];
    uint32_t gathered = CAP + 1;
    if (bin < BINS - 1) {
      const float behind = (float)(bin + 1);
      gather([&](float x, uint32_t) { return fast_bin(x) < behind; });
      cl.sync();
      gathered = peer(0)->n_cand;
    }
    if (gathered <= CAP) {
      cl.sync();  // the others have read it
      if (rank == 0) {
        order(gathered);
        draw_sorted(min(gathered, (uint32_t)p.top_k));
      }
      return;
    }
    cl.sync();  // the others have read the counts and n_cand
    for (uint32_t b = tid; b < BINS; b += THREADS) sh.count[b] = 0;
    if (tid == 0) sh.n_cand = 0;
  }
  for (int phase = 0; phase < 2; phase++) {
    // phase 0: the top_k-th place, by counts; phase 1: the nucleus's border, by mass among the places >= cut
    if (phase == 0 ? !by_k : !by_p) continue;
    const bool mass = phase == 1;
    uint64_t lo = cut, hi = best, above = 0;  // the border lies in [lo, hi]; count or mass over hi
    double goal = 0;
    uint32_t slot = 1;
    if (mass && by_k) {
      cl.sync();  // the others have read the counts of phase 0
      for (uint32_t b = tid; b < BINS; b += THREADS) sh.count[b] = 0;
    }
    for (int round = 0;; round++) {
      int bits = 0;
      if (round) while (((hi - lo) >> bits) >= BINS) bits++;
      auto bin_of = [&](float x, uint64_t pl) -> uint32_t {
        return round ? (uint32_t)((hi - pl) >> bits) : (uint32_t)fast_bin(x);
      };
      const bool everything = round == 0 && lo == 0;  // every value is in [lo, hi]: only its bin matters
      __syncthreads();
      if (everything) {
        each([&](float x, uint32_t) {
          if (x > -INFINITY) atomicAdd(&sh.count[(uint32_t)fast_bin(x)], 1u);
        });
      } else {
        each([&](float x, uint32_t i) {
          const uint64_t pl = place(x, begin + i);
          if (x > -INFINITY && pl >= lo && pl <= hi) atomicAdd(&sh.count[bin_of(x, pl)], 1u);
        });
      }
      cl.sync();
      uint32_t c[4] = {};
      all_counts(c);
      uint32_t c_total;
      const uint32_t c_before = block_before(c[0] + c[1] + c[2] + c[3], sh.warp64, &c_total);
      uint32_t bin_a = 0, bin_b = BINS - 1;  // the border lies in a bin from bin_a to bin_b
      uint64_t mass_above = 0;               // of the bins before bin_a
      uint64_t n_above, n_in;                // places in the bins before, and in them
      auto count_range = [&] {
        uint64_t ca = 0, ci = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const uint32_t b = 4 * tid + j;
          ca += b < bin_a ? c[j] : 0;
          ci += b >= bin_a && b <= bin_b ? c[j] : 0;
        }
        const uint64_t both = block_sum(ca << 32 | ci, sh.warp64);
        n_above = both >> 32, n_in = (uint32_t)both;
      };
      if (tid == 0) sh.found[0] = ~0u, sh.found[1] = ~0u;
      __syncthreads();
      if (!mass) {
        uint64_t run = above + c_before;
#pragma unroll
        for (int j = 0; j < 4; j++) {
          if (run < (uint64_t)p.top_k && run + c[j] >= (uint64_t)p.top_k) sh.found[0] = 4 * tid + j;
          run += c[j];
        }
        __syncthreads();
        bin_a = bin_b = sh.found[0];
        if (bin_a == ~0u) break;  // fewer places than top_k: all are kept
        count_range();
      } else {
        // The guess: counts times the weight at a bin's middle, within a margin.
        double m[4], sum = 0, all, var = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const uint64_t b = 4 * tid + j;
          const uint64_t mid = hi - min(hi - lo, (b << bits) + ((uint64_t)1 << bits) / 2);
          const float y = round ? (unordered((uint32_t)(mid >> 32)) - top) * (float)wt.c
                                : -((float)b + 0.5f) * (float)(RANGE / BINS * 1.4426950408889634);
          m[j] = c[j] ? (double)c[j] * (double)exp2f(y) : 0.0;
          sum += m[j];
          var += m[j] * m[j];
        }
        const double before_m = block_before(sum, sh.warp64b, &all);
        double var_all;
        block_before(var, sh.warp64, &var_all);
        // The bin in which the guessed sums pass `want` (sh.found[which]; ~0: none).
        auto guess = [&](double want, int which) {
          double run = before_m;
#pragma unroll
          for (int j = 0; j < 4; j++) {
            if (run < want && run + m[j] >= want) sh.found[which] = 4 * tid + j;
            run += m[j];
          }
        };
        // A bin's values are off its middle by RANGE / BINS / sqrt(12), all alike where they are few distinct
        // ones (16-bit logits). Errors of hundreds of bins cancel, and those before and behind the border partly
        // do: 0.4 of the standard deviation leaves a few bins, and held in every one of 480 simulated rows.
        const double want = round ? (goal - (double)above) / UNIT : (double)p.top_p * all;
        const double slack = 0.4 * RANGE / BINS / 3.46 * sqrt(var_all) + 3e-5 * all;
        guess(want - slack, 0);
        guess(want + slack, 1);
        __syncthreads();
        // Exact masses of a range of bins to try: it then holds the border, or what lies on one side of it does,
        // so the range that may hold it, [bin_a, bin_b], shrinks every turn. The first turn tries the guess, the
        // later ones a guess from the exact mass before bin_a, which is a few bins off at most. Where all values
        // are in [lo, hi] a thread looks at consecutive ones, as in the draw, keeps its mass before bin_a (`mine`)
        // and collects the range's places: the draw then needs no pass of its own.
        uint32_t try_a = sh.found[0] == ~0u ? 0 : sh.found[0], try_b = sh.found[1] == ~0u ? BINS - 1 : max(sh.found[1], try_a);
        mine = 0;
        for (int turn = 0;; turn++) {
          uint64_t ma = 0, mi = 0, ml = 0;  // in the bins from bin_a to try_a, of the range, behind it (first turn)
          if (everything) {
            const float f0 = (float)bin_a, fa = (float)try_a, fb = try_b == BINS - 1 ? INFINITY : (float)(try_b + 1);
            if (tid == 0) sh.n_here = 0;
            __syncthreads();
            auto collect = [&](float x, uint32_t i) {
              const uint32_t at = atomicAdd(&sh.n_here, 1u);
              if (at < CAP) local[at] = place(x, begin + i);
            };
            if (!turn) {
              for (uint32_t i = i0; i < i1; i += 4) {
                float x[4];
                uint64_t w[4];
#pragma unroll
                for (int j = 0; j < 4; j++) x[j] = i + j < i1 ? value(vals[i + j]) : -INFINITY;
#pragma unroll
                for (int j = 0; j < 4; j++) w[j] = wt.of(x[j]);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                  const float b = fast_bin(x[j]);
                  ml += w[j];
                  ma += b < fa ? w[j] : 0;
                  if (b >= fa && b < fb && x[j] > -INFINITY) {
                    mi += w[j];
                    collect(x[j], i + j);
                  }
                }
              }
              ml -= ma + mi;
            } else {
#pragma unroll 4
              for (uint32_t i = i0; i < i1; i++) {
                const float x = value(vals[i]), b = fast_bin(x);
                if (!(b >= f0 && b < fb && x > -INFINITY)) continue;
                const uint64_t w = wt.of(x);
                if (b < fa) {
                  ma += w;
                } else {
                  mi += w;
                  collect(x, i);
                }
              }
            }
          } else {
            each([&](float x, uint32_t i) {
              const uint64_t pl = place(x, begin + i);
              if (!(x > -INFINITY) || pl < lo || pl > hi) return;
              const uint32_t b = bin_of(x, pl);
              if (b < bin_a || (b > try_b && (round || turn))) return;
              const uint64_t w = wt.of(x);
              if (b < try_a) ma += w;
              else if (b <= try_b) mi += w;
              else ml += w;
            });
          }
          const uint64_t ma_here = ma, mi_here = mi;
          ma = block_sum(ma, sh.warp64);
          mi = block_sum(mi, sh.warp64b);
          ml = block_sum(ml, sh.warp64);
          slot ^= 5;  // 1 and 4 in turn
          if (tid == 0) sh.post[slot] = ma, sh.post[slot + 1] = mi, sh.post[slot + 2] = ml;
          cl.sync();
          uint64_t unused;
          ma = mass_above + add_up(slot, unused), mi = add_up(slot + 1, unused), ml = add_up(slot + 2, unused);
          if (!round && !turn) goal = (double)p.top_p * (double)(ma + mi + ml);
          const bool begins = try_a == bin_a || above + ma == 0 || (double)(above + ma) < goal;
          const bool ends = try_b == bin_b || (double)(above + ma + mi) >= goal;
          if (begins && ends) {
            bin_a = try_a, bin_b = try_b, mass_above = ma;
            mine += ma_here;
          } else if (!begins) {
            bin_b = try_a - 1;
          } else {
            bin_a = try_b + 1, mass_above = ma + mi;
            mine += ma_here + mi_here;
          }
          count_range();
          direct = everything && begins && ends && n_in <= CAP;
          if (direct || (!everything && n_in <= CAP) || (bin_a == bin_b && n_in > CAP)) break;
          // the next range: all that is left, if that is few; else the bin of the new guess and its neighbours
          try_a = bin_a, try_b = bin_b;
          if (n_in <= CAP) continue;
          if (tid == 0) sh.found[0] = (bin_a + bin_b) / 2;
          __syncthreads();
          if (4 * tid <= bin_a && bin_a < 4 * tid + 4) {
            double run = before_m;
#pragma unroll
            for (int j = 0; j < 4; j++) run += 4 * tid + j < bin_a ? m[j] : 0.0;
            sh.anchor = run;
          }
          __syncthreads();
          guess(sh.anchor + (goal - (double)above - (double)mass_above) / UNIT, 0);
          __syncthreads();
          const uint32_t t = min(max(sh.found[0], bin_a), bin_b);
          __syncthreads();
          if (bin_b - bin_a > 2) try_a = max(bin_a, t ? t - 1 : 0), try_b = min(bin_b, t + 1);
          else try_a = try_b = t;
        }
      }
      const bool small = !mass && round == 0 && n_above + n_in <= CAP;  // all the top_k at once
      if (small) {
        bin_a = 0;
        n_in += n_above, n_above = 0;
      }
      if (n_in <= CAP) {
        const float fa = (float)bin_a, fb = bin_b == BINS - 1 ? INFINITY : (float)(bin_b + 1);
        if (direct) {
          push(local);
        } else if (everything) {
          gather([&](float x, uint32_t) { return x > -INFINITY && fast_bin(x) >= fa && fast_bin(x) < fb; });
        } else {
          gather([&](float x, uint32_t i) {
            const uint64_t pl = place(x, begin + i);
            if (!(x > -INFINITY) || pl < lo || pl > hi) return false;
            const uint32_t b = bin_of(x, pl);
            return b >= bin_a && b <= bin_b;
          });
        }
        cl.sync();
        if (small && rank != 0) return;
        if (rank == 0) {
          const uint32_t held = min(sh.n_cand, CAP);  // n_in, as both went by the same bins
          if (small) {
            order(held);
            draw_sorted(min(held, (uint32_t)p.top_k));
            return;
          }
          const uint64_t border = border_among(held, mass, above + (mass ? mass_above : n_above), mass ? goal : (double)p.top_k);
          if (tid == 0) sh.cut = border, sh.n_cand = 0;
        }
        cl.sync();
        cut = peer(0)->cut;
        break;
      }
      // too many: narrow [lo, hi] to what the range holds
      uint64_t mn = ~0ull, mx = 0;
      each([&](float x, uint32_t i) {
        const uint64_t pl = place(x, begin + i);
        if (!(x > -INFINITY) || pl < lo || pl > hi) return;
        const uint32_t b = bin_of(x, pl);
        if (b >= bin_a && b <= bin_b) mn = min(mn, pl), mx = max(mx, pl);
      });
      mx = block_max(mx, sh.warp64);
      mn = ~block_max(~mn, sh.warp64b);
      cl.sync();  // the others have read counts and post
      for (uint32_t b = tid; b < BINS; b += THREADS) sh.count[b] = 0;
      if (tid == 0) sh.post[7] = mn, sh.post[8] = mx;
      cl.sync();
      for (uint32_t i = 0; i < CL; i++) mn = min(mn, peer(i)->post[7]), mx = max(mx, peer(i)->post[8]);
      lo = mn, hi = mx;
      above += mass ? mass_above : n_above;
    }
  }

  // ---- the draw, in the vocabulary's order ----
  const float cut_x = cut ? unordered((uint32_t)(cut >> 32)) : -INFINITY;
  const uint32_t cut_i = ~(uint32_t)cut - begin, best_i = ~(uint32_t)best - begin;  // modulo 2^32, as begin + i is
  auto weight_at = [&](uint32_t i) -> uint64_t {  // 0: not kept
    const float x = value(vals[i]);
    const uint64_t w = wt.of(x);
    const bool in = x > cut_x || (x == cut_x && begin + i <= cut_i + begin);
    return in && (w >= min_weight || i == best_i) ? w : 0;
  };
  if (direct && min_weight == 0) {
    // the search's sums: the values before its range, and of the range those kept
    uint64_t* extra = sh.weight;
    extra[tid] = 0;
    __syncthreads();
    for (uint32_t i = tid; i < sh.n_here; i += THREADS) {
      const uint64_t pl = local[i];
      if (pl >= cut)
        atomicAdd(reinterpret_cast<unsigned long long*>(&extra[(~(uint32_t)pl - begin) / run_len]),
                  (unsigned long long)wt.of(unordered((uint32_t)(pl >> 32))));
    }
    __syncthreads();
    mine += extra[tid];
  } else {
    mine = 0;
#pragma unroll 4
    for (uint32_t i = i0; i < i1; i++) mine += weight_at(i);
  }
  uint64_t cta;
  uint64_t run = block_before(mine, sh.warp64, &cta);
  if (tid == 0) sh.post[9] = cta;
  cl.sync();
  uint64_t before_me;
  const uint64_t total = add_up(9, before_me);
  run += before_me;
  cl.sync();  // the others read post
  const double aim = (double)u * (double)total;
  // one thread of the cluster holds the value at which the sum passes the aim; its warp looks for it
  const uint32_t who = __ballot_sync(~0u, (double)run <= aim && (double)(run + mine) > aim);
  if (who) {
    const uint32_t owner = __ffs(who) - 1;
    run = __shfl_sync(~0u, run, owner);
    const uint32_t j0 = __shfl_sync(~0u, i0, owner), j1 = __shfl_sync(~0u, i1, owner);
    for (uint32_t i = j0; i < j1; i += 32) {
      const uint64_t w = i + lane < j1 ? weight_at(i + lane) : 0;
      uint64_t upto = w;
#pragma unroll
      for (uint32_t o = 1; o < 32; o <<= 1) {
        const uint64_t y = __shfl_up_sync(~0u, upto, o);
        if (lane >= o) upto += y;
      }
      upto += run;
      if (w && (double)upto > aim && (double)(upto - w) <= aim) finish(begin + i + lane, value(vals[i + lane]), total);
      run = __shfl_sync(~0u, upto, 31);
    }
  }
}

template <typename T>
cudaError_t draw_typed(const DrawArgs& a, uint32_t sms, cudaStream_t st) {
  // CTAs a row: as many as let all rows run at once (two CTAs an SM); at least
  // what the row needs of shared memory, at most what leaves a CTA 2048 values.
  uint32_t cl = 1;
  while (cl < MAX_CLUSTER && ((uint64_t)a.vocab * sizeof(T) > (uint64_t)cl * MAX_PART || ((uint64_t)a.n_rows * cl * (cl < 8 ? 1 : 4) <= sms && a.vocab / (cl * 2) >= 2048)))
    cl *= 2;
  const uint32_t chunk = ((a.vocab + cl - 1) / cl + 7) / 8 * 8;
  const size_t smem = sizeof(Shared) + (size_t)chunk * sizeof(T);
  auto* kern = draw_kernel<T>;
  static SmemOnce once;
  cudaError_t e = once.allow((const void*)kern, (int)(sizeof(Shared) + 2 * MAX_PART + 64));
  if (e == cudaSuccess && cl > 8) e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(a.n_rows * cl);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cl, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, a, chunk);
}

}  // namespace

cudaError_t launch_draw(const DrawArgs& a, uint32_t sms, cudaStream_t st) {
  if (!a.n_rows) return cudaSuccess;
  switch (a.type) {
    case ACT_F32: return draw_typed<float>(a, sms, st);
    case ACT_F16: return draw_typed<__half>(a, sms, st);
    default: return draw_typed<__nv_bfloat16>(a, sms, st);
  }
}

}  // namespace sm
