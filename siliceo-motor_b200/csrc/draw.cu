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
// weights are 64-bit fixed-point numbers (2^-43; the exponential is evaluated
// in f64): their sums are exact, whatever the order, and the atomics of a
// histogram cannot change a draw.
//
// A cluster of CTAs holds a row in shared memory and reads it once. The k-th
// largest value and the nucleus's border are found without sorting the row: a
// histogram over the distance from the maximum, then an exact sort of the one
// bin the border lies in (or finer histograms while that bin holds too many).
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <float.h>

#include <algorithm>

#include "kv8.cuh"

namespace cg = cooperative_groups;

namespace sm {
namespace {

constexpr uint32_t THREADS = 512;
constexpr uint32_t BINS = 2048;
constexpr uint32_t CAP = 1024;    // candidates sorted at once
constexpr double UNIT = 8796093022208.0;  // 2^43
constexpr uint32_t MAX_CLUSTER = 16;

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

struct Shared {
  uint32_t count[BINS];
  uint64_t mass[BINS];
  uint64_t cand[CAP];     // gathered places (rank 0's), then sorted
  uint64_t sorted[CAP];
  uint64_t warp64[THREADS / 32], warp64b[THREADS / 32];
  uint64_t post[4];       // what this CTA tells the cluster
  uint64_t got[4];        // what the cluster found
  uint32_t n_cand;
};

__device__ uint64_t block_sum(uint64_t v, uint64_t* tmp) {
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) tmp[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0;
  for (uint32_t i = 0; i < THREADS / 32; i++) v += tmp[i];
  return v;
}
// Exclusive prefix of v over the CTA's threads.
__device__ uint64_t block_before(uint64_t v, uint64_t* tmp, uint64_t* total) {
  const uint32_t lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  uint64_t x = v;
  for (uint32_t o = 1; o < 32; o <<= 1) {
    const uint64_t y = __shfl_up_sync(~0u, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) tmp[w] = x;
  __syncthreads();
  uint64_t before = 0, all = 0;
  for (uint32_t i = 0; i < THREADS / 32; i++) {
    before += i < w ? tmp[i] : 0;
    all += tmp[i];
  }
  *total = all;
  return before + x - v;
}
__device__ uint64_t block_max(uint64_t v, uint64_t* tmp) {
  for (int o = 16; o; o >>= 1) v = max(v, __shfl_xor_sync(~0u, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) tmp[threadIdx.x >> 5] = v;
  __syncthreads();
  for (uint32_t i = 0; i < THREADS / 32; i++) v = max(v, tmp[i]);
  return v;
}

struct Row {
  const float* x;        // this CTA's values in shared memory
  uint32_t n, begin;     // how many, and the first's index
  uint32_t each;         // consecutive values of a thread (odd: no bank conflicts)
  float top;             // the row's maximum
  double inv_t;
  __device__ double w(float v) const { return exp(((double)v - (double)top) * inv_t); }
  __device__ uint64_t fixed(float v) const { return (uint64_t)(w(v) * UNIT + 0.5); }
};

template <typename T>
__global__ void __launch_bounds__(THREADS) draw_kernel(const DrawArgs a, uint32_t chunk) {
  extern __shared__ float4 draw_smem4[];
  Shared& sh = *reinterpret_cast<Shared*>(draw_smem4);
  float* vals = reinterpret_cast<float*>(&sh + 1);
  cg::cluster_group cl = cg::this_cluster();
  const uint32_t CL = cl.num_blocks(), rank = cl.block_rank(), row = blockIdx.x / CL, tid = threadIdx.x;
  const uint32_t V = a.vocab;
  Row r;
  r.begin = min(V, rank * chunk);
  r.n = min(V, r.begin + chunk) - r.begin;
  r.each = (r.n + THREADS - 1) / THREADS | 1;
  r.x = vals;

  // ---- the row's part, into shared memory; its largest ----
  uint64_t best = 0;
  {
    const T* src = (const T*)a.logits + (uint64_t)row * a.ld + r.begin;
    const uint8_t* mk = a.mask ? a.mask + (uint64_t)row * a.ld + r.begin : nullptr;
    for (uint32_t i = tid; i < r.n; i += THREADS) {
      float x = load_logit(src[i]);
      if (!(x > -INFINITY) || (mk && !mk[i])) x = -INFINITY;  // NaN, masked
      x = fminf(x, FLT_MAX) + 0.f;                            // and -0 is 0
      vals[i] = x;
      if (x > -INFINITY) best = max(best, place(x, r.begin + i));
    }
  }
  best = block_max(best, sh.warp64);
  if (tid == 0) sh.post[0] = best, sh.n_cand = 0, sh.got[0] = 0;
  cl.sync();
  for (uint32_t i = 0; i < CL; i++) best = max(best, cl.map_shared_rank(&sh, i)->post[0]);
  const DrawParams p = a.params[row];
  const bool sampled = p.temperature > 0.f;
  if (best == 0 || !sampled) {  // nothing to draw from, or greedy
    if (rank == 0 && tid == 0) {
      a.tokens[row] = best ? (int32_t)(uint32_t)~best : -1;
      if (a.logprobs) a.logprobs[row] = best ? 0.f : -INFINITY;
    }
    cl.sync();  // post is read above
    return;
  }
  r.top = unordered((uint32_t)(best >> 32));
  r.inv_t = 1.0 / (double)p.temperature;
  const uint32_t i0 = min(r.n, tid * r.each), i1 = min(r.n, i0 + r.each);
  float uu = a.u[row];
  uu = uu > 0.f ? fminf(uu, 0.99999994f) : 0.f;
  const double min_p = p.min_p;
  auto peer = [&](uint32_t i) { return cl.map_shared_rank(&sh, i); };

  // One round of the search for a border among the places in [lo, hi]. By
  // count: the border is the `goal`-th largest place. By mass: the place whose
  // preceding mass is still below `goal` of `mass_all`, the last such. `above`
  // is the count (or mass) of the places over hi. First round: bins over the
  // distance from the maximum; later ones over [lo, hi] itself. Leaves in
  // sh.got: {first place of the bin's values as the caller narrows it, bin, above, number in the bin}.
  uint64_t cut = 0;  // places >= cut are kept
  const bool by_k = p.top_k > 0 && (uint32_t)p.top_k < V, by_p = p.top_p < 1.f;
  const float bin_scale = (float)fmin(BINS * r.inv_t / 24.0, (double)FLT_MAX);

  for (int phase = 0; phase < 2; phase++) {
    // phase 0: top-k by counts; phase 1: top-p by mass among the places >= cut
    if (phase == 0 ? !by_k : !by_p) continue;
    const bool mass = phase == 1;
    uint64_t lo = cut, hi = best, above = 0, all = 0;
    for (int round = 0;; round++) {
      int sh_bits = 0;
      if (round) while (((hi - lo) >> sh_bits) >= BINS) sh_bits++;
      auto bin_of = [&](float x, uint64_t pl) -> uint32_t {
        return round ? (uint32_t)((hi - pl) >> sh_bits) : min(BINS - 1, (uint32_t)fminf((r.top - x) * bin_scale, 4e9f));
      };
      for (uint32_t b = tid; b < BINS; b += THREADS) sh.count[b] = 0, sh.mass[b] = 0;
      __syncthreads();
      for (uint32_t i = i0; i < i1; i++) {
        const float x = vals[i];
        const uint64_t pl = place(x, r.begin + i);
        if (x == -INFINITY || pl < lo || pl > hi) continue;
        const uint32_t b = bin_of(x, pl);
        atomicAdd(&sh.count[b], 1u);
        if (mass) atomicAdd(reinterpret_cast<unsigned long long*>(&sh.mass[b]), (unsigned long long)r.fixed(x));
      }
      cl.sync();
      // this CTA adds up the cluster's bins [b0, b0 + per)
      const uint32_t per = BINS / CL, b0 = rank * per;
      uint64_t c_mine = 0, m_mine = 0;  // of this thread's bins: consecutive ones
      const uint32_t tper = (per + THREADS - 1) / THREADS, t0 = min(per, tid * tper), t1 = min(per, t0 + tper);
      uint64_t cs[4] = {}, ms[4] = {};  // BINS / THREADS at most
      for (uint32_t b = t0; b < t1; b++) {
        for (uint32_t i = 0; i < CL; i++) {
          cs[b - t0] += peer(i)->count[b0 + b];
          if (mass) ms[b - t0] += peer(i)->mass[b0 + b];
        }
        c_mine += cs[b - t0], m_mine += ms[b - t0];
      }
      uint64_t c_total, m_total;
      const uint64_t c_before = block_before(c_mine, sh.warp64, &c_total);
      const uint64_t m_before = block_before(m_mine, sh.warp64b, &m_total);
      if (tid == 0) sh.post[1] = c_total, sh.post[2] = m_total;
      cl.sync();
      uint64_t c_run = mass ? 0 : above, m_run = above, m_all = 0;
      for (uint32_t i = 0; i < CL; i++) {
        if (i < rank) c_run += peer(i)->post[1], m_run += peer(i)->post[2];
        m_all += peer(i)->post[2];
      }
      if (mass && !round) all = m_all;
      c_run += c_before, m_run += m_before;
      const double goal = (double)p.top_p * (double)all;
      // the bin with the border: the last whose values begin before the goal
      for (uint32_t b = t0; b < t1; b++) {
        const uint64_t c = cs[b - t0], m = ms[b - t0];
        const bool here = c && (mass ? m_run == 0 || (double)m_run < goal : c_run < (uint64_t)p.top_k);
        const bool next = mass ? (double)(m_run + m) < goal : c_run + c < (uint64_t)p.top_k;
        // the goal lies in this bin, or behind all of them
        if (here && !next)
          for (uint32_t i = 0; i < CL; i++) {
            peer(i)->got[0] = 1, peer(i)->got[1] = b0 + b;
            peer(i)->got[2] = mass ? m_run : c_run, peer(i)->got[3] = c;
          }
        c_run += c, m_run += m;
      }
      cl.sync();
      const bool found = sh.got[0];
      const uint32_t bin = (uint32_t)sh.got[1];
      const uint64_t found_above = sh.got[2];
      const uint32_t n_in = (uint32_t)sh.got[3];
      __syncthreads();
      if (tid == 0) sh.got[0] = 0;
      if (!found) break;  // fewer values than top_k, or a top_p their sum does not reach: all are kept
      above = found_above;
      if (n_in <= CAP) {
        Shared* zero = peer(0);
        for (uint32_t i = i0; i < i1; i++) {
          const float x = vals[i];
          const uint64_t pl = place(x, r.begin + i);
          if (x == -INFINITY || pl < lo || pl > hi || bin_of(x, pl) != bin) continue;
          zero->cand[atomicAdd(&zero->n_cand, 1u)] = pl;
        }
        cl.sync();
        if (rank == 0) {
          for (uint32_t i = tid; i < n_in; i += THREADS) {  // rank each, by counting
            const uint64_t c = sh.cand[i];
            uint32_t before = 0;
            for (uint32_t j = 0; j < n_in; j++) before += sh.cand[j] > c;
            sh.sorted[before] = c;
          }
          if (tid == 0) sh.n_cand = 0;
          __syncthreads();
          uint64_t border = 0;
          if (!mass) {
            border = sh.sorted[p.top_k - 1 - above];
          } else {
            uint64_t mine = 0, total;
            const uint32_t j0 = tid * (CAP / THREADS), j1 = min(n_in, j0 + CAP / THREADS);
            for (uint32_t j = j0; j < j1; j++) mine += r.fixed(unordered((uint32_t)(sh.sorted[j] >> 32)));
            uint64_t run = above + block_before(mine, sh.warp64, &total);
            uint64_t keep = ~0ull;  // the smallest place whose preceding mass is below the goal
            for (uint32_t j = j0; j < j1; j++) {
              if (run == 0 || (double)run < goal) keep = sh.sorted[j];
              run += r.fixed(unordered((uint32_t)(sh.sorted[j] >> 32)));
            }
            border = ~block_max(~keep, sh.warp64);
          }
          __syncthreads();
          if (tid < CL) peer(tid)->got[1] = border;
        }
        cl.sync();
        cut = sh.got[1];
        break;
      }
      // too many in the bin: narrow [lo, hi] to what it holds
      uint64_t mn = ~0ull, mx = 0;
      for (uint32_t i = i0; i < i1; i++) {
        const float x = vals[i];
        const uint64_t pl = place(x, r.begin + i);
        if (x == -INFINITY || pl < lo || pl > hi || bin_of(x, pl) != bin) continue;
        mn = min(mn, pl), mx = max(mx, pl);
      }
      mx = block_max(mx, sh.warp64);
      mn = ~block_max(~mn, sh.warp64b);
      if (tid == 0) sh.post[1] = mn, sh.post[2] = mx;
      cl.sync();
      for (uint32_t i = 0; i < CL; i++) mn = min(mn, peer(i)->post[1]), mx = max(mx, peer(i)->post[2]);
      lo = mn, hi = mx;
      cl.sync();
    }
  }

  // ---- the draw, in the vocabulary's order ----
  auto kept = [&](float x, uint32_t i, double w) {
    const uint64_t pl = place(x, i);
    return x > -INFINITY && pl >= cut && (w >= min_p || pl == best);
  };
  uint64_t mine = 0;
  for (uint32_t i = i0; i < i1; i++) {
    const float x = vals[i];
    if (x == -INFINITY || place(x, r.begin + i) < cut) continue;
    const double w = r.w(x);
    if (kept(x, r.begin + i, w)) mine += (uint64_t)(w * UNIT + 0.5);
  }
  uint64_t cta_total;
  const uint64_t before = block_before(mine, sh.warp64, &cta_total);
  if (tid == 0) sh.post[3] = cta_total;
  cl.sync();
  uint64_t run = before, total = 0;
  for (uint32_t i = 0; i < CL; i++) {
    const uint64_t m = peer(i)->post[3];
    if (i < rank) run += m;
    total += m;
  }
  const double goal = (double)uu * (double)total;
  // one thread of the cluster holds the value at which the sum passes the goal
  if (mine && (double)run <= goal && (double)(run + mine) > goal) {
    for (uint32_t i = i0; i < i1; i++) {
      const float x = vals[i];
      if (x == -INFINITY || place(x, r.begin + i) < cut) continue;
      const double w = r.w(x);
      if (!kept(x, r.begin + i, w)) continue;
      const uint64_t f = (uint64_t)(w * UNIT + 0.5);
      if ((double)run <= goal && (double)(run + f) > goal) {
        a.tokens[row] = (int32_t)(r.begin + i);
        if (a.logprobs) a.logprobs[row] = (float)(((double)x - (double)r.top) * r.inv_t - log((double)total / UNIT));
      }
      run += f;
    }
  }
  cl.sync();  // post is read above
}

template <typename T>
cudaError_t draw_typed(const DrawArgs& a, cudaStream_t st) {
  uint32_t cl = 8;
  while ((a.vocab + cl - 1) / cl > 40 * 1024 && cl < MAX_CLUSTER) cl *= 2;
  while (cl > 1 && a.vocab / cl < 2048) cl /= 2;
  const uint32_t chunk = ((a.vocab + cl - 1) / cl + 7) / 8 * 8;
  const size_t smem = sizeof(Shared) + (size_t)chunk * 4;
  auto* kern = draw_kernel<T>;
  static SmemOnce once;
  cudaError_t e = once.allow((const void*)kern, (int)(sizeof(Shared) + 40 * 1024 * 4 + 64));
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

cudaError_t launch_draw(const DrawArgs& a, cudaStream_t st) {
  if (!a.n_rows) return cudaSuccess;
  switch (a.type) {
    case ACT_F32: return draw_typed<float>(a, st);
    case ACT_F16: return draw_typed<__half>(a, st);
    default: return draw_typed<__nv_bfloat16>(a, st);
  }
}

}  // namespace sm
