// Attention over the 8-bit paged KV cache, streaming form (few rows a
// sequence): decoding and short chunks. kv8_attn_*.cu instantiate it.
//
//   o = sum_j p_j s_v(j) V_j / sum_j p_j,   p_j = exp(scale s_k(j) q.K_j)
//
// over the positions j a row sees; K_j, V_j are codes, s_k, s_v the scales of
// j's page. One pass with a running maximum m of t_j + e_j, where
// t_j = log2 p_j and e_j = exponent of s_v(j): the weights of the products,
// w_j = 2^(t_j + e_j - m + 13), are then relative to the largest
// *contribution* and fit f16 whatever the spread of the pages' scales, while
// the denominator adds 2^(t_j - m + 38) in f32. m is kept a whole number, so
// moving it multiplies by a power of two and rounds nothing. e_j is held to
// -60 .. 127: smaller scales' weights come out smaller instead. m is then at
// most 128 above the largest t_j and at most 60 below it: the denominator's
// terms and sums stay in f32's range (2^28 positions above, 2^-25 of the largest
// term below). Both come from one exponential, 2^(t_j + g_j - m) with
// g_j = max(e_j, 27): it is at most 2^87, and nothing of weight in the
// denominator underflows however large another page's e is. Factors between
// two maxima may be below 2^-126 and still count there (scaled).
//
// Bound by the cache bytes (2 hd a position and head): a warp copies a page at
// a time into shared memory of its own, the next page's K under this page's
// weights and products, its V under the next scores, and computes
// with mma.m16n8k16 in the transposed sense, S^T = K Q^T and O^T = V^T P^T,
// because the few rows of a unit (8, or 16) then are the narrow side n and
// nothing of the MMA is idle. K is the A operand: lane (g, t) holds 16
// consecutive dims of positions g, g + 8, ..., which serve four k-steps whose k
// order is permuted alike in Q's fragments. The weights leave S^T's
// accumulators through movmatrix as P^T's B fragments. V^T is an A operand
// too: lane (g, t) holds dims [16g, 16g + 16) of positions 2t, 2t + 1, 2t + 8,
// 2t + 9, ... and interleaves their bytes in pairs. The codes are exact in f16.
//
// Rows are (token, head of the group) pairs of one sequence and KV head. f32
// rows enter as high and low f16 halves (q and w), two MMAs each: scores and
// products keep 22 bits.
//
// Work is the list of all pages of all (sequence, row block, KV head) units
// laid end to end; every warp takes an equal share, whatever the lengths are,
// which only the device knows. A unit cut between warps of a CTA is merged in
// shared memory, one cut between CTAs by the last of them to arrive.
//
// Measured on B200 (GPU time, launches back to back): 4 sequences of up to
// 131072 positions, 28/4 heads of 128, bf16 rows, int8 codes: 80 us for 422 MB
// (5.3 TB/s, 0.81 of the measured 6515 GB/s); 32 sequences of up to 4096, 32/8
// heads: 47 us for 204 MB. The difference of the two is 6.4 TB/s, what is left
// is about 15 us a launch: 3 us to the first copies, 2 to 5 to the first codes,
// 5 to 9 of merging and of SMs that finish at different times. Row blocks of
// up to 8 rows keep 16 warps an SM (128 registers); 16 rows 12 warps. Some of
// the state spills: 32 bytes a thread with 8 rows, 132 with 16, 92 for f32 rows
// (head_dim 128; 39 and 262 local loads a scheduler in a launch). Without
// the exchanged columns, copies by the lanes' own fragments took 12 shared
// memory cycles more a page than the HBM time of the page.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "kv8.cuh"

namespace sm {
namespace {

constexpr uint32_t TILE = KV8_PAGE;  // positions of a step
constexpr int32_t FOLD_FROM = 1024;  // pages of a unit that one warp adds up
constexpr int32_t FOLD = 64;         // pages whose products the tensor core adds up before they are added in f32
constexpr int32_t SHORT = 4;         // pages of a unit that is never cut: a merge would cost more
constexpr float MINM = -3e38f;       // running maximum of a row that has seen nothing

// Shape of a kernel. HD: head dims, at run time at most HDV. NR: rows of a unit.
template <typename T, uint32_t HDV, uint32_t NR>
struct Shape {
  static constexpr bool SPLIT = sizeof(T) == 4;
  static constexpr uint32_t WARPS = NR == 8 ? (SPLIT && HDV > 64 ? 12 : 16) : (HDV > 64 ? 12 : 16);
  static constexpr uint32_t VALUES = TILE * HDV, SCALES = 2 * VALUES;  // a page: K's codes, V's, then the scales
  static constexpr uint32_t STAGE = SCALES + 128;
  // Byte offset of 16-byte column c of row r. The columns of each 128 bytes are exchanged by the row, so that
  // the 8 lanes of a shared-memory phase, (g, t) with two g for K and with four rows 2t for V, meet 8 of them.
  static __device__ uint32_t at(uint32_t r, uint32_t c) {
    if (HDV == 128) return r * 128 + ((c ^ ((r >> 1 & 3) << 1) ^ ((r & 1) << 2)) << 4);
    return (r >> 1) * 128 + ((((r & 1) << 2 | c) ^ ((r >> 1 & 3) << 1)) << 4);
  }
  // The same for the accesses of a lane, from its first offset `base`: all others are constants away, with the
  // column's bit 2 flipped (64 bytes; areas begin at multiples of 128) or not.
  static __device__ uint32_t copy_at(uint32_t base, uint32_t i) { return (HDV == 128 && (i & 1) ? base ^ 64 : base) + i * 512; }
  static __device__ uint32_t k_at(uint32_t base, uint32_t n, uint32_t sg) { return (sg ? base ^ 64 : base) + n * 8 * HDV; }
  static __device__ uint32_t v_at(uint32_t base, uint32_t half, uint32_t i) {
    return (i & 1 ? base ^ 64 : base) + half * 16 * HDV + (i >> 1) * 8 * HDV + (HDV == 128 ? (i & 1) * 128 : 0);
  }
  static constexpr uint32_t PART = NR * HDV * 4, ML = 128;  // a partial result: o, then m and l
  static constexpr uint32_t RING = STAGE > PART + ML ? STAGE : PART + ML;
  static constexpr uint32_t WARP = RING + PART + ML;  // the second partial lies over the page, done by then
  static constexpr uint32_t TOTAL = WARPS * WARP;
  static __device__ float* part(void* base, uint32_t warp, uint32_t slot) {
    return reinterpret_cast<float*>((char*)base + warp * WARP + (slot ? 0 : RING));
  }
};
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Asynchronous copies into shared memory; zeros where `in` is false.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy8(uint32_t dst, const void* src, bool in) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(in ? 8 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ uint4 lds16(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint2 lds8(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
  return v;
}
// An 8 x 8 matrix of f16 across the warp, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The exponent of a V scale as the weights take it.
__device__ __forceinline__ int v_exponent(uint32_t bits) { return min(max((int)(bits >> 23 & 255) - 127, -60), 127); }

constexpr int SUM_EXP = 38;   // the denominator's exponent beside m
constexpr int LIFT_FROM = 27;  // g = max(e, this)

// x 2^d for whole d <= 0, given f = ex2(d), which is 0 below 2^-126.
__device__ __forceinline__ float scaled(float x, float d, float f) {
  return f == 0.f && x != 0.f ? x * 1.17549435e-38f * ex2(d + 126.f) : x * f;
}

// Codes 0, 1 and 2, 3 of a word as two f16 pairs.
template <uint32_t FMT>
__device__ __forceinline__ void decode4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if (FMT == KV8_E4M3) {
    asm("{ .reg .b16 a, b; mov.b32 {a, b}, %2; cvt.rn.f16x2.e4m3x2 %0, a; cvt.rn.f16x2.e4m3x2 %1, b; }" : "=r"(lo), "=r"(hi) : "r"(w));
  } else {
    w ^= 0x80808080u;  // 0x6400 | byte is 1024 + byte in f16
    const __half2 off = __half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));  // 1152
    uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
    const __half2 x = __hsub2(*reinterpret_cast<__half2*>(&a), off), y = __hsub2(*reinterpret_cast<__half2*>(&b), off);
    lo = *reinterpret_cast<const uint32_t*>(&x), hi = *reinterpret_cast<const uint32_t*>(&y);
  }
}

__device__ __forceinline__ uint32_t pack_half(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void from_f(float x, float& o) { o = x; }
__device__ __forceinline__ void from_f(float x, __half& o) { o = __float2half_rn(x); }
__device__ __forceinline__ void from_f(float x, __nv_bfloat16& o) { o = __float2bfloat16_rn(x); }

// A sequence as the kernel walks it.
struct Seq {
  int32_t len, row0, n_rows;  // positions, first row of q, rows
  int32_t lo, tiles;          // first tile any row sees, tiles of a unit
  int64_t units;              // row blocks x KV heads
};
template <uint32_t NR>
__device__ __forceinline__ Seq seq_of(const Kv8AttnArgs& a, uint32_t s) {
  Seq q;
  const int64_t cap = (int64_t)min(a.table_ld, (uint64_t)(1u << 26)) * KV8_PAGE;
  q.len = a.lens[s];
  const int32_t r0 = a.first[s], r1 = a.first[s + 1];
  q.row0 = min(max(r0, 0), (int32_t)a.n_rows);
  q.n_rows = min(max(r1, 0), (int32_t)a.n_rows) - q.row0;
  if (q.n_rows <= 0) q.n_rows = 0;
  const int64_t held = min(max((int64_t)q.len, (int64_t)0), cap);
  const int64_t from = a.window ? max((int64_t)0, (int64_t)q.len - q.n_rows + 1 - (int64_t)a.window) : 0;
  q.lo = (int32_t)(min(from, held) / TILE);
  q.tiles = max(1, (int32_t)((held + TILE - 1) / TILE) - q.lo);
  q.units = (int64_t)(((int64_t)q.n_rows * a.group + NR - 1) / NR) * a.c.heads;
  return q;
}

template <uint32_t FMT, typename T, uint32_t HDV, uint32_t NR, bool FULL, bool LONG>
__global__ void __launch_bounds__(Shape<T, HDV, NR>::WARPS * 32, 1) kv8_attn_kernel(const Kv8AttnArgs a) {
  using L = Shape<T, HDV, NR>;
  constexpr bool SPLIT = L::SPLIT;
  constexpr float SUM_UNIT = (float)(1u << (SUM_EXP - 13));  // the denominator's factor over the weights'
  constexpr uint32_t WARPS = L::WARPS, THREADS = WARPS * 32;
  constexpr int MT = HDV / 16, SEG = HDV / 64, NB = NR / 8;  // M tiles of O^T, 64-dim segments, n tiles of rows
  extern __shared__ __align__(128) float4 attn_smem4[];
  __shared__ int64_t chunk_base[THREADS + 1];
  __shared__ int64_t warp_sum[WARPS];
  // A warp's partial results: of a unit that began before its share (0), of one that goes on behind it (1).
  struct Piece {
    int64_t unit, end;  // the unit's first page in the list (-1: no partial), and the one behind its last
    uint32_t head, row0, row_base, rows;
  };
  __shared__ Piece piece[WARPS * 2];
  __shared__ uint32_t last_flag[2];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const uint32_t hd = FULL ? HDV : a.c.hd;
  const uint32_t ring = smem_addr(attn_smem4) + warp * L::WARP;
  // Lane (g, t) reads K's rows g, g + 8, .. and V's rows 2t, 2t + 1, 2t + 8, ..
  const uint32_t copy_base = ring + L::at(lane / (HDV / 16), lane % (HDV / 16)), k_base = ring + L::at(g, t);
  const uint32_t v_base = ring + L::VALUES + (HDV == 128 ? L::at(2 * t, g) : L::at(2 * t, g >> 1) + (g & 1) * 8);

  // ---- the tile list: prefix sums over the sequences ----
  const uint32_t per_thread = (a.n_seqs + THREADS - 1) / THREADS;
  {
    const uint32_t s0 = min(a.n_seqs, threadIdx.x * per_thread), s1 = min(a.n_seqs, s0 + per_thread);
    int64_t sum = 0;
    for (uint32_t s = s0; s < s1; s++) {
      const Seq q = seq_of<NR>(a, s);
      sum += q.units * q.tiles;
    }
    int64_t x = sum;
    for (uint32_t o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(~0u, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) warp_sum[warp] = x;
    __syncthreads();
    int64_t before = 0;
    for (uint32_t i = 0; i < warp; i++) before += warp_sum[i];
    chunk_base[threadIdx.x] = before + x - sum;
    if (threadIdx.x == THREADS - 1) chunk_base[THREADS] = before + x;
    if (threadIdx.x < WARPS * 2) piece[threadIdx.x].unit = -1;
    __syncthreads();
  }
  const int64_t total = chunk_base[THREADS];
  // Equal shares, a page more or less, of as many CTAs as have two pages a warp (a short list is not all merging).
  const int64_t ctas = max(min((int64_t)gridDim.x, (total + 2 * WARPS - 1) / (2 * WARPS)), (int64_t)1), n_warps = ctas * WARPS;
  auto share_begin = [&](int64_t w) { return min(w, n_warps) * total / n_warps; };
  auto cta_of = [&](int64_t x) { return ((x + 1) * ctas - 1) / total; };  // the CTA whose share holds page x
  const int64_t my_warp = (int64_t)blockIdx.x * WARPS + warp, x_begin = share_begin(my_warp), x_end = share_begin(my_warp + 1);

  if (!FULL) {  // columns behind hd stay zero
    for (uint32_t i = lane * 16; i < L::SCALES; i += 512)
      *reinterpret_cast<uint4*>((char*)attn_smem4 + warp * L::WARP + i) = make_uint4(0, 0, 0, 0);
    __syncwarp();
  }
  if (x_begin < x_end) {
    // ---- where this warp's share begins ----
    uint32_t seq = 0;
    int64_t seq_base = 0;
    {
      uint32_t lo = 0, hi = THREADS;  // the last chunk that begins at or before x_begin
      while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (chunk_base[mid] <= x_begin) lo = mid; else hi = mid;
      }
      seq = lo * per_thread;
      seq_base = chunk_base[lo];
    }
    Seq sq = seq_of<NR>(a, seq);
    int64_t x = x_begin;
    while (x < x_end) {
      if (x >= seq_base + sq.units * sq.tiles) {
        seq_base += sq.units * sq.tiles;
        sq = seq_of<NR>(a, ++seq);
        continue;
      }
      const int64_t in_seq = x - seq_base;
      const int64_t unit = in_seq >> 31 ? in_seq / sq.tiles : (int64_t)((uint32_t)in_seq / (uint32_t)sq.tiles);
      const int64_t unit_base = seq_base + unit * sq.tiles, unit_end = unit_base + sq.tiles;
      int64_t stop = min(unit_end, x_end);
      if (sq.tiles <= SHORT) {  // not cut: the warp in whose share it begins does all of it
        if (x > unit_base) {
          x = unit_end;
          continue;
        }
        stop = unit_end;
      }
      const uint32_t block = (uint32_t)unit / a.c.heads, head = (uint32_t)unit - block * a.c.heads;
      const uint32_t total_rows = (uint32_t)sq.n_rows * a.group, row_base = block * NR;
      const uint32_t rows = min(NR, total_rows - row_base);

      // Positions of this unit's tiles that every row sees (no mask needed), and that some row sees.
      const int32_t pos_a = sq.len - sq.n_rows + (int32_t)(row_base / a.group);
      const int32_t pos_b = sq.len - sq.n_rows + (int32_t)((row_base + rows - 1) / a.group);
      const int64_t w64 = a.window ? (int64_t)a.window : (int64_t)1 << 40;
      const int32_t all_lo = (int32_t)max((int64_t)0, pos_b + 1 - w64), all_hi = min(pos_a + 1, sq.len);
      const int32_t any_lo = (int32_t)max((int64_t)0, pos_a + 1 - w64), any_hi = min(pos_b + 1, sq.len);

      const int32_t* table = a.table + (uint64_t)seq * a.table_ld;
      int32_t tile = sq.lo + (int32_t)(x - unit_base);
      // of [tile, tile_stop) only the tiles some row sees
      const int32_t tile_stop = min(sq.lo + (int32_t)(stop - unit_base), (int32_t)(((int64_t)max(any_hi, 0) + TILE - 1) / TILE));
      tile = max(tile, any_lo / (int32_t)TILE);
      // Pages: lane l holds the id of page `page0 + l`, and of the 32 behind them.
      int32_t page0 = tile;
      auto page_id = [&](int32_t pg) { return (uint64_t)pg < a.table_ld && pg < tile_stop ? (uint32_t)table[pg] : ~0u; };
      uint32_t ids = page_id(page0 + (int32_t)lane), ids_next = page_id(page0 + 32 + (int32_t)lane);
      auto find = [&](int32_t pg) -> uint32_t {
        if (pg - page0 >= 32) {
          page0 += 32;
          ids = ids_next;
          ids_next = page_id(page0 + 32 + (int32_t)lane);
        }
        return __shfl_sync(~0u, ids, (pg - page0) & 31);
      };
      // K's or V's 32 rows of a page, 512 consecutive bytes a warp and step. Rows at and behind
      // `n` arrive as zeros: behind a sequence's end lies anything.
      auto copy_rows = [&](uint32_t area, const uint8_t* src, int32_t n) {
        if constexpr (FULL) {
          const uint32_t dst = copy_base + area;
          src += lane * 16;
          if (n >= (int32_t)KV8_PAGE) {
#pragma unroll
            for (uint32_t i = 0; i < HDV / 16; i++) copy16(L::copy_at(dst, i), src + i * 512, true);
          } else {
#pragma unroll
            for (uint32_t i = 0; i < HDV / 16; i++) copy16(L::copy_at(dst, i), src + i * 512, (int32_t)((i * 32 + lane) / (HDV / 16)) < n);
          }
          return;
        }
        const uint32_t cpr = hd / 16, dst = ring + area;
#pragma unroll
        for (uint32_t i = 0; i < HDV / 16; i++) {
          if (i >= cpr) break;
          const uint32_t at = i * 32 + lane, row = at / cpr, col = at - row * cpr;
          copy16(dst + L::at(row, col), src + at * 16, (int32_t)row < n);
        }
      };
      auto fetch_k = [&](int32_t pg, uint32_t id) {  // an id outside the pool: no such page, its positions take no part
        if (pg < tile_stop && id < a.c.n_pages) {
          const uint64_t at = ((uint64_t)id * a.c.heads + head) * 2;
          copy_rows(0, a.c.codes + at * KV8_PAGE * hd, KV8_PAGE);
          if (lane == 0) copy8(ring + L::SCALES, a.c.scales + at, true);
        }
        copy_commit();
      };
      auto fetch_v = [&](int32_t pg, uint32_t id) {
        if (pg < tile_stop && id < a.c.n_pages)
          copy_rows(L::VALUES, a.c.codes + (((uint64_t)id * a.c.heads + head) * 2 + 1) * KV8_PAGE * hd,
                    sq.len - pg * (int32_t)TILE);
        copy_commit();
      };
      uint32_t id = find(tile);
      fetch_k(tile, id);
      fetch_v(tile, id);

      // ---- Q's fragments (lane (g, t): rows g of each n tile), and this lane's rows of S^T: 2t, 2t + 1 ----
      uint32_t qf[NB][SEG * 4][SPLIT ? 4 : 2];
      int32_t last_pos[NB][2];  // the last position the row sees
      float mult[NB][2];        // from S to log2 units, apart from the page's scale
#pragma unroll
      for (int nb = 0; nb < NB; nb++) {
        const uint32_t in_block = nb * 8 + g, row = row_base + min(in_block, rows - 1);
        const T* src = (const T*)a.q + (uint64_t)(sq.row0 + row / a.group) * a.ld_q + (uint64_t)(head * a.group + row % a.group) * hd;
        float e[SEG][16];
        uint32_t top = 0;
#pragma unroll
        for (int sg = 0; sg < SEG; sg++) {
          const uint32_t d0 = 64 * sg + 16 * t;
          if (d0 < hd && in_block < rows) {
            uint4 raw[sizeof(T)];
#pragma unroll
            for (uint32_t i = 0; i < sizeof(T); i++) raw[i] = reinterpret_cast<const uint4*>(src + d0)[i];
#pragma unroll
            for (int i = 0; i < 16; i++) e[sg][i] = to_f(reinterpret_cast<const T*>(raw)[i]);
          } else {
#pragma unroll
            for (int i = 0; i < 16; i++) e[sg][i] = 0.f;
          }
#pragma unroll
          for (int i = 0; i < 16; i++) top = max(top, __float_as_uint(e[sg][i]) & 0x7FFFFFFFu);
        }
        top = max(top, __shfl_xor_sync(~0u, top, 1));
        top = max(top, __shfl_xor_sync(~0u, top, 2));
        // The row times 2^k, its largest in [2^14, 2^15): f16 then holds what it can of every element. A row that is
        // not finite becomes NaN as a whole: scores of -inf would look like unseen ones.
        const int ex = (int)(top >> 23) - 127;
        const int k = top == 0 || ex == 128 ? 0 : min(14 - ex, 126);
        const float up = ex == 128 ? NAN : __uint_as_float((uint32_t)(k + 127) << 23);
        const float down = a.scale * 1.4426950408889634f / up;
#pragma unroll
        for (int sg = 0; sg < SEG; sg++)
#pragma unroll
          for (int j = 0; j < 4; j++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
              const float u = e[sg][4 * j + 2 * h] * up, w = e[sg][4 * j + 2 * h + 1] * up;
              const uint32_t p = pack_half(u, w);
              qf[nb][sg * 4 + j][h] = p;
              if constexpr (SPLIT) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&p));
                qf[nb][sg * 4 + j][2 + h] = pack_half(u - f.x, w - f.y);
              }
            }
#pragma unroll
        for (int r = 0; r < 2; r++) {
          mult[nb][r] = __shfl_sync(~0u, down, (2 * t + r) * 4);
          last_pos[nb][r] = sq.len - sq.n_rows + (int32_t)((row_base + min(nb * 8 + 2 * t + r, rows - 1)) / a.group);
        }
      }

      float o[NB][MT][4], m[NB][2], l[NB][2];
#pragma unroll
      for (int nb = 0; nb < NB; nb++) {
#pragma unroll
        for (int j = 0; j < MT; j++)
#pragma unroll
          for (int i = 0; i < 4; i++) o[nb][j][i] = 0.f;
        m[nb][0] = m[nb][1] = MINM, l[nb][0] = l[nb][1] = 0.f;
      }
      // The tensor core cuts its sums off, all to one side: 1.3e-4 of O over 32768 positions of one sign, 5.5e-4
      // over 131072. Where a warp may have more than FOLD_FROM pages of a unit (LONG), 16-bit rows' O goes to a sum
      // in memory every FOLD pages, which is rounded: 1e-5 is left. Code that is there costs 3% where it does not
      // run (4 sequences of up to 131072 positions, 28 pages a warp: 83.5 against 80.6 us), so it is a variant.
      bool has_kept = false;
      auto fold = [&](bool last) {  // the last into o itself
        static_assert(NB * (MT * 4 + 2) * 32 * WARPS <= KV8_KEEP_FLOATS, "O and m of every lane");
        float* kept = a.keep + (uint64_t)blockIdx.x * KV8_KEEP_FLOATS + warp * (NB * (MT * 4 + 2) * 32) + lane;
#pragma unroll
        for (int nb = 0; nb < NB; nb++, kept += (MT * 4 + 2) * 32) {
          float f[2] = {0.f, 0.f};
#pragma unroll
          for (int r = 0; r < 2; r++) {
            if (has_kept) f[r] = ex2(kept[(MT * 4 + r) * 32] - m[nb][r]);
            if (!last) kept[(MT * 4 + r) * 32] = m[nb][r];
          }
#pragma unroll
          for (int j = 0; j < MT; j++) {
            float was[4] = {0.f, 0.f, 0.f, 0.f};
            if (has_kept) {
#pragma unroll
              for (int i = 0; i < 4; i++) was[i] = kept[(j * 4 + i) * 32];
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
              o[nb][j][i] = fmaf(was[i], f[i & 1], o[nb][j][i]);
              if (!last) kept[(j * 4 + i) * 32] = o[nb][j][i], o[nb][j][i] = 0.f;
            }
          }
        }
        has_kept = true;
      };

      for (; tile < tile_stop; tile++) {
        const uint32_t next = find(tile + 1);
        const bool has = id < a.c.n_pages;
        copy_wait<1>();
        __syncwarp();
        // ---- S^T = K Q^T: two tiles of 16 positions ----
        float s[NB][2][4] = {};
        if (has) {
#pragma unroll
          for (int sg = 0; sg < SEG; sg++) {
            uint4 k[4];
#pragma unroll
            for (int n = 0; n < 4; n++) k[n] = lds16(L::k_at(k_base, n, sg));
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
              for (int half = 0; half < 2; half++) {
                uint32_t af[4];
                decode4<FMT>(reinterpret_cast<const uint32_t*>(&k[2 * half])[j], af[0], af[2]);
                decode4<FMT>(reinterpret_cast<const uint32_t*>(&k[2 * half + 1])[j], af[1], af[3]);
#pragma unroll
                for (int nb = 0; nb < NB; nb++) {
                  mma(s[nb][half], af, qf[nb][sg * 4 + j][0], qf[nb][sg * 4 + j][1]);
                  if constexpr (SPLIT) mma(s[nb][half], af, qf[nb][sg * 4 + j][2], qf[nb][sg * 4 + j][3]);
                }
              }
          }
        }
        const uint2 sc = lds8(ring + L::SCALES);
        __syncwarp();
        fetch_k(tile + 1, next);
        uint32_t pf[NB][2][SPLIT ? 4 : 2];
        if (has) {
          // ---- weights: s[nb][half][2 i + r] is position 16 half + 8 i + g, row 2t + r ----
          const float sk = __uint_as_float(sc.x), sv = __uint_as_float(sc.y);
          const int ev = v_exponent(sc.y);
          // the weights' factor 2^13 comes with the scale's fraction
          const int gv = max(ev, LIFT_FROM);
          const float e = (float)ev, lift = (float)(gv - ev), frac = sv * __uint_as_float((uint32_t)(127 + 13 - gv) << 23);
          const float back = __uint_as_float((uint32_t)(127 + SUM_EXP - gv) << 23);
          const int32_t p0 = tile * (int32_t)TILE;
          const bool masked = p0 < all_lo || p0 + (int32_t)TILE > all_hi;
          float f[NB][2];
#pragma unroll
          for (int nb = 0; nb < NB; nb++) f[nb][0] = mult[nb][0] * sk, f[nb][1] = mult[nb][1] * sk;
          // u = t + e, rounded here and then only compared and subtracted: no weight passes 2^13 however large
          // the scores are. Unseen ones are -inf, whatever the codes there were.
#pragma unroll
          for (int nb = 0; nb < NB; nb++)
#pragma unroll
            for (int k = 0; k < 8; k++) {
              float& v = s[nb][k >> 2][k & 3];
              v = fmaf(v, f[nb][k & 1], e);
              if (masked) {
                const int32_t pos = p0 + (int32_t)g + 8 * (k >> 1), last = last_pos[nb][k & 1];
                if (pos > last || (int64_t)pos <= last - w64) v = -INFINITY;
              }
            }
          float top[NB][2];
          bool more = false;
#pragma unroll
          for (int nb = 0; nb < NB; nb++)
#pragma unroll
            for (int r = 0; r < 2; r++) {
              top[nb][r] = fmaxf(fmaxf(s[nb][0][r], s[nb][0][2 + r]), fmaxf(s[nb][1][r], s[nb][1][2 + r]));
              more |= top[nb][r] > m[nb][r];
            }
          if (__any_sync(~0u, more)) {
#pragma unroll
            for (int nb = 0; nb < NB; nb++)
#pragma unroll
              for (int r = 0; r < 2; r++) {
                float x = fmaxf(top[nb][r], MINM);
                x = fmaxf(x, __shfl_xor_sync(~0u, x, 4));
                x = fmaxf(x, __shfl_xor_sync(~0u, x, 8));
                x = fmaxf(x, __shfl_xor_sync(~0u, x, 16));
                // whole: every factor between two maxima is exact
                const float mn = fmaxf(m[nb][r], ceilf(x)), alpha = ex2(m[nb][r] - mn);
                l[nb][r] = scaled(l[nb][r], m[nb][r] - mn, alpha);
                m[nb][r] = mn;
#pragma unroll
                for (int j = 0; j < MT; j++) o[nb][j][r] *= alpha, o[nb][j][2 + r] *= alpha;
              }
          }
#pragma unroll
          for (int nb = 0; nb < NB; nb++) {
            float sum[2] = {0.f, 0.f};
#pragma unroll
            for (int half = 0; half < 2; half++) {
              float w[4];
#pragma unroll
              for (int i = 0; i < 4; i++) {
                const float y = ex2((s[nb][half][i] - m[nb][i & 1]) + lift);
                sum[i & 1] += y;
                w[i] = y * frac;
                if (masked && s[nb][half][i] == -INFINITY) w[i] = 0.f;  // frac may be NaN
              }
#pragma unroll
              for (int i = 0; i < 2; i++) {
                const uint32_t p = pack_half(w[2 * i], w[2 * i + 1]);
                pf[nb][half][i] = transpose8(p);
                if constexpr (SPLIT) {
                  const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&p));
                  pf[nb][half][2 + i] = transpose8(pack_half(w[2 * i] - h.x, w[2 * i + 1] - h.y));
                }
              }
            }
            l[nb][0] = fmaf(sum[0], back, l[nb][0]);
            l[nb][1] = fmaf(sum[1], back, l[nb][1]);
          }
        }
        copy_wait<1>();
        __syncwarp();
        // ---- O^T += V^T P^T ----
        if (has) {
#pragma unroll
          for (int half = 0; half < 2; half++) {
            uint32_t vr[4][HDV / 32];
#pragma unroll
            for (int i = 0; i < 4; i++) {
              if constexpr (HDV == 128) {
                const uint4 v = lds16(L::v_at(v_base, half, i));
                vr[i][0] = v.x, vr[i][1] = v.y, vr[i][2] = v.z, vr[i][3] = v.w;
              } else {
                const uint2 v = lds8(L::v_at(v_base, half, i));
                vr[i][0] = v.x, vr[i][1] = v.y;
              }
            }
#pragma unroll
            for (int j2 = 0; j2 < MT / 2; j2++) {  // words: dims 4 j2 .. 4 j2 + 3 of this lane's
              uint32_t lo[4], hi[4];               // A fragments of M tiles 2 j2 and 2 j2 + 1
#pragma unroll
              for (int n = 0; n < 2; n++) {
                decode4<FMT>(__byte_perm(vr[2 * n][j2], vr[2 * n + 1][j2], 0x5140), lo[2 * n], lo[2 * n + 1]);
                decode4<FMT>(__byte_perm(vr[2 * n][j2], vr[2 * n + 1][j2], 0x7362), hi[2 * n], hi[2 * n + 1]);
              }
#pragma unroll
              for (int nb = 0; nb < NB; nb++) {
                if constexpr (SPLIT) {
                  // The tensor core cuts its sums off: over thousands of positions that bias passes 22 bits. So
                  // f32 rows' products of 16 positions are added to O in f32, rounded.
                  float x[2][4] = {};
                  mma(x[0], lo, pf[nb][half][2], pf[nb][half][3]);
                  mma(x[0], lo, pf[nb][half][0], pf[nb][half][1]);
                  mma(x[1], hi, pf[nb][half][2], pf[nb][half][3]);
                  mma(x[1], hi, pf[nb][half][0], pf[nb][half][1]);
#pragma unroll
                  for (int i = 0; i < 4; i++) o[nb][2 * j2][i] += x[0][i], o[nb][2 * j2 + 1][i] += x[1][i];
                } else {
                  mma(o[nb][2 * j2], lo, pf[nb][half][0], pf[nb][half][1]);
                  mma(o[nb][2 * j2 + 1], hi, pf[nb][half][0], pf[nb][half][1]);
                }
              }
            }
          }
        }
        __syncwarp();
        fetch_v(tile + 1, next);
        id = next;
        if constexpr (LONG)
          if (tile % FOLD == FOLD - 1 && tile + 1 < tile_stop) fold(false);
      }
      if constexpr (LONG)
        if (has_kept) fold(true);
      copy_wait<0>();
      // ---- this piece's result: lane (g, t) holds dims [d0, d0 + HDV / 8) of rows 2t, 2t + 1 ----
      const uint32_t d0 = HDV / 8 * g;
#pragma unroll
      for (int nb = 0; nb < NB; nb++)
#pragma unroll
        for (int r = 0; r < 2; r++) {
          l[nb][r] += __shfl_xor_sync(~0u, l[nb][r], 4);
          l[nb][r] += __shfl_xor_sync(~0u, l[nb][r], 8);
          l[nb][r] += __shfl_xor_sync(~0u, l[nb][r], 16);
        }
      const bool cut_left = x > unit_base, cut_right = stop < unit_end;
      if (!cut_left && !cut_right) {
#pragma unroll
        for (int nb = 0; nb < NB; nb++)
#pragma unroll
          for (int r = 0; r < 2; r++) {
            const uint32_t in_block = nb * 8 + 2 * t + r, row = row_base + in_block;
            if (in_block >= rows || d0 >= hd) continue;
            const float inv = l[nb][r] == 0.f ? 0.f : SUM_UNIT / l[nb][r];
            T* dst = (T*)a.out + (uint64_t)(sq.row0 + row / a.group) * a.ld_out + (uint64_t)(head * a.group + row % a.group) * hd + d0;
            constexpr uint32_t PER = 16 / sizeof(T);
#pragma unroll
            for (uint32_t c = 0; c < HDV / 8 / PER; c++) {
              T v[PER];
#pragma unroll
              for (uint32_t i = 0; i < PER; i++) from_f(o[nb][(c * PER + i) / 2][2 * (i & 1) + r] * inv, v[i]);
              *reinterpret_cast<uint4*>(dst + c * PER) = *reinterpret_cast<uint4*>(v);
            }
          }
      } else {
        const uint32_t slot = cut_left ? 0 : 1;
        __syncwarp();  // the second lies over the page, which other lanes may still be reading
        float* po = L::part(attn_smem4, warp, slot);
        float* ml = po + NR * HDV;
#pragma unroll
        for (int nb = 0; nb < NB; nb++)
#pragma unroll
          for (int r = 0; r < 2; r++) {
            const uint32_t row = nb * 8 + 2 * t + r;
#pragma unroll
            for (int c = 0; c < MT / 2; c++)
              *reinterpret_cast<float4*>(po + row * HDV + d0 + c * 4) =
                  make_float4(o[nb][2 * c][r], o[nb][2 * c][2 + r], o[nb][2 * c + 1][r], o[nb][2 * c + 1][2 + r]);
            if (g == 0) ml[row * 2] = m[nb][r], ml[row * 2 + 1] = l[nb][r];
          }
        if (lane == 0) piece[warp * 2 + slot] = {unit_base, unit_end, head, (uint32_t)sq.row0, row_base, rows};
      }
      x = stop;
    }
  }
  __syncthreads();

  auto store = [&](const Piece& pc, uint32_t row, uint32_t d, float4 o, float l) {
    const float inv = l == 0.f ? 0.f : SUM_UNIT / l;
    const uint32_t r = pc.row_base + row;
    T* dst = (T*)a.out + (uint64_t)(pc.row0 + r / a.group) * a.ld_out + (uint64_t)(pc.head * a.group + r % a.group) * hd + d;
    if (d < hd) from_f(o.x * inv, dst[0]), from_f(o.y * inv, dst[1]), from_f(o.z * inv, dst[2]), from_f(o.w * inv, dst[3]);
  };

  // ---- units cut between warps ----
  // In warp order, slot 0 before slot 1, the pieces of a unit follow one another.
  const int64_t cta_begin = share_begin((int64_t)blockIdx.x * WARPS), cta_end = share_begin((int64_t)(blockIdx.x + 1) * WARPS);
  const int64_t mine = lane < WARPS * 2 ? piece[lane].unit : -1;
  const uint32_t there = __ballot_sync(~0u, mine >= 0);
  const uint32_t before = there & ((1u << lane) - 1);
  const int64_t previous = __shfl_sync(~0u, mine, before ? 31 - __clz(before) : 0);
  uint32_t starts = __ballot_sync(~0u, mine >= 0 && (!before || previous != mine));
  int32_t open[2] = {-1, -1};  // pieces of units that other CTAs share: begun before this one, and in it
  uint32_t taken = 0;  // threads that the units so far occupy: the next unit's items go to those behind them
  while (starts) {
    const uint32_t i = __ffs(starts) - 1;
    starts &= starts - 1;
    const uint32_t ids = there & (starts ? (1u << (__ffs(starts) - 1)) - 1 : ~0u) & ~((1u << i) - 1);  // its pieces
    const Piece pc = piece[i];
    const bool whole = pc.unit >= cta_begin && pc.end <= cta_end;
    const uint32_t side = pc.unit < cta_begin ? 0 : 1;
    float* gpart = a.part + ((uint64_t)blockIdx.x * 2 + side) * KV8_PART_FLOATS;
    if (!whole) open[side] = (int32_t)i;
    const uint32_t items = pc.rows * (HDV / 4), first_item = threadIdx.x >= taken ? threadIdx.x - taken : threadIdx.x + THREADS - taken;
    taken = (taken + items) % THREADS;
    for (uint32_t at = first_item; at < items; at += THREADS) {
      const uint32_t row = at / (HDV / 4), d = at % (HDV / 4) * 4;
      float m = MINM, l = 0.f;
      bool lost = false;  // a factor of l was too small for it
      float4 o = make_float4(0, 0, 0, 0);
      for (uint32_t p = ids; p; p &= p - 1) m = fmaxf(m, L::part(attn_smem4, (__ffs(p) - 1) >> 1, (__ffs(p) - 1) & 1)[NR * HDV + row * 2]);
      for (uint32_t p = ids; p; p &= p - 1) {
        const float* po = L::part(attn_smem4, (__ffs(p) - 1) >> 1, (__ffs(p) - 1) & 1);
        const float2 ml = *reinterpret_cast<const float2*>(po + NR * HDV + row * 2);
        const float f = ex2(ml.x - m);
        const float4 v = *reinterpret_cast<const float4*>(po + row * HDV + d);
        l += f * ml.y, lost |= f == 0.f && ml.y != 0.f;
        o.x += f * v.x, o.y += f * v.y, o.z += f * v.z, o.w += f * v.w;
      }
      if (lost) {
        l = 0.f;
        for (uint32_t p = ids; p; p &= p - 1) {
          const float* ml = L::part(attn_smem4, (__ffs(p) - 1) >> 1, (__ffs(p) - 1) & 1) + NR * HDV + row * 2;
          l += scaled(ml[1], ml[0] - m, ex2(ml[0] - m));
        }
      }
      if (whole) {
        store(pc, row, d, o, l);
      } else {
        __stcg(reinterpret_cast<float4*>(gpart + row * HDV + d), o);
        if (d == 0) __stcg(reinterpret_cast<float2*>(gpart + 16 * KV8_MAX_HD + row * 2), make_float2(m, l));
      }
    }
  }
  if (open[0] < 0 && open[1] < 0) return;
  // ---- units cut between CTAs: the last one to arrive merges, in CTA order ----
  __threadfence();
  __syncthreads();
  if (threadIdx.x < 2) {
    uint32_t last = 0;
    if (open[threadIdx.x] >= 0) {
      const Piece& pc = piece[open[threadIdx.x]];
      const int64_t c0 = cta_of(pc.unit);
      const uint32_t others = (uint32_t)(cta_of(pc.end - 1) - c0);
      last = atomicInc(a.cnt + c0, others) == others;
    }
    last_flag[threadIdx.x] = last;
  }
  __syncthreads();
  for (int side = 0; side < 2; side++) {
    if (last_flag[side]) {
      __threadfence();
      const Piece pc = piece[open[side]];
      const int64_t c0 = cta_of(pc.unit);
      const uint32_t others = (uint32_t)(cta_of(pc.end - 1) - c0);  // CTAs behind the first
      auto part = [&](uint32_t c) { return a.part + ((uint64_t)(c0 + c) * 2 + (c ? 0 : 1)) * KV8_PART_FLOATS; };
      // Every (row, 4 dims) is summed by `ways` threads, each over every ways-th CTA, with
      // the loads of eight in flight; then over the ways, in order.
      constexpr uint32_t ITEMS = NR * (HDV / 4), WAYS = THREADS / ITEMS ? THREADS / ITEMS : 1;
      float* joint = reinterpret_cast<float*>(attn_smem4);  // [WAYS][NR][HDV]
      __shared__ float2 ml_of[WAYS][NR];
      for (uint32_t at = threadIdx.x; at < ITEMS * WAYS; at += THREADS) {
        const uint32_t way = at / ITEMS, row = at % ITEMS / (HDV / 4), d = at % (HDV / 4) * 4;
        if (row >= pc.rows) continue;
        float m = MINM, l = 0.f;
        bool lost = false;
        float4 o = make_float4(0, 0, 0, 0);
        for (uint32_t c = way; c <= others; c += WAYS * 8) {
          float2 ml[8];
          float4 v[8];
#pragma unroll
          for (uint32_t k = 0; k < 8; k++) {
            ml[k] = make_float2(MINM, 0.f);
            v[k] = make_float4(0, 0, 0, 0);
            if (c + k * WAYS <= others) {
              ml[k] = __ldcg(reinterpret_cast<const float2*>(part(c + k * WAYS) + 16 * KV8_MAX_HD + row * 2));
              v[k] = __ldcg(reinterpret_cast<const float4*>(part(c + k * WAYS) + row * HDV + d));
            }
          }
          float mn = m;
#pragma unroll
          for (uint32_t k = 0; k < 8; k++) mn = fmaxf(mn, ml[k].x);
          const float f0 = ex2(m - mn);
          lost |= f0 == 0.f && l != 0.f;
          l *= f0, o.x *= f0, o.y *= f0, o.z *= f0, o.w *= f0;
          m = mn;
#pragma unroll
          for (uint32_t k = 0; k < 8; k++) {
            const float f = ex2(ml[k].x - m);
            l += f * ml[k].y, lost |= f == 0.f && ml[k].y != 0.f;
            o.x += f * v[k].x, o.y += f * v[k].y, o.z += f * v[k].z, o.w += f * v[k].w;
          }
        }
        if (lost) {
          l = 0.f;
          for (uint32_t c = way; c <= others; c += WAYS) {
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(part(c) + 16 * KV8_MAX_HD + row * 2));
            l += scaled(ml.y, ml.x - m, ex2(ml.x - m));
          }
        }
        if (WAYS == 1) {
          store(pc, row, d, o, l);
        } else {
          *reinterpret_cast<float4*>(joint + (way * NR + row) * HDV + d) = o;
          if (d == 0) ml_of[way][row] = make_float2(m, l);
        }
      }
      if (WAYS > 1) {
        __syncthreads();
        for (uint32_t at = threadIdx.x; at < pc.rows * (HDV / 4); at += THREADS) {
          const uint32_t row = at / (HDV / 4), d = at % (HDV / 4) * 4;
          float m = MINM, l = 0.f;
          float4 o = make_float4(0, 0, 0, 0);
          for (uint32_t w = 0; w < WAYS; w++) m = fmaxf(m, ml_of[w][row].x);
          for (uint32_t w = 0; w < WAYS; w++) {
            const float f = ex2(ml_of[w][row].x - m);
            const float4 v = *reinterpret_cast<const float4*>(joint + (w * NR + row) * HDV + d);
            l += scaled(ml_of[w][row].y, ml_of[w][row].x - m, f);
            o.x += f * v.x, o.y += f * v.y, o.z += f * v.z, o.w += f * v.w;
          }
          store(pc, row, d, o, l);
        }
      }
    }
    __syncthreads();
  }
}

// Whether one of `shares` equal shares of the list, in units of `rows` rows, may hold more than FOLD_FROM pages of one.
inline bool folds(const Kv8AttnArgs& a, uint32_t rows, uint32_t shares) {
  const double units = ((double)a.n_rows * a.group / rows + a.n_seqs) * a.c.heads, pages = (double)a.table_ld;
  return pages > FOLD_FROM && units * pages > (double)FOLD_FROM * shares;
}
template <uint32_t FMT, typename T, uint32_t HDV, uint32_t NR, bool FULL, bool LONG = false>
cudaError_t attn_launch(const Kv8AttnArgs& a, uint32_t sms, cudaStream_t st) {
  using L = Shape<T, HDV, NR>;
  static_assert(L::TOTAL <= 220 * 1024, "shared memory");
  if constexpr (!L::SPLIT && !LONG)
    if (folds(a, NR, sms * L::WARPS)) return attn_launch<FMT, T, HDV, NR, FULL, true>(a, sms, st);
  auto* kern = kv8_attn_kernel<FMT, T, HDV, NR, FULL, LONG>;
  static SmemOnce once;
  const cudaError_t e = once.allow((const void*)kern, (int)L::TOTAL);
  if (e != cudaSuccess) return e;
  kern<<<sms, L::WARPS * 32, L::TOTAL, st>>>(a);
  return cudaGetLastError();
}
template <uint32_t FMT, typename T, uint32_t NR>
cudaError_t attn_hd(const Kv8AttnArgs& a, uint32_t sms, cudaStream_t st) {
  if (a.c.hd == 64) return attn_launch<FMT, T, 64, NR, true>(a, sms, st);
  if (a.c.hd == 128) return attn_launch<FMT, T, 128, NR, true>(a, sms, st);
  return attn_launch<FMT, T, 128, NR, false>(a, sms, st);
}
// Units of 8 rows while that is what a sequence has on average (one token of a
// group of up to 8 heads): half the registers, so more warps (32 sequences of
// 3000, 8 KV heads of 128, 8 rows each: 47 against 55 us; of 64: 30 against 38).
// Units of 16 read and decode the cache once for twice the rows (12 rows: 56.9
// against 56.5 us, 24 rows 91 against 105; of 64: 39 and 40, 59 and 55). f32
// rows: always 8, the low halves take the registers. The average is over what
// the host knows: padding rows and idle sequences count.
template <typename T>
cudaError_t attn_typed(const Kv8AttnArgs& a, uint32_t sms, cudaStream_t st) {
  if constexpr (sizeof(T) == 2) {
    if ((uint64_t)a.n_rows * a.group > 8ull * a.n_seqs)
      return a.c.fmt == KV8_E4M3 ? attn_hd<KV8_E4M3, T, 16>(a, sms, st) : attn_hd<KV8_I8, T, 16>(a, sms, st);
  }
  return a.c.fmt == KV8_E4M3 ? attn_hd<KV8_E4M3, T, 8>(a, sms, st) : attn_hd<KV8_I8, T, 8>(a, sms, st);
}

}  // namespace
}  // namespace sm
