// Attention over the 8-bit paged KV cache.
//
//   o = sum_j p_j s_v(j) V_j / sum_j p_j,   p_j = exp(scale s_k(j) q.K_j)
//
// over the positions j a row sees; K_j, V_j are codes, s_k, s_v the scales of
// j's page. One pass with a running maximum m of t_j + e_j, where
// t_j = log2 p_j and e_j = exponent of s_v(j): the weights of the products,
// w_j = 2^(t_j + e_j - m + 13), are then relative to the largest
// *contribution* and fit f16 whatever the spread of the pages' scales, while
// the denominator adds w_j 2^-e_j in f32. m is kept a whole number, so moving
// it multiplies by a power of two and rounds nothing.
//
// Bound by the cache bytes (2 hd a position and head), so nothing passes
// through shared memory: a warp loads a tile of 16 positions straight into
// the registers that mma.m16n8k16 wants. K is the B operand (k = head dims,
// n = positions): lane (g, t) holds 16 consecutive dims of position g, which
// serve four k-steps whose k order is permuted alike in Q's fragments. S's
// accumulators are the A operand of P V. V is its B operand (k = positions,
// n = dims): lane (g, t) loads dims [16g, 16g + 16) of four positions and
// interleaves their bytes in pairs. The codes are exact in f16.
//
// Rows are (token, head of the group) pairs of one sequence and KV head,
// 16 a unit. f32 rows are 8 a unit: rows 0-7 of the MMA carry the high and
// rows 8-15 the low f16 half of q (and of w), so scores and products keep 22
// bits at the cost of rows that a group of 8 would leave empty.
//
// Work is the list of all tiles of all (sequence, row block, KV head) units
// laid end to end; every warp takes an equal share, whatever the lengths are,
// which only the device knows. A unit cut between warps of a CTA is merged in
// shared memory, one cut between CTAs by the last of them to arrive.
#include "kv8.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

namespace sm {
namespace {

constexpr uint32_t WARPS = 8;
constexpr uint32_t TILE = 16;
constexpr uint32_t MAXHD = 128;
constexpr float MINM = -1e30f;  // running maximum of a row that has seen nothing
constexpr uint32_t PART_FLOATS = 16 * (MAXHD + 2);

__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 ldg16(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ uint2 ldg8(const uint8_t* p) {
  uint2 v;
  asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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
template <uint32_t RB>
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
  q.units = (int64_t)(((int64_t)q.n_rows * a.group + RB - 1) / RB) * a.c.heads;
  return q;
}

// One warp's state of one unit.
template <uint32_t HDV, bool SPLIT>
struct Acc {
  static constexpr int NT = HDV / 8, ROWS = SPLIT ? 1 : 2;
  float o[NT][4];
  float m[ROWS], l[ROWS];
  __device__ void clear() {
#pragma unroll
    for (int j = 0; j < NT; j++)
#pragma unroll
      for (int i = 0; i < 4; i++) o[j][i] = 0.f;
#pragma unroll
    for (int r = 0; r < ROWS; r++) m[r] = MINM, l[r] = 0.f;
  }
};

template <uint32_t FMT, typename T, uint32_t HDV>
__global__ void __launch_bounds__(WARPS * 32, 1) kv8_attn_kernel(const Kv8AttnArgs a) {
  constexpr bool SPLIT = sizeof(T) == 4;
  constexpr uint32_t RB = SPLIT ? 8 : 16;
  constexpr int NT = HDV / 8, SEG = HDV / 64, ROWS = SPLIT ? 1 : 2;
  constexpr uint32_t STRIDE = HDV + 4;  // floats between rows of a partial in shared memory
  extern __shared__ float4 attn_smem4[];
  float* part_o = reinterpret_cast<float*>(attn_smem4);       // [WARPS * 2][RB][STRIDE]
  float* part_ml = part_o + WARPS * 2 * RB * STRIDE;          // [WARPS * 2][RB][2]
  __shared__ int64_t chunk_base[WARPS * 32 + 1];
  __shared__ int64_t warp_sum[WARPS];
  __shared__ int64_t piece_unit[WARPS][2];  // tile index where the piece's unit begins, -1: no partial
  __shared__ int64_t piece_end[WARPS][2];   // tile index behind that unit's last
  __shared__ uint32_t piece_seq[WARPS][2], piece_in[WARPS][2];
  __shared__ uint32_t last_flag;
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;

  // ---- the tile list: prefix sums over the sequences ----
  const uint32_t per_thread = (a.n_seqs + WARPS * 32 - 1) / (WARPS * 32);
  {
    const uint32_t s0 = min(a.n_seqs, threadIdx.x * per_thread), s1 = min(a.n_seqs, s0 + per_thread);
    int64_t sum = 0;
    for (uint32_t s = s0; s < s1; s++) {
      const Seq q = seq_of<RB>(a, s);
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
    if (threadIdx.x == WARPS * 32 - 1) chunk_base[WARPS * 32] = before + x;
    if (threadIdx.x < WARPS) piece_unit[threadIdx.x][0] = piece_unit[threadIdx.x][1] = -1;
    __syncthreads();
  }
  const int64_t total = chunk_base[WARPS * 32];
  // Equal shares; at least two tiles, so that a short list is not all merging.
  const int64_t n_warps = (int64_t)gridDim.x * WARPS;
  const int64_t share = max((total + n_warps - 1) / n_warps, (int64_t)2);
  const int64_t x_begin = min(total, ((int64_t)blockIdx.x * WARPS + warp) * share), x_end = min(total, x_begin + share);

  if (x_begin < x_end) {
    // ---- where this warp's share begins ----
    uint32_t seq = 0;
    int64_t seq_base = 0;
    {
      uint32_t lo = 0, hi = WARPS * 32;  // the last chunk that begins at or before x_begin and is not empty
      while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (chunk_base[mid] <= x_begin) lo = mid; else hi = mid;
      }
      seq = lo * per_thread;
      seq_base = chunk_base[lo];
    }
    Seq sq = seq_of<RB>(a, seq);
    while (x_begin >= seq_base + sq.units * sq.tiles) {
      seq_base += sq.units * sq.tiles;
      sq = seq_of<RB>(a, ++seq);
    }
    int64_t x = x_begin;
    while (x < x_end) {
      if (x >= seq_base + sq.units * sq.tiles) {
        seq_base += sq.units * sq.tiles;
        sq = seq_of<RB>(a, ++seq);
        continue;
      }
      const int64_t unit = (x - seq_base) / sq.tiles;
      const int64_t unit_base = seq_base + unit * sq.tiles, unit_end = unit_base + sq.tiles;
      const int64_t stop = min(unit_end, x_end);
      const uint32_t head = (uint32_t)(unit % a.c.heads), block = (uint32_t)(unit / a.c.heads);
      const uint32_t total_rows = (uint32_t)sq.n_rows * a.group, row_base = block * RB;
      const uint32_t rows = min(RB, total_rows - row_base);

      // ---- this lane's rows: g (and g + 8), Q's fragments ----
      int32_t last_pos[ROWS];  // the last position the row sees
      float mult[ROWS];        // from S to log2 units, apart from the page's scale
      uint32_t qf[SEG * 4][4];
#pragma unroll
      for (int r = 0; r < ROWS; r++) {
        const uint32_t in_block = g + 8 * r, row = row_base + min(in_block, rows - 1);
        const uint32_t token = row / a.group, hq = head * a.group + row % a.group;
        last_pos[r] = sq.len - sq.n_rows + (int32_t)token;
        const T* src = (const T*)a.q + (uint64_t)(sq.row0 + token) * a.ld_q + (uint64_t)hq * a.c.hd;
        float e[SEG][16];
        uint32_t top = 0;
#pragma unroll
        for (int sg = 0; sg < SEG; sg++) {
          const uint32_t d0 = 64 * sg + 16 * t;
          if (d0 < a.c.hd && in_block < rows) {
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
        // The row times 2^k, its largest in [2^14, 2^15): f16 then holds what it can of every element.
        const int ex = (int)(top >> 23) - 127;
        const int k = top == 0 || ex == 128 ? 0 : min(14 - ex, 126);
        const float up = __uint_as_float((uint32_t)(k + 127) << 23);
        mult[r] = a.scale * 1.4426950408889634f / up;
#pragma unroll
        for (int sg = 0; sg < SEG; sg++)
#pragma unroll
          for (int j = 0; j < 4; j++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
              const float u = e[sg][4 * j + 2 * h] * up, w = e[sg][4 * j + 2 * h + 1] * up;
              const uint32_t p = pack_half(u, w);
              qf[sg * 4 + j][2 * h + r] = p;
              if (SPLIT) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&p));
                qf[sg * 4 + j][2 * h + 1] = pack_half(u - f.x, w - f.y);
              }
            }
      }
      // Positions of this unit's tiles that every row sees (no mask needed), and that some row sees.
      const int32_t pos_a = sq.len - sq.n_rows + (int32_t)(row_base / a.group);
      const int32_t pos_b = sq.len - sq.n_rows + (int32_t)((row_base + rows - 1) / a.group);
      const int64_t w64 = a.window ? (int64_t)a.window : (int64_t)1 << 40;
      const int32_t all_lo = (int32_t)max((int64_t)0, pos_b + 1 - w64), all_hi = min(pos_a + 1, sq.len);
      const int32_t any_lo = (int32_t)max((int64_t)0, pos_a + 1 - w64), any_hi = min(pos_b + 1, sq.len);

      Acc<HDV, SPLIT> acc;
      acc.clear();
      const int32_t* table = a.table + (uint64_t)seq * a.table_ld;
      int32_t tile = sq.lo + (int32_t)(x - unit_base);
      // of [tile, tile_stop) only the tiles some row sees
      const int32_t tile_stop = min(sq.lo + (int32_t)(stop - unit_base), (int32_t)(((int64_t)max(any_hi, 0) + TILE - 1) / TILE));
      tile = max(tile, any_lo / (int32_t)TILE);
      for (; tile < tile_stop; tile++) {
        const int32_t pg = tile / 2;
        const uint32_t id = (uint64_t)pg < a.table_ld ? (uint32_t)table[pg] : ~0u;
        if (id >= a.c.n_pages) continue;  // no such page: its positions take no part
        const uint64_t at = ((uint64_t)id * a.c.heads + head) * 2;
        const uint8_t* kp = a.c.codes + (at * KV8_PAGE + (tile & 1) * TILE) * a.c.hd;
        const uint8_t* vp = kp + (uint64_t)KV8_PAGE * a.c.hd;
        const float sk = a.c.scales[at], sv = a.c.scales[at + 1];
        uint4 kr[2][SEG];
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
          for (int sg = 0; sg < SEG; sg++)
            kr[n][sg] = 64 * sg + 16 * t < a.c.hd ? ldg16(kp + (n * 8 + g) * a.c.hd + 64 * sg + 16 * t) : make_uint4(0, 0, 0, 0);
        uint32_t vr[4][HDV / 32];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const uint32_t pos = 2 * t + (i & 1) + 8 * (i >> 1), d0 = (HDV / 8) * g;
          const bool in = d0 < a.c.hd && tile * (int32_t)TILE + (int32_t)pos < sq.len;  // behind the end: anything
          if constexpr (HDV == 128) {
            const uint4 v = in ? ldg16(vp + pos * a.c.hd + d0) : make_uint4(0, 0, 0, 0);
            vr[i][0] = v.x, vr[i][1] = v.y, vr[i][2] = v.z, vr[i][3] = v.w;
          } else {
            const uint2 v = in ? ldg8(vp + pos * a.c.hd + d0) : make_uint2(0, 0);
            vr[i][0] = v.x, vr[i][1] = v.y;
          }
        }
        // ---- S = Q K^T ----
        float s[2][4] = {};
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
          for (int sg = 0; sg < SEG; sg++) {
            const uint32_t w[4] = {kr[n][sg].x, kr[n][sg].y, kr[n][sg].z, kr[n][sg].w};
#pragma unroll
            for (int j = 0; j < 4; j++) {
              uint32_t b0, b1;
              decode4<FMT>(w[j], b0, b1);
              mma(s[n], qf[sg * 4 + j], b0, b1);
            }
          }
        // ---- weights ----
        const uint32_t svb = __float_as_uint(sv);
        const int ev = min(max((int)(svb >> 23 & 255) - 127, -60), 126);
        const float e = (float)ev, back = __uint_as_float((uint32_t)(127 - ev) << 23), frac = sv * back;
        const int32_t p0 = tile * (int32_t)TILE;
        const bool masked = p0 < all_lo || p0 + (int32_t)TILE > all_hi;
        float w[ROWS][4];
#pragma unroll
        for (int r = 0; r < ROWS; r++) {
          const float f = mult[r] * sk;
          float top = MINM;
          bool see[4];
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const float v = SPLIT ? s[i >> 1][i & 1] + s[i >> 1][2 + (i & 1)] : s[i >> 1][2 * r + (i & 1)];
            w[r][i] = v;
            see[i] = true;
            if (masked) {
              const int32_t pos = p0 + 2 * (int32_t)t + (i & 1) + 8 * (i >> 1);
              see[i] = pos <= last_pos[r] && (int64_t)pos > last_pos[r] - w64;
            }
            top = fmaxf(top, see[i] ? w[r][i] * f : MINM);
          }
          top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
          top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
          // whole: e - m below is exact, and so is every factor between two maxima
          const float m = fmaxf(acc.m[r], ceilf(top + e));
          if (__any_sync(~0u, m > acc.m[r])) {
            const float alpha = ex2(acc.m[r] - m);
            acc.m[r] = m;
            acc.l[r] *= alpha;
#pragma unroll
            for (int j = 0; j < NT; j++) {
              acc.o[j][2 * r] *= alpha, acc.o[j][2 * r + 1] *= alpha;
              if (SPLIT) acc.o[j][2] *= alpha, acc.o[j][3] *= alpha;
            }
          }
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const float y = see[i] ? ex2(fmaf(w[r][i], f, e - m + 13.f)) : 0.f;
            acc.l[r] += y * back;
            w[r][i] = see[i] ? y * frac : 0.f;
          }
        }
        // ---- O += P V ----
        uint32_t pf[4];
        if (SPLIT) {
#pragma unroll
          for (int n = 0; n < 2; n++) {
            pf[2 * n] = pack_half(w[0][2 * n], w[0][2 * n + 1]);
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&pf[2 * n]));
            pf[2 * n + 1] = pack_half(w[0][2 * n] - f.x, w[0][2 * n + 1] - f.y);
          }
        } else {
#pragma unroll
          for (int n = 0; n < 2; n++)
#pragma unroll
            for (int r = 0; r < ROWS; r++) pf[2 * n + r] = pack_half(w[r][2 * n], w[r][2 * n + 1]);
        }
#pragma unroll
        for (int j4 = 0; j4 < NT / 4; j4++) {
          uint32_t b[4][2];
#pragma unroll
          for (int n = 0; n < 2; n++) {
            decode4<FMT>(__byte_perm(vr[2 * n][j4], vr[2 * n + 1][j4], 0x5140), b[0][n], b[1][n]);
            decode4<FMT>(__byte_perm(vr[2 * n][j4], vr[2 * n + 1][j4], 0x7362), b[2][n], b[3][n]);
          }
#pragma unroll
          for (int j = 0; j < 4; j++) mma(acc.o[j4 * 4 + j], pf, b[j][0], b[j][1]);
        }
      }
      // ---- this piece's result ----
      // Lane (g, t) holds dims [d0, d0 + HDV / 4) of row g (and g + 8).
      const uint32_t d0 = HDV / 4 * t;
#pragma unroll
      for (int r = 0; r < ROWS; r++) {
        acc.l[r] += __shfl_xor_sync(~0u, acc.l[r], 1);
        acc.l[r] += __shfl_xor_sync(~0u, acc.l[r], 2);
        if (SPLIT) {
#pragma unroll
          for (int j = 0; j < NT; j++) acc.o[j][0] += acc.o[j][2], acc.o[j][1] += acc.o[j][3];
        }
      }
      const bool cut_left = x > unit_base, cut_right = stop < unit_end;
      if (!cut_left && !cut_right) {
#pragma unroll
        for (int r = 0; r < ROWS; r++) {
          const uint32_t in_block = g + 8 * r, row = row_base + in_block;
          if (in_block >= rows) continue;
          const float inv = acc.l[r] == 0.f ? 0.f : 1.f / acc.l[r];
          T* dst = (T*)a.out + (uint64_t)(sq.row0 + row / a.group) * a.ld_out + (uint64_t)(head * a.group + row % a.group) * a.c.hd;
#pragma unroll
          for (int h = 0; h < 2; h++) {
            const uint32_t d = d0 + h * NT;
#pragma unroll
            for (uint32_t c = 0; c < NT / (16 / sizeof(T)); c++) {
              T v[16 / sizeof(T)];
#pragma unroll
              for (uint32_t i = 0; i < 16 / sizeof(T); i++) from_f(acc.o[c * (16 / sizeof(T)) + i][2 * r + h] * inv, v[i]);
              if (d + c * (16 / sizeof(T)) < a.c.hd) *reinterpret_cast<uint4*>(dst + d + c * (16 / sizeof(T))) = *reinterpret_cast<uint4*>(v);
            }
          }
        }
      } else {
        const uint32_t slot = cut_left ? 0 : 1;
        float* po = part_o + (warp * 2 + slot) * RB * STRIDE;
        float* ml = part_ml + (warp * 2 + slot) * RB * 2;
#pragma unroll
        for (int r = 0; r < ROWS; r++) {
          const uint32_t row = g + 8 * r;
#pragma unroll
          for (int h = 0; h < 2; h++)
#pragma unroll
            for (int c = 0; c < NT / 4; c++)
              *reinterpret_cast<float4*>(po + row * STRIDE + d0 + h * NT + c * 4) =
                  make_float4(acc.o[4 * c][2 * r + h], acc.o[4 * c + 1][2 * r + h], acc.o[4 * c + 2][2 * r + h], acc.o[4 * c + 3][2 * r + h]);
          if (t == 0) ml[row * 2] = acc.m[r], ml[row * 2 + 1] = acc.l[r];
        }
        if (lane == 0) {
          piece_unit[warp][slot] = unit_base;
          piece_end[warp][slot] = unit_end;
          piece_seq[warp][slot] = seq;
          piece_in[warp][slot] = (uint32_t)unit;
        }
      }
      x = stop;
    }
  }
  __syncthreads();

  // ---- units cut between warps ----
  // In warp order, slot 0 (cut on the left) before slot 1: the pieces of a unit follow one another.
  const int64_t cta_share = share * WARPS, cta_begin = min(total, (int64_t)blockIdx.x * cta_share), cta_end = min(total, cta_begin + cta_share);
  uint32_t i = 0;
  while (i < WARPS * 2) {
    const int64_t base = piece_unit[i >> 1][i & 1];
    if (base < 0) {
      i++;
      continue;
    }
    uint32_t pieces = 1, ids[WARPS];  // a unit has one piece a warp
    ids[0] = i;
    uint32_t k = i + 1;
    for (; k < WARPS * 2; k++) {
      const int64_t b = piece_unit[k >> 1][k & 1];
      if (b < 0) continue;
      if (b != base) break;
      ids[pieces++ & (WARPS - 1)] = k;
    }
    const int64_t end = piece_end[i >> 1][i & 1];
    const uint32_t seq = piece_seq[i >> 1][i & 1], unit = piece_in[i >> 1][i & 1];
    const Seq sq = seq_of<RB>(a, seq);
    const uint32_t head = unit % a.c.heads, row_base = unit / a.c.heads * RB;
    const uint32_t rows = min(RB, (uint32_t)sq.n_rows * a.group - row_base);
    const bool whole = base >= cta_begin && end <= cta_end;
    float* gpart = a.part + ((uint64_t)blockIdx.x * 2 + (base < cta_begin ? 0 : 1)) * PART_FLOATS;
    for (uint32_t at = threadIdx.x; at < rows * (HDV / 4); at += WARPS * 32) {
      const uint32_t row = at / (HDV / 4), d = at % (HDV / 4) * 4;
      float m = MINM, l = 0.f;
      float4 o = make_float4(0, 0, 0, 0);
      for (uint32_t p = 0; p < pieces; p++) m = fmaxf(m, part_ml[(ids[p] * RB + row) * 2]);
      for (uint32_t p = 0; p < pieces; p++) {
        const float f = ex2(part_ml[(ids[p] * RB + row) * 2] - m);
        const float4 v = *reinterpret_cast<const float4*>(part_o + (ids[p] * RB + row) * STRIDE + d);
        l += f * part_ml[(ids[p] * RB + row) * 2 + 1];
        o.x += f * v.x, o.y += f * v.y, o.z += f * v.z, o.w += f * v.w;
      }
      if (whole) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        T* dst = (T*)a.out + (uint64_t)(sq.row0 + (row_base + row) / a.group) * a.ld_out +
                 (uint64_t)(head * a.group + (row_base + row) % a.group) * a.c.hd + d;
        if (d < a.c.hd) from_f(o.x * inv, dst[0]), from_f(o.y * inv, dst[1]), from_f(o.z * inv, dst[2]), from_f(o.w * inv, dst[3]);
      } else {
        __stcg(reinterpret_cast<float4*>(gpart + row * HDV + d), o);
        if (d == 0) __stcg(reinterpret_cast<float2*>(gpart + 16 * MAXHD + row * 2), make_float2(m, l));
      }
    }
    if (!whole) {
      // ---- cut between CTAs: the last one to arrive merges, in CTA order ----
      const int64_t c0 = base / cta_share, c1 = (end - 1) / cta_share;
      __threadfence();
      __syncthreads();
      if (threadIdx.x == 0) last_flag = atomicInc(a.cnt + c0, (uint32_t)(c1 - c0)) == (uint32_t)(c1 - c0);
      __syncthreads();
      if (last_flag) {
        __threadfence();
        for (uint32_t at = threadIdx.x; at < rows * (HDV / 4); at += WARPS * 32) {
          const uint32_t row = at / (HDV / 4), d = at % (HDV / 4) * 4;
          float m = MINM, l = 0.f;
          float4 o = make_float4(0, 0, 0, 0);
          for (int64_t c = c0; c <= c1; c++) {
            const float* p = a.part + ((uint64_t)c * 2 + (c == c0 ? 1 : 0)) * PART_FLOATS;
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(p + 16 * MAXHD + row * 2));
            const float4 v = __ldcg(reinterpret_cast<const float4*>(p + row * HDV + d));
            const float mn = fmaxf(m, ml.x), f0 = ex2(m - mn), f1 = ex2(ml.x - mn);
            m = mn;
            l = l * f0 + ml.y * f1;
            o.x = o.x * f0 + v.x * f1, o.y = o.y * f0 + v.y * f1, o.z = o.z * f0 + v.z * f1, o.w = o.w * f0 + v.w * f1;
          }
          const float inv = l == 0.f ? 0.f : 1.f / l;
          T* dst = (T*)a.out + (uint64_t)(sq.row0 + (row_base + row) / a.group) * a.ld_out +
                   (uint64_t)(head * a.group + (row_base + row) % a.group) * a.c.hd + d;
          if (d < a.c.hd) from_f(o.x * inv, dst[0]), from_f(o.y * inv, dst[1]), from_f(o.z * inv, dst[2]), from_f(o.w * inv, dst[3]);
        }
      }
      __syncthreads();
    }
    i = k;
  }
}

template <uint32_t FMT, typename T, uint32_t HDV>
cudaError_t attn_launch(const Kv8AttnArgs& a, uint32_t sms, cudaStream_t st) {
  constexpr uint32_t RB = sizeof(T) == 4 ? 8 : 16;
  const size_t smem = WARPS * 2 * RB * (HDV + 4 + 2) * sizeof(float);
  auto* kern = kv8_attn_kernel<FMT, T, HDV>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  kern<<<sms, WARPS * 32, smem, st>>>(a);
  return cudaGetLastError();
}
template <uint32_t FMT, typename T>
cudaError_t attn_hd(const Kv8AttnArgs& a, uint32_t sms, cudaStream_t st) {
  return a.c.hd <= 64 ? attn_launch<FMT, T, 64>(a, sms, st) : attn_launch<FMT, T, 128>(a, sms, st);
}
template <uint32_t FMT>
cudaError_t attn_type(const Kv8AttnArgs& a, uint32_t type, uint32_t sms, cudaStream_t st) {
  switch (type) {
    case ACT_F32: return attn_hd<FMT, float>(a, sms, st);
    case ACT_F16: return attn_hd<FMT, __half>(a, sms, st);
    default: return attn_hd<FMT, __nv_bfloat16>(a, sms, st);
  }
}

}  // namespace

uint64_t kv8_attn_part_floats(uint32_t sms) { return (uint64_t)sms * 2 * PART_FLOATS; }
uint32_t kv8_attn_counters(uint32_t sms) { return sms; }

cudaError_t launch_kv8_attn(const Kv8AttnArgs& a, uint32_t type, uint32_t sms, cudaStream_t st) {
  if (!a.n_rows || !a.n_seqs) return cudaSuccess;
  return a.c.fmt == KV8_E4M3 ? attn_type<KV8_E4M3>(a, type, sms, st) : attn_type<KV8_I8>(a, type, sms, st);
}

}  // namespace sm
