// Attention over the 8-bit paged KV cache, tensor-core form (many rows a
// sequence: prompts, chunks of them, long drafts), f16 and bf16 rows.
// kv8_attn_f16.cu and kv8_attn_bf16.cu instantiate it. The weights, their
// scaling and the merging of partial results are those of kv8_attn.cuh.
//
// A unit is 128 (token, head of the group) rows of one sequence and KV head;
// a step is 64 positions (two pages). CTA roles:
//   * eight decode warps read a step's codes (the next step's are in flight
//     meanwhile), turn them into exact f16 and store them as the B operands:
//     K rows as they are (K-major), V rows as they are too (N-major: the
//     transposed operand is the tensor core's work);
//   * one thread issues S = Q K^T (M 128, N 64, Q in tensor memory) and
//     O += P V (M 128, N hd, P in tensor memory, over S), one after the other;
//   * four softmax warps, a row a thread: S from tensor memory, weights, P
//     back; they rescale O when the running maximum has risen by more than 4x
//     (weights keep that much room in f16), and write the results.
// One CTA's scores, weights and products follow one another; the two CTAs of
// an SM overlap each other's. Per step and CTA the tensor pipe needs 512
// cycles, the exponentials (16 a cycle) 512, shared memory about 640.
//
// Work is the list of all steps of all units; every CTA takes an equal share.
// A sequence's row blocks alternate between its first and last ones, so that
// under the causal mask neighbours in the list share the work.
//
// Every wait on an mbarrier is bounded; one that gives up sets the workspace's
// error word and an abort flag, after which the other waits return at once,
// the CTA waits (bounded) for the MMAs it issued, frees its tensor memory and
// leaves.
//
// Measured on B200: 2 sequences, chunks of up to 1024 rows over up to 8192
// positions, 28/4 heads of 128, bf16 rows: 334 us, 482 TFLOP/s of what the rows
// see (0.29 of the measured 1679); the streaming form takes 800. A step takes
// an SM about 2200 cycles, and no unit is busy for all of them: the issue slots
// 0.52, L1's data path 0.38, the tensor pipe 0.23. What counts is the softmax
// warps' latency between a step's two products, which two CTAs an SM overlap
// only in part. At 72 registers a thread they spill (196 bytes; 0.9 million
// local loads a launch). A second S, its product issued before the last step's
// weights are ready, with Q in shared memory, hides the first product and still
// takes 364 us.
#pragma once
#include "kv8_attn.cuh"
#include "tc_common.cuh"
#include "umma.cuh"

#include <type_traits>

namespace sm {
namespace {

constexpr uint32_t CH_ROWS = 128, CH_STEP = 64;
constexpr uint32_t CH_SOFT = 4, CH_DEC = 8, CH_WARPS = CH_SOFT + CH_DEC + 1, CH_THREADS = CH_WARPS * 32;
constexpr uint32_t CH_MIN_SHARE = 2;  // steps of a CTA
constexpr int32_t CH_FOLD = FOLD;  // steps whose products the tensor core adds up before they are added in f32
constexpr uint32_t CH_TCOLS = 256, CH_TS = 0, CH_TQ = 64, CH_TO = 128;  // tensor memory: S (and P over it), Q, O

__device__ __forceinline__ void ch_arrive(uint64_t* b) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(b)) : "memory");
}
// One try (the hardware parks the warp for a while), and a bounded wait; a wait
// that is not urgent sleeps between tries, so that it takes no issue slots.
__device__ __forceinline__ bool ch_try(uint64_t* b, uint32_t parity) {
  uint32_t ok;
  asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
               : "=r"(ok) : "r"(smem_u32(b)), "r"(parity) : "memory");
  return ok;
}
template <bool URGENT>
__device__ __forceinline__ bool ch_wait(uint64_t* b, uint32_t parity, uint32_t* err, volatile uint32_t* abort) {
  for (uint32_t n = 0; n < TC_SPIN_MAX; n++) {
    if (ch_try(b, parity)) return true;
    if (!URGENT) __nanosleep(100);
    if ((n & 31u) == 31u && *abort) return false;
  }
  *abort = 1u;
  atomicOr(err, 1u);
  return false;
}
__device__ __forceinline__ void ch_bar(uint32_t id, uint32_t n) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory"); }
__device__ __forceinline__ bool ch_elect() {
  uint32_t ok;
  asm volatile("{ .reg .pred p; elect.sync _|p, 0xFFFFFFFF; selp.u32 %0, 1, 0, p; }" : "=r"(ok));
  return ok;
}

// A sequence as this kernel walks it: tiles are steps.
__device__ __forceinline__ Seq chunk_seq_of(const Kv8AttnArgs& a, uint32_t s) {
  Seq q;
  const int64_t cap = (int64_t)min(a.table_ld, (uint64_t)(1u << 26)) * KV8_PAGE;
  q.len = a.lens[s];
  const int32_t r0 = a.first[s], r1 = a.first[s + 1];
  q.row0 = min(max(r0, 0), (int32_t)a.n_rows);
  q.n_rows = max(min(max(r1, 0), (int32_t)a.n_rows) - q.row0, 0);
  const int64_t held = min(max((int64_t)q.len, (int64_t)0), cap);
  const int64_t from = a.window ? max((int64_t)0, (int64_t)q.len - q.n_rows + 1 - (int64_t)a.window) : 0;
  q.lo = (int32_t)(min(from, held) / CH_STEP);
  q.tiles = max(1, (int32_t)((held + CH_STEP - 1) / CH_STEP) - q.lo);
  q.units = ((int64_t)q.n_rows * a.group + CH_ROWS - 1) / CH_ROWS * a.c.heads;
  return q;
}

// A CTA's part of a unit.
struct ChunkPiece {
  int64_t unit, end;            // the unit's first step in the list, and the one behind its last
  uint32_t seq, head, row0, row_base, rows;
  int32_t len, pos0;            // the sequence's length, the position of its first row
  int32_t step, stop;           // steps of it to do (those some row sees)
  int32_t all_lo, all_hi;       // positions that every row sees
  bool cut_left, cut_right;
};
struct ChunkWalk {
  int64_t x, x_end, seq_base;
  uint32_t seq;
  Seq sq;
  __device__ bool next(const Kv8AttnArgs& a, ChunkPiece& p) {
    if (x >= x_end) return false;
    while (x >= seq_base + sq.units * sq.tiles) {
      seq_base += sq.units * sq.tiles;
      sq = chunk_seq_of(a, ++seq);
    }
    const int64_t in_seq = x - seq_base;
    const uint32_t unit = (uint32_t)(in_seq >> 31 ? in_seq / sq.tiles : (int64_t)((uint32_t)in_seq / (uint32_t)sq.tiles));
    p.unit = seq_base + (int64_t)unit * sq.tiles;
    p.end = p.unit + sq.tiles;
    const int64_t stop = min(p.end, x_end);
    const uint32_t total = (uint32_t)sq.n_rows * a.group, blocks = (total + CH_ROWS - 1) / CH_ROWS;
    p.head = unit / blocks;
    const uint32_t j = unit - p.head * blocks, block = j & 1 ? blocks - 1 - j / 2 : j / 2;
    p.seq = seq;
    p.row0 = (uint32_t)sq.row0;
    p.row_base = block * CH_ROWS;
    p.rows = min(CH_ROWS, total - p.row_base);
    p.len = sq.len;
    p.pos0 = sq.len - sq.n_rows;
    const int32_t pos_a = p.pos0 + (int32_t)(p.row_base / a.group), pos_b = p.pos0 + (int32_t)((p.row_base + p.rows - 1) / a.group);
    const int64_t w64 = a.window ? (int64_t)a.window : (int64_t)1 << 40;
    p.all_lo = (int32_t)max((int64_t)0, pos_b + 1 - w64), p.all_hi = min(pos_a + 1, sq.len);
    const int32_t any_lo = (int32_t)max((int64_t)0, pos_a + 1 - w64), any_hi = min(pos_b + 1, sq.len);
    p.step = max(sq.lo + (int32_t)(x - p.unit), any_lo / (int32_t)CH_STEP);
    p.stop = min(sq.lo + (int32_t)(stop - p.unit), (int32_t)(((int64_t)max(any_hi, 0) + CH_STEP - 1) / CH_STEP));
    p.cut_left = x > p.unit, p.cut_right = stop < p.end;
    x = stop;
    return true;
  }
};

template <uint32_t FMT, typename T, uint32_t HD, bool LONG>
__global__ void __launch_bounds__(CH_THREADS, 2) kv8_chunk_kernel(const Kv8AttnArgs a) {
  constexpr float SUM_UNIT = (float)(1u << (SUM_EXP - 12));  // the denominator's factor over the weights'
  constexpr uint32_t CORE = 128 + 16;          // 16-byte columns of 8 rows, and a gap: see the decode warps
  constexpr uint32_t GROUP8 = HD / 8 * CORE;   // bytes of 8 positions
  constexpr uint32_t OPERAND = CH_STEP / 8 * GROUP8;  // bytes of a step's K or V
  constexpr uint32_t ITEMS = CH_STEP * HD / 16 / 128;  // 16-code loads of a decode thread
  extern __shared__ __align__(128) float4 attn_smem4[];
  uint8_t* ops = reinterpret_cast<uint8_t*>(attn_smem4);  // K, K, V, V
  __shared__ int64_t chunk_base[CH_THREADS + 1];
  __shared__ int64_t warp_sum[CH_WARPS];
  __shared__ uint64_t full_k[2], full_v[2], empty_k[2], empty_v[2], full_sc[4], s_full, p_full, pv_done, q_full, all_done;
  __shared__ float4 scales[4][2];  // of a step's pages: of K, of V, 1 if the page is there
  __shared__ ChunkPiece open_piece[2];
  __shared__ uint32_t open_flag[2], last_flag[2], s_tmem, s_abort_word;
  __shared__ uint32_t s_gone[3];  // what the softmax warps agree on: a step's (two in turn), a piece's end
  volatile uint32_t* abort = &s_abort_word;
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; i++) {
      mbar_init(&full_k[i], CH_DEC * 16), mbar_init(&full_v[i], CH_DEC * 16);
      mbar_init(&empty_k[i], 1), mbar_init(&empty_v[i], 1);
      open_flag[i] = 0;
    }
    for (int i = 0; i < 4; i++) mbar_init(&full_sc[i], 2);
    mbar_init(&s_full, 1), mbar_init(&pv_done, 1), mbar_init(&all_done, 1);
    mbar_init(&p_full, CH_SOFT * 32), mbar_init(&q_full, CH_SOFT * 32);
    *abort = 0u;
    fence_mbar_init();
  }
  if (warp == CH_WARPS - 1) {
    tmem_alloc(&s_tmem, CH_TCOLS);
    tmem_relinquish();
  }

  // ---- the list of steps: prefix sums over the sequences ----
  const uint32_t per_thread = (a.n_seqs + CH_THREADS - 1) / CH_THREADS;
  {
    const uint32_t s0 = min(a.n_seqs, threadIdx.x * per_thread), s1 = min(a.n_seqs, s0 + per_thread);
    int64_t sum = 0;
    for (uint32_t s = s0; s < s1; s++) {
      const Seq q = chunk_seq_of(a, s);
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
    if (threadIdx.x == CH_THREADS - 1) chunk_base[CH_THREADS] = before + x;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
  }
  const uint32_t tb = s_tmem;
  const int64_t total = chunk_base[CH_THREADS];
  const int64_t share = max((total + gridDim.x - 1) / gridDim.x, (int64_t)CH_MIN_SHARE);
  ChunkWalk walk;
  walk.x = min(total, (int64_t)blockIdx.x * share), walk.x_end = min(total, walk.x + share);
  if (walk.x < walk.x_end) {
    uint32_t lo = 0, hi = CH_THREADS;
    while (hi - lo > 1) {
      const uint32_t mid = (lo + hi) / 2;
      if (chunk_base[mid] <= walk.x) lo = mid; else hi = mid;
    }
    walk.seq = lo * per_thread, walk.seq_base = chunk_base[lo];
    walk.sq = chunk_seq_of(a, walk.seq);
  }
  ChunkPiece pc;
  uint32_t it = 0, n_piece = 0;  // steps and pieces (with steps) so far

  if (warp >= CH_SOFT && warp < CH_SOFT + CH_DEC) {
    // ------------------------------------------------ decode warps: four for K, four for V
    const uint32_t tid = threadIdx.x % 128, is_v = warp >= CH_SOFT + CH_DEC / 2;
    uint64_t *full = is_v ? full_v : full_k, *empty = is_v ? empty_v : empty_k;
    uint8_t* dst = ops + is_v * 2 * OPERAND;
    // An item is 16 codes of a row; a thread's are 128 apart. A warp's 32 are 512 consecutive bytes, and the eight
    // lanes of a shared-memory phase hold four columns of two rows: with 144 bytes a column pair's step they meet
    // different banks (128 bytes would want eight rows a phase, whose loads take eight lines: 348 against 341 us).
    const uint32_t col = HD == 128 ? (lane & 3) | (lane >> 1 & 4) : lane & 3;
    const uint32_t row0 = HD == 128 ? tid / 32 * 4 + (lane >> 2 & 1) + (lane >> 4) * 2 : tid / 4;
    constexpr uint32_t ROWS = 128 / (HD / 16);  // rows between items
    const uint64_t src0 = ((uint64_t)is_v * KV8_PAGE + row0) * HD + col * 16;
    struct Ids { uint32_t id[2]; };  // a step's pages
    auto pages = [&](const ChunkPiece& p, int32_t step) {
      Ids r;
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int32_t pg = step * 2 + h;
        r.id[h] = step < p.stop && (uint64_t)pg < a.table_ld && pg * (int32_t)KV8_PAGE < p.len ? (uint32_t)a.table[(uint64_t)p.seq * a.table_ld + pg] : ~0u;
      }
      return r;
    };
    auto load = [&](const ChunkPiece& p, int32_t step, const Ids& ids, uint4 (&r)[ITEMS]) {
#pragma unroll
      for (uint32_t k = 0; k < ITEMS; k++) {
        const uint32_t row = row0 + k * ROWS, id = ids.id[k * ROWS / KV8_PAGE];
        r[k] = make_uint4(0, 0, 0, 0);
        // V behind the sequence's end: anything lies there
        if (id < a.c.n_pages && (!is_v || step * (int32_t)CH_STEP + (int32_t)row < p.len))
          r[k] = __ldg(reinterpret_cast<const uint4*>(a.c.codes + ((uint64_t)id * a.c.heads + p.head) * 2 * KV8_PAGE * HD + src0 + (k * ROWS) % KV8_PAGE * HD));
      }
    };
    auto put = [&](const ChunkPiece& p, const Ids& ids, const uint4 (&r)[ITEMS]) {
      const uint32_t st = it & 1;
      float2 sc = make_float2(0.f, 0.f);
      const bool brings = !is_v && tid < 2, there = brings && ids.id[tid & 1] < a.c.n_pages;
      if (there) sc = __ldg(reinterpret_cast<const float2*>(a.c.scales) + (uint64_t)ids.id[tid & 1] * a.c.heads + p.head);
      // one warp of the four waits, the others for it at a barrier
      if (it >= 2 && tid < 32) ch_wait<false>(&empty[st], (it / 2 + 1) & 1, a.err, abort);
      if (is_v) ch_bar(3, 128); else ch_bar(2, 128);
#pragma unroll
      for (uint32_t k = 0; k < ITEMS; k++) {
        uint8_t* at = dst + st * OPERAND + (row0 + k * ROWS) / 8 * GROUP8 + col * 2 * CORE + row0 % 8 * 16;
        uint4 lo, hi;
        decode4<FMT>(r[k].x, lo.x, lo.y), decode4<FMT>(r[k].y, lo.z, lo.w);
        decode4<FMT>(r[k].z, hi.x, hi.y), decode4<FMT>(r[k].w, hi.z, hi.w);
        *reinterpret_cast<uint4*>(at) = lo;
        *reinterpret_cast<uint4*>(at + CORE) = hi;
      }
      fence_proxy_async();
      ch_arrive(&full[st]);
      if (brings) {
        // The slot's last readers, the softmax of step it - 4, are done: K's buffer came free after the scores
        // of step it - 2, which follow the weights of step it - 3.
        scales[it & 3][tid] = make_float4(sc.x, sc.y, there ? 1.f : 0.f, 0.f);
        ch_arrive(&full_sc[it & 3]);
      }
      it++;
    };
    // No early way out here: the four warps meet at a barrier each step, and after a wait that gave up
    // (abort is set) the rest of the waits end at once.
    while (walk.next(a, pc)) {
      if (pc.step >= pc.stop) continue;
      // codes one step ahead, page ids two
      uint4 r0[ITEMS], r1[ITEMS];
      Ids i0 = pages(pc, pc.step), i1 = pages(pc, pc.step + 1);
      load(pc, pc.step, i0, r0);
      for (int32_t step = pc.step; step < pc.stop; step += 2) {
        load(pc, step + 1, i1, r1);
        const Ids i2 = pages(pc, step + 2);
        put(pc, i0, r0);
        if (step + 1 >= pc.stop) break;
        load(pc, step + 2, i2, r0);
        const Ids i3 = pages(pc, step + 3);
        put(pc, i1, r1);
        i0 = i2, i1 = i3;
      }
    }
  } else if (warp == CH_WARPS - 1) {
    // ------------------------------------------------ MMAs: the warp as one, an elected lane issues
    const uint32_t s_desc = umma_idesc_f16(CH_ROWS, CH_STEP), o_desc = umma_idesc_f16(CH_ROWS, HD) | 1u << 16;  // B N-major
    const uint64_t k_base = umma_desc_k(smem_u32(ops), CORE, GROUP8);
    // N-major B: 8 positions x 8 dims are 128 bytes, CORE apart; groups of dims follow one another, groups of positions are GROUP8 apart
    const uint64_t v_base = umma_desc_k(smem_u32(ops + 2 * OPERAND), GROUP8, CORE);
    bool gone = false;
    while (walk.next(a, pc) && !gone) {
      if (pc.step >= pc.stop) continue;
      gone = __any_sync(~0u, !ch_wait<true>(&q_full, n_piece++ & 1, a.err, abort));
      for (int32_t step = pc.step; step < pc.stop && !gone; step++, it++) {
        const uint32_t st = it & 1;
        bool ok = ch_wait<true>(&full_k[st], it / 2 & 1, a.err, abort);
        if (it) ok = ok && ch_wait<true>(&pv_done, (it + 1) & 1, a.err, abort);  // P of the last step is read
        gone = __any_sync(~0u, !ok);
        if (gone) break;
        tc_fence_after();
        const uint64_t kd = k_base + st * (OPERAND >> 4), vd = v_base + st * (OPERAND >> 4);
        if (ch_elect()) {
#pragma unroll
          for (uint32_t k = 0; k < HD / 16; k++) umma_ts(tb + CH_TS, tb + CH_TQ + 8 * k, kd + k * (2 * CORE >> 4), s_desc, k != 0);
          umma_commit(&s_full);
          umma_commit(&empty_k[st]);
        }
        __syncwarp();
        ok = ch_wait<true>(&full_v[st], it / 2 & 1, a.err, abort) && ch_wait<true>(&p_full, it & 1, a.err, abort);
        gone = __any_sync(~0u, !ok);
        if (gone) break;
        tc_fence_after();
        const uint32_t more = step != pc.step && !(LONG && step % CH_FOLD == 0);
        if (ch_elect()) {
#pragma unroll
          for (uint32_t k = 0; k < CH_STEP / 16; k++)
            umma_ts(tb + CH_TO, tb + CH_TS + 8 * k, vd + k * (2 * GROUP8 >> 4), o_desc, k != 0 ? 1u : more);
          umma_commit(&pv_done);
          umma_commit(&empty_v[st]);
        }
        __syncwarp();
      }
    }
  } else {
    // ------------------------------------------------ softmax warps: a row a thread
    const uint32_t row = threadIdx.x, tl = tb + (warp * 32 << 16);
    const int64_t w64 = a.window ? (int64_t)a.window : (int64_t)1 << 40;
    static_assert(2 * CH_ROWS * HD <= KV8_KEEP_FLOATS, "O of two CTAs");
    float* kept = a.keep + (uint64_t)blockIdx.x * (CH_ROWS * HD) + row;  // of this row, dims CH_ROWS apart
    float kept_m = MINM;
    bool has_kept = false;
    bool gone = false;  // the CTA gave up: decided by the four warps as one, tensor-memory access is warp-wide
    while (walk.next(a, pc)) {
      float m = MINM, l = 0.f;
      const uint32_t r = pc.row_base + min(row, pc.rows - 1), token = r / a.group, hq = pc.head * a.group + r % a.group;
      if (pc.step < pc.stop && !gone) {
        const int32_t last_pos = pc.pos0 + (int32_t)token;
        float mult;
        {  // the row of Q, times a power of two that brings its largest to [2^14, 2^15), and the scale's sign; or NaN
          const uint4* src = reinterpret_cast<const uint4*>((const T*)a.q + (uint64_t)(pc.row0 + token) * a.ld_q + (uint64_t)hq * HD);
          uint32_t top = 0;
#pragma unroll 4
          for (uint32_t i = 0; i < HD / 8; i++) {
            const uint4 v = src[i];
            const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
            for (int j = 0; j < 8; j++) top = max(top, __float_as_uint(to_f(e[j])) & 0x7FFFFFFFu);
          }
          const int ex = (int)(top >> 23) - 127;
          const int k = top == 0 || ex == 128 ? 0 : min(14 - ex, 126);
          const float up = ex == 128 ? NAN : __uint_as_float((uint32_t)(k + 127) << 23 | (__float_as_uint(a.scale) & 0x80000000u));
          mult = a.scale * 1.4426950408889634f / up;
#pragma unroll
          for (uint32_t c = 0; c < HD / 32; c++) {
            uint32_t q[16];
#pragma unroll
            for (uint32_t i = 0; i < 4; i++) {
              const uint4 v = src[c * 4 + i];
              const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
              for (int j = 0; j < 4; j++) q[i * 4 + j] = row < pc.rows ? pack_half(to_f(e[2 * j]) * up, to_f(e[2 * j + 1]) * up) : 0u;
            }
            tmem_st16(tl + CH_TQ + 16 * c, q);
          }
          tmem_wait_st();
          tc_fence_before();
          ch_arrive(&q_full);
        }
        has_kept = false;
        bool steep = false;  // some page's e is above 52
        for (int32_t step = pc.step; step < pc.stop && !gone; step++, it++) {
          ch_wait<true>(&full_sc[it & 3], it / 4 & 1, a.err, abort);  // the scales come before the scores
          const int32_t p0 = step * (int32_t)CH_STEP;
          float f[2], e[2], back[2], frac[2];
          bool masked = p0 < pc.all_lo || p0 + (int32_t)CH_STEP > pc.all_hi;
          bool here[2];
#pragma unroll
          for (int h = 0; h < 2; h++) {
            const float4 sc = scales[it & 3][h];
            const int ev = v_exponent(__float_as_uint(sc.y));
            // the weights' factor 2^12 comes with the scale's fraction
            e[h] = (float)ev, back[h] = __uint_as_float((uint32_t)(127 + 12 - ev) << 23), frac[h] = sc.y * back[h];
            f[h] = mult * sc.x;
            here[h] = sc.z != 0.f;
            steep |= e[h] > 52.f;
            masked |= !here[h] || !(frac[h] >= 4096.f && frac[h] < 8192.f);
          }
          // columns of this row that it sees: [lo, hi) of each page's 32
          int32_t lo[2] = {0, 0}, hi[2] = {32, 32};
          if (masked) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
              const int64_t first = (int64_t)last_pos - w64 + 1 - (p0 + 32 * h);
              lo[h] = (int32_t)min(max(first, (int64_t)0), (int64_t)32);
              hi[h] = here[h] ? min(max(last_pos + 1 - (p0 + 32 * h), 0), 32) : 0;
            }
          }
          // one warp waits, the others for it at a barrier
          if (warp == 0) {
            ch_wait<true>(&s_full, it & 1, a.err, abort);
            // Two words in turn: the other warps may still be reading the last step's, and all must see the same.
            if (lane == 0) s_gone[it & 1] = *abort;
          }
          ch_bar(1, CH_SOFT * 32);
          gone = s_gone[it & 1];
          if (gone) break;
          tc_fence_after();
          float top = MINM;
          auto largest = [&](auto with_mask) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
              uint32_t s[32];
              tmem_ld32(tl + CH_TS + 32 * h, s);
              tmem_wait_ld();
              float x = -INFINITY;
#pragma unroll
              for (int i = 0; i < 32; i++)
                x = fmaxf(x, !with_mask.value || (i >= lo[h] && i < hi[h]) ? __uint_as_float(s[i]) : -INFINITY);
              if (x > -INFINITY) top = fmaxf(top, fmaf(x, f[h], e[h]));
            }
          };
          if (masked) largest(std::true_type{}); else largest(std::false_type{});
          // O so far to the kept sum; this step's product overwrites it.
          const bool fold = LONG && step != pc.step && step % CH_FOLD == 0;
          if (fold) {
            const float fk = has_kept ? ex2(kept_m - m) : 0.f;
#pragma unroll 1
            for (uint32_t c = 0; c < HD / 16; c++) {
              uint32_t o[16];
              float was[16] = {}, *at = kept + 16 * c * CH_ROWS;
              if (has_kept) {
#pragma unroll
                for (int i = 0; i < 16; i++) was[i] = at[i * CH_ROWS];
              }
              tmem_ld16(tl + CH_TO + 16 * c, o);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 16; i++) at[i * CH_ROWS] = fmaf(was[i], fk, __uint_as_float(o[i]));
            }
            has_kept = true, kept_m = m;
          }
          // Weights up to 2^14 fit f16 (times a scale's fraction): the maximum may lag by a factor 4.
          if (__any_sync(~0u, top - m > 2.f)) {
            const float mn = top - m > 2.f ? ceilf(top) : m, alpha = ex2(m - mn);
            l = scaled(l, m - mn, alpha);
            m = mn;
            if (step != pc.step && !fold) {
#pragma unroll 1
              for (uint32_t c = 0; c < HD / 32; c++) {
                uint32_t o[32];
                tmem_ld32(tl + CH_TO + 32 * c, o);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                tmem_st32(tl + CH_TO + 32 * c, o);
              }
            }
          }
          auto weigh = [&](auto with_mask) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
              // Unmasked: the factor goes into the exponent (exact for a power of two; else off by 2^-16 at most, as
              // |m| is at most 256) and out of l again (4 us of 340 less than multiplying each weight). What underflows is
              // nothing to l while no e is above 52.
              const float c = e[h] - m + __log2f(frac[h]);
              // Masked: 2^(t + g - m), as in the streaming form.
              const float lift = fmaxf((float)LIFT_FROM - e[h], 0.f), low = ex2(-lift), fr = frac[h] * low;
              const float lb = with_mask.value ? back[h] * SUM_UNIT * low : __fdividef(back[h] * SUM_UNIT, frac[h]);
              float sum = 0.f;
#pragma unroll
              for (int half = 0; half < 2; half++) {
                uint32_t s[16], p[8];
                tmem_ld16(tl + CH_TS + 32 * h + 16 * half, s);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 8; i++) {
                  float y[2];
#pragma unroll
                  for (int j = 0; j < 2; j++) {
                    const int col = 16 * half + 2 * i + j;
                    const bool see = !with_mask.value || (col >= lo[h] && col < hi[h]);
                    // large scores: t + e rounded as for the maximum, so that no weight passes 2^14
                    if (with_mask.value) {
                      y[j] = see ? ex2(fmaf(__uint_as_float(s[2 * i + j]), f[h], e[h]) - m + lift) : 0.f;
                      sum += y[j];
                      y[j] = see ? y[j] * fr : 0.f;  // fr may be NaN
                    } else {
                      y[j] = ex2(fmaf(__uint_as_float(s[2 * i + j]), f[h], c));
                      sum += y[j];
                    }
                  }
                  p[i] = pack_half(y[0], y[1]);
                }
                tmem_st8(tl + CH_TS + 16 * h + 8 * half, p);  // over columns already read
              }
              l = fmaf(sum, lb, l);
            }
          };
          if (__any_sync(~0u, masked || steep || fabsf(m) > 256.f)) weigh(std::true_type{}); else weigh(std::false_type{});
          tmem_wait_st();
          tc_fence_before();
          ch_arrive(&p_full);
        }
        if (!gone) {
          if (warp == 0) {
            ch_wait<true>(&pv_done, (it + 1) & 1, a.err, abort);
            if (lane == 0) s_gone[2] = *abort;
          }
          ch_bar(1, CH_SOFT * 32);
          gone = s_gone[2];
        }
        tc_fence_after();
      }
      // ---- this piece's row ----
      const bool whole = !pc.cut_left && !pc.cut_right, some = pc.step < pc.stop;
      const uint32_t side = pc.cut_left ? 0 : 1;
      float* gpart = a.part + ((uint64_t)blockIdx.x * 2 + side) * KV8_CHUNK_PART_FLOATS;
      const float inv = l == 0.f ? 0.f : SUM_UNIT / l;
      T* dst = (T*)a.out + (uint64_t)(pc.row0 + token) * a.ld_out + (uint64_t)hq * HD;
#pragma unroll 1
      for (uint32_t c = 0; c < HD / 16; c++) {
        uint32_t o[16];
        if (some) {
          tmem_ld16(tl + CH_TO + 16 * c, o);
          tmem_wait_ld();
          if (LONG && has_kept) {
            const float fk = ex2(kept_m - m), *at = kept + 16 * c * CH_ROWS;
            float was[16];
#pragma unroll
            for (int i = 0; i < 16; i++) was[i] = at[i * CH_ROWS];
#pragma unroll
            for (int i = 0; i < 16; i++) o[i] = __float_as_uint(fmaf(was[i], fk, __uint_as_float(o[i])));
          }
        } else {
#pragma unroll
          for (int i = 0; i < 16; i++) o[i] = 0;
        }
        if (row >= pc.rows || gone) {
        } else if (whole) {
          T v[16];
#pragma unroll
          for (int i = 0; i < 16; i++) from_f(__uint_as_float(o[i]) * inv, v[i]);
          reinterpret_cast<uint4*>(dst + 16 * c)[0] = reinterpret_cast<uint4*>(v)[0];
          reinterpret_cast<uint4*>(dst + 16 * c)[1] = reinterpret_cast<uint4*>(v)[1];
        } else {
#pragma unroll
          for (int i = 0; i < 4; i++)
            __stcg(reinterpret_cast<uint4*>(gpart + row * HD + 16 * c) + i, make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]));
        }
        __syncwarp();
      }
      if (!whole) {
        if (row < pc.rows) __stcg(reinterpret_cast<float2*>(gpart + CH_ROWS * KV8_MAX_HD) + row, make_float2(m, l));
        if (row == 0) open_piece[side] = pc, open_flag[side] = 1;
      }
      tc_fence_before();  // O and Q are read before the next piece's MMAs
    }
  }

  // ---- teardown: the MMAs are complete (softmax waited for the last), or the CTA gave up and waits for them ----
  __syncwarp();
  if (*abort && warp == CH_WARPS - 1 && ch_elect()) {
    umma_commit(&all_done);  // when all MMAs issued are complete
    for (uint32_t n = 0; n < 1000; n++)
      if (mbar_try(&all_done, 0)) break;
  }
  __syncwarp();
  __threadfence();
  tc_fence_before();
  __syncthreads();
  if (warp == CH_WARPS - 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tb, CH_TCOLS);
  }

  // ---- units cut between CTAs: the last one to arrive merges, in CTA order ----
  if (!open_flag[0] && !open_flag[1]) return;
  if (threadIdx.x < 2) {
    uint32_t last = 0;
    if (open_flag[threadIdx.x]) {
      const ChunkPiece& p = open_piece[threadIdx.x];
      const int64_t c0 = p.unit / share;
      const uint32_t others = (uint32_t)((p.end - 1) / share - c0);
      last = atomicInc(a.cnt + c0, others) == others;
    }
    last_flag[threadIdx.x] = last;
  }
  __syncthreads();
  for (int side = 0; side < 2; side++) {
    if (!last_flag[side]) continue;
    __threadfence();
    const ChunkPiece& p = open_piece[side];
    const int64_t c0 = p.unit / share;
    const uint32_t others = (uint32_t)((p.end - 1) / share - c0);
    auto part = [&](uint32_t c) { return a.part + ((uint64_t)(c0 + c) * 2 + (c ? 0 : 1)) * KV8_CHUNK_PART_FLOATS; };
    auto ml_of = [&](uint32_t c, uint32_t row) { return __ldcg(reinterpret_cast<const float2*>(part(c) + CH_ROWS * KV8_MAX_HD) + row); };
    // A thread a row: its maximum and the factor of its sum; then a thread 8 dims of a row, four pieces' loads in flight.
    float2* of_row = reinterpret_cast<float2*>(ops);
    if (side) __syncthreads();  // the first side's are read
    if (threadIdx.x < p.rows) {
      float m = MINM, l = 0.f;
#pragma unroll 4
      for (uint32_t c = 0; c <= others; c++) m = fmaxf(m, ml_of(c, threadIdx.x).x);
#pragma unroll 4
      for (uint32_t c = 0; c <= others; c++) {
        const float2 ml = ml_of(c, threadIdx.x);
        l += scaled(ml.y, ml.x - m, ex2(ml.x - m));
      }
      of_row[threadIdx.x] = make_float2(m, l == 0.f ? 0.f : SUM_UNIT / l);
    }
    __syncthreads();
    for (uint32_t at = threadIdx.x; at < p.rows * (HD / 8); at += CH_THREADS) {
      const uint32_t row = at / (HD / 8), d = at % (HD / 8) * 8;
      const float2 mi = of_row[row];
      float o[8] = {};
      for (uint32_t c = 0; c <= others; c += 4) {
        float f[4];
        float4 v[4][2];
#pragma unroll
        for (uint32_t k = 0; k < 4; k++) {
          f[k] = MINM;
          v[k][0] = v[k][1] = make_float4(0, 0, 0, 0);
          if (c + k <= others) {
            f[k] = ml_of(c + k, row).x;
            v[k][0] = __ldcg(reinterpret_cast<const float4*>(part(c + k) + row * HD + d));
            v[k][1] = __ldcg(reinterpret_cast<const float4*>(part(c + k) + row * HD + d + 4));
          }
        }
#pragma unroll
        for (uint32_t k = 0; k < 4; k++) {
          f[k] = ex2(f[k] - mi.x);
          const float* x = reinterpret_cast<const float*>(v[k]);
#pragma unroll
          for (int i = 0; i < 8; i++) o[i] += f[k] * x[i];
        }
      }
      const uint32_t r = p.row_base + row;
      T v[8];
#pragma unroll
      for (int i = 0; i < 8; i++) from_f(o[i] * mi.y, v[i]);
      *reinterpret_cast<uint4*>((T*)a.out + (uint64_t)(p.row0 + r / a.group) * a.ld_out + (uint64_t)(p.head * a.group + r % a.group) * HD + d) =
          *reinterpret_cast<uint4*>(v);
    }
  }
}

template <uint32_t FMT, typename T, uint32_t HD, bool LONG = false>
cudaError_t chunk_launch(const Kv8AttnArgs& a, uint32_t sms, cudaStream_t st) {
  if constexpr (!LONG)
    if (folds(a, CH_ROWS, 2 * sms)) return chunk_launch<FMT, T, HD, true>(a, sms, st);
  constexpr uint32_t smem = 4 * CH_STEP * HD * 2 / 128 * (128 + 16);  // four operands of columns CORE apart
  auto* kern = kv8_chunk_kernel<FMT, T, HD, LONG>;
  static SmemOnce once;
  const cudaError_t e = once.allow((const void*)kern, (int)smem);
  if (e != cudaSuccess) return e;
  kern<<<2 * sms, CH_THREADS, smem, st>>>(a);
  return cudaGetLastError();
}

// Rows of a sequence, on average, from which this form is taken. 4 sequences of 4096 positions in the streaming form
// and in this one: 8 KV heads of 128, 62 and 78 us with 112 rows each, 76 and 73 with 160, 106 and 88 with 256, 185
// and 108 with 512; 4 KV heads of 128, 40 and 53, 49 and 64, 65 and 82, 105 and 87; 8 of 64, 40 and 52, 50 and 54, 70
// and 62, 122 and 81. The average is over what the host knows: padding rows and idle sequences count.
constexpr uint32_t CHUNK_MIN_ROWS = 256;
inline bool chunk_takes(const Kv8AttnArgs& a) {
  return (a.c.hd == 64 || a.c.hd == 128) && (uint64_t)a.n_rows * a.group >= (uint64_t)CHUNK_MIN_ROWS * a.n_seqs;
}
template <typename T>
cudaError_t chunk_typed(const Kv8AttnArgs& a, uint32_t sms, cudaStream_t st) {
  if (a.c.hd == 64) return a.c.fmt == KV8_E4M3 ? chunk_launch<KV8_E4M3, T, 64>(a, sms, st) : chunk_launch<KV8_I8, T, 64>(a, sms, st);
  return a.c.fmt == KV8_E4M3 ? chunk_launch<KV8_E4M3, T, 128>(a, sms, st) : chunk_launch<KV8_I8, T, 128>(a, sms, st);
}

}  // namespace
}  // namespace sm
