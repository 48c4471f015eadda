// Attention of many rows over a paged cache (chunks, prompts) on the 5th-generation tensor cores.
//
// A CTA takes two tiles of up to 128 rows (row = new token x query head of one key head, heads of a token side by
// side, so all rows share K and V) and walks the keys in tiles of 128:
//   * warp 9        copies K and V tiles page by page by TMA into a ring (and prefetches the page table), and zeroes the
//                   values behind the context's end (they may be anything, and 0 x NaN is NaN);
//   * warps 10..15  Q8_0 only: int8 tiles and their scales -> f16 operand tiles;
//   * warp 8        one lane issues tcgen05.mma: S_t = Q_t K^T (both from shared memory), O_t += P_t V (P from TMEM);
//   * warps 0..3 and 4..7  softmax of tile 0 and of tile 1, a thread per row: S from TMEM, running maximum and sum in
//                   registers, P back into S's columns (head dimension 64: into columns of its own, so that the next S
//                   need not wait for the product), and the division at the end. The two tiles take turns at the
//                   exponentials: while one's are computed the tensor core works on the other.
// O is rescaled only where a row's maximum grew by more than 2^8 (weights and their sum then stay within f16 and
// f32, and the quotient is the same); a thread owns its row, so that costs the warp that needs it 2 x D columns of TMEM.
// Rows to TMEM lanes: softmax thread r of a tile is lane r. Order of the MMAs, where P shares S's columns: PV of a tile is
// issued before the next S of that tile, and a commit covers all MMAs before it: a full S says that O is complete.
#include "attend.cuh"
#include "attend_launch.h"
#include "tc_common.cuh"
#include "turq_internal.h"

namespace turq {

constexpr int TILE_M = 128, TILE_N = 128;
constexpr int POLY_OF = 8;
constexpr int CONVERT = 192;  // threads that turn int8 into f16

template <int D, bool Q8> struct TileGeomA {
  static constexpr int HALVES = D / 64;
  static constexpr int OPERAND = TILE_N * D * 2;      // a tile of K, V or Q: blocks of 64 columns, 128 rows of 128 bytes each
  static constexpr int STAGES = Q8 ? 3 : (D == 128 ? 4 : 8);
  static constexpr int RAW = Q8 ? TILE_N * D + 1024 : 0;  // int8 rows, scales behind them (1024 bytes of alignment, TILE_N x D / 16 of scales)
  static constexpr int RAW_STAGES = Q8 ? 3 : 0;
  static constexpr int THREADS = Q8 ? 512 : 384;
  static constexpr int REG_SOFT = Q8 ? 192 : 208, REG_REST = Q8 ? 64 : 88;
  static constexpr int SMEM = 2 * OPERAND + STAGES * OPERAND + RAW_STAGES * RAW + 1024;
  static_assert(256 * REG_SOFT + (THREADS - 256) * REG_REST <= THREADS * (Q8 ? 128 : 168), "registers of the launch");
};

__device__ __forceinline__ void tmem_ld32(float* v, uint32_t addr) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,"
      "%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
        "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]),
        "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_ld16(float* v, uint32_t addr) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
                 "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(addr));
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
               "r"(r[14]), "r"(r[15])
               : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(s_u32(bar)) : "memory");
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t acc) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(da), "l"(db),
               "r"(idesc), "r"(acc) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t db, uint32_t idesc, uint32_t acc) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(db),
               "r"(idesc), "r"(acc) : "memory");
}
// The largest of three, one instruction.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// Two f32 at a time, one instruction.
__device__ __forceinline__ uint64_t f2(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void un2(uint64_t v, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// 2^x of two f32 on the FMA units: x = n + f with n the nearest whole number (Cody and Waite; adding 1.5 x 2^23 rounds), 2^f by the
// polynomial of degree 3 that is off by least, relative, on [-1/2, 1/2] (2^-13.7; fitted by Remez' exchange), times 2^n, whose exponent n + 127
// the rounding leaves in the lowest bits. n = -127, where x is held, has the bits of zero: -inf gives 0. NaN stays.
__device__ __forceinline__ float at_least(float x, float low) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(low));
  return r;
}
__device__ __forceinline__ void ex2_pair(uint64_t v, float& x, float& y) {
  un2(v, x, y);
  const uint64_t big = f2(12583039.f, 12583039.f), less = f2(-12583039.f, -12583039.f), one = f2(-1.f, -1.f);
  v = f2(at_least(x, -127.f), at_least(y, -127.f));
  const uint64_t t = add2(v, big);
  const uint64_t f = fma2(add2(t, less), one, v);
  uint64_t p = fma2(f, f2(0.05517166852951050f, 0.05517166852951050f), f2(0.2426111251115799f, 0.2426111251115799f));
  p = fma2(p, f, f2(0.6932609677314758f, 0.6932609677314758f));
  p = fma2(p, f, f2(0.9999280571937561f, 0.9999280571937561f));
  float tx, ty;
  un2(t, tx, ty);
  un2(mul2(p, f2(__int_as_float(__float_as_int(tx) << 23), __int_as_float(__float_as_int(ty) << 23))), x, y);
}

// Bounded: after an expiry the abort flag ends every further wait, and what a loop then does stays within its buffers.
// (In line: a call would not fit the uneven split of registers.)
__device__ __forceinline__ void tile_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  if (!bar_try(bar, parity)) {
    const long long t0 = clock64();
    while (!bar_try(bar, parity)) {
      if (*abort_flag || clock64() - t0 > TC_WAIT_CYCLES) {
        *abort_flag = 1;
        break;
      }
    }
  }
  __syncwarp();  // what follows is done by the warp as one
}

// The 128 threads of a row tile's softmax.
__device__ __forceinline__ void tile_sync(int id) { asm volatile("bar.sync %0, 128;" ::"r"(id) : "memory"); }

__device__ __forceinline__ void turn_wait(int id) { asm volatile("bar.sync %0, 256;" ::"r"(id) : "memory"); }
__device__ __forceinline__ void turn_give(int id) { asm volatile("bar.arrive %0, 256;" ::"r"(id) : "memory"); }

struct TileMaps { CUtensorMap k, v; };

struct Work {
  Span sp;
  int seq, head, tok0, live;     // first new token of the CTA; whether there is any work
  int id, split, splits;         // (index of the tile among those of the call) x heads + head; which piece of its keys
  int begin, end;                // key tiles
};

// What a sequence asks of this kernel: pairs of row tiles, and the most key tiles of one.
struct Ask { int tiles, iters; };
__device__ __forceinline__ Ask ask_of(const AttendArgs& a, const Span& sp, int tokens_per_cta) {
  Ask k{0, 0};
  if (sp.n * a.group > TOKEN_ROWS) {
    k.tiles = ((int)sp.n + tokens_per_cta - 1) / tokens_per_cta;
    k.iters = ((int)sp.ctx + TILE_N - 1) / TILE_N;
  }
  return k;
}

// Block b takes piece b % splits of tile b / splits, a sequence's last (longest) tiles first. How many pieces follows from the tiles
// that there really are, the same for every block. One warp.
__device__ __forceinline__ void find_work(const AttendArgs& a, int tokens_per_cta, Work* w, int lane) {
  if (lane == 0) w->live = 0;
  int total = 0, iters = 0;
  Span sp{};
  Ask ask{0, 0};
  for (int s0 = 0; s0 < a.n_seqs; s0 += 32) {
    ask = Ask{0, 0};
    if (s0 + lane < a.n_seqs) {
      sp = span_of(a, s0 + lane);
      ask = ask_of(a, sp, tokens_per_cta);
    }
    total += __reduce_add_sync(0xFFFFFFFFu, ask.tiles);
    iters = max(iters, __reduce_max_sync(0xFFFFFFFFu, ask.iters));
  }
  const int heads = a.cache.n_heads, ctas = total * heads;
  // (lane i asks for i + 1 pieces)
  const uint32_t mine = (uint32_t)min(tile_split_cost(lane + 1, ctas, iters, a.tile_pieces, a.sms), (int64_t)0x3FFFFFF) << 5 | (uint32_t)lane;
  const int splits = (int)(__reduce_min_sync(0xFFFFFFFFu, mine) & 31u) + 1;
  if (a.tile_pieces > 0 && blockIdx.x == 0 && lane == 0) {
    a.tile_head[0] = splits;
    a.tile_head[1] = ctas;
  }
  const int id = (int)blockIdx.x / splits;
  if (id >= ctas) return;
  int want = id / heads;
  for (int s0 = 0; s0 < a.n_seqs; s0 += 32) {
    if (a.n_seqs > 32) {  // (up to 32: still in registers)
      ask = Ask{0, 0};
      if (s0 + lane < a.n_seqs) {
        sp = span_of(a, s0 + lane);
        ask = ask_of(a, sp, tokens_per_cta);
      }
    }
    int upto = ask.tiles;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int t = __shfl_up_sync(0xFFFFFFFFu, upto, d);
      if (lane >= d) upto += t;
    }
    const int here = __shfl_sync(0xFFFFFFFFu, upto, 31);
    if (want < here) {
      if (want < upto && want >= upto - ask.tiles) {
        const int tile = ask.tiles - 1 - (want - (upto - ask.tiles));
        w->sp = sp;
        w->seq = s0 + lane;
        w->head = id % heads;
        w->tok0 = tile * tokens_per_cta;
        w->id = id;
        w->split = (int)blockIdx.x % splits;
        w->splits = splits;
        const int64_t last = min(sp.n, (int64_t)w->tok0 + tokens_per_cta) - 1;
        const int keys = (int)min(sp.ctx, keys_seen(sp, last, a.causal));
        const int n = (keys + TILE_N - 1) / TILE_N;
        w->begin = n * w->split / splits;  // (32 bits hold 2^23 key tiles x 32)
        w->end = n * (w->split + 1) / splits;
        w->live = 1;
      }
      return;
    }
    want -= here;
  }
}

template <int D, bool Q8, bool BF>
__global__ void __launch_bounds__((TileGeomA<D, Q8>::THREADS), 1)
attend_tiles_kernel(const __grid_constant__ TileMaps maps, const __grid_constant__ AttendArgs a) {
  using G = TileGeomA<D, Q8>;
  constexpr int ST = G::STAGES, OP = G::OPERAND, HB = TILE_N * 128;  // HB: one 64-column block
  constexpr int POLY = D == 128 ? 0 : 1;
  constexpr bool APART = D == 64;                                     // P has columns of its own: S may be written again once it is read
  constexpr uint32_t COL_S = 0, COL_O = 256, COL_P = APART ? 384 : 0;                          // S of tile t at 128 t, O at 256 + D t, P at 384 + 64 t or where S was
  extern __shared__ uint8_t raw[];
  __shared__ __align__(8) uint64_t q_full[2], kv_full[8], kv_empty[8], s_full[2], p_full[2][2], s_read[2], o_full[2], v_fixed, raw_full[3], raw_empty[3];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word;
  __shared__ Work work;
  __shared__ float row_up[2][TILE_M];  // the power of two that a row of Q was divided by
  __shared__ int row_at[2][TILE_M];    // a row's token (of the tile) and, above 8 bits, its head (of the group); -1: no such row
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t smem = (s_u32(raw) + 1023u) & ~1023u;
  const uint32_t sQ = smem, sKV = smem + 2 * OP, sRaw = sKV + ST * OP;
  volatile int* const abort_flag = &abort_word;
  const int tpt = TILE_M / a.group;  // tokens of a tile

  if (threadIdx.x == 32) {
    for (int i = 0; i < 2; i++) { bar_init(&q_full[i], 4); bar_init(&s_full[i], 1); bar_init(&p_full[i][0], 4); bar_init(&p_full[i][1], 4); bar_init(&s_read[i], 4); bar_init(&o_full[i], 1); }
    for (int i = 0; i < ST; i++) { bar_init(&kv_full[i], Q8 ? CONVERT / 32 : 1); bar_init(&kv_empty[i], 1); }
    bar_init(&v_fixed, 1);
    for (int i = 0; i < 3; i++) { bar_init(&raw_full[i], 33); bar_init(&raw_empty[i], CONVERT / 32); }
    abort_word = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (threadIdx.x == 288) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.k) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.v) : "memory");
  }
  // launched behind its predecessor's last block: everything that kernels before it wrote is read from here on
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (warp == 0) find_work(a, 2 * tpt, &work, lane);
  __syncthreads();
  if (!work.live) return;  // (before anything is allocated: a call has blocks for the most tiles and pieces that there may be)
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s_u32(&tmem_slot)), "n"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = tmem_slot;
  const Span sp = work.sp;
  const int seq = work.seq, head = work.head, begin = work.begin, n_iter = work.end - work.begin;
  const int tiles = sp.n - work.tok0 > tpt ? 2 : 1;  // row tiles with rows
  const int ctx = (int)sp.ctx;

  if (warp < 8) {
    // ---------------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(G::REG_SOFT));
    const int t = warp >> 2, r = threadIdx.x & 127;
    // row / group = row x per16 >> 16 for rows and groups up to 128
    const int rt = (int)((r * (65535u / (uint32_t)a.group + 1u)) >> 16), tok = work.tok0 + t * tpt + rt;
    const bool live = rt < tpt && tok < sp.n;
    row_at[t][r] = live ? rt | (r - rt * a.group) << 8 : -1;  // once, and not for every 16 bytes that come or go
    tile_sync(1 + t);
    // Q into the operand layout, D / 8 lanes a row (a row a thread, every load would touch 32 lines: 7300 cycles against 3500); on f16
    // caches a bf16 row by the power of two that its largest element fits. Not where there is no key: the result goes out through the same
    // memory, and nothing between the two would wait for the last thread to have brought its part of Q.
    if (t < tiles && n_iter > 0) {
      constexpr int L = D / 8, ROWS = TILE_M / L;  // rows of a pass
      const int ch = r % L;
      const uint16_t* const qp = a.q + (sp.first + work.tok0 + t * tpt) * a.q_stride + (int64_t)head * a.group * D + 8 * ch;
      uint4 w[L];
#pragma unroll
      for (int i = 0; i < L; i++) {
        const int at = row_at[t][i * ROWS + r / L];
        w[i] = at >= 0 ? *reinterpret_cast<const uint4*>(qp + (at & 255) * a.q_stride + (at >> 8) * D) : make_uint4(0, 0, 0, 0);
      }
      const bool convert = !BF && a.q_bf16;
#pragma unroll
      for (int i = 0; i < L; i++) {
        const int row = i * ROWS + r / L;
        if (convert) {
          uint32_t* x = reinterpret_cast<uint32_t*>(&w[i]);
          uint32_t top = 0;
#pragma unroll
          for (int e = 0; e < 4; e++) top = max(top, max(x[e] & 0x7FFFu, (x[e] >> 16) & 0x7FFFu));
#pragma unroll
          for (int d = 1; d < L; d <<= 1) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
          const int e2 = min(max((int)(top >> 7) - 127, -126), 126);
          const float down = __uint_as_float((uint32_t)(127 - e2) << 23);
          if (ch == 0) row_up[t][row] = __uint_as_float((uint32_t)(127 + e2) << 23);
#pragma unroll
          for (int e = 0; e < 4; e++) x[e] = pack16<false>(__uint_as_float(x[e] << 16) * down, __uint_as_float(x[e] & 0xFFFF0000u) * down);
        }
        asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(sQ + t * OP + (ch >> 3) * HB + row * 128 + (((ch & 7) ^ (row & 7)) << 4)), "r"(w[i].x),
                     "r"(w[i].y), "r"(w[i].z), "r"(w[i].w) : "memory");
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) bar_arrive(&q_full[t]);
      if (convert) tile_sync(1 + t);
    }
    const float mul = !BF && a.q_bf16 && t < tiles && n_iter > 0 ? row_mul(a, row_up[t][r]) : a.scale_log2;
    const int seen = live ? (int)min(sp.ctx, keys_seen(sp, tok, a.causal)) : INT32_MAX;  // rows that do not exist ask for no mask
    // keys that every row of the warp sees
    int least = seen;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) least = min(least, __shfl_xor_sync(0xFFFFFFFFu, least, d));
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // TMEM lane 32 (warp % 4) in the address' upper half
    const uint32_t tS = tmem + lanes + COL_S + 128 * t, tO = tmem + lanes + COL_O + D * t, tP = APART ? tmem + lanes + COL_P + 64 * t : tS;
    float m = -INFINITY, l = 0.f;  // maximum in units of S, as last subtracted; sum of the weights
    float above = 0.f, sub = 0.f;  // maxima above this one are taken over: their weights would be 2^8 and more; maximum x mul
    if (t >= tiles && work.splits > 1 && work.split == 0) a.tile_rows[(int64_t)work.id * (2 * TILE_M) + TILE_M * t + r] = -1;
    if (t < tiles) {
      if (tiles == 2 && t == 1 && n_iter > 0) turn_give(3);
      for (int j = 0; j < n_iter; j++) {
        float s[TILE_N];
        tile_wait(&s_full[t], j & 1, abort_flag);
        tc_after();
        tmem_ld32(s, tS);
        tmem_ld32(s + 32, tS + 32);
        tmem_wait_ld();
        tmem_ld32(s + 64, tS + 64);
        tmem_ld32(s + 96, tS + 96);
        const int k0 = (begin + j) * TILE_N;
        float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        auto largest = [&](int from) {
#pragma unroll
          for (int i = from; i < from + 64; i += 8) {
#pragma unroll
            for (int e = 0; e < 4; e++) top[e] = max3(top[e], s[i + 2 * e], s[i + 2 * e + 1]);
          }
        };
        if (k0 + TILE_N > least) {
          tmem_wait_ld();
          const int lim = seen - k0;
#pragma unroll
          for (int i = 0; i < TILE_N; i++) s[i] = i < lim ? s[i] : -INFINITY;
        }
        largest(0);
        tmem_wait_ld();
        if (APART) {  // all of S is in registers
          tc_before();
          __syncwarp();
          if (lane == 0) bar_arrive(&s_read[t]);
        }
        largest(64);
        const float mt = fmaxf(max3(top[0], top[1], top[2]), top[3]);
        if (j == 0 || __any_sync(0xFFFFFFFFu, mt > above)) {
          if (j == 0) {
            m = mt;
          } else {
            if (APART) {  // otherwise a full S says so
              tile_wait(&o_full[t], (j - 1) & 1, abort_flag);
              tc_after();
            }
            const float m2 = fmaxf(m, mt), f = m2 == -INFINITY ? 1.f : ex2((m - m2) * mul);  // m = -inf: 0 of nothing
            m = m2;
            l *= f;
            float o[16];
#pragma unroll 1
            for (int i = 0; i < D / 16; i++) {
              tmem_ld16(o, tO + 16 * i);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; e++) o[e] *= f;
              tmem_st16(tO + 16 * i, reinterpret_cast<const uint32_t*>(o));
            }
            tmem_wait_st();
          }
          // A weight's exponent is one FMA, s x mul - sub: off by what m x mul loses in rounding, the same for all weights until m changes. From
          // 2^10 on that is 2^-14 and more: such rows (above = m says so) subtract m from their scores before they multiply. Where all rows
          // do, a prompt of 4096 tokens takes a fifth longer (132 us, so 160; head dimension 64 135 and 162), where none does as long.
          sub = m == -INFINITY ? 0.f : m * mul;
          above = m + 8.f / mul;
          if (fabsf(sub) > 1024.f) {
            sub = 0.f;
            above = m;
          }
        }
        if (APART && j > 0) {  // the last weights' product has read them
          tile_wait(&o_full[t], (j - 1) & 1, abort_flag);
          tc_after();
        }
        if (above == m) {  // (or no key seen yet)
          const float mm = m == -INFINITY ? 0.f : m;
#pragma unroll
          for (int i = 0; i < TILE_N; i++) s[i] -= mm;
        }
        // The tiles take turns at the exponentials, which one warp a scheduler can keep busy: together both would take as long as one behind
        // the other, and then both wait for the tensor core at once.
        if (tiles == 2) turn_wait(3 + t);
        const uint64_t times = f2(mul, mul), less = f2(-sub, -sub);
        uint64_t sum[2] = {0, 0};
#pragma unroll
        for (int h = 0; h < TILE_N / 32; h++) {
          uint32_t p[16];
#pragma unroll
          for (int i = 0; i < 16; i++) {
            float x, y;
            const uint64_t e = fma2(f2(s[32 * h + 2 * i], s[32 * h + 2 * i + 1]), times, less);
            if (i % POLY_OF < POLY) {
              ex2_pair(e, x, y);
            } else {
              un2(e, x, y);
              x = ex2(x);
              y = ex2(y);
            }
            sum[i & 1] = add2(sum[i & 1], f2(x, y));
            p[i] = pack16<BF>(x, y);
          }
          tmem_st16(tP + 16 * h, p);
          if (h % 2 == 1) {  // half of the weights: their product may start
            tmem_wait_st();
            tc_before();
            __syncwarp();
            if (lane == 0) bar_arrive(&p_full[t][h / 2]);
          }
        }
        float s0, s1;
        un2(add2(sum[0], sum[1]), s0, s1);
        l += s0 + s1;
        if (tiles == 2 && (t == 0 || j + 1 < n_iter)) turn_give(3 + (t ^ 1));
      }
      if (m == -INFINITY) l = 0.f;  // a row that saw no key
      if (n_iter > 0) {
        tile_wait(&o_full[t], APART ? (n_iter - 1) & 1 : 0, abort_flag);
        tc_after();
      }
      const bool pieces = work.splits > 1;
      const float inv = pieces ? 1.f : l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;  // a row that sees no key gives zeros; NaN stays
      const int64_t piece0 = (int64_t)blockIdx.x * (2 * TILE_M) + TILE_M * t;
      const int64_t out0 = ((work.sp.first + work.tok0 + t * tpt) * a.hq + work.head * a.group) * D;  // of the tile's first row
      if (pieces) {
        a.tile_ml[piece0 + r] = make_float2(joined_max(m, mul), l);
        if (work.split == 0) {
          const int at = row_at[t][r];
          a.tile_rows[(int64_t)work.id * (2 * TILE_M) + TILE_M * t + r] = at < 0 ? -1 : out0 + ((int64_t)(at & 255) * a.hq + (at >> 8)) * D;
        }
      }
      // Rows go out through shared memory, a warp whole rows, for the same reason as Q comes in so (6400 cycles against 3500): through this
      // tile's part of Q, which nothing reads any more, in one go or in two for 32 bits.
      const bool wide = pieces || a.out_dtype == TURQ_F32;
      const uint32_t stage = sQ + t * OP;
      constexpr int L = D / 8;  // 16-byte chunks of a staged row
      const bool store = !*abort_flag;
      const int ch = r % L, shift = wide ? 2 : 1;
      uint8_t* const to = (pieces ? reinterpret_cast<uint8_t*>(a.tile_part + piece0 * D) : static_cast<uint8_t*>(a.out) + (out0 << shift)) + 16 * ch;
      const int64_t token_bytes = (int64_t)a.hq * D << shift;
      auto flush = [&](int pass) {
        tile_sync(1 + t);
#pragma unroll 4
        for (int i = 0; i < L; i++) {
          const int row = i * (TILE_M / L) + r / L, at = row_at[t][row];
          uint4 w;
          asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "r"(stage + row * 2 * D + ((ch ^ (row & 7)) << 4)));
          uint8_t* const p = to + pass * 2 * D + (pieces ? (int64_t)(row * 4 * D) : (at & 255) * token_bytes + (((at >> 8) * D) << shift));
          if (at >= 0 && store) *reinterpret_cast<uint4*>(p) = w;
        }
        tile_sync(1 + t);
      };
#pragma unroll 1
      for (int i = 0; i < D / 32; i++) {
        float o[32];
        if (n_iter > 0) {
          tmem_ld32(o, tO + 32 * i);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int e = 0; e < 32; e++) o[e] = 0.f;
        }
#pragma unroll
        for (int e = 0; e < 32; e++) o[e] *= inv;
        if (wide) {
          const int c = i % (D / 64);
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            asm volatile("st.shared.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(stage + r * 2 * D + (((8 * c + e / 4) ^ (r & 7)) << 4)), "f"(o[e]), "f"(o[e + 1]),
                         "f"(o[e + 2]), "f"(o[e + 3]) : "memory");
          if (c == D / 64 - 1) flush(i / (D / 64));
        } else {
          const bool bf = a.out_dtype == TURQ_BF16;
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            uint32_t w[4];
#pragma unroll
            for (int q = 0; q < 4; q++) w[q] = bf ? pack16<true>(o[e + 2 * q], o[e + 2 * q + 1]) : pack16<false>(o[e + 2 * q], o[e + 2 * q + 1]);
            asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(stage + r * 2 * D + (((4 * i + e / 8) ^ (r & 7)) << 4)), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                         "r"(w[3]) : "memory");
          }
          if (i == D / 32 - 1) flush(0);
        }
        __syncwarp();
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(G::REG_REST));
    if (warp == 8) {
      // -------------------------------------------------------------- MMA
      constexpr uint32_t type = BF ? (1u << 7) | (1u << 10) : 0u;
      constexpr uint32_t id_qk = (1u << 4) | type | ((TILE_N >> 3) << 17) | ((TILE_M >> 4) << 24);
      constexpr uint32_t id_pv = (1u << 4) | type | (1u << 16) | ((D >> 3) << 17) | ((TILE_M >> 4) << 24);  // V: the columns lie side by side
      // rows of 128 swizzled bytes, eight of them 1024 bytes apart; for V also the step from one block of 64 columns to the next
      constexpr uint64_t k_hi = (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
      constexpr uint64_t v_hi = ((uint64_t)(HB >> 4) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
      const uint32_t q_lo = (sQ & 0x3FFFFu) >> 4, kv_lo = (sKV & 0x3FFFFu) >> 4;
      const bool issuer = elect_one();
      auto qk = [&](int t, int stage) {
        if (!issuer) return;
#pragma unroll
        for (int i = 0; i < D / 16; i++) {
          const uint32_t off = (uint32_t)((i >> 2) * (HB >> 4) + 2 * (i & 3));
          mma_ss(tmem + COL_S + 128 * t, k_hi | (uint64_t)(q_lo + t * (OP >> 4) + off), k_hi | (uint64_t)(kv_lo + stage * (OP >> 4) + off), id_qk, i > 0);
        }
        tc_commit(&s_full[t]);
      };
      auto pv = [&](int t, int stage, int half, bool first) {
        if (!issuer) return;
#pragma unroll
        for (int i = TILE_N / 32 * half; i < TILE_N / 32 * (half + 1); i++)
          mma_ts(tmem + COL_O + D * t, tmem + (APART ? COL_P + 64 * t : COL_S + 128 * t) + 8 * i, v_hi | (uint64_t)(kv_lo + stage * (OP >> 4) + 128 * i), id_pv, !first || i > 0);
      };
      if (n_iter > 0) {
        int ks = 0, vs = 1 % ST;  // stages: K_0, V_0, K_1, V_1, ...
        uint32_t kp = 0, vp = 1 >= ST;
        auto next = [](int& s, uint32_t& p) {
          s += 2;
          if (s >= ST) { s -= ST; p ^= 1u; }
        };
        for (int t = 0; t < tiles; t++) tile_wait(&q_full[t], 0, abort_flag);
        tile_wait(&kv_full[ks], kp, abort_flag);
        tc_after();
        for (int t = 0; t < tiles; t++) qk(t, ks);
        if (issuer) tc_commit(&kv_empty[ks]);
        next(ks, kp);
        for (int j = 0; j < n_iter; j++) {
          if (__any_sync(0xFFFFFFFFu, *abort_flag)) break;
          const bool more = j + 1 < n_iter;
          if (!APART) tile_wait(&kv_full[vs], vp, abort_flag);
          if (!APART && !Q8 && (begin + j + 1) * TILE_N > ctx) tile_wait(&v_fixed, 0, abort_flag);
          if (APART && more) {  // the next S as soon as the last is read
            tile_wait(&kv_full[ks], kp, abort_flag);
            for (int t = 0; t < tiles; t++) {
              tile_wait(&s_read[t], j & 1, abort_flag);
              tc_after();
              qk(t, ks);
            }
            if (issuer) tc_commit(&kv_empty[ks]);
          }
          if (APART) tile_wait(&kv_full[vs], vp, abort_flag);
          if (APART && !Q8 && (begin + j + 1) * TILE_N > ctx) tile_wait(&v_fixed, 0, abort_flag);
          for (int t = 0; t < tiles; t++) {
#pragma unroll
            for (int half = 0; half < 2; half++) {
              tile_wait(&p_full[t][half], j & 1, abort_flag);
              tc_after();
              pv(t, vs, half, j == 0);
            }
            if (issuer && (APART || !more)) tc_commit(&o_full[t]);
            if (t == tiles - 1 && issuer) tc_commit(&kv_empty[vs]);
            if (!APART && more) {
              if (t == 0) {
                tile_wait(&kv_full[ks], kp, abort_flag);
                tc_after();
              }
              qk(t, ks);
              if (t == tiles - 1 && issuer) tc_commit(&kv_empty[ks]);
            }
          }
          next(vs, vp);
          next(ks, kp);
        }
      }
      __syncwarp();
    } else if (warp == 9) {
      // -------------------------------------------------------------- copies
      // lane i: the page that key 16 i of the tile begins (boxes of a page's tokens, 16 to 128 of them)
      const int box_shift = min(a.cache.page_shift, 7), box = 1 << box_shift, boxes = TILE_N >> box_shift;
      const int32_t* table = a.page_table + seq * a.table_stride;
      auto page_of = [&](int j) {  // z coordinate of this lane's box in key tile begin + j; -1: behind the context
        const int64_t key = (int64_t)(begin + j) * TILE_N + lane * box;
        if (lane >= boxes || j >= n_iter || key >= ctx) return -1;
        const int64_t p = table[key >> a.cache.page_shift];
        const bool known = p >= 0 && p < a.cache.n_pages;
        if (!known) report(a.status, TURQ_E_INVALID_ARG);
        return known ? (int)(p * a.cache.n_heads + head) : (int)(a.cache.n_pages * a.cache.n_heads);
      };
      int stage = 0, z = page_of(0);
      const int pages_end = (int)(a.cache.n_pages * a.cache.n_heads);
      uint32_t ph = 0;
      for (int j = 0; j < n_iter; j++) {
        if (__any_sync(0xFFFFFFFFu, *abort_flag)) break;
        const int z2 = page_of(j + 1);
        const int y = ((begin + j) * TILE_N + lane * box) & (a.cache.page_size - 1);
        const int n = __popc(__ballot_sync(0xFFFFFFFFu, z >= 0));
#pragma unroll
        for (int kv = 0; kv < 2; kv++) {
          if (!Q8) {
            tile_wait(&kv_empty[stage], ph ^ 1u, abort_flag);
            const uint32_t bar = s_u32(&kv_full[stage]), at = sKV + stage * OP + lane * box * 128;
            if (lane == 0) bar_expect_tx(&kv_full[stage], n * box * D * 2);
            __syncwarp();
            if (z >= 0) {
#pragma unroll
              for (int h = 0; h < G::HALVES; h++) copy_box3(at + h * HB, kv ? &maps.v : &maps.k, 64 * h, y, z, bar);
            }
            if (++stage == ST) { stage = 0; ph ^= 1u; }
          } else {
            tile_wait(&raw_empty[stage], ph ^ 1u, abort_flag);
            const uint32_t bar = s_u32(&raw_full[stage]), at = sRaw + stage * G::RAW;
            if (lane == 0) bar_expect_tx(&raw_full[stage], n * box * D);
            __syncwarp();
            if (z >= 0) copy_box3(at + lane * box * D, kv ? &maps.v : &maps.k, 0, y, z, bar);
            // Scales are too small for boxes (16 of 64 bytes a tile; with pages of 16 tokens head dimension 64 then waits for the copies' rate:
            // one prompt of 8192 tokens 618 us, 541 this way): 16 bytes at a time, zeros where there is no page.
            const __half* const from = kv ? a.cache.vs : a.cache.ks;
#pragma unroll
            for (int i = 0; i < D / 64; i++) {
              constexpr int PER = 256 / D;  // keys whose scales are 16 bytes
              const int key = (i * 32 + lane) * PER, zk = __shfl_sync(0xFFFFFFFFu, z, key >> box_shift);
              const bool have = zk >= 0 && zk < pages_end;
              const __half* const src = from + ((int64_t)(have ? zk : 0) * a.cache.page_size + (((begin + j) * TILE_N + key) & (a.cache.page_size - 1))) * (D / 32);
              asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(sRaw + stage * G::RAW + TILE_N * D + key * (D / 16)), "l"(src), "r"(have ? 16 : 0)
                           : "memory");
            }
            asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(bar) : "memory");
            if (++stage == G::RAW_STAGES) { stage = 0; ph ^= 1u; }
          }
        }
        z = z2;
      }
      if (Q8) asm volatile("cp.async.wait_all;" ::: "memory");  // (after a wait that ran out: nothing is on its way when the block ends)
      // Values behind the context's end. Only this warp can wait for a phase of kv_full that is many on: it knows that the one
      // before is over, as its own wait for the empty stage said.
      if (!Q8 && n_iter > 0 && (begin + n_iter) * TILE_N > ctx) {
        const int i = 2 * (n_iter - 1) + 1, last = i % ST, from = ctx - (begin + n_iter - 1) * TILE_N;
        tile_wait(&kv_full[last], (i / ST) & 1, abort_flag);
        for (int c = lane; c < (TILE_N - from) * (D / 8); c += 32) {
          const int row = from + c / (D / 8), ch = c % (D / 8);
          asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(sKV + last * OP + (ch >> 3) * HB + row * 128 + ((ch & 7) << 4)), "r"(0u) : "memory");
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) bar_arrive(&v_fixed);
      }
    } else if (Q8) {
      // -------------------------------------------------------------- int8 -> f16 operand tiles
      const int id0 = threadIdx.x - 320;
      int rs = 0, stage = 0;
      uint32_t rp = 0, ph = 0;
      __half2 largest = __float2half2_rn(0.f);  // of the scales of keys and values of the context
      for (int j = 0; j < 2 * n_iter; j++) {
        const int keys = ctx - (begin + (j >> 1)) * TILE_N;  // that exist, of this tile
        tile_wait(&raw_full[rs], rp, abort_flag);
        tile_wait(&kv_empty[stage], ph ^ 1u, abort_flag);
        const uint32_t src = sRaw + rs * G::RAW, dst = sKV + stage * OP;
#pragma unroll 3
        for (int i = 0; i < (TILE_N * D / 16 + CONVERT - 1) / CONVERT; i++) {
          const int id = i * CONVERT + id0, row = id / (D / 16), ch = id % (D / 16);
          if (id >= TILE_N * D / 16) break;
          uint4 w;
          asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "r"(src + id * 16));
          uint16_t sc;
          asm volatile("ld.shared.u16 %0, [%1];" : "=h"(sc) : "r"(src + TILE_N * D + (row * (D / 32) + (ch >> 1)) * 2));
          if (row >= keys) sc = 0;  // anything may lie behind the context's end
          const __half2 scale = __half2half2(__ushort_as_half(sc));
          uint32_t h[8];
          halves_of(w.x, scale, h[0], h[1]);
          halves_of(w.y, scale, h[2], h[3]);
          halves_of(w.z, scale, h[4], h[5]);
          halves_of(w.w, scale, h[6], h[7]);
          largest = __hmax2(largest, __habs2(scale));
          const uint32_t to = dst + (ch >> 2) * HB + row * 128;
          const int c0 = ((2 * ch) & 7) ^ (row & 7), c1 = ((2 * ch + 1) & 7) ^ (row & 7);
          asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(to + (c0 << 4)), "r"(h[0]), "r"(h[1]), "r"(h[2]), "r"(h[3]) : "memory");
          asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(to + (c1 << 4)), "r"(h[4]), "r"(h[5]), "r"(h[6]), "r"(h[7]) : "memory");
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
          bar_arrive(&kv_full[stage]);
          bar_arrive(&raw_empty[rs]);
        }
        if (++rs == G::RAW_STAGES) { rs = 0; rp ^= 1u; }
        if (++stage == ST) { stage = 0; ph ^= 1u; }
      }
      report_beyond_f16(a, largest);
    }
  }
  tc_before();
  __syncthreads();
  if (*abort_flag) {
    // a wait ran out: give copies still in flight time to land in this CTA's shared memory
    for (int i = 0; i < 64; i++) __nanosleep(2000);
    if (threadIdx.x == 0) report(a.status, TURQ_E_TIMEOUT);
  }
  if (warp == 8) {
    tc_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(512) : "memory");
  }
}

// The pieces of rows whose keys were cut, in their order: a warp per row, 32 rows a block.
template <int D>
__global__ void __launch_bounds__(256) join_tiles_kernel(const __grid_constant__ AttendArgs a) {
  constexpr int E = D / 32;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int splits = a.tile_head[0], lane = threadIdx.x & 31;
  if (splits <= 1 || (int)blockIdx.x >= a.tile_head[1]) return;
  for (int i = 0; i < 4; i++) {
    const int r = blockIdx.y * 32 + (threadIdx.x >> 5) * 4 + i;
    const int64_t out = a.tile_rows[(int64_t)blockIdx.x * (2 * TILE_M) + r];
    if (out < 0) continue;
    const int64_t piece = (int64_t)blockIdx.x * splits * (2 * TILE_M) + r;
    float mm = -INFINITY, ll = 0.f, o[E];
#pragma unroll
    for (int e = 0; e < E; e++) o[e] = 0.f;
    const float2 mine = lane < splits ? a.tile_ml[piece + (int64_t)lane * (2 * TILE_M)] : make_float2(-INFINITY, 0.f);  // at most 32 of them
    mm = mine.x;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xFFFFFFFFu, mm, d));
    const float f = mm == -INFINITY ? 0.f : ex2((mine.x - mm) * joined_factor(a)), fl = f * mine.y;
#pragma unroll 4
    for (int k = 0; k < splits; k++) {
      const float w = __shfl_sync(0xFFFFFFFFu, f, k);
      const float* p = a.tile_part + (piece + (int64_t)k * (2 * TILE_M)) * D + lane * E;
      ll += __shfl_sync(0xFFFFFFFFu, fl, k);
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        const float2 v = *reinterpret_cast<const float2*>(p + e);
        o[e] += w * v.x;
        o[e + 1] += w * v.y;
      }
    }
    const float inv = ll > 0.f ? 1.f / ll : ll == 0.f ? 0.f : ll;
#pragma unroll
    for (int e = 0; e < E; e += 2) store_out2(a.out, a.out_dtype, out + lane * E + e, o[e] * inv, o[e + 1] * inv);
  }
}

template <int D, bool Q8, bool BF>
static cudaError_t launch_tiles(const turq_kv_cache* kc, const AttendArgs& a, unsigned blocks, cudaStream_t s) {
  using G = TileGeomA<D, Q8>;
  static PerDeviceOnce configured;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (!configured.done(dev)) {
    e = cudaFuncSetAttribute(attend_tiles_kernel<D, Q8, BF>, cudaFuncAttributeMaxDynamicSharedMemorySize, G::SMEM);
    if (e != cudaSuccess) return e;
    configured.set(dev);
  }
  const TileMaps maps{kc->k_tile, kc->v_tile};
  return launch_pdl(attend_tiles_kernel<D, Q8, BF>, dim3(blocks), dim3(G::THREADS), G::SMEM, s, maps, a);
}

cudaError_t launch_attend_tiles(const turq_kv_cache* kc, const AttendArgs& a, unsigned blocks, cudaStream_t s, int* launches) {
  (*launches)++;
  if (kc->head_dim == 128) {
    if (kc->dtype == TURQ_Q8_0) return launch_tiles<128, true, false>(kc, a, blocks, s);
    return kc->dtype == TURQ_BF16 ? launch_tiles<128, false, true>(kc, a, blocks, s) : launch_tiles<128, false, false>(kc, a, blocks, s);
  }
  if (kc->dtype == TURQ_Q8_0) return launch_tiles<64, true, false>(kc, a, blocks, s);
  return kc->dtype == TURQ_BF16 ? launch_tiles<64, false, true>(kc, a, blocks, s) : launch_tiles<64, false, false>(kc, a, blocks, s);
}

cudaError_t launch_join_tiles(const turq_kv_cache* kc, const AttendArgs& a, cudaStream_t s, int* launches) {
  (*launches)++;
  const dim3 grid((unsigned)(a.tile_pieces / 2), 2 * TILE_M / 32);  // two pieces a tile at least
  return kc->head_dim == 64 ? launch_pdl(join_tiles_kernel<64>, grid, dim3(256), 0, s, a) : launch_pdl(join_tiles_kernel<128>, grid, dim3(256), 0, s, a);
}

}  // namespace turq
