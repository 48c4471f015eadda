// Attention of single tokens (up to 16 rows = new tokens x query heads of one key head): bound by the bytes of
// K and V, which every row of a key head shares.
//
// A CTA takes one chunk (plan_token_chunk) of one key head of one sequence, its four warps every fourth step of 16 to 64
// keys. A warp copies its own steps by TMA into its own ring (no CTA-wide barrier in the loop) and keeps its own running
// maximum, sum and output; the four are joined through shared memory at the end. A context of one chunk is then finished;
// the pieces of a longer one go to the workspace and join_tokens_kernel adds them in chunk order.
//
// Products are transposed, S^T = K Q^T and O^T = V^T P^T on mma.sync m16n8k16: keys and value columns fill the 16 rows of
// the wide operand, query rows the 8 columns of the narrow one (one or two tiles of it). The rows are few, so the matrix
// rate does not matter, the accumulators stay in registers, and every key and value is brought into an operand once:
// 16-bit ones by ldmatrix, Q8_0 ones from int8 in registers. There the order of k (of the head's elements) and of m
// (of the value's columns) is the one in which a lane's 16 bytes lie: lane (g, c) multiplies bytes D/4 c .. of keys g and
// g + 8, and columns D/8 g .. of the values of its four keys.
//
// Q8_0 keys and values are rounded to f16 (2^-11 of a value, against the 2^-8 of a block's largest that the
// quantization itself costs); weights are rounded to the 16-bit type before they meet V.
#include "attend.cuh"
#include "attend_launch.h"
#include "tc_common.cuh"
#include "turq_internal.h"

namespace turq {

constexpr int TOK_WARPS = 4;

// A warp's ring: steps of 8 KB of keys and values; of 4 KB for Q8_0 where at most eight query rows leave registers for a fourth
// CTA an SM (their conversion waits for itself: 24 users at 4096 keys 66 us with three, 58 with four, two at 120000 123 and 97). Scales of
// Q8_0 lie behind the steps.
template <int D, bool Q8, int NR> struct TokGeom {
  static constexpr bool FOUR = Q8 && NR == 1;
  static constexpr int CTAS = token_ctas(Q8, NR == 1);
  static constexpr int STAGES = FOUR && D == 128 ? 3 : 2;
  static constexpr int HALF = FOUR ? 2048 : 4096;      // bytes of the keys of a step, and of its values
  static constexpr int ROW = Q8 ? D : 2 * D;           // bytes of a key
  static constexpr int KEYS = HALF / ROW;              // 16 to 64
  static constexpr int BOX = 16 * (Q8 ? D : 128);      // one copy: 16 keys of a 128-byte column block, or of int8
  static constexpr int SC = Q8 ? 16 * (D / 32) * 2 : 0;  // scales of 16 keys: 128 or 64 bytes,
  static constexpr int SC_AT = Q8 ? 128 : 0;             // each copy to a 128-byte boundary, as tensor copies ask for
  static constexpr int SCALES = KEYS / 16 * 2 * SC_AT;   // of a step
  static constexpr int RING = (STAGES * (2 * HALF + SCALES) + 1023) / 1024 * 1024;
  static constexpr int RES = D + 4;                    // floats from one result row to the next: four row pairs x eight columns meet all banks
  static_assert(RING >= 16 * RES * 4 + 128, "the ring holds a warp's result");
};

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
template <bool BF>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (BF)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void copy_box2(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
               ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}

struct TokMaps { CUtensorMap k, v, ks, vs; };

template <int D, bool Q8, bool BF, int NR /* tiles of 8 query rows */>
__global__ void __launch_bounds__(32 * TOK_WARPS, TokGeom<D, Q8, NR>::CTAS) attend_tokens_kernel(const __grid_constant__ TokMaps maps, const __grid_constant__ AttendArgs a) {
  using G = TokGeom<D, Q8, NR>;
  constexpr int TOK_STAGES = G::STAGES, KEYS = G::KEYS, KT = KEYS / 16, KS = D / 16, MT = D / 16, HALVES = Q8 ? 1 : D / 64;
  extern __shared__ uint8_t raw[];
  __shared__ __align__(8) uint64_t full[TOK_WARPS][TOK_STAGES];
  __shared__ int pages[TOKEN_CHUNK_MAX / 16];
  __shared__ int abort_flag;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  const int chunk = blockIdx.x, head = blockIdx.y, seq = blockIdx.z;
  const int64_t lo = (int64_t)chunk * a.chunk;
  const uint32_t base = (s_u32(raw) + 1023u) & ~1023u;
  const uint32_t ring = base + warp * G::RING;
  if (threadIdx.x == 0) {
    abort_flag = 0;
    asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.k) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.v) : "memory");
  }
  if (lane == 0) {
    for (int s = 0; s < TOK_STAGES; s++) bar_init(&full[warp][s], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  // Launched behind its predecessor's last block: everything that kernels before it wrote is read from here on. Beside the tiles of the
  // same call there is nothing to wait for (they started behind those kernels), but one block stays until they are done, so
  // that whoever waits for this launch has waited for both.
  if (!a.beside) asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  // Pages of the chunk, 16 keys each, at the same time as the lengths: entries behind the context are dropped afterwards.
  const int shift = a.cache.page_shift, most = (int)min((int64_t)a.chunk, a.max_context - lo);
  for (int i = threadIdx.x; i < (most + 15) / 16; i += 32 * TOK_WARPS) pages[i] = a.page_table[seq * a.table_stride + ((lo + 16 * i) >> shift)];
  const Span sp = span_of(a, seq);
  const int rows = (int)sp.n * a.group;
  auto leave = [&]() {
    if (a.beside && threadIdx.x == 0 && (blockIdx.x | blockIdx.y | blockIdx.z) == 0) asm volatile("griddepcontrol.wait;" ::: "memory");
  };
  if (sp.n <= 0 || sp.n * a.group > TOKEN_ROWS) return leave();  // none, or the other kernel's
  if (lo >= sp.ctx && chunk > 0 && !a.cluster) return leave();   // (a cluster's blocks stay: they meet at its barriers)
  const int keys = (int)max((int64_t)0, min((int64_t)a.chunk, sp.ctx - lo));  // of this chunk
  const int steps = (keys + KEYS - 1) / KEYS;
  __syncthreads();

  // one step's copies: only boxes that begin inside the context; a page that the cache does not have reads as zeros
  auto issue = [&](int step, int stage) {
    const int k0 = step * KEYS, boxes = min(KT, (keys - k0 + 15) / 16);
    const uint32_t bar = s_u32(&full[warp][stage]), at = ring + stage * 2 * G::HALF, sc = ring + TOK_STAGES * 2 * G::HALF + stage * G::SCALES;
    bar_expect_tx(&full[warp][stage], boxes * (2 * HALVES * G::BOX + 2 * G::SC));
#pragma unroll
    for (int b = 0; b < KT; b++) {
      if (b >= boxes) break;
      const int64_t page = pages[k0 / 16 + b];
      const bool known = page >= 0 && page < a.cache.n_pages;
      if (!known) report(a.status, TURQ_E_INVALID_ARG);
      const int z = (int)((known ? page : a.cache.n_pages) * a.cache.n_heads) + (known ? head : 0);
      const int y = (int)((lo + k0 + 16 * b) & (a.cache.page_size - 1));
#pragma unroll
      for (int h = 0; h < HALVES; h++) {
        copy_box3(at + (b * HALVES + h) * G::BOX, &maps.k, 64 * h, y, z, bar);
        copy_box3(at + G::HALF + (b * HALVES + h) * G::BOX, &maps.v, 64 * h, y, z, bar);
      }
      if (Q8) {
        copy_box2(sc + b * G::SC_AT, &maps.ks, y * (D / 32), z, bar);
        copy_box2(sc + (KT + b) * G::SC_AT, &maps.vs, y * (D / 32), z, bar);
      }
    }
  };
  if (lane == 0)
    for (int s = 0; s < TOK_STAGES; s++)
      if (warp + s * TOK_WARPS < steps) issue(warp + s * TOK_WARPS, s);

  // Q^T, 16 elements x 8 rows: lane (g, c) holds row g. On f16 caches a bf16 row is brought to f16 by a power of two that its
  // largest element fits (the products undo it); rows that do not exist are zeros.
  uint32_t qf[NR][KS][2];
  float mul[NR][2];  // of the rows whose sums this lane holds: 8 j + 2 c + e
  int seen[NR][2];
#pragma unroll
  for (int j = 0; j < NR; j++) {
    const int r = 8 * j + g;
    const bool live = r < rows;
    const uint16_t* qp = a.q + (sp.first + (live ? r / a.group : 0)) * a.q_stride + (int64_t)(head * a.group + (live ? r % a.group : 0)) * D;
#pragma unroll
    for (int s = 0; s < KS; s++)
#pragma unroll
      for (int p = 0; p < 2; p++) qf[j][s][p] = live ? *reinterpret_cast<const uint32_t*>(qp + (Q8 ? (D / 4) * c + 4 * s + 2 * p : 16 * s + 2 * c + 8 * p)) : 0u;
    float f = a.scale_log2;
    if (!BF && a.q_bf16) {
      uint32_t top = 0;  // exponent and fraction of the largest magnitude
#pragma unroll
      for (int s = 0; s < KS; s++)
#pragma unroll
        for (int p = 0; p < 2; p++) top = max(top, max(qf[j][s][p] & 0x7FFFu, (qf[j][s][p] >> 16) & 0x7FFFu));
      top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
      top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
      const int e = min(max((int)(top >> 7) - 127, -126), 126);
      const float down = __uint_as_float((uint32_t)(127 - e) << 23);
      f = row_mul(a, __uint_as_float((uint32_t)(127 + e) << 23));
#pragma unroll
      for (int s = 0; s < KS; s++)
#pragma unroll
        for (int p = 0; p < 2; p++) {
          const uint32_t w = qf[j][s][p];
          qf[j][s][p] = pack16<false>(__uint_as_float(w << 16) * down, __uint_as_float(w & 0xFFFF0000u) * down);
        }
    }
#pragma unroll
    for (int e = 0; e < 2; e++) {
      const int row = 8 * j + 2 * c + e;
      mul[j][e] = __shfl_sync(0xFFFFFFFFu, f, 4 * (2 * c + e));
      seen[j][e] = row < rows ? (int)max((int64_t)0, min((int64_t)keys, keys_seen(sp, row / a.group, a.causal) - lo)) : 0;
    }
  }
  const int least = a.causal ? (int)max((int64_t)0, min((int64_t)keys, keys_seen(sp, 0, true) - lo)) : keys;  // keys that every row sees

  float o[NR][MT][4], m[NR][2], l[NR][2];
#pragma unroll
  for (int j = 0; j < NR; j++) {
#pragma unroll
    for (int i = 0; i < MT; i++) o[j][i][0] = o[j][i][1] = o[j][i][2] = o[j][i][3] = 0.f;
    m[j][0] = m[j][1] = -INFINITY;
    l[j][0] = l[j][1] = 0.f;
  }
  const int r8 = lane & 7, mi = lane >> 3;
  __half2 largest = __float2half2_rn(0.f);  // of the scales of keys and values of the context

  int step = warp, n = 0;  // n: steps taken
  for (; step < steps; step += TOK_WARPS, n++) {
    const int stage = n % TOK_STAGES;
    if (!__all_sync(0xFFFFFFFFu, bar_wait(&full[warp][stage], (n / TOK_STAGES) & 1, &abort_flag))) break;
    const uint32_t at = ring + stage * 2 * G::HALF, sc = ring + TOK_STAGES * 2 * G::HALF + stage * G::SCALES;
    const int k0 = step * KEYS;
    if (Q8) {  // a key's scales (lanes 0 to 15) or a value's each: those behind the context's end are anything
#pragma unroll
      for (int kt = 0; kt < KT; kt++) {
        uint32_t w[D / 64];
        const uint32_t from = sc + ((lane >> 4) * KT + kt) * G::SC_AT + (lane & 15) * (D / 16);
        if (k0 + 16 * kt + (lane & 15) < keys) {
          if (D == 128) asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[D / 64 - 1]) : "r"(from));
          else asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(from));
#pragma unroll
          for (int i = 0; i < D / 64; i++) largest = __hmax2(largest, __habs2(u2h2(w[i])));
        }
      }
    }

    // S^T: lane (g, c) gets keys g and g + 8 of a tile for rows 2c, 2c + 1
    float s[KT][NR][4];
#pragma unroll
    for (int kt = 0; kt < KT; kt++) {
#pragma unroll
      for (int j = 0; j < NR; j++) s[kt][j][0] = s[kt][j][1] = s[kt][j][2] = s[kt][j][3] = 0.f;
      if (!Q8) {
#pragma unroll
        for (int i = 0; i < KS; i++) {
          uint32_t k[4];
          const int ch = 2 * i + (mi >> 1), row = (mi & 1) * 8 + r8;
          ldsm4(k, at + (kt * HALVES + (ch >> 3)) * G::BOX + row * 128 + (((ch & 7) ^ r8) << 4));
#pragma unroll
          for (int j = 0; j < NR; j++) mma_16816<BF>(s[kt][j], k, qf[j][i][0], qf[j][i][1]);
        }
      } else {
        const uint32_t kb = at + kt * G::BOX + g * D, sb = sc + kt * G::SC_AT + (g * (D / 32) + c * D / 128) * 2;
        uint16_t s0, s1;
        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(s0) : "r"(sb));
        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(s1) : "r"(sb + 8 * (D / 32) * 2));
        const __half2 sc0 = __half2half2(__ushort_as_half(s0)), sc1 = __half2half2(__ushort_as_half(s1));
#pragma unroll
        for (int q4 = 0; q4 < D / 64; q4++) {  // 16 bytes of each of the two keys: four k steps
          const int ch = c * (D / 64) + q4, at16 = (D == 128 ? ch ^ g : ch ^ ((g >> 1) & 3)) << 4;
          uint32_t w0[4], w1[4];
          asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w0[0]), "=r"(w0[1]), "=r"(w0[2]), "=r"(w0[3]) : "r"(kb + at16));
          asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w1[0]), "=r"(w1[1]), "=r"(w1[2]), "=r"(w1[3]) : "r"(kb + 8 * D + at16));
#pragma unroll
          for (int i = 0; i < 4; i++) {
            uint32_t k[4];
            halves_of(w0[i], sc0, k[0], k[2]);
            halves_of(w1[i], sc1, k[1], k[3]);
#pragma unroll
            for (int j = 0; j < NR; j++) mma_16816<BF>(s[kt][j], k, qf[j][4 * q4 + i][0], qf[j][4 * q4 + i][1]);
          }
        }
      }
    }
    // weights
    float top[NR][2];
#pragma unroll
    for (int j = 0; j < NR; j++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        top[j][e] = m[j][e];
#pragma unroll
        for (int kt = 0; kt < KT; kt++)
#pragma unroll
          for (int h = 0; h < 2; h++) {
            float& x = s[kt][j][2 * h + e];
            if (k0 + KEYS > least && k0 + 16 * kt + 8 * h + g >= seen[j][e]) x = -INFINITY;
            top[j][e] = fmaxf(top[j][e], x);
          }
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) top[j][e] = fmaxf(top[j][e], __shfl_xor_sync(0xFFFFFFFFu, top[j][e], d));
      }
    bool grew = false;
#pragma unroll
    for (int j = 0; j < NR; j++) grew = grew || top[j][0] > m[j][0] || top[j][1] > m[j][1];
    if (__any_sync(0xFFFFFFFFu, grew)) {
#pragma unroll
      for (int j = 0; j < NR; j++) {
        float was[2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
          was[e] = m[j][e] == -INFINITY ? 0.f : ex2((m[j][e] - top[j][e]) * mul[j][e]);
          m[j][e] = top[j][e];
          l[j][e] *= was[e];
        }
#pragma unroll
        for (int i = 0; i < MT; i++) {
          o[j][i][0] *= was[0]; o[j][i][1] *= was[1];
          o[j][i][2] *= was[0]; o[j][i][3] *= was[1];
        }
      }
    }
    // P^T: the two 8 x 8 tiles of 16 keys turned round
    uint32_t p[KT][NR][2];
#pragma unroll
    for (int j = 0; j < NR; j++) {
      const float sub[2] = {m[j][0] == -INFINITY ? 0.f : m[j][0], m[j][1] == -INFINITY ? 0.f : m[j][1]};
#pragma unroll
      for (int kt = 0; kt < KT; kt++) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const float x = ex2((s[kt][j][2 * h] - sub[0]) * mul[j][0]), y = ex2((s[kt][j][2 * h + 1] - sub[1]) * mul[j][1]);
          l[j][0] += x;
          l[j][1] += y;
          asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(p[kt][j][h]) : "r"(pack16<BF>(x, y)));
        }
      }
    }
    // values, 16 keys at a time
#pragma unroll
    for (int kt = 0; kt < KT; kt++) {
      const int live = keys - k0 - 16 * kt;  // keys of this box that exist: what lies behind may be anything, and 0 x NaN is NaN
      if (!Q8) {
        const uint32_t vb = at + G::HALF + kt * HALVES * G::BOX;
        if (live < 16) {
          for (int i = lane; i < 16 * D / 8; i += 32) {
            const int row = i & 15, ch = i >> 4;
            if (row >= live)
              asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(vb + (ch >> 3) * G::BOX + row * 128 + ((ch & 7) << 4)), "r"(0u) : "memory");
          }
          __syncwarp();
        }
#pragma unroll
        for (int i = 0; i < MT; i++) {
          uint32_t v[4];
          const int row = (mi >> 1) * 8 + r8, ch = 2 * i + (mi & 1);
          ldsm4t(v, vb + (ch >> 3) * G::BOX + row * 128 + (((ch & 7) ^ r8) << 4));
#pragma unroll
          for (int j = 0; j < NR; j++) mma_16816<BF>(o[j][i], v, p[kt][j][0], p[kt][j][1]);
        }
      } else {
        // Lane (g, c): D / 8 columns from D/8 g of keys 2c, 2c + 1, 2c + 8, 2c + 9; tile i's rows g and g + 8 are its columns 2i and
        // 2i + 1. Behind the context's end the quants are some bytes, and a scale of zero makes them zeros.
        const uint32_t vb = at + G::HALF + kt * G::BOX, sb = sc + (KT + kt) * G::SC_AT + (g * D / 256) * 2;
        constexpr int W = D / 32;  // words of a key
        uint32_t w[4][W];
        uint16_t vs[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int row = 2 * c + (i & 1) + 8 * (i >> 1);
          if (D == 128)
            asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[i][0]), "=r"(w[i][1]), "=r"(w[i][2 % W]), "=r"(w[i][3 % W])
                         : "r"(vb + row * D + ((g ^ (row & 7)) << 4)));
          else
            asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[i][0]), "=r"(w[i][1])
                         : "r"(vb + row * D + (((g >> 1) ^ ((row >> 1) & 3)) << 4) + (g & 1) * 8));
          asm volatile("ld.shared.u16 %0, [%1];" : "=h"(vs[i]) : "r"(sb + row * (D / 32) * 2));
          if (row >= live) vs[i] = 0;
        }
        const __half2 sc01 = __halves2half2(__ushort_as_half(vs[0]), __ushort_as_half(vs[1])), sc23 = __halves2half2(__ushort_as_half(vs[2]), __ushort_as_half(vs[3]));
        const __half2 off = __float2half2_rn(1152.f);
#pragma unroll
        for (int i = 0; i < W; i++) {
          const uint32_t x0 = w[0][i] ^ 0x80808080u, x1 = w[1][i] ^ 0x80808080u, x2 = w[2][i] ^ 0x80808080u, x3 = w[3][i] ^ 0x80808080u;
#pragma unroll
          for (int h = 0; h < 2; h++) {  // columns 4i + 2h, + 1
            const uint32_t a01 = __byte_perm(x0, x1, h ? 0x7362 : 0x5140), a23 = __byte_perm(x2, x3, h ? 0x7362 : 0x5140);
            uint32_t v[4];
            v[0] = h22u(__hmul2(__hsub2(pair01(a01), off), sc01));
            v[1] = h22u(__hmul2(__hsub2(pair23(a01), off), sc01));
            v[2] = h22u(__hmul2(__hsub2(pair01(a23), off), sc23));
            v[3] = h22u(__hmul2(__hsub2(pair23(a23), off), sc23));
#pragma unroll
            for (int j = 0; j < NR; j++) mma_16816<BF>(o[j][2 * i + h], v, p[kt][j][0], p[kt][j][1]);
          }
        }
      }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // this stage was read, at a context's end also written, by ordinary accesses
    __syncwarp();
    if (lane == 0 && step + TOK_STAGES * TOK_WARPS < steps) issue(step + TOK_STAGES * TOK_WARPS, stage);
  }
  if (step < steps) {
    // A wait ran out. Nothing more is requested; what has been lands before the ring is used for anything else and before the block ends.
    report(a.status, TURQ_E_TIMEOUT);
    const int own = (steps - warp + TOK_WARPS - 1) / TOK_WARPS;  // this warp's steps: warp, warp + TOK_WARPS, ...
    for (int i = n; i < ring_requested(own, n, TOK_STAGES); i++) {
      const long long t0 = clock64();
      while (!bar_try(&full[warp][i % TOK_STAGES], (i / TOK_STAGES) & 1) && clock64() - t0 < TC_WAIT_CYCLES / 8) {}
    }
  }

  if (Q8) report_beyond_f16(a, largest);

  // the four warps' results: each into its own ring, whose copies have all arrived
  __syncwarp();
  float* const ro = reinterpret_cast<float*>(raw + (ring - s_u32(raw)));
  float* const rml = ro + 16 * G::RES;
#pragma unroll
  for (int j = 0; j < NR; j++) {
#pragma unroll
    for (int e = 0; e < 2; e++) {
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) l[j][e] += __shfl_xor_sync(0xFFFFFFFFu, l[j][e], d);
      const int row = 8 * j + 2 * c + e;
#pragma unroll
      for (int i = 0; i < MT; i++) {
        ro[row * G::RES + (Q8 ? D / 8 * g + 2 * i : 16 * i + g)] = o[j][i][e];
        ro[row * G::RES + (Q8 ? D / 8 * g + 2 * i + 1 : 16 * i + g + 8)] = o[j][i][2 + e];
      }
      if (g == 0) {
        rml[2 * row] = joined_max(m[j][e], mul[j][e]);
        rml[2 * row + 1] = l[j][e];
      }
    }
  }
  __syncthreads();
  const bool whole = sp.ctx <= a.chunk;
  const int64_t item = ((int64_t)seq * a.cache.n_heads + head) * a.max_chunks + chunk;
  const float factor = joined_factor(a);
  const float* const rb = reinterpret_cast<const float*>(raw + (base - s_u32(raw)));
  // where a cluster's blocks leave their piece for one another: row r behind the result of warp r % 4
  const uint32_t left = base + 16 * G::RES * 4 + 128;
  static_assert(16 * G::RES * 4 + 128 + 4 * D * 4 + 32 <= G::RING, "a quarter of the piece's rows fits behind a warp's result");
  for (int i = threadIdx.x; i < rows * (D / 2); i += 32 * TOK_WARPS) {
    const int r = i / (D / 2), d = 2 * (i % (D / 2));
    float mm = -INFINITY, ll = 0.f, x = 0.f, y = 0.f;
#pragma unroll
    for (int w = 0; w < TOK_WARPS; w++) mm = fmaxf(mm, rb[w * (G::RING / 4) + 16 * G::RES + 2 * r]);
#pragma unroll
    for (int w = 0; w < TOK_WARPS; w++) {
      const float* p = rb + w * (G::RING / 4);
      const float f = mm == -INFINITY ? 0.f : ex2((p[16 * G::RES + 2 * r] - mm) * factor);
      const float2 v = *reinterpret_cast<const float2*>(p + r * G::RES + d);
      ll += f * p[16 * G::RES + 2 * r + 1];
      x += f * v.x;
      y += f * v.y;
    }
    if (whole && chunk == 0) {
      const float inv = ll > 0.f ? 1.f / ll : ll == 0.f ? 0.f : ll;  // a row that sees no key gives zeros; NaN stays
      const int t = r / a.group, h = head * a.group + r % a.group;
      store_out2(a.out, a.out_dtype, ((sp.first + t) * a.hq + h) * D + d, x * inv, y * inv);
    } else if (a.cluster) {
      const uint32_t q = left + (r & 3) * G::RING;
      asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(q + ((r >> 2) * D + d) * 4), "f"(x), "f"(y) : "memory");
      if (d == 0) asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(q + 4 * D * 4 + (r >> 2) * 8), "f"(mm), "f"(ll) : "memory");
    } else {
      *reinterpret_cast<float2*>(a.part + (item * a.part_rows + r) * D + d) = make_float2(x, y);
      if (d == 0) *reinterpret_cast<float2*>(a.part_ml + (item * a.part_rows + r) * 2) = make_float2(mm, ll);
    }
  }
  if (!a.cluster) return leave();
  // All chunks of the context are one cluster: its blocks read one another's pieces, each its share of the elements, and add them
  // in chunk order.
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (!whole) {
    const int chunks = (int)((sp.ctx + a.chunk - 1) / a.chunk);
    for (int i = chunk * 32 * TOK_WARPS + threadIdx.x; i < rows * (D / 2); i += a.max_chunks * 32 * TOK_WARPS) {
      const int r = i / (D / 2), d = 2 * (i % (D / 2));
      const uint32_t q = left + (r & 3) * G::RING, qo = q + ((r >> 2) * D + d) * 4, qm = q + 4 * D * 4 + (r >> 2) * 8;
      float2 ml[TOKEN_CLUSTER], v[TOKEN_CLUSTER];
      float mm = -INFINITY, ll = 0.f, x = 0.f, y = 0.f;
#pragma unroll
      for (int k = 0; k < TOKEN_CLUSTER; k++) {
        if (k >= chunks) break;
        asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(ml[k].x), "=f"(ml[k].y) : "r"(map_to_rank(qm, k)));
        asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v[k].x), "=f"(v[k].y) : "r"(map_to_rank(qo, k)));
      }
#pragma unroll
      for (int k = 0; k < TOKEN_CLUSTER; k++)
        if (k < chunks) mm = fmaxf(mm, ml[k].x);
#pragma unroll
      for (int k = 0; k < TOKEN_CLUSTER; k++) {
        if (k >= chunks) break;
        const float f = mm == -INFINITY ? 0.f : ex2((ml[k].x - mm) * factor);
        ll += f * ml[k].y;
        x += f * v[k].x;
        y += f * v[k].y;
      }
      const float inv = ll > 0.f ? 1.f / ll : ll == 0.f ? 0.f : ll;
      const int t = r / a.group, h = head * a.group + r % a.group;
      store_out2(a.out, a.out_dtype, ((sp.first + t) * a.hq + h) * D + d, x * inv, y * inv);
    }
  }
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");  // nobody leaves while its piece is read
  leave();
}

// The pieces of a row, in chunk order: a CTA per row, whose warps take every eighth piece and are added in their order. Its lanes
// first read all maxima and sums at once (a loop over pieces would be as many trips to memory, one behind the other).
template <int D>
__global__ void __launch_bounds__(256) join_tokens_kernel(const __grid_constant__ AttendArgs a) {
  constexpr int WARPS = 8, E = D / 32;
  __shared__ float sh[WARPS][D], sh_l[WARPS];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int r = blockIdx.x, head = blockIdx.y, seq = blockIdx.z, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Span sp = cut_span(a.starts[seq], a.starts[seq + 1], a.contexts[seq], a.n_tokens, a.max_new, a.max_context);
  if (sp.n <= 0 || sp.n * a.group > TOKEN_ROWS || sp.ctx <= a.chunk || r >= sp.n * a.group) return;
  const int chunks = (int)((sp.ctx + a.chunk - 1) / a.chunk);
  const int64_t item0 = ((int64_t)seq * a.cache.n_heads + head) * a.max_chunks;
  const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + item0 * a.part_rows + r;
  const float* po = a.part + (item0 * a.part_rows + r) * D + lane * E;
  float mm = -INFINITY;
  for (int k = lane; k < chunks; k += 32) mm = fmaxf(mm, ml[(int64_t)k * a.part_rows].x);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xFFFFFFFFu, mm, d));
  const float sub = mm == -INFINITY ? 0.f : mm, factor = joined_factor(a);
  float ll = 0.f, o[E];
#pragma unroll
  for (int e = 0; e < E; e++) o[e] = 0.f;
#pragma unroll 4
  for (int k = warp; k < chunks; k += WARPS) {
    const float2 t = ml[(int64_t)k * a.part_rows];
    const float f = ex2((t.x - sub) * factor);
    ll += f * t.y;
    const float* p = po + (int64_t)k * a.part_rows * D;
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      const float2 v = *reinterpret_cast<const float2*>(p + e);
      o[e] += f * v.x;
      o[e + 1] += f * v.y;
    }
  }
#pragma unroll
  for (int e = 0; e < E; e++) sh[warp][lane * E + e] = o[e];
  if (lane == 0) sh_l[warp] = ll;
  __syncthreads();
  const int d = 2 * threadIdx.x;
  if (d < D) {
    float x = 0.f, y = 0.f, l = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; w++) {
      x += sh[w][d];
      y += sh[w][d + 1];
      l += sh_l[w];
    }
    const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
    const int t = r / a.group, h = head * a.group + r % a.group;
    store_out2(a.out, a.out_dtype, ((sp.first + t) * a.hq + h) * D + d, x * inv, y * inv);
  }
}

template <int D, bool Q8, bool BF, int NR>
static cudaError_t launch_tokens_rows(const turq_kv_cache* kc, const AttendArgs& a, cudaStream_t s, int* launches) {
  using G = TokGeom<D, Q8, NR>;
  constexpr int SMEM = TOK_WARPS * G::RING + 1024;
  static PerDeviceOnce configured;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (!configured.done(dev)) {
    e = cudaFuncSetAttribute(attend_tokens_kernel<D, Q8, BF, NR>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(attend_tokens_kernel<D, Q8, BF, NR>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    configured.set(dev);
  }
  const TokMaps maps{kc->k16, kc->v16, kc->ks16, kc->vs16};
  (*launches)++;
  e = launch_pdl_cluster(attend_tokens_kernel<D, Q8, BF, NR>, a.cluster ? (unsigned)a.max_chunks : 0u,
                         dim3((unsigned)a.max_chunks, (unsigned)a.cache.n_heads, (unsigned)a.n_seqs), dim3(32 * TOK_WARPS), SMEM, s, maps, a);
  if (e != cudaSuccess || a.max_chunks == 1 || a.cluster) return e;
  (*launches)++;
  return launch_pdl(join_tokens_kernel<D>, dim3((unsigned)a.part_rows, (unsigned)a.cache.n_heads, (unsigned)a.n_seqs), dim3(256), 0, s, a);
}
template <int D, bool Q8, bool BF>
static cudaError_t launch_tokens(const turq_kv_cache* kc, const AttendArgs& a, cudaStream_t s, int* launches) {
  return a.part_rows <= 8 ? launch_tokens_rows<D, Q8, BF, 1>(kc, a, s, launches) : launch_tokens_rows<D, Q8, BF, 2>(kc, a, s, launches);
}

cudaError_t launch_attend_tokens(const turq_kv_cache* kc, const AttendArgs& a, cudaStream_t s, int* launches) {
  if (kc->head_dim == 128) {
    if (kc->dtype == TURQ_Q8_0) return launch_tokens<128, true, false>(kc, a, s, launches);
    return kc->dtype == TURQ_BF16 ? launch_tokens<128, false, true>(kc, a, s, launches) : launch_tokens<128, false, false>(kc, a, s, launches);
  }
  if (kc->dtype == TURQ_Q8_0) return launch_tokens<64, true, false>(kc, a, s, launches);
  return kc->dtype == TURQ_BF16 ? launch_tokens<64, false, true>(kc, a, s, launches) : launch_tokens<64, false, false>(kc, a, s, launches);
}

}  // namespace turq
