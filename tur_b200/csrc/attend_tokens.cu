// Attention of single tokens (up to 16 rows = new tokens x query heads of one key head): bound by the bytes of
// K and V, which every row of a key head shares.
//
// A CTA takes one chunk (token_chunk) of one key head of one sequence, its four warps every fourth step of 16 to 64
// keys. A warp copies its own steps by TMA into its own ring (no CTA-wide barrier in the loop), multiplies with
// mma.sync (rows x keys: 16 x 8 tiles; the rows are few, so the matrix rate does not matter and the accumulators stay
// in registers) and keeps its own running maximum, sum and output; the four are joined through shared memory at the
// end. A context of one chunk is then finished; the pieces of a longer one go to the workspace and
// join_tokens_kernel adds them in chunk order.
//
// Q8_0 keys and values are converted to f16 (2^-11 of a value, against 2^-8 of a block's largest that the
// quantization itself costs) in registers; weights are rounded to the 16-bit type before they meet V.
#include "attend.cuh"
#include "attend_launch.h"
#include "tc_common.cuh"
#include "turq_internal.h"

namespace turq {

constexpr int TOK_WARPS = 4;
constexpr int TOK_STAGES = 3;

// The bytes of a step: 8 KB of keys and values, with the scales of Q8_0 behind them.
template <int D, bool Q8> struct TokGeom {
  static constexpr int ROW = Q8 ? D : 2 * D;           // bytes of a key
  static constexpr int KEYS = 4096 / ROW;              // 16 to 64
  static constexpr int BOX = 16 * (Q8 ? D : 128);      // one copy: 16 keys of a 128-byte column block, or of int8
  static constexpr int SC = Q8 ? 16 * (D / 32) * 2 : 0;  // scales of 16 keys: 128 or 64 bytes,
  static constexpr int SC_AT = Q8 ? 128 : 0;             // each copy to a 128-byte boundary, as tensor copies ask for
  static constexpr int STAGE = 8192 + (Q8 ? 1024 : 0);
  static constexpr int SCRATCH = Q8 ? 16 * D * 2 : 0;  // 16 values of V as f16
  static constexpr int RING = TOK_STAGES * STAGE + SCRATCH;
  static_assert(KEYS / 16 * 2 * SC_AT <= 1024 && SC <= 128, "scales of a step");
  static_assert(RING >= 16 * D * 4 + 128, "the ring holds a warp's result");
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
template <bool BF>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
  if (BF) {
    const __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&t);
  }
  const __half2 t = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&t);
}
// Four int8 -> half2 pairs (b0, b1), (b2, b3), exact: 1024 + (q + 128) less 1152.
__device__ __forceinline__ void halves_of(uint32_t w, __half2 scale, uint32_t& lo, uint32_t& hi) {
  const uint32_t u = w ^ 0x80808080u;
  const __half2 off = __float2half2_rn(1152.f);
  lo = h22u(__hmul2(__hsub2(pair01(u), off), scale));
  hi = h22u(__hmul2(__hsub2(pair23(u), off), scale));
}

__device__ __forceinline__ void copy_box3(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
               ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}
__device__ __forceinline__ void copy_box2(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
               ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}

struct TokMaps { CUtensorMap k, v, ks, vs; };

constexpr int TOK_CHUNK_MAX = 1024;

template <int D, bool Q8, bool BF>
__global__ void __launch_bounds__(32 * TOK_WARPS, 2) attend_tokens_kernel(const __grid_constant__ TokMaps maps, const __grid_constant__ AttendArgs a) {
  using G = TokGeom<D, Q8>;
  constexpr int KEYS = G::KEYS, NT = KEYS / 8, KS = D / 16, DT = D / 8, G16 = KEYS / 16, HALVES = Q8 ? 1 : D / 64;
  extern __shared__ uint8_t raw[];
  __shared__ __align__(8) uint64_t full[TOK_WARPS][TOK_STAGES];
  __shared__ int pages[TOK_CHUNK_MAX / 16];
  __shared__ int abort_flag;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  const int chunk = blockIdx.x, head = blockIdx.y, seq = blockIdx.z;
  const Span sp = span_of(a, seq);
  const int rows = (int)sp.n * a.group;
  if (sp.n <= 0 || sp.n * a.group > TOKEN_ROWS) return;  // none, or the other kernel's
  const int64_t len = token_chunk(sp.ctx), lo = chunk * len;
  if (lo >= sp.ctx && chunk > 0) return;
  const int keys = (int)max((int64_t)0, min(len, sp.ctx - lo));  // of this chunk
  const int steps = (keys + KEYS - 1) / KEYS;

  // pages of the chunk: of 16 keys each; none (-1) where the table names none of the cache's
  const int shift = a.cache.page_shift;
  for (int i = threadIdx.x; i < (keys + 15) / 16; i += 32 * TOK_WARPS) {
    const int64_t page = a.page_table[seq * a.table_stride + ((lo + 16 * i) >> shift)];
    const bool known = page >= 0 && page < a.cache.n_pages;
    if (!known) report(a.status, TURQ_E_INVALID_ARG);
    pages[i] = known ? (int)(page * a.cache.n_heads + head) : (int)(a.cache.n_pages * a.cache.n_heads);
  }
  const uint32_t base = (s_u32(raw) + 1023u) & ~1023u;
  const uint32_t ring = base + warp * G::RING;
  if (threadIdx.x == 0) abort_flag = 0;
  if (lane == 0) {
    for (int s = 0; s < TOK_STAGES; s++) bar_init(&full[warp][s], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();

  // one step's copies: only boxes that begin inside the context
  auto issue = [&](int step, int stage) {
    const int k0 = step * KEYS, boxes = min(G16, (keys - k0 + 15) / 16);
    const uint32_t bar = s_u32(&full[warp][stage]), at = ring + stage * G::STAGE;
    bar_expect_tx(&full[warp][stage], boxes * (2 * HALVES * G::BOX + 2 * G::SC));
    for (int b = 0; b < boxes; b++) {
      const int z = pages[k0 / 16 + b], y = (int)((lo + k0 + 16 * b) & (a.cache.page_size - 1));
#pragma unroll
      for (int h = 0; h < HALVES; h++) {
        copy_box3(at + (b * HALVES + h) * G::BOX, &maps.k, 64 * h, y, z, bar);
        copy_box3(at + 4096 + (b * HALVES + h) * G::BOX, &maps.v, 64 * h, y, z, bar);
      }
      if (Q8) {
        copy_box2(at + 8192 + b * G::SC_AT, &maps.ks, y * (D / 32), z, bar);
        copy_box2(at + 8192 + (G16 + b) * G::SC_AT, &maps.vs, y * (D / 32), z, bar);
      }
    }
  };
  if (lane == 0)
    for (int s = 0; s < TOK_STAGES; s++)
      if (warp + s * TOK_WARPS < steps) issue(warp + s * TOK_WARPS, s);

  // Q as the 16 x 16 operand. On f16 caches a bf16 row is brought to f16 by a power of two that its largest element
  // fits (the products undo it); rows that do not exist are zeros. The k order is the one in which a lane finds keys:
  // in order for 16-bit types, a lane's own D / 4 consecutive elements for int8.
  uint32_t qf[KS][4];
  float mul[2], seen_f[2];
  int seen[2];
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const int r = g + 8 * i;
    const bool live = r < rows;
    const int t = live ? r / a.group : 0, h = head * a.group + (live ? r % a.group : 0);
    const uint16_t* qp = a.q + (sp.first + t) * a.q_stride + (int64_t)h * D;
    seen[i] = live ? (int)max((int64_t)0, min((int64_t)keys, keys_seen(sp, t, a.causal) - lo)) : 0;
#pragma unroll
    for (int s = 0; s < KS; s++) {
#pragma unroll
      for (int p = 0; p < 2; p++) {
        const int d0 = Q8 ? (D / 4) * c + 4 * s + 2 * p : 16 * s + 2 * c + 8 * p;
        qf[s][i + 2 * p] = live ? *reinterpret_cast<const uint32_t*>(qp + d0) : 0u;
      }
    }
    mul[i] = a.scale_log2;
    if (!BF && a.q_bf16) {
      uint32_t top = 0;  // exponent and fraction of the largest magnitude
#pragma unroll
      for (int s = 0; s < KS; s++)
#pragma unroll
        for (int p = 0; p < 2; p++) top = max(top, max(qf[s][i + 2 * p] & 0x7FFFu, (qf[s][i + 2 * p] >> 16) & 0x7FFFu));
      top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
      top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
      const int e = min(max((int)(top >> 7) - 127, -100), 100);
      const float down = __uint_as_float((uint32_t)(127 - e) << 23);
      mul[i] *= __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
      for (int s = 0; s < KS; s++)
#pragma unroll
        for (int p = 0; p < 2; p++) {
          const uint32_t w = qf[s][i + 2 * p];
          qf[s][i + 2 * p] = pack16<false>(__uint_as_float(w << 16) * down, __uint_as_float(w & 0xFFFF0000u) * down);
        }
    }
  }
  (void)seen_f;
  const int least = a.causal ? (int)max((int64_t)0, min((int64_t)keys, keys_seen(sp, 0, true) - lo)) : keys;  // keys that every row sees

  float o[DT][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < DT; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  bool dead = false;
  const int r8 = lane & 7, mi = lane >> 3;

  for (int step = warp, n = 0; step < steps; step += TOK_WARPS, n++) {
    const int stage = n % TOK_STAGES;
    if (!dead && !bar_wait(&full[warp][stage], (n / TOK_STAGES) & 1, &abort_flag)) {
      dead = true;
      report(a.status, TURQ_E_TIMEOUT);
    }
    __syncwarp();
    const uint32_t at = ring + stage * G::STAGE;
    const int k0 = step * KEYS;
    const bool tail = keys - k0 < KEYS;

    float s[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
      if (!Q8) {
#pragma unroll
        for (int q4 = 0; q4 < D / 32; q4++) {  // four column chunks of 8 keys: two k steps
          uint32_t b[4];
          const int ch = q4 * 4 + mi, row = (nt & 1) * 8 + r8;
          ldsm4(b, at + ((nt >> 1) * HALVES + (ch >> 3)) * G::BOX + row * 128 + (((ch & 7) ^ r8) << 4));
          mma_16816<BF>(s[nt], qf[2 * q4], b[0], b[1]);
          mma_16816<BF>(s[nt], qf[2 * q4 + 1], b[2], b[3]);
        }
      } else {
        // lane (g, c): key g, elements (D / 4) c ..: one block of 32 (D = 128) or half of one
        const int row = (nt & 1) * 8 + g;
        const uint32_t kb = at + (nt >> 1) * G::BOX + row * D;
        uint16_t sc;
        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(sc) : "r"(at + 8192 + (nt >> 1) * G::SC_AT + (row * (D / 32) + c * D / 128) * 2));
        const __half2 scale = __half2half2(__ushort_as_half(sc));
#pragma unroll
        for (int q4 = 0; q4 < D / 64; q4++) {  // 16 bytes: four k steps
          const int ch = c * (D / 64) + q4;
          uint4 w;
          asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w)
                       : "r"(kb + ((D == 128 ? (ch ^ (row & 7)) : ch) << 4)));
          const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int i = 0; i < 4; i++) {
            uint32_t b0, b1;
            halves_of(ww[i], scale, b0, b1);
            mma_16816<BF>(s[nt], qf[4 * q4 + i], b0, b1);
          }
        }
      }
    }
    // weights
    float top[2] = {m[0], m[1]};
    const bool mask = k0 + KEYS > least;
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        float x = s[nt][e] * mul[e >> 1];
        if (mask && k0 + 8 * nt + 2 * c + (e & 1) >= seen[e >> 1]) x = -INFINITY;
        s[nt][e] = x;
        top[e >> 1] = fmaxf(top[e >> 1], x);
      }
    float was[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
      top[i] = fmaxf(top[i], __shfl_xor_sync(0xFFFFFFFFu, top[i], 1));
      top[i] = fmaxf(top[i], __shfl_xor_sync(0xFFFFFFFFu, top[i], 2));
    }
    if (__any_sync(0xFFFFFFFFu, top[0] > m[0] || top[1] > m[1])) {
#pragma unroll
      for (int i = 0; i < 2; i++) {
        was[i] = m[i] == -INFINITY ? 0.f : ex2(m[i] - top[i]);
        m[i] = top[i];
        l[i] *= was[i];
      }
#pragma unroll
      for (int i = 0; i < DT; i++) {
        o[i][0] *= was[0]; o[i][1] *= was[0];
        o[i][2] *= was[1]; o[i][3] *= was[1];
      }
    }
    const float sub[2] = {m[0] == -INFINITY ? 0.f : m[0], m[1] == -INFINITY ? 0.f : m[1]};
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        s[nt][e] = ex2(s[nt][e] - sub[e >> 1]);
        l[e >> 1] += s[nt][e];
      }
    // values, 16 keys at a time
#pragma unroll
    for (int b = 0; b < G16; b++) {
      const uint32_t p[4] = {pack16<BF>(s[2 * b][0], s[2 * b][1]), pack16<BF>(s[2 * b][2], s[2 * b][3]), pack16<BF>(s[2 * b + 1][0], s[2 * b + 1][1]),
                             pack16<BF>(s[2 * b + 1][2], s[2 * b + 1][3])};
      const int live = keys - k0 - 16 * b;  // keys of this box that exist: what lies behind may be anything, and 0 x NaN is NaN
      uint32_t vb;
      if (!Q8) {
        vb = at + 4096 + b * HALVES * G::BOX;
        if (tail && live < 16) {
          for (int i = lane; i < 16 * D / 8; i += 32) {
            const int row = i & 15, ch = i >> 4;
            if (row >= live)
              asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(vb + (ch >> 3) * G::BOX + row * 128 + ((ch & 7) << 4)), "r"(0u) : "memory");
          }
          __syncwarp();
        }
      } else {
        vb = ring + TOK_STAGES * G::STAGE;
        __syncwarp();
#pragma unroll
        for (int i = 0; i < D / 32; i++) {  // 16 bytes of a value: 16 x D / 16 of them
          const int id = i * 32 + lane, row = id / (D / 16), ch = id % (D / 16);
          uint4 w;
          asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w)
                       : "r"(at + 4096 + b * G::BOX + row * D + ((D == 128 ? (ch ^ (row & 7)) : ch) << 4)));
          uint16_t sc;
          asm volatile("ld.shared.u16 %0, [%1];" : "=h"(sc) : "r"(at + 8192 + (G16 + b) * G::SC_AT + (row * (D / 32) + (ch >> 1)) * 2));
          __half2 scale = __half2half2(__ushort_as_half(sc));
          uint32_t h[8];
          halves_of(w.x, scale, h[0], h[1]);
          halves_of(w.y, scale, h[2], h[3]);
          halves_of(w.z, scale, h[4], h[5]);
          halves_of(w.w, scale, h[6], h[7]);
          if (row >= live) {
#pragma unroll
            for (int e = 0; e < 8; e++) h[e] = 0u;
          }
          // 64-column blocks of 16 rows, 16-byte chunks in the order of the 128-byte swizzle
          const uint32_t dst = vb + (ch >> 2) * 2048 + row * 128;
          const int c0 = (2 * ch) & 7;
          asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(dst + ((c0 ^ (row & 7)) << 4)), "r"(h[0]), "r"(h[1]), "r"(h[2]), "r"(h[3]) : "memory");
          asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(dst + (((c0 + 1) ^ (row & 7)) << 4)), "r"(h[4]), "r"(h[5]), "r"(h[6]), "r"(h[7]) : "memory");
        }
        __syncwarp();
      }
#pragma unroll
      for (int dt = 0; dt < DT; dt += 2) {
        uint32_t v[4];
        const int row = (mi & 1) * 8 + r8, ch = dt + (mi >> 1);
        ldsm4t(v, vb + (ch >> 3) * 2048 + row * 128 + (((ch & 7) ^ r8) << 4));
        mma_16816<BF>(o[dt], p, v[0], v[1]);
        mma_16816<BF>(o[dt + 1], p, v[2], v[3]);
      }
    }
    __syncwarp();
    if (lane == 0 && step + TOK_STAGES * TOK_WARPS < steps) {
      // this stage was read (and, at a tail that no later step follows, written) by ordinary accesses
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      issue(step + TOK_STAGES * TOK_WARPS, stage);
    }
  }

  // the four warps' results: each into its own ring, whose copies have all arrived
#pragma unroll
  for (int i = 0; i < 2; i++) {
    l[i] += __shfl_xor_sync(0xFFFFFFFFu, l[i], 1);
    l[i] += __shfl_xor_sync(0xFFFFFFFFu, l[i], 2);
  }
  __syncwarp();
  uint8_t* const mine = raw + (ring - s_u32(raw));
  float* const ro = reinterpret_cast<float*>(mine);
  float* const rml = ro + 16 * D;
#pragma unroll
  for (int dt = 0; dt < DT; dt++) {
    *reinterpret_cast<float2*>(ro + g * D + 8 * dt + 2 * c) = make_float2(o[dt][0], o[dt][1]);
    *reinterpret_cast<float2*>(ro + (g + 8) * D + 8 * dt + 2 * c) = make_float2(o[dt][2], o[dt][3]);
  }
  if (c == 0) {
#pragma unroll
    for (int i = 0; i < 2; i++) {
      rml[2 * (g + 8 * i)] = m[i];
      rml[2 * (g + 8 * i) + 1] = l[i];
    }
  }
  __syncthreads();
  const bool whole = len >= sp.ctx;
  const int64_t item = ((int64_t)seq * a.cache.n_heads + head) * a.max_chunks + chunk;
  const float* const rb = reinterpret_cast<const float*>(raw + (base - s_u32(raw)));
  for (int i = threadIdx.x; i < rows * (D / 2); i += 32 * TOK_WARPS) {
    const int r = i / (D / 2), d = 2 * (i % (D / 2));
    float mm = -INFINITY, ll = 0.f, x = 0.f, y = 0.f;
#pragma unroll
    for (int w = 0; w < TOK_WARPS; w++) mm = fmaxf(mm, rb[w * (G::RING / 4) + 16 * D + 2 * r]);
#pragma unroll
    for (int w = 0; w < TOK_WARPS; w++) {
      const float* p = rb + w * (G::RING / 4);
      const float f = mm == -INFINITY ? 0.f : ex2(p[16 * D + 2 * r] - mm);
      const float2 v = *reinterpret_cast<const float2*>(p + r * D + d);
      ll += f * p[16 * D + 2 * r + 1];
      x += f * v.x;
      y += f * v.y;
    }
    if (whole) {
      const float inv = ll > 0.f ? 1.f / ll : ll == 0.f ? 0.f : ll;  // a row that sees no key gives zeros; NaN stays
      const int t = r / a.group, h = head * a.group + r % a.group;
      store_out2(a.out, a.out_dtype, ((sp.first + t) * a.hq + h) * D + d, x * inv, y * inv);
    } else {
      *reinterpret_cast<float2*>(a.part + (item * a.part_rows + r) * D + d) = make_float2(x, y);
      if (d == 0) *reinterpret_cast<float2*>(a.part_ml + (item * a.part_rows + r) * 2) = make_float2(mm, ll);
    }
  }
}

// The pieces of one key head of a sequence, in chunk order. D / 2 threads a row.
template <int D>
__global__ void __launch_bounds__(256) join_tokens_kernel(const __grid_constant__ AttendArgs a) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int head = blockIdx.x, seq = blockIdx.y;
  const Span sp = cut_span(a.starts[seq], a.starts[seq + 1], a.contexts[seq], a.n_tokens, a.max_new, a.max_context);
  const int64_t len = token_chunk(sp.ctx);
  if (sp.n <= 0 || sp.n * a.group > TOKEN_ROWS || len >= sp.ctx) return;
  const int rows = (int)sp.n * a.group, chunks = (int)token_chunks(sp.ctx);
  const int64_t item0 = ((int64_t)seq * a.cache.n_heads + head) * a.max_chunks;
  for (int i = threadIdx.x; i < rows * (D / 2); i += 256) {
    const int r = i / (D / 2), d = 2 * (i % (D / 2));
    const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + item0 * a.part_rows + r;
    const float* po = a.part + (item0 * a.part_rows + r) * D + d;
    float mm = -INFINITY, ll = 0.f, x = 0.f, y = 0.f;
    for (int k = 0; k < chunks; k++) mm = fmaxf(mm, ml[(int64_t)k * a.part_rows].x);
#pragma unroll 4
    for (int k = 0; k < chunks; k++) {
      const float2 t = ml[(int64_t)k * a.part_rows], v = *reinterpret_cast<const float2*>(po + (int64_t)k * a.part_rows * D);
      const float f = mm == -INFINITY ? 0.f : ex2(t.x - mm);
      ll += f * t.y;
      x += f * v.x;
      y += f * v.y;
    }
    const float inv = ll > 0.f ? 1.f / ll : ll == 0.f ? 0.f : ll;
    const int t = r / a.group, h = head * a.group + r % a.group;
    store_out2(a.out, a.out_dtype, ((sp.first + t) * a.hq + h) * D + d, x * inv, y * inv);
  }
}

template <int D, bool Q8, bool BF>
static cudaError_t launch_tokens(const turq_kv_cache* kc, const AttendArgs& a, cudaStream_t s, int* launches) {
  using G = TokGeom<D, Q8>;
  constexpr int SMEM = TOK_WARPS * G::RING + 1024;
  static PerDeviceOnce configured;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (!configured.done(dev)) {
    e = cudaFuncSetAttribute(attend_tokens_kernel<D, Q8, BF>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
    if (e != cudaSuccess) return e;
    configured.set(dev);
  }
  const TokMaps maps{kc->k16, kc->v16, kc->ks16, kc->vs16};
  attend_tokens_kernel<D, Q8, BF><<<dim3((unsigned)a.max_chunks, (unsigned)a.cache.n_heads, (unsigned)a.n_seqs), 32 * TOK_WARPS, SMEM, s>>>(maps, a);
  e = cudaGetLastError();
  (*launches)++;
  if (e != cudaSuccess || a.max_chunks == 1) return e;
  (*launches)++;
  return launch_pdl(join_tokens_kernel<D>, dim3((unsigned)a.cache.n_heads, (unsigned)a.n_seqs), dim3(256), 0, s, a);
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
