// Between attn_q|k|v and attention: norms of the heads with the position rotation, and the paged cache of
// keys and values that takes them (src/models/qwen3.rs:263-305; src/models/kv_cache.rs:288-525).
//   * rope_table_kernel: cos / sin of position x frequency, in 64 bits (far positions lose their angle in
//     32: a position of 1e5 is known to 4e-3 of a turn's radian there);
//   * head_rows_kernel: one pass over the rows of q, k and v. A row is one head of one token; x / sqrt(mean(x^2)
//     + eps) * w and the rotation are done in registers, and the row goes to a dense tensor or to its page,
//     rounded once or quantized to Q8_0. Every byte is read and written once; for many tokens the issue slots bound it (8192 tokens of
//     40 f32 heads of 128 to bf16: 49 us, 5.1 TB/s, 69% of the slots taken), for few the way through memory (one token 2 us);
//   * kv_read_kernel: slots back into dense rows (4099 tokens of 16 Q8_0 heads of 128 to f32 11 us, 3.9 TB/s).
#include <new>

#include "../../include/turq.h"
#include "actquant.cuh"
#include "device_utils.cuh"
#include "handles.h"
#include "kvcache.cuh"
#include "tc_common.cuh"
#include "turq_internal.h"

namespace turq {

struct Frequencies { double f[64]; };

__global__ void __launch_bounds__(256) rope_table_kernel(const Frequencies fr, int n_freqs, int64_t total, double scale, float2* __restrict__ out) {
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    double s, c;
    sincos((double)(i / n_freqs) * fr.f[i % n_freqs], &s, &c);
    out[i] = make_float2((float)(c * scale), (float)(s * scale));
  }
}

// Four neighbouring elements of a row, whatever their type.
__device__ __forceinline__ void load4(const void* p, int dtype, int64_t i, float (&v)[4]) {
  if (dtype == TURQ_F32) {
    const float4 t = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
    v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
    return;
  }
  const uint2 t = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i);
  float2 a, b;
  if (dtype == TURQ_BF16) {
    a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&t.x));
    b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&t.y));
  } else {
    a = __half22float2(*reinterpret_cast<const __half2*>(&t.x));
    b = __half22float2(*reinterpret_cast<const __half2*>(&t.y));
  }
  v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
}
// 1 / sqrt(v): the hardware's estimate (2^-22) and one step of Newton's method.
__device__ __forceinline__ float inverse_root(float v) {
  const float r = rsqrtf(v);
  return r * fmaf(-0.5f * v * r, r, 1.5f);
}
__device__ __forceinline__ void store4(void* p, int dtype, int64_t i, const float* v) {
  if (dtype == TURQ_F32) {
    *reinterpret_cast<float4*>(static_cast<float*>(p) + i) = make_float4(v[0], v[1], v[2], v[3]);
    return;
  }
  uint2 t;
  if (dtype == TURQ_BF16) {
    *reinterpret_cast<__nv_bfloat162*>(&t.x) = __floats2bfloat162_rn(v[0], v[1]);
    *reinterpret_cast<__nv_bfloat162*>(&t.y) = __floats2bfloat162_rn(v[2], v[3]);
  } else {
    *reinterpret_cast<__half2*>(&t.x) = __floats2half2_rn(v[0], v[1]);
    *reinterpret_cast<__half2*>(&t.y) = __floats2half2_rn(v[2], v[3]);
  }
  *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p) + i) = t;
}

struct HeadRowsArgs {
  const void *q, *k, *v;            // v: only with a cache
  int64_t q_stride, k_stride, v_stride;
  int x_dtype, out_dtype;
  int64_t n_tokens;
  int hq, hkv;                      // hq = 0: keys and values alone
  const float *wq, *wk;
  float eps;
  const float2* table;              // null: no rotation
  int64_t n_positions;
  int half_rot, interleaved;
  const int32_t* positions;
  void *q_out, *k_out;              // k_out: without a cache
  KvPages cache;                    // cache.k null: none
  const int64_t* slots;
  int* status;
};

// A block takes one token, D / 8 lanes a row (a head of q, k or v), ROUNDS rows of a token one behind the other with all their
// loads in flight first: angles and weights are read once, and nothing is divided to find a row. A lane owns four pairs of a
// row, so the rotation stays in its registers: pair p of the rotated part is (p, p + half_rot), or (2p, 2p + 1) interleaved;
// behind it lane j simply has elements 8j .. 8j + 7. half_rot is a multiple of 4: no lane straddles the border.
// X: the type of the rows; KIND: where keys go.
enum RowKind { ROWS_DENSE, ROWS_16BIT, ROWS_Q8 };
template <int D, int ROUNDS, int X, int KIND>
__global__ void __launch_bounds__(256, ROUNDS == 4 ? 4 : 5) head_rows_kernel(const __grid_constant__ HeadRowsArgs a) {
  constexpr int L = D / 8;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int j = threadIdx.x % L, groups = blockDim.x / L;
  const int first = (int)blockIdx.y * ROUNDS * groups + (int)threadIdx.x / L;
  const int rows = a.hq + a.hkv * (a.v ? 2 : 1);
  const int64_t token = blockIdx.x;
  const bool rot = a.table != nullptr && 4 * j < a.half_rot;  // this lane's pairs turn, where the row does
  const bool split = rot && !a.interleaved;                   // and lie half_rot apart

  // A row that does not exist (its lanes stay: the rows of a warp reduce together) reads the last one. Rows and heads are few: where
  // one lies in its token is 32-bit arithmetic, where the token lies is worked out once.
  constexpr int XB = X == TURQ_F32 ? 4 : 2;
  const uint8_t* const qp = static_cast<const uint8_t*>(a.q) + token * a.q_stride * XB;
  const uint8_t* const kp = static_cast<const uint8_t*>(a.k) + token * a.k_stride * XB - (int64_t)a.hq * D * XB;
  const uint8_t* const vp = static_cast<const uint8_t*>(a.v) + token * a.v_stride * XB - (int64_t)(a.hq + a.hkv) * D * XB;
  float x[ROUNDS][8];
#pragma unroll
  for (int u = 0; u < ROUNDS; u++) {
    const int r = min(first + u * groups, rows - 1);
    const bool is_q = r < a.hq, is_v = r >= a.hq + a.hkv, apart = split && !is_v;
    const uint8_t* const src = is_q ? qp : is_v ? vp : kp;
    load4(src, X, r * D + (apart ? 4 * j : 8 * j), reinterpret_cast<float(&)[4]>(x[u][0]));
    load4(src, X, r * D + (apart ? a.half_rot + 4 * j : 8 * j + 4), reinterpret_cast<float(&)[4]>(x[u][4]));
  }
  const int64_t slot = a.slots ? a.slots[token] : -1;
  bool known = true;
  float c[4] = {1.f, 1.f, 1.f, 1.f}, s[4] = {0.f, 0.f, 0.f, 0.f};
  if (a.table) {
    const int64_t pos = a.positions[token];
    known = pos >= 0 && pos < a.n_positions;
    if (!known) *reinterpret_cast<volatile int*>(a.status) = TURQ_E_INVALID_ARG;
    if (rot && known) {
      const float4* t = reinterpret_cast<const float4*>(a.table + pos * a.half_rot + 4 * j);
      const float4 t0 = t[0], t1 = t[1];
      c[0] = t0.x; c[1] = t0.z; c[2] = t1.x; c[3] = t1.z;
      s[0] = t0.y; s[1] = t0.w; s[2] = t1.y; s[3] = t1.w;
    }
  }
  const bool fits = slot < a.cache.n_pages * a.cache.page_size;
  if (KIND != ROWS_DENSE && !fits) *reinterpret_cast<volatile int*>(a.status) = TURQ_E_INVALID_ARG;
  const bool write = KIND != ROWS_DENSE && slot >= 0 && fits && known;
  const int64_t row0 = write ? a.cache.row(slot, 0) : 0;  // of the planes; a page's heads are page_size rows apart

  const int out_bytes = a.out_dtype == TURQ_F32 ? 4 : 2;
  uint8_t* const qo = static_cast<uint8_t*>(a.q_out) + token * a.hq * D * out_bytes;
  uint8_t* const ko = static_cast<uint8_t*>(a.k_out) + (token * a.hkv - a.hq) * D * out_bytes;

#pragma unroll
  for (int u = 0; u < ROUNDS; u++) {
    const int r = first + u * groups;
    const bool live = r < rows, is_q = r < a.hq, is_v = r >= a.hq + a.hkv;
    float* const y = x[u];
    if (a.wq || a.wk) {  // the whole grid the same way: the shuffles need every lane
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 8; e++) ss += y[e] * y[e];
#pragma unroll
      for (int o = 1; o < L; o <<= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
      const float inv = inverse_root(ss / D + a.eps);
      const float* const w = is_q ? a.wq : is_v ? nullptr : a.wk;
      if (w) {
        float wv[8];
        load4(w, TURQ_F32, split ? 4 * j : 8 * j, reinterpret_cast<float(&)[4]>(wv[0]));
        load4(w, TURQ_F32, split ? a.half_rot + 4 * j : 8 * j + 4, reinterpret_cast<float(&)[4]>(wv[4]));
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = y[e] * inv * wv[e];
      }
    }
    if (rot && !is_v) {
      if (a.interleaved) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float p = y[2 * i], q = y[2 * i + 1];
          y[2 * i] = p * c[i] - q * s[i];
          y[2 * i + 1] = q * c[i] + p * s[i];
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float p = y[i], q = y[4 + i];
          y[i] = p * c[i] - q * s[i];
          y[4 + i] = q * c[i] + p * s[i];
        }
      }
    }
    if (!known) {
#pragma unroll
      for (int e = 0; e < 8; e++) y[e] = 0.f;
    }
    const int o0 = split && !is_v ? 4 * j : 8 * j, o1 = split && !is_v ? a.half_rot + 4 * j : 8 * j + 4;
    if (live && (is_q || KIND == ROWS_DENSE)) {
      uint8_t* const out = is_q ? qo : ko;
      store4(out, a.out_dtype, r * D + o0, y);
      store4(out, a.out_dtype, r * D + o1, y + 4);
    }
    if (KIND == ROWS_DENSE) continue;
    const int h = is_v ? r - a.hq - a.hkv : r - a.hq;
    const bool put = write && live && !is_q;
    const int64_t at = row0 + (int64_t)(put ? h : 0) * a.cache.page_size;
    if (KIND == ROWS_16BIT) {
      if (put) {
        void* out = is_v ? a.cache.v : a.cache.k;
        store4(out, a.cache.dtype, at * D + o0, y);
        store4(out, a.cache.dtype, at * D + o1, y + 4);
      }
      continue;
    }
    if (!__any_sync(0xFFFFFFFFu, put)) continue;
    // Q8_0: lane j gets elements 8j .. 8j + 7, so that four lanes hold a block of 32. A group of four elements 4g .. 4g + 3 of a
    // row whose pairs lie apart is the first half of lane g's registers, the second half of lane g - half_rot / 4's, or one
    // of the two of lane g / 2.
    if (a.table && !a.interleaved) {
      float z[8];
#pragma unroll
      for (int b = 0; b < 2; b++) {
        const int g = 2 * j + b, q4 = a.half_rot / 4;
        const int from = !is_v && g < q4 ? g : !is_v && g < 2 * q4 ? g - q4 : g / 2;
        const bool second = !is_v && g < q4 ? false : !is_v && g < 2 * q4 ? true : (g & 1) != 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float lo = __shfl_sync(0xFFFFFFFFu, y[i], from, L), hi = __shfl_sync(0xFFFFFFFFu, y[4 + i], from, L);
          z[4 * b + i] = second ? hi : lo;
        }
      }
#pragma unroll
      for (int e = 0; e < 8; e++) y[e] = z[e];
    }
    uint32_t w0, w1;
    __half d;
    quant_block_q8_0(*reinterpret_cast<const float(*)[8]>(y), w0, w1, d);
    if (put) {
      *reinterpret_cast<uint2*>((is_v ? a.cache.v : a.cache.k) + at * D + 8 * j) = make_uint2(w0, w1);
      if ((j & 3) == 0) (is_v ? a.cache.vs : a.cache.ks)[at * (D / 32) + j / 4] = d;
    }
  }
}

// A block takes one token, D / 8 lanes a row of keys or values, ROUNDS of them one behind the other.
template <int D, int ROUNDS>
__global__ void __launch_bounds__(256) kv_read_kernel(const KvPages c, const int64_t* __restrict__ slots, int out_dtype, void* __restrict__ k_out,
                                                      void* __restrict__ v_out, int* status) {
  constexpr int L = D / 8;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int j = threadIdx.x % L, groups = blockDim.x / L, first = (int)blockIdx.y * ROUNDS * groups + (int)threadIdx.x / L;
  const int64_t token = blockIdx.x, slot = slots[token];
  const bool fits = slot < c.n_pages * c.page_size, there = slot >= 0 && fits;
  if (!fits) *reinterpret_cast<volatile int*>(status) = TURQ_E_INVALID_ARG;
  const int64_t row0 = there ? c.row(slot, 0) : 0;
  uint4 w[ROUNDS];
  float d[ROUNDS];
#pragma unroll
  for (int u = 0; u < ROUNDS; u++) {
    const int r = min(first + u * groups, 2 * c.n_heads - 1);
    const bool is_v = r >= c.n_heads;
    const int64_t at = row0 + (int64_t)(is_v ? r - c.n_heads : r) * c.page_size;
    const uint8_t* src = is_v ? c.v : c.k;
    if (c.dtype == TURQ_Q8_0) {
      const uint2 t = *reinterpret_cast<const uint2*>(src + at * D + 8 * j);
      w[u] = make_uint4(t.x, t.y, 0, 0);
      d[u] = __half2float((is_v ? c.vs : c.ks)[at * (D / 32) + j / 4]);
    } else {
      w[u] = *reinterpret_cast<const uint4*>(src + (at * D + 8 * j) * 2);
    }
  }
#pragma unroll
  for (int u = 0; u < ROUNDS; u++) {
    const int r = first + u * groups;
    if (r >= 2 * c.n_heads) break;
    const bool is_v = r >= c.n_heads;
    const uint32_t t[4] = {w[u].x, w[u].y, w[u].z, w[u].w};
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
      if (c.dtype == TURQ_Q8_0) {
        x[e] = d[u] * (float)(int8_t)(t[e >> 2] >> (8 * (e & 3)));
      } else {
        const uint32_t bits = t[e >> 1] >> (16 * (e & 1));
        x[e] = c.dtype == TURQ_BF16 ? __uint_as_float(bits << 16) : f16_bits_to_f32(bits);
      }
      if (!there) x[e] = 0.f;
    }
    const int64_t o = (token * c.n_heads + (is_v ? r - c.n_heads : r)) * D + 8 * j;
    store4(is_v ? v_out : k_out, out_dtype, o, x);
    store4(is_v ? v_out : k_out, out_dtype, o + 4, x + 4);
  }
}

// Lanes for all rows of a token, 256 at most. Rounds: one where a call has so few tokens that blocks are what it lacks; otherwise two,
// or four where a token has many wide rows (us, 1 / 2 / 4 rounds: 64 tokens of 80 f32 rows of 128 2.6 / 2.7 / 3.3, 8192 of 40 69 / 64 /
// 49, 4099 of 16 bf16 rows of 128 into Q8_0 12.0 / 10.3 / 10.5, 2049 of 60 bf16 rows of 64 10.5 / 8.4 / 8.4).
struct RowGrid { dim3 grid, block; int rounds; };
static RowGrid plan_rows(int64_t n_tokens, int rows, int head_dim, int most = 4) {
  const int lanes = head_dim / 8;
  RowGrid p;
  p.rounds = n_tokens < 256 ? 1 : most == 4 && head_dim == 128 && rows >= 32 ? 4 : 2;
  int threads = ((rows + p.rounds - 1) / p.rounds * lanes + 31) / 32 * 32;
  if (threads > 256) threads = 256;
  const int per_block = threads / lanes * p.rounds;
  p.block = dim3(threads);
  p.grid = dim3((unsigned)n_tokens, (unsigned)((rows + per_block - 1) / per_block));
  return p;
}

template <int D, int X, int KIND>
static cudaError_t launch_rows(const RowGrid& p, const HeadRowsArgs& a, cudaStream_t s) {
  if (p.rounds == 1) return launch_pdl(head_rows_kernel<D, 1, X, KIND>, p.grid, p.block, 0, s, a);
  if (D == 128 && p.rounds == 4) return launch_pdl(head_rows_kernel<D, D == 128 ? 4 : 2, X, KIND>, p.grid, p.block, 0, s, a);
  return launch_pdl(head_rows_kernel<D, 2, X, KIND>, p.grid, p.block, 0, s, a);
}
template <int D, int X>
static cudaError_t launch_rows_kind(const RowGrid& p, const HeadRowsArgs& a, cudaStream_t s) {
  if (!a.cache.k) return launch_rows<D, X, ROWS_DENSE>(p, a, s);
  return a.cache.dtype == TURQ_Q8_0 ? launch_rows<D, X, ROWS_Q8>(p, a, s) : launch_rows<D, X, ROWS_16BIT>(p, a, s);
}
template <int D>
static cudaError_t launch_rows_type(const RowGrid& p, const HeadRowsArgs& a, cudaStream_t s) {
  return a.x_dtype == TURQ_F32 ? launch_rows_kind<D, TURQ_F32>(p, a, s) : a.x_dtype == TURQ_BF16 ? launch_rows_kind<D, TURQ_BF16>(p, a, s) : launch_rows_kind<D, TURQ_F16>(p, a, s);
}
static cudaError_t launch_head_rows(int head_dim, const HeadRowsArgs& a, cudaStream_t s) {
  const RowGrid p = plan_rows(a.n_tokens, a.hq + a.hkv * (a.v ? 2 : 1), head_dim);
  return head_dim == 64 ? launch_rows_type<64>(p, a, s) : launch_rows_type<128>(p, a, s);
}
static cudaError_t launch_kv_read(int head_dim, const KvPages& pages, const int64_t* slots, int64_t n_tokens, int out_dtype, void* k_out, void* v_out, int* status,
                                  cudaStream_t s) {
  const RowGrid p = plan_rows(n_tokens, 2 * pages.n_heads, head_dim, 2);
  auto go = [&](auto kernel) { return launch_pdl(kernel, p.grid, p.block, 0, s, pages, slots, out_dtype, k_out, v_out, status); };
  if (head_dim == 64) return p.rounds == 1 ? go(kv_read_kernel<64, 1>) : go(kv_read_kernel<64, 2>);
  return p.rounds == 1 ? go(kv_read_kernel<128, 1>) : go(kv_read_kernel<128, 2>);
}

}  // namespace turq

namespace {

using turq::api_cuda_fail;
using turq::api_fail;

int32_t elem_bytes(int32_t dtype) { return dtype == TURQ_F32 ? 4 : dtype == TURQ_F16 || dtype == TURQ_BF16 ? 2 : 0; }

// An operand of rows: base and stride in whole 16 bytes, rows that do not overlap.
int32_t check_rows(turq_ctx* ctx, const void* p, int64_t stride, int64_t width, int32_t dtype) {
  if (!p) return api_fail(ctx, TURQ_E_INVALID_ARG, "null argument");
  if (stride < width) return api_fail(ctx, TURQ_E_SHAPE, "the stride of q, k or v is less than the width of its heads");
  if ((uintptr_t)p % 16 != 0 || stride * elem_bytes(dtype) % 16 != 0)
    return api_fail(ctx, TURQ_E_ALIGN, "q, k and v need 16-byte aligned bases and strides of whole 16 bytes");
  return TURQ_OK;
}

int32_t check_tokens(turq_ctx* ctx, int64_t n_tokens, int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim) {
  if (head_dim != 64 && head_dim != 128) return api_fail(ctx, TURQ_E_SHAPE, "head_dim must be 64 or 128");
  if (n_q_heads < 0 || n_kv_heads < 1 || n_q_heads > 65536 || n_kv_heads > 65536) return api_fail(ctx, TURQ_E_SHAPE, "head counts must be in 1..65536");
  if (n_tokens < 0 || n_tokens > INT32_MAX / 2)
    return api_fail(ctx, TURQ_E_SHAPE, "n_tokens out of range");
  return TURQ_OK;
}

// Norm weights, table and positions of a rotating call.
int32_t check_rotation(turq_ctx* ctx, const float* wq, const float* wk, const float* table, int64_t n_positions, int32_t rotary_dim,
                       int32_t head_dim, const int32_t* positions) {
  if (!table || !positions) return api_fail(ctx, TURQ_E_INVALID_ARG, "null argument");
  if (rotary_dim <= 0 || rotary_dim > head_dim || rotary_dim % 8 != 0) return api_fail(ctx, TURQ_E_SHAPE, "rotary_dim must be a multiple of 8 up to head_dim");
  if (n_positions <= 0) return api_fail(ctx, TURQ_E_SHAPE, "the table has no positions");
  if ((uintptr_t)table % 16 != 0 || (uintptr_t)wq % 16 != 0 || (uintptr_t)wk % 16 != 0 || (uintptr_t)positions % 4 != 0)
    return api_fail(ctx, TURQ_E_ALIGN, "table and norm weights must be 16-byte, positions 4-byte aligned");
  return TURQ_OK;
}

int32_t check_cache(turq_ctx* ctx, const turq_kv_cache* cache, const void* slots) {
  if (cache->device != ctx->device) return api_fail(ctx, TURQ_E_INVALID_ARG, "cache and context must live on the same device");
  if (!slots) return api_fail(ctx, TURQ_E_INVALID_ARG, "null argument");
  if ((uintptr_t)slots % 8 != 0) return api_fail(ctx, TURQ_E_ALIGN, "slots must be 8-byte aligned");
  return TURQ_OK;
}

#define TQ_TRY(expr)                      \
  do {                                    \
    const int32_t st__ = (expr);          \
    if (st__ != TURQ_OK) return st__;     \
  } while (0)

int32_t run_head_rows(turq_ctx* ctx, int head_dim, const turq::HeadRowsArgs& a, void* stream, const char* what) {
  turq::DeviceScope on(ctx->device);
  cudaError_t e = on.status;
  if (e == cudaSuccess) e = turq::launch_head_rows(head_dim, a, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return api_cuda_fail(ctx, e, what);
  ctx->launches++;
  return TURQ_OK;
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// A plane [n_pages * heads][page_size][row_elems] for boxes of `tokens` rows and `cols` elements.
bool map_plane(EncodeTiledFn enc, CUtensorMap* map, const turq_kv_cache* kc, CUtensorMapDataType type, int elem, size_t offset, int row_elems,
               int cols, int tokens, CUtensorMapSwizzle swizzle) {
  const cuuint64_t dims[3] = {(cuuint64_t)row_elems, (cuuint64_t)kc->page_size, (cuuint64_t)kc->n_pages * kc->n_kv_heads};
  const cuuint64_t strides[2] = {(cuuint64_t)row_elems * elem, (cuuint64_t)row_elems * elem * kc->page_size};
  const cuuint32_t box[3] = {(cuuint32_t)cols, (cuuint32_t)tokens, 1}, step[3] = {1, 1, 1};
  return enc(map, type, 3, kc->mem + offset, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
bool map_planes(turq_kv_cache* kc) {
  void* p = nullptr;
  cudaDriverEntryPointQueryResult q;
  if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) return false;
  const EncodeTiledFn enc = reinterpret_cast<EncodeTiledFn>(p);
  const int d = kc->head_dim, whole = kc->page_size < 128 ? kc->page_size : 128;
  if (kc->dtype != TURQ_Q8_0) {
    const CUtensorMapDataType t = kc->dtype == TURQ_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    return map_plane(enc, &kc->k16, kc, t, 2, 0, d, 64, 16, CU_TENSOR_MAP_SWIZZLE_128B) &&
           map_plane(enc, &kc->v16, kc, t, 2, kc->off_v, d, 64, 16, CU_TENSOR_MAP_SWIZZLE_128B) &&
           map_plane(enc, &kc->k_tile, kc, t, 2, 0, d, 64, whole, CU_TENSOR_MAP_SWIZZLE_128B) &&
           map_plane(enc, &kc->v_tile, kc, t, 2, kc->off_v, d, 64, whole, CU_TENSOR_MAP_SWIZZLE_128B);
  }
  // Scales: the 16 tokens' lie one behind the other, so a page is one row of its head's plane.
  const CUtensorMapSwizzle swizzle = d == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
  const int per = d / 32;
  auto scales = [&](CUtensorMap* map, size_t offset) {
    const cuuint64_t dims[2] = {(cuuint64_t)kc->page_size * per, (cuuint64_t)kc->n_pages * kc->n_kv_heads};
    const cuuint64_t strides[1] = {(cuuint64_t)kc->page_size * per * 2};
    const cuuint32_t box[2] = {(cuuint32_t)(16 * per), 1}, step[2] = {1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, kc->mem + offset, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
  };
  return map_plane(enc, &kc->k16, kc, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, 0, d, d, 16, swizzle) &&
         map_plane(enc, &kc->v16, kc, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, kc->off_v, d, d, 16, swizzle) &&
         map_plane(enc, &kc->k_tile, kc, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, 0, d, d, whole, CU_TENSOR_MAP_SWIZZLE_NONE) &&
         map_plane(enc, &kc->v_tile, kc, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, kc->off_v, d, d, whole, CU_TENSOR_MAP_SWIZZLE_NONE) && scales(&kc->ks16, kc->off_ks) &&
         scales(&kc->vs16, kc->off_vs);
}

struct CacheShape { size_t off_v, off_ks, off_vs, bytes; bool ok; };
CacheShape cache_shape(int32_t dtype, int64_t n_pages, int32_t page_size, int32_t n_kv_heads, int32_t head_dim) {
  CacheShape c{0, 0, 0, 0, false};
  if (dtype != TURQ_F16 && dtype != TURQ_BF16 && dtype != TURQ_Q8_0) return c;
  if (head_dim != 64 && head_dim != 128) return c;
  if (page_size < 16 || page_size > 256 || (page_size & (page_size - 1)) != 0) return c;
  if (n_pages <= 0 || n_kv_heads <= 0 || n_kv_heads > 65536 || n_pages > INT32_MAX / n_kv_heads) return c;  // page x head is a 31-bit index
  auto up = [](size_t v) { return (v + 255) & ~(size_t)255; };
  const size_t rows = (size_t)n_pages * n_kv_heads * page_size;
  const size_t plane = up(rows * head_dim * (dtype == TURQ_Q8_0 ? 1 : 2)), scales = dtype == TURQ_Q8_0 ? up(rows * (head_dim / 32) * 2) : 0;
  c.off_v = plane;
  c.off_ks = 2 * plane;
  c.off_vs = 2 * plane + scales;
  c.bytes = 2 * plane + 2 * scales;
  c.ok = true;
  return c;
}

}  // namespace

extern "C" {

int32_t turq_rope_table(turq_ctx* ctx, const double* host_freqs, int32_t n_freqs, int64_t n_positions, double scale, float* dev_table, void* stream) {
  if (!ctx || !host_freqs || !dev_table) return api_fail(ctx, TURQ_E_INVALID_ARG, "null argument");
  if (n_freqs <= 0 || n_freqs > 64 || n_freqs % 4 != 0) return api_fail(ctx, TURQ_E_SHAPE, "n_freqs must be a multiple of 4, at most 64");
  if (n_positions <= 0 || n_positions > INT32_MAX) return api_fail(ctx, TURQ_E_SHAPE, "n_positions out of range");
  if ((uintptr_t)dev_table % 16 != 0) return api_fail(ctx, TURQ_E_ALIGN, "dev_table must be 16-byte aligned");
  turq::Frequencies fr{};
  for (int i = 0; i < n_freqs; i++) fr.f[i] = host_freqs[i];
  turq::DeviceScope on(ctx->device);
  if (on.status != cudaSuccess) return api_cuda_fail(ctx, on.status, "rope table launch");
  const int64_t total = n_positions * n_freqs;
  int64_t blocks = (total + 255) / 256;
  if (blocks > 32 * (int64_t)ctx->sm_count) blocks = 32 * (int64_t)ctx->sm_count;
  turq::rope_table_kernel<<<(unsigned)blocks, 256, 0, static_cast<cudaStream_t>(stream)>>>(fr, n_freqs, total, scale, reinterpret_cast<float2*>(dev_table));
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return api_cuda_fail(ctx, e, "rope table launch");
  ctx->launches++;
  return TURQ_OK;
}

int32_t turq_qk_norm_rope(turq_ctx* ctx, const void* dev_q, int64_t q_stride, const void* dev_k, int64_t k_stride, int32_t x_dtype,
                          int64_t n_tokens, int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim, const float* dev_q_weight,
                          const float* dev_k_weight, float eps, const float* dev_table, int64_t n_positions, int32_t rotary_dim,
                          int32_t interleaved, const int32_t* dev_positions, int32_t out_dtype, void* dev_q_out, void* dev_k_out,
                          void* stream) {
  if (!ctx) return TURQ_E_INVALID_ARG;
  if (!elem_bytes(x_dtype) || !elem_bytes(out_dtype)) return api_fail(ctx, TURQ_E_DTYPE, "rows must be F32, F16 or BF16");
  TQ_TRY(check_tokens(ctx, n_tokens, n_q_heads, n_kv_heads, head_dim));
  if (n_q_heads < 1) return api_fail(ctx, TURQ_E_SHAPE, "head counts must be in 1..65536");
  if (n_tokens == 0) return TURQ_OK;
  TQ_TRY(check_rows(ctx, dev_q, q_stride, (int64_t)n_q_heads * head_dim, x_dtype));
  TQ_TRY(check_rows(ctx, dev_k, k_stride, (int64_t)n_kv_heads * head_dim, x_dtype));
  TQ_TRY(check_rotation(ctx, dev_q_weight, dev_k_weight, dev_table, n_positions, rotary_dim, head_dim, dev_positions));
  if (!dev_q_out || !dev_k_out) return api_fail(ctx, TURQ_E_INVALID_ARG, "null argument");
  if ((uintptr_t)dev_q_out % 16 != 0 || (uintptr_t)dev_k_out % 16 != 0) return api_fail(ctx, TURQ_E_ALIGN, "outputs must be 16-byte aligned");
  turq::HeadRowsArgs a{};
  a.q = dev_q; a.k = dev_k;
  a.q_stride = q_stride; a.k_stride = k_stride;
  a.x_dtype = x_dtype; a.out_dtype = out_dtype;
  a.n_tokens = n_tokens; a.hq = n_q_heads; a.hkv = n_kv_heads;
  a.wq = dev_q_weight; a.wk = dev_k_weight; a.eps = eps;
  a.table = reinterpret_cast<const float2*>(dev_table); a.n_positions = n_positions;
  a.half_rot = rotary_dim / 2; a.interleaved = interleaved != 0; a.positions = dev_positions;
  a.q_out = dev_q_out; a.k_out = dev_k_out;
  a.status = ctx->dev_status;
  return run_head_rows(ctx, head_dim, a, stream, "qk_norm_rope launch");
}

size_t turq_kv_cache_bytes(int32_t dtype, int64_t n_pages, int32_t page_size, int32_t n_kv_heads, int32_t head_dim) {
  const CacheShape c = cache_shape(dtype, n_pages, page_size, n_kv_heads, head_dim);
  return c.ok ? c.bytes : 0;
}

int32_t turq_kv_cache_create(turq_ctx* ctx, int32_t dtype, int64_t n_pages, int32_t page_size, int32_t n_kv_heads, int32_t head_dim,
                             void* dev_memory, size_t nbytes, turq_kv_cache** out) {
  if (!ctx || !out) return api_fail(ctx, TURQ_E_INVALID_ARG, "null argument");
  *out = nullptr;
  if (dtype != TURQ_F16 && dtype != TURQ_BF16 && dtype != TURQ_Q8_0) return api_fail(ctx, TURQ_E_DTYPE, "a cache holds F16, BF16 or Q8_0");
  const CacheShape c = cache_shape(dtype, n_pages, page_size, n_kv_heads, head_dim);
  if (!c.ok)
    return api_fail(ctx, TURQ_E_SHAPE, "a cache needs head_dim 64 or 128, pages of 16 to 256 tokens (a power of two), and n_pages * n_kv_heads in 31 bits");
  if (dev_memory && nbytes < c.bytes) return api_fail(ctx, TURQ_E_SHAPE, "dev_memory holds less than turq_kv_cache_bytes");
  if ((uintptr_t)dev_memory % 256 != 0) return api_fail(ctx, TURQ_E_ALIGN, "dev_memory must be 256-byte aligned");
  turq::DeviceScope on(ctx->device);
  if (on.status != cudaSuccess) return api_cuda_fail(ctx, on.status, "cudaSetDevice");
  turq_kv_cache* kc = new (std::nothrow) turq_kv_cache();
  if (!kc) return api_fail(ctx, TURQ_E_INVALID_ARG, "out of host memory");
  kc->device = ctx->device;
  kc->sm_count = ctx->sm_count;
  kc->dtype = dtype;
  kc->n_pages = n_pages;
  kc->page_size = page_size;
  kc->n_kv_heads = n_kv_heads;
  kc->head_dim = head_dim;
  kc->off_v = c.off_v;
  kc->off_ks = c.off_ks;
  kc->off_vs = c.off_vs;
  kc->bytes = c.bytes;
  kc->mem = static_cast<uint8_t*>(dev_memory);
  if (!dev_memory) {
    cudaError_t e = cudaMalloc(reinterpret_cast<void**>(&kc->mem), c.bytes);
    kc->owns = e == cudaSuccess;
    if (e == cudaSuccess) e = cudaMemset(kc->mem, 0, c.bytes);
    if (e == cudaSuccess) e = cudaStreamSynchronize(nullptr);
    if (e != cudaSuccess) {
      cudaGetLastError();
      turq_kv_cache_free(kc);
      return api_cuda_fail(ctx, e, "allocating the cache's pages");
    }
  }
  if (!map_planes(kc)) {
    turq_kv_cache_free(kc);
    return api_fail(ctx, TURQ_E_CUDA, "the driver does not describe the cache's pages as tensors");
  }
  *out = kc;
  return TURQ_OK;
}

int32_t turq_kv_cache_free(turq_kv_cache* cache) {
  if (!cache) return TURQ_E_INVALID_ARG;
  if (cache->owns) {
    turq::DeviceScope on(cache->device);
    cudaFree(cache->mem);
  }
  delete cache;
  return TURQ_OK;
}

int32_t turq_kv_cache_layout(const turq_kv_cache* cache, void** dev_memory, int64_t* offsets) {
  if (!cache) return TURQ_E_INVALID_ARG;
  if (dev_memory) *dev_memory = cache->mem;
  if (offsets) {
    offsets[0] = 0;
    offsets[1] = (int64_t)cache->off_v;
    offsets[2] = (int64_t)cache->off_ks;
    offsets[3] = (int64_t)cache->off_vs;
  }
  return TURQ_OK;
}

int32_t turq_kv_append(turq_ctx* ctx, turq_kv_cache* cache, const void* dev_q, int64_t q_stride, const void* dev_k, int64_t k_stride,
                       const void* dev_v, int64_t v_stride, int32_t x_dtype, int64_t n_tokens, int32_t n_q_heads,
                       const float* dev_q_weight, const float* dev_k_weight, float eps, const float* dev_table, int64_t n_positions,
                       int32_t rotary_dim, int32_t interleaved, const int32_t* dev_positions, const int64_t* dev_slots,
                       int32_t out_dtype, void* dev_q_out, void* stream) {
  if (!ctx || !cache) return api_fail(ctx, TURQ_E_INVALID_ARG, "null argument");
  if (!elem_bytes(x_dtype) || !elem_bytes(out_dtype)) return api_fail(ctx, TURQ_E_DTYPE, "rows must be F32, F16 or BF16");
  const int d = cache->head_dim, hkv = cache->n_kv_heads;
  TQ_TRY(check_tokens(ctx, n_tokens, n_q_heads, hkv, d));
  if (n_q_heads < 1) return api_fail(ctx, TURQ_E_SHAPE, "head counts must be in 1..65536");
  if (n_tokens == 0) return TURQ_OK;
  TQ_TRY(check_rows(ctx, dev_q, q_stride, (int64_t)n_q_heads * d, x_dtype));
  TQ_TRY(check_rows(ctx, dev_k, k_stride, (int64_t)hkv * d, x_dtype));
  TQ_TRY(check_rows(ctx, dev_v, v_stride, (int64_t)hkv * d, x_dtype));
  TQ_TRY(check_rotation(ctx, dev_q_weight, dev_k_weight, dev_table, n_positions, rotary_dim, d, dev_positions));
  TQ_TRY(check_cache(ctx, cache, dev_slots));
  if (!dev_q_out) return api_fail(ctx, TURQ_E_INVALID_ARG, "null argument");
  if ((uintptr_t)dev_q_out % 16 != 0) return api_fail(ctx, TURQ_E_ALIGN, "outputs must be 16-byte aligned");
  turq::HeadRowsArgs a{};
  a.q = dev_q; a.k = dev_k; a.v = dev_v;
  a.q_stride = q_stride; a.k_stride = k_stride; a.v_stride = v_stride;
  a.x_dtype = x_dtype; a.out_dtype = out_dtype;
  a.n_tokens = n_tokens; a.hq = n_q_heads; a.hkv = hkv;
  a.wq = dev_q_weight; a.wk = dev_k_weight; a.eps = eps;
  a.table = reinterpret_cast<const float2*>(dev_table); a.n_positions = n_positions;
  a.half_rot = rotary_dim / 2; a.interleaved = interleaved != 0; a.positions = dev_positions;
  a.q_out = dev_q_out;
  a.cache = turq::pages_of(cache); a.slots = dev_slots;
  a.status = ctx->dev_status;
  return run_head_rows(ctx, d, a, stream, "kv_append launch");
}

int32_t turq_kv_write(turq_ctx* ctx, turq_kv_cache* cache, const void* dev_k, int64_t k_stride, const void* dev_v, int64_t v_stride,
                      int32_t x_dtype, int64_t n_tokens, const int64_t* dev_slots, void* stream) {
  if (!ctx || !cache) return api_fail(ctx, TURQ_E_INVALID_ARG, "null argument");
  if (!elem_bytes(x_dtype)) return api_fail(ctx, TURQ_E_DTYPE, "rows must be F32, F16 or BF16");
  const int d = cache->head_dim, hkv = cache->n_kv_heads;
  TQ_TRY(check_tokens(ctx, n_tokens, 0, hkv, d));
  if (n_tokens == 0) return TURQ_OK;
  TQ_TRY(check_rows(ctx, dev_k, k_stride, (int64_t)hkv * d, x_dtype));
  TQ_TRY(check_rows(ctx, dev_v, v_stride, (int64_t)hkv * d, x_dtype));
  TQ_TRY(check_cache(ctx, cache, dev_slots));
  turq::HeadRowsArgs a{};
  a.k = dev_k; a.v = dev_v;
  a.k_stride = k_stride; a.v_stride = v_stride;
  a.x_dtype = x_dtype;
  a.n_tokens = n_tokens; a.hkv = hkv;
  a.cache = turq::pages_of(cache); a.slots = dev_slots;
  a.status = ctx->dev_status;
  return run_head_rows(ctx, d, a, stream, "kv_write launch");
}

int32_t turq_kv_read(turq_ctx* ctx, const turq_kv_cache* cache, const int64_t* dev_slots, int64_t n_tokens, int32_t out_dtype,
                     void* dev_k_out, void* dev_v_out, void* stream) {
  if (!ctx || !cache) return api_fail(ctx, TURQ_E_INVALID_ARG, "null argument");
  if (!elem_bytes(out_dtype)) return api_fail(ctx, TURQ_E_DTYPE, "rows must be F32, F16 or BF16");
  const int d = cache->head_dim, hkv = cache->n_kv_heads;
  TQ_TRY(check_tokens(ctx, n_tokens, 0, hkv, d));
  if (n_tokens == 0) return TURQ_OK;
  TQ_TRY(check_cache(ctx, cache, dev_slots));
  if (!dev_k_out || !dev_v_out) return api_fail(ctx, TURQ_E_INVALID_ARG, "null argument");
  if ((uintptr_t)dev_k_out % 16 != 0 || (uintptr_t)dev_v_out % 16 != 0) return api_fail(ctx, TURQ_E_ALIGN, "outputs must be 16-byte aligned");
  turq::DeviceScope on(ctx->device);
  if (on.status != cudaSuccess) return api_cuda_fail(ctx, on.status, "kv_read launch");
  const turq::KvPages pages = turq::pages_of(cache);
  const cudaError_t e = turq::launch_kv_read(d, pages, dev_slots, n_tokens, out_dtype, dev_k_out, dev_v_out, ctx->dev_status, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return api_cuda_fail(ctx, e, "kv_read launch");
  ctx->launches++;
  return TURQ_OK;
}

}  // extern "C"
