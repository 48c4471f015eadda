// What the kernels of attention over a paged cache share.
#pragma once
#include "../../include/turq.h"
#include "attend_plan.h"
#include "device_utils.cuh"
#include "kvcache.cuh"
#include "tc_common.cuh"

namespace turq {

struct AttendArgs {
  KvPages cache;
  const uint16_t* q;
  int64_t q_stride;
  int q_bf16;
  int64_t n_tokens;
  int hq, group;
  const int32_t *starts, *contexts, *page_table;
  int64_t table_stride;
  int n_seqs;
  int64_t max_new, max_context;
  float scale_log2;  // scale x log2 e: weights are powers of two
  int causal, out_dtype;
  void* out;
  int* status;
  float *part, *part_ml;  // pieces of rows on their way to the kernel that joins them
  int max_chunks, part_rows;
  int chunk;              // keys of a chunk of a single token's context
  int cluster;            // the chunks of a context are one cluster
  int beside;             // the tokens' launch runs beside the tiles' and need not wait for it before it ends
  // tiles of rows: room for that many pieces (0: no row's keys are cut), their header, maxima and sums, sums, and the rows' places in out
  int tile_pieces, sms;
  int* tile_head;
  float2* tile_ml;
  float* tile_part;
  int64_t* tile_rows;
};

__device__ __forceinline__ void report(int* status, int code) { *reinterpret_cast<volatile int*>(status) = code; }

__device__ __forceinline__ Span span_of(const AttendArgs& a, int i) {
  const Span s = cut_span(a.starts[i], a.starts[i + 1], a.contexts[i], a.n_tokens, a.max_new, a.max_context);
  if (s.cut) report(a.status, TURQ_E_INVALID_ARG);
  return s;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Q8_0 keys and values meet their products in f16: a block whose scale times 127 is beyond f16 (scales above 515.5) would be infinite
// there. It is reported. What a thread has seen of scales' magnitudes, both of a pair; NaN passes through the products by itself.
__device__ __forceinline__ void report_beyond_f16(const AttendArgs& a, __half2 largest) {
  if (__hgt(__low2half(largest), __float2half_rn(515.5f)) || __hgt(__high2half(largest), __float2half_rn(515.5f)))
    report(a.status, TURQ_E_INVALID_ARG);
}

// Scores are compared and subtracted as the products gave them, and multiplied (by scale x log2 e, times what a row of q was divided by)
// afterwards: the product of a large score would be off by its own f32 rounding, in every weight a different one. Where pieces of a row meet,
// their maxima come times the power of two in the row's multiplier, which is exact, and what is left of it, from 1 to 2, is the same for
// all rows: a weight is 2^((maximum - largest) * joined_factor).
__device__ __forceinline__ float row_mul(const AttendArgs& a, float up) {
  return fmaxf(a.scale_log2 * up, __uint_as_float(1u));  // not zero: the score of a key that is not seen is -inf
}
__device__ __forceinline__ float joined_max(float m, float mul) {
  return m == -INFINITY ? m : m * __uint_as_float(__float_as_uint(mul) & 0x7F800000u);
}
__device__ __forceinline__ float joined_factor(const AttendArgs& a) { return __uint_as_float((__float_as_uint(a.scale_log2) & 0x7FFFFFu) | 0x3F800000u); }

// Two f32 rounded to the 16-bit type of the products.
template <bool BF>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
  if (BF) {
    const __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&t);
  }
  const __half2 t = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&t);
}
// Four int8 -> half2 pairs (b0, b1), (b2, b3), exact before the scale: 1024 + (q + 128) less 1152.
__device__ __forceinline__ void halves_of(uint32_t w, __half2 scale, uint32_t& lo, uint32_t& hi) {
  const uint32_t u = w ^ 0x80808080u;
  const __half2 off = __float2half2_rn(1152.f);
  lo = h22u(__hmul2(__hsub2(pair01(u), off), scale));
  hi = h22u(__hmul2(__hsub2(pair23(u), off), scale));
}
// A box of a plane of pages to shared memory, reported to a barrier there.
__device__ __forceinline__ void copy_box3(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
               ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}

// Two neighbouring elements of the output, rounded once.
__device__ __forceinline__ void store_out2(void* out, int dtype, int64_t i, float a, float b) {
  if (dtype == TURQ_F32) *reinterpret_cast<float2*>(static_cast<float*>(out) + i) = make_float2(a, b);
  else if (dtype == TURQ_BF16) *reinterpret_cast<__nv_bfloat162*>(static_cast<__nv_bfloat16*>(out) + i) = __floats2bfloat162_rn(a, b);
  else *reinterpret_cast<__half2*>(static_cast<__half*>(out) + i) = __floats2half2_rn(a, b);
}

}  // namespace turq
