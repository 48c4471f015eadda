// Attention of new tokens over a paged cache (src/models/qwen3.rs:308-505; src/models/attention/cpu_flash).
// out[t, h] = sum_j p_j V_j / sum_j p_j with p_j = exp(scale q . K_j - m), one pass over the keys with the
// running maximum m and sum.
#include <cfloat>

#include "attend.cuh"
#include "attend_launch.h"
#include "turq_internal.h"

namespace turq {

// One warp per row: D / 32 elements a lane.
template <int D>
__global__ void __launch_bounds__(128) attend_rows_kernel(const AttendArgs a) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31, seq = blockIdx.y;
  const Span sp = span_of(a, seq);
  if (sp.n * a.group <= TOKEN_ROWS) return;
  const int64_t row = (int64_t)blockIdx.x * 4 + threadIdx.x / 32;
  if (row >= sp.n * a.hq) return;
  const int64_t t = row / a.hq;
  const int h = (int)(row % a.hq), kv = h / a.group;
  const int64_t seen = keys_seen(sp, t, a.causal);
  float q[E], o[E];
  const uint16_t* qp = a.q + (sp.first + t) * a.q_stride + h * D + lane * E;
#pragma unroll
  for (int e = 0; e < E; e++) {
    q[e] = a.q_bf16 ? __uint_as_float((uint32_t)qp[e] << 16) : f16_bits_to_f32(qp[e]);
    o[e] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int64_t j = 0; j < seen; j++) {
    const int32_t page = a.page_table[seq * a.table_stride + (j >> a.cache.page_shift)];
    const bool known = page >= 0 && page < a.cache.n_pages;
    if (!known) *reinterpret_cast<volatile int*>(a.status) = TURQ_E_INVALID_ARG;
    const int64_t at = a.cache.row(((int64_t)(known ? page : 0) << a.cache.page_shift) + (j & (a.cache.page_size - 1)), kv);
    float k[E], v[E], s = 0.f;
#pragma unroll
    for (int e = 0; e < E; e++) {
      const int64_t i = at * D + lane * E + e;
      if (a.cache.dtype == TURQ_Q8_0) {
        k[e] = (float)reinterpret_cast<const int8_t*>(a.cache.k)[i] * __half2float(a.cache.ks[i / 32]);
        v[e] = (float)reinterpret_cast<const int8_t*>(a.cache.v)[i] * __half2float(a.cache.vs[i / 32]);
      } else {
        const uint16_t kb = reinterpret_cast<const uint16_t*>(a.cache.k)[i], vb = reinterpret_cast<const uint16_t*>(a.cache.v)[i];
        k[e] = a.cache.dtype == TURQ_BF16 ? __uint_as_float((uint32_t)kb << 16) : f16_bits_to_f32(kb);
        v[e] = a.cache.dtype == TURQ_BF16 ? __uint_as_float((uint32_t)vb << 16) : f16_bits_to_f32(vb);
      }
      if (!known) k[e] = v[e] = 0.f;
      s += q[e] * k[e];
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, d);
    s *= a.scale_log2;
    const float m2 = fmaxf(m, s), was = m2 == -INFINITY ? 0.f : exp2f(m - m2), p = m2 == -INFINITY ? 0.f : exp2f(s - m2);
    l = l * was + p;
#pragma unroll
    for (int e = 0; e < E; e++) o[e] = o[e] * was + p * v[e];
    m = m2;
  }
  const int64_t out = ((sp.first + t) * a.hq + h) * D + lane * E;
#pragma unroll
  for (int e = 0; e < E; e++) {
    const float y = l > 0.f ? o[e] / l : 0.f;
    if (a.out_dtype == TURQ_F32) static_cast<float*>(a.out)[out + e] = y;
    else if (a.out_dtype == TURQ_BF16) static_cast<__nv_bfloat16*>(a.out)[out + e] = __float2bfloat16_rn(y);
    else static_cast<__half*>(a.out)[out + e] = __float2half_rn(y);
  }
}

// The workspace: pieces of single tokens' rows, their maxima and sums.
struct AttendWorkspace {
  size_t off_ml = 0, bytes = 0;
  int max_chunks = 1, part_rows = 0;
};
static AttendWorkspace attend_workspace(const turq_kv_cache* kc, int64_t n_tokens, int32_t n_seqs, int32_t n_q_heads, int64_t max_new,
                                        int64_t max_context) {
  AttendWorkspace w;
  const int64_t group = n_q_heads / kc->n_kv_heads, most = max_new < n_tokens ? max_new : n_tokens;
  if (group < 1 || group > TOKEN_ROWS) return w;
  w.max_chunks = (int)token_chunks_max(max_context);
  w.part_rows = (int)(most * group < TOKEN_ROWS ? most * group : TOKEN_ROWS);
  if (w.max_chunks == 1) return w;
  const size_t rows = (size_t)n_seqs * kc->n_kv_heads * w.max_chunks * w.part_rows;
  w.off_ml = rows * kc->head_dim * 4;
  w.bytes = w.off_ml + rows * 8;
  return w;
}

}  // namespace turq

extern "C" {

size_t turq_kv_attention_workspace(const turq_kv_cache* cache, int64_t n_tokens, int32_t n_seqs, int32_t n_q_heads, int64_t max_new,
                                   int64_t max_context) {
  if (!cache || n_tokens <= 0 || n_seqs <= 0 || n_q_heads <= 0 || max_new <= 0 || max_context <= 0) return 0;
  return turq::attend_workspace(cache, n_tokens, n_seqs, n_q_heads, max_new, max_context).bytes;
}

int32_t turq_kv_attention(turq_ctx* ctx, const turq_kv_cache* cache, const void* dev_q, int64_t q_stride, int32_t q_dtype,
                          int64_t n_tokens, int32_t n_q_heads, const int32_t* dev_starts, const int32_t* dev_contexts,
                          const int32_t* dev_page_table, int64_t table_stride, int32_t n_seqs, int64_t max_new, int64_t max_context,
                          float scale, int32_t causal, int32_t out_dtype, void* dev_out, void* dev_workspace, size_t workspace_bytes,
                          void* stream) {
  using turq::api_fail;
  if (!ctx || !cache) return api_fail(ctx, TURQ_E_INVALID_ARG, "null argument");
  if (q_dtype != TURQ_F16 && q_dtype != TURQ_BF16) return api_fail(ctx, TURQ_E_DTYPE, "q must be F16 or BF16");
  if (cache->dtype == TURQ_BF16 && q_dtype != TURQ_BF16) return api_fail(ctx, TURQ_E_DTYPE, "a BF16 cache takes BF16 queries");
  if (out_dtype != TURQ_F32 && out_dtype != TURQ_F16 && out_dtype != TURQ_BF16) return api_fail(ctx, TURQ_E_DTYPE, "out must be F32, F16 or BF16");
  const int d = cache->head_dim, hkv = cache->n_kv_heads;
  if (n_q_heads < 1 || n_q_heads % hkv != 0 || n_q_heads / hkv > 128)
    return api_fail(ctx, TURQ_E_SHAPE, "n_q_heads must be a multiple of the cache's heads, at most 128 to one");
  if (n_tokens < 0 || n_tokens > INT32_MAX / 2 || n_seqs < 0 || n_seqs > 65535 || hkv > 65535) return api_fail(ctx, TURQ_E_SHAPE, "n_tokens or n_seqs out of range");
  if (max_new < 0 || max_new > INT32_MAX / 2 || max_context < 0 || max_context > INT32_MAX / 2) return api_fail(ctx, TURQ_E_SHAPE, "max_new or max_context out of range");
  if (!(scale > 0.f) || scale > FLT_MAX) return api_fail(ctx, TURQ_E_INVALID_ARG, "scale must be positive and finite");
  if (n_tokens == 0 || n_seqs == 0 || max_new == 0) return TURQ_OK;
  if (table_stride < (max_context + cache->page_size - 1) / cache->page_size)
    return api_fail(ctx, TURQ_E_SHAPE, "the page table has fewer pages a sequence than max_context needs");
  if (!dev_q || !dev_starts || !dev_contexts || (!dev_page_table && max_context > 0) || !dev_out) return api_fail(ctx, TURQ_E_INVALID_ARG, "null argument");
  if (q_stride < (int64_t)n_q_heads * d) return api_fail(ctx, TURQ_E_SHAPE, "the stride of q is less than the width of its heads");
  if ((uintptr_t)dev_q % 16 != 0 || q_stride % 8 != 0 || (uintptr_t)dev_out % 16 != 0 || (uintptr_t)dev_workspace % 16 != 0)
    return api_fail(ctx, TURQ_E_ALIGN, "q, out and the workspace must be 16-byte aligned, the stride of q whole 16 bytes");
  if ((uintptr_t)dev_starts % 4 != 0 || (uintptr_t)dev_contexts % 4 != 0 || (uintptr_t)dev_page_table % 4 != 0)
    return api_fail(ctx, TURQ_E_ALIGN, "starts, contexts and the page table must be 4-byte aligned");
  if (cache->device != ctx->device) return api_fail(ctx, TURQ_E_INVALID_ARG, "cache and context must live on the same device");
  if (workspace_bytes > 0 && !dev_workspace) return api_fail(ctx, TURQ_E_INVALID_ARG, "null argument");
  if (workspace_bytes < turq_kv_attention_workspace(cache, n_tokens, n_seqs, n_q_heads, max_new, max_context))
    return api_fail(ctx, TURQ_E_SHAPE, "the workspace is smaller than turq_kv_attention_workspace");
  turq::AttendArgs a{};
  a.cache = turq::pages_of(cache);
  a.q = static_cast<const uint16_t*>(dev_q);
  a.q_stride = q_stride;
  a.q_bf16 = q_dtype == TURQ_BF16;
  a.n_tokens = n_tokens;
  a.hq = n_q_heads;
  a.group = n_q_heads / hkv;
  a.starts = dev_starts;
  a.contexts = dev_contexts;
  a.page_table = dev_page_table;
  a.table_stride = table_stride;
  a.n_seqs = n_seqs;
  a.max_new = max_new;
  a.max_context = max_context;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.causal = causal != 0;
  a.out_dtype = out_dtype;
  a.out = dev_out;
  a.status = ctx->dev_status;
  turq::DeviceScope on(ctx->device);
  if (on.status != cudaSuccess) return turq::api_cuda_fail(ctx, on.status, "attention launch");
  const turq::AttendWorkspace w = turq::attend_workspace(cache, n_tokens, n_seqs, n_q_heads, max_new, max_context);
  a.part = static_cast<float*>(dev_workspace);
  a.part_ml = reinterpret_cast<float*>(static_cast<uint8_t*>(dev_workspace) + w.off_ml);
  a.max_chunks = w.max_chunks;
  a.part_rows = w.part_rows;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaSuccess;
  const int64_t most = max_new < n_tokens ? max_new : n_tokens;
  int launches = 0;
  if (most * a.group > turq::TOKEN_ROWS) {
    const dim3 grid((unsigned)((most * n_q_heads + 3) / 4), (unsigned)n_seqs);
    if (d == 64) turq::attend_rows_kernel<64><<<grid, 128, 0, s>>>(a);
    else turq::attend_rows_kernel<128><<<grid, 128, 0, s>>>(a);
    e = cudaGetLastError();
    launches++;
  }
  if (e == cudaSuccess && a.group <= turq::TOKEN_ROWS) e = turq::launch_attend_tokens(cache, a, s, &launches);
  ctx->launches += launches;
  if (e != cudaSuccess) return turq::api_cuda_fail(ctx, e, "attention launch");
  return TURQ_OK;
}

}  // extern "C"
