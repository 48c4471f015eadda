// Attention of new tokens over a paged cache (src/models/qwen3.rs:308-505; src/models/attention/cpu_flash).
// out[t, h] = sum_j p_j V_j / sum_j p_j with p_j = exp(scale q . K_j - m), one pass over the keys with the
// running maximum m and sum. The entry and the choice between the kernels: up to TOKEN_ROWS rows (new tokens x query
// heads) per key head of a sequence go to attend_tokens.cu, more to attend_tiles.cu. A call may hold both; the lengths
// are on the device, so both are launched and each takes its own.
#include <cfloat>

#include "attend.cuh"
#include "attend_launch.h"
#include "turq_internal.h"

namespace turq {

// The workspace: pieces of single tokens' rows with their maxima and sums, pieces of tiles.
struct AttendWorkspace {
  size_t off_ml = 0, off_tiles = 0, bytes = 0;
  int max_chunks = 1, part_rows = 0, chunk = TOKEN_CHUNK_MAX;
  int64_t pieces = 0;
  bool cluster = false, tokens = false, tiles = false;  // which kernels the call may need
};
static AttendWorkspace attend_workspace(const turq_kv_cache* kc, int64_t n_tokens, int32_t n_seqs, int32_t n_q_heads, int64_t max_new,
                                        int64_t max_context) {
  AttendWorkspace w;
  const int64_t group = n_q_heads / kc->n_kv_heads, most = max_new < n_tokens ? max_new : n_tokens;
  auto up = [](size_t v) { return (v + 255) & ~(size_t)255; };
  if (group < 1 || group > TILE_ROWS / 2) return w;
  w.tokens = group <= TOKEN_ROWS;
  w.tiles = most * group > TOKEN_ROWS;
  if (w.tokens) {
    w.part_rows = (int)(w.tiles ? TOKEN_ROWS : most * group);
    const TokenPlan p = plan_tokens((int64_t)n_seqs * kc->n_kv_heads, max_context, kc->sm_count, token_ctas(kc->dtype == TURQ_Q8_0, w.part_rows <= 8), w.tiles);
    w.chunk = (int)p.chunk;
    w.max_chunks = (int)p.chunks;
    w.cluster = p.cluster;
    if (p.chunks > 1 && !p.cluster) {
      const size_t rows = (size_t)n_seqs * kc->n_kv_heads * p.chunks * w.part_rows;
      w.off_ml = up(rows * kc->head_dim * 4);
      w.off_tiles = w.bytes = w.off_ml + up(rows * 8);
    }
  }
  if (w.tiles) {
    w.pieces = plan_tile_pieces(n_tokens, n_seqs, group, kc->n_kv_heads, max_context, kc->sm_count);
    if (w.pieces > 0) w.bytes += 256 + (size_t)w.pieces * TILE_ROWS * (8 + 8 + (size_t)kc->head_dim * 4);
  }
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
  if (!(scale > 0.f) || scale > FLT_MAX / 2.f) return api_fail(ctx, TURQ_E_INVALID_ARG, "scale must be positive and finite (below 2^127)");
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
  a.chunk = w.chunk;
  a.cluster = w.cluster;
  a.part_rows = w.part_rows;
  a.tile_pieces = (int)w.pieces;
  a.sms = ctx->sm_count;
  if (w.pieces > 0) {
    uint8_t* const t = static_cast<uint8_t*>(dev_workspace) + w.off_tiles;
    a.tile_head = reinterpret_cast<int*>(t);
    a.tile_rows = reinterpret_cast<int64_t*>(t + 256);
    a.tile_ml = reinterpret_cast<float2*>(t + 256 + w.pieces * turq::TILE_ROWS * 8);
    a.tile_part = reinterpret_cast<float*>(t + 256 + w.pieces * turq::TILE_ROWS * 16);
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaSuccess;
  int launches = 0;
  if (w.tiles) {
    int64_t blocks = turq::tile_blocks(n_tokens, n_seqs, a.group, hkv);
    if (blocks < w.pieces) blocks = w.pieces;
    if (blocks > INT32_MAX) return api_fail(ctx, TURQ_E_LIMIT, "more row tiles than a launch takes");
    e = turq::launch_attend_tiles(cache, a, (unsigned)blocks, s, &launches);
  }
  if (e == cudaSuccess && w.tokens) {
    a.beside = w.tiles;
    e = turq::launch_attend_tokens(cache, a, s, &launches);
  }
  if (e == cudaSuccess && w.pieces > 0) e = turq::launch_join_tiles(cache, a, s, &launches);
  ctx->launches += launches;
  if (e != cudaSuccess) return turq::api_cuda_fail(ctx, e, "attention launch");
  return TURQ_OK;
}

}  // extern "C"
