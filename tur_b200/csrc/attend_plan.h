// Index arithmetic of attention over a paged cache, the same on the host (sizes of grids and workspaces, CPU
// tests) and in the kernels.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define TQ_HD __host__ __device__ __forceinline__
#else
#define TQ_HD inline
#endif

namespace turq {

// What the device arrays say of a sequence, cut to what the call allows.
struct Span {
  int64_t first, n;  // rows of q
  int64_t ctx;       // keys
  bool cut;          // something was outside its bounds
};
TQ_HD Span cut_span(int64_t lo, int64_t hi, int64_t ctx, int64_t n_tokens, int64_t max_new, int64_t max_context) {
  Span s;
  s.cut = lo < 0 || hi < lo || hi > n_tokens || hi - lo > max_new || ctx < 0 || ctx > max_context;
  s.first = lo < 0 ? 0 : lo > n_tokens ? n_tokens : lo;
  int64_t end = hi > n_tokens ? n_tokens : hi;
  if (end > s.first + max_new) end = s.first + max_new;
  s.n = end > s.first ? end - s.first : 0;
  s.ctx = ctx < 0 ? 0 : ctx > max_context ? max_context : ctx;
  return s;
}
// Keys that new token t of a sequence sees: all before its own and its own.
TQ_HD int64_t keys_seen(const Span& s, int64_t t, bool causal) {
  if (!causal) return s.ctx;
  const int64_t e = s.ctx - s.n + t + 1;
  return e < 0 ? 0 : e;
}

// ---- single tokens: up to TOKEN_ROWS rows (new tokens x query heads of a key head)
constexpr int TOKEN_ROWS = 16;
// A context is cut into chunks whose length goes by the context alone: a row's bits do not depend on the
// other sequences of the call. Up to sixteen chunks of at least 256 keys while that fills a GPU with one
// sequence of eight heads, not above 1024 keys: a chunk of rows x head_dim f32 leaves the SM and comes back.
TQ_HD int64_t token_chunk(int64_t ctx) {
  const int64_t c = (ctx + 1023) / 1024 * 64;  // ctx / 16 in whole 64s
  return c < 256 ? 256 : c > 1024 ? 1024 : c;
}
TQ_HD int64_t token_chunks(int64_t ctx) { return ctx <= 0 ? 1 : (ctx + token_chunk(ctx) - 1) / token_chunk(ctx); }
// The most chunks that any context up to max_context has (the count falls by one where the length steps up).
TQ_HD int64_t token_chunks_max(int64_t max_context) {
  if (max_context <= 4096) return token_chunks(max_context);
  const int64_t n = (max_context + 1023) / 1024;
  return n < 16 ? 16 : n;
}

}  // namespace turq
