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
// The contexts of a call are cut into chunks of one length, a CTA each, three or four CTAs at a time on an SM. A CTA has costs of its
// own (the way from the lengths over the page table to the first keys, the join of its warps) worth TOKEN_OVERHEAD keys, and 1 to 4 CTAs
// at a time on an SM take TOKEN_DEPTH times as long as the keys of one of them would if they did not share it; a wave that is not the
// only one costs a full one. The length with the least cost is taken, over several waves at most TOKEN_CHUNK_WAVES: sequences differ, and
// the longest should not end alone. Measured, us: one user at 16384 keys (32 heads on 8 of 128, bf16) in chunks of 256 18.4, 512 13.1,
// 1024 17.3; 24 users at 4096 256 81, 1024 70, 2048 70; two at 120000 1024 156, 4480 148; one at 30000 and 31 at 500 2560 42, 6016 77.
constexpr int TOKEN_STEP = 128, TOKEN_CHUNK_MAX = 8192, TOKEN_CHUNK_WAVES = 3200, TOKEN_OVERHEAD = 96;
constexpr int TOKEN_DEPTH[5] = {0, 140, 162, 216, 264};  // hundredths
constexpr int token_ctas(bool q8, bool eight_rows) { return q8 && eight_rows ? 4 : 3; }
inline int64_t plan_token_chunk(int64_t pairs /* sequences x key heads */, int64_t max_context, int sms, int ctas) {
  int64_t best = TOKEN_STEP, cost = -1;
  for (int64_t c = TOKEN_STEP; c <= TOKEN_CHUNK_MAX; c += TOKEN_STEP) {
    const int64_t chunks = max_context <= c ? 1 : (max_context + c - 1) / c, n = pairs * chunks, slots = (int64_t)ctas * sms;
    const int64_t keys = c < max_context ? c : max_context, deep = (n + sms - 1) / sms;
    const int64_t t = (n > slots ? (n + slots - 1) / slots * TOKEN_DEPTH[ctas] : TOKEN_DEPTH[deep]) * (keys + TOKEN_OVERHEAD);
    if (cost < 0 || (t < cost && (n <= slots || c <= TOKEN_CHUNK_WAVES))) {
      cost = t;
      best = c;
    }
    if (c >= max_context) break;
  }
  return best;
}

// Chunks as one cluster, whose blocks join their pieces over shared memory: no workspace, no second launch. Up to eight while all
// run at once anyway, up to sixteen while they also find an SM each (more are hard to place: 3 users at 4096 keys in clusters
// of 16 18.7 us, joined by a launch 11.1). Measured in a captured graph / called one by one, us, one user, 8 heads of 128, cluster
// against launch: 1024 keys 6.2 / - against 6.6 / -, 4096 keys 9.2 / 11.0 against 8.2 / 16.1 (the second launch and the workspace cost
// the host 5); 8192 keys in chunks of 512 12.3 against 9.9, which is why a chunk may not be longer than 256 for it.
constexpr int TOKEN_CLUSTER = 16, TOKEN_CLUSTER_KEYS = 256;
// Beside tiles the tokens get the SMs that those leave, late: chunks for half as many pairs, which are shorter and more, end sooner, while
// whether clusters find room goes by the pairs that there are. us, a chunk of 512 on 4096 keys and so many users at 200 to 6000 (32
// heads on 8 of 128), length by half of the pairs / by all, bf16 and Q8_0: 4 users 62.1 / 63.1 and 66.0 / 67.1, 8 73.5 / 74.7 and 76.7 /
// 84.7, 16 87.3 / 90.9 and 89.3 / 108.4, 32 142.0 / 130.8 and 112.9 / 114.2, 64 205.7 / 205.3 and 177.0 / 175.9; six sequences
// (512 of 8000, 33 of 1000, four users; 40 on 10 of 64, f16) 86.1 / 95.9. Room by half of the pairs too: 8 80.2 and 76.7, 16 95.0 and
// 110.4, 32 136.0 and 134.3.
struct TokenPlan { int64_t chunk, chunks; bool cluster; };
inline TokenPlan plan_tokens(int64_t pairs, int64_t max_context, int sms, int ctas, bool beside = false) {
  TokenPlan p;
  const int64_t sixteenth = (max_context + TOKEN_CLUSTER * TOKEN_STEP - 1) / (TOKEN_CLUSTER * TOKEN_STEP) * TOKEN_STEP;
  p.chunk = plan_token_chunk(beside ? (pairs + 1) / 2 : pairs, max_context, sms, ctas);
  if (sixteenth > p.chunk && sixteenth <= TOKEN_CLUSTER_KEYS && pairs * TOKEN_CLUSTER <= sms) p.chunk = sixteenth;
  p.chunks = max_context <= p.chunk ? 1 : (max_context + p.chunk - 1) / p.chunk;
  p.cluster = p.chunks > 1 && p.chunks <= TOKEN_CLUSTER && pairs * p.chunks <= (int64_t)(p.chunks <= 8 ? ctas : 1) * sms;
  return p;
}

// A warp's ring of copies: how many of its `own` steps have been requested once it has taken `taken` of them (the one that it takes next
// among them). What it has not taken is still on its way.
TQ_HD int ring_requested(int own, int taken, int stages) { return taken + stages < own ? taken + stages : own; }

// ---- tiles of rows: TILE_ROWS rows (two row tiles of the tensor core) a CTA, a CTA an SM
constexpr int TILE_ROWS = 256;
constexpr int TILE_SPLITS = 32;     // pieces of a tile's keys that the join takes
constexpr int TILE_OVERHEAD = 4;    // what a CTA costs beside its key tiles, and what the join does, in key tiles of 128
constexpr int TILE_WAVES = 3;       // pieces are no more than that many CTAs an SM
// Both measured, us (least of four medians; 32 heads on 8 of 128, bf16, but where 40 on 10 of 64, f16). Overhead 2 / 4 / 8: 128 new tokens on
// 20000 keys 59.0 / 59.0 / 59.0, 512 on 8000 74.5 / 74.5 / 74.6, 4 x 200 on 6000 95.5 / 95.4 / 95.5, 512 on 8000 (of 64) 88.5 / 82.4 / 84.5, with
// 33 on 1000 beside it 85.1 / 83.4 / 84.3. Waves 2 / 3 / 4: 128 on 20000 63.3 / 59.0 / 59.2, 512 on 8000 75.9 / 74.5 / 76.0, 1500 on 30000
// 790 / 647 / 606, 300 on 4000 40.4 / 40.2 / 38.8, 4 x 200 on 6000 95.7 / 95.4 / 96.9, 512 on 8000 (of 64) 83.3 / 82.4 / 83.5, 3 x 1000 on their
// own 46.9 / 46.9 / 46.8: 3 is the middle of what small and large calls would take.
// What cutting the keys of each of `ctas` tiles (the longest with `iters` key tiles) into s pieces costs: waves x (key tiles + overhead).
// The kernel takes the s that costs least.
TQ_HD int64_t tile_split_cost(int s, int ctas, int iters, int pieces, int sms) {
  if (s > 1 && ((int64_t)s * ctas > pieces || 2 * s > iters)) return INT32_MAX;
  return (int64_t)((s * ctas + sms - 1) / sms) * ((iters + s - 1) / s + TILE_OVERHEAD) + (s > 1 ? TILE_OVERHEAD : 0);
}
// Pairs of row tiles x key heads that a call has at most (floor(n / p) + sequences is no less than the sum of ceil(n_i / p)).
inline int64_t tile_blocks(int64_t n_tokens, int64_t n_seqs, int64_t group, int64_t heads) {
  const int64_t per_cta = TILE_ROWS / 2 / group * 2;  // tokens
  return (n_seqs == 1 ? (n_tokens + per_cta - 1) / per_cta : n_tokens / per_cta + n_seqs) * heads;
}
// Pieces that a call gets room for: none where its tokens make more tiles than cutting could gain from.
inline int64_t plan_tile_pieces(int64_t n_tokens, int64_t n_seqs, int64_t group, int64_t heads, int64_t max_context, int sms) {
  const int64_t full = n_tokens / (TILE_ROWS / 2 / group * 2) * heads;  // tiles that are full, if all tokens are one sequence's
  int64_t each = (max_context + 127) / 128 / 2;
  if (each > TILE_SPLITS) each = TILE_SPLITS;
  if (2 * full > TILE_WAVES * sms || each < 2) return 0;
  const int64_t most = tile_blocks(n_tokens, n_seqs, group, heads) * each;
  return most < TILE_WAVES * sms ? most : TILE_WAVES * sms;
}

}  // namespace turq
