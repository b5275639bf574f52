// Attention over a conversation's cached context: B x T queries over a 16-bit cache
// (i4_attn_window), one in pages (i4_attn_paged) or an 8-bit one (i4_attn_kv8), under an optional
// sliding window whose first tokens stay visible.
//   out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),  s_j = scale q . k_j,
// over the visible j in one pass, with a running maximum m and sum.
#include "i4_ctx.h"

// the bounds and the workspace of a call
struct i4_span {
  int window, sinks;
  void* workspace;
  int32_t* counters;
};

namespace i4 {

// When the context tiles of many rows are shared out: several sequences whose lengths the host
// does not know (device positions, counts), up to kSharedTiles row tiles of all kv heads, and at
// least kSharedSpan context tiles that a row tile may see.  Measured, shared out against split by
// ctx_split's cost, us: 4 x 400 padded tokens behind up to 9001 positions 184 / 257, 16 x 100
// behind 8000 114 / 209, 16 x 17 behind 16000 103 / 134, 3 x 1000 behind 2000 106 / 102.  The
// parts that runs leave (66 KB each, up to 1024) cost it some 25 us: fewer context tiles, 4 x 400
// behind 1000: 48 / 43, 40 x 8 behind 900: 39 / 32; more row tiles, 8 x 300 of 56 heads behind
// 1000: 105 / 81; and one prompt, whose row tiles the longest-first order evens out: 3000 tokens
// 115 / 84.
static constexpr int kSharedTiles = 1024, kSharedSpan = 32;

// How a call is split: a rule on its sizes alone (no device value), so that the workspace
// can be named before the call.
struct CtxSplit {
  int S, wgs;      // k_ctx_tile's splits; k_ctx_rows' workgroups, or those of a shared-out call
  int64_t parts;   // rows that are written as parts
  int plan;        // entries of a shared-out call's plan, or 0
  size_t bytes() const {
    return (size_t)parts * ((KHD + 2) * 4) + ((size_t)plan * 4 + 255) / 256 * 256;
  }
};
// pages: of a call over pages; share: whether many rows' tiles may be shared out there
static CtxSplit ctx_split(int B, int T, int nq, int nkv, int keys, int window, int sinks,
                          bool pages, bool share) {
  const int R = T * (nq / nkv);
  const bool few = R <= kFewRows;
  // the context tiles of 64 that one row tile sees at most
  const int64_t span = few ? T : (kTileRows + nq / nkv - 1) / (nq / nkv) + 1;
  int64_t tiles = (keys + 63) / 64;
  if (window) {
    const int64_t most = ((int64_t)window + span + 126) / 64 + ((int64_t)sinks + 63) / 64;
    if (most < tiles) tiles = most;
  }
  const int64_t heads = (int64_t)B * nkv;
  if (few) {
    // as many workgroups as the chip holds at once (two a CU), or two or four times that
    // where the heads are too many to share that evenly; at least a tile for each wave
    int64_t w = heads <= 128 ? 512 : heads <= 256 ? 1024 : 2048;
    // Over pages, where heads are few, one workgroup a CU and fewer parts: a kv head's last
    // workgroup reads 32 parts in one round of loads, and another round costs more than it saves
    // in the tiles until they are many.  4 kv heads of one sequence over 30000 positions 20.8 us
    // with 32 parts each, 22.9 with 64, 36.1 with 118, over 60000 30.6 with 32 and 64; one over
    // 30000 20.0, 18.8 and 24.1.  Of several sequences, with 24 parts on average, 48 and (of 4 kv
    // heads 32, all that there are) 64: 2 of 4 over up to 16000 18.4, 22.1, 22.2, up to 100000
    // 71, 77, 77; 2 of one over up to 16000 15.8, 16.8, 16.8, up to 100000 52, 36, 34; 4 of one
    // over up to 100000 56, 43, 45.  8 of 4 over up to 4000 16.6 with 256 workgroups, 19.5 with
    // 512, up to 30000 77 and 79; but 16 of 8 over up to 16000 135 and 108.  (Over one run of rows
    // the splits are what they were: they decide a row's bits.)
    if (pages && heads <= 32) {
      const int parts = B > 1 ? (heads <= 6 && tiles > 400 ? 48 : 24)
                              : (tiles > (heads <= 2 ? 250 : 600) ? 64 : 32);
      w = tiles <= 128 || heads * parts > 256 ? 256 : heads * parts;
    }
    if (w > heads * ((tiles + 3) / 4)) w = heads * ((tiles + 3) / 4);
    if (w <= heads || heads > kShared) w = heads;
    return {1, (int)w, w > heads ? w * kFewRows : 0, 0};
  }
  const int64_t tiled = (R + kTileRows - 1) / kTileRows;
  if (pages && share && B > 1 && B * tiled <= kPlanned && heads * tiled <= kSharedTiles &&
      tiles >= kSharedSpan) {
    const int64_t w = runs_of(heads * tiled * (tiles + kRowTile));
    return {1, (int)w, 2 * w * kTileRows, (int)(B * tiled) + 2};
  }
  // Two workgroups fit a CU: 512 take 2.1 us a tile together, 256 that have their CU to
  // themselves 1.3 us.  Parts cost 1040 bytes a row, written and read, and a launch.
  const int64_t wgs = heads * ((R + kTileRows - 1) / kTileRows), rows = (int64_t)B * T * nq;
  double best = 0;
  int s = 1;
  for (int c = 1; c <= 64 && (c == 1 || c <= tiles / 4); ++c) {
    const int64_t w = wgs * c, rest = w % 512;
    const double rounds = 2.1 * (double)(w / 512) + (rest == 0 ? 0 : rest <= 256 ? 1.3 : 2.1);
    double t = rounds * (double)((tiles + c - 1) / c);
    if (c > 1) t += 4 + (double)rows * c * 1040 / 4e6;
    if (c == 1 || t < best) best = t, s = c;
  }
  return {s, 0, s > 1 ? rows * s : 0, 0};
}

static int launch(CtxArgs& a, int xt, int fmt, int keys, const i4_span& w, hipStream_t stream) {
  const CtxSplit sp = ctx_split(a.B, a.tk.T, a.nq, a.nkv, keys, w.window, w.sinks,
                                fmt == kPaged, a.tk.pos_dev || a.tk.counts);
  a.S = sp.S;
  a.wgs = sp.wgs;
  a.part = (float*)w.workspace;
  a.ml = a.part + sp.parts * KHD;
  a.counters = w.counters;
  a.plan = (int32_t*)(a.ml + 2 * sp.parts);
  a.tiles = (a.R + kTileRows - 1) / kTileRows;
  if (sp.plan) return i4_launch_ctx_shared(a, xt, stream);
  const int64_t grid = a.R <= kFewRows ? sp.wgs : (int64_t)a.tiles * sp.S * a.B * a.nkv;
  if (grid > kMaxGrid) return I4_ERR_SHAPE;
  return a.R <= kFewRows ? i4_launch_ctx_rows(a, xt, fmt, stream)
                         : i4_launch_ctx_tile(a, xt, fmt, stream);
}

}  // namespace i4

static size_t ctx_bytes(int B, int T, int n_heads, int n_kv_heads, int keys, int window, int sinks,
                        bool pages, bool share) {
  if (B < 1 || T < 1 || T > i4::KV_MAX_LEN || n_kv_heads < 1 || n_heads < n_kv_heads ||
      n_heads > 1024 || n_heads % n_kv_heads || keys < 1 || window < 0 || sinks < 0)
    return 0;
  if (n_kv_heads > 1024 || B > 65535) return 0;
  return i4::ctx_split(B, T, n_heads, n_kv_heads, keys, window, sinks, pages, share).bytes();
}

extern "C" {

size_t i4_attn_window_workspace_bytes(int B, int T, int n_heads, int n_kv_heads, int keys,
                                      int window, int sinks) {
  return ctx_bytes(B, T, n_heads, n_kv_heads, keys, window, sinks, false, false);
}
size_t i4_attn_paged_call_bytes(int B, int T, int n_heads, int n_kv_heads, int keys, int window,
                                int sinks, int on_device) {
  return ctx_bytes(B, T, n_heads, n_kv_heads, keys, window, sinks, true, on_device != 0);
}
size_t i4_attn_paged_workspace_bytes(int B, int T, int n_heads, int n_kv_heads, int keys,
                                     int window, int sinks) {
  const size_t split =
      i4_attn_paged_call_bytes(B, T, n_heads, n_kv_heads, keys, window, sinks, 0);
  const size_t shared =
      i4_attn_paged_call_bytes(B, T, n_heads, n_kv_heads, keys, window, sinks, 1);
  return split > shared ? split : shared;
}

// the positions that a call may attend (a host position is checked after this)
static int call_keys(const int32_t* pos_dev, int pos, int T, int len) {
  const int64_t end = (int64_t)pos + T;
  return pos_dev || end > len ? len : end < 1 ? 1 : (int)end;
}

// the checks that both caches share
static int query_check(const void* q, int x_dtype, int dtype, int B, int T, int64_t qbs,
                       int64_t qts, int64_t qhs, int n_heads, int nkv, const int32_t* pos_dev,
                       int pos, const int32_t* counts, int limit, int window, int sinks,
                       float scale, const void* out, const void* workspace, size_t have,
                       size_t need, const int32_t* counters) {
  if (!q || !out) return I4_ERR_NULL;
  if (x_dtype != dtype) return I4_ERR_DTYPE;
  const int rc = i4_check_tokens(B, T, n_heads, nkv, pos_dev, pos, counts, limit);
  if (rc) return rc;
  if (window < 0 || sinks < 0 || (window == 0 && sinks) || !(scale > 0.f) ||
      !(scale < __builtin_inff()))
    return I4_ERR_SHAPE;
  if ((T > 1 && qts < i4::KHD) || (B > 1 && qbs < i4::KHD) || (n_heads > 1 && qhs < i4::KHD))
    return I4_ERR_STRIDE;
  if (((uintptr_t)counters & 3) || ((uintptr_t)q & 15) || ((uintptr_t)out & 15) || (qbs & 7) ||
      (qts & 7) || (qhs & 7))
    return I4_ERR_ALIGN;
  if (need) {
    if (!workspace || have < need) return I4_ERR_WORKSPACE;
    if ((uintptr_t)workspace & 255) return I4_ERR_ALIGN;
  }
  return I4_OK;
}

static i4::CtxArgs ctx_args(const void* q, int B, int T, int64_t qbs, int64_t qts, int64_t qhs, int nq,
                            int nkv, const int32_t* pos_dev, int pos, const int32_t* counts,
                            int window, int sinks, float scale, void* out) {
  i4::CtxArgs a{};
  a.q = (const uint16_t*)q;
  a.qbs = qbs, a.qts = qts, a.qhs = qhs;
  a.out = (uint16_t*)out;
  a.tk = i4::Tokens{pos_dev, counts, pos, T};
  a.w = i4::Bounds{window ? window : INT32_MAX, sinks};
  a.B = B;
  a.nq = nq, a.nkv = nkv, a.G = nq / nkv, a.R = T * (nq / nkv);
  a.c2 = scale * 1.44269504f;
  return a;
}

int i4_attn_window(const void* q, int x_dtype, int T, int64_t q_batch_stride,
                   int64_t q_token_stride, int64_t q_head_stride, int n_heads,
                   const i4_kvcache* cache, const int32_t* pos_dev, int pos,
                   const int32_t* counts, int window, int sinks, float scale, void* out,
                   void* workspace, size_t workspace_bytes, int32_t* counters,
                   hipStream_t stream) {
  using namespace i4;
  int rc = i4_check_kvcache(cache);
  if (rc) return rc;
  const int B = cache->batch, nkv = cache->n_kv_heads;
  const int keys = call_keys(pos_dev, pos, T, cache->max_len);
  rc = query_check(q, x_dtype, cache->dtype, B, T, q_batch_stride, q_token_stride, q_head_stride,
                   n_heads, nkv, pos_dev, pos, counts, cache->max_len, window, sinks, scale, out,
                   workspace, workspace_bytes,
                   i4_attn_window_workspace_bytes(B, T, n_heads, nkv, keys, window, sinks),
                   counters);
  if (rc) return rc;
  CtxArgs a = ctx_args(q, B, T, q_batch_stride, q_token_stride, q_head_stride, n_heads, nkv, pos_dev,
                       pos, counts, window, sinks, scale, out);
  a.c = Cache16{(uint16_t*)cache->k, (uint16_t*)cache->v, cache->batch_stride,
                cache->head_stride, cache->row_stride, cache->max_len};
  a.len = cache->max_len;
  return launch(a, x_dtype, kDense, keys, i4_span{window, sinks, workspace, counters}, stream);
}

int i4_attn_kv8(const void* q, int x_dtype, int T, int64_t q_batch_stride, int64_t q_token_stride,
                int64_t q_head_stride, int n_heads, const i4_kv8cache* cache,
                const int32_t* pos_dev, int pos, const int32_t* counts, int window, int sinks,
                float scale, void* out, void* workspace, size_t workspace_bytes,
                int32_t* counters, hipStream_t stream) {
  using namespace i4;
  int rc = i4_check_kv8cache(cache);
  if (rc) return rc;
  const int B = cache->batch, nkv = cache->n_kv_heads, len = cache->blocks * KBLK;
  const int keys = call_keys(pos_dev, pos, T, len);
  rc = query_check(q, x_dtype, cache->dtype, B, T, q_batch_stride, q_token_stride, q_head_stride,
                   n_heads, nkv, pos_dev, pos, counts, len, window, sinks, scale, out, workspace,
                   workspace_bytes,
                   i4_attn_window_workspace_bytes(B, T, n_heads, nkv, keys, window, sinks),
                   counters);
  if (rc) return rc;
  CtxArgs a = ctx_args(q, B, T, q_batch_stride, q_token_stride, q_head_stride, n_heads, nkv, pos_dev,
                       pos, counts, window, sinks, scale, out);
  a.c8 = Cache8{(uint8_t*)cache->k, (uint8_t*)cache->v, cache->k_scale, cache->v_scale,
                (uint16_t*)cache->k_tail, (uint16_t*)cache->v_tail, cache->blocks};
  a.len = len;
  return launch(a, x_dtype, cache->format, keys, i4_span{window, sinks, workspace, counters},
                stream);
}

int i4_attn_paged(const void* q, int x_dtype, int T, int64_t q_batch_stride,
                  int64_t q_token_stride, int64_t q_head_stride, int n_heads,
                  const i4_pagedcache* cache, const int32_t* pos_dev, int pos,
                  const int32_t* counts, int zero_padding, int window, int sinks, float scale,
                  void* out, void* workspace, size_t workspace_bytes, int32_t* counters,
                  hipStream_t stream) {
  using namespace i4;
  int rc = i4_check_pagedcache(cache);
  if (rc) return rc;
  const int B = cache->batch, nkv = cache->n_kv_heads, len = cache->table_len * cache->page;
  const int keys = call_keys(pos_dev, pos, T, len);
  rc = query_check(q, x_dtype, cache->dtype, B, T, q_batch_stride, q_token_stride, q_head_stride,
                   n_heads, nkv, pos_dev, pos, counts, len, window, sinks, scale, out, workspace,
                   workspace_bytes,
                   i4_attn_paged_call_bytes(B, T, n_heads, nkv, keys, window, sinks,
                                            pos_dev || counts),
                   counters);
  if (rc) return rc;
  CtxArgs a = ctx_args(q, B, T, q_batch_stride, q_token_stride, q_head_stride, n_heads, nkv, pos_dev,
                       pos, counts, window, sinks, scale, out);
  a.pg = i4_pages_of(cache);
  a.zero = zero_padding;
  a.len = len;
  return launch(a, x_dtype, kPaged, keys, i4_span{window, sinks, workspace, counters}, stream);
}

}  // extern "C"
