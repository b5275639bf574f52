// Attention over a conversation's cached context: B x T queries over a 16-bit cache
// (i4_attn_window) or an 8-bit one (i4_attn_kv8), under an optional sliding window whose
// first tokens stay visible.
//   out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),  s_j = scale q . k_j,
// over the visible j in one pass, with a running maximum m and sum.
#include "i4_ctx.h"

// the bounds and the workspace of a call
struct i4_span {
  int window, sinks;
  void* workspace;
};

namespace i4 {

// One wave per query row: lane l holds dims 2l and 2l + 1.
template <int XT, int FMT>
__global__ __launch_bounds__(256) void k_ctx_row(const uint16_t* __restrict__ q, int64_t qbs,
                                                 int64_t qts, int64_t qhs, int nq, int nkv,
                                                 Cache16 c, Cache8 c8, Tokens tk, Bounds w,
                                                 float scale, uint16_t* __restrict__ out,
                                                 int64_t n_rows) {
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);  // (b, t, head)
  if (row >= n_rows) return;
  const int lane = threadIdx.x & 63;
  const int h = (int)(row % nq);
  const int64_t bt = row / nq;
  const int b = (int)(bt / tk.T), t = (int)(bt % tk.T), g = h / (nq / nkv);
  const int n = count_of(tk, b);
  if (t >= n) return;
  u32* dst = (u32*)(out + row * KHD) + lane;
  const int p0 = first_pos(tk, b);
  const int len = FMT < 0 ? c.max_len : c8.blocks * KBLK;
  if (p0 < 0 || p0 >= len || t >= len - p0) {
    *dst = (u32)Half<XT>::QNAN * 0x10001u;
    return;
  }
  const int p = p0 + t, end = p0 + min(n, len - p0), tail0 = end / KBLK * KBLK;
  const u32 qr = *((const u32*)(q + b * qbs + t * qts + h * qhs) + lane);
  const float q0 = Half<XT>::to_f32((uint16_t)qr) * scale;
  const float q1 = Half<XT>::to_f32((uint16_t)(qr >> 16)) * scale;
  const int64_t hb = (int64_t)b * nkv + g;
  float m = -__builtin_inff(), l = 0.f, a0 = 0.f, a1 = 0.f;
  const int lo = max(0, p - w.window + 1), s = min(w.sinks, lo);
  for (int i = 0; i < s + (p + 1 - lo); ++i) {
    const int j = i < s ? i : lo + i - s;
    float k0, k1, v0, v1;
    if (FMT < 0 || j >= tail0) {
      const int64_t o = FMT < 0 ? b * c.bs + g * c.hs + (int64_t)j * c.rs
                                : (hb * KBLK + j - tail0) * KHD;
      const u32 kr = *((const u32*)((FMT < 0 ? c.k : c8.kt) + o) + lane);
      const u32 vr = *((const u32*)((FMT < 0 ? c.v : c8.vt) + o) + lane);
      k0 = Half<XT>::to_f32((uint16_t)kr), k1 = Half<XT>::to_f32((uint16_t)(kr >> 16));
      v0 = Half<XT>::to_f32((uint16_t)vr), v1 = Half<XT>::to_f32((uint16_t)(vr >> 16));
    } else {
      constexpr int F = FMT < 0 ? 0 : FMT;
      const int64_t blk = hb * c8.blocks + j / KBLK;
      const uint8_t *kb = c8.k + blk * KBLK * KHD, *vb = c8.v + blk * KBLK * KHD;
      const float ks = c8.ks[blk], vs = c8.vs[blk];
      const int r = j % KBLK;
      k0 = from_8bit<F>(kb[r * KHD + 2 * lane]) * ks;
      k1 = from_8bit<F>(kb[r * KHD + 2 * lane + 1]) * ks;
      v0 = from_8bit<F>(vb[2 * lane * KBLK + r]) * vs;
      v1 = from_8bit<F>(vb[(2 * lane + 1) * KBLK + r]) * vs;
    }
    const float x = group_sum<64>(q0 * k0 + q1 * k1);
    const float mn = fmaxf(m, x);
    const float f = expf(m - mn), e = expf(x - mn);
    l = l * f + e;
    a0 = a0 * f + e * v0;
    a1 = a1 * f + e * v1;
    m = mn;
  }
  const float inv = 1.0f / l;
  *dst = (u32)Half<XT>::from_f32(a0 * inv) | ((u32)Half<XT>::from_f32(a1 * inv) << 16);
}

// How a call is split: a rule on its sizes alone (no device value), so that the workspace
// can be named before the call.
static int ctx_splits(int B, int T, int nq, int nkv, int keys, int window, int sinks) {
  const int R = T * (nq / nkv);
  if (R > 32) return 1;
  int64_t tiles = (keys + 63) / 64;
  if (window) {
    const int64_t most = ((int64_t)window + T + 126) / 64 + (sinks + 63) / 64;
    if (most < tiles) tiles = most;
  }
  const int64_t want = (1024 + (int64_t)B * nkv - 1) / ((int64_t)B * nkv);
  const int64_t most = (tiles + 3) / 4;  // a tile a wave
  const int64_t s = want < most ? want : most;
  return s < 1 ? 1 : (int)s;
}

static int launch(CtxArgs& a, int B, int xt, int fmt, int keys, const i4_span& w,
                  hipStream_t stream) {
  a.S = ctx_splits(B, a.tk.T, a.nq, a.nkv, keys, w.window, w.sinks);
  if (a.S > 1) {
    a.part = (float*)w.workspace;
    a.ml = a.part + (int64_t)B * a.nkv * a.R * a.S * KHD;
  }
  if (a.R <= 32) return i4_launch_ctx_rows(a, B, xt, fmt, stream);
  const int64_t rows = (int64_t)B * a.tk.T * a.nq;
  const dim3 grid((unsigned)((rows + 3) / 4));
  const float scale = a.c2 * 0.69314718f;
  auto go = [&](auto kern) {
    kern<<<grid, 256, 0, stream>>>(a.q, a.qbs, a.qts, a.qhs, a.nq, a.nkv, a.c, a.c8, a.tk, a.w,
                                   scale, a.out, rows);
  };
  if (xt == I4_F16) {
    if (fmt < 0) go(k_ctx_row<I4_F16, -1>);
    else if (fmt == I4_KV8_INT8) go(k_ctx_row<I4_F16, I4_KV8_INT8>);
    else go(k_ctx_row<I4_F16, I4_KV8_E4M3>);
  } else {
    if (fmt < 0) go(k_ctx_row<I4_BF16, -1>);
    else if (fmt == I4_KV8_INT8) go(k_ctx_row<I4_BF16, I4_KV8_INT8>);
    else go(k_ctx_row<I4_BF16, I4_KV8_E4M3>);
  }
  return hipGetLastError() == hipSuccess ? I4_OK : I4_ERR_LAUNCH;
}

}  // namespace i4

extern "C" {

size_t i4_attn_window_workspace_bytes(int B, int T, int n_heads, int n_kv_heads, int keys,
                                      int window, int sinks) {
  if (B < 1 || T < 1 || T > i4::KV_MAX_LEN || n_kv_heads < 1 || n_heads < n_kv_heads ||
      n_heads > 1024 || n_heads % n_kv_heads || keys < 1 || window < 0 || sinks < 0)
    return 0;
  const int64_t S = i4::ctx_splits(B, T, n_heads, n_kv_heads, keys, window, sinks);
  return S > 1 ? (size_t)((int64_t)B * T * n_heads * S * (i4::KHD + 2) * 4) : 0;
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
                       size_t need) {
  if (!q || !out) return I4_ERR_NULL;
  if (x_dtype != dtype) return I4_ERR_DTYPE;
  const int rc = i4_check_tokens(B, T, n_heads, nkv, pos_dev, pos, counts, limit);
  if (rc) return rc;
  if (window < 0 || sinks < 0 || (window == 0 && sinks) || !(scale > 0.f) ||
      !(scale < __builtin_inff()))
    return I4_ERR_SHAPE;
  if ((T > 1 && qts < i4::KHD) || (B > 1 && qbs < i4::KHD) || (n_heads > 1 && qhs < i4::KHD))
    return I4_ERR_STRIDE;
  if (((uintptr_t)q & 15) || ((uintptr_t)out & 15) || (qbs & 7) || (qts & 7) || (qhs & 7))
    return I4_ERR_ALIGN;
  if (need) {
    if (!workspace || have < need) return I4_ERR_WORKSPACE;
    if ((uintptr_t)workspace & 255) return I4_ERR_ALIGN;
  }
  return I4_OK;
}

static i4::CtxArgs ctx_args(const void* q, int T, int64_t qbs, int64_t qts, int64_t qhs, int nq,
                            int nkv, const int32_t* pos_dev, int pos, const int32_t* counts,
                            int window, int sinks, float scale, void* out) {
  i4::CtxArgs a{};
  a.q = (const uint16_t*)q;
  a.qbs = qbs, a.qts = qts, a.qhs = qhs;
  a.out = (uint16_t*)out;
  a.tk = i4::Tokens{pos_dev, counts, pos, T};
  a.w = i4::Bounds{window ? window : INT32_MAX, sinks};
  a.nq = nq, a.nkv = nkv, a.G = nq / nkv, a.R = T * (nq / nkv);
  a.c2 = scale * 1.44269504f;
  return a;
}

int i4_attn_window(const void* q, int x_dtype, int T, int64_t q_batch_stride,
                   int64_t q_token_stride, int64_t q_head_stride, int n_heads,
                   const i4_kvcache* cache, const int32_t* pos_dev, int pos,
                   const int32_t* counts, int window, int sinks, float scale, void* out,
                   void* workspace, size_t workspace_bytes, hipStream_t stream) {
  using namespace i4;
  int rc = i4_check_kvcache(cache);
  if (rc) return rc;
  const int B = cache->batch, nkv = cache->n_kv_heads;
  const int keys = call_keys(pos_dev, pos, T, cache->max_len);
  rc = query_check(q, x_dtype, cache->dtype, B, T, q_batch_stride, q_token_stride, q_head_stride,
                   n_heads, nkv, pos_dev, pos, counts, cache->max_len, window, sinks, scale, out,
                   workspace, workspace_bytes,
                   i4_attn_window_workspace_bytes(B, T, n_heads, nkv, keys, window, sinks));
  if (rc) return rc;
  CtxArgs a = ctx_args(q, T, q_batch_stride, q_token_stride, q_head_stride, n_heads, nkv, pos_dev,
                       pos, counts, window, sinks, scale, out);
  a.c = Cache16{(uint16_t*)cache->k, (uint16_t*)cache->v, cache->batch_stride,
                cache->head_stride, cache->row_stride, cache->max_len};
  a.len = cache->max_len;
  return launch(a, B, x_dtype, -1, keys, i4_span{window, sinks, workspace}, stream);
}

int i4_attn_kv8(const void* q, int x_dtype, int T, int64_t q_batch_stride, int64_t q_token_stride,
                int64_t q_head_stride, int n_heads, const i4_kv8cache* cache,
                const int32_t* pos_dev, int pos, const int32_t* counts, int window, int sinks,
                float scale, void* out, void* workspace, size_t workspace_bytes,
                hipStream_t stream) {
  using namespace i4;
  int rc = i4_check_kv8cache(cache);
  if (rc) return rc;
  const int B = cache->batch, nkv = cache->n_kv_heads, len = cache->blocks * KBLK;
  const int keys = call_keys(pos_dev, pos, T, len);
  rc = query_check(q, x_dtype, cache->dtype, B, T, q_batch_stride, q_token_stride, q_head_stride,
                   n_heads, nkv, pos_dev, pos, counts, len, window, sinks, scale, out, workspace,
                   workspace_bytes,
                   i4_attn_window_workspace_bytes(B, T, n_heads, nkv, keys, window, sinks));
  if (rc) return rc;
  CtxArgs a = ctx_args(q, T, q_batch_stride, q_token_stride, q_head_stride, n_heads, nkv, pos_dev,
                       pos, counts, window, sinks, scale, out);
  a.c8 = Cache8{(uint8_t*)cache->k, (uint8_t*)cache->v, cache->k_scale, cache->v_scale,
                (uint16_t*)cache->k_tail, (uint16_t*)cache->v_tail, cache->blocks};
  a.len = len;
  return launch(a, B, x_dtype, cache->format, keys, i4_span{window, sinks, workspace}, stream);
}

}  // extern "C"
