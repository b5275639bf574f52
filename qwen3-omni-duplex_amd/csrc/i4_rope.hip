// q/k RMSNorm, rotary embedding and the append to a 16-bit cache, for many tokens: what
// lies between the q|k|v projection and the attention
// (Qwen3OmniMoeThinkerTextAttention.forward, modeling_qwen3_omni_moe.py:1473-1500 in
// transformers 5.15).
//   n_d   = x_d w_d / sqrt(mean(x^2) + eps)
//   out_d = n_d cos(a) - n_{d+64} sin(a),  out_{d+64} = n_{d+64} cos(a) + n_d sin(a),
//   a     = p inv_freq_d,  d < 64,
// all in fp32 and rounded once.  One wave takes one head of one token; lane l holds dims
// 2l and 2l + 1, so dim d +- 64 is lane l ^ 32's.
#include "i4_kv.h"

namespace i4 {

struct RopeFreq {
  float f[KHD / 2];
};

// cos and sin of p f as the sum of two floats: the product's rounding error (up to 2^-25 of
// an angle that grows with the position) is carried to first order.
__device__ inline void angle(float p, float f, float& c, float& s) {
  const float hi = p * f, lo = fmaf(p, f, -hi);
  float s0, c0;
  sincosf(hi, &s0, &c0);
  c = fmaf(-lo, s0, c0);
  s = fmaf(lo, c0, s0);
}

template <int XT>
__global__ __launch_bounds__(256) void k_rope_append(
    const uint16_t* __restrict__ qkv, int64_t bs, int64_t ts, int nq, int nkv,
    const uint16_t* __restrict__ qw, const uint16_t* __restrict__ kw, float eps, RopeFreq rf,
    Tokens tk, int first_row, uint16_t* __restrict__ q_out, Cache16 cache, int limit,
    int64_t n_rows) {
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);  // (b, t, head)
  if (row >= n_rows) return;
  const int lane = threadIdx.x & 63, heads = nq + 2 * nkv;
  const int h = (int)(row % heads);
  const int64_t bt = row / heads;
  const int b = (int)(bt / tk.T), t = (int)(bt % tk.T);
  if (t >= count_of(tk, b)) return;
  const int p0 = first_pos(tk, b);
  // p0 is checked before t is added: a device position may be anything
  const bool ok = p0 >= 0 && p0 < limit && t < limit - p0;
  u32* q_row = (u32*)(q_out + (bt * nq + h) * KHD) + lane;
  if (!ok) {
    if (h < nq) *q_row = (u32)Half<XT>::QNAN * 0x10001u;
    return;
  }
  const int p = p0 + t;
  const u32 raw = *((const u32*)(qkv + b * bs + t * ts + (int64_t)h * KHD) + lane);
  u32 out = raw;
  if (h < nq + nkv) {
    const u32 w = *((const u32*)(h < nq ? qw : kw) + lane);
    const float x0 = Half<XT>::to_f32((uint16_t)raw), x1 = Half<XT>::to_f32((uint16_t)(raw >> 16));
    const float r = 1.0f / sqrtf(group_sum<64>(x0 * x0 + x1 * x1) * (1.0f / KHD) + eps);
    const float n0 = x0 * r * Half<XT>::to_f32((uint16_t)w);
    const float n1 = x1 * r * Half<XT>::to_f32((uint16_t)(w >> 16));
    const float m0 = __shfl_xor(n0, 32), m1 = __shfl_xor(n1, 32);
    const int i = 2 * (lane & 31);
    float c0, s0, c1, s1;
    angle((float)p, rf.f[i], c0, s0);
    angle((float)p, rf.f[i + 1], c1, s1);
    const float sg = lane < 32 ? -1.f : 1.f;
    out = (u32)Half<XT>::from_f32(fmaf(n0, c0, sg * m0 * s0)) |
          ((u32)Half<XT>::from_f32(fmaf(n1, c1, sg * m1 * s1)) << 16);
  }
  if (h < nq) {
    *q_row = out;
    return;
  }
  const int g = (h - nq) % nkv;
  const int slot = first_row < 0 ? p : first_row + t;
  uint16_t* c = h < nq + nkv ? cache.k : cache.v;
  *((u32*)(c + b * cache.bs + g * cache.hs + (int64_t)slot * cache.rs) + lane) = out;
}

}  // namespace i4

extern "C" int i4_rope_append(const void* qkv, int x_dtype, int T, int64_t batch_stride,
                              int64_t token_stride, int n_heads, const void* q_norm_w,
                              const void* k_norm_w, float eps, const float* inv_freq,
                              const int32_t* pos_dev, int pos, int first_row,
                              const int32_t* counts, void* q_out, const i4_kvcache* cache,
                              hipStream_t stream) {
  using namespace i4;
  if (!qkv || !q_norm_w || !k_norm_w || !inv_freq || !q_out) return I4_ERR_NULL;
  int rc = i4_check_kvcache(cache);
  if (rc) return rc;
  if (x_dtype != cache->dtype) return I4_ERR_DTYPE;
  const int nkv = cache->n_kv_heads, B = cache->batch;
  const int limit = first_row < 0 ? cache->max_len : ROPE_MAX_POS;
  rc = i4_check_tokens(B, T, n_heads, nkv, pos_dev, pos, counts, limit);
  if (rc) return rc;
  if (first_row >= 0 && first_row > cache->max_len - T) return I4_ERR_SHAPE;
  const int64_t width = (int64_t)(n_heads + 2 * nkv) * KHD;
  if ((T > 1 && token_stride < width) || (B > 1 && batch_stride < width)) return I4_ERR_STRIDE;
  if (((uintptr_t)qkv & 3) || ((uintptr_t)q_norm_w & 3) || ((uintptr_t)k_norm_w & 3) ||
      ((uintptr_t)q_out & 15) || (token_stride & 1) || (batch_stride & 1))
    return I4_ERR_ALIGN;
  RopeFreq rf;
  for (int i = 0; i < KHD / 2; ++i) rf.f[i] = inv_freq[i];
  const Tokens tk{pos_dev, counts, pos, T};
  const Cache16 c{(uint16_t*)cache->k, (uint16_t*)cache->v, cache->batch_stride,
                  cache->head_stride, cache->row_stride, cache->max_len};
  const int64_t rows = (int64_t)B * T * (n_heads + 2 * nkv);
  const dim3 grid((unsigned)((rows + 3) / 4));
  if (x_dtype == I4_F16)
    k_rope_append<I4_F16><<<grid, 256, 0, stream>>>(
        (const uint16_t*)qkv, batch_stride, token_stride, n_heads, nkv, (const uint16_t*)q_norm_w,
        (const uint16_t*)k_norm_w, eps, rf, tk, first_row, (uint16_t*)q_out, c, limit, rows);
  else
    k_rope_append<I4_BF16><<<grid, 256, 0, stream>>>(
        (const uint16_t*)qkv, batch_stride, token_stride, n_heads, nkv, (const uint16_t*)q_norm_w,
        (const uint16_t*)k_norm_w, eps, rf, tk, first_row, (uint16_t*)q_out, c, limit, rows);
  return hipGetLastError() == hipSuccess ? I4_OK : I4_ERR_LAUNCH;
}
