// q/k RMSNorm, rotary embedding and the append to a 16-bit cache, for many tokens: what
// lies between the q|k|v projection and the attention
// (Qwen3OmniMoeThinkerTextAttention.forward, modeling_qwen3_omni_moe.py:1473-1500 in
// transformers 5.15).
//   n_d   = x_d w_d / sqrt(mean(x^2) + eps)
//   out_d = n_d cos(a) - n_{d+64} sin(a),  out_{d+64} = n_{d+64} cos(a) + n_d sin(a),
//   a     = p inv_freq_d,  d < 64,
// all in fp32 and rounded once.  Bound by the rows' bytes.  A workgroup takes one token: its
// 64 angles are computed once, for all heads; a head is 16 lanes of 8 dims, so that dim
// d +- 64 is 8 lanes away (a rotation by half a DPP row).
#include "i4_kv.h"

namespace i4 {

struct RopeFreq {
  float f[KHD / 2];
};

// cos and sin of p f as the sum of two floats, hi + lo exactly: lo is up to 2^-24 of an angle
// that grows with the position (half a radian at position 2^24), so the rotation by hi is
// followed by a whole one by lo.
__device__ inline void angle(float p, float f, float& c, float& s) {
  const float hi = p * f, lo = fmaf(p, f, -hi);
  float s0, c0, s1, c1;
  sincosf(hi, &s0, &c0);
  sincosf(lo, &s1, &c1);
  c = fmaf(c0, c1, -s0 * s1);
  s = fmaf(s0, c1, c0 * s1);
}

__device__ inline float half_row(float v) {  // the value 8 lanes away within 16
  return dpp_mov<0x128>(v);
}

template <int XT>
__global__ __launch_bounds__(256) void k_rope_append(
    const uint16_t* __restrict__ qkv, int64_t bs, int64_t ts, int nq, int nkv,
    const uint16_t* __restrict__ qw, const uint16_t* __restrict__ kw, float eps, RopeFreq rf,
    Tokens tk, int first_row, uint16_t* __restrict__ q_out, Cache16 cache, int limit) {
  __shared__ __align__(16) float s_c[KHD / 2], s_s[KHD / 2];
  const int b = blockIdx.x / tk.T, t = blockIdx.x % tk.T;
  if (t >= count_of(tk, b)) return;
  const int heads = nq + 2 * nkv, lane = threadIdx.x & 15;
  const int p0 = first_pos(tk, b);
  // p0 is checked before t is added: a device position may be anything
  const bool ok = p0 >= 0 && p0 < limit && t < limit - p0;
  u32x4* q_row = (u32x4*)(q_out + (int64_t)blockIdx.x * nq * KHD) + lane;
  int h = threadIdx.x >> 4;
  if (!ok) {
    for (; h < nq; h += 16) q_row[h * (KHD / 8)] = u32x4{} + (u32)Half<XT>::QNAN * 0x10001u;
    return;
  }
  const int p = p0 + t;
  const u32x4* x_row = (const u32x4*)(qkv + b * bs + t * ts) + lane;
  u32x4 raw = h < heads ? x_row[h * (KHD / 8)] : u32x4{};
  const u32x4 qn = ((const u32x4*)qw)[lane], kn = ((const u32x4*)kw)[lane];
  if (threadIdx.x < KHD / 2) {
    float c, s;
    angle((float)p, rf.f[threadIdx.x], c, s);
    s_c[threadIdx.x] = c;
    s_s[threadIdx.x] = s;
  }
  __syncthreads();
  const int i0 = 8 * (lane & 7);
  float cs[8], sn[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    cs[i] = s_c[i0 + i];
    sn[i] = lane < 8 ? -s_s[i0 + i] : s_s[i0 + i];
  }
  const int64_t slot = (int64_t)(first_row < 0 ? p : first_row + t) * cache.rs + b * cache.bs;
  for (; h < heads; h += 16) {
    const u32x4 next = h + 16 < heads ? x_row[(h + 16) * (KHD / 8)] : u32x4{};
    u32x4 out = raw;
    if (h < nq + nkv) {
      const u32x4 w = h < nq ? qn : kn;
      float x[8], ss = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[2 * i] = Half<XT>::to_f32((uint16_t)raw[i]);
        x[2 * i + 1] = Half<XT>::to_f32((uint16_t)(raw[i] >> 16));
        ss += x[2 * i] * x[2 * i] + x[2 * i + 1] * x[2 * i + 1];
      }
      const float r = 1.0f / sqrtf(group_sum<16>(ss) * (1.0f / KHD) + eps);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[2 * i] *= r * Half<XT>::to_f32((uint16_t)w[i]);
        x[2 * i + 1] *= r * Half<XT>::to_f32((uint16_t)(w[i] >> 16));
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = fmaf(x[i], cs[i], half_row(x[i]) * sn[i]);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        out[i] = (u32)Half<XT>::from_f32(x[2 * i]) | ((u32)Half<XT>::from_f32(x[2 * i + 1]) << 16);
    }
    if (h < nq) {
      q_row[h * (KHD / 8)] = out;
    } else {
      const bool key = h < nq + nkv;
      uint16_t* c = key ? cache.k : cache.v;
      *((u32x4*)(c + slot + (h - nq - (key ? 0 : nkv)) * cache.hs) + lane) = out;
    }
    raw = next;
  }
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
  if ((int64_t)B * T > kMaxGrid) return I4_ERR_SHAPE;
  const int64_t width = (int64_t)(n_heads + 2 * nkv) * KHD;
  if ((T > 1 && token_stride < width) || (B > 1 && batch_stride < width)) return I4_ERR_STRIDE;
  if (((uintptr_t)qkv & 15) || ((uintptr_t)q_norm_w & 15) || ((uintptr_t)k_norm_w & 15) ||
      ((uintptr_t)q_out & 15) || (token_stride & 7) || (batch_stride & 7))
    return I4_ERR_ALIGN;
  RopeFreq rf;
  for (int i = 0; i < KHD / 2; ++i) rf.f[i] = inv_freq[i];
  const Tokens tk{pos_dev, counts, pos, T};
  const Cache16 c{(uint16_t*)cache->k, (uint16_t*)cache->v, cache->batch_stride,
                  cache->head_stride, cache->row_stride, cache->max_len};
  const dim3 grid((unsigned)(B * T));
  if (x_dtype == I4_F16)
    k_rope_append<I4_F16><<<grid, 256, 0, stream>>>(
        (const uint16_t*)qkv, batch_stride, token_stride, n_heads, nkv, (const uint16_t*)q_norm_w,
        (const uint16_t*)k_norm_w, eps, rf, tk, first_row, (uint16_t*)q_out, c, limit);
  else
    k_rope_append<I4_BF16><<<grid, 256, 0, stream>>>(
        (const uint16_t*)qkv, batch_stride, token_stride, n_heads, nkv, (const uint16_t*)q_norm_w,
        (const uint16_t*)k_norm_w, eps, rf, tk, first_row, (uint16_t*)q_out, c, limit);
  return hipGetLastError() == hipSuccess ? I4_OK : I4_ERR_LAUNCH;
}
