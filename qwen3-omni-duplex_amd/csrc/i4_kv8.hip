// The 8-bit KV cache: tokens into blocks of 64 with one scale for each block and head.
//   scale = max(max |x|, 2^-100) / (127 or 448),  element = RNE(x / scale)
// The scale is the correctly rounded fp32 quotient, and an element is the exact quotient
// x / scale rounded once.  A block is rounded when its last token arrives, from the 16-bit
// values of its tokens, so what the cache holds does not depend on how the tokens came
// (one by one, in chunks): the tokens of the unfinished block wait in the tail.
#include "i4_kv.h"

namespace i4 {

// x / s as fp32 rounded to odd: a quotient that fp32 does not hold gets an odd last bit, so
// rounding it to the element's few bits afterwards rounds as the exact quotient would (a
// nearest fp32 quotient could land on a tie that the exact one misses).  inv = 1 / s rounded;
// one Newton step makes the product the quotient to within its last bit, and then the
// remainder of the next fma is exact and says on which side of it the quotient lies.
__device__ inline float quotient_to_odd(float x, float s, float inv) {
  float t = x * inv;
  t = fmaf(fmaf(-t, s, x), inv, t);
  const float r = fmaf(-t, s, x);
  const u32 b = __builtin_bit_cast(u32, t);
  // an even last bit and a remainder: the odd neighbour on the remainder's side (by the sign
  // bit, as t may have underflowed to a zero of x's sign: away from it then)
  const u32 odd = (r > 0.f) == ((b >> 31) == 0) ? b + 1 : b - 1;
  return __builtin_bit_cast(float, r == 0.f || (b & 1) ? b : odd);
}
// four elements in a word
template <int FMT> __device__ inline u32 pack_8bit(float a, float b, float c, float d) {
  if constexpr (FMT == I4_KV8_INT8) {
    const u32 lo = ((u32)(int)rintf(a) & 0xFFu) | (((u32)(int)rintf(b) & 0xFFu) << 8);
    return lo | (((u32)(int)rintf(c) & 0xFFu) << 16) | ((u32)(int)rintf(d) << 24);
  } else {
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (u32)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, lo, true);
  }
}
template <int XT> __device__ inline void widen8(u32x4 x, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = Half<XT>::to_f32((uint16_t)x[i]);
    f[2 * i + 1] = Half<XT>::to_f32((uint16_t)(x[i] >> 16));
  }
}

// Workgroup (touched block i of the sequence, kv head, sequence; keys or values).  The
// block's tokens come from the tail (those before pos, first block only) and the call.
// A finished block is scaled and written; an unfinished one's new tokens go to the tail.
// The first block reads the tail that the last one overwrites, so the first block's
// workgroup does the last, unfinished block too, behind its own.
// Thread t holds dims 8 (t % 16) .. + 7 of tokens 4 (t / 16) .. + 3: whole rows in a wave's
// loads; a key row's 8 bytes are stored as they are, four tokens of a value dim make a word,
// which LDS brings into rows.  4001 tokens of four heads take 8 us, for 2.6 of bytes and some 1
// of quotients (10 instructions an element): two workgroups a CU, each a chain of its own of
// loads, maximum, barrier, quotients, LDS and stores, do not hide each other's waits.
template <int XT, int FMT>
__global__ __launch_bounds__(256) void k_kv8_append(const uint16_t* __restrict__ k,
                                                    const uint16_t* __restrict__ v, int64_t bs,
                                                    int64_t ts, int64_t hs, int nkv, Tokens tk,
                                                    Cache8 c) {
  __shared__ float s_max[4];
  __shared__ __align__(16) u32 s_t[KHD][KBLK / 4 + 1];  // a dim's tokens, padded
  const bool val = blockIdx.y & 1;
  const int g = (blockIdx.y >> 1) % nkv, b = (blockIdx.y >> 1) / nkv;
  const int p0 = first_pos(tk, b), len = c.blocks * KBLK;
  if (p0 < 0 || p0 >= len) return;
  const int n = min(count_of(tk, b), len - p0);
  const int first = p0 / KBLK, r = p0 % KBLK, done = (r + n) / KBLK;  // finished blocks
  const int64_t hb = (int64_t)b * nkv + g;
  const uint16_t* src = (val ? v : k) + b * bs + g * hs;
  uint16_t* tail = (val ? c.vt : c.kt) + hb * KBLK * KHD;
  const int i = blockIdx.x, tid = threadIdx.x;
  const int d0 = 8 * (tid & 15), tok = 4 * (tid >> 4);
  if (i < done) {
    u32x4 x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int at = i * KBLK + tok + j - r;  // the call's token, or one of the tail's
      x[j] = ldg16((at >= 0 ? src + at * ts : tail + (int64_t)(tok + j) * KHD) + d0);
    }
    float f[4][8], m = KV8_TINY;
    bool bad = false;  // an infinity or a NaN
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      widen8<XT>(x[j], f[j]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        bad |= !(fabsf(f[j][e]) < __builtin_inff());
        m = fmaxf(m, fabsf(f[j][e]));
      }
    }
    if (bad) m = __builtin_inff();
    for (int o = 1; o < 64; o <<= 1) m = fmaxf(m, __shfl_xor(m, o));
    if ((tid & 63) == 0) s_max[tid >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
    const bool finite = m < __builtin_inff();
    const float scale = finite ? m / (FMT == I4_KV8_INT8 ? 127.f : 448.f) : __builtin_nanf("");
    const float inv = 1.0f / scale;
    const int64_t blk = hb * c.blocks + first + i;
    uint8_t* dst = (val ? c.v : c.k) + blk * KBLK * KHD;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) f[j][e] = finite ? quotient_to_odd(f[j][e], scale, inv) : 0.f;
    if (val) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        s_t[d0 + e][tid >> 4] = pack_8bit<FMT>(f[0][e], f[1][e], f[2][e], f[3][e]);
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 8; ++j) {  // 16 words a dim
        const int w = 256 * j + tid;
        ((u32*)dst)[w] = s_t[w >> 4][w & 15];
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *(u32x2*)(dst + (tok + j) * KHD + d0) =
            u32x2{pack_8bit<FMT>(f[j][0], f[j][1], f[j][2], f[j][3]),
                  pack_8bit<FMT>(f[j][4], f[j][5], f[j][6], f[j][7])};
    }
    if (tid == 0) (val ? c.vs : c.ks)[blk] = scale;
    __syncthreads();  // the tail has been read
  }
  if (i == 0) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int at = done * KBLK + tok + j - r;
      if (at >= 0 && at < n)
        *(u32x4*)(tail + (int64_t)(tok + j) * KHD + d0) = ldg16(src + at * ts + d0);
    }
  }
}

// The blocks' values in fp32, 16 bytes a lane; value blocks turn through LDS, four dims of
// four tokens at a time.
template <int FMT>
__global__ __launch_bounds__(256) void k_kv8_values(Cache8 c, float* __restrict__ ko,
                                                    float* __restrict__ vo) {
  __shared__ u32 s_t[KHD][KBLK / 4 + 1];
  const int64_t blk = blockIdx.x;
  const int tid = threadIdx.x;
  auto four = [](u32 w, float s) {
    return f32x4{from_8bit<FMT>((uint8_t)w) * s, from_8bit<FMT>((uint8_t)(w >> 8)) * s,
                 from_8bit<FMT>((uint8_t)(w >> 16)) * s, from_8bit<FMT>((uint8_t)(w >> 24)) * s};
  };
  if (blockIdx.y == 0) {
    const u32* src = (const u32*)(c.k + blk * KBLK * KHD);
    const float s = block_scale(c.ks[blk]);
    f32x4* dst = (f32x4*)(ko + blk * KBLK * KHD);
#pragma unroll
    for (int j = 0; j < 8; ++j) dst[256 * j + tid] = four(src[256 * j + tid], s);
    return;
  }
  const u32* src = (const u32*)(c.v + blk * KBLK * KHD);
  const float s = block_scale(c.vs[blk]);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int w = 256 * j + tid;
    s_t[w >> 4][w & 15] = src[w];
  }
  __syncthreads();
  const int d = 4 * (tid & 31);
  f32x4* dst = (f32x4*)(vo + blk * KBLK * KHD) + (tid & 31);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int q = (tid >> 5) + 8 * j;  // tokens 4 q .. + 3
    const u32 w[4] = {s_t[d][q], s_t[d + 1][q], s_t[d + 2][q], s_t[d + 3][q]};
    // bytes (dim, token) -> (token, dim)
    const u32 a = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u);
    const u32 b = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u);
    const u32 e = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u);
    const u32 f = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
    const u32 y[4] = {__builtin_amdgcn_perm(b, a, 0x05040100u),
                      __builtin_amdgcn_perm(b, a, 0x07060302u),
                      __builtin_amdgcn_perm(f, e, 0x05040100u),
                      __builtin_amdgcn_perm(f, e, 0x07060302u)};
#pragma unroll
    for (int i = 0; i < 4; ++i) dst[(4 * q + i) * (KHD / 4)] = four(y[i], s);
  }
}

}  // namespace i4

int i4_check_tokens(int B, int T, int n_heads, int n_kv_heads, const int32_t* pos_dev, int pos,
                    const int32_t* counts, int limit) {
  if (T < 1 || T > i4::KV_MAX_LEN || n_heads < n_kv_heads || n_heads > 1024 ||
      n_heads % n_kv_heads || (int64_t)B * T * (n_heads + 2 * n_kv_heads) >= INT32_MAX)
    return I4_ERR_SHAPE;
  if (((uintptr_t)pos_dev & 3) || ((uintptr_t)counts & 3)) return I4_ERR_ALIGN;
  if (!pos_dev && (pos < 0 || pos > limit - T)) return I4_ERR_SHAPE;
  return I4_OK;
}

int i4_check_kvcache(const i4_kvcache* c) {
  if (!c || !c->k || !c->v) return I4_ERR_NULL;
  if (c->dtype != I4_F16 && c->dtype != I4_BF16) return I4_ERR_DTYPE;
  if (c->head_dim != i4::KHD || c->batch < 1 || c->batch > 65535 || c->n_kv_heads < 1 ||
      c->n_kv_heads > 1024 || c->max_len < 1 || c->max_len > i4::KV_MAX_LEN)
    return I4_ERR_SHAPE;
  if ((c->max_len > 1 && c->row_stride < i4::KHD) ||
      (c->n_kv_heads > 1 && c->head_stride < i4::KHD) ||
      (c->batch > 1 && c->batch_stride < i4::KHD))
    return I4_ERR_STRIDE;
  // one head's rows are addressed with 32-bit byte offsets
  if (c->max_len > 1 && c->row_stride > (((int64_t)1 << 30) - i4::KHD) / (c->max_len - 1))
    return I4_ERR_STRIDE;
  if (((uintptr_t)c->k & 15) || ((uintptr_t)c->v & 15) || (c->row_stride & 7) ||
      (c->head_stride & 7) || (c->batch_stride & 7))
    return I4_ERR_ALIGN;
  return I4_OK;
}

int i4_check_kv8cache(const i4_kv8cache* c) {
  if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale || !c->k_tail || !c->v_tail)
    return I4_ERR_NULL;
  if ((c->dtype != I4_F16 && c->dtype != I4_BF16) ||
      (c->format != I4_KV8_INT8 && c->format != I4_KV8_E4M3))
    return I4_ERR_DTYPE;
  if (c->head_dim != i4::KHD || c->batch < 1 || c->batch > 65535 || c->n_kv_heads < 1 ||
      c->n_kv_heads > 1024 || c->blocks < 1 || c->blocks > i4::KV_MAX_LEN / i4::KBLK ||
      (int64_t)c->batch * c->n_kv_heads * c->blocks >= INT32_MAX)
    return I4_ERR_SHAPE;
  for (const void* p : {(const void*)c->k, (const void*)c->v, (const void*)c->k_scale,
                        (const void*)c->v_scale, (const void*)c->k_tail, (const void*)c->v_tail})
    if ((uintptr_t)p & 15) return I4_ERR_ALIGN;
  return I4_OK;
}

static i4::Cache8 cache8(const i4_kv8cache* c) {
  return i4::Cache8{(uint8_t*)c->k, (uint8_t*)c->v, c->k_scale, c->v_scale,
                    (uint16_t*)c->k_tail, (uint16_t*)c->v_tail, c->blocks};
}

extern "C" int i4_kv8_append(const void* k, const void* v, int x_dtype, int T,
                             int64_t batch_stride, int64_t token_stride, int64_t head_stride,
                             const i4_kv8cache* cache, const int32_t* pos_dev, int pos,
                             const int32_t* counts, hipStream_t stream) {
  using namespace i4;
  if (!k || !v) return I4_ERR_NULL;
  int rc = i4_check_kv8cache(cache);
  if (rc) return rc;
  if (x_dtype != cache->dtype) return I4_ERR_DTYPE;
  const int nkv = cache->n_kv_heads, B = cache->batch;
  rc = i4_check_tokens(B, T, nkv, nkv, pos_dev, pos, counts, cache->blocks * KBLK);
  if (rc) return rc;
  if ((T > 1 && token_stride < KHD) || (B > 1 && batch_stride < KHD) ||
      (nkv > 1 && head_stride < KHD))
    return I4_ERR_STRIDE;
  if (((uintptr_t)k & 15) || ((uintptr_t)v & 15) || (batch_stride & 7) || (token_stride & 7) ||
      (head_stride & 7))
    return I4_ERR_ALIGN;
  if (2 * (int64_t)B * nkv > 65535) return I4_ERR_SHAPE;
  const Tokens tk{pos_dev, counts, pos, T};
  // finished blocks at most (at least one workgroup, for the tail)
  const int r = pos_dev ? KBLK - 1 : pos % KBLK;
  const int most = (r + T) / KBLK;
  const dim3 grid((unsigned)(most > 1 ? most : 1), (unsigned)(2 * B * nkv));
  auto go = [&](auto kern) {
    kern<<<grid, 256, 0, stream>>>((const uint16_t*)k, (const uint16_t*)v, batch_stride,
                                   token_stride, head_stride, nkv, tk, cache8(cache));
  };
  const bool e4 = cache->format == I4_KV8_E4M3;
  if (x_dtype == I4_F16) {
    if (e4) go(k_kv8_append<I4_F16, I4_KV8_E4M3>);
    else go(k_kv8_append<I4_F16, I4_KV8_INT8>);
  } else {
    if (e4) go(k_kv8_append<I4_BF16, I4_KV8_E4M3>);
    else go(k_kv8_append<I4_BF16, I4_KV8_INT8>);
  }
  return hipGetLastError() == hipSuccess ? I4_OK : I4_ERR_LAUNCH;
}

extern "C" int i4_kv8_values(const i4_kv8cache* cache, float* k_out, float* v_out,
                             hipStream_t stream) {
  using namespace i4;
  if (!k_out || !v_out) return I4_ERR_NULL;
  const int rc = i4_check_kv8cache(cache);
  if (rc) return rc;
  if (((uintptr_t)k_out & 15) || ((uintptr_t)v_out & 15)) return I4_ERR_ALIGN;
  const int64_t blocks = (int64_t)cache->batch * cache->n_kv_heads * cache->blocks;
  if (blocks > kMaxGrid) return I4_ERR_SHAPE;
  const dim3 grid((unsigned)blocks, 2);
  if (cache->format == I4_KV8_E4M3)
    k_kv8_values<I4_KV8_E4M3><<<grid, 256, 0, stream>>>(cache8(cache), k_out, v_out);
  else
    k_kv8_values<I4_KV8_INT8><<<grid, 256, 0, stream>>>(cache8(cache), k_out, v_out);
  return hipGetLastError() == hipSuccess ? I4_OK : I4_ERR_LAUNCH;
}
