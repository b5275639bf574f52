// What the kernels of a long conversation's KV cache share: the caches as kernels see
// them, the tokens of a sequence, and the host checks.
#pragma once

#include "i4_common.h"

namespace i4 {

static constexpr int KHD = 128;                // head_dim
static constexpr int KBLK = I4_KV8_BLOCK;      // tokens per 8-bit block
static constexpr int KV_MAX_LEN = 1 << 20;     // positions of a cache
static constexpr int ROPE_MAX_POS = 1 << 24;   // positions that fp32 holds exactly
static constexpr int kMaxGrid = (1 << 24) - 1;  // workgroups of 256 threads: fewer than 2^32
static constexpr float KV8_TINY = 0x1p-100f;   // floor of a block's largest magnitude

// The tokens of the call's sequences: where each begins and how many it has.
struct Tokens {
  const int32_t* pos_dev;  // nullable: pos for every sequence
  const int32_t* counts;   // nullable: T for every sequence
  int32_t pos, T;
};
__device__ inline int first_pos(const Tokens& k, int b) {
  return k.pos_dev ? k.pos_dev[b] : k.pos;
}
__device__ inline int count_of(const Tokens& k, int b) {
  return k.counts ? min(max(k.counts[b], 0), k.T) : k.T;
}

// What a query sees: j <= p, and under a window only j > p - window or j < sinks.
// window == 0 is kept as INT32_MAX (p - window is then below every j).
struct Bounds {
  int32_t window, sinks;
};
__device__ inline bool sees(const Bounds& w, int p, int j) {
  return j <= p && (j > p - w.window || j < w.sinks);
}

// A 16-bit cache (strides in elements).
struct Cache16 {
  uint16_t *k, *v;
  int64_t bs, hs, rs;
  int32_t max_len;
};
// An 8-bit cache: blocks of KBLK tokens, keys [token][dim], values [dim][token].
struct Cache8 {
  uint8_t *k, *v;
  float *ks, *vs;
  uint16_t *kt, *vt;
  int32_t blocks;
};

// A block's scale from what is stored: at least the smallest that the append writes, so that
// nothing is divided by a scale of 0 (an empty cache's, or another quantiser's for a block of
// zeros); NaN stays.  Taken where the scale is used, not where it is loaded: there it would
// wait for the block's loads (a 300-token chunk 40 -> 43.6 us).
__device__ inline float block_scale(float x) {
  constexpr float least = KV8_TINY / 448.f;
  return x < least ? least : x;
}

// 8-bit elements: FMT is I4_KV8_INT8 or I4_KV8_E4M3.
template <int FMT> __device__ inline float from_8bit(uint8_t b) {
  if constexpr (FMT == I4_KV8_INT8) return (float)(int8_t)b;
  else return __builtin_amdgcn_cvt_f32_fp8((int)b, 0);
}

}  // namespace i4

// Host checks (i4_kv8.hip): I4_OK or an error code, made before any launch.
int i4_check_tokens(int B, int T, int n_heads, int n_kv_heads, const int32_t* pos_dev, int pos,
                    const int32_t* counts, int limit);
int i4_check_kvcache(const i4_kvcache* c);
int i4_check_kv8cache(const i4_kv8cache* c);
