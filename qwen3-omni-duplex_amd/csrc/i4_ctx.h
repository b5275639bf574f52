// Attention over a cached context: the call as kernels see it, shared by the kernel for few
// query rows (i4_ctx_rows.hip) and the one for many (i4_ctx_tile.hip).
//
// The queries of one kv head are its rows: row r is token r / G, head r % G of the group of
// G = n_heads / n_kv_heads, so that every key and value is read once for the whole group,
// whatever G is.
#pragma once

#include "i4_kv.h"

namespace i4 {

// Rows of a kv head up to which k_ctx_rows takes a call: as many as a 16-row product holds.
// With a second one (32 rows) it took 138 us against k_ctx_tile's 156 for 16 sequences of 4
// tokens over 32000 16-bit positions (143 against 152 over 8-bit ones), but 26 against 16 for
// one sequence over 8000 (the parts of 32 rows are merged by one workgroup) and 35 against 22
// for 32 over 1000 8-bit ones.  The rule does not look at the batch: the large ones pay for it.
static constexpr int kFewRows = 16;
static constexpr int kShared = I4_CTX_COUNTERS;  // kv heads whose contexts are shared out
static constexpr int kTileRows = 128;    // of a workgroup of k_ctx_tile

struct CtxArgs {
  const uint16_t* q;
  int64_t qbs, qts, qhs;  // strides in elements
  uint16_t* out;          // [B][T][nq][128]
  Cache16 c;              // the 16-bit cache, or
  Cache8 c8;              // the 8-bit one
  Tokens tk;
  Bounds w;
  int32_t nq, nkv, G, R;  // R = T G rows of a kv head
  int32_t len;            // positions of the cache
  int32_t B;
  int32_t tiles;          // row tiles of a kv head
  int32_t S;              // splits of the context (k_ctx_tile), or
  int32_t wgs;            // workgroups that the contexts are shared out to (k_ctx_rows)
  float c2;               // scale log2(e): weights are powers of two
  float* part;            // [B nkv R][S] or [wgs][rows], [128] sums of e v each, then
  float* ml;              // [2] each: maximum and sum
  int32_t* counters;      // nullable: parts of a kv head that are done, 0 between calls
};

// All of the arguments' cache lines asked for at once, at a kernel's start: the compiler
// loads each group of them where it is used, and every such load is a trip to host memory.
__device__ inline void touch(const CtxArgs& a) {
  asm volatile("" ::"s"(a.q), "s"(a.out), "s"(a.c.v), "s"(a.c8.k), "s"(a.c8.vt), "s"(a.tk.counts),
               "s"(a.nq), "s"(a.part), "s"(a.counters));
}

// The context tiles (64 positions) that rows at positions [plo, phi] see: ns tiles with the
// first tokens, then those of the window from tile w0 on; n in all.
struct CtxTiles {
  int ns, w0, n;
  __device__ inline int at(int i) const { return i < ns ? i : w0 + (i - ns); }
};
__device__ inline CtxTiles ctx_tiles(const Bounds& w, int plo, int phi) {
  const int lo = max(0, plo - w.window + 1);  // the first row's first position in the window
  CtxTiles t;
  t.ns = (min(w.sinks, lo) + 63) >> 6;
  t.w0 = max(lo >> 6, t.ns);
  t.n = t.ns + max((phi >> 6) - t.w0 + 1, 0);
  return t;
}
// whether rows at [plo, phi] all see the positions [j, j + n)
__device__ inline bool all_see(const Bounds& w, int plo, int phi, int j, int n) {
  return j + n - 1 <= plo && (j > phi - w.window || j + n <= w.sinks);
}

// The sequence's tokens: rows of the first `have` tokens have an output, those of the first
// `fit` a position inside the cache (the others come out NaN), from position p0 on.
struct CtxSeq {
  int p0, have, fit;
};
__device__ inline CtxSeq ctx_seq(const CtxArgs& a, int b) {
  CtxSeq s;
  s.p0 = first_pos(a.tk, b);
  s.have = count_of(a.tk, b);
  s.fit = s.p0 < 0 || s.p0 >= a.len ? 0 : min(s.have, a.len - s.p0);
  return s;
}
// where row r of a kv head, of token t, has its output
__device__ inline int64_t ctx_out_of(const CtxArgs& a, int b, int g, int r, int t) {
  return (((int64_t)b * a.tk.T + t) * a.nq + g * a.G + r - t * a.G) * KHD;
}
__device__ inline int64_t ctx_out(const CtxArgs& a, int b, int g, int r) {
  return ctx_out_of(a, b, g, r, r / a.G);
}

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// by value: a bit_cast of a vector's element would read element 0
__device__ inline float as_f32(u32 x) { return __builtin_bit_cast(float, x); }

template <int XT> __device__ inline f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (XT == I4_F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <int XT> __device__ inline f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (XT == I4_F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

template <int XT> __device__ inline u32 pack2(float a, float b) {
  if constexpr (XT == I4_F16) return __builtin_bit_cast(u32, f16x2{(_Float16)a, (_Float16)b});
  else return __builtin_bit_cast(u32, bf16x2{(__bf16)a, (__bf16)b});
}
template <int XT> __device__ inline float lo_f32(u32 x) { return Half<XT>::to_f32((uint16_t)x); }
template <int XT> __device__ inline float hi_f32(u32 x) {
  return Half<XT>::to_f32((uint16_t)(x >> 16));
}

// Weights are 2^(x - m + lift) with m at most kLazy below the true maximum.  In fp16 they reach
// 2^(7 + 8) < 65504 and stay normal numbers down to 2^-21 of the largest.  In bf16 they are at
// most 1, so that sums overflow only where those of the plain form do.
static constexpr float kLazy = 8.f;
template <int XT> static constexpr float kLift = XT == I4_F16 ? 7.f : -kLazy;

// Byte N of w as a signed integer, converted: one instruction.  Written out because the
// compiler otherwise splits the loaded words into bytes as soon as they arrive and carries
// those from tile to tile (four registers for one; it spilled).
template <int N> __device__ inline float byte_f32(u32 w) {
  float r;
  if constexpr (N == 0)
    asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_0"
        : "=v"(r) : "v"(w));
  else if constexpr (N == 1)
    asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_1"
        : "=v"(r) : "v"(w));
  else if constexpr (N == 2)
    asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_2"
        : "=v"(r) : "v"(w));
  else
    asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_3"
        : "=v"(r) : "v"(w));
  return r;
}

// two bytes of an 8-bit word (bytes 2 H, 2 H + 1) as a pair of XT values, exactly
template <int FMT, int XT, int H> __device__ inline u32 cvt_pair(u32 w) {
  if constexpr (FMT == I4_KV8_E4M3) {
    if constexpr (XT == I4_F16)
      return __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, H == 1));
    else
      return __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, H == 1));
  } else {
    return pack2<XT>(byte_f32<2 * H>(w), byte_f32<2 * H + 1>(w));
  }
}
// eight bytes as eight XT values
template <int FMT, int XT> __device__ inline u32x4 cvt8(u32 w0, u32 w1) {
  return u32x4{cvt_pair<FMT, XT, 0>(w0), cvt_pair<FMT, XT, 1>(w0), cvt_pair<FMT, XT, 0>(w1),
               cvt_pair<FMT, XT, 1>(w1)};
}

// whether a pair holds an infinity or a NaN
template <int XT> __device__ inline bool not_finite(u32 x) {
  constexpr u32 E = XT == I4_F16 ? 0x7C00u : 0x7F80u;
  return (x & E) == E || ((x >> 16) & E) == E;
}
// the pair with infinities and NaN as zeros
template <int XT> __device__ inline u32 finite_pair(u32 x) {
  constexpr u32 E = XT == I4_F16 ? 0x7C00u : 0x7F80u;
  if ((x & E) == E) x &= 0xFFFF0000u;
  if (((x >> 16) & E) == E) x &= 0x0000FFFFu;
  return x;
}

}  // namespace i4

// i4_ctx_rows.hip / i4_ctx_tile.hip; fmt: -1 (16-bit cache) or I4_KV8_*
int i4_launch_ctx_tile(const i4::CtxArgs& a, int xt, int fmt, hipStream_t s);
int i4_launch_ctx_rows(const i4::CtxArgs& a, int xt, int fmt, hipStream_t s);
