// Rotary embeddings as kernels see them: the table by value, a token's positions, and the
// cosines and sines of their angles.
#pragma once

#include "i4_kv.h"

namespace i4 {

static constexpr int kPairs = I4_ROPE_MAX_PAIRS;

// N: pairs that the kernel has room for.  It travels in the kernel's arguments: nothing to
// allocate, nothing that a graph could find changed.
template <int N> struct RotaryTable {
  float f[N];
  uint8_t axis[N];
  float factor;
  int32_t n;
};
template <int N> inline RotaryTable<N> rotary_table(const i4_rotary* r) {
  RotaryTable<N> t{};
  for (int i = 0; i < r->pairs; ++i) {
    t.f[i] = r->inv_freq[i];
    t.axis[i] = r->axes ? r->axes[i] : 0;
  }
  t.factor = r->factor;
  t.n = r->pairs;
  return t;
}

// Where the angles' positions come from: given for each token, or the tokens' own.
struct Turn {
  const int32_t* pos;  // nullable
  int64_t as, bs;
  int32_t axes;
};
inline Turn turn_of(const i4_turn* t) {  // one axis: whatever a pair's is, it is read there
  return t ? Turn{t->pos, t->axes > 1 ? t->axis_stride : 0, t->batch_stride, t->axes} : Turn{};
}
__device__ inline bool can_turn(int p) { return p > -ROPE_MAX_POS && p < ROPE_MAX_POS; }
// whether all of the positions that token t of sequence b turns by are in range; p: its own
__device__ inline bool turns(const Turn& u, int b, int t, int p) {
  if (!u.pos) return can_turn(p);
  bool ok = true;
  for (int a = 0; a < u.axes; ++a) ok &= can_turn(u.pos[a * u.as + b * u.bs + t]);
  return ok;
}
__device__ inline int turn_pos(const Turn& u, int axis, int b, int t, int p) {
  return u.pos ? u.pos[axis * u.as + b * u.bs + t] : p;
}

// cos and sin of p f.  The product is exact in fp64 (24 bits each), and so, to 2^-52 of up to
// 2^24 f / 2 pi turns, is its share of a turn; the rest after the nearest quarter is at most
// pi / 4 and goes into the Taylor sums in fp32, whose next terms are below 2^-28 there.
__device__ inline void angle_of(int p, float f, float& c, float& s) {
  const double t = (double)p * (double)f * 0.15915494309189533577;
  const double q = rint(4.0 * t);
  const float a = (float)(fma(-0.25, q, t) * 6.2831853071795864769), z = a * a;
  float sn = fmaf(z, 2.7557319e-6f, -1.9841270e-4f);
  sn = fmaf(z, sn, 8.3333333e-3f);
  sn = fmaf(z, sn, -1.6666667e-1f);
  sn = fmaf(z * a, sn, a);
  float cs = fmaf(z, -2.7557319e-7f, 2.4801587e-5f);
  cs = fmaf(z, cs, -1.3888889e-3f);
  cs = fmaf(z, cs, 4.1666667e-2f);
  cs = fmaf(z, cs, -0.5f);
  cs = fmaf(z, cs, 1.0f);
  // a quarter turn more: (c, s) -> (-s, c); q modulo 4 by its exact remainder
  const int k = (int)(q - 4.0 * floor(0.25 * q));
  const float c0 = k & 1 ? sn : cs, s0 = k & 1 ? cs : sn;
  c = k == 1 || k == 2 ? -c0 : c0;
  s = k >= 2 ? -s0 : s0;
}

}  // namespace i4

// Host checks (i4_rotate.hip)
int i4_check_rotary(const i4_rotary* r, const i4_turn* t);
