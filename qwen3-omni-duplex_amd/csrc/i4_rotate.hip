// Rotary embedding of rows of heads: pair (a, b) of a head's dims, turned by the angle
// p inv_freq,
//   a' = (a cos - b sin) factor,  b' = (b cos + a sin) factor,
// with the pair's dims half of the turned part apart, or neighbours.  Bound by the rows' bytes.
//
// A workgroup takes some tokens and all of their heads, so that a token's angles are computed
// once.  An item is two vectors of V elements, V pairs of them (or dims behind the turned ones,
// copied): 16 bytes each where sizes and strides let them.
#include "i4_rotary.h"

namespace i4 {

struct Heads {
  const uint16_t* x;
  uint16_t* y;
  int64_t xb, xt, xh, yb, yt, yh;
  int32_t heads;
};

template <int V> struct Vec;
template <> struct Vec<8> { typedef u32x4 type; };
template <> struct Vec<4> { typedef u32x2 type; };
template <> struct Vec<2> { typedef u32 type; };
template <> struct Vec<1> { typedef uint16_t type; };

template <int V> union Bits {
  typename Vec<V>::type v;
  uint16_t e[V];
};

struct RopeCall {
  Heads q, k;
  Tokens tk;
  Turn turn;
  int32_t rows;   // tokens of all sequences
  int32_t each;   // of them a workgroup
  int32_t hd;     // head_dim
  int32_t items;  // of a head
  int32_t zero;   // whether the padding's rows are set to zero
};

template <int XT, int V, int LAYOUT>
__global__ __launch_bounds__(256) void k_rope(RopeCall a, RotaryTable<kPairs> rt) {
  __shared__ float s_c[4 * kPairs], s_s[4 * kPairs];
  __shared__ int s_ok[4];
  const int n = rt.n, heads = a.q.heads + a.k.heads, row0 = blockIdx.x * a.each;
  const int rows = min(a.each, a.rows - row0);
  for (int i = threadIdx.x; i < rows * n; i += 256) {
    const int r = i / n, j = i - r * n, b = (row0 + r) / a.tk.T, t = (row0 + r) % a.tk.T;
    // the sum wraps where a start is near the ends of its type: out of range either way
    const int p = (int)((u32)first_pos(a.tk, b) + (u32)t);
    if (j == 0) s_ok[r] = turns(a.turn, b, t, p);
    float c, s;
    angle_of(turn_pos(a.turn, rt.axis[j], b, t, p), rt.f[j], c, s);
    s_c[i] = c * rt.factor;
    s_s[i] = s * rt.factor;
  }
  __syncthreads();
  const int total = rows * heads * a.items;
  for (int i = threadIdx.x; i < total; i += 256) {
    const int rh = i / a.items, c = i - rh * a.items;
    const int r = rh / heads, h = rh - r * heads, b = (row0 + r) / a.tk.T, t = (row0 + r) % a.tk.T;
    const bool have = t < count_of(a.tk, b);
    if (!have && !a.zero) continue;
    const bool key = h >= a.q.heads;
    const Heads& g = key ? a.k : a.q;
    const int hh = key ? h - a.q.heads : h;
    const uint16_t* x = g.x + b * g.xb + t * g.xt + hh * g.xh;
    uint16_t* y = g.y + b * g.yb + t * g.yt + hh * g.yh;
    // the item's first pair and its dims
    int d0, d1, pair = V * c;
    if (LAYOUT == I4_ROPE_HALF && pair < n) {
      d0 = pair, d1 = pair + n;
    } else if (LAYOUT == I4_ROPE_HALF) {
      d0 = 2 * n + 2 * (pair - n), d1 = d0 + V;
    } else {
      d0 = 2 * pair, d1 = d0 + V;
    }
    typedef typename Vec<V>::type vec;
    Bits<V> u{}, w{};
    const bool two = d1 < a.hd;
    if (have) {
      u.v = *(const vec*)(x + d0);
      if (two) w.v = *(const vec*)(x + d1);
    }
    if (have && !s_ok[r]) {
#pragma unroll
      for (int e = 0; e < V; ++e) u.e[e] = w.e[e] = Half<XT>::QNAN;
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        uint16_t *pa, *pb;
        if constexpr (LAYOUT == I4_ROPE_HALF) {
          pa = &u.e[e], pb = &w.e[e];
        } else {
          pa = 2 * e < V ? &u.e[2 * e % V] : &w.e[2 * e % V];
          pb = 2 * e + 1 < V ? &u.e[(2 * e + 1) % V] : &w.e[(2 * e + 1) % V];
        }
        if (pair + e < n) {
          const float cs = s_c[r * n + pair + e], sn = s_s[r * n + pair + e];
          const float fa = Half<XT>::to_f32(*pa), fb = Half<XT>::to_f32(*pb);
          *pa = Half<XT>::from_f32(fmaf(fa, cs, -(fb * sn)));
          *pb = Half<XT>::from_f32(fmaf(fb, cs, fa * sn));
        }
      }
    }
    *(vec*)(y + d0) = u.v;
    if (two) *(vec*)(y + d1) = w.v;
  }
}

template <int V>
static void rope_go(const RopeCall& a, const RotaryTable<kPairs>& rt, int layout, bool f16,
                    hipStream_t s) {
  auto go = [&](auto kern) { kern<<<(unsigned)((a.rows + a.each - 1) / a.each), 256, 0, s>>>(a, rt); };
  if (layout == I4_ROPE_HALF) {
    if (f16) go(k_rope<I4_F16, V, I4_ROPE_HALF>);
    else go(k_rope<I4_BF16, V, I4_ROPE_HALF>);
  } else {
    if (f16) go(k_rope<I4_F16, V, I4_ROPE_INTERLEAVED>);
    else go(k_rope<I4_BF16, V, I4_ROPE_INTERLEAVED>);
  }
}

// the rows as the kernel sees them: strides that nothing is stepped by are 0
static Heads heads_of(const i4_heads& g, int B, int T) {
  auto s = [](int n, int64_t x) { return n > 1 ? x : 0; };
  return Heads{(const uint16_t*)g.x, (uint16_t*)g.y, s(B, g.xb), s(T, g.xt), s(g.heads, g.xh),
               s(B, g.yb), s(T, g.yt), s(g.heads, g.yh), g.heads};
}
// elements of a vector that every row's start and stride allow
static int vector_of(const Heads& g, int v) {
  const uint64_t all = ((uint64_t)(uintptr_t)g.x | (uint64_t)(uintptr_t)g.y) / 2 |
                       (uint64_t)(g.xb | g.xt | g.xh | g.yb | g.yt | g.yh);
  while (v > 1 && all % v) v /= 2;
  return v;
}

static int heads_check(const i4_heads* g, int B, int T, int hd) {
  if (!g->x || !g->y) return I4_ERR_NULL;
  if (g->heads < 1 || g->heads > 1024) return I4_ERR_SHAPE;
  if ((g->heads > 1 && (g->xh < hd || g->yh < hd)) || (T > 1 && (g->xt < hd || g->yt < hd)) ||
      (B > 1 && (g->xb < hd || g->yb < hd)))
    return I4_ERR_STRIDE;
  if (((uintptr_t)g->x & 1) || ((uintptr_t)g->y & 1)) return I4_ERR_ALIGN;
  return I4_OK;
}

}  // namespace i4

int i4_check_rotary(const i4_rotary* r, const i4_turn* t) {
  if (!r || !r->inv_freq) return I4_ERR_NULL;
  if (r->pairs < 1 || r->pairs > I4_ROPE_MAX_PAIRS ||
      (r->layout != I4_ROPE_HALF && r->layout != I4_ROPE_INTERLEAVED) ||
      !(r->factor < __builtin_inff()) || !(r->factor > -__builtin_inff()))
    return I4_ERR_SHAPE;
  if (t) {
    if (!t->pos || (t->axes > 1 && !r->axes)) return I4_ERR_NULL;
    if (t->axes < 1 || t->axes > 4) return I4_ERR_SHAPE;
    if ((t->axes > 1 && t->axis_stride < 0) || t->batch_stride < 0) return I4_ERR_STRIDE;
    if ((uintptr_t)t->pos & 3) return I4_ERR_ALIGN;
  }
  for (int i = 0; i < r->pairs; ++i) {
    if (!(__builtin_fabsf(r->inv_freq[i]) <= 16.f)) return I4_ERR_SHAPE;
    if (t && t->axes > 1 && r->axes[i] >= t->axes) return I4_ERR_SHAPE;
  }
  return I4_OK;
}

extern "C" int i4_rope(const i4_heads* q, const i4_heads* k, int x_dtype, int B, int T,
                       int head_dim, const i4_rotary* rotary, const int32_t* pos_dev, int pos,
                       const i4_turn* turn, const int32_t* counts, int zero_padding,
                       hipStream_t stream) {
  using namespace i4;
  if (!q) return I4_ERR_NULL;
  if (x_dtype != I4_F16 && x_dtype != I4_BF16) return I4_ERR_DTYPE;
  if (B < 1 || B > 65535 || T < 1 || T > KV_MAX_LEN || head_dim < 2 || head_dim > 2 * kPairs ||
      head_dim % 2)
    return I4_ERR_SHAPE;
  int rc = i4_check_rotary(rotary, turn);
  if (rc) return rc;
  if (2 * rotary->pairs > head_dim) return I4_ERR_SHAPE;
  rc = heads_check(q, B, T, head_dim);
  if (!rc && k) rc = heads_check(k, B, T, head_dim);
  if (rc) return rc;
  if ((int64_t)B * T > kMaxGrid) return I4_ERR_SHAPE;
  if (((uintptr_t)pos_dev & 3) || ((uintptr_t)counts & 3)) return I4_ERR_ALIGN;
  if (!turn && !pos_dev && (pos <= -ROPE_MAX_POS || pos > ROPE_MAX_POS - T)) return I4_ERR_SHAPE;
  RopeCall a{};
  a.q = heads_of(*q, B, T);
  if (k) a.k = heads_of(*k, B, T);
  // the widest vector that a head's parts and all rows allow
  const int n = rotary->pairs;
  int v = vector_of(a.q, 8);
  if (k) v = vector_of(a.k, v);
  while (v > 1 && (head_dim % v || (rotary->layout == I4_ROPE_HALF && n % v))) v /= 2;
  a.tk = Tokens{pos_dev, counts, pos, T};
  a.turn = turn_of(turn);
  a.rows = B * T;
  a.each = a.rows >= 4096 ? 4 : a.rows >= 2048 ? 2 : 1;
  a.hd = head_dim;
  a.zero = zero_padding;
  a.items = rotary->layout == I4_ROPE_HALF ? n / v + (head_dim - 2 * n + 2 * v - 1) / (2 * v)
                                           : (head_dim + 2 * v - 1) / (2 * v);
  const RotaryTable<kPairs> rt = rotary_table<kPairs>(rotary);
  const bool f16 = x_dtype == I4_F16;
  if (v == 8) rope_go<8>(a, rt, rotary->layout, f16, stream);
  else if (v == 4) rope_go<4>(a, rt, rotary->layout, f16, stream);
  else if (v == 2) rope_go<2>(a, rt, rotary->layout, f16, stream);
  else rope_go<1>(a, rt, rotary->layout, f16, stream);
  return hipGetLastError() == hipSuccess ? I4_OK : I4_ERR_LAUNCH;
}
