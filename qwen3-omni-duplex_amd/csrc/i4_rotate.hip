// Rotary embedding of rows of heads: pair (a, b) of a head's dims, turned by the angle
// p inv_freq,
//   a' = (a cos - b sin) factor,  b' = (b cos + a sin) factor,
// with the pair's dims half of the turned part apart, or neighbours.  Bound by the rows' bytes:
// 6001 tokens of 36 heads of 128 dims take 19.6 us (5.6 TB/s), a token 3.1, which is a launch.
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
  u32 pair[(V + 1) / 2];
};

static constexpr int kTokens = 4;  // of a workgroup at most

template <int XT, int V> __device__ inline void put(Bits<V>& y, const float* x) {
  if constexpr (V == 1) {
    y.e[0] = Half<XT>::from_f32(x[0]);
  } else {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) y.pair[i] = pack2<XT>(x[2 * i], x[2 * i + 1]);
  }
}

struct RopeCall {
  Heads q, k;
  Tokens tk;
  Turn turn;
  int32_t rows;   // tokens of all sequences
  int32_t each;   // of them a workgroup
  int32_t shares;  // workgroups that share the heads of the same tokens
  int32_t hd;     // head_dim
  int32_t items;  // of a head
  int32_t zero;   // whether the padding's rows are set to zero
};

// n / d for 0 <= n < 2^22, d > 0: the reciprocal is off by 2^-23 of the quotient, less than the
// half that is added
__device__ inline int quotient(int n, int d) {
  return (int)(((float)n + 0.5f) * __builtin_amdgcn_rcpf((float)d));
}

template <int XT, int V, int LAYOUT>
__global__ __launch_bounds__(256) void k_rope(RopeCall a, RotaryTable<kPairs> rt) {
  __shared__ __align__(16) float s_c[kTokens * kPairs], s_s[kTokens * kPairs];
  __shared__ int s_state[kTokens];  // of a token: padding, in range, out of range
  enum { kPadding, kGood, kOutside };
  typedef typename Vec<V>::type vec;
  const int n = rt.n, heads = a.q.heads + a.k.heads, row0 = blockIdx.x * a.each;
  const int rows = min(a.each, a.rows - row0), total = rows * heads * a.items;
  const int b0 = row0 / a.tk.T, t0 = row0 - b0 * a.tk.T;
  struct Item {
    Bits<V> u, w;
    uint16_t* y;
    int d0, d1, pair, r;
  };
  auto load = [&](int i) {
    Item m{};
    const int rh = quotient(i, a.items), c = i - rh * a.items;
    const int r = quotient(rh, heads), h = rh - r * heads;
    const int over = quotient(t0 + r, a.tk.T), b = b0 + over, t = t0 + r - over * a.tk.T;
    const bool key = h >= a.q.heads;
    const Heads& g = key ? a.k : a.q;
    const int hh = key ? h - a.q.heads : h;
    const uint16_t* x = g.x + b * g.xb + t * g.xt + hh * g.xh;
    m.y = g.y + b * g.yb + t * g.yt + hh * g.yh;
    m.r = r;
    m.pair = V * c;  // the first one, and its dims
    if (LAYOUT == I4_ROPE_HALF && m.pair < n) {
      m.d0 = m.pair, m.d1 = m.pair + n;
    } else {  // neighbours, or dims behind the turned ones
      m.d0 = 2 * m.pair, m.d1 = m.d0 + V;
    }
    if (t < count_of(a.tk, b)) {
      m.u.v = *(const vec*)(x + m.d0);
      if (m.d1 < a.hd) m.w.v = *(const vec*)(x + m.d1);
    }
    return m;
  };
  const int step = 256 * gridDim.y;
  int i = 256 * blockIdx.y + threadIdx.x;
  Item m{};
  if (i < total) m = load(i);  // on its way while the angles are computed
  for (int j = threadIdx.x; j < rows * n; j += 256) {
    const int r = quotient(j, n), e = j - r * n;
    const int over = quotient(t0 + r, a.tk.T), b = b0 + over, t = t0 + r - over * a.tk.T;
    // the sum wraps where a start is near the ends of its type: out of range either way
    const int p = (int)((u32)first_pos(a.tk, b) + (u32)t);
    if (e == 0)
      s_state[r] = t >= count_of(a.tk, b) ? kPadding : turns(a.turn, b, t, p) ? kGood : kOutside;
    float c, s;
    angle_of(turn_pos(a.turn, rt.axis[e], b, t, p), rt.f[e], c, s);
    s_c[j] = c * rt.factor;
    s_s[j] = s * rt.factor;
  }
  __syncthreads();
  for (; i < total; i += step) {
    Item next{};
    if (i + step < total) next = load(i + step);
    const int state = s_state[m.r];
    if (state != kGood) {
      const uint16_t fill = state == kPadding ? (uint16_t)0 : Half<XT>::QNAN;
#pragma unroll
      for (int e = 0; e < V; ++e) m.u.e[e] = m.w.e[e] = fill;
    } else if (m.pair < n) {
      const int at = m.r * n + m.pair;
      float x[2 * V];  // u's elements, then w's
#pragma unroll
      for (int e = 0; e < V; ++e) {
        x[e] = Half<XT>::to_f32(m.u.e[e]);
        x[V + e] = Half<XT>::to_f32(m.w.e[e]);
      }
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float& fa = x[LAYOUT == I4_ROPE_HALF ? e : 2 * e];
        float& fb = x[LAYOUT == I4_ROPE_HALF ? V + e : 2 * e + 1];
        const int p = LAYOUT == I4_ROPE_HALF ? at + e : min(at + e, m.r * n + n - 1);
        const float cs = s_c[p], sn = s_s[p], u = fa;
        fa = fmaf(u, cs, -(fb * sn));
        fb = fmaf(fb, cs, u * sn);
      }
      const Bits<V> u = m.u, w = m.w;
      put<XT, V>(m.u, x);
      put<XT, V>(m.w, x + V);
      if (LAYOUT != I4_ROPE_HALF && m.pair + V > n) {  // neighbours behind the turned dims
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (m.pair + e >= n) {
            if (2 * e < V) m.u.e[2 * e % V] = u.e[2 * e % V];
            else m.w.e[2 * e % V] = w.e[2 * e % V];
            if (2 * e + 1 < V) m.u.e[(2 * e + 1) % V] = u.e[(2 * e + 1) % V];
            else m.w.e[(2 * e + 1) % V] = w.e[(2 * e + 1) % V];
          }
      }
    }
    if (state != kPadding || a.zero) {
      *(vec*)(m.y + m.d0) = m.u.v;
      if (m.d1 < a.hd) *(vec*)(m.y + m.d1) = m.w.v;
    }
    m = next;
  }
}

// Halves whose number of pairs is not a multiple of 4, in rows that allow 16 bytes: an item is one
// such vector of a head, and its dims' partners, at any distance, come through LDS.
template <int XT>
__global__ __launch_bounds__(256) void k_rope_odd(RopeCall a, RotaryTable<kPairs> rt) {
  constexpr int kPad = 2 * kPairs / 8 * 9;  // dims d at d + d / 8: lanes are 8 dims apart
  __shared__ __align__(16) uint16_t s_x[256 * 8];
  __shared__ float s_c[kTokens * kPad], s_s[kTokens * kPad];
  __shared__ int s_state[kTokens];
  enum { kPadding, kGood, kOutside };
  const int n = rt.n, heads = a.q.heads + a.k.heads, row0 = blockIdx.x * a.each;
  const int rows = min(a.each, a.rows - row0), total = rows * heads;  // heads of all its tokens
  const int b0 = row0 / a.tk.T, t0 = row0 - b0 * a.tk.T;
  const int round = 256 / a.items;  // heads at a time
  const int mine = quotient(threadIdx.x, a.items), d0 = 8 * (threadIdx.x - mine * a.items);
  struct Item {
    u32x4 x;
    uint16_t* y;
    int r;
  };
  auto load = [&](int rh) {
    Item m{};
    if (mine >= round || rh >= total) return m;
    const int r = quotient(rh, heads), h = rh - r * heads;
    const int over = quotient(t0 + r, a.tk.T), b = b0 + over, t = t0 + r - over * a.tk.T;
    const bool key = h >= a.q.heads;
    const Heads& g = key ? a.k : a.q;
    const int hh = key ? h - a.q.heads : h;
    m.y = g.y + b * g.yb + t * g.yt + hh * g.yh + d0;
    m.r = r;
    if (t < count_of(a.tk, b)) m.x = ldg16(g.x + b * g.xb + t * g.xt + hh * g.xh + d0);
    return m;
  };
  int base = blockIdx.y * round;
  Item m = load(base + mine);  // on its way while the angles are computed
  for (int j = threadIdx.x; j < rows * n; j += 256) {
    const int r = quotient(j, n), e = j - r * n;
    const int over = quotient(t0 + r, a.tk.T), b = b0 + over, t = t0 + r - over * a.tk.T;
    const int p = (int)((u32)first_pos(a.tk, b) + (u32)t);  // as in k_rope
    if (e == 0)
      s_state[r] = t >= count_of(a.tk, b) ? kPadding : turns(a.turn, b, t, p) ? kGood : kOutside;
    float c, s;
    angle_of(turn_pos(a.turn, rt.axis[e], b, t, p), rt.f[e], c, s);
    const int lo = r * kPad + e + (e >> 3), f = e + n, hi = r * kPad + f + (f >> 3);
    s_c[lo] = s_c[hi] = c * rt.factor;
    s_s[hi] = s * rt.factor;
    s_s[lo] = -s_s[hi];
  }
  for (; base < total; base += round * gridDim.y) {
    __syncthreads();  // the round before has read s_x
    *(u32x4*)(s_x + 8 * threadIdx.x) = m.x;
    __syncthreads();
    const Item next = load(base + round * gridDim.y + mine);
    if (m.y) {
      const int state = s_state[m.r];
      const uint16_t* x = s_x + 8 * (threadIdx.x - d0 / 8);  // the head's row
      u32x4 out = m.x;
      if (state != kGood) {
        out = u32x4{} + (state == kPadding ? 0u : (u32)Half<XT>::QNAN * 0x10001u);
      } else if (d0 < 2 * n) {
        uint16_t e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int d = min(d0 + i, 2 * n - 1), at = m.r * kPad + d + (d >> 3);
          const float u = Half<XT>::to_f32(x[d]), o = Half<XT>::to_f32(x[d < n ? d + n : d - n]);
          e[i] = d0 + i < 2 * n ? Half<XT>::from_f32(fmaf(u, s_c[at], o * s_s[at])) : x[d0 + i];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) out[i] = e[2 * i] | (u32)e[2 * i + 1] << 16;
      }
      if (state != kPadding || a.zero) *(u32x4*)m.y = out;
    }
    m = next;
  }
}

template <int V>
static void rope_go(const RopeCall& a, const RotaryTable<kPairs>& rt, int layout, bool f16,
                    hipStream_t s) {
  const dim3 grid((unsigned)((a.rows + a.each - 1) / a.each), (unsigned)a.shares);
  auto go = [&](auto kern) { kern<<<grid, 256, 0, s>>>(a, rt); };
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
// Whether the output's rows, which several workgroups write, are distinct: from the smallest
// stride on, each steps over all that the ones before reach.
static bool rows_apart(const i4_heads* g, int B, int T, int hd) {
  int64_t n[3] = {B, T, g->heads}, s[3] = {g->yb, g->yt, g->yh};
  __int128 reach = hd;
  for (int i = 0; i < 3; ++i) {
    int j = -1;
    for (int k = 0; k < 3; ++k)
      if (n[k] > 1 && (j < 0 || s[k] < s[j])) j = k;
    if (j < 0) break;
    if (s[j] < reach) return false;
    reach += (__int128)(n[j] - 1) * s[j];
    n[j] = 1;
  }
  return true;
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
  if (!rows_apart(q, B, T, head_dim) || (k && !rows_apart(k, B, T, head_dim)))
    return I4_ERR_STRIDE;
  if (((uintptr_t)pos_dev & 3) || ((uintptr_t)counts & 3)) return I4_ERR_ALIGN;
  if (!turn && !pos_dev && (pos <= -ROPE_MAX_POS || pos > ROPE_MAX_POS - T)) return I4_ERR_SHAPE;
  RopeCall a{};
  a.q = heads_of(*q, B, T);
  if (k) a.k = heads_of(*k, B, T);
  // the widest vector that a head's parts and all rows allow
  const int n = rotary->pairs;
  const bool half = rotary->layout == I4_ROPE_HALF;
  int v = vector_of(a.q, 8);
  if (k) v = vector_of(a.k, v);
  while (v > 1 && head_dim % v) v /= 2;
  // Through LDS where vectors of 2 or 4 bytes would be left and rows are many: 3000 tokens of 36
  // heads of 72 dims 11.8 us against 21.2 (9 pairs), 11.4 against 13.3 (18), but 12.0 against 9.9
  // (36: 8 bytes), and 1000 of 16 heads of 64 dims (30 pairs) 4.5 against 4.1.
  const bool odd = half && v == 8 && n % 4 && (int64_t)B * T * (q->heads + a.k.heads) >= 1 << 15;
  while (v > 1 && !odd && half && n % v) v /= 2;
  a.tk = Tokens{pos_dev, counts, pos, T};
  a.turn = turn_of(turn);
  a.rows = B * T;
  a.hd = head_dim;
  a.zero = zero_padding;
  a.items = odd ? head_dim / 8 : half ? n / v + (head_dim - 2 * n + 2 * v - 1) / (2 * v)
                                      : (head_dim + 2 * v - 1) / (2 * v);
  // A token a workgroup, or the heads of one shared out where the chip has room: 24 tokens of 72
  // heads of 256 dims 6.7 us with one workgroup a token, 3.3 with five; 400 of them 8.3 with room
  // for 1024 workgroups, 9.5 for 512 and 8.2 for 2048, but 1000 of 36 heads of 128 6.4, 6.4 and
  // 6.9.  Two tokens where there are many (3000 of 36 heads of 128: 12.1, 10.7, 11.3 us with one,
  // two, four), four where a token is less than half a workgroup's items (3000 of 2 heads: 5.5,
  // 4.2, 3.7), one again where it is several rounds of them (3000 of 72 heads of 256: 44.1, 46.6,
  // 48.9).
  const int items = (a.q.heads + a.k.heads) * a.items;
  a.each = a.rows < 1536 || items > 512 ? 1 : items < 128 ? 4 : 2;
  a.shares = 1;
  while (a.shares * 256 < items && (int64_t)a.rows * (a.shares + 1) <= 1024) ++a.shares;
  const RotaryTable<kPairs> rt = rotary_table<kPairs>(rotary);
  const bool f16 = x_dtype == I4_F16;
  if (odd) {
    const dim3 grid((unsigned)((a.rows + a.each - 1) / a.each), (unsigned)a.shares);
    if (f16) k_rope_odd<I4_F16><<<grid, 256, 0, stream>>>(a, rt);
    else k_rope_odd<I4_BF16><<<grid, 256, 0, stream>>>(a, rt);
  } else if (v == 8) rope_go<8>(a, rt, rotary->layout, f16, stream);
  else if (v == 4) rope_go<4>(a, rt, rotary->layout, f16, stream);
  else if (v == 2) rope_go<2>(a, rt, rotary->layout, f16, stream);
  else rope_go<1>(a, rt, rotary->layout, f16, stream);
  return hipGetLastError() == hipSuccess ? I4_OK : I4_ERR_LAUNCH;
}
