// Attention of few query rows (at most 16 per kv head: one token of up to 16 query heads per
// kv head, or two of 8) over a long cached context.  Bound by the bytes of the keys and
// values, so those stream from memory straight into the matrix operands' registers: no LDS,
// no transposition through it.
//
// A wave takes context tiles of its own with a softmax state of its own; the waves of a
// workgroup and then the workgroups that share a kv head's context (Share, below) are merged
// at the end.
//   S^T = K Q^T   (16 keys x 16 rows x 32 dims, v_mfma 16x16x32): lane (m = lane % 16, qd =
//                 lane / 16) supplies key m's dims, and gets the scores of query row m with
//                 keys 4 qd + i of the 16.  The keys of a tile are dealt to the 16-key groups
//                 so that lane qd ends up with the scores of 8 (16-bit cache) or 16 (8-bit)
//                 adjacent keys,
//   O^T = V^T P^T (16 dims x 16 rows x 32 keys): which is the operand layout of P^T: the
//                 weights never leave their lane.  V^T's lane (m, qd) needs dims of the same
//                 keys: from a 16-bit cache a lane loads 16 bytes (dims 8 m .. 8 m + 7) of
//                 each of its 8 keys and pairs them with v_perm; 8-bit value blocks are kept
//                 [dim][token], so 16 bytes are a lane's 16 keys.
// Product t of the eight covers dims 8 m + t; a lane's sums are dims 32 qd + 8 i + t.
//
// The weights enter the product as a sum of two 16-bit numbers (the matrix cores are idle
// most of the time here), off by the square of half a step; sums are fp32.
// The running maximum is only raised when a score exceeds it by 2^kLazy.
#include "i4_ctx.h"

namespace i4 {

// A short call is mostly instruction fetch: the code of a launch comes from L2 at some 70
// cycles a 64-byte line, so what runs once is kept small here (no integer division, rolled
// loops).

// n / d for 0 <= n < 2^22, d > 0: the reciprocal is off by 2^-23 of the quotient, less than
// the half that is added
__device__ inline int udiv(int n, int d) {
  return (int)(((float)n + 0.5f) * __builtin_amdgcn_rcpf((float)d));
}

struct RowAcc {
  f32x4 o[8];
  float m, l;  // l: this lane's keys alone
};

__device__ inline float max_qd(float v) {  // over the lanes of a row (qd)
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ inline float sum_qd(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

// scores (in place) -> weights; c: scale log2(e) (times the keys' scale); key0: the lane's
// first key, key0 + 4 k + i the others
template <int XT, int NK>
__device__ inline void weights(RowAcc& acc, f32x4 (&s)[NK], float c, bool partial, int key0, int p,
                               const Bounds& w) {
  float top = -__builtin_inff();
#pragma unroll
  for (int k = 0; k < NK; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float x = s[k][i] * c;
      if (partial) x = sees(w, p, key0 + 4 * k + i) ? x : -__builtin_inff();
      s[k][i] = x;
      top = fmaxf(top, x);
    }
  if (__builtin_amdgcn_ballot_w64(top > acc.m + kLazy)) {
    const float m = fmaxf(acc.m, max_qd(top));
    const float f = m > acc.m ? __builtin_amdgcn_exp2f(acc.m - m) : 1.f;
    acc.m = m;
    acc.l *= f;
#pragma unroll
    for (int t = 0; t < 8; ++t) acc.o[t] *= f;
  }
  // a row that has seen nothing yet has m = -inf and scores -inf: weights 0
  const float base = acc.m == -__builtin_inff() ? 0.f : acc.m - kLift<XT>;
#pragma unroll
  for (int k = 0; k < NK; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s[k][i] = __builtin_amdgcn_exp2f(s[k][i] - base);
      acc.l += s[k][i];
    }
}

// eight weights as two operands that sum to them
template <int XT> __device__ inline void split8(f32x4 a, f32x4 b, u32x4& hi, u32x4& lo) {
  hi = u32x4{pack2<XT>(a[0], a[1]), pack2<XT>(a[2], a[3]), pack2<XT>(b[0], b[1]),
             pack2<XT>(b[2], b[3])};
  lo = u32x4{pack2<XT>(a[0] - lo_f32<XT>(hi[0]), a[1] - hi_f32<XT>(hi[0])),
             pack2<XT>(a[2] - lo_f32<XT>(hi[1]), a[3] - hi_f32<XT>(hi[1])),
             pack2<XT>(b[0] - lo_f32<XT>(hi[2]), b[1] - hi_f32<XT>(hi[2])),
             pack2<XT>(b[2] - lo_f32<XT>(hi[3]), b[3] - hi_f32<XT>(hi[3]))};
}

// Values are loaded as data that is read once (24 sessions under a window 80 -> 73 us, 32
// over 8 bits 143 -> 139); for the keys, whose lines two loads share, that gains less.
static constexpr int kStream = 2;  // cache-policy bit nt of a buffer access

// 32 positions of a 16-bit cache (or of the tail)
struct Half16 {
  u32x4 k[2][4], v[8];
};
// kr, vr end behind the last row that any query sees: rows past it read as zeros
__device__ inline void load_k16(Half16& h, rsrc_t kr, int row0, u32 stride, int m, int qd) {
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const u32 at = (u32)(row0 + 8 * (m >> 2) + 4 * t + (m & 3)) * stride + 16u * qd;
#pragma unroll
    for (int c = 0; c < 4; ++c)
      h.k[t][c] = __builtin_amdgcn_raw_buffer_load_b128(kr, at + 64u * c, 0, 0);
  }
}
__device__ inline void load_v16(Half16& h, rsrc_t vr, int row0, u32 stride, int m, int qd) {
#pragma unroll
  for (int j = 0; j < 8; ++j)
    h.v[j] = __builtin_amdgcn_raw_buffer_load_b128(vr, (u32)(row0 + 8 * qd + j) * stride + 16u * m,
                                                   0, kStream);
}
template <int XT>
__device__ inline void scores16(const Half16& h, const u32x4 (&q)[4], f32x4 (&s)[2]) {
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < 4; ++c) s[t] = mfma16<XT>(h.k[t][c], q[c], s[t]);
  }
}

// Values that a row does not see must not reach it (0 times an infinity is NaN): before the
// product of a tile that is not seen in full, the values of keys that no row sees are
// cleared; where rows differ, infinities and NaN are taken out and added to the rows that
// see them.
template <int XT>
__device__ inline void clean16(RowAcc& acc, Half16& h, rsrc_t vr, int row0, u32 stride, int key0,
                               int m, int qd, int plo, int phi, int p, const Bounds& w) {
  bool bad = false;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int key = key0 + 8 * qd + j;
    // some row sees it: the last one by position, the first one by the window
    const bool seen = key <= phi && (key > plo - w.window || key < w.sinks);
#pragma unroll
    for (int e = 0; e < 4; ++e) h.v[j][e] = seen ? h.v[j][e] : 0u;
  }
  if (plo == phi) return;
#pragma unroll
  for (int j = 0; j < 8; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) bad |= not_finite<XT>(h.v[j][e]);
  if (!__builtin_amdgcn_ballot_w64(bad)) return;
#pragma unroll
  for (int j = 0; j < 8; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) h.v[j][e] = finite_pair<XT>(h.v[j][e]);
  for (int j = 0; j < 32; ++j) {
    const bool see = sees(w, p, key0 + j);
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // dims 32 qd + 8 i + t
      const u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(
          vr, (u32)(row0 + j) * stride + 64u * qd + 16u * i, 0, 0);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float a = lo_f32<XT>(x[e]), b = hi_f32<XT>(x[e]);
        if (see && !(fabsf(a) < __builtin_inff())) acc.o[2 * e][i] += a;
        if (see && !(fabsf(b) < __builtin_inff())) acc.o[2 * e + 1][i] += b;
      }
    }
  }
}

template <int XT>
__device__ inline void values16(RowAcc& acc, const Half16& h, const f32x4 (&s)[2]) {
  u32x4 hi, lo;
  split8<XT>(s[0], s[1], hi, lo);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    u32x4 a, b;  // dims 8 m + 2 e and 8 m + 2 e + 1 of the lane's 8 keys
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      a[j] = __builtin_amdgcn_perm(h.v[2 * j + 1][e], h.v[2 * j][e], 0x05040100u);
      b[j] = __builtin_amdgcn_perm(h.v[2 * j + 1][e], h.v[2 * j][e], 0x07060302u);
    }
    acc.o[2 * e] = mfma16<XT>(a, hi, acc.o[2 * e]);
    acc.o[2 * e + 1] = mfma16<XT>(b, hi, acc.o[2 * e + 1]);
    acc.o[2 * e] = mfma16<XT>(a, lo, acc.o[2 * e]);
    acc.o[2 * e + 1] = mfma16<XT>(b, lo, acc.o[2 * e + 1]);
  }
}

// 64 positions of an 8-bit cache: one block
struct Block8 {
  u32x4 k[4][2], v[8];
  float ks, vs;
};
__device__ inline void load_k8(Block8& x, const Cache8& c, int64_t blk, int m, int qd) {
  const uint8_t* k = c.k + blk * (KBLK * KHD) + (16 * (m >> 2) + (m & 3)) * KHD + 16 * qd;
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int u = 0; u < 2; ++u) x.k[t][u] = ldg16(k + 4 * t * KHD + 64 * u);
  x.ks = c.ks[blk];
}
__device__ inline void load_v8(Block8& x, const Cache8& c, int64_t blk, int m, int qd) {
  const uint8_t* v = c.v + blk * (KBLK * KHD) + 8 * m * KBLK + 16 * qd;
#pragma unroll
  for (int t = 0; t < 8; ++t) x.v[t] = __builtin_nontemporal_load((const u32x4*)(v + t * KBLK));
  x.vs = c.vs[blk];
}
template <int XT, int FMT>
__device__ inline void scores8(const Block8& x, const u32x4 (&q)[4], f32x4 (&s)[4]) {
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      s[t] = mfma16<XT>(cvt8<FMT, XT>(x.k[t][u][0], x.k[t][u][1]), q[2 * u], s[t]);
      s[t] = mfma16<XT>(cvt8<FMT, XT>(x.k[t][u][2], x.k[t][u][3]), q[2 * u + 1], s[t]);
    }
    __builtin_amdgcn_sched_barrier(0);  // one key group's conversions at a time
  }
}
// The weights take the values' scale; both enter the product as bf16, whose range holds any
// scale: bf16's weights of at most 1 times up to 2^121, fp16's of 2^15 times up to 2^10.  Below
// 2^-133 a product is lost, 2^-125 of the largest weight: with the smallest scale, 2^-109, that
// is an output off by up to 2^-117 a position.  A block with scale NaN is NaN for the rows
// that see one of its keys.
template <int FMT>
__device__ inline void values8(RowAcc& acc, const Block8& x, f32x4 (&s)[4], bool partial, int key0,
                               int p, const Bounds& w) {
  const float vs = block_scale(x.vs);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    s[k] *= vs;
    if (partial)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[k][i] = sees(w, p, key0 + 4 * k + i) ? s[k][i] : 0.f;
  }
  u32x4 hi[2], lo[2];
  split8<I4_BF16>(s[0], s[1], hi[0], lo[0]);
  split8<I4_BF16>(s[2], s[3], hi[1], lo[1]);
#pragma unroll
  for (int t = 0; t < 8; ++t)
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const u32x4 a = cvt8<FMT, I4_BF16>(x.v[t][2 * g], x.v[t][2 * g + 1]);
      acc.o[t] = mfma16<I4_BF16>(a, hi[g], acc.o[t]);
      acc.o[t] = mfma16<I4_BF16>(a, lo[g], acc.o[t]);
      __builtin_amdgcn_sched_barrier(0);
    }
}

// Parts go past the caches of this XCD (sc1), as the workgroup that merges them may run on
// another: stored through, counted when the stores are done, read from memory.
__device__ inline void put_part(rsrc_t r, u32 at, float a, float b, float c, float d) {
  __builtin_amdgcn_raw_buffer_store_b128(
      u32x4{__builtin_bit_cast(u32, a), __builtin_bit_cast(u32, b), __builtin_bit_cast(u32, c),
            __builtin_bit_cast(u32, d)},
      r, at, 0, kCoherent);
}

// The contexts shared out: every workgroup gets up to q tiles of one kv head, and kv head
// (b, g) as many workgroups, one behind the other, as its tiles need, with the smallest q
// for which that is at most a.wgs in all.  Sequences of different ages then take the same
// time; every workgroup works this out for itself from the positions.
struct Share {
  int b, g, first, n;  // kv head and its workgroups [first, first + n)
};
__device__ inline int seq_tiles(const CtxArgs& a, int b) {
  const CtxSeq sq = ctx_seq(a, b);
  return sq.fit > 0 ? ctx_tiles(a.w, sq.p0, sq.p0 + sq.fit - 1).n : 0;
}
__device__ inline int parts_of(int tiles, int q) { return max(udiv(tiles + q - 1, q), 1); }
// the share of workgroup `wg`, or with head >= 0 that of this kv head (b nkv + g); false: none
__device__ inline bool find_share(const CtxArgs& a, int wg, int head, int* s_n, Share& sh) {
  if (a.wgs == a.B * a.nkv) {  // a workgroup each
    const int hb = head < 0 ? wg : head;
    const int b = (int)((uint32_t)hb / (uint32_t)a.nkv);
    sh = Share{b, hb - b * a.nkv, hb, 1};
    return true;
  }
  if (a.B == 1) {
    const int n = seq_tiles(a, 0), most = udiv(a.wgs, a.nkv);  // workgroups for a kv head
    const int parts = parts_of(n, max(parts_of(n, most), 4));
    const int g = head < 0 ? udiv(wg, parts) : head;
    sh = Share{0, g, g * parts, parts};
    return g < a.nkv;
  }
  const int lane = threadIdx.x & 63;
  for (int b = threadIdx.x; b < a.B; b += 256) s_n[b] = seq_tiles(a, b);
  __syncthreads();
  // sums of whole numbers below 2^24, exact in fp32
  auto total = [&](auto of) {
    float n = 0.f;
    for (int b = lane; b < a.B; b += 64) n += (float)of(s_n[b]);
    return (int)group_sum<64>(n) * a.nkv;
  };
  auto fits = [&](int q) {
    return total([&](int n) { return parts_of(n, q); }) <= a.wgs;
  };
  // at least 4: a tile a wave
  int lo = max((total([](int n) { return n; }) + a.wgs - 1) / a.wgs, 4);
  if (!fits(lo)) {
    int hi = 0;  // the longest context: one workgroup each
    for (int b = lane; b < a.B; b += 64) hi = max(hi, s_n[b]);
    for (int o = 1; o < 64; o <<= 1) hi = max(hi, __shfl_xor(hi, o));
    for (++lo; lo < hi;) {
      const int q = (lo + hi) >> 1;
      if (fits(q)) hi = q;
      else lo = q + 1;
    }
  }
  int before = 0;  // workgroups of the sequences before
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const int n = b0 + lane < a.B ? parts_of(s_n[b0 + lane], lo) : 0;
    const int end = before + a.nkv * wave_incl_scan(n);
    const uint64_t hit = __ballot(head < 0 ? wg < end : b0 + lane == head / a.nkv);
    if (hit) {
      const int l = __ffsll((unsigned long long)hit) - 1;
      const int parts = __shfl(n, l), start = __shfl(end, l) - a.nkv * parts;
      if (parts == 0) return false;  // lanes past the last sequence
      const int g = head < 0 ? (wg - start) / parts : head % a.nkv;
      sh = Share{b0 + l, g, start + g * parts, parts};
      return true;
    }
    before = __shfl(end, 63);
  }
  return false;
}

// The rows of a kv head from the parts of its workgroups, by one of them: a row to each half
// of a wave, whose lanes take 4 dims, with U parts in flight (a round of loads past the
// caches takes 1.2 us).
template <int XT, int U>
__device__ inline void merge_rows(const CtxArgs& a, const Share& sh, const CtxSeq& sq) {
  const int d = 4 * (threadIdx.x & 31);
  const int64_t at = (int64_t)sh.first * kFewRows;
  const rsrc_t ml = rsrc(a.ml + 2 * at, 8u * kFewRows * sh.n);
  const rsrc_t part = rsrc(a.part + at * KHD, 4u * KHD * kFewRows * sh.n);
#pragma unroll 1
  for (int r = threadIdx.x >> 5; r < a.R; r += 8) {
    float M = -__builtin_inff(), L = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int s0 = 0; s0 < sh.n; s0 += U) {
      u32x2 v[U];
      u32x4 w[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {  // reads past the parts are zeros: an empty part
        const u32 row = kFewRows * (s0 + i) + r;
        v[i] = __builtin_amdgcn_raw_buffer_load_b64(ml, 8u * row, 0, kCoherent);
        w[i] = __builtin_amdgcn_raw_buffer_load_b128(part, 4u * (KHD * row + d), 0, kCoherent);
      }
      __builtin_amdgcn_sched_barrier(0);
      float mb = M;
#pragma unroll
      for (int i = 0; i < U; ++i) mb = as_f32(v[i][1]) == 0.f ? mb : fmaxf(mb, as_f32(v[i][0]));
      const float f0 = M == mb ? 1.f : __builtin_amdgcn_exp2f(M - mb);
      L *= f0;
      o *= f0;
      M = mb;
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const float l = as_f32(v[i][1]);
        if (l == 0.f) continue;  // its sums were never written
        const float f = __builtin_amdgcn_exp2f(as_f32(v[i][0]) - mb);
        L = fmaf(l, f, L);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = fmaf(as_f32(w[i][e]), f, o[e]);
      }
    }
    const int t = udiv(r, a.G);
    if (t >= sq.have) continue;
    u32x2* y = (u32x2*)(a.out + ctx_out_of(a, sh.b, sh.g, r, t) + d);
    const float inv = 1.0f / L;
    *y = t < sq.fit ? u32x2{pack2<XT>(o[0] * inv, o[1] * inv), pack2<XT>(o[2] * inv, o[3] * inv)}
                    : u32x2{} + (u32)Half<XT>::QNAN * 0x10001u;
  }
}

__device__ inline const uint16_t* query_row(const CtxArgs& a, int b, int g, int r) {
  const int t = udiv(r, a.G);
  return a.q + b * a.qbs + t * a.qts + (int64_t)(g * a.G + r - t * a.G) * a.qhs;
}

// few parts: little code; many: one round of loads (a token over 8191 8-bit positions has 32)
template <int XT>
__device__ inline void merge_share(const CtxArgs& a, const Share& sh, const CtxSeq& sq) {
  if (sh.n <= 8) merge_rows<XT, 8>(a, sh, sq);
  else merge_rows<XT, 32>(a, sh, sq);
}

// A workgroup takes its share of the context of one kv head and all of its rows.
template <int XT, int FMT>
__global__ __launch_bounds__(256, 2) void k_ctx_rows(CtxArgs a) {
  __shared__ __align__(16) float s_o[4][16][KHD + 4];
  __shared__ float s_m[4][16], s_l[4][16];
  __shared__ int s_last;
  touch(a);
  Share sh;
  if (!find_share(a, blockIdx.x, -1, (int*)&s_o[0][0][0], sh)) return;
  const int b = __builtin_amdgcn_readfirstlane(sh.b), g = __builtin_amdgcn_readfirstlane(sh.g);
  const int parts = __builtin_amdgcn_readfirstlane(sh.n);
  const int split = __builtin_amdgcn_readfirstlane(blockIdx.x - sh.first);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, m = lane & 15, qd = lane >> 4;
  const CtxSeq sq = ctx_seq(a, b);
  const int thi = sq.fit - 1;  // the last token with something to attend
  RowAcc acc;
  acc.m = -__builtin_inff();
  acc.l = 0.f;
#pragma unroll
  for (int t = 0; t < 8; ++t) acc.o[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int tm = udiv(m, a.G);  // this lane's row's token
  const int p = m < a.R && tm < sq.fit ? sq.p0 + tm : -1;  // its position; -1 sees nothing
  if (thi >= 0) {
    const int plo = sq.p0, phi = sq.p0 + thi;
    const uint16_t* row = query_row(a, b, g, p < 0 ? 0 : m);  // one that exists
    u32x4 q[4];
#pragma unroll
    for (int c = 0; c < 4; ++c)  // dims as the keys' lanes hold them
      q[c] = ldg16(row + (FMT < 0 ? 32 * c + 8 * qd : 64 * (c >> 1) + 16 * qd + 8 * (c & 1)));
    const CtxTiles ct = ctx_tiles(a.w, plo, phi);
    // this workgroup's tiles, dealt to its waves in turn
    const int each = udiv(ct.n, parts), more = ct.n - each * parts;
    const int i0 = split * each + min(split, more), i1 = i0 + each + (split < more ? 1 : 0);
    if constexpr (FMT < 0) {
      const u32 stride = (u32)a.c.rs * 2u, bytes = (u32)phi * stride + KHD * 2u;
      const int64_t base = b * a.c.bs + g * a.c.hs;
      const rsrc_t kr = rsrc(a.c.k + base, bytes), vr = rsrc(a.c.v + base, bytes);
      Half16 h;
      // halves of 32 positions: 2 i + (0, 1) of tile i
      const int e = 2 * i1;
      int x = 2 * i0 + wave;
      auto pos0 = [&](int y) { return 64 * ct.at(y >> 1) + 32 * (y & 1); };
      if (x < e) {
        load_k16(h, kr, pos0(x), stride, m, qd);
        load_v16(h, vr, pos0(x), stride, m, qd);
      }
      for (; x < e; x += 4) {
        const int j0 = pos0(x);
        const bool partial = !all_see(a.w, plo, phi, j0, 32);
        f32x4 s[2];
        scores16<XT>(h, q, s);
        const int jn = pos0(min(x + 4, e - 1));
        if (x + 4 < e) load_k16(h, kr, jn, stride, m, qd);
        weights<XT, 2>(acc, s, a.c2, partial, j0 + 8 * qd, p, a.w);
        if (partial) clean16<XT>(acc, h, vr, j0, stride, j0, m, qd, plo, phi, p, a.w);
        values16<XT>(acc, h, s);
        if (x + 4 < e) load_v16(h, vr, jn, stride, m, qd);
      }
    } else {
      const int end = sq.p0 + sq.fit, full = end / KBLK;  // finished blocks, then the tail
      const int64_t hblk = ((int64_t)b * a.nkv + g) * a.c8.blocks;
      Block8 x8;
      // the tail's tile is the last one of the list if it is there at all
      const bool tail = i1 == ct.n && i1 > i0 && ct.at(ct.n - 1) >= full;
      const int e = i1 - (tail ? 1 : 0);
      int x = i0 + wave;
      if (x < e) {
        load_k8(x8, a.c8, hblk + ct.at(x), m, qd);
        load_v8(x8, a.c8, hblk + ct.at(x), m, qd);
      }
      for (; x < e; x += 4) {
        const int j0 = 64 * ct.at(x);
        const bool partial = !all_see(a.w, plo, phi, j0, 64);
        f32x4 s[4];
        scores8<XT, FMT>(x8, q, s);
        const float c = a.c2 * block_scale(x8.ks);
        const int64_t nb = hblk + ct.at(min(x + 4, e - 1));
        if (x + 4 < e) load_k8(x8, a.c8, nb, m, qd);
        weights<XT, 4>(acc, s, c, partial, j0 + 16 * qd, p, a.w);
        values8<FMT>(acc, x8, s, partial, j0 + 16 * qd, p, a.w);
        if (x + 4 < e) load_v8(x8, a.c8, nb, m, qd);
      }
      if (tail && wave >= 2) {  // its halves, by the two waves that have the least to do
        const int j0 = full * KBLK + 32 * (wave - 2);
        if (j0 <= phi) {
          const u32 stride = KHD * 2u, bytes = (u32)(phi - full * KBLK + 1) * stride;
          const int64_t base = ((int64_t)b * a.nkv + g) * (KBLK * KHD);
          const rsrc_t kr = rsrc(a.c8.kt + base, bytes), vr = rsrc(a.c8.vt + base, bytes);
          u32x4 qn[4];  // dims in the 16-bit order
#pragma unroll
          for (int c = 0; c < 4; ++c) qn[c] = ldg16(row + 32 * c + 8 * qd);
          Half16 h;
          const int row0 = 32 * (wave - 2);
          load_k16(h, kr, row0, stride, m, qd);
          load_v16(h, vr, row0, stride, m, qd);
          f32x4 s[2];
          scores16<XT>(h, qn, s);
          weights<XT, 2>(acc, s, a.c2, true, j0 + 8 * qd, p, a.w);
          clean16<XT>(acc, h, vr, row0, stride, j0, m, qd, plo, phi, p, a.w);
          values16<XT>(acc, h, s);
        }
      }
    }
  }
  // merge the waves: thread t takes row t / 16, dims 8 (t % 16) .. + 7
  const int r = threadIdx.x >> 4, d0 = 8 * (threadIdx.x & 15), t = udiv(r, a.G);
  __syncthreads();  // s_o has been read
  const float l = sum_qd(acc.l);
  if (qd == 0) {
    s_m[wave][m] = acc.m;
    s_l[wave][m] = l;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int e = 0; e < 8; e += 4)
      *(f32x4*)&s_o[wave][m][32 * qd + 8 * i + e] =
          f32x4{acc.o[e][i], acc.o[e + 1][i], acc.o[e + 2][i], acc.o[e + 3][i]};
  __syncthreads();
  if (r < a.R && t < sq.have) {
    float M = -__builtin_inff(), L = 0.f, o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = 0.f;
    for (int v = 0; v < 4; ++v) M = fmaxf(M, s_m[v][r]);
#pragma unroll 1
    for (int v = 0; v < 4; ++v) {
      if (s_m[v][r] == -__builtin_inff() && s_l[v][r] == 0.f) continue;
      const float f = __builtin_amdgcn_exp2f(s_m[v][r] - M);
      L = fmaf(s_l[v][r], f, L);
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = fmaf(s_o[v][r][d0 + i], f, o[i]);
    }
    if (parts > 1 && t < sq.fit) {
      // this workgroup's rows; an empty part is skipped by its sum
      const int64_t at = (int64_t)blockIdx.x * kFewRows;
      const rsrc_t ml = rsrc(a.ml + 2 * at, 8u * kFewRows);
      const rsrc_t part = rsrc(a.part + at * KHD, 4u * KHD * kFewRows);
      if (d0 == 0)
        __builtin_amdgcn_raw_buffer_store_b64(
            u32x2{__builtin_bit_cast(u32, M), __builtin_bit_cast(u32, L)}, ml, 8u * r, 0,
            kCoherent);
      if (L != 0.f) {
        put_part(part, 4u * (KHD * r + d0), o[0], o[1], o[2], o[3]);
        put_part(part, 4u * (KHD * r + d0 + 4), o[4], o[5], o[6], o[7]);
      }
    } else if (parts == 1) {
      const float inv = 1.0f / L;
      u32x4 y;
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = pack2<XT>(o[2 * i] * inv, o[2 * i + 1] * inv);
      if (t >= sq.fit) y = u32x4{} + (u32)Half<XT>::QNAN * 0x10001u;
      *(u32x4*)(a.out + ctx_out_of(a, b, g, r, t) + d0) = y;
    }
  }
  if (parts == 1 || !a.counters) return;
  // the last of the kv head's workgroups merges their parts; the count returns to 0
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this thread's parts are stored
  __syncthreads();
  int32_t* count = a.counters + b * a.nkv + g;
  if (threadIdx.x == 0)
    s_last =
        __hip_atomic_fetch_add(count, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == parts - 1;
  __syncthreads();
  if (!s_last) return;
  if (threadIdx.x == 0)
    __hip_atomic_store(count, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  merge_share<XT>(a, sh, sq);
}

// The same merge as a launch of its own, a workgroup for each kv head.
template <int XT> __global__ __launch_bounds__(256) void k_ctx_rows_merge(CtxArgs a) {
  __shared__ int s_n[kShared];
  Share sh;
  if (!find_share(a, 0, blockIdx.x, s_n, sh) || sh.n == 1) return;
  merge_share<XT>(a, sh, ctx_seq(a, sh.b));
}

template <int XT, int FMT> static void rows_go(const CtxArgs& a, hipStream_t s) {
  k_ctx_rows<XT, FMT><<<a.wgs, 256, 0, s>>>(a);
  if (a.wgs > a.B * a.nkv && !a.counters) k_ctx_rows_merge<XT><<<a.B * a.nkv, 256, 0, s>>>(a);
}

}  // namespace i4

int i4_launch_ctx_rows(const i4::CtxArgs& a, int xt, int fmt, hipStream_t s) {
  using namespace i4;
  if (xt == I4_F16) {
    if (fmt < 0) rows_go<I4_F16, -1>(a, s);
    else if (fmt == I4_KV8_INT8) rows_go<I4_F16, I4_KV8_INT8>(a, s);
    else rows_go<I4_F16, I4_KV8_E4M3>(a, s);
  } else {
    if (fmt < 0) rows_go<I4_BF16, -1>(a, s);
    else if (fmt == I4_KV8_INT8) rows_go<I4_BF16, I4_KV8_INT8>(a, s);
    else rows_go<I4_BF16, I4_KV8_E4M3>(a, s);
  }
  return hipGetLastError() == hipSuccess ? I4_OK : I4_ERR_LAUNCH;
}
