// Attention of many query rows (prompts and their chunks) over a cached context.  Bound by
// the matrix cores and by LDS reads, which a wave's 32 rows keep in balance.
//
// A workgroup takes 128 rows of one kv head, a wave 32 of them, and walks the context in
// tiles of 64 positions that are double-buffered in LDS.  Everything is computed transposed,
// so that a row's scores, weights and sums stay in the lanes (n, n + 32) of its column:
//   S^T = K Q^T    (32 keys x 32 rows x 16 dims, v_mfma 32x32x16): lane (n, h) gets the
//                  scores of row n with keys 8 (i / 4) + 4 h + i % 4, i < 16;
//   O^T = V^T P^T  (32 dims x 32 rows x 16 keys): that is P^T's operand layout when the
//                  product's k index runs over the keys in the same order, so the weights
//                  are only rounded, never moved.
// V^T's operand: a 16-bit tile is kept [key][dim] as it comes and read with the transposing
// LDS read; an 8-bit value block is [dim][token] already and is stored that way, converted,
// its tokens in the order of the product's k index.
// LDS rows are 256 bytes (K, 16-bit V) or 128 (8-bit V); 16-byte chunk c of row r lies at
// c ^ f(r), so that neither read has bank conflicts.
#include "i4_ctx.h"

namespace i4 {

static constexpr int TKEYS = 64;   // positions of a tile
static constexpr int TBYTES = TKEYS * KHD * 2;  // of a K or V tile in LDS

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef u32 u32x2v __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) unsigned char lds_t;

struct TileAcc {
  f32x16 o[4];  // dims 32 t + 8 (i / 4) + 4 h + i % 4
  float m, l;   // l: this lane's keys alone
};

__device__ inline u32x4 lds_b128(const lds_t* p) {
  return *(const __attribute__((address_space(3))) u32x4*)p;
}
// four rows of four dims each turned: lane i of 16 gets dim i of the rows
__device__ inline u32x2v lds_tr(const lds_t* p) {
  return __builtin_bit_cast(u32x2v, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                        (__attribute__((address_space(3))) s16x4*)p));
}

// 64 rows of a 16-bit cache into LDS (K, then V), straight from memory: each wave instruction
// brings 4 rows.  The loads are not waited for here.  row: of the cache, limited to last.
struct Stage16 {
  u32 k[4], v[4];  // this lane's byte offsets of the chunks within rows
  int row[4];
};
__device__ inline Stage16 stage16_lane(int wave, int lane) {
  Stage16 st;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = 16 * wave + 4 * i + (lane >> 4), c = lane & 15;
    st.row[i] = r;
    st.k[i] = 16u * (c ^ (r & 15));
    st.v[i] = 16u * (c ^ ((r & 7) << 1));
  }
  return st;
}
__device__ inline void load_lds16(const void* base, u32 off, u32 lds) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) u32*)((const char*)base + off),
     (__attribute__((address_space(3))) u32*)(uintptr_t)lds, 16, 0, 0);
}
__device__ inline void wait_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
__device__ inline void stage16(const Stage16& st, const void* k, const void* v, int j0, int last,
                               u32 stride, u32 lds, int wave) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const u32 row = (u32)min(j0 + st.row[i], last) * stride;
    const u32 dst = lds + 1024u * (4 * wave + i);
    load_lds16(k, row + st.k[i], dst);
    load_lds16(v, row + st.v[i], dst + TBYTES);
  }
}

// scores of the tile's 64 keys
template <int XT>
__device__ inline void tile_scores(const lds_t* k, const u32x4 (&q)[8], f32x16 (&s)[2], int n,
                                   int h) {
  const lds_t* row = k + n * 256;
  const int x = (h ^ (n & 15)) * 16;
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) s[t][i] = 0.f;
#pragma unroll
  for (int c = 0; c < 8; ++c)
#pragma unroll
    for (int t = 0; t < 2; ++t)
      s[t] = mfma32<XT>(lds_b128(row + t * 8192 + (x ^ (32 * c))), q[c], s[t]);
}

// scores -> weights in place; c: scale log2(e) (times the keys' scale); key0: the tile's first
// position + 4 h, p: the row's position
__device__ inline void tile_weights(TileAcc& acc, f32x16 (&s)[2], float c, bool partial, int key0,
                                    int p, const Bounds& w) {
  if (partial)
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (!sees(w, p, key0 + 32 * t + 8 * (i >> 2) + (i & 3))) s[t][i] = -__builtin_inff();
  float mx = -__builtin_inff();
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[t][i]);
  mx *= c;  // c > 0
  if (__builtin_amdgcn_ballot_w64(mx > acc.m + kLazy)) {
    const float m = fmaxf(acc.m, fmaxf(mx, __shfl_xor(mx, 32)));
    const float f = m > acc.m ? exp2f(acc.m - m) : 1.f;
    acc.m = m;
    acc.l *= f;
#pragma unroll
    for (int t = 0; t < 4; ++t) acc.o[t] *= f;
  }
  // a row that has seen nothing yet has m = -inf and scores -inf: weights 0
  const float base = acc.m == -__builtin_inff() ? 0.f : acc.m - kLift;
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[t][i] = __builtin_amdgcn_exp2f(fmaf(s[t][i], c, -base));
      acc.l += s[t][i];
    }
}

// the weights of 16 keys (step ks of the tile's four) as the product's operand, and what
// their rounding left
template <int PT> __device__ inline u32x4 weights_hi(const f32x16 (&s)[2], int ks) {
  const f32x16& x = s[ks >> 1];
  const int o = 8 * (ks & 1);
  return u32x4{pack2<PT>(x[o], x[o + 1]), pack2<PT>(x[o + 2], x[o + 3]),
               pack2<PT>(x[o + 4], x[o + 5]), pack2<PT>(x[o + 6], x[o + 7])};
}
template <int PT> __device__ inline u32x4 weights_lo(const f32x16 (&s)[2], int ks, u32x4 hi) {
  const f32x16& x = s[ks >> 1];
  const int o = 8 * (ks & 1);
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    r[i] = pack2<PT>(x[o + 2 * i] - lo_f32<PT>(hi[i]), x[o + 2 * i + 1] - hi_f32<PT>(hi[i]));
  return r;
}

// O^T += V^T P^T for a 16-bit tile.  CLEAN: a tile that some row does not see in full;
// infinities and NaN are taken out of the product (0 times them is NaN) and added to the
// rows that see them.
template <int XT, bool CLEAN>
__device__ __attribute__((always_inline)) inline void tile_values16(TileAcc& acc, const f32x16 (&s)[2], const lds_t* v, int lane,
                                     int key0, int p, const Bounds& w) {
  const int h = lane >> 5, gq = (lane >> 4) & 1, i16 = lane & 15;
  const lds_t* row = v + (4 * h + (i16 >> 2)) * 256 + (i16 & 1) * 8;
  const int x = ((2 * gq + ((i16 & 3) >> 1)) ^ ((4 * h + (i16 >> 2)) << 1)) * 16;
  bool bad = false;
#pragma unroll
  for (int ks = 0; ks < 4; ++ks) {
    const u32x4 b = weights_hi<XT>(s, ks);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const lds_t* at = row + ks * 4096 + (x ^ (64 * t));
      const u32x2v a0 = lds_tr(at), a1 = lds_tr(at + 2048);
      u32x4 a = {a0[0], a0[1], a1[0], a1[1]};
      if constexpr (CLEAN) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          bad |= not_finite<XT>(a[e]);
          a[e] = finite_pair<XT>(a[e]);
        }
      }
      acc.o[t] = mfma32<XT>(a, b, acc.o[t]);
    }
  }
  if constexpr (CLEAN) {
    if (!__builtin_amdgcn_ballot_w64(bad)) return;
    for (int key = 0; key < TKEYS; ++key) {
      const bool see = sees(w, p, key0 + key);
      const lds_t* r = v + key * 256;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // dims 32 t + 8 i + 4 h ..
          const u32x2v y = *(const __attribute__((address_space(3))) u32x2v*)(
              r + ((4 * t + i) ^ ((key & 7) << 1)) * 16 + 8 * h);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float u = lo_f32<XT>(y[e]), z = hi_f32<XT>(y[e]);
            if (see && !(fabsf(u) < __builtin_inff())) acc.o[t][4 * i + 2 * e] += u;
            if (see && !(fabsf(z) < __builtin_inff())) acc.o[t][4 * i + 2 * e + 1] += z;
          }
        }
    }
  }
}

// O^T += V^T P^T for an 8-bit block, in bf16, whose range holds any scale.  TWO: the weights
// as a sum of two (queries in fp16 have three bits more than one bf16 weight)
template <bool TWO>
__device__ inline void tile_values8(TileAcc& acc, const f32x16 (&s)[2], const lds_t* v, int n,
                                    int h) {
  const lds_t* row = v + n * 128;
#pragma unroll
  for (int ks = 0; ks < 4; ++ks) {
    const u32x4 b = weights_hi<I4_BF16>(s, ks);
    u32x4 b2;
    if constexpr (TWO) b2 = weights_lo<I4_BF16>(s, ks, b);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const u32x4 a = lds_b128(row + t * 4096 + (((2 * ks + h) ^ (n & 7)) * 16));
      acc.o[t] = mfma32<I4_BF16>(a, b, acc.o[t]);
      if constexpr (TWO) acc.o[t] = mfma32<I4_BF16>(a, b2, acc.o[t]);
    }
  }
}

// An 8-bit block on its way to LDS: thread t holds 32 bytes of a key's row and of a dim's.
struct Stage8 {
  u32x4 k[2], v[2];
  float ks, vs;
};
__device__ inline void load8(Stage8& st, const Cache8& c, int64_t blk, int tid) {
  const uint8_t *k = c.k + blk * (KBLK * KHD) + tid * 32, *v = c.v + blk * (KBLK * KHD) + tid * 32;
  st.k[0] = ldg16(k);
  st.k[1] = ldg16(k + 16);
  st.v[0] = ldg16(v);
  st.v[1] = ldg16(v + 16);
  st.ks = c.ks[blk];
  st.vs = c.vs[blk];
}
__device__ inline void lds_put(lds_t* p, u32x4 x) {
  *(__attribute__((address_space(3))) u32x4*)p = x;
}
template <int XT, int FMT> __device__ inline void store8(const Stage8& st, lds_t* buf, int tid) {
  const int key = tid >> 2, c0 = 4 * (tid & 3);  // 32 dims: chunks c0 .. c0 + 3
  lds_t* k = buf + key * 256;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    lds_put(k + (((c0 + 2 * i) ^ (key & 15)) * 16), cvt8<FMT, XT>(st.k[i][0], st.k[i][1]));
    lds_put(k + (((c0 + 2 * i + 1) ^ (key & 15)) * 16), cvt8<FMT, XT>(st.k[i][2], st.k[i][3]));
  }
  // 32 tokens of one dim: steps ks = 2 (tid & 1) + i; the product's k index takes tokens
  // 0-3 and 8-11 of a step's 16 in the first half, the others in the second
  const int d = tid >> 1;
  lds_t* v = buf + TBYTES + d * 128;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int c = 4 * (tid & 1) + 2 * i;
    lds_put(v + ((c ^ (d & 7)) * 16), cvt8<FMT, I4_BF16>(st.v[i][0], st.v[i][2]));
    lds_put(v + (((c + 1) ^ (d & 7)) * 16), cvt8<FMT, I4_BF16>(st.v[i][1], st.v[i][3]));
  }
}

// Workgroup (row tile, split, kv head of a sequence); the last rows, which see the most of
// a context, come first.
template <int XT, int FMT>
__global__ __launch_bounds__(256, 2) void k_ctx_tile(CtxArgs a) {
  __shared__ __align__(1024) unsigned char s_tile[2][2 * TBYTES];
  const int heads = (int)gridDim.x / (a.S * a.tiles);  // kv heads of all sequences
  const int hb = blockIdx.x % heads, b = hb / a.nkv, g = hb % a.nkv;
  const int split = blockIdx.x / heads % a.S, rt = a.tiles - 1 - (int)(blockIdx.x / heads / a.S);
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int n = lane & 31, h = lane >> 5;
  const CtxSeq sq = ctx_seq(a, b);
  const int r0 = rt * kTileRows, r = r0 + 32 * wave + n;
  const int tlo = r0 / a.G, thi = min(min(r0 + kTileRows, a.R) - 1, sq.fit * a.G - 1) / a.G;
  const int t = r / a.G;
  const bool mine = r < a.R && t < sq.fit;  // a row with something to attend
  if (sq.fit > tlo) {
    const int plo = sq.p0 + tlo, phi = sq.p0 + thi;
    const int p = mine ? sq.p0 + t : -1;  // -1 sees nothing
    const int rq = mine ? r : r0;         // any row that exists
    const uint16_t* qrow =
        a.q + b * a.qbs + (rq / a.G) * a.qts + (int64_t)(g * a.G + rq % a.G) * a.qhs;
    u32x4 q[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) q[c] = ldg16(qrow + 16 * c + 8 * h);
    TileAcc acc;
    acc.m = -__builtin_inff();
    acc.l = 0.f;
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc.o[u][i] = 0.f;
    const CtxTiles ct = ctx_tiles(a.w, plo, phi);
    const int i0 = (int)((int64_t)ct.n * split / a.S);
    const int i1 = (int)((int64_t)ct.n * (split + 1) / a.S);
    lds_t* lds = (lds_t*)&s_tile[0][0];
    const u32 lds0 = (u32)(uintptr_t)lds;
    const Stage16 st = stage16_lane(wave, lane);
    f32x16 s[2];
    auto attend16 = [&](const lds_t* buf, int j0) {
      const bool partial = !all_see(a.w, plo, phi, j0, TKEYS);
      tile_scores<XT>(buf, q, s, n, h);
      tile_weights(acc, s, a.c2, partial, j0 + 4 * h, p, a.w);
      if (partial) tile_values16<XT, true>(acc, s, buf + TBYTES, lane, j0, p, a.w);
      else tile_values16<XT, false>(acc, s, buf + TBYTES, lane, j0, p, a.w);
    };
    if constexpr (FMT < 0) {
      const u32 stride = (u32)a.c.rs * 2u;
      const uint16_t* k = a.c.k + b * a.c.bs + g * a.c.hs;
      const uint16_t* v = a.c.v + b * a.c.bs + g * a.c.hs;
      if (i0 < i1) stage16(st, k, v, 64 * ct.at(i0), phi, stride, lds0, wave);
      for (int i = i0; i < i1; ++i) {
        const int cur = (i - i0) & 1;
        wait_loads();
        __syncthreads();  // the tile is here, and its other half is free
        if (i + 1 < i1)
          stage16(st, k, v, 64 * ct.at(i + 1), phi, stride, lds0 + (cur ^ 1) * 2 * TBYTES, wave);
        attend16(lds + cur * 2 * TBYTES, 64 * ct.at(i));
      }
    } else {
      const int end = sq.p0 + sq.fit, full = end / KBLK;  // finished blocks, then the tail
      const int64_t hblk = (int64_t)hb * a.c8.blocks;
      // the tail's tile is the last one of the list if it is there at all
      const bool tail = i1 == ct.n && i1 > i0 && ct.at(ct.n - 1) >= full;
      const int e = i1 - (tail ? 1 : 0);
      Stage8 s8;
      float ks = 0.f, vs = 0.f;
      if (i0 < e) {
        load8(s8, a.c8, hblk + ct.at(i0), tid);
        store8<XT, FMT>(s8, lds, tid);
        ks = s8.ks, vs = s8.vs;
      }
      for (int i = i0; i < e; ++i) {
        const int cur = (i - i0) & 1, j0 = 64 * ct.at(i);
        __syncthreads();
        if (i + 1 < e) load8(s8, a.c8, hblk + ct.at(i + 1), tid);
        const bool partial = !all_see(a.w, plo, phi, j0, TKEYS);
        const lds_t* buf = lds + cur * 2 * TBYTES;
        tile_scores<XT>(buf, q, s, n, h);
        if (ks != ks)  // a block that reads as NaN: so do its scores, where they are seen
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int x = 0; x < 16; ++x) s[u][x] = ks;
        tile_weights(acc, s, ks != ks ? a.c2 : a.c2 * ks, partial, j0 + 4 * h, p, a.w);
        // the weights take the values' scale; NaN (a block that reads as NaN) reaches the
        // rows that see one of its keys
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int x = 0; x < 16; ++x) s[u][x] *= vs;
        if (partial)
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int x = 0; x < 16; ++x)
              if (!sees(a.w, p, j0 + 4 * h + 32 * u + 8 * (x >> 2) + (x & 3))) s[u][x] = 0.f;
        tile_values8<XT == I4_F16>(acc, s, buf + TBYTES, n, h);
        if (i + 1 < e) {
          store8<XT, FMT>(s8, lds + (cur ^ 1) * 2 * TBYTES, tid);
          ks = s8.ks, vs = s8.vs;
        }
      }
      if (tail) {
        const int64_t at = (int64_t)hb * (KBLK * KHD);
        __syncthreads();
        stage16(st, a.c8.kt + at, a.c8.vt + at, 0, phi - full * KBLK, KHD * 2u, lds0, wave);
        wait_loads();
        __syncthreads();
        attend16(lds, full * KBLK);
      }
    }
    if (mine) {
      const float l = acc.l + __shfl_xor(acc.l, 32);
      if (a.S > 1) {
        const int64_t at = ((int64_t)hb * a.R + r) * a.S + split;
        if (h == 0) *(float2*)(a.ml + 2 * at) = float2{acc.m, l};
        if (l != 0.f)
#pragma unroll
          for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              *(f32x4*)(a.part + at * KHD + 32 * u + 8 * i + 4 * h) =
                  f32x4{acc.o[u][4 * i], acc.o[u][4 * i + 1], acc.o[u][4 * i + 2],
                        acc.o[u][4 * i + 3]};
      } else {
        uint16_t* y = a.out + ctx_out(a, b, g, r);
        const float inv = 1.0f / l;
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            *(u32x2v*)(y + 32 * u + 8 * i + 4 * h) =
                u32x2v{pack2<XT>(acc.o[u][4 * i] * inv, acc.o[u][4 * i + 1] * inv),
                       pack2<XT>(acc.o[u][4 * i + 2] * inv, acc.o[u][4 * i + 3] * inv)};
      }
    }
  }
  // tokens whose position is outside the cache (the merge writes them when there is one)
  if (a.S == 1 && r < a.R && t >= sq.fit && t < sq.have) {
    u32* y = (u32*)(a.out + ctx_out(a, b, g, r)) + 32 * h;
    for (int i = 0; i < 32; ++i) y[i] = (u32)Half<XT>::QNAN * 0x10001u;
  }
}

}  // namespace i4

int i4_launch_ctx_tile(const i4::CtxArgs& a, int B, int xt, int fmt, hipStream_t s) {
  using namespace i4;
  const dim3 grid((unsigned)(a.tiles * a.S * B * a.nkv));
  auto go = [&](auto kern) { kern<<<grid, 256, 0, s>>>(a); };
  if (xt == I4_F16) {
    if (fmt < 0) go(k_ctx_tile<I4_F16, -1>);
    else if (fmt == I4_KV8_INT8) go(k_ctx_tile<I4_F16, I4_KV8_INT8>);
    else go(k_ctx_tile<I4_F16, I4_KV8_E4M3>);
  } else {
    if (fmt < 0) go(k_ctx_tile<I4_BF16, -1>);
    else if (fmt == I4_KV8_INT8) go(k_ctx_tile<I4_BF16, I4_KV8_INT8>);
    else go(k_ctx_tile<I4_BF16, I4_KV8_E4M3>);
  }
  if (hipGetLastError() != hipSuccess) return I4_ERR_LAUNCH;
  return a.S > 1 ? i4_launch_ctx_merge(a, B, xt, s) : I4_OK;
}
