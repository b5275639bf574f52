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
// c ^ f(r), so that the rows of a read spread over the banks.  Conflicts are left all the same:
// a third of the cycles in which LDS is active (18.3 of 55.0 million for a 6001-token prompt).
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
__device__ inline void lds_put(lds_t* p, u32x4 x) {
  *(__attribute__((address_space(3))) u32x4*)p = x;
}
// four rows of four dims each turned: lane i of 16 gets dim i of the rows
__device__ inline u32x2v lds_tr(const lds_t* p) {
  return __builtin_bit_cast(u32x2v, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                        (__attribute__((address_space(3))) s16x4*)p));
}

// 64 rows of a 16-bit cache into LDS (K, then V), straight from memory: a wave instruction
// brings 4 rows, lane x the 16 bytes that belong at 16 x of its kilobyte.  The loads are not
// waited for here: that is wait_loads(), before the barrier in front of their use.  They are
// written out because the compiler waits for one of its own before the next LDS read of
// whatever address, here for the tile after the one that is read.  m0 says where in LDS; no
// register is written.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // m0 is reserved: nothing else holds it here
__device__ inline void load_lds16(uint64_t base, u32 off, u32 lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
               :
               : "v"(off), "s"(base), "s"(lds)
               : "memory", "m0");
}
#pragma clang diagnostic pop
// every load of this wave (the builtin, so that the compiler knows its own to be there)
__device__ inline void wait_loads() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
  asm volatile("" ::: "memory");
}
// an address that is the same in all lanes
__device__ inline uint64_t uniform(const void* p) {
  const uint64_t x = (uint64_t)p;
  return (uint64_t)(u32)__builtin_amdgcn_readfirstlane((int)x) |
         (uint64_t)(u32)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32;
}
// Row j0 + r of the cache, limited to last.
__device__ inline void stage16(uint64_t k, uint64_t v, int j0, int last, u32 stride, u32 lds,
                               int wave, int lane) {
  const int r4 = lane >> 4, c = lane & 15;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = 16 * wave + 4 * i + r4;
    const u32 row = (u32)min(j0 + r, last) * stride;
    const u32 dst = lds + 1024u * (4 * wave + i);
    load_lds16(k, row + 16u * (c ^ (4 * i + r4)), dst);
    load_lds16(v, row + 16u * (c ^ ((4 * (i & 1) + r4) << 1)), dst + TBYTES);
  }
}

// The same from pages: this wave's 16 rows, which lie in one page (u), from position j on.  A
// missing page's keys are NaN, so that the rows that see one are NaN, and its values 0.
template <int XT>
__device__ inline void stage_pages(const Pages& pg, const PageRows& u, int j, int last, u32 lds,
                                   int wave, int lane) {
  if (u.bad) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      lds_t* dst = (lds_t*)(uintptr_t)(lds + 1024u * (4 * wave + i) + 16u * lane);
      lds_put(dst, u32x4{} + (u32)Half<XT>::QNAN * 0x10001u);
      lds_put(dst + TBYTES, u32x4{});
    }
    return;
  }
  const int r4 = lane >> 4, c = lane & 15;
  const uint64_t k = uniform((const char*)pg.k + u.at), v = uniform((const char*)pg.v + u.at);
  const int most = last - min(j, last & ~15);  // the last row that anything sees
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const u32 row = (u32)min(4 * i + r4, most) * (KHD * 2u);
    const u32 dst = lds + 1024u * (4 * wave + i);
    load_lds16(k, row + 16u * (c ^ (4 * i + r4)), dst);
    load_lds16(v, row + 16u * (c ^ ((4 * (i & 1) + r4) << 1)), dst + TBYTES);
  }
}

// While a wave is among its products it goes before the other one of its SIMD (s_setprio),
// whose vector work fits in between: 293 -> 291 us for a 6001-token prompt, 228 -> 226 for a
// 5000-token one over 8 bits.
//
// Tried and slower: the next tile's scores computed between this tile's exponentials within
// a wave (11 % more cycles: a second set of scores leaves fewer operands read ahead).

// A fence for the scheduler: LDS reads are issued two products ahead of their use, which it
// would undo to save registers (a wave then waits out LDS's latency at every product).
#define I4_ORDER() __builtin_amdgcn_sched_barrier(0)

// x as a value that nothing is known of: what the rare tiles compute from it stays with them
// instead of being prepared in front of the loop, where it took registers from the others.
__device__ inline int opaque(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// scores of the tile's 64 keys
template <int XT>
__device__ inline void tile_scores(const lds_t* k, const u32x4 (&q)[8], f32x16 (&s)[2], int n,
                                   int h) {
  const lds_t* row = k + n * 256;
  const int x = (h ^ (n & 15)) * 16;
  u32x4 a[3][2];
  auto load = [&](int c) {
#pragma unroll
    for (int t = 0; t < 2; ++t) a[c % 3][t] = lds_b128(row + t * 8192 + (x ^ (32 * c)));
  };
  load(0);
  load(1);
  __builtin_amdgcn_s_setprio(1);
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) s[t][i] = 0.f;
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    if (c < 6) load(c + 2);
    I4_ORDER();
#pragma unroll
    for (int t = 0; t < 2; ++t) s[t] = mfma32<XT>(a[c % 3][t], q[c], s[t]);
    I4_ORDER();
  }
  __builtin_amdgcn_s_setprio(0);
}

// whether the maximum has to be raised for these scores, and raising it; c: scale log2(e)
// (times the keys' scale), positive
__device__ inline void tile_max(TileAcc& acc, const f32x16 (&s)[2], float c) {
  float mx = -__builtin_inff();
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[t][i]);
  mx *= c;
  if (__builtin_amdgcn_ballot_w64(mx > acc.m + kLazy)) {
    const float m = fmaxf(acc.m, fmaxf(mx, __shfl_xor(mx, 32)));
    const float f = m > acc.m ? exp2f(acc.m - m) : 1.f;
    acc.m = m;
    acc.l *= f;
#pragma unroll
    for (int t = 0; t < 4; ++t) acc.o[t] *= f;
  }
}
// The weights of 16 keys (step ks of the tile's four) as the product's operand: one 16-bit number
// each.  A second one for what the rounding leaves, as the kernel for few rows has, would make
// the second product twice as long here, where the matrix cores are the bound.  With the sum of
// the rounded weights the error against 64 bits is that of weights and values in fp32 to within
// 2 % where a row sees many keys (relative 0.0017 in bf16 either way, most of it the output's
// own rounding) and 1.2 times it where a window holds few.
template <int PT> __device__ inline u32x4 weights16(const f32x16 (&s)[2], int ks) {
  const f32x16& x = s[ks >> 1];
  const int o = 8 * (ks & 1);
  return u32x4{pack2<PT>(x[o], x[o + 1]), pack2<PT>(x[o + 2], x[o + 3]),
               pack2<PT>(x[o + 4], x[o + 5]), pack2<PT>(x[o + 6], x[o + 7])};
}
// scores -> weights times 2^lift in place; returns their sum.  rounded: as they enter the
// product, so that what rounding adds to the weights is divided out again (two an instruction,
// in the time that the fp32 additions take)
template <int PT>
__device__ inline float tile_weights(const TileAcc& acc, f32x16 (&s)[2], float c, float lift,
                                     bool rounded = true) {
  // a row that has seen nothing yet has m = -inf and scores -inf: weights 0
  const float base = acc.m == -__builtin_inff() ? lift : lift - acc.m;
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i)
      s[t][i] = __builtin_amdgcn_exp2f(fmaf(s[t][i], c, base));
  if (!rounded) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) sum[i & 3] += s[t][i];
  } else {
    constexpr u32 ones = PT == I4_F16 ? 0x3C003C00u : 0x3F803F80u;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      const u32x4 b = weights16<PT>(s, ks);
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[ks] = Half<PT>::dot2(b[i], ones, sum[ks]);
    }
  }
  return (sum[0] + sum[1]) + (sum[2] + sum[3]);
}
// v where the row does not see the key; key0: the tile's first position + 4 h
__device__ inline void tile_mask(f32x16 (&s)[2], int key0, int p, const Bounds& w, float v) {
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if (!sees(w, p, key0 + 32 * t + 8 * (i >> 2) + (i & 3))) s[t][i] = v;
      if ((i & 3) == 3) I4_ORDER();  // few conditions at a time
    }
}

// O^T += V^T P^T for a 16-bit tile
template <int XT>
__device__ inline void tile_values16(TileAcc& acc, const f32x16 (&s)[2], const lds_t* v,
                                     int lane) {
  const int h = lane >> 5, gq = (lane >> 4) & 1, i16 = lane & 15;
  const lds_t* row = v + (4 * h + (i16 >> 2)) * 256 + (i16 & 1) * 8;
  const int x = ((2 * gq + ((i16 & 3) >> 1)) ^ ((4 * h + (i16 >> 2)) << 1)) * 16;
  u32x4 a[3][2];  // two of a step's four products at a time
  auto load = [&](int y) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const lds_t* at = row + (y >> 1) * 4096 + (x ^ (64 * (2 * (y & 1) + u)));
      const u32x2v a0 = lds_tr(at), a1 = lds_tr(at + 2048);
      a[y % 3][u] = u32x4{a0[0], a0[1], a1[0], a1[1]};
    }
  };
  load(0);
  load(1);
  u32x4 b;
  __builtin_amdgcn_s_setprio(1);
#pragma unroll
  for (int y = 0; y < 8; ++y) {
    if (y < 6) load(y + 2);
    if ((y & 1) == 0) b = weights16<XT>(s, y >> 1);
    I4_ORDER();
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int t = 2 * (y & 1) + u;
      acc.o[t] = mfma32<XT>(a[y % 3][u], b, acc.o[t]);
    }
    I4_ORDER();
  }
  __builtin_amdgcn_s_setprio(0);
}

// Values that a row does not see must not reach it, and 0 times an infinity or a NaN would.
// In a tile that some row does not see in full they are cleared in LDS (this thread's 64
// bytes of it; returns whether there were any)
template <int XT> __device__ inline bool clear_not_finite(lds_t* v, int tid) {
  bool bad = false;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    lds_t* at = v + 4096 * j + 16 * tid;
    u32x4 x = lds_b128(at);
    const bool here = not_finite<XT>(x[0]) || not_finite<XT>(x[1]) || not_finite<XT>(x[2]) ||
                      not_finite<XT>(x[3]);
    if (here) {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = finite_pair<XT>(x[e]);
      lds_put(at, x);
    }
    bad |= here;
  }
  return bad;
}
// and added to the rows that see them when all tiles are done: whatever they meet, they stay.
// row(key): the values of a key of the tile at position j0, of which `rows` exist
template <int XT, class Row>
__device__ inline void add_not_finite(TileAcc& acc, Row row, int rows, int j0, int p, int h,
                                      const Bounds& w) {
  for (int key = 0; key < rows; ++key) {
    const bool see = sees(w, p, j0 + key);
    const char* r = row(key) + 8 * h;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // dims 32 t + 8 i + 4 h ..
        const u32x2v y = *(const u32x2v*)(r + 64 * t + 16 * i);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float u = lo_f32<XT>(y[e]), z = hi_f32<XT>(y[e]);
          if (see && !(fabsf(u) < __builtin_inff())) acc.o[t][4 * i + 2 * e] += u;
          if (see && !(fabsf(z) < __builtin_inff())) acc.o[t][4 * i + 2 * e + 1] += z;
        }
      }
  }
}

// O^T += V^T P^T for an 8-bit block
template <int XT>
__device__ inline void tile_values8(TileAcc& acc, const f32x16 (&s)[2], const lds_t* v, int n,
                                    int h) {
  const lds_t* row = v + n * 128;
  u32x4 a[3][2];
  auto load = [&](int y) {
#pragma unroll
    for (int u = 0; u < 2; ++u)
      a[y % 3][u] = lds_b128(row + (2 * (y & 1) + u) * 4096 + ((((y & ~1) + h) ^ (n & 7)) * 16));
  };
  load(0);
  load(1);
  u32x4 b;
  __builtin_amdgcn_s_setprio(1);
#pragma unroll
  for (int y = 0; y < 8; ++y) {
    if (y < 6) load(y + 2);
    if ((y & 1) == 0) b = weights16<XT>(s, y >> 1);
    I4_ORDER();
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int t = 2 * (y & 1) + u;
      acc.o[t] = mfma32<XT>(a[y % 3][u], b, acc.o[t]);
    }
    I4_ORDER();
  }
  __builtin_amdgcn_s_setprio(0);
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
    lds_put(v + ((c ^ (d & 7)) * 16), cvt8<FMT, XT>(st.v[i][0], st.v[i][2]));
    lds_put(v + (((c + 1) ^ (d & 7)) * 16), cvt8<FMT, XT>(st.v[i][1], st.v[i][3]));
  }
}

// The list of context tiles that a call's row tiles see, by all threads of a workgroup: its
// length for one kv head before each row tile m = b a.tiles + rt to s_at [0, M].
__device__ inline Runs plan_runs(const CtxArgs& a, int* s_at, int* s_sum, int most) {
  const int M = a.B * a.tiles, tid = threadIdx.x, each = (M + 255) / 256;
  int sum = 0;
  for (int m = tid * each; m < min(M, (tid + 1) * each); ++m) {
    const int b = m / a.tiles, tlo = (m - b * a.tiles) * kTileRows / a.G;
    const CtxSeq sq = ctx_seq(a, b);
    const int thi = min(((m - b * a.tiles + 1) * kTileRows - 1) / a.G, sq.fit - 1);
    s_at[m] = sum;
    if (sq.fit > tlo) sum += kRowTile + ctx_tiles(a.w, sq.p0 + tlo, sq.p0 + thi).n;
  }
  const int end = wave_incl_scan(sum);
  if ((tid & 63) == 63) s_sum[tid >> 6] = end;
  __syncthreads();
  int before = end - sum, all = 0;
  for (int w = 0; w < 4; ++w) {
    if (w < tid >> 6) before += s_sum[w];
    all += s_sum[w];
  }
  all = __builtin_amdgcn_readfirstlane(all);
  for (int m = tid * each; m < min(M, (tid + 1) * each); ++m) s_at[m] += before;
  if (tid == 0) s_at[M] = all;
  Runs r;
  r.total = (int64_t)all * a.nkv;
  r.wgs = (int)min(runs_of(r.total), (int64_t)most);
  __syncthreads();
  return r;
}

// Workgroup (row tile, split, kv head of a sequence); the last rows, which see the most of
// a context, come first.
// SHARED: every workgroup takes a run of the list of all row tiles' context tiles instead, so
// that all end together however long the sequences are and however many rows are padding.  A row
// tile that lies in one run is done there; of the others each run leaves a part, at most two:
// number 2 w of a row tile that began before run w, 2 w + 1 of one that ends behind it.
template <int XT, int FMT, bool SHARED>
__global__ __launch_bounds__(256, 2) void k_ctx_tile(CtxArgs a) {
  __shared__ __align__(1024) unsigned char s_tile[2][2 * TBYTES];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int n = lane & 31, h = lane >> 5;
  int hb, b, g, split = 0, rt;
  [[maybe_unused]] int run = 0;
  [[maybe_unused]] int64_t at = 0, stop = 0;
  [[maybe_unused]] int* s_at = nullptr;
  if constexpr (SHARED) {
    __shared__ int s_plan[kPlanned + 1], s_sum[4];
    s_at = s_plan;
    const Runs runs = plan_runs(a, s_plan, s_sum, gridDim.x);
    const int M = a.B * a.tiles;
    if (blockIdx.x == 0) {  // for the merge
      for (int m = tid; m <= M; m += 256) a.plan[m] = s_plan[m];
      if (tid == 0) a.plan[M + 1] = runs.wgs;
    }
    // one XCD's workgroups take runs that are neighbours: they read the same contexts
    const int per = runs.wgs >> 3;
    run = per ? (int)(blockIdx.x & 7) * per + (int)(blockIdx.x >> 3) : blockIdx.x;
    if (per ? (int)(blockIdx.x >> 3) >= per : run >= runs.wgs) return;
    at = runs.first(run);
    stop = runs.first(run + 1);
  } else {
    const int heads = (int)gridDim.x / (a.S * a.tiles);  // kv heads of all sequences
    hb = blockIdx.x % heads, b = hb / a.nkv, g = hb % a.nkv;
    split = blockIdx.x / heads % a.S, rt = a.tiles - 1 - (int)(blockIdx.x / heads / a.S);
  }
  do {
    [[maybe_unused]] int from = 0, to = 0;  // SHARED: the context tiles of this row tile
    if constexpr (SHARED) {
      if (at >= stop) break;
      const int M = a.B * a.tiles, one = __builtin_amdgcn_readfirstlane(s_at[M]);
      g = (int)(at / one);
      const int u = (int)(at - (int64_t)g * one);
      int lo = 0, hi = M;  // the row tile that place u is of: s_at[lo] <= u < s_at[hi]
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (__builtin_amdgcn_readfirstlane(s_at[mid]) <= u) lo = mid;
        else hi = mid;
      }
      const int begin = __builtin_amdgcn_readfirstlane(s_at[lo]) + kRowTile;
      const int end = __builtin_amdgcn_readfirstlane(s_at[lo + 1]);
      b = lo / a.tiles, rt = lo - b * a.tiles, hb = b * a.nkv + g;
      const int last = (int)min((int64_t)end, u + (stop - at));
      at += last - u;
      from = max(u - begin, 0), to = last - begin;
      if (to <= from) continue;
      __syncthreads();  // the tiles of the row tile before have been read
    }
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
      const int i0 = SHARED ? from : (int)((int64_t)ct.n * split / a.S);
      const int i1 = SHARED ? to : (int)((int64_t)ct.n * (split + 1) / a.S);
      lds_t* lds = (lds_t*)&s_tile[0][0];
      const u32 lds0 = __builtin_amdgcn_readfirstlane((u32)(uintptr_t)lds);
      f32x16 s[2];
      bool bad = false;  // values that are not finite in a tile that not all rows see in full
      auto whole = [&](int i) { return all_see(a.w, plo, phi, 64 * ct.at(i), TKEYS); };
      auto attend16 = [&](lds_t* buf, int j0, bool edge) {
        if (edge) bad |= __syncthreads_or(clear_not_finite<XT>(buf + TBYTES, tid));
        tile_scores<XT>(buf, q, s, n, h);
        if (edge) tile_mask(s, j0 + 4 * opaque(h), opaque(p), a.w, -__builtin_inff());
        tile_max(acc, s, a.c2);
        acc.l += tile_weights<XT>(acc, s, a.c2, kLift<XT>);
        tile_values16<XT>(acc, s, buf + TBYTES, lane);
      };
      if constexpr (FMT == kPaged) {
        const int32_t* table = a.pg.table + b * a.pg.ts;
        // this wave's 16 positions of tile i; behind the last row's own, that row's
        auto rows_at = [&](int i) {
          return page_rows(a.pg, table, g, min(64 * ct.at(i) + 16 * wave, phi) & ~15);
        };
        PageRows next{};  // looked up a tile before its rows are loaded
        if (i0 < i1) {
          stage_pages<XT>(a.pg, rows_at(i0), 64 * ct.at(i0) + 16 * wave, phi, lds0, wave, lane);
          next = rows_at(min(i0 + 1, i1 - 1));
        }
        for (int i = i0; i < i1; ++i) {
          const int cur = (i - i0) & 1;
          wait_loads();
          __syncthreads();  // the tile is here, and its other half is free
          if (i + 1 < i1) {
            stage_pages<XT>(a.pg, next, 64 * ct.at(i + 1) + 16 * wave, phi,
                            lds0 + (cur ^ 1) * 2 * TBYTES, wave, lane);
            next = rows_at(min(i + 2, i1 - 1));
          }
          attend16(lds + cur * 2 * TBYTES, 64 * ct.at(i), !whole(i));
        }
        if (bad)
          for (int i = i0; i < i1; ++i) {
            const int j0 = 64 * ct.at(i);
            if (!whole(i))
              add_not_finite<XT>(acc, [&](int key) {
                const int j = __builtin_amdgcn_readfirstlane(j0 + key);
                return (const char*)a.pg.v + page_rows(a.pg, table, g, j & ~15).at + (j & 15) * 256;
              }, min(TKEYS, phi - j0 + 1), j0, p, h, a.w);
          }
      } else if constexpr (FMT == kDense) {
        const u32 stride = (u32)a.c.rs * 2u;
        const uint16_t* k = a.c.k + b * a.c.bs + g * a.c.hs;
        const uint16_t* v = a.c.v + b * a.c.bs + g * a.c.hs;
        const uint64_t ku = uniform(k), vu = uniform(v);
        if (i0 < i1) stage16(ku, vu, 64 * ct.at(i0), phi, stride, lds0, wave, lane);
        for (int i = i0; i < i1; ++i) {
          const int cur = (i - i0) & 1;
          wait_loads();
          __syncthreads();  // the tile is here, and its other half is free
          if (i + 1 < i1)
            stage16(ku, vu, 64 * ct.at(i + 1), phi, stride, lds0 + (cur ^ 1) * 2 * TBYTES, wave,
                    lane);
          attend16(lds + cur * 2 * TBYTES, 64 * ct.at(i), !whole(i));
        }
        if (bad)
          for (int i = i0; i < i1; ++i) {
            const int j0 = 64 * ct.at(i);
            if (!whole(i))
              add_not_finite<XT>(acc, [&](int key) {
                return (const char*)v + (int64_t)(j0 + key) * stride;
              }, min(TKEYS, phi - j0 + 1), j0, p, h, a.w);
          }
      } else {
        const int end = sq.p0 + sq.fit, full = end / KBLK;  // finished blocks, then the tail
        const int64_t hblk = (int64_t)hb * a.c8.blocks;
        // the tail's tile is the last one of the list if it is there at all
        const bool tail = i1 == ct.n && i1 > i0 && ct.at(ct.n - 1) >= full;
        const int e = i1 - (tail ? 1 : 0);
        Stage8 s8;
        float ks = 0.f, vs = 0.f;
        // The weights that enter the product take the values' scale, in the exponent; their sum
        // gives it back.  As the 16-bit types' ranges do not hold every scale, it is taken in units
        // of a power of two near it, and the sums so far follow when the unit changes: in fp16
        // where a scale is above it or below an eighth of it, in bf16 above 2^10 or below 2^-60.
        // The unit stays above 2^-30 (bf16: 2^-80) of the largest scale there was, so that the sums
        // do not overflow: what a block of so much smaller values adds is lost to rows that met
        // the larger ones, and to rows of this workgroup that did not see them.
        constexpr bool F16 = XT == I4_F16;
        constexpr float kUp = F16 ? 1.f : 0x1p10f, kDown = F16 ? 0.125f : 0x1p-60f;
        constexpr float kFloor = F16 ? 0x1p-30f : 0x1p-80f;
        float unit = 1.f, per = 1.f, top = 0.f;  // per = 1 / unit
        auto set_unit = [&](float u) {
          const float f = unit / u;
#pragma unroll
          for (int t = 0; t < 4; ++t) acc.o[t] *= f;
          unit = u;
          per = 1.0f / u;
        };
        if (i0 < e) {
          load8(s8, a.c8, hblk + ct.at(i0), tid);
          store8<XT, FMT>(s8, lds, tid);
          ks = block_scale(s8.ks), vs = block_scale(s8.vs);
        }
        for (int i = i0; i < e; ++i) {
          const int cur = (i - i0) & 1, j0 = 64 * ct.at(i);
          __syncthreads();
          if (i + 1 < e) load8(s8, a.c8, hblk + ct.at(i + 1), tid);
          const lds_t* buf = lds + cur * 2 * TBYTES;
          if (ks + vs == ks + vs) {
            tile_scores<XT>(buf, q, s, n, h);
            if (!whole(i)) tile_mask(s, j0 + 4 * opaque(h), opaque(p), a.w, -__builtin_inff());
            const float c = fmaxf(a.c2 * ks, 0x1p-126f);  // above 0: masked scores stay -inf
            tile_max(acc, s, c);
            // the power of two above vs; every block's counts among the largest
            const float near = as_f32((__builtin_bit_cast(u32, vs) & 0x7F800000u) + 0x00800000u);
            top = fmaxf(top, near);
            if (!(vs <= kUp * unit && vs > kDown * unit)) {
              const float u = fmaxf(near, kFloor * top);
              if (u != unit) set_unit(u);
            }
            const float r = F16 ? vs * per : fmaxf(vs * per, 0x1p-100f);
            // (in units of a much larger block an fp16 block's weights may round to 0: then the
            // sum is of the fp32 ones)
            const float sum = tile_weights<XT>(acc, s, c, kLift<XT> + log2f(r), !F16 || r > 0.125f);
            acc.l = fmaf(sum, 1.0f / r, acc.l);
            tile_values8<XT>(acc, s, buf + TBYTES, n, h);
          } else if (j0 <= p && (min(j0 + KBLK - 1, p) > p - a.w.window || j0 < a.w.sinks)) {
            acc.l = __builtin_nanf("");  // a block that reads as NaN, for a row that sees a key
          }
          if (i + 1 < e) {
            store8<XT, FMT>(s8, lds + (cur ^ 1) * 2 * TBYTES, tid);
            ks = block_scale(s8.ks), vs = block_scale(s8.vs);
          }
        }
        if (unit != 1.f) set_unit(1.f);
        if (tail) {
          const int64_t at = (int64_t)hb * (KBLK * KHD);
          const int rows = phi - full * KBLK + 1;
          __syncthreads();
          stage16(uniform(a.c8.kt + at), uniform(a.c8.vt + at), 0, rows - 1, KHD * 2u, lds0, wave,
                  lane);
          wait_loads();
          __syncthreads();
          attend16(lds, full * KBLK, true);
          if (bad)
            add_not_finite<XT>(acc, [&](int key) {
              return (const char*)(a.c8.vt + at) + key * (KHD * 2);
            }, rows, full * KBLK, p, h, a.w);
        }
      }
      if (mine) {
        const float l = acc.l + __shfl_xor(acc.l, 32);
        if (SHARED ? from > 0 || to < ct.n : a.S > 1) {
          const int64_t at = SHARED ? (2 * run + (from == 0)) * kTileRows + (r - r0)
                                    : ((int64_t)hb * a.R + r) * a.S + split;
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
    if constexpr (FMT == kPaged && !SHARED)
      if (a.zero && split == 0 && r < a.R && t >= sq.have) {
        u32* y = (u32*)(a.out + ctx_out(a, b, g, r)) + 32 * h;
        for (int i = 0; i < 32; ++i) y[i] = 0;
      }
    // tokens whose position is outside the cache (the merge writes them when there is one)
    if (!SHARED && a.S == 1 && r < a.R && t >= sq.fit && t < sq.have) {
      u32* y = (u32*)(a.out + ctx_out(a, b, g, r)) + 32 * h;
      for (int i = 0; i < 32; ++i) y[i] = (u32)Half<XT>::QNAN * 0x10001u;
    }
  } while (SHARED);
}

// The splits of rows merged: 32 P lanes a row, each dims 4 (t % 32) .. + 3 of every P-th
// part.  P = 8 (a workgroup a row) keeps many parts in flight at once; few parts take P = 1,
// eight rows a workgroup.
template <int XT, int P> __global__ __launch_bounds__(256) void k_ctx_merge(CtxArgs a, int64_t n) {
  __shared__ __align__(16) float s_o[8][KHD];
  __shared__ float s_m[8], s_l[8];
  const int tid = threadIdx.x, grp = tid >> 5, part = grp % P, d = 4 * (tid & 31);
  const int64_t at = (int64_t)blockIdx.x * (8 / P) + grp / P;  // (sequence, kv head, row)
  const bool here = at < n;
  const int64_t hb = here ? at / a.R : 0;
  const int r = here ? (int)(at % a.R) : 0, t = r / a.G, b = (int)(hb / a.nkv);
  const CtxSeq sq = ctx_seq(a, b);
  float M = -__builtin_inff(), L = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  if (here && t < sq.fit) {
    const float2* ml = (const float2*)a.ml + at * a.S;
    const float* src = a.part + at * a.S * KHD + d;
    constexpr int U = P == 1 ? 2 : 4;
    for (int s0 = part; s0 < a.S; s0 += U * P) {
      float2 v[U];
      f32x4 x[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int s = min(s0 + u * P, a.S - 1);
        v[u] = ml[s];
        x[u] = *(const f32x4*)(src + (int64_t)s * KHD);
        if (s0 + u * P >= a.S) v[u].y = 0.f;
      }
      float mb = M;  // a sum of 0: nothing seen there, no part written
#pragma unroll
      for (int u = 0; u < U; ++u) mb = v[u].y == 0.f ? mb : fmaxf(mb, v[u].x);
      const float f0 = M == mb ? 1.f : exp2f(M - mb);
      L *= f0;
      o *= f0;
      M = mb;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (v[u].y == 0.f) continue;
        const float f = exp2f(v[u].x - M);
        L = fmaf(v[u].y, f, L);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = fmaf(x[u][e], f, o[e]);
      }
    }
  }
  if constexpr (P > 1) {
    *(f32x4*)&s_o[grp][d] = o;
    if (d == 0) s_m[grp] = M, s_l[grp] = L;
    __syncthreads();
    M = -__builtin_inff(), L = 0.f, o = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int i = 0; i < P; ++i) M = s_l[i] == 0.f ? M : fmaxf(M, s_m[i]);
    for (int i = 0; i < P; ++i) {
      if (s_l[i] == 0.f) continue;
      const float f = exp2f(s_m[i] - M);
      L = fmaf(s_l[i], f, L);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = fmaf(s_o[i][d + e], f, o[e]);
    }
  }
  if (!here || t >= sq.have || part != 0) return;
  u32x2* y = (u32x2*)(a.out + ctx_out(a, b, (int)(hb % a.nkv), r) + d);
  if (t >= sq.fit) *y = u32x2{} + (u32)Half<XT>::QNAN * 0x10001u;
  else *y = u32x2{pack2<XT>(o[0] / L, o[1] / L), pack2<XT>(o[2] / L, o[3] / L)};
}

// The parts of row tiles that several runs share, and the rows of other tokens: eight
// rows a workgroup, a row to 32 lanes of 4 dims.
template <int XT> __global__ __launch_bounds__(256) void k_ctx_join(CtxArgs a) {
  const int M = a.B * a.tiles, g = blockIdx.y / M, m = blockIdx.y - g * M;
  const int b = m / a.tiles, rt = m - b * a.tiles, d = 4 * (threadIdx.x & 31);
  const int row = 8 * blockIdx.x + (threadIdx.x >> 5), r = rt * kTileRows + row, t = r / a.G;
  const CtxSeq sq = ctx_seq(a, b);
  if (r >= a.R) return;
  u32x2* y = (u32x2*)(a.out + ctx_out(a, b, g, r) + d);
  if (t >= sq.have) {
    if (a.zero) *y = u32x2{};
    return;
  }
  if (t >= sq.fit) {
    *y = u32x2{} + (u32)Half<XT>::QNAN * 0x10001u;
    return;
  }
  const int one = a.plan[M], begin = a.plan[m] + kRowTile, end = a.plan[m + 1];
  const Runs runs{(int64_t)one * a.nkv, a.plan[M + 1]};
  const int64_t u = (int64_t)g * one;
  const int w0 = runs.of(u + begin), w1 = runs.of(u + end - 1);
  if (w0 == w1) return;
  float top = -__builtin_inff(), L = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  constexpr int U = 4;
  for (int w = w0; w <= w1; w += U) {
    float2 v[U];
    f32x4 x[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int k = min(w + i, w1);
      const int64_t at = (int64_t)(2 * k + (k == w0)) * kTileRows + row;
      v[i] = ((const float2*)a.ml)[at];
      x[i] = *(const f32x4*)(a.part + at * KHD + d);
      if (w + i > w1) v[i].y = 0.f;
    }
    float mb = top;  // a sum of 0: nothing seen there, no part written
#pragma unroll
    for (int i = 0; i < U; ++i) mb = v[i].y == 0.f ? mb : fmaxf(mb, v[i].x);
    const float f0 = top == mb ? 1.f : exp2f(top - mb);
    L *= f0;
    o *= f0;
    top = mb;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (v[i].y == 0.f) continue;
      const float f = exp2f(v[i].x - top);
      L = fmaf(v[i].y, f, L);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = fmaf(x[i][e], f, o[e]);
    }
  }
  *y = u32x2{pack2<XT>(o[0] / L, o[1] / L), pack2<XT>(o[2] / L, o[3] / L)};
}

}  // namespace i4

int i4_launch_ctx_shared(const i4::CtxArgs& a, int xt, hipStream_t s) {
  using namespace i4;
  const dim3 join(kTileRows / 8, (unsigned)(a.B * a.tiles * a.nkv));
  if (xt == I4_F16) k_ctx_tile<I4_F16, kPaged, true><<<a.wgs, 256, 0, s>>>(a);
  else k_ctx_tile<I4_BF16, kPaged, true><<<a.wgs, 256, 0, s>>>(a);
  if (hipGetLastError() != hipSuccess) return I4_ERR_LAUNCH;
  if (xt == I4_F16) k_ctx_join<I4_F16><<<join, 256, 0, s>>>(a);
  else k_ctx_join<I4_BF16><<<join, 256, 0, s>>>(a);
  return hipGetLastError() == hipSuccess ? I4_OK : I4_ERR_LAUNCH;
}

static int launch_merge(const i4::CtxArgs& a, int xt, hipStream_t s) {
  const int64_t rows = (int64_t)a.B * a.nkv * a.R;
  const bool few = a.S <= 16;
  const dim3 grid((unsigned)(few ? (rows + 7) / 8 : rows));
  if (xt == I4_F16) {
    if (few) i4::k_ctx_merge<I4_F16, 1><<<grid, 256, 0, s>>>(a, rows);
    else i4::k_ctx_merge<I4_F16, 8><<<grid, 256, 0, s>>>(a, rows);
  } else {
    if (few) i4::k_ctx_merge<I4_BF16, 1><<<grid, 256, 0, s>>>(a, rows);
    else i4::k_ctx_merge<I4_BF16, 8><<<grid, 256, 0, s>>>(a, rows);
  }
  return hipGetLastError() == hipSuccess ? I4_OK : I4_ERR_LAUNCH;
}

int i4_launch_ctx_tile(const i4::CtxArgs& a, int xt, int fmt, hipStream_t s) {
  using namespace i4;
  const dim3 grid((unsigned)(a.tiles * a.S * a.B * a.nkv));
  auto go = [&](auto kern) { kern<<<grid, 256, 0, s>>>(a); };
  if (xt == I4_F16) {
    if (fmt == kDense) go(k_ctx_tile<I4_F16, kDense, false>);
    else if (fmt == kPaged) go(k_ctx_tile<I4_F16, kPaged, false>);
    else if (fmt == I4_KV8_INT8) go(k_ctx_tile<I4_F16, I4_KV8_INT8, false>);
    else go(k_ctx_tile<I4_F16, I4_KV8_E4M3, false>);
  } else {
    if (fmt == kDense) go(k_ctx_tile<I4_BF16, kDense, false>);
    else if (fmt == kPaged) go(k_ctx_tile<I4_BF16, kPaged, false>);
    else if (fmt == I4_KV8_INT8) go(k_ctx_tile<I4_BF16, I4_KV8_INT8, false>);
    else go(k_ctx_tile<I4_BF16, I4_KV8_E4M3, false>);
  }
  if (hipGetLastError() != hipSuccess) return I4_ERR_LAUNCH;
  return a.S > 1 ? launch_merge(a, xt, s) : I4_OK;
}
