// Rows of the fused q|k|v projection into a cache in pages: RMSNorm of the queries and keys (if
// the model has it), rotary embedding, and keys and values to the rows of their positions'
// pages.  fp32 inside, rounded once.  Bound by the rows' bytes: 5001 tokens of 40 heads take
// 19.2 us (5.3 TB/s), those of 24 sessions 3.9, which is latency.  A workgroup takes one token
// (several share its heads where tokens are few): its angles are computed once; a head is 16
// lanes of 8 dims, so that a half pair's other dim is in a lane pairs / 8 away (8 for a whole
// head: half a DPP row), and a neighbour's is in the same lane.
#include "i4_rotary.h"

namespace i4 {

// How the 8 dims of a lane turn: whole heads in halves, parts in halves, neighbours.
enum { kWhole, kPart, kNext };

struct PagedAppend {
  const uint16_t* qkv;
  int64_t bs, ts;
  const uint16_t *qw, *kw;  // nullable
  uint16_t* q_out;
  Pages pg;
  Tokens tk;
  Turn turn;
  int32_t nq, nkv;
  int32_t zero;  // whether the padding's rows are set to zero
  float eps;
};

template <int XT, int FORM>
__global__ __launch_bounds__(256) void k_paged_append(PagedAppend a, RotaryTable<KHD / 2> rt) {
  __shared__ __align__(16) float s_c[KHD / 2], s_s[KHD / 2];
  const int b = blockIdx.x / a.tk.T, t = blockIdx.x % a.tk.T;
  const bool have = t < count_of(a.tk, b);
  if (!have && !a.zero) return;
  const int heads = a.nq + 2 * a.nkv, lane = threadIdx.x & 15, step = 16 * gridDim.y;
  int h = 16 * blockIdx.y + (threadIdx.x >> 4);
  // on their way while the position, then its page are looked up and the angles computed
  const u32x4* x_row = (const u32x4*)(a.qkv + b * a.bs + t * a.ts) + lane;
  u32x4 raw = have && h < heads ? x_row[h * (KHD / 8)] : u32x4{};
  const u32x4 qn = a.qw ? ((const u32x4*)a.qw)[lane] : u32x4{};
  const u32x4 kn = a.kw ? ((const u32x4*)a.kw)[lane] : u32x4{};
  const int p0 = first_pos(a.tk, b), len = a.pg.table_len << a.pg.shift;
  // p0 is checked before t is added: a device position may be anything
  bool ok = p0 >= 0 && p0 < len && t < len - p0;
  const int p = ok ? p0 + t : 0;
  const PageRows slot = page_rows(a.pg, a.pg.table + b * a.pg.ts, 0, p);
  ok = ok && !slot.bad && turns(a.turn, b, t, p);
  u32x4* q_row = (u32x4*)(a.q_out + (int64_t)blockIdx.x * a.nq * KHD) + lane;
  if (!ok || !have) {
    const u32 fill = have ? (u32)Half<XT>::QNAN * 0x10001u : 0u;
    for (; h < a.nq; h += step) q_row[h * (KHD / 8)] = u32x4{} + fill;
    return;
  }
  const int n = rt.n;
  if (threadIdx.x < KHD / 2) {
    const int i = threadIdx.x;
    float c = 1.f, s = 0.f;
    if (i < n) {
      angle_of(turn_pos(a.turn, rt.axis[i], b, t, p), rt.f[i], c, s);
      c *= rt.factor;
      s *= rt.factor;
    }
    s_c[i] = c;
    s_s[i] = s;
  }
  __syncthreads();
  // the lane's first pair, whether its dims turn, and the lane with their other dims
  const int half = n >> 3;
  const bool low = lane < half;
  const int i0 = FORM == kNext ? 4 * lane : FORM == kWhole ? 8 * (lane & 7)
                                                           : 8 * (low ? lane : lane - half);
  const bool turn = FORM != kPart || lane < 2 * half;
  const int other = (threadIdx.x & 48) | (low ? lane + half : lane - half);
  constexpr int NP = FORM == kNext ? 4 : 8;
  float cs[NP], sn[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int j = (FORM == kPart && !turn) ? 0 : i0 + i;
    cs[i] = s_c[j];
    sn[i] = FORM != kNext && low ? -s_s[j] : s_s[j];
  }
  for (; h < heads; h += step) {
    const u32x4 next = h + step < heads ? x_row[(h + step) * (KHD / 8)] : u32x4{};
    u32x4 out = raw;
    if (h < a.nq + a.nkv) {
      const bool norm = h < a.nq ? a.qw != nullptr : a.kw != nullptr;
      const u32x4 w = h < a.nq ? qn : kn;
      float x[8], y[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[2 * i] = Half<XT>::to_f32((uint16_t)raw[i]);
        x[2 * i + 1] = Half<XT>::to_f32((uint16_t)(raw[i] >> 16));
      }
      if (norm) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) ss += x[2 * i] * x[2 * i] + x[2 * i + 1] * x[2 * i + 1];
        const float r = rsqrtf(group_sum<16>(ss) * (1.0f / KHD) + a.eps);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[2 * i] *= r * Half<XT>::to_f32((uint16_t)w[i]);
          x[2 * i + 1] *= r * Half<XT>::to_f32((uint16_t)(w[i] >> 16));
        }
      }
      if constexpr (FORM == kNext) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float u = x[2 * i], v = x[2 * i + 1];
          const bool in = i0 + i < n;
          y[2 * i] = in ? fmaf(u, cs[i], -(v * sn[i])) : u;
          y[2 * i + 1] = in ? fmaf(v, cs[i], u * sn[i]) : v;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float o = FORM == kWhole ? dpp_mov<0x128>(x[i]) : __shfl(x[i], other);
          y[i] = turn ? fmaf(x[i], cs[i], o * sn[i]) : x[i];
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) out[i] = pack2<XT>(y[2 * i], y[2 * i + 1]);
    }
    if (h < a.nq) {
      q_row[h * (KHD / 8)] = out;
    } else {
      const bool key = h < a.nq + a.nkv;
      char* c = (char*)(key ? a.pg.k : a.pg.v) + slot.at;
      *((u32x4*)(c + (h - a.nq - (key ? 0 : a.nkv)) * a.pg.hs) + lane) = out;
    }
    raw = next;
  }
}

}  // namespace i4

int i4_check_pagedcache(const i4_pagedcache* c) {
  if (!c || !c->k || !c->v || !c->table) return I4_ERR_NULL;
  if (c->dtype != I4_F16 && c->dtype != I4_BF16) return I4_ERR_DTYPE;
  if (c->head_dim != i4::KHD || c->batch < 1 || c->batch > 65535 || c->n_kv_heads < 1 ||
      c->n_kv_heads > 1024 || c->pages < 1 || c->page < 16 || c->page > 1024 ||
      (c->page & (c->page - 1)) || c->table_len < 1 ||
      c->table_len > i4::KV_MAX_LEN / c->page)
    return I4_ERR_SHAPE;
  const int64_t rows = (int64_t)c->page * i4::KHD, most = (int64_t)1 << 48;
  if ((c->pages > 1 && (c->page_stride < rows || c->page_stride > most / c->pages)) ||
      (c->n_kv_heads > 1 && (c->head_stride < rows || c->head_stride > most / c->n_kv_heads)) ||
      (c->batch > 1 && c->table_stride < c->table_len))
    return I4_ERR_STRIDE;
  if (((uintptr_t)c->k & 15) || ((uintptr_t)c->v & 15) || ((uintptr_t)c->table & 3) ||
      (c->page_stride & 7) || (c->head_stride & 7))
    return I4_ERR_ALIGN;
  if (!i4::blocks_apart(rows, c->pages, c->page_stride, c->n_kv_heads, c->head_stride))
    return I4_ERR_STRIDE;
  return I4_OK;
}

i4::Pages i4_pages_of(const i4_pagedcache* c) {
  auto step = [](int n, int64_t stride) { return n > 1 ? stride : 0; };
  return i4::Pages{(uint16_t*)c->k, (uint16_t*)c->v, c->table, 2 * step(c->pages, c->page_stride),
                   2 * step(c->n_kv_heads, c->head_stride), step(c->batch, c->table_stride),
                   c->pages, c->table_len, __builtin_ctz((unsigned)c->page)};
}

extern "C" int i4_paged_append(const void* qkv, int x_dtype, int T, int64_t batch_stride,
                               int64_t token_stride, int n_heads, const void* q_norm_w,
                               const void* k_norm_w, float eps, const i4_rotary* rotary,
                               const int32_t* pos_dev, int pos, const i4_turn* turn,
                               const int32_t* counts, int zero_padding, void* q_out,
                               const i4_pagedcache* cache, hipStream_t stream) {
  using namespace i4;
  if (!qkv || !q_out) return I4_ERR_NULL;
  int rc = i4_check_pagedcache(cache);
  if (!rc) rc = i4_check_rotary(rotary, turn);
  if (rc) return rc;
  if (x_dtype != cache->dtype) return I4_ERR_DTYPE;
  const int nkv = cache->n_kv_heads, B = cache->batch, n = rotary->pairs;
  rc = i4_check_tokens(B, T, n_heads, nkv, pos_dev, pos, counts, cache->table_len * cache->page);
  if (rc) return rc;
  if (n > KHD / 2 || (rotary->layout == I4_ROPE_HALF && n % 8)) return I4_ERR_SHAPE;
  if ((int64_t)B * T > kMaxGrid) return I4_ERR_SHAPE;
  const int64_t width = (int64_t)(n_heads + 2 * nkv) * KHD;
  if ((T > 1 && token_stride < width) || (B > 1 && batch_stride < width)) return I4_ERR_STRIDE;
  if (((uintptr_t)qkv & 15) || ((uintptr_t)q_norm_w & 15) || ((uintptr_t)k_norm_w & 15) ||
      ((uintptr_t)q_out & 15) || (token_stride & 7) || (batch_stride & 7))
    return I4_ERR_ALIGN;
  PagedAppend a{(const uint16_t*)qkv, batch_stride, token_stride, (const uint16_t*)q_norm_w,
                (const uint16_t*)k_norm_w, (uint16_t*)q_out, i4_pages_of(cache),
                Tokens{pos_dev, counts, pos, T}, turn_of(turn), n_heads, nkv, zero_padding, eps};
  const RotaryTable<KHD / 2> rt = rotary_table<KHD / 2>(rotary);
  // The heads of few tokens are shared out, 16 a workgroup at least, while the chip has room for
  // all workgroups at once (8 a CU).  Traced, over four sets of rows and pages: 24 tokens of 40
  // heads 3.9 us against 4.7 with one workgroup a token; 400 of 40 and 500 of 80 heads 4.9 and
  // 6.6 us against 5.5 and 8.1 with room for 512 workgroups, 1000 of 40 6.4 against 7.2 and 7.5
  // with room for 512 and 4096.
  const int heads = n_heads + 2 * nkv;
  int shares = 1;
  while (shares * 16 < heads && (int64_t)B * T * (shares + 1) <= 2048) ++shares;
  const dim3 grid((unsigned)(B * T), (unsigned)shares);
  auto go = [&](auto kern) { kern<<<grid, 256, 0, stream>>>(a, rt); };
  const bool f16 = x_dtype == I4_F16;
  if (rotary->layout == I4_ROPE_INTERLEAVED) {
    if (f16) go(k_paged_append<I4_F16, kNext>);
    else go(k_paged_append<I4_BF16, kNext>);
  } else if (n == KHD / 2) {
    if (f16) go(k_paged_append<I4_F16, kWhole>);
    else go(k_paged_append<I4_BF16, kWhole>);
  } else {
    if (f16) go(k_paged_append<I4_F16, kPart>);
    else go(k_paged_append<I4_BF16, kPart>);
  }
  return hipGetLastError() == hipSuccess ? I4_OK : I4_ERR_LAUNCH;
}
