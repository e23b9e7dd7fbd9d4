// Causal attention of each request's new tokens over its paged KV cache
// (gfx950, 16-bit data, fp32 sums).
//
// Both products run transposed, so that a query row is a lane's column:
// S^T [positions x rows] = K . q^T, then O^T [D x rows] = V^T . P^T.  An
// MFMA result lane holds one row's scores at four positions of a 16-position
// tile; K's rows are taken in an order that makes two such tiles eight
// neighbouring positions, which is the k chunk that the second product's
// operand needs.  So P goes from one product into the next in registers, the
// softmax's maximum and sum are a lane's own values joined over the four
// lanes of a column, and rescaling O is one multiplication a register.  Values
// lie transposed in the cache ([D, page]), so that a chunk of eight positions
// is one 16-byte load; a page is at least eight positions and a power of two.
//
// Masked places: their scores become -inf by selection, and where a tile has
// any, values that are not finite are left out of the product and added in
// for the rows that see them, so what lies behind a request's end or in a
// later token of the chunk reaches no row.
#include <type_traits>

#include "kernels.h"
#include "loads.h"
#include "paged.h"

namespace mlora {

namespace {

constexpr int kPos = 32;  // positions a wave takes at once

// All ones in the 16-bit halves of a word that are infinite or NaN.
template <class T>
__device__ __forceinline__ uint32_t nonfinite_mask(uint32_t w) {
  constexpr uint32_t E = std::is_same<T, BF16>::value ? 0x7f80u : 0x7c00u;
  uint32_t m = 0;
  if ((w & E) == E) m |= 0xffffu;
  if ((w & (E << 16)) == (E << 16)) m |= 0xffff0000u;
  return m;
}

template <int D, int NW, int MT>
struct StreamLds {
  float m[NW][MT * 16];
  float l[NW][MT * 16];
  // A wave's sums; the row padding spreads the transposed stores over the banks.
  float o[NW][MT * 16][D + 4];
};

// Workgroup = (item, key head).  Wave w of NW takes tiles w, w + NW, ... of
// 32 positions, straight from memory into MFMA operands; the waves meet in
// LDS at the end.
template <class T, int D, int NW, int MT>
__global__ __launch_bounds__(NW * 64) void paged_attn_kernel(PagedAttnArgs a) {
  using raw = typename T::raw_t;
  constexpr int KS = D / 32;  // k-steps of the scores
  constexpr int DT = D / 16;  // 16-row tiles of O^T
  constexpr int BM = MT * 16;
  __shared__ StreamLds<D, NW, MT> s;
  const int item = blockIdx.x / a.kv_heads;
  const int head = blockIdx.x - item * a.kv_heads;
  if (item >= a.plan[kApItems]) return;
  const int32_t* w = a.plan + a.shape.items_off + static_cast<int64_t>(item) * kApItemWords;
  const int req = w[0], row0 = w[1], kv0 = w[2], kv1 = w[3], slot = w[4];
  const int first = a.row_indptr[req];
  const int c = a.row_indptr[req + 1] - first;
  const int past = a.kv_lens[req] - c;  // position of the first new token
  const int rows = min(BM, c * a.rep - row0);
  if (rows <= 0) return;
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int col = lane & 15;
  const int g = lane >> 4;
  const int page = 1 << a.page_shift;
  const int32_t* table = a.table + static_cast<int64_t>(req) * a.table_stride;
  const raw* keys = static_cast<const raw*>(a.keys) + static_cast<int64_t>(head) * page * D;
  const raw* values = static_cast<const raw*>(a.values) + static_cast<int64_t>(head) * page * D;

  // q rows as MFMA columns, and the positions that each sees.
  u32x4 qf[MT][KS];
  int lim[MT];  // this lane's row sees positions [0, lim)
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int m = row0 + min(t * 16 + col, rows - 1);
    const int tok = m / a.rep;
    lim[t] = past + tok + 1;
    const raw* q = static_cast<const raw*>(a.q) + static_cast<int64_t>(first + tok) * a.q_stride +
                   static_cast<int64_t>(head * a.rep + (m - tok * a.rep)) * D;
#pragma unroll
    for (int k = 0; k < KS; ++k) qf[t][k] = ld_chunk(q + k * 32 + g * 8);
  }
  const int open = past + row0 / a.rep + 1;  // every row of the tile sees [0, open)

  f32x4 acc[MT][DT];
  float mx[MT], sum[MT];
  bool bad[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    mx[t] = -INFINITY;
    sum[t] = 0.f;
    // A row whose own position the table has no place for.
    bad[t] = lim[t] > (static_cast<int64_t>(a.width) << a.page_shift);
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[t][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  const int ka = (col >> 2) * 8 + (col & 3);  // position of K row `col` of the first tile; the second's is 4 on
  for (int base = kv0 + wave * kPos; base < kv1; base += NW * kPos) {
    // Pages of the chunk of positions this lane loads keys and values of.
    // Chunks past the range read page 0 (their scores are masked).
    const int kp = base + ka, vp = base + g * 8;
    int kid = kp < kv1 ? table[min(kp >> a.page_shift, a.width - 1)] : 0;
    int vid = vp < kv1 ? table[min(vp >> a.page_shift, a.width - 1)] : 0;
    const bool missing = vid < 0 || vid >= a.num_pages;
    if (missing) vid = 0;
    if (kid < 0 || kid >= a.num_pages) kid = 0;
    const raw* kr = keys + static_cast<int64_t>(kid) * a.key_stride + static_cast<int64_t>(kp & (page - 1)) * D + g * 8;
    const raw* vr = values + static_cast<int64_t>(vid) * a.value_stride + static_cast<int64_t>(col) * page + (vp & (page - 1));
    u32x4 kf[2][KS], vf[DT];
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      kf[0][k] = ld_chunk(kr + k * 32);
      kf[1][k] = ld_chunk(kr + 4 * D + k * 32);
    }
#pragma unroll
    for (int d = 0; d < DT; ++d) vf[d] = ld_chunk(vr + static_cast<int64_t>(d) * 16 * page);
    const bool masked = base + kPos > min(open, kv1);  // wave-uniform
    bool any_odd = false;  // a value of the tile is not finite
    if (masked) {
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t nf = nonfinite_mask<T>(vf[d][i]);
          vf[d][i] &= ~nf;
          any_odd |= nf != 0;
        }
      any_odd = __ballot(any_odd) != 0;
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      f32x4 sc[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        sc[0] = T::mma(sc[0], kf[0][k], qf[t][k]);
        sc[1] = T::mma(sc[1], kf[1][k], qf[t][k]);
      }
      // Lane (col, g): positions base + 8 g + i of row t * 16 + col.
      float p[8];
      const int seen = min(lim[t], kv1) - (base + g * 8);
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        p[i] = sc[i >> 2][i & 3] * a.scale_log2;
        if (masked && i >= seen) p[i] = -INFINITY;
        top = fmaxf(top, p[i]);
      }
      bad[t] |= missing && seen > 0;
      top = fmaxf(top, __shfl_xor(top, 16, kWave));
      top = fmaxf(top, __shfl_xor(top, 32, kWave));
      const float now = fmaxf(mx[t], top);
      const float ref = now == -INFINITY ? 0.f : now;  // nothing seen yet: every term below is 0
      const float keep = exp2f(mx[t] - ref);
      mx[t] = now;
      float add = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        p[i] = exp2f(p[i] - ref);
        add += p[i];
      }
      sum[t] = sum[t] * keep + add;  // this lane's positions; joined over the column at the end
      u32x4 pf;
#pragma unroll
      for (int i = 0; i < 4; ++i) pf[i] = T::pack2(p[2 * i], p[2 * i + 1]);
#pragma unroll
      for (int d = 0; d < DT; ++d) {
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[t][d][i] *= keep;
        acc[t][d] = T::mma(acc[t][d], vf[d], pf);
      }
      if (any_odd) {
        // The values left out, for the rows that see them: position z of the
        // tile is in lane group z / 8; row 16 d + 4 g + i of V^T in its lane
        // 4 g + i.
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const u32x4 vd = ld_chunk(vr + static_cast<int64_t>(d) * 16 * page);
#pragma unroll 1
          for (int z = 0; z < kPos; ++z) {
            const int e = z & 7;
            const int from = (z >> 3) * 16;
            float pe = p[0];
#pragma unroll
            for (int i = 1; i < 8; ++i) pe = e == i ? p[i] : pe;
            pe = __shfl(pe, from + col, kWave);
            uint32_t word = vd[0];
#pragma unroll
            for (int i = 1; i < 4; ++i) word = (e >> 1) == i ? vd[i] : word;
            word &= nonfinite_mask<T>(word);
            const bool sees = base + z < min(lim[t], kv1);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t other = __shfl(word, from + g * 4 + i, kWave);
              const float v = T::to_f32(static_cast<raw>((e & 1) ? other >> 16 : other & 0xffffu));
              if (sees && v != 0.f) acc[t][d][i] += pe * v;
            }
          }
        }
      }
    }
  }

  // Columns: the four lanes of a row, then the waves.
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    sum[t] += __shfl_xor(sum[t], 16, kWave);
    sum[t] += __shfl_xor(sum[t], 32, kWave);
    int b = bad[t];
    b |= __shfl_xor(b, 16, kWave);
    b |= __shfl_xor(b, 32, kWave);
    if (g == 0) {
      s.m[wave][t * 16 + col] = mx[t];
      s.l[wave][t * 16 + col] = b ? NAN : sum[t];
    }
#pragma unroll
    for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4*>(&s.o[wave][t * 16 + col][d * 16 + g * 4]) = acc[t][d];
  }
  lds_barrier();
  constexpr int C = D / 4;  // chunks of four columns a row
  for (int i = threadIdx.x; i < BM * C; i += NW * 64) {
    const int r = i / C;
    const int d = (i - r * C) * 4;
    if (r >= rows) continue;
    float m = s.m[0][r];
#pragma unroll
    for (int v = 1; v < NW; ++v) m = fmaxf(m, s.m[v][r]);
    const float ref = m == -INFINITY ? 0.f : m;
    float l = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int v = 0; v < NW; ++v) {
      const float f = exp2f(s.m[v][r] - ref);
      l += s.l[v][r] * f;
      o += *reinterpret_cast<const f32x4*>(&s.o[v][r][d]) * f;
    }
    if (slot >= 0) {
      const int64_t at = (static_cast<int64_t>(slot) * a.kv_heads + head) * BM + r;
      *reinterpret_cast<f32x4*>(a.part + at * D + d) = o;
      if (d == 0) {
        a.ml[at * 2] = m;
        a.ml[at * 2 + 1] = l;
      }
      continue;
    }
    const int mr = row0 + r;
    const int tok = mr / a.rep;
    raw* out = static_cast<raw*>(a.out) + static_cast<int64_t>(first + tok) * a.out_stride +
               static_cast<int64_t>(head * a.rep + (mr - tok * a.rep)) * D + d;
    // Every row sees its own position, so a sum of 0 means scores of -inf only.
    const float inv = l == 0.f ? NAN : 1.f / l;
    uint2 y;
    y.x = T::pack2(o[0] * inv, o[1] * inv);
    y.y = T::pack2(o[2] * inv, o[3] * inv);
    *reinterpret_cast<uint2*>(out) = y;
  }
}

// The parts of a split tile: workgroup = (tile, key head), thread = four
// columns of a row.
template <class T, int D>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedAttnArgs a) {
  using raw = typename T::raw_t;
  constexpr int C = D / 4;
  const int join = blockIdx.x / a.kv_heads;
  const int head = blockIdx.x - join * a.kv_heads;
  if (join >= a.plan[kApJoins]) return;
  const int32_t* w = a.plan + a.shape.joins_off + static_cast<int64_t>(join) * kApJoinWords;
  const int req = w[0], row0 = w[1], slot0 = w[2], parts = w[3];
  const int bm = a.shape.bm;
  const int first = a.row_indptr[req];
  const int rows = min(bm, (a.row_indptr[req + 1] - first) * a.rep - row0);
  for (int i = threadIdx.x; i < rows * C; i += 256) {
    const int r = i / C;
    const int d = (i - r * C) * 4;
    const int64_t step = static_cast<int64_t>(a.kv_heads) * bm;
    const int64_t at = (static_cast<int64_t>(slot0) * a.kv_heads + head) * bm + r;
    float m = -INFINITY;
    for (int p = 0; p < parts; ++p) m = fmaxf(m, a.ml[(at + p * step) * 2]);
    const float ref = m == -INFINITY ? 0.f : m;
    float l = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int p = 0; p < parts; ++p) {
      const float f = exp2f(a.ml[(at + p * step) * 2] - ref);
      l += a.ml[(at + p * step) * 2 + 1] * f;
      o += *reinterpret_cast<const f32x4*>(a.part + (at + p * step) * D + d) * f;
    }
    const int mr = row0 + r;
    const int tok = mr / a.rep;
    raw* out = static_cast<raw*>(a.out) + static_cast<int64_t>(first + tok) * a.out_stride +
               static_cast<int64_t>(head * a.rep + (mr - tok * a.rep)) * D + d;
    const float inv = l == 0.f ? NAN : 1.f / l;
    uint2 y;
    y.x = T::pack2(o[0] * inv, o[1] * inv);
    y.y = T::pack2(o[2] * inv, o[3] * inv);
    *reinterpret_cast<uint2*>(out) = y;
  }
}

template <class T, int D>
hipError_t launch(const PagedAttnArgs& a, hipStream_t stream) {
  const int64_t blocks = static_cast<int64_t>(a.shape.item_cap) * a.kv_heads;
  if (!grid_fits(blocks)) return hipErrorInvalidConfiguration;
  hipLaunchKernelGGL((paged_attn_kernel<T, D, 4, 1>), dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.shape.join_cap == 0) return e;
  hipLaunchKernelGGL((paged_join_kernel<T, D>), dim3(static_cast<unsigned>(a.shape.join_cap * a.kv_heads)), dim3(256), 0,
                     stream, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_paged_attention(const PagedAttnArgs& a, int dtype, int head_dim, hipStream_t stream) {
  if (a.shape.item_cap == 0) return hipSuccess;
  if (dtype == MLORA_BF16) return head_dim == 64 ? launch<BF16, 64>(a, stream) : launch<BF16, 128>(a, stream);
  return head_dim == 64 ? launch<F16, 64>(a, stream) : launch<F16, 128>(a, stream);
}

}  // namespace mlora
