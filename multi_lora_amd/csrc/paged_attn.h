// Causal attention of each request's new tokens over its paged KV cache
// (gfx950, 16-bit data, fp32 sums): the kernels, over pages of 16-bit numbers
// (paged_attn.hip) and of 8-bit codes (KV8; paged_attn8.hip).
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
// Roundings: the weights, for the second product, to the data type (half a
// step of each; their sum is taken before), the result once; scores, sums and
// rescaling are fp32.  (The decoder's q is rounded by the write before.  The
// matrix units take 16-bit operands only; the static cache's attention, which
// uses none, rounds neither.)
//
// Masked places: their scores become -inf by selection, and where a tile has
// any, values that are not finite are left out of the product and added in
// for the rows that see them, so what lies behind a request's end or in a
// later token of the chunk reaches no row.
//
// KV8: pages hold e4m3 codes, and each block of 16 positions of a key head an
// exponent, for keys and for values.  A code times its power of two is a number
// of the data type, so the operands are those of a 16-bit cache that holds the
// values which the codes stand for, and nothing else changes: the conversion
// instruction takes two codes and the scale.  (Against 64 bits, relative to the
// results' norm: 0.0019 to 0.0022 in bf16, where rounding the result alone gives
// 0.0016; the difference is the weights' rounding.)
#pragma once

#include <algorithm>
#include <type_traits>

#include "kernels.h"
#include "loads.h"
#include "paged.h"

namespace mlora {

namespace {

constexpr int kPos = 32;   // positions a wave takes at once
constexpr int kPos8 = 64;  // of 8-bit pages

typedef const __attribute__((address_space(1))) void gvoid_t;
typedef __attribute__((address_space(3))) void lvoid_t;

// All ones in the 16-bit halves of a word that are infinite or NaN.
template <class T>
__device__ __forceinline__ uint32_t nonfinite_mask(uint32_t w) {
  constexpr uint32_t E = std::is_same<T, BF16>::value ? 0x7f80u : 0x7c00u;
  uint32_t m = 0;
  if ((w & E) == E) m |= 0xffffu;
  if ((w & (E << 16)) == (E << 16)) m |= 0xffff0000u;
  return m;
}

// A zero the compiler does not know, made anew at each use: loads at an
// address that has it are not kept in registers over a rare loop.
__device__ __forceinline__ int opaque_zero() {
  int z = 0;
  asm volatile("" : "+s"(z));
  return z;
}

// Element e of a chunk if it is not finite, zeros elsewhere (e < 0: nowhere).
template <class T>
__device__ __forceinline__ u32x4 odd_values(u32x4 v, int e) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    v[i] &= (e >> 1) == i ? nonfinite_mask<T>(v[i]) & ((e & 1) ? 0xffff0000u : 0xffffu) : 0u;
  return v;
}

// Four codes as two words of the data type, times a power of two.
template <class T>
__device__ __forceinline__ uint2 widen4(uint32_t codes, float scale) {
  uint2 w;
  if constexpr (std::is_same<T, BF16>::value) {
    w.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, false));
    w.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, true));
  } else {
    w.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale, false));
    w.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale, true));
  }
  return w;
}
template <class T>
__device__ __forceinline__ u32x4 widen8(uint32_t lo, uint32_t hi, float scale) {
  const uint2 a = widen4<T>(lo, scale), b = widen4<T>(hi, scale);
  return u32x4{a.x, a.y, b.x, b.y};
}
// The power of two of an exponent byte.
__device__ __forceinline__ float scale_of(uint8_t e) { return __uint_as_float(static_cast<uint32_t>(e) << 23); }

// exp2 of what a softmax needs: arguments at most 0 (or NaN); results below
// the smallest normal number are 0.
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// An item of the plan, as every wave of its workgroup reads it.
struct Item {
  int req, row0, kv0, kv1, slot;
  int first, c, past;  // its request's first packed row, new tokens, and position of the first
  int rows;            // query rows of the tile, at most bm
};
__device__ __forceinline__ bool below(int v, int end) { return static_cast<uint32_t>(v) < static_cast<uint32_t>(end); }
__device__ __forceinline__ bool load_item(const PagedAttnArgs& a, const PagedKind& kd, int counter, int item, Item* t) {
  if (item >= min(a.plan[counter], kd.item_cap)) return false;
  const int32_t* w = a.plan + kd.items_off + static_cast<int64_t>(item) * kApItemWords;
  t->req = w[0], t->row0 = w[1], t->kv0 = w[2], t->kv1 = w[3], t->slot = w[4];
  t->first = w[5], t->c = w[6], t->past = w[7];
  // The list is the page tables' own, but a step can be used without one: the
  // launch that fills it may stand in a graph that has not run yet.  What does
  // not fit the call's bounds is skipped, and nothing outside them touched.
  const int room = static_cast<int>(min(static_cast<int64_t>(a.width) << a.page_shift, static_cast<int64_t>(1 << 30)));
  if (!below(t->req, a.n) || !below(t->c, a.rows + 1) || !below(t->first, a.rows - t->c + 1) || !below(t->past, 1 << 30) ||
      !below(t->row0, t->c * a.rep) || t->kv0 < 0 || (t->kv0 < t->kv1 && (t->kv0 & 63) != 0) || t->kv1 > room ||
      t->slot >= kd.slot_cap)
    return false;
  t->rows = min(kd.bm, t->c * a.rep - t->row0);
  return true;
}

// Element offset of query row m of a request inside q or out.
__device__ __forceinline__ int64_t row_offset(const PagedAttnArgs& a, const Item& t, int head, int m, int64_t stride, int d) {
  const int tok = m / a.rep;
  return static_cast<int64_t>(t.first + tok) * stride + static_cast<int64_t>(head * a.rep + (m - tok * a.rep)) * d;
}

// Four columns of a row's result.  Every row sees its own position, so a sum
// of 0 means scores of -inf only.
template <class T>
__device__ __forceinline__ void store_row(typename T::raw_t* out, f32x4 o, float l) {
  const float inv = l == 0.f ? NAN : 1.f / l;
  uint2 y;
  y.x = T::pack2(o[0] * inv, o[1] * inv);
  y.y = T::pack2(o[2] * inv, o[3] * inv);
  *reinterpret_cast<uint2*>(out) = y;
}

template <int D, int NW, int MT>
struct StreamLds {
  float m[NW][MT * 16];
  float l[NW][MT * 16];
  // A wave's sums; the row padding spreads the transposed stores over the banks.
  float o[NW][MT * 16][D + 4];
};

// The end of a short item: a row's sums of four lanes, then those of the waves.
template <class T, int D, int NW, int MT>
__device__ __forceinline__ void stream_meet(const PagedAttnArgs& a, StreamLds<D, NW, MT>& s, const Item& it, int head,
                                            const f32x4 (&acc)[MT][D / 16], const float (&mx)[MT], float (&sum)[MT],
                                            const bool (&bad)[MT]) {
  using raw = typename T::raw_t;
  constexpr int DT = D / 16;
  constexpr int BM = MT * 16;
  const int row0 = it.row0, rows = it.rows;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15;
  const int g = lane >> 4;
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
      const float f = exp2_fast(s.m[v][r] - ref);
      l += s.l[v][r] * f;
      o += *reinterpret_cast<const f32x4*>(&s.o[v][r][d]) * f;
    }
    if (it.slot >= 0) {
      const int64_t at = (static_cast<int64_t>(it.slot) * a.kv_heads + head) * BM + r;
      *reinterpret_cast<f32x4*>(reinterpret_cast<float*>(a.workspace + a.shape.kind[0].part_off) + at * D + d) = o;
      if (d == 0) *reinterpret_cast<float2*>(a.workspace + a.shape.kind[0].ml_off + at * 8) = make_float2(m, l);
    } else {
      store_row<T>(static_cast<raw*>(a.out) + row_offset(a, it, head, row0 + r, a.out_stride, D) + d, o, l);
    }
  }
}

// Short items: wave w of NW takes tiles w, w + NW, ... of 32 positions,
// straight from memory into MFMA operands; the waves meet in LDS at the end.
// Bound by the bytes of K and V, read once each: 64 decoding requests of 200
// to 3985 positions, 295 MB, 60.6 us on average (4.9 TB/s).  Few short ranges
// are bound by their chain: work list, page number, keys, values, meeting (4.7
// us for one request of 203 positions).
template <class T, int D, int NW, int MT>
__device__ __forceinline__ void stream_item(const PagedAttnArgs& a, StreamLds<D, NW, MT>& s, int item, int head) {
  using raw = typename T::raw_t;
  constexpr int KS = D / 32;  // k-steps of the scores
  constexpr int DT = D / 16;  // 16-row tiles of O^T
  Item it;
  if (!load_item(a, a.shape.kind[0], kApShort, item, &it)) return;
  const int row0 = it.row0, rows = it.rows, past = it.past, kv0 = it.kv0, kv1 = it.kv1;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15;
  const int g = lane >> 4;
  const int page = 1 << a.page_shift;
  const int32_t* table = a.table + static_cast<int64_t>(it.req) * a.table_stride;
  const raw* keys = static_cast<const raw*>(a.keys) + static_cast<int64_t>(head) * page * D;
  const raw* values = static_cast<const raw*>(a.values) + static_cast<int64_t>(head) * page * D;

  // q rows as MFMA columns, and the positions that each sees.
  u32x4 qf[MT][KS];
  int lim[MT];  // this lane's row sees positions [0, lim)
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int m = row0 + min(t * 16 + col, rows - 1);
    lim[t] = past + m / a.rep + 1;
    const raw* q = static_cast<const raw*>(a.q) + row_offset(a, it, head, m, a.q_stride, D);
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
  u32x4 kf[2][KS], vf[DT];
  // Pages of the chunks of positions that this lane loads keys and values of.
  // Chunks past the range read page 0 (their scores are masked).
  auto key_page = [&](int base) {
    const int p = base + ka;
    return p < kv1 ? table[min(p >> a.page_shift, a.width - 1)] : 0;
  };
  auto value_page = [&](int base) {
    const int p = base + g * 8;
    return p < kv1 ? table[min(p >> a.page_shift, a.width - 1)] : 0;
  };
  auto in_pool = [&](int id) { return static_cast<uint32_t>(id) < static_cast<uint32_t>(a.num_pages); };
  auto load_keys = [&](int base, int id) {
    const raw* k = keys + static_cast<int64_t>(in_pool(id) ? id : 0) * a.key_stride +
                   static_cast<int64_t>((base + ka) & (page - 1)) * D + g * 8;
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      kf[0][i] = ld_chunk(k + i * 32);
      kf[1][i] = ld_chunk(k + 4 * D + i * 32);
    }
  };
  auto value_rows = [&](int base, int id) {
    return values + static_cast<int64_t>(in_pool(id) ? id : 0) * a.value_stride + static_cast<int64_t>(col) * page +
           ((base + g * 8) & (page - 1));
  };
  auto load_values = [&](const raw* v) {
#pragma unroll
    for (int d = 0; d < DT; ++d) vf[d] = ld_chunk(v + static_cast<int64_t>(d) * 16 * page);
  };

  // Keys of the next tile are asked for as soon as this one's are used, values
  // likewise, so that each is in flight for half of a tile's work at least.
  int base = kv0 + wave * kPos;
  int kid = 0, vid = 0;
  const raw* vr = values;
  if (base < kv1) {
    kid = key_page(base);
    vid = value_page(base);
    load_keys(base, kid);
    vr = value_rows(base, vid);
    load_values(vr);
    kid = key_page(base + NW * kPos);
  }
  for (; base < kv1; base += NW * kPos) {
    const bool more = base + NW * kPos < kv1;
    const bool missing = !in_pool(vid);
    vid = value_page(base + NW * kPos);
    f32x4 sc[MT][2];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      sc[t][0] = sc[t][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        sc[t][0] = T::mma(sc[t][0], kf[0][k], qf[t][k]);
        sc[t][1] = T::mma(sc[t][1], kf[1][k], qf[t][k]);
      }
    }
    if (more) load_keys(base + NW * kPos, kid);
    kid = key_page(base + 2 * NW * kPos);
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
      // Lane (col, g): positions base + 8 g + i of row t * 16 + col.
      float p[8];
      const int seen = min(lim[t], kv1) - (base + g * 8);
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        p[i] = sc[t][i >> 2][i & 3] * a.scale_log2;
        if (masked && i >= seen) p[i] = -INFINITY;
        top = fmaxf(top, p[i]);
      }
      bad[t] |= missing && seen > 0;
      top = fmaxf(top, __shfl_xor(top, 16, kWave));
      top = fmaxf(top, __shfl_xor(top, 32, kWave));
      const float now = fmaxf(mx[t], top);
      const float ref = now == -INFINITY ? 0.f : now;  // nothing seen yet: every term below is 0
      const float keep = exp2_fast(mx[t] - ref);
      mx[t] = now;
      float add = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        p[i] = exp2_fast(p[i] - ref);
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
        // The values left out: one position's at a time, for the rows that see it.
#pragma unroll 1
        for (int z = 0; z < kPos; ++z) {
          const int again = opaque_zero();
          const bool sees = base + z < min(lim[t], kv1);
#pragma unroll
          for (int d = 0; d < DT; ++d) {
            const u32x4 v = odd_values<T>(ld_chunk(vr + again + static_cast<int64_t>(d) * 16 * page), (z >> 3) == g ? z & 7 : -1);
            if (__ballot((v[0] | v[1] | v[2] | v[3]) != 0) == 0) continue;
            const f32x4 part = T::mma(f32x4{0.f, 0.f, 0.f, 0.f}, v, pf);
            if (sees) acc[t][d] += part;
          }
        }
      }
    }
    if (more) {
      vr = value_rows(base + NW * kPos, vid);
      load_values(vr);
    }
  }

  stream_meet<T, D, NW, MT>(a, s, it, head, acc, mx, sum, bad);
}

// Short items over 8-bit pages: a wave takes 64 positions at once, so that a
// lane's 16 bytes of a row of V^T are one block of 16 positions, and its 16
// bytes of a key two steps of the first product.  Lane group g has the positions
// base + 16 g to base + 16 g + 15 of every row's scores: K rows are taken in an
// order that makes them neighbours, four of each of four MFMA tiles.  Bound by
// bytes, and nearly as much by conversions beside the products: 64 decoding
// requests (148 MB) 34.5 us, 4.3 TB/s, three of 8,192 to 32,001 positions (123
// MB) 26.0, 4.7; with waves of fewer registers, three a SIMD, 60 for the first.
template <class T, int D, int NW, int MT>
__device__ __forceinline__ void stream8_item(const PagedAttnArgs& a, StreamLds<D, NW, MT>& s, int item, int head) {
  using raw = typename T::raw_t;
  constexpr int KJ = D / 64;  // 16-byte chunks of a key that a lane loads, two k-steps of the scores each
  constexpr int DT = D / 16;  // 16-row tiles of O^T
  Item it;
  if (!load_item(a, a.shape.kind[0], kApShort, item, &it)) return;
  const int row0 = it.row0, rows = it.rows, past = it.past, kv0 = it.kv0, kv1 = it.kv1;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15;
  const int g = lane >> 4;
  const int page = 1 << a.page_shift;
  const int blocks_shift = a.page_shift - 4;  // blocks of a page
  const int32_t* table = a.table + static_cast<int64_t>(it.req) * a.table_stride;
  const uint8_t* keys = static_cast<const uint8_t*>(a.keys) + static_cast<int64_t>(head) * page * D;
  const uint8_t* values = static_cast<const uint8_t*>(a.values) + static_cast<int64_t>(head) * page * D;

  // q as operands; of two tiles in LDS, where it costs no registers: five tokens
  // for each of 32 requests 17.8 us against 20.4 with 15 of them spilled, for
  // each of 64 of 200 to 3985 positions 50.2 against 71.5.
  constexpr bool QL = MT > 1 && D == 128;
  __shared__ u32x4 q_lds[QL ? MT * 2 * KJ * kWave : 1];
  u32x4 qf[QL ? 1 : MT][2 * KJ];
  int lim[MT];  // this lane's row sees positions [0, lim)
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int m = row0 + min(t * 16 + col, rows - 1);
    lim[t] = past + m / a.rep + 1;
    const raw* q = static_cast<const raw*>(a.q) + row_offset(a, it, head, m, a.q_stride, D);
#pragma unroll
    for (int k = 0; k < 2 * KJ; ++k) {
      if constexpr (!QL) qf[t][k] = ld_chunk(q + (k >> 1) * 64 + g * 16 + (k & 1) * 8);
      else if ((t * 2 * KJ + k) % NW == wave) q_lds[(t * 2 * KJ + k) * kWave + lane] = ld_chunk(q + (k >> 1) * 64 + g * 16 + (k & 1) * 8);
    }
  }
  if constexpr (QL) lds_barrier();
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

  // K row `col` of tile z * 2 + u is position 16 (col >> 2) + 8 z + 4 u + (col & 3).
  const int kblock = col >> 2;
  u32x4 kf[4][KJ], vf[DT];
  uint8_t ks, vs;
  // Pages of the blocks that this lane loads keys and values of.  Blocks past
  // the range read page 0 (their scores are masked).
  auto page_of = [&](int p) { return p < kv1 ? table[min(p >> a.page_shift, a.width - 1)] : 0; };
  auto in_pool = [&](int id) { return static_cast<uint32_t>(id) < static_cast<uint32_t>(a.num_pages); };
  auto scale_at = [&](const uint8_t* scales, int id, int p) {
    return scales[((static_cast<int64_t>(id) * a.kv_heads + head) << blocks_shift) + ((p & (page - 1)) >> 4)];
  };
  auto load_keys = [&](int base, int id) {
    if (!in_pool(id)) id = 0;
    const int p = base + kblock * 16;
    ks = scale_at(a.key_scales, id, p);
    const uint8_t* k = keys + static_cast<int64_t>(id) * a.key_stride + static_cast<int64_t>((p & (page - 1)) + (col & 3)) * D + g * 16;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int j = 0; j < KJ; ++j) kf[t][j] = ld_chunk(k + t * 4 * D + j * 64);
  };
  auto load_values = [&](int base, int id) {
    if (!in_pool(id)) id = 0;
    const int p = base + g * 16;
    vs = scale_at(a.value_scales, id, p);
    const uint8_t* v = values + static_cast<int64_t>(id) * a.value_stride + static_cast<int64_t>(col) * page + (p & (page - 1));
#pragma unroll
    for (int d = 0; d < DT; ++d) vf[d] = ld_chunk(v + static_cast<int64_t>(d) * 16 * page);
  };

  // Keys of the next step are asked for as soon as this one's are used, values
  // likewise, so that each is in flight for half of a step's work at least.
  int base = kv0 + wave * kPos8;
  int kid = 0, vid = 0;
  if (base < kv1) {
    kid = page_of(base + kblock * 16);
    vid = page_of(base + g * 16);
    load_keys(base, kid);
    load_values(base, vid);
    kid = page_of(base + NW * kPos8 + kblock * 16);
  }
  for (; base < kv1; base += NW * kPos8) {
    const bool more = base + NW * kPos8 < kv1;
    const bool missing = !in_pool(vid);
    vid = page_of(base + NW * kPos8 + g * 16);
    f32x4 sc[MT][4];
    const float kscale = scale_of(ks), vscale = scale_of(vs);
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int z = 0; z < 4; ++z) sc[t][z] = f32x4{0.f, 0.f, 0.f, 0.f};
    const u32x4* ql = q_lds + lane + (QL ? opaque_zero() : 0);
#pragma unroll
    for (int k = 0; k < 2 * KJ; ++k) {
      u32x4 qk[MT];
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        if constexpr (QL) qk[t] = ql[(t * 2 * KJ + k) * kWave];
        else qk[t] = qf[t][k];
      }
#pragma unroll
      for (int z = 0; z < 4; ++z) {
        const u32x4 w = kf[z][k >> 1];
        const u32x4 key = (k & 1) ? widen8<T>(w[2], w[3], kscale) : widen8<T>(w[0], w[1], kscale);
#pragma unroll
        for (int t = 0; t < MT; ++t) sc[t][z] = T::mma(sc[t][z], key, qk[t]);
      }
    }
    if (more) load_keys(base + NW * kPos8, kid);
    kid = page_of(base + 2 * NW * kPos8 + kblock * 16);
    const bool masked = base + kPos8 > min(open, kv1);  // wave-uniform
    float keep[MT];
    u32x4 pf[MT][2];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      // Lane (col, g): positions base + 16 g + i of row t * 16 + col.
      float p[16];
      const int seen = min(lim[t], kv1) - (base + g * 16);
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        p[i] = sc[t][i >> 2][i & 3] * a.scale_log2;
      }
      if (masked) {
        asm volatile("");  // (stays a branch)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (i >= seen) p[i] = -INFINITY;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, p[i]);
      bad[t] |= missing && seen > 0;
      top = fmaxf(top, __shfl_xor(top, 16, kWave));
      top = fmaxf(top, __shfl_xor(top, 32, kWave));
      const float now = fmaxf(mx[t], top);
      const float ref = now == -INFINITY ? 0.f : now;  // nothing seen yet: every term below is 0
      keep[t] = exp2_fast(mx[t] - ref);
      mx[t] = now;
      float add = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        p[i] = exp2_fast(p[i] - ref);
        add += p[i];
      }
      sum[t] = sum[t] * keep[t] + add;  // this lane's positions; joined over the column at the end
#pragma unroll
      for (int i = 0; i < 8; ++i) pf[t][i >> 2][i & 3] = T::pack2(p[2 * i], p[2 * i + 1]);
    }
    // Nothing of the hidden positions' handling between the products where none
    // is hidden: 64 requests of 200 to 3985 positions 39.1 us against 40.8 with
    // the handling done always, 39.4 with branches around it.  Two tiles have no
    // registers for a second copy (121 spills) and take the branches.
    if (MT == 1 && !masked) {
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const u32x4 lo = widen8<T>(vf[d][0], vf[d][1], vscale), hi = widen8<T>(vf[d][2], vf[d][3], vscale);
#pragma unroll
        for (int t = 0; t < MT; ++t) {
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[t][d][i] *= keep[t];
          acc[t][d] = T::mma(acc[t][d], lo, pf[t][0]);
          acc[t][d] = T::mma(acc[t][d], hi, pf[t][1]);
        }
      }
    } else {
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const u32x4 all[2] = {widen8<T>(vf[d][0], vf[d][1], vscale), widen8<T>(vf[d][2], vf[d][3], vscale)};
        u32x4 v[2] = {all[0], all[1]};
        bool odd = false;  // a value is not finite
        if (masked) {
          asm volatile("");  // (as above)
#pragma unroll
          for (int z = 0; z < 2; ++z)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t nf = nonfinite_mask<T>(all[z][i]);
              v[z][i] = all[z][i] & ~nf;
              odd |= nf != 0;
            }
        }
#pragma unroll
        for (int t = 0; t < MT; ++t) {
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[t][d][i] *= keep[t];
#pragma unroll
          for (int z = 0; z < 2; ++z) acc[t][d] = T::mma(acc[t][d], v[z], pf[t][z]);
        }
        if (!masked || __ballot(odd) == 0) continue;
        // The values left out: one position's at a time, for the rows that see it.
#pragma unroll
        for (int z = 0; z < 2; ++z) {
#pragma unroll 1
          for (int e = 0; e < 32; ++e) {
            const u32x4 one = odd_values<T>(all[z], (e >> 3) == g ? e & 7 : -1);
            if (__ballot((one[0] | one[1] | one[2] | one[3]) != 0) == 0) continue;
            const int at = base + (e >> 3) * 16 + z * 8 + (e & 7);
#pragma unroll
            for (int t = 0; t < MT; ++t) {
              const f32x4 part = T::mma(f32x4{0.f, 0.f, 0.f, 0.f}, one, pf[t][z]);
              if (at < min(lim[t], kv1)) acc[t][d] += part;
            }
          }
        }
      }
    }
    if (more) load_values(base + NW * kPos8, vid);
  }
  stream_meet<T, D, NW, MT>(a, s, it, head, acc, mx, sum, bad);
}

constexpr int kTile = 64;  // positions of a long item's step
// Chunks from one 1 KB block of a tile (what one load instruction of a wave
// fills) to the next.  With chunk p of a row at p ^ (two of the row's low bits)
// and blocks 64 bytes further apart than they are long, the 16 rows that a
// fragment load takes a chunk of lie in different banks, and all of a lane's
// addresses are two registers and constants.
constexpr int kBlock = 68;

// Long items: 128 rows, 32 a wave, over the same 64 positions; K and V^T of a
// step go straight into LDS, a step ahead, in one of two buffers.  Chunk p of
// a row lies at p ^ (row's low bits), which spreads a fragment's rows over the
// banks.  Bound by the matrix units and the exponentials beside them: 444
// GFLOP (chunks of 4096, 777 and 1301 tokens, 32 heads of 128) take 463 to 474
// us a call, 935 to 960 TFLOP/s, where a library product of 8192^3 has 1606 to
// 1634 in a long run and 1223 in its first calls (504 on average under the
// profiler, 468 at best).  The matrix units are busy in 44 % of the cycles, at
// 1.9 GHz under this load.
// Without the exponentials it takes 4 % less, without the loads 17 %, with half
// of the second product 12 %.
template <int D>
struct TileLds {
  u32x4 k[2][kTile * D / 8 / 64 * kBlock];  // [position][D / 8 chunks]
  u32x4 v[2][D * kTile / 8 / 64 * kBlock];  // [D][8 chunks of positions]
};
// Chunk index of (row, chunk) in a tile whose rows have CPR chunks.
template <int CPR>
__device__ __forceinline__ int swizzle(int row) { return CPR == 16 ? row & 3 : (row >> 1) & 3; }
template <int CPR>
__device__ __forceinline__ int chunk_at(int row, int chunk) {
  constexpr int R = 64 / CPR;  // rows a block
  return row / R * kBlock + (row & (R - 1)) * CPR + (chunk ^ swizzle<CPR>(row));
}

// The softmax's reference of a row is not its largest score so far but one
// against which no weight is above kOver: weights stay in the data type's range,
// and the sums are rescaled a few times a range instead of at every new maximum
// (whose search over raw scores costs as much as the exponentials' arguments).
constexpr float kOver = 256.f;
constexpr float kNoScore = -3.40282347e38f;  // a row's reference before it has seen a score: the lowest number

template <class T, int D, bool KV8>
__device__ __forceinline__ void tile_item(const PagedAttnArgs& a, TileLds<D>& s, int item, int head) {
  using raw = typename T::raw_t;
  constexpr int KS = D / 16;                     // k-steps of the scores
  constexpr int DT = D / 32;                     // 32-row tiles of O^T
  constexpr int NL = kTile * D / 8 / 256;        // instructions a wave loads each of K and V with
  constexpr int KC = D / 8;                      // chunks of a key
  Item it;
  if (!load_item(a, a.shape.kind[1], kApLong, item, &it)) return;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31;
  const int h = lane >> 5;
  const int page = 1 << a.page_shift;
  const int kv0 = it.kv0, kv1 = it.kv1;
  const int32_t* table = a.table + static_cast<int64_t>(it.req) * a.table_stride;

  // The wave's rows; a negative scale goes into q, so that the largest scaled
  // score is the scaled largest one.  A scale of 0 is the least normal number:
  // it makes scores 0 and leaves hidden ones at -inf.
  const float scale = a.scale_log2 == 0.f ? 1.17549435e-38f : fabsf(a.scale_log2);
  const uint32_t flip = a.scale_log2 < 0.f ? 0x80008000u : 0u;
  const int m = it.row0 + min(wave * 32 + col, it.rows - 1);
  const int lim = it.past + m / a.rep + 1;
  u32x4 qf[KS];
  {
    const raw* q = static_cast<const raw*>(a.q) + row_offset(a, it, head, m, a.q_stride, D) + h * 8;
#pragma unroll
    for (int k = 0; k < KS; ++k) qf[k] = ld_chunk(q + k * 16) ^ flip;
  }
  const bool live = wave * 32 < it.rows;
  // All of the wave's rows see [0, open), none sees past shut.
  const int open = min(it.past + (it.row0 + min(wave * 32, it.rows - 1)) / a.rep + 1, kv1);
  const int shut = min(it.past + (it.row0 + min(wave * 32 + 31, it.rows - 1)) / a.rep + 1, kv1);

  f32x16 acc[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[d][r] = 0.f;
  float ref = kNoScore, sum = 0.f;  // sum: of this lane's positions; the two lanes of a row share ref
  int broken = INT32_MAX;           // first position without a page in the pool

  // Lane l's page is that of position base + l of the step.
  auto load_ids = [&](int base) {
    const int p = base + lane;
    return p < kv1 ? table[min(p >> a.page_shift, a.width - 1)] : 0;
  };
  auto check_ids = [&](int ids, int base) {
    if (static_cast<uint32_t>(ids) >= static_cast<uint32_t>(a.num_pages)) {
      broken = min(broken, base + lane);
      ids = 0;
    }
    return static_cast<uint32_t>(ids);
  };
  // 16-bit pages.  An instruction of a wave fills 1 KB of a tile: K rows kr0 + j * 256 / KC,
  // V rows vr0 + j * 32, and chunk p of a row comes from chunk p ^ (row's low
  // bits), the same for every j.  Steps begin at multiples of 64 and pages are
  // powers of two, so a lane's place inside a page moves with the step's only.
  const int kr0 = wave * (64 / KC) + lane / KC;
  const int vr0 = wave * 8 + (lane >> 3);
  const int kc = (lane & (KC - 1)) ^ swizzle<KC>(kr0);
  const int vc = (lane & 7) ^ swizzle<8>(vr0);
  const char* kb = reinterpret_cast<const char*>(a.keys) + (static_cast<int64_t>(head) * page * D + kc * 8) * 2;
  const char* vb = reinterpret_cast<const char*>(a.values) +
                   ((static_cast<int64_t>(head) * D + vr0) * page + (vc * 8 & (page - 1))) * 2;
  const uint32_t kstep = static_cast<uint32_t>(a.key_stride * 2), vstep = static_cast<uint32_t>(a.value_stride * 2);
  auto load_tile = [&](int base, uint32_t ids, int buf) {
    const int in_page = base & (page - 1);
    const char* kp = kb + static_cast<int64_t>(in_page) * (D * 2);
#pragma unroll
    for (int j = 0; j < NL; ++j) {
      const int row = j * (256 / KC) + kr0;
      const uint32_t id = __shfl(ids, row, kWave);
      const char* p = kp + (row & (page - 1)) * (D * 2) + static_cast<uint64_t>(id) * kstep;
      __builtin_amdgcn_global_load_lds((gvoid_t*)p, (lvoid_t*)(&s.k[buf][(j * 4 + wave) * kBlock]), 16, 0, 0);
    }
    const char* vp = vb + in_page * 2 + static_cast<uint64_t>(static_cast<uint32_t>(__shfl(ids, vc * 8, kWave))) * vstep;
#pragma unroll
    for (int j = 0; j < NL; ++j)
      __builtin_amdgcn_global_load_lds((gvoid_t*)(vp + static_cast<int64_t>(j * 32 * 2) * page),
                                       (lvoid_t*)(&s.v[buf][(j * 4 + wave) * kBlock]), 16, 0, 0);
  };

  // 8-bit pages.  A thread loads chunks of 16 codes a step ahead of their use
  // and writes them to LDS as two chunks of the data type, so that the codes are
  // converted once a workgroup and not once a wave: chunks of 4096, 777 and 1301
  // tokens 471 to 493 us, 465 to 474 over 16-bit pages, which need no registers
  // on their way.  K chunk tid + 256 j is
  // chunk kc8 of row kr8 + j * 256 / (D / 16), V chunk tid + 256 j the block vb8
  // of 16 positions of row vr8 + 64 j.
  constexpr int N8 = kTile * D / 16 / 256;
  const int kr8 = tid / (D / 16), kc8 = tid & (D / 16 - 1);
  const int vr8 = tid >> 2, vb8 = tid & 3;
  const int blocks_shift = a.page_shift - 4;
  u32x4 kraw[KV8 ? N8 : 1], vraw[KV8 ? N8 : 1];
  uint8_t ksc[KV8 ? N8 : 1], vsc = 0;
  auto load8 = [&](int base, uint32_t ids) {
    const int in_page = base & (page - 1);
    const uint8_t* k8 = static_cast<const uint8_t*>(a.keys) + static_cast<int64_t>(head) * page * D + kc8 * 16;
    const uint8_t* v8 = static_cast<const uint8_t*>(a.values) + (static_cast<int64_t>(head) * D + vr8) * page;
#pragma unroll
    for (int j = 0; j < N8; ++j) {
      const int row = kr8 + j * (4096 / D);
      const int64_t id = static_cast<uint32_t>(__shfl(ids, row, kWave));
      const int p = (in_page + row) & (page - 1);
      kraw[j] = ld_chunk(k8 + id * a.key_stride + static_cast<int64_t>(p) * D);
      ksc[j] = a.key_scales[((id * a.kv_heads + head) << blocks_shift) + (p >> 4)];
    }
    const int64_t id = static_cast<uint32_t>(__shfl(ids, vb8 * 16, kWave));
    const int p = (in_page + vb8 * 16) & (page - 1);
#pragma unroll
    for (int j = 0; j < N8; ++j) vraw[j] = ld_chunk(v8 + id * a.value_stride + static_cast<int64_t>(j * 64) * page + p);
    vsc = a.value_scales[((id * a.kv_heads + head) << blocks_shift) + (p >> 4)];
  };
  auto widen = [&](int buf) {
#pragma unroll
    for (int j = 0; j < N8; ++j) {
      const int kr = kr8 + j * (4096 / D), vr = vr8 + j * 64;
      s.k[buf][chunk_at<KC>(kr, 2 * kc8)] = widen8<T>(kraw[j][0], kraw[j][1], scale_of(ksc[j]));
      s.k[buf][chunk_at<KC>(kr, 2 * kc8 + 1)] = widen8<T>(kraw[j][2], kraw[j][3], scale_of(ksc[j]));
      s.v[buf][chunk_at<8>(vr, 2 * vb8)] = widen8<T>(vraw[j][0], vraw[j][1], scale_of(vsc));
      s.v[buf][chunk_at<8>(vr, 2 * vb8 + 1)] = widen8<T>(vraw[j][2], vraw[j][3], scale_of(vsc));
    }
  };

  // Row rho of an MFMA tile is position rho with bits 2 and 3 exchanged: a
  // lane's registers 8 s + i are then positions 16 s + 8 h + i.
  const int krow = (col & ~12) | ((col & 4) << 1) | ((col & 8) >> 1);
  // Fragments: k-step k of positions 32 t + krow, and positions 32 t + 16 z of
  // V^T's rows 32 d + col.
  const int ka[2] = {chunk_at<KC>(krow, h), chunk_at<KC>(krow, 2 + h)};
  const int va[2] = {chunk_at<8>(col, h), chunk_at<8>(col, 2 + h)};
  auto k_frag = [&](int buf, int t, int k) { return s.k[buf][ka[k & 1] + t * (32 * KC / 64 * kBlock) + (k >> 1) * 4]; };
  auto v_frag = [&](int buf, int t, int z, int d) { return s.v[buf][va[z] + d * (4 * kBlock) + t * 4]; };
  auto step = [&](int base, int buf) {
    const bool masked = base + kTile > open;  // of the wave
    const int seen = min(lim, kv1) - base - h * 8;
    u32x4 kf[2][KS], vf[2][DT][2], pf[2];
    f32x16 p[2];  // of 32 positions each: scores, then weights
    float top;
    auto load_k = [&](int t) {
#pragma unroll
      for (int k = 0; k < KS; ++k) kf[t][k] = k_frag(buf, t, k);
    };
    auto load_v = [&](int t) {
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int z = 0; z < 2; ++z) vf[t][d][z] = v_frag(buf, t, z, d);
    };
    // S^T of 32 positions x 32 rows.
    auto scores = [&](int t) {
#pragma unroll
      for (int r = 0; r < 16; ++r) p[t][r] = 0.f;
#pragma unroll
      for (int k = 0; k < KS; ++k) p[t] = T::mma32(p[t], kf[t][k], qf[k]);
    };
    auto hide = [&](int t) {
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (t * 32 + (r >> 3) * 16 + (r & 7) >= seen) p[t][r] = -INFINITY;
    };
    auto weights = [&](int t) {
#pragma unroll
      for (int r = 0; r < 16; ++r) p[t][r] = exp2_fast(__builtin_fmaf(p[t][r], scale, -ref));
      top = 0.f;
#pragma unroll
      for (int r = 0; r < 16; r += 2) top = fmaxf(fmaxf(top, p[t][r]), p[t][r + 1]);
    };
    auto rescale = [&](int t) {
      // The scores again: the weights took their place.
#pragma unroll
      for (int r = 0; r < 16; ++r) p[t][r] = 0.f;
#pragma unroll
      for (int k = 0; k < KS; ++k) p[t] = T::mma32(p[t], k_frag(buf, t, k), qf[k]);
      if (masked) {
        asm volatile("");
        hide(t);
      }
      float now = p[t][0];
#pragma unroll
      for (int r = 1; r < 16; ++r) now = fmaxf(now, p[t][r]);
      now = fmaxf(now, __shfl_xor(now, 32, kWave)) * scale;
      now = fmaxf(now, ref);
      const float keep = exp2_fast(ref - now);
      ref = now;
      sum *= keep;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[d][r] *= keep;
#pragma unroll
      for (int r = 0; r < 16; ++r) p[t][r] = exp2_fast(__builtin_fmaf(p[t][r], scale, -ref));
    };
    auto pack = [&](int t) {
#pragma unroll
      for (int r = 0; r < 16; r += 2) pf[r >> 3][(r & 7) >> 1] = T::pack2(p[t][r], p[t][r + 1]);
    };
    auto add_up = [&](int t) {
#pragma unroll
      for (int r = 0; r < 16; r += 2) sum += p[t][r] + p[t][r + 1];
    };
    auto product = [&](int t) {
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int z = 0; z < 2; ++z) acc[d] = T::mma32(acc[d], vf[t][d][z], pf[z]);
    };
    auto drop_odd = [&](int t) {
      bool any = false;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int z = 0; z < 2; ++z)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t nf = nonfinite_mask<T>(vf[t][d][z][i]);
            any |= nf != 0;
            vf[t][d][z][i] &= ~nf;
          }
      return __ballot(any) != 0;
    };
    // The values left out: one position's at a time, for the rows that see it.
    auto add_odd = [&](int t) {
#pragma unroll
      for (int z = 0; z < 2; ++z)
#pragma unroll 1
        for (int e = 0; e < 16; ++e) {
          const int again = opaque_zero();
          const bool sees = base + t * 32 + z * 16 + e < min(lim, kv1);
#pragma unroll
          for (int d = 0; d < DT; ++d) {
            const u32x4 v = odd_values<T>(v_frag(buf, t + again, z, d), (e >> 3) == h ? e & 7 : -1);
            if (__ballot((v[0] | v[1] | v[2] | v[3]) != 0) == 0) continue;
            f32x16 part;
#pragma unroll
            for (int r = 0; r < 16; ++r) part[r] = 0.f;
            part = T::mma32(part, v, pf[z]);
            if (sees)
#pragma unroll
              for (int r = 0; r < 16; ++r) acc[d][r] += part[r];
          }
        }
    };
    bool odd = false;

    // The second half's scores come before the first half's weights, and the
    // first half's product before the second's weights: matrix and vector
    // instructions that do not wait for each other stand next to each other.
    load_k(0);
    load_k(1);
    scores(0);
    __builtin_amdgcn_sched_barrier(0);
    if (masked) {
      asm volatile("");
      hide(0);
    }
    load_v(0);
    scores(1);
    weights(0);
    __builtin_amdgcn_sched_barrier(0);
    if (__any(top > kOver)) rescale(0);
    if (masked) {
      asm volatile("");
      hide(1);
      odd = drop_odd(0);
    }
    pack(0);
    if (odd) add_odd(0);
    product(0);
    weights(1);
    add_up(0);
    load_v(1);
    __builtin_amdgcn_sched_barrier(0);
    if (__any(top > kOver)) rescale(1);
    if (masked) {
      asm volatile("");
      odd = drop_odd(1);
    }
    pack(1);
    if (odd) add_odd(1);
    product(1);
    add_up(1);
  };

  uint32_t ids = 0;
  if (kv0 < kv1) {
    ids = check_ids(load_ids(kv0), kv0);
    if constexpr (KV8) {
      load8(kv0, ids);
      widen(0);
      if (kv0 + kTile < kv1) {
        ids = load_ids(kv0 + kTile);
        load8(kv0 + kTile, check_ids(ids, kv0 + kTile));
      }
      ids = load_ids(kv0 + 2 * kTile);
    } else {
      load_tile(kv0, ids, 0);
      ids = load_ids(kv0 + kTile);
    }
  }
  int buf = 0;
  for (int base = kv0; base < kv1; base += kTile, buf ^= 1) {
    if constexpr (KV8) {
      lds_barrier();  // everyone's part of the step is in LDS, and nobody reads the other buffer
      if (base + kTile < kv1) {
        widen(buf ^ 1);
        if (base + 2 * kTile < kv1) {
          load8(base + 2 * kTile, check_ids(ids, base + 2 * kTile));
          ids = load_ids(base + 3 * kTile);
        }
      }
    } else {
      wait_vmcnt<0>();  // this wave's part of the step has landed
      lds_barrier();    // everyone's has, and nobody reads the other buffer
      if (base + kTile < kv1) {
        load_tile(base + kTile, check_ids(ids, base + kTile), buf ^ 1);
        ids = load_ids(base + 2 * kTile);
      }
    }
    __builtin_amdgcn_sched_barrier(0);  // the next step's loads go out before this one's products
    if (live && base < shut) step(base, buf);
  }

  sum += __shfl_xor(sum, 32, kWave);
  for (int off = 1; off < kWave; off <<= 1) broken = min(broken, __shfl_xor(broken, off, kWave));
  if (broken < lim || lim > (static_cast<int64_t>(a.width) << a.page_shift)) sum = NAN;
  const int r0 = wave * 32 + col;
  if (r0 >= it.rows) return;
  if (it.slot >= 0) {
    const int64_t at = (static_cast<int64_t>(it.slot) * a.kv_heads + head) * kApLongRows + r0;
    float* part = reinterpret_cast<float*>(a.workspace + a.shape.kind[1].part_off) + at * D + h * 4;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int r = 0; r < 16; r += 4)
        *reinterpret_cast<f32x4*>(part + d * 32 + r * 2) = f32x4{acc[d][r], acc[d][r + 1], acc[d][r + 2], acc[d][r + 3]};
    if (h == 0)
      *reinterpret_cast<float2*>(a.workspace + a.shape.kind[1].ml_off + at * 8) = make_float2(ref == kNoScore ? -INFINITY : ref, sum);
  } else {
    raw* out = static_cast<raw*>(a.out) + row_offset(a, it, head, m, a.out_stride, D) + h * 4;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int r = 0; r < 16; r += 4)
        store_row<T>(out + d * 32 + r * 2, f32x4{acc[d][r], acc[d][r + 1], acc[d][r + 2], acc[d][r + 3]}, sum);
  }
}

template <class T, int D, int NW, int MT, bool KV8>
__global__ __launch_bounds__(NW * 64, 2) void paged_short_kernel(PagedAttnArgs a) {
  __shared__ StreamLds<D, NW, MT> s;
  const int item = blockIdx.x / a.kv_heads;
  if constexpr (KV8) stream8_item<T, D, NW, MT>(a, s, item, blockIdx.x - item * a.kv_heads);
  else stream_item<T, D, NW, MT>(a, s, item, blockIdx.x - item * a.kv_heads);
}

// Long items first, then the short ones, which fill the chip as those end, and
// last the workgroups that the host's bounds ask for and the step does not
// need (between the two kinds: 139 us instead of 136 for a prompt of 2048
// tokens beside 128 decoding requests, 114 instead of 99 with four times as
// many of them).  Both kinds in turn from the start: four prompts of 1024
// beside 128 requests 138 us against 157, but 344 against 288 for 2048 tokens
// after 4096 beside 64 requests, whose last long items then start late.  (Over
// 8-bit pages with D 128 five of its 256 registers are spilled.)
template <class T, int D, bool KV8>
__global__ __launch_bounds__(256, 2) void paged_mixed_kernel(PagedAttnArgs a) {
  __shared__ union {
    TileLds<D> tile;
    StreamLds<D, 4, 1> stream;
  } s;
  const int item = blockIdx.x / a.kv_heads;
  const int head = blockIdx.x - item * a.kv_heads;
  const int long_items = max(min(a.plan[kApLong], a.shape.kind[1].item_cap), 0);
  if (item < long_items)
    tile_item<T, D, KV8>(a, s.tile, item, head);
  else if constexpr (KV8)
    stream8_item<T, D, 4, 1>(a, s.stream, item - long_items, head);
  else
    stream_item<T, D, 4, 1>(a, s.stream, item - long_items, head);
}

// The parts of a split tile: workgroup = (tile, key head, block of RB rows),
// thread = four columns of a row.  Short tiles have few rows and up to a
// hundred parts, so the threads left over share the parts (G groups); long
// ones the other way round.  One thread a column group over 34 parts took
// 24 us (three requests of up to 32,000 positions), four 6.7.
template <class T, int D, int RB>
__device__ __forceinline__ void join_rows(const PagedAttnArgs& a, int k, int join, int head, int block, f32x4* os) {
  using raw = typename T::raw_t;
  constexpr int C = D / 4;
  constexpr int G = 256 / (RB * C);
  const PagedKind kd = k ? a.shape.kind[1] : a.shape.kind[0];
  const int32_t* w = a.plan + kd.joins_off + static_cast<int64_t>(join) * kApJoinWords;
  const int slot0 = w[2], parts = w[3];
  Item it;
  it.first = w[0], it.row0 = w[1], it.rows = w[4];
  if (!below(it.rows, kd.bm + 1) || block * RB >= it.rows) return;
  // As in load_item.
  if (!below(it.first, a.rows) || !below(it.row0, 1 << 30) || (it.row0 + it.rows - 1) / a.rep >= a.rows - it.first ||
      !below(parts - 1, kd.slot_cap) || !below(slot0, kd.slot_cap - parts + 1))
    return;
  const int group = threadIdx.x / (RB * C);
  const int i = threadIdx.x - group * (RB * C);
  const int r = min(block * RB + i / C, it.rows - 1);
  const int d = (i & (C - 1)) * 4;
  const int64_t step = static_cast<int64_t>(a.kv_heads) * kd.bm;
  const int64_t at = (static_cast<int64_t>(slot0) * a.kv_heads + head) * kd.bm + r;
  const float* part = reinterpret_cast<const float*>(a.workspace + kd.part_off) + at * D + d;
  const float2* ml = reinterpret_cast<const float2*>(a.workspace + kd.ml_off) + at;
  // The C lanes of a row look at C parts' maxima and sums at once.
  static_assert(RB * C % kWave == 0, "a wave's lanes share the parts they add");
  const int lane = i & (C - 1);
  float m = -INFINITY;
  for (int p = lane; p < parts; p += C) m = fmaxf(m, ml[p * step].x);
#pragma unroll
  for (int off = 1; off < C; off <<= 1) m = fmaxf(m, __shfl_xor(m, off, kWave));
  const float ref = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int p0 = 0; p0 < parts; p0 += C) {
    const float2 x = p0 + lane < parts ? ml[(p0 + lane) * step] : make_float2(-INFINITY, 0.f);
    const float f = exp2_fast(x.x - ref);
    l += x.y * f;
    const int here = min(C, parts - p0);
#pragma unroll 4
    for (int p = group; p < here; p += G)
      o += *reinterpret_cast<const f32x4*>(part + (p0 + p) * step * D) * __shfl(f, (threadIdx.x & 63 & ~(C - 1)) + p, kWave);
  }
#pragma unroll
  for (int off = 1; off < C; off <<= 1) l += __shfl_xor(l, off, kWave);
  if constexpr (G > 1) {
    os[threadIdx.x] = o;
    lds_barrier();
    if (group > 0) return;
#pragma unroll
    for (int v = 1; v < G; ++v) o += os[v * RB * C + i];
  }
  if (block * RB + i / C >= it.rows) return;
  store_row<T>(static_cast<raw*>(a.out) + row_offset(a, it, head, it.row0 + r, a.out_stride, D) + d, o, l);
}

constexpr int kJoinGrid = 2048;  // eight workgroups a CU
constexpr int join_block(int d, int kind) { return kind ? 1024 / d : 256 / d; }  // rows: 8 or 2 of 128 columns

// Workgroups take the row blocks in turn: the host's bound on them is many
// times what most steps have, and starting that many idle ones cost 10 us.
template <class T, int D>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedAttnArgs a, int long_per) {
  __shared__ f32x4 os[256];
  const PagedKind &few = a.shape.kind[0], &many = a.shape.kind[1];
  const int short_per = cdiv(max(min(a.plan[kApJoinRows], few.bm), 0), join_block(D, 0));
  const int long_blocks = max(min(a.plan[kApLong + 1], many.join_cap), 0) * a.kv_heads * long_per;
  const int blocks = long_blocks + max(min(a.plan[kApShort + 1], few.join_cap), 0) * a.kv_heads * short_per;
  for (int u = blockIdx.x; u < blocks; u += gridDim.x) {
    if (u < long_blocks) {
      const int tile = u / long_per;
      const int join = tile / a.kv_heads;
      join_rows<T, D, join_block(D, 1)>(a, 1, join, tile - join * a.kv_heads, u - tile * long_per, os);
    } else {
      const int tile = (u - long_blocks) / short_per;
      const int join = tile / a.kv_heads;
      join_rows<T, D, join_block(D, 0)>(a, 0, join, tile - join * a.kv_heads, u - long_blocks - tile * short_per, os);
      lds_barrier();  // before the next block's sums go where these were read
    }
  }
}

template <class T, int D, bool KV8>
hipError_t launch(const PagedAttnArgs& a, int max_rows, hipStream_t stream) {
  const PagedKind &few = a.shape.kind[0], &many = a.shape.kind[1];
  const int64_t blocks = (static_cast<int64_t>(few.item_cap) + many.item_cap) * a.kv_heads;
  // Row blocks of a tile that hold rows at all.
  const int long_per = cdiv(std::min(many.bm, max_rows), join_block(D, 1));
  const int64_t joins = static_cast<int64_t>(many.join_cap) * a.kv_heads * long_per +
                        static_cast<int64_t>(few.join_cap) * a.kv_heads * cdiv(std::min(few.bm, max_rows), join_block(D, 0));
  if (!grid_fits(blocks) || !grid_fits(joins)) return hipErrorInvalidConfiguration;
  const dim3 grid(static_cast<unsigned>(blocks));
  if (many.item_cap > 0)
    hipLaunchKernelGGL((paged_mixed_kernel<T, D, KV8>), grid, dim3(256), 0, stream, a);
  else if (few.bm == 16)
    hipLaunchKernelGGL((paged_short_kernel<T, D, 4, 1, KV8>), grid, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((paged_short_kernel<T, D, 4, 2, KV8>), grid, dim3(256), 0, stream, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || joins == 0) return e;
  hipLaunchKernelGGL((paged_join_kernel<T, D>), dim3(static_cast<unsigned>(std::min<int64_t>(joins, kJoinGrid))), dim3(256), 0,
                     stream, a, long_per);
  return hipGetLastError();
}

template <bool KV8>
hipError_t launch_of(const PagedAttnArgs& a, int max_new, int dtype, int head_dim, hipStream_t stream) {
  if (a.shape.kind[0].item_cap + a.shape.kind[1].item_cap == 0) return hipSuccess;
  const int max_rows = std::min(max_new, kApLongRows) * a.rep;  // of one request, as far as it matters
  if (dtype == MLORA_BF16)
    return head_dim == 64 ? launch<BF16, 64, KV8>(a, max_rows, stream) : launch<BF16, 128, KV8>(a, max_rows, stream);
  return head_dim == 64 ? launch<F16, 64, KV8>(a, max_rows, stream) : launch<F16, 128, KV8>(a, max_rows, stream);
}

}  // namespace
}  // namespace mlora
