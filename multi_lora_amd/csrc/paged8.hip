// The write of new rows into a paged KV cache of 8-bit codes (gfx950).
//
// A block is 16 neighbouring positions of a page and one key head; its e4m3
// codes (4 exponent and 3 mantissa bits, largest number 448) share a power of
// two, 2^e, for keys and another for values.  With m the largest magnitude of
// the block's new rows, e is the least exponent with m <= 448 * 2^e, or the
// block's own where that is larger and earlier rows are in it.  If it grows, the
// earlier rows' codes are rounded again: their exponents move, so only numbers
// that come to lie below the least normal one (2^-6 * 2^e, a 2^-14 of the
// block's largest) can change.  A power of two also makes a code times its scale
// a number of the data type, which is what attention multiplies with; so e is
// kept in the range for which that holds.
//
// Infinities and NaN become NaN codes and are not counted in m.
#include <type_traits>

#include "kernels.h"
#include "loads.h"
#include "paged.h"

namespace mlora {

namespace {

// Range of the exponents, so that codes * 2^e is exact in the data type: its
// least multiple is 2^(e - 9), its largest 448 * 2^e, or 240 * 2^e at the top,
// where the next code would be infinite.
template <class T>
struct ScaleRange {
  static constexpr int lo = std::is_same<T, BF16>::value ? -117 : -15;
  static constexpr int hi = std::is_same<T, BF16>::value ? 120 : 8;
  // Numbers from here on are infinite in the data type.
  static constexpr float end = std::is_same<T, BF16>::value ? INFINITY : 65520.f;
};

// |x| as an integer, 0 for what is not a number of the data type.
template <class T>
__device__ __forceinline__ uint32_t counted(float x) {
  const float a = fabsf(x);
  return a < ScaleRange<T>::end ? __float_as_uint(a) : 0u;
}

// Least e with m <= 448 * 2^e (448 = 1.75 * 2^8), from m's bits.
template <class T>
__device__ __forceinline__ int exponent_of(uint32_t bits) {
  const int e = static_cast<int>(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(e, ScaleRange<T>::lo), ScaleRange<T>::hi);
}

__device__ __forceinline__ float pow2(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// Four numbers as codes of the exponent, `inv` = 2^-e.
template <class T>
__device__ __forceinline__ uint32_t codes4(const float* x, float inv, int e) {
  float y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    y[i] = x[i] * inv;
    if (e == ScaleRange<T>::hi) y[i] = fminf(fmaxf(y[i], -240.f), 240.f);
    if (!(fabsf(x[i]) < ScaleRange<T>::end)) y[i] = NAN;
  }
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
  return __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
}

// Four codes rounded again for a larger exponent, `ratio` = 2^(old - new).
__device__ __forceinline__ uint32_t moved4(uint32_t w, float ratio) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a[0] * ratio, a[1] * ratio, 0, false);
  return __builtin_amdgcn_cvt_pk_fp8_f32(b[0] * ratio, b[1] * ratio, lo, true);
}

__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) v = max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), off, kWave)));
  return v;
}

// N neighbouring numbers of the data type, or of fp32.
template <class T, int N, bool AL>
__device__ __forceinline__ void load_n(const typename T::raw_t* p, float* f) {
  if constexpr (AL) {
    uint32_t w[N / 2];
    if constexpr (N == 8) *reinterpret_cast<u32x4*>(w) = ld_chunk(p);
    else *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = T::to_f32(static_cast<uint16_t>((i & 1) ? w[i / 2] >> 16 : w[i / 2] & 0xffffu));
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = T::to_f32(p[i]);
  }
}
template <class T, int N, bool AL>
__device__ __forceinline__ void table_n(const void* p, int64_t e, bool f32, float* f) {
  if (f32) {
    const float* t = static_cast<const float*>(p) + e;
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      if constexpr (AL) *reinterpret_cast<f32x4*>(f + i) = *reinterpret_cast<const f32x4*>(t + i);
      else f[i] = t[i], f[i + 1] = t[i + 1], f[i + 2] = t[i + 2], f[i + 3] = t[i + 3];
    }
  } else {
    load_n<T, N, AL>(static_cast<const typename T::raw_t*>(p) + e, f);
  }
}

// x * cos + (x rolled by D / 2) * sin of N columns of the first half and the N
// they pair with; the products are rounded before the sum, as torch's are.
template <class T, int D, int N, bool AL>
__device__ __forceinline__ void rotate(const WriteArgs& a, const typename T::raw_t* x, int r, int e, float* y0, float* y1) {
#pragma clang fp contract(off)
  alignas(16) float lo[N], hi[N], c0[N], c1[N], s0[N], s1[N];
  load_n<T, N, AL>(x + e, lo);
  load_n<T, N, AL>(x + e + D / 2, hi);
  const int64_t at = r * a.rot_stride + e;
  table_n<T, N, AL>(a.cos, at, a.rot_f32, c0);
  table_n<T, N, AL>(a.cos, at + D / 2, a.rot_f32, c1);
  table_n<T, N, AL>(a.sin, at, a.rot_f32, s0);
  table_n<T, N, AL>(a.sin, at + D / 2, a.rot_f32, s1);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float p0 = lo[i] * c0[i], p1 = hi[i] * s0[i], p2 = hi[i] * c1[i], p3 = lo[i] * s1[i];
    y0[i] = p0 + p1;
    y1[i] = p2 + p3;
  }
}

template <class T, int D>
__device__ __forceinline__ void rotate_one(const WriteArgs& a, const typename T::raw_t* x, int r, int e, float* y0, float* y1) {
#pragma clang fp contract(off)
  const int64_t at = r * a.rot_stride + e;
  auto table = [&](const void* p, int64_t i) {
    return a.rot_f32 ? static_cast<const float*>(p)[i] : T::to_f32(static_cast<const typename T::raw_t*>(p)[i]);
  };
  const float lo = T::to_f32(x[e]), hi = T::to_f32(x[e + D / 2]);
  const float p0 = lo * table(a.cos, at), p1 = hi * table(a.sin, at);
  const float p2 = hi * table(a.cos, at + D / 2), p3 = lo * table(a.sin, at + D / 2);
  *y0 = p0 + p1;
  *y1 = p2 + p3;
}

// N (2 or 4) codes in the low bytes of a word.
template <int N>
__device__ __forceinline__ void put_codes(uint8_t* p, uint32_t w) {
  if constexpr (N == 4) *reinterpret_cast<uint32_t*>(p) = w;
  else *reinterpret_cast<uint16_t*>(p) = static_cast<uint16_t>(w);
}
template <int N>
__device__ __forceinline__ uint32_t get_codes(const uint8_t* p) {
  if constexpr (N == 4) return *reinterpret_cast<const uint32_t*>(p);
  else return *reinterpret_cast<const uint16_t*>(p);
}

// A thread rotates 8 columns of a head's first half of q and the 8 they pair with.
template <class T, int D, bool AL>
__device__ __forceinline__ void rotate_q(const WriteArgs& a, int64_t id) {
  using raw = typename T::raw_t;
  constexpr int U = D / 16;  // units a head
  const int per_row = a.heads * U;
  const int r = static_cast<int>(id / per_row);
  if (r >= a.rows) return;
  const int u = static_cast<int>(id - static_cast<int64_t>(r) * per_row);
  const int h = u / U;
  const int e = (u - h * U) * 8;
  float y0[8], y1[8];
  rotate<T, D, 8, AL>(a, static_cast<const raw*>(a.q) + r * a.q_stride + h * D, r, e, y0, y1);
  raw* to = static_cast<raw*>(a.q_out) + r * a.q_out_stride + h * D;
  store_row_chunk<T, AL>(to + e, pack_chunk<T>(y0), 8);
  store_row_chunk<T, AL>(to + e + D / 2, pack_chunk<T>(y1), 8);
}

// The blocks that begin in `window` rows from r0 on.  Lane l looks at row r0 - 1
// + l; bits of lanes: rows that have a slot and are the first of their block
// here, rows that follow one in their block.
struct Blocks {
  int seen;
  uint64_t first, inside;
};
__device__ __forceinline__ Blocks find_blocks(const WriteArgs& a, int r0, int window) {
  const int lane = threadIdx.x & 63;
  const int64_t slots = static_cast<int64_t>(a.num_pages) << a.page_shift;
  const int look = r0 - 1 + lane;
  Blocks b;
  b.seen = lane < window + 16 && look >= 0 && look < a.rows ? a.slots[look] : -1;
  const int before = __shfl_up(b.seen, 1, kWave);
  const bool placed = b.seen >= 0 && b.seen < slots;
  const bool follows = lane > 0 && placed && (b.seen & (kScaleBlock - 1)) != 0 && b.seen == before + 1;
  b.inside = __ballot(follows);
  b.first = __ballot(placed && !follows) & (((1ull << window) - 1) << 1);
  return b;
}
// One of them: its first slot's place, the exponent's, and the new rows.
struct Block {
  int row, n, off;      // first row, rows (at most 16), position of the first
  int64_t id;           // page
  int in_page;          // the block's first position there
  int64_t at;           // index of its exponent
};
__device__ __forceinline__ Block take_block(const WriteArgs& a, const Blocks& b, int l, int r0, int head) {
  Block k;
  const int slot = __builtin_amdgcn_readlane(b.seen, l);
  const int page = 1 << a.page_shift;
  k.n = 1 + __builtin_ctzll(~(b.inside >> (l + 1)));
  k.row = r0 - 1 + l;
  k.off = slot & (kScaleBlock - 1);
  k.id = slot >> a.page_shift;
  k.in_page = slot & (page - 1) & ~(kScaleBlock - 1);
  k.at = ((k.id * a.kv_heads + head) << (a.page_shift - 4)) + (k.in_page >> 4);
  return k;
}
// A stored exponent; it counts where earlier rows are in the block.
template <class T>
__device__ __forceinline__ int stored(uint8_t byte) {
  return min(max(static_cast<int>(byte) - kScaleBias, ScaleRange<T>::lo), ScaleRange<T>::hi);
}
// Four positions of a column of values: positions from j on, of which those
// before `off` keep their (moved) codes and those from `end` on stay as they are.
__device__ __forceinline__ uint32_t merge4(uint32_t codes, uint32_t moved, uint32_t old, int j, int off, int end) {
  uint32_t early = 0, late = 0;
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    if (j + b < off) early |= 0xffu << (8 * b);
    if (j + b >= end) late |= 0xffu << (8 * b);
  }
  return (codes & ~(early | late)) | (moved & early) | (old & late);
}

// Few rows, each in a block of its own more often than not: a wave has the
// block that begins in its row (if one does), for keys or values of one head.
// Which row it begins with does not depend on the slots, so that is read while
// they are on their way.  Bound by that chain: slot, exponent and old codes,
// store.
template <class T, int D, bool AL>
__global__ __launch_bounds__(256, 4) void paged_write8_few_kernel(Write8Args args, int block_groups) {
  using raw = typename T::raw_t;
  const WriteArgs& a = args.w;
  if (static_cast<int>(blockIdx.x) >= block_groups) {
    rotate_q<T, D, AL>(a, (static_cast<int64_t>(blockIdx.x) - block_groups) * 256 + threadIdx.x);
    return;
  }
  constexpr int H = D / 2, N = D / kWave;
  const int page = 1 << a.page_shift;
  const int w = blockIdx.x * 4 + (threadIdx.x >> 6);
  const bool is_v = (w & 1) != 0;
  const int r0 = (w >> 1) / a.kv_heads;
  const int head = (w >> 1) % a.kv_heads;
  if (r0 >= a.rows) return;
  const int lane = threadIdx.x & 63;
  const int e = lane & (H - 1);           // D 64: the upper lanes do what the lower do
  const raw* k = static_cast<const raw*>(a.k) + head * D;
  const raw* v = static_cast<const raw*>(a.v) + head * D + lane;
  float x[2][kScaleBlock];                // keys: the two columns of a pair; values: columns lane and lane + 64; of each row
  auto read = [&](int i) {
    const int64_t r = r0 + i;
    if (!is_v) {
      rotate_one<T, D>(a, k + r * a.k_stride, r0 + i, e, &x[0][i], &x[1][i]);
    } else {
#pragma unroll
      for (int z = 0; z < N; ++z) x[z][i] = T::to_f32(v[r * a.v_stride + z * kWave]);
      if constexpr (N == 1) x[1][i] = 0.f;
    }
  };
  read(0);
  const Blocks found = find_blocks(a, r0, 1);
  if (found.first == 0) return;
  const Block b = take_block(a, found, 1, r0, head);
  uint8_t* scale = (is_v ? args.value_scales : args.key_scales) + b.at;
  const uint8_t byte = *scale;
  uint8_t* keys = static_cast<uint8_t*>(a.keys) + b.id * a.key_stride + (static_cast<int64_t>(head) * page + b.in_page) * D + e;
  uint8_t* values = static_cast<uint8_t*>(a.values) + b.id * a.value_stride + (static_cast<int64_t>(head) * D + lane) * page + b.in_page;
  u32x4 old[N];
  if (is_v && b.n < kScaleBlock)
#pragma unroll
    for (int z = 0; z < N; ++z) old[z] = ld_chunk(values + static_cast<int64_t>(z) * kWave * page);
#pragma unroll
  for (int i = 1; i < kScaleBlock; ++i) {
    if (i < b.n) read(i);
    else x[0][i] = x[1][i] = 0.f;
  }
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < kScaleBlock; ++i) top = max(top, max(counted<T>(x[0][i]), counted<T>(x[1][i])));
  const int was = stored<T>(byte);
  int ex = exponent_of<T>(wave_max(top));
  if (b.off > 0) ex = max(ex, was);
  const float inv = pow2(-ex);
  const bool grows = b.off > 0 && ex > was;
  const float ratio = ldexpf(1.f, was - ex);
  if (!is_v) {
#pragma unroll
    for (int i = 0; i < kScaleBlock; ++i) {
      if (i >= b.n) continue;
      const float y[4] = {x[0][i], x[1][i], 0.f, 0.f};
      const uint32_t c = codes4<T>(y, inv, ex);
      if (lane < H) {
        keys[(b.off + i) * D] = static_cast<uint8_t>(c);
        keys[(b.off + i) * D + H] = static_cast<uint8_t>(c >> 8);
      }
    }
    if (grows && lane < H) {
      for (int i = 0; i < b.off; ++i) {
        const uint32_t c = moved4(keys[i * D] | static_cast<uint32_t>(keys[i * D + H]) << 8, ratio);
        keys[i * D] = static_cast<uint8_t>(c);
        keys[i * D + H] = static_cast<uint8_t>(c >> 8);
      }
    }
  } else {
    // Rows to positions: row i is position off + i.
    float p[N][kScaleBlock];
#pragma unroll
    for (int z = 0; z < N; ++z)
#pragma unroll
      for (int j = 0; j < kScaleBlock; ++j) p[z][j] = x[z][0];
    if (b.n > 1) {
#pragma unroll
      for (int j = 0; j < kScaleBlock; ++j)
#pragma unroll
        for (int i = 1; i < kScaleBlock; ++i)
          if (j - b.off == i)
#pragma unroll
            for (int z = 0; z < N; ++z) p[z][j] = x[z][i];
    }
#pragma unroll
    for (int z = 0; z < N; ++z) {
      u32x4 y;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t c = codes4<T>(p[z] + 4 * i, inv, ex);
        y[i] = b.n < kScaleBlock ? merge4(c, grows ? moved4(old[z][i], ratio) : old[z][i], old[z][i], 4 * i, b.off, b.off + b.n) : c;
      }
      st_chunk(values + static_cast<int64_t>(z) * kWave * page, y);
    }
  }
  if (lane == 0 && (b.off == 0 || grows)) *scale = static_cast<uint8_t>(ex + kScaleBias);
}

// Many rows.  Some workgroups have the cache blocks that begin in kWindow rows,
// for keys or for values of one head; a block is one workgroup's alone, so its
// exponent and codes are changed without atomics.  Its 256 threads share a block
// of 16 x D numbers, 8 (D 64: 4) each: with a wave a block, the kernel's registers
// (136) left the q rows, which the other workgroups rotate, a third of the waves
// (4075 rows 30 us).  Those rows (94 MB) take 24.3 us, 3.9 TB/s; both kinds of
// workgroup in turn 24.3 (4096 tokens of one prompt 24.5, and 29.9).  Bytes need
// 18.4; a thread's eight values are loaded one after the other, each of two bytes
// behind a branch of its own and waited for, after the block's exponent.
constexpr int kWindow = 16;
template <class T, int D, bool AL>
__global__ __launch_bounds__(256) void paged_write8_kernel(Write8Args args, int block_groups) {
  using raw = typename T::raw_t;
  const WriteArgs& a = args.w;
  const int page = 1 << a.page_shift;
  if (static_cast<int>(blockIdx.x) >= block_groups) {
    rotate_q<T, D, AL>(a, (static_cast<int64_t>(blockIdx.x) - block_groups) * 256 + threadIdx.x);
    return;
  }
  __shared__ uint32_t tops[2][4];
  const bool is_v = (blockIdx.x & 1) != 0;
  const int wg = static_cast<int>(blockIdx.x) >> 1;
  const int r0 = wg / a.kv_heads * kWindow;
  const int head = wg % a.kv_heads;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const Blocks found = find_blocks(a, r0, kWindow);  // of every wave
  int turn = 0;
  for (uint64_t todo = found.first; todo != 0; todo &= todo - 1, turn ^= 1) {
    const Block k = take_block(a, found, __builtin_amdgcn_readfirstlane(__builtin_ctzll(todo)), r0, head);
    const int n = k.n, row = k.row, off = k.off, in_page = k.in_page;
    const int64_t id = k.id;
    uint8_t* scale = (is_v ? args.value_scales : args.key_scales) + k.at;
    const int was = stored<T>(*scale);
    // The block's exponent from the threads' widest numbers.
    auto exponent = [&](uint32_t top) {
      top = wave_max(top);
      if (lane == 0) tops[turn][wave] = top;
      lds_barrier();
#pragma unroll
      for (int w = 0; w < 4; ++w) top = max(top, tops[turn][w]);
      const int e = exponent_of<T>(top);
      return off > 0 ? max(e, was) : e;
    };
    if (!is_v) {
      // Thread: row tid / 16, E columns of each half.
      constexpr int E = D / 32;
      const int ri = threadIdx.x >> 4, c = (threadIdx.x & 15) * E;
      uint8_t* keys = static_cast<uint8_t*>(a.keys) + id * a.key_stride + (static_cast<int64_t>(head) * page + in_page) * D + c;
      float y[2][4] = {};
      uint32_t top = 0;
      if (ri < n) {
        const raw* x = static_cast<const raw*>(a.k) + (row + ri) * a.k_stride + head * D;
        if constexpr (E == 4) {
          rotate<T, D, 4, AL>(a, x, row + ri, c, y[0], y[1]);
        } else {
#pragma unroll
          for (int i = 0; i < E; ++i) rotate_one<T, D>(a, x, row + ri, c + i, &y[0][i], &y[1][i]);
        }
#pragma unroll
        for (int i = 0; i < E; ++i) top = max(top, max(counted<T>(y[0][i]), counted<T>(y[1][i])));
      }
      const int e = exponent(top);
      const float inv = pow2(-e);
      const bool grows = off > 0 && e > was;
      if (ri < n) {
#pragma unroll
        for (int z = 0; z < 2; ++z) put_codes<E>(keys + (off + ri) * D + z * (D / 2), codes4<T>(y[z], inv, e));
      }
      if (grows && ri < off) {
        const float ratio = ldexpf(1.f, was - e);
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          uint8_t* old = keys + ri * D + z * (D / 2);
          put_codes<E>(old, moved4(get_codes<E>(old), ratio));
        }
      }
      if (threadIdx.x == 0 && (off == 0 || grows)) *scale = static_cast<uint8_t>(e + kScaleBias);
    } else {
      // Thread: column tid % D, P positions.
      constexpr int P = 16 * D / 256;
      const int d = threadIdx.x & (D - 1), j0 = threadIdx.x / D * P;
      float x[P];
      uint32_t top = 0;
      const raw* v = static_cast<const raw*>(a.v) + head * D + d;
#pragma unroll
      for (int j = 0; j < P; ++j) {
        const int i = j0 + j - off;
        x[j] = i >= 0 && i < n ? T::to_f32(v[(row + i) * a.v_stride]) : 0.f;
      }
      uint32_t* values = reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.values) + id * a.value_stride +
                                                     (static_cast<int64_t>(head) * D + d) * page + in_page + j0);
      uint32_t old[P / 4];
#pragma unroll
      for (int w = 0; w < P / 4; ++w) old[w] = n < kScaleBlock ? values[w] : 0u;
#pragma unroll
      for (int j = 0; j < P; ++j) top = max(top, counted<T>(x[j]));
      const int e = exponent(top);
      const float inv = pow2(-e);
      const bool grows = off > 0 && e > was;
      const float ratio = ldexpf(1.f, was - e);
#pragma unroll
      for (int w = 0; w < P / 4; ++w)
        old[w] = merge4(codes4<T>(x + 4 * w, inv, e), grows ? moved4(old[w], ratio) : old[w], old[w], j0 + 4 * w, off, off + n);
      if constexpr (P == 8) *reinterpret_cast<uint2*>(values) = make_uint2(old[0], old[1]);
      else values[0] = old[0];
      if (threadIdx.x == 0 && (off == 0 || grows)) *scale = static_cast<uint8_t>(e + kScaleBias);
    }
  }
}

// Calls of fewer rows take a wave a row, of more a workgroup a block.  That is
// best where rows and requests go together, as in steps of decoding requests
// or of prompts: 64 requests of one token 4.8 us (24 with a workgroup a block),
// 511 12.5 (38); five drafts of 32 6.5 (8.9), of 64 8.5 (10.4), of 256 18.6 with a
// wave a row and 16.3 with a workgroup a block; 1024 and 2048 tokens of a prompt
// 36.7 and 65.5, 8.4 and 13.6.  It is not best for short prompts alone, of which a
// wave reads 16 rows (64 tokens 12.3 us, 4.3 with a workgroup a block; 300 17.6,
// 4.8; eight of 40 19, 6.8), nor for many requests of one token, whose blocks a
// workgroup takes one after the other (600 39.0 us, 13.8 with a wave a row; 2048
// 81, 39.6): the call has rows and slots, not how many rows a request has.
constexpr int kFewRows = 512;

template <class T, int D, bool AL>
hipError_t launch_write8(const Write8Args& args, hipStream_t stream) {
  const WriteArgs& a = args.w;
  const bool few = a.rows < kFewRows;
  const int64_t rot = (static_cast<int64_t>(a.rows) * a.heads * (D / 16) + 255) / 256;
  const int64_t blocks = few ? (static_cast<int64_t>(a.rows) * a.kv_heads * 2 + 3) / 4
                             : (static_cast<int64_t>(a.rows) + kWindow - 1) / kWindow * a.kv_heads * 2;
  if (!grid_fits(rot + blocks)) return hipErrorInvalidConfiguration;
  const dim3 grid(static_cast<unsigned>(rot + blocks));
  if (few) hipLaunchKernelGGL((paged_write8_few_kernel<T, D, AL>), grid, dim3(256), 0, stream, args, static_cast<int>(blocks));
  else hipLaunchKernelGGL((paged_write8_kernel<T, D, AL>), grid, dim3(256), 0, stream, args, static_cast<int>(blocks));
  return hipGetLastError();
}

template <class T>
hipError_t launch_write8_of(const Write8Args& a, int head_dim, bool aligned, hipStream_t stream) {
  if (head_dim == 64) return aligned ? launch_write8<T, 64, true>(a, stream) : launch_write8<T, 64, false>(a, stream);
  return aligned ? launch_write8<T, 128, true>(a, stream) : launch_write8<T, 128, false>(a, stream);
}

}  // namespace

hipError_t launch_rotary_paged_write8(const Write8Args& a, int dtype, int head_dim, bool aligned, hipStream_t stream) {
  if (a.w.rows == 0) return hipSuccess;
  return dtype == MLORA_BF16 ? launch_write8_of<BF16>(a, head_dim, aligned, stream) : launch_write8_of<F16>(a, head_dim, aligned, stream);
}

}  // namespace mlora
