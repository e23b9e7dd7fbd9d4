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
#include "rotary.h"

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

// Four codes rounded again for an exponent that is `down` more.
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

// Workgroups [0, block_groups): one has the cache blocks that begin in `window`
// rows, for keys or for values of one head; a block is one workgroup's alone, so
// its exponent and codes are changed without atomics.  Its 256 threads share a
// block of 16 x D numbers, 8 (D 64: 4) each: with a wave a block, the kernel's
// registers (136) left the q rows a third of the waves (4075 rows 30.4 us).  The
// rest: a thread rotates 8 columns of a head's first half of q and the 8 they
// pair with.
template <class T, int D, bool AL>
__global__ __launch_bounds__(256) void paged_write8_kernel(Write8Args args, int block_groups, int window) {
  using raw = typename T::raw_t;
  const WriteArgs& a = args.w;
  const int page = 1 << a.page_shift;
  const int64_t slots = static_cast<int64_t>(a.num_pages) << a.page_shift;
  if (static_cast<int>(blockIdx.x) >= block_groups) {
    constexpr int U = D / 16;  // units a head
    const int64_t id = (static_cast<int64_t>(blockIdx.x) - block_groups) * 256 + threadIdx.x;
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
    return;
  }
  __shared__ uint32_t tops[2][4];
  const bool is_v = (blockIdx.x & 1) != 0;
  const int wg = static_cast<int>(blockIdx.x) >> 1;
  const int r0 = wg / a.kv_heads * window;
  const int head = wg % a.kv_heads;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // Lane l of every wave looks at row r0 - 1 + l.  Bits of lanes: rows that have
  // a slot and are the first of their block here, rows that follow one in their block.
  const int look = r0 - 1 + lane;
  const int seen = lane < window + 16 && look >= 0 && look < a.rows ? a.slots[look] : -1;
  const int before = __shfl_up(seen, 1, kWave);
  const bool placed = seen >= 0 && seen < slots;
  const bool follows = lane > 0 && placed && (seen & (kScaleBlock - 1)) != 0 && seen == before + 1;
  const uint64_t inside = __ballot(follows);
  const uint64_t mine = (((1ull << window) - 1) << 1);
  int turn = 0;
  for (uint64_t todo = __ballot(placed && !follows) & mine; todo != 0; todo &= todo - 1, turn ^= 1) {
    const int l = __builtin_amdgcn_readfirstlane(__builtin_ctzll(todo));
    const int slot = __builtin_amdgcn_readlane(seen, l);
    const int n = 1 + __builtin_ctzll(~(inside >> (l + 1)));  // rows of the block, at most 16
    const int row = r0 - 1 + l;
    const int off = slot & (kScaleBlock - 1);
    const int64_t id = slot >> a.page_shift;
    const int in_page = slot & (page - 1) & ~(kScaleBlock - 1);
    const int64_t at = ((id * a.kv_heads + head) << (a.page_shift - 4)) + (in_page >> 4);
    uint8_t* scale = (is_v ? args.value_scales : args.key_scales) + at;
    // A block's exponent counts where earlier rows are in it.
    const int was = min(max(static_cast<int>(*scale) - kScaleBias, ScaleRange<T>::lo), ScaleRange<T>::hi);
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
      // Positions before `off` are earlier rows, those behind the new ones stay as they are.
#pragma unroll
      for (int w = 0; w < P / 4; ++w) {
        uint32_t early = 0, late = 0;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          if (j0 + 4 * w + b < off) early |= 0xffu << (8 * b);
          if (j0 + 4 * w + b >= off + n) late |= 0xffu << (8 * b);
        }
        const uint32_t kept = grows ? moved4(old[w], ratio) : old[w];
        old[w] = (codes4<T>(x + 4 * w, inv, e) & ~(early | late)) | (kept & early) | (old[w] & late);
      }
      if constexpr (P == 8) *reinterpret_cast<uint2*>(values) = make_uint2(old[0], old[1]);
      else values[0] = old[0];
      if (threadIdx.x == 0 && (off == 0 || grows)) *scale = static_cast<uint8_t>(e + kScaleBias);
    }
  }
}

// Rows whose blocks one workgroup looks after.
constexpr int window_rows(int rows) { return rows < 512 ? 1 : 16; }

template <class T, int D>
hipError_t launch_write8(const Write8Args& args, bool aligned, hipStream_t stream) {
  const WriteArgs& a = args.w;
  const int window = window_rows(a.rows);
  const int64_t units = static_cast<int64_t>(a.rows) * a.heads * (D / 16);
  const int64_t rot = (units + 255) / 256;
  const int64_t blocks = (static_cast<int64_t>(a.rows) + window - 1) / window * a.kv_heads * 2;
  if (!grid_fits(rot + blocks)) return hipErrorInvalidConfiguration;
  const dim3 grid(static_cast<unsigned>(rot + blocks));
  if (aligned)
    hipLaunchKernelGGL((paged_write8_kernel<T, D, true>), grid, dim3(256), 0, stream, args, static_cast<int>(blocks), window);
  else
    hipLaunchKernelGGL((paged_write8_kernel<T, D, false>), grid, dim3(256), 0, stream, args, static_cast<int>(blocks), window);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_rotary_paged_write8(const Write8Args& a, int dtype, int head_dim, bool aligned, hipStream_t stream) {
  if (a.w.rows == 0) return hipSuccess;
  if (dtype == MLORA_BF16)
    return head_dim == 64 ? launch_write8<BF16, 64>(a, aligned, stream) : launch_write8<BF16, 128>(a, aligned, stream);
  return head_dim == 64 ? launch_write8<F16, 64>(a, aligned, stream) : launch_write8<F16, 128>(a, aligned, stream);
}

}  // namespace mlora
