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

// x * cos + (x rolled by D / 2) * sin of 8 columns of the first half and the 8
// they pair with; the products are rounded before the sum, as torch's are.
template <class T, int D, bool AL>
__device__ __forceinline__ void rotate8(const WriteArgs& a, const typename T::raw_t* x, int r, int e, float* y0, float* y1) {
#pragma clang fp contract(off)
  const u32x4 lo = load_row_chunk<T, AL>(x, e, 8);
  const u32x4 hi = load_row_chunk<T, AL>(x, e + D / 2, 8);
  float c0[8], c1[8], s0[8], s1[8];
  const char* cs = static_cast<const char*>(a.cos) + r * a.rot_stride * (a.rot_f32 ? 4 : 2);
  const char* sn = static_cast<const char*>(a.sin) + r * a.rot_stride * (a.rot_f32 ? 4 : 2);
  rot_chunk<T, AL>(cs, e, a.rot_f32, c0);
  rot_chunk<T, AL>(cs, e + D / 2, a.rot_f32, c1);
  rot_chunk<T, AL>(sn, e, a.rot_f32, s0);
  rot_chunk<T, AL>(sn, e + D / 2, a.rot_f32, s1);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float x0 = chunk_elem<T>(lo, i), x1 = chunk_elem<T>(hi, i);
    const float p0 = x0 * c0[i], p1 = x1 * s0[i], p2 = x1 * c1[i], p3 = x0 * s1[i];
    y0[i] = p0 + p1;
    y1[i] = p2 + p3;
  }
}

// Blocks [0, block_blocks): a wave has the cache blocks that begin in a few
// rows (of which its first lanes look at the slots), for keys or for values of
// one head; a block is one wave's alone, so its exponent and codes are changed
// without atomics.  The rest: a thread rotates 8 columns of a head's first half
// of q and the 8 they pair with.
template <class T, int D, bool AL>
__global__ __launch_bounds__(256) void paged_write8_kernel(Write8Args args, int block_blocks, int window) {
  using raw = typename T::raw_t;
  const WriteArgs& a = args.w;
  const int page = 1 << a.page_shift;
  const int64_t slots = static_cast<int64_t>(a.num_pages) << a.page_shift;
  if (static_cast<int>(blockIdx.x) >= block_blocks) {
    constexpr int U = D / 16;  // units a head
    const int64_t id = (static_cast<int64_t>(blockIdx.x) - block_blocks) * 256 + threadIdx.x;
    const int per_row = a.heads * U;
    const int r = static_cast<int>(id / per_row);
    if (r >= a.rows) return;
    const int u = static_cast<int>(id - static_cast<int64_t>(r) * per_row);
    const int h = u / U;
    const int e = (u - h * U) * 8;
    float y0[8], y1[8];
    rotate8<T, D, AL>(a, static_cast<const raw*>(a.q) + r * a.q_stride + h * D, r, e, y0, y1);
    raw* to = static_cast<raw*>(a.q_out) + r * a.q_out_stride + h * D;
    store_row_chunk<T, AL>(to + e, pack_chunk<T>(y0), 8);
    store_row_chunk<T, AL>(to + e + D / 2, pack_chunk<T>(y1), 8);
    return;
  }
  const int64_t w = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const bool is_v = (w & 1) != 0;
  const int64_t wg = w >> 1;
  const int64_t first = wg / a.kv_heads * window;
  if (first >= a.rows) return;
  const int r0 = static_cast<int>(first);
  const int head = static_cast<int>(wg % a.kv_heads);
  const int lane = threadIdx.x & 63;
  // Lane l looks at row r0 - 1 + l.  Bits of lanes: rows that have a slot and
  // are the first of their block here, rows that follow one in their block.
  const int look = r0 - 1 + lane;
  const int seen = lane < window + 16 && look >= 0 && look < a.rows ? a.slots[look] : -1;
  const int before = __shfl_up(seen, 1, kWave);
  const bool placed = seen >= 0 && seen < slots;
  const bool follows = lane > 0 && placed && (seen & (kScaleBlock - 1)) != 0 && seen == before + 1;
  const uint64_t inside = __ballot(follows);
  const uint64_t mine = (((1ull << window) - 1) << 1);
  for (uint64_t todo = __ballot(placed && !follows) & mine; todo != 0; todo &= todo - 1) {
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
    if (!is_v) {
      // Lane: row lane >> 2, D / 8 columns of each half.
      constexpr int E = D / 8;
      const int ri = lane >> 2, c = lane & 3;
      float y[2][E];
      uint32_t top = 0;
      if (ri < n) {
        const raw* x = static_cast<const raw*>(a.k) + (row + ri) * a.k_stride + head * D;
#pragma unroll
        for (int e = 0; e < E; e += 8) rotate8<T, D, AL>(a, x, row + ri, c * E + e, y[0] + e, y[1] + e);
#pragma unroll
        for (int i = 0; i < E; ++i) top = max(top, max(counted<T>(y[0][i]), counted<T>(y[1][i])));
      }
      int e = exponent_of<T>(wave_max(top));
      if (off > 0) e = max(e, was);
      const float inv = pow2(-e);
      uint8_t* keys = static_cast<uint8_t*>(a.keys) + id * a.key_stride + (static_cast<int64_t>(head) * page + in_page) * D + c * E;
      if (ri < n) {
        uint32_t* to = reinterpret_cast<uint32_t*>(keys + (off + ri) * D);
#pragma unroll
        for (int i = 0; i < E / 4; ++i) {
          to[i] = codes4<T>(y[0] + 4 * i, inv, e);
          to[D / 8 + i] = codes4<T>(y[1] + 4 * i, inv, e);
        }
      }
      if (off > 0 && e > was && ri < off) {
        const float ratio = ldexpf(1.f, was - e);
        uint32_t* old = reinterpret_cast<uint32_t*>(keys + ri * D);
#pragma unroll
        for (int i = 0; i < E / 4; ++i) {
          old[i] = moved4(old[i], ratio);
          old[D / 8 + i] = moved4(old[D / 8 + i], ratio);
        }
      }
      if (lane == 0 && (off == 0 || e > was)) *scale = static_cast<uint8_t>(e + kScaleBias);
    } else {
      // Lane: columns lane and lane + 64, all 16 positions.
      float x[D / kWave][kScaleBlock];
      uint32_t top = 0;
      const raw* v = static_cast<const raw*>(a.v) + head * D + lane;
#pragma unroll
      for (int j = 0; j < kScaleBlock; ++j) {
        const bool has = j >= off && j < off + n;
#pragma unroll
        for (int d = 0; d < D / kWave; ++d) {
          x[d][j] = has ? T::to_f32(v[(row + j - off) * a.v_stride + d * kWave]) : 0.f;
          top = max(top, counted<T>(x[d][j]));
        }
      }
      uint8_t* values = static_cast<uint8_t*>(a.values) + id * a.value_stride + (static_cast<int64_t>(head) * D + lane) * page + in_page;
      u32x4 old[D / kWave];
      if (n < kScaleBlock)
#pragma unroll
        for (int d = 0; d < D / kWave; ++d) old[d] = ld_chunk(values + static_cast<int64_t>(d) * kWave * page);
      int e = exponent_of<T>(wave_max(top));
      if (off > 0) e = max(e, was);
      const float inv = pow2(-e);
      const float ratio = ldexpf(1.f, was - e);
#pragma unroll
      for (int d = 0; d < D / kWave; ++d) {
        u32x4 y;
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = codes4<T>(x[d] + 4 * i, inv, e);
        if (n < kScaleBlock) {
          // Positions before `off` are earlier rows, those behind the new ones stay as they are.
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t kept = off > 0 && e > was ? moved4(old[d][i], ratio) : old[d][i];
            uint32_t early = 0, late = 0;
#pragma unroll
            for (int b = 0; b < 4; ++b) {
              if (4 * i + b < off) early |= 0xffu << (8 * b);
              if (4 * i + b >= off + n) late |= 0xffu << (8 * b);
            }
            y[i] = (y[i] & ~(early | late)) | (kept & early) | (old[d][i] & late);
          }
        }
        st_chunk(values + static_cast<int64_t>(d) * kWave * page, y);
      }
      if (lane == 0 && (off == 0 || e > was)) *scale = static_cast<uint8_t>(e + kScaleBias);
    }
  }
}

// Rows whose blocks one wave looks after.
constexpr int window_rows(int rows) { return rows < 512 ? 1 : 16; }

template <class T, int D>
hipError_t launch_write8(const Write8Args& args, bool aligned, hipStream_t stream) {
  const WriteArgs& a = args.w;
  const int window = window_rows(a.rows);
  const int64_t units = static_cast<int64_t>(a.rows) * a.heads * (D / 16);
  const int64_t rot = (units + 255) / 256;
  const int64_t waves = (static_cast<int64_t>(a.rows) + window - 1) / window * a.kv_heads * 2;
  const int64_t blocks = (waves + 3) / 4;
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
