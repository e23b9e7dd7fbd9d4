// Rows of activations quantised to 8-bit integers, and products of such rows
// with a weight whose output channels have a scale each (gfx950).
//
// A row's scale is s = max|x| / 127, its codes rint(x / s); a product is
// s * t * sum(codes * codes) + bias.  The sum is exact in 32 bits, whatever the
// order, so every variant below gives the same bits.
#include <algorithm>

#include "int8.h"
#include "kernels.h"
#include "loads.h"

namespace mlora {

namespace {

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x16 __attribute__((ext_vector_type(16)));
typedef const __attribute__((address_space(1))) void gvoid_t;
typedef __attribute__((address_space(3))) void lvoid_t;

constexpr float kLeast = 7.888609052210118e-31f;  // 2^-100: a row's least maximum, so that neither scale leaves fp32
constexpr uint32_t kInfBits = 0x7f800000u;

// |x| as an integer: for what is not negative, floats compare as integers do,
// and NaN is above infinity is above every number.
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// A row's maximum as codes and scale need it.
struct RowScale {
  float top, half;  // divided by 2^8, so that 127 times the maximum stays finite
  float inv, scale;
};
__device__ __forceinline__ RowScale row_scale(uint32_t bits) {
  RowScale s;
  const float top = fmaxf(__uint_as_float(min(bits, kInfBits)), kLeast);
  s.top = top * 0x1p-8f;
  s.half = top * 0x1p-9f;
  s.inv = 127.f / top;
  s.scale = bits >= kInfBits ? NAN : top / 127.f;
  return s;
}

// rint(127 x / top), ties to even.  x * inv is off by some 2^-22 of itself, so
// the nearest integer is off by one only where the quotient is that close to
// halfway; the remainder 127 x - r * top says so exactly (a 16-bit x has at most
// 11 bits, 127 and r have 7, and r is 0 or x at least 2^-8 of top).
__device__ __forceinline__ int code_of(float x, const RowScale& s) {
  float r = __builtin_rintf(x * s.inv);
  const float d = __builtin_fmaf(-r, s.top, x * (127.f * 0x1p-8f));
  const float ad = fabsf(d);
  if (ad >= s.half) {
    const bool odd = (static_cast<int>(r) & 1) != 0;
    if (ad > s.half || odd) r += copysignf(1.f, d);
  }
  return static_cast<int>(r);
}

__device__ __forceinline__ uint32_t pack4(const int* c) {
  return (c[0] & 0xff) | (c[1] & 0xff) << 8 | (c[2] & 0xff) << 16 | static_cast<uint32_t>(c[3]) << 24;
}

// Eight elements of a row from element e on, zeros behind its end.
template <class T, bool AL>
__device__ __forceinline__ void load8(const typename T::raw_t* row, int e, int k, float* f) {
  const int valid = min(max(k - e, 0), 8);
  if constexpr (sizeof(typename T::raw_t) == 2) {
    const u32x4 v = load_row_chunk<T, AL>(row, e, valid);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = chunk_elem<T>(v, i);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = i < valid ? T::to_f32(row[e + i]) : 0.f;
  }
}

constexpr int kQuantKeep = 4;  // chunks of eight elements a thread keeps; longer rows are read twice

// TPR threads a row, eight elements at a time.  Bound by bytes: 2 in and 1 out
// an element.
template <class T, int TPR, bool AL>
__global__ __launch_bounds__(256) void quantize_rows_kernel(QuantArgs a) {
  using raw = typename T::raw_t;
  constexpr int RPB = 256 / TPR;
  __shared__ uint32_t tops[RPB][TPR / 64];
  const int sub = threadIdx.x / TPR;
  const int t = threadIdx.x - sub * TPR;
  const int row = blockIdx.x * RPB + sub;
  const raw* x = static_cast<const raw*>(a.x) + static_cast<int64_t>(min(row, a.rows - 1)) * a.x_stride;
  const int padded = static_cast<int>(int8_padded(a.k));
  float keep[kQuantKeep][8];
  uint32_t top = 0;
#pragma unroll
  for (int c = 0; c < kQuantKeep; ++c) {
    load8<T, AL>(x, (c * TPR + t) * 8, a.k, keep[c]);
  }
#pragma unroll
  for (int c = 0; c < kQuantKeep; ++c)
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, abs_bits(keep[c][i]));
  for (int e = (kQuantKeep * TPR + t) * 8; e < a.k; e += TPR * 8) {
    float f[8];
    load8<T, AL>(x, e, a.k, f);
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, abs_bits(f[i]));
  }
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), off, kWave)));
  if constexpr (TPR > 64) {
    if ((t & 63) == 0) tops[sub][t >> 6] = top;
    lds_barrier();
#pragma unroll
    for (int w = 0; w < TPR / 64; ++w) top = max(top, tops[sub][w]);
  }
  if (row >= a.rows) return;
  const RowScale s = row_scale(top);
  if (t == 0) a.scales[row] = s.scale;
  int8_t* out = a.codes + row * a.codes_stride;
  auto put = [&](int e, const float* f) {
    if (e >= padded) return;
    int q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = code_of(f[i], s);
    *reinterpret_cast<uint2*>(out + e) = make_uint2(pack4(q), pack4(q + 4));
  };
#pragma unroll
  for (int c = 0; c < kQuantKeep; ++c) put((c * TPR + t) * 8, keep[c]);
  for (int e = (kQuantKeep * TPR + t) * 8; e < padded; e += TPR * 8) {
    float f[8];
    load8<T, AL>(x, e, a.k, f);
    put(e, f);
  }
}

// Four columns of a row of the result, n to n + 3.
template <class T>
__device__ __forceinline__ void store4(const Int8Args& a, int m, int n, const i32x4& sum, float as) {
  using raw = typename T::raw_t;
  float y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = min(n + i, a.n - 1);
    y[i] = static_cast<float>(sum[i]) * a.b_scales[c] * as;
    if (a.bias != nullptr) y[i] += T::to_f32(static_cast<const raw*>(a.bias)[c]);
  }
  raw* out = static_cast<raw*>(a.out) + m * a.out_stride + n;
  if (a.vec && n + 4 <= a.n) {
    *reinterpret_cast<uint2*>(out) = make_uint2(T::pack2(y[0], y[1]), T::pack2(y[2], y[3]));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < a.n) out[i] = T::from_f32(y[i]);
  }
}

// Few rows: a workgroup has 16 NT output columns of up to 16 MT rows; its
// waves take the 128-byte pieces of the weight's rows in turn, straight from
// memory into operands (lane l: row l & 15, the 16 bytes 16 (l >> 4) on and
// those 64 further), and add their sums in LDS.
template <class T, int MT, int NT, int NW, int U, bool FUSE>
__global__ __launch_bounds__(NW * 64) void int8_rows_kernel(Int8Args a) {
  using raw = typename T::raw_t;
  extern __shared__ __align__(16) char lds[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15;
  const int g = lane >> 4;
  const int n0 = blockIdx.x * 16 * NT;
  const int m0 = blockIdx.y * 16 * MT;
  const int padded = static_cast<int>(int8_padded(a.k));
  const int pieces = padded / 128;

  const int8_t* wp[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) wp[t] = a.b + static_cast<int64_t>(min(n0 + t * 16 + col, a.n - 1)) * a.b_stride + g * 16;
  const int8_t* xp[MT];
  if constexpr (!FUSE) {
#pragma unroll
    for (int t = 0; t < MT; ++t) xp[t] = a.a + static_cast<int64_t>(min(m0 + t * 16 + col, a.m - 1)) * a.a_stride + g * 16;
  }
  u32x4 wf[U][NT][2], xf[U][MT][2];
  auto load = [&](int u, int piece) {
    const int p = min(piece, pieces - 1) * 128;
#pragma unroll
    for (int t = 0; t < NT; ++t) wf[u][t][0] = ld_chunk(wp[t] + p), wf[u][t][1] = ld_chunk(wp[t] + p + 64);
    if constexpr (!FUSE) {
#pragma unroll
      for (int t = 0; t < MT; ++t) xf[u][t][0] = ld_chunk(xp[t] + p), xf[u][t][1] = ld_chunk(xp[t] + p + 64);
    }
  };
#pragma unroll
  for (int u = 0; u < U; ++u) load(u, wave + u * NW);

  // The workgroup's rows as codes in LDS, rows 64 bytes further apart than
  // they are long: the rows of a fragment then lie in different banks.
  const int pitch = padded + 64;
  uint32_t* tops = reinterpret_cast<uint32_t*>(lds);
  int8_t* codes = reinterpret_cast<int8_t*>(lds) + 64;
  if constexpr (FUSE) {
    static_assert(MT == 1, "one tile of rows");
    if (threadIdx.x < 16) tops[threadIdx.x] = 0;
    lds_barrier();
    const int chunks = padded / 8;
    constexpr int KEEP = 8;  // chunks of a thread: int8_fused
    float keep[KEEP][8];
#pragma unroll
    for (int c = 0; c < KEEP; ++c) {
      const int i = c * NW * 64 + threadIdx.x;
      const int r = i / chunks;
      if (r >= a.m) continue;
      const raw* x = static_cast<const raw*>(a.x) + r * a.x_stride;
      if (a.x_aligned) load8<T, true>(x, (i - r * chunks) * 8, a.k, keep[c]);
      else load8<T, false>(x, (i - r * chunks) * 8, a.k, keep[c]);
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max(top, abs_bits(keep[c][e]));
      atomicMax(&tops[r], top);
    }
    lds_barrier();
#pragma unroll
    for (int c = 0; c < KEEP; ++c) {
      const int i = c * NW * 64 + threadIdx.x;
      const int r = i / chunks;
      if (r >= a.m) continue;
      const RowScale s = row_scale(tops[r]);
      int q[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) q[e] = code_of(keep[c][e], s);
      *reinterpret_cast<uint2*>(codes + r * pitch + (i - r * chunks) * 8) = make_uint2(pack4(q), pack4(q + 4));
    }
    lds_barrier();
  }
  const int8_t* xl = codes + min(col, a.m - 1) * pitch + g * 16;

  i32x4 acc[NT][MT];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[n][m] = i32x4{0, 0, 0, 0};
  for (int p0 = wave; p0 < pieces; p0 += U * NW) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int p = p0 + u * NW;
      if (p < pieces) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if constexpr (FUSE) xf[u][0][h] = *reinterpret_cast<const u32x4*>(xl + p * 128 + h * 64);
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int m = 0; m < MT; ++m)
              acc[n][m] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, wf[u][n][h]),
                                                                __builtin_bit_cast(i32x4, xf[u][m][h]), acc[n][m], 0, 0, 0);
        }
      }
      load(u, p + U * NW);
    }
  }
  // Lane l has rows l & 15 of the tile's m and 4 (l >> 4) on of its n.
  const uint32_t mine = FUSE ? tops[min(col, a.m - 1)] : 0;
  lds_barrier();  // the codes have been read
  i32x4* part = reinterpret_cast<i32x4*>(lds);
  constexpr int S = NT * MT * 64;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int m = 0; m < MT; ++m) part[wave * S + (n * MT + m) * 64 + lane] = acc[n][m];
  lds_barrier();
  for (int i = threadIdx.x; i < S; i += NW * 64) {
    i32x4 sum = part[i];
#pragma unroll
    for (int w = 1; w < NW; ++w) sum += part[w * S + i];
    const int t = i >> 6;
    const int n = n0 + (t / MT) * 16 + g * 4;
    const int m = m0 + (t % MT) * 16 + col;
    if (m < a.m && n < a.n) store4<T>(a, m, n, sum, FUSE ? row_scale(mine).scale : a.a_scales[m]);
  }
}

constexpr int kRowsWaves = 8;
constexpr int kFusedElems = kRowsWaves * 64 * 8 * 8;  // that many elements a workgroup keeps in registers

// Many rows: tiles of TN weight rows by TM rows over K, 128 bytes of each at a
// time in LDS, loaded straight there one step ahead.  Chunk c (16 bytes) of row
// r lies at c ^ (r & 7): a fragment's eight neighbouring rows then lie in
// different banks.
template <class T, int TN, int TM, int WN, int WM>
__global__ __launch_bounds__(WN * WM * 64) void int8_tile_kernel(Int8Args a, int tiles_n, int tiles_m) {
  constexpr int NW = WN * WM;
  constexpr int FN = TN / WN / 32, FM = TM / WM / 32;  // 32x32 blocks of a wave
  constexpr int BLOCKS = (TN + TM) / 8;                // 1 KB blocks (8 rows) of a step
  constexpr int LOADS = BLOCKS / NW;
  static_assert(BLOCKS % NW == 0, "whole blocks a wave");
  constexpr int STAGE = (TN + TM) * 128;
  __shared__ __align__(16) char lds[2 * STAGE];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int steps = static_cast<int>(int8_padded(a.k)) / 128;
  const int tile_n = blockIdx.x % tiles_n, tile_m = blockIdx.x / tiles_n;
  const int n0 = tile_n * TN, m0 = tile_m * TM;

  // Block b of a step: rows 8 b to 8 b + 7 of the weight's tile, then of the other.
  const int8_t* from[LOADS];
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const int r = (wave * LOADS + i) * 8 + (lane >> 3);
    const int chunk = (lane & 7) ^ (r & 7);
    from[i] = (r < TN ? a.b + static_cast<int64_t>(min(n0 + r, a.n - 1)) * a.b_stride
                      : a.a + static_cast<int64_t>(min(m0 + r - TN, a.m - 1)) * a.a_stride) + chunk * 16;
  }
  auto load = [&](int step, int buf) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
      __builtin_amdgcn_global_load_lds((gvoid_t*)(from[i] + static_cast<int64_t>(step) * 128),
                                       (lvoid_t*)(lds + buf * STAGE + (wave * LOADS + i) * 1024), 16, 0, 0);
  };
  const int wn = wave % WN, wm = wave / WN;
  const int row = lane & 31, h = lane >> 5;
  const char* nb = lds + (wn * (TN / WN) + row) * 128;
  const char* mb = lds + (TN + wm * (TM / WM) + row) * 128;
  i32x16 acc[FN][FM];
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int j = 0; j < FM; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;
  load(0, 0);
  int buf = 0;
  for (int s = 0; s < steps; ++s, buf ^= 1) {
    wait_vmcnt<0>();
    lds_barrier();  // the step has landed, and nobody reads the other buffer
    if (s + 1 < steps) load(s + 1, buf ^ 1);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int c = ((k * 2 + h) ^ (row & 7)) * 16 + buf * STAGE;
      i32x4 nf[FN], mf[FM];
#pragma unroll
      for (int i = 0; i < FN; ++i) nf[i] = *reinterpret_cast<const i32x4*>(nb + c + i * 32 * 128);
#pragma unroll
      for (int j = 0; j < FM; ++j) mf[j] = *reinterpret_cast<const i32x4*>(mb + c + j * 32 * 128);
#pragma unroll
      for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(nf[i], mf[j], acc[i][j], 0, 0, 0);
    }
  }
  // Lane l has row l & 31 of a block's m; register r its n 8 (r >> 2) + 4 (l >> 5) + (r & 3).
#pragma unroll
  for (int j = 0; j < FM; ++j) {
    const int m = m0 + wm * (TM / WM) + j * 32 + row;
    if (m >= a.m) continue;
    const float as = a.a_scales[m];
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int n = n0 + wn * (TN / WN) + i * 32 + q * 8 + h * 4;
        if (n < a.n) store4<T>(a, m, n, i32x4{acc[i][j][q * 4], acc[i][j][q * 4 + 1], acc[i][j][q * 4 + 2], acc[i][j][q * 4 + 3]}, as);
      }
  }
}

template <class T, int MT, int NT, int U, bool FUSE>
hipError_t launch_rows(const Int8Args& a, hipStream_t stream) {
  constexpr int NW = kRowsWaves;
  const int codes = FUSE ? 64 + a.m * (static_cast<int>(int8_padded(a.k)) + 64) : 0;
  const int bytes = std::max(codes, NW * NT * MT * 64 * 16);  // at most 64 KB
  const auto kernel = int8_rows_kernel<T, MT, NT, NW, U, FUSE>;
  const dim3 grid(cdiv(a.n, 16 * NT), cdiv(a.m, 16 * MT));
  if (!grid_fits(2 * static_cast<int64_t>(grid.x))) return hipErrorInvalidConfiguration;
  hipLaunchKernelGGL(kernel, grid, dim3(NW * 64), bytes, stream, a);
  return hipGetLastError();
}

template <class T, int TN, int TM, int WN, int WM>
hipError_t launch_tile(const Int8Args& a, hipStream_t stream) {
  const int64_t tn = (static_cast<int64_t>(a.n) + TN - 1) / TN, tm = (static_cast<int64_t>(a.m) + TM - 1) / TM;
  if (!grid_fits(tn * tm * (WN * WM / 4))) return hipErrorInvalidConfiguration;
  hipLaunchKernelGGL((int8_tile_kernel<T, TN, TM, WN, WM>), dim3(static_cast<unsigned>(tn * tm)), dim3(WN * WM * 64), 0, stream, a,
                     static_cast<int>(tn), static_cast<int>(tm));
  return hipGetLastError();
}

template <class T>
hipError_t launch(const Int8Args& a, int cus, hipStream_t stream) {
  if (a.a == nullptr) return launch_rows<T, 1, 1, 4, true>(a, stream);
  if (a.m <= 16) return launch_rows<T, 1, 1, 4, false>(a, stream);
  if (a.m <= 32) return launch_rows<T, 2, 2, 4, false>(a, stream);
  if (a.m <= 64) return launch_rows<T, 4, 2, 4, false>(a, stream);
  auto tiles = [&](int tn, int tm) { return static_cast<int64_t>(cdiv(a.n, tn)) * cdiv(a.m, tm); };
  if (tiles(256, 256) >= cus) return launch_tile<T, 256, 256, 2, 4>(a, stream);
  if (tiles(128, 128) >= cus) return launch_tile<T, 128, 128, 2, 2>(a, stream);
  return launch_tile<T, 64, 64, 2, 2>(a, stream);
}

template <class T, int TPR>
hipError_t launch_quant(const QuantArgs& a, bool aligned, hipStream_t stream) {
  const int64_t blocks = (static_cast<int64_t>(a.rows) + 256 / TPR - 1) / (256 / TPR);
  if (!grid_fits(blocks)) return hipErrorInvalidConfiguration;
  const dim3 grid(static_cast<unsigned>(blocks));
  if (aligned) hipLaunchKernelGGL((quantize_rows_kernel<T, TPR, true>), grid, dim3(256), 0, stream, a);
  else hipLaunchKernelGGL((quantize_rows_kernel<T, TPR, false>), grid, dim3(256), 0, stream, a);
  return hipGetLastError();
}

template <class T>
hipError_t quant_of(const QuantArgs& a, bool aligned, hipStream_t stream) {
  return a.k <= 1024 ? launch_quant<T, 64>(a, aligned, stream) : launch_quant<T, 256>(a, aligned, stream);
}

}  // namespace

bool int8_fused(int m, int k) { return m <= 8 && m * int8_padded(k) <= kFusedElems; }

hipError_t launch_quantize_rows(const QuantArgs& a, int dtype, bool aligned, hipStream_t stream) {
  if (a.rows == 0) return hipSuccess;
  if (dtype == MLORA_BF16) return quant_of<BF16>(a, aligned, stream);
  if (dtype == MLORA_F16) return quant_of<F16>(a, aligned, stream);
  return quant_of<F32>(a, false, stream);
}

hipError_t launch_int8_matmul(const Int8Args& a, int dtype, int cus, hipStream_t stream) {
  if (a.m == 0 || a.n == 0) return hipSuccess;
  return dtype == MLORA_BF16 ? launch<BF16>(a, cus, stream) : launch<F16>(a, cus, stream);
}

}  // namespace mlora
