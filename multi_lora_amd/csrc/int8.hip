// Rows of activations quantised to 8-bit integers, and products of such rows
// with a weight whose output channels have a scale each (gfx950).
//
// A row's scale is s = max|x| / 127, its codes rint(x / s); a product is
// s * t * sum(codes * codes) + bias.  The sum is exact in 32 bits, whatever the
// order, so every variant below gives the same bits.
#include <algorithm>

#include "int8.h"
#include "int8_tile.h"
#include "kernels.h"
#include "loads.h"

namespace mlora {

namespace {

constexpr float kLeast = 7.888609052210118e-31f;  // 2^-100: a row's least maximum, so that neither scale leaves fp32
constexpr uint32_t kInfBits = 0x7f800000u;

// |x| as an integer: for what is not negative, floats compare as integers do,
// and NaN is above infinity is above every number.
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// A row's maximum as codes and scale need it.
struct RowScale {
  float top, inv;  // the maximum divided by 2^8, so that 127 times it stays finite, and 1 over that
  float scale;
};
__device__ __forceinline__ RowScale row_scale(uint32_t bits) {
  RowScale s;
  const float top = fmaxf(__uint_as_float(min(bits, kInfBits)), kLeast);
  s.top = top * 0x1p-8f;
  s.inv = 1.f / s.top;
  s.scale = bits >= kInfBits ? NAN : top / 127.f;
  return s;
}

// rint(127 x / top), ties to even, in the low byte.  The quotient is corrected
// by its remainder, which is exact (127 x has at most 18 bits for a 16-bit x), and
// with that right to its last bit but one: a tie comes out as one, and no other
// quotient is within 2^-19 of itself of one.  Adding 1.5 * 2^23 rounds.
__device__ __forceinline__ uint32_t code_of(float x, const RowScale& s) {
  const float t = x * (127.f * 0x1p-8f);
  const float q = t * s.inv;
  const float exact = __builtin_fmaf(__builtin_fmaf(-q, s.top, t), s.inv, q);
  return __float_as_uint(exact + 12582912.f);
}

// The low bytes of four words.
__device__ __forceinline__ uint32_t pack4(const uint32_t* c) {
  const uint32_t lo = __builtin_amdgcn_perm(c[1], c[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(c[3], c[2], 0x0c0c0400u);
  return __builtin_amdgcn_perm(hi, lo, 0x05040100u);
}

// Eight elements of a row of a 16-bit type from element e on, zeros behind its end.
template <class T, bool AL>
__device__ __forceinline__ void load8(const typename T::raw_t* row, int e, int k, float* f) {
  const u32x4 v = load_row_chunk<T, AL>(row, e, min(max(k - e, 0), 8));
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = chunk_elem<T>(v, i);
}

// Rows from which on a workgroup has more than one of them, where a row fits the
// registers of its share of the waves.
constexpr int kQuantMany = 400;
constexpr int kFusedStep = 8 * 64 * 8;  // elements of one chunk a thread of the register form's workgroup

// The widest of a chunk's elements, as the bits of a float.
template <class T>
__device__ __forceinline__ uint32_t widest(const u32x4& v, uint32_t top) {
  if constexpr (sizeof(typename T::raw_t) == 2) {
    // Of 16-bit numbers, too, magnitudes order as integers; two at a time.
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    u16x2 t = __builtin_bit_cast(u16x2, v[0] & 0x7fff7fffu);
#pragma unroll
    for (int i = 1; i < 4; ++i) t = __builtin_elementwise_max(t, __builtin_bit_cast(u16x2, v[i] & 0x7fff7fffu));
    return max(top, abs_bits(T::to_f32(max(t[0], t[1]))));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) top = max(top, v[i] & 0x7fffffffu);
    return top;
  }
}

// R rows a workgroup (of one band); lane l has row l % R and chunks of 16
// columns.  With two rows, two lanes write 32 bytes side by side, and a wave
// reads 1 KB of each row.  KEEP chunks stay in registers, what a row has more of
// is read twice.  Bound by bytes, 2 in and 1 out an element, and nearly as much
// by its arithmetic: 4075 rows of 4096 13.8 us, 3.6 TB/s, and 11.1 within a call,
// whose workspace the last-level cache holds; 1088 of 14336, one a workgroup of
// 16 waves, 15.8.  Rows that are not aligned are read an element at a time, each
// load behind a branch of its own and waited for: 333 of 1111 4.8 us.
template <class T, int R, int NW, int KEEP, bool AL>
__global__ __launch_bounds__(NW * 64) void quantize_rows_kernel(QuantArgs a) {
  using raw = typename T::raw_t;
  constexpr int V = 16 / T::VEC;              // 16-byte loads of a chunk
  constexpr int STEP = NW * (64 / R) * 16;    // columns of all waves
  __shared__ uint32_t tops[NW][R];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // Workgroups go to the eight XCDs in turn; those of a band take places of one
  // XCD, whose L2 puts together the lines that they share.
  constexpr int PER = 16 / R;
  int id = blockIdx.x;
  if (id < static_cast<int>(gridDim.x) / (8 * PER) * (8 * PER)) {
    const int at = id >> 3;
    id = (at / PER * 8 + (id & 7)) * PER + at % PER;
  }
  const int row = id * R + lane % R;
  const raw* x = static_cast<const raw*>(a.x) + static_cast<int64_t>(min(row, a.rows - 1)) * a.x_stride;
  const int padded = static_cast<int>(int8_padded(a.k));
  const int e0 = (wave * (64 / R) + lane / R) * 16;
  auto load = [&](int e, u32x4 (&v)[V]) {
#pragma unroll
    for (int h = 0; h < V; ++h)
      v[h] = load_row_chunk<T, AL>(x, e + h * T::VEC, min(max(a.k - e - h * T::VEC, 0), static_cast<int>(T::VEC)));
  };
  u32x4 keep[KEEP][V];
  uint32_t top = 0;
#pragma unroll
  for (int c = 0; c < KEEP; ++c) load(e0 + c * STEP, keep[c]);
#pragma unroll
  for (int c = 0; c < KEEP; ++c)
#pragma unroll
    for (int h = 0; h < V; ++h) top = widest<T>(keep[c][h], top);
  for (int e = e0 + KEEP * STEP; e < a.k; e += STEP) {
    u32x4 v[V];
    load(e, v);
#pragma unroll
    for (int h = 0; h < V; ++h) top = widest<T>(v[h], top);
  }
#pragma unroll
  for (int off = R; off < 64; off <<= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), off, kWave)));
  if (lane < R) tops[wave][lane] = top;
  lds_barrier();
#pragma unroll
  for (int w = 0; w < NW; ++w) top = max(top, tops[w][lane % R]);
  if (row >= a.rows) return;
  const RowScale s = row_scale(top);
  if (threadIdx.x < R) a.scales[row] = s.scale;
  const int64_t step = int8_bands(a.rows) * kInt8Block;
  int8_t* out = a.codes + static_cast<int64_t>(row >> 4) * kInt8Block + (row & 15) * 16;
  auto put = [&](int e, const u32x4 (&v)[V]) {
    if (e >= padded) return;
    uint32_t q[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) q[i] = code_of(chunk_elem<T>(v[i / T::VEC], i % T::VEC), s);
    st_chunk(out + (e >> 6) * step + (e >> 4 & 3) * 256, u32x4{pack4(q), pack4(q + 4), pack4(q + 8), pack4(q + 12)});
  };
#pragma unroll
  for (int c = 0; c < KEEP; ++c) put(e0 + c * STEP, keep[c]);
  for (int e = e0 + KEEP * STEP; e < padded; e += STEP) {
    u32x4 v[V];
    load(e, v);
    put(e, v);
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
    y[i] = scaled(sum[i], as, a.b_scales[c]);
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
// waves take the blocks of the bands in turn, straight from memory into
// operands, and add their sums in LDS: no barrier while weights stream.
// KEEP: the rows themselves (of at most KEEP chunks of eight elements a thread)
// are read and quantised by every workgroup, while its first blocks are on
// their way.  Near the weight's bytes where columns fill the chip: 64 rows to
// 28672 of them, K 4096 (117 MB), 27.6 to 28.6 us, 4.1 to 4.3 TB/s.  What keeps
// it from a copy's 5.1: the compiler puts a trip's reloads behind its last
// product, which has waited for all loads before, so that nothing is on its way
// then.  One row to 4096 columns 5.7, of which the bytes need 3.3; the rest is a
// launch's chain and the columns' scales, which are loaded after the products.
// Few columns leave CUs idle and long rows make long trips, since K is not
// split over workgroups: 32 rows to 1024 columns 3.2 us (bytes 0.8), of K 14336
// to 4096 columns 15.8 (11.5), 64 rows 19.3.
template <class T, int MT, int NT, int NW, int U, int KEEP>
__global__ __launch_bounds__(NW * 64) void int8_rows_kernel(Int8Args a) {
  using raw = typename T::raw_t;
  constexpr bool FUSE = KEEP > 0;
  extern __shared__ __align__(16) char lds[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = blockIdx.x * 16 * NT;
  const int m0 = blockIdx.y * 16 * MT;
  const int padded = static_cast<int>(int8_padded(a.k));
  const int pieces = padded / 64;

  const int8_t* wp[NT];
  const int8_t* xp[MT];
#pragma unroll
  for (int t = 0; t < NT; ++t)
    wp[t] = a.b + static_cast<int64_t>(min(n0 / 16 + t, (a.n - 1) / 16)) * kInt8Block + lane * 16;
  if constexpr (!FUSE) {
#pragma unroll
    for (int t = 0; t < MT; ++t)
      xp[t] = a.a + static_cast<int64_t>(min(m0 / 16 + t, (a.m - 1) / 16)) * kInt8Block + lane * 16;
  }
  u32x4 wf[U][NT], xf[U][MT];
  auto load = [&](int u, int piece) {
    const int64_t p = min(piece, pieces - 1);
#pragma unroll
    for (int t = 0; t < NT; ++t) wf[u][t] = ld_chunk(wp[t] + p * a.b_step);
    if constexpr (!FUSE) {
#pragma unroll
      for (int t = 0; t < MT; ++t) xf[u][t] = ld_chunk(xp[t] + p * a.a_step);
    }
  };
#pragma unroll
  for (int u = 0; u < U; ++u) load(u, wave + u * NW);

  // The workgroup's rows as codes in LDS, in the order of blocks of m rows: the
  // 16 bytes at 16 (m c + r) are those of row r and columns 16 c on.
  uint32_t* tops = reinterpret_cast<uint32_t*>(lds);
  int8_t* codes = reinterpret_cast<int8_t*>(lds) + 64;
  if constexpr (FUSE) {
    static_assert(MT == 1, "one band of rows");
    if (threadIdx.x < 16) tops[threadIdx.x] = 0;
    lds_barrier();
    const int chunks = padded / 8;
    float keep[KEEP][8];
#pragma unroll
    for (int c = 0; c < KEEP; ++c) {
      const int i = c * NW * 64 + threadIdx.x;
      const int r = i / chunks;
      if (r >= a.m) continue;
      const raw* x = static_cast<const raw*>(a.x) + r * a.x_stride;
      if (a.x_aligned) load8<T, true>(x, (i - r * chunks) * 8, a.k, keep[c]);
      else load8<T, false>(x, (i - r * chunks) * 8, a.k, keep[c]);
    }
#pragma unroll
    for (int c = 0; c < KEEP; ++c) {
      const int i = c * NW * 64 + threadIdx.x;
      const int r = i / chunks;
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max(top, r < a.m ? abs_bits(keep[c][e]) : 0u);
      // A row has at least 16 chunks: groups of 16 lanes have one row each.
#pragma unroll
      for (int off = 1; off < 16; off <<= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), off, kWave)));
      if ((lane & 15) == 0 && r < a.m) atomicMax(&tops[r], top);
    }
    lds_barrier();
#pragma unroll
    for (int c = 0; c < KEEP; ++c) {
      const int i = c * NW * 64 + threadIdx.x;
      const int r = i / chunks;
      if (r >= a.m) continue;
      const int e = i - r * chunks;
      const RowScale s = row_scale(tops[r]);
      uint32_t q[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) q[j] = code_of(keep[c][j], s);
      *reinterpret_cast<uint2*>(codes + ((e >> 1) * a.m + r) * 16 + (e & 1) * 8) = make_uint2(pack4(q), pack4(q + 4));
    }
    lds_barrier();
  }
  const int8_t* xl = codes + ((lane >> 4) * a.m + min(lane & 15, a.m - 1)) * 16;

  i32x4 acc[NT][MT];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[n][m] = i32x4{0, 0, 0, 0};
  auto multiply = [&](int u, int p) {
    if constexpr (FUSE) xf[u][0] = *reinterpret_cast<const u32x4*>(xl + p * 64 * a.m);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int m = 0; m < MT; ++m)
        acc[n][m] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, wf[u][n]), __builtin_bit_cast(i32x4, xf[u][m]),
                                                          acc[n][m], 0, 0, 0);
  };
  int p = wave;
  for (; p + U * NW < pieces; p += U * NW)
#pragma unroll
    for (int u = 0; u < U; ++u) {
      multiply(u, p + u * NW);
      load(u, p + (u + U) * NW);
    }
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (p + u * NW < pieces) multiply(u, p + u * NW);
  // Lane l has row l & 15 of a band's m and 4 (l >> 4) to + 3 of its n.
  const int col = lane & 15;
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
    const int n = n0 + (t / MT) * 16 + (lane >> 4) * 4;
    const int m = m0 + (t % MT) * 16 + col;
    if (m < a.m && n < a.n) store4<T>(a, m, n, sum, FUSE ? row_scale(mine).scale : a.a_scales[m]);
  }
}

template <class T, int MT, int NT, int NW, int U, int KEEP>
hipError_t launch_rows(const Int8Args& a, hipStream_t stream) {
  const int codes = KEEP > 0 ? 64 + a.m * static_cast<int>(int8_padded(a.k)) : 0;
  const int bytes = std::max(codes, NW * NT * MT * 64 * 16);  // at most 64 KB
  const auto kernel = int8_rows_kernel<T, MT, NT, NW, U, KEEP>;
  const dim3 grid(cdiv(a.n, 16 * NT), cdiv(a.m, 16 * MT));
  if (!grid_fits(2 * static_cast<int64_t>(grid.x))) return hipErrorInvalidConfiguration;
  hipLaunchKernelGGL(kernel, grid, dim3(NW * 64), bytes, stream, a);
  return hipGetLastError();
}

// Rows of a workgroup of the register form, and its columns, in bands: as many
// products as give the chip kFew workgroups, since every band is read anew by
// each workgroup that uses it.  Times in us (K 4096; in a graph, weights cold):
// 64 rows to 4096 columns 5.8 with 2 x 2 bands (256 workgroups), 7.1 with 2 x 4,
// 7.2 with 2 x 1; 128 rows 7.1 with 2 x 4, 8.0 with 2 x 2; 256 rows 10.3 with
// 4 x 4, 10.9 with 2 x 4; 16 rows to 28672 22.4 with 1 x 4, 24.3 with 1 x 1.
constexpr int kFew = 192;
// The register form's loads grow with the rows, and tiles from LDS take over
// where there are more workgroups of 4 x 4 bands than this: 512 rows to 4096
// columns (512 of them) 16.2 against 18.6, and with K 14336 52 against 76; to
// 6144 (768) 24.9 against 22.1; 128 rows to 28672 (896) 44.3 against 34.3.
constexpr int kRegisterTiles = 512;

template <class T>
hipError_t launch(const Int8Args& a, int cus, hipStream_t stream) {
  auto tiles = [&](int tn, int tm) { return static_cast<int64_t>(cdiv(a.n, tn)) * cdiv(a.m, tm); };
  if (a.a == nullptr) {
    // One or two chunks a thread; one band of columns, or four where they fill the chip all the same.
    const bool wide = tiles(64, 16) >= kFew, one = int8_padded(a.k) * a.m <= kFusedStep;
    if (wide) return one ? launch_rows<T, 1, 4, 8, 2, 1>(a, stream) : launch_rows<T, 1, 4, 8, 2, 2>(a, stream);
    return one ? launch_rows<T, 1, 1, 8, 2, 1>(a, stream) : launch_rows<T, 1, 1, 8, 4, 2>(a, stream);
  }
  if (tiles(64, 64) <= kRegisterTiles) {
    if (a.m > 32 && tiles(64, 64) >= kFew) return launch_rows<T, 4, 4, 4, 2, 0>(a, stream);
    if (a.m > 16 && tiles(64, 32) >= kFew) return launch_rows<T, 2, 4, 8, 2, 0>(a, stream);
    if (a.m <= 16 && tiles(64, 16) >= kFew) return launch_rows<T, 1, 4, 8, 2, 0>(a, stream);
    if (a.m > 16 && tiles(32, 32) >= kFew) return launch_rows<T, 2, 2, 8, 2, 0>(a, stream);
    if (tiles(32, 16) >= kFew) return launch_rows<T, 1, 2, 8, 4, 0>(a, stream);
    return launch_rows<T, 1, 1, 8, 2, 0>(a, stream);
  }
  // Tiles: the shape whose rounds over the chip take least, by what a step of a
  // round takes (in hundredths of a us, over all of the CUs; two workgroups of
  // 128 x 128 share a CU).  4075 rows to 6144 columns 98 us with 192 x 256 (2
  // rounds), 104 with 128 x 128 (6), 110 with 256 x 256 (1.5, so 2); 512 to 28672
  // 63 with 256 x 256 (1), 80 with 128 x 128 (3.5); 2048 to 4096 37 with 128 x 128
  // (2), 45 with 192 x 256 (1), 54 with 256 x 256 (1).
  auto rounds = [&](int tn, int tm) { return (tiles(tn, tm) + cus - 1) / cus; };
  const int64_t small = rounds(128, 128) == 1 ? 80 : 60 * rounds(128, 128);
  const int64_t middle = 154 * rounds(192, 256), large = 187 * rounds(256, 256);
  if (small <= middle && small <= large) return launch_tile<T, TileShape<128, 128, 4, 2, 2>>(a, stream);
  if (middle <= large) return launch_tile<T, TileShape<192, 256, 2, 4, 2>>(a, stream);
  return launch_tile<T, TileShape<256, 256, 2, 4, 2>>(a, stream);
}

template <class T, int R, int NW, int KEEP>
hipError_t launch_quant(const QuantArgs& a, bool aligned, hipStream_t stream) {
  const int64_t blocks = (static_cast<int64_t>(a.rows) + R - 1) / R;
  if (!grid_fits(blocks * (NW / 4))) return hipErrorInvalidConfiguration;
  const dim3 grid(static_cast<unsigned>(blocks));
  if (aligned) hipLaunchKernelGGL((quantize_rows_kernel<T, R, NW, KEEP, true>), grid, dim3(NW * 64), 0, stream, a);
  else hipLaunchKernelGGL((quantize_rows_kernel<T, R, NW, KEEP, false>), grid, dim3(NW * 64), 0, stream, a);
  return hipGetLastError();
}

template <class T>
hipError_t quant_of(const QuantArgs& a, bool aligned, hipStream_t stream) {
  // Times in us: 1088 rows of 14336 15.8 with one row a workgroup, 17.3 with two,
  // 18.5 with four; 2048 of 8192 17.2, 14.3 and 14.3; 4075 of 4096 17.1, 13.8 and
  // 14.0; 450 of 4096 3.5, 3.3 and 4.1; 64 of 14336 3.9, 4.5 and 8.0; 600 of 1024
  // 2.8, 3.1 and 2.8.
  if (a.rows < kQuantMany || a.k > 8192)
    return a.k <= 4096 ? launch_quant<T, 1, 4, 1>(a, aligned, stream) : launch_quant<T, 1, 16, 1>(a, aligned, stream);
  if (a.k <= 1024) return launch_quant<T, 4, 4, 1>(a, aligned, stream);
  return a.k <= 4096 ? launch_quant<T, 2, 8, 1>(a, aligned, stream) : launch_quant<T, 2, 8, 2>(a, aligned, stream);
}

}  // namespace

// Quantising inside the product's launch saves the other one's 3.3 us and costs
// every workgroup the rows: one row of 4096 5.8 to 6.0 us against 8.0, two 7.0
// against 8.1, but four 8.9 against 8.1, and one of 14336 16.3 against 16.0.
bool int8_fused(int m, int k) { return m <= 8 && m * int8_padded(k) <= 2 * kFusedStep; }

hipError_t launch_quantize_rows(const QuantArgs& a, int dtype, bool aligned, hipStream_t stream) {
  if (a.rows == 0) return hipSuccess;
  if (dtype == MLORA_BF16) return quant_of<BF16>(a, aligned, stream);
  if (dtype == MLORA_F16) return quant_of<F16>(a, aligned, stream);
  return launch_quant<F32, 4, 4, 1>(a, aligned, stream);
}

hipError_t launch_int8_matmul(const Int8Args& a, int dtype, int cus, hipStream_t stream) {
  if (a.m == 0 || a.n == 0) return hipSuccess;
  return dtype == MLORA_BF16 ? launch<BF16>(a, cus, stream) : launch<F16>(a, cus, stream);
}

}  // namespace mlora
