// Products of many quantised rows: tiles on the matrix units (csrc/int8.hip).
#pragma once

#include "int8.h"
#include "kernels.h"
#include "loads.h"

namespace mlora {

namespace {

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef const __attribute__((address_space(1))) void gvoid_t;
typedef __attribute__((address_space(3))) void lvoid_t;

// A sum (below 2^31) times a row's scale and a channel's, the channel's first
// unless that could leave fp32 where the result does not.  (Scales go from 2^-107
// to 2^121.)
constexpr float kFarScale = 0x1p96f;
__device__ __forceinline__ float scaled(int32_t sum, float row, float channel) {
  const bool far = channel > kFarScale;
  return static_cast<float>(sum) * (far ? row : channel) * (far ? channel : row);
}

// A tile's shape: TN weight rows by TM rows, waves WN by WM, S steps in LDS.  A
// step is two blocks (2 KB) of each band.
template <int TN_, int TM_, int WN_, int WM_, int S_>
struct TileShape {
  static constexpr int TN = TN_, TM = TM_, WN = WN_, WM = WM_, S = S_;
  static constexpr int NW = WN * WM;
  static constexpr int FN = TN / WN / 16, FM = TM / WM / 16;  // bands of a wave
  static constexpr int BLOCKS = (TN + TM) / 8;                // of a step
  static constexpr int LOADS = BLOCKS / NW;                   // of a wave
  static constexpr int EARLY = (LOADS + 1) / 2;               // of them in the second half of a step, the others in the next one's first
  static constexpr int STAGE = BLOCKS * kInt8Block;
  static constexpr int PITCH = TN * 2 + 16;                   // of a row of the result: 16 bytes more, so that rows begin in different banks
  static constexpr int OUT = TM * PITCH;
  static constexpr int BYTES = S * STAGE > OUT ? S * STAGE : OUT;
  static_assert(FN * WN * 16 == TN && FM * WM * 16 == TM && LOADS * NW == BLOCKS, "whole bands and loads a wave");
};

template <class Sh>
struct TileShared {
  __attribute__((aligned(16))) char stage[Sh::BYTES];
  float scale[Sh::TN], bias[Sh::TN];
};

// Tile of workgroup `id` of `tiles_n * tiles_m`.  Workgroups go to the eight
// XCDs in turn; each XCD gets a run of neighbouring tiles, in bands of 4 rows
// of tiles, so that its L2 holds what the tiles share.
__device__ __forceinline__ void pick_tile8(int id, int tiles_n, int tiles_m, int* tn, int* tm) {
  const int total = tiles_n * tiles_m;
  const int per = total >> 3, more = total & 7;
  const int xcd = id & 7, at = id >> 3;
  const int t = xcd * per + min(xcd, more) + at;
  const int band = t / (4 * tiles_n);
  const int rows = min(4, tiles_m - band * 4);
  const int in = t - band * 4 * tiles_n;
  *tn = in / rows;
  *tm = band * 4 + in - *tn * rows;
}

// A tile over K, 128 bytes of each row a step: blocks are loaded straight into
// one of S places in LDS, S - 1 steps ahead, and lie there as they do in memory,
// so that a fragment is one 16-byte load a lane from neighbouring addresses.
// The fragments of the next 64 bytes are read, and loads sent, while this
// one's products run.  Bound by the matrix units at the clock that this load
// allows (1.9 GHz; they are busy in 48 to 55 % of the cycles) and by the loads'
// issue between them: 4075 rows to 6144 columns, K 4096, 95.2 us, 2150 TOP/s
// (replayed from a graph; 113 under a profiler), where a library product without
// scales takes 102 to 103; 8192^3 450 us, 2440 TOP/s (443 to 446).  Three or four
// places in LDS, steps of 64 bytes and groups of waves that share K were no
// faster.
template <class T, class Sh>
__global__ __launch_bounds__(Sh::NW * 64) void int8_tile_kernel(Int8Args a, int tiles_n, int tiles_m) {
  using raw = typename T::raw_t;
  constexpr int TN = Sh::TN, TM = Sh::TM, FN = Sh::FN, FM = Sh::FM, S = Sh::S, STAGE = Sh::STAGE;
  constexpr int LOADS = Sh::LOADS, EARLY = Sh::EARLY, NW = Sh::NW;
  __shared__ TileShared<Sh> s;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int steps = static_cast<int>(int8_padded(a.k)) / 128;
  int tile_n, tile_m;
  pick_tile8(blockIdx.x, tiles_n, tiles_m, &tile_n, &tile_m);
  const int n0 = tile_n * TN, m0 = tile_m * TM;
  const int last_n = (a.n - 1) / 16, last_m = (a.m - 1) / 16;  // bands

  // Block b of a step: half b & 1 of band b >> 1 of the weight's tile, then of the other.
  const int8_t* from[LOADS];
  auto block = [&](int i) { return wave * LOADS + i; };
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const int b = block(i), band = b >> 1;
    from[i] = (band < TN / 16 ? a.b + static_cast<int64_t>(min(n0 / 16 + band, last_n)) * kInt8Block + (b & 1) * a.b_step
                              : a.a + static_cast<int64_t>(min(m0 / 16 + band - TN / 16, last_m)) * kInt8Block + (b & 1) * a.a_step) +
              lane * 16;
  }
  // Block i of step `st`, and on to the next (behind the last one, that is loaded again).
  auto load = [&](int i, int st, int to) {
    __builtin_amdgcn_global_load_lds((gvoid_t*)from[i], (lvoid_t*)(s.stage + to + block(i) * kInt8Block), 16, 0, 0);
    from[i] += st + 1 < steps ? 2 * (block(i) < TN / 8 ? a.b_step : a.a_step) : 0;
  };
#pragma unroll
  for (int st = 0; st < S; ++st)
#pragma unroll
    for (int i = 0; i < (st + 1 < S ? LOADS : EARLY); ++i) load(i, st, st * STAGE);
  for (int i = threadIdx.x; i < TN; i += NW * 64) {
    const int n = min(n0 + i, a.n - 1);
    s.scale[i] = a.b_scales[n];
    s.bias[i] = a.bias != nullptr ? T::to_f32(static_cast<const raw*>(a.bias)[n]) : 0.f;
  }
  const int wn = wave % Sh::WN, wm = wave / Sh::WN;
  const char* nb = s.stage + wn * FN * 2 * kInt8Block + lane * 16;
  const char* mb = s.stage + (TN / 16 + wm * FM) * 2 * kInt8Block + lane * 16;
  i32x4 acc[FN][FM];
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int j = 0; j < FM; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
  i32x4 nf[2][FN], mf[2][FM];
  auto read = [&](int k, int at) {
#pragma unroll
    for (int i = 0; i < FN; ++i) nf[k][i] = *reinterpret_cast<const i32x4*>(nb + at + (i * 2 + k) * kInt8Block);
#pragma unroll
    for (int j = 0; j < FM; ++j) mf[k][j] = *reinterpret_cast<const i32x4*>(mb + at + (j * 2 + k) * kInt8Block);
    __builtin_amdgcn_sched_barrier(0);
  };
  // Products of a half, with the loads [first, end) of step `st` between them.
  auto multiply = [&](int k, int first, int end, int st, int to) {
    constexpr int P = FN * FM;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int i = p / FM, j = p - i * FM;
      acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(nf[k][i], mf[k][j], acc[i][j], 0, 0, 0);
      if (first < end) {
        const int before = p * (end - first) / P, upto = (p + 1) * (end - first) / P;
#pragma unroll
        for (int l = before; l < upto; ++l) load(first + l, st, to);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  wait_vmcnt<(S - 2) * LOADS + EARLY>();  // (the scales' loads, issued later, are waited for by their use)
  lds_barrier();
  read(0, 0);
  // No branch inside a step: the waits before products are then for their own
  // fragments only.
  int at = 0, last = (S - 1) * STAGE;  // places of this step, and of the last one whose loads have begun
  for (int st = 0; st + 1 < steps; ++st) {
    read(1, at);
    multiply(0, EARLY, LOADS, st + S - 1, last);
    // The step's fragments are in registers and the next one has landed, for every wave after the barrier.
    wait_vmcnt<(S - 2) * LOADS>();
    lds_barrier();
    last = at;
    at = at == (S - 1) * STAGE ? 0 : at + STAGE;
    read(0, at);
    multiply(1, 0, EARLY, st + S, last);
  }
  read(1, at);
  multiply(0, 0, 0, 0, 0);
  multiply(1, 0, 0, 0, 0);
  wait_vmcnt<0>();
  lds_barrier();
  // Lane l has row l & 15 of a band's m and 4 (l >> 4) to + 3 of its n.  The
  // result goes through LDS, so that a row is stored whole.
  float as[FM];
#pragma unroll
  for (int j = 0; j < FM; ++j) as[j] = a.a_scales[min(m0 + (wm * FM + j) * 16 + (lane & 15), a.m - 1)];
#pragma unroll
  for (int i = 0; i < FN; ++i) {
    const int n = (wn * FN + i) * 16 + (lane >> 4) * 4;
    const f32x4 bs = *reinterpret_cast<const f32x4*>(&s.scale[n]), bias = *reinterpret_cast<const f32x4*>(&s.bias[n]);
    const bool far = __any(fmaxf(fmaxf(bs[0], bs[1]), fmaxf(bs[2], bs[3])) > kFarScale);
#pragma unroll
    for (int j = 0; j < FM; ++j) {
      const int m = (wm * FM + j) * 16 + (lane & 15);
      float y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = static_cast<float>(acc[i][j][e]) * bs[e] * as[j];
      if (far) {
        asm volatile("");  // (stays a branch)
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = scaled(acc[i][j][e], as[j], bs[e]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (a.bias != nullptr) y[e] += bias[e];
      *reinterpret_cast<uint2*>(s.stage + m * Sh::PITCH + n * 2) = make_uint2(T::pack2(y[0], y[1]), T::pack2(y[2], y[3]));
    }
  }
  lds_barrier();
  constexpr int C = TN / 8;  // chunks of eight columns
  for (int i = threadIdx.x; i < TM * C; i += NW * 64) {
    const int m = i / C, c = i - m * C;
    const int n = n0 + c * 8;
    if (m0 + m >= a.m || n >= a.n) continue;
    const u32x4 v = *reinterpret_cast<const u32x4*>(s.stage + m * Sh::PITCH + c * 16);
    raw* out = static_cast<raw*>(a.out) + static_cast<int64_t>(m0 + m) * a.out_stride + n;
    if (a.wide) {
      store_row_chunk<T, true>(out, v, a.n - n);
    } else if (a.vec && n + 8 <= a.n) {  // rows that begin at multiples of 8 bytes only
      *reinterpret_cast<uint2*>(out) = make_uint2(v[0], v[1]);
      *reinterpret_cast<uint2*>(out + 4) = make_uint2(v[2], v[3]);
    } else {
      store_row_chunk<T, false>(out, v, a.n - n);
    }
  }
}

template <class T, class Sh>
hipError_t launch_tile(const Int8Args& a, hipStream_t stream) {
  const int64_t tn = (static_cast<int64_t>(a.n) + Sh::TN - 1) / Sh::TN, tm = (static_cast<int64_t>(a.m) + Sh::TM - 1) / Sh::TM;
  if (!grid_fits(tn * tm * (Sh::NW / 4))) return hipErrorInvalidConfiguration;
  hipLaunchKernelGGL((int8_tile_kernel<T, Sh>), dim3(static_cast<unsigned>(tn * tm)), dim3(Sh::NW * 64), 0, stream, a,
                     static_cast<int>(tn), static_cast<int>(tm));
  return hipGetLastError();
}

}  // namespace

}  // namespace mlora
