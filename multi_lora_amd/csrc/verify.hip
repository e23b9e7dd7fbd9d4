// Verification of drafted tokens against the target's probabilities (gfx950).
//
// Request i has rows [row_indptr[i], row_indptr[i + 1]) of `target`, one more
// than it has drafts x_0 .. x_{k-1}.  Draft j is accepted while
// u_j * q_j(x_j) < p_j(x_j).  The token after the accepted ones is drawn from
// max(p_j - q_j, 0) at the first rejection j (certain drafts: q is 1 at x_j,
// 0 elsewhere), from p_k after k acceptances: the lowest x whose cumulated
// mass exceeds w times the row's mass.  Products, sums and cumulated sums are
// fp64 and always added in the same order: an answer repeats, and differs from
// that of adding column by column only where w times the mass is within some
// vocab * 2^-53 of it of a column's border.  Mass that is not positive (NaN
// too) counts as none; a residual without mass falls back to p_j, and a row
// without mass has no answer (-1).
//
// Two launches, for one row's sums are needed before its draw: a workgroup
// per 2048 columns of a request's row, which finds the row itself, then a
// workgroup per request that reads the one chunk its draw falls in.  Rows of
// up to 4096 columns are one launch, bound by its chain of reads: 5.3 us for
// one request.  Thirty-two requests of 128,256 fp32 columns (31.8 MB with the
// drafts' rows) take 8.5 us for the sums, 3.7 TB/s, and 4.7 us for the draw
// (averages).
#include "kernels.h"
#include "loads.h"
#include "paged.h"

namespace mlora {

namespace {

struct Row {
  int accepted;   // drafts accepted; the row drawn from is the accepted-th
  bool rejected;  // a draft stands at that row
  int64_t token;  // that draft
  bool live;      // the request has rows in this call
};

// Every wave finds the row for itself, 64 drafts at a time.  The drafts and
// their numbers are asked for together with the row numbers, the two
// probabilities together: two round trips to memory, not four.
template <class T>
__device__ Row find_row(const VerifyArgs& a, int i) {
  using raw = typename T::raw_t;
  const int lane = threadIdx.x & 63;
  int64_t x = lane < a.most ? a.tokens[i * a.token_stride + lane] : -1;
  float u = lane < a.most ? a.accept[i * a.accept_stride + lane] : 0.f;
  const int first = min(max(a.row_indptr[i], 0), a.rows);
  const int end = min(max(a.row_indptr[i + 1], first), a.rows);
  const int k = min(end - first - 1, a.most);
  Row r{0, false, -1, end > first};
  for (int j0 = 0; j0 < k; j0 += kWave) {
    const int j = j0 + lane;
    if (j0 > 0 && j < k) {
      x = a.tokens[i * a.token_stride + j];
      u = a.accept[i * a.accept_stride + j];
    }
    bool no = false;
    if (j < k) {
      no = true;
      if (x >= 0 && x < a.vocab) {
        const raw p = static_cast<const raw*>(a.target)[(first + j) * a.target_stride + x];
        const raw q = a.draft == nullptr
                          ? raw{}
                          : static_cast<const raw*>(a.draft)[i * a.draft_stride0 + j * a.draft_stride1 + x];
        const double qd = a.draft == nullptr ? 1.0 : static_cast<double>(T::to_f32(q));
        no = !(static_cast<double>(u) * qd < static_cast<double>(T::to_f32(p)));
      }
    }
    const uint64_t hit = __ballot(no);
    if (hit != 0) {
      const int l = __ffsll(static_cast<unsigned long long>(hit)) - 1;
      r.accepted = j0 + l;
      r.rejected = true;
      r.token = __shfl(x, l, kWave);
      return r;
    }
  }
  r.accepted = max(k, 0);
  return r;
}

// Mass of column x of the row drawn from: of the residual, and of p.
template <class T>
__device__ __forceinline__ void column(const Row& r, typename T::raw_t p, bool has_q, typename T::raw_t q, int x,
                                       double* rest, double* full) {
  const float f = T::to_f32(p);
  *full = f > 0.f ? static_cast<double>(f) : 0.0;
  if (!r.rejected) {
    *rest = *full;
  } else if (has_q) {
    const double less = static_cast<double>(f) - static_cast<double>(T::to_f32(q));
    *rest = less > 0.0 ? less : 0.0;
  } else {
    *rest = x == r.token ? 0.0 : *full;
  }
}

template <class T>
__device__ __forceinline__ void row_ptrs(const VerifyArgs& a, const Row& r, int i, const typename T::raw_t** p,
                                         const typename T::raw_t** q) {
  using raw = typename T::raw_t;
  const int first = min(max(a.row_indptr[i], 0), a.rows);
  *p = static_cast<const raw*>(a.target) + static_cast<int64_t>(first + r.accepted) * a.target_stride;
  *q = r.rejected && a.draft != nullptr
           ? static_cast<const raw*>(a.draft) + i * a.draft_stride0 + r.accepted * a.draft_stride1
           : nullptr;
}

// Inclusive sum over the wave's lanes, by the data-parallel moves of a row of
// 16 lanes and of rows to the next ones (a lane without a source gets 0).  An
// exchange through the LDS crossbar instead waits for it twelve times a sum.
template <int CTRL, int ROWS>
__device__ __forceinline__ double moved(double v) {
  const unsigned long long b = __builtin_bit_cast(unsigned long long, v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(b & 0xffffffffu), CTRL, ROWS, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(b >> 32), CTRL, ROWS, 0xf, false);
  return __builtin_bit_cast(double, static_cast<unsigned long long>(hi) << 32 | lo);
}
__device__ __forceinline__ double wave_incl_sum(double v) {
  v += moved<0x111, 0xf>(v);  // row_shr:1
  v += moved<0x112, 0xf>(v);  // row_shr:2
  v += moved<0x114, 0xf>(v);  // row_shr:4
  v += moved<0x118, 0xf>(v);  // row_shr:8
  v += moved<0x142, 0xa>(v);  // the last lane of rows 0 and 2 to rows 1 and 3
  v += moved<0x143, 0xc>(v);  // lane 31 to the upper two rows
  return v;
}

template <class T>
__global__ __launch_bounds__(256) void verify_sum_kernel(VerifyArgs a) {
  using raw = typename T::raw_t;
  constexpr int kPer = kVerifyChunk / 256;  // columns a thread
  const int i = blockIdx.x / a.chunks;
  const int c = blockIdx.x - i * a.chunks;
  const Row r = find_row<T>(a, i);
  if (c == 0 && threadIdx.x == 0) a.accepted[i] = r.accepted;
  if (!r.live) return;
  const raw *p, *q;
  row_ptrs<T>(a, r, i, &p, &q);
  // Every load is issued before the first is used; columns past the row's end
  // read its last one again and count nothing.
  raw pv[kPer], qv[kPer];
  const int x0 = c * kVerifyChunk + static_cast<int>(threadIdx.x);
#pragma unroll
  for (int e = 0; e < kPer; ++e) pv[e] = p[min(x0 + e * 256, a.vocab - 1)];
  if (q != nullptr) {
#pragma unroll
    for (int e = 0; e < kPer; ++e) qv[e] = q[min(x0 + e * 256, a.vocab - 1)];
  }
  double rest = 0.0, full = 0.0;
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    const int x = x0 + e * 256;
    double m, f;
    column<T>(r, pv[e], q != nullptr, qv[e], x, &m, &f);
    if (x < a.vocab) {
      rest += m;
      full += f;
    }
  }
  rest = wave_incl_sum(rest);
  full = wave_incl_sum(full);
  __shared__ double part[4][2];
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == kWave - 1) {
    part[wave][0] = rest;
    part[wave][1] = full;
  }
  __syncthreads();
  if (threadIdx.x < 2)
    a.sums[static_cast<int64_t>(blockIdx.x) * 2 + threadIdx.x] =
        part[0][threadIdx.x] + part[1][threadIdx.x] + part[2][threadIdx.x] + part[3][threadIdx.x];
}

// Workgroup = request.  ONE: the row is a single chunk, and this is the only
// launch.  Its time is the chain of what it reads; the waves find the chunk
// each for itself, and meet twice over its columns.
// Four columns a thread: with eight, on 256 and 512 threads, 0.9 us more (2.4
// where a thread has sixteen); two, on 1024 for a chunk, 0.4 more.
constexpr int kDrawColumns = 4;
constexpr int draw_threads(bool one) { return (one ? kVerifyOne : kVerifyChunk) / kDrawColumns; }
template <class T, bool ONE>
__global__ __launch_bounds__(draw_threads(ONE)) void verify_draw_kernel(VerifyArgs a) {
  using raw = typename T::raw_t;
  constexpr int kPer = kDrawColumns;
  constexpr int kThreads = draw_threads(ONE);
  constexpr int kWaves = kThreads / kWave;
  __shared__ double part[kWaves][2];
  __shared__ int hit_s[kWaves], last_s[kWaves];
  const int i = blockIdx.x;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;
  const float last_u = a.last[i];
  int chunk = 0, use = 0;
  double before = 0.0, want = 0.0;
  Row r;
  if constexpr (ONE) {
    r = find_row<T>(a, i);
  } else {
    // The chunk that the draw falls in; a lane takes `per` neighbouring ones.
    const double* sums = a.sums + static_cast<int64_t>(i) * a.chunks * 2;
    const int per = (a.chunks + kWave - 1) / kWave;
    const int c0 = lane * per, c1 = min(c0 + per, a.chunks);
    double rest = 0.0, full = 0.0;
    for (int c = c0; c < c1; ++c) {
      rest += sums[c * 2];
      full += sums[c * 2 + 1];
    }
    const int first = min(max(a.row_indptr[i], 0), a.rows);
    const int end = min(max(a.row_indptr[i + 1], first), a.rows);
    r = Row{a.accepted[i], false, -1, end > first};  // from the first launch's count
    r.rejected = r.accepted < min(end - first - 1, a.most);
    if (r.rejected && a.draft == nullptr) r.token = a.tokens[i * a.token_stride + r.accepted];
    if (r.live) {
      const double rest1 = wave_incl_sum(rest), full1 = wave_incl_sum(full);
      const double total = __shfl(rest1, kWave - 1, kWave);
      use = total > 0.0 ? 0 : 1;
      want = static_cast<double>(last_u) * (use == 0 ? total : __shfl(full1, kWave - 1, kWave));
      double cum = use == 0 ? rest1 - rest : full1 - full;
      double here = 0.0;
      int hit = -1, last = -1;
      for (int c = c0; c < c1; ++c) {
        const double m = sums[c * 2 + use];
        if (m > 0.0) {
          last = c;
          if (hit < 0 && cum + m > want) {
            hit = c;
            here = cum;
          }
        }
        cum += m;
      }
      const uint64_t hits = __ballot(hit >= 0), lasts = __ballot(last >= 0);
      if (hits != 0) {
        const int l = __builtin_ctzll(hits);
        chunk = __shfl(hit, l, kWave);
        before = __shfl(here, l, kWave);
      } else if (lasts != 0) {  // a number of 1 or more: the last column with mass
        chunk = __shfl(last, 63 - __builtin_clzll(lasts), kWave);
        before = -INFINITY;
      } else {
        chunk = -1;
      }
    }
  }
  int64_t token = -1;  // of thread 0
  if (r.live && chunk >= 0) {
    const raw *p, *q;
    row_ptrs<T>(a, r, i, &p, &q);
    const int x0 = chunk * kVerifyChunk + tid * kPer;
    raw pv[kPer], qv[kPer];
#pragma unroll
    for (int e = 0; e < kPer; ++e) pv[e] = p[min(x0 + e, a.vocab - 1)];
    if (q != nullptr) {
#pragma unroll
      for (int e = 0; e < kPer; ++e) qv[e] = q[min(x0 + e, a.vocab - 1)];
    }
    double m[kPer], mine = 0.0, all = 0.0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      double rest, full;
      column<T>(r, pv[e], q != nullptr, qv[e], x0 + e, &rest, &full);
      m[e] = x0 + e < a.vocab ? (use ? full : rest) : 0.0;
      mine += m[e];
      if (ONE && x0 + e < a.vocab) all += full;
    }
    double incl = wave_incl_sum(mine), incl_all = ONE ? wave_incl_sum(all) : 0.0;
    if (lane == kWave - 1) {
      part[wave][0] = incl;
      part[wave][1] = incl_all;
    }
    __syncthreads();
    if constexpr (ONE) {
      double total = 0.0;
      for (int v = 0; v < kWaves; ++v) total += part[v][0];
      if (!(total > 0.0)) {  // nothing left of the residual: the target's row
        use = 1;
        total = 0.0;
        for (int v = 0; v < kWaves; ++v) total += part[v][1];
        incl = incl_all;
        mine = all;
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
          double rest;
          column<T>(r, pv[e], q != nullptr, qv[e], x0 + e, &rest, &m[e]);
          if (x0 + e >= a.vocab) m[e] = 0.0;
        }
      }
      want = static_cast<double>(last_u) * total;
    }
    double cum = before + (incl - mine);
    for (int v = 0; v < wave; ++v) cum += part[v][ONE ? use : 0];
    int hit = -1, last = -1;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      cum += m[e];
      if (m[e] > 0.0) {
        last = x0 + e;
        if (hit < 0 && cum > want) hit = x0 + e;
      }
    }
    const uint64_t hits = __ballot(hit >= 0), lasts = __ballot(last >= 0);
    const int first_hit = hits != 0 ? __shfl(hit, __builtin_ctzll(hits), kWave) : -1;
    const int last_mass = lasts != 0 ? __shfl(last, 63 - __builtin_clzll(lasts), kWave) : -1;
    if (lane == 0) {
      hit_s[wave] = first_hit;
      last_s[wave] = last_mass;
    }
    __syncthreads();
    // No hit where w is 1 or more, or where the chunk's own sum, added in another
    // order, says so within a rounding: the last column with mass.
    for (int v = 0; v < kWaves; ++v) token = max(token, static_cast<int64_t>(last_s[v]));
    for (int v = kWaves - 1; v >= 0; --v)
      if (hit_s[v] >= 0) token = hit_s[v];
  }
  int64_t* out = a.out + static_cast<int64_t>(i) * (a.most + 1);
  for (int j = tid; j <= a.most; j += kThreads)
    out[j] = !r.live ? -1 : j < r.accepted ? a.tokens[i * a.token_stride + j] : j == r.accepted ? token : -1;
  if (ONE && tid == 0) a.accepted[i] = r.accepted;
}

template <class T>
hipError_t launch(const VerifyArgs& a, hipStream_t stream) {
  const int64_t blocks = static_cast<int64_t>(a.n) * a.chunks;
  if (!grid_fits(blocks)) return hipErrorInvalidConfiguration;
  if (a.chunks == 1) {
    hipLaunchKernelGGL((verify_draw_kernel<T, true>), dim3(static_cast<unsigned>(a.n)), dim3(draw_threads(true)), 0, stream, a);
    return hipGetLastError();
  }
  hipLaunchKernelGGL((verify_sum_kernel<T>), dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((verify_draw_kernel<T, false>), dim3(static_cast<unsigned>(a.n)), dim3(draw_threads(false)), 0, stream, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_verify(const VerifyArgs& a, int dtype, hipStream_t stream) {
  if (a.n == 0) return hipSuccess;
  if (dtype == MLORA_F32) return launch<F32>(a, stream);
  return dtype == MLORA_BF16 ? launch<BF16>(a, stream) : launch<F16>(a, stream);
}

}  // namespace mlora
