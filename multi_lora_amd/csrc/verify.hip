// Verification of drafted tokens against the target's probabilities (gfx950).
//
// Request i has rows [row_indptr[i], row_indptr[i + 1]) of `target`, one more
// than it has drafts x_0 .. x_{k-1}.  Draft j is accepted while
// u_j * q_j(x_j) < p_j(x_j).  The token after the accepted ones is drawn from
// max(p_j - q_j, 0) at the first rejection j (certain drafts: q is 1 at x_j,
// 0 elsewhere), from p_k after k acceptances: the lowest x whose cumulated
// mass exceeds w times the row's mass.  Products, sums and cumulated sums are
// fp64, so a draw does not depend on how the row is cut.  Mass that is not
// positive (NaN too) counts as none; a residual without mass falls back to
// p_j, and a row without mass has no answer (-1).
//
// Two launches, for one row's sums are needed before its draw: a workgroup
// per 2048 columns of a request's row, which finds the row itself, then a
// workgroup per request that reads the one chunk its draw falls in.  Rows of
// up to 4096 columns are one launch.
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
  for (int off = 1; off < kWave; off <<= 1) {
    rest += __shfl_xor(rest, off, kWave);
    full += __shfl_xor(full, off, kWave);
  }
  __shared__ double part[4][2];
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) {
    part[wave][0] = rest;
    part[wave][1] = full;
  }
  __syncthreads();
  if (threadIdx.x < 2)
    a.sums[static_cast<int64_t>(blockIdx.x) * 2 + threadIdx.x] =
        part[0][threadIdx.x] + part[1][threadIdx.x] + part[2][threadIdx.x] + part[3][threadIdx.x];
}

// Exclusive sum over the workgroup's 256 threads of `mine`, and the total.
__device__ __forceinline__ double scan256(double mine, double* tmp, double* total) {
  double incl = mine;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) {
    const double y = __shfl_up(incl, off, kWave);
    if (lane >= off) incl += y;
  }
  if (lane == kWave - 1) tmp[wave] = incl;
  __syncthreads();
  double before = 0.0;
  for (int v = 0; v < wave; ++v) before += tmp[v];
  *total = (tmp[0] + tmp[1]) + (tmp[2] + tmp[3]);
  __syncthreads();
  return before + (incl - mine);
}

struct DrawLds {
  double tmp[4];
  double before;
  int hit, last;
};

// Workgroup = request.  ONE: the row is a single chunk, and this is the only
// launch.
template <class T, bool ONE>
__global__ __launch_bounds__(256) void verify_draw_kernel(VerifyArgs a) {
  using raw = typename T::raw_t;
  constexpr int kPer = (ONE ? kVerifyOne : kVerifyChunk) / 256;  // columns a thread
  __shared__ DrawLds s;
  const int i = blockIdx.x;
  const int tid = threadIdx.x;
  Row r;
  if constexpr (ONE) {
    r = find_row<T>(a, i);
    if (tid == 0) a.accepted[i] = r.accepted;
  } else {  // from the first launch's count
    const int first = min(max(a.row_indptr[i], 0), a.rows);
    const int end = min(max(a.row_indptr[i + 1], first), a.rows);
    r = Row{a.accepted[i], false, -1, end > first};
    r.rejected = r.accepted < min(end - first - 1, a.most);
    if (r.rejected) r.token = a.tokens[i * a.token_stride + r.accepted];
  }
  int64_t* out = a.out + static_cast<int64_t>(i) * (a.most + 1);
  for (int j = tid; j <= a.most; j += 256)
    if (j != r.accepted || !r.live) out[j] = r.live && j < r.accepted ? a.tokens[i * a.token_stride + j] : -1;
  if (!r.live) return;
  if (tid == 0) {
    s.hit = INT32_MAX;
    s.last = -1;
  }
  int chunk = 0, use = 0;
  double before = 0.0, want = 0.0;
  if constexpr (!ONE) {
    // The chunk that the draw falls in; a thread takes `per` neighbouring ones.
    const double* sums = a.sums + static_cast<int64_t>(i) * a.chunks * 2;
    const int per = (a.chunks + 255) / 256;
    const int c0 = tid * per, c1 = min(c0 + per, a.chunks);
    double rest = 0.0, full = 0.0, total_rest, total_full;
    for (int c = c0; c < c1; ++c) {
      rest += sums[c * 2];
      full += sums[c * 2 + 1];
    }
    double cum = scan256(rest, s.tmp, &total_rest);
    want = static_cast<double>(a.last[i]) * total_rest;
    if (!(total_rest > 0.0)) {
      cum = scan256(full, s.tmp, &total_full);
      use = 1;
      want = static_cast<double>(a.last[i]) * total_full;
    }
    int hit = INT32_MAX, last = -1;
    double here = 0.0;
    for (int c = c0; c < c1; ++c) {
      const double m = sums[c * 2 + use];
      if (m > 0.0) {
        last = c;
        if (hit == INT32_MAX && cum + m > want) {
          hit = c;
          here = cum;
        }
      }
      cum += m;
    }
    if (hit != INT32_MAX) atomicMin(&s.hit, hit);
    if (last >= 0) atomicMax(&s.last, last);
    __syncthreads();
    chunk = s.hit;
    if (chunk == hit && hit != INT32_MAX) s.before = here;
    if (chunk == INT32_MAX) {  // a number of 1 or more: the last column with mass
      chunk = s.last;
      if (tid == 0) s.before = -INFINITY;
    }
    __syncthreads();
    before = s.before;
    if (chunk < 0) {
      if (tid == 0) out[r.accepted] = -1;
      return;
    }
    if (tid == 0) {
      s.hit = INT32_MAX;
      s.last = -1;
    }
  }
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
  if constexpr (ONE) {
    double rest = 0.0, full = 0.0, total_rest, total_full;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      double re, fu;
      column<T>(r, pv[e], q != nullptr, qv[e], x0 + e, &re, &fu);
      if (x0 + e < a.vocab) {
        rest += re;
        full += fu;
      }
    }
    (void)scan256(rest, s.tmp, &total_rest);
    want = static_cast<double>(a.last[i]) * total_rest;
    if (!(total_rest > 0.0)) {
      (void)scan256(full, s.tmp, &total_full);
      use = 1;
      want = static_cast<double>(a.last[i]) * total_full;
    }
  }
  double m[kPer], mine = 0.0, total;
  int hit = INT32_MAX, last = -1;
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    double re, fu;
    column<T>(r, pv[e], q != nullptr, qv[e], x0 + e, &re, &fu);
    m[e] = x0 + e < a.vocab ? (use ? fu : re) : 0.0;
    if (m[e] > 0.0) last = x0 + e;
    mine += m[e];
  }
  double cum = before + scan256(mine, s.tmp, &total);
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    cum += m[e];
    if (hit == INT32_MAX && m[e] > 0.0 && cum > want) hit = x0 + e;
  }
  if (hit != INT32_MAX) atomicMin(&s.hit, hit);
  if (last >= 0) atomicMax(&s.last, last);
  __syncthreads();
  if (tid == 0) out[r.accepted] = s.hit != INT32_MAX ? s.hit : s.last;  // no mass at all: -1
}

template <class T>
hipError_t launch(const VerifyArgs& a, hipStream_t stream) {
  const int64_t blocks = static_cast<int64_t>(a.n) * a.chunks;
  if (!grid_fits(blocks)) return hipErrorInvalidConfiguration;
  if (a.chunks == 1) {
    hipLaunchKernelGGL((verify_draw_kernel<T, true>), dim3(static_cast<unsigned>(a.n)), dim3(256), 0, stream, a);
    return hipGetLastError();
  }
  hipLaunchKernelGGL((verify_sum_kernel<T>), dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((verify_draw_kernel<T, false>), dim3(static_cast<unsigned>(a.n)), dim3(256), 0, stream, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_verify(const VerifyArgs& a, int dtype, hipStream_t stream) {
  if (a.n == 0) return hipSuccess;
  if (dtype == MLORA_F32) return launch<F32>(a, stream);
  return dtype == MLORA_BF16 ? launch<BF16>(a, stream) : launch<F16>(a, stream);
}

}  // namespace mlora
