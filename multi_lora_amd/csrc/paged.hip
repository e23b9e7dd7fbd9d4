// Page tables of a paged KV cache, and the write of new rows into it
// (gfx950).
#include <algorithm>

#include "kernels.h"
#include "loads.h"
#include "paged.h"

namespace mlora {

namespace {

constexpr int kScanThreads = 1024;
constexpr int kScanWaves = kScanThreads / kWave;

// Scratch words: [0] pages on the stack before the call, [1] pages given
// back, [2] pages wanted, then per request its first freed and first taken
// page (exclusive prefix sums) and the pages it held.
constexpr int kTsTop = 0;
constexpr int kTsFreed = 1;
constexpr int kTsTaken = 2;
constexpr int kTsArrays = 16;

__device__ __forceinline__ int pages_for(int tokens, const TablesArgs& a) {
  const int64_t p = (static_cast<int64_t>(tokens) + (1 << a.page_shift) - 1) >> a.page_shift;
  return static_cast<int>(min(p, static_cast<int64_t>(a.width)));
}

// Tokens request i keeps and gets; sums stay inside 31 bits.
__device__ __forceinline__ int2 lens_of(const TablesArgs& a, int i) {
  const int s = min(max(a.start[i], 0), (1 << 30) - 1);
  const int c = min(max(a.add[i], 0), (1 << 30) - 1);
  return make_int2(s, c);
}

// Page number `t` of the pages wanted in this call: the t-th page given back
// if there is one, else the stack's next entry; -1 when the pool is empty.
__device__ int take_page(const TablesArgs& a, int t, int top, int freed) {
  const int32_t* freed0 = a.scratch + kTsArrays;
  if (t >= freed) {
    const int s = top - 1 - (t - freed);
    return s >= 0 ? a.free[s] : -1;
  }
  int lo = 0, hi = a.n;  // the last request whose first freed page is <= t
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (freed0[mid] <= t) lo = mid;
    else hi = mid;
  }
  const int2 l = lens_of(a, lo);
  return a.table[static_cast<int64_t>(lo) * a.table_stride + pages_for(l.x + l.y, a) + (t - freed0[lo])];
}

// Exclusive sum over the workgroup of a value that fits 31 bits.
__device__ __forceinline__ int scan(int v, int* tmp, int* total) { return block_exclusive_scan<kScanWaves>(v, tmp, total); }

// Prefix sums of rows and pages; one workgroup.
__device__ void scan_requests(const TablesArgs& a, int* tmp) {
  int32_t* freed0 = a.scratch + kTsArrays;
  int32_t* taken0 = freed0 + a.n;
  int32_t* held0 = taken0 + a.n;
  int rows = 0, freed = 0, taken = 0;
  for (int i0 = 0; i0 < a.n; i0 += kScanThreads) {
    const int i = i0 + threadIdx.x;
    int c = 0, f = 0, t = 0;
    if (i < a.n) {
      const int2 l = lens_of(a, i);
      c = l.y;
      const int need = pages_for(l.x + l.y, a);
      const int held = min(max(a.held[i], 0), a.width);
      f = max(held - need, 0);
      t = max(need - held, 0);
      a.kv_lens[i] = l.x + l.y;
      held0[i] = held;
    }
    int total;
    // Rows saturate at the call's rows: later requests then get none.
    const int r0 = scan(min(c, a.rows), tmp, &total);
    if (i < a.n) a.row_indptr[i] = min(rows + r0, a.rows);
    rows = min(rows + total, a.rows);
    const int f0 = scan(f, tmp, &total);
    if (i < a.n) freed0[i] = freed + f0;
    freed += total;
    const int t0 = scan(t, tmp, &total);
    if (i < a.n) taken0[i] = taken + t0;
    taken += total;
  }
  const int top = min(max(a.counts[0], 0), a.num_pages);
  __syncthreads();  // every thread has read counts
  const int have = top + freed;
  for (int i = threadIdx.x; i < a.n; i += kScanThreads) {
    const int2 l = lens_of(a, i);
    const int need = pages_for(l.x + l.y, a);
    const int held = held0[i];
    a.held[i] = need > held ? held + min(need - held, max(have - taken0[i], 0)) : need;
  }
  if (threadIdx.x == 0) {
    a.row_indptr[a.n] = rows;
    a.scratch[kTsTop] = top;
    a.scratch[kTsFreed] = freed;
    a.scratch[kTsTaken] = taken;
    a.counts[0] = max(have - taken, 0);
    a.counts[1] = max(taken - have, 0);
  }
}

// Work list of the step's attention; one workgroup, after scan_requests.
__device__ void build_items(const TablesArgs& a, int* tmp, unsigned long long* wide) {
  const PagedShape& s = a.shape;
  const int room = static_cast<int>(min(static_cast<int64_t>(a.width) << a.page_shift, static_cast<int64_t>(INT32_MAX)));
  if (threadIdx.x < 2) wide[threadIdx.x] = 0;
  __syncthreads();
  unsigned long long work = 0, count = 0;
  for (int i = threadIdx.x; i < a.n; i += kScanThreads) {
    const int c = a.row_indptr[i + 1] - a.row_indptr[i];
    const unsigned long long tiles = (static_cast<unsigned long long>(c) * s.rep + s.bm - 1) / s.bm;
    const int len = min(a.kv_lens[i], room);
    work += tiles * (len - min(c, len) / 2);
    count += tiles;
  }
  for (int off = 1; off < kWave; off <<= 1) {
    work += __shfl_xor(work, off, kWave);
    count += __shfl_xor(count, off, kWave);
  }
  if ((threadIdx.x & 63) == 0) {
    atomicAdd(&wide[0], work);
    atomicAdd(&wide[1], count);
  }
  __syncthreads();
  // Parts of equal length, so that all of them together fill the chip once;
  // tiles that fill it several times over stay whole.
  const unsigned long long part = (wide[0] * a.kv_heads + s.target - 1) / s.target;
  const bool whole = !s.can_split || wide[1] * a.kv_heads >= static_cast<unsigned long long>(kApWhole) * s.target;
  const int split = whole ? INT32_MAX
                          : static_cast<int>(min((max(part, static_cast<unsigned long long>(kApMinSplit)) + 63) / 64 * 64, 1ull << 30));
  int32_t* items = a.plan + s.items_off;
  int32_t* joins = a.plan + s.joins_off;
  int item0 = 0, slot0 = 0, join0 = 0;
  for (int i0 = 0; i0 < a.n; i0 += kScanThreads) {
    const int i = i0 + threadIdx.x;
    int c = 0, len = 0, tiles = 0, parts = 1;
    if (i < a.n) {
      c = a.row_indptr[i + 1] - a.row_indptr[i];
      len = min(a.kv_lens[i], room);
      tiles = static_cast<int>((static_cast<int64_t>(c) * s.rep + s.bm - 1) / s.bm);
      if (len > split) parts = (len + split - 1) / split;
    }
    int n_items, n_slots, n_joins;
    int it = item0 + scan(tiles * parts, tmp, &n_items);
    int sl = slot0 + scan(parts > 1 ? tiles * parts : 0, tmp, &n_slots);
    int jn = join0 + scan(parts > 1 ? tiles : 0, tmp, &n_joins);
    for (int k = tiles - 1; k >= 0; --k) {  // the longest ranges first
      const int last = min((k + 1) * s.bm, c * s.rep) - 1;
      // Positions the tile's last row sees.
      const int end = i < a.n ? min(a.kv_lens[i] - c + last / s.rep + 1, room) : 0;
      const int step = parts > 1 ? ((end + parts - 1) / parts + 63) / 64 * 64 : end;
      const bool fits = it + parts <= s.item_cap && (parts == 1 || (sl + parts <= s.slot_cap && jn < s.join_cap));
      if (!fits) continue;  // the host's bounds rule it out
      if (parts > 1) {
        int32_t* j = joins + static_cast<int64_t>(jn++) * kApJoinWords;
        j[0] = i;
        j[1] = k * s.bm;
        j[2] = sl;
        j[3] = parts;
      }
      for (int p = 0; p < parts; ++p, ++it) {
        int32_t* w = items + static_cast<int64_t>(it) * kApItemWords;
        w[0] = i;
        w[1] = k * s.bm;
        w[2] = min(p * step, end);
        w[3] = p + 1 == parts ? end : min((p + 1) * step, end);
        w[4] = parts > 1 ? sl++ : -1;
      }
    }
    item0 += n_items;
    slot0 += n_slots;
    join0 += n_joins;
  }
  if (threadIdx.x == 0) {
    a.plan[kApItems] = min(item0, s.item_cap);
    a.plan[kApJoins] = min(join0, s.join_cap);
  }
}

__global__ __launch_bounds__(kScanThreads) void tables_scan_kernel(TablesArgs a) {
  __shared__ int tmp[kScanWaves];
  __shared__ unsigned long long wide[2];
  scan_requests(a, tmp);
  if (a.plan != nullptr) {
    __syncthreads();
    build_items(a, tmp, wide);
  }
}

// Blocks [0, row_blocks): positions and slots of 256 rows each; the rest:
// four requests each, one a wave, their pages.  Nothing that one block
// writes is read by another: a freeing request's entries and the stack below
// the pages taken are only read, a taking request's new entries and the
// stack above the pages left only written.
__global__ __launch_bounds__(256) void tables_fill_kernel(TablesArgs a, int row_blocks) {
  const int32_t* freed0 = a.scratch + kTsArrays;
  const int32_t* taken0 = freed0 + a.n;
  const int32_t* held0 = taken0 + a.n;
  const int top = a.scratch[kTsTop], freed = a.scratch[kTsFreed], taken = a.scratch[kTsTaken];
  if (static_cast<int>(blockIdx.x) < row_blocks) {
    const int r = blockIdx.x * 256 + threadIdx.x;
    if (r >= a.rows) return;
    int pos = 0, slot = -1;
    if (r < a.row_indptr[a.n]) {
      int lo = 0, hi = a.n;  // the last request that starts at or before r
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.row_indptr[mid] <= r) lo = mid;
        else hi = mid;
      }
      pos = lens_of(a, lo).x + (r - a.row_indptr[lo]);
      const int pg = pos >> a.page_shift;
      if (pg < a.width) {
        const int id = pg < held0[lo] ? a.table[static_cast<int64_t>(lo) * a.table_stride + pg]
                                      : take_page(a, taken0[lo] + (pg - held0[lo]), top, freed);
        if (id >= 0 && id < a.num_pages) slot = (id << a.page_shift) + (pos & ((1 << a.page_shift) - 1));
      }
    }
    a.positions[r] = pos;
    a.slots[r] = slot;
    return;
  }
  const int i = (blockIdx.x - row_blocks) * 4 + (threadIdx.x >> 6);
  if (i >= a.n) return;
  const int2 l = lens_of(a, i);
  const int need = pages_for(l.x + l.y, a);
  const int held = held0[i];
  int32_t* row = a.table + static_cast<int64_t>(i) * a.table_stride;
  for (int j = held + (threadIdx.x & 63); j < need; j += kWave) row[j] = take_page(a, taken0[i] + (j - held), top, freed);
  for (int j = need + (threadIdx.x & 63); j < held; j += kWave) {
    const int f = freed0[i] + (j - need);
    const int to = top + freed - 1 - f;
    if (f >= taken && to < a.num_pages) a.free[to] = row[j];
  }
}

// ------------------------------------------------------------------- write
// A chunk of 8 table values at p (element index e), as fp32.
template <class T>
__device__ __forceinline__ void rot_chunk(const void* p, int64_t e, bool f32, float* f) {
  if (f32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = static_cast<const float*>(p)[e + i];
  } else {
    const typename T::raw_t* t = static_cast<const typename T::raw_t*>(p) + e;
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = T::to_f32(t[i]);
  }
}

// Blocks [0, rot_blocks): a thread rotates 8 columns of a head's first half
// and the 8 they pair with; x * cos + (x rolled by D / 2) * sin in fp32, one
// rounding.  The rest: a wave takes a row's values of one key head.
template <class T, int D, bool AL>
__global__ __launch_bounds__(256) void paged_write_kernel(WriteArgs a, int rot_blocks) {
  using raw = typename T::raw_t;
  const int page = 1 << a.page_shift;
  if (static_cast<int>(blockIdx.x) < rot_blocks) {
    constexpr int U = D / 16;  // units a head
    const int64_t id = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    const int per_row = (a.heads + a.kv_heads) * U;
    const int64_t r = id / per_row;
    if (r >= a.rows) return;
    const int u = static_cast<int>(id - r * per_row);
    const int h = u / U;
    const int e = (u - h * U) * 8;
    const bool is_q = h < a.heads;
    const raw* x = is_q ? static_cast<const raw*>(a.q) + r * a.q_stride + h * D
                        : static_cast<const raw*>(a.k) + r * a.k_stride + (h - a.heads) * D;
    raw* to;
    if (is_q) {
      to = static_cast<raw*>(a.q_out) + r * a.q_out_stride + h * D;
    } else {
      const int slot = a.slots[r];
      if (slot < 0 || (slot >> a.page_shift) >= a.num_pages) return;
      to = static_cast<raw*>(a.keys) + static_cast<int64_t>(slot >> a.page_shift) * a.key_stride +
           (static_cast<int64_t>(h - a.heads) * page + (slot & (page - 1))) * D;
    }
    const u32x4 lo = load_row_chunk<T, AL>(x, e, 8);
    const u32x4 hi = load_row_chunk<T, AL>(x, e + D / 2, 8);
    float c0[8], c1[8], s0[8], s1[8], y0[8], y1[8];
    rot_chunk<T>(a.cos, r * a.rot_stride + e, a.rot_f32, c0);
    rot_chunk<T>(a.cos, r * a.rot_stride + e + D / 2, a.rot_f32, c1);
    rot_chunk<T>(a.sin, r * a.rot_stride + e, a.rot_f32, s0);
    rot_chunk<T>(a.sin, r * a.rot_stride + e + D / 2, a.rot_f32, s1);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x0 = chunk_elem<T>(lo, i), x1 = chunk_elem<T>(hi, i);
      y0[i] = x0 * c0[i] + x1 * s0[i];
      y1[i] = x1 * c1[i] + x0 * s1[i];
    }
    store_row_chunk<T, AL>(to + e, pack_chunk<T>(y0), 8);
    store_row_chunk<T, AL>(to + e + D / 2, pack_chunk<T>(y1), 8);
    return;
  }
  const int64_t w = (static_cast<int64_t>(blockIdx.x) - rot_blocks) * 4 + (threadIdx.x >> 6);
  const int64_t r = w / a.kv_heads;
  if (r >= a.rows) return;
  const int g = static_cast<int>(w - r * a.kv_heads);
  const int slot = a.slots[r];
  if (slot < 0 || (slot >> a.page_shift) >= a.num_pages) return;
  const raw* v = static_cast<const raw*>(a.v) + r * a.v_stride + g * D;
  raw* to = static_cast<raw*>(a.values) + static_cast<int64_t>(slot >> a.page_shift) * a.value_stride +
            static_cast<int64_t>(g) * D * page + (slot & (page - 1));
  for (int e = threadIdx.x & 63; e < D; e += kWave) to[static_cast<int64_t>(e) * page] = v[e];
}

template <class T, int D>
hipError_t launch_write(const WriteArgs& a, bool aligned, hipStream_t stream) {
  const int64_t units = static_cast<int64_t>(a.rows) * (a.heads + a.kv_heads) * (D / 16);
  const int64_t rot = (units + 255) / 256;
  const int64_t val = (static_cast<int64_t>(a.rows) * a.kv_heads + 3) / 4;
  if (!grid_fits(rot + val)) return hipErrorInvalidConfiguration;
  const dim3 grid(static_cast<unsigned>(rot + val));
  if (aligned)
    hipLaunchKernelGGL((paged_write_kernel<T, D, true>), grid, dim3(256), 0, stream, a, static_cast<int>(rot));
  else
    hipLaunchKernelGGL((paged_write_kernel<T, D, false>), grid, dim3(256), 0, stream, a, static_cast<int>(rot));
  return hipGetLastError();
}

}  // namespace

bool paged_shape(int n, int rows, int max_new, int64_t max_kv, int heads, int kv_heads, int head_dim, int cus,
                 PagedShape* s) {
  *s = PagedShape{};
  if (n < 0 || rows < 0 || max_new < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads != 0) return false;
  s->rep = heads / kv_heads;
  s->bm = kApShortRows;
  s->target = 2 * cus;
  s->can_split = max_kv > kApMinSplit;
  const int64_t tiles = static_cast<int64_t>(rows) * s->rep / s->bm + std::min(n, rows);
  // Parts of a tile: at most its length / split + 1, and the lengths of all
  // tiles sum to at most twice the plan's estimate (len - new / 2).
  const int64_t extra = s->can_split ? 2 * (s->target / kv_heads + 1) : 0;
  const int64_t items = tiles + extra;
  const int64_t slots = s->can_split ? std::min(tiles, kApWhole * static_cast<int64_t>(s->target) / kv_heads + 1) + extra : 0;
  s->item_cap = static_cast<int>(std::min<int64_t>(items, INT32_MAX / 64));
  s->join_cap = static_cast<int>(std::min<int64_t>(tiles, slots / 2));
  if (s->item_cap < items) return false;
  s->slot_cap = static_cast<int>(slots);
  s->items_off = kApHeaderWords;
  s->joins_off = s->items_off + static_cast<size_t>(s->item_cap) * kApItemWords;
  s->plan_bytes = 4 * (s->joins_off + static_cast<size_t>(s->join_cap) * kApJoinWords);
  s->ml_off = static_cast<size_t>(s->slot_cap) * kv_heads * s->bm * head_dim * 4;
  s->ws_bytes = s->ml_off + static_cast<size_t>(s->slot_cap) * kv_heads * s->bm * 2 * 4;
  return true;
}

hipError_t launch_page_tables(const TablesArgs& a, hipStream_t stream) {
  if (a.n == 0 && a.rows == 0) return hipSuccess;
  const int64_t row_blocks = (static_cast<int64_t>(a.rows) + 255) / 256;
  const int64_t blocks = row_blocks + (static_cast<int64_t>(a.n) + 3) / 4;
  if (!grid_fits(blocks)) return hipErrorInvalidConfiguration;
  hipLaunchKernelGGL(tables_scan_kernel, dim3(1), dim3(kScanThreads), 0, stream, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(tables_fill_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream, a,
                     static_cast<int>(row_blocks));
  return hipGetLastError();
}

hipError_t launch_rotary_paged_write(const WriteArgs& a, int dtype, int head_dim, bool aligned, hipStream_t stream) {
  if (a.rows == 0) return hipSuccess;
  if (dtype == MLORA_BF16)
    return head_dim == 64 ? launch_write<BF16, 64>(a, aligned, stream) : launch_write<BF16, 128>(a, aligned, stream);
  return head_dim == 64 ? launch_write<F16, 64>(a, aligned, stream) : launch_write<F16, 128>(a, aligned, stream);
}

}  // namespace mlora
