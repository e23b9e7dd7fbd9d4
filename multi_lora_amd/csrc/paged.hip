// Page tables of a paged KV cache, and the write of new rows into it
// (gfx950).
//
// Tables: request i holds ceil(len_i / page) pages.  Prefix sums over the
// requests of rows, of pages given back and of pages wanted number every page
// that moves; the t-th page wanted is the t-th given back, then the next of
// the free stack, so nothing is claimed by atomics and a step gives the same
// pages every time.  The bytes are kilobytes: launches and the chain of reads
// bound it, hence one workgroup and one launch for all but the largest steps:
// 168 requests of one token 5.6 us, the average of a step and its taking back.
// Beyond, two launches: 8.1 + 3.9 us on average for 4139 rows of 72 requests.
//
// Write: bound by its bytes, read and written once each.  4075 rows of 32 + 2 *
// 8 heads of 128, 102 MB, take 20.5 us on average, 5.0 TB/s, where a copy of 1
// GB has 5.15; 64 rows 3.6.
#include <algorithm>

#include "kernels.h"
#include "loads.h"
#include "paged.h"

namespace mlora {

namespace {

constexpr int kScanThreads = 1024;
constexpr int kScanWaves = kScanThreads / kWave;
// Steps of up to this many requests and rows run as one launch of one
// workgroup; beyond, one workgroup's turns cost more than a second launch.  A
// step and its taking back (of one launch), replayed: 168 requests of one token
// 9.4 us against 15.1 with two launches each, eight prompts of 128 tokens 10.5
// against 15.2; of 512 15.6 against 12.9, of 1024 22.5 against 13.0.
constexpr int kSmallRequests = kScanThreads;
constexpr int kSmallRows = 2048;

// Scratch words: pages on the stack before the call, pages given back, pages
// wanted; then per request its first freed and first taken page (exclusive
// prefix sums), the pages it held, of the work list its first item, slot and
// join and its parts a tile, and its lengths.
constexpr int kTsTop = 0;
constexpr int kTsFreed = 1;
constexpr int kTsTaken = 2;
constexpr int kTsArrays = 16;

__device__ __forceinline__ int pages_for(int tokens, const TablesArgs& a) {
  const int64_t p = (static_cast<int64_t>(tokens) + (1 << a.page_shift) - 1) >> a.page_shift;
  return static_cast<int>(min(p, static_cast<int64_t>(a.width)));
}

// Tokens request i keeps and asks for, as the caller gives them: sums stay
// inside 31 bits, and max_new is kept, for the work list has room for no more.
__device__ __forceinline__ int2 given_lens(const TablesArgs& a, int i) {
  return make_int2(min(max(a.start[i], 0), (1 << 30) - 1), min(max(a.add[i], 0), a.max_new));
}
// Tokens it keeps and gets, from scratch, where the first kernel has put them
// (the caller's may be the step's own kv_lens).
__device__ __forceinline__ int2 lens_of(const TablesArgs& a, int i) {
  const int32_t* start0 = a.scratch + kTsArrays + 7 * a.n;
  return make_int2(start0[i], start0[a.n + i]);
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

// Inclusive sums over the lanes of each row of 16, and over the wave, by lane
// moves (a lane without a source gets 0).
template <int CTRL, int ROWS>
__device__ __forceinline__ int moved(int v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ int row_sum(int v) {
  v += moved<0x111, 0xf>(v);  // row_shr:1
  v += moved<0x112, 0xf>(v);  // row_shr:2
  v += moved<0x114, 0xf>(v);  // row_shr:4
  v += moved<0x118, 0xf>(v);  // row_shr:8
  return v;
}
__device__ __forceinline__ int lane_sum(int v) {
  v = row_sum(v);
  v += moved<0x142, 0xa>(v);  // the last lane of rows 0 and 2 to rows 1 and 3
  v += moved<0x143, 0xc>(v);  // lane 31 to the upper two rows
  return v;
}

// Exclusive sums over the workgroup of N values that fit 31 bits, and their
// totals; the values share the two barriers.
template <int N>
__device__ __forceinline__ void scan(int (&v)[N], int (&total)[N], int (*tmp)[kScanWaves]) {
  static_assert(kScanWaves == 16, "the waves' sums are a row of lanes");
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int x = lane_sum(v[k]);
    if (lane == kWave - 1) tmp[k][wave] = x;
    v[k] = x - v[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int t = row_sum(tmp[k][lane & 15]);
    total[k] = __builtin_amdgcn_readlane(t, 15);
    if (wave > 0) v[k] += __builtin_amdgcn_readlane(t, wave - 1);
  }
  __syncthreads();
}

// Tiles of a request's c new tokens, and which kind they are.
__device__ __forceinline__ int kind_of(const PagedShape& s, int c) {
  return static_cast<int64_t>(c) * s.rep > s.kind[0].bm ? 1 : 0;
}
__device__ __forceinline__ int tiles_of(const PagedShape& s, int c, int kind) {
  const int bm = s.kind[kind].bm;
  return static_cast<int>((static_cast<int64_t>(c) * s.rep + bm - 1) / bm);
}
__device__ __forceinline__ int table_room(const TablesArgs& a) {
  return static_cast<int>(min(static_cast<int64_t>(a.width) << a.page_shift, static_cast<int64_t>(1 << 30)));
}

// What the ranges' split is found from, summed over the workgroup: positions of
// all tiles, tiles and the longest range of each kind.
struct Ranges {
  unsigned long long work[2], tiles[2];
  int longest[2];
};

__device__ __forceinline__ void add_ranges(Ranges& r, unsigned long long (&work)[2], int (&tiles)[2], int (&longest)[2]) {
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    if (__ballot(tiles[k] != 0) == 0) continue;
    for (int off = 1; off < kWave; off <<= 1) {
      work[k] += __shfl_xor(work[k], off, kWave);
      tiles[k] += __shfl_xor(tiles[k], off, kWave);
      longest[k] = max(longest[k], __shfl_xor(longest[k], off, kWave));
    }
    if ((threadIdx.x & 63) == 0) {
      atomicAdd(&r.work[k], work[k]);
      atomicAdd(&r.tiles[k], static_cast<unsigned long long>(tiles[k]));
      atomicMax(&r.longest[k], longest[k]);
    }
  }
}

// Lengths at which the ranges of each kind split: parts of equal length, so
// that all of them together fill the chip once; tiles that fill it several
// times over stay whole.  So do short ranges if the longest is not much longer
// than a part, for the join costs time of its own, more the more tiles it has.
__device__ __forceinline__ void split_lengths(const TablesArgs& a, const Ranges& r, int (&split)[2]) {
  const unsigned long long target = a.shape.target;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const unsigned long long part = (r.work[k] * a.kv_heads + target - 1) / target;
    const unsigned long long least = max(part, static_cast<unsigned long long>(k ? kApMinSplitLong : kApMinSplit));
    split[k] = static_cast<int>((min(least, 1ull << 30) + 63) / 64 * 64);  // (no range is longer than 2^30)
    if (r.tiles[k] * a.kv_heads >= kApWhole * target) split[k] = INT32_MAX;
  }
  const unsigned long long filled = min(2 * r.tiles[0] * a.kv_heads, target);
  const int keep = kApKeep + static_cast<int>(kApKeepFull * filled / target);
  if (r.longest[0] - keep <= split[0]) split[0] = INT32_MAX;
}

// Parts of a tile of `len` positions.  Short ones round up, so that none is
// longer than the others; long ones down, so that all of them still run at
// once (a second turn of a few cost as much as the first: 512 tokens after
// 8192, 121 us in five parts, 109 in three).
__device__ __forceinline__ int parts_of(int len, int split, int kind) {
  return kind ? max(len / split, 1) : len > split ? (len + split - 1) / split : 1;
}

// The items of a kind go on the list in three groups of requests, the longest
// first: what starts last then ends soon after the rest.  300 requests of 100
// positions before 20 of 3000 took 98 us in the requests' order, 81 in this;
// 20 prompts of 300 before four chunks of 300 after 3000 165 and 142.
__device__ __forceinline__ int group_of(const Ranges& r, const int (&split)[2], int len, int parts, int kind) {
  const int longest = kind ? r.longest[1] : min(split[0], r.longest[0]);
  const int64_t all = static_cast<int64_t>(longest) * (kind ? 1 : parts);
  return 2ll * len > all ? 0 : 4ll * len > all ? 1 : 2;
}
struct Groups {  // an item's place from the groups' sums
  int before[3], total[3];
  __device__ int at(int group) const {
    return group == 0 ? before[0] : group == 1 ? total[0] + before[1] : total[0] + total[1] + before[2];
  }
};

// Tile t of a request's `tiles`, those of the longest ranges first, in `parts`
// items.  (The host's bounds leave room for all of them.)
__device__ __forceinline__ void put_items(const TablesArgs& a, const PagedKind& kd, int i, int first, int c, int len, int room,
                                          int tiles, int t, int parts, int it, int sl, int jn) {
  const int row0 = (tiles - 1 - t) * kd.bm;
  const int last = min(row0 + kd.bm, c * a.shape.rep) - 1;
  const int end = min(len - c + last / a.shape.rep + 1, room);  // positions the tile's last row sees
  const int step = ((end + parts - 1) / parts + 63) / 64 * 64;
  if (it + parts > kd.item_cap || (parts > 1 && (sl + parts > kd.slot_cap || jn >= kd.join_cap))) return;
  for (int p = 0; p < parts; ++p) {
    int32_t* w = a.plan + kd.items_off + static_cast<int64_t>(it + p) * kApItemWords;
    w[0] = i;
    w[1] = row0;
    w[2] = min(p * step, end);
    w[3] = p + 1 == parts ? end : min((p + 1) * step, end);
    w[4] = parts > 1 ? sl + p : -1;
    w[5] = first;
    w[6] = c;
    w[7] = len - c;
  }
  if (parts > 1) {
    int32_t* j = a.plan + kd.joins_off + static_cast<int64_t>(jn) * kApJoinWords;
    j[0] = first;
    j[1] = row0;
    j[2] = sl;
    j[3] = parts;
    j[4] = last + 1 - row0;
  }
}

// The last of n ascending numbers (the first is 0) that is at most v.
__device__ __forceinline__ int last_at_most(const int* x, int n, int v) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (x[mid] <= v) lo = mid;
    else hi = mid;
  }
  return lo;
}

// A step of few requests and rows in one workgroup and one launch: thread =
// request for the sums and the work list, then row, then page.
__global__ __launch_bounds__(kScanThreads) void tables_small_kernel(TablesArgs a) {
  __shared__ int tmp[10][kScanWaves];
  __shared__ Ranges ranges;
  __shared__ int join_rows;
  __shared__ int first_s[kSmallRequests], freed_s[kSmallRequests], taken_s[kSmallRequests], need_s[kSmallRequests],
      held_s[kSmallRequests], start_s[kSmallRequests];
  const int i = threadIdx.x;
  const bool plan = a.plan != nullptr;
  const int top = min(max(a.counts[0], 0), a.num_pages);
  int v[3] = {0, 0, 0}, total[3];
  int len = 0, start = 0, need = 0, held = 0;
  if (i == 0) {
    ranges = Ranges{};
    join_rows = 0;
  }
  if (i < a.n) {
    const int2 l = given_lens(a, i);
    start = l.x;
    need = pages_for(l.x + l.y, a);
    held = min(max(a.held[i], 0), a.width);
    v[0] = min(l.y, a.rows + 1);
    v[1] = max(held - need, 0);
    v[2] = max(need - held, 0);
  }
  int c = v[0];
  scan(v, total, tmp);
  const int rows = min(total[0], a.rows), first = min(v[0], a.rows);
  c = min(c, a.rows - first);
  int freed = total[1], taken = total[2];
  if (total[0] > a.rows) {  // some get fewer tokens than asked for, and pages for those only
    int w[2] = {0, 0}, t[2];
    if (i < a.n) {
      need = pages_for(start + c, a);
      w[0] = max(held - need, 0);
      w[1] = max(need - held, 0);
    }
    scan(w, t, tmp);
    v[1] = w[0], v[2] = w[1], freed = t[0], taken = t[1];
  }
  if (i < a.n) {
    len = start + c;
    first_s[i] = first;
    freed_s[i] = v[1];
    taken_s[i] = v[2];
    need_s[i] = need;
    held_s[i] = held;
    start_s[i] = start;
    a.row_indptr[i] = first;
    a.kv_lens[i] = len;
    a.held[i] = need > held ? held + min(need - held, max(top + freed - v[2], 0)) : need;
  }
  if (i == 0) {
    a.row_indptr[a.n] = rows;
    a.counts[0] = max(top + freed - taken, 0);
    a.counts[1] = max(taken - top - freed, 0);
  }
  __syncthreads();

  // As in take_page.
  auto take = [&](int t) {
    if (t >= freed) {
      const int at = top - 1 - (t - freed);
      return at >= 0 ? a.free[at] : -1;
    }
    const int lo = last_at_most(freed_s, a.n, t);
    return a.table[static_cast<int64_t>(lo) * a.table_stride + need_s[lo] + (t - freed_s[lo])];
  };
  for (int r = i; r < a.rows; r += kScanThreads) {
    int pos = 0, slot = -1;
    if (r < rows) {
      const int q = last_at_most(first_s, a.n, r);
      pos = start_s[q] + (r - first_s[q]);
      const int pg = pos >> a.page_shift;
      if (pg < a.width) {
        const int id = pg < held_s[q] ? a.table[static_cast<int64_t>(q) * a.table_stride + pg] : take(taken_s[q] + (pg - held_s[q]));
        if (id >= 0 && id < a.num_pages) slot = (id << a.page_shift) + (pos & ((1 << a.page_shift) - 1));
      }
    }
    a.positions[r] = pos;
    a.slots[r] = slot;
  }
  for (int t = i; t < taken; t += kScanThreads) {
    const int q = last_at_most(taken_s, a.n, t);
    a.table[static_cast<int64_t>(q) * a.table_stride + held_s[q] + (t - taken_s[q])] = take(t);
  }
  for (int f = taken + i; f < freed; f += kScanThreads) {
    const int q = last_at_most(freed_s, a.n, f);
    const int to = top + freed - 1 - f;
    if (to < a.num_pages) a.free[to] = a.table[static_cast<int64_t>(q) * a.table_stride + need_s[q] + (f - freed_s[q])];
  }
  if (!plan) return;

  const PagedShape& s = a.shape;
  const int room = table_room(a);
  const int seen = min(len, room);
  const int kind = kind_of(s, c);
  const int tiles = tiles_of(s, c, kind);
  const unsigned long long positions = static_cast<unsigned long long>(tiles) * seen;
  unsigned long long work[2] = {kind ? 0 : positions, kind ? positions : 0};
  int count[2] = {kind ? 0 : tiles, kind ? tiles : 0};
  int longest[2] = {kind || tiles == 0 ? 0 : seen, kind && tiles > 0 ? seen : 0};
  add_ranges(ranges, work, count, longest);
  __syncthreads();
  int split[2];
  split_lengths(a, ranges, split);
  const int parts = parts_of(seen, kind ? split[1] : split[0], kind);
  const int items = tiles * parts;
  if (kind == 0 && parts > 1 && tiles > 0) atomicMax(&join_rows, c * s.rep);
  const int group = group_of(ranges, split, seen, parts, kind);
  int u[10], sums[10];  // items by kind and group, then slots and joins
#pragma unroll
  for (int k = 0; k < 2; ++k) {
#pragma unroll
    for (int g = 0; g < 3; ++g) u[3 * k + g] = kind == k && group == g ? items : 0;
    u[6 + k] = kind == k && parts > 1 ? items : 0;
    u[8 + k] = kind == k && parts > 1 ? tiles : 0;
  }
  scan(u, sums, tmp);
  const PagedKind kd = kind ? s.kind[1] : s.kind[0];
  const Groups listed = kind ? Groups{{u[3], u[4], u[5]}, {sums[3], sums[4], sums[5]}} : Groups{{u[0], u[1], u[2]}, {sums[0], sums[1], sums[2]}};
  const int it = listed.at(group), sl = kind ? u[7] : u[6], jn = kind ? u[9] : u[8];
  for (int t = 0; t < tiles; ++t) put_items(a, kd, i, first_s[i], c, len, room, tiles, t, parts, it + t * parts, sl + t * parts, jn + t);
  if (i < 2) {
    a.plan[i ? kApLong : kApShort] = min(i ? sums[3] + sums[4] + sums[5] : sums[0] + sums[1] + sums[2], s.kind[i].item_cap);
    a.plan[(i ? kApLong : kApShort) + 1] = min(i ? sums[9] : sums[8], s.kind[i].join_cap);
  }
  if (i == 2) a.plan[kApJoinRows] = join_rows;
}

// Prefix sums of rows, pages and items; one workgroup.
__global__ __launch_bounds__(kScanThreads) void tables_scan_kernel(TablesArgs a) {
  __shared__ int tmp[5][kScanWaves];
  __shared__ Ranges ranges;
  __shared__ int join_rows;
  int32_t* freed0 = a.scratch + kTsArrays;
  int32_t* taken0 = freed0 + a.n;
  int32_t* held0 = taken0 + a.n;
  int32_t* item0 = held0 + a.n;
  int32_t* slot0 = item0 + a.n;
  int32_t* join0 = slot0 + a.n;
  int32_t* parts0 = join0 + a.n;
  const PagedShape& s = a.shape;
  const bool plan = a.plan != nullptr;
  const int room = table_room(a);
  if (threadIdx.x == 0) {
    ranges = Ranges{};
    join_rows = 0;
  }
  int rows = 0, freed = 0, taken = 0;
  unsigned long long work[2] = {0, 0};
  int count[2] = {0, 0}, longest[2] = {0, 0};
  for (int i0 = 0; i0 < a.n; i0 += kScanThreads) {
    const int i = i0 + threadIdx.x;
    int v[3] = {0, 0, 0}, total[3];
    int2 l = make_int2(0, 0);
    int held = 0;
    if (i < a.n) {
      l = given_lens(a, i);
      const int need = pages_for(l.x + l.y, a);
      held = min(max(a.held[i], 0), a.width);
      v[0] = min(l.y, a.rows + 1);
      v[1] = max(held - need, 0);
      v[2] = max(need - held, 0);
      held0[i] = held;
    }
    const int c = v[0];
    scan(v, total, tmp);
    // Rows saturate at the call's rows: later requests then get none.
    const int first = min(rows + v[0], a.rows);
    const int mine = min(c, a.rows - first);
    if (rows + total[0] > a.rows) {  // as in the small kernel
      int w[2] = {0, 0}, t[2];
      if (i < a.n) {
        const int need = pages_for(l.x + mine, a);
        w[0] = max(held - need, 0);
        w[1] = max(need - held, 0);
      }
      scan(w, t, tmp);
      v[1] = w[0], v[2] = w[1], total[1] = t[0], total[2] = t[1];
    }
    if (i < a.n) {
      a.row_indptr[i] = first;
      a.kv_lens[i] = l.x + mine;
      parts0[a.n + i] = l.x;
      parts0[2 * a.n + i] = mine;
      freed0[i] = freed + v[1];
      taken0[i] = taken + v[2];
      if (plan) {
        const int kind = kind_of(s, mine);
        const int tiles = tiles_of(s, mine, kind);
        const int len = min(l.x + mine, room);
        work[kind] += static_cast<unsigned long long>(tiles) * len;
        count[kind] += tiles;
        if (tiles > 0) longest[kind] = max(longest[kind], len);
      }
    }
    rows = min(rows + total[0], a.rows);
    freed += total[1];
    taken += total[2];
  }
  const int top = min(max(a.counts[0], 0), a.num_pages);
  if (plan) add_ranges(ranges, work, count, longest);
  __syncthreads();  // every thread has read counts, and written what others read below
  if (threadIdx.x == 0) {
    a.row_indptr[a.n] = rows;
    a.scratch[kTsTop] = top;
    a.scratch[kTsFreed] = freed;
    a.scratch[kTsTaken] = taken;
    a.counts[0] = max(top + freed - taken, 0);
    a.counts[1] = max(taken - top - freed, 0);
  }
  int split[2] = {INT32_MAX, INT32_MAX};
  if (plan) split_lengths(a, ranges, split);
  const int have = top + freed;
  int base[2][3] = {{0, 0, 0}, {0, 0, 0}};  // items, slots, joins so far of each kind
  for (int i0 = 0; i0 < a.n; i0 += kScanThreads) {
    const int i = i0 + threadIdx.x;
    int c = 0, len = 0;
    if (i < a.n) {
      const int2 l = lens_of(a, i);
      const int need = pages_for(l.x + l.y, a);
      const int held = held0[i];
      a.held[i] = need > held ? held + min(need - held, max(have - taken0[i], 0)) : need;
      c = l.y;
      len = min(l.x + c, room);
    }
    if (!plan) continue;
    const int kind = kind_of(s, c);
    const int tiles = tiles_of(s, c, kind);
    const int parts = parts_of(len, kind ? split[1] : split[0], kind);
    const int items = tiles * parts;
    if (kind == 0 && parts > 1 && tiles > 0) atomicMax(&join_rows, c * s.rep);
    const int group = group_of(ranges, split, len, parts, kind);
#pragma unroll
    for (int k = 0; k < 2; ++k) {  // (the groups of 1024 requests at a time)
      const int mine = kind == k ? items : 0;
      int v[5] = {group == 0 ? mine : 0, group == 1 ? mine : 0, group == 2 ? mine : 0, parts > 1 ? mine : 0,
                  kind == k && parts > 1 ? tiles : 0}, t[5];
      scan(v, t, tmp);
      if (i < a.n && kind == k) {
        item0[i] = base[k][0] + Groups{{v[0], v[1], v[2]}, {t[0], t[1], t[2]}}.at(group);
        slot0[i] = base[k][1] + v[3];
        join0[i] = base[k][2] + v[4];
        parts0[i] = parts;
      }
      base[k][0] += t[0] + t[1] + t[2];
      base[k][1] += t[3];
      base[k][2] += t[4];
    }
  }
  if (!plan) return;
  __syncthreads();
  if (threadIdx.x == 0) a.plan[kApJoinRows] = join_rows;
  if (threadIdx.x < 2) {
    const int k = threadIdx.x;
    a.plan[(k ? kApLong : kApShort)] = min(k ? base[1][0] : base[0][0], s.kind[k].item_cap);
    a.plan[(k ? kApLong : kApShort) + 1] = min(k ? base[1][2] : base[0][2], s.kind[k].join_cap);
  }
}

// Blocks [0, row_blocks): positions and slots of 256 rows each; the rest:
// four requests each, one a wave, their pages and items.  Nothing that one
// block writes is read by another: a freeing request's entries and the stack
// below the pages taken are only read, a taking request's new entries and the
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
  const int lane = threadIdx.x & 63;
  const int2 l = lens_of(a, i);
  const int need = pages_for(l.x + l.y, a);
  const int held = held0[i];
  int32_t* row = a.table + static_cast<int64_t>(i) * a.table_stride;
  for (int j = held + lane; j < need; j += kWave) row[j] = take_page(a, taken0[i] + (j - held), top, freed);
  for (int j = need + lane; j < held; j += kWave) {
    const int f = freed0[i] + (j - need);
    const int to = top + freed - 1 - f;
    if (f >= taken && to < a.num_pages) a.free[to] = row[j];
  }
  if (a.plan == nullptr) return;
  const PagedShape& s = a.shape;
  const int32_t* item0 = held0 + a.n;
  const int first_row = a.row_indptr[i];
  const int c = a.row_indptr[i + 1] - first_row;
  const int len = l.x + c;
  const int kind = kind_of(s, c);
  const PagedKind kd = kind ? s.kind[1] : s.kind[0];
  const int tiles = tiles_of(s, c, kind);
  const int first_item = item0[i], first_slot = item0[a.n + i], first_join = item0[2 * a.n + i], parts = item0[3 * a.n + i];
  const int room = table_room(a);
  for (int t = lane; t < tiles; t += kWave)
    put_items(a, kd, i, first_row, c, len, room, tiles, t, parts, first_item + t * parts, first_slot + t * parts, first_join + t);
}

// ------------------------------------------------------------------- write
// A chunk of 8 table values at element e, as fp32.
template <class T, bool AL>
__device__ __forceinline__ void rot_chunk(const void* p, int64_t e, bool f32, float* f) {
  if (f32) {
    const float* t = static_cast<const float*>(p) + e;
    if constexpr (AL) {
      const f32x4 lo = *reinterpret_cast<const f32x4*>(t), hi = *reinterpret_cast<const f32x4*>(t + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = lo[i], f[4 + i] = hi[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = t[i];
    }
  } else {
    const u32x4 v = load_row_chunk<T, AL>(static_cast<const typename T::raw_t*>(p), static_cast<int>(e), 8);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = chunk_elem<T>(v, i);
  }
}

// Blocks [0, value_blocks): values; they lie transposed in a page, so a row
// alone is D stores of 2 bytes.  A wave looks at the slots around a few rows:
// eight rows whose slots fill a 16-byte chunk of a page are stored as chunks by
// the wave that has the first of them, others one by one.  The rest of the
// blocks: a thread rotates 8 columns of a head's first half and the 8 they pair
// with; x * cos + (x rolled by D / 2) * sin in fp32, one rounding.  (Values
// last: 24.1 us instead of 20.2 for 4075 rows.)
template <class T, int D, bool AL>
__global__ __launch_bounds__(256) void paged_write_kernel(WriteArgs a, int value_blocks) {
  using raw = typename T::raw_t;
  const int page = 1 << a.page_shift;
  const int64_t slots = static_cast<int64_t>(a.num_pages) << a.page_shift;
  if (static_cast<int>(blockIdx.x) >= value_blocks) {
    constexpr int U = D / 16;  // units a head
    const int64_t id = (static_cast<int64_t>(blockIdx.x) - value_blocks) * 256 + threadIdx.x;
    const int per_row = (a.heads + a.kv_heads) * U;
    const int r = static_cast<int>(id / per_row);
    if (r >= a.rows) return;
    const int u = static_cast<int>(id - static_cast<int64_t>(r) * per_row);
    const int h = u / U;
    const int e = (u - h * U) * 8;
    const bool is_q = h < a.heads;
    const raw* x = is_q ? static_cast<const raw*>(a.q) + r * a.q_stride + h * D
                        : static_cast<const raw*>(a.k) + r * a.k_stride + (h - a.heads) * D;
    const u32x4 lo = load_row_chunk<T, AL>(x, e, 8);
    const u32x4 hi = load_row_chunk<T, AL>(x, e + D / 2, 8);
    float c0[8], c1[8], s0[8], s1[8], y0[8], y1[8];
    const char* cs = static_cast<const char*>(a.cos) + r * a.rot_stride * (a.rot_f32 ? 4 : 2);
    const char* sn = static_cast<const char*>(a.sin) + r * a.rot_stride * (a.rot_f32 ? 4 : 2);
    rot_chunk<T, AL>(cs, e, a.rot_f32, c0);
    rot_chunk<T, AL>(cs, e + D / 2, a.rot_f32, c1);
    rot_chunk<T, AL>(sn, e, a.rot_f32, s0);
    rot_chunk<T, AL>(sn, e + D / 2, a.rot_f32, s1);
    raw* to;
    if (is_q) {
      to = static_cast<raw*>(a.q_out) + r * a.q_out_stride + h * D;
    } else {
      const int slot = a.slots[r];
      if (slot < 0 || slot >= slots) return;
      to = static_cast<raw*>(a.keys) + static_cast<int64_t>(slot >> a.page_shift) * a.key_stride +
           (static_cast<int64_t>(h - a.heads) * page + (slot & (page - 1))) * D;
    }
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
  const int64_t w = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int64_t first = w / a.kv_heads * a.value_rows;
  if (first >= a.rows) return;
  const int r0 = static_cast<int>(first);
  const int g = static_cast<int>(w % a.kv_heads);
  const int lane = threadIdx.x & 63;
  // Lane l looks at row r0 - 7 + l.  Bits of lanes: rows with a slot, those in
  // the slot behind the row before, first ones of eight that fill a chunk.
  const int look = r0 - 7 + lane;
  const int seen = lane < a.value_rows + 14 && look >= 0 && look < a.rows ? a.slots[look] : -1;
  const int before = __shfl_up(seen, 1, kWave);
  const uint64_t placed = __ballot(seen >= 0 && seen < slots);
  const uint64_t follows = __ballot(lane > 0 && seen == before + 1);
  uint64_t whole = AL ? placed & __ballot((seen & 7) == 0) : 0;
#pragma unroll
  for (int i = 1; i < 8; ++i) whole &= follows >> i;
  uint64_t covered = whole;
#pragma unroll
  for (int i = 1; i < 8; ++i) covered |= whole << i;
  const uint64_t mine = ((1ull << a.value_rows) - 1) << 7;
  const int64_t head = static_cast<int64_t>(g) * D * page;
  const raw* v = static_cast<const raw*>(a.v) + g * D + lane;
  raw* values = static_cast<raw*>(a.values) + head + static_cast<int64_t>(lane) * page;
  auto place = [&](int slot) { return values + static_cast<int64_t>(slot >> a.page_shift) * a.value_stride + (slot & (page - 1)); };
  for (uint64_t todo = whole & mine; todo != 0; todo &= todo - 1) {
    const int l = __builtin_amdgcn_readfirstlane(__builtin_ctzll(todo));
    const raw* from = v + (r0 - 7 + l) * a.v_stride;
    raw* to = place(__builtin_amdgcn_readlane(seen, l));
#pragma unroll
    for (int e = 0; e < D; e += kWave) {
      u32x4 c;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        c[i] = static_cast<uint32_t>(from[2 * i * a.v_stride + e]) | static_cast<uint32_t>(from[(2 * i + 1) * a.v_stride + e]) << 16;
      st_chunk(to + static_cast<int64_t>(e) * page, c);
    }
  }
  const uint64_t single = placed & mine & ~covered;
  if (single == 0) return;
  // The loads of all of the wave's rows go out before the first store.
  raw x[8][D / kWave];
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < a.value_rows)
#pragma unroll
      for (int e = 0; e < D / kWave; ++e) x[j][e] = v[min(r0 + j, a.rows - 1) * a.v_stride + e * kWave];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if ((single >> (7 + j) & 1) == 0) continue;
    raw* to = place(__builtin_amdgcn_readlane(seen, 7 + j));
#pragma unroll
    for (int e = 0; e < D / kWave; ++e) to[static_cast<int64_t>(e * kWave) * page] = x[j][e];
  }
}

// Rows whose values one wave looks after.  More share the look at the slots and
// ask for more at once, fewer are more waves: 64 decoding requests 3.8 us with
// one row, 4.1 with four, 4.9 with eight; 1000 15.9, 13.0, 13.3; 4096 tokens of
// each of four prompts 136, 99, 92.
constexpr int value_rows(int rows) { return rows < 128 ? 1 : rows < 2048 ? 4 : 8; }

template <class T, int D>
hipError_t launch_write(WriteArgs a, bool aligned, hipStream_t stream) {
  a.value_rows = value_rows(a.rows);
  const int64_t units = static_cast<int64_t>(a.rows) * (a.heads + a.kv_heads) * (D / 16);
  const int64_t rot = (units + 255) / 256;
  const int64_t val = ((static_cast<int64_t>(a.rows) + a.value_rows - 1) / a.value_rows * a.kv_heads + 3) / 4;
  if (!grid_fits(rot + val)) return hipErrorInvalidConfiguration;
  const dim3 grid(static_cast<unsigned>(rot + val));
  if (aligned)
    hipLaunchKernelGGL((paged_write_kernel<T, D, true>), grid, dim3(256), 0, stream, a, static_cast<int>(val));
  else
    hipLaunchKernelGGL((paged_write_kernel<T, D, false>), grid, dim3(256), 0, stream, a, static_cast<int>(val));
  return hipGetLastError();
}

}  // namespace

bool paged_shape(int n, int rows, int max_new, int64_t max_kv, int heads, int kv_heads, int head_dim, int cus,
                 PagedShape* s) {
  *s = PagedShape{};
  if (n < 0 || rows < 0 || max_new < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads != 0) return false;
  s->rep = heads / kv_heads;
  s->target = 2 * cus;
  const int64_t most = static_cast<int64_t>(std::min(max_new, rows)) * s->rep;  // rows of one request
  const int64_t all = static_cast<int64_t>(rows) * s->rep;
  s->kind[0].bm = most <= 16 || most > 32 ? 16 : 32;
  s->kind[1].bm = kApLongRows;
  size_t words = kApHeaderWords, bytes = 0;
  for (int k = 0; k < 2; ++k) {
    PagedKind& kd = s->kind[k];
    const bool occurs = k == 0 ? n > 0 && rows > 0 : most > s->kind[0].bm;
    // A short request has one tile, a long one more than short rows.
    const int64_t tiles = !occurs ? 0
                          : k == 0 ? std::min(n, rows)
                                   : all / kd.bm + std::min<int64_t>(n, all / (s->kind[0].bm + 1));
    // A range splits into parts only where it is longer than `split`, and the
    // lengths of all tiles over the split are at most the parts that fill the
    // chip, target / kv_heads.  So the parts past each tile's first are at most
    // that many; and so are all parts of long tiles that split (they round
    // down), while those of short ones, which round a ratio above 1 up, are
    // fewer than twice as many.  4096 rows of 64 requests, 8 key heads of 128:
    // 43 MB; with room for two parts of every tile it would be 145.
    const int64_t extra = !occurs || max_kv <= (k ? kApMinSplitLong : kApMinSplit + kApKeep) ? 0 : s->target / kv_heads + 1;
    const int64_t slots = extra > 0 ? std::min(tiles + extra, static_cast<int64_t>(k ? 1 : 2) * s->target / kv_heads) : 0;
    if (tiles + extra > INT32_MAX / 64) return false;
    kd.item_cap = static_cast<int>(tiles + extra);
    kd.slot_cap = static_cast<int>(slots);
    kd.join_cap = static_cast<int>(std::min(tiles, slots / 2));
    kd.items_off = words;
    words += static_cast<size_t>(kd.item_cap) * kApItemWords;
    kd.joins_off = words;
    words += static_cast<size_t>(kd.join_cap) * kApJoinWords;
    kd.part_off = bytes;
    bytes += static_cast<size_t>(kd.slot_cap) * kv_heads * kd.bm * head_dim * 4;
    kd.ml_off = bytes;
    bytes += static_cast<size_t>(kd.slot_cap) * kv_heads * kd.bm * 2 * 4;
  }
  s->plan_bytes = 4 * words;
  s->ws_bytes = bytes;
  return true;
}

hipError_t launch_page_tables(const TablesArgs& a, hipStream_t stream) {
  const int64_t row_blocks = (static_cast<int64_t>(a.rows) + 255) / 256;
  const int64_t blocks = row_blocks + (static_cast<int64_t>(a.n) + 3) / 4;
  if (!grid_fits(blocks)) return hipErrorInvalidConfiguration;
  if (a.n <= kSmallRequests && a.rows <= kSmallRows) {
    hipLaunchKernelGGL(tables_small_kernel, dim3(1), dim3(kScanThreads), 0, stream, a);
    return hipGetLastError();
  }
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
