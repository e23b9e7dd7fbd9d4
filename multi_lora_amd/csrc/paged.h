// The paged KV cache: argument structs and sizes shared by csrc/paged.hip,
// csrc/paged_attn.hip, csrc/verify.hip and the C entry points (the layouts
// callers see are in include/mlora_hip.h).
#pragma once

#include "common.h"

namespace mlora {

// ------------------------------------------------------------- attention plan
// The work list of a step's attention (int32 words), built with the page
// tables.  One item is a tile of query rows over a range of positions; every
// key head runs the same items.  Query rows are (token, query head of the key
// head) pairs, token-major: row m of a request is token m / rep, head m % rep.
constexpr int kApHeaderWords = 16;
constexpr int kApItems = 0;      // items
constexpr int kApJoins = 1;      // tiles whose range is split
constexpr int kApItemWords = 8;  // request, first row, first position, end, slot (-1: none)
constexpr int kApJoinWords = 4;  // request, first row, first slot, slots

// Rows a tile of the streaming kernel holds.
constexpr int kApShortRows = 16;
// A range is split only into parts of at least this many positions.
constexpr int kApMinSplit = 256;
// Tiles that fill the chip this many times over are not split.
constexpr int kApWhole = 4;

struct PagedShape {
  int rep;
  int bm;          // query rows a tile
  int target;      // parts (of all key heads) that fill the chip
  int item_cap;    // items and joins the plan has room for
  int join_cap;
  int slot_cap;    // partial results the workspace has room for
  bool can_split;
  size_t items_off, joins_off, plan_bytes;  // words, words, bytes
  size_t ml_off, ws_bytes;                  // bytes
};
// Host bounds only: rows of the step, requests, new tokens of one request,
// longest cache.  False: unsupported.
bool paged_shape(int n, int rows, int max_new, int64_t max_kv, int heads, int kv_heads, int head_dim, int cus,
                 PagedShape* s);

struct TablesArgs {
  int32_t* table;
  int64_t table_stride;
  int32_t *held, *free, *counts;
  int width, num_pages, page_shift;
  int n;
  const int32_t *start, *add;
  int rows;
  int32_t *row_indptr, *kv_lens, *positions, *slots;
  int32_t* scratch;  // kTablesScratch(n) words
  // plan (nullptr: none)
  int32_t* plan;
  PagedShape shape;
  int kv_heads;
};
constexpr int tables_scratch_words(int n) { return 16 + 3 * n; }
hipError_t launch_page_tables(const TablesArgs& a, hipStream_t stream);

struct WriteArgs {
  const void *q, *k, *v;
  int64_t q_stride, k_stride, v_stride;
  const void *cos, *sin;
  int64_t rot_stride;
  int rot_f32;       // tables in fp32, else in the data type
  const int32_t* slots;
  int rows, heads, kv_heads;
  void *keys, *values;
  int64_t key_stride, value_stride;  // elements between pages
  int num_pages, page_shift;
  void* q_out;
  int64_t q_out_stride;
};
hipError_t launch_rotary_paged_write(const WriteArgs& a, int dtype, int head_dim, bool aligned, hipStream_t stream);

struct PagedAttnArgs {
  const void* q;
  int64_t q_stride;
  const void *keys, *values;
  int64_t key_stride, value_stride;
  int num_pages, page_shift;
  const int32_t* table;
  int64_t table_stride;
  int width;
  const int32_t *row_indptr, *kv_lens;
  int n, rows;
  const int32_t* plan;
  void* out;
  int64_t out_stride;
  float* part;       // [slot][kv_heads][bm][D] sums
  float* ml;         // [slot][kv_heads][bm][2] maximum (log2), sum
  int kv_heads, rep;
  float scale_log2;  // scale * log2(e)
  PagedShape shape;
};
hipError_t launch_paged_attention(const PagedAttnArgs& a, int dtype, int head_dim, hipStream_t stream);

struct VerifyArgs {
  const void* target;
  int64_t target_stride;
  const void* draft;               // nullptr: certain drafts
  int64_t draft_stride0, draft_stride1;
  const int64_t* tokens;
  int64_t token_stride;
  const int32_t* row_indptr;
  const float *accept, *last;
  int64_t accept_stride;
  int n, most, rows, vocab;
  int chunks;
  double* sums;                    // [n][chunks][2]
  int32_t* accepted;
  int64_t* out;                    // [n, most + 1]
};
constexpr int kVerifyChunk = 4096;
hipError_t launch_verify(const VerifyArgs& a, int dtype, hipStream_t stream);

}  // namespace mlora
