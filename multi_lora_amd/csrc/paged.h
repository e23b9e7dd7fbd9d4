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
// Requests of few rows are short: their tiles are streamed by a workgroup
// whose waves share the range.  The others are long: tiles of kApLongRows rows
// whose waves share the rows.
constexpr int kApHeaderWords = 16;
constexpr int kApShort = 0;      // items; joins (tiles whose range is split) in the next word
constexpr int kApLong = 2;       // the same
constexpr int kApJoinRows = 4;   // most rows of a split short tile
// An item: request, first row, first position, end, slot (-1: none), the
// request's first packed row, new tokens, and position of the first of them.
// (What the tables know anyway: looked up, it is one more round trip to memory
// in every workgroup, 0.7 us.)
constexpr int kApItemWords = 8;
constexpr int kApJoinWords = 8;  // first packed row, first row, first slot, slots, rows

constexpr int kApLongRows = 128;
// A range is split only into parts of at least this many positions.  A part of
// a long tile writes and reads again 128 rows of sums: 512 tokens after 2000
// beside 32 decoding requests 99 us, with 512 or 2048 here 117 and 115.
constexpr int kApMinSplit = 256;
constexpr int kApMinSplitLong = 1024;
// Short ranges are split only if the longest is longer than a part by kApKeep,
// and by up to kApKeepFull more as the tiles come to fill half the chip: 32
// requests of 400 positions, four tokens each, take 20.5 us in two parts, 14.3
// whole, 32 of 1500 45.0 and 42.4; but one of 700 9.8 in parts and 11.3 whole,
// eight of 1500 beside 56 of 100 21.3 and 27.2.
constexpr int kApKeep = 384;
constexpr int kApKeepFull = 512;
// Tiles that fill the chip this many times over are not split.
constexpr int kApWhole = 4;

// One kind of item: how many the plan and the workspace have room for, and
// where they are.
struct PagedKind {
  int bm;            // query rows a tile
  int item_cap, join_cap, slot_cap;
  size_t items_off, joins_off;  // words of the plan
  size_t part_off, ml_off;      // bytes of the workspace
};
struct PagedShape {
  int rep;
  int target;        // parts (of all key heads) that fill the chip
  PagedKind kind[2]; // short, long (no caps: none can occur)
  size_t plan_bytes, ws_bytes;
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
  int rows, max_new;
  int32_t *row_indptr, *kv_lens, *positions, *slots;
  int32_t* scratch;  // tables_scratch_words(n) words
  // plan (nullptr: none)
  int32_t* plan;
  PagedShape shape;
  int kv_heads;
};
constexpr int tables_scratch_words(int n) { return 16 + 9 * n; }
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
  int value_rows;    // rows whose values a wave looks after (at most 8); set by the launch
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
  const int32_t* plan;
  int n, rows;       // requests, packed rows
  void* out;
  int64_t out_stride;
  // Of each kind at its offsets: sums [slot][kv_heads][bm][D], and the
  // maximum (log2) and sum of weights [slot][kv_heads][bm][2].
  char* workspace;
  int kv_heads, rep;
  float scale_log2;  // scale * log2(e)
  PagedShape shape;
};
hipError_t launch_paged_attention(const PagedAttnArgs& a, int max_new, int dtype, int head_dim, hipStream_t stream);

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
// Columns a workgroup sums, and columns up to which one workgroup does it all.
// Chunks of 2048 against 4096: 32 requests over 128,256 columns 13.6 us against
// 15.1, one over 32,000 7.8 against 9.1; of 1024, 64 requests 21.6 against 17.7.
// One launch for 4096 columns 6.7, two 8.2; for 8192 10.1, two 8.2.
constexpr int kVerifyChunk = 2048;
constexpr int kVerifyOne = 4096;
constexpr int verify_chunks(int vocab) { return vocab <= kVerifyOne ? 1 : (vocab + kVerifyChunk - 1) / kVerifyChunk; }
hipError_t launch_verify(const VerifyArgs& a, int dtype, hipStream_t stream);

}  // namespace mlora
