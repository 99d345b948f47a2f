// Paged key/value cache: the work list shared by the planner (host) and the
// attention kernels, and the launchers behind the C ABI.
//
// A request with n new tokens and a group of G = heads / kv_heads query heads
// on each key head has n * G "packed rows" per key head: packed row i is token
// i / G, query head h * G + i % G.  All of them read the same keys, so tiles of
// packed rows, not of tokens, feed the tensor cores: a single token of grouped
// heads fills G rows, and any G (a power of two or not) packs without holes.
#pragma once

#include "internal.h"

namespace tf {

// One piece of work: `rows` packed rows from row0 of (request, kv_head)
// against key tiles [tile0, tile1).
struct PagedSegment {
  int32_t q_row;    // row of q / out of the request's first new token
  int32_t new_len;  // new tokens of the request
  int32_t kv_len;   // cached tokens, the new ones included
  int32_t request;
  int32_t kv_head;
  int32_t row0;
  int32_t rows;
  int32_t tile0;
  int32_t tile1;
  int32_t part;     // slot of this piece's partial result; -1: the whole result
  int32_t part0;    // first slot and number of the pieces of the same rows
  int32_t parts;
  int32_t counter;  // arrivals of those pieces
  int32_t pad[3];
};
static_assert(sizeof(PagedSegment) == 64, "segments are read as four 16-byte vectors");

constexpr int kSplitRows = 16;  // packed rows of a segment of the few-rows kernel (one m16 MMA tile)
constexpr int kSplitKeys = 32;  // keys per tile
constexpr int kTileRows = 256;  // packed rows of a segment of the tensor-core kernel (two halves of 128)
constexpr int kHalfRows = 128;  // of its form with one half
constexpr int kTileKeys = 128;  // keys per tile

struct PagedArgs {
  const void* q = nullptr;
  int64_t q_stride = 0;
  tf_page_table table{};
  tf_paged_kv kv{};
  const tf_paged_plan* plan = nullptr;
  char* plan_table = nullptr;
  float scale = 1.f;
  int act = TF_DTYPE_F16;
  void* out = nullptr;
  char* workspace = nullptr;
};

// Fills the plan's remaining fields, and the table where it fits.
tf_status paged_plan_make(const int32_t* new_lengths, const int32_t* kv_lengths, tf_paged_plan* plan, char* table,
                          size_t table_capacity);
// Tensor map over pages as [page][64-column half][kv_head * page_size rows][64
// columns], box of box_rows rows by box_columns columns of one page, 128-byte
// swizzle; a page id outside [0, pages) reads zeros.
tf_status make_page_map(void* map, const void* base, const tf_paged_kv& kv, int box_rows, int box_columns);
tf_status launch_paged_split(const PagedArgs& a, cudaStream_t s);
tf_status launch_paged_tile(const PagedArgs& a, cudaStream_t s);
// Workspace of the few-rows kernel's parts: per part and row the maximum, the
// sum, the outputs.  The tensor-core kernels' parts follow it.
inline size_t split_workspace_bytes(const tf_paged_plan& p) {
  return (size_t)p.split_parts * kSplitRows * (2 + p.head_dim) * 4;
}

struct AppendArgs {
  const void* qkv = nullptr;
  int64_t qkv_stride = 0;
  int64_t rows = 0;
  int heads = 0;
  int act = TF_DTYPE_F16;
  const void* q_norm = nullptr;
  const void* k_norm = nullptr;
  float eps = 0.f;
  float theta = 0.f;  // 0: no rotation
  const int32_t* positions = nullptr;
  const int32_t* requests = nullptr;
  tf_page_table table{};
  tf_paged_kv kv{};
  void* q_out = nullptr;
};
tf_status launch_paged_append(const AppendArgs& a, cudaStream_t s);

}  // namespace tf
