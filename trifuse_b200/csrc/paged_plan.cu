// Planner of paged attention: divides the (request, key head, packed rows) x
// key-tile work of one call over the GPU's SMs.  Host code only.
//
// Every thread block gets a list of segments up front, so the kernels need no
// work queue and a call's result does not depend on timing.  Whole items are
// first placed longest-first on the least loaded block.  Where that leaves the
// slowest block more than 1/16 above the mean (few or very unequal items),
// the items are instead laid end to end and cut into equal shares; the pieces
// of a cut item leave partial results that the last of them to finish merges.
// A cut costs the partial results' traffic and the merge, a few percent of a
// long item, so items stay whole where they balance anyway.
#include <string.h>

#include <algorithm>
#include <vector>

#include "paged.h"

namespace tf {

namespace {

struct Item {
  int32_t request, kv_head, row0, rows, q_row, tiles;
};

struct Piece {
  int32_t item, tile0, tile1;
};

// Pieces of all blocks, block by block.
struct Schedule {
  std::vector<Piece> pieces;
  std::vector<int32_t> starts;  // first piece of each block, then the end
};

int current_sms() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) {
    cudaGetLastError();  // no device here: a plan may still be laid out for inspection
    return 148;
  }
  return n;
}

// Divides the items over at most `blocks` blocks.  overhead: cost of starting
// a segment, in tiles; min_piece: smallest piece worth cutting, in tiles.
Schedule divide(const std::vector<Item>& items, int kv_heads, int blocks, int overhead, int min_piece) {
  Schedule out;
  int64_t total = 0;
  for (const Item& it : items) total += it.tiles + overhead;
  const int64_t mean = std::max<int64_t>((total + blocks - 1) / blocks, min_piece + overhead);
  // Longest first; equal items keep their order, so one request's key heads
  // and row blocks run at the same time and share its pages through L2.  The
  // key heads of a row block follow one another with equal lengths, so they
  // are sorted as one.
  std::vector<int32_t> order(items.size()), firsts;
  firsts.reserve(items.size() / kv_heads);
  for (size_t i = 0; i < items.size(); i += kv_heads) firsts.push_back((int32_t)i);
  const auto longer = [&](int32_t a, int32_t b) { return items[a].tiles > items[b].tiles; };
  if (!std::is_sorted(firsts.begin(), firsts.end(), longer)) std::stable_sort(firsts.begin(), firsts.end(), longer);
  for (size_t i = 0; i < order.size(); ++i) order[i] = firsts[i / kv_heads] + (int32_t)(i % kv_heads);
  // Loads as a binary heap of (load, block) in one 64-bit word; the least
  // loaded block is raised in place.
  const int used = (int)std::min<size_t>(blocks, items.size());
  std::vector<uint64_t> heap(used);
  for (int b = 0; b < used; ++b) heap[b] = (uint64_t)b;
  std::vector<int32_t> owner(items.size()), count(used + 1, 0);
  uint64_t most = 0;
  for (int32_t i : order) {
    const uint64_t load = (heap[0] >> 20) + items[i].tiles + overhead;
    const uint64_t b = heap[0] & 0xfffff;
    owner[i] = (int32_t)b;
    ++count[b + 1];
    most = std::max(most, load);
    const uint64_t word = load << 20 | b;
    int at = 0;
    for (int child; (child = 2 * at + 1) < used; at = child) {
      if (child + 1 < used && heap[child + 1] < heap[child]) ++child;
      if (heap[child] >= word) break;
      heap[at] = heap[child];
    }
    heap[at] = word;
  }
  if ((int64_t)most <= mean + mean / 16) {
    for (int b = 0; b < used; ++b) count[b + 1] += count[b];
    out.starts = count;
    out.pieces.resize(items.size());
    for (int32_t i : order) out.pieces[count[owner[i]]++] = {i, 0, items[i].tiles};
    return out;
  }
  // Every cut adds a segment, and a block may close short of a full share, so
  // the share grows until the pieces fit.
  for (int64_t share = mean + overhead;; share += share / 64 + 1) {
    out.pieces.clear();
    out.starts.assign(1, 0);
    int64_t load = 0;
    for (int32_t i : order) {
      int32_t t = 0;
      do {
        const int64_t left = items[i].tiles - t;
        int64_t room = share - load - overhead;
        if (room < min_piece && load > 0) {
          out.starts.push_back((int32_t)out.pieces.size());
          load = 0;
          room = share - overhead;
        }
        int64_t take = std::min(left, room);
        // No crumbs: a rest below min_piece joins this piece.
        if (left - take < min_piece) take = left;
        out.pieces.push_back({i, t, (int32_t)(t + take)});
        load += take + overhead;
        t += (int32_t)take;
      } while (t < items[i].tiles);
    }
    if (load > 0) out.starts.push_back((int32_t)out.pieces.size());
    if ((int)out.starts.size() - 1 <= blocks) return out;
  }
}

struct Layout {
  std::vector<PagedSegment> segments;
  std::vector<int32_t> starts;  // first segment of each block, then the end
  int32_t parts = 0;
  int32_t counters = 0;
};

Layout lay_out(const std::vector<Item>& items, const Schedule& s, const int32_t* new_lengths,
               const int32_t* kv_lengths) {
  Layout out;
  std::vector<int32_t> pieces(items.size(), 0), part0(items.size(), -1), used(items.size(), 0),
      counter(items.size(), -1);
  for (const Piece& p : s.pieces) ++pieces[p.item];
  for (size_t i = 0; i < items.size(); ++i)
    if (pieces[i] > 1) {
      part0[i] = out.parts;
      out.parts += pieces[i];
      counter[i] = out.counters++;
    }
  out.segments.reserve(s.pieces.size());
  for (const Piece& p : s.pieces) {
    const Item& it = items[p.item];
    PagedSegment g{};
    g.q_row = it.q_row;
    g.new_len = new_lengths[it.request];
    g.kv_len = kv_lengths[it.request];
    g.request = it.request;
    g.kv_head = it.kv_head;
    g.row0 = it.row0;
    g.rows = it.rows;
    g.tile0 = p.tile0;
    g.tile1 = p.tile1;
    g.part = part0[p.item] < 0 ? -1 : part0[p.item] + used[p.item]++;
    g.part0 = part0[p.item];
    g.parts = pieces[p.item];
    g.counter = counter[p.item];
    out.segments.push_back(g);
  }
  out.starts = s.starts;
  return out;
}

// The work of one kernel, chosen by a request's packed rows per key head: up to
// kSplitRows go to the few-rows kernel, up to kHalfRows to the tensor-core
// kernel with one half a block and two blocks an SM, more to the one with two
// halves.
enum Kind { kSplit, kHalves1, kHalves2 };

Layout plan_kernel(const int32_t* new_lengths, const int32_t* kv_lengths, const tf_paged_plan& p, Kind kind) {
  const int G = p.heads / p.kv_heads;
  const int block_rows = kind == kSplit ? kSplitRows : kind == kHalves1 ? kHalfRows : kTileRows;
  const int keys = kind == kSplit ? kSplitKeys : kTileKeys;
  std::vector<Item> items;
  int32_t q_row = 0;
  for (int r = 0; r < p.requests; ++r) {
    const int n = new_lengths[r], kv = kv_lengths[r];
    const int64_t rows = (int64_t)n * G;
    if ((rows <= kSplitRows ? kSplit : rows <= kHalfRows ? kHalves1 : kHalves2) == kind)
      for (int64_t row0 = 0; row0 < rows; row0 += block_rows) {
        const int take = (int)std::min<int64_t>(block_rows, rows - row0);
        const int64_t last = (int64_t)kv - n + (row0 + take - 1) / G;  // last key the rows see
        const int32_t tiles = last < 0 ? 0 : (int32_t)(last / keys + 1);
        for (int h = 0; h < p.kv_heads; ++h) items.push_back({r, h, (int32_t)row0, take, q_row, tiles});
      }
    q_row += n;
  }
  // A segment starts in the time of some four small or one large tile; a piece
  // should be worth its partial result (a large tile's keys and values are as
  // many bytes as half a partial result of 256 rows).
  const Schedule s = kind == kSplit ? divide(items, p.kv_heads, current_sms(), 4, 8)
                                    : divide(items, p.kv_heads, current_sms() * (kind == kHalves1 ? 2 : 1), 1, 4);
  return lay_out(items, s, new_lengths, kv_lengths);
}

struct Plans {
  Layout split, half, tile;
  std::vector<PagedSegment> half_merges, tile_merges;
  Plans(const int32_t* new_lengths, const int32_t* kv_lengths, const tf_paged_plan& p)
      : split(plan_kernel(new_lengths, kv_lengths, p, kSplit)),
        half(plan_kernel(new_lengths, kv_lengths, p, kHalves1)),
        tile(plan_kernel(new_lengths, kv_lengths, p, kHalves2)),
        half_merges(cut(half)),
        tile_merges(cut(tile)) {}
  static std::vector<PagedSegment> cut(const Layout& l) {
    std::vector<PagedSegment> out;
    for (const PagedSegment& g : l.segments)
      if (g.part >= 0 && g.part == g.part0) out.push_back(g);
    return out;
  }
};

template <typename V>
size_t put(char* table, size_t at, const std::vector<V>& v) {
  if (table && !v.empty()) memcpy(table + at, v.data(), v.size() * sizeof(V));
  return align_up(at + v.size() * sizeof(V), 16);
}

// Lays the table out, and fills it where `table` is given: the few-rows
// kernel's arrival counters (zero between calls), the kernels' segments, block
// starts and cut row blocks, the rows' positions and requests.
void put_table(const Plans& plans, const int32_t* new_lengths, const int32_t* kv_lengths, tf_paged_plan* p,
               char* table) {
  p->split_blocks = (int32_t)plans.split.starts.size() - 1;
  p->split_parts = plans.split.parts;
  p->split_counters = plans.split.counters;
  p->split_rows = 0;
  for (const PagedSegment& g : plans.split.segments) p->split_rows = std::max(p->split_rows, g.rows);
  p->tile_blocks = (int32_t)plans.tile.starts.size() - 1;
  p->tile_parts = plans.tile.parts;
  p->tile_merges = (int32_t)plans.tile_merges.size();
  p->half_blocks = (int32_t)plans.half.starts.size() - 1;
  p->half_parts = plans.half.parts;
  p->half_merges = (int32_t)plans.half_merges.size();
  size_t at = put(table, 0, std::vector<int32_t>(plans.split.counters, 0));
  p->split_segments_offset = (int64_t)at;
  at = put(table, at, plans.split.segments);
  p->split_starts_offset = (int64_t)at;
  at = put(table, at, plans.split.starts);
  p->tile_segments_offset = (int64_t)at;
  at = put(table, at, plans.tile.segments);
  p->tile_starts_offset = (int64_t)at;
  at = put(table, at, plans.tile.starts);
  p->tile_merges_offset = (int64_t)at;
  at = put(table, at, plans.tile_merges);
  p->half_segments_offset = (int64_t)at;
  at = put(table, at, plans.half.segments);
  p->half_starts_offset = (int64_t)at;
  at = put(table, at, plans.half.starts);
  p->half_merges_offset = (int64_t)at;
  at = put(table, at, plans.half_merges);
  p->positions_offset = (int64_t)at;
  at = align_up(at + (size_t)p->rows * 4, 16);
  p->requests_offset = (int64_t)at;
  p->table_bytes = align_up(at + (size_t)p->rows * 4, 16);
  p->workspace_bytes = split_workspace_bytes(*p) +
                       ((size_t)p->tile_parts * kTileRows + (size_t)p->half_parts * kHalfRows) * (2 + p->head_dim) * 4;
  if (!table) return;
  int32_t* pos = reinterpret_cast<int32_t*>(table + p->positions_offset);
  int32_t* req = reinterpret_cast<int32_t*>(table + p->requests_offset);
  for (int r = 0; r < p->requests; ++r)
    for (int i = 0; i < new_lengths[r]; ++i) {
      *pos++ = kv_lengths[r] - new_lengths[r] + i;
      *req++ = r;
    }
}

}  // namespace

tf_status paged_plan_make(const int32_t* new_lengths, const int32_t* kv_lengths, tf_paged_plan* p, char* table,
                          size_t table_capacity) {
  const Plans plans(new_lengths, kv_lengths, *p);
  put_table(plans, new_lengths, kv_lengths, p, nullptr);
  if (p->table_bytes > table_capacity)
    return set_error(TF_ERR_CAPACITY, "paged plan: table of %zu bytes, %zu needed", table_capacity, p->table_bytes);
  memset(table, 0, p->table_bytes);
  put_table(plans, new_lengths, kv_lengths, p, table);
  return TF_OK;
}

}  // namespace tf
