// Planner of paged attention: divides the (request, key head, packed rows) x
// key-tile work of one call over the GPU's SMs.  Host code only.
//
// Every thread block gets a list of segments up front, so the kernels need no
// work queue and a call's result does not depend on timing.  Three ways to
// divide the items are weighed by the load of the slowest block, in tiles:
//   whole   every item whole, longest first on the least loaded block;
//   even    long items cut into equal pieces of about a block's share, placed
//           the same way;
//   wrap    items laid end to end and cut into equal shares.
// A cut piece costs a partial result and its merge beside a segment's start, so
// items stay whole where they balance within 1/16 of the mean anyway.  (16
// requests of 2048 tokens on 8 key heads, 128 items for 148 blocks: whole 30
// us, wrapped 33; 24 x 5 drafted tokens over 2048, 48 items for 296: 18 us in
// pieces of at least 4 tiles, 15 of at least 2.)
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

// What a kernel's segments cost beside their tiles, in tiles.
struct Costs {
  int start;      // any segment
  int cut;        // a piece of a cut item: its partial result, its part of the merge
  int join;       // a call that cuts at all
  int min_piece;  // smallest piece worth cutting
};

// Places the pieces, in order, each on the least loaded block; most: the load
// of the slowest.
Schedule place(const std::vector<Piece>& pieces, const std::vector<int32_t>& cost, int blocks, int64_t* most) {
  Schedule out;
  // Loads as a binary heap of (load, block) in one 64-bit word; the least
  // loaded block is raised in place.
  const int used = (int)std::min<size_t>(blocks, pieces.size());
  std::vector<uint64_t> heap(used);
  for (int b = 0; b < used; ++b) heap[b] = (uint64_t)b;
  std::vector<int32_t> owner(pieces.size());
  out.starts.assign(used + 1, 0);
  *most = 0;
  for (size_t i = 0; i < pieces.size(); ++i) {
    const uint64_t load = (heap[0] >> 20) + cost[i], b = heap[0] & 0xfffff;
    owner[i] = (int32_t)b;
    ++out.starts[b + 1];
    *most = std::max<int64_t>(*most, (int64_t)load);
    const uint64_t word = load << 20 | b;
    int at = 0;
    for (int child; (child = 2 * at + 1) < used; at = child) {
      if (child + 1 < used && heap[child + 1] < heap[child]) ++child;
      if (heap[child] >= word) break;
      heap[at] = heap[child];
    }
    heap[at] = word;
  }
  for (int b = 0; b < used; ++b) out.starts[b + 1] += out.starts[b];
  out.pieces.resize(pieces.size());
  std::vector<int32_t> next(out.starts.begin(), out.starts.end());
  for (size_t i = 0; i < pieces.size(); ++i) out.pieces[next[owner[i]]++] = pieces[i];
  return out;
}

// Divides the items over at most `blocks` blocks.
Schedule divide(const std::vector<Item>& items, int kv_heads, int blocks, const Costs& c) {
  int64_t total = 0;
  for (const Item& it : items) total += it.tiles + c.start;
  const int64_t mean = std::max<int64_t>((total + blocks - 1) / blocks, c.min_piece + c.start);
  // Longest first; equal items keep their order, so one request's key heads
  // and row blocks run at the same time and share its pages through L2.  The
  // key heads of a row block follow one another with equal lengths, so they
  // are sorted as one.
  std::vector<int32_t> firsts;
  firsts.reserve(items.size() / kv_heads);
  for (size_t i = 0; i < items.size(); i += kv_heads) firsts.push_back((int32_t)i);
  const auto longer = [&](int32_t a, int32_t b) { return items[a].tiles > items[b].tiles; };
  if (!std::is_sorted(firsts.begin(), firsts.end(), longer)) std::stable_sort(firsts.begin(), firsts.end(), longer);
  std::vector<Piece> pieces;
  std::vector<int32_t> cost;
  for (int32_t f : firsts)
    for (int h = 0; h < kv_heads; ++h) {
      pieces.push_back({f + h, 0, items[f].tiles});
      cost.push_back(items[f].tiles + c.start);
    }
  int64_t most = 0;
  Schedule whole = place(pieces, cost, blocks, &most);
  if (most <= mean + mean / 16) return whole;

  const int64_t share = mean - c.start;
  pieces.clear();
  cost.clear();
  for (int32_t f : firsts) {
    const int64_t tiles = items[f].tiles;
    const int64_t n = std::max<int64_t>(1, std::min((tiles + share - 1) / share, tiles / c.min_piece));
    for (int64_t k = 0; k < n; ++k)
      for (int h = 0; h < kv_heads; ++h) {
        pieces.push_back({f + h, (int32_t)(tiles * k / n), (int32_t)(tiles * (k + 1) / n)});
        cost.push_back((int32_t)(tiles * (k + 1) / n - tiles * k / n + c.start + (n > 1 ? c.cut : 0)));
      }
  }
  int64_t most_even = 0;
  Schedule even = place(pieces, cost, blocks, &most_even);
  most_even += c.join;

  // Every cut adds a segment, and a block may close short of a full share, so
  // the share grows until the pieces fit.
  Schedule wrap;
  int64_t most_wrap = 0;
  for (int64_t room_for = mean + c.start + c.cut;; room_for += room_for / 64 + 1) {
    wrap.pieces.clear();
    wrap.starts.assign(1, 0);
    most_wrap = 0;
    int64_t load = 0;
    for (int32_t f : firsts)
      for (int h = 0; h < kv_heads; ++h) {
        const int64_t tiles = items[f].tiles;
        int64_t t = 0;
        do {
          const int64_t left = tiles - t;
          int64_t room = room_for - load - c.start - c.cut;
          if (room < c.min_piece && load > 0) {
            wrap.starts.push_back((int32_t)wrap.pieces.size());
            load = 0;
            room = room_for - c.start - c.cut;
          }
          int64_t take = std::min(left, std::max<int64_t>(room, c.min_piece));
          // No crumbs: a rest below min_piece takes as much from this piece,
          // or joins it.
          if (take < left && left - take < c.min_piece)
            take = left >= 2 * c.min_piece ? left - c.min_piece : left;
          wrap.pieces.push_back({f + h, (int32_t)t, (int32_t)(t + take)});
          load += take + c.start + (take < tiles ? c.cut : 0);
          most_wrap = std::max(most_wrap, load);
          t += take;
        } while (t < tiles);
      }
    if (load > 0) wrap.starts.push_back((int32_t)wrap.pieces.size());
    if ((int)wrap.starts.size() - 1 <= blocks) break;
  }
  most_wrap += c.join;
  if (most <= most_even && most <= most_wrap) return whole;
  return most_even <= most_wrap ? even : wrap;
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
  // In tiles of each kernel: 16 KB a small one, up to 64 KB a large one, whose
  // pieces are merged by a kernel of their own.
  const Costs costs = kind == kSplit ? Costs{2, 6, 0, 4} : Costs{1, 1, 2, 2};
  const Schedule s = divide(items, p.kv_heads, current_sms() * (kind == kHalves1 ? 2 : 1), costs);
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
