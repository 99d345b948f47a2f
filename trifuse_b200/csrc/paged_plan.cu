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
#include <queue>
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

struct Schedule {
  std::vector<std::vector<Piece>> blocks;
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
Schedule divide(const std::vector<Item>& items, int blocks, int overhead, int min_piece) {
  Schedule out;
  int64_t total = 0;
  for (const Item& it : items) total += it.tiles + overhead;
  const int64_t mean = std::max<int64_t>((total + blocks - 1) / blocks, min_piece + overhead);
  std::vector<int32_t> order(items.size());
  for (size_t i = 0; i < order.size(); ++i) order[i] = (int32_t)i;
  // Longest first; equal items keep their order, so one request's key heads
  // and row blocks run at the same time and share its pages through L2.
  std::stable_sort(order.begin(), order.end(),
                   [&](int32_t a, int32_t b) { return items[a].tiles > items[b].tiles; });
  std::vector<std::vector<Piece>> whole(std::min<size_t>(blocks, items.size()));
  using Load = std::pair<int64_t, int32_t>;
  std::priority_queue<Load, std::vector<Load>, std::greater<Load>> loads;
  for (size_t b = 0; b < whole.size(); ++b) loads.push({0, (int32_t)b});
  int64_t most = 0;
  for (int32_t i : order) {
    Load l = loads.top();
    loads.pop();
    whole[l.second].push_back({i, 0, items[i].tiles});
    l.first += items[i].tiles + overhead;
    most = std::max(most, l.first);
    loads.push(l);
  }
  if (most <= mean + mean / 16) {
    out.blocks = std::move(whole);
    return out;
  }
  // Every cut adds a segment, and a block may close short of a full share, so
  // the share grows until the pieces fit.
  for (int64_t share = mean + overhead;; share += share / 64 + 1) {
    out.blocks.clear();
    std::vector<Piece> cur;
    int64_t load = 0;
    for (int32_t i : order) {
      int32_t t = 0;
      do {
        const int64_t left = items[i].tiles - t;
        int64_t room = share - load - overhead;
        if (room < min_piece && !cur.empty()) {
          out.blocks.push_back(std::move(cur));
          cur.clear();
          load = 0;
          room = share - overhead;
        }
        int64_t take = std::min(left, room);
        // No crumbs: a rest below min_piece joins this piece.
        if (left - take < min_piece) take = left;
        cur.push_back({i, t, (int32_t)(t + take)});
        load += take + overhead;
        t += (int32_t)take;
      } while (t < items[i].tiles);
    }
    if (!cur.empty()) out.blocks.push_back(std::move(cur));
    if ((int)out.blocks.size() <= blocks) return out;
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
  for (const auto& b : s.blocks)
    for (const Piece& p : b) ++pieces[p.item];
  for (size_t i = 0; i < items.size(); ++i)
    if (pieces[i] > 1) {
      part0[i] = out.parts;
      out.parts += pieces[i];
      counter[i] = out.counters++;
    }
  for (const auto& b : s.blocks) {
    out.starts.push_back((int32_t)out.segments.size());
    for (const Piece& p : b) {
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
  }
  out.starts.push_back((int32_t)out.segments.size());
  return out;
}

// The work of one kernel: requests of more than kSplitRows packed rows per key
// head go to the tensor-core kernel (whose 128-row products take the same time
// however few rows they hold), the others to the few-rows kernel.
Layout plan_kernel(const int32_t* new_lengths, const int32_t* kv_lengths, const tf_paged_plan& p, bool tile) {
  const int G = p.heads / p.kv_heads;
  const int block_rows = tile ? kTileRows : kSplitRows, keys = tile ? kTileKeys : kSplitKeys;
  std::vector<Item> items;
  int32_t q_row = 0;
  for (int r = 0; r < p.requests; ++r) {
    const int n = new_lengths[r], kv = kv_lengths[r];
    const int64_t rows = (int64_t)n * G;
    if ((rows > kSplitRows) == tile)
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
  // many bytes as half a partial result).
  const Schedule s = tile ? divide(items, current_sms(), 1, 4) : divide(items, current_sms(), 4, 8);
  return lay_out(items, s, new_lengths, kv_lengths);
}

struct Plans {
  Layout split, tile;
  std::vector<PagedSegment> merges;
  Plans(const int32_t* new_lengths, const int32_t* kv_lengths, const tf_paged_plan& p)
      : split(plan_kernel(new_lengths, kv_lengths, p, false)), tile(plan_kernel(new_lengths, kv_lengths, p, true)) {
    for (const PagedSegment& g : tile.segments)
      if (g.part >= 0 && g.part == g.part0) merges.push_back(g);
  }
};

template <typename V>
size_t put(char* table, size_t at, const std::vector<V>& v) {
  if (table && !v.empty()) memcpy(table + at, v.data(), v.size() * sizeof(V));
  return align_up(at + v.size() * sizeof(V), 16);
}

// Lays the table out, and fills it where `table` is given: the few-rows
// kernel's arrival counters (zero between calls), the two kernels' segments and
// block starts, the cut row blocks, the rows' positions and requests.
void put_table(const Plans& plans, const int32_t* new_lengths, const int32_t* kv_lengths, tf_paged_plan* p,
               char* table) {
  p->split_blocks = (int32_t)plans.split.starts.size() - 1;
  p->split_parts = plans.split.parts;
  p->split_counters = plans.split.counters;
  p->tile_blocks = (int32_t)plans.tile.starts.size() - 1;
  p->tile_parts = plans.tile.parts;
  p->merges = (int32_t)plans.merges.size();
  size_t at = put(table, 0, std::vector<int32_t>(plans.split.counters, 0));
  p->split_segments_offset = (int64_t)at;
  at = put(table, at, plans.split.segments);
  p->split_starts_offset = (int64_t)at;
  at = put(table, at, plans.split.starts);
  p->tile_segments_offset = (int64_t)at;
  at = put(table, at, plans.tile.segments);
  p->tile_starts_offset = (int64_t)at;
  at = put(table, at, plans.tile.starts);
  p->merges_offset = (int64_t)at;
  at = put(table, at, plans.merges);
  p->positions_offset = (int64_t)at;
  at = align_up(at + (size_t)p->rows * 4, 16);
  p->requests_offset = (int64_t)at;
  p->table_bytes = align_up(at + (size_t)p->rows * 4, 16);
  p->workspace_bytes = split_workspace_bytes(*p) + (size_t)p->tile_parts * kTileRows * (2 + p->head_dim) * 4;
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

tf_status paged_plan_size(const int32_t* new_lengths, const int32_t* kv_lengths, tf_paged_plan* p) {
  put_table(Plans(new_lengths, kv_lengths, *p), new_lengths, kv_lengths, p, nullptr);
  return TF_OK;
}

tf_status paged_plan_fill(const int32_t* new_lengths, const int32_t* kv_lengths, const tf_paged_plan* p,
                          char* table) {
  const Plans plans(new_lengths, kv_lengths, *p);
  tf_paged_plan again = *p;
  put_table(plans, new_lengths, kv_lengths, &again, nullptr);
  if (memcmp(&again, p, sizeof(again)))
    return set_error(TF_ERR_STATE, "paged plan: lengths or device differ from those the plan was sized for");
  memset(table, 0, p->table_bytes);
  put_table(plans, new_lengths, kv_lengths, &again, table);
  return TF_OK;
}

}  // namespace tf
