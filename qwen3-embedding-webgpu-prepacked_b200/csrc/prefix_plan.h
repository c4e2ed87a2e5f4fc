// Work lists of the shared-prefix attention (host, plain C++).
//
// The query rows of all requests are cut into blocks of `block_tokens`
// consecutive packed tokens, whatever request they belong to: every row sees
// the prefix, so a prefix tile multiplied for a block serves up to
// block_tokens rows however short the requests are. A block's keys are listed
// as tiles of at most 128: tiles of the prefix, then tiles of the packed own
// keys; only tiles with a pair that some row keeps are listed. The lists are
// the same for every kv head.
//
// Kept keys of own query i of a request with n queries and m own keys (m >=
// n, the queries are the last n), at position p = P + m - n + i:
//   full:   prefix keys [0, P) and own keys [0, m - n + i]
//   sparse: of those, the keys at a position < sparse_prefix or > p - window
#pragma once
#include <algorithm>
#include <cstdint>
#include <vector>

namespace qwa {

// One key tile: rows [key, key + width) of the prefix or of the packed own
// keys; width is a multiple of 16 (the MMA's N granularity).
struct PrefixTile {
  int32_t key;
  int32_t info;  // width | kTile* flags
};
constexpr int kTileWidthMask = 0xff;
constexpr int kTileOwn = 1 << 8;    // own keys, not the prefix
// some row drops a column of the tile, or the tile is narrow: its columns past
// the width hold no scores
constexpr int kTileMask = 1 << 9;
// some row drops a key that is in the tensor: values that are not finite in
// its V must not reach that row as 0 * inf
constexpr int kTileGuard = 1 << 10;

// A block of rows and its tiles, for one kv head.
struct PrefixItem {
  int32_t row0;      // first packed query token
  int32_t tokens;    // 1 .. block_tokens
  int32_t head;      // kv head
  int32_t tile_beg;  // tiles [tile_beg, tile_end) of the list
  int32_t tile_end;
  int32_t pad[3];
};

// Kept own keys of one query: packed key rows [lo, hi] (hi its own).
struct PrefixRow {
  int32_t lo, hi;
};

struct PrefixShape {
  int batch, q_heads, kv_heads, prefix_len, sparse, sparse_prefix, window;
  int tile_tokens;   // tokens of one 128-row tile: 128 / (q_heads / kv_heads)
  int block_tokens;  // of a block: tile_tokens or 2 * tile_tokens
};

// Measured: a key tile of a block of two row tiles, and of a block of one (dual), in
// us.
constexpr double kTileUs = 2.14, kDualTileUs = 1.325;

// Arrivals that free a slot of the kernel's ring of key tiles: the commit of the MMAs
// that read it, and each preparing warp's, once it is done with that use. A parity tells
// two neighbouring phases apart and no more. Without their arrivals nothing waited
// for the preparing warps on tiles that need no preparing, and one that was late by a
// whole ring would have taken a phase for the one before it, and never caught up.
constexpr int slot_empty_arrivals(int prep_warps) { return 1 + prep_warps; }

struct PrefixWork {
  std::vector<PrefixItem> items;  // without the head; one per block
  std::vector<PrefixTile> tiles;
  std::vector<PrefixRow> rows;
  std::vector<double> cost;       // of an item among others, us (on a B200)
  // prefix keys that no tile reaches: [gap_beg, gap_end)
  int gap_beg = 0, gap_end = 0;
};

inline int prefix_tile_width(int keys) { return std::min(128, (keys + 15) / 16 * 16); }

// kept pairs of one query head
inline int64_t prefix_kept_pairs(const PrefixShape& s, const int32_t* cu_q, const int32_t* cu_k) {
  int64_t pairs = 0;
  for (int b = 0; b < s.batch; ++b) {
    const int64_t n = cu_q[b + 1] - cu_q[b], m = cu_k[b + 1] - cu_k[b];
    for (int64_t i = 0; i < n; ++i) {
      const int64_t seen = s.prefix_len + m - n + i + 1;
      if (!s.sparse || seen <= s.window) {
        pairs += seen;
        continue;
      }
      pairs += std::min<int64_t>(s.sparse_prefix, seen - s.window) + s.window;
    }
  }
  return pairs;
}

inline PrefixWork build_prefix_work(const PrefixShape& s, const int32_t* cu_q,
                                    const int32_t* cu_k) {
  PrefixWork w;
  const int total = cu_q[s.batch];
  const int P = s.prefix_len;
  // sparse_prefix reaches into the own keys by this many
  const int64_t own_prefix = s.sparse ? std::max(0, s.sparse_prefix - P) : 0;
  w.rows.resize(total);
  std::vector<int> request_of(total);
  for (int b = 0; b < s.batch; ++b) {
    const int n = cu_q[b + 1] - cu_q[b], m = cu_k[b + 1] - cu_k[b];
    for (int i = 0; i < n; ++i) {
      w.rows[cu_q[b] + i] = {cu_k[b], cu_k[b] + m - n + i};
      request_of[cu_q[b] + i] = b;
    }
  }
  // tiles begin at the first key of a span, and reach at most 128 keys on
  w.gap_beg = s.sparse ? std::min(P, (s.sparse_prefix + 127) / 128 * 128) : P;
  w.gap_end = P;
  struct Segment {  // the rows of one request inside a block
    int lo, first_hi, last_hi;
  };
  struct Span {
    int64_t beg, end;
  };
  std::vector<Segment> segs;
  std::vector<Span> spans;
  auto add_span = [&](int64_t beg, int64_t end) {
    if (beg >= end) return;
    if (!spans.empty() && beg <= spans.back().end) {
      spans.back().end = std::max(spans.back().end, end);
      return;
    }
    spans.push_back({beg, end});
  };
  for (int row0 = 0; row0 < total; row0 += s.block_tokens) {
    const int tokens = std::min(s.block_tokens, total - row0);
    segs.clear();
    for (int r = row0; r < row0 + tokens;) {
      const int b = request_of[r];
      const int end = std::min(row0 + tokens, static_cast<int>(cu_q[b + 1]));
      segs.push_back({w.rows[r].lo, w.rows[r].hi, w.rows[end - 1].hi});
      r = end;
    }
    PrefixItem item{};
    item.row0 = row0;
    item.tokens = tokens;
    item.tile_beg = static_cast<int>(w.tiles.size());
    double cost = 0;
    auto emit = [&](int own) {
      int64_t next = 0;
      for (size_t i = 0; i < spans.size();) {
        const int64_t key = std::max(spans[i].beg, next);
        if (key >= spans[i].end) {
          ++i;
          continue;
        }
        // the last key that this tile has to reach
        int64_t last = key;
        for (size_t j = i; j < spans.size() && spans[j].beg < key + 128; ++j)
          last = std::min<int64_t>(spans[j].end, key + 128) - 1;
        const int width = prefix_tile_width(static_cast<int>(last - key + 1));
        bool mask = false, guard = false;
        if (!own) {
          if (s.sparse) {
            int64_t p_max = 0;
            for (const Segment& g : segs)
              p_max = std::max<int64_t>(p_max, static_cast<int64_t>(P) + g.last_hi - g.lo);
            const int64_t end = std::min<int64_t>(key + width, P);
            guard = !(end <= s.sparse_prefix || key + s.window > p_max);
          }
          mask = guard || key + width > P || width < 128;
        } else {
          for (const Segment& g : segs) {
            bool all = key >= g.lo && key + width - 1 <= g.first_hi;
            if (s.sparse)
              all = all && (key + s.window > g.last_hi || key + width <= g.lo + own_prefix);
            guard = guard || !all;
          }
          mask = guard || width < 128;
        }
        w.tiles.push_back({static_cast<int32_t>(key),
                           width | (own ? kTileOwn : 0) | (mask ? kTileMask : 0) |
                               (guard ? kTileGuard : 0)});
        cost += 0.35 + 0.65 * width / 128.0;
        next = key + 128;
      }
    };
    // prefix keys
    spans.clear();
    if (!s.sparse) {
      add_span(0, P);
    } else {
      int64_t p_min = INT64_MAX;
      for (const Segment& g : segs)
        p_min = std::min<int64_t>(p_min, static_cast<int64_t>(P) + g.first_hi - g.lo);
      add_span(0, std::min<int64_t>(P, s.sparse_prefix));
      add_span(std::max<int64_t>(0, p_min - s.window + 1), P);
      w.gap_end = static_cast<int>(
          std::min<int64_t>(w.gap_end, std::max<int64_t>(0, p_min - s.window + 1)));
    }
    emit(0);
    // own keys, request by request (their packed rows ascend)
    spans.clear();
    for (const Segment& g : segs) {
      if (!s.sparse) {
        add_span(g.lo, g.last_hi + 1ll);
        continue;
      }
      add_span(g.lo, std::min<int64_t>(g.last_hi + 1ll, g.lo + own_prefix));
      add_span(std::max<int64_t>(g.lo, static_cast<int64_t>(g.first_hi) - s.window + 1),
               g.last_hi + 1ll);
    }
    emit(1);
    item.tile_end = static_cast<int>(w.tiles.size());
    w.items.push_back(item);
    const int n = item.tile_end - item.tile_beg;
    w.cost.push_back(s.block_tokens == s.tile_tokens ? 2.0 + kDualTileUs * n
                                                     : 3.0 + kTileUs * cost);
  }
  w.gap_end = std::max(w.gap_end, w.gap_beg);
  return w;
}

}  // namespace qwa
