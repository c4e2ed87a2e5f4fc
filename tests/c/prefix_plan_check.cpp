// Checks the work lists of csrc/prefix_plan.h against the keep rule, pair by
// pair. Arguments: P sparse sparse_prefix window group row_tiles (1 or 2), then
// n m of each request. Prints what is wrong and exits 1, or the numbers of kept pairs and
// of tiles.
#include <cstdio>
#include <cstdlib>
#include <map>
#include <vector>

#include "prefix_plan.h"

using namespace qwa;

static int wrong(const char* what, int row, long key) {
  std::printf("%s: row %d key %ld\n", what, row, key);
  return 1;
}

int main(int argc, char** argv) {
  PrefixShape s{};
  s.prefix_len = std::atoi(argv[1]);
  s.sparse = std::atoi(argv[2]);
  s.sparse_prefix = std::atoi(argv[3]);
  s.window = std::atoi(argv[4]);
  const int group = std::atoi(argv[5]);
  s.kv_heads = 1;
  s.q_heads = group;
  s.tile_tokens = 128 / group;
  s.block_tokens = std::atoi(argv[6]) * s.tile_tokens;
  std::vector<int> cu_q(1, 0), cu_k(1, 0);
  for (int i = 7; i + 1 < argc; i += 2) {
    cu_q.push_back(cu_q.back() + std::atoi(argv[i]));
    cu_k.push_back(cu_k.back() + std::atoi(argv[i + 1]));
  }
  s.batch = static_cast<int>(cu_q.size()) - 1;
  const int P = s.prefix_len, total_k = cu_k.back(), total_q = cu_q.back();
  const PrefixWork w = build_prefix_work(s, cu_q.data(), cu_k.data());
  if (total_q && (w.gap_beg < 0 || w.gap_end < w.gap_beg || w.gap_end > P))
    return wrong("gap", w.gap_beg, w.gap_end);
  std::vector<int> seen_rows(total_q, 0);
  long pairs = 0;
  for (const PrefixItem& it : w.items) {
    if (it.tokens < 1 || it.tokens > s.block_tokens) return wrong("tokens", it.row0, it.tokens);
    if (it.tile_end <= it.tile_beg) return wrong("no tiles", it.row0, 0);
    for (int r = it.row0; r < it.row0 + it.tokens; ++r) {
      ++seen_rows[r];
      int b = 0;
      while (cu_q[b + 1] <= r) ++b;
      const int n = cu_q[b + 1] - cu_q[b], m = cu_k[b + 1] - cu_k[b], i = r - cu_q[b];
      const int pos = P + m - n + i;
      if (w.rows[r].lo != cu_k[b] || w.rows[r].hi != cu_k[b] + m - n + i)
        return wrong("row", r, w.rows[r].hi);
      auto keeps = [&](bool own, long key) {
        long at;  // position, -1: not a key of this row
        if (own) {
          if (key < cu_k[b] || key > cu_k[b] + m - n + i) return false;
          at = P + key - cu_k[b];
        } else {
          if (key < 0 || key >= P) return false;
          at = key;
        }
        return !s.sparse || at < s.sparse_prefix || at > pos - s.window;
      };
      std::vector<char> prefix_hit(P, 0), own_hit(total_k, 0);
      for (int j = it.tile_beg; j < it.tile_end; ++j) {
        const PrefixTile t = w.tiles[j];
        const bool own = t.info & kTileOwn;
        const int width = t.info & kTileWidthMask;
        const int limit = own ? total_k : P;
        if (width < 16 || width > 128 || width % 16) return wrong("width", r, width);
        if (t.key < 0 || t.key >= limit) return wrong("tile outside", r, t.key);
        if (!own && t.key < w.gap_end && std::min(t.key + width, P) > w.gap_beg)
          return wrong("tile in the gap", r, t.key);
        for (int c = 0; c < 128; ++c) {
          const long key = t.key + c;
          const bool keep = keeps(own, key);
          if (c >= width) {  // no scores there: must be masked, and nothing lost
            if (!(t.info & kTileMask)) return wrong("narrow without mask", r, key);
            if (keep) return wrong("kept past the width", r, key);
            continue;
          }
          if (!keep && !(t.info & kTileMask)) return wrong("needs mask", r, key);
          if (!keep && key < limit && !(t.info & kTileGuard)) return wrong("needs guard", r, key);
          if (keep) ++(own ? own_hit[key] : prefix_hit[key]);
        }
      }
      for (int key = 0; key < P; ++key) {
        if (prefix_hit[key] != (keeps(false, key) ? 1 : 0)) return wrong("prefix cover", r, key);
        pairs += prefix_hit[key];
      }
      for (int key = 0; key < total_k; ++key) {
        if (own_hit[key] != (keeps(true, key) ? 1 : 0)) return wrong("own cover", r, key);
        pairs += own_hit[key];
      }
    }
  }
  for (int r = 0; r < total_q; ++r)
    if (seen_rows[r] != 1) return wrong("row blocks", r, seen_rows[r]);
  if (pairs != prefix_kept_pairs(s, cu_q.data(), cu_k.data())) return wrong("pairs", 0, pairs);
  std::printf("%ld %zu\n", pairs, w.tiles.size());
  return 0;
}
