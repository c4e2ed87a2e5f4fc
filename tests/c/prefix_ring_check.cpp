// The ring of key tiles of csrc/prefix_attention.cu as the waits and arrivals of its
// roles, run in many orders: the roles end whatever the order is, a tile is copied only into
// a free slot, and the MMAs read the tile that they mean, prepared where it has to be.
// Arguments: slots preparing_warps converts (0 or 1) seed. Prints what is wrong and exits 1.
#include <cstdio>
#include <cstdlib>
#include <deque>
#include <random>
#include <vector>

#include "prefix_plan.h"

struct Barrier {  // phases that complete with `count` arrivals
  int count, pending, phase = 0;
  explicit Barrier(int n) : count(n), pending(n) {}
  void arrive() {
    if (--pending == 0) {
      pending = count;
      ++phase;
    }
  }
  bool done(int parity) const { return (phase & 1) != parity; }
};

struct Op {
  enum Kind { kWait, kArrive, kCopy, kCommit, kPrepare, kRead } kind;
  int bar;     // kWait, kArrive, kCopy (arrives as it lands), kCommit (as the MMAs end)
  int parity;  // kWait
  int slot, use, need;  // of the tile: what a copy or a preparing warp leaves, an MMA expects
};

struct Slot {
  int use = -1, copied = 0, prepared = 0, read = 0;  // of the use in it
};

int main(int, char** argv) {
  const int slots = std::atoi(argv[1]), warps = std::atoi(argv[2]);
  const bool converts = std::atoi(argv[3]) != 0;
  std::mt19937 rng(std::atoi(argv[4]));
  auto chance = [&](int n) { return static_cast<int>(rng() % n) == 0; };
  const int stages = 3, tiles = 60;
  const int arrivals = qwa::slot_empty_arrivals(warps);

  // barriers, by slot: empty, landed, ready, own_go; by stage: full, empty
  std::vector<Barrier> bars;
  auto add = [&](int n, int count) {
    const int at = static_cast<int>(bars.size());
    for (int i = 0; i < n; ++i) bars.emplace_back(count);
    return at;
  };
  const int empty = add(slots, arrivals), landed = add(slots, 1), ready = add(slots, warps),
            own_go = add(slots, 1), full = add(stages, 1), stage_empty = add(stages, warps);

  // the tiles: runs with and without a guard, prefix first
  const bool rare = chance(2);
  const int prefix_tiles = converts ? static_cast<int>(rng() % tiles) : 0;
  std::vector<int> guard(tiles);
  for (int j = 0; j < tiles; ++j) guard[j] = rare ? chance(20) || j == tiles - 1 : chance(2);

  // roles: producer, issuer, preparing warps; each a list of what it does in order
  std::vector<std::vector<Op>> roles(2 + warps);
  auto wait = [&](int role, int bar, int parity) {
    roles[role].push_back({Op::kWait, bar, parity & 1, 0, 0, 0});
  };
  auto arrive = [&](int role, int bar) { roles[role].push_back({Op::kArrive, bar, 0, 0, 0, 0}); };
  std::vector<int> copies(slots, 0), prepared(slots, 0), gos(slots, 0);  // phases so far
  int raw = 0, prev_v = -1;
  for (int j = 0, use = 0; j < tiles; ++j) {
    const bool convert = converts && j < prefix_tiles;
    for (int kv = 0; kv < 2; ++kv, ++use) {
      const int s = use % slots, turn = use / slots, g = raw % stages;
      const bool prepare = convert || (kv == 1 && guard[j]);
      // producer
      if (convert) {
        wait(0, stage_empty + g, (raw / stages + 1) & 1);
        roles[0].push_back({Op::kCopy, full + g, 0, -1, 0, 0});
      } else {
        if (converts) wait(0, own_go + s, gos[s]);
        else wait(0, empty + s, turn + 1);
        roles[0].push_back({Op::kCopy, landed + s, 0, s, use, 0});
      }
      // issuer: S of both row tiles, the PV of the tile before between them
      wait(1, prepare ? ready + s : landed + s, prepare ? prepared[s] : copies[s]);
      roles[1].push_back({Op::kRead, 0, 0, s, use, prepare ? warps : 0});
      if (kv == 0) {
        if (prev_v >= 0) roles[1].push_back({Op::kCommit, empty + prev_v, 0, prev_v, 0, 0});
        roles[1].push_back({Op::kCommit, empty + s, 0, s, 0, 0});
      } else {
        prev_v = s;
        if (j == tiles - 1) roles[1].push_back({Op::kCommit, empty + s, 0, s, 0, 0});
      }
      // preparing warps
      for (int w = 0; w < warps; ++w) {
        const int r = 2 + w;
        wait(r, empty + s, turn + 1);
        if (convert) {
          wait(r, full + g, raw / stages);
          roles[r].push_back({Op::kPrepare, 0, 0, s, use, 0});
          arrive(r, ready + s);
          arrive(r, stage_empty + g);
        } else {
          if (converts && w == 0) arrive(r, own_go + s);
          if (prepare) {
            wait(r, landed + s, copies[s]);
            roles[r].push_back({Op::kPrepare, 0, 0, s, use, 1});
            arrive(r, ready + s);
          }
        }
        if (arrivals > 1) arrive(r, empty + s);
      }
      if (prepare) ++prepared[s];
      if (convert) ++raw;
      else ++copies[s], ++gos[s];
    }
  }

  // any order: a role that is held back moves only when nothing else can, or at random
  const int held = chance(2) ? static_cast<int>(rng() % roles.size()) : -1;
  std::vector<size_t> at(roles.size(), 0);
  std::vector<Op> flying;    // copies, landing in any order
  std::deque<Op> committed;  // MMAs, ending in order
  std::vector<Slot> ring(slots);
  auto wrong = [&](const char* what, int use) {
    std::printf("%s (tile use %d of %d)\n", what, use, 2 * tiles);
    return 1;
  };
  while (true) {
    std::vector<int> can;
    bool over = flying.empty() && committed.empty();
    for (size_t r = 0; r < roles.size(); ++r) {
      if (at[r] == roles[r].size()) continue;
      over = false;
      const Op& op = roles[r][at[r]];
      if (op.kind != Op::kWait || bars[op.bar].done(op.parity)) can.push_back(static_cast<int>(r));
    }
    if (over) return 0;
    const int events = !flying.empty() + !committed.empty();
    if (can.empty() && events == 0) {
      std::printf("no role can move; steps done:");
      for (size_t n : at) std::printf(" %zu", n);
      std::printf("\n");
      return 1;
    }
    if (can.size() + events > 1)  // something else can move
      for (size_t i = 0; i < can.size(); ++i)
        if (can[i] == held) can.erase(can.begin() + i--);
    const size_t pick = rng() % (can.size() + events);
    if (pick < can.size()) {
      const Op& op = roles[can[pick]][at[can[pick]]++];
      if (op.kind == Op::kArrive) bars[op.bar].arrive();
      if (op.kind == Op::kCommit) committed.push_back(op);
      if (op.kind == Op::kCopy) flying.push_back(op);
      if (op.kind == Op::kPrepare) {
        Slot& s = ring[op.slot];
        if (op.need) {  // a guarded tile that has been copied
          if (s.use != op.use || !s.copied) return wrong("prepared another tile", op.use);
        } else if (s.use != op.use) {  // the first warp to convert into the slot
          if (s.use >= 0 && !s.read) return wrong("converted into a slot in use", op.use);
          s = Slot{op.use, 0, 0, 0};
        }
        ++s.prepared;
      }
      if (op.kind == Op::kRead) {
        const Slot& s = ring[op.slot];
        if (s.use != op.use) return wrong("read another tile", op.use);
        if (op.need ? s.prepared != op.need : !s.copied) return wrong("read too early", op.use);
      }
    } else if (pick == can.size() && !flying.empty()) {
      const size_t i = rng() % flying.size();
      const Op op = flying[i];
      flying.erase(flying.begin() + i);
      if (op.slot >= 0) {
        if (ring[op.slot].use >= 0 && !ring[op.slot].read)
          return wrong("copied into a slot in use", op.use);
        ring[op.slot] = Slot{op.use, 1, 0, 0};
      }
      bars[op.bar].arrive();
    } else {
      ring[committed.front().slot].read = 1;
      bars[committed.front().bar].arrive();
      committed.pop_front();
    }
  }
}
