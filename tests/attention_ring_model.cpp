// Host model of the 16-row attention kernel's query ring: a loader and consumers with the kernel's own
// turns (lm_attn_ring.cuh), over barriers whose waits see a phase's parity only. Every order in which the
// sides can take their steps is searched, for every pattern of segments with and without keys.
//   model turns     the kernel's protocol
//   model segments  the mistake that the test plants: buffer and parity by the segment's number, the
//                   consumers arriving in the loader's place for a segment without keys. Its consumers
//                   end each segment together, as the kernel's barriers have it; the turns hold without
// Prints the number of patterns, and of patterns in which a consumer reads another segment's queries or
// the sides wait for one another.
#include <cstdio>
#include <cstring>
#include <set>
#include <vector>

#include "lm_attn_ring.cuh"

namespace {

constexpr int kConsumers = 2;

struct Barrier {
  int count, arrived = 0, phase = 0;
  void arrive() {
    if (++arrived == count) {
      arrived = 0;
      ++phase;
    }
  }
  bool passes(unsigned parity) const { return (phase & 1u) != parity; }
};

struct Side {
  int segment = 0, step = 0;
  lm::AttnQueryTurn turn;
};

struct State {
  Barrier full[2], empty[2];
  int held[2] = {-1, -1};
  Side side[1 + kConsumers];  // 0: the loader
  State() {
    for (int i = 0; i < 2; ++i) full[i].count = 1, empty[i].count = kConsumers;
  }
  std::vector<int> key() const {
    std::vector<int> k;
    for (int i = 0; i < 2; ++i)
      for (int v : {full[i].arrived, full[i].phase, empty[i].arrived, empty[i].phase, held[i]}) k.push_back(v);
    for (const Side& s : side)
      for (int v : {s.segment, s.step, s.turn.taken}) k.push_back(v);
    return k;
  }
};

bool by_segment;  // the planted mistake

int buffer_of(const Side& s) { return by_segment ? s.segment & 1 : s.turn.buffer(); }
unsigned full_parity(const Side& s) { return by_segment ? (s.segment >> 1) & 1u : s.turn.full_parity(); }
unsigned empty_parity(const Side& s) { return by_segment ? full_parity(s) ^ 1u : s.turn.empty_parity(); }

enum Outcome { kBlocked, kMoved, kWrong };

void leave(Side& s, bool keys) {
  if (keys) s.turn.next();
  ++s.segment;
  s.step = 0;
}

// One step of a side: the wait, then (a step later, so that others may come between) what follows it.
Outcome advance(State& st, int who, const std::vector<int>& blocks) {
  Side& s = st.side[who];
  if (s.segment == static_cast<int>(blocks.size())) return kBlocked;
  if (by_segment && who > 0)
    for (int i = 1; i <= kConsumers; ++i)
      if (st.side[i].segment < s.segment) return kBlocked;
  const bool keys = lm::AttnQueryTurn::has_keys(0, blocks[s.segment]);
  const int b = buffer_of(s);
  if (who == 0) {
    if (!keys) {
      leave(s, false);
    } else if (s.step == 0) {
      if (!st.empty[b].passes(empty_parity(s))) return kBlocked;
      s.step = 1;
    } else {
      st.held[b] = s.segment;
      st.full[b].arrive();
      leave(s, true);
    }
    return kMoved;
  }
  if (!keys) {
    if (by_segment) {
      st.empty[b].arrive();
      if (who == 1) st.full[b].arrive();
    }
    leave(s, false);
  } else if (s.step == 0) {
    if (!st.full[b].passes(full_parity(s))) return kBlocked;
    s.step = 1;
  } else {
    if (st.held[b] != s.segment) return kWrong;
    st.empty[b].arrive();
    leave(s, true);
  }
  return kMoved;
}

bool holds(const std::vector<int>& blocks) {
  std::set<std::vector<int>> seen;
  std::vector<State> open(1);
  while (!open.empty()) {
    const State at = open.back();
    open.pop_back();
    if (!seen.insert(at.key()).second) continue;
    bool moved = false, done = true;
    for (int who = 0; who <= kConsumers; ++who) {
      done = done && at.side[who].segment == static_cast<int>(blocks.size());
      State next = at;
      const Outcome o = advance(next, who, blocks);
      if (o == kWrong) return false;
      if (o == kMoved) {
        moved = true;
        open.push_back(next);
      }
    }
    if (!moved && !done) return false;  // they wait for one another
  }
  return true;
}

}  // namespace

int main(int argc, char** argv) {
  by_segment = argc > 1 && std::strcmp(argv[1], "segments") == 0;
  int patterns = 0, broken = 0;
  for (int n = 1; n <= 10; ++n)
    for (int bits = 0; bits < 1 << n; ++bits) {
      std::vector<int> blocks;
      for (int i = 0; i < n; ++i) blocks.push_back(bits >> i & 1);
      ++patterns;
      if (holds(blocks)) continue;
      ++broken;
      if (argc > 2) {  // name them
        for (int v : blocks) std::putchar('0' + v);
        std::putchar('\n');
      }
    }
  std::printf("%d %d\n", patterns, broken);
  return 0;
}
