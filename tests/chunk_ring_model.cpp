// Walks through every order in which the warps of the chunk attention can fill, use and give back the
// positions of its ring of K/V blocks, with the kernel's own rule for filling one
// (mac_b200_chunk_ring.h).  Barriers show one bit of their phase, as the hardware's do.  Prints one line a
// case and leaves with 1 when a position is filled while it is in use, read before it is filled, or
// when the warps come to stand.
//
// The model: kWarps loading warps a group (each fills its share of a position by itself); two issuing warps
// that walk the positions in order, hand a product on each of their own to the tensor cores and give the
// other stream's back at once; the tensor cores, which run a stream's products in order after any time
// and give each position back when its last product has run.  An issuing warp may run ahead as far as the
// barriers of filled positions let it: more than the softmax would.
#include <array>
#include <cstdio>
#include <cstring>
#include <string>
#include <unordered_set>
#include <vector>

#include "../mac_attention_b200/csrc/mac_b200_chunk_ring.h"

namespace {

constexpr int kWarps = 2, kMaxGroups = 3, kMaxStages = 5, kMaxPositions = 32;

struct Barrier {
  unsigned char phases, arrived;
  bool passes(unsigned parity) const { return (phases & 1u) != parity; }
  void arrive(int count) {
    if (++arrived == count) arrived = 0, ++phases;
  }
};
struct State {
  Barrier full[kMaxStages], empty[kMaxStages];
  signed char held[kMaxStages][kWarps];     // the position whose rows lie there, by share
  signed char fills[kMaxGroups][kWarps];    // a loading warp's next position
  signed char looks[2], runs[2];            // a stream's next position to look at / whose product is to run
  signed char given[kMaxPositions];         // streams that gave the position back
};
struct Case {
  const char* name;
  int stages, groups, positions;
  bool dual, rule;                          // rule: wait_to_fill(); else the wait for the given-back phase alone
  bool sound;                               // what the walk has to find
};
// whether stream s has a product on position p (see ring_v() in the kernel)
bool uses(const Case& c, int s, int p) {
  if (c.dual) return true;
  const int n = c.positions;
  const bool is_v = p == n - 1 || (p > 0 && p % 2 == 0);
  const int block = is_v ? (p == n - 1 ? n / 2 : p / 2) - 1 : (p + 1) / 2;
  return block % 2 == s;
}
// applies one move; false: not possible now.  A broken rule is told in `fault`.
bool move(const Case& c, State& x, int kind, int i, std::string& fault) {
  if (kind == 0) {                          // loading warp i fills its share of its next position
    const int g = i / kWarps, w = i % kWarps, p = x.fills[g][w];
    if (p >= c.positions) return false;
    const int st = p % c.stages;
    const unsigned phase = (p / c.stages & 1) ^ 1u;
    auto wait = [&](bool filled) { return (filled ? x.full[st] : x.empty[st]).passes(phase); };
    if (!(c.rule ? mac_b200::wait_to_fill(wait) : wait(false))) return false;
    if (p >= c.stages && x.given[p - c.stages] != 2)
      fault = "position " + std::to_string(p) + " filled over " + std::to_string(p - c.stages) + ", still in use";
    x.held[st][w] = static_cast<signed char>(p);
    x.full[st].arrive(kWarps);
    x.fills[g][w] = static_cast<signed char>(p + c.groups);
    return true;
  }
  auto give_back = [&](int p) {
    x.empty[p % c.stages].arrive(2);
    ++x.given[p];
  };
  auto whole = [&](int p) {
    for (int w = 0; w < kWarps; ++w)
      if (x.held[p % c.stages][w] != p) return false;
    return true;
  };
  if (kind == 1) {                          // issuing warp i looks at its next position
    const int p = x.looks[i];
    if (p >= c.positions || !x.full[p % c.stages].passes(p / c.stages & 1)) return false;
    if (!whole(p)) fault = "position " + std::to_string(p) + " read before it was filled";
    ++x.looks[i];
    if (!uses(c, i, p)) give_back(p);
    return true;
  }
  int p = x.runs[i];                        // the tensor cores run stream i's next product
  while (p < x.looks[i] && !uses(c, i, p)) ++p;
  if (p >= x.looks[i]) return false;
  if (!whole(p)) fault = "position " + std::to_string(p) + " overwritten before its product had run";
  give_back(p);
  x.runs[i] = static_cast<signed char>(p + 1);
  return true;
}

std::string walk(const Case& c, size_t& states) {
  State first;
  std::memset(&first, 0, sizeof(first));
  std::memset(first.held, -1, sizeof(first.held));
  for (int g = 0; g < kMaxGroups; ++g)
    for (int w = 0; w < kWarps; ++w) first.fills[g][w] = static_cast<signed char>(g);
  std::unordered_set<std::string> seen;
  std::vector<State> open{first};
  auto key = [](const State& x) { return std::string(reinterpret_cast<const char*>(&x), sizeof(x)); };
  seen.insert(key(first));
  while (!open.empty()) {
    const State at = open.back();
    open.pop_back();
    bool moved = false;
    for (int kind = 0; kind < 3; ++kind)
      for (int i = 0; i < (kind == 0 ? c.groups * kWarps : 2); ++i) {
        State next = at;
        std::string fault;
        if (!move(c, next, kind, i, fault)) continue;
        if (!fault.empty()) return fault;
        moved = true;
        if (seen.insert(key(next)).second) open.push_back(next);
      }
    bool done = true;
    for (int p = 0; p < c.positions; ++p) done = done && at.given[p] == 2;
    if (!moved && !done) return "the warps stand";
  }
  states = seen.size();
  return "";
}

}  // namespace

int main() {
  using Bf16 = mac_b200::RingShape<false>;
  using E4m3 = mac_b200::RingShape<true>;
  const int spare = E4m3::kStages + E4m3::kSpare;
  const Case cases[] = {
      // the bf16 pool's warps fill every position, one after the other, and wait for nothing else
      {"bf16, streams alternate", Bf16::kStages + Bf16::kSpare, Bf16::kGroups, 30, false, false, true},
      {"bf16, two tiles", Bf16::kStages, Bf16::kGroups, 30, true, false, true},
      {"e4m3, streams alternate, spare position", spare, E4m3::kGroups, 30, false, true, true},
      {"e4m3, streams alternate", E4m3::kStages, E4m3::kGroups, 30, false, true, true},
      {"e4m3, two tiles", E4m3::kStages, E4m3::kGroups, 30, true, true, true},
      // the model sees what a warp that waits for the given-back phase alone does to a ring of four
      {"three groups over four positions, without the first wait", 4, 3, 30, false, false, false},
  };
  int bad = 0;
  for (const Case& c : cases) {
    size_t states = 0;
    const std::string fault = walk(c, states);
    std::printf("%s: %s (%zu states)\n", c.name, fault.empty() ? "sound" : fault.c_str(), states);
    bad += fault.empty() != c.sound;
  }
  return bad != 0;
}
