// Host model of extend_kernel's barriers, on the step order of csrc/extend_steps.h: between the MMA lane,
// the tensor cores and the two softmax warpgroups, and between the producer, its copies and the two
// converters of codes. Every interleaving of the roles over sequences of segments. A wait passes by parity, as mbarrier.try_wait.parity does; a role that waits
// while its phase is two ahead (the wait would pass early) or two behind (it would block for good) is a
// violation, and so is a state from which no role can go on.
//
//   extend_protocol softmax RULE    RULE joined: as the kernel; dual: only one-tile segments joined
//   extend_protocol scales RULE     RULE kept: as the kernel; fewer: the scales of one key tile less are held
//   extend_protocol codes RULE      RULE release: as the kernel; full: converters wait for code_full alone
//
// Prints the number of sequences and of states, or the first violation (exit 1).
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <string>
#include <unordered_set>
#include <vector>

#include "extend_steps.h"

using flb::Steps;

namespace {

enum class Kind { kWait, kArrive, kNeeds };
struct Op {
  Kind kind;
  int bar, phase;   // wait for this phase; one more phase completes; that many have completed, or it is a fault
};
using Program = std::vector<Op>;
struct Model {
  std::vector<Program> roles;
  std::vector<std::string> bars;

  int bar(const std::string& name) {
    for (size_t i = 0; i < bars.size(); ++i)
      if (bars[i] == name) return static_cast<int>(i);
    bars.push_back(name);
    return static_cast<int>(bars.size()) - 1;
  }
  void wait(int role, const std::string& name, int phase) {
    roles[role].push_back({Kind::kWait, bar(name), phase});
  }
  void arrive(int role, const std::string& name) {
    roles[role].push_back({Kind::kArrive, bar(name), 0});
  }
  void needs(int role, const std::string& name, int phases) {
    roles[role].push_back({Kind::kNeeds, bar(name), phases});
  }
};

struct Result {
  long states = 0;
  std::string error;
};

// All interleavings. Programs are straight lines, so the roles' places are the whole state.
Result explore(const Model& m) {
  const size_t roles = m.roles.size(), bars = m.bars.size();
  // Phases each role has completed by its place.
  std::vector<std::vector<std::vector<int>>> done(roles);
  for (size_t r = 0; r < roles; ++r) {
    done[r].assign(m.roles[r].size() + 1, std::vector<int>(bars, 0));
    for (size_t i = 0; i < m.roles[r].size(); ++i) {
      done[r][i + 1] = done[r][i];
      if (m.roles[r][i].kind == Kind::kArrive) ++done[r][i + 1][m.roles[r][i].bar];
    }
  }
  Result result;
  std::unordered_set<uint64_t> seen{0};
  std::vector<uint64_t> todo{0};
  const size_t bits = 64 / roles;
  for (const Program& program : m.roles) {
    if (program.size() >> bits != 0) {
      result.error = "a program is too long for the state";
      return result;
    }
  }
  auto place = [&](uint64_t s, size_t r) {
    return static_cast<size_t>(s >> (bits * r)) & ((size_t{1} << bits) - 1);
  };
  while (!todo.empty()) {
    const uint64_t s = todo.back();
    todo.pop_back();
    ++result.states;
    bool moved = false, ended = true;
    for (size_t r = 0; r < roles; ++r) {
      const size_t at = place(s, r);
      if (at == m.roles[r].size()) continue;
      ended = false;
      const Op& op = m.roles[r][at];
      if (op.kind != Kind::kArrive) {
        int completed = 0;
        for (size_t q = 0; q < roles; ++q) completed += done[q][place(s, q)][op.bar];
        if (op.kind == Kind::kNeeds) {
          if (completed < op.phase) {
            result.error = "role " + std::to_string(r) + " goes on before " + m.bars[op.bar];
            return result;
          }
        } else if (completed < op.phase || completed > op.phase + 1) {
          char text[160];
          std::snprintf(text, sizeof(text), "role %zu waits for phase %d of %s, %d completed", r,
                        op.phase, m.bars[op.bar].c_str(), completed);
          // Reached by the role while the phase before the named one is still open, the wait passes.
          result.error = text;
          return result;
        }
        if (op.kind == Kind::kWait && completed == op.phase) continue;
      }
      moved = true;
      const uint64_t next = s + (uint64_t{1} << (bits * r));
      if (seen.insert(next).second) todo.push_back(next);
    }
    if (!moved && !ended) {
      result.error = "no role can go on";
      return result;
    }
  }
  return result;
}

std::string numbered(const char* name, int i) { return name + std::to_string(i); }

// Roles: 0 the MMA lane, 1 the tensor cores (they work in order, a commit completes what came
// before it), 2 and 3 the softmax warpgroups. K, V and Q are always there. rescale: every step moves
// its reference point, which is when a chain waits for P V of its previous step. With scale_slots > 0 also
// 4, the converter of K, which writes the scales of a tile into one of so many places before the tile.
Model softmax_model(const std::vector<Steps>& segments, int s_bufs, int v_slots, bool rescale,
                    bool join_count0, int k_slots = 0, int scale_slots = 0) {
  Model m;
  m.roles.resize(scale_slots > 0 ? 5 : 4);
  std::vector<int> readers[2];   // steps that each chain has done once it has read the tile's scales
  int chain_steps[2] = {0, 0};
  int n_base = 0, kv_base = 0, p_waits[3] = {0, 0, 0}, o_waits[2] = {0, 0}, joins = 0, issued = 0;
  for (const Steps& s : segments) {
    const int steps = s.count0 + s.count1;
    const int tiles = s.dual ? steps : s.count1;
    const bool joined = join_count0 ? s.joined() : s.dual;
    // The tensor cores may not run ahead of the lane: op i of theirs waits for its issue.
    auto tensor = [&](const std::string& bar) {   // a commit
      m.arrive(0, numbered("issue", issued));
      m.wait(1, numbered("issue", issued), 0);
      ++issued;
      m.arrive(1, bar);
    };
    auto entry_of = [&](int i) {
      return kv_base + (i < s.paired() ? (s.dual ? i : i >> 1) : i - s.count0);
    };
    auto qk = [&](int i) {
      const int entry = entry_of(i);
      if (scale_slots > 0) m.wait(0, numbered("k_full", entry % k_slots), entry / k_slots);
      tensor(numbered("s_full", (n_base + i) % s_bufs));
      if (scale_slots > 0 && (s.dual || s.chain(i) == 1)) tensor(numbered("k_empty", entry % k_slots));
    };
    for (int c = 0; c < 2; ++c) {
      readers[c].resize(kv_base + tiles, chain_steps[c]);
      for (int j = 0; j < s.count(c); ++j) readers[c][kv_base + s.place(c, j)] = ++chain_steps[c];
    }
    for (int at = kv_base; scale_slots > 0 && at < kv_base + tiles; ++at) {
      if (at >= k_slots) m.wait(4, numbered("k_empty", at % k_slots), at / k_slots - 1);
      for (int c = 0; c < 2 && at >= scale_slots; ++c)   // who read the place's last scales has done so
        m.needs(4, numbered("step", c), readers[c][at - scale_slots]);
      m.arrive(4, numbered("scale_full", at % scale_slots));
      m.arrive(4, numbered("k_full", at % k_slots));
    }
    for (int i = 0; i < s_bufs && i < steps; ++i) qk(i);
    for (int i = 0; i < steps; ++i) {
      const int c = s.chain(i), buf = (n_base + i) % s_bufs;
      const int entry = entry_of(i);
      m.wait(0, numbered("p", buf), p_waits[buf]++);
      if (s.dual || c == 1) tensor(numbered("v_empty", entry % v_slots));
      if (i == s.other_last() || i == steps - 1) tensor(numbered("o_full", c));
      if (i + s_bufs < steps) qk(i + s_bufs);
    }
    for (int c = 0; c < 2; ++c) {
      const int role = 2 + c;
      for (int j = 0; j < s.count(c); ++j) {
        const int n = n_base + s.order(c, j);
        m.wait(role, numbered("s_full", n % s_bufs), n / s_bufs);
        if (rescale && j > 0 && s.order(c, j) - s.order(c, j - 1) < s_bufs) {
          const int v = kv_base + s.place(c, j - 1);
          m.wait(role, numbered("v_empty", v % v_slots), v / v_slots);
        }
        if (scale_slots > 0) {
          const int at = kv_base + s.place(c, j);
          m.wait(role, numbered("scale_full", at % scale_slots), at / scale_slots);
          m.arrive(role, numbered("step", c));
        }
        m.arrive(role, numbered("p", n % s_bufs));
      }
      if (s.count(c) > 0) m.wait(role, numbered("o_full", c), o_waits[c]++);
      if (joined) {
        if (c == 1) m.arrive(role, "x_ready");
        m.wait(role, c == 1 ? "x_done" : "x_ready", joins);
        if (c == 0) m.arrive(role, "x_done");
      }
    }
    joins += joined;
    n_base += steps;
    kv_base += tiles;
  }
  return m;
}

long sequences = 0, states = 0;

bool check(const Model& m, const std::string& what) {
  const Result r = explore(m);
  ++sequences;
  states += r.states;
  if (r.error.empty()) return true;
  std::printf("violation: %s: %s\n", what.c_str(), r.error.c_str());
  return false;
}

bool check_softmax(const std::vector<Steps>& segments, bool join_count0) {
  // head_dim 128 and 64, each with the V places of int8 and of 16-bit caches.
  const int shapes[4][2] = {{2, 1}, {2, 2}, {3, 2}, {3, 4}};
  for (const auto& shape : shapes) {
    for (int rescale = 0; rescale < 2; ++rescale) {
      std::string what = "S buffers " + std::to_string(shape[0]) + ", V places " +
                         std::to_string(shape[1]) + ", segments";
      for (const Steps& s : segments)
        what += std::string(s.dual ? " one-tile(" : " two-tile(") + std::to_string(s.count0) + ", " +
                std::to_string(s.count1) + ")";
      if (!check(softmax_model(segments, shape[0], shape[1], rescale, join_count0), what)) return false;
    }
  }
  return true;
}

bool softmax(bool join_count0) {
  // What Walk makes of n key tiles: one-tile segments share them, in two-tile ones the first tile
  // sees as many as the second or one less.
  std::vector<Steps> kinds;
  for (int n = 1; n <= 4; ++n) kinds.push_back({true, (n + 1) / 2, n / 2});
  for (int n = 0; n <= 3; ++n) kinds.push_back({false, n, n});
  for (int n = 0; n <= 2; ++n) kinds.push_back({false, n, n + 1});
  for (const Steps& a : kinds)
    for (const Steps& b : kinds)
      for (const Steps& c : kinds)
        if (!check_softmax({a, b, c}, join_count0)) return false;
  // Longer runs, in a fixed pseudo-random order; segments without a step for chain 0 among them.
  uint32_t x = 12345;
  for (int i = 0; i < 150; ++i) {
    std::vector<Steps> segments;
    for (int k = 0; k < 6; ++k) {
      x = x * 1664525u + 1013904223u;
      const uint32_t pick = x >> 16;
      segments.push_back(pick % 2 ? Steps{false, 0, 1} : kinds[(pick / 2) % kinds.size()]);
    }
    if (!check_softmax(segments, join_count0)) return false;
  }
  return true;
}

bool scales(int held_less) {
  std::vector<Steps> kinds;
  for (int n : {1, 2, 5}) kinds.push_back({true, (n + 1) / 2, n / 2});
  for (int n : {0, 1, 3}) kinds.push_back({false, n, n + 1});
  kinds.push_back({false, 4, 4});
  const int shapes[2][3] = {{2, 1, 2}, {3, 2, 4}};   // S buffers, V and K places at head_dim 128 and 64
  for (const auto& shape : shapes) {
    for (const Steps& a : kinds) {
      for (const Steps& b : kinds) {
        const Model m = softmax_model({a, b, a}, shape[0], shape[1], false, true, shape[2],
                                      shape[2] + shape[0] - held_less);
        if (!check(m, std::to_string(shape[0]) + " S buffers")) return false;
      }
    }
  }
  return true;
}

// Roles: 0 the producer, 1 and 2 the converters of K and V, then one for each place of the ring, whose
// copies land at any time after their issue, in any order among places.
Model codes_model(const std::vector<int>& tiles, int slots, bool wait_release) {
  Model m;
  m.roles.resize(3 + slots);
  int base = 0;
  for (int n : tiles) {
    for (int code = 2 * base; code < 2 * (base + n); ++code) {
      const int slot = code % slots, phase = code / slots;
      if (phase > 0) m.wait(0, numbered("code_empty", slot), phase - 1);
      m.arrive(0, numbered("copy", slot));
      m.wait(3 + slot, numbered("copy", slot), phase);
      m.arrive(3 + slot, numbered("code_full", slot));
    }
    for (int is_v = 0; is_v < 2; ++is_v) {
      for (int i = 0; i < n; ++i) {
        const int code = 2 * base + flb::code_place(is_v, i, n);
        const int slot = code % slots, phase = code / slots;
        if (wait_release && phase > 0) m.wait(1 + is_v, numbered("code_empty", slot), phase - 1);
        m.wait(1 + is_v, numbered("code_full", slot), phase);
        m.arrive(1 + is_v, numbered("code_empty", slot));
      }
    }
    base += n;
  }
  return m;
}

bool codes(bool wait_release) {
  for (int slots : {3, 6}) {   // head_dim 128 and 64
    for (int a = 1; a <= 6; ++a) {
      for (int b = 0; b <= 4; ++b) {
        for (int c = 0; c <= 3; ++c) {
          const std::string what = std::to_string(slots) + " places, segments of " + std::to_string(a) +
                                   ", " + std::to_string(b) + ", " + std::to_string(c) + " tiles";
          if (!check(codes_model({a, b, c}, slots, wait_release), what)) return false;
        }
      }
    }
  }
  return true;
}

}  // namespace

int main(int argc, char** argv) {
  const std::string part = argc > 1 ? argv[1] : "", rule = argc > 2 ? argv[2] : "";
  bool ok;
  if (part == "softmax" && (rule == "joined" || rule == "dual")) {
    ok = softmax(rule == "joined");
  } else if (part == "scales" && (rule == "kept" || rule == "fewer")) {
    ok = scales(rule == "fewer");
  } else if (part == "codes" && (rule == "release" || rule == "full")) {
    ok = codes(rule == "release");
  } else {
    std::printf("usage: extend_protocol softmax joined|dual, scales kept|fewer, or codes release|full\n");
    return 2;
  }
  if (ok) std::printf("%ld sequences, %ld states\n", sequences, states);
  return ok ? 0 : 1;
}
