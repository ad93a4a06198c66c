// Both issuing warps of the attention kernel's ragged forms against a model of what is around them: the K / V
// ring that they share, of which a stage is free when both have released it, their Q tiles, softmax warps
// and epilogue. The warps are coroutines; whatever can happen next is picked at random. Barriers are what
// the hardware has, a phase count of which a wait sees one bit.
#include <ucontext.h>

#include <cstdint>
#include <memory>
#include <random>
#include <vector>

#include "attention_issue.cuh"

namespace {

enum Wrong { NONE, LAPPED, OVERWRITTEN, RELEASED_TWICE, ORDER, DEADLOCK, UNFINISHED };
constexpr int STAGES = trx::AP_STAGES;

struct Item {
  int n, lo[2], hi[2], mask;
};
struct Fill {
  int item, visit;
  bool k;
  bool issued = false, landed = false;
  bool released[2] = {false, false};
};
struct Tile {
  int read = 0;
  int q_issued = 0, q_landed = 0, q_done = 0, q_waited = 0;
  int o_done = 0, o_free = 0, o_waited = 0;
  bool q_pending = false;
  int scores_made = 0, probabilities = 0, products_made = 0;
  std::vector<int> scores, products;  // 1000 * item + visit
  ucontext_t context;
  std::vector<char> stack;
  bool over = false, blocked = false;
};

struct World {
  std::mt19937_64 rng;
  std::vector<Item> items;
  std::vector<Fill> fills;
  std::vector<int> first;
  Tile tile[2];
  Wrong wrong = NONE;
  int item = 0, next_fill = 0, published = 0;
  int landed[STAGES] = {};
  ucontext_t main;
  int running = 0;

  bool fail(Wrong w) {
    if (wrong == NONE) wrong = w;
    return false;
  }
  void yield(int t, bool blocked) {
    tile[t].blocked = blocked;
    swapcontext(&tile[t].context, &main);
  }
  bool mine(const Item& i, int t, int v) const {
    return v >= i.lo[t] && v < i.hi[t] && ((v - i.lo[t]) & i.mask) == 0;
  }
  // what is around the warps: each returns whether it happened
  bool publish() {
    if (item >= static_cast<int>(items.size()) || published > item) return false;
    if (item >= 2 && (tile[0].read < item - 1 || tile[1].read < item - 1)) return false;
    published = item + 1;
    for (int t = 0; t < 2; ++t) tile[t].q_pending = items[item].hi[t] > items[item].lo[t];
    return true;
  }
  bool q_pending() const { return tile[0].q_pending || tile[1].q_pending; }
  bool issue_q(int t) {
    if (published <= item || !tile[t].q_pending || (t == 1 && tile[0].q_pending)) return false;
    if (item > 0 && items[item].n > 0 && next_fill == first[item]) return false;  // its first K ahead
    if (tile[t].q_done < tile[t].q_issued) return false;
    ++tile[t].q_issued;
    tile[t].q_pending = false;
    return true;
  }
  bool issue_fill() {
    if (published <= item || next_fill == first[item + 1]) return false;
    if (q_pending() && (item == 0 || next_fill > first[item])) return false;
    if (next_fill >= STAGES) {
      const Fill& before = fills[next_fill - STAGES];
      if (!before.released[0] || !before.released[1]) return false;
    }
    fills[next_fill++].issued = true;
    return true;
  }
  bool next_item() {
    if (published <= item || q_pending() || next_fill < first[item + 1]) return false;
    ++item;
    publish();
    return true;
  }
  bool land() {
    std::vector<int> flying;
    for (int f = 0; f < next_fill; ++f)
      if (!fills[f].landed) flying.push_back(f);
    if (flying.empty()) return false;
    const int f = flying[rng() % flying.size()];
    fills[f].landed = true;
    ++landed[f % STAGES];
    return true;
  }
  bool land_q(int t) {
    if (tile[t].q_landed == tile[t].q_issued) return false;
    ++tile[t].q_landed;
    return true;
  }
  bool softmax(int t) {
    if (tile[t].probabilities == tile[t].scores_made) return false;
    ++tile[t].probabilities;
    return true;
  }
  bool epilogue(int t) {
    if (tile[t].o_free == tile[t].o_done) return false;
    ++tile[t].o_free;
    return true;
  }
  bool happen(int what) {
    switch (what) {
      case 0: return publish();
      case 1: return issue_q(0);
      case 2: return issue_q(1);
      case 3: return issue_fill();
      case 4: return next_item();
      case 5: return land();
      case 6: return land_q(0);
      case 7: return land_q(1);
      case 8: return softmax(0);
      case 9: return softmax(1);
      case 10: return epilogue(0);
      case 11: return epilogue(1);
      default: {
        Tile& t = tile[what - 12];
        if (t.over) return false;
        running = what - 12;
        swapcontext(&main, &t.context);
        return !t.blocked;
      }
    }
  }
  void run() {
    while (wrong == NONE && !(tile[0].over && tile[1].over)) {
      bool any = false;
      for (int i = 0; i < 10 && !any; ++i) any = happen(static_cast<int>(rng() % 14));
      for (int what = 0; what < 14 && !any; ++what) any = happen(what);
      if (!any && !(tile[0].over && tile[1].over)) fail(DEADLOCK);
    }
  }
  // a wait for a phase of which one bit is compared; `phase` is the one that is meant
  template <class Count>
  bool wait(int t, Count count, int phase) {
    yield(t, false);
    while ((count() & 1) == (phase & 1)) {
      if (wrong != NONE) return false;
      yield(t, true);
    }
    return count() == phase + 1 ? wrong == NONE : fail(LAPPED);
  }
  template <class Count>
  bool there(int t, Count count, int phase) {
    yield(t, false);
    if ((count() & 1) == (phase & 1)) return false;
    if (count() != phase + 1) fail(LAPPED);
    return true;
  }
  void use(int f, bool k) {
    if (!fills[f].landed || fills[f].k != k) fail(ORDER);
    if (f + STAGES < static_cast<int>(fills.size()) && fills[f + STAGES].issued) fail(OVERWRITTEN);
  }
  void warp(int t) {
    Tile& me = tile[t];
    const int count = static_cast<int>(items.size());
    trx::PlainSteps steps{
        [&](trx::AltCursor& c, int i, bool& ok) {
          if (i >= count) return false;
          yield(t, false);  // what came before this is progress
          while (published <= i) {
            if (wrong != NONE) return ok = false;
            yield(t, true);
          }
          c.lo = items[i].lo[t];
          c.hi = items[i].hi[t];
          c.n = items[i].n;
          c.item = i;
          c.v = 0;
          c.mask = items[i].mask;
          me.read = i + 1;
          return true;
        },
        [&](int i) { yield(t, false); return i >= count || published > i; },
        [&](int f) { return wait(t, [&] { return landed[f % STAGES]; }, f / STAGES); },
        [&](int f) { return there(t, [&] { return landed[f % STAGES]; }, f / STAGES); },
        [&](int f) {
          if (fills[f].released[t]) fail(RELEASED_TWICE);
          if (!fills[f].landed) fail(LAPPED);
          fills[f].released[t] = true;
        },
        [&](unsigned parity) {
          if (parity != (me.q_waited & 1u)) return fail(ORDER);
          return wait(t, [&] { return me.q_landed; }, me.q_waited++);
        },
        [&](unsigned) { return there(t, [&] { return me.q_landed; }, me.q_waited); },
        [&](int f) {
          use(f, true);
          if (me.scores.size() != me.products.size()) fail(ORDER);  // its P is not used up yet
          me.scores.push_back(1000 * fills[f].item + fills[f].visit);
          ++me.scores_made;
        },
        [&] { ++me.q_done; },
        [&](unsigned parity) {
          if (parity != (me.o_waited & 1u)) return fail(ORDER);
          return wait(t, [&] { return me.o_free; }, me.o_waited++);
        },
        [&](int f, unsigned acc) {
          if (!wait(t, [&] { return me.probabilities; }, me.products_made++)) return false;
          use(f, false);
          const int v = fills[f].visit, i = fills[f].item;
          if ((acc == 0) != (v == items[i].lo[t]) || me.scores.size() != me.products.size() + 1 ||
              (acc == 0 && me.o_free != me.o_done))
            fail(ORDER);
          me.products.push_back(1000 * i + v);
          return wrong == NONE;
        },
        [&] { ++me.o_done; }};
    trx::plain_issue<trx::AltCursor>(steps);
    me.over = true;
    yield(t, false);
  }
};

World* g_world;
void start() {
  World* w = g_world;
  w->warp(w->running);
}

}  // namespace

extern "C" int issue_pair_model(int count, const int* n, const int* lo0, const int* hi0, const int* lo1,
                                const int* hi1, const int* mask, uint64_t seed) {
  auto world = std::make_unique<World>();
  World& w = *world;
  g_world = world.get();
  w.rng.seed(seed);
  std::vector<int> visits[2];
  for (int i = 0; i < count; ++i) {
    w.items.push_back({n[i], {lo0[i], lo1[i]}, {hi0[i], hi1[i]}, mask[i]});
    w.first.push_back(static_cast<int>(w.fills.size()));
    // K(0), K(1), V(0), K(2), V(1), .. V(n - 1)
    for (int v = 0; v < n[i]; ++v) {
      w.fills.push_back({i, v, true});
      if (v > 0) w.fills.push_back({i, v - 1, false});
    }
    if (n[i] > 0) w.fills.push_back({i, n[i] - 1, false});
    for (int t = 0; t < 2; ++t)
      for (int v = 0; v < n[i]; ++v)
        if (w.mine(w.items[i], t, v)) visits[t].push_back(1000 * i + v);
  }
  w.first.push_back(static_cast<int>(w.fills.size()));
  w.publish();
  for (int t = 0; t < 2; ++t) {
    Tile& me = w.tile[t];
    me.stack.resize(64 << 10);
    getcontext(&me.context);
    me.context.uc_stack.ss_sp = me.stack.data();
    me.context.uc_stack.ss_size = me.stack.size();
    me.context.uc_link = &w.main;
    makecontext(&me.context, start, 0);
  }
  w.run();
  if (w.wrong == NONE) {
    for (int t = 0; t < 2; ++t)
      if (w.tile[t].scores != visits[t] || w.tile[t].products != visits[t]) w.fail(UNFINISHED);
    for (const Fill& f : w.fills)
      if (!f.released[0] || !f.released[1]) w.fail(UNFINISHED);
  }
  return w.wrong;
}
