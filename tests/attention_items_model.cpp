// How the CTAs of a launch come by their work items (next_item of attention_issue.cuh), against a model of the
// grid: a block that has not started either starts as a CTA of its own or is the answer to a request, in any
// order. Blocks hold rows or do not; every one that does has to become an item, once.
#include <cstdint>
#include <random>
#include <vector>

#include "attention_issue.cuh"

namespace {

enum Wrong { NONE, LOST, TWICE, ASKED_AGAIN, WRONG_END, GIVE_UP };

struct Grid {
  std::mt19937_64 rng;
  std::vector<int> waiting;   // blocks that have not started
  std::vector<char> rows;     // whether a block holds any
  std::vector<int> items;     // how often a block has become an item
  bool ordered;               // answers in ascending order
  int take() {
    const size_t i = ordered ? 0 : rng() % waiting.size();
    const int block = waiting[i];
    waiting.erase(waiting.begin() + i);
    return block;
  }
};
struct Cta {
  bool asking = false, refused = false;
  int answer = -1;  // -1: a refusal
};

}  // namespace

// `give_up`: a CTA's request of that number is never answered; it gives up, which loses only what it asked for.
extern "C" int items_model(int blocks, const char* rows, int resident, int ordered, int give_up, uint64_t seed) {
  Grid g;
  g.rng.seed(seed);
  g.rows.assign(rows, rows + blocks);
  g.items.assign(blocks, 0);
  g.ordered = ordered != 0;
  for (int b = 0; b < blocks; ++b) g.waiting.push_back(b);
  std::vector<Cta> ctas;
  Wrong wrong = NONE;
  int asked = 0, unanswered = -1;
  while (true) {
    // as many CTAs as there is room for; one without rows leaves at once
    while (static_cast<int>(ctas.size()) < resident && !g.waiting.empty()) {
      const int block = g.take();
      if (!g.rows[block]) continue;
      ++g.items[block];
      ctas.emplace_back();
    }
    if (ctas.empty()) break;
    const size_t at = g.rng() % ctas.size();  // is done with its item
    Cta& c = ctas[at];
    bool ok = true, more = false;
    trx::next_item(
        [&] {
          if (c.refused) wrong = ASKED_AGAIN;
          c.asking = true;
          c.answer = g.waiting.empty() ? -1 : g.take();
        },
        [&] {
          if (asked++ != give_up) return true;
          unanswered = c.answer;
          return false;
        },
        [&] {
          c.asking = false;
          if (c.answer < 0) {
            c.refused = true;
            return trx::Block::NONE_LEFT;
          }
          if (!g.rows[c.answer]) return trx::Block::NO_ROWS;
          ++g.items[c.answer];
          return trx::Block::ITEM;
        },
        ok, more);
    if (ok != !c.asking || (!ok && more)) wrong = GIVE_UP;
    if (ok && more == c.refused) wrong = WRONG_END;
    if (!ok || !more) ctas.erase(ctas.begin() + at);
    if (wrong != NONE) return wrong;
  }
  for (int b = 0; b < blocks; ++b) {
    if (g.items[b] > 1) return TWICE;
    if (g.items[b] == 0 && g.rows[b] && b != unanswered) return LOST;
  }
  return NONE;
}
