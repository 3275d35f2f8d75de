// Host replay of the paged cache's index arithmetic (htree_cache_index.h, the
// functions the kernels call) over ordinary and damaged device data: lengths
// that are negative, huge or contradict each other, table entries and parents
// out of range.  Checks that
//   * the units of a call fit its launch and its workspace (the launch only
//     where the rows' starts ascend: others leave rows out, and only those);
//   * every row, token, table entry and page a unit touches is inside its
//     buffer, and every tile of every request is taken by exactly one chunk;
//   * walks up a drafted tree end.
// Test infrastructure: built and run by tests/test_cache_replay.py on the CPU.
#include <cstdio>
#include <random>
#include <vector>

#include "htree_cache_index.h"

using namespace htree;

static int fails = 0;
static long calls = 0, units_seen = 0;
#define CHECK(c)                                                       \
  do {                                                                 \
    if (!(c)) {                                                        \
      if (fails < 20) std::printf("FAIL %s (call %ld)\n", #c, calls);  \
      ++fails;                                                         \
    }                                                                  \
  } while (0)

int main() {
  std::mt19937 g(7);
  auto pick = [&](std::vector<int> v) { return v[g() % v.size()]; };
  auto upto = [&](int64_t n) { return (int)(g() % (uint64_t)(n + 1)); };
  for (calls = 0; calls < 4000; ++calls) {
    const bool damaged = calls % 2;
    const int es = pick({2, 4}), Dk = 16 * (1 + upto(15)), Dv = 16 * (1 + upto(15));
    const int Hkv = pick({1, 2, 3, 8}), G = pick({1, 2, 5, 8, 16, 64}), B = 1 + upto(pick({1, 4, 70}));
    const int shift = 4 + upto(4), width = upto(pick({1, 40, 400, 2000})), cap = width << shift;
    const int num_pages = 1 + upto(500), most = pick({1, 4, 30, 200});
    std::vector<int> starts{0}, lens;
    for (int b = 0; b < B; ++b) {
      const int n = upto(most);
      starts.push_back(starts.back() + n);
      lens.push_back(damaged && upto(3) == 0 ? (int)g() : n + upto(cap));
    }
    const int rows = damaged ? upto(starts.back() + 3) : starts.back() + upto(3);
    bool ascend = true;
    if (damaged && calls % 4 == 1)
      for (int& s : starts) if (upto(2) == 0) s = (int)g(), ascend = false;
    if (rows == 0) continue;
    const DraftPlan p = draft_plan(Dk, Dv, es, B, rows, G * Hkv, Hkv, width, 1 << shift);
    CHECK(p.D >= Dk && p.D >= Dv && p.R == 16 * p.MT * p.NW);
    CHECK(p.bytes == (p.target ? p.slots * p.R * (p.D + 2) * 4 + 16 : 0));
    const int KT = draft_tile(p.D, es, p.NW);
    CHECK(KT >= 16 && KT <= 64 && KT % 16 == 0);
    float tiles = 0;
    std::vector<DraftReq> rq;
    for (int b = 0; b < B; ++b) {
      rq.push_back(draft_req(starts[b], starts[b + 1], lens[b], rows));
      const DraftReq& r = rq[b];
      CHECK(r.s0 >= 0 && r.n >= 0 && r.s0 + r.n <= rows && r.len >= 0);
      tiles += (float)draft_tiles(r, cap, KT) * draft_row_groups(r, G, p.R);
    }
    int chunk = draft_chunk(tiles * Hkv, p.target);
    for (int i = upto(3); i > 0 && p.target > 0; --i) chunk = draft_wider(chunk);
    int64_t units = 0, slots = 0;
    for (const DraftReq& r : rq) {
      const int nt = draft_tiles(r, cap, KT), nch = draft_chunks(nt, chunk), part = draft_part(nt, nch);
      CHECK((int64_t)part * nch >= nt && part <= (chunk > 1 ? chunk : 1));
      const int64_t rts = draft_row_groups(r, G, p.R);
      units += draft_pieces(nch, (int)(rts * Hkv));
      if (nch > 1) slots += draft_pieces(nch, (int)(rts * Hkv));
      for (int64_t rt = 0; rt < rts; rt += rts > 40 ? 1 + upto(9) : 1) {
        int next = 0;
        const int even = draft_even(r, G, p.R, 16 * p.MT), r0 = (int)rt * even;
        CHECK(even <= p.R && even * rts >= (int64_t)r.n * G && r0 < r.n * G);
        const DraftSpan whole = draft_span(r, r0, even, G, cap, KT, 0, 1 << 30);
        CHECK(whole.kend >= 0 && whole.kend <= cap && whole.kend <= r.len);
        const int used = (whole.kend + (1 << shift) - 1) >> shift;
        CHECK(used <= width);
        for (int ch = 0; ch < nch; ++ch) {
          const DraftSpan s = draft_span(r, r0, even, G, cap, KT, ch, part);
          ++units_seen;
          CHECK(s.kend == whole.kend && s.t0 <= s.t1);
          CHECK(s.t0 == next);
          next = s.t1;
          for (int t = s.t0; t < s.t1; t += 1 + upto(3))
            for (int i = 0; i < KT; i += 16) {
              const int pi = (t * KT + i) >> shift, off = (t * KT + i) & ((1 << shift) - 1);
              CHECK(pi >= 0 && off + 15 < (1 << shift));
              if (pi >= used) continue;  // taken as no page
              CHECK(pi < width);
              const int pg = cache_page(upto(1) ? (int)g() : upto(num_pages), num_pages);
              CHECK(pg >= -1 && pg < num_pages);
            }
        }
        CHECK(next == (whole.kend + KT - 1) / KT);
        // the rows' tokens and a walk to the root
        for (int64_t x = r0; x < r0 + even && x < (int64_t)r.n * G; ++x) {
          int j = (int)(x / G), steps = 0;
          CHECK(j < r.n && (int64_t)r.s0 + j < rows);
          while (j >= 0) {
            const int up = draft_parent(upto(2) ? j - 1 - upto(3) : (int)g(), j);
            CHECK(up < j);
            j = up;
            CHECK(++steps <= r.n);
          }
        }
      }
    }
    CHECK(slots <= p.slots);
    if (ascend) CHECK(units <= p.units);
    CHECK((p.joins > 0) == (p.target > 0));
    // every unit has one block
    CHECK(p.units % (8 * p.near) == 0);
    if (p.units < 100000) {
      std::vector<char> had((size_t)p.units, 0);
      for (int64_t x = 0; x < p.units; ++x) {
        const int64_t u = draft_near(x, p.near);
        CHECK(u >= 0 && u < p.units && !had[(size_t)u]);
        if (u >= 0 && u < p.units) had[(size_t)u] = 1;
      }
    }
    // page tables: the new pages are those the launch has blocks for
    for (int b = 0; b < B; ++b) {
      const int64_t ctx = lens[b] < 0 ? 0 : lens[b], n = rq[b].n;
      const int64_t had = table_pages(ctx, shift), now = table_pages(ctx + n, shift);
      CHECK(had * (1 << shift) >= ctx && now >= had && now - had <= (n >> shift) + 1);
    }
  }
  std::printf("%ld calls, %ld units, %d failures\n", calls, units_seen, fails);
  return fails != 0;
}
