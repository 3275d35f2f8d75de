// Host replay of how the attention over a paged cache finds its work
// (htree_cache_index.h, the functions the kernels call): every block of a
// launch looks its unit up in the requests' shares, every block of the join its
// pieces.  Checks, over ordinary lengths, that
//   * each (request, group of rows, KV head, chunk) is taken by one block, and
//     its tokens are all of its group's, once;
//   * each unit of a split request has a workspace slot of its own, inside the
//     workspace, and the join reads, for each row, the slots of exactly that
//     row's chunks and stores each row of a split request once, no other;
// and over damaged ones that nothing outside the workspace or the rows is
// touched.  The lanes' sums are made one after the other here.
// Test infrastructure: built and run by tests/test_cache_units.py on the CPU.
#include <cstdio>
#include <map>
#include <random>
#include <tuple>
#include <vector>

#include "htree_cache_index.h"

using namespace htree;

static int fails = 0;
static long calls = 0, units_seen = 0, joined = 0;
#define CHECK(c)                                                      \
  do {                                                                \
    if (!(c)) {                                                       \
      if (fails < 20) std::printf("FAIL %s (call %ld)\n", #c, calls); \
      ++fails;                                                        \
    }                                                                 \
  } while (0)

struct Call {
  int B, rows, H, Hkv, G, width, shift, es, KT;
  DraftPlan p;
  std::vector<int> starts, lens;
  DraftReq req(int b) const { return draft_req(starts[b], starts[b + 1], lens[b], rows); }
  int cap() const { return width << shift; }
};

static int chunk_of(const Call& c) {
  float w = 0.f;
  if (c.p.target > 0)
    for (int b = 0; b < c.B; ++b)
      w += (float)draft_tiles(c.req(b), c.cap(), c.KT) * draft_row_groups(c.req(b), c.G, c.p.R);
  const int chunk = draft_chunk(w * c.Hkv, c.p.target);
  if (c.p.target == 0 || c.B > 64) return chunk;
  return draft_widen(chunk, c.p.target, [&](int x) {
    float units = 0.f;
    for (int b = 0; b < c.B; ++b)
      units += (float)draft_chunks(draft_tiles(c.req(b), c.cap(), c.KT), x) * draft_row_groups(c.req(b), c.G, c.p.R);
    return units * c.Hkv;
  });
}

// the shares' sums up to each request, as the lanes' prefix sums have them
template <typename F>
struct Lookup {
  const Call& c;
  std::vector<DraftShare> share;
  std::vector<int64_t> first, slot;
  Lookup(const Call& c, int chunk, F per) : c(c), first{0}, slot{0} {
    for (int b = 0; b < c.B; ++b) {
      share.push_back(draft_share(c.req(b), c.cap(), c.KT, c.G, c.p.R, c.Hkv, chunk, per));
      first.push_back(first.back() + share.back().pieces);
      slot.push_back(slot.back() + share.back().slots);
    }
  }
  bool find(int64_t u, DraftUnit* o) const {
    for (int b = 0; b < c.B; ++b)
      if (first[b + 1] > u) {
        const DraftShare& s = share[b];
        *o = draft_pick(b, s.nch, s.tiles, s.groups, slot[b], u - first[b], c.Hkv);
        return true;
      }
    return false;
  }
};
template <typename F>
Lookup<F> lookup(const Call& c, int chunk, F per) {
  return Lookup<F>(c, chunk, per);
}

static void check(const Call& c, bool ordinary) {
  const int chunk = chunk_of(c);
  std::map<std::tuple<int, int, int, int>, int64_t> taken;  // b, rt, h, ch -> slot
  std::map<int64_t, int> slots;
  const auto units = lookup(c, chunk, [](int nch) { return nch; });
  for (int64_t x = 0; x < c.p.units; ++x) {
    DraftUnit u;
    if (!units.find(draft_near(x, c.p.near), &u)) continue;
    const DraftPart p = draft_unit_part(u, c.Hkv);
    const DraftReq r = c.req(u.b);
    ++units_seen;
    CHECK(p.h >= 0 && p.h < c.Hkv && p.rt >= 0 && p.rt < u.groups && p.ch >= 0 && p.ch < u.nch);
    CHECK(u.groups == draft_row_groups(r, c.G, c.p.R));
    CHECK((p.slot >= 0) == (u.nch > 1));
    if (u.nch > 1) {
      CHECK(c.p.target > 0 && p.slot < c.p.slots);
      CHECK(slots[p.slot]++ == 0);
    }
    CHECK(taken.emplace(std::make_tuple(u.b, p.rt, p.h, p.ch), p.slot).second);
    const int even = draft_even(r, c.G, c.p.R, 16 * c.p.MT), row0 = p.rt * even;
    CHECK(row0 < r.n * c.G && even <= c.p.R);
    const DraftSpan s = draft_span(r, row0, even, c.G, c.cap(), c.KT, p.ch, u.chunk);
    CHECK(s.t0 >= 0 && s.t0 <= s.t1 && (int64_t)s.t1 * c.KT < (int64_t)c.cap() + c.KT);
    const DraftSpan whole = draft_span(r, row0, even, c.G, c.cap(), c.KT, 0, 1 << 30);
    // even parts: the last chunk ends with the group's tokens
    CHECK(s.t0 == (p.ch * (int64_t)u.chunk < whole.t1 ? p.ch * u.chunk : whole.t1));
    CHECK(p.ch + 1 < u.nch ? s.t1 == (s.t0 + u.chunk < whole.t1 ? s.t0 + u.chunk : whole.t1) : s.t1 == whole.t1);
  }
  if (ordinary) {
    size_t all = 0;
    for (int b = 0; b < c.B; ++b)
      all += (size_t)draft_row_groups(c.req(b), c.G, c.p.R) * c.Hkv * units.share[b].nch;
    CHECK(taken.size() == all);
  }

  // ---- the join: its blocks, in rounds where there are more pieces
  const int OC = c.p.D / 4, sets = 256 / OC, most = c.p.one_round ? 0 : 16 < OC ? 16 : OC;
  std::map<std::tuple<int, int, int>, int> stored;  // b, h, row
  if (c.p.joins > 0) {
    const auto pieces = lookup(c, chunk, [&](int nch) { return draft_join_pieces(nch, most, c.p.R, sets); });
    const int64_t last = pieces.first.back();
    for (int64_t at = 0; at < last && (!c.p.one_round || at < c.p.joins); ++at) {
      DraftUnit u;
      CHECK(pieces.find(at, &u));
      const DraftReq r = c.req(u.b);
      const DraftJoin j = draft_join(u, r, c.G, c.Hkv, c.p.R, 16 * c.p.MT, sets, most);
      CHECK(u.nch > 1 && j.h >= 0 && j.h < c.Hkv && j.rt >= 0 && j.rt < u.groups && j.row >= 0 && j.row < c.p.R);
      CHECK(!j.serial || u.nch <= OC);  // a lane of a set for each chunk
      for (int p = 0; p < (j.serial ? sets : 1); ++p) {
        const int rr = j.row + p, row = j.r0 + rr;
        if (row >= j.nrow) continue;
        CHECK(rr < c.p.R && row < r.n * c.G && (int64_t)r.s0 + row / c.G < c.rows);
        CHECK((stored[std::make_tuple(u.b, j.h, row)]++) == 0);
        ++joined;
        for (int ch = 0; ch < u.nch; ++ch) {
          const int64_t s = j.base + ch * j.step;
          CHECK(s >= 0 && s < c.p.slots);
          const auto it = taken.find(std::make_tuple(u.b, j.rt, j.h, ch));
          if (ordinary) CHECK(it != taken.end());
          if (it != taken.end()) CHECK(it->second == s);
        }
      }
    }
  }
  if (ordinary) {
    size_t all = 0;
    for (int b = 0; b < c.B; ++b)
      if (units.share[b].nch > 1) all += (size_t)c.req(b).n * c.G * c.Hkv;
    CHECK(stored.size() == all);
  }
}

int main() {
  std::mt19937 g(11);
  auto pick = [&](std::vector<int> v) { return v[g() % v.size()]; };
  auto upto = [&](int64_t n) { return (int)(g() % (uint64_t)(n + 1)); };
  for (calls = 0; calls < 1500; ++calls) {
    const bool damaged = calls % 3 == 2;
    Call c;
    c.es = pick({2, 2, 4});
    const int Dk = 16 * (1 + upto(15)), Dv = 16 * (1 + upto(15));
    c.Hkv = pick({1, 2, 3, 8}), c.G = pick({1, 2, 5, 8, 16}), c.H = c.G * c.Hkv;
    c.B = 1 + upto(pick({0, 3, 63, 70, 200}));
    c.shift = 4 + upto(4);
    const int most = c.B > 60 ? pick({1, 4}) : pick({1, 1, 4, 30, 200});
    c.width = 1 + upto(pick({40, 400, 4000}) * 16 >> c.shift);
    c.starts = {0};
    for (int b = 0; b < c.B; ++b) {
      const int n = upto(most);
      c.starts.push_back(c.starts.back() + n);
      const int ctx = upto(3) == 0 ? c.cap() : upto(pick({10, 300, c.cap()}));
      c.lens.push_back(damaged && upto(3) == 0 ? (int)g() : n + ctx);
    }
    c.rows = damaged ? upto(c.starts.back() + 3) : c.starts.back() + upto(3);
    if (damaged && upto(1))
      for (int& s : c.starts)
        if (upto(2) == 0) s = (int)g();
    if (c.rows == 0) continue;
    c.p = draft_plan(Dk, Dv, c.es, c.B, c.rows, c.H, c.Hkv, c.width, 1 << c.shift);
    c.KT = draft_tile(c.p.D, c.es, c.p.NW);
    if (c.p.units > 20000) continue;
    check(c, !damaged);
  }
  // binary search of the page tables: the last request that begins at x or before
  for (int i = 0; i < 2000; ++i) {
    const int B = 1 + upto(70);
    std::vector<int32_t> s{0};
    for (int b = 0; b < B; ++b) s.push_back(s.back() + upto(2) * upto(9));
    for (int x = 0; x < s.back(); ++x) {
      const int b = table_find(s.data(), B, x);
      CHECK(b >= 0 && b < B && s[b] <= x && x < s[b + 1]);
    }
  }
  std::printf("%ld calls, %ld units, %ld rows joined, %d failures\n", calls, units_seen, joined, fails);
  return fails != 0;
}
