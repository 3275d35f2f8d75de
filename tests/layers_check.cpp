// Whether layers of a cache share memory (htree_layers.h), against the bytes
// themselves: small layouts of every kind, each marked byte by byte.
// Test infrastructure: built and run by tests/test_layers.py on the CPU.
#include <cstdio>
#include <random>
#include <vector>

#include "htree_layers.h"

using namespace htree;

static bool mark(std::vector<char>& taken, const Runs& r, int64_t at, int64_t n[3], int64_t st[3]) {
  bool clash = false;
  for (int64_t a = 0; a < n[0]; ++a)
    for (int64_t b = 0; b < n[1]; ++b)
      for (int64_t c = 0; c < n[2]; ++c)
        for (int64_t x = 0; x < r.run; ++x) {
          char& t = taken[at + a * st[0] + b * st[1] + c * st[2] + x];
          clash |= t;
          t = 1;
        }
  return clash;
}

int main() {
  std::mt19937 g(7);
  auto pick = [&](int lo, int hi) { return (int64_t)(lo + (int)(g() % (unsigned)(hi - lo + 1))); };
  long calls = 0, shared = 0, fails = 0;
  for (int i = 0; i < 60000; ++i) {
    const int layers = (int)pick(1, i % 50 ? 4 : 70), kind = (int)pick(0, 4);
    int64_t n[3] = {pick(1, 4), pick(1, 4), pick(1, 3)}, st[2][3], run[2] = {pick(1, 4), pick(1, 4)};
    std::vector<int64_t> at[2];
    if (kind == 0) {  // anything
      for (auto& s : st)
        for (auto& x : s) x = pick(0, 20);
      for (auto& a : at)
        for (int l = 0; l < layers; ++l) a.push_back(pick(0, 300));
    } else if (kind == 1) {  // layers of their own, at places in any order, some too near
      int64_t place = 0;
      std::vector<int64_t> all;
      for (int w = 0; w < 2; ++w) st[w][2] = run[w], st[w][1] = st[w][2] * n[2], st[w][0] = st[w][1] * n[1];
      const int64_t size = std::max(st[0][0], st[1][0]) * n[0];
      for (int l = 0; l < 2 * layers; ++l) all.push_back(place), place += size - (pick(0, 60) == 0) + pick(0, 2);
      if (pick(0, 1)) std::shuffle(all.begin(), all.end(), g);
      at[0].assign(all.begin(), all.begin() + layers), at[1].assign(all.begin() + layers, all.end());
    } else {  // one buffer: keys beside values, layers at one of the places between the strides
      const int64_t both = run[0] + run[1] - (pick(0, 9) == 0);
      int order[4] = {0, 1, 2, 3};  // page, token, head, layer
      std::shuffle(order, order + 4, g);
      int64_t s[4], by = both + pick(0, 2);
      for (int o : order) {
        s[o] = by;
        by *= (o == 3 ? layers : n[o]);
        by += pick(0, 3) - (pick(0, 19) == 0 ? 4 : 0);
      }
      for (int w = 0; w < 2; ++w) {
        for (int d = 0; d < 3; ++d) st[w][d] = std::max<int64_t>(s[d], 0);
        for (int l = 0; l < layers; ++l) at[w].push_back(l * std::max<int64_t>(s[3], 0) + w * run[0]);
      }
      if (kind > 2 && layers > 1)  // some of the layers alone, in any order
        for (auto& a : at) std::shuffle(a.begin(), a.end(), g), a.resize(a.size() - (kind == 4));
    }
    const int L = (int)at[0].size();
    Runs r[2];
    int64_t top = 400;
    for (int w = 0; w < 2; ++w) {
      r[w].at = 0, r[w].run = run[w];
      for (int d = 0; d < 3; ++d) r[w].add(n[d], st[w][d]);
      for (int64_t a : at[w]) top = std::max(top, a + r[w].end());
    }
    const int64_t list = pick(0, (int)std::min<int64_t>(top, 1 << 20)), bytes = pick(0, 2);
    std::vector<char> taken(top + 8, 0);
    bool clash = false;
    for (int w = 0; w < 2; ++w)
      for (int64_t a : at[w]) clash |= mark(taken, r[w], a, n, st[w]);
    for (int64_t x = 0; x < bytes; ++x) clash |= taken[list + x];
    const int64_t base = (int64_t)1 << 40;
    std::vector<void*> p[2];
    for (int w = 0; w < 2; ++w)
      for (int64_t a : at[w]) p[w].push_back((void*)(base + a));
    const Range in[1] = {{(void*)(base + list), bytes}};
    const int rc = layers_apart(r[0], r[1], L, p[0].data(), p[1].data(), in, 1);
    ++calls, shared += clash;
    if (rc != (clash ? HTREE_EOVERLAP : HTREE_OK) && ++fails < 10)
      printf("call %d kind %d layers %d: rc %d, bytes shared %d\n", i, kind, L, rc, clash);
  }
  printf("%ld calls, %ld shared, %ld failures\n", calls, shared, fails);
  return fails != 0;
}
