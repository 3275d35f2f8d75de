// Whether the layers of a paged cache, and the lists that say what moves in
// them, have memory of their own: on the host, to the byte, for any strides
// (keys beside values in one buffer, layers inside pages, heads before tokens).
#pragma once
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <cstdlib>

#include "htree_cache_host.h"

namespace htree {

// Runs of `run` bytes at `at` + i0 step[0] + i1 step[1] + .., 0 <= id < n[d];
// steps descend, no n is 1.
struct Runs {
  static constexpr int kDims = 4;
  int64_t at, run;
  int dims = 0;
  int64_t n[kDims], step[kDims];
  bool huge = false;  // steps past any address

  void add(int64_t count, int64_t by) {
    if (count <= 1) return;
    if (by > ((int64_t)1 << 56) / count) {
      huge = true;
      return;
    }
    int d = dims++;
    for (; d && step[d - 1] < by; --d) n[d] = n[d - 1], step[d] = step[d - 1];
    n[d] = count, step[d] = by;
  }
  int64_t end() const {
    int64_t e = at + run;
    for (int d = 0; d < dims; ++d) e += (n[d] - 1) * step[d];
    return e;
  }
};

// Whether there are whole numbers i[d] in lo[d] .. hi[d] with
// below < x + sum i[d] step[d] < above.  Steps descend and are positive.  Where
// each is at least what the smaller ones span, as in any ordinary layout, two
// numbers a step are looked at; a search of more than kTries gives up, as true.
struct SumSearch {
  static constexpr int kDims = 2 * Runs::kDims, kTries = 1 << 14;
  int dims = 0, tries = 0;
  int64_t lo[kDims], hi[kDims], step[kDims], below, above;
  int64_t rest_lo[kDims + 1], rest_hi[kDims + 1];  // of the sum from d on

  // (in descending order; equal steps become one)
  void add(int64_t l, int64_t h, int64_t by) {
    if (dims && step[dims - 1] == by) {
      lo[dims - 1] += l, hi[dims - 1] += h;
      return;
    }
    lo[dims] = l, hi[dims] = h, step[dims++] = by;
  }
  static int64_t floor_div(int64_t x, int64_t y) { return x / y - (x % y < 0); }
  bool from(int d, int64_t x) {
    if (++tries > kTries) return true;
    if (d == dims) return below < x && x < above;
    const int64_t first = std::max(lo[d], -floor_div(x + rest_hi[d + 1] - below - 1, step[d]));
    const int64_t last = std::min(hi[d], floor_div(above - 1 - x - rest_lo[d + 1], step[d]));
    for (int64_t i = first; i <= last; ++i)
      if (from(d + 1, x + i * step[d])) return true;
    return false;
  }
  bool find(int64_t x) {
    rest_lo[dims] = rest_hi[dims] = 0;
    for (int d = dims - 1; d >= 0; --d) {
      rest_lo[d] = rest_lo[d + 1] + lo[d] * step[d];
      rest_hi[d] = rest_hi[d + 1] + hi[d] * step[d];
    }
    return from(0, x);
  }
};

// whether two of r's own runs share a byte
inline bool runs_overlap(const Runs& r) {
  int64_t span = r.run;
  bool nested = true;
  for (int d = r.dims - 1; d >= 0; --d) {
    if (r.step[d] == 0) return true;
    nested &= r.step[d] >= span;
    span += (r.n[d] - 1) * r.step[d];
  }
  if (nested) return false;
  // two places: their first difference, in the order of the steps, is positive
  for (int f = 0; f < r.dims; ++f) {
    SumSearch s;
    s.below = -r.run, s.above = r.run;
    for (int d = f; d < r.dims; ++d) s.add(d == f ? 1 : 1 - r.n[d], r.n[d] - 1, r.step[d]);
    if (s.find(0)) return true;
  }
  return false;
}

// whether runs of a and of b share a byte (neither's own do: no step is 0)
inline bool runs_overlap(const Runs& a, const Runs& b) {
  if (a.run <= 0 || b.run <= 0 || a.at >= b.end() || b.at >= a.end()) return false;
  SumSearch s;
  s.below = -b.run, s.above = a.run;
  for (int i = 0, j = 0; i < a.dims || j < b.dims;)
    if (j == b.dims || (i < a.dims && a.step[i] >= b.step[j])) s.add(1 - a.n[i], 0, a.step[i]), ++i;
    else s.add(0, b.n[j] - 1, b.step[j]), ++j;
  return s.find(b.at - a.at);
}

// Layers of one layout at p[0 .. n): tensors at even steps are one.  Adds them
// to `out` (room for n); p is sorted where it does not ascend or descend evenly.
inline int layer_runs(Runs layer, int64_t* p, int n, Runs* out) {
  auto even = [&](int a, int b) {  // p[a .. b) at one step
    for (int i = a + 2; i < b; ++i)
      if (p[i] - p[i - 1] != p[a + 1] - p[a]) return false;
    return true;
  };
  if (even(0, n)) {
    if (n > 1 && p[1] < p[0]) std::reverse(p, p + n);
  } else {
    std::sort(p, p + n);
  }
  int made = 0;
  for (int a = 0, b; a < n; a = b) {
    for (b = std::min(a + 2, n); b < n && p[b] - p[b - 1] == p[a + 1] - p[a]; ++b) {
    }
    Runs r = layer;
    r.at = p[a];
    r.add(b - a, b - a > 1 ? p[a + 1] - p[a] : 0);
    out[made++] = r;
  }
  return made;
}

// HTREE_OK if all layers (k and v: a layer's runs, whatever their `at`) and the
// lists `in` have memory of their own.
inline int layers_apart(const Runs& k, const Runs& v, int layers, void* const* k_at, void* const* v_at,
                        const Range* in, int n_in) {
  if (k.huge || v.huge) return HTREE_EUNSUPPORTED;
  constexpr int kFew = 64;
  int64_t few_at[kFew];
  Runs few[2 * kFew];
  void* more = nullptr;
  int64_t* at = few_at;
  Runs* r = few;
  if (layers > kFew) {
    more = std::malloc((size_t)layers * (sizeof(int64_t) + 2 * sizeof(Runs)));
    if (!more) return (int)hipErrorOutOfMemory;
    r = (Runs*)more, at = (int64_t*)(r + 2 * layers);
  }
  auto each = [&](void* const* p) {
    for (int l = 0; l < layers; ++l) at[l] = (int64_t)(uintptr_t)p[l];
    return at;
  };
  int n = layer_runs(k, each(k_at), layers, r);
  n += layer_runs(v, each(v_at), layers, r + n);
  std::sort(r, r + n, [](const Runs& a, const Runs& b) { return a.at < b.at; });
  int rc = HTREE_OK;
  for (int i = 0; i < n && rc == HTREE_OK; ++i) {
    if (r[i].huge) rc = HTREE_EUNSUPPORTED;
    else if (runs_overlap(r[i])) rc = HTREE_EOVERLAP;
  }
  for (int i = 0; i < n && rc == HTREE_OK; ++i) {
    const int64_t end = r[i].end();
    for (int j = i + 1; j < n && r[j].at < end && rc == HTREE_OK; ++j)
      if (runs_overlap(r[i], r[j])) rc = HTREE_EOVERLAP;
    for (int j = 0; j < n_in && rc == HTREE_OK; ++j) {
      Runs list;
      list.at = (int64_t)(uintptr_t)in[j].at, list.run = in[j].bytes;
      if (runs_overlap(r[i], list)) rc = HTREE_EOVERLAP;
    }
  }
  std::free(more);
  return rc;
}

}  // namespace htree
