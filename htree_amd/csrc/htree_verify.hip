// Verification of drafted tokens against the target's probabilities, from
// given uniform numbers.
//
// p and q are the target's and the drafter's probabilities after a row.  At a
// row its drafted children c are tried in turn: with T the mass that is left
// (p at first) and S its sum (1 at first), child c of token x is accepted if
// u_c S q(x) < T(x); a rejected one takes q's mass away, T <- max(T - S q, 0),
// which is max(p - a q, 0) with a the sum of the S so far.  Without a drafter's
// probabilities a draft, however it was chosen, has q = 1 at its token: accepted if
// u_c S < p(x), a rejected one takes its token away.  The walk goes on at the
// accepted child; where none is, the next token is drawn from T.
//
// All sums are fp64: the answers are tokens, and the rounding of an fp32 sum
// over a vocabulary moves the borders between them.
#include <cmath>

#include "htree_cache_host.h"
#include "htree_cache_index.h"
#include "htree_common.h"

namespace htree {

constexpr int kVerifyRows = 1024;    // of a request that are looked at
constexpr int kVerifyThreads = 1024;
constexpr int kVerifyWaves = kVerifyThreads / 64;
constexpr int kVerifyStep = 64 * 8;  // elements that a wave takes at once: 8 a lane
constexpr int kVerifySteps = 4;      // steps in a range, at least; of 16-bit types as many are in flight

// Few requests over a large vocabulary: `parts` blocks share a request's sums.
constexpr int kVerifyParts = 4;        // at most: their waves' sums fill a wave
constexpr int kVerifySplit = 1 << 17;  // elements of a row of p (and q) from which on they do
constexpr int kVerifyFull = 256;       // blocks that fill the GPU
constexpr int64_t kVerifyAll = 1 << 28;  // bytes of a call whose rows are all searched, greedily

// where a request's walk ended, for verify_draw_kernel
struct VerifyEnd {
  double off;
  int32_t row, node, n;  // row -1: the request has none
  int32_t unused;
};

struct VerifyArgs {
  VerifyEnd* ends;  // [B]
  double* sums;     // [B][parts][waves]
  int32_t* largest; // [rows], greedily
  int32_t parts;
  const char *p, *q;
  const int64_t* tokens;
  const int32_t *starts, *parents;
  const float *uniforms, *draws;
  int32_t *kept, *path;
  int64_t* next;
  int64_t p_row, q_row;  // elements
  int32_t B, rows, V;
};

// NV elements from anywhere: rows of an odd vocabulary begin at any element
template <typename T, int NV>
struct __attribute__((packed, aligned(sizeof(T)))) Elements {
  T v[NV];
};

// what an entry counts for: nothing if it is no positive number
template <typename T>
__device__ __forceinline__ float mass(T x) {
  const float f = fmaxf((float)x, 0.f);  // (of a NaN: 0)
  return f < INFINITY ? f : 0.f;
}
__device__ __forceinline__ double left_of(float p, float q, double a) { return fmax((double)p - a * (double)q, 0.0); }

// the value that DPP pattern CTRL brings to a lane, 0 where it brings none
template <int CTRL, int ROWS>
__device__ __forceinline__ double from_lane(double x) {
  const int lo = __builtin_amdgcn_update_dpp(0, __double2loint(x), CTRL, ROWS, 0xf, true);
  const int hi = __builtin_amdgcn_update_dpp(0, __double2hiint(x), CTRL, ROWS, 0xf, true);
  return __hiloint2double(hi, lo);
}
// Sums up to a lane, in the same order whoever asks: within rows of 16 lanes,
// then the rows in front.  A quarter of the time of shuffles through LDS.
__device__ __forceinline__ double wave_scan(double x) {
  x += from_lane<0x111, 0xf>(x);  // from the lane in front,
  x += from_lane<0x112, 0xf>(x);  // two,
  x += from_lane<0x114, 0xf>(x);  // four
  x += from_lane<0x118, 0xf>(x);  // and eight in front
  x += from_lane<0x142, 0xa>(x);  // rows 1, 3: the last lane of the row in front
  x += from_lane<0x143, 0xc>(x);  // rows 2, 3: lane 31
  return x;
}
__device__ __forceinline__ double lane_value(double x, int lane) {
  return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(x), lane),
                          __builtin_amdgcn_readlane(__double2loint(x), lane));
}
__device__ __forceinline__ double wave_sum(double x) { return lane_value(wave_scan(x), 63); }

struct VerifyLds {
  int32_t parent[kVerifyRows], token[kVerifyRows];
  int32_t largest[kVerifyWaves], best[kVerifyRows];
  float p[kVerifyRows], q[kVerifyRows], u[kVerifyRows];
  double red[kVerifyWaves];
  double sums[kVerifyParts * kVerifyWaves];  // of the ranges
  int32_t found;
};

// The first child of `node` behind row c, -1: none.  The same in every wave.
__device__ __forceinline__ int next_child(const VerifyLds& l, int n, int node, int c) {
  const int lane = threadIdx.x & 63;
  for (int g = c + 1; g < n; g += 64) {
    const uint64_t hit = __ballot(g + lane < n && l.parent[min(g + lane, kVerifyRows - 1)] == node);
    if (hit) return g + __builtin_ctzll(hit);
  }
  return -1;
}

// whether a child of `node` before row c has c's token
__device__ __forceinline__ bool had_token(const VerifyLds& l, int node, int c) {
  const int lane = threadIdx.x & 63, x = l.token[c];
  for (int g = node + 1; g < c; g += 64) {
    const int i = min(g + lane, kVerifyRows - 1);
    if (__ballot(g + lane < c && l.parent[i] == node && l.token[i] == x)) return true;
  }
  return false;
}

// What is left of the target's probabilities at a row: max(p - a q, 0), p
// itself (a = 0), or p without the tokens of the row's children.
template <typename T>
struct Left {
  const T *p, *q;  // q: nullptr, nothing of it is taken off
  double off;
  int node, n;     // children that take their tokens away are rows of this parent; n = 0: none do
};

template <typename T>
struct Eight {
  Elements<T, 8> p, q;
};
// The eight elements from e on; where the row ends before, its last eight.
// (V >= 8.)
template <typename T>
__device__ __forceinline__ void load_p(const Left<T>& l, int64_t e, int V, Eight<T>* x) {
  x->p = *(const Elements<T, 8>*)(l.p + min(e, (int64_t)V - 8));
}
template <typename T>
__device__ __forceinline__ void load_q(const Left<T>& l, int64_t e, int V, Eight<T>* x) {
  x->q = *(const Elements<T, 8>*)(l.q + min(e, (int64_t)V - 8));
}

// The largest of eight bit patterns, as unsigned numbers: below infinity's
// all of them are numbers that are not negative.
__device__ __forceinline__ uint32_t most_bits(const Elements<float, 8>& x) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __builtin_bit_cast(uint32_t, x.v[i]));
  return m;
}
template <typename T>
__device__ __forceinline__ uint32_t most_bits(const Elements<T, 8>& x) {
  typedef __attribute__((ext_vector_type(8))) unsigned short u16x8;
  typedef __attribute__((ext_vector_type(2))) unsigned short u16x2;
  const u16x8 v = __builtin_bit_cast(u16x8, x);
  const u16x2 m = __builtin_elementwise_max(__builtin_elementwise_max(v.s01, v.s23),
                                            __builtin_elementwise_max(v.s45, v.s67));
  return max((uint32_t)m.x, (uint32_t)m.y);
}
__device__ __forceinline__ uint32_t infinity_bits(float) { return 0x7f800000u; }
__device__ __forceinline__ uint32_t infinity_bits(__bf16) { return 0x7f80u; }
__device__ __forceinline__ uint32_t infinity_bits(_Float16) { return 0x7c00u; }

// t of those eight elements.  mass() of each would be a third of the instructions:
// only eights that hold something else than finite numbers >= 0 go through it.
template <typename T>
__device__ __forceinline__ void left_eight(const Left<T>& l, Eight<T>& x, double* t) {
  if (most_bits(x.p) >= infinity_bits(T())) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x.p.v[i] = (T)mass(x.p.v[i]);
  }
  if (l.q) {
    if (most_bits(x.q) >= infinity_bits(T())) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x.q.v[i] = (T)mass(x.q.v[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = left_of((float)x.p.v[i], (float)x.q.v[i], l.off);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = (double)(float)x.p.v[i];
  }
}

// What a lane's eight elements from e on count for: those that are there, and
// whose tokens the row's children do not take away (`some`: there may be such).
// The wave's elements are e0 .. e0 + 511.
template <typename T>
__device__ __forceinline__ void count_eight(const Left<T>& l, const VerifyLds& s, Eight<T>& x, int64_t e0, int V,
                                            bool some, double* t) {
  const int lane = threadIdx.x & 63;
  const int64_t e = e0 + lane * 8;
  left_eight(l, x, t);
  int at = lane * 8;  // of the first element, from e0
  if (e0 + kVerifyStep > V) {
    const int64_t over = e - min(e, (int64_t)V - 8);  // elements that the lanes in front have
    at -= (int)over;
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = i < over ? 0.0 : t[i];
  }
  if (!some) return;
  for (int c0 = l.node + 1; c0 < l.n; c0 += 64) {
    const int c = min(c0 + lane, kVerifyRows - 1);
    const int64_t token = s.token[c] - e0;
    uint64_t hit = __ballot(c0 + lane < l.n && s.parent[c] == l.node && token >= 0 && token < kVerifyStep);
    for (; hit; hit &= hit - 1) {
      const int gone = __shfl((int)token, __builtin_ctzll(hit));
#pragma unroll
      for (int i = 0; i < 8; ++i) t[i] = at + i == gone ? 0.0 : t[i];
    }
  }
}

// Element e alone, for vocabularies of less than eight.
template <typename T>
__device__ __forceinline__ double count_one(const Left<T>& l, const VerifyLds& s, int e) {
  for (int c = l.node + 1; c < l.n; ++c)
    if (s.parent[c] == l.node && s.token[c] == e) return 0.0;
  return l.q ? left_of(mass(l.p[e]), mass(l.q[e]), l.off) : (double)mass(l.p[e]);
}

// Range w is the elements w size .. (w + 1) size - 1.
__device__ __forceinline__ int64_t range_size(int V, int ranges) {
  constexpr int once = kVerifySteps * kVerifyStep;
  return (((int64_t)V + once - 1) / once + ranges - 1) / ranges * once;
}

// A wave's sum of range w.  (Taking the children's tokens off the sum
// afterwards would round away what is left beside them.)
template <typename T>
__device__ __forceinline__ double range_sum(const Left<T>& l, const VerifyLds& s, int V, int w, int ranges) {
  constexpr int U = sizeof(T) == 4 ? kVerifySteps / 2 : kVerifySteps;  // steps in flight
  const int lane = threadIdx.x & 63;
  const int64_t size = range_size(V, ranges), e0 = w * size, e1 = min(e0 + size, (int64_t)V);
  bool some = false;  // a child's token in this range
  for (int i = l.node + 1 + lane; i < l.n; i += 64)
    some |= s.parent[i] == l.node && s.token[i] >= e0 && s.token[i] < e1;
  some = __any(some);
  double sum = 0.0;
  for (int64_t e = e0; e < e1; e += U * kVerifyStep) {
    Eight<T> x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) load_p(l, e + u * kVerifyStep + lane * 8, V, &x[u]);
    if (l.q) {
#pragma unroll
      for (int u = 0; u < U; ++u) load_q(l, e + u * kVerifyStep + lane * 8, V, &x[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      double t[8];
      count_eight(l, s, x[u], e + u * kVerifyStep, V, some, t);
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += t[i];
    }
  }
  return wave_sum(sum);
}

// The thread whose share of a cumulative sum first passes t: every thread
// comes with its share `mine` and gets the sum before it, from `base` on.
// Returns that thread, -1 where rounding or the range leaves none; `all` is the
// sum behind the last thread.
__device__ __forceinline__ int find_share(double mine, double base, double t, VerifyLds& s, double* before,
                                          double* all) {
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const double inc = wave_scan(mine);
  __syncthreads();  // what an earlier call left has been read
  if (tid == 0) s.found = 0x7fffffff;
  if (lane == 63) s.red[wv] = inc;
  __syncthreads();
  const double waves = wave_scan(lane < kVerifyWaves ? s.red[lane] : 0.0);
  const double front = base + (wv ? lane_value(waves, wv - 1) : 0.0);
  *all = base + lane_value(waves, 63);
  // the sum before a thread is the one up to its neighbour, to the bit
  const double up = __shfl_up(inc, 1);
  *before = lane ? front + up : front;
  const uint64_t hit = __ballot(mine > 0.0 && front + inc > t);
  if (hit && lane == 0) atomicMin(&s.found, wv * 64 + __builtin_ctzll(hit));
  __syncthreads();
  return s.found == 0x7fffffff ? -1 : s.found;
}

// The first element whose cumulative sum passes `draw` of the total, or where
// rounding leaves none the last with any mass; -1: there is no mass.  The
// ranges' sums (64 at most) are in s.sums.
template <typename T>
__device__ __forceinline__ int64_t find_element(const Left<T>& l, VerifyLds& s, int V, int ranges, float draw) {
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const double part = draw > 0.f ? (double)draw : 0.0;
  if (V < 8) {
    double total = 0.0, sum = 0.0;
    for (int e = 0; e < V; ++e) total += count_one(l, s, e);
    int at = -1;
    for (int e = 0; e < V && !(sum > part * total); ++e) {
      const double x = count_one(l, s, e);
      if (x > 0.0) at = e;
      sum += x;
    }
    return at;
  }
  // its range: the same choice in every wave
  const double mine = lane < ranges ? s.sums[lane] : 0.0, up_to = wave_scan(mine);
  const double t = part * lane_value(up_to, 63);
  const uint64_t any = __ballot(mine > 0.0), pass = __ballot(mine > 0.0 && up_to > t);
  if (!any) return -1;
  const int w = pass ? __builtin_ctzll(pass) : 63 - __builtin_clzll(any);
  double base = w ? lane_value(up_to, w - 1) : 0.0;
  const int64_t size = range_size(V, ranges), e0 = w * size, e1 = min(e0 + size, (int64_t)V);
  __shared__ int64_t token;
  __syncthreads();
  if (tid == 0) token = -1;
  for (int64_t e = e0; e < e1; e += kVerifyThreads * 8) {
    // ranges are whole steps: a wave's elements are in this one or behind it
    const int64_t first = e + wv * kVerifyStep, at = min(first + lane * 8, (int64_t)V - 8);
    double x[8], share = 0.0, before, all;
    if (first < e1) {
      Eight<T> v;
      load_p(l, at, V, &v);
      if (l.q) load_q(l, at, V, &v);
      count_eight(l, s, v, first, V, l.n > 0, x);
#pragma unroll
      for (int i = 0; i < 8; ++i) share += x[i];
    }
    int who = find_share(share, base, t, s, &before, &all);
    const bool passed = who >= 0;
    if (!passed) {
      // the last thread with a share, for when none passes
      __syncthreads();
      if (tid == 0) s.found = -1;
      __syncthreads();
      const uint64_t hit = __ballot(share > 0.0);
      if (hit && (tid & 63) == 0) atomicMax(&s.found, (tid | 63) - __builtin_clzll(hit));
      __syncthreads();
      who = s.found;
    }
    if (tid == who) {
      int last = 0;
      double run = before;
      bool done = false;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (!done && x[i] > 0.0) {
          last = i;
          run += x[i];
          done = passed && run > t;
        }
      token = at + last;
    }
    if (passed) break;
    base = all;
  }
  __syncthreads();
  return token;
}

// The sum over a row, or over part `part` of `parts` of it, by the whole block:
// its waves' shares in s.sums.
template <typename T>
__device__ __forceinline__ double row_sum(const Left<T>& l, VerifyLds& s, int V, int part, int parts) {
  if (V < 8) {
    double all = 0.0;
    for (int e = 0; e < V; ++e) all += count_one(l, s, e);
    return all;
  }
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const double x = range_sum(l, s, V, part * kVerifyWaves + wv, parts * kVerifyWaves);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s.sums[wv] = x;
  __syncthreads();
  const int lane = threadIdx.x & 63;
  return wave_sum(lane < kVerifyWaves ? s.sums[lane] : 0.0);
}

__device__ __forceinline__ int load_row(const VerifyArgs& a, VerifyLds& l, int s0, int i) {
  const int64_t x = a.tokens[s0 + i];
  int up = a.parents ? draft_parent(a.parents[s0 + i], i) : i - 1;
  if (x < 0 || x >= a.V) up = -1;  // no token: no draft
  l.parent[i] = up;
  l.token[i] = (int)x;
  return up;
}

// A request's first row and how many of its rows are looked at.  Its path, but
// for the kept rows behind the first, is written by part 0; a request without
// rows is done with this.
struct Request {
  int s0, n;
};
__device__ __forceinline__ Request open_request(const VerifyArgs& a, int b, int part) {
  const int tid = threadIdx.x;
  const int s0 = min(max(a.starts[b], 0), a.rows), s1 = min(max(a.starts[b + 1], s0), a.rows);
  if (part == 0) {
    // (unsigned: behind the last of 2^31 - 1 rows a signed one would begin again below zero)
    const uint32_t first = s0, last = s1, rows = a.rows;
    for (uint32_t i = first + tid; i < last; i += kVerifyThreads) a.path[i] = i == first ? 0 : -1;
    // rows of no request
    if (b == 0)
      for (uint32_t i = tid; i < first; i += kVerifyThreads) a.path[i] = -1;
    if (b == a.B - 1)
      for (uint32_t i = last + tid; i < rows; i += kVerifyThreads) a.path[i] = -1;
    if (s0 == s1 && tid == 0) {
      a.kept[b] = 0, a.next[b] = -1;
      if (a.parts > 1) a.ends[b].row = -1;
    }
  }
  return {s0, min(s1 - s0, kVerifyRows)};
}

// A block a request: its drafts' tests one after another, the path, then the
// next token from what is left at the last kept row.  With `parts` blocks a
// request each makes the same tests, and a part of the last sums.
// Bound by a chain of latencies (rows, tokens, their elements, the row's first
// loads, two scans: 7 us, three launches took 12 of them) and by the 64-bit
// arithmetic of the sums, 9 instructions an element of p and q.  A chain of 5
// drafts over 32000 fp32 entries 8.8 us; 256 fixed trees over 32768 12.3 us; 16
// trees drawn over 50001 16.4 us, of it 3.5 for each sum between siblings.
template <typename T>
__global__ __launch_bounds__(kVerifyThreads) void verify_drafts_kernel(VerifyArgs a) {
  __shared__ VerifyLds l;
  const int b = blockIdx.x, part = blockIdx.y, tid = threadIdx.x;
  const T *P = (const T*)a.p, *Q = (const T*)a.q;
  const auto [s0, n] = open_request(a, b, part);
  if (n == 0) return;
  const bool writes = part == 0 && tid == 0;
  for (int i = tid; i < n; i += kVerifyThreads) {
    const int up = load_row(a, l, s0, i);
    if (up >= 0) {
      l.p[i] = mass(P[(s0 + up) * a.p_row + l.token[i]]);
      l.q[i] = Q ? mass(Q[(s0 + up) * a.q_row + l.token[i]]) : 1.f;
      const float u = a.uniforms[s0 + i];
      l.u[i] = u > 0.f ? u : 0.f;
    }
  }
  const float draw = a.draws[b];
  __syncthreads();  // also: the path's -1s are written before its places
  Left<T> left = {P + s0 * a.p_row, nullptr, 0.0, 0, 0};
  int node = 0, kept = 1, c = next_child(l, n, 0, 0);
  double S = 1.0, total;
  // one place for the sums over a row, whichever they are for: the code of three
  // would be read from memory by every block
  for (;;) {
    while (c >= 0) {
      const double px = l.p[c], qx = l.q[c], u = l.u[c];
      bool ok, gone = false;
      if (Q) {
        ok = u * S * qx < px - left.off * qx;
      } else {
        gone = had_token(l, node, c);
        ok = !gone && u * S < px;
      }
      if (ok) {
        node = c, S = 1.0;
        left = {P + (s0 + node) * a.p_row, nullptr, 0.0, node, 0};
        if (writes) a.path[s0 + kept] = c;
        ++kept;
      }
      c = next_child(l, n, node, c);
      if (ok) continue;
      if (Q) {
        left.q = Q + (s0 + node) * a.q_row;
        left.off += S;
        break;  // for S, what is left of the mass
      }
      left.node = node, left.n = n;
      if (!gone) S -= px;
    }
    const bool ended = c < 0;
    total = row_sum(left, l, a.V, ended ? part : 0, ended ? a.parts : 1);
    if (!ended) {
      S = total;
      continue;
    }
    if (a.parts > 1 || total > 0.0 || !(left.q || left.n)) break;
    left.q = nullptr, left.n = 0;  // nothing left: from p itself
  }
  if (writes) a.kept[b] = kept;
  if (a.parts > 1) {
    if (tid < kVerifyWaves) a.sums[((int64_t)b * a.parts + part) * kVerifyWaves + tid] = l.sums[tid];
    if (writes) a.ends[b] = {left.off, s0 + node, node, left.n, 0};
    return;
  }
  const int64_t token = find_element(left, l, a.V, kVerifyWaves, draw);
  if (writes) a.next[b] = token;
}

// The next token of a request whose parts' sums are there: 4.2 us.  (The last
// part to finish could draw it, but the fences that show it the others' sums
// wrote back every cache: 160 us for 64 requests of 4 parts.)
template <typename T>
__global__ __launch_bounds__(kVerifyThreads) void verify_draw_kernel(VerifyArgs a) {
  __shared__ VerifyLds l;
  const int b = blockIdx.x, tid = threadIdx.x;
  const VerifyEnd end = a.ends[b];
  if (end.row < 0) return;
  const float draw = a.draws[b];
  const T *P = (const T*)a.p, *Q = (const T*)a.q;
  Left<T> left = {P + end.row * a.p_row, Q && end.off > 0.0 ? Q + end.row * a.q_row : nullptr, end.off, end.node,
                  end.n};
  int ranges = a.parts * kVerifyWaves;
  if (tid < ranges) l.sums[tid] = a.sums[(int64_t)b * ranges + tid];
  for (int i = tid; i < left.n; i += kVerifyThreads) load_row(a, l, end.row - end.node, i);
  __syncthreads();
  const int lane = tid & 63;
  if (!(wave_sum(lane < ranges ? l.sums[lane] : 0.0) > 0.0)) {  // nothing left: from p itself
    left.q = nullptr, left.n = 0, ranges = kVerifyWaves;
    row_sum(left, l, a.V, 0, 1);
  }
  const int64_t token = find_element(left, l, a.V, ranges, draw);
  if (tid == 0) a.next[b] = token;
}

// The index of a row's largest entry, of several the first; -1 where none is
// above -infinity (a NaN is not).  By the whole block.
template <typename T>
__device__ __forceinline__ int row_largest(const T* row, VerifyLds& s, int V) {
  constexpr int U = sizeof(T) == 4 ? kVerifySteps / 2 : kVerifySteps;
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  float most = -INFINITY;
  int at = -1;
  if (V < 8) {
    for (int e = 0; e < V; ++e) {
      const float x = (float)row[e];
      if (x > most) most = x, at = e;
    }
    return at;
  }
  const int64_t size = range_size(V, kVerifyWaves), e0 = wv * size, e1 = min(e0 + size, (int64_t)V);
  for (int64_t e = e0; e < e1; e += U * kVerifyStep) {
    Elements<T, 8> x[U];
    int64_t from[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {  // past the end: the last eight again
      from[u] = min(e + u * kVerifyStep + lane * 8, (int64_t)V - 8);
      x[u] = *(const Elements<T, 8>*)(row + from[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float v = (float)x[u].v[i];
        if (v > most) most = v, at = (int)from[u] + i;
      }
  }
  // (an index of -1 is the largest unsigned one)
  auto better = [&](float v, int i) {
    if (v > most || (v == most && (uint32_t)i < (uint32_t)at)) most = v, at = i;
  };
#pragma unroll
  for (int m = 32; m; m >>= 1) better(__shfl_xor(most, m), __shfl_xor(at, m));
  __syncthreads();
  if (lane == 0) s.p[wv] = most, s.largest[wv] = at;
  __syncthreads();
  most = -INFINITY, at = -1;
  for (int w = 0; w < kVerifyWaves; ++w) better(s.p[w], s.largest[w]);
  return at;
}

// A block a row: its largest entry.
template <typename T>
__global__ __launch_bounds__(kVerifyThreads) void verify_largest_kernel(VerifyArgs a) {
  __shared__ VerifyLds l;
  const int at = row_largest((const T*)a.p + blockIdx.x * a.p_row, l, a.V);
  if (threadIdx.x == 0) a.largest[blockIdx.x] = at;
}

// A block a request, greedily: a draft is kept if its token is the largest
// entry's after the row it was drafted after.  Those of all rows are there
// already, or are found row by row as the walk comes to them.
template <typename T>
__global__ __launch_bounds__(kVerifyThreads) void verify_greedy_kernel(VerifyArgs a) {
  __shared__ VerifyLds l;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const T* P = (const T*)a.p;
  const auto [s0, n] = open_request(a, b, 0);
  if (n == 0) return;
  for (int i = tid; i < n; i += kVerifyThreads) {
    load_row(a, l, s0, i);
    if (a.largest) l.best[i] = a.largest[s0 + i];
  }
  __syncthreads();
  int node = 0, kept = 1, token;
  for (;;) {
    token = a.largest ? l.best[node] : row_largest(P + (s0 + node) * a.p_row, l, a.V);
    int next = -1;
    for (int g = node + 1; g < n && next < 0; g += 64) {
      const int i = min(g + lane, kVerifyRows - 1);
      const uint64_t hit = __ballot(g + lane < n && l.parent[i] == node && l.token[i] == token);
      if (hit) next = g + __builtin_ctzll(hit);
    }
    if (next < 0) break;
    node = next;
    if (tid == 0) a.path[s0 + kept] = node;
    ++kept;
  }
  if (tid == 0) a.kept[b] = kept, a.next[b] = token;
}

// Blocks that share a request's sums: as many as have a CU to themselves.  64
// requests, 2 x 128000 16-bit entries: 15.0 us in two launches, 21.5 in one;
// below 2^17 entries the second launch costs more than the first one saves.
static int verify_parts(int32_t B, int32_t V, bool drawn) {
  const int64_t all = (int64_t)V * (drawn ? 2 : 1);
  if (all < kVerifySplit || 2 * B > kVerifyFull) return 1;
  return kVerifyFull / B < kVerifyParts ? kVerifyFull / B : kVerifyParts;
}

// Whether all rows are searched for their largest entry at once, or only those
// that the walk comes to: one after another, so that the longest path counts.
// 64 requests of 9 rows, 128000 16-bit entries (147 MB): 38 us at once, 67 one
// after another; 256 of 13 rows, 32768 fp32 (436 MB): 80 and 67.
static bool verify_all(int32_t dtype, int32_t rows, int32_t V) {
  return (int64_t)rows * V * (dtype == HTREE_F32 ? 4 : 2) <= kVerifyAll && rows < 1 << 21;  // (blocks of a grid)
}

}  // namespace htree

using namespace htree;

extern "C" int htree_verify_drafts_workspace_bytes(int32_t dtype, int32_t B, int32_t rows, int32_t V, int32_t drawn,
                                                   int32_t greedy, int64_t* bytes) {
  if (!bytes) return HTREE_ENULL;
  if (dtype != HTREE_F32 && dtype != HTREE_BF16 && dtype != HTREE_F16) return HTREE_ESHAPE;
  if (B < 0 || rows < 0 || V < 1 || (greedy && drawn)) return HTREE_ESHAPE;
  if (B > kCacheMaxRequests) return HTREE_EUNSUPPORTED;
  *bytes = 0;
  if (B == 0) return HTREE_OK;
  const int parts = verify_parts(B, V, drawn);
  if (greedy) *bytes = verify_all(dtype, rows, V) ? rows * 4ll : 0;
  else if (parts > 1) *bytes = B * ((int64_t)sizeof(VerifyEnd) + parts * kVerifyWaves * 8);
  return HTREE_OK;
}

extern "C" int htree_verify_drafts(int32_t dtype, int32_t B, int32_t rows, int32_t V, const void* target_probs,
                                   int64_t target_row, const void* draft_probs, int64_t draft_row,
                                   const int64_t* tokens, const int32_t* starts, const int32_t* parents,
                                   const float* uniforms, const float* draws, int32_t* kept, int32_t* path,
                                   int64_t* next_tokens, void* workspace, int64_t workspace_bytes, void* stream) {
  const bool greedy = !uniforms && !draws;
  int64_t need = 0;
  const int rc = htree_verify_drafts_workspace_bytes(dtype, B, rows, V, draft_probs != nullptr, greedy, &need);
  if (rc) return rc;
  if (target_row < 0 || draft_row < 0) return HTREE_ESHAPE;
  if (B == 0) return HTREE_OK;
  if (!starts || (!greedy && !draws) || !kept || !next_tokens) return HTREE_ENULL;
  if (rows && (!target_probs || !tokens || (!greedy && !uniforms) || !path)) return HTREE_ENULL;
  if (need && !workspace) return HTREE_ENULL;
  if (off16(workspace)) return HTREE_EUNSUPPORTED;
  if (workspace_bytes < need) return HTREE_EWORKSPACE;
  const int es = dtype == HTREE_F32 ? 4 : 2;
  const Range in[7] = {{target_probs, rows ? ((rows - 1) * target_row + V) * es : 0},
                       {draft_probs, rows && draft_probs ? ((rows - 1) * draft_row + V) * es : 0},
                       {tokens, rows * 8ll}, {starts, (B + 1) * 4ll}, {parents, parents ? rows * 4ll : 0},
                       {uniforms, uniforms ? rows * 4ll : 0}, {draws, draws ? B * 4ll : 0}};
  const Range out[4] = {{kept, B * 4ll}, {path, rows * 4ll}, {next_tokens, B * 8ll}, {workspace, need}};
  for (int i = 0; i < 4; ++i) {
    for (const Range& y : in)
      if (overlap(out[i], y)) return HTREE_EOVERLAP;
    for (int j = 0; j < i; ++j)
      if (overlap(out[i], out[j])) return HTREE_EOVERLAP;
  }
  VerifyArgs a;
  a.p = (const char*)target_probs, a.q = (const char*)draft_probs;
  a.tokens = tokens, a.starts = starts, a.parents = parents, a.uniforms = uniforms, a.draws = draws;
  a.kept = kept, a.path = path, a.next = next_tokens;
  a.p_row = target_row, a.q_row = draft_row;
  a.B = B, a.rows = rows, a.V = V;
  a.parts = greedy ? 1 : verify_parts(B, V, draft_probs != nullptr);
  a.ends = (VerifyEnd*)workspace;
  a.sums = (double*)(a.ends + B);
  a.largest = greedy && need ? (int32_t*)workspace : nullptr;
  hipStream_t s = (hipStream_t)stream;
#define HTREE_VERIFY(T)                                                                                     \
  do {                                                                                                      \
    if (greedy) {                                                                                           \
      if (a.largest)                                                                                        \
        hipLaunchKernelGGL((verify_largest_kernel<T>), dim3(rows), dim3(kVerifyThreads), 0, s, a);          \
      hipLaunchKernelGGL((verify_greedy_kernel<T>), dim3(B), dim3(kVerifyThreads), 0, s, a);                \
      break;                                                                                                \
    }                                                                                                       \
    hipLaunchKernelGGL((verify_drafts_kernel<T>), dim3(B, a.parts), dim3(kVerifyThreads), 0, s, a);         \
    if (a.parts > 1) hipLaunchKernelGGL((verify_draw_kernel<T>), dim3(B), dim3(kVerifyThreads), 0, s, a);   \
  } while (0)
  if (dtype == HTREE_F32) HTREE_VERIFY(float);
  else if (dtype == HTREE_BF16) HTREE_VERIFY(__bf16);
  else HTREE_VERIFY(_Float16);
#undef HTREE_VERIFY
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? HTREE_OK : (int)e;
}
