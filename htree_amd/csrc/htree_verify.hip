// Verification of drafted tokens against the target's probabilities, from
// given uniform numbers.
//
// p and q are the target's and the drafter's probabilities after a row.  At a
// row its drafted children c are tried in turn: with T the mass that is left
// (p at first) and S its sum (1 at first), child c of token x is accepted if
// u_c S q(x) < T(x); a rejected one takes q's mass away, T <- max(T - S q, 0),
// which is max(p - a q, 0) with a the sum of the S so far.  Without a drafter's
// probabilities a draft is what it is, q = 1 at its token: accepted if
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
constexpr int kVerifySegment = 8192; // elements of a row that a block sums: 8 a thread, 4 times (pick: once)
constexpr int kVerifySum = 256, kVerifyPick = 1024;  // threads

// where a request's walk ended
struct VerifyEnd {
  double off;      // a: T = max(p - a q, 0)
  int32_t row;     // of p and q, -1: the request has no rows
  int32_t node;    // the same within the request; its children are all rejected
};

struct VerifyArgs {
  const char *p, *q;
  const int64_t* tokens;
  const int32_t *starts, *parents;
  const float *uniforms, *draws;
  int32_t *kept, *path;
  int64_t* next;
  VerifyEnd* ends;  // [B]
  double* sums;     // [B][segments][2] of T and of p
  int64_t p_row, q_row;  // elements
  int32_t B, rows, V, segments;
};

// NV elements from anywhere: rows of an odd vocabulary begin at any element
template <typename T, int NV>
struct __attribute__((packed, aligned(sizeof(T)))) Elements {
  T v[NV];
};

// what an entry counts for: nothing if it is no positive number
template <typename T>
__device__ __forceinline__ float mass(T x) {
  const float f = (float)x;
  return f > 0.f && f < INFINITY ? f : 0.f;
}
__device__ __forceinline__ double left_of(float p, float q, double a) { return fmax((double)p - a * (double)q, 0.0); }

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
  for (int m = 32; m; m >>= 1) x += __shfl_xor(x, m);
  return x;
}

// rows s0 .. s0 + n - 1 are request b's
__device__ __forceinline__ int verify_rows(const VerifyArgs& a, int b, int* s0) {
  *s0 = min(max(a.starts[b], 0), a.rows);
  return min(max(a.starts[b + 1], *s0), a.rows) - *s0;
}

struct VerifyLds {
  int32_t parent[kVerifyRows], token[kVerifyRows];
  float p[kVerifyRows], q[kVerifyRows], u[kVerifyRows];
  double red[kVerifyPick / 64];
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

// A block a request: its drafts' tests, one after another, and the path.
template <typename T>
__global__ __launch_bounds__(kVerifyPick) void verify_walk_kernel(VerifyArgs a) {
  __shared__ VerifyLds l;
  const int b = blockIdx.x, tid = threadIdx.x, wv = tid >> 6;
  const T *P = (const T*)a.p, *Q = (const T*)a.q;
  int s0;
  const int rows = verify_rows(a, b, &s0), n = min(rows, kVerifyRows);
  for (int i = tid; i < rows; i += kVerifyPick) a.path[s0 + i] = i ? -1 : 0;
  // rows of no request
  if (b == 0)
    for (int i = tid; i < s0; i += kVerifyPick) a.path[i] = -1;
  if (b == a.B - 1)
    for (int i = s0 + rows + tid; i < a.rows; i += kVerifyPick) a.path[i] = -1;
  if (n == 0) {
    if (tid == 0) {
      a.kept[b] = 0;
      a.ends[b] = {0.0, -1, -1};
    }
    return;
  }
  for (int i = tid; i < n; i += kVerifyPick) {
    const int64_t x = a.tokens[s0 + i];
    int up = a.parents ? draft_parent(a.parents[s0 + i], i) : i - 1;
    if (x < 0 || x >= a.V) up = -1;  // no token: no draft
    l.parent[i] = up;
    l.token[i] = (int)x;
    if (up >= 0) {
      l.p[i] = mass(P[(s0 + up) * a.p_row + x]);
      l.q[i] = Q ? mass(Q[(s0 + up) * a.q_row + x]) : 1.f;
      const float u = a.uniforms[s0 + i];
      l.u[i] = u > 0.f ? u : 0.f;
    }
  }
  __syncthreads();  // also: the path's -1s are written before its places
  int node = 0, kept = 1;
  double off = 0.0, S = 1.0;
  for (int c = next_child(l, n, 0, 0); c >= 0;) {
    const double px = l.p[c], qx = l.q[c], u = l.u[c];
    bool ok, gone = false;
    if (Q) {
      ok = u * S * qx < px - off * qx;
    } else {
      gone = had_token(l, node, c);
      ok = !gone && u * S < px;
    }
    if (ok) {
      node = c, off = 0.0, S = 1.0;
      if (tid == 0) a.path[s0 + kept] = c;
      ++kept;
      c = next_child(l, n, node, c);
      continue;
    }
    c = next_child(l, n, node, c);
    if (!Q) {
      if (!gone) S -= px;
      continue;
    }
    off += S;
    if (c < 0) break;
    // the mass that is left for the next sibling
    constexpr int NV = 16 / (int)sizeof(T);
    const T *pr = P + (s0 + node) * a.p_row, *qr = Q + (s0 + node) * a.q_row;
    double sum = 0.0;
    for (int e = tid * NV; e < a.V; e += kVerifyPick * NV) {
      if (e + NV <= a.V) {
        const Elements<T, NV> x = *(const Elements<T, NV>*)(pr + e), y = *(const Elements<T, NV>*)(qr + e);
#pragma unroll
        for (int i = 0; i < NV; ++i) sum += left_of(mass(x.v[i]), mass(y.v[i]), off);
      } else {
        for (int i = e; i < a.V; ++i) sum += left_of(mass(pr[i]), mass(qr[i]), off);
      }
    }
    sum = wave_sum(sum);
    __syncthreads();
    if ((tid & 63) == 0) l.red[wv] = sum;
    __syncthreads();
    S = 0.0;
    for (int w = 0; w < kVerifyPick / 64; ++w) S += l.red[w];
  }
  if (tid == 0) {
    a.kept[b] = kept;
    a.ends[b] = {off, s0 + node, node};
  }
}

// Bits of the tokens of a segment that the walk's rejected children took away.
__device__ __forceinline__ void taken_bits(const VerifyArgs& a, int b, int node, int64_t e0, uint32_t* bits,
                                           int threads) {
  for (int i = threadIdx.x; i < kVerifySegment / 32; i += threads) bits[i] = 0;
  __syncthreads();
  int s0;
  const int n = min(verify_rows(a, b, &s0), kVerifyRows);
  for (int i = node + 1 + threadIdx.x; i < n; i += threads) {
    const int up = a.parents ? draft_parent(a.parents[s0 + i], i) : i - 1;
    const int64_t x = a.tokens[s0 + i] - e0;
    if (up == node && x >= 0 && x < kVerifySegment && x + e0 < a.V) atomicOr(&bits[x >> 5], 1u << (x & 31));
  }
  __syncthreads();
}

// T and p of the 8 elements from e on; `at` the first one's place in the segment
template <typename T>
__device__ __forceinline__ void load_left(const T* pr, const T* qr, int64_t e, int64_t V, double off,
                                          const uint32_t* bits, int at, double* t, float* p) {
  float q[8];
  if (e + 8 <= V) {
    const Elements<T, 8> x = *(const Elements<T, 8>*)(pr + e);
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = mass(x.v[i]);
    if (qr) {
      const Elements<T, 8> y = *(const Elements<T, 8>*)(qr + e);
#pragma unroll
      for (int i = 0; i < 8; ++i) q[i] = mass(y.v[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      p[i] = e + i < V ? mass(pr[e + i]) : 0.f;
      if (qr) q[i] = e + i < V ? mass(qr[e + i]) : 0.f;
    }
  }
  if (qr) {
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = left_of(p[i], q[i], off);
  } else {
    const uint32_t gone = bits[at >> 5] >> (at & 31);
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = (gone >> i) & 1 ? 0.0 : (double)p[i];
  }
}

// Sums of T and p over a segment (blockIdx.x) of a request's last row.
template <typename T>
__global__ __launch_bounds__(kVerifySum) void verify_sum_kernel(VerifyArgs a) {
  __shared__ uint32_t bits[kVerifySegment / 32];
  __shared__ double red[2][kVerifySum / 64];
  const int b = blockIdx.y, tid = threadIdx.x;
  const VerifyEnd end = a.ends[b];
  if (end.row < 0) return;
  const int64_t e0 = (int64_t)blockIdx.x * kVerifySegment;
  const T* pr = (const T*)a.p + end.row * a.p_row;
  const T* qr = a.q ? (const T*)a.q + end.row * a.q_row : nullptr;
  if (!qr) taken_bits(a, b, end.node, e0, bits, kVerifySum);
  double st = 0.0, sp = 0.0;
#pragma unroll
  for (int r = 0; r < kVerifySegment / (kVerifySum * 8); ++r) {
    const int at = (r * kVerifySum + tid) * 8;
    if (e0 + at >= a.V) break;
    double t[8];
    float p[8];
    load_left(pr, qr, e0 + at, (int64_t)a.V, end.off, bits, at, t, p);
#pragma unroll
    for (int i = 0; i < 8; ++i) st += t[i], sp += (double)p[i];
  }
  st = wave_sum(st), sp = wave_sum(sp);
  if ((tid & 63) == 0) red[0][tid >> 6] = st, red[1][tid >> 6] = sp;
  __syncthreads();
  if (tid < 2) {
    double s = 0.0;
    for (int w = 0; w < kVerifySum / 64; ++w) s += red[tid][w];
    a.sums[((int64_t)b * a.segments + blockIdx.x) * 2 + tid] = s;
  }
}

// The thread whose share of a cumulative sum first passes t: every thread
// comes with its share `mine` and gets the sum before it.  Returns that thread,
// or where rounding leaves none the last one with a share, -1 without any.
// red: kVerifyPick / 64 doubles, found: an int
__device__ __forceinline__ int find_share(double mine, double t, double* red, int* found, double* before) {
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  double inc = mine;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const double x = __shfl_up(inc, m);
    if (lane >= m) inc += x;
  }
  __syncthreads();
  if (tid == 0) *found = 0x7fffffff;
  if (lane == 63) red[wv] = inc;
  __syncthreads();
  double base = 0.0;
  for (int w = 0; w < wv; ++w) base += red[w];
  // the sum before a thread is the sum up to the one in front of it, to the bit
  const double up = __shfl_up(inc, 1);
  *before = lane ? base + up : base;
  const bool pass = mine > 0.0 && base + inc > t;
  uint64_t hit = __ballot(pass);
  if (hit && lane == 0) atomicMin(found, wv * 64 + __builtin_ctzll(hit));
  __syncthreads();
  int at = *found;
  if (at == 0x7fffffff) {
    __syncthreads();
    if (tid == 0) *found = -1;
    __syncthreads();
    hit = __ballot(mine > 0.0);
    if (hit && lane == 0) atomicMax(found, wv * 64 + 63 - __builtin_clzll(hit));
    __syncthreads();
    at = *found;
  }
  return at;
}

// A block a request: the segment whose sum passes the draw, then the token.
template <typename T>
__global__ __launch_bounds__(kVerifyPick) void verify_pick_kernel(VerifyArgs a) {
  __shared__ uint32_t bits[kVerifySegment / 32];
  __shared__ double red[kVerifyPick / 64], pass_s;
  __shared__ int found, seg_s;
  __shared__ double total_s[2];
  const int b = blockIdx.x, tid = threadIdx.x;
  const VerifyEnd end = a.ends[b];
  if (end.row < 0) {
    if (tid == 0) a.next[b] = -1;
    return;
  }
  const double* sums = a.sums + (int64_t)b * a.segments * 2;
  const int per = (a.segments + kVerifyPick - 1) / kVerifyPick;
  const int g0 = min(tid * per, a.segments), g1 = min(g0 + per, a.segments);
  double mine[2] = {0.0, 0.0};
  for (int g = g0; g < g1; ++g) mine[0] += sums[2 * g], mine[1] += sums[2 * g + 1];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const double s = wave_sum(mine[k]);
    __syncthreads();
    if ((tid & 63) == 0) red[tid >> 6] = s;
    __syncthreads();
    if (tid == 0) {
      double all = 0.0;
      for (int w = 0; w < kVerifyPick / 64; ++w) all += red[w];
      total_s[k] = all;
    }
  }
  __syncthreads();
  // no mass left: from p itself, and without any of that no token
  const int k = total_s[0] > 0.0 ? 0 : 1;
  const double total = total_s[k];
  const float d = a.draws[b];
  const double t = (d > 0.f ? (double)d : 0.0) * total;
  double before;
  int at = find_share(mine[k], t, red, &found, &before);
  if (at < 0) {
    if (tid == 0) a.next[b] = -1;
    return;
  }
  if (tid == at) {
    int last = -1, g = g0;
    double sum = before, had = before;
    for (; g < g1; ++g) {
      const double s = sums[2 * g + k];
      if (s > 0.0) {
        last = g, had = sum;
        sum += s;
        if (sum > t) break;
      }
    }
    seg_s = last, pass_s = had;
  }
  __syncthreads();
  const int64_t e0 = (int64_t)seg_s * kVerifySegment;
  const double rest = t - pass_s;
  const bool plain = k == 1;
  const T* pr = (const T*)a.p + end.row * a.p_row;
  const T* qr = a.q ? (const T*)a.q + end.row * a.q_row : nullptr;
  if (!qr) taken_bits(a, b, end.node, e0, bits, kVerifyPick);
  double tt[8];
  float p[8];
  const int first = tid * 8;
  if (e0 + first < a.V) {
    load_left(pr, qr, e0 + first, (int64_t)a.V, end.off, bits, first, tt, p);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) tt[i] = 0.0, p[i] = 0.f;
  }
  double share = 0.0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (plain) tt[i] = (double)p[i];
    share += tt[i];
  }
  at = find_share(share, rest, red, &found, &before);
  if (tid == at) {
    double sum = before;
    int last = 0;
    bool done = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (!done && tt[i] > 0.0) {
        last = i;
        sum += tt[i];
        done = sum > rest;
      }
    }
    a.next[b] = e0 + first + last;
  }
}

template <typename T>
static int verify_launch(const VerifyArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((verify_walk_kernel<T>), dim3(a.B), dim3(kVerifyPick), 0, s, a);
  hipLaunchKernelGGL((verify_sum_kernel<T>), dim3(a.segments, a.B), dim3(kVerifySum), 0, s, a);
  hipLaunchKernelGGL((verify_pick_kernel<T>), dim3(a.B), dim3(kVerifyPick), 0, s, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? HTREE_OK : (int)e;
}

static int verify_segments(int32_t V) { return (int)(((int64_t)V + kVerifySegment - 1) / kVerifySegment); }

}  // namespace htree

using namespace htree;

extern "C" int htree_verify_drafts_workspace_bytes(int32_t B, int32_t V, int64_t* bytes) {
  if (!bytes) return HTREE_ENULL;
  if (B < 0 || V < 1) return HTREE_ESHAPE;
  if (B > kCacheMaxRequests) return HTREE_EUNSUPPORTED;
  *bytes = (int64_t)B * ((int64_t)sizeof(VerifyEnd) + verify_segments(V) * 16ll);
  return HTREE_OK;
}

extern "C" int htree_verify_drafts(int32_t dtype, int32_t B, int32_t rows, int32_t V, const void* target_probs,
                                   int64_t target_row, const void* draft_probs, int64_t draft_row,
                                   const int64_t* tokens, const int32_t* starts, const int32_t* parents,
                                   const float* uniforms, const float* draws, int32_t* kept, int32_t* path,
                                   int64_t* next_tokens, void* workspace, int64_t workspace_bytes, void* stream) {
  int64_t need = 0;
  const int rc = htree_verify_drafts_workspace_bytes(B, V, &need);
  if (rc) return rc;
  if (dtype != HTREE_F32 && dtype != HTREE_BF16 && dtype != HTREE_F16) return HTREE_ESHAPE;
  if (rows < 0 || target_row < 0 || draft_row < 0) return HTREE_ESHAPE;
  if (B == 0) return HTREE_OK;
  if (!starts || !draws || !kept || !next_tokens || !workspace) return HTREE_ENULL;
  if (rows && (!target_probs || !tokens || !uniforms || !path)) return HTREE_ENULL;
  if (off16(workspace)) return HTREE_EUNSUPPORTED;
  if (workspace_bytes < need) return HTREE_EWORKSPACE;
  const int es = dtype == HTREE_F32 ? 4 : 2;
  const Range in[7] = {{target_probs, rows ? ((rows - 1) * target_row + V) * es : 0},
                       {draft_probs, rows && draft_probs ? ((rows - 1) * draft_row + V) * es : 0},
                       {tokens, rows * 8ll}, {starts, (B + 1) * 4ll}, {parents, parents ? rows * 4ll : 0},
                       {uniforms, rows * 4ll}, {draws, B * 4ll}};
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
  a.ends = (VerifyEnd*)workspace;
  a.sums = (double*)(a.ends + B);
  a.p_row = target_row, a.q_row = draft_row;
  a.B = B, a.rows = rows, a.V = V, a.segments = verify_segments(V);
  hipStream_t s = (hipStream_t)stream;
  if (dtype == HTREE_F32) return verify_launch<float>(a, s);
  if (dtype == HTREE_BF16) return verify_launch<__bf16>(a, s);
  return verify_launch<_Float16>(a, s);
}
