// Index arithmetic of the paged cache's kernels (htree_cache.hip,
// htree_draft.h): how an attention call is split into units, which rows,
// tokens and pages a unit touches, which states a piece of the join reads, and
// which pages a request's new tokens get.  Lengths, tables and lists are device
// data that no host checks: the host replays over ordinary and damaged ones
// (tests/cache_replay_check.cpp, tests/cache_units_check.cpp) run these same
// functions.  The kernels alone have the sums over lanes, and the rows' slots
// and positions.
#ifndef HTREE_CACHE_INDEX_H_
#define HTREE_CACHE_INDEX_H_

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace htree {

// Requests of a call, of the page tables and of the attention.  Every block
// sums the lengths of all of them, 64 at a time, so a call's time grows with
// the square: 4096 single tokens over 64 tokens each take 360 us, where their
// bytes take 28; 65536 took 77 ms.
constexpr int kCacheMaxRequests = 4096;

// ------------------------------------------------------- attention's split
// A block's form.  NW = 1: four waves with the same 16 MT rows and tiles of
// their own (few rows); NW = 4: four waves with 16 MT rows each and common
// tiles.
//
// Tokens of a tile: of a wave's own, 8 KB of keys and 8 KB of values (16 KB
// each for fp32 at D 256), the loads that it has in flight while it computes;
// of a block's, twice that.
__host__ __device__ constexpr int draft_tile(int D, int es, int NW = 1) {
  const int n = (NW > 1 ? 16384 : 8192) / (D * es);
  return n > 64 ? 64 : n < 16 ? 16 : n;
}

// whether two blocks of the form with NW = 1 fit a CU (256 registers a lane)
__host__ __device__ constexpr bool draft_two(int D, int MT, int es) {
  return es == 2 ? D * MT <= 128 : D * MT <= 64 || (MT == 1 && D <= 128);
}

// A call's split.  Units: blocks of the launch, R rows of a request and KV
// head each.  Joins: blocks of the second launch, which joins the units of the
// same rows and takes as many rounds as there are rows.
struct DraftPlan {
  int D, MT, NW, R;
  int near;    // groups of rows of a request, on average
  int target;  // units to split into (0: one unit per group of rows)
  bool one_round;  // every piece of the join has a block of its own
  int64_t units, joins, slots, bytes;  // at most
};
__host__ __device__ inline DraftPlan draft_plan(int Dk, int Dv, int es, int B, int rows, int H, int Hkv,
                                                int width, int page_size) {
  DraftPlan p;
  const int m = Dk > Dv ? Dk : Dv;
  p.D = m <= 32 ? 32 : m <= 64 ? 64 : m <= 128 ? 128 : 256;
  const int G = H / Hkv;
  const int64_t per = ((int64_t)rows * G + B - 1) / B;  // rows of a request, on average
  // Blocks of 16 or 32 rows of the first form, or, above 32 rows a request and
  // in 16 bits, of 128 rows of the second.  Requests of 16384 tokens, 4 KV
  // heads, bf16, 64 rows a request: 32 of them at D 128 take 200 us in blocks
  // of 64 rows of the first form and 157 us in the second, 16 at D 64 51.8 and
  // 42 us, 16 at D 32 49.7 and 48.8 us.  At 32 rows and D 128 it is 173 and
  // 148 us, but 16 requests of 1000 tokens take 21.7 and 34.2 us.
  p.MT = per <= 16 ? 1 : 2;
  p.NW = per > 32 && es == 2 ? 4 : 1;
  p.R = 16 * p.MT * p.NW;
  const int64_t rts = ((int64_t)rows * G / p.R + B) * Hkv;
  // blocks that fit the GPU at once
  const int full = (p.NW > 1 ? p.D <= 128 : draft_two(p.D, p.MT, es)) ? 512 : 256;
  p.target = (int64_t)width * page_size <= 1024 ? 0 : full;
  p.near = (int)((per + p.R - 1) / p.R);
  p.near = p.near > 64 ? 64 : p.near;
  p.units = (rts + p.target + 8 * p.near - 1) / (8 * p.near) * (8 * p.near);
  // a group of rows makes R pieces of joining at most; beyond a round, as many
  // blocks as the GPU holds at once (16 trees over 32k: 1024 of them 139.8 us,
  // 2048 138.4 us)
  p.one_round = rts * p.R <= 1024;
  p.joins = p.target == 0 ? 0 : p.one_round ? rts * p.R : 2048;
  // a split request has at most twice the chunks its tokens fill
  p.slots = 2 * (int64_t)p.target;
  p.bytes = p.target == 0 ? 0 : p.slots * p.R * (p.D + 2) * 4 + 16;
  return p;
}

// The unit of block x: of 8 near blocks in a row, those 8 apart take `near`
// units in a row.
__host__ __device__ inline int64_t draft_near(int64_t x, int near) {
  const int64_t all = 8 * (int64_t)near, y = x % all;
  return x - y + y % 8 * near + y / 8;
}

// A request's lengths, held to what the buffers have
struct DraftReq {
  int s0, n;  // first row, rows (new tokens)
  int len;    // tokens
  int ctx;    // tokens before the new ones; negative: the first rows see nothing
};
__host__ __device__ inline DraftReq draft_req(int start, int end, int len, int rows) {
  DraftReq r;
  r.s0 = start < 0 ? 0 : start > rows ? rows : start;
  r.n = (end < r.s0 ? r.s0 : end > rows ? rows : end) - r.s0;
  r.len = len < 0 ? 0 : len;
  r.ctx = r.len - r.n;
  return r;
}

// tiles of a request; cap: tokens its table holds (at most 2^30)
__host__ __device__ inline int draft_tiles(const DraftReq& r, int cap, int KT) {
  return ((r.len < cap ? r.len : cap) + KT - 1) / KT;
}
// groups of rows of a request (and KV head)
__host__ __device__ inline int draft_row_groups(const DraftReq& r, int G, int R) {
  return (int)((r.n * (int64_t)G + R - 1) / R);
}
// Rows of each of them: even parts of the request's, in whole 16 MT of a wave
// (`step`), so that no group is left with a few rows and the time of a full one.
__host__ __device__ inline int draft_even(const DraftReq& r, int G, int R, int step) {
  const int n = r.n * G, groups = draft_row_groups(r, G, R);
  return groups <= 1 ? R : ((n + groups - 1) / groups + step - 1) / step * step;
}
// Pieces of work of a request: groups of rows times pieces of each.  A call
// has at most 2^24 (kDraftMaxUnits); damaged lengths that claim more are cut
// there, so that a wave's sums stay in 32 bits.
constexpr int kDraftMaxUnits = 1 << 24;
__host__ __device__ inline int draft_pieces(int each, int groups) {
  const int64_t n = (int64_t)each * groups;
  return n < kDraftMaxUnits ? (int)n : kDraftMaxUnits;
}
// Tiles of all groups of rows of the requests that a lane sums: lane, lane +
// 64, ...
template <typename F>
__host__ __device__ inline float draft_lane_tiles(int lane, int B, int cap, int KT, int G, int R, F req) {
  float w = 0.f;
  for (int b = lane; b < B; b += 64) {
    const DraftReq r = req(b);
    w += (float)draft_tiles(r, cap, KT) * draft_row_groups(r, G, R);
  }
  return w;
}
// Tiles of a chunk, from the tiles of all groups of rows: an fp32 sum of 64
// terms a lane at most and of 64 lanes, rounded fewer than 100 times on the way
// of any term (100 x 2^-24 is 6e-6), and raised by more than that: the workspace
// is sized for the exact one.  The same for every request, a multiple of the
// block's 4 waves, and so one tile a wave at least.  (A wider chunk and a
// request's even parts are no such multiples.)
__host__ __device__ inline int draft_chunk(float tiles, int target) {
  if (target <= 0) return 1 << 30;
  const float c = tiles * 1.0001f / target;
  return c > (float)(1 << 29) ? 1 << 30 : ((int)c + 4) / 4 * 4;
}
__host__ __device__ inline int draft_wider(int chunk) { return chunk + chunk / 16 + 1; }
// A chunk somewhat larger, where the units(chunk) of the call then all fit the
// GPU at once: else the last few of them start when the others are done.
template <typename F>
__host__ __device__ inline int draft_widen(int chunk, int target, F units) {
  int c = chunk;
  for (int i = 0; i < 4; ++i) {
    if (units(c) <= (float)target) return c;
    c = draft_wider(c);
  }
  return chunk;
}
// chunks of a request, and tiles of each: even parts
__host__ __device__ inline int draft_chunks(int tiles, int chunk) {
  const int n = (int)(((int64_t)tiles + chunk - 1) / chunk);
  return n < 1 ? 1 : n;
}

__host__ __device__ inline int draft_part(int tiles, int chunks) {
  const int n = (tiles + chunks - 1) / chunks;
  return n < 1 ? 1 : n;
}

// Where a block's work is.  The requests whose tokens make more than one chunk
// get workspace slots, one per unit.
struct DraftUnit {
  int b, nch;
  int chunk;   // tiles of each chunk
  int slot;    // of the request's first unit
  int index;   // of the work within the request
  int groups;  // of rows, of one KV head
};
// What a request has of a call's work, where each group of rows of a request
// of `nch` chunks makes per(nch) pieces.
struct DraftShare {
  int nch, tiles;
  int groups;  // of rows, of all KV heads
  int pieces, slots;
};
template <typename F>
__host__ __device__ inline DraftShare draft_share(const DraftReq& r, int cap, int KT, int G, int R, int Hkv,
                                                  int chunk, F per) {
  DraftShare s;
  s.tiles = draft_tiles(r, cap, KT);
  s.nch = draft_chunks(s.tiles, chunk);
  s.groups = draft_row_groups(r, G, R) * Hkv;
  s.pieces = draft_pieces(per(s.nch), s.groups);
  s.slots = draft_pieces(s.nch > 1 ? s.nch : 0, s.groups);
  return s;
}
// the work of request b's share that is `index` pieces into it, `slot` the
// first of the request's slots
__host__ __device__ inline DraftUnit draft_pick(int b, int nch, int tiles, int groups, int64_t slot,
                                                int64_t index, int Hkv) {
  return DraftUnit{b, nch, draft_part(tiles, nch), (int)slot, (int)index, groups / Hkv};
}

// A unit: group of rows rt (fastest), KV head h, chunk ch of a request.  The
// groups of rows of one head and chunk read the same tokens: `near` units in a
// row go to blocks of one of the 8 dies (block x runs on die x % 8), whose L2
// then serves all but the first.
struct DraftPart {
  int h, rt, ch;
  int slot;  // -1: the request has one chunk
};
__host__ __device__ inline DraftPart draft_unit_part(const DraftUnit& u, int Hkv) {
  const uint32_t rest = (uint32_t)u.index / (uint32_t)u.groups;
  DraftPart p;
  p.rt = (int)(u.index - rest * u.groups);
  p.ch = (int)(rest / (uint32_t)Hkv);
  p.h = (int)(rest - p.ch * Hkv);
  p.slot = u.nch > 1 ? u.slot + u.index : -1;
  return p;
}

// A piece of the join: a row of a group of rows, its chunks shared by a
// block's sets, or, of requests of up to `most` chunks, a row for each of the
// `sets`.
__host__ __device__ inline int draft_join_pieces(int nch, int most, int R, int sets) {
  return nch <= 1 ? 0 : nch <= most ? (R + sets - 1) / sets : R;
}
struct DraftJoin {
  int h, rt;
  int r0, nrow;        // rows of the group, from .. to
  int row;             // the first row's place in the group
  bool serial;         // a row for each set
  int64_t base, step;  // slot of chunk c: base + c step
};
__host__ __device__ inline DraftJoin draft_join(const DraftUnit& u, const DraftReq& r, int G, int Hkv, int R,
                                                int step, int sets, int most) {
  DraftJoin j;
  j.serial = u.nch <= most;
  const int per = draft_join_pieces(u.nch, most, R, sets), sub = u.index % per, group = u.index / per;
  j.h = group / u.groups, j.rt = group % u.groups;
  const int even = draft_even(r, G, R, step), end = r.n * G;
  j.r0 = j.rt * even;
  j.nrow = end < j.r0 + even ? end : j.r0 + even;
  j.row = j.serial ? sub * sets : sub;
  j.base = u.slot + group, j.step = (int64_t)u.groups * Hkv;
  return j;
}

// What a unit's rows see: tokens [0, kend), tiles [t0, t1) in its chunk
struct DraftSpan {
  int kend, t0, t1;
};
// (rows row0 .. row0 + R - 1 of it)
__host__ __device__ inline DraftSpan draft_span(const DraftReq& r, int64_t row0, int R, int G, int cap,
                                                int KT, int ch, int chunk) {
  const int64_t nrow = (int64_t)r.n * G, last = (row0 + R < nrow ? row0 + R : nrow) - 1;
  DraftSpan s;
  const int64_t k = (int64_t)r.ctx + last / G + 1;
  s.kend = (int)(k < 0 ? 0 : k > cap ? cap : k);
  const int64_t t0 = (int64_t)ch * chunk, tn = (s.kend + KT - 1) / KT;
  s.t0 = (int)(t0 < tn ? t0 : tn);
  s.t1 = (int)(t0 + chunk < tn ? t0 + chunk : tn);
  return s;
}

// a table entry as a page of the cache, or -1
__host__ __device__ inline int cache_page(int entry, int num_pages) {
  return entry >= 0 && entry < num_pages ? entry : -1;
}

// the token drafted before token j of a request, -1: none
__host__ __device__ inline int draft_parent(int p, int j) { return p >= 0 && p < j ? p : -1; }

// ------------------------------------------------------------ page tables
// pages of n tokens
__host__ __device__ inline int64_t table_pages(int64_t tokens, int shift) {
  return (tokens + (((int64_t)1 << shift) - 1)) >> shift;
}

// last b with s[b] <= x (s ascending, s[0] = 0, x >= 0); B >= 1
__host__ __device__ inline int table_find(const int32_t* s, int B, int x) {
  int lo = 0, hi = B;  // s[lo] <= x, and s[hi] > x or hi == B
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (s[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

}  // namespace htree
#endif  // HTREE_CACHE_INDEX_H_
