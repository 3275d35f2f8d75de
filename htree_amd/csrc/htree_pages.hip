// Pages of a paged key/value cache after a step: accepted drafts moved
// together, requests forked, pages copied, and the pages found that no
// request holds.
#include "htree_cache_host.h"
#include "htree_cache_index.h"
#include "htree_cache_scan.h"
#include "htree_common.h"
#include "htree_layers.h"

namespace htree {

// ----------------------------------------------------------- moving tokens
constexpr int kMoveMost = (1 << 24) - 1;  // blocks of 256 threads along a grid's first dimension
constexpr int kMoveLayers = 64;  // layers of a launch: their pointers are its arguments
// Layers and tokens that a thread reads before it writes the first.  Kept drafts
// are few tokens of many layers, and to find them takes four loads one after
// another: four layers at once 39.6 us for 256 requests and 32 layers, one 47.8.
// Pages are many tokens, found at once: 65 of them, 504 tokens in 16 layers, one
// layer a block 8.5 us, four 8.9; in a list of 256 whose other entries copy
// nothing 12.9 and 12.5.
constexpr int kKeepLayers = 4, kKeepTokens = 4;
constexpr int kCopyLayers = 1, kCopyTokens = 4;

struct MoveArgs {
  char *k[kMoveLayers], *v[kMoveLayers];
  int64_t k_page, k_token, k_head, v_page, v_token, v_head;  // bytes
  int32_t k_pieces, v_pieces;    // 16-byte pieces of a head
  int32_t pieces, k_all;         // of a token, and those of its keys
  int32_t page_shift, num_pages;
  int32_t layers, by;            // of the launch, of a block (blockIdx.y)
};

struct KeepArgs {
  MoveArgs m;
  const int64_t* slots;
  const int32_t *starts, *path, *kept;
  int32_t rows;
};

struct CopyArgs {
  MoveArgs m;
  const int32_t *from, *to, *tokens;
  int32_t columns, parts;  // pieces that a block takes, blocks that share a page's tokens
};

// The column of a token's bytes that a thread owns: one 16-byte piece of a
// head, in the keys' caches or the values'.
struct MoveColumn {
  bool keys;
  int64_t at, page, token;
};
__device__ __forceinline__ MoveColumn move_column(const MoveArgs& m, int piece) {
  MoveColumn c;
  c.keys = piece < m.k_all;
  if (!c.keys) piece -= m.k_all;
  const int per = c.keys ? m.k_pieces : m.v_pieces, h = piece / per;
  c.at = h * (c.keys ? m.k_head : m.v_head) + (int64_t)(piece - h * per) * 16;
  c.page = c.keys ? m.k_page : m.v_page, c.token = c.keys ? m.k_token : m.v_token;
  return c;
}

// The column's pieces of some tokens (from / to: bytes from a layer's base,
// to < 0: read, not written) in the block's layers: all tokens of kLayers layers
// are read before the first of them is written.
template <int kLayers, int kTokens>
__device__ __forceinline__ void move_tokens(const MoveArgs& m, const MoveColumn& c, const int64_t* from,
                                            const int64_t* to) {
  const int l1 = min((int)(blockIdx.y + 1) * m.by, m.layers);
  for (int l0 = blockIdx.y * m.by; l0 < l1; l0 += kLayers) {
    char* base[kLayers];
    f32x4 x[kLayers][kTokens] = {};
#pragma unroll
    for (int l = 0; l < kLayers; ++l) {
      const int at = min(l0 + l, l1 - 1);
      base[l] = c.keys ? m.k[at] : m.v[at];
    }
#pragma unroll
    for (int l = 0; l < kLayers; ++l) {
      if (l0 + l >= l1) break;
#pragma unroll
      for (int i = 0; i < kTokens; ++i) x[l][i] = *(const f32x4*)(base[l] + from[i]);
    }
    // one wait for all that was read: where the stores are conditional the
    // compiler would wait at each, for the stores before it too
#pragma unroll
    for (int l = 0; l < kLayers; ++l)
#pragma unroll
      for (int i = 0; i < kTokens; ++i) asm volatile("" : "+v"(x[l][i]));
#pragma unroll
    for (int l = 0; l < kLayers; ++l) {
      if (l0 + l >= l1) break;
#pragma unroll
      for (int i = 0; i < kTokens; ++i)
        if (to[i] >= 0) *(f32x4*)(base[l] + to[i]) = x[l][i];
    }
  }
}

// Accepted drafts to the front of their request's new tokens: token j comes
// from path[j] >= j.  A thread owns a piece of every token of its request, so
// that the order in which tokens are read and written is its own: four are
// read before the first of them is written, later ones come from places behind
// all that were written.  Bound by the chain start -> path -> slot -> token and
// by memory: 16 requests, one layer 3.9 us; 256 requests, 32 layers of 8 x 128
// bf16 39 us (162 MB, 4.1 TB/s).
__global__ __launch_bounds__(256) void keep_drafts_kernel(KeepArgs a) {
  const int piece = blockIdx.z * blockDim.x + threadIdx.x, b = blockIdx.x;
  if (piece >= a.m.pieces) return;
  const int s0 = min(max(a.starts[b], 0), a.rows), s1 = min(max(a.starts[b + 1], s0), a.rows);
  const int n = s1 - s0, kept = min(a.kept[b], n);
  const MoveColumn c = move_column(a.m, piece);
  const int64_t slots = (int64_t)a.m.num_pages << a.m.page_shift;
  const int64_t mask = ((int64_t)1 << a.m.page_shift) - 1;
  for (uint32_t j0 = 0; j0 < (uint32_t)max(kept, 0); j0 += kKeepTokens) {
    int64_t from[kKeepTokens], to[kKeepTokens];
    bool any = false;
#pragma unroll
    for (int i = 0; i < kKeepTokens; ++i) {
      const int j = (int)j0 + i;
      from[i] = c.at, to[i] = -1;
      if (j >= kept) continue;
      const int p = a.path[s0 + j];
      if (p <= j || p >= n) continue;  // in its place already, or damaged
      const int64_t s = a.slots[s0 + p], d = a.slots[s0 + j];
      if (s < 0 || s >= slots || d < 0 || d >= slots) continue;
      from[i] = c.at + (s >> a.m.page_shift) * c.page + (s & mask) * c.token;
      to[i] = c.at + (d >> a.m.page_shift) * c.page + (d & mask) * c.token;
      any = true;
    }
    if (any) move_tokens<kKeepLayers, kKeepTokens>(a.m, c, from, to);
  }
}

// The first tokens[i] tokens of page from[i] to page to[i]: 65 pages, 504 tokens
// together, in 16 layers of 4 x 128 bf16 8.5 us (33 MB, 3.9 TB/s).  Entries that
// copy nothing have blocks as well: 191 of them in the same list and it takes
// 12.9, 256 of them alone 3.4.  A page to seven others, 16 layers 4.6 us, a launch
// and two loads one after the other.
__global__ __launch_bounds__(256) void copy_pages_kernel(CopyArgs a) {
  const int i = blockIdx.x;
  const int from = cache_page(a.from[i], a.m.num_pages), to = cache_page(a.to[i], a.m.num_pages);
  if (from < 0 || to < 0 || from == to) return;
  const int size = 1 << a.m.page_shift;
  const int n = a.tokens ? min(a.tokens[i], size) : size;
  const int col = threadIdx.x % a.columns, step = 256 / a.columns;
  const int group = blockIdx.z / a.parts, part = blockIdx.z - group * a.parts, piece = group * a.columns + col;
  if (piece >= a.m.pieces || (int)threadIdx.x >= step * a.columns) return;
  const MoveColumn c = move_column(a.m, piece);
  for (int t0 = part * kCopyTokens * step + threadIdx.x / a.columns; t0 < n; t0 += a.parts * kCopyTokens * step) {
    int64_t src[kCopyTokens], dst[kCopyTokens];
#pragma unroll
    for (int u = 0; u < kCopyTokens; ++u) {
      const int t = t0 + u * step;
      src[u] = c.at + from * c.page + min(t, n - 1) * c.token;
      dst[u] = t < n ? c.at + to * c.page + t * c.token : -1;
    }
    move_tokens<kCopyLayers, kCopyTokens>(a.m, c, src, dst);
  }
}

// ----------------------------------------------------------------- forking
struct ForkArgs {
  const int32_t *table, *lens, *source, *free_pages;
  int32_t *out_table, *out_lens, *from, *to, *tokens, *used;
  int64_t table_stride, out_stride;
  int32_t B, N, width, page_shift, num_pages, n_free;
};

// New requests blockIdx.x, + gridDim.x ..: their rows of the table.  Each block
// finds the first child of every request and sums the fresh pages over all new
// ones itself, which is less than a second launch: 4.2 us for 8 new requests,
// 5.3 for 256 out of 256.
__global__ __launch_bounds__(256) void fork_requests_kernel(ForkArgs a) {
  extern __shared__ int32_t fork_lds[];
  __shared__ int64_t red[4];
  int32_t* first = fork_lds;        // [B] the first child of a request
  int32_t* fresh = fork_lds + a.B;  // [N + 1] fresh pages of the new requests before
  const int tid = threadIdx.x;
  const int mask = (1 << a.page_shift) - 1;
  for (int b = tid; b < a.B; b += 256) first[b] = 0x7fffffff;
  __syncthreads();
  for (int i = tid; i < a.N; i += 256) {
    const int s = a.source[i];
    if (s >= 0 && s < a.B) atomicMin(&first[s], i);
  }
  __syncthreads();
  // a fresh page: a partly filled last page that an earlier child holds on to
  auto wants = [&](int i) -> int64_t {
    const int s = a.source[i];
    if (s < 0 || s >= a.B || first[s] == i) return 0;
    const int len = max(a.lens[s], 0);
    return (len & mask) != 0 && (len >> a.page_shift) < a.width;
  };
  const int64_t need = tab_scan(a.N, 0x7fffffff, fresh, red, wants);
  if (blockIdx.x == 0 && tid == 0) a.used[0] = (int32_t)need;
  for (int i = blockIdx.x; i < a.N; i += gridDim.x) {
    int s = a.source[i];
    if (s < 0 || s >= a.B) s = -1;
    const int len = s < 0 ? 0 : max(a.lens[s], 0), full = len >> a.page_shift;
    const int64_t live = min(table_pages(len, a.page_shift), (int64_t)a.width);
    const bool own = fresh[i + 1] > fresh[i];
    const int page = own && fresh[i] < a.n_free ? cache_page(a.free_pages[fresh[i]], a.num_pages) : -1;
    const int32_t* row = a.table + (int64_t)s * a.table_stride;
    for (uint32_t j = tid; j < (uint32_t)a.width; j += 256)  // (a width below 2^31 and 256 pass it)
      a.out_table[(int64_t)i * a.out_stride + j] = j >= live ? -1 : own && (int)j == full ? page : row[j];
    if (tid == 0) {
      a.out_lens[i] = len;
      const int old = own ? cache_page(row[full], a.num_pages) : -1;
      const bool copies = page >= 0 && old >= 0;
      a.from[i] = copies ? old : -1;
      a.to[i] = copies ? page : -1;
      a.tokens[i] = copies ? len & mask : 0;
    }
  }
}

// ------------------------------------------------------------ unused pages
struct UnusedArgs {
  const int32_t *table, *lens, *held;
  uint8_t* flags;   // [tiles * kUnusedTile] 1: held
  int32_t* counts;  // [tiles] unused pages of a tile, nullptr: each block counts
  int32_t *pages, *count;
  int64_t table_stride;
  int32_t B, width, page_shift, num_pages, n_held, tiles;
};
constexpr int kUnusedTile = 4096;        // pages a block counts or lists: 16 a thread
// Tiles that every block counts for itself: a call of 5 of them 9.3 us in a graph
// (10.6 with a launch that counts), 28 12.2 (11.3), 53 14.5 (11.8); the launch
// takes 3 us of the host's time, which bounds such calls outside a graph.
constexpr int kUnusedCounted = 32;
constexpr int kUnusedPiece = 256;        // entries of a row that a wave reads at once, 4 a lane,
// of so many rows: four in the one launch (64 requests of 1024 entries 13.1 us, with
// two 13.5; 256 of 250 13.8 and 14.7), two in unused_mark_kernel (the call's launches
// together, 512 requests of 256 11.8 us, with four 12.7; 300 of 63 9.3 and 10.0)
constexpr int kUnusedPieces = 4, kUnusedMark = 2;
// Calls in one launch: pieces, requests and held pages at most, and pages, whose
// bits fill 32 KB of LDS.  A call, and in brackets the other form's, three launches
// at these sizes: outside a graph, where those are bound by the host, up to 128
// pieces 9.2 to 9.5 us (15.5), 192 10.9 to 11.5 (15.5), 256 12.9 to 14.2 (15.4 to
// 18.1); in a graph 32 pieces 6.7 (9.4), 64 7.1 (9.5), 128 8.9 to 9.5 (9.6), 192
// 10.9 to 11.7 (10.2), 256 13.0 to 14.4 (9.2 to 12.0).  The limit is for calls
// outside one.
constexpr int kUnusedSmall = 256, kUnusedSmallRows = 256, kUnusedSmallHeld = 4096;
constexpr int kUnusedSmallPages = 1 << 18;
constexpr int kUnusedSmallTile = 8192;   // pages a block lists: 8 a thread

struct __attribute__((packed, aligned(4))) Entries {
  int32_t v[4];
};

__device__ __forceinline__ int live_pages(const UnusedArgs& a, int len) {
  return (int)min(table_pages(max(len, 0), a.page_shift), (int64_t)a.width);
}

// N pieces of the table, from piece p0 on: piece p is the (p / B)-th 256
// entries of request p % B, so that first pieces, which have most of the live
// entries, come first.  Reads that would pass a row's end start earlier; what the
// lanes in front have is not marked again, 64 lanes would wait for one word: of a
// lane's four entries those from `lo` to before `hi` count.  (Rows of less than
// four entries: one a lane.)
template <int N>
struct Pieces {
  Entries x[N];
  int lo[N], hi[N];
  bool live[N];  // any of the piece
};
// (less than 2^31 of them)
__device__ __forceinline__ uint32_t piece_count(const UnusedArgs& a) {
  return ((uint32_t)a.width + kUnusedPiece - 1) / kUnusedPiece * a.B;
}
// length(b): of request b.  False, and nothing is read, if none of them is live.
template <int N, typename L>
__device__ __forceinline__ bool load_pieces(const UnusedArgs& a, uint32_t p0, L length, Pieces<N>* c) {
  const int lane = threadIdx.x & 63;
  const uint32_t all = piece_count(a);
  uint32_t q = p0 / (uint32_t)a.B, b = p0 - q * a.B;
  const int32_t* row[N];
  int first[N], live[N];
  bool any = false;
#pragma unroll
  for (int u = 0; u < N; ++u) {
    row[u] = a.table + (int64_t)b * a.table_stride;
    first[u] = (int)q * kUnusedPiece;
    live[u] = p0 + u < all ? live_pages(a, length((int)b)) : 0;
    c->live[u] = live[u] > first[u];
    any |= c->live[u];
    // (past the last piece: that one again)
    if (p0 + u + 1 < all && ++b == (uint32_t)a.B) b = 0, ++q;
  }
  if (!any) return false;
#pragma unroll
  for (int u = 0; u < N; ++u) {
    if (a.width < 4) {
      c->x[u].v[0] = row[u][min(lane, a.width - 1)];
      c->lo[u] = 0, c->hi[u] = lane < live[u] ? 1 : 0;
    } else {
      const int mine = first[u] + lane * 4, at = min(mine, a.width - 4);
      c->x[u] = *(const Entries*)(row[u] + at);
      c->lo[u] = mine - at, c->hi[u] = live[u] - at;
    }
  }
  return true;
}
// f(page) for the pages that count
template <int N, typename F>
__device__ __forceinline__ void mark_pieces(const UnusedArgs& a, const Pieces<N>& c, F f) {
#pragma unroll
  for (int u = 0; u < N; ++u)
    if (c.live[u])
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e >= c.lo[u] && e < c.hi[u] && (uint32_t)c.x[u].v[e] < (uint32_t)a.num_pages)
          f(c.x[u].v[e]);
}

// sum over the block's threads, to all; `red` an int for each wave
template <int WAVES>
__device__ __forceinline__ int block_sum(int x, int* red) {
#pragma unroll
  for (int m = 32; m; m >>= 1) x += __shfl_xor(x, m);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
  __syncthreads();
  int all = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) all += red[w];
  return all;
}

// Lists a block's unused pages, bit i of `bits`: page p0 + i of the thread's N,
// from place `before` of the list on, and -1 in the block's places behind the
// last of `all`.  They go through LDS, so that places are written in order.
template <int WAVES, int N>
__device__ __forceinline__ void list_pages(const UnusedArgs& a, uint32_t bits, int before, int all, int32_t* buf,
                                           int* red) {
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const int64_t p0 = (int64_t)blockIdx.x * (WAVES * 64 * N);
  int inc = __popc(bits);
  const int mine = inc;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const int x = __shfl_up(inc, m);
    if (lane >= m) inc += x;
  }
  __syncthreads();
  if (lane == 63) red[wv] = inc;
  __syncthreads();
  int at = inc - mine, here = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    if (w < wv) at += red[w];
    here += red[w];
  }
  for (; bits; bits &= bits - 1) buf[at++] = (int)(p0 + tid * N + __builtin_ctz(bits));
  __syncthreads();
  for (int i = tid; i < here; i += WAVES * 64) a.pages[(int64_t)before + i] = buf[i];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int64_t p = p0 + i * (WAVES * 64) + tid;
    if (p >= all && p < a.num_pages) a.pages[p] = -1;
  }
  if (blockIdx.x == 0 && tid == 0) a.count[0] = all;
}

// A call in one launch: every block marks all pages that are held, in the bits
// of its LDS, and lists its own part of the others.  Bound by the marks, atomics
// on random words: 41600 live entries of 64 requests, 46620 pages 12.8 us.
__global__ __launch_bounds__(1024) void unused_small_kernel(UnusedArgs a) {
  extern __shared__ uint32_t small_bits[];  // 1: held; pages past the last one too
  __shared__ int32_t buf[kUnusedSmallTile], lens[kUnusedSmallRows];
  __shared__ int red[16];
  const int tid = threadIdx.x, wv = tid >> 6;
  const int words = a.tiles * (kUnusedSmallTile / 32);
  for (int i = tid; i < words; i += 1024) {
    const int left = a.num_pages - i * 32;
    small_bits[i] = left >= 32 ? 0u : left <= 0 ? ~0u : ~0u << left;
  }
  for (int i = tid; i < a.B; i += 1024) lens[i] = a.lens[i];
  __syncthreads();
  auto mark = [&](int page) { atomicOr(&small_bits[page >> 5], 1u << (page & 31)); };
  auto length = [&](int b) { return __builtin_amdgcn_readfirstlane(lens[b]); };
  const uint32_t pieces = piece_count(a);
  for (uint32_t p = __builtin_amdgcn_readfirstlane(wv) * kUnusedPieces; p < pieces; p += 16 * kUnusedPieces) {
    Pieces<kUnusedPieces> c;
    if (load_pieces(a, p, length, &c)) mark_pieces(a, c, mark);
  }
  for (int i = tid; i < a.n_held; i += 1024)
    if ((uint32_t)a.held[i] < (uint32_t)a.num_pages) mark(a.held[i]);
  __syncthreads();
  const int first = blockIdx.x * (kUnusedSmallTile / 32);
  int before = 0, all = 0;
  for (int i = tid; i < words; i += 1024) {
    const int n = 32 - __popc(small_bits[i]);
    all += n;
    if (i < first) before += n;
  }
  before = block_sum<16>(before, red);
  all = block_sum<16>(all, red);
  const uint32_t bits = ~(small_bits[first + tid / 4] >> (tid % 4 * 8)) & 255u;
  list_pages<16, 8>(a, bits, before, all, buf, red);
}

__global__ __launch_bounds__(256) void unused_clear_kernel(uint8_t* flags, int64_t n) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 16;
  if (i < n) *(uint4*)(flags + i) = make_uint4(0, 0, 0, 0);
}

// A wave two pieces of the table (spread over the dies as pieces are numbered: a
// die that had all the first ones took six times as long); the last blocks mark
// the held pages.  Whoever holds a page writes the same 1: no atomics.
// 1.3M entries, each a store to a line of its own, 12 us; all four launches 20.
__global__ __launch_bounds__(256) void unused_mark_kernel(UnusedArgs a) {
  const uint32_t pieces = piece_count(a), blocks = (pieces + 4 * kUnusedMark - 1) / (4 * kUnusedMark);
  if (blockIdx.x >= blocks) {
    const int64_t i = (int64_t)(blockIdx.x - blocks) * 256 + threadIdx.x;
    const int page = i < a.n_held ? cache_page(a.held[i], a.num_pages) : -1;
    if (page >= 0) a.flags[page] = 1;
    return;
  }
  const uint32_t p = (blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * kUnusedMark;
  if (p >= pieces) return;
  Pieces<kUnusedMark> c;
  if (load_pieces(a, p, [&](int b) { return a.lens[b]; }, &c))
    mark_pieces(a, c, [&](int page) { a.flags[page] = 1; });
}

// bit i: page p0 + i is unused
__device__ __forceinline__ uint32_t unused_bits(const UnusedArgs& a, int64_t p0) {
  const uint4 f = *(const uint4*)(a.flags + p0);
  const uint32_t w[4] = {f.x, f.y, f.z, f.w};
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (!((w[i / 4] >> (i % 4 * 8)) & 1) && p0 + i < a.num_pages) bits |= 1u << i;
  return bits;
}

__global__ __launch_bounds__(256) void unused_count_kernel(UnusedArgs a) {
  __shared__ int red[4];
  const int64_t p0 = (int64_t)blockIdx.x * kUnusedTile + threadIdx.x * 16;
  const int n = block_sum<4>(__popc(unused_bits(a, p0)), red);
  if (threadIdx.x == 0) a.counts[blockIdx.x] = n;
}

__global__ __launch_bounds__(256) void unused_list_kernel(UnusedArgs a) {
  __shared__ int32_t buf[kUnusedTile];
  __shared__ int red[4];
  const uint32_t bits = unused_bits(a, (int64_t)blockIdx.x * kUnusedTile + threadIdx.x * 16);
  int before = 0, all = 0;
  if (a.counts) {
    for (int t = threadIdx.x; t < a.tiles; t += 256) {
      const int n = a.counts[t];
      all += n;
      if (t < (int)blockIdx.x) before += n;
    }
  } else {
    // the held ones: their flags' bits, eight tiles in flight
    for (int t0 = 0; t0 < a.tiles; t0 += 8) {
      uint4 f[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        f[i] = *(const uint4*)(a.flags + (int64_t)min(t0 + i, a.tiles - 1) * kUnusedTile + threadIdx.x * 16);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int n = t0 + i < a.tiles ? __popc(f[i].x) + __popc(f[i].y) + __popc(f[i].z) + __popc(f[i].w) : 0;
        all -= n;
        if (t0 + i < (int)blockIdx.x) before -= n;
      }
    }
    if (threadIdx.x == 0) all += a.num_pages, before += (int)blockIdx.x * kUnusedTile;
  }
  before = block_sum<4>(before, red);
  all = block_sum<4>(all, red);
  list_pages<4, 16>(a, bits, before, all, buf, red);
}

// ------------------------------------------------------------------ host
// describes the cache's layers; 0 or an error
static int move_args(const htree_cache* c, int32_t layers, void* const* k, void* const* v, MoveArgs* m) {
  const int rc = cache_check(c);
  if (rc) return rc;
  if (layers < 0) return HTREE_ESHAPE;
  if (layers > 65535) return HTREE_EUNSUPPORTED;
  if (layers && (!k || !v)) return HTREE_ENULL;
  for (int l = 0; l < layers; ++l) {
    if (!k[l] || !v[l]) return HTREE_ENULL;
    if (off16(k[l]) || off16(v[l])) return HTREE_EUNSUPPORTED;
  }
  const int es = cache_es(c);
  m->k_page = c->k_page * es, m->k_token = c->k_token * es, m->k_head = c->k_head * es;
  m->v_page = c->v_page * es, m->v_token = c->v_token * es, m->v_head = c->v_head * es;
  m->k_pieces = c->Dk * es / 16, m->v_pieces = c->Dv * es / 16;
  const int64_t all = (int64_t)c->H_kv * (m->k_pieces + m->v_pieces);
  if (all > (1 << 19)) return HTREE_EUNSUPPORTED;  // a grid's last dimension
  m->pieces = (int32_t)all, m->k_all = c->H_kv * m->k_pieces;
  m->page_shift = log2i(c->page_size), m->num_pages = c->num_pages;
  return HTREE_OK;
}

// HTREE_EOVERLAP where a piece of a layer is another's too, or a list's: blocks
// would write what others read.
template <int N>
static int moves_apart(const htree_cache* c, const MoveArgs& m, int32_t layers, void* const* k, void* const* v,
                       const Range (&lists)[N]) {
  auto layer = [&](int64_t run, int64_t page, int64_t token, int64_t head) {
    Runs r;
    r.at = 0, r.run = run;
    r.add(c->num_pages, page), r.add(c->page_size, token), r.add(c->H_kv, head);
    return r;
  };
  return layers_apart(layer(m.k_pieces * 16, m.k_page, m.k_token, m.k_head),
                      layer(m.v_pieces * 16, m.v_page, m.v_token, m.v_head), layers, k, v, lists, N);
}

// runs f(blocks in y) for 64 layers at a time, `by` of them a block
template <typename F>
static int by_layers(int32_t layers, void* const* k, void* const* v, int by, MoveArgs* m, F f) {
  for (int l = 0; l < layers; l += kMoveLayers) {
    const int n = layers - l < kMoveLayers ? layers - l : kMoveLayers;
    for (int i = 0; i < n; ++i) m->k[i] = (char*)k[l + i], m->v[i] = (char*)v[l + i];
    m->layers = n, m->by = by;
    f((n + by - 1) / by);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
  }
  return HTREE_OK;
}

}  // namespace htree

using namespace htree;

extern "C" int htree_keep_drafts(const htree_cache* c, int32_t layers, void* const* k_layers, void* const* v_layers,
                                 int32_t B, int32_t rows, const int64_t* slots, const int32_t* starts,
                                 const int32_t* path, const int32_t* kept, void* stream) {
  KeepArgs a;
  const int rc = move_args(c, layers, k_layers, v_layers, &a.m);
  if (rc) return rc;
  if (B < 0 || rows < 0) return HTREE_ESHAPE;
  if (B > kCacheMaxRequests) return HTREE_EUNSUPPORTED;
  if (B == 0 || rows == 0 || layers == 0) return HTREE_OK;
  if (!slots || !starts || !path || !kept) return HTREE_ENULL;
  const Range lists[4] = {{slots, rows * 8ll}, {starts, (B + 1) * 4ll}, {path, rows * 4ll}, {kept, B * 4ll}};
  if (const int shared = moves_apart(c, a.m, layers, k_layers, v_layers, lists)) return shared;
  a.slots = slots, a.starts = starts, a.path = path, a.kept = kept, a.rows = rows;
  const unsigned threads = a.m.pieces >= 256 ? 256 : (a.m.pieces + 63) / 64 * 64;
  const unsigned z = (a.m.pieces + threads - 1) / threads;
  // a block for each layer until the GPU is full
  const int by = (int64_t)B * z * layers <= 1024 ? 1 : kKeepLayers;
  return by_layers(layers, k_layers, v_layers, by, &a.m, [&](int y) {
    hipLaunchKernelGGL(keep_drafts_kernel, dim3(B, y, z), dim3(threads), 0, (hipStream_t)stream, a);
  });
}

extern "C" int htree_copy_pages(const htree_cache* c, int32_t layers, void* const* k_layers, void* const* v_layers,
                                int32_t n, const int32_t* from, const int32_t* to, const int32_t* tokens,
                                void* stream) {
  CopyArgs a;
  const int rc = move_args(c, layers, k_layers, v_layers, &a.m);
  if (rc) return rc;
  if (n < 0) return HTREE_ESHAPE;
  if (n > kMoveMost) return HTREE_EUNSUPPORTED;
  if (n == 0 || layers == 0) return HTREE_OK;
  if (!from || !to) return HTREE_ENULL;
  const Range lists[3] = {{from, n * 4ll}, {to, n * 4ll}, {tokens, tokens ? n * 4ll : 0}};
  if (const int shared = moves_apart(c, a.m, layers, k_layers, v_layers, lists)) return shared;
  a.from = from, a.to = to, a.tokens = tokens;
  a.columns = a.m.pieces < 256 ? a.m.pieces : 256;
  // so many blocks that a thread reads its tokens at once, up to 16 a page
  const int once = kCopyTokens * (256 / a.columns), parts = (c->page_size + once - 1) / once;
  a.parts = parts < 16 ? parts : 16;
  const unsigned z = (a.m.pieces + a.columns - 1) / a.columns * a.parts;
  return by_layers(layers, k_layers, v_layers, kCopyLayers, &a.m, [&](int y) {
    hipLaunchKernelGGL(copy_pages_kernel, dim3(n, y, z), dim3(256), 0, (hipStream_t)stream, a);
  });
}

extern "C" int htree_fork_requests(int32_t B, int32_t N, int32_t page_size, int32_t num_pages, int32_t table_width,
                                   int64_t table_stride, int64_t out_stride, int32_t n_free,
                                   const int32_t* block_table, const int32_t* lens, const int32_t* source,
                                   const int32_t* free_pages, int32_t* out_table, int32_t* out_lens,
                                   int32_t* copy_from, int32_t* copy_to, int32_t* copy_tokens, int32_t* pages_used,
                                   void* stream) {
  if (B < 0 || N < 0 || num_pages < 0 || table_width < 0 || n_free < 0) return HTREE_ESHAPE;
  if ((B > 1 && table_stride < table_width) || (N > 1 && out_stride < table_width)) return HTREE_ESHAPE;
  if (page_size < 1 || (page_size & (page_size - 1)) || B > kCacheMaxRequests || N > kCacheMaxRequests)
    return HTREE_EUNSUPPORTED;
  if (N == 0) return HTREE_OK;
  if (!source || !out_lens || !copy_from || !copy_to || !copy_tokens || !pages_used) return HTREE_ENULL;
  if ((B && !lens) || (B && table_width && !block_table) || (table_width && !out_table) || (n_free && !free_pages))
    return HTREE_ENULL;
  const Range in[4] = {{block_table, B && table_width ? ((B - 1) * table_stride + table_width) * 4 : 0},
                       {lens, B * 4ll}, {source, N * 4ll}, {free_pages, n_free * 4ll}};
  const Range out[6] = {{out_table, table_width ? ((N - 1) * out_stride + table_width) * 4 : 0}, {out_lens, N * 4ll},
                        {copy_from, N * 4ll}, {copy_to, N * 4ll}, {copy_tokens, N * 4ll}, {pages_used, 4}};
  for (int i = 0; i < 6; ++i) {
    for (const Range& y : in)
      if (overlap(out[i], y)) return HTREE_EOVERLAP;
    for (int j = 0; j < i; ++j)
      if (overlap(out[i], out[j])) return HTREE_EOVERLAP;
  }
  ForkArgs a;
  a.table = block_table, a.lens = lens, a.source = source, a.free_pages = free_pages;
  a.out_table = out_table, a.out_lens = out_lens, a.from = copy_from, a.to = copy_to, a.tokens = copy_tokens;
  a.used = pages_used;
  a.table_stride = table_stride, a.out_stride = out_stride;
  a.B = B, a.N = N, a.width = table_width, a.page_shift = log2i(page_size), a.num_pages = num_pages;
  a.n_free = n_free;
  hipLaunchKernelGGL(fork_requests_kernel, dim3(N < 512 ? N : 512), dim3(256), (B + N + 1) * 4, (hipStream_t)stream, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? HTREE_OK : (int)e;
}

static int64_t unused_pieces(int32_t B, int32_t table_width) {
  return ((int64_t)table_width + kUnusedPiece - 1) / kUnusedPiece * B;
}
// whether a call runs in one launch
static bool unused_small(int32_t B, int32_t num_pages, int32_t table_width, int32_t n_held) {
  return num_pages <= kUnusedSmallPages && B <= kUnusedSmallRows && n_held <= kUnusedSmallHeld &&
         unused_pieces(B, table_width) <= kUnusedSmall;
}

extern "C" int htree_unused_pages_workspace_bytes(int32_t B, int32_t num_pages, int32_t table_width, int32_t n_held,
                                                  int64_t* bytes) {
  if (!bytes) return HTREE_ENULL;
  if (B < 0 || num_pages < 0 || table_width < 0 || n_held < 0) return HTREE_ESHAPE;
  const int64_t tiles = ((int64_t)num_pages + kUnusedTile - 1) / kUnusedTile;
  *bytes = unused_small(B, num_pages, table_width, n_held) ? 0 : tiles * (kUnusedTile + 4);
  return HTREE_OK;
}

extern "C" int htree_unused_pages(int32_t B, int32_t page_size, int32_t num_pages, int32_t table_width,
                                  int64_t table_stride, const int32_t* block_table, const int32_t* lens,
                                  int32_t n_held, const int32_t* held, int32_t* pages, int32_t* count,
                                  void* workspace, int64_t workspace_bytes, void* stream) {
  int64_t need = 0;
  const int rc = htree_unused_pages_workspace_bytes(B, num_pages, table_width, n_held, &need);
  if (rc) return rc;
  if (B > 1 && table_stride < table_width) return HTREE_ESHAPE;
  if (page_size < 1 || (page_size & (page_size - 1)) || B > kCacheMaxRequests) return HTREE_EUNSUPPORTED;
  if (num_pages == 0) return HTREE_OK;
  if (!pages || !count || (need && !workspace) || (n_held && !held) || (B && !lens) ||
      (B && table_width && !block_table))
    return HTREE_ENULL;
  if (off16(workspace)) return HTREE_EUNSUPPORTED;
  if (workspace_bytes < need) return HTREE_EWORKSPACE;
  const Range in[3] = {{block_table, B && table_width ? ((B - 1) * table_stride + table_width) * 4 : 0},
                       {lens, B * 4ll}, {held, n_held * 4ll}};
  const Range out[3] = {{pages, num_pages * 4ll}, {count, 4}, {workspace, need}};
  for (int i = 0; i < 3; ++i) {
    for (const Range& y : in)
      if (overlap(out[i], y)) return HTREE_EOVERLAP;
    for (int j = 0; j < i; ++j)
      if (overlap(out[i], out[j])) return HTREE_EOVERLAP;
  }
  UnusedArgs a;
  a.table = block_table, a.lens = lens, a.held = held;
  a.pages = pages, a.count = count;
  a.table_stride = table_stride;
  a.B = B, a.width = table_width, a.page_shift = log2i(page_size), a.num_pages = num_pages, a.n_held = n_held;
  hipStream_t s = (hipStream_t)stream;
  if (unused_small(B, num_pages, table_width, n_held)) {
    a.tiles = (num_pages + kUnusedSmallTile - 1) / kUnusedSmallTile;
    a.flags = nullptr, a.counts = nullptr;
    hipLaunchKernelGGL(unused_small_kernel, dim3(a.tiles), dim3(1024), a.tiles * (kUnusedSmallTile / 8), s, a);
  } else {
    a.tiles = (int)(((int64_t)num_pages + kUnusedTile - 1) / kUnusedTile);
    a.flags = (uint8_t*)workspace;
    a.counts = (int32_t*)(a.flags + (int64_t)a.tiles * kUnusedTile);
    const int64_t pieces = unused_pieces(B, table_width);
    const int64_t blocks = (pieces + 4 * kUnusedMark - 1) / (4 * kUnusedMark) + ((int64_t)n_held + 255) / 256;
    if (pieces >= 0x7fffff00 || blocks > kMoveMost) return HTREE_EUNSUPPORTED;
    hipLaunchKernelGGL(unused_clear_kernel, dim3(a.tiles), dim3(256), 0, s, a.flags, (int64_t)a.tiles * kUnusedTile);
    if (blocks) hipLaunchKernelGGL(unused_mark_kernel, dim3((unsigned)blocks), dim3(256), 0, s, a);
    // every block of few tiles counts their flags itself: a launch less
    if (a.tiles <= kUnusedCounted) a.counts = nullptr;
    else hipLaunchKernelGGL(unused_count_kernel, dim3(a.tiles), dim3(256), 0, s, a);
    hipLaunchKernelGGL(unused_list_kernel, dim3(a.tiles), dim3(256), 0, s, a);
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? HTREE_OK : (int)e;
}
