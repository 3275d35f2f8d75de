// Pages of a paged key/value cache after a step: accepted drafts moved
// together, requests forked, pages copied, and the pages found that no
// request holds.
#include "htree_cache_host.h"
#include "htree_cache_index.h"
#include "htree_cache_scan.h"
#include "htree_common.h"

namespace htree {

// ----------------------------------------------------------- moving tokens
constexpr int kMoveLayers = 64;  // layers of a launch: their pointers are its arguments
constexpr int kMoveUnroll = 8;   // tokens that a thread reads before it writes the first

struct MoveArgs {
  char *k[kMoveLayers], *v[kMoveLayers];
  int64_t k_page, k_token, k_head, v_page, v_token, v_head;  // bytes
  int32_t k_pieces, v_pieces;    // 16-byte pieces of a head
  int32_t pieces, k_all;         // of a token, and those of its keys
  int32_t page_shift, num_pages;
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
  int32_t n, columns;  // pieces that a block takes
};

// The column of a token's bytes that a thread owns: one 16-byte piece of a
// head, in the keys' cache or the values'.
struct MoveColumn {
  char* base;
  int64_t page, token;
};
__device__ __forceinline__ MoveColumn move_column(const MoveArgs& m, int layer, int piece) {
  MoveColumn c;
  if (piece < m.k_all) {
    const int h = piece / m.k_pieces;
    c.base = m.k[layer] + h * m.k_head + (int64_t)(piece - h * m.k_pieces) * 16;
    c.page = m.k_page, c.token = m.k_token;
  } else {
    piece -= m.k_all;
    const int h = piece / m.v_pieces;
    c.base = m.v[layer] + h * m.v_head + (int64_t)(piece - h * m.v_pieces) * 16;
    c.page = m.v_page, c.token = m.v_token;
  }
  return c;
}

// Accepted drafts to the front of their request's new tokens: token j comes
// from path[j] >= j.  A thread owns a piece of every token of its request, so
// that the order in which tokens are read and written is its own: eight are
// read before the first of them is written, later ones come from places behind
// all that were written.
__global__ __launch_bounds__(256) void keep_drafts_kernel(KeepArgs a) {
  const int piece = blockIdx.z * blockDim.x + threadIdx.x, b = blockIdx.x;
  if (piece >= a.m.pieces) return;
  const int s0 = min(max(a.starts[b], 0), a.rows), s1 = min(max(a.starts[b + 1], s0), a.rows);
  const int n = s1 - s0, kept = min(a.kept[b], n);
  const MoveColumn c = move_column(a.m, blockIdx.y, piece);
  const int64_t slots = (int64_t)a.m.num_pages << a.m.page_shift;
  const int64_t mask = ((int64_t)1 << a.m.page_shift) - 1;
  for (int j0 = 0; j0 < kept; j0 += kMoveUnroll) {
    uint4 x[kMoveUnroll];
    int64_t to[kMoveUnroll];
#pragma unroll
    for (int i = 0; i < kMoveUnroll; ++i) {
      const int j = j0 + i;
      to[i] = -1;
      if (j >= kept) continue;
      const int p = a.path[s0 + j];
      if (p <= j || p >= n) continue;  // in its place already, or damaged
      const int64_t s = a.slots[s0 + p], d = a.slots[s0 + j];
      if (s < 0 || s >= slots || d < 0 || d >= slots) continue;
      to[i] = d;
      x[i] = *(const uint4*)(c.base + (s >> a.m.page_shift) * c.page + (s & mask) * c.token);
    }
#pragma unroll
    for (int i = 0; i < kMoveUnroll; ++i)
      if (to[i] >= 0) *(uint4*)(c.base + (to[i] >> a.m.page_shift) * c.page + (to[i] & mask) * c.token) = x[i];
  }
}

// The first tokens[i] tokens of page from[i] to page to[i].
__global__ __launch_bounds__(256) void copy_pages_kernel(CopyArgs a) {
  const int i = blockIdx.x;
  const int from = cache_page(a.from[i], a.m.num_pages), to = cache_page(a.to[i], a.m.num_pages);
  if (from < 0 || to < 0 || from == to) return;
  const int size = 1 << a.m.page_shift;
  const int n = a.tokens ? min(a.tokens[i], size) : size;
  const int col = threadIdx.x % a.columns, step = 256 / a.columns;
  const int piece = blockIdx.z * a.columns + col;
  if (piece >= a.m.pieces || (int)threadIdx.x >= step * a.columns) return;
  const MoveColumn c = move_column(a.m, blockIdx.y, piece);
  const char* src = c.base + from * c.page;
  char* dst = c.base + to * c.page;
  for (int t0 = threadIdx.x / a.columns; t0 < n; t0 += kMoveUnroll * step) {
    uint4 x[kMoveUnroll];
#pragma unroll
    for (int u = 0; u < kMoveUnroll; ++u)
      if (t0 + u * step < n) x[u] = *(const uint4*)(src + (t0 + u * step) * c.token);
#pragma unroll
    for (int u = 0; u < kMoveUnroll; ++u)
      if (t0 + u * step < n) *(uint4*)(dst + (t0 + u * step) * c.token) = x[u];
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
// ones itself, which is less than a second launch.
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
    for (int j = tid; j < a.width; j += 256)
      a.out_table[(int64_t)i * a.out_stride + j] = j >= live ? -1 : own && j == full ? page : row[j];
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
  int32_t* counts;  // [tiles] unused pages of a tile
  int32_t *pages, *count;
  int64_t table_stride;
  int32_t B, width, page_shift, num_pages, n_held, tiles;
};
constexpr int kUnusedTile = 4096;  // pages a block counts or lists: 16 a thread

__global__ __launch_bounds__(256) void unused_clear_kernel(uint8_t* flags, int64_t n) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 16;
  if (i < n) *(uint4*)(flags + i) = make_uint4(0, 0, 0, 0);
}

// Whoever holds a page writes the same 1: no atomics.
__global__ __launch_bounds__(256) void unused_mark_kernel(UnusedArgs a) {
  const int b = blockIdx.y;
  if (b == a.B) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < a.n_held; i += (int64_t)gridDim.x * 256) {
      const int pg = cache_page(a.held[i], a.num_pages);
      if (pg >= 0) a.flags[pg] = 1;
    }
    return;
  }
  const int64_t live = min(table_pages(max(a.lens[b], 0), a.page_shift), (int64_t)a.width);
  const int32_t* row = a.table + b * a.table_stride;
  for (int64_t j = (int64_t)blockIdx.x * 256 + threadIdx.x; j < live; j += (int64_t)gridDim.x * 256) {
    const int pg = cache_page(row[j], a.num_pages);
    if (pg >= 0) a.flags[pg] = 1;
  }
}

// sum over the block's 256 threads, to all; `red` 4 ints
__device__ __forceinline__ int block_sum(int x, int* red) {
#pragma unroll
  for (int m = 32; m; m >>= 1) x += __shfl_xor(x, m);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
  __syncthreads();
  return red[0] + red[1] + red[2] + red[3];
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
  const int n = block_sum(__popc(unused_bits(a, p0)), red);
  if (threadIdx.x == 0) a.counts[blockIdx.x] = n;
}

__global__ __launch_bounds__(256) void unused_list_kernel(UnusedArgs a) {
  __shared__ int red[4];
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  int before = 0, all = 0;
  for (int t = tid; t < a.tiles; t += 256) {
    const int n = a.counts[t];
    all += n;
    if (t < (int)blockIdx.x) before += n;
  }
  before = block_sum(before, red);
  all = block_sum(all, red);
  const int64_t p0 = (int64_t)blockIdx.x * kUnusedTile + tid * 16;
  uint32_t bits = unused_bits(a, p0);
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
  int at = before + inc - mine;
  for (int w = 0; w < wv; ++w) at += red[w];
  for (; bits; bits &= bits - 1) a.pages[at++] = (int)(p0 + __builtin_ctz(bits));
  // the list's places behind the last unused page
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (p0 + i >= all && p0 + i < a.num_pages) a.pages[p0 + i] = -1;
  if (blockIdx.x == 0 && tid == 0) a.count[0] = all;
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
  if (all > (1 << 20)) return HTREE_EUNSUPPORTED;
  m->pieces = (int32_t)all, m->k_all = c->H_kv * m->k_pieces;
  m->page_shift = log2i(c->page_size), m->num_pages = c->num_pages;
  return HTREE_OK;
}

// runs f(layers of this launch) for 64 layers at a time
template <typename F>
static int by_layers(int32_t layers, void* const* k, void* const* v, MoveArgs* m, F f) {
  for (int l = 0; l < layers; l += kMoveLayers) {
    const int n = layers - l < kMoveLayers ? layers - l : kMoveLayers;
    for (int i = 0; i < n; ++i) m->k[i] = (char*)k[l + i], m->v[i] = (char*)v[l + i];
    f(n);
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
  a.slots = slots, a.starts = starts, a.path = path, a.kept = kept, a.rows = rows;
  const unsigned threads = a.m.pieces >= 256 ? 256 : (a.m.pieces + 63) / 64 * 64;
  const unsigned z = (a.m.pieces + threads - 1) / threads;
  return by_layers(layers, k_layers, v_layers, &a.m, [&](int n) {
    hipLaunchKernelGGL(keep_drafts_kernel, dim3(B, n, z), dim3(threads), 0, (hipStream_t)stream, a);
  });
}

extern "C" int htree_copy_pages(const htree_cache* c, int32_t layers, void* const* k_layers, void* const* v_layers,
                                int32_t n, const int32_t* from, const int32_t* to, const int32_t* tokens,
                                void* stream) {
  CopyArgs a;
  const int rc = move_args(c, layers, k_layers, v_layers, &a.m);
  if (rc) return rc;
  if (n < 0) return HTREE_ESHAPE;
  if (n == 0 || layers == 0) return HTREE_OK;
  if (!from || !to) return HTREE_ENULL;
  a.from = from, a.to = to, a.tokens = tokens, a.n = n;
  a.columns = a.m.pieces < 256 ? a.m.pieces : 256;
  const unsigned z = (a.m.pieces + a.columns - 1) / a.columns;
  return by_layers(layers, k_layers, v_layers, &a.m, [&](int l) {
    hipLaunchKernelGGL(copy_pages_kernel, dim3(n, l, z), dim3(256), 0, (hipStream_t)stream, a);
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

extern "C" int htree_unused_pages_workspace_bytes(int32_t num_pages, int64_t* bytes) {
  if (!bytes) return HTREE_ENULL;
  if (num_pages < 0) return HTREE_ESHAPE;
  const int64_t tiles = ((int64_t)num_pages + kUnusedTile - 1) / kUnusedTile;
  *bytes = tiles * (kUnusedTile + 4);
  return HTREE_OK;
}

extern "C" int htree_unused_pages(int32_t B, int32_t page_size, int32_t num_pages, int32_t table_width,
                                  int64_t table_stride, const int32_t* block_table, const int32_t* lens,
                                  int32_t n_held, const int32_t* held, int32_t* pages, int32_t* count,
                                  void* workspace, int64_t workspace_bytes, void* stream) {
  if (B < 0 || num_pages < 0 || table_width < 0 || n_held < 0) return HTREE_ESHAPE;
  if (B > 1 && table_stride < table_width) return HTREE_ESHAPE;
  if (page_size < 1 || (page_size & (page_size - 1)) || B > kCacheMaxRequests) return HTREE_EUNSUPPORTED;
  if (num_pages == 0) return HTREE_OK;
  if (!pages || !count || !workspace || (n_held && !held) || (B && !lens) || (B && table_width && !block_table))
    return HTREE_ENULL;
  if (off16(workspace)) return HTREE_EUNSUPPORTED;
  int64_t need = 0;
  htree_unused_pages_workspace_bytes(num_pages, &need);
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
  a.tiles = (int)(((int64_t)num_pages + kUnusedTile - 1) / kUnusedTile);
  a.flags = (uint8_t*)workspace;
  a.counts = (int32_t*)(a.flags + (int64_t)a.tiles * kUnusedTile);
  a.pages = pages, a.count = count;
  a.table_stride = table_stride;
  a.B = B, a.width = table_width, a.page_shift = log2i(page_size), a.num_pages = num_pages, a.n_held = n_held;
  hipStream_t s = (hipStream_t)stream;
  hipLaunchKernelGGL(unused_clear_kernel, dim3(a.tiles), dim3(256), 0, s, a.flags, (int64_t)a.tiles * kUnusedTile);
  const int64_t most = table_width > n_held ? table_width : n_held;
  const unsigned gx = (unsigned)(most <= 1024 ? 1 : most >= 16384 ? 16 : (most + 1023) / 1024);
  if (B + (n_held > 0) > 0)
    hipLaunchKernelGGL(unused_mark_kernel, dim3(gx, B + (n_held > 0)), dim3(256), 0, s, a);
  hipLaunchKernelGGL(unused_count_kernel, dim3(a.tiles), dim3(256), 0, s, a);
  hipLaunchKernelGGL(unused_list_kernel, dim3(a.tiles), dim3(256), 0, s, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? HTREE_OK : (int)e;
}
