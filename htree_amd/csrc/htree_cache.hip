// Serving from a paged key/value cache: block tables and slot maps from
// request lengths, new keys and values written to their slots (rotated by
// their positions), and the entry point of the attention over the cache
// (htree_draft.h).
#include "htree_cache_host.h"
#include "htree_cache_scan.h"
#include "htree_draft.h"

#include <cmath>

namespace htree {

// ---------------------------------------------------------------- tables
// (the lengths' sums of all requests sit in a block's LDS)
constexpr int kTabTile = 256;       // rows, or new pages, that a block takes at a time

struct TabArgs {
  const int32_t *ctx, *add, *parents, *free_pages;
  int32_t *table, *starts, *positions, *lens, *used;
  int64_t* slots;
  int64_t table_stride;
  int32_t B, rows, page_shift, num_pages, width, n_free, page_blocks, tiles;
};

// Blocks 0 .. page_blocks - 1 write the new pages' table entries, the others
// the rows' slots and positions, `tiles` times 256 each.  Each block sums the
// lengths again (two loads and two scans), which is less than a second launch;
// a row's slot comes from the page list itself, not from the entry another
// block may be writing.  Bound by latency (lengths, scans, search, entry):
// 3.6 us for 64 rows of 64 requests, 6.4 us for up to 24 drafted rows of each
// of 256, 8.2 us for 32 whole prompts of up to 32768 rows (12 bytes a row
// out).
__global__ __launch_bounds__(256) void page_tables_kernel(TabArgs a) {
  extern __shared__ int32_t tab_lds[];
  __shared__ int64_t red[4];
  __shared__ int32_t par[kTabTile];
  int32_t* starts = tab_lds;          // [B + 1], rows at most
  int32_t* first = tab_lds + a.B + 1; // [B + 1], new pages of the requests before
  const int tid = threadIdx.x;
  const int P1 = (1 << a.page_shift) - 1;
  tab_scan(a.B, a.rows, starts, red, [&](int b) { return (int64_t)max(a.add[b], 0); });
  auto had = [&](int b) { return table_pages(max(a.ctx[b], 0), a.page_shift); };
  auto now = [&](int b) {
    return table_pages((int64_t)max(a.ctx[b], 0) + (starts[b + 1] - starts[b]), a.page_shift);
  };
  const int64_t need = tab_scan(a.B, 0x7fffffff, first, red, [&](int b) { return now(b) - had(b); });
  auto fresh = [&](int64_t i) {  // i-th new page
    return cache_page(i < a.n_free ? a.free_pages[i] : -1, a.num_pages);
  };

  if ((int)blockIdx.x < a.page_blocks) {
    if (blockIdx.x == 0) {
      for (int b = tid; b <= a.B; b += 256) {
        a.starts[b] = starts[b];
        if (b < a.B)
          a.lens[b] = (int32_t)min((int64_t)max(a.ctx[b], 0) + starts[b + 1] - starts[b], (int64_t)0x7fffffff);
      }
      if (tid == 0) a.used[0] = (int32_t)min(need, (int64_t)0x7fffffff);
    }
    const int64_t total = min(need, (int64_t)0x7fffffff);
    for (int x = 0; x < a.tiles; ++x) {
      const int64_t i = ((int64_t)blockIdx.x * a.tiles + x) * kTabTile + tid;
      if (i >= total) return;
      const int b = table_find(first, a.B, (int)i);
      const int64_t j = had(b) + i - first[b];
      if (j < a.width) a.table[b * a.table_stride + j] = fresh(i);
    }
    return;
  }

  for (int x = 0; x < a.tiles; ++x) {
    const int64_t row0 = ((int64_t)(blockIdx.x - a.page_blocks) * a.tiles + x) * kTabTile, row = row0 + tid;
    if (row0 >= a.rows) return;
    if (a.parents) {
      if (x) __syncthreads();  // the earlier tile's parents have been read
      par[tid] = row < a.rows ? a.parents[row] : -1;
      __syncthreads();
    }
    if (row >= a.rows) continue;
    int64_t slot = -1;
    int pos = -1;
    if (row < starts[a.B]) {
      const int b = table_find(starts, a.B, (int)row);
      const int ctx = max(a.ctx[b], 0), s0 = starts[b], j = (int)row - s0;
      const int64_t at = (int64_t)ctx + j;
      const int64_t pi = at >> a.page_shift, h = had(b);
      if (pi < a.width) {
        const int pg = pi >= h ? fresh(first[b] + pi - h)
                               : cache_page(a.table[b * a.table_stride + pi], a.num_pages);
        if (pg >= 0) slot = ((int64_t)pg << a.page_shift) + (at & P1);
      }
      int64_t depth = j;
      if (a.parents) {
        // up the tree; a parent comes before its children (else: a root)
        depth = 0;
        int i = j;
        while ((i = draft_parent(s0 + i >= row0 ? par[s0 + i - row0] : a.parents[s0 + i], i)) >= 0) ++depth;
      }
      pos = (int)min(ctx + depth, (int64_t)0x7fffffff);
    }
    a.slots[row] = slot;
    a.positions[row] = pos;
  }
}

// ---------------------------------------------------------------- append
struct AppendArgs {
  const char *k, *v, *q;
  char *kc, *vc, *qo;
  const int64_t* slots;
  const int32_t* positions;
  const float *cs, *sn;
  int64_t k_row, k_head, v_row, v_head, q_row, q_head, o_row, o_head;  // bytes
  int64_t kc_page, kc_token, kc_head, vc_page, vc_token, vc_head;      // bytes
  int64_t num_slots;
  int32_t rows, H, Hkv, Dk, Dv, page_shift, rope_rows;
  int32_t lanes;  // of a row: 2^n, at least the pieces of a half of a head (a head, of values)
};

template <int N>
struct AppendVec;
template <>
struct AppendVec<16> {
  typedef uint4 V;
};
template <>
struct AppendVec<8> {
  typedef uint2 V;
};

// x1 c - x2 s and x2 c + x1 s of the pairs (d, d + Dk/2), in fp32, rounded once
template <typename T, int NV>
__device__ __forceinline__ void rotate(const T* x1, const T* x2, const float* c, const float* s, T* y1, T* y2) {
#pragma unroll
  for (int e = 0; e < NV; ++e) {
    const float a = (float)x1[e], b = (float)x2[e];
    y1[e] = (T)(a * c[e] - b * s[e]);
    y2[e] = (T)(b * c[e] + a * s[e]);
  }
}

// heads of one row of q (or k): a lane of its `lanes` takes one chunk of VB
// bytes of each half of a head, lanes / (chunks of a half) heads at a time
template <typename T, int VB>
__device__ __forceinline__ void append_rotate(const char* src, int64_t src_head, char* dst, int64_t dst_head,
                                              int heads, int half, const float* c, const float* s, int lane,
                                              int lanes, int part, int parts) {
  constexpr int NV = VB / (int)sizeof(T);
  typedef typename AppendVec<VB>::V V;
  const int per = half / NV, hpi = lanes / per;
  const int h0 = lane / per, ch = lane - h0 * per;
  if (h0 >= hpi) return;
  float cc[NV], ss[NV];
#pragma unroll
  for (int e = 0; e < NV; ++e) {
    cc[e] = c[ch * NV + e];
    ss[e] = s[ch * NV + e];
  }
  const int64_t hb = (int64_t)half * sizeof(T);
  constexpr int U = 4;
  for (int h = part * hpi + h0; h < heads; h += U * parts * hpi) {
    V x1[U], x2[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int hh = h + i * parts * hpi;
      if (hh < heads) {
        x1[i] = *(const V*)(src + hh * src_head + ch * VB);
        x2[i] = *(const V*)(src + hh * src_head + hb + ch * VB);
      }
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int hh = h + i * parts * hpi;
      if (hh < heads) {
        V y1, y2;
        rotate<T, NV>((const T*)&x1[i], (const T*)&x2[i], cc, ss, (T*)&y1, (T*)&y2);
        *(V*)(dst + hh * dst_head + ch * VB) = y1;
        *(V*)(dst + hh * dst_head + hb + ch * VB) = y2;
      }
    }
  }
}

__device__ __forceinline__ void append_copy(const char* src, int64_t src_head, char* dst, int64_t dst_head,
                                            int heads, int bytes, int lane, int lanes, int part, int parts) {
  const int per = bytes / 16, hpi = lanes / per;
  const int h0 = lane / per, ch = lane - h0 * per;
  if (h0 >= hpi) return;
  constexpr int U = 4;
  for (int h = part * hpi + h0; h < heads; h += U * parts * hpi) {
    f32x4 x[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int hh = h + i * parts * hpi;
      if (hh < heads) x[i] = *(const f32x4*)(src + hh * src_head + ch * 16);
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int hh = h + i * parts * hpi;
      if (hh < heads) *(f32x4*)(dst + hh * dst_head + ch * 16) = x[i];
    }
  }
}

// `lanes` lanes per row (token): a wave where the row has heads enough for
// it, else as many as it has pieces (keys and values of one head of dim 64,
// 2M rows, bf16: 235 us with 8 lanes a row, 1268 us with a wave each).
// blockIdx.y splits a row's heads where there are few rows.  A lane has four
// heads' loads in flight.  Bound by memory, k, v and q once in and once out:
// 32768 rows of 32 query and 2 KV heads of 128, bf16, 115 us (5.4 TB/s, a
// large copy reaches 4.8); 64 such rows 4 to 5 us, most of it the launch and
// the chain slot -> row.
template <typename T, int VB>
__global__ __launch_bounds__(256) void cache_append_kernel(AppendArgs a) {
  const int lanes = a.lanes, lane = threadIdx.x & (lanes - 1);
  const int64_t row = ((int64_t)blockIdx.x * 256 + threadIdx.x) / lanes;
  if (row >= a.rows) return;
  const int part = blockIdx.y, parts = gridDim.y;
  const int64_t slot = a.slots[row];
  const bool rope = a.cs != nullptr;
  int pos = 0;
  bool at = true;
  if (rope) {
    pos = a.positions[row];
    at = pos >= 0 && pos < a.rope_rows;
  }
  const int half = a.Dk / 2;
  const float* c = a.cs + (int64_t)(at ? pos : 0) * half;
  const float* s = a.sn + (int64_t)(at ? pos : 0) * half;
  if (a.q) {
    char* qo = a.qo + row * a.o_row;
    if (at) {
      append_rotate<T, VB>(a.q + row * a.q_row, a.q_head, qo, a.o_head, a.H, half, c, s, lane, lanes, part, parts);
    } else {
      // a row without a position has a query of zeros
      const int n = a.H * (a.Dk * (int)sizeof(T) / 16);
      for (int i = part * lanes + lane; i < n; i += parts * lanes) *(uint4*)(qo + (int64_t)i * 16) = make_uint4(0, 0, 0, 0);
    }
  }
  if (!at || slot < 0 || slot >= a.num_slots) return;
  const int64_t page = slot >> a.page_shift, off = slot & ((1 << a.page_shift) - 1);
  char* kd = a.kc + page * a.kc_page + off * a.kc_token;
  char* vd = a.vc + page * a.vc_page + off * a.vc_token;
  if (rope)
    append_rotate<T, VB>(a.k + row * a.k_row, a.k_head, kd, a.kc_head, a.Hkv, half, c, s, lane, lanes, part, parts);
  else
    append_copy(a.k + row * a.k_row, a.k_head, kd, a.kc_head, a.Hkv, a.Dk * (int)sizeof(T), lane, lanes, part, parts);
  append_copy(a.v + row * a.v_row, a.v_head, vd, a.vc_head, a.Hkv, a.Dv * (int)sizeof(T), lane, lanes, part, parts);
}

// ------------------------------------------------------------------ host
static DraftPlan draft_plan(const htree_cache* c, int B, int rows, int H, int width) {
  return draft_plan(c->Dk, c->Dv, cache_es(c), B, rows, H, c->H_kv, width, c->page_size);
}

static int draft_check(const htree_cache* c, int32_t B, int32_t rows, int32_t H, int32_t width) {
  const int rc = cache_check(c);
  if (rc) return rc;
  if (B < 0 || rows < 0 || H <= 0 || H % c->H_kv || width < 0) return HTREE_ESHAPE;
  if ((int64_t)width * c->page_size > (1 << 30) || B > kCacheMaxRequests) return HTREE_EUNSUPPORTED;
  // 32-bit rows (new tokens x heads of a group), and the units of 16 rows at least
  if ((int64_t)rows * (H / c->H_kv) >= 0x7fffff00ll ||
      ((int64_t)rows * (H / c->H_kv) / 16 + B + 512) * c->H_kv > kDraftMaxUnits)
    return HTREE_EUNSUPPORTED;
  return HTREE_OK;
}

}  // namespace htree

using namespace htree;

extern "C" int htree_page_tables(int32_t B, int32_t rows, int32_t page_size, int32_t num_pages,
                                 int32_t table_width, int64_t table_stride, int32_t n_free,
                                 const int32_t* ctx_lens, const int32_t* new_lens, const int32_t* parents,
                                 int32_t* block_table, const int32_t* free_pages, int32_t* starts,
                                 int64_t* slots, int32_t* positions, int32_t* lens, int32_t* pages_used,
                                 void* stream) {
  if (B < 0 || rows < 0 || num_pages < 0 || table_width < 0 || n_free < 0) return HTREE_ESHAPE;
  if (B > 1 && table_stride < table_width) return HTREE_ESHAPE;
  if (page_size < 1 || (page_size & (page_size - 1)) || B > kCacheMaxRequests) return HTREE_EUNSUPPORTED;
  if (B == 0 && rows == 0) return HTREE_OK;
  if (B == 0) return HTREE_ESHAPE;
  if (!ctx_lens || !new_lens || !starts || !lens || !pages_used) return HTREE_ENULL;
  if ((table_width && !block_table) || (n_free && !free_pages) || (rows && (!slots || !positions))) return HTREE_ENULL;
  // (the lengths of a step are a natural input of the next: a block would read
  // some after another has written them)
  const Range in[4] = {{ctx_lens, B * 4ll}, {new_lens, B * 4ll}, {parents, parents ? rows * 4ll : 0},
                       {free_pages, n_free * 4ll}};
  const Range table = {block_table, table_width ? ((B - 1) * table_stride + table_width) * 4 : 0};
  const Range written[6] = {table, {starts, (B + 1) * 4ll}, {slots, rows * 8ll}, {positions, rows * 4ll},
                            {lens, B * 4ll}, {pages_used, 4}};
  for (const Range& x : written)
    for (const Range& y : in)
      if (overlap(x, y)) return HTREE_EOVERLAP;
  for (const Range& x : written)
    if (&x != written && overlap(x, table)) return HTREE_EOVERLAP;
  TabArgs a;
  a.ctx = ctx_lens, a.add = new_lens, a.parents = parents, a.free_pages = free_pages;
  a.table = block_table, a.starts = starts, a.positions = positions, a.lens = lens, a.used = pages_used;
  a.slots = slots;
  a.table_stride = table_stride;
  a.B = B, a.rows = rows, a.page_shift = log2i(page_size), a.num_pages = num_pages, a.width = table_width;
  a.n_free = n_free;
  // few rows: a tile of 256 a block, for the latency; many: enough tiles that
  // the sums of the lengths do not count
  const int64_t row_tiles = ((int64_t)rows + kTabTile - 1) / kTabTile;
  a.tiles = (int)(row_tiles <= 1024 ? 1 : row_tiles < 8192 ? (row_tiles + 1023) / 1024 : 8);
  // a request's new tokens begin at most one page more than they fill
  const int64_t pages = (int64_t)rows / page_size + B, step = (int64_t)kTabTile * a.tiles;
  a.page_blocks = (int)((pages + step - 1) / step);
  const int64_t grid = a.page_blocks + ((int64_t)rows + step - 1) / step;
  hipLaunchKernelGGL(page_tables_kernel, dim3((unsigned)grid), dim3(256), 2 * (B + 1) * 4, (hipStream_t)stream, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? HTREE_OK : (int)e;
}

extern "C" int htree_cache_append(const htree_cache* c, int32_t rows, int32_t H, const void* k, int64_t k_row,
                                  int64_t k_head, const void* v, int64_t v_row, int64_t v_head, const void* q,
                                  int64_t q_row, int64_t q_head, const int64_t* slots, const int32_t* positions,
                                  const float* cos_table, const float* sin_table, int32_t rope_rows, void* q_out,
                                  void* k_cache, void* v_cache, void* stream) {
  const int rc = cache_check(c);
  if (rc) return rc;
  if (rows < 0) return HTREE_ESHAPE;
  if (rows == 0) return HTREE_OK;
  if (!k || !v || !slots || !k_cache || !v_cache) return HTREE_ENULL;
  const bool rope = cos_table || sin_table;
  if (rope && (!cos_table || !sin_table || !positions)) return HTREE_ENULL;
  if (q && (!rope || !q_out)) return HTREE_ENULL;
  if ((rope && (rope_rows <= 0 || c->Dk % 2)) || (q && H <= 0)) return HTREE_ESHAPE;
  const int es = cache_es(c);
  const int64_t st[6] = {k_row, k_head, v_row, v_head, q ? q_row : 0, q ? q_head : 0};
  for (int64_t s : st)
    if (s < 0 || s * es % 16) return HTREE_EUNSUPPORTED;
  if (off16(k) || off16(v) || off16(q) || off16(q_out) || off16(k_cache) || off16(v_cache)) return HTREE_EUNSUPPORTED;
  // A source in the cache's range: a row could be read after another one's
  // write.  (The two caches' ranges may overlap: keys beside values in a page.)
  const auto rows_end = [&](int64_t row, int64_t head, int heads, int D) {
    return ((rows - 1) * row + (heads - 1) * head + D) * es;
  };
  const auto cache_end = [&](int64_t page, int64_t token, int64_t head, int D) {
    return ((c->num_pages - 1) * page + (c->page_size - 1) * token + (c->H_kv - 1) * head + D) * es;
  };
  const Range from[3] = {{k, rows_end(k_row, k_head, c->H_kv, c->Dk)}, {v, rows_end(v_row, v_head, c->H_kv, c->Dv)},
                         {q, q ? rows_end(q_row, q_head, H, c->Dk) : 0}};
  const Range to[2] = {{k_cache, cache_end(c->k_page, c->k_token, c->k_head, c->Dk)},
                       {v_cache, cache_end(c->v_page, c->v_token, c->v_head, c->Dv)}};
  for (const Range& x : from)
    for (const Range& y : to)
      if (overlap(x, y)) return HTREE_EOVERLAP;
  AppendArgs a;
  a.k = (const char*)k, a.v = (const char*)v, a.q = (const char*)q;
  a.kc = (char*)k_cache, a.vc = (char*)v_cache, a.qo = (char*)q_out;
  a.slots = slots, a.positions = positions, a.cs = rope ? cos_table : nullptr, a.sn = sin_table;
  a.k_row = k_row * es, a.k_head = k_head * es, a.v_row = v_row * es, a.v_head = v_head * es;
  a.q_row = q_row * es, a.q_head = q_head * es;
  a.o_head = (int64_t)c->Dk * es, a.o_row = a.o_head * H;
  a.kc_page = c->k_page * es, a.kc_token = c->k_token * es, a.kc_head = c->k_head * es;
  a.vc_page = c->v_page * es, a.vc_token = c->v_token * es, a.vc_head = c->v_head * es;
  a.num_slots = (int64_t)c->num_pages * c->page_size;
  a.rows = rows, a.H = q ? H : 0, a.Hkv = c->H_kv, a.Dk = c->Dk, a.Dv = c->Dv;
  a.page_shift = log2i(c->page_size), a.rope_rows = rope_rows;
  // 16-byte chunks where a half of a head holds whole ones
  const bool wide = c->Dk * es % 32 == 0;
  const int per_k = rope ? c->Dk / 2 * es / (wide ? 16 : 8) : c->Dk * es / 16, per_v = c->Dv * es / 16;
  const int heads = q ? H : c->H_kv, most = per_k > per_v ? per_k : per_v;
  a.lanes = 1;
  while (a.lanes < 64 && (a.lanes < most || a.lanes < heads * most)) a.lanes *= 2;
  const unsigned gx = (unsigned)(((int64_t)rows * a.lanes + 255) / 256);
  const unsigned gy = gx >= 1024 ? 1 : gx >= 256 ? 2 : 4;
  const dim3 grid(gx, gy);
  hipStream_t s = (hipStream_t)stream;
#define HTREE_APPEND(T)                                                                             \
  if (wide) hipLaunchKernelGGL((cache_append_kernel<T, 16>), grid, dim3(256), 0, s, a);             \
  else hipLaunchKernelGGL((cache_append_kernel<T, 8>), grid, dim3(256), 0, s, a)
  if (c->dtype == HTREE_F32) {
    HTREE_APPEND(float);
  } else if (c->dtype == HTREE_BF16) {
    HTREE_APPEND(__bf16);
  } else {
    HTREE_APPEND(_Float16);
  }
#undef HTREE_APPEND
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? HTREE_OK : (int)e;
}

extern "C" int htree_draft_attention_workspace_bytes(const htree_cache* c, int32_t B, int32_t rows, int32_t H,
                                                     int32_t table_width, int64_t* bytes) {
  if (!bytes) return HTREE_ENULL;
  const int rc = draft_check(c, B, rows, H, table_width);
  if (rc) return rc;
  *bytes = B == 0 || rows == 0 ? 0 : draft_plan(c, B, rows, H, table_width).bytes;
  return HTREE_OK;
}

extern "C" int htree_draft_attention(const htree_cache* c, int32_t B, int32_t rows, int32_t H, int32_t table_width,
                                     int64_t table_stride, float scale, const void* q, int64_t q_row,
                                     int64_t q_head, const void* k_cache, const void* v_cache,
                                     const int32_t* block_table, const int32_t* lens, const int32_t* starts,
                                     const int32_t* parents, void* out, int64_t out_row, int64_t out_head,
                                     void* workspace, int64_t workspace_bytes, void* stream) {
  const int rc = draft_check(c, B, rows, H, table_width);
  if (rc) return rc;
  if (!std::isfinite(scale * kLog2e)) return HTREE_ESHAPE;
  if (B == 0 || rows == 0) return HTREE_OK;
  if (!q || !k_cache || !v_cache || !lens || !starts || !out || (table_width && !block_table)) return HTREE_ENULL;
  if (B > 1 && table_stride < table_width) return HTREE_ESHAPE;
  const int es = cache_es(c);
  const int64_t st[4] = {q_row, q_head, out_row, out_head};
  for (int64_t s : st)
    if (s < 0 || s * es % 16) return HTREE_EUNSUPPORTED;
  if (off16(q) || off16(k_cache) || off16(v_cache) || off16(out) || off16(workspace)) return HTREE_EUNSUPPORTED;
  const DraftPlan p = draft_plan(c, B, rows, H, table_width);
  if (p.bytes > 0 && !workspace) return HTREE_ENULL;
  if (workspace_bytes < p.bytes) return HTREE_EWORKSPACE;
  DraftArgs a;
  a.q = (const char*)q, a.k = (const char*)k_cache, a.v = (const char*)v_cache, a.out = (char*)out;
  a.table = block_table, a.lens = lens, a.starts = starts, a.parents = parents;
  a.ws_o = (float*)workspace;
  a.ws_ml = a.ws_o + p.slots * p.R * p.D;
  a.ws_chunk = (int32_t*)(a.ws_ml + p.slots * p.R * 2);
  a.table_stride = table_stride;
  a.q_row = q_row * es, a.q_head = q_head * es, a.o_row = out_row * es, a.o_head = out_head * es;
  a.k_page = c->k_page * es, a.k_token = c->k_token * es, a.k_head = c->k_head * es;
  a.v_page = c->v_page * es, a.v_token = c->v_token * es, a.v_head = c->v_head * es;
  a.B = B, a.rows = rows, a.Hkv = c->H_kv, a.G = H / c->H_kv, a.Dk = c->Dk, a.Dv = c->Dv;
  a.width = table_width, a.page_shift = log2i(c->page_size), a.num_pages = c->num_pages;
  a.target = p.target;
  a.near = p.near;
  a.one_round = p.one_round;
  a.negate = scale < 0.f;
  a.c = fmaxf(fabsf(scale) * kLog2e, 1e-37f);  // a scale of 0 still multiplies -inf
  a.inv_c = 1.f / a.c;
  hipStream_t s = (hipStream_t)stream;
  if (c->dtype == HTREE_F32) return draft_launch_type<float>(a, p, s);
  if (c->dtype == HTREE_BF16) return draft_launch_type<__bf16>(a, p, s);
  return draft_launch_type<_Float16>(a, p, s);
}
