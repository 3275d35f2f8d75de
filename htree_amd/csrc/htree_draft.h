// Attention of new tokens over a paged key/value cache (gfx950): single
// tokens, drafted trees of tokens, or chunks of a prompt.
//
//   o[r, h] = sum_t p_t v_t,  p = softmax_t(scale q[r, h] . k_t)
//
// over the tokens t of row r's request that it sees: the cached ones, and of
// the new ones its ancestors in the drafted tree (or, without one, those
// before it) and itself.  The G query heads of a KV head and the request's
// new tokens are the rows of one matrix product, so each cached row is read
// once for all of them.
//
// One pass: scores S^T = K Q^T, weights exp2 of the scores against a running
// max, output O^T = V^T P^T, all in matrix products of 16 x 16.  With the
// tokens as the scores' rows, a lane holds the weights of exactly the tokens
// that the second product takes from it: P never leaves the registers.
//
// A block of four waves takes a unit: a group of rows of one (request, KV
// head) and a chunk of its tokens.  Chunks are cut so that the units fill the
// GPU once, whatever the lengths; each block finds its own from the lengths,
// which never leave the device.  Units of one request meet in a second launch
// (draft_join_kernel) through the workspace.
//   draft_kernel: up to 32 rows.  The waves take the chunk's tiles of tokens
//     in turn, each on its own: no barrier until the end, where the four
//     running (max, sum, output) states meet in LDS.
//   draft_rows_kernel: 128 rows.  Each wave has 32 rows of its own and all of
//     them take the same tiles.
//
// What bounds them (bf16, D 128, 16-token pages, launch and join together):
//   64 requests of up to 16384 tokens, one token each, 32/4 heads: the cache's
//     bytes, 276 us (4.9 TB/s).
//   One request of 131008 tokens, 64 drafted, 64/8 heads: 303 us, 906 TFLOP/s,
//     where a library product of 8192 x 8192 reaches 1125: the matrix unit is
//     busy 40% of the time; each tile's softmax, and the latency that two
//     waves per SIMD do not cover, is the rest.
//   One request of 2048 tokens, one token: 7.8 + 4.7 us, a chain of dependent
//     reads (lengths, pages, keys, states) and two launches.
#pragma once

#include "htree_cache_index.h"
#include "htree_common.h"

namespace htree {

struct DraftArgs {
  const char *q, *k, *v;
  char* out;
  const int32_t *table, *lens, *starts, *parents;
  float* ws_o;        // [slots][R][D] output of a unit, relative to its max
  float* ws_ml;       // [slots][R][2] max (log2 units) and sum
  int32_t* ws_chunk;  // tiles of a chunk, for the join
  int64_t table_stride;
  int64_t q_row, q_head, o_row, o_head;                                // bytes
  int64_t k_page, k_token, k_head, v_page, v_token, v_head;            // bytes
  int32_t B, rows, Hkv, G, Dk, Dv, width, page_shift, num_pages;
  int32_t near;       // units that share tokens, on average
  int32_t target;     // units to split into (0: one unit per group of rows)
  int32_t one_round;  // the join's blocks take one piece of work each
  int32_t negate;     // the scale is negative: the queries change sign
  float c, inv_c;     // |scale| * log2(e), not 0
};

template <typename T>
struct DraftT;  // operand types and products of an element type
template <>
struct DraftT<__bf16> {
  typedef bf16x8 V8;
  static __device__ __forceinline__ f32x4 mma(bf16x8 a, bf16x8 b, f32x4 c) { return mma32(a, b, c); }
  static __device__ __forceinline__ f32x4 mma_k16(s16x4 a, s16x4 b, f32x4 c) { return mma16(a, b, c); }
};
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(4))) _Float16 f16x4;
template <>
struct DraftT<_Float16> {
  typedef f16x8 V8;
  static __device__ __forceinline__ f32x4 mma(f16x8 a, f16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 mma_k16(s16x4 a, s16x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4, a),
                                                 __builtin_bit_cast(f16x4, b), c, 0, 0, 0);
  }
};
template <>
struct DraftT<float> {};

template <typename T, int D>
struct DraftShape {
  static constexpr int ES = (int)sizeof(T);
  static constexpr bool F32 = ES == 4;
  static constexpr int ROWB = D * ES;      // bytes of a staged row
  static constexpr int CPR = ROWB / 16;    // its 16-byte chunks
  static constexpr int RPI = 64 / CPR;     // rows of one load of a wave
  static constexpr int NQ = D / 16;        // groups of 4 dims that a lane holds of a row
  // fp32: dims of a lane's V operand read at once
  static constexpr int VW = D / 16 > 4 ? 4 : D / 16;
  static constexpr int OC = D / 4;         // 16-byte chunks of an fp32 row
  static constexpr int OS = OC < 16 ? 7 : 15;
};

// Places of a row's chunk: rows that are read together fall on other banks.
// Keys (and fp32 values): 16 rows, one chunk of each at a time.
template <int CPR>
__device__ __forceinline__ int draft_swz(int row, int chunk) {
  return CPR >= 16 ? chunk ^ (row & 15) : CPR == 8 ? chunk ^ ((row >> 1) & 7) : chunk ^ ((row >> 2) & 3);
}
// 16-bit values: the transposing reads take two chunks of 8 rows at a time.
template <int CPR, bool F32>
__device__ __forceinline__ int draft_swz_v(int row, int chunk) {
  if (F32) return draft_swz<CPR>(row, chunk);
  return CPR >= 16 ? chunk ^ ((row & 7) << 1) : CPR == 8 ? chunk ^ (((row >> 1) & 3) << 1) : chunk ^ (((row >> 2) & 1) << 1);
}

__device__ __forceinline__ uint2 draft_read_tr(const char* p) {
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                       (__attribute__((address_space(3))) s16x4*)(const __attribute__((address_space(3))) void*)p));
}

__device__ __forceinline__ DraftReq draft_request(const DraftArgs& a, int b) {
  return draft_req(a.starts[b], a.starts[b + 1], a.lens[b], a.rows);
}

// Where a block's work is.  Every wave works it out from the lengths: with
// `target` units wanted, a chunk is about the same number of tiles everywhere,
// so a long request gets more units than a short one.

// The u-th piece of work where each group of rows of a request of `nch`
// chunks makes per(nch) pieces; false past the last.
template <int KT, int R, bool JOIN, typename F>
__device__ __forceinline__ bool draft_find(const DraftArgs& a, int64_t u, DraftUnit* o, F per) {
  const int lane = threadIdx.x & 63;
  const int cap = a.width << a.page_shift;
  int chunk;
  if constexpr (JOIN) {
    chunk = max(*a.ws_chunk, 1);
  } else {
    float w = 0.f;
    if (a.target > 0) {
      w = draft_lane_tiles(lane, a.B, cap, KT, a.G, R, [&](int b) { return draft_request(a, b); });
      w = add_xor32(add_xor16(row_sum16(w))) * a.Hkv;
    }
    chunk = draft_chunk(w, a.target);
    if (a.target > 0) {
      if (a.B <= 64)
        chunk = draft_widen(chunk, a.target, [&](int c) {
          float units = 0.f;
          if (lane < a.B) {
            const DraftReq r = draft_request(a, lane);
            units = (float)draft_chunks(draft_tiles(r, cap, KT), c) * draft_row_groups(r, a.G, R);
          }
          return add_xor32(add_xor16(row_sum16(units))) * a.Hkv;
        });
      if (blockIdx.x == 0 && threadIdx.x == 0) *a.ws_chunk = chunk;
    }
  }
  int64_t first = 0, slot = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const int b = b0 + lane;
    DraftShare mine = {};
    if (b < a.B) mine = draft_share(draft_request(a, b), cap, KT, a.G, R, a.Hkv, chunk, per);
    int pu = mine.pieces, ps = mine.slots;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      const int x = __shfl_up(pu, m), y = __shfl_up(ps, m);
      if (lane >= m) pu += x, ps += y;
    }
    const uint64_t hit = __ballot(first + pu > u);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      *o = draft_pick(b0 + l, __builtin_amdgcn_readlane(mine.nch, l), __builtin_amdgcn_readlane(mine.tiles, l),
                      __builtin_amdgcn_readlane(mine.groups, l), slot + __builtin_amdgcn_readlane(ps - mine.slots, l),
                      u - first - __builtin_amdgcn_readlane(pu - mine.pieces, l), a.Hkv);
      return true;
    }
    first += __builtin_amdgcn_readlane(pu, 63);
    slot += __builtin_amdgcn_readlane(ps, 63);
  }
  return false;
}

// the unit of this block
template <int KT, int R>
__device__ __forceinline__ bool draft_unit(const DraftArgs& a, DraftUnit* u, DraftPart* p) {
  if (!draft_find<KT, R, false>(a, draft_near(blockIdx.x, a.near), u, [](int nch) { return nch; })) return false;
  *p = draft_unit_part(*u, a.Hkv);
  p->rt = uniform(p->rt), p->ch = uniform(p->ch), p->h = uniform(p->h);
  return true;
}

// 4 consecutive dims of a lane's row: dims dim(q) .. dim(q) + 3, from the
// accumulators of the products' layouts
template <typename T, int D>
struct DraftQuad {
  using S = DraftShape<T, D>;
  static __device__ __forceinline__ int dim(int q, int g) {
    if constexpr (!S::F32) return 16 * q + 4 * g;
    else if constexpr (S::VW == 4) return 64 * (q >> 2) + 16 * g + 4 * (q & 3);
    else return 8 * g + 4 * q;
  }
  static __device__ __forceinline__ f32x4 get(const f32x4 (&o)[S::NQ], int q) {
    if constexpr (!S::F32) return o[q];
    else if constexpr (S::VW == 4) {
      const int t = q & ~3, i = q & 3;
      return f32x4{o[t][i], o[t + 1][i], o[t + 2][i], o[t + 3][i]};
    } else {
      return f32x4{o[0][2 * q], o[1][2 * q], o[0][2 * q + 1], o[1][2 * q + 1]};
    }
  }
  static __device__ __forceinline__ void add(f32x4 (&o)[S::NQ], int q, int e, float x) {
    if constexpr (!S::F32) o[q][e] += x;
    else if constexpr (S::VW == 4) o[(q & ~3) + e][q & 3] += x;
    else o[e & 1][2 * q + (e >> 1)] += x;
  }
};

// whether a 16-byte piece holds an infinite or NaN element (every exponent
// bit set)
template <typename T>
__device__ __forceinline__ bool draft_odd(uint4 x) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      bad |= (w[i] & 0x7f800000u) == 0x7f800000u;
    } else {
      constexpr uint32_t E = std::is_same<T, __bf16>::value ? 0x7f80u : 0x7c00u;
      bad |= (w[i] & E) == E || ((w[i] >> 16) & E) == E;
    }
  }
  return bad;
}

// What a block knows of its unit
struct DraftCtx {
  int s0, ctx, kend, t0, t1, used, shift;
  int full;  // tokens that every row sees, where their pages exist
  int row0, nrow;          // rows (new tokens x heads of the group) from .. to
  const char *kh, *vh;     // the KV head's keys and values
  const int32_t* tab;      // the request's table
  const int32_t* par;      // its new tokens' parents, or null
};
// The pages of a request's tokens, mostly asked for in ascending order: 64 entries
// of the table in a register of the wave's lanes and the next 64 on their way.
// (Read one by one through the scalar cache they held up the LDS reads, which
// count on the same counter.)
struct DraftPages {
  const int32_t* tab;
  int used, num_pages, shift, at, cur, nxt;
  __device__ __forceinline__ int read(int b) const {
    const int i = b * 64 + (int)__lane_id();
    return cache_page(i < used ? tab[i] : -1, num_pages);
  }
  __device__ __forceinline__ DraftPages(const DraftArgs& a, const DraftCtx& c, int key)
      : tab(c.tab), used(c.used), num_pages(a.num_pages), shift(c.shift), at((key >> c.shift) >> 6) {
    cur = read(at);
    nxt = read(at + 1);
  }
  // page of the 16 tokens from `key`, -1: none (past the end, no page of the cache)
  __device__ __forceinline__ int page(int key) {
    const int pi = key >> shift;
    if (pi >> 6 != at) {
      cur = pi >> 6 == at + 1 ? nxt : read(pi >> 6);
      nxt = read((at = pi >> 6) + 1);
    }
    return __builtin_amdgcn_readlane(cur, pi & 63);
  }
};
template <int KT, int R, int STEP>
__device__ __forceinline__ DraftCtx draft_ctx(const DraftArgs& a, const DraftUnit& u, const DraftPart& p, const DraftReq& rq) {
  DraftCtx c;
  c.s0 = uniform(rq.s0), c.ctx = uniform(rq.ctx);
  c.shift = a.page_shift;
  const int even = draft_even(rq, a.G, R, STEP);
  c.row0 = uniform(p.rt * even);
  c.nrow = uniform(min(rq.n * a.G, c.row0 + even));
  const DraftSpan sp = draft_span(rq, c.row0, even, a.G, a.width << a.page_shift, KT, p.ch, u.chunk);
  c.kend = uniform(sp.kend), c.t0 = uniform(sp.t0), c.t1 = uniform(sp.t1);
  c.used = (c.kend + (1 << c.shift) - 1) >> c.shift;
  // rows behind the request's last see nothing, but are not stored either
  c.full = min(a.parents ? c.ctx : c.ctx + c.row0 / a.G + 1, c.kend);
  c.kh = a.k + p.h * a.k_head;
  c.vh = a.v + p.h * a.v_head;
  c.tab = a.table + u.b * a.table_stride;
  c.par = a.parents ? a.parents + c.s0 : nullptr;
  return c;
}

// The lane, not known to be the same each time: the LDS addresses worked out
// from it are not kept in registers across the loop, which has none to spare.
__device__ __forceinline__ int draft_lane_again() {
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));
  return lane;
}

// A wave's rows and their running softmax: 16 MT rows, in the products'
// layout of one row per lane of 16 (column n16), the lane's group g of 4
// holding a quarter of the tokens (scores) or of the dims (output).
template <typename T, int D, int MT, int KT>
struct DraftWave {
  using S = DraftShape<T, D>;
  using Quad = DraftQuad<T, D>;
  static constexpr int NG = KT / 16, CPR = S::CPR, ROWB = S::ROWB, NQ = S::NQ;
  static constexpr int GROUPS = MT, TILE = KT * ROWB;  // of rows; bytes of a tile's keys
  static constexpr bool F32 = S::F32;
  int n16, g, row0;
  f32x4 qf[MT][F32 ? D / 16 : 1];
  bf16x8 qh[MT][F32 ? 1 : D / 32];
  // The weights are exp2(score c + nm): nm is kUp minus the max they are taken
  // against (0 before there is one), in log2 units; a score past `top`, which
  // is the max and kLag, moves it.
  // fp16 has 11 bits of a weight down to 2^-14 and none below 2^-25: there the
  // max weighs 2^11 and moves after 4 (2^15, and what nm and top are rounded by,
  // is below 65504), so that weights down to 2^-25 of the max keep their bits
  // and each is off by half a step, or 2^-36 of the max.  Against a max of 1,
  // 4096 tokens 20 log2 units below one whose values are zero were 1e-2 off.
  // Moving after 4 and not 8 costs a rescale here and there: two chunks of up
  // to 777 tokens over 1500, 8/2 heads of 64, took 27.8 us for 27.4, a prompt of
  // 2048, 32/4 heads of 128, 78.6 for 76.8.
  static constexpr bool F16 = std::is_same<T, _Float16>::value;
  static constexpr float kUp = F16 ? 11.f : 0.f, kLag = F16 ? 4.f : 8.f;
  float nm[MT], top[MT];
  // Where the max is past kFar log2 units, the product's rounding to fp32 no
  // longer leaves a weight where it belongs (half a unit at 2^24, and past 2^31
  // the max's own weight overflows or is zero).  There the max itself, `top`, is
  // subtracted from the scores before the product, and nm is kUp.
  static constexpr float kFar = 4194304.f;  // 2^22
  int was_far;  // some row of the wave has been there (the same in all lanes)
  // the weights' sum: whole for 16-bit types, which have it from a product
  // with ones, a quarter of it in each lane for fp32
  float l[MT];
  f32x4 o[MT][NQ];

  // new token of lane n16's row of group mt, -1 behind the last row
  __device__ __forceinline__ int token(const DraftArgs& a, const DraftCtx& c, int mt, int n16) const {
    const int r = row0 + mt * 16 + n16;
    return r < c.nrow ? r / a.G : -1;
  }
  __device__ __forceinline__ void init(const DraftArgs& a, const DraftCtx& c, int h, int row) {
    const int lane = threadIdx.x & 63;
    n16 = lane & 15, g = lane >> 4, row0 = row;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const int r = row0 + mt * 16 + n16;
      const bool on = r < c.nrow;
      const int j = on ? r / a.G : 0, hg = on ? r - j * a.G : 0;
      const char* p = a.q + (int64_t)(c.s0 + j) * a.q_row + (int64_t)(h * a.G + hg) * a.q_head;
      if constexpr (F32) {
#pragma unroll
        for (int s = 0; s < D / 16; ++s) {
          const int d = 16 * s + 4 * g;
          const f32x4 x = on && d < a.Dk ? *(const f32x4*)(p + d * 4) : f32x4{0.f, 0.f, 0.f, 0.f};
          qf[mt][s] = a.negate ? -x : x;
        }
      } else {
#pragma unroll
        for (int s = 0; s < D / 32; ++s) {
          const int d = 32 * s + 8 * g;
          uint4 x = on && d < a.Dk ? *(const uint4*)(p + d * 2) : make_uint4(0, 0, 0, 0);
          const uint32_t f = a.negate ? 0x80008000u : 0u;
          x.x ^= f, x.y ^= f, x.z ^= f, x.w ^= f;
          qh[mt][s] = __builtin_bit_cast(bf16x8, x);
        }
      }
      nm[mt] = 0.f;
      top[mt] = -INFINITY;
      l[mt] = 0.f;
#pragma unroll
      for (int q = 0; q < NQ; ++q) o[mt][q] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    was_far = 0;
  }

  // whether row mt's token sees the request's token `key` < kend
  __device__ __forceinline__ bool sees(const DraftArgs& a, const DraftCtx& c, int mt, int key) const {
    int j = token(a, c, mt, n16);
    if (j < 0) return false;
    if (!c.par) return key <= c.ctx + j;
    if (key < c.ctx) return true;
    while (j >= 0 && c.ctx + j > key) j = draft_parent(c.par[j], j);
    return j >= 0 && c.ctx + j == key;
  }

  // Scores of one tile of KT tokens from key0, its keys staged at kb, and the
  // rows' max moved where they call for it.  masked: not every row sees every
  // token; there: the tokens (bits) that exist; between(x, n): called after
  // step x of n of the product.
  template <typename F>
  __device__ __forceinline__ void scores(const DraftArgs& a, const DraftCtx& c, const char* kb, int key0,
                                         bool masked, uint64_t there, f32x4 (&sc)[MT][NG], F between) {
    const int lane = draft_lane_again(), n16 = lane & 15, g = lane >> 4;
    // ---- scores, token x row: a lane holds tokens 4 g .. 4 g + 3 of each
    // group of 16, of row n16.  The operands come from LDS four products
    // ahead (left to itself the compiler reads each where it is used, and the
    // wave waits for every one).
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int i = 0; i < NG; ++i) sc[mt][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    __builtin_amdgcn_s_setprio(1);
    {
      constexpr int NS = NG * (F32 ? D / 16 : D / 32), AHEAD = NS < 4 ? NS : 4;
      // (a row's swizzle and the piece's number are bits of their own)
      const uint32_t k0 = n16 * ROWB + draft_swz<CPR>(n16, g) * 16;
      auto key = [&](int x) {  // step x: 16-byte pieces of group x % NG
        return *(const f32x4*)(kb + (k0 ^ (x / NG * 64)) + x % NG * 16 * ROWB);
      };
      f32x4 f[AHEAD];
#pragma unroll
      for (int x = 0; x < AHEAD; ++x) f[x] = key(x);
#pragma unroll
      for (int x = 0; x < NS; ++x) {
        const int i = x % NG, s = x / NG;
        if constexpr (F32) {
          const f32x4 k4 = f[x % AHEAD];
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
              sc[mt][i] = __builtin_amdgcn_mfma_f32_16x16x4f32(k4[e], qf[mt][s][e], sc[mt][i], 0, 0, 0);
        } else {
          using V8 = typename DraftT<T>::V8;
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
            sc[mt][i] = DraftT<T>::mma(__builtin_bit_cast(V8, f[x % AHEAD]), __builtin_bit_cast(V8, qh[mt][s]), sc[mt][i]);
        }
        if (x + AHEAD < NS) f[x % AHEAD] = key(x + AHEAD);
        between(x, NS);
        __builtin_amdgcn_sched_barrier(0);
      }
    }

    __builtin_amdgcn_s_setprio(0);
    // ---- masks
    if (masked) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        uint64_t see = 0;
        const int tok = token(a, c, mt, n16);
        if (tok >= 0) {
          if (c.par) {
            const int c0 = min(max(c.ctx - key0, 0), 64);  // cached tokens of the tile
            see = c0 == 64 ? ~0ull : (1ull << c0) - 1;
            for (int j = tok; j >= 0 && c.ctx + j >= key0;) {
              if (c.ctx + j - key0 < KT) see |= 1ull << (c.ctx + j - key0);
              j = draft_parent(c.par[j], j);
            }
          } else {
            const int c1 = min(max(c.ctx + tok + 1 - key0, 0), 64);
            see = c1 == 64 ? ~0ull : (1ull << c1) - 1;
          }
        }
        see &= there;
#pragma unroll
        for (int i = 0; i < NG; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!((see >> (16 * i + 4 * g + e)) & 1)) sc[mt][i][e] = -INFINITY;
      }
    }

    // ---- running softmax.  The max that a row's weights are taken against
    // only moves when a score passes it by kLag: the output is seldom rescaled,
    // and the lanes of a row seldom have to compare their scores.
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < NG; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) mx = fmaxf(mx, sc[mt][i][e]);
      if (__any(mx > top[mt])) {
        mx = max_xor32(max_xor16(mx));
        float t = mx + kLag * a.inv_c;
        if (__any(mx > top[mt] && fabsf(t) * a.c >= kFar)) was_far = 1;
        if (mx > top[mt]) {
          float mn = kUp - mx * a.c, al = mn - nm[mt];
          if (was_far) {
            const bool was = far(a, mt);
            if (was) al = top[mt] * a.c - mx * a.c;
            if (fabsf(t) * a.c >= kFar) {
              t = mx;
              if (was) al = (top[mt] - mx) * a.c;
              if (fabsf(mx) * a.c >= kFar) mn = kUp;
            }
          }
          // (before the first score there is nothing to rescale, but NaN stays)
          al = top[mt] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(al);
          nm[mt] = mn;
          top[mt] = t;
          l[mt] *= al;
#pragma unroll
          for (int q = 0; q < NQ; ++q) o[mt][q] *= al;
        }
      }
    }
    if (was_far) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const float m = far(a, mt) ? top[mt] : 0.f;
#pragma unroll
        for (int i = 0; i < NG; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[mt][i][e] -= m;
      }
    }
  }

  // The weights of the tile's tokens and their values, staged at vb.  Output,
  // dim x row: the tokens of a product's k index are those a lane holds, so the
  // weights' registers are its second operand as they are.
  __device__ __forceinline__ void values(const DraftArgs& a, const char* vb, f32x4 (&sc)[MT][NG]) {
    const int lane = draft_lane_again(), n16 = lane & 15, g = lane >> 4;
    auto weigh = [&](int mt, int i, int e) {
      sc[mt][i][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[mt][i][e], a.c, nm[mt]));
    };
    if constexpr (F32) {
      // a step: the dims of one read (VW a lane) times the lane's token e of
      // group i.  The weights of the next group go into the products' shadow.
      constexpr int VW = S::VW, QS = NQ / VW, NS = NG * 4 * QS, AHEAD = 4;
      f32x4 f[AHEAD];
      auto value = [&](int x) {
        const int row = 16 * (x / QS / 4) + 4 * g + x / QS % 4, q = x % QS * VW;
        if constexpr (VW == 4) {
          f[x % AHEAD] = *(const f32x4*)(vb + row * ROWB + draft_swz_v<CPR, F32>(row, 4 * q + n16) * 16);
        } else {
          const f32x2 y = *(const f32x2*)(vb + row * ROWB + draft_swz_v<CPR, F32>(row, n16 >> 1) * 16 + (n16 & 1) * 8);
          f[x % AHEAD] = f32x4{y[0], y[1], 0.f, 0.f};
        }
      };
      auto weights = [&](int i, int e) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          weigh(mt, i, e);
          l[mt] += sc[mt][i][e];
        }
      };
#pragma unroll
      for (int x = 0; x < AHEAD; ++x) value(x);
#pragma unroll
      for (int e = 0; e < 4; ++e) weights(0, e);
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int x = 0; x < NS; ++x) {
        const int i = x / QS / 4, e = x / QS % 4, q = x % QS * VW;
        const f32x4 v = f[x % AHEAD];
#pragma unroll
        for (int w = 0; w < VW; ++w)
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
            o[mt][q + w] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[w], sc[mt][i][e], o[mt][q + w], 0, 0, 0);
        if (x + AHEAD < NS) value(x + AHEAD);
        if (x % QS == 0 && i + 1 < NG) weights(i + 1, e);
        __builtin_amdgcn_sched_barrier(0);
      }
      __builtin_amdgcn_s_setprio(0);
    } else {
      // a transposing read gives lane n16 of group g four tokens of dim n16:
      // it addresses token 4 g + n16 / 4, dims 4 (n16 % 4) ..
      const int row = 4 * g + (n16 >> 2);
      const uint32_t v0 = row * ROWB + draft_swz_v<CPR, F32>(row, (n16 & 3) >> 1) * 16 + (n16 & 1) * 8;
      auto col = [&](int i, int q) { return draft_read_tr(vb + (v0 ^ (q * 32)) + i * 16 * ROWB); };
      // Products of PG groups of 16 tokens at a time, the operands four products
      // ahead.  The weights of the first tokens come before them, those of the
      // next in their shadow: a product holds the matrix unit for four times as
      // long as it holds the wave.
      constexpr int PG = NG == 1 ? 1 : 2, NS = NG / PG * NQ, AHEAD = NS < 4 ? NS : 4;
      constexpr int EL = PG * 4 * MT, EPS = (EL + NQ - 1) / NQ;  // weights of a product's tokens, of a step
      uint2 f[AHEAD][PG];
      auto value = [&](int x) {  // step x: dims x % NQ, groups from x / NQ
#pragma unroll
        for (int y = 0; y < PG; ++y) f[x % AHEAD][y] = col(x / NQ * PG + y, x % NQ);
      };
#pragma unroll
      for (int x = 0; x < AHEAD; ++x) value(x);
      // P rounded to the values' type, which halves the products that a second
      // part of P would take.  Each weight is off by half a step (fp16: or by
      // 2^-36 of the max's), so the output by half a step of
      // sum p |v| / sum p + |output| at most, and mostly by the square root of
      // the tokens' number less.  The sum is taken of the rounded P too, so that
      // the weights still add up to one.
      uint2 p[MT][PG];
      auto round = [&](int i0) {
        typedef __attribute__((ext_vector_type(4))) T T4;
        constexpr uint32_t one = std::is_same<T, __bf16>::value ? 0x3f803f80u : 0x3c003c00u;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
          for (int y = 0; y < PG; ++y) p[mt][y] = __builtin_bit_cast(uint2, __builtin_convertvector(sc[mt][i0 + y], T4));
          f32x4 sum = {0.f, 0.f, 0.f, 0.f};
          l[mt] += product(make_uint2(one, one), make_uint2(one, one), p[mt][0], p[mt][PG - 1], sum)[0];
        }
      };
#pragma unroll
      for (int x = 0; x < EL; ++x) weigh(x / (PG * 4), x / 4 % PG, x % 4);
      round(0);
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int x = 0; x < NS; ++x) {
        const int q = x % NQ, i0 = x / NQ * PG;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
          o[mt][q] = product(f[x % AHEAD][0], f[x % AHEAD][PG - 1], p[mt][0], p[mt][PG - 1], o[mt][q]);
        if (x + AHEAD < NS) value(x + AHEAD);
        if (i0 + PG < NG) {
#pragma unroll
          for (int y = q * EPS; y < (q + 1) * EPS && y < EL; ++y) weigh(y / (PG * 4), i0 + PG + y / 4 % PG, y % 4);
        }
        __builtin_amdgcn_sched_barrier(0);
        if (q == NQ - 1 && i0 + PG < NG) round(i0 + PG);
      }
      __builtin_amdgcn_s_setprio(0);
    }
  }

  // a product over 32 tokens (two groups of 16), or 16 where a tile has no more
  static __device__ __forceinline__ f32x4 product(uint2 a0, uint2 a1, uint2 b0, uint2 b1, f32x4 c) {
    if constexpr (NG == 1) {
      return DraftT<T>::mma_k16(__builtin_bit_cast(s16x4, a0), __builtin_bit_cast(s16x4, b0), c);
    } else {
      using V8 = typename DraftT<T>::V8;
      return DraftT<T>::mma(__builtin_bit_cast(V8, make_uint4(a0.x, a0.y, a1.x, a1.y)),
                            __builtin_bit_cast(V8, make_uint4(b0.x, b0.y, b1.x, b1.y)), c);
    }
  }

  // Adds what the rows that see token `key` take of it, where its values are
  // infinite or NaN and were staged as zeros (l has its weight already).
  __device__ __forceinline__ void odd_token(const DraftArgs& a, const DraftCtx& c, int key, int page) {
    const int at = key & ((1 << c.shift) - 1);
    const T* kp = (const T*)(c.kh + page * a.k_page + at * a.k_token);
    const T* vp = (const T*)(c.vh + page * a.v_page + at * a.v_token);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      if (!__any(sees(a, c, mt, key))) continue;
      float x = 0.f;  // the row's score, a quarter of it in each lane
#pragma unroll
      for (int s = 0; s < (F32 ? D / 16 : D / 32); ++s)
#pragma unroll
        for (int e = 0; e < (F32 ? 4 : 8); ++e) {
          const int d = F32 ? 16 * s + 4 * g + e : 32 * s + 8 * g + e;
          if (d < a.Dk) x += q_at(mt, s, e) * Io<T>::ld(kp + d);
        }
      x = add_xor32(add_xor16(x));
      const bool see = sees(a, c, mt, key);
      // (the sum's order is another than the product's: past kFar a score could
      // pass the max by more than a weight can hold)
      const float p = __builtin_amdgcn_exp2f((far(a, mt) ? fminf(x - top[mt], 0.f) * a.c : x * a.c) + nm[mt]);
#pragma unroll
      for (int q = 0; q < NQ; ++q)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int d = Quad::dim(q, g) + e;
          if (see && d < a.Dv) Quad::add(o[mt], q, e, p * Io<T>::ld(vp + d));
        }
    }
  }
  __device__ __forceinline__ float q_at(int mt, int s, int e) const {
    if constexpr (F32) return qf[mt][s][e];
    else return (float)__builtin_bit_cast(typename DraftT<T>::V8, qh[mt][s])[e];
  }

  // the sum and max (log2 units, less kUp; -inf: none) of row n16 of group mt
  __device__ __forceinline__ float sum(int mt) const {
    return F32 ? add_xor32(add_xor16(l[mt])) : l[mt];
  }
  __device__ __forceinline__ float peak(const DraftArgs& a, int mt) const {
    return top[mt] == -INFINITY ? -INFINITY : far(a, mt) ? top[mt] * a.c - kUp : -nm[mt];
  }
  // whether the max is past kFar (`top` is then the max itself)
  __device__ __forceinline__ bool far(const DraftArgs& a, int mt) const {
    return fabsf(top[mt]) * a.c >= kFar && top[mt] != -INFINITY;
  }

  // the lane's part of row n16 of group mt, times f, into 16 fp32 rows at dst
  __device__ __forceinline__ void put(float* dst, int mt, float f) const {
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      const int ch = Quad::dim(q, g) >> 2;
      *(f32x4*)(dst + n16 * D + ((ch ^ (n16 & S::OS)) << 2)) = Quad::get(o[mt], q) * f;
    }
  }
};

// one chunk of 4 dims of a row, as put() left it
template <typename T, int D>
__device__ __forceinline__ f32x4 draft_got(const float* src, int row, int ch) {
  return *(const f32x4*)(src + row * D + ((ch ^ (row & DraftShape<T, D>::OS)) << 2));
}

// The kernel's arguments, read again: what is needed after the loop over the
// tiles is not kept in scalar registers (spilled to vector lanes) across it.
__device__ __forceinline__ const DraftArgs& draft_args_again() {
  auto p = (const __attribute__((address_space(4))) DraftArgs*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const DraftArgs*)p;
}

// Whether a token's values (row vp of Dv) hold an infinite or NaN one.
template <typename T>
__device__ __forceinline__ bool draft_odd_row(const DraftArgs& a, const char* vp) {
  const int lane = threadIdx.x & 63;
  const bool in = lane * 16 < a.Dv * (int)sizeof(T);
  return __any(in && draft_odd<T>(*(const uint4*)(vp + (in ? lane * 16 : 0))));
}

// stores chunk ch of the request's row r (x: weighted sum, sum: the weights')
template <typename T>
__device__ __forceinline__ void draft_store(const DraftArgs& a, int s0, int h, int r, int ch, f32x4 x, float sum) {
  if (ch * 4 >= a.Dv) return;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;  // a row that sees nothing is zero
  const int j = r / a.G, hg = r - j * a.G;
  typedef __attribute__((ext_vector_type(4))) T T4;
  *(T4*)(a.out + (int64_t)(s0 + j) * a.o_row + (int64_t)(h * a.G + hg) * a.o_head + ch * 4 * sizeof(T)) =
      __builtin_convertvector(x * inv, T4);
}

// Few rows: the four waves of a block have the same 16 MT rows and take the
// chunk's tiles in turn, each through LDS of its own, so that there is no
// barrier before their states meet.  While it works on a tile a wave has the
// loads of its next one in flight: 16 KB a wave, 128 KB a CU.
template <typename T, int D, int MT>
__global__ __launch_bounds__(256, draft_two(D, MT, sizeof(T)) ? 2 : 1) void draft_kernel(DraftArgs a) {
  using S = DraftShape<T, D>;
  constexpr int KT = draft_tile(D, S::ES), NG = KT / 16, CPR = S::CPR, RPI = S::RPI, R = 16 * MT;
  constexpr int NI = KT / RPI, ROWB = S::ROWB, NW = kWavesPerBlock;
  constexpr int WAVE_LDS = 2 * KT * ROWB;
  __shared__ __attribute__((aligned(1024))) char lds[NW * WAVE_LDS];
  __shared__ float ml[NW][R][2];

  DraftUnit u;
  DraftPart part;
  if (!draft_unit<KT, R>(a, &u, &part)) return;  // uniform over the block
  const int lane = threadIdx.x & 63, wv = uniform(threadIdx.x >> 6);
  const DraftReq rq = draft_request(a, u.b);
  const DraftCtx c = draft_ctx<KT, R, 16 * MT>(a, u, part, rq);
  const int row0 = c.row0;
  DraftWave<T, D, MT, KT> w;
  w.init(a, c, part.h, row0);

  char* kb = lds + wv * WAVE_LDS;
  char* vb = kb + KT * ROWB;
  const int lr = lane / CPR, lc = lane % CPR;
  // lanes past the head dim read the row's first chunk and write zeros
  const bool kin = lc * 16 < a.Dk * S::ES, vin = lc * 16 < a.Dv * S::ES;
  const bool whole = a.Dk == D && a.Dv == D;
  const uint32_t koff = lr * (uint32_t)a.k_token + (kin ? lc * 16 : 0);
  const uint32_t voff = lr * (uint32_t)a.v_token + (vin ? lc * 16 : 0);

  DraftPages pg(a, c, (c.t0 + wv) * KT);
  auto pages_of = [&](DraftPages& p, int t, int (&e)[NG]) {
#pragma unroll
    for (int i = 0; i < NG; ++i) e[i] = p.page(t * KT + 16 * i);
  };
  auto pages = [&](int t, int (&e)[NG]) { pages_of(pg, t, e); };
  uint4 kr[NI], vr[NI];
  auto load_k = [&](int t, const int (&e)[NG]) {
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      const char* p = c.kh + (int64_t)max(e[i], 0) * a.k_page + ((t * KT + 16 * i) & ((1 << c.shift) - 1)) * a.k_token;
#pragma unroll
      for (int x = 0; x < NI / NG; ++x) kr[i * (NI / NG) + x] = *(const uint4*)(p + x * RPI * a.k_token + koff);
    }
  };
  auto load_v = [&](int t, const int (&e)[NG]) {
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      const char* p = c.vh + (int64_t)max(e[i], 0) * a.v_page + ((t * KT + 16 * i) & ((1 << c.shift) - 1)) * a.v_token;
#pragma unroll
      for (int x = 0; x < NI / NG; ++x) vr[i * (NI / NG) + x] = *(const uint4*)(p + x * RPI * a.v_token + voff);
    }
  };

  // The lane again, for places in LDS: at D 32 in 16 bits a third block of 32
  // rows fits a CU then (168 registers; 2000 requests of up to 900 tokens, 64/4
  // heads, fp16: 414 us, with two blocks 557).  Elsewhere LDS allows no more
  // blocks, and kept places are up to 2% faster (fp32 at D 32).
  auto place = [&]() { return D == 32 && !S::F32 ? draft_lane_again() : lane; };
  // the staged tile into LDS; the loads of the wave's next one go out
  int ent[NG], nxt[NG];
  int t = c.t0 + wv;
  auto stage = [&]() {
    const int lane2 = place(), lr = lane2 / CPR, lc = lane2 % CPR;
    if (!whole) {
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        if (!kin) kr[i] = make_uint4(0, 0, 0, 0);
        if (!vin) vr[i] = make_uint4(0, 0, 0, 0);
      }
    }
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int row = i * RPI + lr;
      *(uint4*)(kb + row * ROWB + draft_swz<CPR>(row, lc) * 16) = kr[i];
      *(uint4*)(vb + row * ROWB + draft_swz_v<CPR, S::F32>(row, lc) * 16) = vr[i];
    }
#pragma unroll
    for (int i = 0; i < NG; ++i) ent[i] = nxt[i];
    if (t + NW < c.t1) {
      load_k(t + NW, ent);
      load_v(t + NW, ent);
    }
    pages(t + 2 * NW, nxt);
    wave_sync();
  };
  // tiles that some row does not see all of: past `full`, or pages missing
  auto masked = [&]() {
    bool x = (t + 1) * KT > c.full;
#pragma unroll
    for (int i = 0; i < NG; ++i) x |= ent[i] < 0;
    return x;
  };
  // tokens (bits) of tile t that exist
  auto exist = [&]() {
    uint64_t x = 0;
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      const int left = min(max(c.kend - t * KT - 16 * i, 0), 16);
      if (ent[i] >= 0) x |= (uint64_t)((1u << left) - 1u) << (16 * i);
    }
    return x;
  };
  pages(t, ent);
  pages(t + NW, nxt);
  if (t < c.t1) {
    load_k(t, ent);
    load_v(t, ent);
  }
  bool odd = false;  // a token with infinite or NaN values was met
  for (; t < c.t1; t += NW) {
    const bool some = masked();
    uint64_t there = 0;
    if (some) {
      there = exist();
      // Values that a row does not see must not meet the product: 0 x NaN is
      // NaN.  Zeros take the place of those that no row sees, and of
      // infinite or NaN ones, which join at the end.
      const int lr = place() / CPR;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int row = i * RPI + lr;
        if (!((there >> row) & 1)) vr[i] = make_uint4(0, 0, 0, 0);
        const uint64_t hit = __ballot(draft_odd<T>(vr[i]) && vin);
        odd |= hit != 0;
        if ((hit >> (lr * CPR)) & (CPR == 64 ? ~0ull : (1ull << (CPR & 63)) - 1)) vr[i] = make_uint4(0, 0, 0, 0);
      }
    }
    stage();
    f32x4 sc[MT][NG];
    w.scores(a, c, kb, t * KT, some, there, sc, [](int, int) {});
    w.values(a, vb, sc);
    wave_sync();  // this tile's reads come before the next one's writes
  }
  const DraftArgs& z = draft_args_again();
  if (odd) {
    DraftPages again(z, c, (c.t0 + wv) * KT);
    for (t = c.t0 + wv; t < c.t1; t += NW) {
      pages_of(again, t, ent);
      if (!masked()) continue;
      for (uint64_t left = exist(); left; left &= left - 1) {
        const int key = t * KT + __builtin_ctzll(left), p = again.page(key);
        if (draft_odd_row<T>(z, c.vh + p * z.v_page + (key & ((1 << c.shift) - 1)) * z.v_token))
          w.odd_token(z, c, key, p);
      }
    }
  }

  // ---- the four waves' states meet
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const float sum = w.sum(mt);
    if (w.g == 0) {
      ml[wv][mt * 16 + w.n16][0] = w.peak(z, mt);
      ml[wv][mt * 16 + w.n16][1] = sum;
    }
  }
  __syncthreads();
  const int64_t slot = part.slot;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    float mm = -INFINITY;
#pragma unroll
    for (int i = 0; i < NW; ++i) mm = fmaxf(mm, ml[i][mt * 16 + w.n16][0]);
    // a wave that saw no token of the row adds nothing (NaN scores leave the
    // max alone and make sums NaN, which stay)
    const float pk = w.peak(z, mt);
    w.put((float*)(lds + wv * WAVE_LDS), mt, pk == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(pk - mm));
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * S::OC; i += 256) {
      const int row = i / S::OC, ch = i % S::OC, rr = mt * 16 + row;
      if (row0 + rr >= c.nrow) continue;
      f32x4 x = {0.f, 0.f, 0.f, 0.f};
      float big = -INFINITY, sum = 0.f;
#pragma unroll
      for (int j = 0; j < NW; ++j) big = fmaxf(big, ml[j][rr][0]);
#pragma unroll
      for (int j = 0; j < NW; ++j) {
        x += draft_got<T, D>((const float*)(lds + j * WAVE_LDS), row, ch);
        const float mj = ml[j][rr][0];
        sum += mj == -INFINITY ? ml[j][rr][1] : ml[j][rr][1] * __builtin_amdgcn_exp2f(mj - big);
      }
      if (slot >= 0) {
        *(f32x4*)(z.ws_o + (slot * R + rr) * D + ch * 4) = x;
        if (ch == 0) {
          z.ws_ml[(slot * R + rr) * 2] = big;
          z.ws_ml[(slot * R + rr) * 2 + 1] = sum;
        }
      } else {
        draft_store<T>(z, c.s0, part.h, row0 + rr, ch, x, sum);
      }
    }
    __syncthreads();
  }
}

// 16 bytes of each lane into LDS, from `to` on in the order of the lanes
__device__ __forceinline__ void draft_copy16(const char* from, char* to) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from, (lds_void*)to, 16, 0, 0);
}

// A tile, while the next is copied: copy(next, i), i < COPIES, a piece at a
// time between the products (all at once the copies held the wave for as long
// as either product).  The buffers do not overlap and are said not to: else
// the reads of one wait for the copies into the other.
template <int COPIES, typename W, typename F>
__device__ __forceinline__ void draft_step(const DraftArgs& a, const DraftCtx& c, W& w, int key0, bool masked,
                                           uint64_t there, bool on, const char* __restrict__ now,
                                           char* __restrict__ next, F copy) {
  if (!on) {
#pragma unroll
    for (int i = 0; i < COPIES; ++i) copy(next, i);
    return;
  }
  f32x4 sc[W::GROUPS][W::NG];
  w.scores(a, c, now, key0, masked, there, sc, [&](int x, int n) {
#pragma unroll
    for (int i = 0; i < COPIES; ++i)
      if (i * n / COPIES == x) copy(next, i);
  });
  w.values(a, now + W::TILE, sc);
}

// Many rows: each wave of a block has 16 MT rows of its own, and all of them
// take the same tiles, which the block copies into one of two LDS buffers
// (directly, without registers) while it works on the other: one barrier a
// tile.  One request of 131008 tokens, 64 drafted, 64/8 heads of 128, bf16:
// 718 us with 64 rows and tiles of a wave's own, 366 with common tiles, 322
// with the copies straight into LDS, 303 with them spread between the products
// and the waves' priority raised there.
// WHOLE: the head dims are D.
template <typename T, int D, int MT, int NW, int KT, bool WHOLE>
__global__ __launch_bounds__(64 * NW, D <= 128 ? 2 : 1) void draft_rows_kernel(DraftArgs a) {
  using S = DraftShape<T, D>;
  using W = DraftWave<T, D, MT, KT>;
  constexpr int NG = KT / 16, CPR = S::CPR, RPI = S::RPI, R = 16 * MT * NW, ROWB = S::ROWB;
  constexpr int WR = KT / NW;       // rows that a wave copies, in one page
  constexpr int NI = WR / RPI;
  static_assert(WR <= 16 && NI >= 1 && KT <= 64, "a wave copies rows of one page");
  constexpr int STAGE = 2 * KT * ROWB;
  constexpr int PUT = NW * 16 * D * 4;  // the output passes through, 16 rows of each wave
  constexpr int BUF = 2 * STAGE > PUT ? STAGE : PUT / 2;
  __shared__ __attribute__((aligned(1024))) char lds0[BUF];
  __shared__ __attribute__((aligned(1024))) char lds1[BUF];
  __shared__ int odds[NW];

  DraftUnit u;
  DraftPart part;
  if (!draft_unit<KT, R>(a, &u, &part)) return;  // uniform over the block
  const int lane = threadIdx.x & 63, wv = uniform(threadIdx.x >> 6);
  const DraftReq rq = draft_request(a, u.b);
  const DraftCtx c = draft_ctx<KT, R, 16 * MT>(a, u, part, rq);
  const int row0 = c.row0 + wv * 16 * MT;
  const bool on = row0 < c.nrow;  // the wave has rows
  W w;
  w.init(a, c, part.h, row0);

  const int lr = lane / CPR, lc = lane % CPR;
  const int r0 = wv * WR;  // first of the rows this wave copies
  const int kbytes = a.Dk * S::ES, vbytes = a.Dv * S::ES;
  if (!WHOLE) {
    // the places past the head dims: no copy writes them
    for (int i = threadIdx.x * 16; i < STAGE; i += 64 * NW * 16) {
      *(uint4*)(lds0 + i) = make_uint4(0, 0, 0, 0);
      *(uint4*)(lds1 + i) = make_uint4(0, 0, 0, 0);
    }
    __syncthreads();
  }

  // Lane x of a copy writes piece x of a KB of LDS: it reads the piece that
  // belongs there.
  const int row1 = r0 + lr, kc1 = draft_swz<CPR>(row1, lc), vc1 = draft_swz_v<CPR, S::F32>(row1, lc);
  const uint32_t kl = lr * (uint32_t)a.k_token, vl = lr * (uint32_t)a.v_token;
  const char *kp, *vp;  // of the rows to copy
  auto aim = [&](int t, int e) {
    const int at = (t * KT + r0) & ((1 << c.shift) - 1);
    kp = c.kh + (int64_t)max(e, 0) * a.k_page + at * a.k_token;
    vp = c.vh + (int64_t)max(e, 0) * a.v_page + at * a.v_token;
  };
  auto copy = [&](char* buf, int i) {
    // row row1 + x RPI: x's part of the swizzle has bits of its own
    const int x = i >> 1;
    const int kc = (kc1 ^ draft_swz<CPR>(x * RPI, 0)) * 16, vc = (vc1 ^ draft_swz_v<CPR, S::F32>(x * RPI, 0)) * 16;
    char* to = buf + (r0 + x * RPI) * ROWB;
    if (i & 1) {
      if (WHOLE || vc < vbytes) draft_copy16(vp + x * RPI * a.v_token + (vl + vc), to + KT * ROWB);
    } else {
      if (WHOLE || kc < kbytes) draft_copy16(kp + x * RPI * a.k_token + (kl + kc), to);
    }
  };
  DraftPages pg(a, c, c.t0 * KT);
  // the page of the rows that this wave copies (a tile's pages are in one
  // batch of entries)
  auto mine = [&](int t) { return pg.page(t * KT + r0 / 16 * 16); };
  // groups of 16 tokens of a tile without a page
  auto missing = [&](DraftPages& p, int t) {
    uint32_t x = 0;
#pragma unroll
    for (int i = 0; i < NG; ++i) x |= p.page(t * KT + 16 * i) < 0 ? 1u << i : 0u;
    return x;
  };
  // tokens (bits) of tile t that exist
  auto exist = [&](int t, uint32_t gone) {
    uint64_t x = 0;
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      const int left = min(max(c.kend - t * KT - 16 * i, 0), 16);
      if (!((gone >> i) & 1)) x |= (uint64_t)((1u << left) - 1u) << (16 * i);
    }
    return x;
  };
  // whether some row does not see all of tile t
  auto masked = [&](int t, uint32_t gone) { return (t + 1) * KT > c.full || gone != 0; };

  bool odd = false;  // this wave copied a token with infinite or NaN values
  int t = c.t0;
  if (t < c.t1) {
    aim(t, mine(t));
#pragma unroll
    for (int i = 0; i < 2 * NI; ++i) copy(lds0, i);
  }
  auto step = [&](char* now, char* next) {
    const uint32_t gone = missing(pg, t);
    const bool some = masked(t, gone);
    // (past the last tile: this one again, which no one reads)
    const int t2 = min(t + 1, c.t1 - 1);
    aim(t2, mine(t2));
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wave's copies have landed
    __syncthreads();                     // all have, and the other buffer's readers are done
    uint64_t there = 0;
    if (some) {
      // Values that a row does not see must not meet the product: 0 x NaN is
      // NaN.  Each wave puts zeros in the place of those it copied that no row
      // sees, and of infinite or NaN ones, which join at the end.
      there = exist(t, gone);
      const int lane2 = draft_lane_again();
#pragma unroll
      for (int x = 0; x < NI; ++x) {
        const int row = r0 + x * RPI + lane2 / CPR;
        uint4* p = (uint4*)(now + W::TILE + row * ROWB + lane2 % CPR * 16);
        const bool in = (there >> row) & 1;
        const uint64_t hit = __ballot(in && draft_odd<T>(*p));
        odd |= hit != 0;
        if (!in || ((hit >> (lane2 / CPR * CPR)) & (CPR == 64 ? ~0ull : (1ull << (CPR & 63)) - 1)))
          *p = make_uint4(0, 0, 0, 0);
      }
      __syncthreads();
    }
    draft_step<2 * NI>(a, c, w, t * KT, some, there, on, now, next, copy);
    return ++t < c.t1;
  };
  if (t < c.t1)
    while (step(lds0, lds1) && step(lds1, lds0)) {
    }
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): the output passes through the buffers
  const DraftArgs& z = draft_args_again();
  if (lane == 0) odds[wv] = odd;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NW; ++i) odd |= odds[i] != 0;
  if (odd && on) {
    DraftPages again(z, c, c.t0 * KT);
    for (t = c.t0; t < c.t1; ++t) {
      const uint32_t gone = missing(again, t);
      if (!masked(t, gone)) continue;
      for (uint64_t left = exist(t, gone); left; left &= left - 1) {
        const int key = t * KT + __builtin_ctzll(left), p = again.page(key);
        if (draft_odd_row<T>(z, c.vh + p * z.v_page + (key & ((1 << c.shift) - 1)) * z.v_token))
          w.odd_token(z, c, key, p);
      }
    }
  }
  __syncthreads();

  const int64_t slot = part.slot;
  float* my = (float*)(wv < NW / 2 ? lds0 : lds1) + wv % (NW / 2) * 16 * D;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const float l = w.sum(mt), m = w.peak(z, mt);
    w.put(my, mt, 1.f);
    wave_sync();
#pragma unroll
    for (int i = lane; i < 16 * S::OC; i += 64) {
      const int row = i / S::OC, ch = i % S::OC;
      const int r = row0 + mt * 16 + row;
      const float big = __shfl(m, row), sum = __shfl(l, row);
      const f32x4 x = draft_got<T, D>(my, row, ch);
      if (r >= c.nrow) continue;
      if (slot >= 0) {
        const int64_t at = slot * R + wv * 16 * MT + mt * 16 + row;
        *(f32x4*)(z.ws_o + at * D + ch * 4) = x;
        if (ch == 0) {
          z.ws_ml[at * 2] = big;
          z.ws_ml[at * 2 + 1] = sum;
        }
      } else {
        draft_store<T>(z, c.s0, part.h, r, ch, x, sum);
      }
    }
    wave_sync();
  }
}

// Joins the chunks of split requests.  The threads of a block are NP sets of
// D / 4, a set holding a row.  Few chunks: each set takes a row and all its
// chunks; many chunks, or few rows in all: the block takes a row and its sets
// share the chunks.  Bound by the read of the states, and by the launch: 512
// states of 128 rows of 128 (34 MB) 11 us, those of a single token 4.7 us.
constexpr int kJoinSerial = 16;  // or as many as a set has threads
template <typename T, int D, int KT, int R, int STEP>
__global__ __launch_bounds__(256) void draft_join_kernel(DraftArgs a) {
  constexpr int OC = D / 4, NP = 256 / OC;
  __shared__ f32x4 acc[256];
  __shared__ float lsum[NP];
  const int tid = threadIdx.x, p = tid / OC, ch = tid % OC;
  const int most = a.one_round ? 0 : kJoinSerial < OC ? kJoinSerial : OC;
  for (int64_t at = blockIdx.x;; at += gridDim.x) {
    DraftUnit u;
    if (!draft_find<KT, R, true>(a, at, &u, [&](int nch) { return draft_join_pieces(nch, most, R, NP); }))
      return;  // uniform over the block
    const DraftReq rq = draft_request(a, u.b);
    const DraftJoin j = draft_join(u, rq, a.G, a.Hkv, R, STEP, NP, most);
    // (rows of a block ascend: the first one behind the last ends it)
    if (j.r0 + j.row >= j.nrow) {
      if (a.one_round) return;
      continue;
    }
    const bool serial = j.serial;
    const int rr = serial ? j.row + p : j.row, r = j.r0 + rr, h = j.h;
    const bool on = r < j.nrow;
    const int64_t base = j.base, step = j.step;
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
    float sum = 0.f;
    // (a chunk whose tokens the row does not see has max -inf and zeros)
    if (serial) {
      // a lane of the set has a chunk's max and sum
      float mc = -INFINITY, lc = 0.f;
      if (on && ch < u.nch) {
        const float* ml = a.ws_ml + ((base + ch * step) * R + rr) * 2;
        mc = ml[0], lc = ml[1];
      }
      float big = mc;
#pragma unroll
      for (int m = 1; m < OC; m <<= 1) big = fmaxf(big, __shfl_xor(big, m));
      const float f = mc == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mc - big);
      sum = lc * f;
#pragma unroll
      for (int m = 1; m < OC; m <<= 1) sum += __shfl_xor(sum, m);
#pragma unroll 8
      for (int c = 0; c < u.nch; ++c) {
        const float fc = __shfl(f, (tid & 63) / OC * OC + c);
        if (on) x += *(const f32x4*)(a.ws_o + ((base + c * step) * R + rr) * D + ch * 4) * fc;
      }
    } else {
      float big = -INFINITY;
      for (int c = tid & 63; c < u.nch; c += 64) big = fmaxf(big, a.ws_ml[((base + c * step) * R + rr) * 2]);
      big = wave_max(big);
#pragma unroll 4
      for (int c = p; c < u.nch; c += NP) {
        const int64_t i = (base + c * step) * R + rr;
        const float mc = a.ws_ml[i * 2], lc = a.ws_ml[i * 2 + 1];
        const f32x4 oc = *(const f32x4*)(a.ws_o + i * D + ch * 4);
        const float f = mc == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mc - big);
        x += oc * f;
        sum += lc * f;
      }
      acc[tid] = x;
      if (ch == 0) lsum[p] = sum;
      __syncthreads();
      if (p == 0) {
#pragma unroll
        for (int i = 1; i < NP; ++i) {
          x += acc[i * OC + ch];
          sum += lsum[i];
        }
      }
      __syncthreads();
    }
    if (on && (serial || p == 0)) draft_store<T>(a, rq.s0, h, r, ch, x, sum);
    if (a.one_round) return;
  }
}

template <typename T, int D, int MT, int NW>
int draft_launch(const DraftArgs& a, int64_t units, int64_t joins, hipStream_t st) {
  constexpr int KT = draft_tile(D, (int)sizeof(T), NW), R = 16 * MT * NW;
  if constexpr (NW == 1)
    hipLaunchKernelGGL((draft_kernel<T, D, MT>), dim3((unsigned)units), dim3(256), 0, st, a);
  else if (a.Dk == D && a.Dv == D)
    hipLaunchKernelGGL((draft_rows_kernel<T, D, MT, NW, KT, true>), dim3((unsigned)units), dim3(64 * NW), 0, st, a);
  else
    hipLaunchKernelGGL((draft_rows_kernel<T, D, MT, NW, KT, false>), dim3((unsigned)units), dim3(64 * NW), 0, st, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return (int)e;
  if (joins > 0) {
    hipLaunchKernelGGL((draft_join_kernel<T, D, KT, R, 16 * MT>), dim3((unsigned)joins), dim3(256), 0, st, a);
    e = hipGetLastError();
  }
  return e == hipSuccess ? HTREE_OK : (int)e;
}

template <typename T>
int draft_launch_type(const DraftArgs& a, const DraftPlan& p, hipStream_t st);

template <typename T, int D>
int draft_launch_dim(const DraftArgs& a, const DraftPlan& p, hipStream_t st) {
  if constexpr (sizeof(T) == 2) {
    if (p.NW > 1) return draft_launch<T, D, 2, 4>(a, p.units, p.joins, st);
  }
  if (p.MT == 1) return draft_launch<T, D, 1, 1>(a, p.units, p.joins, st);
  return draft_launch<T, D, 2, 1>(a, p.units, p.joins, st);
}

#define HTREE_DRAFT_TYPE(T)                                                        \
  template <>                                                                      \
  int draft_launch_type<T>(const DraftArgs& a, const DraftPlan& p, hipStream_t st) { \
    if (p.D == 32) return draft_launch_dim<T, 32>(a, p, st);                       \
    if (p.D == 64) return draft_launch_dim<T, 64>(a, p, st);                       \
    if (p.D == 128) return draft_launch_dim<T, 128>(a, p, st);                     \
    return draft_launch_dim<T, 256>(a, p, st);                                     \
  }

}  // namespace htree
