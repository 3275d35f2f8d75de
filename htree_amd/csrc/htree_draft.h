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
// One block of four waves takes a unit: 16 MT rows of one (request, KV head)
// and a chunk of its tokens.  The waves take the chunk's tiles of KT tokens
// in turn, each on its own: no barrier until the end, where the four running
// (max, sum, output) states meet in LDS.  Units of one request meet in a
// second launch (draft_join_kernel) through the workspace.
#pragma once

#include "htree_cache_index.h"
#include "htree_common.h"

namespace htree {

struct DraftArgs {
  const char *q, *k, *v;
  char* out;
  const int32_t *table, *lens, *starts, *parents;
  float* ws_o;   // [slots][R][D] output of a unit, relative to its max
  float* ws_ml;  // [slots][R][2] max (log2 units) and sum
  int64_t table_stride;
  int64_t q_row, q_head, o_row, o_head;                                // bytes
  int64_t k_page, k_token, k_head, v_page, v_token, v_head;            // bytes
  int32_t B, rows, H, Hkv, G, Dk, Dv, width, page_shift, num_pages;
  int32_t target;  // units to split into (0: one unit per group of rows)
  float c;         // scale * log2(e)
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

template <typename T, int D, int MT>
struct DraftShape {
  static constexpr int ES = (int)sizeof(T);
  static constexpr bool F32 = ES == 4;
  static constexpr int ROWB = D * ES;      // bytes of a staged row
  static constexpr int CPR = ROWB / 16;    // its 16-byte chunks
  static constexpr int RPI = 64 / CPR;     // rows of one load of a wave
  static constexpr int KT = draft_tile(D, ES);
  static constexpr int NI = KT / RPI;      // loads of a tile's keys
  static constexpr int NG = KT / 16;       // groups of 16 tokens: each in one page
  static constexpr int R = 16 * MT;
  static constexpr int TILE = KT * ROWB;
  static constexpr int WAVE_LDS = 2 * TILE;
  static constexpr int NW = kWavesPerBlock;
  static constexpr int NQ = D / 16;        // groups of 4 dims that a lane holds of a row
  // fp32: dims of a lane's V operand read at once
  static constexpr int VW = D / 16 > 4 ? 4 : D / 16;
};

// place of a row's chunk: rows that are read together fall on other banks
template <int CPR>
__device__ __forceinline__ int draft_swz(int row, int chunk) {
  return CPR >= 16 ? chunk ^ (row & 15) : CPR == 8 ? chunk ^ ((row >> 1) & 7) : chunk ^ ((row >> 2) & 3);
}

__device__ __forceinline__ int64_t wave_sum64(int64_t x) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) x += __shfl_xor((long long)x, m);
  return x;
}

__device__ __forceinline__ DraftReq draft_request(const DraftArgs& a, int b) {
  return draft_req(a.starts[b], a.starts[b + 1], a.lens[b], a.rows);
}

// The unit of this block.  Every wave works it out from the lengths: with
// `target` units wanted, a chunk is the same number of tiles everywhere, so a
// long request gets more units than a short one.  The requests whose tokens
// make more than one chunk get workspace slots, one per unit.
struct DraftUnit {
  int b, h, rt, ch, nch;
  int chunk;     // tiles of a chunk
  int64_t slot;  // of the request's first unit; -1 with one chunk
};

template <int KT, int R>
__device__ __forceinline__ bool draft_unit(const DraftArgs& a, int64_t u, bool groups, DraftUnit* o) {
  const int lane = threadIdx.x & 63;
  const int cap = a.width << a.page_shift;
  int64_t w = 0;
  if (a.target > 0) {
    for (int b = lane; b < a.B; b += 64) {
      const DraftReq r = draft_request(a, b);
      w += draft_tiles(r, cap, KT) * draft_row_groups(r, a.G, R);
    }
    w = wave_sum64(w) * a.Hkv;
  }
  const int chunk = draft_chunk(w, a.target);
  int64_t first = 0, slot = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const int b = b0 + lane;
    int nch = 0;
    int64_t rt = 0;
    if (b < a.B) {
      const DraftReq r = draft_request(a, b);
      nch = draft_chunks(draft_tiles(r, cap, KT), chunk);
      rt = draft_row_groups(r, a.G, R) * a.Hkv;
    }
    // units of a request; with `groups` set only those of split requests
    // count, one for each group of rows
    const int64_t mine = groups ? (nch > 1 ? rt : 0) : nch * rt;
    const int64_t sl = nch > 1 ? nch * rt : 0;
    int64_t pu = mine, ps = sl;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      const int64_t x = __shfl_up((long long)pu, m), y = __shfl_up((long long)ps, m);
      if (lane >= m) pu += x, ps += y;
    }
    const uint64_t hit = __ballot(first + pu > u);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      o->b = b0 + l;
      o->nch = uniform(__shfl(nch, l));
      const int64_t before = first + __shfl((long long)(pu - mine), l);
      const int64_t rts = __shfl((long long)rt, l);
      o->slot = o->nch > 1 ? slot + __shfl((long long)(ps - sl), l) : -1;
      o->chunk = chunk;
      // KV head fastest, then row group, then chunk
      const int64_t i = u - before;
      o->h = uniform((int)(i % a.Hkv));
      const int64_t rest = i / a.Hkv, nrt = rts / a.Hkv;
      o->rt = uniform((int)(rest % nrt));
      o->ch = uniform((int)(rest / nrt));
      return true;
    }
    first += __shfl((long long)pu, 63);
    slot += __shfl((long long)ps, 63);
  }
  return false;
}

// 4 consecutive dims of a lane's row: dims dim(q) .. dim(q) + 3, from the
// accumulators of the products' layouts
template <typename T, int D, int MT>
struct DraftQuad {
  using S = DraftShape<T, D, MT>;
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

template <typename T, int D, int MT>
__global__ __launch_bounds__(256, (MT == 1 && D <= 128) ? 2 : 1) void draft_kernel(DraftArgs a) {
  using S = DraftShape<T, D, MT>;
  using Quad = DraftQuad<T, D, MT>;
  constexpr int KT = S::KT, NI = S::NI, NG = S::NG, CPR = S::CPR, RPI = S::RPI, R = S::R;
  constexpr int ES = S::ES, ROWB = S::ROWB, NQ = S::NQ, NW = S::NW;
  constexpr bool F32 = S::F32;
  __shared__ __attribute__((aligned(16))) char lds[NW * S::WAVE_LDS];
  __shared__ float ml[NW][R][2];

  DraftUnit u;
  if (!draft_unit<KT, R>(a, blockIdx.x, false, &u)) return;  // uniform over the block
  const int lane = threadIdx.x & 63, wv = uniform(threadIdx.x >> 6);
  const int n16 = lane & 15, g = lane >> 4;
  const DraftReq rq = draft_request(a, u.b);
  const int s0 = uniform(rq.s0), ctx = uniform(rq.ctx);
  const int cap = a.width << a.page_shift;
  const int64_t nrow = (int64_t)rq.n * a.G, row0 = (int64_t)u.rt * R;
  const DraftSpan sp = draft_span(rq, row0, R, a.G, cap, KT, u.ch, u.chunk);
  const int kend = uniform(sp.kend), t0 = uniform(sp.t0), t1 = uniform(sp.t1);

  // ---- the rows' queries, as the product's second operand (column n16)
  int tok[MT];  // the row's new token, -1 behind the last row
  int64_t orow[MT];
  f32x4 qf[MT][F32 ? D / 16 : 1];
  typename std::conditional<F32, f32x4, bf16x8>::type qh[MT][F32 ? 1 : D / 32];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int64_t r = row0 + mt * 16 + n16;
    const bool on = r < nrow;
    const int j = on ? (int)(r / a.G) : 0, hg = on ? (int)(r - (int64_t)j * a.G) : 0;
    tok[mt] = on ? j : -1;
    const char* p = a.q + (int64_t)(s0 + j) * a.q_row + (int64_t)(u.h * a.G + hg) * a.q_head;
    if constexpr (F32) {
#pragma unroll
      for (int s = 0; s < D / 16; ++s) {
        const int d = 16 * s + 4 * g;
        qf[mt][s] = on && d < a.Dk ? *(const f32x4*)(p + d * 4) : f32x4{0.f, 0.f, 0.f, 0.f};
      }
    } else {
#pragma unroll
      for (int s = 0; s < D / 32; ++s) {
        const int d = 32 * s + 8 * g;
        const uint4 x = on && d < a.Dk ? *(const uint4*)(p + d * 2) : make_uint4(0, 0, 0, 0);
        qh[mt][s] = __builtin_bit_cast(bf16x8, x);
      }
    }
  }

  float m[MT], l[MT];
  f32x4 o[MT][NQ];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    m[mt] = -INFINITY;
    l[mt] = 0.f;
#pragma unroll
    for (int q = 0; q < NQ; ++q) o[mt][q] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // ---- this wave's tiles
  char* kb = lds + wv * S::WAVE_LDS;
  char* vb = kb + S::TILE;
  const int lr = lane / CPR, lc = lane % CPR;
  // lanes past the head dim read the row's first chunk and write zeros
  const bool kin = lc * 16 < a.Dk * ES, vin = lc * 16 < a.Dv * ES;
  const int64_t koff = lr * a.k_token + (kin ? lc * 16 : 0);
  const int64_t voff = lr * a.v_token + (vin ? lc * 16 : 0);
  const char* kh = a.k + u.h * a.k_head;
  const char* vh = a.v + u.h * a.v_head;
  const int32_t* tab = a.table + u.b * a.table_stride;
  const int used = (kend + (1 << a.page_shift) - 1) >> a.page_shift;  // <= width

  // page of each group of 16 tokens, -1: none (past the end, or no page of the cache)
  auto pages = [&](int t, int (&e)[NG]) {
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      const int pi = (t * KT + 16 * i) >> a.page_shift;
      e[i] = cache_page(t < t1 && pi < used ? tab[pi] : -1, a.num_pages);
    }
  };
  uint4 kr[NI], vr[NI];
  auto load = [&](int t, const int (&e)[NG]) {
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      const int64_t pg = e[i] < 0 ? 0 : e[i];
      const int at = (t * KT + 16 * i) & ((1 << a.page_shift) - 1);
      const char* kp = kh + pg * a.k_page + at * a.k_token;
      const char* vp = vh + pg * a.v_page + at * a.v_token;
#pragma unroll
      for (int x = 0; x < NI / NG; ++x) {
        kr[i * (NI / NG) + x] = *(const uint4*)(kp + (koff + (int64_t)(x * RPI) * a.k_token));
        vr[i * (NI / NG) + x] = *(const uint4*)(vp + (voff + (int64_t)(x * RPI) * a.v_token));
      }
    }
  };

  int ent[NG], nxt[NG];
  int t = t0 + wv;
  pages(t, ent);
  pages(t + NW, nxt);
  if (t < t1) load(t, ent);
  for (; t < t1; t += NW) {
    const int key0 = t * KT;
    // tokens that every row sees need no mask: those before the new ones,
    // in pages that exist
    bool masked = key0 + KT > min(ctx, kend);
#pragma unroll
    for (int i = 0; i < NG; ++i) masked |= ent[i] < 0;
    uint64_t odd = 0;  // tokens with an infinite or NaN value
    if (masked) {
      // Values that no row sees must not meet the product: 0 x NaN is NaN.
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int row = i * RPI + lr;
        if (key0 + row >= kend || ent[i * RPI / 16] < 0) vr[i] = make_uint4(0, 0, 0, 0);
        // every exponent bit set in an element
        bool bad;
        if constexpr (F32) {
          bad = false;
          const uint32_t w[4] = {vr[i].x, vr[i].y, vr[i].z, vr[i].w};
#pragma unroll
          for (int x = 0; x < 4; ++x) bad |= (w[x] & 0x7f800000u) == 0x7f800000u;
        } else {
          constexpr uint32_t E = std::is_same<T, __bf16>::value ? 0x7f80u : 0x7c00u;
          bad = false;
          const uint32_t w[4] = {vr[i].x, vr[i].y, vr[i].z, vr[i].w};
#pragma unroll
          for (int x = 0; x < 4; ++x)
            bad |= (w[x] & E) == E || ((w[x] >> 16) & E) == E;
        }
        uint64_t hit = __ballot(bad && vin);
        if (hit) {
#pragma unroll
          for (int x = 0; x < RPI; ++x) {
            const uint64_t lanes = (CPR == 64 ? ~0ull : ((1ull << (CPR & 63)) - 1)) << ((x * CPR) & 63);
            if (hit & lanes) odd |= 1ull << (i * RPI + x);
          }
          if ((odd >> row) & 1) vr[i] = make_uint4(0, 0, 0, 0);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int row = i * RPI + lr;
      const int at = row * ROWB + draft_swz<CPR>(row, lc) * 16;
      if (!kin) kr[i] = make_uint4(0, 0, 0, 0);
      if (!vin) vr[i] = make_uint4(0, 0, 0, 0);
      *(uint4*)(kb + at) = kr[i];
      *(uint4*)(vb + at) = vr[i];
    }
    int cur[NG];
#pragma unroll
    for (int i = 0; i < NG; ++i) cur[i] = ent[i], ent[i] = nxt[i];
    if (t + NW < t1) load(t + NW, ent);
    pages(t + 2 * NW, nxt);
    wave_sync();

    // ---- scores, token x row: a lane holds tokens 4 g .. 4 g + 3 of each
    // group of 16, of row n16
    f32x4 sc[MT][NG];
#pragma unroll
    for (int i = 0; i < NG; ++i) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) sc[mt][i] = f32x4{0.f, 0.f, 0.f, 0.f};
      const int row = 16 * i + n16;
      const char* p = kb + row * ROWB;
      if constexpr (F32) {
#pragma unroll
        for (int s = 0; s < D / 16; ++s) {
          const f32x4 x = *(const f32x4*)(p + draft_swz<CPR>(row, 4 * s + g) * 16);
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
              sc[mt][i] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], qf[mt][s][e], sc[mt][i], 0, 0, 0);
        }
      } else {
        using V8 = typename DraftT<T>::V8;
#pragma unroll
        for (int s = 0; s < D / 32; ++s) {
          const V8 x = *(const V8*)(p + draft_swz<CPR>(row, 4 * s + g) * 16);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
            sc[mt][i] = DraftT<T>::mma(x, __builtin_bit_cast(V8, qh[mt][s]), sc[mt][i]);
        }
      }
    }

    // ---- to log2 units; masks
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int i = 0; i < NG; ++i) sc[mt][i] *= a.c;
    if (masked) {
      uint64_t there = 0;  // tokens before the end, in pages that exist
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        const int left = min(max(kend - key0 - 16 * i, 0), 16);
        if (cur[i] >= 0) there |= (uint64_t)((1u << left) - 1u) << (16 * i);
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        uint64_t see = 0;
        if (tok[mt] >= 0) {
          if (a.parents) {
            const int c0 = min(max(ctx - key0, 0), 64);  // cached tokens of the tile
            see = c0 == 64 ? ~0ull : (1ull << c0) - 1;
            for (int j = tok[mt]; j >= 0 && ctx + j >= key0;) {
              if (ctx + j - key0 < KT) see |= 1ull << (ctx + j - key0);
              j = draft_parent(a.parents[s0 + j], j);
            }
          } else {
            const int c1 = min(max(ctx + tok[mt] + 1 - key0, 0), 64);
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

    // ---- running softmax
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < NG; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) mx = fmaxf(mx, sc[mt][i][e]);
      mx = max_xor32(max_xor16(mx));
      if (__any(mx > m[mt])) {
        const float mn = fmaxf(m[mt], mx);
        const float al = m[mt] == mn ? 1.f : __builtin_amdgcn_exp2f(m[mt] - mn);
        m[mt] = mn;
        l[mt] *= al;
#pragma unroll
        for (int q = 0; q < NQ; ++q) o[mt][q] *= al;
      }
      const float ref = m[mt] == -INFINITY ? 0.f : m[mt];
#pragma unroll
      for (int i = 0; i < NG; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          sc[mt][i][e] = __builtin_amdgcn_exp2f(sc[mt][i][e] - ref);
          l[mt] += sc[mt][i][e];
        }
    }

    // ---- tokens with infinite or NaN values (their staged rows are zero):
    // only the rows that see them take them
    if (odd) {
      for (uint64_t left = odd; left; left &= left - 1) {
        const int key = __builtin_ctzll(left);
        const int pi = (key0 + key) >> a.page_shift, at = (key0 + key) & ((1 << a.page_shift) - 1);
        const int64_t pg = tab[pi];  // a page of the cache: its values were read
        const char* vp = vh + pg * a.v_page + at * a.v_token;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          float p = 0.f;
#pragma unroll
          for (int i = 0; i < NG; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (key >> 4 == i && (key & 3) == e) p = sc[mt][i][e];
          p = __shfl(p, ((key >> 2) & 3) * 16 + n16);
          // row n16 sees it: not masked (p may be 0 for a very low score)
          bool see = tok[mt] >= 0;
          if (see && a.parents) {
            int j = tok[mt];
            while (j >= 0 && ctx + j > key0 + key) j = draft_parent(a.parents[s0 + j], j);
            see = key0 + key < ctx || (j >= 0 && ctx + j == key0 + key);
          } else if (see) {
            see = key0 + key <= ctx + tok[mt];
          }
#pragma unroll
          for (int q = 0; q < NQ; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int d = Quad::dim(q, g) + e;
              if (see && d < a.Dv) Quad::add(o[mt], q, e, p * Io<T>::ld((const T*)vp + d));
            }
        }
      }
    }

    // ---- output, dim x row: the tokens of a product's k index are those a
    // lane holds, so the scores' registers are its second operand as they are
    if constexpr (F32) {
#pragma unroll
      for (int i = 0; i < NG; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int row = 16 * i + 4 * g + e;
#pragma unroll
          for (int q = 0; q < NQ; q += S::VW) {
            if constexpr (S::VW == 4) {
              const f32x4 x = *(const f32x4*)(vb + row * ROWB + draft_swz<CPR>(row, 4 * q + n16) * 16);
#pragma unroll
              for (int w = 0; w < 4; ++w)
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
                  o[mt][q + w] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[w], sc[mt][i][e], o[mt][q + w], 0, 0, 0);
            } else {
              const f32x2 x = *(const f32x2*)(vb + row * ROWB + draft_swz<CPR>(row, n16 >> 1) * 16 + (n16 & 1) * 8);
#pragma unroll
              for (int w = 0; w < 2; ++w)
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
                  o[mt][q + w] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[w], sc[mt][i][e], o[mt][q + w], 0, 0, 0);
            }
          }
        }
    } else {
      // P rounded to the values' type: a relative half step for each of many
      // tokens, as large as the output's own rounding at most; the sum l is
      // taken of the unrounded P
      uint2 ph[MT][NG];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int i = 0; i < NG; ++i) {
          typedef __attribute__((ext_vector_type(4))) T T4;
          ph[mt][i] = __builtin_bit_cast(uint2, __builtin_convertvector(sc[mt][i], T4));
        }
      // a transposing read gives lane n16 of group g four tokens of dim n16:
      // it addresses token 4 g + n16 / 4, dims 4 (n16 % 4) ..
      auto col = [&](int i, int q) {
        const int row = 16 * i + 4 * g + (n16 >> 2);
        const char* p = vb + row * ROWB + draft_swz<CPR>(row, 2 * q + ((n16 & 3) >> 1)) * 16 + (n16 & 1) * 8;
        return __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) s16x4*)(const __attribute__((address_space(3))) void*)p);
      };
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
        if constexpr (NG == 1) {
          const s16x4 x = col(0, q);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
            o[mt][q] = DraftT<T>::mma_k16(x, __builtin_bit_cast(s16x4, ph[mt][0]), o[mt][q]);
        } else {
          using V8 = typename DraftT<T>::V8;
#pragma unroll
          for (int i = 0; i < NG; i += 2) {
            const uint2 x0 = __builtin_bit_cast(uint2, col(i, q)), x1 = __builtin_bit_cast(uint2, col(i + 1, q));
            const V8 x = __builtin_bit_cast(V8, make_uint4(x0.x, x0.y, x1.x, x1.y));
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
              o[mt][q] = DraftT<T>::mma(
                  x, __builtin_bit_cast(V8, make_uint4(ph[mt][i].x, ph[mt][i].y, ph[mt][i + 1].x, ph[mt][i + 1].y)),
                  o[mt][q]);
          }
        }
      }
    }
    wave_sync();  // this tile's reads come before the next one's writes
  }

  // ---- the four waves' states meet
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    l[mt] = add_xor32(add_xor16(l[mt]));
    if (g == 0) {
      ml[wv][mt * 16 + n16][0] = m[mt];
      ml[wv][mt * 16 + n16][1] = l[mt];
    }
  }
  __syncthreads();
  constexpr int OC = D / 4;           // 16-byte chunks of an fp32 row
  constexpr int OS = OC < 16 ? 7 : 15;
  const bool part = u.nch > 1;
  const int64_t slot = part ? u.slot + (u.ch * draft_row_groups(rq, a.G, R) + u.rt) * a.Hkv + u.h : 0;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; ++w) mm = fmaxf(mm, ml[w][mt * 16 + n16][0]);
    const float f = m[mt] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[mt] - mm);
    // a wave that saw no token of the row adds nothing; NaN states stay NaN
    float* mine = (float*)(lds + wv * S::WAVE_LDS);
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      const f32x4 x = Quad::get(o[mt], q);
      const int ch = Quad::dim(q, g) >> 2;
      *(f32x4*)(mine + n16 * D + ((ch ^ (n16 & OS)) << 2)) = m[mt] == -INFINITY ? x : x * f;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * OC; i += 256) {
      const int row = i / OC, ch = i % OC, rr = mt * 16 + row;
      const int64_t r = row0 + rr;
      if (r >= nrow) continue;
      f32x4 x = {0.f, 0.f, 0.f, 0.f};
      float big = -INFINITY, sum = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) big = fmaxf(big, ml[w][rr][0]);
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        x += *(const f32x4*)((const float*)(lds + w * S::WAVE_LDS) + row * D + ((ch ^ (row & OS)) << 2));
        const float mw = ml[w][rr][0];
        sum += mw == -INFINITY ? ml[w][rr][1] : ml[w][rr][1] * __builtin_amdgcn_exp2f(mw - big);
      }
      if (part) {
        *(f32x4*)(a.ws_o + (slot * R + rr) * D + ch * 4) = x;
        if (ch == 0) {
          a.ws_ml[(slot * R + rr) * 2] = big;
          a.ws_ml[(slot * R + rr) * 2 + 1] = sum;
        }
      } else if (ch * 4 < a.Dv) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;  // a row that sees nothing is zero
        const int j = (int)(r / a.G), hg = (int)(r - (int64_t)j * a.G);
        char* p = a.out + (int64_t)(s0 + j) * a.o_row + (int64_t)(u.h * a.G + hg) * a.o_head + ch * 4 * ES;
        typedef __attribute__((ext_vector_type(4))) T T4;
        *(T4*)p = __builtin_convertvector(x * inv, T4);
      }
    }
    __syncthreads();
  }
}

// Joins the chunks of split requests: one block per row, the threads split
// over the chunks and the row's dims.
template <typename T, int D, int MT>
__global__ __launch_bounds__(256) void draft_join_kernel(DraftArgs a) {
  using S = DraftShape<T, D, MT>;
  constexpr int R = S::R, OC = D / 4, NP = 256 / OC;  // chunks taken at a time
  __shared__ f32x4 acc[256];
  __shared__ float lsum[NP];
  DraftUnit u;
  if (!draft_unit<S::KT, R>(a, blockIdx.x / R, true, &u)) return;
  const int rr = blockIdx.x % R;
  const DraftReq rq = draft_request(a, u.b);
  const int64_t nrow = (int64_t)rq.n * a.G, r = (int64_t)u.rt * R + rr;
  if (r >= nrow) return;
  const int64_t nrt = draft_row_groups(rq, a.G, R);
  const int64_t base = u.slot + (int64_t)u.rt * a.Hkv + u.h, step = nrt * a.Hkv;
  const int tid = threadIdx.x, p = tid / OC, ch = tid % OC;
  float big = -INFINITY;
  for (int c = tid & 63; c < u.nch; c += 64) big = fmaxf(big, a.ws_ml[((base + c * step) * R + rr) * 2]);
  big = wave_max(big);
  f32x4 x = {0.f, 0.f, 0.f, 0.f};
  float sum = 0.f;
#pragma unroll 4
  for (int c = p; c < u.nch; c += NP) {
    const int64_t at = (base + c * step) * R + rr;
    const float mc = a.ws_ml[at * 2], lc = a.ws_ml[at * 2 + 1];
    const f32x4 oc = *(const f32x4*)(a.ws_o + at * D + ch * 4);
    // a chunk whose tokens the row does not see has max -inf and zeros
    // (NaN scores leave the max alone and make the sum NaN)
    const float f = mc == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mc - big);
    x += oc * f;
    sum += lc * f;
  }
  acc[tid] = x;
  if (ch == 0) lsum[p] = sum;
  __syncthreads();
  if (p == 0 && ch * 4 < a.Dv) {
#pragma unroll
    for (int i = 1; i < NP; ++i) {
      x += acc[i * OC + ch];
      sum += lsum[i];
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const int j = (int)(r / a.G), hg = (int)(r - (int64_t)j * a.G);
    char* o = a.out + (int64_t)(rq.s0 + j) * a.o_row + (int64_t)(u.h * a.G + hg) * a.o_head + ch * 4 * S::ES;
    typedef __attribute__((ext_vector_type(4))) T T4;
    *(T4*)o = __builtin_convertvector(x * inv, T4);
  }
}

template <typename T, int D, int MT>
int draft_launch(const DraftArgs& a, int64_t units, int64_t groups, hipStream_t st) {
  hipLaunchKernelGGL((draft_kernel<T, D, MT>), dim3((unsigned)units), dim3(256), 0, st, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return (int)e;
  if (groups > 0) {
    hipLaunchKernelGGL((draft_join_kernel<T, D, MT>), dim3((unsigned)(groups * 16 * MT)), dim3(256), 0, st, a);
    e = hipGetLastError();
  }
  return e == hipSuccess ? HTREE_OK : (int)e;
}

template <typename T>
int draft_launch_type(const DraftArgs& a, int D, int MT, int64_t units, int64_t groups, hipStream_t st);

#define HTREE_DRAFT_TYPE(T)                                                                          \
  template <>                                                                                        \
  int draft_launch_type<T>(const DraftArgs& a, int D, int MT, int64_t units, int64_t groups,         \
                           hipStream_t st) {                                                         \
    switch (D * 8 + MT) {                                                                            \
      case 32 * 8 + 1: return draft_launch<T, 32, 1>(a, units, groups, st);                          \
      case 32 * 8 + 2: return draft_launch<T, 32, 2>(a, units, groups, st);                          \
      case 32 * 8 + 4: return draft_launch<T, 32, 4>(a, units, groups, st);                          \
      case 64 * 8 + 1: return draft_launch<T, 64, 1>(a, units, groups, st);                          \
      case 64 * 8 + 2: return draft_launch<T, 64, 2>(a, units, groups, st);                          \
      case 64 * 8 + 4: return draft_launch<T, 64, 4>(a, units, groups, st);                          \
      case 128 * 8 + 1: return draft_launch<T, 128, 1>(a, units, groups, st);                        \
      case 128 * 8 + 2: return draft_launch<T, 128, 2>(a, units, groups, st);                        \
      case 128 * 8 + 4: return draft_launch<T, 128, 4>(a, units, groups, st);                        \
      case 256 * 8 + 1: return draft_launch<T, 256, 1>(a, units, groups, st);                        \
      default: return draft_launch<T, 256, 2>(a, units, groups, st);                                 \
    }                                                                                                \
  }

}  // namespace htree
