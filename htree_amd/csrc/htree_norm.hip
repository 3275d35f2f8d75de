// Norms of queries and keys by head, with the rotation by position in the same
// pass, and their gradients.
//
//   r = (mean x^2 + eps)^-1/2,  n = x r w,  y = (n1 c - n2 s, n2 c + n1 s)
//   h = (dy1 c + dy2 s, dy2 c - dy1 s),  dw = sum h x r,  g = h w,
//   dx = r (g - x r^2 mean(g x))
//
// with the halves 1, 2 of a head.  Everything is fp32 between one rounding of
// what is read and one of what is written.
#include "htree_cache_host.h"
#include "htree_common.h"

namespace htree {

constexpr int kNormThreads = 256;
constexpr int kNormBlocks = 1024;  // of the backward at most: each leaves a row of partial sums

struct NormSide {  // queries, or keys
  const char *x, *dy;
  char* y;                              // the backward's dx
  const void* w;
  int64_t x_row, x_head, dy_row, dy_head;  // bytes; y is contiguous
  int32_t heads;
};

struct NormArgs {
  NormSide side[2];
  const int32_t* positions;
  const float *cs, *sn;
  float* partial;   // backward: [2][blocks][D]
  int64_t items;    // rows x heads of both sides
  int32_t rows, D, per, lanes, rope_rows, w_f32;
  float eps, inv_d;
};

template <int N>
struct NormVec;
template <>
struct NormVec<16> {
  typedef uint4 V;
};
template <>
struct NormVec<8> {
  typedef uint2 V;
};

// sum over the group of L lanes, to all of them
__device__ __forceinline__ float lanes_sum(float x, int L) {
  for (int m = 1; m < L; m <<= 1) x += __shfl_xor(x, m);
  return x;
}

template <typename T, int NV>
__device__ __forceinline__ void load_weight(const NormArgs& a, const void* w, int at, float* out) {
  if (!w) {
#pragma unroll
    for (int e = 0; e < NV; ++e) out[e] = 1.f;
  } else if (a.w_f32) {
#pragma unroll
    for (int e = 0; e < NV; ++e) out[e] = ((const float*)w)[at + e];
  } else {
#pragma unroll
    for (int e = 0; e < NV; ++e) out[e] = (float)((const T*)w)[at + e];
  }
}

// The rotation of a row, for a lane's NV pairs; false: the row has no position.
template <int NV>
__device__ __forceinline__ bool load_turn(const NormArgs& a, int row, int at, float* c, float* s) {
#pragma unroll
  for (int e = 0; e < NV; ++e) c[e] = 1.f, s[e] = 0.f;
  if (!a.cs) return true;
  const int pos = a.positions[row];
  if (pos < 0 || pos >= a.rope_rows) return false;
  const int64_t o = (int64_t)pos * (a.D / 2) + at;
#pragma unroll
  for (int e = 0; e < NV; ++e) c[e] = a.cs[o + e], s[e] = a.sn[o + e];
  return true;
}

// A head has `lanes` lanes (2^n: LANES, or 0: as the arguments say), the first
// `per` of them with VB bytes of each half, so that a lane has both elements of
// its pairs.  (Four heads of a row a lane, which reads the rotation and the
// weights once for them, took 1 to 2 us longer up to 1000 rows and 234 us instead
// of 227 for 65536.)  Bound by memory, in and out once: 65536 rows of 32/2 heads
// of 128, rotated, bf16, 227 us (5.2 TB/s); 64 such rows 3.5 us, most of it the
// launch.
template <typename T, int VB, int LANES>
__global__ __launch_bounds__(kNormThreads) void head_norm_kernel(NormArgs a) {
  constexpr int NV = VB / (int)sizeof(T);
  typedef typename NormVec<VB>::V V;
  const int L = LANES ? LANES : a.lanes, lane = threadIdx.x & (L - 1);
  const int64_t item = ((int64_t)blockIdx.x * kNormThreads + threadIdx.x) / L;
  if (item >= a.items) return;
  const int all = a.side[0].heads + a.side[1].heads;
  const int row = (int)((uint32_t)item / (uint32_t)all);
  int h = (int)((uint32_t)item - (uint32_t)row * all);
  const int which = h >= a.side[0].heads;
  if (which) h -= a.side[0].heads;
  const NormSide& sd = a.side[which];
  const int half = a.D / 2, at = lane * NV;
  const bool on = lane < a.per;
  const int64_t hb = (int64_t)half * sizeof(T);
  V v1, v2;
  float w1[NV], w2[NV], c[NV], s[NV], ss = 0.f;
  bool there = true;
  const T *p1 = (const T*)&v1, *p2 = (const T*)&v2;
  if (on) {
    const char* x = sd.x + row * sd.x_row + h * sd.x_head + lane * VB;
    v1 = *(const V*)x, v2 = *(const V*)(x + hb);
    load_weight<T, NV>(a, sd.w, at, w1);
    load_weight<T, NV>(a, sd.w, half + at, w2);
    there = load_turn<NV>(a, row, at, c, s);
#pragma unroll
    for (int e = 0; e < NV; ++e) ss += (float)p1[e] * (float)p1[e] + (float)p2[e] * (float)p2[e];
  }
  const float r = rsqrtf(lanes_sum(ss, L) * a.inv_d + a.eps);
  if (!on) return;
  V o1, o2;
  T *q1 = (T*)&o1, *q2 = (T*)&o2;
#pragma unroll
  for (int e = 0; e < NV; ++e) {
    const float n1 = (float)p1[e] * r * w1[e], n2 = (float)p2[e] * r * w2[e];
    q1[e] = (T)(there ? n1 * c[e] - n2 * s[e] : 0.f);
    q2[e] = (T)(there ? n2 * c[e] + n1 * s[e] : 0.f);
  }
  char* y = sd.y + ((int64_t)row * sd.heads + h) * a.D * (int64_t)sizeof(T) + lane * VB;
  *(V*)y = o1;
  *(V*)(y + hb) = o2;
}

// The gradients of x, and each block's share of the weights'.  Blocks walk over
// a side's items in steps of the grid, queries first, so that a lane's sums of
// dw stay in registers.  Bound by memory, x and dy in, dx out once: 65536 rows
// of 32/4 heads of 128, bf16, 380 us (4.8 TB/s).
template <typename T, int VB, int LANES>
__global__ __launch_bounds__(kNormThreads, 4) void head_norm_bwd_kernel(NormArgs a) {
  constexpr int NV = VB / (int)sizeof(T);
  const int L = LANES ? LANES : a.lanes, G = kNormThreads / L;
  typedef typename NormVec<VB>::V V;
  __shared__ float red[kNormThreads * NV * 2];
  const int lane = threadIdx.x & (L - 1), grp = threadIdx.x / L;
  const int half = a.D / 2, at = lane * NV;
  const bool on = lane < a.per;
  const int64_t hb = (int64_t)half * sizeof(T);
#pragma unroll 1
  for (int which = 0; which < 2; ++which) {
    const NormSide& sd = a.side[which];
    if (!sd.heads) continue;
    float w1[NV], w2[NV], d1[NV], d2[NV];
#pragma unroll
    for (int e = 0; e < NV; ++e) d1[e] = d2[e] = 0.f;
    if (on) {
      load_weight<T, NV>(a, sd.w, at, w1);
      load_weight<T, NV>(a, sd.w, half + at, w2);
    }
    const int64_t items = (int64_t)a.rows * sd.heads, step = (int64_t)gridDim.x * G;
    // the next item's halves are read while this one's are computed (of fp32,
    // which has half as much to compute for each byte, that is 4% slower)
    constexpr bool ahead = sizeof(T) == 2;
    V v1, v2, u1, u2;
    int row = 0, h = 0;
    auto load = [&](int64_t item) {
      row = (int)((uint32_t)item / (uint32_t)sd.heads);
      h = (int)((uint32_t)item - (uint32_t)row * sd.heads);
      const char* x = sd.x + row * sd.x_row + h * sd.x_head + lane * VB;
      const char* dy = sd.dy + row * sd.dy_row + h * sd.dy_head + lane * VB;
      v1 = *(const V*)x, v2 = *(const V*)(x + hb);
      u1 = *(const V*)dy, u2 = *(const V*)(dy + hb);
    };
    int64_t item = (int64_t)blockIdx.x * G + grp;
    if (ahead && on && item < items) load(item);
    for (int64_t i0 = (int64_t)blockIdx.x * G; i0 < items; i0 += step, item += step) {
      const bool mine = on && item < items;
      if (!ahead && mine) load(item);
      float c[NV], s[NV];
      const bool there = mine && load_turn<NV>(a, row, at, c, s);
      const V cv1 = v1, cv2 = v2, cu1 = u1, cu2 = u2;
      char* dx = sd.y + (((int64_t)row * sd.heads + h) * a.D) * sizeof(T) + lane * VB;
      if (ahead && on && item + step < items) load(item + step);
      const T *x1 = (const T*)&cv1, *x2 = (const T*)&cv2, *y1 = (const T*)&cu1, *y2 = (const T*)&cu2;
      float g1[NV], g2[NV], ss = 0.f, dot = 0.f;
      if (there) {
#pragma unroll
        for (int e = 0; e < NV; ++e) {
          const float a1 = (float)y1[e], a2 = (float)y2[e], b1 = (float)x1[e], b2 = (float)x2[e];
          g1[e] = a1 * c[e] + a2 * s[e];
          g2[e] = a2 * c[e] - a1 * s[e];
          ss += b1 * b1 + b2 * b2;
          dot += g1[e] * w1[e] * b1 + g2[e] * w2[e] * b2;
        }
      }
      ss = lanes_sum(ss, L), dot = lanes_sum(dot, L);
      if (!mine) continue;
      const float r = rsqrtf(ss * a.inv_d + a.eps), k = r * r * dot * a.inv_d;
      V o1, o2;
      T *q1 = (T*)&o1, *q2 = (T*)&o2;
#pragma unroll
      for (int e = 0; e < NV; ++e) {
        float e1 = 0.f, e2 = 0.f;
        if (there) {
          const float b1 = (float)x1[e], b2 = (float)x2[e];
          e1 = r * (g1[e] * w1[e] - b1 * k);
          e2 = r * (g2[e] * w2[e] - b2 * k);
          d1[e] += g1[e] * (b1 * r);
          d2[e] += g2[e] * (b2 * r);
        }
        q1[e] = (T)e1, q2[e] = (T)e2;
      }
      *(V*)dx = o1;
      *(V*)(dx + hb) = o2;
    }
    if (!a.partial) continue;
    // the groups' sums, in order
    __syncthreads();
#pragma unroll
    for (int e = 0; e < NV; ++e) {
      red[(grp * L + lane) * 2 * NV + e] = d1[e];
      red[(grp * L + lane) * 2 * NV + NV + e] = d2[e];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < a.D; i += kNormThreads) {
      const int second = i >= half, j = i - (second ? half : 0);
      float sum = 0.f;
      for (int g = 0; g < G; ++g) sum += red[(g * L + j / NV) * 2 * NV + second * NV + j % NV];
      a.partial[((int64_t)which * gridDim.x + blockIdx.x) * a.D + i] = sum;
    }
  }
}

struct NormSumArgs {
  const float* partial;
  void* dw[2];
  int32_t blocks, D, w_f32;
};

// The weights' gradients from the blocks' shares: block x, y sums 16 of the D
// columns of side y, 64 threads a column, in a fixed order.  5.4 us of 1024
// shares, eight loads of a thread in flight (9.4 one after another).
template <typename T>
__global__ __launch_bounds__(1024) void head_norm_sum_kernel(NormSumArgs a) {
  __shared__ float red[64][17];
  if (!a.dw[blockIdx.y]) return;
  const int col = threadIdx.x & 15, part = threadIdx.x >> 4, d = blockIdx.x * 16 + col;
  const float* p = a.partial + (int64_t)blockIdx.y * a.blocks * a.D + d;
  float sum = 0.f;
  if (d < a.D)
#pragma unroll 8
    for (int b = part; b < a.blocks; b += 64) sum += p[(int64_t)b * a.D];
  red[part][col] = sum;
  __syncthreads();
  if (part == 0 && d < a.D) {
    float all = 0.f;
    for (int i = 0; i < 64; ++i) all += red[i][col];
    if (a.w_f32) ((float*)a.dw[blockIdx.y])[d] = all;
    else ((T*)a.dw[blockIdx.y])[d] = (T)all;
  }
}

// ------------------------------------------------------------------ host
// lanes of a head: 2^n >= per
static int norm_lanes(int per) {
  int L = 1;
  while (L < per) L *= 2;
  return L;
}

static int norm_blocks(int64_t items, int L) {
  const int64_t n = (items * L + kNormThreads - 1) / kNormThreads;
  return (int)(n < kNormBlocks ? n : kNormBlocks);
}

// 16-byte pieces of 16-bit types make at most 16 lanes a head, of fp32 32; a
// head of odd 8-byte pieces (D % 16, fp32: D % 8) takes the lanes as they come.
#define HTREE_NORM_TYPE(F, T, MOST) \
  if (!wide) F(T, 8, 0);            \
  else if (L == 1) F(T, 16, 1);     \
  else if (L == 2) F(T, 16, 2);     \
  else if (L == 4) F(T, 16, 4);     \
  else if (L == 8) F(T, 16, 8);     \
  else if (L == 16) F(T, 16, 16);   \
  else F(T, 16, MOST)
#define HTREE_NORM_TYPES(F)          \
  if (dtype == HTREE_F32) {          \
    HTREE_NORM_TYPE(F, float, 32);   \
  } else if (dtype == HTREE_BF16) {  \
    HTREE_NORM_TYPE(F, __bf16, 16);  \
  } else {                           \
    HTREE_NORM_TYPE(F, _Float16, 16); \
  }

// sizes, types, strides and pointers that both directions have
static int norm_check(int32_t dtype, int32_t w_dtype, int32_t rows, int32_t H, int32_t H_kv, int32_t D,
                      const int32_t* positions, const float* cs, const float* sn, int32_t rope_rows) {
  if (dtype != HTREE_F32 && dtype != HTREE_BF16 && dtype != HTREE_F16) return HTREE_ESHAPE;
  if (w_dtype != HTREE_F32 && w_dtype != dtype) return HTREE_ESHAPE;
  if (rows < 0 || H < 0 || H_kv < 0 || D <= 0) return HTREE_ESHAPE;
  if (D > 256 || D * (dtype == HTREE_F32 ? 4 : 2) % 16) return HTREE_EUNSUPPORTED;
  if ((int64_t)rows * ((int64_t)H + H_kv) > 0x7fffffff) return HTREE_EUNSUPPORTED;
  if ((cs || sn || positions) && (!cs || !sn || (rows && !positions))) return HTREE_ENULL;
  if (cs && rope_rows <= 0) return HTREE_ESHAPE;
  return HTREE_OK;
}

}  // namespace htree

using namespace htree;

extern "C" int htree_head_norm(int32_t dtype, int32_t w_dtype, int32_t rows, int32_t H, int32_t H_kv, int32_t D,
                               float eps, const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row,
                               int64_t k_head, const void* q_weight, const void* k_weight,
                               const int32_t* positions, const float* cos_table, const float* sin_table,
                               int32_t rope_rows, void* q_out, void* k_out, void* stream) {
  const int rc = norm_check(dtype, w_dtype, rows, H, H_kv, D, positions, cos_table, sin_table, rope_rows);
  if (rc) return rc;
  if (!(eps >= 0.f)) return HTREE_ESHAPE;
  if (rows == 0 || H + H_kv == 0) return HTREE_OK;
  if ((H && (!q || !q_out)) || (H_kv && (!k || !k_out))) return HTREE_ENULL;
  const int es = dtype == HTREE_F32 ? 4 : 2;
  const int64_t st[4] = {q_row, q_head, k_row, k_head};
  for (int64_t s : st)
    if (s < 0 || s * es % 16) return HTREE_EUNSUPPORTED;
  if (off16(q) || off16(k) || off16(q_out) || off16(k_out)) return HTREE_EUNSUPPORTED;
  NormArgs a = {};
  // 16-byte pieces where a half of a head holds whole ones
  const bool wide = D * es % 32 == 0;
  a.per = D / 2 * es / (wide ? 16 : 8);
  const int L = a.lanes = norm_lanes(a.per);
  a.side[0] = {(const char*)q, nullptr, (char*)q_out, q_weight, q_row * es, q_head * es, 0, 0, H};
  a.side[1] = {(const char*)k, nullptr, (char*)k_out, k_weight, k_row * es, k_head * es, 0, 0, H_kv};
  a.positions = positions, a.cs = cos_table, a.sn = sin_table;
  a.items = (int64_t)rows * (H + H_kv);
  if (a.items * L >= (int64_t)1 << 32) return HTREE_EUNSUPPORTED;  // threads of a grid
  a.rows = rows, a.D = D, a.rope_rows = rope_rows, a.w_f32 = w_dtype == HTREE_F32;
  a.eps = eps, a.inv_d = 1.f / D;
  hipStream_t s = (hipStream_t)stream;
  const unsigned blocks = (unsigned)((a.items * L + kNormThreads - 1) / kNormThreads);
#define HTREE_NORM_FWD(T, VB, LANES) \
  hipLaunchKernelGGL((head_norm_kernel<T, VB, LANES>), dim3(blocks), dim3(kNormThreads), 0, s, a)
  HTREE_NORM_TYPES(HTREE_NORM_FWD)
#undef HTREE_NORM_FWD
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? HTREE_OK : (int)e;
}

extern "C" int htree_head_norm_backward_workspace_bytes(int32_t D, int64_t* bytes) {
  if (!bytes) return HTREE_ENULL;
  if (D <= 0) return HTREE_ESHAPE;
  *bytes = 2ll * kNormBlocks * D * 4;
  return HTREE_OK;
}

extern "C" int htree_head_norm_backward(int32_t dtype, int32_t w_dtype, int32_t rows, int32_t H, int32_t H_kv,
                                        int32_t D, float eps, const void* q, int64_t q_row, int64_t q_head,
                                        const void* k, int64_t k_row, int64_t k_head, const void* dq_out,
                                        int64_t dq_row, int64_t dq_head, const void* dk_out, int64_t dk_row,
                                        int64_t dk_head, const void* q_weight, const void* k_weight,
                                        const int32_t* positions, const float* cos_table, const float* sin_table,
                                        int32_t rope_rows, void* dq, void* dk, void* dq_weight, void* dk_weight,
                                        void* workspace, int64_t workspace_bytes, void* stream) {
  const int rc = norm_check(dtype, w_dtype, rows, H, H_kv, D, positions, cos_table, sin_table, rope_rows);
  if (rc) return rc;
  if (!(eps >= 0.f)) return HTREE_ESHAPE;
  if (rows == 0 || H + H_kv == 0) return HTREE_OK;
  if ((H && (!q || !dq_out || !dq)) || (H_kv && (!k || !dk_out || !dk))) return HTREE_ENULL;
  const bool weights = (H && dq_weight) || (H_kv && dk_weight);
  int64_t need = 0;
  htree_head_norm_backward_workspace_bytes(D, &need);
  if (weights && !workspace) return HTREE_ENULL;
  if (weights && workspace_bytes < need) return HTREE_EWORKSPACE;
  const int es = dtype == HTREE_F32 ? 4 : 2;
  const int64_t st[8] = {q_row, q_head, k_row, k_head, dq_row, dq_head, dk_row, dk_head};
  for (int64_t s : st)
    if (s < 0 || s * es % 16) return HTREE_EUNSUPPORTED;
  if (off16(q) || off16(k) || off16(dq_out) || off16(dk_out) || off16(dq) || off16(dk) || off16(workspace))
    return HTREE_EUNSUPPORTED;
  NormArgs a = {};
  const bool wide = D * es % 32 == 0;
  a.per = D / 2 * es / (wide ? 16 : 8);
  const int L = a.lanes = norm_lanes(a.per);
  a.side[0] = {(const char*)q, (const char*)dq_out, (char*)dq, q_weight, q_row * es, q_head * es, dq_row * es,
               dq_head * es, H};
  a.side[1] = {(const char*)k, (const char*)dk_out, (char*)dk, k_weight, k_row * es, k_head * es, dk_row * es,
               dk_head * es, H_kv};
  a.positions = positions, a.cs = cos_table, a.sn = sin_table;
  a.partial = weights ? (float*)workspace : nullptr;
  a.rows = rows, a.D = D, a.rope_rows = rope_rows, a.w_f32 = w_dtype == HTREE_F32;
  a.eps = eps, a.inv_d = 1.f / D;
  const int blocks = norm_blocks((int64_t)rows * (H > H_kv ? H : H_kv), L);
  hipStream_t s = (hipStream_t)stream;
#define HTREE_NORM_BWD(T, VB, LANES) \
  hipLaunchKernelGGL((head_norm_bwd_kernel<T, VB, LANES>), dim3(blocks), dim3(kNormThreads), 0, s, a)
  HTREE_NORM_TYPES(HTREE_NORM_BWD)
#undef HTREE_NORM_BWD
  if (weights) {
    const NormSumArgs w = {a.partial, {H ? dq_weight : nullptr, H_kv ? dk_weight : nullptr}, blocks, D, a.w_f32};
    const dim3 grid((D + 15) / 16, 2);
    if (dtype == HTREE_BF16) hipLaunchKernelGGL((head_norm_sum_kernel<__bf16>), grid, dim3(1024), 0, s, w);
    else if (dtype == HTREE_F16) hipLaunchKernelGGL((head_norm_sum_kernel<_Float16>), grid, dim3(1024), 0, s, w);
    else hipLaunchKernelGGL((head_norm_sum_kernel<float>), grid, dim3(1024), 0, s, w);
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? HTREE_OK : (int)e;
}
