// Query and key heads normed, scaled by a learned weight and turned by their position in one
// pass, and the gradient of that: for a head's row x [D], its weight w and the turn R of
// prefixlm_rotary.hip (linear, its transpose the inverse turn),
//
//   r = 1 / sqrt(mean(x^2) + eps),   y = R (r w x)
//   g = R^T dy,   dw = sum over rows of r g x,   dx = r (w g - x r^2 mean(w g x))
//
// (products of columns; the same weight for all query heads and another for all key heads),
// in fp32 with one rounding of each result; sums over the head run across lanes.
//
// Bound by memory: the forward reads and writes each head once, the gradient reads x and
// dy once and writes dx; nothing is saved for it, r comes again from x.  A group of
// lanes (a power of two, at least 8) owns one head's row at a time, each lane V pairs of columns, so
// that the two sums of a row are a few DPP adds.  A group takes every hp-th head of its token,
// so the angles' series are shared by the heads.  8 x 2048 tokens of 16 / 4 bf16 heads of 128: forward 40.6 us (4.1 TB/s; a
// copy reaches 5.1), gradient 57.9 (4.4 TB/s), the weights' sums 4.1.
//
// dw: the groups of a workgroup walk the tokens with a grid-wide stride and keep their sums in registers, a
// workgroup adds its groups through LDS in a fixed order and stores one row of partial sums,
// and a second kernel adds the rows, in a fixed order too: the result does not depend on timing.
#include <algorithm>
#include <cmath>

#include "prefixlm_common.h"
#include "rotary_turn.h"
#include "strided_overlap.h"

namespace mimir {
namespace {

// A forward of at most this many workgroups, two a CU, takes queries and keys in workgroups of their own, as their round trips
// would follow each other.  16 / 4 bf16 heads of 128, replayed: 8 tokens 5.4 -> 3.8 us, 512 (256 workgroups) 5.9 -> 5.4,
// 1024 (512) 8.0 -> 7.8; beyond, all CUs are busy either way.
constexpr int kFewBlocks = 512;
constexpr int kMaxBlocks = 1024;  // rows of partial sums at most: four workgroups for each of 256 CUs

struct HeadArgs {
  const void* x;
  const void* dy;   // gradient: of the output
  void* y;          // output, or the gradient of x
  const void* w;    // NULL: ones
  int64_t x_sb, x_st, x_sh, dy_sb, dy_st, dy_sh, y_sb, y_st, y_sh;
  int heads;
};
struct NormRotaryArgs {
  HeadArgs q, k;
  const int64_t* turns;
  const void* positions;
  int64_t p_sb, p_st;
  int64_t tokens;      // batch * seqlen
  int S, D;
  int half;            // rotary_dim / 2
  int turning, items;  // items of a head that turn, and all
  int lanes;           // lanes of a group: a power of two, >= items and >= 8
  int hp;              // groups that share a token: each takes every hp-th head
  int idx64, w32;
  float amplitude, eps;
  float* part;         // gradient: [workgroups][2][D]
};

template <typename E, int N>
using Row = E __attribute__((ext_vector_type(N)));

template <int kCtrl>
__device__ __forceinline__ float dpp_add(float x) {
  return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), kCtrl, 0xf, 0xf, false));
}
// Sum over the `lanes` lanes of a group (uniform), on each of them.
__device__ __forceinline__ float group_sum(float x, int lanes) {
  x = dpp_add<0xb1>(x);   // quad_perm: lane ^ 1
  x = dpp_add<0x4e>(x);   // quad_perm: lane ^ 2
  x = dpp_add<0x141>(x);  // row_half_mirror: the other quad of eight
  if (lanes >= 16) x = dpp_add<0x140>(x);  // row_mirror: the other eight of sixteen
  if (lanes >= 32) {
    const int v = __float_as_int(x);
    const auto p = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    const int a = p[0], b = p[1];
    x = __int_as_float(a) + __int_as_float(b);
  }
  if (lanes >= 64) x = xor32_sum(x);
  return x;
}

// What a lane owns of its group's token: the columns of its item and their angles.
template <int V, bool kInterleaved>
struct Item {
  bool any, turn;
  int d1, d2;  // its two runs of V columns: the pairs' halves, or 2 V columns in a row
  float cs[V], sn[V];

  __device__ __forceinline__ void place(const NormRotaryArgs& a, int c) {
    any = c < a.items;
    turn = c < a.turning;
    c = any ? c : 0;
    d1 = turn && !kInterleaved ? c * V : 2 * c * V;
    d2 = turn && !kInterleaved ? d1 + a.half : d1 + V;
  }
  __device__ __forceinline__ void angles(const NormRotaryArgs& a, int c, int64_t b, int64_t i) {
    const int64_t at = b * a.p_sb + i * a.p_st;
    const uint64_t pos = (uint64_t)(a.idx64 ? ((const int64_t*)a.positions)[at] : (int64_t)((const int32_t*)a.positions)[at]);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      sincos_turn(pos * (uint64_t)a.turns[(turn ? c * V : 0) + e], cs[e], sn[e]);
      cs[e] = turn ? cs[e] * a.amplitude : 1.f;
      sn[e] = turn ? sn[e] * a.amplitude : 0.f;
    }
  }
};
// Turns the 2 V columns u | w of an item by +-t.  Interleaved: pair e is elements 2 e and 2 e + 1 of the
// run u | w; else elements e of both.  (Columns that are only passed on have angle 0.)
template <int V, bool kInterleaved>
__device__ __forceinline__ void turn_item(const Item<V, kInterleaved>& it, float sign, float (&u)[V], float (&w)[V]) {
  if constexpr (kInterleaved && V > 1) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      float& p = 2 * e < V ? u[(2 * e) % V] : w[(2 * e) % V];
      float& r = 2 * e + 1 < V ? u[(2 * e + 1) % V] : w[(2 * e + 1) % V];
      const float s = sign * it.sn[e], p0 = p, r0 = r;
      p = p0 * it.cs[e] - r0 * s;
      r = r0 * it.cs[e] + p0 * s;
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float s = sign * it.sn[e], p0 = u[e], r0 = w[e];
      u[e] = p0 * it.cs[e] - r0 * s;
      w[e] = r0 * it.cs[e] + p0 * s;
    }
  }
}

template <int V>
__device__ __forceinline__ void load_weight(const void* p, int w32, bool any, int d, float (&w)[V], bf16_t) {
#pragma unroll
  for (int e = 0; e < V; ++e)
    w[e] = !any ? 0.f : p == nullptr ? 1.f : w32 ? ((const float*)p)[d + e] : (float)((const bf16_t*)p)[d + e];
}
template <int V>
__device__ __forceinline__ void load_weight(const void* p, int, bool any, int d, float (&w)[V], float) {
#pragma unroll
  for (int e = 0; e < V; ++e) w[e] = !any ? 0.f : p == nullptr ? 1.f : ((const float*)p)[d + e];
}

template <typename E, int V, bool kInterleaved>
__global__ __launch_bounds__(256) void norm_rotary_kernel(const NormRotaryArgs a) {
  using R = Row<E, V>;
  constexpr int kBatch = 4;  // heads in flight
  const int c = (int)(threadIdx.x & (a.lanes - 1));
  const uint32_t group = (blockIdx.x * 256u + threadIdx.x) / (uint32_t)a.lanes;  // host: below 2^32 threads
  const uint32_t token = group / (uint32_t)a.hp;
  const int h0 = (int)(group - token * (uint32_t)a.hp);
  if (token >= (uint64_t)a.tokens) return;  // whole groups
  const uint32_t b = token / (uint32_t)a.S, i = token - b * (uint32_t)a.S;
  Item<V, kInterleaved> it;
  it.place(a, c);
  it.angles(a, c, b, i);
  const float inv_d = 1.f / (float)a.D;
  auto heads = [&](const HeadArgs& h) __attribute__((always_inline)) {
    const E* const x = (const E*)h.x + b * h.x_sb + i * h.x_st;
    E* const y = (E*)h.y + b * h.y_sb + i * h.y_st;
    float w1[V], w2[V];
    load_weight<V>(h.w, a.w32, it.any, it.d1, w1, E());
    load_weight<V>(h.w, a.w32, it.any, it.d2, w2, E());
    for (int hb = h0; hb < h.heads; hb += kBatch * a.hp) {
      R x1[kBatch], x2[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const E* row = x + min(hb + j * a.hp, h.heads - 1) * h.x_sh;  // past the last head: that one again
        x1[j] = *(const R*)(row + it.d1);
        x2[j] = *(const R*)(row + it.d2);
      }
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int at = hb + j * a.hp;
        if (at >= h.heads) break;
        float u[V], v[V], sq = 0.f;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          u[e] = (float)x1[j][e];
          v[e] = (float)x2[j][e];
          sq += u[e] * u[e] + v[e] * v[e];
        }
        const float r = rsqrtf(group_sum(it.any ? sq : 0.f, a.lanes) * inv_d + a.eps);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          u[e] *= r * w1[e];
          v[e] *= r * w2[e];
        }
        turn_item<V, kInterleaved>(it, 1.f, u, v);
        if (it.any) {
          R y1, y2;
#pragma unroll
          for (int e = 0; e < V; ++e) {
            y1[e] = (E)u[e];
            y2[e] = (E)v[e];
          }
          E* row = y + at * h.y_sh;
          *(R*)(row + it.d1) = y1;
          *(R*)(row + it.d2) = y2;
        }
      }
    }
  };
  if (gridDim.y == 1 || blockIdx.y == 0) heads(a.q);
  if (gridDim.y == 1 || blockIdx.y == 1) heads(a.k);
}

template <typename E, int V, bool kInterleaved>
__global__ __launch_bounds__(256) void norm_rotary_bwd_kernel(const NormRotaryArgs a) {
  using R = Row<E, V>;
  constexpr int kBatch = 2;  // heads in flight
  const int c = (int)(threadIdx.x & (a.lanes - 1));
  const int per_block = 256 / a.lanes, own = (int)threadIdx.x / a.lanes;
  Item<V, kInterleaved> it;
  it.place(a, c);
  const float inv_d = 1.f / (float)a.D;
  float wq1[V], wq2[V], wk1[V], wk2[V];
  load_weight<V>(a.q.w, a.w32, it.any, it.d1, wq1, E());
  load_weight<V>(a.q.w, a.w32, it.any, it.d2, wq2, E());
  load_weight<V>(a.k.w, a.w32, it.any, it.d1, wk1, E());
  load_weight<V>(a.k.w, a.w32, it.any, it.d2, wk2, E());
  float acc[2][2][V] = {};
  const uint32_t groups = (uint32_t)(a.tokens * a.hp);  // host: below 2^31
  for (uint32_t group = blockIdx.x * per_block + own; group < groups; group += gridDim.x * per_block) {
    const uint32_t token = group / (uint32_t)a.hp;
    const int h0 = (int)(group - token * (uint32_t)a.hp);
    const uint32_t b = token / (uint32_t)a.S, i = token - b * (uint32_t)a.S;
    it.angles(a, c, b, i);
    auto heads = [&](const HeadArgs& h, const float (&w1)[V], const float (&w2)[V], float (&s1)[V], float (&s2)[V])
                     __attribute__((always_inline)) {
      const E* const x = (const E*)h.x + b * h.x_sb + i * h.x_st;
      const E* const dy = (const E*)h.dy + b * h.dy_sb + i * h.dy_st;
      E* const dx = (E*)h.y + b * h.y_sb + i * h.y_st;
      for (int hb = h0; hb < h.heads; hb += kBatch * a.hp) {
        R x1[kBatch], x2[kBatch], g1[kBatch], g2[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
          const int at = min(hb + j * a.hp, h.heads - 1);  // past the last head: that one again
          const E *row = x + at * h.x_sh, *grow = dy + at * h.dy_sh;
          x1[j] = *(const R*)(row + it.d1);
          x2[j] = *(const R*)(row + it.d2);
          g1[j] = *(const R*)(grow + it.d1);
          g2[j] = *(const R*)(grow + it.d2);
        }
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
          const int at = hb + j * a.hp;
          if (at >= h.heads) break;
          float u[V], v[V], p[V], q[V], sq = 0.f, dot = 0.f;
#pragma unroll
          for (int e = 0; e < V; ++e) {
            u[e] = (float)x1[j][e];
            v[e] = (float)x2[j][e];
            p[e] = (float)g1[j][e];
            q[e] = (float)g2[j][e];
          }
          turn_item<V, kInterleaved>(it, -1.f, p, q);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            sq += u[e] * u[e] + v[e] * v[e];
            dot += w1[e] * p[e] * u[e] + w2[e] * q[e] * v[e];
          }
          const float r = rsqrtf(group_sum(it.any ? sq : 0.f, a.lanes) * inv_d + a.eps);
          const float m = group_sum(it.any ? dot : 0.f, a.lanes) * inv_d * r * r;
          R y1, y2;
#pragma unroll
          for (int e = 0; e < V; ++e) {
            s1[e] += r * p[e] * u[e];
            s2[e] += r * q[e] * v[e];
            y1[e] = (E)(r * (w1[e] * p[e] - u[e] * m));
            y2[e] = (E)(r * (w2[e] * q[e] - v[e] * m));
          }
          if (it.any) {
            E* row = dx + at * h.y_sh;
            *(R*)(row + it.d1) = y1;
            *(R*)(row + it.d2) = y2;
          }
        }
      }
    };
    heads(a.q, wq1, wq2, acc[0][0], acc[0][1]);
    heads(a.k, wk1, wk2, acc[1][0], acc[1][1]);
  }
  if (a.part == nullptr) return;
  // One row of partial sums for the workgroup: its groups in order.
  __shared__ float sums[256 * 2 * V];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < V; ++e) {
      sums[e * 256 + threadIdx.x] = acc[t][0][e];
      sums[(V + e) * 256 + threadIdx.x] = acc[t][1][e];
    }
    __syncthreads();
    float* const out = a.part + ((int64_t)blockIdx.x * 2 + t) * a.D;
    for (int n = (int)threadIdx.x; n < a.lanes * 2 * V; n += 256) {
      const int e = n / a.lanes, lane = n % a.lanes;
      if (lane >= a.items) continue;
      double s = 0.0;
      for (int j = 0; j < per_block; ++j) s += sums[e * 256 + j * a.lanes + lane];
      Item<V, kInterleaved> o;
      o.place(a, lane);
      out[e < V ? o.d1 + e : o.d2 + e - V] = (float)s;
    }
  }
}

// The weights' gradients: the rows of partial sums added up, 16 columns a workgroup, in 64 bits (in 32 the error of
// 8 x 2048 tokens of 16 heads was 1.9e-7, three times that of one rounding).
constexpr int kSumCols = 16, kSumRows = 1024 / kSumCols;
struct WeightSumArgs {
  const float* part;
  void* out[2];
  int rows, D, w32;
};
__global__ __launch_bounds__(1024) void norm_weight_sum_kernel(const WeightSumArgs a) {
  __shared__ double sums[kSumRows][kSumCols + 1];
  const int c = threadIdx.x % kSumCols, r0 = threadIdx.x / kSumCols;
  const int col = blockIdx.x * kSumCols + c;
  double s = 0.0;
  if (col < 2 * a.D) {
#pragma unroll 8
    for (int r = r0; r < a.rows; r += kSumRows) s += a.part[(int64_t)r * 2 * a.D + col];
  }
  sums[r0][c] = s;
  __syncthreads();
  for (int n = kSumRows / 2; n > 0; n /= 2) {
    if (r0 < n) sums[r0][c] += sums[r0 + n][c];
    __syncthreads();
  }
  if (r0 != 0 || col >= 2 * a.D) return;
  void* const out = a.out[col / a.D];
  if (out == nullptr) return;
  if (a.w32)
    ((float*)out)[col % a.D] = (float)sums[0][c];
  else
    ((bf16_t*)out)[col % a.D] = (bf16_t)(float)sums[0][c];
}

// By name: of several instantiations launched below, this toolchain drops host stubs.
#define NORM_ROTARY(E, V) \
  template __global__ void norm_rotary_kernel<E, V, true>(const NormRotaryArgs); \
  template __global__ void norm_rotary_kernel<E, V, false>(const NormRotaryArgs); \
  template __global__ void norm_rotary_bwd_kernel<E, V, true>(const NormRotaryArgs); \
  template __global__ void norm_rotary_bwd_kernel<E, V, false>(const NormRotaryArgs);
NORM_ROTARY(bf16_t, 8) NORM_ROTARY(bf16_t, 4) NORM_ROTARY(bf16_t, 2) NORM_ROTARY(bf16_t, 1)
NORM_ROTARY(float, 4) NORM_ROTARY(float, 2) NORM_ROTARY(float, 1)
#undef NORM_ROTARY

template <typename E, int V>
void launch_norm_rotary(const NormRotaryArgs& a, bool interleaved, bool bwd, int64_t blocks, hipStream_t stream) {
  const dim3 grid((unsigned)blocks, !bwd && a.k.heads > 0 && blocks <= kFewBlocks ? 2 : 1), threads(256);
  if (bwd) {
    if (interleaved)
      hipLaunchKernelGGL((norm_rotary_bwd_kernel<E, V, true>), grid, threads, 0, stream, a);
    else
      hipLaunchKernelGGL((norm_rotary_bwd_kernel<E, V, false>), grid, threads, 0, stream, a);
  } else {
    if (interleaved)
      hipLaunchKernelGGL((norm_rotary_kernel<E, V, true>), grid, threads, 0, stream, a);
    else
      hipLaunchKernelGGL((norm_rotary_kernel<E, V, false>), grid, threads, 0, stream, a);
  }
}

// Columns per access: as many as both parts of the head, the addresses and the strides are multiples of,
// up to 16 bytes, while a head still takes the 8 lanes of the smallest group.
int access_columns(const MimirNormRotaryParams& p, bool bwd) {
  const int es = p.dtype == MIMIR_DTYPE_BFLOAT16 ? 2 : 4;
  const bool k = p.num_kv_heads > 0;
  auto fits = [&](int n) {
    if (p.rotary_dim % (2 * n) != 0 || (p.head_dim - p.rotary_dim) % (2 * n) != 0) return false;
    auto at = [&](const void* x, int64_t sb, int64_t st, int64_t sh) {
      return (uintptr_t)x % ((uintptr_t)n * es) == 0 && sb % n == 0 && st % n == 0 && sh % n == 0;
    };
    return at(p.q, p.q_stride_batch, p.q_stride_token, p.q_stride_head) &&
           at(p.q_out, p.q_out_stride_batch, p.q_out_stride_token, p.q_out_stride_head) &&
           (!k || (at(p.k, p.k_stride_batch, p.k_stride_token, p.k_stride_head) &&
                   at(p.k_out, p.k_out_stride_batch, p.k_out_stride_token, p.k_out_stride_head))) &&
           (!bwd || (at(p.dq, p.dq_stride_batch, p.dq_stride_token, p.dq_stride_head) &&
                     (!k || at(p.dk, p.dk_stride_batch, p.dk_stride_token, p.dk_stride_head))));
  };
  int v = 16 / es;
  while (v > 1 && (!fits(v) || p.head_dim / (2 * v) < 8)) v /= 2;
  return v;
}

// Workgroups of the gradient: each group of lanes walks its share of the tokens.
int64_t bwd_blocks(int64_t groups, int lanes) { return std::min<int64_t>((groups * lanes + 255) / 256, kMaxBlocks); }

int run_norm_rotary(const MimirNormRotaryParams* given, bool bwd, void* stream) {
  fail_with(MIMIR_OK, "");
  if (given == nullptr) return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "params is NULL");
  // A dim of one entry has a stride, but no step: none that would keep accesses narrow.
  MimirNormRotaryParams own = *given;
  for (int64_t* s : {&own.q_stride_batch, &own.k_stride_batch, &own.q_out_stride_batch, &own.k_out_stride_batch, &own.dq_stride_batch, &own.dk_stride_batch})
    if (own.batch == 1) *s = 0;
  for (int64_t* s : {&own.q_stride_token, &own.k_stride_token, &own.q_out_stride_token, &own.k_out_stride_token, &own.dq_stride_token, &own.dk_stride_token})
    if (own.seqlen == 1) *s = 0;
  for (int64_t* s : {&own.q_stride_head, &own.q_out_stride_head, &own.dq_stride_head})
    if (own.num_q_heads == 1) *s = 0;
  for (int64_t* s : {&own.k_stride_head, &own.k_out_stride_head, &own.dk_stride_head})
    if (own.num_kv_heads == 1) *s = 0;
  const MimirNormRotaryParams* const p = &own;
  if (p->dtype != MIMIR_DTYPE_FLOAT32 && p->dtype != MIMIR_DTYPE_BFLOAT16)
    return fail_with(MIMIR_ERR_UNSUPPORTED_DTYPE, "normed rotary heads support float32 and bfloat16 tensors only (dtype code " +
                                                      std::to_string(p->dtype) + ")");
  if (p->weight_dtype != MIMIR_DTYPE_FLOAT32 && p->weight_dtype != p->dtype)
    return fail_with(MIMIR_ERR_UNSUPPORTED_DTYPE, "norm weights must be float32 or of the heads' type (dtype code " +
                                                      std::to_string(p->weight_dtype) + ")");
  if (p->batch < 0 || p->seqlen < 0 || p->num_q_heads <= 0 || p->num_kv_heads < 0 || p->head_dim <= 0)
    return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "negative size or non-positive heads / head_dim");
  if (p->head_dim % 2 != 0 || p->rotary_dim % 2 != 0 || p->rotary_dim < 2 || p->rotary_dim > p->head_dim)
    return fail_with(MIMIR_ERR_UNSUPPORTED_SHAPE, "rotary_dim " + std::to_string(p->rotary_dim) + " must be even and in [2, head_dim " +
                                                      std::to_string(p->head_dim) + "], which must be even");
  if (!std::isfinite(p->amplitude) || !std::isfinite(p->eps) || p->eps < 0.f)
    return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "amplitude must be finite, eps finite and not negative");
  const bool k = p->num_kv_heads > 0, sums = bwd && (p->dq_weight != nullptr || p->dk_weight != nullptr);
  const bool empty = p->batch == 0 || p->seqlen == 0;
  if (!empty && (p->q == nullptr || p->q_out == nullptr || (k && (p->k == nullptr || p->k_out == nullptr)) || p->turns == nullptr ||
                 p->positions == nullptr || (bwd && (p->dq == nullptr || (k && p->dk == nullptr)))))
    return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "norm_rotary tensor pointer is NULL");
  if (empty && !sums) return MIMIR_OK;
  const int es = p->dtype == MIMIR_DTYPE_BFLOAT16 ? 2 : 4;
  for (const void* x : {p->q, (const void*)p->q_out, p->k, (const void*)p->k_out, p->dq, p->dk})
    if ((uintptr_t)x % es != 0) return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "norm_rotary tensors must be aligned to their elements");
  const int v = access_columns(*p, bwd);
  NormRotaryArgs a = {};
  a.q = {p->q, p->dq, p->q_out, p->q_weight, p->q_stride_batch, p->q_stride_token, p->q_stride_head, p->dq_stride_batch,
         p->dq_stride_token, p->dq_stride_head, p->q_out_stride_batch, p->q_out_stride_token, p->q_out_stride_head, p->num_q_heads};
  a.k = {p->k, p->dk, p->k_out, p->k_weight, p->k_stride_batch, p->k_stride_token, p->k_stride_head, p->dk_stride_batch,
         p->dk_stride_token, p->dk_stride_head, p->k_out_stride_batch, p->k_out_stride_token, p->k_out_stride_head, p->num_kv_heads};
  a.turns = p->turns;
  a.positions = p->positions;
  a.p_sb = p->positions_stride_batch; a.p_st = p->positions_stride_token;
  a.tokens = (int64_t)p->batch * p->seqlen;
  a.S = std::max(p->seqlen, 1);
  a.D = p->head_dim;
  a.half = p->rotary_dim / 2;
  a.turning = p->rotary_dim / (2 * v);
  a.items = p->head_dim / (2 * v);
  a.idx64 = p->index_int64 != 0;
  a.w32 = p->weight_dtype == MIMIR_DTYPE_FLOAT32;
  a.amplitude = p->amplitude;
  a.eps = p->eps;
  a.lanes = 8;
  while (a.lanes < a.items) a.lanes *= 2;
  if (a.lanes > 64)
    return fail_with(MIMIR_ERR_UNSUPPORTED_SHAPE, "head_dim " + std::to_string(p->head_dim) + " with rotary_dim " + std::to_string(p->rotary_dim) +
                                                      " and these strides is read " + std::to_string(v) + " columns at a time: at most " +
                                                      std::to_string(128 * v) + " columns then");
  // Outputs share no memory with an input, each other or themselves: lanes write what others read.
  const int64_t run = (int64_t)p->head_dim * es;
  auto region = [&](const void* x, int64_t sb, int64_t st, int64_t sh, int heads) {
    return Region{x, run, {p->batch, p->seqlen, heads}, {sb * es, st * es, sh * es}};
  };
  if (!empty) {
    const Region outs[2] = {region(a.q.y, a.q.y_sb, a.q.y_st, a.q.y_sh, a.q.heads), region(a.k.y, a.k.y_sb, a.k.y_st, a.k.y_sh, a.k.heads)};
    const Region ins[4] = {region(a.q.x, a.q.x_sb, a.q.x_st, a.q.x_sh, a.q.heads), region(a.q.dy, a.q.dy_sb, a.q.dy_st, a.q.dy_sh, a.q.heads),
                           region(a.k.x, a.k.x_sb, a.k.x_st, a.k.x_sh, a.k.heads), region(a.k.dy, a.k.dy_sb, a.k.dy_st, a.k.dy_sh, a.k.heads)};
    bool apart = !k || !overlap_each_other(outs[0], outs[1]);
    for (int o = 0; o < (k ? 2 : 1); ++o) {
      apart = apart && !overlaps_itself(outs[o]);
      for (int i = 0; i < (k ? 4 : 2); ++i)
        if (i % 2 == 0 || bwd) apart = apart && !overlap_each_other(outs[o], ins[i]);
    }
    if (!apart) return fail_with(MIMIR_ERR_UNSUPPORTED_SHAPE, "norm_rotary outputs need memory of their own");
  }
  // Four query heads a group, or fewer until there are threads for the whole chip (256 CUs x 16 waves).
  const int heads = std::max(a.q.heads, a.k.heads);
  a.hp = (heads + 3) / 4;
  while (a.hp < heads && a.tokens * a.lanes * a.hp < (int64_t)256 * 16 * 64) a.hp *= 2;
  a.hp = std::min(a.hp, heads);
  const int64_t groups = a.tokens * a.hp;
  const int64_t blocks = bwd ? bwd_blocks(groups, a.lanes) : (groups * a.lanes + 255) / 256;
  if (blocks > kMaxGroups || (bwd && groups > 0x7fffffff)) return fail_with(MIMIR_ERR_UNSUPPORTED_SHAPE, "too many tokens for one launch");
  if (sums) {
    if (p->workspace_bytes < mimir_prefixlm_norm_rotary_workspace_bytes(p) || (p->workspace == nullptr && blocks > 0))
      return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "norm_rotary workspace of " + std::to_string(p->workspace_bytes) + " bytes, needs " +
                                                       std::to_string(mimir_prefixlm_norm_rotary_workspace_bytes(p)));
    if ((uintptr_t)p->workspace % 4 != 0) return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "the workspace must be aligned to 4 bytes");
    a.part = (float*)p->workspace;
  }
  const hipStream_t s = (hipStream_t)stream;
  const bool il = p->interleaved != 0;
  if (blocks > 0) {
    if (es == 2) {
      if (v == 8) launch_norm_rotary<bf16_t, 8>(a, il, bwd, blocks, s);
      else if (v == 4) launch_norm_rotary<bf16_t, 4>(a, il, bwd, blocks, s);
      else if (v == 2) launch_norm_rotary<bf16_t, 2>(a, il, bwd, blocks, s);
      else launch_norm_rotary<bf16_t, 1>(a, il, bwd, blocks, s);
    } else {
      if (v == 4) launch_norm_rotary<float, 4>(a, il, bwd, blocks, s);
      else if (v == 2) launch_norm_rotary<float, 2>(a, il, bwd, blocks, s);
      else launch_norm_rotary<float, 1>(a, il, bwd, blocks, s);
    }
  }
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && sums) {
    const WeightSumArgs w = {a.part, {p->dq_weight, p->dk_weight}, (int)blocks, a.D, a.w32};
    hipLaunchKernelGGL(norm_weight_sum_kernel, dim3((unsigned)((2 * a.D + kSumCols - 1) / kSumCols)), dim3(1024), 0, s, w);
    e = hipGetLastError();
  }
  return e == hipSuccess ? MIMIR_OK : fail_with(MIMIR_ERR_HIP, std::string("norm_rotary launch: ") + hipGetErrorString(e));
}

}  // namespace
}  // namespace mimir

extern "C" size_t mimir_prefixlm_norm_rotary_workspace_bytes(const MimirNormRotaryParams* p) {
  if (p == nullptr || p->head_dim <= 0 || (p->dq_weight == nullptr && p->dk_weight == nullptr)) return 0;
  // at most kMaxBlocks rows, and no more than groups of 8 lanes or more could fill
  const int64_t groups = (int64_t)std::max(p->batch, 0) * std::max(p->seqlen, 0) * std::max(p->num_q_heads, std::max(p->num_kv_heads, 1));
  return (size_t)mimir::bwd_blocks(groups, 64) * 2 * (size_t)p->head_dim * sizeof(float);
}
extern "C" int mimir_prefixlm_norm_rotary(const MimirNormRotaryParams* p, void* stream) {
  return mimir::run_norm_rotary(p, false, stream);
}
extern "C" int mimir_prefixlm_norm_rotary_bwd(const MimirNormRotaryParams* p, void* stream) {
  return mimir::run_norm_rotary(p, true, stream);
}
