// Rotary positions from token positions and a frequency table: pairs of columns of
// each head turned by (position * frequency), in either pair layout, over all or the
// first rotary_dim columns, and the gradient (the inverse turn).
//
// Per pair (a, b) of a head's columns and angle t = 2 pi * frac(position * turns / 2^64):
//   a' = amplitude * (a cos t - b sin t)
//   b' = amplitude * (b cos t + a sin t)
// in fp32 with one rounding to the element type; inverse: t -> -t, which is the
// gradient's map (the turn is orthogonal up to amplitude).  Half layout: pair i is
// columns (i, i + rotary_dim / 2); interleaved: columns (2 i, 2 i + 1).
//
// A frequency is held as the fraction of a turn per position in units of 2^-64, so the
// 64-bit product position * turns, which wraps at whole turns, is the range reduction:
// exact for any position and the given turns, where a product in fp32 is a radian off at a million.  The
// nearest quarter turn comes off as integer bits; what is left, at most pi / 4, is rounded to
// fp32 (2^-28 of a turn at most) and goes through the Taylor series (truncated below 2e-9) of sine and cosine.
//
// Bound by reading and writing the heads once.  A thread owns V pairs of columns of one
// token, computes their angles once and takes every hp-th head of q and k with them, so
// the series are shared by the heads and the loads of several heads are in flight
// together.
#include <algorithm>
#include <cmath>

#include "prefixlm_common.h"
#include "rotary_turn.h"
#include "strided_overlap.h"

namespace mimir {
int fail_with(int code, const std::string& msg);

namespace {

struct RotaryArgs {
  const void *q, *k;
  void *qo, *ko;
  const int64_t* turns;
  const void* positions;
  int64_t q_sb, q_st, q_sh, qo_sb, qo_st, qo_sh, k_sb, k_st, k_sh, ko_sb, ko_st, ko_sh, p_sb, p_st;
  int64_t tokens;      // batch * seqlen
  int S, Hq, H;        // H: heads of q and k together
  int half;            // rotary_dim / 2
  int turning, items;  // items of a head that turn, and with those that are copied
  int hp;              // threads that share a (token, item): each takes every hp-th head
  int idx64;
  float amplitude, sign;
};

template <typename E, int N>
using Row = E __attribute__((ext_vector_type(N)));

// An item is 2 V columns of a head: V pairs, or (past the turned ones) 2 V copied columns.
template <typename E, int V, bool kInterleaved>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryArgs a) {
  using R = Row<E, V>;
  constexpr int kBatch = 4;  // heads in flight
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int c = (int)(id % a.items);
  const int64_t rest = id / a.items;
  const int h0 = (int)(rest % a.hp);
  const int64_t token = rest / a.hp;
  if (token >= a.tokens) return;
  const int64_t b = token / a.S, i = token - b * a.S;
  const bool turn = c < a.turning;
  // the item's two runs of V columns: the pairs' halves, or 2 V columns in a row
  const int d1 = turn && !kInterleaved ? c * V : 2 * c * V;
  const int d2 = turn && !kInterleaved ? d1 + a.half : d1 + V;
  float cs[V], sn[V];
  if (turn) {
    const int64_t at = b * a.p_sb + i * a.p_st;
    const uint64_t pos = (uint64_t)(a.idx64 ? ((const int64_t*)a.positions)[at] : (int64_t)((const int32_t*)a.positions)[at]);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      sincos_turn(pos * (uint64_t)a.turns[c * V + e], cs[e], sn[e]);
      cs[e] *= a.amplitude;
      sn[e] *= a.amplitude * a.sign;
    }
  }
  const E* const q = (const E*)a.q + b * a.q_sb + i * a.q_st;
  const E* const k = (const E*)a.k + b * a.k_sb + i * a.k_st;
  E* const qo = (E*)a.qo + b * a.qo_sb + i * a.qo_st;
  E* const ko = (E*)a.ko + b * a.ko_sb + i * a.ko_st;
  for (int hb = h0; hb < a.H; hb += kBatch * a.hp) {
    R x1[kBatch], x2[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int h = min(hb + j * a.hp, a.H - 1);  // past the last head: that one again
      const E* x = h < a.Hq ? q + h * a.q_sh : k + (h - a.Hq) * a.k_sh;
      x1[j] = *(const R*)(x + d1);
      x2[j] = *(const R*)(x + d2);
    }
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int h = hb + j * a.hp;
      if (h >= a.H) break;
      E* y = h < a.Hq ? qo + h * a.qo_sh : ko + (h - a.Hq) * a.ko_sh;
      R y1 = x1[j], y2 = x2[j];
      if (turn) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          // interleaved: pair e is elements 2 e and 2 e + 1 of the run x1 | x2
          const int u = 2 * e, w = 2 * e + 1;
          const float p = kInterleaved ? (float)(u < V ? x1[j][u % V] : x2[j][u % V]) : (float)x1[j][e];
          const float r = kInterleaved ? (float)(w < V ? x1[j][w % V] : x2[j][w % V]) : (float)x2[j][e];
          const E o1 = (E)(p * cs[e] - r * sn[e]), o2 = (E)(r * cs[e] + p * sn[e]);
          if constexpr (kInterleaved) {
            (u < V ? y1 : y2)[u % V] = o1;
            (w < V ? y1 : y2)[w % V] = o2;
          } else {
            y1[e] = o1;
            y2[e] = o2;
          }
        }
      }
      *(R*)(y + d1) = y1;
      *(R*)(y + d2) = y2;
    }
  }
}

template <typename E, int V>
void launch_rotary(const RotaryArgs& a, bool interleaved, hipStream_t stream) {
  const int64_t blocks = (a.tokens * a.items * a.hp + 255) / 256;
  if (interleaved)
    hipLaunchKernelGGL((rotary_kernel<E, V, true>), dim3((unsigned)blocks), dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((rotary_kernel<E, V, false>), dim3((unsigned)blocks), dim3(256), 0, stream, a);
}

// By name: of several instantiations launched above, this toolchain drops host stubs.
#define ROTARY(E, V) \
  template __global__ void rotary_kernel<E, V, true>(const RotaryArgs); \
  template __global__ void rotary_kernel<E, V, false>(const RotaryArgs);
ROTARY(bf16_t, 8) ROTARY(bf16_t, 4) ROTARY(bf16_t, 2) ROTARY(bf16_t, 1)
ROTARY(float, 4) ROTARY(float, 2) ROTARY(float, 1)
#undef ROTARY

}  // namespace
}  // namespace mimir

extern "C" int mimir_prefixlm_rotary(const MimirRotaryParams* p, void* stream) {
  using mimir::fail_with;
  fail_with(MIMIR_OK, "");
  if (p == nullptr) return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "params is NULL");
  if (p->dtype != MIMIR_DTYPE_FLOAT32 && p->dtype != MIMIR_DTYPE_BFLOAT16)
    return fail_with(MIMIR_ERR_UNSUPPORTED_DTYPE, "rotary positions support float32 and bfloat16 tensors only (dtype code " +
                                                      std::to_string(p->dtype) + ")");
  if (p->batch < 0 || p->seqlen < 0 || p->num_q_heads <= 0 || p->num_kv_heads < 0 || p->head_dim <= 0)
    return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "negative size or non-positive heads / head_dim");
  if (p->head_dim % 2 != 0 || p->rotary_dim % 2 != 0 || p->rotary_dim < 2 || p->rotary_dim > p->head_dim)
    return fail_with(MIMIR_ERR_UNSUPPORTED_SHAPE, "rotary_dim " + std::to_string(p->rotary_dim) + " must be even and in [2, head_dim " +
                                                      std::to_string(p->head_dim) + "], which must be even");
  if (!std::isfinite(p->amplitude)) return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "amplitude must be finite");
  if (p->batch == 0 || p->seqlen == 0) return MIMIR_OK;
  const bool k = p->num_kv_heads > 0;
  if (p->q == nullptr || p->q_out == nullptr || (k && (p->k == nullptr || p->k_out == nullptr)) || p->turns == nullptr ||
      p->positions == nullptr)
    return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "rotary tensor pointer is NULL");
  mimir::RotaryArgs a = {};
  a.q = p->q; a.qo = p->q_out; a.k = p->k; a.ko = p->k_out;
  a.turns = p->turns;
  a.positions = p->positions;
  a.q_sb = p->q_stride_batch; a.q_st = p->q_stride_token; a.q_sh = p->q_stride_head;
  a.qo_sb = p->q_out_stride_batch; a.qo_st = p->q_out_stride_token; a.qo_sh = p->q_out_stride_head;
  a.k_sb = p->k_stride_batch; a.k_st = p->k_stride_token; a.k_sh = p->k_stride_head;
  a.ko_sb = p->k_out_stride_batch; a.ko_st = p->k_out_stride_token; a.ko_sh = p->k_out_stride_head;
  a.p_sb = p->positions_stride_batch; a.p_st = p->positions_stride_token;
  a.tokens = (int64_t)p->batch * p->seqlen;
  a.S = p->seqlen;
  a.Hq = p->num_q_heads;
  a.H = p->num_q_heads + p->num_kv_heads;
  a.half = p->rotary_dim / 2;
  a.idx64 = p->index_int64 != 0;
  a.amplitude = p->amplitude;
  a.sign = p->inverse ? -1.f : 1.f;
  // Columns per access: as many as both parts of the head, the addresses and the strides
  // are multiples of, up to 16 bytes.
  const int es = p->dtype == MIMIR_DTYPE_BFLOAT16 ? 2 : 4;
  int v = 16 / es;
  const int64_t strides[12] = {a.q_sb, a.q_st, a.q_sh, a.qo_sb, a.qo_st, a.qo_sh, a.k_sb, a.k_st, a.k_sh, a.ko_sb, a.ko_st, a.ko_sh};
  auto fits = [&](int n) {
    if (p->rotary_dim % (2 * n) != 0 || (p->head_dim - p->rotary_dim) % (2 * n) != 0) return false;
    for (int s = 0; s < (k ? 12 : 6); ++s)
      if (strides[s] % n != 0) return false;
    const uintptr_t bytes = (uintptr_t)n * es;
    return (uintptr_t)a.q % bytes == 0 && (uintptr_t)a.qo % bytes == 0 && (!k || ((uintptr_t)a.k % bytes == 0 && (uintptr_t)a.ko % bytes == 0));
  };
  while (v > 1 && !fits(v)) v /= 2;
  if ((uintptr_t)a.q % es != 0 || (uintptr_t)a.qo % es != 0 || (k && ((uintptr_t)a.k % es != 0 || (uintptr_t)a.ko % es != 0))) return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "rotary tensors must be aligned to their elements");
  a.turning = p->rotary_dim / (2 * v);
  // In place the columns past rotary_dim are there already.
  const bool in_place = a.q == a.qo && (!k || a.k == a.ko);
  // Threads write what others read: an output is its own input, element by element, or shares nothing with
  // one, with the other output or with itself.
  const int64_t run = (int64_t)(in_place ? p->rotary_dim : p->head_dim) * es;
  auto region = [&](const void* x, int64_t sb, int64_t st, int64_t sh, int heads) {
    return mimir::Region{x, run, {p->batch, p->seqlen, heads}, {sb * es, st * es, sh * es}};
  };
  const mimir::Region q_in = region(a.q, a.q_sb, a.q_st, a.q_sh, a.Hq), k_in = region(a.k, a.k_sb, a.k_st, a.k_sh, a.H - a.Hq);
  const mimir::Region q_out = region(a.qo, a.qo_sb, a.qo_st, a.qo_sh, a.Hq), k_out = region(a.ko, a.ko_sb, a.ko_st, a.ko_sh, a.H - a.Hq);
  auto same = [](const mimir::Region& x, const mimir::Region& y) {
    bool all = x.base == y.base;
    for (int i = 0; i < mimir::Region::kDims; ++i) all = all && (x.size[i] == 1 || x.stride[i] == y.stride[i]);
    return all;
  };
  auto apart = [&](const mimir::Region& out, const mimir::Region& own, const mimir::Region& others) {
    return !overlaps_itself(out) && (same(out, own) || !overlap_each_other(out, own)) && !overlap_each_other(out, others);
  };
  if (!apart(q_out, q_in, k_in) || (k && (!apart(k_out, k_in, q_in) || overlap_each_other(q_out, k_out))))
    return fail_with(MIMIR_ERR_UNSUPPORTED_SHAPE, "rotary outputs need memory of their own: elements that overlap would be turned twice");
  a.items = in_place ? a.turning : p->head_dim / (2 * v);
  // Four heads a thread, all in flight at once, or fewer until there are threads for the whole chip (256 CUs
  // x 16 waves).  One thread for all heads while the tokens fill the chip / so: 16384 tokens, 20 heads of 128,
  // 37.9 / 34.6 us (4.9 TB/s, a large copy's 5.1), 32768 tokens, 40 heads, half turned, 150 / 127 (5.3 TB/s),
  // 24000 tokens, 4 heads, 13.8 / 10.4.  Two or eight heads are within 2%; non-temporal loads or stores slower
  // (127 -> 136, 227).
  a.hp = (a.H + 3) / 4;
  while (a.hp < a.H && a.tokens * a.items * a.hp < (int64_t)256 * 16 * 64) a.hp *= 2;
  a.hp = std::min(a.hp, a.H);
  if ((a.tokens * a.items * a.hp + 255) / 256 > mimir::kMaxGroups) return fail_with(MIMIR_ERR_UNSUPPORTED_SHAPE, "too many tokens for one launch");
  const hipStream_t s = (hipStream_t)stream;
  const bool il = p->interleaved != 0;
  if (es == 2) {
    if (v == 8) mimir::launch_rotary<mimir::bf16_t, 8>(a, il, s);
    else if (v == 4) mimir::launch_rotary<mimir::bf16_t, 4>(a, il, s);
    else if (v == 2) mimir::launch_rotary<mimir::bf16_t, 2>(a, il, s);
    else mimir::launch_rotary<mimir::bf16_t, 1>(a, il, s);
  } else {
    if (v == 4) mimir::launch_rotary<float, 4>(a, il, s);
    else if (v == 2) mimir::launch_rotary<float, 2>(a, il, s);
    else mimir::launch_rotary<float, 1>(a, il, s);
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MIMIR_OK : fail_with(MIMIR_ERR_HIP, std::string("rotary launch: ") + hipGetErrorString(e));
}
