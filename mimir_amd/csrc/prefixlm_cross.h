// Shared by the cross-attention kernels: packed sequences with their gradient
// (prefixlm_cross_bf16.hip, prefixlm_cross_bwd_bf16.hip) and few queries over rows of a static cache
// (prefixlm_states_bf16.hip).
#pragma once

#include <algorithm>

#include "prefixlm_common.h"

namespace mimir {

// Where each sequence's queries and states lie, as rows of q and of k / v.  Packed: cumulative lengths.
// States (cu_q NULL): sequence s is the `per_seq` query rows from s * per_seq on, over the first lengths[r]
// of the `length` positions of cache row r = rows[s] (or s), which starts `pitch` rows of k / v after the row
// before; a row outside the cache has none.
struct SeqTable {
  const int32_t *cu_q, *cu_k;
  const void *lengths, *rows;
  int n, Tq, Tk;
  int per_seq, length, pitch, pool, len64, row64;
};
struct SeqSpan {
  int q0, nq, k0, nk;
};
__device__ __forceinline__ int64_t load_whole(const void* p, int64_t i, int idx64) {
  return idx64 ? ((const int64_t*)p)[i] : (int64_t)((const int32_t*)p)[i];
}
__device__ __forceinline__ SeqSpan seq_span(const SeqTable& t, int s) {
  SeqSpan g;
  if (t.cu_q != nullptr) {  // clamped, so that malformed lengths address nothing outside
    g.q0 = min(max(t.cu_q[s], 0), t.Tq);
    g.nq = min(max(t.cu_q[s + 1], g.q0), t.Tq) - g.q0;
    g.k0 = min(max(t.cu_k[s], 0), t.Tk);
    g.nk = min(max(t.cu_k[s + 1], g.k0), t.Tk) - g.k0;
  } else {
    const int64_t r = t.rows != nullptr ? load_whole(t.rows, s, t.row64) : s;
    const bool ok = r >= 0 && r < t.pool;
    const int64_t len = ok ? load_whole(t.lengths, r, t.len64) : 0;
    g.q0 = s * t.per_seq;
    g.nq = t.per_seq;
    g.k0 = ok ? (int)r * t.pitch : 0;
    g.nk = (int)min(max(len, (int64_t)0), (int64_t)t.length);
  }
  return g;
}

struct CrossArgs {
  const bf16_t *q, *k, *v, *dout;
  bf16_t *o, *o_lo, *dq, *dk, *dv;  // o_lo: contiguous, or NULL
  float* lse2;   // [Hq, Tq]: log2 of the softmax's sum, scale included; -inf for a row without states
  float* delta;  // [Hq, Tq]: rowsum(dO * O), O with its low half
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh, o_st, o_sh, do_st, do_sh, dq_st, dq_sh, dk_st, dk_sh, dv_st, dv_sh;
  int Tq, Hq, Hkv, group;
  const int4* plan_q;  // query tiles: (first row, rows, first state, states), most states first; no rows: padding
  const int4* plan_k;  // tiles of states: (first state, states, first query, queries)
  int cap_q, cap_k;    // entries
  float scale, scale_log2;
};

inline size_t align_up(size_t x) { return (x + 255) & ~(size_t)255; }
// Over at most this many states the forward takes P as two bf16 halves in its product: where few terms make a sum,
// their roundings do not average out, and they would reach dS through delta (dK of 6 sequences over 3 to 20 states: error
// against 64 bits 1.52 of that of rounding the exact result, with two halves 1.44).
constexpr int kSplitStates = 64;

constexpr int kCrossTile = 128;  // query rows or states of a tile
// Entries of a list for any packing of `total` rows into n sequences.
inline int cross_capacity(int total, int n) {
  return total > 0 && n > 0 ? (int)std::min<int64_t>(((int64_t)total + kCrossTile - 1) / kCrossTile + n, 0x7fffffff) : 0;
}

// A query tile of the list (rows 0: padding) and its head.  Unit = list entry * Hkv + kv head on XCD unit % 8, its
// query heads at consecutive slots there: they read the same K and V through one L2.
struct QueryTile {
  int4 item;
  int h, hk;
};
__device__ __forceinline__ QueryTile query_tile(const CrossArgs& a) {
  const int xcd = blockIdx.x % kXcds, slot = blockIdx.x / kXcds;
  const int unit = (slot / a.group) * kXcds + xcd;
  const int rank = min(unit / a.Hkv, a.cap_q - 1), hk = unit % a.Hkv;
  QueryTile t = {load_entry(a.plan_q, rank), hk * a.group + slot % a.group, hk};
  if (unit >= a.cap_q * a.Hkv) t.item.y = 0;
  return t;
}

// The launch in front of the tile kernels: the tile lists, and zeros in the rows outside every sequence.
struct CrossPrologue {
  SeqTable seqs;
  int4 *plan_q, *plan_k;  // NULL: not wanted
  int cap_q, cap_k;
  struct Fill {
    bf16_t* x;            // [rows, H, D]
    int64_t st, sh;
    int by_key, heads;
  } fill[3];
  int nfill, D;
  float* lse2;            // of the filled query rows: -inf
};
hipError_t launch_cross_prologue(const CrossPrologue& p, hipStream_t stream);
hipError_t launch_cross_fwd(const CrossArgs& a, int head_dim, hipStream_t stream);
hipError_t launch_cross_bwd(const CrossArgs& a, int head_dim, hipStream_t stream);

}  // namespace mimir
