// Cross attention of few queries, the decode step of prefixlm_cross_bf16.hip: each request's queries
// (the tokens of all its beams, times the query heads of a kv head: its rows) over one row of a static
// cache of states.  All rows of a request see the same states, so they share one reading of them.
//
// Bound by that reading.  The states of all requests, in units of 64, form one line, which is dealt evenly to
// shares found on the device from the lengths; a share is one workgroup per kv head, the heads of a
// share, whose states are adjacent in memory, side by side.  A workgroup is two waves, each with every second
// 32-state tile of a request in two LDS stages of its own, waiting only for its own copies.  S^T = K Q^T leaves a row in a
// lane, P^T is the B operand of O^T += V^T P^T (prefixlm_fwd_bf16.hip); one or two sets of 32 rows
// take part in each tile.  The waves meet in LDS; a request inside one share is finished there,
// the parts of the others go to the workspace and states_merge_kernel adds them in order.  48 requests of 8 beams over 300 to
// 4096 states, 16 / 4 heads of 128: 48.9 us (4.4 TB/s) and 6.5; one request of 1500 states 7.3 and 5.4, round trips.
//
// Requests of more than 128 rows go to the tile kernel of prefixlm_cross_bf16.hip instead, whatever their number: it splits no
// states and reads them once for each query head (one request of 16384 states, 64 / 8 heads of 128: 128 rows 38 us, 256 rows 281).
#include <algorithm>

#include "prefixlm_cross.h"

namespace mimir {
namespace {

constexpr int kTile = 32;      // states of a wave's tile
constexpr int kShareWaves = 2;
constexpr int kUnit = kTile * kShareWaves;
constexpr int kShareGroups = 512;  // workgroups of all shares and kv heads: two on each of 256 CUs

struct StatesArgs {
  const bf16_t *q, *k, *v;
  bf16_t* o;
  SeqTable seqs;
  int64_t q_st, q_sh, k_sb, k_st, k_sh, v_sb, v_st, v_sh, o_st, o_sh;
  int Hkv, group, rows;  // rows: seq_tokens * group
  int shares;
  float scale_log2;
  float *part_o, *part_ml;  // [row tile][2 shares][Hkv][rows of a tile](D | maximum in log2, sum)
  int4* where;              // of each request, by the first workgroup: first share, shares (0: no states), whether it
                            // begins its first share
};

// The line of units, 64 requests at a time, one a lane.
struct Line {
  int first;  // request of lane 0
  int row;    // cache row
  int keys, units, incl;
  __device__ __forceinline__ void load(const SeqTable& t, int first_, int before, int lane) {
    first = first_;
    row = keys = 0;
    if (first + lane < t.n) {
      const int64_t r = t.rows != nullptr ? load_whole(t.rows, first + lane, t.row64) : first + lane;
      if (r >= 0 && r < t.pool) {
        row = (int)r;
        keys = (int)min(max(load_whole(t.lengths, r, t.len64), (int64_t)0), (int64_t)t.length);
      }
    }
    units = (keys + kUnit - 1) / kUnit;
    incl = before + wave_inclusive_sum(units);
  }
  __device__ __forceinline__ int end() const { return __builtin_amdgcn_readlane(incl, 63); }
};
__device__ __forceinline__ int line_length(const SeqTable& t, Line& line, int lane) {
  int total = 0;
  for (int s = 0; s < t.n; s += 64) {
    line.load(t, s, total, lane);
    total = line.end();
  }
  return total;
}
// A line's units dealt to shares: `each`, and one more to the first `more`.
struct Deal {
  int each, more;
  __device__ __forceinline__ Deal(int total, int shares) : each((int)((uint32_t)total / (uint32_t)shares)), more(total - each * shares) {}
  __device__ __forceinline__ int start(int i) const { return i * each + min(i, more); }
  __device__ __forceinline__ int share_of(int u) const {  // that holds unit u
    const int longer = more * (each + 1);
    return u < longer ? (int)((uint32_t)u / (uint32_t)(each + 1)) : more + (int)((uint32_t)(u - longer) / (uint32_t)max(each, 1));
  }
};
// A share's parts of requests that go on in another: that of its first request, and of its last.
__device__ __forceinline__ int64_t part_slot(const StatesArgs& a, int tile, int share, bool first, int hk, int tile_rows) {
  return ((((int64_t)tile * a.shares + share) * 2 + !first) * a.Hkv + hk) * tile_rows;
}

template <int N>
__device__ __forceinline__ void wait_vmcnt_wide() {
  static_assert(N >= 0 && N < 64, "vmcnt field");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | 0x0F70);
}
__device__ __forceinline__ void lds_barrier() {  // for LDS data alone: copies and stores stay in flight
  __asm__ volatile("" ::: "memory");
  wait_lds();
  __builtin_amdgcn_s_barrier();
  __asm__ volatile("" ::: "memory");
}

// kOnce: the states are read past the caches (the builtin's bit for streaming).
template <int D, int NT, bool kOnce>
__device__ __forceinline__ void states_body(const StatesArgs& a) {
  constexpr int DT = D / 32, KS = D / 16;
  // P enters its product as two bf16 halves where one row tile takes part, which leaves the matrix units idle: error
  // against 64 bits 0.0021 -> 0.0017 of the output, one rounding's, at 54.4 us where 54.2 were spent (48 requests of 300 to 4096
  // states, 32 rows).  Two row tiles (96 rows): 107 us where 99 were spent, so P is rounded to bf16 there.
  constexpr bool kSplit = NT == 1;
  using L = TileLayout<D>;
  constexpr int kInst = (kTile * L::kRowUnits + 63) / 64;  // wave copy instructions per tile
  constexpr int kElems = kInst * 512;
  constexpr int kPitch = D + 4, kRows = 32 * NT;
  // Each stage an object of its own, for both waves: the compiler tells the reads of one from the copies into
  // another.  After a request the second ones hold the waves' partial rows, 32 at a time, with their
  // maxima and sums.
  __shared__ __attribute__((aligned(16))) bf16_t sK0[kShareWaves * kElems];
  __shared__ __attribute__((aligned(16))) bf16_t sV0[kShareWaves * kElems];
  __shared__ __attribute__((aligned(16))) bf16_t sK1[kShareWaves * kElems];
  __shared__ __attribute__((aligned(16))) bf16_t sV1[kShareWaves * kElems];
  static_assert(32 * kPitch * 4 + 32 * 8 <= kShareWaves * kElems * 2, "a wave's partial rows fit one stage object");
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, hi = lane >> 5;
  const int share = blockIdx.x / a.Hkv, hk = blockIdx.x - share * a.Hkv, rt = blockIdx.y;
  bf16_t *const mk0 = sK0 + wave * kElems, *const mv0 = sV0 + wave * kElems;
  bf16_t *const mk1 = sK1 + wave * kElems, *const mv1 = sV1 + wave * kElems;

  Line line;
  const int total = line_length(a.seqs, line, lane);
  const Deal deal(total, a.shares);
  const int u_begin = deal.start(share), u_end = deal.start(share + 1);
  if (blockIdx.x == 0 && rt == 0 && wave == 0) {  // for the merge, which would look all this up again
    int before = 0;
    for (int s = 0; s < a.seqs.n; s += 64) {
      if (a.seqs.n > 64) line.load(a.seqs, s, before, lane);
      before = line.end();
      const int u0 = line.incl - line.units, i0 = deal.share_of(u0);
      if (s + lane < a.seqs.n)
        a.where[s + lane] = line.units > 0 ? make_int4(i0, deal.share_of(line.incl - 1) - i0 + 1, deal.start(i0) == u0, 0) : make_int4(0, 0, 0, 0);
    }
  }
  if (u_begin >= u_end) return;
  if (a.seqs.n > 64) {
    int before = 0;
    for (int s = 0;; s += 64) {
      line.load(a.seqs, s, before, lane);
      before = line.end();
      if (before > u_begin) break;
    }
  }
  uint32_t voffk[kInst], voffv[kInst];
#pragma unroll
  for (int i = 0; i < kInst; ++i) {
    const int u = i * 64 + lane, prow = u / L::kRowUnits, c = u - prow * L::kRowUnits, key = L::unperm(prow);
    const bool data = c < L::kUnits && prow < kTile;
    voffk[i] = data ? (uint32_t)((key * a.k_st + c * 8) * 2) : 0x80000000u;
    voffv[i] = data ? (uint32_t)((key * a.v_st + c * 8) * 2) : 0x80000000u;
  }
  const TileLanes<D> tl(lane);
  const float c2 = a.scale_log2;

  for (int u0 = u_begin; u0 < u_end;) {
    while (line.end() <= u0) line.load(a.seqs, line.first + 64, line.end(), lane);
    const int j = __builtin_ctzll(__builtin_amdgcn_ballot_w64(line.incl > u0));
    const int s = line.first + j;
    const int keys = __builtin_amdgcn_readlane(line.keys, j), crow = __builtin_amdgcn_readlane(line.row, j);
    const int units = __builtin_amdgcn_readlane(line.units, j);
    const int unit0 = u0 - (__builtin_amdgcn_readlane(line.incl, j) - units);
    const int unit1 = min(units, unit0 + u_end - u0);
    const bool whole = unit0 == 0 && unit1 == units, first = u0 == u_begin;
    u0 += unit1 - unit0;
    const int key_end = min(unit1 * kUnit, keys);
    const int t0 = unit0 * kShareWaves + wave;  // this wave's first tile
    const int n_my = t0 * kTile < key_end ? ((key_end + kTile - 1) / kTile - t0 + kShareWaves - 1) / kShareWaves : 0;
    const bf16_t* const kbase = a.k + crow * a.k_sb + hk * a.k_sh;
    const bf16_t* const vbase = a.v + crow * a.v_sb + hk * a.v_sh;
    auto issue = [&](int i, bf16_t* tk, bf16_t* tv) __attribute__((always_inline)) {
      // past the wave's tiles: empty buffers, zeros for a free stage, so that every step waits alike
      const int key0 = (t0 + min(i, max(n_my - 1, 0)) * kShareWaves) * kTile, n = i < n_my ? min(keys - key0, kTile) : 0;
      const __amdgpu_buffer_rsrc_t rk = make_rsrc(kbase + key0 * a.k_st, rows_bytes32(n, (uint32_t)a.k_st, D));
      const __amdgpu_buffer_rsrc_t rv = make_rsrc(vbase + key0 * a.v_st, rows_bytes32(n, (uint32_t)a.v_st, D));
#pragma unroll
      for (int e = 0; e < kInst; ++e)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, (__attribute__((address_space(3))) void*)(tk + e * 512), 16, voffk[e], 0, 0, kOnce ? 2 : 0);
#pragma unroll
      for (int e = 0; e < kInst; ++e)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, (__attribute__((address_space(3))) void*)(tv + e * 512), 16, voffv[e], 0, 0, kOnce ? 2 : 0);
    };
    // Q^T B-operand fragments; lanes past the rows take the last row: their columns are not read
    bf16x8 qf[NT][KS];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = min(rt * kRows + n * 32 + l32, a.rows - 1), t = r / a.group;
      const bf16_t* const qrow = a.q + ((int64_t)s * a.seqs.per_seq + t) * a.q_st + (int64_t)(hk * a.group + r - t * a.group) * a.q_sh + 8 * hi;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) qf[n][ks] = *(const bf16x8*)&qrow[16 * ks];
    }
    issue(0, mk0, mv0);
    issue(1, mk1, mv1);
    f32x16 oacc[NT][DT];
    float m_run[NT], l_run[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m_run[n] = -INFINITY;
      l_run[n] = 0.f;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) oacc[n][dt] = f32x16{};
    }
    auto compute = [&](int i, const bf16_t* sK, const bf16_t* sV) __attribute__((always_inline)) {
      const int key0 = (t0 + i * kShareWaves) * kTile;
      f32x16 st[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) st[n] = f32x16{};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const bf16x8 kf = *(const bf16x8*)&sK[tl.op_base + ks * 16];
#pragma unroll
        for (int n = 0; n < NT; ++n) st[n] = mfma32(kf, qf[n][ks], st[n]);
      }
      bf16x8 pf[NT][2], pl[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        if (key0 + kTile > keys) {  // the last tile reaches past the states
          __asm__ volatile("");
          const int left = keys - key0 - 4 * hi;
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (8 * (r >> 2) + (r & 3) >= left) st[n][r] = -INFINITY;
        }
        float mx = -INFINITY;
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, st[n][r]);
        // P is taken under the running maximum: at most 1, its sum in fp32
        const float m_new = fmaxf(m_run[n], xor32_max(mx));
        const float alpha = m_run[n] == -INFINITY ? 1.f : fast_exp2((m_run[n] - m_new) * c2);
        l_run[n] *= alpha;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) oacc[n][dt] *= alpha;
        m_run[n] = m_new;
        const float mb = m_new == -INFINITY ? 0.f : m_new * c2;
        float lsum = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float pr = fast_exp2(__builtin_fmaf(st[n][r], c2, -mb));
          st[n][r] = pr;
          lsum += pr;
        }
        l_run[n] += lsum;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
          f32x8 t;
#pragma unroll
          for (int e = 0; e < 8; ++e) t[e] = st[n][8 * kk + e];
          pf[n][kk] = to_bf16x8(t);
          if constexpr (kSplit) pl[n][kk] = lo_half(t, pf[n][kk]);
        }
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
          const bf16_t* vp = &sV[tl.tr_base + kk * 16 * L::kRowElems + dt * 32];
          const bf16x8 vf = cat8(lds_read_tr16(vp), lds_read_tr16(vp + L::kTrSecond));
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            oacc[n][dt] = mfma32(vf, pf[n][kk], oacc[n][dt]);
            if constexpr (kSplit) oacc[n][dt] = mfma32(vf, pl[n][kk], oacc[n][dt]);
          }
        }
    };
    // Tile i has landed once at most the copies of tile i + 1 are outstanding; a stage is refilled once this wave's
    // reads of it are done.
    for (int i = 0; i < n_my; i += 2) {
      wait_vmcnt_wide<2 * kInst>();
      __asm__ volatile("" ::: "memory");
      compute(i, mk0, mv0);
      __asm__ volatile("" ::: "memory");
      wait_lds();
      issue(i + 2, mk0, mv0);
      if (i + 1 >= n_my) break;
      wait_vmcnt_wide<2 * kInst>();
      __asm__ volatile("" ::: "memory");
      compute(i + 1, mk1, mv1);
      __asm__ volatile("" ::: "memory");
      wait_lds();
      issue(i + 3, mk1, mv1);
    }
    __asm__ volatile("" ::: "memory");
    wait_vmcnt_wide<0>();  // the last copies
    wait_lds();
    // The waves' partial rows meet in LDS.
    auto area = [&](int w) __attribute__((always_inline)) { return (float*)(w == 0 ? sK1 : sV1); };
    auto ml_of = [&](int w, int r) __attribute__((always_inline)) { return (f32x2*)(area(w) + 32 * kPitch) + r; };
    constexpr int kLanes = D / 4, kRowsAt = 64 / kLanes;  // lanes of a row, four columns each; rows at a time
    const int col = lane % kLanes * 4;
    const int64_t slot = part_slot(a, rt, share, first, hk, kRows);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      lds_barrier();  // both waves are done with their second stages, or with the last rows
      const float l_tot = xor32_sum(l_run[n]);
      if (hi == 0) *ml_of(wave, l32) = f32x2{m_run[n] == -INFINITY ? -INFINITY : m_run[n] * c2, l_tot};
      float* const po = area(wave) + l32 * kPitch;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int rg = 0; rg < 4; ++rg) {
          const f32x4 v = {oacc[n][dt][4 * rg], oacc[n][dt][4 * rg + 1], oacc[n][dt][4 * rg + 2], oacc[n][dt][4 * rg + 3]};
          *(f32x4*)&po[32 * dt + 8 * rg + 4 * hi] = v;
        }
      lds_barrier();
      const int r_first = rt * kRows + n * 32, n_rows = min(a.rows - r_first, 32);
      for (int r0 = wave * kRowsAt; r0 < n_rows; r0 += kShareWaves * kRowsAt) {
        const int rr = r0 + lane / kLanes;
        if (rr >= n_rows) break;
        const f32x2 p = *ml_of(0, rr), q = *ml_of(1, rr);
        const float M = fmaxf(p[0], q[0]);
        // a wave may have had no tile, or only scores of -inf: maximum -inf, sum 0
        const float wp = p[0] == -INFINITY ? 0.f : fast_exp2(p[0] - M), wq = q[0] == -INFINITY ? 0.f : fast_exp2(q[0] - M);
        const float lsum = p[1] * wp + q[1] * wq;
        const f32x4 acc = *(const f32x4*)&area(0)[rr * kPitch + col] * wp + *(const f32x4*)&area(1)[rr * kPitch + col] * wq;
        if (whole) {
          const int r = r_first + rr, t = r / a.group;
          bf16_t* const orow = a.o + ((int64_t)s * a.seqs.per_seq + t) * a.o_st + (int64_t)(hk * a.group + r - t * a.group) * a.o_sh;
          *(bf16x4*)&orow[col] = __builtin_convertvector(acc * (1.f / lsum), bf16x4);
        } else {
          const int64_t at = slot + n * 32 + rr;
          *(f32x4*)&a.part_o[at * D + col] = acc;
          if (col == 0) *(f32x2*)&a.part_ml[at * 2] = f32x2{M, lsum};
        }
      }
    }
    lds_barrier();  // the areas are stages again
  }
}

// One wave per row: the parts of a request that lies in several shares, or zeros for one without states.
template <int D>
__device__ __forceinline__ void states_merge_body(const StatesArgs& a, int tile_rows) {
  constexpr int kLanes = D / 4, kParts = 64 / kLanes;  // lanes of a part's row; parts at a time
  const int lane = threadIdx.x & 63;
  const uint32_t id = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int pair = (int)(id / (uint32_t)a.rows), r = (int)(id - pair * (uint32_t)a.rows), s = pair / a.Hkv, hk = pair - s * a.Hkv;
  if (s >= a.seqs.n) return;
  const int4 where = a.where[s];
  const int i0 = where.x, n = where.y;
  const int t = r / a.group, col = lane % kLanes * 4, sub = lane / kLanes;
  bf16_t* const orow = a.o + ((int64_t)s * a.seqs.per_seq + t) * a.o_st + (int64_t)(hk * a.group + r - t * a.group) * a.o_sh;
  if (n == 0) {
    if (sub == 0) *(bf16x4*)&orow[col] = bf16x4{};
    return;
  }
  if (n == 1) return;  // finished in its share
  const int tile = r / tile_rows;
  // Shares after the first begin inside the request: theirs is the part of their first request.  None is empty: a line
  // of fewer units than shares fills the first ones.  The parts' maxima are met on the way, so that one round trip
  // brings all there is to load.
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  float M = -INFINITY, lsum = 0.f;
  auto add = [&](f32x2 ml, f32x4 o) __attribute__((always_inline)) {
    const float top = fmaxf(M, ml[0]);
    const float old = M == -INFINITY ? 0.f : fast_exp2(M - top), w = ml[0] == -INFINITY ? 0.f : fast_exp2(ml[0] - top);
    lsum = lsum * old + ml[1] * w;
    acc = acc * old + o * w;
    M = top;
  };
  constexpr int kAhead = 8;
  for (int i = sub; i < n; i += kAhead * kParts) {
    f32x2 ml[kAhead];
    f32x4 o[kAhead];
#pragma unroll
    for (int e = 0; e < kAhead; ++e) {
      const int part = min(i + e * kParts, n - 1);  // past the last: that one again
      const int64_t at = part_slot(a, tile, i0 + part, part > 0 || where.z != 0, hk, tile_rows) + r - tile * tile_rows;
      ml[e] = *(const f32x2*)&a.part_ml[at * 2];
      o[e] = *(const f32x4*)&a.part_o[at * D + col];
    }
#pragma unroll
    for (int e = 0; e < kAhead; ++e)
      if (i + e * kParts < n) add(ml[e], o[e]);
  }
#pragma unroll
  for (int off = kLanes; off < 64; off <<= 1) {
    f32x2 ml = {__shfl_xor(M, off, 64), __shfl_xor(lsum, off, 64)};
    f32x4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = __shfl_xor(acc[e], off, 64);
    // (max, sum, row) of both groups joined the same way round on either side
    const bool low = (lane & off) == 0;
    const f32x2 own = {M, lsum};
    const f32x4 mine = acc;
    M = low ? own[0] : ml[0];
    lsum = low ? own[1] : ml[1];
    acc = low ? mine : o;
    add(low ? ml : own, low ? o : mine);
  }
  if (sub == 0) *(bf16x4*)&orow[col] = __builtin_convertvector(acc * (1.f / lsum), bf16x4);
}

template <int D, int NT, bool kOnce>
__global__ __launch_bounds__(kShareWaves * 64, 1) void states_kernel(const StatesArgs a) {
  states_body<D, NT, kOnce>(a);
}
template <int D>
__global__ __launch_bounds__(256) void states_merge_kernel(const StatesArgs a, int tile_rows) {
  states_merge_body<D>(a, tile_rows);
}
// By name: of several instantiations launched below, this toolchain drops host stubs.
template __global__ void states_kernel<64, 1, false>(const StatesArgs);
template __global__ void states_kernel<64, 1, true>(const StatesArgs);
template __global__ void states_kernel<64, 2, false>(const StatesArgs);
template __global__ void states_kernel<128, 1, false>(const StatesArgs);
template __global__ void states_kernel<128, 1, true>(const StatesArgs);
template __global__ void states_kernel<128, 2, false>(const StatesArgs);
template __global__ void states_merge_kernel<64>(const StatesArgs, int);
template __global__ void states_merge_kernel<128>(const StatesArgs, int);

// States of a launch that read past the caches where one row tile reads them, once: more than the 256 MiB in front of
// memory cannot be found there by the next step.  It goes by the positions there are, as the lengths are on the device, so that
// large rows with little in them lose what the caches would hold.  48 requests of 300 to 4096 states, 4 kv heads of 128, other states each
// time: 60.2 us with the caches, 54.2 past them (the same states each time: 48.9 and 53.9).  Two row tiles (96 rows): 99 and 108.
constexpr int64_t kOnceBytes = (int64_t)256 << 20;
constexpr int kManyRows = 128;  // more rows per kv head than this: the tile kernel
struct StatesPlan {
  bool tiles;  // the tile kernel
  int pitch;   // of a cache row, in positions
  int cap;     // entries of its list
  int rows, tile_rows, row_tiles, shares;
  bool once;   // the states are read past the caches
  size_t ml, where, total;  // workspace: parts' rows, then maxima and sums, then the requests' shares
};
StatesPlan states_plan(const MimirStatesParams& p) {
  StatesPlan s = {};
  s.rows = p.seq_tokens * (p.num_q_heads / p.num_kv_heads);
  if (s.rows > kManyRows && p.k_stride_token > 0 && p.v_stride_token > 0 && p.k_stride_row % p.k_stride_token == 0 &&
      p.v_stride_row % p.v_stride_token == 0 && p.k_stride_row / p.k_stride_token == p.v_stride_row / p.v_stride_token) {
    const int64_t pitch = p.cache_rows > 1 ? p.k_stride_row / p.k_stride_token : p.cache_len;
    if (pitch >= 0 && pitch * p.cache_rows <= 0x7fffffff) {
      s.tiles = true;
      s.pitch = (int)pitch;
      s.cap = cross_capacity(p.requests * p.seq_tokens, p.requests);
      s.total = (size_t)s.cap * sizeof(int4);
      return s;
    }
  }
  s.tile_rows = s.rows > 32 ? 64 : 32;
  s.row_tiles = (s.rows + s.tile_rows - 1) / s.tile_rows;
  const int64_t units = (int64_t)p.requests * ((p.cache_len + kUnit - 1) / kUnit);
  const int groups = p.head_dim == 64 ? 2 * kShareGroups : kShareGroups;
  s.shares = (int)std::min<int64_t>(std::max(units, (int64_t)1), std::max(groups / (p.num_kv_heads * s.row_tiles), 1));
  s.once = s.tile_rows == 32 && (int64_t)p.requests * p.cache_len * p.num_kv_heads * p.head_dim * 4 >= kOnceBytes;
  const size_t part_rows = (size_t)s.row_tiles * s.shares * 2 * p.num_kv_heads * s.tile_rows;
  s.ml = align_up(part_rows * p.head_dim * sizeof(float));
  s.where = s.ml + align_up(part_rows * 2 * sizeof(float));
  s.total = s.where + align_up((size_t)p.requests * sizeof(int4));
  return s;
}
bool states_sizes(const MimirStatesParams* p) {
  return p != nullptr && p->requests >= 0 && p->seq_tokens >= 0 && p->cache_rows >= 0 && p->cache_len >= 0 && p->num_kv_heads > 0 &&
         p->num_q_heads > 0 && p->num_q_heads % p->num_kv_heads == 0 && (p->head_dim == 64 || p->head_dim == 128) &&
         (int64_t)p->requests * p->seq_tokens * p->num_q_heads <= 0x7fffffff && (int64_t)p->requests * p->cache_len <= 0x7fffffff;
}

}  // namespace
}  // namespace mimir

extern "C" size_t mimir_prefixlm_states_workspace_bytes(const MimirStatesParams* p) {
  return mimir::states_sizes(p) ? mimir::states_plan(*p).total : 0;
}

extern "C" int mimir_prefixlm_states_attn(const MimirStatesParams* p, void* stream) {
  using namespace mimir;
  fail_with(MIMIR_OK, "");
  if (p == nullptr) return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "params is NULL");
  if (p->dtype != MIMIR_DTYPE_BFLOAT16)
    return fail_with(MIMIR_ERR_UNSUPPORTED_DTYPE, "attention to states supports bfloat16 tensors only (dtype code " + std::to_string(p->dtype) + ")");
  if (p->num_q_heads > 0 && p->num_kv_heads > 0 && p->num_q_heads % p->num_kv_heads != 0)
    return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "Query heads " + std::to_string(p->num_q_heads) + " must be divisible by key/value heads " +
                                                     std::to_string(p->num_kv_heads) + ".");
  if (!states_sizes(p))
    return fail_with(MIMIR_ERR_UNSUPPORTED_SHAPE, "attention to states: negative or too large sizes, or a head_dim that is not 64 or 128 (" +
                                                      std::to_string(p->head_dim) + ")");
  if (!(p->softmax_scale > 1e-30f) || !(p->softmax_scale < 1e30f))
    return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "softmax_scale must be positive and neither below 1e-30 nor above 1e30");
  if (p->requests == 0 || p->seq_tokens == 0) return MIMIR_OK;
  const bool states = p->cache_rows > 0 && p->cache_len > 0;
  if (p->q == nullptr || p->out == nullptr || (states && (p->keys == nullptr || p->values == nullptr || p->lengths == nullptr)))
    return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "attention to states tensor pointer is NULL");
  for (const void* x : {p->q, p->keys, p->values, (const void*)p->out})
    if ((uintptr_t)x % 16 != 0) return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "attention to states needs 16-byte aligned rows");
  for (const int64_t st : {p->q_stride_token, p->q_stride_head, p->k_stride_row, p->k_stride_token, p->k_stride_head, p->v_stride_row,
                           p->v_stride_token, p->v_stride_head, p->out_stride_token, p->out_stride_head})
    if (st % 8 != 0) return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "attention to states needs 16-byte aligned rows");
  for (const int64_t st : {p->q_stride_token, p->k_stride_token, p->v_stride_token, p->out_stride_token})
    if (st < p->head_dim || st >= (1 << 22))
      return fail_with(MIMIR_ERR_UNSUPPORTED_SHAPE, "token strides must be at least head_dim and below 2^22 elements");
  for (const int64_t st : {p->q_stride_head, p->k_stride_row, p->k_stride_head, p->v_stride_row, p->v_stride_head, p->out_stride_head})
    if (st < 0) return fail_with(MIMIR_ERR_UNSUPPORTED_SHAPE, "strides must not be negative");
  const StatesPlan plan = states_plan(*p);
  if (plan.total > 0 && (p->workspace == nullptr || (uintptr_t)p->workspace % 256 != 0 || p->workspace_bytes < plan.total))
    return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "attention to states needs a workspace of " + std::to_string(plan.total) + " bytes aligned to 256");
  SeqTable seqs = {};
  seqs.lengths = p->lengths;
  seqs.rows = p->rows;
  seqs.n = p->requests;
  seqs.Tq = p->requests * p->seq_tokens;
  seqs.per_seq = p->seq_tokens;
  seqs.length = p->cache_len;
  seqs.pitch = plan.pitch;
  seqs.pool = states ? p->cache_rows : 0;
  seqs.len64 = p->lengths_int64 != 0;
  seqs.row64 = p->rows_int64 != 0;
  const int group = p->num_q_heads / p->num_kv_heads;
  hipError_t e;
  if (plan.tiles) {
    if ((int64_t)plan.cap * p->num_q_heads > kMaxGroups - kXcds * p->num_q_heads)
      return fail_with(MIMIR_ERR_UNSUPPORTED_SHAPE, "too many rows for one launch");
    CrossArgs a = {};
    a.q = (const bf16_t*)p->q; a.k = (const bf16_t*)p->keys; a.v = (const bf16_t*)p->values;
    a.o = (bf16_t*)p->out;
    a.q_st = p->q_stride_token; a.q_sh = p->q_stride_head;
    a.k_st = p->k_stride_token; a.k_sh = p->k_stride_head;
    a.v_st = p->v_stride_token; a.v_sh = p->v_stride_head;
    a.o_st = p->out_stride_token; a.o_sh = p->out_stride_head;
    a.Tq = seqs.Tq; a.Hq = p->num_q_heads; a.Hkv = p->num_kv_heads; a.group = group;
    a.plan_q = (const int4*)p->workspace;
    a.cap_q = plan.cap;
    a.scale = p->softmax_scale;
    a.scale_log2 = p->softmax_scale * kLog2e;
    CrossPrologue pro = {};
    pro.seqs = seqs;
    pro.plan_q = (int4*)p->workspace;
    pro.cap_q = plan.cap;
    pro.D = p->head_dim;
    e = launch_cross_prologue(pro, (hipStream_t)stream);
    if (e == hipSuccess) e = launch_cross_fwd(a, p->head_dim, (hipStream_t)stream);
  } else {
    StatesArgs a = {};
    a.q = (const bf16_t*)p->q; a.k = (const bf16_t*)p->keys; a.v = (const bf16_t*)p->values;
    a.o = (bf16_t*)p->out;
    a.seqs = seqs;
    a.q_st = p->q_stride_token; a.q_sh = p->q_stride_head;
    a.k_sb = p->k_stride_row; a.k_st = p->k_stride_token; a.k_sh = p->k_stride_head;
    a.v_sb = p->v_stride_row; a.v_st = p->v_stride_token; a.v_sh = p->v_stride_head;
    a.o_st = p->out_stride_token; a.o_sh = p->out_stride_head;
    a.Hkv = p->num_kv_heads; a.group = group; a.rows = plan.rows;
    a.shares = plan.shares;
    a.scale_log2 = p->softmax_scale * kLog2e;
    a.part_o = (float*)p->workspace;
    a.part_ml = (float*)((char*)p->workspace + plan.ml);
    a.where = (int4*)((char*)p->workspace + plan.where);
    const int64_t merge = ((int64_t)p->requests * p->num_kv_heads * plan.rows + 3) / 4, groups = (int64_t)plan.shares * p->num_kv_heads;
    if (merge > kMaxGroups || groups > kMaxGroups || plan.row_tiles > 65535) return fail_with(MIMIR_ERR_UNSUPPORTED_SHAPE, "too many rows for one launch");
    const dim3 grid((unsigned)groups, (unsigned)plan.row_tiles), threads(kShareWaves * 64);
    const hipStream_t s = (hipStream_t)stream;
    const bool two = plan.tile_rows == 64, wide = p->head_dim == 128;
    if (two && wide) hipLaunchKernelGGL((states_kernel<128, 2, false>), grid, threads, 0, s, a);
    else if (two) hipLaunchKernelGGL((states_kernel<64, 2, false>), grid, threads, 0, s, a);
    else if (wide && plan.once) hipLaunchKernelGGL((states_kernel<128, 1, true>), grid, threads, 0, s, a);
    else if (wide) hipLaunchKernelGGL((states_kernel<128, 1, false>), grid, threads, 0, s, a);
    else if (plan.once) hipLaunchKernelGGL((states_kernel<64, 1, true>), grid, threads, 0, s, a);
    else hipLaunchKernelGGL((states_kernel<64, 1, false>), grid, threads, 0, s, a);
    e = hipGetLastError();
    if (e == hipSuccess) {
      if (p->head_dim == 128) hipLaunchKernelGGL(states_merge_kernel<128>, dim3((unsigned)merge), dim3(256), 0, s, a, plan.tile_rows);
      else hipLaunchKernelGGL(states_merge_kernel<64>, dim3((unsigned)merge), dim3(256), 0, s, a, plan.tile_rows);
      e = hipGetLastError();
    }
  }
  return e == hipSuccess ? MIMIR_OK : fail_with(MIMIR_ERR_HIP, std::string("attention to states launch: ") + hipGetErrorString(e));
}
