// Attention over an 8-bit paged KV cache, bf16 queries, for gfx950 (MI355X).
//
//   decode (at most 32 query rows per kv head, e.g. S = 1):
//     paged_decode_*      appends the new tokens and attends, the workgroups equal shares of all
//                         pages of the call
//     paged_merge_*       adds the partial rows of the shares
//   otherwise:
//     paged_append_*      the new tokens into their pages (prefixlm_paged_append.hip)
//     paged_prefill_*     one workgroup per (batch row, kv head, 128 query rows, key split)
//     paged_merge_splits_* with several splits: adds their partial rows
//
// S^T = K Q^T and O^T += V^T P^T on the matrix cores with an online softmax in fp32: in bf16 (codes
// become bf16 times their page's scale in the conversion instruction, exactly), prefill's first
// product on the codes themselves.  P is rounded to bf16, as everywhere in this library: the one rounding
// between the codes and the output that is not fp32's (and, in prefill, of query elements below 2^-15 of the
// largest of 32 columns).  The sums of P are those of the unrounded ones.
#include <algorithm>
#include <cmath>

#include "prefixlm_paged.h"

namespace mimir {
int fail_with(int code, const std::string& msg);

namespace {

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * 64;
constexpr int kDecRows = 32;        // query rows of the decode kernel per kv head, at most
constexpr float kRefRange = 30.f;   // how far (log2) a tile's reference may lie below the row's maximum

__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// 8-bit operands, 32 columns a lane.  Of each row the first four registers of both lane halves stand under
// 2^(scale - 127) of the lower half's lane, the other four under the upper's.
__device__ __forceinline__ f32x16 mfma8(i32x8 a, i32x8 b, f32x16 c, int a_scale, int b_scale) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 0, 0, 0, a_scale, 0, b_scale);
}

// Four values as codes hi and lo of x = hi + lo * 2^-4, |x| < 2^8: hi's rest is at most 2^4, so lo reaches
// the scale's bottom sixteen times later than it would under hi's.
constexpr int kLoShift = 4;
__device__ __forceinline__ void halves8(float a, float b, float c, float d, int& hi, int& lo) {
  typedef short s16x2 __attribute__((ext_vector_type(2)));
  constexpr float kLoScale = 1.f / (1 << kLoShift);
  hi = encode4(a, b, c, d);
  const f32x2 ab = __builtin_amdgcn_cvt_pk_f32_fp8(hi, false), cd = __builtin_amdgcn_cvt_pk_f32_fp8(hi, true);
  s16x2 x = __builtin_nondeterministic_value(x);  // both halves are written below
  x = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(x, a - ab[0], b - ab[1], kLoScale, false);
  x = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(x, c - cd[0], d - cd[1], kLoScale, true);
  lo = __builtin_bit_cast(int, x);
}

// Combine x over the four 16-lane groups of a wave.
__device__ __forceinline__ float xor16_max(float x) {
  const int xi = __float_as_int(x);
  auto r = __builtin_amdgcn_permlane16_swap(xi, xi, false, false);
  const int a = r[0], b = r[1];
  return fmaxf(__int_as_float(a), __int_as_float(b));
}
__device__ __forceinline__ float xor16_sum(float x) {
  const int xi = __float_as_int(x);
  auto r = __builtin_amdgcn_permlane16_swap(xi, xi, false, false);
  const int a = r[0], b = r[1];
  return __int_as_float(a) + __int_as_float(b);
}

// The largest of the lanes' non-negative values, on every lane (DPP moves; six shuffles through LDS take
// six round trips).
__device__ __forceinline__ int wave_max(int x) {
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false));  // row_shr:1
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false));  // row_shr:2
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false));  // row_shr:4
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false));  // row_shr:8
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false));  // row_bcast:15 into rows 1 and 3
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false));  // row_bcast:31 into rows 2 and 3
  return __builtin_amdgcn_readlane(x, 63);
}

// Between LDS writes and reads of one wave's own: they complete in order, the compiler has to keep it.
__device__ __forceinline__ void wave_lds_fence() {
  __asm__ volatile("" ::: "memory");
  wait_lds();
  __asm__ volatile("" ::: "memory");
}

// ------------------------------------------------------------------ partial rows

// One output row from its n partial rows (maximum in the exp2 domain, sum, unnormalized O) at
// slot(c), c < n: sum_c O_c 2^(m_c - M) / sum_c l_c 2^(m_c - M).  One wave; D / 4 lanes a part row,
// four columns each, kChunk loads in flight.
template <int D, typename Slot>
__device__ __forceinline__ void merge_parts(const PagedArgs& a, int n, int lane, Slot&& slot, bf16_t* orow) {
  constexpr int kChunk = 8, kLanes = D / 4, kParts = 64 / kLanes;
  const int sub = lane / kLanes, col = lane % kLanes * 4;
  float M = -INFINITY, lsum = 0.f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int c0 = 0; c0 < n; c0 += 64) {
    const int in_chunk = min(n - c0, 64);
    const int64_t row = slot(min(c0 + lane, n - 1));
    f32x2 ml = *(const f32x2*)&a.part_ml[2 * row];
    if (lane >= in_chunk) ml = f32x2{-INFINITY, 0.f};
    float m = ml[0];
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
    const float m_new = fmaxf(M, m);
    const float alpha = M == -INFINITY ? 0.f : fast_exp2(M - m_new);
    // no allowed key in this part: its sum is 0 (or NaN, of scores that all were)
    const float w = ml[0] == -INFINITY ? ml[1] : fast_exp2(ml[0] - m_new);
    float l = ml[1] * w;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) l += __shfl_xor(l, off, 64);
    lsum = lsum * alpha + l;
    acc *= alpha;
    M = m_new;
    for (int i0 = 0; i0 < in_chunk; i0 += kChunk * kParts) {
      f32x4 v[kChunk];
#pragma unroll
      for (int i = 0; i < kChunk; ++i) {
        const int src = min(i0 + i * kParts + sub, in_chunk - 1);
        const int64_t at = __shfl(row, src, 64);
        v[i] = *(const f32x4*)&a.part_o[at * D + col];
      }
#pragma unroll
      for (int i = 0; i < kChunk; ++i) {
        const int src = i0 + i * kParts + sub;
        const float wi = __shfl(w, min(src, 63), 64);
        if (src < in_chunk && wi != 0.f) acc += v[i] * wi;
      }
    }
  }
#pragma unroll
  for (int off = kLanes; off < 64; off <<= 1)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] += __shfl_xor(acc[e], off, 64);
  const float inv = lsum != 0.f ? 1.f / lsum : 0.f;  // NaN sums stay NaN
  if (sub == 0) *(bf16x4*)&orow[col] = __builtin_convertvector(acc * inv, bf16x4);
}

// ------------------------------------------------------------------ decode
//
// Bound by the read of the pages (64 rows of 512 to 8000 keys, 16 / 4 heads of 128: 56 us for 299 MB, 5.3 TB/s;
// a large read reaches 6.0) and, for short rows, by a chain of round trips: arguments, lengths, page ids,
// pages (one row of 700 keys 9.9 us).  Each wave streams its own pages straight into registers
// (a page of one head is 16 loads of 16 bytes a lane at head_dim 128): the layouts make
// every load an operand, so there is no LDS round trip and no barrier in the loop.  With the
// matrix instruction's 16 x 16 x 32 form the 64 tokens of a page are dealt so that the
// scores a lane group g holds are tokens 16 g .. 16 g + 15, in order: exactly the tokens of
// the 16-byte load from a value column.  The next page's keys are requested once the scores
// are formed and its values once they are used, so about a page per wave is in flight.
//
// The pages of all batch rows form a line, in units of four (one per wave), dealt evenly to
// shares (one workgroup per share and kv head), so that rows of very different lengths
// keep all CUs busy to the end.  A pair (batch row, kv head) inside one share is
// finished there; the parts of the others are merged by a second kernel.  For batches of
// more than kLineRows rows each pair takes a workgroup.

constexpr int kUnit = kWaves;  // pages of a unit
__device__ __forceinline__ int units_of(int kv) { return (kv + kPage * kUnit - 1) / (kPage * kUnit); }

// The line as each wave sees it, 64 batch rows to a register, one per lane: neither LDS nor barriers,
// whose round trips stood before a wave's first page (one row of 700 keys: 5000 of 18000 cycles).
constexpr int kLineChunks = 4;
constexpr int kLineRows = 64 * kLineChunks;
struct Line {
  PagedRow at[kLineChunks];
  int incl[kLineChunks];  // units up to and with the lane's row
  int total;
  __device__ __forceinline__ Line(const PagedArgs& a, int lane) {
#pragma unroll
    for (int c = 0; c < kLineChunks; ++c) {
      at[c].row = -1, at[c].n = at[c].m = at[c].kv = 0;
      if (64 * c + lane < a.B) at[c] = PagedRow(a, 64 * c + lane);
    }
    total = 0;
#pragma unroll
    for (int c = 0; c < kLineChunks; ++c) {
      incl[c] = total;
      if (64 * c >= a.B) continue;  // uniform
      incl[c] += wave_inclusive_sum(units_of(at[c].kv));
      total = __builtin_amdgcn_readlane(incl[c], 63);
    }
  }
  // The batch row that unit u < total lies in.
  __device__ __forceinline__ int find(int u) const {
#pragma unroll
    for (int c = 0; c < kLineChunks; ++c) {
      const uint64_t past = __builtin_amdgcn_ballot_w64(incl[c] > u);
      if (past != 0) return 64 * c + __builtin_ctzll(past);
    }
    return 0;
  }
  // Of batch row b (uniform): its place, and the units up to and with it.
  __device__ __forceinline__ PagedRow row(int b, int& upto) const {
    PagedRow r;
#pragma unroll
    for (int c = 0; c < kLineChunks; ++c)
      if (c == b >> 6) {
        r.row = __builtin_amdgcn_readlane(at[c].row, b & 63);
        r.n = __builtin_amdgcn_readlane(at[c].n, b & 63);
        r.m = __builtin_amdgcn_readlane(at[c].m, b & 63);
        r.kv = __builtin_amdgcn_readlane(at[c].kv, b & 63);
        upto = __builtin_amdgcn_readlane(incl[c], b & 63);
      }
    return r;
  }
};

// q units to each share, one more to the first r.
struct Deal {
  int q, r;
  __device__ __forceinline__ Deal(int total, int shares) : q(total / shares), r(total - total / shares * shares) {}
  __device__ __forceinline__ int begin(int share) const { return share * q + min(share, r); }
  __device__ __forceinline__ int of(int u) const {  // the share of unit u
    const int longer = r * (q + 1);
    return u < longer ? u / (q + 1) : r + (u - longer) / q;
  }
};
// Part slot (of two per share) of a segment: the one the share begins with, or a later one.
__device__ __forceinline__ int part_slot(int share, bool first) { return 2 * share + !first; }

// Zeros for `heads` heads from h0 on of batch row b.
template <int D>
__device__ __forceinline__ void zero_out(const PagedArgs& a, int b, int h0, int heads) {
  for (int i = threadIdx.x; i < a.S * heads * (D / 8); i += blockDim.x) {
    const int c = i % (D / 8), row = i / (D / 8);
    *(bf16x8*)&a.out[(int64_t)b * a.o_sb + (int64_t)(row / heads) * a.o_st + (int64_t)(h0 + row % heads) * a.o_sh + c * 8] = bf16x8{};
  }
}

template <int D, int NR, bool kPairs>
__device__ __forceinline__ void paged_decode_body(const PagedArgs& a) {
  constexpr int KH = D / 64;   // 16-byte loads of a key row per lane
  constexpr int DT = D / 16;   // column tiles of the output
  constexpr int kRowsMax = 16 * NR;
  constexpr int kPitch = D + 4;
  // Two row tiles of head_dim 128 leave no registers for a page of keys and of values at once: the
  // values are requested when the keys are used, and the other way round.
  constexpr bool kTakeTurns = NR == 2 && D == 128;
  __shared__ __attribute__((aligned(16))) float area[kWaves][kRowsMax * kPitch];
  __shared__ f32x2 area_ml[kWaves][kRowsMax];
  __shared__ __attribute__((aligned(8))) unsigned short s_nan[kWaves][D * 4];  // NaN tokens of each column, by wave

  touch_args<sizeof(PagedArgs)>();
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m16 = lane & 15, g = lane >> 4;
  const int share = blockIdx.x / a.Hkv, hk = blockIdx.x - share * a.Hkv;  // share: the batch row, for pairs
  const int R = a.S * a.G;

  int b = share, u0 = 0, u_end = 1, upto = 0;
  PagedRow r;
  [[maybe_unused]] int incl[kLineChunks];  // of the line
  if constexpr (kPairs) {
    r = PagedRow(a, b);
    if (r.kv == 0) {
      zero_out<D>(a, b, hk * a.G, a.G);
      return;
    }
  } else {
    const Line line(a, lane);
    const Deal deal(line.total, a.shares);
    u0 = deal.begin(share);
    u_end = deal.begin(share + 1);
#pragma unroll
    for (int c = 0; c < kLineChunks; ++c) incl[c] = line.incl[c];
    if (u0 >= u_end) return;
    b = line.find(u0);
    r = line.row(b, upto);
  }

  // offsets of a lane in a page: key rows 16 (m16 / 4) + m16 % 4 (+ 4 per tile), value columns m16 (+ 16)
  const int k_off = (16 * (m16 >> 2) + (m16 & 3)) * D + 16 * g;
  const int v_off = m16 * kPage + 16 * g;
  const float c2 = a.scale_log2;
  const float ref_range = fminf(kRefRange / c2, 3e38f);
  const int u_first = u0;

  for (;;) {
    // The segment: pages [t0, t1) of batch row b.
    int t0 = 0, t1 = (r.kv + kPage - 1) / kPage;
    bool whole = true;
    int u_next = u_end;
    if constexpr (!kPairs) {
      const int units = (t1 + kUnit - 1) / kUnit;
      const int unit0 = u0 - (upto - units), unit1 = min(units, unit0 + u_end - u0);
      whole = unit0 == 0 && unit1 == units;
      u_next = u0 + unit1 - unit0;
      t0 = unit0 * kUnit;
      t1 = min(t1, unit1 * kUnit);
    }
    const int n_my = t0 + wave < t1 ? (t1 - t0 - wave + kUnit - 1) / kUnit : 0;  // this wave's pages

    // Each row's key limit; 0 for queries i >= m.
    int limit[NR];
#pragma unroll
    for (int nr = 0; nr < NR; ++nr) {
      const int i = a.S == 1 ? 0 : (16 * nr + m16) / a.G;
      limit[nr] = 16 * nr + m16 < R && i < r.m ? (a.causal ? min(r.n + i + 1, r.kv) : r.kv) : 0;
    }
    const int limit_min = a.causal ? min(r.n + 1, r.kv) : r.kv;

    // The wave's pages, 64 at a time on its lanes: page id (-1: none) and exponents.
    int ids = -1, ek = 0, ev = 0;
    auto load_ids = [&](int i0) __attribute__((always_inline)) {
      const int t = t0 + wave + kUnit * (i0 + lane);
      ids = t < t1 ? page_id(a, r.row, t) : -1;
      ek = ids >= 0 ? a.ke[ids * a.ke_sp + hk] : 0;
      ev = ids >= 0 ? a.ve[ids * a.ve_sp + hk] : 0;
    };
    i32x4 kreg[4][KH], vreg[DT];
    auto load_keys = [&](int i) __attribute__((always_inline)) {
      const int id = max(__builtin_amdgcn_readlane(ids, i & 63), 0);  // none: page 0, masked
      const uint8_t* p = a.ck + id * a.k_sp + (int64_t)hk * kPage * D;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int h = 0; h < KH; ++h) kreg[t][h] = __builtin_nontemporal_load((const i32x4*)&p[k_off + 4 * t * D + 64 * h]);
    };
    auto load_values = [&](int i) __attribute__((always_inline)) {
      const int id = max(__builtin_amdgcn_readlane(ids, i & 63), 0);
      const uint8_t* p = a.cv + id * a.v_sp + (int64_t)hk * kPage * D;
#pragma unroll
      for (int d = 0; d < DT; ++d) vreg[d] = __builtin_nontemporal_load((const i32x4*)&p[v_off + 16 * kPage * d]);
    };

    // The wave's page with new tokens, if any, is its last (they lie in two pages at most): tokens
    // s0 .. s0 + cnt - 1 of it.  This wave alone reads and writes that page and head in the call, so the
    // codes go to memory and, beside it, straight into the operands.
    constexpr int kUnits = D / 8, kNewRows = 64 / kUnits;  // lanes of a new row, rows at a time
    const int last = t0 + wave + kUnit * (n_my - 1);
    const int new0 = max(r.n, last * kPage), s0 = new0 - last * kPage;
    const int cnt = n_my > 0 ? max(min(r.n + r.m, min(last + 1, a.width) * kPage) - new0, 0) : 0;
    const bf16_t* const x_k = a.kn + (int64_t)b * a.kn_sb + (int64_t)hk * a.kn_sh + (int64_t)(new0 - r.n) * a.kn_st;
    const bf16_t* const x_v = a.vn + (int64_t)b * a.vn_sb + (int64_t)hk * a.vn_sh + (int64_t)(new0 - r.n) * a.vn_st;
    i32x4 k_first = {0, 0, 0, 0}, v_first = {0, 0, 0, 0};  // the lane's first new row, requested with the queries
    constexpr int kQueryBytes = NR * 2 * KH * 64 * 16;
    static_assert(kQueryBytes + 2 * kRowsMax * D <= kRowsMax * kPitch * 4, "the queries and the new codes fit the wave's area");
    uint8_t* const codes = (uint8_t*)area[wave] + kQueryBytes;  // [2][cnt][D]
    auto append = [&](int i, int& e_k, int& e_v) __attribute__((always_inline)) {
      // lane numbers that the compiler cannot see through: what is formed from them here would otherwise be
      // held in registers through the loop over the pages (150 instead of 194 at head_dim 64)
      const int lane = opaque_lane_id(), m16 = lane & 15, g = lane >> 4, x_row = lane / kUnits, x_col = lane % kUnits * 8;
      const bf16_t* const xk = x_k + x_col;
      const bf16_t* const xv = x_v + x_col;
      const int page = __builtin_amdgcn_readlane(ids, i), had_k = e_k, had_v = e_v;
      int most_k = largest_bits(k_first), most_v = largest_bits(v_first);
      for (int t = x_row + kNewRows; t < cnt; t += kNewRows) {
        most_k = max(most_k, largest_bits(*(const i32x4*)&xk[(int64_t)t * a.kn_st]));
        most_v = max(most_v, largest_bits(*(const i32x4*)&xv[(int64_t)t * a.vn_st]));
      }
      e_k = exponent_for(wave_max(most_k));
      e_v = exponent_for(wave_max(most_v));
      if (s0 > 0) {
        e_k = max(e_k, had_k);
        e_v = max(e_v, had_v);
      }
      if (lane == 0) {
        a.ke[page * a.ke_sp + hk] = (int8_t)e_k;
        a.ve[page * a.ve_sp + hk] = (int8_t)e_v;
      }
      uint8_t* const yk = a.ck + page * a.k_sp + (int64_t)hk * kPage * D;
      uint8_t* const yv = a.cv + page * a.v_sp + (int64_t)hk * kPage * D;
      if (__builtin_expect(s0 > 0 && (e_k > had_k || e_v > had_v), 0)) {
        // Now and then (a larger magnitude than the page has seen): the older codes rounded again in memory,
        // and the page read again.
        for (int w = lane; w < s0 * D / 4; w += 64) ((int*)yk)[w] = recode4(((int*)yk)[w], had_k - e_k);
        for (int w = lane; w < 16 * D; w += 64) {
          const int old = ((int*)yv)[w], end = s0 - w % 16 * 4;  // older tokens of the word
          const unsigned keep = end >= 4 ? 0u : (end <= 0 ? ~0u : ~0u << (8 * end));
          ((int*)yv)[w] = (int)(((unsigned)recode4(old, had_v - e_v) & ~keep) | ((unsigned)old & keep));
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
        load_keys(i);
        load_values(i);
      }
      for (int t = x_row; t < cnt; t += kNewRows) {
        const i32x4 xs[2] = {t == x_row ? k_first : *(const i32x4*)&xk[(int64_t)t * a.kn_st],
                             t == x_row ? v_first : *(const i32x4*)&xv[(int64_t)t * a.vn_st]};
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const bf16x8 v = __builtin_bit_cast(bf16x8, xs[w]);
          const int e = w ? e_v : e_k;
          float f[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) f[k] = coded_value((float)v[k], e);
          const i32x2 c = {encode4(f[0], f[1], f[2], f[3]), encode4(f[4], f[5], f[6], f[7])};
          *(i32x2*)&codes[(w * cnt + t) * D + x_col] = c;
          if (w == 0) *(i32x2*)&yk[(s0 + t) * D + x_col] = c;
        }
      }
      wave_lds_fence();
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int j = 16 * (m16 >> 2) + 4 * t + (m16 & 3) - s0;
        if (j >= 0 && j < cnt) {
#pragma unroll
          for (int h = 0; h < KH; ++h) kreg[t][h] = *(const i32x4*)&codes[j * D + 64 * h + 16 * g];
        }
      }
      for (int j = 0; j < cnt; ++j) {
        const int slot = s0 + j, sh = 8 * (slot & 3);
        if (g == slot >> 4) {
          const uint8_t* const x = &codes[(cnt + j) * D + m16];
          unsigned c[DT];
#pragma unroll
          for (int d = 0; d < DT; ++d) c[d] = x[16 * d];
#pragma unroll
          for (int d = 0; d < DT; ++d) yv[(16 * d + m16) * kPage + slot] = (uint8_t)c[d];
#pragma unroll
          for (int w = 0; w < 4; ++w)
            if (w == (slot & 15) >> 2) {  // uniform
#pragma unroll
              for (int d = 0; d < DT; ++d) vreg[d][w] = (int)(((unsigned)vreg[d][w] & ~(0xffu << sh)) | c[d] << sh);
            }
        }
      }
    };

    // Q^T operands: lane holds query row m16 (+ 16), columns 64 h + 16 g + 8 s ..+7; rows past the last
    // take the first (never read).  They wait in LDS, a copy for each wave in its part of the merge's area:
    // registers for them would spill with two row tiles.
    i32x4* const q_lds = (i32x4*)area[wave] + lane;
    i32x4 q_in[NR][2 * KH];
#pragma unroll
    for (int nr = 0; nr < NR; ++nr) {
      const int row = 16 * nr + m16 < R ? 16 * nr + m16 : 0, i = a.S == 1 ? 0 : row / a.G;
      const bf16_t* q = a.q + (int64_t)b * a.q_sb + (int64_t)i * a.q_st + (int64_t)(hk * a.G + row - i * a.G) * a.q_sh + 16 * g;
#pragma unroll
      for (int x = 0; x < 2 * KH; ++x) q_in[nr][x] = *(const i32x4*)&q[64 * (x >> 1) + 8 * (x & 1)];
    }
    if (n_my > 0) {
      load_ids(0);
      const int x_row = lane / kUnits, x_col = lane % kUnits * 8;
      if (x_row < cnt) {
        k_first = *(const i32x4*)&x_k[(int64_t)x_row * a.kn_st + x_col];
        v_first = *(const i32x4*)&x_v[(int64_t)x_row * a.vn_st + x_col];
      }
      load_keys(0);
      if (!kTakeTurns) load_values(0);
    }
#pragma unroll
    for (int nr = 0; nr < NR; ++nr)
#pragma unroll
      for (int x = 0; x < 2 * KH; ++x) q_lds[(nr * 2 * KH + x) * 64] = q_in[nr][x];
    wave_lds_fence();

    f32x4 oacc[NR][DT];
    float m_run[NR], m_top[NR], l_run[NR];  // the sums' reference and the row's maximum so far (scores), the sum
#pragma unroll
    for (int nr = 0; nr < NR; ++nr) {
#pragma unroll
      for (int d = 0; d < DT; ++d) oacc[nr][d] = f32x4{0.f, 0.f, 0.f, 0.f};
      m_run[nr] = m_top[nr] = -INFINITY;
      l_run[nr] = 0.f;
    }
    for (int i = 0; i < n_my; ++i) {
      const int base = (t0 + wave + kUnit * i) * kPage;
      const bool some = __builtin_amdgcn_readlane(ids, i & 63) >= 0;
      int e_k = __builtin_amdgcn_readlane(ek, i & 63), e_v = __builtin_amdgcn_readlane(ev, i & 63);
      const bool appends = cnt > 0 && i + 1 == n_my && some;
      if (appends) {
        if (kTakeTurns) load_values(i);
        append(i & 63, e_k, e_v);
      }
      const float ks = pow2(e_k), vs = pow2(e_v);
      f32x4 st[NR][4];
#pragma unroll
      for (int nr = 0; nr < NR; ++nr)
#pragma unroll
        for (int t = 0; t < 4; ++t) st[nr][t] = f32x4{0.f, 0.f, 0.f, 0.f};
      __asm__ volatile("" ::: "memory");  // read again for every page
#pragma unroll
      for (int h = 0; h < KH; ++h)
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          bf16x8 qf[NR];
#pragma unroll
          for (int nr = 0; nr < NR; ++nr) qf[nr] = __builtin_bit_cast(bf16x8, q_lds[(nr * 2 * KH + 2 * h + s) * 64]);
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const bf16x8 kf = decode8(kreg[t][h][2 * s], kreg[t][h][2 * s + 1], ks);
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) st[nr][t] = mfma16(kf, qf[nr], st[nr][t]);
          }
        }
      if (kTakeTurns) {
        if (!appends) load_values(i);
      } else if (i + 1 < n_my) {
        if (__builtin_expect((i & 63) == 63, 0)) load_ids(i + 1);
        load_keys(i + 1);
      }
      // tokens 16 g + 4 t + e of the page
      const bool edge = !some || base + kPage > limit_min;
      bf16x8 pf[NR][2];
#pragma unroll
      for (int nr = 0; nr < NR; ++nr) {
        if (edge) {
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (!some || base + 16 * g + 4 * t + e >= limit[nr]) st[nr][t][e] = -INFINITY;
        }
        float mx = -INFINITY;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) mx = fmaxf(mx, st[nr][t][e]);
        // Every page's probabilities under its own maximum (but not more than 2^30 below the row's so
        // far, which bounds the sums): its largest is 1, exact in bf16.  (P as the sum of two bf16 numbers, which would
        // leave the output's own rounding alone: 1 to 4% slower with one row tile, up to 8% with two.)
        mx = xor32_max(xor16_max(mx));
        m_top[nr] = fmaxf(m_top[nr], mx);
        const float m_new = fmaxf(mx, m_top[nr] - ref_range);
        const float alpha = m_run[nr] == -INFINITY ? 1.f : fast_exp2((m_run[nr] - m_new) * c2);
        m_run[nr] = m_new;
        const float mb = m_new == -INFINITY ? 0.f : m_new;
        float lsum = 0.f;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            // the difference first: a scaled score of 2^30 is known to 2^6, and rounding it apart from the
            // maximum would give probabilities up to 2^64
            const float p = fast_exp2((st[nr][t][e] - mb) * c2);
            st[nr][t][e] = p;
            lsum += p;
          }
        l_run[nr] = l_run[nr] * alpha + lsum;
#pragma unroll
        for (int d = 0; d < DT; ++d) oacc[nr][d] *= alpha;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          f32x8 x;
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = st[nr][2 * c + (e >> 2)][e & 3];
          pf[nr][c] = to_bf16x8(x);
        }
      }
      bool any_nan = false;
      if (edge) {
        // What lies behind the last token is unwritten; a NaN among the values of tokens that only
        // some of the rows see must not reach the others: it is taken out of the product
        // and put into the rows that see it.
        const int end = (some ? min(r.kv - base, kPage) : 0) - 16 * g;
        unsigned nan = 0;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            vreg[d][w] = codes_before(vreg[d][w], 4 * w, end);
            nan |= nan_codes(vreg[d][w]);
          }
        any_nan = __builtin_amdgcn_ballot_w64(nan != 0) != 0;
        if (__builtin_expect(any_nan, 0)) {
          const int lane = opaque_lane_id(), m16 = lane & 15, g = lane >> 4;
#pragma unroll
          for (int d = 0; d < DT; ++d) {
            unsigned at = 0;  // tokens 16 g + e whose code is NaN
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (((unsigned)vreg[d][e >> 2] >> 8 * (e & 3) & 0x7f) == 0x7f) {
                at |= 1u << e;
                vreg[d][e >> 2] &= (int)~(0xffu << 8 * (e & 3));
              }
            s_nan[wave][(16 * d + m16) * 4 + g] = (unsigned short)at;
          }
          wave_lds_fence();
        }
      }
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const bf16x8 vf = decode8(vreg[d][2 * c], vreg[d][2 * c + 1], vs);
#pragma unroll
          for (int nr = 0; nr < NR; ++nr) oacc[nr][d] = mfma16(vf, pf[nr][c], oacc[nr][d]);
        }
      if (__builtin_expect(any_nan, 0)) {
        const int g = opaque_lane_id() >> 4;
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
          const int n = limit[nr] - base;
          const uint64_t seen = n >= 64 ? ~0ull : (n <= 0 ? 0ull : (1ull << n) - 1);
#pragma unroll
          for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (*(const uint64_t*)&s_nan[wave][(16 * d + 4 * g + e) * 4] & seen) oacc[nr][d][e] = __builtin_nanf("");
        }
        wave_lds_fence();
      }
      if (i + 1 < n_my) {
        if (kTakeTurns) {
          if (__builtin_expect((i & 63) == 63, 0)) load_ids(i + 1);
          load_keys(i + 1);
        } else {
          load_values(i + 1);
        }
      }
    }

    // Merge the waves' rows through LDS.
    const int lane_after = opaque_lane_id(), m16 = lane_after & 15, g = lane_after >> 4, tid = wave * 64 + lane_after;
#pragma unroll
    for (int nr = 0; nr < NR; ++nr) {
      const int row = 16 * nr + m16;
      const float l = xor32_sum(xor16_sum(l_run[nr]));
      if (row < R) {
        if (g == 0) area_ml[wave][row] = f32x2{m_run[nr] == -INFINITY ? -INFINITY : m_run[nr] * c2, l};
#pragma unroll
        for (int d = 0; d < DT; ++d) *(f32x4*)&area[wave][row * kPitch + 16 * d + 4 * g] = oacc[nr][d];
      }
    }
    __syncthreads();
    constexpr int kLanes = D / 4, kRowsAt = kThreads / kLanes;
    const int col = tid % kLanes * 4;
    for (int row = tid / kLanes; row < R; row += kRowsAt) {
      float M = -INFINITY, lsum = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) M = fmaxf(M, area_ml[w][row][0]);
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const f32x2 ml = area_ml[w][row];
        const float wt = ml[0] == -INFINITY ? ml[1] : fast_exp2(ml[0] - M);  // no key: a sum of 0 (or NaN)
        lsum += ml[1] * wt;
        if (wt != 0.f) acc += *(const f32x4*)&area[w][row * kPitch + col] * wt;
      }
      if (whole) {
        const float inv = lsum != 0.f ? 1.f / lsum : 0.f;
        const int i = a.S == 1 ? 0 : row / a.G;
        *(bf16x4*)&a.out[(int64_t)b * a.o_sb + (int64_t)i * a.o_st + (int64_t)(hk * a.G + row - i * a.G) * a.o_sh + col] =
            i < r.m ? __builtin_convertvector(acc * inv, bf16x4) : bf16x4{};
      } else {
        const int64_t slot = ((int64_t)part_slot(share, u0 == u_first) * a.Hkv + hk) * R + row;
        *(f32x4*)&a.part_o[slot * D + col] = acc;
        if (col == 0) *(f32x2*)&a.part_ml[slot * 2] = f32x2{M, lsum};
      }
    }
    if (u_next >= u_end) return;
    u0 = u_next;
    if constexpr (!kPairs) {
      // the next batch row with keys; its place is looked up again rather than held
#pragma unroll
      for (int c = kLineChunks - 1; c >= 0; --c) {
        const uint64_t past = __builtin_amdgcn_ballot_w64(incl[c] > u0);
        if (past != 0) {
          b = 64 * c + __builtin_ctzll(past);
          upto = __builtin_amdgcn_readlane(incl[c], b & 63);
        }
      }
      r = PagedRow(a, b);
    }
    __syncthreads();  // the merge's area is free again
  }
}

#define DECODE(D, NR)                                                                                        \
  __global__ __launch_bounds__(kThreads, 2) void paged_decode_d##D##_r##NR##_kernel(const PagedArgs a) {       \
    paged_decode_body<D, NR, false>(a);                                                                      \
  }                                                                                                          \
  __global__ __launch_bounds__(kThreads, 2) void paged_decode_pairs_d##D##_r##NR##_kernel(const PagedArgs a) { \
    paged_decode_body<D, NR, true>(a);                                                                       \
  }
DECODE(128, 1)
DECODE(128, 2)
DECODE(64, 1)
DECODE(64, 2)
#undef DECODE

// Output rows of the pairs whose pages lie in several shares, one wave per row.
template <int D>
__device__ __forceinline__ void paged_merge_body(const PagedArgs& a) {
  touch_args<sizeof(PagedArgs)>();
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int R = a.S * a.G, groups = (R + kWaves - 1) / kWaves;
  const int row = blockIdx.x % groups * kWaves + wave, pair = blockIdx.x / groups;
  const int b = pair / a.Hkv, hk = pair - b * a.Hkv;
  if (row >= R) return;
  const Line line(a, lane);
  int upto = 0;
  const PagedRow r = line.row(b, upto);
  const int units = units_of(r.kv), before = upto - units;
  const int i = a.S == 1 ? 0 : row / a.G;
  bf16_t* const o = a.out + (int64_t)b * a.o_sb + (int64_t)i * a.o_st + (int64_t)(hk * a.G + row - i * a.G) * a.o_sh;
  if (units == 0 || i >= r.m) {  // a batch row without keys, or a padding query
    if (lane < D / 8) *(bf16x8*)&o[lane * 8] = bf16x8{};
    return;
  }
  const Deal deal(line.total, a.shares);
  const int w0 = deal.of(before), n = deal.of(before + units - 1) - w0 + 1;
  if (n == 1) return;  // written by its share
  const int slot0 = part_slot(w0, before == deal.begin(w0));
  merge_parts<D>(a, n, lane, [&](int c) { return ((int64_t)(c == 0 ? slot0 : part_slot(w0 + c, true)) * a.Hkv + hk) * R + row; }, o);
}
__global__ __launch_bounds__(kThreads) void paged_merge_d128_kernel(const PagedArgs a) { paged_merge_body<128>(a); }
__global__ __launch_bounds__(kThreads) void paged_merge_d64_kernel(const PagedArgs a) { paged_merge_body<64>(a); }

// ------------------------------------------------------------------ prefill
//
// Rows are (token, head) pairs, token-major, 128 to a workgroup, so the G query heads of a
// kv head share its pages, which are copied to LDS as they are while the page before is computed.
//
// The scores run on the 8-bit matrix instruction (32 x 32 x 64, twice the bf16 rate) with the keys' codes as one
// operand, their page's scale going into the instruction, and the queries in two 8-bit halves as the other: hi the
// nearest code, lo that of the rest (halves8), under a power of two of each row and 32 columns.  A code holds four
// significant bits, so the two hold the eight of bf16 in as much matrix time, exactly down to 2^-15 of the largest of
// the 32, the smaller ones to 2^-22 of it: two fp32 half steps of the largest term.  (A third code for what they
// leave, multiplied where a wave's queries leave anything: 8 to 12% slower.)  Against keys converted to bf16: half the
// LDS reads, no conversions, and the queries are split once.
// The output takes P in bf16 and the values' codes converted on their way into the operands, once for each wave.
// P in two halves under its page's maximum, on the codes, lost small probabilities below 2^-21 of the page's
// largest and was slower: it takes ten vector instructions for four, where a conversion of two takes one.  Halves /
// bf16: 8 x 512 tokens on 1024 keys, 16 / 4 heads of 128, 66.6 / 66.4 us, 8 x up to 512 on up to 3000 85.2 / 81.8;
// 8 / 8 heads of 64, 8 x 512 on 1024, 44.5 / 42.0, 4096 on 8192, 8 / 2, 167.7 / 144.9.
// 8 x 512 tokens on 1536 keys, 16 / 4 heads of 128: 68 to 79 us (warm and cool clocks; 77.1 under the counters) for 60
// GFLOP; the vector units are busy 56% and the matrix units 41% of the time, which two waves a SIMD overlap little.
//
// The scores' rows are tokens 32 (m / 4 % 2) + 16 t + 4 (m / 8) + m % 4 for row m of tile t, so that the 32 a
// lane holds are 32 hi .., in order: the 32 bytes of a value column that its half of the lanes reads, eight of them
// for each step of the second product.

constexpr int kRows = kWaves * 32;
constexpr int kTogether = 2;  // pages between two barriers
constexpr int kMaxSplits = 64;

// Whether the batch rows hold about as many cached keys: none differs from the first by more
// than an eighth of the chunk.
__device__ __forceinline__ bool even_lengths(const PagedArgs& a) {
  if (a.B > 64) return false;
  const int n = PagedRow(a, min((int)threadIdx.x & 63, a.B - 1)).n;
  const int64_t off = n - __builtin_amdgcn_readfirstlane(n);
  return __builtin_amdgcn_ballot_w64(8 * (off < 0 ? -off : off) > a.S) == 0;
}

// A padded batch (new_lengths), whose row tiles with queries only the device knows: those alone are cut, each
// into n runs of about as many pages, so that the runs of all are a.slots and one more for each row tile at
// most.  Runs first, then the row tiles without queries.  64 batch rows, one per lane.  Against splits of the
// full batch's tiles, on 1 to so many keys: 8 x up to 512 on 3000 keys, 16 / 4 heads of 128, 97 -> 80.5 us; 3 x up to 200
// on 3000, 32 / 8, 54.6 -> 51.0; 8 x up to 700 on 2000, 8 / 8 heads of 64, 48.7 -> 43.5; 5 x up to 1339 on 1000 58.4 -> 47.0.
constexpr int kDealtRows = 64;
struct Runs {
  PagedRow at;      // of the lane's batch row
  int act, n;       // its row tiles with queries, the runs of each
  int incl, idle;   // up to and with it: runs of all kv heads, and row tiles without queries
  __device__ __forceinline__ Runs(const PagedArgs& a, int lane) {
    at.row = -1, at.n = at.m = at.kv = 0;
    if (lane < a.B) at = PagedRow(a, lane);
    const int tiles = (at.kv + kPage - 1) / kPage;
    act = at.kv > 0 ? (int)((unsigned)(at.m * a.G + kRows - 1) / kRows) : 0;
    const int pages = __builtin_amdgcn_readlane(wave_inclusive_sum(act * a.Hkv * tiles), 63);
    // At head_dim 64 all runs are to be on the chip at once, three per CU: a few more would be a second round (8 x up to
    // 700 tokens on up to 2000 keys 48.6 -> 43.5 us, 5 x up to 1339 on 1000 50.1 -> 47.0, where two per CU take 43.4 and
    // 49.9).  At 128 one per CU and the remainders (two per CU: 8 x up to 512 on up to 3000 80.5 -> 85.6, 4 x up to 100 on
    // up to 3000 29.2 -> 31.0).
    const int all = __builtin_amdgcn_readlane(wave_inclusive_sum(act * a.Hkv), 63);
    int most = max(kTogether, (int)((unsigned)(pages + a.slots - 1) / (unsigned)a.slots));
    for (int tries = a.D == 64 && all <= a.slots ? 12 : 0;; --tries) {
      n = max(1, (int)((unsigned)(tiles + most - 1) / (unsigned)most));
      if (tries == 0 || __builtin_amdgcn_readlane(wave_inclusive_sum(act * a.Hkv * n), 63) <= a.slots) break;
      most += max(1, most / 16);
    }
    const int runs = per(tiles, n);
    n = max(1, (int)((unsigned)(tiles + runs - 1) / (unsigned)runs));
    incl = wave_inclusive_sum(act * a.Hkv * n);
    idle = wave_inclusive_sum(lane < a.B ? (a.n_rt - act) * a.Hkv : 0);
  }
  static __device__ __forceinline__ int per(int tiles, int n) { return max(1, (int)((unsigned)(tiles + n - 1) / (unsigned)n)); }
  __device__ __forceinline__ PagedRow row(int b) const {
    PagedRow r;
    r.row = __builtin_amdgcn_readlane(at.row, b);
    r.n = __builtin_amdgcn_readlane(at.n, b);
    r.m = __builtin_amdgcn_readlane(at.m, b);
    r.kv = __builtin_amdgcn_readlane(at.kv, b);
    return r;
  }
  // The first run of row tile rt < act of (b, hk): the latest row tiles first, they see most.
  __device__ __forceinline__ int first(const PagedArgs& a, int b, int hk, int rt) const {
    const int tiles = __builtin_amdgcn_readlane(act, b), runs = __builtin_amdgcn_readlane(n, b);
    return __builtin_amdgcn_readlane(incl, b) + ((hk - a.Hkv) * tiles + tiles - 1 - rt) * runs;
  }
};

template <int D, bool kRuns>
__device__ __forceinline__ void paged_prefill_body(const PagedArgs& a) {
  constexpr int DT = D / 32, KS = D / 64;
  constexpr int kCopies = D / 64;  // 1 KiB copies of a page's keys, and of its values, per wave
  __shared__ __attribute__((aligned(16))) uint8_t sK[2 * kTogether][kPage * D];
  __shared__ __attribute__((aligned(16))) uint8_t sV[2 * kTogether][kPage * D];
  // of a page that some rows see only part of: which tokens' values are NaN, for each column (64 bits),
  // and whether any are, by wave
  __shared__ __attribute__((aligned(8))) unsigned short s_nan[kTogether][D * 4];
  __shared__ int s_any[kTogether][kWaves];

  touch_args<sizeof(PagedArgs)>();
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, hi = lane >> 5;
  // Later row tiles of a causal chunk see more keys, and workgroups u and u + (CUs) share a CU.  On
  // rows of about the same length they go by rank, the latest first over all pairs, and every
  // other CU-sized run backwards, so that a CU's two are a long and a short one.
  int u = blockIdx.x, split = 0, rt, hk, b, n_valid, per;
  int64_t unit;  // of partial rows
  PagedRow r;
  if constexpr (kRuns) {
    const Runs runs(a, lane);
    const uint64_t past = __builtin_amdgcn_ballot_w64(runs.incl > u);
    unit = u;
    n_valid = 1;
    if (past != 0) {
      b = __builtin_ctzll(past);
      n_valid = __builtin_amdgcn_readlane(runs.n, b);
      const int act = __builtin_amdgcn_readlane(runs.act, b);
      u -= __builtin_amdgcn_readlane(runs.incl, b) - act * a.Hkv * n_valid;
      split = u % n_valid;
      u /= n_valid;
      rt = act - 1 - u % act;
      hk = u / act;
    } else {
      u -= __builtin_amdgcn_readlane(runs.incl, 63);
      const uint64_t rest = __builtin_amdgcn_ballot_w64(runs.idle > u);
      if (rest == 0) return;
      b = __builtin_ctzll(rest);
      const int act = __builtin_amdgcn_readlane(runs.act, b), idle = a.n_rt - act;
      u -= __builtin_amdgcn_readlane(runs.idle, b) - idle * a.Hkv;
      rt = act + u % idle;
      hk = u / idle;
    }
    r = runs.row(b);
    per = Runs::per((r.kv + kPage - 1) / kPage, n_valid);
  } else {
    if (a.splits == 1 && a.causal && even_lengths(a)) {
      const int run = u / a.cus, pairs = gridDim.x / a.n_rt;
      if (run % 2 == 1 && (run + 1) * a.cus <= (int)gridDim.x) u = (2 * run + 1) * a.cus - 1 - u;
      rt = a.n_rt - 1 - u / pairs;
      u %= pairs;
    } else {
      split = u % a.splits;
      u /= a.splits;
      rt = a.n_rt - 1 - u % a.n_rt;
      u /= a.n_rt;
    }
    hk = u % a.Hkv, b = u / a.Hkv;
    r = PagedRow(a, b);
    const int tiles = (r.kv + kPage - 1) / kPage;
    per = max(1, (tiles + a.splits - 1) / a.splits);
    n_valid = (tiles + per - 1) / per;  // splits that hold keys
    if (split > 0 && split >= n_valid) return;
    unit = (((int64_t)b * a.Hkv + hk) * a.n_rt + rt) * a.splits + split;
  }
  const int R = a.S * a.G, Rm = r.kv > 0 ? r.m * a.G : 0;  // rows, and those that attend

  const int row = rt * kRows + wave * 32 + l32;
  const bool row_ok = row < R;
  const int ti = row_ok ? row / a.G : 0;
  const int h = hk * a.G + (row_ok ? row - ti * a.G : 0);
  auto limit_of = [&](int x) { return a.causal ? min(r.n + x / a.G + 1, r.kv) : r.kv; };
  const int limit = row < Rm ? limit_of(row) : 0;
  const int r0 = rt * kRows + wave * 32;
  const bool active = r0 < Rm;
  const int w_max = active ? limit_of(min(r0 + 31, Rm - 1)) : 0, w_min = active ? limit_of(r0) : 0;
  const int wg0 = rt * kRows;
  const int wg_max = wg0 < Rm ? limit_of(min(wg0 + kRows - 1, Rm - 1)) : 0, wg_min = wg0 < Rm ? limit_of(wg0) : 0;
  const int kt0 = split * per;
  const int kt1 = min((wg_max + kPage - 1) / kPage, kt0 + per);

  // 16-byte unit u of token t's key lies at place u ^ k_place(t), of value column d at u ^ v_place(d): the
  // sixteen rows of an operand read then fall on sixteen different places of the banks.
  auto k_place = [](int t) { return D == 128 ? (t >> 1 & 3) | (t >> 3 & 4) : (t >> 2 & 1) | (t >> 4 & 2); };
  auto v_place = [](int d) { return d >> 2 & 3; };
  int id_next[kTogether], ek[kTogether], ev[kTogether];
  bool some[kTogether];
  auto next_id = [&](int kt, int j) { id_next[j] = kt < kt1 ? load_const(a.table, (int64_t)r.row * a.t_st + kt) : -1; };
  auto load_page = [&](int kt, int j, int buf) __attribute__((always_inline)) {
    const int id = id_next[j];
    next_id(kt + kTogether, j);  // ahead: the copies wait for no look at the table
    some[j] = id >= 0 && id < a.num_pages;
    if (kt >= kt1) return;
    const int64_t p = some[j] ? id : 0;  // none: page 0, not attended
    const uint8_t* kp = a.ck + p * a.k_sp + (int64_t)hk * kPage * D;
    const uint8_t* vp = a.cv + p * a.v_sp + (int64_t)hk * kPage * D;
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      const int at = wave * kCopies + i, place = at * 64 + lane;
      const int t = place / (D / 16), d = place / 4;
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(kp + t * D + ((place % (D / 16)) ^ k_place(t)) * 16),
                                       (__attribute__((address_space(3))) void*)(sK[buf] + at * 1024), 16, 0, 0);
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(vp + d * kPage + ((place & 3) ^ v_place(d)) * 16),
                                       (__attribute__((address_space(3))) void*)(sV[buf] + at * 1024), 16, 0, 0);
    }
    ek[j] = a.ke[p * a.ke_sp + hk];
    ev[j] = a.ve[p * a.ve_sp + hk];
  };
  // A page with tokens that some rows of the workgroup do not see: what lies behind the last one is
  // unwritten, and a NaN value must not reach the rows that do not see it (0 times NaN), so
  // both are cleared and the NaN tokens noted.
  auto clean_page = [&](int kt, int j, int buf) {
    unsigned any = 0;
    for (int i = 0; i < kCopies; ++i) {
      const int place = i * kThreads + tid, d = place / 4, t16 = ((place & 3) ^ v_place(d)) * 16;
      i32x4* const at = (i32x4*)&sV[buf][place * 16];
      i32x4 v = *at;
      unsigned nan = 0;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        v[w] = codes_before(v[w], t16 + 4 * w, r.kv - kt * kPage);
        nan |= nan_codes(v[w]);
      }
      unsigned bits = 0;
      if (nan != 0) {
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (((unsigned)v[e >> 2] >> 8 * (e & 3) & 0x7f) == 0x7f) {
            bits |= 1u << e;
            v[e >> 2] &= (int)~(0xffu << 8 * (e & 3));
          }
        any = 1;
      }
      s_nan[j][d * 4 + t16 / 16] = (unsigned short)bits;
      *at = v;
    }
    const int found = __builtin_amdgcn_ballot_w64(any != 0) != 0;
    if (lane == 0) s_any[j][wave] = found;
  };

  if (kt0 < kt1) {
#pragma unroll
    for (int j = 0; j < kTogether; ++j) next_id(kt0 + j, j);
#pragma unroll
    for (int j = 0; j < kTogether; ++j) load_page(kt0 + j, j, j);
  }
  // Q^T operands: the lane's row, columns 64 s + 32 hi ..+31, as codes under 2^(q_scale[s] - 127).
  i32x8 qh[KS], ql[KS];
  int q_scale[KS];
  {
    const bf16_t* q = a.q + (int64_t)b * a.q_sb + (int64_t)ti * a.q_st + (int64_t)h * a.q_sh + 32 * hi;
    i32x4 x[KS][4];  // columns 64 s + 32 hi + 8 j ..+7
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int j = 0; j < 4; ++j) x[s][j] = row < Rm ? *(const i32x4*)&q[64 * s + 8 * j] : i32x4{0, 0, 0, 0};
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      int e01[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int most = max(largest_bits(x[s][2 * c]), largest_bits(x[s][2 * c + 1]));
        const auto both = __builtin_amdgcn_permlane32_swap(most, most, false, false);
        e01[c] = exponent_for(max((int)both[0], (int)both[1]));
      }
      q_scale[s] = 127 + (hi ? e01[1] : e01[0]);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int e = e01[j >> 2];
        const int w0 = x[s][j >> 1][2 * (j & 1)], w1 = x[s][j >> 1][2 * (j & 1) + 1];
        const float f0 = coded_value(__int_as_float(w0 << 16), e), f1 = coded_value(__int_as_float(w0 & 0xffff0000), e);
        const float f2 = coded_value(__int_as_float(w1 << 16), e), f3 = coded_value(__int_as_float(w1 & 0xffff0000), e);
        int c_hi, c_lo;
        halves8(f0, f1, f2, f3, c_hi, c_lo);
        qh[s][j] = c_hi;
        ql[s][j] = c_lo;
      }
    }
  }
  f32x16 oacc[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) oacc[dt] = f32x16{};
  float m_run = -INFINITY, l_run = 0.f;
  const float c2 = a.scale_log2;
  const int k_token = 32 * (l32 >> 2 & 1) + 4 * (l32 >> 3) + (l32 & 3);  // + 16 t
  const int k_base = k_token * D, k_turn = 32 * hi ^ 16 * k_place(k_token);
  const int v_base = l32 * kPage, v_turn = 32 * hi ^ 16 * v_place(l32);

  auto compute = [&](int kt, int j, int buf, int k_scale, int e_v) __attribute__((always_inline)) {
    const int base = kt * kPage;
    if (!active || base >= w_max) return;
    f32x16 st[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      st[t] = f32x16{};
      const uint8_t* const kp = &sK[buf][k_base + t * 16 * D];
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const i32x4 k0 = *(const i32x4*)&kp[k_turn ^ (64 * s)], k1 = *(const i32x4*)&kp[k_turn ^ (64 * s + 16)];
        const i32x8 k = __builtin_shufflevector(k0, k1, 0, 1, 2, 3, 4, 5, 6, 7);
        st[t] = mfma8(k, ql[s], st[t], k_scale, q_scale[s] - kLoShift);
        st[t] = mfma8(k, qh[s], st[t], k_scale, q_scale[s]);
      }
    }
    // tokens 32 hi + 16 t + e
    if (base + kPage > w_min) {
      const int see = limit - base - 32 * hi;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (16 * t + e >= see) st[t][e] = -INFINITY;
    }
    float mx = -INFINITY;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) mx = fmaxf(mx, st[t][e]);
    mx = xor32_max(mx);
    // The reference maximum moves only when it grows by more than 2^8 in probability terms.
    const float m_cand = fmaxf(m_run, mx);
    const bool grow = (m_cand - m_run) * c2 > 8.f;
    if (__builtin_amdgcn_ballot_w64(grow) != 0) {
      const float m_new = grow ? m_cand : m_run;
      const float alpha = m_new == -INFINITY ? 1.f : fast_exp2((m_run - m_new) * c2);
      l_run *= alpha;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) oacc[dt] *= alpha;
      m_run = m_new;
    }
    const float ref = m_run == -INFINITY ? 0.f : m_run, mb = ref * c2;
    // Scaled scores past 2^16 are known to 2^-8 only: their difference is formed before the scale, at an
    // operation more each, or rounding them apart would give probabilities up to 2^(their ulp).
    if (__builtin_amdgcn_ballot_w64(__builtin_fabsf(mb) > 65536.f) != 0) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) st[t][e] = fast_exp2((st[t][e] - ref) * c2);
    } else {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) st[t][e] = fast_exp2(__builtin_fmaf(st[t][e], c2, -mb));
    }
    float lsum = 0.f;
    bf16x8 pf[4];  // tokens 32 hi + 8 s ..+7
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      f32x8 x;
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = st[s >> 1][8 * (s & 1) + e];
      lsum += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
      pf[s] = to_bf16x8(x);
    }
    l_run += lsum;
    const float vs = pow2(e_v);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const uint8_t* const vp = &sV[buf][v_base + dt * 32 * kPage];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const i32x4 v = *(const i32x4*)&vp[half ? v_turn ^ 16 : v_turn];
        oacc[dt] = mfma32(decode8(v[0], v[1], vs), pf[2 * half], oacc[dt]);
        oacc[dt] = mfma32(decode8(v[2], v[3], vs), pf[2 * half + 1], oacc[dt]);
      }
    }
    if (__builtin_expect(base + kPage > wg_min && __builtin_amdgcn_readfirstlane(s_any[j][0] | s_any[j][1] | s_any[j][2] | s_any[j][3]), 0)) {
      // NaN values into the rows that see them
      const int n = limit - base;
      const uint64_t seen = n >= 64 ? ~0ull : (n <= 0 ? 0ull : (1ull << n) - 1);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int d = 32 * dt + 8 * (e >> 2) + 4 * hi + (e & 3);
          if (*(const uint64_t*)&s_nan[j][4 * d] & seen) oacc[dt][e] = __builtin_nanf("");
        }
    }
  };

  for (int kt = kt0, buf = 0; kt < kt1; kt += kTogether, buf ^= kTogether) {
    wait_vmem();  // the pages' copies
    __syncthreads();
    int k_scale[kTogether], e_v[kTogether];
    bool there[kTogether], cleaned = false;
#pragma unroll
    for (int j = 0; j < kTogether; ++j) {
      k_scale[j] = 127 + ek[j], e_v[j] = ev[j], there[j] = some[j];
      if (there[j] && (kt + j) * kPage + kPage > wg_min) {  // uniform
        clean_page(kt + j, j, buf + j);
        cleaned = true;
      }
    }
    if (cleaned) __syncthreads();
#pragma unroll
    for (int j = 0; j < kTogether; ++j) load_page(kt + kTogether + j, j, (buf ^ kTogether) + j);
#pragma unroll
    for (int j = 0; j < kTogether; ++j)
      if (there[j]) compute(kt + j, j, buf + j, k_scale[j], e_v[j]);
  }

  const float l_tot = xor32_sum(l_run);
  if (n_valid <= 1) {
    if (!row_ok) return;
    const float inv = row < Rm && l_tot != 0.f ? 1.f / l_tot : 0.f;
    bf16_t* const o = a.out + (int64_t)b * a.o_sb + (int64_t)ti * a.o_st + (int64_t)h * a.o_sh;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int rg = 0; rg < 4; ++rg) {
        f32x4 t;
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] = row < Rm ? oacc[dt][4 * rg + e] * inv : 0.f;
        *(bf16x4*)&o[32 * dt + 8 * rg + 4 * hi] = __builtin_convertvector(t, bf16x4);
      }
    return;
  }
  const int64_t slot = unit * kRows + wave * 32 + l32;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int rg = 0; rg < 4; ++rg) {
      f32x4 t;
#pragma unroll
      for (int e = 0; e < 4; ++e) t[e] = oacc[dt][4 * rg + e];
      *(f32x4*)&a.part_o[slot * D + 32 * dt + 8 * rg + 4 * hi] = t;
    }
  if (hi == 0) *(f32x2*)&a.part_ml[slot * 2] = f32x2{m_run == -INFINITY ? -INFINITY : m_run * c2, l_tot};
}
__global__ __launch_bounds__(kThreads, 2) void paged_prefill_d128_kernel(const PagedArgs a) { paged_prefill_body<128, false>(a); }
__global__ __launch_bounds__(kThreads, 2) void paged_prefill_d64_kernel(const PagedArgs a) { paged_prefill_body<64, false>(a); }
__global__ __launch_bounds__(kThreads, 2) void paged_prefill_runs_d128_kernel(const PagedArgs a) { paged_prefill_body<128, true>(a); }
__global__ __launch_bounds__(kThreads, 3) void paged_prefill_runs_d64_kernel(const PagedArgs a) { paged_prefill_body<64, true>(a); }

// Of a row tile: its batch row, the parts it is in, and the first of them.
struct Parts {
  PagedRow r;
  int n;
  int64_t first;
  __device__ __forceinline__ Parts(const PagedArgs& a, int b, int hk, int rt) {
    if (a.slots > 0) {
      const Runs runs(a, threadIdx.x & 63);
      r = runs.row(b);
      n = __builtin_amdgcn_readlane(runs.n, b);
      first = runs.first(a, b, hk, rt);
    } else {
      r = PagedRow(a, b);
      const int tiles = (r.kv + kPage - 1) / kPage, per = max(1, (tiles + a.splits - 1) / a.splits);
      n = (tiles + per - 1) / per;
      first = (((int64_t)b * a.Hkv + hk) * a.n_rt + rt) * a.splits;
    }
  }
};

// Adds the partial rows of many key splits (short chunks on long rows), one wave to a row.
template <int D>
__device__ __forceinline__ void paged_merge_many_body(const PagedArgs& a) {
  touch_args<sizeof(PagedArgs)>();
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int R = a.S * a.G, groups = (R + kWaves - 1) / kWaves;
  const int row = blockIdx.x % groups * kWaves + wave, pair = blockIdx.x / groups;
  const int b = pair / a.Hkv, hk = pair - b * a.Hkv;
  if (row >= R) return;
  const Parts parts(a, b, hk, row / kRows);
  const PagedRow& r = parts.r;
  const int n = parts.n;
  if (n <= 1) return;  // written by its split
  const int i = row / a.G;
  bf16_t* const o = a.out + (int64_t)b * a.o_sb + (int64_t)i * a.o_st + (int64_t)(hk * a.G + row - i * a.G) * a.o_sh;
  if (i >= r.m) {  // a padding query
    if (lane < D / 8) *(bf16x8*)&o[lane * 8] = bf16x8{};
    return;
  }
  merge_parts<D>(a, n, lane, [&](int c) { return (parts.first + c) * kRows + row % kRows; }, o);
}
__global__ __launch_bounds__(kThreads) void paged_merge_many_d128_kernel(const PagedArgs a) { paged_merge_many_body<128>(a); }
__global__ __launch_bounds__(kThreads) void paged_merge_many_d64_kernel(const PagedArgs a) { paged_merge_many_body<64>(a); }

// The same for a few splits of many rows, D / 4 lanes to a row and four columns each, four parts at once (a wave to
// a row / so: 8 x 512 on 1536 keys, 8 / 8 heads of 64, two splits, 64.4 / 47.6 us; 100 on 3000, 16 / 4 heads
// of 128, 32 splits, 32.6 / 33.0).
constexpr int kFewSplits = 8;
template <int D>
__device__ __forceinline__ void paged_merge_splits_body(const PagedArgs& a) {
  touch_args<sizeof(PagedArgs)>();
  constexpr int kLanes = D / 4, kRowsAt = kThreads / kLanes, kChunk = 4;
  const int R = a.S * a.G, groups = (R + kRowsAt - 1) / kRowsAt;
  const int pair = blockIdx.x / groups, row0 = (blockIdx.x - pair * groups) * kRowsAt, row = row0 + (int)threadIdx.x / kLanes;
  const int b = pair / a.Hkv, hk = pair - b * a.Hkv, col = threadIdx.x % kLanes * 4;
  // A workgroup's rows lie in one row tile.  One wave looks it up: all four, each over 64 batch rows, made the
  // launch VALU bound (5 x up to 1339 tokens, 8 heads of 64: 9.0 us).
  __shared__ int s_n, s_m;
  __shared__ int64_t s_first;
  if (threadIdx.x < 64) {
    const Parts parts(a, b, hk, row0 / kRows);
    if (threadIdx.x == 0) {
      s_n = parts.n;
      s_m = parts.r.m;
      s_first = parts.first;
    }
  }
  __syncthreads();
  const int n = s_n;
  if (n <= 1 || row >= R) return;  // written by its split
  const int i = row / a.G;
  bf16_t* const out = a.out + (int64_t)b * a.o_sb + (int64_t)i * a.o_st + (int64_t)(hk * a.G + row - i * a.G) * a.o_sh + col;
  if (i >= s_m) {  // a padding query
    *(bf16x4*)out = bf16x4{};
    return;
  }
  const int64_t part = s_first * kRows + row % kRows;  // + kRows each
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  float M = -INFINITY, lsum = 0.f;
  for (int c0 = 0; c0 < n; c0 += kChunk) {
    f32x2 ml[kChunk];
    f32x4 o[kChunk];
#pragma unroll
    for (int c = 0; c < kChunk; ++c) {
      const int64_t at = part + min(c0 + c, n - 1) * kRows;
      ml[c] = *(const f32x2*)&a.part_ml[2 * at];
      o[c] = *(const f32x4*)&a.part_o[at * D + col];
    }
    float m_new = M;
#pragma unroll
    for (int c = 0; c < kChunk; ++c) {
      if (c0 + c >= n) ml[c] = f32x2{-INFINITY, 0.f};
      m_new = fmaxf(m_new, ml[c][0]);
    }
    const float alpha = M == -INFINITY ? 1.f : fast_exp2(M - m_new);  // (what M = -inf has added is 0 or NaN)
    acc *= alpha;
    lsum *= alpha;
    M = m_new;
#pragma unroll
    for (int c = 0; c < kChunk; ++c) {
      const float w = ml[c][0] == -INFINITY ? ml[c][1] : fast_exp2(ml[c][0] - M);  // no key: a sum of 0 (or NaN)
      lsum += ml[c][1] * w;
      if (w != 0.f) acc += o[c] * w;
    }
  }
  const float inv = lsum != 0.f ? 1.f / lsum : 0.f;
  *(bf16x4*)out = __builtin_convertvector(acc * inv, bf16x4);
}
__global__ __launch_bounds__(kThreads) void paged_merge_splits_d128_kernel(const PagedArgs a) { paged_merge_splits_body<128>(a); }
__global__ __launch_bounds__(kThreads) void paged_merge_splits_d64_kernel(const PagedArgs a) { paged_merge_splits_body<64>(a); }

// ------------------------------------------------------------------ host side

struct Plan {
  bool decode, pairs;
  int n_rt, splits, slots;
  int64_t units;  // workgroups of the attention kernel
  size_t workspace_bytes;
};

Plan plan_of(const MimirPagedAttnParams& p) {
  Plan s = {};
  const int64_t cus = device_cu_count(), R = (int64_t)p.seqlen * (p.num_q_heads / p.num_kv_heads);
  const int64_t pairs = (int64_t)p.batch * p.num_kv_heads;
  s.decode = R <= kDecRows;
  s.splits = 1;
  if (s.decode) {
    const int64_t most = (int64_t)p.batch * ((p.table_width + kUnit - 1) / kUnit);  // units of the line
    // One workgroup per pair (nothing to merge, one launch) for short tables, and the longer the more pairs there
    // are to even out, up to 1 MiB of keys and values: the longest pair runs alone.  Shares / pairs, 16 / 4
    // heads of 128: one row of 450 keys 14.3 / 8.8 us, of 1000 14.1 / 12.1, of 2000 13.9 / 19.1; 8 rows of up to
    // 1000 14.7 / 13.8, 1500 14.8 / 17.1; 64 of up to 1000 26.0 / 15.9, 2000 32.0 / 25.9, 8000 62 / 75; 200 of up
    // to 2000 67 / 61; 128 of up to 6000, 32 / 8 heads, 168 / 175.  Heads of 64: 64 of up to 3000, 8 / 8, 32.5 /
    // 25.1, 250 of up to 4000, 8 / 2, 39.1 / 31.6, 48 of up to 4000 17.4 / 29.4.  Twice as long with two row tiles,
    // whose parts are larger (64 rows of up to 2000, 16 / 4 heads of 128, 5 tokens: 54 / 31).
    const int64_t pair_pages = std::max<int64_t>(16, std::min<int64_t>(16 * pairs, 8192) / p.head_dim * (R > 16 ? 2 : 1));
    s.pairs = p.batch > kLineRows || p.table_width <= pair_pages;
    if (s.pairs) {
      s.units = pairs;
    } else {
      // Workgroups per CU: as many as fit at once (registers), two at head_dim 128 or with two row tiles, three
      // else.  Two / three / four, heads of 64: 64 rows of 2000 to 16000 keys, 8 / 8, 90.5 / 89.6 / 95.1 us; 200 rows of
      // 1100 to 9000, 8 / 2, 57.6 / 57.0 / 63.1.  Of 128 two are faster than three or four.
      const int64_t per_cu = p.head_dim == 64 && R <= 16 ? 3 : 2;
      s.units = p.num_kv_heads * std::max<int64_t>(1, std::min(most, per_cu * cus / p.num_kv_heads));
      s.workspace_bytes = (size_t)s.units * 2 * (size_t)R * ((size_t)p.head_dim + 2) * sizeof(float);
    }
    return s;
  }
  s.n_rt = (int)((R + kRows - 1) / kRows);
  const int64_t groups = pairs * s.n_rt;
  s.splits = (int)std::max<int64_t>(1, std::min<int64_t>({(2 * cus + groups * 3 / 4) / groups, p.table_width, kMaxSplits}));
  s.units = groups * s.splits;
  if (p.new_lengths != nullptr && p.batch <= kDealtRows && groups <= 4 * cus && p.table_width <= 1 << 20) {
    s.slots = (int)((p.head_dim == 64 ? 3 : 1) * cus);
    s.units = groups + s.slots;  // runs: pages / per <= slots, and one more for each row tile
  }
  s.workspace_bytes = s.splits > 1 || s.slots > 0 ? (size_t)s.units * kRows * ((size_t)p.head_dim + 2) * sizeof(float) : 0;
  return s;
}

hipError_t launch_paged_attn(const MimirPagedAttnParams& p, const Plan& plan, hipStream_t stream) {
  PagedArgs a = {};
  a.q = (const bf16_t*)p.q;
  a.kn = (const bf16_t*)p.k_new;
  a.vn = (const bf16_t*)p.v_new;
  a.out = (bf16_t*)p.out;
  a.ck = (uint8_t*)p.cache_k;
  a.cv = (uint8_t*)p.cache_v;
  a.ke = p.k_exponents;
  a.ve = p.v_exponents;
  a.table = p.page_table;
  a.lengths = p.cache_lengths;
  a.indices = p.batch_indices;
  a.fresh = p.new_lengths;
  a.q_sb = p.q_stride_batch; a.q_st = p.q_stride_token; a.q_sh = p.q_stride_head;
  a.kn_sb = p.kn_stride_batch; a.kn_st = p.kn_stride_token; a.kn_sh = p.kn_stride_head;
  a.vn_sb = p.vn_stride_batch; a.vn_st = p.vn_stride_token; a.vn_sh = p.vn_stride_head;
  a.o_sb = p.out_stride_batch; a.o_st = p.out_stride_token; a.o_sh = p.out_stride_head;
  a.k_sp = p.k_stride_page; a.v_sp = p.v_stride_page; a.ke_sp = p.ke_stride_page; a.ve_sp = p.ve_stride_page;
  a.t_st = p.table_stride;
  a.B = p.batch;
  a.S = p.seqlen;
  a.num_pages = p.num_pages;
  a.rows = p.table_rows;
  a.width = p.table_width;
  a.Hkv = p.num_kv_heads;
  a.G = p.num_q_heads / p.num_kv_heads;
  a.causal = p.causal != 0;
  a.D = p.head_dim;
  a.idx64 = p.index_int64 != 0;
  a.scale_log2 = std::max(p.softmax_scale * kLog2e, 1.2e-38f);  // a normal number: masked scores times it stay -inf
  a.n_rt = plan.n_rt;
  a.splits = plan.splits;
  a.slots = plan.slots;
  a.cus = device_cu_count();
  a.part_o = (float*)p.workspace;
  const int64_t R = (int64_t)a.S * a.G;
  if (!plan.decode) {
    const hipError_t e = launch_paged_append(a, stream);
    if (e != hipSuccess) return e;
  }
  const dim3 grid((unsigned)plan.units), block(kThreads);
  const dim3 merge((unsigned)((int64_t)a.B * a.Hkv * ((R + kWaves - 1) / kWaves)));
  if (plan.decode) {
    a.shares = (int)(plan.units / a.Hkv);
    a.part_ml = a.part_o + (size_t)plan.units * 2 * R * p.head_dim;
#define DECODE(D, NR)                                                                                             \
  if (plan.pairs)                                                                                                 \
    hipLaunchKernelGGL(paged_decode_pairs_d##D##_r##NR##_kernel, grid, block, 0, stream, a);                        \
  else                                                                                                            \
    hipLaunchKernelGGL(paged_decode_d##D##_r##NR##_kernel, grid, block, 0, stream, a);
    if (a.D == 128 && R <= 16) {
      DECODE(128, 1)
    } else if (a.D == 128) {
      DECODE(128, 2)
    } else if (R <= 16) {
      DECODE(64, 1)
    } else {
      DECODE(64, 2)
    }
#undef DECODE
    if (plan.pairs) return hipGetLastError();
    if (a.D == 128)
      hipLaunchKernelGGL(paged_merge_d128_kernel, merge, block, 0, stream, a);
    else
      hipLaunchKernelGGL(paged_merge_d64_kernel, merge, block, 0, stream, a);
    return hipGetLastError();
  }
  a.part_ml = a.part_o + (size_t)plan.units * kRows * p.head_dim;
  if (a.slots > 0 && a.D == 128)
    hipLaunchKernelGGL(paged_prefill_runs_d128_kernel, grid, block, 0, stream, a);
  else if (a.slots > 0)
    hipLaunchKernelGGL(paged_prefill_runs_d64_kernel, grid, block, 0, stream, a);
  else if (a.D == 128)
    hipLaunchKernelGGL(paged_prefill_d128_kernel, grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL(paged_prefill_d64_kernel, grid, block, 0, stream, a);
  if (plan.splits > 1 || plan.slots > 0) {
    const int rows_at = 4 * kThreads / a.D;
    const dim3 joined((unsigned)((int64_t)a.B * a.Hkv * ((R + rows_at - 1) / rows_at)));
    if (plan.splits > kFewSplits && a.D == 128)
      hipLaunchKernelGGL(paged_merge_many_d128_kernel, merge, block, 0, stream, a);
    else if (plan.splits > kFewSplits)
      hipLaunchKernelGGL(paged_merge_many_d64_kernel, merge, block, 0, stream, a);
    else if (a.D == 128)
      hipLaunchKernelGGL(paged_merge_splits_d128_kernel, joined, block, 0, stream, a);
    else
      hipLaunchKernelGGL(paged_merge_splits_d64_kernel, joined, block, 0, stream, a);
  }
  return hipGetLastError();
}

// A bf16 operand of `heads` heads: pointer, then batch / token / head strides.
int check_rows(const char* name, const void* x, int64_t sb, int64_t st, int64_t sh) {
  if (x == nullptr) return fail_with(MIMIR_ERR_INVALID_ARGUMENT, std::string(name) + " is NULL");
  if ((uintptr_t)x % 16 != 0 || sb < 0 || st < 0 || sh < 0 || sb % 8 != 0 || st % 8 != 0 || sh % 8 != 0)
    return fail_with(MIMIR_ERR_UNSUPPORTED_SHAPE, std::string(name) + " must be 16-byte aligned with non-negative strides that are multiples of 8 elements");
  return MIMIR_OK;
}

bool sizes_ok(const MimirPagedAttnParams* p) {
  return p != nullptr && p->batch >= 0 && p->seqlen >= 0 && p->num_pages >= 0 && p->table_rows >= 0 && p->table_width >= 0 &&
         p->num_q_heads > 0 && p->num_kv_heads > 0 && p->num_q_heads % p->num_kv_heads == 0;
}

}  // namespace
}  // namespace mimir

extern "C" {

size_t mimir_prefixlm_paged_attn_workspace_bytes(const MimirPagedAttnParams* p) {
  if (!mimir::sizes_ok(p) || p->batch == 0 || p->seqlen == 0) return 0;
  return mimir::plan_of(*p).workspace_bytes;
}

int mimir_prefixlm_paged_attn(const MimirPagedAttnParams* p, void* stream) {
  using namespace mimir;
  fail_with(MIMIR_OK, "");
  if (p == nullptr) return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "params is NULL");
  if (p->dtype != MIMIR_DTYPE_BFLOAT16)
    return fail_with(MIMIR_ERR_UNSUPPORTED_DTYPE, "paged attention supports bfloat16 queries only (dtype code " + std::to_string(p->dtype) + ")");
  if (!sizes_ok(p))
    return fail_with(MIMIR_ERR_INVALID_ARGUMENT, p->num_kv_heads > 0 && p->num_q_heads > 0 && p->num_q_heads % p->num_kv_heads != 0
                         ? "Query heads " + std::to_string(p->num_q_heads) + " must be divisible by key/value heads " + std::to_string(p->num_kv_heads) + "."
                         : std::string("negative size or non-positive head count"));
  if (p->head_dim != 64 && p->head_dim != 128)
    return fail_with(MIMIR_ERR_UNSUPPORTED_SHAPE, "head_dim " + std::to_string(p->head_dim) + " is not supported by paged attention (supported: 64, 128)");
  if (!(p->softmax_scale > 0.f) || !std::isfinite(p->softmax_scale))
    return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "softmax_scale must be positive and finite");
  if (p->batch == 0 || p->seqlen == 0) return MIMIR_OK;
  if (p->num_pages == 0 || p->table_width == 0) return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "the cache holds no pages");
  if (p->table_width > (1 << 24)) return fail_with(MIMIR_ERR_UNSUPPORTED_SHAPE, "page tables wider than 2^24 are not supported");
  if (p->page_table == nullptr || p->cache_lengths == nullptr) return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "page_table or cache_lengths is NULL");
  if (p->table_stride < 0) return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "negative table_stride");
  int rc;
  if ((rc = check_rows("q", p->q, p->q_stride_batch, p->q_stride_token, p->q_stride_head)) ||
      (rc = check_rows("k_new", p->k_new, p->kn_stride_batch, p->kn_stride_token, p->kn_stride_head)) ||
      (rc = check_rows("v_new", p->v_new, p->vn_stride_batch, p->vn_stride_token, p->vn_stride_head)) ||
      (rc = check_rows("out", p->out, p->out_stride_batch, p->out_stride_token, p->out_stride_head)))
    return rc;
  if (p->cache_k == nullptr || p->cache_v == nullptr || p->k_exponents == nullptr || p->v_exponents == nullptr)
    return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "cache pointer is NULL");
  const int64_t page = (int64_t)p->num_kv_heads * kPage * p->head_dim;
  if ((uintptr_t)p->cache_k % 16 != 0 || (uintptr_t)p->cache_v % 16 != 0 || p->k_stride_page % 16 != 0 || p->v_stride_page % 16 != 0 ||
      (p->num_pages > 1 && (p->k_stride_page < page || p->v_stride_page < page || p->ke_stride_page < p->num_kv_heads ||
                            p->ve_stride_page < p->num_kv_heads)))
    return fail_with(MIMIR_ERR_UNSUPPORTED_SHAPE, "pages of the cache must be 16-byte aligned and apart");
  const Plan plan = plan_of(*p);
  const int64_t rows = (int64_t)p->seqlen * (p->num_q_heads / p->num_kv_heads), pairs = (int64_t)p->batch * p->num_kv_heads;
  const int64_t append = plan.decode ? 0 : pairs * (((int64_t)p->seqlen + 2 * kPage - 2) / kPage);
  const int64_t merge = plan.workspace_bytes > 0 ? pairs * ((rows + kWaves - 1) / kWaves) : 0;
  if (rows > 0x7fffffff || plan.units > kMaxGroups || append > kMaxGroups || merge > kMaxGroups)
    return fail_with(MIMIR_ERR_UNSUPPORTED_SHAPE, "too many query rows for one call; split the batch");
  if (plan.workspace_bytes > 0 && (p->workspace == nullptr || p->workspace_bytes < plan.workspace_bytes || (uintptr_t)p->workspace % 16 != 0))
    return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "workspace must be 16-byte aligned and hold at least " + std::to_string(plan.workspace_bytes) + " bytes");
  const hipError_t e = launch_paged_attn(*p, plan, (hipStream_t)stream);
  return e == hipSuccess ? MIMIR_OK : fail_with(MIMIR_ERR_HIP, std::string("paged attention launch: ") + hipGetErrorString(e));
}

}  // extern "C"
