// Beam search: the best continuations over a request's beams and the vocabulary, and the rows of
// static caches in the order of the chosen beams.
//
// Selection.  Of logits x[r, w, :], scores s[r, w] and lse = log sum exp x, the `count` largest
// s + x - lse of a request, ties to the lowest (beam, token).  Bound by reading the logits once: one
// workgroup of beam_rows_kernel per piece of a row keeps the piece in registers, and from there
//   * sums exp(x - max) in fp32, a few adds a lane;
//   * finds a threshold that at least `count` elements reach: the count-th largest of a wave's lane maxima,
//     found with ballots two bits at a time (8 steps for bf16), and the largest of that over the waves;
//   * ranks the few elements that reach it and stores the best `count`, in order.
// 48 x 8 rows of 128257 bf16 logits: 27 us (3.3 TB/s). A workgroup computes once its whole piece is there, and the vector units
// issue in 62% of the cycles of CUs with work, 38% of all.
// Within a row larger logits are larger scores, so this needs no lse.  beam_merge_kernel, a workgroup per
// request, joins the pieces' sums, forms the scores of the stored elements in 64 bits, takes the lists whose best reaches
// the count-th largest of 64 groups' best, and ranks what of them does.  (The sums are fp32: all scores of a beam are off by
// the same, less than 2^-19, and beams closer than twice that may change places.)  Masked logits, ended beams and rows of
// ties need no case of their own but for more candidates than the lists hold, which fall back to `count` rounds of a maximum.
//
// Reordering.  Rows of a group take each other's place, so every row is read before any is written: a
// thread owns 16 bytes of the same place in all rows of a group, loads what moves and then stores it.
// Bound by copying: 317 MB of 16 x 8 rows in 63.5 us, 5.0 TB/s.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "prefixlm_common.h"
#include "strided_overlap.h"

namespace mimir {
namespace {

constexpr int kMaxBeams = 32, kMaxCount = 64;
constexpr int kCap = 1024;  // candidates ranked at once
constexpr float kFusedTop = 4096.f;  // log2(e) times it is below 2^13, whose fp32 neighbours are 2^-11 apart

struct SelectArgs {
  const void* logits;
  const float* scores;
  const uint8_t* finished;
  float* out_scores;
  int32_t *out_tokens, *out_rows;
  uint8_t* out_finished;
  int64_t l_sr, l_sw, s_sr, s_sw, f_sr, f_sw;
  int R, W, V, K, end, chunks;
  f32x2* sums;      // [R * W][chunks]: maximum, sum of exp(x - maximum)
  uint64_t* lists;  // [R * W][chunks][K], best first, 0: none
};

// Larger logits have larger codes, equal ones (-0 and 0 among them) equal codes; below that of any finite
// logit lies 0.
__device__ __forceinline__ uint32_t order_code(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float order_value(uint32_t c) { return __uint_as_float(c ^ ((c >> 31) ? 0x80000000u : 0xffffffffu)); }
__device__ __forceinline__ uint64_t list_key(float x, int token) { return (uint64_t)order_code(x) << 32 | (uint32_t)~token; }
__device__ __forceinline__ float key_value(uint64_t k) { return order_value((uint32_t)(k >> 32)); }
__device__ __forceinline__ int key_token(uint64_t k) { return (int)~(uint32_t)k; }

// Over the wave, on every lane, without LDS round trips.
template <typename F>
__device__ __forceinline__ float wave_reduce(float x, F&& f) {
  auto dpp = [&](auto ctrl) __attribute__((always_inline)) {
    const int v = __float_as_int(x);
    return f(x, __int_as_float(__builtin_amdgcn_update_dpp(v, v, decltype(ctrl)::value, 0xf, 0xf, false)));
  };
  x = dpp(std::integral_constant<int, 0xb1>());   // quad_perm: lane ^ 1
  x = dpp(std::integral_constant<int, 0x4e>());   // quad_perm: lane ^ 2
  x = dpp(std::integral_constant<int, 0x141>());  // row_half_mirror: the other quad of eight
  x = dpp(std::integral_constant<int, 0x140>());  // row_mirror: the other eight of sixteen
  const int v = __float_as_int(x);
  const auto p = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  const int a = p[0], b = p[1];
  x = f(__int_as_float(a), __int_as_float(b));
  float lo, hi;
  halves(x, lo, hi);
  return f(lo, hi);
}
// The count-th largest of the wave's codes, or less (0) where so many lanes hold none; from the top bit down to
// `low`, two bits a step.
template <int kLow>
__device__ __forceinline__ uint32_t wave_kth(uint32_t code, int count) {
  uint32_t reach = 0;
#pragma unroll
  for (int bit = 30; bit >= kLow; bit -= 2) {
    const uint32_t one = 1u << bit;
    const int n1 = __builtin_popcountll(__builtin_amdgcn_ballot_w64(code >= reach + one));
    const int n2 = __builtin_popcountll(__builtin_amdgcn_ballot_w64(code >= reach + 2 * one));
    const int n3 = __builtin_popcountll(__builtin_amdgcn_ballot_w64(code >= reach + 3 * one));
    reach += n3 >= count ? 3 * one : n2 >= count ? 2 * one : n1 >= count ? one : 0;
  }
  return reach;
}

// 16 bytes of logits at any address of theirs.
struct __attribute__((packed, aligned(2))) Loose2 {
  i32x4 v;
};
struct __attribute__((packed, aligned(4))) Loose4 {
  i32x4 v;
};
__device__ __forceinline__ i32x4 load_loose(const bf16_t* p) { return ((const Loose2*)p)->v; }
__device__ __forceinline__ i32x4 load_loose(const float* p) { return ((const Loose4*)p)->v; }
// Element e of a vector as it lies in registers.
__device__ __forceinline__ float element(const i32x4& v, int e, bf16_t) {
  return __int_as_float(e % 2 ? v[e / 2] & (int)0xffff0000 : v[e / 2] << 16);
}
__device__ __forceinline__ float element(const i32x4& v, int e, float) { return __int_as_float(v[e]); }
__device__ __forceinline__ void set_element(i32x4& v, int e, bf16_t x) {
  const int b = __builtin_bit_cast(uint16_t, x);
  v[e / 2] = e % 2 ? (v[e / 2] & 0xffff) | b << 16 : (v[e / 2] & (int)0xffff0000) | b;
}
__device__ __forceinline__ void set_element(i32x4& v, int e, float x) { v[e] = __float_as_int(x); }

// Between its uses the piece stays in registers as it was loaded: unpacked once for all of them, the bf16 kernel
// took 162 registers and ran three waves a SIMD.
template <int NV>
__device__ __forceinline__ void keep_packed(i32x4 (&v)[NV]) {
#pragma unroll
  for (int j = 0; j < NV; ++j) __asm__ volatile("" : "+v"(v[j]));
}
template <typename E, int NV>
__global__ __launch_bounds__(256) void beam_rows_kernel(const SelectArgs a) {
  constexpr int kVec = 16 / sizeof(E);
  __shared__ uint64_t keys[kCap];
  __shared__ float wave_max[4], wave_sum[4];
  __shared__ uint32_t wave_code[4];
  __shared__ uint16_t vectors[256 * NV];
  __shared__ int noted, found;
  __shared__ uint64_t round_best[4];
  const int tid = threadIdx.x, wave = tid >> 6;
  const int row = blockIdx.x / a.chunks, chunk = blockIdx.x - row * a.chunks;
  const int r = row / a.W, w = row - r * a.W;
  const float score = a.scores[r * a.s_sr + w * a.s_sw];
  const bool ended = a.finished != nullptr && a.finished[r * a.f_sr + w * a.f_sw] != 0;
  if (ended || !(fabsf(score) < INFINITY)) return;  // the merge does not read this row's pieces
  const E* const x = (const E*)a.logits + r * a.l_sr + w * a.l_sw;
  const int first = chunk * (256 * NV * kVec) + tid * kVec;
  // Vector j holds the tokens from token_of(j) on; past the end it is the row's last whole vector, and -inf where another holds
  // the same tokens.
  auto at_of = [&](int j) __attribute__((always_inline)) { return first + j * 256 * kVec; };
  auto token_of = [&](int j) __attribute__((always_inline)) { return max(min(at_of(j), a.V - kVec), 0); };
  const bool last_chunk = chunk == a.chunks - 1;
  auto mask_vector = [&](int j, i32x4& u) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < kVec; ++e)
      if (token_of(j) + e < at_of(j) || token_of(j) + e >= a.V) set_element(u, e, (E)-INFINITY);
  };
  i32x4 v[NV];
  if (a.V >= kVec) {
#pragma unroll
    for (int j = 0; j < NV; ++j) v[j] = load_loose(x + token_of(j));
  } else {
#pragma unroll
    for (int j = 0; j < NV; ++j) v[j] = i32x4{0, 0, 0, 0};
    for (int e = 0; e < a.V; ++e) set_element(v[0], e, x[e]);
  }
  if (last_chunk) {
#pragma unroll
    for (int j = 0; j < NV; ++j) mask_vector(j, v[j]);
  }
  float most[NV], top = -INFINITY;  // NaN is left out here and comes back in the sum
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    most[j] = -INFINITY;
#pragma unroll
    for (int e = 0; e < kVec; e += 2) most[j] = fmaxf(fmaxf(most[j], element(v[j], e, E())), element(v[j], e + 1, E()));
    top = fmaxf(top, most[j]);
    __builtin_amdgcn_sched_barrier(0);
  }
  keep_packed(v);
  const float wtop = wave_reduce(top, [](float p, float q) { return fmaxf(p, q); });
  // The count-th largest code of the wave's lane maxima: at least `count` elements reach it.
  uint32_t reach = wave_kth<sizeof(E) == 2 ? 16 : 0>(order_code(top), a.K);
  if (sizeof(E) == 2 && reach >> 31 == 0) reach |= 0xffffu;  // a negative bf16's code ends in ones
  if ((tid & 63) == 0) {
    wave_max[wave] = wtop;
    wave_code[wave] = reach;
  }
  if (tid == 0) noted = found = 0;
  __syncthreads();
  const float block_top = fmaxf(fmaxf(wave_max[0], wave_max[1]), fmaxf(wave_max[2], wave_max[3]));
  // exp(x - top) = exp2(x c - top c): one fma with top c rounded, whose rounding (exact by another fma) is taken
  // back from the sum to first order; c's own is one of x - top, not of x.  That rounding grows with top: below
  // kFusedTop it is at most 2^-12 and what the first order leaves (its half square) 2^-26 of the sum.  From there on, as in
  // a piece that is masked with a large finite value, the difference first, which is exact for what counts in the sum.
  const bool near = fabsf(block_top) < kFusedTop;
  const float base = block_top == -INFINITY ? 0.f : block_top, shift = near ? base * kLog2e : 0.f;
  float part[4] = {0.f, 0.f, 0.f, 0.f};
  if (near) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int e = 0; e < kVec; ++e) part[e % 4] += fast_exp2(__builtin_fmaf(element(v[j], e, E()), kLog2e, -shift));
      __builtin_amdgcn_sched_barrier(0);  // a vector at a time, for few registers
    }
  } else {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int e = 0; e < kVec; ++e) part[e % 4] += fast_exp2((element(v[j], e, E()) - base) * kLog2e);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  const float sum = wave_reduce((part[0] + part[1]) + (part[2] + part[3]), [](float p, float q) { return p + q; });
  if ((tid & 63) == 0) wave_sum[wave] = sum;
  const float limit = order_value(max(max(wave_code[0], wave_code[1]), max(wave_code[2], wave_code[3])));
  // The vectors with an element that reaches the limit are noted, and their elements looked at one a thread, from
  // memory: tests of all elements in the registers were a third of the instructions.
#pragma unroll
  for (int j = 0; j < NV; ++j)
    if (most[j] >= limit && most[j] > -INFINITY) {
      const int n = __hip_atomic_fetch_add(&noted, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
      vectors[n] = (uint16_t)(j * 256 + tid);
    }
  __syncthreads();
  const int start = chunk * (256 * NV * kVec);
  for (int i = tid; i < noted * kVec; i += 256) {
    const int at = start + vectors[i / kVec] * kVec, token = max(min(at, a.V - kVec), 0) + i % kVec;
    if (token < at || token >= a.V) continue;  // another vector's, or past the end
    const float y = (float)x[token];
    if (y >= limit && y > -INFINITY) {
      const int n = __hip_atomic_fetch_add(&found, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
      if (n < kCap) keys[n] = list_key(y, token);
    }
  }
  __syncthreads();
  if (tid == 0) {
    const float total = (wave_sum[0] + wave_sum[1]) + (wave_sum[2] + wave_sum[3]);
    const float over = near ? __builtin_fmaf(base, kLog2e, -shift) : 0.f;  // of the exponents, in base 2
    a.sums[blockIdx.x] = f32x2{block_top, total - total * (over * kLn2)};
  }
  uint64_t* const list = a.lists + (int64_t)blockIdx.x * a.K;
  const int n = found;
  if (n <= kCap) {
    for (int i = tid; i < n; i += 256) {
      const uint64_t k = keys[i];
      int rank = 0;
      for (int m = 0; m < n; ++m) rank += keys[m] > k;
      if (rank < a.K) list[rank] = k;
    }
    for (int i = n + tid; i < a.K; i += 256) list[i] = 0;
    return;
  }
  // More than that reach it (long runs of equal logits): the best below the last, `count` times, from memory (to
  // serve from the registers as well, these rounds took 60 more of them).
  uint64_t last = ~0ull;
  for (int i = 0; i < a.K; ++i) {
    uint64_t best = 0;
#pragma unroll 1
    for (int j = 0; j < NV; ++j) {
      i32x4 u = v[0];  // a row of less than a vector
      if (a.V >= kVec) {
        u = load_loose(x + token_of(j));
        if (last_chunk) mask_vector(j, u);
      } else if (j > 0) {
        break;
      }
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        const float y = element(u, e, E());
        const uint64_t k = y > -INFINITY ? list_key(y, token_of(j) + e) : 0;
        if (k < last && k > best) best = k;
      }
    }
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const uint64_t k = __shfl_xor((unsigned long long)best, off, 64);
      best = k > best ? k : best;
    }
    __syncthreads();  // the last round's are read
    if ((tid & 63) == 0) round_best[wave] = best;
    __syncthreads();
#pragma unroll
    for (int m = 0; m < 4; ++m) best = round_best[m] > best ? round_best[m] : best;
    if (tid == 0) list[i] = best;
    last = best;
  }
}

// A continuation of the request: 64-bit score and flat place beam * V + token (a place of -1: none).
struct Choice {
  double score;
  int64_t place;
};
__device__ __forceinline__ bool before(const Choice& p, const Choice& q) {
  return p.score > q.score || (p.score == q.score && p.place < q.place);
}

constexpr int kBeamLanes = 256 / kMaxBeams;  // threads of a beam while sums are joined

__global__ __launch_bounds__(256) void beam_merge_kernel(const SelectArgs a) {
  // A continuation's score is (logit - maximum) + (score - log of the sum), not through the sum of the last two: of large
  // logits that would leave none of the score.
  __shared__ double base[kMaxBeams];  // score - log of the sum of exp(x - maximum)
  __shared__ float row_max[kMaxBeams];
  __shared__ int state[kMaxBeams];    // 0: no continuation, 1: by its lists, 2: ended
  __shared__ float thread_best[256];
  __shared__ int reaching[kCap];      // lists whose best reaches the limit
  __shared__ double held_score[kCap];
  __shared__ int64_t held_place[kCap];
  __shared__ int reached, found;
  __shared__ int64_t chosen[kMaxCount];
  const int tid = threadIdx.x;
  const int r = blockIdx.x;
  const Choice none = {-INFINITY, INT64_MAX};
  const int lists = a.W * a.chunks;
  const uint64_t* const all = a.lists + (int64_t)r * lists * a.K;
  // The best of the first lists, the scores and the pieces' sums: one round trip for all.
  constexpr int kHeads = 4;
  uint64_t head[kHeads];
#pragma unroll
  for (int i = 0; i < kHeads; ++i) head[i] = all[(int64_t)min(tid + 256 * i, lists - 1) * a.K];
  {
    const int w = min(tid / kBeamLanes, a.W - 1), lane = tid % kBeamLanes;
    const float score = a.scores[r * a.s_sr + w * a.s_sw];
    const bool ended = a.finished != nullptr && a.finished[r * a.f_sr + w * a.f_sw] != 0;
    const f32x2* const sums = a.sums + ((int64_t)r * a.W + w) * a.chunks;
    // not written for a beam that is not read: what stands there then is not used
    float m = -INFINITY;
    for (int c = lane; c < a.chunks; c += kBeamLanes) m = fmaxf(m, sums[c][0]);
#pragma unroll
    for (int off = 1; off < kBeamLanes; off <<= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
    double s = 0.0;
    for (int c = lane; c < a.chunks; c += kBeamLanes) {
      const f32x2 ms = sums[c];
      s += ms[0] == -INFINITY && ms[1] == 0.f ? 0.0 : (double)ms[1] * (double)fast_exp2((ms[0] - m) * kLog2e);  // 1 for the largest piece
    }
#pragma unroll
    for (int off = 1; off < kBeamLanes; off <<= 1) s += __shfl_xor(s, off, 64);
    const double log_sum = log(s);
    const bool live = fabsf(score) < INFINITY;
    if (lane == 0 && tid / kBeamLanes < a.W) {
      base[w] = ended ? (double)score : (double)score - log_sum;
      row_max[w] = m;
      state[w] = !live ? 0 : ended ? 2 : fabsf(m) < INFINITY && fabs(log_sum) < INFINITY ? 1 : 0;
    }
  }
  if (tid == 0) reached = found = 0;
  __syncthreads();
  auto choice = [&](int list, int i, uint64_t k) __attribute__((always_inline)) {  // entry i of a list, key k
    const int w = list / a.chunks;
    if (state[w] == 2) return list == w * a.chunks && i == 0 ? Choice{base[w], (int64_t)w * a.V + a.end} : none;
    if (state[w] == 0 || k == 0) return none;
    return Choice{base[w] + ((double)key_value(k) - (double)row_max[w]), (int64_t)w * a.V + key_token(k)};
  };
  auto entry = [&](int list, int i) __attribute__((always_inline)) {
    return choice(list, i, all[(int64_t)list * a.K + i]);
  };
  // At least `count` continuations reach the count-th largest of 64 groups' best; rounding to fp32 keeps the order.
  float best = -INFINITY;
#pragma unroll
  for (int i = 0; i < kHeads; ++i)
    if (tid + 256 * i < lists) best = fmaxf(best, (float)choice(tid + 256 * i, 0, head[i]).score);
  for (int l = tid + 256 * kHeads; l < lists; l += 256) best = fmaxf(best, (float)entry(l, 0).score);
  thread_best[tid] = best;
  __syncthreads();
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < 4; ++i) top = fmaxf(top, thread_best[(tid & 63) + 64 * i]);
  const uint32_t reach = wave_kth<0>(order_code(top), a.K);
  const float limit = order_value(reach);
  auto reaches = [&](const Choice& c) __attribute__((always_inline)) { return c.place != none.place && (float)c.score >= limit; };
  auto note = [&](int list) __attribute__((always_inline)) {
    const int n = __hip_atomic_fetch_add(&reached, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    if (n < kCap) reaching[n] = list;
  };
#pragma unroll
  for (int i = 0; i < kHeads; ++i)
    if (tid + 256 * i < lists && reaches(choice(tid + 256 * i, 0, head[i]))) note(tid + 256 * i);
  for (int l = tid + 256 * kHeads; l < lists; l += 256)
    if (reaches(entry(l, 0))) note(l);
  __syncthreads();
  const int pairs = min(reached, kCap) * a.K;
  for (int p = tid; p < pairs; p += 256) {
    const Choice c = entry(reaching[p / a.K], p % a.K);
    if (!reaches(c)) continue;
    const int n = __hip_atomic_fetch_add(&found, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    if (n < kCap) {
      held_score[n] = c.score;
      held_place[n] = c.place;
    }
  }
  __syncthreads();
  auto put = [&](int i, double score, int64_t place) __attribute__((always_inline)) {
    const int w = (int)(place / a.V), token = (int)(place - (int64_t)w * a.V);
    const int64_t at = (int64_t)r * a.K + i;
    chosen[i] = place;
    a.out_scores[at] = (float)score;
    a.out_tokens[at] = token;
    a.out_rows[at] = r * a.W + w;
    if (a.out_finished != nullptr)
      a.out_finished[at] = (a.finished != nullptr && a.finished[r * a.f_sr + w * a.f_sw] != 0) || token == a.end;
  };
  int n = found;
  if (n <= kCap && reached <= kCap) {
    for (int i = tid; i < n; i += 256) {
      const Choice c = {held_score[i], held_place[i]};
      int rank = 0;
      for (int m = 0; m < n; ++m) rank += before({held_score[m], held_place[m]}, c);
      if (rank < a.K) put(rank, c.score, c.place);
    }
    n = min(n, a.K);
  } else {
    // More than that: the best after the last, `count` times.
    Choice last = {INFINITY, -1};
    for (n = 0; n < a.K; ++n) {
      Choice next = none;
      for (int l = tid; l < lists; l += 256)
        for (int i = 0; i < a.K; ++i) {
          const Choice c = entry(l, i);
          if (c.place == none.place) break;
          if (!before(last, c)) continue;
          if (before(c, next)) next = c;
          break;
        }
      __syncthreads();  // the last round's are read
      held_score[tid] = next.score;
      held_place[tid] = next.place;
      __syncthreads();
      for (int m = 0; m < 256; ++m) {
        const Choice c = {held_score[m], held_place[m]};
        if (before(c, next)) next = c;
      }
      if (next.place == none.place) break;
      if (tid == 0) put(n, next.score, next.place);
      last = next;
    }
  }
  if (n >= a.K) return;
  // All continuations there are have been chosen: the lowest of the other places.
  __syncthreads();
  if (tid != 0) return;
  int64_t place = 0;
  for (int i = n; i < a.K; ++i, ++place) {
    for (int m = 0; m < n; ++m)
      if (chosen[m] == place) {
        ++place;
        m = -1;
      }
    put(i, -INFINITY, place);
  }
}

// ---------------------------------------------------------------- reordering

struct ReorderArgs {
  char* data[MIMIR_REORDER_TENSORS];
  int64_t stride[MIMIR_REORDER_TENSORS];
  void* lengths;
  const void* source;
  int64_t position_bytes;
  int rows, group, max_length, chunks;
  int idx64, src64;
  int past;  // rows are stored past the caches
};
__device__ __forceinline__ int64_t index_at(const void* p, int64_t i, int idx64) {
  return idx64 ? ((const int64_t*)p)[i] : (int64_t)((const int32_t*)p)[i];
}
// The source of row r0 + w within its group, w itself where the given one lies outside.
__device__ __forceinline__ int source_of(const ReorderArgs& a, int r0, int w) {
  const int64_t s = index_at(a.source, r0 + w, a.src64) - r0;
  return s >= 0 && s < a.group ? (int)s : w;
}

// Of tensors that hold more than the 256 MiB in front of memory, rows are stored past the caches: the attention that reads them
// next would not find them there.  16 requests of 8 beams, two layers (512 MiB, 317 MB moved): 72.3 us without, 64.9 with it.
constexpr int64_t kPastBytes = (int64_t)256 << 20;

// Bytes of a row that a workgroup moves: 16 loads of 16 bytes a thread over the rows of a group.
constexpr int reorder_chunk(int group) { return 4096 * (group <= 4 ? 4 : group <= 8 ? 2 : 1); }

template <int kGroup>
__global__ __launch_bounds__(256) void reorder_rows_kernel(const ReorderArgs a) {
  const int tid = threadIdx.x, w = tid & 63;
  const int g = blockIdx.x / a.chunks, chunk = blockIdx.x - g * a.chunks;
  const int r0 = g * a.group;
  int from = w, take = 0;  // lane w: the source of row w, and the positions it takes from it (0: it stays)
  if (w < a.group) {
    from = source_of(a, r0, w);
    const int64_t length = index_at(a.lengths, r0 + from, a.idx64);
    take = from == w || length < 0 ? 0 : (int)min(length, (int64_t)a.max_length);
  }
  // Whole buffers of what a row takes of this chunk, so that no load waits for another's condition: past
  // the end nothing is read, and stores are dropped.
  const int64_t first = (int64_t)chunk * reorder_chunk(kGroup), stride = a.stride[blockIdx.y];
  char* const base = a.data[blockIdx.y] + r0 * stride + first;
  auto rest = [&](int i) __attribute__((always_inline)) {
    const int64_t n = __builtin_amdgcn_readlane(take, i) * a.position_bytes - first;
    return (uint32_t)max(min(n, (int64_t)reorder_chunk(kGroup)), (int64_t)0);
  };
  constexpr int kVecs = reorder_chunk(kGroup) / 4096;
  i32x4 v[kGroup][kVecs];
#pragma unroll
  for (int i = 0; i < kGroup; ++i) {
    const __amdgpu_buffer_rsrc_t r = make_rsrc(base + __builtin_amdgcn_readlane(from, i) * stride, rest(i));
#pragma unroll
    for (int j = 0; j < kVecs; ++j) v[i][j] = buf_load16(r, (uint32_t)(j * 4096 + tid * 16));
  }
#pragma unroll
  for (int i = 0; i < kGroup; ++i) {
    const __amdgpu_buffer_rsrc_t r = make_rsrc(base + i * stride, rest(i));
    if (a.past) {
#pragma unroll
      for (int j = 0; j < kVecs; ++j) __builtin_amdgcn_raw_buffer_store_b128(v[i][j], r, j * 4096 + tid * 16, 0, 2);
    } else {
#pragma unroll
      for (int j = 0; j < kVecs; ++j) __builtin_amdgcn_raw_buffer_store_b128(v[i][j], r, j * 4096 + tid * 16, 0, 0);
    }
  }
}

// A wave per group: every lane reads its source's length before one writes.
__global__ __launch_bounds__(64) void reorder_lengths_kernel(const ReorderArgs a) {
  const int r0 = blockIdx.x * a.group, w = threadIdx.x;
  if (w >= a.group) return;
  const int64_t n = index_at(a.lengths, r0 + source_of(a, r0, w), a.idx64);
  __builtin_amdgcn_wave_barrier();
  if (a.idx64)
    ((int64_t*)a.lengths)[r0 + w] = n;
  else
    ((int32_t*)a.lengths)[r0 + w] = (int32_t)n;
}

// By name: of several instantiations launched below, this toolchain drops host stubs.
template __global__ void beam_rows_kernel<bf16_t, 8>(const SelectArgs);
template __global__ void beam_rows_kernel<bf16_t, 2>(const SelectArgs);
template __global__ void beam_rows_kernel<float, 8>(const SelectArgs);
template __global__ void beam_rows_kernel<float, 2>(const SelectArgs);
template __global__ void reorder_rows_kernel<4>(const ReorderArgs);
template __global__ void reorder_rows_kernel<8>(const ReorderArgs);
template __global__ void reorder_rows_kernel<16>(const ReorderArgs);
template __global__ void reorder_rows_kernel<32>(const ReorderArgs);

// 16-byte vectors a thread of beam_rows_kernel holds: eight, or two where eight leave CUs without work.
struct Pieces {
  int vectors, chunks;
};
Pieces pieces(const MimirBeamSelectParams& p) {
  const int vec = p.dtype == MIMIR_DTYPE_BFLOAT16 ? 8 : 4;
  const int64_t rows = (int64_t)p.requests * p.beams;
  auto cut = [&](int n) { return (int)(((int64_t)p.vocab + 256 * n * vec - 1) / (256 * n * vec)); };
  return rows * cut(8) >= 512 ? Pieces{8, cut(8)} : Pieces{2, cut(2)};
}

size_t sums_bytes(const MimirBeamSelectParams& p, int chunks) {
  return ((size_t)p.requests * (size_t)p.beams * (size_t)chunks * sizeof(f32x2) + 15) & ~(size_t)15;
}
bool select_sizes(const MimirBeamSelectParams* p) {
  return p != nullptr && p->requests >= 0 && p->beams >= 1 && p->beams <= kMaxBeams && p->vocab >= 1 && p->vocab < (1 << 30) &&
         p->count >= 1 && p->count <= kMaxCount && p->count <= (int64_t)p->beams * p->vocab &&
         (int64_t)p->requests * p->beams <= 0x7fffffff;
}

}  // namespace
}  // namespace mimir

extern "C" size_t mimir_prefixlm_beam_select_workspace_bytes(const MimirBeamSelectParams* p) {
  using namespace mimir;
  if (!select_sizes(p)) return 0;
  const int chunks = pieces(*p).chunks;
  return sums_bytes(*p, chunks) + (size_t)p->requests * (size_t)p->beams * (size_t)chunks * (size_t)p->count * sizeof(uint64_t);
}

extern "C" int mimir_prefixlm_beam_select(const MimirBeamSelectParams* p, void* stream) {
  using namespace mimir;
  fail_with(MIMIR_OK, "");
  if (p == nullptr) return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "params is NULL");
  if (p->dtype != MIMIR_DTYPE_FLOAT32 && p->dtype != MIMIR_DTYPE_BFLOAT16)
    return fail_with(MIMIR_ERR_UNSUPPORTED_DTYPE, "beam selection supports float32 and bfloat16 logits only (dtype code " +
                                                      std::to_string(p->dtype) + ")");
  if (!select_sizes(p))
    return fail_with(MIMIR_ERR_UNSUPPORTED_SHAPE, "beam selection of " + std::to_string(p->count) + " among " + std::to_string(p->beams) +
                                                      " beams and " + std::to_string(p->vocab) + " tokens: at most " + std::to_string(kMaxCount) +
                                                      " of at most " + std::to_string(kMaxBeams) + " beams and 2^30 - 1 tokens");
  if (p->end_token >= p->vocab || (p->finished != nullptr && p->end_token < 0))
    return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "end_token " + std::to_string(p->end_token) + " is not one of " + std::to_string(p->vocab) + " tokens");
  if (p->requests == 0) return MIMIR_OK;
  if (p->logits == nullptr || p->scores == nullptr || p->out_scores == nullptr || p->out_tokens == nullptr || p->out_rows == nullptr)
    return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "beam selection tensor pointer is NULL");
  const bool bf16 = p->dtype == MIMIR_DTYPE_BFLOAT16;
  if ((uintptr_t)p->logits % (bf16 ? 2 : 4) != 0) return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "logits must be aligned to their elements");
  if (p->workspace == nullptr || (uintptr_t)p->workspace % 16 != 0 || p->workspace_bytes < mimir_prefixlm_beam_select_workspace_bytes(p))
    return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "beam selection needs a workspace of " +
                                                     std::to_string(mimir_prefixlm_beam_select_workspace_bytes(p)) + " bytes aligned to 16");
  const Pieces cut = pieces(*p);
  const int64_t blocks = (int64_t)p->requests * p->beams * cut.chunks;
  if (blocks > kMaxGroups) return fail_with(MIMIR_ERR_UNSUPPORTED_SHAPE, "too many logits for one launch");
  SelectArgs a = {};
  a.logits = p->logits;
  a.scores = p->scores;
  a.finished = p->finished;
  a.out_scores = p->out_scores;
  a.out_tokens = p->out_tokens;
  a.out_rows = p->out_rows;
  a.out_finished = p->out_finished;
  a.l_sr = p->logits_stride_request; a.l_sw = p->logits_stride_beam;
  a.s_sr = p->scores_stride_request; a.s_sw = p->scores_stride_beam;
  a.f_sr = p->finished_stride_request; a.f_sw = p->finished_stride_beam;
  a.R = p->requests; a.W = p->beams; a.V = p->vocab; a.K = p->count;
  a.end = p->end_token;
  a.chunks = cut.chunks;
  a.sums = (f32x2*)p->workspace;
  a.lists = (uint64_t*)((char*)p->workspace + sums_bytes(*p, cut.chunks));
  const hipStream_t s = (hipStream_t)stream;
  const dim3 grid((unsigned)blocks), threads(256);
  if (bf16 && cut.vectors == 8) hipLaunchKernelGGL((beam_rows_kernel<bf16_t, 8>), grid, threads, 0, s, a);
  else if (bf16) hipLaunchKernelGGL((beam_rows_kernel<bf16_t, 2>), grid, threads, 0, s, a);
  else if (cut.vectors == 8) hipLaunchKernelGGL((beam_rows_kernel<float, 8>), grid, threads, 0, s, a);
  else hipLaunchKernelGGL((beam_rows_kernel<float, 2>), grid, threads, 0, s, a);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess) {
    hipLaunchKernelGGL(beam_merge_kernel, dim3((unsigned)p->requests), threads, 0, s, a);
    e = hipGetLastError();
  }
  return e == hipSuccess ? MIMIR_OK : fail_with(MIMIR_ERR_HIP, std::string("beam selection launch: ") + hipGetErrorString(e));
}

extern "C" int mimir_prefixlm_reorder_rows(const MimirReorderParams* p, void* stream) {
  using namespace mimir;
  fail_with(MIMIR_OK, "");
  if (p == nullptr) return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "params is NULL");
  if (p->rows < 0 || p->max_length < 0 || p->count < 0 || p->count > MIMIR_REORDER_TENSORS)
    return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "negative size, or more than " + std::to_string(MIMIR_REORDER_TENSORS) + " tensors a call");
  if (p->group < 1 || p->group > kMaxBeams || p->rows % p->group != 0)
    return fail_with(MIMIR_ERR_UNSUPPORTED_SHAPE, std::to_string(p->rows) + " rows are no groups of " + std::to_string(p->group) + " (at most " +
                                                      std::to_string(kMaxBeams) + ")");
  if (p->position_bytes <= 0 || p->position_bytes % 16 != 0 || p->position_bytes > (1 << 24))
    return fail_with(MIMIR_ERR_UNSUPPORTED_SHAPE, "a position of " + std::to_string(p->position_bytes) + " bytes is not a multiple of 16 up to 2^24");
  if (p->rows == 0) return MIMIR_OK;
  if (p->lengths == nullptr || p->source == nullptr) return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "lengths or source is NULL");
  const int64_t row_bytes = p->max_length * p->position_bytes;
  ReorderArgs a = {};
  for (int i = 0; i < p->count; ++i) {
    if (p->data[i] == nullptr && row_bytes > 0) return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "cache tensor pointer is NULL");
    if ((uintptr_t)p->data[i] % 16 != 0 || p->stride[i] % 16 != 0)
      return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "cache rows must be aligned to 16 bytes");
    if (p->rows > 1 && p->stride[i] < row_bytes) return fail_with(MIMIR_ERR_UNSUPPORTED_SHAPE, "cache rows must not overlap");
    a.data[i] = (char*)p->data[i];
    a.stride[i] = p->stride[i];
    auto region = [&](int j) { return Region{p->data[j], row_bytes, {p->rows, 1, 1}, {p->stride[j], 0, 0}}; };
    for (int j = 0; j < i && row_bytes > 0; ++j)
      if (overlap_each_other(region(i), region(j))) return fail_with(MIMIR_ERR_UNSUPPORTED_SHAPE, "cache tensors must not share memory");
  }
  a.lengths = p->lengths;
  a.source = p->source;
  a.position_bytes = p->position_bytes;
  a.rows = p->rows; a.group = p->group; a.max_length = p->max_length;
  a.idx64 = p->index_int64 != 0; a.src64 = p->source_int64 != 0;
  const int64_t groups = p->rows / p->group, chunk_bytes = reorder_chunk(p->group), chunks = (row_bytes + chunk_bytes - 1) / chunk_bytes;
  // workgroups of 256 threads, and for the lengths one of 64 a group
  if (groups * chunks > kMaxGroups || chunks > 0x7fffffff || groups > 0xffffffffll / 64) return fail_with(MIMIR_ERR_UNSUPPORTED_SHAPE, "too many positions for one launch");
  a.chunks = (int)chunks;
  a.past = (int64_t)p->count * row_bytes >= kPastBytes / p->rows;
  const hipStream_t s = (hipStream_t)stream;
  hipError_t e = hipSuccess;
  if (p->count > 0 && chunks > 0) {
    const dim3 grid((unsigned)(groups * chunks), (unsigned)p->count), threads(256);
    if (p->group <= 4) hipLaunchKernelGGL(reorder_rows_kernel<4>, grid, threads, 0, s, a);
    else if (p->group <= 8) hipLaunchKernelGGL(reorder_rows_kernel<8>, grid, threads, 0, s, a);
    else if (p->group <= 16) hipLaunchKernelGGL(reorder_rows_kernel<16>, grid, threads, 0, s, a);
    else hipLaunchKernelGGL(reorder_rows_kernel<32>, grid, threads, 0, s, a);
    e = hipGetLastError();
  }
  if (e == hipSuccess && p->update_lengths) {
    hipLaunchKernelGGL(reorder_lengths_kernel, dim3((unsigned)groups), dim3(64), 0, s, a);
    e = hipGetLastError();
  }
  return e == hipSuccess ? MIMIR_OK : fail_with(MIMIR_ERR_HIP, std::string("row reordering launch: ") + hipGetErrorString(e));
}
