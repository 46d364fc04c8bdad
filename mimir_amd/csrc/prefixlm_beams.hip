// Beam search: the best continuations over a request's beams and the vocabulary, and the rows of
// static caches in the order of the chosen beams.
//
// Selection.  Of logits x[r, w, :], scores s[r, w] and lse = log sum exp x, the `count` largest
// s + x - lse of a request, ties to the lowest (beam, token).  Bound by reading the logits once: one
// workgroup of beam_rows_kernel per piece of a row keeps the piece in registers, and from there
//   * sums exp(x - max) in fp32, a few adds a lane;
//   * finds a threshold that at least `count` elements reach: the count-th largest of a wave's lane maxima,
//     bit by bit with ballots (16 steps for bf16), and the largest of that over the waves;
//   * ranks the few elements that reach it and stores the best `count`, in order.
// Within a row larger logits are larger scores, so this needs no lse.  beam_merge_kernel, a workgroup per
// request, joins the pieces' sums in 64 bits, forms the scores of the stored elements in 64 bits (beams
// meet there, whose scores may lie closer than fp32 tells apart), and ranks those that reach the count-th
// largest of its threads' best.  Masked logits, ended beams and rows of ties need no case of their own but
// for more candidates than the lists hold, which fall back to `count` rounds of a maximum.
//
// Reordering.  Rows of a group take each other's place, so every row is read before any is written: a
// thread owns 16 bytes of the same place in all rows of a group, loads what moves and then stores it.
// Bound by copying.
#include <algorithm>
#include <cmath>

#include "prefixlm_common.h"
#include "strided_overlap.h"

namespace mimir {
namespace {

constexpr int kMaxBeams = 32, kMaxCount = 64;
constexpr int kCap = 1024;  // candidates ranked at once

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

template <typename F>
__device__ __forceinline__ float wave_reduce(float x, F&& f) {
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) x = f(x, __shfl_xor(x, off, 64));
  return x;
}

template <typename E, int N>
struct __attribute__((packed, aligned(sizeof(E)))) Loose {  // N elements at any address of theirs
  E v[N];
};

template <typename E, int NV>
__global__ __launch_bounds__(256) void beam_rows_kernel(const SelectArgs a) {
  constexpr int kVec = 16 / sizeof(E);
  __shared__ uint64_t keys[kCap];
  __shared__ float wave_max[4], wave_sum[4];
  __shared__ uint32_t wave_code[4];
  __shared__ int found;
  __shared__ uint64_t round_best[4];
  const int tid = threadIdx.x, wave = tid >> 6;
  const int row = blockIdx.x / a.chunks, chunk = blockIdx.x - row * a.chunks;
  const int r = row / a.W, w = row - r * a.W;
  const float score = a.scores[r * a.s_sr + w * a.s_sw];
  const bool ended = a.finished != nullptr && a.finished[r * a.f_sr + w * a.f_sw] != 0;
  if (ended || !(fabsf(score) < INFINITY)) return;  // the merge does not read this row's pieces
  const E* const x = (const E*)a.logits + r * a.l_sr + w * a.l_sw;
  const int first = chunk * (256 * NV * kVec) + tid * kVec;
  float v[NV][kVec];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int at = first + j * 256 * kVec;
    if (at + kVec <= a.V) {
      const Loose<E, kVec> in = *(const Loose<E, kVec>*)(x + at);
#pragma unroll
      for (int e = 0; e < kVec; ++e) v[j][e] = (float)in.v[e];
    } else {
#pragma unroll
      for (int e = 0; e < kVec; ++e) v[j][e] = at + e < a.V ? (float)x[at + e] : -INFINITY;
    }
  }
  float most[NV], top = -INFINITY;  // NaN is left out here and comes back in the sum
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    most[j] = -INFINITY;
#pragma unroll
    for (int e = 0; e < kVec; ++e) most[j] = fmaxf(most[j], v[j][e]);
    top = fmaxf(top, most[j]);
  }
  const float wtop = wave_reduce(top, [](float p, float q) { return fmaxf(p, q); });
  // The count-th largest code of the wave's lane maxima: at least `count` elements reach it.
  const uint32_t code = order_code(top);
  uint32_t reach = 0;
#pragma unroll
  for (int bit = 31; bit >= (sizeof(E) == 2 ? 16 : 0); --bit) {
    const uint32_t next = reach | 1u << bit;
    if (__builtin_popcountll(__builtin_amdgcn_ballot_w64(code >= next)) >= a.K) reach = next;
  }
  if (sizeof(E) == 2 && reach >> 31 == 0) reach |= 0xffffu;  // a negative bf16's code ends in ones
  if ((tid & 63) == 0) {
    wave_max[wave] = wtop;
    wave_code[wave] = reach;
  }
  if (tid == 0) found = 0;
  __syncthreads();
  const float block_top = fmaxf(fmaxf(wave_max[0], wave_max[1]), fmaxf(wave_max[2], wave_max[3]));
  const float base = block_top == -INFINITY ? 0.f : block_top;
  float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int e = 0; e < kVec; ++e) part[e % 4] += fast_exp2((v[j][e] - base) * kLog2e);
  const float sum = wave_reduce((part[0] + part[1]) + (part[2] + part[3]), [](float p, float q) { return p + q; });
  if ((tid & 63) == 0) wave_sum[wave] = sum;
  const float limit = order_value(max(max(wave_code[0], wave_code[1]), max(wave_code[2], wave_code[3])));
#pragma unroll
  for (int j = 0; j < NV; ++j)
    if (most[j] >= limit) {
#pragma unroll
      for (int e = 0; e < kVec; ++e)
        if (v[j][e] >= limit && v[j][e] > -INFINITY) {
          const int n = __hip_atomic_fetch_add(&found, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
          if (n < kCap) keys[n] = list_key(v[j][e], first + j * 256 * kVec + e);
        }
    }
  __syncthreads();
  if (tid == 0) a.sums[blockIdx.x] = f32x2{block_top, (wave_sum[0] + wave_sum[1]) + (wave_sum[2] + wave_sum[3])};
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
  // More than that reach it (long runs of equal logits): the best below the last, `count` times.
  uint64_t last = ~0ull;
  for (int i = 0; i < a.K; ++i) {
    uint64_t best = 0;
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (most[j] >= limit) {
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          const uint64_t k = v[j][e] > -INFINITY ? list_key(v[j][e], first + j * 256 * kVec + e) : 0;
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

__global__ __launch_bounds__(256) void beam_merge_kernel(const SelectArgs a) {
  __shared__ double base[kMaxBeams];  // score - lse
  __shared__ int state[kMaxBeams];    // 0: no continuation, 1: by its lists, 2: ended
  __shared__ double held_score[kCap];
  __shared__ int64_t held_place[kCap];
  __shared__ double limit_score;
  __shared__ int64_t limit_place;
  __shared__ int found;
  __shared__ int64_t chosen[kMaxCount];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int r = blockIdx.x;
  const Choice none = {-INFINITY, INT64_MAX};
  for (int w = wave; w < a.W; w += 4) {
    const float score = a.scores[r * a.s_sr + w * a.s_sw];
    const bool ended = a.finished != nullptr && a.finished[r * a.f_sr + w * a.f_sw] != 0;
    const bool live = fabsf(score) < INFINITY;
    double lse = 0.0;
    if (live && !ended) {
      const f32x2* const sums = a.sums + ((int64_t)r * a.W + w) * a.chunks;
      float m = -INFINITY;
      for (int c = lane; c < a.chunks; c += 64) m = fmaxf(m, sums[c][0]);
      m = wave_reduce(m, [](float p, float q) { return fmaxf(p, q); });
      double s = 0.0;
      for (int c = lane; c < a.chunks; c += 64) {
        const f32x2 ms = sums[c];
        s += ms[0] == -INFINITY && ms[1] == 0.f ? 0.0 : (double)ms[1] * exp((double)ms[0] - (double)m);
      }
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) s += __shfl_xor(s, off, 64);
      lse = (double)m + log(s);
    }
    if (lane == 0) {
      base[w] = (double)score - lse;
      state[w] = !live || !(fabs(lse) < INFINITY) ? 0 : ended ? 2 : 1;
    }
  }
  if (tid == 0) found = 0;
  __syncthreads();
  const int lists = a.W * a.chunks;
  const uint64_t* const all = a.lists + (int64_t)r * lists * a.K;
  auto choice = [&](int list, int i) __attribute__((always_inline)) {  // entry i of a list, none past its end
    const int w = list / a.chunks;
    if (state[w] == 2) return list == w * a.chunks && i == 0 ? Choice{base[w], (int64_t)w * a.V + a.end} : none;
    if (state[w] == 0) return none;
    const uint64_t k = all[(int64_t)list * a.K + i];
    return k == 0 ? none : Choice{base[w] + (double)key_value(k), (int64_t)w * a.V + key_token(k)};
  };
  Choice best = none;
  for (int l = tid; l < lists; l += 256) {
    const Choice c = choice(l, 0);
    if (before(c, best)) best = c;
  }
  // The count-th best of the threads' best (or the last): what comes before none of them is not chosen.
  held_score[tid] = best.score;
  held_place[tid] = best.place;
  if (tid == 0) {
    limit_score = -INFINITY;
    limit_place = INT64_MAX - 1;
  }
  __syncthreads();
  if (best.place != none.place) {
    int rank = 0;
    for (int m = 0; m < 256; ++m) rank += before({held_score[m], held_place[m]}, best);
    if (rank == a.K - 1) {
      limit_score = best.score;
      limit_place = best.place;
    }
  }
  __syncthreads();
  const Choice limit = {limit_score, limit_place};
  for (int l = tid; l < lists; l += 256)
    for (int i = 0; i < a.K; ++i) {
      const Choice c = choice(l, i);
      if (c.place == none.place || before(limit, c)) break;
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
  if (n <= kCap) {
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
      best = none;
      for (int l = tid; l < lists; l += 256)
        for (int i = 0; i < a.K; ++i) {
          const Choice c = choice(l, i);
          if (c.place == none.place) break;
          if (!before(last, c)) continue;
          if (before(c, best)) best = c;
          break;
        }
      __syncthreads();  // the last round's are read
      held_score[tid] = best.score;
      held_place[tid] = best.place;
      __syncthreads();
      for (int m = 0; m < 256; ++m) {
        const Choice c = {held_score[m], held_place[m]};
        if (before(c, best)) best = c;
      }
      if (best.place == none.place) break;
      if (tid == 0) put(n, best.score, best.place);
      last = best;
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
};
__device__ __forceinline__ int64_t index_at(const void* p, int64_t i, int idx64) {
  return idx64 ? ((const int64_t*)p)[i] : (int64_t)((const int32_t*)p)[i];
}
// The source of row r0 + w within its group, w itself where the given one lies outside.
__device__ __forceinline__ int source_of(const ReorderArgs& a, int r0, int w) {
  const int64_t s = index_at(a.source, r0 + w, a.src64) - r0;
  return s >= 0 && s < a.group ? (int)s : w;
}

template <int kGroup>
__global__ __launch_bounds__(256) void reorder_rows_kernel(const ReorderArgs a) {
  __shared__ int from[kGroup];
  __shared__ int64_t bytes[kGroup];  // that row w takes from its source, 0: it stays
  const int tid = threadIdx.x;
  const int g = blockIdx.x / a.chunks, chunk = blockIdx.x - g * a.chunks;
  const int r0 = g * a.group;
  if (tid < kGroup) {
    int s = tid;
    int64_t n = 0;
    if (tid < a.group) {
      s = source_of(a, r0, tid);
      const int64_t length = index_at(a.lengths, r0 + s, a.idx64);
      n = s == tid || length < 0 ? 0 : min(length, (int64_t)a.max_length) * a.position_bytes;
    }
    from[tid] = s;
    bytes[tid] = n;
  }
  __syncthreads();
  const int64_t at = ((int64_t)chunk * 256 + tid) * 16;
  char* const base = a.data[blockIdx.y] + r0 * a.stride[blockIdx.y] + at;
  const int64_t stride = a.stride[blockIdx.y];
  i32x4 v[kGroup];
#pragma unroll
  for (int w = 0; w < kGroup; ++w)
    if (at < bytes[w]) v[w] = *(const i32x4*)(base + from[w] * stride);
#pragma unroll
  for (int w = 0; w < kGroup; ++w)
    if (at < bytes[w]) *(i32x4*)(base + w * stride) = v[w];
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
  const int64_t groups = p->rows / p->group, chunks = (row_bytes + 4095) / 4096;
  if (groups * chunks > kMaxGroups || chunks > 0x7fffffff) return fail_with(MIMIR_ERR_UNSUPPORTED_SHAPE, "too many positions for one launch");
  a.chunks = (int)chunks;
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
