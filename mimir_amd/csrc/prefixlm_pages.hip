// The rows of a paged cache and the pages they hold: copy, fork, compact, release and
// reserve, on the device alone.
//
// Two kinds of work.  The tables (pages of each row, rows that hold each page) are small
// integers: latency-bound scans, made deterministic by handing out free pages lowest
// first, in the order of the requests, and by counting with commutative integer
// atomics only.  The pool's data moves page by page: a copy, bound by reading and writing
// each moved byte once; its launch also writes the table rows, which the scans leave in
// the workspace.  The number of moves is known on the device only, so the copy's workgroups
// take (move, 16 KiB chunk) units in turn until the list's count ends them.
//
// Measured: 1000 pages of 4 layers, 4 heads of 128 moved (530 MB) 99 us, 5.3 TB/s, after 5.7 of planning; a
// fork of 256 rows of up to 48 pages 28 us: plan 4.1, gather 3.1, take 4.8 and the copies (79 MB) 17; each
// planning launch is 2 us and a few round trips of 0.7.
#include <algorithm>

#include "prefixlm_common.h"

namespace mimir {
int fail_with(int code, const std::string& msg);

namespace {

constexpr int kPageTokens = MIMIR_PAGE_TOKENS;
constexpr int kScan = 1024;               // threads of a scanning workgroup
constexpr int kCopyThreads = 256;
constexpr int kCopyChunk = kCopyThreads * 16 * 4;  // bytes: four 16-byte loads in flight a thread

struct Table {
  int32_t *pages, *lengths, *counts, *missing;
  int64_t stride;
  int rows, width, num_pages;
  __device__ __forceinline__ bool page_ok(int p) const { return p >= 0 && p < num_pages; }
  __device__ __forceinline__ bool row_ok(int r) const { return r >= 0 && r < rows; }
  __device__ __forceinline__ int32_t* row(int r) const { return pages + (int64_t)r * stride; }
};

// counts change by device atomics while others of the workgroup look at them: past the L1
__device__ __forceinline__ int load_count(const int32_t* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Exclusive sum over the workgroup's kScan threads; `total` for all of them.
__device__ __forceinline__ int block_exclusive(int x, int* shared, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int incl = x;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int y = __shfl_up(incl, off, 64);
    if (lane >= off) incl += y;
  }
  __syncthreads();  // shared may still be read from the call before
  if (lane == 63) shared[wave] = incl;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kScan / 64; ++w) {
    const int n = shared[w];
    before += w < wave ? n : 0;
    total += n;
  }
  return before + incl - x;
}

// A thread's kOwn consecutive counts from page p on, as a mask of those that hold(count); pages past the
// last are left out.  Four 16-byte loads where the array allows it.
constexpr int kOwn = 16;
template <typename F>
__device__ __forceinline__ unsigned count_mask(const Table& t, int p, F&& hold) {
  unsigned mask = 0;
  if (p + kOwn <= t.num_pages && (uintptr_t)t.counts % 16 == 0) {
    i32x4 c[kOwn / 4];
#pragma unroll
    for (int e = 0; e < kOwn / 4; ++e) c[e] = ((const i32x4*)(t.counts + p))[e];
#pragma unroll
    for (int e = 0; e < kOwn; ++e) mask |= (hold(c[e / 4][e % 4]) ? 1u : 0u) << e;
  } else {
    for (int e = 0; e < kOwn && p + e < t.num_pages; ++e) mask |= (hold(t.counts[p + e]) ? 1u : 0u) << e;
  }
  return mask;
}

// The free ones of the first pages, as take_free wants them: requested early, they are there by then.
__device__ __forceinline__ unsigned first_free(const Table& t) {
  return count_mask(t, kOwn * (int)threadIdx.x, [](int c) { return c == 0; });
}
// The first `wanted` free pages, ascending, into list; returns how many there are (at most
// wanted).  They count one from here on.  One workgroup of kScan threads, and no other at the time.
__device__ __forceinline__ int take_free(const Table& t, unsigned first, int wanted, int32_t* list, int* shared) {
  int found = 0;
  for (int p0 = 0; p0 < t.num_pages && found < wanted; p0 += kOwn * kScan) {
    const int p = p0 + kOwn * (int)threadIdx.x;
    unsigned free = p0 == 0 ? first : count_mask(t, p, [](int c) { return c == 0; });
    int total;
    int at = found + block_exclusive(__popc(free), shared, total);
    for (; free != 0 && at < wanted; free &= free - 1, ++at) {
      const int page = p + __builtin_ctz(free);
      list[at] = page;
      t.counts[page] = 1;
    }
    found += total;
  }
  __threadfence_block();
  __syncthreads();
  return found < wanted ? found : wanted;
}

// ------------------------------------------------------------------ moving data

struct Pool {
  char* data[4];
  int64_t bytes[4], stride[4];
};

struct CopyArgs {
  Pool pool;
  Table table;
  const int32_t *src, *dst;  // of each move
  const int32_t* n_dev;      // number of moves, on the device; or null: n
  int n, chunks;             // chunks of a page's keys and values
  // what the launch writes beside: fork's rows (entries with kept[i]) ...
  const int32_t *rowbuf, *kept, *dst_rows, *new_len;
  int entries;
  // ... or compact's renamed pages, of those at or past used[0]
  const int32_t *map, *used;
};

__global__ __launch_bounds__(kCopyThreads) void pages_move_kernel(const CopyArgs a) {
  touch_args<sizeof(CopyArgs)>();
  const Table& t = a.table;
  const int64_t threads = (int64_t)gridDim.x * kCopyThreads, id = (int64_t)blockIdx.x * kCopyThreads + threadIdx.x;
  const int n = a.n_dev != nullptr ? *a.n_dev : a.n;
  if (a.rowbuf != nullptr) {
    for (int64_t i = id; i < (int64_t)a.entries * t.width; i += threads) {
      const int e = (int)(i / t.width), j = (int)(i - (int64_t)e * t.width);
      if (!a.kept[e]) continue;
      t.row(a.dst_rows[e])[j] = a.rowbuf[i];
      if (j == 0) t.lengths[a.dst_rows[e]] = a.new_len[e];
    }
  }
  if (a.map != nullptr) {
    const int used = *a.used;
    for (int64_t i = id; i < (int64_t)t.rows * t.width; i += threads) {
      const int r = (int)(i / t.width);
      int32_t* const at = t.row(r) + (i - (int64_t)r * t.width);
      const int p = *at;
      if (p >= used && t.page_ok(p)) *at = a.map[p];
    }
    for (int64_t m = id; m < n; m += threads) {
      t.counts[a.dst[m]] = t.counts[a.src[m]];
      t.counts[a.src[m]] = 0;
    }
  }
  const int key_chunks = (int)((a.pool.bytes[0] + kCopyChunk - 1) / kCopyChunk);
  for (int64_t u = blockIdx.x; u < (int64_t)n * a.chunks; u += gridDim.x) {
    const int m = (int)(u / a.chunks), c = (int)(u - (int64_t)m * a.chunks);
    const int from = a.src[m], to = a.dst[m];
    if (!t.page_ok(from) || !t.page_ok(to)) continue;  // uniform
    const int which = c < key_chunks ? 0 : 1;
    const int64_t at = (int64_t)(c - which * key_chunks) * kCopyChunk, bytes = a.pool.bytes[which];
    const char* const x = a.pool.data[which] + from * a.pool.stride[which];
    char* const y = a.pool.data[which] + to * a.pool.stride[which];
    i32x4 v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int64_t o = at + (e * kCopyThreads + (int)threadIdx.x) * 16;
      if (o < bytes) v[e] = __builtin_nontemporal_load((const i32x4*)(x + o));
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int64_t o = at + (e * kCopyThreads + (int)threadIdx.x) * 16;
      if (o < bytes) __builtin_nontemporal_store(v[e], (i32x4*)(y + o));
    }
    if (c == 0)
      for (int w = 2; w < 4; ++w)
        for (int64_t o = threadIdx.x; o < a.pool.bytes[w]; o += kCopyThreads)
          a.pool.data[w][to * a.pool.stride[w] + o] = a.pool.data[w][from * a.pool.stride[w] + o];
  }
}

// ------------------------------------------------------------------ fork

struct ForkArgs {
  Table t;
  const int32_t *src, *dst;
  int n;
  int32_t *last, *first;  // [rows]: the last entry for a destination, the first kept one of a source
  int32_t *kept, *new_len, *tail, *rowbuf;  // [n], rowbuf [n][width]
  int32_t *from, *to, *free;  // [n]
  int32_t* given_up;          // [1]: whether a last page that several rows hold may have been given up by all
};

// What each entry takes: kept, its length, and its last page (>= 0: an heir's; < -1: a copy of
// page -2 - tail; -1: none).  One workgroup.  The only holder's heir is known here, and then the page
// is held; one that several entries of the table name is looked at again once all have given theirs
// back (fork_heirs): a page that is copied from must not be handed out as another's destination.
__device__ __forceinline__ void fork_plan(const ForkArgs& a) {
  const Table& t = a.t;
  for (int r = threadIdx.x; r < t.rows; r += kScan) {
    a.last[r] = -1;
    a.first[r] = 0x7fffffff;
  }
  if (threadIdx.x == 0) *a.given_up = 0;
  __threadfence_block();
  __syncthreads();
  for (int i = threadIdx.x; i < a.n; i += kScan)
    if (t.row_ok(a.src[i]) && t.row_ok(a.dst[i])) atomicMax(&a.last[a.dst[i]], i);
  __syncthreads();
  for (int i = threadIdx.x; i < a.n; i += kScan) {
    const int s = a.src[i], d = a.dst[i];
    const bool kept = t.row_ok(s) && t.row_ok(d) && s != d && load_count(&a.last[d]) == i;
    a.kept[i] = kept;
    if (kept) atomicMin(&a.first[s], i);
  }
  __threadfence_block();
  __syncthreads();
  for (int i = threadIdx.x; i < a.n; i += kScan) {
    if (!a.kept[i]) continue;
    const int s = a.src[i], len = max(t.lengths[s], 0), full = len / kPageTokens;
    int tail = -1;
    if (len % kPageTokens != 0 && full < t.width && t.page_ok(t.row(s)[full])) {
      const int p = t.row(s)[full];
      const int by = load_count(&a.last[s]);  // the entry that replaces the source
      const bool replaced = by >= 0 && a.src[by] != s, alone = load_count(&t.counts[p]) == 1;
      const bool heir = replaced && alone && load_count(&a.first[s]) == i;
      tail = heir ? p : -2 - p;
      if (replaced && !alone) *a.given_up = 1;  // every writer's value
    }
    a.tail[i] = tail;
    a.new_len[i] = t.lengths[s];
  }
  __threadfence_block();
  __syncthreads();
}

// Entry i's new row into the workspace, its old pages given back and the shared ones counted.
__device__ __forceinline__ void fork_gather(const ForkArgs& a, int i, int thread, int threads) {
  const Table& t = a.t;
  if (!a.kept[i]) return;
  const int32_t *from = t.row(a.src[i]), *old = t.row(a.dst[i]);
  const int len = max(a.new_len[i], 0), full = len / kPageTokens, tail = a.tail[i];
  for (int j = thread; j < t.width; j += threads) {
    const int p = from[j], o = old[j];
    int q = -1;
    if (j < full && t.page_ok(p)) q = p;
    if (j == full && tail >= 0) q = tail;
    a.rowbuf[(int64_t)i * t.width + j] = q;
    if (t.page_ok(o)) atomicSub(&t.counts[o], 1);
    if (q >= 0) atomicAdd(&t.counts[q], 1);
  }
}

// Of last pages that no row holds any more, the first entry that would copy one takes it as it is: the lowest
// entry i leaves i - n in the page's count.  One workgroup.
__device__ __forceinline__ void fork_heirs(const ForkArgs& a) {
  const Table& t = a.t;
  auto unheld = [&](int i) { return a.kept[i] && a.tail[i] < -1 && load_count(&t.counts[-2 - a.tail[i]]) <= 0; };
  for (int i = threadIdx.x; i < a.n; i += kScan)
    if (unheld(i)) atomicMin(&t.counts[-2 - a.tail[i]], i - a.n);
  __syncthreads();
  for (int i = threadIdx.x; i < a.n; i += kScan)
    if (unheld(i) && load_count(&t.counts[-2 - a.tail[i]]) == i - a.n) {
      const int p = -2 - a.tail[i];
      atomicExch(&t.counts[p], 1);
      a.rowbuf[(int64_t)i * t.width + max(a.new_len[i], 0) / kPageTokens] = p;
      a.tail[i] = p;
    }
  __threadfence();  // counts are read through the L1 from here on
  __syncthreads();
}

// Free pages for the last pages that are copied.  One workgroup.
__device__ __forceinline__ void fork_take(const ForkArgs& a, int* shared) {
  const Table& t = a.t;
  unsigned first = first_free(t);
  if (__builtin_expect(*a.given_up != 0, 0)) {  // uniform
    fork_heirs(a);
    first = first_free(t);
  }
  int wanted = 0;
  for (int i0 = 0; i0 < a.n; i0 += kScan) {  // the rank of each request, in a.from for now
    const int i = i0 + threadIdx.x;
    const bool need = i < a.n && a.kept[i] && a.tail[i] < -1;
    int total;
    const int rank = wanted + block_exclusive(need, shared, total);
    if (i < a.n) a.from[i] = need ? rank : -1;
    wanted += total;
  }
  const int got = take_free(t, first, wanted, a.free, shared);
  if (threadIdx.x == 0 && got < wanted) atomicAdd(t.missing, wanted - got);
  for (int i = threadIdx.x; i < a.n; i += kScan) {
    const int rank = a.from[i];
    const bool copy = rank >= 0 && rank < got;
    const int page = copy ? a.free[rank] : -1;
    if (copy) a.rowbuf[(int64_t)i * t.width + max(a.new_len[i], 0) / kPageTokens] = page;
    a.from[i] = copy ? -2 - a.tail[i] : -1;
    a.to[i] = page;
  }
}

__global__ __launch_bounds__(kScan) void fork_plan_kernel(const ForkArgs a) {
  touch_args<sizeof(ForkArgs)>();
  fork_plan(a);
}
__global__ __launch_bounds__(256) void fork_gather_kernel(const ForkArgs a) {
  touch_args<sizeof(ForkArgs)>();
  fork_gather(a, blockIdx.x, threadIdx.x, 256);
}
__global__ __launch_bounds__(kScan) void fork_take_kernel(const ForkArgs a) {
  touch_args<sizeof(ForkArgs)>();
  __shared__ int shared[kScan / 64];
  fork_take(a, shared);
}

// ------------------------------------------------------------------ compact

struct CompactArgs {
  Table t;
  int32_t *used, *n_moves, *map, *from, *to;
};

__global__ __launch_bounds__(kScan) void compact_plan_kernel(const CompactArgs a) {
  touch_args<sizeof(CompactArgs)>();
  __shared__ int shared[kScan / 64];
  const Table& t = a.t;
  // the thread's pages of the first 16384, which it looks at once, and those behind them
  const unsigned first = count_mask(t, kOwn * (int)threadIdx.x, [](int c) { return c > 0; });
  int mine = __popc(first), used;
  for (int p = kOwn * (kScan + (int)threadIdx.x); p < t.num_pages; p += kOwn * kScan)
    mine += __popc(count_mask(t, p, [](int c) { return c > 0; }));
  block_exclusive(mine, shared, used);
  int holes = 0, moves = 0;
  for (int p0 = 0; p0 < t.num_pages; p0 += kOwn * kScan) {
    const int p = p0 + kOwn * (int)threadIdx.x;
    const unsigned held = p0 == 0 ? first : count_mask(t, p, [](int c) { return c > 0; });
    const int left = t.num_pages - p;
    const unsigned inside = left >= kOwn ? (1u << kOwn) - 1 : (left <= 0 ? 0u : (1u << left) - 1);
    const unsigned front = used - p >= kOwn ? (1u << kOwn) - 1 : (used <= p ? 0u : (1u << (used - p)) - 1);  // pages before `used`
    unsigned hole = inside & ~held & front, late = held & ~front;
    // a free page behind `used` stays what it is, should a row name it all the same
    for (unsigned rest = inside & ~held & ~front; rest != 0; rest &= rest - 1) a.map[p + __builtin_ctz(rest)] = p + __builtin_ctz(rest);
    int total;  // of holes in the lower half, of late pages in the upper: at most kOwn * kScan each
    const int before = block_exclusive(__popc(hole) | __popc(late) << 16, shared, total);
    for (int at = holes + (before & 0xffff); hole != 0; hole &= hole - 1) a.to[at++] = p + __builtin_ctz(hole);
    for (int at = moves + (before >> 16 & 0xffff); late != 0; late &= late - 1) a.from[at++] = p + __builtin_ctz(late);
    holes += total & 0xffff;
    moves += total >> 16 & 0xffff;
  }
  __threadfence_block();
  __syncthreads();
  // as many holes before `used` as pages in use behind it
  for (int m = threadIdx.x; m < moves; m += kScan) a.map[a.from[m]] = a.to[m];
  if (threadIdx.x == 0) {
    *a.used = used;
    *a.n_moves = moves;
  }
}

// ------------------------------------------------------------------ release and reserve

// A listed row that comes twice finds its pages gone the second time.
__global__ __launch_bounds__(256) void release_kernel(const Table t, const int32_t* list) {
  const int r = list[blockIdx.x];
  if (!t.row_ok(r)) return;
  for (int j = threadIdx.x; j < t.width; j += 256) {
    const int p = atomicExch(&t.row(r)[j], -1);
    if (t.page_ok(p)) atomicSub(&t.counts[p], 1);
  }
  if (threadIdx.x == 0) t.lengths[r] = 0;
}

struct ReserveArgs {
  Table t;
  const int32_t* new_len;
  int32_t *lack, *free, *got;  // [rows], [num_pages], [1]
};

// Places that row r should hold pages in.
__device__ __forceinline__ int reserve_until(const ReserveArgs& a, int r) {
  const int n = a.new_len[r];
  if (n <= 0) return 0;
  const int64_t pages = ((int64_t)max(a.t.lengths[r], 0) + n + kPageTokens - 1) / kPageTokens;
  return pages < a.t.width ? (int)pages : a.t.width;
}

// One wave per row: the pages it lacks.
__global__ __launch_bounds__(256) void reserve_count_kernel(const ReserveArgs a) {
  touch_args<sizeof(ReserveArgs)>();
  const int r = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (r >= a.t.rows) return;
  const int until = reserve_until(a, r);
  int lack = 0;
  for (int j = lane; j < until; j += 64) lack += !a.t.page_ok(a.t.row(r)[j]);
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) lack += __shfl_xor(lack, off, 64);
  if (lane == 0) a.lack[r] = lack;
}

// lack[r] becomes the rank of the row's first request; the free pages are listed.
__global__ __launch_bounds__(kScan) void reserve_take_kernel(const ReserveArgs a) {
  touch_args<sizeof(ReserveArgs)>();
  __shared__ int shared[kScan / 64];
  const unsigned first = first_free(a.t);
  int64_t wanted = 0;
  for (int r0 = 0; r0 < a.t.rows; r0 += kScan) {
    const int r = r0 + threadIdx.x;
    int total;
    const int rank = block_exclusive(r < a.t.rows ? a.lack[r] : 0, shared, total);
    if (r < a.t.rows) a.lack[r] = (int)(wanted + rank < 0x7fffffff ? wanted + rank : 0x7fffffff);
    wanted += total;
  }
  const int most = wanted < a.t.num_pages ? (int)wanted : a.t.num_pages;
  const int got = take_free(a.t, first, most, a.free, shared);
  if (threadIdx.x == 0) {
    *a.got = got;
    if (got < wanted) atomicAdd(a.t.missing, (int)(wanted - got));
  }
}

__global__ __launch_bounds__(256) void reserve_assign_kernel(const ReserveArgs a) {
  touch_args<sizeof(ReserveArgs)>();
  const int r = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (r >= a.t.rows) return;
  const int until = reserve_until(a, r), got = *a.got;
  int64_t rank = a.lack[r];
  for (int j0 = 0; j0 < until; j0 += 64) {
    const int j = j0 + lane;
    const bool need = j < until && !a.t.page_ok(a.t.row(r)[j]);
    const uint64_t all = __builtin_amdgcn_ballot_w64(need);
    const int64_t mine = rank + __builtin_popcountll(all & ((1ull << lane) - 1));
    if (need) a.t.row(r)[j] = mine < got ? a.free[mine] : -1;
    rank += __builtin_popcountll(all);
  }
}

// Take and assign in one launch of one workgroup, for up to kScan rows: the waves go over the rows that lack pages,
// kAtOnce of them in flight.  Or (kCounts) the count too, over all rows that ask for tokens.
template <bool kCounts>
__device__ __forceinline__ void reserve_place(const ReserveArgs& a) {
  touch_args<sizeof(ReserveArgs)>();
  constexpr int kAtOnce = 4, kWaves = kScan / 64;
  __shared__ int shared[kWaves], s_row[kScan], s_until[kScan], s_rank[kScan];
  const Table& t = a.t;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const unsigned first = first_free(t);
  const int until = tid < t.rows ? reserve_until(a, tid) : 0;
  const int lack = tid >= t.rows ? 0 : (kCounts ? until : a.lack[tid]);
  int listed, wanted;
  const int place = block_exclusive(lack > 0, shared, listed);
  if constexpr (!kCounts) {
    const int rank = block_exclusive(lack, shared, wanted);
    if (lack > 0) s_rank[place] = rank;
  }
  if (lack > 0) {
    s_row[place] = tid;
    s_until[place] = until;
  }
  __syncthreads();
  // each(e, rank, need, row, j): what lane's place j of listed row e needs, rank its requests so far
  auto over_rows = [&](auto&& begin, auto&& each, auto&& end) __attribute__((always_inline)) {
    for (int e0 = wave; e0 < listed; e0 += kAtOnce * kWaves) {
      int row[kAtOnce], stop[kAtOnce], rank[kAtOnce], most = 0;
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        const int e = min(e0 + k * kWaves, listed - 1);
        row[k] = s_row[e];
        stop[k] = e0 + k * kWaves < listed ? s_until[e] : 0;
        rank[k] = begin(e);
        most = max(most, stop[k]);
      }
      for (int j = lane; j - lane < most; j += 64) {
        int p[kAtOnce];
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) p[k] = j < stop[k] ? t.row(row[k])[j] : 0;
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
          const bool need = j < stop[k] && !t.page_ok(p[k]);
          const uint64_t all = __builtin_amdgcn_ballot_w64(need);
          each(rank[k] + __builtin_popcountll(all & ((1ull << lane) - 1)), need, row[k], j);
          rank[k] += __builtin_popcountll(all);
        }
      }
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k)
        if (e0 + k * kWaves < listed) end(e0 + k * kWaves, rank[k]);
    }
  };
  if constexpr (kCounts) {
    over_rows([](int) { return 0; }, [](int, bool, int, int) {}, [&](int e, int n) { if (lane == 0) s_rank[e] = n; });
    __syncthreads();
    const int rank = block_exclusive(tid < listed ? s_rank[tid] : 0, shared, wanted);
    if (tid < listed) s_rank[tid] = rank;
  }
  const int got = take_free(t, first, wanted, a.free, shared);  // (ends with a barrier)
  if (tid == 0 && got < wanted) atomicAdd(t.missing, wanted - got);
  over_rows([&](int e) { return s_rank[e]; },
            [&](int mine, bool need, int row, int j) { if (need) t.row(row)[j] = mine < got ? a.free[mine] : -1; }, [](int, int) {});
}
__global__ __launch_bounds__(kScan) void reserve_place_kernel(const ReserveArgs a) { reserve_place<false>(a); }
__global__ __launch_bounds__(kScan) void reserve_small_kernel(const ReserveArgs a) { reserve_place<true>(a); }

// ------------------------------------------------------------------ host side

int check_table(const MimirPagesParams* p, bool rows) {
  fail_with(MIMIR_OK, "");
  if (p == nullptr) return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "params is NULL");
  if (p->num_pages < 0 || p->rows < 0 || p->width < 0 || p->num_pages > (1 << 30))
    return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "negative size, or over 2^30 pages");
  if (!rows) return MIMIR_OK;
  if (p->pages_stride < p->width) return fail_with(MIMIR_ERR_UNSUPPORTED_SHAPE, "rows of the page table overlap");
  if (p->counts == nullptr || p->missing == nullptr || (p->rows > 0 && (p->lengths == nullptr || (p->width > 0 && p->pages == nullptr))))
    return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "page table pointer is NULL");
  return MIMIR_OK;
}

int check_pool(const MimirPagesParams* p) {
  for (int i = 0; i < 4; ++i) {
    if (p->num_pages > 0 && p->data[i] == nullptr) return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "cache pointer is NULL");
    if (p->data_bytes[i] < 0 || (p->num_pages > 1 && p->data_stride[i] < p->data_bytes[i]))
      return fail_with(MIMIR_ERR_UNSUPPORTED_SHAPE, "pages of the cache overlap");
    if (i < 2 && ((uintptr_t)p->data[i] % 16 != 0 || p->data_bytes[i] % 16 != 0 || p->data_stride[i] % 16 != 0))
      return fail_with(MIMIR_ERR_UNSUPPORTED_SHAPE, "pages of keys and values must be 16-byte aligned");
  }
  return MIMIR_OK;
}

int check_workspace(const MimirPagesParams* p, int items) {
  const size_t need = mimir_prefixlm_pages_workspace_bytes(p, items);
  if (p->workspace == nullptr || p->workspace_bytes < need || (uintptr_t)p->workspace % 16 != 0)
    return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "workspace must be 16-byte aligned and hold at least " + std::to_string(need) + " bytes");
  return MIMIR_OK;
}

Table table_of(const MimirPagesParams& p) {
  return {p.pages, p.lengths, p.counts, p.missing, p.pages_stride, p.rows, p.width, p.num_pages};
}

CopyArgs copy_args(const MimirPagesParams& p) {
  CopyArgs a = {};
  for (int i = 0; i < 4; ++i) {
    a.pool.data[i] = (char*)p.data[i];
    a.pool.bytes[i] = p.data_bytes[i];
    a.pool.stride[i] = p.data_stride[i];
  }
  a.table = table_of(p);
  a.chunks = (int)((p.data_bytes[0] + kCopyChunk - 1) / kCopyChunk + (p.data_bytes[1] + kCopyChunk - 1) / kCopyChunk);
  return a;
}

// Workgroups of the move: one per unit, at most eight per CU (2048 threads).
void launch_move(const CopyArgs& a, int64_t units, hipStream_t s) {
  const int64_t grid = std::min<int64_t>(std::max<int64_t>(units, 1), 256 * 8);
  hipLaunchKernelGGL(pages_move_kernel, dim3((unsigned)grid), dim3(kCopyThreads), 0, s, a);
}

int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MIMIR_OK : fail_with(MIMIR_ERR_HIP, std::string(what) + ": " + hipGetErrorString(e));
}

}  // namespace
}  // namespace mimir

using namespace mimir;

extern "C" {

size_t mimir_prefixlm_pages_workspace_bytes(const MimirPagesParams* p, int32_t items) {
  if (p == nullptr || items < 0 || p->rows < 0 || p->width < 0 || p->num_pages < 0) return 0;
  // fork: six words and a table row per entry, two words per row; compact: three per page;
  // reserve: one per row and page; a few counters
  const int64_t n = items, words = n * ((int64_t)p->width + 6) + 2 * (int64_t)p->rows + 3 * (int64_t)p->num_pages + 16;
  return (size_t)words * sizeof(int32_t);
}

int mimir_prefixlm_pages_copy(const MimirPagesParams* p, const int32_t* source, const int32_t* destination, int32_t n,
                              void* stream) {
  int rc;
  if ((rc = check_table(p, false)) || (rc = check_pool(p))) return rc;
  if (n < 0) return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "negative size");
  if (n == 0 || p->num_pages == 0) return MIMIR_OK;
  if (source == nullptr || destination == nullptr) return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "page list is NULL");
  CopyArgs a = copy_args(*p);
  a.src = source;
  a.dst = destination;
  a.n = n;
  launch_move(a, (int64_t)n * a.chunks, (hipStream_t)stream);
  return launched("page copy launch");
}

int mimir_prefixlm_pages_fork(const MimirPagesParams* p, const int32_t* source, const int32_t* destination, int32_t n,
                              void* stream) {
  int rc;
  if ((rc = check_table(p, true)) || (rc = check_pool(p))) return rc;
  if (n < 0) return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "negative size");
  if (n > kMaxGroups) return fail_with(MIMIR_ERR_UNSUPPORTED_SHAPE, "too many rows for one call");
  if (n == 0 || p->rows == 0) return MIMIR_OK;
  if (source == nullptr || destination == nullptr) return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "row list is NULL");
  if ((rc = check_workspace(p, n))) return rc;
  const hipStream_t s = (hipStream_t)stream;
  ForkArgs f = {};
  f.t = table_of(*p);
  f.src = source;
  f.dst = destination;
  f.n = n;
  int32_t* w = (int32_t*)p->workspace;
  auto take = [&w](int64_t words) { int32_t* at = w; w += words; return at; };
  f.last = take(p->rows); f.first = take(p->rows);
  f.kept = take(n); f.new_len = take(n); f.tail = take(n);
  f.from = take(n); f.to = take(n); f.free = take(n);
  f.rowbuf = take((int64_t)n * p->width);
  f.given_up = take(1);
  // (All three in one workgroup took 26 us for 256 rows of up to 48 pages, a wave's rows one after another.)
  hipLaunchKernelGGL(fork_plan_kernel, dim3(1), dim3(kScan), 0, s, f);
  hipLaunchKernelGGL(fork_gather_kernel, dim3((unsigned)n), dim3(256), 0, s, f);
  hipLaunchKernelGGL(fork_take_kernel, dim3(1), dim3(kScan), 0, s, f);
  CopyArgs a = copy_args(*p);
  a.src = f.from;
  a.dst = f.to;
  a.n = n;
  a.rowbuf = f.rowbuf;
  a.kept = f.kept;
  a.dst_rows = destination;
  a.new_len = f.new_len;
  a.entries = n;
  launch_move(a, std::max<int64_t>((int64_t)n * a.chunks, ((int64_t)n * p->width + kCopyThreads - 1) / kCopyThreads), s);
  return launched("fork launch");
}

int mimir_prefixlm_pages_compact(const MimirPagesParams* p, int32_t* used, void* stream) {
  int rc;
  if ((rc = check_table(p, true)) || (rc = check_pool(p))) return rc;
  if (used == nullptr) return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "used is NULL");
  if ((rc = check_workspace(p, 0))) return rc;
  const hipStream_t s = (hipStream_t)stream;
  CompactArgs c = {};
  c.t = table_of(*p);
  int32_t* w = (int32_t*)p->workspace;
  c.used = used;
  c.n_moves = w;
  c.map = w + 16;
  c.from = c.map + p->num_pages;
  c.to = c.from + p->num_pages;
  hipLaunchKernelGGL(compact_plan_kernel, dim3(1), dim3(kScan), 0, s, c);
  CopyArgs a = copy_args(*p);
  a.src = c.from;
  a.dst = c.to;
  a.n_dev = c.n_moves;
  a.map = c.map;
  a.used = used;
  launch_move(a, std::max<int64_t>((int64_t)p->num_pages / 2 * a.chunks, ((int64_t)p->rows * p->width + kCopyThreads - 1) / kCopyThreads), s);
  return launched("compact launch");
}

int mimir_prefixlm_pages_release(const MimirPagesParams* p, const int32_t* row_list, int32_t n, void* stream) {
  int rc;
  if ((rc = check_table(p, true))) return rc;
  if (n < 0) return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "negative size");
  if (n > kMaxGroups) return fail_with(MIMIR_ERR_UNSUPPORTED_SHAPE, "too many rows for one call");
  if (n == 0 || p->rows == 0) return MIMIR_OK;
  if (row_list == nullptr) return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "row list is NULL");
  hipLaunchKernelGGL(release_kernel, dim3((unsigned)n), dim3(256), 0, (hipStream_t)stream, table_of(*p), row_list);
  return launched("release launch");
}

int mimir_prefixlm_pages_reserve(const MimirPagesParams* p, const int32_t* new_lengths, void* stream) {
  int rc;
  if ((rc = check_table(p, true))) return rc;
  if (p->rows == 0) return MIMIR_OK;
  if (p->rows > 4 * kMaxGroups) return fail_with(MIMIR_ERR_UNSUPPORTED_SHAPE, "too many rows for one call");
  if (new_lengths == nullptr) return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "new_lengths is NULL");
  if ((rc = check_workspace(p, 0))) return rc;
  const hipStream_t s = (hipStream_t)stream;
  ReserveArgs a = {};
  a.t = table_of(*p);
  a.new_len = new_lengths;
  int32_t* w = (int32_t*)p->workspace;
  a.got = w;
  a.lack = w + 16;
  a.free = a.lack + p->rows;
  const int64_t entries = (int64_t)p->rows * p->width;
  // One launch for small tables: 64 rows of 126 places, a page asked for here and there, in a graph 6.3 -> 5.7
  // us, eagerly (the host's time) 19.6 -> 14.3; 256 rows of 126 in a graph 12.7.
  if (p->rows <= 64 && entries <= 8192) {
    hipLaunchKernelGGL(reserve_small_kernel, dim3(1), dim3(kScan), 0, s, a);
    return launched("reserve launch");
  }
  const unsigned grid = (unsigned)((p->rows + 3) / 4);
  hipLaunchKernelGGL(reserve_count_kernel, dim3(grid), dim3(256), 0, s, a);
  // Two for up to 256 rows: 256 of 126 places, a page here and there, 6.3 -> 5.7 us in a graph, 40 rows admitted
  // 19.6 -> 17.2 eagerly, all of them (16000 pages) 28.0 -> 35.0; 500 of 700 rows (11000 pages) 23.9 -> 33.2.
  if (p->rows <= 256 && entries <= 1 << 30) {
    hipLaunchKernelGGL(reserve_place_kernel, dim3(1), dim3(kScan), 0, s, a);
    return launched("reserve launch");
  }
  hipLaunchKernelGGL(reserve_take_kernel, dim3(1), dim3(kScan), 0, s, a);
  hipLaunchKernelGGL(reserve_assign_kernel, dim3(grid), dim3(256), 0, s, a);
  return launched("reserve launch");
}

}  // extern "C"
