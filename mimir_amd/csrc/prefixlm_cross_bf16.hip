// Cross attention: packed queries over another packed set of states, with lengths of their own,
//
//   S = scale Q K^T,  P = softmax over the sequence's states,  O = P V,
//
// grouped heads read in place; a sequence without states has O = 0.  Every query sees every state of
// its sequence, so there is no mask but for the end of the last tile of 64 states.
//
// Forward: one workgroup = 4 waves = 128 query rows of one (sequence, query head), a wave 32 rows, in the
// formulation of prefixlm_fwd_bf16.hip: S^T = K Q^T on v_mfma_f32_32x32x16_bf16 leaves a query row in a
// lane (and its partner half a wave away), so the running maximum and sum are local to it, and P^T leaves the
// accumulator as the B operand of O^T += V^T P^T.  P is rounded to bf16 for that product, its
// sum is not.  K and V tiles come through two LDS stages by direct copies.  Bound by the matrix units: 2 x 8192 queries over
// 16384 states, 32 / 8 heads of 128, in 3.0 ms, 1.05 PFLOP/s (a library product of 8192^3: 1.30).
//
// The launch in front builds the tile list (most states first, by a counting sort in one workgroup),
// so that the tile kernels need neither the longest length nor a search for their sequence.
#include <algorithm>

#include "prefixlm_cross.h"

namespace mimir {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * 64;
constexpr int kBlockN = 64;  // states of an LDS tile

// ---------------------------------------------------------------- the launch in front

constexpr int kPlanThreads = 1024, kBuckets = 256;
constexpr int kFillBlocks = 32;

struct PrologueArgs {
  CrossPrologue p;
  int plans;
};

// Tiles of one side, those with most rows on the other side first.
__device__ __forceinline__ void plan_tiles(const SeqTable& t, bool by_key, int4* list, int cap) {
  __shared__ int counts[kBuckets], most, all, total;
  __shared__ int4 span[kPlanThreads];
  __shared__ int slot[kPlanThreads];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  if (tid == 0) most = all = total = 0;
  for (int i = tid; i < kBuckets; i += kPlanThreads) counts[i] = 0;
  __syncthreads();
  auto at = [&](int s) __attribute__((always_inline)) {  // (own first, own rows, other first, other rows)
    const SeqSpan g = seq_span(t, s);
    return by_key ? make_int4(g.k0, g.nk, g.q0, g.nq) : make_int4(g.q0, g.nq, g.k0, g.nk);
  };
  auto tiles = [](const int4& g) { return (g.y + kCrossTile - 1) / kCrossTile; };
  // Sequences that do not overlap have no more tiles than the list has entries.  Lists that decrease may name any number:
  // counted up to one more than the entries (host: below 2^24), where the sums below would wrap, and then none is listed.
  const int over = cap + 1;
  int own = 0;
  for (int s = tid; s < t.n; s += kPlanThreads) {
    const int4 g = at(s);
    if (g.y > 0) atomicMax(&most, g.w);
    own = min(own + tiles(g), over);
  }
  own = wave_inclusive_sum(own);
  if (lane == 63) atomicAdd(&all, min(own, over));
  __syncthreads();
  if (all > cap) {
    for (int i = tid; i < cap; i += kPlanThreads) list[i] = make_int4(0, 0, 0, 0);
    return;
  }
  const int step = most / kBuckets + 1;
  auto bucket = [&](const int4& g) __attribute__((always_inline)) { return max(kBuckets - 1 - g.w / step, 0); };
  for (int s = tid; s < t.n; s += kPlanThreads) {
    const int4 g = at(s);
    if (g.y > 0) atomicAdd(&counts[bucket(g)], tiles(g));
  }
  __syncthreads();
  if (wave == 0) {  // first entry of each bucket
    int c[kBuckets / 64], sum = 0;
#pragma unroll
    for (int i = 0; i < kBuckets / 64; ++i) {
      c[i] = counts[lane * (kBuckets / 64) + i];
      sum += c[i];
    }
    const int incl = wave_inclusive_sum(sum);
    int first = incl - sum;
#pragma unroll
    for (int i = 0; i < kBuckets / 64; ++i) {
      counts[lane * (kBuckets / 64) + i] = first;
      first += c[i];
    }
    if (lane == 63) total = incl;
  }
  __syncthreads();
  for (int s0 = 0; s0 < t.n; s0 += kPlanThreads) {
    if (s0 + tid < t.n) {
      const int4 g = at(s0 + tid);
      span[tid] = g;
      slot[tid] = g.y > 0 ? atomicAdd(&counts[bucket(g)], tiles(g)) : 0;
    }
    __syncthreads();
    for (int i = wave; i < min(t.n - s0, kPlanThreads); i += kPlanThreads / 64) {
      const int4 g = span[i];
      for (int j = lane; j < tiles(g); j += 64)
        list[slot[i] + j] = make_int4(g.x + j * kCrossTile, min(g.y - j * kCrossTile, kCrossTile), g.z, g.w);
    }
    __syncthreads();
  }
  for (int i = total + tid; i < cap; i += kPlanThreads) list[i] = make_int4(0, 0, 0, 0);
}

// Zeros in the rows before the first and behind the last sequence.
__device__ __forceinline__ void fill_rows(const CrossPrologue& p, const CrossPrologue::Fill& f, int block) {
  const SeqTable& t = p.seqs;
  const int rows = f.by_key ? t.Tk : t.Tq;
  const int32_t* cu = f.by_key ? t.cu_k : t.cu_q;
  const int lo = t.n > 0 ? min(max(cu[0], 0), rows) : rows;
  const int hi = t.n > 0 ? min(max(cu[t.n], lo), rows) : rows;
  const int units = p.D / 8;
  const int64_t per = (int64_t)f.heads * units, total = (int64_t)(lo + rows - hi) * per;
  for (int64_t i = (int64_t)block * kPlanThreads + threadIdx.x; i < total; i += (int64_t)kFillBlocks * kPlanThreads) {
    int64_t row = i / per;
    const int rest = (int)(i - row * per), h = rest / units;
    row += row < lo ? 0 : hi - lo;
    *(i32x4*)&f.x[row * f.st + h * f.sh + (rest - h * units) * 8] = i32x4{0, 0, 0, 0};
    if (p.lse2 != nullptr && !f.by_key && rest == h * units) p.lse2[(int64_t)h * t.Tq + row] = -INFINITY;
  }
}

__global__ __launch_bounds__(kPlanThreads) void cross_prologue_kernel(const PrologueArgs a) {
  int b = blockIdx.x;
  if (b < a.plans) {
    const bool by_key = a.p.plan_q == nullptr || b == 1;
    plan_tiles(a.p.seqs, by_key, by_key ? a.p.plan_k : a.p.plan_q, by_key ? a.p.cap_k : a.p.cap_q);
    return;
  }
  b -= a.plans;
  fill_rows(a.p, a.p.fill[b / kFillBlocks], b % kFillBlocks);
}

// ---------------------------------------------------------------- forward

// Two LDS stages, the same for both bodies of a kernel.
template <int D>
struct FwdStages {
  bf16_t *k0, *v0, *k1, *v1;
};
template <int D>
__device__ __forceinline__ FwdStages<D> fwd_stages() {
  using L = TileLayout<D>;
  __shared__ __attribute__((aligned(16))) bf16_t sK0[L::kElems];
  __shared__ __attribute__((aligned(16))) bf16_t sV0[L::kElems];
  __shared__ __attribute__((aligned(16))) bf16_t sK1[L::kElems];
  __shared__ __attribute__((aligned(16))) bf16_t sV1[L::kElems];
  return FwdStages<D>{sK0, sV0, sK1, sV1};
}

// kSplit: P as two bf16 halves in its product.
template <int D, bool kSplit>
__device__ __forceinline__ void cross_fwd_body(const CrossArgs& a, const QueryTile& tile) {
  constexpr int DT = D / 32;  // 32-row tiles of O^T
  constexpr int KS = D / 16;  // steps of S^T = K Q^T
  using L = TileLayout<D>;
  const FwdStages<D> stages = fwd_stages<D>();
  bf16_t *const sK0 = stages.k0, *const sV0 = stages.v0, *const sK1 = stages.k1, *const sV1 = stages.v1;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31;
  const int hi = lane >> 5;

  const int4 item = tile.item;
  const int h = tile.h, hk = tile.hk, rows = item.y, nk = item.w;
  const int nkt = (nk + kBlockN - 1) / kBlockN;
  const int qa = wave * 32;
  const bool wave_active = qa < rows;
  const int qrow = qa + l32;

  const bf16_t* const qtile = a.q + (int64_t)item.x * a.q_st + (int64_t)h * a.q_sh;
  const __amdgpu_buffer_rsrc_t rq = make_rsrc(qtile, rows_bytes(rows, a.q_st, D));
  const TileLoader<D, kWaves> ldk(a.k_st, wave, lane), ldv(a.v_st, wave, lane);
  const bf16_t* i_k = a.k + (int64_t)item.z * a.k_st + (int64_t)hk * a.k_sh;
  const bf16_t* i_v = a.v + (int64_t)item.z * a.v_st + (int64_t)hk * a.v_sh;
  int i_rows = nk;
  auto issue_next = [&](bf16_t* tk, bf16_t* tv) {
    const int n = min(i_rows, kBlockN);  // (a sequence may span more than 32 bits)
    ldk.issue_at(i_k, rows_bytes32(n, (uint32_t)a.k_st, D), tk);
    ldv.issue_at(i_v, rows_bytes32(n, (uint32_t)a.v_st, D), tv);
    i_k += kBlockN * a.k_st;
    i_v += kBlockN * a.v_st;
    i_rows -= kBlockN;
  };
  if (nkt > 0) issue_next(sK0, sV0);

  // Q^T B-operand fragments: lane holds row qrow, d = 16 ks + 8 hi .. + 7.
  bf16x8 qf[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks)
    qf[ks] = __builtin_bit_cast(bf16x8, buf_load16(rq, (uint32_t)((qrow * a.q_st + 16 * ks + 8 * hi) * 2)));

  f32x16 oacc[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) oacc[dt] = f32x16{};
  float m_run = -INFINITY, l_run = 0.f;
  const float c2 = a.scale_log2;
  const TileLanes<D> tl(lane);

  auto compute = [&](int kt, const bf16_t* sK, const bf16_t* sV) {
    f32x16 st[2];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      st[mt] = f32x16{};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        st[mt] = mfma32(*(const bf16x8*)&sK[tl.op_base + mt * 32 * L::kRowElems + ks * 16], qf[ks], st[mt]);
    }
    if (kt * kBlockN + kBlockN > nk) {  // the last tile reaches past the states
      __asm__ volatile("");             // a real branch: other tiles do not pay for the compares
      const int left = nk - kt * kBlockN - 4 * hi;
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (32 * mt + 8 * (r >> 2) + (r & 3) >= left) st[mt][r] = -INFINITY;
    }
    float mx = -INFINITY;
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, st[mt][r]);
    mx = xor32_max(mx);
    // The reference maximum moves only when the running one grows by more than 2^8 in terms of
    // probabilities: in between these stay below 256, and the sum is taken to the same reference.
    const float m_cand = fmaxf(m_run, mx);
    const bool grow = (m_cand - m_run) * c2 > 8.f;
    if (__builtin_amdgcn_ballot_w64(grow) != 0) {
      const float alpha = grow ? fast_exp2((m_run - m_cand) * c2) : 1.f;
      l_run *= alpha;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) oacc[dt] *= alpha;
      if (grow) m_run = m_cand;
    }
    const float mb = m_run == -INFINITY ? 0.f : m_run * c2;
    float lsum = 0.f;
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float pr = fast_exp2(__builtin_fmaf(st[mt][r], c2, -mb));
        st[mt][r] = pr;
        lsum += pr;
      }
    l_run += lsum;
    bf16x8 pf[4], pl[kSplit ? 4 : 1];
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      f32x8 t;
#pragma unroll
      for (int e = 0; e < 8; ++e) t[e] = st[kk >> 1][(kk & 1) * 8 + e];
      pf[kk] = to_bf16x8(t);
      if constexpr (kSplit) pl[kk] = lo_half(t, pf[kk]);
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        const bf16_t* vp = &sV[tl.tr_base + kk * 16 * L::kRowElems + dt * 32];
        const bf16x8 vt = cat8(lds_read_tr16(vp), lds_read_tr16(vp + L::kTrSecond));
        oacc[dt] = mfma32(vt, pf[kk], oacc[dt]);
        if constexpr (kSplit) oacc[dt] = mfma32(vt, pl[kk], oacc[dt]);
      }
  };

  for (int kt = 0; kt < nkt; kt += 2) {
    wait_vmem();
    __syncthreads();
    if (kt + 1 < nkt) issue_next(sK1, sV1);
    if (wave_active) compute(kt, sK0, sV0);
    if (kt + 1 >= nkt) break;
    wait_vmem();
    __syncthreads();
    if (kt + 2 < nkt) issue_next(sK0, sV0);
    if (wave_active) compute(kt + 1, sK1, sV1);
  }

  // Each wave stages its 32 rows in one K / V stage object, free once every wave is past the
  // tile loop, and stores whole rows.
  __syncthreads();
  if (!wave_active) return;
  const float l_tot = xor32_sum(l_run);
  const float inv = l_tot > 0.f ? 1.f / l_tot : nk > 0 ? __builtin_nanf("") : 0.f;
  constexpr int kPitch = D + 8;  // elements; rows stay 16-byte aligned
  constexpr int kUnits = D / 8;  // 16-byte units per row
  constexpr int kRowsPerInst = 64 / kUnits;
  static_assert(32 * kPitch <= L::kElems, "a wave's rows fit its stage object");
  bf16_t* const stage = wave == 0 ? sK0 : wave == 1 ? sV0 : wave == 2 ? sK1 : sV1;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int rg = 0; rg < 4; ++rg) {
      f32x4 t;
#pragma unroll
      for (int e = 0; e < 4; ++e) t[e] = oacc[dt][4 * rg + e] * inv;
      *(bf16x4*)&stage[l32 * kPitch + 32 * dt + 8 * rg + 4 * hi] = __builtin_convertvector(t, bf16x4);
    }
  if (hi == 0 && a.lse2 != nullptr && qrow < rows)
    a.lse2[(int64_t)h * a.Tq + item.x + qrow] = nk > 0 ? m_run * c2 + fast_log2(l_tot) : -INFINITY;
  // The LDS unit runs one wave's accesses in order: the reads below see the writes above.
  __asm__ volatile("" ::: "memory");
  const int u = lane % kUnits;
  bf16_t* const obase = a.o + (int64_t)(item.x + qa) * a.o_st + (int64_t)h * a.o_sh + u * 8;
#pragma unroll
  for (int j = 0; j < 32 / kRowsPerInst; ++j) {
    const int r = j * kRowsPerInst + lane / kUnits;
    const bf16x8 ov = *(const bf16x8*)&stage[r * kPitch + u * 8];
    if (qa + r < rows) *(bf16x8*)&obase[(int64_t)r * a.o_st] = ov;
  }
  if (a.o_lo == nullptr) return;
  // The low half, another round through the same rows.
  __asm__ volatile("" ::: "memory");
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int rg = 0; rg < 4; ++rg) {
      f32x4 lo;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float t = oacc[dt][4 * rg + e] * inv;
        lo[e] = t - round_to(t, bf16_t());
      }
      *(bf16x4*)&stage[l32 * kPitch + 32 * dt + 8 * rg + 4 * hi] = __builtin_convertvector(lo, bf16x4);
    }
  __asm__ volatile("" ::: "memory");
  bf16_t* const lbase = a.o_lo + ((int64_t)(item.x + qa) * a.Hq + h) * D + u * 8;
#pragma unroll
  for (int j = 0; j < 32 / kRowsPerInst; ++j) {
    const int r = j * kRowsPerInst + lane / kUnits;
    const bf16x8 lv = *(const bf16x8*)&stage[r * kPitch + u * 8];
    if (qa + r < rows) __builtin_nontemporal_store(lv, (bf16x8*)&lbase[(int64_t)r * a.Hq * D]);
  }
}

// The split body in a function of its own, which reads its arguments from the kernel's segment: the plain body keeps
// the registers of a kernel of its own.
template <int D>
__device__ __attribute__((noinline)) void cross_fwd_split(uint64_t seg) {
  const CrossArgs& a = segment_args<CrossArgs>(uniform_segment(seg));
  cross_fwd_body<D, true>(a, query_tile(a));
}
template <int D>
constexpr int kFwdWaves = D == 64 ? 4 : 2;  // waves per SIMD = workgroups per CU
template <int D>
__global__ __attribute__((amdgpu_flat_work_group_size(kThreads, kThreads),
                          amdgpu_waves_per_eu(kFwdWaves<D>, kFwdWaves<D>))) void cross_fwd_kernel(const CrossArgs a) {
  const QueryTile tile = query_tile(a);
  if (tile.item.y == 0) return;
  if (tile.item.w <= kSplitStates)
    cross_fwd_split<D>(kernel_segment());
  else
    cross_fwd_body<D, false>(a, tile);
}
template __global__ void cross_fwd_kernel<64>(const CrossArgs);
template __global__ void cross_fwd_kernel<128>(const CrossArgs);

}  // namespace

hipError_t launch_cross_prologue(const CrossPrologue& p, hipStream_t stream) {
  const PrologueArgs a = {p, (p.plan_q != nullptr) + (p.plan_k != nullptr)};
  const int blocks = a.plans + p.nfill * kFillBlocks;
  if (blocks == 0) return hipSuccess;
  hipLaunchKernelGGL(cross_prologue_kernel, dim3((unsigned)blocks), dim3(kPlanThreads), 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_cross_fwd(const CrossArgs& a, int head_dim, hipStream_t stream) {
  const int64_t units = (int64_t)a.cap_q * a.Hkv;
  if (units == 0) return hipSuccess;
  const dim3 grid((unsigned)((units + kXcds - 1) / kXcds * kXcds * a.group));
  if (head_dim == 128)
    hipLaunchKernelGGL(cross_fwd_kernel<128>, grid, dim3(kThreads), 0, stream, a);
  else
    hipLaunchKernelGGL(cross_fwd_kernel<64>, grid, dim3(kThreads), 0, stream, a);
  return hipGetLastError();
}

namespace {

struct CrossWorkspace {
  size_t plan_q, plan_k, delta, total;
  int cap_q, cap_k;
};
CrossWorkspace cross_workspace(const MimirCrossParams& p, bool backward) {
  CrossWorkspace w;
  w.cap_q = cross_capacity(p.total_q, p.numseqs);
  w.cap_k = backward ? cross_capacity(p.total_k, p.numseqs) : 0;
  w.plan_q = 0;
  w.plan_k = align_up((size_t)w.cap_q * sizeof(int4));
  w.delta = w.plan_k + align_up((size_t)w.cap_k * sizeof(int4));
  w.total = w.delta + (backward ? align_up((size_t)p.total_q * (size_t)p.num_q_heads * sizeof(float)) : 0);
  return w;
}

// Checks what both directions share; MIMIR_OK if the call has work to do or none.
int check_cross(const MimirCrossParams* p, bool backward) {
  if (p == nullptr) return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "params is NULL");
  if (p->dtype != MIMIR_DTYPE_BFLOAT16)
    return fail_with(MIMIR_ERR_UNSUPPORTED_DTYPE, "cross attention supports bfloat16 tensors only (dtype code " + std::to_string(p->dtype) + ")");
  if (p->total_q < 0 || p->total_k < 0 || p->numseqs < 0 || p->num_q_heads <= 0 || p->num_kv_heads <= 0)
    return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "negative size or non-positive heads");
  if (p->num_q_heads % p->num_kv_heads != 0)
    return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "Query heads " + std::to_string(p->num_q_heads) + " must be divisible by key/value heads " +
                                                     std::to_string(p->num_kv_heads) + ".");
  if (p->head_dim != 64 && p->head_dim != 128)
    return fail_with(MIMIR_ERR_UNSUPPORTED_SHAPE, "cross attention supports head_dim 64 and 128, got " + std::to_string(p->head_dim));
  if (!(p->softmax_scale > 1e-30f) || !(p->softmax_scale < 1e30f))
    return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "softmax_scale must be positive and neither below 1e-30 nor above 1e30");
  if ((int64_t)p->num_q_heads * p->head_dim >= (1 << 22))
    return fail_with(MIMIR_ERR_UNSUPPORTED_SHAPE, "a token's query heads must hold fewer than 2^22 elements");
  if ((int64_t)p->total_q * p->num_q_heads > 0x7fffffff || (int64_t)p->total_k * p->num_q_heads > 0x7fffffff)
    return fail_with(MIMIR_ERR_UNSUPPORTED_SHAPE, "too many rows for one call");
  // a workgroup of 256 threads per query tile and head, one of up to 512 per tile of states and kv head
  if ((int64_t)cross_capacity(p->total_q, p->numseqs) * p->num_q_heads > kMaxGroups - kXcds * p->num_q_heads ||
      (backward && (int64_t)cross_capacity(p->total_k, p->numseqs) * p->num_kv_heads > kMaxGroups / 2))
    return fail_with(MIMIR_ERR_UNSUPPORTED_SHAPE, "too many sequences for one launch");
  if (p->numseqs > 0 && (p->cu_seqlens_q == nullptr || p->cu_seqlens_k == nullptr))
    return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "cu_seqlens is NULL");
  struct Tensor {
    const void* x;
    int64_t st, sh;
    int rows;
  };
  const Tensor all[] = {{p->q, p->q_stride_token, p->q_stride_head, p->total_q},
                        {p->out, p->out_stride_token, p->out_stride_head, p->total_q},
                        {p->k, p->k_stride_token, p->k_stride_head, p->total_k},
                        {p->v, p->v_stride_token, p->v_stride_head, p->total_k},
                        {p->dout, p->dout_stride_token, p->dout_stride_head, p->total_q},
                        {p->dq, p->dq_stride_token, p->dq_stride_head, p->total_q},
                        {p->dk, p->dk_stride_token, p->dk_stride_head, p->total_k},
                        {p->dv, p->dv_stride_token, p->dv_stride_head, p->total_k}};
  for (int i = 0; i < (backward ? 8 : 4); ++i) {
    const Tensor& t = all[i];
    if (t.rows == 0) continue;
    if (t.x == nullptr) return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "cross attention tensor pointer is NULL");
    if ((uintptr_t)t.x % 16 != 0 || t.st % 8 != 0 || t.sh % 8 != 0)
      return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "cross attention rows must be 16-byte aligned");
    // 128 rows of a tile are addressed in 31 bits
    if (t.st < p->head_dim || t.st >= (1 << 22) || t.sh < 0)
      return fail_with(MIMIR_ERR_UNSUPPORTED_SHAPE, "token strides must be at least head_dim and below 2^22 elements, head strides not negative");
  }
  if (p->total_q > 0 && backward && (p->lse2 == nullptr || p->out_lo == nullptr))
    return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "lse2 or out_lo is NULL");
  if ((uintptr_t)p->out_lo % 16 != 0) return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "out_lo must be 16-byte aligned");
  const size_t need = cross_workspace(*p, backward).total;
  if (need > 0 && (p->workspace == nullptr || (uintptr_t)p->workspace % 256 != 0 || p->workspace_bytes < need))
    return fail_with(MIMIR_ERR_INVALID_ARGUMENT, "cross attention needs a workspace of " + std::to_string(need) + " bytes aligned to 256");
  return MIMIR_OK;
}

CrossArgs cross_args(const MimirCrossParams& p, const CrossWorkspace& w) {
  CrossArgs a = {};
  a.q = (const bf16_t*)p.q; a.k = (const bf16_t*)p.k; a.v = (const bf16_t*)p.v;
  a.dout = (const bf16_t*)p.dout;
  a.o = (bf16_t*)p.out; a.dq = (bf16_t*)p.dq; a.dk = (bf16_t*)p.dk; a.dv = (bf16_t*)p.dv;
  a.o_lo = (bf16_t*)p.out_lo;
  a.lse2 = p.lse2;
  a.delta = (float*)((char*)p.workspace + w.delta);
  a.q_st = p.q_stride_token; a.q_sh = p.q_stride_head;
  a.k_st = p.k_stride_token; a.k_sh = p.k_stride_head;
  a.v_st = p.v_stride_token; a.v_sh = p.v_stride_head;
  a.o_st = p.out_stride_token; a.o_sh = p.out_stride_head;
  a.do_st = p.dout_stride_token; a.do_sh = p.dout_stride_head;
  a.dq_st = p.dq_stride_token; a.dq_sh = p.dq_stride_head;
  a.dk_st = p.dk_stride_token; a.dk_sh = p.dk_stride_head;
  a.dv_st = p.dv_stride_token; a.dv_sh = p.dv_stride_head;
  a.Tq = p.total_q; a.Hq = p.num_q_heads; a.Hkv = p.num_kv_heads; a.group = p.num_q_heads / p.num_kv_heads;
  a.plan_q = (const int4*)((char*)p.workspace + w.plan_q);
  a.plan_k = (const int4*)((char*)p.workspace + w.plan_k);
  a.cap_q = w.cap_q; a.cap_k = w.cap_k;
  a.scale = p.softmax_scale;
  a.scale_log2 = p.softmax_scale * kLog2e;
  return a;
}

CrossPrologue cross_prologue(const MimirCrossParams& p, const CrossArgs& a) {
  CrossPrologue pro = {};
  pro.seqs.cu_q = p.cu_seqlens_q; pro.seqs.cu_k = p.cu_seqlens_k;
  pro.seqs.n = p.numseqs; pro.seqs.Tq = p.total_q; pro.seqs.Tk = p.total_k;
  if (a.cap_q > 0) pro.plan_q = (int4*)a.plan_q;
  if (a.cap_k > 0) pro.plan_k = (int4*)a.plan_k;
  pro.cap_q = a.cap_q; pro.cap_k = a.cap_k;
  pro.D = p.head_dim;
  return pro;
}

}  // namespace
}  // namespace mimir

extern "C" size_t mimir_prefixlm_cross_workspace_bytes(const MimirCrossParams* p, int32_t backward) {
  if (p == nullptr || p->total_q < 0 || p->total_k < 0 || p->numseqs < 0 || p->num_q_heads <= 0) return 0;
  return mimir::cross_workspace(*p, backward != 0).total;
}

extern "C" int mimir_prefixlm_cross_fwd(const MimirCrossParams* p, void* stream) {
  using namespace mimir;
  fail_with(MIMIR_OK, "");
  const int status = check_cross(p, false);
  if (status != MIMIR_OK || p->total_q == 0) return status;
  const CrossArgs a = cross_args(*p, cross_workspace(*p, false));
  CrossPrologue pro = cross_prologue(*p, a);
  pro.fill[pro.nfill++] = {a.o, a.o_st, a.o_sh, 0, a.Hq};
  pro.lse2 = a.lse2;
  hipError_t e = launch_cross_prologue(pro, (hipStream_t)stream);
  if (e == hipSuccess) e = launch_cross_fwd(a, p->head_dim, (hipStream_t)stream);
  return e == hipSuccess ? MIMIR_OK : fail_with(MIMIR_ERR_HIP, std::string("cross attention launch: ") + hipGetErrorString(e));
}

extern "C" int mimir_prefixlm_cross_bwd(const MimirCrossParams* p, void* stream) {
  using namespace mimir;
  fail_with(MIMIR_OK, "");
  const int status = check_cross(p, true);
  if (status != MIMIR_OK || (p->total_q == 0 && p->total_k == 0)) return status;
  const CrossArgs a = cross_args(*p, cross_workspace(*p, true));
  CrossPrologue pro = cross_prologue(*p, a);
  if (p->total_q > 0) pro.fill[pro.nfill++] = {a.dq, a.dq_st, a.dq_sh, 0, a.Hq};
  if (p->total_k > 0) {
    pro.fill[pro.nfill++] = {a.dk, a.dk_st, a.dk_sh, 1, a.Hkv};
    pro.fill[pro.nfill++] = {a.dv, a.dv_st, a.dv_sh, 1, a.Hkv};
  }
  hipError_t e = launch_cross_prologue(pro, (hipStream_t)stream);
  if (e == hipSuccess) e = launch_cross_bwd(a, p->head_dim, (hipStream_t)stream);
  return e == hipSuccess ? MIMIR_OK : fail_with(MIMIR_ERR_HIP, std::string("cross attention backward launch: ") + hipGetErrorString(e));
}
