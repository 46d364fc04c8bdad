// Cross attention backward, bf16: with P = exp2(S scale log2 e - lse2) and delta = rowsum(dO * O),
//
//   dV = P^T dO,  dP = dO V^T,  dS = P (dP - delta),  dQ = scale dS K,  dK = scale dS^T Q.
//
// Two kernels, each the owner of what it sums, so nothing is added atomically and results do not
// depend on timing: dQ per (query head, 128 query rows), which also forms delta, and then dK / dV per (kv head,
// 128 states), over all query heads of the group and all queries of the sequence, which forms S and dP again.
// delta takes O with its low half: dS is a difference whose rounding errors would else be led by O's
// (error of dQ and dK against 64 bits, in units of one rounding of the exact result: up to 2.3 without, 1.4 with it).
// P and dS are rounded to bf16 for their products.  Both are bound by the matrix units: 8 sequences of 1500 to 2048 queries over
// 1024 to 2048 states, 16 / 4 heads of 128, dQ 270 to 290 us (0.94 PFLOP/s executed at 279), dK / dV 375 to 410 (0.87 at 402, a fifth of it the tail).
// No tile is split over workgroups, so few tiles leave the chip idle: forward and backward of 4096 queries over 77 states (one tile of
// states, 16 / 4 heads) take 402 us, of 16 queries over 8192 states 340.
#include "prefixlm_cross.h"

namespace mimir {
namespace {

// ---------------------------------------------------------------------------
// dK / dV, in the scheme of prefixlm_bwd_dkdv_pair_bf16.hip.  Workgroup = 8 waves.  Waves w and w + 4 own the
// same 32 states (slice w % 4, both on SIMD w % 4) and take the two 32-row halves of every 64-query tile,
// so each keeps partial sums over half of the queries, which are added through LDS at the end.
// Only the K fragments stay in registers; the V tile is staged in LDS once and read as the B operand of
// dP.  With two waves per SIMD one's softmax overlaps the other's MFMAs.  Q and dO tiles with their lse2
// and delta rows come through three LDS stages.  Rows past the queries read as zeros, with lse2 = delta = 0:
// P = 1 there, but dO = 0 and dS = 0.
// ---------------------------------------------------------------------------
constexpr int kKvWaves = 8;
constexpr int kQTile = 64;

template <int D>
__device__ __forceinline__ void cross_dkdv_body(const CrossArgs& a) {
  constexpr int DT = D / 32;
  constexpr int KS = D / 16;
  using L = TileLayout<D>;
  using Loader = TileLoader<D, kKvWaves>;
  constexpr int kStageElems = 2 * L::kElems + 2 * kQTile * 2;  // Q, dO, lse2 + delta (fp32)
  __shared__ __attribute__((aligned(16))) bf16_t sS0[kStageElems];
  __shared__ __attribute__((aligned(16))) bf16_t sS1[kStageElems];
  __shared__ __attribute__((aligned(16))) bf16_t sS2[kStageElems];
  __shared__ __attribute__((aligned(16))) bf16_t sV[2 * L::kElems];
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int slice = wave & 3, qh = wave >> 2;
  const int l32 = lane & 31;
  const int hi = lane >> 5;
  const int rank = blockIdx.x / a.Hkv, hk = blockIdx.x - rank * a.Hkv;
  const int4 item = load_entry(a.plan_k, rank);
  const int keys = item.y, nq = item.w;
  if (keys == 0) return;  // list padding

  const Loader ldq(a.q_st, wave, lane), ldo(a.do_st, wave, lane), ldv(a.v_st, wave, lane);
  const TileLanes<D> tl(lane);
  const float c2 = a.scale_log2;
  const int ka = slice * 32;  // this wave's first state in the tile
  const bool wave_active = ka < keys;
  const int nqt = (nq + kQTile - 1) / kQTile;
  const int n_iter = nqt * a.group;  // (query head, query tile) steps

  const bf16_t* ktile = a.k + (int64_t)item.x * a.k_st + (int64_t)hk * a.k_sh;
  const bf16_t* vtile = a.v + (int64_t)item.x * a.v_st + (int64_t)hk * a.v_sh;
  const uint32_t q_st32 = (uint32_t)a.q_st, o_st32 = (uint32_t)a.do_st;
  const int qh0 = hk * a.group;
  const bf16_t* q_head = a.q + (int64_t)item.z * a.q_st + (int64_t)qh0 * a.q_sh;
  const bf16_t* o_head = a.dout + (int64_t)item.z * a.do_st + (int64_t)qh0 * a.do_sh;
  // one 4-byte row per wave: wave 0 lse2, the others delta (same data to the same place)
  const float* r_head = (wave == 0 ? a.lse2 : a.delta) + (int64_t)qh0 * a.Tq + item.z;
  const bf16_t* i_q = q_head;
  const bf16_t* i_o = o_head;
  const float* i_r = r_head;
  int i_qt = 0, i_rows = nq;
  // Every step issues its copies, also past the last tile (`valid` false: zero bytes are copied, no memory
  // is read), so that the waits are the same on every step.
  auto issue_next = [&](bool valid, bf16_t* stage) {
    const int rows = valid ? min(i_rows, kQTile) : 0;
    ldq.issue_at(i_q, rows_bytes32(rows, q_st32, D), stage);
    ldo.issue_at(i_o, rows_bytes32(rows, o_st32, D), stage + L::kElems);
    float* const tr = (float*)(stage + 2 * L::kElems);
    const __amdgpu_buffer_rsrc_t r = make_rsrc(i_r, (uint32_t)rows * 4u);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(tr + (wave == 0 ? 0 : kQTile)), 4,
                                             (uint32_t)lane * 4u, 0, 0, 0);
    if (++i_qt == nqt) {
      i_qt = 0;
      i_rows = nq;
      q_head += a.q_sh;
      o_head += a.do_sh;
      r_head += a.Tq;
      i_q = q_head;
      i_o = o_head;
      i_r = r_head;
    } else {
      i_rows -= kQTile;
      i_q += kQTile * a.q_st;
      i_o += kQTile * a.do_st;
      i_r += kQTile;
    }
  };

  ldv.issue(vtile, 0, keys, sV);
  ldv.issue(vtile, 64, keys, sV + L::kElems);
  issue_next(n_iter > 0, sS0);
  const __amdgpu_buffer_rsrc_t rk = make_rsrc(ktile, rows_bytes(keys, a.k_st, D));
  bf16x8 kf[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks)
    kf[ks] = __builtin_bit_cast(bf16x8, buf_load16(rk, (uint32_t)(((ka + l32) * a.k_st + 16 * ks + 8 * hi) * 2)));
  issue_next(n_iter > 1, sS1);
  // Copies per issue and wave: the Q and dO loaders share one assignment, so a wave with the last
  // round's instructions (wave 0) issues 2 * kPerWave + 1 with its row, the others two fewer.
  constexpr int kLoadsPerIssue = 2 * Loader::kPerWave + 1;
  auto sync_stage = [&]() {
    if (ldq.has_last)
      stage_barrier<kLoadsPerIssue>();
    else
      stage_barrier<kLoadsPerIssue - 2>();
  };

  f32x16 dkacc[DT], dvacc[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) {
    dkacc[dt] = f32x16{};
    dvacc[dt] = f32x16{};
  }
  const bf16_t* const sVs = sV + (slice >> 1) * L::kElems + tl.op_base + (slice & 1) * 32 * L::kRowElems;

  auto compute = [&](const bf16_t* stage) {
    const bf16_t* const sQ = stage;
    const bf16_t* const sdO = stage + L::kElems;
    const float* const sL = (const float*)(stage + 2 * L::kElems);
    const float* const sD = sL + kQTile;
    f32x16 sc = f32x16{}, dp = f32x16{};
    // Per-step copies of the lane offsets: one register per offset live instead of one per (stage, operand).
    int opb = tl.op_base + qh * 32 * L::kRowElems, trb = tl.tr_base + qh * 32 * L::kRowElems, lrow = 32 * qh + 4 * hi;
    __asm__ volatile("" : "+v"(opb), "+v"(trb), "+v"(lrow));
    // LDS operand reads run two MFMA pairs ahead of their use; the scheduling barriers keep them there.
    bf16x8 qa[KS], oa[KS], va[KS];
    auto rd_a = [&](int ks) {
      qa[ks] = *(const bf16x8*)&sQ[opb + ks * 16];
      oa[ks] = *(const bf16x8*)&sdO[opb + ks * 16];
      va[ks] = *(const bf16x8*)&sVs[ks * 16];
    };
    // dV / dK operand pair j: 16-query step j / DT of this wave's half, 32 columns j % DT
    bf16x8 ot[3], qt[3];
    auto rd_tr = [&](int j) {
      const int o = trb + (j / DT) * 16 * L::kRowElems + (j % DT) * 32;
      ot[j % 3] = cat8(lds_read_tr16(&sdO[o]), lds_read_tr16(&sdO[o + L::kTrSecond]));
      qt[j % 3] = cat8(lds_read_tr16(&sQ[o]), lds_read_tr16(&sQ[o + L::kTrSecond]));
    };
    f32x4 l4[2], d4[2];  // lse2 / delta of the rows of one 16-query step
    auto rd_ld = [&](int s2) {
#pragma unroll
      for (int rg2 = 0; rg2 < 2; ++rg2) {
        l4[rg2] = *(const f32x4*)&sL[lrow + 8 * (2 * s2 + rg2)];
        d4[rg2] = *(const f32x4*)&sD[lrow + 8 * (2 * s2 + rg2)];
      }
    };
    f32x8 tp, tds;
    auto softmax = [&](int s2, int rg2) {  // P and dS of rows 8 (2 s2 + rg2) + 4 hi + e
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = 4 * (2 * s2 + rg2) + e;
        const float pr = fast_exp2(__builtin_fmaf(sc[r], c2, -l4[rg2][e]));
        tp[4 * rg2 + e] = pr;
        tds[4 * rg2 + e] = pr * (dp[r] - d4[rg2][e]);
      }
    };
    rd_a(0);
    rd_a(1);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      __builtin_amdgcn_sched_barrier(0);
      if (ks + 2 < KS) rd_a(ks + 2);
      sc = mfma32(qa[ks], kf[ks], sc);
      dp = mfma32(oa[ks], va[ks], dp);
    }
    rd_ld(0);
    rd_tr(0);
    rd_tr(1);
    __builtin_amdgcn_sched_barrier(0);
    bf16x8 pb[2], db[2];
    softmax(0, 0);
    softmax(0, 1);
    pb[0] = to_bf16x8(tp);
    db[0] = to_bf16x8(tds);
    rd_ld(1);
    // 2 DT dV / dK MFMA pairs; the softmax of the second 16-query step runs beside the first DT.
#pragma unroll
    for (int j = 0; j < 2 * DT; ++j) {
      __builtin_amdgcn_sched_barrier(0);
      if (j + 2 < 2 * DT) rd_tr(j + 2);
      const int dt = j % DT, s2 = j / DT;
      dvacc[dt] = mfma32(ot[j % 3], pb[s2], dvacc[dt]);
      dkacc[dt] = mfma32(qt[j % 3], db[s2], dkacc[dt]);
      if (j == DT / 2 - 1) softmax(1, 0);
      if (j == DT / 2) softmax(1, 1);
      if (j == DT - 1) {
        pb[1] = to_bf16x8(tp);
        db[1] = to_bf16x8(tds);
      }
    }
  };
  int s_qt = 0;  // query tile of the next step
  auto step = [&](const bf16_t* stage) {
    const int qr = s_qt * kQTile + 32 * qh;
    if (++s_qt == nqt) s_qt = 0;
    if (wave_active && qr < nq) compute(stage);
  };
  // After the barrier of step it every wave is done with step it - 1, whose stage then receives tile it + 2.
  for (int it = 0; it < n_iter; it += 3) {
    sync_stage();
    issue_next(it + 2 < n_iter, sS2);
    step(sS0);
    if (it + 1 >= n_iter) break;
    sync_stage();
    issue_next(it + 3 < n_iter, sS0);
    step(sS1);
    if (it + 2 >= n_iter) break;
    sync_stage();
    issue_next(it + 4 < n_iter, sS1);
    step(sS2);
  }
  wait_vmem();  // the copies past the last tile (with n_iter == 0 all of them) are still in flight

  // The second wave of each pair hands its partials over through LDS: blocks of 64 lanes x 16 bytes.
  auto blk = [&](int i) -> bf16_t* {
    bf16_t* const s = i < 2 ? sS0 : i < 4 ? sS1 : i < 6 ? sS2 : sV;
    return s + (i & 1) * L::kElems;
  };
  static_assert(L::kElems * 2 >= DT * 4 * 64 * 16, "a slice's dK or dV (fp32) fits one tile");
  __syncthreads();  // every wave is done with the stages
  f32x4* const pk = (f32x4*)blk(slice) + lane;
  f32x4* const pv = (f32x4*)blk(4 + slice) + lane;
  if (qh == 1) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int rq = 0; rq < 4; ++rq) {
        pk[(dt * 4 + rq) * 64] = f32x4{dkacc[dt][4 * rq], dkacc[dt][4 * rq + 1], dkacc[dt][4 * rq + 2], dkacc[dt][4 * rq + 3]};
        pv[(dt * 4 + rq) * 64] = f32x4{dvacc[dt][4 * rq], dvacc[dt][4 * rq + 1], dvacc[dt][4 * rq + 2], dvacc[dt][4 * rq + 3]};
      }
  }
  __syncthreads();
  if (qh != 0 || ka + l32 >= keys) return;
  const int64_t row = item.x + ka + l32;
  bf16_t* const krow = a.dk + row * a.dk_st + (int64_t)hk * a.dk_sh;
  bf16_t* const vrow = a.dv + row * a.dv_st + (int64_t)hk * a.dv_sh;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int rg = 0; rg < 4; ++rg) {
      const f32x4 k4 = pk[(dt * 4 + rg) * 64], v4 = pv[(dt * 4 + rg) * 64];
      f32x4 tk, tv;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        tk[e] = (dkacc[dt][4 * rg + e] + k4[e]) * a.scale;
        tv[e] = dvacc[dt][4 * rg + e] + v4[e];
      }
      *(bf16x4*)&krow[32 * dt + 8 * rg + 4 * hi] = __builtin_convertvector(tk, bf16x4);
      *(bf16x4*)&vrow[32 * dt + 8 * rg + 4 * hi] = __builtin_convertvector(tv, bf16x4);
    }
}

template <int D>
__global__ __attribute__((amdgpu_flat_work_group_size(kKvWaves * 64, kKvWaves * 64), amdgpu_waves_per_eu(2, 2))) void cross_dkdv_kernel(
    const CrossArgs a) {
  cross_dkdv_body<D>(a);
}
template __global__ void cross_dkdv_kernel<128>(const CrossArgs);

// head_dim 64: K and V fragments both fit the registers, and 4 waves of 32 states each take all 64 rows of
// a query tile: nothing to add up at the end, and three small workgroups per CU overlap each other's
// first loads and stores (48 documents of up to 700 queries over up to 1300 states, 8 heads: the scheme above 99 us, with
// one workgroup of 8 waves per CU).
constexpr int kSmallWaves = 4, kSmallPerSimd = 3;

__global__ __attribute__((amdgpu_flat_work_group_size(kSmallWaves * 64, kSmallWaves * 64), amdgpu_waves_per_eu(kSmallPerSimd, kSmallPerSimd)))
void cross_dkdv_d64_kernel(const CrossArgs a) {
  constexpr int D = 64, DT = D / 32, KS = D / 16;
  using L = TileLayout<D>;
  using Loader = TileLoader<D, kSmallWaves>;
  constexpr int kStageElems = 2 * L::kElems + 2 * kQTile * 2;  // Q, dO, lse2 + delta (fp32)
  __shared__ __attribute__((aligned(16))) bf16_t sS0[kStageElems];
  __shared__ __attribute__((aligned(16))) bf16_t sS1[kStageElems];
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31;
  const int hi = lane >> 5;
  const int rank = blockIdx.x / a.Hkv, hk = blockIdx.x - rank * a.Hkv;
  const int4 item = load_entry(a.plan_k, rank);
  const int keys = item.y, nq = item.w;
  if (keys == 0) return;  // list padding
  const int ka = wave * 32;
  const bool wave_active = ka < keys;
  const int nqt = (nq + kQTile - 1) / kQTile;
  const int n_iter = nqt * a.group;  // (query head, query tile) steps

  // Per tile the Q copy's last instruction is wave 0's, the dO copy's wave 1's; waves 2 and 3 copy the rows.
  static_assert(Loader::kInst == (Loader::kPerWave - 1) * kSmallWaves + 1, "one last-round copy per tile");
  const Loader ldq(a.q_st, wave, lane), ldo(a.do_st, wave, lane, 1);
  const int qh0 = hk * a.group;
  const bf16_t* q_head = a.q + (int64_t)item.z * a.q_st + (int64_t)qh0 * a.q_sh;
  const bf16_t* o_head = a.dout + (int64_t)item.z * a.do_st + (int64_t)qh0 * a.do_sh;
  const float* r_head = (wave == 2 ? a.lse2 : a.delta) + (int64_t)qh0 * a.Tq + item.z;
  const bf16_t* i_q = q_head;
  const bf16_t* i_o = o_head;
  const float* i_r = r_head;
  int i_qt = 0, i_rows = nq;
  auto issue_next = [&](bool valid, bf16_t* stage) {
    const int rows = valid ? min(i_rows, kQTile) : 0;
    ldq.issue_at(i_q, rows_bytes32(rows, (uint32_t)a.q_st, D), stage);
    ldo.issue_at(i_o, rows_bytes32(rows, (uint32_t)a.do_st, D), stage + L::kElems);
    float* const tr = (float*)(stage + 2 * L::kElems);
    const __amdgpu_buffer_rsrc_t r = make_rsrc(i_r, (uint32_t)rows * 4u);
    if (wave >= 2)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(tr + (wave == 2 ? 0 : kQTile)), 4,
                                               (uint32_t)lane * 4u, 0, 0, 0);
    if (++i_qt == nqt) {
      i_qt = 0;
      i_rows = nq;
      q_head += a.q_sh;
      o_head += a.do_sh;
      r_head += a.Tq;
      i_q = q_head;
      i_o = o_head;
      i_r = r_head;
    } else {
      i_rows -= kQTile;
      i_q += kQTile * a.q_st;
      i_o += kQTile * a.do_st;
      i_r += kQTile;
    }
  };
  issue_next(n_iter > 0, sS0);
  const __amdgpu_buffer_rsrc_t rk = make_rsrc(a.k + (int64_t)item.x * a.k_st + (int64_t)hk * a.k_sh, rows_bytes(keys, a.k_st, D));
  const __amdgpu_buffer_rsrc_t rv = make_rsrc(a.v + (int64_t)item.x * a.v_st + (int64_t)hk * a.v_sh, rows_bytes(keys, a.v_st, D));
  bf16x8 kf[KS], vf[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    kf[ks] = __builtin_bit_cast(bf16x8, buf_load16(rk, (uint32_t)(((ka + l32) * a.k_st + 16 * ks + 8 * hi) * 2)));
    vf[ks] = __builtin_bit_cast(bf16x8, buf_load16(rv, (uint32_t)(((ka + l32) * a.v_st + 16 * ks + 8 * hi) * 2)));
  }
  f32x16 dkacc[DT], dvacc[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) {
    dkacc[dt] = f32x16{};
    dvacc[dt] = f32x16{};
  }
  const float c2 = a.scale_log2;
  const TileLanes<D> tl(lane);

  auto compute = [&](const bf16_t* stage, int halves) {
    const bf16_t* const sQ = stage;
    const bf16_t* const sdO = stage + L::kElems;
    const float* const sL = (const float*)(stage + 2 * L::kElems);
    const float* const sD = sL + kQTile;
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {  // 32-row halves of the tile
      if (mt >= halves) break;
      f32x16 sc = f32x16{}, dp = f32x16{};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int o = tl.op_base + mt * 32 * L::kRowElems + ks * 16;
        sc = mfma32(*(const bf16x8*)&sQ[o], kf[ks], sc);
        dp = mfma32(*(const bf16x8*)&sdO[o], vf[ks], dp);
      }
      bf16x8 pb[2], db[2];
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2) {
        f32x8 tp, tds;
#pragma unroll
        for (int rg2 = 0; rg2 < 2; ++rg2) {
          const int qr0 = 32 * mt + 8 * (2 * s2 + rg2) + 4 * hi;
          const f32x4 l4 = *(const f32x4*)&sL[qr0], d4 = *(const f32x4*)&sD[qr0];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = 4 * (2 * s2 + rg2) + e;
            const float pr = fast_exp2(__builtin_fmaf(sc[r], c2, -l4[e]));
            tp[4 * rg2 + e] = pr;
            tds[4 * rg2 + e] = pr * (dp[r] - d4[e]);
          }
        }
        pb[s2] = to_bf16x8(tp);
        db[s2] = to_bf16x8(tds);
      }
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          const int o = tl.tr_base + (2 * mt + s2) * 16 * L::kRowElems + dt * 32;
          dvacc[dt] = mfma32(cat8(lds_read_tr16(&sdO[o]), lds_read_tr16(&sdO[o + L::kTrSecond])), pb[s2], dvacc[dt]);
          dkacc[dt] = mfma32(cat8(lds_read_tr16(&sQ[o]), lds_read_tr16(&sQ[o + L::kTrSecond])), db[s2], dkacc[dt]);
        }
    }
  };
  int s_qt = 0;  // query tile of the next step
  auto step = [&](const bf16_t* stage) {
    const int left = nq - s_qt * kQTile;
    if (++s_qt == nqt) s_qt = 0;
    if (wave_active) compute(stage, left > 32 ? 2 : 1);
  };
  for (int it = 0; it < n_iter; it += 2) {
    stage_barrier<0>();
    issue_next(it + 1 < n_iter, sS1);
    step(sS0);
    if (it + 1 >= n_iter) break;
    stage_barrier<0>();
    issue_next(it + 2 < n_iter, sS0);
    step(sS1);
  }
  wait_vmem();  // copies past the last tile are still in flight
  if (ka + l32 >= keys) return;
  const int64_t row = item.x + ka + l32;
  bf16_t* const krow = a.dk + row * a.dk_st + (int64_t)hk * a.dk_sh;
  bf16_t* const vrow = a.dv + row * a.dv_st + (int64_t)hk * a.dv_sh;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int rg = 0; rg < 4; ++rg) {
      f32x4 tk, tv;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        tk[e] = dkacc[dt][4 * rg + e] * a.scale;
        tv[e] = dvacc[dt][4 * rg + e];
      }
      *(bf16x4*)&krow[32 * dt + 8 * rg + 4 * hi] = __builtin_convertvector(tk, bf16x4);
      *(bf16x4*)&vrow[32 * dt + 8 * rg + 4 * hi] = __builtin_convertvector(tv, bf16x4);
    }
}

// ---------------------------------------------------------------------------
// dQ: the forward's S^T formulation, a query row in a lane, so lse2 and delta are local to it and dS^T is
// the B operand of dQ^T += K^T dS^T.  delta comes from the dO fragments that the kernel holds anyway and the same
// ones of O: a pass of its own over O and dO took 35 us beside the 800 of a training step of 8 x 2048 rows.
// ---------------------------------------------------------------------------
constexpr int kWaves = 4;
constexpr int kThreads = kWaves * 64;
constexpr int kBlockK = 64;

template <int D>
__device__ __forceinline__ void cross_dq_body(const CrossArgs& a) {
  constexpr int DT = D / 32;
  constexpr int KS = D / 16;
  using L = TileLayout<D>;
  __shared__ __attribute__((aligned(16))) bf16_t sK0[L::kElems];
  __shared__ __attribute__((aligned(16))) bf16_t sV0[L::kElems];
  __shared__ __attribute__((aligned(16))) bf16_t sK1[L::kElems];
  __shared__ __attribute__((aligned(16))) bf16_t sV1[L::kElems];
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31;
  const int hi = lane >> 5;
  const QueryTile tile = query_tile(a);
  const int4 item = tile.item;
  const int h = tile.h, hk = tile.hk, rows = item.y, nk = item.w;
  if (rows == 0) return;  // list padding
  const int nkt = (nk + kBlockK - 1) / kBlockK;
  const int qa = wave * 32;
  const bool wave_active = qa < rows;
  const int qrow = qa + l32;

  const __amdgpu_buffer_rsrc_t rq = make_rsrc(a.q + (int64_t)item.x * a.q_st + (int64_t)h * a.q_sh, rows_bytes(rows, a.q_st, D));
  const __amdgpu_buffer_rsrc_t rdo = make_rsrc(a.dout + (int64_t)item.x * a.do_st + (int64_t)h * a.do_sh, rows_bytes(rows, a.do_st, D));
  const TileLoader<D, kWaves> ldk(a.k_st, wave, lane), ldv(a.v_st, wave, lane);
  const bf16_t* i_k = a.k + (int64_t)item.z * a.k_st + (int64_t)hk * a.k_sh;
  const bf16_t* const i_v0 = a.v + (int64_t)item.z * a.v_st + (int64_t)hk * a.v_sh;
  const bf16_t* i_v = i_v0;
  int i_rows = nk;
  auto issue_next = [&](bf16_t* tk, bf16_t* tv) {
    const int n = min(i_rows, kBlockK);
    ldk.issue_at(i_k, rows_bytes32(n, (uint32_t)a.k_st, D), tk);
    ldv.issue_at(i_v, rows_bytes32(n, (uint32_t)a.v_st, D), tv);
    i_k += kBlockK * a.k_st;
    i_v += kBlockK * a.v_st;
    i_rows -= kBlockK;
  };
  if (nkt > 0) issue_next(sK0, sV0);
  bf16x8 qf[KS], dof[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    qf[ks] = __builtin_bit_cast(bf16x8, buf_load16(rq, (uint32_t)((qrow * a.q_st + 16 * ks + 8 * hi) * 2)));
    dof[ks] = __builtin_bit_cast(bf16x8, buf_load16(rdo, (uint32_t)((qrow * a.do_st + 16 * ks + 8 * hi) * 2)));
  }
  const int64_t row_at = (int64_t)h * a.Tq + item.x + qrow;
  const float lse2 = qrow < rows ? a.lse2[row_at] : 0.f;
  float dlt = 0.f;
  {
    const __amdgpu_buffer_rsrc_t ro = make_rsrc(a.o + (int64_t)item.x * a.o_st + (int64_t)h * a.o_sh, rows_bytes(rows, a.o_st, D));
    const int64_t lo_st = (int64_t)a.Hq * D;
    const __amdgpu_buffer_rsrc_t rl = make_rsrc(a.o_lo + (int64_t)item.x * lo_st + (int64_t)h * D, rows_bytes(rows, lo_st, D));
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const bf16x8 ov = __builtin_bit_cast(bf16x8, buf_load16(ro, (uint32_t)((qrow * a.o_st + 16 * ks + 8 * hi) * 2)));
      const bf16x8 lv = __builtin_bit_cast(bf16x8, buf_load16(rl, (uint32_t)((qrow * lo_st + 16 * ks + 8 * hi) * 2)));
#pragma unroll
      for (int e = 0; e < 8; ++e) dlt += ((float)ov[e] + (float)lv[e]) * (float)dof[ks][e];
    }
    dlt = xor32_sum(dlt);
    if (nk == 1) {
      // One state: O is its value and delta is dP, so dS = 0.  Taken from the product that dP comes from, here and in the
      // dK / dV kernel, that holds exactly, and not to the rounding of two sums.
      const __amdgpu_buffer_rsrc_t rv = make_rsrc(i_v0, rows_bytes(1, a.v_st, D));
      f32x16 one = f32x16{};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        one = mfma32(__builtin_bit_cast(bf16x8, buf_load16(rv, (uint32_t)((l32 * a.v_st + 16 * ks + 8 * hi) * 2))), dof[ks], one);
      dlt = __shfl(one[0], l32, 64);  // state 0 is the first half's
    }
    if (hi == 0 && qrow < rows) a.delta[row_at] = dlt;
  }
  f32x16 dqacc[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) dqacc[dt] = f32x16{};
  const float c2 = a.scale_log2;
  const TileLanes<D> tl(lane);

  // kSteps 32-state halves at a time: both at head_dim 128, whose MFMAs then run beside more independent work, one
  // at head_dim 64, where half the scores let four waves share a SIMD.
  constexpr int kSteps = D == 64 ? 1 : 2;
  auto compute = [&](int kt, const bf16_t* sK, const bf16_t* sV) {
#pragma unroll
    for (int m0 = 0; m0 < 2; m0 += kSteps) {
      f32x16 st[kSteps], dpt[kSteps];
#pragma unroll
      for (int mt = 0; mt < kSteps; ++mt) {
        st[mt] = f32x16{};
        dpt[mt] = f32x16{};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const int o = tl.op_base + (m0 + mt) * 32 * L::kRowElems + ks * 16;
          st[mt] = mfma32(*(const bf16x8*)&sK[o], qf[ks], st[mt]);
          dpt[mt] = mfma32(*(const bf16x8*)&sV[o], dof[ks], dpt[mt]);
        }
      }
      if (kt * kBlockK + kBlockK > nk) {  // no P past the states: exp2(0 - lse2) may overflow
        __asm__ volatile("");
        const int left = nk - kt * kBlockK - 32 * m0 - 4 * hi;
#pragma unroll
        for (int mt = 0; mt < kSteps; ++mt)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (32 * mt + 8 * (r >> 2) + (r & 3) >= left) st[mt][r] = -INFINITY;
      }
      bf16x8 sf[2 * kSteps];
#pragma unroll
      for (int kk = 0; kk < 2 * kSteps; ++kk) {
        f32x8 t;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int mt = kk >> 1, r = (kk & 1) * 8 + e;
          t[e] = fast_exp2(__builtin_fmaf(st[mt][r], c2, -lse2)) * (dpt[mt][r] - dlt);
        }
        sf[kk] = to_bf16x8(t);
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int kk = 0; kk < 2 * kSteps; ++kk) {
          const bf16_t* kp = &sK[tl.tr_base + (2 * m0 + kk) * 16 * L::kRowElems + dt * 32];
          dqacc[dt] = mfma32(cat8(lds_read_tr16(kp), lds_read_tr16(kp + L::kTrSecond)), sf[kk], dqacc[dt]);
        }
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

  // Each wave stages its rows in one K / V stage object and stores whole rows.
  __syncthreads();
  if (!wave_active) return;
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
      for (int e = 0; e < 4; ++e) t[e] = dqacc[dt][4 * rg + e] * a.scale;
      *(bf16x4*)&stage[l32 * kPitch + 32 * dt + 8 * rg + 4 * hi] = __builtin_convertvector(t, bf16x4);
    }
  __asm__ volatile("" ::: "memory");  // the LDS unit runs one wave's accesses in order
  const int u = lane % kUnits;
  bf16_t* const dbase = a.dq + (int64_t)(item.x + qa) * a.dq_st + (int64_t)h * a.dq_sh + u * 8;
#pragma unroll
  for (int j = 0; j < 32 / kRowsPerInst; ++j) {
    const int r = j * kRowsPerInst + lane / kUnits;
    const bf16x8 v = *(const bf16x8*)&stage[r * kPitch + u * 8];
    if (qa + r < rows) *(bf16x8*)&dbase[(int64_t)r * a.dq_st] = v;
  }
}

template <int D>
constexpr int kDqWaves = D == 64 ? 4 : 2;  // waves per SIMD = workgroups per CU
template <int D>
__global__ __attribute__((amdgpu_flat_work_group_size(kThreads, kThreads), amdgpu_waves_per_eu(kDqWaves<D>, kDqWaves<D>))) void cross_dq_kernel(
    const CrossArgs a) {
  cross_dq_body<D>(a);
}
template __global__ void cross_dq_kernel<64>(const CrossArgs);
template __global__ void cross_dq_kernel<128>(const CrossArgs);

}  // namespace

hipError_t launch_cross_bwd(const CrossArgs& a, int head_dim, hipStream_t stream) {
  const int64_t units = (int64_t)a.cap_q * a.Hkv;
  if (units > 0) {
    const dim3 grid((unsigned)((units + kXcds - 1) / kXcds * kXcds * a.group));
    if (head_dim == 128)
      hipLaunchKernelGGL(cross_dq_kernel<128>, grid, dim3(kThreads), 0, stream, a);
    else
      hipLaunchKernelGGL(cross_dq_kernel<64>, grid, dim3(kThreads), 0, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if (a.cap_k == 0) return hipSuccess;
  const dim3 grid((unsigned)a.cap_k * (unsigned)a.Hkv);
  if (head_dim == 128)
    hipLaunchKernelGGL(cross_dkdv_kernel<128>, grid, dim3(kKvWaves * 64), 0, stream, a);
  else
    hipLaunchKernelGGL(cross_dkdv_d64_kernel, grid, dim3(kSmallWaves * 64), 0, stream, a);
  return hipGetLastError();
}

}  // namespace mimir
