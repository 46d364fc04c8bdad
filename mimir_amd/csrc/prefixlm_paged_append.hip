// New keys / values into the pages of an 8-bit cache, for gfx950.
//
// One workgroup per (batch row, kv head, page that gets new tokens), for keys and for
// values each.  The page and head take the smallest exponent e with |x| <= 448 * 2^e for
// the new values, but not less than the one they have for older tokens, whose codes are
// rounded again where e grew.  With scales of powers of two that costs them nothing
// but the bits that fall below 2^(e - 9): an 8-bit float keeps its three fraction bits, so a finer
// scale would not make the others more exact either.
//
// Reads the new rows (bf16) and writes their codes; the page's older codes are touched only where the
// exponent grew.  8 x 512 tokens, 4 heads of 128 (13 MB): 7 us, where a copy's rate gives 2.5: bound by its
// chain of round trips (arguments, lengths, page id and rows, exponent, codes).  Values are turned to [D][token] through LDS.
#include "prefixlm_paged.h"

namespace mimir {
namespace {

constexpr int kThreads = 256;

template <int D>
__device__ __forceinline__ void paged_append_body(const PagedArgs& a, int touched) {
  constexpr int kUnits = D / 8;                  // threads of a row
  constexpr int kStep = kThreads / kUnits;       // rows at a time
  constexpr int kPasses = kPage / kStep;
  constexpr int kPitch = D + 4;
  __shared__ uint8_t codes[kPage * kPitch];
  __shared__ int top[kThreads / 64];
  touch_args<sizeof(PagedArgs)>();
  const int tid = threadIdx.x;
  int u = blockIdx.x;
  const int j = u % touched;
  u /= touched;
  const int hk = u % a.Hkv, b = u / a.Hkv;
  const bool values = blockIdx.y == 1;
  const PagedRow r(a, b);
  if (r.m == 0) return;
  const int at = r.n / kPage + j;                // of the row's pages
  const int lo = max(r.n, at * kPage), hi = min(r.n + r.m, min(at + 1, a.width) * kPage);
  if (lo >= hi) return;
  const int page = page_id(a, r.row, at);  // looked at below, when the rows are on their way
  const int s0 = lo - at * kPage, s1 = hi - at * kPage;  // slots of the new tokens
  const bf16_t* const x = values ? a.vn + (int64_t)b * a.vn_sb + (int64_t)hk * a.vn_sh + (int64_t)(lo - r.n) * a.vn_st
                                 : a.kn + (int64_t)b * a.kn_sb + (int64_t)hk * a.kn_sh + (int64_t)(lo - r.n) * a.kn_st;
  const int64_t x_st = values ? a.vn_st : a.kn_st;
  const int row = tid / kUnits, c = tid % kUnits * 8;
  bf16x8 v[kPasses];
  int most = 0;
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int t = p * kStep + row;
    v[p] = bf16x8{};
    if (t < s1 - s0) v[p] = *(const bf16x8*)&x[(int64_t)t * x_st + c];
  }
  if (page < 0) return;
  uint8_t* const y = values ? a.cv + page * a.v_sp + (int64_t)hk * kPage * D : a.ck + page * a.k_sp + (int64_t)hk * kPage * D;
  int8_t* const ey = values ? a.ve + page * a.ve_sp + hk : a.ke + page * a.ke_sp + hk;
  const int had = s0 > 0 ? *ey : kMinExponent;
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    most = max(most, largest_bits(__builtin_bit_cast(i32x4, v[p])));
  }
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) most = max(most, __shfl_xor(most, off, 64));
  if ((tid & 63) == 0) top[tid >> 6] = most;
  __syncthreads();  // and every thread has read the old exponent
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) most = max(most, top[w]);
  const int need = exponent_for(most);
  const int e = s0 > 0 ? max(had, need) : need;
  const int shift = had - e;
  const bool grew = s0 > 0 && shift < 0;
  if (tid == 0) *ey = (int8_t)e;

#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int t = p * kStep + row;
    if (t >= s1 - s0) break;
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = coded_value((float)v[p][i], e);
    const i32x2 w = {encode4(f[0], f[1], f[2], f[3]), encode4(f[4], f[5], f[6], f[7])};
    if (values) {
      *(int*)&codes[(s0 + t) * kPitch + c] = w[0];
      *(int*)&codes[(s0 + t) * kPitch + c + 4] = w[1];
    } else {
      *(i32x2*)&y[(s0 + t) * D + c] = w;
    }
  }
  if (!values) {
    if (grew)
      for (int i = tid * 4; i < s0 * D; i += kThreads * 4) *(int*)&y[i] = recode4(*(const int*)&y[i], shift);
    return;
  }
  __syncthreads();
  // Words of four tokens of four columns at a time: four words of codes, a token each, turned by byte
  // permutes (byte by byte out of LDS, a chunk's launch took 9.3 us; so 6).
  const int w0 = grew ? 0 : s0 / 4, words = (s1 + 3) / 4 - w0;  // words to write, of each column
  for (int i = tid; i < D / 4 * words; i += kThreads) {
    const int q = i / words, t = (i - q * words + w0) * 4;  // columns 4 q ..+3, tokens t ..+3
    unsigned in[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) in[e] = *(const unsigned*)&codes[(t + e) * kPitch + 4 * q];
    const unsigned a01 = __builtin_amdgcn_perm(in[1], in[0], 0x05010400), a23 = __builtin_amdgcn_perm(in[3], in[2], 0x05010400);
    const unsigned b01 = __builtin_amdgcn_perm(in[1], in[0], 0x07030602), b23 = __builtin_amdgcn_perm(in[3], in[2], 0x07030602);
    const unsigned turned[4] = {__builtin_amdgcn_perm(a23, a01, 0x05040100), __builtin_amdgcn_perm(a23, a01, 0x07060302),
                                __builtin_amdgcn_perm(b23, b01, 0x05040100), __builtin_amdgcn_perm(b23, b01, 0x07060302)};
    // bytes of new tokens; the older ones are rounded again where the exponent grew, the others stay
    const int lo = s0 - t, hi_end = s1 - t;
    const unsigned from = lo <= 0 ? ~0u : (lo >= 4 ? 0u : ~0u << (8 * lo)), until = hi_end >= 4 ? ~0u : (1u << (8 * hi_end)) - 1;
    const unsigned fresh = from & until;
#pragma unroll
    for (int c2 = 0; c2 < 4; ++c2) {
      unsigned* const at4 = (unsigned*)&y[(4 * q + c2) * kPage + t];
      unsigned out = turned[c2];
      if (fresh != ~0u) {
        const unsigned old = *at4, kept = grew ? ((unsigned)recode4((int)old, shift) & ~from) | (old & from) : old;
        out = (out & fresh) | (kept & ~fresh);
      }
      *at4 = out;
    }
  }
}

__global__ __launch_bounds__(kThreads) void paged_append_d128_kernel(const PagedArgs a, int touched) {
  paged_append_body<128>(a, touched);
}
__global__ __launch_bounds__(kThreads) void paged_append_d64_kernel(const PagedArgs a, int touched) {
  paged_append_body<64>(a, touched);
}

}  // namespace

hipError_t launch_paged_append(const PagedArgs& a, hipStream_t stream) {
  const int touched = (a.S + 2 * kPage - 2) / kPage;  // pages that S tokens may fall in
  const dim3 grid((unsigned)((int64_t)a.B * a.Hkv * touched), 2);
  if (a.D == 128)
    hipLaunchKernelGGL(paged_append_d128_kernel, grid, dim3(kThreads), 0, stream, a, touched);
  else
    hipLaunchKernelGGL(paged_append_d64_kernel, grid, dim3(kThreads), 0, stream, a, touched);
  return hipGetLastError();
}

}  // namespace mimir
