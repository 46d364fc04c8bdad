// What the kernels of the 8-bit paged cache share: the call, a batch row's place in
// the page table, and the 8-bit codes.
//
// A page holds 64 tokens of every kv head.  Keys lie [token][D], values [D][token]: the
// products read 16 consecutive columns of a key and 16 consecutive tokens of a value
// column, so both operands of the matrix instructions come straight from 16-byte
// loads, without a transpose.  A code times 2^exponent is exact in bf16 (4 significant
// bits, exponents of at least -100 - 9), and the conversion instruction multiplies by a power
// of two on the way, so scaling costs nothing and rounds nothing.
#pragma once

#include "prefixlm_common.h"

namespace mimir {

constexpr int kPage = MIMIR_PAGE_TOKENS;
constexpr int kMinExponent = -100;

struct PagedArgs {
  const bf16_t *q, *kn, *vn;
  bf16_t* out;
  uint8_t *ck, *cv;
  int8_t *ke, *ve;
  const int32_t* table;
  const void *lengths, *indices, *fresh;  // int32 or int64 (idx64); the last two may be null
  int64_t q_sb, q_st, q_sh, kn_sb, kn_st, kn_sh, vn_sb, vn_st, vn_sh, o_sb, o_st, o_sh;
  int64_t k_sp, v_sp, ke_sp, ve_sp, t_st;
  int B, S, num_pages, rows, width, Hkv, G, causal, D, idx64;
  float scale_log2;
  float *part_o, *part_ml;  // partial rows: unnormalized O [D]; maximum (exp2 domain) and sum
  int shares;               // decode: runs of pages, one workgroup per kv head each
  int n_rt, splits, cus;    // prefill: row tiles per (batch row, kv head), key splits of each
  int slots;                // prefill of a padded batch: workgroups to deal its pages to; 0: the splits above
};

__device__ __forceinline__ int64_t paged_index(const void* p, int i, int idx64) {
  return idx64 ? ((const int64_t*)p)[i] : (int64_t)((const int32_t*)p)[i];
}

// A batch row: its table row (-1: outside), tokens held before the call (n), new ones (m) and
// keys to attend (kv; 0 if there is nothing to do).
struct PagedRow {
  int row, n, m, kv;
  __device__ __forceinline__ PagedRow() {}
  __device__ __forceinline__ PagedRow(const PagedArgs& a, int b) {
    const int64_t r = a.indices != nullptr ? paged_index(a.indices, b, a.idx64) : b;
    const int64_t c = paged_index(a.lengths, b, a.idx64);
    const int64_t f = a.fresh != nullptr ? paged_index(a.fresh, b, a.idx64) : a.S;
    const int most = a.width * kPage;
    row = r >= 0 && r < a.rows ? (int)r : -1;
    n = c > most ? most : (int)c;
    m = row < 0 || c < 0 || f < 0 ? 0 : (f > a.S ? a.S : (int)f);
    kv = m > 0 ? min(n + m, most) : 0;
  }
};

// The page of a row's places [64 i, 64 i + 64), -1 if there is none.
__device__ __forceinline__ int page_id(const PagedArgs& a, int row, int i) {
  const int p = a.table[(int64_t)row * a.t_st + i];
  return p >= 0 && p < a.num_pages ? p : -1;
}

// 2^e as a float, e in [-126, 127].
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }

// Eight codes (two words) times `scale`, a power of two, as bf16.
__device__ __forceinline__ bf16x8 decode8(int lo, int hi, float scale) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Non-zero where one of four codes is NaN (all of its lower seven bits set).
__device__ __forceinline__ unsigned nan_codes(int x) { return (((unsigned)x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// A word of four value codes of tokens t.. with those of tokens >= end cleared: what lies
// behind a row's last token is unwritten, and any NaN there would spoil the product.
__device__ __forceinline__ int codes_before(int x, int t, int end) {
  const int n = end - t;
  return n >= 4 ? x : (n <= 0 ? 0 : x & (int)((1u << (8 * n)) - 1));
}

// The exponent that the largest finite magnitude needs, from its bf16 bits (448 = 1.75 * 2^8).
__device__ __forceinline__ int exponent_for(int bits) {
  const int e = (bits >> 7) - 127 - 8 + ((bits & 0x7f) > 96);
  return e > kMinExponent ? e : kMinExponent;
}

// The largest finite magnitude of eight bf16 values, as bits.
__device__ __forceinline__ int largest_bits(i32x4 words) {
  int most = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int bits = words[e >> 1] >> (16 * (e & 1)) & 0x7fff;
    most = max(most, bits < 0x7f80 ? bits : 0);
  }
  return most;
}

// x / 2^e rounded to e4m3, four values to a word; infinities become NaN.
__device__ __forceinline__ float coded_value(float x, int e) {
  return __builtin_fabsf(x) <= 3.4028235e38f ? __builtin_amdgcn_ldexpf(x, -e) : __builtin_nanf("");
}
__device__ __forceinline__ int encode4(float a, float b, float c, float d) {
  int x = __builtin_nondeterministic_value(x);  // both halves are written below
  x = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, x, false);
  return __builtin_amdgcn_cvt_pk_fp8_f32(c, d, x, true);
}
// Four codes times 2^shift, rounded to codes again.
__device__ __forceinline__ int recode4(int x, int shift) {
  const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(x, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(x, true);
  return encode4(__builtin_amdgcn_ldexpf(lo[0], shift), __builtin_amdgcn_ldexpf(lo[1], shift),
                 __builtin_amdgcn_ldexpf(hi[0], shift), __builtin_amdgcn_ldexpf(hi[1], shift));
}

hipError_t launch_paged_append(const PagedArgs& a, hipStream_t stream);

}  // namespace mimir
