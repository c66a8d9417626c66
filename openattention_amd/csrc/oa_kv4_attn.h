// What the attention kernels over the 4-bit paged cache share: arguments, codes to bf16.
#pragma once
#include "oa_paged_attn.h"

namespace kv4 {

using namespace paged;

struct AttnArgs {
  const uint16_t* q; long q_st, q_sh;
  const uint8_t* kc; const uint8_t* ks; const uint8_t* vc; const uint8_t* vs;
  long c_sp, s_sp;                       // bytes between pages
  const int* table; long t_st;
  const int* lens; const int* cu;
  uint16_t* out; long o_st, o_sh;
  float* ws_o; float* ws_ml;             // partial sums, (maximum, sum) by (row, chunk)
  int* ws_flag;                          // by workgroup of oa_kv4_rows.hip
  int B, HKV, G, tokens, max_q, width, NP, lp, chunk, nchunk, ntile;
  unsigned by_g, by_hkv;                 // 2^16 / G + 1; 2^32 / HKV, rounded up (0: HKV is 1)
  int clear;                             // the join sets rows of out that no sequence takes to 0
  float c;                               // scale * log2 e
};

// 8 codes to bf16, scaled by a power of two (all exponent bits set, a scale byte of 255: NaN)
__device__ __forceinline__ bf16x8 from4(unsigned w, float f) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, f, 0);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, f, 1);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, f, 2);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, f, 3);
  const uint4v x = {__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b), __builtin_bit_cast(uint32_t, c),
                    __builtin_bit_cast(uint32_t, d)};
  return __builtin_bit_cast(bf16x8, x);
}
// NQ tiles of 16 rows for each workgroup, the waves on keys of their own (oa_kv4_attn.hip), or 128 rows, 32 to a
// wave, over shared keys (oa_kv4_rows.hip)
void launch_rows(const AttnArgs& a, int head_dim, dim3 grid, hipStream_t st);

}  // namespace kv4
