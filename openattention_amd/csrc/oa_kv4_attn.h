// What the attention kernels over the 4-bit paged cache share: arguments, a sequence's rows and lengths, codes
// to bf16.
#pragma once
#include <cfloat>
#include <type_traits>

#include "oa_common.h"

namespace kv4 {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef unsigned int uint4v __attribute__((ext_vector_type(4)));
typedef unsigned int uint2v __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) short4v lds_short4v;

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * 64;
constexpr int kTile = 32;                // keys per tile
constexpr float kLog2e = 1.4426950408889634f;

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

// what a sequence asks: its rows and how many keys they see
struct Seq {
  int n, r0, R;
  bool bad;                              // more keys than the table or the call covers
};

__device__ __forceinline__ Seq seq_of(const AttnArgs& a, int b) {
  Seq s;
  s.n = max(a.lens[b], 0);
  s.r0 = a.cu ? a.cu[b] : b;
  const int r1 = a.cu ? a.cu[b + 1] : b + 1;
  s.R = s.r0 < 0 || r1 < s.r0 || r1 > a.tokens ? 0 : r1 - s.r0;         // (starts that do not fit the rows: none)
  s.bad = (long)s.n > min((long)a.width << a.lp, (long)a.nchunk * a.chunk);
  return s;
}

__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const f32x2 x = {a, b};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(x, bf16x2));
}
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
// An entry of a table's row, the same for all lanes, by a vector load: scalar loads come back in no order, and
// beside one in flight every wait for LDS waits for all of it.
__device__ __forceinline__ int table_entry(const int* row, int i) {
  int zero;
  asm("v_mov_b32 %0, 0" : "=v"(zero));
  return row[i + zero];
}

// NQ tiles of 16 rows for each workgroup, the waves on keys of their own (oa_kv4_attn.hip), or 128 rows, 32 to a
// wave, over shared keys (oa_kv4_rows.hip)
void launch_rows(const AttnArgs& a, int head_dim, dim3 grid, hipStream_t st);

}  // namespace kv4
