// Query and key rows of a layer: each head's RMS norm and its rotation to the token's position in one
// pass, y = x / sqrt(mean(x^2) + eps) * w, then (y_i, y_(i + D/2)) turned by the angle of pair i:
//   out_i = y_i cos_i - y_(i + D/2) sin_i,   out_(i + D/2) = y_(i + D/2) cos_i + y_i sin_i,
// in fp32, rounded once to the rows' type.  A lane holds 8 dims of each half, so that every pair is in
// one lane and D / 16 lanes are a head: one reduction over 4, 8 or 16 lanes, and loads and stores of 16
// bytes.  The flat map of (token, head) to lanes keeps every lane at work for any number of heads.
// Bound by the rows read and written: 32767 tokens of 40 heads of 128, bf16, 671 MB, 114 us, 5.9 TB/s (a
// large copy moves 5.2); 32 tokens 2.9 us, one launch.  Stores pass by the caches (115 us; 120 through them).
#include "oa_common.h"

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x8m __attribute__((ext_vector_type(8), aligned(16)));    // in memory

template <typename T> struct Vec8;
template <> struct Vec8<__bf16> { typedef bf16x8 type; };
template <> struct Vec8<_Float16> { typedef f16x8 type; };
template <> struct Vec8<float> { typedef f32x8m type; };

constexpr int kThreads = 256;

struct RopeArgs {
  const void* q; long q_st, q_sh;
  const void* k; long k_st, k_sh;
  void* qo; long qo_st, qo_sh;
  void* ko; long ko_st, ko_sh;
  const void* wq; const void* wk;
  const void* pos;
  const float* cos_t; const float* sin_t; long cs_st;
  unsigned units, heads, q_heads;        // (token, head) pairs; heads of a token, query heads first
  int pos64, P;
  float eps;
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) qk_norm_rope_kernel(RopeArgs a) {
  constexpr int kLanes = D / 16;         // lanes of a head
  typedef typename Vec8<T>::type vec;
  const unsigned idx = blockIdx.x * kThreads + threadIdx.x;
  const unsigned u0 = idx / kLanes, lh = idx % kLanes;
  const bool live = u0 < a.units;
  const unsigned u = live ? u0 : a.units - 1;      // (lanes past the end repeat the last head, unstored)
  const unsigned tok = u / a.heads, hd = u - tok * a.heads;
  const bool isq = hd < a.q_heads;
  const T* x = isq ? (const T*)a.q + (long)tok * a.q_st + (long)hd * a.q_sh
                   : (const T*)a.k + (long)tok * a.k_st + (long)(hd - a.q_heads) * a.k_sh;
  const f32x8 lo = __builtin_convertvector(*reinterpret_cast<const vec*>(x + 8 * lh), f32x8);
  const f32x8 hi = __builtin_convertvector(*reinterpret_cast<const vec*>(x + D / 2 + 8 * lh), f32x8);
  const long p = a.pos64 ? ((const long*)a.pos)[tok] : (long)((const int*)a.pos)[tok];
  const long pc = min(max(p, 0l), (long)a.P - 1);
  const float* cr = a.cos_t + pc * a.cs_st + 8 * lh;
  const float* sr = a.sin_t + pc * a.cs_st + 8 * lh;
  const f32x8 c = *reinterpret_cast<const f32x8m*>(cr), s = *reinterpret_cast<const f32x8m*>(sr);
  const T* w = (const T*)(isq ? a.wq : a.wk);
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) ss = fmaf(lo[i], lo[i], fmaf(hi[i], hi[i], ss));
  ss += oa::dpp_f32<0xB1>(ss);
  ss += oa::dpp_f32<0x4E>(ss);
  if (kLanes > 4) ss += oa::dpp_f32<0x141>(ss);
  if (kLanes > 8) ss += oa::dpp_f32<0x140>(ss);
  f32x8 y0 = lo, y1 = hi;
  if (w) {
    const float r = 1.f / sqrtf(ss * (1.f / D) + a.eps);
    const f32x8 w0 = __builtin_convertvector(*reinterpret_cast<const vec*>(w + 8 * lh), f32x8);
    const f32x8 w1 = __builtin_convertvector(*reinterpret_cast<const vec*>(w + D / 2 + 8 * lh), f32x8);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      y0[i] = lo[i] * r * w0[i];
      y1[i] = hi[i] * r * w1[i];
    }
  }
  f32x8 o0, o1;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    o0[i] = y0[i] * c[i] - y1[i] * s[i];
    o1[i] = y1[i] * c[i] + y0[i] * s[i];
  }
  if (p < 0 || p >= a.P) {               // padding: zeros; a position past the tables: NaN
    const float e = p < 0 ? 0.f : __builtin_nanf("");
    o0 = f32x8(e);
    o1 = f32x8(e);
  }
  if (!live) return;
  T* o = isq ? (T*)a.qo + (long)tok * a.qo_st + (long)hd * a.qo_sh
             : (T*)a.ko + (long)tok * a.ko_st + (long)(hd - a.q_heads) * a.ko_sh;
  __builtin_nontemporal_store(__builtin_convertvector(o0, vec), reinterpret_cast<vec*>(o + 8 * lh));
  __builtin_nontemporal_store(__builtin_convertvector(o1, vec), reinterpret_cast<vec*>(o + D / 2 + 8 * lh));
}

template <typename T>
int launch(const RopeArgs& a, int D, hipStream_t st) {
  const unsigned blocks = (unsigned)(((long)a.units * (D / 16) + kThreads - 1) / kThreads);
  switch (D) {
    case 64: hipLaunchKernelGGL((qk_norm_rope_kernel<T, 64>), dim3(blocks), dim3(kThreads), 0, st, a); break;
    case 128: hipLaunchKernelGGL((qk_norm_rope_kernel<T, 128>), dim3(blocks), dim3(kThreads), 0, st, a); break;
    default: hipLaunchKernelGGL((qk_norm_rope_kernel<T, 256>), dim3(blocks), dim3(kThreads), 0, st, a); break;
  }
  return OA_LAUNCH_STATUS();
}

}  // namespace

extern "C" int oa_qk_norm_rope(const void* q, long q_st, long q_sh, const void* k, long k_st, long k_sh, int tokens,
                               int q_heads, int kv_heads, int head_dim, int dtype, const void* pos, int pos_is_64,
                               const float* cos_t, const float* sin_t, long table_stride, int positions,
                               const void* wq, const void* wk, float eps, void* q_out, long qo_st, long qo_sh,
                               void* k_out, long ko_st, long ko_sh, void* stream) {
  if (dtype < 0 || dtype > 2 || (head_dim != 64 && head_dim != 128 && head_dim != 256)) return OA_EINVAL;
  if (tokens < 0 || q_heads < 0 || kv_heads < 0 || positions <= 0 || !(eps >= 0.f) || table_stride % 4) return OA_EINVAL;
  const long units = (long)tokens * ((long)q_heads + kv_heads);
  if (units == 0) return 0;
  if (units > (1L << 27)) return OA_EINVAL;        // (thread indices are 32 bits: units * 16 lanes)
  const int align = dtype == 2 ? 4 : 8;
  auto bad = [&](const void* p, long st, long sh) {
    return !p || (reinterpret_cast<uintptr_t>(p) & 15) || st % align || sh % align;
  };
  auto odd = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; };
  if ((q_heads && (bad(q, q_st, q_sh) || bad(q_out, qo_st, qo_sh))) ||
      (kv_heads && (bad(k, k_st, k_sh) || bad(k_out, ko_st, ko_sh))) || odd(wq) || odd(wk) || !cos_t || !sin_t ||
      odd(cos_t) || odd(sin_t) || !pos)
    return OA_EINVAL;
  RopeArgs a;
  a.q = q; a.q_st = q_st; a.q_sh = q_sh;
  a.k = k; a.k_st = k_st; a.k_sh = k_sh;
  a.qo = q_out; a.qo_st = qo_st; a.qo_sh = qo_sh;
  a.ko = k_out; a.ko_st = ko_st; a.ko_sh = ko_sh;
  a.wq = wq; a.wk = wk; a.pos = pos; a.pos64 = pos_is_64; a.P = positions;
  a.cos_t = cos_t; a.sin_t = sin_t; a.cs_st = table_stride;
  a.units = (unsigned)units; a.heads = (unsigned)(q_heads + kv_heads); a.q_heads = (unsigned)q_heads;
  a.eps = eps;
  const hipStream_t st = (hipStream_t)stream;
  return dtype == 0 ? launch<__bf16>(a, head_dim, st) : dtype == 1 ? launch<_Float16>(a, head_dim, st)
                                                                   : launch<float>(a, head_dim, st);
}
