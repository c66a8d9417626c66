// The 4-bit paged KV cache: rows rounded into it (oa_kv4_write) and read back from it (oa_kv4_read).
//
// A row of a head is held as D / 32 blocks of 32 values: a 4-bit code for each (sign, two bits of
// exponent, one of mantissa: 0, .5, 1, 1.5, 2, 3, 4, 6) and one byte s per block that scales them by
// 2^(s - 127).  2^e is the smallest power of two with max |x| < 7 * 2^e (7 is where the top code would
// round to 8), -125 <= e <= 125, which keeps every value that a code can stand for, down to 0.5 * 2^e, a
// normal fp32 and bf16 number; rounding is to nearest, ties to the even code, at most 6.  A scale that
// is a power of two makes both directions exact but for that one rounding.  Blocks with a value that is
// not finite are held as s = 255: NaN.
// Layout: codes (pages, heads, page, D / 2), scales (pages, heads, page, D / 32), bytes; slot = page id
// * page + offset.
//
// A lane takes 8 values of a row of K and of V (16 bytes of bf16, 4 of codes), four lanes a block, a workgroup one
// head for 16 or 32 successive tokens: where their slots follow each other, as a prompt's do, codes and scales
// are whole lines (by token, all its heads together, writing and reading 32767 tokens took 85 us; K and V by
// workgroups of their own 61; two or four tokens to a lane 58 and 60).
// Bound by the bytes moved: 32767 tokens of 8 heads of 128 in bf16, 170 MB each way, 32 us written (5.3 TB/s) and
// 25 us read back (6.7 TB/s), 58 together; 32 tokens 2.6 us each.  What passes once (rows in, values out) passes
// by the caches (through them 8 us more; codes past the caches too: 12).
#include "oa_common.h"

namespace {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x8m __attribute__((ext_vector_type(8), aligned(16)));    // in memory

template <typename T> struct Vec8;
template <> struct Vec8<__bf16> { typedef bf16x8 type; };
template <> struct Vec8<_Float16> { typedef f16x8 type; };
template <> struct Vec8<float> { typedef f32x8m type; };

constexpr int kThreads = 256;

struct Kv4Args {
  const void* k; long k_st, k_sh;        // rows in (write) or out (read)
  const void* v; long v_st, v_sh;
  const int* slots;
  uint8_t* kc; uint8_t* ks; uint8_t* vc; uint8_t* vs;
  long c_sp, s_sp;                       // bytes between pages of codes and of scales
  int tokens, kv_heads;
  int lp;                                // log2 of the page
  unsigned nslots;
};

// a lane's row: its token, whether it is there, and where its codes and scales lie in their tensors
struct Row {
  int tok;
  unsigned slot;
  bool live;
  long codes, scales;
};

template <int D>
__device__ __forceinline__ Row row_of(const Kv4Args& a, int blk, int head) {
  constexpr int kLanes = D / 8;          // lanes of a row
  Row r;
  r.tok = blk * (kThreads / kLanes) + (int)threadIdx.x / kLanes;
  r.live = r.tok < a.tokens;
  r.slot = r.live ? (unsigned)a.slots[r.tok] : ~0u;
  const unsigned s = r.slot < a.nslots ? r.slot : 0, page = s >> a.lp, off = s & ((1u << a.lp) - 1);
  const long in = ((long)head << a.lp) + off;
  r.codes = (long)page * a.c_sp + in * (D / 2);
  r.scales = (long)page * a.s_sp + in * (D / 32);
  return r;
}

// the lowest byte of each block's first lane, in the row's first lane
template <int D>
__device__ __forceinline__ unsigned scales_of_row(unsigned s) {
  unsigned w = s | (unsigned)__builtin_amdgcn_update_dpp(0, (int)s, 0x104, 0xf, 0xf, true) << 8;      // row_shl 4, 8, 12
  if (D == 128) {
    w |= (unsigned)__builtin_amdgcn_update_dpp(0, (int)s, 0x108, 0xf, 0xf, true) << 16;
    w |= (unsigned)__builtin_amdgcn_update_dpp(0, (int)s, 0x10c, 0xf, 0xf, true) << 24;
  }
  return w;
}

__device__ __forceinline__ unsigned max4(unsigned v) {     // over the lanes of a block
  v = max(v, (unsigned)__builtin_amdgcn_update_dpp((int)v, (int)v, 0xB1, 0xf, 0xf, false));
  return max(v, (unsigned)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x4E, 0xf, 0xf, false));
}

// 8 values of a block of four lanes to codes; the block's scale
__device__ __forceinline__ unsigned to_codes(const f32x8& f, unsigned& scale) {
  unsigned top = 0;                      // of |x| as bits: NaN above infinity above all else
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(f[i]) & 0x7fffffffu);
  top = max4(top);
  const bool fine = top < 0x7f800000u;
  // floor(log2) - 2, one more from 1.75 up: the carry of a quarter into the exponent
  const int e = min(max((int)((top + 0x200000u) >> 23) - 129, -125), 125);
  const float inv = __uint_as_float((unsigned)(127 - e) << 23);
  unsigned c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[0] * inv, f[1] * inv, 1.f, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[2] * inv, f[3] * inv, 1.f, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[4] * inv, f[5] * inv, 1.f, 2);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[6] * inv, f[7] * inv, 1.f, 3);
  scale = fine ? e + 127 : 255;
  return fine ? c : 0u;
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) kv4_write_kernel(Kv4Args a) {
  typedef typename Vec8<T>::type vec;
  const int head = blockIdx.x % a.kv_heads, l = threadIdx.x % (D / 8);
  const Row r = row_of<D>(a, blockIdx.x / a.kv_heads, head);
  const int tok = min(r.tok, a.tokens - 1);          // (lanes past the end repeat the last row, unstored)
  const T* xk = (const T*)a.k + (long)tok * a.k_st + (long)head * a.k_sh + 8 * l;
  const T* xv = (const T*)a.v + (long)tok * a.v_st + (long)head * a.v_sh + 8 * l;
  const vec k = __builtin_nontemporal_load(reinterpret_cast<const vec*>(xk));
  const vec v = __builtin_nontemporal_load(reinterpret_cast<const vec*>(xv));
  unsigned sk, sv;
  const unsigned ck = to_codes(__builtin_convertvector(k, f32x8), sk);
  const unsigned cv = to_codes(__builtin_convertvector(v, f32x8), sv);
  sk = scales_of_row<D>(sk);
  sv = scales_of_row<D>(sv);
  if (r.slot >= a.nslots) return;        // padding
  *reinterpret_cast<unsigned*>(a.kc + r.codes + 4 * l) = ck;
  *reinterpret_cast<unsigned*>(a.vc + r.codes + 4 * l) = cv;
  if (l) return;
  if (D == 128) {
    *reinterpret_cast<unsigned*>(a.ks + r.scales) = sk;
    *reinterpret_cast<unsigned*>(a.vs + r.scales) = sv;
  } else {
    *reinterpret_cast<uint16_t*>(a.ks + r.scales) = (uint16_t)sk;
    *reinterpret_cast<uint16_t*>(a.vs + r.scales) = (uint16_t)sv;
  }
}

__device__ __forceinline__ f32x8 to_values(unsigned c, unsigned s) {
  const float f = s == 255 ? __builtin_nanf("") : __uint_as_float(s << 23);
  const bf16x2 b[4] = {__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, 1.f, 0),
                       __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, 1.f, 1),
                       __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, 1.f, 2),
                       __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, 1.f, 3)};
  f32x8 y;
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = (float)b[i / 2][i % 2] * f;
  return y;
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) kv4_read_kernel(Kv4Args a) {
  typedef typename Vec8<T>::type vec;
  const int head = blockIdx.x % a.kv_heads, l = threadIdx.x % (D / 8);
  const Row r = row_of<D>(a, blockIdx.x / a.kv_heads, head);
  const bool held = r.slot < a.nslots;   // (padding reads slot 0 and gives zeros)
  const unsigned ck = *reinterpret_cast<const unsigned*>(a.kc + r.codes + 4 * l), sk = a.ks[r.scales + l / 4];
  const unsigned cv = *reinterpret_cast<const unsigned*>(a.vc + r.codes + 4 * l), sv = a.vs[r.scales + l / 4];
  const f32x8 k = held ? to_values(ck, sk) : f32x8(0.f), v = held ? to_values(cv, sv) : f32x8(0.f);
  if (!r.live) return;
  T* ok = (T*)a.k + (long)r.tok * a.k_st + (long)head * a.k_sh + 8 * l;
  T* ov = (T*)a.v + (long)r.tok * a.v_st + (long)head * a.v_sh + 8 * l;
  __builtin_nontemporal_store(__builtin_convertvector(k, vec), reinterpret_cast<vec*>(ok));
  __builtin_nontemporal_store(__builtin_convertvector(v, vec), reinterpret_cast<vec*>(ov));
}

// the checks that both directions share
int take(Kv4Args& a, const void* k, long k_st, long k_sh, const void* v, long v_st, long v_sh, int tokens, int kv_heads,
         int D, int align, const int* slots, void* kc, void* ks, void* vc, void* vs, long code_stride, long scale_stride,
         int pages, int page) {
  auto bad = [&](const void* p, long st, long sh) {
    return !p || (reinterpret_cast<uintptr_t>(p) & 15) || st % align || sh % align;
  };
  auto odd = [](const void* p) { return !p || (reinterpret_cast<uintptr_t>(p) & 15) != 0; };
  if ((D != 64 && D != 128) || tokens < 0 || kv_heads <= 0 || pages <= 0 || page < 32 || page > 1024 || (page & (page - 1)) ||
      (long)pages * page > 0x7fffffffL || (long)tokens * kv_heads > (1L << 26))
    return OA_EINVAL;
  a.tokens = tokens;
  if (!tokens) return 0;
  if (bad(k, k_st, k_sh) || bad(v, v_st, v_sh) || odd(kc) || odd(ks) || odd(vc) ||
      odd(vs) || !slots || code_stride < (long)kv_heads * page * (D / 2) || scale_stride < (long)kv_heads * page * (D / 32) ||
      code_stride % 16 || scale_stride % 16)
    return OA_EINVAL;
  a.k = k; a.k_st = k_st; a.k_sh = k_sh;
  a.v = v; a.v_st = v_st; a.v_sh = v_sh;
  a.slots = slots;
  a.kc = (uint8_t*)kc; a.ks = (uint8_t*)ks; a.vc = (uint8_t*)vc; a.vs = (uint8_t*)vs;
  a.c_sp = code_stride; a.s_sp = scale_stride;
  a.kv_heads = kv_heads;
  a.lp = __builtin_ctz(page);
  a.nslots = (unsigned)pages * page;
  return 0;
}

dim3 grid_of(const Kv4Args& a, int D) {
  const int rows = kThreads / (D / 8);
  return dim3((unsigned)((long)((a.tokens + rows - 1) / rows) * a.kv_heads));
}

template <typename T>
void write_rows(const Kv4Args& a, int D, hipStream_t st) {
  if (D == 64) hipLaunchKernelGGL((kv4_write_kernel<T, 64>), grid_of(a, D), dim3(kThreads), 0, st, a);
  else hipLaunchKernelGGL((kv4_write_kernel<T, 128>), grid_of(a, D), dim3(kThreads), 0, st, a);
}
template <typename T>
void read_rows(const Kv4Args& a, int D, hipStream_t st) {
  if (D == 64) hipLaunchKernelGGL((kv4_read_kernel<T, 64>), grid_of(a, D), dim3(kThreads), 0, st, a);
  else hipLaunchKernelGGL((kv4_read_kernel<T, 128>), grid_of(a, D), dim3(kThreads), 0, st, a);
}

}  // namespace

extern "C" int oa_kv4_write(const void* k, long k_st, long k_sh, const void* v, long v_st, long v_sh, int tokens,
                            int kv_heads, int head_dim, int dtype, const int* slots, void* kc, void* ks, void* vc,
                            void* vs, long code_stride, long scale_stride, int pages, int page, void* stream) {
  if (dtype < 0 || dtype > 2) return OA_EINVAL;
  Kv4Args a;
  if (const int e = take(a, k, k_st, k_sh, v, v_st, v_sh, tokens, kv_heads, head_dim, dtype == 2 ? 4 : 8, slots, kc, ks,
                         vc, vs, code_stride, scale_stride, pages, page))
    return e;
  if (!tokens) return 0;
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == 0) write_rows<__bf16>(a, head_dim, st);
  else if (dtype == 1) write_rows<_Float16>(a, head_dim, st);
  else write_rows<float>(a, head_dim, st);
  return OA_LAUNCH_STATUS();
}

extern "C" int oa_kv4_read(const int* slots, const void* kc, const void* ks, const void* vc, const void* vs,
                           long code_stride, long scale_stride, int pages, int page, void* k, long k_st, long k_sh,
                           void* v, long v_st, long v_sh, int tokens, int kv_heads, int head_dim, int dtype,
                           void* stream) {
  if (dtype != 0 && dtype != 2) return OA_EINVAL;  // (fp16 does not hold what a scale may be)
  Kv4Args a;
  if (const int e = take(a, k, k_st, k_sh, v, v_st, v_sh, tokens, kv_heads, head_dim, dtype == 2 ? 4 : 8, slots,
                         const_cast<void*>(kc), const_cast<void*>(ks), const_cast<void*>(vc), const_cast<void*>(vs),
                         code_stride, scale_stride, pages, page))
    return e;
  if (!tokens) return 0;
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == 0) read_rows<__bf16>(a, head_dim, st);
  else read_rows<float>(a, head_dim, st);
  return OA_LAUNCH_STATUS();
}
