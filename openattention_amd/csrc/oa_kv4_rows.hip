// Causal attention over the 4-bit paged cache for many query rows of a KV head (a question, a piece of a
// prompt): the same sums as in oa_kv4_attn.hip, with the keys' codes turned to bf16 once for 128 rows.
//
// One workgroup of four waves takes 128 query rows of a KV head, 32 to a wave, and a chunk of keys.  A tile of 32
// keys is turned to bf16 (V: fp16) by all of them, 16 values of K and of V to a lane (8 where D is 64), into LDS
// tiles that all four read.  Products are v_mfma_f32_32x32x16: S^T = K Q^T, whose lanes hold 16 keys' scores of
// one row, and O^T = V^T P^T with V^T by the LDS transpose reads (the contraction takes keys in the order the
// scores left them).
// Weights and values go into the second product in fp16: weights times 2^7 (11 bits of each, down to 2^-21
// of the maximum; up to 2^8 past it, so that the sums are rescaled in few tiles),
// and values, codes of two bits times 2^(s - ref), exactly, where ref is the largest scale of the block of
// dims in the chunk's first tile.  That holds scales from 2^-13 to 2^13 of ref; a workgroup that meets
// another one leaves a flag, and a second launch does its part again with values in bf16, which holds all, and
// weights in two bf16 terms (both in one kernel spill registers).
// The loop is a pipeline: iteration i issues the products of S(i + 1) and of O += V(i - 1) P(i - 1) between
// the steps of the softmax of S(i), puts tile i + 2 into LDS and requests the codes of tile i + 4.
// Tiles: rows of 2 D bytes, 5 (D = 64: 1) 16-byte places apart, so that rows read or written at one place and
// the transpose reads spread over the banks and every address is one register and a constant (exchanged
// places instead, as in the prompt's kernel, take 16 more registers and spill).
//
// 64 tokens of 32 query heads over 32768 keys of 8 heads, for two sequences (69 GFLOP): 94 us for the call with the
// empty second launch and the join (4.8 and 8.5 under a profiler), 730 TFLOP/s (a large bf16 product reaches 1256).
// The matrix cores are busy 30% of the time, the vector units about 45%, so that neither bounds it; two waves a SIMD
// at 254 registers, which meet every 32 keys.
#include "oa_kv4_attn.h"

namespace {

using namespace kv4;

typedef float float16v __attribute__((ext_vector_type(16)));

constexpr int kWaveRows = 32;
constexpr int kRows = kWaves * kWaveRows;
constexpr int kAhead = 2;                // steps whose LDS operands are requested ahead

__device__ __forceinline__ float16v mfma(bf16x8 a, bf16x8 b, float16v c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float16v mfma16(bf16x8 a, uint4v b, float16v c) {     // both hold fp16
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ uint32_t pack2h(float a, float b) {
  const f32x2 x = {a, b};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(x, f16x2));
}
// 8 codes to fp16, scaled by a power of two (all exponent bits set: NaN)
__device__ __forceinline__ bf16x8 from4h(unsigned w, float f) {
  const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, f, 0);
  const f16x2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, f, 1);
  const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, f, 2);
  const f16x2 d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, f, 3);
  const uint4v x = {__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b), __builtin_bit_cast(uint32_t, c),
                    __builtin_bit_cast(uint32_t, d)};
  return __builtin_bit_cast(bf16x8, x);
}

constexpr int kSpan = 13;                // largest |log2| of a scale over the reference's that fp16 takes
constexpr float kLift = 7.f;             // log2 of what weights are multiplied by
constexpr float kLazy = 8.f;             // log2 of how far a weight may pass 1 before the sums are rescaled

template <bool TWO> struct Weights;      // P^T of a 32-key tile, 16 keys per operand
template <> struct Weights<false> { uint4v hi[2]; };
template <> struct Weights<true> { uint4v hi[2], lo[2]; };       // two bf16 terms

__device__ __forceinline__ float16v value_product(bf16x8 v, const Weights<false>& p, int kk, float16v o) {
  return mfma16(v, p.hi[kk], o);
}
__device__ __forceinline__ float16v value_product(bf16x8 v, const Weights<true>& p, int kk, float16v o) {
  o = mfma(v, __builtin_bit_cast(bf16x8, p.hi[kk]), o);
  return mfma(v, __builtin_bit_cast(bf16x8, p.lo[kk]), o);
}

template <int D, bool TWO>
__global__ void __launch_bounds__(kThreads, 2) kv4_rows_kernel(AttnArgs a) {
  constexpr int kSteps = D / 16;         // products of a score tile, and of a value tile for each term
  constexpr int kDims = D / 32;          // tiles of 32 dims
  constexpr int kRowB = D * 2 + (D == 128 ? 80 : 16), kTileB = kTile * kRowB;
  constexpr int kWords = D / 64;         // words of codes of K and of V that a lane turns to floats
  __shared__ __align__(16) char s_t[6 * kTileB];          // K even, K odd, V of tiles i % 4
  __shared__ unsigned long s_nan[4][kWaves];               // NaN blocks of a masked V tile, by the lanes of each wave
  __shared__ unsigned s_ref[kWaves][8];                    // largest scales of the first V tile, by wave and part
  __shared__ unsigned s_wide;                              // a scale is out of fp16's span

  if (TWO && !a.ws_flag[blockIdx.x]) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n32 = lane & 31, h = lane >> 5;
  const int units = a.B * a.HKV;
  const int bh = blockIdx.x % units, rest = blockIdx.x / units;
  const int ch = rest / a.ntile, row0 = (rest - ch * a.ntile) * kRows;
  const int b = bh / a.HKV, head = bh - b * a.HKV;
  const Seq sq = seq_of(a, b);
  const int rows = min(sq.R, a.max_q) * a.G;
  if (!TWO && tid == 0) a.ws_flag[blockIdx.x] = 0;
  if (row0 >= rows) return;
  const int first = sq.n - sq.R;         // position of the sequence's first query token
  const int hi = sq.bad ? 0 : first + (min(row0 + kRows, rows) - 1) / a.G + 1;         // keys any row sees
  const int all = first + row0 / a.G + 1;                                              // keys every row sees
  const int k0 = ch * a.chunk, k1 = min(k0 + a.chunk, hi);
  if (k0 >= k1 && a.nchunk > 1) return;
  const int n = max(0, (k1 - k0 + kTile - 1) / kTile);     // tiles
  const int nfull = min(n, max(0, (all - k0) / kTile));    // those that every row sees whole

  char* const s_v = s_t + 2 * kTileB;
  // staging: key lane / 8 of the tile, an eighth of its dims
  const int skey = tid >> 3, sg = tid & 7;
  const int* trow = a.table + (long)b * a.t_st;
  const int pmask = (1 << a.lp) - 1;
  const uint8_t* const kc = a.kc + ((long)head << a.lp) * (D / 2);
  const uint8_t* const vc = a.vc + ((long)head << a.lp) * (D / 2);
  const uint8_t* const ks = a.ks + ((long)head << a.lp) * (D / 32);
  const uint8_t* const vs = a.vs + ((long)head << a.lp) * (D / 32);
  const unsigned oc = skey * (D / 2) + sg * (D / 16), os = skey * (D / 32) + sg * D / 256;
  typedef unsigned words __attribute__((ext_vector_type(kWords)));
  // two tiles' codes are on their way, by parity
  struct Staged {
    words k, v;
    unsigned ks, vs, bad;
    int next;                            // the table's entry for the tile after the next
  } st[2];
  auto page_at = [&](int tile) { return table_entry(trow, min((k0 + tile * kTile) >> a.lp, a.width - 1)); };
  auto fetch = [&](Staged& x, int tile, unsigned page) {   // (past the last tile: read, never used)
    // (by lane, though all have the same page: one multiply-add to an address instead of some 20 scalar steps)
    const bool bad = page >= (unsigned)a.NP;
    x.bad = bad ? 0x7f800000u : 0u;
    const unsigned pg = bad ? 0u : page, off = (k0 + tile * kTile) & pmask;
    const unsigned long rc = (unsigned long)pg * (unsigned)a.c_sp + (oc + off * (D / 2));
    const unsigned long rs = (unsigned long)pg * (unsigned)a.s_sp + (os + off * (D / 32));
    x.k = *reinterpret_cast<const words*>(kc + rc);
    x.ks = ks[rs];
    x.v = *reinterpret_cast<const words*>(vc + rc);
    x.vs = vs[rs];
    x.next = page_at(tile + 2);
  };
  char* const sdst = s_t + skey * kRowB + sg * (D / 4);
  unsigned ref = 0, wide = 0;            // this lane's block's reference; it met a scale out of span
  // A lane's V block in a tile: its scale as a float, or zeros instead of its values: those of keys past the last
  // one any row sees (their weights are 0, but what lies there may be anything), and of NaN blocks of a masked
  // tile, which s_nan remembers
  struct Put {
    float f;
    bool out;
  };
  auto put_begin = [&](const Staged& y, int tile) {
    Put t;
    t.out = false;
    if (tile >= nfull) {
      const bool past = k0 + tile * kTile + skey >= hi, nan = y.vs == 255 && !past;
      const unsigned long at = __ballot(nan);
      if (lane == 0) s_nan[tile & 3][wave] = at;
      t.out = nan || past;
    }
    if (TWO) {
      t.f = __uint_as_float(t.out ? 0x3f800000u : y.vs << 23);
    } else {
      unsigned any = y.v[0];
      if constexpr (kWords > 1) any |= y.v[1];
      // (NaN first: its codes are 0 where oa_kv4_write put them, and zeros have no scale to be out of span)
      const bool nan = y.vs == 255 && !t.out, zero = t.out || !(any & 0x77777777u);
      const int x = (int)y.vs - (int)ref;
      if (!zero && !nan && (x < -kSpan || x > kSpan)) wide = 1;
      t.f = __uint_as_float(nan ? 0x7f800000u : zero ? 0x3f800000u : (unsigned)(127 + x) << 23);
    }
    return t;
  };
  auto put_k = [&](const Staged& y, int parity, int i) {
    *reinterpret_cast<bf16x8*>(sdst + parity * kTileB + (i << 4)) = from4(y.k[i], __uint_as_float(y.ks << 23 | y.bad));
  };
  auto put_v = [&](const Put& t, const Staged& y, int tile, int i) {
    const unsigned w = t.out ? 0u : y.v[i];
    *reinterpret_cast<bf16x8*>(sdst + (2 + (tile & 3)) * kTileB + (i << 4)) = TWO ? from4(w, t.f) : from4h(w, t.f);
  };

  // operand addresses (bytes in a tile)
  const int kad = n32 * kRowB + (h << 4);
  const int lr = (lane & 15) >> 2, lc = lane & 3, dsub = (lane >> 4) & 1;
  const int vad = (4 * h + lr) * kRowB + (dsub << 5) + (lc << 3);
  auto key_op = [&](const char* tile, int step) { return *reinterpret_cast<const bf16x8*>(tile + kad + (step << 5)); };
  // V^T of dims 32 db .. and keys 16 kk ..: two transposed reads of 4 keys, 8 apart
  auto val_op = [&](char* tile, int db, int kk) {
    char* const p = tile + vad + (db << 6) + kk * 16 * kRowB;
    const short4v x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4v*)p);
    const short4v y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4v*)(p + 8 * kRowB));
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
  };

  // this lane's row (negated under a negative scale, as the maximum is taken before scaling, and zeros under one of
  // 0, so that masked scores stay -inf) and how many keys it sees (0: no such row)
  const float c = a.c == 0.f ? 1.f : fabsf(a.c);
  const int r = row0 + wave * kWaveRows + n32;
  const int rr = min(r, rows - 1), j = rr / a.G, hd = head * a.G + rr - j * a.G;
  const int lim = r < rows ? first + j + 1 : 0;
  bf16x8 Q[kSteps];
  {
    const unsigned flip = a.c < 0.f ? 0x80008000u : 0u, keep = a.c == 0.f ? 0u : ~0u;
    const uint16_t* p = a.q + (long)(sq.r0 + j) * a.q_st + (long)hd * a.q_sh + 8 * h;
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
      Q[s] = __builtin_bit_cast(bf16x8, (*reinterpret_cast<const uint4v*>(p + 16 * s) ^ uint4v(flip)) & uint4v(keep));
  }

  float16v O[kDims], S0 = float16v(0.f), S1;
  Weights<TWO> P0, P1;
#pragma unroll
  for (int d = 0; d < kDims; ++d) O[d] = float16v(0.f);
  float m = -FLT_MAX, l = 0.f;           // running maximum, scaled, and sum of the lane's keys, times 2^kLift
  bool big = false;                      // a maximum is past 2^24 (uniform)
  if (tid == 0) s_wide = 0;

  if (n > 0) {
    // tiles 0 and 1 and zeros for V(-1), whose weights are 0; then tiles 2 and 3 requested
    fetch(st[0], 0, page_at(0));
    fetch(st[1], 1, page_at(1));
    if (!TWO) {                          // the largest scale of each block of dims in V(0)
      unsigned e = st[0].vs == 255 || k0 + skey >= hi ? 0 : st[0].vs;
#pragma unroll
      for (int x = 1; x < 64; x <<= 1)
        if (x >= 8 || x < 256 / D) e = max(e, (unsigned)__shfl_xor((int)e, x));
      if (lane < 8) s_ref[wave][lane] = e;
      oa::lds_barrier();
      ref = max(max(s_ref[0][sg], s_ref[1][sg]), max(s_ref[2][sg], s_ref[3][sg]));
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const Put t = put_begin(st[x], x);
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        put_k(st[x], x, i);
        put_v(t, st[x], x, i);
      }
    }
#pragma unroll
    for (int i = 0; i < kWords; ++i) *reinterpret_cast<uint4v*>(sdst + 5 * kTileB + (i << 4)) = uint4v(0u);
    P1.hi[0] = P1.hi[1] = uint4v(0u);
    if constexpr (TWO) P1.lo[0] = P1.lo[1] = uint4v(0u);
    fetch(st[0], 2, st[0].next);
    fetch(st[1], 3, st[1].next);
    oa::lds_barrier();
#pragma unroll
    for (int s = 0; s < kSteps; ++s) S0 = mfma(key_op(s_t, s), Q[s], S0);
    oa::lds_barrier();                   // K(0) has been read: its place takes K(2)

    // O += V(tile) P(tile)'s NaN blocks, into the rows that see them (rare)
    auto nan_blocks = [&](int tile) {
#pragma unroll 1
      for (int w = 0; w < kWaves; ++w) {
        unsigned long at = s_nan[tile & 3][w];
        while (at) {
          const int bit = __builtin_ctzl(at), key = k0 + tile * kTile + 8 * w + (bit >> 3), blk = (bit & 7) * D / 256;
          at &= at - 1;
#pragma unroll
          for (int d = 0; d < kDims; ++d)
            if (d == blk && key < lim) O[d] = float16v(__builtin_nanf(""));
        }
      }
    };
    // iteration i (parity odd = i & 1): K(i + 1) is in the other parity's tile
    auto body = [&](auto odd_c, int i, float16v& S, float16v& Sn, const Weights<TWO>& Pp, Weights<TWO>& Pn) {
      constexpr int kOdd = decltype(odd_c)::value;
      char* const kt = s_t + (1 - kOdd) * kTileB;
      char* const vt = s_v + ((i - 1) & 3) * kTileB;
      const Put to = put_begin(st[kOdd], i + 2);
      float mx = -INFINITY, alpha = 1.f, p0 = 0.f;
      bool moved = false;
      Sn = float16v(0.f);
      bf16x8 kop[kSteps], vop[kSteps];
#pragma unroll
      for (int s = 0; s < kAhead; ++s) {
        kop[s] = key_op(kt, s);
        vop[s] = val_op(vt, s >> 1, s & 1);
      }
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        if (s + kAhead < kSteps) {
          kop[s + kAhead] = key_op(kt, s + kAhead);
          vop[s + kAhead] = val_op(vt, (s + kAhead) >> 1, (s + kAhead) & 1);
        }
        Sn = mfma(kop[s], Q[s], Sn);
        O[s >> 1] = value_product(vop[s], Pp, s & 1, O[s >> 1]);
        if (s == 0) {                    // the tile's maximum
          if (i >= nfull) {
#pragma unroll
            for (int r = 0; r < 16; ++r)
              if (k0 + i * kTile + 8 * (r >> 2) + 4 * h + (r & 3) >= lim) S[r] = -INFINITY;
          }
#pragma unroll
          for (int r = 0; r < 16; ++r) mx = fmaxf(mx, S[r]);
        } else if (s == 1) {
          const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
          mx = fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1])) * c;
          moved = __any(mx > m + (big ? 0.f : kLazy));
          if (moved) {
            const float mn = fmaxf(m, mx);
            alpha = __builtin_amdgcn_exp2f(m - mn);
            l *= alpha;
            m = mn;
            // (as in oa_kv4_attn.hip: past 2^24 the product is rounded before the maximum is taken off)
            big = __any(fabsf(m) >= 16777216.f);
          }
          if (big) {
#pragma unroll
            for (int r = 0; r < 16; ++r) S[r] *= c;
          }
        } else {
#pragma unroll
          for (int r = (s - 2) * 16 / (kSteps - 2); r < (s - 1) * 16 / (kSteps - 2); ++r) {
            const float p1 = __builtin_amdgcn_exp2f(fmaf(S[r], big ? 1.f : c, kLift - m));
            l += p1;
            if (r & 1) {
              uint32_t u = TWO ? pack2(p0, p1) : pack2h(p0, p1);
              asm volatile("" : "+v"(u));          // (pinned here: left alone they all sink below the products)
              Pn.hi[r >> 3][(r & 7) >> 1] = u;
              if constexpr (TWO)
                Pn.lo[r >> 3][(r & 7) >> 1] = pack2(p0 - __uint_as_float(u << 16), p1 - __uint_as_float(u & 0xffff0000u));
            }
            p0 = p1;
          }
        }
        if (s >= kSteps - 2 * kWords) {
          const int x = s - (kSteps - 2 * kWords);
          if (x < kWords) put_k(st[kOdd], kOdd, x);
          else put_v(to, st[kOdd], i + 2, x - kWords);
        }
        if (s == kSteps - 1) fetch(st[kOdd], i + 4, st[kOdd].next);
        __builtin_amdgcn_sched_barrier(0);
      }
      if (i > nfull) nan_blocks(i - 1);
      if (moved) {                       // (after O += V(i - 1) P(i - 1), whose weights had the old maximum)
#pragma unroll
        for (int d = 0; d < kDims; ++d) O[d] *= alpha;
      }
      oa::lds_barrier();
    };
    typedef std::integral_constant<int, 0> even_t;
    typedef std::integral_constant<int, 1> odd_t;
    auto finish = [&](const Weights<TWO>& P) {               // V(n - 1) P(n - 1)
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const bf16x8 vop = val_op(s_v + ((n - 1) & 3) * kTileB, s >> 1, s & 1);
        O[s >> 1] = value_product(vop, P, s & 1, O[s >> 1]);
      }
      if (n > nfull) nan_blocks(n - 1);
    };
#pragma unroll 1
    for (int i = 0; i < n; i += 2) {
      body(even_t(), i, S0, S1, P1, P0);
      if (i + 1 < n) body(odd_t(), i + 1, S1, S0, P0, P1);
    }
    if (n & 1) finish(P0);
    else finish(P1);
    if (!TWO) {
      if (wide) s_wide = 1;
#pragma unroll
      for (int d = 0; d < kDims; ++d)    // (a reference of 0: all values were)
        O[d] *= __uint_as_float(max(max(s_ref[0][d * 256 / D], s_ref[1][d * 256 / D]),
                                    max(s_ref[2][d * 256 / D], s_ref[3][d * 256 / D])) << 23);
    }
  }
  if (!TWO) {
    oa::lds_barrier();
    if (tid == 0 && s_wide) a.ws_flag[blockIdx.x] = 1;
  }

  const auto lx = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
  const float L = __uint_as_float(lx[0]) + __uint_as_float(lx[1]);
  if (r >= rows) return;
  if (a.nchunk == 1) {
    const float inv = 1.f / L;
    const bool none = lim <= 0;
    uint16_t* o = a.out + (long)(sq.r0 + j) * a.o_st + (long)hd * a.o_sh + 4 * h;
#pragma unroll
    for (int d = 0; d < kDims; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        f32x4 x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = sq.bad ? __builtin_nanf("") : none ? 0.f : O[d][4 * g + e] * inv;
        *reinterpret_cast<uint2v*>(o + 32 * d + 8 * g) = uint2v{pack2(x[0], x[1]), pack2(x[2], x[3])};
      }
  } else {
    const long at = ((long)(sq.r0 + j) * (a.HKV * a.G) + hd) * a.nchunk + ch;
#pragma unroll
    for (int d = 0; d < kDims; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32x4*>(a.ws_o + at * D + 32 * d + 8 * g + 4 * h) =
            f32x4{O[d][4 * g], O[d][4 * g + 1], O[d][4 * g + 2], O[d][4 * g + 3]};
    if (h == 0) *reinterpret_cast<f32x2*>(a.ws_ml + at * 2) = f32x2{m, L};
  }
}

}  // namespace

namespace kv4 {

void launch_rows(const AttnArgs& a, int head_dim, dim3 grid, hipStream_t st) {
  if (head_dim == 64) {
    hipLaunchKernelGGL((kv4_rows_kernel<64, false>), grid, dim3(kThreads), 0, st, a);
    hipLaunchKernelGGL((kv4_rows_kernel<64, true>), grid, dim3(kThreads), 0, st, a);
  } else {
    hipLaunchKernelGGL((kv4_rows_kernel<128, false>), grid, dim3(kThreads), 0, st, a);
    hipLaunchKernelGGL((kv4_rows_kernel<128, true>), grid, dim3(kThreads), 0, st, a);
  }
}

}  // namespace kv4
