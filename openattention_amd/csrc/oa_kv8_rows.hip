// Causal attention over the 8-bit paged cache for many query rows of a KV head (a question, a piece of a prompt): the
// same sums as in oa_kv8_attn.hip, with the keys' codes turned to 16 bits once for 128 or 256 rows.
//
// One workgroup of four waves takes 128 NR query rows of a KV head, 32 NR to a wave, and a chunk of keys.  A tile of 32
// keys is turned to the queries' type (V: fp16) by all of them, 16 values of K and of V to a lane (8 where D is 64),
// into LDS tiles that all four read.  Products are v_mfma_f32_32x32x16: S^T = K Q^T, whose lanes hold 16 keys' scores of
// one row, and O^T = V^T P^T with V^T by the LDS transpose reads (the contraction takes keys in the order the scores
// left them).  An operand that a wave has read from LDS serves all of its NR products.
// Weights and values go into the second product in fp16: weights times 2^7 (11 bits of each, down to 2^-21 of the
// maximum; up to 2^8 past it, so that the sums are rescaled in few tiles), and values as codes times 2^(e - ref), exactly,
// where ref is a scale that the sums are held in: -15 <= e - ref <= 7 keeps every code's value within fp16.  A block out
// of that span changes ref, and the sums are rescaled by a power of two when its turn comes.  (ref stays within 2^60 of the
// largest: values so much smaller are rounded to a multiple of 2^-84 of it.)
// The loop is a pipeline: iteration i issues the products of S(i + 1) and of O += V(i - 1) P(i - 1) between
// the steps of the softmax of S(i), puts tile i + 2 into LDS and requests the codes of tile i + 4.
// Tiles: rows of 2 D bytes, 5 (D = 64: 1) 16-byte places apart, so that rows read or written at one place and
// the transpose reads spread over the banks and every address is one register and a constant.
#include "oa_kv8_attn.h"

namespace {

using namespace kv8;

typedef float float16v __attribute__((ext_vector_type(16)));

constexpr int kWaveRows = 32;
constexpr int kAhead = 2;                // steps whose LDS operands are requested ahead
constexpr int kUp = 7, kDown = 15;       // e - ref that fp16 takes: 448 * 2^7 and 2^-9 * 2^-15 are fp16 numbers
constexpr int kDeep = 60;                // how far ref goes below the largest
constexpr int kLeast = -117;             // a block's least exponent: zeros, or values that count as such beside others
constexpr float kLift = 7.f;             // log2 of what weights are multiplied by
constexpr float kLazy = 8.f;             // log2 of how far a weight may pass 1 before the sums are rescaled

template <bool HALF>
__device__ __forceinline__ float16v mfma(bf16x8 a, bf16x8 b, float16v c) {
  if constexpr (HALF)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// 2^e, whatever e
__device__ __forceinline__ float any_power(int e) { return power(min(max(e, -126), 127)); }

// NR: groups of 32 rows of a wave
template <int D, int NR, typename T>
__global__ void __launch_bounds__(kThreads, NR == 1 ? 2 : 1) kv8_rows_kernel(AttnArgs a) {
  constexpr bool kHalf = !std::is_same<T, __bf16>::value;
  constexpr int kRows = kWaves * kWaveRows * NR;
  constexpr int kSteps = D / 16;         // products of a score tile, and of a value tile
  constexpr int kDims = D / 32;          // tiles of 32 dims
  constexpr int kRowB = D * 2 + (D == 128 ? 80 : 16), kTileB = kTile * kRowB;
  constexpr int kParts = D / 64;         // groups of 8 codes of K and of V that a lane turns to 16 bits
  __shared__ __align__(16) char s_t[6 * kTileB];          // K even, K odd, V of tiles i % 4
  __shared__ unsigned long s_nan[4][kWaves];               // NaN in a masked V tile, by the lanes of each wave

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n32 = lane & 31, h = lane >> 5;
  const int units = a.B * a.HKV;
  const int bh = blockIdx.x % units, rest = blockIdx.x / units;
  const int ch = rest / a.ntile, row0 = (rest - ch * a.ntile) * kRows;
  const int b = bh / a.HKV, head = bh - b * a.HKV;
  const Seq sq = seq_of(a, b);
  const int rows = min(sq.R, a.max_q) * a.G;
  if (row0 >= rows) return;
  const int first = sq.n - sq.R;         // position of the sequence's first query token
  const int hi = sq.bad ? 0 : first + (min(row0 + kRows, rows) - 1) / a.G + 1;         // keys any row sees
  const int all = first + row0 / a.G + 1;                                              // keys every row sees
  const int k0 = ch * a.chunk, k1 = min(k0 + a.chunk, hi);
  if (k0 >= k1 && a.nchunk > 1) return;
  const int n = max(0, (k1 - k0 + kTile - 1) / kTile);     // tiles
  const int nfull = min(n, max(0, (all - k0) / kTile));    // those that every row sees whole

  char* const s_v = s_t + 2 * kTileB;
  // staging: key tid / 8 of the tile, an eighth of its dims; a tile is successive bytes
  const int skey = tid >> 3, sg = tid & 7;
  const int* trow = a.table + (long)b * a.t_st;
  const int pmask = (1 << a.lp) - 1;
  const uint8_t* const kc = a.kc + ((long)head << a.lp) * D + tid * (D / 8);
  const uint8_t* const vc = a.vc + ((long)head << a.lp) * D + tid * (D / 8);
  const float c = a.c == 0.f ? 1.f : fabsf(a.c);
  typedef unsigned words __attribute__((ext_vector_type(2 * kParts)));
  // two tiles' codes are on their way, by parity
  struct Staged {
    words k, v;
    unsigned ks, vs, bad;
    int next;                            // the table's entry for the tile after the next
  } st[2];
  auto page_at = [&](int tile) { return table_entry(trow, min((k0 + tile * kTile) >> a.lp, a.width - 1)); };
  auto fetch = [&](Staged& x, int tile, unsigned page) {   // (past the last tile: read, never used)
    const bool bad = page >= (unsigned)a.NP;
    x.bad = bad ? 0x7f800000u : 0u;
    const unsigned pg = bad ? 0u : page, off = (k0 + tile * kTile) & pmask;
    const unsigned long at = (unsigned long)pg * (unsigned long)a.c_sp + off * D, as = (unsigned long)pg * (unsigned long)a.s_sp + head;
    x.k = *reinterpret_cast<const words*>(kc + at);
    x.ks = a.ks[as];
    x.v = *reinterpret_cast<const words*>(vc + at);
    x.vs = a.vs[as];
    x.next = page_at(tile + 2);
  };
  char* const sdst = s_t + skey * kRowB + sg * (D / 4);
  int ref = 0, top = -1000;              // the scale of the last tile in LDS, and the largest so far
  // A tile's scales on their way into LDS, and whether this lane's values count as zeros: those of keys past the last
  // one any row sees (their weights are 0, but what lies there may be anything), and NaN of a masked tile, which s_nan
  // remembers
  struct Put {
    float f;
    bool out;
  };
  auto scale_of = [&](const Staged& y) {                   // K's, a factor of the scores
    return fminf(c * __uint_as_float(y.ks << 23), FLT_MAX) + __uint_as_float(y.bad) * 0.f;
  };
  auto put_begin = [&](const Staged& y, int tile) {
    Put t;
    const int e = __builtin_amdgcn_readfirstlane((int)y.vs) - 127;
    top = max(top, e);
    if (e - ref > kUp || (e - ref < -kDown && e > kLeast)) ref = max(e, top - kDeep);
    t.f = any_power(e - ref);
    t.out = false;
    if (tile >= nfull) {
      const bool past = k0 + tile * kTile + skey >= hi;
      unsigned any = 0;
#pragma unroll
      for (int i = 0; i < 2 * kParts; ++i) any |= nan_codes(y.v[i]);
      const unsigned long at = __ballot(any && !past);
      if (lane == 0) s_nan[tile & 3][wave] = at;
      t.out = any || past;
    }
    return t;
  };
  auto put_k = [&](const Staged& y, int parity, int i) {
    *reinterpret_cast<bf16x8*>(sdst + parity * kTileB + (i << 4)) =
        kHalf ? from8h(y.k[2 * i], y.k[2 * i + 1], 1.f) : from8(y.k[2 * i], y.k[2 * i + 1], 1.f);
  };
  auto put_v = [&](const Put& t, const Staged& y, int tile, int i) {
    const unsigned w0 = t.out ? 0u : y.v[2 * i], w1 = t.out ? 0u : y.v[2 * i + 1];
    *reinterpret_cast<bf16x8*>(sdst + (2 + (tile & 3)) * kTileB + (i << 4)) = from8h(w0, w1, t.f);
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

  // this lane's rows (negated under a negative scale, as the maximum is taken before scaling, and zeros under one of
  // 0, so that masked scores stay -inf) and how many keys they see (0: no such row)
  int lim[NR], tok[NR], hd[NR];
  bf16x8 Q[NR][kSteps];
#pragma unroll
  for (int x = 0; x < NR; ++x) {
    const int r = row0 + (wave * NR + x) * kWaveRows + n32, rr = min(r, rows - 1), j = rr / a.G;
    tok[x] = sq.r0 + j;
    hd[x] = head * a.G + rr - j * a.G;
    lim[x] = r < rows ? first + j + 1 : 0;
    const unsigned flip = a.c < 0.f ? 0x80008000u : 0u, keep = a.c == 0.f ? 0u : ~0u;
    const uint16_t* p = a.q + (long)tok[x] * a.q_st + (long)hd[x] * a.q_sh + 8 * h;
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
      Q[x][s] = __builtin_bit_cast(bf16x8, (*reinterpret_cast<const uint4v*>(p + 16 * s) ^ uint4v(flip)) & uint4v(keep));
  }

  struct Weights { uint4v p[2]; };       // P^T of a 32-key tile in fp16, 16 keys per operand
  struct Scores { float16v s[NR]; };
  float16v O[NR][kDims];
  Scores S0, S1;
  Weights P0[NR], P1[NR];
  float m[NR], l[NR];                    // running maximum, scaled, and sum of the lane's keys, times 2^kLift
  bool big[NR];                          // a maximum is past 2^24 (uniform)
#pragma unroll
  for (int x = 0; x < NR; ++x) {
    S0.s[x] = float16v(0.f);
    m[x] = -FLT_MAX;
    l[x] = 0.f;
    big[x] = false;
#pragma unroll
    for (int d = 0; d < kDims; ++d) O[x][d] = float16v(0.f);
  }
  int held = 0;                          // the scale of the sums: they stand for O 2^held

  if (n > 0) {
    // tiles 0 and 1 and zeros for V(-1), whose weights are 0; then tiles 2 and 3 requested
    fetch(st[0], 0, page_at(0));
    fetch(st[1], 1, page_at(1));
    ref = held = __builtin_amdgcn_readfirstlane((int)st[0].vs) - 127;
    float ck0 = scale_of(st[0]), ck1 = scale_of(st[1]);    // of tiles i and i + 1
    int ref0 = 0, ref1 = 0;                                // of tiles i and i + 1
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const Put t = put_begin(st[x], x);
      if (x == 0) ref0 = ref;
      else ref1 = ref;
#pragma unroll
      for (int i = 0; i < kParts; ++i) {
        put_k(st[x], x, i);
        put_v(t, st[x], x, i);
      }
    }
    int refp = ref0;                                       // of tile i - 1
#pragma unroll
    for (int i = 0; i < kParts; ++i) *reinterpret_cast<uint4v*>(sdst + 5 * kTileB + (i << 4)) = uint4v(0u);
#pragma unroll
    for (int x = 0; x < NR; ++x) P1[x].p[0] = P1[x].p[1] = uint4v(0u);
    fetch(st[0], 2, st[0].next);
    fetch(st[1], 3, st[1].next);
    oa::lds_barrier();
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const bf16x8 kop = key_op(s_t, s);
#pragma unroll
      for (int x = 0; x < NR; ++x) S0.s[x] = mfma<kHalf>(kop, Q[x][s], S0.s[x]);
    }
    oa::lds_barrier();                   // K(0) has been read: its place takes K(2)

    // O += V(tile) P(tile)'s NaN, into the rows that see it (rare)
    auto nan_rows = [&](int tile) {
#pragma unroll 1
      for (int w = 0; w < kWaves; ++w) {
        unsigned long at = s_nan[tile & 3][w];
        while (at) {
          const int bit = __builtin_ctzl(at), key = k0 + tile * kTile + 8 * w + (bit >> 3), blk = (bit & 7) * D / 256;
          at &= at - 1;
#pragma unroll
          for (int x = 0; x < NR; ++x)
#pragma unroll
            for (int d = 0; d < kDims; ++d)
              if (d == blk && key < lim[x]) O[x][d] = float16v(__builtin_nanf(""));
        }
      }
    };
    // the sums to the scale of the tile that is added next
    auto rescale = [&](int to) {
      if (held != to) {
        const float f = any_power(held - to);
        held = to;
#pragma unroll
        for (int x = 0; x < NR; ++x)
#pragma unroll
          for (int d = 0; d < kDims; ++d) O[x][d] *= f;
      }
    };
    // iteration i (parity odd = i & 1): K(i + 1) is in the other parity's tile
    auto body = [&](auto odd_c, int i, Scores& S, Scores& Sn, const Weights (&Pp)[NR], Weights (&Pn)[NR]) {
      constexpr int kOdd = decltype(odd_c)::value;
      char* const kt = s_t + (1 - kOdd) * kTileB;
      char* const vt = s_v + ((i - 1) & 3) * kTileB;
      const float ck2 = scale_of(st[kOdd]);
      const Put to = put_begin(st[kOdd], i + 2);
      rescale(refp);
      float mx[NR], alpha[NR], p0[NR];
      bool moved[NR];
#pragma unroll
      for (int x = 0; x < NR; ++x) {
        mx[x] = -INFINITY;
        alpha[x] = 1.f;
        p0[x] = 0.f;
        moved[x] = false;
        Sn.s[x] = float16v(0.f);
      }
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
#pragma unroll
        for (int x = 0; x < NR; ++x) {
          Sn.s[x] = mfma<kHalf>(kop[s], Q[x][s], Sn.s[x]);
          O[x][s >> 1] = mfma<true>(vop[s], __builtin_bit_cast(bf16x8, Pp[x].p[s & 1]), O[x][s >> 1]);
        }
#pragma unroll
        for (int x = 0; x < NR; ++x) {
          float16v& Sx = S.s[x];
          if (s == 0) {                  // the tile's maximum
            if (i >= nfull) {
#pragma unroll
              for (int r = 0; r < 16; ++r)
                if (k0 + i * kTile + 8 * (r >> 2) + 4 * h + (r & 3) >= lim[x]) Sx[r] = -INFINITY;
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) mx[x] = fmaxf(mx[x], Sx[r]);
          } else if (s == 1) {
            const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx[x]), __float_as_uint(mx[x]), false, false);
            mx[x] = fmaxf(__uint_as_float(y[0]), __uint_as_float(y[1])) * ck0;
            moved[x] = __any(mx[x] > m[x] + (big[x] ? 0.f : kLazy));
            if (moved[x]) {
              const float mn = fmaxf(m[x], mx[x]);
              alpha[x] = __builtin_amdgcn_exp2f(m[x] - mn);
              l[x] *= alpha[x];
              m[x] = mn;
              // (as in oa_kv8_attn.hip: past 2^24 the product is rounded before the maximum is taken off)
              big[x] = __any(fabsf(m[x]) >= 16777216.f);
            }
            if (big[x]) {
#pragma unroll
              for (int r = 0; r < 16; ++r) Sx[r] *= ck0;
            }
          } else {
#pragma unroll
            for (int r = (s - 2) * 16 / (kSteps - 2); r < (s - 1) * 16 / (kSteps - 2); ++r) {
              const float p1 = __builtin_amdgcn_exp2f(fmaf(Sx[r], big[x] ? 1.f : ck0, kLift - m[x]));
              l[x] += p1;
              if (r & 1) {
                uint32_t u = pack2h(p0[x], p1);
                asm volatile("" : "+v"(u));        // (pinned here: left alone they all sink below the products)
                Pn[x].p[r >> 3][(r & 7) >> 1] = u;
              }
              p0[x] = p1;
            }
          }
        }
        if (s >= kSteps - 2 * kParts) {
          const int y = s - (kSteps - 2 * kParts);
          if (y < kParts) put_k(st[kOdd], kOdd, y);
          else put_v(to, st[kOdd], i + 2, y - kParts);
        }
        if (s == kSteps - 1) fetch(st[kOdd], i + 4, st[kOdd].next);
        __builtin_amdgcn_sched_barrier(0);
      }
      if (i > nfull) nan_rows(i - 1);
#pragma unroll
      for (int x = 0; x < NR; ++x)
        if (moved[x]) {                  // (after O += V(i - 1) P(i - 1), whose weights had the old maximum)
#pragma unroll
          for (int d = 0; d < kDims; ++d) O[x][d] *= alpha[x];
        }
      ck0 = ck1;
      ck1 = ck2;
      refp = ref0;
      ref0 = ref1;
      ref1 = ref;
      oa::lds_barrier();
    };
    typedef std::integral_constant<int, 0> even_t;
    typedef std::integral_constant<int, 1> odd_t;
    auto finish = [&](const Weights (&P)[NR]) {              // V(n - 1) P(n - 1)
      rescale(refp);
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const bf16x8 vop = val_op(s_v + ((n - 1) & 3) * kTileB, s >> 1, s & 1);
#pragma unroll
        for (int x = 0; x < NR; ++x) O[x][s >> 1] = mfma<true>(vop, __builtin_bit_cast(bf16x8, P[x].p[s & 1]), O[x][s >> 1]);
      }
      if (n > nfull) nan_rows(n - 1);
    };
#pragma unroll 1
    for (int i = 0; i < n; i += 2) {
      body(even_t(), i, S0, S1, P1, P0);
      if (i + 1 < n) body(odd_t(), i + 1, S1, S0, P0, P1);
    }
    if (n & 1) finish(P0);
    else finish(P1);
    const float f = any_power(held);
#pragma unroll
    for (int x = 0; x < NR; ++x)
#pragma unroll
      for (int d = 0; d < kDims; ++d) O[x][d] *= f;
  }

#pragma unroll
  for (int x = 0; x < NR; ++x) {
    const auto lx = __builtin_amdgcn_permlane32_swap(__float_as_uint(l[x]), __float_as_uint(l[x]), false, false);
    const float L = __uint_as_float(lx[0]) + __uint_as_float(lx[1]);
    if (row0 + (wave * NR + x) * kWaveRows + n32 >= rows) continue;
    if (a.nchunk == 1) {
      const float inv = 1.f / L;
      const bool none = lim[x] <= 0;
      uint16_t* o = a.out + (long)tok[x] * a.o_st + (long)hd[x] * a.o_sh + 4 * h;
#pragma unroll
      for (int d = 0; d < kDims; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          f32x4 y;
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] = sq.bad ? __builtin_nanf("") : none ? 0.f : O[x][d][4 * g + e] * inv;
          *reinterpret_cast<uint2v*>(o + 32 * d + 8 * g) = uint2v{pack_out<T>(y[0], y[1]), pack_out<T>(y[2], y[3])};
        }
    } else {
      const long at = ((long)tok[x] * (a.HKV * a.G) + hd[x]) * a.nchunk + ch;
#pragma unroll
      for (int d = 0; d < kDims; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<f32x4*>(a.ws_o + at * D + 32 * d + 8 * g + 4 * h) =
              f32x4{O[x][d][4 * g], O[x][d][4 * g + 1], O[x][d][4 * g + 2], O[x][d][4 * g + 3]};
      if (h == 0) *reinterpret_cast<f32x2*>(a.ws_ml + at * 2) = f32x2{m[x], L};
    }
  }
}

template <int D, typename T>
void launch_rows(const AttnArgs& a, dim3 grid, hipStream_t st) {
  if (a.rows == 128) hipLaunchKernelGGL((kv8_rows_kernel<D, 1, T>), grid, dim3(kThreads), 0, st, a);
  else hipLaunchKernelGGL((kv8_rows_kernel<D, 2, T>), grid, dim3(kThreads), 0, st, a);
}

}  // namespace

namespace kv8 {

void launch_rows(const AttnArgs& a, int head_dim, bool half, dim3 grid, hipStream_t st) {
  if (head_dim == 64) {
    if (half) ::launch_rows<64, _Float16>(a, grid, st);
    else ::launch_rows<64, __bf16>(a, grid, st);
  } else {
    if (half) ::launch_rows<128, _Float16>(a, grid, st);
    else ::launch_rows<128, __bf16>(a, grid, st);
  }
}

}  // namespace kv8
