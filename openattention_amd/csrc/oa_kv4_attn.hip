// Causal attention of the newest tokens of every sequence over a 4-bit paged cache (layout and codes:
// oa_kv4.hip):  out = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale q . k_t - max),  t up to the row's own
// position, in one pass over the keys with a running maximum and sum.
//
// One workgroup of four waves takes 16 NQ query rows of a KV head (row = token * G + head, so that any
// number of query heads fills the tiles) and a chunk of keys (ops.kv4_chunk says how many and why); each wave
// walks its own tiles of 32 keys and the waves join at the end.  With several chunks a second kernel joins them.
//   scores   S^T = K Q^T by v_mfma_f32_16x16x32_bf16: a lane of the K operand holds 32 dims of one key,
//            a block of the cache, whose codes become bf16 with one conversion per pair, scale included
//            (the contraction takes the dims in that order on both sides).  All products are exact.
//   values   O^T = V^T P^T: the weights are the B operand as the scores left them; V goes to bf16 the
//            same way, through the wave's own LDS tile, and comes back by the LDS transpose reads.
// Weights go into the product as two bf16 terms, so that the sum keeps 16 bits of each: up to 8 rows
// the second term sits in the tile's other 8 columns, otherwise it takes a second product.
//
// Bound by the codes read where rows are few: 32 sequences of 32768 keys, 8 KV heads, 1141 MB, 183 us with the
// join, 6.2 TB/s (in a train of launches of more than 2 ms the card slows: 190 to 245); one of 131072 keys 30 us
// (142 MB: 26 us and 4 for the join), where 512 workgroups each begin with three dependent accesses.  A workgroup's
// tile costs 64 conversions, 16 products and about 60 other vector instructions a wave.  Up to 64 rows of a KV head every workgroup turns its own keys to bf16 for 32 of them (64
// rows over 32768 keys, twice: 48 us against 59 in oa_kv4_rows.hip; from 96 rows on that one is faster).
#include "oa_kv4_attn.h"

namespace {

using namespace kv4;

__device__ __forceinline__ float max_groups(float v) {     // over the four 16-lane groups
  const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
  const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(y[0]), __uint_as_float(y[1]));
}
__device__ __forceinline__ float sum_groups(float v) {
  const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(x[0]) + __uint_as_float(x[1]);
  const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(y[0]) + __uint_as_float(y[1]);
}

// what the lanes of a wave exchange through its LDS tile stays in program order (the LDS keeps it)
__device__ __forceinline__ void lane_order() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local"); }

// one tile's codes and scales of this lane: keys lane % 16 and 16 + lane % 16, a quarter of the dims
template <int D>
struct Tile {
  unsigned k[2][D / 32], v[2][D / 32];
  unsigned ks[2], vs[2];
  unsigned bad;                          // the exponent of NaN where the page is outside of the cache
};

// ONCE: codes that no other workgroup reads pass by the caches (32 x 32768 keys: 206 us through them, 187)
template <bool ONCE, int N>
__device__ __forceinline__ void load_words(unsigned (&w)[N], const uint8_t* p) {
  typedef unsigned vec __attribute__((ext_vector_type(N)));
  const vec* q = reinterpret_cast<const vec*>(p);
  const vec x = ONCE ? __builtin_nontemporal_load(q) : *q;
#pragma unroll
  for (int i = 0; i < N; ++i) w[i] = x[i];
}

// NQ tiles of 16 query rows; DUP: at most 8 rows, columns 8.. repeat them for the weights' second terms
template <int D, int NQ, bool DUP>
__global__ void __launch_bounds__(kThreads, NQ > 1 ? 2 : 3) kv4_attn_kernel(AttnArgs a) {
  constexpr int kSteps = D / 32;         // products of a 16 x 16 score tile; words of a lane's codes
  constexpr int kDims = D / 16;          // tiles of 16 dims
  constexpr int kRowB = D * 2;           // bytes of a value row in LDS
  constexpr int kStage = kTile * kRowB;
  constexpr int kCols = DUP ? 8 : 16;
  // value tiles of the waves; at the end their sums, 16 rows of D floats each
  __shared__ __align__(16) char s_v[kWaves * (kStage > 64 * D ? kStage : 64 * D)];
  __shared__ float s_m[kWaves][NQ * 16], s_l[kWaves][NQ * 16];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, g = lane >> 4;
  // (sequence, head) fastest: workgroups go to the XCDs in turn, so that a long sequence's pieces and a
  // batch's short sequences spread over all of them, and the query tiles of a piece meet in one L2.  (Quotients
  // as products: with divisions before the first load 61 sequences of 1 to 16001 keys took 44.7 us for 43.3.)
  const int bh = blockIdx.x, row0 = blockIdx.y * (NQ * kCols), ch = blockIdx.z;
  const int b = a.by_hkv ? (int)__umulhi((unsigned)bh, a.by_hkv) : bh, h = bh - b * a.HKV;
  auto token_of = [&](int r) { return (int)((unsigned)r * a.by_g >> 16); };            // r / G
  // (the table's entries are requested beside the length: what lies past it is not used)
  constexpr int kStride = kWaves * kTile;
  const int k0 = ch * a.chunk, tb = k0 + wave * kTile;
  const int* trow = a.table + (long)b * a.t_st;
  auto page_at = [&](int t0) { return trow[min(t0 >> a.lp, a.width - 1)]; };
  const int page0 = page_at(tb);
  int page = page_at(tb + kStride);
  const Seq sq = seq_of(a, b);
  const int rows = min(sq.R, a.max_q) * a.G;
  if (row0 >= rows) return;
  const int first = sq.n - sq.R;         // position of the sequence's first query token
  const int hi = sq.bad ? 0 : first + token_of(min(row0 + NQ * kCols, rows) - 1) + 1;    // keys any row sees
  const int all = first + token_of(row0) + 1;                                              // keys every row sees
  const int k1 = min(k0 + a.chunk, hi);
  if (k0 >= k1 && a.nchunk > 1) return;

  // a tile's addresses: a scalar base and fixed lane offsets
  const int pmask = (1 << a.lp) - 1;
  const long headc = ((long)h << a.lp) * (D / 2), heads = ((long)h << a.lp) * (D / 32);
  const unsigned oc = col * (D / 2) + g * (D / 8), os = col * (D / 32) + g * D / 128;
  auto load = [&](Tile<D>& t, int t0, int page) {
    const bool bad = (unsigned)page >= (unsigned)a.NP;
    t.bad = bad ? 0x7f800000u : 0u;
    const long pg = bad ? 0 : page, off = t0 & pmask;
    const long bc = pg * a.c_sp + headc + off * (D / 2), bs = pg * a.s_sp + heads + off * (D / 32);
    const uint8_t* kc = a.kc + bc;
    const uint8_t* vc = a.vc + bc;
    const uint8_t* ks = a.ks + bs;
    const uint8_t* vs = a.vs + bs;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      load_words<NQ == 1>(t.k[c], kc + oc + 16 * c * (D / 2));
      t.ks[c] = ks[os + 16 * c * (D / 32)];
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      load_words<NQ == 1>(t.v[c], vc + oc + 16 * c * (D / 2));
      t.vs[c] = vs[os + 16 * c * (D / 32)];
    }
  };
  const int nt = max(0, (k1 - tb + kStride - 1) / kStride);                  // this wave's tiles
  const int nfull = min(nt, max(0, (all - tb - kTile + kStride) / kStride));  // those that every row sees whole
  Tile<D> ta, tc;
  if (nt > 0) load(ta, tb, page0);

  // this lane's columns: rows of q (negated under a negative scale: the maximum is taken before scaling)
  // and how many keys they see (0: no such row)
  const float c = fabsf(a.c);
  const unsigned flip = a.c < 0.f ? 0x80008000u : 0u;
  bf16x8 Q[NQ][kSteps];
  int lim[NQ];
#pragma unroll
  for (int x = 0; x < NQ; ++x) {
    const int r = row0 + x * kCols + (DUP ? col & 7 : col);
    const int rr = min(r, rows - 1), j = token_of(rr), hd = h * a.G + rr - j * a.G;
    lim[x] = r < rows ? first + j + 1 : 0;
    const uint16_t* p = a.q + (long)(sq.r0 + j) * a.q_st + (long)hd * a.q_sh + g * (D / 4);
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const uint4v w = *reinterpret_cast<const uint4v*>(p + 8 * s);
      Q[x][s] = __builtin_bit_cast(bf16x8, w ^ uint4v(flip));
    }
  }

  // LDS tile of 32 value rows; 16-byte chunk x of row r lies at x ^ f(r): 16 rows written at one chunk
  // and 16 rows read at two both spread over all banks
  char* const sv = s_v + wave * kStage;
  auto fsw = [](int r) { return D == 128 ? ((r & 3) << 2) | ((r >> 2) & 3) : ((r >> 1) & 3) << 1; };
  const int wbase = col * kRowB, wf = fsw(col);
  const int lr = 4 * g + ((lane & 15) >> 2), rf = fsw(lr), lc = lane & 3;
  auto val_op = [&](int d) {
    const int ad = lr * kRowB + (((2 * d + (lc >> 1)) ^ rf) << 4) + (lc & 1) * 8;
    const short4v x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4v*)(sv + ad));
    const short4v y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4v*)(sv + ad + 16 * kRowB));
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
  };

  f32x4 O[NQ][kDims];
  float m[NQ], l[NQ];                    // running maximum, scaled, and sum of the lane's keys
  bool big[NQ];                          // a maximum is past 2^24 (uniform)
#pragma unroll
  for (int x = 0; x < NQ; ++x) {
    m[x] = -FLT_MAX;
    l[x] = 0.f;
    big[x] = false;
#pragma unroll
    for (int d = 0; d < kDims; ++d) O[x][d] = f32x4(0.f);
  }


  // tile i from t; tile i + 1 is fetched into n
  auto body = [&](auto mask_c, int i, const Tile<D>& t, Tile<D>& n) {
    constexpr bool MASK = decltype(mask_c)::value;
    const int t0 = tb + i * kStride;
    if (i + 1 < nt) {
      load(n, t0 + kStride, page);
      page = page_at(t0 + 2 * kStride);
    }
    f32x4 S[NQ][2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const float f = __uint_as_float(t.ks[c] << 23 | t.bad);
#pragma unroll
      for (int x = 0; x < NQ; ++x) S[x][c] = f32x4(0.f);
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const bf16x8 kop = from4(t.k[c][s], f);
#pragma unroll
        for (int x = 0; x < NQ; ++x) S[x][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kop, Q[x][s], S[x][c], 0, 0, 0);
      }
    }
    // values into the LDS tile.  In a masked tile keys past the last one any row sees count as zeros (their
    // weights are 0, but what lies there may be anything), and so do NaN blocks of keys that some rows see
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      unsigned e = t.vs[c];
      if (MASK && (t0 + 16 * c + col >= hi || e == 255)) e = 0;
      const float f = __uint_as_float(e << 23);
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
        *reinterpret_cast<bf16x8*>(sv + wbase + 16 * c * kRowB + (((g * (D / 32) + s) ^ wf) << 4)) = from4(t.v[c][s], f);
    }
    lane_order();

    uint4v P[NQ], Plo[NQ];
#pragma unroll
    for (int x = 0; x < NQ; ++x) {
      float v[8];
      float mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = S[x][i >> 2][i & 3];
        if (MASK) v[i] = t0 + 16 * (i >> 2) + 4 * g + (i & 3) < lim[x] ? v[i] * c : -INFINITY;
        mx = fmaxf(mx, v[i]);
      }
      if (!MASK) mx *= c;
      if (__any(mx > m[x])) {
        const float mn = fmaxf(m[x], max_groups(mx)), alpha = __builtin_amdgcn_exp2f(m[x] - mn);
        m[x] = mn;
        l[x] *= alpha;
#pragma unroll
        for (int d = 0; d < kDims; ++d) O[x][d] *= alpha;
        // the maximum rounds S c, so that the fma below leaves up to half its last place: past 2^24 more than
        // the exponential should see, and an infinity in time.  There S c is rounded first, as the maximum is
        big[x] = __any(fabsf(mn) >= 16777216.f);
      }
      if (!MASK && big[x]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= c;
      }
      const float cc = MASK || big[x] ? 1.f : c;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = __builtin_amdgcn_exp2f(MASK ? v[i] - m[x] : fmaf(v[i], cc, -m[x]));
        l[x] += v[i];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t u = pack2(v[2 * i], v[2 * i + 1]);
        const uint32_t lo = pack2(v[2 * i] - __uint_as_float(u << 16), v[2 * i + 1] - __uint_as_float(u & 0xffff0000u));
        P[x][i] = DUP && (lane & 8) ? lo : u;
        Plo[x][i] = lo;
      }
    }
#pragma unroll
    for (int d = 0; d < kDims; ++d) {
      const bf16x8 vop = val_op(d);
#pragma unroll
      for (int x = 0; x < NQ; ++x) {
        O[x][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vop, __builtin_bit_cast(bf16x8, P[x]), O[x][d], 0, 0, 0);
        if (!DUP) O[x][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vop, __builtin_bit_cast(bf16x8, Plo[x]), O[x][d], 0, 0, 0);
      }
    }
    lane_order();
    if (MASK) {                          // NaN blocks, into the rows that see them (rare)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        unsigned long nan = __ballot(t.vs[c] == 255 && t0 + 16 * c + col < hi);
        while (nan) {
          const int at = __builtin_ctzl(nan), key = t0 + 16 * c + (at & 15), blk = (at >> 4) * D / 128;
          nan &= nan - 1;
#pragma unroll
          for (int x = 0; x < NQ; ++x)
#pragma unroll
            for (int d = 0; d < kDims; ++d)
              if (d / 2 == blk && key < lim[x]) O[x][d] = f32x4(__builtin_nanf(""));
        }
      }
    }
  };
  {
    typedef std::integral_constant<bool, false> whole;
    typedef std::integral_constant<bool, true> masked;
    int i = 0;
#pragma unroll 1
    for (; i < nfull; ++i) {             // (two tiles to a turn, without the copies: 186 us for 182)
      body(whole(), i, ta, tc);
      ta = tc;
    }
#pragma unroll 1
    for (; i < nt; ++i) {
      body(masked(), i, ta, tc);
      ta = tc;
    }
  }

  // the four waves' sums, with a common maximum
#pragma unroll
  for (int x = 0; x < NQ; ++x) {
    const float lt = sum_groups(l[x]);
    if (g == 0) {
      s_m[wave][x * 16 + col] = m[x];
      s_l[wave][x * 16 + col] = lt;
    }
  }
  float* const so = reinterpret_cast<float*>(s_v);
#pragma unroll
  for (int x = 0; x < NQ; ++x) {
    __syncthreads();                     // (every wave is done with its tile, or with the previous sums)
    const int sc = x * 16 + col;
    const float M = fmaxf(fmaxf(s_m[0][sc], s_m[1][sc]), fmaxf(s_m[2][sc], s_m[3][sc]));
    const float e = __builtin_amdgcn_exp2f(m[x] - M);
#pragma unroll
    for (int d = 0; d < kDims; ++d)      // 16-byte chunk y of column col at y ^ col
      *reinterpret_cast<f32x4*>(so + (wave * 16 + col) * D + (((4 * d + g) ^ col) << 2)) = O[x][d] * e;
    __syncthreads();
    constexpr int kChunks = D / 4;
    for (int i = threadIdx.x; i < kCols * kChunks; i += kThreads) {
      const int cl = i / kChunks, y = i % kChunks, r = row0 + x * kCols + cl;
      if (r >= rows) continue;
      const int c16 = x * 16 + cl;
      const float Mr = fmaxf(fmaxf(s_m[0][c16], s_m[1][c16]), fmaxf(s_m[2][c16], s_m[3][c16]));
      float L = 0.f;
      f32x4 o = f32x4(0.f);
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        L += s_l[w][c16] * __builtin_amdgcn_exp2f(s_m[w][c16] - Mr);
        o += *reinterpret_cast<const f32x4*>(so + (w * 16 + cl) * D + ((y ^ cl) << 2));
        if (DUP) o += *reinterpret_cast<const f32x4*>(so + (w * 16 + 8 + cl) * D + ((y ^ (8 + cl)) << 2));
      }
      const int j = token_of(r), hd = h * a.G + r - j * a.G;
      if (a.nchunk == 1) {
        const int seen = first + j + 1;
        o = sq.bad ? f32x4(__builtin_nanf("")) : seen > 0 ? o / L : f32x4(0.f);
        *reinterpret_cast<uint2v*>(a.out + (long)(sq.r0 + j) * a.o_st + (long)hd * a.o_sh + 4 * y) =
            uint2v{pack2(o[0], o[1]), pack2(o[2], o[3])};
      } else {
        const long at = ((long)(sq.r0 + j) * (a.HKV * a.G) + hd) * a.nchunk + ch;
        *reinterpret_cast<f32x4*>(a.ws_o + at * D + 4 * y) = o;
        if (y == 0) *reinterpret_cast<f32x2*>(a.ws_ml + at * 2) = f32x2{Mr, L};
      }
    }
  }
}

// Zeros in the rows of out that no sequence takes: those before the first and behind the last by all workgroups
// of the join together, and head hd of sequence b's rows past max_q (all of its rows, where they do not fit) by
// the one of its first row.  In the join, as it costs a launch to fill out beforehand (5 drafts of 7 sequences
// 19.5 us a call, 15.5 here) and the attention kernel 4 to 13 us (one sequence of 131072 keys 30.6 to 35.6, 32 of
// 32768 184 to 197), even where there is nothing to clear.
template <int D>
__device__ __forceinline__ void clear_rows(const AttnArgs& a, int b, int hd, bool own) {
  constexpr int kLanes = D / 4, kRows = kThreads / kLanes;     // lanes of a row, 8 bytes each
  const int y = threadIdx.x % kLanes, x = threadIdx.x / kLanes, heads = a.HKV * a.G;
  auto zero = [&](int tok, int head) {
    *reinterpret_cast<uint2v*>(a.out + (long)tok * a.o_st + (long)head * a.o_sh + 4 * y) = uint2v(0u);
  };
  auto in_out = [&](int t) { return min(max(t, 0), a.tokens); };
  const int lead = in_out(a.cu[0]), tail = in_out(a.cu[a.B]);
  const long n = (long)(lead + a.tokens - tail) * heads, blocks = (long)gridDim.x * gridDim.y;
  for (long i = ((long)blockIdx.y * gridDim.x + blockIdx.x) * kRows + x; i < n; i += blocks * kRows) {
    const int t = (int)(i / heads);
    zero(t < lead ? t : tail + t - lead, (int)(i % heads));
  }
  if (!own) return;
  const int r0 = a.cu[b], r1 = a.cu[b + 1];
  const bool fits = r0 >= 0 && r1 >= r0 && r1 <= a.tokens;
  const int t0 = fits ? r0 + min(r1 - r0, a.max_q) : in_out(r0), t1 = fits ? r1 : in_out(r1);
  for (int t = t0 + x; t < t1; t += kRows) zero(t, hd);
}

// joins a row's chunks: weights exp2(m_i - max m), by groups of D / 4 lanes
template <int D>
__global__ void __launch_bounds__(kThreads) kv4_join_kernel(AttnArgs a) {
  constexpr int kLanes = D / 4, kGroups = kThreads / kLanes;
  __shared__ float s_r[kWaves];
  __shared__ __align__(16) float s_o[kGroups][D];
  __shared__ float s_l[kGroups];
  const int heads = a.HKV * a.G;
  const int hd = blockIdx.x % heads, j = blockIdx.x / heads, b = blockIdx.y;
  const Seq sq = seq_of(a, b);
  if (a.clear) clear_rows<D>(a, b, hd, j == 0);
  if (j >= sq.R) return;
  const int seen = sq.n - sq.R + j + 1, tid = threadIdx.x;
  const int nv = sq.bad || seen <= 0 ? 0 : (seen + a.chunk - 1) / a.chunk;
  const long row = ((long)(sq.r0 + j) * heads + hd) * a.nchunk;
  const float* ml = a.ws_ml + row * 2;
  const int grp = tid / kLanes, y = tid % kLanes;
  constexpr int kAtOnce = 4;             // pieces whose loads are in flight together
  f32x4 x[kAtOnce];
  f32x2 w[kAtOnce];
  auto fetch = [&](int i) {
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const int at = min(i + k * kGroups, nv - 1);
      x[k] = *reinterpret_cast<const f32x4*>(a.ws_o + (row + at) * D + 4 * y);
      w[k] = *reinterpret_cast<const f32x2*>(ml + 2 * at);
    }
  };
  if (grp < nv) fetch(grp);              // (beside the maxima: one sequence of 131072 keys 30.9 us, 32.2 after them)
  float M = -FLT_MAX;
  for (int i = tid; i < nv; i += kThreads) M = fmaxf(M, ml[2 * i]);
  M = oa::wave_max(M);
  if ((tid & 63) == 0) s_r[tid >> 6] = M;
  __syncthreads();
  M = fmaxf(fmaxf(s_r[0], s_r[1]), fmaxf(s_r[2], s_r[3]));
  f32x4 o = f32x4(0.f);
  float L = 0.f;
  for (int i = grp; i < nv; i += kAtOnce * kGroups) {
    if (i > grp) fetch(i);
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      if (i + k * kGroups >= nv) break;
      const float e = __builtin_amdgcn_exp2f(w[k][0] - M);
      L += e * w[k][1];
      o += x[k] * e;
    }
  }
  *reinterpret_cast<f32x4*>(&s_o[grp][4 * y]) = o;
  if (y == 0) s_l[grp] = L;
  __syncthreads();
  if (grp) return;
#pragma unroll
  for (int k = 1; k < kGroups; ++k) {
    o += *reinterpret_cast<const f32x4*>(&s_o[k][4 * y]);
    L += s_l[k];
  }
  o = sq.bad ? f32x4(__builtin_nanf("")) : nv ? o / L : f32x4(0.f);
  *reinterpret_cast<uint2v*>(a.out + (long)(sq.r0 + j) * a.o_st + (long)hd * a.o_sh + 4 * y) =
      uint2v{pack2(o[0], o[1]), pack2(o[2], o[3])};
}

// query rows up to which every workgroup turns its own keys to bf16 (more: oa_kv4_rows.hip)
constexpr int kFewRows = 64;
constexpr long kGrid = 0xffffffffL / kThreads;

template <int D>
int launch(AttnArgs a, hipStream_t st) {
  const long rows = (long)a.max_q * a.G;
  const int cols = rows <= 8 ? 8 : rows <= 16 ? 16 : rows <= kFewRows ? 32 : 128;
  a.ntile = (int)((rows + cols - 1) / cols);
  const long units = (long)a.B * a.HKV, blocks = a.ntile * units * a.nchunk, joins = (long)a.max_q * a.HKV * a.G;
  // (a grid's threads along one axis are counted in 32 bits, its workgroups along the others in 16)
  if (blocks > kGrid || a.nchunk > 65535 || (a.nchunk > 1 && (joins > kGrid || a.B > 65535))) return OA_EINVAL;
  // quotients as products with 2^16 / G + 1 and 2^32 / HKV, rounded up: exact while the number times the divisor is
  // less than that power (rows and G are at most 64 here)
  if (cols < 128 && units * a.HKV > 0xffffffffL) return OA_EINVAL;
  a.by_g = 65536u / a.G + 1;
  a.by_hkv = a.HKV > 1 ? (unsigned)((0x100000000L + a.HKV - 1) / a.HKV) : 0;
  const dim3 grid((unsigned)units, a.ntile, a.nchunk), blk(kThreads);
  if (cols == 8) hipLaunchKernelGGL((kv4_attn_kernel<D, 1, true>), grid, blk, 0, st, a);
  else if (cols == 16) hipLaunchKernelGGL((kv4_attn_kernel<D, 1, false>), grid, blk, 0, st, a);
  else if (cols == 32) hipLaunchKernelGGL((kv4_attn_kernel<D, 2, false>), grid, blk, 0, st, a);
  else launch_rows(a, D, dim3((unsigned)blocks), st);
  if (a.nchunk > 1) hipLaunchKernelGGL((kv4_join_kernel<D>), dim3((unsigned)joins, a.B), blk, 0, st, a);
  return OA_LAUNCH_STATUS();
}

}  // namespace

extern "C" int oa_kv4_attn(const void* q, long q_st, long q_sh, const void* kc, const void* ks, const void* vc,
                           const void* vs, long code_stride, long scale_stride, int pages, int page, const int* table,
                           long table_stride, int width, const int* lens, const int* cu, int sequences, int tokens,
                           int max_q, int q_heads, int kv_heads, int head_dim, float sm_scale, int chunk, int nchunk,
                           float* ws_o, float* ws_ml, int* ws_flag, void* out, long o_st, long o_sh, int clear,
                           void* stream) {
  auto odd = [](const void* p, uintptr_t n) { return !p || (reinterpret_cast<uintptr_t>(p) & (n - 1)) != 0; };
  if ((head_dim != 64 && head_dim != 128) || sequences < 0 || tokens < 0 || max_q <= 0 || kv_heads <= 0 || q_heads <= 0 ||
      q_heads % kv_heads || (long)max_q * (q_heads / kv_heads) > (1L << 30) || pages <= 0 || page < 32 || page > 1024 ||
      (page & (page - 1)) || (long)pages * page > 0x7fffffffL || width <= 0 || (long)width * page > (1L << 30) ||
      table_stride < width || chunk < 128 || chunk % 128 || nchunk <= 0 || (long)nchunk * chunk > (1L << 30) + (1L << 29))
    return OA_EINVAL;
  if (!cu && (max_q != 1 || sequences != tokens)) return OA_EINVAL;
  if (!sequences || !tokens) return 0;
  if (odd(q, 16) || q_st % 8 || q_sh % 8 || odd(out, 8) || o_st % 4 || o_sh % 4 || odd(kc, 16) || odd(ks, 16) || odd(vc, 16) ||
      odd(vs, 16) || !table || !lens || code_stride < (long)kv_heads * page * (head_dim / 2) ||
      scale_stride < (long)kv_heads * page * (head_dim / 32) || code_stride % 16 || scale_stride % 16 ||
      code_stride > 0xffffffffL || scale_stride > 0xffffffffL || !(sm_scale == sm_scale))
    return OA_EINVAL;
  if (out == q) return OA_EINVAL;        // (rows may be read again after others were written)
  if ((nchunk > 1 && (odd(ws_o, 16) || odd(ws_ml, 8))) || ((long)max_q * (q_heads / kv_heads) > kFewRows && odd(ws_flag, 4)))
    return OA_EINVAL;
  AttnArgs a;
  a.q = (const uint16_t*)q; a.q_st = q_st; a.q_sh = q_sh;
  a.kc = (const uint8_t*)kc; a.ks = (const uint8_t*)ks; a.vc = (const uint8_t*)vc; a.vs = (const uint8_t*)vs;
  a.c_sp = code_stride; a.s_sp = scale_stride;
  a.table = table; a.t_st = table_stride; a.lens = lens; a.cu = cu;
  a.out = (uint16_t*)out; a.o_st = o_st; a.o_sh = o_sh;
  a.ws_o = ws_o; a.ws_ml = ws_ml; a.ws_flag = ws_flag;
  a.B = sequences; a.HKV = kv_heads; a.G = q_heads / kv_heads; a.tokens = tokens; a.max_q = max_q;
  a.width = width; a.NP = pages; a.lp = __builtin_ctz(page); a.chunk = chunk; a.nchunk = nchunk;
  a.clear = cu && clear;
  a.c = sm_scale * kLog2e;
  return head_dim == 64 ? launch<64>(a, (hipStream_t)stream) : launch<128>(a, (hipStream_t)stream);
}
