// Page tables of a paged cache kept on the device: the pages, slots and positions of the tokens that
// requests add (oa_kv_pages_extend), and pages given back (oa_kv_pages_truncate).
//
// State: table (requests, width) of page ids (-1: none), lens (requests) tokens held, free (pages) a
// stack of the ids that no request holds and nfree, how many they are (the top is free[nfree - 1]).
// Request i holds ceil(lens_i / page) pages.  An extension pops pages in the order of requests and of
// their pages, a truncation pushes them so that the stack is what it was before the extension that it
// undoes: page k of R popped pages was at nfree - 1 - k, page k of R returned ones goes to
// nfree + R - 1 - k.  Both take effect for all requests or for none; what went wrong is or-ed into
// *status (1: a negative count to add, a length outside of its row of the table; 2: too few free pages, or
// more than a stack can hold; 4: more tokens than the caller has slots for).
//
// One workgroup adds up what every request needs (a scan over the requests, as many threads as there are up
// to 1024), decides, and writes lengths, starts and the stack's height; with few tokens or requests it also
// writes slots and pages.  For many, a second launch does: a lane per token finds its request by bisection
// of the starts, a wave per request moves its returned pages.  Bound by the latency of its few dependent
// accesses: 32 requests that add a token and take it
// back 5.5 us, 1000 that add 360000 tokens and give them back 13.4 (captured calls).
#include "oa_common.h"

namespace {

constexpr int kMost = 1024;              // threads of the planning workgroup
constexpr int kFill = 256;
constexpr int kStarts = 4096;            // starts that a workgroup of the second launch holds in LDS
// tokens up to which the planning workgroup writes the slots itself
constexpr int kAlone = 2048;
constexpr unsigned kFull = 0x7fffffffu;  // what sums stop at

struct PagesArgs {
  const int* count;                      // tokens to add, or to keep
  int* lens;
  int* table; long t_st;
  int* free; int* nfree; int* status;
  int B, width, NP, lp, total;
  int* slots; int* pos; int* cu;
  int* ws;                               // length, first new page of each request (2 B), stack height
};

__device__ __forceinline__ unsigned add_to(unsigned a, unsigned b) { return min(a + b, kFull); }   // (both at most kFull)

// inclusive sum over the lanes of a wave, stopping at kFull
__device__ __forceinline__ unsigned wave_scan(unsigned v) {
  v = add_to(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, false));     // row_shr 1, 2, 4, 8
  v = add_to(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, false));
  v = add_to(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, false));
  v = add_to(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, false));
  v = add_to(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false));     // rows 0 to 1, 2 to 3
  return add_to(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false));  // rows 1 to 2, 3
}

template <int THREADS>
struct Scan {
  unsigned part[2][THREADS / 64];
};

// inclusive sums of two values over the workgroup and their totals
template <int THREADS>
__device__ __forceinline__ void block_scan(Scan<THREADS>& s, unsigned& a, unsigned& b, unsigned& ta, unsigned& tb) {
  a = wave_scan(a);
  b = wave_scan(b);
  if (THREADS == 64) {
    ta = (unsigned)__builtin_amdgcn_readlane((int)a, 63);
    tb = (unsigned)__builtin_amdgcn_readlane((int)b, 63);
    return;
  }
  const int wave = threadIdx.x >> 6;
  __syncthreads();
  if ((threadIdx.x & 63) == 63) {
    s.part[0][wave] = a;
    s.part[1][wave] = b;
  }
  __syncthreads();
  unsigned oa = 0, ob = 0;
  ta = tb = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) {
    if (w == wave) {
      oa = ta;
      ob = tb;
    }
    ta = add_to(ta, s.part[0][w]);
    tb = add_to(tb, s.part[1][w]);
  }
  a = add_to(a, oa);
  b = add_to(b, ob);
}

__device__ __forceinline__ int pages_of(int tokens, int lp) { return (tokens + (1 << lp) - 1) >> lp; }   // (at most 2^30 + page)

// lengths outside of what a row of the table can hold count as its nearest end
__device__ __forceinline__ int held_len(const PagesArgs& a, int i) { return min(max(a.lens[i], 0), a.width << a.lp); }

// slot and position of token t, and, from the first token on a new page, the table's entry.  cu: the starts
__device__ __forceinline__ void fill_token(const PagesArgs& a, const int* cu, const int* len_of, const int* new_of, int t,
                                           int nfree) {
  int lo = 0, n = a.B;                   // the last request that starts at or before t
  while (n > 1) {
    const int half = n >> 1;
    if (cu[lo + half] <= t) lo += half;
    n -= half;
  }
  const int len = len_of[lo], p = len + t - cu[lo], at = p >> a.lp, held = pages_of(len, a.lp);
  int* row = a.table + (long)lo * a.t_st;
  const int id = at >= held ? a.free[nfree - 1 - (new_of[lo] + at - held)] : row[at];
  if (at >= held && (p & ((1 << a.lp) - 1)) == 0) row[at] = id;
  a.slots[t] = (unsigned)id < (unsigned)a.NP ? (id << a.lp) + (p & ((1 << a.lp) - 1)) : -1;
  a.pos[t] = p;
}

// a request's tokens and pages to add; what cannot be is noted in *bad
__device__ __forceinline__ void wanted(const PagesArgs& a, int i, int& len, int& n, int& need, int* bad) {
  n = a.count[i];
  const int have = a.lens[i];
  len = held_len(a, i);
  if (n < 0 || len != have || n > (a.width << a.lp) - len) {
    atomicOr(bad, 1);
    n = 0;
  }
  need = pages_of(len + n, a.lp) - pages_of(len, a.lp);
}

// THREADS: 64 (the requests fit a wave), 256, 1024 (any number of requests)
template <int THREADS>
__global__ void __launch_bounds__(THREADS) pages_extend_kernel(PagesArgs a, int alone) {
  __shared__ Scan<THREADS> s;
  __shared__ int s_bad;
  __shared__ int s_cu[THREADS], s_len[THREADS], s_new[THREADS];
  const int tid = threadIdx.x;
  const bool once = a.B <= THREADS;
  if (tid == 0) s_bad = 0;
  const int nfree = min(max(*a.nfree, 0), a.NP);
  __syncthreads();
  // what all requests need
  unsigned tokens = 0, pages = 0, e0 = 0, e1 = 0;
  int len = 0, n = 0, need = 0;
  for (int i0 = 0; i0 < a.B; i0 += THREADS) {
    const int i = i0 + tid;
    len = n = need = 0;
    if (i < a.B) wanted(a, i, len, n, need, &s_bad);
    unsigned t0, t1;
    e0 = n;
    e1 = need;
    block_scan<THREADS>(s, e0, e1, t0, t1);
    tokens = add_to(tokens, t0);
    pages = add_to(pages, t1);
  }
  __syncthreads();
  const int bad = s_bad | (pages > (unsigned)nfree ? 2 : 0) | (tokens > (unsigned)a.total ? 4 : 0);
  if (bad && tid == 0) *a.status |= bad;
  // starts, lengths (sums that a refused call may have cut short are not used)
  unsigned tok0 = 0, page0 = 0;
  for (int i0 = 0; i0 < a.B; i0 += THREADS) {
    const int i = i0 + tid;
    unsigned t0 = tokens, t1 = pages;
    if (!once) {
      len = n = need = 0;
      if (i < a.B && !bad) wanted(a, i, len, n, need, &s_bad);
      e0 = n;
      e1 = need;
      block_scan<THREADS>(s, e0, e1, t0, t1);
    }
    if (i < a.B) {
      const int end = bad ? 0 : (int)(tok0 + e0), at = bad ? 0 : end - n, page = (int)(page0 + e1) - need;
      a.cu[i + 1] = end;
      if (i == 0) a.cu[0] = 0;
      if (once) {
        s_cu[tid] = at;
        s_len[tid] = len;
        s_new[tid] = page;
      }
      if (!once || !alone) {
        a.ws[i] = len;
        a.ws[a.B + i] = page;
      }
      if (!bad) a.lens[i] = len + n;
    }
    tok0 += t0;
    page0 += t1;
  }
  if (tid == 0) {
    if (!alone) a.ws[2 * a.B] = nfree;
    if (!bad) *a.nfree = nfree - (int)pages;
  }
  if (!alone) return;
  __syncthreads();                       // (starts and lengths of the whole workgroup)
  for (int t = tid; t < a.total; t += THREADS) {
    if (bad || t >= (int)tokens) a.slots[t] = a.pos[t] = -1;
    else if (once) fill_token(a, s_cu, s_len, s_new, t, nfree);
    else fill_token(a, a.cu, a.ws, a.ws + a.B, t, nfree);
  }
}

__global__ void __launch_bounds__(kFill) pages_fill_kernel(PagesArgs a) {
  __shared__ int s_cu[kStarts];
  const int t = blockIdx.x * kFill + threadIdx.x, end = a.cu[a.B], nfree = a.ws[2 * a.B];
  const bool near = a.B <= kStarts;
  if (near) {
    for (int i = threadIdx.x; i < a.B; i += kFill) s_cu[i] = a.cu[i];
    __syncthreads();
  }
  if (t >= a.total) return;
  if (t >= end) a.slots[t] = a.pos[t] = -1;
  else if (near) fill_token(a, s_cu, a.ws, a.ws + a.B, t, nfree);
  else fill_token(a, a.cu, a.ws, a.ws + a.B, t, nfree);
}

// the returned pages of a request, by the lanes of one wave
__device__ __forceinline__ void give_back(const PagesArgs& a, int i, int left, int gone, int first, int top, int lane) {
  int* row = a.table + (long)i * a.t_st + left;
  for (int c = lane; c < gone; c += 64) {
    a.free[top - 1 - (first + c)] = row[c];
    row[c] = -1;
  }
}

template <int THREADS>
__global__ void __launch_bounds__(THREADS) pages_truncate_kernel(PagesArgs a, int alone) {
  __shared__ Scan<THREADS> s;
  __shared__ int s_bad;
  __shared__ int s_left[THREADS], s_gone[THREADS], s_first[THREADS];
  const int tid = threadIdx.x;
  const bool once = a.B <= THREADS;
  if (tid == 0) s_bad = 0;
  const int nfree = min(max(*a.nfree, 0), a.NP);
  __syncthreads();
  unsigned pages = 0, e0 = 0, e1 = 0, t1;
  int gone = 0, keep = 0;
  auto returned = [&](int i) {
    gone = keep = 0;
    if (i < a.B) {
      const int len = held_len(a, i), k = a.count[i];
      if (len != a.lens[i]) atomicOr(&s_bad, 1);
      keep = k < 0 ? len : min(k, len);
      gone = pages_of(len, a.lp) - pages_of(keep, a.lp);
    }
  };
  for (int i0 = 0; i0 < a.B; i0 += THREADS) {
    unsigned t0;
    returned(i0 + tid);
    e0 = gone;
    e1 = 0;
    block_scan<THREADS>(s, e0, e1, t0, t1);
    pages = add_to(pages, t0);
  }
  __syncthreads();
  const int bad = s_bad | (pages > (unsigned)(a.NP - nfree) ? 2 : 0);
  const int top = nfree + (bad ? 0 : (int)pages);
  unsigned page0 = 0;
  for (int i0 = 0; i0 < a.B; i0 += THREADS) {
    const int i = i0 + tid;
    unsigned t0 = pages;
    if (!once) {
      returned(i);
      e0 = gone;
      e1 = 0;
      block_scan<THREADS>(s, e0, e1, t0, t1);
    }
    if (i < a.B) {
      const int left = pages_of(keep, a.lp), first = (int)(page0 + e0) - gone, g = bad ? 0 : gone;
      if (alone) {                       // (then all requests have a thread)
        s_left[tid] = left;
        s_gone[tid] = g;
        s_first[tid] = first;
      } else {
        a.ws[i] = left;
        a.ws[a.B + i] = first;
        a.ws[2 * a.B + 1 + i] = g;
      }
      if (!bad) a.lens[i] = keep;
    }
    page0 = add_to(page0, t0);
  }
  if (tid == 0) {
    if (!alone) a.ws[2 * a.B] = top;
    if (bad) *a.status |= bad;
    else *a.nfree = top;
  }
  if (!alone) return;
  __syncthreads();
  for (int i = tid >> 6; i < a.B; i += THREADS / 64) give_back(a, i, s_left[i], s_gone[i], s_first[i], top, tid & 63);
}

__global__ void __launch_bounds__(kFill) pages_back_kernel(PagesArgs a) {
  const int i = blockIdx.x * (kFill / 64) + (threadIdx.x >> 6);
  if (i >= a.B) return;
  give_back(a, i, a.ws[i], a.ws[2 * a.B + 1 + i], a.ws[a.B + i], a.ws[2 * a.B], threadIdx.x & 63);
}

// requests up to which the planning workgroup moves the returned pages itself (at most its threads)
constexpr int kAloneRows = 256;

int take(PagesArgs& a, const int* count, int* lens, int* table, long t_st, int* free, int* nfree, int* status, int B,
         int width, int NP, int page, int* ws) {
  if (!count || !lens || !table || !free || !nfree || !status || B <= 0 || width <= 0 || t_st < width || NP <= 0 ||
      page < 32 || page > 1024 || (page & (page - 1)) || (long)NP * page > 0x7fffffffL || (long)width * page > (1L << 30) ||
      B > (1 << 24))
    return OA_EINVAL;
  a = PagesArgs{};
  a.count = count; a.lens = lens; a.table = table; a.t_st = t_st; a.free = free; a.nfree = nfree; a.status = status;
  a.B = B; a.width = width; a.NP = NP; a.lp = __builtin_ctz(page); a.ws = ws;
  return 0;
}

}  // namespace

extern "C" int oa_kv_pages_extend(const int* add, int* lens, int* table, long table_stride, int* free, int* nfree,
                                  int* status, int requests, int width, int pages, int page, int total, int* slots,
                                  int* pos, int* cu, int* ws, void* stream) {
  PagesArgs a;
  if (const int e = take(a, add, lens, table, table_stride, free, nfree, status, requests, width, pages, page, ws)) return e;
  if (total < 0 || total > 0x7fffff00 || (total && (!slots || !pos)) || !cu || (!ws && (requests > kMost || total > kAlone)))
    return OA_EINVAL;
  a.total = total; a.slots = slots; a.pos = pos; a.cu = cu;
  const hipStream_t st = (hipStream_t)stream;
  const int alone = total <= kAlone;
  if (requests <= 64 && total <= 256) hipLaunchKernelGGL(pages_extend_kernel<64>, dim3(1), dim3(64), 0, st, a, alone);
  else if (requests <= 256 && total <= 512) hipLaunchKernelGGL(pages_extend_kernel<256>, dim3(1), dim3(256), 0, st, a, alone);
  else hipLaunchKernelGGL(pages_extend_kernel<kMost>, dim3(1), dim3(kMost), 0, st, a, alone);
  if (!alone) hipLaunchKernelGGL(pages_fill_kernel, dim3((total + kFill - 1) / kFill), dim3(kFill), 0, st, a);
  return OA_LAUNCH_STATUS();
}

extern "C" int oa_kv_pages_truncate(const int* keep, int* lens, int* table, long table_stride, int* free, int* nfree,
                                    int* status, int requests, int width, int pages, int page, int* ws, void* stream) {
  PagesArgs a;
  if (const int e = take(a, keep, lens, table, table_stride, free, nfree, status, requests, width, pages, page, ws)) return e;
  if (!ws && requests > kAloneRows) return OA_EINVAL;
  const hipStream_t st = (hipStream_t)stream;
  const int alone = requests <= kAloneRows;
  if (requests <= 16) hipLaunchKernelGGL(pages_truncate_kernel<64>, dim3(1), dim3(64), 0, st, a, alone);
  else if (requests <= 64) hipLaunchKernelGGL(pages_truncate_kernel<256>, dim3(1), dim3(256), 0, st, a, alone);
  else hipLaunchKernelGGL(pages_truncate_kernel<kMost>, dim3(1), dim3(kMost), 0, st, a, alone);
  if (!alone)
    hipLaunchKernelGGL(pages_back_kernel, dim3((requests + kFill / 64 - 1) / (kFill / 64)), dim3(kFill), 0, st, a);
  return OA_LAUNCH_STATUS();
}
