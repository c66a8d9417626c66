// Page tables of a paged cache kept on the device: the pages, slots and positions of the tokens that
// requests add (oa_kv_pages_extend), and pages given back (oa_kv_pages_truncate).
//
// State: table (requests, width) of page ids (-1: none), lens (requests) tokens held, free (pages) a
// stack of the ids that no request holds and nfree, how many they are (the top is free[nfree - 1]).
// Request i holds ceil(lens_i / page) pages.  An extension pops pages in the order of requests and of
// their pages, a truncation pushes them so that the stack is what it was before the extension that it
// undoes: page k of R popped pages was at nfree - 1 - k, page k of R returned ones goes to
// nfree + R - 1 - k.  Both take effect for all requests or for none; what went wrong is or-ed into
// *status (1: a negative count or a request longer than its row of the table; 2: too few free pages, or
// more than a stack can hold; 4: more tokens than the caller has slots for).
//
// One workgroup adds up what every request needs (a scan over the requests), decides, and writes
// lengths, starts and the stack's height; with few tokens it also writes slots and pages.  For many,
// a second launch does: a lane per token finds its request by bisection of the starts.
#include "oa_common.h"

namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kFill = 256;
// tokens up to which the planning workgroup writes the slots itself
constexpr int kAlone = 2048;

struct PagesArgs {
  const int* count;                      // tokens to add, or to keep
  int* lens;
  int* table; long t_st;
  int* free; int* nfree; int* status;
  int B, width, NP, lp, total;
  int* slots; int* pos; int* cu;
  int* ws;                               // length, first new page of each request (2 B), stack height
};

// inclusive sum over the lanes of a wave
__device__ __forceinline__ long wave_scan(long v, int lane) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const long o = __shfl_up(v, d);
    if (lane >= d) v += o;
  }
  return v;
}

struct Scan {
  long part[2][kWaves];
};

// exclusive sums of two values over the workgroup and their totals (two barriers)
__device__ __forceinline__ void block_scan(Scan& s, long a, long b, long& ea, long& eb, long& ta, long& tb) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long ia = wave_scan(a, lane), ib = wave_scan(b, lane);
  __syncthreads();
  if (lane == 63) {
    s.part[0][wave] = ia;
    s.part[1][wave] = ib;
  }
  __syncthreads();
  ea = ia - a;
  eb = ib - b;
  ta = tb = 0;
  for (int w = 0; w < kWaves; ++w) {
    const long x = s.part[0][w], y = s.part[1][w];
    if (w < wave) {
      ea += x;
      eb += y;
    }
    ta += x;
    tb += y;
  }
}

__device__ __forceinline__ long pages_of(long tokens, int lp) { return (tokens + (1L << lp) - 1) >> lp; }

// lengths outside of what a row of the table can hold count as its nearest end
__device__ __forceinline__ long held_len(const PagesArgs& a, int i) {
  return min(max((long)a.lens[i], 0l), (long)a.width << a.lp);
}

// slot and position of token t, and, from the first token on a new page, the table's entry
__device__ __forceinline__ void fill_token(const PagesArgs& a, int t, int nfree) {
  int lo = 0, hi = a.B - 1;              // the last request that starts at or before t
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.cu[mid] <= t) lo = mid;
    else hi = mid - 1;
  }
  const int len = a.ws[lo], p = len + t - a.cu[lo], at = p >> a.lp, held = (int)pages_of(len, a.lp);
  int* row = a.table + (long)lo * a.t_st;
  const int id = at >= held ? a.free[nfree - 1 - (a.ws[a.B + lo] + at - held)] : row[at];
  if (at >= held && (p & ((1 << a.lp) - 1)) == 0) row[at] = id;
  a.slots[t] = (unsigned)id < (unsigned)a.NP ? (id << a.lp) + (p & ((1 << a.lp) - 1)) : -1;
  a.pos[t] = p;
}

__global__ void __launch_bounds__(kThreads) pages_extend_kernel(PagesArgs a, int alone) {
  __shared__ Scan s;
  __shared__ int s_bad;
  const int tid = threadIdx.x;
  if (tid == 0) s_bad = 0;
  __syncthreads();
  const int nfree = min(max(*a.nfree, 0), a.NP);
  // what all requests need
  long tokens = 0, pages = 0;
  for (int i0 = 0; i0 < a.B; i0 += kThreads) {
    const int i = i0 + tid;
    long n = 0, need = 0;
    if (i < a.B) {
      n = a.count[i];
      const long len = held_len(a, i);
      if (n < 0 || len != a.lens[i] || len + n > (long)a.width << a.lp) {
        atomicOr(&s_bad, 1);
        n = 0;
      }
      need = pages_of(len + n, a.lp) - pages_of(len, a.lp);
    }
    long e0, e1, t0, t1;
    block_scan(s, n, need, e0, e1, t0, t1);
    tokens += t0;
    pages += t1;
  }
  __syncthreads();
  const int bad = s_bad | (pages > nfree ? 2 : 0) | (tokens > a.total ? 4 : 0);
  if (bad && tid == 0) *a.status |= bad;
  // starts, lengths
  long tok0 = 0, page0 = 0;
  for (int i0 = 0; i0 < a.B; i0 += kThreads) {
    const int i = i0 + tid;
    long n = 0, need = 0, len = 0;
    if (i < a.B && !bad) {
      n = a.count[i];
      len = a.lens[i];
      need = pages_of(len + n, a.lp) - pages_of(len, a.lp);
    }
    long e0, e1, t0, t1;
    block_scan(s, n, need, e0, e1, t0, t1);
    if (i < a.B) {
      a.cu[i + 1] = (int)(tok0 + e0 + n);
      if (i == 0) a.cu[0] = 0;
      a.ws[i] = (int)len;
      a.ws[a.B + i] = (int)(page0 + e1);
      if (!bad) a.lens[i] = (int)(len + n);
    }
    tok0 += t0;
    page0 += t1;
  }
  if (tid == 0) {
    a.ws[2 * a.B] = nfree;
    if (!bad) *a.nfree = nfree - (int)page0;
  }
  if (!alone) return;
  __syncthreads();                       // (starts and lengths of the whole workgroup, through memory)
  for (int t = tid; t < a.total; t += kThreads) {
    if (t < tok0) fill_token(a, t, nfree);
    else a.slots[t] = a.pos[t] = -1;
  }
}

__global__ void __launch_bounds__(kFill) pages_fill_kernel(PagesArgs a) {
  const int t = blockIdx.x * kFill + threadIdx.x;
  if (t >= a.total) return;
  if (t < a.cu[a.B]) fill_token(a, t, a.ws[2 * a.B]);
  else a.slots[t] = a.pos[t] = -1;
}

// the returned pages of request i, by the lanes of one wave
__device__ __forceinline__ void give_back(const PagesArgs& a, int i, long left, long held, long first, int top, int lane) {
  int* row = a.table + (long)i * a.t_st;
  for (long c = left + lane; c < held; c += 64) {
    a.free[top - 1 - (first + c - left)] = row[c];
    row[c] = -1;
  }
}

__global__ void __launch_bounds__(kThreads) pages_truncate_kernel(PagesArgs a, int alone) {
  __shared__ Scan s;
  const int tid = threadIdx.x;
  const int nfree = min(max(*a.nfree, 0), a.NP);
  long pages = 0;
  for (int i0 = 0; i0 < a.B; i0 += kThreads) {
    const int i = i0 + tid;
    long gone = 0, e0, e1, t0, t1;
    if (i < a.B) {
      const long len = held_len(a, i), keep = a.count[i] < 0 ? len : min((long)a.count[i], len);
      gone = pages_of(len, a.lp) - pages_of(keep, a.lp);
    }
    block_scan(s, gone, 0, e0, e1, t0, t1);
    pages += t0;
  }
  const bool bad = nfree + pages > a.NP;
  if (bad && tid == 0) *a.status |= 2;
  long page0 = 0;
  for (int i0 = 0; i0 < a.B; i0 += kThreads) {
    const int i = i0 + tid;
    long gone = 0, len = 0, keep = 0, e0, e1, t0, t1;
    if (i < a.B) {
      len = held_len(a, i);
      keep = bad || a.count[i] < 0 ? len : min((long)a.count[i], len);
      gone = pages_of(len, a.lp) - pages_of(keep, a.lp);
    }
    block_scan(s, gone, 0, e0, e1, t0, t1);
    if (i < a.B) {
      a.ws[i] = (int)pages_of(keep, a.lp);
      a.ws[a.B + i] = (int)(page0 + e0);
      a.ws[2 * a.B + 1 + i] = (int)gone;
      if (!bad) a.lens[i] = (int)keep;
    }
    page0 += t0;
  }
  if (tid == 0) {
    a.ws[2 * a.B] = nfree + (int)page0;
    if (!bad) *a.nfree = nfree + (int)page0;
  }
  if (!alone) return;
  __syncthreads();
  for (int i = tid >> 6; i < a.B; i += kWaves)
    give_back(a, i, a.ws[i], (long)a.ws[i] + a.ws[2 * a.B + 1 + i], a.ws[a.B + i], nfree + (int)page0, tid & 63);
}

__global__ void __launch_bounds__(kFill) pages_back_kernel(PagesArgs a) {
  const int i = blockIdx.x * (kFill / 64) + (threadIdx.x >> 6);
  if (i >= a.B) return;
  give_back(a, i, a.ws[i], (long)a.ws[i] + a.ws[2 * a.B + 1 + i], a.ws[a.B + i], a.ws[2 * a.B], threadIdx.x & 63);
}

// requests up to which the planning workgroup moves the returned pages itself
constexpr int kAloneRows = 256;

int take(PagesArgs& a, const int* count, int* lens, int* table, long t_st, int* free, int* nfree, int* status, int B,
         int width, int NP, int page, int* ws) {
  if (!count || !lens || !table || !free || !nfree || !status || !ws || B <= 0 || width <= 0 || t_st < width || NP <= 0 ||
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
  if (total < 0 || total > 0x7fffff00 || (total && (!slots || !pos)) || !cu) return OA_EINVAL;
  a.total = total; a.slots = slots; a.pos = pos; a.cu = cu;
  const hipStream_t st = (hipStream_t)stream;
  const int alone = total <= kAlone;
  hipLaunchKernelGGL(pages_extend_kernel, dim3(1), dim3(kThreads), 0, st, a, alone);
  if (!alone) hipLaunchKernelGGL(pages_fill_kernel, dim3((total + kFill - 1) / kFill), dim3(kFill), 0, st, a);
  return OA_LAUNCH_STATUS();
}

extern "C" int oa_kv_pages_truncate(const int* keep, int* lens, int* table, long table_stride, int* free, int* nfree,
                                    int* status, int requests, int width, int pages, int page, int* ws, void* stream) {
  PagesArgs a;
  if (const int e = take(a, keep, lens, table, table_stride, free, nfree, status, requests, width, pages, page, ws)) return e;
  const hipStream_t st = (hipStream_t)stream;
  const int alone = requests <= kAloneRows;
  hipLaunchKernelGGL(pages_truncate_kernel, dim3(1), dim3(kThreads), 0, st, a, alone);
  if (!alone)
    hipLaunchKernelGGL(pages_back_kernel, dim3((requests + kFill / 64 - 1) / (kFill / 64)), dim3(kFill), 0, st, a);
  return OA_LAUNCH_STATUS();
}
