// Block tables, slots and positions of a serving step, from the lengths of its sequences.
//
// With c tokens cached and a added, a sequence needs ceil((c + a) / page) - ceil(c / page) new pages; where its
// tokens and its pages begin are two exclusive prefix sums over the sequences (the second leaves out
// sequences whose tokens have no place, which the first tells).  Every new page has exactly one new token at
// its row 0, so the thread of that token writes the table's entry, and nothing waits for another
// workgroup: each one forms both sums itself, from lengths that are a few KB and in L2, and serves its own run of
// tokens by a search in LDS.
//
// Bound: latency.  The two sums are four trips through LDS and barriers behind one load; the tokens add a
// search, one dependent load (a free page or an old entry) and their stores.
#include "kernels.h"

namespace w4k {
namespace {

constexpr int PT_ITEMS = 4;  // tokens of a thread

// What a sequence asks for, before it is known whether pages are left.
struct Wish {
  long long first, need;  // the first page that is not in the table, and how many
  bool bad, over;
};
__device__ __forceinline__ Wish wish_of(const PagedTables& t, long long c, long long a, long long at) {
  Wish w;
  w.bad = c < 0 || a < 0 || c + a > min((long long)t.stride * t.page, 2147483647LL);
  w.over = a > 0 && at + a > t.tokens;
  // (lengths are 32-bit, and so are the quotients' operands where they count)
  const uint32_t page = (uint32_t)t.page;
  w.first = w.bad ? 0 : ((uint32_t)c + page - 1) / page;
  w.need = w.bad || w.over ? 0 : (long long)(((uint32_t)(c + a) + page - 1) / page) - w.first;
  return w;
}

// Exclusive prefix sum over the workgroup; `total` of all.  sums: one entry per wave.
template <int T>
__device__ __forceinline__ long long exclusive_sum(long long v, long long* sums, long long& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  long long x = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const long long y = __shfl_up(x, d, 64);
    if (lane >= d) x += y;
  }
  if (lane == 63) sums[wave] = x;
  __syncthreads();
  long long before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < T / 64; ++w) {
    const long long s = sums[w];
    if (w < wave) before += s;
    total += s;
  }
  __syncthreads();
  return before + x - v;
}

template <int T>
__global__ __launch_bounds__(T) void paged_tables_kernel(const PagedTables t) {
  __shared__ long long sums[T / 64];
  __shared__ long long tok_at[T], page_at[T];  // where each thread's run of sequences begins
  __shared__ int found[2];
  const int tid = threadIdx.x;
  const int per = (t.nseq + T - 1) / T;
  const int lo = min(tid * per, t.nseq), hi = min(lo + per, t.nseq);
  const long long begin = t.free_range[0];
  const long long left = max(0LL, (long long)t.free_range[1] - begin);
  if (tid == 0) found[0] = found[1] = 0;

  long long mine = 0, all_tokens, all_pages;
  for (int s = lo; s < hi; ++s) mine += max(t.added[s], 0);
  const long long tok0 = exclusive_sum<T>(mine, sums, all_tokens);
  long long need = 0, at = tok0;
  for (int s = lo; s < hi; ++s) {
    const long long a = t.added[s];
    need += wish_of(t, t.cached[s], a, at).need;
    at += max(a, 0LL);
  }
  const long long page0 = exclusive_sum<T>(need, sums, all_pages);
  tok_at[tid] = tok0;
  page_at[tid] = page0;

  if (blockIdx.x == 0) {  // what there is one of per sequence
    long long pre = page0, taken = 0;
    int status = 0;
    at = tok0;
    for (int s = lo; s < hi; ++s) {
      const long long c = t.cached[s], a = t.added[s];
      const Wish w = wish_of(t, c, a, at);
      const bool lacks = w.need > 0 && pre + w.need > left;
      status |= lacks | w.bad << 1 | w.over << 2;
      if (w.need > 0 && !lacks) taken = pre + w.need;
      t.lens[s] = (int)(lacks || w.bad || w.over ? max(c, 0LL) : c + a);
      t.cu[s] = (int)min(at, 2147483647LL);
      at += max(a, 0LL);
      pre += w.need;
      if (s == t.nseq - 1) t.cu[t.nseq] = (int)min(at, 2147483647LL);
    }
    if (status) atomicOr(&found[1], status);
    if (taken) atomicMax(&found[0], (int)taken);
  }
  __syncthreads();
  if (blockIdx.x == 0 && tid == 0) t.result[0] = found[0], t.result[1] = found[1];

  const long long run0 = (long long)blockIdx.x * (T * PT_ITEMS);
#pragma unroll
  for (int k = 0; k < PT_ITEMS; ++k) {
    const long long i = run0 + k * T + tid;
    if (i >= t.tokens) break;
    int slot = -1, pos = -1;
    if (i < all_tokens) {
      // the last run of sequences that begins at or before token i ...
      int a0 = 0;
#pragma unroll
      for (int half = T / 2; half > 0; half >>= 1)
        if (tok_at[a0 + half] <= i) a0 += half;
      // ... and in it the sequence that holds it (there is one: i < all_tokens)
      int s = min(a0 * per, t.nseq - 1);
      long long off = tok_at[a0], pre = page_at[a0];
      while (s < t.nseq - 1 && i >= off + max(t.added[s], 0)) {
        pre += wish_of(t, t.cached[s], t.added[s], off).need;
        off += max(t.added[s], 0);
        ++s;
      }
      const long long c = t.cached[s];
      const Wish w = wish_of(t, c, t.added[s], off);
      if (!(w.bad || w.over || (w.need > 0 && pre + w.need > left))) {
        const uint32_t p = (uint32_t)(c + (i - off)), pg = p / (uint32_t)t.page, r = p - pg * (uint32_t)t.page;
        int* const entry = t.bt + (long long)s * t.stride + pg;
        const bool fresh = (long long)pg >= w.first;
        const int id = fresh ? t.free_pages[begin + pre + ((long long)pg - w.first)] : *entry;
        if (fresh && r == 0) *entry = id;
        pos = (int)p;
        if (id >= 0 && id < t.npages) slot = id * t.page + (int)r;
      }
    }
    t.slots[i] = slot;
    t.positions[i] = pos;
  }
}

}  // namespace

hipError_t launch_paged_tables(const PagedTables& a, hipStream_t s) {
  // up to 256 sequences a thread has one at most, and four waves meet faster than sixteen
  if (a.nseq <= 256) {
    const int per = 256 * PT_ITEMS;
    paged_tables_kernel<256><<<max(1, (a.tokens + per - 1) / per), 256, 0, s>>>(a);
  } else {
    const int per = 1024 * PT_ITEMS;
    paged_tables_kernel<1024><<<max(1, (a.tokens + per - 1) / per), 1024, 0, s>>>(a);
  }
  return hipGetLastError();
}

}  // namespace w4k
