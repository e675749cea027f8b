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
// search, one dependent load (a free page or an old entry) and their stores.  64 sequences with a token each: 2.8 us on the
// device, 4.0 us a call when calls follow each other; 333 prompts with 67317 tokens: 5.6 us.
#include "pages.cuh"

namespace w4k {
namespace {

// Sums saturate at 2^32 - 1: every comparison they enter is with less than 2^31.
__device__ __forceinline__ uint32_t plus(uint32_t a, uint32_t b) { return __builtin_elementwise_add_sat(a, b); }

struct Tables : PagedTables {
  Divider by_page;
  uint32_t most;  // the longest sequence: what a table holds, and positions are ints
};

// What a sequence asks for, before it is known whether pages are left.
struct Wish {
  uint32_t first, need;  // the first page that is not in the table, and how many
  bool bad, over;
};
__device__ __forceinline__ Wish wish_of(const Tables& t, int c, int a, uint32_t at) {
  Wish w;
  const uint32_t all = (uint32_t)c + (uint32_t)a;
  w.bad = c < 0 || a < 0 || all > t.most;
  w.over = a > 0 && plus(at, (uint32_t)a) > (uint32_t)t.tokens;
  const bool none = w.bad || w.over;
  w.first = none || c == 0 ? 0 : t.by_page(c - 1) + 1;
  w.need = none || all == 0 ? 0 : t.by_page((int)all - 1) + 1 - w.first;
  return w;
}

// Exclusive prefix sum over the workgroup; `total` of all.  sums: one entry per wave, not used again before a barrier.
template <int T>
__device__ __forceinline__ uint32_t exclusive_sum(uint32_t v, uint32_t* sums, uint32_t& total) {
  const int wave = threadIdx.x >> 6;
  const uint32_t x = (uint32_t)wave_scan((int)v, 0, [](int a, int b) { return (int)plus((uint32_t)a, (uint32_t)b); });
  if ((threadIdx.x & 63) == 63) sums[wave] = x;
  __syncthreads();
  uint32_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < T / 64; ++w) {
    const uint32_t s = sums[w];
    if (w < wave) before = plus(before, s);
    total = plus(total, s);
  }
  // (a wave's exclusive sum is its neighbour's inclusive one, also where sums saturate)
  const uint32_t left = (uint32_t)__builtin_amdgcn_ds_bpermute(4 * ((threadIdx.x & 63) - 1), (int)x);
  return plus(before, threadIdx.x & 63 ? left : 0u);
}

// ONE: a thread has one sequence at most.
template <int T, bool ONE>
__global__ __launch_bounds__(T) void paged_tables_kernel(const Tables t) {
  __shared__ uint32_t sums[2][T / 64];
  __shared__ uint32_t tok_at[T], page_at[T];  // where each thread's run of sequences begins
  __shared__ int found[2];
  const int tid = threadIdx.x;
  const int per = ONE ? 1 : (t.nseq + T - 1) / T;
  const int lo = min(tid * per, t.nseq), hi = min(lo + per, t.nseq);
  const int begin = t.free_range[0];
  const long long between = (long long)t.free_range[1] - begin;
  const uint32_t left = (uint32_t)max(0LL, between);
  if (tid == 0) found[0] = found[1] = 0;
  // the thread's first sequence stays in registers
  const int c0 = lo < hi ? t.cached[lo] : 0, a0 = lo < hi ? t.added[lo] : 0;
  auto cached = [&](int s) { return ONE || s == lo ? c0 : t.cached[s]; };
  auto added = [&](int s) { return ONE || s == lo ? a0 : t.added[s]; };

  uint32_t mine = 0, all_tokens, all_pages;
  for (int s = lo; s < hi; ++s) mine = plus(mine, (uint32_t)max(added(s), 0));
  const uint32_t tok0 = exclusive_sum<T>(mine, sums[0], all_tokens);
  uint32_t need = 0, at = tok0;
  for (int s = lo; s < hi; ++s) {
    need = plus(need, wish_of(t, cached(s), added(s), at).need);
    at = plus(at, (uint32_t)max(added(s), 0));
  }
  const uint32_t page0 = exclusive_sum<T>(need, sums[1], all_pages);
  tok_at[tid] = tok0;
  page_at[tid] = page0;

  if (blockIdx.x == 0) {  // what there is one of per sequence
    uint32_t pre = page0, taken = 0;
    int status = 0;
    at = tok0;
    for (int s = lo; s < hi; ++s) {
      const int c = cached(s), a = added(s);
      const Wish w = wish_of(t, c, a, at);
      const bool lacks = w.need > 0 && plus(pre, w.need) > left;
      status |= lacks | w.bad << 1 | w.over << 2;
      if (w.need > 0 && !lacks) taken = pre + w.need;
      t.lens[s] = lacks || w.bad || w.over ? max(c, 0) : c + a;
      t.cu[s] = (int)min(at, 2147483647u);
      at = plus(at, (uint32_t)max(a, 0));
      pre = plus(pre, w.need);
      if (s == t.nseq - 1) t.cu[t.nseq] = (int)min(at, 2147483647u);
    }
    if (status) atomicOr(&found[1], status);
    if (taken) atomicMax(&found[0], (int)taken);
  }
  __syncthreads();
  if (blockIdx.x == 0 && tid == 0) t.result[0] = found[0], t.result[1] = found[1];

  const long long i = (long long)blockIdx.x * T + tid;
  if (i >= t.tokens) return;
  int slot = -1, pos = -1;
  if (i < (long long)all_tokens) {
    const uint32_t tok = (uint32_t)i;
    // the last run of sequences that begins at or before the token ...
    int run = 0;
#pragma unroll
    for (int half = T / 2; half > 0; half >>= 1)
      if (tok_at[run + half] <= tok) run += half;
    // ... and in it the sequence that holds it (there is one: tok < all_tokens)
    int s = min(run * per, t.nseq - 1);
    uint32_t off = tok_at[run], pre = page_at[run];
    if constexpr (!ONE)
      while (s < t.nseq - 1 && tok >= plus(off, (uint32_t)max(t.added[s], 0))) {
        pre = plus(pre, wish_of(t, t.cached[s], t.added[s], off).need);
        off = plus(off, (uint32_t)max(t.added[s], 0));
        ++s;
      }
    const int c = t.cached[s];
    const Wish w = wish_of(t, c, t.added[s], off);
    if (!(w.bad || w.over || (w.need > 0 && plus(pre, w.need) > left))) {
      const int p = c + (int)(tok - off), pg = t.by_page(p), r = p - pg * t.page;
      int* const entry = t.bt + (long long)s * t.stride + pg;
      const bool fresh = (uint32_t)pg >= w.first;
      const int id = fresh ? t.free_pages[(long long)begin + pre + ((uint32_t)pg - w.first)] : *entry;
      if (fresh && r == 0) *entry = id;
      pos = p;
      if (id >= 0 && id < t.npages) slot = id * t.page + r;
    }
  }
  t.slots[i] = slot;
  t.positions[i] = pos;
}

}  // namespace

hipError_t launch_paged_tables(const PagedTables& args, hipStream_t s) {
  Tables a;
  (PagedTables&)a = args;
  a.by_page = divider(a.page);
  const long long holds = (long long)a.stride * a.page;
  a.most = holds < 2147483647LL ? (uint32_t)holds : 2147483647u;
  // up to 256 sequences a thread has one at most, and four waves meet faster than sixteen: 3.0 us against 3.4 on the device
  const int T = a.nseq <= 256 ? 256 : 1024;
  const unsigned grid = (unsigned)max(1, (int)(((long long)a.tokens + T - 1) / T));
  if (T == 256) paged_tables_kernel<256, true><<<grid, 256, 0, s>>>(a);
  else if (a.nseq <= 1024) paged_tables_kernel<1024, true><<<grid, 1024, 0, s>>>(a);
  else paged_tables_kernel<1024, false><<<grid, 1024, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace w4k
