// Paged FP8 attention for many rows: the kernel by itself, and how its work is spread.
#include <math.h>

#include "pages_many.cuh"

namespace w4k {
namespace {

template <int D, bool P16>
__global__ __launch_bounds__(PM_WAVES * 64, D <= 128 ? 2 : 1) void pages_many_kernel(const Pages a) {
  __shared__ ManyShared<D, P16> sh;
  many_rows<D, P16>(a, blockIdx.x, blockIdx.y, sh);
}

template <int D>
hipError_t go(const Pages& a, hipStream_t s) {
  const dim3 grid((unsigned)(pages_many_tiles(a, a.few_rows) * a.H), (unsigned)a.many.nsplit);
  if (a.page % 16 == 0) pages_many_kernel<D, true><<<grid, PM_WAVES * 64, 0, s>>>(a);
  else pages_many_kernel<D, false><<<grid, PM_WAVES * 64, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace

long long pages_many_tiles(const PagesArgs& a, int few_rows) {
  const long long rows = (long long)a.tokens * a.group, seqs = rows / (few_rows + 1);
  const long long each = ((long long)a.max_q * a.group + PM_ROWS - 1) / PM_ROWS;
  const long long packed = rows / PM_ROWS + (seqs < a.nseq ? seqs : a.nseq);
  return packed < each * a.nseq ? packed : each * a.nseq;
}

// One round of workgroups (a little less, or a little more), no split shorter than 512 positions, if that takes less time than no
// splits: splits cost what they write and read again and a launch, and shorten the chain of tiles of a workgroup, 1.55 us for
// 64 positions at D = 128 alone on a compute unit, 2.25 next to another one.  1024 tokens of 32 heads take 33 us in one split, 47 in
// two; 512 behind 1500 54 in one, 44 in four; 1024 behind 8000 220 in one, 193 in two.  256 positions at least instead of 512: 150
// calls take the same on average, from 0.9 to 1.3 times as long.
// Splits are cut from max_len, the only length that the host has: under a bound far above the lengths one split does all of a
// sequence (a chunk of 512 tokens at 8192 next to decoding sequences 126 us under its own bound, 222 under four times that).
PagesPlan pages_many_plan(const PagesArgs& a, int few_rows) {
  // (next to a prompt the other sequences have a token each, which is not this kernel's, as far as the host can tell)
  const long long tokens = few_rows && a.tokens - (a.nseq - 1) > a.max_q ? a.tokens - (a.nseq - 1) : few_rows ? a.max_q : a.tokens;
  const long long tiles = (tokens * a.group + PM_ROWS - 1) / PM_ROWS * a.H;
  const long long steps = (a.max_len + PM_TILE - 1) / PM_TILE, most = (a.max_len + 511) / 512;
  const int each = a.D <= 128 ? 2 : 1;  // workgroups of a compute unit
  const double us = 0.4 + 0.6 * a.D / 128;
  auto takes = [&](long long n) {
    // whole rounds, and what is left over: rows of a prompt differ in length, so a few workgroups more are not a whole round more
    const long long full = tiles * n / (256 * each), rest = tiles * n % (256 * each);
    const double last = rest > 256 ? 2.25 : full ? 1.55 * sqrt(rest / 256.0) : 1.55;
    const double chain = (steps + n - 1) / n * us * (full * (each == 2 ? 2.25 : 1.55) + last);
    return n > 1 ? chain + 3.5 + tiles * PM_ROWS * n * (a.D + 2) * 8 / 5e6 : chain;
  };
  const long long down = tiles > 0 ? 256 * each / tiles : 1;
  long long best = 1;
  for (long long n = down; n <= down + 1; ++n) {
    const long long k = n > most ? most : n;
    if (k > 1 && takes(k) < takes(best)) best = k;
  }
  PagesPlan p;
  p.split_len = (int)((steps + best - 1) / best * PM_TILE);
  p.nsplit = (a.max_len + p.split_len - 1) / p.split_len;
  return p;
}

hipError_t launch_pages_many(const Pages& a, hipStream_t s) {
  switch (a.D) {
    case 64: return go<64>(a, s);
    case 96: return go<96>(a, s);
    case 128: return go<128>(a, s);
    default: return go<256>(a, s);
  }
}

}  // namespace w4k
