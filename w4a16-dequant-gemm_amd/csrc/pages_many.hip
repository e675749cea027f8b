// Paged FP8 attention for many rows: the kernel by itself, and how its work is spread.
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

PagesPlan pages_many_plan(const PagesArgs& a) {
  // two workgroups per compute unit where the rows do not give them, no split shorter than 512 positions (256: 150 calls take
  // the same on average, from 0.9 to 1.3 times as long)
  const long long tiles = ((long long)a.tokens * a.group + PM_ROWS - 1) / PM_ROWS * a.H;
  const int most = (a.max_len + 511) / 512;
  long long n = tiles > 0 ? (512 + tiles - 1) / tiles : 1;
  n = n > most ? most : n < 1 ? 1 : n;
  PagesPlan p;
  p.split_len = (int)(((a.max_len + n - 1) / n + PM_TILE - 1) / PM_TILE * PM_TILE);
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
