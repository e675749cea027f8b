// Paged FP8 attention of decoding sequences next to prompts: the work of both kernels in one launch.
//
// Workgroups for few rows come first, half a round of them (plan() has where it is more): they wait for memory, those for many
// rows for the vector ALUs.
// Where no sequence has few rows (only the device knows), they end at once and cost no launch.  A chunk of 512 tokens at 8192
// next to 15 decoding sequences: 125.6 us, 129.6 in two launches, 153 with workgroups of both kinds in turn, eight by eight (one
// kind to one half of the compute units); 36 calls of prompts and chunks: 0.89 of the time of two launches on average, 0.92
// with a whole round for few rows.
#include "pages_few.cuh"
#include "pages_many.cuh"

namespace w4k {
namespace {

template <int D, int NB>
__global__ __launch_bounds__(256, D <= 128 ? 2 : 1) void pages_mixed_kernel(const Pages a, const int tiles) {
  __shared__ union {
    FewShared<D> few;
    ManyShared<D, true> many;
  } sh;
  const int at = (int)blockIdx.x - a.few.grid;
  if (at >= 0) many_rows<D, true>(a, at % tiles, at / tiles, sh.many);
  else few_rows<D, 1, true, NB>(a, blockIdx.x, sh.few);
}

template <int D>
hipError_t go(const Pages& a, hipStream_t s) {
  const int tiles = (int)(pages_many_tiles(a, a.few_rows) * a.H);
  const unsigned grid = (unsigned)a.few.grid + (unsigned)tiles * (unsigned)a.many.nsplit;
  if (a.nseq <= 64) pages_mixed_kernel<D, 1><<<grid, 256, 0, s>>>(a, tiles);
  else pages_mixed_kernel<D, 4><<<grid, 256, 0, s>>>(a, tiles);
  return hipGetLastError();
}

}  // namespace

// (Other pages, and more than 16 query heads to a KV head, are rare next to prompts: two launches.)
bool pages_mixed_applies(const Pages& a) { return a.few.block == 16 && !a.few.alone && a.page % 16 == 0; }

hipError_t launch_pages_mixed(const Pages& a, hipStream_t s) {
  switch (a.D) {
    case 64: return go<64>(a, s);
    case 96: return go<96>(a, s);
    case 128: return go<128>(a, s);
    default: return go<256>(a, s);
  }
}

}  // namespace w4k
