// Paged FP8 attention for few rows: the kernel by itself, and how its work is spread.
#include "pages_few.cuh"

namespace w4k {
namespace {

template <int D, int NT, bool PG4, int NB>
__global__ __launch_bounds__(PF_WAVES * 64) void pages_few_kernel(const Pages a) {
  __shared__ FewShared<D> sh;
  few_rows<D, NT, PG4, NB>(a, blockIdx.x, sh);
}

template <int D, int NT, bool PG4>
void go_share(const Pages& a, hipStream_t s) {
  const unsigned grid = (unsigned)a.few.grid;
  if (a.few.alone) pages_few_kernel<D, NT, PG4, 0><<<grid, 256, 0, s>>>(a);
  else if (a.nseq <= 64) pages_few_kernel<D, NT, PG4, 1><<<grid, 256, 0, s>>>(a);
  else pages_few_kernel<D, NT, PG4, 4><<<grid, 256, 0, s>>>(a);
}
template <int D, int NT>
void go_page(const Pages& a, hipStream_t s) {
  if (a.page % 4 == 0) go_share<D, NT, true>(a, s);
  else go_share<D, NT, false>(a, s);
}
template <int D>
hipError_t go(const Pages& a, hipStream_t s) {
  if (a.few.block == 16) go_page<D, 1>(a, s);
  else go_page<D, 2>(a, s);
  return hipGetLastError();
}

}  // namespace

bool pages_few_applies(const PagesArgs& a) {
  return (a.D == 64 || a.D == 96 || a.D == 128 || a.D == 256) && (((uintptr_t)a.q_k | (uintptr_t)a.q_v) & 15) == 0;
}

FewPlan pages_few_plan(const PagesArgs& a, long long rows, bool half) {
  // What runs at a time: two workgroups per compute unit (three at D = 64: 19.1 us for the ragged ones instead of 18.6), one
  // where LDS leaves no more.
  const int places = a.D == 256 || half ? 256 : 512;
  FewPlan p{};
  p.block = rows <= 16 ? 16 : 32;  // 4 rows in blocks of 32: 91.9 us instead of 89.1 (8 x 32768), 7.5 instead of 6.5 (4 x 300)
  p.blocks = (int)((rows + p.block - 1) / p.block);
  p.rows = rows < p.block ? (int)rows : p.block;
  const long long units = (long long)a.nseq * a.H * p.blocks;
  // Units are not split where many of them fill the card without it (256 sequences of 1000 positions, 32 heads: 321 us against
  // 357 in splits; of 200 to 2000: 355 against 382), and beyond 256 sequences a workgroup does not look for its share (what that
  // costs where one is much longer than the rest: 100000 positions next to 50 .. 1000 973 us, 103 with 256 sequences); nor up to
  // 512 positions, which take less time than a split costs (partial sums, arrival, join): 4 x 300 6.5 us against 8.2.
  p.step_least = a.max_len <= 512 ? 4 : 2;
  p.alone = (a.max_len <= 512 && p.blocks == 1) || a.nseq > 256 || units >= 8 * places ||
            units * ((a.max_len + PF_STEP - 1) / PF_STEP) >= (1ll << 28);  // (quotients of floats: see over())
  // One round of workgroups where the units leave room in it, two where they do not: 384 units of 500 to 4000 positions
  // take 53 us in one, 61 in two (units + places), 160 units 21.5 and 27.
  p.grid = (int)(p.alone ? units : units <= places * 3 / 4 ? places : units + places);
  return p;
}

hipError_t launch_pages_few(const Pages& a, hipStream_t s) {
  switch (a.D) {
    case 64: return go<64>(a, s);
    case 96: return go<96>(a, s);
    case 128: return go<128>(a, s);
    default: return go<256>(a, s);
  }
}

}  // namespace w4k
