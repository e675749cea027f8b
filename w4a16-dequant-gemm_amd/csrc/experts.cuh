// What the kernels of experts' products share: which rows a workgroup multiplies, and the gates' functions.
#pragma once

#include "dq.cuh"
#include "kernels.h"

namespace w4k {

// Some places of one expert, of which a workgroup takes up to TM.
struct ExpertTile {
  int expert, first, rows;  // of the tile; rows 0: there is no such tile
  int column;               // its turn among the tiles of W
};

// Lane l looks after experts e0 + l: where their places begin and end.  Offsets are cut to what `order` has, so that no
// plan leads outside the arrays.
__device__ __forceinline__ void expert_places(const int* __restrict__ offsets, int experts, int pairs, int e0, int& lo, int& hi) {
  const int e = e0 + (int)(threadIdx.x & 63), at = min(e, experts - 1);
  lo = min(max(offsets[at], 0), pairs);
  hi = e < experts ? min(max(offsets[at + 1], lo), pairs) : lo;
}

__device__ __forceinline__ int wave_upto(int v) {  // sum over the lanes up to this one
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(v, o);
    if (lane >= o) v += u;
  }
  return v;
}

// Tile L of the experts' tiles of TM places times `columns` tiles of W, in the experts' order, an expert's places
// fastest: workgroups side by side read the same codes.  L may be any number.  Every wave finds it for itself.
// EVEN: an expert's places are shared out over its tiles in steps of 32.
// SPREAD: consecutive workgroup ids land on different XCDs, each with an L2 of its own: L is turned round so that each
// XCD has a run of the order, whose length is that of the tiles there are, not of the grid.
template <int TM, bool EVEN, bool SPREAD>
__device__ __forceinline__ ExpertTile find_expert_tile(const int* __restrict__ offsets, int experts, int pairs, int columns,
                                                       int L) {
  ExpertTile r{0, 0, 0, 0};
  int lo, hi;
  if constexpr (SPREAD) {
    int all = 0;
    for (int e0 = 0; e0 < experts; e0 += 64) {
      expert_places(offsets, experts, pairs, e0, lo, hi);
      all += (hi - lo + TM - 1) / TM;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) all += __shfl_xor(all, o);
    const int run = (all * columns + 7) >> 3;
    if (L >> 3 >= run) return r;
    L = (L & 7) * run + (L >> 3);
  }
  const int tile = L / columns;  // an expert's tiles times columns begin at a multiple of columns
  int before = 0;
  for (int e0 = 0; e0 < experts; e0 += 64) {
    expert_places(offsets, experts, pairs, e0, lo, hi);
    const int n = (hi - lo + TM - 1) / TM, upto = wave_upto(n);
    const int first = before + upto - n;  // of this lane's expert
    const unsigned long long hit = __ballot(tile >= first && tile < first + n);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      const int count = __shfl(n, l), places = __shfl(hi - lo, l), turn = L - __shfl(first, l) * columns;
      const int per = EVEN ? ((places + count - 1) / count + 31) / 32 * 32 : TM;
      const int m = turn % count * per;
      r.expert = e0 + l;
      r.first = __shfl(lo, l) + m;
      r.rows = min(places - m, per);
      r.column = turn / count;
      break;
    }
    before += __shfl(upto, 63);
  }
  return r;
}

// The most tiles of TM places that `pairs` pairs of `experts` experts can make.
inline long long most_expert_tiles(const ExpertArgs& a, int tm) {
  const long long pairs = (long long)a.tokens * a.top_k;
  return pairs / tm + (pairs < a.experts ? pairs : a.experts);
}

// SiLU; GELU in its tanh form, x / 2 (1 + tanh u) = x / (1 + e^-2u).  In FP32: what exp loses (2^-24 of its argument) is far
// below the half that the result is rounded to.
__device__ __forceinline__ float expert_act(int act, float x) {
  const float u = act == 1 ? x : 1.5957691216057308f * x * (1.f + 0.044715f * x * x);
  return x / (1.f + __expf(-u));
}

// gemm_experts_tile.hip: false (nothing launched) when the arguments are not its.
bool try_experts_tile(const ExpertArgs& a, hipStream_t s, hipError_t* err);
// gemm_experts_step.hip, gemm_experts_few.hip: the same for few rows per expert, of many experts and of few.
bool try_experts_step(const ExpertArgs& a, hipStream_t s, hipError_t* err);
bool try_experts_few(const ExpertArgs& a, hipStream_t s, hipError_t* err);

}  // namespace w4k
