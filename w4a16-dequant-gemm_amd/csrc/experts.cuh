// What the kernels of experts' products share: which rows a workgroup multiplies, and the gates' functions.
#pragma once

#include "dq.cuh"
#include "kernels.h"

namespace w4k {

// One tile of up to TM places of one expert.
struct ExpertTile {
  int expert, first, rows;  // rows 0: there is no such tile
  int tiles;                // of all experts
};

// Tile `tile` of the experts' tiles of TM places, in the experts' order; `tile` may be any number.  Every wave of a
// workgroup finds it for itself: lane l sums the tiles of experts l, l + 64 ... in turns of 64 experts, a scan of a wave
// each.  Offsets are cut to what `order` has, so that no plan leads outside the arrays.
template <int TM>
__device__ __forceinline__ ExpertTile find_expert_tile(const int* __restrict__ offsets, int experts, int pairs, int tile) {
  const int lane = threadIdx.x & 63;
  ExpertTile r{0, 0, 0, 0};
  for (int e0 = 0; e0 < experts; e0 += 64) {
    const int e = min(e0 + lane, experts - 1);
    const int lo = min(max(offsets[e], 0), pairs), hi = min(max(offsets[e + 1], lo), pairs);
    const int n = e0 + lane < experts ? (hi - lo + TM - 1) / TM : 0;
    int upto = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(upto, o);
      if (lane >= o) upto += v;
    }
    const int t = tile - r.tiles - (upto - n);  // the tile's number in this lane's expert
    const unsigned long long hit = __ballot(t >= 0 && t < n);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      r.expert = e0 + l;
      r.first = __shfl(lo + t * TM, l);
      r.rows = __shfl(min(hi - (lo + t * TM), TM), l);
    }
    r.tiles += __shfl(upto, 63);
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

}  // namespace w4k
