// Routing of tokens to experts: scores, choice, weights, and the pairs sorted by expert (w4_route_experts).
//
// Two launches.  The first has a workgroup for a block of tokens, a wave for a token: it chooses experts and counts
// how often the block chose each.  The second sorts: a block's pairs of expert e begin where all pairs of the
// experts before e end, plus what the blocks before it have of e; inside the block they follow by token, and since a token
// chooses an expert once, a pair's place among 64 tokens is the number of bits below its token's in the set of
// those that chose e.  Nothing in it depends on which workgroup comes first.
#include "dq.cuh"
#include "kernels.h"

namespace w4k {
namespace {

constexpr int RT_THREADS = 256, RT_WAVES = RT_THREADS / 64;
constexpr int RT_MAX_E = 1024;
constexpr int RT_MAX_BLOCKS = 1024;  // of tokens: a sorting block reads all blocks' counts

int route_block(int tokens) {  // tokens of a block, a multiple of 64
  const int units = (tokens + 63) / 64;
  return 64 * ((units + RT_MAX_BLOCKS - 1) / RT_MAX_BLOCKS);
}

// The larger of two choices (c, index): of equals, the lower index.
__device__ __forceinline__ bool ahead(double c, int i, double d, int j) { return c > d || (c == d && i < j); }

__device__ __forceinline__ void wave_best(double& c, int& i) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const double d = __shfl_xor(c, o);
    const int j = __shfl_xor(i, o);
    if (ahead(d, j, c, i)) c = d, i = j;
  }
}

// Lane l has experts l, l + 64 ...; a lane of NE of them.  c of an expert that is not to be chosen is -inf.
template <int NE>
__global__ __launch_bounds__(RT_THREADS) void route_kernel(RouteArgs a, int block, uint16_t* __restrict__ counts) {
  __shared__ int count_lds[RT_MAX_E];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int E = a.r.experts, k = a.r.top_k;
  const int per = E / a.r.groups;
  for (int e = t; e < E; e += RT_THREADS) count_lds[e] = 0;
  __syncthreads();
  const int there = a.count ? min(*a.count, a.tokens) : a.tokens;
  const long long first = (long long)blockIdx.x * block;
  const int end = (int)min((long long)a.tokens, first + block);
  for (int tok = (int)first + wave; tok < end; tok += RT_WAVES) {
    int* const ids = a.experts + (long long)tok * k;
    float* const ws = a.weights + (long long)tok * k;
    if (tok >= there) {
      if (lane < k) ids[lane] = -1, ws[lane] = 0.f;
      continue;
    }
    double c[NE];
    float l[NE], top = -INFINITY;
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      const int e = lane + 64 * i;
      l[i] = -INFINITY;
      if (e < E) {
        const long long at = (long long)tok * a.stride + e;
        const float raw = a.f32 ? ((const float*)a.logits)[at] : (float)((const _Float16*)a.logits)[at];
        l[i] = raw != raw ? -INFINITY : fminf(raw, a.f32 ? 3.4028234663852886e38f : 65504.f);
      }
      top = fmaxf(top, l[i]);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    const bool exact = a.r.bias || a.r.groups > 1;
    float total = 0.f;  // of e^(l - top)
    double total_d = 0.0;
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      const bool has = l[i] > -INFINITY;
      c[i] = l[i];
      if (a.r.score == 0) {
        total += has ? expf(l[i] - top) : 0.f;
        if (exact && has) c[i] = exp((double)l[i] - (double)top), total_d += c[i];
      } else if (exact && has) {
        c[i] = 1.0 / (1.0 + exp(-(double)l[i]));
      }
    }
    if (a.r.score == 0) {
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) total += __shfl_xor(total, o), total_d += __shfl_xor(total_d, o);
    }
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      const int e = lane + 64 * i;
      if (a.r.score == 0 && exact && c[i] > -INFINITY) c[i] /= total_d;
      if (a.r.bias && e < E && c[i] > -INFINITY) c[i] += (double)a.r.bias[e];
      if (!(c[i] > -INFINITY)) c[i] = -INFINITY;
    }
    if (a.r.groups > 1) {
      // every group's value by its best two, group g's held by lane g; then the groups that stay
      double mine = -INFINITY;
      for (int g = 0; g < a.r.groups; ++g) {
        double sum = -INFINITY;
        int skip = -1;
        for (int n = 0; n < a.r.group_best; ++n) {
          double b = -INFINITY;
          int at = E;
#pragma unroll
          for (int i = 0; i < NE; ++i) {
            const int e = lane + 64 * i;
            if (e < E && e / per == g && e != skip && ahead(c[i], e, b, at)) b = c[i], at = e;
          }
          wave_best(b, at);
          if (b > -INFINITY) sum = n == 0 ? b : sum + b;
          skip = at;
        }
        if (lane == g) mine = sum;
      }
      unsigned long long kept = 0;
      for (int n = 0; n < a.r.top_groups; ++n) {
        double b = kept >> lane & 1 ? -INFINITY : mine;
        int at = lane;
        wave_best(b, at);
        if (b > -INFINITY) kept |= 1ull << at;
      }
#pragma unroll
      for (int i = 0; i < NE; ++i) {
        const int e = lane + 64 * i;
        if (e < E && !(kept >> (e / per) & 1)) c[i] = -INFINITY;
      }
    }
    // lane j keeps the j-th choice and its logit
    int id = -1;
    float lj = -INFINITY;
    for (int j = 0; j < k; ++j) {
      double b = -INFINITY;
      int at = E;
#pragma unroll
      for (int i = 0; i < NE; ++i)
        if (ahead(c[i], lane + 64 * i, b, at)) b = c[i], at = lane + 64 * i;
      wave_best(b, at);
      if (!(b > -INFINITY)) break;
      float v = 0.f;
#pragma unroll
      for (int i = 0; i < NE; ++i)
        if (lane + 64 * i == at) v = l[i], c[i] = -INFINITY;
      v = __shfl(v, at & 63);
      if (lane == j) id = at, lj = v;
    }
    // Weights that are divided by their sum are taken relative to the largest chosen score: however far below
    // the row's others the chosen ones lie (a bias may choose them), their ratios are kept.
    float most = lj;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor(most, o));
    float w = 0.f;
    if (a.r.score == 0) {
      if (id >= 0) w = a.r.renorm ? expf(lj - most) : expf(lj - top) / total;
    } else if (id >= 0) {  // e^min(l, 0) / (1 + e^-|l|)
      w = expf(fminf(lj, 0.f) - (a.r.renorm ? fminf(most, 0.f) : 0.f)) / (1.f + expf(-fabsf(lj)));
    }
    if (a.r.renorm) {
      float sum = w;
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
      w = id >= 0 ? w / sum : 0.f;
    }
    if (lane < k) {
      ids[lane] = id;
      ws[lane] = w * a.r.scale;
      if (id >= 0) atomicAdd(&count_lds[id], 1);
    }
  }
  __syncthreads();
  for (int e = t; e < E; e += RT_THREADS) counts[(size_t)blockIdx.x * E + e] = (uint16_t)count_lds[e];
}

constexpr int SORT_THREADS = 1024;

__global__ __launch_bounds__(SORT_THREADS) void route_sort_kernel(RouteArgs a, int block, int blocks,
                                                                  const uint16_t* __restrict__ counts) {
  __shared__ int base[RT_MAX_E];                   // where the block's next pair of an expert goes
  __shared__ unsigned long long chose[RT_MAX_E];   // tokens of 64 that chose it
  __shared__ int wave_sum[SORT_THREADS / 64];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int E = a.r.experts, k = a.r.top_k;
  int before = 0, total = 0;
  if (t < E)
    for (int b = 0; b < blocks; ++b) {
      const int n = counts[(size_t)b * E + t];
      if (b < (int)blockIdx.x) before += n;
      total += n;
    }
  int run = total;  // sums over the experts up to this one
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int v = __shfl_up(run, o);
    if (lane >= o) run += v;
  }
  if (lane == 63) wave_sum[wave] = run;
  __syncthreads();
  int all = 0;
  for (int w = 0; w < SORT_THREADS / 64; ++w) {
    if (w < wave) run += wave_sum[w];
    all += wave_sum[w];
  }
  if (t < E) {
    base[t] = run - total + before;
    if (blockIdx.x == 0) a.offsets[t] = run - total;
  }
  if (blockIdx.x == 0 && t == 0) a.offsets[E] = all;
  const long long P = (long long)a.tokens * k;
  for (long long p = all + (long long)blockIdx.x * SORT_THREADS + t; p < P; p += (long long)blocks * SORT_THREADS)
    a.order[p] = -1;
  const long long first = (long long)blockIdx.x * block;
  for (int u = 0; u < block; u += 64) {
    const int t0 = (int)min(first + u, (long long)a.tokens), n = min(64, a.tokens - t0);
    for (int e = t; e < E; e += SORT_THREADS) chose[e] = 0;
    __syncthreads();
    for (int i = t; i < n * k; i += SORT_THREADS) {
      const int e = a.experts[(long long)t0 * k + i];
      if (e >= 0) atomicOr(&chose[e], 1ull << (i / k));
    }
    __syncthreads();
    for (int i = t; i < n * k; i += SORT_THREADS) {
      const int e = a.experts[(long long)t0 * k + i];
      if (e >= 0) a.order[base[e] + __popcll(chose[e] & ((1ull << (i / k)) - 1))] = t0 * k + i;
    }
    __syncthreads();
    if (t < E) base[t] += __popcll(chose[t]);
  }
}

}  // namespace

size_t route_space(const w4_router& r, int tokens) {
  const int block = tokens ? route_block(tokens) : 64;
  return (((size_t)(tokens + block - 1) / block * r.experts * 2) + 15) / 16 * 16;
}

hipError_t launch_route_experts(const RouteArgs& a, hipStream_t s) {
  const int block = a.tokens ? route_block(a.tokens) : 64, blocks = (a.tokens + block - 1) / block;
  uint16_t* const counts = (uint16_t*)a.space;
  const int E = a.r.experts;
  if (blocks) {
    if (E <= 64) route_kernel<1><<<blocks, RT_THREADS, 0, s>>>(a, block, counts);
    else if (E <= 128) route_kernel<2><<<blocks, RT_THREADS, 0, s>>>(a, block, counts);
    else if (E <= 256) route_kernel<4><<<blocks, RT_THREADS, 0, s>>>(a, block, counts);
    else if (E <= 512) route_kernel<8><<<blocks, RT_THREADS, 0, s>>>(a, block, counts);
    else route_kernel<16><<<blocks, RT_THREADS, 0, s>>>(a, block, counts);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  route_sort_kernel<<<blocks ? blocks : 1, SORT_THREADS, 0, s>>>(a, block, blocks, counts);
  return hipGetLastError();
}

}  // namespace w4k
