// The weighted sum of a token's rows, a norm behind the block, its gate, the residual stream and the norm ahead of the
// next block (w4_residual_norm), in one pass over the data: a workgroup has a token and keeps its row in FP32 registers
// from the first sum to the last rounding, so each input is read once and each output written once.
#include "dq.cuh"
#include "kernels.h"

namespace w4k {
namespace {

// A piece is eight consecutive elements.  Rows of any length begin at any half, and the card loads 16 bytes from any
// address, so a piece is one load whatever its alignment; the last of a row is cut short.
__device__ __forceinline__ void load_halves(const w4_half* p, int n, float v[8]) {
  if (n == 8) {
    h8 x;
    __builtin_memcpy(&x, p, 16);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)x[e];
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < n ? half_bits_to_float(p[e]) : 0.f;
  }
}
__device__ __forceinline__ void load_floats(const float* p, int n, float v[8]) {
  if (n == 8) {
    __builtin_memcpy(v, p, 32);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < n ? p[e] : 0.f;
  }
}
__device__ __forceinline__ void store_halves(w4_half* p, int n, const float v[8]) {
  if (n == 8) {
    h8 x;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = (_Float16)v[e];
    __builtin_memcpy(p, &x, 16);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) p[e] = __builtin_bit_cast(uint16_t, (_Float16)v[e]);
  }
}
__device__ __forceinline__ void store_floats(float* p, int n, const float v[8]) {
  if (n == 8) {
    __builtin_memcpy(p, v, 32);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) p[e] = v[e];
  }
}

constexpr int RN_MAX_THREADS = 1024;

// Sum over the workgroup, in the same order for every thread.
__device__ __forceinline__ float group_sum(float v, float* lds) {
  const int waves = blockDim.x >> 6;
  v = wave_sum_to_lane63(v);
  if ((threadIdx.x & 63) == 63) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  float sum = 0.f;
  for (int w = 0; w < waves; ++w) sum += lds[w];
  __syncthreads();
  return sum;
}

// PIECES: of a thread, every blockDim-th.
template <int PIECES>
__global__ __launch_bounds__(RN_MAX_THREADS) void residual_norm_kernel(NormArgs a) {
  __shared__ float lds[RN_MAX_THREADS / 64];
  const int D = a.n.dim, t = threadIdx.x, step = blockDim.x;
  const long long tok = blockIdx.x, row = tok * D;
  float b[PIECES][8];
  auto left = [&](int i) { return min(8, D - 8 * (t + i * step)); };
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    const int n = left(i), at = 8 * (t + i * step);
#pragma unroll
    for (int e = 0; e < 8; ++e) b[i][e] = 0.f;
    if (n <= 0) continue;
    for (int j = 0; j < a.terms; ++j) {
      const float w = a.weights ? a.weights[tok * a.terms + j] : 1.f;
      if (w == 0.f) continue;
      float v[8];
      load_halves(a.y + (tok * a.terms + j) * D + at, n, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) b[i][e] += w * v[e];
    }
    if (a.shared) {
      float v[8];
      load_halves(a.shared + row + at, n, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) b[i][e] += v[e];
    }
  }
  // x becomes its norm without the weight
  auto norm = [&]() {
    if (a.n.centred) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < PIECES; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) sum += b[i][e];
      const float mean = group_sum(sum, lds) / (float)D;
#pragma unroll
      for (int i = 0; i < PIECES; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) b[i][e] = e < left(i) ? b[i][e] - mean : 0.f;
    }
    float sq = 0.f;
#pragma unroll
    for (int i = 0; i < PIECES; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) sq += b[i][e] * b[i][e];
    const float f = 1.f / sqrtf(group_sum(sq, lds) / (float)D + a.n.eps);
#pragma unroll
    for (int i = 0; i < PIECES; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) b[i][e] *= f;
  };
  auto scaled = [&](int i, const w4_half* weight, const w4_half* bias) {
    const int n = left(i), at = 8 * (t + i * step);
    float v[8];
    load_halves(weight + at, n, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) b[i][e] *= v[e];
    if (!bias) return;
    load_halves(bias + at, n, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) b[i][e] += v[e];
  };
  if (a.n.post) norm();
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    const int n = left(i), at = 8 * (t + i * step);
    if (n <= 0) continue;
    if (a.n.post) scaled(i, a.n.post, a.n.post_bias);
    float v[8];
    if (a.n.gate) {
      load_halves(a.n.gate + tok * a.n.gate_stride + at, n, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) b[i][e] *= v[e];
    }
    if (a.f32) load_floats((const float*)a.residual + row + at, n, v);
    else load_halves((const w4_half*)a.residual + row + at, n, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) b[i][e] = v[e] + a.n.residual_scale * b[i][e];
    if (a.f32) store_floats((float*)a.residual_out + row + at, n, b[i]);
    else store_halves((w4_half*)a.residual_out + row + at, n, b[i]);
  }
  if (!a.h) return;
  norm();
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    const int n = left(i);
    if (n <= 0) continue;
    scaled(i, a.n.pre, a.n.pre_bias);
    store_halves(a.h + row + 8 * (t + i * step), n, b[i]);
  }
}

}  // namespace

hipError_t launch_residual_norm(const NormArgs& a, hipStream_t s) {
  const int pieces = (a.n.dim + 7) / 8, threads = pieces >= RN_MAX_THREADS ? RN_MAX_THREADS : (pieces + 63) / 64 * 64;
  if (pieces <= RN_MAX_THREADS) residual_norm_kernel<1><<<a.tokens, threads, 0, s>>>(a);
  else if (pieces <= 2 * RN_MAX_THREADS) residual_norm_kernel<2><<<a.tokens, threads, 0, s>>>(a);
  else residual_norm_kernel<4><<<a.tokens, threads, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace w4k
