// New tokens into a paged FP8 cache: FP16 rows to E4M3 under one FP16 scale per (page, head, side).
//
// A unit of L threads owns one run -- the new tokens of one page, which stand side by side in the slot list --
// of one head and side, so nothing is shared between units: it finds the run's length, the largest magnitude of
// its rows (kept in registers: one pass over the data), the page's scale, and writes the codes.
//   scale: the smallest half >= amax / 448, so nothing saturates; an older page's scale is only ever raised, by
//   a power of two, which leaves the codes of its older rows what they were in value but for subnormals --
//   raised to the new maximum itself, a page of n tokens would round its first rows up to n times.
//   code: RNE(x / s).  Quotients of two halves are exact ties or 2^-17 away from one, so a quotient that is right
//   to the last bit of an FP32 is enough; x * (1 / s) with one residual step is.
// Bound: HBM for prompts (3 bytes per element), behind the chain of slots, rows, scale and codes: 4096 tokens of 8 heads, D = 128,
// on pages of 16 take 8.6 us, 2.9 TB/s (at the rate of a large copy: 4.9 us).  Latency for a decode step: 64 tokens 4.5 us.
#include "pages.cuh"

namespace w4k {
namespace {

constexpr int QP_KEEP = 8;  // pieces of 8 elements that a lane keeps between the two steps

struct QuantPages {
  const w4_half *k, *v;
  uint8_t *q_k, *q_v;
  w4_half *s_k, *s_v;
  const int* slots;
  int* status;
  long long row_stride;
  int H, D, page, npages, tokens;
  int chunk;  // tokens whose runs a unit looks for
  uint32_t units;
  Divider by_page, by_row;  // pages of slots, rows of pieces
};

__device__ __forceinline__ float half_up(float amax) {
  const float want = amax / 448.0f;
  const uint16_t h = __builtin_bit_cast(uint16_t, (_Float16)want);
  const float f = half_bits_to_float(h);
  return f * 448.0f < amax ? half_bits_to_float(h + 1) : f;  // (11 bits times 3: exact)
}

// Largest magnitude of halves as bits (what is not finite is 0x7C00 and more), two at a time.
typedef uint16_t s2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t max_bits(const u4& x, uint32_t m) {
  s2 t = __builtin_bit_cast(s2, m);
#pragma unroll
  for (int i = 0; i < 4; ++i) t = __builtin_elementwise_max(t, __builtin_bit_cast(s2, x[i] & 0x7FFF7FFFu));
  return __builtin_bit_cast(uint32_t, t);
}
// ... leaving out what is not finite
__device__ __forceinline__ uint32_t max_finite_bits(const u4& x, uint32_t m) {
  u4 y;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    y[i] = x[i];
    if ((x[i] & 0x7FFFu) >= 0x7C00u) y[i] &= 0xFFFF0000u;
    if ((x[i] & 0x7FFF0000u) >= 0x7C000000u) y[i] &= 0xFFFFu;
  }
  return max_bits(y, m);
}

// Four codes of x / s, r = 1 / s; 0 where r is 0.  (No quotient of a finite x is over 448.)
template <bool ODD>
__device__ __forceinline__ uint32_t encode4(const float* x, float s, float r) {
  float q[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = x[i] * r;
    q[i] = __builtin_fmaf(-__builtin_fmaf(a, s, -x[i]), r, a);  // (signs so that -0 stays what it is)
    if (ODD && !(fabsf(x[i]) <= 65504.0f)) q[i] = x[i] != x[i] || r == 0.0f ? 0.0f : x[i] > 0.0f ? 448.0f : -448.0f;
  }
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], w, true);
}

// Four codes times a power of two below 1; NaN codes keep their byte.
__device__ __forceinline__ uint32_t recode4(uint32_t w, float f) {
  float x[4];
  uint32_t nan = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t b = (w >> (8 * i)) & 0xFFu;
    // bits 6..0 as exponent and significand are 2^-120 times the E4M3 value, subnormals included
    const float mag = __builtin_bit_cast(float, (b & 0x7Fu) << 20) * 0x1p120f * f;
    x[i] = b & 0x80u ? -mag : mag;
    if ((b & 0x7Fu) == 0x7Fu) nan |= 0xFFu << (8 * i);
  }
  int p = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
  return ((uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], p, true) & ~nan) | (w & nan);
}

// VEC: elements of a piece (8: 16-byte loads; 4: rows of any alignment).  L: threads of a unit.
template <int VEC, int L>
__global__ __launch_bounds__(256) void quantize_pages_kernel(const QuantPages a) {
  constexpr int W = L < 64 ? L : 64;  // tokens whose slots are looked at together
  __shared__ uint32_t tops[4];
  const uint32_t unit = (blockIdx.x * 256u + threadIdx.x) / L;
  if (unit >= a.units) return;  // (a unit's threads leave together)
  const int lane = threadIdx.x & (L - 1), wl = threadIdx.x & (W - 1);
  const uint32_t sides = 2u * a.H;
  const int c0 = (int)(unit / sides) * a.chunk;
  const uint32_t hs = unit % sides;
  const int h = (int)(hs >> 1);
  const bool vside = hs & 1;
  const w4_half* const src = (vside ? a.v : a.k) + (long long)h * a.D;
  uint8_t* const pool = (vside ? a.q_v : a.q_k) + (long long)h * a.npages * a.page * a.D;
  w4_half* const scales = (vside ? a.s_v : a.s_k) + (long long)h * a.npages;
  const int rows = a.npages * a.page;
  const int per_row = a.D / VEC;

  // ---- the slots from the one before the unit's first token on: which tokens begin a run, which go on with one
  const int mine = c0 - 1 + wl;
  const int at_mine = mine >= 0 && mine < a.tokens ? a.slots[mine] : -1;
  const int at_prev = __shfl_up(at_mine, 1, W);
  const bool valid = at_mine >= 0 && at_mine < rows;
  const bool on = valid && at_prev >= 0 && at_prev + 1 == at_mine && at_mine - a.by_page(at_mine) * a.page != 0;
  auto bits = [&](bool x) -> unsigned long long {
    const unsigned long long all = __builtin_amdgcn_ballot_w64(x);
    return W == 64 ? all : (all >> ((threadIdx.x & 63) & ~(W - 1))) & ((1ull << (W & 63)) - 1);
  };
  const unsigned long long goes_on = bits(on && wl > 0);
  unsigned long long begins = bits(valid && !on && wl > 0 && wl <= a.chunk);
  for (; begins; begins &= begins - 1) {
    const int first = __builtin_ctzll(begins), t = c0 - 1 + first;
    const int slot = __shfl(at_mine, first, W);
    const int pg = a.by_page(slot), r0 = slot - pg * a.page;
    int n = 1 + (first + 1 < 64 ? __builtin_ctzll(~(goes_on >> (first + 1))) : 0);
    if (first + n == W) {  // (perhaps past what has been looked at)
      const int room = min(a.page - r0, a.tokens - t);
      while (n < room) {
        const int j = n + wl;
        const unsigned long long more = bits(j < room && a.slots[t + min(j, room - 1)] == slot + j);
        const int got = W == 64 && more == ~0ull ? 64 : __builtin_ctzll(~more);
        n += got;
        if (got < W) break;
      }
    }
    const float old = r0 ? half_bits_to_float(scales[pg]) : 0.0f;
    // ---- the largest magnitude
    const int pieces = n * per_row;
    u4 keep[QP_KEEP];
    auto load = [&](int e) -> u4 {
      const int r = a.by_row(e), d = (e - r * per_row) * VEC;
      const w4_half* const p = src + (long long)(t + r) * a.row_stride + d;
      if constexpr (VEC == 8) {
        return *(const u4*)p;
      } else {
        return u4{p[0] | (uint32_t)p[1] << 16, p[2] | (uint32_t)p[3] << 16, 0u, 0u};
      }
    };
#pragma unroll
    for (int i = 0; i < QP_KEEP; ++i) {
      const int e = lane + i * L;
      keep[i] = e < pieces ? load(e) : u4{0u, 0u, 0u, 0u};
    }
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < QP_KEEP; ++i) top = max_bits(keep[i], top);
    for (int e = lane + QP_KEEP * L; e < pieces; e += L) top = max_bits(load(e), top);
    const bool odd = (top & 0xFFFFu) >= 0x7C00u || top >= 0x7C000000u;  // the thread has something that is not finite
    if (odd) {
      top = 0;
#pragma unroll
      for (int i = 0; i < QP_KEEP; ++i) top = max_finite_bits(keep[i], top);
      for (int e = lane + QP_KEEP * L; e < pieces; e += L) top = max_finite_bits(load(e), top);
      atomicOr(a.status, 1);
    }
    top = max(top & 0xFFFFu, top >> 16);
#pragma unroll
    for (int d = W / 2; d > 0; d >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d, 64));
    if constexpr (L > 64) {
      if (wl == 0) tops[threadIdx.x >> 6] = top;
      __syncthreads();
      top = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
      __syncthreads();
    }
    // ---- the page's scale
    float s = half_up(half_bits_to_float(top)), lowered = 1.0f;
    if (old > 0.0f) {
      float now = old;
      while (now < s) now *= 2.0f, lowered *= 0.5f;
      s = now;
    }
    uint8_t* const at = pool + (long long)pg * a.page * a.D;
    if (lowered < 1.0f) {  // older rows under the raised scale
      const int words = r0 * (a.D / 4);
      for (int e = lane; e < words; e += L) ((uint32_t*)at)[e] = recode4(((const uint32_t*)at)[e], lowered);
    }
    // ---- the codes
    const float r = s > 0.0f ? 1.0f / s : 0.0f;
    auto store = [&](int e, const u4& x) {
      uint32_t w[2];
#pragma unroll
      for (int p = 0; p < VEC / 4; ++p) {
        float f[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = half_bits_to_float((x[2 * p + (i >> 1)] >> (16 * (i & 1))) & 0xFFFFu);
        w[p] = odd ? encode4<true>(f, s, r) : encode4<false>(f, s, r);
      }
      uint8_t* const dst = at + (long long)r0 * a.D + (long long)e * VEC;
      if constexpr (VEC == 8) *(u2*)dst = u2{w[0], w[1]};
      else *(uint32_t*)dst = w[0];
    };
#pragma unroll
    for (int i = 0; i < QP_KEEP; ++i)
      if (lane + i * L < pieces) store(lane + i * L, keep[i]);
    for (int e = lane + QP_KEEP * L; e < pieces; e += L) store(e, load(e));
    if (lane == 0) scales[pg] = __builtin_bit_cast(uint16_t, (_Float16)s);
  }
}

}  // namespace

hipError_t launch_quantize_f8_pages(const w4_f8_pages_view& p, const w4_half* k, const w4_half* v, long long row_stride,
                                    const int* slots, int tokens, int* status, hipStream_t s) {
  QuantPages a{k, v, (uint8_t*)p.q_k, (uint8_t*)p.q_v, (w4_half*)p.s_k, (w4_half*)p.s_v, slots, status, row_stride,
               p.H, p.D, p.page, p.npages, tokens, 1, 0, {}, {}};
  const bool wide = p.D % 8 == 0 && row_stride % 8 == 0 && (((uintptr_t)k | (uintptr_t)v) & 15) == 0 &&
                    (((uintptr_t)p.q_k | (uintptr_t)p.q_v) & 7) == 0;
  // Threads for the rows of a page, so that they are read once (4096 tokens, pages of 16, D = 128: 8.6 us with 64 threads, 14.5
  // with 256, 57 with 16; 64 tokens: 4.5, 6.0, 4.6); and so many tokens to a unit that most units begin a run where
  // there are more units than the card has places (up to 1024 tokens of 8 heads: one each): 16 tokens to 64 threads take
  // 8.6 us there, 8 tokens 12.5, 24 tokens 8.9.
  const long long pieces = (long long)p.page * p.D / (wide ? 8 : 4);
  const int L = pieces <= 32 ? 16 : pieces <= QP_KEEP * 64 ? 64 : 256;
  a.chunk = (long long)tokens * 2 * p.H * L <= (1 << 20) || (p.page == 1 && tokens < (1 << 23) / p.H) ? 1 : L == 16 ? 4 : L == 64 ? 16 : 48;
  const long long units = ((long long)tokens + a.chunk - 1) / a.chunk * 2 * p.H;
  a.units = (uint32_t)units;
  a.by_page = divider(p.page), a.by_row = divider(p.D / (wide ? 8 : 4));
  const unsigned grid = (unsigned)((units * L + 255) / 256);
#define GO(L)                                                               \
  do {                                                                      \
    if (wide) quantize_pages_kernel<8, L><<<grid, 256, 0, s>>>(a);          \
    else quantize_pages_kernel<4, L><<<grid, 256, 0, s>>>(a);               \
  } while (0)
  if (L == 16) GO(16);
  else if (L == 64) GO(64);
  else GO(256);
#undef GO
  return hipGetLastError();
}

}  // namespace w4k
