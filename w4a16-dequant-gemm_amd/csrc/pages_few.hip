// Paged FP8 attention for few rows: one token per sequence, or a handful, for the query heads of one KV head.
//
// A workgroup takes one (sequence, KV head) and a split of its positions; its four waves take tiles of 32
// positions in turn, each with a softmax of its own, and meet once at the end.  With up to 16 NT rows as columns:
//   scores  S[t][row] = sum_d K[t][d] q[row][d]   v_mfma_f32_16x16x32_f16, A = K rows, B = queries; the codes are converted
//           by the hardware (two per instruction, exact) and the page's scale enters the scores, not the elements
//   output  O^T[d][row] += sum_t V[t][d] w[t][row]  A = V transposed: ds_read_b64_tr_b8 takes 8 positions x 16 d out
//           of LDS with a lane's 8 positions of one d side by side; B = the weights straight from the score registers
//           (lane (row, r): positions 4r .. 4r+3 and 16+4r .. 16+4r+3 of the tile, which the reads of V follow)
// K and V tiles reach LDS as whole rows by direct loads (16 bytes a lane, two slots per wave), with pieces swapped
// by row so that neither read has bank conflicts.  Page ids and scales of the split lie in a table in LDS.
// Bound: HBM, 2 D bytes per position and KV head.
#include <type_traits>

#include "pages.cuh"

namespace w4k {
namespace {

constexpr int PF_TILE = 32, PF_WAVES = 4, PF_RING = 2;
constexpr int PF_STEP = PF_TILE * PF_WAVES;  // positions that a workgroup's waves take together
constexpr int PF_TABLE = 512;                // pages of a split
typedef __attribute__((address_space(3))) void* lds_ptr;
typedef int i2 __attribute__((ext_vector_type(2)));

struct Entry {
  int row0;        // first row of the page in its head's pool; -1: no page of the pool
  float skc, sv;   // scale of K times c, scale of V
  float lsv;       // log2 of the latter
};

__device__ __forceinline__ h8 codes_to_half(uint32_t lo, uint32_t hi) {
  const h2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true);
  const h2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
  return h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// PG4: pages of a multiple of 4 rows (four neighbouring positions have one page).
template <int D, int NT, bool PG4>
__global__ __launch_bounds__(PF_WAVES * 64) void pages_few_kernel(const Pages a) {
  constexpr int P = D / 16, NC = D / 32, NE = D / 16;  // 16-byte pieces of a row, MFMAs of a score, of an output
  constexpr bool WIDE = P % 4 == 0;                    // K operands by 16-byte reads
  constexpr int SIDE = PF_TILE * D, SLOT = 2 * SIDE, KI = SIDE / 1024;
  constexpr int LDW = D + 4;  // floats of a merge row: O[D], denominator, M
  static_assert(16 * LDW * 4 <= PF_RING * SLOT, "the merge rows take the ring's place");
  __shared__ __attribute__((aligned(16))) uint8_t ring[PF_WAVES][PF_RING * SLOT];
  __shared__ Entry table[PF_TABLE];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c16 = lane & 15, q4 = lane >> 4;
  const int s = blockIdx.x / a.H, h = blockIdx.x - s * a.H, split = blockIdx.y;
  const Seq q = sequence(a, s);
  const int rows = q.n * a.group, heads = a.H * a.group;
  if (q.n <= 0 || rows > a.few_rows) return;
  const int ns = max(1, splits(a.few, q.len));
  if (split >= ns) return;
  const int s0 = split * a.few.split_len, s1 = min(q.len, s0 + a.few.split_len);
  const float c = 1.44269504088896340736f / sqrtf((float)D);

  // ---- the split's pages
  const int j0 = page_of(a, s0), pages = s1 > s0 ? page_of(a, s1 - 1) - j0 + 1 : 0;
  for (int i = tid; i < pages; i += PF_WAVES * 64) {
    const int id = a.bt[(long long)s * a.stride + j0 + i];
    Entry e{-1, 0.0f, 0.0f, 0.0f};
    if (id >= 0 && id < a.npages) {
      e.row0 = id * a.page;
      e.skc = half_bits_to_float(a.s_k[(long long)h * a.npages + id]) * c;
      e.sv = half_bits_to_float(a.s_v[(long long)h * a.npages + id]);
      e.lsv = fmaxf(__log2f(e.sv), PG_LOG2_FLOOR);
    }
    table[i] = e;
  }
  // ---- queries: lane (row c16, q4) of MFMA m holds 8 elements from kcol(m)
  auto kcol = [&](int m) { return WIDE ? 16 * (4 * (m >> 1) + q4) + 8 * (m & 1) : 8 * (4 * m + q4); };
  h8 qop[NT][NC];
  int sees[NT];  // positions that the lane's row sees
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int row = min(16 * t + c16, rows - 1), tok = row / a.group, head = row - tok * a.group;
    const w4_half* const qp = a.q + (long long)(q.q0 + tok) * a.q_stride + (long long)(h * a.group + head) * D;
#pragma unroll
    for (int m = 0; m < NC; ++m) __builtin_memcpy(&qop[t][m], qp + kcol(m), 16);
    sees[t] = a.causal ? q.shown + tok : q.len;
  }
  __syncthreads();

  const uint8_t* const kbase = a.q_k + (long long)h * a.npages * a.page * D;
  const uint8_t* const vbase = a.q_v + (long long)h * a.npages * a.page * D;
  const uint32_t lds_wave = (uint32_t)(uintptr_t)(lds_ptr)ring + (uint32_t)wave * (PF_RING * SLOT);
  // Pieces swapped by row: 16 rows x one piece of K, and the 8 rows x one piece of V that a group of 16
  // lanes reads, fall on different banks.
  auto kswz = [](int r) { return P == 16 ? r & 15 : P == 8 ? (r >> 1) & 7 : P == 4 ? (r >> 2) & 3 : 0; };
  auto vswz = [](int r) {
    const int hi = (r >> 4) & 1;
    return P == 16 ? (r & 7) | hi << 3 : P == 8 ? ((r >> 1) & 3) | hi << 2 : P == 4 ? ((r >> 2) & 1) | hi << 1 : 0;
  };
  auto dma16 = [](const uint8_t* from, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off nt" : : "v"(from), "s"(lds) : "memory", "m0");
  };
  // Table entry of a position of the split.
  auto entry = [&](int t) { return page_of(a, t) - j0; };

  // Requests the tile at t0 into slot sl; returns which of its rows are there.
  auto request = [&](int sl, int t0) -> uint32_t {
    const int t = t0 + (lane & 31);
    bool there = t < s1;
    const int j = there ? page_of(a, t) : j0;
    const int row0 = table[j - j0].row0;
    there = there && row0 >= 0;
    const int row = there ? row0 + (t - j * a.page) : 0;  // (others read row 0 and drop it)
    const uint32_t at = lds_wave + sl * SLOT;
#pragma unroll
    for (int i = 0; i < KI; ++i) {
      const int u = i * 64 + lane, r = u / P, piece = u % P;
      const long long off = (long long)__shfl(row, r, 64) * D;
      dma16(kbase + off + 16 * (piece ^ kswz(r)), at + i * 1024);
      dma16(vbase + off + 16 * (piece ^ vswz(r)), at + SIDE + i * 1024);
    }
    return (uint32_t)__builtin_amdgcn_ballot_w64(there);
  };

  f4 o[NT][NE];
  float M[NT], l[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    M[t] = -INFINITY, l[t] = 0.0f;
#pragma unroll
    for (int e = 0; e < NE; ++e) o[t][e] = f4{0.f, 0.f, 0.f, 0.f};
  }

  const int vrow = (c16 >> 1) < 4 ? 4 * q4 + (c16 >> 1) : 16 + 4 * q4 + (c16 >> 1) - 4;

  // WHOLE: every position of the tile is there and every row sees it.
  auto compute = [&](int sl, int t0, uint32_t there, auto whole) {
    constexpr bool WHOLE = decltype(whole)::value;
    const uint8_t* const slot = ring[wave] + sl * SLOT;
    f4 sc[NT][2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int r = 16 * j + c16;
      const uint8_t* const kr = slot + r * D;
#pragma unroll
      for (int t = 0; t < NT; ++t) sc[t][j] = f4{0.f, 0.f, 0.f, 0.f};
      if constexpr (WIDE) {
#pragma unroll
        for (int i = 0; i < P / 4; ++i) {
          const u4 w = *(const u4*)(kr + 16 * ((4 * i + q4) ^ kswz(r)));
          const h8 k0 = codes_to_half(w[0], w[1]), k1 = codes_to_half(w[2], w[3]);
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            sc[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qop[t][2 * i], sc[t][j], 0, 0, 0);
            sc[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, qop[t][2 * i + 1], sc[t][j], 0, 0, 0);
          }
        }
      } else {
#pragma unroll
        for (int m = 0; m < NC; ++m) {
          const u2 w = *(const u2*)(kr + 8 * (4 * m + q4));
          const h8 k0 = codes_to_half(w[0], w[1]);
#pragma unroll
          for (int t = 0; t < NT; ++t) sc[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qop[t][m], sc[t][j], 0, 0, 0);
        }
      }
    }
    // the scales of the lane's eight positions
    float skc[8], sv[8], lsv[8];
#pragma unroll
    for (int k = 0; k < 8; k += PG4 ? 4 : 1) {
      const int t = t0 + 16 * (k >> 2) + 4 * q4 + (k & 3);
      const Entry e = table[WHOLE || t < s1 ? entry(t) : 0];
#pragma unroll
      for (int i = 0; i < (PG4 ? 4 : 1); ++i) skc[k + i] = e.skc, sv[k + i] = e.sv, lsv[k + i] = e.lsv;
    }
    h8 pop[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float top = -INFINITY;
      bool see[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int at = 16 * (k >> 2) + 4 * q4 + (k & 3);
        see[k] = WHOLE || (((there >> at) & 1) && t0 + at < sees[t]);
      }
      if constexpr (PG4 && WHOLE) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const f4 x = sc[t][j];
          const float m4 = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
          top = fmaxf(top, __builtin_fmaf(m4, skc[4 * j], lsv[4 * j]));
        }
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float y = __builtin_fmaf(sc[t][k >> 2][k & 3], skc[k], lsv[k]);
          top = fmaxf(top, see[k] ? y : -INFINITY);
        }
      }
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      const float m_new = fmaxf(M[t], top);
      const float use = m_new == -INFINITY ? 0.0f : m_new;
      if (__builtin_amdgcn_ballot_w64(m_new > M[t]) != 0) {  // wave-uniform
        const float alpha = __builtin_amdgcn_exp2f(M[t] - use);
#pragma unroll
        for (int e = 0; e < NE; ++e) o[t][e] *= alpha;
        l[t] *= alpha;
      }
      M[t] = m_new;
      float w[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        float p = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][k >> 2][k & 3], skc[k], -use));
        w[k] = p * sv[k];
        if (!WHOLE && !see[k]) p = w[k] = 0.0f;
        l[t] += p;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) pop[t][k] = (_Float16)w[k];
    }
    // rows that are not there are anything, and 0 times that may be NaN
    uint32_t mask[2] = {~0u, ~0u};
    if constexpr (!WHOLE) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint32_t b = there >> (16 * j + 4 * q4);
        mask[j] = (b & 1 ? 0xFFu : 0u) | (b & 2 ? 0xFF00u : 0u) | (b & 4 ? 0xFF0000u : 0u) | (b & 8 ? 0xFF000000u : 0u);
      }
    }
    const uint8_t* const vr = slot + SIDE + vrow * D + 8 * (c16 & 1);
#pragma unroll
    for (int e = 0; e < NE; ++e) {
      const i2 w = __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) i2*)(vr + 16 * (e ^ vswz(vrow))));
      const h8 v = codes_to_half((uint32_t)w[0] & mask[0], (uint32_t)w[1] & mask[1]);
#pragma unroll
      for (int t = 0; t < NT; ++t) o[t][e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pop[t], o[t][e], 0, 0, 0);
    }
  };

  // ---- tiles of this wave: s0 + 32 (wave + 4 it)
  const int nit = (s1 - s0 + PF_STEP - 1) / PF_STEP;
  auto tile_start = [&](int it) { return s0 + PF_TILE * (wave + PF_WAVES * it); };
  uint32_t there[PF_RING];
#pragma unroll
  for (int d = 0; d < PF_RING; ++d)
    if (d < nit) there[d] = request(d, tile_start(d));
  for (int it0 = 0; it0 < nit; it0 += PF_RING) {
#pragma unroll
    for (int d = 0; d < PF_RING; ++d) {
      const int it = it0 + d;
      if (it < nit) {
        // tile `it` has landed; the ones after it may be in flight
        if (it + PF_RING <= nit) asm volatile("s_waitcnt vmcnt(%0)" : : "n"((PF_RING - 1) * 2 * KI) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
        if (there[d] == ~0u && tile_start(it) + PF_TILE <= q.shown) compute(d, tile_start(it), there[d], std::true_type{});
        else if (there[d]) compute(d, tile_start(it), there[d], std::false_type{});
        asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");  // the slot has been read: refill it
        if (it + PF_RING < nit) there[d] = request(d, tile_start(it + PF_RING));
      }
    }
  }

  // ---- the four waves' sums in wave order
  float* const mine = (float*)ring[wave] + c16 * LDW;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    float den = l[t];
    den += __shfl_xor(den, 16, 64);
    den += __shfl_xor(den, 32, 64);
#pragma unroll
    for (int e = 0; e < NE; ++e) *(f4*)(mine + 16 * e + 4 * q4) = o[t][e];
    if (q4 == 0) mine[D] = den, mine[D + 1] = M[t];
    __syncthreads();
    const int here = min(16, rows - 16 * t);
    for (int i = tid; i < here * (D / 2); i += PF_WAVES * 64) {
      const int r = i / (D / 2), d = 2 * (i - r * (D / 2));
      float top = -INFINITY, sum0 = 0.0f, sum1 = 0.0f, den4 = 0.0f;
#pragma unroll
      for (int w = 0; w < PF_WAVES; ++w) top = fmaxf(top, ((const float*)ring[w])[r * LDW + D + 1]);
      const float use = top == -INFINITY ? 0.0f : top;
#pragma unroll
      for (int w = 0; w < PF_WAVES; ++w) {
        const float* const p = (const float*)ring[w] + r * LDW;
        const float e = __builtin_amdgcn_exp2f(p[D + 1] - use);
        sum0 += e * p[d], sum1 += e * p[d + 1], den4 += e * p[D];
      }
      const int row = 16 * t + r, tok = row / a.group, head = row - tok * a.group;
      const long long at = (long long)(q.q0 + tok) * heads + h * a.group + head;
      if (ns == 1) {
        const float inv = den4 == 0.0f ? 0.0f : 1.0f / den4;
        const h2 v = h2{(_Float16)(sum0 * inv), (_Float16)(sum1 * inv)};
        w4_half* const dst = a.out + at * D + d;
        dst[0] = (uint16_t)as_u32(v), dst[1] = (uint16_t)(as_u32(v) >> 16);
      } else {
        float* const dst = part_of(a, at, split);
        dst[2 + d] = sum0, dst[3 + d] = sum1;
        if (d == 0) dst[0] = top, dst[1] = den4;
      }
    }
    if (t + 1 < NT) __syncthreads();
  }
}

template <int D>
hipError_t go(const Pages& a, hipStream_t s) {
  const dim3 grid((unsigned)a.nseq * a.H, (unsigned)a.few.nsplit);
  const bool pg4 = a.page % 4 == 0;
#define GO(NT)                                                          \
  do {                                                                  \
    if (pg4) pages_few_kernel<D, NT, true><<<grid, 256, 0, s>>>(a);     \
    else pages_few_kernel<D, NT, false><<<grid, 256, 0, s>>>(a);        \
  } while (0)
  if (a.few_rows <= 16) GO(1);
  else if (a.few_rows <= 32) GO(2);
  else if constexpr (D <= 128) GO(4);
#undef GO
  return hipGetLastError();
}

}  // namespace

int pages_few_most(const PagesArgs& a) {
  if (a.D != 64 && a.D != 96 && a.D != 128 && a.D != 256) return 0;
  if (((uintptr_t)a.q_k | (uintptr_t)a.q_v) & 15) return 0;
  return a.D == 256 ? 32 : 64;  // (registers: the sums of 64 rows x 256 elements take all of them)
}

PagesPlan pages_few_plan(const PagesArgs& a, int rows) {
  (void)rows;
  const long long units = (long long)a.nseq * a.H;
  long long n = (1024 + units - 1) / units;
  const long long most = a.max_len <= 512 ? 1 : (a.max_len + 255) / 256;
  n = n < 1 ? 1 : n > most ? most : n;
  long long len = ((a.max_len + n - 1) / n + PF_STEP - 1) / PF_STEP * PF_STEP;
  const long long room = (long long)(PF_TABLE - 2) * a.page / PF_STEP * PF_STEP;  // (a split may begin inside a page)
  if (len > room) len = room;
  PagesPlan p;
  p.split_len = (int)len;
  p.nsplit = (int)((a.max_len + len - 1) / len);
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
