// Products of a few rows per expert with the experts' packed matrices: decode steps, whose time is the reading of codes.
//
// A workgroup multiplies up to 16 MT places of one expert with 32 of its rows (gated: 16 of the gate and the 16 of the way
// up for the same columns).  Its four waves share K out in chunks of 128; a wave asks for all codes, scales and rows of x of four
// chunks at once and waits for no other wave before the end, where the four sums are added in the waves' order.
// v_mfma_f32_16x16x32_f16: lane l brings row l % 16 and eight consecutive k; of a chunk it has k 32 (l / 16) .. + 31, so that
// its codes are one 16-byte load and lie in one group of 32 or more, and its part of a row of x is 64 bytes side by side.
#include "experts.cuh"

namespace w4k {
namespace {

constexpr int EF_WAVES = 4;

template <int FMT, bool GATED, int MT>
__global__ __launch_bounds__(64 * EF_WAVES) void experts_few_kernel(ExpertArgs a, int columns) {
  constexpr bool MX = FMT == 2;
  constexpr int U = 4 / MT;  // chunks asked for at once
  __shared__ float sums[EF_WAVES][2][MT][4][64];
  const int pairs = a.tokens * a.top_k;
  const ExpertTile tile = find_expert_tile<16 * MT, false, true>(a.offsets, a.experts, pairs, columns, blockIdx.x);
  const int rows = __builtin_amdgcn_readfirstlane(tile.rows);
  if (rows == 0) return;
  const int expert = __builtin_amdgcn_readfirstlane(tile.expert), first = __builtin_amdgcn_readfirstlane(tile.first);
  const int c0 = __builtin_amdgcn_readfirstlane(tile.column) * (GATED ? 16 : 32);
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int r = lane & 15, q = lane >> 4;
  const int K = a.v.K, G = MX ? a.v.B : a.v.G, gs = a.v.gs;
  const int R = a.v.N / a.experts, width = GATED ? R / 2 : R;
  const int chunks = (K + 127) >> 7, per = (chunks + EF_WAVES - 1) / EF_WAVES;
  const int c_end = min(chunks, (wave + 1) * per);

  // this lane's rows of W (columns past the last repeat it and are not stored)
  const char* const codes = (const char*)a.v.q + (size_t)expert * R * (K >> 1);
  uint32_t wo[2];
  size_t so[2], zo[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int row = GATED ? min(c0 + r, width - 1) + i * width : min(c0 + 16 * i + r, width - 1);
    wo[i] = (uint32_t)row * (uint32_t)(K >> 1);
    so[i] = ((size_t)expert * R + row) * G;
    zo[i] = ((size_t)expert * R + row) * words(G);
  }
  const w4_half* xr[MT];
  bool there[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int place = first + min(16 * m + r, rows - 1);
    int from = place;
    if (a.from_tokens) {
      const int pair = a.order[place];
      from = pair >= 0 && pair < pairs ? (uint32_t)pair / (uint32_t)a.top_k : 0;
    }
    there[m] = 16 * m + r < rows;
    xr[m] = a.x + (size_t)from * K + 32 * q;
  }
  uint32_t mask = 0x00F0000Fu, magic = 0x54006400u;
  asm volatile("" : "+s"(mask));   // opaque: otherwise they come back as literals of two
  asm volatile("" : "+v"(magic));  // separate instructions

  f4 acc[2][MT];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[i][m] = f4{0.f, 0.f, 0.f, 0.f};

  for (int cb = wave * per; cb < c_end; cb += U) {
    u4 w[U][2], xv[U][MT][4];
    uint32_t sc[U][2], z[U][2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      // (a slice of 32 k behind the end of K, or a chunk behind the wave's last: fetched from the row's start, times 0)
      const int k = (cb + u) * 128 + 32 * q;
      const bool inside = cb + u < c_end && k < K;
      const int kk = inside ? k : 0;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        w[u][i] = *(const u4*)(codes + (wo[i] + (kk >> 1)));
        if constexpr (MX) {
          sc[u][i] = ((const uint8_t*)a.v.scales)[so[i] + (kk >> 5)];
        } else {
          const int g = kk / gs;
          sc[u][i] = ((const uint16_t*)a.v.scales)[so[i] + g];
          z[u][i] = FMT == 1 ? a.v.zeros[zo[i] + (g >> 3)] >> (4 * (g & 7)) & 0xFu : 8u;
        }
      }
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          xv[u][m][j] = u4{0u, 0u, 0u, 0u};
          if (there[m] && inside) xv[u][m][j] = *(const u4*)(xr[m] + (cb + u) * 128 + 8 * j);
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          h8 av;
          if constexpr (MX) {
            h2 n[4];
            dq_mx(w[u][i][j], mx_scale(sc[u][i]), n);
            av = __builtin_bit_cast(h8, u4{as_u32(n[0]), as_u32(n[1]), as_u32(n[2]), as_u32(n[3])});
          } else {
            av = expand_word(w[u][i][j], as_h2(0xD400E400u | (z[u][i] << 20) | z[u][i]), splat_bits(sc[u][i]), mask, magic);
          }
#pragma unroll
          for (int m = 0; m < MT; ++m)
            acc[i][m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, __builtin_bit_cast(h8, xv[u][m][j]), acc[i][m], 0, 0, 0);
        }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int e = 0; e < 4; ++e) sums[wave][i][m][e][lane] = acc[i][m][e];
  __syncthreads();
  // lane l of a 16 x 16 tile holds columns 4 (l / 16) + e of place l % 16
  constexpr int COLS = GATED ? 16 : 32;
  for (int o = t; o < COLS * 16 * MT; o += 64 * EF_WAVES) {
    const int col = o % COLS, m = o / COLS;  // column and place of the tile
    if (m >= rows || c0 + col >= width) continue;
    const int e = col & 3, l = (col >> 2 & 3) * 16 + (m & 15), i = GATED ? 0 : col >> 4;
    float y = 0.f, up = 0.f;
#pragma unroll
    for (int w = 0; w < EF_WAVES; ++w) {
      y += sums[w][i][m >> 4][e][l];
      if (GATED) up += sums[w][1][m >> 4][e][l];
    }
    if (GATED) y = expert_act(a.act, y) * up;
    const int pair = a.order[first + m];
    if (pair < 0 || pair >= pairs) continue;
    a.out[(size_t)(a.to_pairs ? pair : first + m) * width + c0 + col] = __builtin_bit_cast(uint16_t, (_Float16)y);
  }
}

template <int FMT, bool GATED, int MT>
hipError_t go(const ExpertArgs& a, hipStream_t s) {
  const int R = a.v.N / a.experts, columns = GATED ? (R / 2 + 15) / 16 : (R + 31) / 32;
  const long long grid = (most_expert_tiles(a, 16 * MT) * columns + 7) / 8 * 8;
  if (grid > 0x7FFFFFFFLL) return hipErrorInvalidConfiguration;
  experts_few_kernel<FMT, GATED, MT><<<dim3((unsigned)grid), dim3(64 * EF_WAVES), 0, s>>>(a, columns);
  return hipGetLastError();
}

template <int FMT>
hipError_t go_rows(const ExpertArgs& a, hipStream_t s) {
  const long long pairs = (long long)a.tokens * a.top_k;
  const bool two = pairs >= 12LL * a.experts;
  if (a.act) return two ? go<FMT, true, 2>(a, s) : go<FMT, true, 1>(a, s);
  return two ? go<FMT, false, 2>(a, s) : go<FMT, false, 1>(a, s);
}

}  // namespace

bool try_experts_few(const ExpertArgs& a, hipStream_t s, hipError_t* err) {
  const WView& v = a.v;
  if (v.K % 32 || (!v.mx && v.gs % 32)) return false;
  if ((long long)(v.N / a.experts) * v.K / 2 >= 1LL << 32) return false;  // offsets of 32 bits into an expert's codes
  if ((((uintptr_t)v.q | (uintptr_t)a.x) & 15) || ((uintptr_t)v.scales & 1) || ((uintptr_t)v.zeros & 3)) return false;
  *err = v.mx ? go_rows<2>(a, s) : v.symmetric ? go_rows<0>(a, s) : go_rows<1>(a, s);
  return true;
}

}  // namespace w4k
