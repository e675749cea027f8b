// Products of some rows per expert with the experts' packed matrices, where many experts have a few: decode steps of many
// sequences, whose time is the reading of codes.
//
// A workgroup multiplies up to 16 places of one expert with 128 of its rows, 32 a wave (gated: 16 of the gate and the 16 of
// the way up for the same columns), in stages of 256 k.  Everything goes global -> LDS (no registers) in whole lines: a
// load instruction that takes 16 bytes of each of 64 rows, as the operands need them, holds the memory path four times as
// long.  The rows of x are fetched once for the four waves; a wave's codes, scales and zero-points are its own.  Three stage
// buffers, one barrier a stage.
// v_mfma_f32_16x16x32_f16: lane l brings row l % 16 and eight consecutive k; of a stage it has k 64 (l / 16) .. + 63, two
// 16-byte pieces of codes and eight of x.
#include <atomic>

#include "experts.cuh"

namespace w4k {
namespace {

typedef __attribute__((address_space(3))) void* lds_ptr;

constexpr int ES_WAVES = 4, ES_STAGES = 3;
constexpr int ES_W = 4096;            // a wave's codes of a stage: 32 rows of 128 bytes
constexpr int ES_X = 16 * 512;        // rows of x
constexpr int ES_X_AT = ES_WAVES * ES_W, ES_P_AT = ES_X_AT + ES_X;

// How the groups of W4 lie in a stage (GM): 0 two (gs 128), 1 four, 2 eight (gs 32, and MXFP4's blocks), 3 at most four of any
// size that is a multiple of 32, from 96 on.  What a row needs of a stage: a run of dwords of scales, which begins at any
// half (MXFP4: byte) of its first, and words of zero-points; one dword of 32 rows is half a load instruction.
constexpr int es_scales(int fmt, int gm) { return fmt == 2 ? 3 : gm == 0 ? 2 : gm == 2 ? 5 : 3; }
constexpr int es_zeros(int fmt, int gm) { return fmt != 1 ? 0 : gm == 3 ? 2 : 1; }
constexpr int es_param_loads(int fmt, int gm) { return (es_scales(fmt, gm) + es_zeros(fmt, gm) + 1) / 2; }
constexpr int es_stage(int fmt, int gm) { return ES_P_AT + ES_WAVES * es_param_loads(fmt, gm) * 256; }

extern __shared__ __attribute__((aligned(16))) uint8_t es_lds[];

// Where 16-byte piece p of a row lies.  A load instruction writes lane l's 16 bytes at 16 l: eight rows of codes, two of x;
// which piece a lane fetches is chosen so that the sixteen rows of a read (same p) fall on sixteen distinct bank groups.
__device__ __forceinline__ int es_w_key(int R) { return (R >> 1) & 7; }
__device__ __forceinline__ int es_w_at(int R, int p) { return R * 128 + (p ^ es_w_key(R)) * 16; }
__device__ __forceinline__ int es_x_at(int R, int p) { return R * 512 + (p ^ (R & 15)) * 16; }

// (asm, as in the tile kernels: the compiler must not wait for these before an LDS read; M0 carries the LDS address)
__device__ __forceinline__ void es_dma16(const void* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(off), "s"(base), "s"(lds) : "memory", "m0");
}
__device__ __forceinline__ void es_dma4(const void* at, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" : : "v"(at), "s"(lds) : "memory", "m0");
}

// XI: load instructions of x per wave and stage, for up to 8 XI places.
template <int FMT, bool GATED, int GM, int XI>
__device__ __forceinline__ void experts_step(const ExpertArgs& a, const ExpertTile& tile, uint32_t group_mul) {
  constexpr bool MX = FMT == 2, ASYM = FMT == 1;
  constexpr int PS = es_scales(FMT, GM), PZ = es_zeros(FMT, GM), PI = es_param_loads(FMT, GM);
  constexpr int LOADS = 4 + XI + PI, STAGE = es_stage(FMT, GM);
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int r = lane & 15, q = lane >> 4;
  const int K = a.v.K, G = MX ? a.v.B : a.v.G, wg = words(G), pairs = a.tokens * a.top_k;
  const int R = a.v.N / a.experts, width = GATED ? R / 2 : R;
  const int c0 = tile.column * (GATED ? 64 : 128) + wave * (GATED ? 16 : 32);  // first output column of the wave
  // row of the expert that row n of the wave's 32 is; columns past the last repeat it and are not stored
  auto row_of = [&](int n) {
    return GATED ? min(c0 + (n & 15), width - 1) + (n & 16 ? width : 0) : min(c0 + n, width - 1);
  };
  const int stages = (K + 255) >> 8;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_ptr)es_lds;

  const char* const wb = (const char*)a.v.q + (size_t)tile.expert * R * (K >> 1);
  const char* const xb = (const char*)(a.from_tokens ? a.x : a.x + (size_t)tile.first * K);
  uint32_t wo[4], xo[XI];
  int wp[4], xp[XI];  // pieces that the lane fetches
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int n = 8 * i + (lane >> 3);
    wp[i] = (lane & 7) ^ es_w_key(n);
    wo[i] = (uint32_t)row_of(n) * (uint32_t)(K >> 1) + 16 * wp[i];
  }
#pragma unroll
  for (int i = 0; i < XI; ++i) {
    const int m = 2 * (wave + ES_WAVES * i) + (lane >> 5), place = min(m, tile.rows - 1);
    uint32_t from = place;
    if (a.from_tokens) {
      const int pair = a.order[tile.first + place];
      from = pair >= 0 && pair < pairs ? (uint32_t)pair / (uint32_t)a.top_k : 0;
    }
    xp[i] = (lane & 31) ^ (m & 15);
    xo[i] = from * (uint32_t)(K * 2) + 16 * xp[i];
  }
  // parameters: this lane's dwords of a stage (entry e: dword e / 32 of row e % 32)
  const size_t row0 = (size_t)tile.expert * R;
  const size_t sc_last = ((size_t)a.v.N * G >> (MX ? 2 : 1)) - 1, zw_last = (size_t)a.v.N * wg - 1;
  auto first_group = [&](uint32_t d) { return MX ? 8 * d : GM == 3 ? __umulhi(16 * d, group_mul) : (2u << GM) * d; };
  const size_t pn = row0 + row_of(lane & 31);
  auto request = [&](int d, uint32_t buf) {
    const uint32_t dd = (uint32_t)min(d, stages - 1), st = lds0 + buf;
    const bool tail = dd * 256 + 256 > (uint32_t)K;  // pieces behind the end of a row are fetched from its part that is there
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t off = wo[i];
      if (tail && dd * 256 + 32 * wp[i] >= (uint32_t)K) off -= 16 * wp[i];
      es_dma16(wb + dd * 128, off, st + wave * ES_W + i * 1024);
    }
#pragma unroll
    for (int i = 0; i < XI; ++i) {
      uint32_t off = xo[i];
      if (tail && dd * 256 + 8 * xp[i] >= (uint32_t)K) off -= 16 * xp[i];
      es_dma16(xb + dd * 512, off, st + ES_X_AT + (wave + ES_WAVES * i) * 1024);
    }
    const uint32_t g = first_group(dd);
#pragma unroll
    for (int i = 0; i < PI; ++i) {
      const int e = 2 * i + (lane >> 5);
      const uint32_t* at = (const uint32_t*)a.v.scales + min(((pn * G + g) >> (MX ? 2 : 1)) + min(e, PS - 1), sc_last);
      if (ASYM && e >= PS) at = a.v.zeros + min(pn * wg + (g >> 3) + min(e - PS, PZ - 1), zw_last);
      es_dma4(at, st + ES_P_AT + (wave * PI + i) * 256);
    }
  };

  uint32_t mask = 0x00F0000Fu, magic = 0x54006400u;
  asm volatile("" : "+s"(mask));   // opaque: otherwise they come back as literals of two
  asm volatile("" : "+v"(magic));  // separate instructions
  f4 acc[2] = {f4{0.f, 0.f, 0.f, 0.f}, f4{0.f, 0.f, 0.f, 0.f}};
  uint32_t first[2];  // entry of the row's first scale in the whole array: its place in a dword
#pragma unroll
  for (int i = 0; i < 2; ++i) first[i] = (uint32_t)((row0 + row_of(16 * i + r)) * G);
  const uint8_t* const mine = es_lds + wave * ES_W;
  const uint8_t* const xs = es_lds + ES_X_AT;
  const uint8_t* const ps = es_lds + ES_P_AT + wave * PI * 256;
  uint32_t b0 = 0, b1 = STAGE, b2 = 2 * STAGE;
  request(0, b0);
  request(1, b1);
#pragma unroll 1
  for (int d = 0; d < stages; ++d) {
    // stage d has landed (outstanding: stage d + 1), for every wave behind the barrier, where nobody reads stage d - 1 any more
    __builtin_amdgcn_s_waitcnt(waitcnt_vm(LOADS));
    __syncthreads();
    request(d + 2, b2);
    __builtin_amdgcn_sched_barrier(0);
    const uint32_t g0 = first_group(d);
    u4 w[2][2];
    uint32_t sc[2][2], zw[2][2];  // of the lane's two pieces of a row
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        w[i][p] = *(const u4*)(mine + b0 + es_w_at(16 * i + r, 2 * q + p));
        // group of the piece, counted from the stage's first
        const uint32_t n = MX || GM == 2 ? 2 * q + p : GM == 1 ? q : GM == 0 ? q >> 1 : __umulhi(2 * (8 * d + 2 * q + p), group_mul) - g0;
        if (p && !MX && GM < 2) {
          sc[i][1] = sc[i][0], zw[i][1] = zw[i][0];
          continue;
        }
        const uint32_t at = n + ((first[i] + g0) & (MX ? 3 : 1));
        if constexpr (MX) {
          sc[i][p] = ps[b0 + (at >> 2) * 128 + (16 * i + r) * 4 + (at & 3)];
        } else {
          sc[i][p] = *(const uint16_t*)(ps + b0 + (at >> 1) * 128 + (16 * i + r) * 4 + (at & 1) * 2);
          const uint32_t g = g0 + n;
          zw[i][p] = 8;
          if (ASYM)
            zw[i][p] = *(const uint32_t*)(ps + b0 + (PS + (GM == 3 ? (g >> 3) - (g0 >> 3) : 0)) * 128 + (16 * i + r) * 4) >> (4 * (g & 7)) & 0xFu;
        }
      }
    const bool tail = d * 256 + 256 > K;
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      u4 x = *(const u4*)(xs + b0 + es_x_at(r, 8 * q + s));
      const int p = s >> 2;
      const bool past = d * 256 + 64 * q + 32 * p >= K;
      if (tail && past) x = u4{0u, 0u, 0u, 0u};  // what was fetched there counts as 0, and so do its codes
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        h8 av;
        if constexpr (MX) {
          h2 n[4];
          dq_mx(w[i][p][s & 3], tail && past ? 0.f : mx_scale(sc[i][p]), n);
          av = __builtin_bit_cast(h8, u4{as_u32(n[0]), as_u32(n[1]), as_u32(n[2]), as_u32(n[3])});
        } else {
          av = expand_word(w[i][p][s & 3], as_h2(0xD400E400u + zw[i][p] * 0x00100001u), splat_bits(tail && past ? 0u : sc[i][p]), mask, magic);
        }
        acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, __builtin_bit_cast(h8, x), acc[i], 0, 0, 0);
      }
    }
    const uint32_t old = b0;
    b0 = b1;
    b1 = b2;
    b2 = old;
  }
  __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));  // nothing may still be writing LDS at exit

  // lane l of a 16 x 16 tile holds columns 4 (l / 16) + e of place l % 16
  if (r >= tile.rows) return;
  const int place = tile.first + r, pair = a.order[place];
  if (pair < 0 || pair >= pairs) return;
  w4_half* const out = a.out + (size_t)(a.to_pairs ? pair : place) * width;
#pragma unroll
  for (int i = 0; i < (GATED ? 1 : 2); ++i) {
    const int col = c0 + 16 * i + 4 * q;
    h4 y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = (_Float16)(GATED ? expert_act(a.act, acc[0][e]) * acc[1][e] : acc[i][e]);
    if (col + 4 <= width) {
      __builtin_memcpy(out + col, &y, 8);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (col + e < width) out[col + e] = __builtin_bit_cast(uint16_t, (_Float16)y[e]);
    }
  }
}

template <int FMT, bool GATED, int GM>
__global__ __launch_bounds__(64 * ES_WAVES, 2) void experts_step_kernel(ExpertArgs a, int columns, uint32_t group_mul) {
  const ExpertTile tile = find_expert_tile<16, false, true>(a.offsets, a.experts, a.tokens * a.top_k, columns, blockIdx.x);
  const int rows = __builtin_amdgcn_readfirstlane(tile.rows);
  if (rows == 0) return;
  const ExpertTile u{__builtin_amdgcn_readfirstlane(tile.expert), __builtin_amdgcn_readfirstlane(tile.first), rows,
                     __builtin_amdgcn_readfirstlane(tile.column)};
  if (rows > 8) return experts_step<FMT, GATED, GM, 2>(a, u, group_mul);
  experts_step<FMT, GATED, GM, 1>(a, u, group_mul);
}

template <int FMT, bool GATED, int GM>
hipError_t go(const ExpertArgs& a, hipStream_t s) {
  // more than 64 KB of LDS has to be granted per device, once
  constexpr int LDS = ES_STAGES * es_stage(FMT, GM);
  static std::atomic<bool> granted[64] = {};
  int dev = 0;
  if (hipError_t e = hipGetDevice(&dev); e != hipSuccess) return e;
  if (dev < 0 || dev >= 64 || !granted[dev]) {
    const hipError_t e = hipFuncSetAttribute((const void*)experts_step_kernel<FMT, GATED, GM>,
                                             hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
    if (e != hipSuccess) return e;
    if (dev >= 0 && dev < 64) granted[dev] = true;
  }
  const int R = a.v.N / a.experts, columns = GATED ? (R / 2 + 63) / 64 : (R + 127) / 128;
  const long long grid = (most_expert_tiles(a, 16) * columns + 7) / 8 * 8;
  if (grid > 0x7FFFFFFFLL) return hipErrorInvalidConfiguration;
  // the group of slice n of 32 k is (2 n group_mul) >> 32
  const uint32_t d = a.v.mx ? 1 : a.v.gs / 32, mul = (uint32_t)(((1ull << 31) + d - 1) / d);
  experts_step_kernel<FMT, GATED, GM><<<dim3((unsigned)grid), dim3(64 * ES_WAVES), LDS, s>>>(a, columns, mul);
  return hipGetLastError();
}

template <int FMT, int GM>
hipError_t go_act(const ExpertArgs& a, hipStream_t s) {
  return a.act ? go<FMT, true, GM>(a, s) : go<FMT, false, GM>(a, s);
}

template <int FMT>
hipError_t go_groups(const ExpertArgs& a, hipStream_t s) {
  if (a.v.gs == 128) return go_act<FMT, 0>(a, s);
  if (a.v.gs == 64) return go_act<FMT, 1>(a, s);
  if (a.v.gs == 32) return go_act<FMT, 2>(a, s);
  return go_act<FMT, 3>(a, s);
}

}  // namespace

bool try_experts_step(const ExpertArgs& a, hipStream_t s, hipError_t* err) {
  const WView& v = a.v;
  const long long G = v.mx ? v.B : v.G, R = v.N / a.experts, pairs = (long long)a.tokens * a.top_k;
  if (v.K % 32 || (!v.mx && v.gs % 32) || v.K >= 1 << 20) return false;
  if ((long long)v.N * G % (v.mx ? 4 : 2)) return false;  // the dword around the last scale lies inside the array
  // offsets of 32 bits: an expert's codes, rows of x
  if (R * v.K / 2 >= 1LL << 32 || (a.from_tokens && (long long)a.tokens * v.K * 2 >= 1LL << 32)) return false;
  if ((((uintptr_t)v.q | (uintptr_t)a.x) & 15) || ((uintptr_t)v.scales & 3) || ((uintptr_t)v.zeros & 3)) return false;
  if ((pairs < a.experts ? pairs : a.experts) * R < 256 * 128) return false;
  *err = v.mx ? go_act<2, 2>(a, s) : v.symmetric ? go_groups<0>(a, s) : go_groups<1>(a, s);
  return true;
}

}  // namespace w4k
