// Paged FP8 attention for few rows: one token per sequence, or a handful, for the query heads of one KV head.
//
// A workgroup takes one (sequence, KV head) and a split of its positions; its four waves take tiles of 32
// positions in turn, each with a softmax of its own, and meet once at the end.  Blocks of 16 NT rows are the columns of
//   scores  S[t][row] = sum_d K[t][d] q[row][d]   v_mfma_f32_16x16x32_f16, A = K rows, B = queries; the codes are converted
//           by the hardware (two per instruction, exact) and the page's scale enters the scores, not the elements
//   output  O^T[d][row] += sum_t V[t][d] w[t][row]  A = V transposed: ds_read_b64_tr_b8 takes 8 positions x 16 d out
//           of LDS with a lane's 8 positions of one d side by side; B = the weights straight from the score registers
//           (lane (row, r): positions 4r .. 4r+3 and 16+4r .. 16+4r+3 of the tile, which the reads of V follow)
// K and V tiles reach LDS as whole rows by direct loads (16 bytes a lane, two slots per wave), with pieces swapped
// by row so that neither read has bank conflicts.  Page ids and scales of the split lie in a table in LDS.
// Workgroups find their splits from the lengths on the device; the last one of a unit joins its partial sums in place.
// Bound: HBM, 2 D bytes per position and KV head: 8 sequences of 32768 positions, 8 KV heads of 4 query heads, D = 128:
// 90 us, 6.0 TB/s (a large read: 7.0).  Short or ragged caches are bound by the chain of lengths, page ids, scales, tiles, join: 29 sequences of 400
// to 6007 positions, 4 KV heads, D = 64: 18.5 us, 2.7 TB/s; 4 of up to 300: 6.4 us; 5 tokens in each of 16 sequences of
// up to 1505: 19.2 us.  (On one pool again and again, which the last-level cache holds; cold 1 to 2 us more.)
#pragma once

#include <type_traits>

#include "pages.cuh"

namespace w4k {
namespace {

constexpr int PF_TILE = 32, PF_WAVES = 4, PF_RING = 2;
constexpr int PF_STEP = PF_TILE * PF_WAVES;  // positions that a workgroup's waves take together
constexpr int PF_TABLE = 512;                // pages that are looked up at a time
constexpr int PF_JOIN = 384;                 // most partial sums (rows times splits) that one workgroup joins

// A workgroup's share: a split of a sequence for one KV head and a block of rows.
struct Share {
  int s, h, block, split, ns, len;  // ns splits of len positions each; s < 0: none
  int first;                        // the unit's first workgroup
};

// ceil(u / k) for u below 2^24 and r = 1 / k to the last bits: the quotient is right, or one off
__device__ __forceinline__ int over(int u, int k, float r) {
  const int n = (int)((float)u * r), left = u - n * k;
  return n + (left > 0 ? 1 : left <= -k ? -1 : 0);
}
__device__ __forceinline__ int over(int u, int k) { return over(u, k, __builtin_amdgcn_rcpf((float)k)); }

// What a sequence has: positions in steps of 128, and blocks of rows; 0: it is not this kernel's.
struct Wants {
  int steps, blocks;
};
__device__ __forceinline__ Wants wants_of(const Pages& a, int s) {
  const Seq q = sequence_of_lane(a, min(s, a.nseq - 1));
  const int rows = q.n * a.group;
  const bool none = s >= a.nseq || q.n <= 0 || rows > a.few_rows;
  return Wants{none ? 0 : max(1, (q.len + PF_STEP - 1) / PF_STEP), none ? 0 : (rows + a.few.block - 1) / a.few.block};
}

// Splits of k steps, the same k for all, as short as the grid allows: with U steps in all units and A units,
// U / k + A workgroups are always enough, and U / k have to be; in between four k are tried.  So one
// long sequence among short ones is spread over the card, and equal ones are cut into one round of
// workgroups.  NB: 64 sequences a register.
template <int NB>
__device__ __forceinline__ Share find_share(const Pages& a, int wg) {
  const int lane = threadIdx.x & 63;
  int u[NB], units[NB], U = 0, A = 0, longest = 0;
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const Wants w = wants_of(a, 64 * b + lane);
    u[b] = w.steps, units[b] = w.blocks * a.H;
  }
#pragma unroll
  for (int b = 0; b < NB; ++b) U += u[b] * units[b], A += units[b], longest = max(longest, u[b]);
  const int work = wave_total(U), free = a.few.grid - wave_total(A);
  longest = wave_most(longest);
  // (a unit's last workgroup joins its rows' splits: no more than PF_JOIN of them)
  const int least = max(a.few.step_least, (int)(((long long)longest * a.few.rows + PF_JOIN - 1) / PF_JOIN));
  const int lo = max(least, (int)((float)work / (float)a.few.grid)), hi = max(least, (int)((float)work / (float)free) + 1);
  int k = hi;
#pragma unroll
  for (int c = 3; c >= 0; --c) {
    const int t = lo + (hi - lo) / 4 * c;
    const float r = __builtin_amdgcn_rcpf((float)t);
    int n = 0;
#pragma unroll
    for (int b = 0; b < NB; ++b) n += over(u[b], t, r) * units[b];
    if (wave_total(n) <= a.few.grid) k = t;
  }
  Share x{-1, 0, 0, 0, 0, k * PF_STEP, 0};
  int left = wg;
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const int n = over(u[b], k), sum = wave_prefix(n * units[b]);
    const uint64_t past = __builtin_amdgcn_ballot_w64(sum > left);
    if (x.s < 0 && past) {
      const int at = __builtin_ctzll(past);
      x.s = __builtin_amdgcn_readfirstlane(64 * b + at);
      x.ns = __builtin_amdgcn_readlane(n, at);
      const int in = __builtin_amdgcn_readfirstlane(left) - __builtin_amdgcn_readlane(sum - n * units[b], at);
      const int unit = over(in + 1, x.ns) - 1;
      x.split = in - unit * x.ns;
      x.block = unit / a.H;
      x.h = unit - x.block * a.H;
    }
    left -= __builtin_amdgcn_readlane(sum, 63);
  }
  x.first = wg - x.split;
  return x;
}

template <int D>
struct FewShared {
  __attribute__((aligned(16))) uint8_t ring[PF_WAVES][PF_RING * 2 * PF_TILE * D];
  PageEntry table[PF_TABLE];
  int scaleless;  // a page of the split has a V scale of 0
  uint32_t arrived;
};
// Workgroup wg.  PG4: pages of a multiple of 4 rows (four neighbouring positions have one page, and one read of its scales: 18.5 us
// against 19.5 without for the 29 ragged sequences).
// NB: how many times 64 sequences find_share() looks at (1: 18.5 us for 29 of them, 4: 20.2); 0: no unit is split.
template <int D, int NT, bool PG4, int NB>
__device__ __forceinline__ void few_rows(const Pages& a, const int wg, FewShared<D>& sh) {
  constexpr int P = D / 16, NC = D / 32, NE = D / 16;  // 16-byte pieces of a row, MFMAs of a score, of an output
  constexpr bool WIDE = P % 4 == 0;                    // K operands by 16-byte reads
  constexpr int SIDE = PF_TILE * D, SLOT = 2 * SIDE, KI = SIDE / 1024;
  constexpr int LDW = D + 4;  // floats of a merge row: O[D], denominator, M
  static_assert(16 * LDW * 4 <= PF_RING * SLOT, "the merge rows take the ring's place");
  auto& ring = sh.ring;
  auto& table = sh.table;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c16 = lane & 15, q4 = lane >> 4;
  Share x;
  if constexpr (NB == 0) {
    const int unit = wg / a.H;
    x = Share{unit / a.few.blocks, wg - unit * a.H, unit % a.few.blocks, 0, 1, a.max_len, wg};
  } else {
    x = find_share<NB>(a, wg);
    if (x.s < 0) return;
  }
  x.block = __builtin_amdgcn_readfirstlane(x.block);
  x.s = __builtin_amdgcn_readfirstlane(x.s), x.h = __builtin_amdgcn_readfirstlane(x.h);
  x.split = __builtin_amdgcn_readfirstlane(x.split), x.ns = __builtin_amdgcn_readfirstlane(x.ns);
  x.len = __builtin_amdgcn_readfirstlane(x.len), x.first = __builtin_amdgcn_readfirstlane(x.first);
  const int s = x.s, h = x.h, ns = x.ns, s0 = x.split * x.len;
  // ---- the first pages of the split, asked for next to what the sequence is
  const int stretch = (int)min((long long)(PF_TABLE - 2) * a.page / PF_STEP * PF_STEP, (long long)x.len);
  constexpr int EACH = PF_TABLE / (PF_WAVES * 64);
  int id[EACH];
  auto look_up = [&](int j0, int pages) {
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
      id[k] = a.bt[(long long)s * a.stride + j0 + min(tid + k * PF_WAVES * 64, pages - 1)];
    }
  };
  look_up(page_of(a, s0), page_of(a, min(a.max_len, s0 + stretch) - 1) - page_of(a, s0) + 1);
  const Seq q = sequence(a, s);
  const int all = q.n * a.group, heads = a.H * a.group, r0 = x.block * a.few.block, rows = min(all - r0, a.few.block);
  if (q.n <= 0 || rows <= 0 || all > a.few_rows) return;
  // positions that the block's first row sees, and its last
  const int shown = a.causal ? q.shown + r0 / a.group : q.len;
  const int shown_last = a.causal ? q.shown + (r0 + rows - 1) / a.group : q.len;
  const int s1 = min(min(q.len, shown_last), s0 + x.len);
  const float c = 1.44269504088896340736f / sqrtf((float)D);

  // ---- queries: lane (row c16, q4) of MFMA m holds 8 elements from kcol(m)
  auto kcol = [&](int m) { return WIDE ? 16 * (4 * (m >> 1) + q4) + 8 * (m & 1) : 8 * (4 * m + q4); };
  h8 qop[NT][NC];
  int sees[NT];  // positions that the lane's row sees
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int row = r0 + min(16 * t + c16, rows - 1), tok = row / a.group, head = row - tok * a.group;
    const w4_half* const qp = a.q + (long long)(q.q0 + tok) * a.q_stride + (long long)(h * a.group + head) * D;
#pragma unroll
    for (int m = 0; m < NC; ++m) __builtin_memcpy(&qop[t][m], qp + kcol(m), 16);
    sees[t] = a.causal ? q.shown + tok : q.len;
  }

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
  int j0 = 0;  // first page of the table
  // Requests the tile at t0 into slot sl; returns which of its positions are there.
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
      load_to_lds(kbase + off + 16 * (piece ^ kswz(r)), at + i * 1024);
      load_to_lds(vbase + off + 16 * (piece ^ vswz(r)), at + SIDE + i * 1024);
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

  bool no_scales = false;
  const int vrow = (c16 >> 1) < 4 ? 4 * q4 + (c16 >> 1) : 16 + 4 * q4 + (c16 >> 1) - 4;

  auto compute = [&](uint8_t* slot, int t0, uint32_t there) {
    if (t0 + PF_TILE > shown && shown_last > shown) {  // wave-uniform: some rows see what others do not
      int own = lane, from = vrow;  // (unknown to the compiler, which keeps addresses of this way out of the loop's registers)
      asm volatile("" : "+v"(own), "+v"(from));
      u4* const v = (u4*)(slot + SIDE) + own;
      uint32_t nan = 0;
#pragma unroll
      for (int i = 0; i < KI; ++i) {
        const u4 w = v[64 * i];
        nan |= has_nan_code(w[0]) | has_nan_code(w[1]) | has_nan_code(w[2]) | has_nan_code(w[3]);
      }
      if (__builtin_amdgcn_ballot_w64(nan != 0) != 0) {
        const uint32_t mine = there >> (4 * q4);
        h8 seen[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int at = 16 * (k >> 2) + (k & 3);
            seen[t][k] = ((mine >> at) & 1) && at < sees[t] - t0 - 4 * q4 ? (_Float16)1.0f : (_Float16)0.0f;
          }
#pragma unroll
        for (int e = 0; e < NE; ++e) {
          __builtin_amdgcn_sched_barrier(0);  // (one at a time: registers are for the way that is taken)
          const u2 w = read_transposed(slot + SIDE + from * D + 8 * (own & 1) + 16 * (e ^ vswz(from)));
          const h8 ones = codes_to_half(nan_codes(w[0]) & 0x38383838u, nan_codes(w[1]) & 0x38383838u);  // 0x38: 1
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            f4 n = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, seen[t], f4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i) n[i] = n[i] > 0.0f ? __builtin_nanf("") : 0.0f;
            o[t][e] += n;
          }
        }
#pragma unroll 1
        for (int i = 0; i < KI; ++i) {
          u4 w = v[64 * i];
#pragma unroll
          for (int j = 0; j < 4; ++j) w[j] &= ~nan_codes(w[j]);
          v[64 * i] = w;
        }
        asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
      }
    }
    f4 sc[NT][2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint8_t* const kr = slot + 16 * j * D + c16 * D;
#pragma unroll
      for (int t = 0; t < NT; ++t) sc[t][j] = f4{0.f, 0.f, 0.f, 0.f};
      if constexpr (WIDE) {
#pragma unroll
        for (int i = 0; i < P / 4; ++i) {
          const u4 w = *(const u4*)(kr + 16 * ((4 * i + q4) ^ kswz(c16)));
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
    // register k = 4 j + i of a row's scores is position 16 j + 4 q4 + i
    if (there != ~0u || t0 + PF_TILE > shown) {  // wave-uniform
      const uint32_t mine = there >> (4 * q4);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int left = sees[t] - t0 - 4 * q4;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int at = 16 * (k >> 2) + (k & 3);
          if (!((mine >> at) & 1) || at >= left) sc[t][k >> 2][k & 3] = -INFINITY;
        }
      }
    }
    if (there != ~0u || no_scales) {
      const int t = min(t0 + (lane & 31), s1 - 1);
      const bool here = (there >> (lane & 31)) & 1;
      if (lane < PF_TILE && (!here || !has_scale(table[page_of(a, t) - j0]))) clear_row<P>(slot + SIDE + lane * D, here);
      asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
    }
    const int last = (s1 - 1) - t0;  // (positions past the split have the last one's entry)
    constexpr int SAME = PG4 ? 4 : 1;
    float skc[8 / SAME], lsv[8 / SAME], inv[8 / SAME];
#pragma unroll
    for (int k = 0; k < 8; k += SAME) {
      const PageEntry e = table[page_of(a, t0 + min(16 * (k >> 2) + 4 * q4 + (k & 3), last)) - j0];
      skc[k / SAME] = e.skc, lsv[k / SAME] = e.lsv, inv[k / SAME] = e.inv;
    }
    h8 pop[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float top = -INFINITY;
#pragma unroll
      for (int k = 0; k < 8; k += SAME) {
        float m = sc[t][k >> 2][k & 3];
#pragma unroll
        for (int i = 1; i < SAME; ++i) m = fmaxf(m, sc[t][k >> 2][(k & 3) + i]);
        top = fmaxf(top, __builtin_fmaf(m, skc[k / SAME], lsv[k / SAME]));
      }
      top = max_over_32(max_over_16(top));
      if (__builtin_amdgcn_ballot_w64(top > M[t] + PG_SLACK) != 0) {  // wave-uniform
        const float m_new = fmaxf(M[t], top);
        const float alpha = m_new == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(M[t] - m_new);
#pragma unroll
        for (int e = 0; e < NE; ++e) o[t][e] *= alpha;
        l[t] *= alpha;
        M[t] = m_new;
      }
      const float use = M[t] == -INFINITY ? 0.0f : M[t] - PG_LIFT;
#pragma unroll
      for (int k = 0; k < 8; k += SAME) {
        const float add = lsv[k / SAME] - use;
        float sum = 0.0f;
#pragma unroll
        for (int i = k; i < k + SAME; ++i) {
          const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][i >> 2][i & 3], skc[k / SAME], add));
          sum += w;
          pop[t][i] = (_Float16)w;
        }
        l[t] = __builtin_fmaf(sum, inv[k / SAME], l[t]);
      }
    }
    const uint8_t* const vr = slot + SIDE + vrow * D + 8 * (c16 & 1);
#pragma unroll
    for (int e = 0; e < NE; ++e) {
      const u2 w = read_transposed(vr + 16 * (e ^ vswz(vrow)));
      const h8 v = codes_to_half(w[0], w[1]);
#pragma unroll
      for (int t = 0; t < NT; ++t) o[t][e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pop[t], o[t][e], 0, 0, 0);
    }
  };

  // ---- stretches of the split whose pages fit the table; in each, the wave's tiles: c0 + 32 (wave + 4 it)
  for (int c0 = s0; c0 < s1; c0 += stretch) {
    const int c1 = min(s1, c0 + stretch);
    j0 = page_of(a, c0);
    const int pages = page_of(a, c1 - 1) - j0 + 1;
    if (c0 > s0) {
      __syncthreads();  // the table is still being read
      look_up(j0, pages);
    }
    // (what the first tile waits for is a table entry; the scales come with the tile, and are loaded as halves and
    // without a branch so that nothing waits for them here)
    _Float16 sk[EACH], sv[EACH];
    if (tid == 0) sh.scaleless = 0;
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
      const int i = tid + k * PF_WAVES * 64;
      if (id[k] < 0 || id[k] >= a.npages) id[k] = -1;
      const long long at = (long long)h * a.npages + max(id[k], 0);
      sk[k] = ((const _Float16*)a.s_k)[at], sv[k] = ((const _Float16*)a.s_v)[at];
      if (i < pages) table[i].row0 = id[k] < 0 ? -1 : id[k] * a.page;
    }
    __syncthreads();
    const int nit = (c1 - c0 + PF_STEP - 1) / PF_STEP;
    auto tile_start = [&](int it) { return c0 + PF_TILE * (wave + PF_WAVES * it); };
    uint32_t there[PF_RING];
#pragma unroll
    for (int d = 0; d < PF_RING; ++d)
      if (d < nit) there[d] = request(d, tile_start(d));
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
      const int i = tid + k * PF_WAVES * 64;
      if (i < pages) {
        PageEntry e{id[k] < 0 ? -1 : id[k] * a.page, 1.0f, PG_NO_SCALE, 0x1p25f};
        if (id[k] >= 0) set_scales(e, (float)sk[k], (float)sv[k], c);
        if (!has_scale(e)) sh.scaleless = 1;
        table[i] = e;
      }
    }
    __syncthreads();
    no_scales = sh.scaleless != 0;
    for (int it0 = 0; it0 < nit; it0 += PF_RING) {
#pragma unroll
      for (int d = 0; d < PF_RING; ++d) {
        const int it = it0 + d;
        if (it < nit) {
          // tile `it` has landed; the ones after it may be in flight
          if (it + PF_RING <= nit) asm volatile("s_waitcnt vmcnt(%0)" : : "n"((PF_RING - 1) * 2 * KI) : "memory");
          else asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
          if (there[d]) compute(ring[wave] + d * SLOT, tile_start(it), there[d]);
          asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");  // the slot has been read: refill it
          if (it + PF_RING < nit) there[d] = request(d, tile_start(it + PF_RING));
        }
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
      const int row = r0 + 16 * t + r, tok = row / a.group, head = row - tok * a.group;
      const long long at = (long long)(q.q0 + tok) * heads + h * a.group + head;
      if (ns == 1) {
        const float inv = den4 == 0.0f ? 0.0f : 1.0f / den4;
        const h2 v = h2{(_Float16)(sum0 * inv), (_Float16)(sum1 * inv)};
        w4_half* const dst = a.out + at * D + d;
        dst[0] = (uint16_t)as_u32(v), dst[1] = (uint16_t)(as_u32(v) >> 16);
      } else {
        float* const dst = a.few_part + ((long long)wg * a.few.rows + 16 * t + r) * (D + 2);
        publish(dst + 2 + d, sum0, sum1);
        if (d == 0) publish(dst, top, den4);
      }
    }
    if (t + 1 < NT) __syncthreads();
  }
  if (NB == 0 || ns == 1) return;

  // The unit's workgroup that finishes last joins its splits.  Each counts itself once its partial sums have been
  // written (the stores have come back); the counter wraps to 0 with the last one.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0)
    sh.arrived = __builtin_amdgcn_atomic_inc32(&a.count[x.first << a.count_shift], (uint32_t)(ns - 1), __ATOMIC_RELAXED,
                                            "agent");
  __syncthreads();
  if (sh.arrived != (uint32_t)(ns - 1)) return;
  const long long pitch = (long long)a.few.rows * (D + 2);
  auto join = [&](auto rows_at_a_time, auto batch) {  // (of a wave; the first again where there are no more)
    constexpr int N = decltype(rows_at_a_time)::value;
    for (int i0 = wave; i0 < rows; i0 += N * PF_WAVES) {
      const float* from[N];
      w4_half* to[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int r = i0 + i * PF_WAVES < rows ? i0 + i * PF_WAVES : i0, row = r0 + r, tok = row / a.group;
        from[i] = a.few_part + x.first * pitch + r * (D + 2);
        to[i] = a.out + ((long long)(q.q0 + tok) * heads + h * a.group + (row - tok * a.group)) * D;
      }
      join_rows<N, decltype(batch)::value, true>(from, pitch, ns, D, to);
    }
  };
  if (rows <= PF_WAVES) join(std::integral_constant<int, 1>{}, std::integral_constant<int, 16>{});
  else if (rows <= 2 * PF_WAVES || ns > 8) join(std::integral_constant<int, 2>{}, std::integral_constant<int, 8>{});
  else join(std::integral_constant<int, 5>{}, std::integral_constant<int, 4>{});
}

}  // namespace
}  // namespace w4k
