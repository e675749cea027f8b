// Paged FP8 attention for many rows: prompts and chunks of them.
//
// A workgroup takes 128 rows of one (sequence, KV head) -- row = token * group + head, so the heads of a group
// share what is read -- and the positions of a split; a wave has 32 rows as the columns of
//   scores  S[t][row] = sum_d K[t][d] q[row][d]    v_mfma_f32_32x32x16_f16, A = 32 K rows, B = queries (in registers)
//   output  O^T[d][row] += sum_t V[t][d] w[t][row]  A = 32 d of V transposed, B = the weights straight from the score registers:
//           lane (row, half f) has positions 8 g + 4 f .. + 3 of the 32, and the transposed reads of V follow that
// Tiles of 64 positions go through three slots of LDS: whole rows by direct loads, requested two tiles ahead, one
// barrier per tile.  Codes are converted by each wave after it has read them: half the LDS traffic of
// converted tiles, which would take as long as the matrix products.
// Weights are formed as 2^(x + log2(sv) - M) at once; the denominator takes a page's sum times 1 / sv.
// Bound: vector ALUs and matrix cores in turn -- 128 conversions of two codes, 32 exponentials and some 230 other instructions for
// a wave's tile of 64 positions, then 32 matrix products: the first are busy 0.62 of the time, the second 0.38, and little of
// one runs beside the other.  Two prompts of 4096 and 3777 tokens, 8 KV heads of 4 query heads, D = 128: 313 to 323 us by
// card, 800 TFLOP/s (a large library product of halves: 1330).
#pragma once

#include "pages.cuh"

namespace w4k {
namespace {

constexpr int PM_ROWS = 128, PM_TILE = 64, PM_WAVES = 4;
constexpr int PM_SLOTS = 3;  // one is multiplied, one lands, one is requested
constexpr int PM_TABLE = 512;  // pages that are looked up at a time
typedef float f16v __attribute__((ext_vector_type(16)));

// Tiles of rows that a sequence has here.
__device__ __forceinline__ int tiles_of(const Pages& a, int s) {
  const int rows = sequence_of_lane(a, s).n * a.group;
  return rows <= a.few_rows ? 0 : (rows + PM_ROWS - 1) / PM_ROWS;
}

template <int D, bool P16>
struct ManyShared {
  __attribute__((aligned(16))) uint8_t ring[PM_SLOTS][2 * PM_TILE * D];
  PageEntry table[PM_TABLE];
  __attribute__((aligned(16))) float scale_of[P16 ? 1 : PM_SLOTS][3][PM_TILE];  // skc, lsv, inv of each position
  int odd;  // a page of the table is none of the pool, or has a V scale of 0
};
// Workgroup wg of a split.
// P16: pages of a multiple of 16 rows: eight of a lane's scores in a row have one page, the same in all lanes.  Otherwise
// the scales of a tile's positions are laid out one by one when it is requested: 345 us for the two prompts instead of
// 325 (same card).
template <int D, bool P16>
__device__ __forceinline__ void many_rows(const Pages& a, const int wg, const int split, ManyShared<D, P16>& sh) {
  constexpr int P = D / 16, NE = D / 32;  // pieces of a row, 32-element blocks of it
  constexpr int SIDE = PM_TILE * D, SLOT = 2 * SIDE, LOADS = 2 * P / PM_WAVES;
  auto& ring = sh.ring;
  auto& table = sh.table;
  auto& scale_of = sh.scale_of;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c32 = lane & 31, half = lane >> 5;
  // heads first: the workgroups of one head's pages run on one XCD where there are eight heads
  const int h = wg % a.H;
  // ---- which tile of which sequence: 64 sequences at a time, the lanes sum up their tiles
  int s = 0, left = wg / a.H, count = 0;
  for (int base = 0;; base += 64) {
    if (base >= a.nseq) return;
    count = tiles_of(a, min(base + lane, a.nseq - 1));
    if (base + lane >= a.nseq) count = 0;
    const int sum = wave_prefix(count);
    const uint64_t past = __builtin_amdgcn_ballot_w64(sum > left);
    if (past) {
      const int at = __builtin_ctzll(past);
      left -= __builtin_amdgcn_readlane(sum - count, at);
      count = __builtin_amdgcn_readlane(count, at);
      s = __builtin_amdgcn_readfirstlane(base + at);
      break;
    }
    left -= __builtin_amdgcn_readlane(sum, 63);
  }
  // later tokens first: under a causal mask they have the most to do
  const int tile = __builtin_amdgcn_readfirstlane(count - 1 - left);
  const Seq q = sequence(a, s);
  const int rows = q.n * a.group, heads = a.H * a.group, r0 = tile * PM_ROWS;
  const int ns = max(1, splits(a.many, q.len));
  if (split >= ns) return;
  const float c = 1.44269504088896340736f / sqrtf((float)D);
  // positions that the workgroup's rows see, that the wave's rows see, that all of the wave's rows see
  const int w0 = r0 + 32 * wave;
  auto seen_by = [&](int row) { return a.causal ? min(q.len, q.shown + min(row, rows - 1) / a.group) : q.len; };
  const int s0 = split * a.many.split_len, s1 = min(seen_by(r0 + PM_ROWS - 1), s0 + a.many.split_len);
  const int wave_end = w0 < rows ? min(s1, seen_by(w0 + 31)) : 0, wave_all = seen_by(w0);
  const int all_see = seen_by(r0);
  const int row = min(w0 + c32, rows - 1), tok = row / a.group;
  const int sees = seen_by(row);
  const long long at = (long long)(q.q0 + tok) * heads + h * a.group + (row - tok * a.group);

  // ---- queries: step m of the lane's half holds 8 elements from 16 (2 (m / 2) + half) + 8 (m % 2)
  h8 qop[P];
  {
    const w4_half* const qp = a.q + (long long)(q.q0 + tok) * a.q_stride + (long long)(h * a.group + (row - tok * a.group)) * D;
#pragma unroll
    for (int m = 0; m < P; ++m) __builtin_memcpy(&qop[m], qp + 16 * (2 * (m >> 1) + half) + 8 * (m & 1), 16);
  }

  const uint8_t* const kbase = a.q_k + (long long)h * a.npages * a.page * D;
  const uint8_t* const vbase = a.q_v + (long long)h * a.npages * a.page * D;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_ptr)ring;
  // pieces swapped by row: 16 K rows x one piece, and 8 V rows x two pieces, on different banks
  auto kswz = [](int r) { return P == 16 ? r & 15 : P == 8 ? (r >> 1) & 7 : P == 4 ? (r >> 2) & 3 : 0; };
  auto vswz = [](int r) {
    const int hi = (r >> 3) & 1;
    return P == 16 ? ((r & 3) | hi << 2) << 1 : P == 8 ? (((r >> 1) & 1) | hi << 1) << 1 : P == 4 ? hi << 1 : 0;
  };

  f16v o[NE];
#pragma unroll
  for (int e = 0; e < NE; ++e) o[e] = f16v{};
  float M = -INFINITY, l = 0.0f;
  int j0 = 0;  // first page of the table
  bool odd_pages = false;
  uint32_t lane_off[LOADS];  // of the wave's loads: a lane's bytes past the first row
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const int n = wave * LOADS + i, u = (n % P) * 64 + lane, r = u / P;
    lane_off[i] = (r - (n % P) * (64 / P)) * D + 16 * ((u % P) ^ (n >= P ? vswz(r) : kswz(r)));
  }

  // Requests the wave's share of the tile at t0 into slot sl; returns which of its positions are there, and which of
  // their rows of V count (`fine`: there, under a scale that is not 0).
  auto request = [&](int sl, int t0, uint64_t& fine) -> uint64_t {
    if constexpr (P16 && 64 % P == 0) {
      // Whole tiles of pages of whole 16s: the rows of a load lie side by side on one page, so its place is a scalar and
      // a lane adds what it always adds.
      if (t0 + PM_TILE <= s1 && !odd_pages) {
        int first[LOADS];
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
          const int n = wave * LOADS + i, r = (n % P) * (64 / P), t = t0 + (r & ~15), j = page_of(a, t);
          first[i] = table[j - j0].row0 + (t - j * a.page) + (r & 15);
        }
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
          const int n = wave * LOADS + i;
          load_to_lds((n >= P ? vbase : kbase) + (long long)__builtin_amdgcn_readfirstlane(first[i]) * D, lane_off[i],
                      lds0 + sl * SLOT + n * 1024);
        }
        fine = ~0ull;
        return ~0ull;
      }
    }
    const int t = t0 + lane;
    bool there = t < s1;
    const int j = there ? page_of(a, t) : j0;
    const PageEntry e = table[j - j0];
    there = there && e.row0 >= 0;
    if (!P16 && lane >> 4 == wave) scale_of[sl][0][lane] = e.skc, scale_of[sl][1][lane] = e.lsv, scale_of[sl][2][lane] = e.inv;
    const int row = there ? e.row0 + (t - j * a.page) : 0;  // (others read row 0 and drop it)
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int n = wave * LOADS + i, u = (n % P) * 64 + lane, r = u / P, piece = u % P;
      const long long off = (long long)__shfl(row, r, 64) * D;
      const bool v = n >= P;
      load_to_lds((v ? vbase : kbase) + off + 16 * (piece ^ (v ? vswz(r) : kswz(r))), lds0 + sl * SLOT + n * 1024);
    }
    fine = __builtin_amdgcn_ballot_w64(there && has_scale(e));
    return __builtin_amdgcn_ballot_w64(there);
  };

  const int i16 = lane & 15;
  const int vrow = ((i16 >> 1) < 4 ? (i16 >> 1) : 4 + (i16 >> 1)) + 4 * half;  // of the 16 positions of a step

  // A tile's three steps.  Reads of LDS stand together ahead of what uses them, so that one latency is waited for and
  // not one per matrix product: all of a tile's K (D = 256: a half), and its V before the softmax.
  f16v sc[2];
  constexpr int VG = NE > 4 ? 0 : NE < 4 || P16 ? 4 : 2;  // steps of 16 positions whose V is read ahead, as registers allow
  u2 vraw[VG ? VG : 1][NE];
  h8 pop[4];
  auto scores = [&](const uint8_t* slot) {
    constexpr int KG = P <= 8 ? P / 2 : 4;
#pragma unroll
    for (int b = 0; b < 2; ++b) sc[b] = f16v{};
#pragma unroll
    for (int g = 0; g < P / 2; g += KG) {
      u4 w[2][KG];
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < KG; ++i) w[b][i] = *(const u4*)(slot + 32 * b * D + c32 * D + 16 * ((2 * (g + i) + half) ^ kswz(c32)));
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < KG; ++i)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          sc[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(codes_to_half(w[b][i][0], w[b][i][1]), qop[2 * (g + i)], sc[b], 0, 0, 0);
          sc[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(codes_to_half(w[b][i][2], w[b][i][3]), qop[2 * (g + i) + 1], sc[b], 0, 0, 0);
        }
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  auto v_of = [&](const uint8_t* slot, int kk, int e, int from, int l) {
    return slot + SIDE + 16 * kk * D + from * D + 8 * (l & 1) + 16 * ((2 * e + ((l >> 4) & 1)) ^ vswz(from));
  };
  auto read_v = [&](const uint8_t* slot, int kk, int e) {
    return read_transposed(v_of(slot, kk, e, vrow, lane));
  };
  constexpr int SAME = 8;
  float skc[4], lsv[4], inv[4];
  // register k = 16 b + 4 g + i of the scores is position 32 b + 8 g + 4 half + i
  auto position = [&](int k) { return 32 * (k >> 4) + 8 * ((k >> 2) & 3) + 4 * half + (k & 3); };
  auto read_scales = [&](int t0) {
    if constexpr (P16)
#pragma unroll
      for (int k = 0; k < 32; k += SAME) {  // (positions past the split have the last one's)
        const PageEntry e = table[page_of(a, min(t0 + position(k) - 4 * half, s1 - 1)) - j0];
        skc[k / SAME] = e.skc, lsv[k / SAME] = e.lsv, inv[k / SAME] = e.inv;
      }
  };
  auto weights = [&](int sl, int t0, uint64_t there, uint64_t fine) {
    uint8_t* const slot = ring[sl];
    if (fine != ~0ull) {
      // (every wave writes the same, also what it makes of what another one wrote, before its own reads)
      if (!((fine >> lane) & 1)) clear_row<P>(slot + SIDE + lane * D, (there >> lane) & 1);
      asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
    }
#pragma unroll
    for (int kk = 0; kk < VG; ++kk)
#pragma unroll
      for (int e = 0; e < NE; ++e) vraw[kk][e] = read_v(slot, kk, e);
    __builtin_amdgcn_sched_barrier(0);
    if (there != ~0ull || t0 + PM_TILE > wave_all) {  // wave-uniform
      const uint64_t mine = there >> (4 * half);
      const int left = sees - t0 - 4 * half;
#pragma unroll
      for (int k = 0; k < 32; ++k) {
        const int at = position(k) - 4 * half;
        if (!((mine >> at) & 1) || at >= left) sc[k >> 4][k & 15] = -INFINITY;
      }
    }
    float top = -INFINITY;
    if constexpr (P16) {
#pragma unroll
      for (int k = 0; k < 32; k += SAME) {
        float m = sc[k >> 4][k & 15];
#pragma unroll
        for (int i = 1; i < SAME; ++i) m = fmaxf(m, sc[k >> 4][(k & 15) + i]);
        top = fmaxf(top, __builtin_fmaf(m, skc[k / SAME], lsv[k / SAME]));
      }
    } else {
#pragma unroll
      for (int k = 0; k < 32; k += 4) {
        const f4 z = *(const f4*)&scale_of[sl][0][position(k)], v = *(const f4*)&scale_of[sl][1][position(k)];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float y = __builtin_fmaf(sc[k >> 4][(k & 15) + i], z[i], v[i]);
          sc[k >> 4][(k & 15) + i] = y;
          top = fmaxf(top, y);
        }
      }
    }
    top = max_over_32(top);
    if (__builtin_amdgcn_ballot_w64(top > M + PG_SLACK) != 0) {  // wave-uniform
      const float m_new = fmaxf(M, top);
      const float alpha = m_new == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(M - m_new);
#pragma unroll
      for (int e = 0; e < NE; ++e) o[e] *= alpha;
      l *= alpha;
      M = m_new;
    }
    const float use = M == -INFINITY ? 0.0f : M - PG_LIFT;
    // (denominators take the weights as they are in FP32: under a small scale of V the halves lose what they need)
    if constexpr (P16) {
#pragma unroll
      for (int k0 = 0; k0 < 32; k0 += SAME) {
        const float add = lsv[k0 / SAME] - use;
        float sum = 0.0f;
#pragma unroll
        for (int k = k0; k < k0 + SAME; ++k) {
          const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[k >> 4][k & 15], skc[k0 / SAME], add));
          sum += w;
          pop[k >> 3][k & 7] = (_Float16)w;
        }
        l = __builtin_fmaf(sum, inv[k0 / SAME], l);
      }
    } else {
#pragma unroll
      for (int k0 = 0; k0 < 32; k0 += 4) {
        const f4 z = *(const f4*)&scale_of[sl][2][position(k0)];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int k = k0 + i;
          const float w = __builtin_amdgcn_exp2f(sc[k >> 4][k & 15] - use);
          l = __builtin_fmaf(w, z[i], l);
          pop[k >> 3][k & 7] = (_Float16)w;
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  auto add_values = [&](const uint8_t* slot) {
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {  // 16 positions
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        const u2 w = kk < VG ? vraw[kk < VG ? kk : 0][e] : read_v(slot, kk, e);
        o[e] = __builtin_amdgcn_mfma_f32_32x32x16_f16(codes_to_half(w[0], w[1]), pop[kk], o[e], 0, 0, 0);
      }
      if (kk >= VG) __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto barrier = []() {
    asm volatile("" : : : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" : : : "memory");
  };

  // A tile that the first of the workgroup's rows does not see all of, with a NaN code of V in it: the rows that see the code
  // are NaN, then it is taken out for the others.  (All waves look at the whole tile, so they agree on the barriers.)
  auto nan_codes_of = [&](uint8_t* slot, int t0, uint64_t there) {
    int own = lane, from = vrow;  // (unknown to the compiler, which keeps addresses of this way out of the loop's registers)
    asm volatile("" : "+v"(own), "+v"(from));
    u4* const v = (u4*)(slot + SIDE);
    uint32_t nan = 0;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const u4 w = v[64 * i + own];
      nan |= has_nan_code(w[0]) | has_nan_code(w[1]) | has_nan_code(w[2]) | has_nan_code(w[3]);
    }
    if (__builtin_amdgcn_ballot_w64(nan != 0) == 0) return;
    const uint64_t mine = there >> (4 * (own >> 5));
    const int left = sees - t0 - 4 * (own >> 5);
#pragma unroll
    for (int e = 0; e < NE; ++e) {
      f16v n = f16v{};
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        __builtin_amdgcn_sched_barrier(0);  // (one at a time: registers are for the way that is taken)
        const u2 w = read_transposed(v_of(slot, kk, e, from, own));
        h8 seen;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int at = position(8 * kk + k) - 4 * half;  // (a constant)
          seen[k] = ((mine >> at) & 1) && at < left ? (_Float16)1.0f : (_Float16)0.0f;
        }
        const h8 ones = codes_to_half(nan_codes(w[0]) & 0x38383838u, nan_codes(w[1]) & 0x38383838u);  // 0x38: 1
        n = __builtin_amdgcn_mfma_f32_32x32x16_f16(ones, seen, n, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) n[i] = n[i] > 0.0f ? __builtin_nanf("") : 0.0f;
      o[e] += n;
    }
    asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
    barrier();
#pragma unroll 1
    for (int i = tid; i < SIDE / 16; i += PM_WAVES * 64) {
      u4 w = v[i];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] &= ~nan_codes(w[j]);
      v[i] = w;
    }
    asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
    barrier();
  };

  // ---- stretches of the split whose pages fit the table
  const int stretch = (int)min((long long)(PM_TABLE - 2) * a.page / PM_TILE * PM_TILE, (long long)a.many.split_len);
  for (int c0 = s0; c0 < s1; c0 += stretch) {
    const int c1 = min(s1, c0 + stretch);
    j0 = page_of(a, c0);
    const int pages = page_of(a, c1 - 1) - j0 + 1;
    __syncthreads();  // (the table and the slots of the stretch before are still being read)
    if (tid == 0) sh.odd = 0;
    __syncthreads();
    for (int i = tid; i < pages; i += PM_WAVES * 64) {
      const PageEntry e = page_entry(a, s, h, j0 + i, c);
      table[i] = e;
      if (e.row0 < 0 || !has_scale(e)) sh.odd = 1;
    }
    __syncthreads();
    odd_pages = __builtin_amdgcn_readfirstlane(sh.odd) != 0;
    const int nit = (c1 - c0 + PM_TILE - 1) / PM_TILE;
    // (what is known of the tile at hand, and of the next one)
    uint64_t there = 0, fine = 0, there1 = 0, fine1 = 0;
    there = request(0, c0, fine);
    if (1 < nit) there1 = request(1, c0 + PM_TILE, fine1);
    // (a wave's scales are read by the others behind the next barrier, which waits for no store by itself; later tiles' are
    // waited for at the end of the tile that requests them)
    if constexpr (!P16) asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
    int sl = 0;
#pragma unroll 1
    for (int it = 0; it < nit; ++it) {
      const int t0 = c0 + PM_TILE * it;
      // the wave's share of tile `it` has landed (the next tile's may be in flight), then everybody's, and nobody
      // reads the slot before it any more
      if (it + 1 < nit) asm volatile("s_waitcnt vmcnt(%0)" : : "n"(LOADS) : "memory");
      else asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
      barrier();
      uint64_t there2 = 0, fine2 = 0;
      if (it + 2 < nit) there2 = request(sl == 0 ? 2 : sl - 1, t0 + 2 * PM_TILE, fine2);
      if (t0 + PM_TILE > all_see && s1 > all_see) nan_codes_of(ring[sl], t0, there);  // uniform
      if (t0 < wave_end && there) {
        read_scales(t0);
        scores(ring[sl]);
        weights(sl, t0, there, fine);
        add_values(ring[sl]);
      }
      asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
      there = there1, fine = fine1, there1 = there2, fine1 = fine2;
      sl = sl == 2 ? 0 : sl + 1;
    }
  }

  l += __shfl_xor(l, 32, 64);
  if (w0 + c32 >= rows) return;
  // element 32 e + 8 g + 4 half + i of the row is o[e][4 g + i]
  if (ns == 1) {
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    w4_half* const dst = a.out + at * D + 4 * half;
#pragma unroll
    for (int e = 0; e < NE; ++e)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const u2 v = u2{as_u32(h2{(_Float16)(o[e][4 * g] * inv), (_Float16)(o[e][4 * g + 1] * inv)}),
                        as_u32(h2{(_Float16)(o[e][4 * g + 2] * inv), (_Float16)(o[e][4 * g + 3] * inv)})};
        __builtin_memcpy(dst + 32 * e + 8 * g, &v, 8);
      }
  } else {
    float* const dst = part_of(a, at, split);
    if (half == 0) dst[0] = M, dst[1] = l;
#pragma unroll
    for (int e = 0; e < NE; ++e)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        float* const p = dst + 2 + 32 * e + 8 * g + 4 * half;
        *(float2*)p = float2{o[e][4 * g], o[e][4 * g + 1]};
        *(float2*)(p + 2) = float2{o[e][4 * g + 2], o[e][4 * g + 3]};
      }
  }
}

}  // namespace
}  // namespace w4k
