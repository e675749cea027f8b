// What the kernels of paged FP8 attention share: which rows a sequence has, where a position lies, and
// how the parts of a row that several workgroups formed are joined.
//
// A row is one query token and head.  For position t on page p with scales sk, sv and a row's raw dot product s of
// codes, its score in units of log2 is x = s sk c, c = log2(e) / sqrt(D), and its weight on the raw V codes is
// 2^x sv.  Sums are kept relative to M, the running maximum of x + log2(sv): the weights that enter the matrix
// product in FP16 then have one range whatever the scales are, and the denominators, 2^(x - M), stay in FP32.
// (Relative to the maximum of x alone, weights of pages whose V scale is small would fall below FP16's range.)
// Both are kept 2^PG_LIFT times as large, which falls out of their quotient: M may lag behind by PG_SLACK, so weights go up
// to 2^14 of the 2^16 that a half holds (room for what rounding does to exponents as long as scores are below 2^24), and
// only those 2^-20 of the largest and less lose bits.  A token that takes nearly all of the softmax and has no values
// is ordinary; without the lift, others 2^-25 below it were lost in the numerator and there in the denominator.
#pragma once

#include "dq.cuh"
#include "kernels.h"

namespace w4k {

// t / d for 0 <= t < 2^31 without a division
struct Divider {
  uint32_t magic;
  int shift;
  __device__ __forceinline__ int operator()(int t) const { return (int)(__umulhi(2u * (uint32_t)t, magic) >> shift); }
};
inline Divider divider(int d) {
  Divider v{0, 0};
  while ((1ll << v.shift) < d) ++v.shift;
  v.magic = (uint32_t)((1ull << (31 + v.shift)) / (uint32_t)d + 1);
  return v;
}

// Sums and maxima over a wave by lane moves inside the vector ALU (an exchange through LDS takes a hundred cycles a
// step): inclusive from lane 0 on, so lane 63 has them all.
template <int CTRL, int ROWS>
__device__ __forceinline__ int moved(int x, int none) {
  return __builtin_amdgcn_update_dpp(none, x, CTRL, ROWS, 0xF, false);
}
template <typename F>
__device__ __forceinline__ int wave_scan(int x, int none, F f) {
  x = f(x, moved<0x111, 0xF>(x, none));  // the lane 1, 2, 4, 8 before, in rows of 16
  x = f(x, moved<0x112, 0xF>(x, none));
  x = f(x, moved<0x114, 0xF>(x, none));
  x = f(x, moved<0x118, 0xF>(x, none));
  x = f(x, moved<0x142, 0xA>(x, none));  // lane 15 of rows 0 and 2 into rows 1 and 3
  x = f(x, moved<0x143, 0xC>(x, none));  // lane 31 into rows 2 and 3
  return x;
}
__device__ __forceinline__ int wave_prefix(int x) {
  return wave_scan(x, 0, [](int a, int b) { return a + b; });
}
__device__ __forceinline__ int wave_total(int x) { return __builtin_amdgcn_readlane(wave_prefix(x), 63); }
__device__ __forceinline__ int wave_most(int x) {  // of values that are not negative
  return __builtin_amdgcn_readlane(wave_scan(x, 0, [](int a, int b) { return max(a, b); }), 63);
}
// The larger of a value and the one 32 (16) lanes away.
__device__ __forceinline__ float max_over_32(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
  return fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}
__device__ __forceinline__ float max_over_16(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
  return fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}

struct PagesPlan {
  int split_len, nsplit;  // positions per split, splits of the longest sequence
};

// How the kernel for few rows spreads its work.  Lengths are known on the device alone: its workgroups
// find their splits from them (pages_few.hip).
struct FewPlan {
  int grid;        // workgroups
  int step_least;  // a split has 128 times this positions at least
  int alone;       // 1: no unit (a block of a sequence's rows of one KV head) is split
  int block;       // rows of a block: 16 or 32
  int blocks;      // most of a sequence
  int rows;        // rows of a unit that the workspace has room for
};

// Sequences of up to few_rows rows per KV head are the kernel's for few rows, the others the one for many.
struct Pages : PagesArgs {
  Divider by_page;
  int few_rows;
  bool mixed;  // both kernels' work in one launch
  FewPlan few;
  PagesPlan many;
  uint32_t* count;  // few rows: arrivals of a unit, at its first workgroup's number << count_shift
  int count_shift;
  float* few_part;  // [workgroup][row][D + 2]: M, denominator, O
  float* part;      // many rows: [row][split][D + 2]
};
// The workspace begins with a fixed room for counters: wherever another call's partial sums begin, no
// call finds anything but zeros where it counts.  Counters are spread over it, because arrivals on one line wait for
// each other.
constexpr int PG_COUNTERS = 16384;

// pages_few.hip.  Whether its kernel takes this call's dimensions, and how it spreads sequences of up to so many rows
// per KV head; half: over half of the card.
bool pages_few_applies(const PagesArgs& a);
FewPlan pages_few_plan(const PagesArgs& a, long long rows, bool half = false);
hipError_t launch_pages_few(const Pages& a, hipStream_t s);
// pages_many.hip.  Most tiles of a call's sequences: whole ones, and one that is not for each sequence that has more than
// few_rows.
long long pages_many_tiles(const PagesArgs& a, int few_rows);
PagesPlan pages_many_plan(const PagesArgs& a, int few_rows);
hipError_t launch_pages_many(const Pages& a, hipStream_t s);
// pages_mixed.hip.  Whether one launch can do the work of both, as a.few spreads it.
bool pages_mixed_applies(const Pages& a);
hipError_t launch_pages_mixed(const Pages& a, hipStream_t s);

__device__ __forceinline__ int page_of(const Pages& a, int t) { return a.by_page(t); }

// Sequence that holds packed token `tok`; -1: none.
__device__ __forceinline__ int sequence_of(const Pages& a, int tok) {
  if (!a.cu) return tok < a.nseq ? tok : -1;
  int lo = 0, hi = a.nseq;  // cu[lo] <= tok < cu[hi]
  if (tok < a.cu[0] || tok >= a.cu[a.nseq]) return -1;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.cu[mid] <= tok) lo = mid;
    else hi = mid;
  }
  return lo;
}

// A sequence's queries and positions.  What lies outside the packed tokens, the tables or the bounds of the
// call is left out.
struct Seq {
  int q0, n, len, shown;  // first packed token, tokens, positions; the first token sees shown positions, each next one more
};
__device__ __forceinline__ Seq sequence_from(const Pages& a, int q0, int end, int len) {
  Seq q;
  q.q0 = q0;
  q.n = q0 < 0 ? 0 : min(min(end, a.tokens) - q0, a.max_q);
  q.len = max(0, min(len, a.max_len));
  q.shown = a.causal ? len - (end - q0) + 1 : q.len;
  return q;
}
// (Three loads together: each of them under the condition that needs it is a trip to the cache of its own, which is
// what the empty statement and the lane reads prevent.)
__device__ __forceinline__ Seq sequence(const Pages& a, int s) {  // s: the same in all lanes
  const int* const cu = a.cu ? a.cu + s : a.lens + s;
  const int q0 = __builtin_amdgcn_readfirstlane(cu[0]), end = __builtin_amdgcn_readfirstlane(cu[a.cu ? 1 : 0]);
  const int len = __builtin_amdgcn_readfirstlane(a.lens[s]);
  return sequence_from(a, a.cu ? q0 : s, a.cu ? end : s + 1, len);
}
__device__ __forceinline__ Seq sequence_of_lane(const Pages& a, int s) {
  const int* const cu = a.cu ? a.cu : a.lens;
  int q0 = cu[s], end = cu[s + (a.cu ? 1 : 0)], len = a.lens[s];
  asm volatile("" : "+v"(q0), "+v"(end), "+v"(len));
  return sequence_from(a, a.cu ? q0 : s, a.cu ? end : s + 1, len);
}

__device__ __forceinline__ int splits(const PagesPlan& p, int len) { return (len + p.split_len - 1) / p.split_len; }
// Partial sums pass between workgroups of one launch by stores and loads of agent scope, which go where every XCD sees
// them (a fence instead would write the whole L2 of an XCD back).
__device__ __forceinline__ void publish(float* p, float x, float y) {
  const uint64_t v = __builtin_bit_cast(uint32_t, x) | ((uint64_t)__builtin_bit_cast(uint32_t, y) << 32);
  __hip_atomic_store((uint64_t*)p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 published(const float* p) {
  const uint64_t v = __hip_atomic_load((const uint64_t*)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return float2{__builtin_bit_cast(float, (uint32_t)v), __builtin_bit_cast(float, (uint32_t)(v >> 32))};
}
// One wave joins the splits of N rows into their outputs: every lane has its columns, and all loads of BATCH splits are in
// flight at once.  SAME: the sums come from workgroups of the same launch.
template <int N, int BATCH, bool SAME>
__device__ __forceinline__ void join_rows(const float* const (&part)[N], long long pitch, int ns, int D,
                                          w4_half* const (&out)[N]) {
  for (int d0 = 2 * (threadIdx.x & 63); d0 < D; d0 += 128) {
    float M[N], den[N], sum0[N], sum1[N];
#pragma unroll
    for (int r = 0; r < N; ++r) M[r] = -INFINITY, den[r] = sum0[r] = sum1[r] = 0.0f;
    for (int t0 = 0; t0 < ns; t0 += BATCH) {
      float2 ml[N][BATCH], col[N][BATCH];
#pragma unroll
      for (int t = 0; t < BATCH; ++t)
#pragma unroll
        for (int r = 0; r < N; ++r) {
          const float* const p = part[r] + min(t0 + t, ns - 1) * pitch;
          ml[r][t] = SAME ? published(p) : *(const float2*)p;
          col[r][t] = SAME ? published(p + 2 + d0) : *(const float2*)(p + 2 + d0);
        }
#pragma unroll
      for (int r = 0; r < N; ++r) {
        float m = M[r];
#pragma unroll
        for (int t = 0; t < BATCH; ++t) m = fmaxf(m, ml[r][t].x);  // (the last split again where there are no more)
        const float use = m == -INFINITY ? 0.0f : m, alpha = __builtin_amdgcn_exp2f(M[r] - use);
        M[r] = m;
        den[r] *= alpha, sum0[r] *= alpha, sum1[r] *= alpha;
#pragma unroll
        for (int t = 0; t < BATCH; ++t) {
          const float w = t0 + t < ns ? __builtin_amdgcn_exp2f(ml[r][t].x - use) : 0.0f;
          den[r] += w * ml[r][t].y, sum0[r] += w * col[r][t].x, sum1[r] += w * col[r][t].y;
        }
      }
    }
#pragma unroll
    for (int r = 0; r < N; ++r) {
      const float inv = den[r] == 0.0f ? 0.0f : 1.0f / den[r];
      const h2 v = h2{(_Float16)(sum0[r] * inv), (_Float16)(sum1[r] * inv)};
      out[r][d0] = (uint16_t)as_u32(v), out[r][d0 + 1] = (uint16_t)(as_u32(v) >> 16);
    }
  }
}
__device__ __forceinline__ float* part_of(const Pages& a, long long row, int split) {
  return a.part + (row * a.many.nsplit + split) * (a.D + 2);
}

// A page of a split or a stretch of one, in LDS.  Where the V scale is 0 the kernels read zeros for the codes that are numbers.
struct PageEntry {
  int row0;   // first row of the page in its head's pool; -1: no page of the pool
  float skc;  // scale of K times c, not 0 (a masked score, -infinity, stays that when multiplied)
  float lsv;  // log2 of the scale of V (at least -24: a half); PG_NO_SCALE where it is 0
  float inv;  // 2^-lsv
};
constexpr float PG_SLACK = 8.0f;  // sums are rescaled only when the maximum has risen by this
constexpr float PG_LIFT = 6.0f;
constexpr float PG_NO_SCALE = -25.0f;
__device__ __forceinline__ bool has_scale(const PageEntry& e) { return e.lsv > -24.5f; }
__device__ __forceinline__ void set_scales(PageEntry& e, float sk, float sv, float c) {
  e.skc = fmaxf(sk * c, 1e-30f);
  if (sv > 0.0f) e.lsv = __log2f(sv), e.inv = 1.0f / sv;
}
__device__ __forceinline__ PageEntry page_entry(const Pages& a, int s, int h, int j, float c) {
  const int id = a.bt[(long long)s * a.stride + j];
  PageEntry e{-1, 1.0f, PG_NO_SCALE, 0x1p25f};
  if (id >= 0 && id < a.npages) {
    e.row0 = id * a.page;
    const long long at = (long long)h * a.npages + id;
    set_scales(e, half_bits_to_float(a.s_k[at]), half_bits_to_float(a.s_v[at]), c);
  }
  return e;
}

// Eight E4M3 codes as halves (exact).
__device__ __forceinline__ h8 codes_to_half(uint32_t lo, uint32_t hi) {
  const h2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true);
  const h2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
  return h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Causal rows of a tile that do not see all of it.  A weight of 0 does not keep a NaN code of V out of a matrix product, so
// tiles that hold one (0x7F, 0xFF) go a second way: the codes without it, and a product of what is NaN with what a row sees.
__device__ __forceinline__ uint32_t has_nan_code(uint32_t w) { return ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u; }
__device__ __forceinline__ uint32_t nan_codes(uint32_t w) {  // 0xFF at each
  const uint32_t x = has_nan_code(w) >> 7;
  return (x << 8) - x;
}

// What is left of a row of V in LDS that does not count: zeros where no position is there (it may hold anything, and 0
// times that may be NaN), the NaN codes under a scale of 0, which are NaN all the same.  (The end of every short sequence
// comes this way: zeros are stored without a read, 4 x 300 positions 6.4 us against 7.1.)
template <int PIECES>
__device__ __forceinline__ void clear_row(uint8_t* row, bool there) {
  if (!there) {
#pragma unroll 1
    for (int i = 0; i < PIECES; ++i) *(u4*)(row + 16 * i) = u4{0u, 0u, 0u, 0u};
  } else {
#pragma unroll 1
    for (int i = 0; i < PIECES; ++i) {
      u4 w = *(const u4*)(row + 16 * i);
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] &= nan_codes(w[j]);
      *(u4*)(row + 16 * i) = w;
    }
  }
}

typedef __attribute__((address_space(3))) void* lds_ptr;
typedef int i2 __attribute__((ext_vector_type(2)));
// 8 rows x 16 bytes read transposed by 16 lanes: lane i gives the address of half a row (row i / 2) and gets byte i of
// the eight rows.
__device__ __forceinline__ u2 read_transposed(const uint8_t* p) {
  const i2 w = __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) i2*)p);
  return u2{(uint32_t)w[0], (uint32_t)w[1]};
}
// 16 bytes a lane straight into LDS at `lds` + 16 * lane.
__device__ __forceinline__ void load_to_lds(const uint8_t* from, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off nt" : : "v"(from), "s"(lds) : "memory", "m0");
}

__device__ __forceinline__ void load_to_lds(const uint8_t* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1 nt" : : "v"(off), "s"(base), "s"(lds) : "memory", "m0");
}

__device__ __forceinline__ float f8_to_float(uint32_t b) {
  const float m = __builtin_bit_cast(float, (b & 0x7Fu) << 20) * 0x1p120f;
  const float v = (b & 0x7Fu) == 0x7Fu ? __builtin_nanf("") : m;
  return b & 0x80u ? -v : v;
}

}  // namespace w4k
