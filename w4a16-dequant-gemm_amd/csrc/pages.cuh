// What the kernels of paged FP8 attention share: which rows a sequence has, where a position lies, and
// how the parts of a row that several workgroups formed are joined.
//
// A row is one query token and head.  For position t on page p with scales sk, sv and a row's raw dot product s of
// codes, its score in units of log2 is x = s sk c, c = log2(e) / sqrt(D), and its weight on the raw V codes is
// 2^x sv.  Sums are kept relative to M, the running maximum of x + log2(sv): the weights that enter the matrix
// product in FP16 then stay at most 1 whatever the scales are, and the denominators, 2^(x - M), stay in FP32.
// (Relative to the maximum of x alone, weights of pages whose V scale is small would fall below FP16's range.)
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

struct PagesPlan {
  int split_len, nsplit;  // positions per split, splits of the longest sequence
};

// Sequences of up to few_rows rows per KV head are the kernel's for few rows, the others the one for many.
struct Pages : PagesArgs {
  Divider by_page;
  int few_rows;
  PagesPlan few, many;
  int slots;        // splits of a row that the workspace has room for
  float* part;      // [row][slots][D + 2]: M, denominator, O
  uint32_t* count;  // arrivals, for the kernel for few rows; null: the join kernel has its rows
  int count_shift;  // (sequence, KV head) units are 2^count_shift counters apart
};
// The workspace begins with a fixed room for counters: wherever another call's partial sums begin, no
// call finds anything but zeros where it counts.  Counters are spread over it, because arrivals on one line wait for
// each other.
constexpr int PG_COUNTERS = 16384;

// pages_few.hip.  Most rows of a sequence and KV head that its kernel takes; 0: not this call's dimensions.
int pages_few_most(const PagesArgs& a);
PagesPlan pages_few_plan(const PagesArgs& a, int rows);
hipError_t launch_pages_few(const Pages& a, hipStream_t s);
// Whether the last workgroup of every unit joins its splits itself.
bool pages_few_joins(const PagesArgs& a, const PagesPlan& p, int rows);
// pages_many.hip
bool pages_many_applies(const PagesArgs& a);
PagesPlan pages_many_plan(const PagesArgs& a);
hipError_t launch_pages_many(const Pages& a, hipStream_t s);

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
__device__ __forceinline__ Seq sequence(const Pages& a, int s) {
  Seq q;
  q.q0 = a.cu ? a.cu[s] : s;
  const int end = a.cu ? a.cu[s + 1] : s + 1;
  q.n = q.q0 < 0 ? 0 : min(min(end, a.tokens) - q.q0, a.max_q);
  const int len = a.lens[s];
  q.len = max(0, min(len, a.max_len));
  q.shown = a.causal ? len - (end - q.q0) + 1 : q.len;
  return q;
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
// One wave joins the splits of a row into its output.
template <int BATCH>
__device__ __forceinline__ void join_row(const float* part, int ns, int D, w4_half* out) {
  const int lane = threadIdx.x & 63, pitch = D + 2;
  float M = -INFINITY, den = 0.0f;
  for (int t0 = 0; t0 < ns; t0 += 64) {
    const float2 ml = published(part + (long long)min(t0 + lane, ns - 1) * pitch);
    float m = t0 + lane < ns ? ml.x : -INFINITY;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
    m = fmaxf(M, m);
    const float use = m == -INFINITY ? 0.0f : m;
    float w = t0 + lane < ns ? __builtin_amdgcn_exp2f(ml.x - use) * ml.y : 0.0f;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) w += __shfl_xor(w, d, 64);
    den = den * __builtin_amdgcn_exp2f(M - use) + w;
    M = m;
  }
  const float use = M == -INFINITY ? 0.0f : M, inv = den == 0.0f ? 0.0f : 1.0f / den;
  for (int d0 = 2 * lane; d0 < D; d0 += 128) {
    float sum0 = 0.0f, sum1 = 0.0f;
    for (int t0 = 0; t0 < ns; t0 += BATCH) {
      float2 col[BATCH];
      float m[BATCH];
#pragma unroll
      for (int t = 0; t < BATCH; ++t) {
        const float* const p = part + (long long)min(t0 + t, ns - 1) * pitch;
        col[t] = published(p + 2 + d0), m[t] = published(p).x;
      }
#pragma unroll
      for (int t = 0; t < BATCH; ++t) {
        const float w = t0 + t < ns ? __builtin_amdgcn_exp2f(m[t] - use) : 0.0f;
        sum0 += w * col[t].x, sum1 += w * col[t].y;
      }
    }
    const h2 v = h2{(_Float16)(sum0 * inv), (_Float16)(sum1 * inv)};
    out[d0] = (uint16_t)as_u32(v), out[d0 + 1] = (uint16_t)(as_u32(v) >> 16);
  }
}
__device__ __forceinline__ float* part_of(const Pages& a, long long row, int split) {
  return a.part + (row * a.slots + split) * (a.D + 2);
}

// A page of a split or a stretch of one, in LDS.  Where the V scale is 0 the kernels read zeros for the codes.
struct PageEntry {
  int row0;   // first row of the page in its head's pool; -1: no page of the pool
  float skc;  // scale of K times c, not 0 (a masked score, -infinity, stays that when multiplied)
  float lsv;  // log2 of the scale of V (at least -24: a half); PG_NO_SCALE where it is 0
  float inv;  // 2^-lsv
};
constexpr float PG_NO_SCALE = -25.0f;
__device__ __forceinline__ bool has_scale(const PageEntry& e) { return e.lsv > -24.5f; }
__device__ __forceinline__ PageEntry page_entry(const Pages& a, int s, int h, int j, float c) {
  const int id = a.bt[(long long)s * a.stride + j];
  PageEntry e{-1, 1.0f, PG_NO_SCALE, 0x1p25f};
  if (id >= 0 && id < a.npages) {
    e.row0 = id * a.page;
    e.skc = fmaxf(half_bits_to_float(a.s_k[(long long)h * a.npages + id]) * c, 1e-30f);
    const float sv = half_bits_to_float(a.s_v[(long long)h * a.npages + id]);
    if (sv > 0.0f) e.lsv = __log2f(sv), e.inv = 1.0f / sv;
  }
  return e;
}

// Eight E4M3 codes as halves (exact).
__device__ __forceinline__ h8 codes_to_half(uint32_t lo, uint32_t hi) {
  const h2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true);
  const h2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
  return h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
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

__device__ __forceinline__ float f8_to_float(uint32_t b) {
  const float m = __builtin_bit_cast(float, (b & 0x7Fu) << 20) * 0x1p120f;
  const float v = (b & 0x7Fu) == 0x7Fu ? __builtin_nanf("") : m;
  return b & 0x80u ? -v : v;
}

}  // namespace w4k
