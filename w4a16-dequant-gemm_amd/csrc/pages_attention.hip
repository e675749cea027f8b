// Attention of packed queries over a paged FP8 cache: plan, general kernel, and the join of split rows.
#include "pages.cuh"

namespace w4k {
namespace {

// ---- any head dimension, page size and alignment -----------------------------------------------
// A workgroup takes rows of one split in turn, tiles of 256 positions: a thread forms one position's score, then owns
// four columns of O for every (256 / (D / 4))-th position of the tile.  Nothing is shared between the heads of a group and
// no matrix core is used: 8 x 32768 positions at D = 128 took it 1035 us (the kernel for few rows: 90), two prompts of 4096
// tokens 34.5 ms (the one for many: 313 us).  Bound: the vector ALUs.
__global__ __launch_bounds__(256) void pages_general_kernel(const Pages a) {
  __shared__ float qs[512], red[4], weight[256], o4[256][4];
  __shared__ long long at[256];  // offset of a position's row in the codes; -1: not seen
  const int tid = threadIdx.x, D = a.D, heads = a.H * a.group;
  const int all_rows = a.tokens * heads;
  for (int row = blockIdx.x; row < all_rows; row += gridDim.x) {
    __syncthreads();  // (the row before has been read)
    const int tok = row / heads, head = row - tok * heads, h = head / a.group;
    const int s = sequence_of(a, tok);
    if (s < 0) continue;
    const Seq q = sequence(a, s);
    const int i = tok - q.q0;
    if (i >= q.n || q.n * a.group <= a.few_rows) continue;
    const int end = min(q.len, a.causal ? q.shown + i : q.len);  // positions that the row sees
    const int ns = max(1, splits(a.many, q.len));
    const int split = blockIdx.y;
    if (split >= ns) continue;
    const int s0 = split * a.many.split_len, s1 = min(end, s0 + a.many.split_len);
    const float c = 1.44269504088896340736f / sqrtf((float)D);
    const uint8_t* const kp = a.q_k + (long long)h * a.npages * a.page * D;
    const uint8_t* const vp = a.q_v + (long long)h * a.npages * a.page * D;
    for (int d = tid; d < D; d += 256) qs[d] = half_bits_to_float(a.q[(long long)tok * a.q_stride + (long long)head * D + d]);
    const int cols = D / 4, groups = 256 / cols, g = tid / cols, col = tid - g * cols;
    float M = -INFINITY, l = 0.0f, o[4] = {};
    __syncthreads();
    for (int t0 = s0; t0 < s1; t0 += 256) {
      const int t = t0 + tid;
      float x = -INFINITY, y = -INFINITY, sv = 0.0f;
      long long off = -1;
      if (t < s1) {
        const int j = page_of(a, t);
        const int id = a.bt[(long long)s * a.stride + j];
        if (id >= 0 && id < a.npages) {
          off = ((long long)id * a.page + (t - j * a.page)) * D;
          const uint32_t* const row = (const uint32_t*)(kp + off);
          float dot = 0.0f;
          for (int d = 0; d < D; d += 4) {
            const uint32_t w = row[d / 4];
#pragma unroll
            for (int e = 0; e < 4; ++e) dot = __builtin_fmaf(qs[d + e], f8_to_float((w >> (8 * e)) & 0xFFu), dot);
          }
          sv = half_bits_to_float(a.s_v[(long long)h * a.npages + id]);
          x = dot * (half_bits_to_float(a.s_k[(long long)h * a.npages + id]) * c);
          y = x + (sv > 0.0f ? __log2f(sv) : -25.0f);
        }
      }
      at[tid] = off;
      float m = y;
#pragma unroll
      for (int d = 32; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
      if ((tid & 63) == 0) red[tid >> 6] = m;
      __syncthreads();
      const float m_new = fmaxf(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), M);
      const float use = m_new == -INFINITY ? 0.0f : m_new;
      const float alpha = exp2f(M - use);
      const float p = off >= 0 ? exp2f(x - use) : 0.0f;
      weight[tid] = p * sv;
      M = m_new;
      l = l * alpha + p;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] *= alpha;
      __syncthreads();
      if (g < groups) {
        const int here = min(256, s1 - t0);
        for (int k = g; k < here; k += groups)
          if (at[k] >= 0) {
            const uint32_t w = *(const uint32_t*)(vp + at[k] + 4 * col);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(weight[k], f8_to_float((w >> (8 * e)) & 0xFFu), o[e]);
          }
      }
      __syncthreads();
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) l += __shfl_xor(l, d, 64);
    if ((tid & 63) == 0) red[tid >> 6] = l;
#pragma unroll
    for (int e = 0; e < 4; ++e) o4[tid][e] = o[e];
    __syncthreads();
    l = red[0] + red[1] + red[2] + red[3];
    float* const part = part_of(a, row, split);
    for (int d = tid; d < D; d += 256) {
      float sum = 0.0f;
      for (int k = 0; k < groups; ++k) sum += o4[k * cols + d / 4][d & 3];
      if (ns > 1) part[2 + d] = sum;
      else a.out[(long long)row * D + d] = __builtin_bit_cast(uint16_t, (_Float16)(l == 0.0f ? 0.0f : sum / l));
    }
    if (ns > 1 && tid == 0) part[0] = M, part[1] = l;
  }
}

// ---- rows that several workgroups formed ----------------------------------------------------------
// A wave joins four heads of a token: what is read is twice what the output is times the splits, and all of it is asked
// for at once (four splits of four rows).
constexpr int PJ_ROWS = 4;
__global__ __launch_bounds__(256) void pages_join_kernel(const Pages a, const int blocks) {
  const int heads = a.H * a.group;
  const int tok = (int)(blockIdx.x / blocks);
  const int head = ((int)(blockIdx.x % blocks) * 4 + (threadIdx.x >> 6)) * PJ_ROWS;
  const int s = sequence_of(a, tok);
  if (s < 0 || head >= heads) return;
  const Seq q = sequence(a, __builtin_amdgcn_readfirstlane(s));
  if (tok - q.q0 >= q.n || q.n * a.group <= a.few_rows) return;
  const int ns = splits(a.many, q.len);
  if (ns <= 1) return;
  const float* from[PJ_ROWS];
  w4_half* to[PJ_ROWS];
#pragma unroll
  for (int i = 0; i < PJ_ROWS; ++i) {  // (the last head again where there are no more)
    const long long row = (long long)tok * heads + min(head + i, heads - 1);
    from[i] = part_of(a, row, 0), to[i] = a.out + row * a.D;
  }
  join_rows<PJ_ROWS, 4, false>(from, a.D + 2, ns, a.D, to);
}

PagesPlan general_plan(const PagesArgs& a) {
  // enough splits for four workgroups per compute unit, none shorter than a tile
  const long long rows = (long long)a.tokens * a.H * a.group;
  const int most = (a.max_len + 255) / 256;
  long long n = rows > 0 ? 1024 / rows : 1;
  n = n < 1 ? 1 : n > most ? most : n;
  PagesPlan p;
  p.split_len = (int)(((a.max_len + n - 1) / n + 255) / 256 * 256);
  p.nsplit = (a.max_len + p.split_len - 1) / p.split_len;
  return p;
}

constexpr double FEW_WORK = 7e8;

// Which kernels take the call's sequences, how they split them, and where the workspace's parts lie.
size_t plan(Pages& a) {
  const long long rows = (long long)a.max_q * a.group;
  const bool fast = pages_few_applies(a);
  a.few = FewPlan{};
  a.many = PagesPlan{a.max_len, 1};
  a.few_rows = 0;
  a.mixed = false;
  // Decode and a few tokens per sequence are the kernel's for few rows (8 x 32768 positions 89 us, 175 by the one for many; five
  // tokens each in 16 sequences 19.2 and 24.5).  So is everything up to FEW_WORK (what the scores of all rows come to
  // at most): one launch that cuts rows into blocks of 32 and positions into splits takes 0.5 to 1.2 of the time there that the
  // kernel for many rows, which waits for tile after tile, and its join take, above that 0.7 to 2.4 (140 calls of 1e8
  // to 2.5e9).  Decoding sequences next to prompts: 125 us with the work of both kernels, 147 with the one for many alone.
  if (fast) a.few = pages_few_plan(a, rows);
  const double work = (double)a.tokens * a.H * a.group * a.max_len * a.D;
  if (fast && (rows <= 32 || a.max_q == 1 || (work <= FEW_WORK && !a.few.alone))) {
    a.few_rows = (int)rows;
  } else if (fast && a.group <= 32 && a.nseq > 1) {  // decoding sequences next to prompts
    a.few_rows = (a.group + 15) / 16 * 16;
    // over half of the card where its units are split then, else over all of it (256 sequences of 900 to 7680 positions and 8 KV
    // heads, one with a chunk of 512: 508 us so in one launch, 529 in two); two launches where they are split in neither
    a.few = pages_few_plan(a, a.few_rows, true);
    a.mixed = pages_mixed_applies(a);
    if (!a.mixed) {
      a.few = pages_few_plan(a, a.few_rows);
      a.mixed = pages_mixed_applies(a);
    }
  }
  if (rows > a.few_rows) a.many = fast ? pages_many_plan(a, a.few_rows) : general_plan(a);
  size_t floats = 0;
  a.count = nullptr;
  if (a.few_rows && !a.few.alone) {
    a.count = (uint32_t*)a.space;
    a.count_shift = 0;
    while ((long long)a.few.grid << (a.count_shift + 1) <= PG_COUNTERS) ++a.count_shift;
    a.few_part = (float*)a.space + PG_COUNTERS;
    floats = (size_t)a.few.grid * a.few.rows * (a.D + 2);
  }
  a.part = (float*)a.space + PG_COUNTERS + floats;
  if (a.many.nsplit > 1) floats += (size_t)a.tokens * a.H * a.group * a.many.nsplit * (a.D + 2);
  return floats ? (PG_COUNTERS + floats) * sizeof(float) : 0;
}

}  // namespace

size_t pages_attention_space(const PagesArgs& args) {
  Pages a;
  (PagesArgs&)a = args;
  return plan(a);
}

void pages_attention_plan(const PagesArgs& args, int* out) {
  Pages a;
  (PagesArgs&)a = args;
  plan(a);
  const bool more = (long long)a.max_q * a.group > a.few_rows;
  out[0] = !pages_few_applies(a) ? 0 : !more ? 1 : !a.few_rows ? 2 : a.mixed ? 4 : 3;
  out[1] = a.few_rows;
  out[2] = a.many.split_len;
  out[3] = a.many.nsplit;
}

hipError_t launch_pages_attention(const PagesArgs& args, hipStream_t s) {
  Pages a;
  (PagesArgs&)a = args;
  a.by_page = divider(a.page);
  plan(a);
  const long long rows = (long long)a.tokens * a.H * a.group;
  const bool more = (long long)a.max_q * a.group > a.few_rows, fast = pages_few_applies(a);
  hipError_t e = hipSuccess;
  if (a.mixed) e = launch_pages_mixed(a, s);
  else if (a.few_rows) e = launch_pages_few(a, s);
  if (e == hipSuccess && more && fast) {
    if (!a.mixed) e = launch_pages_many(a, s);
  } else if (e == hipSuccess && more) {
    pages_general_kernel<<<dim3((unsigned)(rows < (1 << 20) ? rows : 1 << 20), a.many.nsplit), 256, 0, s>>>(a);
    e = hipGetLastError();
  }
  if (e == hipSuccess && a.many.nsplit > 1) {
    const int blocks = (a.H * a.group + 4 * PJ_ROWS - 1) / (4 * PJ_ROWS);
    pages_join_kernel<<<(unsigned)a.tokens * blocks, 256, 0, s>>>(a, blocks);
    e = hipGetLastError();
  }
  return e;
}

}  // namespace w4k
