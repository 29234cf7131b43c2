// kh_paged_select.hip - the pages a cheap score picks for each drafted token
// (kh_paged, KH_PAGED_SELECT).
//
// Score of page b for token i and kv head c: (sum of the group's queries) .
// k_means[b][c]. Products and sums are in 64 bits: whether a page is picked
// hangs on the order of two scores, and 64 bits leave no rounding that two
// orders of summing could disagree about where 32 would.
//
// First kernel: 16 lanes hold one page's mean (as doubles) and take the dot
// product with every token's query sum from the LDS, so the means are read
// once per 16 tokens. Second kernel, a workgroup per (token, kv head): the
// top-th largest score by its bits, 8 at a time from the highest (counts in
// the LDS), until a digit's bin is taken whole; then one ordered sweep writes
// the columns, ties in order of column.
#include <algorithm>

#include "kh_paged.hpp"

namespace kh {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr int kTokens = 16;         // query sums in the LDS at a time
constexpr int kMostDim = 256;
constexpr int kPagesPerGroup = 64;  // pages of a workgroup of the first kernel

__device__ __forceinline__ int held_pages(const kh_paged &p, int s) {
  const int64_t most = (int64_t)p.width * p.page_size;
  const int64_t n = p.lengths[s];
  const int64_t len = n < 0 ? 0 : n > most ? most : n;
  return (int)((len + p.page_size - 1) / p.page_size);
}

__device__ __forceinline__ double act(const void *p, int64_t i, int type) {
  if (type == KH_TYPE_F32) return static_cast<const float *>(p)[i];
  if (type == KH_TYPE_BF16) return (double)(float)static_cast<const __bf16 *>(p)[i];
  return (double)(float)static_cast<const _Float16 *>(p)[i];
}

// A score's bits in its order: larger score, larger key. NaN is 0, below -inf.
__device__ __forceinline__ uint64_t key_of(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  if (x != x) return 0;
  return u >> 63 ? ~u : u | (1ull << 63);
}

// keys[s][n][c][width]
__global__ __launch_bounds__(kThreads) void scores_kernel(const kh_paged p, uint64_t *keys) {
  __shared__ double sums[kTokens][kMostDim];
  const int s = blockIdx.y / p.kv_heads, c = blockIdx.y - s * p.kv_heads;
  const int held = held_pages(p, s);
  const int b0 = blockIdx.x * kPagesPerGroup;
  if (b0 >= held) return;
  const int group = p.heads / p.kv_heads;
  const int lane16 = threadIdx.x & 15, sub = threadIdx.x >> 4;   // 16 pages at a time
  for (int n0 = blockIdx.z * kTokens; n0 < p.draft; n0 += gridDim.z * kTokens) {
    const int nn = min(kTokens, p.draft - n0);
    __syncthreads();
    for (int i = threadIdx.x; i < nn * p.dim; i += kThreads) {
      const int n = i / p.dim, d = i - n * p.dim;
      double sum = 0.0;
      for (int h = 0; h < group; ++h)
        sum += act(p.q, s * p.q_s + (n0 + n) * p.q_n + (int64_t)(c * group + h) * p.q_h + d, p.act_type);
      sums[n][d] = sum;
    }
    __syncthreads();
    for (int b = b0 + sub; b < min(b0 + kPagesPerGroup, held); b += 16) {
      const int page = p.table[s * p.table_s + b];
      const bool there = page >= 0 && page < p.pages;   // else: every score 0
      const float *mean = p.k_means + (there ? page * p.m_p + c * p.m_h : 0);
      // dimensions 4 lane16 .. + 4 of every 64
      double x[kMostDim / 16];
#pragma unroll
      for (int i = 0; i < kMostDim / 64; ++i) {
        const int d = 64 * i + 4 * lane16;
        const bool in = d < p.dim;
        const f32x4 y = *reinterpret_cast<const f32x4 *>(mean + (in ? d : 0));
#pragma unroll
        for (int e = 0; e < 4; ++e) x[4 * i + e] = in && there ? (double)y[e] : 0.0;
      }
      for (int n = 0; n < nn; ++n) {
        double dot = 0.0;
#pragma unroll
        for (int i = 0; i < kMostDim / 64; ++i) {
          const int d = 64 * i + 4 * lane16;
          if (d < p.dim) {
#pragma unroll
            for (int e = 0; e < 4; ++e) dot = fma(x[4 * i + e], sums[n][d + e], dot);
          }
        }
#pragma unroll
        for (int step = 8; step; step /= 2) dot += __shfl_xor(dot, step);
        if (lane16 == 0)
          keys[(((int64_t)s * p.draft + n0 + n) * p.kv_heads + c) * p.width + b] =
              b == held - 1 ? ~0ull : key_of(dot);
      }
    }
  }
}

__global__ __launch_bounds__(kThreads) void top_kernel(const kh_paged p, const uint64_t *all) {
  __shared__ int count[256];
  __shared__ int above[2], wave_count[2][4];
  const int c = blockIdx.x % p.kv_heads, sn = blockIdx.x / p.kv_heads;
  const int s = sn / p.draft, n = sn - s * p.draft;
  const int held = held_pages(p, s);
  const uint64_t *keys = all + ((int64_t)sn * p.kv_heads + c) * p.width;
  int32_t *out = p.selected + s * p.sel_s + n * p.sel_n + c * p.sel_h;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int take = min(held, p.top);
  for (int i = take + tid; i < p.top; i += kThreads) out[i] = -1;
  if (take == held) {
    for (int i = tid; i < held; i += kThreads) out[i] = i;
    return;
  }
  // the take-th largest key: its digits from the top; `need` of the keys that
  // share the digits found so far are still to be taken
  uint64_t found = 0, known = 0;   // digits found, and the bits they cover
  int need = take;
  for (int shift = 56; shift >= 0; shift -= 8) {
    count[tid] = 0;
    __syncthreads();
    for (int i = tid; i < held; i += kThreads) {
      const uint64_t k = keys[i];
      if ((k & known) == found) atomicAdd(&count[(k >> shift) & 255], 1);
    }
    __syncthreads();
    // thread t: how many lie in the bins above bin t (a wave's suffix sums)
    const int mine = count[tid];
    int run = mine;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int o = __shfl_down(run, d);
      if (lane + d < 64) run += o;
    }
    if (lane == 0) wave_count[0][wave] = run;
    __syncthreads();
    int over = run - mine;
    for (int i = wave + 1; i < 4; ++i) over += wave_count[0][i];
    if (over < need && over + mine >= need) {
      above[0] = tid;
      above[1] = over;
    }
    __syncthreads();
    found |= (uint64_t)above[0] << shift;
    known |= 255ull << shift;
    need -= above[1];
    const bool whole = count[above[0]] == need;
    __syncthreads();
    if (whole) break;
  }
  // keys above the digits found are taken, and the first `need` that equal them
  int written = 0, equal = 0;
  for (int i0 = 0; i0 < held; i0 += kThreads) {
    const int i = i0 + tid;
    const uint64_t k = i < held ? keys[i] & known : 0;
    const bool same = i < held && k == found, more = i < held && k > found;
    const uint64_t same_mask = __ballot(same), before = (1ull << lane) - 1;
    if (lane == 0) wave_count[0][wave] = __popcll(same_mask);
    __syncthreads();
    int rank = equal + __popcll(same_mask & before);
    for (int j = 0; j < wave; ++j) rank += wave_count[0][j];
    const bool in = more || (same && rank < need);
    const uint64_t in_mask = __ballot(in);
    if (lane == 0) wave_count[1][wave] = __popcll(in_mask);
    __syncthreads();
    int at = written + __popcll(in_mask & before);
    for (int j = 0; j < wave; ++j) at += wave_count[1][j];
    if (in) out[at] = i;
    for (int j = 0; j < 4; ++j) {
      equal += wave_count[0][j];
      written += wave_count[1][j];
    }
    __syncthreads();
  }
}

}  // namespace

size_t select_workspace_floats(const kh_paged &p) {
  return 2 * (size_t)p.batch * p.draft * p.kv_heads * p.width;
}

hipError_t launch_select(const kh_paged &p, float *workspace, hipStream_t stream) {
  if (p.batch == 0 || p.draft == 0 || p.top == 0) return hipSuccess;
  uint64_t *keys = reinterpret_cast<uint64_t *>(workspace);
  if (p.width > 0) {
    const unsigned chunks = (unsigned)((p.width + kPagesPerGroup - 1) / kPagesPerGroup);
    const unsigned heads = (unsigned)p.batch * p.kv_heads;
    const dim3 grid(chunks, heads, (unsigned)((p.draft + kTokens - 1) / kTokens));
    scores_kernel<<<grid, kThreads, 0, stream>>>(p, keys);
  }
  top_kernel<<<(unsigned)((int64_t)p.batch * p.draft * p.kv_heads), kThreads, 0, stream>>>(p, keys);
  return hipGetLastError();
}

}  // namespace kh
