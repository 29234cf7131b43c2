// kh_paged_select.hip - the pages a cheap score picks for each drafted token
// (kh_paged, KH_PAGED_SELECT).
//
// Score of page b for token i and kv head c: (sum of the group's queries) .
// k_means[b][c]. Products and sums are in 64 bits: whether a page is picked
// hangs on the order of two scores, and 64 bits leave no rounding that two
// orders of summing could disagree about where 32 would.
//
// First kernel: 16 lanes hold one page's mean (as doubles) and take the dot
// product with every token's query sum from the LDS, four tokens at a time, so
// the means are read once per 16 tokens. Second kernel, a workgroup per (token,
// kv head): the top-th largest score by its bits, 11 at a time from the highest
// (sign and exponent first; counts in the LDS), until a digit's bin is taken
// whole; then one ordered sweep writes the columns, ties in order of column.
// Up to 2048 scores stay in registers meanwhile.
//
// Measured: 16 sequences of up to 512 pages, 8 heads of 128 (17 MB of means)
// 13.5 and 6.4 us; 13 tokens over 1024 pages, 2 sequences, 13.2 (38 with the dot
// products' lane sums through the LDS) and 8.2; 125 pages of 12 heads of 64 4.4
// and 5.4. Both are chains of a few dependent loads, not their bytes.
#include <algorithm>

#include "kh_paged.hpp"

namespace kh {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int kThreads = 256;
constexpr int kTokens = 16;         // query sums in the LDS at a time
constexpr int kPagesPerGroup = 32;  // pages of a workgroup of the first kernel
constexpr int kDigit = 11;          // bits of a score looked at together
constexpr int kHeld = 8;            // scores of a thread in registers

__device__ __forceinline__ int held_pages(const kh_paged &p, int s) {
  const int64_t most = (int64_t)p.width * p.page_size;
  const int64_t n = p.lengths[s];
  const int64_t len = n < 0 ? 0 : n > most ? most : n;
  return (int)((len + p.page_size - 1) / p.page_size);
}

// A score's bits in its order: larger score, larger key. NaN is 0, below -inf.
__device__ __forceinline__ uint64_t key_of(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  if (x != x) return 0;
  return u >> 63 ? ~u : u | (1ull << 63);
}

// n adjacent values of q as doubles added to sum
template <int N>
__device__ __forceinline__ void add_acts(const void *p, int64_t i, int type, double (&sum)[N]) {
  if (type == KH_TYPE_F32) {
    const f32x4 a = *reinterpret_cast<const f32x4 *>(static_cast<const float *>(p) + i);
#pragma unroll
    for (int e = 0; e < N; ++e) sum[e] += (double)a[e];
  } else {
    const u32x2 a = *reinterpret_cast<const u32x2 *>(static_cast<const uint16_t *>(p) + i);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const uint32_t half = a[e / 2] >> (16 * (e & 1)) & 0xffffu;
      sum[e] += (double)(type == KH_TYPE_BF16 ? __uint_as_float(half << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)half));
    }
  }
}

template <int CTRL>
__device__ __forceinline__ double dpp64(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xF, 0xF, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, 0xF, 0xF, false);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double sum16(double x) {   // over the 16 lanes of a row
  x += dpp64<0xB1>(x);    // quad_perm [1,0,3,2]
  x += dpp64<0x4E>(x);    // quad_perm [2,3,0,1]
  x += dpp64<0x141>(x);   // row_half_mirror
  x += dpp64<0x140>(x);   // row_mirror
  return x;
}

// keys[s][n][c][width]. DG: 64-wide groups of dimensions.
template <int DG>
__global__ __launch_bounds__(kThreads) void scores_kernel(const kh_paged p, uint64_t *keys) {
  __shared__ __attribute__((aligned(16))) double sums[kTokens][64 * DG];
  const int s = blockIdx.y / p.kv_heads, c = blockIdx.y - s * p.kv_heads;
  const int b0 = blockIdx.x * kPagesPerGroup;
  const int lane16 = threadIdx.x & 15, sub = threadIdx.x >> 4;   // 16 pages at a time
  int named[kPagesPerGroup / 16];   // (asked for along with the length)
#pragma unroll
  for (int r = 0; r < kPagesPerGroup / 16; ++r) named[r] = p.table[s * p.table_s + min(b0 + 16 * r + sub, p.width - 1)];
  const int held = held_pages(p, s);
  if (b0 >= held) return;
  const int group = p.heads / p.kv_heads;
  // this lane's part of its pages' means: dimensions 4 lane16 .. + 4 of every 64
  constexpr int kRounds = kPagesPerGroup / 16;
  f32x4 mean[kRounds][DG];
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int b = b0 + 16 * r + sub;
    const int page = b < held ? named[r] : -1;
    const bool there = page >= 0 && page < p.pages;   // else: every score 0
    const float *at = p.k_means + (there ? page * p.m_p + c * p.m_h : 0);
#pragma unroll
    for (int i = 0; i < DG; ++i) {
      const int d = 64 * i + 4 * lane16;
      const f32x4 y = *reinterpret_cast<const f32x4 *>(at + (d < p.dim ? d : 0));
      mean[r][i] = there && d < p.dim ? y : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
  }
  const int quads = 16 * DG;
  for (int n0 = blockIdx.z * kTokens; n0 < p.draft; n0 += gridDim.z * kTokens) {
    const int nn = min(kTokens, p.draft - n0);
    const int padded = (nn + 3) & ~3;
    for (int i = threadIdx.x; i < padded * quads; i += kThreads) {
      const int n = i / quads, d = 4 * (i - n * quads);
      double sum[4] = {0.0, 0.0, 0.0, 0.0};
      if (n < nn && d < p.dim) {
        const int64_t at = s * p.q_s + (n0 + n) * p.q_n + (int64_t)(c * group) * p.q_h + d;
#pragma unroll 4
        for (int h = 0; h < group; ++h) add_acts(p.q, at + h * p.q_h, p.act_type, sum);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) sums[n][d + e] = sum[e];
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      const int b = b0 + 16 * r + sub;
      for (int n = 0; n < padded; n += 4) {
        double dot[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
        for (int i = 0; i < DG; ++i)
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) dot[t] = fma((double)mean[r][i][e], sums[n + t][64 * i + 4 * lane16 + e], dot[t]);
#pragma unroll
        for (int t = 0; t < 4; ++t) dot[t] = sum16(dot[t]);
        // (lane t of the 16 writes token n + t)
        double mine = dot[0];
#pragma unroll
        for (int t = 1; t < 4; ++t) mine = lane16 == t ? dot[t] : mine;
        if (lane16 < 4 && n + lane16 < nn && b < held)
          keys[(((int64_t)s * p.draft + n0 + n + lane16) * p.kv_heads + c) * p.width + b] =
              b == held - 1 ? ~0ull : key_of(mine);
      }
    }
    __syncthreads();
  }
}

__global__ __launch_bounds__(kThreads) void top_kernel(const kh_paged p, const uint64_t *all) {
  constexpr int kBins = 1 << kDigit, kPer = kBins / kThreads;
  __shared__ int count[kBins];
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
  uint64_t mine[kHeld];
#pragma unroll
  for (int j = 0; j < kHeld; ++j) mine[j] = j * kThreads + tid < held ? keys[j * kThreads + tid] : 0;
  // the take-th largest key: its digits from the top; `need` of the keys that
  // share the digits found so far are still to be taken
  uint64_t found = 0, known = 0;   // digits found, and the bits they cover
  int need = take;
  for (int shift = 64 - kDigit;;) {
    for (int i = tid; i < kBins; i += kThreads) count[i] = 0;
    __syncthreads();
    auto see = [&](uint64_t k) {
      if ((k & known) == found) atomicAdd(&count[(k >> shift) & (kBins - 1)], 1);
    };
#pragma unroll
    for (int j = 0; j < kHeld; ++j)
      if (j * kThreads + tid < held) see(mine[j]);
    for (int i = kHeld * kThreads + tid; i < held; i += kThreads) see(keys[i]);
    __syncthreads();
    // thread t has bins kPer t ..: how many lie in the bins above them
    int here[kPer], own = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) own += here[j] = count[tid * kPer + j];
    int run = own;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int o = __shfl_down(run, d);
      if (lane + d < 64) run += o;
    }
    if (lane == 0) wave_count[0][wave] = run;
    __syncthreads();
    int over = run - own;
    for (int i = wave + 1; i < 4; ++i) over += wave_count[0][i];
    if (over < need && over + own >= need) {
#pragma unroll
      for (int j = kPer - 1; j >= 0; --j) {
        if (over < need && over + here[j] >= need) {
          above[0] = tid * kPer + j;
          above[1] = over;
        }
        over += here[j];
      }
    }
    __syncthreads();
    found |= (uint64_t)above[0] << shift;   // (a last digit that overlaps the one before agrees with it)
    known |= (uint64_t)(kBins - 1) << shift;
    need -= above[1];
    const bool whole = count[above[0]] == need;
    __syncthreads();
    if (whole || shift == 0) break;
    shift = max(shift - kDigit, 0);
  }
  // keys above the digits found are taken, and the first `need` that equal them
  int written = 0, equal = 0;
  auto sweep = [&](int i, uint64_t k) {
    const bool same = i < held && (k & known) == found, more = i < held && (k & known) > found;
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
  };
#pragma unroll
  for (int j = 0; j < kHeld; ++j)
    if (j * kThreads < held) sweep(j * kThreads + tid, mine[j]);
  for (int i0 = kHeld * kThreads; i0 < held; i0 += kThreads) sweep(i0 + tid, i0 + tid < held ? keys[i0 + tid] : 0);
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
    switch ((p.dim + 63) / 64) {
      case 1: scores_kernel<1><<<grid, kThreads, 0, stream>>>(p, keys); break;
      case 2: scores_kernel<2><<<grid, kThreads, 0, stream>>>(p, keys); break;
      default: scores_kernel<4><<<grid, kThreads, 0, stream>>>(p, keys);
    }
  }
  top_kernel<<<(unsigned)((int64_t)p.batch * p.draft * p.kv_heads), kThreads, 0, stream>>>(p, keys);
  return hipGetLastError();
}

}  // namespace kh
