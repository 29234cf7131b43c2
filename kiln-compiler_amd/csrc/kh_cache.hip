// kh_cache.hip - what moves a paged cache's tokens: appending new ones
// (kh_cache_append) and copying pages (kh_cache_copy).
//
// append: a workgroup per (layer, sequence, kv head, page that may be written
// to). Its threads take 8 adjacent dimensions of a token each; the mean of the
// page's keys is summed in fp32 over the same threads' tokens (the ones the
// page held before are read, the new ones are at hand), then over the threads
// in order, so it depends on nothing but the page's contents.
// Measured: 12 layers x 64 sequences x 8 heads of 128, up to 23 tokens each,
// 45.8 us (2.7 TB/s; one token at a time per thread, types told apart in the
// loop, took 67): short chains of dependent loads in 6000 workgroups.
// copy: the page numbers travel in the kernel's arguments (256 pairs a
// launch), so that a call needs no upload that a later one could overtake. 301
// pages of 128 KB, K and V in 12 layers (1.9 GB both ways) take 345 us, 5.5 TB/s,
// where a 2 GiB device copy moves 4.9.
#include <algorithm>
#include <cstring>
#include <vector>

#include "kh_paged.hpp"

namespace kh {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int kThreads = 256;

__device__ __forceinline__ void load8(const void *p, int64_t i, int type, float (&x)[8]) {
  if (type == KH_TYPE_F32) {
#pragma unroll
    for (int j = 0; j < 8; j += 4) {
      const f32x4 a = *reinterpret_cast<const f32x4 *>(static_cast<const float *>(p) + i + j);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[j + e] = a[e];
    }
    return;
  }
  const u32x4 a = *reinterpret_cast<const u32x4 *>(static_cast<const uint16_t *>(p) + i);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t half = a[e / 2] >> (16 * (e & 1)) & 0xffffu;
    x[e] = type == KH_TYPE_BF16 ? __uint_as_float(half << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)half);
  }
}

// x stored at element i of p in `type`; x becomes the values that were stored
__device__ __forceinline__ void store8(void *p, int64_t i, int type, float (&x)[8]) {
  if (type == KH_TYPE_F32) {
#pragma unroll
    for (int j = 0; j < 8; j += 4)
      *reinterpret_cast<f32x4 *>(static_cast<float *>(p) + i + j) = f32x4{x[j], x[j + 1], x[j + 2], x[j + 3]};
  } else if (type == KH_TYPE_BF16) {
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    v8 y;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      y[e] = (__bf16)x[e];
      x[e] = (float)y[e];
    }
    *reinterpret_cast<v8 *>(static_cast<__bf16 *>(p) + i) = y;
  } else {
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    v8 y;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      y[e] = (_Float16)x[e];
      x[e] = (float)y[e];
    }
    *reinterpret_cast<v8 *>(static_cast<_Float16 *>(p) + i) = y;
  }
}

// How many rows of sequence s count: those before the first outside [0, draft).
__device__ __forceinline__ int counted_rows(const kh_cache_append_op &a, int s) {
  if (!a.rows) return a.accept;
  for (int i = 0; i < a.accept; i += 64) {
    const int lane = threadIdx.x & 63;
    const int r = i + lane < a.accept ? a.rows[s * a.rows_s + i + lane] : -1;
    const uint64_t bad = __ballot(r < 0 || r >= a.draft);
    if (bad) return i + __builtin_ctzll(bad);
  }
  return a.accept;
}

constexpr int kAhead = 4;   // tokens of a thread whose loads are in flight together: of those that are there
constexpr int kPair = 2;    // ... and of the new ones, k and v of each

// CT, AT: element types of the cache and of the new tokens.
template <int CT, int AT>
__global__ __launch_bounds__(kThreads) void append_kernel(const kh_cache_append_op a) {
  __shared__ float sums[kThreads][8 + 1];
  const int s = blockIdx.y / a.kv_heads, c = blockIdx.y - s * a.kv_heads, layer = blockIdx.z;
  const int64_t len = a.lengths[s];
  if (len < 0) return;
  const int64_t col = len / a.page_size + blockIdx.x;
  if (col >= a.width || col * a.page_size >= len + a.accept) return;   // (before rows are counted)
  const int page = a.table[s * a.table_s + col];
  const int count = counted_rows(a, s);
  const int64_t first = col * a.page_size;
  // the page's slots [lo, hi) are written, those before lo are there
  const int lo = (int)(len > first ? len - first : 0);
  const int hi = (int)min(len + count - first, (int64_t)a.page_size);
  if (lo >= hi || page < 0 || page >= a.pages) return;

  const int chunks = a.dim / 8;                 // threads of a token
  const int side = kThreads / chunks;           // tokens at a time
  const int t = threadIdx.x / chunks, d = (threadIdx.x - t * chunks) * 8;
  float sum[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  if (t < side) {
    const int64_t kp_at = layer * a.kp_l + page * a.kp_p + c * a.kp_h + d;
    const int64_t vp_at = layer * a.vp_l + page * a.vp_p + c * a.vp_h + d;
    const int64_t k_at = layer * a.k_l + s * a.k_s + c * a.k_h + d, v_at = layer * a.v_l + s * a.v_s + c * a.v_h + d;
    const int64_t i0 = first - len;              // slot j gets row i0 + j
    if (a.k_means) {
      for (int j = t; j < lo; j += kAhead * side) {
        float x[kAhead][8];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
#pragma unroll
          for (int e = 0; e < 8; ++e) x[i][e] = 0.0f;
          if (j + i * side < lo) load8(a.k_pages, kp_at + (j + i * side) * a.kp_t, CT, x[i]);
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
#pragma unroll
          for (int e = 0; e < 8; ++e) sum[e] += x[i][e];
      }
    }
    for (int j = lo + t; j < hi; j += kPair * side) {
      float x[kPair][8], y[kPair][8];
#pragma unroll
      for (int i = 0; i < kPair; ++i) {
        if (j + i * side >= hi) continue;
        int64_t r = i0 + j + i * side;
        if (a.rows) r = a.rows[s * a.rows_s + r];
        load8(a.k, k_at + r * a.k_n, AT, x[i]);
        load8(a.v, v_at + r * a.v_n, AT, y[i]);
      }
#pragma unroll
      for (int i = 0; i < kPair; ++i) {
        const int slot = j + i * side;
        if (slot >= hi) continue;
        store8(a.k_pages, kp_at + slot * a.kp_t, CT, x[i]);
        store8(a.v_pages, vp_at + slot * a.vp_t, CT, y[i]);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] += x[i][e];
      }
    }
  }
  if (!a.k_means) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) sums[threadIdx.x][e] = sum[e];
  __syncthreads();
  for (int i = threadIdx.x; i < a.dim; i += kThreads) {
    float total = 0.0f;
    for (int j = 0; j < side; ++j) total += sums[j * chunks + i / 8][i & 7];
    a.k_means[layer * a.m_l + page * a.m_p + c * a.m_h + i] = total / (float)hi;
  }
}

// ---------------------------------------------------------------------------

constexpr int kPairs = 256;    // pages of a launch
constexpr int kChunk = 16384;  // bytes of a page that a workgroup copies

struct CopyArgs {
  kh_pool pool[KH_MAX_POOLS];
  int n_pools;
  int32_t source[kPairs], target[kPairs];
};

template <class T>
__global__ __launch_bounds__(kThreads) void copy_kernel(const CopyArgs a) {
  int i = 0;
  int64_t layer = blockIdx.z;
  while (layer >= a.pool[i].layers) layer -= a.pool[i++].layers;   // (the grid has one z per layer of a pool)
  const kh_pool &pool = a.pool[i];
  const int64_t at = (int64_t)blockIdx.x * kChunk;
  if (at >= pool.page_bytes) return;
  const int64_t n = min((int64_t)kChunk, pool.page_bytes - at) / (int64_t)sizeof(T);
  char *base = static_cast<char *>(pool.base) + layer * pool.layer_bytes + at;
  const T *from = reinterpret_cast<const T *>(base + a.source[blockIdx.y] * pool.page_bytes);
  T *to = reinterpret_cast<T *>(base + a.target[blockIdx.y] * pool.page_bytes);
  // (the whole chunk in flight; each byte is read and written once: past the caches)
  T x[kChunk / kThreads / sizeof(T)];
#pragma unroll
  for (int i = 0; i < (int)(kChunk / kThreads / sizeof(T)); ++i) {
    const int64_t j = (int64_t)i * kThreads + threadIdx.x;
    if (j < n) x[i] = __builtin_nontemporal_load(from + j);
  }
#pragma unroll
  for (int i = 0; i < (int)(kChunk / kThreads / sizeof(T)); ++i) {
    const int64_t j = (int64_t)i * kThreads + threadIdx.x;
    if (j < n) __builtin_nontemporal_store(x[i], to + j);
  }
}

// -- CPU meaning ----------------------------------------------------------------

float host_value(const void *p, int64_t i, int type) {
  if (type == KH_TYPE_F32) return static_cast<const float *>(p)[i];
  if (type == KH_TYPE_BF16) return (float)static_cast<const __bf16 *>(p)[i];
  return (float)static_cast<const _Float16 *>(p)[i];
}
float host_store(void *p, int64_t i, int type, float x) {
  if (type == KH_TYPE_F32) return static_cast<float *>(p)[i] = x;
  if (type == KH_TYPE_BF16) return (float)(static_cast<__bf16 *>(p)[i] = (__bf16)x);
  return (float)(static_cast<_Float16 *>(p)[i] = (_Float16)x);
}

}  // namespace

hipError_t launch_append(const kh_cache_append_op &a, hipStream_t stream) {
  if (!a.layers || !a.batch || !a.accept) return hipSuccess;
  const unsigned pages = (unsigned)((a.accept - 1) / a.page_size + 2);
  const dim3 grid(pages, (unsigned)a.batch * a.kv_heads, (unsigned)a.layers);
  switch (3 * a.cache_type + a.act_type) {
    case 0: append_kernel<0, 0><<<grid, kThreads, 0, stream>>>(a); break;
    case 1: append_kernel<0, 1><<<grid, kThreads, 0, stream>>>(a); break;
    case 2: append_kernel<0, 2><<<grid, kThreads, 0, stream>>>(a); break;
    case 3: append_kernel<1, 0><<<grid, kThreads, 0, stream>>>(a); break;
    case 4: append_kernel<1, 1><<<grid, kThreads, 0, stream>>>(a); break;
    case 5: append_kernel<1, 2><<<grid, kThreads, 0, stream>>>(a); break;
    case 6: append_kernel<2, 0><<<grid, kThreads, 0, stream>>>(a); break;
    case 7: append_kernel<2, 1><<<grid, kThreads, 0, stream>>>(a); break;
    default: append_kernel<2, 2><<<grid, kThreads, 0, stream>>>(a);
  }
  return hipGetLastError();
}

void host_append(const kh_cache_append_op &a) {
  for (int layer = 0; layer < a.layers; ++layer)
    for (int s = 0; s < a.batch; ++s) {
      const int64_t len = a.lengths[s];
      if (len < 0) continue;
      int count = 0;
      while (count < a.accept && (!a.rows || (a.rows[s * a.rows_s + count] >= 0 && a.rows[s * a.rows_s + count] < a.draft)))
        ++count;
      for (int64_t col = len / a.page_size; col < a.width && col * a.page_size < len + count; ++col) {
        const int page = a.table[s * a.table_s + col];
        if (page < 0 || page >= a.pages) continue;
        const int64_t start = col * a.page_size, hi = std::min<int64_t>(len + count, start + a.page_size);
        if (std::max(len, start) >= hi) continue;   // nothing is written to it
        for (int c = 0; c < a.kv_heads; ++c) {
          const int64_t kp = layer * a.kp_l + page * a.kp_p + c * a.kp_h, vp = layer * a.vp_l + page * a.vp_p + c * a.vp_h;
          for (int d = 0; d < a.dim; ++d) {
            double sum = 0.0;
            for (int64_t pos = start; pos < hi; ++pos) {
              if (pos >= len) {
                const int64_t r = a.rows ? a.rows[s * a.rows_s + pos - len] : pos - len;
                host_store(a.k_pages, kp + (pos - start) * a.kp_t + d, a.cache_type,
                           host_value(a.k, layer * a.k_l + s * a.k_s + r * a.k_n + c * a.k_h + d, a.act_type));
                host_store(a.v_pages, vp + (pos - start) * a.vp_t + d, a.cache_type,
                           host_value(a.v, layer * a.v_l + s * a.v_s + r * a.v_n + c * a.v_h + d, a.act_type));
              }
              sum += host_value(a.k_pages, kp + (pos - start) * a.kp_t + d, a.cache_type);
            }
            if (a.k_means) a.k_means[layer * a.m_l + page * a.m_p + c * a.m_h + d] = (float)(sum / (double)(hi - start));
          }
        }
      }
    }
}

hipError_t launch_copy(const kh_pool *pools, int n_pools, const int32_t *source, const int32_t *target, int n,
                       hipStream_t stream) {
  CopyArgs a;
  a.n_pools = n_pools;
  int64_t layers = 0, most = 0;
  bool wide = true;
  for (int i = 0; i < n_pools; ++i) {
    a.pool[i] = pools[i];
    layers += pools[i].layers;
    if (pools[i].layers) most = std::max(most, pools[i].page_bytes);
    wide = wide && pools[i].page_bytes % 16 == 0 && pools[i].layer_bytes % 16 == 0 && (uintptr_t)pools[i].base % 16 == 0;
  }
  if (!layers || !most) return hipSuccess;
  for (int done = 0; done < n; done += kPairs) {
    const int part = std::min(kPairs, n - done);
    std::memcpy(a.source, source + done, part * sizeof(int32_t));
    std::memcpy(a.target, target + done, part * sizeof(int32_t));
    const dim3 grid((unsigned)((most + kChunk - 1) / kChunk), (unsigned)part, (unsigned)layers);
    if (wide) copy_kernel<u32x4><<<grid, kThreads, 0, stream>>>(a);
    else copy_kernel<uint32_t><<<grid, kThreads, 0, stream>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace kh
