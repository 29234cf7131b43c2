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

#include "kh_mx4.hpp"
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

// Append into 4-bit pages: as append_kernel, the 4 lanes of a block agree on its
// largest. The mean is that of the values stored. 12 layers of 16 prompts of 256
// tokens, 8 heads of 128, bf16: 255 MB in 84 us (3 TB/s; 65 and 3.9 at best), bound by
// the rows' loads; 1 or 4 rows ahead (kPair) were no faster than 2.
template <int AT>
__global__ __launch_bounds__(kThreads) void append_mx4_kernel(const kh_cache_append_op a) {
  __shared__ float sums[kThreads][8 + 1];
  const int s = blockIdx.y / a.kv_heads, c = blockIdx.y - s * a.kv_heads, layer = blockIdx.z;
  const int64_t len = a.lengths[s];
  if (len < 0) return;
  const int64_t col = len / a.page_size + blockIdx.x;
  if (col >= a.width || col * a.page_size >= len + a.accept) return;
  const int page = a.table[s * a.table_s + col];
  const int count = counted_rows(a, s);
  const int64_t first = col * a.page_size;
  const int lo = (int)(len > first ? len - first : 0);
  const int hi = (int)min(len + count - first, (int64_t)a.page_size);
  if (lo >= hi || page < 0 || page >= a.pages) return;

  const int chunks = a.dim / 8;                 // threads of a token: whole groups of 4
  const int side = kThreads / chunks;
  const int t = threadIdx.x / chunks, d = (threadIdx.x - t * chunks) * 8;
  float sum[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  if (t < side) {
    uint8_t *kp = static_cast<uint8_t *>(a.k_pages) + (layer * a.kp_l + page * a.kp_p + c * a.kp_h);
    uint8_t *vp = static_cast<uint8_t *>(a.v_pages) + (layer * a.vp_l + page * a.vp_p + c * a.vp_h);
    const int64_t k_at = layer * a.k_l + s * a.k_s + c * a.k_h + d, v_at = layer * a.v_l + s * a.v_s + c * a.v_h + d;
    const int64_t i0 = first - len;
    if (a.k_means) {
      for (int j = t; j < lo; j += kAhead * side) {
        uint32_t code[kAhead], e[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          const int slot = j + i * side < lo ? j + i * side : j;
          code[i] = *reinterpret_cast<const uint32_t *>(kp + mx_key_code(slot, d, a.dim));
          e[i] = kp[mx_key_scale(slot, d, a.dim, a.page_size)];
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          float x[8];
          mx_unpack(code[i], mx_scale(e[i]), x);
#pragma unroll
          for (int q = 0; q < 8; ++q) sum[q] += j + i * side < lo ? x[q] : 0.0f;
        }
      }
    }
    for (int j = lo + t; j < hi; j += kPair * side) {
      float x[kPair][8], y[kPair][8];
#pragma unroll
      for (int i = 0; i < kPair; ++i) {
        int64_t r = i0 + (j + i * side < hi ? j + i * side : j);
        if (a.rows) r = a.rows[s * a.rows_s + r];
        load8(a.k, k_at + r * a.k_n, AT, x[i]);
        load8(a.v, v_at + r * a.v_n, AT, y[i]);
      }
#pragma unroll
      for (int i = 0; i < kPair; ++i) {
        const int slot = j + i * side;
        uint32_t km = mx_most(x[i]), vm = mx_most(y[i]);
        km = quad_max(km);
        vm = quad_max(vm);
        if (slot >= hi) continue;   // (the same for a block's 4 lanes)
        const uint32_t ke = mx_scale_of(km), ve = mx_scale_of(vm), kw = mx_pack(x[i], ke);
        *reinterpret_cast<uint32_t *>(kp + mx_key_code(slot, d, a.dim)) = kw;
        *reinterpret_cast<uint32_t *>(vp + mx_value_code(slot, d, a.dim)) = mx_pack(y[i], ve);
        if (!(d & 31)) {
          kp[mx_key_scale(slot, d, a.dim, a.page_size)] = (uint8_t)ke;
          vp[mx_value_scale(slot, d, a.dim, a.page_size)] = (uint8_t)ve;
        }
        float z[8];
        mx_unpack(kw, mx_scale(ke), z);
#pragma unroll
        for (int q = 0; q < 8; ++q) sum[q] += z[q];
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
// Cached tokens as dense rows: a thread takes 8 dimensions of 4 tokens that lie
// together (slots 4 j .. 4 j + 3), which is what 16 bytes of a 4-bit page's
// values hold, and writes a row's 8 of each. Bound by what it writes: of the same
// prompts about 880 MB, zeros behind the shorter ones among them, in 147 us (6 TB/s).

template <int CT, int OT>
__global__ __launch_bounds__(kThreads) void read_kernel(const kh_cache_read_op a) {
  const int chunks = a.dim / 8;
  const int s = blockIdx.y, layer = blockIdx.z;
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int64_t group = i / (a.kv_heads * chunks);
  const int rest = (int)(i - group * (a.kv_heads * chunks)), c = rest / chunks, d = (rest - c * chunks) * 8;
  const int64_t start = a.starts[s], end = a.ends[s];
  const int64_t p0 = (start & ~(int64_t)3) + 4 * group;       // (start may be negative: rounds down)
  if (p0 >= start + a.tokens) return;
  const int64_t col = p0 >= 0 ? p0 / a.page_size : a.width;
  int page = -1;
  if (p0 < end && col < a.width) page = a.table[s * a.table_s + col];
  const bool in = page >= 0 && page < a.pages;
  const int slot = in ? (int)(p0 - col * a.page_size) : 0;
  const int there = in ? (int)min(end - p0, (int64_t)4) : 0;   // tokens of the four that are there
  float x[4][8], y[4][8];
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) x[j][e] = y[j][e] = 0.0f;
  if (in) {
    if constexpr (CT == KH_TYPE_MX4) {
      const uint8_t *kp = static_cast<const uint8_t *>(a.k_pages) + (layer * a.kp_l + page * a.kp_p + c * a.kp_h);
      const uint8_t *vp = static_cast<const uint8_t *>(a.v_pages) + (layer * a.vp_l + page * a.vp_p + c * a.vp_h);
      const u32x4 vw = *reinterpret_cast<const u32x4 *>(vp + mx_value_code(slot, d, a.dim));
      const uint32_t ve = *reinterpret_cast<const uint32_t *>(vp + mx_value_scale(slot, d, a.dim, a.page_size));
      uint32_t kw[4], ke[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        kw[j] = *reinterpret_cast<const uint32_t *>(kp + mx_key_code(slot + j, d, a.dim));
        ke[j] = kp[mx_key_scale(slot + j, d, a.dim, a.page_size)];
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (j >= there) continue;
        mx_unpack(kw[j], mx_scale(ke[j]), x[j]);
        mx_unpack(vw[j], mx_scale(ve >> (8 * j) & 255u), y[j]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (j >= there) continue;
        load8(a.k_pages, layer * a.kp_l + page * a.kp_p + c * a.kp_h + (slot + j) * a.kp_t + d, CT, x[j]);
        load8(a.v_pages, layer * a.vp_l + page * a.vp_p + c * a.vp_h + (slot + j) * a.vp_t + d, CT, y[j]);
      }
    }
  }
  const int64_t row = (int64_t)a.kv_heads * a.dim;
  const int64_t to = ((int64_t)layer * a.batch + s) * a.tokens * row + c * a.dim + d;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t n = p0 + j - start;
    if (n < 0 || n >= a.tokens) continue;
    store8(a.k, to + n * row, OT, x[j]);
    store8(a.v, to + n * row, OT, y[j]);
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
  if (a.cache_type == KH_TYPE_MX4) {
    switch (a.act_type) {
      case KH_TYPE_F32: append_mx4_kernel<KH_TYPE_F32><<<grid, kThreads, 0, stream>>>(a); break;
      case KH_TYPE_BF16: append_mx4_kernel<KH_TYPE_BF16><<<grid, kThreads, 0, stream>>>(a); break;
      default: append_mx4_kernel<KH_TYPE_F16><<<grid, kThreads, 0, stream>>>(a);
    }
    return hipGetLastError();
  }
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

template <int CT>
static void launch_read_of(const kh_cache_read_op &a, dim3 grid, hipStream_t stream) {
  switch (a.out_type) {
    case KH_TYPE_F32: read_kernel<CT, KH_TYPE_F32><<<grid, kThreads, 0, stream>>>(a); break;
    case KH_TYPE_BF16: read_kernel<CT, KH_TYPE_BF16><<<grid, kThreads, 0, stream>>>(a); break;
    default: read_kernel<CT, KH_TYPE_F16><<<grid, kThreads, 0, stream>>>(a);
  }
}

int64_t read_blocks(const kh_cache_read_op &a) {
  return (((int64_t)a.tokens + 6) / 4 * a.kv_heads * (a.dim / 8) + kThreads - 1) / kThreads;
}

hipError_t launch_read(const kh_cache_read_op &a, hipStream_t stream) {
  if (!a.layers || !a.batch || !a.tokens) return hipSuccess;
  const dim3 grid((unsigned)read_blocks(a), (unsigned)a.batch, (unsigned)a.layers);
  switch (a.cache_type) {
    case KH_TYPE_F32: launch_read_of<KH_TYPE_F32>(a, grid, stream); break;
    case KH_TYPE_BF16: launch_read_of<KH_TYPE_BF16>(a, grid, stream); break;
    case KH_TYPE_F16: launch_read_of<KH_TYPE_F16>(a, grid, stream); break;
    default: launch_read_of<KH_TYPE_MX4>(a, grid, stream);
  }
  return hipGetLastError();
}

// Element (page's head at `at`, slot t, dimension d) of pages of any type.
static float host_page_value(const void *pages, int64_t at, int64_t row, int t, int d, int dim, int page_size, int type, bool keys) {
  if (type != KH_TYPE_MX4) return host_value(pages, at + t * row + d, type);
  const uint8_t *p = static_cast<const uint8_t *>(pages) + at;
  const uint32_t code = p[keys ? mx_key_code(t, d, dim) : mx_value_code(t, d, dim)] >> (4 * (d & 1)) & 15u;
  return mx_value(code, p[keys ? mx_key_scale(t, d, dim, page_size) : mx_value_scale(t, d, dim, page_size)]);
}

void host_read(const kh_cache_read_op &a) {
  int64_t to = 0;
  for (int layer = 0; layer < a.layers; ++layer)
    for (int s = 0; s < a.batch; ++s)
      for (int64_t n = 0; n < a.tokens; ++n)
        for (int c = 0; c < a.kv_heads; ++c)
          for (int d = 0; d < a.dim; ++d, ++to) {
            const int64_t pos = a.starts[s] + n, col = pos < 0 ? a.width : pos / a.page_size;
            const int page = pos < a.ends[s] && col < a.width ? a.table[s * a.table_s + col] : -1;
            float x = 0.0f, y = 0.0f;
            if (page >= 0 && page < a.pages) {
              const int t = (int)(pos - col * a.page_size);
              x = host_page_value(a.k_pages, layer * a.kp_l + page * a.kp_p + c * a.kp_h, a.kp_t, t, d, a.dim, a.page_size, a.cache_type, true);
              y = host_page_value(a.v_pages, layer * a.vp_l + page * a.vp_p + c * a.vp_h, a.vp_t, t, d, a.dim, a.page_size, a.cache_type, false);
            }
            host_store(a.k, to, a.out_type, x);
            host_store(a.v, to, a.out_type, y);
          }
}

// A token's row of a head into a 4-bit page.
static void host_store_mx4(void *pages, int64_t at, int t, int dim, int page_size, bool keys, const float *x) {
  uint8_t *p = static_cast<uint8_t *>(pages) + at;
  for (int b = 0; b < dim; b += kMxBlock) {
    uint32_t most = 0;
    for (int d = b; d < b + kMxBlock; ++d) most = std::max(most, mx_bits(x[d]) & 0x7fffffffu);
    const uint32_t e = mx_scale_of(most);
    p[keys ? mx_key_scale(t, b, dim, page_size) : mx_value_scale(t, b, dim, page_size)] = (uint8_t)e;
    for (int d = b; d < b + kMxBlock; ++d) {
      uint8_t &byte = p[keys ? mx_key_code(t, d, dim) : mx_value_code(t, d, dim)];
      const uint32_t code = mx_code(x[d], e);
      byte = (uint8_t)(d & 1 ? (byte & 0x0f) | code << 4 : (byte & 0xf0) | code);
    }
  }
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
          if (a.cache_type == KH_TYPE_MX4) {
            std::vector<float> row((size_t)a.dim);
            for (int64_t pos = std::max(len, start); pos < hi; ++pos) {
              const int64_t r = a.rows ? a.rows[s * a.rows_s + pos - len] : pos - len;
              for (int d = 0; d < a.dim; ++d) row[(size_t)d] = host_value(a.k, layer * a.k_l + s * a.k_s + r * a.k_n + c * a.k_h + d, a.act_type);
              host_store_mx4(a.k_pages, kp, (int)(pos - start), a.dim, a.page_size, true, row.data());
              for (int d = 0; d < a.dim; ++d) row[(size_t)d] = host_value(a.v, layer * a.v_l + s * a.v_s + r * a.v_n + c * a.v_h + d, a.act_type);
              host_store_mx4(a.v_pages, vp, (int)(pos - start), a.dim, a.page_size, false, row.data());
            }
          }
          for (int d = 0; d < a.dim; ++d) {
            double sum = 0.0;
            for (int64_t pos = start; pos < hi; ++pos) {
              if (pos >= len && a.cache_type != KH_TYPE_MX4) {
                const int64_t r = a.rows ? a.rows[s * a.rows_s + pos - len] : pos - len;
                host_store(a.k_pages, kp + (pos - start) * a.kp_t + d, a.cache_type,
                           host_value(a.k, layer * a.k_l + s * a.k_s + r * a.k_n + c * a.k_h + d, a.act_type));
                host_store(a.v_pages, vp + (pos - start) * a.vp_t + d, a.cache_type,
                           host_value(a.v, layer * a.v_l + s * a.v_s + r * a.v_n + c * a.v_h + d, a.act_type));
              }
              sum += host_page_value(a.k_pages, kp, a.kp_t, (int)(pos - start), d, a.dim, a.page_size, a.cache_type, true);
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
