// kh_paged_attn.hpp - attention of drafted tokens over a paged cache (kh_paged).
//
// One item is (sequence, kv head, up to 16 RT query rows: all (token, head of
// the group) pairs, or with picked pages one token's heads). Its keys are cut
// into tiles of 32: the cached ones (two half tiles of 16, each within one
// page, since a page holds a multiple of 16), then the new ones. All items'
// tiles in a row are dealt to the workgroups in equal ranges, so a batch of
// ragged lengths loads every workgroup alike and one long sequence fills the
// chip; the four waves of a workgroup take a range's tiles in turn. A range
// that ends inside an item leaves (m, l, O) in the workspace, which a second
// kernel joins; an item within one range is finished here. Where no item can
// have many tiles, a workgroup takes a whole item instead and one kernel is
// enough.
//
// A wave holds its tile in registers: scores S^T = K Q^T, so that a lane has
// its query's scores (lane li = lane & 15) for keys 4 g + r (g = lane >> 4),
// which is how O^T += V^T P^T takes the weights back without a move; V^T's
// operand needs 8 keys of one dimension per lane, which a lane makes from 8
// rows' 16-byte pieces by 32 byte permutes. One pass over the keys with
// running maximum and sum (base 2, fp32). The next tile's K is loaded once
// this one's scores are made, its V once this one's weights are used, into the
// same registers: one to two tiles are in flight per wave without any for
// themselves, and the page numbers come by scalar loads, which do not queue
// behind them.
//
// fp32 activations over a 16-bit cache keep fp32's accuracy: a bf16 product's
// three parts x = x1 + x2 + x3 of 8 bits each hold all 24 bits of q and of a
// weight, and K and V are exact, so three passes lose nothing; fp16 parts
// hold 11 bits each, two passes are off by 2^-21, with q scaled by a power of
// two per row and the weights by 2^14 to stay clear of fp16's subnormals. Under
// 16-bit activations q is exact as it is and the weights are two parts: 16 bits
// of bf16 and 22 of fp16, so that nothing rounds by as much as the result's own
// 8 or 11 do. NQ and NW: parts of q and of the weights; one and one rounds
// both to the cache's type (a plan whose products are bf16 asks for that). The
// parts of a number all have its sign and none is 0 alone, so that an infinite
// key or value gives what it gives in one product (split8).
//
// What bounds it, measured (one MI355X; a 2 GiB copy moves 4.9 TB/s, reads and
// writes together): long caches the reading of K and V - 131072 bf16 tokens of
// 8 heads of 128, one fp32 query of 32 heads, 104 us (5.2 TB/s) and 7 us for
// the join; 32 sequences of 0 to 8192 tokens 122 us (4.7 TB/s) and 7; 48 pages
// of 128 tokens picked for each of 13 tokens 102 us (653 MB, 6.4 TB/s: tokens
// share pages). Short ones latency: a launch, the length, the first loads and
// one tile are 7 us, each further tile of a wave 1.5 us (a K load's latency and
// the products behind it), which is why a whole item takes eight waves: 27-token
// trees over 1024 tokens, 12 heads of 64, 30.6 us with four, 23.8 with eight.
// Tiles of 64 keys for 64-wide heads, and page numbers staged in the LDS, were
// both slower (32.7 us there; 137 for the 32 sequences): the first tile waits
// longer, and nothing that comes after was waiting for them.
//
// A window leaves tiles out and masks those on its edge row by row: 32 sequences
// of up to 120000 bf16 tokens, a window of 4096 and 4 sinks, 102 us (536 MB, 5.3
// TB/s) and 7 for the join, as much as caches of 4096 tokens take.
#pragma once

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "kh_mx4.hpp"
#include "kh_paged.hpp"

namespace kh {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kTile = kPagedTile;
constexpr int kThreads = 256;
constexpr int kWaves = kPagedWaves;
constexpr float kWeightExp = 14.0f;   // fp16 weights are 2^14 softmax weights

// ---------------------------------------------------------------------------
// The tiles of all items in a row.

struct Plan {   // ranges: the first `extra` of `each` + 1 tiles, the others of `each`
  int count, each, extra;
};

// int32 operands through the constant address space: a wave-uniform index
// then becomes a scalar load (the kernels write none of them).
typedef const __attribute__((address_space(4))) int32_t *const_ints;
__device__ __forceinline__ const_ints ints_of(const int32_t *p) { return (const_ints)(uintptr_t)p; }

template <class W>
__device__ __forceinline__ int clamp_len(W &w, int s) {
  const int n = ints_of(w.p.lengths)[s];
  const int64_t most = (int64_t)w.p.width * w.p.page_size;
  return n < 0 ? 0 : (n > most ? (int)most : n);
}

// The tiles of the cached tokens that count: all of them, or under a window
// those of the first `sinks` tokens and those from the first key that the
// shallowest new token sees; tile t is tile t of the sequence below `head`, t +
// skip from there on.
// (WIN: whether there may be a window; kernels are built with and without, as
// its few scalars would not fit beside the others.)
struct Span {
  int tiles, head, skip;
};

template <bool WIN, class W>
__device__ __forceinline__ Span span_of(W &w, int len) {
  const int all = (len + w.tile - 1) / w.tile;
  Span r = {all, all, 0};
  if (WIN && w.p.window) {
    const int from = max(len - w.p.window + 1, 0) / w.tile;
    r.head = (min(w.p.sinks, len) + w.tile - 1) / w.tile;
    r.skip = max(from - r.head, 0);
    r.tiles = all - r.skip;
  }
  return r;
}

// Do new tokens differ in which keys they see of the 32 (64) from `pos` on, or
// see none of some? (A new token's window starts at len + depth - window + 1.)
template <bool WIN, class W>
__device__ __forceinline__ bool on_edge(W &w, int len, int pos, int keys) {
  return WIN && w.p.window && pos + keys > w.p.sinks && pos <= len - w.p.window + w.p.draft - 1;
}

// Bits of the 32 keys from `pos` on that lie in the window or are sinks: `first`
// is the window's first key.
__device__ __forceinline__ uint32_t window_bits(int first, int sinks, int pos) {
  const int lo = first - pos, hi = sinks - pos;
  const uint32_t in = lo <= 0 ? ~0u : lo >= 32 ? 0u : ~0u << lo;
  return in | (hi <= 0 ? 0u : hi >= 32 ? ~0u : (1u << hi) - 1);
}

template <bool WIN, class W>
__device__ __forceinline__ int tiles_of(W &w, int len) {
  return (w.sel_tiles ? w.sel_tiles : span_of<WIN>(w, len).tiles) + w.draft_tiles;
}

// first[s] = tiles of one item of the sequences before s, for s <= batch; LEAD: tiles
// that an item counts for besides its own, in front of them (what beginning one costs).
template <bool WIN, int LEAD, class W>
__device__ __forceinline__ void scan_tiles(W &w, int *first, int *wave_sums) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n = w.p.batch;
  const int per = (n + kThreads - 1) / kThreads;
  const int lo = threadIdx.x * per;
  int sum = 0;
  for (int i = lo; i < min(lo + per, n); ++i) sum += tiles_of<WIN>(w, clamp_len(w, i)) + LEAD;
  int run = sum;   // inclusive over the wave
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int o = __shfl_up(run, d);
    if (lane >= d) run += o;
  }
  if (lane == 63) wave_sums[wave] = run;
  __syncthreads();
  int at = run - sum;
  for (int i = 0; i < wave; ++i) at += wave_sums[i];
  for (int i = lo; i < min(lo + per, n); ++i) {
    first[i] = at;
    at += tiles_of<WIN>(w, clamp_len(w, i)) + LEAD;
  }
  if (lo < n && lo + per >= n) first[n] = at;
  __syncthreads();
}

template <int LEAD, class W>
__device__ __forceinline__ Plan plan_of(W &w, const int *first) {
  Plan r;
  const uint32_t total = (uint32_t)__builtin_amdgcn_readfirstlane(first[w.p.batch]) * (uint32_t)w.items;
  // a tile per wave at least, or as many tiles as a beginning counts for
  const uint32_t least = LEAD ? 2 * LEAD : kWaves;
  const uint32_t want = (total + least - 1) / least;
  r.count = (int)min(want, (uint32_t)w.grid);
  r.each = (int)(total / (uint32_t)r.count);
  r.extra = (int)(total - (uint32_t)r.each * r.count);
  return r;
}

__device__ __forceinline__ int range_start(const Plan &r, int w) { return r.each * w + min(w, r.extra); }

// The range that holds tile x.
__device__ __forceinline__ int range_of(const Plan &r, int x) {
  const int longer = r.extra * (r.each + 1);
  return x < longer ? (int)((uint32_t)x / (uint32_t)(r.each + 1)) : r.extra + (int)((uint32_t)(x - longer) / (uint32_t)r.each);
}

// Which sequence tile x of the row lies in (first[] counts one item's tiles).
template <class W>
__device__ __forceinline__ int sequence_of(W &w, const int *first, int x) {
  int lo = 0, hi = w.p.batch - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (first[mid] * w.items <= x) lo = mid;
    else hi = mid - 1;
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

// ---------------------------------------------------------------------------

// Which rows of the drafted tokens' paths see which of them: bit j of row i.
// Also the unused tokens. Doubling: after k rounds a row holds its nearest
// 2^k ancestors.
struct Paths {
  uint32_t bits[kMaxDraft][kMaxDraft / 32];
  int16_t next[kMaxDraft];   // the next ancestor beyond those held; -1 none, -2 the token is unused
  int16_t depth[kMaxDraft];  // ancestors of the token (under a window)
};

template <bool WIN, class W>
__device__ __forceinline__ void build_paths(W &w, int s, int len, Paths &t) {
  const int i = threadIdx.x, n = w.p.draft;
  const int32_t *parents = w.p.parents + s * w.p.parents_s;
  const int words = (n + 31) / 32;
  if (i < n) {
    const int p = parents[i];
    t.next[i] = p >= -1 && p < i ? p : -2;
    for (int k = 0; k < words; ++k) t.bits[i][k] = k == i / 32 ? 1u << (i & 31) : 0u;
  }
  __syncthreads();
  for (int round = 0; round < w.rounds; ++round) {
    uint32_t got[kMaxDraft / 32];
    int next = -1;
    if (i < n) {
      next = t.next[i];
      const int from = next < 0 ? i : next;
#pragma unroll
      for (int k = 0; k < kMaxDraft / 32; ++k)
        if (k < words) got[k] = t.bits[i][k] | t.bits[from][k];
      if (next >= 0) next = t.next[next];
    }
    __syncthreads();
    if (i < n) {
#pragma unroll
      for (int k = 0; k < kMaxDraft / 32; ++k)
        if (k < words) t.bits[i][k] = got[k];
      t.next[i] = (int16_t)next;
    }
    __syncthreads();
  }
  if (WIN && w.p.window) {
    if (i < n) {
      int depth = -1;
      for (int k = 0; k < words; ++k) depth += __builtin_popcount(t.bits[i][k]);
      t.depth[i] = (int16_t)depth;
      if (w.p.window < n) {   // ancestors out of the window: the path is walked again
        for (int k = 0; k < words; ++k) t.bits[i][k] = 0u;
        int j = i;
        for (int back = 0; back <= depth; ++back) {
          if (back < w.p.window || len + depth - back < w.p.sinks) t.bits[i][j / 32] |= 1u << (j & 31);
          j = max(parents[j], 0);
        }
      }
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------

template <int CT>
struct Cache;   // element type of the cache
template <>
struct Cache<KH_TYPE_F32> {
  typedef float T;
};
template <>
struct Cache<KH_TYPE_BF16> {
  typedef __bf16 T;
  typedef bf16x8 V8;
  __device__ static f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};
template <>
struct Cache<KH_TYPE_F16> {
  typedef _Float16 T;
  typedef f16x8 V8;
  __device__ static f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};

// 4-bit pages: values are bf16 ones (kh_mx4.hpp), the products bf16's
template <>
struct Cache<KH_TYPE_MX4> : Cache<KH_TYPE_BF16> {};

// n (4 or 8) adjacent activations from element i, fp32 or T, 16-byte (8-byte) aligned
template <class T, int N>
__device__ __forceinline__ void load_acts(const void *p, int64_t i, bool fp32, float (&x)[N]) {
  if (sizeof(T) == 4 || fp32) {
#pragma unroll
    for (int j = 0; j < N; j += 4) {
      const f32x4 a = *reinterpret_cast<const f32x4 *>(static_cast<const float *>(p) + i + j);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[j + e] = a[e];
    }
  } else {
    typedef T vec __attribute__((ext_vector_type(N)));
    const vec a = *reinterpret_cast<const vec *>(static_cast<const T *>(p) + i);
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = (float)a[j];
  }
}

template <class T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  typedef T pair __attribute__((ext_vector_type(2)));
  const pair v = {(T)a, (T)b};
  return __builtin_bit_cast(uint32_t, v);
}

// x's leading bits as a T, toward zero, as a float
template <class T>
__device__ __forceinline__ float leading(float x) {
  if constexpr (std::is_same<T, __bf16>::value) return __uint_as_float(__float_as_uint(x) & 0xffff0000u);
  else return (float)__builtin_amdgcn_cvt_pkrtz(x, x)[0];
}

// x as NP parts of type T: the leading bits of x, those of what is left, and
// last the nearest to that. No part has the other sign, and none is 0 under an
// x that T can tell from 0 (the smallest normal of bf16 or the smallest
// subnormal of fp16 stands in): an infinite key or value then meets no part
// that makes a NaN of it (0 inf, inf - inf), as it would not meet x.
// One part is the nearest to x. SIGNED: x may be negative.
template <class T, int NP, bool SIGNED>
__device__ __forceinline__ void split8(const float (&x)[8], u32x4 (&out)[NP]) {
  if constexpr (NP == 1) {
#pragma unroll
    for (int m = 0; m < 4; ++m) out[0][m] = pack2<T>(x[2 * m], x[2 * m + 1]);
    return;
  }
  constexpr float kLeast = std::is_same<T, __bf16>::value ? 0x1p-126f : 0x1p-24f;
  float rest[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) rest[j] = SIGNED ? fabsf(x[j]) : x[j];
#pragma unroll
  for (int part = 0; part < NP; ++part) {
    if (part + 1 < NP) {
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        const float a = rest[2 * m], b = rest[2 * m + 1];
        if constexpr (std::is_same<T, __bf16>::value)
          out[part][m] = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
        else
          out[part][m] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a, b));
      }
      // (the median: not below kLeast, nor above x where x is)
#pragma unroll
      for (int j = 0; j < 8; ++j) rest[j] = __builtin_amdgcn_fmed3f(rest[j] - leading<T>(rest[j]), kLeast, rest[j]);
    } else {
#pragma unroll
      for (int m = 0; m < 4; ++m) out[part][m] = pack2<T>(rest[2 * m], rest[2 * m + 1]);
    }
    if constexpr (SIGNED) {
#pragma unroll
      for (int m = 0; m < 4; ++m)
        out[part][m] |= __float_as_uint(x[2 * m]) >> 31 << 15 | (__float_as_uint(x[2 * m + 1]) & 0x80000000u);
    }
  }
}

// x (not negative) as parts that meet no infinite value: as split8, without what
// that needs.
template <class T, int NP>
__device__ __forceinline__ void split_finite(const float (&x)[8], u32x4 (&out)[NP]) {
  float rest[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) rest[j] = x[j];
#pragma unroll
  for (int part = 0; part < NP; ++part) {
#pragma unroll
    for (int m = 0; m < 4; ++m)
      out[part][m] = part + 1 < NP ? __builtin_amdgcn_perm(__float_as_uint(rest[2 * m + 1]), __float_as_uint(rest[2 * m]), 0x07060302u)
                                   : pack2<T>(rest[2 * m], rest[2 * m + 1]);
#pragma unroll
    for (int j = 0; j < 8; ++j) rest[j] -= leading<T>(rest[j]);
  }
}

__device__ __forceinline__ float max16x32(float v) {   // over the four lane groups of a query
  float2 p = row_pair(v);
  v = fmaxf(p.x, p.y);
  p = half_pair(v);
  return fmaxf(p.x, p.y);
}
__device__ __forceinline__ float sum16x32(float v) {
  float2 p = row_pair(v);
  v = p.x + p.y;
  p = half_pair(v);
  return p.x + p.y;
}

// One tile's keys and values in a lane's registers. K: lane (li, g) holds of
// key 16 h + li the dimensions 32 ks + 8 g .. + 8; V: of key 16 (j >> 2) + 4 g
// + (j & 3) the dimensions VD li .. + VD of every 16 VD.
template <int CT, int DT>
struct Tile {
  static constexpr int KS = DT / 32;
  static constexpr int KW = CT == KH_TYPE_F32 ? 8 : 4;         // words of 8 elements
  static constexpr int VD = DT >= 128 ? 8 : 4;                 // adjacent dimensions of a lane
  static constexpr int VC = DT / (16 * VD);                    // chunks of 16 VD dimensions
  static constexpr int VW = CT == KH_TYPE_F32 ? VD : VD / 2;   // words of VD elements
  uint32_t k[2][KS][KW];
  uint32_t v[8][VC][VW];
};

template <int N>
__device__ __forceinline__ void load_words(const void *p, uint32_t (&x)[N]) {
  if constexpr (N == 2) {
    const u32x2 a = *static_cast<const u32x2 *>(p);
    x[0] = a[0];
    x[1] = a[1];
  } else {
#pragma unroll
    for (int j = 0; j < N; j += 4) {
      const u32x4 a = static_cast<const u32x4 *>(p)[j / 4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[j + e] = a[e];
    }
  }
}

// Where a tile's halves lie (uniform over the wave): rows of `valid` keys each.
template <class T>
struct Source {
  const T *k[2], *v[2];
  int k_row, v_row;    // elements from a key to the next
  int valid[2];
  int draft;           // index among the new tokens' tiles, -1 for a cached one
  int pos;             // a cached tile's first key
  bool edge;           // not every row sees the same of its keys
};

// The kernel's arguments are read where they are used, through a pointer that
// fresh() makes opaque: hoisted to the start they would fill the scalar
// registers and spill.
typedef const __attribute__((address_space(4))) PagedWork const_work;
__device__ __forceinline__ const_work &fresh() {
  uint64_t args = (uint64_t)(uintptr_t)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(args));
  return *(const_work *)(uintptr_t)args;
}

// WHOLE: a workgroup per item, of eight waves where the registers allow two on
// a SIMD (one alone waits about 1.5 us a tile for its loads); else ranges.
template <int CT, int NQ, int NW, int DT, int RT, bool WHOLE, bool WIN>
__global__ __launch_bounds__(64 * paged_waves(DT, RT, WHOLE), RT * DT > 128 ? 1 : 2) void paged_attn_kernel(const PagedWork) {
  constexpr int WAVES = paged_waves(DT, RT, WHOLE);
  typedef typename Cache<CT>::T T;
  typedef Tile<CT, DT> Regs;
  constexpr bool F32 = CT == KH_TYPE_F32;
  constexpr int KS = Regs::KS, VD = Regs::VD, VC = Regs::VC;
  constexpr int RM = 16 * RT;
  constexpr int NT = DT / 16;                  // 16-wide tiles of O^T: (chunk, t)
  constexpr bool SCALED_Q = CT == KH_TYPE_F16 && NQ > 1;
  constexpr float kBias = CT == KH_TYPE_F16 ? kWeightExp : 0.0f;

  __shared__ int first[WHOLE ? 1 : kMaxBatch + 1];
  __shared__ int wave_sums[kWaves];
  __shared__ Paths paths;
  __shared__ f32x4 o_share[WAVES / 2][RT][NT][64];
  __shared__ float ml_share[WAVES / 2][2][RM];

  const int lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  int me = blockIdx.x, at = 0, end = 1;
  if constexpr (!WHOLE) {
    const_work &w = fresh();
    scan_tiles<WIN, 0>(w, first, wave_sums);
    const Plan plan = plan_of<0>(w, first);
    if (me >= plan.count) return;
    // neighbouring ranges on the same XCD: they share row blocks' keys
    const int xcd = me & 7, per = plan.count >> 3, rest = plan.count & 7;
    me = xcd * per + min(xcd, rest) + (me >> 3);
    at = range_start(plan, me);
    end = range_start(plan, me + 1);
  }

  int paths_of = -1;   // sequence whose paths the LDS holds
  while (at < end) {
    const_work &w = fresh();
    int s, item, t0, t1, tiles, len;
    if constexpr (WHOLE) {
      s = (int)((uint32_t)me / (uint32_t)w.items);
      item = me - s * w.items;
      len = clamp_len(w, s);
      tiles = tiles_of<WIN>(w, len);
      t0 = 0;
      t1 = tiles;
      at = end;
    } else {
      s = sequence_of(w, first, at);
      len = clamp_len(w, s);
      tiles = tiles_of<WIN>(w, len);
      const int in_seq = at - __builtin_amdgcn_readfirstlane(first[s]) * w.items;
      item = (int)((uint32_t)in_seq / (uint32_t)tiles);
      t0 = in_seq - item * tiles;
      t1 = min(tiles, t0 + (end - at));
      at += t1 - t0;
    }
    const int cached = tiles - w.draft_tiles;
    const Span span = span_of<WIN>(w, len);
    // item = (kv head, [token,] row block)
    const int c = (int)((uint32_t)item / (uint32_t)w.per_head);
    const int b = item - c * w.per_head;
    const bool sel = w.sel_tiles;
    const int token = sel ? (int)((uint32_t)b / (uint32_t)w.blocks) : 0;
    const int row0 = (sel ? b - token * w.blocks : b) * RM;
    const bool act32 = w.p.act_type == KH_TYPE_F32;

    const bool has_draft = t1 > cached;
    const bool tree = w.p.parents != nullptr;
    if ((has_draft || WIN) && tree && paths_of != s) {
      __syncthreads();   // the last item's rows have read the table
      build_paths<WIN>(w, s, len, paths);
      paths_of = s;
    }

    // -- where tile t lies; the first tile at or after t with a key, in steps of the waves
    const_work &wt = fresh();
    const T *kp = static_cast<const T *>(wt.p.k_pages) + c * wt.p.kp_h, *vp = static_cast<const T *>(wt.p.v_pages) + c * wt.p.vp_h;
    const int64_t kp_p = wt.p.kp_p, vp_p = wt.p.vp_p;
    const int kp_t = (int)wt.p.kp_t, vp_t = (int)wt.p.vp_t, half_shift = wt.half_shift, pages = wt.p.pages;
    const const_ints row_of_table = ints_of(wt.p.table) + s * wt.p.table_s;
    auto find = [&](int &t, Source<T> &r) {
      for (; t < t1; t += WAVES) {
        if (t >= cached) {
          const_work &w = fresh();
          r.draft = t - cached;
          if constexpr (WIN) r.edge = false;
          const int n0 = kTile * r.draft;
          r.k_row = (int)w.p.k_n;
          r.v_row = (int)w.p.v_n;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            r.valid[h] = min(max(w.p.draft - (n0 + 16 * h), 0), 16);
            const int n = r.valid[h] ? n0 + 16 * h : 0;
            r.k[h] = static_cast<const T *>(w.p.k) + (s * w.p.k_s + c * w.p.k_h + n * w.p.k_n);
            r.v[h] = static_cast<const T *>(w.p.v) + (s * w.p.v_s + c * w.p.v_h + n * w.p.v_n);
          }
          return;
        }
        r.draft = -1;
        r.k_row = kp_t;
        r.v_row = vp_t;
        const int real = t < span.head ? t : t + span.skip;
        if constexpr (WIN) {
          r.pos = kTile * real;
          r.edge = on_edge<WIN>(fresh(), len, r.pos, kTile);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int j = 2 * real + h;
          int col = j >> half_shift, pos = 16 * j;
          const int slot = (j & ((1 << half_shift) - 1)) * 16;
          bool in = true;
          if (sel) {
            const_work &w = fresh();
            const int rank = col;
            in = rank < w.p.top;
            const const_ints list = ints_of(w.p.selected) + (s * w.p.sel_s + token * w.p.sel_n + c * w.p.sel_h);
            const int before = in && rank > 0 ? list[rank - 1] : -1;
            col = in ? list[rank] : 0;
            in = in && col > before && col >= 0 && col < w.p.width;
            pos = in ? col * w.p.page_size + slot : len;
          }
          in = in && pos < len;
          const int page = in ? row_of_table[col] : 0;
          in = in && page >= 0 && page < pages;
          r.valid[h] = in ? min(len - pos, 16) : 0;
          const int there = in ? page : 0;
          r.k[h] = kp + (there * kp_p + (int64_t)(slot * kp_t));
          r.v[h] = vp + (there * vp_p + (int64_t)(slot * vp_t));
        }
        if (r.valid[0] | r.valid[1]) return;
      }
    };

    // a new tile of fp32 activations over a 16-bit cache is rounded as it is loaded
    auto rounds = [&](const Source<T> &r) { return !F32 && act32 && r.draft >= 0; };
    const int dim = wt.p.dim;
    auto load_k = [&](const Source<T> &r, Regs &x) {
      const void *base = rounds(r) ? fresh().p.k : nullptr;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = min(li, max(r.valid[h], 1) - 1) * r.k_row;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const int d = 32 * ks + 8 * g, in = d < dim ? d : 0;
          if (!rounds(r)) {
            load_words(r.k[h] + (uint32_t)(row + in), x.k[h][ks]);
          } else if constexpr (!F32) {
            // (r.k counts elements of T, the activations are fp32: twice its size)
            const float *y = static_cast<const float *>(base) + (r.k[h] - static_cast<const T *>(base)) + (row + in);
            const f32x4 lo = *reinterpret_cast<const f32x4 *>(y), hi = *reinterpret_cast<const f32x4 *>(y + 4);
            x.k[h][ks][0] = pack2<T>(lo[0], lo[1]);
            x.k[h][ks][1] = pack2<T>(lo[2], lo[3]);
            x.k[h][ks][2] = pack2<T>(hi[0], hi[1]);
            x.k[h][ks][3] = pack2<T>(hi[2], hi[3]);
          }
        }
      }
    };
    auto load_v = [&](const Source<T> &r, Regs &x) {
      const void *base = rounds(r) ? fresh().p.v : nullptr;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = min(4 * g + i, max(r.valid[h], 1) - 1) * r.v_row;
#pragma unroll
          for (int vc = 0; vc < VC; ++vc) {
            const int d = 16 * VD * vc + VD * li, in = d < dim ? d : 0;
            if (!rounds(r)) {
              load_words(r.v[h] + (uint32_t)(row + in), x.v[4 * h + i][vc]);
            } else if constexpr (!F32) {
              const float *y = static_cast<const float *>(base) + (r.v[h] - static_cast<const T *>(base)) + (row + in);
#pragma unroll
              for (int e = 0; e < VD; e += 4) {
                const f32x4 z = *reinterpret_cast<const f32x4 *>(y + e);
                x.v[4 * h + i][vc][e / 2] = pack2<T>(z[0], z[1]);
                x.v[4 * h + i][vc][e / 2 + 1] = pack2<T>(z[2], z[3]);
              }
            }
          }
        }
      }
    };

    Regs x;
    Source<T> here;
    int t = t0 + wave;
    find(t, here);
    if (t < t1) {
      load_k(here, x);
      load_v(here, x);
    }

    // this lane's query rows
    const_work &wq = fresh();
    int row_token[RT], row_head[RT];
    bool row_ok[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int r = row0 + rt * 16 + li;
      row_ok[rt] = r < wq.rows;
      const int rr = row_ok[rt] ? r : 0;
      row_token[rt] = sel ? token : (int)((uint32_t)rr / (uint32_t)wq.group);
      row_head[rt] = c * wq.group + (sel ? rr : rr - row_token[rt] * wq.group);
    }
    u32x4 q16[F32 ? 1 : NQ][RT][KS];
    float q32[F32 ? RT : 1][F32 ? KS : 1][8];
    // products to the base-2 domain; positive, so that a masked -inf stays one: q
    // takes a negative scale's sign, or a zero (so that 0 inf is NaN), under which
    // the smallest number does
    float mult[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float y[KS][8];
      const int64_t base = s * wq.p.q_s + row_token[rt] * wq.p.q_n + row_head[rt] * wq.p.q_h;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int d = 32 * ks + 8 * g;
        const bool in = row_ok[rt] && (d < dim);
        load_acts<T>(wq.p.q, base + (in ? d : 0), act32, y[ks]);
#pragma unroll
        for (int j = 0; j < 8; ++j) y[ks][j] = in ? y[ks][j] : 0.0f;
      }
      float up = wq.scale2 > 0.0f ? 1.0f : wq.scale2 < 0.0f ? -1.0f : wq.scale2;
      mult[rt] = fabsf(wq.scale2);
      if constexpr (SCALED_Q) {
        float most = 0.0f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int j = 0; j < 8; ++j) most = fmaxf(most, fabsf(y[ks][j]));
        most = max16x32(most);
        // the power of two that brings the largest to [2^14, 2^15)
        int e = (int)((__float_as_uint(most) >> 23) & 255) - 127;
        e = most == 0.0f || e == 128 ? 0 : min(max(14 - e, -126), 126);
        up *= __uint_as_float((uint32_t)(e + 127) << 23);
        mult[rt] *= __uint_as_float((uint32_t)(127 - e) << 23);
      }
      mult[rt] = fmaxf(mult[rt], 0x1p-126f);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
        for (int j = 0; j < 8; ++j) y[ks][j] *= up;
        if constexpr (F32) {
#pragma unroll
          for (int j = 0; j < 8; ++j) q32[rt][ks][j] = y[ks][j];
        } else {
          u32x4 parts[NQ];
          split8<T, NQ, true>(y[ks], parts);
#pragma unroll
          for (int n = 0; n < NQ; ++n) q16[n][rt][ks] = parts[n];
        }
      }
    }

    f32x4 o[RT][VC][VD];
    float m[RT], l[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      m[rt] = -INFINITY;
      l[rt] = 0.0f;
#pragma unroll
      for (int vc = 0; vc < VC; ++vc)
#pragma unroll
        for (int i = 0; i < VD; ++i) o[rt][vc][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    while (t < t1) {
      int t_next = t + WAVES;
      Source<T> next;
      find(t_next, next);

      if (dim < DT) {   // beyond dim: whatever was read meets q = 0, which needs it finite
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
          if (32 * ks + 8 * g >= dim) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int e = 0; e < Regs::KW; ++e) x.k[h][ks][e] = 0;
          }
      }
      // (products of different sums next to each other: each waits for the one before in its own)
      f32x4 sc[RT][2];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int h = 0; h < 2; ++h) sc[rt][h] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      if constexpr (F32) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
              for (int h = 0; h < 2; ++h)
                sc[rt][h] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(x.k[h][ks][j]), q32[rt][ks][j], sc[rt][h], 0, 0, 0);
      } else {
#pragma unroll
        for (int n = NQ - 1; n >= 0; --n)
#pragma unroll
          for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const u32x4 a = {x.k[h][ks][0], x.k[h][ks][1], x.k[h][ks][2], x.k[h][ks][3]};
                sc[rt][h] = Cache<CT>::mma(a, q16[n][rt][ks], sc[rt][h]);
              }
      }
      if (t_next < t1) load_k(next, x);

      uint32_t odd = 0;   // this lane group's keys with a value that is not finite (where rows see different keys)
      uint32_t see[RT];
      const bool masked = here.draft >= 0 || (WIN && here.edge);   // rows see different keys
      const bool partly = masked || (here.valid[0] & here.valid[1]) < 16;
      if (partly) {
        // which of the tile's keys this lane's rows attend to
        const uint32_t there = ((1u << here.valid[0]) - 1) | ((1u << here.valid[1]) - 1) << 16;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          see[rt] = there;
          if (here.draft >= 0) {
            const int i = row_token[rt] - kTile * here.draft;   // chain: the tokens up to its own
            see[rt] &= tree ? paths.bits[row_token[rt]][here.draft] : (i < 0 ? 0u : i >= 31 ? ~0u : (2u << i) - 1);
            if (WIN && !tree) {   // (a tree's bits know the window)
              const_work &w = fresh();
              see[rt] &= window_bits(row_token[rt] - w.p.window + 1, w.p.sinks - len, kTile * here.draft);
            }
          } else if (WIN && here.edge) {
            const_work &w = fresh();
            const int depth = tree ? (int)paths.depth[row_token[rt]] : row_token[rt];
            see[rt] &= window_bits(len - w.p.window + 1 + depth, w.p.sinks, here.pos);
          }
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (!(see[rt] >> (16 * (j >> 2) + 4 * g + (j & 3)) & 1)) sc[rt][j >> 2][j & 3] = -INFINITY;
        }
        // values behind the last key (a page's unwritten slots): their weight
        // is 0, which needs them finite
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (4 * g + (j & 3) >= here.valid[j >> 2]) {
#pragma unroll
            for (int vc = 0; vc < VC; ++vc)
#pragma unroll
              for (int e = 0; e < Regs::VW; ++e) x.v[j][vc][e] = 0;
          }
        // a new token's value that is not finite must not reach rows that do
        // not attend to it through 0 * inf: it is taken out of the product
        // here and added by hand below
        if (masked) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int vc = 0; vc < VC; ++vc)
#pragma unroll
              for (int e = 0; e < Regs::VW; ++e) {
                const uint32_t u = x.v[j][vc][e];
                if constexpr (F32) {
                  if ((u & 0x7f800000u) == 0x7f800000u) {
                    x.v[j][vc][e] = 0;
                    odd |= 1u << j;
                  }
                } else {
                  constexpr uint32_t kExp = CT == KH_TYPE_BF16 ? 0x7f80u : 0x7c00u;
                  const bool lo = (u & kExp) == kExp, hi = (u >> 16 & kExp) == kExp;
                  if (lo || hi) {
                    x.v[j][vc][e] = (lo ? 0u : u & 0xffffu) | (hi ? 0u : u & 0xffff0000u);
                    odd |= 1u << j;
                  }
                }
              }
        }
      }

      // the running softmax of this lane's rows (the four lane groups of a row agree on m)
      float pr[RT][8];
      u32x4 parts[F32 ? 1 : RT][NW];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        float most = sc[rt][0][0];
#pragma unroll
        for (int j = 1; j < 8; ++j) most = fmaxf(most, sc[rt][j >> 2][j & 3]);
        most = max16x32(most);
        // m is kBias below the largest score, so that weights reach 2^kBias; any
        // rounding of it is the same for every key and is scaled out again
        const float m_new = fmaxf(m[rt], fmaf(most, mult[rt], -kBias));
        const float zero = m_new == -INFINITY ? 0.0f : m_new;   // nothing seen yet: every weight is 0
        const float shrink = __builtin_amdgcn_exp2f(m[rt] - zero);
        m[rt] = m_new;
        // past 2^22 a rounding of m is a factor of 2^(1/4) and more: fp16 weights could overflow
        const bool far = CT == KH_TYPE_F16 && __any(fabsf(m_new) > 0x1p22f);
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          pr[rt][j] = fmaf(sc[rt][j >> 2][j & 3], mult[rt], -zero);
        }
        if (far) {
#pragma unroll
          for (int j = 0; j < 8; ++j) pr[rt][j] = pr[rt][j] > kBias ? kBias : pr[rt][j];   // (a NaN stays)
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          pr[rt][j] = __builtin_amdgcn_exp2f(pr[rt][j]);
          sum += pr[rt][j];
        }
        l[rt] = fmaf(l[rt], shrink, sum);
        if (__any(shrink != 1.0f)) {
#pragma unroll
          for (int vc = 0; vc < VC; ++vc)
#pragma unroll
            for (int i = 0; i < VD; ++i) o[rt][vc][i] *= shrink;
        }
        if constexpr (!F32) split8<T, NW, false>(pr[rt], parts[rt]);
      }
      if constexpr (F32) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int vc = 0; vc < VC; ++vc)
#pragma unroll
            for (int i = 0; i < VD; ++i)
#pragma unroll
              for (int rt = 0; rt < RT; ++rt)
                o[rt][vc][i] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(x.v[j][vc][i]), pr[rt][j], o[rt][vc][i], 0, 0, 0);
      } else {
#pragma unroll
        for (int vc = 0; vc < VC; ++vc)
#pragma unroll
          for (int i0 = 0; i0 < VD; i0 += 4) {
            u32x4 a[4];   // 8 keys of dimensions i0 ..
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                a[i][e] = __builtin_amdgcn_perm(x.v[2 * e + 1][vc][(i0 + i) / 2], x.v[2 * e][vc][(i0 + i) / 2],
                                                i & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
            for (int n = NW - 1; n >= 0; --n)
#pragma unroll
              for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) o[rt][vc][i0 + i] = Cache<CT>::mma(a[i], parts[rt][n], o[rt][vc][i0 + i]);
          }
      }
      if (t_next < t1) load_v(next, x);

      if (__builtin_expect(__any(odd != 0), 0)) {
        const_work &w = fresh();
        for (int key = 0; key < kTile; ++key) {   // the values taken out, by hand
          const int j = 4 * (key >> 4) + (key & 3), from = (key & 15) >> 2;
          if (!__any(g == from && (odd >> j & 1))) continue;
          const int n = min(kTile * here.draft + key, w.p.draft - 1);
          const int64_t row = s * w.p.v_s + c * w.p.v_h + n * w.p.v_n;
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) {
            float mine = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) mine = e == j ? pr[rt][e] : mine;
            const float weight = __shfl(mine, li + 16 * from);
            if (!(see[rt] >> key & 1)) continue;
#pragma unroll
            for (int vc = 0; vc < VC; ++vc)
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const int d = 16 * VD * vc + VD * (4 * g + r);
                float y[VD];
                if (!WIN || here.draft >= 0) {
                  load_acts<T>(w.p.v, row + (d < dim ? d : 0), act32, y);
                } else {   // (a cached one)
                  load_acts<T>(key & 16 ? here.v[1] : here.v[0], (int64_t)(key & 15) * here.v_row + (d < dim ? d : 0), false, y);
                }
#pragma unroll
                for (int i = 0; i < VD; ++i) {
                  const float z = (float)(T)y[i];
                  if (!(fabsf(z) < INFINITY)) o[rt][vc][i][r] += weight * z;
                }
              }
          }
        }
      }
      here = next;
      t = t_next;
    }

    // -- the waves' parts joined, in a fixed order
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      l[rt] = sum16x32(l[rt]);
      // an unused token's rows: marked by l = -1 in the part that holds its tile
      if (has_draft && tree && wave == 0 && paths.next[row_token[rt]] == -2) l[rt] = -1.0f;
    }
    auto put = [&](int to) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
        for (int vc = 0; vc < VC; ++vc)
#pragma unroll
          for (int i = 0; i < VD; ++i) o_share[to][rt][vc * VD + i][lane] = o[rt][vc][i];
        if (g == 0) {
          ml_share[to][0][rt * 16 + li] = m[rt];
          ml_share[to][1][rt * 16 + li] = l[rt];
        }
      }
    };
    auto join = [&](int from) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const float mo = ml_share[from][0][rt * 16 + li], lo = ml_share[from][1][rt * 16 + li];
        const float mn = fmaxf(m[rt], mo), zero = mn == -INFINITY ? 0.0f : mn;
        const float a = __builtin_amdgcn_exp2f(m[rt] - zero), b2 = __builtin_amdgcn_exp2f(mo - zero);
        l[rt] = l[rt] < 0.0f || lo < 0.0f ? -1.0f : l[rt] * a + lo * b2;
        m[rt] = mn;
#pragma unroll
        for (int vc = 0; vc < VC; ++vc)
#pragma unroll
          for (int i = 0; i < VD; ++i) o[rt][vc][i] = o[rt][vc][i] * a + o_share[from][rt][vc * VD + i][lane] * b2;
      }
    };
#pragma unroll
    for (int step = WAVES / 2; step; step /= 2) {
      if (t1 - t0 <= step) continue;   // (waves from `step` on had no tile)
      if (wave >= step && wave < 2 * step) put(wave - step);
      __syncthreads();
      if (wave < step) join(wave);
      if (step > 1) __syncthreads();
    }
    if (wave == 0) {
      const_work &w = fresh();
      const bool done = WHOLE || (t0 == 0 && t1 == tiles);
      // (t0 > 0: this range's first part; else its last)
      const int64_t slot = 2 * (int64_t)me + (t0 > 0 ? 0 : 1);
      float *part = w.part + slot * RM * DT;
      float *stats = w.part + 2 * (int64_t)w.grid * RM * DT + slot * RM * 2;
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        if (!row_ok[rt]) continue;
        if (!done && g == 0) {
          stats[2 * (rt * 16 + li)] = m[rt];
          stats[2 * (rt * 16 + li) + 1] = l[rt];
        }
        const float norm = 1.0f / l[rt];
        const int64_t out = s * w.p.o_s + row_token[rt] * w.p.o_n + row_head[rt] * w.p.o_h;
#pragma unroll
        for (int vc = 0; vc < VC; ++vc)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int d = 16 * VD * vc + VD * (4 * g + r);
            if (d >= dim) continue;
            float y[VD];
#pragma unroll
            for (int i = 0; i < VD; ++i) y[i] = o[rt][vc][i][r];
            float *to = part + (rt * 16 + li) * DT + d;
            if (done) {
#pragma unroll
              for (int i = 0; i < VD; ++i) y[i] = l[rt] < 0.0f ? 0.0f : y[i] * norm;
              to = static_cast<float *>(w.p.out) + out + d;
            }
            if (F32 || act32 || !done) {
#pragma unroll
              for (int i = 0; i < VD; i += 4) *reinterpret_cast<f32x4 *>(to + i) = f32x4{y[i], y[i + 1], y[i + 2], y[i + 3]};
            } else if constexpr (!F32) {
#pragma unroll
              for (int i = 0; i < VD; i += 4)
                *reinterpret_cast<u32x2 *>(static_cast<T *>(w.p.out) + out + d + i) = u32x2{pack2<T>(y[i], y[i + 1]), pack2<T>(y[i + 2], y[i + 3])};
            }
          }
      }
    }
    if (!WHOLE && at < end) __syncthreads();   // the shared parts are free again
  }
}

// ---------------------------------------------------------------------------
// Many rows (kWideRows and more) over a 16-bit cache: the matrix cores decide,
// not the loads. A workgroup's four waves take 32 rows each and share a tile
// of 64 keys in the LDS, copied while the tile before is used; 32x32x16
// products give a lane half its row's 32 scores of a block, so a row's maximum
// takes one exchange of lane halves instead of two, and each operand read from
// the LDS serves 32 rows. V^T operands come from transposing LDS reads.
//
// Measured: 4 sequences of 3604 to 32768 tokens, 64 drafted tokens of 8 heads a
// group (512 rows over 4 fp16 heads of 128) 174 us and 13 for the join (weights in
// one part 146, where paged_attn_kernel on 64 rows a wave took 369). K and V are
// fetched once for each of an item's four row blocks, 562 MiB for 142: equal
// ranges cut the blocks at different keys, so they do not meet in an XCD's L2.
// That is 3.4 TB/s; at 2.4 GHz the matrix instructions are busy 26% of the
// time, VALU 35% (10.6 for each of them), the LDS 9% (no conflicts). Tried
// without gain, with weights in one part: the second block's exponentials
// between the first block's products (146 us; fp32 activations slower), eight
// waves of 256 rows with two tiles copied ahead (150 us).
//
// Over 4-bit pages threads make a tile's bf16 values out of codes that were loaded
// a tile before, where other caches copy to the LDS; q of fp16 takes two bf16 parts. 64
// tokens of 4 sequences, 32 query heads on 4 of 128, up to 32768 tokens, fp16: 235
// to 242 us (228 at best) and 13.5 for the join (8 more with split8, which is for caches
// that hold infinities), 53% of the rate of a large matrix product. Without gain: one wave a SIMD
// (292), the products' operands read a step ahead (231 to 238).

// Chunk swizzle of K and V rows in the LDS, 16-byte chunks: a 128-bit read
// meets in one LDS cycle rows {0-3, 12-15, 20-27}, distinct mod 16, so every
// row mod 16 (mod 8 of each parity, two 64-wide rows to 256 bytes) has a chunk
// of its own; a transposing read's 32 lanes address 4 adjacent rows at the same
// 4 chunks, which a row's low bits move to other ones.
template <int DT>
__device__ __forceinline__ int swz_wide(int r) {
  if constexpr (DT == 128) return (r & 3) << 2 | (r >> 2 & 3);
  else return (r >> 1 & 1) << 2 | (r >> 2 & 3);
}

typedef __attribute__((address_space(3))) void lds_void;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
typedef float f32x16 __attribute__((ext_vector_type(16)));

template <int CT>
__device__ __forceinline__ f32x16 mma32(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (CT != KH_TYPE_F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// 64 lanes' 16 bytes at base + voff to LDS address lds + 16 lane (a wave-uniform base)
__device__ __forceinline__ void copy_rows(const void *base, uint32_t voff, uint32_t lds) {
  const uint64_t v = (uint64_t)(uintptr_t)base;
  const uint64_t at = (uint64_t)__builtin_amdgcn_readfirstlane((uint32_t)(v >> 32)) << 32 |
                      (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)v);
  const uint32_t to = __builtin_amdgcn_readfirstlane(lds);
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(voff), "s"(at), "s"(to)
               : "memory", "m0");
}

__device__ __forceinline__ void copies_landed() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((7 << 4) | (15 << 8));   // vmcnt(0)
  asm volatile("" ::: "memory");
}

constexpr int kWideSpots = 512;

template <int CT, int NQ, int NW, int DT, bool WIN>
__global__ __launch_bounds__(kThreads, 2) void paged_wide_kernel(const PagedWork) {
  typedef typename Cache<CT>::T T;
  constexpr int TK = 64, NH = 4;               // keys of a tile, its parts of 16
  constexpr int KS = DT / 16, NT = DT / 32;    // chunks of 16 dimensions in S^T, tiles of 32 in O^T
  constexpr int RB = DT * 2, CH = RB / 16;     // bytes and chunks of a row
  constexpr int RPI = 64 / CH;                 // rows of a copy
  constexpr int RM = 32 * kWaves;
  constexpr int PART = 16 * RB, SIDE = NH * PART;   // bytes of 16 keys, of a tile's K or V
  constexpr bool MX = CT == KH_TYPE_MX4;
  constexpr int LEAD = MX ? kMxWideLead : 0;
  typedef std::conditional_t<MX && NQ == 2, _Float16, T> A;   // 16-bit activations
  constexpr bool SCALED_Q = CT == KH_TYPE_F16 && NQ > 1;
  constexpr float kBias = CT == KH_TYPE_F16 ? kWeightExp : 0.0f;

  __shared__ __attribute__((aligned(256))) unsigned char tiles_lds[2][2][SIDE];   // [buffer][K, V]
  __shared__ int first[kMaxWideBatch + 1];
  __shared__ int wave_sums[kWaves];
  __shared__ Paths paths;
  __shared__ uint32_t spots[kWideSpots];
  __shared__ uint32_t odd_keys[kMaxDraft / TK][2];   // new tokens with a value that is not finite, by tile
  __shared__ uint32_t odd_edge[WIN ? 2 : 1];         // keys of a tile on a window's edge with such a value
  __shared__ uint32_t nan_blocks[MX ? 2 : 1][MX ? TK : 1];   // 4-bit pages: [buffer][key], a byte per block whose values are set aside

  const int lane = threadIdx.x & 63, row = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  int me = blockIdx.x, at = 0, end = 1;
  const bool whole = fresh().whole;
  if (!whole) {
    const_work &w = fresh();
    scan_tiles<WIN, LEAD>(w, first, wave_sums);
    const Plan plan = plan_of<LEAD>(w, first);
    if (me >= plan.count) return;
    const int xcd = me & 7, per = plan.count >> 3, rest = plan.count & 7;
    me = xcd * per + min(xcd, rest) + (me >> 3);
    at = range_start(plan, me);
    end = range_start(plan, me + 1);
  }
  int paths_of = -1;
  while (at < end) {
    const_work &w = fresh();
    int s, item, t0, t1, tiles, len;
    if (whole) {
      s = (int)((uint32_t)me / (uint32_t)w.items);
      item = me - s * w.items;
      len = clamp_len(w, s);
      tiles = tiles_of<WIN>(w, len);
      t0 = 0;
      t1 = tiles;
      at = end;
    } else {
      s = sequence_of(w, first, at);
      len = clamp_len(w, s);
      tiles = tiles_of<WIN>(w, len);
      const int in_seq = at - __builtin_amdgcn_readfirstlane(first[s]) * w.items;
      item = (int)((uint32_t)in_seq / (uint32_t)(tiles + LEAD));
      t0 = in_seq - item * (tiles + LEAD);
      t1 = min(tiles + LEAD, t0 + (end - at));
      at += t1 - t0;
      if constexpr (LEAD > 0) {
        t0 = max(t0 - LEAD, 0);
        t1 = max(t1 - LEAD, 0);
        if (t1 == 0) continue;
      }
    }
    const int cached = tiles - w.draft_tiles;
    const int c = (int)((uint32_t)item / (uint32_t)w.per_head);
    const int b = item - c * w.per_head;
    const bool sel = w.sel_tiles;
    const int token = sel ? (int)((uint32_t)b / (uint32_t)w.blocks) : 0;
    const int row0 = (sel ? b - token * w.blocks : b) * RM;
    const bool act32 = w.p.act_type == KH_TYPE_F32;
    const bool has_draft = t1 > cached;
    const bool tree = w.p.parents != nullptr;
    const int dim = w.p.dim;
    const Span span = span_of<WIN>(w, len);
    if ((has_draft || WIN) && tree && paths_of != s) {
      __syncthreads();
      build_paths<WIN>(w, s, len, paths);
      paths_of = s;
    }

    // places of the cached parts of tiles [c0, c1), by all threads
    const int half_mask = (1 << w.half_shift) - 1;
    auto stage = [&](int c0, int c1) {
      const_work &w = fresh();
      const int32_t *table = w.p.table + s * w.p.table_s;
      for (int at = NH * c0 + (int)threadIdx.x; at < NH * min(c1, cached); at += kThreads) {
        const int j = at < NH * span.head ? at : at + NH * span.skip;
        int col = j >> w.half_shift, pos = 16 * j;
        bool in = true;
        if (sel) {
          const int rank = col;
          in = rank < w.p.top;
          const int32_t *list = w.p.selected + (s * w.p.sel_s + token * w.p.sel_n + c * w.p.sel_h);
          const int before = in && rank > 0 ? list[rank - 1] : -1;
          col = in ? list[rank] : 0;
          in = in && col > before && col >= 0 && col < w.p.width;
          pos = in ? col * w.p.page_size + (j & half_mask) * 16 : len;
        }
        in = in && pos < len;
        const int page = in ? table[col] : -1;
        in = in && page >= 0 && page < w.p.pages;
        spots[at - NH * c0] = in ? (uint32_t)page * 32u + (uint32_t)min(len - pos, 16) : 0u;
      }
    };
    stage(t0, min(t1, t0 + kWideSpots / NH));

    // this lane's query row: chunk 2 ks + half of its dimensions
    const_work &wq = fresh();
    const int r_item = row0 + 32 * wave + row;
    const bool row_ok = r_item < wq.rows;
    const int rr = row_ok ? r_item : 0;
    const int row_token = sel ? token : (int)((uint32_t)rr / (uint32_t)wq.group);
    const int row_head = c * wq.group + (sel ? rr : rr - row_token * wq.group);
    u32x4 q[NQ][KS];
    float mult = fabsf(wq.scale2);
    {
      float y[KS][8];
      const int64_t base = s * wq.p.q_s + row_token * wq.p.q_n + row_head * wq.p.q_h;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int d = 16 * ks + 8 * half;
        const bool in = row_ok && d < dim;
        load_acts<A>(wq.p.q, base + (in ? d : 0), act32, y[ks]);
#pragma unroll
        for (int j = 0; j < 8; ++j) y[ks][j] = in ? y[ks][j] : 0.0f;
      }
      float up = wq.scale2 > 0.0f ? 1.0f : wq.scale2 < 0.0f ? -1.0f : wq.scale2;
      if constexpr (SCALED_Q) {
        float most = 0.0f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int j = 0; j < 8; ++j) most = fmaxf(most, fabsf(y[ks][j]));
        const float2 both = half_pair(most);
        most = fmaxf(both.x, both.y);
        int e = (int)((__float_as_uint(most) >> 23) & 255) - 127;   // to [2^14, 2^15)
        e = most == 0.0f || e == 128 ? 0 : min(max(14 - e, -126), 126);
        up *= __uint_as_float((uint32_t)(e + 127) << 23);
        mult *= __uint_as_float((uint32_t)(127 - e) << 23);
      }
      mult = fmaxf(mult, 0x1p-126f);   // (as there)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
        for (int j = 0; j < 8; ++j) y[ks][j] *= up;
        u32x4 parts[NQ];
        split8<T, NQ, true>(y[ks], parts);
#pragma unroll
        for (int n = 0; n < NQ; ++n) q[n][ks] = parts[n];
      }
    }

    f32x16 o[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[t][r] = 0.0f;
    float m = -INFINITY, l = 0.0f;

    const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_void *)tiles_lds;
    // copies of tile t into buffer `to`: wave i takes its part i, row by row in
    // RB bytes, chunk x of row r at x ^ swz_wide(r)
    const int crow = lane / CH, cpos = lane % CH;
    auto fetch = [&](int t, int c0, int to) {
      const_work &w = fresh();
      const uint32_t k_lds = lds0 + (uint32_t)(to * 2 * SIDE + wave * PART), v_lds = k_lds + SIDE;
      if (t < cached) {
        const int j = NH * (t < span.head ? t : t + span.skip) + wave, slot = (j & half_mask) * 16;
        const int page = (int)(__builtin_amdgcn_readfirstlane(spots[NH * (t - c0) + wave]) >> 5);
        const T *kb = static_cast<const T *>(w.p.k_pages) + (c * w.p.kp_h + page * w.p.kp_p + slot * w.p.kp_t);
        const T *vb = static_cast<const T *>(w.p.v_pages) + (c * w.p.vp_h + page * w.p.vp_p + slot * w.p.vp_t);
#pragma unroll
        for (int i = 0; i < 16 / RPI; ++i) {
          const int r = RPI * i + crow, d = 8 * (cpos ^ swz_wide<DT>(r)), in = d < dim ? d : 0;
          copy_rows(kb, (uint32_t)(r * (int)w.p.kp_t + in) * 2u, k_lds + i * 1024);
          copy_rows(vb, (uint32_t)(r * (int)w.p.vp_t + in) * 2u, v_lds + i * 1024);
        }
        return;
      }
      // new tokens: rounded to the cache's type, what is not finite in V set aside
      const int n0 = TK * (t - cached) + 16 * wave;
      uint32_t odd = 0;
#pragma unroll 1
      for (int i = 0; i < 16 / RPI; ++i) {   // (rolled: its registers would come on top of the loop's)
        const int r = RPI * i + crow, d = 8 * (cpos ^ swz_wide<DT>(r)), in = d < dim ? d : 0;
        const int n = n0 + r;
        const bool there = n < w.p.draft;
        float y[8], z[8];
        const int64_t nn = there ? n : 0;
        load_acts<T>(w.p.k, s * w.p.k_s + c * w.p.k_h + nn * w.p.k_n + in, act32, y);
        load_acts<T>(w.p.v, s * w.p.v_s + c * w.p.v_h + nn * w.p.v_n + in, act32, z);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const bool fine = fabsf((float)(T)z[e]) < INFINITY;
          if (there && !fine) odd |= 1u << r;
          z[e] = there && fine ? z[e] : 0.0f;
        }
        u32x4 kw[1], vw[1];
        split8<T, 1, true>(y, kw);
        split8<T, 1, true>(z, vw);
        *(lds_u32x4 *)(uintptr_t)(k_lds + i * 1024 + lane * 16) = kw[0];
        *(lds_u32x4 *)(uintptr_t)(v_lds + i * 1024 + lane * 16) = vw[0];
      }
      if (odd) atomicOr(&odd_keys[t - cached][wave >> 1], odd << (16 * (wave & 1)));
    };
    // 4-bit pages: a thread takes 16 bytes of K (32 dimensions of a key) or V (8
    // of 4 keys) a turn, loads them a tile ahead of the one that is written to
    // the LDS, which is a tile ahead of the one in use
    constexpr int TURNS = 4 * DT / kThreads, KN = DT / 32, VN = DT / 8;   // 16-byte pieces of a key's K, of 4 keys' V
    u32x4 raw[MX ? TURNS : 1];
    uint32_t raw_e[MX ? TURNS : 1];   // a scale byte, or 4
    auto piece = [&](int i, bool &values) {
      const int x = i * kThreads + (int)threadIdx.x;
      values = DT == 128 ? i == 1 : wave >= 2;
      return values ? x - 2 * DT : x;
    };
    auto load_raw = [&](int t, int c0) {
      if (t >= cached) return;
      const_work &w = fresh();
#pragma unroll
      for (int i = 0; i < TURNS; ++i) {
        bool values;
        const int x = piece(i, values);
        const int key = values ? 4 * (x / VN) : x / KN, d = values ? 8 * (x % VN) : 32 * (x % KN), in = d < dim ? d : 0;
        const int part = NH * (t < span.head ? t : t + span.skip) + (key >> 4), slot = (part & half_mask) * 16 + (key & 15);
        const int64_t page = spots[NH * (t - c0) + (key >> 4)] >> 5;
        const uint8_t *at = static_cast<const uint8_t *>(values ? w.p.v_pages : w.p.k_pages) +
                            (values ? c * w.p.vp_h + page * w.p.vp_p : c * w.p.kp_h + page * w.p.kp_p);
        raw[i] = *reinterpret_cast<const u32x4 *>(at + (uint32_t)(values ? mx_value_code(slot, in, dim) : mx_key_code(slot, in, dim)));
        if (values) raw_e[i] = *reinterpret_cast<const uint32_t *>(at + (uint32_t)mx_value_scale(slot, in, dim, w.p.page_size));
        else raw_e[i] = at[(uint32_t)mx_key_scale(slot, in, dim, w.p.page_size)];
      }
    };
    // tile t, of `valid` keys, into buffer `to`; new tokens are read and rounded here
    auto expand = [&](int t, int to, const int (&valid)[NH]) {
      const_work &w = fresh();
      const uint32_t k_lds = lds0 + (uint32_t)(to * 2 * SIDE), v_lds = k_lds + SIDE;
      const bool masked = t >= cached || (WIN && on_edge<WIN>(w, len, TK * (t < span.head ? t : t + span.skip), TK));
#pragma unroll
      for (int i = 0; i < TURNS; ++i) {
        bool values;
        const int x = piece(i, values);
        const int key = values ? 4 * (x / VN) : x / KN, d = values ? 8 * (x % VN) : 32 * (x % KN), in = d < dim ? d : 0;
        if (t >= cached) {
          const int n0 = TK * (t - cached);
          if (values) raw_e[i] = 0;
#pragma unroll 1
          for (int j = 0; j < 4; ++j) {   // 8 dimensions of K, or of one of V's 4 keys (rolled: its registers would come on top)
            if (!values) break;
            float y[8];
            load_acts<A>(w.p.v, s * w.p.v_s + c * w.p.v_h + (int64_t)min(n0 + key + j, w.p.draft - 1) * w.p.v_n + in, act32, y);
            uint32_t most = mx_most(y);
            most = max(most, (uint32_t)__shfl_xor((int)most, 1));
            most = max(most, (uint32_t)__shfl_xor((int)most, 2));
            const uint32_t e8 = mx_scale_of(most), word = mx_pack(y, e8);
            raw_e[i] |= e8 << (8 * j);
            raw[i][0] = j == 0 ? word : raw[i][0];
            raw[i][1] = j == 1 ? word : raw[i][1];
            raw[i][2] = j == 2 ? word : raw[i][2];
            raw[i][3] = j == 3 ? word : raw[i][3];
          }
          if (!values) {
            const int64_t base = s * w.p.k_s + c * w.p.k_h + (int64_t)min(n0 + key, w.p.draft - 1) * w.p.k_n + in;
            uint32_t most = 0;
#pragma unroll 1
            for (int j = 0; j < 4; ++j) {
              float y[8];
              load_acts<A>(w.p.k, base + 8 * j, act32, y);
              most = max(most, mx_most(y));
            }
            raw_e[i] = mx_scale_of(most);
#pragma unroll 1
            for (int j = 0; j < 4; ++j) {
              float y[8];
              load_acts<A>(w.p.k, base + 8 * j, act32, y);
              const uint32_t word = mx_pack(y, raw_e[i]);
              raw[i][0] = j == 0 ? word : raw[i][0];
              raw[i][1] = j == 1 ? word : raw[i][1];
              raw[i][2] = j == 2 ? word : raw[i][2];
              raw[i][3] = j == 3 ? word : raw[i][3];
            }
          }
        }
        const int h = key >> 4, there = h == 0 ? valid[0] : h == 1 ? valid[1] : h == 2 ? valid[2] : valid[3];
        const float k_scale = mx_scale(raw_e[i] & 255u);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          // K: dimensions d + 8 j of the key; V: dimensions d of key + j
          const int r = values ? key + j : key, chunk = values ? d / 8 : d / 8 + j;
          const uint32_t e8 = raw_e[i] >> (8 * j) & 255u;
          float scale = values ? mx_scale(e8) : k_scale;
          uint32_t word = raw[i][j];
          bool none = !values && d >= dim;       // K beyond dim meets q = 0, which needs it finite
          if (values) {
            const bool behind = (r & 15) >= there;   // (their weight is 0, which needs them finite)
            const bool aside = masked && e8 > kMxMost && !behind;
            if (masked && !(d & 31)) reinterpret_cast<uint8_t *>(&nan_blocks[to][r])[d >> 5] = aside && d < dim ? 1 : 0;
            none = behind || aside;
          }
          u32x4 y = {mx_pair<0>(word, scale), mx_pair<1>(word, scale), mx_pair<2>(word, scale), mx_pair<3>(word, scale)};
          if (none) y = u32x4{0, 0, 0, 0};
          *(lds_u32x4 *)(uintptr_t)((values ? v_lds : k_lds) + (uint32_t)(r * RB + ((chunk ^ swz_wide<DT>(r)) * 16))) = y;
        }
      }
    };
    // the tile at or after t that has a key; valid[] of its parts
    auto find = [&](int &t, int c0, int c1, int (&valid)[NH]) {
      for (; t < c1; ++t) {
        if (t >= cached) {
          const int n0 = TK * (t - cached), n = fresh().p.draft;
#pragma unroll
          for (int h = 0; h < NH; ++h) valid[h] = min(max(n - n0 - 16 * h, 0), 16);
          return;
        }
        int any = 0;
#pragma unroll
        for (int h = 0; h < NH; ++h) {
          valid[h] = (int)(__builtin_amdgcn_readfirstlane(spots[NH * (t - c0) + h]) & 31);
          any |= valid[h];
        }
        if (any) return;
      }
    };

    if (threadIdx.x < 2 * (kMaxDraft / TK)) odd_keys[threadIdx.x >> 1][threadIdx.x & 1] = 0;
    int buffer = 0;
    for (int c0 = t0; c0 < t1; c0 += kWideSpots / NH) {
      const int c1 = min(t1, c0 + kWideSpots / NH);
      if (c0 > t0) stage(c0, c1);   // (behind the last tile's barrier: no wave reads the old places)
      __syncthreads();
      int t = c0, valid[NH];
      find(t, c0, c1, valid);
      if constexpr (MX) {
        if (t < c1) {
          load_raw(t, c0);
          expand(t, buffer, valid);
          int t_next = t + 1, valid_next[NH];
          find(t_next, c0, c1, valid_next);
          if (t_next < c1) load_raw(t_next, c0);
        }
      } else {
        if (t < c1) fetch(t, c0, buffer);
      }
      while (t < c1) {
        int t_next = t + 1, valid_next[NH];
        find(t_next, c0, c1, valid_next);
        if constexpr (!MX) copies_landed();
        __syncthreads();   // this tile is there, and no wave reads the other buffer
        if constexpr (MX) {
          if (t_next < c1) {
            expand(t_next, buffer ^ 1, valid_next);
            int t_then = t_next + 1, valid_then[NH];
            find(t_then, c0, c1, valid_then);
            if (t_then < c1) load_raw(t_then, c0);
          }
        } else {
          if (t_next < c1) fetch(t_next, c0, buffer ^ 1);
        }
        const uint32_t k_lds = lds0 + (uint32_t)(buffer * 2 * SIDE), v_lds = k_lds + SIDE;
        const int draft = t >= cached ? t - cached : -1;
        int fewest = valid[0] & valid[1] & valid[2] & valid[3];
        const int pos = TK * (t < span.head ? t : t + span.skip);
        const bool edge = WIN && draft < 0 && on_edge<WIN>(fresh(), len, pos, TK);
        const bool partly = draft >= 0 || edge || fewest < 16;
        if constexpr (WIN && !MX) if (edge) {
          // a value that is not finite must not reach rows that do not see its
          // key: set aside, as a new token's is
          if (threadIdx.x < 2) odd_edge[threadIdx.x] = 0;
          __syncthreads();
#pragma unroll 1
          for (int i = 0; i < SIDE / (16 * kThreads); ++i) {
            const int chunk = i * kThreads + (int)threadIdx.x, r = chunk / CH;
            u32x4 x = *(lds_u32x4 *)(uintptr_t)(v_lds + chunk * 16);
            constexpr uint32_t kExp = CT == KH_TYPE_BF16 ? 0x7f80u : 0x7c00u;
            bool odd = false;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const bool lo = (x[e] & kExp) == kExp, hi = (x[e] >> 16 & kExp) == kExp;
              odd |= lo | hi;
              x[e] = (lo ? 0u : x[e] & 0xffffu) | (hi ? 0u : x[e] & 0xffff0000u);
            }
            const int there = r < 16 ? valid[0] : r < 32 ? valid[1] : r < 48 ? valid[2] : valid[3];
            const int d = 8 * ((chunk % CH) ^ swz_wide<DT>(r));
            if (odd) {
              *(lds_u32x4 *)(uintptr_t)(v_lds + chunk * 16) = x;
              if ((r & 15) < there && d < dim) atomicOr(&odd_edge[r >> 5], 1u << (r & 31));
            }
          }
          __syncthreads();
        }
        if (!MX && draft < 0 && fewest < 16) {
          // values behind the last key (a page's unwritten slots): their weight
          // is 0, which needs them finite
#pragma unroll
          for (int i = 0; i < SIDE / (16 * kThreads); ++i) {
            const int chunk = i * kThreads + (int)threadIdx.x, r = chunk / CH;
            const int there = r < 16 ? valid[0] : r < 32 ? valid[1] : r < 48 ? valid[2] : valid[3];
            if ((r & 15) >= there) *(lds_u32x4 *)(uintptr_t)(v_lds + chunk * 16) = u32x4{0, 0, 0, 0};
          }
          __syncthreads();
        }
        if (!MX && dim < DT) {   // K beyond dim meets q = 0, which needs it finite
#pragma unroll
          for (int i = 0; i < SIDE / (16 * kThreads); ++i) {
            const int chunk = i * kThreads + (int)threadIdx.x, r = chunk / CH, x = (chunk % CH) ^ swz_wide<DT>(r);
            if (8 * x >= dim) *(lds_u32x4 *)(uintptr_t)(k_lds + chunk * 16) = u32x4{0, 0, 0, 0};
          }
          __syncthreads();
        }

        // scores of the two blocks of 32 keys: register r of a lane is key 8 (r >> 2) + 4 half + (r & 3)
        f32x16 sc[2];
        const uint32_t k_at = k_lds + (uint32_t)row * RB + (uint32_t)(half ^ swz_wide<DT>(row)) * 16u;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int r = 0; r < 16; ++r) sc[kb][r] = 0.0f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          u32x4 k[2];
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
            k[kb] = *(const lds_u32x4 *)(uintptr_t)((k_at ^ (uint32_t)(2 * ks * 16)) + (uint32_t)(kb * 32 * RB));
#pragma unroll
          for (int n = NQ - 1; n >= 0; --n)
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) sc[kb] = mma32<CT>(k[kb], q[n][ks], sc[kb]);
          if (ks & 1) __builtin_amdgcn_sched_barrier(0);   // (all operands read ahead would not fit the registers)
        }

        uint32_t see[2];
        if (partly) {
#pragma unroll
          for (int kb = 0; kb < 2; ++kb) {
            see[kb] = ((1u << valid[2 * kb]) - 1) | ((1u << valid[2 * kb + 1]) - 1) << 16;
            if (draft >= 0) {
              const int word = 2 * draft + kb, i = row_token - 32 * word;   // chain: the tokens up to its own
              see[kb] &= tree ? (word < kMaxDraft / 32 ? paths.bits[row_token][word] : 0u)
                              : (i < 0 ? 0u : i >= 31 ? ~0u : (2u << i) - 1);
              if (WIN && !tree) {   // (a tree's bits know the window)
                const_work &w = fresh();
                see[kb] &= window_bits(row_token - w.p.window + 1, w.p.sinks - len, 32 * word);
              }
            } else if (WIN && edge) {
              const_work &w = fresh();
              const int depth = tree ? (int)paths.depth[row_token] : row_token;
              see[kb] &= window_bits(len - w.p.window + 1 + depth, w.p.sinks, pos + 32 * kb);
            }
#pragma unroll
            for (int r = 0; r < 16; ++r)
              if (!(see[kb] >> (8 * (r >> 2) + 4 * half + (r & 3)) & 1)) sc[kb][r] = -INFINITY;
          }
        }
        float most = sc[0][0];
#pragma unroll
        for (int r = 1; r < 32; ++r) most = fmaxf(most, sc[r >> 4][r & 15]);
        const float2 both = half_pair(most);
        most = fmaxf(both.x, both.y);
        // (see paged_attn_kernel: m is kBias below the largest score)
        const float m_new = fmaxf(m, fmaf(most, mult, -kBias));
        const float zero = m_new == -INFINITY ? 0.0f : m_new;
        const float shrink = __builtin_amdgcn_exp2f(m - zero);
        m = m_new;
        const bool far = CT == KH_TYPE_F16 && __any(fabsf(m_new) > 0x1p22f);
#pragma unroll
        for (int r = 0; r < 32; ++r) sc[r >> 4][r & 15] = fmaf(sc[r >> 4][r & 15], mult, -zero);
        if (far) {
#pragma unroll
          for (int r = 0; r < 32; ++r) sc[r >> 4][r & 15] = sc[r >> 4][r & 15] > kBias ? kBias : sc[r >> 4][r & 15];
        }
        float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int r = 0; r < 32; ++r) {
          sc[r >> 4][r & 15] = __builtin_amdgcn_exp2f(sc[r >> 4][r & 15]);
          sum[r & 3] += sc[r >> 4][r & 15];
        }
        l = fmaf(l, shrink, (sum[0] + sum[1]) + (sum[2] + sum[3]));
        if (__any(shrink != 1.0f)) {
#pragma unroll
          for (int t2 = 0; t2 < NT; ++t2) o[t2] *= shrink;
        }
        // O^T += V^T P^T, 16 keys at a time: a lane's keys are its registers 8 i .. 8 i + 7,
        // V^T's operand two transposing reads, in each of which lane (a4, b4) = (lane % 16 / 4,
        // lane % 4) of 16 addresses dimensions 4 b4 .. + 4 of the 16 in key row a4
        const int a4 = (lane & 15) >> 2, g1 = (lane >> 4) & 1;
        const uint32_t v_row = (uint32_t)(4 * half + a4) * RB + (uint32_t)(lane & 1) * 8u;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float y[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = sc[i >> 1][8 * (i & 1) + e];
          u32x4 parts[NW];
          if constexpr (MX) split_finite<T, NW>(y, parts);
          else split8<T, NW, false>(y, parts);
          u32x4 v[NT];
#pragma unroll
          for (int t2 = 0; t2 < NT; ++t2) {
            s16x4 x[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const int r = 16 * i + 8 * j + 4 * half + a4;
              const int chunk = (4 * t2 + 2 * g1 + ((lane & 2) >> 1)) ^ swz_wide<DT>(r);
              x[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                  (lds_s16x4 *)(uintptr_t)(v_lds + v_row + (uint32_t)((16 * i + 8 * j) * RB + chunk * 16)));
            }
            v[t2] = __builtin_bit_cast(u32x4, __builtin_shufflevector(x[0], x[1], 0, 1, 2, 3, 4, 5, 6, 7));
          }
#pragma unroll
          for (int n = NW - 1; n >= 0; --n)
#pragma unroll
            for (int t2 = 0; t2 < NT; ++t2) o[t2] = mma32<CT>(v[t2], parts[n], o[t2]);
          if (i & 1) __builtin_amdgcn_sched_barrier(0);
        }

        if constexpr (MX) {
          if (draft >= 0 || (WIN && edge)) {
            const uint32_t set_aside = nan_blocks[buffer][lane] & (DT == 64 ? 0xffffu : ~0u);   // (bytes of its blocks)
            if (__builtin_expect(__any(set_aside != 0), 0)) {
              for (int key = 0; key < TK; ++key) {
                const uint32_t blocks = __builtin_amdgcn_readlane(set_aside, key);
                if (!blocks || !((key >> 5 ? see[1] : see[0]) >> (key & 31) & 1)) continue;
#pragma unroll
                for (int t2 = 0; t2 < NT; ++t2)
                  if (blocks >> (8 * t2) & 1) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) o[t2][r] = NAN;
                  }
              }
            }
          }
        } else if (draft >= 0 || (WIN && edge)) {
          const uint32_t *set_aside = !WIN || draft >= 0 ? odd_keys[draft] : odd_edge;
          const uint32_t odd[2] = {set_aside[0], set_aside[1]};
          if (__builtin_expect(__any((odd[0] | odd[1]) != 0), 0)) {
            const_work &w = fresh();
            for (int key = 0; key < TK; ++key) {   // the values set aside, by hand
              if (!(odd[key >> 5] >> (key & 31) & 1)) continue;
              const int kk = key & 31, reg = 4 * (kk >> 3) + (kk & 3), from = kk >> 2 & 1;
              float mine = 0.0f;
#pragma unroll
              for (int r = 0; r < 32; ++r) mine = r == 16 * (key >> 5) + reg ? sc[r >> 4][r & 15] : mine;
              const float weight = __shfl(mine, row + 32 * from);
              if (!((key >> 5 ? see[1] : see[0]) >> kk & 1)) continue;
              int64_t from_row = s * w.p.v_s + c * w.p.v_h + (int64_t)(TK * draft + key) * w.p.v_n;
              if (WIN && draft < 0) {   // a cached one
                const int64_t page = spots[NH * (t - c0) + (key >> 4)] >> 5;
                const int slot = ((pos + key) & (w.p.page_size - 1));
                from_row = c * w.p.vp_h + page * w.p.vp_p + slot * w.p.vp_t;
              }
#pragma unroll
              for (int t2 = 0; t2 < NT; ++t2)
#pragma unroll
                for (int a = 0; a < 4; ++a) {
                  const int d = 32 * t2 + 8 * a + 4 * half;
                  float y[4];
                  load_acts<T>(!WIN || draft >= 0 ? w.p.v : w.p.v_pages, from_row + (d < dim ? d : 0), (!WIN || draft >= 0) && act32, y);
#pragma unroll
                  for (int e = 0; e < 4; ++e) {
                    const float z = (float)(T)y[e];
                    if (!(fabsf(z) < INFINITY)) o[t2][4 * a + e] += weight * z;
                  }
                  __builtin_amdgcn_sched_barrier(0);
                }
            }
          }
        }
#pragma unroll
        for (int h = 0; h < NH; ++h) valid[h] = valid_next[h];
        t = t_next;
        buffer ^= 1;
      }
      __syncthreads();   // all waves are done with this stretch's places, tiles and marks
    }

    // -- a wave's rows are its own: finished, or this range's part of them
    const_work &we = fresh();
    const float2 sums = half_pair(l);
    l = sums.x + sums.y;
    if (has_draft && tree && paths.next[row_token] == -2) l = -1.0f;   // an unused token's row
    if (row_ok) {
      const bool done = t0 == 0 && t1 == tiles;
      const int64_t slot = 2 * (int64_t)me + (t0 > 0 ? 0 : 1);
      const int r = 32 * wave + row;
      float *to = we.part + (slot * RM + r) * DT;
      if (!done && half == 0) {
        float *stats = we.part + 2 * (int64_t)we.grid * RM * DT + (slot * RM + r) * 2;
        stats[0] = m;
        stats[1] = l;
      }
      const int64_t out = s * we.p.o_s + row_token * we.p.o_n + row_head * we.p.o_h;
      if (done) to = static_cast<float *>(we.p.out) + out;
      const float norm = done ? 1.0f / l : 1.0f;
#pragma unroll
      for (int t2 = 0; t2 < NT; ++t2)
#pragma unroll
        for (int a = 0; a < 4; ++a) {
          const int d = 32 * t2 + 8 * a + 4 * half;
          if (d >= dim) continue;
          float y[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] = done && l < 0.0f ? 0.0f : o[t2][4 * a + e] * norm;
          if (act32 || !done) *reinterpret_cast<f32x4 *>(to + d) = f32x4{y[0], y[1], y[2], y[3]};
          else *reinterpret_cast<u32x2 *>(static_cast<A *>(we.p.out) + out + d) = u32x2{pack2<A>(y[0], y[1]), pack2<A>(y[2], y[3])};
        }
    }
  }
}

// The parts of rows that few ranges share, joined: a wave per row, in range
// order.
template <int DT, int LEAD>
__global__ __launch_bounds__(kThreads) void paged_join_rows_kernel(const PagedWork w) {
  constexpr int RM = 32 * kWaves;
  constexpr int PER = DT / 64;
  __shared__ int first[kMaxWideBatch + 1];
  __shared__ int wave_sums[kWaves];
  const kh_paged &p = w.p;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  scan_tiles<true, LEAD>(w, first, wave_sums);
  const Plan plan = plan_of<LEAD>(w, first);
  const int s = blockIdx.x / w.items, item = blockIdx.x - s * w.items;
  const int tiles = tiles_of<true>(w, clamp_len(w, s));
  const int x = first[s] * w.items + item * (tiles + LEAD) + LEAD;
  const int w0 = range_of(plan, x), w1 = range_of(plan, x + tiles - 1);
  if (w0 == w1) return;
  const int c = item / w.per_head, b = item - c * w.per_head;
  const int token = w.sel_tiles ? b / w.blocks : 0;
  const int row0 = (w.sel_tiles ? b - token * w.blocks : b) * RM;
  const bool in = lane * PER < p.dim;
  const int r = blockIdx.y * kWaves + wave;
  {
    if (row0 + r >= w.rows) return;
    const int n = w.sel_tiles ? token : (row0 + r) / w.group;
    const int head = c * w.group + (w.sel_tiles ? row0 + r : row0 + r - n * w.group);
    auto stat = [&](int i) { return w.part + 2 * (int64_t)w.grid * RM * DT + ((2 * (int64_t)(w0 + i) + (i == 0 ? 1 : 0)) * RM + r) * 2; };
    const int count = w1 - w0 + 1;
    float m = -INFINITY, l = 0.0f, o[PER];
    bool unused = false;
    for (int i = lane; i < count; i += 64) m = fmaxf(m, stat(i)[0]);
    m = wave_max(m);
    if (m == -INFINITY) m = 0.0f;
#pragma unroll
    for (int e = 0; e < PER; ++e) o[e] = 0.0f;
#pragma unroll 4
    for (int i = 0; i < count; ++i) {
      const float a = __builtin_amdgcn_exp2f(stat(i)[0] - m), li = stat(i)[1];
      l = fmaf(a, li, l);
      unused |= li < 0.0f;
      const float *part = w.part + ((2 * (int64_t)(w0 + i) + (i == 0 ? 1 : 0)) * RM + r) * DT + (in ? lane * PER : 0);
#pragma unroll
      for (int e = 0; e < PER; ++e) o[e] = fmaf(a, part[e], o[e]);
    }
    const float norm = 1.0f / l;
    const int64_t to = s * p.o_s + n * p.o_n + head * p.o_h;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const int d = lane * PER + e;
      if (d >= p.dim) continue;
      const float y = unused ? 0.0f : o[e] * norm;
      if (p.act_type == KH_TYPE_F32) static_cast<float *>(p.out)[to + d] = y;
      else if (p.act_type == KH_TYPE_BF16) static_cast<__bf16 *>(p.out)[to + d] = (__bf16)y;
      else static_cast<_Float16 *>(p.out)[to + d] = (_Float16)y;
    }
  }
}

// The parts of the items that more than one range touched, joined: a
// workgroup per row. Weights first, a part per lane, then the weighted sums,
// every fourth part to a wave, then the waves' sums in order.
template <int DT, int RT, int LEAD>
__global__ __launch_bounds__(kThreads) void paged_join_kernel(const PagedWork w) {
  constexpr int RM = 16 * RT;
  constexpr int PER = DT / 64;   // dimensions of a lane
  __shared__ int first[kMaxBatch + 1];
  __shared__ int wave_sums[kWaves];
  __shared__ float sums[kWaves][DT];
  __shared__ float weights[64];
  const kh_paged &p = w.p;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  scan_tiles<true, LEAD>(w, first, wave_sums);
  const Plan plan = plan_of<LEAD>(w, first);
  const int s = blockIdx.x / w.items, item = blockIdx.x - s * w.items;
  const int tiles = tiles_of<true>(w, clamp_len(w, s));
  const int x = first[s] * w.items + item * (tiles + LEAD) + LEAD;
  const int w0 = range_of(plan, x), w1 = range_of(plan, x + tiles - 1);
  if (w0 == w1) return;   // finished by its one range
  const int c = item / w.per_head, b = item - c * w.per_head;
  const int token = w.sel_tiles ? b / w.blocks : 0;
  const int row0 = (w.sel_tiles ? b - token * w.blocks : b) * RM;
  const int r = blockIdx.y;
  if (row0 + r >= w.rows) return;
  const int n = w.sel_tiles ? token : (row0 + r) / w.group;
  const int head = c * w.group + (w.sel_tiles ? row0 + r : row0 + r - n * w.group);
  const float *stats = w.part + 2 * (int64_t)w.grid * RM * DT + 2 * r;
  // part i of the item: the last part of range w0, then the first of the others
  auto slot = [&](int i) { return 2 * (int64_t)(w0 + i) + (i == 0 ? 1 : 0); };
  const int count = w1 - w0 + 1;
  float m = -INFINITY;
  for (int i = lane; i < count; i += 64) m = fmaxf(m, stats[slot(i) * RM * 2]);
  m = wave_max(m);
  if (m == -INFINITY) m = 0.0f;
  float l = 0.0f, o[PER];
  bool unused = false;
#pragma unroll
  for (int e = 0; e < PER; ++e) o[e] = 0.0f;
  const bool in = lane * PER < p.dim;   // (dim is a multiple of 8, PER at most 4)
  for (int i0 = 0; i0 < count; i0 += 64) {
    const int here = min(count - i0, 64);
    if (lane < here && wave == 0) {
      const float *st = stats + slot(i0 + lane) * RM * 2;
      weights[lane] = __builtin_amdgcn_exp2f(st[0] - m);
      l += weights[lane] * st[1];
      unused |= st[1] < 0.0f;
    }
    __syncthreads();
#pragma unroll 8
    for (int i = wave; i < here; i += kWaves) {
      const float *part = w.part + (slot(i0 + i) * RM + r) * DT + (in ? lane * PER : 0);
      const float a = weights[i];
#pragma unroll
      for (int e = 0; e < PER; ++e) o[e] = fmaf(a, part[e], o[e]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int e = 0; e < PER; ++e) sums[wave][lane * PER + e] = o[e];
  __syncthreads();
  if (wave) return;
  l = wave_sum(l);
  unused = __any(unused);
  const float norm = 1.0f / l;
  const int64_t at = s * p.o_s + n * p.o_n + head * p.o_h;
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    const int d = lane * PER + e;
    if (d >= p.dim) continue;
    float y = 0.0f;
    for (int i = 0; i < kWaves; ++i) y += sums[i][d];
    y = unused ? 0.0f : y * norm;
    if (p.act_type == KH_TYPE_F32) static_cast<float *>(p.out)[at + d] = y;
    else if (p.act_type == KH_TYPE_BF16) static_cast<__bf16 *>(p.out)[at + d] = (__bf16)y;
    else static_cast<_Float16 *>(p.out)[at + d] = (_Float16)y;
  }
}

template <int CT, int NQ, int NW, int DT, int RT, bool WIN>
void launch_both(const PagedWork &w, hipStream_t stream) {
  if (w.whole) {
    paged_attn_kernel<CT, NQ, NW, DT, RT, true, WIN><<<w.grid, 64 * paged_waves(DT, RT, true), 0, stream>>>(w);
  } else {
    paged_attn_kernel<CT, NQ, NW, DT, RT, false, WIN><<<w.grid, kThreads, 0, stream>>>(w);
    const dim3 grid((unsigned)(w.p.batch * w.items), (unsigned)std::min(w.rows, 16 * RT));
    paged_join_kernel<DT, RT, 0><<<grid, kThreads, 0, stream>>>(w);
  }
}

template <int CT, int NQ, int NW, int DT, bool WIN>
void launch_wide(const PagedWork &w, hipStream_t stream) {
  paged_wide_kernel<CT, NQ, NW, DT, WIN><<<w.grid, kThreads, 0, stream>>>(w);
  if (!w.whole) {
    const dim3 grid((unsigned)(w.p.batch * w.items), (unsigned)((std::min(w.rows, 32 * kWaves) + kWaves - 1) / kWaves));
    paged_join_rows_kernel<DT, CT == KH_TYPE_MX4 ? kMxWideLead : 0><<<grid, kThreads, 0, stream>>>(w);
  }
}

template <int CT, int NQ, int NW, bool WIN>
void launch_sizes(const PagedWork &w, int dt, int rt, hipStream_t stream) {
  if (dt == 256) launch_both<CT, NQ, NW, 256, 1, WIN>(w, stream);
  else if (rt == kWideBlocks) {
    if constexpr (CT != KH_TYPE_F32) {
      if (dt == 128) launch_wide<CT, NQ, NW, 128, WIN>(w, stream);
      else launch_wide<CT, NQ, NW, 64, WIN>(w, stream);
    }
  } else if (dt == 128) {
    if (rt == 1) launch_both<CT, NQ, NW, 128, 1, WIN>(w, stream);
    else launch_both<CT, NQ, NW, 128, 2, WIN>(w, stream);
  } else {
    if (rt == 1) launch_both<CT, NQ, NW, 64, 1, WIN>(w, stream);
    else launch_both<CT, NQ, NW, 64, 2, WIN>(w, stream);
  }
}

template <int CT, int NQ, int NW>
hipError_t launch_passes(const PagedWork &w, int dt, int rt, hipStream_t stream) {
  if (w.p.window) launch_sizes<CT, NQ, NW, true>(w, dt, rt, stream);
  else launch_sizes<CT, NQ, NW, false>(w, dt, rt, stream);
  return hipGetLastError();
}

}  // namespace
}  // namespace kh
