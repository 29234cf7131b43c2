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
// kernel joins; an item within one range is finished here.
//
// A wave holds its tile in registers: scores S^T = K Q^T, so that a lane has
// its query's scores (lane li = lane & 15) for keys 4 g + r (g = lane >> 4),
// which is how O^T += V^T P^T takes the weights back without a move; V^T's
// operand needs 8 keys of one dimension per lane, which a lane makes from 8
// rows' 16-byte pieces by 32 byte permutes. One pass over the keys with
// running maximum and sum (base 2, fp32).
//
// fp32 activations over a 16-bit cache keep fp32's accuracy: a bf16 product's
// three parts x = x1 + x2 + x3 of 8 bits each hold all 24 bits of q and of a
// weight, and K and V are exact, so three passes lose nothing; fp16 parts
// hold 11 bits each, two passes 22, with q scaled by a power of two per row
// and the weights by 2^14 to stay clear of fp16's subnormals.
#pragma once

#include <algorithm>
#include <cmath>
#include <type_traits>

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

struct Plan {
  int64_t total;   // tiles of the batch
  int64_t count;   // workgroups that take part
};

__device__ __forceinline__ int clamp_len(const PagedWork &w, int s) {
  const int n = w.p.lengths[s];
  const int64_t most = (int64_t)w.p.width * w.p.page_size;
  return n < 0 ? 0 : (n > most ? (int)most : n);
}

__device__ __forceinline__ int tiles_of(const PagedWork &w, int len) {
  return (w.sel_tiles ? w.sel_tiles : (len + kTile - 1) / kTile) + w.draft_tiles;
}

// first[s] = tiles of one item of the sequences before s, for s <= batch.
__device__ __forceinline__ void scan_tiles(const PagedWork &w, int *first, int *wave_sums) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n = w.p.batch;
  const int per = (n + kThreads - 1) / kThreads;
  const int lo = threadIdx.x * per;
  int sum = 0;
  for (int i = lo; i < min(lo + per, n); ++i) sum += tiles_of(w, clamp_len(w, i));
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
    at += tiles_of(w, clamp_len(w, i));
  }
  if (lo < n && lo + per >= n) first[n] = at;
  __syncthreads();
}

__device__ __forceinline__ Plan plan_of(const PagedWork &w, const int *first) {
  Plan r;
  r.total = (int64_t)first[w.p.batch] * w.items;
  // a tile per wave at least
  const int64_t want = (r.total + kWaves - 1) / kWaves;
  r.count = want < w.grid ? (want < 1 ? 1 : want) : w.grid;
  return r;
}

__device__ __forceinline__ int64_t range_start(const Plan &r, int64_t w) { return r.total * w / r.count; }

// The workgroup whose range holds tile x.
__device__ __forceinline__ int64_t range_of(const Plan &r, int64_t x) {
  return ((x + 1) * r.count + r.total - 1) / r.total - 1;
}

// Which sequence tile x of the row lies in (first[] counts one item's tiles).
__device__ __forceinline__ int sequence_of(const PagedWork &w, const int *first, int64_t x) {
  int lo = 0, hi = w.p.batch - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if ((int64_t)first[mid] * w.items <= x) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// ---------------------------------------------------------------------------

// Which rows of the drafted tokens' paths see which of them: bit j of row i.
// Also the unused tokens. Doubling: after k rounds a row holds its nearest
// 2^k ancestors.
struct Paths {
  uint32_t bits[kMaxDraft][kMaxDraft / 32];
  int16_t next[kMaxDraft];   // the next ancestor beyond those held; -1 none, -2 the token is unused
};

__device__ void build_paths(const PagedWork &w, int s, Paths &t) {
  const int i = threadIdx.x, n = w.p.draft;
  const int32_t *parents = w.p.parents + s * w.p.parents_s;
  if (i < n) {
    const int p = parents[i];
    t.next[i] = p >= -1 && p < i ? p : -2;
    for (int k = 0; k < w.draft_tiles; ++k) t.bits[i][k] = k == i / 32 ? 1u << (i & 31) : 0u;
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
        if (k < w.draft_tiles) got[k] = t.bits[i][k] | t.bits[from][k];
      if (next >= 0) next = t.next[next];
    }
    __syncthreads();
    if (i < n) {
#pragma unroll
      for (int k = 0; k < kMaxDraft / 32; ++k)
        if (k < w.draft_tiles) t.bits[i][k] = got[k];
      t.next[i] = (int16_t)next;
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

__device__ __forceinline__ float load_act(const void *p, int64_t i, int type) {
  if (type == KH_TYPE_F32) return static_cast<const float *>(p)[i];
  if (type == KH_TYPE_BF16) return (float)static_cast<const __bf16 *>(p)[i];
  return (float)static_cast<const _Float16 *>(p)[i];
}

// n (4 or 8) adjacent activations from element i, 16-byte (8-byte) aligned
template <int N>
__device__ __forceinline__ void load_acts(const void *p, int64_t i, int type, float (&x)[N]) {
  if (type == KH_TYPE_F32) {
#pragma unroll
    for (int j = 0; j < N; j += 4) {
      const f32x4 a = *reinterpret_cast<const f32x4 *>(static_cast<const float *>(p) + i + j);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[j + e] = a[e];
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < N; j += 4) {
    const u32x2 a = *reinterpret_cast<const u32x2 *>(static_cast<const uint16_t *>(p) + i + j);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t half = (a[e / 2] >> (16 * (e & 1))) & 0xffffu;
      x[j + e] = type == KH_TYPE_BF16 ? __uint_as_float(half << 16)
                                      : (float)__builtin_bit_cast(_Float16, (uint16_t)half);
    }
  }
}

template <class T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  typedef T pair __attribute__((ext_vector_type(2)));
  const pair v = {(T)a, (T)b};
  return __builtin_bit_cast(uint32_t, v);
}

// x as NP parts of type T, the first the nearest to x, each next the nearest
// to what the ones before leave.
template <class T, int NP>
__device__ __forceinline__ void split8(const float (&x)[8], u32x4 (&out)[NP]) {
  float rest[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) rest[j] = x[j];
#pragma unroll
  for (int part = 0; part < NP; ++part) {
#pragma unroll
    for (int m = 0; m < 4; ++m) out[part][m] = pack2<T>(rest[2 * m], rest[2 * m + 1]);
    if (part + 1 < NP) {
#pragma unroll
      for (int j = 0; j < 8; ++j) rest[j] -= (float)(T)rest[j];
    }
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
  int valid[2];       // keys of each half
  int draft;          // index of the tile among the new tokens' tiles, -1 for a cached one
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

// Where the two halves of a cached tile lie.
struct Spot {
  int page[2], slot[2], valid[2];
};

// FULL: dim == DT, every lane's pieces lie inside a row.
template <int CT, int NP, int DT, int RT, bool FULL>
__global__ __launch_bounds__(kThreads, (RT == 1 && DT <= 128) ? 2 : 1) void paged_attn_kernel(const PagedWork w) {
  typedef typename Cache<CT>::T T;
  typedef Tile<CT, DT> Regs;
  constexpr bool F32 = CT == KH_TYPE_F32;
  constexpr int KS = Regs::KS, VD = Regs::VD, VC = Regs::VC;
  constexpr int RM = 16 * RT;
  constexpr int NT = DT / 16;                  // 16-wide tiles of O^T: (chunk, t)
  constexpr bool SCALED_P = CT == KH_TYPE_F16;
  constexpr bool SCALED_Q = CT == KH_TYPE_F16 && NP > 1;

  __shared__ int first[kMaxBatch + 1];
  __shared__ int wave_sums[kWaves];
  __shared__ Paths paths;
  __shared__ f32x4 o_share[2][RT][NT][64];
  __shared__ float ml_share[2][2][RM];

  const kh_paged &p = w.p;
  const int lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  scan_tiles(w, first, wave_sums);
  const Plan plan = plan_of(w, first);
  // neighbouring ranges on the same XCD: they share row blocks' keys
  int me = blockIdx.x;
  if (me >= plan.count) return;
  {
    const int xcd = me & 7, per = (int)plan.count >> 3, rest = (int)plan.count & 7;
    me = xcd * per + min(xcd, rest) + (me >> 3);
  }
  const int64_t begin = range_start(plan, me), end = range_start(plan, me + 1);

  int paths_of = -1;   // sequence whose paths the LDS holds
  int64_t at = begin;
  while (at < end) {
    const int s = sequence_of(w, first, at);
    const int len = clamp_len(w, s);
    const int tiles = tiles_of(w, len);
    const int64_t in_seq = at - (int64_t)first[s] * w.items;
    const int item = (int)(in_seq / tiles);
    const int t0 = (int)(in_seq - (int64_t)item * tiles);
    const int t1 = (int)min((int64_t)tiles, t0 + (end - at));
    at += t1 - t0;
    const int cached = tiles - w.draft_tiles;
    // item = (kv head, [token,] row block)
    const int per_head = w.items / p.kv_heads;
    const int c = item / per_head;
    const int b = item - c * per_head;
    const int token = w.sel_tiles ? b / w.blocks : 0;
    const int row0 = (w.sel_tiles ? b - token * w.blocks : b) * RM;

    const bool has_draft = t1 > cached;
    if (has_draft && p.parents && paths_of != s) {
      __syncthreads();   // the last item's rows have read the table
      build_paths(w, s, paths);
      paths_of = s;
    }

    // this lane's query rows
    int row_token[RT], row_head[RT];
    bool row_ok[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int r = row0 + rt * 16 + li;
      row_ok[rt] = r < w.rows;
      const int rr = row_ok[rt] ? r : 0;
      row_token[rt] = w.sel_tiles ? token : rr / w.group;
      row_head[rt] = c * w.group + (w.sel_tiles ? rr : rr - row_token[rt] * w.group);
    }
    u32x4 q16[F32 ? 1 : NP][RT][KS];
    float q32[F32 ? RT : 1][F32 ? KS : 1][8];
    float mult[RT];   // scores to the base-2 domain
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float x[KS][8];
      const int64_t base = s * p.q_s + row_token[rt] * p.q_n + row_head[rt] * p.q_h;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int d = 32 * ks + 8 * g;
        const bool in = row_ok[rt] && (FULL || d < p.dim);
        load_acts(p.q, base + (in ? d : 0), p.act_type, x[ks]);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[ks][j] = in ? x[ks][j] : 0.0f;
      }
      mult[rt] = w.scale2;
      float up = 1.0f;
      if constexpr (SCALED_Q) {
        float most = 0.0f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int j = 0; j < 8; ++j) most = fmaxf(most, fabsf(x[ks][j]));
        most = max16x32(most);
        // the power of two that brings the largest to [2^14, 2^15)
        int e = (int)((__float_as_uint(most) >> 23) & 255) - 127;
        e = most == 0.0f || e == 128 ? 0 : min(max(14 - e, -126), 126);
        up = __uint_as_float((uint32_t)(e + 127) << 23);
        mult[rt] = w.scale2 * __uint_as_float((uint32_t)(127 - e) << 23);
      }
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        if constexpr (F32) {
#pragma unroll
          for (int j = 0; j < 8; ++j) q32[rt][ks][j] = x[ks][j];
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) x[ks][j] *= up;
          u32x4 parts[NP];
          split8<T, NP>(x[ks], parts);
#pragma unroll
          for (int n = 0; n < NP; ++n) q16[n][rt][ks] = parts[n];
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
        for (int t = 0; t < VD; ++t) o[rt][vc][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    // -- where a cached tile lies (uniform over the wave)
    auto spot = [&](int t) {
      Spot r;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int j = 2 * t + h;
        int col = j >> w.half_shift, pos = 16 * j;
        r.slot[h] = (j & ((1 << w.half_shift) - 1)) * 16;
        bool in = true;
        if (w.sel_tiles) {
          const int rank = col;
          in = rank < p.top;
          const int32_t *list = p.selected + s * p.sel_s + token * p.sel_n + c * p.sel_h;
          const int before = in && rank > 0 ? list[rank - 1] : -1;
          col = in ? list[rank] : 0;
          in = in && col > before && col >= 0 && col < p.width;
          pos = in ? col * p.page_size + r.slot[h] : len;
        }
        in = in && pos < len;
        const int page = in ? p.table[s * p.table_s + col] : 0;
        in = in && page >= 0 && page < p.pages;
        r.page[h] = in ? page : 0;
        r.valid[h] = in ? min(len - pos, 16) : 0;
      }
      return r;
    };

    auto load_cached = [&](const Spot &at_, Regs &x) {
      x.draft = -1;
      const T *kp = static_cast<const T *>(p.k_pages), *vp = static_cast<const T *>(p.v_pages);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        x.valid[h] = at_.valid[h];
        const T *kb = kp + (at_.page[h] * p.kp_p + c * p.kp_h + at_.slot[h] * p.kp_t);
        const T *vb = vp + (at_.page[h] * p.vp_p + c * p.vp_h + at_.slot[h] * p.vp_t);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const int d = 32 * ks + 8 * g;
          load_words(kb + (uint32_t)(li * (int)p.kp_t + (FULL || d < p.dim ? d : 0)), x.k[h][ks]);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int vc = 0; vc < VC; ++vc) {
            const int d = 16 * VD * vc + VD * li;
            load_words(vb + (uint32_t)((4 * g + r) * (int)p.vp_t + (FULL || d < p.dim ? d : 0)), x.v[4 * h + r][vc]);
          }
      }
    };

    // new tokens 32 j ..: their k and v rounded to the cache's type
    auto load_new = [&](int j, Regs &x) {
      x.draft = j;
      auto to_words = [&](const float *y, uint32_t *out, int n) {
        for (int e = 0; e < n; ++e)
          if constexpr (F32) out[e] = __float_as_uint(y[e]);
          else if (!(e & 1)) out[e / 2] = pack2<T>(y[e], y[e + 1]);
      };
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        x.valid[h] = min(max(p.draft - (32 * j + 16 * h), 0), 16);
        const int64_t kn = min(32 * j + 16 * h + li, p.draft - 1);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const int d = 32 * ks + 8 * g;
          float y[8];
          load_acts(p.k, s * p.k_s + kn * p.k_n + c * p.k_h + (FULL || d < p.dim ? d : 0), p.act_type, y);
          to_words(y, x.k[h][ks], 8);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int vc = 0; vc < VC; ++vc) {
            const int d = 16 * VD * vc + VD * li;
            const int64_t vn = min(32 * j + 16 * h + 4 * g + r, p.draft - 1);
            float y[VD];
            load_acts(p.v, s * p.v_s + vn * p.v_n + c * p.v_h + (FULL || d < p.dim ? d : 0), p.act_type, y);
            to_words(y, x.v[4 * h + r][vc], VD);
          }
      }
    };

    auto compute = [&](Regs &x) {
      // rows past a dimension's end: whatever was read meets q = 0, which needs it finite
      if constexpr (!FULL) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
          if (32 * ks + 8 * g >= p.dim) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int e = 0; e < Regs::KW; ++e) x.k[h][ks][e] = 0;
          }
      }
      // values behind the last key of a half: whatever they hold (a page's
      // unwritten slots), their weight is 0, which needs them finite
      if (x.valid[0] < 16 || x.valid[1] < 16) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (4 * g + (j & 3) >= x.valid[j >> 2]) {
#pragma unroll
            for (int vc = 0; vc < VC; ++vc)
#pragma unroll
              for (int e = 0; e < Regs::VW; ++e) x.v[j][vc][e] = 0;
          }
      }
      uint32_t see[RT];   // which of the tile's keys this lane's rows attend to
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const uint32_t there = ((1u << x.valid[0]) - 1) | ((1u << x.valid[1]) - 1) << 16;
        see[rt] = there;
        if (x.draft >= 0) {
          const int i = row_token[rt] - 32 * x.draft;   // chain: the tokens up to its own
          see[rt] &= p.parents ? paths.bits[row_token[rt]][x.draft]
                               : (i < 0 ? 0u : i >= 31 ? ~0u : (2u << i) - 1);
        }
      }
      // a new token's value that is not finite must not reach rows that do not
      // attend to it through 0 * inf: it is taken out of the product here and
      // added by hand below
      uint32_t odd = 0;   // keys of this lane's group with such a value
      if (x.draft >= 0) {
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

#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        f32x4 sc[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          sc[h] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
          if constexpr (F32) {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
              for (int j = 0; j < 8; ++j)
                sc[h] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(x.k[h][ks][j]), q32[rt][ks][j], sc[h], 0, 0, 0);
          } else {
#pragma unroll
            for (int n = NP - 1; n >= 0; --n)
#pragma unroll
              for (int ks = 0; ks < KS; ++ks) {
                const u32x4 a = {x.k[h][ks][0], x.k[h][ks][1], x.k[h][ks][2], x.k[h][ks][3]};
                sc[h] = Cache<CT>::mma(a, q16[n][rt][ks], sc[h]);
              }
          }
        }
        // the running softmax of this lane's row (the four lane groups of a row agree on m)
        float pr[8], most = -INFINITY;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const bool on = see[rt] >> (16 * (j >> 2) + 4 * g + (j & 3)) & 1;
          pr[j] = on ? sc[j >> 2][j & 3] * mult[rt] : -INFINITY;
          most = fmaxf(most, pr[j]);
        }
        const float m_new = fmaxf(m[rt], max16x32(most));
        const float zero = m_new == -INFINITY ? 0.0f : m_new;   // nothing seen yet: every weight is 0
        const float shrink = __builtin_amdgcn_exp2f(m[rt] - zero);
        m[rt] = m_new;
        l[rt] *= shrink;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          pr[j] = __builtin_amdgcn_exp2f(pr[j] - zero + (SCALED_P ? kWeightExp : 0.0f));
          l[rt] += pr[j];
        }
        if (__any(shrink != 1.0f)) {
#pragma unroll
          for (int vc = 0; vc < VC; ++vc)
#pragma unroll
            for (int t = 0; t < VD; ++t) o[rt][vc][t] *= shrink;
        }
        if constexpr (F32) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int vc = 0; vc < VC; ++vc)
#pragma unroll
              for (int t = 0; t < VD; ++t)
                o[rt][vc][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(x.v[j][vc][t]), pr[j], o[rt][vc][t], 0, 0, 0);
        } else {
          u32x4 parts[NP];
          split8<T, NP>(pr, parts);
#pragma unroll
          for (int vc = 0; vc < VC; ++vc)
#pragma unroll
            for (int t = 0; t < VD; ++t) {
              u32x4 a;   // 8 keys of dimension t
#pragma unroll
              for (int e = 0; e < 4; ++e)
                a[e] = __builtin_amdgcn_perm(x.v[2 * e + 1][vc][t / 2], x.v[2 * e][vc][t / 2],
                                             t & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
              for (int n = NP - 1; n >= 0; --n) o[rt][vc][t] = Cache<CT>::mma(a, parts[n], o[rt][vc][t]);
            }
        }
        if (x.draft >= 0 && __any(odd != 0)) {
          for (int key = 0; key < 32; ++key) {   // rare: the values taken out, by hand
            const int j = 4 * (key >> 4) + (key & 3), from = (key & 15) >> 2;
            if (!__any(g == from && (odd >> j & 1))) continue;
            float mine = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) mine = e == j ? pr[e] : mine;
            const float weight = __shfl(mine, li + 16 * from);
            const bool on = see[rt] >> key & 1;
            const int64_t vn = min(32 * x.draft + key, p.draft - 1);
            for (int vc = 0; vc < VC; ++vc)
#pragma unroll
              for (int t = 0; t < VD; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                  const int d = 16 * VD * vc + VD * (4 * g + r) + t;
                  if (d < p.dim && on) {
                    const float y = (float)(T)load_act(p.v, s * p.v_s + vn * p.v_n + c * p.v_h + d, p.act_type);
                    if (!(fabsf(y) < INFINITY)) {
#pragma unroll
                      for (int vv = 0; vv < VC; ++vv)
                        if (vv == vc) o[rt][vv][t][r] += weight * y;
                    }
                  }
                }
          }
        }
      }
    };

    for (int t = t0 + wave; t < t1; t += kWaves) {
      Regs x;
      if (t < cached) {
        const Spot here = spot(t);
        if ((here.valid[0] | here.valid[1]) == 0) continue;
        load_cached(here, x);
      } else {
        load_new(t - cached, x);
      }
      compute(x);
    }

    // -- the four waves' parts joined, in wave order
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      l[rt] = sum16x32(l[rt]);
      // an unused token's rows: marked by l = -1 in the part that holds its tile
      if (has_draft && p.parents && wave == 0 && paths.next[row_token[rt]] == -2) l[rt] = -1.0f;
    }
    auto put = [&](int to) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
        for (int vc = 0; vc < VC; ++vc)
#pragma unroll
          for (int t = 0; t < VD; ++t) o_share[to][rt][vc * VD + t][lane] = o[rt][vc][t];
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
          for (int t = 0; t < VD; ++t) o[rt][vc][t] = o[rt][vc][t] * a + o_share[from][rt][vc * VD + t][lane] * b2;
      }
    };
    if (wave >= 2) put(wave - 2);
    __syncthreads();
    if (wave < 2) join(wave);
    __syncthreads();
    if (wave == 1) put(0);
    __syncthreads();
    if (wave == 0) {
      join(0);
      const bool whole = t0 == 0 && t1 == tiles;
      // (t0 > 0: this range's first part; else its last)
      const int64_t slot = 2 * (int64_t)me + (t0 > 0 ? 0 : 1);
      float *part = w.part + slot * RM * DT;
      float *stats = w.part + 2 * (int64_t)w.grid * RM * DT + slot * RM * 2;
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        if (!row_ok[rt]) continue;
        if (!whole && g == 0) {
          stats[2 * (rt * 16 + li)] = m[rt];
          stats[2 * (rt * 16 + li) + 1] = l[rt];
        }
        const float norm = l[rt] < 0.0f ? 0.0f : 1.0f / l[rt];
        const int64_t out = s * p.o_s + row_token[rt] * p.o_n + row_head[rt] * p.o_h;
#pragma unroll
        for (int vc = 0; vc < VC; ++vc)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int d = 16 * VD * vc + VD * (4 * g + r);
            if (!FULL && d >= p.dim) continue;
            float y[VD];
#pragma unroll
            for (int t = 0; t < VD; ++t) y[t] = o[rt][vc][t][r];
            if (!whole) {
#pragma unroll
              for (int t = 0; t < VD; t += 4)
                *reinterpret_cast<f32x4 *>(part + (rt * 16 + li) * DT + d + t) = f32x4{y[t], y[t + 1], y[t + 2], y[t + 3]};
              continue;
            }
#pragma unroll
            for (int t = 0; t < VD; ++t) y[t] = l[rt] < 0.0f ? 0.0f : y[t] * norm;
            if (p.act_type == KH_TYPE_F32) {
#pragma unroll
              for (int t = 0; t < VD; t += 4)
                *reinterpret_cast<f32x4 *>(static_cast<float *>(p.out) + out + d + t) = f32x4{y[t], y[t + 1], y[t + 2], y[t + 3]};
            } else {
#pragma unroll
              for (int t = 0; t < VD; t += 4) {
                u32x2 pair;
                if (p.act_type == KH_TYPE_BF16) pair = u32x2{pack2<__bf16>(y[t], y[t + 1]), pack2<__bf16>(y[t + 2], y[t + 3])};
                else pair = u32x2{pack2<_Float16>(y[t], y[t + 1]), pack2<_Float16>(y[t + 2], y[t + 3])};
                *reinterpret_cast<u32x2 *>(static_cast<uint16_t *>(p.out) + out + d + t) = pair;
              }
            }
          }
      }
    }
    __syncthreads();   // the shared parts are free again
  }
}

// The parts of the items that more than one range touched, joined: one wave
// per row, two passes over the parts (the largest maximum, then the weighted
// sum in range order).
template <int DT, int RT>
__global__ __launch_bounds__(kThreads) void paged_join_kernel(const PagedWork w) {
  constexpr int RM = 16 * RT;
  constexpr int PER = DT / 64;   // dimensions of a lane
  __shared__ int first[kMaxBatch + 1];
  __shared__ int wave_sums[kWaves];
  const kh_paged &p = w.p;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  scan_tiles(w, first, wave_sums);
  const Plan plan = plan_of(w, first);
  const int s = blockIdx.x / w.items, item = blockIdx.x - s * w.items;
  const int tiles = tiles_of(w, clamp_len(w, s));
  const int64_t x = (int64_t)first[s] * w.items + (int64_t)item * tiles;
  const int64_t w0 = range_of(plan, x), w1 = range_of(plan, x + tiles - 1);
  if (w0 == w1) return;   // finished by its one range
  const int per_head = w.items / p.kv_heads;
  const int c = item / per_head, b = item - c * per_head;
  const int token = w.sel_tiles ? b / w.blocks : 0;
  const int row0 = (w.sel_tiles ? b - token * w.blocks : b) * RM;
  const int r = blockIdx.y * kWaves + wave;
  if (row0 + r >= w.rows || r >= RM) return;
  const int n = w.sel_tiles ? token : (row0 + r) / w.group;
  const int head = c * w.group + (w.sel_tiles ? row0 + r : row0 + r - n * w.group);
  const float *stats = w.part + 2 * (int64_t)w.grid * RM * DT + 2 * r;
  // part i of the item: the last part of range w0, then the first of the others
  auto slot = [&](int64_t i) { return 2 * (w0 + i) + (i == 0 ? 1 : 0); };
  const int64_t count = w1 - w0 + 1;
  float m = -INFINITY;
  bool unused = false;
  for (int64_t i = lane; i < count; i += 64) {
    m = fmaxf(m, stats[slot(i) * RM * 2]);
    unused |= stats[slot(i) * RM * 2 + 1] < 0.0f;
  }
  m = wave_max(m);
  unused = __any(unused);
  if (m == -INFINITY) m = 0.0f;
  float l = 0.0f, o[PER];
#pragma unroll
  for (int e = 0; e < PER; ++e) o[e] = 0.0f;
#pragma unroll 4
  for (int64_t i = 0; i < count; ++i) {
    const int64_t at = slot(i);
    const float a = __builtin_amdgcn_exp2f(stats[at * RM * 2] - m);
    l += a * stats[at * RM * 2 + 1];
    const float *part = w.part + (at * RM + r) * DT + lane * PER;
#pragma unroll
    for (int e = 0; e < PER; ++e) o[e] += lane * PER + e < p.dim ? a * part[e] : 0.0f;
  }
  const float norm = 1.0f / l;
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    const int d = lane * PER + e;
    if (d >= p.dim) continue;
    const float y = unused ? 0.0f : o[e] * norm;
    const int64_t at = s * p.o_s + n * p.o_n + head * p.o_h + d;
    if (p.act_type == KH_TYPE_F32) static_cast<float *>(p.out)[at] = y;
    else if (p.act_type == KH_TYPE_BF16) static_cast<__bf16 *>(p.out)[at] = (__bf16)y;
    else static_cast<_Float16 *>(p.out)[at] = (_Float16)y;
  }
}

template <int CT, int NP, int DT, int RT>
void launch_both(const PagedWork &w, hipStream_t stream) {
  if (w.p.dim == DT) paged_attn_kernel<CT, NP, DT, RT, true><<<w.grid, kThreads, 0, stream>>>(w);
  else paged_attn_kernel<CT, NP, DT, RT, false><<<w.grid, kThreads, 0, stream>>>(w);
  if (w.grid > 1) {
    const dim3 grid((unsigned)(w.p.batch * w.items), (unsigned)((std::min(w.rows, 16 * RT) + kWaves - 1) / kWaves));
    paged_join_kernel<DT, RT><<<grid, kThreads, 0, stream>>>(w);
  }
}

template <int CT, int NP>
hipError_t launch_typed(const PagedWork &w, int dt, int rt, hipStream_t stream) {
  constexpr bool kFour = CT != KH_TYPE_F32 && NP == 1;
  if (dt == 256) launch_both<CT, NP, 256, 1>(w, stream);
  else if (dt == 128) {
    if (rt == 1) launch_both<CT, NP, 128, 1>(w, stream);
    else if (rt == 2 || !kFour) launch_both<CT, NP, 128, 2>(w, stream);
    else if constexpr (kFour) launch_both<CT, NP, 128, 4>(w, stream);
  } else {
    if (rt == 1) launch_both<CT, NP, 64, 1>(w, stream);
    else if (rt == 2 || !kFour) launch_both<CT, NP, 64, 2>(w, stream);
    else if constexpr (kFour) launch_both<CT, NP, 64, 4>(w, stream);
  }
  return hipGetLastError();
}

}  // namespace
}  // namespace kh
