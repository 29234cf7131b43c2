// kh_paged_mx4.hpp - attention over a paged cache in 4 bits (kh_mx4.hpp), few rows
// an item: what paged_attn_kernel (kh_paged_attn.hpp) is to the other caches.
//
// Items, ranges, the products' shapes and the running softmax are as there.
// Codes become bf16 numbers as they are used, exactly, so products are bf16's with
// q and the weights in parts: one and two under bf16 activations, two and two
// under fp16 ones, three and three under fp32 ones. What differs follows from a
// token being 17/64 of the bytes:
//   a tile is 64 keys: the loads of one are as many bytes as a bf16 tile's of 17,
//     and what a tile costs beside its keys - the exchange of maxima, the scalar
//     work of finding its pages - is paid half as often;
//   a lane's loads are 16 bytes: K's 32 dimensions of one key (a block, under one
//     scale), V's 8 dimensions of 4 keys;
//   where a wave's next 16 tiles lie is worked out by its lanes at once, a part
//     of 16 keys each: a scalar load and 64-bit products a tile are what bounded
//     the first version of this kernel;
//   new tokens are rounded once an item, into pages of their own in the LDS.
//
// What it measured (one token, 8 kv heads of 128, 32 query heads, bf16): one
// sequence of 131072 tokens 33 us, 4.3 TB/s of the 5.2 that a copy reaches; 32
// ragged ones up to 8192, 41.5 us, 3.6 TB/s (medians; 31.3 and 38.8 at best). What is missing is beginning and
// ending an item, a chain of dependent loads (length, page, codes) and a join,
// which kMxLead counts. Cached and new tokens' tiles are loops of their own, and
// the cached one always asks for a next tile: while a wave could meet either, the
// wait for this tile's V was one for the next one's K too (39 and 45 us). Two
// tiles in flight a wave, registers for two waves a SIMD alone, and tiles of 32
// keys were slower. Many rows under fp32 activations (27 drafted tokens of 16
// sequences, a window of 1021: 68 us, 17.5 of them products at the matrix cores'
// rate) are bound by one wave a SIMD: three products a pair of operands each way
// and their parts take 400 registers.
#pragma once

#include "kh_paged_attn.hpp"

namespace kh {
namespace {

constexpr int kMxTile = kWideTile;   // keys of a tile: 4 parts of 16

// A tile in a lane's registers. K: codes of the DT / 4 dimensions from DT / 4 g on
// of key 16 h + li, and their blocks' scales; V: codes of 8 dimensions of keys 16 h
// + 4 g .. + 4 (heads of 64: of which this lane uses 4 dimensions, its neighbour
// the others), and the keys' scales, a byte each.
template <int DT>
struct MxTile {
  static constexpr int KS = DT / 32;                      // steps of 32 dimensions (8 a lane)
  static constexpr int VD = DT >= 128 ? 8 : 4;            // adjacent dimensions of a lane's V
  static constexpr int VC = DT / (16 * VD);
  static constexpr int PD = DT / 4;                       // ... of its K
  static constexpr int PW = PD < 32 ? 2 : 4;              // words of one block's share
  static constexpr int PB = PD < 32 ? 1 : PD / 32;        // blocks
  uint32_t k[4][PB][PW], ke[4][PB];
  uint32_t v[4][VC][4], ve[4][VC];
};

// 8 adjacent activations as they lie in memory: asked for early, made floats later.
struct Raw8 {
  u32x4 w[2];
};
__device__ __forceinline__ void load_raw8(const void *p, int64_t i, bool fp32, Raw8 &r) {
  if (fp32) {
#pragma unroll
    for (int j = 0; j < 2; ++j) r.w[j] = *reinterpret_cast<const u32x4 *>(static_cast<const float *>(p) + i + 4 * j);
  } else {
    r.w[0] = *reinterpret_cast<const u32x4 *>(static_cast<const uint16_t *>(p) + i);
  }
}
template <class A>
__device__ __forceinline__ void raw_values(const Raw8 &r, bool fp32, float (&x)[8]) {
  typedef A vec __attribute__((ext_vector_type(8)));
  const vec a = __builtin_bit_cast(vec, r.w[0]);
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = fp32 ? __uint_as_float(r.w[j >> 2][j & 3]) : (float)a[j];
}

// The new tokens of (s, c) into two 4-bit pages in the LDS, rounded as
// kh_cache_append does: a thread takes 8 dimensions of a token (its i-th, of
// draft dim / 8), the 4 lanes of a block agree on its largest.
template <class W>
__device__ __forceinline__ void load_new(W &w, int s, int c, int i, bool act32, Raw8 &k, Raw8 &v) {
  const int chunks = w.p.dim / 8, t = i / chunks, d = (i - t * chunks) * 8;
  load_raw8(w.p.k, s * w.p.k_s + c * w.p.k_h + t * w.p.k_n + d, act32, k);
  load_raw8(w.p.v, s * w.p.v_s + c * w.p.v_h + t * w.p.v_n + d, act32, v);
}
template <class A>
__device__ __forceinline__ void store_new(int dim, int i, int page, uint8_t *keys, bool act32, const Raw8 &k, const Raw8 &v) {
  const int chunks = dim / 8, t = i / chunks, d = (i - t * chunks) * 8;
  uint8_t *values = keys + mx_page_bytes(page, dim);
  float x[8], y[8];
  raw_values<A>(k, act32, x);
  raw_values<A>(v, act32, y);
  const uint32_t ke = mx_scale_of(quad_max(mx_most(x))), ve = mx_scale_of(quad_max(mx_most(y)));
  *reinterpret_cast<uint32_t *>(keys + mx_key_code(t, d, dim)) = mx_pack(x, ke);
  *reinterpret_cast<uint32_t *>(values + mx_value_code(t, d, dim)) = mx_pack(y, ve);
  if (!(d & 31)) {
    keys[mx_key_scale(t, d, dim, page)] = (uint8_t)ke;
    values[mx_value_scale(t, d, dim, page)] = (uint8_t)ve;
  }
}

// WHOLE: a workgroup of eight waves per item; else ranges, four waves.
template <int NQ, int NW, int DT, int RT, bool WHOLE, bool WIN>
__global__ __launch_bounds__(64 * paged_waves(DT, RT, WHOLE), RT * DT > 128 ? 1 : 2) void paged_mx4_kernel(const PagedWork) {
  constexpr int WAVES = paged_waves(DT, RT, WHOLE);
  typedef MxTile<DT> Regs;
  typedef Cache<KH_TYPE_MX4> C;
  typedef std::conditional_t<NQ == 2, _Float16, __bf16> A;   // 16-bit activations
  constexpr int KS = Regs::KS, VD = Regs::VD, VC = Regs::VC, PD = Regs::PD, PW = Regs::PW, PB = Regs::PB;
  constexpr int RM = 16 * RT;
  constexpr int NT = DT / 16;

  __shared__ int first[WHOLE ? 1 : kMaxBatch + 1];
  __shared__ int wave_sums[kWaves];
  __shared__ Paths paths;
  __shared__ f32x4 o_share[WAVES / 2][RT][NT][64];
  __shared__ float ml_share[WAVES / 2][2][RM];
  extern __shared__ __attribute__((aligned(16))) uint8_t new_lds[];   // the new tokens' K and V, a page of each

  const int lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  int me = blockIdx.x, at = 0, end = 1;
  if constexpr (!WHOLE) {
    const_work &w = fresh();
    scan_tiles<WIN, kMxLead>(w, first, wave_sums);
    const Plan plan = plan_of<kMxLead>(w, first);
    if (me >= plan.count) return;
    const int xcd = me & 7, per = plan.count >> 3, rest = plan.count & 7;
    me = xcd * per + min(xcd, rest) + (me >> 3);
    at = range_start(plan, me);
    end = range_start(plan, me + 1);
  }

  int paths_of = -1;   // sequence whose paths the LDS holds
  int new_of = -1;     // (sequence, kv head) whose new tokens
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
      item = (int)((uint32_t)in_seq / (uint32_t)(tiles + kMxLead));
      t0 = in_seq - item * (tiles + kMxLead);
      t1 = min(tiles + kMxLead, t0 + (end - at));
      at += t1 - t0;
      t0 = max(t0 - kMxLead, 0);
      t1 = max(t1 - kMxLead, 0);
      if (t1 == 0) continue;
    }
    const int cached = tiles - w.draft_tiles;
    const Span span = span_of<WIN>(w, len);
    const int c = (int)((uint32_t)item / (uint32_t)w.per_head);
    const int b = item - c * w.per_head;
    const bool sel = w.sel_tiles;
    const int token = sel ? (int)((uint32_t)b / (uint32_t)w.blocks) : 0;
    const int row0 = (sel ? b - token * w.blocks : b) * RM;
    const bool act32 = NQ == 3 || (NQ == 1 && w.p.act_type == KH_TYPE_F32);
    const bool has_draft = WHOLE || t1 > cached;
    const bool tree = w.p.parents != nullptr;
    if ((has_draft || WIN) && tree && paths_of != s) {
      __syncthreads();   // the last item's rows have read the table
      build_paths<WIN>(w, s, len, paths);
      paths_of = s;
    }

    const_work &wt = fresh();
    const int dim = wt.p.dim, page_size = wt.p.page_size, half_shift = wt.half_shift;
    const int new_page = (wt.p.draft + 15) & ~15;
    const uint8_t *kp = static_cast<const uint8_t *>(wt.p.k_pages) + c * wt.p.kp_h, *vp = static_cast<const uint8_t *>(wt.p.v_pages) + c * wt.p.vp_h;

    // this lane's query rows, and its share of the new tokens: asked for before the
    // pages, whose loads wait for the table's
    int row_token[RT], row_head[RT];
    bool row_ok[RT];
    Raw8 q_raw[RT][KS];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int r = row0 + rt * 16 + li;
      row_ok[rt] = r < wt.rows;
      const int rr = row_ok[rt] ? r : 0;
      row_token[rt] = sel ? token : (int)((uint32_t)rr / (uint32_t)wt.group);
      row_head[rt] = c * wt.group + (sel ? rr : rr - row_token[rt] * wt.group);
      const int64_t base = s * wt.p.q_s + row_token[rt] * wt.p.q_n + row_head[rt] * wt.p.q_h;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int d = PD * g + 8 * ks;
        load_raw8(wt.p.q, base + (row_ok[rt] && d < dim ? d : 0), act32, q_raw[rt][ks]);
      }
    }
    const bool make_new = has_draft && new_of != s * wt.p.kv_heads + c;
    const bool mine = make_new && (int)threadIdx.x < wt.p.draft * (dim / 8);
    Raw8 new_k, new_v;
    if (mine) load_new(fresh(), s, c, threadIdx.x, act32, new_k, new_v);

    // where this lane's share of a part lies in it, and of its scales
    constexpr int PAIR = VD == 8 ? 1 : 2;   // lanes of 8 of V's dimensions
    uint32_t k_at[PB], ke_at[PB], v_at[VC], ve_at[VC];
#pragma unroll
    for (int i = 0; i < PB; ++i) {
      const int d = PD * g + 32 * i, in = d < dim ? d : 0;
      k_at[i] = mx_key_code(li, in, dim);
      ke_at[i] = li * (dim / kMxBlock) + in / kMxBlock;
    }
#pragma unroll
    for (int vc = 0; vc < VC; ++vc) {
      const int d = 16 * VD * vc + 8 * (li / PAIR), in = d < dim ? d : 0;
      v_at[vc] = mx_value_code(4 * g, in, dim);
      ve_at[vc] = (g * (dim / kMxBlock) + in / kMxBlock) * 4;
    }

    // -- where tiles lie: lane 4 i + h keeps part h of this wave's i-th tile from `batch` on
    const int last = min(t1, cached);   // cached tiles end here
    int batch = t0 + wave;
    int spot_keys = 0;                  // its keys
    uint64_t spot_k = 0, spot_v = 0;    // its page (none: the first)
    uint64_t some = 0, full = 0;        // parts with keys, with 16 of them
    auto stage = [&] {
      const_work &w = fresh();
      const int t = batch + WAVES * (lane >> 2), h = lane & 3;
      spot_keys = 0;
      int page = 0;
      if (t < last) {
        const int real = t < span.head ? t : t + span.skip, j = 4 * real + h;
        int col = j >> half_shift, pos = 16 * j;
        bool in = true;
        if (sel) {
          const int rank = col;
          in = in && rank < w.p.top;
          const int32_t *list = w.p.selected + (s * w.p.sel_s + token * w.p.sel_n + c * w.p.sel_h);
          const int before = in && rank > 0 ? list[rank - 1] : -1;
          col = in ? list[rank] : 0;
          in = in && col > before && col >= 0 && col < w.p.width;
          pos = in ? col * page_size + (j & ((1 << half_shift) - 1)) * 16 : len;
        }
        in = in && pos < len;
        page = in ? w.p.table[s * w.p.table_s + col] : -1;
        in = in && page >= 0 && page < w.p.pages;
        spot_keys = in ? min(len - pos, 16) : 0;
        page = in ? page : 0;
      }
      spot_k = (uint64_t)(page * w.p.kp_p);
      spot_v = (uint64_t)(page * w.p.vp_p);
      some = __ballot(spot_keys > 0);
      full = __ballot(spot_keys == 16);
    };
    struct Spot {
      int i;       // of the batch
      int t;       // the tile, `last` and more: none
      int real;    // its place in the sequence (a new one's: among the new ones)
      uint32_t keys;   // of its parts, a byte each: 0x10101010 where it has all 64
      uint32_t edge;   // not every row sees the same of its keys
    };
    auto keys_of = [](const Spot &r, int h) { return (int)(r.keys >> (8 * h) & 255u); };
    // the next tile with a key
    auto find = [&](Spot &r, int from) {
      for (;;) {
        const uint64_t left = from < 16 ? some >> (4 * from) : 0;
        if (left) {
          r.i = from + (__builtin_ctzll(left) >> 2);
          r.t = batch + WAVES * r.i;
          r.real = r.t < span.head ? r.t : r.t + span.skip;
          r.edge = WIN && on_edge<WIN>(fresh(), len, kMxTile * r.real, kMxTile);
          r.keys = 0x10101010u;
          if ((full >> (4 * r.i) & 15) != 15) {
            r.keys = 0;
#pragma unroll
            for (int h = 0; h < 4; ++h) r.keys |= (uint32_t)__builtin_amdgcn_readlane(spot_keys, 4 * r.i + h) << (8 * h);
          }
          return;
        }
        batch += 16 * WAVES;
        if (batch >= last) {
          r.t = last;
          r.i = r.real = 0;   // (a page of the pool's all the same)
          return;
        }
        stage();
        from = 0;
      }
    };
    auto lane_of = [&](uint64_t x, int from) {
      return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), from) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)x, from));
    };
    // (a page holds whole parts: rows behind the last key are read too, and masked)
    auto load_k = [&](const Spot &r, Regs &x) {
      int64_t page = 0;
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const int slot = ((4 * r.real + h) & ((1 << half_shift) - 1)) * 16;   // first token of the part in its page
        if (h == 0 || half_shift < 2) page = lane_of(spot_k, 4 * r.i + h);    // (pages of 64 tokens hold the tile)
        const uint8_t *from = kp + (page + slot * (dim / 2)), *e = kp + (page + page_size * (dim / 2) + slot * (dim / kMxBlock));
#pragma unroll
        for (int i = 0; i < PB; ++i) {
          load_words(from + k_at[i], x.k[h][i]);
          x.ke[h][i] = e[ke_at[i]];
        }
      }
    };
    auto load_v = [&](const Spot &r, Regs &x) {
      int64_t page = 0;
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const int slot = ((4 * r.real + h) & ((1 << half_shift) - 1)) * 16;
        if (h == 0 || half_shift < 2) page = lane_of(spot_v, 4 * r.i + h);
        const uint8_t *from = vp + (page + slot * (dim / 2)), *e = vp + (page + page_size * (dim / 2) + slot * (dim / kMxBlock));
#pragma unroll
        for (int vc = 0; vc < VC; ++vc) {
          load_words(from + v_at[vc], x.v[h][vc]);
          x.ve[h][vc] = *reinterpret_cast<const uint32_t *>(e + ve_at[vc]);
        }
      }
    };
    // a tile of new tokens, from the LDS (parts behind the last hold the first's)
    auto load_new_tile = [&](const Spot &r, Regs &x) {
      const uint8_t *values = new_lds + mx_page_bytes(new_page, dim);
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const int slot = keys_of(r, h) ? kMxTile * r.real + 16 * h : 0, code = slot * (dim / 2), scale = new_page * (dim / 2) + slot * (dim / kMxBlock);
#pragma unroll
        for (int i = 0; i < PB; ++i) {
          load_words(new_lds + code + k_at[i], x.k[h][i]);
          x.ke[h][i] = new_lds[scale + ke_at[i]];
        }
#pragma unroll
        for (int vc = 0; vc < VC; ++vc) {
          load_words(values + code + v_at[vc], x.v[h][vc]);
          x.ve[h][vc] = *reinterpret_cast<const uint32_t *>(values + scale + ve_at[vc]);
        }
      }
    };

    Regs x;
    Spot here;
    here.t = last;
    if (batch < last) {
      stage();
      find(here, 0);
    }
    if (here.t < last) {
      load_k(here, x);
      load_v(here, x);
    }
    if (make_new) {
      new_of = s * wt.p.kv_heads + c;
      if (mine) store_new<A>(dim, threadIdx.x, new_page, new_lds, act32, new_k, new_v);
      for (int i = threadIdx.x + blockDim.x; i < wt.p.draft * (dim / 8); i += blockDim.x) {   // (whole groups of 4 lanes)
        load_new(fresh(), s, c, i, act32, new_k, new_v);
        store_new<A>(dim, i, new_page, new_lds, act32, new_k, new_v);
      }
      __syncthreads();
    }

    // the query rows' parts
    u32x4 q[NQ][RT][KS];
    // products to the base-2 domain; positive, so that a masked -inf stays one: q
    // takes a negative scale's sign, or a zero (so that 0 inf is NaN), under which
    // the smallest number does
    const_work &wq = fresh();
    const float mult = fmaxf(fabsf(wq.scale2), 0x1p-126f);
    const float up = wq.scale2 > 0.0f ? 1.0f : wq.scale2 < 0.0f ? -1.0f : wq.scale2;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const bool in = row_ok[rt] && PD * g + 8 * ks < dim;
        float y[8];
        raw_values<A>(q_raw[rt][ks], act32, y);
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = in ? y[j] * up : 0.0f;
        u32x4 parts[NQ];
        split8<__bf16, NQ, true>(y, parts);
#pragma unroll
        for (int n = 0; n < NQ; ++n) q[n][rt][ks] = parts[n];
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

    // A tile's products. The loads of the next one's K go between the first product
    // and the softmax, of its V behind the second: always as many, so that a wait
    // for this tile's V leaves the next one's K in flight.
    auto consume = [&](const Spot &here, auto is_new, auto load_next_k, auto load_next_v) {
      constexpr bool NEW = decltype(is_new)::value;
      f32x4 sc[RT][4];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int h = 0; h < 4; ++h) sc[rt][h] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      // (dimensions beyond dim hold the first block's values, which meet q = 0)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        u32x4 a[4];
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          const uint32_t word = x.k[h][ks / PW][ks % PW];
          const float scale = mx_scale_raw(x.ke[h][ks / PW]);
          a[h] = u32x4{mx_pair<0>(word, scale), mx_pair<1>(word, scale), mx_pair<2>(word, scale), mx_pair<3>(word, scale)};
        }
#pragma unroll
        for (int n = NQ - 1; n >= 0; --n)
#pragma unroll
          for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int h = 0; h < 4; ++h) sc[rt][h] = C::mma(a[h], q[n][rt][ks], sc[rt][h]);
      }
      load_next_k();

      uint32_t odd = 0;        // bit 16 vc + 4 h + i: this lane's V of that key is NaN, and set aside
      uint32_t see[RT][2];
      const bool masked = NEW || (WIN && here.edge);   // rows see different keys
      const bool partly = masked || here.keys != 0x10101010u;
      if (partly) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          const uint32_t there = ((1u << keys_of(here, 2 * kb)) - 1) | ((1u << keys_of(here, 2 * kb + 1)) - 1) << 16;
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) {
            see[rt][kb] = there;
            if constexpr (NEW) {
              const int word = 2 * here.real + kb, i = row_token[rt] - 32 * word;   // chain: the tokens up to its own
              see[rt][kb] &= tree ? (word < kMaxDraft / 32 ? paths.bits[row_token[rt]][word] : 0u) : (i < 0 ? 0u : i >= 31 ? ~0u : (2u << i) - 1);
              if (WIN && !tree) {   // (a tree's bits know the window)
                const_work &w = fresh();
                see[rt][kb] &= window_bits(row_token[rt] - w.p.window + 1, w.p.sinks - len, 32 * word);
              }
            } else if (WIN && here.edge) {
              const_work &w = fresh();
              const int depth = tree ? (int)paths.depth[row_token[rt]] : row_token[rt];
              see[rt][kb] &= window_bits(len - w.p.window + 1 + depth, w.p.sinks, kMxTile * here.real + 32 * kb);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j)
              if (!(see[rt][kb] >> (16 * (j >> 2) + 4 * g + (j & 3)) & 1)) sc[rt][2 * kb + (j >> 2)][j & 3] = -INFINITY;
          }
        }
        // values behind the last key, and new ones or ones that not every row sees,
        // of a block that is NaN: any scale will do for a weight of 0, and NaN is
        // added by hand below
#pragma unroll
        for (int h = 0; h < 4; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int vc = 0; vc < VC; ++vc) {
              const uint32_t e8 = x.ve[h][vc] >> (8 * i) & 255u;
              const bool behind = 4 * g + i >= keys_of(here, h);
              if (e8 > kMxMost && (behind || masked)) {
                x.ve[h][vc] ^= (e8 ^ 127u) << (8 * i);
                if (!behind) odd |= 1u << (16 * vc + 4 * h + i);
              }
            }
      }

      // the running softmax of this lane's rows (the four lane groups of a row agree on m)
      u32x4 parts[RT][2][NW];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        float most = sc[rt][0][0];
#pragma unroll
        for (int j = 1; j < 16; ++j) most = fmaxf(most, sc[rt][j >> 2][j & 3]);
        most = max16x32(most);
        const float m_new = fmaxf(m[rt], most * mult);
        const float zero = m_new == -INFINITY ? 0.0f : m_new;   // nothing seen yet: every weight is 0
        const float shrink = __builtin_amdgcn_exp2f(m[rt] - zero);
        m[rt] = m_new;
        float sum[2] = {0.0f, 0.0f};
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          float pr[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            pr[j] = __builtin_amdgcn_exp2f(fmaf(sc[rt][2 * kb + (j >> 2)][j & 3], mult, -zero));
            sum[kb] += pr[j];
          }
          split_finite<__bf16, NW>(pr, parts[rt][kb]);
        }
        l[rt] = fmaf(l[rt], shrink, sum[0] + sum[1]);
        if (__any(shrink != 1.0f)) {
#pragma unroll
          for (int vc = 0; vc < VC; ++vc)
#pragma unroll
            for (int i = 0; i < VD; ++i) o[rt][vc][i] *= shrink;
        }
      }
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int vc = 0; vc < VC; ++vc)
#pragma unroll
          for (int i0 = 0; i0 < VD; i0 += 4) {
            uint32_t pairs[8][2];   // two dimensions of a key each
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const int h = 2 * kb + (j >> 2), i = j & 3;
              // (the conversion reads bits 23 to 30 alone)
              const uint32_t e = i == 3 ? x.ve[h][vc] >> 1 : x.ve[h][vc] << (23 - 8 * i);
              const float scale = __uint_as_float(e);
              const uint32_t word = x.v[h][vc][i] >> (VD == 8 ? 0 : 16 * (li & 1));
              pairs[j][0] = i0 ? mx_pair<2>(word, scale) : mx_pair<0>(word, scale);
              pairs[j][1] = i0 ? mx_pair<3>(word, scale) : mx_pair<1>(word, scale);
            }
            u32x4 a[4];   // 8 keys of dimensions i0 ..
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                a[i][e] = __builtin_amdgcn_perm(pairs[2 * e + 1][i / 2], pairs[2 * e][i / 2], i & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
            for (int n = NW - 1; n >= 0; --n)
#pragma unroll
              for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) o[rt][vc][i0 + i] = C::mma(a[i], parts[rt][kb][n], o[rt][vc][i0 + i]);
          }
      load_next_v();

      if (__builtin_expect(__any(odd != 0), 0)) {   // the blocks set aside, by hand
        for (int key = 0; key < kMxTile; ++key) {
          const int j = 4 * (key >> 4) + (key & 3), from = (key & 15) >> 2;
          if (!__any(g == from && (odd & (0x00010001u << j)) != 0)) continue;
#pragma unroll
          for (int r = 0; r < 4; ++r) {   // (a row of O^T holds lane 4 g + r's dimensions)
            const uint32_t theirs = (uint32_t)__shfl((int)odd, 4 * g + r + 16 * from);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
              for (int vc = 0; vc < VC; ++vc)
                if ((theirs >> (16 * vc + j) & 1) && (((uint64_t)see[rt][1] << 32 | see[rt][0]) >> key & 1)) {
#pragma unroll
                  for (int i = 0; i < VD; ++i) o[rt][vc][i][r] = NAN;
                }
          }
        }
      }
    };
    while (here.t < last) {
      Spot next;
      consume(here, std::false_type(), [&] {
        find(next, here.i + 1);
        load_k(next, x);
      }, [&] { load_v(next, x); });
      here = next;
    }
    if (has_draft) {   // new tokens' tiles of this wave
      for (int t = max(cached, t0) + ((wave - (max(cached, t0) - t0)) & (WAVES - 1)); t < t1; t += WAVES) {
        const_work &w = fresh();
        here.real = t - cached;
        here.keys = 0;
#pragma unroll
        for (int h = 0; h < 4; ++h) here.keys |= (uint32_t)min(max(w.p.draft - (kMxTile * here.real + 16 * h), 0), 16) << (8 * h);
        load_new_tile(here, x);
        consume(here, std::true_type(), [] {}, [] {});
      }
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
            if (act32 || !done) {
#pragma unroll
              for (int i = 0; i < VD; i += 4) *reinterpret_cast<f32x4 *>(to + i) = f32x4{y[i], y[i + 1], y[i + 2], y[i + 3]};
            } else {
#pragma unroll
              for (int i = 0; i < VD; i += 4)
                *reinterpret_cast<u32x2 *>(static_cast<A *>(w.p.out) + out + d + i) = u32x2{pack2<A>(y[i], y[i + 1]), pack2<A>(y[i + 2], y[i + 3])};
            }
          }
      }
    }
    if (!WHOLE && at < end) __syncthreads();   // the shared parts and the new tokens' pages are free again
  }
}

template <int NQ, int NW, int DT, int RT, bool WIN>
void launch_mx4_rows(const PagedWork &w, hipStream_t stream) {
  const unsigned lds = 2 * (unsigned)mx_page_bytes((w.p.draft + 15) & ~15, w.p.dim);   // the new tokens
  if (w.whole) {
    paged_mx4_kernel<NQ, NW, DT, RT, true, WIN><<<w.grid, 64 * paged_waves(DT, RT, true), lds, stream>>>(w);
  } else {
    paged_mx4_kernel<NQ, NW, DT, RT, false, WIN><<<w.grid, kThreads, lds, stream>>>(w);
    const dim3 grid((unsigned)(w.p.batch * w.items), (unsigned)std::min(w.rows, 16 * RT));
    paged_join_kernel<DT, RT, kMxLead><<<grid, kThreads, 0, stream>>>(w);
  }
}

template <int NQ, int NW, bool WIN>
void launch_mx4_sizes(const PagedWork &w, int dt, int rt, hipStream_t stream) {
  if (dt == 256) launch_mx4_rows<NQ, NW, 256, 1, WIN>(w, stream);
  else if (rt == kWideBlocks) {
    if constexpr (NQ < 3) {   // (not under fp32 activations)
      if (dt == 128) launch_wide<KH_TYPE_MX4, NQ, NW, 128, WIN>(w, stream);
      else launch_wide<KH_TYPE_MX4, NQ, NW, 64, WIN>(w, stream);
    }
  } else if (dt == 128) {
    if (rt == 1) launch_mx4_rows<NQ, NW, 128, 1, WIN>(w, stream);
    else launch_mx4_rows<NQ, NW, 128, 2, WIN>(w, stream);
  } else {
    if (rt == 1) launch_mx4_rows<NQ, NW, 64, 1, WIN>(w, stream);
    else launch_mx4_rows<NQ, NW, 64, 2, WIN>(w, stream);
  }
}

template <int NQ, int NW>
hipError_t launch_mx4(const PagedWork &w, int dt, int rt, hipStream_t stream) {
  if (w.p.window) launch_mx4_sizes<NQ, NW, true>(w, dt, rt, stream);
  else launch_mx4_sizes<NQ, NW, false>(w, dt, rt, stream);
  return hipGetLastError();
}

}  // namespace
}  // namespace kh
