// kh_paged_attn.hip - how attention over a paged cache (kh_paged_attn.hpp) is
// dealt out: rows of an item, workgroups, workspace.
#include <algorithm>

#include "kh_paged.hpp"

namespace kh {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

// Whole items or ranges. A whole item of n keys takes eight waves about 8 us
// and 9 ns a key whatever else runs, ranges and their join 14 us and the time
// that the chip's loads take: one sequence of 8 heads of 128, bf16, 1000 keys
// 17.7 (whole) and 18.1 us (ranges), 1280 keys 19.7 and 18.2, 2000 keys 26.2
// and 14.3. With an item for half the compute units whole items lose little of
// the chip: 128 items of 1000 keys 20.6 and 27.6 us, of 2000 keys 30.9 and 33.3,
// of 4000 keys 51.3 and 53.3, 512 items of 4000 keys 193 and 194 (fp32
// activations 198 and 194). Four waves (many rows, wide heads) take about twice
// as long a key. The number of keys is that of the table's columns: lengths are
// on the device, so short sequences under a wide table run as ranges.
constexpr int kWholeKeys = 1280, kWholeManyKeys = 4096, kWholeSlowKeys = 1024;

// Over 4-bit pages (paged_mx4_kernel, tiles of 64 keys) the two meet elsewhere. 16
// rows an item, eight waves, bf16, 8 heads of 128: 8 items of 2000 keys 17.7 (whole)
// and 22.7 us (ranges), of 4000 keys 25.5 and 22.2; 128 items of 4000 keys 25.9 and
// 28.6, of 8000 keys 44.2 and 39.4. 32 rows an item, four waves: 256 items of 4000
// keys 45 and 62, of 8000 keys 92 and 103 (heads of 64, eight waves: 62 and 96). Four
// waves and few items (heads of 256 now) as 16 items of 32 rows did: 1000 keys 23.2
// and 30.1, 2000 keys 33.8 and 30.5.
constexpr int kMxWholeKeys = 2560, kMxWholeSlowKeys = 1536, kMxWholeManyKeys = 4096, kMxWholeManyRowsKeys = 8192;

int padded_dim(int d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }

// 16-row blocks of an item: one or two by its rows, what the registers of a
// lane hold beside a tile (a 256-wide head's fill them with one). Many rows over
// a 16-bit cache take paged_wide_kernel: from half as many as its 128, where two
// blocks of 32 would read K and V twice (12 heads of 64, 1000 tokens, 4
// sequences, bf16 under fp32 queries: 64 rows 29.5 us there, 32 rows 31.7 here).
constexpr int kWideRows = 48;
// Over 4-bit pages a row block's own reading of K and V costs little (they are
// small and stay in the L2) and what splits 128 rows' keys much (64 KB of parts a
// range), so paged_wide_kernel is for long ones, rows that fill its blocks, and 16-bit
// activations (its parts of fp32 ones do not fit the registers): 16 sequences of 27
// tokens, 108 rows a head, bf16 4000 keys 91.8 us there and 113 here, 1000 keys 60.3 and
// 50.7; 64 rows a head, 8000 keys, 147 and 109; 108 rows, fp32, 8000 keys 316 and 254; 512
// rows, fp16, 8000 keys 113 and 111, 32768 keys 254 and 335.
constexpr int kMxWideKeys = 4096;

// Keys of an item, at most: the table's or the picked pages', or the window's.
int64_t most_keys(const kh_paged &p) {
  const int64_t keys = (int64_t)(p.top ? p.top : p.width) * p.page_size;
  return p.window ? std::min(keys, (int64_t)p.window + p.sinks) : keys;
}

int row_blocks(const kh_paged &p) {
  const int rows = (p.top ? 1 : p.draft) * (p.heads / p.kv_heads);
  const int dt = padded_dim(p.dim);
  if (p.cache_type == KH_TYPE_MX4) {
    const int filled = (rows + 16 * kWideBlocks - 1) / (16 * kWideBlocks) * 16 * kWideBlocks;
    if (dt < 256 && 4 * rows >= 3 * filled && (p.act_type != KH_TYPE_F32 || p.one_pass) && most_keys(p) > kMxWideKeys && p.batch <= kMaxWideBatch)
      return kWideBlocks;
  } else if (p.cache_type != KH_TYPE_F32 && dt < 256 && rows >= kWideRows && p.batch <= kMaxWideBatch) return kWideBlocks;
  if (rows <= 16 || dt == 256) return 1;
  // items of 32 rows that leave compute units without work are cut into 16: 64 rows of 8
  // heads of 128, 250 keys 11.3 us and 16.1 in 32s, 8000 keys 26.3 and 30.6; of 16 sequences
  // 20.6 and 15.7, 124 and 110
  if (p.cache_type == KH_TYPE_MX4 && (int64_t)p.batch * p.kv_heads * (p.top ? p.draft : 1) * ((rows + 31) / 32) < current_device().cus) return 1;
  return 2;
}

PagedWork work_of(const kh_paged &p) {
  PagedWork w;
  w.p = p;
  w.group = p.heads / p.kv_heads;
  const int rm = 16 * row_blocks(p);
  w.rows = (p.top ? 1 : p.draft) * w.group;
  w.blocks = (w.rows + rm - 1) / rm;
  w.per_head = w.blocks * (p.top ? p.draft : 1);
  w.items = p.kv_heads * w.per_head;
  w.half_shift = 0;
  while ((16 << w.half_shift) < p.page_size) ++w.half_shift;
  w.tile = rm == 16 * kWideBlocks || p.cache_type == KH_TYPE_MX4 ? kWideTile : kPagedTile;
  w.draft_tiles = (p.draft + w.tile - 1) / w.tile;
  w.sel_tiles = (int)(((int64_t)p.top * p.page_size + w.tile - 1) / w.tile);
  w.rounds = 0;
  while ((1 << w.rounds) < p.draft) ++w.rounds;
  w.scale2 = p.scale * kLog2e;
  int64_t cached = ((int64_t)p.width * p.page_size + w.tile - 1) / w.tile;
  // (a window's keys, those before it in its first tile, and the sinks')
  if (p.window) cached = std::min(cached, ((int64_t)p.window + w.tile - 2) / w.tile + 1 + ((int64_t)p.sinks + w.tile - 1) / w.tile);
  const int64_t per_item = (w.sel_tiles ? w.sel_tiles : cached) + w.draft_tiles;
  const int64_t items = (int64_t)w.items * p.batch;
  // workgroups: one per item where none can have many tiles; else what the
  // chip holds at once, or a tile per wave of the most tiles the table has room for
  const bool eight = rm != 16 * kWideBlocks && paged_waves(padded_dim(p.dim), rm / 16, true) == 8;
  const bool many = 2 * items >= current_device().cus;
  const int64_t most_whole = p.cache_type == KH_TYPE_MX4 && rm != 16 * kWideBlocks
                                 ? (many ? (rm == 16 ? kMxWholeManyKeys : kMxWholeManyRowsKeys) : eight ? kMxWholeKeys : kMxWholeSlowKeys)
                             : !eight ? kWholeSlowKeys
                             : many   ? kWholeManyKeys
                                      : kWholeKeys;
  w.whole = per_item * w.tile <= most_whole;
  const bool two = rm == 16 * kWideBlocks || rm * padded_dim(p.dim) <= 16 * 128;   // workgroups of a CU
  const int cap = current_device().cus * (two ? 2 : 1);
  w.grid = (int)(w.whole ? items : std::min<int64_t>((per_item * items + kPagedWaves - 1) / kPagedWaves, cap));
  w.part = nullptr;
  return w;
}

}  // namespace

size_t paged_workspace_floats(const kh_paged &p) {
  const PagedWork w = work_of(p);
  if (w.whole) return 0;
  return 2 * (size_t)w.grid * 16 * row_blocks(p) * (padded_dim(p.dim) + 2);
}

int64_t paged_threads(const kh_paged &p) {
  if (p.batch == 0 || p.draft == 0) return 0;
  const PagedWork w = work_of(p);
  const int rt = row_blocks(p);
  const int waves = rt == kWideBlocks ? kPagedWaves : paged_waves(padded_dim(p.dim), rt, w.whole);
  return (int64_t)p.batch * w.items * 64 * (w.whole ? waves : kPagedWaves);   // (ranges: the join)
}

hipError_t launch_paged(const kh_paged &p, float *workspace, hipStream_t stream) {
  if (p.batch == 0 || p.draft == 0) return hipSuccess;
  PagedWork w = work_of(p);
  w.part = workspace;
  const int dt = padded_dim(p.dim), rt = row_blocks(p);
  const bool fp32 = p.act_type == KH_TYPE_F32;
  switch (p.cache_type) {
    case KH_TYPE_F32: return launch_paged_f32(w, dt, rt, stream);
    case KH_TYPE_MX4:
      return (p.act_type == KH_TYPE_F16 ? launch_paged_mx4x2 : fp32 && !p.one_pass ? launch_paged_mx4x3 : launch_paged_mx4w2)(w, dt, rt, stream);
    case KH_TYPE_BF16:
      return (p.one_pass ? launch_paged_bf16 : fp32 ? launch_paged_bf16x3 : launch_paged_bf16w2)(w, dt, rt, stream);
    default: return (p.one_pass ? launch_paged_f16 : fp32 ? launch_paged_f16x2 : launch_paged_f16w2)(w, dt, rt, stream);
  }
}

}  // namespace kh
