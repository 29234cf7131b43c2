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

int padded_dim(int d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }

// 16-row blocks of an item: one or two by its rows, what the registers of a
// lane hold beside a tile (a 256-wide head's fill them with one). Many rows over
// a 16-bit cache take paged_wide_kernel: from half as many as its 128, where two
// blocks of 32 would read K and V twice (12 heads of 64, 1000 tokens, 4
// sequences, bf16 under fp32 queries: 64 rows 29.5 us there, 32 rows 31.7 here).
constexpr int kWideRows = 48;

int row_blocks(const kh_paged &p) {
  const int rows = (p.top ? 1 : p.draft) * (p.heads / p.kv_heads);
  const int dt = padded_dim(p.dim);
  if (p.cache_type != KH_TYPE_F32 && dt < 256 && rows >= kWideRows && p.batch <= kMaxWideBatch) return kWideBlocks;
  return rows <= 16 || dt == 256 ? 1 : 2;
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
  w.tile = rm == 16 * kWideBlocks ? kWideTile : kPagedTile;
  w.draft_tiles = (p.draft + w.tile - 1) / w.tile;
  w.sel_tiles = (int)(((int64_t)p.top * p.page_size + w.tile - 1) / w.tile);
  w.rounds = 0;
  while ((1 << w.rounds) < p.draft) ++w.rounds;
  w.scale2 = p.scale * kLog2e;
  const int64_t per_item = (w.sel_tiles ? w.sel_tiles : ((int64_t)p.width * p.page_size + w.tile - 1) / w.tile) + w.draft_tiles;
  const int64_t items = (int64_t)w.items * p.batch;
  // workgroups: one per item where none can have many tiles; else what the
  // chip holds at once, or a tile per wave of the most tiles the table has room for
  const bool eight = rm != 16 * kWideBlocks && paged_waves(padded_dim(p.dim), rm / 16, true) == 8;
  const int64_t most_whole = !eight ? kWholeSlowKeys : 2 * items >= current_device().cus ? kWholeManyKeys : kWholeKeys;
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
    case KH_TYPE_BF16:
      return (p.one_pass ? launch_paged_bf16 : fp32 ? launch_paged_bf16x3 : launch_paged_bf16w2)(w, dt, rt, stream);
    default: return (p.one_pass ? launch_paged_f16 : fp32 ? launch_paged_f16x2 : launch_paged_f16w2)(w, dt, rt, stream);
  }
}

}  // namespace kh
