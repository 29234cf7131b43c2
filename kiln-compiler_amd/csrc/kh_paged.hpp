// kh_paged.hpp - shared by the kernels of the paged cache's operators.
#pragma once

#include <string>

#include "kh_common.hpp"
#include "kh_internal.hpp"

namespace kh {

// Checks of a kh_paged's sizes, types and strides (pointers aside); false
// with `err` set, `unsupported` telling a size no kernel is built for from a
// malformed one.
bool check_paged(const kh_paged &p, std::string &err, bool &unsupported);
// ... and of its pointers: null ones, alignment.
bool check_paged_pointers(const kh_paged &p, std::string &err);

size_t paged_workspace_floats(const kh_paged &p);
// Work items of the largest of an attention's launches.
int64_t paged_threads(const kh_paged &p);
hipError_t launch_paged(const kh_paged &p, float *workspace, hipStream_t stream);
size_t select_workspace_floats(const kh_paged &p);
hipError_t launch_select(const kh_paged &p, float *workspace, hipStream_t stream);
void host_paged(const kh_paged &p);
// The operands of a PAGED launch of a plan at the addresses ptrs.
kh_paged paged_of_launch(const kh_launch &L);
void patch_paged(kh_paged &p, const kh_launch &L, float *const *ptrs);

// What the host works out for the kernels.
struct PagedWork {
  kh_paged p;
  int group;       // query heads of a kv head
  int rows;        // query rows of an item's sequence part: draft * group, or group with picked pages
  int blocks;      // row blocks of `rows`
  int items;       // items of a sequence: kv_heads * blocks (* draft with picked pages)
  int per_head;    // items of a kv head
  int half_shift;  // page_size = 16 << half_shift
  int tile;        // keys of a tile
  int draft_tiles;
  int sel_tiles;   // tiles of the picked pages, 0 without
  int whole;       // a workgroup per item, no second kernel
  int grid;        // workgroups of the first kernel
  int rounds;      // doublings that cover the longest path
  float scale2;    // scale * log2(e)
  float *part;     // [workgroup][2][16 RT rows][DT], then [workgroup][2][16 RT][2] m and l
};

// The kernels of one cache type (kh_paged_attn.hpp) and number of parts of q and
// of the weights (1 and 1; x3, x2: as many of both; w2: 1 and 2), on dt-wide
// heads and rt blocks of 16 rows.
hipError_t launch_paged_f32(const PagedWork &w, int dt, int rt, hipStream_t stream);
hipError_t launch_paged_bf16(const PagedWork &w, int dt, int rt, hipStream_t stream);
hipError_t launch_paged_bf16w2(const PagedWork &w, int dt, int rt, hipStream_t stream);
hipError_t launch_paged_bf16x3(const PagedWork &w, int dt, int rt, hipStream_t stream);
hipError_t launch_paged_f16(const PagedWork &w, int dt, int rt, hipStream_t stream);
hipError_t launch_paged_f16w2(const PagedWork &w, int dt, int rt, hipStream_t stream);
hipError_t launch_paged_f16x2(const PagedWork &w, int dt, int rt, hipStream_t stream);

constexpr int kPagedTile = 32;     // keys of a tile
constexpr int kWideTile = 64;      // ... of paged_wide_kernel
constexpr int kWideBlocks = 8;     // its rows, in 16s
constexpr int kMaxWideBatch = 1024;
constexpr int kPagedWaves = 4;     // waves of a workgroup
// ... of paged_attn_kernel: eight where it takes whole items and two fit a SIMD
constexpr int paged_waves(int dt, int rt, bool whole) { return whole && rt * dt <= 128 ? 8 : kPagedWaves; }
constexpr int kMaxDraft = 256;     // new tokens of a sequence: a workgroup's table of paths fits the LDS
constexpr int kMaxBatch = 4096;    // sequences of a call: each workgroup scans their lengths

inline int type_bytes(int t) { return t == KH_TYPE_F32 ? 4 : 2; }

}  // namespace kh
