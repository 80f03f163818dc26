// What a list launch carries in its kernel arguments: the ranges of memory its waves walk, cut into tiles.  Shared by
// the host packing (list_api.hip) and the kernels (list_kernels.hip.h); plain structs, no HIP types.
//
// The ranges travel by value (at most 4 KiB of kernel arguments per launch), so a call needs no device-side table, no
// staging copy and no state that outlives it: two calls at once, on any streams, share nothing, and a captured graph
// holds its own copy.  A list of more ranges than fit becomes several launches.
#pragma once
#include <stdint.h>

namespace yafsdp {

// ---- norm / scale: one wave per tile of 4 KiB ---------------------------------------------------------
constexpr int kListTileBytes = 4096;
constexpr int kListMax = 240;  // ranges per launch: 16 bytes each

struct ListRange {
  uint64_t addr;      // first element
  uint32_t tile_end;  // tiles of this launch up to and including this range's
  uint32_t tail;      // bits 0-12: end of the range inside its last tile (1 .. 4096 bytes); bits 30-31: dtype
};
// A range's tiles start at the 128-byte line that holds its first element, so every 16-byte access is aligned and no
// cache line is shared by two tiles of one range.
struct ListArgs {
  int32_t n;         // ranges
  uint32_t n_tiles;  // of all of them
  ListRange r[kListMax];
};
static_assert(sizeof(ListArgs) <= 3856, "kernel arguments hold at most 4 KiB");

// ---- AdamW: one wave per tile of 512 elements ---------------------------------------------------------
constexpr int kListAdamTile = 512;
constexpr int kListAdamMax = 80;  // ranges per launch: 48 bytes each

struct ListAdamRange {
  uint64_t p, g, m, v, out;
  uint32_t tile_end;
  uint32_t tail;  // elements in the last tile (1 .. 512)
};
struct ListAdamArgs {
  int32_t n;
  uint32_t n_tiles;
  ListAdamRange r[kListAdamMax];
};
static_assert(sizeof(ListAdamArgs) <= 3856, "kernel arguments hold at most 4 KiB");

enum : int { LIST_NORM_1 = 1, LIST_NORM_2 = 2, LIST_NORM_INF = 3 };

// partial sums of one call (doubles in the caller's workspace) and workgroups of one launch
constexpr int kListMaxPartials = 8192;
constexpr int kListBlock = 256;
constexpr int kListGrid = 2048;

}  // namespace yafsdp
