// What a list launch works from: the ranges of memory its waves walk, cut into tiles.  Shared by the host packing
// (list_api.hip) and the kernels (list_kernels.hip.h); plain structs, no HIP types.
//
// Up to kListMax (kListAdamMax) ranges travel by value in the kernel arguments (at most 4 KiB per launch).  A longer list
// is first written to the caller's workspace, where the one launch that does the work reads it: by one kernel that
// fetches it from a pinned staging slot (stage_slots.h), or, while a graph is being captured and when every slot is
// still unread, by kernels that carry it in THEIR arguments, 3840 bytes each.  Either way no call waits for another,
// two calls at once share nothing, and a captured graph holds its own list.
#pragma once
#include <stdint.h>

namespace yafsdp {

// ---- norm / scale: one wave per tile of 4 KiB ---------------------------------------------------------
// A range's tiles start at the 128-byte line that holds its first element, so every 16-byte access is aligned and no
// cache line is shared by two tiles of one range.
constexpr int kListTileBytes = 4096;
constexpr int kListMax = 240;

struct ListArgs {
  int32_t n;                    // ranges
  uint32_t n_tiles;             // of all of them
  uint32_t tile_end[kListMax];  // tiles up to and including this range's
  uint32_t tail[kListMax];      // bits 0-12: end of the range inside its last tile (1 .. 4096 bytes); bits 30-31: dtype
  uint64_t addr[kListMax];      // first element
};
struct ListRef {  // the same in the workspace
  int32_t n;
  uint32_t n_tiles;
  const uint32_t* tile_end;
  const uint32_t* tail;
  const uint64_t* addr;
};

// ---- AdamW: one wave per tile of 256 elements ---------------------------------------------------------
// A range's tiles start at the 256-byte boundary below its first parameter (64 elements: whole lines of the 16-bit
// arrays too).  Ranges cut from buffers of one layout have their other arrays at the matching places.
constexpr int kListAdamTile = 256;
constexpr int kListAdamMax = 80;

struct ListAdamRange {
  uint64_t p, g, m, v, out;
};
struct ListAdamArgs {
  int32_t n;
  uint32_t n_tiles;
  uint32_t tile_end[kListAdamMax];
  uint32_t tail[kListAdamMax];  // end of the range inside its last tile (1 .. 256)
  ListAdamRange r[kListAdamMax];
};
struct ListAdamRef {
  int32_t n;
  uint32_t n_tiles;
  const uint32_t* tile_end;
  const uint32_t* tail;
  const ListAdamRange* r;
};

// ---- staging of longer lists --------------------------------------------------------------------------
constexpr int kListStageWords = 960;  // per launch; the workspace holds whole pieces
struct ListStageArgs {
  alignas(16) uint32_t word[kListStageWords];
};
static_assert(sizeof(ListArgs) <= 3856 && sizeof(ListAdamArgs) <= 3856 && sizeof(ListStageArgs) <= 3856,
              "kernel arguments hold at most 4 KiB");

constexpr int kListFetchBlock = 1024;

enum : int { LIST_NORM_1 = 1, LIST_NORM_2 = 2, LIST_NORM_INF = 3 };

constexpr int kListNormBlock = 256;
constexpr int kListNormGrid = 1024;  // = the most partial sums of one call (doubles in the caller's workspace)
constexpr int kListNormLongGrid = 512;
constexpr int kListNormLongRange = 1024;
constexpr int kListSmallBlock = 1024;
constexpr int kListSmallTiles = 128;
constexpr int kListScaleBlock = 64;
constexpr int kListClipBlock = 256;
constexpr int kListClipGrid = 1024;
constexpr int kListClipTiles = 32768;
constexpr int kListAdamBlock = 64;

}  // namespace yafsdp
