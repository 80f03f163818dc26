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
constexpr int kListMax = 320;

// A range in 64 bits: where its first element lies (48 bits: device addresses are below 2^47), the end of the range inside
// its last tile minus one (12 bits) and its dtype.
constexpr int kListAddrBits = 48, kListTailBits = 12;
constexpr uint64_t list_word(uint64_t addr, uint32_t tail, int dtype) {
  return addr | uint64_t(tail - 1) << kListAddrBits | uint64_t(dtype) << (kListAddrBits + kListTailBits);
}

struct ListArgs {
  int32_t n;                    // ranges
  uint32_t n_tiles;             // of all of them
  uint32_t tile_end[kListMax];  // tiles up to and including this range's
  uint64_t range[kListMax];     // list_word
};
struct ListRef {  // the same in the workspace
  int32_t n;
  uint32_t n_tiles;
  const uint32_t* tile_end;
  const uint64_t* range;
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

// ---- launch shapes, measured on MI355X (random data; times of whole calls) ------------------------------
// Norm: a grid that loops, one partial sum per workgroup (kListNormGrid doubles of the caller's workspace).  Fewer waves
// stream long ranges faster (436 MB in 9 ranges: 65.6 us with 512 workgroups, 68.4 with 1024), but where ranges are
// short, so that a wave needs a new one for almost every tile, twice the waves hide the lookups (1427 ragged tensors,
// 346 MB: 87 us and 68; 64 ranges of 8 MB: 84.7 and 82.4).  Long: at least kListNormLongRange tiles a range on average,
// two strides of the smaller grid (16 ranges of 16 MB: 41.5 and 43.0).
constexpr int kListNormBlock = 256;
constexpr int kListNormGrid = 1024;
constexpr int kListNormLongGrid = 512;
constexpr int kListNormLongRange = 4096;
// One workgroup for the whole call while that is faster than one launch more: norm of 128 tiles 11.8 us against 13.4, of
// 256 tiles 18.6 against 14.0; clipping 64 tiles 11.4 against 13.6, 128 tiles 16.4 against 14.3.
constexpr int kListSmallBlock = 1024;
constexpr int kListSmallNormTiles = 128;
constexpr int kListSmallClipTiles = 96;
// Scaling: one tile per wave and one wave per workgroup (1.74 GB: 570 us; two and four waves per workgroup 605 and 595,
// grids that loop 670).  Up to kListClipTiles tiles a looping grid that also joins the partial sums saves the
// finishing launch: 32 MB 22.5 -> 19.8 us, 134 MB 67.2 -> 67.0, beyond that it loses (268 MB 126 -> 128, 536 MB 246 -> 255).
constexpr int kListScaleBlock = 64;
constexpr int kListClipBlock = 256;
constexpr int kListClipGrid = 1024;
constexpr int kListClipTiles = 32768;
// AdamW: one tile of 256 elements per wave, one wave per workgroup (a layer of 218 M elements, 6.1 GB: 1011 us; tiles
// of 512 and 1024 elements 1038 and 1050; two and four waves per workgroup with tiles of 512 1051 and 1075).
constexpr int kListAdamBlock = 64;
// A wave per tile takes several launches beyond this many workgroups (17 GB of scaling; 1.07 G elements of AdamW): 2^28
// lanes, a sixteenth of the 2^32 that a grid stays below.  Each is 5 ms of work, so the 5 us of one launch more are
// 0.1 %, and lists that need several still fit a card.  (Waves that loop instead cost 0.4-1.5 % at every size.)
constexpr uint32_t kListMaxGrid = 1u << 22;

}  // namespace yafsdp
