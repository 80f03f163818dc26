// C ABI of the list entry points: argument checks, packing of the ranges into launches.  Declarations are in
// include/yafsdp_hip.h.
#include <algorithm>
#include <cstring>
#include <type_traits>
#include <vector>

#include "../../include/yafsdp_hip.h"
#include "adam_scalars.h"
#include "launch.h"
#include "list_args.h"
#include "stage_slots.h"

using namespace yafsdp;

namespace {

struct Span {
  uintptr_t lo, hi;
};
struct Range {
  uintptr_t addr;
  uint64_t bytes;
  int dtype;
};
struct AdamRange {
  uintptr_t p, g, m, v, out;
  uint64_t numel;
};

inline bool valid_dtype(int dt) { return dt == DT_F32 || dt == DT_BF16 || dt == DT_F16; }
inline int item_size(int dt) { return dt == DT_F32 ? 4 : 2; }
inline bool aligned_to(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
// more elements than any address space holds: refused before a size is computed from them
constexpr int64_t kMaxNumel = int64_t(1) << 46;

// Sorts by address; lists usually come in ascending order, which costs one pass.
void sort_spans(std::vector<Span>& s) {
  const auto less = [](const Span& a, const Span& b) { return a.lo < b.lo; };
  if (!std::is_sorted(s.begin(), s.end(), less)) std::sort(s.begin(), s.end(), less);
}
// True if no two of the sorted spans share a byte.
bool disjoint(const std::vector<Span>& s) {
  for (size_t i = 1; i < s.size(); i++)
    if (s[i - 1].hi > s[i].lo) return false;
  return true;
}
// True if one of the sorted disjoint spans shares a byte with the one given.
bool touches(const std::vector<Span>& s, const void* data, size_t bytes) {
  const uintptr_t lo = reinterpret_cast<uintptr_t>(data);
  const auto it = std::lower_bound(s.begin(), s.end(), lo, [](const Span& a, uintptr_t at) { return a.hi <= at; });
  return it != s.end() && it->lo < lo + bytes;
}
// Adds sorted spans to sorted spans.
void merge_spans(std::vector<Span>& into, const std::vector<Span>& s) {
  const size_t mid = into.size();
  into.insert(into.end(), s.begin(), s.end());
  std::inplace_merge(into.begin(), into.begin() + mid, into.end(), [](const Span& a, const Span& b) { return a.lo < b.lo; });
}

// The list as ranges of memory: empty tensors left out, neighbours in memory of one dtype joined.
int collect(const yafsdp_list_entry* entries, int64_t n, std::vector<Range>& out) {
  if (n < 0 || (n > 0 && entries == nullptr)) return YAFSDP_ERR_INVALID_ARGUMENT;
  int last[3] = {-1, -1, -1};  // the newest range of each dtype
  for (int64_t i = 0; i < n; i++) {
    const yafsdp_list_entry& e = entries[i];
    if (!valid_dtype(e.dtype)) return YAFSDP_ERR_UNSUPPORTED_DTYPE;
    if (e.numel < 0 || (e.numel > 0 && e.data == nullptr)) return YAFSDP_ERR_INVALID_ARGUMENT;
    if (e.numel > kMaxNumel) return YAFSDP_ERR_TOO_LARGE;
    if (e.numel == 0) continue;
    const int size = item_size(e.dtype);
    if (!aligned_to(e.data, size)) return YAFSDP_ERR_MISALIGNED;
    const uintptr_t addr = reinterpret_cast<uintptr_t>(e.data);
    const uint64_t bytes = uint64_t(e.numel) * size;
    if (addr >> kListAddrBits != 0) return YAFSDP_ERR_INVALID_ARGUMENT;  // no device address
    int& l = last[e.dtype];
    if (l >= 0 && out[l].addr + out[l].bytes == addr) {
      out[l].bytes += bytes;
      continue;
    }
    l = int(out.size());
    out.push_back(Range{addr, bytes, e.dtype});
  }
  return YAFSDP_OK;
}

// Tiles so far; false when a launch cannot count them.
struct Tiles {
  uint64_t count = 0;
  bool add(uint64_t n) { return (count += n) <= uint64_t(INT32_MAX); }
};

// Where a range ends, and its tiles, counted from the 128-byte line that holds its first element.
uint64_t end_of(const Range& r) { return (r.addr & 127) + r.bytes; }
uint64_t tiles_of(const Range& r) { return (end_of(r) + kListTileBytes - 1) / kListTileBytes; }

// Whether two spans share a byte.
bool share(const Span& a, const Span& b) { return a.lo < b.hi && b.lo < a.hi; }
Span span_of(const void* data, size_t bytes) {
  const uintptr_t lo = reinterpret_cast<uintptr_t>(data);
  return Span{lo, lo + bytes};
}

// The workspace, which every call writes, against the ranges and the scalars; with `written`, the ranges (which are
// rewritten) against each other and against the scalars that the waves read meanwhile.
int check_memory(const std::vector<Range>& ranges, bool written, const float* scalars, int n_scalars,
                 const void* workspace, size_t workspace_bytes) {
  const Span scratch = span_of(workspace, workspace_bytes), scalar = span_of(scalars, n_scalars * sizeof(float));
  bool shared = share(scratch, scalar);
  Tiles tiles;
  std::vector<Span> spans;
  if (written) spans.reserve(ranges.size());
  for (const Range& r : ranges) {
    if (!tiles.add(tiles_of(r))) return YAFSDP_ERR_TOO_LARGE;
    const Span s{r.addr, r.addr + r.bytes};
    shared |= share(s, scratch);
    if (!written) continue;
    shared |= share(s, scalar);
    spans.push_back(s);
  }
  if (shared) return YAFSDP_ERR_OVERLAP;
  sort_spans(spans);
  return disjoint(spans) ? YAFSDP_OK : YAFSDP_ERR_OVERLAP;
}

// workgroups of `block` lanes, one wave per tile, at most `cap`
int grid_of(uint32_t n_tiles, int block, int cap) {
  const int per = block / 64;
  return int(std::min((int64_t(n_tiles) + per - 1) / per, int64_t(cap)));
}

constexpr size_t kPartialBytes = size_t(kListNormGrid) * sizeof(double);
constexpr size_t kAdamRecordWords = sizeof(ListAdamRange) / sizeof(uint32_t);
static_assert((kAdamRecordWords + 2) % 4 == 0, "whole 16-byte vectors");

// 32-bit words of a staged list of n ranges: whole 16-byte vectors.
size_t list_words(size_t n) { return (3 * n + 3) / 4 * 4; }
size_t adam_words(size_t n) { return (kAdamRecordWords + 2) * n; }

// Bytes of `words` 32-bit words in the workspace: whole pieces of kListStageWords.
size_t staged_bytes(size_t words) {
  return (words + kListStageWords - 1) / kListStageWords * kListStageWords * sizeof(uint32_t);
}

// The process's staging slots (never freed: kernels may read them until the end).
StageSlots& slots() {
  static StageSlots* s = new StageSlots;
  return *s;
}
// False without pinned memory; allocated at the first call.  Call with the slots' mutex held.
bool have_slots(StageSlots& s) {
  static bool tried = false;
  if (!tried) {
    tried = true;
    // an allocation is not part of anybody's graph capture
    hipStreamCaptureMode mode = hipStreamCaptureModeRelaxed;
    const bool exchanged = hipThreadExchangeStreamCaptureMode(&mode) == hipSuccess;
    void* block = nullptr;
    if (hipHostMalloc(&block, StageSlots::kBlockBytes, hipHostMallocPortable | hipHostMallocMapped | hipHostMallocCoherent) ==
        hipSuccess)
      s.attach(block);
    else
      (void)hipGetLastError();  // without pinned memory the other route serves
    if (exchanged) (void)hipThreadExchangeStreamCaptureMode(&mode);
  }
  return s.attached();
}

bool capturing(hipStream_t stream) {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(stream, &status) != hipSuccess) {
    (void)hipGetLastError();
    return true;
  }
  return status != hipStreamCaptureStatusNone;
}

// Sends `words` (a multiple of 4) to the workspace: one launch through a staging slot, or a launch per kListStageWords.
// What a captured graph replays has to be in the graph itself, so a capture always takes the second route.
int stage(const std::vector<uint32_t>& words, void* dst, hipStream_t stream) {
  const size_t bytes = words.size() * sizeof(uint32_t);
  if (!capturing(stream)) {
    StageSlots& s = slots();
    int slot = -1;
    uint32_t number = 0;
    {
      std::lock_guard<std::mutex> lock(s.mutex);
      if (have_slots(s)) slot = s.claim(bytes, &number);
    }
    if (slot >= 0) {
      std::memcpy(s.data(slot), words.data(), bytes);
      const hipError_t e = launch_list_fetch(s.data(slot), dst, uint32_t(bytes / 16),
                                             reinterpret_cast<uint32_t*>(s.done(slot)), number, StageSlots::pieces(bytes),
                                             stream);
      if (e == hipSuccess) return YAFSDP_OK;
      std::lock_guard<std::mutex> lock(s.mutex);
      s.abandon(slot);
      return int(e);
    }
  }
  ListStageArgs a{};
  for (size_t i = 0; i < words.size(); i += kListStageWords) {
    std::copy_n(words.data() + i, std::min(words.size() - i, size_t(kListStageWords)), a.word);
    const hipError_t e = launch_list_stage(a, static_cast<uint32_t*>(dst) + i, stream);
    if (e != hipSuccess) return int(e);
  }
  return YAFSDP_OK;
}
static_assert(StageSlots::kPieceBytes == size_t(kListFetchBlock) * 16, "a workgroup reads a piece");

// What the kernels know of range r.
bool cut(const Range& r, Tiles& tiles, uint32_t* tile_end, uint64_t* word) {
  const uint64_t n = tiles_of(r);
  if (!tiles.add(n)) return false;
  *tile_end = uint32_t(tiles.count);
  *word = list_word(r.addr, uint32_t(end_of(r) - (n - 1) * kListTileBytes), r.dtype);
  return true;
}
static_assert(kListTileBytes == 1 << kListTailBits, "the end inside a tile, minus one, has kListTailBits bits");

int pack(const std::vector<Range>& ranges, ListArgs& a) {
  Tiles tiles;
  a.n = int32_t(ranges.size());
  for (int k = 0; k < a.n; k++)
    if (!cut(ranges[k], tiles, &a.tile_end[k], &a.range[k])) return YAFSDP_ERR_TOO_LARGE;
  a.n_tiles = uint32_t(tiles.count);
  return YAFSDP_OK;
}

// The list behind the partial sums of the workspace: the ranges, then where their tiles end.
int pack_and_stage(const std::vector<Range>& ranges, void* workspace, hipStream_t stream, ListRef& a) {
  const size_t n = ranges.size();
  std::vector<uint32_t> words(list_words(n));
  Tiles tiles;
  for (size_t k = 0; k < n; k++) {
    uint64_t word;
    if (!cut(ranges[k], tiles, &words[2 * n + k], &word)) return YAFSDP_ERR_TOO_LARGE;
    std::memcpy(&words[2 * k], &word, sizeof(word));
  }
  uint32_t* base = reinterpret_cast<uint32_t*>(static_cast<char*>(workspace) + kPartialBytes);
  a = ListRef{int32_t(n), uint32_t(tiles.count), base + 2 * n, reinterpret_cast<const uint64_t*>(base)};
  return stage(words, base, stream);
}

// f(meta) with the list in the kernel arguments or, where it is too long for them, in the workspace
template <class F>
int with_list(const std::vector<Range>& ranges, void* workspace, hipStream_t stream, F f) {
  if (ranges.size() <= size_t(kListMax)) {
    ListArgs a;
    const int rc = pack(ranges, a);
    return rc != YAFSDP_OK ? rc : f(a);
  }
  ListRef a;
  const int rc = pack_and_stage(ranges, workspace, stream, a);
  return rc != YAFSDP_OK ? rc : f(a);
}

template <class META>
int norm_or_clip_launches(const META& a, int norm, float max_norm, double* partials, float* norm_and_coef, bool clip,
                          hipStream_t stream) {
  const bool long_ranges = a.n_tiles / uint32_t(a.n) >= uint32_t(kListNormLongRange);
  const int count = grid_of(a.n_tiles, kListNormBlock, long_ranges ? kListNormLongGrid : kListNormGrid);
  hipError_t e = launch_list_norm(norm, a, partials, count, stream);
  if (e != hipSuccess) return int(e);
  if (clip && a.n_tiles <= uint32_t(kListClipTiles))
    return int(launch_list_clip(norm, a, partials, count, max_norm, norm_and_coef,
                                grid_of(a.n_tiles, kListClipBlock, kListClipGrid), stream));
  e = launch_list_finish(norm, partials, count, max_norm, norm_and_coef, stream);
  if (e != hipSuccess || !clip) return int(e);
  return int(launch_list_scale(a, norm_and_coef + 1, stream));
}

int norm_or_clip(const yafsdp_list_entry* entries, int64_t n, int norm, double max_norm, void* workspace,
                 size_t workspace_bytes, float* norm_and_coef, hipStream_t stream, bool clip) {
  if (norm != LIST_NORM_1 && norm != LIST_NORM_2 && norm != LIST_NORM_INF) return YAFSDP_ERR_INVALID_ARGUMENT;
  const size_t need = yafsdp_list_workspace_bytes(n);
  if (n < 0 || workspace == nullptr || norm_and_coef == nullptr || workspace_bytes < need)
    return YAFSDP_ERR_INVALID_ARGUMENT;
  if (!aligned_to(workspace, 16) || !aligned_to(norm_and_coef, 4)) return YAFSDP_ERR_MISALIGNED;
  std::vector<Range> ranges;
  int rc = collect(entries, n, ranges);
  if (rc == YAFSDP_OK) rc = check_memory(ranges, clip, norm_and_coef, 2, workspace, need);
  if (rc != YAFSDP_OK) return rc;
  return with_list(ranges, workspace, stream, [&](const auto& a) {
    if constexpr (std::is_same<std::decay_t<decltype(a)>, ListArgs>::value)
      if (a.n_tiles <= uint32_t(clip ? kListSmallClipTiles : kListSmallNormTiles))
        return int(launch_list_small(norm, clip, a, static_cast<float>(max_norm), norm_and_coef, stream));
    return norm_or_clip_launches(a, norm, static_cast<float>(max_norm), static_cast<double*>(workspace), norm_and_coef,
                                 clip, stream);
  });
}

}  // namespace

extern "C" {

size_t yafsdp_list_workspace_bytes(int64_t n) {
  return kPartialBytes + (n > kListMax ? staged_bytes(list_words(size_t(n))) : 0);
}

size_t yafsdp_list_adamw_workspace_bytes(int64_t n) {
  return n > kListAdamMax ? staged_bytes(adam_words(size_t(n))) : 0;
}

int yafsdp_list_norm(const yafsdp_list_entry* entries, int64_t n, int norm, double max_norm, void* workspace,
                     size_t workspace_bytes, float* norm_and_coef, void* stream) try {
  return norm_or_clip(entries, n, norm, max_norm, workspace, workspace_bytes, norm_and_coef,
                      static_cast<hipStream_t>(stream), false);
} catch (...) {
  return YAFSDP_ERR_OUT_OF_MEMORY;
}

int yafsdp_list_clip(const yafsdp_list_entry* entries, int64_t n, int norm, double max_norm, void* workspace,
                     size_t workspace_bytes, float* norm_and_coef, void* stream) try {
  return norm_or_clip(entries, n, norm, max_norm, workspace, workspace_bytes, norm_and_coef,
                      static_cast<hipStream_t>(stream), true);
} catch (...) {
  return YAFSDP_ERR_OUT_OF_MEMORY;
}

int yafsdp_list_scale(const yafsdp_list_entry* entries, int64_t n, const float* coef, void* workspace,
                      size_t workspace_bytes, void* stream_) try {
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  const size_t need = yafsdp_list_workspace_bytes(n);
  if (n < 0 || coef == nullptr || workspace == nullptr || workspace_bytes < need) return YAFSDP_ERR_INVALID_ARGUMENT;
  if (!aligned_to(coef, 4) || !aligned_to(workspace, 16)) return YAFSDP_ERR_MISALIGNED;
  std::vector<Range> ranges;
  int rc = collect(entries, n, ranges);
  if (rc == YAFSDP_OK) rc = check_memory(ranges, true, coef, 1, workspace, need);
  if (rc != YAFSDP_OK || ranges.empty()) return rc;
  return with_list(ranges, workspace, stream, [&](const auto& a) {
    return int(launch_list_scale(a, coef, stream));
  });
} catch (...) {
  return YAFSDP_ERR_OUT_OF_MEMORY;
}

int yafsdp_list_adamw(const yafsdp_adamw_entry* entries, int64_t n, int grad_dtype, int out16_dtype, double lr,
                      double beta1, double beta2, double eps, double weight_decay, int64_t step,
                      const float* grad_scale, int flags, void* workspace, size_t workspace_bytes,
                      void* stream_) try {
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  if (n < 0 || step < 1 || (n > 0 && entries == nullptr)) return YAFSDP_ERR_INVALID_ARGUMENT;
  const size_t need = yafsdp_list_adamw_workspace_bytes(n);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return YAFSDP_ERR_INVALID_ARGUMENT;
  if (need > 0 && !aligned_to(workspace, 16)) return YAFSDP_ERR_MISALIGNED;
  // out16_dtype F32: no 16-bit copy
  if (!valid_dtype(grad_dtype) || !valid_dtype(out16_dtype)) return YAFSDP_ERR_UNSUPPORTED_DTYPE;
  if (grad_scale != nullptr && !aligned_to(grad_scale, 4)) return YAFSDP_ERR_MISALIGNED;
  const bool has_out = out16_dtype != DT_F32, zero = (flags & YAFSDP_ADAM_ZERO_GRAD) != 0;
  const uint64_t gsize = uint64_t(item_size(grad_dtype));
  std::vector<AdamRange> ranges;
  for (int64_t i = 0; i < n; i++) {
    const yafsdp_adamw_entry& e = entries[i];
    if (e.numel < 0) return YAFSDP_ERR_INVALID_ARGUMENT;
    if (e.numel > kMaxNumel) return YAFSDP_ERR_TOO_LARGE;
    if (e.numel == 0) continue;
    if (e.param == nullptr || e.grad == nullptr || e.exp_avg == nullptr || e.exp_avg_sq == nullptr ||
        (has_out && e.out16 == nullptr))
      return YAFSDP_ERR_INVALID_ARGUMENT;
    if (!aligned_to(e.param, 4) || !aligned_to(e.exp_avg, 4) || !aligned_to(e.exp_avg_sq, 4) ||
        !aligned_to(e.grad, gsize) || (has_out && !aligned_to(e.out16, 2)))
      return YAFSDP_ERR_MISALIGNED;
    const AdamRange r{reinterpret_cast<uintptr_t>(e.param), reinterpret_cast<uintptr_t>(e.grad),
                      reinterpret_cast<uintptr_t>(e.exp_avg), reinterpret_cast<uintptr_t>(e.exp_avg_sq),
                      has_out ? reinterpret_cast<uintptr_t>(e.out16) : 0, uint64_t(e.numel)};
    if (!ranges.empty()) {  // fragments that follow each other in every buffer are one range
      AdamRange& l = ranges.back();
      if (l.p + 4 * l.numel == r.p && l.g + gsize * l.numel == r.g && l.m + 4 * l.numel == r.m &&
          l.v + 4 * l.numel == r.v && (!has_out || l.out + 2 * l.numel == r.out)) {
        l.numel += r.numel;
        continue;
      }
    }
    ranges.push_back(r);
  }
  // what is written (the workspace too) shares no byte with anything else; gradients that are only read may share theirs
  std::vector<Span> written, spans(ranges.size());
  const auto add = [&](uintptr_t AdamRange::*member, uint64_t size, bool is_written) {
    for (size_t i = 0; i < ranges.size(); i++)
      spans[i] = Span{ranges[i].*member, ranges[i].*member + size * ranges[i].numel};
    sort_spans(spans);
    if (is_written) merge_spans(written, spans);
  };
  if (need > 0) written.push_back(span_of(workspace, need));
  add(&AdamRange::p, 4, true);
  add(&AdamRange::m, 4, true);
  add(&AdamRange::v, 4, true);
  if (has_out) add(&AdamRange::out, 2, true);
  add(&AdamRange::g, gsize, zero);
  if (!disjoint(written)) return YAFSDP_ERR_OVERLAP;
  if (grad_scale != nullptr && touches(written, grad_scale, sizeof(float))) return YAFSDP_ERR_OVERLAP;
  size_t w = 0;
  for (size_t i = 0; i < spans.size() && !zero; i++) {  // the gradients, sorted, against what is written
    while (w < written.size() && written[w].hi <= spans[i].lo) w++;
    if (w < written.size() && written[w].lo < spans[i].hi) return YAFSDP_ERR_OVERLAP;
  }
  if (ranges.empty()) return YAFSDP_OK;
  const AdamScalars s = adam_scalars(lr, beta1, beta2, eps, weight_decay, step, flags);
  const size_t k = ranges.size();
  std::vector<uint32_t> tile_end(k), tail(k);
  Tiles tiles;
  for (size_t i = 0; i < k; i++) {
    const uint64_t end = (ranges[i].p & 255) / 4 + ranges[i].numel, t = (end + kListAdamTile - 1) / kListAdamTile;
    if (!tiles.add(t)) return YAFSDP_ERR_TOO_LARGE;
    tile_end[i] = uint32_t(tiles.count);
    tail[i] = uint32_t(end - (t - 1) * kListAdamTile);
  }
  const uint32_t n_tiles = uint32_t(tiles.count);
  const auto record = [&](size_t i) {
    return ListAdamRange{ranges[i].p, ranges[i].g, ranges[i].m, ranges[i].v, ranges[i].out};
  };
  if (k <= size_t(kListAdamMax)) {
    ListAdamArgs a;
    a.n = int32_t(k);
    a.n_tiles = n_tiles;
    for (size_t i = 0; i < k; i++) {
      a.r[i] = record(i);
      a.tile_end[i] = tile_end[i];
      a.tail[i] = tail[i];
    }
    return int(launch_list_adamw(grad_dtype, out16_dtype, a, s, grad_scale, stream));
  }
  std::vector<uint32_t> words(adam_words(k));
  for (size_t i = 0; i < k; i++) {
    const ListAdamRange r = record(i);
    std::memcpy(&words[kAdamRecordWords * i], &r, sizeof(r));
  }
  std::copy(tile_end.begin(), tile_end.end(), words.begin() + kAdamRecordWords * k);
  std::copy(tail.begin(), tail.end(), words.begin() + (kAdamRecordWords + 1) * k);
  const int rc = stage(words, workspace, stream);
  if (rc != YAFSDP_OK) return rc;
  const uint32_t* base = static_cast<const uint32_t*>(workspace);
  const ListAdamRef a{int32_t(k), n_tiles, base + kAdamRecordWords * k, base + (kAdamRecordWords + 1) * k,
                      static_cast<const ListAdamRange*>(workspace)};
  return int(launch_list_adamw(grad_dtype, out16_dtype, a, s, grad_scale, stream));
} catch (...) {
  return YAFSDP_ERR_OUT_OF_MEMORY;
}

}  // extern "C"
