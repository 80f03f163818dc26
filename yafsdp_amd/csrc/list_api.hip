// C ABI of the list entry points: argument checks, packing of the ranges into launches.  Declarations are in
// include/yafsdp_hip.h.
#include <algorithm>
#include <new>
#include <vector>

#include "../../include/yafsdp_hip.h"
#include "adam_scalars.h"
#include "launch.h"
#include "list_args.h"

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

// True if no two spans share a byte.  Lists usually come in ascending order (or nearly), which costs one pass.
bool disjoint(std::vector<Span>& s) {
  bool ascending = true;
  for (size_t i = 1; i < s.size() && ascending; i++) ascending = s[i - 1].hi <= s[i].lo;
  if (ascending) return true;
  std::sort(s.begin(), s.end(), [](const Span& a, const Span& b) { return a.lo < b.lo; });
  for (size_t i = 1; i < s.size(); i++)
    if (s[i - 1].hi > s[i].lo) return false;
  return true;
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

int check_disjoint(const std::vector<Range>& ranges) {
  std::vector<Span> spans;
  spans.reserve(ranges.size());
  for (const Range& r : ranges) spans.push_back(Span{r.addr, r.addr + r.bytes});
  return disjoint(spans) ? YAFSDP_OK : YAFSDP_ERR_OVERLAP;
}

// One launch's arguments from ranges [first, first + a.n); returns the first range of the next launch.
int pack(const std::vector<Range>& ranges, size_t first, ListArgs& a, size_t* next) {
  uint64_t tiles = 0;
  size_t i = first;
  a.n = 0;
  for (; i < ranges.size() && a.n < kListMax; i++) {
    const Range& r = ranges[i];
    const uint64_t end = (r.addr & 127) + r.bytes;  // counted from the line that holds the first element
    const uint64_t n = (end + kListTileBytes - 1) / kListTileBytes;
    if (tiles + n > uint64_t(INT32_MAX)) {
      if (a.n == 0) return YAFSDP_ERR_TOO_LARGE;
      break;
    }
    tiles += n;
    const uint32_t tail = uint32_t(end - (n - 1) * kListTileBytes);
    a.r[a.n++] = ListRange{r.addr, uint32_t(tiles), tail | uint32_t(r.dtype) << 30};
  }
  a.n_tiles = uint32_t(tiles);
  *next = i;
  return YAFSDP_OK;
}

int grid_of(uint32_t n_tiles, int cap) {
  const int per = kListBlock / 64;
  const int64_t g = (int64_t(n_tiles) + per - 1) / per;
  return int(g < cap ? g : cap);
}

// The partial sums of every range into the workspace; *count receives how many.
int norm_launches(const std::vector<Range>& ranges, int norm, double* partials, int* count, hipStream_t stream) {
  const int64_t launches = (int64_t(ranges.size()) + kListMax - 1) / kListMax;
  // (a launch of fewer ranges for the sake of its tile count happens beyond 8 TB only; it is refused below)
  int64_t cap = launches > 0 ? kListMaxPartials / launches : 0;
  if (launches > 0 && cap < 1) return YAFSDP_ERR_TOO_LARGE;
  cap = std::min<int64_t>(cap, kListGrid);
  *count = 0;
  ListArgs a;
  for (size_t i = 0; i < ranges.size();) {
    const int rc = pack(ranges, i, a, &i);
    if (rc != YAFSDP_OK) return rc;
    const int grid = grid_of(a.n_tiles, int(cap));
    if (*count + grid > kListMaxPartials) return YAFSDP_ERR_TOO_LARGE;
    const hipError_t e = launch_list_norm(norm, a, partials + *count, grid, stream);
    if (e != hipSuccess) return int(e);
    *count += grid;
  }
  return YAFSDP_OK;
}

int scale_launches(const std::vector<Range>& ranges, const float* coef, hipStream_t stream) {
  ListArgs a;
  for (size_t i = 0; i < ranges.size();) {
    const int rc = pack(ranges, i, a, &i);
    if (rc != YAFSDP_OK) return rc;
    const hipError_t e = launch_list_scale(a, coef, grid_of(a.n_tiles, kListGrid), stream);
    if (e != hipSuccess) return int(e);
  }
  return YAFSDP_OK;
}

int norm_or_clip(const yafsdp_list_entry* entries, int64_t n, int norm, double max_norm, void* workspace,
                 size_t workspace_bytes, float* norm_and_coef, hipStream_t stream, bool clip) {
  if (norm != LIST_NORM_1 && norm != LIST_NORM_2 && norm != LIST_NORM_INF) return YAFSDP_ERR_INVALID_ARGUMENT;
  if (workspace == nullptr || norm_and_coef == nullptr || workspace_bytes < yafsdp_list_workspace_bytes())
    return YAFSDP_ERR_INVALID_ARGUMENT;
  if (!aligned_to(workspace, 8) || !aligned_to(norm_and_coef, 4)) return YAFSDP_ERR_MISALIGNED;
  std::vector<Range> ranges;
  int rc = collect(entries, n, ranges);
  if (rc == YAFSDP_OK && clip) rc = check_disjoint(ranges);
  if (rc != YAFSDP_OK) return rc;
  double* partials = static_cast<double*>(workspace);
  int count = 0;
  rc = norm_launches(ranges, norm, partials, &count, stream);
  if (rc != YAFSDP_OK) return rc;
  const hipError_t e = launch_list_finish(norm, partials, count, static_cast<float>(max_norm), norm_and_coef, stream);
  if (e != hipSuccess) return int(e);
  return clip ? scale_launches(ranges, norm_and_coef + 1, stream) : YAFSDP_OK;
}

}  // namespace

extern "C" {

size_t yafsdp_list_workspace_bytes(void) { return size_t(kListMaxPartials) * sizeof(double); }

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

int yafsdp_list_scale(const yafsdp_list_entry* entries, int64_t n, const float* coef, void* stream) try {
  if (coef == nullptr) return YAFSDP_ERR_INVALID_ARGUMENT;
  if (!aligned_to(coef, 4)) return YAFSDP_ERR_MISALIGNED;
  std::vector<Range> ranges;
  int rc = collect(entries, n, ranges);
  if (rc == YAFSDP_OK) rc = check_disjoint(ranges);
  if (rc != YAFSDP_OK) return rc;
  return scale_launches(ranges, coef, static_cast<hipStream_t>(stream));
} catch (...) {
  return YAFSDP_ERR_OUT_OF_MEMORY;
}

int yafsdp_list_adamw(const yafsdp_adamw_entry* entries, int64_t n, int grad_dtype, int out16_dtype, double lr,
                      double beta1, double beta2, double eps, double weight_decay, int64_t step,
                      const float* grad_scale, int flags, void* stream) try {
  if (n < 0 || step < 1 || (n > 0 && entries == nullptr)) return YAFSDP_ERR_INVALID_ARGUMENT;
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
  // what is written shares no byte with anything else; gradients that are only read may share theirs
  std::vector<Span> written, read;
  for (const AdamRange& r : ranges) {
    written.push_back(Span{r.p, r.p + 4 * r.numel});
    (zero ? written : read).push_back(Span{r.g, r.g + gsize * r.numel});
    written.push_back(Span{r.m, r.m + 4 * r.numel});
    written.push_back(Span{r.v, r.v + 4 * r.numel});
    if (has_out) written.push_back(Span{r.out, r.out + 2 * r.numel});
  }
  if (!disjoint(written)) return YAFSDP_ERR_OVERLAP;
  std::sort(written.begin(), written.end(), [](const Span& a, const Span& b) { return a.lo < b.lo; });
  for (const Span& g : read) {
    // the first written span that ends behind the gradient's start
    const auto it = std::upper_bound(written.begin(), written.end(), g.lo,
                                     [](uintptr_t lo, const Span& s) { return lo < s.hi; });
    if (it != written.end() && it->lo < g.hi) return YAFSDP_ERR_OVERLAP;
  }
  const AdamScalars s = adam_scalars(lr, beta1, beta2, eps, weight_decay, step, flags);
  ListAdamArgs a;
  for (size_t i = 0; i < ranges.size();) {
    uint64_t tiles = 0;
    a.n = 0;
    for (; i < ranges.size() && a.n < kListAdamMax; i++) {
      const AdamRange& r = ranges[i];
      const uint64_t k = (r.numel + kListAdamTile - 1) / kListAdamTile;
      if (tiles + k > uint64_t(INT32_MAX)) {
        if (a.n == 0) return YAFSDP_ERR_TOO_LARGE;
        break;
      }
      tiles += k;
      a.r[a.n++] = ListAdamRange{r.p, r.g, r.m, r.v, r.out, uint32_t(tiles),
                                 uint32_t(r.numel - (k - 1) * kListAdamTile)};
    }
    a.n_tiles = uint32_t(tiles);
    const int64_t grid = (int64_t(tiles) + kListBlock / 64 - 1) / (kListBlock / 64);
    const hipError_t e = launch_list_adamw(grad_dtype, out16_dtype, a, s, grad_scale, int(grid),
                                           static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return int(e);
  }
  return YAFSDP_OK;
} catch (...) {
  return YAFSDP_ERR_OUT_OF_MEMORY;
}

}  // extern "C"
