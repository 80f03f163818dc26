// Optimizer-side passes over a list of separate tensors: norm (1, 2, inf), scaling by a device-resident coefficient,
// AdamW.  Nothing here is a contraction: all of it is bound by memory.
//
// Work is cut into wave-sized tiles (4 KiB for the norm and the scaling, 256 elements for AdamW); a wave looks the range
// that holds its tile up by a binary search with scalar loads.  (Searching with one vector load and a ballot per 64
// ranges measured slower: from the kernel arguments 97 us against 87 on 1427 tensors, because those are far away, and
// from the workspace 74 against 69, because a vector load queues behind the data's.)
//
// Reached on MI355X (kernel alone, traced): norm of 436 MB of bf16 6.5-6.7 TB/s and of 1.74 GB 7.0 TB/s (a read-only pass 7.2);
// scaling 1.74 GB 6.3 TB/s (a copy 6.36); AdamW of 218 M elements 6.05 TB/s, with 573 ragged tensors 6.1 (a mover of its
// streams without arithmetic 6.1-6.2).  What is left is the 4-5 us per launch that run below full rate.
#pragma once
#include "adam_elem.hip.h"
#include "elem.hip.h"
#include "launch.h"
#include "list_args.h"

namespace yafsdp {

// Index of this wave in the grid, known to be wave-uniform.
template <int BLOCK>
__device__ __forceinline__ uint32_t global_wave() {
  return __builtin_amdgcn_readfirstlane(blockIdx.x * (BLOCK / 64) + (threadIdx.x >> 6));
}

// A list as the kernels read it: through the constant address space (scalar loads), from the kernel arguments (the
// first parameter of the kernel) or from the workspace.
struct ListView {
  const YAFSDP_CONST_AS uint32_t* tile_end;
  const YAFSDP_CONST_AS uint64_t* range;
  int n;
  uint32_t n_tiles;
};
struct ListAdamView {
  const YAFSDP_CONST_AS uint32_t* tile_end;
  const YAFSDP_CONST_AS uint32_t* tail;
  const YAFSDP_CONST_AS ListAdamRange* r;
  int n;
  uint32_t n_tiles;
};

template <class T>
__device__ __forceinline__ const YAFSDP_CONST_AS T* as_const(const T* p) {
  return (const YAFSDP_CONST_AS T*)reinterpret_cast<uintptr_t>(p);
}
template <class ARGS>
__device__ __forceinline__ const YAFSDP_CONST_AS ARGS* first_argument() {
  return (const YAFSDP_CONST_AS ARGS*)__builtin_amdgcn_kernarg_segment_ptr();
}
__device__ __forceinline__ ListView list_view(const ListArgs&) {
  const YAFSDP_CONST_AS ListArgs* a = first_argument<ListArgs>();
  return ListView{a->tile_end, a->range, a->n, a->n_tiles};
}
__device__ __forceinline__ ListView list_view(const ListRef& a) {
  return ListView{as_const(a.tile_end), as_const(a.range), a.n, a.n_tiles};
}
__device__ __forceinline__ ListAdamView list_view(const ListAdamArgs&) {
  const YAFSDP_CONST_AS ListAdamArgs* a = first_argument<ListAdamArgs>();
  return ListAdamView{a->tile_end, a->tail, a->r, a->n, a->n_tiles};
}
__device__ __forceinline__ ListAdamView list_view(const ListAdamRef& a) {
  return ListAdamView{as_const(a.tile_end), as_const(a.tail), as_const(a.r), a.n, a.n_tiles};
}

// First range, from `lo` on, whose tiles end behind tile t (t < n_tiles).
template <class VIEW>
__device__ __forceinline__ int find_range(const VIEW& a, uint32_t t, int lo = 0) {
  int hi = a.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (t >= a.tile_end[mid]) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

// Writes one piece of a long list into the workspace: 16 bytes per lane, one load.
__global__ void __launch_bounds__(kListStageWords / 4) list_stage_kernel(ListStageArgs, u32x4* dst) {
  const YAFSDP_CONST_AS u32x4* a = reinterpret_cast<const YAFSDP_CONST_AS u32x4*>(first_argument<ListStageArgs>()->word);
  dst[threadIdx.x] = a[threadIdx.x];
}

// The same from pinned host memory in one launch; each workgroup marks its piece as read (StageSlots).
__global__ void __launch_bounds__(kListFetchBlock)
list_fetch_kernel(const u32x4* src, u32x4* dst, uint32_t n, uint32_t* done, uint32_t number) {
  const uint32_t i = blockIdx.x * kListFetchBlock + threadIdx.x;
  if (i < n) dst[i] = src[i];
  __syncthreads();
  if (threadIdx.x == 0) __hip_atomic_store(done + blockIdx.x, number, __ATOMIC_RELEASE, __HIP_MEMORY_SCOPE_SYSTEM);
}

// The ranges' addresses are integers in the list: said to be global memory here, so that the accesses need no flat ones.
#define YAFSDP_GLOBAL_AS __attribute__((address_space(1)))
template <class T>
__device__ __forceinline__ YAFSDP_GLOBAL_AS T* global_at(uint64_t addr) {
  return (YAFSDP_GLOBAL_AS T*)addr;
}

// Bytes [lo, hi) of one 4-KiB tile.
struct ListTile {
  uint64_t base;  // 128-byte aligned
  int lo, hi;
  int dtype;
};

// Tile t of a range (list_word) whose tiles are [begin, end).
__device__ __forceinline__ ListTile tile_of(uint64_t range, uint32_t begin, uint32_t end, uint32_t t) {
  const uint64_t addr = range & ((uint64_t(1) << kListAddrBits) - 1);
  const uint32_t rest = uint32_t(range >> kListAddrBits);
  ListTile x;
  x.base = (addr & ~uint64_t(127)) + uint64_t(t - begin) * kListTileBytes;
  x.lo = t == begin ? int(addr & 127) : 0;
  x.hi = t + 1 == end ? int(rest & ((1u << kListTailBits) - 1)) + 1 : kListTileBytes;
  x.dtype = int(rest >> kListTailBits);
  return x;
}

// Looks tiles up in ascending order; a tile of the same range as the one before costs nothing.
struct TileCursor {
  const ListView& a;
  int k;
  uint32_t begin, end;
  uint64_t range;

  __device__ __forceinline__ explicit TileCursor(const ListView& view) : a(view), k(-1), begin(0), end(0) {}
  __device__ __forceinline__ ListTile tile(uint32_t t) {
    if (t >= end) {
      k = find_range(a, t, k + 1);
      begin = k > 0 ? a.tile_end[k - 1] : 0;
      end = a.tile_end[k];
      range = a.range[k];
    }
    return tile_of(range, begin, end, t);
  }
};

// values every lane of the wave holds alike, as scalars
__device__ __forceinline__ float uniform(float x) {
  return bits_to_f32(__builtin_amdgcn_readfirstlane(f32_to_bits(x)));
}
__device__ __forceinline__ ListTile uniform(const ListTile& x) {
  ListTile y;
  y.base = uint64_t(__builtin_amdgcn_readfirstlane(uint32_t(x.base >> 32))) << 32 |
           uint32_t(__builtin_amdgcn_readfirstlane(uint32_t(x.base)));
  y.lo = __builtin_amdgcn_readfirstlane(x.lo);
  y.hi = __builtin_amdgcn_readfirstlane(x.hi);
  y.dtype = __builtin_amdgcn_readfirstlane(x.dtype);
  return y;
}

// A lane's share of a tile: every 64th of its 256 16-byte vectors, zeros where a vector is not wholly inside [lo, hi).
constexpr int kTileVecs = kListTileBytes / 1024;
struct TileData {
  u32x4 v[kTileVecs];
};
__device__ __forceinline__ bool whole(const ListTile& x) { return x.lo == 0 && x.hi == kListTileBytes; }
__device__ __forceinline__ int vec_offset(int j) { return (j * 64 + int(threadIdx.x & 63)) * 16; }
__device__ __forceinline__ bool inside(const ListTile& x, int off) { return off >= x.lo && off + 16 <= x.hi; }

// Non-temporal in either branch: the compiler merges a load that both share, and drops the hint unless both have it.
__device__ __forceinline__ TileData load_tile(const ListTile& x) {
  TileData d;
  if (whole(x)) {
#pragma unroll
    for (int j = 0; j < kTileVecs; j++) d.v[j] = __builtin_nontemporal_load(global_at<const u32x4>(x.base + vec_offset(j)));
  } else {
#pragma unroll
    for (int j = 0; j < kTileVecs; j++) {
      d.v[j] = u32x4{0u, 0u, 0u, 0u};
      if (inside(x, vec_offset(j))) d.v[j] = __builtin_nontemporal_load(global_at<const u32x4>(x.base + vec_offset(j)));
    }
  }
  return d;
}

// Calls elem(offset) for the elements of the (at most two) vectors that the tile's first and last byte cut: up to 7 at
// either end, one per lane.
template <int SIZE, class E>
__device__ __forceinline__ void cut_elements(const ListTile& x, E elem) {
  const int lane = threadIdx.x & 63;
  const int lo16 = (x.lo + 15) & ~15, hi16 = x.hi & ~15;
  const int head_end = lo16 < x.hi ? lo16 : x.hi;
  const int tail_begin = hi16 > lo16 ? hi16 : lo16;
  const int h = x.lo + lane * SIZE, t = tail_begin + lane * SIZE;
  if (h < head_end) elem(h);
  if (t < x.hi) elem(t);
}

template <class S>
__device__ __forceinline__ void unpack_vec(u32x4 v, float (&f)[16 / S::kSize]) {
  if constexpr (S::kSize == 4) {
#pragma unroll
    for (int i = 0; i < 4; i++) f[i] = bits_to_f32(v[i]);
  } else {
    Unit<S> u;
    u.v[0] = v;
    unpack<S>(u, f);
  }
}

template <class S>
__device__ __forceinline__ u32x4 pack_vec(const float (&f)[16 / S::kSize]) {
  if constexpr (S::kSize == 4) {
    return u32x4{f32_to_bits(f[0]), f32_to_bits(f[1]), f32_to_bits(f[2]), f32_to_bits(f[3])};
  } else {
    return pack<S>(f).v[0];
  }
}

// ------------------------------------------------------------------- norm ----
// Sums are held in binary64: the square of a binary32 number is exact there and neither overflows nor underflows, so
// the order of the additions moves the result by no more than the last bits of binary64.  The largest magnitude is
// taken as an unsigned integer (the bits without the sign): ordered like the values, with every NaN above infinity, so
// a NaN anywhere becomes the result.
template <int NORM>
struct NormAcc {
  double s[2] = {0.0, 0.0};
  uint32_t m = 0;

  __device__ __forceinline__ void add(float x, int i) {
    if constexpr (NORM == LIST_NORM_INF) {
      const uint32_t b = f32_to_bits(x) & 0x7FFFFFFFu;
      m = b > m ? b : m;
    } else if constexpr (NORM == LIST_NORM_1) {
      s[i & 1] += double(__builtin_fabsf(x));
    } else {
      s[i & 1] = __fma_rn(double(x), double(x), s[i & 1]);
    }
  }
  __device__ __forceinline__ double value() const {
    if constexpr (NORM == LIST_NORM_INF) return double(m);
    else return s[0] + s[1];
  }
};

template <int NORM>
__device__ __forceinline__ double norm_join(double a, double b) {
  if constexpr (NORM == LIST_NORM_INF) return a > b ? a : b;  // bit patterns as whole numbers: exact, never NaN
  else return a + b;
}

// block_sum's order, for either kind of partial result.  Valid in thread 0.
template <int NORM, int BLOCK>
__device__ __forceinline__ double block_join(double v, double* lds) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = norm_join<NORM>(v, __shfl_down(v, off, 64));
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (lane == 0) lds[wave] = v;
  __syncthreads();
  double t = 0.0;
  if (threadIdx.x == 0) {
#pragma unroll
    for (int w = 0; w < BLOCK / 64; w++) t = norm_join<NORM>(t, lds[w]);
  }
  return t;
}

template <int NORM, class S>
__device__ __forceinline__ void norm_tile_of(const ListTile& x, const TileData& d, NormAcc<NORM>& acc) {
  constexpr int kPer = 16 / S::kSize;
#pragma unroll
  for (int j = 0; j < kTileVecs; j++) {
    float f[kPer];
    unpack_vec<S>(d.v[j], f);
#pragma unroll
    for (int i = 0; i < kPer; i++) acc.add(f[i], i);
  }
  if (!whole(x))
    cut_elements<S::kSize>(
        x, [&](int off) { acc.add(to_f32<S>(*global_at<const typename S::storage>(x.base + off)), 0); });
}
template <int NORM>
__device__ __forceinline__ void norm_tile(const ListTile& x, const TileData& d, NormAcc<NORM>& acc) {
  if (x.dtype == DT_F32) norm_tile_of<NORM, F32>(x, d, acc);
  else if (x.dtype == DT_BF16) norm_tile_of<NORM, BF16>(x, d, acc);
  else norm_tile_of<NORM, F16>(x, d, acc);
}

// f(tile, its data) for tiles w, w + step, ... below n: the next tile is looked up (`at`) and its loads are issued while
// those of the tile before are still in flight.
template <class A, class F>
__device__ __forceinline__ void stream_tiles(uint32_t w, uint32_t step, uint32_t n, A at, F f) {
  if (w >= n) return;
  ListTile x = at(w);
  TileData d = load_tile(x);
  for (uint32_t t = w + step; t < n; t += step) {
    const ListTile y = at(t);
    const TileData e = load_tile(y);
    f(x, d);
    x = y;
    d = e;
  }
  f(x, d);
}
// ... over the whole grid
template <int BLOCK, class F>
__device__ __forceinline__ void stream_list(const ListView& a, F f) {
  TileCursor cursor(a);
  stream_tiles(global_wave<BLOCK>(), gridDim.x * (BLOCK / 64), a.n_tiles, [&](uint32_t t) { return cursor.tile(t); }, f);
}

// partials[blockIdx.x] = this workgroup's share of the norm's sum
template <int NORM, class META, int BLOCK>
__global__ void __launch_bounds__(BLOCK) list_norm_kernel(META meta, double* partials) {
  __shared__ double lds[BLOCK / 64];
  const ListView a = list_view(meta);
  NormAcc<NORM> acc;
  stream_list<BLOCK>(a, [&](const ListTile& x, const TileData& d) { norm_tile<NORM>(x, d, acc); });
  const double total = block_join<NORM, BLOCK>(acc.value(), lds);
  if (threadIdx.x == 0) partials[blockIdx.x] = total;
}

// norm and clip coefficient from the joined total, in binary32 as clip_coef_kernel computes them
template <int NORM>
__device__ __forceinline__ void norm_and_coef_of(double total, float max_norm, float& norm, float& coef) {
  if constexpr (NORM == LIST_NORM_INF) norm = bits_to_f32(uint32_t(total));
  else if constexpr (NORM == LIST_NORM_1) norm = float(total);
  else norm = float(__builtin_sqrt(total));
  coef = __fdiv_rn(max_norm, __fadd_rn(norm, 1e-6f));
  if (coef > 1.0f) coef = 1.0f;  // a NaN stays
}

// The joined total of at most kListNormGrid partial sums, valid in thread 0.  One latency: a lane's loads are all in
// flight at once (448 tensors clipped, 59 MB: 36.6 us; one after the other 37.4), and four waves join sooner than
// sixteen (norm of 300 fp16 tensors: 29.8 us and 30.5).
template <int NORM, int BLOCK>
__device__ __forceinline__ double join_partials(const double* partials, int count, double* lds) {
  constexpr int kPer = kListNormGrid / BLOCK;
  static_assert(kPer * BLOCK == kListNormGrid, "whole rounds");
  double v[kPer];
#pragma unroll
  for (int j = 0; j < kPer; j++) {
    const int i = int(threadIdx.x) + j * BLOCK;
    v[j] = i < count ? partials[i] : 0.0;
  }
#pragma unroll
  for (int j = 1; j < kPer; j++) v[0] = norm_join<NORM>(v[0], v[j]);
  return block_join<NORM, BLOCK>(v[0], lds);
}

template <int NORM, int BLOCK>
__global__ void __launch_bounds__(BLOCK)
list_finish_kernel(const double* partials, int count, float max_norm, float* norm_and_coef) {
  __shared__ double lds[BLOCK / 64];
  const double total = join_partials<NORM, BLOCK>(partials, count, lds);
  if (threadIdx.x == 0) {
    float norm, coef;
    norm_and_coef_of<NORM>(total, max_norm, norm, coef);
    norm_and_coef[0] = norm;
    norm_and_coef[1] = coef;
  }
}

// ------------------------------------------------------------------ scale ----
// x = round(float(x) * c) in place; nothing is touched when c is exactly 1 (x * 1 == x).
template <class S>
__device__ __forceinline__ void scale_tile_of(const ListTile& x, const TileData& d, float c) {
  constexpr int kPer = 16 / S::kSize;
  const bool all = whole(x);
#pragma unroll
  for (int j = 0; j < kTileVecs; j++) {
    float f[kPer];
    unpack_vec<S>(d.v[j], f);
#pragma unroll
    for (int i = 0; i < kPer; i++) f[i] = opaque(__fmul_rn(opaque(f[i]), c));
    if (all || inside(x, vec_offset(j)))
      __builtin_nontemporal_store(pack_vec<S>(f), global_at<u32x4>(x.base + vec_offset(j)));
  }
  if (!all)
    cut_elements<S::kSize>(x, [&](int off) {
      YAFSDP_GLOBAL_AS typename S::storage* p = global_at<typename S::storage>(x.base + off);
      *p = from_f32<S>(opaque(__fmul_rn(opaque(to_f32<S>(*p)), c)));
    });
}
__device__ __forceinline__ void scale_tile(const ListTile& x, const TileData& d, float c) {
  if (x.dtype == DT_F32) scale_tile_of<F32>(x, d, c);
  else if (x.dtype == DT_BF16) scale_tile_of<BF16>(x, d, c);
  else scale_tile_of<F16>(x, d, c);
}

// one tile per wave, from tile `first` on
template <class META, int BLOCK>
__global__ void __launch_bounds__(BLOCK) list_scale_kernel(META meta, uint32_t first, const float* coef) {
  const float c = *as_const(coef);
  if (c == 1.0f) return;
  const ListView a = list_view(meta);
  const uint32_t t = first + global_wave<BLOCK>();
  if (t >= a.n_tiles) return;
  const ListTile x = TileCursor(a).tile(t);
  scale_tile(x, load_tile(x), c);
}

// list_finish_kernel and the scaling in one launch, for a list of medium size: every workgroup joins the partial sums
// for itself (the same additions in the same order), the first one also reports norm and coefficient.
template <int NORM, class META, int BLOCK>
__global__ void __launch_bounds__(BLOCK)
list_clip_kernel(META meta, const double* partials, int count, float max_norm, float* norm_and_coef) {
  __shared__ double lds[BLOCK / 64];
  __shared__ float shared_coef;
  const ListView a = list_view(meta);
  const double total = join_partials<NORM, BLOCK>(partials, count, lds);
  if (threadIdx.x == 0) {
    float norm, coef;
    norm_and_coef_of<NORM>(total, max_norm, norm, coef);
    shared_coef = coef;
    if (blockIdx.x == 0) {
      norm_and_coef[0] = norm;
      norm_and_coef[1] = coef;
    }
  }
  __syncthreads();
  const float c = uniform(shared_coef);
  if (c == 1.0f) return;
  stream_list<BLOCK>(a, [&](const ListTile& x, const TileData& d) { scale_tile(x, d, c); });
}

// A short list (at most kListSmallNormTiles tiles) in one launch of one workgroup: norm, coefficient and (CLIP) the scaling.
// The ranges' lanes first write every tile's place to LDS.  A wave scales the tiles it has read itself, so nothing but
// the joined total passes between waves; the first kHeld tiles of a wave are loaded at once and stay in its registers.
template <int NORM, bool CLIP, int BLOCK>
__global__ void __launch_bounds__(BLOCK) list_small_kernel(ListArgs, float max_norm, float* norm_and_coef) {
  static_assert(BLOCK >= kListMax && kListSmallClipTiles <= kListSmallNormTiles, "a lane per range, room for every tile");
  constexpr int kHeld = 4, kWaves = BLOCK / 64;
  __shared__ double lds[kWaves];
  __shared__ float shared_coef;
  __shared__ ListTile tiles[kListSmallNormTiles];
  const YAFSDP_CONST_AS ListArgs* a = first_argument<ListArgs>();
  const uint32_t n_tiles = a->n_tiles;
  const int i = threadIdx.x;
  if (i < a->n) {
    const uint32_t begin = i > 0 ? a->tile_end[i - 1] : 0, end = a->tile_end[i];
    const uint64_t range = a->range[i];
    for (uint32_t t = begin; t < end; t++) tiles[t] = tile_of(range, begin, end, t);
  }
  __syncthreads();
  const uint32_t wave = global_wave<BLOCK>(), rest = wave + kHeld * kWaves;
  const auto at = [&](uint32_t t) { return uniform(tiles[t]); };
  TileData held[kHeld];
#pragma unroll
  for (int j = 0; j < kHeld; j++)
    if (wave + j * kWaves < n_tiles) held[j] = load_tile(at(wave + j * kWaves));
  NormAcc<NORM> acc;
#pragma unroll
  for (int j = 0; j < kHeld; j++)
    if (wave + j * kWaves < n_tiles) norm_tile<NORM>(at(wave + j * kWaves), held[j], acc);
  stream_tiles(rest, kWaves, n_tiles, at, [&](const ListTile& x, const TileData& d) { norm_tile<NORM>(x, d, acc); });
  const double total = block_join<NORM, BLOCK>(acc.value(), lds);
  if (i == 0) {
    float norm, coef;
    norm_and_coef_of<NORM>(total, max_norm, norm, coef);
    norm_and_coef[0] = norm;
    norm_and_coef[1] = coef;
    shared_coef = coef;
  }
  if constexpr (CLIP) {
    __syncthreads();
    const float c = uniform(shared_coef);
    if (c == 1.0f) return;
#pragma unroll
    for (int j = 0; j < kHeld; j++)
      if (wave + j * kWaves < n_tiles) scale_tile(at(wave + j * kWaves), held[j], c);
    stream_tiles(rest, kWaves, n_tiles, at, [&](const ListTile& x, const TileData& d) { scale_tile(x, d, c); });
  }
}

// ------------------------------------------------------------------ AdamW ----
// adam_elem on each element: same operations, same roundings, same bits as adamw_kernel.  A 16-bit gradient enters as
// the binary32 number it stands for; its product with grad_scale is rounded to binary32 (a grad.mul_ beforehand would
// round it to 16 bits).  O is F32 for "no 16-bit copy".  Tiles are counted from a 256-byte boundary of the parameters:
// with tiles from the first element of each tensor, two waves share a line at every tile's ends in all four or five
// arrays, and 573 ragged tensors took 280 us instead of 222.
template <class G>
__device__ __forceinline__ float adam_grad(float g) {
  if constexpr (G::kId == DT_F16) return opaque(g);
  else return g;
}

// a quad at any element-aligned address, non-temporal
template <class T>
__device__ __forceinline__ Quad<T> load_nt(const YAFSDP_GLOBAL_AS typename T::storage* p) {
  Quad<T> q;
  q.v = __builtin_nontemporal_load((const YAFSDP_GLOBAL_AS typename T::quad_unaligned*)p);
  return q;
}
template <class T>
__device__ __forceinline__ void store_nt(YAFSDP_GLOBAL_AS typename T::storage* p, const Quad<T>& q) {
  __builtin_nontemporal_store(q.v, (YAFSDP_GLOBAL_AS typename T::quad_unaligned*)p);
}

// one tile per wave, from tile `first_tile` on
template <class G, class O, class META, int BLOCK>
__global__ void __launch_bounds__(BLOCK)
list_adamw_kernel(META meta, uint32_t first_tile, AdamScalars s, const float* grad_scale) {
  constexpr bool kOut = !same_t<O, F32>::value;
  static_assert(kListAdamTile == 256, "a wave holds a tile as one quad per lane");
  typedef typename G::storage g_t;
  const ListAdamView a = list_view(meta);
  const uint32_t t = first_tile + global_wave<BLOCK>();
  if (t >= a.n_tiles) return;
  const bool scaled = grad_scale != nullptr;
  float gs = 1.0f;
  if (scaled) gs = *as_const(grad_scale);
  const int lane = threadIdx.x & 63;
  const int k = find_range(a, t);
  const uint32_t begin = k > 0 ? a.tile_end[k - 1] : 0;
  const uint64_t p0 = a.r[k].p;
  // elements [lo, hi) of the tile; element e of it is element first + e of the range
  const int head = int(p0 & 255) / 4, lo = t == begin ? head : 0, hi = t + 1 == a.tile_end[k] ? int(a.tail[k]) : kListAdamTile;
  const int64_t first = int64_t(t - begin) * kListAdamTile - head;
  YAFSDP_GLOBAL_AS float* p = global_at<float>(p0) + first;
  YAFSDP_GLOBAL_AS g_t* g = global_at<g_t>(a.r[k].g) + first;
  YAFSDP_GLOBAL_AS float* m = global_at<float>(a.r[k].m) + first;
  YAFSDP_GLOBAL_AS float* v = global_at<float>(a.r[k].v) + first;
  YAFSDP_GLOBAL_AS typename O::storage* out = global_at<typename O::storage>(kOut ? a.r[k].out : 0) + first;
  const int e4 = lane * 4;
  if (e4 >= lo && e4 + 4 <= hi) {
    const Quad<F32> qp = load_nt<F32>(p + e4);
    const Quad<G> qg = load_nt<G>(g + e4);
    const Quad<F32> qm = load_nt<F32>(m + e4);
    const Quad<F32> qv = load_nt<F32>(v + e4);
    float fp[4], fg[4], fm[4], fv[4];
    unpack_quad<F32>(qp, fp);
    unpack_quad<G>(qg, fg);
    unpack_quad<F32>(qm, fm);
    unpack_quad<F32>(qv, fv);
#pragma unroll
    for (int i = 0; i < 4; i++) adam_elem(fp[i], adam_grad<G>(fg[i]), fm[i], fv[i], s, scaled, gs);
    store_nt<F32>(p + e4, pack_quad<F32>(fp));
    store_nt<F32>(m + e4, pack_quad<F32>(fm));
    store_nt<F32>(v + e4, pack_quad<F32>(fv));
    if constexpr (kOut) store_nt<O>(out + e4, pack_quad<O>(fp));
    if (s.flags & ADAM_ZERO_GRAD) {
      const float z[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      store_nt<G>(g + e4, pack_quad<G>(z));
    }
  }
  if (lo == 0 && hi == kListAdamTile) return;
  // the elements of quads that the tile's first and last element cut: up to 3 at either end, lanes 0-3 and 4-7
  const int lo4 = (lo + 3) & ~3, hi4 = hi & ~3;
  const int e = lane < 4 ? lo + lane : (hi4 > lo4 ? hi4 : lo4) + lane - 4;
  if (lane < 8 && e < (lane < 4 && lo4 < hi ? lo4 : hi)) {
    float fp = p[e], fm = m[e], fv = v[e];
    adam_elem(fp, adam_grad<G>(to_f32<G>(g[e])), fm, fv, s, scaled, gs);
    p[e] = fp;
    m[e] = fm;
    v[e] = fv;
    if constexpr (kOut) out[e] = from_f32<O>(fp);
    if (s.flags & ADAM_ZERO_GRAD) g[e] = from_f32<G>(0.0f);
  }
}

}  // namespace yafsdp
