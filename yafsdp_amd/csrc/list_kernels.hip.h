// Optimizer-side passes over a list of separate tensors: norm (1, 2, inf), scaling by a device-resident coefficient,
// AdamW.  Nothing here is a contraction: all of it is bound by memory.
//
// Work is cut into wave-sized tiles (4 KiB for the norm and the scaling, 512 elements for AdamW); a wave finds the
// range that holds its tile in the kernel arguments, which it reads through the constant address space (scalar loads).
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

// First range of the launch whose tiles end behind tile t (t < n_tiles).
template <class ARGS>
__device__ __forceinline__ int find_range(const YAFSDP_CONST_AS ARGS* a, uint32_t t) {
  int lo = 0, hi = a->n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (t >= a->r[mid].tile_end) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

// The kernel arguments where they lie: the first parameter of every kernel here is its list.
template <class ARGS>
__device__ __forceinline__ const YAFSDP_CONST_AS ARGS* list_args() {
  return (const YAFSDP_CONST_AS ARGS*)__builtin_amdgcn_kernarg_segment_ptr();
}

// Bytes [lo, hi) of one 4-KiB tile.
struct ListTile {
  char* base;  // 128-byte aligned
  int lo, hi;
  int dtype;
};

__device__ __forceinline__ ListTile list_tile(const YAFSDP_CONST_AS ListArgs* a, uint32_t t) {
  const int k = find_range(a, t);
  const uint32_t begin = k > 0 ? a->r[k - 1].tile_end : 0;
  const uint64_t addr = a->r[k].addr;
  const uint32_t tail = a->r[k].tail;
  ListTile x;
  x.base = reinterpret_cast<char*>(addr & ~uint64_t(127)) + uint64_t(t - begin) * kListTileBytes;
  x.lo = t == begin ? int(addr & 127) : 0;
  x.hi = t + 1 == a->r[k].tile_end ? int(tail & 0x1FFFu) : kListTileBytes;
  x.dtype = int(tail >> 30);
  return x;
}

// Calls vec(offset) for every 16-byte vector of this lane that lies inside the tile and elem(offset) for the elements
// of the (at most two) vectors that the tile's first and last byte cut: up to 7 at either end.
template <int SIZE, class V, class E>
__device__ __forceinline__ void walk_partial_tile(const ListTile& x, V vec, E elem) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int j = 0; j < kListTileBytes / 1024; j++) {
    const int off = (j * 64 + lane) * 16;
    if (off >= x.lo && off + 16 <= x.hi) vec(off);
  }
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
__device__ __forceinline__ void norm_tile(const ListTile& x, NormAcc<NORM>& acc) {
  constexpr int kPer = 16 / S::kSize;
  const int lane = threadIdx.x & 63;
  if (x.lo == 0 && x.hi == kListTileBytes) {
    u32x4 v[kListTileBytes / 1024];
#pragma unroll
    for (int j = 0; j < kListTileBytes / 1024; j++)
      v[j] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(x.base + (j * 64 + lane) * 16));
#pragma unroll
    for (int j = 0; j < kListTileBytes / 1024; j++) {
      float f[kPer];
      unpack_vec<S>(v[j], f);
#pragma unroll
      for (int i = 0; i < kPer; i++) acc.add(f[i], i);
    }
  } else {
    walk_partial_tile<S::kSize>(
        x,
        [&](int off) {
          float f[kPer];
          unpack_vec<S>(*reinterpret_cast<const u32x4*>(x.base + off), f);
#pragma unroll
          for (int i = 0; i < kPer; i++) acc.add(f[i], i);
        },
        [&](int off) { acc.add(to_f32<S>(*reinterpret_cast<const typename S::storage*>(x.base + off)), 0); });
  }
}

// partials[blockIdx.x] = this workgroup's share of the norm's sum
template <int NORM, int BLOCK>
__global__ void __launch_bounds__(BLOCK) list_norm_kernel(ListArgs, double* partials) {
  __shared__ double lds[BLOCK / 64];
  const YAFSDP_CONST_AS ListArgs* a = list_args<ListArgs>();
  const uint32_t n_tiles = a->n_tiles, waves = gridDim.x * (BLOCK / 64);
  NormAcc<NORM> acc;
  for (uint32_t t = global_wave<BLOCK>(); t < n_tiles; t += waves) {
    const ListTile x = list_tile(a, t);
    if (x.dtype == DT_F32) norm_tile<NORM, F32>(x, acc);
    else if (x.dtype == DT_BF16) norm_tile<NORM, BF16>(x, acc);
    else norm_tile<NORM, F16>(x, acc);
  }
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

template <int NORM, int BLOCK>
__device__ __forceinline__ double join_partials(const double* partials, int count, double* lds) {
  double acc = 0.0;
  for (int i = threadIdx.x; i < count; i += BLOCK) acc = norm_join<NORM>(acc, partials[i]);
  return block_join<NORM, BLOCK>(acc, lds);
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
__device__ __forceinline__ void scale_tile(const ListTile& x, float c) {
  constexpr int kPer = 16 / S::kSize;
  const int lane = threadIdx.x & 63;
  if (x.lo == 0 && x.hi == kListTileBytes) {
    u32x4 v[kListTileBytes / 1024];
#pragma unroll
    for (int j = 0; j < kListTileBytes / 1024; j++)
      v[j] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(x.base + (j * 64 + lane) * 16));
#pragma unroll
    for (int j = 0; j < kListTileBytes / 1024; j++) {
      float f[kPer];
      unpack_vec<S>(v[j], f);
#pragma unroll
      for (int i = 0; i < kPer; i++) f[i] = opaque(__fmul_rn(opaque(f[i]), c));
      __builtin_nontemporal_store(pack_vec<S>(f), reinterpret_cast<u32x4*>(x.base + (j * 64 + lane) * 16));
    }
  } else {
    walk_partial_tile<S::kSize>(
        x,
        [&](int off) {
          float f[kPer];
          u32x4* p = reinterpret_cast<u32x4*>(x.base + off);
          unpack_vec<S>(*p, f);
#pragma unroll
          for (int i = 0; i < kPer; i++) f[i] = opaque(__fmul_rn(opaque(f[i]), c));
          *p = pack_vec<S>(f);
        },
        [&](int off) {
          typename S::storage* p = reinterpret_cast<typename S::storage*>(x.base + off);
          *p = from_f32<S>(opaque(__fmul_rn(opaque(to_f32<S>(*p)), c)));
        });
  }
}

template <int BLOCK>
__global__ void __launch_bounds__(BLOCK) list_scale_kernel(ListArgs, const float* coef) {
  const YAFSDP_CONST_AS ListArgs* a = list_args<ListArgs>();
  const float c = *reinterpret_cast<const YAFSDP_CONST_AS float*>(reinterpret_cast<uintptr_t>(coef));
  if (c == 1.0f) return;
  const uint32_t n_tiles = a->n_tiles, waves = gridDim.x * (BLOCK / 64);
  for (uint32_t t = global_wave<BLOCK>(); t < n_tiles; t += waves) {
    const ListTile x = list_tile(a, t);
    if (x.dtype == DT_F32) scale_tile<F32>(x, c);
    else if (x.dtype == DT_BF16) scale_tile<BF16>(x, c);
    else scale_tile<F16>(x, c);
  }
}

// ------------------------------------------------------------------ AdamW ----
// adam_elem on each element: same operations, same roundings, same bits as adamw_kernel.  A
// 16-bit gradient enters as the binary32 number it stands for; its product with grad_scale is rounded to binary32 (a
// grad.mul_ beforehand would round it to 16 bits).  O is F32 for "no 16-bit copy".
template <class G>
__device__ __forceinline__ float adam_grad(float g) {
  if constexpr (G::kId == DT_F16) return opaque(g);
  else return g;
}

template <class G, class O, int BLOCK>
__global__ void __launch_bounds__(BLOCK) list_adamw_kernel(ListAdamArgs, AdamScalars s, const float* grad_scale) {
  constexpr bool kOut = !same_t<O, F32>::value;
  constexpr int kQuads = kListAdamTile / 256;
  typedef typename G::storage g_t;
  const YAFSDP_CONST_AS ListAdamArgs* a = list_args<ListAdamArgs>();
  const bool scaled = grad_scale != nullptr;
  float gs = 1.0f;
  if (scaled) gs = *reinterpret_cast<const YAFSDP_CONST_AS float*>(reinterpret_cast<uintptr_t>(grad_scale));
  const uint32_t n_tiles = a->n_tiles, waves = gridDim.x * (BLOCK / 64);
  const int lane = threadIdx.x & 63;
  for (uint32_t t = global_wave<BLOCK>(); t < n_tiles; t += waves) {
    const int k = find_range(a, t);
    const uint32_t begin = k > 0 ? a->r[k - 1].tile_end : 0;
    const int n = t + 1 == a->r[k].tile_end ? int(a->r[k].tail) : kListAdamTile;
    const uint64_t first = uint64_t(t - begin) * kListAdamTile;
    float* p = reinterpret_cast<float*>(a->r[k].p) + first;
    g_t* g = reinterpret_cast<g_t*>(a->r[k].g) + first;
    float* m = reinterpret_cast<float*>(a->r[k].m) + first;
    float* v = reinterpret_cast<float*>(a->r[k].v) + first;
    typename O::storage* out = kOut ? reinterpret_cast<typename O::storage*>(a->r[k].out) + first : nullptr;
    Quad<F32> qp[kQuads], qm[kQuads], qv[kQuads];
    Quad<G> qg[kQuads];
#pragma unroll
    for (int j = 0; j < kQuads; j++) {
      const int e = (j * 64 + lane) * 4;
      if (e + 4 <= n) {
        qp[j] = load_quad<F32, true>(p + e);
        qg[j] = load_quad<G, true>(g + e);
        qm[j] = load_quad<F32, true>(m + e);
        qv[j] = load_quad<F32, true>(v + e);
      }
    }
#pragma unroll
    for (int j = 0; j < kQuads; j++) {
      const int e = (j * 64 + lane) * 4;
      if (e + 4 <= n) {
        float fp[4], fg[4], fm[4], fv[4];
        unpack_quad<F32>(qp[j], fp);
        unpack_quad<G>(qg[j], fg);
        unpack_quad<F32>(qm[j], fm);
        unpack_quad<F32>(qv[j], fv);
#pragma unroll
        for (int i = 0; i < 4; i++) adam_elem(fp[i], adam_grad<G>(fg[i]), fm[i], fv[i], s, scaled, gs);
        store_quad<F32, true>(p + e, pack_quad<F32>(fp));
        store_quad<F32, true>(m + e, pack_quad<F32>(fm));
        store_quad<F32, true>(v + e, pack_quad<F32>(fv));
        if constexpr (kOut) store_quad<O, true>(out + e, pack_quad<O>(fp));
        if (s.flags & ADAM_ZERO_GRAD) {
          const float z[4] = {0.0f, 0.0f, 0.0f, 0.0f};
          store_quad<G, true>(g + e, pack_quad<G>(z));
        }
      }
    }
    const int e = (n & ~3) + lane;  // up to 3 elements behind the last quad of a range
    if (e < n) {
      float fp = p[e], fm = m[e], fv = v[e];
      adam_elem(fp, adam_grad<G>(to_f32<G>(g[e])), fm, fv, s, scaled, gs);
      p[e] = fp;
      m[e] = fm;
      v[e] = fv;
      if constexpr (kOut) out[e] = from_f32<O>(fp);
      if (s.flags & ADAM_ZERO_GRAD) g[e] = from_f32<G>(0.0f);
    }
  }
}

}  // namespace yafsdp
