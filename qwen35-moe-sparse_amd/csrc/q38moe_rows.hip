// Tokens to expert-sorted rows and back (differentiable experts of the caller's own between the two), on the
// permutation of q38moe_permute.hip: pair p = t*k + j of token t goes to row inv[p]; pairs whose index lies outside
// [0, E) have no row, and the rows behind the last filled one are theirs to be zero.
//
//   spread:   dst[inv[p]] = src[t] (* w[p]),  dst[r] = 0 for r >= filled,  dw[p] = <src[t], y[inv[p]]>
//   collect:  out[t] = sum_j src[inv[p]] (* w[p])
//
// spread without w is the dispatch, collect without w its gradient; collect with w is the combine, spread with w and y its
// gradients. Products and sums are fp32, each output is rounded once. Both run one wave per token: a wave's instruction
// covers 1 KiB of a row, and the loads of two such pieces of all k rows are issued before any is used. Both are bound by
// memory: 16384 tokens of 1024 bf16 by 5 take 36 us there (201 MB, 5.6 TB/s), 35 back, and 68 for both gradients of the
// combine (369 MB, 5.4 TB/s). Rows are written past the caches, which the next reader's 168 MB would not find there anyway:
// through them the four passes take 195 us together instead of 174.
#include <type_traits>

#include "q38moe_common.h"
#include "q38moe_kernels.h"

namespace q38 {
namespace {

template <typename E>
constexpr int VEC = 16 / sizeof(E);  // elements of a 16-byte load

constexpr int ROWS_SMALL = 4096;  // pairs of a dispatch in one launch

template <typename E>
__device__ __forceinline__ void unpack16(u32x4_t v, float (&f)[VEC<E>]) {
  if constexpr (std::is_same<E, float>::value) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) unpack_bf16x2(v[i], f[2 * i], f[2 * i + 1]);
  }
}

template <typename E>
__device__ __forceinline__ u32x4_t pack16(const float (&f)[VEC<E>]) {
  u32x4_t v;
  if constexpr (std::is_same<E, float>::value) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __float_as_uint(f[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = pack_bf16x2(f[2 * i], f[2 * i + 1]);
  }
  return v;
}

__device__ __forceinline__ float weight_of(const void* w, bool f32, int64_t p) {
  return f32 ? static_cast<const float*>(w)[p] : bf16_to_f32(static_cast<const uint16_t*>(w)[p]);
}

__device__ __forceinline__ float wave_add(float v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// The rows of token t's pairs (-1: none), wave-uniform. Dispatch takes them from its indices and leaves -1 in the plan for the
// pairs that have none; everything after it looks at the plan alone, so that indices changed since reach nothing, and a plan
// that does not hold rows (below P = T*k) leads to none.
template <int KT, typename IdxT>
__device__ __forceinline__ void pair_rows(const IdxT* idx, int32_t* inv, int64_t t, int NE, int64_t P, int64_t (&row)[KT]) {
#pragma unroll
  for (int j = 0; j < KT; ++j) {
    bool ok = true;
    if constexpr (!std::is_void<IdxT>::value) {
      const int64_t e = (int64_t)idx[t * KT + j];
      ok = __builtin_amdgcn_readfirstlane((int)(e >= 0 && e < NE)) != 0;
    }
    const int64_t r = (int64_t)__builtin_amdgcn_readfirstlane(inv[t * KT + j]);
    row[j] = ok && r >= 0 && r < P ? r : (int64_t)-1;
    if constexpr (!std::is_void<IdxT>::value)
      if (!ok && (threadIdx.x & 63) == 0) inv[t * KT + j] = -1;
  }
}

template <typename E, typename IdxT, int KT>
__global__ __launch_bounds__(256) void spread_kernel(const E* __restrict__ src, const void* __restrict__ w, bool w_f32,
                                                     const E* __restrict__ y, const IdxT* __restrict__ idx,
                                                     int32_t* __restrict__ inv,
                                                     const int32_t* __restrict__ starts,
                                                     const int32_t* __restrict__ counts, E* __restrict__ dst,
                                                     void* __restrict__ dw, int64_t T, int h, int NE) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int64_t t = (int64_t)blockIdx.x * 4 + wave;
  if (t >= T) return;
  int64_t row[KT];
  pair_rows<KT, IdxT>(idx, inv, t, NE, T * KT, row);
  float s[KT], acc[KT];
#pragma unroll
  for (int j = 0; j < KT; ++j) {
    s[j] = w != nullptr ? weight_of(w, w_f32, t * KT + j) : 1.0f;
    acc[j] = 0.0f;
  }
  // U pieces of the row at c, c + 64 VEC, ...
  auto piece = [&](auto pieces, int c) {
    constexpr int U = decltype(pieces)::value, P = 64 * VEC<E>;
    u32x4_t a[U], b[U][KT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      a[u] = ld16(src + t * h + c + u * P);
      if (y != nullptr) {
#pragma unroll
        for (int j = 0; j < KT; ++j)
          b[u][j] = row[j] >= 0 ? ld16_stream(y + row[j] * h + c + u * P) : (u32x4_t){0u, 0u, 0u, 0u};
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float f[VEC<E>];
      unpack16<E>(a[u], f);
#pragma unroll
      for (int j = 0; j < KT; ++j) {
        if (row[j] < 0) continue;
        if (y != nullptr) {
          float g[VEC<E>];
          unpack16<E>(b[u][j], g);
#pragma unroll
          for (int i = 0; i < VEC<E>; ++i) acc[j] = fmaf(f[i], g[i], acc[j]);
        }
        if (dst != nullptr) {
          u32x4_t v = a[u];
          if (w != nullptr) {
            float g[VEC<E>];
#pragma unroll
            for (int i = 0; i < VEC<E>; ++i) g[i] = f[i] * s[j];
            v = pack16<E>(g);
          }
          st16_stream(dst + row[j] * h + c + u * P, v);
        }
      }
    }
  };
  // (Two pieces of y's rows at a time cost more registers than they hide: both gradients 75 us against 67.)
  int c = lane * VEC<E>;
  if (y == nullptr)
    for (; c + 64 * VEC<E> < h; c += 128 * VEC<E>) piece(std::integral_constant<int, 2>{}, c);
  for (; c < h; c += 64 * VEC<E>) piece(std::integral_constant<int, 1>{}, c);
  if (dw != nullptr) {
#pragma unroll
    for (int j = 0; j < KT; ++j) {
      const float r = wave_add(acc[j]);
      if (lane == 0) {
        if (w_f32) static_cast<float*>(dw)[t * KT + j] = r;
        else static_cast<uint16_t*>(dw)[t * KT + j] = (uint16_t)f32_to_bf16_rne(r);
      }
    }
  }
  if (dst != nullptr) {  // of the T*k rows, wave t looks after the zeros among rows t*k .. t*k + k - 1
    const int64_t filled = (int64_t)starts[NE - 1] + counts[NE - 1];
#pragma unroll
    for (int j = 0; j < KT; ++j) {
      const int64_t r = t * KT + j;
      if (r < filled) continue;
      for (int c = lane * VEC<E>; c < h; c += 64 * VEC<E>) st16(dst + r * h + c, (u32x4_t){0u, 0u, 0u, 0u});
    }
  }
}

// Dispatch of up to ROWS_SMALL pairs in one launch instead of three (histogram, permutation, spread): every block takes all
// pairs' experts into LDS and counts them, and a wave finds its token's rows as starts[e] + the earlier pairs of the same
// expert, 64 at a time by ballots, which is the stable order of the permutation. Between them the blocks write the whole
// plan. 305 pairs take 5.4 us on the GPU and 9.5 with the host's part, in three launches 8.7 and 16; 2560 pairs 8.8 and
// 9.6, 10.1 and 16.5; at 4096 the ballots cost as much as the launches (k = 2: 9.1 and 9.2 us on the GPU; k = 8: 11.9 and
// 10.4, but 11.6 and 16 with the host).
template <typename E, typename IdxT, int KT>
__global__ __launch_bounds__(256) void dispatch_small_kernel(const E* __restrict__ src, const IdxT* __restrict__ idx,
                                                             int32_t* __restrict__ counts, int32_t* __restrict__ starts,
                                                             int32_t* __restrict__ perm, int32_t* __restrict__ inv,
                                                             E* __restrict__ dst, int64_t T, int h, int NE) {
  constexpr int NONE = 255;
  __shared__ uint8_t ids[ROWS_SMALL];
  __shared__ int cnt[64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int P = (int)T * KT;
  if (threadIdx.x < 64) cnt[threadIdx.x] = 0;
  __syncthreads();
  for (int p = threadIdx.x; p < P; p += 256) {
    const int64_t e = (int64_t)idx[p];
    const bool ok = e >= 0 && e < NE;
    ids[p] = ok ? (uint8_t)e : (uint8_t)NONE;
    if (ok) atomicAdd(&cnt[e], 1);
  }
  __syncthreads();
  const int c = cnt[lane];  // lane = expert; none beyond NE
  int end = c;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(end, o);
    if (lane >= o) end += u;
  }
  const int start = end - c, filled = __shfl(end, 63);
  if (blockIdx.x == 0 && wave == 0 && lane < NE) {
    counts[lane] = c;
    starts[lane] = start;
  }
  const int t = (int)blockIdx.x * 4 + wave;
  if (t >= T) return;
  int e[KT], row[KT];
#pragma unroll
  for (int j = 0; j < KT; ++j) {
    e[j] = __builtin_amdgcn_readfirstlane((int)ids[t * KT + j]);
    row[j] = 0;
  }
  int p0 = 0;
  for (; p0 + 256 <= t * KT; p0 += 256) {  // all before the token's own pairs
    int v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] = ids[p0 + 64 * u + lane];
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int j = 0; j < KT; ++j) row[j] += __popcll(ballot64(v[u] == e[j]));
  }
  for (; p0 < t * KT + KT; p0 += 64) {
    const int p = p0 + lane, v = p < P ? (int)ids[p] : NONE;
#pragma unroll
    for (int j = 0; j < KT; ++j) row[j] += __popcll(ballot64(v == e[j] && p < t * KT + j));
  }
#pragma unroll
  for (int j = 0; j < KT; ++j) {
    row[j] = e[j] == NONE ? -1 : row[j] + __shfl(start, e[j] & 63);
    row[j] = __builtin_amdgcn_readfirstlane(row[j]);
    if (lane == 0) {
      inv[t * KT + j] = row[j];
      if (row[j] >= 0) perm[row[j]] = t * KT + j;
    }
  }
  for (int k = lane * VEC<E>; k < h; k += 64 * VEC<E>) {
    const u32x4_t v = ld16(src + (int64_t)t * h + k);
#pragma unroll
    for (int j = 0; j < KT; ++j) {
      if (row[j] >= 0) st16(dst + (int64_t)row[j] * h + k, v);
      if (t * KT + j >= filled) st16(dst + (int64_t)(t * KT + j) * h + k, (u32x4_t){0u, 0u, 0u, 0u});
    }
  }
}

template <typename E, int KT>
__global__ __launch_bounds__(256) void collect_kernel(const E* __restrict__ src, const void* __restrict__ w, bool w_f32,
                                                      int32_t* __restrict__ inv, E* __restrict__ out, int64_t T, int h) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int64_t t = (int64_t)blockIdx.x * 4 + wave;
  if (t >= T) return;
  int64_t row[KT];
  pair_rows<KT, void>(nullptr, inv, t, 0, T * KT, row);
  float s[KT];
#pragma unroll
  for (int j = 0; j < KT; ++j) s[j] = w != nullptr ? weight_of(w, w_f32, t * KT + j) : 1.0f;
  auto piece = [&](auto pieces, int c) {
    constexpr int U = decltype(pieces)::value, P = 64 * VEC<E>;
    u32x4_t b[U][KT];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < KT; ++j)
        b[u][j] = row[j] >= 0 ? ld16_stream(src + row[j] * h + c + u * P) : (u32x4_t){0u, 0u, 0u, 0u};
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float a[VEC<E>];
#pragma unroll
      for (int i = 0; i < VEC<E>; ++i) a[i] = 0.0f;
#pragma unroll
      for (int j = 0; j < KT; ++j) {
        if (row[j] < 0) continue;  // its weight may be anything
        float g[VEC<E>];
        unpack16<E>(b[u][j], g);
#pragma unroll
        for (int i = 0; i < VEC<E>; ++i) a[i] = fmaf(g[i], s[j], a[i]);
      }
      st16(out + t * h + c + u * P, pack16<E>(a));
    }
  };
  int c = lane * VEC<E>;
  for (; c + 64 * VEC<E> < h; c += 128 * VEC<E>) piece(std::integral_constant<int, 2>{}, c);
  if (c < h) piece(std::integral_constant<int, 1>{}, c);
}

template <typename E, typename IdxT>
hipError_t spread_k(const void* src, const void* w, bool w_f32, const void* y, const void* idx, int32_t* inv,
                    const int32_t* starts, const int32_t* counts, void* dst, void* dw, int64_t T, int h, int NE, int k,
                    hipStream_t st) {
  const dim3 grid((unsigned)((T + 3) / 4));
#define Q38_SPREAD(KT)                                                                                              \
  case KT:                                                                                                          \
    hipLaunchKernelGGL((spread_kernel<E, IdxT, KT>), grid, dim3(256), 0, st, (const E*)src, w, w_f32, (const E*)y,  \
                       (const IdxT*)idx, inv, starts, counts, (E*)dst, dw, T, h, NE);                               \
    break;
  switch (k) {
    Q38_SPREAD(1) Q38_SPREAD(2) Q38_SPREAD(3) Q38_SPREAD(4) Q38_SPREAD(5) Q38_SPREAD(6) Q38_SPREAD(7) Q38_SPREAD(8)
    default: return hipErrorInvalidValue;
  }
#undef Q38_SPREAD
  return hipGetLastError();
}

template <typename E, typename IdxT>
hipError_t dispatch_small_k(const void* src, const void* idx, int32_t* counts, int32_t* starts, int32_t* perm, int32_t* inv,
                            void* dst, int64_t T, int h, int NE, int k, hipStream_t st) {
  const dim3 grid((unsigned)((T + 3) / 4));
#define Q38_DISPATCH(KT)                                                                                          \
  case KT:                                                                                                        \
    hipLaunchKernelGGL((dispatch_small_kernel<E, IdxT, KT>), grid, dim3(256), 0, st, (const E*)src,               \
                       (const IdxT*)idx, counts, starts, perm, inv, (E*)dst, T, h, NE);                           \
    break;
  switch (k) {
    Q38_DISPATCH(1) Q38_DISPATCH(2) Q38_DISPATCH(3) Q38_DISPATCH(4) Q38_DISPATCH(5) Q38_DISPATCH(6) Q38_DISPATCH(7)
    Q38_DISPATCH(8)
    default: return hipErrorInvalidValue;
  }
#undef Q38_DISPATCH
  return hipGetLastError();
}

template <typename E>
hipError_t collect_k(const void* src, const void* w, bool w_f32, int32_t* inv, void* out, int64_t T, int h, int k,
                     hipStream_t st) {
  const dim3 grid((unsigned)((T + 3) / 4));
#define Q38_COLLECT(KT)                                                                                             \
  case KT:                                                                                                          \
    hipLaunchKernelGGL((collect_kernel<E, KT>), grid, dim3(256), 0, st, (const E*)src, w, w_f32, inv, (E*)out, T, h); \
    break;
  switch (k) {
    Q38_COLLECT(1) Q38_COLLECT(2) Q38_COLLECT(3) Q38_COLLECT(4) Q38_COLLECT(5) Q38_COLLECT(6) Q38_COLLECT(7)
    Q38_COLLECT(8)
    default: return hipErrorInvalidValue;
  }
#undef Q38_COLLECT
  return hipGetLastError();
}

template <typename E>
hipError_t spread_any(const void* src, const void* w, bool w_f32, const void* y, const void* idx, bool idx64, int32_t* inv,
                      const int32_t* starts, const int32_t* counts, void* dst, void* dw, int64_t T, int h, int NE, int k,
                      hipStream_t st) {
  if (idx == nullptr) return spread_k<E, void>(src, w, w_f32, y, idx, inv, starts, counts, dst, dw, T, h, NE, k, st);
  if (idx64) return spread_k<E, int64_t>(src, w, w_f32, y, idx, inv, starts, counts, dst, dw, T, h, NE, k, st);
  return spread_k<E, int32_t>(src, w, w_f32, y, idx, inv, starts, counts, dst, dw, T, h, NE, k, st);
}

}  // namespace

hipError_t launch_spread_rows(const void* src, const void* w, bool w_f32, const void* y, const void* idx, bool idx64,
                              int32_t* inv, const int32_t* starts, const int32_t* counts, void* dst, void* dw, int64_t T,
                              int h, int E, int k, bool bf16, hipStream_t st) {
  if (T == 0) return hipSuccess;
  return bf16 ? spread_any<uint16_t>(src, w, w_f32, y, idx, idx64, inv, starts, counts, dst, dw, T, h, E, k, st)
              : spread_any<float>(src, w, w_f32, y, idx, idx64, inv, starts, counts, dst, dw, T, h, E, k, st);
}

bool dispatch_is_small(int64_t T, int k) { return T > 0 && T * k <= ROWS_SMALL; }

hipError_t launch_dispatch_small(const void* src, const void* idx, bool idx64, int32_t* counts, int32_t* starts,
                                 int32_t* perm, int32_t* inv, void* dst, int64_t T, int h, int E, int k, bool bf16,
                                 hipStream_t st) {
  if (!dispatch_is_small(T, k)) return hipErrorInvalidValue;
  if (bf16)
    return idx64 ? dispatch_small_k<uint16_t, int64_t>(src, idx, counts, starts, perm, inv, dst, T, h, E, k, st)
                 : dispatch_small_k<uint16_t, int32_t>(src, idx, counts, starts, perm, inv, dst, T, h, E, k, st);
  return idx64 ? dispatch_small_k<float, int64_t>(src, idx, counts, starts, perm, inv, dst, T, h, E, k, st)
               : dispatch_small_k<float, int32_t>(src, idx, counts, starts, perm, inv, dst, T, h, E, k, st);
}

hipError_t launch_collect_rows(const void* src, const void* w, bool w_f32, const int32_t* inv, void* out, int64_t T, int h,
                               int k, bool bf16, hipStream_t st) {
  if (T == 0) return hipSuccess;
  int32_t* const plan = const_cast<int32_t*>(inv);  // only read without indices
  return bf16 ? collect_k<uint16_t>(src, w, w_f32, plan, out, T, h, k, st)
              : collect_k<float>(src, w, w_f32, plan, out, T, h, k, st);
}

}  // namespace q38
