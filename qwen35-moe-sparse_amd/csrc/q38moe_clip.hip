// Global norm of many tensors, and the tensors scaled to a largest norm.
//
//   N = (sum over all tensors and elements of |g|^p)^(1/p), p = 1, 2 or infinity (the largest |g|; a NaN stays one)
//   out = g * min(1, max_norm / (N + 1e-6)), one fp32 product rounded to the output's type
//
// Both passes are bound by memory: each element is read for the norm and once more for the product, since the
// coefficient needs all of them. The tensors' addresses and sizes go to the kernels by value, 96 tensors to a launch, so
// a call copies nothing to the device, can be captured, and takes two launches for up to 96 tensors. Elements are
// dealt in chunks, a block taking a run of neighbouring chunks. Sums are kept in fp64: squares of fp32 neither
// overflow nor vanish, and the order of the partial sums, which is fixed, hardly matters; at about six VALU
// operations per element against 15 that the memory's rate leaves, the conversions cost no time.
#include <type_traits>

#include "q38moe_common.h"
#include "q38moe_kernels.h"

namespace q38 {
namespace {

constexpr int CLIP_CHUNK = 16384;  // elements of a chunk

__device__ __forceinline__ double clip_fold(int ord, double a, double b) {
  if (ord != CLIP_INF) return a + b;
  return a != a || b != b ? __builtin_nan("") : (a > b ? a : b);
}

// One element's term.
template <int ORD>
__device__ __forceinline__ double clip_term(double acc, float f) {
  if constexpr (ORD == CLIP_L2) {
    const double d = (double)f;
    return __builtin_fma(d, d, acc);
  } else if constexpr (ORD == CLIP_L1) {
    return acc + (double)fabsf(f);
  } else {
    return clip_fold(CLIP_INF, acc, (double)fabsf(f));
  }
}

__device__ __forceinline__ double shfl_xor_d(double v, int o) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __shfl_xor((int)(uint32_t)u, o), hi = __shfl_xor((int)(uint32_t)(u >> 32), o);
  return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}

// The block's 256 values folded, in every thread (fixed order).
__device__ __forceinline__ double block_fold(int ord, double v, double* lds) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v = clip_fold(ord, v, shfl_xor_d(v, o));
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) lds[wave] = v;
  __syncthreads();
  return clip_fold(ord, clip_fold(ord, lds[0], lds[1]), clip_fold(ord, lds[2], lds[3]));
}

// The tensor that holds chunk c: the last one that starts at or before it.
__device__ __forceinline__ int tensor_of(const ClipTable& t, int64_t c) {
  int lo = 0, hi = t.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= c) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

template <int ORD>
__device__ __forceinline__ double chunk_norm_bf16(const uint16_t* p, int n, double acc) {
  const int tid = threadIdx.x;
  double a[4] = {acc, 0.0, 0.0, 0.0};
  int i = 0;
  if ((reinterpret_cast<uintptr_t>(p) & 15) == 0) {
    for (; i + 8192 <= n; i += 8192) {
      u32x4_t v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = ld16(p + i + 2048 * u + 8 * tid);
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float x, y;
          unpack_bf16x2(v[u][q], x, y);
          a[q] = clip_term<ORD>(a[q], x);
          a[q] = clip_term<ORD>(a[q], y);
        }
    }
    for (; i + 8 * tid + 8 <= n; i += 2048) {
      const u32x4_t v = ld16(p + i + 8 * tid);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float x, y;
        unpack_bf16x2(v[q], x, y);
        a[q] = clip_term<ORD>(a[q], x);
        a[q] = clip_term<ORD>(a[q], y);
      }
    }
    i = n & ~7;  // what 16-byte loads leave
  }
  for (int j = i + tid; j < n; j += 256) a[0] = clip_term<ORD>(a[0], bf16_to_f32(p[j]));
  return clip_fold(ORD, clip_fold(ORD, a[0], a[1]), clip_fold(ORD, a[2], a[3]));
}

template <int ORD>
__device__ __forceinline__ double chunk_norm_f32(const float* p, int n, double acc) {
  const int tid = threadIdx.x;
  double a[4] = {acc, 0.0, 0.0, 0.0};
  int i = 0;
  if ((reinterpret_cast<uintptr_t>(p) & 15) == 0) {
    for (; i + 4096 <= n; i += 4096) {
      u32x4_t v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = ld16(p + i + 1024 * u + 4 * tid);
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int q = 0; q < 4; ++q) a[q] = clip_term<ORD>(a[q], __uint_as_float(v[u][q]));
    }
    for (; i + 4 * tid + 4 <= n; i += 1024) {
      const u32x4_t v = ld16(p + i + 4 * tid);
#pragma unroll
      for (int q = 0; q < 4; ++q) a[q] = clip_term<ORD>(a[q], __uint_as_float(v[q]));
    }
    i = n & ~3;
  }
  for (int j = i + tid; j < n; j += 256) a[0] = clip_term<ORD>(a[0], p[j]);
  return clip_fold(ORD, clip_fold(ORD, a[0], a[1]), clip_fold(ORD, a[2], a[3]));
}

// partial[blockIdx.x] = this block's sum (or maximum).
template <int ORD>
__global__ __launch_bounds__(256) void norm_partial_kernel(const ClipTable t, double* __restrict__ partial) {
  __shared__ double lds[4];
  const int64_t chunks = t.first[t.n];
  const int64_t per = (chunks + gridDim.x - 1) / gridDim.x;
  const int64_t c0 = (int64_t)blockIdx.x * per, c1 = min(c0 + per, chunks);
  double acc = 0.0;
  if (c0 < c1) {
    int i = tensor_of(t, c0);
    for (int64_t c = c0; c < c1; ++c) {
      while (c >= t.first[i + 1]) ++i;
      const int64_t at = (c - t.first[i]) * CLIP_CHUNK;
      const int n = (int)min((int64_t)CLIP_CHUNK, t.numel[i] - at);
      acc = t.src_f32[i] ? chunk_norm_f32<ORD>(static_cast<const float*>(t.src[i]) + at, n, acc)
                         : chunk_norm_bf16<ORD>(static_cast<const uint16_t*>(t.src[i]) + at, n, acc);
    }
  }
  const double s = block_fold(ORD, acc, lds);
  if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

// The norm from all partials, in every thread of a 256-thread block.
__device__ __forceinline__ float norm_of(const double* partial, int n, int ord, double* lds) {
  double acc = 0.0;
  for (int i = threadIdx.x; i < n; i += 256) acc = clip_fold(ord, acc, partial[i]);
  const double s = block_fold(ord, acc, lds);
  return (float)(ord == CLIP_L2 ? sqrt(s) : s);
}

__global__ __launch_bounds__(256) void norm_finish_kernel(const double* __restrict__ partial, int n, int ord,
                                                          float* __restrict__ norm) {
  __shared__ double lds[4];
  const float v = norm_of(partial, n, ord, lds);
  if (threadIdx.x == 0) *norm = v;
}

// 4 elements as floats, and back: 8 or 16 bytes per lane, a wave's instruction whole lines either way.
__device__ __forceinline__ f32x4_t load4(const float* p) {
  return __builtin_nontemporal_load(reinterpret_cast<const f32x4_t*>(p));
}
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ f32x4_t load4(const uint16_t* p) {
  const u32x2_t v = __builtin_nontemporal_load(reinterpret_cast<const u32x2_t*>(p));
  f32x4_t f;
  float a, b;
  unpack_bf16x2(v[0], a, b);
  f[0] = a;
  f[1] = b;
  unpack_bf16x2(v[1], a, b);
  f[2] = a;
  f[3] = b;
  return f;
}
__device__ __forceinline__ void store4(float* p, f32x4_t f) {
  __builtin_nontemporal_store(f, reinterpret_cast<f32x4_t*>(p));
}
__device__ __forceinline__ void store4(uint16_t* p, f32x4_t f) {
  __builtin_nontemporal_store((u32x2_t){pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3])},
                              reinterpret_cast<u32x2_t*>(p));
}

template <typename S, typename D>
__device__ __forceinline__ void chunk_scale(const S* p, D* o, int n, float c) {
  const int tid = threadIdx.x;
  int i = 0;
  if ((reinterpret_cast<uintptr_t>(p) & (4 * sizeof(S) - 1)) == 0 &&
      (reinterpret_cast<uintptr_t>(o) & (4 * sizeof(D) - 1)) == 0) {
    for (; i + 4096 <= n; i += 4096) {
      f32x4_t f[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) f[u] = load4(p + i + 1024 * u + 4 * tid);
#pragma unroll
      for (int u = 0; u < 4; ++u) store4(o + i + 1024 * u + 4 * tid, f[u] * c);
    }
    for (; i + 4 * tid + 4 <= n; i += 1024) store4(o + i + 4 * tid, load4(p + i + 4 * tid) * c);
    i = n & ~3;
  }
  for (int j = i + tid; j < n; j += 256) {
    float f;
    if constexpr (sizeof(S) == 2) f = bf16_to_f32(p[j]);
    else f = p[j];
    f *= c;
    if constexpr (sizeof(D) == 2) o[j] = (uint16_t)f32_to_bf16_rne(f);
    else o[j] = f;
  }
}

// out = g * coefficient. The norm comes from the partials, summed by every block for itself, and block 0 stores it in *norm; or from
// *norm where there are none (more than one launch's partials are summed once instead). A block takes the chunks of its
// run backwards: the last ones that the first pass read are still in the caches (123 MB bf16: 48 us, 5.1 TB/s). That holds
// within a launch; of more than 96 tensors the launches come in the first pass's order, and one of 1 GB, read again after
// the three others, is read from memory (4.06 GB fp32: 4 x 430 us, 4.7 TB/s). In place with a coefficient of 1 nothing is
// written (the tensors already hold the result).
__global__ __launch_bounds__(256) void clip_scale_kernel(const ClipTable t, const double* __restrict__ partial,
                                                         int npartial, int ord, float max_norm, bool in_place,
                                                         float* __restrict__ norm) {
  __shared__ double lds[4];
  float N;
  if (npartial > 0) {
    N = norm_of(partial, npartial, ord, lds);
    if (blockIdx.x == 0 && threadIdx.x == 0) *norm = N;
  } else {
    N = *norm;
  }
  const float ratio = max_norm / (N + 1e-6f);
  const float c = ratio > 1.0f ? 1.0f : ratio;  // a NaN stays one
  if (in_place && c == 1.0f) return;
  const int64_t chunks = t.first[t.n];
  const int64_t per = (chunks + gridDim.x - 1) / gridDim.x;
  const int64_t c0 = (int64_t)blockIdx.x * per, c1 = min(c0 + per, chunks);
  if (c0 >= c1) return;
  int i = tensor_of(t, c1 - 1);
  for (int64_t k = c1 - 1; k >= c0; --k) {
    while (k < t.first[i]) --i;
    const int64_t at = (k - t.first[i]) * CLIP_CHUNK;
    const int n = (int)min((int64_t)CLIP_CHUNK, t.numel[i] - at);
    if (t.src_f32[i]) {
      const float* p = static_cast<const float*>(t.src[i]) + at;
      if (t.dst_f32[i]) chunk_scale(p, static_cast<float*>(t.dst[i]) + at, n, c);
      else chunk_scale(p, static_cast<uint16_t*>(t.dst[i]) + at, n, c);
    } else {
      const uint16_t* p = static_cast<const uint16_t*>(t.src[i]) + at;
      if (t.dst_f32[i]) chunk_scale(p, static_cast<float*>(t.dst[i]) + at, n, c);
      else chunk_scale(p, static_cast<uint16_t*>(t.dst[i]) + at, n, c);
    }
  }
}

}  // namespace

int clip_chunk() { return CLIP_CHUNK; }

static unsigned clip_grid(const ClipTable& t) {
  const int64_t chunks = t.first[t.n];
  return (unsigned)(chunks < CLIP_BLOCKS ? (chunks > 0 ? chunks : 1) : CLIP_BLOCKS);
}

hipError_t launch_norm_partial(const ClipTable& t, int ord, double* partial, int* blocks, hipStream_t st) {
  const dim3 grid(clip_grid(t));
  *blocks = (int)grid.x;
  if (ord == CLIP_L2) hipLaunchKernelGGL(norm_partial_kernel<CLIP_L2>, grid, dim3(256), 0, st, t, partial);
  else if (ord == CLIP_L1) hipLaunchKernelGGL(norm_partial_kernel<CLIP_L1>, grid, dim3(256), 0, st, t, partial);
  else hipLaunchKernelGGL(norm_partial_kernel<CLIP_INF>, grid, dim3(256), 0, st, t, partial);
  return hipGetLastError();
}

hipError_t launch_norm_finish(const double* partial, int n, int ord, float* norm, hipStream_t st) {
  hipLaunchKernelGGL(norm_finish_kernel, dim3(1), dim3(256), 0, st, partial, n, ord, norm);
  return hipGetLastError();
}

hipError_t launch_clip_scale(const ClipTable& t, const double* partial, int npartial, int ord, float max_norm,
                             bool in_place, float* norm, hipStream_t st) {
  hipLaunchKernelGGL(clip_scale_kernel, dim3(clip_grid(t)), dim3(256), 0, st, t, partial, npartial, ord, max_norm,
                     in_place, norm);
  return hipGetLastError();
}

}  // namespace q38
