// Norms of queries and keys for each head and their rotation by position, in one pass, and the gradients.
//
//   n = x rsqrt(mean(x^2) + eps) w',  w' = 1 + w or w  (n = x without weights)
//   y[i] = n[i] cos a_i - n[i + r/2] sin a_i,  y[i + r/2] = n[i + r/2] cos a_i + n[i] sin a_i  (i < r/2),  y[i] = n[i] (i >= r)
//   a_i = position[axis_i] * inv_freq[i]
// and back, with dn the rotation of dy by -a, g = dn w', xh = x rstd:
//   dx = rstd (g - xh mean(g xh)),  dw = sum over tokens and heads of dn xh.
// fp32 throughout, one rounding of each result. The angle is a product in 64 bits, reduced to a fraction of a turn there
// (in 32 bits a position of 10^6 leaves an angle uncertain by 0.06); its sine and cosine are those of an fp32 fraction of a turn
// and of what it leaves of the angle (which alone is up to 2^-23, and all of a sine near half a turn).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "q38moe_common.h"
#include "q38moe_kernels.h"

namespace q38 {
namespace {

constexpr int ROPE_THREADS = 256;
constexpr int ROPE_TURNS = 2048;  // (cos, sin) pairs that a block keeps

template <bool BF16>
__device__ __forceinline__ void rope_ld4(const void* base, int64_t at, float* v) {
  if constexpr (BF16) {
    const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(base) + at);
    unpack_bf16x2(u.x, v[0], v[1]);
    unpack_bf16x2(u.y, v[2], v[3]);
  } else {
    const f32x4_t u = *reinterpret_cast<const f32x4_t*>(static_cast<const float*>(base) + at);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = u[e];
  }
}

template <bool BF16>
__device__ __forceinline__ void rope_st4(void* base, int64_t at, const float* v) {
  if constexpr (BF16)
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(base) + at) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
  else
    *reinterpret_cast<f32x4_t*>(static_cast<float*>(base) + at) = f32x4_t{v[0], v[1], v[2], v[3]};
}

// The turns of tokens t0 .. t0 + n: turns[token][i] = (cos a_i, sin a_i). An axis outside [0, p.axes) gives NaN.
__device__ __forceinline__ void rope_turns(const RopeArgs& p, int64_t t0, int n, float2* turns) {
  const int half = p.rot / 2;
  for (int u = threadIdx.x; u < n * half; u += ROPE_THREADS) {
    const int tok = u / half, i = u - tok * half;
    const int axis = p.axis_of != nullptr ? p.axis_of[i] : 0;
    float2 cs = make_float2(__builtin_nanf(""), __builtin_nanf(""));
    if (axis >= 0 && axis < p.axes) {
      const int64_t at = axis * p.T + t0 + tok;
      const double pos = p.pos64 ? (double)static_cast<const int64_t*>(p.pos)[at] : (double)static_cast<const int32_t*>(p.pos)[at];
      double turn = pos * (double)p.inv_freq[i] * 0.15915494309189533577;
      turn -= rint(turn);
      const float near = (float)turn, more = (float)(6.283185307179586 * (turn - (double)near));
      float s, c;
      sincospif(2.0f * near, &s, &c);
      cs = make_float2(fmaf(-more, s, c), fmaf(more, c, s));  // the rest of the angle, at most 2^-23: to the first order
    }
    turns[u] = cs;
  }
}

// A lane's 8 features of a head: unit u < rot / 8 holds 4 u .. + 3 and their partners rot / 2 further on, the others
// 8 u .. + 7, so that a rotation stays within a lane.
struct RopeUnit {
  int lo, hi;
  bool turned, there;
};
__device__ __forceinline__ RopeUnit rope_unit(int u, int d, int rot) {
  const bool turned = u < rot / 8;
  return {turned ? 4 * u : 8 * u, turned ? rot / 2 + 4 * u : 8 * u + 4, turned, 8 * u < d};
}

template <bool BF16>
__device__ __forceinline__ void rope_weight(const void* w, const RopeUnit& un, bool plus1, float* out) {
#pragma unroll
  for (int e = 0; e < 8; ++e) out[e] = 1.0f;
  if (w == nullptr || !un.there) return;
  rope_ld4<BF16>(w, un.lo, out);
  rope_ld4<BF16>(w, un.hi, out + 4);
#pragma unroll
  for (int e = 0; e < 8; ++e) out[e] += plus1 ? 1.0f : 0.0f;
}

template <int LPH>
__device__ __forceinline__ float head_sum(float v) {
#pragma unroll
  for (int o = 1; o < LPH; o <<= 1) v += __shfl_xor(v, o);
  return v;
}

// One block per p.tokens tokens, LPH lanes per head (d / 8 up to a power of two), every head of a token in turn: the turns of
// a token are made once for all of its heads. HBM-bound: 16384 tokens x 40 heads of 64 bf16 take 40 us (median; 168 MB, 4.2 TB/s; a
// large copy reaches 5.1), 4097 x 18 of 256 19.0 us (76 MB, 4.0 TB/s).
template <bool BF16, int LPH>
__global__ __launch_bounds__(ROPE_THREADS) void rope_kernel(RopeArgs p) {
  __shared__ float2 turns[ROPE_TURNS];
  const int64_t t0 = (int64_t)blockIdx.x * p.tokens;
  const int n = (int)min((int64_t)p.tokens, p.T - t0);
  rope_turns(p, t0, n, turns);
  const RopeUnit un = rope_unit(threadIdx.x % LPH, p.d, p.rot);
  float wq[8], wk[8];
  rope_weight<BF16>(p.wq, un, p.plus1, wq);
  rope_weight<BF16>(p.wk, un, p.plus1, wk);
  __syncthreads();
  const int heads = p.H + p.KV, rows = n * heads;
  for (int r = threadIdx.x / LPH; r < rows; r += ROPE_THREADS / LPH) {
    const int tok = r / heads, h = r - tok * heads;
    const bool isq = h < p.H;
    const int64_t t = t0 + tok;
    const void* src = isq ? p.q : p.k;
    const int64_t from = isq ? t * p.q_token + h * p.q_head : t * p.k_token + (h - p.H) * p.k_head;
    float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (un.there) {
      rope_ld4<BF16>(src, from + un.lo, x);
      rope_ld4<BF16>(src, from + un.hi, x + 4);
    }
    if ((isq ? p.wq : p.wk) != nullptr) {
      float s = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) s = fmaf(x[e], x[e], s);
      const float rstd = rsqrtf(head_sum<LPH>(s) / (float)p.d + p.eps);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = x[e] * rstd * (isq ? wq[e] : wk[e]);
    }
    if (!un.there) continue;
    if (un.turned) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 cs = turns[tok * (p.rot / 2) + un.lo + e];
        const float a = x[e], b = x[e + 4];
        x[e] = a * cs.x - b * cs.y;
        x[e + 4] = b * cs.x + a * cs.y;
      }
    }
    void* dst = isq ? p.q_out : p.k_out;
    const int64_t to = isq ? (t * p.H + h) * p.d : (t * p.KV + h - p.H) * p.d;
    rope_st4<BF16>(dst, to + un.lo, x);
    rope_st4<BF16>(dst, to + un.hi, x + 4);
  }
}

// The gradients: blocks take groups of p.tokens tokens in turn; a lane keeps the weights' gradients of its 8 features, the
// block's go to partial[block][2][d] and rope_dw_kernel adds them in a fixed order. HBM-bound: 16384 tokens x 40 heads of 64 bf16
// take 58 us (median; 252 MB, 4.3 TB/s); 6 and 8 blocks a CU instead of 4, and two rows at a time, take as long.
template <bool BF16, int LPH>
__global__ __launch_bounds__(ROPE_THREADS) void rope_backward_kernel(RopeArgs p, const void* __restrict__ dyq,
                                                                     const void* __restrict__ dyk, float* __restrict__ partial) {
  __shared__ float2 turns[ROPE_TURNS];
  __shared__ float sums[ROPE_THREADS * 8];
  const RopeUnit un = rope_unit(threadIdx.x % LPH, p.d, p.rot);
  float wq[8], wk[8], aq[8], ak[8];
  rope_weight<BF16>(p.wq, un, p.plus1, wq);
  rope_weight<BF16>(p.wk, un, p.plus1, wk);
#pragma unroll
  for (int e = 0; e < 8; ++e) aq[e] = ak[e] = 0.0f;
  const int heads = p.H + p.KV;
  for (int64_t t0 = (int64_t)blockIdx.x * p.tokens; t0 < p.T; t0 += (int64_t)gridDim.x * p.tokens) {
    const int n = (int)min((int64_t)p.tokens, p.T - t0), rows = n * heads;
    __syncthreads();
    rope_turns(p, t0, n, turns);
    __syncthreads();
    for (int r = threadIdx.x / LPH; r < rows; r += ROPE_THREADS / LPH) {
      const int tok = r / heads, h = r - tok * heads;
      const bool isq = h < p.H, normed = (isq ? p.wq : p.wk) != nullptr;
      const int64_t t = t0 + tok;
      const int64_t from = isq ? t * p.q_token + h * p.q_head : t * p.k_token + (h - p.H) * p.k_head;
      const int64_t to = isq ? (t * p.H + h) * p.d : (t * p.KV + h - p.H) * p.d;
      float x[8] = {0, 0, 0, 0, 0, 0, 0, 0}, g[8] = {0, 0, 0, 0, 0, 0, 0, 0};
      if (un.there) {
        rope_ld4<BF16>(isq ? dyq : dyk, to + un.lo, g);
        rope_ld4<BF16>(isq ? dyq : dyk, to + un.hi, g + 4);
        if (normed) {
          rope_ld4<BF16>(isq ? p.q : p.k, from + un.lo, x);
          rope_ld4<BF16>(isq ? p.q : p.k, from + un.hi, x + 4);
        }
      }
      if (un.there && un.turned) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 cs = turns[tok * (p.rot / 2) + un.lo + e];
          const float a = g[e], b = g[e + 4];
          g[e] = a * cs.x + b * cs.y;
          g[e + 4] = b * cs.x - a * cs.y;
        }
      }
      if (normed) {
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) s = fmaf(x[e], x[e], s);
        const float rstd = rsqrtf(head_sum<LPH>(s) / (float)p.d + p.eps);
        float dot = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[e] *= rstd;
          if (isq) aq[e] = fmaf(g[e], x[e], aq[e]);
          else ak[e] = fmaf(g[e], x[e], ak[e]);
          g[e] *= isq ? wq[e] : wk[e];
          dot = fmaf(g[e], x[e], dot);
        }
        dot = head_sum<LPH>(dot) / (float)p.d;
#pragma unroll
        for (int e = 0; e < 8; ++e) g[e] = rstd * (g[e] - x[e] * dot);
      }
      if (!un.there) continue;
      rope_st4<BF16>(isq ? p.q_out : p.k_out, to + un.lo, g);
      rope_st4<BF16>(isq ? p.q_out : p.k_out, to + un.hi, g + 4);
    }
  }
  if (partial == nullptr) return;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    __syncthreads();
    if (un.there) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        sums[(threadIdx.x / LPH) * p.d + (e < 4 ? un.lo + e : un.hi + e - 4)] = which == 0 ? aq[e] : ak[e];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < p.d; c += ROPE_THREADS) {
      float s = 0.0f;
      for (int r = 0; r < ROPE_THREADS / LPH; ++r) s += sums[r * p.d + c];
      partial[((int64_t)blockIdx.x * 2 + which) * p.d + c] = s;
    }
  }
}

// dw[which][c] = sum over blocks of partial[block][which][c], in fp64: 16 columns a block, 64 threads each (16 threads: 4.8 us
// where these take 3, of 1024 blocks' sums).
template <bool BF16>
__global__ __launch_bounds__(1024) void rope_dw_kernel(const float* __restrict__ partial, int blocks, int d, void* dwq, void* dwk) {
  __shared__ double s[64][17];
  const int which = blockIdx.y, c = blockIdx.x * 16 + threadIdx.x % 16, g = threadIdx.x / 16;
  double v = 0.0;
  if (c < d) {
#pragma unroll 8
    for (int b = g; b < blocks; b += 64) v += (double)partial[((int64_t)b * 2 + which) * d + c];
  }
  s[g][threadIdx.x % 16] = v;
  __syncthreads();
  void* dst = which == 0 ? dwq : dwk;
  if (threadIdx.x < 16 && c < d && dst != nullptr) {
    double sum = 0.0;
    for (int r = 0; r < 64; ++r) sum += s[r][threadIdx.x];
    if (BF16) static_cast<uint16_t*>(dst)[c] = (uint16_t)f32_to_bf16_rne((float)sum);
    else static_cast<float*>(dst)[c] = (float)sum;
  }
}

// Calls f(std::integral_constant<int, lanes per head>).
template <class F>
void with_lanes(int d, F f) {
  if (d <= 8) f(std::integral_constant<int, 1>());
  else if (d <= 16) f(std::integral_constant<int, 2>());
  else if (d <= 32) f(std::integral_constant<int, 4>());
  else if (d <= 64) f(std::integral_constant<int, 8>());
  else if (d <= 128) f(std::integral_constant<int, 16>());
  else f(std::integral_constant<int, 32>());
}

// Tokens of a block: about 8 rows for every slot of LPH lanes, fewer where that leaves CUs without a block.
int rope_tokens(const RopeArgs& p) {
  int lanes = 1;
  while (lanes * 8 < p.d) lanes *= 2;
  const int64_t most = std::max<int64_t>(1, 8 * (ROPE_THREADS / lanes) / (p.H + p.KV));
  const int64_t fill = std::max<int64_t>(1, p.T / (4 * (int64_t)device_cus()));
  return (int)std::min({most, fill, (int64_t)(ROPE_TURNS / std::max(1, p.rot / 2))});
}

}  // namespace

hipError_t launch_rope(RopeArgs p, bool bf16, hipStream_t st) {
  if (p.T == 0) return hipSuccess;
  p.tokens = rope_tokens(p);
  const dim3 grid((unsigned)((p.T + p.tokens - 1) / p.tokens));
  with_lanes(p.d, [&](auto lph) {
    if (bf16) hipLaunchKernelGGL((rope_kernel<true, decltype(lph)::value>), grid, dim3(ROPE_THREADS), 0, st, p);
    else hipLaunchKernelGGL((rope_kernel<false, decltype(lph)::value>), grid, dim3(ROPE_THREADS), 0, st, p);
  });
  return hipGetLastError();
}

int rope_backward_blocks(const RopeArgs& p) {
  const int64_t groups = (p.T + rope_tokens(p) - 1) / rope_tokens(p);
  return (int)std::min<int64_t>(groups, 4 * (int64_t)device_cus());
}

hipError_t launch_rope_backward(RopeArgs p, const void* dyq, const void* dyk, float* partial, void* dwq, void* dwk, bool bf16,
                                hipStream_t st) {
  p.tokens = rope_tokens(p);
  const int blocks = rope_backward_blocks(p);
  if (blocks > 0) {
    with_lanes(p.d, [&](auto lph) {
      constexpr int L = decltype(lph)::value;
      if (bf16) hipLaunchKernelGGL((rope_backward_kernel<true, L>), dim3(blocks), dim3(ROPE_THREADS), 0, st, p, dyq, dyk, partial);
      else hipLaunchKernelGGL((rope_backward_kernel<false, L>), dim3(blocks), dim3(ROPE_THREADS), 0, st, p, dyq, dyk, partial);
    });
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if (dwq == nullptr && dwk == nullptr) return hipSuccess;
  const dim3 grid((unsigned)((p.d + 15) / 16), 2);
  if (bf16) hipLaunchKernelGGL(rope_dw_kernel<true>, grid, dim3(1024), 0, st, partial, blocks, p.d, dwq, dwk);
  else hipLaunchKernelGGL(rope_dw_kernel<false>, grid, dim3(1024), 0, st, partial, blocks, p.d, dwq, dwk);
  return hipGetLastError();
}

}  // namespace q38
