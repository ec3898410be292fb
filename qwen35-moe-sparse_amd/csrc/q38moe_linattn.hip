// Linear attention with a decay for each head: for prompts and training in chunks of 64 tokens, and one token at a time.
//
//   S_t = e^g S_{t-1} + k_t v_t^T,   o_t = scale S_t^T q_t                     (S fp32 [dk, dv] per sequence and head)
// In a chunk that starts with the state S, with i, j its tokens:
//   o_i = scale (sum_{j <= i} e^{g (i - j)} (q_i . k_j) v_j + e^{g (i + 1)} S^T q_i)
//   S' = e^{g C} S + sum_j e^{g (C - 1 - j)} k_j v_j^T
// Every gradient is the same sum with the roles exchanged: dq that of (dO, v, k) over S^T; dk and dv those of (v, dO, q) and
// (k, q, dO) with the tokens taken backwards over the gradient of the state. So one kernel makes them all, forwards or
// backwards in time.
//
// A sequence is cut into segments of whole chunks that workgroups take at once: la_kernel<OUT = false> makes what each adds
// to the state, la_carry_kernel runs over the segments, la_kernel<OUT = true> goes through the chunks of each with the state
// in its accumulators.
//
// bf16 roundings: the weighted scores and the state that queries read, each once, as operands of the matrix units; what
// goes into the state itself is split into three bf16 parts (24 bits), so that the state is as exact as in fp32.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "q38moe_common.h"
#include "q38moe_kernels.h"

namespace q38 {
namespace {

constexpr int LA_C = 64;  // tokens of a chunk

typedef short la_i16x4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ uint2 la_read_tr(const uint8_t* lds) {
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) la_i16x4_t*)(
                                       uintptr_t)((const __attribute__((address_space(3))) uint8_t*)lds)));
}

__device__ __forceinline__ f32x4_t mfma16x16x4(float a, float b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// Byte of 16-byte column `col` of row `row` in a tile of rows of `bytes` bytes: the low three bits of the column are mixed with
// the row's, so that 8 rows' same column lies in 8 different bank groups.
__device__ __forceinline__ int la_at(int row, int col, int bytes) { return row * bytes + ((col ^ (row & 7)) << 4); }

// e^{g n} to 24 + 24 bits.
__device__ __forceinline__ float2 la_decay2(double g, int64_t n) {
  const double x = n == 0 ? 1.0 : exp(g * (double)n);
  const float hi = (float)x;
  return make_float2(hi, isinf(hi) || isnan(hi) ? 0.0f : (float)(x - (double)hi));
}

// Segment `seg` (OUT; else of those with another behind them, whose states are kept in a.mid): its sequence, that one's
// first token and length, and the place in it. `there` is false past the last one.
struct LaPlace {
  int seq, s, len, nseg;
  int64_t start;  // packed: the sequence's first token
  bool there;
};
template <bool OUT>
__device__ __forceinline__ LaPlace la_place(const LaArgs& a, int seg) {
  LaPlace p;
  if (a.plan == nullptr) {
    const int per = OUT ? a.nseg : a.nseg - 1;
    p = {seg / per, seg % per, a.S, a.nseg, 0, true};
    return p;
  }
  const int32_t* first = a.plan;
  auto before = [&](int n) { return OUT ? first[n] : first[n] - n; };
  p.there = seg < before(a.N);
  int lo = 0, hi = a.N - 1;  // the last sequence that starts at or before seg
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (before(mid) <= seg) lo = mid;
    else hi = mid - 1;
  }
  p.seq = lo;
  p.s = seg - before(lo);
  p.nseg = first[lo + 1] - first[lo];
  p.start = a.plan[a.N + 1 + lo];
  p.len = a.plan[2 * a.N + 1 + lo];
  return p;
}
// The place in a.mid of the state behind the sequence's first segment.
__device__ __forceinline__ int64_t la_slot(const LaArgs& a, int seq) {
  return a.plan == nullptr ? (int64_t)seq * (a.nseg - 1) : (int64_t)a.plan[seq] - seq;
}

// Packed sequences: first segment of each (and their number), first token and length. Offsets are brought into order and
// into [0, S], so that no later access leaves the tensors whatever they are.
__global__ __launch_bounds__(1024) void la_plan_kernel(const int32_t* __restrict__ cu, int32_t* __restrict__ plan, int N, int S,
                                                       int L) {
  __shared__ int tops[16], sums[16];
  __shared__ int top0, sum0;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (tid == 0) {
    top0 = 0;
    sum0 = 0;
  }
  __syncthreads();
  // end[n] = max over m <= n + 1 of cu[m], clamped: a running maximum; then a running sum of segments.
  for (int n0 = 0; n0 < N; n0 += 1024) {
    const int n = n0 + tid;
    int end = n < N ? min(max(cu[n + 1], 0), S) : 0;
    if (n == 0) end = max(end, min(max(cu[0], 0), S));
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(end, o);
      if (lane >= o) end = max(end, v);
    }
    if (lane == 63) tops[wave] = end;
    __syncthreads();
    int before = top0;
    for (int w = 0; w < wave; ++w) before = max(before, tops[w]);
    end = max(end, before);
    int start = __shfl_up(end, 1);
    if (lane == 0) start = before;
    if (n == 0) start = min(max(cu[0], 0), S);
    const int segs = n < N ? max(1, (end - start + L - 1) / L) : 0;
    int sum = segs;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(sum, o);
      if (lane >= o) sum += v;
    }
    if (lane == 63) sums[wave] = sum;
    __syncthreads();
    int base = sum0;
    for (int w = 0; w < wave; ++w) base += sums[w];
    if (n < N) {
      plan[n] = base + sum - segs;
      plan[N + 1 + n] = start;
      plan[2 * N + 1 + n] = end - start;
      if (n == N - 1) plan[N] = base + sum;
    }
    __syncthreads();
    if (tid == 1023) {
      top0 = end;
      sum0 = base + sum;
    }
    __syncthreads();
  }
}

// Rows of [T, heads, dv] that belong to no sequence: zeros.
__global__ __launch_bounds__(256) void la_gap_kernel(void* o, const int32_t* __restrict__ plan, int N, int64_t T, int row_bytes) {
  const int64_t from = plan[N + 1], to = plan[N + 1 + N - 1] + plan[2 * N + 1 + N - 1];
  const int per = row_bytes / 16;
  for (int64_t r = (int64_t)blockIdx.x * 64; r < min((int64_t)(blockIdx.x + 1) * 64, T); ++r) {
    if (r >= from && r < to) continue;
    for (int c = threadIdx.x; c < per; c += 256) st16(static_cast<uint8_t*>(o) + r * row_bytes + 16 * c, u32x4_t{0, 0, 0, 0});
  }
}

// 64 rows of up to D features on their way from memory to LDS, zero behind the last row and the last feature.
template <int BYTES>  // of a row of the tile
struct LaStage {
  static constexpr int COLS = BYTES / 16, N = LA_C * COLS / 256;
  u32x4_t r[N];
  template <bool REV>
  __device__ __forceinline__ void load(const uint8_t* base, int64_t stride, int len, int j0, int rows, int bytes) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (int)threadIdx.x + 256 * i, row = c / COLS, col = c % COLS, j = j0 + row;
      r[i] = u32x4_t{0, 0, 0, 0};
      if (row < rows && 16 * col < bytes) r[i] = ld16(base + (int64_t)(REV ? len - 1 - j : j) * stride + 16 * col);
    }
  }
  __device__ __forceinline__ void store(uint8_t* lds) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (int)threadIdx.x + 256 * i;
      *reinterpret_cast<u32x4_t*>(lds + la_at(c / COLS, c % COLS, BYTES)) = r[i];
    }
  }
};

// acc += rows of the tile (16 of them, the lane's is `row`) times the lane's column q, contiguous features.
template <bool BF16, int BYTES>
__device__ __forceinline__ f32x4_t la_dot(const uint8_t* tile, int row, int lq, const u32x4_t* q, f32x4_t acc) {
#pragma unroll
  for (int s = 0; s < BYTES / 64; ++s) {
    const u32x4_t x = *reinterpret_cast<const u32x4_t*>(tile + la_at(row, 4 * s + lq, BYTES));
    if constexpr (BF16) {
      acc = mfma16x16x32(x, q[s], acc);
    } else {
      const f32x4_t xf = __builtin_bit_cast(f32x4_t, x), qf = __builtin_bit_cast(f32x4_t, q[s]);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc = mfma16x16x4(xf[e], qf[e], acc);
    }
  }
  return acc;
}

// bf16: features 16 t .. of tokens 32 u + {4 lq + e, 16 + 4 lq + e} of a row-major tile, feature 16 t + lr in this lane.
template <int BYTES>
__device__ __forceinline__ u32x4_t la_column(const uint8_t* tile, int u, int t, int lr, int lq) {
  const int row = 32 * u + 4 * lq + (lr >> 2);
  const uint8_t* at = tile + la_at(row, 2 * t + ((lr & 3) >> 1), BYTES) + 8 * (lr & 1);
  const uint2 x = la_read_tr(at), y = la_read_tr(at + 16 * BYTES);
  return u32x4_t{x.x, x.y, y.x, y.y};
}
// fp32: feature 16 t + lr of token `row`.
template <int BYTES>
__device__ __forceinline__ float la_value(const uint8_t* tile, int row, int t, int lr) {
  return *reinterpret_cast<const float*>(tile + la_at(row, 4 * t + (lr >> 2), BYTES) + 4 * (lr & 3));
}

// One segment of one head. Wave w has queries 16 w .. of each chunk (scores as [key, query] tiles, outputs as [feature,
// query] tiles, so that scores go from accumulators to operands within a lane) and the state's columns w DV / 4 .. .
template <bool BF16, int DK, int DV, bool REV, bool OUT>
__global__ __launch_bounds__(256) void la_kernel(LaArgs a) {
  constexpr int ES = BF16 ? 2 : 4, KB = DK * ES, VB = DV * ES, NA = DK / 16, NB = DV / 64, NT = DV / 16;
  __shared__ __attribute__((aligned(16))) uint8_t Ks[LA_C * KB];
  __shared__ __attribute__((aligned(16))) uint8_t Vs[LA_C * VB];
  __shared__ __attribute__((aligned(16))) uint8_t Ss[OUT ? DV * KB : 16];  // the state as operand: [dv][dk]
  __shared__ float tab[LA_C + 1];
  const int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, lq = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int seg = (int)(blockIdx.x / a.H), h = (int)(blockIdx.x % a.H);
  const LaPlace p = la_place<OUT>(a, seg);
  if (!p.there) return;
  const double g = (double)a.g[h];
  if (tid <= LA_C) tab[tid] = la_decay2(g, tid).x;
  const float2 whole = la_decay2(g, LA_C);
  const int64_t first = a.plan == nullptr ? 0 : p.start;
  const int64_t sb = a.plan == nullptr ? p.seq : 0;
  auto at = [&](const LaTensor& t) {
    return static_cast<const uint8_t*>(t.p) + ES * (sb * t.sb + first * t.st + (int64_t)(h / t.div) * t.sh);
  };
  const uint8_t *qp = at(a.q), *kp = at(a.k), *vp = at(a.v);
  const int64_t qs = a.q.st * ES, ks = a.k.st * ES, vs = a.v.st * ES;
  const int begin = p.s * a.L, end = min(p.len, begin + a.L);
  const bool last = p.s == p.nseg - 1, keep = !OUT || (last && a.s1 != nullptr);

  // The state the segment starts with.
  f32x4_t S[NA][NB];
  const int64_t slot = la_slot(a, p.seq) + p.s;
  auto mid = [&](int64_t s, int i, int b) {
    return reinterpret_cast<f32x4_t*>(a.mid + (s * a.H + h) * (DK * DV) + (((w * NA + i) * NB + b) * 64 + lane) * 4);
  };
  auto user = [&](int i, int b, int e) {  // of the caller's state
    const int dk = 16 * i + 4 * lq + e, dv = 16 * (w * NB + b) + lr;
    return dk < a.dk && dv < a.dv ? ((int64_t)p.seq * a.H + h) * a.dk * a.dv + (a.turned ? dv * a.dk + dk : dk * a.dv + dv) : -1;
  };
#pragma unroll
  for (int i = 0; i < NA; ++i)
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      S[i][b] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
      if (!OUT) continue;
      if (p.s > 0) {
        S[i][b] = *mid(slot - 1, i, b);
      } else if (a.s0 != nullptr) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int64_t u = user(i, b, e);
          if (u >= 0) S[i][b][e] = a.s0[u];
        }
      }
    }
  auto publish = [&]() {
#pragma unroll
    for (int i = 0; i < NA; ++i)
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const int row = 16 * (w * NB + b) + lr;
        if constexpr (BF16) {
          uint8_t* to = Ss + la_at(row, 2 * i + (lq >> 1), KB) + 8 * (lq & 1);
          *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16x2(S[i][b][0], S[i][b][1]), pack_bf16x2(S[i][b][2], S[i][b][3]));
        } else {
          *reinterpret_cast<f32x4_t*>(Ss + la_at(row, 4 * i + lq, KB)) = S[i][b];
        }
      }
  };
  LaStage<KB> kst;
  LaStage<VB> vst;
  u32x4_t q[KB / 64], qn[KB / 64];
  auto fetch = [&](int j0) {
    const int rows = min(LA_C, end - j0);
    kst.template load<REV>(kp, ks, p.len, j0, rows, a.dk * ES);
    vst.template load<REV>(vp, vs, p.len, j0, rows, a.dv * ES);
    if (OUT) {
      const int j = j0 + 16 * w + lr;
#pragma unroll
      for (int s = 0; s < KB / 64; ++s) {
        qn[s] = u32x4_t{0, 0, 0, 0};
        if (j < end && 64 * s + 16 * lq < a.dk * ES)
          qn[s] = ld16(qp + (int64_t)(REV ? p.len - 1 - j : j) * qs + 64 * s + 16 * lq);
      }
    }
  };
  if (begin < end) {
    fetch(begin);
    kst.store(Ks);
    vst.store(Vs);
  }
  if (OUT) publish();
  for (int j0 = begin; j0 < end; j0 += LA_C) {
    const int rows = min(LA_C, end - j0);
    const bool more = j0 + LA_C < end;
    __syncthreads();
    if (OUT) {
#pragma unroll
      for (int s = 0; s < KB / 64; ++s) q[s] = qn[s];
    }
    if (more) fetch(j0 + LA_C);
    if (OUT) {
      f32x4_t o[NT], P[4];
      const float read = a.inter * tab[16 * w + lr + 1 - a.lag];
#pragma unroll
      for (int t = 0; t < NT; ++t)
        o[t] = la_dot<BF16, KB>(Ss, 16 * t + lr, lq, q, f32x4_t{0.0f, 0.0f, 0.0f, 0.0f}) * read;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        P[t] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
        if (t > w) continue;
        P[t] = la_dot<BF16, KB>(Ks, 16 * t + lr, lq, q, P[t]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int n = 16 * (w - t) + lr - 4 * lq - e;  // tokens between key and query
          P[t][e] = n >= 0 ? P[t][e] * (a.intra * tab[n < 0 ? 0 : n]) : 0.0f;
        }
      }
      if constexpr (BF16) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          if (2 * u > w) continue;
          const f32x4_t x = P[2 * u], y = P[2 * u + 1];
          const u32x4_t f = {pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
#pragma unroll
          for (int t = 0; t < NT; ++t) o[t] = mfma16x16x32(la_column<VB>(Vs, u, t, lr, lq), f, o[t]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (j > w) continue;
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int t = 0; t < NT; ++t) o[t] = mfma16x16x4(la_value<VB>(Vs, 16 * j + 4 * lq + e, t, lr), P[j][e], o[t]);
        }
      }
      // Lane: features 16 t + 4 lq .. + 3 of query 16 w + lr.
      const int j = j0 + 16 * w + lr;
      if (j < end) {
        const int64_t to = sb * a.ob + (first + (REV ? p.len - 1 - j : j)) * a.ot + (int64_t)h * a.oh;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const int c = 16 * t + 4 * lq;
          if (c >= a.dv) continue;
          if (BF16 && !a.o_f32)
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.o) + to + c) =
                make_uint2(pack_bf16x2(o[t][0], o[t][1]), pack_bf16x2(o[t][2], o[t][3]));
          else
            *reinterpret_cast<f32x4_t*>(static_cast<float*>(a.o) + to + c) = o[t];
        }
      }
    }
    if (more || keep) {
      const float2 full = rows == LA_C ? whole : la_decay2(g, rows);
#pragma unroll
      for (int i = 0; i < NA; ++i)
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int e = 0; e < 4; ++e) S[i][b][e] = fmaf(S[i][b][e], full.x, S[i][b][e] * full.y);
      const int gap = rows - 1 + a.lag;
      if constexpr (BF16) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          u32x4_t part[NB][3];
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            const u32x4_t v = la_column<VB>(Vs, u, w * NB + b, lr, lq);
#pragma unroll
            for (int z = 0; z < 4; ++z) {
              const int n = 32 * u + 16 * (z >> 1) + 4 * lq + 2 * (z & 1);  // token of the first of the two
              float x0, x1;
              unpack_bf16x2(v[z], x0, x1);
              x0 = n < rows ? x0 * (a.gain * tab[gap - min(n, gap)]) : 0.0f;
              x1 = n + 1 < rows ? x1 * (a.gain * tab[gap - min(n + 1, gap)]) : 0.0f;
#pragma unroll
              for (int y = 0; y < 3; ++y) {
                const uint32_t b0 = __float_as_uint(x0), b1 = __float_as_uint(x1);
                part[b][y][z] = __builtin_amdgcn_perm(b1, b0, 0x07060302u);  // the high halves
                x0 -= __uint_as_float(b0 & 0xffff0000u);
                x1 -= __uint_as_float(b1 & 0xffff0000u);
              }
            }
          }
#pragma unroll
          for (int i = 0; i < NA; ++i) {
            const u32x4_t k = la_column<KB>(Ks, u, i, lr, lq);
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
              for (int y = 0; y < 3; ++y) S[i][b] = mfma16x16x32(k, part[b][y], S[i][b]);
          }
        }
      } else {
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int n = 16 * t + 4 * lq + e;
            float v[NB];
#pragma unroll
            for (int b = 0; b < NB; ++b)
              v[b] = n < rows ? la_value<VB>(Vs, n, w * NB + b, lr) * (a.gain * tab[gap - min(n, gap)]) : 0.0f;
#pragma unroll
            for (int i = 0; i < NA; ++i) {
              const float k = la_value<KB>(Ks, n, i, lr);
#pragma unroll
              for (int b = 0; b < NB; ++b) S[i][b] = mfma16x16x4(k, v[b], S[i][b]);
            }
          }
      }
    }
    if (!more) break;
    __syncthreads();
    kst.store(Ks);
    vst.store(Vs);
    if (OUT) publish();
  }
  if (!keep) return;
#pragma unroll
  for (int i = 0; i < NA; ++i)
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      if (!OUT) {
        *mid(slot, i, b) = S[i][b];
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int64_t u = user(i, b, e);
          if (u >= 0) a.s1[u] = S[i][b][e];
        }
      }
    }
}

// mid[s] = e^{g L} (the state before segment s) + mid[s]: the state behind every segment but a sequence's last. A thread has 4
// elements of one state; reads run LA_AHEAD segments ahead.
constexpr int LA_AHEAD = 8;
template <int DK, int DV>
__global__ __launch_bounds__(256) void la_carry_kernel(LaArgs a) {
  constexpr int NA = DK / 16, NB = DV / 64;
  const int seq = (int)(blockIdx.x / a.H), h = (int)(blockIdx.x % a.H);
  const int idx = (int)(blockIdx.y * 256 + threadIdx.x);
  const int n = (a.plan == nullptr ? a.nseg : a.plan[seq + 1] - a.plan[seq]) - 1;
  if (n <= 0) return;
  const int64_t slot = la_slot(a, seq);
  const float2 whole = la_decay2((double)a.g[h], a.L);
  f32x4_t S = {0.0f, 0.0f, 0.0f, 0.0f};
  if (a.s0 != nullptr) {
    const int lane = idx & 63, b = (idx >> 6) % NB, i = (idx >> 6) / NB % NA, w = (idx >> 6) / NB / NA;
    const int dv = 16 * (w * NB + b) + (lane & 15);
    const int64_t base = ((int64_t)seq * a.H + h) * a.dk * a.dv;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int dk = 16 * i + 4 * (lane >> 4) + e;
      if (dk < a.dk && dv < a.dv) S[e] = a.s0[base + (a.turned ? dv * a.dk + dk : dk * a.dv + dv)];
    }
  }
  f32x4_t* p = reinterpret_cast<f32x4_t*>(a.mid + (slot * a.H + h) * (DK * DV) + 4 * idx);
  const int64_t step = (int64_t)a.H * DK * DV / 4;
  for (int s = 0; s < n; s += LA_AHEAD) {
    f32x4_t x[LA_AHEAD];
#pragma unroll
    for (int u = 0; u < LA_AHEAD; ++u)
      if (s + u < n) x[u] = p[(s + u) * step];
#pragma unroll
    for (int u = 0; u < LA_AHEAD; ++u) {
      if (s + u >= n) break;
#pragma unroll
      for (int e = 0; e < 4; ++e) S[e] = fmaf(S[e], whole.x, fmaf(S[e], whole.y, x[u][e]));
      p[(s + u) * step] = S;
    }
  }
}

// out[t][hk][c] = sum over the G heads that share hk of x[t][hk G + i][c], fp32 in, one rounding.
template <bool BF16>
__global__ __launch_bounds__(256) void la_group_kernel(const float* __restrict__ x, void* __restrict__ out, int64_t n4, int G, int d4) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n4; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / d4;
    const int c = (int)(i - row * d4);
    f32x4_t s = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int j = 0; j < G; ++j) s += *reinterpret_cast<const f32x4_t*>(x + ((row * G + j) * d4 + c) * 4);
    if (BF16)
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + 4 * i) = make_uint2(pack_bf16x2(s[0], s[1]), pack_bf16x2(s[2], s[3]));
    else
      *reinterpret_cast<f32x4_t*>(static_cast<float*>(out) + 4 * i) = s;
  }
}

// One token: S = e^g S + k v^T in place, o = scale S^T q. Workgroup: 32 columns of one state, thread: 4 columns of every 32nd
// row; HBM-bound, 8 bytes per element of the states.
template <bool BF16>
__global__ __launch_bounds__(256) void la_step_kernel(LaStepArgs a) {
  constexpr int ES = BF16 ? 2 : 4;
  __shared__ f32x4_t part[4][8];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int cols = (a.dv + 31) / 32;
  const int ct = (int)(blockIdx.x % cols), h = (int)(blockIdx.x / cols) % a.H;
  const int64_t b = blockIdx.x / cols / a.H;
  const int c = 32 * ct + 4 * (tid & 7);
  const bool there = c < a.dv;
  const int64_t to = (b * a.H + h) * a.dv + c;
  const int64_t slot = a.slots != nullptr ? a.slots[b] : b;
  auto load1 = [&](const LaTensor& t, int i) {
    const uint8_t* at = static_cast<const uint8_t*>(t.p) + ES * (b * t.st + (int64_t)(h / t.div) * t.sh + i);
    return BF16 ? bf16_to_f32(*reinterpret_cast<const uint16_t*>(at)) : *reinterpret_cast<const float*>(at);
  };
  f32x4_t o = {0.0f, 0.0f, 0.0f, 0.0f};
  if (slot >= 0 && slot < a.pool) {
    const float lam = (float)exp((double)a.g[h]);
    f32x4_t v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (there) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = load1(a.v, c + e);
    }
    float* S = a.state + (slot * a.H + h) * (int64_t)(a.dk * a.dv) + c;
#pragma unroll 4
    for (int r = tid >> 3; r < a.dk; r += 32) {
      if (!there) continue;
      f32x4_t s = *reinterpret_cast<const f32x4_t*>(S + (int64_t)r * a.dv);
      const float k = load1(a.k, r), q = load1(a.q, r);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[e] = fmaf(s[e], lam, k * v[e]);
        o[e] = fmaf(s[e], q, o[e]);
      }
      *reinterpret_cast<f32x4_t*>(S + (int64_t)r * a.dv) = s;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      o[e] += __shfl_xor(o[e], 8);
      o[e] += __shfl_xor(o[e], 16);
      o[e] += __shfl_xor(o[e], 32);
    }
  }
  if (lane < 8) part[w][lane] = o;
  __syncthreads();
  if (tid < 8 && there) {
    o = (part[0][tid] + part[1][tid]) + (part[2][tid] + part[3][tid]);
    o = o * a.scale;
    if (BF16)
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + to) = make_uint2(pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]));
    else
      *reinterpret_cast<f32x4_t*>(static_cast<float*>(a.out) + to) = o;
  }
}

template <bool BF16, int DK, int DV, bool REV>
hipError_t la_run(const LaArgs& a, int64_t segs, hipStream_t st) {
  const int64_t inner = segs - a.N;  // segments with another behind them, at most
  if (inner > 0) {
    hipLaunchKernelGGL((la_kernel<BF16, DK, DV, REV, false>), dim3((unsigned)(inner * a.H)), dim3(256), 0, st, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((la_carry_kernel<DK, DV>), dim3((unsigned)(a.N * a.H), DK * DV / 1024), dim3(256), 0, st, a);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL((la_kernel<BF16, DK, DV, REV, true>), dim3((unsigned)(segs * a.H)), dim3(256), 0, st, a);
  return hipGetLastError();
}

template <bool BF16, bool REV>
hipError_t la_run_d(const LaArgs& a, int64_t segs, hipStream_t st) {
  if (a.dk <= 64) return a.dv <= 64 ? la_run<BF16, 64, 64, REV>(a, segs, st) : la_run<BF16, 64, 128, REV>(a, segs, st);
  return a.dv <= 64 ? la_run<BF16, 128, 64, REV>(a, segs, st) : la_run<BF16, 128, 128, REV>(a, segs, st);
}

}  // namespace

int la_segment_tokens(int64_t T, int64_t N, int H) {
  // Segments of at least 8 chunks, as many as give every CU two workgroups.
  const int64_t want = std::max<int64_t>(1, 2 * (int64_t)device_cus() / H);
  const int64_t chunks = (T + LA_C * want - 1) / (LA_C * want);
  return (int)std::min<int64_t>(std::max<int64_t>(chunks, 8), 1 << 20) * LA_C;
}

int64_t la_padded_state(int dk, int dv) { return (int64_t)(dk <= 64 ? 64 : 128) * (dv <= 64 ? 64 : 128); }

hipError_t launch_la_plan(const int32_t* cu, int32_t* plan, int N, int S, int L, hipStream_t st) {
  hipLaunchKernelGGL(la_plan_kernel, dim3(1), dim3(1024), 0, st, cu, plan, N, S, L);
  return hipGetLastError();
}

hipError_t launch_la_gap(void* o, const int32_t* plan, int N, int64_t T, int row_bytes, hipStream_t st) {
  hipLaunchKernelGGL(la_gap_kernel, dim3((unsigned)((T + 63) / 64)), dim3(256), 0, st, o, plan, N, T, row_bytes);
  return hipGetLastError();
}

hipError_t launch_la(const LaArgs& a, int64_t segs, bool backwards, bool bf16, hipStream_t st) {
  if (backwards) return bf16 ? la_run_d<true, true>(a, segs, st) : la_run_d<false, true>(a, segs, st);
  return bf16 ? la_run_d<true, false>(a, segs, st) : la_run_d<false, false>(a, segs, st);
}

hipError_t launch_la_group(const float* x, void* out, int64_t rows, int G, int d, bool bf16, hipStream_t st) {
  const int64_t n4 = rows * (d / 4);
  const dim3 grid((unsigned)std::min<int64_t>((n4 + 255) / 256, 16 * (int64_t)device_cus()));
  if (n4 == 0) return hipSuccess;
  if (bf16) hipLaunchKernelGGL(la_group_kernel<true>, grid, dim3(256), 0, st, x, out, n4, G, d / 4);
  else hipLaunchKernelGGL(la_group_kernel<false>, grid, dim3(256), 0, st, x, out, n4, G, d / 4);
  return hipGetLastError();
}

hipError_t launch_la_step(const LaStepArgs& a, bool bf16, hipStream_t st) {
  const int64_t blocks = a.B * a.H * ((a.dv + 31) / 32);
  if (blocks == 0) return hipSuccess;
  if (bf16) hipLaunchKernelGGL(la_step_kernel<true>, dim3((unsigned)blocks), dim3(256), 0, st, a);
  else hipLaunchKernelGGL(la_step_kernel<false>, dim3((unsigned)blocks), dim3(256), 0, st, a);
  return hipGetLastError();
}

}  // namespace q38
