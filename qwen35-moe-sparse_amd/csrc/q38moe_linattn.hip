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
// bf16 roundings: the weighted scores and the state that queries read are operands of the matrix units in two bf16 parts (16
// bits: off by 2^-16 of themselves at most, where rounding a result leaves 2^-8 of that): a result is as near to exact as its own
// rounding. With the state in one part it was 0.0021 off (norm of the error over the result's), so 0.0017, for 4 x 4096 tokens x 16
// heads of 128 forward and back in 346 us, not 331. What goes into the state itself is split into three parts (24 bits), so that
// the state is as exact as in fp32.
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

// A tile of rows of BYTES bytes: where row `row` has its 16-byte column `col`. The columns are mixed with the row so that the
// lanes that a read serves at once (16 bytes: rows 0-3 and 12-15 of a column and 4-11 of the next; 8 bytes, transposing: two
// columns of 8 rows, or four half ones; 4 bytes, fp32: one column of rows 4 apart) find their data in different banks. Half columns
// of bf16 tiles are exchanged in every other row where `swapped` says so (la_row's reads).
template <bool BF16, int BYTES>
struct LaTile {
  static __device__ __forceinline__ int key(int row) { return !BF16 ? row & 15 : BYTES == 128 ? row & 6 : 2 * (row & 7); }
  static __device__ __forceinline__ int at(int row, int col) { return row * BYTES + ((col ^ key(row)) << 4); }
  static __device__ __forceinline__ bool swapped(int row) { return (BYTES == 128 ? row >> 1 : row) & 1; }
};

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
  // The last sequence that starts at or before seg: the wave's lanes look at 64 places at once.
  int lo = 0;
  for (int step = a.N; step > 1;) {
    const int each = (step + 63) / 64, n = lo + each * ((int)threadIdx.x & 63);
    const uint64_t at = ballot64(n < min(lo + step, a.N) && before(n) <= seg);
    lo += each * max(0, 63 - __builtin_clzll(at | 1));
    step = each;
  }
  lo = __builtin_amdgcn_readfirstlane(lo);
  p.seq = lo;
  p.s = __builtin_amdgcn_readfirstlane(seg - before(lo));
  p.nseg = __builtin_amdgcn_readfirstlane(first[lo + 1] - first[lo]);
  p.start = __builtin_amdgcn_readfirstlane(a.plan[a.N + 1 + lo]);
  p.len = __builtin_amdgcn_readfirstlane(a.plan[2 * a.N + 1 + lo]);
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

// Rows 64 block .. of `out` (row_bytes each) that belong to no packed sequence: zeros. The workgroups behind those of the
// segments do this.
__device__ __forceinline__ void la_gap(const LaArgs& a, void* out, int row_bytes, int block) {
  const int32_t* start = a.plan + a.N + 1;
  const int from = start[0], to = start[a.N - 1] + start[2 * a.N - 1], per = row_bytes / 16;
  for (int r = 64 * block; r < min(64 * (block + 1), a.S); ++r) {
    if (r >= from && r < to) continue;
    for (int c = threadIdx.x; c < per; c += blockDim.x)
      st16(static_cast<uint8_t*>(out) + (int64_t)r * row_bytes + 16 * c, u32x4_t{0, 0, 0, 0});
  }
}

// 64 rows of features on their way from memory to LDS, zero behind the last row and the last feature.
template <bool BF16, int BYTES, int THREADS>
struct LaStage {
  using Tile = LaTile<BF16, BYTES>;
  static constexpr int COLS = BYTES / 16, N = (LA_C * COLS + THREADS - 1) / THREADS, ROWS = THREADS / COLS;
  static constexpr bool EVEN = N * ROWS == LA_C;
  u32x4_t r[N];
  const uint8_t* at;  // the thread's first piece of the next 64 rows
  int64_t step;       // bytes from row to row, negative backwards
  __device__ __forceinline__ void start(const uint8_t* base, int64_t stride, int j0) {
    step = stride;
    at = base + (j0 + (int)threadIdx.x / COLS) * stride + 16 * ((int)threadIdx.x % COLS);
  }
  __device__ __forceinline__ void load(int tid, int rows, int bytes) {
    const int row = tid / COLS, col = tid % COLS;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      r[i] = u32x4_t{0, 0, 0, 0};
      if (row + ROWS * i < rows && 16 * col < bytes) r[i] = ld16(at + ROWS * i * step);
    }
    at += LA_C * step;
  }
  // SWAP: with the 8-byte halves of odd rows' columns exchanged.
  template <bool SWAP>
  __device__ __forceinline__ void store(int tid, uint8_t* lds) const {
    const int row = tid / COLS, col = tid % COLS;
    static_assert(ROWS % 4 == 0, "the rows of a thread are all swapped or none");
    const bool swap = SWAP && Tile::swapped(row);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (EVEN || row + ROWS * i < LA_C)
        *reinterpret_cast<u32x4_t*>(lds + Tile::at(row + ROWS * i, col)) =
            swap ? u32x4_t{r[i][2], r[i][3], r[i][0], r[i][1]} : r[i];
  }
  // The next 64 rows straight into a tile, asynchronously. Places behind the last row or feature get others of the same kind,
  // since a copy cannot leave zeros: rows that are not stored, and features that meet zeros of the state and of the keys.
  __device__ __forceinline__ void copy(int tid, uint8_t* lds, int rows, int bytes) {
    static_assert(EVEN, "every thread copies");
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int row = tid / COLS + ROWS * i, col = tid % COLS ^ Tile::key(row);
      load_lds16(at + (min(row, rows - 1) - tid / COLS) * step + 16 * (min(col, bytes / 16 - 1) - tid % COLS),
                 lds + 16 * (THREADS * i + (tid & ~63)));
    }
    at += LA_C * step;
  }
};

// Two pieces of 4 tokens (rows `row` + {0, 16}) of one feature, transposed out of a row-major bf16 tile: the lane addresses 4
// features at byte `at` of its row (lr / 4 of the 4 rows) and gets feature lr of the 16 that its group addresses.
template <int BYTES>
__device__ __forceinline__ u32x4_t la_column(const uint8_t* at) {
  const uint2 x = la_read_tr(at), y = la_read_tr(at + 16 * BYTES);
  return u32x4_t{x.x, x.y, y.x, y.y};
}

__device__ __forceinline__ u32x4_t la_pack(f32x4_t x, f32x4_t y) {
  return u32x4_t{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
}

// What la_pack(x, y) left, rounded. An infinity leaves a NaN.
__device__ __forceinline__ u32x4_t la_left(f32x4_t x, f32x4_t y, u32x4_t packed) {
#pragma unroll
  for (int z = 0; z < 4; ++z) {
    float x0, x1;
    unpack_bf16x2(packed[z], x0, x1);
    f32x4_t& of = z < 2 ? x : y;
    of[2 * (z & 1)] -= x0;
    of[2 * (z & 1) + 1] -= x1;
  }
  return la_pack(x, y);
}

// x, but not as the compiler knows it: what follows from it is made again in every chunk rather than kept in registers that
// the loop lacks.
__device__ __forceinline__ int afresh(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// Waves on a SIMD that the LDS of la_kernel's workgroups allows, at most 4: the limit of its registers.
constexpr int la_waves(bool bf16, int dk, int dv, bool out) {
  return bf16 ? (out && dk == 128 && dv == 64 ? 2 : 4) : out && dk == 128 && dv == 64 ? 1 : 2;
}

// The scores of a chunk: units of 32 keys (32 u ..) and 16 queries (16 t ..), those with a key at or before a query.
constexpr int LA_UNITS = 6;
__device__ __forceinline__ int la_unit_queries(int unit) { return (0x201233 >> (4 * unit)) & 15; }
__device__ __forceinline__ int la_unit_keys(int unit) { return (0x22 >> unit) & 1; }
constexpr int la_unit(int t, int u) { return t == 3 ? u : t == 2 ? 2 + 3 * u : 4 - t; }

// First of the 4 rows of the state that accumulator tile i has in lanes 16 q .. : bf16 tiles 2 u and 2 u + 1 share groups of 8
// rows, so that a lane's rows of both, rounded, are 8 features in a row: an operand against the queries as they lie.
template <bool BF16>
__device__ __forceinline__ int la_row(int i, int q) {
  return BF16 ? 32 * (i >> 1) + 8 * q + 4 * (i & 1) : 16 * i + 4 * q;
}

// bf16: one unit's scores, weighted, to `to` as operands: rounded, and behind the units what that left. KEYS_SWAPPED: the keys' odd
// rows lie with the halves of their columns exchanged. row_at: see la_kernel.
constexpr int LA_SCORES = LA_UNITS * 1024;
template <int BYTES, bool KEYS_SWAPPED>
__device__ __forceinline__ void la_scores(const uint8_t* keys, const uint8_t* queries, uint8_t* to, int unit, int lr, int lq,
                                          int row_at, float intra, const float2* tab) {
  const int t = la_unit_queries(unit), u = la_unit_keys(unit);
  auto key = [&](const uint8_t* at) {
    const u32x4_t k = *reinterpret_cast<const u32x4_t*>(at);
    return KEYS_SWAPPED && LaTile<true, BYTES>::swapped(lr) ? u32x4_t{k[2], k[3], k[0], k[1]} : k;
  };
  f32x4_t P[2];
  P[0] = P[1] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int s = 0; s < BYTES / 64; ++s) {
    const uint8_t* x = keys + (row_at ^ (64 * s)) + 32 * BYTES * u;
    const u32x4_t q = *reinterpret_cast<const u32x4_t*>(queries + (row_at ^ (64 * s)) + 16 * BYTES * t);
    P[0] = mfma16x16x32(key(x), q, P[0]);
    if (2 * u + 1 <= t) P[1] = mfma16x16x32(key(x + 16 * BYTES), q, P[1]);
  }
  float decay[2][4];
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) decay[k][e] = tab[max(16 * (t - 2 * u - k) + lr - 4 * lq - e, 0)].x;
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) asm volatile("" : "+v"(decay[k][e]));  // all at once, none behind a branch on its place
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int n = 16 * (t - 2 * u - k) + lr - 4 * lq - e;  // tokens between key and query
      P[k][e] = n >= 0 ? P[k][e] * (intra * decay[k][e]) : 0.0f;
    }
  const u32x4_t high = la_pack(P[0], P[1]);
#pragma unroll
  for (int z = 0; z < 4; ++z) {
    float x0, x1;
    unpack_bf16x2(high[z], x0, x1);
    const int e = 2 * (z & 1);
    const float y0 = P[z >> 1][e] - x0, y1 = P[z >> 1][e + 1] - x1;
    P[z >> 1][e] = y0 == y0 ? y0 : 0.0f;  // an infinity leaves nothing
    P[z >> 1][e + 1] = y1 == y1 ? y1 : 0.0f;
  }
  uint8_t* const at = to + (unit * 64 + 16 * lq + lr) * 16;
  *reinterpret_cast<u32x4_t*>(at) = high;
  *reinterpret_cast<u32x4_t*>(at + LA_SCORES) = la_pack(P[0], P[1]);
}

// bf16: S = e^{g rows} S + the chunk's k v^T. v: the wave's column's tokens as operands; k: the row-major tile of BYTES a row, its
// odd rows' halves exchanged. The weighted values are split into three bf16 parts.
template <int BYTES, int NA>
__device__ __forceinline__ void la_add(f32x4_t (&S)[NA], const uint8_t* keys, const u32x4_t (&v)[2], float2 full, const float* add,
                                       int column_at, int lq) {
#pragma unroll
  for (int i = 0; i < NA; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) S[i][e] = fmaf(S[i][e], full.x, S[i][e] * full.y);
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    __builtin_amdgcn_sched_barrier(0);
    u32x4_t part[3];
#pragma unroll
    for (int z = 0; z < 4; ++z) {
      const int n = 32 * u + 16 * (z >> 1) + 4 * lq + 2 * (z & 1);  // token of the first of the two
      float x0, x1;
      unpack_bf16x2(v[u][z], x0, x1);
      x0 *= add[n];
      x1 *= add[n + 1];
#pragma unroll
      for (int y = 0; y < 3; ++y) {
        const uint32_t b0 = __float_as_uint(x0), b1 = __float_as_uint(x1);
        part[y][z] = __builtin_amdgcn_perm(b1, b0, 0x07060302u);  // the high halves
        x0 -= __uint_as_float(b0 & 0xffff0000u);
        x1 -= __uint_as_float(b1 & 0xffff0000u);
      }
    }
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      // The reads of few rows at a time: more of them in flight would push the loop's state out of the registers.
      if (i % 2 == 0) __builtin_amdgcn_sched_barrier(0);
      const u32x4_t k = la_column<BYTES>(keys + (column_at ^ (64 * (i >> 1) + 8 * (i & 1))) + 32 * BYTES * u);
#pragma unroll
      for (int y = 0; y < 3; ++y) S[i] = mfma16x16x32(k, part[y], S[i]);
    }
  }
}

// The segment and the head of workgroup b. Heads that share keys and values run on one XCD (b runs on XCD b % 8) and find them in
// its L2 (39 heads on 13 of 64, 2 x 2049 tokens: 25.0 -> 23.2 us). Ordinary heads are spread over the XCDs, each head's segments
// on few of them, so that its states are found there too.
struct LaUnit {
  int seg, h, shared;  // the head, and the one that it shares keys and values with others in
};
__device__ __forceinline__ LaUnit la_unit_of(const LaArgs& a, unsigned b) {
  const unsigned G = a.group, Hk = G == 1 ? a.H : a.H / G, i = b / 8, j = G == 1 ? i : i / G, u = 8 * j + b % 8, seg = u / Hk;
  const int shared = (int)(u - seg * Hk);
  return {(int)seg, (int)(shared * G + (i - j * G)), shared};
}
__host__ __device__ __forceinline__ unsigned la_units(const LaArgs& a, unsigned segs) {
  return (segs * (a.H / a.group) + 7) / 8 * 8 * a.group;
}

// A score of a later key is zero, but zero times a NaN or an infinity among its values is a NaN. So values that are not finite are
// looked for, once a chunk, and where there are any their terms are added one by one, of keys at or before the query alone, and
// zeros take their place for the product (la_weigh_infinite). A wave that has just added them to its columns of the state need
// look at one row of that alone: each is a sum over all of the column's values.
__device__ __forceinline__ bool la_any_infinite(float x) {
  return ballot64((__float_as_uint(x) & 0x7f800000u) == 0x7f800000u) != 0;
}
__device__ __forceinline__ bool la_any_infinite(const u32x4_t (&v)[2]) {
  uint32_t any = 0;
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int z = 0; z < 4; ++z) any |= (v[u][z] & 0x7f807f80u) + 0x00800080u;  // carries out of an exponent of ones
  return ballot64((any & 0x80008000u) != 0) != 0;
}
__device__ __forceinline__ bool la_any_infinite(const f32x4_t (&v)[4]) {
  uint32_t any = 0;
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) any |= (__float_as_uint(v[t][e]) & 0x7f800000u) + 0x00800000u;
  return ballot64((any & 0x80000000u) != 0) != 0;
}
__device__ __forceinline__ bool la_infinite(float x) { return !(fabsf(x) <= 3.402823466e38f); }

// x of that lane of the wave (__shfl would keep the lane's own number in a register all through the loop).
__device__ __forceinline__ uint32_t la_lane(uint32_t x, int lane) {
  return (uint32_t)__builtin_amdgcn_ds_bpermute(4 * lane, (int)x);
}

// o[t] += the terms of values that are not finite. value(n, c): token n's value of column c of the wave's 16, where the lane at
// 16 ((n / 4) % 4) + c holds it; score(t, n): that of token n for query 16 t + lr.
template <class Value, class Score>
__device__ __forceinline__ void la_weigh_infinite(f32x4_t (&o)[4], int lr, int lq, Value value, Score score) {
#pragma unroll 1
  for (int n = 0; n < LA_C; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float x = value(n, 4 * lq + e);
      if (!la_infinite(x)) continue;
#pragma unroll
      for (int t = 0; t < 4; ++t)
        if (n <= 16 * t + lr) o[t][e] += score(t, n) * x;
    }
}
// bf16: o[t] += scores times values.
__device__ __forceinline__ void la_weigh(f32x4_t (&o)[4], const u32x4_t (&v)[2], const uint8_t* scores, int lane) {
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int u = 0; u <= t / 2; ++u)
#pragma unroll
      for (int part = 0; part < 2 * LA_SCORES; part += LA_SCORES)
        o[t] = mfma16x16x32(v[u], *reinterpret_cast<const u32x4_t*>(scores + (la_unit(t, u) * 64 + lane) * 16 + part), o[t]);
}
__device__ __forceinline__ void la_weigh_infinite(f32x4_t (&o)[4], u32x4_t (&v)[2], const uint8_t* scores, int lane) {
  const int lr = lane & 15, lq = lane >> 4;
  la_weigh_infinite(
      o, lr, lq,
      [&](int n, int c) {
        const int z = 2 * ((n >> 4) & 1) + ((n >> 1) & 1);
        const u32x4_t x = n < 32 ? u32x4_t(v[0]) : u32x4_t(v[1]);
        const uint32_t word = la_lane(z == 0 ? x[0] : z == 1 ? x[1] : z == 2 ? x[2] : x[3], 16 * ((n >> 2) & 3) + c);
        return __uint_as_float(n & 1 ? word & 0xffff0000u : word << 16);
      },
      [&](int t, int n) {
        const int unit = t == 3 ? n >> 5 : t == 2 ? 2 + 3 * (n >> 5) : 4 - t, lane = 16 * ((n >> 2) & 3) + lr;
        const uint8_t* at = scores + (unit * 64 + lane) * 16 + 8 * ((n >> 4) & 1) + 2 * (n & 3);
        auto part = [](const uint8_t* x) { return bf16_to_f32(*reinterpret_cast<const uint16_t*>(x)); };
        return part(at) + part(at + LA_SCORES);
      });
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int z = 0; z < 4; ++z) {
      const uint32_t x = v[u][z];
      v[u][z] = ((x & 0x7f80u) == 0x7f80u ? 0u : x & 0xffffu) | ((x & 0x7f800000u) == 0x7f800000u ? 0u : x & 0xffff0000u);
    }
}
// The same in fp32.
__device__ __forceinline__ void la_weigh(f32x4_t (&o)[4], const f32x4_t (&v)[4], const uint8_t* scores, int lane) {
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int k = 0; k <= t; ++k) {
      const f32x4_t s = *reinterpret_cast<const f32x4_t*>(scores + ((2 * la_unit(t, k / 2) + k % 2) * 64 + lane) * 16);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[t] = mfma16x16x4(v[k][e], s[e], o[t]);
    }
}
__device__ __forceinline__ void la_weigh_infinite(f32x4_t (&o)[4], f32x4_t (&v)[4], const uint8_t* scores, int lane) {
  const int lr = lane & 15, lq = lane >> 4;
  la_weigh_infinite(
      o, lr, lq,
      [&](int n, int c) {
        uint32_t word = 0;  // by masks: an index that varies would put the values into memory
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) word |= n >> 4 == t && (n & 3) == e ? __float_as_uint(v[t][e]) : 0u;
        return __uint_as_float(la_lane(word, 16 * ((n >> 2) & 3) + c));
      },
      [&](int t, int n) {
        const int k = n >> 4, unit = t == 3 ? k >> 1 : t == 2 ? 2 + 3 * (k >> 1) : 4 - t, lane = 16 * ((n >> 2) & 3) + lr;
        return *reinterpret_cast<const float*>(scores + ((2 * unit + (k & 1)) * 64 + lane) * 16 + 4 * (n & 3));
      });
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) v[t][e] = la_infinite(v[t][e]) ? 0.0f : v[t][e];
}

// tab[n] = e^{g n} for n <= 64; put[n] = what token n of a whole chunk adds to the state with, gain e^{g (63 - n + lag)}, then
// zeros.
__device__ __forceinline__ void la_tables(float2* tab, float* put, double g, float gain, int lag, int tid) {
  if (tid <= LA_C) tab[tid] = la_decay2(g, tid);
  if (tid >= 128 && tid < 256) put[tid - 128] = tid - 128 < LA_C ? gain * la_decay2(g, LA_C - 1 - (tid - 128) + lag).x : 0.0f;
}

// Where the caller's state has the lane's element e of tile i, column col: [dk][dv], or [dv][dk] with turned; -1 outside of it.
template <bool BF16>
__device__ __forceinline__ int la_user(const LaArgs& a, int i, int e, int lq, int col) {
  const int row = la_row<BF16>(0, lq), more = la_row<BF16>(i, 0) + e;  // row + more
  const int at = a.turned ? col * a.dk + row + more : row * a.dv + col + more * a.dv;
  return row + more < a.dk && col < a.dv ? at : -1;
}

// The same of a state in a.mid that a call with dk and dv exchanged left, in tiles of NA rows: from the lane's own part, of row
// 16 w + lr and columns la_row(0, lq) .., by what i and e add.
template <bool BF16, int NA>
__device__ __forceinline__ int la_turned(int i, int e, int w, int lr, int lq) {
  const int row = 16 * w + lr;
  const int tile = BF16 ? 2 * (row >> 5) + ((row >> 2) & 1) : row >> 4, q = BF16 ? (row >> 3) & 3 : (row >> 2) & 3;
  const int own = (64 * tile + 16 * q) * 4 + (row & 3);
  return BF16 ? own + (lq >> 1) * (256 * NA) + 32 * (lq & 1) + (i >> 1) * (512 * NA) + 16 * (i & 1) + 4 * e
              : own + 16 * lq + i * (256 * NA) + 4 * e;
}

// One segment of one head; DV / 16 waves. Wave w has columns 16 w .. of the state and of the outputs for all 64 queries of a
// chunk (outputs as [column, query] tiles), and some of the scores' six [32 keys, 16 queries] units, which go through LDS. The
// state stays in accumulators, which, in two bf16 parts, are the operand that queries read (la_row). A column's tokens come out of the
// transposing LDS read in the order in which an accumulator holds the scores' keys, once for the outputs and for the state.
// Two barriers a chunk: tiles and scores are read behind one, scores and the next tiles written behind the other.
// 4 x 4096 tokens x 16 heads of 128 bf16 (MI355X; median, and least, of 27 passes) take 86 (75) us with OUT (302 MB, 3.5 TB/s; a large
// copy reaches 5.1), 41 (36) without (163 MB, 4.0 TB/s): bound by memory and vector instructions, which are busy 62 % of the time,
// the matrix units 33 % (60 and 35 without; counters at 65536 tokens). fp32: 267 and 119 us, matrix units busy 58 and 35 %.
template <bool BF16, int DK, int DV, bool REV, bool OUT>
__global__ __launch_bounds__(4 * DV, la_waves(BF16, DK, DV, OUT)) void la_kernel(LaArgs a) {
  constexpr int ES = BF16 ? 2 : 4, KB = DK * ES, VB = DV * ES, NA = DK / 16, W = DV / 16, THREADS = 4 * DV;
  __shared__ __attribute__((aligned(16))) uint8_t Ks[LA_C * KB];
  __shared__ __attribute__((aligned(16))) uint8_t Vs[LA_C * VB];
  // Queries go straight to LDS, to the other of two tiles; narrow ones through registers like keys and values, so that four
  // workgroups' LDS fit on a CU.
  constexpr bool COPY = !(BF16 && DK == 64 && DV == 64);
  __shared__ __attribute__((aligned(16))) uint8_t Qs[1 + COPY][OUT ? LA_C * KB : 16];
  __shared__ __attribute__((aligned(16))) uint8_t Ps[OUT ? 2 * LA_SCORES : 16];
  __shared__ float2 tab[LA_C + 1];  // e^{g n} to 48 bits
  __shared__ float put[2 * LA_C];   // what a token adds to the state with: of a chunk's 64, then zeros
  const int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, lq = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  if (OUT && blockIdx.x >= la_units(a, a.segs)) {
    la_gap(a, a.o, a.H * a.dv * (a.o_f32 ? 4 : ES), blockIdx.x - la_units(a, a.segs));
    return;
  }
  const LaUnit unit = la_unit_of(a, blockIdx.x);
  const int seg = unit.seg, h = unit.h;
  if (seg >= (OUT ? a.segs : a.segs - a.N)) return;
  const LaPlace p = la_place<OUT>(a, seg);
  if (!p.there) return;
  const int64_t first = a.plan == nullptr ? 0 : p.start;
  const int64_t sb = a.plan == nullptr ? p.seq : 0;
  auto start = [&](auto& stage, const LaTensor& t, int j0) {
    const int head = t.div == 1 ? h : unit.shared;
    const uint8_t* base = static_cast<const uint8_t*>(t.p) + ES * (sb * t.sb + first * t.st + (int64_t)head * t.sh);
    if (REV) stage.start(base + (int64_t)(p.len - 1) * t.st * ES, -t.st * ES, j0);
    else stage.start(base, t.st * ES, j0);
  };
  const int begin = p.s * a.L, end = min(p.len, begin + a.L);
  const bool last = p.s == p.nseg - 1, keep = !OUT || (last && a.s1 != nullptr);

  LaStage<BF16, KB, THREADS> kst, qst;
  LaStage<BF16, VB, THREADS> vst;
  start(kst, a.k, begin);
  start(vst, a.v, begin);
  if (OUT) start(qst, a.q, begin);
  auto fetch = [&](int rows) {
    const int tid = afresh((int)threadIdx.x);
    if (OUT && !COPY) qst.load(tid, rows, a.dk * ES);
    kst.load(tid, rows, a.dk * ES);
    vst.load(tid, rows, a.dv * ES);
  };
  auto copy = [&](int rows, uint8_t* queries) {
    if (OUT && COPY) qst.copy(afresh((int)threadIdx.x), queries, rows, a.dk * ES);
  };
  const double g = (double)a.g[h];
  // Rows la_row(i, lq) .. + 3, column 16 w + lr.
  f32x4_t S[NA];
  const float* before = a.mid + ((la_slot(a, p.seq) + p.s - 1) * a.H + h) * (DK * DV);
  const int64_t user = ((int64_t)p.seq * a.H + h) * a.dk * a.dv;
  if (OUT && p.s > 0 && a.mid_turned) {
#pragma unroll
    for (int i = 0; i < NA; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) S[i][e] = before[la_turned<BF16, DV / 16>(i, e, w, lr, lq)];
  } else if (OUT && p.s > 0) {
#pragma unroll
    for (int i = 0; i < NA; ++i) S[i] = *reinterpret_cast<const f32x4_t*>(before + ((w * NA + i) * 64 + lane) * 4);
  } else if (OUT && a.s0 != nullptr) {
#pragma unroll
    for (int i = 0; i < NA; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int at = la_user<BF16>(a, i, e, lq, 16 * w + lr);
        const float x = (a.s0 + user)[max(at, 0)];
        S[i][e] = at >= 0 ? x : 0.0f;
      }
  } else {
#pragma unroll
    for (int i = 0; i < NA; ++i) S[i] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  }
  // The first tiles are on their way while the decays are made (before the state, which is waited for first: 2048 tokens x 16
  // heads of 128 take 42.4 us, so 40.2).
  if (begin < end) {
    copy(min(LA_C, end - begin), Qs[0]);
    fetch(min(LA_C, end - begin));
  }
  la_tables(tab, put, g, a.gain, a.lag, tid);
  auto stage = [&]() {
    const int tid = afresh((int)threadIdx.x);
    kst.template store<BF16>(tid, Ks);
    vst.template store<false>(tid, Vs);
    if (OUT && !COPY) qst.template store<false>(tid, Qs[0]);
    if (OUT && COPY) wait_vmcnt0();  // the queries' copy
  };
  if (begin < end) stage();
  for (int j0 = begin, par = 0; j0 < end; j0 += LA_C, par ^= 1) {
    const int rows = min(LA_C, end - j0);
    const bool more = j0 + LA_C < end;
    __syncthreads();
    if (more) fetch(min(LA_C, end - j0 - LA_C));
    const uint8_t* const Q = Qs[COPY ? par : 0];
    const int lane = afresh(tid & 63), lr = lane & 15, lq = lane >> 4;
    using KeyTile = LaTile<BF16, KB>;
    using ValueTile = LaTile<BF16, VB>;
    // Row 16 t + lr, column 4 s + lq: row_at ^ 64 (s % 4), + 256 (s / 4), + 16 KB t.
    const int row_at = KeyTile::at(lr, lq);
    // bf16: rows 4 lq + lr / 4, features la_row(i, lr % 4) ..: column_at ^ (64 (i / 2) + 8 (i % 2)).
    const int column_at = KeyTile::at(4 * lq + (lr >> 2), lr & 3) + 8 * KeyTile::swapped(lr >> 2);
    const int value_at = ValueTile::at(4 * lq + (lr >> 2), 2 * w + ((lr & 3) >> 1)) + 8 * (lr & 1);
    f32x4_t o[4];  // [query tile]
    if constexpr (OUT) {
      // Scores of queries 16 t + lr with keys 32 u + {4 lq .., 16 + 4 lq ..}, weighted.
      for (int unit = w; unit < LA_UNITS; unit += W) {
        if constexpr (BF16) {
          la_scores<KB, true>(Ks, Q, Ps, unit, lr, lq, row_at, a.intra, tab);
        } else {
          const int t = la_unit_queries(unit), u = la_unit_keys(unit);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            f32x4_t P = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int s = 0; s < KB / 64; ++s) {
              const int at = (row_at ^ (64 * (s & 3))) + 256 * (s >> 2);
              const f32x4_t x = *reinterpret_cast<const f32x4_t*>(Ks + at + 16 * KB * (2 * u + k));
              const f32x4_t y = *reinterpret_cast<const f32x4_t*>(Q + at + 16 * KB * t);
#pragma unroll
              for (int e = 0; e < 4; ++e) P = mfma16x16x4(x[e], y[e], P);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int n = 16 * (t - 2 * u - k) + lr - 4 * lq - e;  // tokens between key and query
              P[e] = n >= 0 ? P[e] * (a.intra * tab[max(n, 0)].x) : 0.0f;
            }
            *reinterpret_cast<f32x4_t*>(Ps + ((2 * unit + k) * 64 + lane) * 16) = P;
          }
        }
      }
      // What the queries read from the state.
#pragma unroll
      for (int t = 0; t < 4; ++t) o[t] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int s = 0; s < KB / 64; ++s) {
        u32x4_t x, left;
        if constexpr (BF16) x = la_pack(S[2 * s], S[2 * s + 1]), left = la_left(S[2 * s], S[2 * s + 1], x);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const u32x4_t y = *reinterpret_cast<const u32x4_t*>(Q + (row_at ^ (64 * (s & 3))) + 256 * (s >> 2) + 16 * KB * t);
          if constexpr (BF16) {
            o[t] = mfma16x16x32(left, y, mfma16x16x32(x, y, o[t]));
          } else {
            const f32x4_t yf = __builtin_bit_cast(f32x4_t, y);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[t] = mfma16x16x4(S[s][e], yf[e], o[t]);
          }
        }
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) o[t] = o[t] * (a.inter * tab[16 * t + lr + 1 - a.lag].x);
      // Behind this chunk's reads of queries: a read of either tile waits for copies under way.
      if (more) copy(min(LA_C, end - j0 - LA_C), Qs[COPY ? par ^ 1 : 0]);
    }
    // The wave's columns of the values: bf16 as operands, tokens 32 u + {4 lq .., 16 + 4 lq ..}; fp32 tokens 16 t + 4 lq .. .
    u32x4_t v[2];
    f32x4_t vf[4];
    if constexpr (BF16) {
#pragma unroll
      for (int u = 0; u < 2; ++u) v[u] = la_column<VB>(Vs + value_at + 32 * VB * u);
    } else {
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          vf[t][e] = *reinterpret_cast<const float*>(Vs + ValueTile::at(16 * t + 4 * lq + e, 4 * w + (lr >> 2)) + 4 * (lr & 3));
    }
    if (more || keep) {
      const float2 full = tab[rows];
      const float* add = put + LA_C - rows;  // zero behind the last row
      if constexpr (BF16) {
        la_add<KB>(S, Ks, v, full, add, column_at, lq);
      } else {
#pragma unroll
        for (int i = 0; i < NA; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) S[i][e] = fmaf(S[i][e], full.x, S[i][e] * full.y);
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int n = 16 * t + 4 * lq + e;
            const float x = vf[t][e] * add[n];
#pragma unroll
            for (int i = 0; i < NA; ++i)
              S[i] = mfma16x16x4(*reinterpret_cast<const float*>(Ks + KeyTile::at(n, 4 * i + (lr >> 2)) + 4 * (lr & 3)), x, S[i]);
          }
      }
    }
    __syncthreads();
    if (more) stage();
    if constexpr (OUT) {
      const int lane = afresh((int)threadIdx.x) & 63, lr = lane & 15, lq = lane >> 4;
      const int c = 16 * w + 4 * lq;
      if constexpr (BF16) {
        if (__builtin_expect(more || keep ? la_any_infinite(S[0][0]) : la_any_infinite(v), 0)) la_weigh_infinite(o, v, Ps, lane);
        la_weigh(o, v, Ps, lane);
      } else {
        if (__builtin_expect(more || keep ? la_any_infinite(S[0][0]) : la_any_infinite(vf), 0))
          la_weigh_infinite(o, vf, Ps, lane);
        la_weigh(o, vf, Ps, lane);
      }
      const int64_t out = sb * a.ob + (first + (REV ? p.len - 1 - j0 - lr : j0 + lr)) * a.ot + (int64_t)h * a.oh + c;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        if (j0 + 16 * t + lr >= end || c >= a.dv) continue;
        const int64_t to = out + (int64_t)(REV ? -(16 * t) : 16 * t) * a.ot;
        if (BF16 && !a.o_f32)
          *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.o) + to) =
              make_uint2(pack_bf16x2(o[t][0], o[t][1]), pack_bf16x2(o[t][2], o[t][3]));
        else
          *reinterpret_cast<f32x4_t*>(static_cast<float*>(a.o) + to) = o[t];
      }
    }
  }
  if (!keep) return;
  const int own = afresh(tid & 63);
#pragma unroll
  for (int i = 0; i < NA; ++i) {
    if (!OUT) {
      *reinterpret_cast<f32x4_t*>(a.mid + ((la_slot(a, p.seq) + p.s) * a.H + h) * (DK * DV) + ((w * NA + i) * 64 + own) * 4) = S[i];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int at = la_user<BF16>(a, i, e, own >> 4, 16 * w + (own & 15));
        if (at >= 0) (a.s1 + user)[at] = S[i][e];
      }
    }
  }
}

// dk and dv of one segment of one head together, bf16, backwards in time with T = the gradient of the state [dk, dv]:
//   dv_j = scale sum_{i >= j} e^{g (i - j)} (k_j . q_i) dO_i + e^{g j'} T^T k_j     (j' tokens from the chunk's start, backwards)
//   dk_j = scale sum_{i >= j} e^{g (i - j)} (v_j . dO_i) q_i + e^{g j'} T v_j
// DV / 16 waves make dv and hold T as la_kernel's hold S; DK / 16 more make dk and read T, in two bf16 parts, from LDS, where the
// first ones leave it once a chunk. One pass over q, k, v and dO instead of two over three of them each, and T made once:
// 4 x 4096 tokens x 16 heads of 128 (MI355X; median, and least, of 27 passes) take 139 (121) us (419 MB, 3.0 TB/s; vector units busy
// 47 % of the time, matrix units 27), two passes of la_kernel 2 x 86 and another carry.
template <int DK, int DV>
__global__ __launch_bounds__(4 * (DK + DV), DK == DV ? 4 : 3) void la_back_kernel(LaBackArgs a) {
  constexpr int KB = DK * 2, VB = DV * 2, NA = DK / 16, WV = DV / 16, WK = DK / 16, THREADS = 4 * (DK + DV);
  __shared__ __attribute__((aligned(16))) uint8_t Qs[LA_C * KB], Ks[LA_C * KB], Vs[LA_C * VB], Ds[LA_C * VB];
  __shared__ __attribute__((aligned(16))) uint8_t Ts[2][DV * KB];
  __shared__ __attribute__((aligned(16))) uint8_t Ps[2][2 * LA_SCORES];
  __shared__ float2 tab[LA_C + 1];
  __shared__ float put[2 * LA_C];
  const int tid = threadIdx.x;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const bool first_waves = w < WV;
  const int wc = first_waves ? w : w - WV;  // columns 16 wc .. of dv or dk
  if (blockIdx.x >= la_units(a.s, a.s.segs)) {
    const int block = blockIdx.x - la_units(a.s, a.s.segs), es = a.s.o_f32 ? 4 : 2;
    if (a.dk_out != nullptr) la_gap(a.s, a.dk_out, a.s.H * a.s.dk * es, block);
    if (a.dv_out != nullptr) la_gap(a.s, a.dv_out, a.s.H * a.s.dv * es, block);
    return;
  }
  const LaUnit unit = la_unit_of(a.s, blockIdx.x);
  const int seg = unit.seg, h = unit.h;
  if (seg >= a.s.segs) return;
  const LaPlace p = la_place<true>(a.s, seg);
  if (!p.there) return;
  const int64_t first = a.s.plan == nullptr ? 0 : p.start;
  const int64_t sb = a.s.plan == nullptr ? p.seq : 0;
  const int begin = p.s * a.s.L, end = min(p.len, begin + a.s.L);
  const bool keep = p.s == p.nseg - 1 && a.s.s1 != nullptr;
  auto start = [&](auto& stage, const LaTensor& t) {
    const int head = t.div == 1 ? h : unit.shared;
    const uint8_t* base = static_cast<const uint8_t*>(t.p) + 2 * (sb * t.sb + first * t.st + (int64_t)head * t.sh);
    stage.start(base + (int64_t)(p.len - 1) * t.st * 2, -t.st * 2, begin);
  };
  using KeyTile = LaTile<true, KB>;
  using ValueTile = LaTile<true, VB>;
  LaStage<true, KB, THREADS> qst, kst;
  LaStage<true, VB, THREADS> vst, dst;
  start(qst, a.s.k);
  start(dst, a.s.v);
  start(kst, a.k);
  start(vst, a.v);
  auto fetch = [&](int rows) {
    const int tid = afresh((int)threadIdx.x);
    qst.load(tid, rows, a.s.dk * 2);
    kst.load(tid, rows, a.s.dk * 2);
    vst.load(tid, rows, a.s.dv * 2);
    dst.load(tid, rows, a.s.dv * 2);
  };
  auto stage = [&]() {
    const int tid = afresh((int)threadIdx.x);
    qst.template store<true>(tid, Qs);
    kst.template store<false>(tid, Ks);
    vst.template store<false>(tid, Vs);
    dst.template store<false>(tid, Ds);
  };
  const double g = (double)a.s.g[h];
  if (begin < end) fetch(min(LA_C, end - begin));

  f32x4_t T[NA];  // first waves: rows la_row(i, lq) .., column 16 w + lr
  const int64_t user = ((int64_t)p.seq * a.s.H + h) * a.s.dk * a.s.dv;
  {
    const int lane = tid & 63, lr = lane & 15, lq = lane >> 4;
    if (first_waves && p.s > 0) {
      const float* before = a.s.mid + ((la_slot(a.s, p.seq) + p.s - 1) * a.s.H + h) * (DK * DV);
#pragma unroll
      for (int i = 0; i < NA; ++i) T[i] = *reinterpret_cast<const f32x4_t*>(before + ((w * NA + i) * 64 + lane) * 4);
    } else if (first_waves && a.s.s0 != nullptr) {
#pragma unroll
      for (int i = 0; i < NA; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int at = la_user<true>(a.s, i, e, lq, 16 * w + lr);
          const float x = (a.s.s0 + user)[max(at, 0)];
          T[i][e] = at >= 0 ? x : 0.0f;
        }
    } else {
#pragma unroll
      for (int i = 0; i < NA; ++i) T[i] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    }
  }
  la_tables(tab, put, g, a.s.gain, 1, tid);
  // Ts is [dv][dk], two parts; rows 8 apart, which its transposing reads take together, are mixed as those 4 apart of other tiles are.
  auto state = [&](int row, int col) { return row * KB + ((col ^ KeyTile::key((row & 3) | ((row >> 1) & 4))) << 4); };
  auto publish = [&](int lr, int lq) {
#pragma unroll
    for (int u = 0; u < NA / 2; ++u) {
      const u32x4_t x = la_pack(T[2 * u], T[2 * u + 1]);
      *reinterpret_cast<u32x4_t*>(Ts[0] + state(16 * wc + lr, 4 * u + lq)) = x;
      *reinterpret_cast<u32x4_t*>(Ts[1] + state(16 * wc + lr, 4 * u + lq)) = la_left(T[2 * u], T[2 * u + 1], x);
    }
  };
  if (begin < end) {
    stage();
    if (first_waves) publish(tid & 15, (tid >> 4) & 3);
  }
  for (int j0 = begin; j0 < end; j0 += LA_C) {
    const int rows = min(LA_C, end - j0);
    const bool more = j0 + LA_C < end;
    __syncthreads();
    if (more) fetch(min(LA_C, end - j0 - LA_C));
    const int lane = afresh(tid & 63), lr = lane & 15, lq = lane >> 4;
    f32x4_t o[4];
    u32x4_t v[2];
#pragma unroll
    for (int t = 0; t < 4; ++t) o[t] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    if (first_waves) {
      const int row_at = KeyTile::at(lr, lq);
      const int column_at = KeyTile::at(4 * lq + (lr >> 2), lr & 3) + 8 * KeyTile::swapped(lr >> 2);
      const int value_at = ValueTile::at(4 * lq + (lr >> 2), 2 * wc + ((lr & 3) >> 1)) + 8 * (lr & 1);
      for (int unit = wc; unit < LA_UNITS; unit += WV)
        la_scores<KB, true>(Qs, Ks, Ps[0], unit, lr, lq, row_at, a.s.intra, tab);
#pragma unroll
      for (int s = 0; s < KB / 64; ++s) {
        // T as the wave itself published it: reads cost less than making it again.
        const u32x4_t x = *reinterpret_cast<const u32x4_t*>(Ts[0] + state(16 * wc + lr, 4 * s + lq));
        const u32x4_t left = *reinterpret_cast<const u32x4_t*>(Ts[1] + state(16 * wc + lr, 4 * s + lq));
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const u32x4_t y = *reinterpret_cast<const u32x4_t*>(Ks + (row_at ^ (64 * s)) + 16 * KB * t);
          o[t] = mfma16x16x32(left, y, mfma16x16x32(x, y, o[t]));
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) v[u] = la_column<VB>(Ds + value_at + 32 * VB * u);
      if (more || keep) la_add<KB>(T, Qs, v, tab[rows], put + LA_C - rows, column_at, lq);
    } else {
      const int row_at = ValueTile::at(lr, lq);
      const int value_at =
          KeyTile::at(4 * lq + (lr >> 2), 2 * wc + ((lr & 3) >> 1)) + 8 * ((lr & 1) ^ KeyTile::swapped(lr >> 2));
      // Row 16 wc + lr of T, columns 32 s + 8 lq .. + 3 and the 4 behind them.
      int state_at[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) state_at[i] = state(8 * lq + 4 * i + (lr >> 2), 2 * wc + ((lr & 3) >> 1)) + 8 * (lr & 1);
      for (int unit = wc; unit < LA_UNITS; unit += WK)
        la_scores<VB, false>(Ds, Vs, Ps[1], unit, lr, lq, row_at, a.s.intra, tab);
#pragma unroll
      for (int s = 0; s < VB / 64; ++s) {
        u32x4_t x[2];
#pragma unroll
        for (int part = 0; part < 2; ++part) {
          const uint2 a = la_read_tr(Ts[part] + state_at[0] + 32 * KB * s), b = la_read_tr(Ts[part] + state_at[1] + 32 * KB * s);
          x[part] = u32x4_t{a.x, a.y, b.x, b.y};
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const u32x4_t y = *reinterpret_cast<const u32x4_t*>(Vs + (row_at ^ (64 * s)) + 16 * VB * t);
          o[t] = mfma16x16x32(x[1], y, mfma16x16x32(x[0], y, o[t]));
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) v[u] = la_column<KB>(Qs + value_at + 32 * KB * u);
    }
    __syncthreads();
    if (more) {
      stage();
      if (first_waves) publish(lr, lq);
    }
    const int me = afresh((int)threadIdx.x) & 63, mr = me & 15, mq = me >> 4;
    const uint8_t* const P = Ps[first_waves ? 0 : 1];
#pragma unroll
    for (int t = 0; t < 4; ++t) o[t] = o[t] * tab[16 * t + mr].x;
    if (__builtin_expect(first_waves && (more || keep) ? la_any_infinite(T[0][0]) : la_any_infinite(v), 0))
      la_weigh_infinite(o, v, P, me);
    la_weigh(o, v, P, me);
    const int c = 16 * wc + 4 * mq, d = first_waves ? a.s.dv : a.s.dk;
    void* const to = first_waves ? a.dv_out : a.dk_out;
    const int64_t ot = (int64_t)a.s.H * d, out = sb * a.s.S * ot + (first + p.len - 1 - j0 - mr) * ot + (int64_t)h * d + c;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      if (j0 + 16 * t + mr >= end || c >= d || to == nullptr) continue;
      if (a.s.o_f32)
        *reinterpret_cast<f32x4_t*>(static_cast<float*>(to) + out - 16 * t * ot) = o[t];
      else
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(to) + out - 16 * t * ot) =
            make_uint2(pack_bf16x2(o[t][0], o[t][1]), pack_bf16x2(o[t][2], o[t][3]));
    }
  }
  if (!keep || !first_waves) return;
  const int own = afresh(tid & 63);
#pragma unroll
  for (int i = 0; i < NA; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int at = la_user<true>(a.s, i, e, own >> 4, 16 * w + (own & 15));
      if (at >= 0) (a.s.s1 + user)[at] = T[i][e];
    }
}

// mid[s] = e^{g L} (the state before segment s) + mid[s]: the state behind every segment but a sequence's last. A thread has 4
// elements of one state, and the reads of the next LA_AHEAD segments are on their way while those of the last are added (31
// segments of 16 heads of 128 without 14.2 us, with 11.1; the median of 27 passes of 65536 tokens 12.7, 65 MB at 5.1 TB/s).
constexpr int LA_AHEAD = 8;
template <bool BF16, int DK, int DV>
__global__ __launch_bounds__(256) void la_carry_kernel(LaArgs a) {
  constexpr int NA = DK / 16;
  const int seq = (int)(blockIdx.x / a.H), h = (int)(blockIdx.x % a.H);
  const int idx = (int)(blockIdx.y * 256 + threadIdx.x);
  const int n = (a.plan == nullptr ? a.nseg : a.plan[seq + 1] - a.plan[seq]) - 1;
  if (n <= 0) return;
  const int64_t slot = la_slot(a, seq);
  const float2 whole = la_decay2((double)a.g[h], a.L);
  f32x4_t S = {0.0f, 0.0f, 0.0f, 0.0f};
  if (a.s0 != nullptr) {
    const int lane = idx & 63, i = (idx >> 6) % NA, dv = 16 * ((idx >> 6) / NA) + (lane & 15);
    const int64_t base = ((int64_t)seq * a.H + h) * a.dk * a.dv;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int dk = la_row<BF16>(i, lane >> 4) + e;
      if (dk < a.dk && dv < a.dv) S[e] = a.s0[base + (a.turned ? dv * a.dk + dk : dk * a.dv + dv)];
    }
  }
  f32x4_t* p = reinterpret_cast<f32x4_t*>(a.mid + (slot * a.H + h) * (DK * DV) + 4 * idx);
  const int64_t step = (int64_t)a.H * DK * DV / 4;
  f32x4_t x[2][LA_AHEAD];
  auto read = [&](f32x4_t (&to)[LA_AHEAD], int s) {
#pragma unroll
    for (int u = 0; u < LA_AHEAD; ++u)
      if (s + u < n) to[u] = p[(s + u) * step];
  };
  auto write = [&](f32x4_t (&from)[LA_AHEAD], int s) {
#pragma unroll
    for (int u = 0; u < LA_AHEAD; ++u) {
      if (s + u >= n) break;
#pragma unroll
      for (int e = 0; e < 4; ++e) S[e] = fmaf(S[e], whole.x, fmaf(S[e], whole.y, from[u][e]));
      p[(s + u) * step] = S;
    }
  };
  read(x[0], 0);
  for (int s = 0; s < n; s += 2 * LA_AHEAD) {
    read(x[1], s + LA_AHEAD);
    write(x[0], s);
    read(x[0], s + 2 * LA_AHEAD);
    write(x[1], s + LA_AHEAD);
  }
}

// out[t][hk][c] = sum over the G heads that share hk of x[t][hk G + i][c], fp32 in, one rounding; of two such in one launch.
template <bool BF16>
__global__ __launch_bounds__(256) void la_group_kernel(LaGroup a, LaGroup b, int64_t rows, int G) {
  const LaGroup g = blockIdx.y == 0 ? a : b;
  const int d4 = g.d / 4;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * d4; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / d4;
    const int c = (int)(i - row * d4);
    f32x4_t s = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int j = 0; j < G; ++j) s += *reinterpret_cast<const f32x4_t*>(g.x + ((row * G + j) * d4 + c) * 4);
    if (BF16)
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(g.out) + 4 * i) =
          make_uint2(pack_bf16x2(s[0], s[1]), pack_bf16x2(s[2], s[3]));
    else
      *reinterpret_cast<f32x4_t*>(static_cast<float*>(g.out) + 4 * i) = s;
  }
}

// One token: S = e^g S + k v^T in place, o = scale S^T q. Workgroup: 32 columns of one state, thread: 4 columns of every 32nd
// row; HBM-bound, 8 bytes per element of the states: 256 sequences x 16 heads of 128 x 128, a pool of 320, take 116 us (median; 541
// MB, 4.7 TB/s).
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
  bool mine = slot >= 0 && slot < a.pool;
  // Not one that an earlier sequence has: both would write it. 1024 slots are looked at at once: 4096 sequences x 16 heads of 128
  // take 1903 us, 1910 without slots (256 at a time 1937), 4096 x 2 of 64 49 and 42 (55), 16384 x 2 of 64 348 and 193 (473): all
  // workgroups' looks grow with the square of the sequences, and beyond some thousands of few and narrow heads they show.
  if (mine && a.slots != nullptr) {
    bool before = false;
    const int32_t *at = a.slots + tid, *const end = a.slots + b;
    for (; at + 3 * 256 < end; at += 4 * 256) {
#pragma unroll
      for (int i = 0; i < 4; ++i) before |= at[256 * i] == (int32_t)slot;
    }
    for (; at < end; at += 256) before |= *at == (int32_t)slot;
    mine = !__syncthreads_or(before);
  }
  if (mine) {
    // In two floats: one is off by up to 2^-25 of the state in the same direction at every token, which adds up (after 20000 tokens of
    // g = -1e-5 3e-4, and below -3e-8 nothing would be forgotten at all).
    const float2 lam = la_decay2((double)a.g[h], 1);
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
        s[e] = fmaf(s[e], lam.x, fmaf(s[e], lam.y, k * v[e]));
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

unsigned la_blocks(const LaArgs& a) { return la_units(a, a.segs) + (a.plan != nullptr ? (unsigned)(a.S + 63) / 64 : 0); }

// What every segment adds to the state, and the states between them, into a.mid.
template <bool BF16, int DK, int DV, bool REV>
hipError_t la_states(const LaArgs& a, hipStream_t st) {
  const int64_t inner = a.segs - a.N;  // segments with another behind them, at most
  if (inner == 0) return hipSuccess;
  hipLaunchKernelGGL((la_kernel<BF16, DK, DV, REV, false>), dim3(la_units(a, (unsigned)inner)), dim3(4 * DV), 0, st, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((la_carry_kernel<BF16, DK, DV>), dim3((unsigned)(a.N * a.H), DK * DV / 1024), dim3(256), 0, st, a);
  return hipGetLastError();
}

template <bool BF16, int DK, int DV, bool REV>
hipError_t la_run(const LaArgs& a, bool states, hipStream_t st) {
  if (states) {
    const hipError_t e = la_states<BF16, DK, DV, REV>(a, st);
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL((la_kernel<BF16, DK, DV, REV, true>), dim3(la_blocks(a)), dim3(4 * DV), 0, st, a);
  return hipGetLastError();
}

template <int DK, int DV>
hipError_t la_run_back(const LaBackArgs& a, hipStream_t st) {
  const hipError_t e = la_states<true, DK, DV, true>(a.s, st);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((la_back_kernel<DK, DV>), dim3(la_blocks(a.s)), dim3(4 * (DK + DV)), 0, st, a);
  return hipGetLastError();
}

// Calls f<DK, DV>(): the widths up to 64 or 128.
template <class F>
hipError_t la_widths(int dk, int dv, F f) {
  if (dk <= 64) return dv <= 64 ? f.template operator()<64, 64>() : f.template operator()<64, 128>();
  return dv <= 64 ? f.template operator()<128, 64>() : f.template operator()<128, 128>();
}

struct LaForwards {
  const LaArgs& a;
  bool states, bf16;
  hipStream_t st;
  template <int DK, int DV>
  hipError_t operator()() const {
    return bf16 ? la_run<true, DK, DV, false>(a, states, st) : la_run<false, DK, DV, false>(a, states, st);
  }
};
struct LaBackwards {
  const LaArgs& a;
  hipStream_t st;
  template <int DK, int DV>
  hipError_t operator()() const {
    return la_run<false, DK, DV, true>(a, true, st);
  }
};
struct LaBackBoth {
  const LaBackArgs& a;
  hipStream_t st;
  template <int DK, int DV>
  hipError_t operator()() const {
    return la_run_back<DK, DV>(a, st);
  }
};

}  // namespace

// Workgroups of la_kernel, or (back) of la_back_kernel, that a CU holds, by their LDS and registers.
static int la_per_cu(bool bf16, int dk, int dv, bool back) {
  const bool narrow = dk <= 64 && dv <= 64;
  return back ? (narrow ? 2 : 1) : bf16 ? (narrow ? 4 : 2) : narrow ? 2 : 1;
}

// As long segments as still give every CU the workgroups that it holds: more segments cost more states to write and read (64 KB
// at widths of 128, as much as 64 tokens' queries to outputs), fewer leave CUs idle. 16 heads with half, all, twice and four times
// as many as a CU holds: 4 x 4096 tokens of 128 bf16 forward and back 462, 359, 390, 458 us, 65536 tokens forward 473, 425, 444, 473,
// of 64 195, 220, 238, 263 (289 with a quarter); 16384 tokens fp32 forward of 128 694, 367, 368, 384, of 64 161, 133, 141.
int la_segment_tokens(int64_t N, int64_t S, bool packed, int H, bool bf16, int dk, int dv, bool back) {
  const int per_cu = la_per_cu(bf16, dk, dv, back);
  const int64_t want = std::max<int64_t>(1, (int64_t)per_cu * device_cus() / H);
  const int64_t chunks = std::max<int64_t>(1, (S + LA_C - 1) / LA_C);
  // Two chunks of bf16 are quicker in one launch than in three, of fp32, which take longer, not. 128 tokens x 16 heads of 128
  // forward in one and in two segments: bf16 15.2 and 17.3 us, fp32 34.6 and 31.5 (and back 107 and 84); of 64 10.3 and 12.8, 17.5 and
  // 17.6 (59 and 53). Three chunks of bf16 in one and in three: 19.8 and 17.7, of 64 13.4 and 12.9.
  if (!packed && bf16 && chunks <= 2) return 2 * LA_C;
  // Packed: sequences end inside of segments, half a one each, so these are made longer, up to a third; twice as long where the
  // sequences alone fill the CUs and few of them have a second segment. 16 heads of 128 forward with n = want, 3/4, 1/2 of it and by
  // the rule, the mean of eight drawn sets: 8191 tokens in 8 sequences 88, 83, 90, 79 us, in 23 84, 79, 89, 79, in 100 97, 96, 88, 88;
  // 32768 in 3 247, 270, 293, 235, in 12 264, 265, 303, 254, in 120 261, 254, 234, 234. Of 64: 8191 in 23 44, 41, 42, 42 (fp32 98,
  // 95, 114, 95), 32768 in 12 111, 105, 114, 102, in 120 116, 120, 133, 121.
  const int64_t n = !packed         ? std::max<int64_t>(1, want / std::max<int64_t>(1, N))
                    : N >= 2 * want ? std::max<int64_t>(1, want / 2)
                                    : std::max({want - N / 2, want * 3 / 4, (int64_t)1});
  // A segment of one chunk costs twice its bytes in states, which pays while half of the workgroups' places are empty (of
  // la_back_kernel's to the last one): 1024 tokens x 16 heads of 128 forward with one and two chunks a segment 26.2 and 27.5 us,
  // 2048 tokens 38.3 and 33.2, of 64 4096 tokens 30.3 and 25.9.
  const bool two = !packed && bf16 && !back && 2 * chunks > n;
  return (int)std::max<int64_t>(two ? 2 : 1, (chunks + n - 1) / n) * LA_C;
}

int64_t la_padded_state(int dk, int dv) { return (int64_t)(dk <= 64 ? 64 : 128) * (dv <= 64 ? 64 : 128); }

hipError_t launch_la_plan(const int32_t* cu, int32_t* plan, int N, int S, int L, hipStream_t st) {
  hipLaunchKernelGGL(la_plan_kernel, dim3(1), dim3(1024), 0, st, cu, plan, N, S, L);
  return hipGetLastError();
}

hipError_t launch_la(const LaArgs& a, bool states, bool bf16, hipStream_t st) {
  return la_widths(a.dk, a.dv, LaForwards{a, states, bf16, st});
}

hipError_t launch_la_backwards_f32(const LaArgs& a, hipStream_t st) {
  return la_widths(a.dk, a.dv, LaBackwards{a, st});
}

hipError_t launch_la_back_bf16(const LaBackArgs& a, hipStream_t st) {
  return la_widths(a.s.dk, a.s.dv, LaBackBoth{a, st});
}

hipError_t launch_la_group(const LaGroup& a, const LaGroup& b, int64_t rows, int G, bool bf16, hipStream_t st) {
  const LaGroup first = a.out != nullptr ? a : b;
  const int both = a.out != nullptr && b.out != nullptr;
  const int64_t n4 = rows * ((both ? std::max(a.d, b.d) : first.d) / 4);
  if (first.out == nullptr || n4 == 0) return hipSuccess;
  const dim3 grid((unsigned)std::min<int64_t>((n4 + 255) / 256, 16 * (int64_t)device_cus()), 1 + both);
  if (bf16) hipLaunchKernelGGL(la_group_kernel<true>, grid, dim3(256), 0, st, first, b, rows, G);
  else hipLaunchKernelGGL(la_group_kernel<false>, grid, dim3(256), 0, st, first, b, rows, G);
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
