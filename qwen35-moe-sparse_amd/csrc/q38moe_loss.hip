// Softmax cross entropy of a linear head, without its logits, and its gradient.
//
//   z = x W^T,  lse[t] = log sum_v exp z[t,v],  loss[t] = lse[t] - z[t, target[t]]
//   s[t,v] = exp(z[t,v] - lse[t]) - [v = target[t]],  dx = g (s W),  dW = g (s^T x)
//
// The forward pass multiplies tiles of the vocabulary by tiles of tokens and keeps of each only its rows' maximum and
// sum of exponentials (fp32) and the target's logit. The backward pass takes the vocabulary in pieces whose s [T, piece]
// fits a bounded workspace: it multiplies again (the logits were not kept), turns the fp32 accumulators into s, and
// multiplies s by W and by x. s is rounded to the operands' type for the matrix units (bf16: by up to 2^-8 of each
// value), before the loss's scalar gradient g, which the outputs' epilogues apply: the target's -1 + p, most of s's norm,
// then is -1 where p is below half a step, 2^-9, and loses only that p (1e-4 of the gradient at a vocabulary of 4000),
// where g (-1 + p) would carry the rounding of g, the same one, into every row. A gradient per row has to go into s, since
// dW sums over rows. What the rows' gradients share is taken out of them first: u, the largest without its power of two, so that
// one that all rows have rounds as the scalar does (1777 x 256 x 4096 against float64, g = 0.5637 in every row: dx and dW are
// off by 0.0017 of their norm; with g whole in s 0.0026, of which 0.0019 lie in the result's own direction). Where g / u is
// no power of two the target's entry rounds too, once as every other (random g: 0.0022). In fp32 g stays whole.
//
// Rows whose target is the ignored one leave the problem first: a stable partition lists the others, their x is copied
// next to each other, and the products run over those rows only, so neither the work nor a NaN in a masked row counts.
//
// One kernel does the four products. C[m, n] = sum_k A[m, k] B[n, k] on 256 x 256 tiles (128 x 128 or 64 x 64 where those are
// few), four waves, each a quarter of the tile in 32x32 blocks: at one wave per SIMD with 128 x 128 elements each operand byte
// read from LDS is used 128 times, which keeps LDS reads at half of the matrix units' time. An operand is either
// K-contiguous (KC: rows of 128 bytes per K step) or K-strided (KS: K rows of the tile's columns, fragments by the
// transposing LDS read in bf16), so s, x and W are used as they lie:
//     z^T : A = W (KC), B = x (KC);   dx^T : A = W (KS), B = s (KC);   dW^T : A = x (KS), B = s (KS).
// A K step is 128 bytes of K. Two steps lie in LDS (four or eight with 64 x 64 tiles, whose products wait for memory), copied
// there by buffer loads that write LDS directly; reads out of range give zeros, which are the tails of every dimension. The
// tokens (or vocabulary rows) are the lanes of the accumulators and the reduced or stored dimension their registers, so the
// softmax's maxima and sums are in-lane but for one exchange.
//
// What bounds it. The matrix units need 2051 clocks for a step of a 256 x 256 tile. With all CUs at work on random bf16
// data the chip lowers its clock to 1.7 - 1.9 GHz: MFMAs alone take 1.09 us a step, with their LDS reads 1.23, with the
// copies to LDS out of the L2 1.33 (all zeros: 0.94, 0.96, 1.04), and with a stream of its own per CU 1.94; this kernel,
// whose tiles share the streams eight by four, takes 1.7, in dx, whose s comes from memory, 2.1 and more. Smallest and
// median time of nine steps in a row: 16384 x 1024 x 10112 z 311 and 326 us (1090 and 1041 TFLOP/s), s 2 x 169 and 180, dx
// 2 x 163 and 194, dW 2 x 168 and 182; 4099 x 2048 x 50021 z 703 and 732 (1195 and 1147), s 2 x 381 and 397, dx 2 x 425 and
// 450, dW 2 x 403 and 423. Few tokens are bound by the latency of W's way into LDS: 61 x 1024 x 10112 z 10 us for 20.7 MB.
#include "q38moe_common.h"
#include "q38moe_kernels.h"

namespace q38 {
namespace {

enum { KC = 0, KS = 1 };
enum { EPI_LSE = 0, EPI_S = 1, EPI_OUT = 2 };

constexpr float LOG2E = 1.4426950408889634f;

typedef short ls_i16x4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __builtin_amdgcn_readfirstlane(v); }

// 16 bytes per lane from p + voff + soff to LDS at lds + 16 lane, zeros where voff + soff reaches `bytes` (raw buffer, no
// format).
__device__ __forceinline__ void ls_dma(const uint8_t* p, int64_t bytes, uint32_t voff, uint32_t soff, uint32_t lds) {
  const uint64_t a = (uint64_t)(uintptr_t)p;
  const uint32_t n = bytes <= 0 ? 0u : (bytes >= 0xffffffffll ? 0xffffffffu : (uint32_t)bytes);
  const u32x4_t r = {uniform((uint32_t)a), uniform((uint32_t)(a >> 32) & 0xffffu), uniform(n), 0x00020000u};
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(lds), "v"(voff), "s"(r), "s"(soff) : "memory", "m0");
}
// 16 bytes to p + off (p uniform), through the XCD's L2 (scope sc1): what a kernel leaves there has to be written back
// before the next one starts. For whole lines: s of 1024 x 1024 x 10112 36 -> 34 us, of 1024 x 1024 x 5056 21.3 -> 19.6, dW
// 47 -> 44.8; fp32, whose lanes store parts of lines, 43.6 -> 47. Past it (non-temporal) s is not found by its readers
// either (dx 32.7 -> 41 us).
__device__ __forceinline__ void ls_store_through(void* p, uint32_t off, u32x4_t v) {
  const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(p, (short)0, -1, 0x00020000);
  __builtin_amdgcn_raw_buffer_store_b128(v, r, (int)off, 0, 16);
}
__device__ __forceinline__ uint32_t ls_lds_addr(const void* p) {
  return uniform((uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p);
}
// This wave's LDS operations are done, and so are the others'.
__device__ __forceinline__ void ls_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

__device__ __forceinline__ uint2 ls_read_tr(const uint8_t* p) {
  const ls_i16x4_t v = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (__attribute__((address_space(3))) ls_i16x4_t*)(uintptr_t)((const __attribute__((address_space(3))) uint8_t*)p));
  return __builtin_bit_cast(uint2, v);
}

// One tile operand: R rows (KC) or columns (KS) of it, F32 elements or bf16.
template <bool F32, int R, int L>
struct Operand {
  static constexpr int ESZ = F32 ? 4 : 2;
  static constexpr int BK = 128 / ESZ;        // K elements of a step
  static constexpr int NDMA = R / 32;         // copies per wave and step
  static constexpr int PITCH = L == KC ? 128 : R * ESZ;
  static constexpr int LPR = PITCH / 16;      // lanes per LDS row of a copy
  static constexpr int NOFF = L == KC ? 4 : R / 64;  // lane offsets of a wave's fragments

  // Offset of copy j's 16 bytes of this lane from the operand's base: rows are ld bytes apart. Chunk c of row r lies at
  // c ^ swz(r): the 16 lanes that read together then cover the 64 banks.
  static __device__ __forceinline__ uint32_t voff(int j, int wave, int lane, uint32_t ld) {
    const int row = wave * (L == KC ? R / 4 : BK / 4) + j * (64 / LPR) + lane / LPR;
    const int sw = L == KC ? (row >> 1) & 7 : (F32 ? 8 * ((row >> 2) & 1) : ks_swz(row));
    return (uint32_t)row * ld + 16u * (uint32_t)((lane % LPR) ^ sw);
  }

  // KS, bf16: the four K rows that a half-wave's transposing read takes 64 bytes of lie in different banks.
  static __device__ __forceinline__ int ks_swz(int row) { return R == 64 ? 4 * ((row >> 1) & 1) : 4 * (row & 3); }

  // This lane's LDS offset of fragments: of K substep i (KC; block b adds 32 rows) or of block i (KS; substep u adds
  // rows).
  static __device__ __forceinline__ int foff(int i, int half, int lane) {
    const int r0 = half * (R / 2);
    if constexpr (L == KC) {
      const int row = r0 + (lane & 31);
      return row * 128 + 16 * ((2 * i + (lane >> 5)) ^ ((row >> 1) & 7));
    } else if constexpr (F32) {
      const int col = r0 + 32 * i + (lane & 31);
      return 4 * (lane >> 5) * PITCH + 16 * ((col >> 2) ^ (8 * (lane >> 5))) + 4 * (col & 3);
    } else {
      const int g = lane >> 4, gi = lane & 15;
      const int row = 8 * (g >> 1) + (gi >> 2), col = r0 + 32 * i + 16 * (g & 1) + 4 * (gi & 3);
      return row * PITCH + 16 * ((col >> 3) ^ ks_swz(row)) + 2 * (col & 7);
    }
  }

  // Fragment of block b, substep u (a quarter of the step's K): 16 bytes of K per lane.
  static __device__ __forceinline__ u32x4_t frag(const uint8_t* lds, const int (&off)[NOFF], int b, int u) {
    if constexpr (L == KC) {
      return ld16(lds + off[u] + b * 32 * 128);
    } else if constexpr (F32) {
      const uint8_t* p = lds + off[b] + u * 8 * PITCH;
      u32x4_t v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = *reinterpret_cast<const uint32_t*>(p + e * PITCH);
      return v;
    } else {
      const uint8_t* p = lds + off[b] + u * 16 * PITCH;
      const uint2 a = ls_read_tr(p), c = ls_read_tr(p + 4 * PITCH);
      return (u32x4_t){a.x, a.y, c.x, c.y};
    }
  }
};

// acc += A B: inline asm with the accumulator in its own AGPRs, as the four-wave gate/up kernel does it and for its
// reasons; two wait states cover a VALU write of an operand right before it.
template <bool F32>
__device__ __forceinline__ void ls_mfma(f32x16_t& acc, u32x4_t a, u32x4_t b) {
  if constexpr (F32) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      asm volatile("s_nop 1\n\tv_mfma_f32_32x32x2_f32 %0, %1, %2, %0" : "+a"(acc) : "v"(a[e]), "v"(b[e]));
  } else {
    asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+a"(acc) : "v"(a), "v"(b));
  }
}
// acc = 0 by the matrix unit, which has nothing else to do between two tiles (16 VALU writes would cost the epilogue their
// time).
__device__ __forceinline__ void ls_zero(f32x16_t& acc) {
  const u32x4_t z = {0u, 0u, 0u, 0u};
  asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %1, 0" : "+a"(acc) : "v"(z));
}
// Wait states between the last MFMA and VALU reads of its result (16 passes).
__device__ __forceinline__ void ls_drain() { asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7" ::: "memory"); }

// A block's accumulators in VGPRs, at this place of the instruction order (left to itself the compiler moves all of a
// tile's out at once, and spills).
__device__ __forceinline__ f32x16_t ls_take(const f32x16_t& a) {
  f32x16_t v = a;
  asm volatile("" : "+v"(v));
  return v;
}

// v = with where a value's row 8 (q / 4) + q % 4 of the block is `left` or beyond. (The comparisons stay at their place: as
// invariants of the blocks' loop their masks would not fit the SGPRs.)
__device__ __forceinline__ void ls_mask(f32x16_t& v, int left, float with) {
  asm volatile("" : "+v"(left));
#pragma unroll
  for (int q = 0; q < 16; ++q)
    if (8 * (q >> 2) + (q & 3) >= left) v[q] = with;
}

// {m, s} of two sets of values as one.
__device__ __forceinline__ void lse_join(float& m, float& s, float m2, float s2) {
  const float top = fmaxf(m, m2);
  const float ref = top == -__builtin_inff() ? 0.0f : top;
  s = s * __builtin_amdgcn_exp2f((m - ref) * LOG2E) + s2 * __builtin_amdgcn_exp2f((m2 - ref) * LOG2E);
  m = top;
}

struct LsParams {
  const uint8_t* A;      // KC [M, K], KS [K, M]
  const uint8_t* B;      // KC [N, K], KS [K, N]
  const uint8_t* alt;    // the operand that holds tokens where every row counts (the uncopied x)
  int64_t lda, ldb;      // bytes between rows
  int64_t M, N, K;       // extents (the tokens' one: an upper bound)
  int64_t m_rows;        // rows (KC) or columns of A that exist, <= M: the others of M multiply zeros
  const int32_t* count;  // tokens that count (device)
  int64_t T;             // tokens of the call
  const int32_t* rows;   // original row of a counted token
  // EPI_LSE, EPI_S
  int64_t v0;            // first vocabulary row of the piece
  float2* part;          // {max, sum} [2 ceil(M / BM), T]
  const int32_t* tgt;    // target per counted token
  const void* raw;       // EPI_LSE without a list of rows: the targets as they are (count NULL: all T)
  bool raw64;
  float* zt;             // the target's logit
  uint32_t* done;        // EPI_LSE: cleared for ls_finish_kernel
  const float* lse;      // EPI_S: per counted token
  const float* g_row;    // its gradient, or NULL
  const float* g_unit;   // bf16: what is taken out of it before s is rounded, or NULL
  // EPI_S, EPI_OUT
  void* out;             // s, or the gradient
  int64_t ldo;           // elements between rows of out
  const float* g_scale;  // the loss's gradient, or the unit of the rows' (NULL: 1)
  const float* r_scale;  // the reduction's factor (NULL: 1)
  float* acc;            // tiles' sums over the pieces so far (fp32, in the accumulators' own order), or NULL
  bool first, last;      // piece: acc holds nothing yet; out is written (else acc)
  float* split;          // partial sums of split tiles, a tile after another
  uint32_t slots;        // workgroups that run at once
  bool whole;            // no tile is split
};

// How a product's tiles are dealt to `slots` workgroups: whole rounds of them take their tile over all of K. The `rest` of
// a last, partial round is split over K, where that pays, and the partial sums are joined afterwards, in one of two ways:
//   parts > 0: every tile into `parts` runs of `per` steps, run by run, so that workgroups that share rows of the operands
//              read them at the same time (at most two items per workgroup);
//   parts = 0: all steps of the rest evenly, `per` neighbouring ones to a workgroup, which reach over at most two tiles, a
//              tile cut at most 17-fold.
// In steps' time (1.7 us on 256 x 256): an item costs 3 beside its own; equal parts (up to 8) 4 and 16 for each round of
// partial sums, even runs 42. 64 x 64 tiles have a sixteenth of the partial sums, 5 a round, but their joining waits once
// for each part, 1 in bf16 and 0.5 in fp32, and may have 16 (dx of 16 x 256 x 10112 in fp32 with the rest of the call: 42
// us, with 8 parts 50). Measured: 80 tiles of 256 steps 164 us in 3 parts and 197 in even runs, 136 tiles of 392 steps 500
// and 425. Even runs share no operand rows: bf16 tiles of 128 x 128, whose step takes half as long, then wait for memory,
// 2.5 times as long (376 tiles of 158 steps: 257 us in even runs, 160 whole).
struct LsPlan {
  uint32_t full, rest, steps, per, parts;
  uint32_t cost;  // of the last, partial round
};
constexpr uint32_t LS_CUTS = 16;

// The time of `rest` tiles in about q equal parts each, and those.
template <bool F32, int BM>
__host__ __device__ inline uint32_t ls_parts(uint32_t rest, uint32_t steps, uint32_t slots, uint32_t q, uint32_t& per,
                                             uint32_t& parts) {
  per = (steps + q - 1) / q;
  parts = (steps + per - 1) / per;
  const uint32_t load = rest * parts;
  const uint32_t join = BM == 64 ? 5 * load / slots + (F32 ? parts / 2 : parts) : 4 + 16 * load / slots;
  return (load + slots - 1) / slots * (per + 3) + join;
}
template <int BM>
__host__ __device__ inline bool ls_may(uint32_t rest, uint32_t steps, uint32_t slots, uint32_t q) {
  return q <= (BM == 64 ? LS_CUTS : 8) && q <= steps && rest * q <= 2 * slots;
}

// The plan but for equal parts.
template <bool F32, int BM>
__host__ __device__ inline LsPlan ls_unparted(uint32_t tiles, uint32_t steps, uint32_t slots) {
  const uint32_t rest = tiles % slots;
  if (rest == 0) return LsPlan{tiles, 0, steps, steps, 1, 0};
  const uint32_t even = (uint32_t)(((uint64_t)rest * steps + slots - 1) / slots);
  const uint32_t least = (steps + LS_CUTS - 1) / LS_CUTS, run = even > least ? even : least;
  const uint32_t run_cost = (!F32 && BM == 128 ? run * 5 / 2 : run) + 42;
  if (run_cost < steps + 3) return LsPlan{tiles - rest, rest, steps, run, 0, run_cost};
  return LsPlan{tiles, 0, steps, steps, 1, steps + 3};
}

template <bool F32, int BM>
LsPlan ls_plan(uint32_t tiles, uint32_t steps, uint32_t slots) {
  LsPlan pl = ls_unparted<F32, BM>(tiles, steps, slots);
  const uint32_t rest = tiles % slots;
  for (uint32_t q = 2; rest != 0 && ls_may<BM>(rest, steps, slots, q); ++q) {
    uint32_t per, parts;
    const uint32_t cost = ls_parts<F32, BM>(rest, steps, slots, q, per, parts);
    if (cost < pl.cost) pl = LsPlan{tiles - rest, rest, steps, per, parts, cost};
  }
  return pl;
}

// The same by a wave, a lane for each q: one after another their divisions take 2 us a kernel and 4 with 16 of them (dx of
// 1 x 256 x 1000, a product and its joining: 21 and 27 us with the rest of the call, so 18.6).
template <bool F32, int BM>
__device__ __forceinline__ LsPlan ls_plan_wave(uint32_t tiles, uint32_t steps, uint32_t slots) {
  const LsPlan pl = ls_unparted<F32, BM>(tiles, steps, slots);
  const uint32_t rest = tiles % slots, q = 2 + (threadIdx.x & 15);
  if (rest == 0 || steps < 2) return pl;
  uint32_t per = 0, parts = 0, key = 0xffffffffu;
  if (ls_may<BM>(rest, steps, slots, q)) key = ls_parts<F32, BM>(rest, steps, slots, q, per, parts) << 5 | q;  // < 2^26
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) key = min(key, (uint32_t)__shfl_xor((int)key, o));
  key = uniform(key);
  if ((key >> 5) >= pl.cost) return pl;
  const int at = (int)(key & 31) - 2;
  return LsPlan{tiles - rest, rest, steps, uniform((uint32_t)__shfl((int)per, at)), uniform((uint32_t)__shfl((int)parts, at)),
                key >> 5};
}

// Workgroups that share a CU.
constexpr int ls_per_cu(int bm, int epi) { return bm == 128 || (bm == 64 && epi != EPI_OUT) ? 2 : 1; }

// A target id as an int, -1 where it lies outside of one's range.
__device__ __forceinline__ int32_t raw_target(const void* targets, bool idx64, int64_t t) {
  if (!idx64) return static_cast<const int32_t*>(targets)[t];
  const int64_t v = static_cast<const int64_t*>(targets)[t];
  return v < 0 || v > 0x7fffffff ? -1 : (int32_t)v;
}

// Position of a work item: tile (m, n) and its K steps; part: its index among the partial sums, or -1 for a whole tile.
struct LsItem {
  int m, n, part, k0, nk;
  uint32_t tile;
};

__device__ __forceinline__ void ls_tile(uint32_t t, uint32_t ntm, uint32_t ntn, int& m, int& n) {
  const uint32_t grp = t / (8u * ntn), rem = t - grp * 8u * ntn;
  const uint32_t gm = min(8u, ntm - grp * 8u), q = rem / gm;
  n = (int)q;
  m = (int)(grp * 8u + rem - q * gm);
}

template <bool F32, int BM, int BN, int LA, int LB, int EPI>
__global__ __launch_bounds__(256, ls_per_cu(BM, EPI)) void ls_gemm_kernel(const LsParams p) {
  using OA = Operand<F32, BM, LA>;
  using OB = Operand<F32, BN, LB>;
  constexpr int MB = BM / 64, NB = BN / 64;  // 32x32 blocks of a wave
  constexpr int SLOT = (BM + BN) * 128;
  constexpr int NS = BM != 64 ? 2 : ls_per_cu(BM, EPI) == 1 ? 8 : 4;  // steps in LDS: few tiles wait for memory, many for the matrix units
  constexpr int BK = OA::BK, ESZ = OA::ESZ;
  __shared__ __align__(1024) uint8_t lds[NS * SLOT];
  // Staging of bf16 outputs, 32 rows of out by BM / 2 columns per wave (beside the slots: copies for the next item run
  // meanwhile).
  constexpr bool STAGED = !F32 && (EPI == EPI_S || EPI == EPI_OUT);
  __shared__ __align__(1024) uint8_t stage[STAGED ? 4 * 32 * BM : 16];
  constexpr bool TO_ROWS = EPI == EPI_OUT && LB == KC;  // dx: rows of out through `rows`
  constexpr int CH = BM / 16, RPI = 64 / CH;  // 16-byte chunks of a staged row, rows of a store
  constexpr int KB = 32 / RPI < 4 ? 32 / RPI : 4;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = (int)uniform((uint32_t)tid >> 6);
  const int wm = wave >> 1, wn = wave & 1;

  uint8_t* const stw = stage + (STAGED ? wave * 32 * BM : 0);

  if (EPI == EPI_LSE && blockIdx.x == 0 && tid == 0) *p.done = 0;

  // Tokens are N of z^T and dx^T, K of dW^T.
  const int64_t cnt = p.count != nullptr ? (int64_t)load_uniform(p.count) : p.T;
  const bool all = cnt >= p.T;
  constexpr bool tok_k = LB == KS;
  const int64_t N = tok_k ? p.N : cnt, K = tok_k ? cnt : p.K;
  const uint8_t* const A = tok_k && all && p.alt != nullptr ? p.alt : p.A;
  const uint8_t* const B = !tok_k && all && p.alt != nullptr ? p.alt : p.B;
  const uint32_t ntm = (uint32_t)((p.M + BM - 1) / BM), ntn = (uint32_t)((N + BN - 1) / BN);
  const int steps = (int)((K + BK - 1) / BK);
  const uint32_t tiles = ntm * ntn;  // < 2^31: the callers' limits on T and V

  // Work items of neighbouring blocks on an XCD are neighbouring tiles: 8 tiles of M by as many of N as it has room for.
  const uint32_t G = gridDim.x;
  const uint32_t first = (G & 7) == 0 ? (blockIdx.x & 7) * (G >> 3) + (blockIdx.x >> 3) : blockIdx.x;
  const LsPlan pl = EPI == EPI_OUT && !p.whole ? ls_plan_wave<F32, BM>(tiles, (uint32_t)steps, p.slots)
                                               : LsPlan{tiles, 0, (uint32_t)steps, (uint32_t)steps, 1, 0};
  // Of n items that are fewer than the blocks: this block's, or n. Each XCD has an eighth, neighbours, for its first blocks
  // (dealt like whole rounds, they would all go to the first XCDs: dW of 1777 x 1024 x 10112 with the rest of the call 106
  // us, so 119; the fp32 forward of 1024 x 512 x 10112 106 and 134).
  auto partial = [&](uint32_t n) -> uint32_t {
    if ((G & 7) != 0) return min((uint32_t)blockIdx.x, n);
    const uint32_t share = (n + 7) >> 3, i = blockIdx.x >> 3, at = (blockIdx.x & 7) * share + i;
    return i < share ? min(at, n) : n;
  };
  const float unit = EPI == EPI_S && p.g_unit != nullptr ? load_uniform(p.g_unit) : 1.0f;
  // This block's items: its tiles of the whole rounds, then (with the grid of p.slots blocks) its share of the rest.
  const uint32_t whole = pl.full / G, left = pl.full - whole * G, last_tile = partial(left);
  const uint32_t rounds = whole + (last_tile < left ? 1 : 0);
  const uint32_t load = pl.rest * pl.parts, load1 = load / G, load_left = load - load1 * G, last_part = partial(load_left);
  uint32_t lo = 0, cut = 0, hi = 0;  // even runs: steps lo .. cut - 1 of its first tile, cut .. hi - 1 of the next
  uint32_t total = rounds;
  if (EPI == EPI_OUT && pl.rest != 0) {
    if (pl.parts != 0) {
      total += load1 + (last_part < load_left ? 1 : 0);
    } else {
      const uint32_t units = pl.rest * pl.steps;  // < 2^29
      lo = min(first * pl.per, units);
      hi = min(lo + pl.per, units);
      cut = hi > lo ? min((lo / pl.steps + 1) * pl.steps, hi) : lo;
      total += (hi > lo ? 1 : 0) + (hi > cut ? 1 : 0);
    }
  }
  if (total == 0) return;
  auto item_of = [&](uint32_t r) {
    LsItem it = {0, 0, -1, 0, max(1, steps), r < whole ? first + r * G : whole * G + last_tile};  // no step at all: one of zeros
    if (EPI == EPI_OUT && r >= rounds) {
      const uint32_t s = r - rounds;
      if (pl.parts != 0) {
        const uint32_t q = s < load1 ? first + s * G : load1 * G + last_part, part = q / pl.rest;
        it.tile = pl.full + q - part * pl.rest;
        it.k0 = (int)(part * pl.per);
        it.nk = (int)min(pl.per, pl.steps - part * pl.per);
        it.part = (int)q;
      } else {
        const uint32_t from = s == 0 ? lo : cut, to = s == 0 ? cut : hi, q = from / pl.steps;
        it.tile = pl.full + q;
        it.k0 = (int)(from - q * pl.steps);
        it.nk = (int)(to - from);
        if (to - from < pl.steps) it.part = (int)(2 * first + s);
      }
    }
    ls_tile(it.tile, ntm, ntn, it.m, it.n);
    return it;
  };

  uint32_t va[OA::NDMA], vb[OB::NDMA];
#pragma unroll
  for (int j = 0; j < OA::NDMA; ++j) va[j] = OA::voff(j, wave, lane, (uint32_t)p.lda);
#pragma unroll
  for (int j = 0; j < OB::NDMA; ++j) vb[j] = OB::voff(j, wave, lane, (uint32_t)p.ldb);
  int fa[OA::NOFF], fb[OB::NOFF];
#pragma unroll
  for (int i = 0; i < OA::NOFF; ++i) fa[i] = OA::foff(i, wm, lane);
#pragma unroll
  for (int i = 0; i < OB::NOFF; ++i) fb[i] = BM * 128 + OB::foff(i, wn, lane);

  // The stream of K steps over this block's items, as the loads see it: `c` and its step, the operands' resources and the
  // K offset of a KC operand's rows (a KS operand's base moves instead: its end has to bound the step's K rows).
  uint32_t c_item = 0;
  LsItem c = item_of(c_item);
  int c_step = 0;
  uint32_t c_soff = 0;
  const uint8_t *pa, *pb;
  int64_t na, nb;  // bytes from pa, pb to the operands' ends
  auto enter = [&]() {
    const bool live = c_item < total;
    const int64_t k = (int64_t)c.k0 * BK, ma = (int64_t)c.m * BM, mb = (int64_t)c.n * BN;
    c_soff = 0;
    if (LA == KC) {
      pa = A + ma * p.lda + k * ESZ;
      na = live && k < K ? min((int64_t)BM, p.m_rows - ma) * p.lda - k * ESZ : 0;
    } else {
      pa = A + k * p.lda + ma * ESZ;
      na = live ? (K - k) * p.lda - ma * ESZ : 0;
    }
    if (LB == KC) {
      pb = B + mb * p.ldb + k * ESZ;
      nb = live && k < K ? min((int64_t)BN, N - mb) * p.ldb - k * ESZ : 0;
    } else {
      pb = B + k * p.ldb + mb * ESZ;
      nb = live ? (K - k) * p.ldb - mb * ESZ : 0;
    }
  };
  auto advance = [&]() {
    if (++c_step < c.nk) {
      c_soff += 128;
      if (LA == KS) pa += BK * p.lda, na -= BK * p.lda;
      if (LB == KS) pb += BK * p.ldb, nb -= BK * p.ldb;
      return;
    }
    c_step = 0;
    if (++c_item < total) c = item_of(c_item);
    enter();
  };

  // Position q of the stream lies in slot q % NS. Its slot is free once every wave has read its last fragments: in the
  // last quarter of q the first half of position q + NS is copied over it, in the first quarter of q + 1 the second,
  // and with two slots both have at least two quarters to arrive. (All in one quarter is 5 % slower, over three or four
  // quarters 2 % slower; the same loads through registers, a whole step ahead of their LDS stores, 2 % slower: at full
  // rate the chip's power decides, and the registers' way costs more of it.)
  constexpr int NC = OA::NDMA + OB::NDMA, Q = MB * NB;
  constexpr int C3 = NC / 2, C0 = NC - C3;
  const uint32_t lds0 = ls_lds_addr(lds);
  auto copy = [&](int j, int slot) {
    const uint32_t to = lds0 + (uint32_t)slot * SLOT;
    if (j < OA::NDMA) ls_dma(pa, na, va[j], LA == KC ? c_soff : 0u, to + wave * (BM * 32) + j * 1024);
    else ls_dma(pb, nb, vb[j - OA::NDMA], LB == KC ? c_soff : 0u, to + BM * 128 + wave * (BN * 32) + (j - OA::NDMA) * 1024);
  };
  enter();
#pragma unroll 1
  for (int q = 0; q < NS - 1; ++q) {
#pragma unroll
    for (int j = 0; j < NC; ++j) copy(j, q);
    advance();
  }
#pragma unroll
  for (int j = 0; j < C3; ++j) copy(j, NS - 1);
  asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((NS - 2) * NC + C3) : "memory");

  f32x16_t acc[MB][NB];
#pragma unroll
  for (int q = 0; q < MB * NB; ++q) ls_zero(acc[q / NB][q % NB]);
  u32x4_t fr[2][MB + NB];  // fragments of two quarters: A's, then B's
  auto read = [&](int j, const uint8_t* base, int u) {
    return j < MB ? OA::frag(base, fa, j, u) : OB::frag(base, fb, j - MB, u);
  };
#pragma unroll
  for (int j = 0; j < MB + NB; ++j) fr[0][j] = read(j, lds, 0);
  LsItem it = item_of(0);
  uint32_t item = 0;
  int slot = 0;
  // What a tile's tokens bring to its epilogue: the target, lse and gradient, or the row of out; lane l holds token 32 j +
  // l % 32's. Read at the tile's start: in the epilogue each read would wait for memory, and for the copies under way
  // before it.
  int32_t tk[NB];
  float tl[NB], tg[NB];
  auto tokens = [&]() {
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const int64_t n = (int64_t)it.n * BN + wn * (BN / 2) + 32 * j + (lane & 31);
      const bool ok = n < N;
      tk[j] = -1;
      if constexpr (EPI == EPI_LSE) {
        if (ok) tk[j] = p.raw != nullptr ? raw_target(p.raw, p.raw64, n) : p.tgt[n];
      } else if constexpr (EPI == EPI_S) {
        tl[j] = 0.0f;
        tg[j] = 1.0f;
        if (ok) {
          tk[j] = p.tgt[n];
          tl[j] = p.lse[n];
          if (p.g_row != nullptr) tg[j] = p.g_row[n];
        }
      } else if (TO_ROWS) {
        tk[j] = (int32_t)n;
        if (!all && ok) tk[j] = p.rows[n];
      }
    }
  };
  tokens();
#pragma unroll 1
  for (;;) {
#pragma unroll 1
    for (int s = 0; s < it.nk; ++s) {
      const int then = slot + 1 < NS ? slot + 1 : 0, before = slot > 0 ? slot - 1 : NS - 1;
      const uint8_t* base = lds + slot * SLOT;
      const uint8_t* next = lds + then * SLOT;
      // A quarter multiplies fr[half], reads fragments u of src into the other half after the first MFMAs, in the order of
      // their use, and stores and reloads quarter `part` of the loads after the others.
      auto quarter = [&](int half, const uint8_t* src, int u, int from, int cn, int to) {
#pragma unroll
        for (int q = 0; q < Q; ++q) {
          ls_mfma<F32>(acc[q / NB][q % NB], fr[half][q / NB], fr[half][MB + q % NB]);
#pragma unroll
          for (int e = 0; e < MB + NB; ++e)
            if (e * Q / (MB + NB) / 2 == q) {
              const int j = e == 0 ? 0 : (e <= NB ? MB + e - 1 : e - NB);
              fr[half ^ 1][j] = read(j, src, u);
            }
#pragma unroll
          for (int e = cn * q / Q; e < cn * (q + 1) / Q; ++e) copy(from + e, to);
        }
      };
      quarter(0, base, 1, C3, C0, before);
      quarter(1, base, 2, 0, 0, slot);
      quarter(0, base, 3, 0, 0, slot);
      advance();
      // This wave's copies of the next step have landed (those of the NS - 2 positions behind it may be under way), its
      // reads of this slot are done, and so are the others'.
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NS - 2) * NC) : "memory");
      ls_barrier();
      if constexpr (NS == 2) {  // the tokens' reads have landed with the copies: no wait for them later
#pragma unroll
        for (int j = 0; j < NB; ++j) {
          asm volatile("" : "+v"(tk[j]));
          if constexpr (EPI == EPI_S) asm volatile("" : "+v"(tl[j]), "+v"(tg[j]));
        }
      }
      quarter(1, next, 0, 0, C3, slot);
      slot = then;
    }
    ls_drain();

    // acc[i][j][q] of lane l: m = 32 i + 8 (q / 4) + 4 (l / 32) + q % 4 of the wave's rows, n = 32 j + l % 32.
    const int64_t mw = (int64_t)it.m * BM + wm * (BM / 2), nw = (int64_t)it.n * BN + wn * (BN / 2);
    const int lh = lane >> 5;
    const int mleft = (int)min((int64_t)(BM / 2), p.m_rows - mw);  // rows of the wave that exist (may be <= 0)
    float scale = 1.0f;
    const bool to_out = EPI != EPI_OUT || (it.part < 0 && p.last);  // else to the partial sums or the pieces' sums
    if (EPI == EPI_OUT && to_out) {
      if (p.g_scale != nullptr) scale *= *p.g_scale;
      if (p.r_scale != nullptr) scale *= *p.r_scale;
    }
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const int64_t n = nw + 32 * j + (lane & 31);
      const bool n_ok = n < N;
      // Where the token's target lies among the wave's rows, and what the softmax needs.
      const int rel = EPI == EPI_OUT ? -1 : tk[j] - (EPI == EPI_S ? (int)p.v0 : 0) - (int)mw;
      const float lse = EPI == EPI_S ? tl[j] : 0.0f;
      float g = EPI == EPI_S ? tg[j] : 1.0f;
      if (EPI == EPI_S && !F32 && p.g_row != nullptr) g /= unit;
      const int64_t row = TO_ROWS ? (int64_t)tk[j] : n;
      float mx = -__builtin_inff(), sum = 0.0f;
#pragma unroll
      for (int i = 0; i < MB; ++i) {
        f32x16_t v = ls_take(acc[i][j]);
        ls_zero(acc[i][j]);
        if constexpr (EPI == EPI_LSE) {
          if (mleft < BM / 2) ls_mask(v, mleft - 4 * lh - 32 * i, -__builtin_inff());
          float top = mx;
#pragma unroll
          for (int q = 0; q < 16; ++q) top = fmaxf(top, v[q]);
          const float ref = top == -__builtin_inff() ? 0.0f : top;
          float part[2] = {sum * __builtin_amdgcn_exp2f((mx - ref) * LOG2E), 0.0f};
#pragma unroll
          for (int q = 0; q < 16; ++q) part[q & 1] += __builtin_amdgcn_exp2f((v[q] - ref) * LOG2E);
          mx = top;
          sum = part[0] + part[1];
          if (__any((rel >> 5) == i)) {
#pragma unroll
            for (int q = 0; q < 16; ++q)
              if (rel == 32 * i + 8 * (q >> 2) + 4 * lh + (q & 3)) p.zt[n] = v[q];
          }
        } else {
          if constexpr (EPI == EPI_S) {
#pragma unroll
            for (int q = 0; q < 16; ++q) v[q] = __builtin_amdgcn_exp2f((v[q] - lse) * LOG2E);
            if (__any((rel >> 5) == i)) {
#pragma unroll
              for (int q = 0; q < 16; ++q)
                if (rel == 32 * i + 8 * (q >> 2) + 4 * lh + (q & 3)) v[q] -= 1.0f;
            }
            if (p.g_row != nullptr) v *= g;
            if (mleft < BM / 2) ls_mask(v, mleft - 4 * lh - 32 * i, 0.0f);
          } else {
            // The accumulators' own order: block (i, j) of wave w at 1024 ((w MB + i) NB + j), its quarters 256 apart, 4
            // per lane.
            const int64_t at = (((int64_t)wave * MB + i) * NB + j) * 1024 + 4 * lane;
            if (it.part < 0 && !p.first) {
              const float* a = p.acc + (int64_t)it.tile * (BM * BN) + at;
#pragma unroll
              for (int q4 = 0; q4 < 4; ++q4) {
                const f32x4_t f = *reinterpret_cast<const f32x4_t*>(a + 256 * q4);
#pragma unroll
                for (int q = 0; q < 4; ++q) v[4 * q4 + q] += f[q];
              }
            }
            if (!to_out) {
              float* a = (it.part < 0 ? p.acc + (int64_t)it.tile * (BM * BN) : p.split + (int64_t)it.part * (BM * BN)) + at;
#pragma unroll
              for (int q4 = 0; q4 < 4; ++q4)
                *reinterpret_cast<f32x4_t*>(a + 256 * q4) =
                    (f32x4_t){v[4 * q4], v[4 * q4 + 1], v[4 * q4 + 2], v[4 * q4 + 3]};
              continue;
            }
            v *= scale;
          }
          const int mstore = EPI == EPI_S ? BM / 2 : mleft;  // s: whole tiles; the others' rows are a multiple of 64
          if constexpr (F32) {
            if (n_ok && 32 * i < mstore) {
#pragma unroll
              for (int q4 = 0; q4 < 4; ++q4)
                *reinterpret_cast<f32x4_t*>(static_cast<float*>(p.out) + row * p.ldo + mw + 32 * i + 8 * q4 + 4 * lh) =
                    (f32x4_t){v[4 * q4], v[4 * q4 + 1], v[4 * q4 + 2], v[4 * q4 + 3]};
            }
          } else {
            // Through the wave's staging area, 32 rows of out by BM / 2 columns, so that stores write whole lines: 16-byte
            // chunk c of row r at c ^ r.
            const int r = lane & 31;
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4)
              *reinterpret_cast<uint2*>(stw + r * BM + 16 * ((4 * i + q4) ^ (r & (CH - 1))) + 8 * lh) =
                  make_uint2(pack_bf16x2(v[4 * q4], v[4 * q4 + 1]), pack_bf16x2(v[4 * q4 + 2], v[4 * q4 + 3]));
          }
        }
      }
      if constexpr (EPI == EPI_LSE) {
        const float mx2 = __shfl_xor(mx, 32), sum2 = __shfl_xor(sum, 32);
        lse_join(mx, sum, mx2, sum2);
        if (n_ok && lh == 0) p.part[((int64_t)it.m * 2 + wm) * p.T + n] = make_float2(mx, sum);
      } else if constexpr (STAGED) {
        if (!to_out) continue;
        const int mstore = EPI == EPI_S ? BM / 2 : mleft, c = lane % CH;
#pragma unroll
        for (int k0 = 0; k0 < 32 / RPI; k0 += KB) {  // several reads under way: one at a time the tile's 32 would wait for one another
          u32x4_t w[KB];
#pragma unroll
          for (int k = 0; k < KB; ++k) {
            const int rr = (k0 + k) * RPI + lane / CH;
            w[k] = ld16(stw + rr * BM + 16 * (c ^ (rr & (CH - 1))));
          }
#pragma unroll
          for (int k = 0; k < KB; ++k) {
            const int rr = (k0 + k) * RPI + lane / CH;
            const int64_t nn = nw + 32 * j + rr;
            const int r = TO_ROWS ? __shfl(tk[j], rr) : 32 * j + rr;
            if (nn < N && 8 * c < mstore) {
              if constexpr (TO_ROWS) st16(static_cast<uint16_t*>(p.out) + r * p.ldo + mw + 8 * c, w[k]);
              else ls_store_through(static_cast<uint16_t*>(p.out) + nw * p.ldo + mw,
                                    2u * ((uint32_t)r * (uint32_t)p.ldo + 8u * (uint32_t)c), w[k]);
            }
          }
        }
      }
    }
    if (++item >= total) break;
    it = item_of(item);
    tokens();
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

// Partition of the rows: rows[0 .. n-1] those that count, ascending, rows[n .. T-1] the ignored ones, *count = n, tgt[i]
// the target of rows[i] (-1: outside the vocabulary), and where given lse_c[i] = lse[rows[i]], g_c[i] = g[rows[i]], *unit the
// unit of those g.
struct LsList {
  int32_t *rows, *tgt, *count;
  const float* lse;
  float* lse_c;
  const float* g;
  float* g_c;
  float* unit;
};
constexpr int LS_RUNS = 8, LS_LIST = LS_RUNS * 1024;  // rows that a block of 1024 lists at a time, in runs of 1024

// Places of rows t0 .. t0 + LS_LIST - 1, of which `kept` before them count, by ballots and a scan of the waves' counts:
// place(t, i, v) for each, i its place in the list and v its target. Returns how many of them count.
template <typename IdxT, typename F>
__device__ __forceinline__ int ls_places(const IdxT* targets, int64_t ignore, int64_t T, int64_t t0, int64_t kept, int* sums,
                                         F place) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int64_t v[LS_RUNS];
  uint64_t mask[LS_RUNS];
#pragma unroll
  for (int e = 0; e < LS_RUNS; ++e) {
    const int64_t t = t0 + e * 1024 + tid;
    v[e] = t < T ? (int64_t)targets[t] : ignore;
  }
#pragma unroll
  for (int e = 0; e < LS_RUNS; ++e) {
    mask[e] = ballot64(v[e] != ignore);  // the places behind T hold ignore
    if (lane == 0) sums[e * 16 + wave] = __popcll(mask[e]);
  }
  __syncthreads();
  if (wave == 0) {  // exclusive prefix sums of the LS_RUNS * 16 counts
    const int a = sums[2 * lane], b = sums[2 * lane + 1];
    int s = a + b;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int u = __shfl_up(s, o);
      if (lane >= o) s += u;
    }
    sums[2 * lane] = s - a - b;
    sums[2 * lane + 1] = s - b;
    if (lane == 63) sums[LS_RUNS * 16] = s;
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < LS_RUNS; ++e) {
    const int64_t t = t0 + e * 1024 + tid;
    if (t >= T) break;
    const int64_t before = kept + sums[e * 16 + wave] + __popcll(mask[e] & ((1ull << lane) - 1));
    place(t, v[e] != ignore ? before : T - 1 - (t - before), v[e]);  // the ignored ones from the end
  }
  const int n = sums[LS_RUNS * 16];
  __syncthreads();
  return n;
}

// top: the largest finite g and -g so far.
__device__ __forceinline__ void ls_put(const LsList& l, int64_t t, int64_t i, int64_t v, int64_t ignore, int V,
                                       float (&top)[2]) {
  l.rows[i] = (int32_t)t;
  if (v == ignore) return;
  l.tgt[i] = v >= 0 && v < V ? (int32_t)v : -1;
  if (l.lse != nullptr) l.lse_c[i] = l.lse[t];
  if (l.g == nullptr) return;
  const float g = l.g[t];
  l.g_c[i] = g;
  if (fabsf(g) < __builtin_inff()) top[0] = fmaxf(top[0], g), top[1] = fmaxf(top[1], -g);
}

// *unit = the finite g of the largest size without its power of two, in [1, 2) with g's sign (1 where it is zero or
// subnormal; the positive one of two that are as large): by a block of 1024, of whose threads each has met `top`. Of the
// rows' g only this is taken out before s is rounded, so that their range stays what it is; with the sign, because the
// matrix unit's sums of -a are not exactly those of a.
__device__ __forceinline__ void ls_store_unit(float* unit, float (&top)[2], float (*red)[2]) {
#pragma unroll
  for (int e = 0; e < 2; ++e) {
#pragma unroll
    for (int o = 32; o; o >>= 1) top[e] = fmaxf(top[e], __shfl_xor(top[e], o));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6][e] = top[e];
  }
  __syncthreads();
  if (threadIdx.x != 0) return;
#pragma unroll
  for (int w = 1; w < 16; ++w) top[0] = fmaxf(top[0], red[w][0]), top[1] = fmaxf(top[1], red[w][1]);
  const float g = top[1] > top[0] ? -top[1] : top[0];
  *unit = fabsf(g) < 0x1p-126f ? 1.0f : __uint_as_float((__float_as_uint(g) & 0x807fffffu) | 0x3f800000u);
}

// The list by one block (16384 rows: 4.5 us with the targets in the caches, 9 without; with 1024 rows at a time 14.5).
template <typename IdxT>
__global__ __launch_bounds__(1024) void ls_rows_kernel(const IdxT* __restrict__ targets, int64_t ignore, int64_t T, int V,
                                                       LsList l) {
  __shared__ int sums[LS_RUNS * 16 + 1];
  __shared__ float red[16][2];
  int64_t kept = 0;  // rows that count, so far
  float top[2] = {0.0f, 0.0f};
  for (int64_t t0 = 0; t0 < T; t0 += LS_LIST)
    kept += ls_places(targets, ignore, T, t0, kept, sums,
                      [&](int64_t t, int64_t i, int64_t v) { ls_put(l, t, i, v, ignore, V, top); });
  if (threadIdx.x == 0) *l.count = (int32_t)kept;
  if (l.unit != nullptr) ls_store_unit(l.unit, top, red);
}

__device__ __forceinline__ void ls_copy_row(const uint8_t* x, uint8_t* xc, uint8_t* zero, int64_t i, int64_t r, bool counts,
                                            int bytes) {
  for (int c = 16 * (threadIdx.x & 63); c < bytes; c += 1024) {
    if (counts) st16(xc + i * bytes + c, ld16(x + r * bytes + c));
    else st16(zero + r * bytes + c, (u32x4_t){0u, 0u, 0u, 0u});
  }
}

// Up to LS_LIST rows: the list and ls_gather_kernel's copies in one launch. Every block makes the list, the first one
// stores it, and each copies the 16 rows of its places: 2 us a call less than two launches at 61 to 4096 rows (1777 rows,
// 40 % ignored: 5 and 7.5 with the gap between), 0.5 to 1 at 8192.
template <typename IdxT>
__global__ __launch_bounds__(1024) void ls_list_kernel(const IdxT* __restrict__ targets, int64_t ignore, int64_t T, int V,
                                                       LsList l, const uint8_t* __restrict__ x, uint8_t* __restrict__ xc,
                                                       uint8_t* __restrict__ zero, int bytes) {
  __shared__ int sums[LS_RUNS * 16 + 1];
  __shared__ int own[16];
  __shared__ float red[16][2];
  float top[2] = {0.0f, 0.0f};
  const int n = ls_places(targets, ignore, T, 0, 0, sums, [&](int64_t t, int64_t i, int64_t v) {
    if (blockIdx.x == 0) ls_put(l, t, i, v, ignore, V, top);
    if ((int)(i >> 4) == (int)blockIdx.x) own[i & 15] = (int)t;
  });
  if (blockIdx.x == 0 && threadIdx.x == 0) *l.count = n;
  if (blockIdx.x == 0 && l.unit != nullptr) ls_store_unit(l.unit, top, red);
  const int wave = (int)uniform(threadIdx.x >> 6);
  const int64_t i = (int64_t)blockIdx.x * 16 + wave;
  if (n >= T || i >= T || (i >= n && zero == nullptr)) return;
  ls_copy_row(x, xc, zero, i, (int64_t)own[wave], i < n, bytes);
}

// xc[i] = x[rows[i]] for the rows that count, unless all do; zero[rows[i]] = 0 for the others (zero may be NULL). One wave per
// row, rows of `bytes` bytes.
__global__ __launch_bounds__(256) void ls_gather_kernel(const uint8_t* __restrict__ x, const int32_t* __restrict__ rows,
                                                        const int32_t* __restrict__ count, uint8_t* __restrict__ xc,
                                                        uint8_t* __restrict__ zero, int64_t T, int bytes) {
  const int64_t n = load_uniform(count);
  if (n >= T) return;
  const int64_t i = (int64_t)blockIdx.x * 4 + (int)uniform(threadIdx.x >> 6);
  if (i >= T || (i >= n && zero == nullptr)) return;
  ls_copy_row(x, xc, zero, i, (int64_t)rows[i], i < n, bytes);
}

// lse and loss of R rows per block from their partial maxima and sums, which its 1024 / R groups of lanes share; rows that
// do not count get loss 0. Few rows wait for the groups' loads, many for the blocks' sums to reach the last one: 16 rows to
// a block up to 2048 rows, else 64 (61 rows of 316 entries 3.8 and 5.7 us; 1777 7.2 and 7.4; with the mean of 4099 13.9 and
// 10.8, of 16384 27 and 10). Rows are those of the list, or with `raw` the call's own. Then *reduced = the sum of all
// losses (mean: over the rows that count; 0 where none does), *row_scale = the factor of every row's gradient: by the block
// that is done last, from the blocks' sums in their order (*done is 0 before and after).
template <int R>
__global__ __launch_bounds__(1024) void ls_finish_kernel(const float2* __restrict__ part, int entries,
                                                         const float* __restrict__ zt, const int32_t* __restrict__ tgt,
                                                         const int32_t* __restrict__ rows,
                                                         const int32_t* __restrict__ count, const void* raw, bool raw64,
                                                         int64_t ignore, int V, int64_t T, float* __restrict__ loss,
                                                         float* __restrict__ lse, bool mean, double* block_sum,
                                                         int32_t* block_n, uint32_t* done, float* __restrict__ reduced,
                                                         float* __restrict__ row_scale) {
  __shared__ float2 red[16][R];
  __shared__ bool last;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, group = threadIdx.x / R;
  const int64_t n = raw != nullptr ? T : (int64_t)load_uniform(count);
  const int64_t i = (int64_t)blockIdx.x * R + (lane & (R - 1));
  float m = -__builtin_inff(), s = 0.0f;
  auto join_lanes = [&]() {  // the wave's groups, each lane with all of its row's
#pragma unroll
    for (int o = R; o < 64; o <<= 1) lse_join(m, s, __shfl_xor(m, o), __shfl_xor(s, o));
  };
  if (i < n) {
#pragma unroll 4
    for (int e = group; e < entries; e += 1024 / R) {
      const float2 v = part[(int64_t)e * T + i];
      lse_join(m, s, v.x, v.y);
    }
  }
  join_lanes();
  if (lane < R) red[wave][lane] = make_float2(m, s);
  __syncthreads();
  if (wave == 0) {
    m = -__builtin_inff(), s = 0.0f;
#pragma unroll
    for (int w = 0; w < 16; w += 64 / R) {
      const float2 v = red[w + lane / R][lane & (R - 1)];
      lse_join(m, s, v.x, v.y);
    }
    join_lanes();
    double sum = 0.0;
    int c = 0;
    if (i < T && lane < R) {
      const int64_t r = raw != nullptr ? i : (int64_t)rows[i];
      int tg = -1;
      bool in = i < n;
      if (raw != nullptr) {
        const int64_t v = raw64 ? static_cast<const int64_t*>(raw)[i] : (int64_t)static_cast<const int32_t*>(raw)[i];
        in = v != ignore;
        tg = v >= 0 && v < V ? (int)v : -1;
      } else if (in) {
        tg = tgt[i];
      }
      float l = 0.0f, z = 0.0f;
      if (in) {
        z = tg < 0 ? __builtin_nanf("") : m + logf(s);  // a target outside the vocabulary shows as NaN
        l = tg < 0 ? z : z - zt[i];
        sum = (double)l;
        c = 1;
      }
      loss[r] = l;
      if (lse != nullptr) lse[r] = z;
    }
    if (reduced != nullptr) {
#pragma unroll
      for (int o = 32; o; o >>= 1) {
        const uint64_t u = __builtin_bit_cast(uint64_t, sum);
        const uint32_t lo = __shfl_xor((int)(uint32_t)u, o), hi = __shfl_xor((int)(uint32_t)(u >> 32), o);
        sum += __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
        c += __shfl_xor(c, o);
      }
      if (lane == 0) {
        __hip_atomic_store(block_sum + blockIdx.x, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(block_n + blockIdx.x, c, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last = __hip_atomic_fetch_add(done, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
      }
    }
  }
  if (reduced == nullptr) return;
  __syncthreads();
  if (!last) return;
  __shared__ double sums[1024];
  __shared__ int64_t ns[1024];
  double a = 0.0;
  int64_t k = 0;
  for (int b = threadIdx.x; b < (int)gridDim.x; b += 1024) {
    a += __hip_atomic_load(block_sum + b, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    k += __hip_atomic_load(block_n + b, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  sums[threadIdx.x] = a;
  ns[threadIdx.x] = k;
  __syncthreads();
  for (int o = 512; o; o >>= 1) {
    if ((int)threadIdx.x < o) {
      sums[threadIdx.x] += sums[threadIdx.x + o];
      ns[threadIdx.x] += ns[threadIdx.x + o];
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    const double d = mean ? (double)(ns[0] > 0 ? ns[0] : 1) : 1.0;
    *reduced = (float)(sums[0] / d);
    if (row_scale != nullptr) *row_scale = (float)(1.0 / d);
    *done = 0;
  }
}

// The split tiles of a product (ls_gemm_kernel with the same parameters): their parts in order and the earlier pieces' sums,
// to out or to the pieces' sums. A thread takes 8 consecutive m of one n, in the accumulators' order 4 at a time (32 of them
// leave too few loads under way: 80 tiles of 256 x 256 in 3 parts 16.5 us, so 18.1; 36 of 64 x 64 in fp32 5.9 and 7.2).
template <typename E, int BM, int BN, bool TOK_K>
__global__ __launch_bounds__(256) void ls_join_kernel(const LsParams p) {
  constexpr int BK = 128 / sizeof(E), NB = BN / 64, W = 2, PER = BM * BN / (4 * W);  // groups of four values of a thread, threads of a tile
  const int64_t cnt = (int64_t)load_uniform(p.count);
  const int64_t N = TOK_K ? p.N : cnt, K = TOK_K ? cnt : p.K;
  const uint32_t ntm = (uint32_t)((p.M + BM - 1) / BM), ntn = (uint32_t)((N + BN - 1) / BN);
  const LsPlan pl = ls_plan_wave<sizeof(E) == 4, BM>(ntm * ntn, (uint32_t)((K + BK - 1) / BK), p.slots);
  float scale = 1.0f;
  if (p.last && p.g_scale != nullptr) scale *= *p.g_scale;
  if (p.last && p.r_scale != nullptr) scale *= *p.r_scale;
  for (uint32_t id = blockIdx.x * 256 + threadIdx.x; id < pl.rest * PER; id += gridDim.x * 256) {
    const uint32_t q = id / PER, in = id - q * PER;
    // Its partial sums: one per part, or one per workgroup whose run of steps meets the tile (one alone has written it).
    const uint32_t lo = q * pl.steps;
    const uint32_t c0 = pl.parts != 0 ? 0 : lo / pl.per, c1 = pl.parts != 0 ? pl.parts - 1 : (lo + pl.steps - 1) / pl.per;
    if (c0 == c1) continue;
    const int ln = in & 31, k0 = (int)(in >> 5) % (8 / W) * W, blk = (int)(in >> 5) / (8 / W);  // block (w MB + i) NB + j
    int tm, tn;
    ls_tile(pl.full + q, ntm, ntn, tm, tn);
    const int j = blk % NB, i = blk / NB % (BM / 64), w = blk / NB / (BM / 64);
    const int64_t m = (int64_t)tm * BM + (w >> 1) * (BM / 2) + 32 * i, n = (int64_t)tn * BN + (w & 1) * (BN / 2) + 32 * j + ln;
    if (m >= p.M || n >= N) continue;
    f32x4_t v[W];  // m = 4 (k0 + k)
    const int64_t at = (int64_t)blk * 1024 + 4 * ln;
#pragma unroll
    for (int k = 0; k < W; ++k) v[k] = (f32x4_t){0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t c = c0; c <= c1; ++c) {
      // Even runs: the tile is the second of the workgroup's, or the first.
      const uint32_t part = pl.parts != 0 ? c * pl.rest + q : 2 * c + (c * pl.per < lo ? 1 : 0);
      const float* a = p.split + (int64_t)part * (BM * BN) + at;
#pragma unroll
      for (int k = 0; k < W; ++k) v[k] += *reinterpret_cast<const f32x4_t*>(a + 128 * (k0 + k));
    }
    float* const c = p.acc + (int64_t)(pl.full + q) * (BM * BN) + at;
    if (!p.first) {
#pragma unroll
      for (int k = 0; k < W; ++k) v[k] += *reinterpret_cast<const f32x4_t*>(c + 128 * (k0 + k));
    }
    if (!p.last) {
#pragma unroll
      for (int k = 0; k < W; ++k) *reinterpret_cast<f32x4_t*>(c + 128 * (k0 + k)) = v[k];
      continue;
    }
    E* const o = static_cast<E*>(p.out) + (TOK_K || cnt >= p.T ? n : (int64_t)p.rows[n]) * p.ldo + m + 4 * k0;
#pragma unroll
    for (int k = 0; k < W; ++k) {
      v[k] *= scale;
      if constexpr (sizeof(E) == 4) *reinterpret_cast<f32x4_t*>(o + 4 * k) = v[k];
      else if (k & 1)
        st16(o + 4 * (k - 1), (u32x4_t){pack_bf16x2(v[k - 1][0], v[k - 1][1]), pack_bf16x2(v[k - 1][2], v[k - 1][3]),
                                        pack_bf16x2(v[k][0], v[k][1]), pack_bf16x2(v[k][2], v[k][3])});
    }
  }
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

uint32_t ls_slots(int bm, int epi) { return (uint32_t)(device_cus() * ls_per_cu(bm, epi)); }

template <bool F32, int BM, int BN, int LA, int LB, int EPI>
hipError_t ls_gemm(LsParams p, hipStream_t st) {
  p.slots = ls_slots(BM, EPI);
  // dW's tiles do not depend on the rows that count, and fewer of those (fewer steps) make splitting no better: where T rows
  // leave the tiles whole there is nothing to join (1777 x 1024 x 10112: 4 us).
  if (EPI == EPI_OUT && LB == KS)
    p.whole = ls_plan<F32, BM>((uint32_t)(ceil_div(p.M, BM) * ceil_div(p.N, BN)),
                               (uint32_t)ceil_div(p.K, 128 / (F32 ? 4 : 2)), p.slots).rest == 0;
  const int64_t tiles = ceil_div(p.M, BM) * ceil_div(p.N, BN);
  const unsigned grid = EPI == EPI_OUT || tiles > p.slots ? p.slots : (unsigned)tiles;
  hipLaunchKernelGGL((ls_gemm_kernel<F32, BM, BN, LA, LB, EPI>), dim3(grid), dim3(256), 0, st, p);
  const hipError_t e = hipGetLastError();
  if (EPI != EPI_OUT || p.whole || e != hipSuccess) return e;
  using E = typename std::conditional<F32, float, uint16_t>::type;
  hipLaunchKernelGGL((ls_join_kernel<E, BM, BN, LB == KS>), dim3(1024), dim3(256), 0, st, p);
  return hipGetLastError();
}

// Tile side of the products over the vocabulary, whose tiles stay whole. bf16: 64 where one round of such tiles, two to a
// CU, is all (61 x 1024 x 10112 forward and dx: 15.6 and 36 us, with 128 18.5 and 42; 128 tokens 17.1 and 38, 18.5 and 42;
// 2 rounds, 200 tokens: 25.5 and 51, 18.8 and 47). Else a round of 256 x 256 tiles takes 30 us at h = 1024 and one of 128 x
// 128, two to a CU, 17 (16384 x 1024 x 10112: 302 and 350 us; 1777 tokens: 60 and 51; 300: 30 and 17). fp32 multiplies at a
// sixteenth of the rate, so that a large tile's reuse is worth nothing, and the work on the busiest CU decides: 64 where it
// gets at most three times as many of those as of 128 (of 64 tokens the larger tile is half empty: 61 x 2048 x 50021
// forward 155 and 244 us; 100 x 1024 x 10112 45 and 71; three for one, 200 tokens, 69 and 72, 2600 x 512 x 2000 67 and 72;
// seven for two, 700 tokens, 137 and 129).
int tile_z(int64_t M, int64_t N, bool f32) {
  const int64_t cus = device_cus(), n64 = ceil_div(M, 64) * ceil_div(N, 64), n128 = ceil_div(M, 128) * ceil_div(N, 128);
  if (f32) return ceil_div(n64, cus) <= 3 * ceil_div(n128, cus) ? 64 : 128;
  if (n64 <= 2 * cus) return 64;
  return 7 * ceil_div(ceil_div(M, 256) * ceil_div(N, 256), cus) <= 4 * ceil_div(n128, 2 * cus) ? 256 : 128;
}

// A bf16 product's time over K that may be split, in steps of its tiles.
template <int B>
uint64_t ls_cost(int64_t M, int64_t N, int64_t steps) {
  const uint32_t tiles = (uint32_t)(ceil_div(M, B) * ceil_div(N, B)), slots = ls_slots(B, EPI_OUT);
  return (uint64_t)(tiles / slots) * (uint64_t)(steps + 3) + ls_plan<false, B>(tiles, (uint32_t)steps, slots).cost +
         (B == 256 ? 2 * ((tiles + slots - 1) / slots) : 0);  // its longer epilogue
}

// Of the gradients' products, whose tiles can be split over K. 64 (with eight steps in LDS) for few tiles of 128, or for at
// most one per two CUs and little K (dx of 61 x 1024 x 10112: 37 and 49 us with the rest of the call; of 400 x 1024 x
// 30000, 32 tiles, 173 and 116, in fp32 of 400 x 1024 x 10112 224 and 192; dw of 2600 x 512 x 2000 39 and 47, of 1500 x
// 1024 x 2000, 128 tiles of 24 steps, 42 and 47, of 700 x 256 x 10112, 158 tiles, 35 and 28). Else bf16 takes 128 or 256 by
// the time that the plan gives either, a step of 256 being worth 1.6 (two of 128 to a CU): dx of 1280 x 1024 x 10112 88 and
// 100 us, of 1536 x 2048 x 50021 762 and 648; dw of 100 x 1024 x 10112 28 and 30, of 6000 x 1024 x 10112 290 and 321, of
// 1536 x 2048 x 50021 727 and 667. fp32 has no use for 256.
int tile_k(int64_t M, int64_t N, int64_t steps, bool f32) {
  const int64_t cus = device_cus(), n128 = ceil_div(M, 128) * ceil_div(N, 128);
  if (8 * n128 < cus || (2 * n128 <= cus && n128 * steps <= (f32 ? 16 : 12) * cus)) return 64;
  if (f32) return 128;
  return 8 * ls_cost<256>(M, N, steps) <= 5 * ls_cost<128>(M, N, steps) ? 256 : 128;
}

int ls_finish_rows(int64_t T) { return T <= 2048 ? 16 : 64; }

// Bytes of a product's partial sums, and of its running sums.
size_t split_bytes(int64_t M, int64_t N, int b) {
  const int64_t most = 2 * (int64_t)ls_slots(b, EPI_OUT), cuts = ceil_div(M, b) * ceil_div(N, b) * LS_CUTS * 2;
  return 4 * (size_t)(b * b) * (size_t)(cuts < most ? cuts : most);
}
size_t acc_bytes(int64_t M, int64_t N, int b) { return 4 * (size_t)(b * b) * (size_t)(ceil_div(M, b) * ceil_div(N, b)); }

size_t up(size_t v) { return (v + 255) / 256 * 256; }

struct Layout {
  size_t rows, tgt, count, xc, part, zt, bsum, bn, done, lse, g, unit, s, acc, split, end;
  int entries;             // of the forward's partial sums
  int64_t piece;           // vocabulary rows of a piece (multiple of 256)
  int pieces;
  int tile_s, tile_x, tile_w;  // tile sides of the forward's or s's, dx's and dw's products
  bool raw;                // forward: no list of rows, every row's logits
};

constexpr int64_t PIECE_BYTES = (int64_t)256 << 20;

Layout layout(int64_t T, int h, int V, bool f32, bool fwd, bool need_x, bool need_w) {
  Layout l = {};
  const size_t esz = f32 ? 4 : 2;
  size_t off = 0;
  auto take = [&](size_t n) {
    const size_t at = off;
    off = up(off + n);
    return at;
  };
  l.raw = fwd && T <= 256;  // few tokens: skipping rows would save less than the launch that lists them costs
  l.rows = take(l.raw ? 0 : 4 * T);
  l.tgt = take(l.raw ? 0 : 4 * T);
  l.count = take(4);
  l.xc = take(l.raw ? 0 : esz * T * h);
  l.tile_s = tile_z(V, T, f32);
  if (fwd) {
    l.entries = (int)(2 * ceil_div(V, l.tile_s));
    l.part = take(8 * (size_t)l.entries * T);
    l.zt = take(4 * T);
    l.bsum = take(8 * ceil_div(T, ls_finish_rows(T)));
    l.bn = take(4 * ceil_div(T, ls_finish_rows(T)));
    l.done = take(4);
  } else {
    const int64_t vt = ceil_div(V, 256);
    int64_t most = PIECE_BYTES / ((int64_t)esz * T) / 256;
    if (most < 1) most = 1;
    l.pieces = (int)ceil_div(vt, most);
    const int64_t pt = ceil_div(vt, l.pieces);
    l.pieces = (int)ceil_div(vt, pt);
    l.piece = pt * 256;
    l.lse = take(4 * T);
    l.g = take(4 * T);
    l.unit = take(4);
    l.s = take(esz * (size_t)T * l.piece);
    const int64_t bk = f32 ? 32 : 64, n = l.piece < V ? l.piece : V;
    l.tile_s = tile_z(n, T, f32);
    l.tile_x = tile_k(h, T, ceil_div(n, bk), f32);
    l.tile_w = tile_k(h, n, ceil_div(T, bk), f32);
    l.acc = take(need_x && l.pieces > 1 ? acc_bytes(h, T, l.tile_x) : 0);
    const size_t sx = need_x ? split_bytes(h, T, l.tile_x) : 0, sw = need_w ? split_bytes(h, n, l.tile_w) : 0;
    l.split = take(sx > sw ? sx : sw);
  }
  l.end = off;
  return l;
}

template <typename P>
P* at(void* base, size_t off) {
  return reinterpret_cast<P*>(static_cast<char*>(base) + off);
}

#define LS_TRY(e)                       \
  do {                                  \
    const hipError_t e_ = (e);          \
    if (e_ != hipSuccess) return e_;    \
  } while (0)

// The list of rows and their copies.
template <typename IdxT>
hipError_t ls_rows(const IdxT* targets, int64_t ignore, int64_t T, int V, const LsList& l, const void* x, void* xc, void* zero,
                   int bytes, hipStream_t st) {
  const uint8_t* from = static_cast<const uint8_t*>(x);
  uint8_t *to = static_cast<uint8_t*>(xc), *zeros = static_cast<uint8_t*>(zero);
  if (T <= LS_LIST) {
    hipLaunchKernelGGL(ls_list_kernel<IdxT>, dim3((unsigned)ceil_div(T, 16)), dim3(1024), 0, st, targets, ignore, T, V, l,
                       from, to, zeros, bytes);
    return hipGetLastError();
  }
  hipLaunchKernelGGL(ls_rows_kernel<IdxT>, dim3(1), dim3(1024), 0, st, targets, ignore, T, V, l);
  LS_TRY(hipGetLastError());
  hipLaunchKernelGGL(ls_gather_kernel, dim3((unsigned)ceil_div(T, 4)), dim3(256), 0, st, from, l.rows, l.count, to, zeros, T,
                     bytes);
  return hipGetLastError();
}

hipError_t ls_rows_any(const void* targets, bool idx64, int64_t ignore, int64_t T, int V, const LsList& l, const void* x,
                       void* xc, void* zero, int bytes, hipStream_t st) {
  return idx64 ? ls_rows(static_cast<const int64_t*>(targets), ignore, T, V, l, x, xc, zero, bytes, st)
               : ls_rows(static_cast<const int32_t*>(targets), ignore, T, V, l, x, xc, zero, bytes, st);
}

template <bool F32, int LA, int LB, int EPI>
hipError_t ls_gemm_any(const LsParams& p, int tile, hipStream_t st) {
  if (tile == 64) return ls_gemm<F32, 64, 64, LA, LB, EPI>(p, st);
  if constexpr (!F32)
    if (tile == 256) return ls_gemm<F32, 256, 256, LA, LB, EPI>(p, st);
  return ls_gemm<F32, 128, 128, LA, LB, EPI>(p, st);
}

template <bool F32>
hipError_t ce_forward(const void* x, const void* w, const void* targets, bool idx64, int64_t ignore, float* loss,
                      float* lse, float* reduced, float* row_scale, bool mean, int64_t T, int h, int V, void* ws,
                      hipStream_t st) {
  const Layout l = layout(T, h, V, F32, true, false, false);
  int32_t* rows = at<int32_t>(ws, l.rows);
  int32_t* tgt = at<int32_t>(ws, l.tgt);
  int32_t* count = at<int32_t>(ws, l.count);
  const int64_t rb = (int64_t)h * (F32 ? 4 : 2);
  if (!l.raw) {
    const LsList list = {rows, tgt, count, nullptr, nullptr, nullptr, nullptr, nullptr};
    LS_TRY(ls_rows_any(targets, idx64, ignore, T, V, list, x, at<void>(ws, l.xc), nullptr, (int)rb, st));
  }
  LsParams p = {};
  p.A = static_cast<const uint8_t*>(w);
  p.B = l.raw ? static_cast<const uint8_t*>(x) : at<const uint8_t>(ws, l.xc);
  p.alt = static_cast<const uint8_t*>(x);
  p.lda = p.ldb = rb;
  p.M = p.m_rows = V;
  p.N = p.T = T;
  p.K = h;
  p.count = l.raw ? nullptr : count;
  p.raw = l.raw ? targets : nullptr;
  p.raw64 = idx64;
  p.part = at<float2>(ws, l.part);
  p.tgt = tgt;
  p.zt = at<float>(ws, l.zt);
  p.done = at<uint32_t>(ws, l.done);
  LS_TRY((ls_gemm_any<F32, KC, KC, EPI_LSE>(p, l.tile_s, st)));
  const int per = ls_finish_rows(T);
  hipLaunchKernelGGL(per == 16 ? ls_finish_kernel<16> : ls_finish_kernel<64>, dim3((unsigned)ceil_div(T, per)), dim3(1024), 0, st,
                     p.part, l.entries, p.zt, tgt, rows, count, p.raw, idx64, ignore, V, T, loss, lse, mean,
                     at<double>(ws, l.bsum), at<int32_t>(ws, l.bn), p.done, reduced, row_scale);
  return hipGetLastError();
}

template <bool F32>
hipError_t ce_backward(const float* g, bool g_rows, const float* r_scale, const void* x, const void* w,
                       const void* targets, bool idx64, int64_t ignore, const float* lse, void* dx, void* dw, int64_t T,
                       int h, int V, void* ws, hipStream_t st) {
  const Layout l = layout(T, h, V, F32, false, dx != nullptr, dw != nullptr);
  int32_t* rows = at<int32_t>(ws, l.rows);
  int32_t* tgt = at<int32_t>(ws, l.tgt);
  int32_t* count = at<int32_t>(ws, l.count);
  const int64_t rb = (int64_t)h * (F32 ? 4 : 2);
  const int64_t esz = F32 ? 4 : 2;
  float* unit = g_rows && !F32 ? at<float>(ws, l.unit) : nullptr;
  const LsList list = {rows, tgt, count, lse, at<float>(ws, l.lse), g_rows ? g : nullptr, at<float>(ws, l.g), unit};
  LS_TRY(ls_rows_any(targets, idx64, ignore, T, V, list, x, at<void>(ws, l.xc), dx, (int)rb, st));
  const uint8_t* xc = at<const uint8_t>(ws, l.xc);
  const float* scale = g_rows ? unit : g;
  for (int i = 0; i < l.pieces; ++i) {
    const int64_t v0 = (int64_t)i * l.piece, n = V - v0 < l.piece ? V - v0 : l.piece;
    const int64_t pitch = ceil_div(n, 256) * 256;
    const uint8_t* wp = static_cast<const uint8_t*>(w) + v0 * rb;
    LsParams p = {};
    p.T = T;
    p.count = count;
    // s [T, pitch]
    p.A = wp;
    p.B = xc;
    p.alt = static_cast<const uint8_t*>(x);
    p.lda = p.ldb = rb;
    p.N = T;
    p.K = h;
    p.v0 = v0;
    p.tgt = tgt;
    p.lse = at<float>(ws, l.lse);
    p.g_row = g_rows ? at<float>(ws, l.g) : nullptr;
    p.g_unit = unit;
    p.out = at<void>(ws, l.s);
    p.ldo = pitch;
    p.M = pitch;  // whole tiles: the columns behind the piece become zeros
    p.m_rows = n;
    LS_TRY((ls_gemm_any<F32, KC, KC, EPI_S>(p, l.tile_s, st)));
    LsParams q = {};
    q.B = at<const uint8_t>(ws, l.s);
    q.lda = rb;
    q.ldb = pitch * esz;
    q.M = q.m_rows = h;
    q.T = T;
    q.count = count;
    q.rows = rows;
    q.ldo = h;
    q.g_scale = scale;
    q.r_scale = r_scale;
    q.split = at<float>(ws, l.split);
    if (dx != nullptr) {
      q.A = wp;
      q.N = T;
      q.K = n;
      q.out = dx;
      q.acc = at<float>(ws, l.acc);
      q.first = i == 0;
      q.last = i == l.pieces - 1;
      LS_TRY((ls_gemm_any<F32, KS, KC, EPI_OUT>(q, l.tile_x, st)));
    }
    if (dw != nullptr) {
      q.A = xc;
      q.alt = static_cast<const uint8_t*>(x);
      q.N = n;
      q.K = T;
      q.out = static_cast<uint8_t*>(dw) + v0 * rb;
      q.first = q.last = true;
      LS_TRY((ls_gemm_any<F32, KS, KS, EPI_OUT>(q, l.tile_w, st)));
    }
  }
  return hipSuccess;
}

}  // namespace

size_t linear_ce_workspace(int64_t T, int h, int V, bool f32, bool forward, bool need_x, bool need_w) {
  return layout(T, h, V, f32, forward, need_x, need_w).end;
}

hipError_t launch_linear_ce_forward(const void* x, const void* w, const void* targets, bool idx64, int64_t ignore,
                                    float* loss, float* lse, float* reduced, float* row_scale, bool mean, int64_t T,
                                    int h, int V, void* ws, bool f32, hipStream_t st) {
  return f32 ? ce_forward<true>(x, w, targets, idx64, ignore, loss, lse, reduced, row_scale, mean, T, h, V, ws, st)
             : ce_forward<false>(x, w, targets, idx64, ignore, loss, lse, reduced, row_scale, mean, T, h, V, ws, st);
}

hipError_t launch_linear_ce_backward(const float* g, bool g_rows, const float* r_scale, const void* x, const void* w,
                                     const void* targets, bool idx64, int64_t ignore, const float* lse, void* dx,
                                     void* dw, int64_t T, int h, int V, void* ws, bool f32, hipStream_t st) {
  return f32 ? ce_backward<true>(g, g_rows, r_scale, x, w, targets, idx64, ignore, lse, dx, dw, T, h, V, ws, st)
             : ce_backward<false>(g, g_rows, r_scale, x, w, targets, idx64, ignore, lse, dx, dw, T, h, V, ws, st);
}

}  // namespace q38
