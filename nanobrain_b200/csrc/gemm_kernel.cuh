// Matrix products of the gated feed-forward block on the tensor cores, with what surrounds them in their epilogues:
//
//   kGemmGate   a = x Wg^T, b = x Wu^T over one pass of x; h = act(a) b and the checkpoint of a and b leave
//   kGemmDact   dh = dy Wd; with a and b from the checkpoint da = dh b act'(a) and db = dh act(a) leave (and h again)
//   kGemmPlain  up to four products of one launch, e.g. dx = da Wg + db Wu, dWg = da^T x, dWu = db^T x, dWd = dy^T h
//
// One persistent CTA per SM: warps 0 and 2 drive TMA, one thread of warp 1 issues tcgen05.mma, warps 4-11 are two epilogue
// warpgroups. A unit is an output tile of 128 rows x up to 256 columns over a range of 64-deep steps. A and B tiles
// are 64 elements (128 bytes, swizzled) x rows whichever way the matrix lies in memory: where the inner index runs
// along memory the tile is a K-major operand, otherwise an MN-major one, so no product needs a transposed copy.
// Accumulators are two sets of 256 tensor-memory columns: the epilogue of a unit runs under the products of the next.
//
// Large products are made by pairs of CTAs (cta_group::2) on tiles of 256 rows x 256 columns: each CTA loads its 128 rows
// of A and half of B. What bounds one CTA's 128 x 256 tile is its shared memory's port (128 bytes a clock): a 64-deep
// step takes 512 clocks of MMAs, but its 48 KB are written once and read once, 768 clocks. A pair's CTA moves 32 KB. Measured
// on 26253 x 768 x 2048 (one training step; boards differ by 5 %): gate 126-130 us (1.27-1.31 PFLOP/s), y 63-64 (1.29-1.31),
// activation's backward 93-96 (0.86-0.89, 440 MB), dx and the weight gradients, five products, 267-279 (1.48-1.55).
#pragma once

#include <cuda_fp16.h>

#include "ptx.cuh"

namespace nb {

constexpr int kGemmRows = 128, kGemmDepth = 64, kGemmMaxCols = 256;
constexpr int kGemmBytesA = kGemmRows * kGemmDepth * 2, kGemmBytesB = kGemmMaxCols * kGemmDepth * 2;
constexpr int kGroup = 32;  // features of a token that share a scale in the checkpoint

enum GemmKind { kGemmGate = 0, kGemmDact = 1, kGemmPlain = 2 };

// A warp's 32 rows x 32 features of a and b in the checkpoint: [a, b][chunk of 16 bytes][row], then a word of both scales
// (bf16) per row. Contiguous, so a bulk copy moves it.
template <int kBits>
struct CodeBlock {
  static constexpr int kWords = kGroup * kBits / 32;  // of a lane's 32 values
  static constexpr int kChunks = kWords / 4;          // of 16 bytes
  static constexpr int kScales = 2 * kChunks * 512;   // where they begin
  static constexpr int kBytes = kBits ? kScales + 128 : 0;
};

// Shared memory: stages, then a part for every epilogue warp (boxes for TMA's stores, code blocks), then barriers.
constexpr int kEpilogueWarps = 8, kGemmThreads = 128 + 32 * kEpilogueWarps;
template <int kKind, int kBits, int kCtas>
struct GemmLayout {
  static constexpr int kStageBytes = kGemmBytesA + kGemmBytesB / kCtas;
  static constexpr int kBoxes = kKind == kGemmPlain ? 4096 : kKind == kGemmGate ? 2048 : (kBits == 8 ? 3 : 2) * 2048;
  static constexpr int kSlots = kKind == kGemmDact && kBits == 8 ? 2 : 1;  // code blocks under way
  static constexpr int kWarpBytes = (kBoxes + kSlots * CodeBlock<kBits>::kBytes + 1023) / 1024 * 1024;
  static constexpr int kMost = 232448 - 1024 - 512 - kEpilogueWarps * kWarpBytes;
  static constexpr int kStages = kMost / kStageBytes < 6 ? kMost / kStageBytes : 6;
  static constexpr int kWarps = kStages * kStageBytes;
  static constexpr int kBars = kWarps + kEpilogueWarps * kWarpBytes;
  static constexpr int kBytes = kBars + 512 + 1024;  // (+ 1024: the base is aligned by hand)
};

struct GemmProblem {
  CUtensorMap a[2], b[2], c;  // a, b: of the two ranges of steps (gate: b of Wg and Wu)
  const __nv_bfloat16* bias;  // per column, or NULL
  float* partial;             // [split][row tile][column tile][columns / 4][128 rows][4], where splits > 1
  int32_t m, n;               // rows and columns of the output
  int32_t row_tiles, col_tiles, cols;  // tiles of 128 rows per CTA of the team; cols: of a tile
  uint32_t by_col_tiles, by_shift;     // u / col_tiles = u * by_col_tiles >> by_shift for u < 2^31
  int32_t steps0, steps;      // 64-deep steps of the first range, of both
  int32_t splits, split_steps;
  int32_t a_mn, b_mn;         // the operand's inner index does not run along memory
};

// The units of a launch, dealt to the teams (CTAs or pairs) in a fixed manner: `n_long` units (the problems with more
// steps come first in the list) in turns; the teams left with one long unit fewer then take `extra` short ones each, and
// the rest of the short units goes round again.
struct GemmDeal {
  int32_t n_long, n_short, extra;
};
template <int kCtas>
struct GemmTurns {
  int team, teams, n_long, n_short, mine, extra, rest;  // long units of this team; where its other short units begin
  __device__ __forceinline__ explicit GemmTurns(const GemmDeal& d) {
    teams = int(gridDim.x) / kCtas, team = int(blockIdx.x) / kCtas;
    n_long = d.n_long, n_short = d.n_short;
    mine = extra = 0, rest = team;
    if (n_long > 0) {
      const int rem = n_long % teams;
      mine = n_long / teams + (team < rem);
      if (team >= rem) extra = d.extra;
      rest = (teams - rem) * d.extra + team;
      first_extra = n_long + (team - rem) * d.extra;
    }
  }
  __device__ __forceinline__ int unit(int i) const {  // the i-th of this team; -1: no more
    if (i < mine) return team + i * teams;
    i -= mine;
    if (i < extra) return first_extra + i;
    const int at = rest + (i - extra) * teams;
    return at < n_short ? n_long + at : -1;
  }
  int first_extra = 0;
};

template <int kProblems>
struct GemmParams {
  GemmProblem p[kProblems];
  GemmDeal deal;
  // the gate's and its backward's
  CUtensorMap map_db, map_h;   // backward (p[0].c is that of da, forward of h)
  const __nv_bfloat16* bias_up;
  uint8_t* codes;     // checkpoint: [row tile][group][warp] code blocks
  float* col_sums;    // backward, or NULL: [row tile][warp][2 x hidden] sums of da and db over 32 rows
  int32_t groups, hidden;
};

// A second parameter, so that the parameters' size leaves a remainder of 24 by 64 (tensor maps make GemmParams a multiple of
// 64): the host needs 0.3 us more to launch a kernel with another remainder than 24 or 32.
struct GemmTail {
  int32_t* status;
  int32_t pad[4];
};
static_assert(sizeof(GemmTail) == 24, "the remainder that is cheap to launch");

struct GemmUnit {
  int problem, row, col, begin, end, split;
};
template <int kProblems>
__device__ __forceinline__ GemmUnit gemm_unit(const GemmParams<kProblems>& g, int u) {
  GemmUnit r;
  int i = 0;
  if constexpr (kProblems > 1) {
#pragma unroll 1
    for (; i < kProblems - 1; ++i) {
      const int n = g.p[i].row_tiles * g.p[i].col_tiles * g.p[i].splits;
      if (u < n) break;
      u -= n;
    }
  }
  const GemmProblem& p = g.p[i];
  r.problem = i;
  r.split = 0;
  if (p.splits > 1) {
    const int tiles = p.row_tiles * p.col_tiles;
    r.split = u / tiles;
    u -= r.split * tiles;
  }
  r.row = int(uint64_t(uint32_t(u)) * p.by_col_tiles >> p.by_shift);
  r.col = u - r.row * p.col_tiles;
  r.begin = r.split * p.split_steps;
  r.end = min(r.begin + p.split_steps, p.steps);
  return r;
}

// ---- activations ---------------------------------------------------------------------------
constexpr int kActSilu = 0, kActGelu = 1;

// gate(a) and, for the backward, its slope.
//   silu: a s with s = 1 / (1 + e^-a); slope s (1 + a (1 - s)).
//   gelu: a Phi(a); slope Phi + a phi. Phi by Abramowitz and Stegun 7.1.26: with z = |a| / sqrt 2, t = 1 / (1 + 0.3275911 z),
//   erfc(z) = t (a1 + t (a2 + t (a3 + t (a4 + t a5)))) e^-z^2, off by at most 1.5e-7; its exponential is phi's as well.
// Both take one exponential and one reciprocal. A large negative a must give 0 and not 0 x inf: e^-a overflows to inf,
// whose reciprocal is 0. The epilogues are bound by their instructions, so two values go through one packed instruction.
__device__ __forceinline__ float fast_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
__device__ __forceinline__ void split(float2 v, float& x, float& y) { x = v.x, y = v.y; }
__device__ __forceinline__ float2 exp2_of(float2 v) {
  float x, y;
  split(v, x, y);
  return make_float2(fast_exp2(x), fast_exp2(y));
}
__device__ __forceinline__ float2 rcp_of(float2 v) {
  float x, y;
  split(v, x, y);
  return make_float2(fast_rcp(x), fast_rcp(y));
}
// 1 / (1 + e^-a), or Phi(a) with e = e^(-a^2 / 2).
__device__ __forceinline__ float2 sigmoid_of(float2 a) {
  return rcp_of(__fadd2_rn(exp2_of(__fmul2_rn(a, both(-1.4426950408889634f))), both(1.f)));
}
__device__ __forceinline__ float2 phi_of(float2 a, float2& e) {
  const float2 mag = make_float2(fabsf(a.x), fabsf(a.y));
  const float2 t = rcp_of(__ffma2_rn(mag, both(0.3275911f * 0.70710678118654752f), both(1.f)));
  e = exp2_of(__fmul2_rn(__fmul2_rn(a, both(-0.72134752044448170f)), a));
  float2 q = __ffma2_rn(t, both(1.061405429f), both(-1.453152027f));
  q = __ffma2_rn(t, q, both(1.421413741f));
  q = __ffma2_rn(t, q, both(-0.284496736f));
  q = __ffma2_rn(t, q, both(0.254829592f));
  q = __fmul2_rn(__fmul2_rn(t, both(0.5f)), __fmul2_rn(q, e));  // Phi(-|a|)
  float x, y, qx, qy;
  split(a, x, y);
  split(q, qx, qy);
  return make_float2(x < 0.f ? qx : 1.f - qx, y < 0.f ? qy : 1.f - qy);
}
template <int kAct>
__device__ __forceinline__ float2 gate_of(float2 a) {
  float2 e;
  if constexpr (kAct == kActSilu) return __fmul2_rn(a, sigmoid_of(a));
  else return __fmul2_rn(a, phi_of(a, e));
}
template <int kAct>
__device__ __forceinline__ void gate_and_slope(float2 a, float2& gate, float2& slope) {
  if constexpr (kAct == kActSilu) {
    const float2 s = sigmoid_of(a);
    gate = __fmul2_rn(a, s);
    slope = __ffma2_rn(gate, __ffma2_rn(s, both(-1.f), both(1.f)), s);
  } else {
    float2 e;
    const float2 phi = phi_of(a, e);
    gate = __fmul2_rn(a, phi);
    slope = __ffma2_rn(__fmul2_rn(a, both(0.39894228040143268f)), e, phi);
  }
}
template <int kAct>
__device__ __forceinline__ float gate_of(float a) {
  float x, y;
  split(gate_of<kAct>(both(a)), x, y);
  return x;
}

// ---- the checkpoint ------------------------------------------------------------------------
// 32 features of a token share a scale. 16 bits: fp16 of v / 2^k with the group's largest magnitude in [2^14, 2^15), so
// every value within 2^-29 of it keeps 11 bits (bf16 would keep 8 and cost the gradients a rounding as large as that
// of their own operands). 8 bits: round(v / s), s = max |v| / 127 rounded up to bf16. A group with a value that is not
// finite is NaN as a whole in 8 bits; in 16 bits its scale is 1.
// (four chains of maxima)
__device__ __forceinline__ float abs_max32(const float (&v)[32]) {
  float m[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) m[i] = max3_nan(fabsf(v[i]), fabsf(v[i + 4]), fabsf(v[i + 8]));
#pragma unroll
  for (int j = 12; j < 28; j += 8)
#pragma unroll
    for (int i = 0; i < 4; ++i) m[i] = max3_nan(m[i], fabsf(v[j + i]), fabsf(v[j + 4 + i]));
#pragma unroll
  for (int i = 0; i < 4; ++i) m[i] = max3_nan(m[i], fabsf(v[28 + i]), 0.f);
  return max3_nan(max3_nan(m[0], m[1], m[2]), m[3], 0.f);
}

// Returns the scale as the upper half of its fp32 bits.
template <int kBits>
__device__ __forceinline__ uint32_t encode(const float (&v)[32], uint32_t (&w)[CodeBlock<kBits>::kWords]) {
  const float m = abs_max32(v);
  if constexpr (kBits == 16) {
    uint32_t e = __float_as_uint(m) >> 23;
    e = e == 255u ? 141u : max(e, 15u);
    const float2 inv = both(__uint_as_float((268u - e) << 23));
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float x, y;
      split(__fmul2_rn(make_float2(v[2 * i], v[2 * i + 1]), inv), x, y);
      const __half2 h = __floats2half2_rn(x, y);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return (e - 14u) << 7;
  } else {
    uint32_t s = (__float_as_uint(__fdiv_rn(m, 127.f)) + 0xFFFFu) >> 16;
    float inv = __fdividef(1.f, __uint_as_float(s << 16));
    if (!(m < __uint_as_float(0x7F800000u))) s = 0x7FC0u, inv = 0.f;   // (also NaN)
    else if (s < 0x0D80u) s = 0u, inv = 0.f;                            // below 2^-100: zeros
    // Adding 1.5 * 2^23 + 128 rounds to a whole number, whose low byte is kept: the code + 128.
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t b[4];
#pragma unroll
      for (int k = 0; k < 4; k += 2) {
        float x, y;
        split(__ffma2_rn(make_float2(v[4 * i + k], v[4 * i + k + 1]), both(inv), both(12583040.f)), x, y);
        b[k] = __float_as_uint(x), b[k + 1] = __float_as_uint(y);
      }
      w[i] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    }
    return s;
  }
}

// Values 2 i and 2 i + 1 of a lane's (i known at compile time).
template <int kBits, int kWords>
__device__ __forceinline__ float2 decode(const uint32_t (&w)[kWords], int i, float2 scale) {
  if constexpr (kBits == 16) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    return __fmul2_rn(make_float2(f.x, f.y), scale);
  } else {
    // Put into the low byte of 2^23: 2^23 + 128 + code.
    const uint32_t u = w[i >> 1];
    const float x = __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7440 | (2 * (i & 1)))),
                y = __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7440 | (2 * (i & 1) + 1)));
    return __fmul2_rn(__fadd2_rn(make_float2(x, y), both(-8388736.f)), scale);
  }
}

// Sum of each of 16 values over the warp's lanes; lane l receives that of value l % 16.
__device__ __forceinline__ float column_sums(float (&v)[16], int lane) {
#pragma unroll
  for (int off = 8; off > 0; off >>= 1) {
    const bool up = (lane & off) != 0;
#pragma unroll
    for (int i = 0; i < off; ++i) {
      const float keep = up ? v[i + off] : v[i], send = up ? v[i] : v[i + off];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, send, off);
    }
  }
  return v[0] + __shfl_xor_sync(0xffffffffu, v[0], 16);
}

__device__ __forceinline__ void add_bias32(float (&v)[32], const __nv_bfloat16* bias, int col, int n) {
  if (bias == nullptr) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (col + 8 * i >= n) break;  // (n is a multiple of 8)
    const uint4 b = *reinterpret_cast<const uint4*>(bias + col + 8 * i);
    const uint32_t u[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[8 * i + 2 * k] += __uint_as_float(u[k] << 16);
      v[8 * i + 2 * k + 1] += __uint_as_float(u[k] & 0xFFFF0000u);
    }
  }
}

// The wait for a load from tensor memory, as something that its registers depend on: nothing computed from them may be
// moved in front of it.
__device__ __forceinline__ void tmem_wait_ld32(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                 "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]),
                 "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]),
                 "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28])
               :
               : "memory");
  asm volatile("" : "+r"(r[29]), "+r"(r[30]), "+r"(r[31]) : : "memory");
}
__device__ __forceinline__ void tmem_ld32f(uint32_t taddr, float (&v)[32]) {
  uint32_t r[32];
  tmem_ld32(taddr, r);
  tmem_wait_ld32(r);
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

// 32 values of a row of a box that TMA stores, 64 columns wide (`half` of it): the chunks of 16 bytes where its swizzle
// expects them.
__device__ __forceinline__ void stage_half_row(uint32_t box, int row, int half, const float (&v)[32]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    st_shared_v4(box + swz128(row, half * 4 + i), pack_bf16(v[8 * i], v[8 * i + 1]), pack_bf16(v[8 * i + 2], v[8 * i + 3]),
                 pack_bf16(v[8 * i + 4], v[8 * i + 5]), pack_bf16(v[8 * i + 6], v[8 * i + 7]));
}
// 16 values (`half` of 32) of a row of a box that TMA stores, 32 columns wide, where its swizzle expects them.
__device__ __forceinline__ void stage_half16(uint32_t box, int row, int half, const uint32_t (&w)[8]) {
#pragma unroll
  for (int i = 0; i < 2; ++i)
    st_shared_v4(box + row * 64 + (((2 * half + i) ^ ((row >> 1) & 3)) << 4), w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
}
__device__ __forceinline__ uint4 ld_shared_v4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}

// ---- the kernel ----------------------------------------------------------------------------
template <int kCtas, int kKind, int kAct, int kBits, int kProblems>
__global__ void __launch_bounds__(kGemmThreads, 1) gemm_kernel(const __grid_constant__ GemmParams<kProblems> g,
                                                                const __grid_constant__ GemmTail tail) {
  using L = GemmLayout<kKind, kBits, kCtas>;
  constexpr int kStages = L::kStages;
  constexpr bool kPair = kCtas == 2;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t bars = base + L::kBars;
  const uint32_t full = bars, empty = bars + 8 * kStages, acc_full = bars + 16 * kStages, acc_empty = acc_full + 16,
                 codes_full = acc_empty + 16, tmem_slot = codes_full + 16 * kEpilogueWarps, abort_at = tmem_slot + 4;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem_raw + (abort_at - smem_u32(smem_raw)));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = kPair ? int(cluster_rank()) : 0;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(full + 8 * i, 1), mbar_init(empty + 8 * i, 1);
    for (int i = 0; i < 2; ++i) mbar_init(acc_full + 8 * i, 1), mbar_init(acc_empty + 8 * i, kEpilogueWarps * kCtas);
    if constexpr (kKind == kGemmDact)
      for (int i = 0; i < 2 * kEpilogueWarps; ++i) mbar_init(codes_full + 8 * i, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  pdl_wait();
  if (warp == 1) {
    if constexpr (kPair) tmem_alloc_pair(tmem_slot, 512), tmem_relinquish_pair();
    else tmem_alloc(tmem_slot, 512), tmem_relinquish();
    tc_fence_before();
  }
  __syncwarp();
  if constexpr (kPair) cluster_sync();  // the other CTA's barriers are there
  else __syncthreads();
  tc_fence_after();
  pdl_launch_dependents();  // behind the allocation: the next kernel's blocks may ask for columns too
  uint32_t tmem;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(tmem_slot));

  const GemmTurns<kCtas> turns(g.deal);
  if (warp == 0 || warp == 2) {
    // One thread loads A's tiles, another one B's, both elected: issuing a step's four loads of MN-major blocks took a single
    // thread, chosen by its lane, nearly the 512 clocks of the step's MMAs (dx and the weight gradients of 26253 x 768 x 2048:
    // 300 us; two threads chosen by their lanes 316, as they look at what their waits return; two elected ones 267).
    if (elect_one()) {
      const bool for_a = warp == 0;
      const auto load = [&](uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
        if constexpr (kPair) tma_load_2d_pair(dst, map, bar, c0, c1);
        else tma_load_2d(dst, map, bar, c0, c1);
      };
      int stage = 0;
      uint32_t phase = 0;
      // It ends where one of its waits gave up: more arrivals than a phase expects, while bytes are due, are not defined.
      bool live = true;
      for (int i = 0; live; ++i) {
        const int id = turns.unit(i);
        if (id < 0) break;
        const GemmUnit u = gemm_unit(g, id);
        const GemmProblem& p = g.p[u.problem];
        const int cols = p.cols, mine = cols / kCtas;  // columns of the tile, and those that this CTA loads
        const int row0 = (u.row * kCtas + rank) * kGemmRows, steps0 = p.steps0;
        // Blocks of 64 columns of an MN-major tile (a pair's 96 take two), 0: a K-major one.
        const int a_blocks = p.a_mn ? 2 : 0, b_blocks = p.b_mn ? (mine + 63) / 64 : 0;
        const uint32_t bytes = kCtas * (kGemmBytesA + uint32_t(b_blocks ? b_blocks * 64 : mine) * (kGemmDepth * 2));
        // The gate's tile has columns of a, then as many of b: in a pair rank 0 holds those of a and rank 1 those of b.
        const int half = cols / 2, col0 = kKind == kGemmGate ? u.col * half : u.col * cols + rank * mine;
        const CUtensorMap* map = for_a ? &p.a[0] : &p.b[kKind == kGemmGate && kPair ? rank : 0];
        const int blocks = for_a ? a_blocks : b_blocks, first = for_a ? row0 : col0;
        for (int s = u.begin; s < u.end; ++s) {
          live = mbar_wait(empty + 8 * stage, phase ^ 1, abort_flag);
          if (!live) break;
          const uint32_t at = base + stage * L::kStageBytes + (for_a ? 0 : kGemmBytesA);
          uint32_t bar = full + 8 * stage;
          if (for_a && rank == 0) mbar_arrive_expect_tx(bar, bytes);  // (all loads of both CTAs count on rank 0's barrier)
          if constexpr (kPair) bar = map_to_rank(bar, 0);
          const int second = kKind == kGemmPlain && s >= steps0;
          const int k = (second ? s - steps0 : s) * kGemmDepth;
          if (blocks) {
            for (int b = 0; b < blocks; ++b) load(at + b * 8192, map + second, bar, first + b * 64, k);
          } else {
            load(at, map + second, bar, k, first);
            if constexpr (kKind == kGemmGate && !kPair)
              if (!for_a) load(at + half * 128, map + 1, bar, k, first);
          }
          if (++stage == kStages) stage = 0, phase ^= 1;
        }
      }
      // The MMAs' arrivals on this CTA's barriers (rank 0's in a pair) are in before it may end.
      for (int s = 0; s < kStages && live; ++s) {
        live = mbar_wait(empty + 8 * stage, phase ^ 1, abort_flag);
        if (++stage == kStages) stage = 0, phase ^= 1;
      }
    }
  } else if (warp == 1) {
    if (rank == 0 && elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      // (No look at what the waits return: a test between wait and MMAs made the products 30 % slower, and behind a wait that
      // gave up these MMAs and arrivals, each a whole phase of its barrier, do no harm.)
      for (int i = 0;; ++i) {
        const int id = turns.unit(i);
        if (id < 0) break;
        const GemmUnit u = gemm_unit(g, id);
        const GemmProblem& p = g.p[u.problem];
        const uint32_t idesc = make_idesc(kGemmRows * kCtas, p.cols, p.a_mn, p.b_mn);
        const uint64_t step_a = p.a_mn ? 2048 >> 4 : 32 >> 4, step_b = p.b_mn ? 2048 >> 4 : 32 >> 4;
        const uint32_t acc = tmem + (i & 1) * kGemmMaxCols;
        mbar_wait(acc_empty + 8 * (i & 1), ((i >> 1) & 1) ^ 1, abort_flag);
        tc_fence_after();
        for (int s = u.begin; s < u.end; ++s) {
          mbar_wait(full + 8 * stage, phase, abort_flag);
          tc_fence_after();
          const uint32_t at_a = base + stage * L::kStageBytes;
          uint64_t da = make_sdesc(at_a, 8192, 1024), db = make_sdesc(at_a + kGemmBytesA, 8192, 1024);
#pragma unroll
          for (int k = 0; k < kGemmDepth / 16; ++k) {
            if constexpr (kPair) mma_ss_pair(acc, da, db, idesc, s > u.begin || k > 0);
            else mma_ss(acc, da, db, idesc, s > u.begin || k > 0);
            da += step_a, db += step_b;
          }
          if constexpr (kPair) tc_commit_pair(empty + 8 * stage);
          else tc_commit(empty + 8 * stage);
          if (++stage == kStages) stage = 0, phase ^= 1;
        }
        if constexpr (kPair) tc_commit_pair(acc_full + 8 * (i & 1));
        else tc_commit(acc_full + 8 * (i & 1));
      }
    }
  } else if (warp >= 4) {
    // A warp works by itself on its 32 rows (its lane is the row) and on every other 32 (plain: 64) columns, hands boxes of 32
    // rows to TMA and waits for no other warp. (Four warps that met at two barriers per box spent 17 % of their time there.)
    // Twelve warps that store whole sectors from their registers instead save 5 of 125 us in the gate with 16 bits and no
    // biases (26253 x 768 x 2048), but what else uses the load and store unit queues behind such stores: with biases
    // the gate took 130 instead of 108 us in 8 bits, the activation's backward with its column sums 155 instead of 118.
    const int wg = (warp >> 2) - 1, quarter = warp & 3;
    [[maybe_unused]] const uint32_t own = base + L::kWarps + (warp - 4) * L::kWarpBytes;
    const uint32_t lanes = uint32_t(quarter) << 21;
    const uint32_t acc_free = kPair ? map_to_rank(acc_empty, 0) : acc_empty;  // where the MMAs' issuer waits
    constexpr int kB = kBits ? kBits : 16;
    using Block = CodeBlock<kB>;
    const auto rows_of = [&](const GemmUnit& u) { return (u.row * kCtas + rank) * kGemmRows; };
    const auto code_block = [&](const GemmUnit& u, int f) {
      return g.codes + ((int64_t(u.row * kCtas + rank) * g.groups + f / kGroup) * 4 + quarter) * Block::kBytes;
    };

    // The backward's code blocks are requested as soon as there is room.
    [[maybe_unused]] struct { int i, blk; GemmUnit u; bool live; } ahead{-1, 0, {}, true};
    [[maybe_unused]] uint32_t piece = 0;
    [[maybe_unused]] const uint32_t my_codes = codes_full + 16 * (warp - 4);
    [[maybe_unused]] const auto request = [&](uint32_t slot) {  // the next piece's
      if constexpr (kKind == kGemmDact) {
        const int cols = g.p[0].cols;
        ahead.blk += 64;
        while (ahead.live && (ahead.i < 0 || ahead.blk >= cols || ahead.u.col * cols + ahead.blk >= g.hidden ||
                              (kPair && rows_of(ahead.u) >= g.p[0].m))) {
          const int id = turns.unit(++ahead.i);
          ahead.live = id >= 0;
          if (ahead.live) ahead.u = gemm_unit(g, id);
          ahead.blk = wg * 32;
        }
        if (ahead.live && lane == 0) {
          mbar_arrive_expect_tx(my_codes + 8 * slot, Block::kBytes);
          bulk_load(own + L::kBoxes + slot * Block::kBytes, code_block(ahead.u, ahead.u.col * cols + ahead.blk), Block::kBytes,
                    my_codes + 8 * slot);
        }
      }
    };
    if constexpr (kKind == kGemmDact)
      for (int i = 0; i < L::kSlots; ++i) request(i);

    [[maybe_unused]] bool live = true;
    for (int i = 0; live; ++i) {
      const int id = turns.unit(i);
      if (id < 0) break;
      const GemmUnit u = gemm_unit(g, id);
      const GemmProblem& p = g.p[u.problem];
      const uint32_t acc = tmem + lanes + (i & 1) * kGemmMaxCols;
      if (!__all_sync(0xffffffffu, mbar_wait(acc_full + 8 * (i & 1), (i >> 1) & 1, abort_flag))) break;
      tc_fence_after();
      const int row0 = rows_of(u), row = row0 + quarter * 32;  // of the tile, of the warp
      if (kPair && row0 >= p.m) {
        // the pair's second half lies behind the last row
      } else if constexpr (kKind == kGemmGate) {
        const int half = p.cols / 2;
#pragma unroll 1
        for (int blk = wg * 32; blk < half; blk += 64) {
          const int f = u.col * half + blk;
          if (f >= g.hidden) break;
          [[maybe_unused]] const uint32_t block = own + L::kBoxes;
          float a[32], b[32];
          [[maybe_unused]] uint32_t w[Block::kWords], scales = 0;
          tmem_ld32f(acc + blk, a);
          add_bias32(a, p.bias, f, g.hidden);
          if (lane == 0) bulk_wait_group_read0();  // the boxes in front have left
          __syncwarp();
          if constexpr (kBits > 0) {
            scales = encode<kB>(a, w);
#pragma unroll
            for (int c = 0; c < Block::kChunks; ++c)
              st_shared_v4(block + c * 512 + lane * 16, w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
          }
#pragma unroll
          for (int k = 0; k < 32; k += 2) split(gate_of<kAct>(make_float2(a[k], a[k + 1])), a[k], a[k + 1]);
          tmem_ld32f(acc + half + blk, b);
          add_bias32(b, g.bias_up, f, g.hidden);
          if constexpr (kBits > 0) {
            scales |= encode<kB>(b, w) << 16;
#pragma unroll
            for (int c = 0; c < Block::kChunks; ++c)
              st_shared_v4(block + (Block::kChunks + c) * 512 + lane * 16, w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
            asm volatile("st.shared.b32 [%0], %1;" ::"r"(block + Block::kScales + lane * 4), "r"(scales) : "memory");
          }
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            uint32_t v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k)
              v[k] = pack_bf16(a[16 * q + 2 * k] * b[16 * q + 2 * k], a[16 * q + 2 * k + 1] * b[16 * q + 2 * k + 1]);
            stage_half16(own, lane, q, v);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&p.c, own, f, row);
            if constexpr (kBits > 0) bulk_store(code_block(u, f), block, Block::kBytes);
            bulk_commit_group();
          }
        }
      } else if constexpr (kKind == kGemmDact) {
#pragma unroll 1
        for (int blk = wg * 32; blk < p.cols; blk += 64) {
          const int f = u.col * p.cols + blk;
          if (f >= g.hidden) break;
          const uint32_t slot = piece % L::kSlots, codes = own + L::kBoxes + slot * Block::kBytes;
          live = __all_sync(0xffffffffu, mbar_wait(my_codes + 8 * slot, (piece / L::kSlots) & 1, abort_flag));
          if (!live) break;
          uint32_t scales;
          asm volatile("ld.shared.b32 %0, [%1];" : "=r"(scales) : "r"(codes + Block::kScales + lane * 4) : "memory");
          const float2 sa = both(__uint_as_float(scales << 16)), sb = both(__uint_as_float(scales & 0xFFFF0000u));
          uint32_t wa[Block::kWords], wb[Block::kWords], r[32];
          tmem_ld32(acc + blk, r);
#pragma unroll
          for (int c = 0; c < Block::kChunks; ++c) {
            const uint4 x = ld_shared_v4(codes + c * 512 + lane * 16),
                        y = ld_shared_v4(codes + (Block::kChunks + c) * 512 + lane * 16);
            wa[4 * c] = x.x, wa[4 * c + 1] = x.y, wa[4 * c + 2] = x.z, wa[4 * c + 3] = x.w;
            wb[4 * c] = y.x, wb[4 * c + 1] = y.y, wb[4 * c + 2] = y.z, wb[4 * c + 3] = y.w;
          }
          // The block has been read, by every lane, before the copy that refills it may write: without the fence nothing orders
          // these loads in front of the async proxy's writes, and one in some 25000 calls found the next block's values.
          fence_proxy_async_smem();
          __syncwarp();
          request(slot);
          tmem_wait_ld32(r);
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            float d[16], e[16];
            uint32_t vd[8], ve[8], vh[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const float2 a = decode<kB>(wa, 8 * q + k, sa), b = decode<kB>(wb, 8 * q + k, sb),
                           dh = make_float2(__uint_as_float(r[16 * q + 2 * k]), __uint_as_float(r[16 * q + 2 * k + 1]));
              float2 gate, slope;
              gate_and_slope<kAct>(a, gate, slope);
              split(__fmul2_rn(dh, gate), e[2 * k], e[2 * k + 1]);
              split(__fmul2_rn(__fmul2_rn(dh, b), slope), d[2 * k], d[2 * k + 1]);
              vd[k] = pack_bf16(d[2 * k], d[2 * k + 1]);
              ve[k] = pack_bf16(e[2 * k], e[2 * k + 1]);
              if constexpr (kBits == 8) {
                float x, y;
                split(__fmul2_rn(gate, b), x, y);
                vh[k] = pack_bf16(x, y);
              }
            }
            if (q == 0) {
              if (lane == 0) bulk_wait_group_read0();  // the boxes in front have left
              __syncwarp();
            }
            stage_half16(own, lane, q, vd);
            stage_half16(own + 2048, lane, q, ve);
            if constexpr (kBits == 8) stage_half16(own + 4096, lane, q, vh);
            if (q == 1) {
              fence_proxy_async_smem();
              __syncwarp();
              if (lane == 0) {
                tma_store_2d(&p.c, own, f, row);
                tma_store_2d(&g.map_db, own + 2048, f, row);
                if constexpr (kBits == 8) tma_store_2d(&g.map_h, own + 4096, f, row);
                bulk_commit_group();
              }
            }
            if (g.col_sums != nullptr) {
              const int fq = f + 16 * q;
              float* sums = g.col_sums + (int64_t(row0 / kGemmRows) * 4 + quarter) * (2 * int64_t(g.hidden));
              const float sd = column_sums(d, lane), se = column_sums(e, lane);
              const int at = fq + (lane & 15);
              if (at < g.hidden) sums[(lane < 16 ? 0 : g.hidden) + at] = lane < 16 ? sd : se;
            }
          }
          ++piece;
        }
      } else {
        const int c0 = u.col * p.cols;
        if (p.splits > 1) {
          float4* out = reinterpret_cast<float4*>(p.partial) +
                        ((int64_t(u.split) * p.row_tiles * kCtas + row0 / kGemmRows) * p.col_tiles + u.col) *
                            (int64_t(p.cols) / 4 * kGemmRows) + quarter * 32 + lane;
#pragma unroll 1
          for (int blk = wg * 32; blk < p.cols; blk += 64) {
            float v[32];
            tmem_ld32f(acc + blk, v);
#pragma unroll
            for (int k = 0; k < 8; ++k)
              out[(blk / 4 + k) * kGemmRows] = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
          }
        } else {
#pragma unroll 1
          for (int blk = wg * 64; blk < p.cols; blk += 128) {
            if (c0 + blk >= p.n) break;
            if (lane == 0) bulk_wait_group_read0();
            __syncwarp();
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              float v[32];
              tmem_ld32f(acc + blk + q * 32, v);
              add_bias32(v, p.bias, c0 + blk + q * 32, p.n);
              stage_half_row(own, lane, q, v);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) tma_store_2d(&p.c, own, c0 + blk, row), bulk_commit_group();
          }
        }
      }
      if (!live) break;
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (kPair) mbar_arrive_cluster(acc_free + 8 * (i & 1));
        else mbar_arrive(acc_free + 8 * (i & 1));
      }
    }
    if (lane == 0) bulk_wait_group<0>();
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0) report_abort(abort_flag, tail.status);
  __syncwarp();
  if constexpr (kPair) cluster_sync();  // nothing of this CTA is used by the other one any more
  if (warp == 1) {
    tc_fence_after();
    if constexpr (kPair) tmem_dealloc_pair(tmem, 512);
    else tmem_dealloc(tmem, 512);
  }
  // Neither SM of a pair takes a block of the next kernel, which may want tensor memory for itself, before both CTAs have
  // given theirs back.
  __syncwarp();
  if constexpr (kPair) cluster_sync();
}

}  // namespace nb
