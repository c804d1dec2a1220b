// Norms of queries and keys per head with the rotation by position in the same pass (include/nb_block.h).
//
// With r = (mean x^2 + eps)^-1/2 and n = x r w the result is y = R(theta) n, where R turns each of the head's 32 pairs
// by the angle theta_i = sum_a position_a freq_ai of its token. Backward: dn = R(-theta) dy, dw = sum dn x r and, with
// g = dn w, dx = r (g - x r^2 mean(g x)); r is computed again from x, which is read anyway.
//
// Bound by memory traffic: 2 bytes per value read and written once (forward), three tensors read or written in the
// backward. A warp takes a token with all its heads, so that the token's 32 angles are computed once, one per lane,
// and handed around by shuffles. Four lanes share a row of 64 values: lane j of them holds values [8j, 8j+8) and
// [32+8j, 32+8j+8), which contain both partners of every pair in either order of pairs, so the rotation needs no
// exchange and every access is 16 bytes. A lane keeps its eight pairs as first and second partners, two pairs to a
// packed instruction: with one value per instruction the kernels took 35 (forward) and 72 us (backward) on 26253 tokens of
// 12 + 12 heads, bound by their instructions; now 33 and 54 (161 and 242 MB: 4.9 and 4.5 TB/s). Sums are in fp32; the one
// rounding is that of the result to bf16. Angles are products and sums in 64 bits, and whole turns are taken off there: position 2^20 at
// frequency 1 would keep an error of 0.03 in fp32.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "../../include/nb_block.h"
#include "host.h"
#include "ptx.cuh"

namespace {

constexpr int kDim = 64, kPairs = 32;
constexpr int kWarps = 8, kThreads = kWarps * 32;
constexpr int kRowsAtOnce = 8;          // of a warp: four lanes a row
constexpr int kBwdBlocksMax = 1184;     // blocks of the backward, whose partial sums of dw the workspace holds

struct Side {
  const __nv_bfloat16* x;
  const __nv_bfloat16* dy;
  __nv_bfloat16* y;
  int64_t xs[3], ys[3], gs[3];  // batch, token, head
  const float* weight;
  const void* pos;
  int64_t ps[2];                // batch, token
  int32_t heads, tokens;
};
struct Params {
  Side s[2];
  int64_t units, units_q;       // tokens, or tokens of both sides one after the other
  int32_t shared;               // queries and keys of a token are one unit
  int32_t one_batch;
  int32_t axes, pos_type, interleaved;
  const float* freqs;
  float eps;
  float* partial;               // backward: [blocks][2][64]
};

using nb::add_f32x2;
using nb::fma_f32x2;
using nb::mul_f32x2;
using nb::pack_f32x2;
using nb::unpack_f32x2;

__device__ __forceinline__ uint64_t both(float v) { return pack_f32x2(v, v); }
__device__ __forceinline__ float sum_of(uint64_t v) {
  float x, y;
  unpack_f32x2(v, x, y);
  return x + y;
}

// The warp's number, known to be the same for its lanes: what follows from it can live in uniform registers.
__device__ __forceinline__ int warp_index() { return __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0); }

// The position coordinates of a token, as they lie in memory.
struct Position {
  int64_t at[NB_ROPE_MAX_AXES];
};
__device__ __forceinline__ void load_position(const Params& p, const Side& s, int64_t batch, int64_t token, Position& v) {
  const int64_t at = batch * s.ps[0] + token * s.ps[1];
#pragma unroll
  for (int a = 0; a < NB_ROPE_MAX_AXES; ++a) {
    if (a >= p.axes) break;
    if (p.pos_type == NB_POSITION_I64) v.at[a] = static_cast<const int64_t*>(s.pos)[at + a];
    else v.at[a] = static_cast<const int32_t*>(s.pos)[at + a];  // (or the bits of a float)
  }
}
// cos and sin of the token's angle of pair `lane`.
__device__ __forceinline__ float2 turn_of(const Params& p, const Position& v, int lane) {
  if (p.axes == 0) return make_float2(1.f, 0.f);
  double angle = 0.0;
#pragma unroll
  for (int a = 0; a < NB_ROPE_MAX_AXES; ++a) {
    if (a >= p.axes) break;
    const double pos = p.pos_type == NB_POSITION_F32 ? double(__int_as_float(int(v.at[a]))) : double(v.at[a]);
    angle = fma(pos, double(p.freqs[a * kPairs + lane]), angle);
  }
  // Whole turns off, in 64 bits; the rest in half turns, which need no reduction.
  const double turns = angle * 0.15915494309189533577;
  float sn, cs;
  sincospif(float(2.0 * (turns - rint(turns))), &sn, &cs);
  return make_float2(cs, sn);
}

// Pair e (0..7) of a lane with column block j: 8j + e, or interleaved 4j + e of the first eight values and 16 + 4j + e of
// the others.
template <bool kInter>
__device__ __forceinline__ int pair_of(int j, int e) {
  return kInter ? (e < 4 ? 4 * j + e : 16 + 4 * j + (e - 4)) : 8 * j + e;
}
// cos and sin of the lane's pairs, from the lanes that hold them.
template <bool kInter>
__device__ __forceinline__ void spread(float2 mine, int j, uint64_t (&c)[4], uint64_t (&s)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int p0 = pair_of<kInter>(j, 2 * i), p1 = pair_of<kInter>(j, 2 * i + 1);
    c[i] = pack_f32x2(__shfl_sync(0xffffffffu, mine.x, p0), __shfl_sync(0xffffffffu, mine.x, p1));
    s[i] = pack_f32x2(__shfl_sync(0xffffffffu, mine.y, p0), __shfl_sync(0xffffffffu, mine.y, p1));
  }
}

// A lane's 16 values as the first and second partners of its eight pairs.
template <bool kInter>
__device__ __forceinline__ void partners(const uint4& lo, const uint4& hi, uint64_t (&a)[4], uint64_t (&b)[4]) {
  const uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const auto low = [](uint32_t v) { return __uint_as_float(v << 16); };
    const auto high = [](uint32_t v) { return __uint_as_float(v & 0xFFFF0000u); };
    if constexpr (kInter) {
      a[i] = pack_f32x2(low(w[2 * i]), low(w[2 * i + 1]));
      b[i] = pack_f32x2(high(w[2 * i]), high(w[2 * i + 1]));
    } else {
      a[i] = pack_f32x2(low(w[i]), high(w[i]));
      b[i] = pack_f32x2(low(w[4 + i]), high(w[4 + i]));
    }
  }
}
template <bool kInter>
__device__ __forceinline__ void store16(__nv_bfloat16* p, int j, const uint64_t (&a)[4], const uint64_t (&b)[4]) {
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a0, a1, b0, b1;
    unpack_f32x2(a[i], a0, a1);
    unpack_f32x2(b[i], b0, b1);
    if constexpr (kInter) w[2 * i] = nb::pack_bf16(a0, b0), w[2 * i + 1] = nb::pack_bf16(a1, b1);
    else w[i] = nb::pack_bf16(a0, a1), w[4 + i] = nb::pack_bf16(b0, b1);
  }
  *reinterpret_cast<uint4*>(p + 8 * j) = make_uint4(w[0], w[1], w[2], w[3]);
  *reinterpret_cast<uint4*>(p + 32 + 8 * j) = make_uint4(w[4], w[5], w[6], w[7]);
}
// Where value `a` or `b` of pair e of column block j lies in the row.
template <bool kInter>
__device__ __forceinline__ int column_of(int j, int e, bool second) {
  const int pair = pair_of<kInter>(j, e);
  return kInter ? 2 * pair + second : pair + 32 * second;
}

// (a, b) turned by the angles, or back (s negated).
__device__ __forceinline__ void rotate(uint64_t (&a)[4], uint64_t (&b)[4], const uint64_t (&c)[4], const uint64_t (&s)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint64_t x = a[i], y = b[i], n = s[i] ^ 0x8000000080000000ull;
    a[i] = fma_f32x2(y, n, mul_f32x2(x, c[i]));
    b[i] = fma_f32x2(x, s[i], mul_f32x2(y, c[i]));
  }
}
__device__ __forceinline__ float sum4(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}
// (mean x^2 + eps)^-1/2 of the row.
__device__ __forceinline__ float root_of(const uint64_t (&a)[4], const uint64_t (&b)[4], float eps) {
  uint64_t ss = mul_f32x2(a[0], a[0]);
#pragma unroll
  for (int i = 1; i < 4; ++i) ss = fma_f32x2(a[i], a[i], ss);
#pragma unroll
  for (int i = 0; i < 4; ++i) ss = fma_f32x2(b[i], b[i], ss);
  return rsqrtf(sum4(sum_of(ss)) * (1.f / kDim) + eps);
}

// A warp's way through its units (tokens of one side, or of both) and their groups of eight rows. All of it is the same for
// the warp's lanes.
struct Walk {
  int64_t unit, batch, token;
  int side, r0, split, rows;  // rows from `split` on are keys
  bool live;
};
__device__ __forceinline__ void enter(const Params& p, Walk& w) {
  w.live = w.unit < p.units;
  if (!w.live) return;
  w.side = p.shared || w.unit < p.units_q ? 0 : 1;
  const uint32_t at = uint32_t(w.side ? w.unit - p.units_q : w.unit), len = uint32_t(p.s[w.side].tokens);
  const uint32_t b = p.one_batch ? 0 : at / len;
  w.batch = b, w.token = at - b * len;
  w.r0 = 0;
  w.split = w.side ? 0 : p.s[0].heads;
  w.rows = w.split + (p.shared || w.side ? p.s[1].heads : 0);
}
__device__ __forceinline__ Walk begin(const Params& p, int warp) {
  Walk w{};
  w.unit = int64_t(blockIdx.x) * kWarps + warp;
  enter(p, w);
  return w;
}
__device__ __forceinline__ void advance(const Params& p, Walk& w) {
  w.r0 += kRowsAtOnce;
  if (w.r0 < w.rows) return;
  w.unit += int64_t(gridDim.x) * kWarps;
  enter(p, w);
}
// A lane's row of the group in a tensor with these strides.
template <typename T>
__device__ __forceinline__ T* row_of(T* q, const int64_t (&sq)[3], T* k, const int64_t (&sk)[3], const Walk& w, int row) {
  return row < w.split ? q + w.batch * sq[0] + w.token * sq[1] + row * sq[2]
                       : k + w.batch * sk[0] + w.token * sk[1] + (row - w.split) * sk[2];
}

// The weights of both sides in shared memory, as the lanes hold them: [side][j][first, second][8 pairs].
template <bool kInter>
__device__ __forceinline__ void load_weights(const Params& p, float* w) {
  if (threadIdx.x < 2 * kDim) {
    const int side = threadIdx.x / kDim, j = (threadIdx.x >> 4) & 3, second = (threadIdx.x >> 3) & 1, e = threadIdx.x & 7;
    const float* src = p.s[side].weight;
    w[threadIdx.x] = src != nullptr ? src[column_of<kInter>(j, e, second)] : 1.f;
  }
  __syncthreads();
}
__device__ __forceinline__ void weights_of(const float* w, int side, int j, uint64_t (&a)[4], uint64_t (&b)[4]) {
  const float* at = w + side * kDim + j * 16;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(at + 4 * i), y = *reinterpret_cast<const ulonglong2*>(at + 8 + 4 * i);
    a[2 * i] = x.x, a[2 * i + 1] = x.y, b[2 * i] = y.x, b[2 * i + 1] = y.y;
  }
}

// ---- forward -------------------------------------------------------------------------------
// The next group's rows (and the next token's position) are under way while a group is computed.
constexpr int kFwdBlocks = 4;  // per SM

template <bool kInter>
__global__ void __launch_bounds__(kThreads, kFwdBlocks) qk_fwd_kernel(const __grid_constant__ Params p) {
  __shared__ __align__(16) float w_smem[2 * kDim];
  nb::pdl_wait();
  nb::pdl_launch_dependents();
  load_weights<kInter>(p, w_smem);
  const int lane = threadIdx.x & 31, j = lane & 3, slot = lane >> 2;
  uint4 lo = {}, hi = {};
  Position pos;
  const auto load = [&](const Walk& w) {
    const int row = w.r0 + slot;
    if (row < w.rows) {
      const __nv_bfloat16* x = row_of(p.s[0].x, p.s[0].xs, p.s[1].x, p.s[1].xs, w, row);
      lo = *reinterpret_cast<const uint4*>(x + 8 * j);
      hi = *reinterpret_cast<const uint4*>(x + 32 + 8 * j);
    }
    if (w.r0 == 0) load_position(p, p.s[w.side], w.batch, w.token, pos);
  };
  Walk w = begin(p, warp_index());
  if (w.live) load(w);
  uint64_t c[4], s[4];
  while (w.live) {
    const Walk now = w;
    uint64_t a[4], b[4], wa[4], wb[4];
    partners<kInter>(lo, hi, a, b);
    if (now.r0 == 0) spread<kInter>(turn_of(p, pos, lane), j, c, s);
    advance(p, w);
    if (w.live) load(w);
    const int row = now.r0 + slot, side = row >= now.split;
    const uint64_t r = both(root_of(a, b, p.eps));
    weights_of(w_smem, side, j, wa, wb);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      a[i] = mul_f32x2(mul_f32x2(a[i], r), wa[i]);
      b[i] = mul_f32x2(mul_f32x2(b[i], r), wb[i]);
    }
    rotate(a, b, c, s);
    if (row < now.rows) store16<kInter>(row_of(p.s[0].y, p.s[0].ys, p.s[1].y, p.s[1].ys, now, row), j, a, b);
  }
}

// ---- backward ------------------------------------------------------------------------------
constexpr int kBwdBlocks = 2;  // per SM

template <bool kInter>
__global__ void __launch_bounds__(kThreads, kBwdBlocks) qk_bwd_kernel(const __grid_constant__ Params p) {
  __shared__ __align__(16) float w_smem[2 * kDim];
  // Every lane's sums of dw of both sides. In registers they are 32 of 128, and the rest spills: 180 instead of 165 us on
  // 32 x 4096 tokens of 8 + 8 heads. (Three blocks of 80 registers spill as well: 217.)
  __shared__ __align__(16) ulonglong2 dw_smem[kWarps][2][4][32];
  const int lane = threadIdx.x & 31, warp = warp_index(), j = lane & 3, slot = lane >> 2;
#pragma unroll
  for (int i = 0; i < 4; ++i) dw_smem[warp][0][i][lane] = dw_smem[warp][1][i][lane] = make_ulonglong2(0, 0);
  nb::pdl_wait();
  nb::pdl_launch_dependents();
  load_weights<kInter>(p, w_smem);
  uint4 lo = {}, hi = {}, glo = {}, ghi = {};
  Position pos;
  const auto load = [&](const Walk& w) {
    const int row = w.r0 + slot;
    if (row < w.rows) {
      const __nv_bfloat16* x = row_of(p.s[0].x, p.s[0].xs, p.s[1].x, p.s[1].xs, w, row);
      const __nv_bfloat16* g = row_of(p.s[0].dy, p.s[0].gs, p.s[1].dy, p.s[1].gs, w, row);
      lo = *reinterpret_cast<const uint4*>(x + 8 * j);
      hi = *reinterpret_cast<const uint4*>(x + 32 + 8 * j);
      glo = *reinterpret_cast<const uint4*>(g + 8 * j);
      ghi = *reinterpret_cast<const uint4*>(g + 32 + 8 * j);
    }
    if (w.r0 == 0) load_position(p, p.s[w.side], w.batch, w.token, pos);
  };
  Walk w = begin(p, warp);
  if (w.live) load(w);
  uint64_t c[4], s[4];
  while (w.live) {
    const Walk now = w;
    uint64_t a[4], b[4], ga[4], gb[4], wa[4], wb[4];
    partners<kInter>(lo, hi, a, b);
    partners<kInter>(glo, ghi, ga, gb);
    if (now.r0 == 0) {
      float2 turn = turn_of(p, pos, lane);
      turn.y = -turn.y;
      spread<kInter>(turn, j, c, s);
    }
    advance(p, w);
    if (w.live) load(w);
    const int row = now.r0 + slot, side = row >= now.split;
    const uint64_t r = both(root_of(a, b, p.eps));
    rotate(ga, gb, c, s);  // dn
    weights_of(w_smem, side, j, wa, wb);
    uint64_t gx = 0;
    ulonglong2* dw = &dw_smem[warp][side][0][lane];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      a[i] = mul_f32x2(a[i], r), b[i] = mul_f32x2(b[i], r);  // x r
      const uint64_t ta = mul_f32x2(ga[i], a[i]), tb = mul_f32x2(gb[i], b[i]);
      if (row < now.rows) {
        const ulonglong2 sum = dw[i * 32];
        dw[i * 32] = make_ulonglong2(add_f32x2(sum.x, ta), add_f32x2(sum.y, tb));
      }
      gx = fma_f32x2(ta, wa[i], gx);
      gx = fma_f32x2(tb, wb[i], gx);
    }
    const uint64_t mean = both(sum4(sum_of(gx)) * (-1.f / kDim));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      ga[i] = mul_f32x2(r, fma_f32x2(a[i], mean, mul_f32x2(ga[i], wa[i])));
      gb[i] = mul_f32x2(r, fma_f32x2(b[i], mean, mul_f32x2(gb[i], wb[i])));
    }
    if (row < now.rows) store16<kInter>(row_of(p.s[0].y, p.s[0].ys, p.s[1].y, p.s[1].ys, now, row), j, ga, gb);
  }
  // The block's sums of dw, a column per thread: over its warps and their eight rows, in order.
  __syncthreads();
  if (threadIdx.x < 2 * kDim) {
    const int sd = threadIdx.x / kDim, cj = (threadIdx.x >> 4) & 3, second = (threadIdx.x >> 3) & 1, e = threadIdx.x & 7;
    float v = 0.f;
    for (int k = 0; k < kWarps; ++k)
#pragma unroll
      for (int l = 0; l < 8; ++l)
        v += reinterpret_cast<const float*>(&dw_smem[k][sd][e >> 1][4 * l + cj])[2 * second + (e & 1)];
    p.partial[int64_t(blockIdx.x) * 2 * kDim + sd * kDim + column_of<kInter>(cj, e, second)] = v;
  }
}

// dw of both sides from the blocks' sums, always in the same order: a block takes 16 columns, 64 threads a column (one
// block for all of them waited 7 us for its loads).
constexpr int kDwColumns = 16;
__global__ void __launch_bounds__(1024) qk_dw_kernel(const float* partial, int blocks, float* dwq, float* dwk) {
  __shared__ float part[64][kDwColumns + 1];
  nb::pdl_wait();
  nb::pdl_launch_dependents();
  const int c = threadIdx.x & (kDwColumns - 1), lane = threadIdx.x / kDwColumns, col = blockIdx.x * kDwColumns + c;
  float v = 0.f;
#pragma unroll 8
  for (int b = lane; b < blocks; b += 64) v += partial[b * 2 * kDim + col];
  part[lane][c] = v;
  __syncthreads();
  if (threadIdx.x < kDwColumns) {
    v = 0.f;
#pragma unroll
    for (int k = 0; k < 64; ++k) v += part[k][c];
    (col < kDim ? dwq : dwk)[col % kDim] = v;
  }
}

// ---- host ----------------------------------------------------------------------------------
template <typename... KArgs, typename... Args>
int launch(void (*kernel)(KArgs...), unsigned grid, unsigned threads, void* stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, KArgs(args)...) == cudaSuccess ? NB_ATTN_OK : NB_ATTN_ERR_LAUNCH;
}

int check_tensor(const nb_attn_tensor& t) {
  if (t.ptr == nullptr) return NB_ATTN_ERR_NULL;
  if ((reinterpret_cast<uintptr_t>(t.ptr) & 15u) != 0 || t.stride_batch % 8 || t.stride_token % 8 || t.stride_head % 8)
    return NB_ATTN_ERR_ALIGN;
  return NB_ATTN_OK;
}

int make_side(const nb_qk_side& in, const nb_qk_norm_rope_args& a, bool bwd, Side* out) {
  if (in.heads <= 0 || in.tokens < 0 || in.heads > 65535) return NB_ATTN_ERR_SHAPE;
  if (int64_t(in.tokens) * a.batch > INT32_MAX) return NB_ATTN_ERR_SHAPE;
  if (bwd && in.d_weight == nullptr) return NB_ATTN_ERR_NULL;
  if (in.tokens > 0 && a.batch > 0) {  // (a side without tokens has no addresses)
    if (int rc = check_tensor(in.x)) return rc;
    if (int rc = check_tensor(in.y)) return rc;
    if (bwd)
      if (int rc = check_tensor(in.dy)) return rc;
    if (a.axes > 0 && in.positions == nullptr) return NB_ATTN_ERR_NULL;
  }
  *out = Side{};
  out->x = static_cast<const __nv_bfloat16*>(in.x.ptr);
  out->y = static_cast<__nv_bfloat16*>(in.y.ptr);
  out->dy = static_cast<const __nv_bfloat16*>(in.dy.ptr);
  const nb_attn_tensor* t[3] = {&in.x, &in.y, &in.dy};
  int64_t* s[3] = {out->xs, out->ys, out->gs};
  for (int i = 0; i < 3; ++i) s[i][0] = t[i]->stride_batch, s[i][1] = t[i]->stride_token, s[i][2] = t[i]->stride_head;
  out->weight = in.weight;
  out->pos = in.positions;
  out->ps[0] = in.position_stride_batch, out->ps[1] = in.position_stride_token;
  out->heads = in.heads, out->tokens = in.tokens;
  return NB_ATTN_OK;
}

int make_params(const nb_qk_norm_rope_args* a, bool bwd, Params* p) {
  if (a == nullptr) return NB_ATTN_ERR_NULL;
  if (a->batch < 0 || a->axes < 0 || a->axes > NB_ROPE_MAX_AXES || a->position_type < 0 || a->position_type > 2)
    return NB_ATTN_ERR_SHAPE;
  if (a->axes > 0 && a->freqs == nullptr) return NB_ATTN_ERR_NULL;
  *p = Params{};
  if (int rc = make_side(a->q, *a, bwd, &p->s[0])) return rc;
  if (int rc = make_side(a->k, *a, bwd, &p->s[1])) return rc;
  const Side &q = p->s[0], &k = p->s[1];
  // A token's angles serve its queries and its keys where both have the same positions.
  p->shared = q.tokens == k.tokens &&
              (a->axes == 0 || (q.pos == k.pos && q.ps[0] == k.ps[0] && q.ps[1] == k.ps[1]));
  p->units_q = int64_t(a->batch) * q.tokens;
  p->units = p->units_q + (p->shared ? 0 : int64_t(a->batch) * k.tokens);
  // Batches that follow on one another in every tensor are one long batch: no division per token.
  p->one_batch = a->batch == 1;
  const auto follows = [](const int64_t* s, int64_t tokens) { return s[0] == tokens * s[1]; };
  if (!p->one_batch) {
    p->one_batch = true;
    for (const Side& s : p->s)
      p->one_batch = p->one_batch && follows(s.xs, s.tokens) && follows(s.ys, s.tokens) && (!bwd || follows(s.gs, s.tokens)) &&
                     (a->axes == 0 || follows(s.ps, s.tokens));
  }
  p->axes = a->axes, p->pos_type = a->position_type, p->interleaved = a->interleaved != 0;
  p->freqs = a->freqs, p->eps = a->eps;
  return NB_ATTN_OK;
}

}  // namespace

extern "C" int nb_qk_norm_rope_fwd(const nb_qk_norm_rope_args* args, void* stream) {
  Params p;
  if (int rc = make_params(args, false, &p)) return rc;
  int sms = 0;
  if (int rc = nb::host_prepare(&sms)) return rc;
  if (p.units == 0) return NB_ATTN_OK;
  const int64_t blocks = (p.units + kWarps - 1) / kWarps, most = int64_t(sms) * kFwdBlocks;
  return launch(p.interleaved ? qk_fwd_kernel<true> : qk_fwd_kernel<false>, unsigned(blocks < most ? blocks : most), kThreads,
                stream, p);
}

extern "C" size_t nb_qk_norm_rope_bwd_workspace_bytes(void) { return size_t(kBwdBlocksMax) * 2 * kDim * sizeof(float); }

extern "C" int nb_qk_norm_rope_bwd(const nb_qk_norm_rope_args* args, void* stream) {
  Params p;
  if (int rc = make_params(args, true, &p)) return rc;
  if (args->workspace == nullptr || args->workspace_bytes < nb_qk_norm_rope_bwd_workspace_bytes())
    return NB_ATTN_ERR_WORKSPACE;
  if ((reinterpret_cast<uintptr_t>(args->workspace) & 15u) != 0) return NB_ATTN_ERR_ALIGN;
  int sms = 0;
  if (int rc = nb::host_prepare(&sms)) return rc;
  p.partial = static_cast<float*>(args->workspace);
  int64_t blocks = (p.units + kWarps - 1) / kWarps;
  const int64_t most = int64_t(sms) * kBwdBlocks < kBwdBlocksMax ? int64_t(sms) * kBwdBlocks : kBwdBlocksMax;
  if (blocks > most) blocks = most;
  if (blocks > 0)
    if (int rc = launch(p.interleaved ? qk_bwd_kernel<true> : qk_bwd_kernel<false>, unsigned(blocks), kThreads, stream, p))
      return rc;
  return launch(qk_dw_kernel, unsigned(2 * kDim / kDwColumns), 1024u, stream, static_cast<const float*>(p.partial), int(blocks), args->q.d_weight,
                args->k.d_weight);
}
