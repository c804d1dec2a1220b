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
// exchange and every access is 16 bytes. Sums are in fp32; the one rounding is that of the result to bf16.
// Angles are products and sums in 64 bits, and whole turns are taken off there: position 2^20 at frequency 1 would keep
// an error of 0.03 in fp32.
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
  int32_t axes, pos_type, interleaved;
  const float* freqs;
  float eps;
  float* partial;               // backward: [blocks][2][64]
};

__device__ __forceinline__ float2 unpack2(uint32_t v) {
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
}

// cos and sin of the token's angle of pair `lane`.
__device__ __forceinline__ float2 turn_of(const Params& p, const Side& s, int64_t batch, int64_t token, int lane) {
  if (p.axes == 0) return make_float2(1.f, 0.f);
  const int64_t at = batch * s.ps[0] + token * s.ps[1];
  double angle = 0.0;
  for (int a = 0; a < p.axes; ++a) {
    double pos;
    if (p.pos_type == NB_POSITION_I64) pos = double(static_cast<const int64_t*>(s.pos)[at + a]);
    else if (p.pos_type == NB_POSITION_I32) pos = double(static_cast<const int32_t*>(s.pos)[at + a]);
    else pos = double(static_cast<const float*>(s.pos)[at + a]);
    angle = fma(pos, double(p.freqs[a * kPairs + lane]), angle);
  }
  // Whole turns off, in 64 bits; the rest in half turns, which need no reduction.
  const double turns = angle * 0.15915494309189533577;
  float sn, cs;
  sincospif(float(2.0 * (turns - rint(turns))), &sn, &cs);
  return make_float2(cs, sn);
}

// The eight (cos, sin) that a lane with column block j needs, from the lanes that hold them: those of its values'
// pairs, 8j + e, or interleaved 4j + e (first eight values) and 16 + 4j + e (the others), e < 4.
__device__ __forceinline__ void spread(float2 mine, int j, bool interleaved, float (&c)[8], float (&s)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int src = interleaved ? (e < 4 ? 4 * j + e : 16 + 4 * j + (e - 4)) : 8 * j + e;
    c[e] = __shfl_sync(0xffffffffu, mine.x, src);
    s[e] = __shfl_sync(0xffffffffu, mine.y, src);
  }
}

// v: a lane's 16 values, first the eight of block j, then those of block 4 + j. Turned by the angles, or back.
template <bool kBack>
__device__ __forceinline__ void rotate(float (&v)[16], const float (&c)[8], const float (&s)[8], bool interleaved) {
  if (interleaved) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float a = v[2 * e], b = v[2 * e + 1], t = kBack ? -s[e] : s[e];
      v[2 * e] = a * c[e] - b * t;
      v[2 * e + 1] = b * c[e] + a * t;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float a = v[e], b = v[8 + e], t = kBack ? -s[e] : s[e];
      v[e] = a * c[e] - b * t;
      v[8 + e] = b * c[e] + a * t;
    }
  }
}

__device__ __forceinline__ void to_float(const uint4& lo, const uint4& hi, float (&v)[16]) {
  const uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 f = unpack2(w[i]);
    v[2 * i] = f.x, v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void store16(__nv_bfloat16* p, int j, const float (&v)[16]) {
  uint4 lo, hi;
  lo.x = nb::pack_bf16(v[0], v[1]), lo.y = nb::pack_bf16(v[2], v[3]);
  lo.z = nb::pack_bf16(v[4], v[5]), lo.w = nb::pack_bf16(v[6], v[7]);
  hi.x = nb::pack_bf16(v[8], v[9]), hi.y = nb::pack_bf16(v[10], v[11]);
  hi.z = nb::pack_bf16(v[12], v[13]), hi.w = nb::pack_bf16(v[14], v[15]);
  *reinterpret_cast<uint4*>(p + 8 * j) = lo;
  *reinterpret_cast<uint4*>(p + 32 + 8 * j) = hi;
}
__device__ __forceinline__ float sum4(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}

// What a unit is: a token of one side, or of both.
struct Unit {
  int side, rows;          // the first row's side; rows of the unit
  int64_t batch, token;
};
__device__ __forceinline__ Unit unit_of(const Params& p, int64_t u) {
  Unit r;
  r.side = p.shared || u < p.units_q ? 0 : 1;
  const uint32_t at = uint32_t(r.side ? u - p.units_q : u), len = uint32_t(p.s[r.side].tokens);
  const uint32_t b = at / len;
  r.batch = b, r.token = at - b * len;
  r.rows = p.shared ? p.s[0].heads + p.s[1].heads : p.s[r.side].heads;
  return r;
}

// The weights of both sides in shared memory: [2][64].
__device__ __forceinline__ void load_weights(const Params& p, float* w) {
  if (threadIdx.x < 2 * kDim) {
    const float* src = p.s[threadIdx.x / kDim].weight;
    w[threadIdx.x] = src != nullptr ? src[threadIdx.x % kDim] : 1.f;
  }
  __syncthreads();
}
__device__ __forceinline__ void weights_of(const float* w, int side, int j, float (&v)[16]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float4 f = *reinterpret_cast<const float4*>(w + side * kDim + (i >> 1) * 32 + 8 * j + (i & 1) * 4);
    v[4 * i] = f.x, v[4 * i + 1] = f.y, v[4 * i + 2] = f.z, v[4 * i + 3] = f.w;
  }
}

// ---- forward -------------------------------------------------------------------------------
constexpr int kFwdDeep = 3;  // groups of eight rows whose loads are under way together (12 + 12 heads: all of a token)

__global__ void __launch_bounds__(kThreads) qk_fwd_kernel(const __grid_constant__ Params p) {
  __shared__ __align__(16) float w_smem[2 * kDim];
  nb::pdl_wait();
  nb::pdl_launch_dependents();
  load_weights(p, w_smem);
  const int lane = threadIdx.x & 31, j = lane & 3, slot = lane >> 2;
  const int64_t step = int64_t(gridDim.x) * kWarps;
  for (int64_t u = int64_t(blockIdx.x) * kWarps + (threadIdx.x >> 5); u < p.units; u += step) {
    const Unit unit = unit_of(p, u);
    float c[8], s[8];
    for (int r0 = 0; r0 < unit.rows; r0 += kFwdDeep * kRowsAtOnce) {
      uint4 lo[kFwdDeep], hi[kFwdDeep];
#pragma unroll
      for (int d = 0; d < kFwdDeep; ++d) {
        const int row = r0 + d * kRowsAtOnce + slot;
        if (row < unit.rows) {
          const int side = p.shared ? row >= p.s[0].heads : unit.side;
          const Side& sd = p.s[side];
          const int head = p.shared && side ? row - p.s[0].heads : row;
          const __nv_bfloat16* x = sd.x + unit.batch * sd.xs[0] + unit.token * sd.xs[1] + head * sd.xs[2];
          lo[d] = *reinterpret_cast<const uint4*>(x + 8 * j);
          hi[d] = *reinterpret_cast<const uint4*>(x + 32 + 8 * j);
        } else {
          lo[d] = hi[d] = make_uint4(0, 0, 0, 0);
        }
      }
      if (r0 == 0) spread(turn_of(p, p.s[unit.side], unit.batch, unit.token, lane), j, p.interleaved, c, s);
#pragma unroll
      for (int d = 0; d < kFwdDeep; ++d) {
        if (r0 + d * kRowsAtOnce >= unit.rows) break;
        const int row = r0 + d * kRowsAtOnce + slot;
        const int side = p.shared ? row >= p.s[0].heads : unit.side;
        float v[16], w[16];
        to_float(lo[d], hi[d], v);
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) ss = fmaf(v[i], v[i], ss);
        const float r = rsqrtf(sum4(ss) * (1.f / kDim) + p.eps);
        weights_of(w_smem, side, j, w);
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] *= r * w[i];
        rotate<false>(v, c, s, p.interleaved);
        if (row < unit.rows) {
          const Side& sd = p.s[side];
          const int head = p.shared && side ? row - p.s[0].heads : row;
          store16(sd.y + unit.batch * sd.ys[0] + unit.token * sd.ys[1] + head * sd.ys[2], j, v);
        }
      }
    }
  }
}

// ---- backward ------------------------------------------------------------------------------
constexpr int kBwdDeep = 2;

__global__ void __launch_bounds__(kThreads, 2) qk_bwd_kernel(const __grid_constant__ Params p) {
  __shared__ __align__(16) float w_smem[2 * kDim];
  __shared__ float dw_smem[kWarps][2 * kDim];
  nb::pdl_wait();
  nb::pdl_launch_dependents();
  load_weights(p, w_smem);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, j = lane & 3, slot = lane >> 2;
  float dw[2][16];
#pragma unroll
  for (int i = 0; i < 16; ++i) dw[0][i] = dw[1][i] = 0.f;
  const int64_t step = int64_t(gridDim.x) * kWarps;
  for (int64_t u = int64_t(blockIdx.x) * kWarps + warp; u < p.units; u += step) {
    const Unit unit = unit_of(p, u);
    float c[8], s[8];
    for (int r0 = 0; r0 < unit.rows; r0 += kBwdDeep * kRowsAtOnce) {
      uint4 lo[kBwdDeep], hi[kBwdDeep], glo[kBwdDeep], ghi[kBwdDeep];
#pragma unroll
      for (int d = 0; d < kBwdDeep; ++d) {
        const int row = r0 + d * kRowsAtOnce + slot;
        if (row < unit.rows) {
          const int side = p.shared ? row >= p.s[0].heads : unit.side;
          const Side& sd = p.s[side];
          const int head = p.shared && side ? row - p.s[0].heads : row;
          const __nv_bfloat16* x = sd.x + unit.batch * sd.xs[0] + unit.token * sd.xs[1] + head * sd.xs[2];
          const __nv_bfloat16* g = sd.dy + unit.batch * sd.gs[0] + unit.token * sd.gs[1] + head * sd.gs[2];
          lo[d] = *reinterpret_cast<const uint4*>(x + 8 * j);
          hi[d] = *reinterpret_cast<const uint4*>(x + 32 + 8 * j);
          glo[d] = *reinterpret_cast<const uint4*>(g + 8 * j);
          ghi[d] = *reinterpret_cast<const uint4*>(g + 32 + 8 * j);
        } else {
          lo[d] = hi[d] = glo[d] = ghi[d] = make_uint4(0, 0, 0, 0);
        }
      }
      if (r0 == 0) spread(turn_of(p, p.s[unit.side], unit.batch, unit.token, lane), j, p.interleaved, c, s);
#pragma unroll
      for (int d = 0; d < kBwdDeep; ++d) {
        if (r0 + d * kRowsAtOnce >= unit.rows) break;
        const int row = r0 + d * kRowsAtOnce + slot;
        const int side = p.shared ? row >= p.s[0].heads : unit.side;
        float v[16], g[16], w[16];
        to_float(lo[d], hi[d], v);
        to_float(glo[d], ghi[d], g);
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) ss = fmaf(v[i], v[i], ss);
        const float r = rsqrtf(sum4(ss) * (1.f / kDim) + p.eps);
        rotate<true>(g, c, s, p.interleaved);  // dn
        weights_of(w_smem, side, j, w);
        float gx = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          v[i] *= r;  // x r
          const float t = g[i] * v[i];
          if (row < unit.rows) {
            if (side) dw[1][i] += t;
            else dw[0][i] += t;
          }
          gx = fmaf(t, w[i], gx);
        }
        const float mean = sum4(gx) * (1.f / kDim);
#pragma unroll
        for (int i = 0; i < 16; ++i) g[i] = r * (g[i] * w[i] - v[i] * mean);
        if (row < unit.rows) {
          const Side& sd = p.s[side];
          const int head = p.shared && side ? row - p.s[0].heads : row;
          store16(sd.y + unit.batch * sd.ys[0] + unit.token * sd.ys[1] + head * sd.ys[2], j, g);
        }
      }
    }
  }
  // The block's sums of dw: over the eight rows of a warp, then over its warps in order.
#pragma unroll
  for (int side = 0; side < 2; ++side)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float v = dw[side][i];
      v += __shfl_xor_sync(0xffffffffu, v, 4);
      v += __shfl_xor_sync(0xffffffffu, v, 8);
      v += __shfl_xor_sync(0xffffffffu, v, 16);
      if (slot == 0) dw_smem[warp][side * kDim + (i >> 3) * 32 + 8 * j + (i & 7)] = v;
    }
  __syncthreads();
  if (threadIdx.x < 2 * kDim) {
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < kWarps; ++k) v += dw_smem[k][threadIdx.x];
    p.partial[int64_t(blockIdx.x) * 2 * kDim + threadIdx.x] = v;
  }
}

// dw of both sides from the blocks' sums, always in the same order: 8 threads a column.
__global__ void __launch_bounds__(1024) qk_dw_kernel(const float* partial, int blocks, float* dwq, float* dwk) {
  __shared__ float part[8][2 * kDim];
  nb::pdl_wait();
  nb::pdl_launch_dependents();
  const int col = threadIdx.x & 127, lane = threadIdx.x >> 7;
  float v = 0.f;
#pragma unroll 8
  for (int b = lane; b < blocks; b += 8) v += partial[b * 2 * kDim + col];
  part[lane][col] = v;
  __syncthreads();
  if (threadIdx.x < 2 * kDim) {
    v = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) v += part[k][threadIdx.x];
    (threadIdx.x < kDim ? dwq : dwk)[threadIdx.x % kDim] = v;
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
  if (in.tokens > 0) {  // (a side without tokens has no addresses)
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
  if (a->batch <= 0 || a->axes < 0 || a->axes > NB_ROPE_MAX_AXES || a->position_type < 0 || a->position_type > 2)
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
  const int64_t blocks = (p.units + kWarps - 1) / kWarps, most = int64_t(sms) * 3;
  return launch(qk_fwd_kernel, unsigned(blocks < most ? blocks : most), kThreads, stream, p);
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
  const int64_t most = int64_t(sms) * 2 < kBwdBlocksMax ? int64_t(sms) * 2 : kBwdBlocksMax;
  if (blocks > most) blocks = most;
  if (blocks > 0)
    if (int rc = launch(qk_bwd_kernel, unsigned(blocks), kThreads, stream, p)) return rc;
  return launch(qk_dw_kernel, 1u, 1024u, stream, static_cast<const float*>(p.partial), int(blocks), args->q.d_weight,
                args->k.d_weight);
}
