// The gated feed-forward block of include/nb_block.h: host side, the form for few tokens and the kernels that finish
// what gemm_kernel.cuh leaves in parts.
//
// Forward: one launch for a, b and h (kGemmGate), one for y. Backward: one for da, db (kGemmDact), one for dx and the
// three weight gradients together (kGemmPlain), and where needed one that adds split products up and two for the biases.
#include <cuda_runtime.h>

#include <algorithm>
#include <mutex>

#include "../../include/nb_block.h"
#include "gemm_kernel.cuh"
#include "host.h"

namespace {

using namespace nb;
using bf16 = __nv_bfloat16;

// ---- few tokens, forward only ----------------------------------------------------------------
// Bound by reading the weights once, from as many SMs and with as many loads under way as there can be: a block takes 16
// features (rows of Wg and Wu, or of Wd), its warps deal their 32-deep chunks out, and the block adds the warps' sums up.
// The products are mma.sync's of 16 features x 8 tokens: with one token per multiply-add the time grew with the tokens
// (768 x 2048, weights from memory, us: 1 token 7.1, 8 tokens 29; now 6.7, 7.2, 16 tokens 9.3), and the tiles of the large
// kernels occupy 16 to 48 SMs (17 for up to 128 tokens, and so faster from 17 tokens on: 32 tokens take 20 here). A
// lane's 16 bytes are eight neighbouring k of its row; the order of k inside a chunk does not matter as long as weights and
// tokens have the same.
constexpr int kFewTokens = 16, kFewRows = 16;
constexpr int kFewGateWarps = 8, kFewDownWarps = 16;

__device__ __forceinline__ void mma_16x8(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 32 deep: rows g and g + 8 of the features, row g of the tokens.
__device__ __forceinline__ void mma_chunk(float (&c)[4], const uint4& lo, const uint4& hi, const uint4& x) {
  mma_16x8(c, lo.x, hi.x, lo.y, hi.y, x.x, x.y);
  mma_16x8(c, lo.z, hi.z, lo.w, hi.w, x.z, x.w);
}

struct FewParams {
  const bf16 *x, *w0, *w1, *bias0, *bias1;
  bf16* out;
  int64_t xs, w0s, w1s, outs;
  int32_t tokens, in, out_n;
};

// 16 bytes of row `row`, zeros behind the last row or column.
__device__ __forceinline__ uint4 few_load(const bf16* m, int64_t stride, int row, int rows, int k, int n) {
  return row < rows && k < n ? *reinterpret_cast<const uint4*>(m + row * stride + k) : make_uint4(0, 0, 0, 0);
}

// Adds up the warps' sums of output i = (token, feature) of the block.
template <int kWarps, int kTiles>
__device__ __forceinline__ float few_total(const float (&part)[kWarps][kFewRows][8 * kTiles], int token, int feature) {
  float v = 0.f;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) v += part[w][feature][token];
  return v;
}
template <int kWarps, int kTiles>
__device__ __forceinline__ void few_put(float (&part)[kWarps][kFewRows][8 * kTiles], const float (&acc)[kTiles][4], int warp,
                                        int lane) {
  const int g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int i = 0; i < kTiles; ++i) {
    part[warp][g][8 * i + 2 * t] = acc[i][0], part[warp][g][8 * i + 2 * t + 1] = acc[i][1];
    part[warp][g + 8][8 * i + 2 * t] = acc[i][2], part[warp][g + 8][8 * i + 2 * t + 1] = acc[i][3];
  }
}

template <int kAct, int kTiles>  // tiles of eight tokens
__global__ void __launch_bounds__(kFewGateWarps * 32) few_gate_kernel(const __grid_constant__ FewParams p) {
  __shared__ float part_a[kFewGateWarps][kFewRows][8 * kTiles], part_b[kFewGateWarps][kFewRows][8 * kTiles];
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, f0 = blockIdx.x * kFewRows;
  float a[kTiles][4] = {}, b[kTiles][4] = {};
#pragma unroll 3
  for (int k = warp * 32 + (lane & 3) * 8; k < (p.in + 31) / 32 * 32; k += kFewGateWarps * 32) {
    const uint4 g0 = few_load(p.w0, p.w0s, f0 + g, p.out_n, k, p.in), g1 = few_load(p.w0, p.w0s, f0 + g + 8, p.out_n, k, p.in);
    const uint4 u0 = few_load(p.w1, p.w1s, f0 + g, p.out_n, k, p.in), u1 = few_load(p.w1, p.w1s, f0 + g + 8, p.out_n, k, p.in);
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
      const uint4 x = few_load(p.x, p.xs, 8 * i + g, p.tokens, k, p.in);
      mma_chunk(a[i], g0, g1, x);
      mma_chunk(b[i], u0, u1, x);
    }
  }
  few_put(part_a, a, warp, lane);
  few_put(part_b, b, warp, lane);
  __syncthreads();
  for (int i = threadIdx.x; i < kFewRows * 8 * kTiles; i += kFewGateWarps * 32) {
    const int token = i / kFewRows, feature = i % kFewRows, f = f0 + feature;
    if (token >= p.tokens || f >= p.out_n) continue;
    const float bg = p.bias0 != nullptr ? __bfloat162float(p.bias0[f]) : 0.f;
    const float bu = p.bias1 != nullptr ? __bfloat162float(p.bias1[f]) : 0.f;
    const float va = few_total<kFewGateWarps, kTiles>(part_a, token, feature) + bg;
    const float vb = few_total<kFewGateWarps, kTiles>(part_b, token, feature) + bu;
    p.out[token * p.outs + f] = __float2bfloat16(gate_of<kAct>(va) * vb);
  }
}

constexpr int kFewAhead = 4;  // chunks of a warp's weights requested before the kernel in front is done
template <int kTiles>
__global__ void __launch_bounds__(kFewDownWarps * 32) few_down_kernel(const __grid_constant__ FewParams p) {
  __shared__ float part[kFewDownWarps][kFewRows][8 * kTiles];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, d0 = blockIdx.x * kFewRows;
  const int k0 = warp * 32 + (lane & 3) * 8;
  constexpr int kStep = kFewDownWarps * 32;
  // The gate kernel, which comes right in front, does not write weights.
  uint4 lo[kFewAhead], hi[kFewAhead];
#pragma unroll
  for (int i = 0; i < kFewAhead; ++i) {
    lo[i] = few_load(p.w0, p.w0s, d0 + g, p.out_n, k0 + i * kStep, p.in);
    hi[i] = few_load(p.w0, p.w0s, d0 + g + 8, p.out_n, k0 + i * kStep, p.in);
  }
  pdl_wait();
  pdl_launch_dependents();
  float y[kTiles][4] = {};
#pragma unroll
  for (int i = 0; i < kFewAhead; ++i) {
    if (warp * 32 + i * kStep >= p.in) break;
#pragma unroll
    for (int t = 0; t < kTiles; ++t) mma_chunk(y[t], lo[i], hi[i], few_load(p.x, p.xs, 8 * t + g, p.tokens, k0 + i * kStep, p.in));
  }
#pragma unroll 2
  for (int k = k0 + kFewAhead * kStep; k < (p.in + 31) / 32 * 32; k += kStep) {
    const uint4 w0 = few_load(p.w0, p.w0s, d0 + g, p.out_n, k, p.in), w1 = few_load(p.w0, p.w0s, d0 + g + 8, p.out_n, k, p.in);
#pragma unroll
    for (int t = 0; t < kTiles; ++t) mma_chunk(y[t], w0, w1, few_load(p.x, p.xs, 8 * t + g, p.tokens, k, p.in));
  }
  few_put(part, y, warp, lane);
  __syncthreads();
  for (int i = threadIdx.x; i < kFewRows * 8 * kTiles; i += kFewDownWarps * 32) {
    const int token = i / kFewRows, feature = i % kFewRows, d = d0 + feature;
    if (token >= p.tokens || d >= p.out_n) continue;
    const float bias = p.bias0 != nullptr ? __bfloat162float(p.bias0[d]) : 0.f;
    p.out[token * p.outs + d] = __float2bfloat16(few_total<kFewDownWarps, kTiles>(part, token, feature) + bias);
  }
}

// ---- what is left in parts ---------------------------------------------------------------------
// The sum of a split product's parts, in their order. A thread takes a row's eight columns.
struct SplitItem {
  const float4* partial;
  bf16* out;
  int64_t stride;
  int32_t rows, n, row_tiles, col_tiles, cols, splits;
  int64_t pieces;  // of 8 columns x 1 row, over whole tiles
};
struct SplitParams {
  SplitItem item[4];
  int32_t n_items;
};
__global__ void __launch_bounds__(256) split_sum_kernel(const __grid_constant__ SplitParams p) {
  pdl_wait();
  pdl_launch_dependents();
  int64_t at = int64_t(blockIdx.x) * 256 + threadIdx.x;
  int i = 0;
  while (i < p.n_items && at >= p.item[i].pieces) at -= p.item[i++].pieces;
  if (i == p.n_items) return;
  const SplitItem& s = p.item[i];
  const int row = int(at % kGemmRows);
  const int64_t block = at / kGemmRows;  // (tile, eight columns)
  const int per = s.cols / 8;
  const int tile = int(block / per), oct = int(block % per);
  const int64_t whole = int64_t(s.row_tiles) * s.col_tiles * (s.cols / 4) * kGemmRows;
  const float4* src = s.partial + (int64_t(tile) * (s.cols / 4) + 2 * oct) * kGemmRows + row;
  float4 a = src[0], b = src[kGemmRows];
  for (int k = 1; k < s.splits; ++k) {
    const float4 x = src[k * whole], y = src[k * whole + kGemmRows];
    a.x += x.x, a.y += x.y, a.z += x.z, a.w += x.w;
    b.x += y.x, b.y += y.y, b.z += y.z, b.w += y.w;
  }
  const int64_t r = int64_t(tile / s.col_tiles) * kGemmRows + row;
  const int c = (tile % s.col_tiles) * s.cols + 8 * oct;
  if (r < s.rows && c < s.n)
    *reinterpret_cast<uint4*>(s.out + r * s.stride + c) =
        make_uint4(pack_bf16(a.x, a.y), pack_bf16(a.z, a.w), pack_bf16(b.x, b.y), pack_bf16(b.z, b.w));
}

// Sums of a matrix' columns over chunks of kSumRows rows: a block takes 64 columns.
constexpr int kSumRows = 512;
constexpr int kDirectRows = 4096;  // up to so many rows the last kernel reads the matrix itself: a launch less
struct ColPartialParams {
  const bf16* m;
  int64_t stride, rows;
  float* out;
  int32_t n;
};
__global__ void __launch_bounds__(256) col_partial_kernel(const __grid_constant__ ColPartialParams p) {
  __shared__ float part[32][65];
  const bf16* m = p.m;
  const int64_t stride = p.stride, rows = p.rows;
  const int n = p.n;
  float* out = p.out;
  pdl_wait();
  pdl_launch_dependents();
  const int oct = threadIdx.x & 7, lane = threadIdx.x >> 3, c = blockIdx.x * 64 + oct * 8;
  float s[8] = {};
  const int64_t first = int64_t(blockIdx.y) * kSumRows, last = first + kSumRows < rows ? first + kSumRows : rows;
  if (c < n) {
#pragma unroll 4
    for (int64_t r = first + lane; r < last; r += 32) {
      const uint4 v = *reinterpret_cast<const uint4*>(m + r * stride + c);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) s[2 * i] += __uint_as_float(w[i] << 16), s[2 * i + 1] += __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) part[lane][oct * 8 + i] = s[i];
  __syncthreads();
  if (threadIdx.x < 64 && blockIdx.x * 64 + threadIdx.x < n) {
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) v += part[i][threadIdx.x];
    out[int64_t(blockIdx.y) * n + blockIdx.x * 64 + threadIdx.x] = v;
  }
}

struct ColItem {
  const void* from;      // fp32 or bf16 [rows][stride]
  bf16* out;
  int64_t stride;
  int32_t rows, n, blocks;
  int32_t is_bf16;
};
struct ColParams {
  ColItem item[3];
  int32_t n_items;
};
__global__ void __launch_bounds__(1024) col_sum_kernel(const __grid_constant__ ColParams p) {
  __shared__ float part[32][33];
  pdl_wait();
  pdl_launch_dependents();
  int b = blockIdx.x, i = 0;
  while (b >= p.item[i].blocks) b -= p.item[i++].blocks;
  const ColItem& s = p.item[i];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = b * 32 + lane;
  float v = 0.f;
  if (c < s.n) {
    if (s.is_bf16) {
#pragma unroll 8
      for (int r = warp; r < s.rows; r += 32) v += __bfloat162float(static_cast<const bf16*>(s.from)[r * s.stride + c]);
    } else {
#pragma unroll 8
      for (int r = warp; r < s.rows; r += 32) v += static_cast<const float*>(s.from)[r * s.stride + c];
    }
  }
  part[warp][lane] = v;
  __syncthreads();
  if (warp == 0 && c < s.n) {
    v = 0.f;
#pragma unroll
    for (int k = 0; k < 32; ++k) v += part[k][lane];
    s.out[c] = __float2bfloat16(v);
  }
}

// ---- host --------------------------------------------------------------------------------------
template <typename... KArgs>
int launch_cluster(void (*kernel)(KArgs...), int cluster, dim3 grid, unsigned threads, size_t smem, void* stream,
                   const KArgs&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = unsigned(cluster), attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...) == cudaSuccess ? NB_ATTN_OK : NB_ATTN_ERR_LAUNCH;
}
template <typename Arg>
int launch(void (*kernel)(Arg), dim3 grid, unsigned threads, size_t smem, void* stream, const Arg& arg) {
  return launch_cluster(kernel, 1, grid, threads, smem, stream, arg);
}

// A GEMM kernel needs its shared memory allowed once per device.
constexpr int kMaxDevices = 64;
template <int kCtas, int kKind, int kAct, int kBits, int kProblems>
int launch_gemm(const GemmParams<kProblems>& g, int sms, int32_t* status, void* stream) {
  static std::mutex mutex;
  static bool ready[kMaxDevices];
  auto* kernel = gemm_kernel<kCtas, kKind, kAct, kBits, kProblems>;
  using L = GemmLayout<kKind, kBits, kCtas>;
  constexpr int kSmem = L::kBytes;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return NB_ATTN_ERR_DEVICE;
  {
    std::lock_guard<std::mutex> lock(mutex);
    if (!ready[dev]) {
      if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) != cudaSuccess)
        return NB_ATTN_ERR_LAUNCH;
      ready[dev] = true;
    }
  }
  const int units = g.deal.n_long + g.deal.n_short, teams = std::min(units, sms / kCtas);
  return launch_cluster(kernel, kCtas, dim3(unsigned(teams * kCtas)), kGemmThreads, kSmem, stream, g, GemmTail{status, {}});
}
template <int kKind, int kAct, int kBits, int kProblems>
int launch_gemm(const GemmParams<kProblems>& g, int ctas, int sms, int32_t* status, void* stream) {
  return ctas == 2 ? launch_gemm<2, kKind, kAct, kBits, kProblems>(g, sms, status, stream)
                   : launch_gemm<1, kKind, kAct, kBits, kProblems>(g, sms, status, stream);
}

int div_up(int64_t a, int64_t b) { return int((a + b - 1) / b); }
// Rows of hidden features in scratch begin on lines of 128 bytes.
int64_t padded(int hidden) { return (int64_t(hidden) + 63) / 64 * 64; }
size_t align256(size_t n) { return (n + 255) / 256 * 256; }

// Teams of one or two CTAs, and the columns of their tiles, by the clocks that a team's share of the tiles takes. A 64-deep
// step's MMAs take two clocks a column; its operands cross the port of a CTA's shared memory (128 bytes a clock) twice.
// A tile's epilogue takes `epilogue` clocks a column and runs under the next tile's products; the last one does not.
struct Tiling {
  int ctas, cols, row_tiles, col_tiles;
  double clocks;
};
constexpr double kPlainClocks = 8, kGateClocks = 26, kDactClocks = 30;  // per column and CTA
double step_clocks(const Tiling& t) { return std::max(2.0 * t.cols, 256.0 + 2.0 * t.cols / t.ctas); }
Tiling tiling(int64_t m, int n, int steps, int sms, int ctas, int cols, double epilogue) {
  Tiling t{ctas, cols, div_up(m, int64_t(ctas) * kGemmRows), div_up(n, cols), 0.0};
  const int64_t tiles = int64_t(t.row_tiles) * t.col_tiles, teams = sms / ctas;
  t.clocks = double((tiles + teams - 1) / teams) * (std::max(steps * step_clocks(t), epilogue * cols) + 400.0) + epilogue * cols +
             1000.0 * ctas;
  return t;
}
Tiling best_tiling(int64_t m, int n, int steps, int sms, double epilogue) {
  Tiling best = tiling(m, n, steps, sms, 2, kGemmMaxCols, epilogue);
  for (int ctas = 2; ctas >= 1; --ctas)
    for (int cols = kGemmMaxCols; cols >= 64; cols -= 64) {
      const Tiling t = tiling(m, n, steps, sms, ctas, cols, epilogue);
      if (t.clocks < 0.98 * best.clocks) best = t;
    }
  return best;
}

int check_matrix(const nb_matrix& m, int64_t cols) {
  if (m.ptr == nullptr) return NB_ATTN_ERR_NULL;
  if ((reinterpret_cast<uintptr_t>(m.ptr) & 15u) != 0 || m.stride % 8 != 0 || m.stride < cols || m.stride >> 36) return NB_ATTN_ERR_ALIGN;
  return NB_ATTN_OK;
}
int check_bias(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0 ? NB_ATTN_ERR_ALIGN : NB_ATTN_OK; }

constexpr int kMaxWidth = 1 << 20;
int check_shape(const nb_gated_mlp_shape& s) {
  if (s.tokens <= 0 || s.dim <= 0 || s.hidden <= 0 || s.dim % 8 || s.hidden % 8) return NB_ATTN_ERR_SHAPE;
  if (s.dim > kMaxWidth || s.hidden > kMaxWidth || s.tokens > INT32_MAX - kGemmRows) return NB_ATTN_ERR_SHAPE;
  // Tiles are counted in 32 bits, of 64 columns at the least.
  const int64_t rows = div_up(s.tokens, kGemmRows);
  if (rows * div_up(std::max(s.dim, s.hidden), 64) > INT32_MAX / 4) return NB_ATTN_ERR_SHAPE;
  if (s.activation != NB_ACT_SILU && s.activation != NB_ACT_GELU) return NB_ATTN_ERR_SHAPE;
  if (s.checkpoint < NB_CHECKPOINT_NONE || s.checkpoint > NB_CHECKPOINT_8BIT) return NB_ATTN_ERR_SHAPE;
  return NB_ATTN_OK;
}

size_t code_bytes(const nb_gated_mlp_shape& s) {
  const size_t blocks = size_t(div_up(s.tokens, kGemmRows)) * div_up(s.hidden, kGroup) * 4;
  return blocks * (s.checkpoint == NB_CHECKPOINT_8BIT ? CodeBlock<8>::kBytes : CodeBlock<16>::kBytes);
}

// Boxes of an operand whose inner index runs along memory: 64 deep x rows; of the others: 64 x 64.
int map_k_major(CUtensorMap* m, const nb_matrix& t, int64_t rows, int64_t cols, int box_rows) {
  return host_matrix_map(m, t.ptr, rows, cols, t.stride, box_rows, 64);
}
int map_mn_major(CUtensorMap* m, const nb_matrix& t, int64_t rows, int64_t cols) {
  return host_matrix_map(m, t.ptr, rows, cols, t.stride, 64, 64);
}

#define NB_TRY(expr)                 \
  do {                               \
    if (const int rc_ = (expr)) return rc_; \
  } while (0)

template <int kAct, int kTiles>
int launch_few(const nb_gated_mlp_fwd_args& a, void* stream) {
  const nb_gated_mlp_shape& s = a.shape;
  FewParams p{};
  p.x = static_cast<const bf16*>(a.x.ptr), p.xs = a.x.stride;
  p.w0 = static_cast<const bf16*>(a.w_gate.ptr), p.w0s = a.w_gate.stride;
  p.w1 = static_cast<const bf16*>(a.w_up.ptr), p.w1s = a.w_up.stride;
  p.bias0 = static_cast<const bf16*>(a.b_gate), p.bias1 = static_cast<const bf16*>(a.b_up);
  p.out = static_cast<bf16*>(a.h.ptr), p.outs = a.h.stride;
  p.tokens = int(s.tokens), p.in = s.dim, p.out_n = s.hidden;
  NB_TRY(launch(few_gate_kernel<kAct, kTiles>, dim3(div_up(s.hidden, kFewRows)), kFewGateWarps * 32, 0, stream, p));
  FewParams d{};
  d.x = p.out, d.xs = p.outs;
  d.w0 = static_cast<const bf16*>(a.w_down.ptr), d.w0s = a.w_down.stride;
  d.bias0 = static_cast<const bf16*>(a.b_down);
  d.out = static_cast<bf16*>(a.y.ptr), d.outs = a.y.stride;
  d.tokens = int(s.tokens), d.in = s.hidden, d.out_n = s.dim;
  return launch(few_down_kernel<kTiles>, dim3(div_up(s.dim, kFewRows)), kFewDownWarps * 32, 0, stream, d);
}
template <int kAct>
int launch_few(const nb_gated_mlp_fwd_args& a, void* stream) {
  return a.shape.tokens <= 8 ? launch_few<kAct, 1>(a, stream) : launch_few<kAct, 2>(a, stream);
}

template <int kKind, int kAct>
int launch_bits(const GemmParams<1>& g, int checkpoint, int ctas, int sms, int32_t* status, void* stream) {
  switch (checkpoint) {
    case NB_CHECKPOINT_16BIT: return launch_gemm<kKind, kAct, 16, 1>(g, ctas, sms, status, stream);
    case NB_CHECKPOINT_8BIT: return launch_gemm<kKind, kAct, 8, 1>(g, ctas, sms, status, stream);
  }
  if constexpr (kKind == kGemmGate) return launch_gemm<kKind, kAct, 0, 1>(g, ctas, sms, status, stream);
  return NB_ATTN_ERR_SHAPE;
}
template <int kKind>
int launch_act(const GemmParams<1>& g, const nb_gated_mlp_shape& s, int ctas, int sms, int32_t* status, void* stream) {
  return s.activation == NB_ACT_SILU ? launch_bits<kKind, kActSilu>(g, s.checkpoint, ctas, sms, status, stream)
                                     : launch_bits<kKind, kActGelu>(g, s.checkpoint, ctas, sms, status, stream);
}

// The kernels divide unit numbers (below 2^31) by the column tiles: with 2^(k-1) < d <= 2^k, ceil(2^(31+k) / d) is below 2^32
// and its product's excess, below u / 2^31, does not reach the next whole number.
void set_col_tiles(GemmProblem* p, int col_tiles) {
  int k = 0;
  while ((int64_t(1) << k) < col_tiles) ++k;
  p->col_tiles = col_tiles;
  p->by_shift = uint32_t(31 + k);
  p->by_col_tiles = uint32_t(((uint64_t(1) << (31 + k)) + col_tiles - 1) / col_tiles);
}

void set_tiles(GemmProblem* p, int64_t rows, int n, const Tiling& t, int steps0, int steps) {
  p->m = int(rows), p->n = n;
  p->row_tiles = t.row_tiles, p->cols = t.cols;
  set_col_tiles(p, t.col_tiles);
  p->steps0 = steps0, p->steps = steps;
  p->splits = 1, p->split_steps = steps;
}

// A product behind da and db: [m][n] over `steps` 64-deep steps, in tiles and parts of the steps.
enum { kDWGate = 0, kDWUp = 1, kDWDown = 2, kDx = 3, kProducts = 4 };
struct Product {
  bool wanted;
  int64_t m;
  int n, steps;
  Tiling tiles;
  int splits, split_steps;
  size_t part_bytes;  // fp32 sums of the parts, where there are several
  double unit_clocks() const { return step_clocks(tiles) * split_steps; }
  double clocks() const { return step_clocks(tiles) * steps * tiles.row_tiles * tiles.col_tiles; }
  int units() const { return tiles.row_tiles * tiles.col_tiles * splits; }
};
// Where the backward's scratch lies in the workspace, and how its products are cut.
struct BwdPlan {
  size_t da, db, h, col_sums, dy_sums, parts[kProducts], bytes;
  int ctas;
  Product p[kProducts];
  double clocks;
};

// The products by teams of `ctas`.
void plan_products(BwdPlan* plan, const nb_gated_mlp_bwd_args& a, int sms, int ctas) {
  const nb_gated_mlp_shape& s = a.shape;
  const int tokens = div_up(s.tokens, kGemmDepth), hidden = div_up(s.hidden, kGemmDepth);
  plan->ctas = ctas;
  plan->p[kDWGate] = {a.d_w_gate.ptr != nullptr, s.hidden, s.dim, tokens};
  plan->p[kDWUp] = {a.d_w_up.ptr != nullptr, s.hidden, s.dim, tokens};
  plan->p[kDWDown] = {a.d_w_down.ptr != nullptr, s.dim, s.hidden, tokens};
  plan->p[kDx] = {a.dx.ptr != nullptr, s.tokens, s.dim, 2 * hidden};
  double total = 0.0;
  for (Product& p : plan->p) {
    const int cols = div_up(div_up(p.n, div_up(p.n, kGemmMaxCols)), 64) * 64;
    p.tiles = tiling(p.m, p.n, p.steps, sms, ctas, cols, kPlainClocks);
    if (p.wanted) total += p.clocks();
  }
  // A unit that runs over all steps may be more than a team's even share of the launch's work. Then it is cut into parts of
  // about half a share, which are added up by another launch (fp32, in a fixed order): worth while from some 12000 clocks
  // on, with parts of 6000 at the least. (26253 x 768 x 2048: nothing is cut; 820 tokens of it: dx, 35 -> 25 us with the sum.)
  const double share = total / (sms / ctas);
  double longest = 0.0;
  for (Product& p : plan->p) {
    const double unit = step_clocks(p.tiles) * p.steps;
    int splits = 1;
    if (unit > 0.8 * share && unit > 12000.0) splits = std::min(32, int(unit / std::max(0.5 * share, 6000.0)) + 1);
    splits = std::max(splits, div_up(p.steps, 1 << 18));  // (a unit stays far below the time after which a wait gives up)
    p.split_steps = div_up(p.steps, splits);
    p.splits = div_up(p.steps, p.split_steps);
    const size_t tiles = size_t(p.tiles.row_tiles) * ctas * p.tiles.col_tiles;
    p.part_bytes = p.wanted && p.splits > 1 ? tiles * p.tiles.cols * kGemmRows * 4 * p.splits : 0;
    if (p.wanted) longest = std::max(longest, p.unit_clocks());
  }
  plan->clocks = std::max(share + 0.25 * longest, longest) + 1000.0 * ctas;
}

BwdPlan plan_bwd(const nb_gated_mlp_bwd_args& a, int sms) {
  const nb_gated_mlp_shape& s = a.shape;
  BwdPlan p{}, single{};
  plan_products(&p, a, sms, 2);  // (all products of the launch have teams of one size)
  plan_products(&single, a, sms, 1);
  if (single.clocks < 0.98 * p.clocks) p = single;
  size_t at = 0;
  const auto take = [&at](size_t n) {
    const size_t here = at;
    at += align256(n);
    return here;
  };
  const size_t hidden_bytes = size_t(s.tokens) * padded(s.hidden) * 2, row_tiles = size_t(div_up(s.tokens, kGemmRows));
  p.da = take(hidden_bytes), p.db = take(hidden_bytes);
  p.h = take(s.checkpoint == NB_CHECKPOINT_8BIT ? hidden_bytes : 0);
  p.col_sums = take(a.d_b_gate != nullptr || a.d_b_up != nullptr ? row_tiles * 4 * 2 * s.hidden * 4 : 0);
  p.dy_sums = take(a.d_b_down != nullptr && s.tokens > kDirectRows ? size_t(div_up(s.tokens, kSumRows)) * s.dim * 4 : 0);
  for (int i = 0; i < kProducts; ++i) p.parts[i] = take(p.p[i].part_bytes);
  p.bytes = std::max<size_t>(at, 256);
  return p;
}

}  // namespace

extern "C" size_t nb_gated_mlp_checkpoint_bytes(const nb_gated_mlp_shape* shape) {
  if (shape == nullptr || check_shape(*shape) != NB_ATTN_OK || shape->checkpoint == NB_CHECKPOINT_NONE) return 0;
  return code_bytes(*shape);
}

extern "C" int nb_gated_mlp_fwd(const nb_gated_mlp_fwd_args* args, void* stream) {
  if (args == nullptr) return NB_ATTN_ERR_NULL;
  const nb_gated_mlp_shape& s = args->shape;
  NB_TRY(check_shape(s));
  NB_TRY(check_matrix(args->x, s.dim));
  NB_TRY(check_matrix(args->w_gate, s.dim));
  NB_TRY(check_matrix(args->w_up, s.dim));
  NB_TRY(check_matrix(args->w_down, s.hidden));
  NB_TRY(check_matrix(args->y, s.dim));
  NB_TRY(check_matrix(args->h, s.hidden));
  for (const void* b : {args->b_gate, args->b_up, args->b_down}) NB_TRY(check_bias(b));
  if (s.checkpoint != NB_CHECKPOINT_NONE) {
    if (args->checkpoint == nullptr) return NB_ATTN_ERR_NULL;
    if ((reinterpret_cast<uintptr_t>(args->checkpoint) & 255u) != 0) return NB_ATTN_ERR_ALIGN;
  }
  int sms = 0;
  NB_TRY(host_prepare(&sms));
  if (s.checkpoint == NB_CHECKPOINT_NONE && s.tokens <= kFewTokens)
    return s.activation == NB_ACT_SILU ? launch_few<kActSilu>(*args, stream) : launch_few<kActGelu>(*args, stream);

  const int steps = div_up(s.dim, kGemmDepth);
  GemmParams<1> g{};
  GemmProblem& p = g.p[0];
  // (a tile has as many columns of a as of b)
  const Tiling tg = best_tiling(s.tokens, 2 * s.hidden, steps, sms, kGateClocks);
  const int cols = tg.cols;
  set_tiles(&p, s.tokens, s.hidden, tg, steps, steps);
  set_col_tiles(&p, div_up(s.hidden, cols / 2));
  NB_TRY(map_k_major(&p.a[0], args->x, s.tokens, s.dim, kGemmRows));
  NB_TRY(map_k_major(&p.b[0], args->w_gate, s.hidden, s.dim, cols / 2));
  NB_TRY(map_k_major(&p.b[1], args->w_up, s.hidden, s.dim, cols / 2));
  NB_TRY(host_matrix_map(&p.c, args->h.ptr, s.tokens, s.hidden, args->h.stride, 32, kGroup));
  p.bias = static_cast<const bf16*>(args->b_gate);
  g.bias_up = static_cast<const bf16*>(args->b_up);
  g.codes = static_cast<uint8_t*>(args->checkpoint);
  g.groups = div_up(s.hidden, kGroup), g.hidden = s.hidden;
  g.deal.n_short = p.row_tiles * p.col_tiles;

  GemmParams<1> d{};
  GemmProblem& q = d.p[0];
  const int down_steps = div_up(s.hidden, kGemmDepth);
  const Tiling td = best_tiling(s.tokens, s.dim, down_steps, sms, kPlainClocks);
  set_tiles(&q, s.tokens, s.dim, td, down_steps, down_steps);
  NB_TRY(map_k_major(&q.a[0], args->h, s.tokens, s.hidden, kGemmRows));
  NB_TRY(map_k_major(&q.b[0], args->w_down, s.dim, s.hidden, td.cols / td.ctas));
  NB_TRY(host_matrix_map(&q.c, args->y.ptr, s.tokens, s.dim, args->y.stride, 32, 64));
  q.bias = static_cast<const bf16*>(args->b_down);
  d.deal.n_short = q.row_tiles * q.col_tiles;
  NB_TRY(launch_act<kGemmGate>(g, s, tg.ctas, sms, args->status, stream));
  return launch_gemm<kGemmPlain, 0, 0, 1>(d, td.ctas, sms, args->status, stream);
}

extern "C" size_t nb_gated_mlp_bwd_workspace_bytes(const nb_gated_mlp_bwd_args* args) {
  int sms = 0;
  if (args == nullptr || check_shape(args->shape) != NB_ATTN_OK || host_prepare(&sms) != NB_ATTN_OK) return 0;
  return plan_bwd(*args, sms).bytes;
}

extern "C" int nb_gated_mlp_bwd(const nb_gated_mlp_bwd_args* args, void* stream) {
  if (args == nullptr) return NB_ATTN_ERR_NULL;
  const nb_gated_mlp_bwd_args& a = *args;
  const nb_gated_mlp_shape& s = a.shape;
  NB_TRY(check_shape(s));
  if (s.checkpoint == NB_CHECKPOINT_NONE) return NB_ATTN_ERR_SHAPE;
  NB_TRY(check_matrix(a.x, s.dim));
  NB_TRY(check_matrix(a.w_gate, s.dim));
  NB_TRY(check_matrix(a.w_up, s.dim));
  NB_TRY(check_matrix(a.w_down, s.hidden));
  NB_TRY(check_matrix(a.dy, s.dim));
  if (s.checkpoint == NB_CHECKPOINT_16BIT) NB_TRY(check_matrix(a.h, s.hidden));
  if (a.dx.ptr != nullptr) NB_TRY(check_matrix(a.dx, s.dim));
  if (a.d_w_gate.ptr != nullptr) NB_TRY(check_matrix(a.d_w_gate, s.dim));
  if (a.d_w_up.ptr != nullptr) NB_TRY(check_matrix(a.d_w_up, s.dim));
  if (a.d_w_down.ptr != nullptr) NB_TRY(check_matrix(a.d_w_down, s.hidden));
  if (a.d_b_down != nullptr && s.tokens > int64_t(65535) * kSumRows) return NB_ATTN_ERR_SHAPE;  // (the sums' grid)
  if (a.checkpoint == nullptr) return NB_ATTN_ERR_NULL;
  if ((reinterpret_cast<uintptr_t>(a.checkpoint) & 255u) != 0 || (reinterpret_cast<uintptr_t>(a.workspace) & 255u) != 0)
    return NB_ATTN_ERR_ALIGN;
  int sms = 0;
  NB_TRY(host_prepare(&sms));
  const BwdPlan plan = plan_bwd(a, sms);
  if (a.workspace == nullptr || a.workspace_bytes < plan.bytes) return NB_ATTN_ERR_WORKSPACE;
  char* ws = static_cast<char*>(a.workspace);
  const int64_t stride = padded(s.hidden);
  const nb_matrix da{ws + plan.da, stride}, db{ws + plan.db, stride};
  const nb_matrix h = s.checkpoint == NB_CHECKPOINT_8BIT ? nb_matrix{ws + plan.h, stride} : a.h;
  const int row_tiles = div_up(s.tokens, kGemmRows);

  // dh = dy Wd with the activation's backward behind it. (Needed for every gradient but those of Wd, in 16 bits, and bd.)
  const bool hidden_grads = a.dx.ptr != nullptr || a.d_w_gate.ptr != nullptr || a.d_w_up.ptr != nullptr ||
                            a.d_b_gate != nullptr || a.d_b_up != nullptr;
  const bool dact = hidden_grads || (a.d_w_down.ptr != nullptr && s.checkpoint == NB_CHECKPOINT_8BIT);
  GemmParams<1> act{};
  Tiling act_tiling{};
  if (dact) {
    GemmParams<1>& g = act;
    GemmProblem& p = g.p[0];
    const int steps = div_up(s.dim, kGemmDepth);
    act_tiling = best_tiling(s.tokens, s.hidden, steps, sms, kDactClocks);
    set_tiles(&p, s.tokens, s.hidden, act_tiling, steps, steps);
    p.b_mn = 1;
    NB_TRY(map_k_major(&p.a[0], a.dy, s.tokens, s.dim, kGemmRows));
    NB_TRY(map_mn_major(&p.b[0], a.w_down, s.dim, s.hidden));
    NB_TRY(host_matrix_map(&p.c, da.ptr, s.tokens, s.hidden, da.stride, 32, kGroup));
    NB_TRY(host_matrix_map(&g.map_db, db.ptr, s.tokens, s.hidden, db.stride, 32, kGroup));
    if (s.checkpoint == NB_CHECKPOINT_8BIT)
      NB_TRY(host_matrix_map(&g.map_h, h.ptr, s.tokens, s.hidden, h.stride, 32, kGroup));
    if (a.d_b_gate != nullptr || a.d_b_up != nullptr) g.col_sums = reinterpret_cast<float*>(ws + plan.col_sums);
    g.codes = static_cast<uint8_t*>(const_cast<void*>(a.checkpoint));
    g.groups = div_up(s.hidden, kGroup), g.hidden = s.hidden;
    g.deal.n_short = p.row_tiles * p.col_tiles;
  }

  // dx and the weight gradients, the longer units first.
  GemmParams<kProducts> g{};
  SplitParams sums{};
  int n = 0;
  const auto add = [&](int which, const nb_matrix& out) -> int {
    const Product& from = plan.p[which];
    if (!from.wanted) return NB_ATTN_OK;
    const bool dx = which == kDx;
    GemmProblem& p = g.p[n++];
    set_tiles(&p, from.m, from.n, from.tiles, dx ? from.steps / 2 : from.steps, from.steps);
    p.splits = from.splits, p.split_steps = from.split_steps;
    p.a_mn = !dx, p.b_mn = 1;
    if (dx) {
      NB_TRY(map_k_major(&p.a[0], da, s.tokens, s.hidden, kGemmRows));
      NB_TRY(map_k_major(&p.a[1], db, s.tokens, s.hidden, kGemmRows));
      NB_TRY(map_mn_major(&p.b[0], a.w_gate, s.hidden, s.dim));
      NB_TRY(map_mn_major(&p.b[1], a.w_up, s.hidden, s.dim));
    } else {
      NB_TRY(map_mn_major(&p.a[0], which == kDWGate ? da : which == kDWUp ? db : a.dy, s.tokens, from.m));
      NB_TRY(map_mn_major(&p.b[0], which == kDWDown ? h : a.x, s.tokens, from.n));
    }
    if (p.splits == 1) return host_matrix_map(&p.c, out.ptr, from.m, from.n, out.stride, 32, 64);
    p.partial = reinterpret_cast<float*>(ws + plan.parts[which]);
    SplitItem& i = sums.item[sums.n_items++];
    i.partial = reinterpret_cast<const float4*>(p.partial);
    i.out = static_cast<bf16*>(out.ptr), i.stride = out.stride;
    i.rows = int(from.m), i.n = from.n, i.row_tiles = p.row_tiles * plan.ctas, i.col_tiles = p.col_tiles, i.cols = p.cols;
    i.splits = p.splits;
    i.pieces = int64_t(i.row_tiles) * p.col_tiles * (p.cols / 8) * kGemmRows;
    return NB_ATTN_OK;
  };
  const Product &dx = plan.p[kDx], &dw = plan.p[kDWGate];
  const bool dw_first = dw.unit_clocks() >= dx.unit_clocks();
  if (!dw_first) NB_TRY(add(kDx, a.dx));
  NB_TRY(add(kDWGate, a.d_w_gate));
  NB_TRY(add(kDWUp, a.d_w_up));
  NB_TRY(add(kDWDown, a.d_w_down));
  if (dw_first) NB_TRY(add(kDx, a.dx));
  if (dact) NB_TRY(launch_act<kGemmDact>(act, s, act_tiling.ctas, sms, a.status, stream));
  if (n > 0) {
    int dw_units = 0;
    for (int i = 0; i < kDx; ++i) dw_units += plan.p[i].wanted ? plan.p[i].units() : 0;
    const int dx_units = dx.wanted ? dx.units() : 0;
    g.deal.n_long = dw_first ? dw_units : dx_units, g.deal.n_short = dw_first ? dx_units : dw_units;
    const int teams = std::min(dw_units + dx_units, sms / plan.ctas), rem = g.deal.n_long % teams;
    if (g.deal.n_short > 0 && rem > 0) {
      const double ratio = dw.unit_clocks() / dx.unit_clocks();
      g.deal.extra = std::min(int(dw_first ? ratio : 1.0 / ratio), g.deal.n_short / (teams - rem));
    }
    NB_TRY((launch_gemm<kGemmPlain, 0, 0, kProducts>(g, plan.ctas, sms, a.status, stream)));
  }
  if (sums.n_items > 0) {
    int64_t pieces = 0;
    for (int i = 0; i < sums.n_items; ++i) pieces += sums.item[i].pieces;
    NB_TRY(launch(split_sum_kernel, dim3(unsigned((pieces + 255) / 256)), 256, 0, stream, sums));
  }

  // Biases.
  ColParams cols{};
  const auto add_col = [&](void* out, const void* from, bool is_bf16, int64_t stride, int rows, int width) {
    if (out == nullptr) return;
    cols.item[cols.n_items++] = ColItem{from, static_cast<bf16*>(out), stride, rows, width, div_up(width, 32), is_bf16};
  };
  const float* sums_at = reinterpret_cast<const float*>(ws + plan.col_sums);
  add_col(a.d_b_gate, sums_at, false, 2 * int64_t(s.hidden), row_tiles * 4, s.hidden);
  add_col(a.d_b_up, sums_at + s.hidden, false, 2 * int64_t(s.hidden), row_tiles * 4, s.hidden);
  if (s.tokens <= kDirectRows) {
    add_col(a.d_b_down, a.dy.ptr, true, a.dy.stride, int(s.tokens), s.dim);
  } else if (a.d_b_down != nullptr) {
    float* dy_sums = reinterpret_cast<float*>(ws + plan.dy_sums);
    const int chunks = div_up(s.tokens, kSumRows);
    NB_TRY(launch(col_partial_kernel, dim3(div_up(s.dim, 64), chunks), 256, 0, stream,
                  ColPartialParams{static_cast<const bf16*>(a.dy.ptr), a.dy.stride, s.tokens, dy_sums, s.dim}));
    add_col(a.d_b_down, dy_sums, false, s.dim, chunks, s.dim);
  }
  if (cols.n_items > 0) {
    int blocks = 0;
    for (int i = 0; i < cols.n_items; ++i) blocks += cols.item[i].blocks;
    NB_TRY(launch(col_sum_kernel, dim3(blocks), 1024, 0, stream, cols));
  }
  return NB_ATTN_OK;
}
