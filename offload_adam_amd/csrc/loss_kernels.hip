// Softmax cross entropy of a linear head, z = x W^T, without ever holding z.
//
// Forward: the tiled product of oa_gemm.hpp with an epilogue that folds each
// token's tile of logits into a running maximum and sum of exponentials (one pair
// per token and tile) and picks out the target's logit; a second kernel joins the
// pairs into lse_t = log sum_v exp z[t,v] and the losses lse_t - z[t,y_t].
//
// Backward, in pieces of the vocabulary: the product again, with an epilogue that
// turns each logit into d[t,v] = exp(z[t,v] - lse_t) - [v = y_t] and stores it in 16
// bits, as [t][v] and as [v][t]; then dx += d W_piece (fp32) and dw_piece = d^T x.
//
// Bound by the matrix cores: 2 T V H operations forward, 6 T V H backward (z is
// computed again).  Logits, maxima, sums and the sums over tokens and vocabulary are
// fp32; d is rounded once to the 16-bit type of x and W, as it would be by a
// framework that stores the logits' gradient.

#include <math.h>

#include <type_traits>

#include "oa_gemm.hpp"

#pragma clang fp contract(off)

namespace oa {
namespace {

using namespace gemm;

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kCombineTokens = 32, kCombineParts = 8;
constexpr int kCombineThreads = kCombineTokens * kCombineParts;
constexpr int kReduceThreads = 1024;

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// (maximum, sum of exp(z - maximum)) of two disjoint sets of logits.
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2) {
  const float top = fmaxf(m, m2);
  const float at = top == -INFINITY ? 0.0f : top;  // two empty sets: 0 * exp(-inf), not exp(nan)
  s = s * exp2_hw((m - at) * kLog2e) + s2 * exp2_hw((m2 - at) * kLog2e);
  m = top;
}

template <class T>
struct Store16;
template <>
struct Store16<Bf16> {
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    return f32x2_to_bf16x2_bits(a, b);
  }
};
template <>
struct Store16<F16> {
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const _Float16 lo = (_Float16)a, hi = (_Float16)b;
    return (uint32_t)__builtin_bit_cast(uint16_t, lo) |
           ((uint32_t)__builtin_bit_cast(uint16_t, hi) << 16);
  }
};

// ------------------------------------------------------------------- forward

struct StatsEpilogue {
  const int64_t* target;
  int64_t tokens, vocab;
  f32x2* part;      // [vocabulary tile][token]: maximum, sum
  float* z_target;  // [token]

  template <class Tl>
  __device__ __forceinline__ void operator()(Tl& t, int64_t row_q, int64_t row_p, int tq, int,
                                             uint8_t* lds) const {
    f32x2* all = reinterpret_cast<f32x2*>(lds);  // [wave along q][token of the tile]
    __syncthreads();
    const int64_t v0 = row_q + t.q0();
    const bool whole = row_q + Tl::BQ <= vocab;
#pragma unroll
    for (int b = 0; b < Tl::PT; ++b) {
      const int64_t token = row_p + t.p0() + 16 * b;
      const int64_t y = token < tokens ? target[token] : -1;
      const int64_t rel64 = y - v0;
      const int rel = rel64 >= 0 && rel64 < Tl::BQ && y < vocab ? (int)rel64 : -1;
      float m = -INFINITY, hit = 0.0f;
      bool found = false;
#pragma unroll
      for (int a = 0; a < Tl::QT; ++a)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (!whole && v0 + 16 * a + i >= vocab) t.acc[a][b][i] = -INFINITY;
          const float z = t.acc[a][b][i];
          m = fmaxf(m, z);
          if (rel == 16 * a + i) {
            hit = z;
            found = true;
          }
        }
      if (found) z_target[token] = hit;
      const float at = (m == -INFINITY ? 0.0f : m) * kLog2e;
      float s = 0.0f;
#pragma unroll
      for (int a = 0; a < Tl::QT; ++a)
#pragma unroll
        for (int i = 0; i < 4; ++i) s += exp2_hw(fmaf(t.acc[a][b][i], kLog2e, -at));
      // the four lanes that hold this token's logits
      join(m, s, __shfl_xor(m, 16, kWave), __shfl_xor(s, 16, kWave));
      join(m, s, __shfl_xor(m, 32, kWave), __shfl_xor(s, 32, kWave));
      if (t.lane < 16) all[t.wq * Tl::BP + t.p0() + 16 * b] = f32x2{m, s};
    }
    __syncthreads();
    for (int i = threadIdx.x; i < Tl::BP; i += Tl::kThreads) {
      f32x2 v = all[i];
      float m = v[0], s = v[1];
#pragma unroll
      for (int w = 1; w < Tl::kWavesQ; ++w) join(m, s, all[w * Tl::BP + i][0], all[w * Tl::BP + i][1]);
      if (row_p + i < tokens) part[(int64_t)tq * tokens + row_p + i] = f32x2{m, s};
    }
  }
};

// Joins a token's tiles: eight lanes per token, then the eight.  A target outside
// [0, vocab) that is not `ignore` makes the loss NaN.
__global__ void __launch_bounds__(kCombineThreads)
ce_combine_kernel(const f32x2* __restrict__ part, const float* __restrict__ z_target,
                  const int64_t* __restrict__ target, int64_t tokens, int64_t vocab,
                  int64_t ignore, int tiles, float* __restrict__ lse_out,
                  float* __restrict__ loss_out, float* __restrict__ block_sum,
                  int* __restrict__ block_count) {
  __shared__ f32x2 all[kCombineParts][kCombineTokens];
  const int col = threadIdx.x % kCombineTokens, row = threadIdx.x / kCombineTokens;
  const int64_t token = (int64_t)blockIdx.x * kCombineTokens + col;
  float m = -INFINITY, s = 0.0f;
  if (token < tokens)
    for (int j = row; j < tiles; j += kCombineParts) {
      const f32x2 v = part[(int64_t)j * tokens + token];
      join(m, s, v[0], v[1]);
    }
  all[row][col] = f32x2{m, s};
  __syncthreads();
  if (threadIdx.x >= kWave) return;
  float loss = 0.0f;
  bool used = false;
  if (threadIdx.x < kCombineTokens && token < tokens) {
    for (int j = 1; j < kCombineParts; ++j) join(m, s, all[j][col][0], all[j][col][1]);
    const float lse = m + logf(s);
    lse_out[token] = lse;
    const int64_t y = target[token];
    used = y != ignore;
    if (used) loss = y >= 0 && y < vocab ? lse - z_target[token] : NAN;
    if (loss_out) loss_out[token] = loss;
  }
  const float total = wave_sum(loss);
  const int count = __popcll(__ballot(used));
  if (threadIdx.x == 0) {
    block_sum[blockIdx.x] = total;
    block_count[blockIdx.x] = count;
  }
}

// Sum over the workgroups of the kernel above, in a fixed order, and the number of
// tokens that took part.
__global__ void __launch_bounds__(kReduceThreads)
ce_reduce_kernel(const float* __restrict__ block_sum, const int* __restrict__ block_count,
                 int blocks, int mean, float* __restrict__ loss_out, float* __restrict__ count_out) {
  __shared__ float sums[kReduceThreads / kWave];
  __shared__ int counts[kReduceThreads / kWave];
  float s = 0.0f;
  int c = 0;
  for (int i = threadIdx.x; i < blocks; i += kReduceThreads) {
    s += block_sum[i];
    c += block_count[i];
  }
  s = wave_sum(s);
  for (int off = kWave / 2; off > 0; off >>= 1) c += __shfl_xor(c, off, kWave);
  if (threadIdx.x % kWave == 0) {
    sums[threadIdx.x / kWave] = s;
    counts[threadIdx.x / kWave] = c;
  }
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int w = 1; w < kReduceThreads / kWave; ++w) {
    s += sums[w];
    c += counts[w];
  }
  *count_out = (float)c;
  if (loss_out) *loss_out = mean ? s / (float)c : s;  // nothing took part: 0 / 0
}

// ------------------------------------------------------------------ backward

// Factors of a token.  The 16-bit d has to survive in fp16 too, whose smallest
// normal number (6e-5) is far above a probability times a gradient of 1 / tokens:
// there d is held times 2^15, and in [v][t] relative to the largest gradient.
struct TokenFactors {
  float* held;    // d -> [v][t]; 0: the token takes no part
  float* dx;      // sum over v -> dx
  float* dw;      // one element: sum over t -> dw
};
constexpr float kF16Lift = 32768.0f;

__global__ void __launch_bounds__(kReduceThreads)
ce_factors_kernel(const float* __restrict__ grad, int per_token, int mean,
                  const float* __restrict__ count, const int64_t* __restrict__ target,
                  int64_t tokens, int64_t padded, int64_t vocab, int64_t ignore, int f16,
                  TokenFactors f) {
  __shared__ float tops[kReduceThreads / kWave];
  const float lift = f16 ? kF16Lift : 1.0f;
  float top = 0.0f;
  for (int64_t i = threadIdx.x; i < padded; i += kReduceThreads) {
    float g = 0.0f;
    if (i < tokens && target[i] != ignore) {
      g = grad[per_token ? i : 0];
      if (mean) g = g / *count;
      if (target[i] < 0 || target[i] >= vocab) g = NAN;
    }
    f.held[i] = g;
    f.dx[i] = g / lift;
    top = fmaxf(top, fabsf(g));
  }
  if (!f16) {
    if (threadIdx.x == 0) *f.dw = 1.0f;
    return;
  }
  top = wave_max(top);
  if (threadIdx.x % kWave == 0) tops[threadIdx.x / kWave] = top;
  __syncthreads();
  for (int w = 0; w < kReduceThreads / kWave; ++w) top = fmaxf(top, tops[w]);
  if (threadIdx.x == 0) *f.dw = top / lift;
  // each lane rescales what it wrote itself
  for (int64_t i = threadIdx.x; i < padded; i += kReduceThreads) {
    const float g = f.held[i];
    if (g != 0.0f) f.held[i] = g / top * lift;
  }
}

template <class T>
struct ProbEpilogue {
  const int64_t* target;
  const float* lse;
  const float* held;
  int64_t tokens, vocab;  // of the piece: targets and columns count from its first row
  int64_t first;          // first vocabulary row of the piece
  uint16_t* d;            // [token][ld_d]
  uint16_t* d_t;          // [vocabulary row of the piece][ld_t]
  int64_t ld_d, ld_t;
  float lift;

  template <class Tl>
  __device__ __forceinline__ void operator()(Tl& t, int64_t row_q, int64_t row_p, int, int,
                                             uint8_t*) const {
    const int64_t v0 = row_q + t.q0();
#pragma unroll
    for (int b = 0; b < Tl::PT; ++b) {
      const int64_t token = row_p + t.p0() + 16 * b;
      const bool here = token < tokens;
      const float h = here ? held[token] : 0.0f;
      const bool used = h != 0.0f;
      const float at = (here ? lse[token] : 0.0f) * kLog2e;
      const int64_t rel64 = (here ? target[token] - first : -1) - v0;
      const int rel = rel64 >= 0 && rel64 < Tl::BQ ? (int)rel64 : -1;
#pragma unroll
      for (int a = 0; a < Tl::QT; ++a) {
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float p = exp2_hw(fmaf(t.acc[a][b][i], kLog2e, -at));
          if (rel == 16 * a + i) p -= 1.0f;
          v[i] = used && v0 + 16 * a + i < vocab ? p : 0.0f;
        }
        const u32x2 w = {Store16<T>::pack(v[0] * lift, v[1] * lift),
                         Store16<T>::pack(v[2] * lift, v[3] * lift)};
        if (d) *reinterpret_cast<u32x2*>(d + token * ld_d + v0 + 16 * a) = w;
        if (d_t) {
          const u32x2 u = {Store16<T>::pack(v[0] * h, v[1] * h),
                           Store16<T>::pack(v[2] * h, v[3] * h)};
          uint16_t* o = d_t + (v0 + 16 * a) * ld_t + token;
          o[0] = (uint16_t)u[0];
          o[ld_t] = (uint16_t)(u[0] >> 16);
          o[2 * ld_t] = (uint16_t)u[1];
          o[3 * ld_t] = (uint16_t)(u[1] >> 16);
        }
      }
    }
  }
};

// dx of one piece, added to the pieces before it: [slice][token][hidden] fp32.
struct SumEpilogue {
  float* sum;
  int64_t tokens, hidden;
  int first;  // nothing is there yet

  template <class Tl>
  __device__ __forceinline__ void operator()(Tl& t, int64_t row_q, int64_t row_p, int, int slice,
                                             uint8_t*) const {
    float* base = sum + (int64_t)slice * tokens * hidden;
#pragma unroll
    for (int b = 0; b < Tl::PT; ++b) {
      const int64_t token = row_p + t.p0() + 16 * b;
      if (token >= tokens) continue;
#pragma unroll
      for (int a = 0; a < Tl::QT; ++a) {
        const int64_t h = row_q + t.q0() + 16 * a;
        if (h >= hidden) continue;  // hidden is a multiple of 8: four at a time
        f32x4* o = reinterpret_cast<f32x4*>(base + token * hidden + h);
        f32x4 v = t.acc[a][b];
        if (!first) v += *o;
        *o = v;
      }
    }
  }
};

template <class T>
struct WeightGradEpilogue {
  uint16_t* dw;
  int64_t rows, hidden;
  const float* factor;

  template <class Tl>
  __device__ __forceinline__ void operator()(Tl& t, int64_t row_q, int64_t row_p, int, int,
                                             uint8_t*) const {
    const float f = *factor;
#pragma unroll
    for (int b = 0; b < Tl::PT; ++b) {
      const int64_t row = row_p + t.p0() + 16 * b;
      if (row >= rows) continue;
#pragma unroll
      for (int a = 0; a < Tl::QT; ++a) {
        const int64_t h = row_q + t.q0() + 16 * a;
        if (h >= hidden) continue;
        const f32x4 v = t.acc[a][b] * f;
        const u32x2 w = {Store16<T>::pack(v[0], v[1]), Store16<T>::pack(v[2], v[3])};
        *reinterpret_cast<u32x2*>(dw + row * hidden + h) = w;
      }
    }
  }
};

// Slices of the fp32 sums -> dx in 16 bits, four elements per lane.
template <class T>
__global__ void __launch_bounds__(256)
ce_dx_kernel(const float* __restrict__ sum, int slices, const float* __restrict__ held,
             const float* __restrict__ factor, int64_t tokens, int64_t hidden,
             uint16_t* __restrict__ dx) {
  const int64_t quads = tokens * hidden / 4;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= quads) return;
  const int64_t token = i * 4 / hidden;
  f32x4 v = reinterpret_cast<const f32x4*>(sum)[i];
  for (int s = 1; s < slices; ++s) v += reinterpret_cast<const f32x4*>(sum)[s * quads + i];
  v = held[token] == 0.0f ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : v * factor[token];
  reinterpret_cast<u32x2*>(dx)[i] =
      u32x2{Store16<T>::pack(v[0], v[1]), Store16<T>::pack(v[2], v[3])};
}

// out[c][r] = in[r][c] of 16-bit elements, 64 x 64 per workgroup; rows from `rows` up
// to ld_out, and rows whose keep[] is 0, read as zero.
constexpr int kTrTile = 64;
__global__ void __launch_bounds__(256)
transpose16_kernel(const uint16_t* __restrict__ in, int64_t ld_in, int64_t rows, int64_t cols,
                   const float* __restrict__ keep, uint16_t* __restrict__ out, int64_t ld_out) {
  __shared__ uint16_t tile[kTrTile][kTrTile + 2];
  const int64_t r0 = (int64_t)blockIdx.x * kTrTile, c0 = (int64_t)blockIdx.y * kTrTile;
#pragma unroll
  for (int k = 0; k < 2; ++k) {  // eight consecutive columns of a row per lane
    const int i = threadIdx.x + 256 * k, r = i / 8, c = i % 8 * 8;
    u16x8 v = {0, 0, 0, 0, 0, 0, 0, 0};
    if (r0 + r < rows && c0 + c < cols && (!keep || keep[r0 + r] != 0.0f))
      v = *reinterpret_cast<const u16x8*>(in + (r0 + r) * ld_in + c0 + c);
#pragma unroll
    for (int j = 0; j < 8; ++j) tile[r][c + j] = v[j];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int i = threadIdx.x + 256 * k, c = i / 8, r = i % 8 * 8;
    if (c0 + c >= cols) continue;
    u16x8 v;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = tile[r + j][c];
    *reinterpret_cast<u16x8*>(out + (c0 + c) * ld_out + r0 + r) = v;
  }
}

int transpose16(const void* in, int64_t ld_in, int64_t rows, int64_t cols, const float* keep,
                void* out, int64_t ld_out, hipStream_t s) {
  hipLaunchKernelGGL(transpose16_kernel,
                     dim3((unsigned)(ld_out / kTrTile), (unsigned)tiles_along(cols, kTrTile)),
                     dim3(256), 0, s, static_cast<const uint16_t*>(in), ld_in, rows, cols, keep,
                     static_cast<uint16_t*>(out), ld_out);
  return launch_status();
}

// --------------------------------------------------------------- host side

int64_t up_to(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

// Carves a workspace; with a null base it only counts.
struct Carver {
  uint8_t* base;
  size_t used = 0;
  template <class P>
  P* take(int64_t count) {
    P* p = reinterpret_cast<P*>(base ? base + used : nullptr);
    used += (size_t)up_to(count * (int64_t)sizeof(P), 256);
    return p;
  }
};

struct ForwardPlan {
  bool large;
  int tiles;
  int blocks;
  f32x2* part;
  float *z_target, *block_sum;
  int* block_count;
  size_t bytes;
  ForwardPlan(int64_t tokens, int64_t vocab, void* ws) {
    large = large_tiles_fill(vocab, tokens);
    tiles = (int)tiles_along(vocab, large ? 256 : 128);
    blocks = (int)tiles_along(tokens, kCombineTokens);
    Carver c{static_cast<uint8_t*>(ws)};
    part = c.take<f32x2>((int64_t)tiles * tokens);
    z_target = c.take<float>(tokens);
    block_sum = c.take<float>(blocks);
    block_count = c.take<int>(blocks);
    bytes = c.used;
  }
};

// Elements of d that a piece of the vocabulary may hold: 64 Mi (128 MiB, twice).  A
// larger piece saves passes over the fp32 sums of dx (one read and write per piece).
constexpr int64_t kPieceElems = (int64_t)64 << 20;

struct BackwardPlan {
  int64_t padded;       // tokens, rounded up to whole tiles
  int64_t piece;        // vocabulary rows of a piece, whole tiles
  int slices;           // of the dx product
  float *held, *dx_factor, *dw_factor;
  uint16_t *d, *d_t, *x_t, *w_t;
  float* sum;
  size_t bytes;
  BackwardPlan(int64_t tokens, int64_t hidden, int64_t vocab, bool want_dx, bool want_dw, void* ws) {
    padded = up_to(tokens, 256);
    const int64_t whole = up_to(vocab, 256);
    int64_t most = kPieceElems / padded / 256 * 256;
    if (most < 256) most = 256;
    const int64_t pieces = tiles_along(whole, (int)(most < whole ? most : whole));
    piece = up_to(tiles_along(whole, (int)pieces), 256);
    slices = slices_for(hidden, tokens, piece * 2);
    Carver c{static_cast<uint8_t*>(ws)};
    held = c.take<float>(padded);
    dx_factor = c.take<float>(padded);
    dw_factor = c.take<float>(1);
    d = want_dx ? c.take<uint16_t>(padded * piece) : nullptr;
    w_t = want_dx ? c.take<uint16_t>(hidden * piece) : nullptr;
    sum = want_dx ? c.take<float>(slices * tokens * hidden) : nullptr;
    d_t = want_dw ? c.take<uint16_t>(padded * piece) : nullptr;
    x_t = want_dw ? c.take<uint16_t>(hidden * padded) : nullptr;
    bytes = c.used;
  }
};

template <class T, class E>
int product(const Problem& pr, bool large, int slices, const E& e, hipStream_t s) {
  return large ? launch_tiles<Large<T>, E>(pr, slices, e, s)
               : launch_tiles<Small<T>, E>(pr, slices, e, s);
}

struct Head {
  const uint8_t *x, *w;
  int64_t ldx, ldw;  // elements
  const int64_t* target;
  int64_t tokens, hidden, vocab, ignore;
};

Problem logits_problem(const Head& h, int64_t first, int64_t rows) {
  Problem pr{};
  pr.q = Operand{h.w + first * h.ldw * 2, h.ldw * 2, rows};
  pr.p = Operand{h.x, h.ldx * 2, h.tokens};
  pr.k_bytes = (int)(h.hidden * 2);
  return pr;
}

template <class T>
int forward(const Head& h, int reduction, float* loss, float* lse, float* count, void* ws,
            hipStream_t s) {
  const ForwardPlan plan(h.tokens, h.vocab, ws);
  if (h.tokens > 0) {
    const StatsEpilogue e{h.target, h.tokens, h.vocab, plan.part, plan.z_target};
    int rc = product<T>(logits_problem(h, 0, h.vocab), plan.large, 1, e, s);
    if (rc) return rc;
    hipLaunchKernelGGL(ce_combine_kernel, dim3((unsigned)plan.blocks), dim3(kCombineThreads), 0, s,
                       plan.part, plan.z_target, h.target, h.tokens, h.vocab, h.ignore, plan.tiles,
                       lse, reduction == OA_LOSS_NONE ? loss : nullptr, plan.block_sum,
                       plan.block_count);
    rc = launch_status();
    if (rc) return rc;
  }
  hipLaunchKernelGGL(ce_reduce_kernel, dim3(1), dim3(kReduceThreads), 0, s, plan.block_sum,
                     plan.block_count, plan.blocks, reduction == OA_LOSS_MEAN,
                     reduction == OA_LOSS_NONE ? nullptr : loss, count);
  return launch_status();
}

template <class T>
int backward(const Head& h, int reduction, const float* lse, const float* count,
             const float* grad, uint16_t* dx, uint16_t* dw, void* ws, hipStream_t s) {
  const BackwardPlan plan(h.tokens, h.hidden, h.vocab, dx != nullptr, dw != nullptr, ws);
  const bool f16 = std::is_same<T, F16>::value;
  const TokenFactors f{plan.held, plan.dx_factor, plan.dw_factor};
  hipLaunchKernelGGL(ce_factors_kernel, dim3(1), dim3(kReduceThreads), 0, s, grad,
                     (int)(reduction == OA_LOSS_NONE), (int)(reduction == OA_LOSS_MEAN), count,
                     h.target, h.tokens, plan.padded, h.vocab, h.ignore, (int)f16, f);
  int rc = launch_status();
  if (rc) return rc;
  if (dw) {
    rc = transpose16(h.x, h.ldx, h.tokens, h.hidden, plan.held, plan.x_t, plan.padded, s);
    if (rc) return rc;
  }
  for (int64_t first = 0; first < h.vocab; first += plan.piece) {
    const int64_t rows = h.vocab - first < plan.piece ? h.vocab - first : plan.piece;
    Problem pr = logits_problem(h, first, rows);
    const bool large = large_tiles_fill(rows, h.tokens);
    const ProbEpilogue<T> pe{h.target, lse,      plan.held,  h.tokens, rows,
                             first,    plan.d,   plan.d_t,   plan.piece, plan.padded,
                             f16 ? kF16Lift : 1.0f};
    rc = product<T>(pr, large, 1, pe, s);
    if (rc) return rc;
    const int64_t tile = large ? 256 : 128;
    if (dx) {
      rc = transpose16(h.w + first * h.ldw * 2, h.ldw, rows, h.hidden, nullptr, plan.w_t,
                       plan.piece, s);
      if (rc) return rc;
      Problem px{};
      px.q = Operand{reinterpret_cast<uint8_t*>(plan.w_t), plan.piece * 2, h.hidden};
      px.p = Operand{reinterpret_cast<uint8_t*>(plan.d), plan.piece * 2, h.tokens};
      px.k_bytes = (int)(up_to(rows, tile) * 2);
      const SumEpilogue se{plan.sum, h.tokens, h.hidden, (int)(first == 0)};
      rc = product<T>(px, plan.slices == 1 && large_tiles_fill(h.hidden, h.tokens), plan.slices,
                      se, s);
      if (rc) return rc;
    }
    if (dw) {
      Problem pw{};
      pw.q = Operand{reinterpret_cast<uint8_t*>(plan.x_t), plan.padded * 2, h.hidden};
      pw.p = Operand{reinterpret_cast<uint8_t*>(plan.d_t), plan.padded * 2, rows};
      pw.k_bytes = (int)(up_to(h.tokens, tile) * 2);
      const WeightGradEpilogue<T> we{dw + first * h.hidden, rows, h.hidden, plan.dw_factor};
      rc = product<T>(pw, large_tiles_fill(h.hidden, rows), 1, we, s);
      if (rc) return rc;
    }
  }
  if (dx) {
    const int64_t quads = h.tokens * h.hidden / 4;
    hipLaunchKernelGGL(ce_dx_kernel<T>, dim3((unsigned)tiles_along(quads, 256)), dim3(256), 0, s,
                       plan.sum, plan.slices, plan.held, plan.dx_factor, h.tokens, h.hidden, dx);
    rc = launch_status();
  }
  return rc;
}

int check_head(const Head& h, int dtype, int reduction) {
  if (dtype != OA_BF16 && dtype != OA_F16) return OA_EINVAL;
  if (reduction != OA_LOSS_NONE && reduction != OA_LOSS_MEAN && reduction != OA_LOSS_SUM)
    return OA_EINVAL;
  if (h.tokens < 0 || h.hidden <= 0 || h.vocab <= 0 || !h.w) return OA_EINVAL;
  if (h.tokens > 0 && (!h.x || !h.target)) return OA_EINVAL;
  if (h.ldw < h.hidden || (h.tokens > 1 && h.ldx < h.hidden)) return OA_EINVAL;
  if (h.hidden % 8 || h.ldx % 8 || h.ldw % 8 || !aligned_to(h.x, 16) || !aligned_to(h.w, 16) ||
      !aligned_to(h.target, 8))
    return OA_EALIGN;
  if (h.ldx > (1 << 20) || h.ldw > (1 << 20) || h.tokens > (1 << 22) || h.vocab > (1 << 24))
    return OA_ERANGE;
  return 0;
}

}  // namespace
}  // namespace oa

using namespace oa;

extern "C" size_t oa_linear_ce_workspace_bytes(int64_t tokens, int64_t hidden, int64_t vocab,
                                               int backward, int want_dx, int want_dw) {
  if (tokens < 0 || hidden <= 0 || vocab <= 0) return 0;
  // never 0: the workspace of an empty batch is a valid pointer too
  if (!backward) return ForwardPlan(tokens, vocab, nullptr).bytes + 256;
  return BackwardPlan(tokens, hidden, vocab, want_dx != 0, want_dw != 0, nullptr).bytes + 256;
}

extern "C" int oa_linear_ce_forward(const void* x, int64_t ldx, const void* w, int64_t ldw,
                                    int dtype, const int64_t* target, int64_t tokens,
                                    int64_t hidden, int64_t vocab, int64_t ignore_index,
                                    int reduction, float* loss, float* lse, float* count,
                                    void* workspace, size_t workspace_bytes, void* stream) {
  const Head h{static_cast<const uint8_t*>(x), static_cast<const uint8_t*>(w), ldx, ldw, target,
               tokens, hidden, vocab, ignore_index};
  int rc = check_head(h, dtype, reduction);
  if (rc) return rc;
  if (!loss || !lse || !count || !workspace) return OA_EINVAL;
  if (!aligned_to(workspace, 256) || !aligned_to(loss, 4) || !aligned_to(lse, 4) ||
      !aligned_to(count, 4))
    return OA_EALIGN;
  if (workspace_bytes < oa_linear_ce_workspace_bytes(tokens, hidden, vocab, 0, 0, 0))
    return OA_EINVAL;
  hipStream_t s = static_cast<hipStream_t>(stream);
  return dtype == OA_BF16 ? forward<Bf16>(h, reduction, loss, lse, count, workspace, s)
                          : forward<F16>(h, reduction, loss, lse, count, workspace, s);
}

extern "C" int oa_linear_ce_backward(const void* x, int64_t ldx, const void* w, int64_t ldw,
                                     int dtype, const int64_t* target, int64_t tokens,
                                     int64_t hidden, int64_t vocab, int64_t ignore_index,
                                     int reduction, const float* lse, const float* count,
                                     const float* grad, void* dx, void* dw, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  const Head h{static_cast<const uint8_t*>(x), static_cast<const uint8_t*>(w), ldx, ldw, target,
               tokens, hidden, vocab, ignore_index};
  int rc = check_head(h, dtype, reduction);
  if (rc) return rc;
  if (tokens == 0 || !lse || !count || !grad || !workspace || (!dx && !dw)) return OA_EINVAL;
  if (!aligned_to(workspace, 256) || !aligned_to(lse, 4) || !aligned_to(count, 4) ||
      !aligned_to(grad, 4) || !aligned_to(dx, 16) || !aligned_to(dw, 16))
    return OA_EALIGN;
  if (workspace_bytes <
      oa_linear_ce_workspace_bytes(tokens, hidden, vocab, 1, dx != nullptr, dw != nullptr))
    return OA_EINVAL;
  hipStream_t s = static_cast<hipStream_t>(stream);
  uint16_t *gx = static_cast<uint16_t*>(dx), *gw = static_cast<uint16_t*>(dw);
  return dtype == OA_BF16
             ? backward<Bf16>(h, reduction, lse, count, grad, gx, gw, workspace, s)
             : backward<F16>(h, reduction, lse, count, grad, gx, gw, workspace, s);
}
