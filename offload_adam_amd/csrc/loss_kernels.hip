// Softmax cross entropy of a linear head, z = x W^T, without ever holding z.
//
// Forward: the tiled product of oa_gemm.hpp with an epilogue that folds each
// token's tile of logits into a maximum and a sum of exponentials (one pair per token and
// tile) and picks out the target's logit; a second kernel joins the pairs into
// lse_t = log sum_v exp z[t,v] and the losses lse_t - z[t,y_t].
//
// Backward, in pieces of the vocabulary: the product again, with an epilogue that
// turns each logit into d[t,v] = exp(z[t,v] - lse_t) - [v = y_t] and stores it in 16
// bits; then dx += d W_piece (fp32) and dw_piece = d^T x, which read W, d and x as they
// lie (line by line along the dimension that is summed over).
//
// Bound by the matrix cores: 2 T V H operations forward, 6 T V H backward (z is
// computed again).  4096 tokens, 2048 hidden, 32000 words, bf16: 410 to 475 us forward;
// backward, in two pieces, each 213 to 260 for d, 182 to 230 for dx and 195 to 225 for dw, by
// the clock that power allows.  Logits, maxima, sums and the sums over tokens and vocabulary are
// fp32; lse_t is one fp32 number, which makes d off by 2^-24 of its magnitude; d is rounded once
// to the 16-bit type of x and W, which the products need and which a framework that stores the
// logits' gradient does too.

#include <math.h>

#include <type_traits>

#include "oa_gemm.hpp"

#pragma clang fp contract(off)

namespace oa {
namespace {

using namespace gemm;

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kCombineTokens = 8, kCombineParts = 32;
constexpr int kCombineThreads = kCombineTokens * kCombineParts;
constexpr int kReduceThreads = 1024;

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// exp(z - m) is exp2(fma(z, log2e, -at)) * unrounded(m, at) with at = m * log2e rounded: one
// fma per logit, and what the rounding of `at` makes of all of a token's exponentials (2^-24 of
// |m|) is taken back once.
__device__ __forceinline__ float unrounded(float m, float at) {
  return fabsf(at) < INFINITY ? exp2_hw(-fmaf(m, kLog2e, -at)) : 1.0f;
}

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

// A token's column among a lane's (kLines * u + i for element i of quad u), or -1.  Few
// tiles hold the target of any of their tokens, so what is done for it stays out of the
// loops over all logits.
template <class Tl>
__device__ __forceinline__ int column_of(int64_t rel) {
  return rel >= 0 && rel < Tl::kQuads * kLines && rel % kLines < 4 ? (int)rel : -1;
}
template <class Tl>
__device__ __forceinline__ float logit_at(const Tl& t, int b, int rel) {
  float z = 0.0f;
#pragma unroll
  for (int u = 0; u < Tl::kQuads; ++u)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (rel == kLines * u + i) z = t.quad(u, b)[i];
  return z;
}

// A lane's columns from `left` on hold no logit: their exponentials are 0.  `any`: the tile
// has such columns.
template <class Tl>
__device__ __forceinline__ void drop_columns(Tl& t, int64_t left, bool any) {
  if (!any) return;
#pragma unroll
  for (int u = 0; u < Tl::kQuads; ++u)
#pragma unroll
    for (int b = 0; b < Tl::kColumns; ++b) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (kLines * u + i >= left) t.acc[u][b][i] = -INFINITY;
      asm volatile("" : "+a"(t.acc[u][b]));  // stays where it is; the other registers are few
    }
}

// ------------------------------------------------------------------- forward

// Each token's maximum and sum of exponentials over the tile.  Per logit one fma, one
// exponential and an addition: 8 of the 52 us that a tile with 2048 of k takes.
struct StatsEpilogue {
  const int64_t* target;
  int64_t tokens, vocab;
  f32x2* part;      // [vocabulary tile][token]: maximum, sum
  float* z_target;  // [token]

  template <class Tl>
  __device__ __forceinline__ void operator()(Tl& t, int64_t row_q, int64_t row_p, const Place& place,
                                             uint8_t* lds) const {
    f32x2* all = reinterpret_cast<f32x2*>(lds);  // [wave along q][token of the tile]
    const int64_t v0 = row_q + t.q0();
    drop_columns(t, vocab - v0, row_q + Tl::BQ > vocab);
#pragma unroll
    for (int b = 0; b < Tl::kColumns; ++b) {
      const int64_t token = row_p + t.p0() + kLines * b;
      float m = -INFINITY;
#pragma unroll
      for (int u = 0; u < Tl::kQuads; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) m = fmaxf(m, t.quad(u, b)[i]);
      const float from = m == -INFINITY ? 0.0f : m, at = from * kLog2e;
      float s = 0.0f;
#pragma unroll
      for (int u = 0; u < Tl::kQuads; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) s += exp2_hw(fmaf(t.quad(u, b)[i], kLog2e, -at));
      s *= unrounded(from, at);
      const int64_t y = token < tokens ? target[token] : -1;
      const int rel = column_of<Tl>(y < vocab ? y - v0 : -1);
      if (__any(rel >= 0)) {
        const float hit = logit_at(t, b, rel);
        if (rel >= 0) z_target[token] = hit;
      }
      // the four lanes that hold this token's logits
      join(m, s, __shfl_xor(m, 16, kWave), __shfl_xor(s, 16, kWave));
      join(m, s, __shfl_xor(m, 32, kWave), __shfl_xor(s, 32, kWave));
      if (t.lane < kLines) all[t.wq * Tl::BP + t.p0() + kLines * b] = f32x2{m, s};
    }
    __syncthreads();
    for (int i = threadIdx.x; i < Tl::BP; i += Tl::kThreads) {
      f32x2 v = all[i];
      float m = v[0], s = v[1];
#pragma unroll
      for (int w = 1; w < Tl::kWavesQ; ++w) join(m, s, all[w * Tl::BP + i][0], all[w * Tl::BP + i][1]);
      if (row_p + i < tokens) part[(int64_t)place.tq * tokens + row_p + i] = f32x2{m, s};
    }
  }
};

struct Losses {
  const float* z_target;
  const int64_t* target;
  int64_t tokens, vocab, ignore;
  float *lse, *loss;  // loss: of every token, or NULL

  // A token whose logits have this maximum and sum: its loss, 0 if it takes no part.  A
  // target outside [0, vocab) that is not `ignore` makes it NaN.
  __device__ __forceinline__ float finish(int64_t token, float m, float s, bool& used) const {
    const float l = logf(s);
    lse[token] = m + l;
    const int64_t y = target[token];
    used = y != ignore;
    // the difference of the large ones first: l alone is as small as the loss may be
    const float v = !used ? 0.0f : y >= 0 && y < vocab ? m - z_target[token] + l : NAN;
    if (loss) loss[token] = v;
    return v;
  }
};

// This lane's share of a token's tiles.
__device__ __forceinline__ void join_tiles(const f32x2* part, int64_t tokens, int64_t token,
                                           int tiles, int row, float& m, float& s) {
  m = -INFINITY;
  s = 0.0f;
  if (token >= tokens) return;
#pragma unroll 4
  for (int j = row; j < tiles; j += kCombineParts) {
    const f32x2 v = part[(int64_t)j * tokens + token];
    join(m, s, v[0], v[1]);
  }
}

// Joins a token's tiles: 32 lanes per token, eight to a wave, then the lanes (a chain of
// loads and exponentials is what this takes: 8 us with 8 lanes per token and 125 tiles, 4
// with 32).
__global__ void __launch_bounds__(kCombineThreads)
ce_combine_kernel(const f32x2* __restrict__ part, const Losses a, int tiles,
                  float* __restrict__ block_sum, int* __restrict__ block_count) {
  __shared__ f32x2 all[kCombineThreads / kWave][kCombineTokens];
  const int col = threadIdx.x % kCombineTokens, row = threadIdx.x / kCombineTokens;
  const int64_t token = (int64_t)blockIdx.x * kCombineTokens + col;
  float m, s;
  join_tiles(part, a.tokens, token, tiles, row, m, s);
#pragma unroll
  for (int off = kCombineTokens; off < kWave; off <<= 1) {
    const float m2 = __shfl_xor(m, off, kWave), s2 = __shfl_xor(s, off, kWave);
    join(m, s, m2, s2);
  }
  if (threadIdx.x % kWave < kCombineTokens) all[threadIdx.x / kWave][col] = f32x2{m, s};
  __syncthreads();
  if (threadIdx.x >= kWave) return;
  float loss = 0.0f;
  bool used = false;
  if (threadIdx.x < kCombineTokens && token < a.tokens) {
#pragma unroll
    for (int w = 1; w < kCombineThreads / kWave; ++w) join(m, s, all[w][col][0], all[w][col][1]);
    loss = a.finish(token, m, s, used);
  }
  const float total = wave_sum(loss);
  const int count = __popcll(__ballot(used));
  if (threadIdx.x == 0) {
    block_sum[blockIdx.x] = total;
    block_count[blockIdx.x] = count;
  }
}

// The same and the sum over all tokens, of up to kFewLosses, 32 at a time: one launch
// instead of two where a launch is what counts.
constexpr int64_t kFewLosses = 128;
__global__ void __launch_bounds__(kReduceThreads)
ce_few_losses_kernel(const f32x2* __restrict__ part, const Losses a, int tiles, int mean,
                     float* __restrict__ loss_out, float* __restrict__ count_out) {
  constexpr int kTokens = kReduceThreads / kCombineParts;
  __shared__ f32x2 all[kReduceThreads / kWave][kTokens];
  const int col = threadIdx.x % kTokens, row = threadIdx.x / kTokens;
  float total = 0.0f, count = 0.0f;
  for (int64_t first = 0; first < a.tokens; first += kTokens) {
    float m, s;
    join_tiles(part, a.tokens, first + col, tiles, row, m, s);
    const float m2 = __shfl_xor(m, kTokens, kWave), s2 = __shfl_xor(s, kTokens, kWave);
    join(m, s, m2, s2);
    __syncthreads();
    if (threadIdx.x % kWave < kTokens) all[threadIdx.x / kWave][col] = f32x2{m, s};
    __syncthreads();
    if (row == 0 && first + col < a.tokens) {
#pragma unroll
      for (int w = 1; w < kReduceThreads / kWave; ++w) join(m, s, all[w][col][0], all[w][col][1]);
      bool used;
      total += a.finish(first + col, m, s, used);
      count += used ? 1.0f : 0.0f;
    }
  }
  if (threadIdx.x >= kWave) return;
  total = wave_sum(total);
  count = wave_sum(count);
  if (threadIdx.x != 0) return;
  *count_out = count;
  *loss_out = mean ? total / count : total;  // nothing took part: 0 / 0
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
  *loss_out = mean ? s / (float)c : s;  // nothing took part: 0 / 0
}

// ------------------------------------------------------------------ backward

// Factors of a token with gradient g.  One g for all (mean, sum), bf16: it goes into the
// fp32 sums, and d is stored as it is: the target's element, which often outweighs all
// others together, is then close to -1, which 16 bits hold exactly, where -g they do not
// (98 tokens, 31151 words, random logits, a sum times a random g: gradients off by 1.9e-3
// of their size, 1.7e-3 of it the rounding of the results, against 2.6e-3).  One g per
// token, bf16: d is stored times g, and everything else is 1.  fp16, whose smallest normal
// number (6e-5) is far above a probability times a gradient of 1 / tokens: g = top m 2^(a + b)
// with top the largest finite |g| of all tokens and 1/2 < |m| <= 1; d is stored times
// 2^15 m 2^a, x times 2^b, and the rest goes into the fp32 sums.  Both are exact but for
// fp16's smallest step, 2^-25 off at most: 2^(-40 - a) of d and 2^(-25 - b) of x.  So b goes
// down to -8 first, x then being exact from 2^-6 on, then a to -12, where the error of d
// is 2^-28 (of 131072 probabilities together no more than the rounding of the target's
// element), and b takes what is left under 2^-20.  (All of it in b left x four of its eleven
// bits at 2^-20.)
struct TokenFactors {
  float* d;   // of d as it is stored; 0: the token takes no part
  float* x;   // of x for dw
  float* dx;  // of the sum over v
  float* dw;  // one element: of the sum over t
};
constexpr float kF16Lift = 32768.0f;

struct Gradient {
  const float *grad, *count;
  const int64_t* target;
  int64_t tokens, vocab, ignore;
  int per_token, mean;

  __device__ __forceinline__ bool takes_part(int64_t token) const {
    return target[token] != ignore;
  }
  // NaN for a target that is none
  __device__ __forceinline__ float fault(int64_t token) const {
    const int64_t y = target[token];
    return y < 0 || y >= vocab ? NAN : 0.0f;
  }
};

// Factors, and x for dw: rows that take no part become zeros, whatever they hold.  Eight
// elements of x per lane; without `out`, one token.  Everything but fp16 with one gradient
// per token, whose factors depend on each other.
template <class T>
__global__ void __launch_bounds__(256)
ce_token_kernel(const Gradient a, const TokenFactors f, const uint16_t* __restrict__ x,
                int64_t ldx, int64_t hidden, uint16_t* __restrict__ out) {
  constexpr float kLift = std::is_same<T, F16>::value ? kF16Lift : 1.0f;
  const int64_t per_row = out ? hidden / 8 : 1;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= a.tokens * per_row) return;
  const int64_t token = i / per_row, c = i % per_row * 8;
  const bool used =
      a.takes_part(token) && !(a.per_token && a.grad[token] + a.fault(token) == 0.0f);
  if (c == 0) {
    float d = 0.0f, dx = 0.0f;
    if (used) {
      if (a.per_token) {
        d = a.grad[token] + a.fault(token);
        dx = 1.0f;
      } else {
        d = kLift + a.fault(token);
        dx = (a.mean ? a.grad[0] / *a.count : a.grad[0]) / kLift + a.fault(token);
      }
    }
    f.d[token] = d;
    f.dx[token] = dx;
  }
  if (i == 0) {
    float dw = 1.0f;
    // no token takes part: 0 times whatever the gradient is
    if (!a.per_token)
      dw = *a.count == 0.0f ? 0.0f : (a.mean ? a.grad[0] / *a.count : a.grad[0]) / kLift;
    *f.dw = dw;
  }
  if (!out) return;
  u32x4 w = {0u, 0u, 0u, 0u};
  if (used) w = *reinterpret_cast<const u32x4*>(x + token * ldx + c);
  *reinterpret_cast<u32x4*>(out + token * hidden + c) = w;
}

// fp16, one gradient per token.
__global__ void __launch_bounds__(kReduceThreads)
ce_factors_kernel(const Gradient a, const TokenFactors f) {
  __shared__ float tops[kReduceThreads / kWave];
  float top = 0.0f;
  for (int64_t i = threadIdx.x; i < a.tokens; i += kReduceThreads) {
    const float g = a.takes_part(i) ? a.grad[i] + a.fault(i) : 0.0f;
    f.d[i] = g;
    if (fabsf(g) < INFINITY) top = fmaxf(top, fabsf(g));
  }
  top = wave_max(top);
  if (threadIdx.x % kWave == 0) tops[threadIdx.x / kWave] = top;
  __syncthreads();
  for (int w = 0; w < kReduceThreads / kWave; ++w) top = fmaxf(top, tops[w]);
  if (top == 0.0f) top = 1.0f;
  if (threadIdx.x == 0) *f.dw = top / kF16Lift;
  // each lane goes over what it wrote itself
  for (int64_t i = threadIdx.x; i < a.tokens; i += kReduceThreads) {
    const float g = f.d[i];
    if (!(fabsf(g) < INFINITY)) {  // infinities and NaN stay in their row of dx
      f.d[i] = g;
      f.x[i] = f.dx[i] = 1.0f;
      continue;
    }
    int e = 0;
    float m = g == 0.0f ? 0.0f : frexpf(g / top, &e);
    if (fabsf(m) == 0.5f) {
      m *= 2.0f;
      e -= 1;
    }
    const int a = e > -8 ? 0 : e < -20 ? -12 : e + 8;
    const float power = ldexpf(1.0f, e - a);
    f.d[i] = ldexpf(m * kF16Lift, a);
    f.x[i] = m == 0.0f ? 0.0f : power;
    f.dx[i] = m == 0.0f ? 0.0f : top * power / kF16Lift;
  }
}

// d of the tile, 16 bits, through LDS to whole rows: 14 of 58 us with 2048 of k, of which the
// stores of all CUs at once (128 KB each) are 8.
template <class T>
struct ProbEpilogue {
  const int64_t* target;
  const float* lse;
  const float* factor;
  int64_t tokens, rows;  // rows of the piece
  int64_t first;         // its first vocabulary row
  uint16_t* d;           // [token][ld]
  int64_t ld;

  template <class Tl>
  __device__ __forceinline__ void operator()(Tl& t, int64_t row_q, int64_t row_p, const Place&,
                                             uint8_t* lds) const {
    const int64_t v0 = row_q + t.q0();
    drop_columns(t, rows - v0, row_q + Tl::BQ > rows);
    float h[Tl::kColumns], at[Tl::kColumns];
#pragma unroll
    for (int b = 0; b < Tl::kColumns; ++b) {
      const int64_t token = row_p + t.p0() + kLines * b;
      const bool here = token < tokens;
      const float l = here ? lse[token] : 0.0f;
      h[b] = here ? factor[token] : 0.0f;
      at[b] = l * kLog2e;
      if (h[b] != 0.0f) h[b] *= unrounded(l, at[b]);
    }
    auto p = [&](float z, int b) { return exp2_hw(fmaf(z, kLog2e, -at[b])); };
    t.rows16(
        lds,
        [&](int u, int b) {
          const f32x4 z = t.quad(u, b);
          const uint32_t lo = Store16<T>::pack(p(z[0], b) * h[b], p(z[1], b) * h[b]);
          const uint32_t hi = Store16<T>::pack(p(z[2], b) * h[b], p(z[3], b) * h[b]);
          // a token that takes no part: 0, whatever its logits are
          return u32x2{h[b] == 0.0f ? 0u : lo, h[b] == 0.0f ? 0u : hi};
        },
        [&] {  // 1 off the target's
#pragma unroll
          for (int b = 0; b < Tl::kColumns; ++b) {
            const int64_t token = row_p + t.p0() + kLines * b;
            const int64_t y = token < tokens ? target[token] - first : -1;
            const int rel = column_of<Tl>(y < rows ? y - v0 : -1);
            if (!__any(rel >= 0)) continue;
            const float z = logit_at(t, b, rel);
            if (rel >= 0 && h[b] != 0.0f) {
              const float one = p(z, b) * unrounded(lse[token], at[b]);  // or less
              t.put16(lds, rel, b,
                      (uint16_t)Store16<T>::pack((one - 1.0f) * factor[token], 0.0f));
            }
          }
        },
        [&](int p, int q, u32x4 v) {
          if (row_p + p < tokens) *reinterpret_cast<u32x4*>(d + (row_p + p) * ld + row_q + q) = v;
        });
  }
};

// dx of one piece, added to the pieces before it: [slice][token][hidden] fp32.
struct SumEpilogue {
  float* sum;
  int64_t tokens, hidden;
  int first;  // nothing is there yet

  template <class Tl>
  __device__ __forceinline__ void operator()(Tl& t, int64_t row_q, int64_t row_p, const Place& place,
                                             uint8_t* lds) const {
    float* base = sum + ((int64_t)place.slice * tokens + row_p) * hidden + row_q;
    t.rows32(lds, [&](int p, int q, f32x4 v) {
      if (row_p + p >= tokens || row_q + q >= hidden) return;  // hidden is a multiple of 8
      f32x4* o = reinterpret_cast<f32x4*>(base + p * hidden + q);
      *o = first ? v : *o + v;
    });
  }
};

// dx itself, where all of it is one product.
template <class T>
struct DxEpilogue {
  uint16_t* dx;
  int64_t tokens, hidden;
  const float* factor;

  template <class Tl>
  __device__ __forceinline__ void operator()(Tl& t, int64_t row_q, int64_t row_p, const Place&,
                                             uint8_t* lds) const {
    float f[Tl::kColumns];
#pragma unroll
    for (int b = 0; b < Tl::kColumns; ++b) {
      const int64_t token = row_p + t.p0() + kLines * b;
      f[b] = token < tokens ? factor[token] : 0.0f;
    }
    t.rows16(
        lds,
        [&](int u, int b) {
          const f32x4 v = t.quad(u, b) * f[b];
          const uint32_t lo = Store16<T>::pack(v[0], v[1]), hi = Store16<T>::pack(v[2], v[3]);
          return u32x2{f[b] == 0.0f ? 0u : lo, f[b] == 0.0f ? 0u : hi};
        },
        [] {},
        [&](int p, int q, u32x4 v) {
          if (row_p + p < tokens && row_q + q < hidden)
            *reinterpret_cast<u32x4*>(dx + (row_p + p) * hidden + row_q + q) = v;
        });
  }
};

template <class T>
struct WeightGradEpilogue {
  uint16_t* dw;
  int64_t rows, hidden;
  const float* factor;

  template <class Tl>
  __device__ __forceinline__ void operator()(Tl& t, int64_t row_q, int64_t row_p, const Place&,
                                             uint8_t* lds) const {
    const float f = *factor;
    t.rows16(
        lds,
        [&](int u, int b) {
          const f32x4 v = t.quad(u, b) * f;
          return u32x2{Store16<T>::pack(v[0], v[1]), Store16<T>::pack(v[2], v[3])};
        },
        [] {},
        [&](int p, int q, u32x4 v) {
          if (row_p + p < rows && row_q + q < hidden)
            *reinterpret_cast<u32x4*>(dw + (row_p + p) * hidden + row_q + q) = v;
        });
  }
};

// Slices of the fp32 sums -> dx in 16 bits, four elements per lane.
template <class T>
__global__ void __launch_bounds__(256)
ce_dx_kernel(const float* __restrict__ sum, int slices, const float* __restrict__ factor,
             int64_t tokens, int64_t hidden, uint16_t* __restrict__ dx) {
  const int64_t quads = tokens * hidden / 4;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= quads) return;
  const float f = factor[i * 4 / hidden];
  f32x4 v = reinterpret_cast<const f32x4*>(sum)[i];
#pragma unroll 8
  for (int s = 1; s < slices; ++s) v += reinterpret_cast<const f32x4*>(sum)[s * quads + i];
  v = f == 0.0f ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : v * f;
  reinterpret_cast<u32x2*>(dx)[i] =
      u32x2{Store16<T>::pack(v[0], v[1]), Store16<T>::pack(v[2], v[3])};
}

template <class T>
__device__ __forceinline__ void unpack(uint32_t w, float& a, float& b) {
  if (std::is_same<T, Bf16>::value) {
    a = bf16lo_to_f32(w);
    b = bf16hi_to_f32(w);
  } else {
    a = (float)__builtin_bit_cast(_Float16, (uint16_t)w);
    b = (float)__builtin_bit_cast(_Float16, (uint16_t)(w >> 16));
  }
}

// x for dw with factors: rows that take no part become zeros.  Eight elements per lane.
template <class T>
__global__ void __launch_bounds__(256)
ce_x_kernel(const uint16_t* __restrict__ x, int64_t ldx, const float* __restrict__ factor,
            int64_t tokens, int64_t hidden, uint16_t* __restrict__ out) {
  const int64_t per_row = hidden / 8;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= tokens * per_row) return;
  const int64_t token = i / per_row, c = i % per_row * 8;
  const float f = factor[token];
  u32x4 w = {0u, 0u, 0u, 0u};
  if (f != 0.0f) {
    w = *reinterpret_cast<const u32x4*>(x + token * ldx + c);
    if (f != 1.0f)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float a, b;
        unpack<T>(w[k], a, b);
        w[k] = Store16<T>::pack(a * f, b * f);
      }
  }
  *reinterpret_cast<u32x4*>(out + token * hidden + c) = w;
}

// --------------------------------------------------------------- host side

struct ForwardPlan {
  Cut cut;
  int tiles;
  int blocks;
  f32x2* part;
  float *z_target, *block_sum;
  int* block_count;
  size_t bytes;
  ForwardPlan(int64_t tokens, int64_t hidden, int64_t vocab, void* ws) {
    cut = cut_for(vocab, tokens > 0 ? tokens : 1, steps_of(hidden * 2), kNoSlices);
    tiles = (int)tiles_along(vocab, cut.large ? 256 : 128);
    blocks = (int)tiles_along(tokens, kCombineTokens);
    Carver c{static_cast<uint8_t*>(ws)};
    part = c.take<f32x2>((int64_t)tiles * tokens);
    z_target = c.take<float>(tokens);
    block_sum = c.take<float>(blocks);
    block_count = c.take<int>(blocks);
    bytes = c.used;
  }
};

// Elements of d that a piece of the vocabulary may hold: 64 Mi (128 MiB).  A larger
// piece saves passes over the fp32 sums of dx (one read and write per piece).  Its rows are
// limited too: the product for dw addresses 64 lines of d with 32 bits.
constexpr int64_t kPieceElems = (int64_t)64 << 20, kPieceRows = (int64_t)4 << 20;

struct BackwardPlan {
  int64_t piece;  // vocabulary rows of a piece, whole tiles
  Cut dx_cut;
  TokenFactors f;
  uint16_t *d, *x;
  float* sum;
  size_t bytes;
  BackwardPlan(int64_t tokens, int64_t hidden, int64_t vocab, bool want_dx, bool want_dw, void* ws) {
    const int64_t whole = up_to(vocab, 256);
    int64_t most = kPieceElems / tokens / 256 * 256;
    if (most < 256) most = 256;
    if (most > kPieceRows) most = kPieceRows;
    if (most > whole) most = whole;
    piece = up_to(tiles_along(whole, tiles_along(whole, most)), 256);
    dx_cut = cut_for(hidden, tokens, steps_of(piece * 2), kAllTiles);
    Carver c{static_cast<uint8_t*>(ws)};
    f.d = c.take<float>(tokens);
    f.x = c.take<float>(tokens);
    f.dx = c.take<float>(tokens);
    f.dw = c.take<float>(1);
    d = c.take<uint16_t>(tokens * piece);
    // one piece in one slice is dx as it stands
    sum = want_dx && (piece < vocab || dx_cut.slices > 1)
              ? c.take<float>(dx_cut.slices * tokens * hidden)
              : nullptr;
    x = want_dw ? c.take<uint16_t>(tokens * hidden) : nullptr;
    bytes = c.used;
  }
};

struct Head {
  const uint8_t *x, *w;
  int64_t ldx, ldw;  // elements
  const int64_t* target;
  int64_t tokens, hidden, vocab, ignore;
};

Problem logits_problem(const Head& h, int64_t first, int64_t rows) {
  Problem pr{};
  pr.q = Operand{h.w + first * h.ldw * 2, h.ldw * 2, rows, 0};
  pr.p = Operand{h.x, h.ldx * 2, h.tokens, 0};
  pr.k_bytes = (int)(h.hidden * 2);
  return pr;
}

template <class T>
int forward(const Head& h, int reduction, float* loss, float* lse, float* count, void* ws,
            hipStream_t s) {
  const ForwardPlan plan(h.tokens, h.hidden, h.vocab, ws);
  if (h.tokens > 0) {
    const StatsEpilogue e{h.target, h.tokens, h.vocab, plan.part, plan.z_target};
    int rc = launch_product<T, false, false>(logits_problem(h, 0, h.vocab), plan.cut, e, s);
    if (rc) return rc;
    const Losses a{plan.z_target, h.target, h.tokens, h.vocab, h.ignore, lse,
                   reduction == OA_LOSS_NONE ? loss : nullptr};
    if (reduction != OA_LOSS_NONE && h.tokens <= kFewLosses) {
      hipLaunchKernelGGL(ce_few_losses_kernel, dim3(1), dim3(kReduceThreads), 0, s, plan.part, a,
                         plan.tiles, reduction == OA_LOSS_MEAN, loss, count);
      return launch_status();
    }
    hipLaunchKernelGGL(ce_combine_kernel, dim3((unsigned)plan.blocks), dim3(kCombineThreads), 0, s,
                       plan.part, a, plan.tiles, plan.block_sum, plan.block_count);
    rc = launch_status();
    if (rc) return rc;
  }
  if (reduction == OA_LOSS_NONE) return 0;
  hipLaunchKernelGGL(ce_reduce_kernel, dim3(1), dim3(kReduceThreads), 0, s, plan.block_sum,
                     plan.block_count, plan.blocks, reduction == OA_LOSS_MEAN, loss, count);
  return launch_status();
}

template <class T>
int backward(const Head& h, int reduction, const float* lse, const float* count,
             const float* grad, uint16_t* dx, uint16_t* dw, void* ws, hipStream_t s) {
  const BackwardPlan plan(h.tokens, h.hidden, h.vocab, dx != nullptr, dw != nullptr, ws);
  const TokenFactors& f = plan.f;
  const Gradient a{grad, count, h.target, h.tokens, h.vocab, h.ignore,
                   reduction == OA_LOSS_NONE, reduction == OA_LOSS_MEAN};
  const uint16_t* x = reinterpret_cast<const uint16_t*>(h.x);
  const unsigned x_blocks = (unsigned)tiles_along(h.tokens * (dw ? h.hidden / 8 : 1), 256);
  const bool joint = std::is_same<T, F16>::value && reduction == OA_LOSS_NONE;
  if (joint)
    hipLaunchKernelGGL(ce_factors_kernel, dim3(1), dim3(kReduceThreads), 0, s, a, f);
  else
    hipLaunchKernelGGL(ce_token_kernel<T>, dim3(x_blocks), dim3(256), 0, s, a, f, x, h.ldx,
                       h.hidden, plan.x);
  int rc = launch_status();
  if (rc) return rc;
  if (joint && dw) {
    hipLaunchKernelGGL(ce_x_kernel<T>, dim3(x_blocks), dim3(256), 0, s, x, h.ldx, f.x, h.tokens,
                       h.hidden, plan.x);
    rc = launch_status();
    if (rc) return rc;
  }
  for (int64_t first = 0; first < h.vocab; first += plan.piece) {
    const int64_t rows = h.vocab - first < plan.piece ? h.vocab - first : plan.piece;
    const ProbEpilogue<T> pe{h.target, lse, f.d, h.tokens, rows, first, plan.d, plan.piece};
    rc = launch_product<T, false, false>(logits_problem(h, first, rows),
                                         cut_for(rows, h.tokens, steps_of(h.hidden * 2), kNoSlices), pe,
                                         s);
    if (rc) return rc;
    if (dx) {
      Problem px{};
      px.q = Operand{h.w + first * h.ldw * 2, h.ldw * 2, h.hidden, rows};
      px.p = Operand{reinterpret_cast<uint8_t*>(plan.d), plan.piece * 2, h.tokens, 0};
      px.k_bytes = (int)(up_to(rows, 8) * 2);
      if (plan.sum) {
        const SumEpilogue se{plan.sum, h.tokens, h.hidden, (int)(first == 0)};
        rc = launch_product<T, true, false>(px, plan.dx_cut, se, s);
      } else {
        const DxEpilogue<T> de{dx, h.tokens, h.hidden, f.dx};
        rc = launch_product<T, true, false>(px, plan.dx_cut, de, s);
      }
      if (rc) return rc;
    }
    if (dw) {
      Problem pw{};
      pw.q = Operand{reinterpret_cast<uint8_t*>(plan.x), h.hidden * 2, h.hidden, h.tokens};
      pw.p = Operand{reinterpret_cast<uint8_t*>(plan.d), plan.piece * 2, rows, h.tokens};
      pw.k_bytes = (int)(up_to(h.tokens, 8) * 2);
      const WeightGradEpilogue<T> we{dw + first * h.hidden, rows, h.hidden, f.dw};
      rc = launch_product<T, true, true>(
          pw, cut_for(h.hidden, rows, steps_of(pw.k_bytes), kNoSlices), we, s);
      if (rc) return rc;
    }
  }
  if (plan.sum) {
    const int64_t quads = h.tokens * h.hidden / 4;
    hipLaunchKernelGGL(ce_dx_kernel<T>, dim3((unsigned)tiles_along(quads, 256)), dim3(256), 0, s,
                       plan.sum, plan.dx_cut.slices, f.dx, h.tokens, h.hidden, dx);
    rc = launch_status();
  }
  return rc;
}

constexpr int64_t kMostTokens = 1 << 22, kMostHidden = 1 << 20, kMostVocab = 1 << 24;

int check_head(const Head& h, int dtype, int reduction) {
  if (dtype != OA_BF16 && dtype != OA_F16) return OA_EINVAL;
  if (reduction != OA_LOSS_NONE && reduction != OA_LOSS_MEAN && reduction != OA_LOSS_SUM)
    return OA_EINVAL;
  if (h.tokens < 0 || h.hidden <= 0 || h.vocab <= 0 || !h.w) return OA_EINVAL;
  if (h.tokens > 0 && (!h.x || !h.target)) return OA_EINVAL;
  if (h.ldw < h.hidden || h.ldx < h.hidden) return OA_EINVAL;
  if (h.hidden % 8 || h.ldx % 8 || h.ldw % 8 || !aligned_to(h.x, 16) || !aligned_to(h.w, 16) ||
      !aligned_to(h.target, 8))
    return OA_EALIGN;
  if (h.ldx > kMostHidden || h.ldw > kMostHidden || h.tokens > kMostTokens ||
      h.vocab > kMostVocab)
    return OA_ERANGE;
  return 0;
}

}  // namespace
}  // namespace oa

using namespace oa;

extern "C" size_t oa_linear_ce_workspace_bytes(int64_t tokens, int64_t hidden, int64_t vocab,
                                               int backward, int want_dx, int want_dw) {
  if (tokens < 0 || hidden <= 0 || vocab <= 0) return 0;
  if (tokens > kMostTokens || hidden > kMostHidden || vocab > kMostVocab) return 0;
  // never 0: the workspace of an empty batch is a valid pointer too
  if (!backward) return ForwardPlan(tokens, hidden, vocab, nullptr).bytes + 256;
  if (tokens == 0) return 0;
  return BackwardPlan(tokens, hidden, vocab, want_dx != 0, want_dw != 0, nullptr).bytes;
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
