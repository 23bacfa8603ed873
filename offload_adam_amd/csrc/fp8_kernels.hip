// 8-bit floating-point weights (e4m3 codes, one e8m0 scale per 128 x 128 block) and the
// linear layer on them.
//
// A scale is the smallest power of two that brings the largest magnitude of its block
// to 448 or less, so that scaling is exact and a code is one rounding of its element;
// the matrix instruction of gfx950 applies such scales by itself.  Elements that are
// not finite take no part in the scale and become NaN.
//
//   y  = xq wq^T     xq: blocks of 1 x 128 along the inputs      (T x K) (N x K)^T
//   dx = gq wq       gq: blocks of 1 x 128 along the outputs     (T x N) (N x K)
//   dw = gt^T xt     gt, xt: blocks of 128 x 1 along the tokens  (T x N)^T (T x K)
//
// Products accumulate in fp32 and are rounded once, to the type of x.  4096 tokens, 4096 ->
// 14336, bf16: forward 13 us to encode x and 206 to 230 for y (2.1 to 2.3 PFLOP/s); backward
// 60 to encode, 174 to 195 for dx, 193 to 230 for dw, by the clock that power allows.

#include <math.h>

#include <type_traits>

#include "oa_gemm.hpp"

#pragma clang fp contract(off)

namespace oa {
namespace {

using namespace gemm;

constexpr int kBlock = 128;
constexpr int kThreads = 256;  // 16 x 16 lanes, each 8 rows x 8 columns of a block
constexpr int kPatch = 8;

int64_t blocks_of(int64_t v) { return (v + kBlock - 1) / kBlock; }

template <int DT>
__device__ __forceinline__ float load1(const void* base, int64_t i) {
  if (DT == OA_F32) return static_cast<const float*>(base)[i];
  const uint16_t h = static_cast<const uint16_t*>(base)[i];
  return DT == OA_BF16 ? bf16_bits_to_f32(h) : (float)__builtin_bit_cast(_Float16, h);
}

// Vectors that are aligned to an element only: one access all the same.
typedef uint32_t u32x4_2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2_2 __attribute__((ext_vector_type(2), aligned(2)));
typedef float f32x4_4 __attribute__((ext_vector_type(4), aligned(4)));

// Eight elements as they lie in memory.
template <int DT>
struct Octet {
  static constexpr int kWords = DT == OA_F32 ? 2 : 1;
  u32x4 w[kWords];

  __device__ __forceinline__ void load(const void* base, int64_t i) {
    const uint8_t* p = static_cast<const uint8_t*>(base) + i * (DT == OA_F32 ? 4 : 2);
#pragma unroll
    for (int k = 0; k < kWords; ++k) {
      if (DT == OA_F32)
        w[k] = __builtin_bit_cast(u32x4, f32x4(*reinterpret_cast<const f32x4_4*>(p + 16 * k)));
      else
        w[k] = *reinterpret_cast<const u32x4_2*>(p + 16 * k);
    }
  }
  __device__ __forceinline__ float operator[](int k) const {
    if (DT == OA_F32) return __uint_as_float(w[k / 4 % kWords][k % 4]);
    const uint16_t h = (uint16_t)(w[0][k / 2 % 4] >> (16 * (k % 2)));
    return DT == OA_BF16 ? bf16_bits_to_f32(h) : (float)__builtin_bit_cast(_Float16, h);
  }
};

template <int DT>
__device__ __forceinline__ void load8(const void* base, int64_t i, float (&x)[8]) {
  Octet<DT> o;
  o.load(base, i);
#pragma unroll
  for (int k = 0; k < 8; ++k) x[k] = o[k];
}

template <int DT>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
  if (DT == OA_BF16) return f32x2_to_bf16x2_bits(a, b);
  const _Float16 lo = (_Float16)a, hi = (_Float16)b;
  return (uint32_t)__builtin_bit_cast(uint16_t, lo) |
         ((uint32_t)__builtin_bit_cast(uint16_t, hi) << 16);
}

template <int DT>
__device__ __forceinline__ void store1(void* base, int64_t i, float v) {
  if (DT == OA_F32) static_cast<float*>(base)[i] = v;
  else static_cast<uint16_t*>(base)[i] = (uint16_t)pack16<DT>(v, 0.0f);
}

template <int DT>
__device__ __forceinline__ void store4(void* base, int64_t i, f32x4 v) {
  if (DT == OA_F32) *reinterpret_cast<f32x4*>(static_cast<float*>(base) + i) = v;
  else
    *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(base) + i) =
        u32x2{pack16<DT>(v[0], v[1]), pack16<DT>(v[2], v[3])};
}

// e8m0 byte of a set whose largest finite magnitude is m: 448 = 1.75 * 2^8, so the
// exponent of m, one more if its mantissa is over 1.75, less 8; at least 2^-126, and 1
// for a set of zeros.
__device__ __forceinline__ uint32_t scale_of(float m) {
  const uint32_t u = __float_as_uint(m);
  const int b = (int)((u + 0x1FFFFFu) >> 23) - 8;
  return u == 0 ? 127u : (uint32_t)(b < 1 ? 1 : b);
}
// 1 / scale, exactly
__device__ __forceinline__ float down_of(uint32_t scale) {
  return __uint_as_float((254u - scale) << 23);
}
__device__ __forceinline__ float scale_value(uint32_t b) {
  return __uint_as_float(b == 0 ? 0x00400000u : b == 255 ? 0x7FC00000u : b << 23);
}

__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

// A matrix to encode: rows `stride` elements apart.
struct Source {
  const void* base;
  int64_t stride, rows, cols;
};

// Largest of 16 neighbouring lanes, in all of them.
__device__ __forceinline__ float max_of_16(float v) {
  auto other = [](float x, auto ctrl) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), decltype(ctrl)::value, 0xF,
                                                   0xF, true));
  };
  v = fmaxf(v, other(v, std::integral_constant<int, 0xB1>{}));   // 1 0 3 2 of each four
  v = fmaxf(v, other(v, std::integral_constant<int, 0x4E>{}));   // 2 3 0 1
  v = fmaxf(v, other(v, std::integral_constant<int, 0x141>{}));  // mirrored eights
  return fmaxf(v, other(v, std::integral_constant<int, 0x140>{}));  // mirrored sixteens
}

// One lane's 8 x 8 patch of block (br, bc): rows r .. r+7, columns c .. c+7 of it; what lies
// outside the source reads as zero.  `vec`: rows are 16-byte aligned, whole octets, and
// 128 of them span less than 2^31 bytes.  Else an octet is one load that may cross a line,
// and the last one of a row, if it is not whole, eight: a gradient of 5064 x 14085 in fp16
// to both kinds of codes takes 64 us, 91 with single elements throughout; 5064 x 14080, 59.
template <int DT>
__device__ __forceinline__ void load_patch(const Source& m, int64_t br, int64_t bc, int r, int c,
                                           bool vec, float (&v)[kPatch][kPatch]) {
  constexpr int kSize = DT == OA_F32 ? 4 : 2;
  const int64_t first = br * kBlock, left = m.rows - first, c0 = bc * kBlock + c;
  const int rows = left < kBlock ? (int)left : kBlock;
  Octet<DT> o[kPatch];
  if (vec) {
    const uint8_t* base = static_cast<const uint8_t*>(m.base) + first * m.stride * kSize;
    const int pitch = (int)m.stride * kSize;
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t*>(base), 0, (rows - 1) * pitch + (int)m.cols * kSize, 0x00020000);
    const int at = c0 < m.cols ? r * pitch + (int)c0 * kSize : kOut;
#pragma unroll
    for (int p = 0; p < kPatch; ++p)
#pragma unroll
      for (int k = 0; k < Octet<DT>::kWords; ++k)
        o[p].w[k] = __builtin_bit_cast(
            u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                       rsrc, r + p < rows ? at + p * pitch + 16 * k : kOut, 0, 0));
#pragma unroll
    for (int p = 0; p < kPatch; ++p)
#pragma unroll
      for (int j = 0; j < kPatch; ++j) v[p][j] = o[p][j];
  } else if (c0 + kPatch <= m.cols) {
    // rows past the end: some row that is there, and zeros in its place
#pragma unroll
    for (int p = 0; p < kPatch; ++p)
      o[p].load(m.base, (first + (r + p < rows ? r + p : 0)) * m.stride + c0);
#pragma unroll
    for (int p = 0; p < kPatch; ++p)
#pragma unroll
      for (int j = 0; j < kPatch; ++j) v[p][j] = r + p < rows ? o[p][j] : 0.0f;
  } else {
#pragma unroll
    for (int p = 0; p < kPatch; ++p)
#pragma unroll
      for (int j = 0; j < kPatch; ++j)
        v[p][j] = r + p < rows && c0 + j < m.cols
                      ? load1<DT>(m.base, (first + r + p) * m.stride + c0 + j)
                      : 0.0f;
  }
}

// Infinities of a patch as NaN: they have no code.
__device__ __forceinline__ void drop_infinities(float (&v)[kPatch][kPatch]) {
  float top = 0.0f;
#pragma unroll
  for (int p = 0; p < kPatch; ++p)
#pragma unroll
    for (int j = 0; j < kPatch; ++j) top = fmaxf(top, fabsf(v[p][j]));
  if (top == INFINITY) {
#pragma unroll
    for (int p = 0; p < kPatch; ++p)
#pragma unroll
      for (int j = 0; j < kPatch; ++j)
        if (fabsf(v[p][j]) == INFINITY) v[p][j] = NAN;
  }
}

// -------------------------------------------------------------- weight codec

// One workgroup per 128 x 128 block: one read of the source, one write of the codes.  Bound
// by HBM: 14336 x 4096, 57 us from fp32 (293 MB), 27 from bf16 (176 MB, part of them still
// in the memory-side cache).
template <int DT>
__global__ void __launch_bounds__(kThreads)
fp8_encode_kernel(const Source m, uint32_t blocks_c, bool vec, uint8_t* __restrict__ q,
                  uint8_t* __restrict__ scales) {
  __shared__ float tops[kThreads / kWave];
  const int64_t br = blockIdx.x / blocks_c, bc = blockIdx.x % blocks_c;
  const int r = threadIdx.x / 16 * kPatch, c = threadIdx.x % 16 * kPatch;
  const int64_t r0 = br * kBlock + r, c0 = bc * kBlock + c;
  float v[kPatch][kPatch];
  load_patch<DT>(m, br, bc, r, c, vec, v);
  drop_infinities(v);
  float top = 0.0f;
#pragma unroll
  for (int p = 0; p < kPatch; ++p)
#pragma unroll
    for (int j = 0; j < kPatch; ++j) top = fmaxf(top, fabsf(v[p][j]));
  top = wave_max(top);
  if (threadIdx.x % kWave == 0) tops[threadIdx.x / kWave] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / kWave; ++w) top = fmaxf(top, tops[w]);
  const uint32_t s = scale_of(top);
  const float down = down_of(s);
  if (threadIdx.x == 0) scales[blockIdx.x] = (uint8_t)s;
#pragma unroll
  for (int p = 0; p < kPatch; ++p) {
    if (r0 + p >= m.rows || c0 >= m.cols) continue;  // a multiple of 16 columns
    float* x = v[p];
    *reinterpret_cast<u32x2*>(q + (r0 + p) * m.cols + c0) =
        u32x2{encode4(x[0] * down, x[1] * down, x[2] * down, x[3] * down),
              encode4(x[4] * down, x[5] * down, x[6] * down, x[7] * down)};
  }
}

__device__ __forceinline__ void decode4(uint32_t w, float s, float* x) {
  const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
  const f32x2 b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  x[0] = a[0] * s;
  x[1] = a[1] * s;
  x[2] = b[0] * s;
  x[3] = b[1] * s;
}

// 16 codes per lane (cols is a multiple of 16: one row, one block).  14336 x 4096 to bf16:
// 28 us for 176 MB.
template <int DT>
__global__ void __launch_bounds__(kThreads)
fp8_decode_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ scales, int64_t rows,
                  int64_t cols, int64_t blocks_c, void* __restrict__ out, int64_t out_stride,
                  bool vec) {
  const int64_t per_row = cols / 16;
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (i >= rows * per_row) return;
  const int64_t r = i / per_row, c = i % per_row * 16;
  const float s = scale_value(scales[r / kBlock * blocks_c + c / kBlock]);
  const u32x4 w = *reinterpret_cast<const u32x4*>(q + r * cols + c);
  float x[16];
#pragma unroll
  for (int k = 0; k < 4; ++k) decode4(w[k], s, x + 4 * k);
  const int64_t o = r * out_stride + c;
  if (vec) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      store4<DT>(out, o + 4 * k, f32x4{x[4 * k], x[4 * k + 1], x[4 * k + 2], x[4 * k + 3]});
  } else {
    for (int k = 0; k < 16; ++k) store1<DT>(out, o + k, x[k]);
  }
}

// ----------------------------------------------------------- operand encoder

// A matrix [rows][cols] as operands of the products, in one read of it:
struct Encoded {
  uint8_t* q;        // codes [rows][ld], blocks of 1 x 128 along the columns
  uint8_t* scales;   // packed, rows x column blocks
  int64_t ld, scale_stride;
  uint8_t* qt;       // codes [cols][ld_t], blocks of 128 x 1 along the rows
  uint8_t* scales_t; // packed, cols x row blocks
  int64_t ld_t, scale_stride_t;
  float* sums;       // [row block][cols]: sums over 128 rows
  void* sum;         // [cols], in the type of the source: with one row block, instead
};

// One or two of them in a launch.
struct Operands {
  Source m[2];
  Encoded e[2];
  uint32_t blocks_c[2];
  bool vec[2];
  uint32_t first;  // workgroups of m[0]
};

// One workgroup per 128 x 128 block.  4096 x 14336 in bf16 to both kinds of codes: 52
// us for 235 MB.
template <int DT>
__global__ void __launch_bounds__(kThreads)
fp8_operand_kernel(const Operands all) {
  const bool second = blockIdx.x >= all.first;
  const Source m = second ? all.m[1] : all.m[0];
  const Encoded e = second ? all.e[1] : all.e[0];
  const uint32_t blocks_c = second ? all.blocks_c[1] : all.blocks_c[0];
  const uint32_t block = blockIdx.x - (second ? all.first : 0);
  const bool vec = second ? all.vec[1] : all.vec[0];
  constexpr int kWaves = kThreads / kWave;
  // [column][row], 16-byte pieces of a column at piece ^ (column / 16): lanes that write
  // together meet different banks
  __shared__ __align__(16) uint8_t tile[kBlock][kBlock + 16];
  __shared__ __align__(16) float part[kWaves][kBlock];
  const int64_t br = block / blocks_c, bc = block % blocks_c;
  const int wave = threadIdx.x / kWave, rg = threadIdx.x / 16, cg = threadIdx.x % 16;
  const int r = rg * kPatch, c = cg * kPatch;
  const int64_t r0 = br * kBlock + r, c0 = bc * kBlock + c;
  float v[kPatch][kPatch];
  load_patch<DT>(m, br, bc, r, c, vec, v);

  // one number per column of this lane's, from its rows, over the rows of the block
  auto over_rows = [&](float (&a)[kPatch], auto join) {
#pragma unroll
    for (int j = 0; j < kPatch; ++j) {
      a[j] = join(a[j], __shfl_xor(a[j], 16, kWave));
      a[j] = join(a[j], __shfl_xor(a[j], 32, kWave));
    }
    if (threadIdx.x % kWave < 16) {
#pragma unroll
      for (int j = 0; j < kPatch; j += 4)
        *reinterpret_cast<f32x4*>(&part[wave][c + j]) = f32x4{a[j], a[j + 1], a[j + 2], a[j + 3]};
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kPatch; j += 4) {
      f32x4 all = *reinterpret_cast<const f32x4*>(&part[0][c + j]);
#pragma unroll
      for (int w = 1; w < kWaves; ++w) {
        const f32x4 one = *reinterpret_cast<const f32x4*>(&part[w][c + j]);
#pragma unroll
        for (int i = 0; i < 4; ++i) all[i] = join(all[i], one[i]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) a[j + i] = all[i];
    }
  };
  if (e.sums || e.sum) {
    float s[kPatch];
#pragma unroll
    for (int j = 0; j < kPatch; ++j) {
      s[j] = 0.0f;
#pragma unroll
      for (int p = 0; p < kPatch; ++p) s[j] += v[p][j];
    }
    over_rows(s, [](float a, float b) { return a + b; });
    if (rg == 0) {
#pragma unroll
      for (int j = 0; j < kPatch; ++j)
        if (c0 + j < m.cols) {
          if (e.sum) store1<DT>(e.sum, c0 + j, s[j]);
          else e.sums[br * m.cols + c0 + j] = s[j];
        }
    }
    __syncthreads();
  }
  drop_infinities(v);
  if (e.q) {
#pragma unroll
    for (int p = 0; p < kPatch; ++p) {
      float top = 0.0f;
#pragma unroll
      for (int j = 0; j < kPatch; ++j) top = fmaxf(top, fabsf(v[p][j]));
      const uint32_t s = scale_of(max_of_16(top));
      const float down = down_of(s);
      if (r0 + p < m.rows) {
        const float* x = v[p];
        *reinterpret_cast<u32x2*>(e.q + (r0 + p) * e.ld + c0) =
            u32x2{encode4(x[0] * down, x[1] * down, x[2] * down, x[3] * down),
                  encode4(x[4] * down, x[5] * down, x[6] * down, x[7] * down)};
        if (cg == 0) e.scales[packed_scale_at(r0 + p, bc, e.scale_stride)] = (uint8_t)s;
      }
    }
  }
  if (!e.qt) return;
  float top[kPatch];
#pragma unroll
  for (int j = 0; j < kPatch; ++j) {
    top[j] = 0.0f;
#pragma unroll
    for (int p = 0; p < kPatch; ++p) top[j] = fmaxf(top[j], fabsf(v[p][j]));
  }
  over_rows(top, [](float a, float b) { return fmaxf(a, b); });
#pragma unroll
  for (int j = 0; j < kPatch; ++j) {
    const uint32_t s = scale_of(top[j]);
    const float d = down_of(s);
    if (rg == 0 && c0 + j < m.cols)
      e.scales_t[packed_scale_at(c0 + j, br, e.scale_stride_t)] = (uint8_t)s;
    *reinterpret_cast<u32x2*>(&tile[c + j][(rg / 2 ^ cg / 2) * 16 + rg % 2 * 8]) =
        u32x2{encode4(v[0][j] * d, v[1][j] * d, v[2][j] * d, v[3][j] * d),
              encode4(v[4][j] * d, v[5][j] * d, v[6][j] * d, v[7][j] * d)};
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int i = threadIdx.x + kThreads * k, col = i / 8, piece = i % 8;
    if (bc * kBlock + col < m.cols)
      *reinterpret_cast<u32x4*>(e.qt + (bc * kBlock + col) * e.ld_t + br * kBlock + piece * 16) =
          *reinterpret_cast<const u32x4*>(&tile[col][(piece ^ col / 16) * 16]);
  }
}

// The row operand alone (codes in blocks of 1 x 128 along the columns): 16 lanes to a
// block, eight elements to a lane, columns from `cols` up to e.ld zero.  4096 x 4096 in bf16:
// 13 us for 50 MB; 16384 x 14336: 130 us for 705 MB.
template <int DT>
__global__ void __launch_bounds__(kThreads)
fp8_rows_kernel(const Source m, const Encoded e) {
  const int64_t per_row = e.ld / kPatch;
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int64_t r = i / per_row, c = i % per_row * kPatch;
  if (r >= m.rows) return;  // 16 lanes together: rows are whole blocks long
  float x[kPatch] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
  if (c < m.cols) load8<DT>(m.base, r * m.stride + c, x);  // whole octets
  float top = 0.0f;
#pragma unroll
  for (int j = 0; j < kPatch; ++j) {
    if (fabsf(x[j]) == INFINITY) x[j] = NAN;
    top = fmaxf(top, fabsf(x[j]));
  }
  const uint32_t s = scale_of(max_of_16(top));
  const float down = down_of(s);
  *reinterpret_cast<u32x2*>(e.q + r * e.ld + c) =
      u32x2{encode4(x[0] * down, x[1] * down, x[2] * down, x[3] * down),
            encode4(x[4] * down, x[5] * down, x[6] * down, x[7] * down)};
  if (threadIdx.x % 16 == 0) e.scales[packed_scale_at(r, c / kBlock, e.scale_stride)] = (uint8_t)s;
}

// Column sums: the row blocks' sums in order.
template <int DT>
__global__ void __launch_bounds__(kThreads)
fp8_column_sum_kernel(const float* __restrict__ sums, int64_t blocks_r, int64_t cols,
                      void* __restrict__ out) {
  const int64_t c = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (c >= cols) return;
  float s = 0.0f;
  for (int64_t b = 0; b < blocks_r; ++b) s += sums[b * cols + c];
  store1<DT>(out, c, s);
}

// ------------------------------------------------------------------ products

// The product, plus the bias of its columns, in the caller's type.  Whole octets of a row
// are one store, aligned or not: 5064 x 14085 x 240 takes 52 us, 136 with single elements
// for rows that are not aligned; 5064 x 14080 x 240, 47.
template <int DT>
struct StoreEpilogue {
  void* out;
  int64_t rows, cols;  // p, q
  const void* bias;    // by q, or NULL

  template <class Tl>
  __device__ __forceinline__ void operator()(Tl& t, int64_t row_q, int64_t row_p, const Place&,
                                             uint8_t* lds) const {
    if (bias) {
#pragma unroll
      for (int u = 0; u < Tl::kQuads; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int64_t q = row_q + t.q0() + kLines * u + i;
          const float add = q < cols ? load1<DT>(bias, q) : 0.0f;
#pragma unroll
          for (int b = 0; b < Tl::kColumns; ++b) t.acc[u][b][i] += add;
        }
    }
    if constexpr (DT == OA_F32) {
      t.rows32(lds, [&](int p, int q, f32x4 v) {
        if (row_p + p >= rows) return;
        float* o = static_cast<float*>(out) + (row_p + p) * cols + row_q + q;
        if (row_q + q + 4 <= cols) *reinterpret_cast<f32x4_4*>(o) = v;
        else
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (row_q + q + i < cols) o[i] = v[i];
      });
    } else {
      t.rows16(
          lds,
          [&](int u, int b) {
            const f32x4 v = t.quad(u, b);
            return u32x2{pack16<DT>(v[0], v[1]), pack16<DT>(v[2], v[3])};
          },
          [] {},
          [&](int p, int q, u32x4 v) {
            if (row_p + p >= rows) return;
            uint16_t* o = static_cast<uint16_t*>(out) + (row_p + p) * cols + row_q + q;
            if (row_q + q + 8 <= cols) *reinterpret_cast<u32x4_2*>(o) = v;
            else
#pragma unroll
              for (int i = 0; i < 8; ++i)
                if (row_q + q + i < cols) o[i] = (uint16_t)(v[i / 2] >> (16 * (i % 2)));
          });
    }
  }
};

// The same where some tiles are cut along k: their slices go to fp32 tiles of their own,
// [number of the tile][slice][row][column], with as many rows as there are when those are
// less than a tile's.
template <int DT>
struct CutEpilogue {
  StoreEpilogue<DT> whole;
  float* part;
  int slices, area;  // of a slice's tile, elements

  template <class Tl>
  __device__ __forceinline__ void operator()(Tl& t, int64_t row_q, int64_t row_p,
                                             const Place& place, uint8_t* lds) const {
    if (place.slice < 0) {
      whole(t, row_q, row_p, place, lds);
      return;
    }
    float* out = part + ((int64_t)place.number * slices + place.slice) * area;
    t.rows32(lds, [&](int p, int q, f32x4 v) {
      if (row_p + p < whole.rows && row_q + q < whole.cols)
        *reinterpret_cast<f32x4*>(out + p * Tl::BQ + q) = v;
    });
  }
};

// ---- few tokens.  Bound by reading the weight once.  A workgroup makes 16 columns of y;
// each of its waves takes every WAVES-th step of k, its fragments straight from memory to
// registers (16 rows of 128 bytes each), two or four steps ahead of the products, so that
// the loads of all waves of a CU cover the latency, multiplies them with all the tokens, one or
// two tiles of 16, and the waves' sums meet in LDS, in order.  ENCODE: x comes as it is
// and every workgroup makes the codes for itself, in LDS, while its weights are on the way.
template <int DT>
struct Few {
  const uint8_t *w, *ws;
  int64_t out_f;
  int in_f, blocks_k;
  Source x;            // ENCODE
  const uint8_t *xq, *xs;  // else
  int64_t ldx;         // of the codes
  int64_t xs_stride;
  int tokens;
  const void* bias;
  void* y;
};

constexpr int kFewCodes = 16384, kFewEncodeTokens = 16;  // ENCODE: codes, and tokens, at most

template <int DT, int TILES, int WAVES, bool ENCODE>
__global__ void __launch_bounds__(WAVES* kWave) fp8_few_kernel(const Few<DT> a) {
  static_assert(!ENCODE || TILES == 1, "a workgroup encodes the tokens of one tile");
  constexpr int kLanes = WAVES * kWave;
  constexpr int kFewAhead = ENCODE ? 4 : 2;  // codes of x on their way take registers too
  constexpr int kPieces = ENCODE ? kFewCodes / kPatch / kLanes : 1;
  __shared__ __align__(16) float sums[WAVES][TILES][kLines][kLines + 4];  // [token][column]
  __shared__ __align__(16) uint8_t codes[ENCODE ? kFewCodes : 16];
  __shared__ uint8_t scales[ENCODE ? kFewCodes / kBlock : 1];
  const int lane = threadIdx.x % kWave;
  // the same in all lanes, and known to be: a matrix instruction does not look at which
  // lanes are switched off
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int64_t n0 = (int64_t)blockIdx.x * kLines;
  const int r = lane % kLines, k0 = lane / kLines * 32;
  // What is not there reads as zero by the descriptors' ranges, without a branch: behind one
  // the compiler does not know how many loads are on their way, and waits for all.
  const int rows = a.out_f - n0 < kLines ? (int)(a.out_f - n0) : kLines;
  const auto w_rsrc = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint8_t*>(a.w + n0 * a.in_f), 0, rows * a.in_f, 0x00020000);
  const auto ws_rsrc = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint8_t*>(a.ws + n0 / kBlock * a.blocks_k), 0, a.blocks_k, 0x00020000);
  const auto xq_rsrc = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint8_t*>(a.xq), 0, a.tokens * (int)a.ldx, 0x00020000);
  const auto xs_rsrc = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint8_t*>(a.xs), 0, a.blocks_k * (int)a.xs_stride, 0x00020000);
  auto load16 = [](auto rsrc, int at) {
    return __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, at, 0, 0));
  };
  f32x4 acc[TILES];
#pragma unroll
  for (int t = 0; t < TILES; ++t) acc[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  Octet<DT> x[kPieces];
  const int per_row = (int)a.ldx / kPatch;
  if (ENCODE) {
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
      const int i = threadIdx.x + j * kLanes;
      const int token = i / per_row, c = i % per_row * kPatch;
      x[j] = Octet<DT>{};
      if (token >= a.tokens) continue;
      if (c < a.in_f) x[j].load(a.x.base, token * a.x.stride + c);
    }
  }
  auto fetch = [&](int step, i32x8& q, int& sq, i32x8 (&p)[TILES], int (&sp)[TILES]) {
    const int k = step * kStepBytes + k0;
    const i32x4 lo = load16(w_rsrc, k < a.in_f ? r * a.in_f + k : kOut);
    const i32x4 hi = load16(w_rsrc, k + 16 < a.in_f ? r * a.in_f + k + 16 : kOut);
    q = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    sq = __builtin_amdgcn_raw_buffer_load_b8(ws_rsrc, step, 0, 0);
    if constexpr (!ENCODE) {
#pragma unroll
      for (int t = 0; t < TILES; ++t) {
        const int token = t * kLines + r;
        const bool in = step < a.blocks_k && token < a.tokens;  // rows are whole steps long
        const int at = in ? token * (int)a.ldx + k : kOut;
        p[t] = __builtin_shufflevector(load16(xq_rsrc, at), load16(xq_rsrc, at + 16), 0, 1, 2, 3,
                                       4, 5, 6, 7);
        sp[t] = __builtin_amdgcn_raw_buffer_load_b8(
            xs_rsrc, in ? (int)packed_scale_at(token, step, a.xs_stride) : kOut, 0, 0);
      }
    }
  };
  i32x8 q[kFewAhead], p[kFewAhead][TILES];
  int sq[kFewAhead], sp[kFewAhead][TILES];
#pragma unroll
  for (int i = 0; i < kFewAhead; ++i) fetch(wave + i * WAVES, q[i], sq[i], p[i], sp[i]);

  if (ENCODE) {
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
      const int i = threadIdx.x + j * kLanes;
      if (j * kLanes >= a.tokens * per_row) break;
      float v[kPatch], top = 0.0f;
#pragma unroll
      for (int e = 0; e < kPatch; ++e) {
        v[e] = fabsf(x[j][e]) == INFINITY ? NAN : x[j][e];
        top = fmaxf(top, fabsf(v[e]));
      }
      const uint32_t s = scale_of(max_of_16(top));
      const float d = down_of(s);
      *reinterpret_cast<u32x2*>(codes + i * kPatch) =
          u32x2{encode4(v[0] * d, v[1] * d, v[2] * d, v[3] * d),
                encode4(v[4] * d, v[5] * d, v[6] * d, v[7] * d)};
      if (i % 16 == 0) scales[i / 16] = (uint8_t)s;
    }
    __syncthreads();
  }
  for (int step = wave; step < a.blocks_k; step += kFewAhead * WAVES) {
#pragma unroll
    for (int i = 0; i < kFewAhead; ++i) {
      const int at = step + i * WAVES;
      if constexpr (ENCODE) {
        const bool in = at < a.blocks_k && r < a.tokens;
        const uint8_t* c = codes + (in ? r * (int)a.ldx + at * kStepBytes + k0 : 0);
        const i32x4 lo = *reinterpret_cast<const i32x4*>(c);
        const i32x4 hi = *reinterpret_cast<const i32x4*>(c + 16);
        const int s = scales[in ? r * a.blocks_k + at : 0];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          p[i][0][j] = in ? lo[j] : 0;
          p[i][0][4 + j] = in ? hi[j] : 0;
        }
        sp[i][0] = in ? s : 0;
      }
      // steps past the last: zeros
#pragma unroll
      for (int t = 0; t < TILES; ++t)
        acc[t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(q[i], p[i][t], acc[t], 0, 0, 0,
                                                                  sq[i], 0, sp[i][t]);
      fetch(at + kFewAhead * WAVES, q[i], sq[i], p[i], sp[i]);
    }
  }
#pragma unroll
  for (int t = 0; t < TILES; ++t) {
    asm volatile("" : "+v"(acc[t]));  // here, on every lane
    *reinterpret_cast<f32x4*>(&sums[wave][t][r][lane / kLines * 4]) = acc[t];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < TILES * kLines * kLines; i += kLanes) {
    const int token = i / kLines, c = i % kLines;
    if (token >= a.tokens || n0 + c >= a.out_f) continue;
    float v = 0.0f;
#pragma unroll
    for (int g = 0; g < WAVES; ++g) v += sums[g][token / kLines][token % kLines][c];
    if (a.bias) v += load1<DT>(a.bias, n0 + c);
    store1<DT>(a.y, token * a.out_f + n0 + c, v);
  }
}

template <int DT, int TILES, bool ENCODE>
void launch_few(const Few<DT>& a, int waves, hipStream_t s) {
  const dim3 grid((unsigned)tiles_along(a.out_f, kLines)), block(waves * kWave);
  if (waves == 4)
    hipLaunchKernelGGL((fp8_few_kernel<DT, TILES, 4, ENCODE>), grid, block, 0, s, a);
  else
    hipLaunchKernelGGL((fp8_few_kernel<DT, TILES, 8, ENCODE>), grid, block, 0, s, a);
}

// Slices of the cut tiles -> results, four columns of a row per lane.
template <int DT>
__global__ void __launch_bounds__(kThreads)
fp8_join_kernel(const CutEpilogue<DT> e, int side, uint32_t first, uint32_t tiles_p,
                uint32_t tiles_q) {
  const uint32_t per_tile = (uint32_t)((e.area / 4 + kThreads - 1) / kThreads);
  const uint32_t number = blockIdx.x / per_tile;
  const int i = (int)((blockIdx.x - number * per_tile) * kThreads + threadIdx.x) * 4;
  uint32_t tp, tq;
  tile_at(first + number, tiles_p, tiles_q, tp, tq);
  const int64_t row = (int64_t)tp * side + i / side, col = (int64_t)tq * side + i % side;
  if (i >= e.area || row >= e.whole.rows || col >= e.whole.cols) return;
  const float* part = e.part + (int64_t)number * e.slices * e.area + i;
  f32x4 v = *reinterpret_cast<const f32x4*>(part);
#pragma unroll 8
  for (int s = 1; s < e.slices; ++s)
    v += *reinterpret_cast<const f32x4*>(part + (int64_t)s * e.area);
  const int64_t at = row * e.whole.cols + col;
  const int left = e.whole.cols - col < 4 ? (int)(e.whole.cols - col) : 4;
  if (e.whole.bias) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < left) v[k] += load1<DT>(e.whole.bias, col + k);
  }
  if (left < 4) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < left) store1<DT>(e.whole.out, at + k, v[k]);
  } else if constexpr (DT == OA_F32) {
    *reinterpret_cast<f32x4_4*>(static_cast<float*>(e.whole.out) + at) = v;
  } else {
    *reinterpret_cast<u32x2_2*>(static_cast<uint16_t*>(e.whole.out) + at) =
        u32x2{pack16<DT>(v[0], v[1]), pack16<DT>(v[2], v[3])};
  }
}

// A product's rows and columns, how it is cut, and the partial sums of its slices.
struct Output {
  int64_t rows = 0, cols = 0, tiles_p = 0, tiles_q = 0, side = 0;
  Cut cut{false, 1, 0};
  float* part = nullptr;
  Output() {}
  Output(int64_t rows_, int64_t cols_, int64_t k_bytes, Carver& c) : rows(rows_), cols(cols_) {
    cut = cut_for(cols, rows, steps_of(k_bytes), kLastTiles);
    side = cut.large ? 256 : 128;
    tiles_p = tiles_along(rows, side);
    tiles_q = tiles_along(cols, side);
    if (cut.slices > 1) part = c.take<float>(cut_tiles() * cut.slices * area());
  }
  int64_t cut_tiles() const { return tiles_p * tiles_q - cut.whole; }
  int64_t area() const { return side * (rows < side ? rows : side); }
};

template <int DT, bool Q_PACKED, bool Q_LINES>
int multiply(const Problem& pr, const Output& o, const void* bias, void* out, hipStream_t s) {
  typedef E4m3<Q_PACKED> T;
  const StoreEpilogue<DT> whole{out, o.rows, o.cols, bias};
  if (o.cut.slices == 1) return launch_product<T, Q_LINES, false>(pr, o.cut, whole, s);
  const CutEpilogue<DT> e{whole, o.part, o.cut.slices, (int)o.area()};
  int rc = launch_product<T, Q_LINES, false>(pr, o.cut, e, s);
  if (rc) return rc;
  const int64_t blocks = o.cut_tiles() * tiles_along(o.area() / 4, kThreads);
  hipLaunchKernelGGL(fp8_join_kernel<DT>, dim3((unsigned)blocks), dim3(kThreads), 0, s, e,
                     (int)o.side, (uint32_t)o.cut.whole, (uint32_t)o.tiles_p, (uint32_t)o.tiles_q);
  return launch_status();
}

bool vector_rows(const Source& m, int dtype) {
  const int64_t per = dtype == OA_F32 ? 4 : 8;
  return m.cols % 8 == 0 && m.stride % per == 0 && m.stride < (1 << 21) && m.cols < (1 << 21) &&
         aligned_to(m.base, 16);
}

template <int DT>
int encode_operands(int count, const Source* const* m, const Encoded* const* e, hipStream_t s) {
  Operands all{};
  int64_t blocks = 0;
  for (int i = 0; i < count; ++i) {
    all.m[i] = *m[i];
    all.e[i] = *e[i];
    all.blocks_c[i] = (uint32_t)blocks_of(m[i]->cols);
    all.vec[i] = vector_rows(*m[i], DT);
    blocks += blocks_of(m[i]->cols) * blocks_of(m[i]->rows);
    if (i == 0) all.first = (uint32_t)blocks;
  }
  if (blocks > 0x7FFFFFFF) return OA_ERANGE;
  hipLaunchKernelGGL(fp8_operand_kernel<DT>, dim3((unsigned)blocks), dim3(kThreads), 0, s, all);
  return launch_status();
}

template <int DT>
int encode_rows(const Source& m, const Encoded& e, hipStream_t s) {
  const int64_t lanes = m.rows * (e.ld / kPatch);
  hipLaunchKernelGGL(fp8_rows_kernel<DT>, dim3((unsigned)((lanes + kThreads - 1) / kThreads)),
                     dim3(kThreads), 0, s, m, e);
  return launch_status();
}

struct Layer {
  const uint8_t *q, *scales;
  int64_t out_f, in_f;
};

// Whether the kernel for few tokens takes a call.  It reads every token's codes once per 16
// columns, the tiles once per 128, but those take two more launches and half the bytes they
// move in LDS are for rows that hold no token.  Weights that come from HBM, bf16: 14336 -> 4096,
// 13 and 21 us for 1 and 16 tokens, 23 and 24 with tiles; 4096 -> 14336, 14 and 22 against 22
// and 22; beyond 16 tokens, 4096 -> 14336, 27 against 20 for 24, but a small weight gains for
// longer: 4096 -> 4096, 10 against 13.  Only very wide weights turn earlier: 4096 -> 128256,
// 101 against 114 for 4 tokens, 124 against 114 for 8.
bool takes_few(const Layer& w, int64_t tokens) {
  return tokens <= kLines || (tokens <= 2 * kLines && w.out_f * w.in_f <= (1 << 24));
}
// Waves of its workgroups: a CU that has only one of them needs more loads in flight from
// it.  4 / 8 waves, weights that come from HBM, bf16, 1 token: 4096 -> 14336, 14.4, 14.3 us;
// 2048 -> 5632, 5.5, 6.3; 4096 -> 4096, 6.3, 6.0; 14336 -> 4096, 13.4, 13.2; 2 tokens there,
// 19.3, 16.0; 8 tokens: 4096 -> 14336, 19.7, 21.1; 14336 -> 4096, 19.9, 18.2.
int few_waves(const Layer& w) { return tiles_along(w.out_f, kLines) > 256 ? 4 : 8; }

struct ForwardPlan {
  Encoded x{};
  Output y;
  size_t bytes;
  ForwardPlan(int64_t tokens, int64_t in_f, int64_t out_f, bool few, void* ws) {
    Carver c{static_cast<uint8_t*>(ws)};
    x.ld = up_to(in_f, kBlock);
    x.scale_stride = up_to(tokens, 256);
    x.q = c.take<uint8_t>(tokens * x.ld);
    x.scales = c.take<uint8_t>(blocks_of(in_f) * x.scale_stride);
    if (!few) y = Output(tokens, out_f, in_f, c);
    bytes = c.used;
  }
};

template <int DT>
int forward(const Source& x, const Layer& w, const void* bias, void* y, void* ws, hipStream_t s) {
  const bool few = takes_few(w, x.rows);
  const ForwardPlan plan(x.rows, w.in_f, w.out_f, few, ws);
  if (few) {
    const int tokens = (int)x.rows;
    const bool encode = tokens <= kFewEncodeTokens && tokens * plan.x.ld <= kFewCodes;
    const int waves = few_waves(w);
    const Few<DT> a{w.q, w.scales, w.out_f, (int)w.in_f, (int)blocks_of(w.in_f),
                    x, plan.x.q, plan.x.scales, plan.x.ld,
                    plan.x.scale_stride, tokens, bias, y};
    if (encode) {
      launch_few<DT, 1, true>(a, waves, s);
      return launch_status();
    }
    const int rc = encode_rows<DT>(x, plan.x, s);
    if (rc) return rc;
    if (tokens <= kLines) launch_few<DT, 1, false>(a, waves, s);
    else launch_few<DT, 2, false>(a, waves, s);
    return launch_status();
  }
  int rc = encode_rows<DT>(x, plan.x, s);
  if (rc) return rc;
  Problem pr{};
  pr.q = Operand{w.q, w.in_f, w.out_f, 0};
  pr.p = Operand{plan.x.q, plan.x.ld, x.rows, 0};
  pr.sq = Scales{w.scales, 1, blocks_of(w.in_f), blocks_of(w.out_f)};
  pr.sp = Scales{plan.x.scales, plan.x.scale_stride, 0, 0};
  pr.k_bytes = (int)w.in_f;
  return multiply<DT, false, false>(pr, plan.y, bias, y, s);
}

struct BackwardPlan {
  Encoded g{}, x{};
  Output dx, dw;
  size_t bytes;
  BackwardPlan(int64_t tokens, int64_t in_f, int64_t out_f, bool want_dx, bool want_dw,
               bool want_db, void* ws) {
    Carver c{static_cast<uint8_t*>(ws)};
    const int64_t padded_t = up_to(tokens, kBlock), padded_n = up_to(out_f, kBlock);
    if (want_dx) {
      g.ld = padded_n;
      g.scale_stride = up_to(tokens, 256);
      g.q = c.take<uint8_t>(tokens * g.ld);
      g.scales = c.take<uint8_t>(blocks_of(out_f) * g.scale_stride);
      dx = Output(tokens, in_f, padded_n, c);
    }
    if (want_dw) {
      g.ld_t = x.ld_t = padded_t;
      g.scale_stride_t = up_to(out_f, 256);
      x.scale_stride_t = up_to(in_f, 256);
      g.qt = c.take<uint8_t>(out_f * padded_t);
      g.scales_t = c.take<uint8_t>(blocks_of(tokens) * g.scale_stride_t);
      x.qt = c.take<uint8_t>(in_f * padded_t);
      x.scales_t = c.take<uint8_t>(blocks_of(tokens) * x.scale_stride_t);
      dw = Output(out_f, in_f, padded_t, c);
    }
    if (want_db && tokens > kBlock) g.sums = c.take<float>(blocks_of(tokens) * out_f);
    bytes = c.used;
  }
};

template <int DT>
int backward(const Source& g, const Source& x, const Layer& w, void* dx, void* dw, void* db,
             void* ws, hipStream_t s) {
  BackwardPlan plan(g.rows, w.in_f, w.out_f, dx != nullptr, dw != nullptr, db != nullptr, ws);
  if (!plan.g.sums) plan.g.sum = db;
  const Source* sources[2] = {&g, &x};
  const Encoded* codes[2] = {&plan.g, &plan.x};
  int rc = encode_operands<DT>(dw ? 2 : 1, sources, codes, s);
  if (rc) return rc;
  if (dx) {
    // the weight as it lies: line by line along the outputs, which are summed over
    const int64_t bc = blocks_of(w.in_f);
    Problem pr{};
    pr.q = Operand{w.q, w.in_f, w.in_f, w.out_f};
    pr.p = Operand{plan.g.q, plan.g.ld, g.rows, 0};
    pr.sq = Scales{w.scales, bc, 1, bc};
    pr.sp = Scales{plan.g.scales, plan.g.scale_stride, 0, 0};
    pr.k_bytes = (int)plan.g.ld;
    rc = multiply<DT, false, true>(pr, plan.dx, nullptr, dx, s);
    if (rc) return rc;
  }
  if (dw) {
    Problem pr{};
    pr.q = Operand{plan.x.qt, plan.x.ld_t, w.in_f, 0};
    pr.p = Operand{plan.g.qt, plan.g.ld_t, w.out_f, 0};
    pr.sq = Scales{plan.x.scales_t, plan.x.scale_stride_t, 0, 0};
    pr.sp = Scales{plan.g.scales_t, plan.g.scale_stride_t, 0, 0};
    pr.k_bytes = (int)plan.x.ld_t;
    rc = multiply<DT, true, false>(pr, plan.dw, nullptr, dw, s);
    if (rc) return rc;
  }
  if (plan.g.sums) {
    hipLaunchKernelGGL(fp8_column_sum_kernel<DT>,
                       dim3((unsigned)((w.out_f + kThreads - 1) / kThreads)), dim3(kThreads), 0, s,
                       plan.g.sums, blocks_of(g.rows), w.out_f, db);
    rc = launch_status();
  }
  return rc;
}

bool known(int dtype) { return dtype == OA_F32 || dtype == OA_BF16 || dtype == OA_F16; }
uintptr_t size_of(int dtype) { return dtype == OA_F32 ? 4 : 2; }

constexpr int64_t kMostRows = (int64_t)1 << 22;  // of an operand; also its longest row

int check_codec(const void* q, const void* scales, int64_t rows, int64_t cols) {
  if (rows < 0 || cols < 0 || cols % 16 || (rows > 0 && cols > 0 && (!q || !scales)))
    return OA_EINVAL;
  if (!aligned_to(q, 16)) return OA_EALIGN;
  if (blocks_of(rows) * blocks_of(cols) > 0x7FFFFFFF ||
      (cols > 0 && rows > ((int64_t)0x7FFFFFFF * kThreads) / (cols / 16)))
    return OA_ERANGE;
  return 0;
}

int check_layer(const Layer& w, int64_t tokens, int dtype) {
  if (!known(dtype) || tokens <= 0 || w.out_f <= 0 || w.in_f <= 0 || w.in_f % 16 || !w.q ||
      !w.scales)
    return OA_EINVAL;
  if (!aligned_to(w.q, 16)) return OA_EALIGN;
  if (tokens > kMostRows || w.out_f > kMostRows || w.in_f > kMostRows) return OA_ERANGE;
  return 0;
}

int check_source(const Source& m, int dtype) {
  if (!m.base || (m.rows > 1 && m.stride < m.cols)) return OA_EINVAL;
  return aligned_to(m.base, size_of(dtype)) ? 0 : OA_EALIGN;
}

}  // namespace
}  // namespace oa

using namespace oa;

extern "C" int oa_quant_fp8(const void* src, int src_dtype, int64_t src_row_stride, int64_t rows,
                            int64_t cols, void* q, void* scales, void* stream) {
  int rc = check_codec(q, scales, rows, cols);
  if (rc) return rc;
  if (!known(src_dtype) || src_row_stride < 0) return OA_EINVAL;
  if (rows == 0 || cols == 0) return 0;
  const Source m{src, src_row_stride, rows, cols};
  rc = check_source(m, src_dtype);
  if (rc) return rc;
  const bool vec = vector_rows(m, src_dtype);
  const uint32_t bc = (uint32_t)blocks_of(cols);
  const dim3 grid((unsigned)(bc * blocks_of(rows)));
  hipStream_t s = static_cast<hipStream_t>(stream);
  uint8_t *qb = static_cast<uint8_t*>(q), *sb = static_cast<uint8_t*>(scales);
  switch (src_dtype) {
    case OA_F32:
      hipLaunchKernelGGL(fp8_encode_kernel<OA_F32>, grid, dim3(kThreads), 0, s, m, bc, vec, qb, sb);
      break;
    case OA_BF16:
      hipLaunchKernelGGL(fp8_encode_kernel<OA_BF16>, grid, dim3(kThreads), 0, s, m, bc, vec, qb, sb);
      break;
    default:
      hipLaunchKernelGGL(fp8_encode_kernel<OA_F16>, grid, dim3(kThreads), 0, s, m, bc, vec, qb, sb);
  }
  return launch_status();
}

extern "C" int oa_dequant_fp8(const void* q, const void* scales, int64_t rows, int64_t cols,
                              void* out, int out_dtype, int64_t out_row_stride, void* stream) {
  int rc = check_codec(q, scales, rows, cols);
  if (rc) return rc;
  if (!known(out_dtype) || (rows > 1 && out_row_stride < cols)) return OA_EINVAL;
  if (rows == 0 || cols == 0) return 0;
  if (!out) return OA_EINVAL;
  if (!aligned_to(out, size_of(out_dtype))) return OA_EALIGN;
  const bool vec = out_row_stride % 8 == 0 && aligned_to(out, 16);
  const int64_t bc = blocks_of(cols), lanes = rows * (cols / 16);
  const dim3 grid((unsigned)((lanes + kThreads - 1) / kThreads));
  hipStream_t s = static_cast<hipStream_t>(stream);
  const uint8_t *qb = static_cast<const uint8_t*>(q), *sb = static_cast<const uint8_t*>(scales);
  switch (out_dtype) {
    case OA_F32:
      hipLaunchKernelGGL(fp8_decode_kernel<OA_F32>, grid, dim3(kThreads), 0, s, qb, sb, rows, cols,
                         bc, out, out_row_stride, vec);
      break;
    case OA_BF16:
      hipLaunchKernelGGL(fp8_decode_kernel<OA_BF16>, grid, dim3(kThreads), 0, s, qb, sb, rows,
                         cols, bc, out, out_row_stride, vec);
      break;
    default:
      hipLaunchKernelGGL(fp8_decode_kernel<OA_F16>, grid, dim3(kThreads), 0, s, qb, sb, rows, cols,
                         bc, out, out_row_stride, vec);
  }
  return launch_status();
}

extern "C" size_t oa_fp8_linear_workspace_bytes(int64_t tokens, int64_t in_features,
                                                int64_t out_features, int backward, int want_dx,
                                                int want_dw, int want_db) {
  if (tokens <= 0 || in_features <= 0 || out_features <= 0) return 0;
  if (tokens > kMostRows || in_features > kMostRows || out_features > kMostRows) return 0;
  if (!backward) {
    const bool few = takes_few(Layer{nullptr, nullptr, out_features, in_features}, tokens);
    return ForwardPlan(tokens, in_features, out_features, few, nullptr).bytes;
  }
  return BackwardPlan(tokens, in_features, out_features, want_dx != 0, want_dw != 0, want_db != 0,
                      nullptr)
      .bytes;
}

extern "C" int oa_fp8_linear_forward(const void* x, int64_t ldx, int dtype, int64_t tokens,
                                     const void* q, const void* scales, const void* bias,
                                     int64_t out_features, int64_t in_features, void* y,
                                     void* workspace, size_t workspace_bytes, void* stream) {
  const Layer w{static_cast<const uint8_t*>(q), static_cast<const uint8_t*>(scales), out_features,
                in_features};
  int rc = check_layer(w, tokens, dtype);
  if (rc) return rc;
  const Source m{x, ldx, tokens, in_features};
  rc = check_source(m, dtype);
  if (rc) return rc;
  if (!y || !workspace ||
      workspace_bytes < oa_fp8_linear_workspace_bytes(tokens, in_features, out_features, 0, 0, 0, 0))
    return OA_EINVAL;
  if (!aligned_to(y, size_of(dtype)) || !aligned_to(bias, size_of(dtype)) ||
      !aligned_to(workspace, 256))
    return OA_EALIGN;
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case OA_F32: return forward<OA_F32>(m, w, bias, y, workspace, s);
    case OA_BF16: return forward<OA_BF16>(m, w, bias, y, workspace, s);
    default: return forward<OA_F16>(m, w, bias, y, workspace, s);
  }
}

extern "C" int oa_fp8_linear_backward(const void* grad, int64_t ldg, const void* x, int64_t ldx,
                                      int dtype, int64_t tokens, const void* q,
                                      const void* scales, int64_t out_features,
                                      int64_t in_features, void* dx, void* dw, void* db,
                                      void* workspace, size_t workspace_bytes, void* stream) {
  const Layer w{static_cast<const uint8_t*>(q), static_cast<const uint8_t*>(scales), out_features,
                in_features};
  int rc = check_layer(w, tokens, dtype);
  if (rc) return rc;
  const Source mg{grad, ldg, tokens, out_features}, mx{x, ldx, tokens, in_features};
  rc = check_source(mg, dtype);
  if (rc) return rc;
  if (dw) {
    rc = check_source(mx, dtype);
    if (rc) return rc;
  }
  if ((!dx && !dw && !db) || !workspace ||
      workspace_bytes < oa_fp8_linear_workspace_bytes(tokens, in_features, out_features, 1,
                                                      dx != nullptr, dw != nullptr, db != nullptr))
    return OA_EINVAL;
  if (!aligned_to(dx, size_of(dtype)) || !aligned_to(dw, size_of(dtype)) ||
      !aligned_to(db, size_of(dtype)) || !aligned_to(workspace, 256))
    return OA_EALIGN;
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case OA_F32: return backward<OA_F32>(mg, mx, w, dx, dw, db, workspace, s);
    case OA_BF16: return backward<OA_BF16>(mg, mx, w, dx, dw, db, workspace, s);
    default: return backward<OA_F16>(mg, mx, w, dx, dw, db, workspace, s);
  }
}
