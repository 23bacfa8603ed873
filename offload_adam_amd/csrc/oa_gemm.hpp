// Tiled matrix product on the matrix cores, shared by the loss and the 8-bit
// floating-point kernels:
//
//     out[p][q] = sum_k P[p][k] * Q[q][k]          (both operands contiguous along k)
//
// A workgroup owns a BP x BQ tile of `out` and walks k in steps of 128 bytes per
// row (64 bf16 / fp16 or 128 e4m3 elements).  Both operands' next step travels
// from HBM to LDS with 16-byte direct loads (no registers in between) while the
// current one is multiplied; LDS holds two steps.  A row of a step is eight
// 16-byte chunks; chunk c of row r sits at position c ^ (r & 7), which spreads the
// eight rows that a quarter-wave reads together over all banks.  A direct load
// writes LDS in lane order, so the permutation is applied to the source address.
//
// A lane of a matrix instruction supplies chunks l/16 and l/16 + 4 of row l%16.
// Which k elements those are does not matter as long as both operands agree, so
// the three element types share every address computation.
//
// Q is the first operand of the matrix instruction: a lane then holds four
// consecutive q of one p, which is the contiguous direction of `out`.
//
// Rows past the end of an operand and chunks past the end of k are out of the
// buffer descriptor's range and read as zero.
#pragma once

#include "oa_common.hpp"

namespace oa {
namespace gemm {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int kStepBytes = 128;  // bytes of one row that one k step covers
constexpr int kChunks = kStepBytes / 16;

struct Bf16 {
  static constexpr bool kScaled = false;
  template <int, int>
  static __device__ __forceinline__ f32x4 mma(const i32x4 (&q)[2], const i32x4 (&p)[2], f32x4 c,
                                              int, int) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, q[0]),
                                                __builtin_bit_cast(bf16x8, p[0]), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, q[1]),
                                                   __builtin_bit_cast(bf16x8, p[1]), c, 0, 0, 0);
  }
};

struct F16 {
  static constexpr bool kScaled = false;
  template <int, int>
  static __device__ __forceinline__ f32x4 mma(const i32x4 (&q)[2], const i32x4 (&p)[2], f32x4 c,
                                              int, int) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, q[0]),
                                               __builtin_bit_cast(f16x8, p[0]), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, q[1]),
                                                  __builtin_bit_cast(f16x8, p[1]), c, 0, 0, 0);
  }
};

// e4m3 with one e8m0 scale per row and step: the matrix instruction takes each
// lane's scale with its row and applies it for free.  It adds the products of 8
// consecutive k at the exponent of the largest of them, with 13 bits under its leading
// one (the rest is cut off), and those sums and the accumulator in fp32.  That is some
// 2^-14 of a result, under the rounding of the codes (2^-4 each) and of a 16-bit result;
// multiplying decoded values instead would keep 24 bits at half the rate.
struct E4m3 {
  static constexpr bool kScaled = true;
  template <int BYTE_Q, int BYTE_P>
  static __device__ __forceinline__ f32x4 mma(const i32x4 (&q)[2], const i32x4 (&p)[2], f32x4 c,
                                              int sq, int sp) {
    const i32x8 a = __builtin_shufflevector(q[0], q[1], 0, 1, 2, 3, 4, 5, 6, 7);
    const i32x8 b = __builtin_shufflevector(p[0], p[1], 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, BYTE_Q, sq, BYTE_P, sp);
  }
};

// An operand: rows of `ld` bytes (16-byte aligned), k_bytes of each taking part
// (a multiple of 16).
struct Operand {
  const uint8_t* base;
  int64_t ld;
  int64_t rows;
};

// Where the scales of an e4m3 operand are.  `packed`: one byte per row and step, as
// [step][row group of 64][16] dwords, byte j of dword i = row 16 j + i of the group,
// so that a lane's dword serves four matrix tiles; rows go up to a multiple of 256.
// Otherwise one byte per 128 rows and step.
struct Scales {
  const uint8_t* base;
  int64_t step_stride;   // bytes from one step to the next
  int64_t block_stride;  // not packed: bytes from one block of 128 rows to the next
  int64_t blocks;        // not packed: number of those
  bool packed;
};

// Byte of (row, step) in a packed array.
__host__ __device__ inline int64_t packed_scale_at(int64_t row, int64_t step, int64_t step_stride) {
  return step * step_stride + row / 64 * 64 + row % 16 * 4 + row / 16 % 4;
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t tile_rsrc(const Operand& o, int64_t row0,
                                                            int tile_rows) {
  int64_t rows = o.rows - row0;
  rows = rows < 0 ? 0 : (rows > tile_rows ? tile_rows : rows);
  const uint8_t* base = o.base + (rows > 0 ? row0 * o.ld : 0);
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base), 0, (int)(rows * o.ld),
                                           0x00020000);
}

// The tile of workgroup b: consecutive workgroups go to the 8 XCDs in turn, and
// each XCD gets one contiguous run of tile numbers, numbered so that a run covers
// blocks of kGroup tiles along p: the operands of the tiles that an XCD has in
// flight together then come out of its own L2.
constexpr int kGroup = 8;
__device__ __forceinline__ void tile_of(uint32_t b, uint32_t tiles_p, uint32_t tiles_q,
                                        uint32_t& tp, uint32_t& tq) {
  const uint32_t total = tiles_p * tiles_q;
  const uint32_t per = total / kXcds, extra = total % kXcds;
  const uint32_t x = b % kXcds, j = b / kXcds;
  const uint32_t id = x * per + (x < extra ? x : extra) + j;
  const uint32_t group = id / (kGroup * tiles_q);
  const uint32_t first = group * kGroup;
  const uint32_t wide = tiles_p - first < kGroup ? tiles_p - first : kGroup;
  const uint32_t in = id - first * tiles_q;
  tp = first + in % wide;
  tq = in / wide;
}

template <class T, int BQ_, int BP_, int WQ, int WP>
struct Tile {
  static constexpr int BQ = BQ_, BP = BP_;
  static constexpr int kWavesQ = WQ, kWavesP = WP, kWaves = WQ * WP, kThreads = kWave * kWaves;
  static constexpr int QR = BQ / WQ, PR = BP / WP;  // rows of each operand that a wave owns
  static constexpr int QT = QR / 16, PT = PR / 16;
  static constexpr int kLoadsQ = BQ / 8 / kWaves, kLoadsP = BP / 8 / kWaves;
  static constexpr int kBytesQ = BQ * kStepBytes, kBytesP = BP * kStepBytes;
  static_assert(kLoadsQ * 8 * kWaves == BQ && kLoadsP * 8 * kWaves == BP, "tile / waves");

  f32x4 acc[QT][PT];
  int lane, wave, wq, wp;

  __device__ __forceinline__ Tile() {
    lane = threadIdx.x & (kWave - 1);
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    wq = wave % WQ;
    wp = wave / WQ;
  }

  // First q / p of this lane's results relative to the tile: result i of acc[a][b]
  // is (q0() + 16 a + i, p0() + 16 b).
  __device__ __forceinline__ int q0() const { return wq * QR + 4 * (lane / 16); }
  __device__ __forceinline__ int p0() const { return wp * PR + lane % 16; }

  template <int N>
  __device__ __forceinline__ void fetch(__amdgpu_buffer_rsrc_t rsrc, int ld, int step, int k_bytes,
                                        uint8_t* lds) const {
    const int c = (lane % 8) ^ (lane / 8);
    const int k = step * kStepBytes + c * 16;
    const int row = wave * N * 8 + lane / 8;
    const int off = k < k_bytes ? row * ld + k : 0x7FFFFF00;
#pragma unroll
    for (int i = 0; i < N; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rsrc,
          reinterpret_cast<__attribute__((address_space(3))) void*>(
              reinterpret_cast<uintptr_t>(lds + (wave * N + i) * 8 * kStepBytes)),
          16, k < k_bytes ? off + i * 8 * ld : off, 0, 0, 0);
  }

  // Scales of this lane's rows, four 16-row tiles to a dword.
  static constexpr int kScalesQ = (QT + 3) / 4, kScalesP = (PT + 3) / 4;

  template <int A, int B>
  __device__ __forceinline__ void multiply_row(const i32x4 (&fq)[2], const i32x4 (&fp)[PT][2],
                                               const int (&sq)[kScalesQ],
                                               const int (&sp)[kScalesP]) {
    if constexpr (B < PT) {
      acc[A][B] = T::template mma<A % 4, B % 4>(fq, fp[B], acc[A][B], sq[A / 4], sp[B / 4]);
      multiply_row<A, B + 1>(fq, fp, sq, sp);
    }
  }

  template <int A>
  __device__ __forceinline__ void multiply_rows(const uint8_t* q, int o0, int o1,
                                                const i32x4 (&fp)[PT][2],
                                                const int (&sq)[kScalesQ],
                                                const int (&sp)[kScalesP]) {
    if constexpr (A < QT) {
      i32x4 fq[2];
      fq[0] = *reinterpret_cast<const i32x4*>(q + A * 16 * kStepBytes + o0);
      fq[1] = *reinterpret_cast<const i32x4*>(q + A * 16 * kStepBytes + o1);
      multiply_row<A, 0>(fq, fp, sq, sp);
      multiply_rows<A + 1>(q, o0, o1, fp, sq, sp);
    }
  }

  __device__ __forceinline__ void multiply(const uint8_t* lq, const uint8_t* lp,
                                           const int (&sq)[kScalesQ], const int (&sp)[kScalesP]) {
    const int r = lane % 16, g = lane / 16;
    const uint8_t* q = lq + (wq * QR + r) * kStepBytes;
    const uint8_t* p = lp + (wp * PR + r) * kStepBytes;
    const int o0 = (g ^ (r & 7)) * 16, o1 = ((g + 4) ^ (r & 7)) * 16;
    i32x4 fp[PT][2];
#pragma unroll
    for (int b = 0; b < PT; ++b) {
      fp[b][0] = *reinterpret_cast<const i32x4*>(p + b * 16 * kStepBytes + o0);
      fp[b][1] = *reinterpret_cast<const i32x4*>(p + b * 16 * kStepBytes + o1);
    }
    multiply_rows<0>(q, o0, o1, fp, sq, sp);
  }

  template <int N>
  __device__ __forceinline__ void load_scales(const Scales& s, int64_t row0, int step,
                                              int (&out)[N]) const {
    if constexpr (T::kScaled) {
      if (s.packed) {
        const uint32_t* d = reinterpret_cast<const uint32_t*>(s.base + (int64_t)step * s.step_stride) +
                            row0 / 64 * 16 + lane % 16;
#pragma unroll
        for (int j = 0; j < N; ++j) out[j] = (int)(d[16 * j] >> (8 * (row0 / 16 % 4)));
      } else {
        int64_t block = row0 / 128;  // a tile may hang over the last block
        if (block >= s.blocks) block = s.blocks - 1;
        const int v = s.base[block * s.block_stride + step * s.step_stride] * 0x01010101;
#pragma unroll
        for (int j = 0; j < N; ++j) out[j] = v;
      }
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) out[j] = 0;
    }
  }

  // The products of steps [step0, step1) of the tile at (row_q, row_p).
  __device__ __forceinline__ void run(const Operand& oq, const Operand& op, int64_t row_q,
                                      int64_t row_p, int k_bytes, int step0, int step1,
                                      const Scales& scq, const Scales& scp, uint8_t* lq0,
                                      uint8_t* lq1, uint8_t* lp0, uint8_t* lp1) {
#pragma unroll
    for (int a = 0; a < QT; ++a)
#pragma unroll
      for (int b = 0; b < PT; ++b) acc[a][b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const auto rq = tile_rsrc(oq, row_q, BQ), rp = tile_rsrc(op, row_p, BP);
    const int ldq = (int)oq.ld, ldp = (int)op.ld;
    const int64_t mine_q = row_q + wq * QR, mine_p = row_p + wp * PR;
    int sq[kScalesQ], sp[kScalesP], nsq[kScalesQ], nsp[kScalesP];
    const int begin = step0 < step1 ? step0 : 0;  // an empty slice: any scale that is there
    load_scales(scq, mine_q, begin, sq);
    load_scales(scp, mine_p, begin, sp);
    // steps from step1 on read as zero
    const int k_end = k_bytes < step1 * kStepBytes ? k_bytes : step1 * kStepBytes;
    fetch<kLoadsQ>(rq, ldq, step0, k_end, lq0);
    fetch<kLoadsP>(rp, ldp, step0, k_end, lp0);
    int s = step0;
    for (; s + 1 < step1; s += 2) {
      wait();
      load_scales(scq, mine_q, s + 1, nsq);
      load_scales(scp, mine_p, s + 1, nsp);
      fetch<kLoadsQ>(rq, ldq, s + 1, k_end, lq1);
      fetch<kLoadsP>(rp, ldp, s + 1, k_end, lp1);
      multiply(lq0, lp0, sq, sp);
      wait();
      const int next = s + 2 < step1 ? s + 2 : s + 1;  // scales past the end are not there
      load_scales(scq, mine_q, next, sq);
      load_scales(scp, mine_p, next, sp);
      fetch<kLoadsQ>(rq, ldq, s + 2, k_end, lq0);
      fetch<kLoadsP>(rp, ldp, s + 2, k_end, lp0);
      multiply(lq1, lp1, nsq, nsp);
    }
    wait();
    if (s < step1) multiply(lq0, lp0, sq, sp);
    // The results exist here, on every lane: a matrix instruction that moved into a
    // branch of the epilogue would lose the operands of the lanes that do not take it.
#pragma unroll
    for (int a = 0; a < QT; ++a)
#pragma unroll
      for (int b = 0; b < PT; ++b) asm volatile("" : "+v"(acc[a][b]));
  }

  // This wave's direct loads have landed in LDS, and every wave of the workgroup has
  // come this far: its loads have landed too, and it is done reading the other buffers.
  static __device__ __forceinline__ void wait() {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  }
};

// One product.  `slices` workgroups share a tile, each with its own run of k steps;
// what becomes of their results is the epilogue's business.
struct Problem {
  Operand q, p;
  Scales sq, sp;  // e4m3 only
  int k_bytes;
  int steps_per_slice;
  uint32_t tiles_q, tiles_p;
};

inline int steps_of(int64_t k_bytes) { return (int)((k_bytes + kStepBytes - 1) / kStepBytes); }

template <class T, class E>
__global__ void __launch_bounds__(T::kThreads) product_kernel(const Problem pr, const E epilogue) {
  __shared__ __align__(16) uint8_t lq0[T::kBytesQ], lq1[T::kBytesQ];
  __shared__ __align__(16) uint8_t lp0[T::kBytesP], lp1[T::kBytesP];
  T t;
  uint32_t tp, tq;
  const uint32_t tiles = pr.tiles_p * pr.tiles_q;
  const uint32_t slice = blockIdx.x / tiles;
  tile_of(blockIdx.x - slice * tiles, pr.tiles_p, pr.tiles_q, tp, tq);
  const int64_t row_q = (int64_t)tq * T::BQ, row_p = (int64_t)tp * T::BP;
  const int steps = (pr.k_bytes + kStepBytes - 1) / kStepBytes;
  const int step0 = (int)slice * pr.steps_per_slice;
  const int step1 = step0 + pr.steps_per_slice < steps ? step0 + pr.steps_per_slice : steps;
  t.run(pr.q, pr.p, row_q, row_p, pr.k_bytes, step0, step1, pr.sq, pr.sp, lq0, lq1, lp0, lp1);
  epilogue(t, row_q, row_p, (int)tq, (int)slice, lq0);
}

// Tile sizes.  256 x 256 with 8 waves reads each byte of LDS for 2 (q) or 4 (p)
// waves and is the fastest where it fills the chip; with fewer tiles than three
// quarters of the 256 CUs the 128 x 128 tile, two workgroups to a CU, leaves fewer
// of them idle.  Measured in bf16: 4096 x 14336 x 4096 takes 471 us with the large
// tile and 539 us with the small one; 1000 x 1020 x 520 takes 17.7 against 8.4 us.
template <class T>
using Large = Tile<T, 256, 256, 2, 4>;
template <class T>
using Small = Tile<T, 128, 128, 2, 2>;
constexpr int64_t kFillTiles = 192;

inline int64_t tiles_along(int64_t rows, int tile) { return (rows + tile - 1) / tile; }

inline bool large_tiles_fill(int64_t rows_q, int64_t rows_p) {
  return tiles_along(rows_q, 256) * tiles_along(rows_p, 256) >= kFillTiles;
}

// Workgroups that share a tile along k: enough that the chip is filled, no slice
// shorter than 8 steps (a slice pays one pass over its partial results).
inline int slices_for(int64_t rows_q, int64_t rows_p, int64_t k_bytes) {
  const int64_t tiles = tiles_along(rows_q, 128) * tiles_along(rows_p, 128);
  int64_t s = 2 * kFillTiles / tiles;
  const int64_t most = steps_of(k_bytes) / 8;
  if (s > most) s = most;
  return (int)(s < 1 ? 1 : s);
}

template <class T, class E>
int launch_tiles(Problem pr, int slices, const E& epilogue, hipStream_t stream) {
  const int64_t tq = tiles_along(pr.q.rows, T::BQ), tp = tiles_along(pr.p.rows, T::BP);
  if (tq * tp * slices > 0x7FFFFFFF) return OA_ERANGE;
  pr.tiles_q = (uint32_t)tq;
  pr.tiles_p = (uint32_t)tp;
  const int steps = steps_of(pr.k_bytes);
  pr.steps_per_slice = (steps + slices - 1) / slices;
  hipLaunchKernelGGL((product_kernel<T, E>), dim3((unsigned)(tq * tp * slices)),
                     dim3(T::kThreads), 0, stream, pr, epilogue);
  return launch_status();
}

// A tile's rows, and the offsets inside it, have to fit the buffer descriptor.
inline bool operand_fits(const Operand& o, int64_t k_bytes) {
  return o.ld > 0 && o.ld <= (1 << 22) && k_bytes <= o.ld && o.ld % 16 == 0 &&
         aligned_to(o.base, 16) && k_bytes % 16 == 0;
}

}  // namespace gemm
}  // namespace oa
