// Quantization to 8-bit floating point (e4m3) with one scale per block of 128.
//
// A block is 1 x 128 along a row (an activation, a gradient), 1 x 128 along a column (the
// same tensors as operands of a weight gradient, which reduces over the rows), or 128 x 128
// (a weight). With amax the block's largest magnitude, the scale is
//   e8m0: 2^e, e the least with amax / 2^e <= 448, in [-126, 127] (a byte e + 127), or
//   FP32: r(a r(1 / 448)), a = max(amax, 2^-100),
// and q = rne(x * factor): 1 / scale exactly under e8m0; under FP32 r(448 r(1 / a)), within
// 2^-23 of 448 / a, so that x * factor is at most 448 (1 + 2^-22), which rounds to 448. A block
// with an infinity or a NaN gets the e8m0 NaN (255) or the FP32 scale inf / NaN, so that all of it
// dequantizes to NaN (beside an infinity the FP32 factor is 0, and 0 times inf is NaN). Magnitudes
// are compared as integers, which ranks NaN above infinity above every number, so none is lost in the
// max.
//
// HBM-bound: x is read once (2 or 4 bytes an element), every form wanted of it written once
// (1 byte each). 16384 x 5632 BF16 by rows and columns takes 82 us, 4.5 TB/s (the card copies at
// 4.8); an 8960 x 1280 FP32 weight in both forms 15.5 us, 4.4 TB/s. A workgroup of 256 threads
// takes a 128 x 128 tile, in which all three kinds of block are whole, and holds it in
// registers as 8 x 8 elements per thread: thread t has rows 8 (t >> 4) .., columns
// 8 (t & 15) ... A row's 16 threads are neighbouring lanes; a column's 16 threads are four lanes
// in each of the four waves. The transposed form goes through LDS so that its rows leave as
// whole 128-byte lines.
#pragma once

#include "common.h"

namespace ws {

constexpr int kQBlock = 128;
constexpr float kE4M3Max = 448.0f;
enum QuantScale { kScaleE8M0 = 0, kScaleF32 = 1 };
enum QuantForm { kQuantRows = 1, kQuantCols = 2, kQuantBlocks = 4 };

struct QuantParams {
  const void* x;
  long ldx;
  int rows, cols, col_tiles;
  int q_cols, qt_cols;
  // Element (r, c) of q at r * ldq + c; columns past `cols` up to q_cols, the next multiple of
  // 16, are written as zeros. The transposed form likewise with rows and columns exchanged.
  unsigned char* q;  long ldq;
  unsigned char* qt; long ldqt;
  // Scale (r, b): e8m0 byte at r * ld + b, FP32 at b * ld + r.
  void* scale;   long ld_scale;
  void* scale_t; long ld_scale_t;
};

// The scale of a block from the bits of its largest magnitude, and its inverse.
template <int SCALE>
__device__ __forceinline__ float block_inverse(unsigned amax_bits, unsigned& scale) {
  if constexpr (SCALE == kScaleE8M0) {
    int code = (int)(amax_bits >> 23) - 8 + ((amax_bits & 0x7fffffu) > 0x600000u);
    code = code < 1 ? 1 : code;
    if (amax_bits >= 0x7f800000u) code = 255;
    scale = (unsigned)code;
    return __uint_as_float(code == 255 ? 0x7fc00000u : (unsigned)(254 - code) << 23);
  } else {
    // 2^-100 keeps the factor finite; the bits of a NaN stay the larger ones.
    const unsigned floor_bits = 27u << 23;
    const float a = __uint_as_float(amax_bits > floor_bits ? amax_bits : floor_bits);
    scale = __float_as_uint(a * (1.0f / kE4M3Max));
    return (1.0f / a) * kE4M3Max;
  }
}
template <int SCALE>
__device__ __forceinline__ void store_scale(void* base, long ld, long r, long b, unsigned v) {
  if constexpr (SCALE == kScaleE8M0) static_cast<unsigned char*>(base)[r * ld + b] = (unsigned char)v;
  else static_cast<unsigned*>(base)[b * ld + r] = v;
}

// Four FP32 values -> four e4m3 bytes (round to nearest even).
__device__ __forceinline__ unsigned pack_e4m3(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

// Element e (0..7) of a thread's row piece as FP32: BF16 pairs in four words, or FP32 words.
template <bool F32>
struct QuantRow {
  unsigned w[F32 ? 8 : 4];
  __device__ __forceinline__ float at(int e) const {
    if constexpr (F32) return __uint_as_float(w[e]);
    else return (e & 1) ? hi_bf16(w[e >> 1]) : lo_bf16(w[e >> 1]);
  }
  __device__ __forceinline__ unsigned magnitude(int e) const {
    return __float_as_uint(at(e)) & 0x7fffffffu;
  }
};

// VEC: rows start on 16-byte boundaries (and their strides keep them there), so that whole
// pieces of eight elements are loaded as vectors; others are loaded one element at a time.
// R: rows per thread, 8, or 1 for few rows quantized by rows (tiles of 16 x 128).
template <bool F32, int SCALE, int FORM, bool VEC, int R>
static __global__ void __launch_bounds__(256) quantize_kernel(const QuantParams p) {
  constexpr bool kRows = FORM & kQuantRows, kCols = FORM & kQuantCols, kBlocks = FORM & kQuantBlocks;
  static_assert(!kBlocks || !kRows, "a tile has row scales or one block scale");
  static_assert(R == 8 || FORM == kQuantRows, "whole blocks of 128 rows");
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int tr = blockIdx.x / p.col_tiles, tc = blockIdx.x % p.col_tiles;
  const int r0 = tr * 16 * R + R * (t >> 4), c0 = tc * kQBlock + 8 * (t & 15);
  const int left = p.cols - c0;  // columns of this thread's pieces inside the matrix

  QuantRow<F32> x[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const bool ok = r0 + r < p.rows;
    if (VEC && ok && left >= 8) {
      if constexpr (F32) {
        const auto* src = reinterpret_cast<const u32x4_t*>(static_cast<const float*>(p.x) + (long)(r0 + r) * p.ldx + c0);
        const u32x4_t a = src[0], b = src[1];
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          x[r].w[d] = a[d];
          x[r].w[4 + d] = b[d];
        }
      } else {
        const u32x4_t a = *reinterpret_cast<const u32x4_t*>(
            static_cast<const unsigned short*>(p.x) + (long)(r0 + r) * p.ldx + c0);
#pragma unroll
        for (int d = 0; d < 4; ++d) x[r].w[d] = a[d];
      }
    } else {
#pragma unroll
      for (int d = 0; d < (F32 ? 8 : 4); ++d) x[r].w[d] = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (!ok || e >= left) continue;
        const long at = (long)(r0 + r) * p.ldx + c0 + e;
        if constexpr (F32) x[r].w[e] = static_cast<const unsigned*>(p.x)[at];
        else x[r].w[e >> 1] |= (unsigned)static_cast<const unsigned short*>(p.x)[at] << (16 * (e & 1));
      }
    }
  }

  __shared__ unsigned amax[4][kQBlock];
  __shared__ unsigned char tile[kCols || kBlocks ? kQBlock : 1][kQBlock + 16];
  float inv_block = 0.0f;
  if constexpr (kBlocks) {
    unsigned m = 0;
#pragma unroll
    for (int r = 0; r < 8; ++r)
#pragma unroll
      for (int e = 0; e < 8; ++e) m = max(m, x[r].magnitude(e));
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) m = max(m, (unsigned)__shfl_xor((int)m, off, kWave));
    if (lane == 0) amax[wave][0] = m;
    __syncthreads();
    m = max(max(amax[0][0], amax[1][0]), max(amax[2][0], amax[3][0]));
    unsigned scale;
    inv_block = block_inverse<SCALE>(m, scale);
    if (t == 0) {
      store_scale<SCALE>(p.scale, p.ld_scale, tr, tc, scale);
      if (p.qt) store_scale<SCALE>(p.scale_t, p.ld_scale_t, tc, tr, scale);
    }
  }
  if constexpr (kRows || kBlocks) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float inv = inv_block;
      if constexpr (kRows) {
        unsigned m = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) m = max(m, x[r].magnitude(e));
#pragma unroll
        for (int off = 8; off >= 1; off >>= 1) m = max(m, (unsigned)__shfl_xor((int)m, off, kWave));
        unsigned scale;
        inv = block_inverse<SCALE>(m, scale);
        if ((t & 15) == 0 && r0 + r < p.rows) store_scale<SCALE>(p.scale, p.ld_scale, r0 + r, tc, scale);
      }
      if (r0 + r < p.rows && c0 < p.q_cols) {
        u32x2_t o;
#pragma unroll
        for (int d = 0; d < 2; ++d)
          o[d] = pack_e4m3(x[r].at(4 * d) * inv, x[r].at(4 * d + 1) * inv, x[r].at(4 * d + 2) * inv,
                           x[r].at(4 * d + 3) * inv);
        *reinterpret_cast<u32x2_t*>(p.q + (long)(r0 + r) * p.ldq + c0) = o;
      }
    }
  }
  if constexpr (kCols || kBlocks) {
    if (!kCols && !p.qt) return;  // uniform
    // Transposed: this thread's eight columns, eight row bytes each, into LDS rows of the
    // transposed tile, then whole rows out.
    if constexpr (kCols) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        unsigned m = 0;
#pragma unroll
        for (int r = 0; r < 8; ++r) m = max(m, x[r].magnitude(e));
        m = max(m, (unsigned)__shfl_xor((int)m, 16, kWave));
        m = max(m, (unsigned)__shfl_xor((int)m, 32, kWave));
        if (lane < 16) amax[wave][8 * lane + e] = m;
      }
      __syncthreads();
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int c = 8 * (t & 15) + e;
      float inv = inv_block;
      if constexpr (kCols) {
        unsigned scale;
        inv = block_inverse<SCALE>(max(max(amax[0][c], amax[1][c]), max(amax[2][c], amax[3][c])), scale);
        if (t < 16 && tc * kQBlock + c < p.cols)
          store_scale<SCALE>(p.scale_t, p.ld_scale_t, tc * kQBlock + c, tr, scale);
      }
      u32x2_t o;
#pragma unroll
      for (int d = 0; d < 2; ++d)
        o[d] = pack_e4m3(x[4 * d].at(e) * inv, x[4 * d + 1].at(e) * inv, x[4 * d + 2].at(e) * inv,
                         x[4 * d + 3].at(e) * inv);
      *reinterpret_cast<u32x2_t*>(&tile[c][8 * (t >> 4)]) = o;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = 32 * i + (t >> 3), byte = 16 * (t & 7);
      if (tc * kQBlock + c < p.cols && tr * kQBlock + byte < p.qt_cols)
        *reinterpret_cast<u32x4_t*>(p.qt + (long)(tc * kQBlock + c) * p.ldqt + tr * kQBlock + byte) =
            *reinterpret_cast<const u32x4_t*>(&tile[c][byte]);
    }
  }
}

// Bytes (r, c) at r * s_row + c * s_col into rows of ldd bytes (a multiple of 16), zeros past
// `cols`: an operand that the product's 16-byte loads cannot read as it is.
static __global__ void __launch_bounds__(256) pack_bytes_kernel(const unsigned char* src, long s_row,
                                                                long s_col, unsigned char* dst,
                                                                long ldd, long rows, long cols) {
  const long pieces = ldd / 16;
  const long i = blockIdx.x * 256L + threadIdx.x;
  if (i >= rows * pieces) return;
  const long r = i / pieces, c = 16 * (i % pieces);
  u32x4_t v = {0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < 16; ++e)
    if (c + e < cols) v[e >> 2] |= (unsigned)src[r * s_row + (c + e) * s_col] << (8 * (e & 3));
  *reinterpret_cast<u32x4_t*>(dst + r * ldd + c) = v;
}

}  // namespace ws
