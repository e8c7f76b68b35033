// Residual addition and RMSNorm in one pass, the norm in BF16 or in 8 bits, and its backward.
//
//   s = r(x + residual)                in the residual stream's type, BF16 or FP32
//   rstd = 1 / sqrt(mean(s^2) + eps),  y = s rstd w
//
// of the rounded s, which is what the next addition reads. y is rounded once: to BF16, or to
// e4m3 with a scale per block of 128 (quant.h), from FP32 either way. With g = dy w and the
// stream's own upstream gradient ds,
//   d = ds + rstd (g - s rstd^2 mean(g s)),  dweight = sum over rows of dy s rstd,
// and d is the gradient of both inputs, rounded to the type of each. The backward reads s anyway and
// takes rstd from it again, so that nothing but the stream is kept for it.
//
// HBM-bound: each input is read once and each output written once, with the row in registers
// between. A row's pieces of eight columns lie on consecutive lanes, so that 16 lanes hold a block
// of 128.
#pragma once

#include "quant.h"

namespace ws {

struct AddNormParams {
  const unsigned short* x; long ldx;
  const void* residual; long ldr;  // the stream's type
  const float* w;
  int rows, d;
  float eps;
  unsigned short* y;               // [rows, d]
  void* stream;                    // [rows, d], the stream's type
  unsigned char* q; long ldq;      // bytes past d up to q_cols, the next multiple of 16, are zeros
  int q_cols;
  void* scale; long ld_scale;
};

// 16 bytes at any address of their elements: the vector instructions do not need more.
typedef unsigned u32x4_any2 __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned u32x4_any4 __attribute__((ext_vector_type(4), aligned(4)));

// Eight elements from element `at` on, of which `left` exist (zeros for the others). WHOLE: rows are
// whole pieces, so that left is at least eight or at most zero.
template <bool F32, bool WHOLE>
__device__ __forceinline__ void load_piece(QuantRow<F32>& v, const void* base, long at, int left) {
  if (left >= 8) {
    if constexpr (F32) {
      const auto* src = reinterpret_cast<const u32x4_any4*>(static_cast<const float*>(base) + at);
      const u32x4_t a = src[0], b = src[1];
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        v.w[d] = a[d];
        v.w[4 + d] = b[d];
      }
    } else {
      const u32x4_t a = *reinterpret_cast<const u32x4_any2*>(static_cast<const unsigned short*>(base) + at);
#pragma unroll
      for (int d = 0; d < 4; ++d) v.w[d] = a[d];
    }
    return;
  }
#pragma unroll
  for (int d = 0; d < (F32 ? 8 : 4); ++d) v.w[d] = 0;
  if (WHOLE || left <= 0) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (e >= left) continue;
    if constexpr (F32) v.w[e] = static_cast<const unsigned*>(base)[at + e];
    else v.w[e >> 1] |= (unsigned)static_cast<const unsigned short*>(base)[at + e] << (16 * (e & 1));
  }
}
template <bool F32, bool WHOLE>
__device__ __forceinline__ void store_piece(const QuantRow<F32>& v, void* base, long at, int left) {
  if (left >= 8) {
    if constexpr (F32) {
      auto* dst = reinterpret_cast<u32x4_any4*>(static_cast<float*>(base) + at);
      dst[0] = u32x4_t{v.w[0], v.w[1], v.w[2], v.w[3]};
      dst[1] = u32x4_t{v.w[4], v.w[5], v.w[6], v.w[7]};
    } else {
      *reinterpret_cast<u32x4_any2*>(static_cast<unsigned short*>(base) + at) =
          u32x4_t{v.w[0], v.w[1], v.w[2], v.w[3]};
    }
    return;
  }
  if (WHOLE || left <= 0) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (e >= left) continue;
    if constexpr (F32) static_cast<unsigned*>(base)[at + e] = v.w[e];
    else static_cast<unsigned short*>(base)[at + e] = (unsigned short)(v.w[e >> 1] >> (16 * (e & 1)));
  }
}
template <bool F32>
__device__ __forceinline__ QuantRow<F32> round_piece(const float (&f)[8]) {
  QuantRow<F32> v;
  if constexpr (F32) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v.w[e] = __float_as_uint(f[e]);
  } else {
#pragma unroll
    for (int d = 0; d < 4; ++d) v.w[d] = pack_bf16x2(f[2 * d], f[2 * d + 1]);
  }
  return v;
}

// The sum of v over the WPR waves of a row, in wave order. `slot` differs between two sums with no
// barrier but theirs between them, so that one barrier per sum is enough.
template <int WPR>
__device__ __forceinline__ float row_sum(float v, float (*red)[4], int slot, int lane, int wave) {
  v = wave_sum(v);
  if constexpr (WPR == 1) return v;
  if (lane == 0) red[slot][wave] = v;
  __syncthreads();
  return (red[slot][0] + red[slot][1]) + (red[slot][2] + red[slot][3]);
}

enum AddNormOut { kNormBF16 = 0, kNormE8M0 = 1, kNormF32Scales = 2 };

// WPR waves take a row (1: four rows per workgroup; 4: one), NC pieces per lane: d is at most
// 512 NC WPR. ADD: there is a residual; without one s is x, and no stream is written.
template <bool F32, bool ADD, int OUT, int NC, int WPR, bool WHOLE>
static __global__ void __launch_bounds__(256) add_rmsnorm_kernel(const AddNormParams p) {
  __shared__ float red[2][4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = WPR == 1 ? blockIdx.x * 4 + wave : blockIdx.x;
  if (WPR == 1 && row >= p.rows) return;
  const int c0 = 8 * (WPR == 1 ? lane : (int)threadIdx.x);
  QuantRow<F32> s[NC];
  {
    QuantRow<false> x[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = c0 + i * 512 * WPR;
      load_piece<false, WHOLE>(x[i], p.x, (long)row * p.ldx + c, p.d - c);
      if constexpr (ADD) load_piece<F32, WHOLE>(s[i], p.residual, (long)row * p.ldr + c, p.d - c);
    }
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      float f[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = ADD ? x[i].at(e) + s[i].at(e) : x[i].at(e);
      s[i] = round_piece<F32>(f);
      const int c = c0 + i * 512 * WPR;
      if constexpr (ADD) store_piece<F32, WHOLE>(s[i], p.stream, (long)row * p.d + c, p.d - c);
    }
  }
  float acc = 0.0f;
#pragma unroll
  for (int i = 0; i < NC; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) acc += s[i].at(e) * s[i].at(e);
  acc = row_sum<WPR>(acc, red, 0, lane, wave);
  const float r = 1.0f / sqrtf(acc / (float)p.d + p.eps);
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int c = c0 + i * 512 * WPR, left = p.d - c;
    QuantRow<true> w;
    load_piece<true, WHOLE>(w, p.w, c, left);
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = (s[i].at(e) * r) * w.at(e);
    if constexpr (OUT == kNormBF16) {
      store_piece<false, WHOLE>(round_piece<false>(f), p.y, (long)row * p.d + c, left);
    } else {
      constexpr int SCALE = OUT == kNormE8M0 ? kScaleE8M0 : kScaleF32;
      unsigned m = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) m = max(m, __float_as_uint(f[e]) & 0x7fffffffu);
#pragma unroll
      for (int off = 8; off >= 1; off >>= 1) m = max(m, (unsigned)__shfl_xor((int)m, off, kWave));
      unsigned scale;
      const float inv = block_inverse<SCALE>(m, scale);
      if ((lane & 15) == 0 && left > 0) store_scale<SCALE>(p.scale, p.ld_scale, row, c / kQBlock, scale);
      if (c < p.q_cols) {
        u32x2_t o;
#pragma unroll
        for (int d = 0; d < 2; ++d)
          o[d] = pack_e4m3(f[4 * d] * inv, f[4 * d + 1] * inv, f[4 * d + 2] * inv, f[4 * d + 3] * inv);
        *reinterpret_cast<u32x2_t*>(p.q + (long)row * p.ldq + c) = o;
      }
    }
  }
}

struct AddNormGradParams {
  const void* s;                            // [rows, d], the stream's type
  const float* w;
  float eps;
  const unsigned short* dy; long ld_dy;
  const void* ds; long ld_ds;               // the stream's type; unused without DS
  int rows, d;
  unsigned short* dx;                       // [rows, d] BF16
  float* dresidual;                         // [rows, d]: an FP32 stream's gradient (null: not wanted)
  float* partial;                           // [gridDim.x, d]: dweight of a workgroup's rows
};

// Each lane keeps the weight and the weight gradient of its columns in registers over all rows of
// its waves, so that the gradient's partial sums cost one row of FP32 per workgroup.
template <bool F32, bool DS, int NC, int WPR, bool WHOLE>
static __global__ void __launch_bounds__(256) add_rmsnorm_bwd_kernel(const AddNormGradParams p) {
  __shared__ float red[4][4];
  __shared__ float sums[WPR == 1 ? 3 : 1][WPR == 1 ? 512 * NC : 1];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c0 = 8 * (WPR == 1 ? lane : (int)threadIdx.x);
  constexpr int kRows = 4 / WPR;  // rows of a workgroup at a time
  float w[NC][8], dw[NC][8];
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int c = c0 + i * 512 * WPR;
    QuantRow<true> v;
    load_piece<true, WHOLE>(v, p.w, c, p.d - c);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      w[i][e] = v.at(e);
      dw[i][e] = 0.0f;
    }
  }
  int slot = 0;
  for (int row = blockIdx.x * kRows + (WPR == 1 ? wave : 0); row < p.rows; row += gridDim.x * kRows) {
    QuantRow<F32> s[NC], ds[NC];
    QuantRow<false> dy[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = c0 + i * 512 * WPR, left = p.d - c;
      load_piece<F32, WHOLE>(s[i], p.s, (long)row * p.d + c, left);
      load_piece<false, WHOLE>(dy[i], p.dy, (long)row * p.ld_dy + c, left);
      if constexpr (DS) load_piece<F32, WHOLE>(ds[i], p.ds, (long)row * p.ld_ds + c, left);
    }
    float dot = 0.0f, square = 0.0f;
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        dot += (dy[i].at(e) * w[i][e]) * s[i].at(e);
        square += s[i].at(e) * s[i].at(e);
      }
    dot = row_sum<WPR>(dot, red, 2 * slot, lane, wave);
    square = row_sum<WPR>(square, red, 2 * slot + 1, lane, wave);
    slot ^= 1;
    const float r = 1.0f / sqrtf(square / (float)p.d + p.eps);
    const float m = dot / (float)p.d * (r * r);
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = c0 + i * 512 * WPR, left = p.d - c;
      if constexpr (!F32) {  // keeps s and dy packed over the sums; unpacked they cost a workgroup's registers
#pragma unroll
        for (int e = 0; e < 4; ++e) asm volatile("" : "+v"(s[i].w[e]), "+v"(dy[i].w[e]));
      }
      float f[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float se = s[i].at(e), ge = dy[i].at(e);
        f[e] = r * (ge * w[i][e] - se * m);
        if constexpr (DS) f[e] += ds[i].at(e);
        dw[i][e] += ge * (se * r);
      }
      store_piece<false, WHOLE>(round_piece<false>(f), p.dx, (long)row * p.d + c, left);
      if constexpr (F32)
        if (p.dresidual) store_piece<true, WHOLE>(round_piece<true>(f), p.dresidual, (long)row * p.d + c, left);
    }
  }
  // The waves' sums in wave order.
  if constexpr (WPR == 1) {
    if (wave > 0) {
#pragma unroll
      for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) sums[wave - 1][512 * i + 64 * e + lane] = dw[i][e];
    }
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int q = 0; q < 3; ++q)
#pragma unroll
      for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) dw[i][e] += sums[q][512 * i + 64 * e + lane];
  }
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int c = c0 + i * 512 * WPR;
    store_piece<true, WHOLE>(round_piece<true>(dw[i]), p.partial, (long)blockIdx.x * p.d + c, p.d - c);
  }
}

}  // namespace ws
