// Epilogues of the LM head's logits product for the token scores (scores.h): row statistics,
// and the logits' gradient. The logits themselves exist only in the accumulators, in FP32.
#pragma once

#include "gemm_fast.h"
#include "scores.h"

namespace ws {

// Per row, over this wave's FB * 16 columns: the largest logit m, S and W (scores.h), one partial
// per (row, wave column block), and the token's logit. The four lanes l, l^16, l^32, l^48 share a row.
struct FEpiScoreStats {
  template <int FA, int FB>
  __device__ __forceinline__ static void run(const GemmParams& p, Acc16<FA, FB>& acc, int m_base,
                                             int n_base, int lane, int tm, int tn, int wn,
                                             unsigned char* stage) {
    opaque_lane(lane);
    const int part = n_base / (FB * 16);
    const int c0 = 4 * (lane >> 4);  // this lane's first column of each 16-column block
    const int ncols = p.N - n_base;  // columns of this wave inside the vocabulary
    const float scale = p.logit_scale * kLog2e;
#pragma unroll
    for (int i = 0; i < FA; ++i) {
      const int m = m_base + 16 * i + (lane & 15);
      const bool mok = m < p.M;
      // The row's token as a column of this wave's (-1 if outside).
      const long trel = (mok ? p.targets[m] : -1) - n_base;
      const int t = trel >= 0 && trel < FB * 16 && trel < ncols ? (int)trel : -1;
      // Columns past the vocabulary add e^-inf = 0. (A branch of the whole wave: as selections,
      // in every wave, they spilled registers and cost 8000 x 32768 x 1280 6 % of its time.)
      if (ncols < FB * 16) {
        asm volatile("");
#pragma unroll
        for (int j = 0; j < FB; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (16 * j + c0 + e >= ncols) acc.v[i][j][e] = -INFINITY;
      }
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < FB; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) mx = fmaxf(mx, acc.v[i][j][e]);
      // The token's logit only in the waves where some row's token falls in these columns.
      if (__builtin_amdgcn_ballot_w64(t >= 0) != 0) {
        float tv = 0.0f;
#pragma unroll
        for (int j = 0; j < FB; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) tv = 16 * j + c0 + e == t ? acc.v[i][j][e] : tv;
        if (t >= 0 && (t & 12) == c0) p.tgt_logit[m] = tv;
      }
      mx = fmaxf(mx, __shfl_xor(mx, 16, kWave));
      mx = fmaxf(mx, __shfl_xor(mx, 32, kWave));
      ScoreStats st = {mx, 0.0f, 0.0f};
      const float ref = score_ref(mx);
#pragma unroll
      for (int j = 0; j < FB; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) score_add(st, (acc.v[i][j][e] - ref) * scale);
      st.s += __shfl_xor(st.s, 16, kWave);
      st.s += __shfl_xor(st.s, 32, kWave);
      st.w += __shfl_xor(st.w, 16, kWave);
      st.w += __shfl_xor(st.w, 32, kWave);
      if (mok && lane < 16 && part < p.parts_per_row) {
        const long at = (long)m * p.parts_per_row + part;
        p.part_max[at] = st.m;
        p.part_sum[at] = st.s;
        p.part_wsum[at] = st.w;
      }
    }
  }
};

// The logits' gradient, rounded once to BF16 for the two products that read it, through the
// wave's LDS staging rows into c [M, ldc] (ldc the vocabulary, a multiple of 8, or padded past it
// with zeros to a multiple of 64) as 16-byte row pieces.
struct FEpiScoreGrad {
  template <int FA, int FB>
  __device__ __forceinline__ static void run(const GemmParams& p, Acc16<FA, FB>& acc, int m_base,
                                             int n_base, int lane, int tm, int tn, int wn,
                                             unsigned char* stage) {
    // LPR lanes cover a row of the wave tile (8 columns each), RPI rows per instruction.
    constexpr int LPR = FB * 2, RPI = 64 / LPR, NQ = FA * 16 / RPI;
    static_assert(64 % LPR == 0 && NQ >= 1, "whole rows per instruction");
    opaque_lane(lane);
    const int c0 = 4 * (lane >> 4), ncols = p.N - n_base;
    const float scale = p.logit_scale;
#pragma unroll
    for (int i = 0; i < FA; ++i) {
      const int m = m_base + 16 * i + (lane & 15);
      const bool mok = m < p.M;
      const f32x4_t c = mok ? *reinterpret_cast<const f32x4_t*>(p.row_coef + 4L * m) : f32x4_t{0.f, 0.f, 0.f, 0.f};
      const long trel = (mok ? p.targets[m] : -1) - n_base;
      const int t = trel >= 0 && trel < FB * 16 && trel < ncols ? (int)trel : -1;
      // A row without upstream gradient has none, whatever its logits.
      const bool none = c[1] == 0.0f && c[2] == 0.0f && c[3] == 0.0f;
      const bool some = __builtin_amdgcn_ballot_w64(t >= 0) != 0;
#pragma unroll
      for (int j = 0; j < FB; ++j) {
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[e] = score_grad(acc.v[i][j][e] * scale - c[0], c);
          if (some && 16 * j + c0 + e == t) v[e] += c[3];
          if (none || (ncols < FB * 16 && 16 * j + c0 + e >= ncols)) v[e] = 0.0f;
        }
        const u32x2_t w = {pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
        *reinterpret_cast<u32x2_t*>(stage + (16 * i + (lane & 15)) * epi_row<FB>() + (16 * j + c0) * 2) = w;
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): this wave's staging writes landed
    const int c8 = 8 * (lane % LPR);
    const bool full = n_base + c8 + 7 < (int)p.ldc;
    __amdgpu_buffer_rsrc_t rc = make_rsrc(p.c + (long)m_base * p.ldc + n_base, 0x7fffffff);
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      const int r = RPI * q + lane / LPR;
      const bool ok = m_base + r < p.M && full;
      const u32x4_t v = *reinterpret_cast<const u32x4_t*>(stage + r * epi_row<FB>() + c8 * 2);
      __builtin_amdgcn_raw_buffer_store_b128(v, rc, store_off(ok, (long)r * p.ldc + c8, 2), 0, kEpiNT);
    }
  }
};

}  // namespace ws
