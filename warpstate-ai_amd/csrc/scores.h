// Token scores: of each row of logits l (scaled by 1 / temperature), the log probability of a
// given token, the entropy, and the k likeliest tokens,
//   lse = m + log S,  S = sum e^(l - m),  W = sum e^(l - m) (l - m),  m = max l,
//   logprob = l_t - lse,  entropy = log S - W / S,
// and their gradient, with g and h the upstream gradients of logprob and entropy:
//   dl_j = g [j = t] - p_j (g + h (log p_j + entropy)),  p_j = e^(l_j - lse).
// A part of a row is summed up as (m, S, W); parts join by rescaling to the larger maximum m':
//   S' = e^(m - m') S,  W' = e^(m - m') (W + (m - m') S).
// Logits of -inf (a vocabulary mask) have p = 0 and add nothing; a row of nothing else has no
// distribution and gets NaN. A token of -100 has logprob 0 and no g; another token outside the
// vocabulary gets NaN. All sums are FP32.
#pragma once

#include "common.h"

namespace ws {

constexpr long kIgnored = -100;

struct ScoreStats {
  float m, s, w;
};
// l - m where l may be -inf: 0 then, for products with a zero weight.
__device__ __forceinline__ float score_shift(float l, float m) { return l == -INFINITY ? 0.0f : l - m; }
// The finite reference point for a maximum that may be -inf (nothing seen yet).
__device__ __forceinline__ float score_ref(float m) { return m == -INFINITY ? 0.0f : m; }
__device__ __forceinline__ void score_add(ScoreStats& a, float l, float ref) {
  const float e = exp_e(l - ref);
  a.s += e;
  a.w += e * score_shift(l, ref);
}
__device__ __forceinline__ ScoreStats score_join(const ScoreStats& a, const ScoreStats& b) {
  ScoreStats r;
  r.m = fmaxf(a.m, b.m);
  const float ref = score_ref(r.m);
  const float ea = exp_e(a.m - ref), eb = exp_e(b.m - ref);
  r.s = ea * a.s + eb * b.s;
  r.w = ea * (a.w + score_shift(a.m, ref) * a.s) + eb * (b.w + score_shift(b.m, ref) * b.s);
  return r;
}
__device__ __forceinline__ ScoreStats score_join_wave(ScoreStats v) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) {
    const ScoreStats o = {__shfl_xor(v.m, off, kWave), __shfl_xor(v.s, off, kWave), __shfl_xor(v.w, off, kWave)};
    v = score_join(v, o);
  }
  return v;
}

// Outputs of a row. `target` is the scaled logit of its token (read only where that is valid).
struct ScoreOut {
  float *lse, *logprob, *entropy;
};
__device__ __forceinline__ float score_finish(const ScoreOut& o, long row, const ScoreStats& st, long token,
                                              long vocab, float target) {
  const float log_s = log_e(st.s), lse = st.m + log_s;
  o.lse[row] = lse;
  o.entropy[row] = log_s - st.w / st.s;
  o.logprob[row] = token == kIgnored ? 0.0f : token >= 0 && token < vocab ? target - lse : NAN;
  return lse;
}

// ---------------------------------------------------------------------------------------
// From logits [rows, vocab] in memory. HBM-bound: each logit is read once. A workgroup of 256
// threads takes 256 * EPT logits of a row into registers: the maximum, then the sums against
// it, and the part's k likeliest tokens. Rows longer than that are split over workgroups and
// joined by score_join_kernel.
//
// The k largest of a part, by (logit, lowest id first): an order-preserving integer of the logit with the
// complemented id below it makes every key different. The part's 64 groups of four threads
// give their largest keys; the k-th largest of those, T, is at most the part's k-th largest key,
// so every key >= T is a candidate, and in ordinary data few others are. They are collected in
// LDS (in any order) and each is placed by the number of larger ones.
constexpr int kScoreGroups = 64;
constexpr int kMaxTopK = kScoreGroups;
constexpr int kScoreCandidates = 2048;
constexpr int kMaxScoreParts = 64;

// Ascending in the logit's order; -0 as 0. The lowest key, 0, is no logit's (-inf has
// 0x007fffff) and stands for places past the vocabulary.
__device__ __forceinline__ unsigned score_key(float x) {
  const unsigned u = __float_as_uint(x + 0.0f);
  return u ^ ((unsigned)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float score_unkey(unsigned k) {
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
__device__ __forceinline__ unsigned long score_pack(unsigned key, unsigned id) {
  return (unsigned long)key << 32 | (unsigned)~id;
}
__device__ __forceinline__ unsigned long shfl_xor_u64(unsigned long v, int off) {
  const unsigned lo = (unsigned)__shfl_xor((int)v, off, kWave), hi = (unsigned)__shfl_xor((int)(v >> 32), off, kWave);
  return (unsigned long)hi << 32 | lo;
}

// Eight logits from `src`, `left` of them inside the row (any alignment: 16-byte loads need
// none on this target), -inf past it.
template <bool F32>
__device__ __forceinline__ void load_logits8(const void* src, long at, long left, float (&x)[8]) {
  if (left >= 8) {
    if constexpr (F32) {
      f32x4_t v[2];
      __builtin_memcpy(v, static_cast<const float*>(src) + at, 32);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = v[e >> 2][e & 3];
    } else {
      u32x4_t v;
      __builtin_memcpy(&v, static_cast<const unsigned short*>(src) + at, 16);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = (e & 1) ? hi_bf16(v[e >> 1]) : lo_bf16(v[e >> 1]);
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    x[e] = -INFINITY;
    if (e < left) {
      if constexpr (F32) x[e] = static_cast<const float*>(src)[at + e];
      else x[e] = bf16_bits_to_f32(static_cast<const unsigned short*>(src)[at + e]);
    }
  }
}
template <bool F32>
__device__ __forceinline__ float load_logit(const void* src, long at) {
  if constexpr (F32) return static_cast<const float*>(src)[at];
  else return bf16_bits_to_f32(static_cast<const unsigned short*>(src)[at]);
}

struct ScoreParams {
  const void* logits;
  long ld;
  int rows, vocab, parts, top_k;
  float inv_t;
  const long* tokens;
  ScoreOut out;
  float* top_logprobs;
  long* top_ids;
  // Partial results of split rows, [rows][parts] and [rows][parts][top_k].
  f32x4_t* stats;
  unsigned long* keys;
};

__device__ __forceinline__ void score_top(const ScoreParams& p, long row, int i, unsigned long key, float lse) {
  p.top_logprobs[row * p.top_k + i] = score_unkey((unsigned)(key >> 32)) * p.inv_t - lse;
  p.top_ids[row * p.top_k + i] = (long)(unsigned)~(unsigned)key;
}

template <bool F32, int EPT, bool TOPK>
static __global__ void __launch_bounds__(256) score_rows_kernel(const ScoreParams p) {
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const long row = blockIdx.x / p.parts;
  const int part = blockIdx.x % p.parts;
  const int first = part * 256 * EPT + 8 * t;  // element e of piece i: id first + 2048 i + e
  float x[EPT];
#pragma unroll
  for (int i = 0; i < EPT / 8; ++i) {
    float v[8];
    load_logits8<F32>(p.logits, row * p.ld + first + 2048 * i, (long)p.vocab - (first + 2048 * i), v);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[8 * i + e] = v[e];
  }

  __shared__ float red[3][4];
  __shared__ unsigned long groups[TOPK ? kScoreGroups : 1], cand[TOPK ? kScoreCandidates : 1], best[TOPK ? kMaxTopK : 1];
  __shared__ unsigned long threshold, reduce4[4];
  __shared__ int count;

  float mx = x[0];
#pragma unroll
  for (int i = 1; i < EPT; ++i) mx = fmaxf(mx, x[i]);
  mx = wave_max(mx);
  if (lane == 0) red[0][wave] = mx;
  unsigned long mine = 0;
  if constexpr (TOPK) {
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      const int id = first + 2048 * (i / 8) + i % 8;
      const unsigned long key = score_pack(id < p.vocab ? score_key(x[i]) : 0u, (unsigned)id);
      mine = key > mine ? key : mine;
    }
    unsigned long group = mine;
#pragma unroll
    for (int off = 1; off <= 2; off <<= 1) {
      const unsigned long o = shfl_xor_u64(group, off);
      group = o > group ? o : group;
    }
    if ((t & 3) == 0) groups[t >> 2] = group;
    if (t == 0) count = 0;
  }
  __syncthreads();
  ScoreStats st;
  st.m = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3])) * p.inv_t;
  st.s = st.w = 0.0f;
  const float ref = score_ref(st.m);
#pragma unroll
  for (int i = 0; i < EPT; ++i) score_add(st, x[i] * p.inv_t, ref);
  st.s = wave_sum(st.s);
  st.w = wave_sum(st.w);
  if (lane == 0) {
    red[1][wave] = st.s;
    red[2][wave] = st.w;
  }
  if constexpr (TOPK) {
    if (wave == 0) {
      const unsigned long my = groups[lane];
      int larger = 0;
      for (int g = 0; g < kScoreGroups; ++g) larger += groups[g] > my;
      if (larger == p.top_k - 1) threshold = my;
    }
  }
  __syncthreads();
  st.s = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
  st.w = (red[2][0] + red[2][1]) + (red[2][2] + red[2][3]);
  if constexpr (TOPK) {
    const unsigned long T = threshold;
    if (mine >= T) {
#pragma unroll
      for (int i = 0; i < EPT; ++i) {
        const int id = first + 2048 * (i / 8) + i % 8;
        const unsigned long key = score_pack(id < p.vocab ? score_key(x[i]) : 0u, (unsigned)id);
        if (key >= T) {
          const int at = atomicAdd(&count, 1);
          if (at < kScoreCandidates) cand[at] = key;
        }
      }
    }
    __syncthreads();
    const int n = count;
    if (n <= kScoreCandidates) {
      for (int c = t; c < n; c += 256) {
        const unsigned long my = cand[c];
        int larger = 0;
        for (int o = 0; o < n; ++o) larger += cand[o] > my;
        if (larger < p.top_k) best[larger] = my;
      }
      __syncthreads();
    } else {
      // More candidates than LDS holds (the largest logits crowded into few threads): one
      // maximum at a time.
      unsigned long last = ~0ul;
      for (int k = 0; k < p.top_k; ++k) {
        unsigned long m = 0;
#pragma unroll
        for (int i = 0; i < EPT; ++i) {
          const int id = first + 2048 * (i / 8) + i % 8;
          const unsigned long key = score_pack(id < p.vocab ? score_key(x[i]) : 0u, (unsigned)id);
          m = key < last && key > m ? key : m;
        }
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) {
          const unsigned long o = shfl_xor_u64(m, off);
          m = o > m ? o : m;
        }
        if (lane == 0) reduce4[wave] = m;
        __syncthreads();
        const unsigned long a = reduce4[0] > reduce4[1] ? reduce4[0] : reduce4[1];
        const unsigned long b = reduce4[2] > reduce4[3] ? reduce4[2] : reduce4[3];
        last = a > b ? a : b;
        if (t == 0) best[k] = last;
        __syncthreads();
      }
    }
  }
  if (p.parts > 1) {
    if (t == 0) p.stats[blockIdx.x] = f32x4_t{st.m, st.s, st.w, 0.0f};
    if (TOPK && t < p.top_k) p.keys[(long)blockIdx.x * p.top_k + t] = best[t];
    return;
  }
  const long token = p.tokens[row];
  const float lse = st.m + log_e(st.s);
  if (t == 0) {
    const bool valid = token >= 0 && token < p.vocab;
    score_finish(p.out, row, st, token, p.vocab,
                 valid ? load_logit<F32>(p.logits, row * p.ld + token) * p.inv_t : 0.0f);
  }
  if (TOPK && t < p.top_k) score_top(p, row, t, best[t], lse);
}

// Joins the parts of split rows, one wave per row: lane i holds part i (at most 64), its sums
// and the head of its sorted keys; each of the k steps takes the largest head.
template <bool F32>
static __global__ void __launch_bounds__(256) score_join_kernel(const ScoreParams p) {
  const int lane = threadIdx.x & 63;
  const long row = blockIdx.x * 4L + (threadIdx.x >> 6);
  if (row >= p.rows) return;
  ScoreStats st = {-INFINITY, 0.0f, 0.0f};
  const long part = row * p.parts + lane;
  if (lane < p.parts) {
    const f32x4_t v = p.stats[part];
    st = ScoreStats{v[0], v[1], v[2]};
  }
  st = score_join_wave(st);
  const float lse = st.m + log_e(st.s);
  if (lane == 0) {
    const long token = p.tokens[row];
    const bool valid = token >= 0 && token < p.vocab;
    score_finish(p.out, row, st, token, p.vocab,
                 valid ? load_logit<F32>(p.logits, row * p.ld + token) * p.inv_t : 0.0f);
  }
  const unsigned long* keys = p.keys + part * p.top_k;
  int at = 0;
  unsigned long head = p.top_k > 0 && lane < p.parts ? keys[0] : 0ul;
  for (int k = 0; k < p.top_k; ++k) {
    unsigned long m = head;
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) {
      const unsigned long o = shfl_xor_u64(m, off);
      m = o > m ? o : m;
    }
    if (lane == 0) score_top(p, row, k, m, lse);
    if (head == m && lane < p.parts) head = ++at < p.top_k ? keys[at] : 0ul;
  }
}

// ---------------------------------------------------------------------------------------
// Coefficients of a row's gradient, dl_j / temperature = [j = t] c[3] - p_j (c[1] + c[2] log p_j)
// with c[0] = lse. c[1] is NaN for a token that has no score.
static __global__ void __launch_bounds__(256) score_coef_kernel(const long* tokens, const float* lse,
                                                                const float* entropy, const float* dlogprob,
                                                                const float* dentropy, float inv_t, int rows,
                                                                int vocab, f32x4_t* coef) {
  const int row = blockIdx.x * 256 + threadIdx.x;
  if (row >= rows) return;
  const long token = tokens[row];
  const bool valid = token >= 0 && token < vocab;
  const float g = dlogprob && token != kIgnored ? (valid ? dlogprob[row] : NAN) : 0.0f;
  const float h = dentropy ? dentropy[row] : 0.0f;
  coef[row] = f32x4_t{lse[row], h == 0.0f ? inv_t * g : inv_t * (g + h * entropy[row]), inv_t * h, inv_t * g};
}

// One gradient value from a scaled logit. p = 0 gives 0 (log p is -inf there).
__device__ __forceinline__ float score_grad(float l, const f32x4_t& c) {
  const float logp = l - c[0], pr = exp_e(logp);
  return pr == 0.0f ? 0.0f : -pr * (c[1] + c[2] * logp);
}

template <bool F32>
static __global__ void __launch_bounds__(256) score_grad_kernel(const ScoreParams p, const float* dlogprob,
                                                                const float* dentropy, void* out, long ld_out,
                                                                int segments) {
  const long row = blockIdx.x / segments;
  const int id0 = (int)(blockIdx.x % segments) * 2048 + 8 * threadIdx.x;
  if (id0 >= p.vocab) return;
  const long token = p.tokens[row];
  const bool valid = token >= 0 && token < p.vocab;
  const float g = dlogprob && token != kIgnored ? (valid ? dlogprob[row] : NAN) : 0.0f;
  const float h = dentropy ? dentropy[row] : 0.0f;
  // A row without upstream gradient has none, whatever its logits.
  const bool none = g == 0.0f && h == 0.0f;
  const f32x4_t c = {p.out.lse[row], h == 0.0f ? p.inv_t * g : p.inv_t * (g + h * p.out.entropy[row]),
                     p.inv_t * h, p.inv_t * g};
  float x[8];
  const long left = (long)p.vocab - id0;
  if (none) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = 0.0f;
  } else {
    load_logits8<F32>(p.logits, row * p.ld + id0, left, x);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = score_grad(x[e] * p.inv_t, c);
      if (id0 + e == token) x[e] += c[3];
    }
  }
  const long at = row * ld_out + id0;
  if constexpr (F32) {
    float* o = static_cast<float*>(out) + at;
    if (left >= 8) {
      __builtin_memcpy(o, x, 32);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < left) o[e] = x[e];
    }
  } else {
    auto* o = static_cast<unsigned short*>(out) + at;
    u32x4_t v;
#pragma unroll
    for (int d = 0; d < 4; ++d) v[d] = pack_bf16x2(x[2 * d], x[2 * d + 1]);
    if (left >= 8) {
      __builtin_memcpy(o, &v, 16);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < left) o[e] = (unsigned short)(v[e >> 1] >> (16 * (e & 1)));
    }
  }
}

// ---------------------------------------------------------------------------------------
// From the LM head's products: joins the parts' statistics of a row, one wave per row.
static __global__ void __launch_bounds__(256) score_combine_kernel(const float* pm, const float* ps,
                                                                   const float* pw, int parts,
                                                                   const float* target, const long* tokens,
                                                                   ScoreOut out, int rows, int vocab) {
  const int lane = threadIdx.x & 63;
  const long row = blockIdx.x * 4L + (threadIdx.x >> 6);
  if (row >= rows) return;
  ScoreStats st = {-INFINITY, 0.0f, 0.0f};
  for (int q = lane; q < parts; q += 64) {
    const long i = row * parts + q;
    st = score_join(st, ScoreStats{pm[i], ps[i], pw[i]});
  }
  st = score_join_wave(st);
  if (lane == 0) {
    const long token = tokens[row];
    score_finish(out, row, st, token, vocab, token >= 0 && token < vocab ? target[row] : 0.0f);
  }
}

}  // namespace ws
