// Token scores: of each row of logits l (scaled by 1 / temperature), the log probability of a
// given token, the entropy, and the k likeliest tokens,
//   lse = m + log S,  S = sum e^(l - m),  W = sum e^(l - m) (l - m),  m = max l,
//   logprob = (l_t - m) - log S,  entropy = log S - W / S,
// and their gradient, with g and h the upstream gradients of logprob and entropy:
//   dl_j = g [j = t] - p_j (g + h (log p_j + entropy)),  p_j = e^(l_j - lse).
// A part of a row is summed up as (m, S, W); parts join by rescaling to the larger maximum m':
//   S' = e^(m - m') S,  W' = e^(m - m') (W + (m - m') S).
// Logits of -inf (a vocabulary mask) have p = 0 and add nothing; a row of nothing else has no
// distribution and gets NaN. A token of -100 has logprob 0 and no g; another token outside the
// vocabulary gets NaN. All sums are FP32.
#pragma once

#include <type_traits>

#include "common.h"

namespace ws {

constexpr long kIgnored = -100;

// Logits and their maxima m are held as they are given: only a distance l - m, at most 0, is
// scaled, by log2 e / temperature, so that e^(l - m) is the hardware's base-2 exponential and W is in
// units of log 2. (Scaled first, finite logits above 2.36e38, such as a mask of the type's
// lowest value, would overflow, and at 1e10 the scaled maximum's own rounding is hundreds.) A
// distance beyond FP32's range is -inf, which adds nothing.
struct ScoreStats {
  float m, s, w;
};
__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }
// The finite reference point for a maximum that may be -inf (nothing seen yet).
__device__ __forceinline__ float score_ref(float m) { return m == -INFINITY ? 0.0f : m; }
// Adds a logit y above the reference point. y = -inf adds nothing: the bound keeps 0 y from
// being a NaN.
__device__ __forceinline__ void score_add(ScoreStats& a, float y) {
  const float e = exp2_hw(y);
  a.s += e;
  a.w = __builtin_fmaf(e, fmaxf(y, -1e30f), a.w);
}
__device__ __forceinline__ ScoreStats score_join(const ScoreStats& a, const ScoreStats& b, float scale) {
  ScoreStats r;
  r.m = fmaxf(a.m, b.m);
  const float ref = score_ref(r.m);
  const float ya = (a.m - ref) * scale, yb = (b.m - ref) * scale;
  const float ea = exp2_hw(ya), eb = exp2_hw(yb);
  r.s = __builtin_fmaf(ea, a.s, eb * b.s);
  // (An empty part has m = -inf, s = w = 0.)
  r.w = ea * __builtin_fmaf(fmaxf(ya, -1e30f), a.s, a.w) + eb * __builtin_fmaf(fmaxf(yb, -1e30f), b.s, b.w);
  return r;
}
// Joins the values of `lanes` (a power of two) neighbouring lanes.
__device__ __forceinline__ ScoreStats score_join_lanes(ScoreStats v, int lanes, float scale) {
  for (int off = lanes / 2; off >= 1; off >>= 1) {
    const ScoreStats o = {__shfl_xor(v.m, off, kWave), __shfl_xor(v.s, off, kWave), __shfl_xor(v.w, off, kWave)};
    v = score_join(v, o, scale);
  }
  return v;
}

// Outputs of a row. `target` is its token's logit (read only where the token is valid).
struct ScoreOut {
  float *lse, *logprob, *entropy;
};
// log2 S of finished sums.
__device__ __forceinline__ float score_log(const ScoreStats& st) { return __builtin_amdgcn_logf(st.s); }
// A logit's log probability. The largest logit's own term makes S at least 1, so it is at most 0.
__device__ __forceinline__ float score_logprob(float l, float m, float log_s, float inv_t) {
  return (l - m) * inv_t - log_s * kLn2;
}
__device__ __forceinline__ void score_finish(const ScoreOut& o, long row, const ScoreStats& st, long token,
                                             long vocab, float target, float inv_t) {
  const float log_s = score_log(st);
  o.lse[row] = st.m * inv_t + log_s * kLn2;
  o.entropy[row] = (log_s - st.w / st.s) * kLn2;
  o.logprob[row] = token == kIgnored               ? 0.0f
                   : token >= 0 && token < vocab ? score_logprob(target, st.m, log_s, inv_t)
                                                   : NAN;
}

// ---------------------------------------------------------------------------------------
// From logits [rows, vocab] in memory. HBM-bound: each logit is read once. A workgroup of 256
// threads takes 256 * EPT logits of a row into registers: the maximum, then the sums against
// it, and the part's k likeliest tokens. Rows longer than that are split over workgroups and
// joined by score_join_kernel.
//
// The k largest of a part, by (logit, lowest id first). The part's groups (the threads, or for
// k up to 32 the 64 groups of four threads) give their largest logits; a T that at least k of
// those reach is at most the part's k-th largest logit, so every logit >= T is a candidate, and
// in ordinary data few others are. T is the k-th largest group cut to 16 bits of its key (an
// order-preserving integer of the logit), found bit by bit with ballots over the groups, in
// every wave alike. Each wave collects its candidates in LDS as keys above the complemented
// id, so that all are different, and each is placed by the number of larger ones. Rows with
// many logits equal to T (a mask that leaves fewer than k, say) go another way
// (score_top_slow): the threshold there is the k-th largest of the groups' largest keys, which
// tells equal logits apart by their ids, and if the largest logits crowd into few threads, so
// that even that leaves too many, the keys are taken one maximum at a time.
//
// Few registers (eight workgroups on a compute unit), no scratch and few barriers are what it is
// built for: 4096 x 32768 with the top 20 took 128 us while every logit's 64-bit key was formed
// and compared in 121 registers, 125 with 112 bytes of scratch for a call, 83 inlined, 78 with the
// 64 groups for k up to 32 (a quarter of the comparisons for a few more candidates: k = 32 90.6 ->
// 87.7, k = 48 99.4 -> 104.4), 80 with distances taken before they are scaled, an operation more for
// each logit. Of that the sums take 70 (no top, 3.8 TB/s; 67 while logits were scaled first).
constexpr int kScoreGroups = 64;
constexpr int kMaxTopK = kScoreGroups;
constexpr int kScoreCandidates = 2048, kScoreWaveCandidates = kScoreCandidates / 4;
constexpr int kScoreFewK = 32;
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
  float inv_t, scale;  // 1 / temperature, and that times log2 e
  const long* tokens;
  ScoreOut out;
  float* top_logprobs;
  long* top_ids;
  // Partial results of split rows, [rows][parts] and [rows][parts][top_k].
  f32x4_t* stats;
  unsigned long* keys;
};

__device__ __forceinline__ void score_top(const ScoreParams& p, long row, int i, unsigned long key,
                                          const ScoreStats& st, float log_s) {
  p.top_logprobs[row * p.top_k + i] = score_logprob(score_unkey((unsigned)(key >> 32)), st.m, log_s, p.inv_t);
  p.top_ids[row * p.top_k + i] = (long)(unsigned)~(unsigned)key;
}

__device__ __forceinline__ unsigned long max_u64(unsigned long a, unsigned long b) { return a > b ? a : b; }

constexpr int kScoreWaves = 4;
struct ScoreShared {
  unsigned long group_keys[kScoreGroups], cand[kScoreCandidates], best[kMaxTopK], reduce[kScoreWaves], threshold;
  int count, wave_count[kScoreWaves];
};

// A part's logits read again, eight at a time: f(key) of each inside the row.
template <bool F32, int EPT, class F>
__device__ __forceinline__ void score_each_key(const ScoreParams& p, long row, int first, F&& f) {
#pragma unroll 1
  for (int i = 0; i < EPT / 8; ++i) {
    const int id = first + 2048 * i;
    const long left = (long)p.vocab - id;
    float v[8];
    load_logits8<F32>(p.logits, row * p.ld + id, left, v);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < left) f(score_pack(score_key(v[e]), (unsigned)(id + e)));
  }
}

// The part's k largest keys into sh.best where the list of candidates overflowed.
template <bool F32, int EPT>
__device__ __forceinline__ void score_top_slow(const ScoreParams& p, long row, int first, ScoreShared& sh) {
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, k = p.top_k;
  if (t == 0) sh.count = 0;
  unsigned long mine = 0;
  score_each_key<F32, EPT>(p, row, first, [&](unsigned long key) { mine = max_u64(mine, key); });
  unsigned long g = max_u64(mine, shfl_xor_u64(mine, 1));
  g = max_u64(g, shfl_xor_u64(g, 2));
  if ((t & 3) == 0) sh.group_keys[t >> 2] = g;
  if (t == 0) sh.threshold = 0;
  __syncthreads();
  if (wave == 0) {
    const unsigned long my = sh.group_keys[lane];
    int larger = 0;
    for (int o = 0; o < kScoreGroups; ++o) larger += sh.group_keys[o] > my;
    if (larger == k - 1 && my != 0) sh.threshold = my;
  }
  __syncthreads();
  const unsigned long T = sh.threshold;
  if (mine >= T) {
    score_each_key<F32, EPT>(p, row, first, [&](unsigned long key) {
      if (key < T) return;
      const int at = atomicAdd(&sh.count, 1);
      if (at < kScoreCandidates) sh.cand[at] = key;
    });
  }
  __syncthreads();
  const int n = sh.count;
  if (n <= kScoreCandidates) {
    for (int c = t; c < n; c += 256) {
      const unsigned long my = sh.cand[c];
      int larger = 0;
      for (int o = 0; o < n; ++o) larger += sh.cand[o] > my;
      if (larger < k) sh.best[larger] = my;
    }
    // A part with fewer logits than k: the lowest key, which no logit has, for the others.
    for (int c = n + t; c < k; c += 256) sh.best[c] = 0;
    __syncthreads();
    return;
  }
  unsigned long last = ~0ul;
  for (int q = 0; q < k; ++q) {
    unsigned long m = 0;
    score_each_key<F32, EPT>(p, row, first, [&](unsigned long key) { m = key < last && key > m ? key : m; });
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) m = max_u64(m, shfl_xor_u64(m, off));
    if (lane == 0) sh.reduce[wave] = m;
    __syncthreads();
    last = max_u64(max_u64(sh.reduce[0], sh.reduce[1]), max_u64(sh.reduce[2], sh.reduce[3]));
    if (t == 0) sh.best[q] = last;
    __syncthreads();
  }
}

template <bool F32, int EPT, bool TOPK>
static __global__ void __launch_bounds__(256) score_rows_kernel(const ScoreParams p) {
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const long row = blockIdx.x / p.parts;
  // Element e of piece i: id first + 2048 i + e.
  const int first = (int)(blockIdx.x % p.parts) * 256 * EPT + 8 * t;
  float x[EPT];
#pragma unroll
  for (int i = 0; i < EPT / 8; ++i) {
    float v[8];
    const int id = first + 2048 * i;
    load_logits8<F32>(p.logits, row * p.ld + id, (long)p.vocab - id, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[8 * i + e] = v[e];
  }
  __shared__ __attribute__((aligned(16))) float groups[256];
  __shared__ float red[2][kScoreWaves];
  __shared__ std::conditional_t<TOPK, ScoreShared, int> sh;
  float mx = x[0];
#pragma unroll
  for (int i = 1; i < EPT; ++i) mx = fmaxf(mx, x[i]);
  groups[t] = mx;
  __syncthreads();
  const f32x4_t group = *reinterpret_cast<const f32x4_t*>(&groups[4 * lane]);
  const float four = fmaxf(fmaxf(group[0], group[1]), fmaxf(group[2], group[3]));
  ScoreStats st;
  st.m = wave_max(four);
  st.s = st.w = 0.0f;
  if constexpr (TOPK) {
    unsigned T = 0;
    if (p.top_k <= kScoreFewK) {
      const unsigned key = score_key(four);
#pragma unroll
      for (int b = 31; b >= 16; --b) {
        const unsigned with = T | 1u << b;
        if (__builtin_popcountll(__builtin_amdgcn_ballot_w64(key >= with)) >= p.top_k) T = with;
      }
    } else {
      const unsigned key[4] = {score_key(group[0]), score_key(group[1]), score_key(group[2]), score_key(group[3])};
#pragma unroll
      for (int b = 31; b >= 16; --b) {
        const unsigned with = T | 1u << b;
        int n = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) n += __builtin_popcountll(__builtin_amdgcn_ballot_w64(key[e] >= with));
        if (n >= p.top_k) T = with;
      }
    }
    // Keys up to -inf's leave too many: the other way.
    int found = kScoreWaveCandidates + 1;
    if (T > 0x007fffffu) {
      const float cut = score_unkey(T);
      found = 0;
#pragma unroll
      for (int i = 0; i < EPT; ++i) {
        const bool hit = x[i] >= cut;
        const unsigned long hits = __builtin_amdgcn_ballot_w64(hit);
        if (hits != 0) {
          const int at = found + (int)__builtin_amdgcn_mbcnt_hi((unsigned)(hits >> 32),
                                                                 __builtin_amdgcn_mbcnt_lo((unsigned)hits, 0));
          if (hit && at < kScoreWaveCandidates)
            sh.cand[wave * kScoreWaveCandidates + at] =
                score_pack(score_key(x[i]), (unsigned)(first + 2048 * (i / 8) + i % 8));
          found += __builtin_popcountll(hits);
        }
      }
    }
    if (lane == 0) sh.wave_count[wave] = found;
  }
  const float ref = score_ref(st.m);
#pragma unroll
  for (int i = 0; i < EPT; ++i) score_add(st, (x[i] - ref) * p.scale);
  st.s = wave_sum(st.s);
  st.w = wave_sum(st.w);
  if (lane == 0) {
    red[0][wave] = st.s;
    red[1][wave] = st.w;
  }
  __syncthreads();
  st.s = (red[0][0] + red[0][1]) + (red[0][2] + red[0][3]);
  st.w = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
  if constexpr (TOPK) {
    int n[kScoreWaves], most = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kScoreWaves; ++w) {
      n[w] = __builtin_amdgcn_readfirstlane(sh.wave_count[w]);
      most = max(most, n[w]);
      all += n[w];
    }
    // (A NaN compares false: a row of them can leave fewer than k.)
    if (most > kScoreWaveCandidates || all < p.top_k) {
      __syncthreads();  // every thread has read the counts
      score_top_slow<F32, EPT>(p, row, first, sh);
    } else {
      for (int c = lane; c < n[wave]; c += 64) {
        const unsigned long my = sh.cand[wave * kScoreWaveCandidates + c];
        int larger = 0;
#pragma unroll
        for (int w = 0; w < kScoreWaves; ++w)
#pragma unroll 4
          for (int o = 0; o < n[w]; ++o) larger += sh.cand[w * kScoreWaveCandidates + o] > my;
        if (larger < p.top_k) sh.best[larger] = my;
      }
      __syncthreads();
    }
  }
  if (p.parts > 1) {
    if (t == 0) p.stats[blockIdx.x] = f32x4_t{st.m, st.s, st.w, 0.0f};
    if constexpr (TOPK) {
      if (t < p.top_k) p.keys[(long)blockIdx.x * p.top_k + t] = sh.best[t];
    }
    return;
  }
  if (t == 0) {
    const long token = p.tokens[row];
    const bool valid = token >= 0 && token < p.vocab;
    score_finish(p.out, row, st, token, p.vocab, valid ? load_logit<F32>(p.logits, row * p.ld + token) : 0.0f,
                 p.inv_t);
  }
  if constexpr (TOPK) {
    if (t < p.top_k) score_top(p, row, t, sh.best[t], st, score_log(st));
  }
}

// Joins the parts of split rows, blockDim.x / threads rows per workgroup. The first `lanes` lanes
// of a row's threads (a power of two, at least the parts) join its sums. A key's place among the
// row's is the number of larger keys in every part's sorted list, found by bisection in LDS,
// four lists side by side and `per_key` neighbouring lanes on a key (one row of 16 parts, 8 keys
// each: 8.0 us with one list after the other, 6.3 with four at once, 3.8 with four lanes a
// key; 4096 rows of 4 parts, 20 keys each: 7.5, 7.1, and 12 while the largest head was taken
// over and over). With more keys than threads, neighbouring threads take the parts' keys of one
// place, so that whole waves skip the places whose keys are below what the k-th largest is at least
// (scores of 2048 rows of 16 parts, 64 keys each, 245 -> 208 us, 20 each 157 -> 150; 4 parts of 20,
// with fewer keys than threads, would take 1 us longer).
constexpr int kScoreJoinAt = 4, kScoreJoinThreads = 1024;
template <bool F32>
static __global__ void __launch_bounds__(kScoreJoinThreads) score_join_kernel(const ScoreParams p, int threads,
                                                                              int lanes, int per_key) {
  extern __shared__ unsigned long join_keys[];
  __shared__ float joined[4][2];
  const int t = threadIdx.x % threads, slot = threadIdx.x / threads;
  const long row = (long)blockIdx.x * (blockDim.x / threads) + slot;
  const int k = p.top_k, total = p.parts * k;
  const bool ok = row < p.rows;
  unsigned long* keys = join_keys + slot * total;
  // (All requested before any is waited for; a row past the last reads the last one's.)
  const long at = ok ? row : p.rows - 1;
  const long token = p.tokens[at];
  const f32x4_t part = p.stats[at * p.parts + min(t, p.parts - 1)];
  const unsigned long key = k ? p.keys[at * total + min(t, total - 1)] : 0;
  const float target = token >= 0 && token < p.vocab ? load_logit<F32>(p.logits, at * p.ld + token) : 0.0f;
  if (t < total) keys[t] = key;
  for (int i = t + threads; i < total; i += threads) keys[i] = p.keys[at * total + i];
  ScoreStats st = {-INFINITY, 0.0f, 0.0f};
  if (t < p.parts) st = ScoreStats{part[0], part[1], part[2]};
  st = score_join_lanes(st, lanes, p.scale);
  if (ok && t == 0) {
    score_finish(p.out, row, st, token, p.vocab, target, p.inv_t);
    joined[slot][0] = st.m;
    joined[slot][1] = score_log(st);
  }
  if (k == 0) return;  // uniform
  __syncthreads();
  if (!ok) return;
  st.m = joined[slot][0];
  const float log_s = joined[slot][1];
  int most = 1;  // the largest power of two up to k
  while (2 * most <= k) most *= 2;
  const bool many = total > threads;  // (uniform: then per_key is 1)
  unsigned long bound = 0;
  if (many) {
    // The row's k-th largest key is at least each part's k-th, and at least the least of the
    // parts' j-th, as `parts` times j reach k.
    const int part_of = t % lanes;
    unsigned long least = ~0ul;
    if (part_of < p.parts) {
      least = keys[part_of * k + (k - 1) / p.parts];
      bound = keys[part_of * k + k - 1];
    }
    for (int off = lanes / 2; off; off >>= 1) {
      const unsigned long o = shfl_xor_u64(least, off);
      least = o < least ? o : least;
      bound = max_u64(bound, shfl_xor_u64(bound, off));
    }
    bound = max_u64(bound, least);
  }
  for (int i = t / per_key; i < total; i += threads / per_key) {
    const unsigned long my = keys[many ? i % p.parts * k + i / p.parts : i];
    int larger = my < bound ? k : 0;
    for (int q = t % per_key * kScoreJoinAt; q < p.parts && larger < k; q += per_key * kScoreJoinAt) {
      // Keys of these parts' descending lists that are larger (a part past the last: none).
      int n[kScoreJoinAt] = {};
      for (int step = most; step; step >>= 1) {
        unsigned long other[kScoreJoinAt];
#pragma unroll
        for (int u = 0; u < kScoreJoinAt; ++u)
          other[u] = keys[min(q + u, p.parts - 1) * k + min(n[u] + step, k) - 1];
#pragma unroll
        for (int u = 0; u < kScoreJoinAt; ++u)
          n[u] += (q + u < p.parts) & (n[u] + step <= k) & (other[u] > my) ? step : 0;
      }
#pragma unroll
      for (int u = 0; u < kScoreJoinAt; ++u) larger += n[u];
    }
    for (int off = per_key / 2; off; off >>= 1) larger += __shfl_xor(larger, off, kWave);
    // (The key 0 of a part with fewer logits than k is never among the row's k largest.)
    if (larger < k && my != 0 && t % per_key == 0) score_top(p, row, larger, my, st, log_s);
  }
}

// ---------------------------------------------------------------------------------------
// A log probability's upstream gradient: none for an ignored token; of a token that has no score,
// NaN unless it is zero (a row outside the loss).
__device__ __forceinline__ float score_upstream(const float* dlogprob, long row, long token, bool valid) {
  const float g = dlogprob && token != kIgnored ? dlogprob[row] : 0.0f;
  return valid || g == 0.0f ? g : NAN;
}

// Coefficients of a row's gradient, dl_j / temperature = [j = t] c[3] - p_j (c[1] + c[2] log p_j)
// with c[0] = lse. c[1] is NaN for a token that has no score but a gradient.
static __global__ void __launch_bounds__(256) score_coef_kernel(const long* tokens, const float* lse,
                                                                const float* entropy, const float* dlogprob,
                                                                const float* dentropy, float inv_t, int rows,
                                                                int vocab, f32x4_t* coef) {
  const int row = blockIdx.x * 256 + threadIdx.x;
  if (row >= rows) return;
  const long token = tokens[row];
  const bool valid = token >= 0 && token < vocab;
  const float g = score_upstream(dlogprob, row, token, valid);
  const float h = dentropy ? dentropy[row] : 0.0f;
  coef[row] = f32x4_t{lse[row], h == 0.0f ? inv_t * g : inv_t * (g + h * entropy[row]), inv_t * h, inv_t * g};
}

// One gradient value from a log probability. p = 0 gives 0 (log p may be -inf there).
__device__ __forceinline__ float score_grad(float logp, const f32x4_t& c) {
  const float pr = exp_e(logp);
  return pr == 0.0f ? 0.0f : -pr * (c[1] + c[2] * logp);
}

// A probability taken from an lse of up to this size is off by at most half a step of it, 2^-17.
// Beyond, where the step comes to hide the sum of the row's distances (and with a mask of the
// type's lowest value all of it), a row's gradient sums the row again (4096 x 32768 BF16 logits
// 132 -> 596 us if every row is such, 1000 x 10883 38 -> 41).
constexpr float kLseReach = 256.0f;

// (m, S) of a whole row, by all of a workgroup's 256 threads (W is left out).
template <bool F32>
__device__ __forceinline__ ScoreStats score_row_sum(const ScoreParams& p, long row) {
  const int t = threadIdx.x;
  __shared__ float red[2][kScoreWaves];
  ScoreStats st = {-INFINITY, 0.0f, 0.0f};
#pragma unroll 1
  for (int id = 8 * t; id < p.vocab; id += 2048) {
    float x[8];
    load_logits8<F32>(p.logits, row * p.ld + id, (long)p.vocab - id, x);
    ScoreStats piece = {x[0], 0.0f, 0.0f};
#pragma unroll
    for (int e = 1; e < 8; ++e) piece.m = fmaxf(piece.m, x[e]);
    const float ref = score_ref(piece.m);
#pragma unroll
    for (int e = 0; e < 8; ++e) piece.s += exp2_hw((x[e] - ref) * p.scale);
    st = score_join(st, piece, p.scale);
  }
  st = score_join_lanes(st, kWave, p.scale);
  if ((t & 63) == 0) {
    red[0][t >> 6] = st.m;
    red[1][t >> 6] = st.s;
  }
  __syncthreads();
  st = ScoreStats{red[0][0], red[1][0], 0.0f};
#pragma unroll
  for (int w = 1; w < kScoreWaves; ++w) st = score_join(st, ScoreStats{red[0][w], red[1][w], 0.0f}, p.scale);
  return st;
}

// A workgroup takes every `segments`-th piece of 2048 logits of a row: one piece, or, where the
// gradient goes over the logits, all of them (no other workgroup may have written what it sums).
template <bool F32>
static __global__ void __launch_bounds__(256) score_grad_kernel(const ScoreParams p, const float* dlogprob,
                                                                const float* dentropy, void* out, long ld_out,
                                                                int segments) {
  const long row = blockIdx.x / segments;
  const long token = p.tokens[row];
  const bool valid = token >= 0 && token < p.vocab;
  const float g = score_upstream(dlogprob, row, token, valid);
  const float h = dentropy ? dentropy[row] : 0.0f;
  // A row without upstream gradient has none, whatever its logits.
  const bool none = g == 0.0f && h == 0.0f;
  // log p = (l - m) / temperature - log_s.
  float m = 0.0f, log_s = p.out.lse[row];
  if (!none && !(fabsf(log_s) < kLseReach)) {  // (the same for the whole workgroup)
    const ScoreStats st = score_row_sum<F32>(p, row);
    m = st.m;
    log_s = score_log(st) * kLn2;
  }
  const f32x4_t c = {0.0f, h == 0.0f ? p.inv_t * g : p.inv_t * (g + h * p.out.entropy[row]), p.inv_t * h,
                     p.inv_t * g};
#pragma unroll 1
  for (long id0 = blockIdx.x % segments * 2048L + 8 * threadIdx.x; id0 < p.vocab; id0 += segments * 2048L) {
    float x[8];
    const long left = p.vocab - id0;
    if (none) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = 0.0f;
    } else {
      load_logits8<F32>(p.logits, row * p.ld + id0, left, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = score_grad((x[e] - m) * p.inv_t - log_s, c);
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
}

// ---------------------------------------------------------------------------------------
// From the LM head's products: joins the parts' statistics of a row, one wave per row.
static __global__ void __launch_bounds__(256) score_combine_kernel(const float* pm, const float* ps,
                                                                   const float* pw, int parts,
                                                                   const float* target, const long* tokens,
                                                                   ScoreOut out, int rows, int vocab,
                                                                   float inv_t) {
  const int lane = threadIdx.x & 63;
  const long row = blockIdx.x * 4L + (threadIdx.x >> 6);
  if (row >= rows) return;
  ScoreStats st = {-INFINITY, 0.0f, 0.0f};
  for (int q = lane; q < parts; q += 64) {
    const long i = row * parts + q;
    st = score_join(st, ScoreStats{pm[i], ps[i], pw[i]}, inv_t * kLog2e);
  }
  st = score_join_lanes(st, kWave, inv_t * kLog2e);
  if (lane == 0) {
    const long token = tokens[row];
    score_finish(out, row, st, token, vocab, token >= 0 && token < vocab ? target[row] : 0.0f, inv_t);
  }
}

}  // namespace ws
