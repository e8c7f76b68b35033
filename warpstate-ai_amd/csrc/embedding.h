// Embedding lookup with scaling, and the table's gradient by sorted tokens.
//
//   y[t] = r(scale W[token t]),   dW[v] = scale sum over t with token t = v of dy[t]
//
// The gradient's sums are FP32 and taken in the order of t (in pieces of it for tokens that occur
// often), so that a call gives the same bits every time: the tokens' positions are sorted by
// token first, stably, and each row of the table is then written once, zeros included.
//
// HBM-bound: rows of the table and of y once; dy once and the table's gradient once. The sort reads
// the tokens, some hundred kilobytes that stay in L2.
#pragma once

#include "residual_norm.h"

namespace ws {

constexpr long kIgnoredToken = -100;

// A wave per token, 64 x 8 columns at a time. Ignored tokens get zeros, others outside the
// vocabulary NaN; neither reads the table.
template <bool TF32, bool OF32, bool VEC>
static __global__ void __launch_bounds__(256) embed_lookup_kernel(const void* table, long ld, const long* tokens,
                                                                  int rows, int vocab, int d, float scale, void* y) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = blockIdx.x * 4 + wave;
  if (row >= rows) return;
  const long token = tokens[row];
  const bool known = token >= 0 && token < vocab;
  const float fill = token == kIgnoredToken ? 0.0f : __uint_as_float(0x7fc00000u);
#pragma unroll 4
  for (int c = 8 * lane; c < d; c += 512) {
    QuantRow<TF32> v;
    if (known) load_piece<TF32, VEC>(v, table, token * ld + c, d - c);
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = known ? v.at(e) * scale : fill;
    store_piece<OF32, VEC>(round_piece<OF32>(f), y, (long)row * d + c, d - c);
  }
}

// Positions of the tokens sorted by token, stably: perm[start[v] .. start[v + 1]) are those of
// token v in order; positions of tokens outside the vocabulary are left out. A workgroup owns
// `range` tokens of the vocabulary and reads all positions twice, each of its sixteen waves a
// sixteenth of them: it counts its own tokens by wave and the ones below its range, which is
// where its part of perm begins, and then places its own. No workgroup waits for another.
constexpr int kSortWaves = 16, kSortRange = 512;

static __global__ void __launch_bounds__(64 * kSortWaves) embed_sort_kernel(const long* __restrict__ tokens, int rows,
                                                                            int vocab, int range,
                                                                            int* __restrict__ start,
                                                                            int* __restrict__ perm) {
  __shared__ int count[kSortWaves][kSortRange];
  __shared__ int below[kSortWaves], scan[kSortWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lo = blockIdx.x * range, n = min(range, vocab - lo);
  const int slice = cdiv(cdiv(rows, 64), kSortWaves) * 64;
  const int begin = min((long)rows, (long)wave * slice), end = min((long)rows, (long)begin + slice);
  int* const mine = count[wave];
  for (int r = lane; r < n; r += 64) mine[r] = 0;
  __syncthreads();
  int less = 0;
#pragma unroll 4
  for (int t = begin + lane; t < end; t += 64) {
    const long token = tokens[t];
    less += token >= 0 && token < lo;
    if (token >= lo && token < lo + n) atomicAdd(&mine[token - lo], 1);
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) less += __shfl_xor(less, off, kWave);
  if (lane == 0) below[wave] = less;
  __syncthreads();
  // Thread r: token lo + r over all waves, then the running sum over the tokens.
  int total = 0;
  if (tid < n)
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) total += count[w][tid];
  int upto = total;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int other = __shfl_up(upto, off, kWave);
    if (lane >= off) upto += other;
  }
  if (lane == 63) scan[wave] = upto;
  __syncthreads();
  int at = upto - total;
#pragma unroll
  for (int w = 0; w < kSortWaves; ++w) at += below[w] + (w < wave ? scan[w] : 0);
  if (tid < n) {
    start[lo + tid] = at;
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) {
      const int c = count[w][tid];
      count[w][tid] = at;
      at += c;
    }
    if (lo + tid == vocab - 1) start[vocab] = at;
  }
  __syncthreads();
  for (int t0 = begin; t0 < end; t0 += 64) {
    const int t = t0 + lane;
    const long token = t < end ? tokens[t] : -1;
    const bool member = token >= lo && token < lo + n;
    const int r = member ? (int)(token - lo) : -1;
    // One token of the 64 positions at a time; its lanes are in the order of the positions.
    for (unsigned long todo = __builtin_amdgcn_ballot_w64(member); todo != 0;) {
      const int v = __builtin_amdgcn_readlane(r, __builtin_ctzl(todo));
      const unsigned long same = __builtin_amdgcn_ballot_w64(r == v);
      const int first = mine[v];
      if (r == v) perm[first + __builtin_popcountl(same & ((1ul << lane) - 1))] = t;
      mine[v] = first + __builtin_popcountl(same);  // by every lane, the same value
      todo &= ~same;
    }
  }
}

struct EmbedGradParams {
  const void* dy; long ld_dy;
  const long* tokens;
  const int* start;
  const int* perm;
  int vocab, d;
  float scale;
  void* out; long ld_out;
  // Tokens with more than `piece` positions are summed in pieces of perm that begin at multiples
  // of `piece`: the part of one that begins before piece p or with it goes to row 2 p of
  // `partial`, the part of one that begins inside it and runs past it to row 2 p + 1.
  int piece, pieces;
  float* partial; long ld_partial;
};
enum EmbedOut { kEmbedBF16 = 0, kEmbedF32 = 1, kEmbedAdd = 2 };

// Sum of dy at perm[begin .. end) for the 8 NC columns at c, c + 512, ..: the positions of 64 rows
// are one load, a position on each lane, then four rows of dy at a time are in flight. All 64 lanes
// come here, those past the last column too: each holds a position that the others read.
template <bool GF32, int NC, bool VEC>
__device__ __forceinline__ void embed_sum(const EmbedGradParams& p, int begin, int end, int c, int lane,
                                          float (&acc)[NC][8]) {
#pragma unroll
  for (int i = 0; i < NC; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[i][e] = 0.0f;
  constexpr int kAhead = GF32 ? 2 : 4;
  for (int b = begin; b < end; b += 64) {
    const int n = min(64, end - b);
    const int rows = lane < n ? p.perm[b + lane] : 0;
    for (int j = 0; j < n; j += kAhead) {
      QuantRow<GF32> v[kAhead][NC];
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        const long row = __builtin_amdgcn_readlane(rows, min(j + a, n - 1));
#pragma unroll
        for (int i = 0; i < NC; ++i)
          load_piece<GF32, VEC>(v[a][i], p.dy, row * p.ld_dy + c + 512 * i, p.d - c - 512 * i);
      }
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        if (j + a >= n) break;
#pragma unroll
        for (int i = 0; i < NC; ++i)
#pragma unroll
          for (int e = 0; e < 8; ++e) acc[i][e] += v[a][i].at(e);
      }
    }
  }
}

template <int OUT, bool VEC>
__device__ __forceinline__ void embed_store(const EmbedGradParams& p, int v, int c, float (&acc)[8]) {
  const long at = v * p.ld_out + c;
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] *= p.scale;
  if constexpr (OUT == kEmbedAdd) {
    QuantRow<true> old;
    load_piece<true, VEC>(old, p.out, at, p.d - c);
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] += old.at(e);
  }
  store_piece<OUT != kEmbedBF16, VEC>(round_piece<OUT != kEmbedBF16>(acc), p.out, at, p.d - c);
}

// A wave per piece of the sorted positions, then a wave per row of the table.
template <bool GF32, int OUT, bool VEC>
static __global__ void __launch_bounds__(256) embed_grad_kernel(const EmbedGradParams p) {
  constexpr int NC = 4;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long task = blockIdx.x * 4L + wave;
  float acc[NC][8];
  if (task < p.pieces) {
    const int total = p.start[p.vocab], begin = (int)task * p.piece;
    if (begin >= total) return;
    const int end = (int)min((long)total, (long)begin + p.piece);
    const long first = p.tokens[p.perm[begin]], last = p.tokens[p.perm[end - 1]];
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      if (part == 1 && last == first) break;
      const long v = part ? last : first;
      const int s = p.start[v], e = p.start[v + 1];
      if (e - s <= p.piece) continue;
      for (int c0 = 0; c0 < p.d; c0 += 512 * NC) {
        const int c = c0 + 8 * lane;
        embed_sum<GF32, NC, VEC>(p, part ? s : begin, part ? end : min(e, end), c, lane, acc);
#pragma unroll
        for (int i = 0; i < NC; ++i)
          if (c + 512 * i < p.d)
            store_piece<true, true>(round_piece<true>(acc[i]), p.partial,
                                    (2 * task + part) * p.ld_partial + c + 512 * i, 8);
      }
    }
    return;
  }
  const int v = (int)(task - p.pieces);
  if (v >= p.vocab) return;
  const int s = p.start[v], e = p.start[v + 1];
  if (e - s > p.piece || (OUT == kEmbedAdd && s == e)) return;
  for (int c0 = 0; c0 < p.d; c0 += 512 * NC) {
    const int c = c0 + 8 * lane;
    embed_sum<GF32, NC, VEC>(p, s, e, c, lane, acc);
#pragma unroll
    for (int i = 0; i < NC; ++i)
      if (c + 512 * i < p.d) embed_store<OUT, VEC>(p, v, c + 512 * i, acc[i]);
  }
}

// Adds the pieces of the token that begins in piece blockIdx.x and runs past it, in their order.
template <int OUT, bool VEC>
static __global__ void __launch_bounds__(256) embed_join_kernel(const EmbedGradParams p) {
  const int total = p.start[p.vocab], q = blockIdx.x, begin = q * p.piece;
  if (begin >= total) return;
  const int end = (int)min((long)total, (long)begin + p.piece);
  const long v = p.tokens[p.perm[end - 1]];
  const int s = p.start[v], e = p.start[v + 1];
  if (e - s <= p.piece || s < begin) return;
  const int c = 8 * (blockIdx.y * 256 + threadIdx.x);
  if (c >= p.d) return;
  QuantRow<true> x;
  load_piece<true, true>(x, p.partial, (2L * q + (s > begin)) * p.ld_partial + c, 8);
  float acc[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = x.at(i);
#pragma unroll 4
  for (int next = q + 1; (long)next * p.piece < e; ++next) {
    load_piece<true, true>(x, p.partial, 2L * next * p.ld_partial + c, 8);
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] += x.at(i);
  }
  embed_store<OUT, VEC>(p, (int)v, c, acc);
}

}  // namespace ws
