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
typedef unsigned u32x2_any2 __attribute__((ext_vector_type(2), aligned(2)));

// A wave per token, 64 x 8 columns at a time. Ignored tokens get zeros, others outside the
// vocabulary NaN; neither reads the table.
template <bool TF32, bool OF32, bool WHOLE>
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
    if (known) load_piece<TF32, WHOLE>(v, table, token * ld + c, d - c);
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = known ? v.at(e) * scale : fill;
    store_piece<OF32, WHOLE>(round_piece<OF32>(f), y, (long)row * d + c, d - c);
  }
}

// Positions of the tokens sorted by token, stably: perm[start[v] .. start[v + 1]) are those of
// token v in order; positions of tokens outside the vocabulary are left out. A workgroup owns
// `range` tokens of the vocabulary and reads all positions twice, each of its sixteen waves a
// sixteenth of them: it counts its own tokens by wave and the ones below its range, which is
// where its part of perm begins, and then places its own. No workgroup waits for another.
constexpr int kSortWaves = 16, kSortRange = 512, kSortAhead = 16;

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
  // kSortAhead tokens a lane at a time, as distances from the range's first; outside the vocabulary, or
  // past the end, kNoToken.
  constexpr int kNoToken = 0x7fffffff;
  auto load = [&](int t0, int (&r)[kSortAhead]) {
    long token[kSortAhead];
#pragma unroll
    for (int a = 0; a < kSortAhead; ++a) token[a] = t0 + 64 * a + lane < end ? tokens[t0 + 64 * a + lane] : -1;
#pragma unroll
    for (int a = 0; a < kSortAhead; ++a) r[a] = token[a] >= 0 && token[a] < vocab ? (int)token[a] - lo : kNoToken;
  };
  int less = 0, r[kSortAhead];
  for (int t0 = begin; t0 < end; t0 += 64 * kSortAhead) {
    load(t0, r);
#pragma unroll
    for (int a = 0; a < kSortAhead; ++a) {
      less += r[a] < 0;
      if (r[a] >= 0 && r[a] < n) atomicAdd(&mine[r[a]], 1);
    }
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
  for (int t0 = begin; t0 < end; t0 += 64 * kSortAhead) {
    if (end - begin > 64 * kSortAhead) load(t0, r);  // else they are there still
#pragma unroll
    for (int a = 0; a < kSortAhead; ++a) {
      // One token of the 64 positions at a time; its lanes are in the order of the positions.
      for (unsigned long todo = __builtin_amdgcn_ballot_w64(r[a] >= 0 && r[a] < n); todo != 0;) {
        const int v = __builtin_amdgcn_readlane(r[a], __builtin_ctzl(todo));
        const unsigned long same = __builtin_amdgcn_ballot_w64(r[a] == v);
        const int first = mine[v];
        if (r[a] == v) perm[first + __builtin_popcountl(same & ((1ul << lane) - 1))] = t0 + 64 * a + lane;
        mine[v] = first + __builtin_popcountl(same);  // by every lane, the same value
        todo &= ~same;
      }
    }
  }
}

struct EmbedGradParams {
  const void* dy; long ld_dy;
  const long* tokens; int rows;
  const int* start;
  const int* perm;
  int vocab, d;
  int group;  // rows of the table that a wave takes, fewer than 64
  float scale;
  void* out; long ld_out;
  // Tokens with more than `piece` positions are summed in pieces of perm that begin at multiples
  // of `piece`: the part of one that begins before piece p or with it goes to row 2 p of
  // `partial`, the part of one that begins inside it and runs past it to row 2 p + 1.
  int piece, pieces;
  float* partial; long ld_partial;
};
enum EmbedOut { kEmbedBF16 = 0, kEmbedF32 = 1, kEmbedAdd = 2 };

// W elements of a row, 8 or 4: an FP32 output's pieces are four columns wide, so that a wave's stores
// cover whole lines (16384 x 2048 into 32768 rows, the kernel alone, us, pieces of 8 / 4: 83 / 75).
template <bool F32, int W>
struct EmbedPiece {
  unsigned w[F32 ? W : W / 2];
  __device__ __forceinline__ float at(int e) const {
    if constexpr (F32) return __uint_as_float(w[e]);
    else return (e & 1) ? hi_bf16(w[e >> 1]) : lo_bf16(w[e >> 1]);
  }
};
template <bool F32, int W, bool WHOLE>
__device__ __forceinline__ EmbedPiece<F32, W> embed_load(const void* base, long at, int left) {
  constexpr int kWords = F32 ? W : W / 2;
  EmbedPiece<F32, W> v;
  const char* src = static_cast<const char*>(base) + at * (F32 ? 4 : 2);
  if (left >= W) {
    if constexpr (kWords == 2) {
      const u32x2_t a = *reinterpret_cast<const u32x2_any2*>(src);
      v.w[0] = a[0];
      v.w[1] = a[1];
    } else {
#pragma unroll
      for (int q = 0; q < kWords / 4; ++q) {
        const u32x4_t a = reinterpret_cast<const u32x4_any2*>(src)[q];
#pragma unroll
        for (int d = 0; d < 4; ++d) v.w[4 * q + d] = a[d];
      }
    }
    return v;
  }
#pragma unroll
  for (int d = 0; d < kWords; ++d) v.w[d] = 0;
  if (WHOLE || left <= 0) return v;
#pragma unroll
  for (int e = 0; e < W; ++e) {
    if (e >= left) continue;
    if constexpr (F32) v.w[e] = reinterpret_cast<const unsigned*>(src)[e];
    else v.w[e >> 1] |= (unsigned)reinterpret_cast<const unsigned short*>(src)[e] << (16 * (e & 1));
  }
  return v;
}
template <bool F32, int W, bool WHOLE, bool NT = false>
__device__ __forceinline__ void embed_write(const float (&f)[W], void* base, long at, int left) {
  char* dst = static_cast<char*>(base) + at * (F32 ? 4 : 2);
  if (left >= W) {
    if constexpr (F32) {
#pragma unroll
      for (int q = 0; q < W / 4; ++q) {
        const u32x4_t v = {__float_as_uint(f[4 * q]), __float_as_uint(f[4 * q + 1]), __float_as_uint(f[4 * q + 2]),
                           __float_as_uint(f[4 * q + 3])};
        if constexpr (NT) __builtin_nontemporal_store(v, reinterpret_cast<u32x4_any4*>(dst) + q);
        else reinterpret_cast<u32x4_any4*>(dst)[q] = v;
      }
    } else {
      static_assert(F32 || W == 8, "BF16 pieces are 16 bytes");
      const u32x4_t v = {pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[W - 4], f[W - 3]),
                         pack_bf16x2(f[W - 2], f[W - 1])};
      if constexpr (NT) __builtin_nontemporal_store(v, reinterpret_cast<u32x4_any2*>(dst));
      else *reinterpret_cast<u32x4_any2*>(dst) = v;
    }
    return;
  }
  if (WHOLE || left <= 0) return;
#pragma unroll
  for (int e = 0; e < W; ++e) {
    if (e >= left) continue;
    if constexpr (F32) reinterpret_cast<float*>(dst)[e] = f[e];
    else reinterpret_cast<unsigned short*>(dst)[e] = to_bf16_bits(f[e]);
  }
}

// Walks the positions [begin, end) of perm with the sums of dy over the NC pieces of W columns at c,
// c + 64 W, ..: the positions of 64 rows are one load, a position on each lane (so all 64 lanes come here, those
// past the last column too), and then kAhead rows of dy at a time are in flight. `before(at, acc)`
// comes before the row at position `at` is added, and may store the sums and clear them.
template <bool GF32, int NC, int W, bool WHOLE, class Before>
__device__ __forceinline__ void embed_walk(const EmbedGradParams& p, int begin, int end, int c, int lane,
                                           float (&acc)[NC][W], Before&& before) {
  constexpr int kAhead = GF32 ? 2 : 4;
  for (int b = begin; b < end; b += 64) {
    const int n = min(64, end - b);
    const int rows = lane < n ? p.perm[b + lane] : 0;
    for (int j = 0; j < n; j += kAhead) {
      EmbedPiece<GF32, W> v[kAhead][NC];
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        const long row = __builtin_amdgcn_readlane(rows, min(j + a, n - 1));
#pragma unroll
        for (int i = 0; i < NC; ++i)
          v[a][i] = embed_load<GF32, W, WHOLE>(p.dy, row * p.ld_dy + c + 64 * W * i, p.d - c - 64 * W * i);
      }
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        if (j + a >= n) break;
        before(b + j + a);
#pragma unroll
        for (int i = 0; i < NC; ++i)
#pragma unroll
          for (int e = 0; e < W; ++e) acc[i][e] += v[a][i].at(e);
      }
    }
  }
}
template <int NC, int W>
__device__ __forceinline__ void embed_clear(float (&acc)[NC][W]) {
#pragma unroll
  for (int i = 0; i < NC; ++i)
#pragma unroll
    for (int e = 0; e < W; ++e) acc[i][e] = 0.0f;
}

template <int OUT, int W, bool WHOLE, bool NT>
__device__ __forceinline__ void embed_store(const EmbedGradParams& p, long v, int c, float (&acc)[W]) {
  const long at = v * p.ld_out + c;
#pragma unroll
  for (int e = 0; e < W; ++e) acc[e] *= p.scale;
  if constexpr (OUT == kEmbedAdd) {
    const auto old = embed_load<true, W, WHOLE>(p.out, at, p.d - c);
#pragma unroll
    for (int e = 0; e < W; ++e) acc[e] += old.at(e);
  }
  embed_write<OUT != kEmbedBF16, W, WHOLE, NT>(acc, p.out, at, p.d - c);
}

// A wave per piece of the sorted positions, then a wave per `group` rows of the table, whose
// positions lie one after the other: the rows of dy of all of them are requested as one run, so
// that a row with one token or none, the usual one, does not wait for its own chain of loads. NT:
// the output goes around the caches.
template <bool GF32, int OUT, bool WHOLE, bool NT>
static __global__ void __launch_bounds__(256) embed_grad_kernel(const EmbedGradParams p) {
  constexpr int W = OUT == kEmbedBF16 ? 8 : 4, NC = 32 / W, kSpan = 64 * W;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long task = blockIdx.x * 4L + wave;
  float acc[NC][W];
  if (task < p.pieces) {
    const int total = p.start[p.vocab], begin = (int)task * p.piece;
    if (begin >= total) return;
    const int end = (int)min((long)total, (long)begin + p.piece);
    const long first = p.tokens[p.perm[begin]], last = p.tokens[p.perm[end - 1]];
#pragma unroll 1
    for (int part = 0; part < 2; ++part) {
      if (part == 1 && last == first) break;
      const long v = part ? last : first;
      const int s = p.start[v], e = p.start[v + 1];
      if (e - s <= p.piece) continue;
      for (int c0 = 0; c0 < p.d; c0 += kSpan * NC) {
        const int c = c0 + W * lane;
        embed_clear(acc);
        embed_walk<GF32, NC, W, WHOLE>(p, part ? s : begin, part ? end : min(e, end), c, lane, acc, [](int) {});
#pragma unroll
        for (int i = 0; i < NC; ++i)
          if (c + kSpan * i < p.d)
            embed_write<true, W, true>(acc[i], p.partial, (2 * task + part) * p.ld_partial + c + kSpan * i, W);
      }
    }
    return;
  }
  const long v0 = (task - p.pieces) * p.group;
  if (v0 >= p.vocab) return;
  const int rows = (int)min((long)p.group, p.vocab - v0);
  // Lane r: where row r's positions begin (lane `rows`: where the last one's end).
  const int begins = p.start[v0 + min(lane, rows)];
  for (int c0 = 0; c0 < p.d; c0 += kSpan * NC) {
    const int c = c0 + W * lane;
    int r = 0;
    // Row r is complete: stored, unless its token is summed in pieces (or nothing is added to it).
    auto store = [&]() {
      const int n = __builtin_amdgcn_readlane(begins, r + 1) - __builtin_amdgcn_readlane(begins, r);
      if (n <= p.piece && (OUT != kEmbedAdd || n > 0)) {
#pragma unroll
        for (int i = 0; i < NC; ++i)
          if (c + kSpan * i < p.d) embed_store<OUT, W, WHOLE, NT>(p, v0 + r, c + kSpan * i, acc[i]);
      }
      embed_clear(acc);
      ++r;
    };
    embed_clear(acc);
    // Runs of rows between tokens that are summed in pieces.
    while (r < rows) {
      int to = r;
      while (to < rows && __builtin_amdgcn_readlane(begins, to + 1) - __builtin_amdgcn_readlane(begins, to) <= p.piece) ++to;
      embed_walk<GF32, NC, W, WHOLE>(p, __builtin_amdgcn_readlane(begins, r), __builtin_amdgcn_readlane(begins, to), c, lane, acc,
                                [&](int at) {
                                  while (at >= __builtin_amdgcn_readlane(begins, r + 1)) store();
                                });
      while (r < to || (r == to && r < rows)) store();  // the rest of the run, and the token after it
    }
  }
}

// At most 64 tokens need no sorting: every wave holds them all, one on a lane, and a row of the table
// takes the lanes with its token in their order.
constexpr int kFewTokens = 64;

template <bool GF32, int OUT, bool WHOLE>
static __global__ void __launch_bounds__(256) embed_few_kernel(const EmbedGradParams p) {
  constexpr int W = OUT == kEmbedBF16 ? 8 : 4, NC = 32 / W, kSpan = 64 * W;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long v0 = (blockIdx.x * 4L + wave) * p.group;
  if (v0 >= p.vocab) return;
  const int rows = (int)min((long)p.group, p.vocab - v0);
  const long token = lane < p.rows ? p.tokens[lane] : -1;
  for (int c0 = 0; c0 < p.d; c0 += kSpan * NC) {
    const int c = c0 + W * lane;
    for (int r = 0; r < rows; ++r) {
      unsigned long todo = __builtin_amdgcn_ballot_w64(token == v0 + r);
      if (OUT == kEmbedAdd && todo == 0) continue;
      float acc[NC][W];
      embed_clear(acc);
      while (todo != 0) {
        constexpr int kAhead = 2;
        EmbedPiece<GF32, W> v[kAhead][NC];
        int n = 0;
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
          // (Past the last one some row is read, and not added.)
          const long row = todo != 0 ? __builtin_ctzl(todo) : 0;
          if (todo != 0) ++n;
          todo &= todo - 1;
#pragma unroll
          for (int i = 0; i < NC; ++i)
            v[a][i] = embed_load<GF32, W, WHOLE>(p.dy, row * p.ld_dy + c + kSpan * i, p.d - c - kSpan * i);
        }
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
          if (a >= n) break;
#pragma unroll
          for (int i = 0; i < NC; ++i)
#pragma unroll
            for (int e = 0; e < W; ++e) acc[i][e] += v[a][i].at(e);
        }
      }
#pragma unroll
      for (int i = 0; i < NC; ++i)
        if (c + kSpan * i < p.d) embed_store<OUT, W, WHOLE, false>(p, v0 + r, c + kSpan * i, acc[i]);
    }
  }
}

// Adds the pieces of the token that begins in piece blockIdx.x and runs past it, in their order: a
// quarter of them on each wave, 64 W columns a workgroup.
template <int OUT, bool WHOLE>
static __global__ void __launch_bounds__(256) embed_join_kernel(const EmbedGradParams p) {
  const int total = p.start[p.vocab], q = blockIdx.x, begin = q * p.piece;
  if (begin >= total) return;
  const int end = (int)min((long)total, (long)begin + p.piece);
  const long v = p.tokens[p.perm[end - 1]];
  const int s = p.start[v], e = p.start[v + 1];
  if (e - s <= p.piece || s < begin) return;
  constexpr int W = OUT == kEmbedBF16 ? 8 : 4;
  __shared__ float sums[4][W][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = W * (blockIdx.y * 64 + lane);
  const int n = cdiv(e, p.piece) - q, share = cdiv(n, 4);  // pieces q .. q + n - 1
  float acc[W] = {};
  constexpr int kAhead = 8;
  const int to = min(n, (wave + 1) * share);
  for (int i = wave * share; i < to; i += kAhead) {
    EmbedPiece<true, W> x[kAhead];
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      const long row = 2L * (q + i + a) + (i + a == 0 && s > begin);
      x[a] = embed_load<true, W, true>(p.partial, row * p.ld_partial + c, i + a < to && c < p.d ? W : 0);
    }
#pragma unroll
    for (int a = 0; a < kAhead; ++a)
#pragma unroll
      for (int k = 0; k < W; ++k) acc[k] += x[a].at(k);
  }
#pragma unroll
  for (int k = 0; k < W; ++k) sums[wave][k][lane] = acc[k];
  __syncthreads();
  if (wave > 0 || c >= p.d) return;
#pragma unroll
  for (int k = 0; k < W; ++k) acc[k] = (sums[0][k][lane] + sums[1][k][lane]) + (sums[2][k][lane] + sums[3][k][lane]);
  embed_store<OUT, W, WHOLE, false>(p, v, c, acc);
}

}  // namespace ws
