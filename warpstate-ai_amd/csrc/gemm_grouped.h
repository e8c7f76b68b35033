// Products grouped by expert: rows sorted by expert, each expert's with a weight of its own.
//
//   rows t in [offsets[e], offsets[e + 1]):  C[t] = A[t] B_e          (forward, input gradient)
//   G_e = sum over those t of dY[t]^T X[t]                            (weight gradient)
//
// The offsets are on the device and the host knows only their number, so the grid is sized for
// the most tiles that any offsets make, and a workgroup finds its tile from them: every wave
// runs over the groups, one or more on a lane, with a running sum of their tiles, and takes the group
// whose tiles hold its index. Offsets are clamped to [0, rows]: whatever they hold, no access leaves the
// operands. Rows before the first offset and behind the last form two groups without a
// product, and get zeros.
//
// A group's tiles are those of a product of its own (gemm_fast.h, gemm_ring.h): the same loads, LDS
// layouts, k-loops and epilogues, with the group's first row and row count in the place of the
// matrix's. With few rows for each group the weights' bytes are the bound, and the kernel at
// the end streams them.
#pragma once

#include "gemm_ring.h"
#include "residual_norm.h"

namespace ws {

struct GroupedParams {
  OperandDesc a;                // rows of all groups
  OperandDesc b;                // group 0's weight as the product's B
  long b_group;                 // elements from one group's weight to the next
  const long* offsets;          // [groups + 1]
  int groups, rows, N, K, tiles_n;
  int b_rows;                   // columns of the product that the weight has; those up to N get zeros
  int chunk;                    // groups on each of 64 lanes
  int run;                      // tiles of a workgroup, one after the other (not 256 x 256)
  int most;                     // tiles that the grid is sized for
  int pieces_most;              // a last round of at most so many 256 x 256 tiles goes in pieces
  unsigned short* c; long ldc;
  int per;                      // k-tiles of a slice of the reduction (grouped_ring_kernel<SLICED>)
  float* partial;               // [slices, rows, N]
};

struct GroupTile {
  int group;     // -1: rows of no group
  int lo, hi;    // its rows
  int index;     // the tile within the group
};

__device__ __forceinline__ int group_offset(const GroupedParams& p, int g) {
  return (int)min((long)p.rows, max(0L, p.offsets[min(g, p.groups)]));
}

// A lane's groups, `chunk` from lane * chunk on: their tiles of BM rows (the grid's `most` at most), and
// the running sum over the lanes. lo, hi: the rows where chunk is 1 (up to 64 groups).
struct GroupLanes {
  int lo, hi, tiles, upto;
};
__device__ __forceinline__ int lanes_upto(int tiles, int lane) {
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int other = __shfl_up(tiles, off, kWave);
    if (lane >= off) tiles += other;
  }
  return tiles;
}
template <int BM>
__device__ __forceinline__ int row_tiles(const GroupedParams& p, int lo, int hi) {
  return hi > lo ? cdiv(hi - lo, BM) * p.tiles_n : 0;
}
template <int BM>
__device__ __forceinline__ GroupLanes group_lanes(const GroupedParams& p, int lane) {
  GroupLanes v;
  v.lo = group_offset(p, lane * p.chunk);  // past the last group: its end, twice
  v.hi = v.tiles = 0;
  if (p.chunk == 1) {
    v.hi = group_offset(p, lane + 1);
    v.tiles = row_tiles<BM>(p, v.lo, v.hi);
  } else {
    constexpr int kAhead = 8;
    int lo = v.lo;
    for (int b = 0; b < p.chunk; b += kAhead) {
      int hi[kAhead];
#pragma unroll
      for (int a = 0; a < kAhead; ++a) hi[a] = group_offset(p, lane * p.chunk + b + a + 1);
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        if (b + a < p.chunk) v.tiles = min(p.most, v.tiles + row_tiles<BM>(p, lo, hi[a]));
        lo = hi[a];
      }
    }
  }
  v.upto = lanes_upto(v.tiles, lane);
  return v;
}

// The tiles that there are, `most` at most (what offsets that do not decrease make): the groups', those of the
// rows before the first offset and of those behind the last.
template <int BM>
__device__ __forceinline__ int count_tiles(const GroupedParams& p, int lane, GroupLanes& v) {
  v = group_lanes<BM>(p, lane);
  return min(p.most, __builtin_amdgcn_readlane(v.upto, 63) + row_tiles<BM>(p, 0, group_offset(p, 0)) +
                         row_tiles<BM>(p, group_offset(p, p.groups), p.rows));
}

// The tile at index w, below count_tiles' total.
template <int BM>
__device__ __forceinline__ GroupTile find_tile(const GroupedParams& p, int w, int lane, GroupLanes v) {
  const int grouped = __builtin_amdgcn_readlane(v.upto, 63);
  if (w >= grouped) {
    w -= grouped;
    const int first = group_offset(p, 0), before = row_tiles<BM>(p, 0, first);
    return w < before ? GroupTile{-1, 0, first, w} : GroupTile{-1, group_offset(p, p.groups), p.rows, w - before};
  }
  int l = __builtin_ctzl(__builtin_amdgcn_ballot_w64(w < v.upto)), base = 0;
  if (p.chunk > 1) {  // the same over the groups of that lane, 64 at a time
    w -= __builtin_amdgcn_readlane(v.upto - v.tiles, l);
    base = l * p.chunk;
    for (const int end = base + p.chunk;; base += 64) {
      v.lo = group_offset(p, base + lane);
      v.hi = group_offset(p, base + lane + 1);
      v.tiles = base + lane < end ? row_tiles<BM>(p, v.lo, v.hi) : 0;
      v.upto = lanes_upto(v.tiles, lane);
      const unsigned long past = __builtin_amdgcn_ballot_w64(w < v.upto);
      l = past != 0 ? __builtin_ctzl(past) : 0;
      if (past != 0 || base + 64 >= end) break;
      w -= __builtin_amdgcn_readlane(v.upto, 63);
    }
  }
  return GroupTile{base + l, __builtin_amdgcn_readlane(v.lo, l), __builtin_amdgcn_readlane(v.hi, l),
                   w - __builtin_amdgcn_readlane(v.upto - v.tiles, l)};
}
// The tile after t, at index w: in its group, or the first of one of the next four, or searched for.
template <int BM>
__device__ __forceinline__ GroupTile next_tile(const GroupedParams& p, GroupTile t, int w, int lane) {
  if (++t.index < row_tiles<BM>(p, t.lo, t.hi)) return t;
  if (t.group >= 0) {
    const int last = min(t.group + 4, p.groups - 1);
    for (int g = t.group + 1; g <= last; ++g) {
      const int lo = group_offset(p, g), hi = group_offset(p, g + 1);
      if (hi > lo) return GroupTile{g, lo, hi, 0};
    }
  }
  return find_tile<BM>(p, w, lane, group_lanes<BM>(p, lane));
}

// What the epilogues read of a GEMM's parameters.
__device__ __forceinline__ GemmParams store_params(unsigned short* c, long ldc, int M, int N) {
  GemmParams e{};
  e.c = c;
  e.ldc = ldc;
  e.M = M;
  e.N = N;
  return e;
}

// A piece of the last round's tiles: BM x BN of tile whole + x / pieces, the (x % pieces)-th by rows. Its
// sums have the 256 x 256 tile's order, so the bits do not tell which of the two made them.
template <class Cfg, int BMODE>
__device__ __forceinline__ void grouped_piece(const GroupedParams& p, int whole, int x, unsigned char* smem, int lane,
                                              int wave) {
  constexpr int kAcross = kFBN / Cfg::BN, kPieces = kFBM / Cfg::BM * kAcross;
  const GroupTile t = find_tile<kFBM>(p, whole + x / kPieces, lane, group_lanes<kFBM>(p, lane));
  int tm, tn;
  tile_position(t.index, cdiv(t.hi - t.lo, kFBM), p.tiles_n, tm, tn);
  const int piece = x % kPieces;
  const int row0 = t.lo + tm * kFBM + piece / kAcross * Cfg::BM, col0 = tn * kFBN + piece % kAcross * Cfg::BN;
  if (row0 >= t.hi || col0 >= p.N) return;
  const int wm = wave / Cfg::WN, wn = wave % Cfg::WN;
  OperandDesc b = p.b;
  b.ptr += max(t.group, 0) * p.b_group;
  Acc16<Cfg::FA, Cfg::FB> acc;
  ring_k_loop<Cfg, kKContig, BMODE, false>(acc, p.a, row0, t.hi, b, col0, p.b_rows, 0, p.K, 0,
                                           t.group < 0 ? 0 : cdiv(p.K, kFBK), smem, wave, lane);
  const GemmParams e = store_params(p.c, p.ldc, t.hi, p.N);
  FEpiStore<false, false>::run(e, acc, row0 + wm * Cfg::TM, col0 + wn * Cfg::TN, lane, tm, tn, wn,
                               smem + wave * epi_wave<Cfg::FA, Cfg::FB>());
  __builtin_amdgcn_s_barrier();  // the next piece's loads go where the staging was
}

// 256 x 256 tiles, a workgroup per compute unit looping over them. A last round that would leave most
// units idle goes in pieces of 64 x 128 or 128 x 128 instead, so that all of them take part (us of R
// tiles on 256 units, whole / in pieces: reduction 512, R 32 14.7 / 8.2, R 64 14.6 / 9.8; 2048, R 32
// 36 / 17, R 64 36 / 22, R 96 36 / 39; 8192, R 32 121 / 52, R 64 121 / 74).
typedef RingCfg<64, 128, 2, 4, 4> Piece64;
typedef RingCfg<128, 128, 4, 2, 4> Piece128;

template <int BMODE>
__global__ void __launch_bounds__(kFNT) grouped_fast_kernel(const GroupedParams p) {
  constexpr int TM = kFBM / kFWM, TN = kFBN / kFWN;
  extern __shared__ __attribute__((aligned(1024))) unsigned char fsmem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / kFWN, wn = wave % kFWN;
  const unsigned lds0 = (unsigned)(unsigned long)(__attribute__((address_space(3))) unsigned char*)fsmem;
  const unsigned abase = lds0 + frag_base<kKContig>(wm * TM, lane);
  const unsigned bbase = lds0 + 2 * kFTileBytes + frag_base<BMODE>(wn * TN, lane);
  GroupLanes v;
  const int total = count_tiles<kFBM>(p, lane, v), rest = total % (int)gridDim.x;
  const int whole = rest <= p.pieces_most ? total - rest : total;
  for (int w = blockIdx.x; w < whole; w += gridDim.x) {
    // The groups are read again for each tile: kept over the k-loop they would cost it registers.
    int l = lane;
    opaque_lane(l);
    const GroupTile t = find_tile<kFBM>(p, xcd_remap(w, whole, gridDim.x), l, group_lanes<kFBM>(p, l));
    int tm, tn;
    tile_position(t.index, cdiv(t.hi - t.lo, kFBM), p.tiles_n, tm, tn);
    const int row0 = t.lo + tm * kFBM, col0 = tn * kFBN;
    OperandDesc b = p.b;
    b.ptr += max(t.group, 0) * p.b_group;
    Acc16<4, 8> acc;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) acc.v[i][j] = f32x4_v{0.f, 0.f, 0.f, 0.f};
    fast_k_loop<kKContig, BMODE, false>(acc, p.a, row0, t.hi, b, col0, p.b_rows, 0, p.K, 0,
                                        t.group < 0 ? 0 : cdiv(p.K, kFBK), fsmem, fsmem + 2 * kFTileBytes, abase,
                                        bbase, wave, lane);
    const GemmParams e = store_params(p.c, p.ldc, t.hi, p.N);
    FEpiStore<false, false>::run(e, acc, row0 + wm * TM, col0 + wn * TN, lane, tm, tn, wn, fsmem + wave * kFStageWave);
    __builtin_amdgcn_s_barrier();
  }
  if (whole == total) return;
  int l = lane;
  opaque_lane(l);
  if (rest * 8 <= (int)gridDim.x) {
    for (int x = blockIdx.x; x < rest * 8; x += gridDim.x)
      grouped_piece<Piece64, BMODE>(p, whole, xcd_remap(x, rest * 8, gridDim.x), fsmem, l, wave);
  } else {
    for (int x = blockIdx.x; x < rest * 4; x += gridDim.x)
      grouped_piece<Piece128, BMODE>(p, whole, xcd_remap(x, rest * 4, gridDim.x), fsmem, l, wave);
  }
}

// The wave's accumulators as FP32 rows of out [M, N], through its LDS staging rows in two halves, so
// that the stores cover whole lines; NT: they go around the caches. (Stored from the fragments, 64 bytes of
// each of 16 rows at a time, and through them, a step of eight experts' 11264 x 2048 masters over
// 16384 rows took 2000 us instead of 1960.)
template <bool NT, int FA, int FB>
__device__ __forceinline__ void store_f32(float* out, int M, int N, Acc16<FA, FB>& acc, int m_base, int n_base, int lane,
                                          unsigned char* stage) {
  constexpr int kRow = FB * 64 + 16, LPR = FB * 4, RPI = 64 / LPR, HA = FA / 2, NQ = HA * 16 / RPI;
  static_assert(FA % 2 == 0 && 64 % LPR == 0 && NQ >= 1 && HA * 16 * kRow <= epi_wave<FA, FB>(), "half a tile is staged");
  opaque_lane(lane);
  __amdgpu_buffer_rsrc_t rg = make_rsrc(out + (long)m_base * N + n_base, 0x7fffffff);
  const int c4 = 4 * (lane % LPR);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int i = 0; i < HA; ++i)
#pragma unroll
      for (int j = 0; j < FB; ++j)
        *reinterpret_cast<f32x4_v*>(stage + (16 * i + (lane & 15)) * kRow + (16 * j + 4 * (lane >> 4)) * 4) =
            acc.v[h * HA + i][j];
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): this wave's staging writes landed
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      const int r = RPI * q + lane / LPR, m = 16 * HA * h + r;
      const bool ok = m_base + m < M && n_base + c4 + 3 < N;  // N is a multiple of 8
      const u32x4_t v = *reinterpret_cast<const u32x4_t*>(stage + r * kRow + c4 * 4);
      __builtin_amdgcn_raw_buffer_store_b128(v, rg, store_off(ok, (long)m * N + c4, 4), 0, NT ? kEpiNT : 0);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}
// Smaller tiles, one workgroup each. SLICED: slice blockIdx.y of the reduction, in FP32, for
// grouped_join_kernel.
template <class Cfg, int BMODE, bool SLICED>
__global__ void __launch_bounds__(Cfg::NT) grouped_ring_kernel(const GroupedParams p) {
  constexpr int FA = Cfg::FA, FB = Cfg::FB, TM = Cfg::TM, TN = Cfg::TN;
  extern __shared__ __attribute__((aligned(1024))) unsigned char rsmem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / Cfg::WN, wn = wave % Cfg::WN;
  GroupLanes v;
  const int total = count_tiles<Cfg::BM>(p, lane, v), blocks = cdiv(total, p.run);
  if ((int)blockIdx.x >= blocks) return;
  int w = xcd_remap(blockIdx.x, blocks, kRingWindow) * p.run;
  const int end = min(total, w + p.run);
  GroupTile t = find_tile<Cfg::BM>(p, w, lane, v);
  while (true) {
    int tm, tn;
    tile_position(t.index, cdiv(t.hi - t.lo, Cfg::BM), p.tiles_n, tm, tn);
    const int row0 = t.lo + tm * Cfg::BM, col0 = tn * Cfg::BN;
    OperandDesc b = p.b;
    b.ptr += max(t.group, 0) * p.b_group;
    const int tiles = t.group < 0 ? 0 : cdiv(p.K, kFBK), kb = SLICED ? blockIdx.y * p.per : 0;
    Acc16<FA, FB> acc;
    ring_k_loop<Cfg, kKContig, BMODE, false>(acc, p.a, row0, t.hi, b, col0, p.b_rows, 0, p.K, kb,
                                             SLICED ? min(tiles, kb + p.per) : tiles, rsmem, wave, lane);
    if constexpr (SLICED) {
      store_f32<false>(p.partial + (long)blockIdx.y * p.rows * p.N, t.hi, p.N, acc, row0 + wm * TM, col0 + wn * TN, lane,
                       rsmem + wave * epi_wave<FA, FB>());
    } else {
      const GemmParams e = store_params(p.c, p.ldc, t.hi, p.N);
      FEpiStore<false, false>::run(e, acc, row0 + wm * TM, col0 + wn * TN, lane, tm, tn, wn,
                                   rsmem + wave * epi_wave<FA, FB>());
    }
    if (SLICED || ++w >= end) return;
    __builtin_amdgcn_s_barrier();  // the next tile's loads go where the staging was
    t = next_tile<Cfg::BM>(p, t, w, lane);
  }
}

// The slices' sums in their order, eight columns a thread.
static __global__ void __launch_bounds__(256) grouped_join_kernel(const float* partial, int slices, long rows, int N,
                                                                  unsigned short* c, long ldc) {
  const long at = (blockIdx.x * 256L + threadIdx.x) * 8, size = rows * N;
  if (at >= size) return;
  float sum[8] = {};
#pragma unroll 4
  for (int i = 0; i < slices; ++i) {
    const f32x4_v* src = reinterpret_cast<const f32x4_v*>(partial + i * size + at);
    const f32x4_v a = src[0], b = src[1];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      sum[e] += a[e];
      sum[4 + e] += b[e];
    }
  }
  const long row = at / N;
  *reinterpret_cast<u32x4_t*>(c + row * ldc + (at - row * N)) =
      u32x4_t{pack_bf16x2(sum[0], sum[1]), pack_bf16x2(sum[2], sum[3]), pack_bf16x2(sum[4], sum[5]), pack_bf16x2(sum[6], sum[7])};
}

// --------------------------------------------------------------------------------------
// Weight gradients: [M, N] per group, reduced over the group's rows.

struct GroupedGradParams {
  const unsigned short *a, *b;  // [rows, M] and [rows, N]
  long lda, ldb;
  const long* offsets;
  int groups, rows, M, N, tiles_m, tiles_n;
  void* g;                      // [groups, M, N], BF16 or FP32
};

__device__ __forceinline__ void grad_rows(const GroupedGradParams& p, int g, int& lo, int& hi) {
  auto at = [&](int i) { return (int)min((long)p.rows, max(0L, p.offsets[i])); };
  lo = at(g);
  hi = at(g + 1);
}
struct GradTile {
  OperandDesc a, b;
  int group, K, tm, tn;
};
// Groups in the order in which their tiles are dealt out, lane r the group with the r-th most rows:
// the tiles of one group take as long as it has rows, and long ones that come last leave the others
// waiting. (16384 rows in eight groups, gradients of 2048 x 2048 in BF16: 168 -> 134 us.) More than
// kOrdered groups keep their own order: finding another takes a small tile's workgroup too long.
constexpr int kOrdered = 16;
__device__ __forceinline__ int grad_order(const GroupedGradParams& p, int lane) {
  if (p.groups > kOrdered) return lane;
  int lo = 0, hi = 0;
  if (lane < p.groups) grad_rows(p, lane, lo, hi);
  const int rows = max(0, hi - lo);
  int rank = lane < p.groups ? 0 : lane;
  for (int j = 0; j < p.groups; ++j) {
    const int other = __builtin_amdgcn_readlane(rows, j);
    if (lane < p.groups) rank += other > rows || (other == rows && j < lane);
  }
  return __builtin_amdgcn_ds_permute(4 * rank, lane);
}
__device__ __forceinline__ GradTile grad_tile(const GroupedGradParams& p, int w, int order) {
  const int per = p.tiles_m * p.tiles_n, place = w / per;
  GradTile t;
  t.group = p.groups > kOrdered ? place : __builtin_amdgcn_readlane(order, place);
  tile_position(w - place * per, p.tiles_m, p.tiles_n, t.tm, t.tn);
  int lo, hi;
  grad_rows(p, t.group, lo, hi);
  t.K = max(0, hi - lo);
  t.a = OperandDesc{p.a + lo * p.lda, 1, p.lda};
  t.b = OperandDesc{p.b + lo * p.ldb, 1, p.ldb};
  return t;
}
template <bool F32, int FA, int FB>
__device__ __forceinline__ void grad_store(const GroupedGradParams& p, const GradTile& t, Acc16<FA, FB>& acc, int m_base,
                                           int n_base, int lane, int wn, unsigned char* stage) {
  const long at = (long)t.group * p.M * p.N;
  if constexpr (F32) {
    store_f32<true>(static_cast<float*>(p.g) + at, p.M, p.N, acc, m_base, n_base, lane, stage);
  } else {
    const GemmParams e = store_params(static_cast<unsigned short*>(p.g) + at, p.N, p.M, p.N);
    FEpiStore<false, false>::run(e, acc, m_base, n_base, lane, t.tm, t.tn, wn, stage);
  }
}

template <bool F32>
__global__ void __launch_bounds__(kFNT) grouped_grad_fast_kernel(const GroupedGradParams p) {
  constexpr int TM = kFBM / kFWM, TN = kFBN / kFWN;
  extern __shared__ __attribute__((aligned(1024))) unsigned char fsmem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / kFWN, wn = wave % kFWN;
  const unsigned lds0 = (unsigned)(unsigned long)(__attribute__((address_space(3))) unsigned char*)fsmem;
  const unsigned abase = lds0 + frag_base<kMNContig>(wm * TM, lane);
  const unsigned bbase = lds0 + 2 * kFTileBytes + frag_base<kMNContig>(wn * TN, lane);
  const int total = p.groups * p.tiles_m * p.tiles_n, order = grad_order(p, lane);
  for (int w = blockIdx.x; w < total; w += gridDim.x) {
    // Every other round runs backwards, so that a unit with a long tile in one has a short one in the next.
    const int round = w / (int)gridDim.x, base = round * gridDim.x, x = xcd_remap(w, total, gridDim.x);
    const GradTile t = grad_tile(p, round & 1 ? 2 * base + min((int)gridDim.x, total - base) - 1 - x : x, order);
    Acc16<4, 8> acc;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) acc.v[i][j] = f32x4_v{0.f, 0.f, 0.f, 0.f};
    fast_k_loop<kMNContig, kMNContig, false>(acc, t.a, t.tm * kFBM, p.M, t.b, t.tn * kFBN, p.N, 0, t.K, 0,
                                             cdiv(t.K, kFBK), fsmem, fsmem + 2 * kFTileBytes, abase, bbase, wave, lane);
    grad_store<F32>(p, t, acc, t.tm * kFBM + wm * TM, t.tn * kFBN + wn * TN, lane, wn, fsmem + wave * kFStageWave);
    __builtin_amdgcn_s_barrier();
  }
}

template <class Cfg, bool F32>
__global__ void __launch_bounds__(Cfg::NT) grouped_grad_ring_kernel(const GroupedGradParams p) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char rsmem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / Cfg::WN, wn = wave % Cfg::WN;
  const GradTile t = grad_tile(p, xcd_remap(blockIdx.x, gridDim.x, kRingWindow), grad_order(p, lane));
  Acc16<Cfg::FA, Cfg::FB> acc;
  ring_k_loop<Cfg, kMNContig, kMNContig, false>(acc, t.a, t.tm * Cfg::BM, p.M, t.b, t.tn * Cfg::BN, p.N, 0, t.K, 0,
                                                cdiv(t.K, kFBK), rsmem, wave, lane);
  grad_store<F32>(p, t, acc, t.tm * Cfg::BM + wm * Cfg::TM, t.tn * Cfg::BN + wn * Cfg::TN, lane, wn,
                  rsmem + wave * epi_wave<Cfg::FA, Cfg::FB>());
}

// --------------------------------------------------------------------------------------
// Few rows for each group: tiles of 16 rows x COLS columns, one workgroup of four waves, each
// with a quarter of the reduction (64 of every 256 k, so that together they read whole rows of the
// weight). Fragments go from memory to registers as they are: a lane's piece is 16 bytes of one row,
// and a k-tile's two pieces of a row are one line. The waves' sums are added through LDS, in
// wave order. Rows past the group's read its last one and are not stored; columns past the weight's
// read its last one, and what they get, up to N, is no part of the result. Operands have any alignment and
// any K: the pieces need none.
//
// The weights' bytes are the bound. Neighbouring tiles run on one XCD, so that what it reads at a time is one
// run of the weight, and two k-tiles are in flight: with four, the registers leave fewer workgroups
// (32 rows in 8 groups of 5632 x 2048, launch order and four / these 40 / 34 us, 40 rows in 8 of 2048 x 8192 61 / 50).
constexpr int kFewRows = 16;
typedef bf16x8_t bf16x8_any __attribute__((aligned(2)));

// RUN: p.run tiles of a workgroup, for which the registers leave fewer of them.
template <int COLS, bool RUN>
static __global__ void __launch_bounds__(256) grouped_few_kernel(const GroupedParams p) {
  constexpr int BM = kFewRows, NJ = COLS / 16;
  __shared__ float sums[4][BM][COLS + 4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  GroupLanes v;
  const int total = count_tiles<BM>(p, lane, v), run = RUN ? p.run : 1, blocks = cdiv(total, run);
  if ((int)blockIdx.x >= blocks) return;
  int w = xcd_remap(blockIdx.x, blocks, kRingWindow) * run;
  const int end = min(total, w + run);
  GroupTile t = find_tile<BM>(p, w, lane, v);
  while (true) {
    const int tm = t.index / p.tiles_n, tn = t.index - tm * p.tiles_n;
    const int row0 = t.lo + tm * BM, col0 = tn * COLS;
    f32x4_v acc[NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[j] = f32x4_v{0.f, 0.f, 0.f, 0.f};
    if (t.group >= 0) {
      const int r = lane & 15, q = 8 * (lane >> 4);
      const unsigned short* const a = p.a.ptr + (long)min(row0 + r, t.hi - 1) * p.a.s_row + q;
      const unsigned short* b[NJ];
#pragma unroll
      for (int j = 0; j < NJ; ++j)
        b[j] = p.b.ptr + t.group * p.b_group + (long)min(col0 + 16 * j + r, p.b_rows - 1) * p.b.s_row + q;
      // U k-tiles at a time, all of their pieces requested before the first product.
      auto steps = [&](int k, auto count, auto load) {
        constexpr int U = decltype(count)::value;
        bf16x8_t fa[U][2], fb[U][2][NJ];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            const int at = k + 256 * u + 32 * s;
#pragma unroll
            for (int j = 0; j < NJ; ++j) fb[u][s][j] = load(b[j], at);
            fa[u][s] = load(a, at);
          }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int j = 0; j < NJ; ++j)
              acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[u][s][j], fa[u][s], acc[j], 0, 0, 0);
      };
      const auto whole = [](const unsigned short* row, int at) -> bf16x8_t { return *reinterpret_cast<const bf16x8_any*>(row + at); };
      constexpr int U = 2;
      int k = 64 * wave;
      for (; k + 256 * (U - 1) + 64 <= p.K; k += 256 * U) steps(k, std::integral_constant<int, U>{}, whole);
      for (; k + 64 <= p.K; k += 256) steps(k, std::integral_constant<int, 1>{}, whole);
      if (k < p.K)
        steps(k, std::integral_constant<int, 1>{}, [&](const unsigned short* row, int at) {
          const int left = p.K - at - q;
          if (left >= 8) return whole(row, at);
          u32x4_t v = {0, 0, 0, 0};
#pragma unroll
          for (int e = 0; e < 7; ++e)
            if (e < left) v[e >> 1] |= (unsigned)row[at + e] << (16 * (e & 1));
          return __builtin_bit_cast(bf16x8_t, v);
        });
    }
#pragma unroll
    for (int j = 0; j < NJ; ++j)
      *reinterpret_cast<f32x4_v*>(&sums[wave][lane & 15][16 * j + 4 * (lane >> 4)]) = acc[j];
    __syncthreads();
    const int m = threadIdx.x / (COLS / 2), n = 2 * (threadIdx.x % (COLS / 2));
    if (m < BM) {
      float v2[2];
#pragma unroll
      for (int e = 0; e < 2; ++e)
        v2[e] = (sums[0][m][n + e] + sums[1][m][n + e]) + (sums[2][m][n + e] + sums[3][m][n + e]);
      if (row0 + m < t.hi && col0 + n < p.N)  // N is a multiple of 8
        *reinterpret_cast<unsigned*>(p.c + (long)(row0 + m) * p.ldc + col0 + n) = pack_bf16x2(v2[0], v2[1]);
    }
    if (!RUN || ++w >= end) return;
    __syncthreads();  // the sums have been read
    t = next_tile<BM>(p, t, w, lane);
  }
}

// --------------------------------------------------------------------------------------
// Matrices of any width as the products read them, and back: rows [rows_in, cols_in] of each group into
// rows [rows_out, cols_out], what lies past the input written as zeros and what lies past the output
// left out. Element (g, r, c) at g * group + r * ld + c on either side.
struct CopyRowsParams {
  const void* in; long group_in, ld_in; int rows_in, cols_in;
  void* out; long group_out, ld_out; int rows_out, cols_out;
  long rows;  // of all groups' output
};

template <bool IN32, bool OUT32>
static __global__ void __launch_bounds__(256) copy_rows_kernel(const CopyRowsParams p) {
  const int lane = threadIdx.x & 63;
  for (long row = blockIdx.x * 4L + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); row < p.rows; row += gridDim.x * 4L) {
    const long g = row / p.rows_out;
    const int r = (int)(row - g * p.rows_out), cols = r < p.rows_in ? p.cols_in : 0;
#pragma unroll 4
    for (int c = 8 * lane; c < p.cols_out; c += 512) {
      QuantRow<IN32> v;
      load_piece<IN32, false>(v, p.in, g * p.group_in + r * p.ld_in + c, cols - c);
      float f[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = v.at(e);
      store_piece<OUT32, false>(round_piece<OUT32>(f), p.out, g * p.group_out + r * p.ld_out + c, p.cols_out - c);
    }
  }
}

}  // namespace ws
