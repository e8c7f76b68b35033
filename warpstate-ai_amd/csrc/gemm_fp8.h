// Product of two e4m3 matrices with a scale per block of 128 along the reduction:
//   C[m, n] = sum_b sA[m, b] sB[n, b] sum_{k in block b} A[m, k] B[n, k],
// A [M, K] and B [N, K] (nn.Linear layout) with contiguous rows, C in BF16. Sums are FP32
// between the instruction's groups of eight products; within a group each product is cut at
// 2^-13 of the largest one's power of two (measured: beside a product of 1, one of 2^-13 is
// kept and one of 2^-14 lost; between groups, 2^-23 is kept). That costs about 1e-4 of a
// result's size, against 2e-3 of its BF16 rounding, and is why FP32 results are not offered:
// products of BF16 operands, with twice the matrix-pipe time, give those.
//
// A 128-byte row piece of e4m3 is one scale block and also exactly what 64 BF16 values take,
// so a k-tile is one block and the operand tiles, their direct-to-LDS loads, their swizzle
// and the accumulator layout are those of the BF16 kernels (gemm_fast.h, gemm_ring.h), with
// K counted in pairs of bytes by the loaders. Where those run two v_mfma_f32_16x16x32_bf16
// on a pair of 16-byte chunks, one v_mfma_f32_16x16x128_f8f6f4 takes both chunks: the same
// matrix-pipe time per k-tile for twice the products. The chunks (l >> 4) and 4 + (l >> 4) of
// a row go to lane l: the k order is another than the instruction's own, but the same for
// both operands, and a block has one scale.
//
// Rates (the 256 x 256 tile, e8m0 / FP32 scales, B in blocks, one product in a loop): 8192 x 10240 x
// 2048 141 / 171 us (2.4 / 2.0 PFLOP/s), 16384 x 2048 x 11264 241 / 309 us (3.1 / 2.4; 2.6 to 2.8 under
// e8m0 in the clock that a training step's other products leave), where BF16 products reach
// 1.4 to 1.5 and the instruction alone, in a loop on registers, 4.6. Between the two stand the
// chain of a k-tile (fragment reads behind a barrier, then the MFMAs), the epilogue (about 4 us
// a tile, a fifth of one with 16 k-tiles) and the clock under load.
//
// Scales. e8m0: the instruction's own block scales (v_mfma_scale), no arithmetic beside it. A
// lane gives the scale byte of its operand row; a dword holds the four bytes of four k-tiles, and is
// shifted by one byte per k-tile. FP32: the block's product starts from zero, and
// acc = fma(product, sA * sB, acc), four FP32 operations per MFMA beside it; sA * sB has to be in
// FP32's range.
#pragma once

#include "gemm_ring.h"
#include "quant.h"

namespace ws {

typedef int i32x8_t __attribute__((ext_vector_type(8)));

// Scales of an operand: (r, b) as an e8m0 byte at r * ld + b (ld a multiple of 4, base 4-byte
// aligned, rows readable to the next multiple of 4) or as FP32 at b * ld + r (for B with a
// scale per row, base 16-byte aligned and ld a multiple of 4); one row of scales per
// 2^shift operand rows.
struct Fp8Scale {
  const void* ptr;
  long ld;
  int shift;
};
// Tiles of the raster from `whole` on are split along K into `splits` slices of slice_kt
// k-tiles (a multiple of 4: a dword of e8m0 scales), whose FP32 sums go to blocks of
// BM x BN floats (tile, slice) of `partials`; fp8_join_kernel adds them.
struct Fp8Params {
  Fp8Scale a, b;
  int whole, splits, slice_kt;
  float* partials;
};

__device__ __forceinline__ i32x8_t join_frag(bf16x8_t lo, bf16x8_t hi) {
  const u32x4_t a = __builtin_bit_cast(u32x4_t, lo), b = __builtin_bit_cast(u32x4_t, hi);
  return i32x8_t{(int)a[0], (int)a[1], (int)a[2], (int)a[3], (int)b[0], (int)b[1], (int)b[2], (int)b[3]};
}

// (Functions of their own: with template-dependent arguments the builtin's target check fails
// on the compiler's host pass.)
__device__ __forceinline__ f32x4_v mfma_e4m3_scaled(i32x8_t b, i32x8_t a, f32x4_v c, unsigned sb,
                                                    unsigned sa) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b, a, c, 0, 0, 0, (int)sb, 0, (int)sa);
}
__device__ __forceinline__ f32x4_v mfma_e4m3(i32x8_t b, i32x8_t a, f32x4_v c) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b, a, c, 0, 0, 0, 0, 0, 0);
}

__device__ __forceinline__ unsigned load_u32(__amdgpu_buffer_rsrc_t rs, unsigned off, unsigned soff) {
  return __builtin_amdgcn_raw_buffer_load_b32(rs, off, soff, 0);
}

// The scales of one wave's FA x FB blocks for one k-tile at a time: load() requests them and
// ready() makes them usable once they are there. BROW: B has a scale per row; otherwise the
// wave's columns lie in one block of 128.
//
// e8m0: a lane requests the dword of one row, so that one load covers 64 rows and four k-tiles,
// and ready() hands lane l the words of rows 16 i + (l & 15) through the LDS crossbar. (With a load
// per block, 4 lanes asking for each of its 16 rows, the 12 loads every four k-tiles cost a
// 11264 x 2048 x 16384 product a fifth of its time: 411 us against 324 with B in blocks.) FP32: a
// load per block, every k-tile; through the crossbar 512 x 4096 x 4096 took 20.0 us against 18.6.
//
// OWN (the next request follows at once): every word goes to a register of its own. Sharing the
// request's, the next request would go to another, and be waited for and copied within the same
// k-tile, with the operand loads ahead of it (e8m0, B in blocks, 16 x 11264 x 2048: 64 x 128 tiles
// 16.1 -> 12.4 us, 64 x 64 10.8 -> 9.8).
template <int SCALE, bool BROW, int FA, int FB>
struct WaveScales {
  static constexpr bool kE8 = SCALE == kScaleE8M0;
  static constexpr int NB = BROW ? FB : 1;
  static constexpr int kWords = kE8 || !BROW ? 1 : 4;  // per B block: a lane's four columns under FP32
  static constexpr int LA = kE8 ? (16 * FA + 63) / 64 : FA;
  static constexpr int LB = kE8 && BROW ? (16 * FB + 63) / 64 : NB;
  const char *base_a, *base_b;
  long step_a, step_b;  // bytes per k-tile
  unsigned off_a[LA], off_b[LB];
  unsigned a[FA], b[NB][kWords];
  unsigned raw_a[LA], raw_b[LB][kWords];

  // m_base, n_base: first row and column of the wave's tile.
  __device__ __forceinline__ void init(const Fp8Params& p, int m_base, int n_base, int M, int N,
                                       int lane) {
    // A wave past the last row or column reads the last one's scales (four columns' at a time
    // for a scale per row under FP32); nothing of it is stored.
    const long ra = min(m_base, M - 1) >> p.a.shift;
    const long rb = min(n_base, kWords == 4 ? (N - 1) & ~3 : N - 1) >> p.b.shift;
    const long row_a = kE8 ? p.a.ld : 4, row_b = kE8 ? p.b.ld : 4;  // bytes per row
    base_a = static_cast<const char*>(p.a.ptr) + ra * row_a;
    base_b = static_cast<const char*>(p.b.ptr) + rb * row_b;
    step_a = kE8 ? 1 : 4 * p.a.ld;
    step_b = kE8 ? 1 : 4 * p.b.ld;
#pragma unroll
    for (int i = 0; i < LA; ++i) {
      const int row = m_base + (kE8 ? 64 * i + lane % (FA < 4 ? 16 * FA : 64) : 16 * i + (lane & 15));
      off_a[i] = (unsigned)(((min(row, M - 1) >> p.a.shift) - ra) * row_a);
    }
#pragma unroll
    for (int j = 0; j < LB; ++j) {
      if constexpr (!BROW) off_b[j] = 0;
      else if constexpr (kE8) off_b[j] = (unsigned)((min(n_base + 64 * j + lane % (FB < 4 ? 16 * FB : 64), N - 1) - rb) * p.b.ld);
      else off_b[j] = (unsigned)(4 * (min(n_base + 16 * j + 4 * (lane >> 4), (N - 1) & ~3) - rb));
    }
  }
  // Requests the scales of k-tile kt (e8m0: of kt .. kt + 3, kt a multiple of 4).
  __device__ __forceinline__ void load(int kt) {
    __amdgpu_buffer_rsrc_t ra = make_rsrc(base_a + kt * step_a, 0x7fffffff);
    __amdgpu_buffer_rsrc_t rb = make_rsrc(base_b + kt * step_b, 0x7fffffff);
#pragma unroll
    for (int i = 0; i < LA; ++i) raw_a[i] = load_u32(ra, off_a[i], 0);
#pragma unroll
    for (int j = 0; j < LB; ++j) {
      if constexpr (kWords == 1) {
        raw_b[j][0] = load_u32(rb, off_b[j], 0);
      } else {
        const u32x4_t v = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(rb, off_b[j], 0, 0));
#pragma unroll
        for (int e = 0; e < 4; ++e) raw_b[j][e] = v[e];
      }
    }
  }
  // After a load(): the words to the lanes that use them.
  template <bool OWN>
  __device__ __forceinline__ void ready(int lane) {
    auto take = [](unsigned word) {
      if (OWN) asm volatile("" : "+v"(word));
      return word;
    };
    auto from = [&](unsigned word, int block) {
      return (unsigned)__builtin_amdgcn_ds_bpermute(4 * (16 * (block % 4) + (lane & 15)), (int)word);
    };
#pragma unroll
    for (int i = 0; i < FA; ++i) a[i] = kE8 ? from(raw_a[i / (kE8 ? 4 : 1)], i) : take(raw_a[kE8 ? 0 : i]);
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      if constexpr (kE8 && BROW) {
        b[j][0] = from(raw_b[j / 4][0], j);
      } else {
#pragma unroll
        for (int e = 0; e < kWords; ++e) b[j][e] = take(raw_b[j][e]);
      }
    }
  }
  // e8m0: on to the next k-tile's byte.
  __device__ __forceinline__ void shift() {
#pragma unroll
    for (int i = 0; i < FA; ++i) a[i] >>= 8;
#pragma unroll
    for (int j = 0; j < NB; ++j) b[j][0] >>= 8;
  }
  // Scaled product of A block i and B block j, added to acc (e8m0).
  __device__ __forceinline__ void mac(f32x4_v& acc, i32x8_t fb, i32x8_t fa, int i, int j) const {
    if constexpr (kE8) acc = mfma_e4m3_scaled(fb, fa, acc, b[BROW ? j : 0][0], a[i]);
    else add(acc, mfma_e4m3(fb, fa, f32x4_v{0.f, 0.f, 0.f, 0.f}), i, j);
  }
  // FP32: acc += p times the blocks' scales.
  __device__ __forceinline__ void add(f32x4_v& acc, f32x4_v p, int i, int j) const {
    const float sa = __uint_as_float(a[i]);
    if constexpr (BROW) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        acc[e] = __builtin_fmaf(p[e], sa * __uint_as_float(b[j][e < kWords ? e : 0]), acc[e]);
    } else {
      const float s = sa * __uint_as_float(b[0][0]);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] = __builtin_fmaf(p[e], s, acc[e]);
    }
  }
};

// BF16 output through the wave's LDS staging rows, as 16-byte row pieces. Outputs that are no
// whole aligned vectors (GemmParams::vec_out 0) leave the staging rows element by element.
struct Fp8Epi {
  template <int FA, int FB>
  __device__ __forceinline__ static void run(const GemmParams& p, Acc16<FA, FB>& acc, int m_base,
                                             int n_base, int lane, int tm, int tn, int wn,
                                             unsigned char* stage) {
    if (p.vec_out) {
      FEpiStore<false, false>::run(p, acc, m_base, n_base, lane, tm, tn, wn, stage);
      return;
    }
    constexpr int kRow = epi_row<FB>(), LPR = FB * 2, RPI = 64 / LPR;
    opaque_lane(lane);
#pragma unroll
    for (int i = 0; i < FA; ++i)
#pragma unroll
      for (int j = 0; j < FB; ++j) {
        const u32x2_t w = {pack_bf16x2(acc.v[i][j][0], acc.v[i][j][1]), pack_bf16x2(acc.v[i][j][2], acc.v[i][j][3])};
        *reinterpret_cast<u32x2_t*>(stage + (16 * i + (lane & 15)) * kRow + (16 * j + 4 * (lane >> 4)) * 2) = w;
      }
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): this wave's staging writes landed
    const int c8 = 8 * (lane % LPR);
#pragma unroll 1
    for (int r = lane / LPR; r < FA * 16; r += RPI) {
      if (m_base + r >= p.M) break;
      const auto* src = reinterpret_cast<const unsigned short*>(stage + r * kRow + c8 * 2);
      unsigned short* out = p.c + (long)(m_base + r) * p.ldc + n_base + c8;
#pragma unroll 1
      for (int e = 0; e < 8 && n_base + c8 + e < p.N; ++e) out[e] = src[e];
    }
  }
};

// A tile's sums as FP32, rows of `width` floats; `block` is this wave's first element.
template <int FA, int FB>
__device__ __forceinline__ void fp8_partial(Acc16<FA, FB>& acc, float* block, int width, int lane) {
  opaque_lane(lane);
#pragma unroll
  for (int i = 0; i < FA; ++i)
#pragma unroll
    for (int j = 0; j < FB; ++j)
      *reinterpret_cast<f32x4_v*>(block + (16 * i + (lane & 15)) * width + 16 * j + 4 * (lane >> 4)) = acc.v[i][j];
}

// Adds the slices of split tiles in order and rounds once. blockIdx.y is the tile after
// `whole`; a block of 256 threads takes 1024 elements.
template <int BM, int BN>
static __global__ void __launch_bounds__(256) fp8_join_kernel(const GemmParams p, const Fp8Params sp, int window) {
  int tm, tn;
  tile_position(xcd_remap(sp.whole + blockIdx.y, p.total_tiles, window), p.tiles_m, p.tiles_n, tm, tn);
  const int e = (blockIdx.x * 256 + threadIdx.x) * 4;
  const int m = tm * BM + e / BN, n = tn * BN + e % BN;
  if (m >= p.M || n >= p.N) return;
  const float* src = sp.partials + (long)blockIdx.y * sp.splits * (BM * BN) + e;
  f32x4_v v = *reinterpret_cast<const f32x4_v*>(src);
  for (int s = 1; s < sp.splits; ++s) v += *reinterpret_cast<const f32x4_v*>(src + (long)s * (BM * BN));
  unsigned short* out = p.c + (long)m * p.ldc + n;
  if (p.vec_out) {
    *reinterpret_cast<u32x2_t*>(out) = u32x2_t{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < p.N) out[i] = to_bf16_bits(v[i]);
  }
}

// Macro-tiles up to 128 x 128 (RingCfg): S LDS stages, one workgroup per tile, or per
// slice of a tile's k-tiles. The scales of a
// k-tile are requested before the operand loads of the same turn, so the waits that count
// operand loads only wait for more than they need.
template <class Cfg, int SCALE, bool BROW>
__global__ void __launch_bounds__(Cfg::NT) gemm_fp8_ring_kernel(const GemmParams p, const Fp8Params sp) {
  constexpr int FA = Cfg::FA, FB = Cfg::FB, S = Cfg::S;
  constexpr int TM = Cfg::TM, TN = Cfg::TN;
  extern __shared__ __attribute__((aligned(1024))) unsigned char rsmem[];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / Cfg::WN, wn = wave % Cfg::WN;
  const int kb = blockIdx.y * sp.slice_kt, ke = min(cdiv(p.K, kFBK), kb + sp.slice_kt);

  int tm, tn;
  tile_position(xcd_remap(blockIdx.x, p.total_tiles, kRingWindow), p.tiles_m, p.tiles_n, tm, tn);
  const int row0_a = tm * Cfg::BM, row0_b = tn * Cfg::BN;

  RingTile<Cfg::BM, Cfg::NT, kKContig, false> la;
  RingTile<Cfg::BN, Cfg::NT, kKContig, false> lb;
  la.init(p.a, row0_a, p.M, 0, wave, lane);
  lb.init(p.b, row0_b, p.N, 0, wave, lane);
  constexpr int kWaitLoads = (RingTile<Cfg::BM, Cfg::NT, kKContig, false>::kIns +
                              RingTile<Cfg::BN, Cfg::NT, kKContig, false>::kIns) * (S - 2);

  Acc16<FA, FB> acc;
#pragma unroll
  for (int i = 0; i < FA; ++i)
#pragma unroll
    for (int j = 0; j < FB; ++j) acc.v[i][j] = f32x4_v{0.f, 0.f, 0.f, 0.f};

  auto issue = [&](int kt, int stage) {
    unsigned char* st = rsmem + stage * Cfg::kStage;
    la.issue(p.a, row0_a, kt * kFBK, p.K, st, wave, lane);
    lb.issue(p.b, row0_b, kt * kFBK, p.K, st + Cfg::kTileA, wave, lane);
  };
  WaveScales<SCALE, BROW, FA, FB> sc;
  sc.init(sp, row0_a + wm * TM, row0_b + wn * TN, p.M, p.N, lane);
  sc.load(kb);
#pragma unroll
  for (int s = 0; s + 1 < S; ++s) issue(kb + s, s);
  int rd = 0, wr = S - 1;
  for (int kt = kb; kt < ke; ++kt) {
    __builtin_amdgcn_s_waitcnt(wait_vmcnt(kWaitLoads));
    __builtin_amdgcn_s_barrier();
    constexpr int kStep = SCALE == kScaleE8M0 ? 4 : 1;  // k-tiles of one request
    if (kt % kStep == 0) {
      sc.template ready<true>(lane);
      if (kt + kStep < ke) sc.load(kt + kStep);
    } else {
      sc.shift();
    }
    // Stage wr was read in the previous k-tile, which every wave has left (barrier).
    issue(kt + S - 1, wr);
    wr = wr + 1 == S ? 0 : wr + 1;
    __builtin_amdgcn_sched_barrier(0);
    const unsigned char* sa = rsmem + rd * Cfg::kStage;
    const unsigned char* sb = sa + Cfg::kTileA;
    i32x8_t af[FA], bf[FB];
#pragma unroll
    for (int i = 0; i < FA; ++i)
      af[i] = join_frag(read_frag(sa, wm * TM + 16 * i, 0, lane), read_frag(sa, wm * TM + 16 * i, 1, lane));
#pragma unroll
    for (int j = 0; j < FB; ++j)
      bf[j] = join_frag(read_frag(sb, wn * TN + 16 * j, 0, lane), read_frag(sb, wn * TN + 16 * j, 1, lane));
#pragma unroll
    for (int i = 0; i < FA; ++i)
#pragma unroll
      for (int j = 0; j < FB; ++j) sc.mac(acc.v[i][j], bf[j], af[i], i, j);
    rd = rd + 1 == S ? 0 : rd + 1;
    // This wave's fragment reads are complete (its MFMAs have issued) before the barrier
    // that lets other waves' loads overwrite the stage.
    __builtin_amdgcn_sched_barrier(0);
  }
  // The loads past the last k-tile land, and every wave is done reading, before the
  // epilogue's staging writes.
  __builtin_amdgcn_s_waitcnt(wait_vmcnt(0));
  __builtin_amdgcn_s_barrier();
  if (sp.splits > 1) {
    fp8_partial(acc, sp.partials + ((long)blockIdx.x * sp.splits + blockIdx.y) * (Cfg::BM * Cfg::BN) +
                         wm * TM * Cfg::BN + wn * TN, Cfg::BN, lane);
    return;
  }
  Fp8Epi::run(p, acc, row0_a + wm * TM, row0_b + wn * TN, lane, tm, tn, wn,
           rsmem + wave * epi_wave<FA, FB>());
}

// 256 x 256 tiles: the two-group pipeline of gemm_fast.h (its comment has the schedule), A in
// two LDS stages and B in three. A k-tile is 24 fragment reads and 32 MFMAs, as many LDS bytes
// and as much matrix-pipe time as there. The scales are requested at the head of a read phase,
// ahead of its operand loads: a wait that leaves those in flight has then seen the scales.
// Fragment of the 16-row block at `at` (its lane's first chunk): the chunks c and c ^ 4.
__device__ __forceinline__ i32x8_t fp8_frag(const unsigned char* tile, unsigned at) {
  return join_frag(*reinterpret_cast<const bf16x8_t*>(tile + at), *reinterpret_cast<const bf16x8_t*>(tile + (at ^ 64)));
}

// Keeps what made these values before the LDS reads and barriers that follow.
__device__ __forceinline__ void pin(f32x4_v& a, f32x4_v& b) {
  asm volatile("" : "+v"(a), "+v"(b)::"memory");
}

template <int SCALE, bool BROW>
__global__ void __launch_bounds__(kFNT) gemm_fp8_kernel(const GemmParams p, const Fp8Params sp) {
  constexpr int TM = kFBM / kFWM, TN = kFBN / kFWN;  // 64 x 128
  constexpr int FA = TM / 16, FB = TN / 16;          // 4 x 8
  extern __shared__ __attribute__((aligned(1024))) unsigned char fsmem[];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / kFWN, wn = wave % kFWN;
  const bool first = wave < 4;  // the group that runs a phase ahead and loads A
  const int items = sp.whole + (p.total_tiles - sp.whole) * sp.splits;

  unsigned char* const sA = fsmem;
  unsigned char* const sB = fsmem + 2 * kFTileBytes;
  const unsigned aoff = frag_base<kKContig>(wm * TM, lane), boff = frag_base<kKContig>(wn * TN, lane);

  for (int w = blockIdx.x; w < items; w += gridDim.x) {
    const bool slice = w >= sp.whole;
    const int piece = w - sp.whole, tile = slice ? sp.whole + piece / sp.splits : w;
    const int kb = slice ? piece % sp.splits * sp.slice_kt : 0;
    const int ke = slice ? min(cdiv(p.K, kFBK), kb + sp.slice_kt) : cdiv(p.K, kFBK);
    int tm, tn;
    tile_position(xcd_remap(tile, p.total_tiles, gridDim.x), p.tiles_m, p.tiles_n, tm, tn);
    const int row0_a = tm * kFBM, row0_b = tn * kFBN;
    Acc16<FA, FB> acc;
#pragma unroll
    for (int i = 0; i < FA; ++i)
#pragma unroll
      for (int j = 0; j < FB; ++j) acc.v[i][j] = f32x4_v{0.f, 0.f, 0.f, 0.f};
    WaveScales<SCALE, BROW, FA, FB> sc;
    sc.init(sp, row0_a + wm * TM, row0_b + wn * TN, p.M, p.N, lane);
    if (SCALE == kScaleE8M0) sc.load(kb);

    // This wave's share of its group's operand tile: one quarter, eight loads of 8 rows each,
    // 32 rows apart. Rows past the matrix take the last one's bytes (their results are not
    // stored), so the offsets need no registers of their own: three instructions per load,
    // against eight registers, which the FP32 scales' partial products need.
    const int gw = wave & 3, r0 = gw * 8 + (lane >> 3), c16 = 16 * ((lane & 7) ^ swz(r0));
    const int r_last = (first ? p.M - row0_a : p.N - row0_b) - 1;
    const unsigned ld = (unsigned)(2 * (first ? p.a.s_row : p.b.s_row));
    const unsigned short* base = first ? p.a.ptr + (long)row0_a * p.a.s_row : p.b.ptr + (long)row0_b * p.b.s_row;
    auto load = [&](int kt, unsigned char* stage, auto whole) {
      __amdgpu_buffer_rsrc_t rs = make_rsrc(base + (long)kt * kFBK, 0x7fffffff);
      unsigned char* dst = stage + gw * 1024;
      int r = r0;
      asm volatile("" : "+v"(r));  // not hoisted out of the loop
      // Chunks at k >= K land as zeros.
      const bool ok = decltype(whole)::value || kt * kFBK + (c16 >> 1) < p.K;
#pragma unroll
      for (int i = 0; i < kFIns; ++i) {
        const unsigned off = __umul24((unsigned)min(r + 32 * i, r_last), ld) + (unsigned)c16;
        dma16(rs, dst + i * 4096, ok ? off : kOOB);
      }
    };
    if (first) {
      load(kb, sA, std::false_type{});
      __builtin_amdgcn_s_waitcnt(wait_vmcnt(0));
    } else {
      load(kb, sB, std::false_type{});
      if (kb + 1 < ke) {
        load(kb + 1, sB + kFTileBytes, std::false_type{});
        __builtin_amdgcn_s_waitcnt(wait_vmcnt(kFIns));  // B(kb)
      } else {
        __builtin_amdgcn_s_waitcnt(wait_vmcnt(0));
      }
    }
    __builtin_amdgcn_s_barrier();
    if (!first) __builtin_amdgcn_s_barrier();  // one phase behind from here on
    unsigned ast = 0, bst = 0;  // byte offsets of the k-tile's stages
    // k-tile kt; the last two (TAIL) load nothing past the end, and the one before them may
    // load a ragged one. (With the ragged case in the loop, as a branch, the compiler loses
    // count of the loads that follow the scales' and waits for those of the k-tile ahead.)
    auto k_tile = [&](int kt, auto tail, auto whole) {
      constexpr bool TAIL = decltype(tail)::value;
      // Read phase. A(kt + 1) goes to the stage A(kt - 1) used and B(kt + 2) to the one
      // B(kt - 1) used: both groups have read those.
      // e8m0 scales are requested four k-tiles ahead (the last request is repeated: with one left
      // out, as a branch, the compiler loses count of the loads after it; requested where they are
      // used, 8192 x 8192 x 8192 with B's scales by rows took 416 us against 404). FP32 scales, which
      // would take more registers than there are, for this MFMA phase.
      if constexpr (SCALE == kScaleF32) {
        sc.load(kt);
      } else if ((kt & 3) == 0) {
        sc.template ready<true>(lane);
        sc.load(min(kt + 4, (ke - 1) & ~3));
      } else {
        sc.shift();
      }
      __builtin_amdgcn_sched_barrier(0);
      if (!TAIL)
        load(first ? kt + 1 : kt + 2,
             first ? sA + (ast ^ kFTileBytes) : sB + (bst == 0 ? 2 * kFTileBytes : bst - kFTileBytes), whole);
      else if (first && kt + 1 < ke)
        load(kt + 1, sA + (ast ^ kFTileBytes), whole);
      __builtin_amdgcn_sched_barrier(0);
      i32x8_t fa[FA], fb[FB / 2];
#pragma unroll
      for (int i = 0; i < FA; ++i) fa[i] = fp8_frag(sA + ast, aoff + 2048 * i);
#pragma unroll
      for (int j = 0; j < FB / 2; ++j) fb[j] = fp8_frag(sB + bst, boff + 2048 * j);
      __builtin_amdgcn_sched_barrier(0);
      // B(kt + 1) has landed (only the second group has older operand loads in flight here; the
      // first would wait for the scales just requested), and this wave's reads are done. In the last k-tile neither group has a load in flight from
      // here on, so that the first group's epilogue may stage through LDS.
      if (!TAIL && !first) __builtin_amdgcn_s_waitcnt(wait_vmcnt(kFIns));
      if (TAIL && !first) __builtin_amdgcn_s_waitcnt(wait_vmcnt(0));
      if constexpr (SCALE == kScaleF32) sc.template ready<false>(lane);
      __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
      __builtin_amdgcn_s_barrier();
      __builtin_amdgcn_sched_barrier(0);
      // MFMA phase. The second half of B's blocks is read into the first half's registers as
      // those are used up; B(kt)'s stage is not refilled before the next phase but one. In the
      // last k-tile a wave of the second group that is ahead would stage its output over blocks
      // that another still reads: the group meets once its reads are done, at a barrier that
      // the first group takes before its epilogue.
      auto reads_done = [&] {
        if (TAIL && !first && kt + 1 == ke) {
          __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
          __builtin_amdgcn_s_barrier();
        }
      };
      if constexpr (SCALE == kScaleE8M0) {
#pragma unroll
        for (int j = 0; j < FB; ++j) {
#pragma unroll
          for (int i = 0; i < FA; ++i) sc.mac(acc.v[i][j], fb[j % (FB / 2)], fa[i], i, j);
          pin(acc.v[0][j], acc.v[1][j]);
          pin(acc.v[2][j], acc.v[3][j]);
          if (j < FB / 2) fb[j] = fp8_frag(sB + bst, boff + 2048 * (j + FB / 2));
          if (j == FB / 2 - 1) reads_done();
          // (Left to the scheduler, all four reads go through one block's registers, each
          // waited for at once.)
          __builtin_amdgcn_sched_barrier(0);
        }
      } else {
        // The additions of two blocks run behind the next two blocks' MFMAs.
        f32x4_v prod[2][2];
#pragma unroll
        for (int q = 0; q <= 2 * FB; ++q) {
          const int j = q / 2, i = 2 * (q % 2);
          if (q < 2 * FB) {
            prod[q & 1][0] = mfma_e4m3(fb[j % (FB / 2)], fa[i], f32x4_v{0.f, 0.f, 0.f, 0.f});
            prod[q & 1][1] = mfma_e4m3(fb[j % (FB / 2)], fa[i + 1], f32x4_v{0.f, 0.f, 0.f, 0.f});
            pin(prod[q & 1][0], prod[q & 1][1]);
            if (i == 2 && j < FB / 2) fb[j] = fp8_frag(sB + bst, boff + 2048 * (j + FB / 2));
            if (i == 2 && j == FB / 2 - 1) reads_done();
          }
          if (q > 0) {
            const int jp = (q - 1) / 2, ip = 2 * ((q - 1) % 2);
            sc.add(acc.v[ip][jp], prod[(q - 1) & 1][0], ip, jp);
            sc.add(acc.v[ip + 1][jp], prod[(q - 1) & 1][1], ip + 1, jp);
            pin(acc.v[ip][jp], acc.v[ip + 1][jp]);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      if (first) __builtin_amdgcn_s_waitcnt(wait_vmcnt(0));  // A(kt + 1) has landed
      // The second group's last MFMA phase ends the loop: the first group is past it.
      if (!TAIL || first || kt + 1 < ke) __builtin_amdgcn_s_barrier();
      __builtin_amdgcn_sched_barrier(0);
      ast ^= kFTileBytes;
      bst = bst == 2 * kFTileBytes ? 0 : bst + kFTileBytes;
    };
    int kt = kb;
    for (; kt + 3 < ke; ++kt) k_tile(kt, std::false_type{}, std::true_type{});
    if (kt + 2 < ke) k_tile(kt++, std::false_type{}, std::false_type{});
    for (; kt < ke; ++kt) k_tile(kt, std::true_type{}, std::false_type{});
    if (first) __builtin_amdgcn_s_barrier();  // the second group's reads of the last k-tile
    if (slice)
      fp8_partial(acc, sp.partials + (long)piece * (kFBM * kFBN) + wm * TM * kFBN + wn * TN, kFBN, lane);
    else
      Fp8Epi::run(p, acc, row0_a + wm * TM, row0_b + wn * TN, lane, tm, tn, wn, fsmem + wave * kFStageWave);
    __builtin_amdgcn_s_barrier();
  }
}

// Few rows of A (at most 32: decoding, a short prompt): bound by reading B once. A workgroup of
// eight waves takes all rows and 16 columns (sixteen waves, with fewer k-tiles each, were slower
// everywhere: 1 x 11264 x 2048 10.5 us against 8.2); the waves share the k-tiles in turn and
// read their fragments straight from memory (B's rows as whole 128-byte lines, A's from L2), the
// next kAhead k-tiles requested before the current ones are used, and their partial products
// are added in LDS in wave order. 1 x 2048 x 5632: 6.2 us, of which reading B at the card's copy rate
// takes 2.4.
template <int FA, int SCALE, bool BROW>
__global__ void __launch_bounds__(512) gemm_fp8_skinny_kernel(const GemmParams p, const Fp8Params sp) {
  constexpr int kWaves = 8, kAhead = 4;
  constexpr bool kE8 = SCALE == kScaleE8M0;
  constexpr int kSB = kE8 || !BROW ? 1 : 4;
  __shared__ f32x4_v red[kWaves][FA][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = blockIdx.x * 16;
  const int ke = cdiv(p.K, kFBK);
  const long lda = 2 * p.a.s_row, ldb = 2 * p.b.s_row;
  const int kb = 2 * p.K;  // bytes of a row
  const unsigned char *pa[FA], *pb;
  const char *psa[FA], *psb;
  const int chunk = 16 * (lane >> 4);
#pragma unroll
  for (int i = 0; i < FA; ++i) {
    const int r = min(16 * i + (lane & 15), p.M - 1);
    pa[i] = reinterpret_cast<const unsigned char*>(p.a.ptr) + r * lda + chunk;
    const long q = r >> sp.a.shift;
    psa[i] = static_cast<const char*>(sp.a.ptr) + (kE8 ? q * sp.a.ld : 4 * q);
  }
  {
    const int r = min(n0 + (lane & 15), p.N - 1);
    pb = reinterpret_cast<const unsigned char*>(p.b.ptr) + r * ldb + chunk;
    // FP32 by rows: a lane's four columns at once (past the end the last whole four).
    const long q = kSB == 4 ? min(n0 + 4 * (lane >> 4), (p.N - 1) & ~3) : r >> sp.b.shift;
    psb = static_cast<const char*>(sp.b.ptr) + (kE8 ? q * sp.b.ld : 4 * q);
  }
  const long step_a = kE8 ? 1 : 4 * sp.a.ld, step_b = kE8 ? 1 : 4 * sp.b.ld;
  struct Piece {
    i32x8_t a[FA], b;
    unsigned sa[FA], sb[kSB];
  };
  auto load8 = [&](const unsigned char* row, int kt) {
    const u32x4_t zero = {0, 0, 0, 0};
    const int at = kt * 128;
    const u32x4_t lo = at + chunk < kb ? *reinterpret_cast<const u32x4_t*>(row + at) : zero;
    const u32x4_t hi = at + 64 + chunk < kb ? *reinterpret_cast<const u32x4_t*>(row + at + 64) : zero;
    return join_frag(__builtin_bit_cast(bf16x8_t, lo), __builtin_bit_cast(bf16x8_t, hi));
  };
  auto fetch = [&](Piece& x, int kt) {
    if (kt >= ke) return;  // uniform
    x.b = load8(pb, kt);
#pragma unroll
    for (int i = 0; i < FA; ++i) x.a[i] = load8(pa[i], kt);
#pragma unroll
    for (int i = 0; i < FA; ++i) {
      const char* q = psa[i] + kt * step_a;
      x.sa[i] = kE8 ? (unsigned)*reinterpret_cast<const unsigned char*>(q) : *reinterpret_cast<const unsigned*>(q);
    }
    const char* q = psb + kt * step_b;
    if constexpr (kSB == 4) {
      const u32x4_t v = *reinterpret_cast<const u32x4_t*>(q);
#pragma unroll
      for (int e = 0; e < 4; ++e) x.sb[e] = v[e];
    } else {
      x.sb[0] = kE8 ? (unsigned)*reinterpret_cast<const unsigned char*>(q) : *reinterpret_cast<const unsigned*>(q);
    }
  };
  f32x4_v acc[FA];
#pragma unroll
  for (int i = 0; i < FA; ++i) acc[i] = f32x4_v{0.f, 0.f, 0.f, 0.f};
  auto use = [&](const Piece& x, int kt) {
    if (kt >= ke) return;  // uniform
#pragma unroll
    for (int i = 0; i < FA; ++i) {
      if constexpr (kE8) {
        acc[i] = mfma_e4m3_scaled(x.b, x.a[i], acc[i], x.sb[0], x.sa[i]);
      } else {
        const f32x4_v v = mfma_e4m3(x.b, x.a[i], f32x4_v{0.f, 0.f, 0.f, 0.f});
#pragma unroll
        for (int e = 0; e < 4; ++e)
          acc[i][e] = __builtin_fmaf(v[e], __uint_as_float(x.sa[i]) * __uint_as_float(x.sb[kSB == 4 ? e : 0]), acc[i][e]);
      }
    }
  };
  Piece piece[kAhead];
#pragma unroll
  for (int u = 0; u < kAhead; ++u) fetch(piece[u], wave + u * kWaves);
  for (int kt = wave; kt < ke; kt += kAhead * kWaves) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      use(piece[u], kt + u * kWaves);
      fetch(piece[u], kt + (u + kAhead) * kWaves);
    }
  }
#pragma unroll
  for (int i = 0; i < FA; ++i) red[wave][i][lane] = acc[i];
  __syncthreads();
  for (int q = threadIdx.x; q < FA * 64; q += 512) {
    const int blk = q >> 6, l = q & 63;
    f32x4_v v = red[0][blk][l];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) v += red[w][blk][l];
    const int m = 16 * blk + (l & 15), n = n0 + 4 * (l >> 4);
    if (m >= p.M) continue;
    unsigned short* out = p.c + (long)m * p.ldc + n;
    if (p.vec_out) {
      if (n + 3 < p.N) *reinterpret_cast<u32x2_t*>(out) = u32x2_t{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < p.N) out[e] = to_bf16_bits(v[e]);
    }
  }
}

}  // namespace ws
