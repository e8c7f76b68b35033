// C ABI: quantization to e4m3 in blocks of 128 and the block-scaled 8-bit product.
#include "../../include/warpstate_hip.h"
#include "gemm_fp8.h"
#include "launch.h"

using namespace ws;

namespace {

// Workgroups of 256 threads in one launch, which has fewer than 2^32 threads.
bool fits_launch(long blocks) { return blocks < 1L << 24; }

template <bool F32, int SCALE, int FORM, int R = 8>
int run_quantize(const QuantParams& p, bool vec, hipStream_t s) {
  const long tiles = (long)cdiv(p.rows, 16 * R) * p.col_tiles;
  if (!fits_launch(tiles)) return set_error(kInvalid, "too many 128 x 128 tiles");
  if constexpr (FORM == kQuantRows && R == 8) {
    // Few tiles: a row per thread (1 x 5632: 5.9 -> 2.9 us).
    if (tiles < device_cus()) return run_quantize<F32, SCALE, FORM, 1>(p, vec, s);
  }
  if (vec)
    hipLaunchKernelGGL((quantize_kernel<F32, SCALE, FORM, true, R>), dim3((unsigned)tiles), dim3(256), 0, s, p);
  else
    hipLaunchKernelGGL((quantize_kernel<F32, SCALE, FORM, false, R>), dim3((unsigned)tiles), dim3(256), 0, s, p);
  return hip_check(hipGetLastError(), "quantize launch");
}
template <bool F32, int SCALE>
int dispatch_quantize(const QuantParams& p, int form, bool vec, hipStream_t s) {
  switch (form) {
    case kQuantRows: return run_quantize<F32, SCALE, kQuantRows>(p, vec, s);
    case kQuantCols: return run_quantize<F32, SCALE, kQuantCols>(p, vec, s);
    case kQuantRows | kQuantCols: return run_quantize<F32, SCALE, kQuantRows | kQuantCols>(p, vec, s);
    case kQuantBlocks: return run_quantize<F32, SCALE, kQuantBlocks>(p, vec, s);
  }
  return set_error(kInvalid, "unknown quantization form %d", form);
}

// How a product runs: a macro-tile (FastTile), or kTileFew, and the slices along K of the
// tiles from `whole` on.
constexpr int kTileFew = kFastTiles;
struct Fp8Plan {
  int tile, whole, splits, slice_kt;
  long partials;  // floats
};

// us of adding `splits` slices of `tiles` tiles (written and read once, mostly in cache).
inline float join_time(long tiles, int bm, int bn, int splits) {
  return 3.0f + (float)tiles * (float)(bm * bn) * 8.0f * (float)splits / 6e6f;
}

// The macro-tile by the BF16 kernels' cost table: a k-tile of 128 bytes a row takes as many LDS
// bytes and as much matrix-pipe time in either type.
Fp8Plan fp8_plan(long m, long n, long k, bool brow, int scale_type) {
  const long pairs = k / 2;  // the loaders' count
  const int kt = cdiv(pairs, kFBK), cus = device_cus();
  Fp8Plan best{kTileFew, 0, 1, kt, 0};
  // Few rows: reading A's fragments once per 16 columns costs less than tiles' prologues until
  // the columns fill the card with tiles (16 rows) or with workgroups of 16 columns (32 rows,
  // a reduction that eight waves share in few steps). us of e8m0 products, few rows' kernel /
  // the best tile: 16 x 8192 x 2048 7.5 / 9.6, 16 x 16384 x 2048 12.3 / 9.9, 32 x 4096 x 2048 6.1 /
  // 8.5, 32 x 6144 x 2048 10.4 / 9.4, 32 x 2048 x 5632 11.7 / 13.0, 32 x 2048 x 8192 17.7 / 12.5 (the
  // rule's edge), 32 x 2048 x 11264 21.1 / 15.8. Up to 16 rows the rule does not ask for K:
  // 16 x 2048 x 5632 8.9 / 12.3, x 8192 12.5 / 11.9, x 11264 14.6 / 14.8, x 16384 22.0 / 17.5, 8 rows
  // x 16384 18.0 / 17.2, one row x 16384 13.0 / 17.1.
  if (m <= 16 ? cdiv(n, 64) < cus : m <= 32 && cdiv(n, 16) <= cus && k <= 8192) return best;
  float t = 1e30f;
  for (int tile = 0; tile < kFastTiles; ++tile) {
    if (tile == kTile256 && scale_type == kScaleF32 && brow) continue;  // (would not fit the registers)
    const TileCost& c = tile_cost(tile, kKContig, kKContig);
    const long tiles = (long)cdiv(m, c.bm) * cdiv(n, c.bn);
    const int whole = tile == kTile256 ? (int)(tiles / cus * cus) : 0;
    const long rest = tiles - whole;
    float plain = tile_time(tile, m, n, pairs, kKContig, kKContig, cus, false, kEpiStore);
    if (plain < t) {
      t = plain;
      best = Fp8Plan{tile, (int)tiles, 1, kt, 0};
    }
    const int room = cus * (c.pair > 0.0f ? 2 : 1);  // workgroups at once
    for (int want = 2; rest > 0 && want <= 16 && rest * want <= room; ++want) {
      const int slice = cdiv(cdiv(kt, want), 4) * 4, splits = cdiv(kt, slice);
      if (splits < 2 || rest * splits > room) continue;
      const bool paired = rest * splits > cus;
      float time = (float)(whole / cus) * (c.alone * (float)kt + c.fixed) +
                   (paired ? c.pair : c.alone) * (float)slice + c.fixed + join_time(rest, c.bm, c.bn, splits);
      if (time < t) {
        t = time;
        best = Fp8Plan{tile, whole, splits, slice, rest * splits * c.bm * c.bn};
      }
    }
  }
  return best;
}

template <int BM, int BN>
int run_join(const GemmParams& p, const Fp8Params& sp, int window, hipStream_t s) {
  hipLaunchKernelGGL((fp8_join_kernel<BM, BN>), dim3(BM * BN / 1024, p.total_tiles - sp.whole), dim3(256), 0, s, p,
                     sp, window);
  return hip_check(hipGetLastError(), "8-bit product join launch");
}
template <class Cfg, int SCALE, bool BROW>
int run_fp8_ring(GemmParams p, const Fp8Params& sp, hipStream_t s) {
  const void* kern = reinterpret_cast<const void*>(&gemm_fp8_ring_kernel<Cfg, SCALE, BROW>);
  if (int rc = ensure_lds(kern, Cfg::kLds)) return rc;
  p.tiles_m = cdiv(p.M, Cfg::BM);
  p.tiles_n = cdiv(p.N, Cfg::BN);
  p.total_tiles = p.tiles_m * p.tiles_n;
  hipLaunchKernelGGL((gemm_fp8_ring_kernel<Cfg, SCALE, BROW>), dim3(p.total_tiles, sp.splits), dim3(Cfg::NT),
                     Cfg::kLds, s, p, sp);
  if (int rc = hip_check(hipGetLastError(), "8-bit product launch")) return rc;
  return sp.splits > 1 ? run_join<Cfg::BM, Cfg::BN>(p, sp, kRingWindow, s) : kOk;
}
template <int SCALE, bool BROW>
int run_fp8_256(GemmParams p, const Fp8Params& sp, hipStream_t s) {
  const void* kern = reinterpret_cast<const void*>(&gemm_fp8_kernel<SCALE, BROW>);
  if (int rc = ensure_lds(kern, kFLdsBytes)) return rc;
  p.tiles_m = cdiv(p.M, kFBM);
  p.tiles_n = cdiv(p.N, kFBN);
  p.total_tiles = p.tiles_m * p.tiles_n;
  const int cus = device_cus(), items = sp.whole + (p.total_tiles - sp.whole) * sp.splits;
  const int grid = items < cus ? items : cus;
  hipLaunchKernelGGL((gemm_fp8_kernel<SCALE, BROW>), dim3(grid), dim3(kFNT), kFLdsBytes, s, p, sp);
  if (int rc = hip_check(hipGetLastError(), "8-bit product launch")) return rc;
  return sp.splits > 1 ? run_join<kFBM, kFBN>(p, sp, grid, s) : kOk;
}
template <int FA, int SCALE, bool BROW>
int run_fp8_skinny(const GemmParams& p, const Fp8Params& sp, hipStream_t s) {
  hipLaunchKernelGGL((gemm_fp8_skinny_kernel<FA, SCALE, BROW>), dim3(cdiv(p.N, 16)), dim3(512), 0, s, p, sp);
  return hip_check(hipGetLastError(), "8-bit product launch");
}
template <int SCALE, bool BROW>
int run_fp8_few(const GemmParams& p, const Fp8Params& sp, hipStream_t s) {
  return p.M <= 16 ? run_fp8_skinny<1, SCALE, BROW>(p, sp, s) : run_fp8_skinny<2, SCALE, BROW>(p, sp, s);
}
template <int SCALE, bool BROW>
int run_fp8(const GemmParams& p, const Fp8Params& sp, int tile, hipStream_t s) {
  switch (tile) {
    case kTileFew: return run_fp8_few<SCALE, BROW>(p, sp, s);
    case kTile256:
      if constexpr (SCALE == kScaleE8M0 || !BROW) return run_fp8_256<SCALE, BROW>(p, sp, s);
      break;
    case kTile128x2: return run_fp8_ring<Ring128x2, SCALE, BROW>(p, sp, s);
    case kTile128x1: return run_fp8_ring<Ring128x1, SCALE, BROW>(p, sp, s);
    case kTile64x128: return run_fp8_ring<Ring64x128, SCALE, BROW>(p, sp, s);
    case kTile64: return run_fp8_ring<Ring64, SCALE, BROW>(p, sp, s);
  }
  return set_error(kInvalid, "no 8-bit macro-tile %d", tile);
}

int check_scale(const Fp8Scale& s, long rows, long k_blocks, int type, bool vec4, const char* which) {
  if (!s.ptr) return set_error(kInvalid, "null scale pointer (%s)", which);
  const long scale_rows = (rows + (1L << s.shift) - 1) >> s.shift;
  if (type == kScaleE8M0) {
    if (s.ld < k_blocks || s.ld % 4 || !al(s.ptr, 4))
      return set_error(kInvalid, "e8m0 scales of %s need 4-byte aligned rows that hold every block", which);
    if (256 * s.ld + 4 >= 0x7fffffffL) return set_error(kInvalid, "scale rows of %s are too long", which);
  } else if (s.ld < scale_rows || !al(s.ptr, vec4 ? 16 : 4) || (vec4 && s.ld % 4)) {
    return set_error(kInvalid, "FP32 scales of %s need a column of every row's scales per block%s", which,
                     vec4 ? ", in aligned groups of four" : "");
  }
  return kOk;
}

}  // namespace

extern "C" int ws_fp8_quantize(const void* x, int64_t ldx, int x_f32, int64_t rows, int64_t cols,
                               int form, int scale_type, void* q, int64_t ldq, void* scale,
                               int64_t ld_scale, void* qt, int64_t ldqt, void* scale_t,
                               int64_t ld_scale_t, void* stream) {
  if (!x) return set_error(kInvalid, "null operand pointer");
  if (rows < 1 || cols < 1 || !fits_i32(rows) || !fits_i32(cols) || rows > 0x7fffff00L || cols > 0x7fffff00L)
    return set_error(kInvalid, "invalid quantization sizes rows=%ld cols=%ld", (long)rows, (long)cols);
  if (ldx < cols) return set_error(kInvalid, "leading dimension < cols");
  if (x_f32 != 0 && x_f32 != 1) return set_error(kInvalid, "unknown input type %d", x_f32);
  if (scale_type != kScaleE8M0 && scale_type != kScaleF32)
    return set_error(kInvalid, "unknown scale type %d", scale_type);
  if (form != kQuantRows && form != kQuantCols && form != (kQuantRows | kQuantCols) && form != kQuantBlocks)
    return set_error(kInvalid, "unknown quantization form %d", form);
  const bool e8 = scale_type == kScaleE8M0;
  const long row_blocks = cdiv(rows, kQBlock), col_blocks = cdiv(cols, kQBlock);
  const long scale_rows = form == kQuantBlocks ? row_blocks : rows;
  const long scale_rows_t = form == kQuantBlocks ? col_blocks : cols;
  if (form != kQuantCols) {
    if (!q || !scale) return set_error(kInvalid, "null output pointer");
    if (ldq < cols || ldq % 16 || !al(q, 16))
      return set_error(kInvalid, "quantized rows need 16-byte aligned storage of a multiple of 16 bytes");
    if (ld_scale < (e8 ? col_blocks : scale_rows) || (!e8 && !al(scale, 4)))
      return set_error(kInvalid, "scale leading dimension too small");
  }
  if ((form & kQuantCols) || qt) {
    if (!qt || !scale_t) return set_error(kInvalid, "null output pointer");
    if (ldqt < rows || ldqt % 16 || !al(qt, 16))
      return set_error(kInvalid, "quantized columns need 16-byte aligned storage of a multiple of 16 bytes");
    if (ld_scale_t < (e8 ? row_blocks : scale_rows_t) || (!e8 && !al(scale_t, 4)))
      return set_error(kInvalid, "transposed scale leading dimension too small");
  }
  QuantParams p{};
  p.x = x;
  p.ldx = ldx;
  p.rows = (int)rows; p.cols = (int)cols; p.col_tiles = (int)col_blocks;
  p.q_cols = (int)((cols + 15) / 16 * 16);
  p.qt_cols = (int)((rows + 15) / 16 * 16);
  p.q = static_cast<unsigned char*>(q);
  p.ldq = ldq;
  p.qt = static_cast<unsigned char*>(qt);
  p.ldqt = ldqt;
  p.scale = scale;
  p.ld_scale = ld_scale;
  p.scale_t = scale_t;
  p.ld_scale_t = ld_scale_t;
  const bool vec = al(x, 16) && ldx % (x_f32 ? 4 : 8) == 0;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (x_f32)
    return e8 ? dispatch_quantize<true, kScaleE8M0>(p, form, vec, s)
              : dispatch_quantize<true, kScaleF32>(p, form, vec, s);
  return e8 ? dispatch_quantize<false, kScaleE8M0>(p, form, vec, s)
            : dispatch_quantize<false, kScaleF32>(p, form, vec, s);
}

extern "C" int ws_fp8_pack(const void* src, int64_t s_row, int64_t s_col, void* dst, int64_t ldd,
                           int64_t rows, int64_t cols, void* stream) {
  if (!src || !dst) return set_error(kInvalid, "null operand pointer");
  if (rows < 1 || cols < 1 || !fits_i32(rows) || !fits_i32(cols) || s_row < 1 || s_col < 1)
    return set_error(kInvalid, "invalid matrix to pack");
  if (ldd < cols || ldd % 16 || !al(dst, 16))
    return set_error(kInvalid, "packed rows need 16-byte aligned storage of a multiple of 16 bytes");
  const long blocks = (rows * (ldd / 16) + 255) / 256;
  if (!fits_launch(blocks)) return set_error(kInvalid, "matrix to pack is too large");
  hipLaunchKernelGGL(pack_bytes_kernel, dim3((unsigned)blocks), dim3(256), 0, static_cast<hipStream_t>(stream),
                     static_cast<const unsigned char*>(src), (long)s_row, (long)s_col,
                     static_cast<unsigned char*>(dst), (long)ldd, (long)rows, (long)cols);
  return hip_check(hipGetLastError(), "pack launch");
}

extern "C" int ws_fp8_mm_plan(int64_t m, int64_t n, int64_t k, int b_block_rows, int scale_type,
                              int64_t* workspace_bytes, int* splits) {
  if (m < 1 || n < 1 || k < 1 || !fits_i32(m) || !fits_i32(n) || !fits_i32(k)) {
    set_error(kInvalid, "matrix sizes must be positive 32-bit integers");
    return -1;
  }
  const Fp8Plan plan = fp8_plan(m, n, k, b_block_rows == 1, scale_type);
  if (workspace_bytes) *workspace_bytes = plan.partials * 4;
  if (splits) *splits = plan.splits;
  return plan.tile;
}

extern "C" int64_t ws_fp8_mm_workspace_bytes(int64_t m, int64_t n, int64_t k, int b_block_rows,
                                             int scale_type) {
  int64_t bytes = 0;
  ws_fp8_mm_plan(m, n, k, b_block_rows, scale_type, &bytes, nullptr);
  return bytes;
}

extern "C" int ws_fp8_mm(const void* a, int64_t lda, const void* scale_a, int64_t ld_scale_a,
                         int a_block_rows, const void* b, int64_t ldb, const void* scale_b,
                         int64_t ld_scale_b, int b_block_rows, int scale_type, void* c, int64_t ldc,
                         int64_t m, int64_t n, int64_t k, void* workspace, void* stream) {
  if (!a || !b || !c) return set_error(kInvalid, "null operand pointer");
  if (m < 1 || n < 1 || k < 1 || !fits_i32(m) || !fits_i32(n) || !fits_i32(k))
    return set_error(kInvalid, "matrix sizes must be positive 32-bit integers (m=%ld n=%ld k=%ld)",
                     (long)m, (long)n, (long)k);
  if (k % 16 || lda % 16 || ldb % 16 || lda < k || ldb < k || !al(a, 16) || !al(b, 16))
    return set_error(kInvalid, "8-bit operands need rows of whole 16-byte pieces (ws_fp8_pack)");
  if (257 * lda >= 0x7fffffffL || 257 * ldb >= 0x7fffffffL)
    return set_error(kInvalid, "operand rows are too long: 257 rows span 2 GiB or more");
  if (scale_type != kScaleE8M0 && scale_type != kScaleF32)
    return set_error(kInvalid, "unknown scale type %d", scale_type);
  if ((a_block_rows != 1 && a_block_rows != kQBlock) || (b_block_rows != 1 && b_block_rows != kQBlock))
    return set_error(kInvalid, "a scale covers 1 or 128 rows");
  if (ldc < n) return set_error(kInvalid, "output leading dimension < n");
  if (!al(c, 2)) return set_error(kInvalid, "misaligned output");
  if (int rc = check_out_stride(ldc, 2, "output")) return rc;
  const Fp8Plan plan = fp8_plan(m, n, k, b_block_rows == 1, scale_type);
  if (plan.partials && (!workspace || !al(workspace, 16)))
    return set_error(kInvalid, "this product needs a 16-byte aligned workspace");
  const Fp8Params sp{{scale_a, ld_scale_a, a_block_rows == 1 ? 0 : 7}, {scale_b, ld_scale_b, b_block_rows == 1 ? 0 : 7},
                     plan.whole, plan.splits, plan.slice_kt, static_cast<float*>(workspace)};
  const long k_blocks = cdiv(k, kQBlock);
  if (int rc = check_scale(sp.a, m, k_blocks, scale_type, false, "A")) return rc;
  if (int rc = check_scale(sp.b, n, k_blocks, scale_type, b_block_rows == 1, "B")) return rc;
  GemmParams p{};
  // The loaders count K in pairs of bytes.
  p.a = OperandDesc{static_cast<const unsigned short*>(a), lda / 2, 1};
  p.b = OperandDesc{static_cast<const unsigned short*>(b), ldb / 2, 1};
  p.M = (int)m; p.N = (int)n; p.K = (int)(k / 2);
  p.c = static_cast<unsigned short*>(c);
  p.ldc = ldc;
  p.vec_out = n % 4 == 0 && ldc % 4 == 0 && al(c, 8);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool brow = b_block_rows == 1;
  if (scale_type == kScaleE8M0)
    return brow ? run_fp8<kScaleE8M0, true>(p, sp, plan.tile, s) : run_fp8<kScaleE8M0, false>(p, sp, plan.tile, s);
  return brow ? run_fp8<kScaleF32, true>(p, sp, plan.tile, s) : run_fp8<kScaleF32, false>(p, sp, plan.tile, s);
}
