// C ABI: products grouped by expert.
#include <cmath>

#include "../../include/warpstate_hip.h"
#include "gemm_grouped.h"
#include "launch.h"

using namespace ws;

namespace {

// (Every workgroup searches all groups.)
constexpr int64_t kMaxGroups = 16384, kMaxRows = 1L << 30;
// Workgroups of a launch (of up to 512 threads, which have to be fewer than 2^32); and a product's tiles, of which
// a workgroup takes several: the search adds up to 66 times their number in 32 bits.
constexpr int64_t kMaxBlocks = 1L << 22, kMaxTiles = 1L << 24;
// Beside FastTile: the kernel for few rows, tiles of 32 and of 16 columns.
constexpr int kTileFew = kFastTiles, kTileFew16 = kFastTiles + 1;
// The most 256 x 256 tiles for 256 compute units whose round goes in pieces (grouped_fast_kernel).
constexpr int kPiecesOf256 = 64;

// The most slices of a reduction (never 256 x 256 tiles nor two 128 x 128 a unit, which others were faster than in
// slices), and the least k-tiles of one.
constexpr int kMaxSlices = 8, kSliceTiles = 4;

int64_t up8(int64_t n) { return (n + 7) / 8 * 8; }
int tile_rows(int tile) {
  switch (tile) {
    case kTile256: return 256;
    case kTile128x2:
    case kTile128x1: return 128;
    case kTileFew:
    case kTileFew16: return kFewRows;
    default: return 64;
  }
}
int tile_cols(int tile) {
  return tile == kTileFew ? 32 : tile == kTileFew16 ? 16 : tile == kTile256 ? 256 : tile == kTile64 ? 64 : 128;
}
// Tiles of `rows` rows that any offsets make at most: a group ends in a part of one. (The rows of
// no group form two more.)
int64_t most_tiles(int64_t rows, int64_t groups, int bm) {
  const int64_t used = groups + 2 < rows ? groups + 2 : rows;
  return rows / bm + used;
}

// The tiles that the grid of a product with n columns is sized for. Those of 256 x 256 are the fewest.
int64_t grid_tiles(int64_t rows, int64_t groups, int64_t n, int tile) {
  return most_tiles(rows, groups, tile_rows(tile)) * cdiv(n, tile_cols(tile));
}
int64_t grad_tiles(int64_t groups, int64_t m, int64_t n, int tile) {
  return groups * cdiv(m, tile_rows(tile)) * cdiv(n, tile_cols(tile));
}

// Tiles of a workgroup, one after the other: with a short reduction, finding one among the groups takes longer than
// its product (us, one / several: 512 rows, one each in 512 groups of 2048 x 16, 135 / 34, 4096 in 256 of 2048 x 64 45 / 31).
// With any reduction, as many as bring the workgroups down to what a launch takes.
int tiles_of_run(int64_t tiles, int64_t k) {
  const int64_t most = tiles / (4 * (int64_t)device_cus()), run = k > 256 || most < 2 ? 1 : most < 16 ? most : 16;
  const int64_t least = (tiles + kMaxBlocks - 1) / kMaxBlocks;
  return (int)(run < least ? least : run);
}

// The tile for rows that are spread over the groups, by the cost table of single products, for the
// rows of the tiles that a group of average size makes (its last one is half full on average, and
// there is one); and the slices of a long reduction whose tiles leave units idle (us, whole / in slices: 64 rows
// in 2 groups of 2048 x 11264 50 / 25, 494 in 3 of 960 x 9704 46 / 29, 64 in 8 of 2048 x 5632 34 / 37). What is
// added to the table was fitted to 440 drawn sizes: over the 427 that the kernel for few rows does not take, the choice
// is 3 % behind the best tile and slices, 2 % for reductions up to 2048 (the table alone 19 and 5 %, the best tiles
// without slices 15 %).
struct GroupedPlan {
  int tile, slices;
};
GroupedPlan pick_grouped(int64_t rows, int64_t groups, int64_t n, int64_t k, int bmode) {
  const int64_t used = groups < rows ? groups : rows;
  if (bmode == kKContig) {
    // Up to 6 rows for each group, above which some groups take two tiles of 16 (us, this kernel / the best other):
    // 48 rows in 8 groups of 5632 x 2048 41 / 41, of 1024 x 8192 29 / 31, 64 rows 41 / 43 and 44 / 31; 256 in 32 of
    // 1024 x 1280 20 / 17. Up to 16 where its tiles leave units idle, and larger ones more so, or 8 where the reduction is
    // long enough for many slices: 32 in 2 of 2048 x 2048 8 / 9.5, of 2048 x 11264 32 / 23, 32 in 4 of 1024 x 4096
    // 9 / 12, 64 13 / 12; 128 in 8 of 512 x 1280 6 / 8.5.
    const int64_t tiles = (int64_t)cdiv(n, 32) * (used + rows / 16), cus = device_cus();
    if ((rows <= 6 * used || (rows <= (k < 4096 ? 16 : 8) * used && tiles <= cus)) &&
        grid_tiles(rows, groups, n, kTileFew) < kMaxTiles) {
      // Tiles of 16 columns, whose rows of x are read twice as often, for idle units, and for long
      // reductions with very few rows (32 / 16 columns): 48 rows in 8 groups of 512 x 2048 7.7 / 6.0, 96 8.1 /
      // 9.4; 32 in 8 of 5632 x 2048 41 / 35; 32 in 8 of 7168 x 1472 30.5 / 32.5; 256 in 32 of 1024 x 2048 29.5 / 32.
      const bool narrow = 4 * tiles <= 3 * cus || (k >= 2048 && rows <= 6 * used);
      return {narrow && grid_tiles(rows, groups, n, kTileFew16) <= kMaxBlocks ? kTileFew16 : kTileFew, 1};
    }
  }
  // Two workgroups on a unit with few stages hide less of what comes from HBM, one with more hides more.
  static const float slower[kFastTiles] = {1.0f, 1.2f, 0.9f, 1.0f, 1.0f};
  GroupedPlan best = {kTile256, 1};
  float t = 0.0f;
  for (int tile = 0; tile < kFastTiles; ++tile) {
    if (tile != kTile256 && grid_tiles(rows, groups, n, tile) >= kMaxTiles) continue;
    const int64_t bm = tile_rows(tile), cus = device_cus();
    int64_t wide = rows + used * bm / 2;
    if (wide < used * bm) wide = used * bm;
    // Many groups make some tiles more or fewer: a round that is just full is not counted on.
    if (used >= 16) wide += (int64_t)(0.2f * (float)bm * std::sqrt((float)used));
    // What the tiles read, each weight once for every tile of rows, at the caches' rate, and what HBM gives. (1000
    // rows in 8 groups of 2048 x 5632: 64 x 128, by the table, 83 us, 128 x 128 61.)
    const float fn = (float)n, fk = 2.0f * (float)k, frows = (float)rows, fused = (float)used;
    float read = ((float)(rows / bm + used) * fn * fk + (float)cdiv(n, tile_cols(tile)) * frows * fk) / 12e6f;
    const float once = (fused * fn * fk + frows * (2.0f * fn + fk)) / 7e6f;
    if (read < once) read = once;
    for (int slices = 1; slices <= (tile == kTile256 || tile == kTile128x2 ? 1 : kMaxSlices); slices *= 2) {
      if (slices > 1 && (k < (int64_t)slices * kSliceTiles * kFBK || grid_tiles(rows, groups, n, tile) > kMaxBlocks)) break;
      float ti = slower[tile] * tile_time(tile, wide, n, k, kKContig, bmode, cus, false, kEpiStore, slices);
      if (tile == kTile256) {
        const TileCost& c = tile_cost(tile, kKContig, bmode);
        const int64_t tiles = cdiv(wide, 256) * (int64_t)cdiv(n, 256), rest = tiles % cus;
        const float kt = (float)cdiv(k, kFBK);
        if (rest * 256 <= kPiecesOf256 * cus)
          ti = (float)(tiles / cus) * (c.alone * kt + c.fixed) + (rest * 8 <= cus ? 0.45f : 0.62f) * kt + 4.0f;
      }
      if (ti < read) ti = read;
      // The second kernel, and the slices' sums there and back.
      if (slices > 1) ti += 4.0f + frows * fn * (float)(8 * slices) / 4e6f;
      if ((tile == 0 && slices == 1) || ti < t) {
        best = {tile, slices};
        t = ti;
      }
    }
  }
  return best;
}
int pick_grad(int64_t rows, int64_t groups, int64_t m, int64_t n) {
  int best = kTile256;
  float t = 0.0f;
  for (int tile = 0; tile < kFastTiles; ++tile) {
    const int64_t bm = tile_rows(tile);
    // With a k-tile or less for each group the smaller tile's stores start sooner (64 groups of 512 x
    // 1280 over 4096 rows, BF16, 26 / 24 us; 8 of 5632 x 2048 over 32, FP32, 82 / 76).
    if (tile == kTile256 ? rows <= kFBK * groups : grad_tiles(groups, m, n, tile) >= kMaxBlocks) continue;
    const float ti = tile_time(tile, groups * (cdiv(m, bm) * bm), n, cdiv(rows, groups), kMNContig, kMNContig, device_cus(),
                               false, kEpiF32);
    if (t == 0.0f || ti < t) {
      best = tile;
      t = ti;
    }
  }
  return best;
}

int check_sizes(int64_t groups, int64_t rows, int64_t n, int64_t k) {
  if (groups < 1 || groups > kMaxGroups) return set_error(kInvalid, "1 to %ld groups, not %ld", (long)kMaxGroups, (long)groups);
  if (rows < 0 || n < 1 || k < 1 || rows > kMaxRows || !fits_i32(n) || !fits_i32(k))
    return set_error(kInvalid, "invalid grouped product shape (%ld rows, %ld x %ld)", (long)rows, (long)n, (long)k);
  return kOk;
}
// The width of the weights' rows.
int check_width(int64_t width) {
  return width % 8 == 0 ? kOk : set_error(kInvalid, "grouped products take weight rows of a multiple of 8, not %ld", (long)width);
}
// Rows of whole, aligned 16-byte pieces, 256 of which span less than 2 GiB.
int check_rows(const void* p, int64_t ld, int64_t rows, int64_t cols, const char* what) {
  if (!al(p, 16) || ld % 8 != 0) return set_error(kInvalid, "%s rows must be 16-byte aligned", what);
  if (rows > 1 && ld < cols) return set_error(kInvalid, "%s rows overlap", what);
  return check_out_stride(ld > cols ? ld : cols, 2, what);
}

int check_tiles(int64_t tiles, int64_t most, int64_t rows, int64_t groups, int64_t n, int64_t k) {
  return tiles < most ? kOk
                      : set_error(kInvalid, "too many tiles (%ld rows, %ld groups of %ld x %ld)", (long)rows, (long)groups,
                                  (long)n, (long)k);
}
// What the weight gradient asks of sizes alone: where 256 x 256 tiles are few enough, so are those that are chosen.
int check_grad(int64_t rows, int64_t groups, int64_t n, int64_t k, int elem_bytes) {
  if (int rc = check_out_stride(k, elem_bytes, "dweight")) return rc;
  return check_tiles(grad_tiles(groups, n, k, kTile256), kMaxBlocks, rows, groups, n, k);
}

template <class Cfg, int BMODE, bool CUT = true>
int launch_ring(const GroupedParams& p, int slices, int64_t grid, hipStream_t s) {
  auto run = [&](auto kernel) {
    if (int rc = ensure_lds(reinterpret_cast<const void*>(kernel), Cfg::kLds)) return rc;
    hipLaunchKernelGGL(kernel, dim3((unsigned)cdiv(grid, p.run), slices), dim3(Cfg::NT), Cfg::kLds, s, p);
    return hip_check(hipGetLastError(), "grouped product launch");
  };
  if constexpr (!CUT) return run(&grouped_ring_kernel<Cfg, BMODE, false>);
  if (slices == 1) return run(&grouped_ring_kernel<Cfg, BMODE, false>);
  if (int rc = run(&grouped_ring_kernel<Cfg, BMODE, CUT>)) return rc;
  hipLaunchKernelGGL(grouped_join_kernel, dim3((unsigned)cdiv((int64_t)p.rows * p.N, 2048)), dim3(256), 0, s, p.partial, slices,
                     (long)p.rows, p.N, p.c, p.ldc);
  return hip_check(hipGetLastError(), "grouped product join launch");
}
template <int BMODE>
int launch_whole(GroupedParams p, int64_t grid, hipStream_t s) {
  const void* kern = reinterpret_cast<const void*>(&grouped_fast_kernel<BMODE>);
  static_assert(Piece64::kLds <= kFLdsBytes && Piece128::kLds <= kFLdsBytes && Piece64::NT == kFNT && Piece128::NT == kFNT,
                "pieces run in the workgroup of a 256 x 256 tile");
  if (int rc = ensure_lds(kern, kFLdsBytes)) return rc;
  // (All units, also for fewer tiles: these may go in pieces.)
  const int cus = device_cus();
  p.pieces_most = kPiecesOf256 * cus / 256;
  hipLaunchKernelGGL((grouped_fast_kernel<BMODE>), dim3((unsigned)(grid * 8 < cus ? grid * 8 : cus)), dim3(kFNT), kFLdsBytes, s, p);
  return hip_check(hipGetLastError(), "grouped product launch");
}
template <int BMODE>
int run_tile(const GroupedParams& p, GroupedPlan plan, int64_t grid, hipStream_t s) {
  const int tile = plan.tile, slices = plan.slices;
  switch (tile) {
    case kTile256: return launch_whole<BMODE>(p, grid, s);
    case kTile128x2: return launch_ring<Ring128x2, BMODE, false>(p, 1, grid, s);
    case kTile128x1: return launch_ring<Ring128x1, BMODE>(p, slices, grid, s);
    case kTile64x128: return launch_ring<Ring64x128, BMODE>(p, slices, grid, s);
    case kTile64: return launch_ring<Ring64, BMODE>(p, slices, grid, s);
  }
  if constexpr (BMODE == kKContig) {
    // (Several tiles a workgroup are of 32 columns: 16 are for idle units, or for reductions above 256.)
    const auto kernel = tile == kTileFew16 ? grouped_few_kernel<16, false>
                        : p.run > 1        ? grouped_few_kernel<32, true>
                                           : grouped_few_kernel<32, false>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)cdiv(grid, p.run)), dim3(256), 0, s, p);
    return hip_check(hipGetLastError(), "grouped product launch");
  }
  return set_error(kInvalid, "no grouped tile %d", tile);
}

template <class Cfg>
int launch_grad_ring(const GroupedGradParams& p, bool f32, int64_t grid, hipStream_t s) {
  auto run = [&](auto kernel) {
    if (int rc = ensure_lds(reinterpret_cast<const void*>(kernel), Cfg::kLds)) return rc;
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(Cfg::NT), Cfg::kLds, s, p);
    return hip_check(hipGetLastError(), "grouped weight gradient launch");
  };
  return f32 ? run(&grouped_grad_ring_kernel<Cfg, true>) : run(&grouped_grad_ring_kernel<Cfg, false>);
}

}  // namespace

extern "C" int ws_grouped_tile(int64_t rows, int64_t groups, int64_t n, int64_t k, int form) {
  if (rows < 1 || check_sizes(groups, rows, n, k)) return -1;
  if (form == WS_GROUPED_GRAD) return grad_tiles(groups, n, k, kTile256) < kMaxBlocks ? pick_grad(rows, groups, n, k) : -1;
  if ((form != WS_GROUPED_NT && form != WS_GROUPED_NN) || grid_tiles(rows, groups, n, kTile256) >= kMaxTiles) return -1;
  return pick_grouped(rows, groups, n, k, form == WS_GROUPED_NT ? kKContig : kMNContig).tile;
}

extern "C" int ws_grouped_backward_check(int64_t rows, int64_t groups, int64_t n, int64_t k, int dx, int dweight,
                                         int dweight_f32) {
  if (int rc = check_sizes(groups, rows, n, k)) return rc;
  const int64_t wide_n = up8(n), wide_k = up8(k);
  if (int rc = check_out_stride(wide_n > wide_k ? wide_n : wide_k, 2, "gradient")) return rc;
  if (dx && rows > 0) {
    if (int rc = check_tiles(grid_tiles(rows, groups, wide_k, kTile256), kMaxTiles, rows, groups, n, k)) return rc;
  }
  return dweight ? check_grad(rows, groups, n, wide_k, dweight_f32 ? 4 : 2) : kOk;
}

extern "C" int64_t ws_grouped_workspace_floats(int64_t rows, int64_t groups, int64_t n, int64_t k, int form) {
  if (rows < 1 || check_sizes(groups, rows, n, k) || (form != WS_GROUPED_NT && form != WS_GROUPED_NN)) return 0;
  const int slices = pick_grouped(rows, groups, n, k, form == WS_GROUPED_NT ? kKContig : kMNContig).slices;
  return slices > 1 ? slices * rows * up8(n) : 0;
}

extern "C" int ws_grouped_mm(const void* x, int64_t ldx, const void* weight, int64_t ld_weight, int64_t group_stride,
                             int form, const int64_t* offsets, int64_t groups, int64_t rows, int64_t n, int64_t k,
                             void* y, int64_t ldy, float* workspace, void* stream) {
  if (form != WS_GROUPED_NT && form != WS_GROUPED_NN) return set_error(kInvalid, "unknown form %d", form);
  if (int rc = check_sizes(groups, rows, n, k)) return rc;
  if (rows == 0) return kOk;
  if (!x || !weight || !offsets || !y) return set_error(kInvalid, "null pointer");
  const bool nt = form == WS_GROUPED_NT;
  const GroupedPlan plan = pick_grouped(rows, groups, n, k, nt ? kKContig : kMNContig);
  const int tile = plan.tile;
  const int64_t wide = up8(n);
  if (tile == kTileFew || tile == kTileFew16) {  // operands of any alignment and width
    if (rows > 1 && ldx < k) return set_error(kInvalid, "x rows overlap");
    if (ld_weight < k) return set_error(kInvalid, "weight rows overlap");
    if (!al(x, 2) || !al(weight, 2) || group_stride < 0) return set_error(kInvalid, "operands must be aligned to their elements");
  } else {
    if (int rc = check_width(nt ? k : n)) return rc;
    if (int rc = check_rows(x, ldx, rows, up8(k), "x")) return rc;
    if (int rc = check_rows(weight, ld_weight, 2, nt ? k : n, "weight")) return rc;
    if (group_stride % 8 != 0 || group_stride < 0) return set_error(kInvalid, "weights must be 16-byte aligned");
  }
  if (int rc = check_rows(y, ldy, rows, wide, "y")) return rc;
  if (plan.slices > 1 && !workspace) return set_error(kInvalid, "null pointer");
  if (!al(workspace, 16)) return set_error(kInvalid, "the workspace must be 16-byte aligned");
  GroupedParams p{};
  p.per = cdiv(cdiv(k, kFBK), plan.slices);
  p.partial = workspace;
  p.a = OperandDesc{static_cast<const unsigned short*>(x), ldx, 1};
  p.b = OperandDesc{static_cast<const unsigned short*>(weight), nt ? ld_weight : 1, nt ? 1 : ld_weight};
  p.b_group = group_stride;
  p.offsets = reinterpret_cast<const long*>(offsets);
  p.groups = (int)groups;
  p.rows = (int)rows;
  p.N = (int)wide;
  p.K = (int)k;
  p.b_rows = (int)n;
  p.tiles_n = cdiv(wide, tile_cols(tile));
  p.c = static_cast<unsigned short*>(y);
  p.ldc = ldy;
  if (int rc = check_tiles(grid_tiles(rows, groups, n, kTile256), kMaxTiles, rows, groups, n, k)) return rc;
  const int64_t grid = grid_tiles(rows, groups, n, tile);
  p.most = (int)grid;
  p.chunk = cdiv(groups, 64);
  p.run = tile == kTile256 || tile == kTileFew16 || plan.slices > 1 ? 1 : tiles_of_run(grid, k);
  hipStream_t s = static_cast<hipStream_t>(stream);
  return nt ? run_tile<kKContig>(p, plan, grid, s) : run_tile<kMNContig>(p, plan, grid, s);
}

extern "C" int ws_grouped_weight_grad(const void* dy, int64_t ld_dy, const void* x, int64_t ldx, const int64_t* offsets,
                                      int64_t groups, int64_t rows, int64_t n, int64_t k, void* dweight,
                                      int dweight_f32, void* stream) {
  if (int rc = check_sizes(groups, rows, n, k)) return rc;
  if (int rc = check_width(k)) return rc;
  if (!dweight || !offsets || (rows > 0 && (!dy || !x))) return set_error(kInvalid, "null pointer");
  if (int rc = check_rows(dy, ld_dy, rows, up8(n), "dy")) return rc;
  if (int rc = check_rows(x, ldx, rows, k, "x")) return rc;
  if (!al(dweight, 16)) return set_error(kInvalid, "the weight gradient must be 16-byte aligned");
  if (int rc = check_grad(rows, groups, n, k, dweight_f32 ? 4 : 2)) return rc;
  const int tile = pick_grad(rows, groups, n, k);
  GroupedGradParams p{};
  p.a = static_cast<const unsigned short*>(dy);
  p.lda = ld_dy;
  p.b = static_cast<const unsigned short*>(x);
  p.ldb = ldx;
  p.offsets = reinterpret_cast<const long*>(offsets);
  p.groups = (int)groups;
  p.rows = (int)rows;
  p.M = (int)n;
  p.N = (int)k;
  p.tiles_m = cdiv(n, tile_rows(tile));
  p.tiles_n = cdiv(k, tile_cols(tile));
  p.g = dweight;
  const int64_t grid = grad_tiles(groups, n, k, tile);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool f32 = dweight_f32 != 0;
  switch (tile) {
    case kTile128x2: return launch_grad_ring<Ring128x2>(p, f32, grid, s);
    case kTile128x1: return launch_grad_ring<Ring128x1>(p, f32, grid, s);
    case kTile64x128: return launch_grad_ring<Ring64x128>(p, f32, grid, s);
    case kTile64: return launch_grad_ring<Ring64>(p, f32, grid, s);
  }
  auto run = [&](auto kernel) {
    if (int rc = ensure_lds(reinterpret_cast<const void*>(kernel), kFLdsBytes)) return rc;
    const int cus = device_cus();
    hipLaunchKernelGGL(kernel, dim3((unsigned)(grid < cus ? grid : cus)), dim3(kFNT), kFLdsBytes, s, p);
    return hip_check(hipGetLastError(), "grouped weight gradient launch");
  };
  return f32 ? run(&grouped_grad_fast_kernel<true>) : run(&grouped_grad_fast_kernel<false>);
}

extern "C" int ws_copy_rows(const void* in, int in_f32, int64_t group_in, int64_t ld_in, int64_t rows_in, int64_t cols_in,
                            void* out, int out_f32, int64_t group_out, int64_t ld_out, int64_t rows_out, int64_t cols_out,
                            int64_t groups, void* stream) {
  if (groups < 0 || rows_in < 0 || rows_out < 0 || cols_in < 0 || cols_out < 0 || !fits_i32(rows_in) ||
      !fits_i32(rows_out) || !fits_i32(cols_in + 512) || !fits_i32(cols_out + 512) || groups > 1L << 24)
    return set_error(kInvalid, "invalid sizes of copied rows");
  if (groups == 0 || rows_out == 0 || cols_out == 0) return kOk;
  if (!out || (!in && rows_in > 0 && cols_in > 0)) return set_error(kInvalid, "null pointer");
  if (!in_f32 && out_f32) return set_error(kInvalid, "rows are copied in their type or rounded to BF16");
  if ((rows_out > 1 && ld_out < cols_out) || (groups > 1 && group_out < ld_out * (rows_out - 1) + cols_out))
    return set_error(kInvalid, "rows overlap");
  CopyRowsParams p{in, group_in, ld_in, (int)rows_in, (int)cols_in, out, group_out, ld_out, (int)rows_out, (int)cols_out, groups * rows_out};
  const int64_t blocks = p.rows < 4 * kMaxBlocks ? cdiv(p.rows, 4) : kMaxBlocks;
  auto run = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), 0, static_cast<hipStream_t>(stream), p);
    return hip_check(hipGetLastError(), "row copy launch");
  };
  return in_f32 ? (out_f32 ? run(&copy_rows_kernel<true, true>) : run(&copy_rows_kernel<true, false>))
                : run(&copy_rows_kernel<false, false>);
}
