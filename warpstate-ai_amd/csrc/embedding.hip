// C ABI: embedding lookup and the table's gradient.
#include "../../include/warpstate_hip.h"
#include "embedding.h"
#include "launch.h"

using namespace ws;

namespace {

// The sort reads every token for each 512 of the vocabulary: 0.3 s at these limits.
constexpr int64_t kMaxTokens = 1L << 24, kMaxVocab = 1L << 22, kMaxWidth = 1L << 20;

int check_table(int64_t rows, int64_t vocab, int64_t d, int64_t ld) {
  if (rows < 0 || vocab < 1 || d < 1 || rows > kMaxTokens || vocab > kMaxVocab || d > kMaxWidth)
    return set_error(kInvalid, "invalid embedding shape (%ld tokens, %ld x %ld)", (long)rows, (long)vocab, (long)d);
  if (vocab > 1 && ld < d) return set_error(kInvalid, "rows overlap");
  return kOk;
}
// Positions of one piece of a token that occurs more often: 32, or as many as leave 1024 pieces.
int64_t piece_rows(int64_t rows) { return rows <= 32 * 1024 ? 32 : (rows + 1023) / 1024; }

struct GradLayout {
  int64_t piece, pieces, start, perm, partial, bytes, ld_partial;
};
GradLayout grad_layout(int64_t rows, int64_t vocab, int64_t d) {
  if (rows <= kFewTokens) return GradLayout{};
  auto up = [](int64_t n) { return (n + 255) / 256 * 256; };
  GradLayout l;
  l.piece = piece_rows(rows);
  l.pieces = rows > l.piece ? (rows + l.piece - 1) / l.piece : 0;  // otherwise no token occurs more often
  l.ld_partial = (d + 7) / 8 * 8;
  l.start = 0;
  l.perm = up(4 * (vocab + 1));
  l.partial = l.perm + up(4 * rows);
  l.bytes = l.partial + up(8 * l.pieces * l.ld_partial);
  return l;
}

// A gradient that the memory-side cache does not hold beside its input goes around it: 16384 rows into
// 32768 x 2048 FP32 (268 MB), all kernels, 94 -> 70 us; BF16 (134 MB) 65 -> 67.
bool past_caches(int64_t bytes) { return bytes > 256L << 20; }

// (Through the caches at any size: few rows of dy are there to be kept, and 64 tokens into 32768 x 2048 FP32
// measure 48 us either way.)
template <bool GF32, int OUT>
int launch_few(const EmbedGradParams& p, bool whole, hipStream_t s) {
  const dim3 grid((unsigned)cdiv(cdiv(p.vocab, p.group), 4)), block(256);
  if (whole) hipLaunchKernelGGL((embed_few_kernel<GF32, OUT, true>), grid, block, 0, s, p);
  else hipLaunchKernelGGL((embed_few_kernel<GF32, OUT, false>), grid, block, 0, s, p);
  return hip_check(hipGetLastError(), "embedding gradient launch");
}

template <bool GF32, int OUT>
int launch_grad(const EmbedGradParams& p, int64_t rows, bool whole, hipStream_t s) {
  const dim3 grid((unsigned)cdiv(p.pieces + cdiv(p.vocab, p.group), 4)), block(256);
  const bool nt = OUT != kEmbedAdd && past_caches(p.d * ((int64_t)p.vocab * (OUT == kEmbedBF16 ? 2 : 4) + rows * (GF32 ? 4 : 2)));
  auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, s, p); };
  if constexpr (OUT != kEmbedAdd) {
    if (whole && nt) run(&embed_grad_kernel<GF32, OUT, true, true>);
  }
  if (whole && !nt) run(&embed_grad_kernel<GF32, OUT, true, false>);
  if (!whole) run(&embed_grad_kernel<GF32, OUT, false, false>);
  if (int rc = hip_check(hipGetLastError(), "embedding gradient launch")) return rc;
  if (p.pieces == 0) return kOk;
  const dim3 join(p.pieces, cdiv(p.d, OUT == kEmbedBF16 ? 512 : 256));
  if (whole) hipLaunchKernelGGL((embed_join_kernel<OUT, true>), join, block, 0, s, p);
  else hipLaunchKernelGGL((embed_join_kernel<OUT, false>), join, block, 0, s, p);
  return hip_check(hipGetLastError(), "embedding gradient join launch");
}

}  // namespace

extern "C" int ws_embedding(const void* table, int64_t ld_table, int table_f32, const int64_t* tokens, int64_t rows,
                            int64_t vocab, int64_t d, float scale, void* y, int y_f32, void* stream) {
  if (int rc = check_table(rows, vocab, d, ld_table)) return rc;
  if (rows == 0) return kOk;
  if (!table || !tokens || !y) return set_error(kInvalid, "null pointer");
  const bool whole = d % 8 == 0;
  auto run = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(cdiv(rows, 4)), dim3(256), 0, static_cast<hipStream_t>(stream), table,
                       (long)ld_table, reinterpret_cast<const long*>(tokens), (int)rows, (int)vocab, (int)d, scale, y);
    return hip_check(hipGetLastError(), "embedding launch");
  };
  if (table_f32)
    return y_f32 ? (whole ? run(&embed_lookup_kernel<true, true, true>) : run(&embed_lookup_kernel<true, true, false>))
                 : (whole ? run(&embed_lookup_kernel<true, false, true>) : run(&embed_lookup_kernel<true, false, false>));
  return y_f32 ? (whole ? run(&embed_lookup_kernel<false, true, true>) : run(&embed_lookup_kernel<false, true, false>))
               : (whole ? run(&embed_lookup_kernel<false, false, true>) : run(&embed_lookup_kernel<false, false, false>));
}

extern "C" int64_t ws_embedding_backward_workspace_bytes(int64_t rows, int64_t vocab, int64_t d) {
  if (rows < 0 || vocab < 1 || d < 1 || rows > kMaxTokens || vocab > kMaxVocab || d > kMaxWidth) return 0;
  return grad_layout(rows, vocab, d).bytes;
}

extern "C" int ws_embedding_backward(const void* dy, int64_t ld_dy, int dy_f32, const int64_t* tokens, int64_t rows,
                                     int64_t vocab, int64_t d, float scale, void* dtable, int64_t ld_dtable,
                                     int mode, void* workspace, void* stream) {
  if (int rc = check_table(rows, vocab, d, ld_dtable)) return rc;
  if (mode < WS_EMBED_WRITE_BF16 || mode > WS_EMBED_ADD_F32) return set_error(kInvalid, "unknown gradient mode %d", mode);
  const bool few = rows <= kFewTokens;
  if (!dtable || (!workspace && !few) || (rows > 0 && (!dy || !tokens))) return set_error(kInvalid, "null pointer");
  if (rows > 1 && ld_dy < d) return set_error(kInvalid, "rows overlap");
  if (!al(workspace, 16)) return set_error(kInvalid, "the workspace must be 16-byte aligned");
  const GradLayout l = grad_layout(rows, vocab, d);
  char* const work = static_cast<char*>(workspace);
  EmbedGradParams p{};
  p.dy = dy;
  p.ld_dy = ld_dy;
  p.tokens = reinterpret_cast<const long*>(tokens);
  p.rows = (int)rows;
  p.start = reinterpret_cast<int*>(work + l.start);
  p.perm = reinterpret_cast<int*>(work + l.perm);
  p.vocab = (int)vocab;
  p.d = (int)d;
  // A row of the table for each wave, so that frequent tokens next to each other do not wait for one another;
  // two, or four, where most rows are empty and their waves take longer than up to 4 KB of zeros (us, all kernels,
  // 1 / 2 / 4 rows a wave, tokens of a Zipf distribution in any order and, in brackets, with the frequent ones
  // adjacent: 16384 into 32768 x 2048 FP32 65 / 68 / 68 (99 / 99 / 113); 7000 into 32768 x 1280 BF16 55 / 49 / 42
  // (60 / 67 / 81); 2000 into 32768 x 2048 FP32 58 / 62 / 60; 100 into 32768 x 1280 BF16 29 / 23 / 21).
  const int64_t row_bytes = d * (mode == WS_EMBED_WRITE_BF16 ? 2 : 4);
  p.group = 64 * rows < vocab ? 4 : 4 * rows < vocab && row_bytes <= 4096 ? 2 : 1;
  p.scale = scale;
  p.out = dtable;
  p.ld_out = ld_dtable;
  p.piece = (int)l.piece;
  p.pieces = (int)l.pieces;
  p.partial = reinterpret_cast<float*>(work + l.partial);
  p.ld_partial = l.ld_partial;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool whole = d % 8 == 0;
#define WS_GRAD(RUN_, ...)                                                                                       \
  (dy_f32 ? (mode == WS_EMBED_WRITE_BF16  ? RUN_<true, kEmbedBF16>(__VA_ARGS__)                                  \
             : mode == WS_EMBED_WRITE_F32 ? RUN_<true, kEmbedF32>(__VA_ARGS__)                                   \
                                          : RUN_<true, kEmbedAdd>(__VA_ARGS__))                                  \
          : (mode == WS_EMBED_WRITE_BF16  ? RUN_<false, kEmbedBF16>(__VA_ARGS__)                                 \
             : mode == WS_EMBED_WRITE_F32 ? RUN_<false, kEmbedF32>(__VA_ARGS__)                                  \
                                          : RUN_<false, kEmbedAdd>(__VA_ARGS__)))
  if (few) return WS_GRAD(launch_few, p, whole, s);
  // A workgroup per compute unit, more where their ranges would pass the counters' space.
  int64_t range = cdiv(vocab, device_cus());
  if (range > kSortRange) range = kSortRange;
  hipLaunchKernelGGL(embed_sort_kernel, dim3(cdiv(vocab, range)), dim3(64 * kSortWaves), 0, s, p.tokens, (int)rows,
                     (int)vocab, (int)range, const_cast<int*>(p.start), const_cast<int*>(p.perm));
  if (int rc = hip_check(hipGetLastError(), "embedding sort launch")) return rc;
  return WS_GRAD(launch_grad, p, rows, whole, s);
#undef WS_GRAD
}
