// C ABI: token scores (log probability, entropy, likeliest tokens) and their gradients, from
// logits and from the LM head's operands.
#include "../../include/warpstate_hip.h"
#include "lm_head.h"
#include "score_epilogue.h"
#include "scores.h"

using namespace ws;

namespace {

constexpr int kLargeEpt = 32, kSmallEpt = 8;
// 1 / temperature: a normal FP32 number, and finite times log2 e.
bool good_inv_t(float inv_t) { return inv_t >= 0x1p-126f && inv_t <= 2.3e38f; }

// Logits per thread: 8 (parts of 2048) while 32 would leave most compute units without a
// workgroup, as long as 64 parts cover the row.
int score_ept(long rows, long vocab) {
  const long parts = cdiv(vocab, 256 * kLargeEpt);
  return rows * parts < 2 * device_cus() && cdiv(vocab, 256 * kSmallEpt) <= kMaxScoreParts ? kSmallEpt
                                                                                           : kLargeEpt;
}
int score_parts(long rows, long vocab) { return cdiv(vocab, 256 * score_ept(rows, vocab)); }

template <bool F32, int EPT>
void launch_rows(const ScoreParams& p, hipStream_t s) {
  const dim3 grid((unsigned)((long)p.rows * p.parts));
  if (p.top_k > 0) hipLaunchKernelGGL((score_rows_kernel<F32, EPT, true>), grid, dim3(256), 0, s, p);
  else hipLaunchKernelGGL((score_rows_kernel<F32, EPT, false>), grid, dim3(256), 0, s, p);
}
// A launch has fewer than 2^32 threads, so more workgroups of 256 go in several launches.
constexpr long kMaxLaunchBlocks = (1L << 24) - 1;
long launch_row_count(long blocks_per_row) { return kMaxLaunchBlocks / blocks_per_row; }

// The rows from `first` on, at most `count` of them.
ScoreParams some_rows(ScoreParams p, long first, long count, bool f32) {
  p.rows = (int)(p.rows - first < count ? p.rows - first : count);
  p.logits = static_cast<const char*>(p.logits) + first * p.ld * (f32 ? 4 : 2);
  p.tokens += first;
  p.out.lse += first;
  p.out.entropy += first;
  if (p.out.logprob) p.out.logprob += first;
  if (p.top_k) {
    p.top_logprobs += first * p.top_k;
    p.top_ids += first * p.top_k;
  }
  if (p.stats) p.stats += first * p.parts;
  if (p.keys) p.keys += first * p.parts * p.top_k;
  return p;
}

template <bool F32>
int run_scores(const ScoreParams& all, int ept, hipStream_t s) {
  const long count = launch_row_count(all.parts);
  if (all.rows > count) {
    for (long first = 0; first < all.rows; first += count)
      if (int rc = run_scores<F32>(some_rows(all, first, count, F32), ept, s)) return rc;
    return kOk;
  }
  const ScoreParams& p = all;
  if (ept == kSmallEpt) launch_rows<F32, kSmallEpt>(p, s);
  else launch_rows<F32, kLargeEpt>(p, s);
  if (int rc = hip_check(hipGetLastError(), "token score launch")) return rc;
  if (p.parts == 1) return kOk;
  int lanes = 2, threads = 64, per_key = 1;
  while (lanes < p.parts) lanes *= 2;
  const int total = p.parts * p.top_k;
  // Enough rows fill the card with a thread per key.
  if (p.rows < device_cus())
    while (per_key * kScoreJoinAt < p.parts && 2 * per_key * total <= kScoreJoinThreads) per_key *= 2;
  while (threads < total * per_key && threads < (per_key > 1 ? kScoreJoinThreads : 256)) threads *= 2;
  const int block = threads > 256 ? threads : 256, rows = block / threads;
  hipLaunchKernelGGL((score_join_kernel<F32>), dim3(cdiv(p.rows, rows)), dim3(block), rows * total * 8, s, p, threads,
                     lanes, per_key);
  return hip_check(hipGetLastError(), "token score join launch");
}

int check_logits(const void* logits, long ld, int f32, long rows, long vocab, const void* tokens, float inv_t) {
  if (!logits || !tokens) return set_error(kInvalid, "null operand pointer");
  if (rows < 1 || vocab < 1 || !fits_i32(rows) || vocab > (long)kMaxScoreParts * 256 * kLargeEpt)
    return set_error(kInvalid, "token scores take at least one row and 1 to %ld logits a row",
                     (long)kMaxScoreParts * 256 * kLargeEpt);
  if (ld < vocab) return set_error(kInvalid, "leading dimension < vocab");
  if (f32 != 0 && f32 != 1) return set_error(kInvalid, "unknown logit type %d", f32);
  if (!good_inv_t(inv_t)) return set_error(kInvalid, "the temperature must lie between 4.4e-39 and 8.5e37");
  if (!fits_i32(rows * cdiv(vocab, 2048))) return set_error(kInvalid, "too many logits for one launch");
  return kOk;
}

}  // namespace

extern "C" int64_t ws_token_scores_workspace_bytes(int64_t rows, int64_t vocab, int64_t top_k) {
  if (rows < 1 || vocab < 1 || top_k < 0) return 0;
  const long parts = score_parts(rows, vocab);
  return parts == 1 ? 0 : rows * parts * (16 + 8 * top_k);
}

extern "C" int ws_token_scores(const void* logits, int64_t ld, int f32, const int64_t* tokens,
                               int64_t rows, int64_t vocab, float inv_temperature, int64_t top_k,
                               void* workspace, float* lse, float* logprob, float* entropy,
                               float* top_logprobs, int64_t* top_ids, void* stream) {
  if (int rc = check_logits(logits, ld, f32, rows, vocab, tokens, inv_temperature)) return rc;
  if (!lse || !logprob || !entropy) return set_error(kInvalid, "null output pointer");
  if (top_k < 0 || top_k > kMaxTopK || top_k > vocab)
    return set_error(kInvalid, "top_k must lie in [0, min(%d, vocab)]", kMaxTopK);
  if (top_k && (!top_logprobs || !top_ids)) return set_error(kInvalid, "null output pointer");
  const int ept = score_ept(rows, vocab);
  ScoreParams p{};
  p.logits = logits;
  p.ld = ld;
  p.rows = (int)rows; p.vocab = (int)vocab; p.top_k = (int)top_k;
  p.parts = score_parts(rows, vocab);
  p.inv_t = inv_temperature;
  p.scale = inv_temperature * kLog2e;
  p.tokens = reinterpret_cast<const long*>(tokens);
  p.out = ScoreOut{lse, logprob, entropy};
  p.top_logprobs = top_logprobs;
  p.top_ids = reinterpret_cast<long*>(top_ids);
  if (p.parts > 1) {
    if (!workspace || !al(workspace, 16)) return set_error(kInvalid, "the workspace must be 16-byte aligned");
    p.stats = static_cast<f32x4_t*>(workspace);
    p.keys = reinterpret_cast<unsigned long*>(p.stats + rows * p.parts);
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  return f32 ? run_scores<true>(p, ept, s) : run_scores<false>(p, ept, s);
}

extern "C" int ws_token_scores_backward(const void* logits, int64_t ld, int f32, const int64_t* tokens,
                                        int64_t rows, int64_t vocab, float inv_temperature,
                                        const float* lse, const float* entropy, const float* dlogprob,
                                        const float* dentropy, void* dlogits, int64_t ld_out, void* stream) {
  if (int rc = check_logits(logits, ld, f32, rows, vocab, tokens, inv_temperature)) return rc;
  if (!lse || !entropy || !dlogits) return set_error(kInvalid, "null pointer");
  if (ld_out < vocab) return set_error(kInvalid, "output leading dimension < vocab");
  ScoreParams p{};
  p.logits = logits;
  p.ld = ld;
  p.rows = (int)rows; p.vocab = (int)vocab;
  p.inv_t = inv_temperature;
  p.scale = inv_temperature * kLog2e;
  p.tokens = reinterpret_cast<const long*>(tokens);
  p.out = ScoreOut{const_cast<float*>(lse), nullptr, const_cast<float*>(entropy)};
  const auto* x = static_cast<const char*>(logits);
  const auto* dx = static_cast<const char*>(dlogits);
  const long size = f32 ? 4 : 2, span = ((rows - 1) * ld + vocab) * size, dspan = ((rows - 1) * ld_out + vocab) * size;
  const bool in_place = x < dx + dspan && dx < x + span;
  const int segments = in_place ? 1 : cdiv(vocab, 2048);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const long count = launch_row_count(segments);
  for (long first = 0; first < rows; first += count) {
    const ScoreParams q = some_rows(p, first, count, f32);
    const float* g = dlogprob ? dlogprob + first : nullptr;
    const float* h = dentropy ? dentropy + first : nullptr;
    void* out = static_cast<char*>(dlogits) + first * ld_out * size;
    const dim3 grid((unsigned)((long)q.rows * segments));
    if (f32)
      hipLaunchKernelGGL((score_grad_kernel<true>), grid, dim3(256), 0, s, q, g, h, out, (long)ld_out, segments);
    else
      hipLaunchKernelGGL((score_grad_kernel<false>), grid, dim3(256), 0, s, q, g, h, out, (long)ld_out, segments);
  }
  return hip_check(hipGetLastError(), "token score gradient launch");
}

// --- from the LM head's operands ------------------------------------------------------------

namespace {

int check_head(const void* hidden, long ld_hidden, const void* weight, long ld_weight, const void* tokens,
               long rows, long vocab, long d, float inv_t, GemmParams& p) {
  if (!hidden || !weight || !tokens) return set_error(kInvalid, "null operand pointer");
  if (rows < 1 || vocab < 1 || d < 1 || !fits_i32(rows) || !fits_i32(vocab) || !fits_i32(d))
    return set_error(kInvalid, "invalid LM-head sizes rows=%ld vocab=%ld d=%ld", rows, vocab, d);
  // (64 threads a row join its parts, in one launch of fewer than 2^32.)
  if (rows >= 1L << 26) return set_error(kInvalid, "too many rows for one launch");
  if (ld_hidden < d || ld_weight < d) return set_error(kInvalid, "leading dimension < d");
  if (!good_inv_t(inv_t)) return set_error(kInvalid, "the temperature must lie between 4.4e-39 and 8.5e37");
  p = GemmParams{};
  p.a = OperandDesc{static_cast<const unsigned short*>(hidden), ld_hidden, 1};
  p.b = OperandDesc{static_cast<const unsigned short*>(weight), ld_weight, 1};  // B = W^T
  p.M = (int)rows; p.N = (int)vocab; p.K = (int)d;
  p.vec_out = 1;
  p.logit_scale = inv_t;
  if (operand_mode(p.a, rows, d, 256) != kKContig || operand_mode(p.b, vocab, d, 256) != kKContig ||
      !fast_ok(p, kKContig, kKContig, false))
    return set_error(kInvalid, "hidden and weight need 16-byte aligned rows of a multiple of 8 elements");
  return kOk;
}
// The logits product's macro-tile: with few rows most compute units would idle on 256 x 256,
// where reading the head weight is what bounds it (us, 256 x 256 / the choice: 64 x 2048 over
// 32768 46 / 30, of which the weight takes 28 at the card's copy rate; 512 x 1280 over 10883
// 36 / 27; 1000 rows over 32768 108 / 107).
int head_tile(long rows, long vocab, long d) {
  const int tile = pick_tile(rows, vocab, d, kKContig, kKContig, false, kEpiStore);
  return tile == kTile256 || tile == kTile128x2 ? tile : kTile64x128;
}
// One partial per column block of a wave: 128 columns, or 64 of the smaller tiles.
long head_parts(int tile, long vocab) { return (long)cdiv(vocab, tile == kTile256 ? 256 : 128) * 2; }

template <class Epi>
int run_head(const GemmParams& p, int tile, hipStream_t s) {
  switch (tile) {
    case kTile256: return run_fast<kKContig, kKContig, false, Epi>(p, kFusedCfg, s);
    case kTile128x2: return run_ring<Ring128x2, kKContig, kKContig, false, Epi>(p, 1, s);
    default: return run_ring<Ring64x128, kKContig, kKContig, false, Epi>(p, 1, s);
  }
}

}  // namespace

extern "C" int64_t ws_linear_token_scores_workspace_floats(int64_t rows, int64_t vocab, int64_t d) {
  if (rows < 1 || vocab < 1 || d < 1) return 0;
  return rows * (3 * head_parts(head_tile(rows, vocab, d), vocab) + 1);
}

extern "C" int ws_linear_token_scores(const void* hidden, int64_t ld_hidden, const void* weight,
                                      int64_t ld_weight, const int64_t* tokens, int64_t rows,
                                      int64_t vocab, int64_t d, float inv_temperature, float* workspace,
                                      float* lse, float* logprob, float* entropy, void* stream) {
  GemmParams p;
  if (int rc = check_head(hidden, ld_hidden, weight, ld_weight, tokens, rows, vocab, d, inv_temperature, p))
    return rc;
  if (!workspace || !lse || !logprob || !entropy) return set_error(kInvalid, "null output pointer");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int tile = head_tile(rows, vocab, d);
  const long parts = head_parts(tile, vocab);
  p.targets = reinterpret_cast<const long*>(tokens);
  p.part_max = workspace;
  p.part_sum = p.part_max + rows * parts;
  p.part_wsum = p.part_sum + rows * parts;
  p.tgt_logit = p.part_wsum + rows * parts;
  p.parts_per_row = (int)parts;
  if (int rc = run_head<FEpiScoreStats>(p, tile, s)) return rc;
  hipLaunchKernelGGL(score_combine_kernel, dim3(cdiv(rows, 4)), dim3(256), 0, s, p.part_max, p.part_sum,
                     p.part_wsum, p.parts_per_row, p.tgt_logit, p.targets, ScoreOut{lse, logprob, entropy},
                     (int)rows, (int)vocab, inv_temperature);
  return hip_check(hipGetLastError(), "token score combine launch");
}

// Workspace of the backward: [rows x 4 FP32 coefficients][chunk x row BF16 logit gradients]
// [splits x chunk x d FP32 dHidden partials], each part 256-byte aligned.
extern "C" int64_t ws_linear_token_scores_backward_workspace_bytes(int64_t rows, int64_t vocab, int64_t d,
                                                                   int64_t chunk_rows) {
  if (rows < 1 || vocab < 1 || d < 1 || chunk_rows < 1) return 0;
  const long chunk = chunk_rows < rows ? chunk_rows : rows;
  const int splits = ce_dh_splits(chunk, d, vocab);
  return round256(rows * 16) + round256(chunk * ce_row(vocab) * 2) +
         (splits > 1 ? round256((long)splits * chunk * d * 4) : 0);
}

extern "C" int ws_linear_token_scores_backward(const void* hidden, int64_t ld_hidden, const void* weight,
                                               int64_t ld_weight, const void* weight_t,
                                               const int64_t* tokens, const float* lse,
                                               const float* entropy, const float* dlogprob,
                                               const float* dentropy, int64_t rows, int64_t vocab, int64_t d,
                                               float inv_temperature, void* workspace, int64_t chunk_rows,
                                               void* dhidden, int64_t ld_dhidden, void* dweight,
                                               int64_t ld_dweight, int dweight_bf16, void* stream) {
  GemmParams p;
  if (int rc = check_head(hidden, ld_hidden, weight, ld_weight, tokens, rows, vocab, d, inv_temperature, p))
    return rc;
  if (!lse || !entropy || !workspace || (!dhidden && !dweight)) return set_error(kInvalid, "null pointer");
  if (!al(workspace, 256)) return set_error(kInvalid, "workspace must be 256-byte aligned");
  const long chunk = chunk_rows < rows ? chunk_rows : rows;
  const long ldg = ce_row(vocab);
  if (chunk_rows < 1 || !fits_i32(chunk * ldg)) return set_error(kInvalid, "bad chunk_rows");
  if (int rc = check_out_stride(ldg, 2, "logit-gradient chunk")) return rc;
  if (dhidden) {
    if (ld_dhidden < d) return set_error(kInvalid, "dhidden leading dimension < d");
    if (int rc = check_out_stride(ld_dhidden, 2, "dhidden")) return rc;
    if (int rc = check_out_stride(d, 4, "dhidden partial")) return rc;
  }
  if (dweight) {
    if (ld_dweight < d) return set_error(kInvalid, "dweight leading dimension < d");
    if (int rc = check_out_stride(ld_dweight, 4, "dweight")) return rc;
    if (dweight_bf16 && (ld_dweight != d || chunk < rows))
      return set_error(kInvalid, "a BF16 weight gradient is contiguous and of one chunk");
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto* base = static_cast<unsigned char*>(workspace);
  auto* coef = reinterpret_cast<f32x4_t*>(base);
  auto* gl = reinterpret_cast<unsigned short*>(base + round256(rows * 16));
  auto* partials = reinterpret_cast<float*>(base + round256(rows * 16) + round256(chunk * ldg * 2));
  const int splits = ce_dh_splits(chunk, d, vocab);
  hipLaunchKernelGGL(score_coef_kernel, dim3(cdiv(rows, 256)), dim3(256), 0, s,
                     reinterpret_cast<const long*>(tokens), lse, entropy, dlogprob, dentropy, inv_temperature,
                     (int)rows, (int)vocab, coef);
  if (int rc = hip_check(hipGetLastError(), "token score coefficient launch")) return rc;
  for (long start = 0; start < rows; start += chunk) {
    const CeChunk c{static_cast<const unsigned short*>(hidden) + start * ld_hidden, ld_hidden, start,
                    rows - start < chunk ? rows - start : chunk, ldg};
    GemmParams g = p;
    g.a.ptr = c.hidden;
    g.M = (int)c.r;
    g.c = gl;
    g.ldc = ldg;
    g.targets = reinterpret_cast<const long*>(tokens) + start;
    g.row_coef = reinterpret_cast<const float*>(coef + start);
    if (int rc = run_head<FEpiScoreGrad>(g, head_tile(c.r, vocab, d), s)) return rc;
    if (dweight && dweight_bf16) {
      if (int rc = ws_mm(gl, 1, ldg, c.hidden, ld_hidden, 1, dweight, vocab, d, c.r, 1, 0, stream)) return rc;
    } else if (dweight) {
      if (int rc = ce_chunk_weight_grad(c, gl, vocab, d, static_cast<float*>(dweight), ld_dweight, start == 0,
                                        nullptr, s, false))
        return rc;
    }
    if (dhidden) {
      if (int rc = ce_chunk_dhidden(c, gl, weight, ld_weight, weight_t, vocab, d, splits, chunk, partials,
                                    static_cast<unsigned short*>(dhidden) + start * ld_dhidden, ld_dhidden,
                                    nullptr, s))
        return rc;
    }
  }
  return kOk;
}
