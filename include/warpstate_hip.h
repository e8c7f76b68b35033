/*
 * warpstate_hip.h -- C ABI of the MI355X (gfx950) BF16 matmul hot path of WarpState.
 *
 * Every entry point takes raw device pointers, element strides and sizes, plus the
 * hipStream_t to launch on (passed as void*; from Python it is
 * torch.cuda.current_stream().cuda_stream of the calling thread). The library launches
 * work on that stream and returns; it never allocates, frees or synchronises. The caller
 * allocates every output and workspace. Outputs must not alias inputs, except the FP32
 * gradient buffers of ws_mm_accumulate_f32 and ws_mm_accumulate_f32_group (updated in
 * place) and the output of
 * ws_sigmoid_backward_cols (which may be its dout).
 *
 * Return value: 0 on success, 1 for an invalid argument (nothing was launched), 2 for a
 * HIP runtime error. ws_last_error() returns the calling thread's last message.
 *
 * Size limits: sizes are positive 32-bit integers. Kernels address a 256-row output tile
 * with 32-bit offsets from the tile's first row, so 256 rows of every output must span
 * less than 2 GiB (a BF16 row stride below 4,194,303 elements, an FP32 one below
 * 2,097,151); wider outputs are rejected with status 1. Operands past the corresponding
 * bound take a slower loader with 64-bit addresses instead.
 *
 * Numerics: BF16 operands, FP32 accumulation in MFMA, BF16 round-to-nearest-even
 * outputs, at the rounding points of the reference's PyTorch path.
 *
 * `algorithm` (GEMM entry points): 0 = "tiled" (one workgroup per output tile),
 * 1 = "persistent" (one resident workgroup per CU slot striding over tiles),
 * 2 = "persistent_tma" (persistent, with the reference's TMA preconditions checked by the
 * caller). `tile`: 0 = the vector kernels' macro-tile for these sizes (256x256 to 64x64, see
 * ws_gemm_tile; 256x256 with 8 waves for operands that the vector loaders refuse), 1 = the
 * general kernel's 128x128 macro-tile (4 waves).
 *
 * Reference citations are path:line in gtausa197-svg/WarpState-AI.
 */
#ifndef WARPSTATE_HIP_H
#define WARPSTATE_HIP_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Last error message of the calling thread ("" if none). */
const char* ws_last_error(void);

/* Library version string. */
const char* ws_version(void);

/*
 * C[m,n] = bf16(A[m,k] @ B[k,n]), C row-contiguous with leading dimension n.
 * A element (i,j) at a + i*a_s0 + j*a_s1, B element (i,j) at b + i*b_s0 + j*b_s1; any
 * positive strides. Replaces the kernel launches of launch_mm
 * (ops/matmul_kernels.py:167-205): `_matmul_kernel` (:81-108) for "tiled"/"persistent"
 * and `warpstate::persistent_tma_mm` (:135-159) for "persistent_tma".
 */
int ws_mm(const void* a, int64_t a_s0, int64_t a_s1, const void* b, int64_t b_s0, int64_t b_s1,
          void* c, int64_t m, int64_t n, int64_t k, int algorithm, int tile, void* stream);

/*
 * Paired up/gate projection with SwiGLU epilogue: packed[m, 2h] = bf16(A @ B) (up in
 * columns [0,h), gate in [h,2h)), act[m,h] = bf16(r?(silu(gate)) * up), where silu runs
 * on the BF16-rounded gate and is itself rounded iff eager_rounding. Replaces the launch
 * of `_paired_swiglu_mm_kernel` in launch_swiglu_mm (ops/matmul_epilogue.py:86-142).
 */
int ws_swiglu_mm(const void* a, int64_t a_s0, int64_t a_s1, const void* b, int64_t b_s0,
                 int64_t b_s1, void* packed, void* act, int64_t m, int64_t h, int64_t k,
                 int eager_rounding, int algorithm, int tile, void* stream);

/* The macro-tile that ws_mm, ws_swiglu_mm (tile 0), ws_residual_mm, ws_rmsnorm_gate_mm and
 * ws_swiglu_backward_mm run an [m, n] output with reduction k on, for operands that the vector
 * loaders take: 0 = 256 x 256, 1 = 128 x 128 (two workgroups per CU), 2 = 128 x 128 (one),
 * 3 = 64 x 128, 4 = 64 x 64; -1 for invalid sizes. `n` is the packed width 2h of the paired
 * SwiGLU projection and h of the SwiGLU backward. Operands: A [m, k] with k or (token-major)
 * m contiguous, B [k, n] with k or n contiguous. Launches nothing. */
enum WsEpilogue {
  WS_EPI_STORE = 0,
  WS_EPI_RESIDUAL = 1,
  WS_EPI_SIGMOID = 2,
  WS_EPI_SWIGLU = 3,
  WS_EPI_SWIGLU_BACKWARD = 4
};
int ws_gemm_tile(int64_t m, int64_t n, int64_t k, int a_token_major, int b_n_contiguous,
                 int epilogue);

/* The same for one FP32 gradient (ws_mm_accumulate_f32, or ws_mm_store_f32 with `store`) of
 * token-major operands whose caller allows `splits` k-slices; *slices (may be null) receives
 * the slices of a smaller tile, or `splits` for 256 x 256 tiles. Launches nothing. */
int ws_mm_f32_tile(int64_t m, int64_t n, int64_t k, int64_t splits, int store, int* slices);

/* Standalone SwiGLU of a contiguous packed [rows, 2h] BF16 projection; replaces
 * bf16_swiglu (ops/activation_execution.py:58-70). */
int ws_swiglu_forward(const void* packed, void* out, int64_t rows, int64_t h, int eager_rounding,
                      void* stream);

/* SwiGLU backward: out[rows, 2h] = (dUp | dGate) from packed [rows, 2h] and contiguous
 * grad [rows, h]; replaces `_swiglu_backward` (ops/activation_execution.py:73-81). */
int ws_swiglu_backward(const void* packed, const void* grad, void* out, int64_t rows, int64_t h,
                       int eager_rounding, void* stream);

/* BF16 RMSNorm forward of contiguous x [rows, d] with FP32 weight; writes y and the FP32
 * row rsqrt; replaces bf16_rmsnorm (ops/activation_execution.py:161-173). */
int ws_rmsnorm_forward(const void* x, const float* weight, void* y, float* rstd, int64_t rows,
                       int64_t d, float eps, int eager_rounding, void* stream);

/* Floats of the `partial` workspace ws_rmsnorm_backward needs: one partial row of d floats
 * per 8 to 32 rows up to d = 2048, per 4 to 32 rows above, depending on the row count. */
int64_t ws_rmsnorm_backward_partial_floats(int64_t rows, int64_t d);

/* RMSNorm backward: dx [rows, d] BF16 and dweight [d] FP32 from x, weight, rstd and a
 * contiguous grad; replaces `_rms_backward` (ops/activation_execution.py:176-194). Any
 * width d <= 8192 and any buffer alignment (d % 8 == 0 with 16-byte aligned x, grad and dx
 * takes the vector kernel, everything else a generic one with the same arithmetic). */
int ws_rmsnorm_backward(const void* x, const float* weight, const float* rstd, const void* grad,
                        void* dx, float* dweight, float* partial, int64_t rows, int64_t d,
                        int eager_rounding, void* stream);

/* Allocation-free variant of ws_rmsnorm_backward: the same kernels and results, with the
 * weight-gradient partials in a static 4 MiB device array of the library instead of a
 * caller workspace. No counterpart in the reference: it is for callers that cannot
 * allocate (code under HIP graph capture, tight serving loops, harnesses that forbid
 * hipMalloc). It calls no allocator, and none of its row kernels uses runtime-allocated
 * private memory. Limits: d <= 8192 and ws_rmsnorm_backward_partial_floats(rows, d) <=
 * ws_rmsnorm_backward_static_max_partial_floats() (2^20; e.g. 16384 x 2048); larger
 * sizes return an error. Each GPU holds its own copy of the array until the process
 * ends; calls that overlap on one GPU share it and race. */
int ws_rmsnorm_backward_static(const void* x, const float* weight, const float* rstd,
                               const void* grad, void* dx, float* dweight, int64_t rows,
                               int64_t d, int eager_rounding, void* stream);

/* Partial floats the static scratch of ws_rmsnorm_backward_static holds. */
int64_t ws_rmsnorm_backward_static_max_partial_floats(void);

/* out[cols, rows] = transpose(in[rows, cols]) for BF16 (in has row stride ld_in, out is
 * contiguous). Used to give weight-side GEMM operands a contiguous reduction dimension:
 * the input gradient dX = dY @ W (ops/matmul_execution.py:239) then reads W^T rows.
 * No reference counterpart (a layout step of this implementation). */
int ws_transpose_bf16(const void* in, int64_t ld_in, void* out, int64_t rows, int64_t cols,
                      void* stream);

/*
 * RMSNorm-prologue projection with gate sigmoid: out[m,n] = bf16(y @ B) with
 * y = r(r(x * rstd) * r(norm_weight)), then out[:, gate_begin:gate_end] = r(sigmoid(out)).
 * The prologue is one pass over x that writes y into `normed` [m, k] (row-contiguous,
 * caller-allocated; it is also the saved input of the projection's weight gradient) and
 * rstd [m]; the GEMM then reads y. Restates RMSNorm.forward (warpstate/model.py:22-28) ->
 * in_proj (warpstate/model.py:93, 109) -> torch.sigmoid on the gate slice
 * (warpstate/model.py:174). x needs a unit column stride.
 */
int ws_rmsnorm_gate_mm(const void* x, int64_t x_s0, const float* norm_weight, float eps,
                       float* rstd, void* normed, const void* b, int64_t b_s0, int64_t b_s1,
                       void* out, int64_t m, int64_t n, int64_t k, int64_t gate_begin,
                       int64_t gate_end, void* stream);

/* Gradient through the gate sigmoid of ws_rmsnorm_gate_mm's output: dp = dout, except
 * columns [gate_begin, gate_end) where dp = r(dout * (1 - out) * out) with `out` the forward
 * output (torch.sigmoid's backward, warpstate/model.py:174). dp may be dout itself (then
 * only the gate columns are rewritten). */
int ws_sigmoid_backward_cols(const void* dout, int64_t ld_dout, const void* out, int64_t ld_out,
                             void* dp, int64_t ld_dp, int64_t rows, int64_t cols,
                             int64_t gate_begin, int64_t gate_end, void* stream);

/* Down projection with residual add: out[m,n] = r(residual[m,n] + r(A @ B)), residual
 * row stride ld_residual (warpstate/model.py:178 under BF16 residuals,
 * ops/residual_experiment.py:25-58). */
int ws_residual_mm(const void* a, int64_t a_s0, int64_t a_s1, const void* b, int64_t b_s0,
                   int64_t b_s1, const void* residual, int64_t ld_residual, void* out, int64_t m,
                   int64_t n, int64_t k, void* stream);

/*
 * Down-projection dgrad with SwiGLU-backward epilogue: dact = r(grad @ B) (grad [m,k] =
 * dY, B [k,h] = W_down of nn.Linear layout [k,h]) is never stored; from the saved packed
 * [m,2h] projection it writes dpacked [m,2h] = (dUp | dGate). Restates `_mm_backward`'s
 * dX (ops/matmul_execution.py:239) followed by `_swiglu_backward_kernel`
 * (ops/activation_execution.py:36-55).
 */
int ws_swiglu_backward_mm(const void* grad, int64_t g_s0, int64_t g_s1, const void* b,
                          int64_t b_s0, int64_t b_s1, const void* packed, void* dpacked,
                          int64_t m, int64_t h, int64_t k, int eager_rounding, void* stream);

/* Floats of the workspace ws_mm_accumulate_f32 needs for an [m, n] gradient with
 * reduction k and `splits` (0 when splits <= 1), on the current device. */
int64_t ws_mm_accumulate_workspace_floats(int64_t m, int64_t n, int64_t k, int64_t splits);

/*
 * Weight-gradient GEMM accumulated into an FP32 buffer: G[m,n] += f32(r(A @ B)) when
 * round_bf16 (the BF16 dW then AccumulateGrad of test_gradient_execution.py:243-246 and
 * ops/matmul_execution.py:243), or G += A @ B in FP32 otherwise (the "direct_fp32_addmm"
 * variant of ops/benchmark_gradient_accumulation.py:141-144). splits > 1 lets the
 * reduction be split through `workspace`: for operands with a contiguous reduction or row
 * dimension the 256 x 256 tiles that fill whole rounds of the GPU accumulate directly and
 * the remaining tiles' k-range is shared evenly by all compute units (FP32 partial sums,
 * added in k order, rounded once); other layouts use `splits` even k-slices.
 */
int ws_mm_accumulate_f32(const void* a, int64_t a_s0, int64_t a_s1, const void* b, int64_t b_s0,
                         int64_t b_s1, float* g, int64_t ldg, int64_t m, int64_t n, int64_t k,
                         int round_bf16, float* workspace, int64_t splits, void* stream);

/* One weight gradient of a grouped accumulation: G[m, n] (row stride ldg) += A[m, k] B[k, n],
 * with A and B given by pointer and (row, column) element strides as in ws_mm. */
typedef struct ws_accumulate_problem {
  const void* a;
  int64_t a_s0, a_s1;
  const void* b;
  int64_t b_s0, b_s1;
  float* g;
  int64_t ldg;
  int64_t m, n;
} ws_accumulate_problem;

/* Floats of the workspace ws_mm_accumulate_f32_group needs for these problems (0 when
 * none), on the current device. */
int64_t ws_mm_accumulate_group_workspace_floats(const ws_accumulate_problem* problems, int count,
                                                int64_t k);

/*
 * Up to four weight-gradient accumulations with the same reduction length k (the token
 * count) in one launch, each with the numerics of ws_mm_accumulate_f32 (round_bf16 as
 * there): the weight gradients of one backward stage, computed together instead of as
 * separate AccumulateGrad steps (ops/matmul_execution.py:243 once per weight; fused, new).
 * Their 256 x 256 tiles form one raster: whole rounds of the GPU run directly, the rest
 * is shared evenly by all compute units through `workspace`, so a gradient with fewer
 * tiles than compute units fills the GPU together with the others. The gradients must not
 * overlap. When the problems' operand layouts differ or do not take the fast loader, the
 * call runs ws_mm_accumulate_f32 per problem (split-K through `workspace` when given).
 */
int ws_mm_accumulate_f32_group(const ws_accumulate_problem* problems, int count, int64_t k,
                               int round_bf16, float* workspace, void* stream);

/*
 * G = f32(r(A @ B)) (or the FP32 product when round_bf16 is 0): ws_mm_accumulate_f32 and
 * ws_mm_accumulate_f32_group with the gradient buffers written instead of updated, so
 * they need no clearing and are never read. Same arguments, workspace sizes
 * (ws_mm_accumulate_workspace_floats, ws_mm_accumulate_group_workspace_floats) and
 * paths. This is the BF16 weight gradient of F.linear under autocast widened to FP32,
 * the value AccumulateGrad adds to an FP32 master's .grad
 * (ops/matmul_execution.py:243; test_gradient_execution.py:243-246), produced in one
 * FP32 pass for an adapter that returns it through autograd (new).
 */
int ws_mm_store_f32(const void* a, int64_t a_s0, int64_t a_s1, const void* b, int64_t b_s0,
                    int64_t b_s1, float* g, int64_t ldg, int64_t m, int64_t n, int64_t k,
                    int round_bf16, float* workspace, int64_t splits, void* stream);
int ws_mm_store_f32_group(const ws_accumulate_problem* problems, int count, int64_t k,
                          int round_bf16, float* workspace, void* stream);

/* Or-ed into a leading dimension of the LM-head gradient calls (ld_dweight of
 * ws_linear_ce_backward and ws_linear_ce_fused, ld_unit of ws_linear_ce_fused_backward):
 * dweight is written instead of accumulated into, so that it needs no clearing and is not
 * read before it is written. */
#define WS_WRITE_DWEIGHT ((int64_t)1 << 62)

/* Number of per-row partials (floats per row of part_max / part_sum) for `vocab`. */
int64_t ws_linear_ce_parts(int64_t vocab);

/*
 * Fused LM-head cross-entropy forward. hidden [rows, d] (row stride ld_hidden, unit column
 * stride), weight [vocab, d] (nn.Embedding / tied head layout, row stride ld_weight),
 * int64 targets with -100 ignored. Writes per-token FP32 loss, lse, the target logit,
 * mean = sum(loss) / max(1, count) and the int64 valid-token count. `logits` (nullable): when given, the rounded
 * BF16 logits are also stored there ([rows, vocab], row stride vocab; vocab % 4 == 0,
 * 16-byte aligned; both operands row-contiguous) for a backward that reads them instead
 * of recomputing the GEMM. Without it the logits exist only in registers.
 * Restates the chunked head of WarpStateLM.forward (warpstate/model.py:316-334) and
 * `_full_loss` (ops/loss_experiment.py:14-19).
 */
int ws_linear_ce_forward(const void* hidden, int64_t ld_hidden, const void* weight,
                         int64_t ld_weight, const int64_t* targets, int64_t rows, int64_t vocab,
                         int64_t d, float* part_max, float* part_sum, float* target_logit,
                         float* lse, float* loss, float* mean, int64_t* count, void* logits,
                         void* stream);

/* Bytes of the workspace ws_linear_ce_backward needs for `chunk_rows`-row chunks. */
int64_t ws_linear_ce_workspace_bytes(int64_t rows, int64_t vocab, int64_t d, int64_t chunk_rows);

/*
 * Fused LM-head cross-entropy backward: dhidden [rows, d] = r(r(g (softmax - onehot)) @ W)
 * with g = grad_mean / max(1, count), zero rows for ignored targets. Rows are processed
 * chunk_rows at a time: the BF16 logit gradients of one chunk ([chunk_rows, vocab], never
 * the whole batch) go to the 256-byte aligned `workspace` and feed that chunk's dHidden
 * GEMM, split over the vocab with FP32 partials when the chunk alone would not fill the
 * GPU. `weight_t` (nullable) is the head weight transposed, [d, vocab] contiguous; when
 * given, the dHidden GEMM reads it instead of `weight`, unless the vocabulary is no multiple
 * of 8 and the vector kernels take the chunk. `dweight` (nullable, FP32
 * [vocab, d], row stride ld_dweight) receives the tied head weight's gradient, accumulated
 * per chunk as dweight += f32(r(G_chunk^T @ hidden_chunk)): the BF16 weight gradient of the
 * chunk's F.linear followed by FP32 accumulation (warpstate/model.py:321-331 under BF16
 * autocast, test_gradient_execution.py:243-246). `logits` (nullable): the logits the
 * forward stored; each chunk's logit gradients then come from one elementwise pass over
 * them (same arithmetic, same bits) instead of a recomputing GEMM. Restates autograd of
 * warpstate/model.py:321-334.
 */
int ws_linear_ce_backward(const void* hidden, int64_t ld_hidden, const void* weight,
                          int64_t ld_weight, const void* weight_t, const int64_t* targets,
                          const float* lse, const int64_t* count, const float* grad_mean,
                          int64_t rows, int64_t vocab, int64_t d, void* workspace,
                          int64_t chunk_rows, void* dhidden, int64_t ld_dhidden, float* dweight,
                          int64_t ld_dweight, const void* logits, void* stream);

/*
 * Fused LM-head cross-entropy in one pass: the outputs of ws_linear_ce_forward plus the
 * gradients for a unit upstream gradient of the mean, dhidden [rows, d] BF16 and (nullable)
 * dweight [vocab, d] FP32 (+=), with the numerics of ws_linear_ce_backward at grad_mean = 1.
 * Rows go chunk_rows at a time through the workspace of ws_linear_ce_workspace_bytes: the
 * chunk's logits GEMM stores its BF16 logits in the workspace chunk (the whole [rows, vocab]
 * logits never exist), the chunk's row statistics give its lse and loss, one elementwise
 * pass turns the stored logits into the logit gradients in place, and they feed the
 * chunk's dHidden and head-weight GEMMs: one logits GEMM per row instead of the forward's
 * and the backward's. `weight_t` as in ws_linear_ce_backward. Restates
 * warpstate/model.py:316-334 with its autograd.
 */
int ws_linear_ce_fused(const void* hidden, int64_t ld_hidden, const void* weight,
                       int64_t ld_weight, const void* weight_t, const int64_t* targets,
                       int64_t rows, int64_t vocab, int64_t d, float* part_max, float* part_sum,
                       float* target_logit, float* lse, float* loss, float* mean, int64_t* count,
                       void* workspace, int64_t chunk_rows, void* dhidden, int64_t ld_dhidden,
                       float* dweight, int64_t ld_dweight, void* stream);

/*
 * Backward of ws_linear_ce_fused for the actual upstream gradient grad_mean (device FP32
 * scalar): dhidden [rows, d] BF16 (row stride ld_dhidden) and, when given, dweight
 * [vocab, d] FP32 (contiguous, +=). When grad_mean is +-2^e with |e| <= 32, scaling
 * commutes with every rounding that stays in the normal range, and the results are
 * grad_mean * dhidden_unit and dweight + grad_mean * dweight_unit: the two-pass backward's
 * results bit for bit (dweight up to summation order into a nonzero buffer), except for
 * elements that are subnormal before or after the scaling. Otherwise it runs the two-pass
 * backward (ws_linear_ce_backward's arguments). The choice is made on the device, without a host synchronisation: both paths
 * are launched and the kernels of the one not taken exit at once.
 */
int ws_linear_ce_fused_backward(const void* hidden, int64_t ld_hidden, const void* weight,
                                int64_t ld_weight, const void* weight_t, const int64_t* targets,
                                const float* lse, const int64_t* count, const float* grad_mean,
                                int64_t rows, int64_t vocab, int64_t d, void* workspace,
                                int64_t chunk_rows, const void* dhidden_unit, int64_t ld_unit,
                                const float* dweight_unit, void* dhidden, int64_t ld_dhidden,
                                float* dweight, void* stream);

/*
 * The second phase of ws_linear_ce_forward on its own: lse and loss per row from the
 * statistics partials part_max / part_sum ([rows, ws_linear_ce_parts(vocab)]) and the
 * target logits, then mean = sum(loss) / max(1, count) and the int64 count (the combine
 * step of the chunked head, warpstate/model.py:326-334, ops/loss_experiment.py:18-19).
 */
int ws_linear_ce_combine(const float* part_max, const float* part_sum, const float* target_logit,
                         const int64_t* targets, float* lse, float* loss, float* mean,
                         int64_t* count, int64_t rows, int64_t vocab, void* stream);

/*
 * Logit gradients from BF16 logits: out = r(scale (exp(l - lse) - onehot)), zero rows for
 * ignored targets, `scale` a device FP32 scalar; `out` may be `logits` (in place). vocab % 4
 * == 0, row strides multiples of 8, 16-byte aligned buffers. The elementwise pass of the
 * fused loss (autograd of F.cross_entropy on BF16 logits, warpstate/model.py:328-334).
 */
int ws_linear_ce_logit_grad(const void* logits, int64_t ld_logits, const int64_t* targets,
                            const float* lse, const float* scale, void* out, int64_t ld_out,
                            int64_t rows, int64_t vocab, void* stream);

/*
 * Packed attention-backward gradient layout: out [B, N*C, 5*H*D] BF16 (token-major rows of
 * [q | k | v | gate | u], each H*D wide) from the saved head-major [B, N, H, C, D] BF16
 * tensors q_memory, q_local, tanh_k, k_local, v_local, memory, local, gate, u_write, tanh_u,
 * k_write [B, N, H, D, C], grad_y [B, N*C, H*D] and FP32 rope tables sin, cos [C, D]; all
 * contiguous. `scale` multiplies memory in the gate gradient (head_dim^-0.5).
 * `algorithm`: 0 = "profile" (two passes through the caller's head-major BF16 scratch_q and
 * scratch_k, the reference's profiled two-kernel baseline), 1 = "paired" (q/k pass, then
 * v/gate/u pass), 2 = "single" (one pass). All three give identical bits. Replaces the
 * launches of prepare_layout (ops/backward_layout.py:213-276) of the kernels at :116-210.
 */
int ws_backward_layout(const void* q_memory, const void* q_local, const float* sin,
                       const float* cos, const void* k_write, const void* tanh_k,
                       const void* k_local, const void* v_local, const void* grad_y,
                       const void* memory, const void* local, const void* gate,
                       const void* u_write, const void* tanh_u, void* out, int64_t batch,
                       int64_t chunks, int64_t heads, int64_t chunk_size, int64_t head_dim,
                       float scale, int algorithm, void* scratch_q, void* scratch_k,
                       void* stream);

/* --- 8-bit products -------------------------------------------------------------------
 *
 * e4m3 (OCP, largest finite value 448) matrices with one scale per block of 128: 1 x 128
 * along the reduction, or 128 x 128. Scale types: WS_SCALE_E8M0, a byte e + 127 for 2^e (255:
 * NaN), scale (r, b) at r * ld + b; WS_SCALE_F32, a float, scale (r, b) at b * ld + r, where r
 * counts rows, or groups of 128 rows, and b the blocks along the reduction.
 */
enum WsScaleType { WS_SCALE_E8M0 = 0, WS_SCALE_F32 = 1 };
enum WsQuantForm { WS_QUANT_ROWS = 1, WS_QUANT_COLUMNS = 2, WS_QUANT_BLOCKS = 4 };

/* x [rows, cols] (row stride ldx, BF16 or, with x_f32, FP32) to e4m3. `form`:
 *   WS_QUANT_ROWS     q [rows, cols], scale [rows, ceil(cols / 128)];
 *   WS_QUANT_COLUMNS  qt [cols, rows] (transposed), scale_t [cols, ceil(rows / 128)];
 *   both of them      from one read of x;
 *   WS_QUANT_BLOCKS   q [rows, cols], scale [ceil(rows / 128), ceil(cols / 128)], and, with qt,
 *                     the same values transposed: qt [cols, rows], scale_t the transpose of scale.
 * Scales: e8m0, the least power of two (at least 2^-126) under which the block's magnitudes
 * are at most 448; FP32, a (1 / 448) with a = max(amax, 2^-100). q = rne(x / scale) (FP32
 * scales: x times 448 (1 / a); every operation rounded to FP32). A block with an infinity or a
 * NaN gets the scale NaN (e8m0) or its amax / 448 (FP32). ldq and ldqt are multiples of 16 and
 * their buffers 16-byte aligned; bytes past cols (rows of x for qt) up to the next multiple of
 * 16 are written as zeros. */
int ws_fp8_quantize(const void* x, int64_t ldx, int x_f32, int64_t rows, int64_t cols, int form,
                    int scale_type, void* q, int64_t ldq, void* scale, int64_t ld_scale, void* qt,
                    int64_t ldqt, void* scale_t, int64_t ld_scale_t, void* stream);

/* Byte matrix src (r, c) at r * s_row + c * s_col into dst rows of ldd bytes (a multiple of 16,
 * 16-byte aligned), zeros past cols: an operand of ws_fp8_mm from any layout. */
int ws_fp8_pack(const void* src, int64_t s_row, int64_t s_col, void* dst, int64_t ldd, int64_t rows,
                int64_t cols, void* stream);

/* BF16 C [m, n] (row stride ldc) = sum over blocks b of scale_a scale_b (A_b B_b^T) with e4m3 A
 * [m, k] (row stride lda) and B [n, k] (nn.Linear layout, row stride ldb), FP32 accumulation (of
 * groups of eight products whose terms the instruction cuts at 13 bits below the largest). k,
 * lda and ldb are multiples of 16 and the operands 16-byte aligned (bytes past a matrix's own
 * reduction have to be zero: ws_fp8_pack). *_block_rows is 1 (a scale per row and block) or 128
 * (per 128 rows and block). e8m0 scales: 4-byte aligned, ld a multiple of 4, rows readable to
 * the next multiple of 4 bytes. FP32 scales of B with b_block_rows 1: 16-byte aligned, ld a multiple of
 * 4. `workspace`: 16-byte aligned, ws_fp8_mm_workspace_bytes (null if that is 0): slices of the
 * reduction where the tiles alone would leave compute units idle. */
int64_t ws_fp8_mm_workspace_bytes(int64_t m, int64_t n, int64_t k, int b_block_rows, int scale_type);
/* What ws_fp8_mm runs these sizes on, without a launch: 0 256 x 256, 1 and 2 128 x 128 (two or
 * one workgroup on a compute unit), 3 64 x 128, 4 64 x 64, 5 the kernel for few rows; -1 for
 * invalid sizes. workspace_bytes and splits (slices of the reduction) are nullable. */
int ws_fp8_mm_plan(int64_t m, int64_t n, int64_t k, int b_block_rows, int scale_type,
                   int64_t* workspace_bytes, int* splits);
int ws_fp8_mm(const void* a, int64_t lda, const void* scale_a, int64_t ld_scale_a, int a_block_rows,
              const void* b, int64_t ldb, const void* scale_b, int64_t ld_scale_b, int b_block_rows,
              int scale_type, void* c, int64_t ldc, int64_t m, int64_t n, int64_t k,
              void* workspace, void* stream);

/* --- token scores ---------------------------------------------------------------------
 *
 * For each row of logits l (times inv_temperature, 2^-126 to 2.3e38): logprob = l[token] - lse,
 * entropy = lse - sum p l, lse = log sum e^l, FP32. A token of -100 has logprob 0 and takes no
 * gradient; any other token outside [0, vocab) gets NaN. Logits of -inf have probability 0; a row
 * of nothing else gets NaN. Finite logits of any size have scores (a mask of the type's lowest
 * value among them): only their distances to the row's largest are scaled.
 */

/* From logits [rows, vocab] (row stride ld, BF16 or, with f32, FP32; any alignment of their
 * type; vocab at most 524288). top_k (0 to min(64, vocab)): top_ids and top_logprobs [rows,
 * top_k] receive the largest logits' ids and log probabilities, largest first, equal logits by
 * their lowest id. `workspace`: 16-byte aligned, ws_token_scores_workspace_bytes (null if that
 * is 0). */
int64_t ws_token_scores_workspace_bytes(int64_t rows, int64_t vocab, int64_t top_k);
int ws_token_scores(const void* logits, int64_t ld, int f32, const int64_t* tokens, int64_t rows,
                    int64_t vocab, float inv_temperature, int64_t top_k, void* workspace, float* lse,
                    float* logprob, float* entropy, float* top_logprobs, int64_t* top_ids,
                    void* stream);
/* dlogits [rows, vocab] (row stride ld_out, the logits' type; may be the logits) of
 * sum(dlogprob logprob + dentropy entropy); either of the two may be null (zero). lse and
 * entropy are the forward's; a row with |lse| of 256 or more is summed again, in distances. A row
 * whose two upstream gradients are zero gets zeros. */
int ws_token_scores_backward(const void* logits, int64_t ld, int f32, const int64_t* tokens,
                             int64_t rows, int64_t vocab, float inv_temperature, const float* lse,
                             const float* entropy, const float* dlogprob, const float* dentropy,
                             void* dlogits, int64_t ld_out, void* stream);

/* From hidden [rows, d] and the head weight [vocab, d] (BF16, 16-byte aligned rows, d a
 * multiple of 8): the logits are the FP32 products, and exist in registers only. */
int64_t ws_linear_token_scores_workspace_floats(int64_t rows, int64_t vocab, int64_t d);
int ws_linear_token_scores(const void* hidden, int64_t ld_hidden, const void* weight,
                           int64_t ld_weight, const int64_t* tokens, int64_t rows, int64_t vocab,
                           int64_t d, float inv_temperature, float* workspace, float* lse,
                           float* logprob, float* entropy, void* stream);
/* Gradients of sum(dlogprob logprob + dentropy entropy): dhidden [rows, d] BF16 and dweight
 * [vocab, d] FP32 or, with dweight_bf16 (one chunk, ld_dweight = d), BF16 (written), each
 * nullable. The logits are recomputed chunk_rows rows at a time, and their gradient, rounded to
 * BF16, feeds the two products. weight_t: null, or the weight transposed ([d, vocab], vocab a
 * multiple of 8). Probabilities are e^(l - lse) with lse in FP32, off by up to 2^-24 |lse| as the
 * FP32 logits themselves are. `workspace`: 256-byte aligned. */
int64_t ws_linear_token_scores_backward_workspace_bytes(int64_t rows, int64_t vocab, int64_t d,
                                                        int64_t chunk_rows);
int ws_linear_token_scores_backward(const void* hidden, int64_t ld_hidden, const void* weight,
                                    int64_t ld_weight, const void* weight_t, const int64_t* tokens,
                                    const float* lse, const float* entropy, const float* dlogprob,
                                    const float* dentropy, int64_t rows, int64_t vocab, int64_t d,
                                    float inv_temperature, void* workspace, int64_t chunk_rows,
                                    void* dhidden, int64_t ld_dhidden, void* dweight,
                                    int64_t ld_dweight, int dweight_bf16, void* stream);

/* --- residual norm ---------------------------------------------------------------------
 *
 * s = r(x + residual) in the residual stream's type (BF16, or FP32 with stream_f32), then the
 * RMSNorm of the rounded s: y = s rstd w, rstd = 1 / sqrt(mean(s^2) + eps), rounded once. x is BF16,
 * the weight FP32; up to 2^30 rows of 1 to 8192 columns, row strides in elements, outputs contiguous.
 */

/* y [rows, d] BF16, stream_out [rows, d] = s. */
int ws_add_rmsnorm(const void* x, int64_t ldx, const void* residual, int64_t ld_residual,
                   int stream_f32, const float* weight, float eps, int64_t rows, int64_t d, void* y,
                   void* stream_out, void* stream);
/* The unrounded y quantized by rows (WS_QUANT_ROWS of ws_fp8_quantize): q, ldq, scale and
 * ld_scale as there. With a null residual s is x and stream_out is null. */
int ws_rmsnorm_quantize(const void* x, int64_t ldx, const void* residual, int64_t ld_residual,
                        int stream_f32, const float* weight, float eps, int64_t rows, int64_t d,
                        int scale_type, void* q, int64_t ldq, void* scale, int64_t ld_scale,
                        void* stream_out, void* stream);
/* With stream_in [rows, d] = s and the forward's eps, dy BF16 and dstream (nullable: zero) in the
 * stream's type: dx [rows, d] BF16, the gradient of x and of a BF16 residual; dresidual (nullable)
 * the same in FP32 for an FP32 stream; dweight [d]. `partial`: ws_add_rmsnorm_backward_partial_floats
 * (which follows the device's compute units; null if that is 0). */
int64_t ws_add_rmsnorm_backward_partial_floats(int64_t rows, int64_t d);
int ws_add_rmsnorm_backward(const void* stream_in, int stream_f32, const float* weight,
                            float eps, const void* dy, int64_t ld_dy, const void* dstream,
                            int64_t ld_dstream, int64_t rows, int64_t d, void* dx, float* dresidual,
                            float* dweight, float* partial, void* stream);

/* --- embedding -------------------------------------------------------------------------
 *
 * y [rows, d] (BF16, or FP32 with y_f32) = scale * table[token] from a BF16 or FP32 table [vocab,
 * d] (row stride ld_table). A token of -100 is ignored: its row is zeros. Any other token outside
 * [0, vocab) gets NaN. Up to 2^22 rows of 2^20 columns of the table, and 2^24 tokens.
 */
int ws_embedding(const void* table, int64_t ld_table, int table_f32, const int64_t* tokens,
                 int64_t rows, int64_t vocab, int64_t d, float scale, void* y, int y_f32,
                 void* stream);
/* dtable [vocab, d] = scale * the sums of dy's rows (BF16, or FP32 with dy_f32) by token, FP32 in
 * the order of the rows: the same bits on every call. Written in BF16 or FP32, or added to FP32
 * values that are there (rows without tokens then stay as they are, unread). Tokens outside the
 * vocabulary, ignored ones among them, take no part. `workspace`: 16-byte aligned,
 * ws_embedding_backward_workspace_bytes (null if that is 0). */
enum WsEmbedGrad { WS_EMBED_WRITE_BF16 = 0, WS_EMBED_WRITE_F32 = 1, WS_EMBED_ADD_F32 = 2 };
int64_t ws_embedding_backward_workspace_bytes(int64_t rows, int64_t vocab, int64_t d);
int ws_embedding_backward(const void* dy, int64_t ld_dy, int dy_f32, const int64_t* tokens,
                          int64_t rows, int64_t vocab, int64_t d, float scale, void* dtable,
                          int64_t ld_dtable, int mode, void* workspace, void* stream);

/* --- products grouped by expert --------------------------------------------------------
 *
 * Rows sorted by expert: rows offsets[e] to offsets[e + 1] of x belong to group e (offsets: groups + 1
 * int64 on the device, not decreasing). The offsets are read on the device only, and no value of theirs
 * leads an access out of the operands; decreasing ones leave rows of the result unspecified. BF16
 * operands, FP32 sums, 16-byte aligned rows, weight rows of a multiple of 8 elements, 1 to 16384
 * groups, up to 2^30 rows; in tiles of 256 x 256, fewer than 2^24 for a product, (rows / 256 + groups + 2)
 * ceil(n / 256), and fewer than 2^22 for a weight gradient, groups ceil(n / 256) ceil(k / 256). The other width, n below, may be any; rows of that width reach to its
 * next multiple of 8: y's are written up to there, and dy's, like x's under WS_GROUPED_NN, have
 * to hold zeros.
 */

/* y [rows, n] BF16 = x [rows, k] times the transpose of the group's weight [n, k] (WS_GROUPED_NT:
 * a projection; k a multiple of 8), or times its weight [k, n] itself (WS_GROUPED_NN: the input
 * gradient of one; n a multiple of 8), both row-major with row stride ld_weight, group_stride elements
 * from one group's to the next. Where ws_grouped_tile is 5 or 6, x and the weights may have any k, any
 * strides and the alignment of their elements. Rows before the first offset and behind the last get
 * zeros. The sums of the tiles have one order, those of the kernel for few rows, and of long
 * reductions that are cut in slices, another. `workspace`:
 * 16-byte aligned, ws_grouped_workspace_floats (which follows the device's compute units; null if that
 * is 0). */
enum WsGroupedForm { WS_GROUPED_NT = 0, WS_GROUPED_NN = 1, WS_GROUPED_GRAD = 2 };
int ws_grouped_mm(const void* x, int64_t ldx, const void* weight, int64_t ld_weight,
                  int64_t group_stride, int form, const int64_t* offsets, int64_t groups,
                  int64_t rows, int64_t n, int64_t k, void* y, int64_t ldy, float* workspace, void* stream);
int64_t ws_grouped_workspace_floats(int64_t rows, int64_t groups, int64_t n, int64_t k, int form);
/* dweight [groups, n, k] (contiguous, BF16 or FP32) = the sums over each group's rows of
 * dy^T x, dy [rows, n] and x [rows, k]; a group without rows gets zeros. */
int ws_grouped_weight_grad(const void* dy, int64_t ld_dy, const void* x, int64_t ldx,
                           const int64_t* offsets, int64_t groups, int64_t rows, int64_t n,
                           int64_t k, void* dweight, int dweight_f32, void* stream);
/* Whether the gradients of a product y = x w^T of these sizes, with widths padded to multiples of 8, fit what
 * the calls above take: dx (WS_GROUPED_NN) and dweight where asked for. No launch; for a forward that would
 * otherwise be recorded in vain. */
int ws_grouped_backward_check(int64_t rows, int64_t groups, int64_t n, int64_t k, int dx, int dweight,
                              int dweight_f32);
/* Matrices of any width as these products take them, and back: for each group, rows [rows_in, cols_in]
 * into rows [rows_out, cols_out] with zeros past the input's last row and column, rows and columns past
 * the output's left out. BF16 or FP32, in the input's type or rounded from FP32 to BF16; any alignment
 * of the types. Up to 2^24 groups. */
int ws_copy_rows(const void* in, int in_f32, int64_t group_in, int64_t ld_in, int64_t rows_in,
                 int64_t cols_in, void* out, int out_f32, int64_t group_out, int64_t ld_out,
                 int64_t rows_out, int64_t cols_out, int64_t groups, void* stream);
/* What these sizes run on, without a launch (WS_GROUPED_GRAD: the weight gradient): 0 256 x 256,
 * 1 and 2 128 x 128 (two or one workgroup on a compute unit), 3 64 x 128, 4 64 x 64, 5 and 6 the kernel
 * for few rows (tiles of 32 or 16 columns); -1 for invalid sizes. */
int ws_grouped_tile(int64_t rows, int64_t groups, int64_t n, int64_t k, int form);

#ifdef __cplusplus
}
#endif

#endif /* WARPSTATE_HIP_H */
