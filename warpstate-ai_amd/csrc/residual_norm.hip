// C ABI: residual addition with RMSNorm (BF16 or 8-bit result) and its backward.
#include "../../include/warpstate_hip.h"
#include "launch.h"
#include "residual_norm.h"
#include "rowops.h"

using namespace ws;

namespace {

constexpr int64_t kMaxWidth = 8192, kMaxRows = 1L << 30;
// Rows of one launch: fewer than 2^32 threads.
constexpr int64_t kLaunchRows = 1L << 22;

int check_shape(int64_t rows, int64_t d) {
  if (rows < 0 || d < 1 || rows > kMaxRows) return set_error(kInvalid, "invalid RMSNorm shape");
  if (d > kMaxWidth) return set_error(kInvalid, "RMSNorm takes rows of at most %ld columns (got %ld)", kMaxWidth, (long)d);
  return kOk;
}
// Few rows leave compute units idle at one wave a row: four waves take it then, and rows of more
// than 2048 columns, whose pieces would not fit one wave's registers.
int waves_per_row(int64_t rows, int64_t d) { return d > 2048 || rows <= 4L * device_cus() ? 4 : 1; }

template <bool F32, bool ADD, int OUT, int NC, int WPR, bool WHOLE>
int launch_forward(AddNormParams p, hipStream_t s) {
  hipLaunchKernelGGL((add_rmsnorm_kernel<F32, ADD, OUT, NC, WPR, WHOLE>), dim3(WPR == 1 ? cdiv(p.rows, 4) : p.rows),
                     dim3(256), 0, s, p);
  return hip_check(hipGetLastError(), "residual norm launch");
}
template <bool F32, bool ADD, int OUT, bool WHOLE>
int run_forward(const AddNormParams& p, hipStream_t s) {
  if (waves_per_row(p.rows, p.d) == 4)
    return p.d <= 2048 ? launch_forward<F32, ADD, OUT, 1, 4, WHOLE>(p, s)
         : p.d <= 4096 ? launch_forward<F32, ADD, OUT, 2, 4, WHOLE>(p, s)
                       : launch_forward<F32, ADD, OUT, 4, 4, WHOLE>(p, s);
  return p.d <= 512    ? launch_forward<F32, ADD, OUT, 1, 1, WHOLE>(p, s)
         : p.d <= 1024 ? launch_forward<F32, ADD, OUT, 2, 1, WHOLE>(p, s)
                       : launch_forward<F32, ADD, OUT, 4, 1, WHOLE>(p, s);
}
template <int OUT>
int dispatch_forward(AddNormParams p, bool f32, hipStream_t s) {
  const int size = f32 ? 4 : 2;
  const bool add = p.residual != nullptr;
  const bool whole = p.d % 8 == 0;
  for (int64_t left = p.rows; left > 0; left -= kLaunchRows) {
    p.rows = (int)(left < kLaunchRows ? left : kLaunchRows);
    int rc;
    if (OUT != kNormBF16 && !add)
      rc = whole ? run_forward<false, OUT == kNormBF16, OUT, true>(p, s) : run_forward<false, OUT == kNormBF16, OUT, false>(p, s);
    else if (f32)
      rc = whole ? run_forward<true, true, OUT, true>(p, s) : run_forward<true, true, OUT, false>(p, s);
    else
      rc = whole ? run_forward<false, true, OUT, true>(p, s) : run_forward<false, true, OUT, false>(p, s);
    if (rc) return rc;
    p.x += kLaunchRows * p.ldx;
    if (add) {
      p.residual = static_cast<const char*>(p.residual) + kLaunchRows * p.ldr * size;
      p.stream = static_cast<char*>(p.stream) + kLaunchRows * p.d * size;
    }
    if (OUT == kNormBF16) {
      p.y += kLaunchRows * p.d;
    } else {
      p.q += kLaunchRows * p.ldq;
      p.scale = static_cast<char*>(p.scale) + kLaunchRows * (OUT == kNormE8M0 ? p.ld_scale : 4);
    }
  }
  return kOk;
}

// Up to 8 rows take one workgroup, two rows a wave, which writes the weight's gradient itself: one launch
// less and no partial sums to allocate. Rows of 2048 columns, one workgroup or several and a reduction:
// 8 rows 6.0 or 7.5 us, 16 rows 9.5 or 7.5 us.
bool one_group(int64_t rows, int64_t d) { return rows <= 8 && d <= 2048; }

// Workgroups of the backward: two on a compute unit, each with one partial row of the weight's
// gradient.
int backward_groups(int64_t rows, int64_t d) {
  if (one_group(rows, d)) return 1;
  const int per = waves_per_row(rows, d) == 4 ? 1 : 4;
  const int64_t most = 2L * device_cus(), need = cdiv(rows, per);
  return (int)(need < most ? need : most);
}

template <bool F32, bool DS, int NC, int WPR, bool WHOLE>
int launch_backward(const AddNormGradParams& p, hipStream_t s) {
  hipLaunchKernelGGL((add_rmsnorm_bwd_kernel<F32, DS, NC, WPR, WHOLE>), dim3(backward_groups(p.rows, p.d)), dim3(256), 0, s, p);
  return hip_check(hipGetLastError(), "residual norm backward launch");
}
template <bool F32, bool DS, bool WHOLE>
int run_backward(const AddNormGradParams& p, hipStream_t s) {
  if (!one_group(p.rows, p.d) && waves_per_row(p.rows, p.d) == 4)
    return p.d <= 2048 ? launch_backward<F32, DS, 1, 4, WHOLE>(p, s)
         : p.d <= 4096 ? launch_backward<F32, DS, 2, 4, WHOLE>(p, s)
                       : launch_backward<F32, DS, 4, 4, WHOLE>(p, s);
  return p.d <= 512    ? launch_backward<F32, DS, 1, 1, WHOLE>(p, s)
         : p.d <= 1024 ? launch_backward<F32, DS, 2, 1, WHOLE>(p, s)
                       : launch_backward<F32, DS, 4, 1, WHOLE>(p, s);
}
template <bool F32>
int dispatch_backward(const AddNormGradParams& p, bool whole, hipStream_t s) {
  if (p.ds) return whole ? run_backward<F32, true, true>(p, s) : run_backward<F32, true, false>(p, s);
  return whole ? run_backward<F32, false, true>(p, s) : run_backward<F32, false, false>(p, s);
}

}  // namespace

extern "C" int ws_add_rmsnorm(const void* x, int64_t ldx, const void* residual, int64_t ld_residual, int stream_f32,
                              const float* weight, float eps, int64_t rows, int64_t d, void* y, void* stream_out,
                              void* stream) {
  if (int rc = check_shape(rows, d)) return rc;
  if (rows == 0) return kOk;
  if (!x || !residual || !weight || !y || !stream_out) return set_error(kInvalid, "null pointer");
  if (rows > 1 && (ldx < d || ld_residual < d)) return set_error(kInvalid, "rows overlap");
  AddNormParams p{};
  p.x = static_cast<const unsigned short*>(x);
  p.ldx = ldx;
  p.residual = residual;
  p.ldr = ld_residual;
  p.w = weight;
  p.rows = (int)rows;
  p.d = (int)d;
  p.eps = eps;
  p.y = static_cast<unsigned short*>(y);
  p.stream = stream_out;
  return dispatch_forward<kNormBF16>(p, stream_f32 != 0, static_cast<hipStream_t>(stream));
}

extern "C" int ws_rmsnorm_quantize(const void* x, int64_t ldx, const void* residual, int64_t ld_residual,
                                   int stream_f32, const float* weight, float eps, int64_t rows, int64_t d,
                                   int scale_type, void* q, int64_t ldq, void* scale, int64_t ld_scale,
                                   void* stream_out, void* stream) {
  if (int rc = check_shape(rows, d)) return rc;
  if (scale_type != WS_SCALE_E8M0 && scale_type != WS_SCALE_F32) return set_error(kInvalid, "unknown scale type %d", scale_type);
  if (rows == 0) return kOk;
  if (!x || !weight || !q || !scale || (residual != nullptr) != (stream_out != nullptr))
    return set_error(kInvalid, "null pointer");
  if (rows > 1 && (ldx < d || (residual && ld_residual < d))) return set_error(kInvalid, "rows overlap");
  const int64_t wide = (d + 15) / 16 * 16, blocks = cdiv(d, kQBlock);
  if (ldq % 16 != 0 || ldq < wide || !al(q, 16)) return set_error(kInvalid, "8-bit rows must be whole 16-byte pieces");
  if (ld_scale < (scale_type == WS_SCALE_E8M0 ? blocks : rows)) return set_error(kInvalid, "scale rows overlap");
  AddNormParams p{};
  p.x = static_cast<const unsigned short*>(x);
  p.ldx = ldx;
  p.residual = residual;
  p.ldr = ld_residual;
  p.w = weight;
  p.rows = (int)rows;
  p.d = (int)d;
  p.eps = eps;
  p.stream = stream_out;
  p.q = static_cast<unsigned char*>(q);
  p.ldq = ldq;
  p.q_cols = (int)wide;
  p.scale = scale;
  p.ld_scale = ld_scale;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool f32 = stream_f32 != 0 && residual;
  return scale_type == WS_SCALE_E8M0 ? dispatch_forward<kNormE8M0>(p, f32, s) : dispatch_forward<kNormF32Scales>(p, f32, s);
}

extern "C" int64_t ws_add_rmsnorm_backward_partial_floats(int64_t rows, int64_t d) {
  if (rows < 1 || d < 1 || d > kMaxWidth || rows > kMaxRows) return 0;
  const int groups = backward_groups(rows, d);
  return groups > 1 ? groups * d : 0;
}

extern "C" int ws_add_rmsnorm_backward(const void* stream_in, int stream_f32, const float* weight, float eps,
                                       const void* dy, int64_t ld_dy, const void* dstream, int64_t ld_dstream,
                                       int64_t rows, int64_t d, void* dx, float* dresidual, float* dweight,
                                       float* partial, void* stream) {
  if (int rc = check_shape(rows, d)) return rc;
  if (rows < 1) return set_error(kInvalid, "invalid RMSNorm shape");
  if (!stream_in || !weight || !dy || !dx || !dweight || (!partial && backward_groups(rows, d) > 1))
    return set_error(kInvalid, "null pointer");
  if (dresidual && !stream_f32) return set_error(kInvalid, "a BF16 stream's gradient is dx");
  if (rows > 1 && (ld_dy < d || (dstream && ld_dstream < d))) return set_error(kInvalid, "rows overlap");
  AddNormGradParams p{};
  p.s = stream_in;
  p.w = weight;
  p.eps = eps;
  p.dy = static_cast<const unsigned short*>(dy);
  p.ld_dy = ld_dy;
  p.ds = dstream;
  p.ld_ds = ld_dstream;
  p.rows = (int)rows;
  p.d = (int)d;
  p.dx = static_cast<unsigned short*>(dx);
  p.dresidual = dresidual;
  const int groups = backward_groups(rows, d);
  p.partial = groups > 1 ? partial : dweight;
  const bool whole = d % 8 == 0;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (int rc = stream_f32 ? dispatch_backward<true>(p, whole, s) : dispatch_backward<false>(p, whole, s)) return rc;
  if (groups == 1) return kOk;
  const bool vec_reduce = d % 4 == 0 && al(partial, 16);
  hipLaunchKernelGGL(vec_reduce ? rms_weight_reduce_kernel<true> : rms_weight_reduce_kernel<false>,
                     dim3(cdiv(d, kRmsReduceCols)), dim3(256), 0, s, partial, dweight, groups, (int)d, 0);
  return hip_check(hipGetLastError(), "residual norm weight reduce launch");
}
