// extern "C" surface of the 4-bit matrices (declared in include/flux_cuda.h): argument checks, then one launch on the
// context's stream. The context is looked at last, so every other refusal can be provoked without a GPU.
#include <math.h>

#include "context.cuh"
#include "fp4.cuh"

using namespace fx;

namespace {

// The context's device for the length of a call, whichever one the calling thread works on.
struct OnDevice {
  int before = -1;
  explicit OnDevice(int device) {
    if (cudaGetDevice(&before) != cudaSuccess || before == device) before = -1;
    else cudaSetDevice(device);
  }
  ~OnDevice() {
    if (before >= 0) cudaSetDevice(before);
  }
};

bool is_dtype(int d) { return d == FLUX_CUDA_F32 || d == FLUX_CUDA_F16 || d == FLUX_CUDA_BF16; }
int size_of(int d) { return d == FLUX_CUDA_F32 ? 4 : 2; }

int refuse(const char *op, const char *what) {
  set_error("%s: %s", op, what);
  return FLUX_CUDA_ERR_ARG;
}

int check_matrix(const char *op, const char *name, const flux_cuda_fp4 *q) {
  const char *why = nullptr;
  if (!q) why = "is null";
  else if (q->format != FLUX_CUDA_NVFP4 && q->format != FLUX_CUDA_MXFP4) why = "has an unknown format";
  else if (q->rows < 0 || q->cols < 1) why = "needs rows >= 0 and cols >= 1";
  else if (q->rows > 0 && (!q->codes || !q->scales)) why = "has no memory";
  else if ((reinterpret_cast<uintptr_t>(q->codes) & 15) || (reinterpret_cast<uintptr_t>(q->scales) & 15))
    why = "needs codes and scales on 16-byte boundaries";
  else if (!isfinite(q->scale)) why = "has a scale that is not finite";
  if (!why) return FLUX_CUDA_OK;
  set_error("%s: %s %s", op, name, why);
  return FLUX_CUDA_ERR_ARG;
}

// A plain matrix of `rows` x `cols` elements with row pitch ld.
int check_plain(const char *op, const char *name, const void *p, int dtype, long long ld, long long rows, long long cols) {
  const char *why = nullptr;
  if (!is_dtype(dtype)) why = "has an unknown type";
  else if (rows > 0 && cols > 0 && !p) why = "is null";
  else if (reinterpret_cast<uintptr_t>(p) & (size_of(dtype) - 1)) why = "is not aligned to its type";
  else if (ld < cols) why = "has a row pitch below its width";
  if (!why) return FLUX_CUDA_OK;
  set_error("%s: %s %s", op, name, why);
  return FLUX_CUDA_ERR_ARG;
}

// Quantising and back take blocks of 32 rows x 256 columns.
bool too_large(const flux_cuda_fp4 &q) { return fp4_row_tiles(q.rows) * 4 * ((q.cols + 255LL) / 256) > 0x7FFFFFFF; }

int finish(const char *op, int rc) {
  if (rc == 0) return FLUX_CUDA_OK;
  if (rc == FP4_ERR_MAP) {
    set_error("%s: tensor map refused", op);
  } else {
    set_error("%s: launch failed: %s", op, cudaGetErrorString(static_cast<cudaError_t>(rc)));
    cudaGetLastError();  // it has been reported
  }
  return FLUX_CUDA_ERR_CUDA;
}

}  // namespace

extern "C" {

long long flux_cuda_fp4_code_bytes(int rows, int cols) {
  if (rows < 0 || cols < 1) return -1;
  return rows * fp4_pitch(cols);
}

long long flux_cuda_fp4_scale_bytes(int rows, int cols, int format) {
  if (rows < 0 || cols < 1 || (format != FLUX_CUDA_NVFP4 && format != FLUX_CUDA_MXFP4)) return -1;
  return fp4_row_tiles(rows) * fp4_chunks(cols, format) * 512;
}

int flux_cuda_fp4_quantize(flux_cuda_ctx *ctx, const void *x, int dtype, long long ldx, const flux_cuda_fp4 *q) {
  const char *op = "fp4_quantize";
  int rc = check_matrix(op, "q", q);
  if (rc || (rc = check_plain(op, "x", x, dtype, ldx, q->rows, q->cols))) return rc;
  int e;
  if (too_large(*q)) return refuse(op, "q is too large for one launch");
  if (frexpf(q->scale, &e) != 0.5f || e < -99 || e > 101) return refuse(op, "q's scale is not a power of two in 2^-100 .. 2^100");
  if (!ctx) return refuse(op, "null context");
  if (q->rows == 0) return FLUX_CUDA_OK;
  OnDevice on(ctx->device);
  return finish(op, launch_fp4_quantize(x, dtype, ldx, *q, ctx->stream));
}

int flux_cuda_fp4_dequantize(flux_cuda_ctx *ctx, const flux_cuda_fp4 *q, void *out, int dtype, long long ld) {
  const char *op = "fp4_dequantize";
  int rc = check_matrix(op, "q", q);
  if (rc || (rc = check_plain(op, "out", out, dtype, ld, q->rows, q->cols))) return rc;
  if (too_large(*q)) return refuse(op, "q is too large for one launch");
  if (!ctx) return refuse(op, "null context");
  if (q->rows == 0) return FLUX_CUDA_OK;
  OnDevice on(ctx->device);
  return finish(op, launch_fp4_dequantize(*q, out, dtype, ld, ctx->err_dev + 1, ctx->stream));
}

int flux_cuda_gemm_fp4(flux_cuda_ctx *ctx, const flux_cuda_fp4 *x, const flux_cuda_fp4 *w, void *out, int dtype,
                       long long ld_out, const float *gate, const float *residual, long long ld_residual) {
  const char *op = "gemm_fp4";
  int rc = check_matrix(op, "x", x);
  if (rc || (rc = check_matrix(op, "w", w)) || (rc = check_plain(op, "out", out, dtype, ld_out, x->rows, w->rows))) return rc;
  if (x->format != w->format) return refuse(op, "x and w have different formats");
  if (x->cols != w->cols) return refuse(op, "x and w have different widths");
  if (gate && (rc = check_plain(op, "gate", gate, FLUX_CUDA_F32, w->rows, 1, w->rows))) return rc;
  if (residual) {
    if ((rc = check_plain(op, "residual", residual, FLUX_CUDA_F32, ld_residual, x->rows, w->rows))) return rc;
    if (residual == out && (dtype != FLUX_CUDA_F32 || ld_residual != ld_out))
      return refuse(op, "residual may be out itself only in f32 and with the same row pitch");
  }
  if (ld_out >= (1LL << 30) || (residual && ld_residual >= (1LL << 30))) return refuse(op, "a row pitch is above 2^30 - 1");
  if (fp4_row_tiles(x->rows) * fp4_row_tiles(w->rows) > 0x3FFFFFFF) return refuse(op, "too many output tiles");
  if (!ctx) return refuse(op, "null context");
  if (x->rows == 0 || w->rows == 0) return FLUX_CUDA_OK;
  OnDevice on(ctx->device);
  Fp4GemmArgs a = {*x, *w, out, dtype, ld_out, gate, residual, ld_residual};
  return finish(op, launch_gemm_fp4(a, ctx->device, ctx->num_sms, ctx->err_dev, ctx->stream));
}

int flux_cuda_gemv_fp4(flux_cuda_ctx *ctx, const void *x, int x_dtype, long long ldx, int rows, const flux_cuda_fp4 *w,
                       void *out, int dtype, long long ld_out) {
  const char *op = "gemv_fp4";
  int rc = check_matrix(op, "w", w);
  if (rc) return rc;
  if (rows < 0 || rows > FP4_GEMV_MAX_ROWS) return refuse(op, "takes 0 to 16 rows");
  if (w->cols > FP4_GEMV_MAX_COLS) return refuse(op, "takes up to 65536 columns");
  if ((rc = check_plain(op, "x", x, x_dtype, ldx, rows, w->cols)) ||
      (rc = check_plain(op, "out", out, dtype, ld_out, rows, w->rows)))
    return rc;
  if (!ctx) return refuse(op, "null context");
  if (rows == 0 || w->rows == 0) return FLUX_CUDA_OK;
  OnDevice on(ctx->device);
  return finish(op, launch_gemv_fp4(x, x_dtype, ldx, rows, *w, out, dtype, ld_out, ctx->device, ctx->err_dev + 1,
                                    ctx->stream));
}

}  // extern "C"
