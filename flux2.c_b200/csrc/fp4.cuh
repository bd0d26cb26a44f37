// 4-bit matrices: e2m1 codes with one factor per block of 16 columns (e4m3) or 32 columns (a power of two), the
// device helpers that read and write them, and the launchers behind the flux_cuda_fp4_* / _gemm_fp4 / _gemv_fp4 entry
// points.
//
// Storage. Codes: row r is 16 * ceil(cols / 32) bytes, the even column of a pair in the low half of its byte; columns
// past the end hold code 0. Factors: one byte per row and block, in tiles of 128 rows x 4 blocks (512 bytes) whose
// byte order is the one tcgen05.cp .32x128b.warpx4 wants, so that a tile goes from global memory to shared memory to
// TMEM as it lies: byte (r % 32) * 16 + (r % 128 / 32) * 4 + b % 4 of tile [r / 128][b / 4]; rows and blocks past the
// end hold 0.
#pragma once
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "flux_cuda.h"
#include "ptx.cuh"

namespace fx {

inline long long fp4_pitch(int cols) { return 16LL * ((static_cast<long long>(cols) + 31) / 32); }
inline long long fp4_blocks(int cols, int format) { return (static_cast<long long>(cols) + format - 1) / format; }
inline long long fp4_chunks(int cols, int format) { return (fp4_blocks(cols, format) + 3) / 4; }
inline long long fp4_row_tiles(int rows) { return (static_cast<long long>(rows) + 127) / 128; }

struct Fp4GemmArgs {
  flux_cuda_fp4 x, w;  // [M, K] and [N, K], the same format
  void *out;
  int dtype;
  long long ld_out;
  const float *gate;      // [N] or null
  const float *residual;  // f32 [M, N] or null; may be `out` itself
  long long ld_residual;
};

// All return 0, the cudaError_t (above 0) of the launch, or FP4_ERR_MAP for a tensor map the driver refuses.
static constexpr int FP4_ERR_MAP = -4;
int launch_fp4_quantize(const void *x, int dtype, long long ldx, const flux_cuda_fp4 &q, cudaStream_t st);
int launch_fp4_dequantize(const flux_cuda_fp4 &q, void *out, int dtype, long long ld, int *sat, cudaStream_t st);
int launch_gemm_fp4(const Fp4GemmArgs &a, int device, int num_sms, int *err, cudaStream_t st);
int launch_gemv_fp4(const void *x, int x_dtype, long long ldx, int rows, const flux_cuda_fp4 &w, void *out, int dtype,
                    long long ld_out, int device, int *sat, cudaStream_t st);
// For the current device, once per context: large shared memory, and how many clusters the device holds at once.
int fp4_gemm_init(int device);
int fp4_gemv_init(int device);

static constexpr int FP4_GEMV_MAX_ROWS = 16, FP4_GEMV_MAX_COLS = 65536;  // what eight SMs' shared memory holds of x

template <int DT>
constexpr int FP4_SIZE = DT == FLUX_CUDA_F32 ? 4 : 2;

// One f32 value as an output element; f16 saturates (the caller counts through `mx`).
template <int DT>
__device__ __forceinline__ void fp4_store(void *out, long long i, float v, float &mx) {
  if (DT == FLUX_CUDA_F32) {
    reinterpret_cast<float *>(out)[i] = v;
  } else if (DT == FLUX_CUDA_F16) {
    mx = fmaxf(mx, fabsf(v));
    reinterpret_cast<uint16_t *>(out)[i] = static_cast<uint16_t>(pack_f16x2(v, 0.f));
  } else {
    reinterpret_cast<uint16_t *>(out)[i] = static_cast<uint16_t>(pack_bf16x2(v, 0.f));
  }
}

// Eight f32 values to eight codes, v[0] in the lowest four bits; round to nearest even, at most +-6.
__device__ __forceinline__ uint32_t fp4_pack8(const float (&v)[8]) {
  uint32_t r;
  asm("{\n\t"
      ".reg .b8 t0, t1, t2, t3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 t0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 t1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 t2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 t3, %8, %7;\n\t"
      "mov.b32 %0, {t0, t1, t2, t3};\n\t"
      "}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}
// Eight codes to four f16 pairs (exact).
__device__ __forceinline__ void fp4_unpack8(uint32_t c, uint32_t (&h)[4]) {
  asm("{\n\t"
      ".reg .b8 t0, t1, t2, t3;\n\t"
      "mov.b32 {t0, t1, t2, t3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, t0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, t1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, t2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, t3;\n\t"
      "}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(c));
}
// A block factor's byte as f32 (exact; the formats' NaN gives NaN).
template <int BLOCK>
__device__ __forceinline__ float fp4_factor(uint32_t byte) {
  if (BLOCK == 32) {
    // 2^(byte - 127); byte 0 is the subnormal 2^-127
    const uint32_t bits = byte == 255 ? 0x7FC00000u : byte == 0 ? 0x00400000u : byte << 23;
    return __uint_as_float(bits);
  }
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(byte)));
  return __half2float(__ushort_as_half(static_cast<uint16_t>(h & 0xFFFFu)));
}

// Two f32 operations in one instruction.
__device__ __forceinline__ uint64_t f2_pack(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void f2_unpack(uint64_t v, float &lo, float &hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t f2_mul(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
// A word of another CTA's shared memory (an address from map_to_cta).
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

}  // namespace fx
