// Quantising to and from 4-bit matrices (layout in fp4.cuh).
//
// Mathematics, per row and block with xs = x / scale and a = max |xs|:
//   blocks of 16:  s = a / 6 rounded to e4m3 (nearest, ties to even, at most 448);  code = e2m1(xs / s)
//   blocks of 32:  s = 2^(floor(log2 a) - 2), exponent within [-127, 127];          code = e2m1(xs / s)
// e2m1() rounds to nearest, ties to even, at most +-6. A block that holds an infinity or a NaN gets the format's NaN as
// its factor. Both roundings are those of the exact quotients: a / 6 is first rounded to odd, and xs / s is a correctly
// rounded quotient, which cannot land on a rounding border the exact one is not on (the factor has four significant
// bits, so the border b has t = b s with at most seven, and |x - t| >= ulp(x) >= 2^-24 |t| keeps the quotient at least
// half an ulp away).
//
// Bound by memory: every element is read once, 0.56 bytes per element are written. A block of 256 threads owns 128 rows x
// 256 columns, 16 consecutive columns per thread, so that a thread has a whole block of 16 (half a block of 32) in
// registers and the factors of a tile leave as whole 512-byte tiles.
#include "fp4.cuh"

namespace fx {

static constexpr int Q_ROWS = 128, Q_COLS = 256, Q_THREADS = 256;

template <int DT>
__device__ __forceinline__ float q_load1(const void *x, long long i) {
  if (DT == FLUX_CUDA_F32) return reinterpret_cast<const float *>(x)[i];
  const uint16_t h = reinterpret_cast<const uint16_t *>(x)[i];
  if (DT == FLUX_CUDA_F16) return __half2float(__ushort_as_half(h));
  return __uint_as_float(static_cast<uint32_t>(h) << 16);
}

template <int DT>
__device__ __forceinline__ void q_expand(uint32_t w, float &lo, float &hi) {
  if (DT == FLUX_CUDA_F16) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w));
    lo = f.x, hi = f.y;
  } else {
    lo = bf16_lo(w), hi = bf16_hi(w);
  }
}

// 16 consecutive elements starting at element i, all in range; ALIGN: bytes the address is a multiple of (16) or 0.
template <int DT, int ALIGN>
__device__ __forceinline__ void q_load16(const void *x, long long i, float (&v)[16]) {
  if (ALIGN == 0) {
#pragma unroll
    for (int k = 0; k < 16; ++k) v[k] = q_load1<DT>(x, i + k);
  } else if (DT == FLUX_CUDA_F32) {
    const float4 *p = reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(x) + i);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float4 f = __ldg(p + k);
      v[4 * k] = f.x, v[4 * k + 1] = f.y, v[4 * k + 2] = f.z, v[4 * k + 3] = f.w;
    }
  } else {
    const uint4 *p = reinterpret_cast<const uint4 *>(reinterpret_cast<const uint16_t *>(x) + i);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const uint4 u = __ldg(p + k);
      q_expand<DT>(u.x, v[8 * k], v[8 * k + 1]);
      q_expand<DT>(u.y, v[8 * k + 2], v[8 * k + 3]);
      q_expand<DT>(u.z, v[8 * k + 4], v[8 * k + 5]);
      q_expand<DT>(u.w, v[8 * k + 6], v[8 * k + 7]);
    }
  }
}

// Codes of 16 columns and the factor byte of their block. For blocks of 32 the two threads of a block exchange their
// maxima, so the whole warp must call this.
template <int BLOCK>
__device__ __forceinline__ uint32_t q_encode(float (&v)[16], float inv_scale, uint2 &codes) {
  uint32_t top = 0;
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    v[k] *= inv_scale;
    top = max(top, __float_as_uint(v[k]) & 0x7FFFFFFFu);  // NaN compares above infinity
  }
  if (BLOCK == 32) top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  const bool bad = top >= 0x7F800000u;
  uint32_t byte;
  if (BLOCK == 32) {
    const int e = static_cast<int>(top >> 23) - 2;
    byte = bad ? 255u : static_cast<uint32_t>(e > 0 ? e : 0);
    const float r = bad ? 0.f : __uint_as_float((254u - byte) << 23);  // 2^-(byte - 127): the quotient is exact
#pragma unroll
    for (int k = 0; k < 16; ++k) v[k] = bad ? 0.f : v[k] * r;
  } else {
    // a / 6 rounded to odd: truncated, with the lowest bit set where something was cut off; rounding that to e4m3 is
    // rounding the exact quotient
    const float a = __uint_as_float(top);
    float q = __fdiv_rz(a, 6.0f);
    if (__fmaf_rn(-q, 6.0f, a) != 0.f) q = __uint_as_float(__float_as_uint(q) | 1u);
    uint16_t e;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(e) : "f"(0.f), "f"(q));
    byte = bad ? 0x7Fu : (e & 0xFFu);
    const float s = bad ? 0.f : fp4_factor<16>(byte);
    const float r = s > 0.f ? __frcp_rn(s) : 0.f;
    // Markstein's correction: with r the correctly rounded reciprocal, fma(fma(-q, s, x), r, q) is the correctly
    // rounded quotient
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const float x = bad ? 0.f : v[k];
      const float q0 = x * r;
      v[k] = __fmaf_rn(__fmaf_rn(-q0, s, x), r, q0);
    }
  }
  float lo[8], hi[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) lo[k] = v[k], hi[k] = v[8 + k];
  codes = make_uint2(fp4_pack8(lo), fp4_pack8(hi));
  return byte;
}

template <int DT, int BLOCK, int ALIGN>
__global__ void __launch_bounds__(Q_THREADS) fp4_quantize_kernel(const void *__restrict__ x, long long ldx, int rows,
                                                                 int cols, float inv_scale, uint8_t *__restrict__ codes,
                                                                 long long pitch, uint8_t *__restrict__ scales,
                                                                 long long chunks, int col_tiles) {
  constexpr int CH = Q_COLS / (4 * BLOCK);  // factor tiles per block of threads
  __shared__ __align__(16) uint8_t fac[CH * 512];
  pdl_launch_dependents();
  const long long rt = blockIdx.x / col_tiles;
  const int ct = blockIdx.x % col_tiles;
  const int cx = threadIdx.x & 15, ry = threadIdx.x >> 4;
  const int here = static_cast<int>(rows - rt * Q_ROWS < Q_ROWS ? rows - rt * Q_ROWS : Q_ROWS);
  const long long c0 = static_cast<long long>(ct) * Q_COLS + cx * 16;
  if (threadIdx.x < CH * 32) reinterpret_cast<uint4 *>(fac)[threadIdx.x] = make_uint4(0, 0, 0, 0);
  __syncthreads();
#pragma unroll 4
  for (int it = 0; it < Q_ROWS / 16; ++it) {
    const int rl = it * 16 + ry;
    if (it * 16 >= here) break;  // uniform in the block
    const long long r = rt * Q_ROWS + rl;
    float v[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) v[k] = 0.f;
    if (rl < here) {
      if (c0 + 16 <= cols) {
        q_load16<DT, ALIGN>(x, r * ldx + c0, v);
      } else {
#pragma unroll
        for (int k = 0; k < 16; ++k)
          if (c0 + k < cols) v[k] = q_load1<DT>(x, r * ldx + c0 + k);
      }
    }
    uint2 cd;
    const uint32_t byte = q_encode<BLOCK>(v, inv_scale, cd);
    if (rl < here) {
      if (c0 / 2 + 8 <= pitch) *reinterpret_cast<uint2 *>(codes + r * pitch + c0 / 2) = cd;
      const int b = cx * 16 / BLOCK;
      if (BLOCK == 16 || !(cx & 1))
        fac[(b >> 2) * 512 + (rl & 31) * 16 + (rl >> 5) * 4 + (b & 3)] = static_cast<uint8_t>(c0 < cols ? byte : 0u);
    }
  }
  __syncthreads();
  const long long chunk = static_cast<long long>(ct) * CH + (threadIdx.x >> 5);
  if (threadIdx.x < CH * 32 && chunk < chunks)
    *reinterpret_cast<uint4 *>(scales + (rt * chunks + chunk) * 512 + (threadIdx.x & 31) * 16) =
        reinterpret_cast<const uint4 *>(fac)[threadIdx.x];
}

int launch_fp4_quantize(const void *x, int dtype, long long ldx, const flux_cuda_fp4 &q, cudaStream_t st) {
  const int col_tiles = (q.cols + Q_COLS - 1) / Q_COLS;
  const long long blocks = fp4_row_tiles(q.rows) * col_tiles;
  const int size = dtype == FLUX_CUDA_F32 ? 4 : 2;
  const bool vec = !(reinterpret_cast<uintptr_t>(x) & 15) && !((ldx * size) & 15);
  uint8_t *codes = static_cast<uint8_t *>(q.codes), *scales = static_cast<uint8_t *>(q.scales);
  const long long pitch = fp4_pitch(q.cols), chunks = fp4_chunks(q.cols, q.format);
  const float inv = 1.0f / q.scale;
#define FX_Q(DT, BL, AL)                                                                                       \
  fp4_quantize_kernel<DT, BL, AL><<<static_cast<unsigned>(blocks), Q_THREADS, 0, st>>>(x, ldx, q.rows, q.cols, inv, codes, \
                                                                                       pitch, scales, chunks, col_tiles)
#define FX_Q2(DT)                                  \
  do {                                             \
    if (q.format == 16) {                          \
      if (vec) FX_Q(DT, 16, 16);                   \
      else FX_Q(DT, 16, 0);                        \
    } else {                                       \
      if (vec) FX_Q(DT, 32, 16);                   \
      else FX_Q(DT, 32, 0);                        \
    }                                              \
  } while (0)
  if (dtype == FLUX_CUDA_F32) FX_Q2(FLUX_CUDA_F32);
  else if (dtype == FLUX_CUDA_F16) FX_Q2(FLUX_CUDA_F16);
  else FX_Q2(FLUX_CUDA_BF16);
#undef FX_Q2
#undef FX_Q
  return cudaGetLastError() == cudaSuccess ? 0 : -8;
}

// ------------------------------------------------------------------------------------------------
// The values a 4-bit matrix stands for: the product with the matrix's own scale is rounded to f32 and then to the output
// type, everything else is exact. Same tiling as above; bound by writing the values.
// ------------------------------------------------------------------------------------------------
template <int DT, int BLOCK, int ALIGN>
__global__ void __launch_bounds__(Q_THREADS) fp4_dequantize_kernel(const uint8_t *__restrict__ codes, long long pitch,
                                                                   const uint8_t *__restrict__ scales, long long chunks,
                                                                   int rows, int cols, float scale, void *__restrict__ out,
                                                                   long long ld, int col_tiles, int *sat) {
  constexpr int CH = Q_COLS / (4 * BLOCK);
  __shared__ __align__(16) uint8_t fac[CH * 512];
  pdl_launch_dependents();
  const long long rt = blockIdx.x / col_tiles;
  const int ct = blockIdx.x % col_tiles;
  const int cx = threadIdx.x & 15, ry = threadIdx.x >> 4;
  const int here = static_cast<int>(rows - rt * Q_ROWS < Q_ROWS ? rows - rt * Q_ROWS : Q_ROWS);
  const long long c0 = static_cast<long long>(ct) * Q_COLS + cx * 16;
  const long long chunk = static_cast<long long>(ct) * CH + (threadIdx.x >> 5);
  if (threadIdx.x < CH * 32)
    reinterpret_cast<uint4 *>(fac)[threadIdx.x] =
        chunk < chunks ? __ldg(reinterpret_cast<const uint4 *>(scales + (rt * chunks + chunk) * 512) + (threadIdx.x & 31))
                       : make_uint4(0, 0, 0, 0);
  __syncthreads();
  float mx = 0.f;
  if (c0 < cols) {
#pragma unroll 4
    for (int it = 0; it < Q_ROWS / 16; ++it) {
      const int rl = it * 16 + ry;
      if (rl >= here) break;
      const long long r = rt * Q_ROWS + rl;
      const uint2 cd = __ldg(reinterpret_cast<const uint2 *>(codes + r * pitch + c0 / 2));
      const int b = cx * 16 / BLOCK;
      const float s = fp4_factor<BLOCK>(fac[(b >> 2) * 512 + (rl & 31) * 16 + (rl >> 5) * 4 + (b & 3)]);
      // code * e4m3 is exact. A power of two may take a code out of the f32 range that a small scale brings back: then
      // the scale comes first.
      const bool scale_first = BLOCK == 32 && fabsf(scale) < 1.0f;
      const float first = scale_first ? scale : s, second = scale_first ? s : scale;
      float v[16];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        uint32_t h[4];
        fp4_unpack8(k ? cd.y : cd.x, h);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h[j]));
          v[8 * k + 2 * j] = f.x * first * second;
          v[8 * k + 2 * j + 1] = f.y * first * second;
        }
      }
      const long long at = r * ld + c0;
      if (ALIGN && c0 + 16 <= cols) {
        if (DT == FLUX_CUDA_F32) {
          float4 *p = reinterpret_cast<float4 *>(reinterpret_cast<float *>(out) + at);
#pragma unroll
          for (int k = 0; k < 4; ++k) p[k] = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
        } else {
          uint4 *p = reinterpret_cast<uint4 *>(reinterpret_cast<uint16_t *>(out) + at);
          uint32_t w[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) w[k] = pack_16x2_t(v[2 * k], v[2 * k + 1], DT == FLUX_CUDA_F16, mx);
          p[0] = make_uint4(w[0], w[1], w[2], w[3]);
          p[1] = make_uint4(w[4], w[5], w[6], w[7]);
        }
      } else {
#pragma unroll
        for (int k = 0; k < 16; ++k)
          if (c0 + k < cols) fp4_store<DT>(out, at + k, v[k], mx);
      }
    }
  }
  sat_report(sat, DT == FLUX_CUDA_F16, mx);
}

int launch_fp4_dequantize(const flux_cuda_fp4 &q, void *out, int dtype, long long ld, int *sat, cudaStream_t st) {
  const int col_tiles = (q.cols + Q_COLS - 1) / Q_COLS;
  const long long blocks = fp4_row_tiles(q.rows) * col_tiles;
  const int size = dtype == FLUX_CUDA_F32 ? 4 : 2;
  const bool vec = !(reinterpret_cast<uintptr_t>(out) & 15) && !((ld * size) & 15);
  const uint8_t *codes = static_cast<const uint8_t *>(q.codes), *scales = static_cast<const uint8_t *>(q.scales);
  const long long pitch = fp4_pitch(q.cols), chunks = fp4_chunks(q.cols, q.format);
#define FX_D(DT, BL, AL)                                                                                                   \
  fp4_dequantize_kernel<DT, BL, AL><<<static_cast<unsigned>(blocks), Q_THREADS, 0, st>>>(codes, pitch, scales, chunks, q.rows, \
                                                                                         q.cols, q.scale, out, ld, col_tiles, sat)
#define FX_D2(DT)                                  \
  do {                                             \
    if (q.format == 16) {                          \
      if (vec) FX_D(DT, 16, 16);                   \
      else FX_D(DT, 16, 0);                        \
    } else {                                       \
      if (vec) FX_D(DT, 32, 16);                   \
      else FX_D(DT, 32, 0);                        \
    }                                              \
  } while (0)
  if (dtype == FLUX_CUDA_F32) FX_D2(FLUX_CUDA_F32);
  else if (dtype == FLUX_CUDA_F16) FX_D2(FLUX_CUDA_F16);
  else FX_D2(FLUX_CUDA_BF16);
#undef FX_D2
#undef FX_D
  return cudaGetLastError() == cudaSuccess ? 0 : -8;
}

}  // namespace fx
