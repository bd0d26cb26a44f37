// A few rows of f32 / f16 / bf16 times a 4-bit matrix: out[m, n] = w.scale * sum_k x[m, k] w[n, k], the activations not
// quantised. The form for single tokens and for the modulation vectors of a schedule; bound by reading the packed
// weights once (0.56 bytes per weight).
//
// One warp takes the four weight rows r, r + 32, r + 64, r + 96 of a 128-row tile, because one 16-byte piece of a factor
// tile holds the factors of exactly these rows for four blocks; a lane takes 32 consecutive codes (16 bytes) of each per
// step, so a step of the warp covers 1024 codes of four rows. x is laid out once per block in shared memory as f32, in
// the order in which the lanes read it ([piece of 4][lane]: no bank conflicts), for up to four rows of x at a time; more
// rows are further blocks, whose weights then come from L2. Sums are f32: per lane over its codes, then over the warp.
#include "fp4.cuh"

namespace fx {

static constexpr int V_THREADS = 512;
static constexpr int V_SMEM_MAX = 200 * 1024;

__device__ __forceinline__ float v_load(const void *x, int dt, long long i) {
  if (dt == FLUX_CUDA_F32) return reinterpret_cast<const float *>(x)[i];
  const uint16_t h = reinterpret_cast<const uint16_t *>(x)[i];
  return dt == FLUX_CUDA_F16 ? __half2float(__ushort_as_half(h)) : __uint_as_float(static_cast<uint32_t>(h) << 16);
}

// S rows of x per block (blockIdx.y * S ...). STAGED: x lies in shared memory; otherwise (K too long) it is read from
// global memory.
template <int S, int BLOCK, bool STAGED>
__global__ void __launch_bounds__(V_THREADS) gemv_fp4_kernel(const void *__restrict__ x, int x_dt, long long ldx, int rows,
                                                             const uint8_t *__restrict__ codes, long long pitch,
                                                             const uint8_t *__restrict__ scales, long long chunks,
                                                             float scale, int N, int K, void *__restrict__ out, int dt,
                                                             long long ld, int *sat) {
  extern __shared__ float4 xs[];  // [S][steps][8][32]
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int steps = (K + 1023) / 1024;
  const int m0 = blockIdx.y * S;
  if (STAGED) {
    float *f = reinterpret_cast<float *>(xs);
    for (int i = threadIdx.x; i < S * steps * 1024; i += V_THREADS) {
      // destination order: [row][step][piece j][lane][4]
      const int e = i & 3, l = (i >> 2) & 31, j = (i >> 7) & 7, st = (i >> 10) % steps, s = (i >> 10) / steps;
      const long long k = static_cast<long long>(st) * 1024 + l * 32 + j * 4 + e;
      f[i] = (m0 + s < rows && k < K) ? v_load(x, x_dt, (m0 + s) * ldx + k) : 0.f;
    }
    __syncthreads();
  }
  const long long quads = (static_cast<long long>(N) + 127) / 128 * 32;
  float mx = 0.f;
  for (long long t = blockIdx.x * static_cast<long long>(V_THREADS / 32) + (threadIdx.x >> 5); t < quads;
       t += static_cast<long long>(gridDim.x) * (V_THREADS / 32)) {
    const long long n0 = t / 32 * 128 + t % 32;  // rows n0 + 32 q
    if (n0 >= N) continue;
    float acc[4][S];
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int s = 0; s < S; ++s) acc[q][s] = 0.f;
    for (int st = 0; st < steps; ++st) {
      const long long byte = st * 512LL + lane * 16;
      uint4 w[4];
#pragma unroll
      for (int q = 0; q < 4; ++q)
        w[q] = (byte < pitch && n0 + 32 * q < N) ? __ldg(reinterpret_cast<const uint4 *>(codes + (n0 + 32 * q) * pitch + byte))
                                                 : make_uint4(0, 0, 0, 0);
      // 32 codes are two blocks of 16 (half of a factor word) or one of 32 (a quarter)
      const long long blk = (st * 1024LL + lane * 32) / BLOCK;
      uint4 sf = make_uint4(0, 0, 0, 0);
      if (blk / 4 < chunks)
        sf = __ldg(reinterpret_cast<const uint4 *>(scales + ((n0 / 128) * chunks + blk / 4) * 512 + (n0 % 32) * 16));
      const int sh = static_cast<int>(blk & 3) * 8;
      const uint32_t fw[4] = {sf.x >> sh, sf.y >> sh, sf.z >> sh, sf.w >> sh};
#pragma unroll
      for (int half = 0; half < 2; ++half) {  // 16 codes each
        float4 xv[S][4];
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (STAGED) {
              xv[s][j] = xs[((s * steps + st) * 8 + half * 4 + j) * 32 + lane];
            } else {
              float e[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const long long k = st * 1024LL + lane * 32 + half * 16 + j * 4 + i;
                e[i] = (m0 + s < rows && k < K) ? v_load(x, x_dt, (m0 + s) * ldx + k) : 0.f;
              }
              xv[s][j] = make_float4(e[0], e[1], e[2], e[3]);
            }
          }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float f = fp4_factor<BLOCK>((BLOCK == 16 ? fw[q] >> (half * 8) : fw[q]) & 0xFFu);
          float part[S];
#pragma unroll
          for (int s = 0; s < S; ++s) part[s] = 0.f;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const uint32_t word = half == 0 ? (c == 0 ? w[q].x : w[q].y) : (c == 0 ? w[q].z : w[q].w);
            uint32_t h[4];
            fp4_unpack8(word, h);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&h[2 * j]));
              const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&h[2 * j + 1]));
#pragma unroll
              for (int s = 0; s < S; ++s) {
                const float4 v = xv[s][2 * c + j];
                part[s] = fmaf(a.x, v.x, part[s]);
                part[s] = fmaf(a.y, v.y, part[s]);
                part[s] = fmaf(b.x, v.z, part[s]);
                part[s] = fmaf(b.y, v.w, part[s]);
              }
            }
          }
#pragma unroll
          for (int s = 0; s < S; ++s) acc[q][s] = fmaf(f, part[s], acc[q][s]);
        }
      }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int s = 0; s < S; ++s) {
        const float v = warp_sum(acc[q][s]) * scale;
        const long long n = n0 + 32 * q;
        if (lane == 0 && n < N && m0 + s < rows) {
          const long long at = (m0 + s) * ld + n;
          if (dt == FLUX_CUDA_F32) fp4_store<FLUX_CUDA_F32>(out, at, v, mx);
          else if (dt == FLUX_CUDA_F16) fp4_store<FLUX_CUDA_F16>(out, at, v, mx);
          else fp4_store<FLUX_CUDA_BF16>(out, at, v, mx);
        }
      }
  }
  sat_report(sat, dt == FLUX_CUDA_F16, mx);
}

template <int S, int BLOCK, bool STAGED>
static cudaError_t v_launch(dim3 grid, size_t smem, cudaStream_t st, const void *x, int x_dt, long long ldx, int rows,
                            const flux_cuda_fp4 &w, void *out, int dt, long long ld, int *sat) {
  if (smem > 48 * 1024) {
    cudaError_t e = cudaFuncSetAttribute(gemv_fp4_kernel<S, BLOCK, STAGED>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         V_SMEM_MAX);
    if (e != cudaSuccess) return e;
  }
  gemv_fp4_kernel<S, BLOCK, STAGED><<<grid, V_THREADS, smem, st>>>(
      x, x_dt, ldx, rows, static_cast<const uint8_t *>(w.codes), fp4_pitch(w.cols),
      static_cast<const uint8_t *>(w.scales), fp4_chunks(w.cols, w.format), w.scale, w.rows, w.cols, out, dt, ld, sat);
  return cudaGetLastError();
}

int launch_gemv_fp4(const void *x, int x_dtype, long long ldx, int rows, const flux_cuda_fp4 &w, void *out, int dtype,
                    long long ld_out, int num_sms, int *sat, cudaStream_t st) {
  const long long steps = (static_cast<long long>(w.cols) + 1023) / 1024;
  int s = rows == 1 ? 1 : rows == 2 ? 2 : 4;
  while (s > 1 && s * steps * 4096 > V_SMEM_MAX) s /= 2;
  const bool staged = s * steps * 4096 <= V_SMEM_MAX;
  const size_t smem = staged ? static_cast<size_t>(s * steps * 4096) : 0;
  const long long warps = fp4_row_tiles(w.rows) * 32;
  const long long want = (warps + V_THREADS / 32 - 1) / (V_THREADS / 32);
  dim3 grid(static_cast<unsigned>(want < num_sms ? want : num_sms), (rows + s - 1) / s);
  cudaError_t e;
#define FX_V(S, ST)                                                                                                     \
  e = w.format == 16 ? v_launch<S, 16, ST>(grid, smem, st, x, x_dtype, ldx, rows, w, out, dtype, ld_out, sat)             \
                     : v_launch<S, 32, ST>(grid, smem, st, x, x_dtype, ldx, rows, w, out, dtype, ld_out, sat)
  if (!staged) FX_V(1, false);
  else if (s == 1) FX_V(1, true);
  else if (s == 2) FX_V(2, true);
  else FX_V(4, true);
#undef FX_V
  return e == cudaSuccess ? 0 : -8;
}

}  // namespace fx
