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
// Bound by memory: every element is read once, 0.56 bytes per element are written. A thread owns 16 consecutive columns of
// the four rows r, r + 32, r + 64, r + 96 of a 128-row tile: a whole block of 16 (half a block of 32) per row in registers,
// 128 to 256 bytes of loads in flight per thread, and of the factors exactly what lies in one 16-byte piece of a factor
// tile, so the four lanes of a chunk put a piece together with shuffles and store it whole. No shared memory, no barrier:
// rows beyond the last cost one predicate, which keeps a single token at the price of a launch.
#include <math.h>

#include "fp4.cuh"
#include "launch.cuh"

namespace fx {

static constexpr int Q_COLS = 256;  // columns per block of threads: 16 threads of 16
static constexpr int Q_THREADS = 128;  // 8 rows r per block of threads, 32 rows of the matrix

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

// 16 consecutive elements as 32-bit words. From a 32-byte aligned address in loads of 32 bytes; from any other one in the
// aligned 16-byte pieces that hold them, shifted into place.
template <int DT>
struct Raw16 {
  static constexpr int N = DT == FLUX_CUDA_F32 ? 16 : 8;
  uint32_t w[N];
};
template <int DT>
__device__ __forceinline__ void q_load_aligned(const char *p, Raw16<DT> &raw) {
#pragma unroll
  for (int k = 0; k < Raw16<DT>::N; k += 8)
    asm volatile("ld.global.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(raw.w[k]), "=r"(raw.w[k + 1]), "=r"(raw.w[k + 2]), "=r"(raw.w[k + 3]), "=r"(raw.w[k + 4]),
                   "=r"(raw.w[k + 5]), "=r"(raw.w[k + 6]), "=r"(raw.w[k + 7])
                 : "l"(p + k * 4));
}
// The pieces around [p, p + 16 elements): N / 4 + 1 of them, the last one only if p is not 16-byte aligned.
template <int DT>
__device__ __forceinline__ void q_load_shifted(const char *p, Raw16<DT> &raw) {
  constexpr int N = Raw16<DT>::N;
  const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p)) & 15;
  const uint4 *g = reinterpret_cast<const uint4 *>(p - off);
  uint32_t t[N + 4];
#pragma unroll
  for (int k = 0; k <= N / 4; ++k) {
    uint4 u = make_uint4(0, 0, 0, 0);
    if (k < N / 4 || off) u = __ldg(g + k);
    t[4 * k] = u.x, t[4 * k + 1] = u.y, t[4 * k + 2] = u.z, t[4 * k + 3] = u.w;
  }
#pragma unroll
  for (int k = 0; k < N + 2; ++k) t[k] = off & 8 ? t[k + 2] : t[k];
#pragma unroll
  for (int k = 0; k < N + 1; ++k) t[k] = off & 4 ? t[k + 1] : t[k];
#pragma unroll
  for (int k = 0; k < N; ++k) raw.w[k] = DT == FLUX_CUDA_F32 ? t[k] : __funnelshift_r(t[k], t[k + 1], (off & 2) * 8);
}
template <int DT>
__device__ __forceinline__ void q_expand16(const Raw16<DT> &raw, float (&v)[16]) {
#pragma unroll
  for (int k = 0; k < 16; ++k)
    if (DT == FLUX_CUDA_F32) v[k] = __uint_as_float(raw.w[k % Raw16<DT>::N]);
    else if (!(k & 1)) q_expand<DT>(raw.w[k / 2], v[k], v[k + 1]);
}

// The largest of three magnitudes, NaN if one of them is.
__device__ __forceinline__ float max3_abs(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(fabsf(a)), "f"(fabsf(b)), "f"(fabsf(c)));
  return r;
}

// Codes of 16 columns and the factor byte of their block. inv_scale is a power of two, and the division by the matrix's scale
// is exact whatever f32 makes of it: whether a block is finite is asked of x itself, and a quotient that f32 cannot hold is
// either kept at the largest f32 (beyond it) or never formed (below it). For blocks of 32 the two threads of a block exchange
// their maxima, so the whole warp must call this.
template <int BLOCK>
__device__ __forceinline__ uint32_t q_encode(float (&v)[16], float inv_scale, uint2 &codes) {
  float a = fabsf(v[0]);
#pragma unroll
  for (int k = 1; k < 15; k += 2) a = max3_abs(a, v[k], v[k + 1]);
  uint32_t top = __float_as_uint(max3_abs(a, a, v[15])) & 0x7FFFFFFFu;  // NaN compares above infinity
  if (BLOCK == 32) top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  const bool bad = top >= 0x7F800000u;
  if (bad) {
#pragma unroll
    for (int k = 0; k < 16; ++k) v[k] = 0.f;
  }
  uint32_t byte;
  float q[16];
  if (BLOCK == 32) {
    // the factor's and the scale's powers of two in one, 2^-shift, so that the quotient is exact. (The exponent of a subnormal
    // maximum is that of its product with 2^24; where no scale raises it, the factor is the least one anyway.)
    const int k = 127 - static_cast<int>(__float_as_uint(inv_scale) >> 23);  // the scale is 2^k
    int e = static_cast<int>(top >> 23) - 2;
    if (e < 0 && k < 0) e = static_cast<int>(__float_as_uint(__uint_as_float(top) * 0x1p24f) >> 23) - 26;
    e = top == 0 ? 0 : min(max(e - k, 0), 254);
    byte = bad ? 255u : static_cast<uint32_t>(e);
    const int shift = 127 - e - k;  // -125 .. 151
    float r = bad ? 0.f : __uint_as_float(static_cast<uint32_t>(min(shift, 127) + 127) << 23);
    if (shift > 127) {  // only tiny x: nothing overflows on the way
      const float rest = __uint_as_float(static_cast<uint32_t>(shift) << 23);
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] *= rest;
    }
    const uint64_t r2 = f2_pack(r, r);
#pragma unroll
    for (int i = 0; i < 16; i += 2) f2_unpack(f2_mul(f2_pack(v[i], v[i + 1]), r2), q[i], q[i + 1]);
  } else {
    a = __uint_as_float(bad ? 0u : top);
    if (inv_scale != 1.0f) {
      a *= inv_scale;
#pragma unroll
      for (int k = 0; k < 16; ++k) v[k] *= inv_scale;
      if (a > 3.402823466e38f) {  // the largest factor, and codes of 6 for what is beyond f32
        a = 3.402823466e38f;
#pragma unroll
        for (int k = 0; k < 16; ++k) v[k] = fminf(fmaxf(v[k], -a), a);
      }
      // A quotient below the normal range is not exact, but its block has the factor 0 or its code is 0.
    }
    // a / 6 rounded to odd (truncated, with the lowest bit set where something was cut off): rounding that to e4m3 is
    // rounding the exact quotient
    float t = a * (1.0f / 6.0f);  // within one unit of a / 6; the residual's sign tells on which side
    const float rest = __fmaf_rn(-t, 6.0f, a);
    uint32_t bits = __float_as_uint(t);
    if (rest < 0.f) bits -= 1;
    if (rest != 0.f) bits |= 1;
    t = __uint_as_float(bits);
    uint16_t e;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(e) : "f"(0.f), "f"(t));
    byte = bad ? 0x7Fu : (e & 0xFFu);
    const float s = fp4_factor<16>(e & 0xFFu);
    float r = 0.f;
    if (s > 0.f) {  // one Newton step: the correctly rounded reciprocal for every one of the 126 factors
      asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
      r = __fmaf_rn(__fmaf_rn(-s, r, 1.0f), r, r);
    }
    // Markstein's correction: with r the correctly rounded reciprocal, fma(fma(-q, s, x), r, q) is the correctly
    // rounded quotient
    const uint64_t r2 = f2_pack(r, r), s2 = f2_pack(-s, -s);
#pragma unroll
    for (int k = 0; k < 16; k += 2) {
      const uint64_t x2 = f2_pack(v[k], v[k + 1]), q2 = f2_mul(x2, r2);
      f2_unpack(f2_fma(f2_fma(q2, s2, x2), r2, q2), q[k], q[k + 1]);
    }
  }
  float lo[8], hi[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) lo[k] = q[k], hi[k] = q[8 + k];
  codes = make_uint2(fp4_pack8(lo), fp4_pack8(hi));
  return byte;
}

// VEC: x and its row pitch are multiples of 32 bytes. Grid: [row tiles][4 groups of 8 rows r][column tiles].
template <int DT, int BLOCK, bool VEC>
__global__ void __launch_bounds__(Q_THREADS) fp4_quantize_kernel(const void *__restrict__ x, long long ldx, int rows,
                                                                 int cols, float inv_scale, uint8_t *__restrict__ codes,
                                                                 long long pitch, uint8_t *__restrict__ scales,
                                                                 long long chunks, int col_tiles) {
  pdl_launch_dependents();
  const int ct = blockIdx.x % col_tiles, rg = blockIdx.x / col_tiles % 4;
  const long long rt = blockIdx.x / col_tiles / 4;
  const int cx = threadIdx.x & 15, r32 = rg * 8 + (threadIdx.x >> 4);
  const long long c0 = static_cast<long long>(ct) * Q_COLS + cx * 16, r0 = rt * 128 + r32;
  const char *base = static_cast<const char *>(x), *end = base + ((rows - 1) * ldx + cols) * FP4_SIZE<DT>;
  Raw16<DT> raw[4];
  bool whole[4];  // all 16 elements are in `raw`
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const char *p = base + ((r0 + 32 * q) * ldx + c0) * FP4_SIZE<DT>;
    whole[q] = r0 + 32 * q < rows && c0 + 16 <= cols;
    if (VEC) {
      if (whole[q]) q_load_aligned<DT>(p, raw[q]);
    } else {
      // the 16-byte pieces around the elements must lie inside the matrix themselves
      const uintptr_t lo = reinterpret_cast<uintptr_t>(p) & ~uintptr_t(15);
      whole[q] = whole[q] && lo >= reinterpret_cast<uintptr_t>(base) &&
                 ((reinterpret_cast<uintptr_t>(p) + 16 * FP4_SIZE<DT> + 15) & ~uintptr_t(15)) <= reinterpret_cast<uintptr_t>(end);
      if (whole[q]) q_load_shifted<DT>(p, raw[q]);
    }
  }
  uint32_t word[4];  // the factors of this lane's chunk of four blocks
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    word[q] = 0;
    const bool live = r0 + 32 * q < rows;
    if (!__any_sync(0xffffffffu, live)) continue;
    float v[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) v[k] = 0.f;
    if (live) {
      if (whole[q]) {
        q_expand16<DT>(raw[q], v);
      } else {
        const long long at = (r0 + 32 * q) * ldx + c0;
#pragma unroll
        for (int k = 0; k < 16; ++k)
          if (c0 + k < cols) v[k] = q_load1<DT>(x, at + k);
      }
    }
    uint2 cd;
    uint32_t byte = q_encode<BLOCK>(v, inv_scale, cd);
    if (live && c0 / 2 + 8 <= pitch) *reinterpret_cast<uint2 *>(codes + (r0 + 32 * q) * pitch + c0 / 2) = cd;
    if (c0 >= cols) byte = 0;
    if (BLOCK == 16) {  // lanes 4 i .. 4 i + 3 hold the four blocks of a chunk
      byte |= __shfl_xor_sync(0xffffffffu, byte, 1) << 8;
      byte |= __shfl_xor_sync(0xffffffffu, byte, 2) << 16;
    } else {  // lanes 8 i, + 2, + 4, + 6
      byte |= __shfl_xor_sync(0xffffffffu, byte, 2) << 8;
      byte |= __shfl_xor_sync(0xffffffffu, byte, 4) << 16;
    }
    word[q] = byte;
  }
  const long long chunk = c0 / (4 * BLOCK);
  if (!(cx & (BLOCK == 16 ? 3 : 7)) && chunk < chunks)
    *reinterpret_cast<uint4 *>(scales + (rt * chunks + chunk) * 512 + r32 * 16) = make_uint4(word[0], word[1], word[2], word[3]);
}

int launch_fp4_quantize(const void *x, int dtype, long long ldx, const flux_cuda_fp4 &q, cudaStream_t st) {
  const int col_tiles = static_cast<int>((q.cols + (Q_COLS - 1LL)) / Q_COLS);
  const long long blocks = fp4_row_tiles(q.rows) * 4 * col_tiles;
  const int size = dtype == FLUX_CUDA_F32 ? 4 : 2;
  const bool vec = !(reinterpret_cast<uintptr_t>(x) & 31) && !((ldx * size) & 31);
  uint8_t *codes = static_cast<uint8_t *>(q.codes), *scales = static_cast<uint8_t *>(q.scales);
  const long long pitch = fp4_pitch(q.cols), chunks = fp4_chunks(q.cols, q.format);
  const float inv = 1.0f / q.scale;
  PdlOff no_overlap;  // the kernels do not wait for a predecessor themselves
  const dim3 grid(static_cast<unsigned>(blocks)), threads(Q_THREADS);
  cudaError_t e;
#define FX_Q(DT, BL, AL) \
  e = launch_kernel(fp4_quantize_kernel<DT, BL, AL>, grid, threads, 0, st, 1, x, ldx, q.rows, q.cols, inv, codes, pitch, scales, chunks, col_tiles)
#define FX_Q2(DT)                                  \
  do {                                             \
    if (q.format == 16) {                          \
      if (vec) FX_Q(DT, 16, true);                 \
      else FX_Q(DT, 16, false);                    \
    } else {                                       \
      if (vec) FX_Q(DT, 32, true);                 \
      else FX_Q(DT, 32, false);                    \
    }                                              \
  } while (0)
  if (dtype == FLUX_CUDA_F32) FX_Q2(FLUX_CUDA_F32);
  else if (dtype == FLUX_CUDA_F16) FX_Q2(FLUX_CUDA_F16);
  else FX_Q2(FLUX_CUDA_BF16);
#undef FX_Q2
#undef FX_Q
  return e;
}

// ------------------------------------------------------------------------------------------------
// The values a 4-bit matrix stands for, rounded once. Same tiling as above; bound by writing the values.
//
// PLAIN scales are 0 and the normal powers of two: code * factor * scale in two multiplications is exact, or, for results
// below f32's normal range, rounded once more only where a 16-bit type has 0 anyway. Under any other scale the product has
// up to 30 bits, and rounding it to f32 on the way to a 16-bit type may put it on the middle between two values that it is
// not on. It is rounded to odd then (truncated, with the lowest bit set where something was cut off), which later roundings to
// fewer bits cannot tell from the exact product. The scale's power of two stays out of that and joins the factor's.
// Measured at 9728 x 9216: to bf16 38.6 us (37.0 under a plain scale), blocks of 32 to f16 42.5 (36.8); f32 needs no second
// rounding: 28.7 us at 4096 x 9216 (29.9).
// ------------------------------------------------------------------------------------------------
struct DqScale {
  float scale, mant;  // scale = mant * 2^exp with 1 <= |mant| < 2
  int exp;
};
// Two products a b rounded to odd; minus_b is -b.
__device__ __forceinline__ void dq_odd(uint64_t a, uint64_t b, uint64_t minus_b, float &lo, float &hi) {
  uint64_t p;
  asm("mul.rz.f32x2 %0, %1, %2;" : "=l"(p) : "l"(a), "l"(b));
  float cut_lo, cut_hi;
  f2_unpack(p, lo, hi);
  f2_unpack(f2_fma(a, minus_b, p), cut_lo, cut_hi);  // exact
  if (cut_lo != 0.f) lo = __uint_as_float(__float_as_uint(lo) | 1u);
  if (cut_hi != 0.f) hi = __uint_as_float(__float_as_uint(hi) | 1u);
}
// value * mant * 2^k where that may be no normal f32.
template <int DT>
__device__ __noinline__ float dq_far(float value, float mant, int k) {
  const double d = static_cast<double>(value) * mant * __longlong_as_double(static_cast<long long>(k + 1023) << 52);  // exact
  if (DT == FLUX_CUDA_F32) return __double2float_rn(d);
  const float f = __double2float_rz(d);
  return static_cast<double>(f) == d ? f : __uint_as_float(__float_as_uint(f) | 1u);
}
// Eight codes under a factor's byte as f32 values that are to be rounded to the type.
template <int DT, int BLOCK, bool PLAIN>
__device__ __forceinline__ void dq_values(uint32_t c, uint32_t byte, const DqScale &S, float *v) {
  uint32_t h[4];
  fp4_unpack8(c, h);
  const float s = fp4_factor<BLOCK>(byte);
  if (PLAIN) {
    // code * e4m3 is exact. A power of two may take a code out of the f32 range that a small scale brings back: then the
    // scale comes first.
    const bool scale_first = BLOCK == 32 && fabsf(S.scale) < 1.0f;
    const float first = scale_first ? S.scale : s, second = scale_first ? s : S.scale;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h[j]));
      v[2 * j] = f.x * first * second;
      v[2 * j + 1] = f.y * first * second;
    }
    return;
  }
  const float factor = BLOCK == 16 || byte == 255 ? s : 1.0f;
  int k = BLOCK == 16 || byte == 255 ? S.exp : S.exp + static_cast<int>(byte) - 127;
  if (!(c & 0x77777777u)) k = 0;  // zeros, those past the end of the matrix among them
  if (k >= -100 && k <= 110) {    // mant * code (* e4m3) is within 2^-10 .. 2^13: normal products, and exact rests of them
    const float two = factor * __uint_as_float(static_cast<uint32_t>(k + 127) << 23);
    const uint64_t two2 = f2_pack(two, two), mant2 = f2_pack(S.mant, S.mant), minus2 = f2_pack(-S.mant, -S.mant);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h[j]));
      const uint64_t value = f2_mul(f2_pack(f.x, f.y), two2);
      if (DT == FLUX_CUDA_F32) f2_unpack(f2_mul(value, mant2), v[2 * j], v[2 * j + 1]);
      else dq_odd(value, mant2, minus2, v[2 * j], v[2 * j + 1]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h[j / 2]));
      v[j] = dq_far<DT>((j & 1 ? f.y : f.x) * factor, S.mant, k);
    }
  }
}

template <int DT>
struct OutElement {
  using T = uint16_t;
};
template <>
struct OutElement<FLUX_CUDA_F32> {
  using T = uint32_t;
};

// VEC: out and its row pitch are multiples of 32 bytes: 16 columns per thread in stores of 32 bytes. Otherwise the lanes of
// a warp store neighbouring columns, so that the stores of an odd pitch still fill whole sectors.
template <int DT, int BLOCK, bool VEC, bool PLAIN>
__global__ void __launch_bounds__(Q_THREADS) fp4_dequantize_kernel(const uint8_t *__restrict__ codes, long long pitch,
                                                                   const uint8_t *__restrict__ scales, long long chunks,
                                                                   int rows, int cols, DqScale S, void *__restrict__ out,
                                                                   long long ld, int col_tiles, int *sat) {
  pdl_launch_dependents();
  const int ct = blockIdx.x % col_tiles, rg = blockIdx.x / col_tiles % 4;
  const long long rt = blockIdx.x / col_tiles / 4;
  const int cx = threadIdx.x & 15, r32 = rg * 8 + (threadIdx.x >> 4);
  const long long c0 = static_cast<long long>(ct) * Q_COLS + cx * 16, r0 = rt * 128 + r32;
  uint2 cd[4];
#pragma unroll
  for (int q = 0; q < 4; ++q)
    cd[q] = c0 / 2 + 8 <= pitch && r0 + 32 * q < rows
                ? __ldg(reinterpret_cast<const uint2 *>(codes + (r0 + 32 * q) * pitch + c0 / 2))
                : make_uint2(0, 0);
  const long long chunk = c0 / (4 * BLOCK);
  uint4 f4 = make_uint4(0, 0, 0, 0);
  if (chunk < chunks && r0 < rows) f4 = __ldg(reinterpret_cast<const uint4 *>(scales + (rt * chunks + chunk) * 512 + r32 * 16));
  const int sh = (cx * 16 / BLOCK & 3) * 8;
  const uint32_t fw[4] = {f4.x >> sh, f4.y >> sh, f4.z >> sh, f4.w >> sh};
  float mx = 0.f;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const long long r = r0 + 32 * q;
    const uint32_t byte = fw[q] & 0xFFu;
    float top = 0.f;
    if (VEC && c0 + 16 <= cols) {
      if (r >= rows) continue;
      float v[16];
      dq_values<DT, BLOCK, PLAIN>(cd[q].x, byte, S, v);
      dq_values<DT, BLOCK, PLAIN>(cd[q].y, byte, S, v + 8);
      char *p = reinterpret_cast<char *>(out) + (r * ld + c0) * FP4_SIZE<DT>;
      uint32_t w[Raw16<DT>::N];
#pragma unroll
      for (int k = 0; k < Raw16<DT>::N; ++k)
        w[k] = DT == FLUX_CUDA_F32 ? __float_as_uint(v[k]) : pack_16x2_t(v[2 * k & 15], v[2 * k + 1 & 15], DT == FLUX_CUDA_F16, mx);
#pragma unroll
      for (int k = 0; k < Raw16<DT>::N; k += 8)
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p + k * 4), "r"(w[k]), "r"(w[k + 1]),
                     "r"(w[k + 2]), "r"(w[k + 3]), "r"(w[k + 4]), "r"(w[k + 5]), "r"(w[k + 6]), "r"(w[k + 7])
                     : "memory");
    } else if (VEC) {
      if (r >= rows || c0 >= cols) continue;
      float v[16];
      dq_values<DT, BLOCK, PLAIN>(cd[q].x, byte, S, v);
      dq_values<DT, BLOCK, PLAIN>(cd[q].y, byte, S, v + 8);
#pragma unroll
      for (int k = 0; k < 16; ++k)
        if (c0 + k < cols) fp4_store<DT>(out, r * ld + c0 + k, v[k], mx);
    } else {
      // through shared memory, so that the lanes of a warp store neighbouring elements of a row
      using E = typename OutElement<DT>::T;
      __shared__ __align__(16) E stage[Q_THREADS / 32][2][Q_COLS];
      float v[16];
      dq_values<DT, BLOCK, PLAIN>(cd[q].x, byte, S, v);
      dq_values<DT, BLOCK, PLAIN>(cd[q].y, byte, S, v + 8);
      const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
      uint4 *mine = reinterpret_cast<uint4 *>(&stage[warp][lane >> 4][cx * 16]);
      uint32_t w[Raw16<DT>::N];
#pragma unroll
      for (int k = 0; k < Raw16<DT>::N; ++k)
        w[k] = DT == FLUX_CUDA_F32 ? __float_as_uint(v[k]) : pack_16x2_t(v[2 * k & 15], v[2 * k + 1 & 15], DT == FLUX_CUDA_F16, top);
      __syncwarp();
#pragma unroll
      for (int k = 0; k < Raw16<DT>::N / 4; ++k) mine[k] = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
      __syncwarp();
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const long long row = r - (threadIdx.x >> 4 & 1) + h, c = static_cast<long long>(ct) * Q_COLS + lane;
        E *p = reinterpret_cast<E *>(out) + row * ld + c;
#pragma unroll
        for (int k = 0; k < Q_COLS / 32; ++k)
          if (row < rows && c + 32 * k < cols) p[32 * k] = stage[warp][h][32 * k + lane];
      }
      if (r < rows && c0 < cols) mx = fmaxf(mx, top);
    }
  }
  sat_report(sat, DT == FLUX_CUDA_F16, mx);
}

int launch_fp4_dequantize(const flux_cuda_fp4 &q, void *out, int dtype, long long ld, int *sat, cudaStream_t st) {
  const int col_tiles = static_cast<int>((q.cols + (Q_COLS - 1LL)) / Q_COLS);
  const long long blocks = fp4_row_tiles(q.rows) * 4 * col_tiles;
  const int size = dtype == FLUX_CUDA_F32 ? 4 : 2;
  const bool vec = !(reinterpret_cast<uintptr_t>(out) & 31) && !((ld * size) & 31);
  const uint8_t *codes = static_cast<const uint8_t *>(q.codes), *scales = static_cast<const uint8_t *>(q.scales);
  const long long pitch = fp4_pitch(q.cols), chunks = fp4_chunks(q.cols, q.format);
  DqScale S = {q.scale, 0.f, 0};
  bool plain = true;
  if (q.scale != 0.f) {
    S.mant = 2.0f * frexpf(q.scale, &S.exp), --S.exp;
    plain = fabsf(S.mant) == 1.0f && S.exp >= -126;
  }
  PdlOff no_overlap;
  const dim3 grid(static_cast<unsigned>(blocks)), threads(Q_THREADS);
  cudaError_t e;
#define FX_D(DT, BL, AL, PL)                                                                                                 \
  e = launch_kernel(fp4_dequantize_kernel<DT, BL, AL, PL>, grid, threads, 0, st, 1, codes, pitch, scales, chunks, q.rows, q.cols, S, \
                    out, ld, col_tiles, sat)
#define FX_D1(DT, BL, AL)            \
  do {                               \
    if (plain) FX_D(DT, BL, AL, true); \
    else FX_D(DT, BL, AL, false);    \
  } while (0)
#define FX_D2(DT)                   \
  do {                              \
    if (q.format == 16) {           \
      if (vec) FX_D1(DT, 16, true); \
      else FX_D1(DT, 16, false);    \
    } else {                        \
      if (vec) FX_D1(DT, 32, true); \
      else FX_D1(DT, 32, false);    \
    }                               \
  } while (0)
  if (dtype == FLUX_CUDA_F32) FX_D2(FLUX_CUDA_F32);
  else if (dtype == FLUX_CUDA_F16) FX_D2(FLUX_CUDA_F16);
  else FX_D2(FLUX_CUDA_BF16);
#undef FX_D2
#undef FX_D1
#undef FX_D
  return e;
}

}  // namespace fx
