// Product of two 4-bit matrices on the block-scaled tensor-core path (layout in fp4.cuh):
//
//   out[m, n] = residual[m, n] + gate[n] * (x.scale * w.scale * sum_k x[m, k] w[n, k])
//
// tcgen05.mma kind::mxf4nvf4 / mxf4 multiplies e2m1 operands from shared memory by factors that lie in TMEM and
// accumulates in f32. The weights are the instruction's A operand (128 output columns n on the TMEM lanes), the rows x
// its B operand (output rows m on the TMEM columns): a single token costs a 16-wide instruction instead of a padded
// 128-row tile, and in the epilogue the 32 lanes of a warp hold 32 neighbouring columns of one output row, so plain
// stores are coalesced for any width and pitch.
//
// One k-slice is 256 codes = 128 bytes of a row, the span of the 128-byte swizzle; it is fetched by TMA together with
// the factor tiles it needs, which tcgen05.cp moves from shared memory to TMEM as they lie. What a tensor map reads past
// the end is zero codes and zero factors, so no size needs to be a multiple of anything.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <float.h>
#include <math.h>
#include <string.h>

#include "fp4.cuh"
#include "launch.cuh"

namespace fx {

static constexpr int F_BN = 128;                  // output columns (rows of w) per CTA
static constexpr int F_KB = 128;                  // bytes of a row per k-slice: 256 codes
static constexpr int F_W_BYTES = F_BN * F_KB;     // 16 KB
static constexpr int F_THREADS = 192;             // producer, issuer and four epilogue warps
static constexpr int F2_THREADS = 320;            // the same with eight epilogue warps

struct alignas(64) Fp4GemmParams {
  CUtensorMap tm_w, tm_x;    // codes as bytes [rows, pitch], boxes of 128 bytes, 128-byte swizzle
  CUtensorMap tm_ws, tm_xs;  // factor tiles as u32 [row tiles, chunks, 128]
  int M, N, slices;          // k-slices of 256 codes
  int tiles_m, tiles;
  int splits;                // CTAs of a cluster that share one output tile, each with its part of the k-slices
  float alpha;               // x.scale * w.scale
  float scale_x, scale_w;    // STEPS: the two
  void *out;
  const float *gate, *residual;
  uint32_t pitch, res_pitch;  // bytes from row to row of out and residual
  int *err;
};

// Instruction descriptor of tcgen05.mma with block factors: [4,6) factor id of B, [7,10) A format and [10,12) B format
// (1 = e2m1), [17,23) N >> 3, 23 factor type (0 e4m3, 1 power of two), [27,29) M >> 7, [29,31) factor id of A. Both
// operands K-major. The factor id picks the bytes of a 32-bit TMEM column: 0, or 2 for the upper half of a pair.
__host__ __device__ constexpr uint32_t fp4_idesc(int M, int N, int block, uint32_t id) {
  return (id << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(N >> 3) << 17) | ((block == 32 ? 1u : 0u) << 23) |
         (static_cast<uint32_t>(M >> 7) << 27) | (id << 29);
}

// D[tmem] (+)= A[smem] * B[smem] with block factors in TMEM; 64 codes of K. Issued by ONE thread; PAIR: for both CTAs of a
// pair (M = 256, each CTA holding 128 rows of A and half of the rows of B).
template <int BLOCK, bool PAIR>
__device__ __forceinline__ void fp4_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb,
                                        uint32_t accumulate) {
#define FX_MMA(GROUP, KIND)                                                                              \
  asm volatile(                                                                                          \
      "{\n\t"                                                                                            \
      ".reg .pred p;\n\t"                                                                                \
      "setp.ne.b32 p, %6, 0;\n\t"                                                                        \
      "tcgen05.mma.cta_group::" GROUP ".kind::" KIND " [%0], %1, %2, %3, [%4], [%5], p;\n\t"             \
      "}\n" ::"r"(d),                                                                                    \
      "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate)                                      \
      : "memory")
  if (BLOCK == 16) {
    if (PAIR) FX_MMA("2", "mxf4nvf4.block_scale.scale_vec::4X");
    else FX_MMA("1", "mxf4nvf4.block_scale.scale_vec::4X");
  } else {
    if (PAIR) FX_MMA("2", "mxf4.block_scale.scale_vec::2X");
    else FX_MMA("1", "mxf4.block_scale.scale_vec::2X");
  }
#undef FX_MMA
}

// One 512-byte factor tile from shared memory to four TMEM columns, repeated in the four lane groups.
template <bool PAIR>
__device__ __forceinline__ void fp4_copy_factors(uint32_t taddr, uint64_t sdesc) {
  if (PAIR) asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(sdesc) : "memory");
  else asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(sdesc) : "memory");
}
// Shared-memory descriptor of a factor tile: no swizzle, groups of 8 rows x 16 bytes at a stride of 128 bytes.
__device__ __forceinline__ uint64_t fp4_factor_desc(uint32_t smem_addr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((smem_addr & 0x3FFFF) >> 4);
  d |= static_cast<uint64_t>(128 >> 4) << 16;
  d |= static_cast<uint64_t>(128 >> 4) << 32;
  d |= 1ull << 46;
  return d;
}

// tma_load_2d_pair for three dimensions: into this CTA's shared memory, bytes counted on a barrier of the pair's leader.
__device__ __forceinline__ void tma_load_3d_pair(void *smem_dst, const CUtensorMap *m, uint32_t bar_cluster_addr, int x,
                                                 int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, "
      "%5}], [%2];" ::"r"(smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(bar_cluster_addr), "r"(x), "r"(y), "r"(z)
      : "memory");
}

// Arrival on a barrier of the pair's leader that orders no memory: what it releases is TMEM whose loads have completed. The
// releasing form waits for the epilogue's global stores, a thousand cycles in which the tensor pipe stood still.
__device__ __forceinline__ void mbar_arrive_cluster_relaxed(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// The residual of 16 output rows of this thread's column, requested well before fp4_emit wants it (a load takes most of a
// microsecond, and the stores in between keep the compiler from moving it). Only where there is one.
__device__ __forceinline__ void fp4_residual(float (&v)[16], int rows, const uint8_t *res, uint32_t res_pitch) {
  if (rows >= 16) {
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = __ldcg(reinterpret_cast<const float *>(res + static_cast<uint64_t>(res_pitch) * j));
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j)
      v[j] = j < rows ? __ldcg(reinterpret_cast<const float *>(res + static_cast<uint64_t>(res_pitch) * j)) : 0.f;
  }
}
// What the sums of column n are multiplied by: x.scale * w.scale * gate. STEPS = false: in one step, for calls whose alpha is a
// normal f32 and that have no gate, or alpha = 1. Otherwise the product may be no normal f32 although the result is one;
// it is then three factors that take a sum the same way, so that nothing on the way leaves f32 unless the result does.
// (Sums are 0 or 2^-149 .. 2^128, so powers of two beyond 2^300 need not be told apart.)
// Instances of their own, because the multiplications cost every other call 0.2 - 0.3 us of exposed epilogue, even behind a
// branch (1024 x 6144 x 2560: 13.6 -> 13.9 us).
struct Fp4Factor {
  float a, pre, pre2;
};
template <bool STEPS>
__device__ __forceinline__ Fp4Factor fp4_column(const Fp4GemmParams &P, int n) {
  if (!STEPS) return {P.gate ? P.alpha * P.gate[n] : P.alpha, 1.0f, 1.0f};
  const double t = static_cast<double>(P.scale_x) * P.scale_w * (P.gate ? P.gate[n] : 1.0f);
  const float a = static_cast<float>(t);
  if (t == 0 || !(fabs(t) < __longlong_as_double(0x7FF0000000000000LL)) || (fabsf(a) >= 1.17549435e-38f && fabsf(a) <= 3.402823466e38f))
    return {a, 1.0f, 1.0f};
  const long long bits = __double_as_longlong(t);
  const double mant = __longlong_as_double((bits & 0x800FFFFFFFFFFFFFLL) | 0x3FF0000000000000LL);  // t = mant 2^e
  const int e = min(max(static_cast<int>(bits >> 52 & 0x7FF) - 1023, -300), 300), k = e / 3;
  const auto two = [](int i) { return __uint_as_float(static_cast<uint32_t>(i + 127) << 23); };
  return {static_cast<float>(mant) * two(k), two(k), two(e - 2 * k)};
}
template <bool STEPS>
__device__ __forceinline__ float fp4_scaled(float sum, float pre, float pre2) {
  return STEPS ? sum * pre * pre2 : sum;
}
// Epilogue of 16 output rows of this thread's column n, starting at `out`: f from fp4_column, v the residual if any. Each row's
// address is one multiply-add of its own (row pitches are 32 bits, checked on the host), and whole blocks carry no
// predicates: one warp per scheduler has nothing to hide a chain of 64-bit additions or a branch behind. Checked and
// addressed row by row a store cost 150 cycles, along a chain 32.
template <int DT, bool STEPS>
__device__ __forceinline__ void fp4_emit(const uint32_t (&r)[16], float (&v)[16], bool residual, int rows, uint8_t *out,
                                         uint32_t pitch, const Fp4Factor &f, float &mx) {
  if (residual) {
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = fmaf(f.a, fp4_scaled<STEPS>(__uint_as_float(r[j]), f.pre, f.pre2), v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = f.a * fp4_scaled<STEPS>(__uint_as_float(r[j]), f.pre, f.pre2);
  }
  if (rows >= 16) {
    if (DT == FLUX_CUDA_F32) {
#pragma unroll
      for (int j = 0; j < 16; ++j) *reinterpret_cast<float *>(out + static_cast<uint64_t>(pitch) * j) = v[j];
    } else {
#pragma unroll
      for (int j = 0; j < 16; j += 2) {  // one conversion for two rows
        const uint32_t w = pack_16x2_t(v[j], v[j + 1], DT == FLUX_CUDA_F16, mx);
        *reinterpret_cast<uint16_t *>(out + static_cast<uint64_t>(pitch) * j) = static_cast<uint16_t>(w);
        *reinterpret_cast<uint16_t *>(out + static_cast<uint64_t>(pitch) * (j + 1)) = static_cast<uint16_t>(w >> 16);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (j < rows) fp4_store<DT>(out + static_cast<uint64_t>(pitch) * j, 0, v[j], mx);
  }
}

// The second half of a split tile: rows [m, m_end) of the tile, every fourth one this warp's, four neighbouring columns
// per lane, the parts of up to SP CTAs added in rank order. R rows' parts (16 loads) are requested before the first is
// used: a load from another SM takes most of a microsecond.
template <int DT, int SP, int R, bool STEPS>
__device__ __forceinline__ void fp4_join(uint32_t part, int splits, int m, int m_end, int n, int N, uint8_t *out,
                                         long long pitch, const uint8_t *res, long long res_pitch,
                                         const Fp4GemmParams &P, const Fp4Factor (&early)[4], float &mx) {
  Fp4Factor f[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = STEPS ? early[i] : fp4_column<STEPS>(P, n + i < N ? n + i : N - 1);
  for (; m < m_end; m += 4 * R) {
    float4 v[SP][R];
    float y[R][4];  // the residual, all of it requested before anything is stored (it may be `out`)
#pragma unroll
    for (int s = 0; s < SP; ++s) {
      if (s >= splits) break;
      const uint32_t from = map_to_cta(part, s);
#pragma unroll
      for (int j = 0; j < R; ++j) v[s][j] = ld_cluster_f32x4(from + (m + 4 * j < m_end ? m + 4 * j : m) * F_BN * 4);
    }
#pragma unroll
    for (int j = 0; j < R; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        y[j][i] = res && m + 4 * j < m_end && n + i < N
                      ? __ldcg(reinterpret_cast<const float *>(res + (m + 4 * j) * res_pitch + i * 4))
                      : 0.f;
#pragma unroll
    for (int j = 0; j < R; ++j) {
      float4 a = v[0][j];
#pragma unroll
      for (int s = 1; s < SP; ++s)
        if (s < splits) a.x += v[s][j].x, a.y += v[s][j].y, a.z += v[s][j].z, a.w += v[s][j].w;
      y[j][0] = fmaf(f[0].a, fp4_scaled<STEPS>(a.x, f[0].pre, f[0].pre2), y[j][0]);
      y[j][1] = fmaf(f[1].a, fp4_scaled<STEPS>(a.y, f[1].pre, f[1].pre2), y[j][1]);
      y[j][2] = fmaf(f[2].a, fp4_scaled<STEPS>(a.z, f[2].pre, f[2].pre2), y[j][2]);
      y[j][3] = fmaf(f[3].a, fp4_scaled<STEPS>(a.w, f[3].pre, f[3].pre2), y[j][3]);
    }
#pragma unroll
    for (int j = 0; j < R; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (m + 4 * j < m_end && n + i < N) fp4_store<DT>(out + (m + 4 * j) * pitch, i, y[j][i], mx);
  }
}

// ------------------------------------------------------------------------------------------------
// One CTA per 128 (n) x BM (m) tile, or a cluster of `splits` CTAs that each take a part of K and add their parts in
// rank order through distributed shared memory (no workspace, no atomics, the same bits every time).
// ------------------------------------------------------------------------------------------------
// DEEP (the lowest tiles only): nine k-slices under way and one CTA per SM instead of four and two, for products whose few
// CTAs each have that many slices: 1 x 2560 x 9728 then waits for memory once instead of twice.
template <int BM, int BLOCK, bool DEEP>
struct FCfg {
  static constexpr int CHUNKS = 256 / (4 * BLOCK);  // factor tiles per k-slice
  static constexpr int X_BYTES = BM * F_KB;
  static constexpr int S_BYTES = CHUNKS * 512;
  static constexpr int STAGE_BYTES = F_W_BYTES + X_BYTES + 2 * S_BYTES;
  static constexpr int STAGES = DEEP ? 9 : BM >= 128 ? 3 : 4;
  static constexpr int SMEM = STAGES * STAGE_BYTES + 256;
  static constexpr int SF_COLS = CHUNKS * 4;
  static constexpr int TMEM_COLS = BM + 2 * SF_COLS <= 64 ? 64 : BM + 2 * SF_COLS <= 128 ? 128 : 256;
  static_assert(STAGE_BYTES % 1024 == 0, "the swizzled operands of every stage start on 1024 bytes");
  static_assert(BM * F_BN * 4 <= STAGES * STAGE_BYTES, "the partial tile of a split fits the operand ring");
  static_assert(BM + 2 * SF_COLS <= TMEM_COLS, "accumulator and factors fit the allocation");
};

template <int BM, int BLOCK, int DT, bool DEEP, bool STEPS>
__global__ void __launch_bounds__(F_THREADS, DEEP ? 1 : 2) gemm_fp4_kernel(const __grid_constant__ Fp4GemmParams P) {
  using C = FCfg<BM, BLOCK, DEEP>;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + C::STAGES * C::STAGE_BYTES);
  uint64_t *empty = full + C::STAGES;
  uint64_t *tfull = empty + C::STAGES;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(tfull + 1);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(tfull, 1);
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 1) tmem_alloc(tmem_slot, C::TMEM_COLS);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  const uint32_t sfa = tmem + BM, sfb = sfa + C::SF_COLS;
  pdl_launch_dependents();
  pdl_wait();

  const int rank = blockIdx.x % P.splits, tile = blockIdx.x / P.splits;
  const int m0 = (tile % P.tiles_m) * BM, n0 = (tile / P.tiles_m) * F_BN;
  const int kb0 = static_cast<int>(static_cast<long long>(P.slices) * rank / P.splits);
  const int kb1 = static_cast<int>(static_cast<long long>(P.slices) * (rank + 1) / P.splits);
  auto fail = [&](int code) {
    *abort_flag = 1;
    atomicCAS(P.err, 0, code);
  };

  if (warp == 0) {
    if (lane == 0) {
      for (int kb = kb0; kb < kb1; ++kb) {
        const int i = kb - kb0, s = i % C::STAGES;
        if (!mbar_wait(&empty[s], ((i / C::STAGES) & 1) ^ 1, abort_flag)) {
          fail(KERR_WAIT_EMPTY);
          break;
        }
        uint8_t *sw = smem + s * C::STAGE_BYTES, *sx = sw + F_W_BYTES, *ss = sx + C::X_BYTES;
        mbar_arrive_expect_tx(&full[s], C::STAGE_BYTES);
        tma_load_2d(sw, &P.tm_w, &full[s], kb * F_KB, n0);
        tma_load_2d(sx, &P.tm_x, &full[s], kb * F_KB, m0);
        tma_load_3d(ss, &P.tm_ws, &full[s], 0, kb * C::CHUNKS, n0 / 128);
        tma_load_3d(ss + C::S_BYTES, &P.tm_xs, &full[s], 0, kb * C::CHUNKS, m0 / 128);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    const bool leader = elect_one();
    const uint32_t base = smem_u32(smem);
    bool ok = true;
    for (int kb = kb0; kb < kb1; ++kb) {
      const int i = kb - kb0, s = i % C::STAGES;
      if (!mbar_wait_warp(&full[s], (i / C::STAGES) & 1, abort_flag)) {
        if (lane == 0) fail(KERR_WAIT_FULL);
        ok = false;
        break;
      }
      tc_fence_after_sync();
      const uint32_t sw = base + s * C::STAGE_BYTES, sx = sw + F_W_BYTES, ss = sx + C::X_BYTES;
      const uint64_t wd = make_smem_desc_sw128(sw, 16, 1024), xd = make_smem_desc_sw128(sx, 16, 1024);
      // a 64-row tile may be the upper half of a factor tile's rows: columns 2 and 3 of its four
      const uint32_t sfx = sfb + (BM == 64 ? (m0 & 64) / 32 : 0);
      if (leader) {
#pragma unroll
        for (int c = 0; c < C::CHUNKS; ++c) {
          fp4_copy_factors<false>(sfa + 4 * c, fp4_factor_desc(ss + 512 * c));
          fp4_copy_factors<false>(sfb + 4 * c, fp4_factor_desc(ss + C::S_BYTES + 512 * c));
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int c = BLOCK == 16 ? k : k >> 1;
          const uint32_t id = BLOCK == 16 ? 0 : (k & 1) * 2;
          fp4_mma<BLOCK, false>(tmem, wd + 2 * k, xd + 2 * k, fp4_idesc(F_BN, BM, BLOCK, id), sfa + 4 * c, sfx + 4 * c,
                         (i | k) ? 1u : 0u);
        }
        tc_commit(&empty[s]);
      }
    }
    if (ok && leader) tc_commit(tfull);
    __syncwarp();
  } else {
    const int q = warp & 3;  // the lane group of TMEM this warp may read
    const int nl = q * 32 + lane, n = n0 + nl;
    const int live = P.M - m0 < BM ? P.M - m0 : BM;
    const Fp4Factor f = fp4_column<STEPS>(P, n < P.N ? n : P.N - 1);
    Fp4Factor f4[4];  // of the columns that this lane joins; worked out behind the products where that takes a while
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = n0 + lane * 4 + i;
      if (STEPS) f4[i] = P.splits > 1 ? fp4_column<STEPS>(P, c < P.N ? c : P.N - 1) : f;
    }
    float mx = 0.f;
    const long long pitch = P.pitch, res_pitch = P.res_pitch;
    uint8_t *out = static_cast<uint8_t *>(P.out) + m0 * pitch + n * static_cast<long long>(FP4_SIZE<DT>);
    const uint8_t *res = P.residual ? reinterpret_cast<const uint8_t *>(P.residual) + m0 * res_pitch + n * 4LL : nullptr;
    constexpr int STEP = 16;
    const bool direct = P.splits == 1 && n < P.N;
    float v[16];
    if (direct && res) fp4_residual(v, live, res, P.res_pitch);
    const bool ok = mbar_wait_warp(tfull, 0, abort_flag);
    if (!ok && lane == 0) fail(KERR_WAIT_TMEM_FULL);
    tc_fence_after_sync();
    float *part = reinterpret_cast<float *>(smem);  // every MMA has read its operands by now
    if (ok) {
#pragma unroll 1  // see the pair kernel
      for (int c = 0; c < BM; c += STEP) {
        if (c >= live) break;
        uint32_t r[STEP];
        const uint32_t at = tmem + c + (static_cast<uint32_t>(q * 32) << 16);
        tc_ld_32x16(at, r);
        tc_wait_ld();
        if (P.splits > 1) {
#pragma unroll
          for (int j = 0; j < STEP; ++j) part[(c + j) * F_BN + nl] = __uint_as_float(r[j]);
        } else if (direct) {
          float next[16];
          if (res) fp4_residual(next, live - c - STEP, res + (c + STEP) * res_pitch, P.res_pitch);
          fp4_emit<DT, STEPS>(r, v, res != nullptr, live - c, out + c * pitch, P.pitch, f, mx);
          if (res) {
#pragma unroll
            for (int j = 0; j < STEP; ++j) v[j] = next[j];
          }
        }
      }
    }
    if (P.splits > 1) {
      __syncwarp();
      cluster_sync_all();
      // every CTA of the cluster finishes its share of the tile's rows
      if (ok) {
        const int first = live * rank / P.splits + q, end = live * (rank + 1) / P.splits, nj = n0 + lane * 4;
        const uint32_t mine = smem_u32(part) + lane * 16;
        uint8_t *o = static_cast<uint8_t *>(P.out) + m0 * pitch + nj * static_cast<long long>(FP4_SIZE<DT>);
        const uint8_t *r = P.residual ? reinterpret_cast<const uint8_t *>(P.residual) + m0 * res_pitch + nj * 4LL : nullptr;
        if (P.splits <= 2) fp4_join<DT, 2, 8, STEPS>(mine, P.splits, first, end, nj, P.N, o, pitch, r, res_pitch, P, f4, mx);
        else if (P.splits <= 4) fp4_join<DT, 4, 4, STEPS>(mine, P.splits, first, end, nj, P.N, o, pitch, r, res_pitch, P, f4, mx);
        else fp4_join<DT, 8, 2, STEPS>(mine, P.splits, first, end, nj, P.N, o, pitch, r, res_pitch, P, f4, mx);
      }
    }
    sat_report(P.err + 1, DT == FLUX_CUDA_F16, mx);
  }
  if (P.splits > 1) {
    if (warp < 2) cluster_sync_all();  // the barrier between writing and adding the parts counts every thread
    __syncwarp();
    cluster_sync_all();  // nobody leaves while another CTA still reads its part
  }
  if (*abort_flag) {  // copies still in flight land before the shared memory is given back
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000LL) __nanosleep(1000);
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, C::TMEM_COLS);
  }
}

// ------------------------------------------------------------------------------------------------
// Large products: a pair of CTAs on neighbouring SMs owns a 256 (n) x 256 (m) tile. Each CTA stages its own 128 rows of w
// and half (128) of the rows of x: 38 KB per k-slice and SM for 512 tensor cycles (a 128 x 256 tile per CTA would need 54
// KB). The factors of x are needed in full by both CTAs. Bound by the delivery of operands: shared memory takes 600 cycles of
// the slice (38 KB written, 32 KB read by the multiplications, 6 KB of factors copied, 128 bytes per cycle), and the L2
// delivers 12 TB/s; a slice takes 822 cycles at 1500 MHz and 925 at 1965, so part of it does not follow the SM clock. At
// 8192 x 8192 x 8192 (211 us) a sixth slice under way takes 224, without the factor copies it is 209, without the factors'
// loads 206.
//
// TMEM holds 512 columns: two accumulators of 256 and 48 columns of factors do not fit, so the second accumulator starts
// at column 208 and shares 48 columns with the first. The epilogue takes those columns first and releases the accumulator
// to the next tile's products as soon as it has them in registers; by then the tile before last has long been drained.
// ------------------------------------------------------------------------------------------------
template <int BLOCK>
struct F2Cfg {
  static constexpr int CHUNKS = 256 / (4 * BLOCK);
  static constexpr int X_BYTES = 128 * F_KB;
  static constexpr int S_BYTES = CHUNKS * 512;
  static constexpr int STAGE_BYTES = F_W_BYTES + X_BYTES + 3 * S_BYTES;
  static constexpr int STAGES = BLOCK == 16 ? 5 : 6;
  static constexpr int SMEM = STAGES * STAGE_BYTES + 256;
  static constexpr int SFA = 464, SFB = SFA + 4 * CHUNKS;  // TMEM columns of the factors
  static constexpr int ACC1 = 208, SHARED = 48;
  static_assert(STAGE_BYTES % 1024 == 0 && SMEM <= 232448, "stages are aligned and fit");
  static_assert(SFB + 8 * CHUNKS <= 512 && ACC1 + 256 <= SFA && ACC1 + SHARED == 256, "TMEM columns");
};

template <int BLOCK, int DT, bool STEPS>
__global__ void __launch_bounds__(F2_THREADS, 1) gemm2_fp4_kernel(const __grid_constant__ Fp4GemmParams P) {
  using C = F2Cfg<BLOCK>;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + C::STAGES * C::STAGE_BYTES);  // used in the leader only
  uint64_t *empty = full + C::STAGES;                                                // both CTAs
  uint64_t *tfull = empty + C::STAGES;                                               // both CTAs
  uint64_t *drained = tfull + 2;  // leader only, 16 arrivals: the shared columns of a tile are in registers
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drained + 1);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int pair = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(&tfull[0], 1);
    mbar_init(&tfull[1], 1);
    mbar_init(drained, 16);
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 1) tmem_alloc_pair(tmem_slot, 512);
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  pdl_launch_dependents();
  pdl_wait();
  auto fail = [&](int code) {
    *abort_flag = 1;
    atomicCAS(P.err, 0, code);
  };

  if (warp == 0) {
    if (lane == 0) {
      uint32_t it = 0;
      bool ok = true;
      for (int tile = pair; ok && tile < P.tiles; tile += num_pairs) {
        const int m0 = (tile % P.tiles_m) * 256, n0 = (tile / P.tiles_m) * 256 + static_cast<int>(rank) * 128;
        for (int kb = 0; kb < P.slices; ++kb, ++it) {
          const int s = it % C::STAGES;
          if (!mbar_wait(&empty[s], ((it / C::STAGES) & 1) ^ 1, abort_flag)) {
            fail(KERR_WAIT_EMPTY);
            ok = false;
            break;
          }
          uint8_t *sw = smem + s * C::STAGE_BYTES, *sx = sw + F_W_BYTES, *ss = sx + C::X_BYTES;
          const uint32_t bar = map_to_cta(smem_u32(&full[s]), 0);
          if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * C::STAGE_BYTES);  // both CTAs' bytes
          tma_load_2d_pair(sw, &P.tm_w, bar, kb * F_KB, n0);
          tma_load_2d_pair(sx, &P.tm_x, bar, kb * F_KB, m0 + static_cast<int>(rank) * 128);
          tma_load_3d_pair(ss, &P.tm_ws, bar, 0, kb * C::CHUNKS, n0 / 128);
          tma_load_3d_pair(ss + C::S_BYTES, &P.tm_xs, bar, 0, kb * C::CHUNKS, m0 / 128);
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (rank == 0) {
      const bool leader = elect_one();
      const uint32_t base = smem_u32(smem);
      uint32_t it = 0, t = 0;
      bool ok = true;
      for (int tile = pair; ok && tile < P.tiles; tile += num_pairs, ++t) {
        if (t > 0 && !mbar_wait_warp(drained, (t - 1) & 1, abort_flag)) {
          if (lane == 0) fail(KERR_WAIT_TMEM_EMPTY);
          break;
        }
        tc_fence_after_sync();
        const uint32_t d = tmem + (t & 1) * C::ACC1;
        for (int kb = 0; kb < P.slices; ++kb, ++it) {
          const int s = it % C::STAGES;
          if (!mbar_wait_warp(&full[s], (it / C::STAGES) & 1, abort_flag)) {
            if (lane == 0) fail(KERR_WAIT_FULL);
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t sw = base + s * C::STAGE_BYTES, sx = sw + F_W_BYTES, ss = sx + C::X_BYTES;
          const uint64_t wd = make_smem_desc_sw128(sw, 16, 1024), xd = make_smem_desc_sw128(sx, 16, 1024);
          if (leader) {
#pragma unroll
            for (int c = 0; c < C::CHUNKS; ++c) {
              fp4_copy_factors<true>(tmem + C::SFA + 4 * c, fp4_factor_desc(ss + 512 * c));
              fp4_copy_factors<true>(tmem + C::SFB + 8 * c, fp4_factor_desc(ss + C::S_BYTES + 512 * c));
              fp4_copy_factors<true>(tmem + C::SFB + 8 * c + 4, fp4_factor_desc(ss + 2 * C::S_BYTES + 512 * c));
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int c = BLOCK == 16 ? k : k >> 1;
              const uint32_t id = BLOCK == 16 ? 0 : (k & 1) * 2;
              fp4_mma<BLOCK, true>(d, wd + 2 * k, xd + 2 * k, fp4_idesc(256, 256, BLOCK, id), tmem + C::SFA + 4 * c,
                                   tmem + C::SFB + 8 * c, (kb | k) ? 1u : 0u);
            }
            tc_commit_pair(&empty[s], 3);
          }
        }
        if (ok && leader) tc_commit_pair(&tfull[t & 1], 3);
      }
    }
    __syncwarp();
  } else {
    const int q = warp & 3, half = warp >= 6;
    float mx = 0.f;
    uint32_t t = 0;
    for (int tile = pair; tile < P.tiles; tile += num_pairs, ++t) {
      const int m0 = (tile % P.tiles_m) * 256, n = (tile / P.tiles_m) * 256 + static_cast<int>(rank) * 128 + q * 32 + lane;
      const int live = n < P.N ? (P.M - m0 < 256 ? P.M - m0 : 256) : 0;
      const Fp4Factor f = fp4_column<STEPS>(P, n < P.N ? n : P.N - 1);
      const uint32_t acc = tmem + (t & 1) * C::ACC1 + (static_cast<uint32_t>(q * 32) << 16);
      const long long pitch = P.pitch, res_pitch = P.res_pitch;
      uint8_t *out = static_cast<uint8_t *>(P.out) + m0 * pitch + n * static_cast<long long>(FP4_SIZE<DT>);
      const uint8_t *res = P.residual ? reinterpret_cast<const uint8_t *>(P.residual) + m0 * res_pitch + n * 4LL : nullptr;
      // Two warps share a lane group and take every other sixteen columns, in an order that starts with the columns the
      // accumulators share (the last 48 of the lower one, the first 48 of the upper one): once the first two loads of
      // each are done the next tile's products may start. Two warps per scheduler, because the epilogue is bound by
      // instruction latency (8 instructions and 26 cycles per column with one); the loop is not unrolled further, because
      // 40 KB of straight-line code ran at the speed of instruction fetches and took the issuer's loop out of the cache.
      const int shared = (t & 1) ? 0 : C::ACC1;
      uint32_t r0[16], r1[16];
      float v0[16], v1[16];
      auto column = [&](int i) { return (shared + 16 * (2 * i + half)) & 255; };
      auto finish = [&](const uint32_t (&r)[16], float (&v)[16], int c) {
        fp4_emit<DT, STEPS>(r, v, res != nullptr, live - c, out + c * pitch, P.pitch, f, mx);
      };
      auto fetch = [&](float (&v)[16], int c) {
        if (res) fp4_residual(v, live - c, res + c * res_pitch, P.res_pitch);
      };
      fetch(v0, column(0));  // while the tile is still being computed
      fetch(v1, column(1));
      if (!mbar_wait_warp(&tfull[t & 1], (t >> 1) & 1, abort_flag)) {
        if (lane == 0) fail(KERR_WAIT_TMEM_FULL);
        break;
      }
      tc_fence_after_sync();
      tc_ld_32x16(acc + column(0), r0);
      tc_ld_32x16(acc + column(1), r1);
      tc_wait_ld();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster_relaxed(map_to_cta(smem_u32(drained), 0));
#pragma unroll 1
      for (int i = 0; i < 8; i += 2) {
        finish(r0, v0, column(i));
        if (i < 6) {
          tc_ld_32x16(acc + column(i + 2), r0);
          fetch(v0, column(i + 2));
        }
        finish(r1, v1, column(i + 1));
        if (i < 6) {
          tc_ld_32x16(acc + column(i + 3), r1);
          fetch(v1, column(i + 3));
        }
        tc_wait_ld();
      }
    }
    sat_report(P.err + 1, DT == FLUX_CUDA_F16, mx);
  }
  if (*abort_flag) {
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000LL) __nanosleep(1000);
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();  // neither CTA leaves while the other may still read its shared memory or signal its barriers
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc_pair(tmem, 512);
  }
}

// ---------------------------------------------------------------------------------------------- host
static PFN_cuTensorMapEncodeTiled_v12000 g_encode4 = nullptr;

template <int BM, int BLOCK, int DT, bool DEEP>
static bool opt_in_one() {
  const int smem = FCfg<BM, BLOCK, DEEP>::SMEM;
  return cudaFuncSetAttribute(gemm_fp4_kernel<BM, BLOCK, DT, DEEP, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) ==
             cudaSuccess &&
         cudaFuncSetAttribute(gemm_fp4_kernel<BM, BLOCK, DT, DEEP, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) ==
             cudaSuccess;
}
template <int BM, bool DEEP>
static bool opt_in() {
  return opt_in_one<BM, 16, FLUX_CUDA_F32, DEEP>() && opt_in_one<BM, 16, FLUX_CUDA_F16, DEEP>() &&
         opt_in_one<BM, 16, FLUX_CUDA_BF16, DEEP>() && opt_in_one<BM, 32, FLUX_CUDA_F32, DEEP>() &&
         opt_in_one<BM, 32, FLUX_CUDA_F16, DEEP>() && opt_in_one<BM, 32, FLUX_CUDA_BF16, DEEP>();
}

template <int BLOCK, int DT>
static bool opt_in_pair_one() {
  const int smem = F2Cfg<BLOCK>::SMEM;
  return cudaFuncSetAttribute(gemm2_fp4_kernel<BLOCK, DT, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) ==
             cudaSuccess &&
         cudaFuncSetAttribute(gemm2_fp4_kernel<BLOCK, DT, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) ==
             cudaSuccess;
}
template <int BLOCK>
static bool opt_in_pair() {
  return opt_in_pair_one<BLOCK, FLUX_CUDA_F32>() && opt_in_pair_one<BLOCK, FLUX_CUDA_F16>() &&
         opt_in_pair_one<BLOCK, FLUX_CUDA_BF16>();
}

// Clusters of 1 to 8 CTAs that a device holds at once with one CTA per SM: the GPCs' numbers of SMs are no multiples of most
// sizes, so they are fewer than the SMs make (33 of four, 15 of eight). The query counts one CTA per SM for the kernels of
// which two fit as well; those are taken to fit twice.
static int g_fp4_clusters[64][9];

static void count_clusters(int *counts) {
  for (int s = 1; s <= 8; ++s) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(1024 / s * s);
    cfg.blockDim = dim3(F_THREADS);
    cfg.dynamicSmemBytes = FCfg<32, 16, true>::SMEM;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = s;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;  // none: this size is not used
    if (cudaOccupancyMaxActiveClusters(&n, gemm_fp4_kernel<32, 16, FLUX_CUDA_BF16, true, false>, &cfg) != cudaSuccess) cudaGetLastError();
    counts[s] = s == 1 && n < 1 ? 1 : n;
  }
}

int fp4_gemm_init(int device) {
  if (device < 0 || device >= 64) return -1;
  if (!g_encode4) {
    void *fn = nullptr;
    cudaDriverEntryPointQueryResult qres;
    cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &qres);
    if (e != cudaSuccess || qres != cudaDriverEntryPointSuccess || !fn) return -1;
    g_encode4 = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
  }
  const bool ok = opt_in<16, false>() && opt_in<16, true>() && opt_in<32, false>() && opt_in<32, true>() && opt_in<64, false>() &&
                  opt_in<128, false>() && opt_in_pair<16>() && opt_in_pair<32>();
  if (!ok) return -2;
  count_clusters(g_fp4_clusters[device]);
  return 0;
}

// The codes of a matrix as bytes, in boxes of box_rows x 128.
static int map_codes(CUtensorMap *m, const flux_cuda_fp4 &q, uint32_t box_rows) {
  const cuuint64_t pitch = static_cast<cuuint64_t>(fp4_pitch(q.cols));
  cuuint64_t dims[2] = {pitch, static_cast<cuuint64_t>(q.rows)};
  cuuint64_t strides[1] = {pitch};
  cuuint32_t box[2] = {F_KB, box_rows}, one[2] = {1, 1};
  CUresult r = g_encode4(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, q.codes, dims, strides, box, one,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : FP4_ERR_MAP;
}
// Its factor tiles, in boxes of `chunks` tiles of one group of 128 rows (or `row_tiles` such groups).
static int map_factors(CUtensorMap *m, const flux_cuda_fp4 &q, uint32_t chunks, uint32_t row_tiles) {
  cuuint64_t dims[3] = {128, static_cast<cuuint64_t>(fp4_chunks(q.cols, q.format)),
                        static_cast<cuuint64_t>(fp4_row_tiles(q.rows))};
  cuuint64_t strides[2] = {512, dims[1] * 512};
  cuuint32_t box[3] = {128, chunks, row_tiles}, one[3] = {1, 1, 1};
  CUresult r = g_encode4(m, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, q.scales, dims, strides, box, one,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : FP4_ERR_MAP;
}

template <int BM, int BLOCK, bool DEEP, bool STEPS>
static cudaError_t launch_steps(const Fp4GemmParams &P, unsigned grid, int dtype, cudaStream_t st) {
  const size_t smem = FCfg<BM, BLOCK, DEEP>::SMEM;
  const dim3 g(grid), t(F_THREADS);
  if (dtype == FLUX_CUDA_F32)
    return launch_kernel(gemm_fp4_kernel<BM, BLOCK, FLUX_CUDA_F32, DEEP, STEPS>, g, t, smem, st, P.splits, P);
  if (dtype == FLUX_CUDA_F16)
    return launch_kernel(gemm_fp4_kernel<BM, BLOCK, FLUX_CUDA_F16, DEEP, STEPS>, g, t, smem, st, P.splits, P);
  return launch_kernel(gemm_fp4_kernel<BM, BLOCK, FLUX_CUDA_BF16, DEEP, STEPS>, g, t, smem, st, P.splits, P);
}
template <int BM, int BLOCK, bool DEEP>
static cudaError_t launch_one(const Fp4GemmParams &P, unsigned grid, int dtype, bool steps, cudaStream_t st) {
  return steps ? launch_steps<BM, BLOCK, DEEP, true>(P, grid, dtype, st) : launch_steps<BM, BLOCK, DEEP, false>(P, grid, dtype, st);
}

template <int BLOCK, bool STEPS>
static cudaError_t launch_pair_steps(const Fp4GemmParams &P, unsigned grid, int dtype, cudaStream_t st) {
  const size_t smem = F2Cfg<BLOCK>::SMEM;
  const dim3 g(grid), t(F2_THREADS);
  if (dtype == FLUX_CUDA_F32) return launch_kernel(gemm2_fp4_kernel<BLOCK, FLUX_CUDA_F32, STEPS>, g, t, smem, st, 2, P);
  if (dtype == FLUX_CUDA_F16) return launch_kernel(gemm2_fp4_kernel<BLOCK, FLUX_CUDA_F16, STEPS>, g, t, smem, st, 2, P);
  return launch_kernel(gemm2_fp4_kernel<BLOCK, FLUX_CUDA_BF16, STEPS>, g, t, smem, st, 2, P);
}
template <int BLOCK>
static cudaError_t launch_pair(const Fp4GemmParams &P, unsigned grid, int dtype, bool steps, cudaStream_t st) {
  return steps ? launch_pair_steps<BLOCK, true>(P, grid, dtype, st) : launch_pair_steps<BLOCK, false>(P, grid, dtype, st);
}

// Which kernel, tile height and split a product gets: the least of the times below, in microseconds, whose constants are
// measured on a B200 (148 SMs) and matter only relative to one another.
//   One CTA per tile: 2.5 to start and stop, a k-slice 0.33 while the ring's latency bounds it (0.45 with the three stages
//   of the 128-row tile; nine deep, 1.2 once and 0.06 per slice while they fit) and its bytes over 12 TB/s of L2 when many
//   CTAs run (a pitch off the 128-byte lines costs 1.6 times as much), as many clusters at once as the device holds; a split
//   adds a cluster launch and the exchange of the partial tile.
//   Pairs: a k-slice 0.35, an epilogue of 2 that the next tile's products hide.
// Measured at 1024 x 1024 x 1024: 64 rows 4.8, 128 rows 5.8, pairs 7.0; 512 x 2560 x 9728: 128 rows 20.8 alone, 16.2 split
// three ways, pairs 19.2; 1 x 2560 x 9728: 16.0 alone, 6.1 split six ways, 5.9 deep; 32 x 2560 x 9728: 7.7 split eight ways,
// 6.9 six ways deep; 1 x 19456 x 2560: 8.1, deep 12.7; 128 x 2560 x 2560: 64 rows 6.8 alone, 7.6 split in two.
struct Fp4Choice {
  int bm, splits;  // bm 256: pairs
  bool deep;
};
static Fp4Choice fp4_choose(long long M, long long N, int slices, long long pitch, int num_sms, const int *clusters) {
  const long long tn = (N + F_BN - 1) / F_BN;
  Fp4Choice best = {128, 1, false};
  double least = 1e30;
  for (int bm = 16; bm <= 128; bm *= 2) {
    if (bm < 64 && M > bm) continue;  // a tile starts on half a factor tile at the least
    const long long tiles = tn * ((M + bm - 1) / bm);
    for (int deep = 0; deep <= (bm < 64); ++deep)
      for (int s = 1; s <= 8 && s <= slices; ++s) {
        const long long at_once = clusters[s] * (deep ? 1LL : 2LL);
        if (at_once < 1 || tiles * s > 0x7FFFFFFF) continue;  // the latter: more CTAs than a launch takes
        const int n = (slices + s - 1) / s;
        const double active = static_cast<double>(tiles < at_once ? tiles : at_once) * s, waves = (tiles + at_once - 1) / at_once;
        const double latency = deep ? 1.2 + (n <= 9 ? 0.06 : 0.15) * n : (bm == 128 ? 0.45 : 0.33) * n;
        const double bytes = n * active * (F_W_BYTES + bm * F_KB + 4096) / 12e6 * (pitch % 128 ? 1.6 : 1.0);
        const double t = 2.5 + waves * (latency > bytes ? latency : bytes) + (s == 1 ? waves * bm * 0.012 : waves * (1.0 + 0.05 * s + 0.04 * bm));
        if (t < least) least = t, best = {bm, s, deep != 0};
      }
    if (bm >= M) break;  // a taller tile would only be emptier
  }
  if (M > 128) {
    const long long tiles = (M + 255) / 256 * ((N + 255) / 256), pairs = num_sms / 2;
    const double waves = (tiles + pairs - 1) / pairs, main = slices * 0.35 * (pitch % 128 ? 1.3 : 1.0) + 0.4;
    if (2.5 + waves * (main > 2.0 ? main : 2.0) + 2.0 < least) best = {256, 1, false};
  }
  return best;
}

int launch_gemm_fp4(const Fp4GemmArgs &a, int device, int num_sms, int *err, cudaStream_t st) {
  Fp4GemmParams P;
  memset(&P, 0, sizeof(P));
  const long long M = a.x.rows, N = a.w.rows;  // up to 2^31 - 1: rounding up to tiles wants more bits
  const int block = a.x.format;
  const int slices = static_cast<int>((static_cast<long long>(a.x.cols) + 255) / 256);
  const Fp4Choice choice = fp4_choose(M, N, slices, fp4_pitch(a.x.cols), num_sms, g_fp4_clusters[device]);
  const int bm = choice.bm;
  const bool pair = bm == 256;
  const uint32_t chunks = 256 / (4 * block);
  if (map_codes(&P.tm_w, a.w, F_BN) || map_codes(&P.tm_x, a.x, pair ? 128 : bm) || map_factors(&P.tm_ws, a.w, chunks, 1) ||
      map_factors(&P.tm_xs, a.x, chunks, pair ? 2 : 1))
    return FP4_ERR_MAP;
  P.M = a.x.rows;
  P.N = a.w.rows;
  P.slices = slices;
  P.tiles_m = static_cast<int>((M + bm - 1) / bm);
  P.splits = choice.splits;
  P.alpha = a.x.scale * a.w.scale;
  P.scale_x = a.x.scale;
  P.scale_w = a.w.scale;
  const bool normal = (fabsf(P.alpha) >= FLT_MIN && fabsf(P.alpha) <= FLT_MAX) || a.x.scale == 0 || a.w.scale == 0;
  const bool steps = !normal || (a.gate && P.alpha != 1.0f);
  P.out = a.out;
  P.pitch = static_cast<uint32_t>(a.ld_out * (a.dtype == FLUX_CUDA_F32 ? 4 : 2));
  P.gate = a.gate;
  P.residual = a.residual;
  P.res_pitch = static_cast<uint32_t>(a.ld_residual * 4);
  P.err = err;
  if (pair) {
    const long long pair_tiles = P.tiles_m * ((N + 255) / 256);
    P.tiles = static_cast<int>(pair_tiles);
    const int pairs = pair_tiles < num_sms / 2 ? P.tiles : num_sms / 2;
    cudaError_t e = block == 16 ? launch_pair<16>(P, 2 * pairs, a.dtype, steps, st)
                                 : launch_pair<32>(P, 2 * pairs, a.dtype, steps, st);
    return e;
  }
  const unsigned grid = static_cast<unsigned>(P.tiles_m * ((N + F_BN - 1) / F_BN) * P.splits);
  cudaError_t e;
#define FX_G(BM, DEEP)                                                      \
  e = block == 16 ? launch_one<BM, 16, DEEP>(P, grid, a.dtype, steps, st) \
                  : launch_one<BM, 32, DEEP>(P, grid, a.dtype, steps, st)
  if (bm == 16 && choice.deep) FX_G(16, true);
  else if (bm == 16) FX_G(16, false);
  else if (bm == 32 && choice.deep) FX_G(32, true);
  else if (bm == 32) FX_G(32, false);
  else if (bm == 64) FX_G(64, false);
  else FX_G(128, false);
#undef FX_G
  return e;
}

}  // namespace fx
