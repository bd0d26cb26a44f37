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
#include <string.h>

#include "fp4.cuh"
#include "launch.cuh"

namespace fx {

static constexpr int F_BN = 128;                  // output columns (rows of w) per CTA
static constexpr int F_KB = 128;                  // bytes of a row per k-slice: 256 codes
static constexpr int F_W_BYTES = F_BN * F_KB;     // 16 KB
static constexpr int F_THREADS = 192;

struct alignas(64) Fp4GemmParams {
  CUtensorMap tm_w, tm_x;    // codes as bytes [rows, pitch], boxes of 128 bytes, 128-byte swizzle
  CUtensorMap tm_ws, tm_xs;  // factor tiles as u32 [row tiles, chunks, 128]
  int M, N, slices;          // k-slices of 256 codes
  int tiles_m;
  int splits;                // CTAs of a cluster that share one output tile, each with its part of the k-slices
  float alpha;
  void *out;
  long long ld;
  const float *gate, *residual;
  long long ld_res;
  int *err;
};

// Instruction descriptor of tcgen05.mma with block factors: [4,6) factor id of B, [7,10) A format and [10,12) B format
// (1 = e2m1), [17,23) N >> 3, 23 factor type (0 e4m3, 1 power of two), [27,29) M >> 7, [29,31) factor id of A. Both
// operands K-major. The factor id picks the bytes of a 32-bit TMEM column: 0, or 2 for the upper half of a pair.
__host__ __device__ constexpr uint32_t fp4_idesc(int M, int N, int block, uint32_t id) {
  return (id << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(N >> 3) << 17) | ((block == 32 ? 1u : 0u) << 23) |
         (static_cast<uint32_t>(M >> 7) << 27) | (id << 29);
}

// D[tmem] (+)= A[smem] * B[smem] with block factors in TMEM; 64 codes of K. Issued by ONE thread.
template <int BLOCK>
__device__ __forceinline__ void fp4_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb,
                                        uint32_t accumulate) {
  if (BLOCK == 16)
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n\t"
        "}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t"
        "}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate)
        : "memory");
}

// One 512-byte factor tile from shared memory to four TMEM columns, repeated in the four lane groups.
__device__ __forceinline__ void fp4_copy_factors(uint32_t taddr, uint64_t sdesc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(sdesc) : "memory");
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

__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// ------------------------------------------------------------------------------------------------
// One CTA per 128 (n) x BM (m) tile, or a cluster of `splits` CTAs that each take a part of K and add their parts in
// rank order through distributed shared memory (no workspace, no atomics, the same bits every time).
// ------------------------------------------------------------------------------------------------
template <int BM, int BLOCK>
struct FCfg {
  static constexpr int CHUNKS = 256 / (4 * BLOCK);  // factor tiles per k-slice
  static constexpr int X_BYTES = BM * F_KB;
  static constexpr int S_BYTES = CHUNKS * 512;
  static constexpr int STAGE_BYTES = F_W_BYTES + X_BYTES + 2 * S_BYTES;
  static constexpr int STAGES = BM >= 128 ? 3 : 4;
  static constexpr int SMEM = STAGES * STAGE_BYTES + 256 + 1024;
  static constexpr int SF_COLS = CHUNKS * 4;
  static constexpr int TMEM_COLS = BM + 2 * SF_COLS <= 64 ? 64 : BM + 2 * SF_COLS <= 128 ? 128 : 256;
  static_assert(STAGE_BYTES % 1024 == 0, "the swizzled operands of every stage start on 1024 bytes");
  static_assert(BM * F_BN * 4 <= STAGES * STAGE_BYTES, "the partial tile of a split fits the operand ring");
  static_assert(BM + 2 * SF_COLS <= TMEM_COLS, "accumulator and factors fit the allocation");
};

template <int BM, int BLOCK, int DT>
__global__ void __launch_bounds__(F_THREADS) gemm_fp4_kernel(const __grid_constant__ Fp4GemmParams P) {
  using C = FCfg<BM, BLOCK>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
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
      if (leader) {
#pragma unroll
        for (int c = 0; c < C::CHUNKS; ++c) {
          fp4_copy_factors(sfa + 4 * c, fp4_factor_desc(ss + 512 * c));
          fp4_copy_factors(sfb + 4 * c, fp4_factor_desc(ss + C::S_BYTES + 512 * c));
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int c = BLOCK == 16 ? k : k >> 1;
          const uint32_t id = BLOCK == 16 ? 0 : (k & 1) * 2;
          fp4_mma<BLOCK>(tmem, wd + 2 * k, xd + 2 * k, fp4_idesc(F_BN, BM, BLOCK, id), sfa + 4 * c, sfb + 4 * c,
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
    const bool ok = mbar_wait_warp(tfull, 0, abort_flag);
    if (!ok && lane == 0) fail(KERR_WAIT_TMEM_FULL);
    tc_fence_after_sync();
    const int live = P.M - m0 < BM ? P.M - m0 : BM;
    const float g = P.gate && n < P.N ? P.gate[n] : 1.0f;
    float mx = 0.f;
    auto emit = [&](int m, float acc) {
      float v = g * (P.alpha * acc);
      if (P.residual) v += P.residual[static_cast<long long>(m) * P.ld_res + n];
      fp4_store<DT>(P.out, static_cast<long long>(m) * P.ld + n, v, mx);
    };
    constexpr int STEP = BM < 32 ? 16 : 32;
    float *part = reinterpret_cast<float *>(smem);  // every MMA has read its operands by now
    if (ok) {
      for (int c = 0; c < BM; c += STEP) {
        if (c >= live) break;
        uint32_t r[STEP];
        const uint32_t at = tmem + c + (static_cast<uint32_t>(q * 32) << 16);
        if constexpr (STEP == 16) tc_ld_32x16(at, r);
        else tc_ld_32x32(at, r);
        tc_wait_ld();
        if (P.splits > 1) {
#pragma unroll
          for (int j = 0; j < STEP; ++j) part[(c + j) * F_BN + nl] = __uint_as_float(r[j]);
        } else if (n < P.N) {
#pragma unroll
          for (int j = 0; j < STEP; ++j)
            if (c + j < live) emit(m0 + c + j, __uint_as_float(r[j]));
        }
      }
    }
    if (P.splits > 1) {
      __syncwarp();
      cluster_sync_all();
      // every CTA of the cluster finishes its share of the tile's rows, adding the parts in rank order
      if (ok && n < P.N) {
        const uint32_t mine = smem_u32(part) + nl * 4;
        for (int m = rank; m < live; m += P.splits) {
          float acc = 0.f;
          for (int s = 0; s < P.splits; ++s) acc += ld_cluster_f32(map_to_cta(mine + m * F_BN * 4, s));
          emit(m0 + m, acc);
        }
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

// ---------------------------------------------------------------------------------------------- host
static PFN_cuTensorMapEncodeTiled_v12000 g_encode4 = nullptr;

template <int BM, int BLOCK>
static cudaError_t opt_in() {
  cudaError_t e = cudaFuncSetAttribute(gemm_fp4_kernel<BM, BLOCK, FLUX_CUDA_F32>,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize, FCfg<BM, BLOCK>::SMEM);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(gemm_fp4_kernel<BM, BLOCK, FLUX_CUDA_F16>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             FCfg<BM, BLOCK>::SMEM);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(gemm_fp4_kernel<BM, BLOCK, FLUX_CUDA_BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             FCfg<BM, BLOCK>::SMEM);
  return e;
}

int fp4_gemm_init() {
  if (!g_encode4) {
    void *fn = nullptr;
    cudaDriverEntryPointQueryResult qres;
    cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &qres);
    if (e != cudaSuccess || qres != cudaDriverEntryPointSuccess || !fn) return -1;
    g_encode4 = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
  }
  const bool ok = opt_in<16, 16>() == cudaSuccess && opt_in<16, 32>() == cudaSuccess && opt_in<32, 16>() == cudaSuccess &&
                  opt_in<32, 32>() == cudaSuccess && opt_in<64, 16>() == cudaSuccess && opt_in<64, 32>() == cudaSuccess &&
                  opt_in<128, 16>() == cudaSuccess && opt_in<128, 32>() == cudaSuccess;
  return ok ? 0 : -2;
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
  return r == CUDA_SUCCESS ? 0 : -4;
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
  return r == CUDA_SUCCESS ? 0 : -4;
}

template <int BM, int BLOCK>
static cudaError_t launch_one(const Fp4GemmParams &P, unsigned grid, int dtype, cudaStream_t st) {
  const size_t smem = FCfg<BM, BLOCK>::SMEM;
  if (dtype == FLUX_CUDA_F32)
    return launch_kernel(gemm_fp4_kernel<BM, BLOCK, FLUX_CUDA_F32>, dim3(grid), dim3(F_THREADS), smem, st, P.splits, P);
  if (dtype == FLUX_CUDA_F16)
    return launch_kernel(gemm_fp4_kernel<BM, BLOCK, FLUX_CUDA_F16>, dim3(grid), dim3(F_THREADS), smem, st, P.splits, P);
  return launch_kernel(gemm_fp4_kernel<BM, BLOCK, FLUX_CUDA_BF16>, dim3(grid), dim3(F_THREADS), smem, st, P.splits, P);
}

int launch_gemm_fp4(const Fp4GemmArgs &a, int num_sms, int *err, cudaStream_t st) {
  Fp4GemmParams P;
  memset(&P, 0, sizeof(P));
  const int M = a.x.rows, N = a.w.rows, block = a.x.format;
  const int bm = M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : 128;
  const uint32_t chunks = 256 / (4 * block);
  if (map_codes(&P.tm_w, a.w, F_BN) || map_codes(&P.tm_x, a.x, bm) || map_factors(&P.tm_ws, a.w, chunks, 1) ||
      map_factors(&P.tm_xs, a.x, chunks, 1))
    return -4;
  P.M = M;
  P.N = N;
  P.slices = static_cast<int>((static_cast<long long>(a.x.cols) + 255) / 256);
  P.tiles_m = (M + bm - 1) / bm;
  const long long tiles = static_cast<long long>(P.tiles_m) * ((N + F_BN - 1) / F_BN);
  P.splits = 1;
  while (P.splits < 8 && tiles * P.splits * 2 <= 2LL * num_sms && P.splits * 2 <= P.slices) P.splits *= 2;
  P.alpha = a.x.scale * a.w.scale;
  P.out = a.out;
  P.ld = a.ld_out;
  P.gate = a.gate;
  P.residual = a.residual;
  P.ld_res = a.ld_residual;
  P.err = err;
  const unsigned grid = static_cast<unsigned>(tiles * P.splits);
  cudaError_t e;
#define FX_G(BM) e = block == 16 ? launch_one<BM, 16>(P, grid, a.dtype, st) : launch_one<BM, 32>(P, grid, a.dtype, st)
  if (bm == 16) FX_G(16);
  else if (bm == 32) FX_G(32);
  else if (bm == 64) FX_G(64);
  else FX_G(128);
#undef FX_G
  return e == cudaSuccess ? 0 : -8;
}

}  // namespace fx
