// A few rows of f32 / f16 / bf16 times a 4-bit matrix: out[m, n] = w.scale * sum_k x[m, k] w[n, k], the activations not
// quantised. The form for single tokens and for the modulation vectors of a schedule. Bound by reading the packed weights
// once (0.56 bytes per weight) and by decoding them.
//
// Decoding: a code and its factor are an exact bf16 value (at most six significant bits). The three magnitude bits of a
// code, put at the border of a bf16's exponent and mantissa, are the code's value times 2^-126 (the code for 0.5 becomes a
// subnormal), so a mask, an integer multiplication, a mask and one packed multiplication by factor * 2^110 (blocks of 32:
// 2^(e + 126)) make two weights. Multiplying in f32 instead takes two conversions and one multiply-add per weight and row of x: measured 17 us
// for one row and 36 for four (19456 x 2560), bound by instructions.
//
// Products: mma.sync m16n8k16 on bf16, 16 weight rows by 8 columns, f32 sums. x is split into bf16 parts (bf16 1,
// f16 2, f32 3), each a column of its own, so every product is exact and all rows of x share one decoding (up to 32 columns,
// more rows are further blocks). (tcgen05 wants its operands in
// shared memory; decoded weights go from registers to the multiplication here.)
//
// A warp takes 32 weight rows at a time (a "unit": rows r + 32 q, r = 8 neighbours, q = 0..3, because one 16-byte piece of
// a factor tile holds the factors of exactly the rows r + 32 q for four blocks) in steps of 256 columns, a 128-byte line of
// each row: a lane loads twice 32 consecutive codes of its four rows, and because sums do not care for order, those are its
// columns in the multiplication too. The loads go to a ring in shared memory, asynchronously and without barriers, so that a
// step is on its way while one is computed without costing registers; 64 bytes of a row at a time into registers came to 2.1
// TB/s. x lies in shared memory in the order of the multiplication's registers. K is split among the CTAs of a cluster, so
// that x fits and the units of a cluster are many enough to be shared out evenly; the warps of a CTA take equal stretches of
// its (unit, step) pairs, wherever these begin and end. Partial sums are added in a fixed order through (distributed) shared
// memory: no workspace, no atomics, the same bits every time.
#include <math.h>

#include "fp4.cuh"
#include "launch.cuh"

namespace fx {

static constexpr int V_WARPS = 16, V_THREADS = 32 * V_WARPS;  // one block per SM
static constexpr int V_STEP_BYTES = 8 * 512 + 512;             // a warp's codes and factors of a step
static_assert(V_STEP_BYTES >= 32 * 32 * 4, "32 columns of sums fit the places of a step");
static constexpr int V_RING = 2 * V_WARPS * V_STEP_BYTES;      // two steps per warp
static constexpr int V_SMEM_MAX = 227 * 1024 - V_RING;         // what is left for x and the sums

struct GemvFp4Params {
  const void *x;
  int x_vec;  // x and its row pitch are multiples of 16 bytes
  long long ldx;
  int rows, group;  // rows of x; rows of x per block, each in PARTS columns
  const uint8_t *codes, *scales;
  long long pitch, chunks;
  float scale, scale2;  // what a sum is multiplied by; the second is 1 unless f32 cannot hold the two as one
  int N, K, steps;  // steps of 256 columns
  int kparts;       // K is split among this many CTAs of a cluster
  int part_steps;   // most steps of a CTA
  int clusters;
  long long units;
  void *out;
  int dt;
  long long ld;
  int *sat;
  uint2 by;  // 2^12 + 2^6 and 2^8 + 2^2 (v_place); not constants, which the compiler would take apart into shifts
};

// Where a lane's pieces of the next step lie. Rows past the last one read it instead (their sums are dropped).
struct VRows {
  const uint8_t *codes[4], *factors;
};
template <int BLOCK>
__device__ __forceinline__ VRows v_rows(const GemvFp4Params &P, long long unit, int step, int lane) {
  const int g = lane >> 2, t = lane & 3, r32 = static_cast<int>(unit & 3) * 8 + g;
  const long long n0 = (unit >> 2) * 128 + r32;
  VRows r;
#pragma unroll
  for (int q = 0; q < 4; ++q)
    r.codes[q] = P.codes + (n0 + 32 * q < P.N ? n0 + 32 * q : P.N - 1) * P.pitch + step * 128 + t * 16;
  r.factors = P.scales + ((unit >> 2) * P.chunks + step * (64 / BLOCK) + t * 8 / BLOCK) * 512 + r32 * 16;
  return r;
}
// 16 bytes from global to shared memory, asynchronously; zeros where there is nothing to read.
__device__ __forceinline__ void v_copy16(uint32_t dst, const uint8_t *src, bool in) {
  if (in) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(dst), "r"(0) : "memory");
}
// A step of a unit: the codes into this lane's places, [half of the step][4 rows][lane], and the pieces of factors into the
// warp's, [half][piece][8 neighbours], by the first of the lanes that share one; and on to the next step. left, chunks: bytes
// of codes and chunks of factors from here to the end of the row.
template <int BLOCK>
__device__ __forceinline__ void v_fetch(uint32_t dst, VRows &r, int step, int lane, int code_end, int factor_end) {
  constexpr int PIECES = 32 / BLOCK;  // of half a step: two chunks of 64 columns, or one of 128
  const int g = lane >> 2, t = lane & 3, p = t * 8 / BLOCK;
  const int left = code_end - step * 128 - t * 16, chunks = factor_end - step * 2 * PIECES - p;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int q = 0; q < 4; ++q) v_copy16(dst + (h * 4 + q) * 512 + lane * 16, r.codes[q] + h * 64, left > h * 64);
    if (t * 8 % BLOCK == 0)
      v_copy16(dst + 8 * 512 + ((h * PIECES + p) * 8 + g) * 16, r.factors + h * PIECES * 512, chunks > h * PIECES);
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) r.codes[q] += 128;
  r.factors += 2 * PIECES * 512;
  asm volatile("cp.async.commit_group;" ::: "memory");
}
__device__ __forceinline__ uint4 v_ring(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ uint32_t v_mul2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// Eight codes to four bf16 pairs (codes i and i + 4) times m (a pair of equal factors). One multiplication by 2^a + 2^b puts
// a masked code's sign and its magnitude where they belong at once; the copies that land elsewhere are masked off. (With a
// shift and a mask for each the decoding was bound by the integer pipe: 275 of its instructions per 128 codes and lane.)
__device__ __forceinline__ uint32_t v_place(uint32_t code, uint32_t by) { return (code * by) & 0x81C081C0u; }
__device__ __forceinline__ void v_decode(uint32_t w, uint32_t m, uint2 by, uint32_t (&p)[4]) {
  const uint32_t v = w >> 8;
  p[0] = v_mul2(v_place(w & 0x000F000Fu, by.x), m);
  p[1] = v_mul2(v_place(w & 0x00F000F0u, by.y), m);
  p[2] = v_mul2(v_place(v & 0x000F000Fu, by.x), m);
  p[3] = v_mul2(v_place(v & 0x00F000F0u, by.y), m);
}
__device__ __forceinline__ void v_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                      uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The same onto zeros: the start of a chain.
__device__ __forceinline__ void v_mma0(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// The bf16 parts of a value, the largest first (8 bits of the magnitude each), the second times 2^7 and the third times 2^15:
// as they are the lower parts of numbers below 2^-110 would lie among the subnormal bf16 numbers, whose digits end at 2^-133.
// Taken up so far a part is not above the value itself, so no sum leaves f32 earlier; of f32 numbers below 2^-124 the digit
// 2^-149 is cut off.
__device__ __forceinline__ constexpr float v_up(int part) { return part == 0 ? 128.f : 256.f; }  // from one part to the next
template <int PARTS>
__device__ __forceinline__ void v_split(float x, uint32_t (&p)[PARTS]) {
  const bool finite = (__float_as_uint(x) & 0x7F800000u) != 0x7F800000u;
  if (!finite && x != x) x = __uint_as_float(0x7FC00000u);
#pragma unroll
  for (int i = 0; i < PARTS; ++i) {
    const uint32_t top = __float_as_uint(x) & 0xFFFF0000u;
    p[i] = top >> 16;
    x = finite ? (x - __uint_as_float(top)) * v_up(i) : 0.f;
  }
}

// Elements of x, whose type has PARTS parts; eight of them from a 16-byte aligned address.
template <int PARTS>
__device__ __forceinline__ float v_load(const void *x, long long i) {
  if (PARTS == 3) return __ldg(reinterpret_cast<const float *>(x) + i);
  const uint16_t h = __ldg(reinterpret_cast<const uint16_t *>(x) + i);
  return PARTS == 2 ? __half2float(__ushort_as_half(h)) : __uint_as_float(static_cast<uint32_t>(h) << 16);
}
template <int PARTS>
__device__ __forceinline__ void v_load8(const void *x, long long i, float (&v)[8]) {
  if (PARTS == 3) {
    const float4 *p = reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(x) + i);
    const float4 a = __ldg(p), b = __ldg(p + 1);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
    const uint4 a = __ldg(reinterpret_cast<const uint4 *>(reinterpret_cast<const uint16_t *>(x) + i));
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (PARTS == 2) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[j]));
        v[2 * j] = f.x, v[2 * j + 1] = f.y;
      } else {
        v[2 * j] = bf16_lo(w[j]), v[2 * j + 1] = bf16_hi(w[j]);
      }
    }
  }
}

// NH: 8 NH columns per block at most (group * PARTS of them, part by part); PARTS: bf16 parts of x.
template <int NH, int PARTS, int BLOCK>
__global__ void __launch_bounds__(V_THREADS, 1) gemv_fp4_kernel(const __grid_constant__ GemvFp4Params P) {
  // the ring, then x [2 part_steps][4][columns][4], then sums [units + 2 V_WARPS][group][32]
  extern __shared__ uint4 shared[];
  uint4 *xs = shared + V_RING / 16;
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int part = blockIdx.x % P.kparts, cluster = blockIdx.x / P.kparts;
  const int G = P.group, m0 = blockIdx.y * G, C = G * PARTS;
  const int s0 = static_cast<int>(static_cast<long long>(P.steps) * part / P.kparts),
            s1 = static_cast<int>(static_cast<long long>(P.steps) * (part + 1) / P.kparts), L = s1 - s0;
  const long long u0 = P.units * cluster / P.clusters;
  const int nu = static_cast<int>(P.units * (cluster + 1) / P.clusters - u0);
  float *sums = reinterpret_cast<float *>(xs + 2 * P.part_steps * 16 * C);

  // this warp's stretch of the nu * L pairs, unit by unit
  auto begin_of = [&](int w) { return static_cast<int>(static_cast<long long>(nu) * L * w / V_WARPS); };
  const int first = begin_of(warp), last = begin_of(warp + 1);
  int u = first / L, st = first - u * L;
  VRows rows = v_rows<BLOCK>(P, u0 + (u < nu ? u : 0), s0 + st, lane);
  const int code_end = static_cast<int>(P.pitch), factor_end = static_cast<int>(P.chunks);
  // lanes beyond the columns repeat the last one: the sums they take part in are dropped
  int x_lane[NH];
#pragma unroll
  for (int nh = 0; nh < NH; ++nh) x_lane[nh] = (g + 8 * nh < C ? g + 8 * nh : C - 1) * 4 + t;
  const uint32_t ring = smem_u32(shared) + warp * 2 * V_STEP_BYTES;
  const uint32_t my_factors = 8 * 512 + (t * 8 / BLOCK * 8 + g) * 16;
  if (first < last) v_fetch<BLOCK>(ring, rows, s0 + st, lane, code_end, factor_end);  // the weights do not wait for x
  for (int i = threadIdx.x; i < 2 * L * 16 * G; i += V_THREADS) {  // eight consecutive columns of a row
    const int c8 = i % (2 * L * 16), m = i / (2 * L * 16);
    const int sx = c8 >> 4, tt = (c8 >> 2) & 3, jj = c8 & 3;
    const long long k = s0 * 256LL + sx * 128 + tt * 32 + jj * 8, at = (m0 + m) * P.ldx + k;
    uint32_t p[8][PARTS];
    float v[8];
    if (P.x_vec && m0 + m < P.rows && k + 8 <= P.K) {
      v_load8<PARTS>(P.x, at, v);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = m0 + m < P.rows && k + e < P.K ? v_load<PARTS>(P.x, at + e) : 0.f;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v_split<PARTS>(v[e], p[e]);
#pragma unroll
    for (int h = 0; h < PARTS; ++h)  // columns i and i + 4 in a register, as the codes are decoded
      xs[((sx * 4 + jj) * C + h * G + m) * 4 + tt] = make_uint4(p[0][h] | p[4][h] << 16, p[1][h] | p[5][h] << 16,
                                                                      p[2][h] | p[6][h] << 16, p[3][h] | p[7][h] << 16);
  }
  __syncthreads();

  for (int at = first; at < last; ++u) {
    const bool begins = st == 0;
    const int stop = st + (last - at) < L ? st + (last - at) : L;
    float d[2][NH][4];
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int h = 0; h < NH; ++h) d[a][h][0] = d[a][h][1] = d[a][h][2] = d[a][h][3] = 0.f;
    // a unit that this warp does not do alone: its sums go to a place of the warp's own, one for the stretch's first unit
    // and one for its last
    float *mine = sums + (begins && stop == L ? u : nu + 2 * warp + (at == first ? 0 : 1)) * G * 32;
    for (; st < stop; ++st, ++at) {
      if (at + 1 < last) {
        if (st + 1 == L) rows = v_rows<BLOCK>(P, u0 + u + 1, s0, lane);
        v_fetch<BLOCK>(ring + ((at + 1 - first) & 1) * V_STEP_BYTES, rows, s0 + (st + 1 == L ? 0 : st + 1), lane, code_end, factor_end);
        asm volatile("cp.async.wait_group 1;" ::: "memory");
      } else {
        asm volatile("cp.async.wait_group 0;" ::: "memory");
      }
      __syncwarp();  // the factors were copied by other lanes; nobody overwrites them before the multiplications below
#pragma unroll 1
      for (int half = 0; half < 2; ++half) {
        const uint32_t here = ring + ((at - first) & 1) * V_STEP_BYTES;
        uint4 cur[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) cur[q] = v_ring(here + (half * 4 + q) * 512 + lane * 16);
        const uint4 f4 = v_ring(here + my_factors + half * (32 / BLOCK) * 128);
        // this lane's factors: two blocks of 16 per row (half of a factor word), or one of 32 (a quarter of it)
        const uint32_t fw[4] = {f4.x, f4.y, f4.z, f4.w};
        uint32_t m[4][2];
        uint32_t over[4];
        bool wide = false;  // blocks of 32: a factor above 2, or NaN, somewhere in the warp
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if (BLOCK == 16) {
            uint32_t h;
            asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(fw[q] >> (t & 1) * 16)));
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h));
            m[q][0] = __byte_perm(__float_as_uint(f.x * 0x1p110f), 0, 0x3232);
            m[q][1] = __byte_perm(__float_as_uint(f.y * 0x1p110f), 0, 0x3232);
          } else {
            const uint32_t b = fw[q] >> t * 8 & 0xFFu;
            m[q][0] = m[q][1] = (b + 126u) * 0x00800080u;  // 2^(e + 126), twice
            wide |= b > 128u;
          }
        }
        if (BLOCK == 32) {
          wide = __any_sync(0xffffffffu, wide);
          if (wide) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const uint32_t b = fw[q] >> t * 8 & 0xFFu;
              m[q][0] = m[q][1] = b == 255u ? 0x7FC07FC0u : (min(b, 128u) + 126u) * 0x00800080u;  // 2^(min(e, 1) + 126)
              over[q] = (b > 128u && b < 255u ? b - 1u : 127u) * 0x00800080u;                     // the rest: 2^(e - 1)
            }
          }
        }
        const uint4 *xp = xs + (2 * st + half) * 16 * C;
        // The instruction truncates its sums: chains of more than 128 columns are added with rounding. (One chain over all of
        // K was 2.8e-6 off, relative, at K = 9216.)
        float e[2][NH][4];
#pragma unroll
        for (int jj = 0; jj < 4; ++jj) {
          uint32_t a[4][4];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const uint32_t w = jj == 0 ? cur[q].x : jj == 1 ? cur[q].y : jj == 2 ? cur[q].z : cur[q].w;
            v_decode(w, m[q][jj >> 1], P.by, a[q]);
            if (BLOCK == 32 && wide) {
#pragma unroll
              for (int i = 0; i < 4; ++i) a[q][i] = v_mul2(a[q][i], over[q]);
            }
          }
#pragma unroll
          for (int nh = 0; nh < NH; ++nh) {
            const uint4 b = xp[jj * C * 4 + x_lane[nh]];
#pragma unroll
            for (int tile = 0; tile < 2; ++tile) {
              if (jj == 0) v_mma0(e[tile][nh], a[2 * tile][0], a[2 * tile + 1][0], a[2 * tile][1], a[2 * tile + 1][1], b.x, b.y);
              else v_mma(e[tile][nh], a[2 * tile][0], a[2 * tile + 1][0], a[2 * tile][1], a[2 * tile + 1][1], b.x, b.y);
              v_mma(e[tile][nh], a[2 * tile][2], a[2 * tile + 1][2], a[2 * tile][3], a[2 * tile + 1][3], b.z, b.w);
            }
          }
        }
#pragma unroll
        for (int tile = 0; tile < 2; ++tile)
#pragma unroll
          for (int nh = 0; nh < NH; ++nh)
#pragma unroll
            for (int i = 0; i < 4; ++i) d[tile][nh][i] += e[tile][nh][i];
      }
    }
    st = 0;
    // through the places of the step that was just used: the columns of a row of x are added, the smallest parts first
    float *swap = reinterpret_cast<float *>(shared) + (warp * 2 + ((at - 1 - first) & 1)) * (V_STEP_BYTES / 4);
    __syncwarp();
#pragma unroll
    for (int tile = 0; tile < 2; ++tile)
#pragma unroll
      for (int nh = 0; nh < NH; ++nh)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int c = nh * 8 + 2 * t + (i & 1), q = 2 * tile + (i >> 1);
          if (c < C) swap[c * 32 + q * 8 + g] = d[tile][nh][i];
        }
    __syncwarp();
    for (int m = 0; m < G; ++m) {
      float y = swap[((PARTS - 1) * G + m) * 32 + lane];
#pragma unroll
      for (int h = PARTS - 2; h >= 0; --h) y = fmaf(y, 1.0f / v_up(h), swap[(h * G + m) * 32 + lane]);
      mine[m * 32 + lane] = y;
    }
    __syncwarp();
  }
  __syncthreads();
  // units in pieces: the pieces in the order of the warps (unit i is pairs [i L, i L + L))
  for (int i = warp; i < nu; i += V_WARPS) {
    const int lo = i * L, hi = lo + L;
    int w0 = static_cast<int>(static_cast<long long>(lo) * V_WARPS / (nu * L));
    while (w0 + 1 < V_WARPS && begin_of(w0 + 1) <= lo) ++w0;
    if (begin_of(w0) <= lo && begin_of(w0 + 1) >= hi) continue;  // one warp's alone
    for (int m = 0; m < G; ++m) {
      float y = 0.f;
      for (int w = w0; w < V_WARPS && begin_of(w) < hi; ++w)
        if (begin_of(w) < begin_of(w + 1)) y += sums[((nu + 2 * w + (begin_of(w) >= lo ? 0 : 1)) * G + m) * 32 + lane];
      sums[(i * G + m) * 32 + lane] = y;
    }
  }
  // and the parts in the order of the cluster's CTAs
  if (P.kparts > 1) cluster_sync_all();
  else __syncthreads();
  float mx = 0.f;
  const int count = nu * G * 32;
  for (int i = part * V_THREADS + threadIdx.x; i < count; i += P.kparts * V_THREADS) {
    const int rl = i & 31, m = (i >> 5) % G, u = (i >> 5) / G;
    float y = 0.f;
    if (P.kparts > 1) {
      const uint32_t at = smem_u32(sums + i);
      float p[8];
#pragma unroll
      for (int c = 0; c < 8; ++c)
        if (c < P.kparts) p[c] = ld_cluster_f32(map_to_cta(at, c));
#pragma unroll
      for (int c = 0; c < 8; ++c)
        if (c < P.kparts) y += p[c];
    } else {
      y = sums[i];
    }
    const long long unit_i = u0 + u, n = (unit_i >> 2) * 128 + (unit_i & 3) * 8 + (rl & 7) + 32 * (rl >> 3);
    if (n < P.N && m0 + m < P.rows) {
      y *= P.scale;
      if (P.scale2 != 1.0f) y *= P.scale2;
      const long long at = (m0 + m) * P.ld + n;
      if (P.dt == FLUX_CUDA_F32) fp4_store<FLUX_CUDA_F32>(P.out, at, y, mx);
      else if (P.dt == FLUX_CUDA_F16) fp4_store<FLUX_CUDA_F16>(P.out, at, y, mx);
      else fp4_store<FLUX_CUDA_BF16>(P.out, at, y, mx);
    }
  }
  sat_report(P.sat, P.dt == FLUX_CUDA_F16, mx);
  if (P.kparts > 1) cluster_sync_all();  // nobody leaves while another CTA still reads its sums
}

// Clusters of 1, 2, 4 and 8 blocks that a device holds at once, one block per SM (the GPCs' numbers of SMs are no multiples of
// eight, so they are fewer than the SMs make).
static int g_clusters[64][4];
template <int NH, int PARTS>
static bool v_opt_in() {
  return cudaFuncSetAttribute(gemv_fp4_kernel<NH, PARTS, 16>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              V_RING + V_SMEM_MAX) == cudaSuccess &&
         cudaFuncSetAttribute(gemv_fp4_kernel<NH, PARTS, 32>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              V_RING + V_SMEM_MAX) == cudaSuccess;
}
int fp4_gemv_init(int device) {
  if (device < 0 || device >= 64) return -1;
  if (!v_opt_in<1, 1>() || !v_opt_in<2, 1>() || !v_opt_in<1, 2>() || !v_opt_in<2, 2>() || !v_opt_in<4, 2>() || !v_opt_in<1, 3>() ||
      !v_opt_in<2, 3>() || !v_opt_in<3, 3>() || !v_opt_in<4, 3>())
    return -2;
  for (int i = 0; i < 4; ++i) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(128 << i);
    cfg.blockDim = dim3(V_THREADS);
    cfg.dynamicSmemBytes = V_RING + V_SMEM_MAX;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1 << i;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;  // none: this size is not used unless x needs it
    if (cudaOccupancyMaxActiveClusters(&n, gemv_fp4_kernel<1, 1, 16>, &cfg) != cudaSuccess) cudaGetLastError();
    g_clusters[device][i] = n;
  }
  return 0;
}

template <int NH, int PARTS, int BLOCK>
static cudaError_t v_launch(dim3 grid, size_t smem, cudaStream_t st, const GemvFp4Params &P) {
  PdlOff plain;  // a grid of this kind that may follow a persistent cluster kernel goes out in plain stream order
  return launch_kernel(gemv_fp4_kernel<NH, PARTS, BLOCK>, grid, dim3(V_THREADS), smem, st, P.kparts, P);
}

int launch_gemv_fp4(const void *x, int x_dtype, long long ldx, int rows, const flux_cuda_fp4 &w, void *out, int dtype,
                    long long ld_out, int device, int *sat, cudaStream_t st) {
  GemvFp4Params P = {};
  P.x = x, P.ldx = ldx, P.rows = rows;
  P.x_vec = !(reinterpret_cast<uintptr_t>(x) & 15) && !(ldx * (x_dtype == FLUX_CUDA_F32 ? 4 : 2) & 15);
  P.codes = static_cast<const uint8_t *>(w.codes), P.scales = static_cast<const uint8_t *>(w.scales);
  P.pitch = fp4_pitch(w.cols), P.chunks = fp4_chunks(w.cols, w.format);
  // Blocks of 16: the factors go in as factor * 2^110, against codes * 2^-126. In one step with the scale, because the sum
  // times 2^16 may be beyond f32 where the result is not.
  P.scale = w.format == 16 ? w.scale * 65536.0f : w.scale, P.scale2 = 1.0f;
  if (isinf(P.scale)) P.scale = w.scale, P.scale2 = 65536.0f;
  P.N = w.rows, P.K = w.cols;
  P.steps = (w.cols + 255) / 256;
  P.out = out, P.dt = dtype, P.ld = ld_out, P.sat = sat;
  P.by = make_uint2((1u << 12) + (1u << 6), (1u << 8) + (1u << 2));
  P.units = fp4_row_tiles(w.rows) * 4;
  const int parts = x_dtype == FLUX_CUDA_BF16 ? 1 : x_dtype == FLUX_CUDA_F16 ? 2 : 3;
  // Rows of x per block (evenly shared out, up to 32 columns), and K in as many CTAs as it takes to fit them.
  const int blocks_of_rows = (rows * parts + 31) / 32;
  P.group = (rows + blocks_of_rows - 1) / blocks_of_rows;
  auto x_bytes = [&](int group, int kparts) {
    return static_cast<long long>((P.steps + kparts - 1) / kparts) * 512 * parts * group;
  };
  const long long sums_room = 16384;
  P.kparts = 1;
  while (P.kparts < 8 && P.kparts * 2 <= P.steps && x_bytes(P.group, P.kparts) > V_SMEM_MAX - sums_room * (1 + (P.group > 4))) P.kparts *= 2;
  while (P.group > 1 && x_bytes(P.group, P.kparts) + (2 * V_WARPS + 1) * 128LL * P.group > V_SMEM_MAX) P.group = (P.group + 1) / 2;
  const int sets = (rows + P.group - 1) / P.group;
  // Of the ways to split K further, as long as a warp gets a step, the one that ends first: clusters at once, and how evenly
  // the units go into them.
  auto held = [&](int kparts) {
    const long long n = g_clusters[device][kparts == 1 ? 0 : kparts == 2 ? 1 : kparts == 4 ? 2 : 3] / sets;
    return n < 1 ? 1 : n > P.units ? P.units : n;
  };
  // in steps of a warp: what the busiest cluster's warps do, a quarter for joining parts, and laying out x (a fifth of a
  // step for every 16 bytes and thread)
  auto longest = [&](int kparts) {
    const long long n = held(kparts), pairs = (P.units + n - 1) / n * ((P.steps + kparts - 1) / kparts);
    return static_cast<double>(pairs) / V_WARPS + 0.25 * (kparts > 1) + 0.2 * x_bytes(P.group, kparts) / (16 * V_THREADS);
  };
  int split = P.kparts;
  for (int k = P.kparts * 2, i = P.kparts == 1 ? 1 : P.kparts == 2 ? 2 : 3; k <= 8 && k <= P.steps; k *= 2, ++i)
    if (g_clusters[device][i] > 0 && longest(k) < longest(split)) split = k;
  P.kparts = split;
  // What a choice comes to: the sums of a cluster's units lie next to x, so where x leaves little room there are more clusters
  // than the device holds at once, in rounds that lay out x again.
  struct Plan {
    long long clusters, rounds;
    double time;  // in steps of a warp and 8 columns, as above, with what a round costs at the least
  };
  auto plan = [&](int group, int kparts) {
    const int sets = (rows + group - 1) / group, i = kparts == 1 ? 0 : kparts == 2 ? 1 : kparts == 4 ? 2 : 3;
    const long long x = x_bytes(group, kparts), room = (V_SMEM_MAX - x) / (128LL * group) - 2 * V_WARPS;
    const long long at_once = g_clusters[device][i] < 1 ? 1 : g_clusters[device][i];
    Plan p;
    p.clusters = at_once / sets < 1 ? 1 : at_once / sets > P.units ? P.units : at_once / sets;
    if (P.units > p.clusters * room) p.clusters = (P.units + room - 1) / room;
    p.rounds = (p.clusters * sets + at_once - 1) / at_once;
    const long long pairs = (P.units + p.clusters - 1) / p.clusters * ((P.steps + kparts - 1) / kparts);
    const double step[4] = {1.0, 1.3, 1.6, 1.7};  // of 8, 16, 24 and 32 columns
    p.time = p.rounds * (0.5 + pairs * step[(group * parts - 1) / 8] / V_WARPS + 0.4 * x / (16 * V_THREADS) + 0.25 * (kparts > 1));
    return p;
  };
  Plan chosen = plan(P.group, P.kparts);
  // Several rounds: the least of all choices that fit. (18432 x 9216: 7 f32 rows 309 -> 93 us as four sets of two, 12 bf16 rows
  // 225 -> 63, 16 f16 rows of 19456 x 2560: 55 -> 37; over 24 such sizes the choice is within a tenth of the best one.)
  if (chosen.rounds > 1) {
    for (int group = 1; group <= rows && group * parts <= 32; ++group)
      for (int kparts = 1, i = 0; kparts <= 8 && kparts <= P.steps; kparts *= 2, ++i) {
        if (g_clusters[device][i] < 1 || x_bytes(group, kparts) + (2 * V_WARPS + 1) * 128LL * group > V_SMEM_MAX) continue;
        const Plan p = plan(group, kparts);
        if (p.time < chosen.time) chosen = p, P.group = group, P.kparts = kparts;
      }
  }
  const int groups = (rows + P.group - 1) / P.group;
  const long long clusters = chosen.clusters;
  P.part_steps = (P.steps + P.kparts - 1) / P.kparts;
  P.clusters = static_cast<int>(clusters);
  const size_t smem = static_cast<size_t>(V_RING + x_bytes(P.group, P.kparts) +
                                          ((P.units + clusters - 1) / clusters + 2 * V_WARPS) * 128 * P.group);
  const dim3 grid(static_cast<unsigned>(clusters * P.kparts), groups);
  cudaError_t e;
#define FX_V(NH, PARTS) e = w.format == 16 ? v_launch<NH, PARTS, 16>(grid, smem, st, P) : v_launch<NH, PARTS, 32>(grid, smem, st, P)
  const int nh = (P.group * parts + 7) / 8;
  if (parts == 1) {
    if (nh == 1) FX_V(1, 1);
    else FX_V(2, 1);
  } else if (parts == 2) {
    if (nh == 1) FX_V(1, 2);
    else if (nh == 2) FX_V(2, 2);
    else FX_V(4, 2);
  } else {
    if (nh == 1) FX_V(1, 3);
    else if (nh == 2) FX_V(2, 3);
    else if (nh == 3) FX_V(3, 3);
    else FX_V(4, 3);
  }
#undef FX_V
  return e;
}

}  // namespace fx
