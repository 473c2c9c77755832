/* The block-scaled product of large aligned operands to half and bfloat16, on tiles of 256 x 256.
 *
 * Eight waves, two per SIMD, own 128 x 64 of the tile each: 128 accumulator registers, so that the multiply-adds outside the
 * matrix cores (32 for every row of blocks) need no moves between register files, and a second wave on the SIMD whose
 * matrix instructions run beside them (bare loops: 1.7 PFLOP/s with one wave per SIMD, 3.4 with two, 4.1 without the
 * multiply-adds). The slab's 64 KB go from memory straight to LDS, one slab ahead of the matrix instructions, with one
 * barrier per slab: an element is loaded once per 256 of the other operand, half of what 128 x 128 tiles load. Row i of
 * blocks is multiplied while the fragment of row i + 1 is read and the sums of row i - 1 are scaled and added.
 *
 * 8192^3 from e4m3 codes of Gaussian data to bfloat16: 480 us, 2.29 PFLOP/s; 384 us (2.86) when all codes are equal. The
 * difference is the power that changing operand bits draw, which is the bound: orders of the tiles, fragments read further
 * ahead or before the barrier, wave priorities and 32 x 32 x 64 instructions (8 % slower) change neither figure. */
#pragma once
#include "och_gemm_f8_tile.h"
#pragma clang diagnostic ignored "-Winline-asm"

namespace och {

#define OCH_F8_PIPE 256
#define OCH_F8_PIPE_THREADS 512

/* one float per lane from memory to LDS, as load_to_lds moves sixteen bytes */
static __device__ __forceinline__ void load_float_to_lds(const char *base, uint32_t offset, uint32_t target)
{
   asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" : : "s"(target), "v"(offset), "s"(base) : "memory");
}

/* The four loads of a slab's 256 rows that a wave issues, 1 KB each: chunks 64 (4 wave + e) + lane. Rows that do not exist
   repeat the last (KC) or the last sixteen (!KC: the number of rows is a multiple of 16 there). */
template <bool KC> struct F8PipeLoads
{
   typedef F8Slab<KC, OCH_F8_PIPE> L;
   uint32_t offset[4];                    /* bytes from the slab's first element */
   __device__ __forceinline__ void start(uint32_t wave, uint32_t lane, int64_t ld, uint32_t rows)
   {
#pragma unroll
      for (int e = 0; e < 4; e++)
      {  uint32_t row, k;
         L::where(64 * (4 * wave + e) + lane, row, k);
         const uint32_t last = KC ? rows - 1 : rows - 16;
         row = row < last ? row : last;
         offset[e] = KC ? row * (uint32_t)ld + k : row + k * (uint32_t)ld;
      }
   }
   __device__ __forceinline__ void issue(int e, const char *slab, uint32_t target) const { load_to_lds(slab, offset[e], target + 1024 * e); }
};

/* COLUMNS columns of R rows of finished sums from LDS to C */
template <int DT, int R, uint32_t PITCH, uint32_t COLUMNS, int THREADS> __device__ __forceinline__ void f8_pipe_write(const F8GemmParams &p, const char *lds, uint32_t m0, uint32_t n0)
{
   typedef typename Wide<DT>::E E;
#pragma unroll 1
   for (uint32_t q = threadIdx.x; q < COLUMNS * (R / 8); q += THREADS)
   {  const uint32_t c = q / (R / 8), m = m0 + q % (R / 8) * 8, n = n0 + c;
      if (m >= p.M || n >= p.N) continue;
      const och_f32x4v *from = reinterpret_cast<const och_f32x4v *>(lds + c * PITCH + q % (R / 8) * 32);
      const och_f32x4v lo = from[0], hi = from[1];
      E *to = reinterpret_cast<E *>(p.C) + (int64_t)m + (int64_t)n * p.ldC;
      const int64_t valid = (int64_t)p.M - m;
      Wide8<DT> v;
      if (p.beta != 0.0f) v.load(to, valid);
#pragma unroll
      for (int e = 0; e < 8; e++)
      {  float x = p.alpha * (e < 4 ? lo[e % 4] : hi[e % 4]);
         if (p.beta != 0.0f) x = __builtin_fmaf(p.beta, v.get(e), x);
         v.put(e, x);
      }
      v.store(to, valid);
   }
}

template <bool AKC, bool BKC, bool E5A, bool E5B, bool ROWS>
__global__ __launch_bounds__(OCH_F8_PIPE_THREADS, 2) void gemm_f8_pipe_kernel(const F8GemmParams p)
{
   constexpr int R = OCH_F8_PIPE, THREADS = OCH_F8_PIPE_THREADS, TI = 8, TJ = 4;
   constexpr uint32_t OPERAND = R * OCH_F8_SLAB, SCALES = 2 * OPERAND, BUF = 2 * OPERAND + 2 * R * 4;
   extern __shared__ __align__(16) char lds_pipe[];
   char *const lds = lds_pipe;
   uint32_t tm, tn;
   f8_tile_of(blockIdx.x, p.tiles_m, p.tiles_n, tm, tn);
   const uint32_t m0 = tm * R, n0 = tn * R;
   const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave % 2 * 128, wn = wave / 2 * 64;
   const och_f32x4v zero = { 0, 0, 0, 0 };
   och_f32x4v acc[TI][TJ];
#pragma unroll
   for (int i = 0; i < TI; i++)
#pragma unroll
      for (int j = 0; j < TJ; j++) acc[i][j] = zero;

   F8PipeLoads<AKC> la; F8PipeLoads<BKC> lb;
   la.start(wave, lane, p.ldA, p.M - m0); lb.start(wave, lane, p.ldB, p.N - n0);
   const char *nextA = (const char *)p.A + (AKC ? (int64_t)m0 * p.ldA : (int64_t)m0), *nextB = (const char *)p.B + (BKC ? (int64_t)n0 * p.ldB : (int64_t)n0);
   const int64_t stepA = AKC ? OCH_F8_SLAB : OCH_F8_SLAB * p.ldA, stepB = BKC ? OCH_F8_SLAB : OCH_F8_SLAB * p.ldB;
   /* waves 0 .. 3 bring the scales of 64 rows of A each, 4 .. 7 those of columns of B */
   const bool forA = wave < 4;
   const uint32_t line = (forA ? m0 : n0) + 64 * (wave % 4) + lane, most = (forA ? p.M : p.N) - 1;
   const int64_t scale_line = forA ? p.sa_m : p.sb_n, scale_step = (forA ? p.sa_k : p.sb_k) * 4;
   const uint32_t scale_first = (forA ? m0 : n0) >> (forA ? p.shiftA : p.shiftB);
   const char *nextS = (const char *)((forA ? p.SA : p.SB) + (int64_t)scale_first * scale_line);
   const uint32_t scale_offset = (((line < most ? line : most) >> (forA ? p.shiftA : p.shiftB)) - scale_first) * (uint32_t)scale_line * 4;
   const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
   auto fetch = [&](uint32_t buf)
   {
#pragma unroll
      for (int e = 0; e < 4; e++) { la.issue(e, nextA, buf + 4096 * wave); lb.issue(e, nextB, buf + OPERAND + 4096 * wave); }
      load_float_to_lds(nextS, scale_offset, buf + SCALES + 256 * wave);
      nextA += stepA; nextB += stepB; nextS += scale_step;
   };
   const uint32_t whole = p.K / OCH_F8_SLAB, end = (p.K + OCH_F8_SLAB - 1) / OCH_F8_SLAB;
   if (whole > 0) fetch(lds0);
   for (uint32_t s = 0, turn = 0; s < end; s++, turn ^= 1)
   {  char *buf = lds + turn * BUF;
      const float *sA = reinterpret_cast<const float *>(buf + SCALES), *sB = sA + R;
      if (s >= whole)
      {  /* the rest of K, chunk by chunk through registers */
         F8Stage<AKC, R, THREADS> ra; F8Stage<BKC, R, THREADS> rb;
         __syncthreads();
         ra.load_border(p.A, p.ldA, m0, s * OCH_F8_SLAB, p.M, p.K); ra.store(buf, false);
         rb.load_border(p.B, p.ldB, n0, s * OCH_F8_SLAB, p.N, p.K); rb.store(buf + OPERAND, false);
         load_float_to_lds(nextS, scale_offset, lds0 + turn * BUF + SCALES + 256 * wave);
      }
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      if (s + 1 < whole) fetch(lds0 + (turn ^ 1) * BUF);
      och_i32x8 b[TJ]; float t[TJ];
#pragma unroll
      for (int j = 0; j < TJ; j++)
      {  b[j] = f8_fragment<BKC, R>(buf + OPERAND, wn + 16 * j);
         t[j] = sB[wn + 16 * j + lane % 16];
         if (!ROWS) t[j] *= sA[wm];
      }
      och_i32x8 a = f8_fragment<AKC, R>(buf, wm);
      och_f32x4v part[2][TJ], rs[2];
#pragma unroll
      for (int i = 0; i <= TI; i++)
      {  if (i < TI)
         {  const och_i32x8 now = a;
            if (i < TI - 1) a = f8_fragment<AKC, R>(buf, wm + 16 * (i + 1));
            if (ROWS) rs[i % 2] = *reinterpret_cast<const och_f32x4v *>(sA + wm + 16 * i + 4 * (lane / 16));
#pragma unroll
            for (int j = 0; j < TJ; j++) part[i % 2][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(now, b[j], zero, E5A ? 1 : 0, E5B ? 1 : 0, 0, 0, 0, 0);
         }
         if (i > 0)
         {  const int o = (i - 1) % 2, q = i > 0 ? i - 1 : 0;
#pragma unroll
            for (int j = 0; j < TJ; j++)
#pragma unroll
               for (int r = 0; r < 4; r++) acc[q][j][r] = __builtin_fmaf(part[o][j][r], ROWS ? rs[o][r] * t[j] : t[j], acc[q][j][r]);
#pragma unroll
            for (int j = 0; j < TJ; j++) asm volatile("" : "+v"(acc[q][j]));
         }
         if (i > 0 && i < TI)
         {
#pragma unroll
            for (int j = 0; j < TJ; j++) { __builtin_amdgcn_sched_group_barrier(0x8, 1, 0); __builtin_amdgcn_sched_group_barrier(0x2, ROWS ? 8 : 4, 0); }
         }
         __builtin_amdgcn_sched_barrier(0);
      }
   }
   /* C leaves through LDS, 128 columns at a time as floats with a pitch that spreads neighbouring columns over the banks, in
      pieces of eight rows: memory sees 512 consecutive bytes of a column */
   constexpr uint32_t PITCH = R * 4 + 16, HALF = 128;
   static_assert(HALF * PITCH <= 2 * BUF, "half a tile fits where the slabs were");
#pragma unroll 1
   for (uint32_t pass = 0; pass < 2; pass++)
   {  __syncthreads();
      if (wave / 4 == pass)
      {  char *mine = lds + (wn % HALF + lane % 16) * PITCH + (wm + 4 * (lane / 16)) * 4;
#pragma unroll
         for (int j = 0; j < TJ; j++)
#pragma unroll
            for (int i = 0; i < TI; i++) *reinterpret_cast<och_f32x4v *>(mine + 16 * j * PITCH + 64 * i) = acc[i][j];
      }
      __syncthreads();
      if (p.dtypeC == OCH_HALF) f8_pipe_write<OCH_HALF, R, PITCH, HALF, THREADS>(p, lds, m0, n0 + pass * HALF);
      else                      f8_pipe_write<OCH_BFLOAT16, R, PITCH, HALF, THREADS>(p, lds, m0, n0 + pass * HALF);
   }
}

template <bool E5A, bool E5B, bool ROWS> static int gemm_f8_pipe_launch(const F8GemmParams &p, bool akc, bool bkc, hipStream_t stream)
{
   const size_t lds = 2 * (2 * OCH_F8_PIPE * OCH_F8_SLAB + 2 * OCH_F8_PIPE * 4);
   auto go = [&](auto kernel) -> int
   {  OCH_CHECK_HIP(hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
      hipLaunchKernelGGL(kernel, dim3(p.tiles_m * p.tiles_n), dim3(OCH_F8_PIPE_THREADS), lds, stream, p);
      OCH_CHECK_LAUNCH();
      return 0;
   };
   return akc ? (bkc ? go(gemm_f8_pipe_kernel<true, true, E5A, E5B, ROWS>) : go(gemm_f8_pipe_kernel<true, false, E5A, E5B, ROWS>))
              : (bkc ? go(gemm_f8_pipe_kernel<false, true, E5A, E5B, ROWS>) : go(gemm_f8_pipe_kernel<false, false, E5A, E5B, ROWS>));
}
template <bool E5A, bool E5B> static int gemm_f8_pipe(const F8GemmParams &p, bool akc, bool bkc, hipStream_t stream)
{  return p.shiftA == 0 ? gemm_f8_pipe_launch<E5A, E5B, true>(p, akc, bkc, stream) : gemm_f8_pipe_launch<E5A, E5B, false>(p, akc, bkc, stream); }

} /* namespace och */
