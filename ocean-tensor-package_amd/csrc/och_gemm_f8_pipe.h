/* The block-scaled product of large aligned operands to half and bfloat16, on tiles of 256 x 256.
 *
 * Eight waves, two per SIMD, own 128 x 64 of the tile each: 128 accumulator registers, so that the multiply-adds outside the
 * matrix cores (32 for every row of blocks) need no moves between register files, and a second wave on the SIMD whose
 * matrix instructions run beside them. The slab's 64 KB go from memory straight to LDS: an element is loaded once per 256
 * of the other operand, half of what 128 x 128 tiles load. Step i of a slab multiplies row i of blocks while the fragment of
 * row i + 1 is read and the sums of row i - 1 are scaled and added. The one barrier of a slab stands in front of its last
 * step, when the fragments of that step are in registers: behind it the next slab is complete, its first fragments are read
 * during the last step, and this slab's buffer is free. The loads of the slab after the next go there, two or three to a
 * step: a wave that issues all nine in a row waits for the memory pipe instead of multiplying (8192^3 on equal codes: 385 us,
 * spread over a step each 405, two or three to a step 358, with the barrier and the first fragments moved into the last
 * step 340).
 *
 * 8192^3 to bfloat16: 340 us, 3.24 PFLOP/s, when all codes are equal (bare loops of these matrix instructions and additions:
 * 4.5 PFLOP/s on equal codes, 3.3 on changing ones), 465 us, 2.36 PFLOP/s, on random codes: what bounds it is the power that
 * changing operand bits draw. Orders of the tiles, fragments read further ahead, wave priorities and two barriers with one
 * and a half slabs in flight changed nothing or lost; 32 x 32 x 64 instructions are 8 % slower. */
#pragma once
#include "och_gemm_f8_tile.h"
#pragma clang diagnostic ignored "-Winline-asm"

namespace och {

#define OCH_F8_PIPE 256
#define OCH_F8_PIPE_THREADS 512

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
   const uint32_t whole = p.K / OCH_F8_SLAB, slabs = (p.K + OCH_F8_SLAB - 1) / OCH_F8_SLAB;
   /* load x (0 .. 8) of slab s, which goes to buffer s mod 2 */
   auto load = [&](int x, uint32_t s)
   {  const uint32_t buf = lds0 + (s & 1) * BUF;
      if (x < 8)
      {  if (x % 2) lb.issue(x / 2, nextB, buf + OPERAND + 4096 * wave);
         else       la.issue(x / 2, nextA, buf + 4096 * wave);
      }
      else
      {  load_float_to_lds(nextS, scale_offset, buf + SCALES + 256 * wave);
         nextA += stepA; nextB += stepB; nextS += scale_step;
      }
   };
   /* the slab inside which K ends: chunk by chunk through registers (once per tile, not overlapped with anything) */
   auto load_rest = [&]()
   {  const uint32_t buf = (whole & 1) * BUF;
      uint32_t q = threadIdx.x;
      asm volatile("" : "+v"(q));                 /* nothing of this is worth a register in the loop */
#pragma unroll 1
      for (; q < F8Slab<AKC, R>::CHUNKS; q += THREADS)
      {  const och_u32x4 va = f8_any_chunk<AKC, R>(p.A, p.ldA, m0, whole * OCH_F8_SLAB, p.M, p.K, q), vb = f8_any_chunk<BKC, R>(p.B, p.ldB, n0, whole * OCH_F8_SLAB, p.N, p.K, q);
         *reinterpret_cast<och_u32x4 *>(lds + buf + 16 * q) = va;
         *reinterpret_cast<och_u32x4 *>(lds + buf + OPERAND + 16 * q) = vb;
      }
      load_float_to_lds(nextS, scale_offset, lds0 + buf + SCALES + 256 * wave);
   };
   och_i32x8 a, b[TJ]; float ta = 1, t[TJ], told[TJ];            /* told: the slab before's */
   och_f32x4v part[2][TJ], rs = zero;
#pragma unroll
   for (int j = 0; j < TJ; j++) { part[(TI - 1) % 2][j] = zero; told[j] = 0; }
   auto scales_of = [&](const char *buf) { return reinterpret_cast<const float *>(buf + SCALES); };
   auto column = [&](const char *buf, int j)
   {  b[j] = f8_fragment<BKC, R>(buf + OPERAND, wn + 16 * j);
      t[j] = scales_of(buf)[R + wn + 16 * j + lane % 16];
   };
   auto row_scales = [&](const char *buf, int i) { if (ROWS) rs = *reinterpret_cast<const och_f32x4v *>(scales_of(buf) + wm + 16 * i + 4 * (lane / 16)); };
   auto multiply = [&](int i, int j, const och_i32x8 &now)
   {  part[i % 2][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(now, b[j], zero, E5A ? 1 : 0, E5B ? 1 : 0, 0, 0, 0, 0); };
   /* the sums of block (i, j), scaled; the empty statement keeps the addition where it is written */
   auto add = [&](int i, int j, const float (&w)[TJ])
   {
#pragma unroll
      for (int r = 0; r < 4; r++) acc[i][j][r] = __builtin_fmaf(part[i % 2][j][r], ROWS ? rs[r] * w[j] : w[j], acc[i][j][r]);
      asm volatile("" : "+v"(acc[i][j]));
   };
   if (slabs > 0)
   {  if (whole > 0)
      {
#pragma unroll
         for (int x = 0; x < 9; x++) load(x, 0);
      }
      else load_rest();
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      if (whole > 1) { load(0, 1); load(1, 1); }
      else if (slabs > 1) load_rest();
      a = f8_fragment<AKC, R>(lds, wm);
      if (!ROWS) ta = scales_of(lds)[wm];
#pragma unroll
      for (int j = 0; j < TJ; j++) column(lds, j);
      for (uint32_t s = 0; s < slabs; s++)
      {  const char *buf = lds + (s & 1) * BUF, *next = lds + ((s + 1) & 1) * BUF;
         const bool more = s + 1 < whole;                      /* slab s + 1 is being loaded */
#pragma unroll
         for (int i = 0; i < TI - 1; i++)
         {  const och_i32x8 now = a;
            if (more)
            {  if (i == 0) { load(2, s + 1); load(3, s + 1); load(4, s + 1); }
               if (i == 1) { load(5, s + 1); load(6, s + 1); }
               if (i == 2) { load(7, s + 1); load(8, s + 1); }
            }
            a = f8_fragment<AKC, R>(buf, wm + 16 * (i + 1));
            if (i > 0) row_scales(buf, i - 1);                 /* (row 0 finds those of the slab before's last row) */
#pragma unroll
            for (int j = 0; j < TJ; j++) multiply(i, j, now);
#pragma unroll
            for (int j = 0; j < TJ; j++) { if (i == 0) add(TI - 1, j, told); else add(i > 0 ? i - 1 : 0, j, t); }
            if (i == 0 && !ROWS)
            {
#pragma unroll
               for (int j = 0; j < TJ; j++) t[j] *= ta;
            }
#pragma unroll
            for (int j = 0; j < TJ; j++) { __builtin_amdgcn_sched_group_barrier(0x8, 1, 0); __builtin_amdgcn_sched_group_barrier(0x2, ROWS ? 8 : 4, 0); }
            __builtin_amdgcn_sched_barrier(0);
         }
         och_f32x4v last = zero;
         if (ROWS) { row_scales(buf, TI - 1); last = rs; row_scales(buf, TI - 2); }
         asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
         __syncthreads();
         if (s + 2 < whole) { load(0, s + 2); load(1, s + 2); }
         else if (s + 2 == whole && slabs > whole) load_rest();
         const och_i32x8 now = a;
         a = f8_fragment<AKC, R>(next, wm);                    /* (behind the last slab: of no use, and none is made of it) */
         if (!ROWS) ta = scales_of(next)[wm];
#pragma unroll
         for (int j = 0; j < TJ; j++)
         {  multiply(TI - 1, j, now);
            add(TI - 2, j, t);
            told[j] = t[j];
            column(next, j);
            __builtin_amdgcn_sched_barrier(0);
         }
         rs = last;
      }
   }
#pragma unroll
   for (int j = 0; j < TJ; j++) add(TI - 1, j, told);
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
      if (p.dtypeC == OCH_HALF) f8_store_columns<OCH_HALF, R, PITCH, HALF, THREADS>(p, lds, m0, n0 + pass * HALF);
      else                      f8_store_columns<OCH_BFLOAT16, R, PITCH, HALF, THREADS>(p, lds, m0, n0 + pass * HALF);
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
