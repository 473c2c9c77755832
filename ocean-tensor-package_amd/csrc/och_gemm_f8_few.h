/* The block-scaled product for few columns (at most 64 tokens), both operands contiguous along k and 16-byte aligned: what
 * a decoding step asks for. It reads every code of A once, so memory bounds it; the matrix instructions, of which most
 * columns may be idle, are nearly free.
 *
 * A workgroup owns 16 TM rows of A and all columns; its W waves share out the slabs of 128 k (wave w takes slabs w, w + W,
 * ...), so that a few thousand waves are in flight whatever M is. The workgroups of a die (every eighth) begin at different
 * slabs, or else they would all read the same k of rows that lie a power of two apart, which one channel of the die's cache
 * serves: 8192 x 16 x 8192 14.8 us instead of 19.2. Every wave has a slot of its own in LDS that loads from memory fill
 * directly, eight rows of 128 consecutive bytes per load: with fragments loaded straight into registers a load covers sixteen
 * rows of 64 bytes, which the first-level cache serves at 15 instead of 38 bytes a cycle. No wave waits for another before the
 * end, where the waves' sums meet in LDS and are added in the order of the waves. Two tiles of rows share the columns' codes
 * where there are more than 16 columns and rows enough: these come from the second-level cache once per workgroup and slab.
 *
 * Measured, three sets of operands in turn: 14336 x 1 x 4096 10.5 us (5.6 TB/s), 8192 x 16 x 8192 11.8 us (5.7 TB/s), 8192 x
 * 48 x 8192 14.5 us (4.7 TB/s). Every 16 columns more cost 1.5 to 3 us, their codes being read by all 256 workgroups. Two slots
 * per wave, the next but one slab under way, change nothing at these sizes. On 128 x 128 tiles 16, 22 and 22 us. */
#pragma once
#include "och_gemm_f8_tile.h"
#pragma clang diagnostic ignored "-Winline-asm"

namespace och {

#define OCH_F8_STREAM (192u << 20)      /* bytes of A from which on it is loaded past the caches, whose last level holds 256 MB */

static constexpr uint32_t f8_few_waves(int TN) { return TN == 1 ? 16 : 8; }      /* at most, per workgroup: more than 16 columns need over 128 registers */
static constexpr uint32_t f8_few_slot(int TM, int TN) { return (uint32_t)(TM + TN) * 16 * OCH_F8_SLAB + 512; }      /* codes, 64 scales of A, 64 of B */

/* sixteen bytes per lane from memory to LDS as load_to_lds moves them, past the caches */
static __device__ __forceinline__ void stream_to_lds(const char *base, uint32_t offset, uint32_t target)
{
   asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt" : : "s"(target), "v"(offset), "s"(base) : "memory");
}

/* `stream`: A is larger than what the caches could hold until the next call (28672 x 1 x 8192: 37.5 us past them, 43.1 through
   them; A's of 60 MB that take turns in them: 12.2 and 10.7) */
template <bool E5A, bool E5B, bool WIDE, int TM, int TN>
__global__ __launch_bounds__(64 * f8_few_waves(TN)) void gemm_f8_few_kernel(const F8GemmParams p, bool stream)
{
   typedef F8Slab<true, 32> L;
   constexpr uint32_t SLOT = f8_few_slot(TM, TN), SLOT_B = TM * 16 * OCH_F8_SLAB, SLOT_SCALES = SLOT - 512;
   extern __shared__ __align__(16) char lds_few[];
   const uint32_t lane = threadIdx.x & 63, g = lane / 16, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), W = blockDim.x / 64;
   const uint32_t m0 = blockIdx.x * 16 * TM;
   char *slot = lds_few + wave * SLOT;
   const uint32_t target = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)slot;
   const och_f32x4v zero = { 0, 0, 0, 0 };
   och_f32x4v acc[TM][TN];

   /* the wave's loads: load e covers rows 8 e .. + 7 of A (then columns of B), lane l the l mod 8-th slot of row l / 8;
      rows and columns that do not exist repeat the last one */
   uint32_t row0, k0, oa[2 * TM], ob[2 * TN];
   L::where(lane, row0, k0);
   const char *rowsA = (const char *)p.A + (int64_t)m0 * p.ldA, *rowsB = (const char *)p.B;
#pragma unroll
   for (int e = 0; e < 2 * TM; e++)
   {  const uint32_t r = row0 + 8 * e, last = p.M - 1 - m0;
      oa[e] = (r < last ? r : last) * (uint32_t)p.ldA + k0;
   }
#pragma unroll
   for (int e = 0; e < 2 * TN; e++)
   {  const uint32_t r = row0 + 8 * e, last = p.N - 1;
      ob[e] = (r < last ? r : last) * (uint32_t)p.ldB + k0;
   }
   /* lane l brings the scales of row l and of column l */
   const uint32_t last_row = p.M - 1 - m0 < 16 * TM - 1 ? p.M - 1 - m0 : 16 * TM - 1, last_column = p.N - 1 < 16 * TN - 1 ? p.N - 1 : 16 * TN - 1;
   const uint32_t osa = (((m0 + (lane < last_row ? lane : last_row)) >> p.shiftA) - (m0 >> p.shiftA)) * (uint32_t)p.sa_m * 4;
   const uint32_t osb = ((lane < last_column ? lane : last_column) >> p.shiftB) * (uint32_t)p.sb_n * 4;
   const char *scalesA = (const char *)(p.SA + (int64_t)(m0 >> p.shiftA) * p.sa_m), *scalesB = (const char *)p.SB;
#pragma unroll
   for (int i = 0; i < TM; i++)
#pragma unroll
      for (int j = 0; j < TN; j++) acc[i][j] = zero;
   auto fetch = [&](uint32_t s)
   {  if (stream)
      {
#pragma unroll
         for (int e = 0; e < 2 * TM; e++) stream_to_lds(rowsA + (uint64_t)s * OCH_F8_SLAB, oa[e], target + 1024 * e);
      }
      else
      {
#pragma unroll
         for (int e = 0; e < 2 * TM; e++) load_to_lds(rowsA + (uint64_t)s * OCH_F8_SLAB, oa[e], target + 1024 * e);
      }
#pragma unroll
      for (int e = 0; e < 2 * TN; e++) load_to_lds(rowsB + (uint64_t)s * OCH_F8_SLAB, ob[e], target + SLOT_B + 1024 * e);
      load_float_to_lds(scalesA + (int64_t)s * p.sa_k * 4, osa, target + SLOT_SCALES);
      load_float_to_lds(scalesB + (int64_t)s * p.sb_k * 4, osb, target + SLOT_SCALES + 256);
   };
   /* the slot's slab: fragments to registers, then (the slot is free) `next`, then the product */
   auto use = [&](auto next)
   {  och_i32x8 ca[TM], cb[TN]; och_f32x4v r0[TM]; float t0[TN];
      const float *rs = reinterpret_cast<const float *>(slot + SLOT_SCALES), *t = rs + 64;
#pragma unroll
      for (int i = 0; i < TM; i++) { ca[i] = f8_fragment<true, 32>(slot, 16 * i); r0[i] = *reinterpret_cast<const och_f32x4v *>(rs + 16 * i + 4 * g); }
#pragma unroll
      for (int j = 0; j < TN; j++) { cb[j] = f8_fragment<true, 32>(slot + SLOT_B, 16 * j); t0[j] = t[16 * j + lane % 16]; }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      next();
      F8Operand<WIDE> fb[TN];
#pragma unroll
      for (int j = 0; j < TN; j++) fb[j].template set<E5B>(cb[j]);
#pragma unroll
      for (int i = 0; i < TM; i++)
      {  F8Operand<WIDE> fa;
         fa.template set<E5A>(ca[i]);
#pragma unroll
         for (int j = 0; j < TN; j++)
         {  const och_f32x4v part = f8_block<E5A, E5B>(fa, fb[j]);
#pragma unroll
            for (int r = 0; r < 4; r++) acc[i][j][r] = __builtin_fmaf(part[r], r0[i][r] * t0[j], acc[i][j][r]);
         }
      }
   };
   const uint32_t whole = p.K / OCH_F8_SLAB, turns = wave < whole ? (whole - wave + W - 1) / W : 0;
   uint32_t turn = turns ? blockIdx.x / 8 % turns : 0;
   if (turns) fetch(wave + turn * W);
   for (uint32_t i = 0; i < turns; i++)
   {  turn = turn + 1 < turns ? turn + 1 : 0;
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      use([&]() { if (i + 1 < turns) fetch(wave + turn * W); });
   }
   if (p.K % OCH_F8_SLAB != 0 && whole % W == wave)
   {  /* the rest of K: its chunks through registers, zeros behind the end */
      const int64_t valid = (int64_t)(p.K % OCH_F8_SLAB) - k0;
#pragma unroll
      for (int e = 0; e < 2 * TM; e++)
         *reinterpret_cast<och_u32x4 *>(slot + 1024 * e + 16 * lane) = f8_border_chunk((const uint8_t *)rowsA + (uint64_t)whole * OCH_F8_SLAB + oa[e], valid, p.K);
#pragma unroll
      for (int e = 0; e < 2 * TN; e++)
         *reinterpret_cast<och_u32x4 *>(slot + SLOT_B + 1024 * e + 16 * lane) = f8_border_chunk((const uint8_t *)rowsB + (uint64_t)whole * OCH_F8_SLAB + ob[e], valid, p.K);
      float *rest = reinterpret_cast<float *>(slot + SLOT_SCALES);
      rest[lane] = *reinterpret_cast<const float *>(scalesA + (int64_t)whole * p.sa_k * 4 + osa);
      rest[64 + lane] = *reinterpret_cast<const float *>(scalesB + (int64_t)whole * p.sb_k * 4 + osb);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      use([]() { });
   }
   __syncthreads();
   /* wave w's sums: [w][column][row], a column's rows together */
   constexpr uint32_t COLUMN = 16 * TM, PLANE = COLUMN * 16 * TN;
   static_assert(PLANE * 4 <= SLOT, "the sums lie where the slots were");
   float *mine = reinterpret_cast<float *>(lds_few) + wave * PLANE;
#pragma unroll
   for (int j = 0; j < TN; j++)
#pragma unroll
      for (int i = 0; i < TM; i++) *reinterpret_cast<och_f32x4v *>(mine + (16 * j + lane % 16) * COLUMN + 16 * i + 4 * g) = acc[i][j];
   __syncthreads();
   for (uint32_t e = threadIdx.x; e < PLANE / 4; e += blockDim.x)
   {  const uint32_t n = e / (COLUMN / 4), m = m0 + e % (COLUMN / 4) * 4;
      if (n >= p.N || m >= p.M) continue;
      och_f32x4v v = zero;
      for (uint32_t w = 0; w < W; w++) v += *reinterpret_cast<const och_f32x4v *>(reinterpret_cast<const float *>(lds_few) + w * PLANE + 4 * e);
      const int64_t at = (int64_t)m + (int64_t)n * p.ldC;
      if (p.dtypeC == OCH_FLOAT)     f8_finish4<OCH_FLOAT>(p.C, at, v, p.alpha, p.beta, p.M - m);
      else if (p.dtypeC == OCH_HALF) f8_finish4<OCH_HALF>(p.C, at, v, p.alpha, p.beta, p.M - m);
      else                           f8_finish4<OCH_BFLOAT16>(p.C, at, v, p.alpha, p.beta, p.M - m);
   }
}

template <bool E5A, bool E5B, bool WIDE, int TM, int TN> static int gemm_f8_few_launch(const F8GemmParams &p, hipStream_t stream)
{
   auto kernel = gemm_f8_few_kernel<E5A, E5B, WIDE, TM, TN>;
   /* waves per workgroup: eight per compute unit over all, no more than slabs or than their slots fit into 160 KB */
   const uint32_t slabs = (uint32_t)(((uint64_t)p.K + OCH_F8_SLAB - 1) / OCH_F8_SLAB), groups = (p.M + 16 * TM - 1) / (16 * TM);
   uint32_t waves = (uint32_t)((8ull * gemm_compute_units() + groups - 1) / groups);
   if (waves > f8_few_waves(TN)) waves = f8_few_waves(TN);
   if (waves > slabs) waves = slabs > 0 ? slabs : 1;
   if (waves > 163840 / f8_few_slot(TM, TN)) waves = 163840 / f8_few_slot(TM, TN);
   if (groups > most_groups(64 * waves)) return set_error("gemm_scaled: a result of %u x %u has too many tiles", p.M, p.N);
   const size_t lds = (size_t)waves * f8_few_slot(TM, TN);
   if (lds > 65536) OCH_CHECK_HIP(hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
   hipLaunchKernelGGL(kernel, dim3(groups), dim3(64 * waves), lds, stream, p, (uint64_t)p.M * p.K >= OCH_F8_STREAM);
   OCH_CHECK_LAUNCH();
   return 0;
}
/* Up to 32 columns the bfloat16 instructions take 0.5 to 1.5 % more time (8192 x 16 x 8192 11.76 us and 11.71, 8192 x 32 x 8192
   13.0 and 12.8, 14336 x 1 x 4096 10.5 and 10.4), so 16-bit results have float sums as well. With more columns they would take 3 to
   20 % (8192 x 48 x 8192 15.4 us and 14.5, 14336 x 64 x 4096 with a scale per row of A 22.6 and 18.8). */
template <bool E5A, bool E5B> static int gemm_f8_few(const F8GemmParams &p, hipStream_t stream)
{
   if (p.N <= 16) return gemm_f8_few_launch<E5A, E5B, true, 1, 1>(p, stream);
   /* single tiles of rows where pairs would leave compute units idle: 4096 x 32 x 14336 12.9 us against 16.2 */
   const bool single = p.M <= 16u * (uint32_t)gemm_compute_units(), wide = p.dtypeC == OCH_FLOAT;
   if (p.N <= 32) return single ? gemm_f8_few_launch<E5A, E5B, true, 1, 2>(p, stream) : gemm_f8_few_launch<E5A, E5B, true, 2, 2>(p, stream);
#define OCH_GO(TN) (single ? (wide ? gemm_f8_few_launch<E5A, E5B, true, 1, TN>(p, stream) : gemm_f8_few_launch<E5A, E5B, false, 1, TN>(p, stream)) \
                           : (wide ? gemm_f8_few_launch<E5A, E5B, true, 2, TN>(p, stream) : gemm_f8_few_launch<E5A, E5B, false, 2, TN>(p, stream)))
   return p.N <= 48 ? OCH_GO(3) : OCH_GO(4);
#undef OCH_GO
}

} /* namespace och */
