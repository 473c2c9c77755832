/* och_gemm_scaled: products of 8-bit floats with one scale per block of 128 k (and per row or per 128 rows) of either
 * operand. No counterpart in the reference.
 *
 * The matrix cores multiply a whole block of 128 k (one v_mfma_f32_16x16x128_f8f6f4, or four bfloat16 ones where the
 * result is float); the 16 x 16 sums of a block are multiplied by the two scales and added to the float accumulators
 * outside them, four multiply-adds per lane beside 32 or 64 cycles of matrix work.
 */
#include "och_gemm_f8.h"

namespace och {

/* Any operands: a workgroup of four waves owns 64 x 64 of C (each wave 32 x 32); a slab of 128 k of both operands goes
   through registers to LDS. Chunks of 16 bytes that lie inside the matrix are one load, whatever their alignment; those
   at its border are loaded byte by byte, those outside are zero. */
template <bool KC, int R, int THREADS>
__device__ __forceinline__ void f8_load_slab(const uint8_t *mat, int64_t ld, uint32_t r0, uint32_t k0, uint32_t rows, uint32_t K, char *slab)
{
   typedef F8Slab<KC, R> L;
   constexpr int NV = (int)L::CHUNKS / THREADS;
   och_u32x4 v[NV];
#pragma unroll
   for (int i = 0; i < NV; i++)
   {  uint32_t row, k;
      L::where(threadIdx.x + THREADS * i, row, k);
      const int64_t gr = (int64_t)r0 + row, gk = (int64_t)k0 + k;
      const uint8_t *at = mat + (KC ? gk + gr * ld : gr + gk * ld);
      const int64_t valid = KC ? (gr < rows ? (int64_t)K - gk : 0) : (gk < K ? (int64_t)rows - gr : 0);
      if (valid >= 16) v[i] = *reinterpret_cast<const och_u32x4_any *>(at);
      else
      {  uint32_t w[4] = { 0, 0, 0, 0 };
#pragma unroll
         for (int e = 0; e < 16; e++) if (e < valid) w[e / 4] |= (uint32_t)at[e] << (8 * (e % 4));
         v[i].x = w[0]; v[i].y = w[1]; v[i].z = w[2]; v[i].w = w[3];
      }
   }
#pragma unroll
   for (int i = 0; i < NV; i++) *reinterpret_cast<och_u32x4 *>(slab + 16 * (threadIdx.x + THREADS * i)) = v[i];
}

template <bool AKC, bool BKC, bool E5A, bool E5B, bool WIDE>
__global__ __launch_bounds__(256) void gemm_f8_any_kernel(const F8GemmParams p)
{
   constexpr int R = 64;
   __shared__ __align__(16) char lds[2 * R * OCH_F8_SLAB];
   const uint32_t m0 = blockIdx.x % p.tiles_m * R, n0 = blockIdx.x / p.tiles_m * R;
   const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave % 2 * 32, wn = wave / 2 * 32;
   och_f32x4v acc[2][2];
   const och_f32x4v zero = { 0, 0, 0, 0 };
#pragma unroll
   for (int i = 0; i < 2; i++)
#pragma unroll
      for (int j = 0; j < 2; j++) acc[i][j] = zero;
   /* the scales of this lane's rows and columns; those outside C repeat the last one inside */
   const float *sa[2][4], *sb[2];
#pragma unroll
   for (int i = 0; i < 2; i++)
   {  const uint32_t n = n0 + wn + 16 * i + lane % 16;
      sb[i] = p.SB + (int64_t)((n < p.N ? n : p.N - 1) >> p.shiftB) * p.sb_n;
#pragma unroll
      for (int r = 0; r < 4; r++)
      {  const uint32_t m = m0 + wm + 16 * i + 4 * (lane / 16) + r;
         sa[i][r] = p.SA + (int64_t)((m < p.M ? m : p.M - 1) >> p.shiftA) * p.sa_m;
      }
   }
   const uint32_t slabs = (p.K + OCH_F8_SLAB - 1) / OCH_F8_SLAB;
   for (uint32_t s = 0; s < slabs; s++)
   {  f8_load_slab<AKC, R, 256>(p.A, p.ldA, m0, s * OCH_F8_SLAB, p.M, p.K, lds);
      f8_load_slab<BKC, R, 256>(p.B, p.ldB, n0, s * OCH_F8_SLAB, p.N, p.K, lds + R * OCH_F8_SLAB);
      __syncthreads();
      F8Operand<WIDE> a[2], b[2];
#pragma unroll
      for (int i = 0; i < 2; i++)
      {  a[i].template set<E5A>(f8_fragment<AKC, R>(lds, wm + 16 * i));
         b[i].template set<E5B>(f8_fragment<BKC, R>(lds + R * OCH_F8_SLAB, wn + 16 * i));
      }
#pragma unroll
      for (int j = 0; j < 2; j++)
      {  const float t = sb[j][(int64_t)s * p.sb_k];
#pragma unroll
         for (int i = 0; i < 2; i++)
         {  const och_f32x4v part = f8_block<E5A, E5B>(a[i], b[j]);
#pragma unroll
            for (int r = 0; r < 4; r++) acc[i][j][r] = __builtin_fmaf(part[r], sa[i][r][(int64_t)s * p.sa_k] * t, acc[i][j][r]);
         }
      }
      __syncthreads();
   }
#pragma unroll
   for (int j = 0; j < 2; j++)
   {  const uint32_t n = n0 + wn + 16 * j + lane % 16;
#pragma unroll
      for (int i = 0; i < 2; i++)
#pragma unroll
         for (int r = 0; r < 4; r++)
         {  const uint32_t m = m0 + wm + 16 * i + 4 * (lane / 16) + r;
            if (m >= p.M || n >= p.N) continue;
            const int64_t at = (int64_t)m + (int64_t)n * p.ldC;
            if (p.dtypeC == OCH_FLOAT)     f8_finish<OCH_FLOAT>(p.C, at, acc[i][j][r], p.alpha, p.beta);
            else if (p.dtypeC == OCH_HALF) f8_finish<OCH_HALF>(p.C, at, acc[i][j][r], p.alpha, p.beta);
            else                           f8_finish<OCH_BFLOAT16>(p.C, at, acc[i][j][r], p.alpha, p.beta);
         }
   }
}

template <bool E5A, bool E5B, bool WIDE> static int gemm_f8_any(F8GemmParams p, bool akc, bool bkc, hipStream_t stream)
{
   p.tiles_m = (p.M + 63) / 64; p.tiles_n = (p.N + 63) / 64;
   const uint64_t blocks = (uint64_t)p.tiles_m * p.tiles_n;
   if (blocks > 0x7FFFFFFFull) return set_error("gemm_scaled: too many tiles");
   const dim3 grid((unsigned)blocks);
   if (akc && bkc) hipLaunchKernelGGL((gemm_f8_any_kernel<true, true, E5A, E5B, WIDE>), grid, dim3(256), 0, stream, p);
   else if (akc)   hipLaunchKernelGGL((gemm_f8_any_kernel<true, false, E5A, E5B, WIDE>), grid, dim3(256), 0, stream, p);
   else if (bkc)   hipLaunchKernelGGL((gemm_f8_any_kernel<false, true, E5A, E5B, WIDE>), grid, dim3(256), 0, stream, p);
   else            hipLaunchKernelGGL((gemm_f8_any_kernel<false, false, E5A, E5B, WIDE>), grid, dim3(256), 0, stream, p);
   OCH_CHECK_LAUNCH();
   return 0;
}

/* float results take the wide sums, 16-bit ones the 8-bit matrix instruction */
template <bool E5A, bool E5B> static int gemm_f8_dispatch(const F8GemmParams &p, bool akc, bool bkc, hipStream_t stream)
{
   return p.dtypeC == OCH_FLOAT ? gemm_f8_any<E5A, E5B, true>(p, akc, bkc, stream) : gemm_f8_any<E5A, E5B, false>(p, akc, bkc, stream);
}

} /* namespace och */

using namespace och;

extern "C" int och_gemm_scaled(int dtypeA, int dtypeB, int dtypeC, char transA, char transB, size_t M, size_t N, size_t K, float alpha,
                               const void *A, ptrdiff_t ldA, const float *SA, ptrdiff_t ldSA, size_t blockA,
                               const void *B, ptrdiff_t ldB, const float *SB, ptrdiff_t ldSB, size_t blockB,
                               float beta, void *C, ptrdiff_t ldC, och_stream stream)
{
   if (!code_type(dtypeA) || !code_type(dtypeB)) return set_error("gemm_scaled: the operands are float8_e4m3 or float8_e5m2 (got %d, %d)", dtypeA, dtypeB);
   if (!wide_type(dtypeC)) return set_error("gemm_scaled: the result is half, bfloat16 or float (got %d)", dtypeC);
   if ((transA != 'N' && transA != 'T') || (transB != 'N' && transB != 'T')) return set_error("gemm_scaled: transposition flags are 'N' or 'T' (got '%c', '%c')", transA, transB);
   if ((blockA != 1 && blockA != OCH_F8_BLOCK) || (blockB != 1 && blockB != OCH_F8_BLOCK))
      return set_error("gemm_scaled: a scale covers 1 or 128 rows of op(A) and columns of op(B) (got %zu, %zu)", blockA, blockB);
   if (M == 0 || N == 0) return 0;
   if (M > 0x7FFFFFFFull || N > 0x7FFFFFFFull || K > 0x7FFFFF00ull) return set_error("gemm_scaled: a side of %zu x %zu x %zu is too long", M, N, K);
   if (C == nullptr) return set_error("gemm_scaled: null pointer argument");
   if (ldC < (ptrdiff_t)M) return set_error("gemm_scaled: ldC = %td is smaller than M = %zu", ldC, M);
   if ((uintptr_t)C % wide_size(dtypeC) != 0 || (uintptr_t)SA % 4 != 0 || (uintptr_t)SB % 4 != 0) return set_error("gemm_scaled: misaligned pointer");
   const bool akc = transA == 'T', bkc = transB == 'N';
   if (K > 0)
   {  if (A == nullptr || B == nullptr || SA == nullptr || SB == nullptr) return set_error("gemm_scaled: null pointer argument");
      const size_t kb = (K + OCH_F8_BLOCK - 1) / OCH_F8_BLOCK, mb = (M + blockA - 1) / blockA, nb = (N + blockB - 1) / blockB;
      if (ldA < (ptrdiff_t)(akc ? K : M) || ldB < (ptrdiff_t)(bkc ? K : N)) return set_error("gemm_scaled: ldA = %td or ldB = %td is smaller than its matrix", ldA, ldB);
      if (ldSA < (ptrdiff_t)(akc ? kb : mb) || ldSB < (ptrdiff_t)(bkc ? kb : nb)) return set_error("gemm_scaled: ldSA = %td or ldSB = %td is smaller than its matrix of scales", ldSA, ldSB);
   }
   F8GemmParams p;
   memset(&p, 0, sizeof(p));
   p.A = (const uint8_t *)A; p.B = (const uint8_t *)B; p.C = (char *)C; p.SA = SA; p.SB = SB; p.ldA = ldA; p.ldB = ldB; p.ldC = ldC;
   /* the scales of a matrix are a matrix of the same orientation */
   p.sa_m = akc ? ldSA : 1; p.sa_k = akc ? 1 : ldSA; p.sb_n = bkc ? ldSB : 1; p.sb_k = bkc ? 1 : ldSB;
   p.shiftA = blockA == 1 ? 0 : 7; p.shiftB = blockB == 1 ? 0 : 7;
   p.M = (uint32_t)M; p.N = (uint32_t)N; p.K = (uint32_t)K; p.alpha = alpha; p.beta = beta; p.dtypeC = dtypeC;
   const bool e5a = dtypeA == OCH_FLOAT8_E5M2, e5b = dtypeB == OCH_FLOAT8_E5M2;
   hipStream_t s = as_stream(stream);
   return e5a ? (e5b ? gemm_f8_dispatch<true, true>(p, akc, bkc, s) : gemm_f8_dispatch<true, false>(p, akc, bkc, s))
              : (e5b ? gemm_f8_dispatch<false, true>(p, akc, bkc, s) : gemm_f8_dispatch<false, false>(p, akc, bkc, s));
}
