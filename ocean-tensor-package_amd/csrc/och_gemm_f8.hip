/* och_gemm_scaled: products of 8-bit floats with one scale per block of 128 k (and per row or per 128 rows) of either
 * operand. No counterpart in the reference.
 *
 * The matrix cores multiply a whole block of 128 k (one v_mfma_f32_16x16x128_f8f6f4, or four bfloat16 ones where the
 * result is float or has up to 32 columns); the 16 x 16 sums of a block are multiplied by the two scales and added to the float accumulators
 * outside them, four multiply-adds per lane beside 32 or 64 cycles of matrix work.
 *
 * The two scales are multiplied with each other first, which is once per column and block where a scale of A covers 128
 * rows; either one times the sums would be once more per element. So their product has to lie within float's range, and
 * callers are told so; sums times a single scale would leave the range for other pairs (1e35 times a sum of 1e7).
 */
#include "och_gemm_f8_tile.h"
#include <math.h>

namespace och {

/* adds the shares of K in order and finishes the elements: four rows of a column per thread, eight planes' loads under way
   together */
template <int DT> __global__ __launch_bounds__(256) void gemm_f8_join_kernel(const F8GemmParams p, uint32_t shares)
{
   const uint32_t pitch = f8_plane_pitch(p.M);
   const uint64_t q = (uint64_t)blockIdx.x * 256 + threadIdx.x, plane = (uint64_t)pitch * p.N;
   const uint32_t n = (uint32_t)(q / (pitch / 4)), m = (uint32_t)(q % (pitch / 4)) * 4;
   if (n >= p.N) return;
   och_f32x4v s = { 0, 0, 0, 0 };
   for (uint32_t t = 0; t < shares; t += 8)
   {  och_f32x4v v[8];
#pragma unroll
      for (uint32_t u = 0; u < 8; u++) v[u] = *reinterpret_cast<const och_f32x4v *>(p.partial + (t + u < shares ? t + u : shares - 1) * plane + 4 * q);
#pragma unroll
      for (int u = 0; u < 8; u++) asm volatile("" : "+v"(v[u]));      /* all eight, before the first is waited for */
#pragma unroll
      for (uint32_t u = 0; u < 8; u++) if (t + u < shares) s += v[u];
   }
   f8_finish4<DT>(p.C, (int64_t)m + (int64_t)n * p.ldC, s, p.alpha, p.beta, p.M - m);
}

/* Shares of K for a product of few tiles: what takes the least time by these figures, in microseconds. A block of 128 k
   takes a tile 1.0 (float results: 1.5; operands that cannot be pipelined: 3.4), half as much again where two workgroups share
   a compute unit; the second kernel 4, and a plane 0.05 and its bytes written and read at 5 TB/s. To bfloat16, 1024 x 1024 x
   4096: one share 37.6 us, four 21.3, eight 24.5; 2048 x 1024 x 1024: one share 13.7, two 21.0; 524 x 121 x 10112: twelve shares
   16.0, twenty 14.4, forty 16.8. Pairs of groups on a tile work like two workgroups on a unit and need no plane of their own.
   Blocks per share at the least of blocks * slab + blocks of K / blocks * plane, and the numbers of shares that fill every unit
   once and twice, are compared with one. */
static uint64_t gemm_f8_shares(uint64_t tiles, uint64_t slabs, uint64_t plane_bytes, uint64_t units, bool wide, bool piped, bool *pair)
{
   uint64_t best = 1, most = 2 * units / tiles;
   const uint64_t fit = OCH_GEMM_WORKSPACE / plane_bytes;
   if (most > slabs) most = slabs;
   if (most > fit) most = fit;
   const double slab = !piped ? 3.4 : wide ? 1.5 : 1.0, plane = 0.05 + (double)plane_bytes * 2 / 5e6;
   const uint64_t blocks = 1 + (uint64_t)sqrt((double)slabs * plane / slab);
   const uint64_t tries[6] = { 1, (slabs + blocks - 1) / blocks, blocks > 1 ? (slabs + blocks - 2) / (blocks - 1) : most, (slabs + 2 * blocks - 1) / (2 * blocks), units / tiles, most };
   double least = INFINITY;
   *pair = false;
   for (int i = 0; i < 6; i++)
   {  uint64_t s = tries[i] < most ? tries[i] : most;
      if (s < 1) s = 1;
      const uint64_t own = (slabs + s - 1) / s;
      const double join = s > 1 ? 4.0 + (double)s * plane : 0;
      const double single = (double)own * slab * (tiles * s > units ? 1.5 : 1.0) + join, twin = (double)((own + 1) / 2) * slab * 1.5 + 0.5 + join;
      if (single < least) { least = single; best = s; *pair = false; }
      if (piped && own > 1 && tiles * s <= units && twin < least) { least = twin; best = s; *pair = true; }
   }
   return best;
}

/* A product on 128 x 128 tiles, K cut into shares where that is quicker */
static int gemm_f8_tiles(F8GemmParams p, bool e5a, bool e5b, bool akc, bool bkc, hipStream_t stream)
{
   p.tiles_m = (p.M + OCH_F8_TILE - 1) / OCH_F8_TILE; p.tiles_n = (p.N + OCH_F8_TILE - 1) / OCH_F8_TILE;
   const uint64_t tiles = (uint64_t)p.tiles_m * p.tiles_n, slabs = ((uint64_t)p.K + OCH_F8_SLAB - 1) / OCH_F8_SLAB, units = (uint64_t)gemm_compute_units();
   if (tiles > most_groups(OCH_F8_TILE_THREADS)) return set_error("gemm_scaled: a result of %u x %u has too many tiles", p.M, p.N);
   const bool piped = (akc || p.M >= 16) && (bkc || p.N >= 16) && p.ldA < (1 << 24) && p.ldB < (1 << 24);
   bool pair;
   uint64_t shares = gemm_f8_shares(tiles, slabs, (uint64_t)f8_plane_pitch(p.M) * p.N * sizeof(float), units, p.dtypeC == OCH_FLOAT, piped, &pair);
   if (shares >= 2)
   {  char *ws;
      if (stream_gemm_workspace(stream, &ws) != 0) return -1;
      p.partial = reinterpret_cast<float *>(ws);
      p.share_slabs = (uint32_t)((slabs + shares - 1) / shares);
      shares = (slabs + p.share_slabs - 1) / p.share_slabs;
   }
   else shares = 1;
   const dim3 grid((unsigned)tiles, (unsigned)shares);
   const int status = e5a ? (e5b ? gemm_f8_tile_55(p, akc, bkc, pair, grid, stream) : gemm_f8_tile_54(p, akc, bkc, pair, grid, stream))
                          : (e5b ? gemm_f8_tile_45(p, akc, bkc, pair, grid, stream) : gemm_f8_tile_44(p, akc, bkc, pair, grid, stream));
   if (status != 0 || p.share_slabs == 0) return status;
   const dim3 join((unsigned)(((uint64_t)f8_plane_pitch(p.M) / 4 * p.N + 255) / 256));
   if (p.dtypeC == OCH_FLOAT)     hipLaunchKernelGGL(gemm_f8_join_kernel<OCH_FLOAT>, join, dim3(256), 0, stream, p, (uint32_t)shares);
   else if (p.dtypeC == OCH_HALF) hipLaunchKernelGGL(gemm_f8_join_kernel<OCH_HALF>, join, dim3(256), 0, stream, p, (uint32_t)shares);
   else                           hipLaunchKernelGGL(gemm_f8_join_kernel<OCH_BFLOAT16>, join, dim3(256), 0, stream, p, (uint32_t)shares);
   OCH_CHECK_LAUNCH();
   return 0;
}

/* Whether a product of aligned operands is quicker on 256 x 256 tiles (one workgroup per compute unit) than on 128 x 128
   (two): rounds of the compute units times the work of a round over its rate. Measured rates on full rounds of aligned
   operands: 2.3 and 1.5 PFLOP/s. */
static bool gemm_f8_large(size_t M, size_t N)
{
   const double units = gemm_compute_units(), small = (double)((M + 127) / 128) * (double)((N + 127) / 128), large = (double)((M + 255) / 256) * (double)((N + 255) / 256);
   return ceil(large / units) * 4 / 2.3 < ceil(small / (2 * units)) * 2 / 1.5;
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
   /* few columns on their own kernel, which loads 16 bytes at a time and counts bytes within its rows in 32 bits */
   const bool aligned = (((uintptr_t)A | (uintptr_t)B | (uintptr_t)ldA | (uintptr_t)ldB) & 15) == 0, near = ldA < (1 << 25) && ldB < (1 << 25) && ldSA < (1 << 24) && ldSB < (1 << 24);
   if (N <= 64 && akc && bkc && aligned && near)
      return e5a ? (e5b ? gemm_f8_few_55(p, s) : gemm_f8_few_54(p, s)) : (e5b ? gemm_f8_few_45(p, s) : gemm_f8_few_44(p, s));
   /* float results need the wide sums, and chunks of 16 rows must not pass the end of an operand that is contiguous along them */
   if (dtypeC != OCH_FLOAT && aligned && ldA < (1 << 24) && ldB < (1 << 24) && ldSA < (1 << 22) && ldSB < (1 << 22) && (akc || M % 16 == 0) && (bkc || N % 16 == 0) && gemm_f8_large(M, N))
   {  p.tiles_m = (p.M + 255) / 256; p.tiles_n = (p.N + 255) / 256;
      if ((uint64_t)p.tiles_m * p.tiles_n > most_groups(512)) return set_error("gemm_scaled: a result of %u x %u has too many tiles", p.M, p.N);
      return e5a ? (e5b ? gemm_f8_pipe_55(p, akc, bkc, s) : gemm_f8_pipe_54(p, akc, bkc, s)) : (e5b ? gemm_f8_pipe_45(p, akc, bkc, s) : gemm_f8_pipe_44(p, akc, bkc, s));
   }
   return gemm_f8_tiles(p, e5a, e5b, akc, bkc, s);
}
