/* och_quantize_blocks: a matrix to 8-bit float codes with one float scale per block of 128 x 1, 1 x 128 or 128 x 128.
 * No counterpart in the reference, which has no 8-bit floats.
 *
 *    a = max(max |x| over the block, 2^-100),  scale = a / c,  code = round(clamp(x * (c / a), -c, c)),  c the largest code
 *
 * One pass over the data: a block's values stay in registers between the maximum and the conversion, so the traffic is
 * the matrix once in and the codes and scales once out; that is what bounds it.
 */
#include "och_float8.h"

namespace och {

struct QuantizeParams
{
   const char *X; uint8_t *Q; float *S;
   int64_t  ldX, ldQ, ldS;              /* in elements */
   int64_t  M, N;
   uint32_t bm;                         /* blocks along M: ceil(M / 128) */
   uint64_t blocks;
};

/* Blocks of 128 x 1: sixteen lanes own a block, eight elements each; a workgroup of 256 handles sixteen blocks at a time */
template <int DT, int CODE>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const QuantizeParams p)
{
   typedef typename Wide<DT>::E E;
   const uint64_t b = (uint64_t)blockIdx.x * 16 + threadIdx.x / 16;
   const bool live = b < p.blocks;
   const int64_t j = live ? (int64_t)(b / p.bm) : 0;
   const uint32_t kb = live ? (uint32_t)(b - (uint64_t)j * p.bm) : 0;
   const int64_t i = (int64_t)kb * OCH_F8_BLOCK + (threadIdx.x % 16) * 8, valid = live ? p.M - i : 0;
   Wide8<DT> v;
   v.load(reinterpret_cast<const E *>(p.X) + i + j * p.ldX, valid);
   uint32_t m = 0;
#pragma unroll
   for (int e = 0; e < 8; e++) m = umax(m, magnitude_bits(v.get(e)));
   float scale, factor; bool bad;
   block_scale<CODE>(row16_max(m), scale, factor, bad);
   och_u32x2 q;
   q.x = code4<CODE>(v.get(0), v.get(1), v.get(2), v.get(3), factor, bad);
   q.y = code4<CODE>(v.get(4), v.get(5), v.get(6), v.get(7), factor, bad);
   store_codes(p.Q + i + j * p.ldQ, q, valid);
   if (live && threadIdx.x % 16 == 0) p.S[kb + j * p.ldS] = scale;
}

/* Blocks of 1 x 128 and 128 x 128 (WHOLE): a workgroup of 256 owns 128 x 128 elements; thread t holds rows
   8 (t % 16) .. + 7 of columns t / 16 + 16 c, c = 0 .. 7. Maxima over the columns meet in LDS. */
template <int DT, int CODE, bool WHOLE>
__global__ __launch_bounds__(256) void quantize_tile_kernel(const QuantizeParams p)
{
   typedef typename Wide<DT>::E E;
   __shared__ uint32_t part[16][OCH_F8_BLOCK];
   const uint32_t kb = blockIdx.x % p.bm;
   const int64_t nb = blockIdx.x / p.bm;
   const int ti = threadIdx.x % 16, tj = threadIdx.x / 16;
   const int64_t i = (int64_t)kb * OCH_F8_BLOCK + ti * 8, j0 = nb * OCH_F8_BLOCK + tj, valid = p.M - i;
   Wide8<DT> v[8];
   uint32_t m[8] = { 0, 0, 0, 0, 0, 0, 0, 0 };
#pragma unroll
   for (int c = 0; c < 8; c++)
      v[c].load(reinterpret_cast<const E *>(p.X) + i + (j0 + 16 * c) * p.ldX, j0 + 16 * c < p.N ? valid : 0);
#pragma unroll
   for (int c = 0; c < 8; c++)
#pragma unroll
      for (int e = 0; e < 8; e++) m[e] = umax(m[e], magnitude_bits(v[c].get(e)));
#pragma unroll
   for (int e = 0; e < 8; e++) part[tj][ti * 8 + e] = m[e];
   __syncthreads();
#pragma unroll
   for (int e = 0; e < 8; e++)
   {  m[e] = part[0][ti * 8 + e];
#pragma unroll
      for (int t = 1; t < 16; t++) m[e] = umax(m[e], part[t][ti * 8 + e]);
   }
   if (WHOLE)
   {  uint32_t all = m[0];
#pragma unroll
      for (int e = 1; e < 8; e++) all = umax(all, m[e]);
      all = row16_max(all);
#pragma unroll
      for (int e = 0; e < 8; e++) m[e] = all;
   }
   float scale[8], factor[8]; bool bad[8];
#pragma unroll
   for (int e = 0; e < 8; e++) block_scale<CODE>(m[e], scale[e], factor[e], bad[e]);
#pragma unroll
   for (int c = 0; c < 8; c++)
   {  uint8_t q[8];
#pragma unroll
      for (int e = 0; e < 8; e++) q[e] = (uint8_t)code4<CODE>(v[c].get(e), 0, 0, 0, factor[e], bad[e]);
      och_u32x2 w;
      w.x = q[0] | q[1] << 8 | q[2] << 16 | (uint32_t)q[3] << 24; w.y = q[4] | q[5] << 8 | q[6] << 16 | (uint32_t)q[7] << 24;
      store_codes(p.Q + i + (j0 + 16 * c) * p.ldQ, w, j0 + 16 * c < p.N ? valid : 0);
   }
   if (WHOLE) { if (threadIdx.x == 0) p.S[kb + nb * p.ldS] = scale[0]; }
   else if (tj == 0)
   {
#pragma unroll
      for (int e = 0; e < 8; e++) if (e < valid) p.S[i + e + nb * p.ldS] = scale[e];
   }
}

template <int DT, int CODE>
static int quantize_launch(const QuantizeParams &p, bool rows, bool whole, hipStream_t stream)
{
   const uint64_t groups = rows ? (p.blocks + 15) / 16 : (uint64_t)p.bm * ((p.N + OCH_F8_BLOCK - 1) / OCH_F8_BLOCK);
   if (groups > 0x7FFFFFFFull) return set_error("quantize_blocks: the matrix has too many blocks");
   const dim3 grid((unsigned)groups);
   if (rows)       hipLaunchKernelGGL((quantize_rows_kernel<DT, CODE>), grid, dim3(256), 0, stream, p);
   else if (whole) hipLaunchKernelGGL((quantize_tile_kernel<DT, CODE, true>), grid, dim3(256), 0, stream, p);
   else            hipLaunchKernelGGL((quantize_tile_kernel<DT, CODE, false>), grid, dim3(256), 0, stream, p);
   OCH_CHECK_LAUNCH();
   return 0;
}

} /* namespace och */

using namespace och;

extern "C" int och_quantize_blocks(int dtype, int code, size_t M, size_t N, const void *X, ptrdiff_t ldX, size_t block_m, size_t block_n,
                                   void *Q, ptrdiff_t ldQ, float *S, ptrdiff_t ldS, och_stream stream)
{
   if (!wide_type(dtype)) return set_error("quantize_blocks is available for half, bfloat16 and float (got %d)", dtype);
   if (!code_type(code)) return set_error("quantize_blocks: the codes are float8_e4m3 or float8_e5m2 (got %d)", code);
   const bool rows = block_m == OCH_F8_BLOCK && block_n == 1, whole = block_m == OCH_F8_BLOCK && block_n == OCH_F8_BLOCK;
   if (!rows && !whole && !(block_m == 1 && block_n == OCH_F8_BLOCK))
      return set_error("quantize_blocks: blocks are 128 x 1, 1 x 128 or 128 x 128 (got %zu x %zu)", block_m, block_n);
   if (M == 0 || N == 0) return 0;
   if (M > 0x7FFFFFFFull || N > 0x7FFFFFFFull) return set_error("quantize_blocks: a side of %zu elements is too long", M > N ? M : N);
   if (X == nullptr || Q == nullptr || S == nullptr) return set_error("quantize_blocks: null pointer argument");
   const size_t sm = (M + block_m - 1) / block_m;
   if (ldX < (ptrdiff_t)M || ldQ < (ptrdiff_t)M || ldS < (ptrdiff_t)sm)
      return set_error("quantize_blocks: a leading dimension (%td, %td, %td) is smaller than its matrix (%zu, %zu, %zu)", ldX, ldQ, ldS, M, M, sm);
   if ((uintptr_t)X % wide_size(dtype) != 0 || (uintptr_t)S % 4 != 0) return set_error("quantize_blocks: misaligned pointer");
   QuantizeParams p;
   p.X = (const char *)X; p.Q = (uint8_t *)Q; p.S = S; p.ldX = ldX; p.ldQ = ldQ; p.ldS = ldS; p.M = (int64_t)M; p.N = (int64_t)N;
   p.bm = (uint32_t)((M + OCH_F8_BLOCK - 1) / OCH_F8_BLOCK); p.blocks = (uint64_t)p.bm * N;
#define OCH_GO(DT) (code == OCH_FLOAT8_E4M3 ? quantize_launch<DT, OCH_FLOAT8_E4M3>(p, rows, whole, as_stream(stream)) \
                                            : quantize_launch<DT, OCH_FLOAT8_E5M2>(p, rows, whole, as_stream(stream)))
   return OCH_BY_WIDE(dtype, OCH_GO);
#undef OCH_GO
}
