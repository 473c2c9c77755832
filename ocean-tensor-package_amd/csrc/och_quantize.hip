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
   uint64_t blocks, first;              /* blocks of 128 x 1; workgroup 0's place in the whole */
};

/* Blocks of 128 x 1: sixteen lanes own a block, eight elements each, and take OCH_QUANTIZE_VECTORS blocks, sixteen apart,
   whose loads are under way together. 8192 x 8192 bfloat16 values to codes: 33.3 us (6.1 TB/s of reads and writes);
   through the caches 36.8 with two blocks, 38.5 with one, 37.1 with four. */
#define OCH_QUANTIZE_VECTORS 2
template <int DT, int CODE, bool NT>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const QuantizeParams p)
{
   constexpr int V = OCH_QUANTIZE_VECTORS;
   typedef typename Wide<DT>::E E;
   Wide8<DT> x[V];
   int64_t i[V], j[V], valid[V];
   uint32_t kb[V];
#pragma unroll
   for (int v = 0; v < V; v++)
   {  const uint64_t b = ((p.first + blockIdx.x) * V + v) * 16 + threadIdx.x / 16;
      const bool live = b < p.blocks;
      if (p.blocks >> 32 == 0) j[v] = (uint32_t)b / p.bm;
      else                     j[v] = (int64_t)(b / p.bm);
      kb[v] = (uint32_t)(b - (uint64_t)j[v] * p.bm);
      if (!live) { j[v] = 0; kb[v] = 0; }
      i[v] = (int64_t)kb[v] * OCH_F8_BLOCK + (threadIdx.x % 16) * 8;
      valid[v] = live ? p.M - i[v] : INT64_MIN;
      x[v].template load<NT>(reinterpret_cast<const E *>(p.X) + i[v] + j[v] * p.ldX, valid[v]);
   }
#pragma unroll
   for (int v = 0; v < V; v++)
   {  uint32_t m = 0;
#pragma unroll
      for (int w = 0; w < Wide8<DT>::WORDS * 4; w++) m = word_max<DT>(m, word_magnitude<DT>(x[v].raw[w / 4][w % 4]));
      if (DT != OCH_FLOAT) m = umax(word_float_bits<DT>(m, 0), word_float_bits<DT>(m, 1));
      float scale, factor; bool bad;
      block_scale<CODE>(row16_max(m), scale, factor, bad);
      och_u32x2 q;
      q.x = code4<CODE>(x[v].get(0), x[v].get(1), x[v].get(2), x[v].get(3), factor, bad);
      q.y = code4<CODE>(x[v].get(4), x[v].get(5), x[v].get(6), x[v].get(7), factor, bad);
      store_codes<NT>(p.Q + i[v] + j[v] * p.ldQ, q, valid[v]);
      if (valid[v] > 0 && threadIdx.x % 16 == 0) p.S[kb[v] + j[v] * p.ldS] = scale;
   }
}

/* Blocks of 1 x 128 and 128 x 128 (WHOLE): a workgroup of 256 owns 128 x 128 elements; thread t holds rows
   8 (t % 16) .. + 7 of columns t / 16 + 16 c, c = 0 .. 7. The maxima over the columns are taken in registers first, then
   over the four groups of lanes of the wave, and then the four waves' meet in LDS.
   8192 x 4096 floats in 128 x 128 blocks: 29.6 us (5.7 TB/s), 31.6 where all sixteen threads of a column meet in LDS.
   Halfs in 1 x 128 blocks: 5120 x 4096, columns of whole cache lines, 11.4 us (5.6 TB/s); 5003 x 4001 17.3 us (3.5 TB/s), with 64
   rows to a workgroup 20.2: neighbouring tiles share lines and run on different dies, so that 39 % more is read and 21 % more
   written than the matrix holds. */
template <int DT, int CODE, bool WHOLE, bool NT>
__global__ __launch_bounds__(256) void quantize_tile_kernel(const QuantizeParams p)
{
   typedef typename Wide<DT>::E E;
   constexpr int WORDS = Wide8<DT>::WORDS * 4, PER = 8 / WORDS;    /* of a thread; elements in a word */
   __shared__ och_u32x4 part[4][16][WORDS / 4];
   const uint32_t tile = (uint32_t)p.first + blockIdx.x, kb = tile % p.bm;
   const int64_t nb = tile / p.bm;
   const int ti = threadIdx.x % 16, tj = threadIdx.x / 16;
   const int64_t i = (int64_t)kb * OCH_F8_BLOCK + ti * 8, j0 = nb * OCH_F8_BLOCK + tj, valid = p.M - i;
   Wide8<DT> v[8];
   uint32_t m[WORDS];
#pragma unroll
   for (int c = 0; c < 8; c++)
      v[c].template load<NT>(reinterpret_cast<const E *>(p.X) + i + (j0 + 16 * c) * p.ldX, j0 + 16 * c < p.N ? valid : 0);
#pragma unroll
   for (int w = 0; w < WORDS; w++)
   {  m[w] = 0;
#pragma unroll
      for (int c = 0; c < 8; c++) m[w] = word_max<DT>(m[w], word_magnitude<DT>(v[c].raw[w / 4][w % 4]));
   }
   if (WHOLE)
   {
#pragma unroll
      for (int w = 1; w < WORDS; w++) m[0] = word_max<DT>(m[0], m[w]);
      if (PER == 2) m[0] = umax(m[0] & 0xFFFFu, m[0] >> 16);
      m[0] = row16_max(m[0]);
   }
#pragma unroll
   for (int w = 0; w < (WHOLE ? 1 : WORDS); w++)
   {  m[w] = word_max<DT>(m[w], (uint32_t)__shfl_xor((int)m[w], 16));
      m[w] = word_max<DT>(m[w], (uint32_t)__shfl_xor((int)m[w], 32));
   }
   if (threadIdx.x % 64 < 16)
   {
#pragma unroll
      for (int w = 0; w < (WHOLE ? 1 : WORDS); w++) part[tj / 4][ti][w / 4][w % 4] = m[w];
   }
   __syncthreads();
#pragma unroll
   for (int g = 0; g < 4; g++)
#pragma unroll
      for (int w = 0; w < (WHOLE ? 1 : WORDS); w++) m[w] = word_max<DT>(m[w], part[g][ti][w / 4][w % 4]);
   float scale[8], factor[8]; bool bad[8];
#pragma unroll
   for (int e = 0; e < 8; e++) block_scale<CODE>(WHOLE ? word_float_bits<DT>(m[0], 0) : word_float_bits<DT>(m[e / PER], e % PER), scale[e], factor[e], bad[e]);
   uint32_t keep[2] = { 0, 0 };                       /* 0xFF in the bytes of good blocks */
#pragma unroll
   for (int e = 0; e < 8; e++) keep[e / 4] |= bad[e] ? 0u : 0xFFu << 8 * (e % 4);
#pragma unroll
   for (int c = 0; c < 8; c++)
   {  och_u32x2 q;
      q.x = code4<CODE>(v[c].get(0) * factor[0], v[c].get(1) * factor[1], v[c].get(2) * factor[2], v[c].get(3) * factor[3]);
      q.y = code4<CODE>(v[c].get(4) * factor[4], v[c].get(5) * factor[5], v[c].get(6) * factor[6], v[c].get(7) * factor[7]);
      q.x = (q.x & keep[0]) | (0x7F7F7F7Fu & ~keep[0]); q.y = (q.y & keep[1]) | (0x7F7F7F7Fu & ~keep[1]);
      store_codes<NT>(p.Q + i + (j0 + 16 * c) * p.ldQ, q, j0 + 16 * c < p.N ? valid : 0);
   }
   if (WHOLE) { if (threadIdx.x == 0) p.S[kb + nb * p.ldS] = scale[0]; }
   else if (tj == 0)
   {
#pragma unroll
      for (int e = 0; e < 8; e++) if (e < valid) p.S[i + e + nb * p.ldS] = scale[e];
   }
}

template <int DT, int CODE, bool NT>
static int quantize_launch(QuantizeParams p, bool rows, bool whole, hipStream_t stream)
{
   const uint64_t groups = rows ? (p.blocks + 16 * OCH_QUANTIZE_VECTORS - 1) / (16 * OCH_QUANTIZE_VECTORS) : (uint64_t)p.bm * ((p.N + OCH_F8_BLOCK - 1) / OCH_F8_BLOCK);
   if (!rows && groups > 0xFFFFFFFFull) return set_error("quantize_blocks: the matrix has too many blocks");
   for (p.first = 0; p.first < groups; p.first += most_groups(256))
   {  const uint64_t left = groups - p.first;
      const dim3 grid((unsigned)(left < most_groups(256) ? left : most_groups(256)));
      if (rows)       hipLaunchKernelGGL((quantize_rows_kernel<DT, CODE, NT>), grid, dim3(256), 0, stream, p);
      else if (whole) hipLaunchKernelGGL((quantize_tile_kernel<DT, CODE, true, NT>), grid, dim3(256), 0, stream, p);
      else            hipLaunchKernelGGL((quantize_tile_kernel<DT, CODE, false, NT>), grid, dim3(256), 0, stream, p);
      OCH_CHECK_LAUNCH();
   }
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
   /* 8192 x 8192 bfloat16 values in blocks of 128 x 1: 33.3 us past the caches, 36.7 through them; 5003 x 4001 halfs, whose
      columns do not begin on whole lines, 22.5 against 17.2 */
   const size_t es = wide_size(dtype);
   const bool nt = streams(X, ldX * es, (uint64_t)M * N * es) && streams(Q, ldQ, (uint64_t)M * N);
#define OCH_GO_CODE(DT, CODE) (nt ? quantize_launch<DT, CODE, true>(p, rows, whole, as_stream(stream)) : quantize_launch<DT, CODE, false>(p, rows, whole, as_stream(stream)))
#define OCH_GO(DT) (code == OCH_FLOAT8_E4M3 ? OCH_GO_CODE(DT, OCH_FLOAT8_E4M3) : OCH_GO_CODE(DT, OCH_FLOAT8_E5M2))
   return OCH_BY_WIDE(dtype, OCH_GO);
#undef OCH_GO
#undef OCH_GO_CODE
}
