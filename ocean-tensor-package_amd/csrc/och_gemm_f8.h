/* Block-scaled products of 8-bit floats, C <- alpha * sum over blocks of 128 k of (scale of A) (scale of B) (A B over
 * the block) + beta * C, column-major: what the kernels share. */
#pragma once
#include "och_gemm.h"
#include "och_float8.h"
#include "och_gemm_f8_slab.h"

namespace och {

typedef int   och_i32x8 __attribute__((ext_vector_type(8)));
typedef int   och_f8i32x4 __attribute__((ext_vector_type(4)));
typedef int   och_f8i32x2 __attribute__((ext_vector_type(2)));
typedef float och_f32x4v __attribute__((ext_vector_type(4)));

struct F8GemmParams
{
   const uint8_t *A, *B; char *C; const float *SA, *SB;
   int64_t  ldA, ldB, ldC;              /* in elements */
   int64_t  sa_m, sa_k, sb_n, sb_k;     /* elements of SA / SB from one scale to the next along op(A)'s rows / op(B)'s columns and along the blocks of k */
   uint32_t shiftA, shiftB;             /* rows of op(A) / columns of op(B) per scale: 1 << shift */
   uint32_t M, N, K;
   float    alpha, beta;
   int      dtypeC;
   uint32_t tiles_m, tiles_n;
   /* few tiles and a long K: workgroup (x, y) computes share y of tile x, share_slabs blocks of 128 k, and leaves its sums
      in plane y of `partial`; a second kernel adds the planes in order. 0: every tile has the whole K */
   uint32_t share_slabs;
   float   *partial;
};
/* rows of a plane of partial sums: whole groups of four */
__host__ __device__ static inline uint32_t f8_plane_pitch(uint32_t M) { return (M + 3) & ~3u; }
int gemm_f8_tile_44(const F8GemmParams &p, bool akc, bool bkc, bool pair, dim3 grid, hipStream_t stream);
int gemm_f8_tile_45(const F8GemmParams &p, bool akc, bool bkc, bool pair, dim3 grid, hipStream_t stream);
int gemm_f8_tile_54(const F8GemmParams &p, bool akc, bool bkc, bool pair, dim3 grid, hipStream_t stream);
int gemm_f8_tile_55(const F8GemmParams &p, bool akc, bool bkc, bool pair, dim3 grid, hipStream_t stream);
int gemm_f8_pipe_44(const F8GemmParams &p, bool akc, bool bkc, hipStream_t stream);
int gemm_f8_pipe_45(const F8GemmParams &p, bool akc, bool bkc, hipStream_t stream);
int gemm_f8_pipe_54(const F8GemmParams &p, bool akc, bool bkc, hipStream_t stream);
int gemm_f8_pipe_55(const F8GemmParams &p, bool akc, bool bkc, hipStream_t stream);
int gemm_f8_few_44(const F8GemmParams &p, hipStream_t stream);
int gemm_f8_few_45(const F8GemmParams &p, hipStream_t stream);
int gemm_f8_few_54(const F8GemmParams &p, hipStream_t stream);
int gemm_f8_few_55(const F8GemmParams &p, hipStream_t stream);

typedef __bf16 och_bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 och_bf16x8 __attribute__((ext_vector_type(8)));

/* The sums of 16 x 16 products over a block of 128 k, in one of two ways.
 *
 * v_mfma_f32_16x16x128_f8f6f4 takes the codes as they are, 32 cycles for the block. Of every eight products that it adds
 * at once (the eight k that lie together in a register pair) it keeps the bits down to 2^-13 of the largest one's leading
 * bit and cuts the others off (measured: with 2^16 and -2^16 among the eight, 2^3 survives and 2^2 does not; across the
 * eights, and in the older fp8 instructions alike, 24 bits do). On Gaussian operands that is about 1e-4 of the result's
 * norm: half a rounding to half, a twentieth of one to bfloat16.
 * WIDE: the codes become bfloat16, which holds them exactly, and four v_mfma_f32_16x16x32_bf16 of 16 cycles add their
 * exact products with 24 bits: sums as good as float ones, at half the matrix rate, for results that are float and wherever
 * memory bounds the product anyway (the kernel of few columns, up to 32 of them). */
template <bool WIDE> struct F8Operand;
template <> struct F8Operand<false>
{  och_i32x8 v;
   template <bool E5> __device__ __forceinline__ void set(och_i32x8 codes) { v = codes; }
};
template <> struct F8Operand<true>
{  och_bf16x8 v[4];
   template <bool E5> __device__ __forceinline__ void set(och_i32x8 codes)
   {
#pragma unroll
      for (int q = 0; q < 4; q++)
      {  och_bf16x2 t[4];
#pragma unroll
         for (int h = 0; h < 2; h++)
         {  const unsigned c = (unsigned)codes[2 * q + h];
            t[2 * h]     = E5 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(c, 1.0f, false) : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, 1.0f, false);
            t[2 * h + 1] = E5 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(c, 1.0f, true)  : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, 1.0f, true);
         }
         v[q] = __builtin_shufflevector(__builtin_shufflevector(t[0], t[1], 0, 1, 2, 3), __builtin_shufflevector(t[2], t[3], 0, 1, 2, 3), 0, 1, 2, 3, 4, 5, 6, 7);
      }
   }
};
template <bool E5A, bool E5B> __device__ __forceinline__ och_f32x4v f8_block(const F8Operand<false> &a, const F8Operand<false> &b)
{  const och_f32x4v zero = { 0, 0, 0, 0 };
   return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a.v, b.v, zero, E5A ? 1 : 0, E5B ? 1 : 0, 0, 0, 0, 0);
}
template <bool E5A, bool E5B> __device__ __forceinline__ och_f32x4v f8_block(const F8Operand<true> &a, const F8Operand<true> &b)
{  och_f32x4v c = { 0, 0, 0, 0 };
#pragma unroll
   for (int q = 0; q < 4; q++) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v[q], b.v[q], c, 0, 0, 0);
   return c;
}
/* a row of TJ blocks; the wide instructions of two blocks alternate, because each needs the sums of the one before */
template <bool E5A, bool E5B, int TJ> __device__ __forceinline__ void f8_row(const F8Operand<false> &a, const F8Operand<false> (&b)[TJ], och_f32x4v (&part)[TJ])
{
#pragma unroll
   for (int j = 0; j < TJ; j++) part[j] = f8_block<E5A, E5B>(a, b[j]);
}
template <bool E5A, bool E5B, int TJ> __device__ __forceinline__ void f8_row(const F8Operand<true> &a, const F8Operand<true> (&b)[TJ], och_f32x4v (&part)[TJ])
{  const och_f32x4v zero = { 0, 0, 0, 0 };
   static_assert(TJ % 2 == 0, "pairs of blocks");
#pragma unroll
   for (int x = 0; x < 4 * TJ; x++)
   {  const int j = x / 8 * 2 + x % 2, q = x / 2 % 4;
      part[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v[q], b[j].v[q], q == 0 ? zero : part[j], 0, 0, 0);
   }
}

/* the fragment of rows row0 .. + 15 (row0 a multiple of 16) of a slab in LDS */
template <bool KC, int R> __device__ __forceinline__ och_i32x8 f8_fragment(const char *slab, uint32_t row0)
{
   typedef F8Slab<KC, R> L;
   const uint32_t lane = threadIdx.x & 63, g = lane / 16;
   och_i32x8 f;
   if (KC)
   {  const uint32_t row = row0 + lane % 16;
      const och_f8i32x4 lo = *reinterpret_cast<const och_f8i32x4 *>(slab + L::at_row(row, g));
      const och_f8i32x4 hi = *reinterpret_cast<const och_f8i32x4 *>(slab + L::at_row(row, 4 + g));
      f = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
   }
   else
   {  och_f8i32x2 t[4];
#pragma unroll
      for (int i = 0; i < 4; i++)
         t[i] = __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) och_f8i32x2 *)(slab + L::at_k(row0, 16 * g + 64 * (i / 2) + 8 * (i % 2), lane)));
      f = __builtin_shufflevector(__builtin_shufflevector(t[0], t[1], 0, 1, 2, 3), __builtin_shufflevector(t[2], t[3], 0, 1, 2, 3), 0, 1, 2, 3, 4, 5, 6, 7);
   }
   return f;
}

/* one float per lane from memory to LDS, as load_to_lds moves sixteen bytes */
static __device__ __forceinline__ void load_float_to_lds(const char *base, uint32_t offset, uint32_t target)
{
   asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" : : "s"(target), "v"(offset), "s"(base) : "memory");
}

/* one element of C: s is the finished sum */
template <int DT> __device__ __forceinline__ void f8_finish(char *C, int64_t at, float s, float alpha, float beta)
{  typedef typename Wide<DT>::E E;
   E *c = reinterpret_cast<E *>(C) + at;
   float v = alpha * s;
   if (beta != 0.0f) v = __builtin_fmaf(beta, Wide<DT>::get(*c), v);
   *c = Wide<DT>::put(v);
}

} /* namespace och */
