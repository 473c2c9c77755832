/* What the block-scaled 8-bit float operations (och_quantize.hip, och_rms_norm.hip, och_gemm_f8*.hip) share: vectors of
 * eight elements of the wide types, the conversion to 8-bit codes, and the rule that makes a scale out of a block's
 * largest magnitude.
 *
 * half and bfloat16 are converted by the hardware here (round to nearest even, subnormal numbers kept), not by the
 * reference's half routines, which flush small values: the data comes from and goes to other programs' layers.
 *
 * A block's magnitudes are compared as bit patterns without the sign: for every IEEE type these order like the values,
 * with infinity above all finite values and NaN above infinity, so one unsigned maximum also finds both. */
#pragma once
#include "och_common.h"

namespace och {

#define OCH_F8_BLOCK 128

typedef unsigned int och_u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int och_u32x4 __attribute__((ext_vector_type(4)));
/* accesses aligned to the element only: the device runs with unaligned access enabled */
typedef och_u32x4 och_u32x4_any __attribute__((aligned(1)));
typedef och_u32x2 och_u32x2_any __attribute__((aligned(1)));

template <int DT> struct Wide;
template <> struct Wide<OCH_FLOAT>
{  typedef float E;
   static __device__ __forceinline__ float get(E x) { return x; }
   static __device__ __forceinline__ E put(float x) { return x; }
};
template <> struct Wide<OCH_HALF>
{  typedef _Float16 E;
   static __device__ __forceinline__ float get(E x) { return (float)x; }
   static __device__ __forceinline__ E put(float x) { return (E)x; }
};
template <> struct Wide<OCH_BFLOAT16>
{  typedef __bf16 E;
   static __device__ __forceinline__ float get(E x) { return (float)x; }
   static __device__ __forceinline__ E put(float x) { return (E)x; }
};

/* eight neighbouring elements; only the first `valid` of them exist (valid <= 0: none), the others read as zero and are
   not written */
template <int DT> struct Wide8
{
   typedef typename Wide<DT>::E E;
   static constexpr int WORDS = (int)sizeof(E) * 8 / 16;
   union { och_u32x4 raw[WORDS]; E e[8]; };
   /* NT: past the caches (see streams()) */
   template <bool NT = false> __device__ __forceinline__ void load(const E *at, int64_t valid)
   {  if (valid >= 8)
      {  const och_u32x4_any *from = reinterpret_cast<const och_u32x4_any *>(at);
#pragma unroll
         for (int w = 0; w < WORDS; w++) raw[w] = NT ? __builtin_nontemporal_load(from + w) : from[w];
      }
      else
      {
#pragma unroll
         for (int i = 0; i < 8; i++) e[i] = (i < valid) ? at[i] : (E)0.0f;
      }
   }
   template <bool NT = false> __device__ __forceinline__ void store(E *at, int64_t valid) const
   {  if (valid >= 8)
      {  och_u32x4_any *to = reinterpret_cast<och_u32x4_any *>(at);
#pragma unroll
         for (int w = 0; w < WORDS; w++)
         {  const och_u32x4_any x = raw[w];
            if (NT) __builtin_nontemporal_store(x, to + w); else to[w] = x;
         }
      }
      else
      {
#pragma unroll
         for (int i = 0; i < 8; i++) if (i < valid) at[i] = e[i];
      }
   }
   __device__ __forceinline__ float get(int i) const { return Wide<DT>::get(e[i]); }
   __device__ __forceinline__ void put(int i, float x) { e[i] = Wide<DT>::put(x); }
};

__device__ __forceinline__ uint32_t magnitude_bits(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }
__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }

/* largest value over the row of 16 lanes, in all of its lanes */
template <int CTRL> __device__ __forceinline__ uint32_t dpp_max(uint32_t x)
{  return umax(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xF, 0xF, true)); }
__device__ __forceinline__ uint32_t row16_max(uint32_t x)
{  x = dpp_max<0xB1>(x); x = dpp_max<0x4E>(x); x = dpp_max<0x141>(x); return dpp_max<0x140>(x); }

/* Largest magnitudes of elements as they lie in memory, word by word: one float or two 16-bit elements in a word, which are
   compared without being converted */
typedef unsigned short och_u16x2 __attribute__((ext_vector_type(2)));
template <int DT> __device__ __forceinline__ uint32_t word_magnitude(uint32_t w) { return w & (DT == OCH_FLOAT ? 0x7FFFFFFFu : 0x7FFF7FFFu); }
template <int DT> __device__ __forceinline__ uint32_t word_max(uint32_t a, uint32_t b)
{  if (DT == OCH_FLOAT) return umax(a, b);
   return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(och_u16x2, a), __builtin_bit_cast(och_u16x2, b)));
}
/* element i of the word, as the bits of a float */
template <int DT> __device__ __forceinline__ uint32_t word_float_bits(uint32_t w, int i)
{  if constexpr (DT == OCH_FLOAT) return w;
   else return __float_as_uint(Wide<DT>::get(__builtin_bit_cast(typename Wide<DT>::E, (unsigned short)(w >> 16 * i))));
}

template <int CODE> struct Code8 { static constexpr float MOST = (CODE == OCH_FLOAT8_E4M3) ? 448.0f : 57344.0f; };

/* scale and factor of a block by the bits of its largest magnitude: values are multiplied by the factor before they are
   rounded to codes, codes times the scale give the values back. Magnitudes below 2^-100 count as 2^-100, which keeps both
   numbers finite and normal; a block that holds an infinity or a NaN gets scale NaN.

   Both quotients are correctly rounded, in far fewer instructions than a general division takes, whose cases (subnormal
   numbers, overflow, zero) cannot occur: a quotient by a reciprocal, and one correction by its exact remainder (Markstein,
   IBM J. Res. Dev. 34, 1990). a 2^-20 keeps the reciprocal normal for every a. All 2^23 significands of a were compared with
   the division for both types; powers of two scale every step exactly. */
template <int CODE> __device__ __forceinline__ void block_scale(uint32_t largest, float &scale, float &factor, bool &bad)
{  constexpr float MOST = Code8<CODE>::MOST, INVERSE = 1.0f / MOST, SMALL = 0x1p-20f;
   bad = largest >= 0x7F800000u;
   const float a = fmaxf(__uint_as_float(largest), 0x1p-100f);
   float q = a * INVERSE;
   q = __builtin_fmaf(__builtin_fmaf(-MOST, q, a), INVERSE, q);
   scale = bad ? __uint_as_float(0x7FC00000u) : q;
   const float d = a * SMALL;
   float r = __builtin_amdgcn_rcpf(d);
   r = __builtin_fmaf(__builtin_fmaf(-d, r, 1.0f), r, r);
   q = (MOST * SMALL) * r;
   factor = __builtin_fmaf(__builtin_fmaf(-d, q, MOST * SMALL), r, q);
}

/* four codes of values that are multiplied by their factors, round to nearest even. The product can pass the largest code by one rounding, from where the
   conversion comes back to the largest code: what it rounds to, not what it is given, decides about overflow */
template <int CODE> __device__ __forceinline__ uint32_t code4(float a, float b, float c, float d)
{  int r = 0;
   if (CODE == OCH_FLOAT8_E4M3) { r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, r, false); r = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true); }
   else                         { r = __builtin_amdgcn_cvt_pk_bf8_f32(a, b, r, false); r = __builtin_amdgcn_cvt_pk_bf8_f32(c, d, r, true); }
   return (uint32_t)r;
}
/* the same with one factor; a block with an infinity or a NaN is 0x7F throughout, a NaN of both code types */
template <int CODE> __device__ __forceinline__ uint32_t code4(float a, float b, float c, float d, float factor, bool bad)
{  return bad ? 0x7F7F7F7Fu : code4<CODE>(a * factor, b * factor, c * factor, d * factor); }

/* eight codes to memory, the first `valid` of them */
template <bool NT = false> __device__ __forceinline__ void store_codes(uint8_t *at, och_u32x2 q, int64_t valid)
{  if (valid >= 8)
   {  const och_u32x2_any x = q;
      if (NT) __builtin_nontemporal_store(x, reinterpret_cast<och_u32x2_any *>(at)); else *reinterpret_cast<och_u32x2_any *>(at) = x;
   }
   else
   {
#pragma unroll
      for (int i = 0; i < 8; i++) if (i < valid) at[i] = (uint8_t)((i < 4 ? q.x : q.y) >> (8 * (i & 3)));
   }
}

/* host: whether a matrix of so many bytes is moved past the caches: large ones, of which little would be found there again,
   whose columns begin on whole cache lines, because a line that two accesses share would be moved twice */
static inline bool streams(const void *at, uint64_t column_bytes, uint64_t bytes) { return bytes >= (32u << 20) && ((uintptr_t)at | column_bytes) % 128 == 0; }
/* host: a launch has fewer than 2^32 threads; more work than that goes out in pieces of this many workgroups of `threads` */
static constexpr uint64_t most_groups(uint64_t threads) { return 0xFFFFFFFFull / threads; }
/* host: types that the three operations take */
static inline bool wide_type(int dtype) { return dtype == OCH_HALF || dtype == OCH_BFLOAT16 || dtype == OCH_FLOAT; }
static inline bool code_type(int dtype) { return dtype == OCH_FLOAT8_E4M3 || dtype == OCH_FLOAT8_E5M2; }
static inline size_t wide_size(int dtype) { return dtype == OCH_FLOAT ? 4 : 2; }

#define OCH_BY_WIDE(DTYPE, CALL) (DTYPE == OCH_FLOAT ? CALL(OCH_FLOAT) : DTYPE == OCH_HALF ? CALL(OCH_HALF) : CALL(OCH_BFLOAT16))

} /* namespace och */
