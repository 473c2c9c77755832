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
   __device__ __forceinline__ void load(const E *at, int64_t valid)
   {  if (valid >= 8)
      {
#pragma unroll
         for (int w = 0; w < WORDS; w++) raw[w] = reinterpret_cast<const och_u32x4_any *>(at)[w];
      }
      else
      {
#pragma unroll
         for (int i = 0; i < 8; i++) e[i] = (i < valid) ? at[i] : (E)0.0f;
      }
   }
   __device__ __forceinline__ void store(E *at, int64_t valid) const
   {  if (valid >= 8)
      {
#pragma unroll
         for (int w = 0; w < WORDS; w++) reinterpret_cast<och_u32x4_any *>(at)[w] = raw[w];
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
{  return umax(x, (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, CTRL, 0xF, 0xF, false)); }
__device__ __forceinline__ uint32_t row16_max(uint32_t x)
{  x = dpp_max<0xB1>(x); x = dpp_max<0x4E>(x); x = dpp_max<0x141>(x); return dpp_max<0x140>(x); }

template <int CODE> struct Code8 { static constexpr float MOST = (CODE == OCH_FLOAT8_E4M3) ? 448.0f : 57344.0f; };

/* scale and factor of a block by the bits of its largest magnitude: values are multiplied by the factor before they are
   rounded to codes, codes times the scale give the values back. Magnitudes below 2^-100 count as 2^-100, which keeps both
   numbers finite and normal; a block that holds an infinity or a NaN gets scale NaN. */
template <int CODE> __device__ __forceinline__ void block_scale(uint32_t largest, float &scale, float &factor, bool &bad)
{  bad = largest >= 0x7F800000u;
   const float a = fmaxf(__uint_as_float(largest), 0x1p-100f);
   scale = bad ? __uint_as_float(0x7FC00000u) : a / Code8<CODE>::MOST;
   factor = Code8<CODE>::MOST / a;
}

/* four codes, round to nearest even. The product with the factor can pass the largest code by one rounding: the clamp
   keeps it there, because what the conversion makes of larger values depends on a mode bit */
template <int CODE> __device__ __forceinline__ uint32_t code4(float a, float b, float c, float d, float factor, bool bad)
{  constexpr float M = Code8<CODE>::MOST;
   a = __builtin_amdgcn_fmed3f(a * factor, -M, M); b = __builtin_amdgcn_fmed3f(b * factor, -M, M);
   c = __builtin_amdgcn_fmed3f(c * factor, -M, M); d = __builtin_amdgcn_fmed3f(d * factor, -M, M);
   int r = 0;
   if (CODE == OCH_FLOAT8_E4M3) { r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, r, false); r = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true); }
   else                         { r = __builtin_amdgcn_cvt_pk_bf8_f32(a, b, r, false); r = __builtin_amdgcn_cvt_pk_bf8_f32(c, d, r, true); }
   return bad ? 0x7F7F7F7Fu : (uint32_t)r;            /* 0x7F is a NaN of both code types */
}

/* eight codes to memory, the first `valid` of them */
__device__ __forceinline__ void store_codes(uint8_t *at, och_u32x2 q, int64_t valid)
{  if (valid >= 8) *reinterpret_cast<och_u32x2_any *>(at) = q;
   else
   {
#pragma unroll
      for (int i = 0; i < 8; i++) if (i < valid) at[i] = (uint8_t)((i < 4 ? q.x : q.y) >> (8 * (i & 3)));
   }
}

/* host: types that the three operations take */
static inline bool wide_type(int dtype) { return dtype == OCH_HALF || dtype == OCH_BFLOAT16 || dtype == OCH_FLOAT; }
static inline bool code_type(int dtype) { return dtype == OCH_FLOAT8_E4M3 || dtype == OCH_FLOAT8_E5M2; }
static inline size_t wide_size(int dtype) { return dtype == OCH_FLOAT ? 4 : 2; }

#define OCH_BY_WIDE(DTYPE, CALL) (DTYPE == OCH_FLOAT ? CALL(OCH_FLOAT) : DTYPE == OCH_HALF ? CALL(OCH_HALF) : CALL(OCH_BFLOAT16))

} /* namespace och */
