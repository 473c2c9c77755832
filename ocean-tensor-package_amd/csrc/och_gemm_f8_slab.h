/* How a slab of 128 k of an 8-bit operand lies in LDS, for the block-scaled product: arithmetic only, so that a host
 * program can walk through it. R rows (of op(A), or columns of op(B)) by 128 k are R * 8 chunks of 16 bytes, chunk q at
 * byte 16 q.
 *
 * KC (contiguous along k in memory): chunk q holds 16 consecutive k of row q / 8; the 16 k at 16 c lie in slot
 *    c ^ (row mod 8), so that the lanes that read the same k of neighbouring rows meet different banks.
 * !KC (contiguous along the rows): chunk q holds 16 consecutive rows of k = q / (R / 16); the rows at 16 c lie in slot
 *    c ^ twist(k), so that the eight k of a transposing read meet different banks.
 *
 * A fragment is 32 bytes per lane: lane l holds row l mod 16, and with g = l / 16 the k of 16 g .. + 15 and of
 * 64 + 16 g .. + 15. The matrix instruction pairs byte b of group g of A with byte b of group g of B, so any order of the
 * k inside the slab gives the product as long as both operands use the same. */
#pragma once
#ifndef OCH_SLAB_FN
#define OCH_SLAB_FN __device__ __forceinline__
#endif
#include <stdint.h>

namespace och {

#define OCH_F8_SLAB 128

template <bool KC, int R> struct F8Slab
{
   static constexpr uint32_t BYTES = R * OCH_F8_SLAB, CHUNKS = R * 8;
   static constexpr uint32_t PER_K = R / 16;                              /* !KC: chunks per k */
   static constexpr uint32_t SHIFT = PER_K >= 8 ? 0 : PER_K == 4 ? 1 : 2; /* !KC: neighbouring k that fill 128 bytes together share a twist */
   static_assert(R % 32 == 0 && R >= 32 && R <= 256, "32, 64, 128 or 256 rows");
   static OCH_SLAB_FN uint32_t twist(uint32_t k) { return (k >> SHIFT) & (PER_K >= 8 ? 7 : PER_K - 1); }
   /* what chunk q holds: its first row and first k */
   static OCH_SLAB_FN void where(uint32_t q, uint32_t &row, uint32_t &k)
   {  if (KC) { row = q / 8; k = 16 * ((q % 8) ^ (row % 8)); }
      else    { k = q / PER_K; row = 16 * ((q % PER_K) ^ twist(k)); }
   }
   /* KC: byte of the 16 k at 16 c of a row */
   static OCH_SLAB_FN uint32_t at_row(uint32_t row, uint32_t c) { return row * 128 + 16 * (c ^ (row % 8)); }
   /* !KC: byte that a lane reads for the transposing read of rows row0 .. + 15 (row0 a multiple of 16), k0 .. + 7 (k0 a
      multiple of 8): in every group of 16 lanes, lanes 2 e and 2 e + 1 read the 16 rows of k0 + e, and lane i of the group
      receives row i of k0 .. k0 + 7 */
   static OCH_SLAB_FN uint32_t at_k(uint32_t row0, uint32_t k0, uint32_t lane)
   {  const uint32_t e = (lane % 16) / 2;              /* twist(k0 + e) is twist(e) */
      return (k0 + e) * R + 16 * ((row0 / 16) ^ twist(e)) + 8 * (lane % 2);
   }
};

} /* namespace och */
