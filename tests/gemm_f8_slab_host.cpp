/* Host walk through the LDS layout of the block-scaled 8-bit product (csrc/och_gemm_f8_slab.h), for
   tests/test_gemm_f8_layout_cpu.py: a slab of known bytes is brought into an LDS image chunk by chunk, and every byte that
   a matrix instruction would get is compared with the element it has to be. Also checked: the chunks cover the slab once,
   reads stay inside it, and the banks that neighbouring lanes of a read meet. Returns the number of violations. */
#include <string.h>
#include <vector>
#define OCH_SLAB_FN inline
#include "och_gemm_f8_slab.h"

using namespace och;

template <bool KC, int R> static long check()
{
   typedef F8Slab<KC, R> L;
   long bad = 0;
   std::vector<uint16_t> lds(L::BYTES, 0xFFFF);             /* element number of every LDS byte: row * 128 + k */
   for (uint32_t q = 0; q < L::CHUNKS; q++)
   {  uint32_t row, k;
      L::where(q, row, k);
      for (uint32_t e = 0; e < 16; e++)
      {  const uint32_t r = row + (KC ? 0 : e), kk = k + (KC ? e : 0);
         if (r >= R || kk >= 128 || lds[16 * q + e] != 0xFFFF) { bad++; continue; }
         lds[16 * q + e] = (uint16_t)(r * 128 + kk);
      }
   }
   std::vector<int> seen(L::BYTES, 0);
   for (uint16_t v : lds) { if (v == 0xFFFF) bad++; else seen[v]++; }
   for (int s : seen) if (s != 1) bad++;
   for (uint32_t row0 = 0; row0 < R; row0 += 16)
   {  if (KC)
         for (uint32_t lane = 0; lane < 64; lane++)
            for (uint32_t half = 0; half < 2; half++)
            {  const uint32_t row = row0 + lane % 16, c = 4 * half + lane / 16, at = L::at_row(row, c);
               if (at + 16 > L::BYTES || at % 16) { bad++; continue; }
               for (uint32_t e = 0; e < 16; e++) if (lds[at + e] != row * 128 + 16 * c + e) bad++;
               if (lane % 8 == 0)                            /* eight neighbouring lanes cover all 128 bytes once */
               {  uint32_t slots = 0;
                  for (uint32_t x = 0; x < 8; x++) slots |= 1u << (L::at_row(row0 + (lane + x) % 16, 4 * half + (lane + x) / 16) / 16 % 8);
                  if (slots != 0xFF) bad++;
               }
            }
      else
         for (uint32_t g = 0; g < 4; g++)
            for (uint32_t i = 0; i < 4; i++)
            {  const uint32_t k0 = 16 * g + 64 * (i / 2) + 8 * (i % 2);
               uint32_t slots = 0;
               for (uint32_t lane = 0; lane < 16; lane++)
               {  const uint32_t at = L::at_k(row0, k0, 16 * g + lane);
                  if (at + 8 > L::BYTES || at % 8) { bad++; continue; }
                  for (uint32_t e = 0; e < 8; e++)           /* rows row0 + 8 (lane mod 2) + e of k0 + lane / 2 */
                     if (lds[at + e] != (row0 + 8 * (lane % 2) + e) * 128 + k0 + lane / 2) bad++;
                  slots |= 1u << (at / 8 % 16);
               }
               if (slots != 0xFFFF) bad++;                   /* sixteen lanes cover 128 bytes of banks once */
            }
   }
   return bad;
}

extern "C" long gemm_f8_slab_check(int kc, int rows)
{
   switch (rows)
   {  case 32:  return kc ? check<true, 32>() : check<false, 32>();
      case 64:  return kc ? check<true, 64>() : check<false, 64>();
      case 128: return kc ? check<true, 128>() : check<false, 128>();
      case 256: return kc ? check<true, 256>() : check<false, 256>();
   }
   return -1;
}
