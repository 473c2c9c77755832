/* block-scaled products of e4m3 (A) and e4m3 (B) on 128 x 128 tiles */
#include "och_gemm_f8_tile.h"
namespace och { int gemm_f8_tile_44(const F8GemmParams &p, bool akc, bool bkc, bool pair, dim3 grid, hipStream_t stream) { return gemm_f8_tile<false, false>(p, akc, bkc, pair, grid, stream); } }
