/* block-scaled products of e4m3 (A) and e5m2 (B) on 128 x 128 tiles */
#include "och_gemm_f8_tile.h"
namespace och { int gemm_f8_tile_45(const F8GemmParams &p, bool akc, bool bkc, bool pair, dim3 grid, hipStream_t stream) { return gemm_f8_tile<false, true>(p, akc, bkc, pair, grid, stream); } }
