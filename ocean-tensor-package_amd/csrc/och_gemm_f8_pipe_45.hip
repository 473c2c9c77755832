/* block-scaled products of e4m3 (A) and e5m2 (B) on 256 x 256 tiles */
#include "och_gemm_f8_pipe.h"
namespace och { int gemm_f8_pipe_45(const F8GemmParams &p, bool akc, bool bkc, hipStream_t stream) { return gemm_f8_pipe<false, true>(p, akc, bkc, stream); } }
