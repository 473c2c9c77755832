/* block-scaled products of e5m2 (A) and e4m3 (B) on 256 x 256 tiles */
#include "och_gemm_f8_pipe.h"
namespace och { int gemm_f8_pipe_54(const F8GemmParams &p, bool akc, bool bkc, hipStream_t stream) { return gemm_f8_pipe<true, false>(p, akc, bkc, stream); } }
