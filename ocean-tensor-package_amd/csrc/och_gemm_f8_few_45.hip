/* block-scaled products of e4m3 (A) and e5m2 (B) with few columns */
#include "och_gemm_f8_few.h"
namespace och { int gemm_f8_few_45(const F8GemmParams &p, hipStream_t stream) { return gemm_f8_few<false, true>(p, stream); } }
