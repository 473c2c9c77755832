/* block-scaled products of e5m2 (A) and e5m2 (B) with few columns */
#include "och_gemm_f8_few.h"
namespace och { int gemm_f8_few_55(const F8GemmParams &p, hipStream_t stream) { return gemm_f8_few<true, true>(p, stream); } }
