// Attention of any lengths: the fp32 forward kernels.
#include "long_attention.hpp"

int la::forward_fp32(const LaParams& p, const Cut& c, hipStream_t st) { return run_forward_t<EF32>(p, c, st); }
