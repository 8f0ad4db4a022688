// Attention of any lengths: the fp16 forward kernels.
#include "long_attention.hpp"

int la::forward_fp16(const LaParams& p, const Cut& c, hipStream_t st) { return run_forward_t<E16<true>>(p, c, st); }
