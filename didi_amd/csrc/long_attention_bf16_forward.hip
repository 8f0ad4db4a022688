// Attention of any lengths: the bf16 forward kernels.
#include "long_attention.hpp"

int la::forward_bf16(const LaParams& p, const Cut& c, hipStream_t st) { return run_forward_t<E16<false>>(p, c, st); }
