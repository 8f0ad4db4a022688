// Attention of any lengths: the bf16 backward kernels.
#include "long_attention.hpp"

int la::backward_bf16(const LaParams& p, const Plan& z, void* dtable, hipStream_t st) { return run_backward_t<E16<false>>(p, z, dtable, st); }
