// Attention of any lengths: the fp16 backward kernels.
#include "long_attention.hpp"

int la::backward_fp16(const LaParams& p, const Plan& z, void* dtable, hipStream_t st) { return run_backward_t<E16<true>>(p, z, dtable, st); }
