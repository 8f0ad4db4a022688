// Attention of any lengths: the fp32 backward kernels.
#include "long_attention.hpp"

int la::backward_fp32(const LaParams& p, const Plan& z, void* dtable, hipStream_t st) { return run_backward_t<EF32>(p, z, dtable, st); }
