// Attention of any lengths: the forward on split planes (joined and multiplied in fp32).
#include "long_attention.hpp"

int la::forward_planes(const LaParams& p, const Cut& c, bool f16, hipStream_t st) {
    return f16 ? run_forward_t<EPlanes<true>>(p, c, st) : run_forward_t<EPlanes<false>>(p, c, st);
}
