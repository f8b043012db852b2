// The fp32 group norm kernels (group_norm.h).
#include "group_norm.h"

template hipError_t dc::gn::launch_vec<float>(bool, const GnArgs&, const Plan&, hipStream_t);
