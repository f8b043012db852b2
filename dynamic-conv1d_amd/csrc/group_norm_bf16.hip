// The bf16 group norm kernels (group_norm.h).
#include "group_norm.h"

template hipError_t dc::gn::launch_vec<dc::bf16>(bool, const GnArgs&, const Plan&, hipStream_t);
