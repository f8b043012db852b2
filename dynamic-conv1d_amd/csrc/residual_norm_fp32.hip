// The fp32 residual norm kernels (residual_norm.h).
#include "residual_norm.h"

template hipError_t dc::rn::launch_vec<float>(bool, const dc::rn::Args&, const dc::rn::Plan&, bool, hipStream_t);
