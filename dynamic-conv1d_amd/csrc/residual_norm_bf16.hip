// The bf16 residual norm kernels (residual_norm.h).
#include "residual_norm.h"

template hipError_t dc::rn::launch_vec<dc::bf16>(bool, const dc::rn::Args&, const dc::rn::Plan&, bool, hipStream_t);
