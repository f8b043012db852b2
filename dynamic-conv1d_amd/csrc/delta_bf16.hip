// The bf16 gated delta rule kernels (delta_mfma.h).
#include "delta_mfma.h"

template hipError_t dc::dr::launch<dc::bf16, 2>(dc::dr::Stage, const dc::dr::Args&, int, hipStream_t);
