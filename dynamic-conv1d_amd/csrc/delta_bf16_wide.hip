// The bf16 gated delta rule kernels for float32 results (delta_mfma.h).
#include "delta_mfma.h"

template hipError_t dc::dr::launch<dc::bf16, 3>(dc::dr::Stage, const dc::dr::Args&, int, hipStream_t);
