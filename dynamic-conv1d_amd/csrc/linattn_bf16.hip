// The bf16 linear attention kernels (linattn_mfma.h).
#include "linattn_mfma.h"

template hipError_t dc::la::launch<dc::bf16>(const dc::la::Args&, int, int, bool, bool, hipStream_t);
