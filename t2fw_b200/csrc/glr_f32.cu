// The gated linear recurrence's kernels for fp32 storage.
#include "glr_scan.cuh"

namespace t2fw {
T2FW_GLR_INSTANTIATE(float);
}
