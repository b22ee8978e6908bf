// The gated linear recurrence's kernels for bf16 storage.
#include "glr_scan.cuh"

namespace t2fw {
T2FW_GLR_INSTANTIATE(__nv_bfloat16);
}
