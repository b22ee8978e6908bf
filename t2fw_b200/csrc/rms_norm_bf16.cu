// The root-mean-square norm's kernels for bf16 storage.
#include "rms_norm.cuh"

namespace t2fw {
T2FW_RMS_FORWARD(__nv_bfloat16, false);
T2FW_RMS_FORWARD(__nv_bfloat16, true);
T2FW_RMS_BACKWARD(__nv_bfloat16);
}
