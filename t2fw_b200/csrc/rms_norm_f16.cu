// The root-mean-square norm's kernels for fp16 storage.
#include "rms_norm.cuh"

namespace t2fw {
T2FW_RMS_FORWARD(__half, false);
T2FW_RMS_FORWARD(__half, true);
T2FW_RMS_BACKWARD(__half);
}
