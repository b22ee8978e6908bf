// The root-mean-square norm's kernels for fp32 storage.
#include "rms_norm.cuh"

namespace t2fw {
T2FW_RMS_FORWARD(float, false);
T2FW_RMS_FORWARD(float, true);
T2FW_RMS_BACKWARD(float);
}
