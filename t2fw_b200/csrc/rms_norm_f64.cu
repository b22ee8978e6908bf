// The root-mean-square norm's kernels for fp64 storage.
#include "rms_norm.cuh"

namespace t2fw {
T2FW_RMS_FORWARD(double, false);
T2FW_RMS_BACKWARD(double);
}
