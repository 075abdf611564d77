// The gated delta rule's kernels, activations of float.
#define BF_DELTA_KERNELS
#include "gated_delta.h"

template struct bf::DeltaLaunch<float>;
