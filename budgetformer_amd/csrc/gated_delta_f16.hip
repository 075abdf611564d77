// The gated delta rule's kernels, activations of _Float16.
#define BF_DELTA_KERNELS
#include "gated_delta.h"

template struct bf::DeltaLaunch<_Float16>;
