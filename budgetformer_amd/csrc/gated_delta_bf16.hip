// The gated delta rule's kernels, activations of __bf16.
#define BF_DELTA_KERNELS
#include "gated_delta.h"

template struct bf::DeltaLaunch<__bf16>;
