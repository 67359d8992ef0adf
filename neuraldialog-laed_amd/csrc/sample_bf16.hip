// Filtered sampling: the bf16 kernels (laed_sample.h).
#include "laed_sample.h"

void laed_sample_launch_bf16(const SampleArgs& a, hipStream_t stream) { launch<laed_bf16>(a, stream); }
