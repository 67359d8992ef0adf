// Filtered sampling: the fp16 kernels (laed_sample.h).
#include "laed_sample.h"

void laed_sample_launch_f16(const SampleArgs& a, hipStream_t stream) { launch<laed_f16>(a, stream); }
