// Filtered sampling: the C entry and the fp32 kernels (laed_sample.h).
#include "laed_sample.h"

void laed_sample_launch_f32(const SampleArgs& a, hipStream_t stream) { launch<float>(a, stream); }

extern "C" int laed_sample_rows(const void* logits, int64_t ld, int64_t N, int V, int dtype, const float* u, uint64_t seed,
                                uint64_t offset, double temperature, const float* temperature_rows, int64_t top_k,
                                const int64_t* top_k_rows, double top_p, const float* top_p_rows, double min_p,
                                const float* min_p_rows, int64_t* ids, float* logp, void* stream) {
    LAED_CHECK_ARG(N >= 0 && N <= INT32_MAX && V >= 1, "sample_rows: bad size");
    LAED_CHECK_ARG(dtype >= LAED_F32 && dtype <= LAED_F16, "sample_rows: unknown dtype %d", dtype);
    LAED_CHECK_ARG(V <= (1 << 28), "sample_rows: V must not exceed 2^28");
    LAED_CHECK_ARG(temperature_rows || temperature >= 0.0, "sample_rows: temperature must be >= 0 (0 = greedy)");
    LAED_CHECK_ARG(top_p_rows || (top_p >= 0.0 && top_p <= 1.0), "sample_rows: top_p must lie in [0, 1]");
    LAED_CHECK_ARG(min_p_rows || (min_p >= 0.0 && min_p <= 1.0), "sample_rows: min_p must lie in [0, 1]");
    if (N == 0) return 0;
    LAED_CHECK_ARG(logits && ids, "sample_rows: null pointer");
    int lg = 0;
    while ((1ll << lg) < V) ++lg;
    SampleArgs a = {logits, ld, N, 0, V, 62 - lg < 46 ? 62 - lg : 46, u, seed, offset, temperature, temperature_rows, top_k, top_k_rows,
                    top_p, top_p_rows, min_p, min_p_rows, ids, logp};
    if (dtype == LAED_BF16) laed_sample_launch_bf16(a, (hipStream_t)stream);
    else if (dtype == LAED_F16) laed_sample_launch_f16(a, (hipStream_t)stream);
    else laed_sample_launch_f32(a, (hipStream_t)stream);
    LAED_LAUNCH_CHECK("sample_rows");
    return 0;
}
