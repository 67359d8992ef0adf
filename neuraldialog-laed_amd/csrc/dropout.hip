// Dropout whose keep decisions are drawn from the counter generator where they are used: forward and backward each draw
// them again from (seed, offset), so no mask is written, read or kept for the backward pass.
//   y = keep ? x * 1/(1-p) : 0  (+ residual),   keep(i) = uniform01(seed, offset + i) >= p
// The draw of logical element i is the one laed_dropout_keep_mask puts at place i: a stored mask and this kernel agree.
#include "laed_dtypes.h"
#include <math.h>

namespace {

struct DropArgs {
    const void* x;
    const void* residual;
    void* y;
    int64_t d0, d1, d2;                    // logical shape, row-major numbering of the draws
    int64_t xs0, xs1, rs0, rs1, ys0, ys1;  // element strides of the two outer dimensions (the last one is dense)
    float p, scale;
    unsigned thr;                          // keep <=> 24-bit draw >= thr, thr = ceil(p 2^24)
    uint64_t seed, offset;
    const uint64_t* rng;                   // device (seed, offset), or NULL
};

// first version: one element per thread and turn
template <typename T>
__global__ __launch_bounds__(256) void dropout_kernel(DropArgs a) {
    const uint64_t seed = a.rng ? a.rng[0] : a.seed, offset = a.rng ? a.rng[1] : a.offset;
    const T* x = (const T*)a.x;
    const T* res = (const T*)a.residual;
    T* y = (T*)a.y;
    const int64_t n = a.d0 * a.d1 * a.d2;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t r = i / a.d2, c = i - r * a.d2, r0 = r / a.d1, r1 = r - r0 * a.d1;
        const bool keep = uniform01(seed, offset + (uint64_t)i) >= a.p;
        float v = keep ? laed_to_float(x[r0 * a.xs0 + r1 * a.xs1 + c]) * a.scale : 0.f;
        if (res != nullptr) v += laed_to_float(res[r0 * a.rs0 + r1 * a.rs1 + c]);
        y[r0 * a.ys0 + r1 * a.ys1 + c] = laed_from_float<T>(v);
    }
}

}   // namespace

extern "C" int laed_dropout(const void* x, int64_t xs0, int64_t xs1, const void* residual, int64_t rs0, int64_t rs1,
                            void* y, int64_t ys0, int64_t ys1, int64_t d0, int64_t d1, int64_t d2, int dtype, float p,
                            uint64_t seed, uint64_t offset, const void* rng, void* stream) {
    LAED_CHECK_ARG(d0 >= 0 && d1 >= 0 && d2 >= 0, "dropout: negative dimension");
    LAED_CHECK_ARG(p >= 0.f && p <= 1.f, "dropout: p must lie in [0, 1]");
    LAED_CHECK_ARG(dtype >= LAED_F32 && dtype <= LAED_F16, "dropout: unknown dtype %d", dtype);
    if (d0 == 0 || d1 == 0 || d2 == 0) return 0;
    LAED_CHECK_ARG(x && y, "dropout: null pointer");
    LAED_CHECK_ARG(d0 <= INT64_MAX / d1 / d2, "dropout: too many elements");
    DropArgs a = {x, residual, y, d0, d1, d2, xs0, xs1, rs0, rs1, ys0, ys1, p, p < 1.f ? (float)(1.0 / (1.0 - (double)p)) : 0.f,
                  (unsigned)ceilf(p * 16777216.0f), seed, offset, (const uint64_t*)rng};
    const int64_t n = d0 * d1 * d2;
    const int grid = (int)(cdiv64(n, 256) < 65536 ? cdiv64(n, 256) : 65536);
#define LAUNCH(T) hipLaunchKernelGGL((dropout_kernel<T>), dim3(grid), dim3(256), 0, (hipStream_t)stream, a)
    LAED_BY_DTYPE(dtype, LAUNCH);
#undef LAUNCH
    LAED_LAUNCH_CHECK("dropout");
    return 0;
}
