// Dropout whose keep decisions are drawn from the counter generator where they are used: forward and backward each draw
// them again from (seed, offset), so no mask is written, read or kept for the backward pass.
//   y = keep ? x * 1/(1-p) : 0  (+ residual),   keep(i) = uniform01(seed, offset + i) >= p
// The draw of logical element i is the one laed_dropout_keep_mask puts at place i: a stored mask and this kernel agree.
//
// fp32 is HBM-bound: 163840 x 1024 in 245 us a pass, 5.5 TB/s (one element per thread and turn: 465 us).  16-bit tensors move
// half as much per draw and are bound by the hash's 64-bit products: 16384 x 1024 bf16 in 21 us, 0.8 elements per picosecond.
#include "laed_dtypes.h"
#include <math.h>

namespace {

struct DropArgs {
    const void* x;
    const void* residual;
    void* y;
    int64_t d0, d1, d2;                    // logical shape, row-major numbering of the draws
    int64_t xs0, xs1, rs0, rs1, ys0, ys1;  // element strides of the two outer dimensions (the last one is dense)
    float scale;
    unsigned thr;                          // keep <=> 24-bit draw >= thr, thr = ceil(p 2^24)
    uint64_t seed, offset;
    const uint64_t* rng;                   // device (seed, offset), or NULL
    int64_t block0, last;                  // dense tensors: this launch's first block, and the last one of all
};

// Elements e0 .. e0 + VW of one row: the generator's index advances by one per element, so its product with the odd constant
// advances by the constant; of the hash's last product only the upper word is needed (the draw is its top 24 bits).
template <typename T, int VW>
__device__ __forceinline__ void drop_vec(const laed_vec<T, VW>& x, const laed_vec<T, VW>* res, laed_vec<T, VW>& y, uint64_t key,
                                         uint64_t index, unsigned thr, float scale) {
    uint64_t step = index * 0xD6E8FEB86659FD93ull;
#pragma unroll
    for (int e = 0; e < VW; ++e) {
        const unsigned draw = (unsigned)(mix64(key ^ step) >> 40);
        step += 0xD6E8FEB86659FD93ull;
        float v = draw >= thr ? laed_to_float(x.v[e]) * scale : 0.f;
        if (res != nullptr) v += laed_to_float(res->v[e]);
        y.v[e] = laed_from_float<T>(v);
    }
}

// Dense tensors: one row of n elements.  A block takes UNITS x 256 vectors of 16 bytes; a thread issues all its loads before
// it draws.  The tail that does not fill a vector is taken element by element by the last block's first threads.
// VW = 1: tensors that do not start on 16 bytes.
template <typename T, int VW, bool RES>
__global__ __launch_bounds__(256) void dropout_flat_kernel(DropArgs a) {
    constexpr int UNITS = 4;
    using V = laed_vec<T, VW>;
    const uint64_t key = mix64(a.rng ? a.rng[0] : a.seed), offset = a.rng ? a.rng[1] : a.offset;
    const V* x = (const V*)a.x;
    const V* res = (const V*)a.residual;
    V* y = (V*)a.y;
    const int64_t block = a.block0 + blockIdx.x, nv = a.d2 / VW, first = block * (256 * UNITS) + threadIdx.x;
    V xv[UNITS], rv[UNITS];
#pragma unroll
    for (int k = 0; k < UNITS; ++k)
        if (first + k * 256 < nv) {
            xv[k] = x[first + k * 256];
            if (RES) rv[k] = res[first + k * 256];
        }
#pragma unroll
    for (int k = 0; k < UNITS; ++k)
        if (first + k * 256 < nv) {
            V yv;
            drop_vec<T, VW>(xv[k], RES ? &rv[k] : nullptr, yv, key, offset + (uint64_t)(first + k * 256) * VW, a.thr, a.scale);
            y[first + k * 256] = yv;
        }
    if (VW > 1 && block == a.last && threadIdx.x < a.d2 - nv * VW) {
        const int64_t i = nv * VW + threadIdx.x;
        laed_vec<T, 1> x1 = {{((const T*)a.x)[i]}}, r1, y1;
        if (RES) r1.v[0] = ((const T*)a.residual)[i];
        drop_vec<T, 1>(x1, RES ? &r1 : nullptr, y1, key, offset + (uint64_t)i, a.thr, a.scale);
        ((T*)a.y)[i] = y1.v[0];
    }
}

// Strided tensors: rows of d2 elements, d2 a multiple of VW and every row on a vector boundary (VW = 1 otherwise).
template <typename T, int VW, bool RES>
__global__ __launch_bounds__(256) void dropout_rows_kernel(DropArgs a) {
    using V = laed_vec<T, VW>;
    const uint64_t key = mix64(a.rng ? a.rng[0] : a.seed), offset = a.rng ? a.rng[1] : a.offset;
    const int64_t per = a.d2 / VW, n = a.d0 * a.d1 * per;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        int64_t r, r0;
        if (n <= 0xffffffffll) {                                   // 32-bit divisions, a fraction of the 64-bit ones' cost
            r = (unsigned)i / (unsigned)per;
            r0 = (unsigned)r / (unsigned)a.d1;
        } else {
            r = i / per;
            r0 = r / a.d1;
        }
        const int64_t c = (i - r * per) * VW, r1 = r - r0 * a.d1;
        const V xv = *(const V*)((const T*)a.x + r0 * a.xs0 + r1 * a.xs1 + c);
        V rv, yv;
        if (RES) rv = *(const V*)((const T*)a.residual + r0 * a.rs0 + r1 * a.rs1 + c);
        drop_vec<T, VW>(xv, RES ? &rv : nullptr, yv, key, offset + (uint64_t)i * VW, a.thr, a.scale);
        *(V*)((T*)a.y + r0 * a.ys0 + r1 * a.ys1 + c) = yv;
    }
}

template <typename T, int VW>
void launch(DropArgs a, hipStream_t stream) {
    if (a.d0 * a.d1 == 1) {
        // a grid holds fewer than 2^32 threads: longer tensors (from 2^34 single elements on) go in several launches
        const int64_t blocks = cdiv64(cdiv64(a.d2, VW), 1024), most = 1 << 23;
        a.last = blocks - 1;
        for (a.block0 = 0; a.block0 < blocks; a.block0 += most) {
            const dim3 grid((unsigned)(blocks - a.block0 < most ? blocks - a.block0 : most));
            if (a.residual) hipLaunchKernelGGL((dropout_flat_kernel<T, VW, true>), grid, dim3(256), 0, stream, a);
            else hipLaunchKernelGGL((dropout_flat_kernel<T, VW, false>), grid, dim3(256), 0, stream, a);
        }
        return;
    }
    const int64_t blocks = cdiv64(a.d0 * a.d1 * (a.d2 / VW), 256);
    const unsigned grid = (unsigned)(blocks < (1 << 20) ? blocks : (1 << 20));
    if (a.residual) hipLaunchKernelGGL((dropout_rows_kernel<T, VW, true>), dim3(grid), dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((dropout_rows_kernel<T, VW, false>), dim3(grid), dim3(256), 0, stream, a);
}

template <typename T>
void dispatch(const DropArgs& a, hipStream_t stream) {
    constexpr int vw = 16 / sizeof(T);
    const bool flat = a.d0 * a.d1 == 1;
    const auto on = [&](const void* p, int64_t s0, int64_t s1) {
        return p == nullptr || (aligned16(p) && (flat || (s0 % vw == 0 && s1 % vw == 0)));
    };
    if ((flat || a.d2 % vw == 0) && on(a.x, a.xs0, a.xs1) && on(a.y, a.ys0, a.ys1) && on(a.residual, a.rs0, a.rs1))
        launch<T, vw>(a, stream);
    else
        launch<T, 1>(a, stream);
}

}   // namespace

extern "C" int laed_dropout(const void* x, int64_t xs0, int64_t xs1, const void* residual, int64_t rs0, int64_t rs1,
                            void* y, int64_t ys0, int64_t ys1, int64_t d0, int64_t d1, int64_t d2, int dtype, double p,
                            uint64_t seed, uint64_t offset, const void* rng, void* stream) {
    LAED_CHECK_ARG(d0 >= 0 && d1 >= 0 && d2 >= 0, "dropout: negative dimension");
    LAED_CHECK_ARG(p >= 0.0 && p <= 1.0, "dropout: p must lie in [0, 1]");
    LAED_CHECK_ARG(dtype >= LAED_F32 && dtype <= LAED_F16, "dropout: unknown dtype %d", dtype);
    if (d0 == 0 || d1 == 0 || d2 == 0) return 0;
    LAED_CHECK_ARG(x && y, "dropout: null pointer");
    LAED_CHECK_ARG(d0 <= (1ll << 40) / d1 / d2, "dropout: more than 2^40 elements");
    // the decision goes by p in fp32, as laed_dropout_keep_mask's; the factor by p itself: 1 / (1 - p) of the rounded p is off by
    // 4 half steps of fp32 at p = 0.9 and by 16 at 0.99
    DropArgs a = {x, residual, y, d0, d1, d2, xs0, xs1, rs0, rs1, ys0, ys1, p < 1.0 ? (float)(1.0 / (1.0 - p)) : 0.f,
                  (unsigned)ceilf((float)p * 16777216.0f), seed, offset, (const uint64_t*)rng, 0, 0};
#define LAUNCH(T) dispatch<T>(a, (hipStream_t)stream)
    LAED_BY_DTYPE(dtype, LAUNCH);
#undef LAUNCH
    LAED_LAUNCH_CHECK("dropout");
    return 0;
}
