// Gated linear recurrence  h_t = z_t h_{t-1} + (1 - z_t) x_t,  z_t = sigmoid(f_t),  and its backward pass
//   g_t = dout_t + z_{t+1} g_{t+1};  dx_t = (1 - z_t) g_t;  df_t = g_t (h_{t-1} - x_t) z_t (1 - z_t);  dh0 = z_0 g_0.
// A position t >= lengths[b] is an identity step (z = 1): nothing is read there, the outputs and gradients are zeros.
// For the backward pass the forward one keeps the fp32 state in front of every block of SCAN_BLOCK steps; the backward pass
// runs a block forward again from there, so neither the states nor the gates are stored and the states it uses are the
// fp32 ones whatever the tensors' type.
#include "laed_dtypes.h"

namespace {

constexpr int SCAN_BLOCK = 16;

struct ScanArgs {
    const void* gi;                       // (f | x) halves of the last dimension, element (t, b, c) at t*gst + b*gsb + c
    int64_t gst, gsb;
    const float* h0;                      // [B][H] or NULL (zeros)
    const int64_t* lengths;               // [B] or NULL
    int T, B, H, reverse;
    void* out; int64_t ost, osb;          // forward
    float* hT;
    float* tape;                          // [ceil(T / SCAN_BLOCK)][B][H] or NULL
    const void* dout; int64_t dst, dsb;   // backward
    const float* dhT;
    void* dgi; int64_t qst, qsb;
    float* dh0;
};

// z and 1 - z, each to full relative precision: the smaller one from e^-|f| / (1 + e^-|f|), the larger one as 1 - smaller
// (rounded to nearest; no systematic error accumulates over a long product of z).
__device__ __forceinline__ void gate(float f, float& z, float& u) {
    const float e = __builtin_amdgcn_exp2f(fabsf(f) * -1.44269504088896341f);
    const float s = e * __builtin_amdgcn_rcpf(1.0f + e), l = 1.0f - s;
    z = f >= 0.f ? l : s;
    u = f >= 0.f ? s : l;
}

// first version: one thread per channel walks the whole sequence
template <typename T>
__global__ __launch_bounds__(256) void scan_fwd_kernel(ScanArgs a) {
    const int64_t C = (int64_t)a.B * a.H, c = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (c >= C) return;
    const int64_t b = c / a.H, k = c - b * a.H;
    const T* gi = (const T*)a.gi + b * a.gsb + k;
    T* out = (T*)a.out + b * a.osb + k;
    const int64_t len = a.lengths ? a.lengths[b] : a.T;
    float h = a.h0 ? a.h0[c] : 0.f;
    for (int s = 0; s < a.T; ++s) {
        const int64_t t = a.reverse ? a.T - 1 - s : s;
        if (a.tape && s % SCAN_BLOCK == 0) a.tape[s / SCAN_BLOCK * C + c] = h;
        float o = 0.f;
        if (t < len) {
            float z, u;
            gate(laed_to_float(gi[t * a.gst]), z, u);
            h = fmaf(z, h, u * laed_to_float(gi[t * a.gst + a.H]));
            o = h;
        }
        out[t * a.ost] = laed_from_float<T>(o);
    }
    if (a.hT) a.hT[c] = h;
}

template <typename T>
__global__ __launch_bounds__(256) void scan_bwd_kernel(ScanArgs a) {
    const int64_t C = (int64_t)a.B * a.H, c = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (c >= C) return;
    const int64_t b = c / a.H, k = c - b * a.H;
    const T* gi = (const T*)a.gi + b * a.gsb + k;
    const T* dout = a.dout ? (const T*)a.dout + b * a.dsb + k : nullptr;
    T* dgi = (T*)a.dgi + b * a.qsb + k;
    const int64_t len = a.lengths ? a.lengths[b] : a.T;
    float g = a.dhT ? a.dhT[c] : 0.f;      // z_{t+1} g_{t+1}
    for (int blk = (a.T + SCAN_BLOCK - 1) / SCAN_BLOCK - 1; blk >= 0; --blk) {
        float hp[SCAN_BLOCK], z[SCAN_BLOCK], u[SCAN_BLOCK], x[SCAN_BLOCK];
        float h = a.tape[blk * C + c];
        const int s0 = blk * SCAN_BLOCK;
#pragma unroll
        for (int i = 0; i < SCAN_BLOCK; ++i) {
            const int64_t t = a.reverse ? a.T - 1 - (s0 + i) : s0 + i;
            hp[i] = h; z[i] = 1.f; u[i] = 0.f; x[i] = 0.f;
            if (s0 + i < a.T && t < len) {
                gate(laed_to_float(gi[t * a.gst]), z[i], u[i]);
                x[i] = laed_to_float(gi[t * a.gst + a.H]);
                h = fmaf(z[i], h, u[i] * x[i]);
            }
        }
#pragma unroll
        for (int i = SCAN_BLOCK - 1; i >= 0; --i) {
            const int64_t t = a.reverse ? a.T - 1 - (s0 + i) : s0 + i;
            if (s0 + i >= a.T) continue;
            float df = 0.f, dx = 0.f;
            if (t < len) {
                if (dout) g += laed_to_float(dout[t * a.dst]);
                dx = u[i] * g;
                df = g * (hp[i] - x[i]) * (z[i] * u[i]);
                g *= z[i];
            }
            dgi[t * a.qst] = laed_from_float<T>(df);
            dgi[t * a.qst + a.H] = laed_from_float<T>(dx);
        }
    }
    if (a.dh0) a.dh0[c] = g;
}

}   // namespace

extern "C" int64_t laed_gated_scan_tape(int T, int B, int H) {
    if (T <= 0 || B <= 0 || H <= 0) return 0;
    return cdiv64(T, SCAN_BLOCK) * B * H;
}

extern "C" int laed_gated_scan_fwd(const void* gi, int64_t gi_st, int64_t gi_sb, const float* h0, const int64_t* lengths,
                                   int T, int B, int H, int dtype, int reverse, void* out, int64_t out_st, int64_t out_sb,
                                   float* hT, float* tape, void* stream) {
    LAED_CHECK_ARG(T >= 0 && B >= 0 && H >= 0, "gated_scan_fwd: negative dimension");
    LAED_CHECK_ARG(dtype >= LAED_F32 && dtype <= LAED_F16, "gated_scan_fwd: unknown dtype %d", dtype);
    if (B == 0 || H == 0) return 0;
    LAED_CHECK_ARG(T == 0 || (gi && out), "gated_scan_fwd: null pointer");
    ScanArgs a = {};
    a.gi = gi; a.gst = gi_st; a.gsb = gi_sb; a.h0 = h0; a.lengths = lengths; a.T = T; a.B = B; a.H = H; a.reverse = reverse;
    a.out = out; a.ost = out_st; a.osb = out_sb; a.hT = hT; a.tape = tape;
    const int64_t blocks = cdiv64((int64_t)B * H, 256);
    LAED_CHECK_ARG(blocks <= INT32_MAX, "gated_scan_fwd: B * H too large");
#define LAUNCH(T_) hipLaunchKernelGGL((scan_fwd_kernel<T_>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, a)
    LAED_BY_DTYPE(dtype, LAUNCH);
#undef LAUNCH
    LAED_LAUNCH_CHECK("gated_scan_fwd");
    return 0;
}

extern "C" int laed_gated_scan_bwd(const void* gi, int64_t gi_st, int64_t gi_sb, const float* tape, const int64_t* lengths,
                                   const void* dout, int64_t dout_st, int64_t dout_sb, const float* dhT, int T, int B, int H,
                                   int dtype, int reverse, void* dgi, int64_t dgi_st, int64_t dgi_sb, float* dh0, void* stream) {
    LAED_CHECK_ARG(T >= 0 && B >= 0 && H >= 0, "gated_scan_bwd: negative dimension");
    LAED_CHECK_ARG(dtype >= LAED_F32 && dtype <= LAED_F16, "gated_scan_bwd: unknown dtype %d", dtype);
    if (B == 0 || H == 0) return 0;
    LAED_CHECK_ARG(T == 0 || (gi && tape && dgi), "gated_scan_bwd: null pointer");
    ScanArgs a = {};
    a.gi = gi; a.gst = gi_st; a.gsb = gi_sb; a.tape = (float*)tape; a.lengths = lengths; a.T = T; a.B = B; a.H = H;
    a.reverse = reverse; a.dout = dout; a.dst = dout_st; a.dsb = dout_sb; a.dhT = dhT; a.dgi = dgi; a.qst = dgi_st; a.qsb = dgi_sb;
    a.dh0 = dh0;
    const int64_t blocks = cdiv64((int64_t)B * H, 256);
    LAED_CHECK_ARG(blocks <= INT32_MAX, "gated_scan_bwd: B * H too large");
#define LAUNCH(T_) hipLaunchKernelGGL((scan_bwd_kernel<T_>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, a)
    LAED_BY_DTYPE(dtype, LAUNCH);
#undef LAUNCH
    LAED_LAUNCH_CHECK("gated_scan_bwd");
    return 0;
}
