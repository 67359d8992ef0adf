// Gated linear recurrence  h_t = z_t h_{t-1} + (1 - z_t) x_t,  z_t = sigmoid(f_t),  and its backward pass
//   g_t = dout_t + z_{t+1} g_{t+1};  dx_t = (1 - z_t) g_t;  df_t = g_t (h_{t-1} - x_t) z_t (1 - z_t);  dh0 = z_0 g_0.
// A position t >= lengths[b] is an identity step (z = 1): nothing is read there, the outputs and gradients are zeros.
//
// A stretch of steps maps the state in front of it to the state behind it by  h -> A h + b  with A = product of z and b the
// stretch's own recurrence from zero, and stretches compose: time is split three ways over
//   lanes' registers   LSTEP steps per wave, loaded at once (the loads in flight that HBM needs)
//   waves of a block   a tile of `waves` x LSTEP steps; (A, b) go through LDS, one barrier per tile, every wave folds all
//                      of them itself and so keeps the tile's end state in registers without a second exchange
//   blocks             few channels and a long time axis: `segs` segments of tiles; a first launch reduces each segment to
//                      (A, b), a second one folds them into the state in front of each segment, the third one is the scan
// For the backward pass the forward one keeps the fp32 state in front of every tile (1 / tile of the outputs' size); the
// backward pass runs a tile forward again from there, so neither states nor gates are stored, and the states it uses are the
// fp32 ones whatever the tensors' type: 3 reads and 2 writes an element, where stored states would take 4 and 2.
//
// HBM-bound (about 75 cycles of arithmetic per 64 elements and pass against 200 and more of memory).  Measured on one MI355X:
// 4096 x 40 x 1024 fp32 forward 398 us (5.1 TB/s), backward 797 us (4.2 TB/s); 2 x 16384 x 1024 bf16 72 us (29 the reduction, 6 the
// fold, 37 the scan) and 92 us (25, 7, 60); one thread per channel took 1423 us for the first pair and 16.7 ms for the second.
// LSTEP x 8 bytes a lane: 4 channels of 16 bits forward, 2 of either type backward (4 need 255 registers: one block per
// CU, 77 us instead of 60 on the long case).
#include "laed_dtypes.h"

namespace {

constexpr int LSTEP = 8;
constexpr int MAXW = 8;

struct ScanArgs {
    const void* gi;                       // (f | x) halves of the last dimension, element (t, b, c) at t*gst + b*gsb + c
    int64_t gst, gsb;
    const float* h0;                      // [B][H] or NULL (zeros)
    const int64_t* lengths;               // [B] or NULL
    int T, B, H, reverse;
    int waves, tiles, segs, seg_tiles;    // tile = waves * LSTEP steps; segment = seg_tiles tiles
    void* out; int64_t ost, osb;          // forward
    float* hT;
    float* tape;                          // [tiles][B][H] or NULL
    const void* dout; int64_t dst, dsb;   // backward
    const float* dhT;
    void* dgi; int64_t qst, qsb;
    float* dh0;
    float* ws;                            // segs > 1: [segs][2][B*H], (A, b) of each segment, b replaced by the state in front
};

// How time is divided: a function of the sizes alone, so that the backward call finds the forward call's tape.
struct ScanPlan { int waves, tiles, segs, seg_tiles; };

ScanPlan scan_plan(int T, int B, int H) {
    ScanPlan p;
    const int longest = MAXW * LSTEP;
    p.tiles = (int)cdiv64(T, longest);
    if (p.tiles < 1) p.tiles = 1;
    p.waves = (int)cdiv64(T, (int64_t)p.tiles * LSTEP);            // balanced: 65 steps are 2 tiles of 40, not 64 + 1
    if (p.waves < 1) p.waves = 1;
    p.tiles = (int)cdiv64(T, p.waves * LSTEP);
    // blocks of 64 x 2 channels; 1024 of them are four (with 4 channels a lane, two) per CU: against 512, the long case's
    // passes took 29 and 37 us instead of 41 and 49.  From 512 strips on one segment, which reads the inputs once.  Forward + backward
    // in us, one segment | this rule's number (inputs not in the caches):
    //   strips   bf16 T 1024   bf16 T 4096   fp32 T 1024   fp32 T 4096
    //       64    231 |  96     926 |  226    148 | 104     597 |  333
    //      128    247 | 119     988 |  428    165 | 155     644 |  604
    //      256    267 | 216    1055 |  809    221 | 321     813 | 1179
    //      511    399 | 536    1551 | 2054    515 | 738    2246 | 2944
    // So the border of 512 is right for neither type: 16 bits gain up to 256 strips, fp32 up to 128, and between there and
    // 512 the second read costs more than the blocks gain.
    const int64_t strips = cdiv64((int64_t)B * H, 128);
    int64_t segs = strips >= 512 ? 1 : cdiv64(1024, strips);
    if (segs > p.tiles / 2) segs = p.tiles / 2;                    // a segment is two tiles at least: its block folds, then scans
    if (segs < 1) segs = 1;
    p.seg_tiles = (int)cdiv64(p.tiles, segs);
    if (p.seg_tiles < 1) p.seg_tiles = 1;
    p.segs = (int)cdiv64(p.tiles, p.seg_tiles);
    if (p.segs < 1) p.segs = 1;
    return p;
}

// z and 1 - z, each to full relative precision: the smaller one from e^-|f| / (1 + e^-|f|), the larger one as 1 - smaller
// (rounded to nearest; no systematic error accumulates over a long product of z).
__device__ __forceinline__ void gate(float f, float& z, float& u) {
    const float e = __builtin_amdgcn_exp2f(fabsf(f) * -1.44269504088896341f);
    const float s = e * __builtin_amdgcn_rcpf(1.0f + e), l = 1.0f - s;
    z = f >= 0.f ? l : s;
    u = f >= 0.f ? s : l;
}

// The same in one register: the smaller gate with f's sign (an identity step is +0: z = 1, 1 - z = 0).
__device__ __forceinline__ float signed_gate(float f) {
    const float e = __builtin_amdgcn_exp2f(fabsf(f) * -1.44269504088896341f);
    return copysignf(e * __builtin_amdgcn_rcpf(1.0f + e), f);
}
__device__ __forceinline__ void gates_of(float sg, float& z, float& u) {
    const float s = fabsf(sg), l = 1.0f - s;
    const bool open = __float_as_int(sg) >= 0;
    z = open ? l : s;
    u = open ? s : l;
}

template <int VW> struct Chan { float v[VW]; };

// One lane's place: VW channels of one sequence.
template <int VW>
struct Lane {
    int64_t c, b, k;
    int len;
    bool on;
    __device__ __forceinline__ Lane(const ScanArgs& a, int64_t group) {
        const int64_t C = (int64_t)a.B * a.H;
        c = group * VW;
        on = c < C;
        if (!on) c = 0;
        b = c / a.H;
        k = c - b * a.H;
        len = a.T;
        if (a.lengths) {
            const int64_t l = a.lengths[b];
            len = l < 0 ? 0 : (l < a.T ? (int)l : a.T);
        }
        if (!on) len = 0;
    }
};

template <typename T, int VW>
__device__ __forceinline__ Chan<VW> load_ch(const T* p) {
    const laed_vec<T, VW> r = *reinterpret_cast<const laed_vec<T, VW>*>(p);
    Chan<VW> c;
#pragma unroll
    for (int j = 0; j < VW; ++j) c.v[j] = laed_to_float(r.v[j]);
    return c;
}
template <typename T, int VW>
__device__ __forceinline__ void store_ch(T* p, const Chan<VW>& c) {
    laed_vec<T, VW> r;
#pragma unroll
    for (int j = 0; j < VW; ++j) r.v[j] = laed_from_float<T>(c.v[j]);
    *reinterpret_cast<laed_vec<T, VW>*>(p) = r;
}
template <int VW> __device__ __forceinline__ Chan<VW> zeros() {
    Chan<VW> c;
#pragma unroll
    for (int j = 0; j < VW; ++j) c.v[j] = 0.f;
    return c;
}

// step s of the walk is position t = s (or T-1-s); real = inside the sequence
__device__ __forceinline__ int position(const ScanArgs& a, int s) { return a.reverse ? a.T - 1 - s : s; }

// AGG: only (A, b) of the segment.  Grid: x = strips of 64 VW channels, y = segments.
template <typename T, int VW, bool AGG>
__global__ __launch_bounds__(64 * MAXW) void scan_fwd_kernel(ScanArgs a) {
    __shared__ Chan<VW> sA[2][MAXW][64], sB[2][MAXW][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = a.waves;
    const Lane<VW> me(a, (int64_t)blockIdx.x * 64 + lane);
    const int64_t C = (int64_t)a.B * a.H;
    const int seg = blockIdx.y, tile0 = seg * a.seg_tiles, tile1 = tile0 + a.seg_tiles < a.tiles ? tile0 + a.seg_tiles : a.tiles;
    const T* gi = (const T*)a.gi + me.b * a.gsb + me.k;
    T* out = AGG ? nullptr : (T*)a.out + me.b * a.osb + me.k;
    Chan<VW> h = zeros<VW>(), At;
    if (AGG) {
#pragma unroll
        for (int j = 0; j < VW; ++j) At.v[j] = 1.f;
    } else if (me.on) {
        const float* from = a.segs > 1 ? a.ws + (int64_t)(2 * seg + 1) * C : a.h0;
        if (from) h = load_ch<float, VW>(from + me.c);
    }
    for (int tile = tile0; tile < tile1; ++tile) {
        const int s0 = (tile * waves + wave) * LSTEP;
        Chan<VW> z[LSTEP], ux[LSTEP];
#pragma unroll
        for (int i = 0; i < LSTEP; ++i) {
            const int t = position(a, s0 + i);
            z[i] = ux[i] = zeros<VW>();
            if (s0 + i < a.T && t < me.len) {
                z[i] = load_ch<T, VW>(gi + t * a.gst);
                ux[i] = load_ch<T, VW>(gi + t * a.gst + a.H);
            }
        }
        if (!AGG && a.tape && wave == 0 && me.on) store_ch<float, VW>(a.tape + (int64_t)tile * C + me.c, h);
        Chan<VW> A, b = zeros<VW>();
#pragma unroll
        for (int j = 0; j < VW; ++j) A.v[j] = 1.f;
#pragma unroll
        for (int i = 0; i < LSTEP; ++i) {
            const bool real = s0 + i < a.T && position(a, s0 + i) < me.len;
#pragma unroll
            for (int j = 0; j < VW; ++j) {
                float zz, u;
                gate(z[i].v[j], zz, u);
                z[i].v[j] = real ? zz : 1.f;
                ux[i].v[j] = real ? u * ux[i].v[j] : 0.f;
                A.v[j] *= z[i].v[j];
                b.v[j] = fmaf(z[i].v[j], b.v[j], ux[i].v[j]);
            }
        }
        Chan<VW> hs = h;                                           // the state in front of this wave's steps
        if (waves > 1) {
            const int buf = tile & 1;
            sA[buf][wave][lane] = A;
            sB[buf][wave][lane] = b;
            __syncthreads();
            for (int w = 0; w < waves; ++w) {
                const Chan<VW> Aw = sA[buf][w][lane], bw = sB[buf][w][lane];
#pragma unroll
                for (int j = 0; j < VW; ++j) {
                    if (w == wave) hs.v[j] = h.v[j];
                    h.v[j] = fmaf(Aw.v[j], h.v[j], bw.v[j]);
                    if (AGG) At.v[j] *= Aw.v[j];
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < VW; ++j) {
                h.v[j] = fmaf(A.v[j], h.v[j], b.v[j]);
                if (AGG) At.v[j] *= A.v[j];
            }
        }
        if (AGG) continue;
#pragma unroll
        for (int i = 0; i < LSTEP; ++i) {
            const int t = position(a, s0 + i);
            Chan<VW> o;
#pragma unroll
            for (int j = 0; j < VW; ++j) {
                hs.v[j] = fmaf(z[i].v[j], hs.v[j], ux[i].v[j]);
                o.v[j] = t < me.len ? hs.v[j] : 0.f;
            }
            if (s0 + i < a.T && me.on) store_ch<T, VW>(out + t * a.ost, o);
        }
    }
    if (wave != 0 || !me.on) return;
    if (AGG) {
        store_ch<float, VW>(a.ws + (int64_t)(2 * seg) * C + me.c, At);
        store_ch<float, VW>(a.ws + (int64_t)(2 * seg + 1) * C + me.c, h);
    } else if (a.hT && seg == a.segs - 1) {
        store_ch<float, VW>(a.hT + me.c, h);
    }
}

// Folds the segments' (A, b): b of segment s becomes the state in front of it.  Backward: from the last segment to the first.
template <bool BWD>
__global__ __launch_bounds__(64) void scan_carry_kernel(float* __restrict__ ws, const float* __restrict__ first, int64_t C, int segs) {
    const int64_t c = (int64_t)blockIdx.x * 64 + threadIdx.x;
    if (c >= C) return;
    float h = first ? first[c] : 0.f;
    constexpr int AHEAD = 16;                                      // loads in flight; only the products wait for one another
    for (int i0 = 0; i0 < segs; i0 += AHEAD) {
        float A[AHEAD], b[AHEAD];
#pragma unroll
        for (int q = 0; q < AHEAD; ++q) {
            const int i = i0 + q < segs ? i0 + q : segs - 1;
            const int64_t at = (int64_t)(2 * (BWD ? segs - 1 - i : i)) * C + c;
            A[q] = ws[at];
            b[q] = ws[at + C];
        }
#pragma unroll
        for (int q = 0; q < AHEAD; ++q)
            if (i0 + q < segs) {
                ws[(int64_t)(2 * (BWD ? segs - 1 - i0 - q : i0 + q)) * C + c + C] = h;
                h = fmaf(A[q], h, b[q]);
            }
    }
}

// at most 128 registers: four waves per SIMD, two blocks per CU (131 without the bound: one)
template <typename T, int VW, bool AGG>
__global__ __launch_bounds__(64 * MAXW, 4) void scan_bwd_kernel(ScanArgs a) {
    __shared__ Chan<VW> sA[2][MAXW][64], sB[2][MAXW][64], sD[2][MAXW][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = a.waves;
    const Lane<VW> me(a, (int64_t)blockIdx.x * 64 + lane);
    const int64_t C = (int64_t)a.B * a.H;
    const int seg = blockIdx.y, tile0 = seg * a.seg_tiles, tile1 = tile0 + a.seg_tiles < a.tiles ? tile0 + a.seg_tiles : a.tiles;
    const T* gi = (const T*)a.gi + me.b * a.gsb + me.k;
    const T* dout = a.dout ? (const T*)a.dout + me.b * a.dsb + me.k : nullptr;
    T* dgi = AGG ? nullptr : (T*)a.dgi + me.b * a.qsb + me.k;
    Chan<VW> g = zeros<VW>(), At;                                  // g: z_{t+1} g_{t+1} behind the current tile
    if (AGG) {
#pragma unroll
        for (int j = 0; j < VW; ++j) At.v[j] = 1.f;
    } else if (me.on) {
        const float* from = a.segs > 1 ? a.ws + (int64_t)(2 * seg + 1) * C : a.dhT;
        if (from) g = load_ch<float, VW>(from + me.c);
    }
    for (int tile = tile1 - 1; tile >= tile0; --tile) {
        const int s0 = (tile * waves + wave) * LSTEP;
        laed_vec<T, VW> f[LSTEP], x[LSTEP], d[LSTEP];
        Chan<VW> hs = zeros<VW>();
#pragma unroll
        for (int i = 0; i < LSTEP; ++i) {
            const int t = position(a, s0 + i);
            f[i] = x[i] = d[i] = laed_vec<T, VW>();
            if (s0 + i < a.T && t < me.len) {
                f[i] = *reinterpret_cast<const laed_vec<T, VW>*>(gi + t * a.gst);
                if (!AGG) x[i] = *reinterpret_cast<const laed_vec<T, VW>*>(gi + t * a.gst + a.H);
                if (dout) d[i] = *reinterpret_cast<const laed_vec<T, VW>*>(dout + t * a.dst);
            }
        }
        if (!AGG && me.on) hs = load_ch<float, VW>(a.tape + (int64_t)tile * C + me.c);
        Chan<VW> sg[LSTEP], A, b = zeros<VW>(), q = zeros<VW>();
#pragma unroll
        for (int j = 0; j < VW; ++j) A.v[j] = 1.f;
#pragma unroll
        for (int i = 0; i < LSTEP; ++i) {
            const bool real = s0 + i < a.T && position(a, s0 + i) < me.len;
#pragma unroll
            for (int j = 0; j < VW; ++j) {
                float z, u;
                sg[i].v[j] = real ? signed_gate(laed_to_float(f[i].v[j])) : 0.f;
                gates_of(sg[i].v[j], z, u);
                A.v[j] *= z;
                if (!AGG) b.v[j] = fmaf(z, b.v[j], u * laed_to_float(x[i].v[j]));
            }
        }
#pragma unroll
        for (int i = LSTEP - 1; i >= 0; --i)
#pragma unroll
            for (int j = 0; j < VW; ++j) {
                float z, u;
                gates_of(sg[i].v[j], z, u);
                q.v[j] = z * (laed_to_float(d[i].v[j]) + q.v[j]);
            }
        Chan<VW> gs = g;
        if (waves > 1) {
            const int buf = tile & 1;
            sA[buf][wave][lane] = A;
            sD[buf][wave][lane] = q;
            if (!AGG) sB[buf][wave][lane] = b;
            __syncthreads();
            if (!AGG)
                for (int w = 0; w < wave; ++w) {
                    const Chan<VW> Aw = sA[buf][w][lane], bw = sB[buf][w][lane];
#pragma unroll
                    for (int j = 0; j < VW; ++j) hs.v[j] = fmaf(Aw.v[j], hs.v[j], bw.v[j]);
                }
            for (int w = waves - 1; w >= 0; --w) {
                const Chan<VW> Aw = sA[buf][w][lane], qw = sD[buf][w][lane];
#pragma unroll
                for (int j = 0; j < VW; ++j) {
                    if (w == wave) gs.v[j] = g.v[j];
                    g.v[j] = fmaf(Aw.v[j], g.v[j], qw.v[j]);
                    if (AGG) At.v[j] *= Aw.v[j];
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < VW; ++j) {
                g.v[j] = fmaf(A.v[j], g.v[j], q.v[j]);
                if (AGG) At.v[j] *= A.v[j];
            }
        }
        if (AGG) continue;
        Chan<VW> e[LSTEP];                                         // h_{t-1} - x_t
#pragma unroll
        for (int i = 0; i < LSTEP; ++i)
#pragma unroll
            for (int j = 0; j < VW; ++j) {
                float z, u;
                gates_of(sg[i].v[j], z, u);
                const float xv = laed_to_float(x[i].v[j]);
                e[i].v[j] = hs.v[j] - xv;
                hs.v[j] = fmaf(z, hs.v[j], u * xv);
            }
#pragma unroll
        for (int i = LSTEP - 1; i >= 0; --i) {
            const int t = position(a, s0 + i);
            Chan<VW> df, dx;
#pragma unroll
            for (int j = 0; j < VW; ++j) {
                float z, u;
                gates_of(sg[i].v[j], z, u);
                const float at = gs.v[j] + laed_to_float(d[i].v[j]);
                dx.v[j] = u * at;
                df.v[j] = dx.v[j] * (e[i].v[j] * z);
                gs.v[j] = z * at;
                if (t >= me.len) { dx.v[j] = 0.f; df.v[j] = 0.f; }
            }
            if (s0 + i < a.T && me.on) {
                store_ch<T, VW>(dgi + t * a.qst, df);
                store_ch<T, VW>(dgi + t * a.qst + a.H, dx);
            }
        }
    }
    if (wave != 0 || !me.on) return;
    if (AGG) {
        store_ch<float, VW>(a.ws + (int64_t)(2 * seg) * C + me.c, At);
        store_ch<float, VW>(a.ws + (int64_t)(2 * seg + 1) * C + me.c, g);
    } else if (a.dh0 && seg == 0) {
        store_ch<float, VW>(a.dh0 + me.c, g);
    }
}

// Channels per lane: 8 bytes of the type forward, two channels backward (registers), where every row of every tensor starts
// on such a boundary; one channel otherwise.
bool rows_on(const void* p, int64_t st, int64_t sb, int vw, int es) {
    return ((uintptr_t)p % (vw * es)) == 0 && st % vw == 0 && sb % vw == 0;
}

template <typename T, int VW>
void launch_fwd(const ScanArgs& a, hipStream_t stream) {
    const int64_t C = (int64_t)a.B * a.H;
    const unsigned strips = (unsigned)cdiv64(C, 64 * VW);
    const dim3 block(64 * a.waves);
    if (a.segs > 1) {
        hipLaunchKernelGGL((scan_fwd_kernel<T, VW, true>), dim3(strips, a.segs), block, 0, stream, a);
        hipLaunchKernelGGL((scan_carry_kernel<false>), dim3((unsigned)cdiv64(C, 64)), dim3(64), 0, stream, a.ws, a.h0, C, a.segs);
    }
    hipLaunchKernelGGL((scan_fwd_kernel<T, VW, false>), dim3(strips, a.segs), block, 0, stream, a);
}
template <typename T, int VW>
void launch_bwd(const ScanArgs& a, hipStream_t stream) {
    const int64_t C = (int64_t)a.B * a.H;
    const unsigned strips = (unsigned)cdiv64(C, 64 * VW);
    const dim3 block(64 * a.waves);
    if (a.segs > 1) {
        hipLaunchKernelGGL((scan_bwd_kernel<T, VW, true>), dim3(strips, a.segs), block, 0, stream, a);
        hipLaunchKernelGGL((scan_carry_kernel<true>), dim3((unsigned)cdiv64(C, 64)), dim3(64), 0, stream, a.ws, a.dhT, C, a.segs);
    }
    hipLaunchKernelGGL((scan_bwd_kernel<T, VW, false>), dim3(strips, a.segs), block, 0, stream, a);
}

// A grid holds fewer than 2^32 threads, 64 of them per strip and wave: more sequences than that go in several launches, each with
// a tape of its own.  (A strip's number as an argument of the kernel instead: 431 us for 398 in the forward pass of
// 4096 x 40 x 1024 fp32, from the same registers.)
template <typename T, typename F>
void over_sequences(const ScanArgs& a, F launch) {
    const int64_t fit = (1ll << 31) / a.waves / a.H, most = fit > 1 ? fit : 1;
    for (int64_t b0 = 0; b0 < a.B; b0 += most) {
        ScanArgs p = a;
        p.B = (int)(a.B - b0 < most ? a.B - b0 : most);
        const int64_t c0 = b0 * a.H;
        const auto states = [&](auto q) { return q ? q + c0 : q; };
        p.gi = (const T*)a.gi + b0 * a.gsb;
        p.h0 = states(a.h0); p.hT = states(a.hT); p.dhT = states(a.dhT); p.dh0 = states(a.dh0);
        p.lengths = a.lengths ? a.lengths + b0 : nullptr;
        p.tape = a.tape ? a.tape + c0 * a.tiles : nullptr;
        p.out = a.out ? (T*)a.out + b0 * a.osb : nullptr;
        p.dout = a.dout ? (const T*)a.dout + b0 * a.dsb : nullptr;
        p.dgi = a.dgi ? (T*)a.dgi + b0 * a.qsb : nullptr;
        launch(p);
    }
}

template <typename T>
void dispatch(const ScanArgs& a, bool bwd, hipStream_t stream) {
    constexpr int es = sizeof(T), wide = 8 / sizeof(T), narrow = 2;
    auto ok = [&](int vw) {
        return a.H % vw == 0 && rows_on(a.gi, a.gst, a.gsb, vw, es) &&
               (bwd ? rows_on(a.dgi, a.qst, a.qsb, vw, es) && (!a.dout || rows_on(a.dout, a.dst, a.dsb, vw, es))
                    : rows_on(a.out, a.ost, a.osb, vw, es)) &&
               ((uintptr_t)a.h0 | (uintptr_t)a.hT | (uintptr_t)a.tape | (uintptr_t)a.dhT | (uintptr_t)a.dh0 | (uintptr_t)a.ws) % (vw * 4) == 0;
    };
    const bool vectors = bwd ? ok(narrow) : ok(wide);
    over_sequences<T>(a, [&](const ScanArgs& p) {
        if (vectors) bwd ? launch_bwd<T, narrow>(p, stream) : launch_fwd<T, wide>(p, stream);
        else bwd ? launch_bwd<T, 1>(p, stream) : launch_fwd<T, 1>(p, stream);
    });
}

int scan_args(ScanArgs& a, const char* what, const void* gi, int64_t gst, int64_t gsb, const int64_t* lengths, int T, int B, int H,
              int dtype, int reverse, float* ws, int64_t ws_floats) {
    LAED_CHECK_ARG(dtype >= LAED_F32 && dtype <= LAED_F16, "%s: unknown dtype %d", what, dtype);
    LAED_CHECK_ARG(cdiv64((int64_t)B * H, 64) <= INT32_MAX, "%s: B * H too large", what);
    LAED_CHECK_ARG(T <= INT32_MAX - 64, "%s: T too large", what);
    const ScanPlan p = scan_plan(T, B, H);
    LAED_CHECK_ARG((int64_t)H * p.waves <= (1ll << 31), "%s: H too large", what);      // one sequence's threads fit a grid
    LAED_CHECK_ARG(p.segs == 1 || (ws && ws_floats >= laed_gated_scan_workspace(T, B, H)), "%s: workspace too small", what);
    a.gi = gi; a.gst = gst; a.gsb = B > 1 ? gsb : 0; a.lengths = lengths; a.T = T; a.B = B; a.H = H; a.reverse = reverse;
    a.waves = p.waves; a.tiles = p.tiles; a.segs = p.segs; a.seg_tiles = p.seg_tiles; a.ws = ws;
    return 0;
}

}   // namespace

extern "C" int64_t laed_gated_scan_tape(int T, int B, int H) {
    if (T <= 0 || B <= 0 || H <= 0) return 0;
    return (int64_t)scan_plan(T, B, H).tiles * B * H;
}

extern "C" int64_t laed_gated_scan_workspace(int T, int B, int H) {
    if (T <= 0 || B <= 0 || H <= 0) return 0;
    const ScanPlan p = scan_plan(T, B, H);
    return p.segs > 1 ? (int64_t)2 * p.segs * B * H : 0;
}

extern "C" int laed_gated_scan_fwd(const void* gi, int64_t gi_st, int64_t gi_sb, const float* h0, const int64_t* lengths,
                                   int T, int B, int H, int dtype, int reverse, void* out, int64_t out_st, int64_t out_sb,
                                   float* hT, float* tape, float* ws, int64_t ws_floats, void* stream) {
    ScanArgs a = {};
    LAED_CHECK_ARG(T >= 0 && B >= 0 && H >= 0, "gated_scan_fwd: negative dimension");
    if (B == 0 || H == 0) return 0;
    LAED_TRY(scan_args(a, "gated_scan_fwd", gi, gi_st, gi_sb, lengths, T, B, H, dtype, reverse, ws, ws_floats));
    LAED_CHECK_ARG(T == 0 || (gi && out), "gated_scan_fwd: null pointer");
    a.h0 = h0; a.out = out; a.ost = out_st; a.osb = B > 1 ? out_sb : 0; a.hT = hT; a.tape = T > 0 ? tape : nullptr;
#define LAUNCH(T_) dispatch<T_>(a, false, (hipStream_t)stream)
    LAED_BY_DTYPE(dtype, LAUNCH);
#undef LAUNCH
    LAED_LAUNCH_CHECK("gated_scan_fwd");
    return 0;
}

extern "C" int laed_gated_scan_bwd(const void* gi, int64_t gi_st, int64_t gi_sb, const float* tape, const int64_t* lengths,
                                   const void* dout, int64_t dout_st, int64_t dout_sb, const float* dhT, int T, int B, int H,
                                   int dtype, int reverse, void* dgi, int64_t dgi_st, int64_t dgi_sb, float* dh0,
                                   float* ws, int64_t ws_floats, void* stream) {
    ScanArgs a = {};
    LAED_CHECK_ARG(T >= 0 && B >= 0 && H >= 0, "gated_scan_bwd: negative dimension");
    if (B == 0 || H == 0) return 0;
    LAED_TRY(scan_args(a, "gated_scan_bwd", gi, gi_st, gi_sb, lengths, T, B, H, dtype, reverse, ws, ws_floats));
    LAED_CHECK_ARG(T == 0 || (gi && tape && dgi), "gated_scan_bwd: null pointer");
    a.tape = (float*)tape; a.dout = dout; a.dst = dout_st; a.dsb = B > 1 ? dout_sb : 0; a.dhT = dhT;
    a.dgi = dgi; a.qst = dgi_st; a.qsb = B > 1 ? dgi_sb : 0;
    a.dh0 = dh0;
    if (T == 0) a.tiles = 0;
#define LAUNCH(T_) dispatch<T_>(a, true, (hipStream_t)stream)
    LAED_BY_DTYPE(dtype, LAUNCH);
#undef LAUNCH
    LAED_LAUNCH_CHECK("gated_scan_bwd");
    return 0;
}
