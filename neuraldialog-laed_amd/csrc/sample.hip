// One token per row from logits under temperature, top-k, top-p and min-p, from a given (or generated) uniform number.
//   y_i = (l_i - max l) / tau, w_i = e^{y_i}; rank by (l descending, index ascending)
//   top-k keeps ranks < k; top-p keeps, of those, the tokens in front of which less than p of their mass lies (the first one
//   always); min-p keeps w_i >= min_p.  The token drawn is the first one IN VOCABULARY ORDER whose cumulative kept weight
//   exceeds u * total.  -inf and NaN are masked; a row with nothing left gives -1.
// Weights are 64-bit fixed-point numbers (w 2^fb, fb = 62 - ceil(log2 V), at most 46), computed in 64-bit floating point
// and rounded once: sums are exact, so neither the order of the atomics nor the split over threads changes a result, and a
// border is off by at most V 2^-fb-1 of the largest weight -- a fp32 sum over a vocabulary would put a draw on the wrong
// side of a border once in a few hundred rows.
#include "laed_dtypes.h"
#include <math.h>

typedef unsigned long long u64;

namespace {

constexpr int NBINS = 2048;
constexpr int CAP = 1024;                 // candidates ranked in LDS
constexpr int MAXW = 16;                  // waves per block

struct SampleArgs {
    const void* logits;
    int64_t ld, N;
    int V, fb;
    const float* u;
    uint64_t seed, offset;
    double temperature; const float* temperature_rows;
    int64_t top_k; const int64_t* top_k_rows;
    double top_p; const float* top_p_rows;
    double min_p; const float* min_p_rows;
    int64_t* ids;
    float* logp;
};

struct Shared {
    u64 hist[NBINS];
    u64 cw[CAP];
    unsigned ckey[CAP];
    int cidx[CAP];
    u64 wsum[MAXW];
    float wmax[MAXW];
    unsigned kmin, kmax, n;
    int bin, result;
    u64 acc, last, total;
};

// ordered image of a float: larger value, larger key (l + 0.0f has turned -0 into 0; NaN never comes here)
__device__ __forceinline__ unsigned key_of(float l) {
    const unsigned b = __float_as_uint(l);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float value_of(unsigned k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }

// what a row's passes need
struct Row {
    float m;                              // largest logit
    double c2;                            // log2(e) / tau
    double cut2;                          // log2(min_p): keep y2 >= cut2
    float bins;                           // linear bins per unit of logit
    int fb;
    unsigned tkey;                        // kept: key > tkey, or key == tkey and index <= tidx
    int tidx;

    __device__ __forceinline__ double y2(float l) const { return l == m ? 0.0 : ((double)l - (double)m) * c2; }
    // 2^y2 as a fixed-point number with fb binary places.  2^f on [-1/2, 1/2] by the series of e^{f ln 2} up to the 12th
    // power (remainder below 2^-52), adding 2^52 rounds to an integer in the low bits of the mantissa.
    __device__ __forceinline__ u64 weight(float l) const {
        const double y = y2(l);
        if (!(y > -(double)(fb + 2))) return 0;
        const double n = rint(y), f = (y - n) * 0.693147180559945309417;
        double p = 1.0 / 479001600.0;
        p = fma(p, f, 1.0 / 39916800.0);
        p = fma(p, f, 1.0 / 3628800.0);
        p = fma(p, f, 1.0 / 362880.0);
        p = fma(p, f, 1.0 / 40320.0);
        p = fma(p, f, 1.0 / 5040.0);
        p = fma(p, f, 1.0 / 720.0);
        p = fma(p, f, 1.0 / 120.0);
        p = fma(p, f, 1.0 / 24.0);
        p = fma(p, f, 1.0 / 6.0);
        p = fma(p, f, 0.5);
        p = fma(p, f, 1.0);
        p = fma(p, f, 1.0);
        p = ldexp(p, (int)n + fb) + 4503599627370496.0;
        return (u64)__double_as_longlong(p) & 0x000fffffffffffffull;
    }
    __device__ __forceinline__ int bin(float l) const {
        const float d = l == m ? 0.f : m - l;
        return (int)fminf(d * bins, (float)(NBINS - 1));
    }
    __device__ __forceinline__ bool kept(float l, int i) const {
        const unsigned k = key_of(l);
        return l > -INFINITY && (k > tkey || (k == tkey && i <= tidx));
    }
};

__device__ __forceinline__ u64 wave_sum64(u64 v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
__device__ __forceinline__ u64 wave_scan64(u64 v, int lane) {      // inclusive
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const u64 t = __shfl_up(v, o, 64);
        if (lane >= o) v += t;
    }
    return v;
}

// The row's elements in vocabulary order: 16-byte vectors from the aligned address at or below the row's start (vectors that
// stick out of the row are read element by element); wave w walks a contiguous stretch of them.  Elements outside the row
// come as -inf.
template <typename T>
struct Walk {
    static constexpr int VW = 16 / sizeof(T);
    const T* p;
    int V, shift, nvec, per_wave;
    __device__ __forceinline__ Walk(const T* row, int V_, int waves) : V(V_) {
        shift = (int)(((uintptr_t)row & 15) / sizeof(T));
        p = row - shift;
        nvec = (V + shift + VW - 1) / VW;
        per_wave = ((nvec + waves - 1) / waves + 63) / 64 * 64;
    }
    __device__ __forceinline__ void load(int vec, float (&l)[VW]) const {
        const int first = vec * VW - shift;
        if (first >= 0 && first + VW <= V) {
            const laed_vec<T, VW> v = *reinterpret_cast<const laed_vec<T, VW>*>(p + (int64_t)vec * VW);
#pragma unroll
            for (int e = 0; e < VW; ++e) l[e] = laed_to_float(v.v[e]);
        } else {
#pragma unroll
            for (int e = 0; e < VW; ++e)
                l[e] = (first + e >= 0 && first + e < V) ? laed_to_float(p[vec * VW + e]) : -INFINITY;
        }
#pragma unroll
        for (int e = 0; e < VW; ++e) l[e] = l[e] > -INFINITY ? l[e] + 0.0f : -INFINITY;       // NaN is masked, -0 becomes 0
    }
    // f(index, logit) for this thread's elements
    template <typename F> __device__ __forceinline__ void each(int wave, int lane, F f) const {
        for (int j = 0; j < per_wave; j += 64) {
            const int vec = wave * per_wave + j + lane;
            if (vec >= nvec) break;
            float l[VW];
            load(vec, l);
#pragma unroll
            for (int e = 0; e < VW; ++e) f(vec * VW - shift + e, l[e]);
        }
    }
};

// Bins [0, NBINS) hold weights, best first: finds the first bin at which base + cumulative weight reaches `want` and puts
// (bin, weight in front of it) into shared memory; bin = -1 if the whole is less than `want`.
__device__ __forceinline__ void find_bin(Shared& sh, u64 base, u64 want, int tid, int lane, int wave, int nt) {
    const int per = NBINS / nt;
    if (tid == 0) sh.bin = -1;
    u64 mine = 0;
    for (int i = 0; i < per; ++i) mine += sh.hist[tid * per + i];
    const u64 inc = wave_scan64(mine, lane);
    if (lane == 63) sh.wsum[wave] = inc;
    __syncthreads();
    u64 front = base + inc - mine;
    for (int w = 0; w < wave; ++w) front += sh.wsum[w];
    if (front < want && front + mine >= want) {                    // exactly one thread
        for (int i = 0; i < per; ++i) {
            const u64 v = sh.hist[tid * per + i];
            if (front + v >= want) { sh.bin = tid * per + i; sh.acc = front; break; }
            front += v;
        }
    }
    __syncthreads();
}

// First element in vocabulary order at which the cumulative weight exceeds `target`; its index in sh.result (-1: none).
template <typename T, typename W>
__device__ __forceinline__ void locate(Shared& sh, const Walk<T>& walk, u64 target, int tid, int lane, int wave, int waves, W weight) {
    u64 mine = 0;
    walk.each(wave, lane, [&](int i, float l) { mine += weight(i, l); });
    mine = wave_sum64(mine);
    if (tid == 0) sh.result = -1;
    if (lane == 0) sh.wsum[wave] = mine;
    __syncthreads();
    u64 front = 0;
    for (int w = 0; w < wave; ++w) front += sh.wsum[w];
    if (front <= target && front + mine > target) {                // exactly one wave
        for (int j = 0; j < walk.per_wave; j += 64) {              // wave-uniform
            const int vec = wave * walk.per_wave + j + lane;
            float l[Walk<T>::VW];
            u64 v = 0;
            if (vec < walk.nvec) {
                walk.load(vec, l);
                for (int e = 0; e < Walk<T>::VW; ++e) v += weight(vec * Walk<T>::VW - walk.shift + e, l[e]);
            }
            const u64 inc = wave_scan64(v, lane), all = __shfl(inc, 63, 64);
            if (front + all > target) {
                u64 at = front + inc - v;
                if (at <= target && at + v > target) {             // exactly one lane
                    for (int e = 0; e < Walk<T>::VW; ++e) {
                        at += weight(vec * Walk<T>::VW - walk.shift + e, l[e]);
                        if (at > target) { sh.result = vec * Walk<T>::VW - walk.shift + e; break; }
                    }
                }
                break;
            }
            front += all;
        }
    }
    __syncthreads();
}

// Narrows (row.tkey, row.tidx) to the last element in rank order in front of which less than `want` lies -- elements counted
// (MASS = false) or their weights.  A histogram over linear bins of the logit finds the bin that holds it; the bin's
// elements are ranked in LDS, and if they are too many the bin is divided by its own range of values until they fit or are
// all equal; equal ones are taken in vocabulary order.
template <bool MASS, typename T>
__device__ void narrow(Shared& sh, Row& row, const Walk<T>& walk, u64 want, int tid, int lane, int wave, int waves, int nt) {
    for (int i = tid; i < NBINS; i += nt) sh.hist[i] = 0;
    __syncthreads();
    walk.each(wave, lane, [&](int i, float l) {
        if (!row.kept(l, i)) return;
        const u64 w = MASS ? row.weight(l) : 1;
        if (w) atomicAdd(&sh.hist[row.bin(l)], w);
    });
    __syncthreads();
    find_bin(sh, 0, want, tid, lane, wave, nt);
    if (sh.bin < 0) return;                                        // less than `want` in all: everything stays
    const int bin = sh.bin;
    u64 acc = sh.acc;
    unsigned klo = 0, khi = 0xffffffffu;
    for (;;) {                                                     // at most 4 turns: a turn divides the range by 2048
        __syncthreads();
        if (tid == 0) { sh.n = 0; sh.kmin = 0xffffffffu; sh.kmax = 0; sh.last = 0; }
        __syncthreads();
        unsigned kmin = 0xffffffffu, kmax = 0;
        walk.each(wave, lane, [&](int i, float l) {
            if (!row.kept(l, i) || row.bin(l) != bin) return;
            const unsigned k = key_of(l);
            if (k < klo || k > khi) return;
            kmin = k < kmin ? k : kmin;
            kmax = k > kmax ? k : kmax;
            const unsigned at = atomicAdd(&sh.n, 1u);
            if (at < CAP) { sh.ckey[at] = k; sh.cidx[at] = i; sh.cw[at] = MASS ? row.weight(l) : 1; }
        });
        if (kmax >= kmin) { atomicMin(&sh.kmin, kmin); atomicMax(&sh.kmax, kmax); }
        __syncthreads();
        const unsigned n = sh.n;
        kmin = sh.kmin; kmax = sh.kmax;
        if (n <= CAP) {
            for (unsigned i = tid; i < n; i += nt) {
                const unsigned k = sh.ckey[i];
                const int x = sh.cidx[i];
                u64 before = acc;
                for (unsigned j = 0; j < n; ++j)
                    before += (sh.ckey[j] > k || (sh.ckey[j] == k && sh.cidx[j] < x)) ? sh.cw[j] : 0;
                if (before < want) atomicMax(&sh.last, ((u64)~k << 32) | (unsigned)x);
            }
            __syncthreads();
            row.tkey = ~(unsigned)(sh.last >> 32);
            row.tidx = (int)(unsigned)sh.last;
            return;
        }
        if (kmin == kmax) {
            const u64 w = MASS ? row.weight(value_of(kmin)) : 1;   // > 0: the bin's weight crosses `want`
            const u64 r = (want - acc + w - 1) / w;                // that many of the equal ones stay
            if (r < n) {
                locate(sh, walk, r - 1, tid, lane, wave, waves,
                       [&](int i, float l) { return (u64)(row.kept(l, i) && key_of(l) == kmin); });
                row.tidx = sh.result;
            } else if (row.tkey != kmin) {
                row.tidx = 0x7fffffff;
            }
            row.tkey = kmin;
            return;
        }
        const unsigned range = kmax - kmin;
        const int bits = 32 - __clz(range), shift = bits > 11 ? bits - 11 : 0;
        for (int i = tid; i < NBINS; i += nt) sh.hist[i] = 0;
        __syncthreads();
        walk.each(wave, lane, [&](int i, float l) {
            if (!row.kept(l, i) || row.bin(l) != bin) return;
            const unsigned k = key_of(l);
            if (k < kmin || k > kmax) return;
            const u64 w = MASS ? row.weight(l) : 1;
            if (w) atomicAdd(&sh.hist[(kmax - k) >> shift], w);
        });
        __syncthreads();
        find_bin(sh, acc, want, tid, lane, wave, nt);
        acc = sh.acc;
        khi = kmax - ((unsigned)sh.bin << shift);
        const unsigned width = (1u << shift) - 1;
        klo = khi - kmin > width ? khi - width : kmin;
    }
}

// first version: one block per row, every pass reads the row again
template <typename T>
__global__ __launch_bounds__(1024) void sample_rows_kernel(SampleArgs a) {
    __shared__ Shared sh;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, nt = blockDim.x, waves = nt >> 6;
    for (int64_t r = blockIdx.x; r < a.N; r += gridDim.x) {
        __syncthreads();
        const Walk<T> walk((const T*)a.logits + r * a.ld, a.V, waves);
        Row row;
        float m = -INFINITY;
        walk.each(wave, lane, [&](int, float l) { m = fmaxf(m, l); });
        m = wave_max(m);
        if (lane == 0) sh.wmax[wave] = m;
        __syncthreads();
        for (int w = 0; w < waves; ++w) m = fmaxf(m, sh.wmax[w]);
        if (m == -INFINITY) {                                      // nothing to draw from
            if (tid == 0) { a.ids[r] = -1; if (a.logp) a.logp[r] = -INFINITY; }
            continue;
        }
        const double tau = a.temperature_rows ? (double)a.temperature_rows[r] : a.temperature;
        const int64_t k = a.top_k_rows ? a.top_k_rows[r] : a.top_k;
        const double p = a.top_p_rows ? (double)a.top_p_rows[r] : a.top_p;
        const double mp = a.min_p_rows ? (double)a.min_p_rows[r] : a.min_p;
        row.m = m;
        row.fb = a.fb;
        row.tkey = 0;
        row.tidx = 0x7fffffff;
        if (!(tau > 0.0)) {                                        // greedy: the first largest one
            locate(sh, walk, 0, tid, lane, wave, waves, [&](int, float l) { return (u64)(l == m); });
            if (tid == 0) { a.ids[r] = sh.result; if (a.logp) a.logp[r] = 0.f; }
            continue;
        }
        row.c2 = 1.4426950408889634074 / tau;
        row.bins = (float)fmin(64.0 / tau, 1e30);
        row.cut2 = mp > 0.0 ? log2(mp < 1.0 ? mp : 1.0) : -INFINITY;
        if (k > 0 && k < a.V) narrow<false>(sh, row, walk, (u64)k, tid, lane, wave, waves, nt);
        if (p < 1.0) {
            u64 mass = 0;
            walk.each(wave, lane, [&](int i, float l) { if (row.kept(l, i)) mass += row.weight(l); });
            mass = wave_sum64(mass);
            __syncthreads();
            if (lane == 0) sh.wsum[wave] = mass;
            __syncthreads();
            mass = 0;
            for (int w = 0; w < waves; ++w) mass += sh.wsum[w];
            __syncthreads();
            const double goal = ceil(p * (double)mass);            // in front of a kept token: less than p of the mass
            narrow<true>(sh, row, walk, goal > 1.0 ? (u64)goal : 1, tid, lane, wave, waves, nt);
        }
        auto drawn = [&](int i, float l) { return row.kept(l, i) && row.y2(l) >= row.cut2 ? row.weight(l) : (u64)0; };
        u64 total = 0;
        walk.each(wave, lane, [&](int i, float l) { total += drawn(i, l); });
        total = wave_sum64(total);
        __syncthreads();
        if (lane == 0) sh.wsum[wave] = total;
        __syncthreads();
        total = 0;
        for (int w = 0; w < waves; ++w) total += sh.wsum[w];
        __syncthreads();
        float u = a.u ? a.u[r] : uniform01(a.seed, a.offset + (uint64_t)r);
        u = u > 0.f ? (u < 1.f ? u : 0x1.fffffep-1f) : 0.f;
        const u64 target = __umul64hi((u64)(u * 0x1p64f), total);  // floor(u * total)
        locate(sh, walk, target, tid, lane, wave, waves, drawn);
        if (tid == 0) {
            const int id = sh.result;
            a.ids[r] = id;
            if (a.logp) {
                float l = laed_to_float(((const T*)a.logits + r * a.ld)[id]) + 0.0f;
                a.logp[r] = (float)((l == m ? 0.0 : ((double)l - (double)m) / tau) - (log((double)total) - a.fb * 0.693147180559945309417));
            }
        }
    }
}

}   // namespace

extern "C" int laed_sample_rows(const void* logits, int64_t ld, int64_t N, int V, int dtype, const float* u, uint64_t seed,
                                uint64_t offset, double temperature, const float* temperature_rows, int64_t top_k,
                                const int64_t* top_k_rows, double top_p, const float* top_p_rows, double min_p,
                                const float* min_p_rows, int64_t* ids, float* logp, void* stream) {
    LAED_CHECK_ARG(N >= 0 && V >= 1, "sample_rows: bad size");
    LAED_CHECK_ARG(dtype >= LAED_F32 && dtype <= LAED_F16, "sample_rows: unknown dtype %d", dtype);
    LAED_CHECK_ARG(V <= (1 << 28), "sample_rows: V must not exceed 2^28");
    LAED_CHECK_ARG(temperature_rows || temperature >= 0.0, "sample_rows: temperature must be >= 0 (0 = greedy)");
    LAED_CHECK_ARG(top_p_rows || (top_p >= 0.0 && top_p <= 1.0), "sample_rows: top_p must lie in [0, 1]");
    LAED_CHECK_ARG(min_p_rows || (min_p >= 0.0 && min_p <= 1.0), "sample_rows: min_p must lie in [0, 1]");
    if (N == 0) return 0;
    LAED_CHECK_ARG(logits && ids, "sample_rows: null pointer");
    int lg = 0;
    while ((1ll << lg) < V) ++lg;
    SampleArgs a = {logits, ld, N, V, 62 - lg < 46 ? 62 - lg : 46, u, seed, offset, temperature, temperature_rows, top_k, top_k_rows,
                    top_p, top_p_rows, min_p, min_p_rows, ids, logp};
    const unsigned grid = (unsigned)(N < (1 << 20) ? N : (1 << 20));
    const unsigned nt = V <= 4096 ? 256 : 1024;
#define LAUNCH(T) hipLaunchKernelGGL((sample_rows_kernel<T>), dim3(grid), dim3(nt), 0, (hipStream_t)stream, a)
    LAED_BY_DTYPE(dtype, LAUNCH);
#undef LAUNCH
    LAED_LAUNCH_CHECK("sample_rows");
    return 0;
}
