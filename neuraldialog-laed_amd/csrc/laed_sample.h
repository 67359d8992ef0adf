// One token per row from logits under temperature, top-k, top-p and min-p, from a given (or generated) uniform number.
//   y_i = (l_i - max l) / tau, w_i = e^{y_i}; rank by (l descending, index ascending)
//   top-k keeps ranks < k; top-p keeps, of those, the tokens in front of which less than p of their mass lies (the first one
//   always); min-p keeps w_i >= min_p.  The token drawn is the first one IN VOCABULARY ORDER whose cumulative kept weight
//   exceeds u * total.  -inf and NaN are masked; a row with nothing left gives -1.
// Weights are 64-bit fixed-point numbers (w 2^fb, fb = 62 - ceil(log2 V), at most 46): sums are exact, so neither the order
// of the atomics nor the split over threads changes a result.  A weight is off by 2^-35 of itself (the series below) and
// half a unit; over n kept tokens such errors move a border by about 2^-35 / sqrt(n) of the whole -- a fp32 sum over a
// vocabulary would put a draw on the wrong side of a border once in a few hundred rows.
//
// Bound by vector instructions: a row of 50000 is one CU's, and every instruction per element and pass costs 0.33 us.  4096 x 50000
// under top-p: 714 us, of 16 rows a CU one after the other -- reading 7 us, histogram of the weights 12, border 8, weights
// of the kept 8, token 5 (reading the row again in every pass: 2750 us).  64 x 50000 under all filters 40 us, one row of 10004 12 us.
#pragma once
#include "laed_dtypes.h"
#include <math.h>

typedef unsigned long long u64;

struct SampleArgs {
    const void* logits;
    int64_t ld, N;
    int64_t row0;                         // first row of this launch
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

// one translation unit per element type: each holds half a dozen large kernels
void laed_sample_launch_f32(const SampleArgs& a, hipStream_t stream);
void laed_sample_launch_bf16(const SampleArgs& a, hipStream_t stream);
void laed_sample_launch_f16(const SampleArgs& a, hipStream_t stream);

namespace {

constexpr int NBINS = 2048;
constexpr int CAP = 512;                  // candidates ranked in LDS
constexpr int FEW = 512;                  // a top-k up to this is finished among its tokens alone
constexpr int STEPS = 1024;               // table steps per octave
constexpr unsigned PER_BIN = 16;          // steps per bin
constexpr int FAR = 200 * STEPS;          // weights below 2^-200 are 0
constexpr int MAXW = 16;                  // waves per block
constexpr int QUEUE = 64 + 4 * 64;        // a wave's worth left over and four elements of every lane

// A token in an order: the larger `rank` goes first.
struct Entry { u64 rank, weight; };

struct Shared {
    double pow2[STEPS];                   // 2^(fb - i / STEPS)
    union {
        struct { u64 hist[NBINS]; Entry cand[CAP]; };
        float queue[MAXW][QUEUE];         // when the filters are done: logits that wait for their weight, by wave
    };
    u64 before[CAP];
    Entry few[FEW];                       // the tokens of a small top-k
    u64 wsum[MAXW];
    float wmax[MAXW];
    unsigned n, nfew;
    int bin, result;
    u64 acc, want, last, kmin, kmax;
};

// ordered image of a float: larger value, larger key (-0 has been turned into 0; NaN never comes here)
__device__ __forceinline__ unsigned key_of(float l) {
    const unsigned b = __float_as_uint(l);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float value_of(unsigned k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }

// `l` moved by a few floats, at most to an infinity
__device__ __forceinline__ float nudged(double l, int by) {
    const float f = (float)fmin(fmax(l, -3.4028234663852886e38), 3.4028234663852886e38) + 0.0f;
    const unsigned k = key_of(f) + by;
    return value_of(k < 0x007fffffu ? 0x007fffffu : (k > 0xff800000u ? 0xff800000u : k));
}

// 2^(-i / STEPS) by the series of e^{-i ln 2 / STEPS} up to the 16th power (remainder below 2^-57), once per block
__device__ __forceinline__ double pow2_step(int i) {
    const double x = i * (-0.693147180559945309417 / STEPS);
    double p = 1.0;
#pragma unroll
    for (int k = 16; k > 0; --k) p = fma(p * x, 1.0 / k, 1.0);
    return p;
}

// one value for the whole wave, kept in scalar registers: the passes' constants would be spilled as vector registers
__device__ __forceinline__ float uniform(float x) { return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(x))); }
__device__ __forceinline__ u64 uniform(u64 b) {
    const unsigned lo = (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)b), hi = (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)(b >> 32));
    return ((u64)hi << 32) | lo;
}
__device__ __forceinline__ double uniform(double x) { return __longlong_as_double((long long)uniform((u64)__double_as_longlong(x))); }

// what a row's passes need; all of it uniform
struct Row {
    const double* pow2;
    double md, c, per_step;               // largest logit, steps per unit of logit (STEPS log2(e) / tau) and 1 / c
    float m;
    double cut;                           // -STEPS log2(min_p)
    float tval;                           // kept: l > tval, or l == tval and index <= tidx
    int tidx;

    // steps below the largest one, 0 .. FAR (-inf and NaN: FAR)
    __device__ __forceinline__ double steps(float l) const { return fmin((md - (double)l) * c, (double)FAR); }
    // Adding 1.5 2^52 leaves the nearest whole number of steps in the low word: what bins and the table go by.
    static __device__ __forceinline__ unsigned whole(double y) { return (unsigned)__double_as_longlong(y + 6755399441055744.0); }
    // e^{(l - m) / tau} as a fixed-point number with fb binary places, y = steps(l).  With k whole steps and r = y - k:
    // 2^(-k / STEPS) from the table and the exponent, times 1 + q, q = e^{-r ln 2 / STEPS} - 1 <= 3.4e-4 to second order and in
    // fp32 -- a relative error of 2^-35 at most, another one in every element, where fp32 alone would leave 2^-22.  Adding 2^52
    // rounds to an integer in the low bits of the mantissa.  17 instructions; every one costs 0.33 us per pass over a
    // row of 50000 held by one CU (a series of 11 terms without the table: 30).
    __device__ __forceinline__ u64 weight(double y, int& k) const {
        const double t = y + 6755399441055744.0;
        k = (int)(unsigned)__double_as_longlong(t);
        const float r = (float)(y - (t - 6755399441055744.0));
        const float x = r * (float)(0.693147180559945309417 / STEPS), q = x * fmaf(x, 0.5f, -1.0f);
        const double w = pow2[k & (STEPS - 1)];
        const u64 bits = (u64)__double_as_longlong(fma(w, (double)q, w));
        unsigned hi = (unsigned)(bits >> 32) - ((unsigned)(k & ~(STEPS - 1)) << 10);
        asm volatile("" : "+v"(hi));                               // one 32-bit subtraction, not a 64-bit one
        const double p = __longlong_as_double((long long)(((u64)hi << 32) | (unsigned)bits)) + 4503599627370496.0;
        return (u64)__double_as_longlong(p) & 0x000fffffffffffffull;
    }
    __device__ __forceinline__ u64 weight(float l) const {
        int k;
        return weight(steps(l), k);
    }
    __device__ __forceinline__ bool kept(float l, int i) const { return (int)(l > tval) | ((int)(l == tval) & (int)(i <= tidx)); }
    // the weight it is drawn with: kept, and at most `cut` steps below the largest one
    __device__ __forceinline__ u64 drawn(float l, int i) const {
        const double y = steps(l);
        int k;
        const u64 v = weight(y, k);
        return ((int)kept(l, i) & (int)(y <= cut)) ? v : 0;
    }
};

// sum over the wave: inside rows of 16 lanes by DPP (no address registers to keep), across them by two shuffles
template <int O> __device__ __forceinline__ u64 row_add64(u64 v) {
    const unsigned lo = (unsigned)laed_bfly32_i<O>((int)(unsigned)v), hi = (unsigned)laed_bfly32_i<O>((int)(unsigned)(v >> 32));
    return v + (((u64)hi << 32) | lo);
}
__device__ __forceinline__ u64 wave_sum64(u64 v) {
    v = row_add64<1>(v);
    v = row_add64<2>(v);
    v = row_add64<4>(v);
    v = row_add64<8>(v);
    v += __shfl_xor(v, 16, 64);
    v += __shfl_xor(v, 32, 64);
    return v;
}
__device__ __forceinline__ u64 wave_scan64(u64 v, int lane) {      // inclusive
    asm volatile("" : "+v"(lane));                                 // its six masks are made here each time, not kept in between
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const u64 t = __shfl_up(v, o, 64);
        if (lane >= o) v += t;
    }
    return v;
}

// A row in vocabulary order: 16-byte vectors from the aligned address at or below its start (vectors that stick out of the
// row are read element by element); wave w walks a contiguous stretch of them, 64 at a time.  Elements outside the row and
// NaN come as -inf, -0 as 0.  A row whose maximum is +inf is walked as 0 where it is +inf and -inf elsewhere.
template <typename T>
struct Place {
    static constexpr int VW = 16 / sizeof(T);
    const T* p;
    int V, shift, nvec, turns, group, wave, lane;                  // turns: vectors per lane; group: a fourth of them, rounded up
    bool infinite;
    __device__ __forceinline__ Place(const T* row, int V_, int waves, int wave_, int lane_) : V(V_), wave(wave_), lane(lane_), infinite(false) {
        const u64 at = uniform((u64)(uintptr_t)row);               // a descriptor in vector registers would be read lane by lane
        shift = (int)((at & 15) / sizeof(T));
        p = (const T*)(uintptr_t)(at & ~15ull);
        nvec = (V + shift + VW - 1) / VW;
        turns = ((nvec + waves - 1) / waves + 63) / 64;
        group = (turns + 3) / 4;
    }
    __device__ __forceinline__ int vec_of(int j) const { return (wave * turns + j) * 64 + lane; }
    __device__ __forceinline__ int index_of(int vec, int e) const { return vec * VW - shift + e; }
    __device__ __forceinline__ float clean(float l) const {
        l = l > -INFINITY ? l + 0.0f : -INFINITY;
        return infinite ? (l == INFINITY ? 0.f : -INFINITY) : l;
    }
    __device__ __forceinline__ laed_vec<T, VW> raw(int vec) const {
        laed_vec<T, VW> v;
        const int first = vec * VW - shift;
        if (first >= 0 && first + VW <= V) {
            v = *reinterpret_cast<const laed_vec<T, VW>*>(p + (int64_t)vec * VW);
        } else {
#pragma unroll
            for (int e = 0; e < VW; ++e) v.v[e] = (first + e >= 0 && first + e < V) ? p[(int64_t)vec * VW + e] : (T)-INFINITY;
        }
        return v;
    }
};

// the row read from memory in every pass: any length
template <typename T>
struct Stream : Place<T> {
    using Place<T>::VW;
    __device__ __forceinline__ Stream(const T* row, int V_, int waves, int wave_, int lane_) : Place<T>(row, V_, waves, wave_, lane_) {}
    __device__ __forceinline__ float load() {                      // -> this thread's maximum
        float m = -INFINITY;
        each([&](int, float l) { m = fmaxf(m, l); });
        return m;
    }
    __device__ __forceinline__ void squash() { this->infinite = true; }
    // f(index, logit) for this thread's elements
    template <typename F> __device__ __forceinline__ void each(F f) {
        for (int j = 0; j < this->turns; ++j) {
            const int vec = this->vec_of(j);
            if (vec >= this->nvec) break;
            const laed_vec<T, VW> v = this->raw(vec);
#pragma unroll
            for (int e = 0; e < VW; ++e) f(this->index_of(vec, e), this->clean(laed_to_float(v.v[e])));
        }
    }
    template <typename W> __device__ __forceinline__ void sums(u64 (&sum)[4], W weight) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int end = this->group * (g + 1) < this->turns ? this->group * (g + 1) : this->turns;
            for (int j = this->group * g; j < end; ++j) {
                const int vec = this->vec_of(j);
                if (vec >= this->nvec) break;
                const laed_vec<T, VW> v = this->raw(vec);
#pragma unroll
                for (int e = 0; e < VW; ++e) sum[g] += weight(this->index_of(vec, e), this->clean(laed_to_float(v.v[e])));
            }
        }
    }
    __device__ __forceinline__ void kept_sums(u64 (&sum)[4], const Row& row, float*) {
        sums(sum, [&](int i, float l) { return row.drawn(l, i); });
    }
};

// the row held in registers, NV vectors per thread: read from memory once
template <typename T, int NV>
struct Held : Place<T> {
    using Place<T>::VW;
    laed_vec<T, VW> v[NV];
    static __device__ __forceinline__ unsigned (&words(laed_vec<T, VW>& x))[4] { return reinterpret_cast<unsigned (&)[4]>(x); }
    __device__ __forceinline__ Held(const T* row, int V_, int waves, int wave_, int lane_) : Place<T>(row, V_, waves, wave_, lane_) {
        this->group = (NV + 3) / 4;                                // known to the compiler
    }
    __device__ __forceinline__ float load() {
        // all loads first: the whole vectors through a buffer descriptor of exactly their bytes (one 32-bit offset each, 0 for
        // what lies outside), then the row's first and last vector, which may stick out of it, and -inf behind it
        const int whole0 = this->shift ? 1 : 0, whole1 = (this->V + this->shift) / VW, base = this->vec_of(0);
        const auto rows = __builtin_amdgcn_make_buffer_rsrc((void*)(uintptr_t)uniform((u64)(uintptr_t)(this->p + whole0 * VW)), 0,
                                                            __builtin_amdgcn_readfirstlane((whole1 > whole0 ? whole1 - whole0 : 0) * 16), 0x00027000);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const auto got = __builtin_amdgcn_raw_buffer_load_b128(rows, (base + 64 * j - whole0) * 16, 0, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i) words(v[j])[i] = got[i];
        }
        laed_vec<T, VW> head = this->raw(0), tail = this->raw(this->nvec - 1), none;
#pragma unroll
        for (int e = 0; e < VW; ++e) none.v[e] = (T)-INFINITY;
        float m = -INFINITY;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int vec = base + 64 * j;
            const bool first = vec < whole0, last = vec >= whole1, beyond = vec >= this->nvec || j >= this->turns;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                unsigned x = words(v[j])[i];
                x = last ? words(tail)[i] : x;
                x = first ? words(head)[i] : x;
                words(v[j])[i] = beyond ? words(none)[i] : x;
            }
#pragma unroll
            for (int e = 0; e < VW; ++e) {
                const float l = this->clean(laed_to_float(v[j].v[e]));
                v[j].v[e] = laed_from_float<T>(l);                 // the same number
                m = fmaxf(m, l);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        return m;
    }
    __device__ __forceinline__ void squash() {
        this->infinite = true;                                     // for what is read again
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < VW; ++e) v[j].v[e] = laed_from_float<T>(laed_to_float(v[j].v[e]) == INFINITY ? 0.f : -INFINITY);
    }
    // f(index, logit, group) for this thread's elements, done(group) behind each group (a fourth of NV vectors).  The empty asm
    // statements keep the compiler from carrying per-element results (bins, 64-bit copies) from one pass to the next: a
    // register or more per element, spilled, where recomputing costs a few instructions.
    template <typename F, typename D> __device__ __forceinline__ void each_in_group(F f, D done) {
        constexpr int G = (NV + 3) / 4;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
#pragma unroll
            for (int i = 0; i < 4; ++i) asm volatile("" : "+v"(words(v[j])[i]));
        }
        int base = this->index_of(this->vec_of(0), 0);
        asm volatile("" : "+v"(base));
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            if (j < this->turns) {
#pragma unroll
                for (int e = 0; e < VW; ++e) {
                    f(base + 64 * VW * j + e, laed_to_float(v[j].v[e]), j / G, e);
                    if (e & 1) __builtin_amdgcn_sched_barrier(0);          // two elements' weights in flight, not the whole row's
                }
            }
            if (j % G == G - 1 || j == NV - 1) done(j / G);
        }
    }
    template <typename F> __device__ __forceinline__ void each(F f) {
        each_in_group([&](int i, float l, int, int) { f(i, l); }, [](int) {});
    }
    template <typename W> __device__ __forceinline__ void sums(u64 (&sum)[4], W weight) {
        each_in_group([&](int i, float l, int g, int) { sum[g] += weight(i, l); }, [](int) {});
    }
    // sums of row.drawn.  The kept logits are few, and spread: they are packed into the wave's queue, whose 64 next ones are
    // weighed at a time, so that every lane weighs a kept one (packing costs 6 instructions an element, weighing 20).
    __device__ __forceinline__ void kept_sums(u64 (&sum)[4], const Row& row, float* queue) {
        int n = 0;                                                 // uniform
        u64 acc = 0;
        const auto weigh = [&](float l) {
            const double y = row.steps(l);
            int k;
            const u64 v = row.weight(y, k);
            return y <= row.cut ? v : 0;
        };
        each_in_group(
            [&](int i, float l, int, int e) {
                const bool keep = row.kept(l, i);
                const u64 mask = __ballot(keep);
                if (keep) queue[__builtin_amdgcn_mbcnt_hi((unsigned)(mask >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)mask, (unsigned)n))] = l;
                n += __popcll(mask);
                if (e % 4 == 3) {
                    // other lanes' entries of the same wave: the LDS takes a wave's accesses in order, the fences keep
                    // the compiler to it
                    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                    while (n >= 64) {
                        n -= 64;
                        acc += weigh(queue[n + this->lane]);
                    }
                    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                }
            },
            [&](int g) {                                           // what is left in the queue is this group's own
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                if (this->lane < n) acc += weigh(queue[this->lane]);
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                n = 0;
                sum[g] = acc;
                acc = 0;
            });
    }
};

struct Who { int tid, lane, wave, waves, nt; };

// Bins hold weights, best first: finds the first bin at which the cumulative weight reaches `want` -- or, with share >= 0,
// that share of the whole (rounded up, 1 at least) -- and leaves (bin, weight in front of it, want) in shared memory;
// bin = -1 if the whole is less than `want`.
__device__ __forceinline__ void find_bin(Shared& sh, const Who& w, u64 want, double share) {
    const int per = NBINS / w.nt;
    if (w.tid == 0) sh.bin = -1;
    u64 mine = 0;
    for (int i = 0; i < per; ++i) mine += sh.hist[w.tid * per + i];
    const u64 inc = wave_scan64(mine, w.lane);
    if (w.lane == 63) sh.wsum[w.wave] = inc;
    __syncthreads();
    u64 front = inc - mine, whole = 0;
    for (int i = 0; i < w.waves; ++i) {
        if (i < w.wave) front += sh.wsum[i];
        whole += sh.wsum[i];
    }
    if (share >= 0.0) {
        const double goal = ceil(share * (double)whole);
        want = goal > 1.0 ? (u64)goal : 1;
    }
    if (front < want && front + mine >= want) {                    // exactly one thread, if any
        for (int i = 0; i < per; ++i) {
            const u64 v = sh.hist[w.tid * per + i];
            if (front + v >= want) { sh.bin = w.tid * per + i; sh.acc = front; sh.want = want; break; }
            front += v;
        }
    }
    __syncthreads();
}

// First element in vocabulary order at which the cumulative weight exceeds share / 2^64 of the whole; its index in sh.result
// (-1: none).  -> the whole.  `sums`: this thread's part of the weight of each of the wave's four groups of vectors; the group
// that holds the element is read again.
template <typename R, typename W>
__device__ __forceinline__ u64 locate(Shared& sh, const Who& w, R& row, u64 (&sums)[4], u64 share, u64 fixed_target, W weight) {
    constexpr int VW = R::VW;
#pragma unroll
    for (int g = 0; g < 4; ++g) sums[g] = wave_sum64(sums[g]);
    __syncthreads();
    if (w.lane == 0) {
        sh.wsum[w.wave] = sums[0] + sums[1] + sums[2] + sums[3];
        if (w.wave == 0) sh.result = -1;
    }
    __syncthreads();
    u64 front = 0, whole = 0;
    for (int i = 0; i < w.waves; ++i) {
        if (i < w.wave) front += sh.wsum[i];
        whole += sh.wsum[i];
    }
    const u64 target = share ? __umul64hi(share, whole) : fixed_target;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        if (front <= target && front + sums[g] > target) {         // one group of one wave
            bool open = true;
            const int end = row.group * (g + 1) < row.turns ? row.group * (g + 1) : row.turns;
#pragma unroll 1
            for (int j0 = row.group * g; j0 < end && open; j0 += 4) {
                u64 v[4], all[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int vec = row.vec_of(j0 + q);
                    v[q] = 0;
                    if (j0 + q < end && vec < row.nvec) {
                        const auto x = row.raw(vec);
#pragma unroll
                        for (int e = 0; e < VW; ++e) v[q] += weight(row.index_of(vec, e), row.clean(laed_to_float(x.v[e])));
                    }
                }
#pragma unroll
                for (int q = 0; q < 4; ++q) all[q] = wave_sum64(v[q]);
                int hit = -1;
                u64 mine = 0;
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    if (open) {
                        if (front + all[q] > target) { open = false; hit = j0 + q; mine = v[q]; }
                        else front += all[q];
                    }
                if (open) continue;
                u64 at = front + wave_scan64(mine, w.lane) - mine;
                if (at <= target && at + mine > target) {          // exactly one lane
                    const int vec = row.vec_of(hit);
                    int found = -1;
#pragma unroll 1
                    for (int e = 0; e < VW && found < 0; ++e) {
                        const int i = row.index_of(vec, e);
                        if (i >= 0 && i < row.V) at += weight(i, row.clean(laed_to_float(row.p[(int64_t)vec * VW + e])));
                        if (at > target) found = i;
                    }
                    sh.result = found;
                }
            }
            break;
        }
        front += sums[g];
    }
    __syncthreads();
    return whole;
}

__device__ __forceinline__ u64 block_sum(Shared& sh, const Who& w, u64 mine) {
    mine = wave_sum64(mine);
    __syncthreads();
    if (w.lane == 0) sh.wsum[w.wave] = mine;
    __syncthreads();
    u64 all = 0;
    for (int i = 0; i < w.waves; ++i) all += sh.wsum[i];
    return all;
}

// More than CAP candidates in a bin (equal logits, or a tail that the linear bins do not reach): bisection over the ordered
// bit patterns between the bin's smallest and largest value, one pass each (at most 32), then the equal ones in vocabulary
// order.  Each pass costs what the histogram's does.  Rare in fp32; in 16 bits a long vocabulary's tail is full of equal
// logits (64 rows of 100000 bf16 under top-p 0.9: 197 us, 33 under a temperature alone).
template <bool MASS, typename R>
__device__ __forceinline__ void bisect(Shared& sh, const Who& w, Row& row, R& walk, u64 need) {
    unsigned lo = (unsigned)sh.kmin, hi = (unsigned)sh.kmax;
    const float top = value_of(hi);
    u64 above;
    for (;;) {                                                     // the largest key that weighs `need` with those above it
        const bool found = lo == hi;
        const unsigned probe = found ? lo + 1 : lo + (hi - lo + 1) / 2;
        const float from = value_of(probe);
        u64 mine = 0;
        walk.each([&](int i, float l) {
            const bool in = (int)(l >= from) & (int)(l <= top) & (int)row.kept(l, i);
            mine += in ? (MASS ? row.weight(l) : 1) : 0;
        });
        const u64 sum = block_sum(sh, w, mine);
        above = sum;
        if (found) break;
        if (sum >= need) lo = probe;
        else hi = probe - 1;
    }
    const float tie = value_of(lo);
    const u64 each = MASS ? row.weight(tie) : 1;                   // > 0: the equal ones' weight crosses `need`
    const u64 stay = (need - above + each - 1) / each;             // that many of them stay
    const auto one = [&](int i, float l) { return (u64)((int)(l == tie) & (int)row.kept(l, i)); };
    u64 sums[4] = {0, 0, 0, 0};
    walk.sums(sums, one);
    locate(sh, w, walk, sums, 0, stay - 1, one);
    const int hit = sh.result;                                     // -1: all of them
    row.tidx = __builtin_amdgcn_readfirstlane(hit >= 0 ? hit : (row.tval == tie ? row.tidx : 0x7fffffff));
    row.tval = uniform(tie);
}

// Leaves in sh.before[i] `base` and the weights of the entries in front of entry i of n: groups of threads share one entry's
// comparisons (n^2 / threads of them each).  n <= CAP.
__device__ __forceinline__ void rank(Shared& sh, const Who& w, const Entry* e, int n, u64 base) {
    for (int i = w.tid; i < n; i += w.nt) sh.before[i] = base;
    __syncthreads();
    const int lg = n > 1 ? 32 - __clz(n - 1) : 0, per = w.nt >> lg, groups = per > 0 ? per : 1, part = (n + groups - 1) / groups;
    for (int q = w.tid; q < groups << lg; q += w.nt) {
        const int i = q & ((1 << lg) - 1), j0 = (q >> lg) * part, j1 = j0 + part < n ? j0 + part : n;
        if (i >= n) continue;
        const u64 mine = e[i].rank;
        u64 sum = 0;
#pragma unroll 4
        for (int j = j0; j < j1; ++j) {
            const Entry x = e[j];
            sum += x.rank > mine ? x.weight : 0;
        }
        if (sum) atomicAdd(&sh.before[i], sum);
    }
    __syncthreads();
}

// one thread each in draw_few
__device__ __forceinline__ int few_limit(const Who& w) { return w.nt < FEW ? w.nt : FEW; }

// rank order of the filters: larger logit first, then lower index
__device__ __forceinline__ u64 rank_of(float l, int i) { return ((u64)key_of(l) << 32) | (unsigned)~i; }

// Narrows (row.tval, row.tidx) to the last element in rank order in front of which less than `want` lies -- elements counted
// (MASS = false, nothing narrowed before) or their weights (then `share` of the kept mass is wanted).  A histogram over linear
// bins of the logit finds the bin that holds it; the bin's range of floats picks the candidates in a second pass, and they are
// ranked in LDS.  A count of at most few_limit also collects the elements it keeps (sh.few, sh.nfew) on the way.
// Returns false, nothing narrowed, where the candidates are too many and BISECTS is false.  sh.hist is zero on entry.
template <bool MASS, bool BISECTS, typename R>
__device__ __forceinline__ bool narrow(Shared& sh, const Who& w, Row& row, R& walk, u64 want, double share) {
    const float per_unit = NBINS / 32.0f;                          // counted: 32 units of logit, whatever the temperature
    const auto bin_of = [&](float l) {
        if (MASS) {
            const int b = Row::whole(row.steps(l)) / PER_BIN;      // 64 bins per octave, 32 octaves
            return b < NBINS - 1 ? b : NBINS - 1;
        }
        return (int)fminf((row.m - l) * per_unit, (float)(NBINS - 1));
    };
    if (w.tid == 0) { sh.n = 0; sh.nfew = 0; sh.kmin = ~0ull; sh.kmax = 0; sh.last = 0; }
    if (!MASS) {
        walk.each([&](int, float l) { if (l > -INFINITY) atomicAdd(&sh.hist[bin_of(l)], 1ull); });
    } else if (row.tval == -INFINITY) {
        walk.each([&](int, float l) {
            int k;
            const u64 v = row.weight(row.steps(l), k);
            const int b = k < (NBINS - 1) * PER_BIN ? k / PER_BIN : NBINS - 1;
            if (k < FAR) atomicAdd(&sh.hist[b], v);
        });
    } else {
        walk.each([&](int i, float l) { if (row.kept(l, i)) atomicAdd(&sh.hist[bin_of(l)], row.weight(l)); });
    }
    __syncthreads();
    find_bin(sh, w, want, share);
    if (sh.bin < 0) return true;                                   // less than `want` in all: everything stays
    const int bin = __builtin_amdgcn_readfirstlane(sh.bin);
    // The candidates are the bin's elements; its range of logits only spares the others the bin's arithmetic.  A bin goes by the
    // rounded distance from the largest logit (off by half a step of the distance in fp32), and near logit 0 that is far more
    // than a few floats of the logit: the range is wider by 2^-23 of the distance d, twice that rounding, and, for its own
    // rounding to fp32, by 16 floats.  side: 1 the upper end of bin b, -1 the lower end of the bin in front of b.
    const auto edge = [&](int b, int side) {
        const double d = MASS ? (b * (double)PER_BIN - 0.5) * row.per_step : b / (double)per_unit;
        return nudged(row.md - d * (1.0 - side * 0x1p-23), 16 * side);
    };
    const bool few = !MASS && want <= (u64)few_limit(w);
    const float hi = uniform(few || bin == 0 ? row.m : edge(bin, 1)), lo = uniform(bin == NBINS - 1 ? -INFINITY : edge(bin + 1, -1));
    walk.each([&](int i, float l) {
        if ((int)(l >= lo) & (int)(l <= hi) && l > -INFINITY) {
            const int b = bin_of(l);
            if (b == bin && row.kept(l, i)) {
                const unsigned at = atomicAdd(&sh.n, 1u);
                if (at < CAP) sh.cand[at].rank = rank_of(l, i);
            }
            if (few && b < bin) sh.few[atomicAdd(&sh.nfew, 1u)].rank = rank_of(l, i);      // fewer than want of them
        }
    });
    __syncthreads();
    const unsigned n = sh.n;
    if constexpr (!BISECTS) {
        if (n > CAP) return false;
    } else if (n > CAP) {
        unsigned kmin = 0xffffffffu, kmax = 0;
        walk.each([&](int i, float l) {
            if (l > -INFINITY && bin_of(l) == bin && row.kept(l, i)) {
                const unsigned k = key_of(l);
                kmin = k < kmin ? k : kmin;
                kmax = k > kmax ? k : kmax;
            }
        });
        if (kmin <= kmax) { atomicMin(&sh.kmin, (u64)kmin); atomicMax(&sh.kmax, (u64)kmax); }
        __syncthreads();
        bisect<MASS>(sh, w, row, walk, sh.want - sh.acc);
        if (few) {                                                 // collected anew, by the exact border
            __syncthreads();
            if (w.tid == 0) sh.nfew = 0;
            __syncthreads();
            walk.each([&](int i, float l) { if (row.kept(l, i)) sh.few[atomicAdd(&sh.nfew, 1u)].rank = rank_of(l, i); });
        }
        return true;
    }
    for (int i = w.tid; i < (int)n; i += w.nt) sh.cand[i].weight = MASS ? row.weight(value_of((unsigned)(sh.cand[i].rank >> 32))) : 1;
    rank(sh, w, sh.cand, (int)n, sh.acc);                          // (its first barrier covers the weights)
    want = sh.want;
    for (int i = w.tid; i < (int)n; i += w.nt)
        if (sh.before[i] < want) {
            atomicMax(&sh.last, ~sh.cand[i].rank);
            if (few) sh.few[atomicAdd(&sh.nfew, 1u)].rank = sh.cand[i].rank;
        }
    __syncthreads();
    const u64 last = ~sh.last;
    row.tval = uniform(value_of((unsigned)(last >> 32)));
    row.tidx = __builtin_amdgcn_readfirstlane(~(int)(unsigned)last);
    return true;
}

// The rest of the row among the tokens of a small top-k: nucleus, min-p and draw by ranking alone.  -> token, total weight
__device__ __forceinline__ u64 draw_few(Shared& sh, const Who& w, const Row& row, double p, u64 share) {
    const int n = (int)sh.nfew, i = w.tid;
    u64 rank_i = 0, weight = 0;
    if (i < n) {
        rank_i = sh.few[i].rank;
        weight = row.weight(value_of((unsigned)(rank_i >> 32)));
        sh.few[i].weight = weight;
    }
    if (p < 1.0) {
        rank(sh, w, sh.few, n, 0);
        u64 mass = wave_sum64(weight);
        if (w.lane == 0) sh.wsum[w.wave] = mass;
        __syncthreads();
        mass = 0;
        for (int q = 0; q < w.waves; ++q) mass += sh.wsum[q];
        const double goal = ceil(p * (double)mass);                // in front of a kept token: less than p of the mass
        if (i < n && sh.before[i] >= (goal > 1.0 ? (u64)goal : 1)) weight = 0;
        __syncthreads();
    }
    if (i < n && !(row.steps(value_of((unsigned)(rank_i >> 32))) <= row.cut)) weight = 0;
    // by index: the entry in front of which target or less lies, and with which more does
    if (i < n) sh.few[i] = {(u64)(unsigned)rank_i, weight};        // ~index: the lower index goes first
    if (w.tid == 0) sh.result = -1;
    u64 total = wave_sum64(weight);
    if (w.lane == 0) sh.wsum[w.wave] = total;
    rank(sh, w, sh.few, n, 0);
    total = 0;
    for (int q = 0; q < w.waves; ++q) total += sh.wsum[q];
    const u64 target = __umul64hi(share, total);                   // floor(u * total)
    if (i < n && sh.before[i] <= target && sh.before[i] + weight > target) sh.result = (int)~(unsigned)rank_i;
    __syncthreads();
    return total;
}

__device__ __forceinline__ void clear_bins(Shared& sh, const Who& w) {
    for (int i = w.tid; i < NBINS; i += w.nt) sh.hist[i] = 0;
}

// Draws row r.  Returns false, nothing written, for a row that needs the bisection where BISECTS is false.
template <bool BISECTS, typename T, typename R>
__device__ __forceinline__ bool draw_row(Shared& sh, const Who& w, const SampleArgs& a, int64_t r) {
    R walk((const T*)a.logits + r * a.ld, a.V, w.waves, w.wave, w.lane);
    clear_bins(sh, w);
    for (int i = w.tid; i < STEPS; i += w.nt) sh.pow2[i] = ldexp(pow2_step(i), a.fb);
    float m = wave_max(walk.load());
    if (w.lane == 0) sh.wmax[w.wave] = m;
    __syncthreads();
    for (int i = 0; i < w.waves; ++i) m = fmaxf(m, sh.wmax[i]);
    if (m == -INFINITY) {                                          // nothing to draw from
        if (w.tid == 0) { a.ids[r] = -1; if (a.logp) a.logp[r] = -INFINITY; }
        return true;
    }
    if (m == INFINITY) { walk.squash(); m = 0.f; }
    // settings are read where they are used: a number that waits through the passes costs them registers
    const auto setting = [&](const float* rows, double all) {
        int64_t at = r;
        asm volatile("" : "+s"(at));
        return rows ? (double)rows[at] : all;
    };
    const double tau = setting(a.temperature_rows, a.temperature);
    if (!(tau > 0.0)) {                                            // greedy: the first largest one
        int best = 0x7fffffff;
        walk.each([&](int i, float l) { best = l == m && i < best ? i : best; });
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            const int other = __shfl_xor(best, o, 64);
            best = other < best ? other : best;
        }
        if (w.lane == 0) sh.before[w.wave] = (u64)best;
        __syncthreads();
        for (int i = 0; i < w.waves; ++i) best = (int)sh.before[i] < best ? (int)sh.before[i] : best;
        if (w.tid == 0) { a.ids[r] = best; if (a.logp) a.logp[r] = 0.f; }
        return true;
    }
    Row row;
    row.pow2 = sh.pow2;
    row.m = uniform(m);
    row.md = uniform((double)m);
    row.c = uniform(fmin(STEPS * 1.4426950408889634074 / tau, 1e300));    // finite: 0 c is 0; floats differ by 1e-45 and more, so from
                                                                           // 1e300 on only equals of the largest one have a weight
    row.per_step = uniform(tau * (0.693147180559945309417 / STEPS));
    row.tval = -INFINITY;
    row.tidx = -1;
    const int64_t k = a.top_k_rows ? a.top_k_rows[r] : a.top_k;
    bool few = false;
    if (k > 0 && k < a.V) {
        if (!narrow<false, BISECTS>(sh, w, row, walk, (u64)k, -1.0)) return false;
        few = k <= few_limit(w) && sh.bin >= 0;
        __syncthreads();
        if (!few) {
            clear_bins(sh, w);
            __syncthreads();
        }
    }
    const double p = setting(a.top_p_rows, a.top_p);
    if (!few && p < 1.0 && !narrow<true, BISECTS>(sh, w, row, walk, 0, p > 0.0 ? p : 0.0)) return false;
    const double mp = setting(a.min_p_rows, a.min_p);
    row.cut = uniform(mp > 0.0 ? -STEPS * log2(mp < 1.0 ? mp : 1.0) : 2.0 * FAR);
    float u = a.u ? a.u[r] : uniform01(a.seed, a.offset + (uint64_t)r);
    u = u > 0.f ? (u < 1.f ? u : 0x1.fffffep-1f) : 0.f;
    const u64 share = (u64)(u * 0x1p64f);
    u64 total;
    if (few) {
        total = draw_few(sh, w, row, p, share);
    } else {
        u64 sums[4] = {0, 0, 0, 0};
        if (row.tval == -INFINITY && mp <= 0.0) walk.sums(sums, [&](int, float l) { return row.weight(l); });      // everything
        else walk.kept_sums(sums, row, sh.queue[w.wave]);
        total = locate(sh, w, walk, sums, share, 0, [&](int i, float l) { return row.drawn(l, i); });
    }
    if (w.tid == 0) {
        const int id = sh.result;
        a.ids[r] = id;
        if (a.logp && id < 0) a.logp[r] = -INFINITY;               // no element in front of the row is ever read
        else if (a.logp) {
            const double l = (double)walk.clean(laed_to_float(((const T*)a.logits + r * a.ld)[id]));
            a.logp[r] = (float)((l - (double)m) / setting(a.temperature_rows, a.temperature) - log(ldexp((double)total, -a.fb)));      // one token alone: exactly 0
        }
    }
    return true;
}

// One block per row.  R: the row held in registers (read from memory once), or Stream, reading it again in every pass.
template <typename T, typename R, int NT>
__global__ __launch_bounds__(NT) void sample_rows_kernel(SampleArgs a) {
    __shared__ Shared sh;
    const Who w = {(int)threadIdx.x, (int)threadIdx.x & 63, __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), NT / 64, NT};
    const int64_t r = a.row0 + blockIdx.x;
    if constexpr (std::is_same<R, Stream<T>>::value) {
        draw_row<true, T, R>(sh, w, a, r);
    } else if (!draw_row<false, T, R>(sh, w, a, r)) {
        __syncthreads();
        draw_row<true, T, Stream<T>>(sh, w, a, r);
    }
}

// a grid holds fewer than 2^32 threads: more rows than that go in several launches
template <typename T, typename R, int NT>
void go(SampleArgs a, hipStream_t stream) {
    constexpr int64_t most = (1ll << 31) / NT;
    for (a.row0 = 0; a.row0 < a.N; a.row0 += most) {
        const int64_t rows = a.N - a.row0 < most ? a.N - a.row0 : most;
        hipLaunchKernelGGL((sample_rows_kernel<T, R, NT>), dim3((unsigned)rows), dim3(NT), 0, stream, a);
    }
}

template <typename T>
void launch(const SampleArgs& a, hipStream_t stream) {
    const int64_t nvec = (a.V + 2 * (16 / sizeof(T)) - 2) / (16 / sizeof(T));      // the row's start may lie inside a vector
    // The row in registers, as few vectors a thread as hold it.  Up to 8 of them nothing is spilled; 13 spill 28 registers (fp32; 53
    // in 16 bits), 16 spill 171 (238 to 241).  fp32 rows of 50000, 64 and 1024 of them under top-p 0.9: 13 vectors 39 and 173 us, 16
    // 53 and 274, the row read again in every pass 53 and 237.  Rows that only 16 hold: 60000 fp32 52 and 294 us, read again
    // 60 and 267; 128003 bf16 under a temperature 43 and 217 us, read again 45 and 205.
    // 256 threads per row where they hold it and rows are many: several rows share a CU and overlap their phases (2000 fp32, top-p:
    // 4096 rows 68 us against 186 with 1024 threads).  Fewer than 256 rows get 1024 threads, which has turned out to be
    // a little slower too (64 rows 12.9 us against 11.6).
    if (nvec <= 512 && (a.N >= 256 || nvec <= 256)) go<T, Held<T, 2>, 256>(a, stream);
    else if (nvec <= 1024 * 4) go<T, Held<T, 4>, 1024>(a, stream);
    else if (nvec <= 1024 * 8) go<T, Held<T, 8>, 1024>(a, stream);
    else if (nvec <= 1024 * 13) go<T, Held<T, 13>, 1024>(a, stream);
    else if (nvec <= 1024 * 16) go<T, Held<T, 16>, 1024>(a, stream);
    else go<T, Stream<T>, 1024>(a, stream);
}

}   // namespace
