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
constexpr int CAP = 512;                  // candidates ranked in LDS
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
    u64 cw[CAP], before[CAP];
    unsigned ckey[CAP];
    int cidx[CAP];
    u64 wsum[MAXW];
    float wmax[MAXW];
    unsigned kmin, kmax, n;
    int bin, result;
    u64 acc, want, last;
};

// ordered image of a float: larger value, larger key (-0 has been turned into 0; NaN never comes here)
__device__ __forceinline__ unsigned key_of(float l) {
    const unsigned b = __float_as_uint(l);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float value_of(unsigned k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }

// what a row's passes need
struct Row {
    float m;                              // largest logit
    double md, c2;                        // the same, log2(e) / tau
    double cut2;                          // log2(min_p): keep y2 >= cut2
    float bins;                           // linear bins per unit of logit
    int fb;
    float tval;                           // kept: l > tval, or l == tval and index <= tidx
    int tidx;

    __device__ __forceinline__ double y2(float l) const { return ((double)l - md) * c2; }
    // 2^y2 as a fixed-point number with fb binary places.  y2 = n + f with |f| <= 1/2 (adding 1.5 2^52 leaves n in the low
    // word), 2^f by the series of e^{f ln 2} up to the 11th power (remainder below 2^-47, the size of the final rounding),
    // adding 2^52 rounds to an integer in the low bits of the mantissa.  22 fp64 instructions, no branch; -inf gives 0.
    __device__ __forceinline__ u64 weight(float l) const {
        const double y = fmax(y2(l), -200.0), t = y + 6755399441055744.0, f = y - (t - 6755399441055744.0);
        constexpr double L = 0.693147180559945309417;
        constexpr double c2_ = L * L / 2, c3 = c2_ * L / 3, c4 = c3 * L / 4, c5 = c4 * L / 5, c6 = c5 * L / 6, c7 = c6 * L / 7,
                         c8 = c7 * L / 8, c9 = c8 * L / 9, c10 = c9 * L / 10, c11 = c10 * L / 11;
        double p = fma(c11, f, c10);
        p = fma(p, f, c9);
        p = fma(p, f, c8);
        p = fma(p, f, c7);
        p = fma(p, f, c6);
        p = fma(p, f, c5);
        p = fma(p, f, c4);
        p = fma(p, f, c3);
        p = fma(p, f, c2_);
        p = fma(p, f, L);
        p = fma(p, f, 1.0);
        p = ldexp(p, (int)(unsigned)__double_as_longlong(t) + fb) + 4503599627370496.0;
        return (u64)__double_as_longlong(p) & 0x000fffffffffffffull;
    }
    __device__ __forceinline__ int bin(float l) const { return (int)fminf((m - l) * bins, (float)(NBINS - 1)); }
    __device__ __forceinline__ bool kept(float l, int i) const { return (int)(l > tval) | ((int)(l == tval) & (int)(i <= tidx)); }
    __device__ __forceinline__ u64 drawn(float l, int i) const { return ((int)kept(l, i) & (int)(y2(l) >= cut2)) ? weight(l) : 0; }
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

// A row in vocabulary order: 16-byte vectors from the aligned address at or below its start (vectors that stick out of the
// row are read element by element); wave w walks a contiguous stretch of them, 64 at a time.  Elements outside the row and
// NaN come as -inf, -0 as 0.  A row whose maximum is +inf is walked as 0 where it is +inf and -inf elsewhere.
template <typename T>
struct Place {
    static constexpr int VW = 16 / sizeof(T);
    const T* p;
    int V, shift, nvec, turns, wave, lane;
    bool infinite;
    __device__ __forceinline__ Place(const T* row, int V_, int waves, int wave_, int lane_) : V(V_), wave(wave_), lane(lane_), infinite(false) {
        shift = (int)(((uintptr_t)row & 15) / sizeof(T));
        p = row - shift;
        nvec = (V + shift + VW - 1) / VW;
        turns = ((nvec + waves - 1) / waves + 63) / 64;
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
};

// the row held in registers, NV vectors per thread: read from memory once
template <typename T, int NV>
struct Held : Place<T> {
    using Place<T>::VW;
    laed_vec<T, VW> v[NV];
    static __device__ __forceinline__ unsigned (&words(laed_vec<T, VW>& x))[4] { return reinterpret_cast<unsigned (&)[4]>(x); }
    __device__ __forceinline__ Held(const T* row, int V_, int waves, int wave_, int lane_) : Place<T>(row, V_, waves, wave_, lane_) {}
    __device__ __forceinline__ float load() {
        // all loads first, from whole vectors (a clamped address where this thread's lies elsewhere); then the row's first and
        // last vector, which may stick out of it, and -inf behind it
        const int whole0 = this->shift ? 1 : 0, whole1 = (this->V + this->shift) / VW, base = this->vec_of(0);
        if (whole1 > whole0) {
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                int vec = base + 64 * j;
                vec = vec < whole0 ? whole0 : (vec < whole1 ? vec : whole1 - 1);
                if (j < this->turns) v[j] = *reinterpret_cast<const laed_vec<T, VW>*>(this->p + (int64_t)vec * VW);
            }
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
    // The empty asm statements keep the compiler from carrying per-element results (bins, 64-bit copies) from one pass to the
    // next: a register or more per element, spilled, where recomputing costs a few instructions.
    template <typename F> __device__ __forceinline__ void each(F f) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
#pragma unroll
            for (int i = 0; i < 4; ++i) asm volatile("" : "+v"(words(v[j])[i]));
        }
        int base = this->index_of(this->vec_of(0), 0);
        asm volatile("" : "+v"(base));
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (j < this->turns) {
#pragma unroll
                for (int e = 0; e < VW; ++e) {
                    f(base + 64 * VW * j + e, laed_to_float(v[j].v[e]));
                    if (e & 1) __builtin_amdgcn_sched_barrier(0);  // two elements' weights in flight, not the whole row's
                }
            }
    }
};

struct Who { int tid, lane, wave, waves, nt; };

// Bins hold weights, best first: finds the first bin at which base + cumulative weight reaches `want` -- or, with share >= 0,
// that share of the whole (rounded up, 1 at least) -- and leaves (bin, weight in front of it, want) in shared memory;
// bin = -1 if the whole is less than `want`.
__device__ __forceinline__ void find_bin(Shared& sh, const Who& w, u64 base, u64 want, double share) {
    const int per = NBINS / w.nt;
    if (w.tid == 0) sh.bin = -1;
    u64 mine = 0;
    for (int i = 0; i < per; ++i) mine += sh.hist[w.tid * per + i];
    const u64 inc = wave_scan64(mine, w.lane);
    if (w.lane == 63) sh.wsum[w.wave] = inc;
    __syncthreads();
    u64 front = base + inc - mine, whole = 0;
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

// First element in vocabulary order at which the cumulative weight exceeds `target`; its index in sh.result (-1: none).
// `mine`: this thread's sum of weight(i, l).
template <typename R, typename W>
__device__ __forceinline__ void locate(Shared& sh, const Who& w, const R& row, u64 mine, u64 target, W weight) {
    constexpr int VW = R::VW;
    mine = wave_sum64(mine);
    if (w.tid == 0) sh.result = -1;
    __syncthreads();
    if (w.lane == 0) sh.wsum[w.wave] = mine;
    __syncthreads();
    u64 front = 0;
    for (int i = 0; i < w.wave; ++i) front += sh.wsum[i];
    if (front <= target && front + mine > target) {                // exactly one wave
        for (int j = 0; j < row.turns; ++j) {                      // read again: 1 / waves of the row
            const int vec = row.vec_of(j);
            float l[VW];
            u64 v = 0;
            if (vec < row.nvec) {
                const auto r = row.raw(vec);
#pragma unroll
                for (int e = 0; e < VW; ++e) {
                    l[e] = row.clean(laed_to_float(r.v[e]));
                    v += weight(row.index_of(vec, e), l[e]);
                }
            }
            const u64 inc = wave_scan64(v, w.lane), all = __shfl(inc, 63, 64);
            if (front + all > target) {
                u64 at = front + inc - v;
                if (at <= target && at + v > target) {             // exactly one lane
                    int hit = -1;
#pragma unroll
                    for (int e = 0; e < VW; ++e) {
                        at += weight(row.index_of(vec, e), l[e]);
                        if (hit < 0 && at > target) hit = row.index_of(vec, e);
                    }
                    sh.result = hit;
                }
                break;
            }
            front += all;
        }
    }
    __syncthreads();
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
// order.  Rare: each pass costs what the histogram's does.
template <bool MASS, typename R>
__device__ __forceinline__ void bisect(Shared& sh, const Who& w, Row& row, R& walk, u64 need) {
    unsigned lo = sh.kmin, hi = sh.kmax;
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
    u64 mine = 0;
    walk.each([&](int i, float l) { mine += one(i, l); });
    locate(sh, w, walk, mine, stay - 1, one);
    const int hit = sh.result;                                     // -1: all of them
    row.tidx = hit >= 0 ? hit : (row.tval == tie ? row.tidx : 0x7fffffff);
    row.tval = tie;
}

// Narrows (row.tval, row.tidx) to the last element in rank order in front of which less than `want` lies -- elements counted
// (MASS = false) or their weights (then `want` is the share of the kept mass).  A histogram over linear bins of the logit
// finds the bin that holds it, and the bin's elements are ranked in LDS.  sh.hist is zero on entry.
template <bool MASS, typename R>
__device__ __forceinline__ void narrow(Shared& sh, const Who& w, Row& row, R& walk, u64 want, double share) {
    walk.each([&](int i, float l) {
        if (!MASS) {
            if (l > -INFINITY) atomicAdd(&sh.hist[row.bin(l)], 1ull);
        } else {
            const u64 v = row.kept(l, i) ? row.weight(l) : 0;
            if (v) atomicAdd(&sh.hist[row.bin(l)], v);
        }
    });
    if (w.tid == 0) { sh.n = 0; sh.kmin = 0xffffffffu; sh.kmax = 0; sh.last = 0; }
    __syncthreads();
    find_bin(sh, w, 0, want, share);
    if (sh.bin < 0) return;                                        // less than `want` in all: everything stays
    const int bin = sh.bin;
    walk.each([&](int i, float l) {
        if (row.bin(l) == bin && l > -INFINITY && row.kept(l, i)) {
            const unsigned at = atomicAdd(&sh.n, 1u);
            if (at < CAP) { sh.ckey[at] = key_of(l); sh.cidx[at] = i; }
        }
    });
    __syncthreads();
    unsigned n = sh.n;
    if (n > CAP) {
        unsigned kmin = 0xffffffffu, kmax = 0;
        walk.each([&](int i, float l) {
            if (row.bin(l) == bin && l > -INFINITY && row.kept(l, i)) {
                const unsigned k = key_of(l);
                kmin = k < kmin ? k : kmin;
                kmax = k > kmax ? k : kmax;
            }
        });
        if (kmin <= kmax) { atomicMin(&sh.kmin, kmin); atomicMax(&sh.kmax, kmax); }
        __syncthreads();
        bisect<MASS>(sh, w, row, walk, sh.want - sh.acc);
        return;
    }
    // rank the n candidates: groups of threads share one candidate's comparisons
    const u64 acc = sh.acc;
    want = sh.want;
    int n2 = 1;
    while (n2 < (int)n) n2 <<= 1;
    for (int i = w.tid; i < (int)n; i += w.nt) {
        sh.cw[i] = MASS ? row.weight(value_of(sh.ckey[i])) : 1;
        sh.before[i] = acc;
    }
    __syncthreads();
    const int groups = w.nt > n2 ? w.nt / n2 : 1, part = ((int)n + groups - 1) / groups;
    for (int q = w.tid; q < groups * n2; q += w.nt) {
        const int i = q & (n2 - 1), j0 = q / n2 * part, j1 = j0 + part < (int)n ? j0 + part : (int)n;
        if (i >= (int)n) continue;
        const unsigned k = sh.ckey[i];
        const int x = sh.cidx[i];
        u64 sum = 0;
        for (int j = j0; j < j1; ++j) sum += (sh.ckey[j] > k || (sh.ckey[j] == k && sh.cidx[j] < x)) ? sh.cw[j] : 0;
        if (sum) atomicAdd(&sh.before[i], sum);
    }
    __syncthreads();
    for (int i = w.tid; i < (int)n; i += w.nt)
        if (sh.before[i] < want) atomicMax(&sh.last, ((u64)~sh.ckey[i] << 32) | (unsigned)sh.cidx[i]);
    __syncthreads();
    row.tval = value_of(~(unsigned)(sh.last >> 32));
    row.tidx = (int)(unsigned)sh.last;
}

__device__ __forceinline__ void clear_bins(Shared& sh, const Who& w) {
    for (int i = w.tid; i < NBINS; i += w.nt) sh.hist[i] = 0;
}

template <typename T, typename R>
__device__ __forceinline__ void draw_row(Shared& sh, const Who& w, const SampleArgs& a, int64_t r) {
    R walk((const T*)a.logits + r * a.ld, a.V, w.waves, w.wave, w.lane);
    clear_bins(sh, w);
    float m = wave_max(walk.load());
    if (w.lane == 0) sh.wmax[w.wave] = m;
    __syncthreads();
    for (int i = 0; i < w.waves; ++i) m = fmaxf(m, sh.wmax[i]);
    if (m == -INFINITY) {                                          // nothing to draw from
        if (w.tid == 0) { a.ids[r] = -1; if (a.logp) a.logp[r] = -INFINITY; }
        return;
    }
    if (m == INFINITY) { walk.squash(); m = 0.f; }
    const double tau = a.temperature_rows ? (double)a.temperature_rows[r] : a.temperature;
    const int64_t k = a.top_k_rows ? a.top_k_rows[r] : a.top_k;
    const double p = a.top_p_rows ? (double)a.top_p_rows[r] : a.top_p;
    const double mp = a.min_p_rows ? (double)a.min_p_rows[r] : a.min_p;
    if (!(tau > 0.0)) {                                            // greedy: the first largest one
        const auto first = [&](int, float l) { return (u64)(l == m); };
        u64 mine = 0;
        walk.each([&](int i, float l) { mine += first(i, l); });
        locate(sh, w, walk, mine, 0, first);
        if (w.tid == 0) { a.ids[r] = sh.result; if (a.logp) a.logp[r] = 0.f; }
        return;
    }
    Row row;
    row.m = m;
    row.md = (double)m;
    row.fb = a.fb;
    row.tval = -INFINITY;
    row.tidx = -1;
    row.c2 = fmin(1.4426950408889634074 / tau, 1e300);
    row.bins = (float)fmin(64.0 / tau, 1e30);
    row.cut2 = mp > 0.0 ? log2(mp < 1.0 ? mp : 1.0) : -INFINITY;
    if (k > 0 && k < a.V) {
        narrow<false>(sh, w, row, walk, (u64)k, -1.0);
        __syncthreads();
        clear_bins(sh, w);
        __syncthreads();
    }
    if (p < 1.0) narrow<true>(sh, w, row, walk, 0, p > 0.0 ? p : 0.0);
    const auto drawn = [&](int i, float l) { return row.drawn(l, i); };
    u64 mine = 0;
    walk.each([&](int i, float l) { mine += drawn(i, l); });
    __syncthreads();
    u64 total = wave_sum64(mine);
    if (w.lane == 0) sh.wsum[w.wave] = total;
    __syncthreads();
    total = 0;
    for (int i = 0; i < w.waves; ++i) total += sh.wsum[i];
    float u = a.u ? a.u[r] : uniform01(a.seed, a.offset + (uint64_t)r);
    u = u > 0.f ? (u < 1.f ? u : 0x1.fffffep-1f) : 0.f;
    const u64 target = __umul64hi((u64)(u * 0x1p64f), total);      // floor(u * total)
    locate(sh, w, walk, mine, target, drawn);
    if (w.tid == 0) {
        const int id = sh.result;
        a.ids[r] = id;
        if (a.logp) {
            const double l = (double)walk.clean(laed_to_float(((const T*)a.logits + r * a.ld)[id]));
            a.logp[r] = (float)((l - row.md) / tau - (log((double)total) - a.fb * 0.693147180559945309417));
        }
    }
}

// One block per row.  R: the row held in registers (read from memory once), or Stream, reading it again in every pass.
template <typename T, typename R, int NT>
__global__ __launch_bounds__(NT) void sample_rows_kernel(SampleArgs a) {
    __shared__ Shared sh;
    const Who w = {(int)threadIdx.x, (int)threadIdx.x & 63, (int)threadIdx.x >> 6, NT / 64, NT};
    draw_row<T, R>(sh, w, a, blockIdx.x);
}

template <typename T, typename R, int NT>
void go(const SampleArgs& a, unsigned grid, hipStream_t stream) {
    hipLaunchKernelGGL((sample_rows_kernel<T, R, NT>), dim3(grid), dim3(NT), 0, stream, a);
}

template <typename T>
void launch(const SampleArgs& a, hipStream_t stream) {
    const unsigned grid = (unsigned)a.N;
    const int64_t nvec = (a.V + 2 * (16 / sizeof(T)) - 2) / (16 / sizeof(T));      // the row's start may lie inside a vector
    // 256 threads per row where they hold it and rows are many: several rows share a CU and overlap their phases
    if (nvec <= 512 && (a.N >= 256 || nvec <= 256)) go<T, Held<T, 2>, 256>(a, grid, stream);
    else if (nvec <= 1024 * 2) go<T, Held<T, 2>, 1024>(a, grid, stream);
    else if (nvec <= 1024 * 4) go<T, Held<T, 4>, 1024>(a, grid, stream);
    else if (nvec <= 1024 * 8) go<T, Held<T, 8>, 1024>(a, grid, stream);
    else if (nvec <= 1024 * 13) go<T, Held<T, 13>, 1024>(a, grid, stream);
    else if (nvec <= 1024 * 16) go<T, Held<T, 16>, 1024>(a, grid, stream);
    else go<T, Stream<T>, 1024>(a, grid, stream);
}

}   // namespace

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
    SampleArgs a = {logits, ld, N, V, 62 - lg < 46 ? 62 - lg : 46, u, seed, offset, temperature, temperature_rows, top_k, top_k_rows,
                    top_p, top_p_rows, min_p, min_p_rows, ids, logp};
#define LAUNCH(T) launch<T>(a, (hipStream_t)stream)
    LAED_BY_DTYPE(dtype, LAUNCH);
#undef LAUNCH
    LAED_LAUNCH_CHECK("sample_rows");
    return 0;
}
