// Sampling with temperature, top-k, top-p and min-p from one uniform number a row (q35_sample).
//
// Candidates are ranked by logit, equal ones by id. Every filter keeps a prefix of the ranking, so what is
// kept is a count of first places, and the draw is a place too: the one in whose share of the kept mass the
// number falls. Weights are exp((l - max) / T) in 64 bits, held as whole multiples of 2^-S (2^S times the number
// of candidates stays below 2^62): sums are exact, so they do not depend on their order, and places next to
// each other in mass are told apart down to 2^-S of the largest weight.
//
// A row is cut into slices, a workgroup each. The first launch finds the largest logit; the second counts
// candidates and mass by bins of (max - l) / T, down to 36, below which weights are 0; the third
// gathers the candidates of the bins that the borders and the draw may lie in (a border that is known to a bin
// leaves the next one open to as much mass, so mostly to a bin as well). The workgroup that is done last
// with a row plans that, or sorts the candidates and finds the exact places. A small top_k needs no counts: the largest
// logits of 64 parts of the row, which the first launch leaves, bound its candidates, and the second launch gathers
// them and draws. Rows of one slice take one launch. Where the open bins hold more than kList candidates (that many equal
// logits, or a whole row within less than a temperature), the places are found by radix descent over the row.
//
// One row of 151936 with a top_k of 20 takes 15.5 us (by counts 22.5), 48 with settings of all kinds 46 us. The logits
// are read two or three times, 29 MB of 48 rows in about 5 us each; the rest is one workgroup's chain of steps at the end
// of each launch (settling 64 candidates takes 3.5 us, 2048 5) and, of many rows, the weights: 12 instructions in
// 64 bits each and an addition of 64 bits in LDS (together 6 us), and the listing of those in open bins (3 us). Flat
// rows have longer lists (one of 151936 at a temperature of 5, top_p 0.95: 41 us; 2000 equal logits on top 47, 8000 105).
#include "dev_q4.hpp"
#include "launch_q4.hpp"

namespace q35k {
namespace {

__device__ __forceinline__ void put_token(const SampleArgs& a, int b, int token) {
    a.token[b] = token;
    if (a.feed) a.feed[b] = max(token, 0);
}

constexpr int kThreads = 1024;

// ordered bits of a logit: larger logits have larger keys, both zeros one, a NaN counts as -inf
__device__ __forceinline__ uint32_t key_of(float x) {
    x = x == x ? x + 0.0f : -INFINITY;
    const uint32_t b = __float_as_uint(x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
constexpr uint32_t kKeyNone = 0x007fffffu;  // -inf
constexpr uint32_t kKeyInf = 0xff800000u;   // +inf

// Bins of 1/128 of a depth, down to 36. (Wider ones below 12 cost a batch 1 us less, but there lies the bulk of a row with one
// token far above it, thousands of candidates a bin.)
constexpr int kBins = 36 * 128;         // and one for what has no weight

// 2^(-y / 512) for 0 <= y < 2^15: y = n + f, |f| <= 1/2, so it is 2^-(n div 512) 2^-(n mod 512 / 512) 2^(-f / 512), the second
// factor from a table and the last by four terms of its series (the fifth is below 2^-55).
struct ExpTable {
    double t[512];
    __device__ __forceinline__ void fill() {
        if (threadIdx.x < 512) t[threadIdx.x] = exp2(-static_cast<double>(threadIdx.x) / 512.0);
    }
};
constexpr double kLn2 = 0.69314718055994530942;
__device__ __forceinline__ double exp2_minus(double y, const ExpTable& e) {
    constexpr double kWhole = 0x1.8p52, kStep = kLn2 / 512.0;
    const double m = y + kWhole, f = y - (m - kWhole);  // n in the last bits of m
    const int n = static_cast<int>(__builtin_bit_cast(uint64_t, m));
    double p = fma(f, kStep * kStep * kStep * kStep / 24.0, -kStep * kStep * kStep / 6.0);
    p = fma(f, p, kStep * kStep / 2.0);
    p = fma(f, p, -kStep);
    p = fma(f, p, 1.0);
    // 2^-(n div 512) straight into the exponent
    const uint64_t r = __builtin_bit_cast(uint64_t, e.t[n & 511] * p);
    return __builtin_bit_cast(double, r - (static_cast<uint64_t>(static_cast<uint32_t>(n >> 9) << 20) << 32));
}

constexpr float kLeastT = 1e-36f;  // below this the bins' arithmetic in fp32 would not do

struct Weigher {
    double top, rt, unit;
    float top32, rt32;
    const ExpTable& table;
    bool inf;
    __device__ __forceinline__ Weigher(uint32_t key, float T, double unit_, const ExpTable& e)
        : top(of_key(key)), rt(512.0 / kLn2 / static_cast<double>(T)), unit(unit_), top32(of_key(key)),
          rt32(static_cast<float>(rt * (kLn2 / 4.0))), table(e), inf(key == kKeyInf) {}
    // (max - l) / T in units of ln 2 / 512: infinite or a NaN where a candidate is ruled out
    __device__ double depth(float l) const {
        if (inf) return l == INFINITY ? 0.0 : INFINITY;
        return (top - static_cast<double>(l)) * rt;
    }
    __device__ double depth(uint32_t key) const { return depth(of_key(key)); }
    // The same in fp32, for bins: whatever its rounding, larger logits have no larger ones, and all with
    // weight are below kBins (a weight ends at 35.4).
    __device__ float place(float l) const {
        if (inf) return l == INFINITY ? 0.0f : INFINITY;
        return l > -INFINITY ? fminf(top32 - l, 3.4e38f) * rt32 : INFINITY;
    }
    static constexpr double kDeepest = 36.0 * 512.0 / kLn2;
    // the weight in 64 bits, of the largest
    __device__ double share(uint32_t key) const {
        const double y = depth(key);
        return y < kDeepest ? exp2_minus(y, table) : 0.0;
    }
    // a whole number of units: rounded by what 2^52 more leaves of it
    __device__ uint64_t units_within(double depth) const {
        return __builtin_bit_cast(uint64_t, fma(exp2_minus(depth, table), unit, 0x1p52)) & 0xfffffffffffffull;
    }
    __device__ uint64_t units(double depth) const { return depth < kDeepest ? units_within(depth) : 0; }
    __device__ uint64_t operator()(uint32_t key) const { return units(depth(key)); }
};

// Of a mass `total`: the unit that the last candidate of a top_p below 1 holds, and the drawn one.
__device__ __forceinline__ uint64_t top_p_place(float p, uint64_t total) {
    const double want = ceil(static_cast<double>(p) * static_cast<double>(total));
    return want >= 1.0 ? min(static_cast<uint64_t>(want), total) - 1 : 0;
}
__device__ __forceinline__ uint64_t drawn_place(float u, uint64_t total) {
    return min(static_cast<uint64_t>(floor(static_cast<double>(u > 0.0f ? fminf(u, 1.0f) : 0.0f) * static_cast<double>(total))), total - 1);
}

// ---- by bins
constexpr int kParts = 64;              // of a row, every slice having some of each
constexpr int kFew = 2048;              // most lists are shorter
constexpr int kList = 8192;             // candidates that can be listed: some bins of a flat row
constexpr int kMostK = 1024;            // top_k up to this: every candidate that it may leave is listed
constexpr int kBuckets = kThreads;
// Candidates of one bucket up to which counting sorts it (of one row, 100 equal ones by counting 32.3 us in all, by comparing all
// 31.6; 500 51.5 and 36).
constexpr uint32_t kCrowd = 64;
constexpr int kPer = (kBins + kThreads) / kThreads;

// a candidate in the ranking's order: larger ones first
__device__ __forceinline__ uint64_t entry_of(uint32_t key, int id) { return static_cast<uint64_t>(key) << 32 | static_cast<uint32_t>(~id); }

// What is asked of a row.
struct Question {
    int k;                              // 0: all
    float p, m, u;
    bool few;                           // a small top_k: counts alone lead to its candidates
    __device__ __forceinline__ Question(const SampleArgs& a, int b)
        : k(a.top_k ? max(a.top_k[b], 0) : 0), p(a.top_p ? a.top_p[b] : 1.0f), m(a.min_p ? a.min_p[b] : 0.0f), u(a.u[b]),
          few(k > 0 && k <= kMostK) {}
};

// The open bins, in up to four ranges, apart and in order (empty ones have hi < lo): all their candidates are
// listed.
struct Plan {
    int lo[4], hi[4];
    uint64_t mass[4], end[4];           // mass before the range, and with it
    uint64_t all;                       // mass of the row
    int k_range, m_range;               // where the last candidate of top_k and the first that min_p may leave out
                                        // are; -1: they leave out nothing that has weight
    uint32_t k_at;                      // the place of the former in its range
};

// What a row's workgroups share, in the workspace. Cleared by the first launch.
struct Row {
    uint64_t mass[kBins];
    uint32_t count[kBins];
    uint32_t listed, counted, gathered, done;
    Plan plan;
    uint64_t list[kList];
};

struct Work {
    union {
        struct {
            uint64_t mass[kBins + 1];   // by bin, then of the bins before
            uint32_t count[kBins + 1];
        } bins;
        struct {
            uint64_t list[kList], run[kList];
            uint32_t at[kBuckets];
        } pick;
        uint32_t part[kThreads / 64][kParts];
    };
    Plan plan;
    ExpTable exp;
    uint64_t wave_mass[kThreads / 64];
    uint32_t wave_count[kThreads / 64];
    uint32_t in_range[4];
    uint32_t listed, base, last;
};

__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
    const auto step = [&](int o) { v = max(v, static_cast<uint32_t>(o)); };
    step(dpp_i<0xB1>(static_cast<int>(v)));
    step(dpp_i<0x4E>(static_cast<int>(v)));
    step(dpp_i<0x141>(static_cast<int>(v)));
    step(dpp_i<0x140>(static_cast<int>(v)));
    step(__builtin_amdgcn_ds_swizzle(static_cast<int>(v), 0x401F));
    return max(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), 0)),
               static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), 32)));
}
__device__ __forceinline__ uint64_t wave_top(uint64_t v) {
    const uint32_t hi = wave_max_u32(static_cast<uint32_t>(v >> 32));
    const uint32_t lo = wave_max_u32(static_cast<uint32_t>(v >> 32) == hi ? static_cast<uint32_t>(v) : 0u);
    return static_cast<uint64_t>(hi) << 32 | lo;
}
// the sum of the threads before this one; `waves` has a place for each wave, one use between barriers
template <typename U>
__device__ __forceinline__ U block_scan(U v, U* waves) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const U in = wave_scan(v);
    if ((threadIdx.x & 63) == 63) waves[wave] = in;
    __syncthreads();
    const U sums = wave_scan(waves[threadIdx.x & (kThreads / 64 - 1)]);
    return in - v + (wave ? lane_of(sums, wave - 1) : U{0});
}

// What workgroups of one row leave each other within a launch passes through these and atomic additions: they
// go to where all of them look, past the caches that do not.
template <typename U>
__device__ __forceinline__ U shared_load(const U* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
template <typename U>
__device__ __forceinline__ void shared_store(U* p, U v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
// f(logit, id) for ids [i, e), i a multiple of four: sixteen are on their way at a time, whatever f does.
template <typename F>
__device__ __forceinline__ void each_logit(const float* x, int i, int e, const F& f) {
    int j = i + 4 * threadIdx.x;
    if ((reinterpret_cast<uintptr_t>(x) & 15) == 0) {
        constexpr int kBatch = 4;
        const int last = (e - 4) & ~3;  // the last whole four
        for (; j <= last; j += 4 * kBatch * kThreads) {
            float4 l[kBatch];
#pragma unroll
            for (int n = 0; n < kBatch; ++n) l[n] = *reinterpret_cast<const float4*>(x + min(j + 4 * n * kThreads, last));
#pragma unroll
            for (int n = 0; n < kBatch; ++n) {
                const int id = j + 4 * n * kThreads;
                if (id <= last) f(l[n].x, id), f(l[n].y, id + 1), f(l[n].z, id + 2), f(l[n].w, id + 3);
            }
        }
        j = max(last + 4, i) + threadIdx.x;
        if (j < e) f(x[j], j);
        return;
    }
    constexpr int kBatch = 16;
    for (j = i + threadIdx.x; j < e; j += kBatch * kThreads) {
        float l[kBatch];
#pragma unroll
        for (int n = 0; n < kBatch; ++n) l[n] = x[min(j + n * kThreads, e - 1)];
#pragma unroll
        for (int n = 0; n < kBatch; ++n)
            if (j + n * kThreads < e) f(l[n], j + n * kThreads);
    }
}

// The largest entry of ids [i, e); where the temperature is not 0 only its key matters, and `parts` (may be null)
// gets the largest keys of kParts parts of the ids, by way of `spread`, kThreads floats of LDS.
__device__ __forceinline__ uint64_t slice_top(const float* x, int i, int e, bool greedy, uint64_t* waves, uint32_t* parts, float* spread) {
    uint64_t top = 0;
    float m = -INFINITY;                // fmaxf passes over a NaN
    if (greedy) each_logit(x, i, e, [&](float l, int j) { top = max(top, entry_of(key_of(l), j)); });
    else each_logit(x, i, e, [&](float l, int) { m = fmaxf(m, l); });
    if (!greedy) {
        if (parts) {                    // a part: the same lane of every wave
            spread[threadIdx.x] = m;
            __syncthreads();
            if (threadIdx.x < kParts) {
#pragma unroll
                for (int w = 1; w < kThreads / kParts; ++w) m = fmaxf(m, spread[w * kParts + threadIdx.x]);
                parts[threadIdx.x] = key_of(m);
            }
        }
        top = entry_of(key_of(m), 0);
    }
    top = wave_top(top);
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x / 64] = top;
    __syncthreads();
    return wave_top(waves[threadIdx.x & (kThreads / 64 - 1)]);
}
// a lane's of the slices' tops; the row's is the wave_top of these
__device__ __forceinline__ uint64_t lane_top(const uint64_t* tops, int slices) {
    uint64_t top = 0;
    for (int i = threadIdx.x & 63; i < slices; i += 64) top = max(top, tops[i]);
    return top;
}

// greedy and empty rows, and rows without a candidate: true if there is nothing more to do
__device__ __forceinline__ bool plain_row(const SampleArgs& a, int b, float T, uint64_t top, bool writes) {
    const uint32_t key = static_cast<uint32_t>(top >> 32);
    if (T > 0.0f && key != kKeyNone) return false;
    if (writes && T >= 0.0f) {
        put_token(a, b, key == kKeyNone ? -1 : static_cast<int>(~static_cast<uint32_t>(top)));
        if (a.prob) a.prob[b] = key == kKeyNone ? 0.0f : 1.0f;
    }
    return true;
}

__device__ __forceinline__ void clear_bins(Work& sh) {
    for (int i = threadIdx.x; i <= kBins; i += kThreads) sh.bins.mass[i] = 0, sh.bins.count[i] = 0;
}
// Masses by bin, and counts where there is a top_k; counts alone for a small one. (The additions in LDS bound
// this: one of 64 bits takes more of its time than the weight.)
__device__ __forceinline__ void count_slice(const float* x, int i, int e, const Question& q, const Weigher& w, Work& sh) {
    const bool counts = q.k > 0, masses = !q.few;
    each_logit(x, i, e, [&](float l, int) {
        const float z = w.place(l);
        if (!(z < kBins)) return;
        const int bin = static_cast<int>(z);
        if (counts) atomicAdd(&sh.bins.count[bin], 1u);
        if (masses) atomicAdd(reinterpret_cast<unsigned long long*>(&sh.bins.mass[bin]), static_cast<unsigned long long>(w.units_within(w.depth(l))));
    });
}

// bins' counts and masses become those of the bins before; the totals stand behind the last
__device__ __forceinline__ void add_up(Work& sh) {
    uint64_t m[kPer], im = 0;
    uint32_t n[kPer], in = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int b = threadIdx.x * kPer + i;
        m[i] = b < kBins ? sh.bins.mass[b] : 0, n[i] = b < kBins ? sh.bins.count[b] : 0;
        im += m[i], in += n[i];
    }
    im = block_scan(im, sh.wave_mass);
    in = block_scan(in, sh.wave_count);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int b = threadIdx.x * kPer + i;
        if (b <= kBins) sh.bins.mass[b] = im, sh.bins.count[b] = in;
        im += m[i], in += n[i];
    }
    __syncthreads();
}

// the bin that holds unit x of the mass (x below the total) or candidate x: 64 steps of kBins / 64 bins, then one by one
template <bool BY_MASS>
__device__ __forceinline__ int bin_of(uint64_t x, const Work& sh) {
    static_assert(kBins % 64 == 0 && kBins / 64 <= 128);
    const int lane = threadIdx.x & 63;
    const auto before = [&](int b) { return BY_MASS ? sh.bins.mass[b] : static_cast<uint64_t>(sh.bins.count[b]); };
    const int base = (__popcll(__ballot(before(lane * (kBins / 64)) <= x)) - 1) * (kBins / 64);
    int n = __popcll(__ballot(before(min(base + lane, kBins)) <= x));
    if (n == 64 && kBins / 64 > 64) n += __popcll(__ballot(lane < kBins / 64 - 64 && before(min(base + 64 + lane, kBins)) <= x));
    return base + n - 1;
}

// Makes the plan, once all is counted and added up: one wave.
__device__ __forceinline__ void make_plan(const Question& q, Work& sh) {
    Plan& p = sh.plan;
    const uint64_t* mass = sh.bins.mass;
    const uint32_t* count = sh.bins.count;
    int l[4] = {0, 0, 0, 0}, h[4] = {-1, -1, -1, -1};
    int k_range = -1, m_range = -1, k_bin = 0, m_bin = -1;
    uint64_t lo = mass[kBins], hi = lo; // the total lies within
    if (q.few) {
        // all that top_k may leave; what is behind a rank of kBins bins has no weight
        h[0] = static_cast<uint32_t>(q.k) < count[kBins] ? bin_of<false>(q.k - 1, sh) : kBins - 1;
        k_range = static_cast<uint32_t>(q.k) < count[kBins] ? 0 : -1;
        m_range = q.m > 0.0f ? 0 : -1;
    } else {
        if (q.k > 0 && static_cast<uint32_t>(q.k) < count[kBins]) {
            k_range = 0;
            k_bin = l[0] = h[0] = bin_of<false>(q.k - 1, sh);
            lo = max(mass[l[0]], uint64_t{1}), hi = mass[l[0] + 1];
        }
        if (q.p < 1.0f) {
            l[1] = h[1] = bin_of<true>(top_p_place(q.p, lo), sh);
            if (hi != lo) h[1] = bin_of<true>(top_p_place(q.p, hi), sh);
            lo = max(mass[l[1]], uint64_t{1}), hi = min(hi, mass[h[1] + 1]);
        }
        if (q.m > 0.0f) {
            // candidates next to the border are compared one by one
            const double z = q.m < 1.0f ? -log(static_cast<double>(q.m)) : 0.0;
            const auto bin = [](double depth) { return static_cast<int>(fminf(static_cast<float>(depth * 128.0), kBins)); };
            l[2] = bin(fmax(z - 1e-4, 0.0)), h[2] = min(bin(z + 1e-4), kBins - 1);
            if (l[2] < kBins) {
                m_bin = l[2];
                lo = min(lo, max(mass[l[2]], uint64_t{1})), hi = min(hi, mass[h[2] + 1]);
            } else {
                l[2] = 0, h[2] = -1;    // only what has no weight is left out
            }
        }
        l[3] = h[3] = bin_of<true>(drawn_place(q.u, lo), sh);
        if (hi != lo) h[3] = bin_of<true>(drawn_place(q.u, hi), sh);
        // in order, those that meet as one
#pragma unroll
        for (int i = 0; i < 3; ++i)
#pragma unroll
            for (int j = 0; j < 3; ++j)
                if (h[j + 1] >= l[j + 1] && (h[j] < l[j] || l[j + 1] < l[j])) {
                    const int x = l[j], y = h[j];
                    l[j] = l[j + 1], h[j] = h[j + 1], l[j + 1] = x, h[j + 1] = y;
                }
#pragma unroll
        for (int i = 0; i < 3; ++i)
#pragma unroll
            for (int j = i + 1; j < 4; ++j)
                if (h[i] >= l[i] && h[j] >= l[j] && l[j] <= h[i] + 1) h[i] = max(h[i], h[j]), l[j] = 0, h[j] = -1;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (k_range >= 0 && l[i] <= k_bin && k_bin <= h[i]) k_range = i;
            if (m_bin >= 0 && l[i] <= m_bin && m_bin <= h[i]) m_range = i;
        }
    }
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) p.lo[i] = l[i], p.hi[i] = h[i], p.mass[i] = h[i] < l[i] ? 0 : mass[l[i]], p.end[i] = h[i] < l[i] ? 0 : mass[h[i] + 1];
        p.all = mass[kBins];
        p.k_range = k_range, p.m_range = m_range;
        p.k_at = k_range < 0 ? 0 : q.k - 1 - count[p.lo[k_range]];
        }
}

// Ids [i, e) of the open bins, to the workgroup's list; sh.listed counts on where it is full.
__device__ __forceinline__ void gather(const float* x, int i, int e, const Weigher& w, const Plan& p, Work& sh) {
    uint32_t lo[4], bins[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) lo[r] = p.lo[r], bins[r] = p.hi[r] + 1 - p.lo[r];
    each_logit(x, i, e, [&](float l, int j) {
        const uint32_t bin = static_cast<uint32_t>(fminf(w.place(l), kBins));  // kBins where there is no weight: no range's
        bool in = false;
#pragma unroll
        for (int r = 0; r < 4; ++r) in |= bin - lo[r] < bins[r];
        if (in) {
            const uint32_t at = atomicAdd(&sh.listed, 1u);
            if (at < kList) sh.pick.list[at] = entry_of(key_of(l), j);
        }
    });
}

// sh.pick.list's first n entries in their order, by a bitonic network.
__device__ __forceinline__ void sort_list(int n, Work& sh) {
    int N = 64;
    while (N < n) N *= 2;
    for (int i = n + threadIdx.x; i < N; i += kThreads) sh.pick.list[i] = 0;
    for (int run = 2; run <= N; run *= 2)
        for (int d = run / 2; d > 0; d /= 2) {
            __syncthreads();
            for (int i = threadIdx.x; i < N / 2; i += kThreads) {
                const int at = 2 * i - (i & (d - 1));
                const uint64_t x = sh.pick.list[at], y = sh.pick.list[at + d];
                if ((x < y) == ((at & run) == 0)) sh.pick.list[at] = y, sh.pick.list[at + d] = x;
            }
        }
    __syncthreads();
}

// The exact places, from the n <= kEach kThreads candidates of the open bins in sh.pick.list.
template <int kEach>
__device__ __forceinline__ void settle(const SampleArgs& a, int b, const Question& q, int n, const Weigher& w, Work& sh) {
    const Plan& p = sh.plan;
    const int t = threadIdx.x, lane = t & 63, wave = t / 64;
    // Sorted by buckets of equal width in depth, a few candidates each, and within one by counting; where one holds many, by
    // comparing all (2000 equal ones: 47 us in all, by counting 219).
    sh.pick.at[t] = 0;
    if (t < 4) sh.in_range[t] = 0;
    __syncthreads();
    float width[4], wide = 0.0f;        // bins before the range
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        width[r] = wide;
        wide += p.hi[r] + 1 - p.lo[r];
    }
    const float scale = static_cast<float>(kBuckets) / wide;
    uint64_t mine[kEach];
    int of[kEach];
    uint32_t place[kEach];
    bool crowded = false;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const bool there = t + i * kThreads < n;
        mine[i] = there ? sh.pick.list[t + i * kThreads] : 0;
        const float z = w.place(of_key(static_cast<uint32_t>(mine[i] >> 32)));
        float before = 0.0f;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const bool in = there && z >= p.lo[r] && z < p.hi[r] + 1;
            if (in) before = width[r] + (z - p.lo[r]);
            const uint64_t v = __ballot(in);
            if (v && lane == 0) atomicAdd(&sh.in_range[r], static_cast<uint32_t>(__popcll(v)));
        }
        of[i] = min(static_cast<int>(before * scale), kBuckets - 1);
        place[i] = there ? atomicAdd(&sh.pick.at[of[i]], 1u) : 0;
        crowded |= place[i] >= kCrowd;
    }
    if (__syncthreads_or(crowded)) {
        sort_list(n, sh);
    } else {
        sh.pick.at[t] = block_scan(sh.pick.at[t], sh.wave_count);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            if (t + i * kThreads < n) sh.pick.list[sh.pick.at[of[i]] + place[i]] = mine[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            if (t + i * kThreads >= n) continue;
            const uint32_t first = sh.pick.at[of[i]], end = of[i] + 1 < kBuckets ? sh.pick.at[of[i] + 1] : n;
            place[i] = first;
            for (uint32_t j = first; j < end; ++j) place[i] += sh.pick.list[j] > mine[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            if (t + i * kThreads < n) sh.pick.list[place[i]] = mine[i];
        __syncthreads();
    }
    // running masses
    uint64_t m[kEach], in = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int at = t * kEach + i;
        m[i] = at < n ? w(static_cast<uint32_t>(sh.pick.list[at] >> 32)) : 0;
        in += m[i];
    }
    if (t == 0) sh.listed = 0;
    in = block_scan(in, sh.wave_mass);
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        in += m[i];
        sh.pick.run[t * kEach + i] = in;
    }
    const auto first_of = [&](int r) {  // in the list
        uint32_t f = 0;
        for (int i = 0; i < r; ++i) f += sh.in_range[i];
        return f;
    };
    if (p.m_range >= 0) {               // how many of that range's candidates min_p leaves
        const uint32_t first = first_of(p.m_range), end = first + sh.in_range[p.m_range];
        uint32_t c = 0;
        for (uint32_t i = first + t; i < end; i += kThreads) c += w.share(static_cast<uint32_t>(sh.pick.list[i] >> 32)) >= q.m;
        if (c) atomicAdd(&sh.listed, c);
    }
    __syncthreads();
    if (wave) return;
    const auto run = [&](uint32_t i) { return i ? sh.pick.run[i - 1] : 0; };  // of the first i
    // mass up to and with candidate i of the list, in range r
    const auto up_to = [&](uint32_t i, int r) { return p.mass[r] + run(i + 1) - run(first_of(r)); };
    // the listed candidate that holds unit x of the row's mass, and its range: one wave
    int range = 0;
    const auto holder = [&](uint64_t x) -> uint32_t {
        for (int r = 0; r < 4; ++r)
            if (q.few ? r == 0 : p.mass[r] <= x && x < p.end[r]) range = r;
        uint32_t low = first_of(range), count = n - low;
        const uint64_t at = x - p.mass[range] + run(low);
        while (count > 0) {             // the first i with run(i + 1) > at, 64 steps at a time
            const uint32_t step = (count + 63) / 64;
            const uint32_t i = low + (lane + 1) * step;
            const uint32_t k = __popcll(__ballot(i <= low + count && run(min(i, static_cast<uint32_t>(n))) <= at));
            low += k * step;
            count = step == 1 ? 0 : min(step, count - min(count, k * step));
        }
        return low;
    };
    uint64_t total = q.few ? run(n) : p.all;
    if (p.k_range >= 0) total = up_to(first_of(p.k_range) + p.k_at, p.k_range);
    if (q.p < 1.0f) {
        const uint32_t i = holder(top_p_place(q.p, total));
        total = up_to(i, range);
    }
    if (p.m_range >= 0) {
        const uint32_t first = first_of(p.m_range);
        const uint64_t most = p.mass[p.m_range] + run(first + sh.listed) - run(first);
        total = min(total, max(most, static_cast<uint64_t>(w.unit)));  // the first place stays
    }
    const uint32_t at = holder(drawn_place(q.u, total));
    if (lane == 0) {
        put_token(a, b, static_cast<int>(~static_cast<uint32_t>(sh.pick.list[at])));
        if (a.prob) a.prob[b] = static_cast<float>(static_cast<double>(run(at + 1) - run(at)) / static_cast<double>(total));
    }
}

// The same for up to 64 candidates, a lane's being `mine`, by one wave: sorted by counting.
__device__ __forceinline__ void settle_wave(const SampleArgs& a, int b, const Question& q, int n, uint64_t mine, const Weigher& w, Work& sh) {
    const Plan& p = sh.plan;
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int i = 0; i < n; ++i) before += lane_of(mine, i) > mine;
    __builtin_amdgcn_wave_barrier();    // what the list held has been read
    if (lane < n) sh.pick.list[before] = mine;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    mine = sh.pick.list[min(lane, max(n - 1, 0))];
    const uint32_t key = static_cast<uint32_t>(mine >> 32);
    const uint64_t sums = wave_scan(lane < n ? w(key) : uint64_t{0});
    const auto run = [&](int i) { return i ? lane_of(sums, i - 1) : uint64_t{0}; };  // of the first i
    const float z = w.place(of_key(key));
    const auto in_range = [&](int r) { return __popcll(__ballot(lane < n && z >= p.lo[r] && z < p.hi[r] + 1)); };
    const int f1 = in_range(0), f2 = f1 + in_range(1), f3 = f2 + in_range(2), f4 = f3 + in_range(3);
    const auto first_of = [&](int r) { return r == 0 ? 0 : r == 1 ? f1 : r == 2 ? f2 : r == 3 ? f3 : f4; };
    const auto up_to = [&](int i, int r) { return p.mass[r] + run(i + 1) - run(first_of(r)); };
    int range = 0;
    const auto holder = [&](uint64_t x) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (q.few ? r == 0 : p.mass[r] <= x && x < p.end[r]) range = r;
        const uint64_t at = x - p.mass[range] + run(first_of(range));
        return min(__popcll(__ballot(lane < n && sums <= at)), n - 1);
    };
    uint64_t total = q.few ? run(n) : p.all;
    if (p.k_range >= 0) total = up_to(first_of(p.k_range) + p.k_at, p.k_range);
    if (q.p < 1.0f) {
        const int i = holder(top_p_place(q.p, total));
        total = up_to(i, range);
    }
    if (p.m_range >= 0) {
        const int f = first_of(p.m_range), e = first_of(p.m_range + 1);
        const int c = __popcll(__ballot(lane >= f && lane < e && w.share(key) >= q.m));
        total = min(total, max(p.mass[p.m_range] + run(f + c) - run(f), static_cast<uint64_t>(w.unit)));  // the first place stays
    }
    const int at = holder(drawn_place(q.u, total));
    if (lane == at) {
        put_token(a, b, static_cast<int>(~static_cast<uint32_t>(mine)));
        if (a.prob) a.prob[b] = static_cast<float>(static_cast<double>(w(key)) / static_cast<double>(total));
    }
}

// ---- by descent
// f(logit) for the whole row, with few copies of f: the next four are on their way while f has these.
template <typename F>
__device__ __forceinline__ void each_of_row(const float* x, int V, const F& f) {
    constexpr int kBatch = 4;
    float l[2][kBatch];
    const auto load = [&](float (&to)[kBatch], int j) {
#pragma unroll
        for (int n = 0; n < kBatch; ++n) to[n] = x[min(j + n * kThreads, V - 1)];
    };
    load(l[0], threadIdx.x);
#pragma unroll 1
    for (int j = threadIdx.x; j < V; j += kBatch * kThreads) {
        load(l[1], j + kBatch * kThreads);
#pragma unroll
        for (int n = 0; n < kBatch; ++n)
            if (j + n * kThreads < V) f(l[0][n]);
#pragma unroll
        for (int n = 0; n < kBatch; ++n) l[0][n] = l[1][n];
    }
}

// A place in the ranking: the candidates with larger keys, and `nth` with the same key, are before it.
struct Place {
    uint32_t key, nth;
    uint64_t mass;                      // of the larger keys
};
// The place that holds unit `left` of the mass (by_mass) or has `left` candidates before it. There is one. The key's first
// twelve bits, the next, and the last eight, each by counts and masses of what agrees so far; a thread adds
// those of equal bits in a row at once, as a row of equal logits would wait for one place.
__device__ __forceinline__ Place find(const float* x, int V, const Weigher& w, uint64_t left, bool by_mass, Work& sh) {
    static_assert(kBins >= 4096);
    Place p{0, 0, 0};
#pragma unroll 1
    for (int shift = 20; shift >= 0; shift = shift == 20 ? 8 : shift - 8) {
        const int bits = shift ? 12 : 8;
        const uint32_t last = (1u << bits) - 1, all = shift == 20 ? 0 : ~0u;
        __syncthreads();
        clear_bins(sh);
        __syncthreads();
        uint32_t place = 0, n = 0;      // of the candidates not yet added
        uint64_t m = 0;
        const auto add = [&] {
            if (n) atomicAdd(&sh.bins.count[place], n);
            if (m) atomicAdd(reinterpret_cast<unsigned long long*>(&sh.bins.mass[place]), static_cast<unsigned long long>(m));
        };
        each_of_row(x, V, [&](float l) {
            const uint32_t k = key_of(l);
            if ((k >> shift >> bits & all) != p.key) return;
            const uint32_t to = last - (k >> shift & last);  // larger keys first
            if (to != place) {
                add();
                place = to, n = 0, m = 0;
            }
            ++n, m += w(k);
        });
        add();
        __syncthreads();
        add_up(sh);
        const int bin = by_mass ? bin_of<true>(left, sh) : bin_of<false>(left, sh);
        left -= by_mass ? sh.bins.mass[bin] : sh.bins.count[bin];
        p.mass += sh.bins.mass[bin];
        p.key = p.key << bits | (last - bin);
    }
    const uint64_t each = by_mass ? w(p.key) : 1;
    p.nth = static_cast<uint32_t>(each ? left / each : 0);
    return p;
}

// The places by descent, for rows whose open bins hold too many candidates, or next to temperature 0. One workgroup reads the
// row three times a place (one of 151936, top_p 0.95: at a temperature of 100 410 us, all equal 510).
__device__ __forceinline__ void sample_by_descent(const SampleArgs& a, int b, const Question& q, const Weigher& w, Work& sh) {
    const float* x = a.logits + b * a.ld;
    // the mass of those that have at least `least` of the largest weight
    const auto mass_of = [&](float least) {
        uint64_t s = 0;
        each_of_row(x, a.V, [&](float l) {
            const uint32_t key = key_of(l);
            if (w.share(key) >= least) s += w(key);
        });
        s = wave_scan(s);
        __syncthreads();
        if ((threadIdx.x & 63) == 63) sh.wave_mass[threadIdx.x / 64] = s;
        __syncthreads();
        return lane_of(wave_scan(sh.wave_mass[threadIdx.x & (kThreads / 64 - 1)]), kThreads / 64 - 1);
    };
    const bool by_k = q.k > 0 && q.k < a.V;
    uint64_t total = by_k ? 0 : mass_of(0.0f);
    Place at{};
#pragma unroll 1
    for (int step = 0; step < 3; ++step) {  // the last of top_k, of top_p, the drawn one
        if (step == 0 ? !by_k : step == 1 && !(q.p < 1.0f)) continue;
        if (step == 2 && q.m > 0.0f) total = min(total, max(mass_of(q.m), static_cast<uint64_t>(w.unit)));  // the first place stays
        at = find(x, a.V, w, step == 0 ? q.k - 1 : step == 1 ? top_p_place(q.p, total) : drawn_place(q.u, total), step > 0, sh);
        if (step < 2) total = at.mass + (at.nth + 1ull) * w(at.key);
    }
    // the nth candidate with that key: every wave counts those of a stretch, and the one that has it looks again
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    constexpr int kBatch = 8, kWaves = kThreads / 64;
    const int stretch = ((a.V + kWaves - 1) / kWaves + 63) & ~63, begin = wave * stretch, end = min(begin + stretch, a.V);
    const auto each_vote = [&](const auto& f) {
        for (int i = begin; i < end; i += 64 * kBatch) {
            float l[kBatch];
#pragma unroll
            for (int j = 0; j < kBatch; ++j) l[j] = x[min(i + 64 * j + lane, end - 1)];
#pragma unroll
            for (int j = 0; j < kBatch; ++j)
                if (f(i + 64 * j, __ballot(i + 64 * j + lane < end && key_of(l[j]) == at.key))) return;
        }
    };
    uint32_t n = 0;
    each_vote([&](int, uint64_t vote) { return n += __popcll(vote), false; });
    if (lane == 0) sh.wave_count[wave] = n;
    __syncthreads();
    uint32_t before = 0;
    for (int i = 0; i < wave; ++i) before += sh.wave_count[i];
    if (at.nth < before || at.nth >= before + n) return;
    each_vote([&](int i, uint64_t vote) {
        const uint32_t c = __popcll(vote);
        if (at.nth >= before + c) return before += c, false;
        if ((vote >> lane & 1) && before + __popcll(vote & ((1ull << lane) - 1)) == at.nth) {
            put_token(a, b, i + lane);
            if (a.prob) a.prob[b] = static_cast<float>(static_cast<double>(w(at.key)) / static_cast<double>(total));
        }
        return true;
    });
}

__device__ __forceinline__ int slice_begin(int V, int slices, int i) {
    return i == slices ? V : static_cast<int>(static_cast<int64_t>(V) * i / slices) & ~3;
}

__global__ __launch_bounds__(kThreads) void sample_top_kernel(SampleArgs a, int slices, uint64_t* tops, uint32_t* parts, Row* rows) {
    __shared__ uint64_t waves[kThreads / 64];
    __shared__ float spread[kThreads];
    const int b = blockIdx.y, s = blockIdx.x;
    Row& r = rows[b];
    for (int i = s * kThreads + threadIdx.x; i < kBins; i += slices * kThreads) r.mass[i] = 0, r.count[i] = 0;
    if (s == 0 && threadIdx.x == 0) r.listed = 0, r.counted = 0, r.gathered = 0, r.done = 0;
    if (!(a.temperature[b] >= 0.0f)) return;  // an empty place
    const uint64_t top =
        slice_top(a.logits + b * a.ld, slice_begin(a.V, slices, s), slice_begin(a.V, slices, s + 1), a.temperature[b] == 0.0f, waves,
                  parts + (static_cast<int64_t>(b) * slices + s) * kParts, spread);
    if (threadIdx.x == 0) tops[b * slices + s] = top;
}

// Whether this workgroup is the last of the row's to come here. What the workgroups leave each other are atomic additions
// and shared_store's alone, which are done, where all look, once their wave has waited for them; every wave does before
// the barrier, behind which the ticket is drawn. So a workgroup that draws the last ticket finds, by atomic reads
// (shared_load), all of the others', and the ticket needs no release or acquire, which would write back and drop the
// whole second cache. Plain stores and loads would need them: those of a row's plan go to the next launch.
__device__ __forceinline__ bool last_of(uint32_t* ticket, int slices, Work& sh) {
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vector memory, nothing outstanding
    __syncthreads();
    if (threadIdx.x == 0)
        sh.last = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == static_cast<uint32_t>(slices) - 1;
    __syncthreads();
    return sh.last;
}

// The slice's candidates of the open bins, to the row's list; the row's last workgroup settles it. True for that one
// where they were too many.
__device__ __forceinline__ bool gather_and_settle(const SampleArgs& a, int b, int i, int e, int slices, const Question& q, const Weigher& w, Row& r, Work& sh) {
    gather(a.logits + b * a.ld, i, e, w, sh.plan, sh);
    __syncthreads();
    const uint32_t own = sh.listed;
    if (threadIdx.x == 0 && own) sh.base = atomicAdd(&r.listed, own);
    __syncthreads();
    for (uint32_t j = threadIdx.x; j < own && sh.base + j < kList; j += kThreads) shared_store(&r.list[sh.base + j], sh.pick.list[j]);
    if (!last_of(&r.gathered, slices, sh)) return false;
    const uint32_t n = shared_load(&r.listed);
    if (n > kList) return true;
    if (n <= 64) {
        const uint32_t lane = threadIdx.x & 63;
        if (threadIdx.x < 64) settle_wave(a, b, q, n, lane < n ? shared_load(&r.list[lane]) : uint64_t{0}, w, sh);
        return false;
    }
    for (uint32_t j = threadIdx.x; j < n; j += kThreads) sh.pick.list[j] = shared_load(&r.list[j]);
    n <= kFew ? settle<kFew / kThreads>(a, b, q, n, w, sh) : settle<kList / kThreads>(a, b, q, n, w, sh);
    return false;
}

// The largest logits of 64 parts of the row are logits of 64 candidates, so the k-th of them is no larger than the row's
// k-th: a top_k of at most 64 has its candidates in that one's bin and above. True with the plan made; false where less
// than k parts have a candidate with weight.
__device__ __forceinline__ bool plan_by_parts(const Question& q, uint32_t key, const Weigher& w, Work& sh) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x / 64;
    sh.part[wave][lane] = key;
    __syncthreads();
    if (wave == 0) {
#pragma unroll
        for (int i = 1; i < kThreads / 64; ++i) key = max(key, sh.part[i][lane]);
        // the first bits of the k-th, bit by bit
        uint32_t bound = 0;
        for (uint32_t bit = 0x80000000u; bit >= 0x1000u; bit >>= 1)
            if (__popcll(__ballot(key >= (bound | bit))) >= q.k) bound |= bit;
        if (lane == 0) {
            const float z = w.place(of_key(bound));
            Plan& p = sh.plan;
            for (int r = 0; r < 4; ++r) p.lo[r] = 0, p.hi[r] = -1, p.mass[r] = 0, p.end[r] = 0;
            p.hi[0] = z < kBins ? static_cast<int>(z) : -1;
            p.all = 0;
            p.k_range = 0, p.m_range = q.m > 0.0f ? 0 : -1, p.k_at = q.k - 1;
            sh.listed = 0;
        }
    }
    __syncthreads();
    return sh.plan.hi[0] >= 0;
}

__global__ __launch_bounds__(kThreads) void sample_count_kernel(SampleArgs a, double unit, int slices, const uint64_t* tops, const uint32_t* parts,
                                                                Row* rows) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    Work& sh = *reinterpret_cast<Work*>(lds);
    const int b = blockIdx.y, s = blockIdx.x;
    // all that is read is asked for before the first of it is used (an empty row's may be anything)
    const float T = a.temperature[b];
    const Question q(a, b);
    uint64_t top = lane_top(tops + b * slices, slices);
    uint32_t part_key = kKeyNone;       // this thread's of the parts
    const uint32_t* own = parts + static_cast<int64_t>(b) * slices * kParts;
    for (int i = threadIdx.x / kParts; i < slices; i += kThreads / kParts) part_key = max(part_key, own[i * kParts + (threadIdx.x & (kParts - 1))]);
    sh.exp.fill();
    if (!(T >= 0.0f)) return;
    const bool by_parts = q.k > 0 && q.k <= kParts;
    top = wave_top(top);
    if (plain_row(a, b, T, top, s == 0 && threadIdx.x == 0) || T < kLeastT) return;
    const Weigher w(static_cast<uint32_t>(top >> 32), T, unit, sh.exp);
    __syncthreads();
    Row& r = rows[b];
    const int begin = slice_begin(a.V, slices, s), end = slice_begin(a.V, slices, s + 1);
    // (one row of 151936, top_k 20: 15.5 us in all, by counts 22.5)
    if (by_parts) {
        if (plan_by_parts(q, part_key, w, sh)) {
            const bool many = gather_and_settle(a, b, begin, end, slices, q, w, r, sh);
            if (threadIdx.x == 0 && sh.last) r.done = many ? 2 : 1;
            return;
        }
        __syncthreads();
    }
    clear_bins(sh);
    __syncthreads();
    count_slice(a.logits + b * a.ld, begin, end, q, w, sh);
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += kThreads) {
        if (sh.bins.count[i]) atomicAdd(&r.count[i], sh.bins.count[i]);
        if (sh.bins.mass[i]) atomicAdd(reinterpret_cast<unsigned long long*>(&r.mass[i]), static_cast<unsigned long long>(sh.bins.mass[i]));
    }
    if (!last_of(&r.counted, slices, sh)) return;
    for (int i = threadIdx.x; i < kBins; i += kThreads) {
        if (q.k) sh.bins.count[i] = shared_load(&r.count[i]);
        if (!q.few) sh.bins.mass[i] = shared_load(&r.mass[i]);
    }
    __syncthreads();
    add_up(sh);
    if (threadIdx.x < 64) {
        make_plan(q, sh);
        if (threadIdx.x == 0) r.plan = sh.plan;
    }
}

__global__ __launch_bounds__(kThreads) void sample_draw_kernel(SampleArgs a, double unit, int slices, const uint64_t* tops, Row* rows) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    Work& sh = *reinterpret_cast<Work*>(lds);
    const int b = blockIdx.y, s = blockIdx.x;
    Row& r = rows[b];
    const uint32_t done = r.done;
    if (done == 1) return;
    // all that is read is asked for before the first of it is used (an empty row's may be anything)
    const float T = a.temperature[b];
    const Question q(a, b);
    const uint32_t plan = threadIdx.x < sizeof(Plan) / 4 ? reinterpret_cast<const uint32_t*>(&r.plan)[threadIdx.x] : 0;
    uint64_t top = lane_top(tops + b * slices, slices);
    sh.exp.fill();
    if (!(T >= 0.0f)) return;
    if (threadIdx.x < sizeof(Plan) / 4) reinterpret_cast<uint32_t*>(&sh.plan)[threadIdx.x] = plan;
    if (threadIdx.x == 0) sh.listed = 0;
    top = wave_top(top);
    if (plain_row(a, b, T, top, false)) return;
    const Weigher w(static_cast<uint32_t>(top >> 32), T, unit, sh.exp);
    __syncthreads();
    // by descent where the open bins hold too many (done is 2 where that is known), and next to temperature 0
    bool descend = (T < kLeastT || done) && s == 0;
    if (T >= kLeastT && !done) descend = gather_and_settle(a, b, slice_begin(a.V, slices, s), slice_begin(a.V, slices, s + 1), slices, q, w, r, sh);
    if (descend) sample_by_descent(a, b, q, w, sh);
}

// a row of one slice
__global__ __launch_bounds__(kThreads) void sample_row_kernel(SampleArgs a, double unit) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    Work& sh = *reinterpret_cast<Work*>(lds);
    const int b = blockIdx.x;
    const float T = a.temperature[b];
    if (!(T >= 0.0f)) return;
    const Question q(a, b);
    const float* x = a.logits + b * a.ld;
    clear_bins(sh);
    sh.exp.fill();
    const uint64_t top = slice_top(x, 0, a.V, T == 0.0f, sh.wave_mass, nullptr, nullptr);
    if (plain_row(a, b, T, top, threadIdx.x == 0)) return;
    const Weigher w(static_cast<uint32_t>(top >> 32), T, unit, sh.exp);
    __syncthreads();
    if (T >= kLeastT) {
        count_slice(x, 0, a.V, q, w, sh);
        __syncthreads();
        add_up(sh);
        if (threadIdx.x < 64) make_plan(q, sh);
        if (threadIdx.x == 0) sh.listed = 0;
        __syncthreads();
        gather(x, 0, a.V, w, sh.plan, sh);
        __syncthreads();
        const uint32_t n = sh.listed;
        if (n <= 64) {
            const uint32_t lane = threadIdx.x & 63;
            if (threadIdx.x < 64) settle_wave(a, b, q, n, lane < n ? sh.pick.list[lane] : 0, w, sh);
            return;
        }
        if (n <= kList) {
            n <= kFew ? settle<kFew / kThreads>(a, b, q, n, w, sh) : settle<kList / kThreads>(a, b, q, n, w, sh);
            return;
        }
        __syncthreads();
    }
    sample_by_descent(a, b, q, w, sh);
}

// Workgroups a row: one for each 4096 logits, up to 256 in all. From 129 rows on each has one, and one launch (in graphs, top_p
// 0.95 of 151936: 128 rows 79 us, 129 95, 256 109).
int sample_slices(int B, int V) { return std::max(1, std::min((V + 4095) / 4096, 256 / std::min(B, 256))); }

}  // namespace

uint64_t sample_workspace_bytes(int B, int V) {
    const int slices = sample_slices(B, V);
    return slices == 1 ? 16 : static_cast<uint64_t>(B) * (sizeof(Row) + (8 + 4 * kParts) * slices);
}

hipError_t launch_sample(const SampleArgs& a, hipStream_t s) {
    int bits = 0;
    while ((1ll << bits) < a.V) ++bits;
    const double unit = ldexp(1.0, std::min(62 - bits, 50));
    const int slices = sample_slices(a.B, a.V);
    static AllowedLds allowed_row, allowed_count, allowed_draw;
    if (slices == 1) {
        const hipError_t e = allowed_row(reinterpret_cast<const void*>(sample_row_kernel), sizeof(Work));
        if (e != hipSuccess) return e;
        klaunch(sample_row_kernel, dim3(a.B), dim3(kThreads), sizeof(Work), s, a, unit);
        return hipGetLastError();
    }
    hipError_t e = allowed_count(reinterpret_cast<const void*>(sample_count_kernel), sizeof(Work));
    if (e == hipSuccess) e = allowed_draw(reinterpret_cast<const void*>(sample_draw_kernel), sizeof(Work));
    if (e != hipSuccess) return e;
    Row* rows = static_cast<Row*>(a.ws);
    uint64_t* tops = reinterpret_cast<uint64_t*>(rows + a.B);
    uint32_t* parts = reinterpret_cast<uint32_t*>(tops + static_cast<int64_t>(a.B) * slices);
    const dim3 grid(slices, a.B);
    klaunch(sample_top_kernel, grid, dim3(kThreads), 0, s, a, slices, tops, parts, rows);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    klaunch(sample_count_kernel, grid, dim3(kThreads), sizeof(Work), s, a, unit, slices, static_cast<const uint64_t*>(tops),
            static_cast<const uint32_t*>(parts), rows);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    klaunch(sample_draw_kernel, grid, dim3(kThreads), sizeof(Work), s, a, unit, slices, static_cast<const uint64_t*>(tops), rows);
    return hipGetLastError();
}

}  // namespace q35k
