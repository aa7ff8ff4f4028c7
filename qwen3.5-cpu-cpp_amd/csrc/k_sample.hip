// Sampling with temperature, top-k, top-p and min-p from one uniform number a row (q35_sample).
//
// Candidates are ranked by logit, equal ones by id. Every filter keeps a prefix of the ranking, so what is
// kept is a count of first places, and the draw is a place too: the one in whose share of the kept mass the
// number falls. Weights are exp((l - max) / T) in 64 bits, held as whole multiples of 2^-S (2^S times the number
// of candidates stays below 2^62): sums are exact, so they do not depend on their order, and places next to
// each other in mass are told apart down to 2^-S of the largest weight.
//
// A row is cut into slices, a workgroup each. The first launch finds the largest logit; the second counts
// candidates and mass by bins of 1/128 of (max - l) / T, down to 36, below which weights are 0; the third
// reads off which bins the borders and the draw may lie in (a border that is known to a bin leaves the next one
// open to as much mass, so mostly to a bin as well), gathers their candidates, and the workgroup that is done
// last sorts those and finds the exact places. Rows of one slice take one launch. Where the open bins
// hold more than kList candidates (thousands of equal logits), it finds the places by radix descent over
// the row instead.
#include "dev_common.hpp"
#include "launch_q4.hpp"

namespace q35k {
namespace {

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

constexpr int kBins = 36 * 128;  // and one for what has no weight

struct Weigher {
    double top, rt, unit;
    bool inf;
    __device__ Weigher(uint32_t key, float T, double unit_) : top(of_key(key)), rt(1.0 / static_cast<double>(T)), unit(unit_), inf(key == kKeyInf) {}
    // (max - l) / T
    __device__ double depth(uint32_t key) const {
        if (inf) return key == kKeyInf ? 0.0 : INFINITY;
        if (key == kKeyNone) return INFINITY;
        const double d = top - static_cast<double>(of_key(key));
        return d == 0.0 ? 0.0 : d * rt;
    }
    static __device__ int bin(double depth) { return static_cast<int>(fmin(depth * 128.0, static_cast<double>(kBins))); }
    // the weight in 64 bits, of the largest
    __device__ double share(uint32_t key) const {
        const double z = depth(key);
        return z < 36.0 ? exp(-z) : 0.0;
    }
    __device__ uint64_t units(double depth) const { return depth < 36.0 ? static_cast<uint64_t>(rint(exp(-depth) * unit)) : 0; }
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

// A place in the ranking: the candidates with larger keys, and `nth` with the same key, are before it.
struct Place {
    uint32_t key;
    uint32_t nth;
    uint64_t count, mass;  // of the larger keys
};

struct Shared {
    uint32_t count[256];
    uint64_t mass[256];
    uint64_t red[kThreads / 64];
    Place place;
    uint64_t left;
    uint32_t prefix;
};

__device__ uint64_t block_sum_u64(uint64_t v, Shared& sh) {
    for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.red[threadIdx.x / 64] = v;
    __syncthreads();
    uint64_t t = 0;
    for (int i = 0; i < kThreads / 64; ++i) t += sh.red[i];
    return t;
}

// The place that holds unit `at` of the mass (BY_MASS) or has `at` candidates before it. There is one.
template <bool BY_MASS>
__device__ Place find(const float* x, int V, const Weigher& w, uint64_t at, Shared& sh) {
    uint32_t prefix = 0;
    Place p{0, 0, 0, 0};
    uint64_t left = at;
    for (int shift = 24; shift >= 0; shift -= 8) {
        __syncthreads();
        if (threadIdx.x < 256) sh.count[threadIdx.x] = 0, sh.mass[threadIdx.x] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < V; i += kThreads) {
            const uint32_t k = key_of(x[i]);
            if (shift < 24 && (k >> (shift + 8)) != prefix) continue;
            atomicAdd(&sh.count[k >> shift & 255], 1u);
            const uint64_t m = w(k);
            if (m) atomicAdd(reinterpret_cast<unsigned long long*>(&sh.mass[k >> shift & 255]), static_cast<unsigned long long>(m));
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            int d = 255;
            for (; d > 0; --d) {
                const uint64_t n = BY_MASS ? sh.mass[d] : sh.count[d];
                if (left < n) break;
                left -= n;
                p.count += sh.count[d];
                p.mass += sh.mass[d];
            }
            sh.place = p;
            sh.left = left;
            sh.prefix = prefix << 8 | static_cast<uint32_t>(d);
        }
        __syncthreads();
        p = sh.place;
        left = sh.left;
        prefix = sh.prefix;
    }
    p.key = prefix;
    const uint64_t each = BY_MASS ? w(prefix) : 1;
    p.nth = static_cast<uint32_t>(each ? left / each : 0);
    return p;
}

// The places by descent over the whole row: for rows whose open bins hold too many candidates.
__device__ void sample_by_descent(const SampleArgs& a, int b, uint32_t top, const Weigher& w, Shared& sh) {
    const float* x = a.logits + b * a.ld;
    uint64_t total;
    const int k = a.top_k ? a.top_k[b] : 0;
    const float tp = a.top_p ? a.top_p[b] : 1.0f, mp = a.min_p ? a.min_p[b] : 0.0f;
    uint32_t last = kKeyNone;  // the last key that is kept
    if (k > 0 && k < a.V) {
        const Place p = find<false>(x, a.V, w, k - 1, sh);
        last = p.key;
        total = p.mass + (p.nth + 1ull) * w(p.key);
    } else {
        uint64_t s = 0;
        for (int i = threadIdx.x; i < a.V; i += kThreads) s += w(key_of(x[i]));
        total = block_sum_u64(s, sh);
    }
    if (tp < 1.0f) {
        const Place p = find<true>(x, a.V, w, top_p_place(tp, total), sh);
        last = p.key;
        total = p.mass + (p.nth + 1ull) * w(p.key);
    }
    if (mp > 0.0f && !(w.share(last) >= mp)) {
        uint64_t s = 0;
        for (int i = threadIdx.x; i < a.V; i += kThreads) {
            const uint32_t key = key_of(x[i]);
            if (w.share(key) >= mp) s += w(key);
        }
        total = max(block_sum_u64(s, sh), w(top));  // the first place stays
    }
    const Place at = find<true>(x, a.V, w, drawn_place(a.u[b], total), sh);
    // the nth candidate with that key
    uint32_t seen = 0;
    for (int i0 = 0; i0 < a.V; i0 += kThreads) {
        const int i = i0 + threadIdx.x;
        const bool same = i < a.V && key_of(x[i]) == at.key;
        const uint64_t vote = __ballot(same);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) sh.red[threadIdx.x / 64] = __popcll(vote);
        __syncthreads();
        uint32_t before = seen, all = 0;
        for (int j = 0; j < kThreads / 64; ++j) {
            if (j < static_cast<int>(threadIdx.x / 64)) before += static_cast<uint32_t>(sh.red[j]);
            all += static_cast<uint32_t>(sh.red[j]);
        }
        before += __popcll(vote & ((1ull << (threadIdx.x & 63)) - 1));
        if (same && before == at.nth) {
            a.token[b] = i;
            if (a.prob) a.prob[b] = static_cast<float>(static_cast<double>(w(at.key)) / static_cast<double>(total));
        }
        seen += all;
        if (seen > at.nth) return;  // the same for every thread
    }
}

// ---- by bins
constexpr int kList = 4096;             // candidates of the open bins
constexpr int kPer = (kBins + 1 + kThreads - 1) / kThreads;

// a candidate in the ranking's order: larger ones first
__device__ __forceinline__ uint64_t entry_of(uint32_t key, int id) { return static_cast<uint64_t>(key) << 32 | static_cast<uint32_t>(~id); }

// What a row's workgroups share, in the workspace. Cleared by the first launch.
struct Row {
    uint64_t mass[kBins];
    uint32_t count[kBins];
    uint32_t listed, done;
    uint64_t list[kList];
};

struct Work {
    union {
        struct {
            uint64_t mass[kBins + 2];   // by bin, then of the bins before
            uint32_t count[kBins + 2];
            uint64_t list[kList], run[kList];
            uint64_t wave_mass[kThreads / 64];
            uint32_t wave_count[kThreads / 64];
            uint64_t found;
            uint32_t listed, last;
        } s;
        Shared descent;
    };
};

// largest entry of ids [i, e)
__device__ uint64_t slice_top(const float* x, int i, int e, Work& sh) {
    uint64_t top = 0;
    for (int j = i + threadIdx.x; j < e; j += kThreads) top = max(top, entry_of(key_of(x[j]), j));
    for (int d = 1; d < 64; d <<= 1) top = max(top, static_cast<uint64_t>(__shfl_xor(static_cast<unsigned long long>(top), d)));
    if ((threadIdx.x & 63) == 0) sh.s.wave_mass[threadIdx.x / 64] = top;
    __syncthreads();
    for (int j = 0; j < kThreads / 64; ++j) top = max(top, sh.s.wave_mass[j]);
    __syncthreads();
    return top;
}

// greedy and empty rows, and rows without a candidate: true if there is nothing more to do
__device__ bool plain_row(const SampleArgs& a, int b, float T, uint64_t top, bool writes) {
    const uint32_t key = static_cast<uint32_t>(top >> 32);
    if (T > 0.0f && key != kKeyNone) return false;
    if (writes && T >= 0.0f) {
        a.token[b] = key == kKeyNone ? -1 : static_cast<int>(~static_cast<uint32_t>(top));
        if (a.prob) a.prob[b] = key == kKeyNone ? 0.0f : 1.0f;
    }
    return true;
}

__device__ void clear_bins(Work& sh) {
    for (int i = threadIdx.x; i < kBins + 2; i += kThreads) sh.s.mass[i] = 0, sh.s.count[i] = 0;
}
__device__ void count_slice(const float* x, int i, int e, const Weigher& w, Work& sh) {
    for (int j = i + threadIdx.x; j < e; j += kThreads) {
        const double z = w.depth(key_of(x[j]));
        if (!(z < 36.0)) continue;
        const int bin = Weigher::bin(z);
        atomicAdd(&sh.s.count[bin], 1u);
        atomicAdd(reinterpret_cast<unsigned long long*>(&sh.s.mass[bin]), static_cast<unsigned long long>(w.units(z)));
    }
}

// bins' counts and masses become those of the bins before; the totals stand behind the last
__device__ void add_up(Work& sh) {
    const int t = threadIdx.x, lane = t & 63, wave = t / 64;
    uint64_t m = 0;
    uint32_t n = 0;
    for (int i = 0; i < kPer; ++i) {
        const int b = t * kPer + i;
        if (b < kBins) m += sh.s.mass[b], n += sh.s.count[b];
    }
    uint64_t im = m;
    uint32_t in = n;
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t om = __shfl_up(static_cast<unsigned long long>(im), d);
        const uint32_t on = __shfl_up(in, d);
        if (lane >= d) im += om, in += on;
    }
    if (lane == 63) sh.s.wave_mass[wave] = im, sh.s.wave_count[wave] = in;
    __syncthreads();
    im -= m, in -= n;
    for (int i = 0; i < wave; ++i) im += sh.s.wave_mass[i], in += sh.s.wave_count[i];
    for (int i = 0; i < kPer; ++i) {
        const int b = t * kPer + i;
        if (b > kBins) break;
        const uint64_t bm = sh.s.mass[b];
        const uint32_t bn = sh.s.count[b];
        sh.s.mass[b] = im, sh.s.count[b] = in;
        if (b < kBins) im += bm, in += bn;
    }
    __syncthreads();
}

// the bin that holds unit x of the mass (x below the total) or candidate x
template <bool BY_MASS>
__device__ int bin_of(uint64_t x, Work& sh) {
    for (int b = threadIdx.x; b < kBins; b += kThreads) {
        const uint64_t lo = BY_MASS ? sh.s.mass[b] : sh.s.count[b], hi = BY_MASS ? sh.s.mass[b + 1] : sh.s.count[b + 1];
        if (lo <= x && x < hi) sh.s.found = b;
    }
    __syncthreads();
    const int b = static_cast<int>(sh.s.found);
    __syncthreads();
    return b;
}

// Bins that are open: up to four ranges [lo, hi], in order, apart.
struct Open {
    int lo[4], hi[4], n = 0;
    __device__ void add(int l, int h) {
        for (int i = 0; i < n;) {       // ranges that meet become one
            if (l <= hi[i] + 1 && lo[i] <= h + 1) {
                l = min(l, lo[i]), h = max(h, hi[i]);
                --n;
                for (int j = i; j < n; ++j) lo[j] = lo[j + 1], hi[j] = hi[j + 1];
            } else {
                ++i;
            }
        }
        int i = n++;
        for (; i > 0 && lo[i - 1] > l; --i) lo[i] = lo[i - 1], hi[i] = hi[i - 1];
        lo[i] = l, hi[i] = h;
    }
    __device__ bool holds(int b) const {
        bool in = false;
        for (int i = 0; i < n; ++i) in |= lo[i] <= b && b <= hi[i];
        return in;
    }
    // candidates of the open bins before bin b
    __device__ uint32_t before(int b, const Work& sh) const {
        uint32_t c = 0;
        for (int i = 0; i < n; ++i)
            if (lo[i] < b) c += sh.s.count[min(hi[i] + 1, b)] - sh.s.count[lo[i]];
        return c;
    }
};

// What is asked of a row, and where by its bins the answers may lie.
struct Question {
    int k;                              // 0: no top_k that leaves weight out
    float tp, mp, u;
    int bk, bm_lo, bm_hi;
    Open open;
};
__device__ Question ask(const SampleArgs& a, int b, Work& sh) {
    Question q;
    const int k = a.top_k ? a.top_k[b] : 0;
    q.k = k > 0 && static_cast<uint32_t>(k) < sh.s.count[kBins] ? k : 0;
    q.tp = a.top_p ? a.top_p[b] : 1.0f;
    q.mp = a.min_p ? a.min_p[b] : 0.0f;
    q.u = a.u[b];
    q.bk = q.bm_lo = q.bm_hi = 0;
    uint64_t lo = sh.s.mass[kBins], hi = lo;  // the total lies within
    if (q.k) {
        q.bk = bin_of<false>(q.k - 1, sh);
        q.open.add(q.bk, q.bk);
        lo = max(sh.s.mass[q.bk], uint64_t{1}), hi = sh.s.mass[q.bk + 1];
    }
    if (q.tp < 1.0f) {
        const int l = bin_of<true>(top_p_place(q.tp, lo), sh), h = bin_of<true>(top_p_place(q.tp, hi), sh);
        q.open.add(l, h);
        lo = max(sh.s.mass[l], uint64_t{1}), hi = min(hi, sh.s.mass[h + 1]);
    }
    if (q.mp > 0.0f) {
        // depths next to the border are compared one by one
        const double z = q.mp < 1.0f ? -log(static_cast<double>(q.mp)) : 0.0;
        q.bm_lo = Weigher::bin(fmax(z - 1e-6, 0.0)), q.bm_hi = min(Weigher::bin(z + 1e-6), kBins - 1);
        if (q.bm_lo < kBins) {
            q.open.add(q.bm_lo, q.bm_hi);
            lo = min(lo, max(sh.s.mass[q.bm_lo], uint64_t{1})), hi = min(hi, sh.s.mass[q.bm_hi + 1]);
        } else {
            q.mp = 0.0f;                // only what has no weight is left out
        }
    }
    q.open.add(bin_of<true>(drawn_place(q.u, lo), sh), bin_of<true>(drawn_place(q.u, hi), sh));
    return q;
}

// ids [i, e) of the open bins, to a list
__device__ void gather(const float* x, int i, int e, const Weigher& w, const Open& open, uint64_t* list, uint32_t* listed) {
    for (int j = i + threadIdx.x; j < e; j += kThreads) {
        const uint32_t key = key_of(x[j]);
        const double z = w.depth(key);
        if (z < 36.0 && open.holds(Weigher::bin(z))) list[atomicAdd(listed, 1u)] = entry_of(key, j);
    }
}

// The exact places, from the n candidates of the open bins in sh.s.list.
__device__ void settle(const SampleArgs& a, int b, int n, const Weigher& w, const Question& q, Work& sh) {
    const int t = threadIdx.x, lane = t & 63, wave = t / 64;
    int size = 64;
    while (size < n) size *= 2;
    for (int i = n + t; i < size; i += kThreads) sh.s.list[i] = 0;
    __syncthreads();
    // bitonic sort, largest first
    for (int k = 2; k <= size; k *= 2)
        for (int j = k / 2; j > 0; j /= 2) {
            for (int p = t; p < size / 2; p += kThreads) {
                const int i = 2 * p - (p & (j - 1));
                const uint64_t x = sh.s.list[i], y = sh.s.list[i + j];
                if ((x < y) == ((i & k) == 0)) sh.s.list[i] = y, sh.s.list[i + j] = x;
            }
            __syncthreads();
        }
    // running masses
    constexpr int kEach = kList / kThreads;
    uint64_t m[kEach], sum = 0;
    for (int i = 0; i < kEach; ++i) {
        const int at = t * kEach + i;
        m[i] = at < n ? w(static_cast<uint32_t>(sh.s.list[at] >> 32)) : 0;
        sum += m[i];
    }
    uint64_t in = sum;
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t o = __shfl_up(static_cast<unsigned long long>(in), d);
        if (lane >= d) in += o;
    }
    if (lane == 63) sh.s.wave_mass[wave] = in;
    __syncthreads();
    in -= sum;
    for (int i = 0; i < wave; ++i) in += sh.s.wave_mass[i];
    for (int i = 0; i < kEach; ++i) {
        in += m[i];
        sh.s.run[t * kEach + i] = in;
    }
    __syncthreads();
    const auto run = [&](uint32_t i) { return i ? sh.s.run[i - 1] : 0; };  // of the first i
    // the listed candidate that holds unit x of the row's mass
    const auto holder = [&](uint64_t x) {
        const int bin = bin_of<true>(x, sh);
        const uint32_t first = q.open.before(bin, sh);
        const uint64_t at = x - sh.s.mass[bin] + run(first);
        for (int i = t; i < n; i += kThreads)
            if (run(i) <= at && at < run(i + 1)) sh.s.found = i | static_cast<uint64_t>(bin) << 32;
        __syncthreads();
        const uint64_t f = sh.s.found;
        __syncthreads();
        return f;
    };
    const auto up_to = [&](uint32_t i, int bin) { return sh.s.mass[bin] + run(i + 1) - run(q.open.before(bin, sh)); };
    uint64_t total = sh.s.mass[kBins];
    if (q.k) total = up_to(q.open.before(q.bk, sh) + (q.k - 1 - sh.s.count[q.bk]), q.bk);
    if (q.tp < 1.0f) {
        const uint64_t f = holder(top_p_place(q.tp, total));
        total = up_to(static_cast<uint32_t>(f), static_cast<int>(f >> 32));
    }
    if (q.mp > 0.0f) {
        const uint32_t first = q.open.before(q.bm_lo, sh), end = q.open.before(q.bm_hi + 1, sh);
        if (t == 0) sh.s.listed = 0;
        __syncthreads();
        uint32_t c = 0;
        for (uint32_t i = first + t; i < end; i += kThreads) c += w.share(static_cast<uint32_t>(sh.s.list[i] >> 32)) >= q.mp;
        if (c) atomicAdd(&sh.s.listed, c);
        __syncthreads();
        const uint64_t most = sh.s.mass[q.bm_lo] + run(first + sh.s.listed) - run(first);
        total = min(total, max(most, static_cast<uint64_t>(w.unit)));  // the first place stays
    }
    const uint32_t at = static_cast<uint32_t>(holder(drawn_place(q.u, total)));
    if (t == 0) {
        const uint64_t e = sh.s.list[at];
        a.token[b] = static_cast<int>(~static_cast<uint32_t>(e));
        if (a.prob) a.prob[b] = static_cast<float>(static_cast<double>(run(at + 1) - run(at)) / static_cast<double>(total));
    }
}

__device__ __forceinline__ int slice_begin(int V, int slices, int i) { return static_cast<int>(static_cast<int64_t>(V) * i / slices); }

__global__ __launch_bounds__(kThreads) void sample_top_kernel(SampleArgs a, int slices, uint64_t* tops, Row* rows) {
    __shared__ Work sh;
    const int b = blockIdx.y, s = blockIdx.x;
    Row& r = rows[b];
    for (int i = s * kThreads + threadIdx.x; i < kBins; i += slices * kThreads) r.mass[i] = 0, r.count[i] = 0;
    if (s == 0 && threadIdx.x == 0) r.listed = 0, r.done = 0;
    if (!(a.temperature[b] >= 0.0f)) return;  // an empty place
    const uint64_t top = slice_top(a.logits + b * a.ld, slice_begin(a.V, slices, s), slice_begin(a.V, slices, s + 1), sh);
    if (threadIdx.x == 0) tops[b * slices + s] = top;
}

__device__ uint64_t row_top(const uint64_t* tops, int slices) {
    uint64_t top = 0;
    for (int i = 0; i < slices; ++i) top = max(top, tops[i]);
    return top;
}

__global__ __launch_bounds__(kThreads) void sample_count_kernel(SampleArgs a, double unit, int slices, const uint64_t* tops, Row* rows) {
    __shared__ Work sh;
    const int b = blockIdx.y, s = blockIdx.x;
    const float T = a.temperature[b];
    if (!(T > 0.0f)) return;
    const uint64_t top = row_top(tops + b * slices, slices);
    if (plain_row(a, b, T, top, false)) return;
    const Weigher w(static_cast<uint32_t>(top >> 32), T, unit);
    clear_bins(sh);
    __syncthreads();
    count_slice(a.logits + b * a.ld, slice_begin(a.V, slices, s), slice_begin(a.V, slices, s + 1), w, sh);
    __syncthreads();
    Row& r = rows[b];
    for (int i = threadIdx.x; i < kBins; i += kThreads)
        if (sh.s.count[i]) {
            atomicAdd(&r.count[i], sh.s.count[i]);
            atomicAdd(reinterpret_cast<unsigned long long*>(&r.mass[i]), static_cast<unsigned long long>(sh.s.mass[i]));
        }
}

__global__ __launch_bounds__(kThreads) void sample_draw_kernel(SampleArgs a, double unit, int slices, const uint64_t* tops, Row* rows) {
    __shared__ Work sh;
    const int b = blockIdx.y, s = blockIdx.x;
    const float T = a.temperature[b];
    if (!(T >= 0.0f)) return;
    const uint64_t top = row_top(tops + b * slices, slices);
    if (plain_row(a, b, T, top, s == 0 && threadIdx.x == 0)) return;
    const Weigher w(static_cast<uint32_t>(top >> 32), T, unit);
    Row& r = rows[b];
    for (int i = threadIdx.x; i < kBins; i += kThreads) sh.s.mass[i] = r.mass[i], sh.s.count[i] = r.count[i];
    __syncthreads();
    add_up(sh);
    const Question q = ask(a, b, sh);
    const uint32_t n = q.open.before(kBins, sh);
    if (n <= kList) gather(a.logits + b * a.ld, slice_begin(a.V, slices, s), slice_begin(a.V, slices, s + 1), w, q.open, r.list, &r.listed);
    // the workgroup that is done last sees what all have listed
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) sh.s.last = atomicAdd(&r.done, 1u) == static_cast<uint32_t>(slices) - 1;
    __syncthreads();
    if (!sh.s.last) return;
    __threadfence();
    if (n > kList) {
        __syncthreads();
        sample_by_descent(a, b, static_cast<uint32_t>(top >> 32), w, sh.descent);
        return;
    }
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) sh.s.list[i] = r.list[i];
    settle(a, b, n, w, q, sh);
}

// a row of one slice
__global__ __launch_bounds__(kThreads) void sample_row_kernel(SampleArgs a, double unit) {
    __shared__ Work sh;
    const int b = blockIdx.x;
    const float T = a.temperature[b];
    if (!(T >= 0.0f)) return;
    const float* x = a.logits + b * a.ld;
    clear_bins(sh);
    const uint64_t top = slice_top(x, 0, a.V, sh);
    if (plain_row(a, b, T, top, threadIdx.x == 0)) return;
    const Weigher w(static_cast<uint32_t>(top >> 32), T, unit);
    count_slice(x, 0, a.V, w, sh);
    __syncthreads();
    add_up(sh);
    const Question q = ask(a, b, sh);
    const uint32_t n = q.open.before(kBins, sh);
    if (n > kList) {
        __syncthreads();
        sample_by_descent(a, b, static_cast<uint32_t>(top >> 32), w, sh.descent);
        return;
    }
    if (threadIdx.x == 0) sh.s.listed = 0;
    __syncthreads();
    gather(x, 0, a.V, w, q.open, sh.s.list, &sh.s.listed);
    __syncthreads();
    settle(a, b, n, w, q, sh);
}

int sample_slices(int B, int V) { return std::max(1, std::min((V + 4095) / 4096, 512 / std::min(B, 512))); }

}  // namespace

uint64_t sample_workspace_bytes(int B, int V) {
    const int slices = sample_slices(B, V);
    return slices == 1 ? 16 : static_cast<uint64_t>(B) * (sizeof(Row) + 8 * slices);
}

hipError_t launch_sample(const SampleArgs& a, hipStream_t s) {
    int bits = 0;
    while ((1ll << bits) < a.V) ++bits;
    const double unit = ldexp(1.0, std::min(62 - bits, 50));
    const int slices = sample_slices(a.B, a.V);
    if (slices == 1) {
        klaunch(sample_row_kernel, dim3(a.B), dim3(kThreads), 0, s, a, unit);
        return hipGetLastError();
    }
    Row* rows = static_cast<Row*>(a.ws);
    uint64_t* tops = reinterpret_cast<uint64_t*>(rows + a.B);
    const dim3 grid(slices, a.B);
    klaunch(sample_top_kernel, grid, dim3(kThreads), 0, s, a, slices, tops, rows);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    klaunch(sample_count_kernel, grid, dim3(kThreads), 0, s, a, unit, slices, static_cast<const uint64_t*>(tops), rows);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    klaunch(sample_draw_kernel, grid, dim3(kThreads), 0, s, a, unit, slices, static_cast<const uint64_t*>(tops), rows);
    return hipGetLastError();
}

}  // namespace q35k
