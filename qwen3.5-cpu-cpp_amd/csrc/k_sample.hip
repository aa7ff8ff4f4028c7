// Sampling with temperature, top-k, top-p and min-p from one uniform number a row (q35_sample).
//
// Candidates are ranked by logit, equal ones by id. Every filter keeps a prefix of the ranking, so what is
// kept is a count of first places, and the draw is a place too: the one in whose share of the kept mass the
// number falls. All are found by radix descent over the logits' ordered bits, with a count and a mass per
// digit. Weights are exp((l - max) / T) in 64 bits, held as whole multiples of 2^-S (2^S times the number
// of candidates stays below 2^62): sums are exact, so they do not depend on their order, and places next to
// each other in mass are told apart down to 2^-S of the largest weight.
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

struct Weigher {
    double top, t, unit;
    bool inf;
    __device__ uint64_t operator()(uint32_t key) const {
        if (inf) return key == kKeyInf ? static_cast<uint64_t>(unit) : 0;
        if (key == kKeyNone) return 0;
        return static_cast<uint64_t>(rint(share(key) * unit));
    }
    // the weight in 64 bits, of the largest
    __device__ double share(uint32_t key) const {
        if (inf) return key == kKeyInf ? 1.0 : 0.0;
        if (key == kKeyNone) return 0.0;
        const double d = static_cast<double>(of_key(key)) - top;
        return d == 0.0 ? 1.0 : exp(d / t);
    }
};

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

__global__ __launch_bounds__(kThreads) void sample_kernel(SampleArgs a, double unit) {
    __shared__ Shared sh;
    const int b = blockIdx.x;
    const float* x = a.logits + b * a.ld;
    const float T = a.temperature[b];
    if (!(T >= 0.0f)) return;  // an empty place
    uint32_t top = 0;
    for (int i = threadIdx.x; i < a.V; i += kThreads) top = max(top, key_of(x[i]));
    for (int d = 1; d < 64; d <<= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), d)));
    if ((threadIdx.x & 63) == 0) sh.red[threadIdx.x / 64] = top;
    __syncthreads();
    for (int i = 0; i < kThreads / 64; ++i) top = max(top, static_cast<uint32_t>(sh.red[i]));
    __syncthreads();
    if (top == kKeyNone) {  // nothing to choose
        if (threadIdx.x == 0) {
            a.token[b] = -1;
            if (a.prob) a.prob[b] = 0.0f;
        }
        return;
    }
    const Weigher w{static_cast<double>(of_key(top)), static_cast<double>(T), unit, top == kKeyInf};
    Place at{top, 0, 0, 0};
    double prob = 1.0;
    if (T > 0.0f) {
        uint64_t total;
        const int k = a.top_k ? a.top_k[b] : 0;
        const float tp = a.top_p ? a.top_p[b] : 1.0f, mp = a.min_p ? a.min_p[b] : 0.0f;
        uint32_t last = kKeyNone;  // the last key that is kept, with `n` candidates of it
        uint64_t n = ~0ull;
        if (k > 0 && k < a.V) {
            const Place p = find<false>(x, a.V, w, k - 1, sh);
            last = p.key, n = p.nth + 1ull;
            total = p.mass + n * w(p.key);
        } else {
            uint64_t s = 0;
            for (int i = threadIdx.x; i < a.V; i += kThreads) s += w(key_of(x[i]));
            total = block_sum_u64(s, sh);
        }
        if (tp < 1.0f) {
            const double want = ceil(static_cast<double>(tp) * static_cast<double>(total));
            const uint64_t pos = want >= 1.0 ? min(static_cast<uint64_t>(want), total) - 1 : 0;
            const Place p = find<true>(x, a.V, w, pos, sh);
            last = p.key, n = p.nth + 1ull;
            total = p.mass + n * w(p.key);
        }
        if (mp > 0.0f && !(w.share(last) >= mp)) {
            uint64_t s = 0;
            for (int i = threadIdx.x; i < a.V; i += kThreads) {
                const uint32_t key = key_of(x[i]);
                if (w.share(key) >= mp || key == top) s += w(key);
            }
            total = block_sum_u64(s, sh);
            // a minimum above 1 keeps the first place alone
            if (mp > 1.0f) total = w(top);
        }
        const float u = a.u[b];
        const double t = floor(static_cast<double>(u > 0.0f ? u : 0.0f) * static_cast<double>(total));
        at = find<true>(x, a.V, w, min(static_cast<uint64_t>(t), total - 1), sh);
        prob = static_cast<double>(w(at.key)) / static_cast<double>(total);
    }
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
            if (a.prob) a.prob[b] = static_cast<float>(prob);
        }
        seen += all;
        if (seen > at.nth) return;  // the same for every thread
    }
}

}  // namespace

uint64_t sample_workspace_bytes(int B, int V) { return 16; }

hipError_t launch_sample(const SampleArgs& a, hipStream_t s) {
    int bits = 0;
    while ((1ll << bits) < a.V) ++bits;
    klaunch(sample_kernel, dim3(a.B), dim3(kThreads), 0, s, a, ldexp(1.0, std::min(62 - bits, 50)));
    return hipGetLastError();
}

}  // namespace q35k
