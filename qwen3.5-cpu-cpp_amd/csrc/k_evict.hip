// Eviction of cache rows by score (q35_kv_evict): which rows stay is chosen per (sequence, kv
// head), the surviving rows beyond the budget are then copied into the slots that evicted rows
// leave. Sources lie at or above `keep` and destinations below it, so the copies are independent
// and only as many rows move as were evicted below `keep`.
//
// Choosing is a radix selection of the keep-th largest 32-bit key over 11 + 11 + 10 bits with
// histograms in LDS (after the first 11 mostly few keys are left, which are then compared with one
// another: 1152 rows 10.0 us a call, 11.3 by three passes; with up to 64 keys for few instead of 256
// the same), then a pass that ranks the rows in slot order: of the rows equal to that
// key the lowest slots stay, and the number of rows kept before a row gives its place in the move
// lists. Up to kRegRows rows one workgroup holds all keys in registers and does it in one
// launch. Longer caches are cut into slices of kSlice rows, a workgroup each, in three launches:
// the keys and their histogram; from all slices' histograms the bin of the wanted key, and the
// slice's keys that lie in it (candidates); from all candidates the key itself, and the slice's
// ranks. What every slice needs of the others it forms for itself, so no launch has a single
// workgroup: 131072 rows of two heads 22 us against 56 with one workgroup that
// finds the key and slices that count the rows before them. One workgroup and slices, whole calls in us, bf16
// caches of two heads cut to 7/8, 1 / 4 / 24 sequences: 4096 rows 12.1 / 13.0 / 19.4 and 19.5 / 20.4 / 27.4; 4097
// (16 keys a thread instead of 4) 19.3 / 20.4 / 27.2 and 19.6 / 21.3 / 29.8; 8192 21.9 / 23.6 / 37.1 and 20.8 /
// 22.0 / 37.9; 16384 26.7 / 28.9 / 57.5 and 21.6 / 25.0 / 55.4; beyond, 16385 and 32768 rows of one sequence
// 22.3 and 24.5. So the border is where the registers end, and slices would do for a few sequences from 6000
// rows on.
#include "dev_common.hpp"
#include "launch.hpp"

namespace q35k {
namespace {

constexpr int kSelThreads = 1024, kSelWaves = kSelThreads / 64;
constexpr int kBins = 2048;
constexpr int kRegRows = 16384;      // most rows of the one-launch selection (16 keys a thread)
constexpr int kSlice = 4096;         // rows of a slice of a longer cache
constexpr int kCandidates = 16384;   // keys of one bin held in LDS
constexpr int kFew = kSelThreads / 4; // keys of one bin that are compared with one another

// Order of the rows: larger keys stay. Rows kept whatever their weight come first, a NaN
// last; -0 equals 0.
__device__ __forceinline__ uint32_t row_key(float score, int pos, int n_sink, int64_t recent) {
    if (pos < n_sink || pos >= recent) return 0xffffffffu;
    if (!(score == score)) return 0u;
    const uint32_t u = __float_as_uint(score + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ int lanes_below(uint64_t mask) {
    return __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(mask >> 32),
                                     __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(mask), 0));
}

// Sums over the lanes up to each one's, by shifts within rows of 16 lanes and broadcasts of a row's
// and of half a wave's last lane (no LDS: six exchanges through it take 0.35 us).
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, true);
    return v;
}

// One (sequence, kv head): its arrays, its rows n, and whether there is anything to choose.
struct Cache {
    int64_t bk;
    int n;
    bool choose;
    const float* score;
    const int* pos;
    float* score_out;  // null where scores stay in their array
    int* pos_out;
    int64_t recent;
};
__device__ __forceinline__ Cache cache_of(const KvEvictArgs& a, int h, int b) {
    Cache c;
    c.bk = static_cast<int64_t>(b) * a.NKV + h;
    c.n = a.len[b];
    c.choose = c.n > a.keep && c.n <= a.cap;
    c.score = a.score + c.bk * a.cap;
    c.pos = a.pos + c.bk * a.cap;
    c.score_out = a.score_out != a.score ? a.score_out + c.bk * a.cap : nullptr;
    c.pos_out = a.pos_out != a.pos ? a.pos_out + c.bk * a.cap : nullptr;
    c.recent = static_cast<int64_t>(a.next_pos[b]) - a.n_recent;
    return c;
}
// Rows [t0, t1) of a cache within its budget (or of none): they stay where they are.
__device__ __forceinline__ void keep_all(const KvEvictArgs& a, const Cache& c, int t0, int t1) {
    if (c.n <= a.cap)
        for (int t = t0 + threadIdx.x; t < min(t1, c.n); t += blockDim.x) {
            if (c.score_out) c.score_out[t] = c.score[t];
            if (c.pos_out) c.pos_out[t] = c.pos[t];
        }
    if (t0 == 0 && threadIdx.x == 0) a.head[c.bk] = make_int2(c.n, 0);
}

// The bin, from the top, that holds the want-th largest of the counted keys, how many of its keys are
// wanted and how many it has. c0, c1: the counts of this thread's bins kBins - 1 - 2 tid and the next
// lower.
__device__ __forceinline__ uint3 find_bin(uint32_t c0, uint32_t c1, uint32_t want, uint32_t* wsum, uint32_t* found) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, hi_bin = kBins - 1 - 2 * tid;
    const uint32_t inc = wave_scan(c0 + c1);
    if (lane == 63) wsum[wave] = inc;
    __syncthreads();
    uint32_t before = inc - c0 - c1;
    for (int w = 0; w < wave; ++w) before += wsum[w];
    if (before < want && want <= before + c0 + c1) {  // one thread
        const bool first = want <= before + c0;
        found[0] = first ? hi_bin : hi_bin - 1;
        found[1] = want - before - (first ? 0 : c0);
        found[2] = first ? c0 : c1;
    }
    __syncthreads();
    return make_uint3(found[0], found[1], found[2]);
}

// The last key that stays and how many of the keys equal to it do; each(f) calls f on every key of
// the thread (each key of the cache is some thread's). From pass `pass` on, among the keys whose
// higher bits are `prefix`.
template <class Each>
__device__ __forceinline__ uint2 radix_limit(uint32_t* hist, uint32_t* wsum, uint32_t* found, int pass, uint32_t prefix,
                                             uint32_t want, Each&& each) {
    const int tid = threadIdx.x;
    __shared__ uint32_t few[kFew], listed;
    uint32_t left = 0xffffffffu;
    for (; pass < 3 && left > kFew; ++pass) {
        const int bits = pass < 2 ? 11 : 10, shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
        hist[tid] = hist[tid + kSelThreads] = 0;
        __syncthreads();
        each([&](uint32_t key) {
            if (pass == 0 || (key >> (shift + bits)) == prefix) atomicAdd(&hist[(key >> shift) & ((1u << bits) - 1)], 1u);
        });
        __syncthreads();
        const uint3 r = find_bin(hist[kBins - 1 - 2 * tid], hist[kBins - 2 - 2 * tid], want, wsum, found);
        prefix = (prefix << bits) | r.x;
        want = r.y;
        left = r.z;
    }
    if (pass == 3) return make_uint2(prefix, want);
    // few keys share the bits so far: each is compared with all
    if (tid == 0) listed = 0;
    __syncthreads();
    each([&](uint32_t key) {
        if (key >> (pass == 1 ? 21 : 10) == prefix) few[atomicAdd(&listed, 1u)] = key;
    });
    __syncthreads();
    // (four threads a key, a quarter of the comparisons each)
    const uint32_t key = few[min(static_cast<uint32_t>(tid >> 2), left - 1)];
    uint32_t above = 0, equal = 0;
#pragma unroll 4
    for (uint32_t i = tid & 3; i < left; i += 4) {
        above += few[i] > key;
        equal += few[i] == key;
    }
    above += dpp_i<0xB1>(above), equal += dpp_i<0xB1>(equal);
    above += dpp_i<0x4E>(above), equal += dpp_i<0x4E>(equal);
    if (above < want && want <= above + equal) {  // the wanted key: every thread that has it writes the same
        found[0] = key;
        found[1] = want - above;
    }
    __syncthreads();
    return make_uint2(found[0], found[1]);
}

// Rows kept so far in slot order, and what becomes of 64 rows (a lane each) after them.
struct Ranks {
    uint32_t gt, eq;   // rows above the limit, and equal to it, in earlier slots
};
__device__ __forceinline__ void rank_rows(const KvEvictArgs& a, const Cache& c, Ranks& r, uint2 limit, uint32_t stay, int t,
                                          bool in, uint32_t key) {
    const uint64_t gt = __ballot(in && key > limit.x), eq = __ballot(in && key == limit.x);
    const uint32_t eqb = r.eq + lanes_below(eq);
    const uint32_t before = r.gt + lanes_below(gt) + min(eqb, limit.y);
    const bool kept = in && (key > limit.x || (key == limit.x && eqb < limit.y));
    if (in && t < a.keep && !kept) a.to[c.bk * a.most + t - before] = t;
    if (kept && t >= a.keep) a.from[c.bk * a.most + before - stay] = t;
    if (kept && t < a.keep) {
        if (c.score_out) c.score_out[t] = c.score[t];
        if (c.pos_out) c.pos_out[t] = c.pos[t];
    }
    r.gt += __popcll(gt);
    r.eq += __popcll(eq);
}

// Counts over the workgroup's waves: rows above the limit and equal to it in earlier waves, and, of
// all, below `keep`. c: this wave's four counts (above, equal, and both below `keep`).
__device__ __forceinline__ Ranks wave_ranks(uint32_t (&cnt)[4][kSelWaves], const uint32_t (&c)[4], uint2 limit, uint32_t& stay) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (lane == 0)
        for (int i = 0; i < 4; ++i) cnt[i][wave] = c[i];
    __syncthreads();
    Ranks r{0, 0};
    uint32_t gt_low = 0, eq_low = 0;
    for (int w = 0; w < kSelWaves; ++w) {
        if (w < wave) r.gt += cnt[0][w], r.eq += cnt[1][w];
        gt_low += cnt[2][w], eq_low += cnt[3][w];
    }
    stay = gt_low + min(eq_low, limit.y);
    return r;
}

// grid (NKV, B): a whole cache of up to KPT * 1024 rows, wave w holding KPT times 64 rows.
template <int KPT>
__global__ __launch_bounds__(kSelThreads) void kv_select_kernel(KvEvictArgs a) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const Cache c = cache_of(a, blockIdx.x, blockIdx.y);
    if (!c.choose) {
        keep_all(a, c, 0, static_cast<int>(a.cap));
        return;
    }
    __shared__ uint32_t hist[kBins], wsum[kSelWaves], found[3], cnt[4][kSelWaves];
    // (waves take whole groups of 64 in turn of slots; the rows are spread over all waves)
    const int per = (c.n + kSelThreads - 1) / kSelThreads, w0 = wave * per * 64;  // per <= KPT
    float sc[KPT];
    int ps[KPT];
#pragma unroll
    for (int j = 0; j < KPT; ++j) {
        const int t = min(w0 + 64 * j + lane, c.n - 1);
        sc[j] = c.score[t];
        ps[j] = c.pos[t];
    }
    uint32_t key[KPT];
#pragma unroll
    for (int j = 0; j < KPT; ++j) key[j] = row_key(sc[j], ps[j], a.n_sink, c.recent);
    const auto in = [&](int j) { return j < per && w0 + 64 * j + lane < c.n; };
    const uint2 limit = radix_limit(hist, wsum, found, 0, 0, a.keep, [&](auto&& f) {
#pragma unroll
        for (int j = 0; j < KPT; ++j)
            if (in(j)) f(key[j]);
    });
    uint32_t n4[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < KPT; ++j) {
        const bool low = w0 + 64 * j + lane < a.keep;
        const uint64_t gt = __ballot(in(j) && key[j] > limit.x), eq = __ballot(in(j) && key[j] == limit.x);
        const uint64_t lo = __ballot(low);
        n4[0] += __popcll(gt), n4[1] += __popcll(eq), n4[2] += __popcll(gt & lo), n4[3] += __popcll(eq & lo);
    }
    uint32_t stay;
    Ranks r = wave_ranks(cnt, n4, limit, stay);
    if (tid == 0) a.head[c.bk] = make_int2(a.keep, a.keep - static_cast<int>(stay));
#pragma unroll
    for (int j = 0; j < KPT; ++j) rank_rows(a, c, r, limit, stay, w0 + 64 * j + lane, in(j), key[j]);
}

// grid (slices, NKV, B): the keys of a slice's rows and their histogram over the highest 11 bits.
__global__ __launch_bounds__(kSelThreads) void kv_keys_kernel(KvEvictArgs a) {
    const int tid = threadIdx.x;
    const Cache c = cache_of(a, blockIdx.y, blockIdx.z);
    const int t0 = blockIdx.x * kSlice;
    if (!c.choose) {
        keep_all(a, c, t0, t0 + kSlice);
        return;
    }
    if (t0 >= c.n) return;
    __shared__ uint32_t hist[kBins];
    hist[tid] = hist[tid + kSelThreads] = 0;
    float sc[4];
    int ps[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int t = min(t0 + kSelThreads * j + tid, c.n - 1);
        sc[j] = c.score[t];
        ps[j] = c.pos[t];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int t = t0 + kSelThreads * j + tid;
        const uint32_t key = row_key(sc[j], ps[j], a.n_sink, c.recent);
        if (t < c.n) {
            a.keys[c.bk * a.cap + t] = key;
            atomicAdd(&hist[key >> 21], 1u);
        }
    }
    __syncthreads();
    // (a slice's counts fit 16 bits)
    a.hist[(c.bk * gridDim.x + blockIdx.x) * (kBins / 2) + tid] = hist[2 * tid] | hist[2 * tid + 1] << 16;
}

// sums of N counts over the workgroup, to every thread
template <int N>
__device__ __forceinline__ void block_sums(uint32_t (&s)[N], uint32_t (*red)[kSelWaves]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        s[i] = wave_scan(s[i]);
        if (lane == 63) red[i][wave] = s[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        s[i] = 0;
        for (int w = 0; w < kSelWaves; ++w) s[i] += red[i][w];
    }
}

// grid (slices, NKV, B): the bin of the wanted key; of this slice the candidates, in slot order
// (over its keys' place in `cand`), and how many rows of earlier slices lie in higher bins, how
// many candidates there are, and how many of either kind lie below `keep`. Slice 0 notes
// the bin and how many of its keys are wanted.
__global__ __launch_bounds__(kSelThreads) void kv_bin_kernel(KvEvictArgs a) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, slices = gridDim.x, slice = blockIdx.x;
    const Cache c = cache_of(a, blockIdx.y, blockIdx.z);
    const int t0 = slice * kSlice;
    if (!c.choose || t0 >= c.n) return;
    __shared__ uint32_t wsum[kSelWaves], found[3], red[3][kSelWaves], wcnt[kSelWaves];
    const int w0 = t0 + wave * 256;  // wave w holds four times 64 rows
    uint32_t key[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) key[j] = a.keys[c.bk * a.cap + min(w0 + 64 * j + lane, c.n - 1)];
    const int used = (c.n + kSlice - 1) / kSlice;
    const uint32_t* h = a.hist + c.bk * slices * (kBins / 2) + kBins / 2 - 1 - tid;
    uint32_t c0 = 0, c1 = 0, e0 = 0, e1 = 0;  // of all slices, of earlier ones
#pragma unroll 16
    for (int i = 0; i < used; ++i) {
        const uint32_t x = h[static_cast<int64_t>(i) * (kBins / 2)];
        c0 += x >> 16, c1 += x & 0xffffu;
        if (i < slice) e0 += x >> 16, e1 += x & 0xffffu;
    }
    const uint3 top = find_bin(c0, c1, a.keep, wsum, found);
    const uint32_t bin = kBins - 1 - 2 * tid;
    uint32_t s[3] = {(bin > top.x ? e0 : 0) + (bin - 1 > top.x && bin > 0 ? e1 : 0), 0, 0};
    uint32_t mine = 0;  // candidates of this wave
    uint64_t is[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int t = w0 + 64 * j + lane;
        const bool cand = t < c.n && key[j] >> 21 == top.x;
        is[j] = __ballot(cand);
        mine += __popcll(is[j]);
        s[1] += t < c.n && t < a.keep && key[j] >> 21 > top.x;
        s[2] += cand && t < a.keep;
    }
    if (lane == 0) wcnt[wave] = mine;
    block_sums(s, red);
    uint32_t at = 0, total = 0;
    for (int w = 0; w < kSelWaves; ++w) {
        if (w < wave) at += wcnt[w];
        total += wcnt[w];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (is[j] >> lane & 1) a.cand[c.bk * a.cap + t0 + at + lanes_below(is[j])] = key[j];
        at += __popcll(is[j]);
    }
    if (tid == 0) {
        a.slice[c.bk * slices + slice] = make_uint4(s[0], total, s[1], s[2]);
        if (slice == 0) a.limit[c.bk] = make_uint2(top.x, top.y);
    }
}

// grid (slices, NKV, B): the last key that stays, from the candidates of all slices (in LDS, or where
// they do not fit, many equal ones, found again in every pass), then the ranks of this slice's
// rows.
__global__ __launch_bounds__(kSelThreads) void kv_rank_kernel(KvEvictArgs a) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, slices = gridDim.x, slice = blockIdx.x;
    const Cache c = cache_of(a, blockIdx.y, blockIdx.z);
    const int t0 = slice * kSlice;
    if (!c.choose || t0 >= c.n) return;
    __shared__ uint32_t hist[kBins], wsum[kSelWaves], found[3], cnt[4][kSelWaves], red[4][kSelWaves];
    __shared__ uint32_t cand[kCandidates];
    const int used = (c.n + kSlice - 1) / kSlice, low = a.keep / kSlice;  // `keep` lies in slice `low`
    const uint4* sl = a.slice + c.bk * slices;
    const uint2 top = a.limit[c.bk];
    const int w0 = t0 + wave * 256;
    uint32_t key[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) key[j] = a.keys[c.bk * a.cap + min(w0 + 64 * j + lane, c.n - 1)];
    const uint4 here = sl[slice], edge = sl[low];
    // candidates of all slices; of those before this one; of those below `keep`
    uint32_t s[3] = {0, 0, 0};
    for (int i = tid; i < used; i += kSelThreads) {
        const uint32_t n = sl[i].y;
        s[0] += n;
        if (i < slice) s[1] += n;
        if (i < low) s[2] += n;
    }
    block_sums(s, red);
    const uint32_t total = s[0], before = s[1], below = s[2] + edge.w;
    // f(key, place in slot order) for every candidate, a wave per slice
    const auto listed = [&](auto&& f) {
        uint32_t off = 0;
        for (int i0 = 0; i0 < used; i0 += 16) {  // counts of sixteen slices at a time, one a lane
            const uint32_t mine = lane < 16 && i0 + lane < used ? sl[i0 + lane].y : 0, inc = wave_scan(mine);
            const uint32_t n = __shfl(mine, wave), first = off + __shfl(inc, wave) - n;
            for (uint32_t k = lane; k < n; k += 64) f(a.cand[c.bk * a.cap + (i0 + wave) * static_cast<int64_t>(kSlice) + k], first + k);
            off += __shfl(inc, 15);
        }
    };
    const bool fits = total <= kCandidates;
    if (fits) listed([&](uint32_t k, uint32_t at) { cand[at] = k; });
    __syncthreads();
    const auto each = [&](auto&& f) {
        if (!fits) return listed(f);
        for (uint32_t i = tid; i < total; i += 4 * kSelThreads) {  // (four reads on their way at once)
            uint32_t k[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) k[j] = cand[min(i + j * kSelThreads, total - 1)];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (i + j * kSelThreads < total) f(k[j], i + j * kSelThreads);
        }
    };
    const uint2 limit = radix_limit(hist, wsum, found, 1, top.x, top.y, [&](auto&& f) { each([&](uint32_t k, uint32_t) { f(k); }); });
    uint32_t q[4] = {0, 0, 0, 0};  // before this slice: above, equal; below `keep`: above, equal
    each([&](uint32_t k, uint32_t at) {
        const uint32_t gt = k > limit.x, eq = k == limit.x;
        if (at < before) q[0] += gt, q[1] += eq;
        if (at < below) q[2] += gt, q[3] += eq;
    });
    __syncthreads();  // `red` again
    block_sums(q, red);
    uint32_t n4[4] = {0, 0, 0, 0};
    const auto in = [&](int j) { return w0 + 64 * j + lane < c.n; };
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        n4[0] += __popcll(__ballot(in(j) && key[j] > limit.x));
        n4[1] += __popcll(__ballot(in(j) && key[j] == limit.x));
    }
    uint32_t ignored;
    Ranks r = wave_ranks(cnt, n4, limit, ignored);
    r.gt += here.x + q[0];
    r.eq += q[1];
    const uint32_t stay = edge.x + edge.z + q[2] + min(q[3], limit.y);
    if (slice == 0 && tid == 0) a.head[c.bk] = make_int2(a.keep, a.keep - static_cast<int>(stay));
#pragma unroll
    for (int j = 0; j < 4; ++j) rank_rows(a, c, r, limit, stay, w0 + 64 * j + lane, in(j), key[j]);
}

constexpr int kMoveUnits = 1024;  // 16-byte units of K (and of V) per workgroup

// grid (chunks, NKV, B): copies rows from[i] -> to[i] of K and V with their scores and
// positions, four 16-byte units of each per thread.
template <int UNITS>  // units of a row
__global__ __launch_bounds__(256) void kv_move_kernel(KvEvictArgs a) {
    constexpr int R = kMoveUnits / UNITS;
    const int h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
    const int64_t bk = static_cast<int64_t>(b) * a.NKV + h;
    const int2 head = a.head[bk];
    if (blockIdx.x == 0 && h == 0 && tid == 0) a.new_len[b] = head.x;
    const int i0 = blockIdx.x * R, m = head.y;
    if (i0 >= m) return;
    const int* to = a.to + bk * a.most;
    const int* from = a.from + bk * a.most;
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    u32x4* K = static_cast<u32x4*>(a.k) + bk * a.cap * UNITS;
    u32x4* V = static_cast<u32x4*>(a.v) + bk * a.cap * UNITS;
    const int u = tid % UNITS;
    u32x4 kr[4], vr[4];
    int64_t src[4], dst[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {  // rows past the last: the last again, not stored
        const int i = i0 + (j * 256 + tid) / UNITS, ic = min(i, m - 1);
        src[j] = static_cast<int64_t>(from[ic]) * UNITS + u;
        dst[j] = i < m ? static_cast<int64_t>(to[ic]) * UNITS + u : -1;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        kr[j] = __builtin_nontemporal_load(K + src[j]);
        vr[j] = __builtin_nontemporal_load(V + src[j]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (dst[j] >= 0) {
            __builtin_nontemporal_store(kr[j], K + dst[j]);
            __builtin_nontemporal_store(vr[j], V + dst[j]);
        }
    if (tid < R && i0 + tid < m) {
        const int s = from[i0 + tid], d = to[i0 + tid];
        a.score_out[bk * a.cap + d] = a.score[bk * a.cap + s];
        a.pos_out[bk * a.cap + d] = a.pos[bk * a.cap + s];
    }
}

// rows that may have to move: no more than stay and no more than lie beyond
int most_moved(int64_t cap, int keep) {
    return static_cast<int>(std::max<int64_t>(0, std::min<int64_t>(keep, cap - keep)));
}
// slices of a long cache (0: chosen in one launch, or never longer than `keep`)
int slices_of(int64_t cap, int keep) {
    return cap <= kRegRows || cap <= keep ? 0 : static_cast<int>((cap + kSlice - 1) / kSlice);
}

}  // namespace

int64_t kv_evict_workspace_ints(int B, int NKV, int64_t cap, int keep) {
    const int64_t slices = slices_of(cap, keep);
    return static_cast<int64_t>(B) * NKV *
           (2 + 2 * static_cast<int64_t>(most_moved(cap, keep)) + (slices ? 2 * cap + slices * (kBins / 2 + 4) + 2 : 0)) + 4;
}

void kv_evict_carve(KvEvictArgs& a, int* ws) {
    const int64_t bk = static_cast<int64_t>(a.B) * a.NKV, slices = slices_of(a.cap, a.keep);
    a.most = most_moved(a.cap, a.keep);
    if (slices) {
        a.slice = reinterpret_cast<uint4*>(ws);  // widest elements first: every array stays aligned
        ws += 4 * bk * slices;
        a.hist = reinterpret_cast<uint32_t*>(ws);
        ws += bk * slices * (kBins / 2);
        a.limit = reinterpret_cast<uint2*>(ws);
        ws += 2 * bk;
        a.keys = reinterpret_cast<uint32_t*>(ws) + 2 * bk;
        a.cand = a.keys + bk * a.cap;
    }
    a.head = reinterpret_cast<int2*>(ws);
    ws += 2 * bk + (slices ? 2 * bk * a.cap : 0);
    a.to = ws;
    a.from = a.to + bk * a.most;
}

hipError_t launch_kv_evict(const KvEvictArgs& a, hipStream_t s) {
    const dim3 each(a.NKV, a.B);
    if (const int slices = slices_of(a.cap, a.keep)) {
        const dim3 cut(slices, a.NKV, a.B);
        klaunch(kv_keys_kernel, cut, kSelThreads, 0, s, a);
        klaunch(kv_bin_kernel, cut, kSelThreads, 0, s, a);
        klaunch(kv_rank_kernel, cut, kSelThreads, 0, s, a);
    } else if (a.cap <= 4 * kSelThreads || a.cap <= a.keep) {
        klaunch(kv_select_kernel<4>, each, kSelThreads, 0, s, a);
    } else {
        klaunch(kv_select_kernel<16>, each, kSelThreads, 0, s, a);
    }
    const int units = a.kv_bf16 ? 32 : 64, rows = kMoveUnits / units;
    const dim3 grid(std::max(1, (a.most + rows - 1) / rows), a.NKV, a.B);
    if (a.kv_bf16) klaunch(kv_move_kernel<32>, grid, 256, 0, s, a);
    else klaunch(kv_move_kernel<64>, grid, 256, 0, s, a);
    return hipGetLastError();
}

}  // namespace q35k
