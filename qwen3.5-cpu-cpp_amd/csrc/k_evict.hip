// Eviction of cache rows by score (q35_kv_evict): which rows stay is chosen by one workgroup
// per (sequence, kv head), the surviving rows beyond the budget are then copied into the
// slots that evicted rows leave. Sources lie at or above `keep` and destinations below it, so
// the copies are independent and only as many rows move as were evicted below `keep`.
#include "dev_common.hpp"
#include "launch.hpp"

namespace q35k {
namespace {

constexpr int kSelThreads = 1024, kSelWaves = kSelThreads / 64;
constexpr int kBins = 2048;

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

// Radix selection of the `keep`-th largest key over 11 + 11 + 10 bits (LDS histograms), then
// one pass that ranks the rows in slot order: of the rows equal to that key the lowest slots
// stay, and a row's rank among the kept ones gives its place in the move lists.
__global__ __launch_bounds__(kSelThreads) void kv_select_kernel(KvEvictArgs a) {
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t bk = static_cast<int64_t>(b) * a.NKV + h;
    const int n = a.len[b], keep = a.keep;
    int2* head = a.head + bk;
    if (n < 0 || n > a.cap) {
        if (tid == 0) *head = make_int2(n, 0);
        return;
    }
    const float* score = a.score + bk * a.cap;
    const int* pos = a.pos + bk * a.cap;
    float* score_out = a.score_out + bk * a.cap;
    int* pos_out = a.pos_out + bk * a.cap;
    const bool copy_s = a.score_out != a.score, copy_p = a.pos_out != a.pos;
    if (n <= keep) {
        for (int t = tid; t < n; t += kSelThreads) {
            if (copy_s) score_out[t] = score[t];
            if (copy_p) pos_out[t] = pos[t];
        }
        if (tid == 0) *head = make_int2(n, 0);
        return;
    }
    const int64_t recent = static_cast<int64_t>(a.next_pos[b]) - a.n_recent;
    __shared__ uint32_t hist[kBins];
    __shared__ uint32_t wsum[kSelWaves];
    __shared__ uint32_t found[2];
    uint32_t prefix = 0, want = keep;  // the wanted key is the want-th largest among those of this prefix
    int shift = 21;
    for (int pass = 0; pass < 3; ++pass) {
        const int bits = pass < 2 ? 11 : 10;
        for (int i = tid; i < kBins; i += kSelThreads) hist[i] = 0;
        __syncthreads();
        for (int t = tid; t < n; t += kSelThreads) {
            const uint32_t key = row_key(score[t], pos[t], a.n_sink, recent);
            if (pass == 0 || (key >> (shift + bits)) == prefix) atomicAdd(&hist[(key >> shift) & ((1u << bits) - 1)], 1u);
        }
        __syncthreads();
        // rows in bins above each pair of bins: thread i holds bins 2i, 2i + 1 from the top
        const int hi_bin = kBins - 1 - 2 * tid;
        const uint32_t c0 = hist[hi_bin], c1 = hist[hi_bin - 1];
        uint32_t inc = c0 + c1;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t up = __shfl_up(inc, o);
            if (lane >= o) inc += up;
        }
        if (lane == 63) wsum[wave] = inc;
        __syncthreads();
        uint32_t before = inc - c0 - c1;
        for (int w = 0; w < wave; ++w) before += wsum[w];
        if (before < want && want <= before + c0 + c1) {  // one thread
            const bool first = want <= before + c0;
            found[0] = first ? hi_bin : hi_bin - 1;
            found[1] = want - before - (first ? 0 : c0);
        }
        __syncthreads();
        prefix = (prefix << bits) | found[0];
        want = found[1];
        shift -= pass == 0 ? 11 : 10;
        __syncthreads();
    }
    const uint32_t limit = prefix;  // rows above it stay, and the first `want` equal ones

    // per-wave ranges of slots: rows above the limit and equal to it, and those below `keep`
    __shared__ uint32_t cnt[4][kSelWaves];
    const int per = (n + kSelWaves * 64 - 1) / (kSelWaves * 64) * 64;
    const int w0 = min(n, wave * per), w1 = min(n, w0 + per);
    uint32_t c[4] = {0, 0, 0, 0};
    for (int t0 = w0; t0 < w1; t0 += 64) {
        const int t = t0 + lane;
        const uint32_t key = t < w1 ? row_key(score[t], pos[t], a.n_sink, recent) : 0u;
        const uint64_t gt = __ballot(t < w1 && key > limit), eq = __ballot(t < w1 && key == limit);
        const uint64_t low = __ballot(t < keep);
        c[0] += __popcll(gt);
        c[1] += __popcll(eq);
        c[2] += __popcll(gt & low);
        c[3] += __popcll(eq & low);
    }
    if (lane == 0)
        for (int i = 0; i < 4; ++i) cnt[i][wave] = c[i];
    __syncthreads();
    uint32_t gt_before = 0, eq_before = 0, gt_low = 0, eq_low = 0;
    for (int w = 0; w < kSelWaves; ++w) {
        if (w < wave) {
            gt_before += cnt[0][w];
            eq_before += cnt[1][w];
        }
        gt_low += cnt[2][w];
        eq_low += cnt[3][w];
    }
    const uint32_t stay = gt_low + min(eq_low, want);  // kept rows below `keep`
    if (tid == 0) *head = make_int2(keep, keep - static_cast<int>(stay));
    int* to = a.to + bk * a.most;
    int* from = a.from + bk * a.most;
    for (int t0 = w0; t0 < w1; t0 += 64) {
        const int t = t0 + lane;
        const bool in = t < w1;
        const float sc = in ? score[t] : 0.0f;
        const int ps = in ? pos[t] : 0;
        const uint32_t key = row_key(sc, ps, a.n_sink, recent);
        const uint64_t gt = __ballot(in && key > limit), eq = __ballot(in && key == limit);
        const uint32_t eqb = eq_before + lanes_below(eq);
        const uint32_t kept_before = gt_before + lanes_below(gt) + min(eqb, want);
        const bool kept = in && (key > limit || (key == limit && eqb < want));
        if (in && t < keep && !kept) to[t - kept_before] = t;
        if (kept && t >= keep) from[kept_before - stay] = t;
        if (kept && t < keep) {
            if (copy_s) score_out[t] = sc;
            if (copy_p) pos_out[t] = ps;
        }
        gt_before += __popcll(gt);
        eq_before += __popcll(eq);
    }
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
    uint4* K = static_cast<uint4*>(a.k) + bk * a.cap * UNITS;
    uint4* V = static_cast<uint4*>(a.v) + bk * a.cap * UNITS;
    const int u = tid % UNITS;
    uint4 kr[4], vr[4];
    int dst[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int i = i0 + (j * 256 + tid) / UNITS;
        dst[j] = -1;
        if (i < m) {
            const int64_t s = from[i];
            dst[j] = to[i];
            kr[j] = K[s * UNITS + u];
            vr[j] = V[s * UNITS + u];
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (dst[j] >= 0) {
            K[static_cast<int64_t>(dst[j]) * UNITS + u] = kr[j];
            V[static_cast<int64_t>(dst[j]) * UNITS + u] = vr[j];
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

}  // namespace

int64_t kv_evict_workspace_ints(int B, int NKV, int64_t cap, int keep) {
    return static_cast<int64_t>(B) * NKV * (2 + 2 * static_cast<int64_t>(most_moved(cap, keep)));
}

void kv_evict_carve(KvEvictArgs& a, int* ws) {
    const int64_t bk = static_cast<int64_t>(a.B) * a.NKV;
    a.most = most_moved(a.cap, a.keep);
    a.head = reinterpret_cast<int2*>(ws);
    a.to = ws + 2 * bk;
    a.from = a.to + bk * a.most;
}

hipError_t launch_kv_evict(const KvEvictArgs& a, hipStream_t s) {
    klaunch(kv_select_kernel, dim3(a.NKV, a.B), kSelThreads, 0, s, a);
    const int units = a.kv_bf16 ? 32 : 64, rows = kMoveUnits / units;
    const dim3 grid(std::max(1, (a.most + rows - 1) / rows), a.NKV, a.B);
    if (a.kv_bf16) klaunch(kv_move_kernel<32>, grid, 256, 0, s, a);
    else klaunch(kv_move_kernel<64>, grid, 256, 0, s, a);
    return hipGetLastError();
}

}  // namespace q35k
