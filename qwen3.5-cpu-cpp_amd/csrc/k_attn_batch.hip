// Attention of a batch of continuations: one token per sequence over a prefix that all share
// and each sequence's own cache, in three launches: the queries and the appended rows
// (prep), partial outputs over pieces of the keys (attend), and their merge with the gate,
// which also adds the softmax weights to the own rows' scores (combine).
#include <cmath>

#include "dev_common.hpp"
#include "launch.hpp"

namespace q35k {
namespace {

constexpr int kHD = 256;

// fp32 -> bf16, round to nearest even, NaN stays NaN
__device__ __forceinline__ uint16_t to_bf16(float x) { return x == x ? f32_to_bf16(x) : uint16_t{0x7fc0}; }

// slot of the new row, -1 where the place is empty or the cache full
__device__ __forceinline__ int new_slot(const AttnBatchArgs& a, int b) {
    const int n = a.own_len[b];
    return n >= 0 && n < a.cap ? n : -1;
}

// stride of the rows of raw scores: whole tiles
__host__ __device__ inline int64_t raw_stride(int64_t cap) { return (cap + 31) / 32 * 32; }

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef short i16x8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));

// 2^e
__device__ __forceinline__ float pow2(int e) { return __uint_as_float(static_cast<uint32_t>(127 + e) << 23); }
// the power of two that brings a largest magnitude (its bits) into [2^14, 2^15), as far as 2^+-100
__device__ __forceinline__ int row_exp(uint32_t bits) { return min(max(141 - static_cast<int>(bits >> 23), -100), 100); }
// what undoes it; NaN for a row of 2^115 or more, an infinity or a NaN (whose other entries the parts
// would lose, and the row's outputs be finite and wrong)
__device__ __forceinline__ float row_scale(uint32_t bits, int e) { return bits < 0x79000000u ? pow2(-e) : NAN; }
// Scores are formed over 2^kScoreExp times their query's scale: a sum of scaled products (below 2^39) times
// its key's 2^100 at most then stays below 2^123.
constexpr int kScoreExp = 16;

// theta^(-2i / ROT), formed on the host: 32 double-precision powers cost the kernel 1 us
struct RopeFreq {
    double f[kHD / 2];
};

// Dims 4 lane .. + 3 of query row `row`.
__device__ __forceinline__ void store_query(const AttnBatchArgs& a, int64_t row, int lane, float4 y) {
    if (a.kv_bf16) {  // three exact bf16 parts, [row][3][HD]
        uint32_t lo[3], hi[3];
        split3_pair(y.x, y.y, lo[0], lo[1], lo[2]);
        split3_pair(y.z, y.w, hi[0], hi[1], hi[2]);
#pragma unroll
        for (int q = 0; q < 3; ++q) static_cast<uint2*>(a.Qs)[(row * 3 + q) * 64 + lane] = make_uint2(lo[q], hi[q]);
        return;
    }
    *reinterpret_cast<float4*>(a.Qa + row * kHD + 4 * lane) = y;
    if (!a.Qs) return;
    // two fp16 parts of the row scaled by a power of two, [row][2][HD]
    const float mx = wave_max(fmaxf(fmaxf(fabsf(y.x), fabsf(y.y)), fmaxf(fabsf(y.z), fabsf(y.w))));
    const int e = row_exp(__float_as_uint(mx));
    uint2 h, l;
    split2h_pair(y.x * pow2(e), y.y * pow2(e), h.x, l.x);
    split2h_pair(y.z * pow2(e), y.w * pow2(e), h.y, l.y);
    static_cast<uint2*>(a.Qs)[(row * 2 + 0) * 64 + lane] = h;
    static_cast<uint2*>(a.Qs)[(row * 2 + 1) * 64 + lane] = l;
    if (lane == 0) a.Qscale[row] = row_scale(__float_as_uint(mx), e - kScoreExp);
}

// grid ((NQ + NKV) / 4, B), a wave per row: rmsnorm (1 + w) + RoPE of a query row, or of the new key
// row -> own cache, with its value row. Angles in double, one lane each. Query rows, times
// 1 / sqrt(HD), are stored as the attention reads them: as they are (Qa) where it multiplies in
// fp32, and split into the parts of its 16-bit products (Qs), which each workgroup would split again.
__global__ __launch_bounds__(256) void attn_batch_prep_kernel(AttnBatchArgs a, RopeFreq freq) {
    const int b = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = blockIdx.x * 4 + wave;
    __shared__ __align__(16) float buf[4][kHD];
    __shared__ float cs[2][kHD / 2];
    const bool is_q = r < a.NQ, there = r < a.NQ + a.NKV;
    const int kh = is_q ? r / a.GRP : min(r - a.NQ, a.NKV - 1);
    // (requested before the lengths are known: rows of empty places are there to be read)
    const int64_t bk = static_cast<int64_t>(b) * a.NKV + kh;
    const float* src = is_q ? a.qg + (static_cast<int64_t>(b) * a.NQ + r) * 2 * kHD : a.k_new + bk * kHD;
    const float4 x = *reinterpret_cast<const float4*>(src + 4 * lane);
    const float4 w = *reinterpret_cast<const float4*>((is_q ? a.q_norm : a.k_norm) + 4 * lane);
    const float4 v = *reinterpret_cast<const float4*>(a.v_new + bk * kHD + 4 * lane);
    const int half = a.ROT / 2, pos = a.pos[b], slot = new_slot(a, b);
    const int64_t qrow = (static_cast<int64_t>(kh) * a.B + b) * a.GRP + (r - kh * a.GRP);
    if (slot < 0) {
        if (is_q) store_query(a, qrow, lane, make_float4(0.f, 0.f, 0.f, 0.f));
        return;
    }
    for (int i = threadIdx.x; i < half; i += 256) {
        double sn, cn;
        sincos(static_cast<double>(pos) * freq.f[i], &sn, &cn);
        cs[0][i] = static_cast<float>(cn);
        cs[1][i] = static_cast<float>(sn);
    }
    const double ss = wave_sum(static_cast<double>(x.x) * x.x + static_cast<double>(x.y) * x.y + static_cast<double>(x.z) * x.z +
                               static_cast<double>(x.w) * x.w);
    const float inv = 1.0f / sqrtf(static_cast<float>(ss / kHD) + a.eps);
    float y[4] = {x.x * inv * (1.0f + w.x), x.y * inv * (1.0f + w.y), x.z * inv * (1.0f + w.z), x.w * inv * (1.0f + w.w)};
    *reinterpret_cast<float4*>(&buf[wave][4 * lane]) = make_float4(y[0], y[1], y[2], y[3]);
    __syncthreads();
    if (!there) return;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int d = 4 * lane + e;
        if (d < a.ROT) {
            const int i = d < half ? d : d - half;
            const float c = cs[0][i], s = cs[1][i];
            y[e] = d < half ? y[e] * c - buf[wave][i + half] * s : y[e] * c + buf[wave][i] * s;
        }
    }
    if (is_q) {  // scaled by 1 / sqrt(HD), exact
        store_query(a, qrow, lane, make_float4(y[0] * 0.0625f, y[1] * 0.0625f, y[2] * 0.0625f, y[3] * 0.0625f));
        return;
    }
    const int64_t row = bk * a.cap + slot;
    if (a.kv_bf16) {
        const auto pair = [](float lo, float hi) { return to_bf16(lo) | static_cast<uint32_t>(to_bf16(hi)) << 16; };
        static_cast<uint2*>(a.k_own)[row * (kHD / 4) + lane] = make_uint2(pair(y[0], y[1]), pair(y[2], y[3]));
        static_cast<uint2*>(a.v_own)[row * (kHD / 4) + lane] = make_uint2(pair(v.x, v.y), pair(v.z, v.w));
    } else {
        static_cast<float4*>(a.k_own)[row * (kHD / 4) + lane] = make_float4(y[0], y[1], y[2], y[3]);
        static_cast<float4*>(a.v_own)[row * (kHD / 4) + lane] = v;
    }
    if (a.own_pos && lane == 0) a.own_pos[row] = pos;
}

constexpr float kLog2e = 1.44269504088896341f;
constexpr int kKT = 32;         // keys per tile of the 16-bit matrix products
constexpr int kWaitVm = 0x0f70; // s_waitcnt: vector memory, nothing outstanding

// What one workgroup does: rows [row0, rows) of one list of query rows over keys [lo, hi) of one
// cache, and where its partial result goes.
struct Item {

    int64_t q0;             // first query row, of all
    int rows, row0;
    int lo, hi;
    const void *K, *V;      // row 0 of the cache
    float* part;            // [rows][HD]
    float2* ml;             // [rows]
    float* raw;             // scores of the rows, stride raw_stride, indexed by key (own caches; may be null)
    int64_t raw_stride;
    bool narrow;            // at most 16 rows, shared by the workgroup's waves
};

// Items [0, prefix_items) are (piece, kv head, row block) of the prefix, the others (piece, kv
// head, sequence) of the own caches. Workgroups go to the 8 XCDs in turn: the row blocks that
// read one piece get numbers 8 apart, so that one L2 fetches it for all of them.
__host__ __device__ inline int prefix_items(const AttnBatchPlan& p, int NKV) { return (p.pieces * NKV + 7) / 8 * 8 * p.nblk; }
__device__ __forceinline__ bool item_of(const AttnBatchArgs& a, int i, Item& it) {
    const int pairs = a.plan.pieces * a.NKV, prefix = prefix_items(a.plan, a.NKV);

    const int64_t row_bytes = a.kv_bf16 ? kHD * 2 : kHD * 4;
    if (i < prefix) {
        const int blk = (i >> 3) % a.plan.nblk, pair = (i >> 3) / a.plan.nblk * 8 + (i & 7);
        if (pair >= pairs) return false;
        const int piece = pair / a.NKV, kh = pair - piece * a.NKV;
        it.rows = a.B * a.GRP;
        it.row0 = blk * a.plan.block;
        it.q0 = static_cast<int64_t>(kh) * it.rows;
        it.lo = piece * a.plan.pkeys;
        it.hi = static_cast<int>(min(a.P, static_cast<int64_t>(it.lo) + a.plan.pkeys));
        it.K = static_cast<const char*>(a.k_prefix) + kh * a.prefix_cap * row_bytes;
        it.V = static_cast<const char*>(a.v_prefix) + kh * a.prefix_cap * row_bytes;
        const int64_t row = (static_cast<int64_t>(kh) * a.plan.pieces + piece) * it.rows;
        it.part = a.part_p + row * kHD;
        it.ml = a.ml_p + row;
        it.raw = nullptr;
        it.raw_stride = 0;
        it.narrow = a.plan.block == kBatchNarrow;
        return true;
    }
    i -= prefix;
    // first pieces first, as later ones may be empty, and each piece of a cache another XCD's
    const int pairs_own = a.B * a.NKV, piece = i / pairs_own;
    i = (i - piece * pairs_own + piece) % pairs_own;
    const int kh = i % a.NKV, b = i / a.NKV;
    const int slot = new_slot(a, b);
    const int64_t lo = static_cast<int64_t>(piece) * a.plan.okeys;
    if (slot < 0 || lo > slot) return false;
    const int64_t bk = static_cast<int64_t>(b) * a.NKV + kh;
    it.rows = a.GRP;
    it.row0 = 0;
    it.q0 = (static_cast<int64_t>(kh) * a.B + b) * a.GRP;
    it.lo = static_cast<int>(lo);
    it.hi = static_cast<int>(min(static_cast<int64_t>(slot) + 1, lo + a.plan.okeys));
    it.K = static_cast<const char*>(a.k_own) + bk * a.cap * row_bytes;
    it.V = static_cast<const char*>(a.v_own) + bk * a.cap * row_bytes;
    const int64_t row = (bk * a.plan.own + piece) * a.GRP;
    it.part = a.part_o + row * kHD;
    it.ml = a.ml_o + row;
    it.raw_stride = raw_stride(a.cap);
    it.raw = a.own_score ? a.raw + bk * a.GRP * it.raw_stride : nullptr;
    it.narrow = true;
    return true;
}

// eight floats as three 16-byte operands, the exact bf16 parts of each
__device__ __forceinline__ void split3_8(const float (&x)[8], bf16x8 (&part)[3]) {
    uint32_t p[3][4];
#pragma unroll
    for (int e = 0; e < 4; ++e) split3_pair(x[2 * e], x[2 * e + 1], p[0][e], p[1][e], p[2][e]);
#pragma unroll
    for (int q = 0; q < 3; ++q) part[q] = __builtin_bit_cast(bf16x8, make_uint4(p[q][0], p[q][1], p[q][2], p[q][3]));
}

// Query row r16 of a wave's 16 (past the last: the last again), dims 32 c + 8 g4 .. + 7, in NP parts.
template <int NP, class X8>
__device__ __forceinline__ void load_query(const AttnBatchArgs& a, const Item& it, int first, int r16, int g4, X8 (&q)[NP][8]) {
    const uint4* src = static_cast<const uint4*>(a.Qs) + (it.q0 + min(first + r16, it.rows - 1)) * NP * 32 + g4;
#pragma unroll
    for (int p = 0; p < NP; ++p)
#pragma unroll
        for (int c = 0; c < 8; ++c) q[p][c] = __builtin_bit_cast(X8, src[32 * p + 4 * c]);
}

// max and sum over the four lanes r16 + 16 g of a query (the 16- and 32-lane swaps of gfx950)
template <class F>
__device__ __forceinline__ float over_query(float v, F&& f) {
    auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(int, v), __builtin_bit_cast(int, v), false, false);
    v = f(__builtin_bit_cast(float, static_cast<int>(r[0])), __builtin_bit_cast(float, static_cast<int>(r[1])));
    r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(int, v), __builtin_bit_cast(int, v), false, false);
    return f(__builtin_bit_cast(float, static_cast<int>(r[0])), __builtin_bit_cast(float, static_cast<int>(r[1])));
}
__device__ __forceinline__ float query_max(float v) {
    return over_query(v, [](float x, float y) { return fmaxf(x, y); });
}
__device__ __forceinline__ float query_sum(float v) {
    return over_query(v, [](float x, float y) { return x + y; });
}

// Online softmax of N scores of the lane's query (four lanes r16 + 16 g share it), each s times the
// power of two `unit`: s becomes weights, (m, l) the query's running maximum (in the units of s) and
// sum. Returns the factor of the output so far. The reference maximum moves only when a score
// exceeds it by more than 8 / unit, so weights reach e^8. e^y as the native 2^(y log2 e) of the
// exactly formed exponent. The maximum starts at kNoMax: with a score of -inf alone it stays there, and the
// weight is 0.
constexpr float kNoMax = -3.402823466e38f;  // the lowest float
template <int N>
__device__ __forceinline__ float softmax_step(float (&s)[N], float unit, float& m, float& l) {
    float tm;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(tm) : "v"(s[0]), "v"(s[1]), "v"(s[2]));
#pragma unroll
    for (int i = 3; i + 1 < N; i += 2) asm("v_max3_f32 %0, %0, %1, %2" : "+v"(tm) : "v"(s[i]), "v"(s[i + 1]));
    if constexpr (N % 2 == 0) asm("v_max_f32 %0, %0, %1" : "+v"(tm) : "v"(s[N - 1]));
    tm = query_max(tm);
    const float k = unit * kLog2e;
    const float m_new = (tm - m) * unit > 8.0f ? tm : m;
    const float f = __builtin_amdgcn_exp2f((m - m_new) * k);
    float ps = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        s[i] = __builtin_amdgcn_exp2f((s[i] - m_new) * k);
        ps += s[i];
    }
    l = l * f + query_sum(ps);
    m = m_new;
    return f;
}

// the lane's outputs times its query's factor, which is mostly 1
template <int N>
__device__ __forceinline__ void rescale(float f, floatx4 (&o)[N]) {
    if (!__any(f != 1.0f)) return;
#pragma unroll
    for (int t = 0; t < N; ++t) o[t] *= f;
}

// The 16-byte chunk (dims 8 c ..) of row r of a 32-key tile of bf16 lies in LDS at chunk
// 32 r + (c ^ f(r)): f(r) = r % 16 for keys, so that the 16 rows that one operand read takes
// lie on all 64 banks, and 2 r % 16 for values, whose transposed reads take two neighbouring
// chunks of eight rows.
__device__ __forceinline__ int k_off(int r16, int g4) { return r16 * 512 + ((g4 ^ r16) << 4); }   // ^ (c << 6)
__device__ __forceinline__ int v_off(int r16, int g4) {                                            // ^ (t << 5)
    const int row = 4 * g4 + (r16 >> 2);
    return row * 512 + ((((2 * row) & 15) + ((r16 & 3) >> 1)) << 4) + (r16 & 1) * 8;
}

// Order of a run of STEPS steps of READS LDS reads and PRODUCTS matrix products on what they
// return: the reads of two steps first, then those of each next step under the products of one
// (left alone, the compiler reads and waits step by step, 100 to 200 cycles each).
template <int STEPS, int READS, int PRODUCTS>
__device__ __forceinline__ void reads_ahead() {
    constexpr int kRead = 0x100, kProduct = 0x8, kAhead = STEPS < 2 ? STEPS : 2;
    __builtin_amdgcn_sched_group_barrier(kRead, kAhead * READS, 0);
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        __builtin_amdgcn_sched_group_barrier(kProduct, PRODUCTS, 0);
        if (i + kAhead < STEPS) __builtin_amdgcn_sched_group_barrier(kRead, READS, 0);
    }
}

// scores of keys past the last
__device__ __forceinline__ void mask_tail(float (&s)[8], int k0, int hi, int g4) {
    if (k0 + kKT <= hi) return;  // uniform
    asm volatile("");            // (a branch: seventeen instructions that only the last tile needs)
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (k0 + 16 * (i >> 2) + 4 * g4 + (i & 3) >= hi) s[i] = -INFINITY;
}

// dims 16 t + r16 of keys 4 g4 .. + 3 of the tile's first half, then of its second
template <class X8>
__device__ __forceinline__ X8 v_operand(const uint4* V, int off) {
    typedef __attribute__((address_space(3))) i16x4 lds4;
    const char* p = reinterpret_cast<const char*>(V) + off;
    const i16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)p);
    const i16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(p + 16 * 512));
    const i16x8 x = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(X8, x);
}

// One 32-key tile of a bf16 cache for the 16 query rows of a wave, on v_mfma_f32_16x16x32_bf16.
// Queries and weights are the exact sums of three bf16 parts, K and V one part as they are, so every
// product is exact in fp32.
//   S^T = K Q^T by 16-key halves: lane (r16, g4) ends with keys 4 g4 + v of both for query r16
//   O^T += V^T P^T: those eight weights are the B operand as they lie, its k slots 8 g4 .. + 7
//         being keys 4 g4 .. + 3 of the first half and of the second, which transposed LDS reads
//         give V too; lane (r16, g4) ends with dims 16 t + 4 g4 + v of query r16, so that a
//         query's factors stay in its lanes
// T tiles of 16 dims from t0 on (a narrow workgroup's waves share the dims and each form all scores).
template <int T>
__device__ __forceinline__ void bf16_tile(const uint4 (&Kc)[1024], const uint4 (&Vc)[1024], const bf16x8 (&qp)[3][8], int k0,
                                          int hi, int r16, int g4, int t0, float* raw, float& m, float& l, floatx4 (&o)[T]) {
    floatx4 St[2];
    int ko = k_off(r16, g4), vo = v_off(r16, g4);
    asm volatile("" : "+v"(ko), "+v"(vo));  // formed per tile: kept, the 24 addresses would spill
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
        floatx4 sa[2], sb[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) sa[e] = sb[e] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < 8; c += 2) {
            bf16x8 k[2];
#pragma unroll
            for (int e = 0; e < 2; ++e)
                k[e] = *reinterpret_cast<const bf16x8*>(reinterpret_cast<const char*>(Kc) + hf * 16 * 512 + (ko ^ ((c + e) << 6)));
#pragma unroll
            for (int e = 0; e < 2; ++e) sb[e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k[e], qp[2][c + e], sb[e], 0, 0, 0);
#pragma unroll
            for (int e = 0; e < 2; ++e) sa[e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k[e], qp[0][c + e], sa[e], 0, 0, 0);
#pragma unroll
            for (int e = 0; e < 2; ++e) sb[e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k[e], qp[1][c + e], sb[e], 0, 0, 0);
        }
        St[hf] = (sb[0] + sb[1]) + (sa[0] + sa[1]);
    }
    reads_ahead<8, 2, 6>();
    float p[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = St[i >> 2][i & 3];
    if (raw) {  // (rows of raw are whole tiles)
        *reinterpret_cast<floatx4*>(raw + k0 + 4 * g4) = St[0];
        *reinterpret_cast<floatx4*>(raw + k0 + 16 + 4 * g4) = St[1];
    }
    mask_tail(p, k0, hi, g4);
    rescale(softmax_step(p, 1.0f, m, l), o);
    bf16x8 pa[3];
    split3_8(p, pa);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int t = 0; t < T; t += 2) {
        bf16x8 v[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) v[e] = v_operand<bf16x8>(Vc, vo ^ ((t0 + t + e) << 5));
#pragma unroll
        for (int q = 2; q >= 0; --q)
#pragma unroll
            for (int e = 0; e < 2; ++e) o[t + e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v[e], pa[q], o[t + e], 0, 0, 0);
    }
    reads_ahead<T / 2, 4, 6>();
}

// A wave's unnormalised output (dims 16 (t0 + t) + 4 g4 + v of row first + r16) and, from the
// wave that is asked, the rows' (max, sum).
template <int T>
__device__ __forceinline__ void store_part(const Item& it, int first, int r16, int g4, int t0, const floatx4 (&o)[T], float m,
                                           float l, bool with_ml) {
    const int row = first + r16;
    if (row >= it.rows) return;
    float* dst = it.part + static_cast<int64_t>(row) * kHD + 16 * t0 + 4 * g4;
#pragma unroll
    for (int t = 0; t < T; ++t) *reinterpret_cast<floatx4*>(dst + 16 * t) = o[t];
    if (with_ml && g4 == 0) it.ml[row] = make_float2(m, l);
}

// 16 bytes a lane from memory straight into LDS: lane i's go to dst + i.
__device__ __forceinline__ void copy_16(const uint4* src, uint4* dst) {
    __builtin_amdgcn_global_load_lds(reinterpret_cast<const __attribute__((address_space(1))) void*>(reinterpret_cast<uintptr_t>(src)),
                                     (__attribute__((address_space(3))) void*)dst, 16, 0, 0);
}

// bf16 caches: four waves, two workgroups per compute unit. Tiles are copied from memory
// straight into LDS (16 bytes a lane, the swizzle in the source address), the next one while
// this one is multiplied. Wide: 64 query rows, 16 a wave. Narrow: 16 rows, the waves share the
// dims of P V.
__global__ __launch_bounds__(256, 2) void attn_batch_bf16_kernel(AttnBatchArgs a) {
    // (separate arrays: the compiler then knows that a copy into one need not be waited for
    // before reads of another)
    __shared__ __align__(16) uint4 K0[1024], V0[1024], K1[1024], V1[1024];
    Item it;
    if (!item_of(a, blockIdx.x, it)) return;
    const int lane = threadIdx.x & 63, r16 = lane & 15, g4 = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    auto copy = [&](int k0, uint4* K, uint4* V) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {  // two rows of K and of V per instruction
            const int c = 64 * (4 * wave + j), row = 2 * (4 * wave + j) + (lane >> 5), pos = lane & 31;
            const int64_t at = static_cast<int64_t>(min(k0 + row, it.hi - 1)) * 32;
            const uint4* ks = static_cast<const uint4*>(it.K) + at + (pos ^ (row & 15));
            const uint4* vs = static_cast<const uint4*>(it.V) + at + (pos ^ ((2 * row) & 15));
            copy_16(ks, K + c);
            copy_16(vs, V + c);
        }
    };
    copy(it.lo, K0, V0);
    const int first = it.narrow ? it.row0 : it.row0 + 16 * wave;
    bf16x8 qp[3][8];
    load_query(a, it, first, r16, g4, qp);
    float m = kNoMax, l = 0.0f;
    auto walk = [&](auto& o, int t0, float* raw, bool live) {
#pragma unroll
        for (auto& x : o) x = floatx4{0.f, 0.f, 0.f, 0.f};
        auto tile = [&](int k0, const uint4 (&Kc)[1024], const uint4 (&Vc)[1024], uint4* Kn, uint4* Vn) {
            __builtin_amdgcn_s_waitcnt(kWaitVm);  // this wave's share of the tile
            lds_barrier();                        // every share; every wave is done with the other buffer
            if (k0 + kKT < it.hi) copy(k0 + kKT, Kn, Vn);  // uniform
            if (live) bf16_tile(Kc, Vc, qp, k0, it.hi, r16, g4, t0, raw, m, l, o);
        };
        for (int k0 = it.lo; k0 < it.hi; k0 += 2 * kKT) {
            tile(k0, K0, V0, K1, V1);
            if (k0 + kKT < it.hi) tile(k0 + kKT, K1, V1, K0, V0);
        }
    };
    if (it.narrow) {
        floatx4 o[4];
        float* raw = it.raw && wave == 0 && r16 < it.rows ? it.raw + r16 * it.raw_stride : nullptr;
        walk(o, 4 * wave, raw, true);
        store_part(it, first, r16, g4, 4 * wave, o, m, l, wave == 0);
    } else {
        floatx4 o[16];
        walk(o, 0, nullptr, first < it.rows);
        store_part(it, first, r16, g4, 0, o, m, l, true);
    }
}

// eight floats times s as two fp16 parts h = fp16(x), l = fp16(x - h): |x - h - l| <= 2^-23 |x|
// (the mixed-precision fused multiply-adds round straight to fp16; in instructions: the compiler
// forms the upper h twice, five for a pair instead of four)
__device__ __forceinline__ void split2_8(const float (&x)[8], float s, halfx8 (&part)[2]) {
    uint32_t h[4], l[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        asm("v_fma_mixlo_f16 %0, %1, %2, 0" : "=v"(h[e]) : "v"(x[2 * e]), "v"(s));
        asm("v_fma_mixhi_f16 %0, %1, %2, 0" : "+v"(h[e]) : "v"(x[2 * e + 1]), "v"(s));
        asm("v_fma_mixlo_f16 %0, %1, %2, -%3 op_sel_hi:[0,0,1]" : "=v"(l[e]) : "v"(x[2 * e]), "v"(s), "v"(h[e]));
        asm("v_fma_mixhi_f16 %0, %1, %2, -%3 op_sel:[0,0,1] op_sel_hi:[0,0,1]" : "+v"(l[e]) : "v"(x[2 * e + 1]), "v"(s), "v"(h[e]));
    }
    part[0] = __builtin_bit_cast(halfx8, make_uint4(h[0], h[1], h[2], h[3]));
    part[1] = __builtin_bit_cast(halfx8, make_uint4(l[0], l[1], l[2], l[3]));
}
// largest |x| (in instructions: the compiler would first quieten each operand)
__device__ __forceinline__ float max8(const float (&x)[8]) {
    float m;
    asm("v_max3_f32 %0, |%1|, |%2|, |%3|" : "=v"(m) : "v"(x[0]), "v"(x[1]), "v"(x[2]));
    asm("v_max3_f32 %0, %0, |%1|, |%2|" : "+v"(m) : "v"(x[3]), "v"(x[4]));
    asm("v_max3_f32 %0, %0, |%1|, |%2|" : "+v"(m) : "v"(x[5]), "v"(x[6]));
    return fmaxf(m, fabsf(x[7]));
}
// A tile of an fp32 cache in LDS: two fp16 parts of K and of V, and what undoes their rows' scales.
//
// fp32 caches run on v_mfma_f32_16x16x32_f16. Every operand row (a query, a key, a value row, a
// query's weights over the tile) is scaled by a power of two that brings its largest entry into
// [2^14, 2^15) and split into two fp16 parts; the three part products of lowest order are summed
// (the fourth is below 2^-22 of the product) and the scales undone exactly: a key's in the scores,
// a value row's in the weights before their own scaling, and that one, which the output is kept in,
// at the end. The weights' scale is set by the largest weight times value row of a tile where
// the softmax's reference moves and where it would be left upwards, so nothing is lost relative to the
// largest such product so far, whatever rows lie beside it.
struct alignas(1024) F32Tile {  // (aligned, so that a swizzled offset is one exclusive or on the address)
    uint4 K[2][1024], V[2][1024];
    float kscale[kKT], vscale[kKT];
};
struct F32Query {
    halfx8 p[2][8];  // row first + r16, dims 32 c + 8 g4 .. + 7
    float scale;
};

// Dims 8 c .. + 7 and 128 + 8 c .. + 7 of row `row` of a tile's K or V: 16 lanes hold the row.
__device__ __forceinline__ void f32_stage(F32Tile& tile, bool v, int row, int c, const floatx4 (&y)[4]) {
    float x[2][8];
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i >> 3][i & 7] = y[i >> 2][i & 3];
    uint32_t mx = __float_as_uint(fmaxf(max8(x[0]), max8(x[1])));
    mx = max(mx, static_cast<uint32_t>(dpp_i<0xB1>(mx)));
    mx = max(mx, static_cast<uint32_t>(dpp_i<0x4E>(mx)));
    mx = max(mx, static_cast<uint32_t>(dpp_i<0x141>(mx)));
    mx = max(mx, static_cast<uint32_t>(dpp_i<0x140>(mx)));
    const int e = row_exp(mx);
    const int at = 32 * row + (c ^ ((v ? 2 * row : row) & 15));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        halfx8 p[2];
        split2_8(x[i], pow2(e), p);
#pragma unroll
        for (int q = 0; q < 2; ++q) (v ? tile.V : tile.K)[q][at + 16 * i] = __builtin_bit_cast(uint4, p[q]);
    }
    if (c == 0) (v ? tile.vscale : tile.kscale)[row] = row_scale(mx, v ? e : e + kScoreExp);
}

// Byte address in LDS, to be offset by exclusive or.
__device__ __forceinline__ uint32_t lds_at(const void* p) {
    return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const void*)p));
}
template <class X>
__device__ __forceinline__ X lds_read(uint32_t at) {
    return *reinterpret_cast<__attribute__((address_space(3))) const X*>(static_cast<uintptr_t>(at));
}

// Scores of query r16 of the wave, over its scale (the stored one, with 2^kScoreExp): keys 4 g4 + v of the tile's first half, then of
// its second.
__device__ __forceinline__ void f32_scores(const F32Tile& tile, const F32Query& q, int r16, int g4, float (&p)[8]) {
    uint32_t ko = lds_at(&tile) + k_off(r16, g4);
    asm volatile("" : "+v"(ko));  // addresses formed per tile: kept, they would spill
    floatx4 St[2];
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
        floatx4 s[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) s[e] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < 8; c += 2) {
            halfx8 k[2][2];
#pragma unroll
            for (int h = 1; h >= 0; --h)
#pragma unroll
                for (int e = 0; e < 2; ++e) k[h][e] = lds_read<halfx8>((ko ^ ((c + e) << 6)) + h * 16384 + hf * 8192);
#pragma unroll
            for (int e = 0; e < 2; ++e) s[e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[1][e], q.p[0][c + e], s[e], 0, 0, 0);
#pragma unroll
            for (int e = 0; e < 2; ++e) s[e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[0][e], q.p[1][c + e], s[e], 0, 0, 0);
#pragma unroll
            for (int e = 0; e < 2; ++e) s[e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[0][e], q.p[0][c + e], s[e], 0, 0, 0);
        }
        St[hf] = s[0] + s[1];
    }
    reads_ahead<8, 4, 6>();
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
        const floatx4 ks = *reinterpret_cast<const floatx4*>(tile.kscale + 16 * hf + 4 * g4);
#pragma unroll
        for (int v = 0; v < 4; ++v) p[4 * hf + v] = St[hf][v] * ks[v];
    }
}

// O^T += V^T P^T, O in units of 2^-exp for the lane's query; f: the softmax's factor of O so far.
__device__ __forceinline__ void f32_output(const F32Tile& tile, float (&p)[8], float f, int r16, int g4, int& exp, floatx4 (&o)[16]) {
    uint32_t vo = lds_at(&tile) + 32768 + v_off(r16, g4);
    asm volatile("" : "+v"(vo));
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
        const floatx4 vs = *reinterpret_cast<const floatx4*>(tile.vscale + 16 * hf + 4 * g4);
#pragma unroll
        for (int v = 0; v < 4; ++v) p[4 * hf + v] *= vs[v];
    }
    const int e = row_exp(__float_as_uint(query_max(max8(p))));  // the largest weight is brought to [2^14, 2^15)
    const bool move = f != 1.0f || e < exp;
    if (__any(move)) {
        int to = move ? e : exp;
        if (__any(to > exp && f > 0.0f)) {
            // up no further than keeps O, by its present largest, below 2^90 (a tile adds less than 2^36, and
            // terms that it would take further are below 2^-59 of that largest)
            float mx = 0.0f;
#pragma unroll
            for (int t = 0; t < 16; ++t)
                mx = fmaxf(fmaxf(fmaxf(mx, fabsf(o[t][0])), fmaxf(fabsf(o[t][1]), fabsf(o[t][2]))), fabsf(o[t][3]));
            mx = query_max(mx) * f;
            if (mx > 0.0f) to = min(to, exp + max(216 - static_cast<int>(__float_as_uint(mx) >> 23), 0));
        }
        const int step = to - exp;
        const int s1 = min(max(step, -126), 126), s2 = min(max(step - s1, -126), 126);
        const float g = (f * pow2(s1)) * pow2(s2);
#pragma unroll
        for (int t = 0; t < 16; ++t) o[t] *= g;
        exp = to;
    }
    halfx8 pp[2];
    split2_8(p, pow2(exp), pp);
    asm("s_nop 1" : "+v"(pp[0]), "+v"(pp[1]));  // two states between a vector write and a product's read (the compiler sees no such write)
    // steps of 32 dims: the next but one's reads go with this one's products
    constexpr int kAhead = 2, kSteps = 8;
    halfx8 v[kAhead + 1][2][2];
    const auto read = [&](int u) {
        typedef __attribute__((address_space(3))) i16x4 lds4;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int d = 0; d < 2; ++d) {
                const uint32_t at = (vo ^ ((2 * u + d) << 5)) + h * 16384;
                const i16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds4*>(static_cast<uintptr_t>(at)));
                const i16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds4*>(static_cast<uintptr_t>(at + 8192)));
                const i16x8 z = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
                v[u % (kAhead + 1)][h][d] = __builtin_bit_cast(halfx8, z);
            }
    };
#pragma unroll
    for (int u = 0; u < kAhead; ++u) read(u);
#pragma unroll
    for (int u = 0; u < kSteps; ++u) {
        __builtin_amdgcn_sched_barrier(0);
        if (u + kAhead < kSteps) read(u + kAhead);
        const halfx8(&w)[2][2] = v[u % (kAhead + 1)];
#pragma unroll
        for (int d = 0; d < 2; ++d) o[2 * u + d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w[0][d], pp[1], o[2 * u + d], 0, 0, 0);
#pragma unroll
        for (int d = 0; d < 2; ++d) o[2 * u + d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w[1][d], pp[0], o[2 * u + d], 0, 0, 0);
#pragma unroll
        for (int d = 0; d < 2; ++d) o[2 * u + d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w[0][d], pp[0], o[2 * u + d], 0, 0, 0);
    }
}

// Wide: 128 query rows, 16 a wave. Tiles come through registers and are split once for all waves
// into the other of two buffers, one barrier a tile. Of the two waves that share a matrix core one
// stages before its products with K and the other after, so that one's vector work runs beside the
// other's products. A product takes its matrix core 17.5 cycles and an issue slot 9, a vector
// instruction 4: a tile's 192 products and 620 vector instructions take a core 4300 of its 5200 cycles. 3.1 us
// a tile of 128 rows and 32 keys, 1040 TFLOP/s in fp16 products over the compute units, where a large
// fp16 matrix product reaches 1221. (Four waves of 32 rows, which read half as much of LDS, softmax and
// staging interleaved with the products one by one: 4.0 us.)
__device__ __forceinline__ void f32_wide(const AttnBatchArgs& a, const Item& it, F32Tile* tiles) {
    const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, g4 = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int first = it.row0 + 16 * wave;
    const bool live = first < it.rows;  // uniform per wave
    floatx4 st[2][4];  // dims 8 c .. + 7 and 128 + 8 c .. + 7 of a row of K, of V
    const int row = tid >> 4, c = tid & 15;
    const auto load = [&](int k0) {
        const int64_t at = static_cast<int64_t>(min(k0 + row, it.hi - 1)) * kHD + 8 * c;
#pragma unroll
        for (int v = 0; v < 2; ++v) {
            const floatx4* src = reinterpret_cast<const floatx4*>(static_cast<const float*>(v ? it.V : it.K) + at);
#pragma unroll
            for (int i = 0; i < 4; ++i) st[v][i] = src[(i >> 1) * 32 + (i & 1)];
        }
    };
    const auto stage = [&](F32Tile& dst) {
#pragma unroll
        for (int v = 0; v < 2; ++v) f32_stage(dst, v, row, c, st[v]);
    };
    load(it.lo);
    F32Query q;
    load_query(a, it, first, r16, g4, q.p);
    q.scale = a.Qscale[it.q0 + min(first + r16, it.rows - 1)];
    stage(tiles[0]);
    load(it.lo + kKT);  // (past the end: the last row again)
    float m = kNoMax, l = 0.0f;
    int exp = 100;
    floatx4 o[16];
#pragma unroll
    for (auto& x : o) x = floatx4{0.f, 0.f, 0.f, 0.f};
    lds_barrier();
    int cur = 0;
    for (int k0 = it.lo; k0 < it.hi; k0 += kKT) {
        const bool more = k0 + kKT < it.hi;  // uniform
        const auto next = [&]() {
            if (!more) return;
            stage(tiles[cur ^ 1]);
            load(k0 + 2 * kKT);
        };
        if (wave < 4) next();
        float p[8], f = 1.0f;
        if (live) {
            __builtin_amdgcn_s_setprio(1);  // products before the other wave's vector work: 2% of the whole
            f32_scores(tiles[cur], q, r16, g4, p);
            __builtin_amdgcn_s_setprio(0);
            mask_tail(p, k0, it.hi, g4);
            f = softmax_step(p, q.scale, m, l);
        }
        if (wave >= 4) next();
        __builtin_amdgcn_s_setprio(1);
        if (live) f32_output(tiles[cur], p, f, r16, g4, exp, o);
        __builtin_amdgcn_s_setprio(0);
        cur ^= 1;
        lds_barrier();  // every wave is done with this tile, every share of the next one is in
    }
    if (!live) return;
#pragma unroll
    for (auto& x : o) x *= pow2(-exp);
    store_part(it, first, r16, g4, 0, o, m * q.scale, l, true);
}

// Narrow: 16 query rows on v_mfma_f32_16x16x4_f32, K and V straight from memory as its operands, no
// staging and no barrier in the loop (splitting a tile costs more vector work than its products
// here: 2.4 us a tile against 1.4). The eight waves take 16 keys in turn and are merged at the end.
//   S^T = K Q^T: lane (r16, g4) loads dims 16 u + 4 g4 .. + 3 of key r16; the k slot g4 of product
//         (u, e) is dim 16 u + 4 g4 + e on both sides
//   O^T += V^T P^T: product (v, t, e) takes the weights of keys 4 g4 + v as they lie and dims
//         64 t + 4 r16 + e of those keys; lane (r16, g4) ends with dims 64 t + 16 g4 + 4 i + e of
//         query r16 in o[4 t + e][i]
// K and V of the wave's next 16 keys are on their way while this 16's products run; the queries are
// read from LDS as they are needed, which is what leaves registers for both.
__device__ __forceinline__ void f32_narrow(const AttnBatchArgs& a, const Item& it, float* buf, float (*ms)[16], float (*ls)[16]) {
    const int lane = threadIdx.x & 63, r16 = lane & 15, g4 = lane >> 4, wave = threadIdx.x >> 6;
    const float *K = static_cast<const float*>(it.K), *V = static_cast<const float*>(it.V);
    float4 k[16], vv[4][4];
    const auto load_k = [&](int k0) {  // keys past the last: it again
        const float* kr = K + static_cast<int64_t>(min(k0 + r16, it.hi - 1)) * kHD + 4 * g4;
#pragma unroll
        for (int u = 0; u < 16; ++u) k[u] = *reinterpret_cast<const float4*>(kr + 16 * u);
    };
    const auto load_v = [&](int k0) {
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            const float* vr = V + static_cast<int64_t>(min(k0 + 4 * g4 + v, it.hi - 1)) * kHD + 4 * r16;
#pragma unroll
            for (int t = 0; t < 4; ++t) vv[v][t] = *reinterpret_cast<const float4*>(vr + 64 * t);
        }
    };
    const int first = it.lo + 16 * wave;
    // query rows 2 wave, + 1 into LDS, a row's 16-byte chunks c at c ^ row (rows past the last: it again)
    float4 qrow[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
        qrow[i] = *reinterpret_cast<const float4*>(a.Qa + (it.q0 + min(it.row0 + 2 * wave + i, it.rows - 1)) * kHD + 4 * lane);
    load_k(first);
    load_v(first);
#pragma unroll
    for (int i = 0; i < 2; ++i)
        *reinterpret_cast<float4*>(buf + (2 * wave + i) * kHD + 4 * (lane ^ (2 * wave + i))) = qrow[i];
    lds_barrier();
    float* raw = it.raw && r16 < it.rows ? it.raw + r16 * it.raw_stride : nullptr;
    float m = kNoMax, l = 0.0f;
    floatx4 o[16];
#pragma unroll
    for (auto& x : o) x = floatx4{0.f, 0.f, 0.f, 0.f};
    int qo = r16 * kHD * 4 + ((g4 ^ r16) << 4);  // bytes; ^ (u << 6): chunk 4 u + g4
    for (int k0 = first; k0 < it.hi; k0 += 128) {
        const bool more = k0 + 128 < it.hi;  // uniform per wave
        asm volatile("" : "+v"(qo));
        floatx4 s[4];
#pragma unroll
        for (auto& x : s) x = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < 16; ++u) {
            const float4 q = *reinterpret_cast<const float4*>(reinterpret_cast<const char*>(buf) + (qo ^ (u << 6)));
            s[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[u].x, q.x, s[0], 0, 0, 0);
            s[1] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[u].y, q.y, s[1], 0, 0, 0);
            s[2] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[u].z, q.z, s[2], 0, 0, 0);
            s[3] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[u].w, q.w, s[3], 0, 0, 0);
        }
        reads_ahead<16, 1, 4>();
        __builtin_amdgcn_sched_barrier(0);
        if (more) load_k(k0 + 128);
        const floatx4 St = (s[0] + s[1]) + (s[2] + s[3]);
        if (raw) *reinterpret_cast<floatx4*>(raw + k0 + 4 * g4) = St;  // (rows of raw are whole tiles)
        float p[4];
#pragma unroll
        for (int v = 0; v < 4; ++v) p[v] = k0 + 4 * g4 + v < it.hi ? St[v] : -INFINITY;
        rescale(softmax_step(p, 1.0f, m, l), o);
#pragma unroll
        for (int v = 0; v < 4; ++v)
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                o[4 * t] = __builtin_amdgcn_mfma_f32_16x16x4f32(vv[v][t].x, p[v], o[4 * t], 0, 0, 0);
                o[4 * t + 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(vv[v][t].y, p[v], o[4 * t + 1], 0, 0, 0);
                o[4 * t + 2] = __builtin_amdgcn_mfma_f32_16x16x4f32(vv[v][t].z, p[v], o[4 * t + 2], 0, 0, 0);
                o[4 * t + 3] = __builtin_amdgcn_mfma_f32_16x16x4f32(vv[v][t].w, p[v], o[4 * t + 3], 0, 0, 0);
            }
        __builtin_amdgcn_sched_barrier(0);
        if (more) load_v(k0 + 128);
    }
    // merge of the waves; one without keys has maximum kNoMax, and output and sum 0
    if (g4 == 0) {
        ms[wave][r16] = m;
        ls[wave][r16] = l;
    }
    lds_barrier();  // (and every wave is done with the queries)
    float top = ms[0][r16];
#pragma unroll
    for (int w = 1; w < 8; ++w) top = fmaxf(top, ms[w][r16]);
    rescale(__builtin_amdgcn_exp2f((m - top) * kLog2e), o);
    const int n = min(16, it.rows - it.row0);
    if (wave == 0 && g4 == 0 && r16 < n) {
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < 8; ++w) sum += ls[w][r16] * __builtin_amdgcn_exp2f((ms[w][r16] - top) * kLog2e);
        it.ml[it.row0 + r16] = make_float2(top, sum);
    }
    // (rows' 16-byte chunks c at c ^ row % 16: the 16 lanes of a store lie on all banks)
    if (r16 < n) {
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<float4*>(buf + (wave * 16 + r16) * kHD + 4 * ((16 * t + 4 * g4 + i) ^ r16)) =
                    make_float4(o[4 * t][i], o[4 * t + 1][i], o[4 * t + 2][i], o[4 * t + 3][i]);
    }
    lds_barrier();
    for (int r = wave; r < n; r += 8) {
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < 8; ++w) {
            const float4 x = *reinterpret_cast<const float4*>(buf + (w * 16 + r) * kHD + 4 * (lane ^ r));
            y.x += x.x, y.y += x.y, y.z += x.z, y.w += x.w;
        }
        *reinterpret_cast<float4*>(it.part + static_cast<int64_t>(it.row0 + r) * kHD + 4 * lane) = y;
    }
}

// fp32 caches: eight waves, one workgroup per compute unit.
__global__ __launch_bounds__(512, 1) void attn_batch_f32_kernel(AttnBatchArgs a) {
    __shared__ __align__(16) F32Tile tiles[2];
    __shared__ float small[2][8][16];
    Item it;
    if (!item_of(a, blockIdx.x, it)) return;
    if (it.narrow) f32_narrow(a, it, reinterpret_cast<float*>(tiles), small[0], small[1]);
    else f32_wide(a, it, tiles);
}

constexpr int kCombWaves = 8, kCombAhead = 8;

// The (max, sum) of piece i of row g of (b, kh): the prefix's pieces, then the own cache's.
__device__ __forceinline__ int64_t piece_row(const AttnBatchArgs& a, int b, int kh, int g, int i) {
    return i < a.plan.pieces
               ? (static_cast<int64_t>(kh) * a.plan.pieces + i) * a.B * a.GRP + b * a.GRP + g
               : ((static_cast<int64_t>(b) * a.NKV + kh) * a.plan.own + i - a.plan.pieces) * a.GRP + g;
}
__device__ __forceinline__ float2 piece_ml(const AttnBatchArgs& a, int b, int kh, int g, int i) {
    return (i < a.plan.pieces ? a.ml_p : a.ml_o)[piece_row(a, b, kh, g, i)];
}
// (max, sum) over n pieces, by the lanes of a wave; first: the lane's first piece's
__device__ __forceinline__ float2 merge_ml(const AttnBatchArgs& a, int b, int kh, int g, int n, int lane, float2& first) {
    first = lane < n ? piece_ml(a, b, kh, g, lane) : make_float2(-INFINITY, 0.0f);
    float m = first.x;
    for (int i = lane + 64; i < n; i += 64) m = fmaxf(m, piece_ml(a, b, kh, g, i).x);
    m = wave_max(m);
    float l = first.y * __builtin_amdgcn_exp2f((first.x - m) * kLog2e);
    for (int i = lane + 64; i < n; i += 64) {
        const float2 x = piece_ml(a, b, kh, g, i);
        l += x.y * __builtin_amdgcn_exp2f((x.x - m) * kLog2e);
    }
    return make_float2(m, wave_sum(l));
}

// Workgroups [0, B NQ): one output row each. A wave takes every eighth piece, a lane four dims; the
// partial outputs of a wave's first pieces are on their way while the pieces' factors e^(their
// maximum - the row's) are formed, into LDS. Then the gate.
// The others (with own_score): 512 own rows of a (sequence, kv head) each: their weights, summed
// over the heads of the group in order, into the scores.
__global__ __launch_bounds__(kCombWaves * 64) void attn_batch_combine_kernel(AttnBatchArgs a) {
    extern __shared__ __align__(16) float fac[];  // a factor per piece
    __shared__ __align__(16) float part[kCombWaves][kHD];
    __shared__ float ms[16], ls[16];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rows = a.B * a.NQ;
    if (static_cast<int>(blockIdx.x) >= rows) {
        const int chunks = static_cast<int>((a.cap + 511) / 512);
        const int64_t bk = (blockIdx.x - rows) / chunks;
        const int chunk = (blockIdx.x - rows) % chunks;
        const int b = static_cast<int>(bk / a.NKV), kh = static_cast<int>(bk % a.NKV);
        const int slot = new_slot(a, b);
        if (slot < 0 || chunk * 512LL > slot) return;
        const int n = a.plan.pieces + slot / a.plan.okeys + 1;
        for (int g = wave; g < a.GRP; g += kCombWaves) {
            float2 first;
            const float2 x = merge_ml(a, b, kh, g, n, lane, first);
            if (lane == 0) ms[g] = x.x, ls[g] = 1.0f / x.y;
        }
        __syncthreads();
        const int64_t t = chunk * 512LL + tid;
        if (t > slot) return;
        float w = 0.0f;
        for (int g = 0; g < a.GRP; ++g)
            w += __builtin_amdgcn_exp2f((a.raw[(bk * a.GRP + g) * raw_stride(a.cap) + t] - ms[g]) * kLog2e) * ls[g];
        float* sc = a.own_score + bk * a.cap + t;
        *sc = t == slot ? w : *sc + w;
        return;
    }
    const int h = blockIdx.x % a.NQ, b = blockIdx.x / a.NQ;
    const int len = a.own_len[b];
    if (len < 0) return;
    float* out = a.out + (static_cast<int64_t>(b) * a.NQ + h) * kHD + 4 * lane;
    if (len >= a.cap) {
        if (wave == 0) *reinterpret_cast<float4*>(out) = make_float4(NAN, NAN, NAN, NAN);
        return;
    }
    const int kh = h / a.GRP, g = h - kh * a.GRP, n = a.plan.pieces + len / a.plan.okeys + 1;
    const float4 gate = *reinterpret_cast<const float4*>(a.qg + (static_cast<int64_t>(b) * a.NQ + h) * 2 * kHD + kHD + 4 * lane);
    const auto partial = [&](int i) {
        return *reinterpret_cast<const float4*>((i < a.plan.pieces ? a.part_p : a.part_o) + piece_row(a, b, kh, g, i) * kHD + 4 * lane);
    };
    float4 x[kCombAhead];
#pragma unroll
    for (int j = 0; j < kCombAhead; ++j)
        if (wave + j * kCombWaves < n) x[j] = partial(wave + j * kCombWaves);  // uniform
    float2 first;
    const float2 all = merge_ml(a, b, kh, g, n, lane, first);  // every wave the same
    if (tid < min(n, 64)) fac[tid] = __builtin_amdgcn_exp2f((first.x - all.x) * kLog2e);
    for (int i = tid + 64; i < n; i += kCombWaves * 64) fac[i] = __builtin_amdgcn_exp2f((piece_ml(a, b, kh, g, i).x - all.x) * kLog2e);
    lds_barrier();
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
    const auto add = [&](float4 v, float f) { y.x += v.x * f, y.y += v.y * f, y.z += v.z * f, y.w += v.w * f; };
#pragma unroll
    for (int j = 0; j < kCombAhead; ++j)
        if (wave + j * kCombWaves < n) add(x[j], fac[wave + j * kCombWaves]);
#pragma unroll 4
    for (int i = wave + kCombAhead * kCombWaves; i < n; i += kCombWaves) add(partial(i), fac[i]);
    *reinterpret_cast<float4*>(&part[wave][4 * lane]) = y;
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int w = 1; w < kCombWaves; ++w) {
        const float4 x = *reinterpret_cast<const float4*>(&part[w][4 * lane]);
        y.x += x.x, y.y += x.y, y.z += x.z, y.w += x.w;
    }
    *reinterpret_cast<float4*>(out) = make_float4((y.x / all.y) * sigmoid_f(gate.x), (y.y / all.y) * sigmoid_f(gate.y),
                                                  (y.z / all.y) * sigmoid_f(gate.z), (y.w / all.y) * sigmoid_f(gate.w));
}

struct Carve {
    int64_t q, qs, sc, pp, mp, po, mo, raw, total;  // float offsets, multiples of 4
    bool split;
};
Carve carve_of(const AttnBatchArgs& a) {
    const auto up4 = [](int64_t x) { return (x + 3) / 4 * 4; };
    const int64_t rows = static_cast<int64_t>(a.B) * a.NQ;
    const AttnBatchPlan p = attn_batch_plan(a.B, a.GRP, a.NKV, a.P, a.cap, a.kv_bf16, device_cu_count());
    Carve c{};
    c.split = a.kv_bf16 || p.block == batch_wide(false);
    c.q = 0;
    c.qs = c.q + (a.kv_bf16 ? 0 : rows * kHD);
    c.sc = c.qs + (a.kv_bf16 ? rows * (3 * kHD / 2) : c.split ? rows * kHD : 0);
    c.pp = c.sc + (c.split && !a.kv_bf16 ? up4(rows) : 0);
    c.mp = c.pp + rows * p.pieces * kHD;
    c.po = c.mp + up4(rows * p.pieces * 2);
    c.mo = c.po + rows * p.own * kHD;
    c.raw = c.mo + up4(rows * p.own * 2);
    c.total = c.raw + (a.own_score ? rows * raw_stride(a.cap) : 0);
    return c;
}

}  // namespace

int64_t attn_batch_workspace_floats(const AttnBatchArgs& a) { return carve_of(a).total; }

void attn_batch_carve(AttnBatchArgs& a, float* ws) {
    const Carve c = carve_of(a);
    a.plan = attn_batch_plan(a.B, a.GRP, a.NKV, a.P, a.cap, a.kv_bf16, device_cu_count());
    a.Qa = ws + c.q;
    a.Qs = c.split ? ws + c.qs : nullptr;
    a.Qscale = ws + c.sc;
    a.part_p = ws + c.pp;
    a.ml_p = reinterpret_cast<float2*>(ws + c.mp);
    a.part_o = ws + c.po;
    a.ml_o = reinterpret_cast<float2*>(ws + c.mo);
    a.raw = ws + c.raw;
}

bool attn_batch_launches(const AttnBatchArgs& a) {
    const AttnBatchPlan p = attn_batch_plan(a.B, a.GRP, a.NKV, a.P, a.cap, a.kv_bf16, device_cu_count());
    const int64_t pairs = static_cast<int64_t>(a.B) * a.NKV, most = UINT32_MAX;  // threads of a launch
    const int64_t attend = (static_cast<int64_t>(p.pieces) * a.NKV + 7) / 8 * 8 * p.nblk + pairs * p.own;
    const int64_t combine = static_cast<int64_t>(a.B) * a.NQ + (a.own_score ? (a.cap + 511) / 512 * pairs : 0);
    return attend <= most / (a.kv_bf16 ? 256 : 512) && combine <= most / (kCombWaves * 64);
}

hipError_t launch_attn_batch(const AttnBatchArgs& a, hipStream_t s) {
    // a function of theta and the width alone, kept for the next call of this host thread
    static thread_local RopeFreq freq;
    static thread_local double theta = 0.0;
    static thread_local int rot = -1;
    if (theta != a.theta || rot != a.ROT) {
        for (int i = 0; i < a.ROT / 2; ++i) freq.f[i] = std::pow(a.theta, -static_cast<double>(2 * i) / a.ROT);
        theta = a.theta;
        rot = a.ROT;
    }
    klaunch(attn_batch_prep_kernel, dim3((a.NQ + a.NKV + 3) / 4, a.B), 256, 0, s, a, freq);
    const uint32_t prefix = prefix_items(a.plan, a.NKV), own = a.B * a.NKV * a.plan.own;
    if (a.kv_bf16) klaunch(attn_batch_bf16_kernel, dim3(prefix + own), 256, 0, s, a);
    else klaunch(attn_batch_f32_kernel, dim3(prefix + own), 512, 0, s, a);
    const uint32_t scores = a.own_score ? static_cast<uint32_t>((a.cap + 511) / 512) * a.B * a.NKV : 0;
    klaunch(attn_batch_combine_kernel, dim3(a.B * a.NQ + scores), kCombWaves * 64, (a.plan.pieces + a.plan.own) * 4, s, a);
    return hipGetLastError();
}

}  // namespace q35k
