// Attention of a batch of continuations: one token per sequence over a prefix that all share
// and each sequence's own cache, in three launches: the queries and the appended rows
// (prep), partial outputs over pieces of the keys (attend), and their merge with the gate,
// which also adds the softmax weights to the own rows' scores (combine).
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

// grid ((NQ + NKV) / 4, B), a wave per row: rmsnorm (1 + w) + RoPE of a query row -> Qa, or of the
// new key row -> own cache, with its value row. Angles in double, one lane each.
__global__ __launch_bounds__(256) void attn_batch_prep_kernel(AttnBatchArgs a) {
    const int b = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = blockIdx.x * 4 + wave;
    __shared__ __align__(16) float buf[4][kHD];
    __shared__ float cs[2][kHD / 2];
    const int slot = new_slot(a, b);
    const bool is_q = r < a.NQ, there = r < a.NQ + a.NKV;
    const int kh = is_q ? r / a.GRP : min(r - a.NQ, a.NKV - 1);
    float* q = a.Qa + ((static_cast<int64_t>(kh) * a.B + b) * a.GRP + (r - kh * a.GRP)) * kHD + 4 * lane;
    if (slot < 0) {
        if (is_q) *reinterpret_cast<float4*>(q) = make_float4(0.f, 0.f, 0.f, 0.f);
        return;
    }
    const int64_t bk = static_cast<int64_t>(b) * a.NKV + kh;
    const float* src = is_q ? a.qg + (static_cast<int64_t>(b) * a.NQ + r) * 2 * kHD : a.k_new + bk * kHD;
    const float4 x = *reinterpret_cast<const float4*>(src + 4 * lane);
    const float4 w = *reinterpret_cast<const float4*>((is_q ? a.q_norm : a.k_norm) + 4 * lane);
    const float4 v = *reinterpret_cast<const float4*>(a.v_new + bk * kHD + 4 * lane);
    const int half = a.ROT / 2, pos = a.pos[b];
    for (int i = threadIdx.x; i < half; i += 256) {
        const double ang = static_cast<double>(pos) * pow(a.theta, -static_cast<double>(2 * i) / a.ROT);
        double sn, cn;
        sincos(ang, &sn, &cn);
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
        *reinterpret_cast<float4*>(q) = make_float4(y[0] * 0.0625f, y[1] * 0.0625f, y[2] * 0.0625f, y[3] * 0.0625f);
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

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef short i16x8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
constexpr float kLog2e = 1.44269504088896341f;
constexpr int kKT = 32;         // keys per tile of the 16-bit matrix products
constexpr int kWaitVm = 0x0f70; // s_waitcnt: vector memory, nothing outstanding

// What one workgroup does: rows [row0, rows) of one list of query rows over keys [lo, hi) of one
// cache, and where its partial result goes.
struct Item {
    const float* Q;         // query rows [rows][HD]
    int rows, row0;
    int lo, hi;
    const void *K, *V;      // row 0 of the cache
    float* part;            // [rows][HD]
    float2* ml;             // [rows]
    float* raw;             // scores of the rows, stride raw_stride, indexed by key (own caches; may be null)
    int64_t raw_stride;
    bool narrow;            // at most 16 rows, shared by the workgroup's waves
};

// Workgroups [0, prefix) are (piece, kv head, row block) of the prefix, the others (piece, kv
// head, sequence) of the own caches. Workgroups go to the 8 XCDs in turn: the row blocks that
// read one piece get numbers 8 apart, so that one L2 fetches it for all of them.
__device__ __forceinline__ bool item_of(const AttnBatchArgs& a, Item& it) {
    const int pairs = a.plan.pieces * a.NKV, groups = (pairs + 7) / 8;
    const int prefix = groups * 8 * a.plan.nblk;
    int i = blockIdx.x;
    const int64_t row_bytes = a.kv_bf16 ? kHD * 2 : kHD * 4;
    if (i < prefix) {
        const int blk = (i >> 3) % a.plan.nblk, pair = (i >> 3) / a.plan.nblk * 8 + (i & 7);
        if (pair >= pairs) return false;
        const int piece = pair / a.NKV, kh = pair - piece * a.NKV;
        it.rows = a.B * a.GRP;
        it.row0 = blk * a.plan.block;
        it.Q = a.Qa + static_cast<int64_t>(kh) * it.rows * kHD;
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
    const int piece = i % a.plan.own;
    i /= a.plan.own;
    const int kh = i % a.NKV, b = i / a.NKV;
    const int slot = new_slot(a, b);
    const int64_t lo = static_cast<int64_t>(piece) * a.plan.okeys;
    if (slot < 0 || lo > slot) return false;
    const int64_t bk = static_cast<int64_t>(b) * a.NKV + kh;
    it.rows = a.GRP;
    it.row0 = 0;
    it.Q = a.Qa + (static_cast<int64_t>(kh) * a.B + b) * a.GRP * kHD;
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

// Query row r16 of a wave's 16 (past the last: the last again), dims 32 c + 8 g4 .. + 7, as three
// bf16 parts.
__device__ __forceinline__ void load_query(const Item& it, int first, int r16, int g4, bf16x8 (&qp)[3][8]) {
    const float* src = it.Q + static_cast<int64_t>(min(first + r16, it.rows - 1)) * kHD + 8 * g4;
#pragma unroll
    for (int c = 0; c < 8; ++c) {
        const float4 u = *reinterpret_cast<const float4*>(src + 32 * c), w = *reinterpret_cast<const float4*>(src + 32 * c + 4);
        const float x[8] = {u.x, u.y, u.z, u.w, w.x, w.y, w.z, w.w};
        bf16x8 p[3];
        split3_8(x, p);
#pragma unroll
        for (int q = 0; q < 3; ++q) qp[q][c] = p[q];
    }
}

// Online softmax of N scores of the lane's query (four lanes r16 + 16 g share it): s becomes
// weights, (m, l) the query's running maximum and sum. Returns the factor of the output so
// far. The reference maximum moves only when a score exceeds it by more than 8; a query without
// a key yet keeps -inf and weight 0. e^y as the native 2^(y log2 e) of the exactly formed
// exponent.
template <int N>
__device__ __forceinline__ float softmax_step(float (&s)[N], float& m, float& l) {
    float tm = s[0];
#pragma unroll
    for (int i = 1; i < N; ++i) tm = fmaxf(tm, s[i]);
    tm = fmaxf(tm, __shfl_xor(tm, 16));
    tm = fmaxf(tm, __shfl_xor(tm, 32));
    const float m_new = tm > m + 8.0f ? tm : m;
    const bool live = m_new != -INFINITY;
    const float f = live ? __builtin_amdgcn_exp2f((m - m_new) * kLog2e) : 1.0f;
    float ps = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        s[i] = live ? __builtin_amdgcn_exp2f((s[i] - m_new) * kLog2e) : 0.0f;
        ps += s[i];
    }
    ps += __shfl_xor(ps, 16);
    ps += __shfl_xor(ps, 32);
    l = l * f + ps;
    m = m_new;
    return f;
}

// o[.][v] (query rows 4 g4 + v) times the factors of lanes 4 g4 + v
template <int N>
__device__ __forceinline__ void rescale(float f, int g4, floatx4 (&o)[N]) {
    if (!__any(f != 1.0f)) return;
    float fr[4];
#pragma unroll
    for (int v = 0; v < 4; ++v) fr[v] = __shfl(f, 4 * g4 + v);
#pragma unroll
    for (int t = 0; t < N; ++t)
#pragma unroll
        for (int v = 0; v < 4; ++v) o[t][v] *= fr[v];
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

// scores of keys past the last
__device__ __forceinline__ void mask_tail(float (&s)[8], int k0, int hi, int g4) {
    if (k0 + kKT <= hi) return;  // uniform
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
//   O += P V: those eight weights are the A operand as they lie, its k slots 8 g4 .. + 7 being
//         keys 4 g4 .. + 3 of the first half and of the second, which transposed LDS reads give V too;
//         lane (r16, g4) ends with dims 16 t + r16 of queries 4 g4 + v
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
        for (int c = 0; c < 8; ++c) {
            const bf16x8 k = *reinterpret_cast<const bf16x8*>(reinterpret_cast<const char*>(Kc) + hf * 16 * 512 + (ko ^ (c << 6)));
            sb[c & 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, qp[2][c], sb[c & 1], 0, 0, 0);
            sb[c & 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, qp[1][c], sb[c & 1], 0, 0, 0);
            sa[c & 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, qp[0][c], sa[c & 1], 0, 0, 0);
        }
        St[hf] = (sb[0] + sb[1]) + (sa[0] + sa[1]);
    }
    float p[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = St[i >> 2][i & 3];
    if (raw) {  // (rows of raw are whole tiles)
        *reinterpret_cast<floatx4*>(raw + k0 + 4 * g4) = St[0];
        *reinterpret_cast<floatx4*>(raw + k0 + 16 + 4 * g4) = St[1];
    }
    mask_tail(p, k0, hi, g4);
    const float f = softmax_step(p, m, l);
    rescale(f, g4, o);
    bf16x8 pa[3];
    split3_8(p, pa);
#pragma unroll
    for (int t = 0; t < T; ++t) {
        const bf16x8 v = v_operand<bf16x8>(Vc, vo ^ ((t0 + t) << 5));
#pragma unroll
        for (int q = 2; q >= 0; --q) o[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pa[q], v, o[t], 0, 0, 0);
    }
}

// A wave's unnormalised output (dims 16 (t0 + t) + r16 of rows first + 4 g4 + v) and, from the
// wave that is asked, the rows' (max, sum).
template <int T>
__device__ __forceinline__ void store_part(const Item& it, int first, int r16, int g4, int t0, const floatx4 (&o)[T], float m,
                                           float l, bool with_ml) {
#pragma unroll
    for (int v = 0; v < 4; ++v) {
        const int row = first + 4 * g4 + v;
        if (row < it.rows) {
            float* dst = it.part + static_cast<int64_t>(row) * kHD + 16 * t0 + r16;
#pragma unroll
            for (int t = 0; t < T; ++t) dst[16 * t] = o[t][v];
        }
    }
    if (with_ml && g4 == 0 && first + r16 < it.rows) it.ml[first + r16] = make_float2(m, l);
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
    if (!item_of(a, it)) return;
    const int lane = threadIdx.x & 63, r16 = lane & 15, g4 = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    auto copy = [&](int k0, uint4* K, uint4* V) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {  // two rows of K and of V per instruction
            const int c = 64 * (4 * wave + j), row = 2 * (4 * wave + j) + (lane >> 5), pos = lane & 31;
            const int64_t at = static_cast<int64_t>(min(k0 + row, it.hi - 1)) * 32;
            const uint4* ks = static_cast<const uint4*>(it.K) + at + (pos ^ (row & 15));
            const uint4* vs = static_cast<const uint4*>(it.V) + at + (pos ^ ((2 * row) & 15));
            __builtin_amdgcn_global_load_lds(
                reinterpret_cast<const __attribute__((address_space(1))) void*>(reinterpret_cast<uintptr_t>(ks)),
                (__attribute__((address_space(3))) void*)(K + c), 16, 0, 0);
            __builtin_amdgcn_global_load_lds(
                reinterpret_cast<const __attribute__((address_space(1))) void*>(reinterpret_cast<uintptr_t>(vs)),
                (__attribute__((address_space(3))) void*)(V + c), 16, 0, 0);
        }
    };
    copy(it.lo, K0, V0);
    const int first = it.narrow ? it.row0 : it.row0 + 16 * wave;
    bf16x8 qp[3][8];
    load_query(it, first, r16, g4, qp);
    float m = -INFINITY, l = 0.0f;
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

typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));

// 2^e
__device__ __forceinline__ float pow2(int e) { return __uint_as_float(static_cast<uint32_t>(127 + e) << 23); }

// eight floats times s as two fp16 parts h = fp16(x), l = fp16(x - h): |x - h - l| <= 2^-23 |x|
__device__ __forceinline__ void split2_8(const float (&x)[8], float s, halfx8 (&part)[2]) {
    uint32_t h[4], l[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) split2h_pair(x[2 * e] * s, x[2 * e + 1] * s, h[e], l[e]);
    part[0] = __builtin_bit_cast(halfx8, make_uint4(h[0], h[1], h[2], h[3]));
    part[1] = __builtin_bit_cast(halfx8, make_uint4(l[0], l[1], l[2], l[3]));
}
__device__ __forceinline__ float max8(const float (&x)[8]) {
    float m = fabsf(x[0]);
#pragma unroll
    for (int e = 1; e < 8; ++e) m = fmaxf(m, fabsf(x[e]));
    return m;
}

// fp32 caches, wide: 64 query rows, 16 a wave, 32-key tiles, on v_mfma_f32_16x16x32_f16. Every
// operand row (a query, a key, a value row, a query's weights over the tile) is scaled by a power
// of two that brings its largest entry into [2^14, 2^15) and split into two fp16 parts; the three
// part products of lowest order are summed (the fourth is below 2^-22 of the product) and the
// scales undone exactly: a key's in the scores, a value row's in the weights before their own
// scaling, and that one as the tile's products, summed from zero, are added to the output. So
// nothing is lost relative to the largest weight times value row of the tile, whatever rows lie
// beside it.
// A tile's rows come through registers and are split once for the four waves: K of the next tile
// while V is multiplied, V while K is.
__device__ __forceinline__ void f32_wide(const Item& it, uint4 (*Kc)[1024], uint4 (*Vc)[1024], float* kscale, float* vscale) {
    const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, g4 = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int first = it.row0 + 16 * wave;
    const bool live = first < it.rows;  // uniform per wave
    float4 st[8];
    auto load = [&](const void* cache, int k0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t at = static_cast<int64_t>(min(k0 + (tid >> 5) + 8 * i, it.hi - 1)) * kHD + 8 * (tid & 31);
            const float4* s = reinterpret_cast<const float4*>(static_cast<const float*>(cache) + at);
            st[2 * i] = s[0], st[2 * i + 1] = s[1];
        }
    };
    auto store = [&](uint4 (*dst)[1024], float* scale, int mul) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = (tid >> 5) + 8 * i, c = tid & 31;
            const float x[8] = {st[2 * i].x, st[2 * i].y, st[2 * i].z, st[2 * i].w,
                                st[2 * i + 1].x, st[2 * i + 1].y, st[2 * i + 1].z, st[2 * i + 1].w};
            float mx = max8(x);  // over the row: the 32 lanes of half a wave
            mx = fmaxf(mx, dpp_f<0xB1>(mx));
            mx = fmaxf(mx, dpp_f<0x4E>(mx));
            mx = fmaxf(mx, dpp_f<0x141>(mx));
            mx = fmaxf(mx, dpp_f<0x140>(mx));
            mx = fmaxf(mx, swz16_f(mx));
            const int e = split_row_exp(mx);
            halfx8 p[2];
            split2_8(x, pow2(e), p);
#pragma unroll
            for (int q = 0; q < 2; ++q) dst[q][32 * row + (c ^ ((mul * row) & 15))] = __builtin_bit_cast(uint4, p[q]);
            if (c == 0) scale[row] = pow2(-e);
        }
    };
    load(it.K, it.lo);
    halfx8 qp[2][8];
    float qscale;
    {
        const float* src = it.Q + static_cast<int64_t>(min(first + r16, it.rows - 1)) * kHD + 8 * g4;
        float4 u[16];
        float mx = 0.0f;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            u[2 * c] = *reinterpret_cast<const float4*>(src + 32 * c);
            u[2 * c + 1] = *reinterpret_cast<const float4*>(src + 32 * c + 4);
        }
#pragma unroll
        for (auto& x : u) mx = fmaxf(mx, fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))));
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const int e = split_row_exp(mx);
        qscale = pow2(-e);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            const float x[8] = {u[2 * c].x, u[2 * c].y, u[2 * c].z, u[2 * c].w,
                                u[2 * c + 1].x, u[2 * c + 1].y, u[2 * c + 1].z, u[2 * c + 1].w};
            halfx8 p[2];
            split2_8(x, pow2(e), p);
            qp[0][c] = p[0], qp[1][c] = p[1];
        }
    }
    store(Kc, kscale, 1);
    load(it.V, it.lo);
    float m = -INFINITY, l = 0.0f;
    floatx4 o[16];
#pragma unroll
    for (auto& x : o) x = floatx4{0.f, 0.f, 0.f, 0.f};
    store(Vc, vscale, 2);
    lds_barrier();
    for (int k0 = it.lo; k0 < it.hi; k0 += kKT) {
        const bool more = k0 + kKT < it.hi;  // uniform
        if (more) load(it.K, k0 + kKT);
        int ko = k_off(r16, g4), vo = v_off(r16, g4);
        asm volatile("" : "+v"(ko), "+v"(vo));  // formed per tile: kept, the 24 addresses would spill
        float p[8], f = 1.0f;
        if (live) {
            floatx4 St[2];
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                floatx4 sa[2], sb[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) sa[e] = sb[e] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    halfx8 k[2];
#pragma unroll
                    for (int q = 0; q < 2; ++q)
                        k[q] = *reinterpret_cast<const halfx8*>(reinterpret_cast<const char*>(Kc[q]) + hf * 16 * 512 + (ko ^ (c << 6)));
                    sb[c & 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[1], qp[0][c], sb[c & 1], 0, 0, 0);
                    sb[c & 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[0], qp[1][c], sb[c & 1], 0, 0, 0);
                    sa[c & 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[0], qp[0][c], sa[c & 1], 0, 0, 0);
                }
                St[hf] = (sb[0] + sb[1]) + (sa[0] + sa[1]);
            }
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                const floatx4 ks = *reinterpret_cast<const floatx4*>(kscale + 16 * hf + 4 * g4);
#pragma unroll
                for (int v = 0; v < 4; ++v) p[4 * hf + v] = (St[hf][v] * qscale) * ks[v];
            }
            mask_tail(p, k0, it.hi, g4);
            f = softmax_step(p, m, l);
        }
        lds_barrier();  // every wave is done with K, every share of V is in
        if (more) {
            store(Kc, kscale, 1);
            load(it.V, k0 + kKT);
        }
        if (live) {
            rescale(f, g4, o);
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                const floatx4 vs = *reinterpret_cast<const floatx4*>(vscale + 16 * hf + 4 * g4);
#pragma unroll
                for (int v = 0; v < 4; ++v) p[4 * hf + v] *= vs[v];
            }
            float mx = max8(p);
            mx = fmaxf(mx, __shfl_xor(mx, 16));
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const int e = split_row_exp(mx);
            halfx8 pp[2];
            split2_8(p, pow2(e), pp);
            const float undo = pow2(-e);
            float er[4];
#pragma unroll
            for (int v = 0; v < 4; ++v) er[v] = __shfl(undo, 4 * g4 + v);
#pragma unroll
            for (int t = 0; t < 16; ++t) {
                const halfx8 v0 = v_operand<halfx8>(Vc[0], vo ^ (t << 5)), v1 = v_operand<halfx8>(Vc[1], vo ^ (t << 5));
                floatx4 x = floatx4{0.f, 0.f, 0.f, 0.f};
                x = __builtin_amdgcn_mfma_f32_16x16x32_f16(pp[1], v0, x, 0, 0, 0);
                x = __builtin_amdgcn_mfma_f32_16x16x32_f16(pp[0], v1, x, 0, 0, 0);
                x = __builtin_amdgcn_mfma_f32_16x16x32_f16(pp[0], v0, x, 0, 0, 0);
#pragma unroll
                for (int v = 0; v < 4; ++v) o[t][v] += x[v] * er[v];
            }
        }
        lds_barrier();  // every wave is done with V, every share of the next K is in
        if (more) store(Vc, vscale, 2);
    }
    store_part(it, first, r16, g4, 0, o, m, l, true);
}

// fp32 caches, narrow: 16 query rows on v_mfma_f32_16x16x4_f32 with K and V straight from memory
// as its operands, no LDS and no barrier in the loop; the four waves take 16 keys in turn and are
// merged at the end.
//   S^T = K Q^T: lane (r16, g4) loads dims 16 u + 4 g4 .. + 3 of key r16; the k slot g4 of product
//         (u, e) is dim 16 u + 4 g4 + e on both sides
//   O += P V: product (v, t, e) takes the weights of keys 4 g4 + v as they lie and dims
//         64 t + 4 r16 + e of those keys; lane (r16, g4) ends with dims 64 t + 4 r16 + e of rows 4 g4 + .
__device__ __forceinline__ void f32_narrow(const Item& it, float* buf, float (*ms)[16], float (*ls)[16]) {
    const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, g4 = lane >> 4, wave = tid >> 6;
    float4 q[16];
    {
        const float* src = it.Q + static_cast<int64_t>(min(it.row0 + r16, it.rows - 1)) * kHD + 4 * g4;
#pragma unroll
        for (int u = 0; u < 16; ++u) q[u] = *reinterpret_cast<const float4*>(src + 16 * u);
    }
    const float *K = static_cast<const float*>(it.K), *V = static_cast<const float*>(it.V);
    float* raw = it.raw && r16 < it.rows ? it.raw + r16 * it.raw_stride : nullptr;
    float m = -INFINITY, l = 0.0f;
    floatx4 o[16];
#pragma unroll
    for (auto& x : o) x = floatx4{0.f, 0.f, 0.f, 0.f};
    for (int k0 = it.lo + 16 * wave; k0 < it.hi; k0 += 64) {
        floatx4 s[4];
#pragma unroll
        for (auto& x : s) x = floatx4{0.f, 0.f, 0.f, 0.f};
        float4 k[16];
        const float* kr = K + static_cast<int64_t>(min(k0 + r16, it.hi - 1)) * kHD + 4 * g4;
#pragma unroll
        for (int u = 0; u < 16; ++u) k[u] = *reinterpret_cast<const float4*>(kr + 16 * u);
#pragma unroll
        for (int u = 0; u < 16; ++u) {
            s[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[u].x, q[u].x, s[0], 0, 0, 0);
            s[1] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[u].y, q[u].y, s[1], 0, 0, 0);
            s[2] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[u].z, q[u].z, s[2], 0, 0, 0);
            s[3] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[u].w, q[u].w, s[3], 0, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);  // V takes K's registers
        float4 vv[4][4];
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            const float* vr = V + static_cast<int64_t>(min(k0 + 4 * g4 + v, it.hi - 1)) * kHD + 4 * r16;
#pragma unroll
            for (int t = 0; t < 4; ++t) vv[v][t] = *reinterpret_cast<const float4*>(vr + 64 * t);
        }
        const floatx4 St = (s[0] + s[1]) + (s[2] + s[3]);
        if (raw) *reinterpret_cast<floatx4*>(raw + k0 + 4 * g4) = St;
        float p[4];
#pragma unroll
        for (int v = 0; v < 4; ++v) p[v] = k0 + 4 * g4 + v < it.hi ? St[v] : -INFINITY;
        const float f = softmax_step(p, m, l);
        rescale(f, g4, o);
#pragma unroll
        for (int v = 0; v < 4; ++v)
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                o[4 * t] = __builtin_amdgcn_mfma_f32_16x16x4f32(p[v], vv[v][t].x, o[4 * t], 0, 0, 0);
                o[4 * t + 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(p[v], vv[v][t].y, o[4 * t + 1], 0, 0, 0);
                o[4 * t + 2] = __builtin_amdgcn_mfma_f32_16x16x4f32(p[v], vv[v][t].z, o[4 * t + 2], 0, 0, 0);
                o[4 * t + 3] = __builtin_amdgcn_mfma_f32_16x16x4f32(p[v], vv[v][t].w, o[4 * t + 3], 0, 0, 0);
            }
    }
    // merge of the waves; one without keys has maximum -inf and weight 0
    if (g4 == 0) {
        ms[wave][r16] = m;
        ls[wave][r16] = l;
    }
    lds_barrier();
    const float top = fmaxf(fmaxf(ms[0][r16], ms[1][r16]), fmaxf(ms[2][r16], ms[3][r16]));
    const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - top) * kLog2e);
    rescale(f, g4, o);
    const int n = min(16, it.rows - it.row0);
    if (wave == 0 && g4 == 0 && r16 < n) {
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w)
            if (ms[w][r16] != -INFINITY) sum += ls[w][r16] * __builtin_amdgcn_exp2f((ms[w][r16] - top) * kLog2e);
        it.ml[it.row0 + r16] = make_float2(top, sum);
    }
#pragma unroll
    for (int v = 0; v < 4; ++v)
        if (4 * g4 + v < n) {
#pragma unroll
            for (int t = 0; t < 4; ++t)
                *reinterpret_cast<float4*>(buf + (wave * 16 + 4 * g4 + v) * kHD + 64 * t + 4 * r16) =
                    make_float4(o[4 * t][v], o[4 * t + 1][v], o[4 * t + 2][v], o[4 * t + 3][v]);
        }
    lds_barrier();
    for (int r = wave; r < n; r += 4) {
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float4 x = *reinterpret_cast<const float4*>(buf + (w * 16 + r) * kHD + 4 * lane);
            y.x += x.x, y.y += x.y, y.z += x.z, y.w += x.w;
        }
        *reinterpret_cast<float4*>(it.part + static_cast<int64_t>(it.row0 + r) * kHD + 4 * lane) = y;
    }
}

// fp32 caches: four waves, two workgroups per compute unit.
__global__ __launch_bounds__(256, 2) void attn_batch_f32_kernel(AttnBatchArgs a) {
    __shared__ __align__(16) uint4 lds[2][2][1024];
    __shared__ __align__(16) float small[2][4][16];
    Item it;
    if (!item_of(a, it)) return;
    if (it.narrow) f32_narrow(it, reinterpret_cast<float*>(lds), small[0], small[1]);
    else f32_wide(it, lds[0], lds[1], &small[0][0][0], &small[1][0][0]);
}

constexpr int kCombWaves = 8;

// The (max, sum) of piece i of row g of (b, kh): the prefix's pieces, then the own cache's.
__device__ __forceinline__ int64_t piece_row(const AttnBatchArgs& a, int b, int kh, int g, int i) {
    return i < a.plan.pieces
               ? (static_cast<int64_t>(kh) * a.plan.pieces + i) * a.B * a.GRP + b * a.GRP + g
               : ((static_cast<int64_t>(b) * a.NKV + kh) * a.plan.own + i - a.plan.pieces) * a.GRP + g;
}
__device__ __forceinline__ float2 piece_ml(const AttnBatchArgs& a, int b, int kh, int g, int i) {
    return (i < a.plan.pieces ? a.ml_p : a.ml_o)[piece_row(a, b, kh, g, i)];
}
// (max, sum) over n pieces, by the lanes of a wave
__device__ __forceinline__ float2 merge_ml(const AttnBatchArgs& a, int b, int kh, int g, int n, int lane) {
    float m = -INFINITY, l = 0.0f;
    for (int i = lane; i < n; i += 64) m = fmaxf(m, piece_ml(a, b, kh, g, i).x);
    m = wave_max(m);
    for (int i = lane; i < n; i += 64) {
        const float2 x = piece_ml(a, b, kh, g, i);
        l += x.y * __builtin_amdgcn_exp2f((x.x - m) * kLog2e);
    }
    return make_float2(m, wave_sum(l));
}

// Workgroups [0, B NQ): one output row each. The pieces' factors e^(their maximum - the row's) / sum
// first, into LDS, so that the partial outputs stream with nothing between their loads: a wave
// takes every eighth piece, a lane four dims. Then the gate.
// The others (with own_score): 512 own rows of a (sequence, kv head) each: their weights, summed
// over the heads of the group in order, into the scores.
__global__ __launch_bounds__(kCombWaves * 64) void attn_batch_combine_kernel(AttnBatchArgs a) {
    extern __shared__ __align__(16) float fac[];  // a factor per piece
    __shared__ __align__(16) float part[kCombWaves][kHD];
    __shared__ float ms[16], ls[16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
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
            const float2 x = merge_ml(a, b, kh, g, n, lane);
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
    const float2 all = merge_ml(a, b, kh, g, n, lane);  // every wave the same
    for (int i = tid; i < n; i += kCombWaves * 64)
        fac[i] = __builtin_amdgcn_exp2f((piece_ml(a, b, kh, g, i).x - all.x) * kLog2e);
    __syncthreads();
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int i = wave; i < n; i += kCombWaves) {
        const float4 x = *reinterpret_cast<const float4*>((i < a.plan.pieces ? a.part_p : a.part_o) + piece_row(a, b, kh, g, i) * kHD + 4 * lane);
        const float f = fac[i];
        y.x += x.x * f, y.y += x.y * f, y.z += x.z * f, y.w += x.w * f;
    }
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
    int64_t q, pp, mp, po, mo, raw, total;  // float offsets, multiples of 4
};
Carve carve_of(const AttnBatchArgs& a) {
    const auto up4 = [](int64_t x) { return (x + 3) / 4 * 4; };
    const int64_t rows = static_cast<int64_t>(a.B) * a.NQ;
    const AttnBatchPlan p = attn_batch_plan(a.B, a.GRP, a.NKV, a.P, a.cap, a.kv_bf16, device_cu_count());
    Carve c{};
    c.q = 0;
    c.pp = c.q + rows * kHD;
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
    a.part_p = ws + c.pp;
    a.ml_p = reinterpret_cast<float2*>(ws + c.mp);
    a.part_o = ws + c.po;
    a.ml_o = reinterpret_cast<float2*>(ws + c.mo);
    a.raw = ws + c.raw;
}

hipError_t launch_attn_batch(const AttnBatchArgs& a, hipStream_t s) {
    klaunch(attn_batch_prep_kernel, dim3((a.NQ + a.NKV + 3) / 4, a.B), 256, 0, s, a);
    const uint32_t prefix = (a.plan.pieces * a.NKV + 7) / 8 * 8 * a.plan.nblk, own = a.B * a.NKV * a.plan.own;
    if (a.kv_bf16) klaunch(attn_batch_bf16_kernel, dim3(prefix + own), 256, 0, s, a);
    else klaunch(attn_batch_f32_kernel, dim3(prefix + own), 256, 0, s, a);
    const uint32_t scores = a.own_score ? static_cast<uint32_t>((a.cap + 511) / 512) * a.B * a.NKV : 0;
    klaunch(attn_batch_combine_kernel, dim3(a.B * a.NQ + scores), kCombWaves * 64, (a.plan.pieces + a.plan.own) * 4, s, a);
    return hipGetLastError();
}

}  // namespace q35k
