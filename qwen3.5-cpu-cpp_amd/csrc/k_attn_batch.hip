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

// grid (B, NQ + NKV), one thread per dim: rmsnorm (1 + w) + RoPE of a query row -> Qa, or of
// the new key row -> own cache, with its value row.
__global__ __launch_bounds__(256) void attn_batch_prep_kernel(AttnBatchArgs a) {
    const int b = blockIdx.x, r = blockIdx.y, d = threadIdx.x;
    __shared__ float buf[kHD];
    __shared__ double red[4];
    const int slot = new_slot(a, b);
    const bool is_q = r < a.NQ;
    const int kh = is_q ? r / a.GRP : r - a.NQ;
    float* q = a.Qa + ((static_cast<int64_t>(kh) * a.B + b) * a.GRP + (r - kh * a.GRP)) * kHD + d;
    if (slot < 0) {
        if (is_q) *q = 0.0f;
        return;
    }
    const float* src = is_q ? a.qg + (static_cast<int64_t>(b) * a.NQ + r) * 2 * kHD
                            : a.k_new + (static_cast<int64_t>(b) * a.NKV + kh) * kHD;
    const float x = src[d];
    const double ss = block_sum(static_cast<double>(x) * x, red);
    const float inv = 1.0f / sqrtf(static_cast<float>(ss / kHD) + a.eps);
    float y = x * inv * (1.0f + (is_q ? a.q_norm : a.k_norm)[d]);
    buf[d] = y;
    __syncthreads();
    if (d < a.ROT) {
        const int half = a.ROT / 2, i = d < half ? d : d - half;
        const double ang = static_cast<double>(a.pos[b]) * pow(a.theta, -static_cast<double>(2 * i) / a.ROT);
        const float c = static_cast<float>(cos(ang)), s = static_cast<float>(sin(ang));
        y = d < half ? buf[i] * c - buf[i + half] * s : buf[i + half] * c + buf[i] * s;
    }
    if (is_q) {
        *q = y * 0.0625f;  // 1 / sqrt(HD), exact
        return;
    }
    const int64_t row = (static_cast<int64_t>(b) * a.NKV + kh) * a.cap + slot;
    const float v = a.v_new[(static_cast<int64_t>(b) * a.NKV + kh) * kHD + d];
    if (a.kv_bf16) {
        static_cast<uint16_t*>(a.k_own)[row * kHD + d] = to_bf16(y);
        static_cast<uint16_t*>(a.v_own)[row * kHD + d] = to_bf16(v);
    } else {
        static_cast<float*>(a.k_own)[row * kHD + d] = y;
        static_cast<float*>(a.v_own)[row * kHD + d] = v;
    }
    if (a.own_pos && d == 0) a.own_pos[row] = a.pos[b];
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

// dims 16 t + r16 of keys 4 g4 .. + 3 of the tile's first half, then of its second
__device__ __forceinline__ bf16x8 v_operand(const uint4* V, int off) {
    typedef __attribute__((address_space(3))) i16x4 lds4;
    const char* p = reinterpret_cast<const char*>(V) + off;
    const i16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)p);
    const i16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(p + 16 * 512));
    const i16x8 x = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(bf16x8, x);
}

// One 32-key tile for the 16 query rows of a wave, on v_mfma_f32_16x16x32_bf16. Every fp32
// operand is the exact sum of three bf16 parts; with a bf16 cache K and V are one part each and
// every product is exact, else the six part products of lowest order are summed (the others
// are below 2^-23 of the product).
//   S^T = K Q^T by 16-key halves: lane (r16, g4) ends with keys 4 g4 + v of both for query r16
//   O += P V: those eight weights are the A operand as they lie, its k slots 8 g4 .. + 7 being
//         keys 4 g4 .. + 3 of the first half and of the second, which transposed LDS reads give V too;
//         lane (r16, g4) ends with dims 16 t + r16 of queries 4 g4 + v
// T tiles of 16 dims from t0 on (a narrow workgroup's waves share the dims and each form all scores).
template <int NP, int T>
__device__ __forceinline__ void tile_products(const uint4 (&Kc)[NP][1024], const uint4 (&Vc)[NP][1024], const bf16x8 (&qp)[3][8],
                                              int k0, int hi, int r16, int g4, int t0, float* raw, float& m, float& l,
                                              floatx4 (&o)[T]) {
    constexpr int lo_part[6] = {2, 1, 0, 1, 0, 0}, hi_part[6] = {0, 1, 2, 0, 1, 0};  // smallest products first
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
            bf16x8 kop[NP];
#pragma unroll
            for (int p = 0; p < NP; ++p)
                kop[p] = *reinterpret_cast<const bf16x8*>(reinterpret_cast<const char*>(&Kc[p][0]) + hf * 16 * 512 + (ko ^ (c << 6)));
            floatx4& b = sb[c & 1];
            if constexpr (NP == 1) {
                b = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kop[0], qp[2][c], b, 0, 0, 0);
                b = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kop[0], qp[1][c], b, 0, 0, 0);
                sa[c & 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kop[0], qp[0][c], sa[c & 1], 0, 0, 0);
            } else {
#pragma unroll
                for (int i = 0; i < 6; ++i) {
                    floatx4& s = i < 5 ? b : sa[c & 1];
                    s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kop[lo_part[i] % NP], qp[hi_part[i]][c], s, 0, 0, 0);
                }
            }
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
    if (k0 + kKT > hi) {  // uniform
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (k0 + 16 * (i >> 2) + 4 * g4 + (i & 3) >= hi) p[i] = -INFINITY;
    }
    const float f = softmax_step(p, m, l);
    rescale(f, g4, o);
    bf16x8 pa[3];
    split3_8(p, pa);
#pragma unroll
    for (int t = 0; t < T; ++t) {
        bf16x8 vb[NP];
#pragma unroll
        for (int q = 0; q < NP; ++q) vb[q] = v_operand(&Vc[q][0], vo ^ ((t0 + t) << 5));
        if constexpr (NP == 1) {
#pragma unroll
            for (int q = 2; q >= 0; --q) o[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pa[q], vb[0], o[t], 0, 0, 0);
        } else {
#pragma unroll
            for (int i = 0; i < 6; ++i)
                o[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pa[lo_part[i]], vb[hi_part[i] % NP], o[t], 0, 0, 0);
        }
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
    __shared__ __align__(16) uint4 K0[1][1024], V0[1][1024], K1[1][1024], V1[1][1024];
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
    copy(it.lo, &K0[0][0], &V0[0][0]);
    const int first = it.narrow ? it.row0 : it.row0 + 16 * wave;
    bf16x8 qp[3][8];
    load_query(it, first, r16, g4, qp);
    float m = -INFINITY, l = 0.0f;
    auto walk = [&](auto& o, int t0, float* raw, bool live) {
#pragma unroll
        for (auto& x : o) x = floatx4{0.f, 0.f, 0.f, 0.f};
        auto tile = [&](int k0, const uint4 (&Kc)[1][1024], const uint4 (&Vc)[1][1024], uint4* Kn, uint4* Vn) {
            __builtin_amdgcn_s_waitcnt(kWaitVm);  // this wave's share of the tile
            lds_barrier();                        // every share; every wave is done with the other buffer
            if (k0 + kKT < it.hi) copy(k0 + kKT, Kn, Vn);  // uniform
            if (live) tile_products<1>(Kc, Vc, qp, k0, it.hi, r16, g4, t0, raw, m, l, o);
        };
        for (int k0 = it.lo; k0 < it.hi; k0 += 2 * kKT) {
            tile(k0, K0, V0, &K1[0][0], &V1[0][0]);
            if (k0 + kKT < it.hi) tile(k0 + kKT, K1, V1, &K0[0][0], &V0[0][0]);
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

// fp32 caches, wide: 128 query rows, 16 a wave. A tile's rows are loaded into registers under
// the products of the one before, split into three bf16 parts and stored to LDS once for all
// eight waves.
__device__ __forceinline__ void f32_wide(const Item& it, uint4 (&Kc)[3][1024], uint4 (&Vc)[3][1024]) {
    const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, g4 = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int first = it.row0 + 16 * wave;
    float4 kst[4], vst[4];
    auto load = [&](int k0) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int row = (tid >> 5) + 16 * i;
            const int64_t at = static_cast<int64_t>(min(k0 + row, it.hi - 1)) * kHD + 8 * (tid & 31);
            const float4 *ks = reinterpret_cast<const float4*>(static_cast<const float*>(it.K) + at),
                         *vs = reinterpret_cast<const float4*>(static_cast<const float*>(it.V) + at);
            kst[2 * i] = ks[0], kst[2 * i + 1] = ks[1];
            vst[2 * i] = vs[0], vst[2 * i + 1] = vs[1];
        }
    };
    auto store = [&]() {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int row = (tid >> 5) + 16 * i, c = tid & 31;
            bf16x8 p[3];
            const float k8[8] = {kst[2 * i].x, kst[2 * i].y, kst[2 * i].z, kst[2 * i].w,
                                 kst[2 * i + 1].x, kst[2 * i + 1].y, kst[2 * i + 1].z, kst[2 * i + 1].w};
            split3_8(k8, p);
#pragma unroll
            for (int q = 0; q < 3; ++q) Kc[q][32 * row + (c ^ (row & 15))] = __builtin_bit_cast(uint4, p[q]);
            const float v8[8] = {vst[2 * i].x, vst[2 * i].y, vst[2 * i].z, vst[2 * i].w,
                                 vst[2 * i + 1].x, vst[2 * i + 1].y, vst[2 * i + 1].z, vst[2 * i + 1].w};
            split3_8(v8, p);
#pragma unroll
            for (int q = 0; q < 3; ++q) Vc[q][32 * row + (c ^ ((2 * row) & 15))] = __builtin_bit_cast(uint4, p[q]);
        }
    };
    load(it.lo);
    bf16x8 qp[3][8];
    load_query(it, first, r16, g4, qp);
    float m = -INFINITY, l = 0.0f;
    floatx4 o[16];
#pragma unroll
    for (auto& x : o) x = floatx4{0.f, 0.f, 0.f, 0.f};
    store();
    lds_barrier();
    for (int k0 = it.lo; k0 < it.hi; k0 += kKT) {
        load(min(k0 + kKT, it.hi - 1));
        if (first < it.rows) tile_products<3>(Kc, Vc, qp, k0, it.hi, r16, g4, 0, nullptr, m, l, o);  // uniform per wave
        lds_barrier();  // every wave is done with this tile
        if (k0 + kKT < it.hi) {
            store();
            lds_barrier();
        }
    }
    store_part(it, first, r16, g4, 0, o, m, l, true);
}

// fp32 caches, narrow: 16 query rows on v_mfma_f32_16x16x4_f32 with K and V straight from memory
// as its operands, no LDS and no barrier in the loop; the eight waves take 16 keys in turn and are
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
    for (int k0 = it.lo + 16 * wave; k0 < it.hi; k0 += 128) {
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
    // merge of the waves, eight rows at a time; a wave without keys has maximum -inf and weight 0
    if (g4 == 0) {
        ms[wave][r16] = m;
        ls[wave][r16] = l;
    }
    lds_barrier();
    float top = ms[0][r16];
#pragma unroll
    for (int w = 1; w < 8; ++w) top = fmaxf(top, ms[w][r16]);
    const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - top) * kLog2e);
    rescale(f, g4, o);
    const int n = min(16, it.rows - it.row0);
    if (wave == 0 && g4 == 0 && r16 < n) {
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < 8; ++w)
            if (ms[w][r16] != -INFINITY) sum += ls[w][r16] * __builtin_amdgcn_exp2f((ms[w][r16] - top) * kLog2e);
        it.ml[it.row0 + r16] = make_float2(top, sum);
    }
    for (int r0 = 0; r0 < n; r0 += 8) {
        if (r0) lds_barrier();
        if (g4 >> 1 == r0 >> 3) {
#pragma unroll
            for (int v = 0; v < 4; ++v)
#pragma unroll
                for (int t = 0; t < 4; ++t)
                    *reinterpret_cast<float4*>(buf + (wave * 8 + 4 * (g4 & 1) + v) * kHD + 64 * t + 4 * r16) =
                        make_float4(o[4 * t][v], o[4 * t + 1][v], o[4 * t + 2][v], o[4 * t + 3][v]);
        }
        lds_barrier();
        const int r = tid >> 6;
        if (r0 + r < n) {
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < 8; ++w) {
                const float4 x = *reinterpret_cast<const float4*>(buf + (w * 8 + r) * kHD + 4 * lane);
                y.x += x.x, y.y += x.y, y.z += x.z, y.w += x.w;
            }
            *reinterpret_cast<float4*>(it.part + static_cast<int64_t>(it.row0 + r0 + r) * kHD + 4 * lane) = y;
        }
    }
}

__global__ __launch_bounds__(512, 1) void attn_batch_f32_kernel(AttnBatchArgs a) {
    __shared__ __align__(16) uint4 lds[2][3][1024];
    Item it;
    if (!item_of(a, it)) return;
    if (it.narrow) {
        float(*ms)[16] = reinterpret_cast<float(*)[16]>(&lds[1][2][0]);  // behind 64 KB of rows
        f32_narrow(it, reinterpret_cast<float*>(lds), ms, ms + 8);
    } else {
        f32_wide(it, lds[0], lds[1]);
    }
}

// The (max, sum) of row g of (b, kh) over all its pieces; f(i, m, l) for each.
template <class F>
__device__ __forceinline__ void pieces_of(const AttnBatchArgs& a, int b, int kh, int g, int n_own, F&& f) {
    for (int i = 0; i < a.plan.pieces; ++i) {
        const int64_t row = (static_cast<int64_t>(kh) * a.plan.pieces + i) * a.B * a.GRP + b * a.GRP + g;
        f(a.part_p + row * kHD, a.ml_p[row]);
    }
    for (int i = 0; i < n_own; ++i) {
        const int64_t row = ((static_cast<int64_t>(b) * a.NKV + kh) * a.plan.own + i) * a.GRP + g;
        f(a.part_o + row * kHD, a.ml_o[row]);
    }
}

// grid (NQ, B), one thread per dim: merges the pieces, divides, gates.
__global__ __launch_bounds__(256) void attn_batch_combine_kernel(AttnBatchArgs a) {
    const int h = blockIdx.x, b = blockIdx.y, d = threadIdx.x;
    const int n = a.own_len[b];
    if (n < 0) return;
    float* out = a.out + (static_cast<int64_t>(b) * a.NQ + h) * kHD + d;
    if (n >= a.cap) {
        *out = NAN;
        return;
    }
    const int kh = h / a.GRP, g = h - kh * a.GRP, n_own = n / a.plan.okeys + 1;
    float m = -INFINITY, l = 0.0f, o = 0.0f;
    pieces_of(a, b, kh, g, n_own, [&](const float*, float2 ml) { m = fmaxf(m, ml.x); });
    pieces_of(a, b, kh, g, n_own, [&](const float* po, float2 ml) {
        const float f = expf(ml.x - m);
        l += ml.y * f;
        o += po[d] * f;
    });
    const float gate = a.qg[(static_cast<int64_t>(b) * a.NQ + h) * 2 * kHD + kHD + d];
    *out = (o / l) * sigmoid_f(gate);
}

// grid (cap / 256, NKV, B): the weights of the own rows, summed over the heads of the group
// in their order, into the scores.
__global__ __launch_bounds__(256) void attn_batch_score_kernel(AttnBatchArgs a) {
    const int kh = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
    const int slot = new_slot(a, b);
    const int64_t t = static_cast<int64_t>(blockIdx.x) * 256 + tid;
    if (slot < 0 || blockIdx.x * 256LL > slot) return;
    __shared__ float ms[16], ls[16];
    if (tid < a.GRP) {
        float m = -INFINITY, l = 0.0f;
        const int n_own = slot / a.plan.okeys + 1;
        pieces_of(a, b, kh, tid, n_own, [&](const float*, float2 ml) { m = fmaxf(m, ml.x); });
        pieces_of(a, b, kh, tid, n_own, [&](const float*, float2 ml) { l += ml.y * expf(ml.x - m); });
        ms[tid] = m;
        ls[tid] = l;
    }
    __syncthreads();
    if (t > slot) return;
    const int64_t bk = static_cast<int64_t>(b) * a.NKV + kh;
    float w = 0.0f;
    for (int g = 0; g < a.GRP; ++g) w += expf(a.raw[(bk * a.GRP + g) * raw_stride(a.cap) + t] - ms[g]) / ls[g];
    float* sc = a.own_score + bk * a.cap + t;
    *sc = t == slot ? w : *sc + w;
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
    klaunch(attn_batch_prep_kernel, dim3(a.B, a.NQ + a.NKV), 256, 0, s, a);
    const uint32_t prefix = (a.plan.pieces * a.NKV + 7) / 8 * 8 * a.plan.nblk, own = a.B * a.NKV * a.plan.own;
    if (a.kv_bf16) klaunch(attn_batch_bf16_kernel, dim3(prefix + own), 256, 0, s, a);
    else klaunch(attn_batch_f32_kernel, dim3(prefix + own), 512, 0, s, a);
    klaunch(attn_batch_combine_kernel, dim3(a.NQ, a.B), 256, 0, s, a);
    if (a.own_score)
        klaunch(attn_batch_score_kernel, dim3(static_cast<uint32_t>((a.cap + 255) / 256), a.NKV, a.B), 256, 0, s, a);
    return hipGetLastError();
}

}  // namespace q35k
