// Products with 4-bit weights and group scales: Y[m][n] = R[m][n] + sum_g s[n][g] sum_{k in g}
// X[m][k] (c[n][k] - z[n][g]), and the kernels that make such weights. The layout of packed weights
// is in launch_q4.hpp.
#include <cstdint>
#include <type_traits>

#include "dev_q4.hpp"
#include "launch_q4.hpp"

namespace q35k {
namespace {

constexpr int kThreads = 512, kWaves = 8;

// ---- rows of X as pairs of fp16 values
// An entry of X times the power of two that brings its group's largest to [2^14, 2^15) is hi + lo, two fp16 values, to 2^-22
// of itself (or 2^-39 of the largest); a code less its zero is an fp16 value; so products on the fp16 matrix cores are
// exact, and their sums, of one group, are in fp32. An entry keeps its bits beside one that is far larger: where one a group
// of 64 is 10^4 times the others and its weights are 0, outputs of 2048 k are off by 4e-8 of their norm. (As 24-bit multiples
// of a unit of the largest, for the integer cores, by 7e-4, for a tenth less time where weights are all there is to read.)
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));

template <int G>
__device__ __forceinline__ uint32_t group_max(uint32_t v) {  // over the G / 8 lanes that hold a group
    v = max(v, static_cast<uint32_t>(dpp_i<0xB1>(static_cast<int>(v))));
    v = max(v, static_cast<uint32_t>(dpp_i<0x4E>(static_cast<int>(v))));
    if constexpr (G >= 64) v = max(v, static_cast<uint32_t>(dpp_i<0x141>(static_cast<int>(v))));
    if constexpr (G >= 128) v = max(v, static_cast<uint32_t>(dpp_i<0x140>(static_cast<int>(v))));
    return v;
}
// Sums over groups are in units of this, so that the largest scale times the largest factor, 2^16 2^113, stays below 2^128.
constexpr float kUnit = 4.0f;
// Eight entries of a group, whose other lanes hold the rest, as pairs in the order in which a word's codes come apart (0 2 4
// 6 1 3 5 7); returns what undoes the power of two, over kUnit. An infinity or a NaN is its own first part, with a second of
// 0, beside which the group's finite entries do not matter: they are brought below 2^15 whatever they are.
template <int G>
__device__ __forceinline__ float split8(const float (&x)[8], h8& hi, h8& lo) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
    top = group_max<G>(top);
    const bool finite = top < 0x7f800000u;
    const int e = top == 0 ? 0 : finite ? min(15 - __builtin_amdgcn_frexp_expf(__uint_as_float(top)), 100) : 15 - 128;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        constexpr int kOrder[8] = {0, 2, 4, 6, 1, 3, 5, 7};
        const v2f y = {ldexpf(x[kOrder[i]], e), ldexpf(x[kOrder[i + 1]], e)};
        const h2 a = __builtin_convertvector(y, h2);
        const v2f rest = {finite ? y[0] - static_cast<float>(a[0]) : 0.0f, finite ? y[1] - static_cast<float>(a[1]) : 0.0f};
        const h2 b = __builtin_convertvector(rest, h2);
        hi[i] = a[0], hi[i + 1] = a[1], lo[i] = b[0], lo[i + 1] = b[1];
    }
    return ldexpf(1.0f / kUnit, -e);
}
// the eight of a row that is in a block of 256 k: the part of 32 k, and the lanes c, that they belong to
template <int G>
__device__ __forceinline__ void place8(int eight, int& mi, int& c) {
    if constexpr (G == 32) mi = eight >> 2, c = eight & 3;
    else mi = eight >> 4 << 2 | (eight >> 3 & 1) << 1 | (eight & 1), c = eight >> 1 & 3;
}

// eight codes less their zero: zero1 = -(1024 + zero), zero16 = -(64 + zero), twice each. A code becomes fp16 as the
// last bits of 1024 + code, or of 1024 + 16 code.
__device__ __forceinline__ h8 less_zero(uint32_t w, h2 zero1, h2 zero16) {
    const h2 sixteenth = {static_cast<_Float16>(0.0625f), static_cast<_Float16>(0.0625f)};
    const uint32_t v = w >> 8;
    const h2 a = __builtin_bit_cast(h2, (w & 0x000f000fu) ^ 0x64086408u) + zero1;
    const h2 b = __builtin_elementwise_fma(__builtin_bit_cast(h2, (w & 0x00f000f0u) ^ 0x64806480u), sixteenth, zero16);
    const h2 c = __builtin_bit_cast(h2, (v & 0x000f000fu) ^ 0x64086408u) + zero1;
    const h2 d = __builtin_elementwise_fma(__builtin_bit_cast(h2, (v & 0x00f000f0u) ^ 0x64806480u), sixteenth, zero16);
    return h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// eight entries of a row from k on, 0 behind its end
__device__ __forceinline__ void load8(const float* row, int k, int K, bool wide, float (&x)[8]) {
    const float* src = row + k;
    if (wide && k + 8 <= K) {
        const v4f a = reinterpret_cast<const v4f*>(src)[0], b = reinterpret_cast<const v4f*>(src)[1];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = k + i < K ? src[i] : 0.0f;
    }
}

// An image of R rows of X (fewer may be there) over some blocks of 256 k, the operand of the products as it is read: [block][8 of
// 32 k][c] of 2 R places of 16 bytes, a row's eight entries' first parts and second ones in turn; then the groups' factors
// [group][R]. The places are moved on by image_turn, so that of the writers, who hold eights of one row, few
// meet in a bank; it is the same for c = 0 and 1, and for 2 and 3, whose readers are served together.
__host__ __device__ constexpr int image_bytes(int R) { return R * 1024; }
template <int G>
__host__ __device__ constexpr int meta_bytes(int R) { return R * (256 / G) * 4; }
template <int R>
__device__ __forceinline__ int image_turn(int mi, int c) { return R == 1 ? 0 : 2 * (mi & 3) + R * (c >> 1); }

// Makes the image of k [k0, k0 + kn) (kn a multiple of 256). A wave keeps to one row.
template <int G, int R>
__device__ __forceinline__ void make_image(const float* X, int64_t ldx, int K, int rows, int k0, int kn, uint8_t* img, uint8_t* meta,
                                           int lane, int wave) {
    constexpr int step = kThreads / R;
    const int count = kn / 8, first = wave / R * 64 + lane, r = wave & (R - 1);
    if (r >= rows) return;
    const bool wide = (ldx & 3) == 0 && (reinterpret_cast<uintptr_t>(X) & 15) == 0;
    constexpr int kBatch = R == 1 ? 1 : 4;  // requested together
    for (int id0 = first; id0 < count; id0 += kBatch * step) {
        float x[kBatch][8];
#pragma unroll
        for (int n = 0; n < kBatch; ++n) load8(X + r * ldx, k0 + min(id0 + n * step, count - 1) * 8, K, wide, x[n]);
#pragma unroll
        for (int n = 0; n < kBatch; ++n) {
            const int id = id0 + n * step;
            if (id >= count) break;     // 32 lanes are in or out together
            h8 hi, lo;
            const float factor = split8<G>(x[n], hi, lo);
            const int b = id >> 5, w = id & 31;  // the block, the eight in it
            int mi, c;
            place8<G>(w, mi, c);
            const int at = 2 * r + image_turn<R>(mi, c);
            uint8_t* to = img + b * image_bytes(R) + (mi * 4 + c) * R * 32;
            *reinterpret_cast<h8*>(to + (at & (2 * R - 1)) * 16) = hi;
            *reinterpret_cast<h8*>(to + ((at + 1) & (2 * R - 1)) * 16) = lo;
            if (w % (G / 8) == 0) reinterpret_cast<float*>(meta)[(b * (256 / G) + w / (G / 8)) * R + r] = factor;
        }
    }
}

// ---- the products
// A 16 x 16 x 32 fp16 product takes 16 rows of weights and, on its other side, up to eight rows of X as two parts each: lane
// 16 c + n holds, side by side, the two parts' sums of row c (of four rows; of eight, of rows 2 c and 2 c + 1; of one, of
// that row in every c) and weight row n, and only there are they added, scaled and added up in fp32. A group is one such
// product for every 32 k.
//
// A workgroup's waves take tiles of 16 weight rows, `ks` waves a tile, which share its k by blocks of 256 and
// add up in LDS. Weights go from memory to registers kDepth blocks ahead: with two, three workgroups' registers fit a
// compute unit (the head of 151936 rows 33.7 us, four ahead 38.0).
constexpr int kDepth = 2;

template <int G, bool ZP>
struct Unit {
    static constexpr int kScales = 256 / G, kWords = ZP ? kScales : kScales / 2, kBytes = 2048 + 64 * kWords;
    uint4 c[2];
    uint32_t s[kWords];
    __device__ void load(const uint8_t* u, int lane) {
        c[0] = *reinterpret_cast<const uint4*>(u + 16 * lane);
        c[1] = *reinterpret_cast<const uint4*>(u + 1024 + 16 * lane);
        const uint32_t* p = reinterpret_cast<const uint32_t*>(u + 2048) + (lane & 15) * kWords;
        if constexpr (kWords >= 4) {
#pragma unroll
            for (int i = 0; i < kWords; i += 4) {
                const uint4 v = *reinterpret_cast<const uint4*>(p + i);
                s[i] = v.x, s[i + 1] = v.y, s[i + 2] = v.z, s[i + 3] = v.w;
            }
        } else if constexpr (kWords == 2) {
            const uint2 v = *reinterpret_cast<const uint2*>(p);
            s[0] = v.x, s[1] = v.y;
        } else {
            s[0] = *p;
        }
    }
    __device__ float scale(int g) const { return half_bits(ZP ? s[g] : g & 1 ? s[g / 2] >> 16 : s[g / 2]); }
    __device__ int zero(int g) const { return static_cast<int>(s[g]) >> 16; }
    __device__ uint32_t word(int i) const {
        const uint4& v = c[i / 4];
        return (i & 3) == 0 ? v.x : (i & 3) == 1 ? v.y : (i & 3) == 2 ? v.z : v.w;
    }
};

// the zero points of a group as less_zero takes them
template <bool ZP, typename U>
__device__ __forceinline__ void zeros_of(const U& u, int g, h2& zero1, h2& zero16) {
    zero1 = h2{static_cast<_Float16>(-1032.0f), static_cast<_Float16>(-1032.0f)};
    zero16 = h2{static_cast<_Float16>(-72.0f), static_cast<_Float16>(-72.0f)};
    if constexpr (ZP) {
        const _Float16 z = static_cast<_Float16>(static_cast<short>(-u.zero(g)));
        const h2 zz = {z, z};
        zero1 += zz, zero16 += zz;
    }
}

// What a lane reads of the images for one group: the parts that it holds of the operand and its rows' factors.
template <int G, int R>
struct Operand {
    static constexpr int kEach = G / 32, kRows = R == 8 ? 2 : 1;
    h8 x[kEach];
    float factor[kRows];
    __device__ void load(const uint8_t* img, const uint8_t* meta, const int (&place)[4], int g) {
#pragma unroll
        for (int m = 0; m < kEach; ++m) x[m] = *reinterpret_cast<const h8*>(img + (g * kEach + m) * R * 128 + place[(g * kEach + m) & 3]);
        if constexpr (kRows == 2) {
            const v2f f = *reinterpret_cast<const v2f*>(meta + g * R * 4);
            factor[0] = f[0], factor[1] = f[1];
        } else {
            factor[0] = *reinterpret_cast<const float*>(meta + g * R * 4);
        }
    }
};

// A block of 256 k of a tile: img: the block's image; place[mi % 4]: this lane's bytes in the part of 32 k; meta: its place in
// the block's factors. What a group needs from LDS is asked for a group ahead.
template <int G, bool ZP, int R>
__device__ __forceinline__ void multiply(const Unit<G, ZP>& u, const uint8_t* img, const uint8_t* meta, const int (&place)[4],
                                         float (&acc)[R == 8 ? 2 : 1]) {
    typedef Operand<G, R> O;
    O o[2];
    o[0].load(img, meta, place, 0);
#pragma unroll
    for (int g = 0; g < 256 / G; ++g) {
        if (g + 1 < 256 / G) o[(g + 1) & 1].load(img, meta, place, g + 1);
        const O& x = o[g & 1];
        h2 zero1, zero16;
        zeros_of<ZP>(u, g, zero1, zero16);
        v4f d = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int m = 0; m < O::kEach; ++m)
            d = __builtin_amdgcn_mfma_f32_16x16x32_f16(x.x[m], less_zero(u.word(g * O::kEach + m), zero1, zero16), d, 0, 0, 0);
        const float sw = u.scale(g);
#pragma unroll
        for (int j = 0; j < O::kRows; ++j) acc[j] = fmaf(d[2 * j] + d[2 * j + 1], sw * x.factor[j], acc[j]);
    }
}

template <int G, bool ZP, int R>
__global__ __launch_bounds__(kThreads) void q4_mul_kernel(Q4MulArgs a, int most, int ks, int chunk) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    constexpr int kRows = R == 8 ? 2 : 1, kImage = image_bytes(R), kMeta = meta_bytes<G>(R);
    typedef Unit<G, ZP> U;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane >> 4, n = lane & 15;
    const int r0 = blockIdx.y * most, rows = min(most, a.M - r0);
    const int tiles = (a.N + 15) / 16, blocks = (a.K + 255) / 256, rt = kWaves / ks, part = wave & (ks - 1);
    const int sets = (tiles + rt - 1) / rt;
    uint8_t* meta = lds + kImage * chunk;
    float* red = reinterpret_cast<float*>(meta + kMeta * chunk);
    // this lane's places: rows that are not there hold whatever, as do the sums over them
    const int part_of = 2 * (R == 8 ? n >> 1 : R == 4 ? n >> 2 : 0) + (n & 1);
    int place[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) place[i] = c * R * 32 + ((part_of + image_turn<R>(i, c)) & (2 * R - 1)) * 16;
    const uint8_t* meta_lane = meta + (R == 8 ? c * 8 : R == 4 ? c * 4 : 0);
    const bool one = chunk >= blocks;   // one image serves all tiles
    bool made = false;
    U u[kDepth];
    // blocks b0 + part, + ks, .. of the set's tile, the first ones
    const auto load = [&](int set, int b0, int its) {
        const uint8_t* w = a.W + (static_cast<int64_t>(min(set * rt + wave / ks, tiles - 1)) * blocks + b0 + part) * U::kBytes;
#pragma unroll
        for (int i = 0; i < kDepth; ++i)
            if (i < its) u[i].load(w + i * ks * U::kBytes, lane);
        return w;
    };
    const uint8_t* w = nullptr;
    for (int set = blockIdx.x; set < sets; set += gridDim.x) {
        const int tile = set * rt + wave / ks;
        float acc[kRows];
#pragma unroll
        for (int j = 0; j < kRows; ++j) acc[j] = 0.0f;
        for (int b0 = 0; b0 < blocks; b0 += chunk) {
            const int bn = min(chunk, blocks - b0), its = (bn - part + ks - 1) / ks;
            if (!one || !made) {
                w = load(set, b0, its);
                if (made) lds_barrier();
                make_image<G, R>(a.X + r0 * a.ldx, a.ldx, a.K, rows, b0 * 256, bn * 256, lds, meta, lane, wave);
                made = true;
                lds_barrier();
            }
            const uint8_t *img = lds + part * kImage, *factors = meta_lane + part * kMeta;
            for (int i = 0; i < its; i += kDepth) {
#pragma unroll
                for (int j = 0; j < kDepth; ++j)
                    if (i + j < its) {
                        multiply<G, ZP, R>(u[j], img, factors, place, acc);
                        img += ks * kImage, factors += ks * kMeta;
                        if (i + j + kDepth < its) u[j].load(w + (i + j + kDepth) * ks * U::kBytes, lane);
                    }
            }
        }
        // the next set's first blocks, before this one's end
        if (one && set + static_cast<int>(gridDim.x) < sets) w = load(set + gridDim.x, 0, (blocks - part + ks - 1) / ks);
        const auto store = [&](int j, float y) {
            const int r = kRows * c + j, col = tile * 16 + n;
            if (r < rows && tile < tiles && col < a.N) {
                const int64_t at = r0 + r;
                a.Y[at * a.ldy + col] = fmaf(y, kUnit, a.R ? a.R[at * a.ldr + col] : 0.0f);
            }
        };
        if (ks == 1) {
#pragma unroll
            for (int j = 0; j < kRows; ++j) store(j, acc[j]);
            continue;
        }
#pragma unroll
        for (int j = 0; j < kRows; ++j) red[(wave * kRows + j) * 64 + lane] = acc[j];
        lds_barrier();
#pragma unroll
        for (int j = 0; j < kRows; ++j)
            if ((j & (ks - 1)) == part) {
                float y = 0.0f;
                for (int i = 0; i < ks; ++i) y += red[((wave - part + i) * kRows + j) * 64 + lane];
                store(j, y);
            }
        lds_barrier();
    }
}

// ---- the products of many rows
// Sixteen rows of X against sixteen of weights, 32 k at a time, each of their two parts a product. A group of 64 k costs a
// tile and 16 rows some 32 instructions and four products. 4096 rows of 8224 x 2048 take 395 us (349 TFLOP/s of products
// by X as it is, twice that of fp16 products); both pipes are busy in turn. Small products are bound by what comes first,
// X's image, which every workgroup makes.
constexpr int kManyRows = 16, kManyBytes = 16 * 1024, kPair = 2, kManyDepth = 2;
template <int G>
__host__ __device__ constexpr int many_bytes() { return kManyBytes + 256 / G * kManyRows * 4; }

// The image of a block of 256 k: [8 of 32 k][lo, hi][c] of 16 places of 16 bytes, a row's eight entries, moved on by many_turn
// as above; then the groups' factors [group][16].
__device__ __forceinline__ int many_turn(int mi, int c) { return 2 * (mi & 3) + 8 * (c >> 1); }
template <int G>
__device__ __forceinline__ void make_many(const float* X, int64_t ldx, int K, int rows, int k0, int blocks, uint8_t* img, uint8_t* meta,
                                          int lane, int wave) {
    const int count = blocks * 32;
    const bool wide = (ldx & 3) == 0 && (reinterpret_cast<uintptr_t>(X) & 15) == 0;
    constexpr int kBatch = 4;           // requested together
    for (int r = wave; r < rows; r += kWaves)
        for (int id0 = lane; id0 < count; id0 += kBatch * 64) {
            float x[kBatch][8];
#pragma unroll
            for (int n = 0; n < kBatch; ++n) load8(X + r * ldx, k0 + min(id0 + n * 64, count - 1) * 8, K, wide, x[n]);
#pragma unroll
            for (int n = 0; n < kBatch; ++n) {
                const int o = id0 + n * 64;
                if (o >= count) break;  // 32 lanes are in or out together
                h8 hi, lo;
                const float factor = split8<G>(x[n], hi, lo);
                const int b = o >> 5, w = o & 31;  // the block, the eight in it
                int mi, c;
                place8<G>(w, mi, c);
                uint8_t* at = img + b * kManyBytes + mi * 2048 + c * 256 + ((r + many_turn(mi, c)) & 15) * 16;
                *reinterpret_cast<h8*>(at) = lo;
                *reinterpret_cast<h8*>(at + 1024) = hi;
                if (w % (G / 8) == 0) reinterpret_cast<float*>(meta)[(b * (256 / G) + w / (G / 8)) * kManyRows + r] = factor;
            }
        }
}

// A block of 256 k of two tiles. img: the block's image; place[mi % 4]: this lane's bytes in the part of 32 k.
template <int G, bool ZP>
__device__ __forceinline__ void multiply_many(const Unit<G, ZP> (&u)[kPair], const uint8_t* img, const uint8_t* meta, const int (&place)[4],
                                              float (&acc)[kPair][4]) {
    constexpr int kEach = G / 32;
    h8 x[2][kEach][2];
    v4f factor[2];
    const auto load = [&](int g) {
#pragma unroll
        for (int m = 0; m < kEach; ++m)
#pragma unroll
            for (int p = 0; p < 2; ++p)
                x[g & 1][m][p] = *reinterpret_cast<const h8*>(img + (g * kEach + m) * 2048 + p * 1024 + place[(g * kEach + m) & 3]);
        factor[g & 1] = *reinterpret_cast<const v4f*>(meta + g * kManyRows * 4);
    };
    load(0);
#pragma unroll
    for (int g = 0; g < 256 / G; ++g) {
        if (g + 1 < 256 / G) load(g + 1);
        h8 w[kPair][kEach];
        v4f d[kPair];
#pragma unroll
        for (int t = 0; t < kPair; ++t) {
            h2 zero1, zero16;
            zeros_of<ZP>(u[t], g, zero1, zero16);
#pragma unroll
            for (int m = 0; m < kEach; ++m) w[t][m] = less_zero(u[t].word(g * kEach + m), zero1, zero16);
        }
        // the two tiles' in turn: a product waits for the one before of its own
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
            for (int m = 0; m < kEach; ++m)
#pragma unroll
                for (int t = 0; t < kPair; ++t)
                    d[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[g & 1][m][p], w[t][m], p || m ? d[t] : v4f{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int t = 0; t < kPair; ++t) {
            const float sw = u[t].scale(g);
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[t][r] = fmaf(d[t][r], sw * factor[g & 1][r], acc[t][r]);
        }
#pragma unroll
        for (int t = 0; t < kPair; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) pin(acc[t][r]);
    }
}

// As q4_mul_kernel, a wave's share being two tiles.
template <int G, bool ZP>
__global__ __launch_bounds__(kThreads) void q4_mul_many_kernel(Q4MulArgs a, int most, int ks, int chunk) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    constexpr int kMeta = 256 / G * kManyRows * 4;
    typedef Unit<G, ZP> U;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane >> 4, n = lane & 15;
    const int r0 = blockIdx.y * most, rows = min(most, a.M - r0);
    const int tiles = (a.N + 15) / 16, pairs = (tiles + 1) / 2, blocks = (a.K + 255) / 256, rt = kWaves / ks, part = wave & (ks - 1);
    const int sets = (pairs + rt - 1) / rt;
    uint8_t* meta = lds + kManyBytes * chunk;
    float* red = reinterpret_cast<float*>(meta + kMeta * chunk);
    // rows that are not there hold whatever, as do the sums over them
    int place[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) place[i] = c * 256 + ((n + many_turn(i, c)) & 15) * 16;
    const bool one = chunk >= blocks;   // one image serves all tiles
    bool made = false;
    for (int set = blockIdx.x; set < sets; set += gridDim.x) {
        const int tile = (set * rt + wave / ks) * 2;
        const uint8_t* w[kPair];
#pragma unroll
        for (int t = 0; t < kPair; ++t) w[t] = a.W + static_cast<int64_t>(min(tile + t, tiles - 1)) * blocks * U::kBytes;
        float acc[kPair][4];
#pragma unroll
        for (int t = 0; t < kPair; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[t][r] = 0.0f;
        for (int b0 = 0; b0 < blocks; b0 += chunk) {
            const int bn = min(chunk, blocks - b0);
            U u[kManyDepth][kPair];
#pragma unroll
            for (int i = 0; i < kManyDepth; ++i)
                if (part + i * ks < bn) {
#pragma unroll
                    for (int t = 0; t < kPair; ++t) u[i][t].load(w[t] + (b0 + part + i * ks) * U::kBytes, lane);
                }
            if (!one || !made) {
                if (made) lds_barrier();
                make_many<G>(a.X + r0 * a.ldx, a.ldx, a.K, rows, b0 * 256, bn, lds, meta, lane, wave);
                made = true;
                lds_barrier();
            }
            for (int b = part; b < bn; b += kManyDepth * ks) {
#pragma unroll
                for (int i = 0; i < kManyDepth; ++i) {
                    const int at = b + i * ks;
                    if (at < bn) {
                        multiply_many<G, ZP>(u[i], lds + at * kManyBytes, meta + at * kMeta + c * 16, place, acc);
                        if (at + kManyDepth * ks < bn) {
#pragma unroll
                            for (int t = 0; t < kPair; ++t) u[i][t].load(w[t] + (b0 + at + kManyDepth * ks) * U::kBytes, lane);
                        }
                    }
                }
            }
        }
        const auto store = [&](int t, int r, float y) {
            const int row = 4 * c + r, col = (tile + t) * 16 + n;
            if (row < rows && tile + t < tiles && col < a.N) {
                const int64_t at = r0 + row;
                a.Y[at * a.ldy + col] = fmaf(y, kUnit, a.R ? a.R[at * a.ldr + col] : 0.0f);
            }
        };
        if (ks == 1) {
#pragma unroll
            for (int t = 0; t < kPair; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) store(t, r, acc[t][r]);
            continue;
        }
#pragma unroll
        for (int t = 0; t < kPair; ++t) reinterpret_cast<v4f*>(red)[(wave * kPair + t) * 64 + lane] = v4f{acc[t][0], acc[t][1], acc[t][2], acc[t][3]};
        lds_barrier();
#pragma unroll
        for (int t = 0; t < kPair; ++t)
            if ((t & (ks - 1)) == part) {
                v4f y = {0.0f, 0.0f, 0.0f, 0.0f};
                for (int i = 0; i < ks; ++i) y += reinterpret_cast<const v4f*>(red)[((wave - part + i) * kPair + t) * 64 + lane];
#pragma unroll
                for (int r = 0; r < 4; ++r) store(t, r, y[r]);
            }
        lds_barrier();
    }
}

// 16 lanes a group. Without zero points the entry of the largest magnitude becomes code 0, -8 steps:
// scale = -entry / 8; with them the codes span [min(least, 0), max(largest, 0)]. Scales are rounded to
// fp16 first and codes chosen by the rounded scale. A group with an infinity or a NaN, or whose scale fp16 does not
// hold, gets scale NaN. Done once a model: 151936 x 2048 from bf16 take 352 us (2.2 TB/s; a copy's rate would be 152), from fp32
// 382 (272), a lane's short loads, maxima over lanes and divisions.
template <bool BF16, int G>
__global__ __launch_bounds__(256) void q4_quantize_kernel(const void* W, int N, int K, uint8_t* codes, uint16_t* scales, uint8_t* zeros) {
    constexpr int per = G / 16, kBytes = per * (BF16 ? 2 : 4);
    const int groups = (K + G - 1) / G, lane = threadIdx.x & 15;
    const int64_t id = static_cast<int64_t>(blockIdx.x) * 16 + threadIdx.x / 16;
    if (id >= static_cast<int64_t>(N) * groups) return;  // whole groups of 16 lanes leave
    const int64_t n = static_cast<uint32_t>(id) / groups;  // below 2^27
    const int g = static_cast<int>(static_cast<uint32_t>(id) % groups), k0 = g * G + lane * per;
    float x[per];
    if (k0 + per <= K && K % per == 0 && reinterpret_cast<uintptr_t>(W) % kBytes == 0) {  // in one piece
        struct alignas(kBytes < 16 ? kBytes : 16) Piece {
            uint32_t w[kBytes / 4];
        };
        const Piece v = *reinterpret_cast<const Piece*>(static_cast<const uint8_t*>(W) + (n * K + k0) * (BF16 ? 2 : 4));
#pragma unroll
        for (int i = 0; i < per; ++i) {
            if constexpr (BF16) x[i] = i & 1 ? bf16_hi(v.w[i / 2]) : bf16_lo(v.w[i / 2]);
            else x[i] = __uint_as_float(v.w[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < per; ++i) {
            if constexpr (BF16) x[i] = k0 + i < K ? bf16_to_f32(static_cast<const uint16_t*>(W)[n * K + k0 + i]) : 0.0f;
            else x[i] = k0 + i < K ? static_cast<const float*>(W)[n * K + k0 + i] : 0.0f;
        }
    }
    float lo = 0.0f, hi = 0.0f;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < per; ++i) {
        lo = fminf(lo, x[i]);
        hi = fmaxf(hi, x[i]);
        bad |= !(fabsf(x[i]) < INFINITY);
    }
    for (int d = 1; d < 16; d <<= 1) {
        lo = fminf(lo, __shfl_xor(lo, d, 16));
        hi = fmaxf(hi, __shfl_xor(hi, d, 16));
        bad |= static_cast<bool>(__shfl_xor(static_cast<int>(bad), d, 16));
    }
    uint16_t sb = bits_half(zeros ? (hi - lo) / 15.0f : (hi > -lo ? hi : lo) * -0.125f);
    if (bad || (sb & 0x7fff) >= 0x7c00) bad = true, sb = 0x7e00;
    const float s = half_bits(sb);
    const bool none = bad || s == 0.0f;
    const float zero = !zeros || none ? 8.0f : fminf(fmaxf(rintf(-lo / s), 0.0f), 15.0f);
    if (lane == 0) {
        scales[id] = sb;
        if (zeros) zeros[id] = static_cast<uint8_t>(zero);
    }
#pragma unroll
    for (int i = 0; i < per; i += 2) {
        uint32_t c[2];
#pragma unroll
        for (int j = 0; j < 2; ++j)
            c[j] = k0 + i + j >= K ? 0u
                   : none ? static_cast<uint32_t>(zero)
                          : static_cast<uint32_t>(fminf(fmaxf(rintf(x[i + j] / s) + zero, 0.0f), 15.0f));
        if (k0 + i < K) codes[n * ((K + 1) / 2) + (k0 + i) / 2] = static_cast<uint8_t>(c[0] | c[1] << 4);
    }
}

// A workgroup a unit: a thread per dword of codes (four bytes of them in their order, in one load where rows allow it), then
// per scale. Done once a model: 151936 x 2048 take 125 us (2.7 TB/s; at a copy's rate 64), by loads of four bytes a row.
__global__ __launch_bounds__(256) void q4_pack_kernel(const uint8_t* codes, const uint16_t* scales, const uint8_t* zeros, int N, int K,
                                                      int G, int unit, uint8_t* packed) {
    const int words = unit / 4, blocks = (K + 255) / 256, groups = (K + G - 1) / G;
    const int t = static_cast<int>(blockIdx.x / blocks), s = static_cast<int>(blockIdx.x % blocks);
    const bool wide = (K & 7) == 0 && (reinterpret_cast<uintptr_t>(codes) & 3) == 0;
    for (int w = threadIdx.x; w < words; w += 256) {
        uint32_t out = 0;
        if (w < 512) {
            const int h = w / 256, l = w / 4 % 64, i = w & 3, c = l / 16;
            const int n = t * 16 + (l & 15), k = s * 256 + 128 * h + (G == 32 ? 32 * i + 8 * c : 64 * (i / 2) + 16 * c + 8 * (i & 1));
            const uint8_t* row = codes + static_cast<int64_t>(n) * ((K + 1) / 2);
            if (n < N && k < K && wide) {
                const uint32_t b = *reinterpret_cast<const uint32_t*>(row + k / 2), even = b & 0x0f0f0f0fu, odd = b >> 4 & 0x0f0f0f0fu;
                out = (__builtin_amdgcn_perm(odd, even, 0x05010400u) | __builtin_amdgcn_perm(odd, even, 0x07030602u) << 4) ^ 0x88888888u;
            } else if (n < N) {
                for (int j = 0; j < 8; ++j) {
                    if (k + j >= K) break;
                    const uint32_t b = row[(k + j) / 2];
                    out |= (((j & 1 ? b >> 4 : b) & 15u) ^ 8u) << (8 * (j & 3) + (j & 4));
                }
            }
        } else {
            const int per = 256 / G, e = (w - 512) * (zeros ? 1 : 2);  // first scale of this dword
            for (int j = 0; j < (zeros ? 1 : 2); ++j) {
                const int n = t * 16 + (e + j) / per, g = s * per + (e + j) % per;
                if (n >= N || g >= groups) continue;
                const int64_t at = static_cast<int64_t>(n) * groups + g;
                if (zeros) out = scales[at] | static_cast<uint32_t>((zeros[at] & 15) - 8) << 16;
                else out |= static_cast<uint32_t>(scales[at]) << (16 * j);
            }
        }
        reinterpret_cast<uint32_t*>(packed)[static_cast<int64_t>(blockIdx.x) * words + w] = out;
    }
}

// Rows a block and its image's, waves a tile, workgroups a block of rows, blocks of 256 k an image holds.
struct Q4Plan {
    int most, image, row_blocks, ks, wgs, chunk;
    uint32_t lds;
};
template <int G, bool ZP>
void q4_fit(Q4Plan& p, int N, int K) {
    const bool many = p.image == kManyRows;
    const int blocks = q4_blocks(K), each = many ? many_bytes<G>() : image_bytes(p.image) + meta_bytes<G>(p.image);
    const int red = p.ks > 1 ? kWaves * (many ? 4 * kPair : p.image == 8 ? 2 : 1) * 256 : 0;
    p.chunk = std::min(blocks, (160 * 1024 - red) / each);
    p.lds = each * p.chunk + red;
}
template <int G, bool ZP>
Q4Plan q4_plan(int M, int N, int K) {
    Q4Plan p{};
    const int blocks = q4_blocks(K), tiles = q4_tiles(N);
    // Blocks of four rows fill the chip sooner, of eight read and unpack the weights less often (K 2048: 64 x 2048 in
    // fours 7.9 us, in eights 6.9; 8 x 8224 8.9 and 7.1; 32 x 2048 6.2 and 6.1; 12 x 2048 5.1 and 5.2; 8 x 2048 4.6 and 5.1;
    // 16 x 2048 x 6144 9.4 and 11.1).
    p.image = M == 1 ? 1 : tiles * ((M + 3) / 4) <= 1024 || M <= 4 ? 4 : 8;
    // Sixteen rows, and two tiles a wave, where rows and tiles are many (48 x 8224 x 2048 13.7 us, by eights 15.7; 32 x
    // 8224 13.0 and 14.7; 16 x 151936 54 and 62; 12 x 50000 18.8 and 23.8), else by fewer, whose smaller images are made
    // sooner (24 x 8224 10.7 us, by sixteens 12.4; 16 x 12288 10.1 and 11.0; 64 x 2048 6.9 and 8.3; 8 x 151936 39.5 and 51.7).
    if (M > 8 && static_cast<int64_t>(tiles) * M >= 16384) {
        p.image = kManyRows;
        p.row_blocks = (M + p.image - 1) / p.image;
        p.most = (M + p.row_blocks - 1) / p.row_blocks;
        // Waves that share a pair of tiles: as many as make the rounds of a workgroup a compute unit, each of so many blocks
        // of k and half a block's time for joining, least (48 x 8224 x 2048, two 13.7 us, one 18.4, four 16.0; 64 x 8224 x
        // 2048, four 17.9, two 18.7; 1024 x 8224 x 2048, one 107, two 116).
        const int pairs = (tiles + 1) / 2, most_wgs = std::max(1, 256 / p.row_blocks);
        int64_t best = INT64_MAX;
        for (int ks = 1; ks <= kWaves && (ks == 1 || ks <= blocks); ks *= 2) {
            const int sets = (pairs + kWaves / ks - 1) / (kWaves / ks), wgs = std::min(sets, most_wgs);
            const int64_t cost = static_cast<int64_t>((sets + wgs - 1) / wgs) * (2 * ((blocks + ks - 1) / ks) + (ks > 1));
            if (cost < best) best = cost, p.ks = ks, p.wgs = wgs;
        }
        q4_fit<G, ZP>(p, N, K);
        return p;
    }
    p.row_blocks = (M + p.image - 1) / p.image;
    p.most = (M + p.row_blocks - 1) / p.row_blocks;
    // Waves share a tile while there are not enough tiles: up to eight waves a compute unit, for one row up to 32
    // (1 x 12288 x 2048, eight waves a tile 5.8 us, two 6.1, one 7.8; 1 x 151936, one 33.9, two 36.2, eight 40.6; 8 x 8224,
    // two 7.2, eight 7.4, one 9.4).
    p.ks = kWaves;
    while (p.ks > 1 && (static_cast<int64_t>(tiles) * p.row_blocks * p.ks > (M == 1 ? 8192 : 2048) || p.ks / 2 >= blocks)) p.ks /= 2;
    const int rt = kWaves / p.ks, sets = (tiles + rt - 1) / rt;
    // two workgroups a compute unit go on from tile to tile (the head of 151936 rows: 33.5 us, by one 39.6, by all at once 34.2)
    p.wgs = std::min(sets, std::max(1, 512 / p.row_blocks));
    q4_fit<G, ZP>(p, N, K);
    return p;
}

template <int G, bool ZP, int R>
hipError_t launch_q4_form(const Q4MulArgs& a, const Q4Plan& p, hipStream_t s) {
    static AllowedLds allowed;
    const hipError_t e = allowed(reinterpret_cast<const void*>(q4_mul_kernel<G, ZP, R>), 160 * 1024);
    if (e != hipSuccess) return e;
    klaunch(q4_mul_kernel<G, ZP, R>, dim3(p.wgs, p.row_blocks), dim3(kThreads), p.lds, s, a, p.most, p.ks, p.chunk);
    return hipGetLastError();
}

template <int G, bool ZP>
hipError_t launch_q4_many(const Q4MulArgs& a, const Q4Plan& p, hipStream_t s) {
    static AllowedLds allowed;
    const hipError_t e = allowed(reinterpret_cast<const void*>(q4_mul_many_kernel<G, ZP>), 160 * 1024);
    if (e != hipSuccess) return e;
    klaunch(q4_mul_many_kernel<G, ZP>, dim3(p.wgs, p.row_blocks), dim3(kThreads), p.lds, s, a, p.most, p.ks, p.chunk);
    return hipGetLastError();
}

template <int G, bool ZP>
hipError_t launch_q4_plan(const Q4MulArgs& a, const Q4Plan& p, hipStream_t s) {
    return p.image == kManyRows ? launch_q4_many<G, ZP>(a, p, s) : p.image == 1 ? launch_q4_form<G, ZP, 1>(a, p, s) : p.image == 4 ? launch_q4_form<G, ZP, 4>(a, p, s) : launch_q4_form<G, ZP, 8>(a, p, s);
}

}  // namespace

hipError_t launch_q4_mul(const Q4MulArgs& a, hipStream_t s) {
    const auto go = [&](auto g, auto z) {
        constexpr int G = decltype(g)::value;
        constexpr bool Z = decltype(z)::value;
        return launch_q4_plan<G, Z>(a, q4_plan<G, Z>(a.M, a.N, a.K), s);
    };
    const auto by_zeros = [&](auto g) { return a.zeros ? go(g, std::true_type()) : go(g, std::false_type()); };
    return a.G == 32   ? by_zeros(std::integral_constant<int, 32>())
           : a.G == 64 ? by_zeros(std::integral_constant<int, 64>())
                       : by_zeros(std::integral_constant<int, 128>());
}

hipError_t launch_q4_quantize(const void* W, bool bf16, int N, int K, int G, uint8_t* codes, uint16_t* scales, uint8_t* zeros,
                              hipStream_t s) {
    const dim3 grid(static_cast<uint32_t>((static_cast<int64_t>(N) * ((K + G - 1) / G) + 15) / 16));
    const auto go = [&](auto g) {
        constexpr int kG = decltype(g)::value;
        klaunch(bf16 ? q4_quantize_kernel<true, kG> : q4_quantize_kernel<false, kG>, grid, dim3(256), 0, s, W, N, K, codes, scales, zeros);
    };
    G == 32 ? go(std::integral_constant<int, 32>()) : G == 64 ? go(std::integral_constant<int, 64>()) : go(std::integral_constant<int, 128>());
    return hipGetLastError();
}

hipError_t launch_q4_pack(const uint8_t* codes, const uint16_t* scales, const uint8_t* zeros, int N, int K, int G, uint8_t* packed,
                          hipStream_t s) {
    const int unit = q4_unit_bytes(G, zeros != nullptr);
    const int64_t units = static_cast<int64_t>(q4_tiles(N)) * q4_blocks(K);
    klaunch(q4_pack_kernel, dim3(static_cast<uint32_t>(units)), dim3(256), 0, s, codes, scales, zeros, N, K, G, unit, packed);
    return hipGetLastError();
}

}  // namespace q35k
