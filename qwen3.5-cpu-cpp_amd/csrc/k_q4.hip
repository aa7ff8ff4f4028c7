// Products with 4-bit weights and group scales: Y[m][n] = R[m][n] + sum_g s[n][g] sum_{k in g}
// X[m][k] (c[n][k] - z[n][g]), and the kernels that make such weights. The layout of packed weights
// is in launch_q4.hpp.
#include <mutex>
#include <type_traits>

#include "dev_q4.hpp"
#include "launch_q4.hpp"

namespace q35k {
namespace {

constexpr int kThreads = 512, kWaves = 8;

// ---- rows of X as whole numbers
// A group of a row's entries becomes multiples of a power of two, each three signed bytes: integer products
// with 4-bit codes are exact.
struct Digits {
    uint32_t d[3][2];                   // eight entries: plane, four bytes each
};
// the multiples of eight entries whose group's largest magnitude has the bits `top`, and 2^-e / 16 (codes are
// multiplied as 16 times themselves); NaN for a group with an infinity or a NaN
__device__ __forceinline__ Digits digits8(const float* x, uint32_t top, float& scale) {
    const float m = __uint_as_float(top);
    const int e = multiple_exp(m);
    const bool ok = top < 0x7f800000u && top != 0;
    scale = top >= 0x7f800000u ? NAN : ldexpf(0.0625f, ok ? -e : 0);
    uint32_t y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = signed_digits(ok ? static_cast<int>(rintf(ldexpf(x[i], e))) : 0);
    Digits r;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        r.d[0][h] = plane<0>(y[4 * h], y[4 * h + 1], y[4 * h + 2], y[4 * h + 3]);
        r.d[1][h] = plane<1>(y[4 * h], y[4 * h + 1], y[4 * h + 2], y[4 * h + 3]);
        r.d[2][h] = plane<2>(y[4 * h], y[4 * h + 1], y[4 * h + 2], y[4 * h + 3]);
    }
    return r;
}
template <int G>
__device__ __forceinline__ uint32_t group_max(uint32_t v) {  // over the G / 8 lanes that hold a group
    v = max(v, static_cast<uint32_t>(dpp_i<0xB1>(static_cast<int>(v))));
    v = max(v, static_cast<uint32_t>(dpp_i<0x4E>(static_cast<int>(v))));
    if constexpr (G >= 64) v = max(v, static_cast<uint32_t>(dpp_i<0x141>(static_cast<int>(v))));
    if constexpr (G >= 128) v = max(v, static_cast<uint32_t>(dpp_i<0x140>(static_cast<int>(v))));
    return v;
}
template <int G>
__device__ __forceinline__ int group_sum(int v) {
    v += dpp_i<0xB1>(v);
    v += dpp_i<0x4E>(v);
    if constexpr (G >= 64) v += dpp_i<0x141>(v);
    if constexpr (G >= 128) v += dpp_i<0x140>(v);
    return v;
}

// An image of R rows of X (fewer may be there) over some blocks of 64 k, the operand of the products as it is
// read: digit d of row r at k 64 b + 16 c + j in byte ((4 b + c) R + r) 48 + 16 d + j; then the groups' factors
// [group][R], floats, or with zero points four words: the sums of the three digits and the factor's bits.
template <int G, bool ZP>
__host__ __device__ constexpr int meta_bytes(int R, int k) { return R * (k / G) * (ZP ? 16 : 4); }

// Makes the image of k [k0, k0 + kn) (kn a multiple of 256) with the threads first, first + step, ..
template <int G, bool ZP, int R>
__device__ __forceinline__ void make_image(const float* X, int64_t ldx, int K, int rows, int k0, int kn, uint8_t* img, uint8_t* meta,
                                           int first, int step) {
    const int per = kn / 8;
    const bool wide = (ldx & 3) == 0 && (reinterpret_cast<uintptr_t>(X) & 15) == 0;
    for (int id = first; id < rows * per; id += step) {  // 32 lanes are in or out together
        const int r = R == 1 ? 0 : id / per, kk = (R == 1 ? id : id % per) * 8, k = k0 + kk;
        const float* src = X + r * ldx + k;
        float x[8];
        if (wide && k + 8 <= K) {
            const float4 a = reinterpret_cast<const float4*>(src)[0], b = reinterpret_cast<const float4*>(src)[1];
            x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = k + i < K ? src[i] : 0.0f;
        }
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
        float scale;
        const Digits d = digits8(x, group_max<G>(top), scale);
        uint8_t* at = img + ((kk >> 4) * R + r) * 48 + (kk & 8);
#pragma unroll
        for (int p = 0; p < 3; ++p) *reinterpret_cast<uint2*>(at + 16 * p) = make_uint2(d.d[p][0], d.d[p][1]);
        const int g = kk / G * R + r;
        if constexpr (ZP) {
            int s[3];
#pragma unroll
            for (int p = 0; p < 3; ++p)
                s[p] = group_sum<G>(__builtin_amdgcn_sdot4(static_cast<int>(d.d[p][1]), 0x01010101,
                                                           __builtin_amdgcn_sdot4(static_cast<int>(d.d[p][0]), 0x01010101, 0, false), false));
            if (kk % G == 0) reinterpret_cast<int4*>(meta)[g] = make_int4(s[0], s[1], s[2], __float_as_int(scale));
        } else {
            if (kk % G == 0) reinterpret_cast<float*>(meta)[g] = scale;
        }
    }
}

// The images of all blocks of R rows, in the workspace, then their factors.
template <int G, bool ZP, int R>
__global__ __launch_bounds__(256) void q4_image_kernel(const float* X, int64_t ldx, int M, int K, int most, uint8_t* img, uint8_t* meta) {
    const int r0 = blockIdx.y * most, kp = (K + 255) / 256 * 256;
    make_image<G, ZP, R>(X + r0 * ldx, ldx, K, min(most, M - r0), 0, kp, img + static_cast<int64_t>(blockIdx.y) * R * 3 * kp,
                         meta + static_cast<int64_t>(blockIdx.y) * meta_bytes<G, ZP>(R, kp), blockIdx.x * 256 + threadIdx.x, gridDim.x * 256);
}

// ---- the products
// A 16 x 16 x 64 integer product takes 16 rows of weights and, on its other side, four rows of X as four times
// three digits (the fourth row of each four is never looked at): lane 16 c + n holds the three digits' sums of
// row c of the four and weight row n side by side, and only there are they put together, scaled and added
// in fp32. A group is one such product (two for 128, one of depth 32 for 32), so sums are exact until they
// are scaled. Zero points start the sums at -16 zero x (sum of the digits).
//
// A workgroup's waves take tiles of 16 weight rows, `ks` waves a tile, which share its k by blocks of 256 and
// add up in LDS. Weights go from memory to registers kDepth blocks ahead.
constexpr int kDepth = 4;

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

// A block of 256 k: `img` and `meta` are this lane's places in the images of that block.
template <int G, bool ZP, int R>
__device__ __forceinline__ void multiply(const Unit<G, ZP>& u, const uint8_t* img, const uint8_t* meta, float* acc) {
    constexpr int QN = (R + 3) / 4;
#pragma unroll
    for (int g = 0; g < 256 / G; ++g) {
        const float sw = u.scale(g);
        // eight codes a word: bytes of 16 times the low and the high ones
        v4i b[G == 128 ? 2 : 1];
        if constexpr (G == 32) {
            const uint32_t w = u.word(g);
            b[0] = v4i{static_cast<int>(w << 4 & 0xf0f0f0f0u), static_cast<int>(w & 0xf0f0f0f0u), 0, 0};
        } else {
#pragma unroll
            for (int h = 0; h < G / 64; ++h) {
                const uint32_t w0 = u.word(2 * (g * (G / 64) + h)), w1 = u.word(2 * (g * (G / 64) + h) + 1);
                b[h] = v4i{static_cast<int>(w0 << 4 & 0xf0f0f0f0u), static_cast<int>(w0 & 0xf0f0f0f0u),
                           static_cast<int>(w1 << 4 & 0xf0f0f0f0u), static_cast<int>(w1 & 0xf0f0f0f0u)};
            }
        }
#pragma unroll
        for (int q = 0; q < QN; ++q) {
            float sx;
            v4i d = {0, 0, 0, 0};
            if constexpr (ZP) {
                const v4i t = *reinterpret_cast<const v4i*>(meta + (g * R + 4 * q) * 16);
                const int z = -16 * u.zero(g);
                d = v4i{z * t[0], z * t[1], z * t[2], 0};
                sx = __int_as_float(t[3]);
            } else {
                sx = *reinterpret_cast<const float*>(meta + (g * R + 4 * q) * 4);
            }
            if constexpr (G == 32) {
                const v2i a = *reinterpret_cast<const v2i*>(img + (g >> 1) * R * 192 + (g & 1) * R * 96 + q * 192);
                d = __builtin_amdgcn_mfma_i32_16x16x32_i8(__builtin_bit_cast(long, a), __builtin_bit_cast(long, v2i{b[0][0], b[0][1]}), d, 0, 0, 0);
            } else {
#pragma unroll
                for (int h = 0; h < G / 64; ++h) {
                    const v4i a = *reinterpret_cast<const v4i*>(img + (g * (G / 64) + h) * R * 192 + q * 192);
                    d = __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b[h], d, 0, 0, 0);
                }
            }
            acc[q] = fmaf(from_digits(d), sw * sx, acc[q]);
        }
    }
}

// From memory straight into LDS, a KB a wave at a time: a workgroup's copy of `bytes` (a multiple of 4, `to` 16-byte
// aligned; the rest behind the last 16 dword by dword).
__device__ __forceinline__ void copy_to_lds(uint8_t* to, const uint8_t* from, int bytes) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const auto glob = [](const uint8_t* p) {
        return reinterpret_cast<const __attribute__((address_space(1))) void*>(reinterpret_cast<uintptr_t>(p));
    };
    const auto local = [](uint8_t* p) { return reinterpret_cast<__attribute__((address_space(3))) void*>(reinterpret_cast<uintptr_t>(p)); };
    const int whole = bytes & ~15;
    for (int o = wave * 1024; o < whole; o += kWaves * 1024)
        if (o + 16 * lane < whole) __builtin_amdgcn_global_load_lds(glob(from + o + 16 * lane), local(to + o), 16, 0, 0);
    if (wave == 0 && 4 * lane < bytes - whole) __builtin_amdgcn_global_load_lds(glob(from + whole + 4 * lane), local(to + whole), 4, 0, 0);
}

template <int G, bool ZP, int R, bool PRE>
__global__ __launch_bounds__(kThreads) void q4_mul_kernel(Q4MulArgs a, int most, int ks, int chunk) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    constexpr int QN = (R + 3) / 4, kMeta = meta_bytes<G, ZP>(R, 256);
    typedef Unit<G, ZP> U;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane >> 4, n = lane & 15;
    const int r0 = blockIdx.y * most, rows = min(most, a.M - r0);
    const int tiles = (a.N + 15) / 16, blocks = (a.K + 255) / 256, rt = kWaves / ks, part = wave & (ks - 1);
    const int sets = (tiles + rt - 1) / rt;
    uint8_t* meta = lds + R * 768 * chunk;
    float* red = reinterpret_cast<float*>(meta + kMeta * chunk);
    // this lane's places: rows that are not there hold whatever, as do the sums over them
    const int digit = min(n & 3, 2), row = min(n >> 2, R - 1);
    const uint8_t* img_lane = lds + (G == 32 ? ((c >> 1) * R + row) * 48 + (c & 1) * 8 : (c * R + row) * 48) + digit * 16;
    const uint8_t* meta_lane = meta + min(c, R - 1) * (ZP ? 16 : 4);
    const bool one = chunk >= blocks;   // one image serves all tiles
    bool made = false;
    for (int set = blockIdx.x; set < sets; set += gridDim.x) {
        const int tile = set * rt + wave / ks;
        const uint8_t* W = a.W + static_cast<int64_t>(min(tile, tiles - 1)) * blocks * U::kBytes;
        float acc[QN];
#pragma unroll
        for (int q = 0; q < QN; ++q) acc[q] = 0.0f;
        for (int b0 = 0; b0 < blocks; b0 += chunk) {
            const int bn = min(chunk, blocks - b0), its = (bn - part + ks - 1) / ks;  // blocks b0 + part + i ks
            const uint8_t* w = W + static_cast<int64_t>(b0 + part) * U::kBytes;
            U u[kDepth];
#pragma unroll
            for (int i = 0; i < kDepth; ++i)
                if (i < its) u[i].load(w + i * ks * U::kBytes, lane);
            if (!one || !made) {
                if (made) lds_barrier();
                if constexpr (PRE) {
                    const int kp = blocks * 256;
                    const uint8_t *img = static_cast<const uint8_t*>(a.ws) + static_cast<int64_t>(blockIdx.y) * R * 3 * kp,
                                  *factors = static_cast<const uint8_t*>(a.ws) + static_cast<int64_t>(gridDim.y) * R * 3 * kp +
                                             static_cast<int64_t>(blockIdx.y) * kMeta * blocks;
                    copy_to_lds(lds, img + static_cast<int64_t>(b0) * R * 768, bn * R * 768);
                    copy_to_lds(meta, factors + static_cast<int64_t>(b0) * kMeta, bn * kMeta);
                    __builtin_amdgcn_s_waitcnt(0x0f70);  // vector memory, nothing outstanding
                } else {
                    make_image<G, ZP, R>(a.X + r0 * a.ldx, a.ldx, a.K, rows, b0 * 256, bn * 256, lds, meta, threadIdx.x, kThreads);
                }
                made = true;
                lds_barrier();
            }
            const uint8_t *img = img_lane + part * R * 768, *factors = meta_lane + part * kMeta;
            for (int i = 0; i < its; i += kDepth) {
#pragma unroll
                for (int j = 0; j < kDepth; ++j)
                    if (i + j < its) {
                        multiply<G, ZP, R>(u[j], img, factors, acc);
#pragma unroll
                        for (int q = 0; q < QN; ++q) pin(acc[q]);
                        img += ks * R * 768, factors += ks * kMeta;
                        if (i + j + kDepth < its) u[j].load(w + (i + j + kDepth) * ks * U::kBytes, lane);
                    }
            }
        }
        const auto store = [&](int q, float y) {
            const int r = 4 * q + c, col = tile * 16 + n;
            if (r < rows && tile < tiles && col < a.N) {
                const int64_t at = r0 + r;
                a.Y[at * a.ldy + col] = y + (a.R ? a.R[at * a.ldr + col] : 0.0f);
            }
        };
        if (ks == 1) {
#pragma unroll
            for (int q = 0; q < QN; ++q) store(q, acc[q]);
            continue;
        }
#pragma unroll
        for (int q = 0; q < QN; ++q) red[(wave * QN + q) * 64 + lane] = acc[q];
        lds_barrier();
#pragma unroll
        for (int q = 0; q < QN; ++q)
            if ((q & (ks - 1)) == part) {
                float y = 0.0f;
                for (int i = 0; i < ks; ++i) y += red[((wave - part + i) * QN + q) * 64 + lane];
                store(q, y);
            }
        lds_barrier();
    }
}

// 16 lanes a group. Without zero points the entry of the largest magnitude becomes code 0, -8 steps:
// scale = -entry / 8; with them the codes span [min(least, 0), max(largest, 0)]. Scales are rounded to
// fp16 first and codes chosen by the rounded scale. A group with an infinity or a NaN gets scale NaN.
template <bool BF16>
__global__ __launch_bounds__(256) void q4_quantize_kernel(const void* W, int N, int K, int G, uint8_t* codes, uint16_t* scales,
                                                          uint8_t* zeros) {
    const int groups = (K + G - 1) / G, lane = threadIdx.x & 15;
    const int64_t id = static_cast<int64_t>(blockIdx.x) * 16 + threadIdx.x / 16;
    if (id >= static_cast<int64_t>(N) * groups) return;  // whole groups of 16 lanes leave
    const int64_t n = id / groups;
    const int g = static_cast<int>(id % groups), k0 = g * G + lane * (G / 16), per = G / 16;
    const auto entry = [&](int k) -> float {
        if (k >= K) return 0.0f;
        if constexpr (BF16) return bf16_to_f32(static_cast<const uint16_t*>(W)[n * K + k]);
        else return static_cast<const float*>(W)[n * K + k];
    };
    float lo = 0.0f, hi = 0.0f;
    bool bad = false;
    for (int i = 0; i < per; ++i) {
        const float x = entry(k0 + i);
        lo = fminf(lo, x);
        hi = fmaxf(hi, x);
        bad |= !(fabsf(x) < INFINITY);
    }
    for (int d = 1; d < 16; d <<= 1) {
        lo = fminf(lo, __shfl_xor(lo, d, 16));
        hi = fmaxf(hi, __shfl_xor(hi, d, 16));
        bad |= static_cast<bool>(__shfl_xor(static_cast<int>(bad), d, 16));
    }
    const uint16_t sb = bad ? 0x7e00 : bits_half(zeros ? (hi - lo) / 15.0f : (hi > -lo ? hi : lo) * -0.125f);
    const float s = half_bits(sb);
    const bool none = bad || s == 0.0f;
    const float zero = !zeros || none ? 8.0f : fminf(fmaxf(rintf(-lo / s), 0.0f), 15.0f);
    if (lane == 0) {
        scales[id] = sb;
        if (zeros) zeros[id] = static_cast<uint8_t>(zero);
    }
    for (int i = 0; i < per; i += 2) {
        uint32_t c[2];
        for (int j = 0; j < 2; ++j)
            c[j] = k0 + i + j >= K ? 0u
                   : none ? static_cast<uint32_t>(zero)
                          : static_cast<uint32_t>(fminf(fmaxf(rintf(entry(k0 + i + j) / s) + zero, 0.0f), 15.0f));
        if (k0 + i < K) codes[n * ((K + 1) / 2) + (k0 + i) / 2] = static_cast<uint8_t>(c[0] | c[1] << 4);
    }
}

// a thread per dword of codes, then per scale
__global__ __launch_bounds__(256) void q4_pack_kernel(const uint8_t* codes, const uint16_t* scales, const uint8_t* zeros, int N, int K,
                                                      int G, int unit, int64_t units, uint8_t* packed) {
    const int words = unit / 4, blocks = (K + 255) / 256, groups = (K + G - 1) / G;
    const int64_t id = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (id >= units * words) return;
    const int64_t u = id / words;
    const int w = static_cast<int>(id % words), t = static_cast<int>(u / blocks), s = static_cast<int>(u % blocks);
    uint32_t out = 0;
    if (w < 512) {
        const int h = w / 256, l = w / 4 % 64, i = w & 3, c = l / 16;
        const int n = t * 16 + (l & 15), k = s * 256 + 128 * h + (G == 32 ? 32 * i + 8 * c : 64 * (i / 2) + 16 * c + 8 * (i & 1));
        if (n < N)
            for (int j = 0; j < 8; ++j) {
                if (k + j >= K) break;
                const uint32_t b = codes[static_cast<int64_t>(n) * ((K + 1) / 2) + (k + j) / 2];
                out |= (((j & 1 ? b >> 4 : b) & 15u) ^ 8u) << (8 * (j & 3) + (j & 4));
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
    reinterpret_cast<uint32_t*>(packed)[id] = out;
}

// Rows a block and its image's, waves a tile, workgroups, blocks of 256 k an image holds, and whether the images are
// made by a launch of their own.
struct Q4Plan {
    int most, image, row_blocks, ks, wgs, chunk;
    bool pre;
    uint32_t lds;
};
template <int G, bool ZP>
void q4_fit(Q4Plan& p, int N, int K) {
    const int blocks = q4_blocks(K), each = p.image * 768 + meta_bytes<G, ZP>(p.image, 256);
    const int red = p.ks > 1 ? kWaves * ((p.image + 3) / 4) * 256 : 0;
    p.chunk = std::min(blocks, std::max(1, (160 * 1024 - red) / each));
    p.lds = each * p.chunk + red;
}
template <int G, bool ZP>
Q4Plan q4_plan(int M, int N, int K) {
    Q4Plan p{};
    const int blocks = q4_blocks(K), tiles = q4_tiles(N);
    p.row_blocks = (M + 15) / 16;
    p.most = (M + p.row_blocks - 1) / p.row_blocks;
    p.image = p.most == 1 ? 1 : p.most <= 4 ? 4 : p.most <= 8 ? 8 : 16;
    p.pre = p.most > 4;
    p.ks = 8;
    while (p.ks > 1 && tiles * p.ks * p.row_blocks >= 2 * kWaves * 256) p.ks /= 2;
    while (p.ks > 1 && p.ks / 2 >= blocks) p.ks /= 2;
    const int rt = kWaves / p.ks, sets = (tiles + rt - 1) / rt;
    p.wgs = std::min(sets, std::max(1, 256 / p.row_blocks));
    q4_fit<G, ZP>(p, N, K);
    return p;
}

template <int G, bool ZP, int R, bool PRE>
hipError_t launch_q4_form(const Q4MulArgs& a, const Q4Plan& p, hipStream_t s) {
    static std::once_flag once;         // LDS beyond the default limit
    static hipError_t limit;
    std::call_once(once, [] {
        limit = hipFuncSetAttribute(reinterpret_cast<const void*>(q4_mul_kernel<G, ZP, R, PRE>), hipFuncAttributeMaxDynamicSharedMemorySize,
                                    160 * 1024);
    });
    if (limit != hipSuccess) return limit;
    if constexpr (PRE) {
        const int kp = q4_blocks(a.K) * 256;
        uint8_t* ws = static_cast<uint8_t*>(a.ws);
        klaunch(q4_image_kernel<G, ZP, R>, dim3((p.most * kp / 8 + 255) / 256, p.row_blocks), dim3(256), 0, s, a.X, a.ldx, a.M, a.K, p.most, ws,
                ws + static_cast<int64_t>(p.row_blocks) * R * 3 * kp);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    klaunch(q4_mul_kernel<G, ZP, R, PRE>, dim3(p.wgs, p.row_blocks), dim3(kThreads), p.lds, s, a, p.most, p.ks, p.chunk);
    return hipGetLastError();
}

template <int G, bool ZP>
hipError_t launch_q4_plan(const Q4MulArgs& a, const Q4Plan& p, hipStream_t s) {
    if (p.pre) return p.image == 4 ? launch_q4_form<G, ZP, 4, true>(a, p, s) : p.image == 8 ? launch_q4_form<G, ZP, 8, true>(a, p, s) : launch_q4_form<G, ZP, 16, true>(a, p, s);
    return p.image == 1 ? launch_q4_form<G, ZP, 1, false>(a, p, s) : p.image == 4 ? launch_q4_form<G, ZP, 4, false>(a, p, s) : launch_q4_form<G, ZP, 8, false>(a, p, s);
}

}  // namespace

uint64_t q4_mul_workspace_bytes(int M, int N, int K, int G) {
    const uint64_t kp = static_cast<uint64_t>(q4_blocks(K)) * 256;
    return (M + 15) / 16 * 16 * (3 * kp + kp / G * 16);
}

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
    const int64_t n = static_cast<int64_t>(N) * ((K + G - 1) / G);
    klaunch(bf16 ? q4_quantize_kernel<true> : q4_quantize_kernel<false>, dim3(static_cast<uint32_t>((n + 15) / 16)), dim3(256), 0, s, W,
            N, K, G, codes, scales, zeros);
    return hipGetLastError();
}

hipError_t launch_q4_pack(const uint8_t* codes, const uint16_t* scales, const uint8_t* zeros, int N, int K, int G, uint8_t* packed,
                          hipStream_t s) {
    const int unit = q4_unit_bytes(G, zeros != nullptr);
    const int64_t units = static_cast<int64_t>(q4_tiles(N)) * q4_blocks(K), n = units * (unit / 4);
    klaunch(q4_pack_kernel, dim3(static_cast<uint32_t>((n + 255) / 256)), dim3(256), 0, s, codes, scales, zeros, N, K, G, unit, units,
            packed);
    return hipGetLastError();
}

}  // namespace q35k
