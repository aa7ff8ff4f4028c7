// Products with 4-bit weights and group scales: Y[m][n] = R[m][n] + sum_g s[n][g] sum_{k in g}
// X[m][k] (c[n][k] - z[n][g]), and the kernels that make such weights. The layout of packed weights
// is in launch_q4.hpp.
#include "dev_common.hpp"
#include "launch_q4.hpp"

namespace q35k {
namespace {

__device__ __forceinline__ float half_bits(uint32_t h) {
    return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(h)));
}
__device__ __forceinline__ uint16_t bits_half(float x) { return __builtin_bit_cast(uint16_t, static_cast<_Float16>(x)); }

// One wave an output, k spread over its lanes.
__global__ __launch_bounds__(256) void q4_mul_kernel(Q4MulArgs a) {
    const int lane = threadIdx.x & 63, n = blockIdx.x * 4 + threadIdx.x / 64, m = blockIdx.y;
    if (n >= a.N) return;
    const int unit = 2048 + 16 * (256 / a.G) * (a.zeros ? 4 : 2), blocks = (a.K + 255) / 256, r = n & 15;
    float acc = 0.0f;
    for (int k = lane; k < a.K; k += 64) {
        const uint8_t* u = a.W + (static_cast<int64_t>(n / 16) * blocks + k / 256) * unit;
        const int h = k / 128 % 2, kk = k & 127;
        int i, c;
        if (a.G == 32) {
            i = kk / 32;
            c = kk / 8 % 4;
        } else {
            c = kk / 16 % 4;
            i = 2 * (kk / 64) + kk / 8 % 2;
        }
        const uint32_t w = *reinterpret_cast<const uint32_t*>(u + 1024 * h + 16 * (16 * c + r) + 4 * i);
        const int j = k & 7, q = static_cast<int>(w << (28 - 8 * (j & 3) - (j & 4))) >> 28;
        const int g = (k & 255) / a.G;
        float scale;
        int zero = 0;
        if (a.zeros) {
            const uint32_t s = reinterpret_cast<const uint32_t*>(u + 2048)[r * (256 / a.G) + g];
            scale = half_bits(s);
            zero = static_cast<int>(s) >> 16;
        } else {
            scale = half_bits(reinterpret_cast<const uint16_t*>(u + 2048)[r * (256 / a.G) + g]);
        }
        acc = fmaf(a.X[m * a.ldx + k], scale * static_cast<float>(q - zero), acc);
    }
    acc = wave_sum(acc);
    if (lane == 0) a.Y[m * a.ldy + n] = acc + (a.R ? a.R[m * a.ldr + n] : 0.0f);
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

}  // namespace

uint64_t q4_mul_workspace_bytes(int M, int N, int K, int G) { return 16; }

hipError_t launch_q4_mul(const Q4MulArgs& a, hipStream_t s) {
    klaunch(q4_mul_kernel, dim3((a.N + 3) / 4, a.M), dim3(256), 0, s, a);
    return hipGetLastError();
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
