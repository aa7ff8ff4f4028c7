#pragma once
// Host-side launchers of the kernels of a decode step held in 4 bits: products with 4-bit weights
// (k_q4.hip), attention over a cache of 4-bit rows (k_attn_q4.hip), sampling (k_sample.hip).
// Shapes are checked by the callers (c_api_q4.hip, runtime.hip) before launching.
#include <atomic>
#include <cstdint>

#include "launch.hpp"

namespace q35k {

// ---------------------------------------------------------------- 4-bit weights
// Packed weights: units of 16 rows x 256 k, unit (t, s) of row tile t and k block s at
// (t * blocks + s) * unit bytes: 2048 bytes of codes, then each row's scales side by side (fp16, or
// with zero points dwords fp16 | (zero - 8) << 16). Rows and k beyond N and K hold code 0 and scale 0.
// A code is the 4 bits of (code - 8) in two's complement; lane l = 16 c + n of a wave finds row n's codes
// at 1024 h + 16 l, in four dwords i of eight codes j (low nibbles of the four bytes j = 0..3, high ones 4..7):
//   groups of 64, 128: k = 128 h + 64 (i / 2) + 16 c + 8 (i % 2) + j
//   groups of 32:      k = 128 h + 32 i + 8 c + j
constexpr int kQ4Rows = 16, kQ4Block = 256;
inline int q4_tiles(int N) { return (N + kQ4Rows - 1) / kQ4Rows; }
inline int q4_blocks(int K) { return (K + kQ4Block - 1) / kQ4Block; }
inline int q4_unit_bytes(int G, bool zeros) { return 2048 + kQ4Rows * (kQ4Block / G) * (zeros ? 4 : 2); }

struct Q4MulArgs {
    const float* X;
    const uint8_t* W;                   // packed
    const float* R;                     // may be null, may be Y
    float* Y;
    int64_t ldx, ldr, ldy;
    int M, N, K, G;
    bool zeros;
};
hipError_t launch_q4_mul(const Q4MulArgs& a, hipStream_t s);
// bf16 or fp32 W [N][K] -> codes [N][(K + 1) / 2], scales and (zeros not null) zeros [N][groups]
hipError_t launch_q4_quantize(const void* W, bool bf16, int N, int K, int G, uint8_t* codes, uint16_t* scales, uint8_t* zeros,
                              hipStream_t s);
hipError_t launch_q4_pack(const uint8_t* codes, const uint16_t* scales, const uint8_t* zeros, int N, int K, int G, uint8_t* packed,
                          hipStream_t s);

// ---------------------------------------------------------------- 4-bit cache rows
// A row: 256 codes in 128 bytes (dim 2 i in the low nibble of byte i), and for each 64 dims fp16
// (step, least) in a dword, step in the low half: x = least + step * code.
constexpr int kQ4RowBytes = 128, kQ4RowScales = 4;

struct AttnQ4Args {
    int B, NQ, NKV, GRP, ROT;
    int64_t cap;
    double theta;
    float eps;
    const int *len, *pos;               // device
    const float *qg, *k_new, *v_new, *q_norm, *k_norm;
    uint8_t *k, *v;
    uint32_t *k_scale, *v_scale;
    float* out;
    float* ws;
};
int64_t attn_q4_workspace_floats(const AttnQ4Args& a);
hipError_t launch_attn_q4(const AttnQ4Args& a, hipStream_t s);

struct KvQ4Args {
    int B, NKV;
    bool bf16, shared;
    int64_t rows_cap, cap;
    const int *begin, *end;             // device; begin may be null
    void *k_rows, *v_rows;
    uint8_t *k, *v;
    uint32_t *k_scale, *v_scale;
};
hipError_t launch_kv_q4(const KvQ4Args& a, bool store, hipStream_t s);

// ---------------------------------------------------------------- sampling
struct SampleArgs {
    int B, V;
    int64_t ld;
    const float *logits, *temperature;
    const int* top_k;                   // the three filters may be null: off
    const float *top_p, *min_p;
    const float* u;
    int* token;
    float* prob;                        // may be null
    void* ws;
    int* feed = nullptr;                // may be null: the token for a step to take, 0 where there is none
};
uint64_t sample_workspace_bytes(int B, int V);
hipError_t launch_sample(const SampleArgs& a, hipStream_t s);

// Lets a kernel have more LDS than the default limit, once a device.
struct AllowedLds {
    std::atomic<uint64_t> devices{0};
    hipError_t operator()(const void* kernel, int bytes) {
        int dev = 0;
        hipError_t e = hipGetDevice(&dev);
        if (e != hipSuccess || (dev < 64 && (devices.load() >> dev & 1))) return e;
        e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e == hipSuccess && dev < 64) devices.fetch_or(uint64_t{1} << dev);
        return e;
    }
};

}  // namespace q35k
