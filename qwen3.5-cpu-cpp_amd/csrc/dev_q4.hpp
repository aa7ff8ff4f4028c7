#pragma once
// Device helpers of the 4-bit operators: fp16 scales; fp32 values as whole multiples of a power of two in
// three signed bytes, for exact products on the integer matrix cores; sums over a wave's lanes.
#include "dev_common.hpp"

namespace q35k {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef int v2i __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float half_bits(uint32_t h) {
    return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(h)));
}
__device__ __forceinline__ uint16_t bits_half(float x) { return __builtin_bit_cast(uint16_t, static_cast<_Float16>(x)); }

// Values whose largest magnitude is m as multiples of 2^-e: x = i 2^-e, |i| <= 8355711 = 127 (2^16 + 2^8 + 1), with
// the largest above 2^21.99, so that a value is off by at most 2^-23 of the largest. Values below 2^-100
// are multiples of that.
__device__ __forceinline__ int multiple_exp(float m) {
    int e = 23 - __builtin_amdgcn_frexp_expf(m);
    if (ldexpf(m, e) > 8355711.0f) --e;
    return min(e, 100);
}
// such an i = d2 2^16 + d1 2^8 + d0 as its signed digits, d0, d1, d2 in bytes 0, 1, 2 (byte 3: anything)
__device__ __forceinline__ uint32_t signed_digits(int i) { return (static_cast<uint32_t>(i) + 0x8080u) ^ 0x8080u; }
// byte p of each of four words, side by side
template <int P>
__device__ __forceinline__ uint32_t plane(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __builtin_amdgcn_perm(b, a, 0x0c0c0400u + P * 0x0101u) | __builtin_amdgcn_perm(d, c, 0x04000c0cu + P * 0x01010000u);
}
// three digits' sums of products as one number; its bits beyond 24 are rounded
__device__ __forceinline__ float from_digits(v4i d) {
    return fmaf(static_cast<float>(d[2] * 256 + d[1]), 256.0f, static_cast<float>(d[0]));
}

// Here the value exists: without it the compiler puts off what follows the products, whose sums (four
// registers for one value) then outnumber the registers.
__device__ __forceinline__ void pin(float& x) { asm volatile("" : "+v"(x)); }

// Sums of the lanes up to and with each: lanes 1, 2, 4, 8 before within a row of 16, then the rows before.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t moved(uint32_t v) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xF, false));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t moved(uint64_t v) {
    return static_cast<uint64_t>(moved<CTRL, ROWS>(static_cast<uint32_t>(v >> 32))) << 32 | moved<CTRL, ROWS>(static_cast<uint32_t>(v));
}
template <typename U>
__device__ __forceinline__ U wave_scan(U v) {
    v += moved<0x111, 0xF>(v);
    v += moved<0x112, 0xF>(v);
    v += moved<0x114, 0xF>(v);
    v += moved<0x118, 0xF>(v);
    v += moved<0x142, 0xA>(v);
    v += moved<0x143, 0xC>(v);
    return v;
}
__device__ __forceinline__ uint32_t lane_of(uint32_t v, int l) { return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), l)); }
__device__ __forceinline__ uint64_t lane_of(uint64_t v, int l) {
    return static_cast<uint64_t>(lane_of(static_cast<uint32_t>(v >> 32), l)) << 32 | lane_of(static_cast<uint32_t>(v), l);
}

}  // namespace q35k
