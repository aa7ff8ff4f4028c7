// Attention over caches of 4-bit rows (q35_attn_q4), and such rows from and to fp32 or bf16 caches
// (q35_kv_q4_store, q35_kv_q4_load). The layout of a row is in launch_q4.hpp.
//
// A row is quantized by 64 dims: least = fp16(min), step = fp16((max - least) / 15), code =
// round((x - least) / step), all from 64-bit values rounded to fp32 and then fp16: a value next to the
// border of two codes is on the same side for whoever computes it from the same inputs.
#include "dev_common.hpp"
#include "launch_q4.hpp"

namespace q35k {
namespace {

constexpr int kHD = 256;

__device__ __forceinline__ float half_bits(uint32_t h) {
    return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(h)));
}
__device__ __forceinline__ uint32_t bits_half(float x) {
    return __builtin_bit_cast(uint16_t, static_cast<_Float16>(x));
}
// fp16 through fp32: without the barrier the two roundings are compiled as one
__device__ __forceinline__ uint32_t bits_half(double x) {
    float f = static_cast<float>(x);
    asm("" : "+v"(f));
    return bits_half(f);
}
// least and step of a (step, least) dword
__device__ __forceinline__ float step_of(uint32_t s) { return half_bits(s & 0xffffu); }
__device__ __forceinline__ float least_of(uint32_t s) { return half_bits(s >> 16); }

__device__ __forceinline__ double min16(double v) {
    v = fmin(v, dpp_d<0xB1>(v));
    v = fmin(v, dpp_d<0x4E>(v));
    v = fmin(v, dpp_d<0x141>(v));
    return fmin(v, dpp_d<0x140>(v));
}
__device__ __forceinline__ int or16(int v) {
    v |= dpp_i<0xB1>(v);
    v |= dpp_i<0x4E>(v);
    v |= dpp_i<0x141>(v);
    return v | dpp_i<0x140>(v);
}

// A wave quantizes a row: lane l holds dims 4 l .. 4 l + 3, so 16 lanes are one group. Returns the lane's
// four codes (two bytes) and its group's (step, least). A group with an infinity or a NaN, or whose step
// or least value fp16 does not hold, has no values: both are NaN.
__device__ __forceinline__ uint32_t quantize4(const double* x, uint32_t& scale) {
    double lo = x[0], hi = x[0];
    int bad = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        lo = fmin(lo, x[i]);
        hi = fmax(hi, x[i]);
        bad |= !(fabs(x[i]) < static_cast<double>(INFINITY));
    }
    lo = min16(lo);
    hi = -min16(-hi);
    const uint32_t lb = bits_half(lo);
    const double least = half_bits(lb);
    const double d = (hi - least) / 15.0;
    const uint32_t sb = bits_half(d > 0.0 ? d : 0.0);
    const double step = half_bits(sb);
    if (or16(bad) || !(step < 65520.0) || !(fabs(least) < 65520.0)) {
        scale = 0x7e007e00u;
        return 0;
    }
    scale = sb | lb << 16;
    uint32_t c = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const double n = step == 0.0 ? 0.0 : rint((x[i] - least) / step);
        c |= static_cast<uint32_t>(fmin(fmax(n, 0.0), 15.0)) << (4 * i);
    }
    return c;
}

// A wave a row: the batch's query rows (normed, rotated, scaled, to the workspace), then the new
// key rows (normed, rotated) and value rows, quantized and appended at slot len[b].
__global__ __launch_bounds__(256) void attn_q4_prep_kernel(AttnQ4Args a, float* q) {
    __shared__ double row[4][kHD], cs[4][kHD];
    const int lane = threadIdx.x & 63, w = threadIdx.x / 64;
    const int64_t id = static_cast<int64_t>(blockIdx.x) * 4 + w;
    const int per = a.NQ + 2 * a.NKV;
    const int b = static_cast<int>(id / per), r = static_cast<int>(id % per);
    const int len = b < a.B ? a.len[b] : -1;
    const bool on = len >= 0 && len < a.cap, is_q = r < a.NQ, is_k = !is_q && r < a.NQ + a.NKV;
    const int h = is_q ? r : is_k ? r - a.NQ : r - a.NQ - a.NKV;
    double x[4] = {0, 0, 0, 0};
    if (on) {
        const float* src = is_q ? a.qg + (static_cast<int64_t>(b) * a.NQ + h) * 2 * kHD
                                : (is_k ? a.k_new : a.v_new) + (static_cast<int64_t>(b) * a.NKV + h) * kHD;
        const float4 f = reinterpret_cast<const float4*>(src)[lane];
        x[0] = f.x, x[1] = f.y, x[2] = f.z, x[3] = f.w;
        if (is_q || is_k) {
            const double ss = wave_sum(x[0] * x[0] + x[1] * x[1] + x[2] * x[2] + x[3] * x[3]);
            const double inv = 1.0 / sqrt(ss / kHD + static_cast<double>(a.eps));
            const float4 nw = reinterpret_cast<const float4*>(is_q ? a.q_norm : a.k_norm)[lane];
            x[0] *= inv * (1.0 + nw.x), x[1] *= inv * (1.0 + nw.y), x[2] *= inv * (1.0 + nw.z), x[3] *= inv * (1.0 + nw.w);
            const int half = a.ROT / 2;
            for (int i = lane; i < half; i += 64) {
                const double ang = static_cast<double>(a.pos[b]) * pow(a.theta, -static_cast<double>(2 * i) / a.ROT);
                cs[w][i] = cos(ang);
                cs[w][128 + i] = sin(ang);
            }
            for (int i = 0; i < 4; ++i) row[w][4 * lane + i] = x[i];
        }
    }
    __syncthreads();
    if (!on) return;
    if (is_q || is_k) {
        const int half = a.ROT / 2;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = 4 * lane + i;
            if (d < half) x[i] = x[i] * cs[w][d] - row[w][d + half] * cs[w][128 + d];
            else if (d < a.ROT) x[i] = x[i] * cs[w][d - half] + row[w][d - half] * cs[w][128 + d - half];
        }
    }
    if (is_q) {
        reinterpret_cast<float4*>(q + (static_cast<int64_t>(b) * a.NQ + h) * kHD)[lane] =
            make_float4(static_cast<float>(x[0] * 0.0625), static_cast<float>(x[1] * 0.0625), static_cast<float>(x[2] * 0.0625),
                        static_cast<float>(x[3] * 0.0625));
        return;
    }
    uint32_t scale;
    const uint32_t c = quantize4(x, scale);
    const int64_t at = (static_cast<int64_t>(b) * a.NKV + h) * a.cap + len;
    reinterpret_cast<uint16_t*>(is_k ? a.k : a.v)[at * 64 + lane] = static_cast<uint16_t>(c);
    if ((lane & 15) == 0) (is_k ? a.k_scale : a.v_scale)[at * 4 + lane / 16] = scale;
}

// a wave per query head: the keys one after another
__global__ __launch_bounds__(64) void attn_q4_kernel(AttnQ4Args a, const float* q) {
    const int lane = threadIdx.x, h = blockIdx.x, b = blockIdx.y;
    const int len = a.len[b];
    if (len < 0) return;
    const int64_t o = static_cast<int64_t>(b) * a.NQ + h;
    float4* out = reinterpret_cast<float4*>(a.out + o * kHD) + lane;
    if (len >= a.cap) {  // nothing was appended
        *out = make_float4(NAN, NAN, NAN, NAN);
        return;
    }
    const float4 x = reinterpret_cast<const float4*>(q + o * kHD)[lane];
    float m = -INFINITY, l = 0.0f;
    float acc[4] = {0, 0, 0, 0};
    for (int t = 0; t <= len; ++t) {
        const int64_t at = (static_cast<int64_t>(b) * a.NKV + h / a.GRP) * a.cap + t;
        const uint32_t kc = reinterpret_cast<const uint16_t*>(a.k)[at * 64 + lane], ks = a.k_scale[at * 4 + lane / 16];
        const uint32_t vc = reinterpret_cast<const uint16_t*>(a.v)[at * 64 + lane], vs = a.v_scale[at * 4 + lane / 16];
        const auto val = [](uint32_t c, int i, uint32_t s) { return fmaf(step_of(s), static_cast<float>(c >> (4 * i) & 15u), least_of(s)); };
        const float s = wave_sum(x.x * val(kc, 0, ks) + x.y * val(kc, 1, ks) + x.z * val(kc, 2, ks) + x.w * val(kc, 3, ks));
        const float mn = fmaxf(m, s), al = expf(m - mn), p = expf(s - mn);
        m = mn;
        l = l * al + p;
        for (int i = 0; i < 4; ++i) acc[i] = acc[i] * al + p * val(vc, i, vs);
    }
    const float4 g = reinterpret_cast<const float4*>(a.qg + o * 2 * kHD + kHD)[lane];
    *out = make_float4(acc[0] / l * sigmoid_f(g.x), acc[1] / l * sigmoid_f(g.y), acc[2] / l * sigmoid_f(g.z), acc[3] / l * sigmoid_f(g.w));
}

// whether rows [i, e) of sequence b are there
__device__ __forceinline__ bool range_of(const KvQ4Args& a, int b, int& i, int& e) {
    i = a.begin ? a.begin[b] : 0;
    e = a.end[b];
    return i >= 0 && e > i && e <= a.cap && e <= a.rows_cap;
}

// a wave a row of K or of V at a time: blockIdx.y = 2 (b NKV + h) + (0: K, 1: V)
template <bool BF16, bool STORE>
__global__ __launch_bounds__(256) void kv_q4_kernel(KvQ4Args a) {
    const int lane = threadIdx.x & 63;
    for (int64_t id = blockIdx.y; id < 2ll * a.B * a.NKV; id += gridDim.y) {
        const int b = static_cast<int>(id / 2 / a.NKV), h = static_cast<int>(id / 2 % a.NKV), v = static_cast<int>(id & 1);
        int i, e;
        if (!range_of(a, b, i, e)) continue;
        const int64_t from = (static_cast<int64_t>(a.shared ? 0 : b) * a.NKV + h) * a.rows_cap, to = (id / 2) * a.cap;
        for (int64_t t = i + blockIdx.x * 4 + threadIdx.x / 64; t < e; t += gridDim.x * 4) {
            void* rows = v ? a.v_rows : a.k_rows;
            uint16_t* codes = reinterpret_cast<uint16_t*>(v ? a.v : a.k) + (to + t) * 64 + lane;
            uint32_t* scale = (v ? a.v_scale : a.k_scale) + (to + t) * 4 + lane / 16;
            float f[4];
            if constexpr (STORE) {
                if constexpr (BF16) {
                    const uint2 u = static_cast<const uint2*>(rows)[(from + t) * 64 + lane];
                    f[0] = bf16_lo(u.x), f[1] = bf16_hi(u.x), f[2] = bf16_lo(u.y), f[3] = bf16_hi(u.y);
                } else {
                    const float4 u = static_cast<const float4*>(rows)[(from + t) * 64 + lane];
                    f[0] = u.x, f[1] = u.y, f[2] = u.z, f[3] = u.w;
                }
                const double x[4] = {f[0], f[1], f[2], f[3]};
                uint32_t sc;
                const uint32_t c = quantize4(x, sc);
                *codes = static_cast<uint16_t>(c);
                if ((lane & 15) == 0) *scale = sc;
            } else {
                const uint32_t c = *codes, sc = *scale;
                for (int j = 0; j < 4; ++j) f[j] = fmaf(step_of(sc), static_cast<float>(c >> (4 * j) & 15u), least_of(sc));
                if constexpr (BF16) {
                    uint32_t p[4];
                    for (int j = 0; j < 4; ++j) p[j] = f[j] == f[j] ? f32_to_bf16(f[j]) : 0x7fc0u;
                    static_cast<uint2*>(rows)[(from + t) * 64 + lane] = make_uint2(p[0] | p[1] << 16, p[2] | p[3] << 16);
                } else {
                    static_cast<float4*>(rows)[(from + t) * 64 + lane] = make_float4(f[0], f[1], f[2], f[3]);
                }
            }
        }
    }
}

}  // namespace

int64_t attn_q4_workspace_floats(const AttnQ4Args& a) { return static_cast<int64_t>(a.B) * a.NQ * kHD; }

hipError_t launch_attn_q4(const AttnQ4Args& a, hipStream_t s) {
    const int64_t rows = static_cast<int64_t>(a.B) * (a.NQ + 2 * a.NKV);
    klaunch(attn_q4_prep_kernel, dim3(static_cast<uint32_t>((rows + 3) / 4)), dim3(256), 0, s, a, a.ws);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    klaunch(attn_q4_kernel, dim3(a.NQ, a.B), dim3(64), 0, s, a, static_cast<const float*>(a.ws));
    return hipGetLastError();
}

hipError_t launch_kv_q4(const KvQ4Args& a, bool store, hipStream_t s) {
    const int64_t n = std::min(a.cap, a.rows_cap), y = std::min<int64_t>(2ll * a.B * a.NKV, 32768);
    const dim3 grid(static_cast<uint32_t>(std::min<int64_t>((n + 3) / 4, std::max<int64_t>(1, 8192 / y))), static_cast<uint32_t>(y));
    if (store) klaunch(a.bf16 ? kv_q4_kernel<true, true> : kv_q4_kernel<false, true>, grid, dim3(256), 0, s, a);
    else klaunch(a.bf16 ? kv_q4_kernel<true, false> : kv_q4_kernel<false, false>, grid, dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace q35k
