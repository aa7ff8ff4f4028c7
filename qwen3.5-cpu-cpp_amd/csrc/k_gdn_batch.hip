// The recurrent gated delta rule for a batch of sequences with a few tokens each
// (q35_gdn_batch): one workgroup per (sequence, v-head), the 128 x 128 state in registers
// through all tokens of the sequence, read once and written once.
//
// The rule is column-separable, so a wave owns 32 columns and needs no other wave: lane l holds
// rows 16 (l / 8) .. + 15 of columns 4 (l % 8) .. + 3 of its slice, and the column sums S^T k and
// S^T q reduce over the lane's rows and then over the 8 row groups by lane swaps. What the
// waves share goes through LDS for kTok tokens at a time: the conv window + SiLU of the
// head's q, k and v channels, the l2 norms, decay and beta before the recurrence, the gated norm
// of the readout after it.
#include "dev_common.hpp"
#include "launch.hpp"

namespace q35k {
namespace {

constexpr int kD = 128;
constexpr int kTok = 8;  // tokens per pass through LDS

// sum over the 8 lanes l, l ^ 8, ..., l ^ 56: a DPP rotation by 8 within each 16-lane row, then
// the 16- and 32-lane swaps of gfx950
__device__ __forceinline__ float row8_sum(float v) {
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x128, 0xF, 0xF, false));
    auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(int, v), __builtin_bit_cast(int, v), false, false);
    v = __builtin_bit_cast(float, static_cast<int>(r[0])) + __builtin_bit_cast(float, static_cast<int>(r[1]));
    r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(int, v), __builtin_bit_cast(int, v), false, false);
    return __builtin_bit_cast(float, static_cast<int>(r[0])) + __builtin_bit_cast(float, static_cast<int>(r[1]));
}

// rows [first, first + n) of sequence b, within the rows there are
__device__ __forceinline__ void rows_of(const GdnBatchArgs& a, int b, int& first, int& n) {
    first = a.row0 ? min(max(a.row0[b], 0), a.rows) : b;
    n = a.row0 ? max(min(a.row0[b + 1], a.rows) - first, 0) : 1;
}

// A channel of the ring after n tokens: slot i receives the last input of a position equal to i mod 4,
// from this call's rows or, where the batch is forked, from the ring that was read.
__device__ __forceinline__ void store_ring(const GdnBatchArgs& a, const float* rin, float* rout, uint32_t pos, int row, int n,
                                           bool fork, int ch, int CONV) {
#pragma unroll
    for (int i = 1; i <= 4; ++i) {  // the i-th input from the end
        const int64_t o = static_cast<int64_t>((pos + n - i) & 3) * CONV + ch;
        if (i <= n) rout[o] = a.qkv[static_cast<int64_t>(row + n - i) * a.ld_qkv + ch];
        else if (fork) rout[o] = rin[o];
    }
}

// ONE: a token per sequence (row0 null); the ring is written here then, by the workgroup that
// owns the channel. With more tokens a later token's slot is one that another workgroup may
// still have to read where v-heads share a k-head: gdn_batch_ring_kernel writes it afterwards.
template <bool ONE>
__global__ __launch_bounds__(256) void gdn_batch_kernel(GdnBatchArgs a) {
    constexpr int TC = ONE ? 1 : kTok;
    const int vh = blockIdx.x, b = blockIdx.y;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (a.pos[b] < 0) return;
    const uint32_t pos = a.pos[b];
    int row, n;
    rows_of(a, b, row, n);
    const bool fork = a.state_in != a.state;
    if (!ONE && n == 0 && !fork) return;
    const int rep = a.VH / a.KH, kh = vh / rep;
    const int KD = a.KH * kD, CONV = 2 * KD + a.VH * kD;
    __shared__ __align__(16) float x_s[TC][3 * kD];  // q, k, v after the window
    __shared__ __align__(16) float o_s[TC][kD];
    __shared__ float ab_s[TC][2];

    // channels of this thread: q or k channel tid, and v channel tid % 128 (both halves of the
    // workgroup, so that no load sits under a branch)
    const float* rin = a.ring_in + b * a.s_ring_in;
    float* rout = a.ring + b * a.s_ring;
    const int ch[2] = {tid < kD ? kh * kD + tid : KD + kh * kD + tid - kD, 2 * KD + vh * kD + (tid & (kD - 1))};
    float win[2][3];
    float4 w[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        w[c] = *reinterpret_cast<const float4*>(a.conv_w + static_cast<int64_t>(ch[c]) * 4);
#pragma unroll
        for (int i = 0; i < 3; ++i) win[c][i] = rin[static_cast<int64_t>((pos + 1 + i) & 3) * CONV + ch[c]];
    }
    // the state slice
    const int rg = lane >> 3, col = 32 * wave + 4 * (lane & 7);
    const int64_t soff = static_cast<int64_t>(vh) * kD * kD + (16 * rg) * kD + col;
    const float* Sin = a.state_in + b * a.s_state_in + soff;
    float4 s[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = *reinterpret_cast<const float4*>(Sin + i * kD);
    const float decay = -expf(a.A_log[vh]), dt = a.dt_bias[vh];

    // the rows of a pass are requested together: tokens past the last are the last again
    constexpr int ZT = (TC + 3) / 4;
    for (int t0 = 0; t0 < n; t0 += TC) {
        const int m = min(TC, n - t0);
        float x[2][TC], z[ZT][2], ab[2];
#pragma unroll
        for (int t = 0; t < TC; ++t) {
            const float* qkv = a.qkv + static_cast<int64_t>(row + t0 + min(t, m - 1)) * a.ld_qkv;
#pragma unroll
            for (int c = 0; c < 2; ++c) x[c][t] = qkv[ch[c]];
        }
        {
            const int64_t r = static_cast<int64_t>(row + t0 + min(tid, m - 1)) * a.ld_ba + vh;
            ab[0] = a.a[r];
            ab[1] = a.b[r];
        }
        if (a.norm_w) {
#pragma unroll
            for (int i = 0; i < ZT; ++i) {
                const float* zr = a.z + static_cast<int64_t>(row + t0 + min(wave + 4 * i, m - 1)) * a.ld_z + vh * kD;
                z[i][0] = zr[lane];
                z[i][1] = zr[lane + 64];
            }
        }
        if (t0) __syncthreads();
#pragma unroll
        for (int t = 0; t < TC; ++t) {
            if (t >= m) break;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float acc = 0.0f;
                acc += w[c].x * win[c][0];
                acc += w[c].y * win[c][1];
                acc += w[c].z * win[c][2];
                acc += w[c].w * x[c][t];
                if (ONE && (c ? tid < kD : vh % rep == 0)) {
                    rout[static_cast<int64_t>(pos & 3) * CONV + ch[c]] = x[c][t];
                    if (fork) {
#pragma unroll
                        for (int i = 0; i < 3; ++i) rout[static_cast<int64_t>((pos + 1 + i) & 3) * CONV + ch[c]] = win[c][i];
                    }
                }
                win[c][0] = win[c][1];
                win[c][1] = win[c][2];
                win[c][2] = x[c][t];
                if (c == 0 || tid < kD) x_s[t][c ? 2 * kD + tid : tid] = silu_f(acc);
            }
        }
        if (tid < m) {
            ab_s[tid][0] = expf(decay * softplus_f(ab[0] + dt));
            ab_s[tid][1] = sigmoid_f(ab[1]);
        }
        __syncthreads();
        // l2 norms (eps 1e-6, sums of squares in double) of q and k; q also scaled by DK^-1/2
        for (int i = wave; i < 2 * m; i += 4) {
            float* v = &x_s[i >> 1][(i & 1) * kD];
            const float u0 = v[lane], u1 = v[lane + 64];
            const double ss = wave_sum(static_cast<double>(u0) * u0 + static_cast<double>(u1) * u1);
            const float inv = 1.0f / sqrtf(static_cast<float>(ss) + 1e-6f);
            const float sc = i & 1 ? 1.0f : 1.0f / sqrtf(static_cast<float>(kD));
            v[lane] = (u0 * inv) * sc;
            v[lane + 64] = (u1 * inv) * sc;
        }
        __syncthreads();
        for (int t = 0; t < m; ++t) {
            const float alpha = ab_s[t][0], beta = ab_s[t][1];
            const float4* k4 = reinterpret_cast<const float4*>(&x_s[t][kD + 16 * rg]);
            const float4* q4 = reinterpret_cast<const float4*>(&x_s[t][16 * rg]);
            const float4 v4 = *reinterpret_cast<const float4*>(&x_s[t][2 * kD + col]);
            float kn[16], qn[16];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float4 u = k4[j], y = q4[j];
                kn[4 * j] = u.x, kn[4 * j + 1] = u.y, kn[4 * j + 2] = u.z, kn[4 * j + 3] = u.w;
                qn[4 * j] = y.x, qn[4 * j + 1] = y.y, qn[4 * j + 2] = y.z, qn[4 * j + 3] = y.w;
            }
            float4 km = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[i].x *= alpha, s[i].y *= alpha, s[i].z *= alpha, s[i].w *= alpha;
                km.x += s[i].x * kn[i], km.y += s[i].y * kn[i], km.z += s[i].z * kn[i], km.w += s[i].w * kn[i];
            }
            km.x = row8_sum(km.x), km.y = row8_sum(km.y), km.z = row8_sum(km.z), km.w = row8_sum(km.w);
            const float4 d = make_float4((v4.x - km.x) * beta, (v4.y - km.y) * beta, (v4.z - km.z) * beta,
                                         (v4.w - km.w) * beta);
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[i].x += kn[i] * d.x, s[i].y += kn[i] * d.y, s[i].z += kn[i] * d.z, s[i].w += kn[i] * d.w;
                o.x += s[i].x * qn[i], o.y += s[i].y * qn[i], o.z += s[i].z * qn[i], o.w += s[i].w * qn[i];
            }
            o.x = row8_sum(o.x), o.y = row8_sum(o.y), o.z = row8_sum(o.z), o.w = row8_sum(o.w);
            if (rg == 0) *reinterpret_cast<float4*>(&o_s[t][col]) = o;
        }
        __syncthreads();
        // readout, with the gated norm (src/forward_pass.cpp:86-93) where there is one
#pragma unroll
        for (int i = 0; i < ZT; ++i) {
            const int t = wave + 4 * i;
            if (t >= m) break;
            float o0 = o_s[t][lane], o1 = o_s[t][lane + 64];
            float* out = a.out + static_cast<int64_t>(row + t0 + t) * (a.VH * kD) + vh * kD;
            if (a.norm_w) {
                const double ss = wave_sum(static_cast<double>(o0) * o0 + static_cast<double>(o1) * o1);
                const float inv = 1.0f / sqrtf(static_cast<float>(ss / kD) + a.eps);
                o0 = a.norm_w[lane] * (o0 * inv) * silu_f(z[i][0]);
                o1 = a.norm_w[lane + 64] * (o1 * inv) * silu_f(z[i][1]);
            }
            out[lane] = o0;
            out[lane + 64] = o1;
        }
    }
    float* Sout = a.state + b * a.s_state + soff;
#pragma unroll
    for (int i = 0; i < 16; ++i) *reinterpret_cast<float4*>(Sout + i * kD) = s[i];
    if (!ONE && (fork || rep == 1)) {  // no other workgroup reads what is written here
        if (vh % rep == 0) store_ring(a, rin, rout, pos, row, n, fork, ch[0], CONV);
        if (tid < kD) store_ring(a, rin, rout, pos, row, n, fork, ch[1], CONV);
    }
}

// grid (CONV / 256, B): the rings, in place, where v-heads share a k-head's channels.
__global__ __launch_bounds__(256) void gdn_batch_ring_kernel(GdnBatchArgs a) {
    const int b = blockIdx.y, CONV = (2 * a.KH + a.VH) * kD, ch = blockIdx.x * 256 + threadIdx.x;
    if (a.pos[b] < 0 || ch >= CONV) return;
    int row, n;
    rows_of(a, b, row, n);
    float* ring = a.ring + b * a.s_ring;
    store_ring(a, ring, ring, a.pos[b], row, n, false, ch, CONV);
}

}  // namespace

hipError_t launch_gdn_batch(const GdnBatchArgs& a, hipStream_t s) {
    const dim3 grid(a.VH, a.B);
    if (!a.row0) {
        klaunch(gdn_batch_kernel<true>, grid, 256, 0, s, a);
    } else {
        klaunch(gdn_batch_kernel<false>, grid, 256, 0, s, a);
        if (a.state_in == a.state && a.VH != a.KH)
            klaunch(gdn_batch_ring_kernel, dim3(((2 * a.KH + a.VH) * kD + 255) / 256, a.B), 256, 0, s, a);
    }
    return hipGetLastError();
}

}  // namespace q35k
