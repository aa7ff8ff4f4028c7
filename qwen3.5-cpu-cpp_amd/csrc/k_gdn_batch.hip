// The recurrent gated delta rule for a batch of sequences with a few tokens each
// (q35_gdn_batch): one workgroup per (sequence, v-head), the 128 x 128 state in registers
// through all tokens of the sequence, read once and written once.
//
// The rule is column-separable, so a wave owns 128 / W columns (W waves) and needs no other wave:
// lane l holds R rows of columns 4 (l % C) .. + 3 of its slice (C lanes side by side, 64 / C row
// groups), and the column sums S^T k and S^T q reduce over the lane's rows and then over the row
// groups by lane swaps. Both sums are taken of the old state, as o = S_new^T q = alpha S^T q + (k.q) d:
// one reduction a token, off the update's path. What the waves share goes through LDS for kTok
// tokens at a time: the conv window + SiLU of the head's q, k and v channels, the l2 norms, k.q,
// decay and beta before the recurrence, the gated norm of the readout after it.
#include "dev_common.hpp"
#include "launch.hpp"

namespace q35k {
namespace {

constexpr int kD = 128;
constexpr int kTok = 8;  // tokens per pass through LDS

// Four sums over the row groups (lanes C apart), one a lane: those of the r-th 16 lanes end with component
// 0, 2, 1, 3 for r = 0 .. 3. The 32- and 16-lane swaps of gfx950 add two values at once, rotations within
// the 16 lanes the rest: 7 instructions, where four sums in every lane take 28.
template <int C>
__device__ __forceinline__ float group_sums(float4 v) {
    const auto add = [](auto r) {
        return __builtin_bit_cast(float, static_cast<int>(r[0])) + __builtin_bit_cast(float, static_cast<int>(r[1]));
    };
    const auto bits = [](float x) { return __builtin_bit_cast(int, x); };
    const float a = add(__builtin_amdgcn_permlane32_swap(bits(v.x), bits(v.y), false, false));
    const float b = add(__builtin_amdgcn_permlane32_swap(bits(v.z), bits(v.w), false, false));
    float s = add(__builtin_amdgcn_permlane16_swap(bits(a), bits(b), false, false));
    if constexpr (C == 4) s += dpp_f<0x124>(s);  // rotation by 4
    return s + dpp_f<0x128>(s);                  // by 8
}
__device__ __forceinline__ int component(int lane) { return (lane >> 5) + (lane >> 3 & 2); }
// the way back: all four components in every lane
__device__ __forceinline__ float4 all_components(float s) {
    const int i = __builtin_bit_cast(int, s);
    const auto r = __builtin_amdgcn_permlane16_swap(i, i, false, false);
    const auto p = __builtin_amdgcn_permlane32_swap(r[0], r[0], false, false), q = __builtin_amdgcn_permlane32_swap(r[1], r[1], false, false);
    const auto f = [](auto x) { return __builtin_bit_cast(float, static_cast<int>(x)); };
    return make_float4(f(p[0]), f(p[1]), f(q[0]), f(q[1]));
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
template <bool ONE, int W>
__global__ __launch_bounds__(64 * W) void gdn_batch_kernel(GdnBatchArgs a) {
    constexpr int TC = ONE ? 1 : kTok, NCH = 3 * kD > 64 * W ? 2 : 1;  // channels a thread
    constexpr int C = 32 / W, R = kD * C / 64;
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
    __shared__ float ab_s[TC][3];                    // decay, beta, k.q

    // channels of this thread, of the head's q, k and v channels in order (the threads beyond the
    // last take it again, so that no load sits under a branch)
    const float* rin = a.ring_in + b * a.s_ring_in;
    float* rout = a.ring + b * a.s_ring;
    int ch[NCH];
    bool mine[NCH], keeps[NCH];
    float win[NCH][3];
    float4 w[NCH];
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
        const int i = tid + 64 * W * c, j = min(i, 3 * kD - 1);
        ch[c] = j < kD ? kh * kD + j : j < 2 * kD ? KD + kh * kD + j - kD : 2 * KD + vh * kD + j - 2 * kD;
        mine[c] = i < 3 * kD;
        keeps[c] = mine[c] && (i >= 2 * kD || vh % rep == 0);  // this workgroup writes the channel's ring
        w[c] = *reinterpret_cast<const float4*>(a.conv_w + static_cast<int64_t>(ch[c]) * 4);
#pragma unroll
        for (int k = 0; k < 3; ++k) win[c][k] = rin[static_cast<int64_t>((pos + 1 + k) & 3) * CONV + ch[c]];
    }
    // the state slice
    const int rg = lane / C, col = 4 * C * wave + 4 * (lane % C), one = col + component(lane);
    const int64_t soff = static_cast<int64_t>(vh) * kD * kD + (R * rg) * kD + col;
    const float* Sin = a.state_in + b * a.s_state_in + soff;
    float4 s[R];
#pragma unroll
    for (int i = 0; i < R; ++i) s[i] = *reinterpret_cast<const float4*>(Sin + i * kD);
    const float decay = -expf(a.A_log[vh]), dt = a.dt_bias[vh];

    // the rows of a pass are requested together: tokens past the last are the last again
    constexpr int ZT = (TC + W - 1) / W;
    for (int t0 = 0; t0 < n; t0 += TC) {
        const int m = min(TC, n - t0);
        float x[NCH][TC], z[ZT][2], ab[2];
#pragma unroll
        for (int t = 0; t < TC; ++t) {
            const float* qkv = a.qkv + static_cast<int64_t>(row + t0 + min(t, m - 1)) * a.ld_qkv;
#pragma unroll
            for (int c = 0; c < NCH; ++c) x[c][t] = qkv[ch[c]];
        }
        {
            const int64_t r = static_cast<int64_t>(row + t0 + min(tid, m - 1)) * a.ld_ba + vh;
            ab[0] = a.a[r];
            ab[1] = a.b[r];
        }
        if (a.norm_w) {
#pragma unroll
            for (int i = 0; i < ZT; ++i) {
                const float* zr = a.z + static_cast<int64_t>(row + t0 + min(wave + W * i, m - 1)) * a.ld_z + vh * kD;
                z[i][0] = zr[lane];
                z[i][1] = zr[lane + 64];
            }
        }
        if (t0) lds_barrier();
        // four tokens at a time, so that their activations run side by side
#pragma unroll
        for (int g = 0; g < TC; g += 4) {
            if (g >= m) break;  // uniform
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
#pragma unroll
                for (int t = g; t < min(g + 4, TC); ++t) {  // (those past the last go nowhere)
                    float acc = 0.0f;
                    acc += w[c].x * win[c][0];
                    acc += w[c].y * win[c][1];
                    acc += w[c].z * win[c][2];
                    acc += w[c].w * x[c][t];
                    if (ONE && keeps[c]) {
                        rout[static_cast<int64_t>(pos & 3) * CONV + ch[c]] = x[c][t];
                        if (fork) {
#pragma unroll
                            for (int i = 0; i < 3; ++i) rout[static_cast<int64_t>((pos + 1 + i) & 3) * CONV + ch[c]] = win[c][i];
                        }
                    }
                    win[c][0] = win[c][1];
                    win[c][1] = win[c][2];
                    win[c][2] = x[c][t];
                    if (mine[c]) x_s[t][tid + 64 * W * c] = silu_f(acc);
                }
            }
        }
        if (tid < m) {
            ab_s[tid][0] = expf(decay * softplus_f(ab[0] + dt));
            ab_s[tid][1] = sigmoid_f(ab[1]);
        }
        lds_barrier();
        // l2 norms (eps 1e-6, sums in double) of q and k; q also scaled by DK^-1/2
        for (int t = wave; t < m; t += W) {
            float *q = &x_s[t][0], *k = &x_s[t][kD];
            const float q0 = q[lane], q1 = q[lane + 64], k0 = k[lane], k1 = k[lane + 64];
            const double qq = wave_sum(static_cast<double>(q0) * q0 + static_cast<double>(q1) * q1);
            const double kk = wave_sum(static_cast<double>(k0) * k0 + static_cast<double>(k1) * k1);
            const double kq = wave_sum(static_cast<double>(q0) * k0 + static_cast<double>(q1) * k1);
            const float iq = 1.0f / sqrtf(static_cast<float>(qq) + 1e-6f), ik = 1.0f / sqrtf(static_cast<float>(kk) + 1e-6f);
            const float sc = 1.0f / sqrtf(static_cast<float>(kD));
            q[lane] = (q0 * iq) * sc, q[lane + 64] = (q1 * iq) * sc;
            k[lane] = k0 * ik, k[lane + 64] = k1 * ik;
            if (lane == 0) ab_s[t][2] = static_cast<float>(kq * (static_cast<double>(iq) * ik * sc));
        }
        lds_barrier();
        for (int t = 0; t < m; ++t) {
            const float alpha = ab_s[t][0], beta = ab_s[t][1], kq = ab_s[t][2];
            const float v = x_s[t][2 * kD + one];
            float kn[R], qn[R];
#pragma unroll
            for (int j = 0; j < R; j += 4) {
                const float4 u = *reinterpret_cast<const float4*>(&x_s[t][kD + R * rg + j]);
                const float4 y = *reinterpret_cast<const float4*>(&x_s[t][R * rg + j]);
                kn[j] = u.x, kn[j + 1] = u.y, kn[j + 2] = u.z, kn[j + 3] = u.w;
                qn[j] = y.x, qn[j + 1] = y.y, qn[j + 2] = y.z, qn[j + 3] = y.w;
            }
            float4 km = make_float4(0.f, 0.f, 0.f, 0.f), o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int i = 0; i < R; ++i) {
                s[i].x *= alpha, s[i].y *= alpha, s[i].z *= alpha, s[i].w *= alpha;
                km.x += s[i].x * kn[i], km.y += s[i].y * kn[i], km.z += s[i].z * kn[i], km.w += s[i].w * kn[i];
                o.x += s[i].x * qn[i], o.y += s[i].y * qn[i], o.z += s[i].z * qn[i], o.w += s[i].w * qn[i];
            }
            // (a lane forms one component of d and of the readout)
            const float d1 = (v - group_sums<C>(km)) * beta;
            const float4 d = all_components(d1);
#pragma unroll
            for (int i = 0; i < R; ++i)
                s[i].x += kn[i] * d.x, s[i].y += kn[i] * d.y, s[i].z += kn[i] * d.z, s[i].w += kn[i] * d.w;
            const float o1 = group_sums<C>(o) + kq * d1;
            if ((lane & 15) < C) o_s[t][one] = o1;
        }
        lds_barrier();
        // readout, with the gated norm (src/forward_pass.cpp:86-93) where there is one
#pragma unroll
        for (int i = 0; i < ZT; ++i) {
            const int t = wave + W * i;
            if (t >= m) break;  // uniform
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
    for (int i = 0; i < R; ++i) *reinterpret_cast<float4*>(Sout + i * kD) = s[i];
    if (!ONE && (fork || rep == 1)) {  // no other workgroup reads what is written here
#pragma unroll
        for (int c = 0; c < NCH; ++c)
            if (keeps[c]) store_ring(a, rin, rout, pos, row, n, fork, ch[c], CONV);
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
    // eight waves a head while the token loop bounds the time, else four. Eight and four waves: 3 sequences
    // of 16 heads, 8 tokens, 13.2 us and 14.6; 20 of 0..8 19.0 and 20.3, 40 26.5 and 29.3, 64 34.4 and
    // 34.0; of one token 18 10.9 and 10.6, 64 26.9 and 24.2
    const bool few = static_cast<int64_t>(a.VH) * a.B <= device_cu_count() * (a.row0 ? 3 : 1);
    if (!a.row0) {
        if (few) klaunch(gdn_batch_kernel<true, 8>, grid, 512, 0, s, a);
        else klaunch(gdn_batch_kernel<true, 4>, grid, 256, 0, s, a);
    } else {
        if (few) klaunch(gdn_batch_kernel<false, 8>, grid, 512, 0, s, a);
        else klaunch(gdn_batch_kernel<false, 4>, grid, 256, 0, s, a);
        if (a.state_in == a.state && a.VH != a.KH)
            klaunch(gdn_batch_ring_kernel, dim3(((2 * a.KH + a.VH) * kD + 255) / 256, a.B), 256, 0, s, a);
    }
    return hipGetLastError();
}

}  // namespace q35k
