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
        *q = y;
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

template <bool KVB>
__device__ __forceinline__ float cache_at(const void* c, int64_t i) {
    if constexpr (KVB) return bf16_to_f32(static_cast<const uint16_t*>(c)[i]);
    else return static_cast<const float*>(c)[i];
}

// Workgroups of the prefix first ((piece, kv head, sequence)), then of the own caches ((piece,
// sequence, kv head)): the GRP query rows of one sequence over a piece of the keys, 64 at a
// time, scores by (key, row) pairs, outputs by dims.
template <bool KVB>
__global__ __launch_bounds__(256) void attn_batch_kernel(AttnBatchArgs a) {
    __shared__ float q[16][kHD];
    __shared__ float p[16][64];
    __shared__ float ms[16], ls[16], fs[16];
    const int tid = threadIdx.x;
    const int n_prefix = a.plan.pieces * a.NKV * a.B;
    const bool own = static_cast<int>(blockIdx.x) >= n_prefix;
    int i = own ? blockIdx.x - n_prefix : blockIdx.x;
    const int np = own ? a.plan.own : a.plan.pieces, piece = i % np;
    i /= np;
    const int kh = i % a.NKV, b = i / a.NKV;
    const int slot = new_slot(a, b);
    if (slot < 0) return;
    const int64_t lo = static_cast<int64_t>(piece) * (own ? a.plan.okeys : a.plan.pkeys);
    const int64_t hi = min(own ? static_cast<int64_t>(slot) + 1 : a.P, lo + (own ? a.plan.okeys : a.plan.pkeys));
    if (lo >= hi) return;
    const int64_t base = own ? (static_cast<int64_t>(b) * a.NKV + kh) * a.cap : kh * a.prefix_cap;
    const void *K = own ? a.k_own : a.k_prefix, *V = own ? a.v_own : a.v_prefix;
    const int G = a.GRP;
    const float* Q = a.Qa + (static_cast<int64_t>(kh) * a.B + b) * G * kHD;
    for (int g = 0; g < G; ++g) q[g][tid] = Q[g * kHD + tid];
    if (tid < 16) {
        ms[tid] = -INFINITY;
        ls[tid] = 0.0f;
    }
    float o[16];
#pragma unroll
    for (int g = 0; g < 16; ++g) o[g] = 0.0f;
    for (int64_t k0 = lo; k0 < hi; k0 += 64) {
        __syncthreads();
        const int n = static_cast<int>(min<int64_t>(64, hi - k0));
        for (int e = tid; e < G * 64; e += 256) {
            const int g = e >> 6, k = e & 63;
            float s = -INFINITY;
            if (k < n) {
                s = 0.0f;
                for (int d = 0; d < kHD; ++d) s += q[g][d] * cache_at<KVB>(K, (base + k0 + k) * kHD + d);
                s *= 0.0625f;
                if (own && a.own_score)
                    a.raw[((static_cast<int64_t>(b) * a.NKV + kh) * G + g) * a.cap + k0 + k] = s;
            }
            p[g][k] = s;
        }
        __syncthreads();
        if (tid < G) {
            float m = ms[tid];
            for (int k = 0; k < n; ++k) m = fmaxf(m, p[tid][k]);
            const float f = m == -INFINITY ? 1.0f : expf(ms[tid] - m);
            float l = ls[tid] * f;
            for (int k = 0; k < n; ++k) {
                p[tid][k] = m == -INFINITY ? 0.0f : expf(p[tid][k] - m);
                l += p[tid][k];
            }
            ms[tid] = m;
            ls[tid] = l;
            fs[tid] = f;
        }
        __syncthreads();
#pragma unroll
        for (int g = 0; g < 16; ++g)
            if (g < G) o[g] *= fs[g];
        for (int k = 0; k < n; ++k) {
            const float v = cache_at<KVB>(V, (base + k0 + k) * kHD + tid);
#pragma unroll
            for (int g = 0; g < 16; ++g)
                if (g < G) o[g] += p[g][k] * v;
        }
    }
    const int64_t row = own ? ((static_cast<int64_t>(b) * a.NKV + kh) * a.plan.own + piece) * G
                            : (static_cast<int64_t>(kh) * a.plan.pieces + piece) * a.B * G + b * G;
    float* po = (own ? a.part_o : a.part_p) + row * kHD;
    float2* ml = (own ? a.ml_o : a.ml_p) + row;
#pragma unroll
    for (int g = 0; g < 16; ++g)
        if (g < G) po[g * kHD + tid] = o[g];
    if (tid < G) ml[tid] = make_float2(ms[tid], ls[tid]);
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
    for (int g = 0; g < a.GRP; ++g) w += expf(a.raw[(bk * a.GRP + g) * a.cap + t] - ms[g]) / ls[g];
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
    c.total = c.raw + (a.own_score ? up4(rows * a.cap) : 0);
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
    const dim3 grid(a.B * a.NKV * (a.plan.pieces + a.plan.own));
    if (a.kv_bf16) klaunch(attn_batch_kernel<true>, grid, 256, 0, s, a);
    else klaunch(attn_batch_kernel<false>, grid, 256, 0, s, a);
    klaunch(attn_batch_combine_kernel, dim3(a.NQ, a.B), 256, 0, s, a);
    if (a.own_score)
        klaunch(attn_batch_score_kernel, dim3(static_cast<uint32_t>((a.cap + 255) / 256), a.NKV, a.B), 256, 0, s, a);
    return hipGetLastError();
}

}  // namespace q35k
