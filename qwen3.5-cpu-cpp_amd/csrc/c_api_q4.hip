// C ABI of the operators of a decode step held in 4 bits (q35_matmul_q4 and what makes its weights,
// q35_attn_q4, q35_kv_q4_store / _load) and of q35_sample: sizes and pointers are checked here, lengths
// and settings that only the device knows are bounded in the kernels.
#include <hip/hip_runtime.h>

#include "../host/q35_internal.h"
#include "launch_q4.hpp"

namespace {

q35_status launched(hipError_t e, const char* what) {
    return e == hipSuccess ? Q35_OK : q35::fail(Q35_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// [p, p + n) and [q, q + m) share a byte
bool overlap(const void* p, uint64_t n, const void* q, uint64_t m) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(p), y = reinterpret_cast<uintptr_t>(q);
    return n && m && x < y + m && y < x + n;
}

// An array of a call. What is written may overlap nothing else (what is read may be the same array twice).
struct Part {
    const void* p;
    uint64_t n;
    bool out;
};
template <int N>
bool written_overlaps(const Part (&part)[N]) {
    for (int i = 0; i < N; ++i)
        for (int j = i + 1; j < N; ++j)
            if ((part[i].out || part[j].out) && overlap(part[i].p, part[i].n, part[j].p, part[j].n)) return true;
    return false;
}

// The kernels run on the current device: a stream of another one is refused.
q35_status check_stream(hipStream_t s, const char* who) {
    if (!s) return Q35_OK;
    int dev = -1, sdev = -1;
    hipError_t e = hipGetDevice(&dev);
    if (e == hipSuccess) e = hipStreamGetDevice(s, &sdev);
    if (e != hipSuccess) return q35::fail(Q35_ERR_HIP, "%s: %s", who, hipGetErrorString(e));
    if (dev != sdev)
        return q35::fail(Q35_ERR_ARG, "%s: the stream belongs to device %d but device %d is current", who, sdev, dev);
    return Q35_OK;
}

// Of q35_matmul_q4, which leaves it alone: X's images lie in LDS, and waves that share a tile add up there.
constexpr uint64_t kMulWorkspace = 16;
constexpr int64_t kMostWeights = 1ll << 32;  // N x K: a kernel's threads stay below the 2^32 of a grid

q35_status q4_sizes(int32_t N, int32_t K, int32_t group, const char* who) {
    if (N < 1 || K < 1) return q35::fail(Q35_ERR_ARG, "%s: %d rows of %d weights", who, N, K);
    if (group != 32 && group != 64 && group != 128) return q35::fail(Q35_ERR_UNSUPPORTED, "%s: groups of %d", who, group);
    // rows and k are padded to units of 16 x 256
    if ((N + 15ll) / 16 * 16 * ((K + 255ll) / 256 * 256) > kMostWeights)
        return q35::fail(Q35_ERR_UNSUPPORTED, "%s: %d rows of %d weights", who, N, K);
    return Q35_OK;
}

q35_status attn_q4_sizes(const q35_attn_q4_args* args, const char* who, q35k::AttnQ4Args* out) {
    if (!args) return q35::fail(Q35_ERR_ARG, "%s: null args", who);
    const q35_attn_q4_args& g = *args;
    if (g.head_dim != 256) return q35::fail(Q35_ERR_UNSUPPORTED, "%s: head_dim must be 256", who);
    if (g.batch <= 0 || g.q_heads <= 0 || g.kv_heads <= 0 || g.q_heads % g.kv_heads != 0)
        return q35::fail(Q35_ERR_ARG, "%s: bad batch or head counts", who);
    if (g.q_heads / g.kv_heads > 16) return q35::fail(Q35_ERR_UNSUPPORTED, "%s: GQA group %d", who, g.q_heads / g.kv_heads);
    if (static_cast<int64_t>(g.batch) * g.q_heads > 1 << 22 || g.batch > 65535 || g.q_heads > 4096)
        return q35::fail(Q35_ERR_UNSUPPORTED, "%s: batch %d of %d heads", who, g.batch, g.q_heads);
    if (g.rotary_dim < 0 || g.rotary_dim > 256 || (g.rotary_dim & 1))
        return q35::fail(Q35_ERR_ARG, "%s: rotary_dim %d", who, g.rotary_dim);
    if (g.capacity < 1 || g.capacity > INT32_MAX / 2)
        return q35::fail(Q35_ERR_RANGE, "%s: caches of %lld rows", who, static_cast<long long>(g.capacity));
    q35k::AttnQ4Args a{};
    a.B = g.batch;
    a.NQ = g.q_heads;
    a.NKV = g.kv_heads;
    a.GRP = g.q_heads / g.kv_heads;
    a.ROT = g.rotary_dim;
    a.cap = g.capacity;
    *out = a;
    return Q35_OK;
}

q35_status kv_q4(const q35_kv_q4_args* args, bool store, q35_stream s, const char* who) {
    if (!args) return q35::fail(Q35_ERR_ARG, "%s: null args", who);
    const q35_kv_q4_args& g = *args;
    if (g.head_dim != 256) return q35::fail(Q35_ERR_UNSUPPORTED, "%s: head_dim must be 256", who);
    if (g.batch <= 0 || g.kv_heads <= 0) return q35::fail(Q35_ERR_ARG, "%s: bad batch or head count", who);
    if (g.batch > 65535 || g.kv_heads > 65535 || static_cast<int64_t>(g.batch) * g.kv_heads > 1 << 24)
        return q35::fail(Q35_ERR_UNSUPPORTED, "%s: batch %d of %d heads", who, g.batch, g.kv_heads);
    if (g.kv_dtype != 0 && g.kv_dtype != 1) return q35::fail(Q35_ERR_ARG, "%s: kv_dtype %d", who, g.kv_dtype);
    if (g.shared_rows != 0 && (g.shared_rows != 1 || !store))
        return q35::fail(Q35_ERR_ARG, "%s: shared_rows %d", who, g.shared_rows);
    if (g.capacity < 1 || g.capacity > INT32_MAX / 2 || g.rows_capacity < 1 || g.rows_capacity > INT32_MAX / 2)
        return q35::fail(Q35_ERR_RANGE, "%s: caches of %lld and %lld rows", who, static_cast<long long>(g.rows_capacity),
                         static_cast<long long>(g.capacity));
    if (!g.end || !g.k_rows || !g.v_rows || !g.k || !g.v || !g.k_scale || !g.v_scale)
        return q35::fail(Q35_ERR_ARG, "%s: null pointer", who);
    if (!aligned(g.k_rows, 16) || !aligned(g.v_rows, 16) || !aligned(g.k, 16) || !aligned(g.v, 16) || !aligned(g.k_scale, 16) ||
        !aligned(g.v_scale, 16))
        return q35::fail(Q35_ERR_ARG, "%s: caches must be 16-byte aligned", who);
    const uint64_t heads = static_cast<uint64_t>(g.batch) * g.kv_heads, n = heads * g.capacity;
    const uint64_t wide = (g.shared_rows ? g.kv_heads : heads) * g.rows_capacity * 256 * (g.kv_dtype ? 2 : 4);
    const uint64_t batch = g.batch * 4ull;
    const Part part[] = {{g.k_rows, wide, !store}, {g.v_rows, wide, !store}, {g.k, n * 128, store}, {g.v, n * 128, store},
                         {g.k_scale, n * 16, store}, {g.v_scale, n * 16, store}, {g.begin, g.begin ? batch : 0, false}, {g.end, batch, false}};
    if (written_overlaps(part)) return q35::fail(Q35_ERR_ARG, "%s: an output overlaps another array", who);
    const q35_status st = check_stream(static_cast<hipStream_t>(s), who);
    if (st != Q35_OK) return st;
    q35k::KvQ4Args a{};
    a.B = g.batch;
    a.NKV = g.kv_heads;
    a.bf16 = g.kv_dtype == 1;
    a.shared = g.shared_rows == 1;
    a.rows_cap = g.rows_capacity;
    a.cap = g.capacity;
    a.begin = g.begin;
    a.end = g.end;
    a.k_rows = g.k_rows;
    a.v_rows = g.v_rows;
    a.k = g.k;
    a.v = g.v;
    a.k_scale = static_cast<uint32_t*>(g.k_scale);
    a.v_scale = static_cast<uint32_t*>(g.v_scale);
    return launched(q35k::launch_kv_q4(a, store, static_cast<hipStream_t>(s)), who);
}

}  // namespace

extern "C" {

uint64_t q35_q4_packed_bytes(int32_t N, int32_t K, int32_t group, int32_t has_zeros) {
    if (q4_sizes(N, K, group, "q35_q4_packed_bytes") != Q35_OK) return 0;
    return static_cast<uint64_t>(q35k::q4_tiles(N)) * q35k::q4_blocks(K) * q35k::q4_unit_bytes(group, has_zeros != 0);
}

q35_status q35_q4_quantize(const void *W, int32_t w_dtype, int32_t N, int32_t K, int32_t group, uint8_t *codes, uint16_t *scales,
                           uint8_t *zeros, q35_stream s) {
    const char* who = "q35_q4_quantize";
    q35_status st = q4_sizes(N, K, group, who);
    if (st != Q35_OK) return st;
    if (w_dtype != 0 && w_dtype != 1) return q35::fail(Q35_ERR_ARG, "%s: w_dtype %d", who, w_dtype);
    if (!W || !codes || !scales) return q35::fail(Q35_ERR_ARG, "%s: null pointer", who);
    if (!aligned(W, w_dtype ? 2 : 4) || !aligned(scales, 2)) return q35::fail(Q35_ERR_ARG, "%s: unaligned pointer", who);
    const uint64_t groups = static_cast<uint64_t>(N) * ((K + group - 1) / group);
    const struct { const void* p; uint64_t n; } part[] = {{W, static_cast<uint64_t>(N) * K * (w_dtype ? 2 : 4)},
                                                          {codes, static_cast<uint64_t>(N) * ((K + 1) / 2)},
                                                          {scales, groups * 2}, {zeros, zeros ? groups : 0}};
    for (int i = 0; i < 4; ++i)
        for (int j = i + 1; j < 4; ++j)
            if (overlap(part[i].p, part[i].n, part[j].p, part[j].n)) return q35::fail(Q35_ERR_ARG, "%s: arrays overlap", who);
    st = check_stream(static_cast<hipStream_t>(s), who);
    if (st != Q35_OK) return st;
    return launched(q35k::launch_q4_quantize(W, w_dtype == 1, N, K, group, codes, scales, zeros, static_cast<hipStream_t>(s)), who);
}

q35_status q35_q4_pack(const uint8_t *codes, const uint16_t *scales, const uint8_t *zeros, int32_t N, int32_t K, int32_t group,
                       void *packed, q35_stream s) {
    const char* who = "q35_q4_pack";
    q35_status st = q4_sizes(N, K, group, who);
    if (st != Q35_OK) return st;
    if (!codes || !scales || !packed) return q35::fail(Q35_ERR_ARG, "%s: null pointer", who);
    if (!aligned(packed, 16) || !aligned(scales, 2)) return q35::fail(Q35_ERR_ARG, "%s: packed must be 16-byte aligned", who);
    const uint64_t groups = static_cast<uint64_t>(N) * ((K + group - 1) / group), out = q35_q4_packed_bytes(N, K, group, zeros != nullptr);
    if (overlap(packed, out, codes, static_cast<uint64_t>(N) * ((K + 1) / 2)) || overlap(packed, out, scales, groups * 2) ||
        overlap(packed, out, zeros, zeros ? groups : 0))
        return q35::fail(Q35_ERR_ARG, "%s: packed overlaps an input", who);
    st = check_stream(static_cast<hipStream_t>(s), who);
    if (st != Q35_OK) return st;
    return launched(q35k::launch_q4_pack(codes, scales, zeros, N, K, group, static_cast<uint8_t*>(packed), static_cast<hipStream_t>(s)),
                    who);
}

uint64_t q35_matmul_q4_workspace_bytes(int32_t M, int32_t N, int32_t K, int32_t group) {
    const char* who = "q35_matmul_q4_workspace_bytes";
    if (q4_sizes(N, K, group, who) != Q35_OK) return 0;
    if (M < 1 || M > Q35_MATMUL_Q4_MOST_ROWS) {
        q35::fail(Q35_ERR_UNSUPPORTED, "%s: %d rows", who, M);
        return 0;
    }
    return kMulWorkspace;
}

q35_status q35_matmul_q4(const float *X, int64_t ldx, const void *packed, int32_t has_zeros, int32_t M, int32_t N, int32_t K,
                         int32_t group, const float *R, int64_t ldr, float *Y, int64_t ldy, void *workspace,
                         uint64_t workspace_bytes, q35_stream s) {
    const char* who = "q35_matmul_q4";
    q35_status st = q4_sizes(N, K, group, who);
    if (st != Q35_OK) return st;
    if (M < 1) return q35::fail(Q35_ERR_ARG, "%s: %d rows", who, M);
    if (M > Q35_MATMUL_Q4_MOST_ROWS) return q35::fail(Q35_ERR_UNSUPPORTED, "%s: %d rows", who, M);
    if (has_zeros != 0 && has_zeros != 1) return q35::fail(Q35_ERR_ARG, "%s: has_zeros %d", who, has_zeros);
    if (!X || !packed || !Y || !workspace) return q35::fail(Q35_ERR_ARG, "%s: null pointer", who);
    constexpr int64_t kMost = 1ll << 40;  // elements: offsets stay within 64 bits
    if (ldx < K || ldy < N || (R && ldr < N) || ldx > kMost || ldy > kMost || (R && ldr > kMost))
        return q35::fail(Q35_ERR_ARG, "%s: bad leading dimension", who);
    if (!aligned(packed, 16) || !aligned(workspace, 16) || !aligned(X, 4) || !aligned(Y, 4) || !aligned(R, 4))
        return q35::fail(Q35_ERR_ARG, "%s: packed and workspace must be 16-byte aligned", who);
    const auto span = [](int64_t ld, int64_t rows, int64_t n) { return static_cast<uint64_t>(ld * (rows - 1) + n) * 4; };
    if (overlap(Y, span(ldy, M, N), X, span(ldx, M, K)) || overlap(Y, span(ldy, M, N), packed, q35_q4_packed_bytes(N, K, group, has_zeros)) ||
        (R && !(R == Y && ldr == ldy) && overlap(Y, span(ldy, M, N), R, span(ldr, M, N))))
        return q35::fail(Q35_ERR_ARG, "%s: Y overlaps an input (R may be Y itself)", who);
    if (workspace_bytes < kMulWorkspace)
        return q35::fail(Q35_ERR_ARG, "%s: workspace of %llu bytes, needs %llu", who,
                         static_cast<unsigned long long>(workspace_bytes), static_cast<unsigned long long>(kMulWorkspace));
    st = check_stream(static_cast<hipStream_t>(s), who);
    if (st != Q35_OK) return st;
    q35k::Q4MulArgs a{};
    a.X = X;
    a.W = static_cast<const uint8_t*>(packed);
    a.R = R;
    a.Y = Y;
    a.ldx = ldx;
    a.ldr = ldr;
    a.ldy = ldy;
    a.M = M;
    a.N = N;
    a.K = K;
    a.G = group;
    a.zeros = has_zeros != 0;
    return launched(q35k::launch_q4_mul(a, static_cast<hipStream_t>(s)), who);
}

uint64_t q35_attn_q4_workspace_bytes(const q35_attn_q4_args *args) {
    q35k::AttnQ4Args a{};
    if (attn_q4_sizes(args, "q35_attn_q4_workspace_bytes", &a) != Q35_OK) return 0;
    return static_cast<uint64_t>(q35k::attn_q4_workspace_floats(a)) * 4;
}

q35_status q35_attn_q4(const q35_attn_q4_args *args, q35_stream s) {
    const char* who = "q35_attn_q4";
    q35k::AttnQ4Args a{};
    q35_status st = attn_q4_sizes(args, who, &a);
    if (st != Q35_OK) return st;
    const q35_attn_q4_args& g = *args;
    if (!g.len || !g.pos || !g.qg || !g.k_new || !g.v_new || !g.q_norm || !g.k_norm || !g.k || !g.v || !g.k_scale || !g.v_scale ||
        !g.out || !g.workspace)
        return q35::fail(Q35_ERR_ARG, "%s: null pointer", who);
    for (const void* p : {static_cast<const void*>(g.qg), static_cast<const void*>(g.k_new), static_cast<const void*>(g.v_new),
                          static_cast<const void*>(g.q_norm), static_cast<const void*>(g.k_norm), static_cast<const void*>(g.k),
                          static_cast<const void*>(g.v), static_cast<const void*>(g.k_scale), static_cast<const void*>(g.v_scale),
                          static_cast<const void*>(g.out), static_cast<const void*>(g.workspace)})
        if (!aligned(p, 16)) return q35::fail(Q35_ERR_ARG, "%s: rows, caches and workspace must be 16-byte aligned", who);
    const uint64_t n = static_cast<uint64_t>(g.batch) * g.kv_heads * g.capacity;
    const uint64_t need = static_cast<uint64_t>(q35k::attn_q4_workspace_floats(a)) * 4;
    const uint64_t batch = g.batch * 4ull, row = 256 * batch;
    const Part part[] = {{g.k, n * 128, true}, {g.v, n * 128, true}, {g.k_scale, n * 16, true}, {g.v_scale, n * 16, true},
                         {g.out, row * g.q_heads, true}, {g.workspace, need, true}, {g.qg, row * g.q_heads * 2, false},
                         {g.k_new, row * g.kv_heads, false}, {g.v_new, row * g.kv_heads, false}, {g.q_norm, 1024, false},
                         {g.k_norm, 1024, false}, {g.len, batch, false}, {g.pos, batch, false}};
    if (written_overlaps(part)) return q35::fail(Q35_ERR_ARG, "%s: an output overlaps another array", who);
    if (g.workspace_bytes < need)
        return q35::fail(Q35_ERR_ARG, "%s: workspace of %llu bytes, needs %llu", who,
                         static_cast<unsigned long long>(g.workspace_bytes), static_cast<unsigned long long>(need));
    st = check_stream(static_cast<hipStream_t>(s), who);
    if (st != Q35_OK) return st;
    a.theta = g.rope_theta;
    a.eps = g.eps;
    a.len = g.len;
    a.pos = g.pos;
    a.qg = g.qg;
    a.k_new = g.k_new;
    a.v_new = g.v_new;
    a.q_norm = g.q_norm;
    a.k_norm = g.k_norm;
    a.k = g.k;
    a.v = g.v;
    a.k_scale = static_cast<uint32_t*>(g.k_scale);
    a.v_scale = static_cast<uint32_t*>(g.v_scale);
    a.out = g.out;
    a.ws = static_cast<float*>(g.workspace);
    return launched(q35k::launch_attn_q4(a, static_cast<hipStream_t>(s)), who);
}

q35_status q35_kv_q4_store(const q35_kv_q4_args *args, q35_stream s) { return kv_q4(args, true, s, "q35_kv_q4_store"); }
q35_status q35_kv_q4_load(const q35_kv_q4_args *args, q35_stream s) { return kv_q4(args, false, s, "q35_kv_q4_load"); }

static q35_status sample_sizes(const q35_sample_args *args, const char *who) {
    if (!args) return q35::fail(Q35_ERR_ARG, "%s: null args", who);
    if (args->batch <= 0 || args->vocab <= 0) return q35::fail(Q35_ERR_ARG, "%s: %d rows of %d logits", who, args->batch, args->vocab);
    if (args->batch > 65535 || args->vocab > 1 << 22)
        return q35::fail(Q35_ERR_UNSUPPORTED, "%s: %d rows of %d logits", who, args->batch, args->vocab);
    return Q35_OK;
}

uint64_t q35_sample_workspace_bytes(const q35_sample_args *args) {
    if (sample_sizes(args, "q35_sample_workspace_bytes") != Q35_OK) return 0;
    return q35k::sample_workspace_bytes(args->batch, args->vocab);
}

q35_status q35_sample(const q35_sample_args *args, q35_stream s) {
    const char* who = "q35_sample";
    q35_status st = sample_sizes(args, who);
    if (st != Q35_OK) return st;
    const q35_sample_args& g = *args;
    if (g.ld_logits < g.vocab || g.ld_logits > 1ll << 40) return q35::fail(Q35_ERR_ARG, "%s: bad leading dimension", who);
    if (!g.logits || !g.temperature || !g.u || !g.token || !g.workspace) return q35::fail(Q35_ERR_ARG, "%s: null pointer", who);
    if (!aligned(g.workspace, 16) || !aligned(g.logits, 4)) return q35::fail(Q35_ERR_ARG, "%s: workspace must be 16-byte aligned", who);
    const uint64_t need = q35k::sample_workspace_bytes(g.batch, g.vocab);
    if (g.workspace_bytes < need)
        return q35::fail(Q35_ERR_ARG, "%s: workspace of %llu bytes, needs %llu", who,
                         static_cast<unsigned long long>(g.workspace_bytes), static_cast<unsigned long long>(need));
    const uint64_t batch = g.batch * 4ull;
    const auto settings = [&](const void* p) { return Part{p, p ? batch : 0, false}; };
    const Part part[] = {{g.logits, static_cast<uint64_t>((g.batch - 1) * g.ld_logits + g.vocab) * 4, false}, settings(g.temperature),
                         settings(g.top_k), settings(g.top_p), settings(g.min_p), settings(g.u), {g.token, batch, true},
                         {g.prob, g.prob ? batch : 0, true}, {g.workspace, need, true}};
    if (written_overlaps(part)) return q35::fail(Q35_ERR_ARG, "%s: an output overlaps another array", who);
    st = check_stream(static_cast<hipStream_t>(s), who);
    if (st != Q35_OK) return st;
    q35k::SampleArgs a{};
    a.B = g.batch;
    a.V = g.vocab;
    a.ld = g.ld_logits;
    a.logits = g.logits;
    a.temperature = g.temperature;
    a.top_k = g.top_k;
    a.top_p = g.top_p;
    a.min_p = g.min_p;
    a.u = g.u;
    a.token = g.token;
    a.prob = g.prob;
    a.ws = g.workspace;
    return launched(q35k::launch_sample(a, static_cast<hipStream_t>(s)), who);
}

}  // extern "C"
