// C ABI of the operators for a batch of continuations (q35_attn_batch, q35_kv_evict,
// q35_gdn_batch): sizes and pointers are checked here, lengths that only the device knows are
// bounded in the kernels.
#include <hip/hip_runtime.h>

#include "../host/q35_internal.h"
#include "launch.hpp"

namespace {

q35_status launched(hipError_t e, const char* what) {
    return e == hipSuccess ? Q35_OK : q35::fail(Q35_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}

bool a16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// [p, p + n) and [q, q + m) share a byte
bool overlap(const void* p, uint64_t n, const void* q, uint64_t m) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(p), y = reinterpret_cast<uintptr_t>(q);
    return x < y + m && y < x + n;
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

constexpr int64_t kMostRows = 1 << 24;  // batch x query heads, batch x kv heads

// Sizes of q35_attn_batch (what its workspace depends on).
q35_status attn_batch_sizes(const q35_attn_batch_args* args, const char* who, q35k::AttnBatchArgs* out) {
    if (!args) return q35::fail(Q35_ERR_ARG, "%s: null args", who);
    const q35_attn_batch_args& g = *args;
    if (g.head_dim != 256) return q35::fail(Q35_ERR_UNSUPPORTED, "%s: head_dim must be 256", who);
    if (g.batch <= 0 || g.q_heads <= 0 || g.kv_heads <= 0 || g.q_heads % g.kv_heads != 0)
        return q35::fail(Q35_ERR_ARG, "%s: bad batch or head counts", who);
    if (g.q_heads / g.kv_heads > 16) return q35::fail(Q35_ERR_UNSUPPORTED, "%s: GQA group %d", who, g.q_heads / g.kv_heads);
    if (static_cast<int64_t>(g.batch) * g.q_heads > kMostRows || g.batch > 65535 || g.q_heads > 4096)
        return q35::fail(Q35_ERR_UNSUPPORTED, "%s: batch %d of %d heads", who, g.batch, g.q_heads);
    if (g.rotary_dim < 0 || g.rotary_dim > 256 || (g.rotary_dim & 1))
        return q35::fail(Q35_ERR_ARG, "%s: rotary_dim %d", who, g.rotary_dim);
    if (g.kv_dtype != 0 && g.kv_dtype != 1) return q35::fail(Q35_ERR_ARG, "%s: kv_dtype %d", who, g.kv_dtype);
    if (g.prefix_len < 0 || g.prefix_len > g.prefix_capacity || g.own_capacity < 1 || g.prefix_capacity > INT32_MAX / 2 ||
        g.own_capacity > INT32_MAX / 2)
        return q35::fail(Q35_ERR_RANGE, "%s: prefix of %lld rows in %lld, own caches of %lld", who,
                         static_cast<long long>(g.prefix_len), static_cast<long long>(g.prefix_capacity),
                         static_cast<long long>(g.own_capacity));
    if (g.own_score && (g.own_capacity + 511) / 512 * g.batch * g.kv_heads + static_cast<int64_t>(g.batch) * g.q_heads > INT32_MAX)
        return q35::fail(Q35_ERR_UNSUPPORTED, "%s: scores of %d caches of %lld rows", who, g.batch * g.kv_heads,
                         static_cast<long long>(g.own_capacity));
    q35k::AttnBatchArgs a{};
    a.B = g.batch;
    a.NQ = g.q_heads;
    a.NKV = g.kv_heads;
    a.GRP = g.q_heads / g.kv_heads;
    a.ROT = g.rotary_dim;
    a.kv_bf16 = g.kv_dtype == 1;
    a.P = g.prefix_len;
    a.prefix_cap = g.prefix_capacity;
    a.cap = g.own_capacity;
    a.own_score = g.own_score;
    *out = a;
    return Q35_OK;
}

q35_status evict_sizes(const q35_kv_evict_args* args, const char* who) {
    if (!args) return q35::fail(Q35_ERR_ARG, "%s: null args", who);
    const q35_kv_evict_args& g = *args;
    if (g.head_dim != 256) return q35::fail(Q35_ERR_UNSUPPORTED, "%s: head_dim must be 256", who);
    if (g.batch <= 0 || g.kv_heads <= 0) return q35::fail(Q35_ERR_ARG, "%s: bad batch or head count", who);
    if (g.batch > 65535 || g.kv_heads > 65535 || static_cast<int64_t>(g.batch) * g.kv_heads > kMostRows)
        return q35::fail(Q35_ERR_UNSUPPORTED, "%s: batch %d of %d heads", who, g.batch, g.kv_heads);
    if (g.kv_dtype != 0 && g.kv_dtype != 1) return q35::fail(Q35_ERR_ARG, "%s: kv_dtype %d", who, g.kv_dtype);
    if (g.capacity < 1 || g.capacity > INT32_MAX / 2)
        return q35::fail(Q35_ERR_RANGE, "%s: capacity %lld", who, static_cast<long long>(g.capacity));
    if (g.keep < 1 || g.n_sink < 0 || g.n_recent < 0 || static_cast<int64_t>(g.n_sink) + g.n_recent > g.keep)
        return q35::fail(Q35_ERR_ARG, "%s: keep %d with %d first and %d recent rows", who, g.keep, g.n_sink, g.n_recent);
    return Q35_OK;
}

}  // namespace

extern "C" {

uint64_t q35_attn_batch_workspace_bytes(const q35_attn_batch_args* args) {
    q35k::AttnBatchArgs a{};
    if (attn_batch_sizes(args, "q35_attn_batch_workspace_bytes", &a) != Q35_OK) return 0;
    return static_cast<uint64_t>(q35k::attn_batch_workspace_floats(a)) * 4;
}

q35_status q35_attn_batch(const q35_attn_batch_args* args, q35_stream s) {
    const char* who = "q35_attn_batch";
    q35k::AttnBatchArgs a{};
    q35_status st = attn_batch_sizes(args, who, &a);
    if (st != Q35_OK) return st;
    const q35_attn_batch_args& g = *args;
    if (!q35k::attn_batch_launches(a))
        return q35::fail(Q35_ERR_UNSUPPORTED, "%s: batch %d of %d / %d heads is more than one launch holds", who, g.batch,
                         g.q_heads, g.kv_heads);
    if (!g.own_len || !g.pos || !g.qg || !g.k_new || !g.v_new || !g.q_norm || !g.k_norm || !g.k_own || !g.v_own ||
        !g.out || !g.workspace || (g.prefix_len > 0 && (!g.k_prefix || !g.v_prefix)))
        return q35::fail(Q35_ERR_ARG, "%s: null pointer", who);
    if (!a16(g.qg) || !a16(g.k_new) || !a16(g.v_new) || !a16(g.q_norm) || !a16(g.k_norm) || !a16(g.k_own) ||
        !a16(g.v_own) || !a16(g.out) || !a16(g.workspace) || (g.prefix_len > 0 && (!a16(g.k_prefix) || !a16(g.v_prefix))))
        return q35::fail(Q35_ERR_ARG, "%s: rows, caches and workspace must be 16-byte aligned", who);
    const uint64_t need = static_cast<uint64_t>(q35k::attn_batch_workspace_floats(a)) * 4;
    if (g.workspace_bytes < need)
        return q35::fail(Q35_ERR_ARG, "%s: workspace of %llu bytes, needs %llu", who,
                         static_cast<unsigned long long>(g.workspace_bytes), static_cast<unsigned long long>(need));
    st = check_stream(static_cast<hipStream_t>(s), who);
    if (st != Q35_OK) return st;
    a.theta = g.rope_theta;
    a.eps = g.eps;
    a.own_len = g.own_len;
    a.pos = g.pos;
    a.qg = g.qg;
    a.k_new = g.k_new;
    a.v_new = g.v_new;
    a.q_norm = g.q_norm;
    a.k_norm = g.k_norm;
    a.k_prefix = g.k_prefix;
    a.v_prefix = g.v_prefix;
    a.k_own = g.k_own;
    a.v_own = g.v_own;
    a.own_pos = g.own_pos;
    a.out = g.out;
    q35k::attn_batch_carve(a, static_cast<float*>(g.workspace));
    return launched(q35k::launch_attn_batch(a, static_cast<hipStream_t>(s)), who);
}

uint64_t q35_kv_evict_workspace_bytes(const q35_kv_evict_args* args) {
    if (evict_sizes(args, "q35_kv_evict_workspace_bytes") != Q35_OK) return 0;
    return static_cast<uint64_t>(q35k::kv_evict_workspace_ints(args->batch, args->kv_heads, args->capacity, args->keep)) * 4;
}

q35_status q35_kv_evict(const q35_kv_evict_args* args, q35_stream s) {
    const char* who = "q35_kv_evict";
    q35_status st = evict_sizes(args, who);
    if (st != Q35_OK) return st;
    const q35_kv_evict_args& g = *args;
    if (!g.len || !g.next_pos || !g.score || !g.pos || !g.k || !g.v || !g.score_out || !g.pos_out || !g.new_len ||
        !g.workspace)
        return q35::fail(Q35_ERR_ARG, "%s: null pointer", who);
    if (!a16(g.k) || !a16(g.v) || !a16(g.workspace))
        return q35::fail(Q35_ERR_ARG, "%s: caches and workspace must be 16-byte aligned", who);
    const uint64_t rows = static_cast<uint64_t>(g.batch) * g.kv_heads * g.capacity;
    if ((g.score_out != g.score && overlap(g.score_out, rows * 4, g.score, rows * 4)) ||
        (g.pos_out != g.pos && overlap(g.pos_out, rows * 4, g.pos, rows * 4)) ||
        (g.new_len != g.len && overlap(g.new_len, g.batch * 4ull, g.len, g.batch * 4ull)) ||
        overlap(g.k, rows * 256 * (g.kv_dtype ? 2 : 4), g.v, rows * 256 * (g.kv_dtype ? 2 : 4)))
        return q35::fail(Q35_ERR_ARG, "%s: an output overlaps another array", who);
    const uint64_t need = q35_kv_evict_workspace_bytes(args);
    if (g.workspace_bytes < need)
        return q35::fail(Q35_ERR_ARG, "%s: workspace of %llu bytes, needs %llu", who,
                         static_cast<unsigned long long>(g.workspace_bytes), static_cast<unsigned long long>(need));
    st = check_stream(static_cast<hipStream_t>(s), who);
    if (st != Q35_OK) return st;
    q35k::KvEvictArgs a{};
    a.B = g.batch;
    a.NKV = g.kv_heads;
    a.kv_bf16 = g.kv_dtype == 1;
    a.keep = g.keep;
    a.n_sink = g.n_sink;
    a.n_recent = g.n_recent;
    a.cap = g.capacity;
    a.len = g.len;
    a.next_pos = g.next_pos;
    a.score = g.score;
    a.pos = g.pos;
    a.k = g.k;
    a.v = g.v;
    a.score_out = g.score_out;
    a.pos_out = g.pos_out;
    a.new_len = g.new_len;
    q35k::kv_evict_carve(a, static_cast<int*>(g.workspace));
    return launched(q35k::launch_kv_evict(a, static_cast<hipStream_t>(s)), who);
}

q35_status q35_gdn_batch(const q35_gdn_batch_args* args, q35_stream s) {
    const char* who = "q35_gdn_batch";
    if (!args) return q35::fail(Q35_ERR_ARG, "%s: null args", who);
    const q35_gdn_batch_args& g = *args;
    if (g.head_dim_k != 128 || g.head_dim_v != 128 || g.conv_kernel != 4)
        return q35::fail(Q35_ERR_UNSUPPORTED, "%s: needs DK == DV == 128 and conv kernel 4", who);
    if (g.batch <= 0 || g.rows <= 0 || g.k_heads <= 0 || g.v_heads <= 0 || g.v_heads % g.k_heads != 0)
        return q35::fail(Q35_ERR_ARG, "%s: bad batch, row or head counts", who);
    if (g.batch > 65535 || g.v_heads > 4096 || g.k_heads > 4096)
        return q35::fail(Q35_ERR_UNSUPPORTED, "%s: batch %d of %d heads", who, g.batch, g.v_heads);
    if (!g.row0 && g.rows < g.batch)
        return q35::fail(Q35_ERR_ARG, "%s: %d rows for %d sequences of one token", who, g.rows, g.batch);
    if (!g.pos || !g.qkv || !g.b || !g.a || !g.conv_w || !g.A_log || !g.dt_bias || !g.conv_ring || !g.state || !g.out)
        return q35::fail(Q35_ERR_ARG, "%s: null pointer", who);
    if (g.norm_w && !g.z) return q35::fail(Q35_ERR_ARG, "%s: the gated norm needs z", who);
    if (!g.conv_ring_in != !g.state_in) return q35::fail(Q35_ERR_ARG, "%s: conv_ring_in and state_in come together", who);
    const int64_t conv = (2LL * g.k_heads + g.v_heads) * 128, ring = 4 * conv, state = g.v_heads * 16384LL;
    if (g.ld_qkv < conv || (g.norm_w && g.ld_z < g.v_heads * 128LL) || g.ld_ba < g.v_heads)
        return q35::fail(Q35_ERR_ARG, "%s: leading dimension too small", who);
    if (g.stride_ring < ring || g.stride_state < state || (g.state_in && g.stride_state_in != 0 && g.stride_state_in < state) ||
        (g.state_in && g.stride_ring_in != 0 && g.stride_ring_in < ring))
        return q35::fail(Q35_ERR_ARG, "%s: sequences' rings or states overlap", who);
    if (!a16(g.conv_w) || !a16(g.conv_ring) || !a16(g.state) || !a16(g.conv_ring_in) || !a16(g.state_in) ||
        g.stride_state % 4 != 0 || g.stride_state_in % 4 != 0)
        return q35::fail(Q35_ERR_ARG, "%s: conv_w, rings and states must be 16-byte aligned, the states' strides multiples of 4", who);
    const auto span = [&](int64_t stride, int64_t one) { return static_cast<uint64_t>(stride * (g.batch - 1) + one) * 4; };
    if (g.state_in && (overlap(g.state_in, span(g.stride_state_in, state), g.state, span(g.stride_state, state)) ||
                       overlap(g.conv_ring_in, span(g.stride_ring_in, ring), g.conv_ring, span(g.stride_ring, ring))))
        return q35::fail(Q35_ERR_ARG, "%s: the rings or states read overlap the ones written (NULL: in place)", who);
    const q35_status st = check_stream(static_cast<hipStream_t>(s), who);
    if (st != Q35_OK) return st;
    q35k::GdnBatchArgs a{};
    a.B = g.batch;
    a.rows = g.rows;
    a.KH = g.k_heads;
    a.VH = g.v_heads;
    a.eps = g.eps;
    a.row0 = g.row0;
    a.pos = g.pos;
    a.qkv = g.qkv;
    a.z = g.z;
    a.b = g.b;
    a.a = g.a;
    a.ld_qkv = g.ld_qkv;
    a.ld_z = g.ld_z;
    a.ld_ba = g.ld_ba;
    a.conv_w = g.conv_w;
    a.A_log = g.A_log;
    a.dt_bias = g.dt_bias;
    a.norm_w = g.norm_w;
    a.ring_in = g.state_in ? g.conv_ring_in : g.conv_ring;
    a.state_in = g.state_in ? g.state_in : g.state;
    a.s_ring_in = g.state_in ? g.stride_ring_in : g.stride_ring;
    a.s_state_in = g.state_in ? g.stride_state_in : g.stride_state;
    a.ring = g.conv_ring;
    a.state = g.state;
    a.s_ring = g.stride_ring;
    a.s_state = g.stride_state;
    a.out = g.out;
    return launched(q35k::launch_gdn_batch(a, static_cast<hipStream_t>(s)), who);
}

}  // extern "C"
