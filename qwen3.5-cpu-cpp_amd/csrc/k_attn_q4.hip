// Attention over caches of 4-bit rows (q35_attn_q4), and such rows from and to fp32 or bf16 caches
// (q35_kv_q4_store, q35_kv_q4_load). The layout of a row is in launch_q4.hpp.
//
// A row is quantized by 64 dims: least = fp16(min), step = fp16((max - least) / 15), code =
// round((x - least) / step), all from 64-bit values rounded to fp32 and then fp16: a value next to the
// border of two codes is on the same side for whoever computes it from the same inputs.
#include <cmath>

#include "dev_q4.hpp"
#include "launch_q4.hpp"

namespace q35k {
namespace {

constexpr int kHD = 256;

// fp16 through fp32: without the barrier the two roundings are compiled as one
__device__ __forceinline__ uint32_t bits_half(double x) {
    float f = static_cast<float>(x);
    asm("" : "+v"(f));
    return q35k::bits_half(f);
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
// Over the 16 lanes of a row; all of them are there, so that a move becomes part of the instruction that uses it.
template <int CTRL>
__device__ __forceinline__ int row_i(int x) { return __builtin_amdgcn_mov_dpp(x, CTRL, 0xF, 0xF, true); }
template <int CTRL>
__device__ __forceinline__ float row_f(float x) { return __builtin_bit_cast(float, row_i<CTRL>(__builtin_bit_cast(int, x))); }
__device__ __forceinline__ int max16(int v) {
    v = max(v, row_i<0xB1>(v));
    v = max(v, row_i<0x4E>(v));
    v = max(v, row_i<0x141>(v));
    return max(v, row_i<0x140>(v));
}
// of values that are not negative (a NaN is above all)
__device__ __forceinline__ float max16_abs(float v) { return __builtin_bit_cast(float, max16(__builtin_bit_cast(int, v))); }
// by bits in the values' order, as fmaxf takes an instruction more a step
__device__ __forceinline__ float max16(float v) {
    const auto order = [](int b) { return b ^ (b >> 31 & 0x7fffffff); };
    return __builtin_bit_cast(float, order(max16(order(__builtin_bit_cast(int, v)))));
}
__device__ __forceinline__ int sum16(int v) {
    v += row_i<0xB1>(v);
    v += row_i<0x4E>(v);
    v += row_i<0x141>(v);
    return v + row_i<0x140>(v);
}
__device__ __forceinline__ float sum16(float v) {
    v += row_f<0xB1>(v);
    v += row_f<0x4E>(v);
    v += row_f<0x141>(v);
    return v + row_f<0x140>(v);
}
__device__ __forceinline__ float exp2_f(float x) { return __builtin_amdgcn_exp2f(x); }
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

// The same of a row of fp32 values, in fp32 where that decides it: a quotient is off by less than 2^-22 of itself, so
// one that is further than 2^-16 from the middle between two codes, and a step further than 16 of its last places from
// the middle between two of fp16, falls to the same side in 64 bits. A row in some 40 takes the way above instead.
__device__ __forceinline__ uint32_t quantize4(const float* x, uint32_t& scale) {
    const float lo = -max16(fmaxf(fmaxf(-x[0], -x[1]), fmaxf(-x[2], -x[3]))), hi = max16(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])));
    const uint32_t lb = q35k::bits_half(lo);
    const float least = half_bits(lb), d = (hi - least) * (1.0f / 15.0f);
    const uint32_t db = __float_as_uint(d), off = (db & 0x1fffu) - 0x0ff0u;
    bool sure = d > 6.2e-5f && d < 4000.0f && off > 0x20u;
#pragma unroll
    for (int i = 0; i < 4; ++i) sure &= fabsf(x[i]) < 60000.0f;
    const uint32_t sb = q35k::bits_half(d);
    const float inv = __builtin_amdgcn_rcpf(half_bits(sb));
    scale = sb | lb << 16;
    uint32_t c = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float q = (x[i] - least) * inv, r = rintf(q);
        sure &= fabsf(fabsf(q - r) - 0.5f) > 0x1p-16f;
        c |= static_cast<uint32_t>(fminf(fmaxf(r, 0.0f), 15.0f)) << (4 * i);
    }
    if (__all(sure)) return c;
    const double y[4] = {x[0], x[1], x[2], x[3]};
    return quantize4(y, scale);
}

// theta^(-2i / ROT), formed on the host
struct RopeFreq {
    double f[kHD / 2];
};

// What lanes of a wave have written to LDS is there for its other lanes.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}
// What the products read of a query head lies in LDS: the three digits of its row, by quads of heads: [quad][group
// of 64 dims][c][head of the quad][digit] 16 bytes, the dims 16 c .. + 15 of the group in the order in which a
// cache row's nibbles come apart (0 2 4 6 1 3 5 7 8 10 ..); and per head and group (2^-e, which is the row's, and the
// sum of the group's multiples, which the rows' least values are multiplied by).
constexpr int kQuadBytes = 4 * 4 * 4 * 3 * 16;

// A wave norms a row (lane l: dims 4 l .. + 3) and rotates it by the angles in cs (cosines, then sines from 128 on),
// through 2 KB of LDS of its own.
__device__ __forceinline__ void norm_rotate(double* x, const float4& w, float eps, int rot, const double* cs, double* row) {
    const int lane = threadIdx.x & 63, half = rot / 2;
    const double ss = wave_sum(x[0] * x[0] + x[1] * x[1] + x[2] * x[2] + x[3] * x[3]);
    const double inv = 1.0 / sqrt(ss / kHD + static_cast<double>(eps));
    x[0] *= inv * (1.0 + w.x), x[1] *= inv * (1.0 + w.y), x[2] *= inv * (1.0 + w.z), x[3] *= inv * (1.0 + w.w);
#pragma unroll
    for (int i = 0; i < 4; ++i) row[4 * lane + i] = x[i];
    wave_sync();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int d = 4 * lane + i;
        if (d < half) x[i] = x[i] * cs[d] - row[d + half] * cs[128 + d];
        else if (d < rot) x[i] = x[i] * cs[d - half] + row[d - half] * cs[128 + d - half];
    }
    wave_sync();
}

// A normed, rotated query row, times log2(e) / sqrt(HD), as digits: head h of the kv head's. One unit serves the row (a unit
// for each 64 dims took 1.5% more of a batch's time): an entry is off by 2^-23 of the largest of all 256.
__device__ __forceinline__ void place_query(const double* x, int h, uint8_t* qbuf, float2* fbuf) {
    const int lane = threadIdx.x & 63;
    constexpr double kScale = 0.0625 * 1.4426950408889634;
    float f[4];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[i] = static_cast<float>(x[i] * kScale);
        top = max(top, __float_as_uint(f[i]) & 0x7fffffffu);
    }
    top = static_cast<uint32_t>(max16(static_cast<int>(top)));
    const auto row_top = [&](int l) { return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(top), l)); };
    top = max(max(row_top(0), row_top(16)), max(row_top(32), row_top(48)));
    const bool ok = top < 0x7f800000u && top != 0;
    const int e = ok ? multiple_exp(__uint_as_float(top)) : 0;
    int sum = 0;
    uint32_t y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int v = ok ? static_cast<int>(rintf(ldexpf(f[i], e))) : 0;
        sum += v;
        y[i] = signed_digits(v);
    }
    sum = sum16(sum);
    const int g = lane >> 4, c = lane >> 2 & 3, o = lane & 3;
    uint8_t* at = qbuf + (h / 4) * kQuadBytes + ((g * 4 + c) * 4 + h % 4) * 48 + (o >> 1) * 8 + (o & 1) * 2;
#pragma unroll
    for (int p = 0; p < 3; ++p) {  // dims 4 o, 4 o + 2 and 4 o + 1, 4 o + 3 of the sixteen
        *reinterpret_cast<uint16_t*>(at + 16 * p) = static_cast<uint16_t>((y[0] >> (8 * p) & 0xffu) | (y[2] >> (8 * p) & 0xffu) << 8);
        *reinterpret_cast<uint16_t*>(at + 16 * p + 4) = static_cast<uint16_t>((y[1] >> (8 * p) & 0xffu) | (y[3] >> (8 * p) & 0xffu) << 8);
    }
    if ((lane & 15) == 0) {
        const float s = top >= 0x7f800000u ? NAN : ldexpf(1.0f, -e);
        fbuf[h * 4 + g] = make_float2(s, static_cast<float>(sum));
    }
}

// sixteen codes of two words as bytes: the even nibbles of each, then the odd ones
__device__ __forceinline__ v4i bytes_of(v2i w) {
    return v4i{w[0] & 0x0f0f0f0f, static_cast<int>(static_cast<uint32_t>(w[0]) >> 4 & 0x0f0f0f0fu), w[1] & 0x0f0f0f0f,
               static_cast<int>(static_cast<uint32_t>(w[1]) >> 4 & 0x0f0f0f0fu)};
}
// 16 times sixteen signed codes
__device__ __forceinline__ v4i bytes_of_signed(v2i w) {
    constexpr int kHigh = static_cast<int>(0xf0f0f0f0u);
    return v4i{w[0] << 4 & kHigh, w[0] & kHigh, w[1] << 4 & kHigh, w[1] & kHigh};
}

constexpr int kTile = 64;       // keys a wave takes at a time
constexpr int kVBytes = kTile * kQ4RowBytes, kPBytes = 4 * 4 * 4 * 3 * 16, kFreshBytes = kQ4RowBytes + 16;

// A workgroup's share: a piece of one head's rows.
struct Share {
    int b, head, piece, pieces, first;  // of `pieces` of that head, the first one's workgroup being `first`
    int rounds;                         // of tiles for all waves, a piece
};
constexpr int kMostShared = 512;        // sequences and workgroups up to which rows are shared out

// The batch's rows shared out among `groups` workgroups: pieces of as many rounds as are needed for all to have
// one, so that long sequences get many and none waits for another's. Every wave finds the same.
__device__ __forceinline__ Share share_out(const AttnQ4Args& a, int groups, int w, int waves) {
    constexpr int kEach = kMostShared / 64;
    if (a.B == 1) {                     // the same without the sums (1 x 700 14.3 us, with them 15.3; 1 x 131072 30.3 and 32.0)
        const int len = a.len[0], all = len < 0 ? 0 : len < a.cap ? len / (waves * kTile) + 1 : 1, per = static_cast<uint32_t>(groups) / a.NKV;
        const int r = max(static_cast<int>((static_cast<uint32_t>(all) + per - 1) / per), 1), np = (static_cast<uint32_t>(all) + r - 1) / r;
        if (w >= np * a.NKV) return {-1, 0, 0, 0, 0, r};
        const int head = static_cast<uint32_t>(w) / np;
        return {0, head, w - head * np, np, head * np, r};
    }
    const int lane = threadIdx.x & 63, round = waves * kTile, blocks = (a.B + 63) / 64;
    int rounds[kEach], total = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int b = i * 64 + lane, len = i < blocks && b < a.B ? a.len[b] : -1;
        rounds[i] = len < 0 ? 0 : len < a.cap ? len / round + 1 : 1;  // one to say that nothing was appended
        total += rounds[i];
    }
    const auto sum = [](int v) { return static_cast<int>(lane_of(wave_scan(static_cast<uint32_t>(v)), 63)); };
    // whole rounds of all heads stay below 2^31: rows of a cache below 2^30, of a batch below 2^39 / 256
    int r = max((sum(total) + groups / a.NKV - 1) / (groups / a.NKV), 1);
    const auto pieces_of = [&](int i) { return (rounds[i] + r - 1) / r; };
    for (;;) {
        int n = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            if (i < blocks) n += pieces_of(i);
        if (sum(n) * a.NKV <= groups) break;
        r += max(r / 8, 1);             // ends: with r the longest, every head has one
    }
    Share s{-1, 0, 0, 0, 0, r};
    int before = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        if (i >= blocks || s.b >= 0) break;
        const int n = pieces_of(i) * a.NKV, upto = before + static_cast<int>(wave_scan(static_cast<uint32_t>(n)));
        const uint64_t mine = __ballot(w < upto);
        if (mine) {
            const int l = __ffsll(static_cast<unsigned long long>(mine)) - 1;
            const int np = __builtin_amdgcn_readlane(n, l) / a.NKV, start = __builtin_amdgcn_readlane(upto, l) - np * a.NKV;
            s.b = i * 64 + l;
            s.head = (w - start) / np;
            s.piece = (w - start) % np;
            s.pieces = np;
            s.first = start + s.head * np;
        }
        before = __builtin_amdgcn_readlane(upto, 63);
    }
    return s;
}

struct Partials {
    float* o;                           // [workgroups][GRP][HD]
    float2* ml;                         // [workgroups][GRP] (max, sum)
    int2* where;                        // [B][NKV] first workgroup, workgroups
};

// Four waves (or eight) a piece of one cache's keys, tiles of 64 keys a wave, for all query heads of the kv head.
//
// Scores: a 16 x 16 x 64 integer product takes four heads as four times three digits (the fourth row is never
// looked at) and 16 keys over a group of 64 dims; lane 16 c + n then holds head c's three sums for key n, and
//   s = 2^-e sum_g (step_g sum_d i_d code_d + least_g sum_d i_d).
// Weights: p = 2^(s - tile's largest) <= 1 is multiplied by its value row's step, which differs by group, and becomes
// multiples of a 4190000th of the tile's largest such product (of one below 1e-30, 0): p step (code - 8) summed over 64
// keys is again one integer product, heads and digits by 16 dims. A lane's four weights (of keys n, n + 16, ..) are one word of that
// operand, so P's order of keys is theirs, and value rows are read transposed (16 x 16 nibbles at a time) in that
// order. The rest, sum_t p_t (least_t + 8 step_t), is a sum a head and group. (By code - 8 both are means of values of
// both signs: of 131072 rows the outputs are 6e-7 off, by code and least 3.2e-6.)
//
// The matrix cores do the products in passing; what a tile costs is some 1200 instructions around them (5k cycles of
// a wave), and what a call costs is mostly that workgroups are short: 1 x 131072 (16/2 heads), 73 MB, takes 30 us, of
// which 24 are this kernel's: 1 to share the rows out, 3 to request what it reads, 4 for its queries, 12 for two tiles
// a wave, 2 to join the waves. 40 sequences of up to 8192, 94 MB, take 41 us; 1 x 700 (8/2 heads) 14.3. (Figures here and
// below: calls replayed from a graph, over three sets of inputs, all of one run.)
template <int HQ, int kWaves>
__global__ __launch_bounds__(kWaves * 64, HQ > 2 || kWaves > 4 ? 1 : 2) void attn_q4_kernel(AttnQ4Args a, RopeFreq freq, int shared, Partials part) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane >> 4, n = lane & 15;
    // every head whole, or the rows shared out
    Share share{static_cast<int>(blockIdx.x) / a.NKV, static_cast<int>(blockIdx.x) % a.NKV, 0, 1, static_cast<int>(blockIdx.x), 0};
    if (shared) share = share_out(a, shared, blockIdx.x, kWaves);
    if (share.b < 0) return;            // no share left
    const int b = share.b, hk = share.head, len = a.len[b];
    if (len < 0) return;
    if (len >= a.cap) {  // nothing was appended
        for (int i = threadIdx.x; i < a.GRP * kHD; i += kWaves * 64) a.out[(static_cast<int64_t>(b) * a.NQ + hk * a.GRP) * kHD + i] = NAN;
        if (shared && threadIdx.x == 0) part.where[b * a.NKV + hk] = make_int2(0, 1);
        return;
    }
    const int rows = len + 1, piece_len = share.rounds * kWaves * kTile, first = share.piece * piece_len;
    const int end = share.piece + 1 == share.pieces ? rows : first + piece_len;
    const int64_t bk = static_cast<int64_t>(b) * a.NKV + hk;
    const bool fresh = end == rows;     // the new row is this piece's
    // the piece's rows; offsets within it stay within 32 bits
    const int count = end - first;
    const int64_t row0 = bk * a.cap + first;
    const uint8_t *K = a.k + row0 * kQ4RowBytes, *V = a.v + row0 * kQ4RowBytes;
    const uint8_t *KS = reinterpret_cast<const uint8_t*>(a.k_scale) + row0 * 16, *VS = reinterpret_cast<const uint8_t*>(a.v_scale) + row0 * 16;

    // the queries, for all waves, the angles, and each wave's value rows and weights
    constexpr int JB = HQ < 2 ? HQ : 2;  // quads whose weights lie in LDS at a time
    uint8_t* qbuf = lds;
    float2* fbuf = reinterpret_cast<float2*>(lds + HQ * kQuadBytes);
    double* cs = reinterpret_cast<double*>(lds + HQ * (kQuadBytes + 128));
    uint8_t* fresh_row = lds + HQ * (kQuadBytes + 128) + 2048;  // K's and V's: the codes and the steps
    uint8_t* vbuf = fresh_row + 2 * kFreshBytes + wave * (kVBytes + JB * kPBytes);
    uint8_t* pbuf = vbuf + kVBytes;

    // A tile's keys, key and value steps, and value rows: whole tiles by constant places of a lane, the last one's
    // missing rows as copies of the last row (their scores are masked).
    v2i k[4][4];
    v4i ks[4], vs[4], v[8];
    const auto load_k = [&](int t0) {
        const uint8_t *kt = K + static_cast<int64_t>(t0) * kQ4RowBytes, *st = KS + static_cast<int64_t>(t0) * 16;
        const bool whole = t0 + kTile <= count;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const uint32_t r = whole ? 16 * t + n : min(16 * t + n, count - 1 - t0);
#pragma unroll
            for (int g = 0; g < 4; ++g) k[t][g] = *reinterpret_cast<const v2i*>(kt + (r * kQ4RowBytes + 8 * c) + 32 * g);
            ks[t] = *reinterpret_cast<const v4i*>(st + r * 16);
        }
    };
    const auto load_v = [&](int t0) {
        const uint8_t* vt = V + static_cast<int64_t>(t0) * kQ4RowBytes;
        const bool whole = t0 + kTile <= count;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t r = whole ? 8 * i + (lane >> 3) : min(8 * i + (lane >> 3), count - 1 - t0);
            v[i] = *reinterpret_cast<const v4i*>(vt + (r * kQ4RowBytes + 16 * (lane & 7)));
        }
    };
    // a row's eight 16-byte pieces lie in LDS in an order that spreads the rows over the banks; its codes as code - 8
    const auto place_v = [&] {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            *reinterpret_cast<v4i*>(vbuf + (8 * i + (lane >> 3)) * kQ4RowBytes + 16 * ((lane & 7) ^ (lane >> 3))) = v[i] ^ static_cast<int>(0x88888888u);
    };
    const auto load_vs = [&](int t0) {
        const uint8_t* st = VS + static_cast<int64_t>(t0) * 16;
        const bool whole = t0 + kTile <= count;
#pragma unroll
        for (int t = 0; t < 4; ++t)
            vs[t] = *reinterpret_cast<const v4i*>(st + static_cast<uint32_t>(whole ? 16 * t + n : min(16 * t + n, count - 1 - t0)) * 16);
    };

    float m[HQ], l[HQ], lo[HQ][4], o[HQ][16];
#pragma unroll
    for (int j = 0; j < HQ; ++j) {
        m[j] = -INFINITY;
        l[j] = 0.0f;
#pragma unroll
        for (int g = 0; g < 4; ++g) lo[j][g] = 0.0f;
#pragma unroll
        for (int d = 0; d < 16; ++d) o[j][d] = 0.0f;
    }

    // nibble n of the transposed 16 keys: which key its place in the operand is
    const int spot = (n & 8) + (n & 1) * 4 + ((n & 7) >> 1), key = 16 * (spot & 3) + 4 * c + (spot >> 2);
    int t0 = wave * kTile;
    constexpr int kHeads = (4 * HQ + kWaves - 1) / kWaves;  // query heads a wave makes
    float4 qx[kHeads];
    const float4 qw = reinterpret_cast<const float4*>(a.q_norm)[lane];
#pragma unroll
    for (int i = 0; i < kHeads; ++i)
        qx[i] = reinterpret_cast<const float4*>(a.qg + (static_cast<int64_t>(b) * a.NQ + hk * a.GRP + min(wave + i * kWaves, a.GRP - 1)) * 2 * kHD)[lane];
    const int angle = min(static_cast<int>(threadIdx.x), kHD / 2 - 1);
    const double f = freq.f[angle];
    const int pos = a.pos[b];
    __builtin_amdgcn_sched_barrier(0);  // loads come back in order: what is used first is asked for first
    if (t0 < count) {                   // on its way while the queries are made
        load_k(t0);
        load_v(t0);
        load_vs(t0);
    }
    __builtin_amdgcn_sched_barrier(0);
    if (static_cast<int>(threadIdx.x) < a.ROT / 2) sincos(static_cast<double>(pos) * f, &cs[128 + angle], &cs[angle]);
    lds_barrier();
    double* row = reinterpret_cast<double*>(vbuf);  // before the values are there
    if (fresh) {
        if (wave >= kWaves - 2) {
            const bool is_k = wave == kWaves - 2;
            const float4 f = reinterpret_cast<const float4*>((is_k ? a.k_new : a.v_new) + bk * kHD)[lane];
            double x[4] = {f.x, f.y, f.z, f.w};
            if (is_k) norm_rotate(x, reinterpret_cast<const float4*>(a.k_norm)[lane], a.eps, a.ROT, cs, row);
            uint32_t scale;
            const uint32_t code = quantize4(x, scale);
            const int64_t at = bk * a.cap + len;
            uint8_t* row = fresh_row + (is_k ? 0 : kFreshBytes);
            reinterpret_cast<uint16_t*>(row)[lane] = static_cast<uint16_t>(code);
            reinterpret_cast<uint16_t*>(is_k ? a.k : a.v)[at * 64 + lane] = static_cast<uint16_t>(code);
            if (n == 0) {
                reinterpret_cast<uint32_t*>(row + kQ4RowBytes)[c] = scale;
                (is_k ? a.k_scale : a.v_scale)[at * 4 + c] = scale;
            }
        }
    }
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
        if (wave + i * kWaves >= a.GRP) break;
        double x[4] = {qx[i].x, qx[i].y, qx[i].z, qx[i].w};
        norm_rotate(x, qw, a.eps, a.ROT, cs, row);
        place_query(x, wave + i * kWaves, qbuf, fbuf);
    }
    lds_barrier();
    for (; t0 < count; t0 += kWaves * kTile) {
        if (fresh && t0 + kTile >= count) {  // the new row, and its copies, from LDS: in the cache it may not be yet
            const int last = count - 1 - t0;
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                if (16 * t + n < last) continue;
#pragma unroll
                for (int g = 0; g < 4; ++g) k[t][g] = *reinterpret_cast<const v2i*>(fresh_row + 8 * c + 32 * g);
                ks[t] = *reinterpret_cast<const v4i*>(fresh_row + kQ4RowBytes);
                vs[t] = *reinterpret_cast<const v4i*>(fresh_row + kFreshBytes + kQ4RowBytes);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (8 * i + (lane >> 3) >= last) v[i] = *reinterpret_cast<const v4i*>(fresh_row + kFreshBytes + 16 * (lane & 7));
        }
        float s[HQ][4];
#pragma unroll
        for (int j = 0; j < HQ; ++j)
#pragma unroll
            for (int t = 0; t < 4; ++t) s[j][t] = 0.0f;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            v4i q[HQ];
            float f[HQ];
#pragma unroll
            for (int j = 0; j < HQ; ++j) {
                q[j] = *reinterpret_cast<const v4i*>(qbuf + j * kQuadBytes + ((g * 4 + c) * 4 + (n >> 2)) * 48 + min(n & 3, 2) * 16);
                f[j] = fbuf[(j * 4 + c) * 4 + g].y;
            }
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const v4i kb = bytes_of(k[t][g]);
                const uint32_t sc = ks[t][g];
                const float step = step_of(sc), least = least_of(sc);
#pragma unroll
                for (int j = 0; j < HQ; ++j) {
                    const v4i d = __builtin_amdgcn_mfma_i32_16x16x64_i8(q[j], kb, v4i{0, 0, 0, 0}, 0, 0, 0);
                    s[j][t] = fmaf(from_digits(d), step, fmaf(least, f[j], s[j][t]));
                    if constexpr (HQ > 2) pin(s[j][t]);
                }
            }
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int j = 0; j < HQ; ++j) pin(s[j][t]);
        }
#pragma unroll
        for (int j = 0; j < HQ; ++j) {
            const float unit = fbuf[(j * 4 + c) * 4].x;
#pragma unroll
            for (int t = 0; t < 4; ++t) s[j][t] *= unit;
        }
        const int next = t0 + kWaves * kTile;
        place_v();
        if (next < count) {
            load_k(next);
            load_v(next);
        }
        float alpha[HQ], beta[HQ];
#pragma unroll
        for (int j = 0; j < HQ; ++j) {
            if (t0 + kTile > count) {
#pragma unroll
                for (int t = 0; t < 4; ++t) s[j][t] = t0 + 16 * t + n < count ? s[j][t] : -INFINITY;
            }
            const float top = max16(fmaxf(fmaxf(s[j][0], s[j][1]), fmaxf(s[j][2], s[j][3])));
            const float ref = top == -INFINITY ? 0.0f : top, mn = fmaxf(m[j], top), mref = mn == -INFINITY ? 0.0f : mn;
            alpha[j] = exp2_f(m[j] - mref);
            beta[j] = exp2_f(top - mref);
            m[j] = mn;
#pragma unroll
            for (int t = 0; t < 4; ++t) s[j][t] = exp2_f(s[j][t] - ref);
            l[j] = fmaf(l[j], alpha[j], beta[j] * ((s[j][0] + s[j][1]) + (s[j][2] + s[j][3])));
        }
#pragma unroll
        for (int j0 = 0; j0 < HQ; j0 += JB) {
            // weights times steps, in units of the tile's largest such product: digits through LDS into the
            // operand's order
            float unit[JB][4];
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                float st[4], le[4];
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    st[t] = step_of(vs[t][g]);
                    le[t] = fmaf(st[t], 8.0f, least_of(vs[t][g]));
                }
#pragma unroll
                for (int j = j0; j < j0 + JB; ++j) {
                    float x[4], part_lo = 0.0f;
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        x[t] = s[j][t] * st[t];
                        part_lo = fmaf(s[j][t], le[t], part_lo);
                    }
                    lo[j][g] = fmaf(lo[j][g], alpha[j], beta[j] * part_lo);
                    const float big = max16_abs(fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3]))));
                    const float inv = big > 1e-30f ? 4190000.0f * __builtin_amdgcn_rcpf(big) : 0.0f;
                    unit[j - j0][g] = beta[j] * big * (0.0625f / 4190000.0f);
                    uint32_t y[4];
#pragma unroll
                    for (int t = 0; t < 4; ++t)  // 1.5 2^23 + i: i in the low bits
                        y[t] = (__float_as_uint(fmaf(x[t], inv, 12582912.0f)) + (0x8080u - 0x4b400000u)) ^ 0x8080u;
                    uint8_t* at = pbuf + (j - j0) * kPBytes + (g * 4 + (n >> 2)) * 192 + c * 48 + 4 * (n & 3);
                    // bytes 0 and 1 of two words each, then of all four
                    const uint32_t a01 = __builtin_amdgcn_perm(y[1], y[0], 0x05010400u), a23 = __builtin_amdgcn_perm(y[3], y[2], 0x05010400u);
                    *reinterpret_cast<uint32_t*>(at) = __builtin_amdgcn_perm(a23, a01, 0x05040100u);
                    *reinterpret_cast<uint32_t*>(at + 16) = __builtin_amdgcn_perm(a23, a01, 0x07060302u);
                    *reinterpret_cast<uint32_t*>(at + 32) = plane<2>(y[0], y[1], y[2], y[3]);
                    pin(lo[j][g]);
                    pin(unit[j - j0][g]);
                }
            }
            if (j0 + JB >= HQ && next < count) load_vs(next);
#pragma unroll
            for (int j = j0; j < j0 + JB; ++j)
                if (__any(alpha[j] != 1.0f)) {
#pragma unroll
                    for (int d = 0; d < 16; ++d) o[j][d] *= alpha[j];
                }
            wave_sync();
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                v4i p[JB];
#pragma unroll
                for (int j = 0; j < JB; ++j)
                    p[j] = *reinterpret_cast<const v4i*>(pbuf + j * kPBytes + (g * 4 + c) * 192 + (n >> 2) * 48 + min(n & 3, 2) * 16);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int d = 4 * g + i;  // dims 16 d .. + 15
                    const v2i w = __builtin_amdgcn_ds_read_tr4_b64_v2i32(reinterpret_cast<__attribute__((address_space(3))) v2i*>(
                        reinterpret_cast<uintptr_t>(vbuf + key * kQ4RowBytes + 16 * ((d >> 1) ^ (key & 7)) + 8 * (d & 1))));
                    const v4i vb = bytes_of_signed(w);
#pragma unroll
                    for (int j = 0; j < JB; ++j) {
                        o[j0 + j][d] = fmaf(from_digits(__builtin_amdgcn_mfma_i32_16x16x64_i8(p[j], vb, v4i{0, 0, 0, 0}, 0, 0, 0)),
                                            unit[j][g], o[j0 + j][d]);
                        if constexpr (HQ > 2) pin(o[j0 + j][d]);
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < JB; ++j) pin(o[j0 + j][4 * g + i]);
            }
            wave_sync();
        }
    }
    if (shared && share.piece == 0 && threadIdx.x == 0) part.where[bk] = make_int2(share.first, share.pieces);
    // The waves' parts: each scaled to the largest maximum of all, then added.
    __syncthreads();
    float2* wml = reinterpret_cast<float2*>(lds);
    float* wo = reinterpret_cast<float*>(lds + kWaves * HQ * 4 * 8);
#pragma unroll
    for (int j = 0; j < HQ; ++j) {
        l[j] = sum16(l[j]);
        if (n == 0) wml[wave * HQ * 4 + 4 * j + c] = make_float2(m[j], l[j]);
#pragma unroll
        for (int g = 0; g < 4; ++g) lo[j][g] = sum16(lo[j][g]);
    }
    lds_barrier();
#pragma unroll
    for (int j = 0; j < HQ; ++j) {
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) top = fmaxf(top, wml[w * HQ * 4 + 4 * j + c].x);
        const float f = exp2_f(m[j] - (top == -INFINITY ? 0.0f : top));
#pragma unroll
        for (int d = 0; d < 16; ++d) wo[((wave * HQ + j) * 4 + c) * kHD + 16 * d + n] = f * (o[j][d] + lo[j][d / 4]);
    }
    lds_barrier();
    for (int i = threadIdx.x; i < a.GRP * (kHD / 4); i += kWaves * 64) {
        const int h = i / (kHD / 4), d = i % (kHD / 4);
        v4f x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) x += reinterpret_cast<const v4f*>(wo + (w * HQ * 4 + h) * kHD)[d];
        float m_all = -INFINITY, l_all = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) m_all = fmaxf(m_all, wml[w * HQ * 4 + h].x);
        const float ref = m_all == -INFINITY ? 0.0f : m_all;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) l_all = fmaf(exp2_f(wml[w * HQ * 4 + h].x - ref), wml[w * HQ * 4 + h].y, l_all);
        if (share.pieces == 1) {        // all there is
            const int64_t at = static_cast<int64_t>(b) * a.NQ + hk * a.GRP + h;
            const v4f g = reinterpret_cast<const v4f*>(a.qg + at * 2 * kHD + kHD)[d];
            reinterpret_cast<v4f*>(a.out + at * kHD)[d] = v4f{x[0] / l_all * sigmoid_f(g[0]), x[1] / l_all * sigmoid_f(g[1]),
                                                              x[2] / l_all * sigmoid_f(g[2]), x[3] / l_all * sigmoid_f(g[3])};
        } else {
            const int64_t at = static_cast<int64_t>(blockIdx.x) * a.GRP + h;
            reinterpret_cast<v4f*>(part.o + at * kHD)[d] = x;
            if (d == 0) part.ml[at] = make_float2(m_all, l_all);
        }
    }
}

// The pieces' parts of a query head, and the gate: four workgroups a head, 64 dims each, in which sixteen threads take
// four dims each of every kSlots-th piece.
template <int kSlots>
__global__ __launch_bounds__(16 * kSlots) void attn_q4_combine_kernel(AttnQ4Args a, Partials part) {
    __shared__ v4f ws[kSlots][16];
    __shared__ float2 wml[kSlots];
    const int d = threadIdx.x & 15, s = threadIdx.x >> 4, h = blockIdx.x >> 2, quarter = blockIdx.x & 3, b = blockIdx.y, hk = h / a.GRP;
    // asked for together (an empty place's may be anything)
    const int len = a.len[b];
    const int2 where = part.where[static_cast<int64_t>(b) * a.NKV + hk];
    const int64_t o = static_cast<int64_t>(b) * a.NQ + h;
    const v4f g = reinterpret_cast<const v4f*>(a.qg + o * 2 * kHD + kHD)[quarter * 16 + d];
    const int np = where.y;
    if (len < 0 || np == 1) return;     // one: written by its workgroup
    const int64_t first = static_cast<int64_t>(where.x) * a.GRP + h % a.GRP;
    float m = -INFINITY, l = 0.0f;
    v4f x = {0.0f, 0.0f, 0.0f, 0.0f};
    constexpr int kBatch = 8;           // requested together
    for (int i0 = s; i0 < np; i0 += kSlots * kBatch) {
        float2 ml[kBatch];
        v4f v[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const int64_t at = first + static_cast<int64_t>(min(i0 + kSlots * k, np - 1)) * a.GRP;
            ml[k] = part.ml[at];
            v[k] = reinterpret_cast<const v4f*>(part.o + at * kHD)[quarter * 16 + d];
        }
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            if (i0 + kSlots * k >= np) break;
            const float mn = fmaxf(m, ml[k].x), ref = mn == -INFINITY ? 0.0f : mn, f = exp2_f(m - ref), e = exp2_f(ml[k].x - ref);
            m = mn;
            l = l * f + ml[k].y * e;
            x = x * f + v[k] * e;
        }
    }
    ws[s][d] = x;
    if (d == 0) wml[s] = make_float2(m, l);
    __syncthreads();
    if (s) return;
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < kSlots; ++i) top = fmaxf(top, wml[i].x);
    top = top == -INFINITY ? 0.0f : top;
    l = 0.0f;
    x = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < kSlots; ++i) {
        const float f = exp2_f(wml[i].x - top);
        l = fmaf(wml[i].y, f, l);
        x += ws[i][d] * f;
    }
    reinterpret_cast<v4f*>(a.out + o * kHD)[quarter * 16 + d] =
        v4f{x[0] / l * sigmoid_f(g[0]), x[1] / l * sigmoid_f(g[1]), x[2] / l * sigmoid_f(g[2]), x[3] / l * sigmoid_f(g[3])};
}

// whether rows [i, e) of sequence b are there
__device__ __forceinline__ bool range_of(const KvQ4Args& a, int b, int& i, int& e) {
    i = a.begin ? a.begin[b] : 0;
    e = a.end[b];
    return i >= 0 && e > i && e <= a.cap && e <= a.rows_cap;
}

// A wave takes kKvRows rows of K or of V at a time, requested together; blockIdx.y = 2 (b NKV + h) + (0: K, 1: V).
// Bound by memory: 8192 fp32 rows of two heads, 38 MB, take 9.7 us (4.0 TB/s; by single rows with divisions in 64 bits
// 15.2); reading five caches of up to 4099 rows back as bf16 8.2 us (before 10.3).
constexpr int kKvRows = 4;
template <bool BF16>
__global__ __launch_bounds__(256) void kv_q4_store_kernel(KvQ4Args a) {
    const int lane = threadIdx.x & 63;
    for (int64_t id = blockIdx.y; id < 2ll * a.B * a.NKV; id += gridDim.y) {
        const int b = static_cast<int>(id / 2 / a.NKV), h = static_cast<int>(id / 2 % a.NKV), v = static_cast<int>(id & 1);
        int i, e;
        if (!range_of(a, b, i, e)) continue;
        const void* rows = v ? a.v_rows : a.k_rows;
        const int64_t from = (static_cast<int64_t>(a.shared ? 0 : b) * a.NKV + h) * a.rows_cap, to = (id / 2) * a.cap;
        for (int64_t t = i + (blockIdx.x * 4 + threadIdx.x / 64) * kKvRows; t < e; t += gridDim.x * 4 * kKvRows) {
            v4f x[kKvRows];
#pragma unroll
            for (int r = 0; r < kKvRows; ++r) {
                const int64_t at = (from + min(t + r, static_cast<int64_t>(e - 1))) * 64 + lane;
                if constexpr (BF16) {
                    const uint2 u = static_cast<const uint2*>(rows)[at];
                    x[r] = v4f{bf16_lo(u.x), bf16_hi(u.x), bf16_lo(u.y), bf16_hi(u.y)};
                } else {
                    x[r] = static_cast<const v4f*>(rows)[at];
                }
            }
#pragma unroll
            for (int r = 0; r < kKvRows; ++r) {
                if (t + r >= e) break;
                const float f[4] = {x[r][0], x[r][1], x[r][2], x[r][3]};
                uint32_t sc;
                const uint32_t c = quantize4(f, sc);
                reinterpret_cast<uint16_t*>(v ? a.v : a.k)[(to + t + r) * 64 + lane] = static_cast<uint16_t>(c);
                if ((lane & 15) == 0) (v ? a.v_scale : a.k_scale)[(to + t + r) * 4 + lane / 16] = sc;
            }
        }
    }
}

// A lane writes 16 bytes: 4 values of a row of fp32, 8 of one of the two rows of bf16 that a wave takes together.
template <bool BF16>
__global__ __launch_bounds__(256) void kv_q4_load_kernel(KvQ4Args a) {
    constexpr int kLanes = BF16 ? 32 : 64, kEach = kHD / kLanes, kTogether = 64 / kLanes, kTake = kKvRows * kTogether;
    const int lane = threadIdx.x & (kLanes - 1), which = (threadIdx.x & 63) / kLanes;
    for (int64_t id = blockIdx.y; id < 2ll * a.B * a.NKV; id += gridDim.y) {
        const int b = static_cast<int>(id / 2 / a.NKV), h = static_cast<int>(id / 2 % a.NKV), v = static_cast<int>(id & 1);
        int i, e;
        if (!range_of(a, b, i, e)) continue;
        const int64_t to = (static_cast<int64_t>(b) * a.NKV + h) * a.rows_cap, from = (id / 2) * a.cap;
        for (int64_t t = i + (blockIdx.x * 4 + threadIdx.x / 64) * kTake; t < e; t += gridDim.x * 4 * kTake) {
            uint32_t code[kKvRows], sc[kKvRows];
#pragma unroll
            for (int r = 0; r < kKvRows; ++r) {
                const int64_t at = from + min(t + r * kTogether + which, static_cast<int64_t>(e - 1));
                if constexpr (BF16) code[r] = reinterpret_cast<const uint32_t*>(v ? a.v : a.k)[at * 32 + lane];
                else code[r] = reinterpret_cast<const uint16_t*>(v ? a.v : a.k)[at * 64 + lane];
                sc[r] = (v ? a.v_scale : a.k_scale)[at * 4 + lane / (kLanes / 4)];
            }
#pragma unroll
            for (int r = 0; r < kKvRows; ++r) {
                if (t + r * kTogether + which >= e) break;
                const float step = step_of(sc[r]), least = least_of(sc[r]);
                float f[kEach];
#pragma unroll
                for (int j = 0; j < kEach; ++j) f[j] = fmaf(step, static_cast<float>(code[r] >> (4 * j) & 15u), least);
                v4i w;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if constexpr (BF16) {
                        const float x = f[2 * j], y = f[2 * j + 1];
                        w[j] = static_cast<int>((x == x ? f32_to_bf16(x) : 0x7fc0u) | (y == y ? f32_to_bf16(y) : 0x7fc0u) << 16);
                    } else {
                        w[j] = __builtin_bit_cast(int, f[j]);
                    }
                }
                static_cast<v4i*>(v ? a.v_rows : a.k_rows)[(to + t + r * kTogether + which) * kLanes + lane] = w;
            }
        }
    }
}

}  // namespace

namespace {

struct AttnQ4Plan {
    int quads, waves, groups, shared;
};
AttnQ4Plan attn_q4_plan(const AttnQ4Args& a) {
    AttnQ4Plan p{};
    p.quads = a.GRP <= 4 ? 1 : a.GRP <= 8 ? 2 : 4;
    p.waves = 4;
    const int64_t heads = static_cast<int64_t>(a.B) * a.NKV;
    p.groups = static_cast<int>(heads);
    // A workgroup a head. (Of 512 heads and more, and by the few pieces left of nearly as many, a sequence that is far longer than
    // the others takes its own time: 255 x 16/2 of up to 2000 rows, one of 131072, 981 us, 256 1880, where one alone takes 30.)
    if (heads >= kMostShared || a.cap <= 4 * kTile) return p;
    const bool eight = p.quads <= 2;    // their registers allow it
    // A workgroup a head of eight waves where that is one tile a wave (1 x 300, 8/2 heads 11.4 us, rows shared out 13.4;
    // 40 x 512, 16/2 17.7 and 21.3; 1 x 1024, 8/2 18.8 and 14.7), or two and heads are many (90 x 1024, 16/2 25.7 and
    // 34.6; 40 x up to 1024 24.4 and 21.5).
    if (eight && (a.cap <= 8 * kTile || (a.cap <= 16 * kTile && heads >= 128))) {
        p.waves = 8;
        return p;
    }
    // Else rows are shared out: eight waves a compute unit, or as many workgroups as there can be rounds. Two
    // workgroups of four waves, or one of eight, half as many to be merged, where sequences are few and one round of
    // all of them may not do (1 x 131072, 16/2 30.9 us, by fours 31.5; 20 x up to 8192 29.8 and 31.2; 1 x 16384 19.7 and
    // 18.2; 40 x up to 8192 44.1 and 41.0).
    if (eight && heads <= 40 && heads * a.cap >= kMostShared * 4 * kTile) p.waves = 8;
    const int64_t each = p.waves * kTile, most = kMostShared * 4 / p.waves;  // most >= heads: every head has a workgroup
    p.groups = p.shared = static_cast<int>(std::min<int64_t>(most / a.NKV, a.B * ((a.cap + each - 1) / each)) * a.NKV);
    return p;
}

template <int HQ, int kWaves>
hipError_t launch_attend(const AttnQ4Args& a, const RopeFreq& freq, const AttnQ4Plan& p, const Partials& part, hipStream_t s) {
    const uint32_t lds = std::max(HQ * (kQuadBytes + 128) + 2048 + 2 * kFreshBytes + kWaves * (kVBytes + std::min(HQ, 2) * kPBytes), kWaves * HQ * 4 * (kHD * 4 + 8));
    static AllowedLds allowed;
    hipError_t e = allowed(reinterpret_cast<const void*>(attn_q4_kernel<HQ, kWaves>), static_cast<int>(lds));
    if (e != hipSuccess) return e;
    klaunch(attn_q4_kernel<HQ, kWaves>, dim3(p.groups), dim3(kWaves * 64), lds, s, a, freq, p.shared, part);
    e = hipGetLastError();
    if (e != hipSuccess || !p.shared) return e;
    // Workgroups of 512 threads where there is at most one for a compute unit (256 pieces of 16 heads 30.9 us in all, with
    // 256 threads 31.9; three pieces of 8 heads 14.3 and 13.8), else of 256 (40 sequences 42.0, with 512 46.0).
    const dim3 grid(a.NQ * 4, a.B);
    if (static_cast<int64_t>(a.NQ) * 4 * a.B <= 256) klaunch(attn_q4_combine_kernel<32>, grid, dim3(512), 0, s, a, part);
    else klaunch(attn_q4_combine_kernel<16>, grid, dim3(256), 0, s, a, part);
    return hipGetLastError();
}

}  // namespace

int64_t attn_q4_workspace_floats(const AttnQ4Args& a) {
    const AttnQ4Plan p = attn_q4_plan(a);
    return p.shared ? static_cast<int64_t>(p.groups) * a.GRP * (kHD + 2) + 2ll * a.B * a.NKV : 64;
}

hipError_t launch_attn_q4(const AttnQ4Args& a, hipStream_t s) {
    const AttnQ4Plan p = attn_q4_plan(a);
    RopeFreq freq{};
    for (int i = 0; i < a.ROT / 2; ++i) freq.f[i] = std::pow(a.theta, -static_cast<double>(2 * i) / a.ROT);
    Partials part;
    part.o = a.ws;
    part.ml = reinterpret_cast<float2*>(a.ws + static_cast<int64_t>(p.groups) * a.GRP * kHD);
    part.where = reinterpret_cast<int2*>(part.ml + static_cast<int64_t>(p.groups) * a.GRP);
    if (p.waves == 8) return p.quads == 1 ? launch_attend<1, 8>(a, freq, p, part, s) : launch_attend<2, 8>(a, freq, p, part, s);
    return p.quads == 1   ? launch_attend<1, 4>(a, freq, p, part, s)
           : p.quads == 2 ? launch_attend<2, 4>(a, freq, p, part, s)
                          : launch_attend<4, 4>(a, freq, p, part, s);
}

hipError_t launch_kv_q4(const KvQ4Args& a, bool store, hipStream_t s) {
    const int64_t n = std::min(a.cap, a.rows_cap), y = std::min<int64_t>(2ll * a.B * a.NKV, 32768), each = 4 * kKvRows * (a.bf16 && !store ? 2 : 1);
    const dim3 grid(static_cast<uint32_t>(std::min<int64_t>((n + each - 1) / each, std::max<int64_t>(1, 8192 / y))), static_cast<uint32_t>(y));
    if (store) klaunch(a.bf16 ? kv_q4_store_kernel<true> : kv_q4_store_kernel<false>, grid, dim3(256), 0, s, a);
    else klaunch(a.bf16 ? kv_q4_load_kernel<true> : kv_q4_load_kernel<false>, grid, dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace q35k
