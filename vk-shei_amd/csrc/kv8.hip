// The 8-bit paged K/V cache: rotating and appending rows, reading rows back,
// and the attention that reads it.
//
// A block of 16 tokens of one kv head has one scale for K and one for V, so a
// token costs 2 * head_dim bytes per head and half a byte of scale instead of
// 4 * head_dim bytes: the decode, an HBM stream of the cache, moves half as
// much.  K rows are plain rows.  V keeps four tokens of a dimension side by
// side ([4][head_dim][4] bytes per block): that is the order in which the P.V
// MFMA wants its operand, so V needs no transposition through LDS.
#include <algorithm>

#include "common.hpp"
#include "kernels.hpp"

namespace mslim {

namespace {

template <int FMT>
struct Format;
template <>
struct Format<kFormatE4m3> {
    // largest value 448 = 1.75 * 2^8
    static constexpr int kExponent = 9;
    static constexpr uint32_t kMantissa = 0x600000u;
};
template <>
struct Format<kFormatInt8> {
    // largest value 127 = 1.984375 * 2^6
    static constexpr int kExponent = 7;
    static constexpr uint32_t kMantissa = 0x7E0000u;
};

// The scale of values whose largest magnitude has the bits `amax`: the
// smallest power of two, 2^-126 at least, with amax <= largest * scale.  NaN
// where a value is not finite: its block stands for NaN until it is begun
// anew, so a value that 8 bits cannot hold is never a wrong number.
// Powers of two make every later change of a block's scale an exact shift of
// the values it stands for, so growing it costs at most the bits that the
// larger scale has not, however often it grows; an E4M3 value loses nothing
// against a finer scale, an INT8 value at most one bit.
template <int FMT>
__device__ __forceinline__ float scale_of(uint32_t amax) {
    if (amax >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
    // amax = m * 2^e2 with 1 <= m < 2 (subnormals end at the bound anyway)
    const int e2 = (int)(amax >> 23) - 127;
    const int e = e2 + 1 - Format<FMT>::kExponent + ((amax & 0x7fffffu) > Format<FMT>::kMantissa ? 1 : 0);
    return __uint_as_float((uint32_t)(max(e, -126) + 127) << 23);
}

// Four values, divided by their scale, as bytes.  Round to nearest, halves to
// even; a quotient beyond the format's range by a rounding ends at its edge.
template <int FMT>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
    if constexpr (FMT == kFormatE4m3) {
        auto edge = [](float x) { return x > 448.0f ? 448.0f : x < -448.0f ? -448.0f : x; };
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(edge(a), edge(b), 0, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(edge(c), edge(d), w, true);
        return (uint32_t)w;
    } else {
        auto whole = [](float x) { return (uint32_t)(int)rintf(fminf(fmaxf(x, -127.0f), 127.0f)) & 0xffu; };
        return whole(a) | whole(b) << 8 | whole(c) << 16 | whole(d) << 24;
    }
}

// The value of byte i of four.
template <int FMT>
__device__ __forceinline__ float byte_value(uint32_t w, int i) {
    if constexpr (FMT == kFormatE4m3) {
        switch (i) {
        case 0: return __builtin_amdgcn_cvt_f32_fp8((int)w, 0);
        case 1: return __builtin_amdgcn_cvt_f32_fp8((int)w, 1);
        case 2: return __builtin_amdgcn_cvt_f32_fp8((int)w, 2);
        default: return __builtin_amdgcn_cvt_f32_fp8((int)w, 3);
        }
    } else {
        return (float)(int8_t)(w >> (8 * i));
    }
}

// Four bytes of an older scale under a larger one.
template <int FMT>
__device__ __forceinline__ uint32_t rescale4(uint32_t w, float ratio) {
    return encode4<FMT>(byte_value<FMT>(w, 0) * ratio, byte_value<FMT>(w, 1) * ratio, byte_value<FMT>(w, 2) * ratio,
                        byte_value<FMT>(w, 3) * ratio);
}

// Eight bytes as BF16 values of their format, exactly: both formats' values
// have at most eight significant bits.
template <int FMT>
__device__ __forceinline__ bf16x8_t widen8(uint32_t lo, uint32_t hi) {
    uint32_t w[4];
    if constexpr (FMT == kFormatE4m3) {
        w[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false));
        w[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true));
        w[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false));
        w[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t s = i < 2 ? lo : hi;
            const uint32_t x = __float_as_uint((float)(int8_t)(s >> (16 * (i & 1))));
            const uint32_t y = __float_as_uint((float)(int8_t)(s >> (16 * (i & 1) + 8)));
            w[i] = __builtin_amdgcn_perm(y, x, 0x07060302u);
        }
    }
    return __builtin_bit_cast(bf16x8_t, make_uint4(w[0], w[1], w[2], w[3]));
}

__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#pragma unroll
    for (int mask = 1; mask < 64; mask <<= 1) v = max(v, (uint32_t)__shfl_xor((int)v, mask, 64));
    return v;
}

// c and s of a rotary pair: the angle is position * turn periods in 64 bits,
// reduced to half a period there, so positions keep their full accuracy
// however far they are; the functions and the rotation are in 32.
__device__ __forceinline__ float2 turn_cs(int64_t position, double turn) {
    const double t = (double)position * turn;
    float s, c;
    sincospif((float)(2.0 * (t - rint(t))), &s, &c);
    return make_float2(c, s);
}

// Index of the 16-token block that holds token t (>= 0) of a sequence, or -1
// where the table names no page of the pool.
__device__ __forceinline__ int64_t block_of(const Kv8Cache &c, int b, int head, int64_t t) {
    const int64_t page = c.table[(int64_t)b * c.pages_per_seq + (t >> c.shift)];
    if (page < 0 || page >= c.pool_pages) return -1;
    return ((page * c.kv_heads + head) << (c.shift - 4)) + ((t & ((1 << c.shift) - 1)) >> 4);
}

struct AppendArgs {
    Kv8Cache cache;
    const uint16_t *q, *k, *v;
    uint16_t *q_out;
    const int32_t *positions;
    int batch, tokens, q_heads;
    int blocks;     // 16-token blocks that `tokens` rows can reach
    int kv_groups;  // workgroups of a block: four kv heads each
    int64_t kv_workgroups;
    Kv8Turns turns;
};

__device__ __forceinline__ void unpack8(const uint4 &w, float (&x)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = bf16_lo(u[i]);
        x[2 * i + 1] = bf16_hi(u[i]);
    }
}

// Eight rotate-half pairs (x[i], p[i]) -> (x c - p s, p c + x s).
__device__ __forceinline__ void rotate8(float (&x)[8], float (&p)[8], const float2 *cs) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float2 t = cs[i];
        const float lo = __fsub_rn(__fmul_rn(x[i], t.x), __fmul_rn(p[i], t.y));
        p[i] = __fadd_rn(__fmul_rn(p[i], t.x), __fmul_rn(x[i], t.y));
        x[i] = lo;
    }
}

// The first kv_workgroups workgroups write the cache, a wavefront per (block,
// kv head); the others rotate a row of Q each.  The rows of a block that are
// not new and lie before the new ones are read only where the block's scale
// grows; the rows behind keep their bytes.  NI: units of 8 pairs of a lane.
template <int FMT, int NI, bool ROTATE>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a) {
    __shared__ float2 cs_lds[16 * 16 * NI * 2];  // [16 rows][half <= 32 * NI]
    const Kv8Cache &c = a.cache;
    const int d = c.head_dim, half = d / 2;
    const int hc = half / 8;  // units per head row
    const int tid = threadIdx.x;
    if ((int64_t)blockIdx.x >= a.kv_workgroups) {
        if constexpr (ROTATE) {
            const int64_t row = blockIdx.x - a.kv_workgroups;  // batch * tokens
            const int64_t position = (int64_t)a.positions[row / a.tokens] + row % a.tokens;
            for (int f = tid; f < half; f += 256) cs_lds[f] = turn_cs(position, a.turns.turn[f]);
            __syncthreads();
            const uint16_t *src = a.q + row * a.q_heads * d;
            uint16_t *dst = a.q_out + row * a.q_heads * d;
            for (int u = tid; u < a.q_heads * hc; u += 256) {
                const int at = u / hc * d + u % hc * 8;
                float x[8], p[8];
                unpack8(*reinterpret_cast<const uint4 *>(src + at), x);
                unpack8(*reinterpret_cast<const uint4 *>(src + at + half), p);
                rotate8(x, p, cs_lds + u % hc * 8);
                auto pack = [](const float (&y)[8]) {
                    return make_uint4(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]), pack_bf16x2(y[4], y[5]),
                                      pack_bf16x2(y[6], y[7]));
                };
                *reinterpret_cast<uint4 *>(dst + at) = pack(x);
                *reinterpret_cast<uint4 *>(dst + at + half) = pack(p);
            }
        }
        return;
    }
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int group = (int)(blockIdx.x % a.kv_groups);
    const int64_t bj = blockIdx.x / a.kv_groups;
    const int b = (int)(bj / a.blocks);
    const int64_t pos = a.positions[b];
    const int64_t base = ((pos >> 4) + bj % a.blocks) * 16;  // first token of the block
    const int64_t capacity = (int64_t)c.pages_per_seq << c.shift;
    const int64_t lo64 = max(max(pos, base), (int64_t)0);
    const int64_t hi64 = min(min(pos + a.tokens, base + 16), capacity);
    if (base < 0 || lo64 >= hi64) return;  // uniform over the workgroup
    const int lo = (int)(lo64 - base), n = (int)(hi64 - lo64);
    const int64_t row0 = (int64_t)b * a.tokens + (lo64 - pos);  // of k and v
    if constexpr (ROTATE) {
        for (int u = tid; u < n * half; u += 256)
            cs_lds[u] = turn_cs(lo64 + u / half, a.turns.turn[u % half]);
        __syncthreads();
    }
    const int head = group * 4 + wave;
    if (head >= c.kv_heads) return;
    const int64_t block = block_of(c, b, head, base);
    if (block < 0) return;

    // K: lane's units are (row, 8 pairs).
    uint8_t *kb = c.k + block * 16 * d;
    float x[NI][8], p[NI][8];
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int u = lane + 64 * i;
        if (u < n * hc) {
            const int r = u / hc, at = u % hc * 8;
            const uint16_t *src = a.k + ((row0 + r) * c.kv_heads + head) * d + at;
            unpack8(*reinterpret_cast<const uint4 *>(src), x[i]);
            unpack8(*reinterpret_cast<const uint4 *>(src + half), p[i]);
            if constexpr (ROTATE) rotate8(x[i], p[i], cs_lds + r * half + at);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                amax = max(amax, max(__float_as_uint(x[i][j]) & 0x7fffffffu, __float_as_uint(p[i][j]) & 0x7fffffffu));
        }
    }
    float2 *scale_at = reinterpret_cast<float2 *>(c.scales) + block;
    float2 old = make_float2(0.0f, 0.0f);
    if (lo > 0) old = *scale_at;
    // The scale that covers old rows and new ones; NaN on either side stays.
    auto cover = [&](uint32_t top, float before) {
        const float fresh = scale_of<FMT>(top);
        return lo > 0 && !(fresh > before || fresh != fresh) ? before : fresh;
    };
    // What a value is multiplied by to become a byte; a NaN scale has zeros.
    auto inverse = [](float s) { return s == s ? __fdiv_rn(1.0f, s) : 0.0f; };
    const float ks = cover(wave_max(amax), old.x);
    const float ki = inverse(ks);
    auto times = [](float v, float by) { return by == 0.0f ? 0.0f : v * by; };
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int u = lane + 64 * i;
        if (u < n * hc) {
            uint8_t *dst = kb + (lo + u / hc) * d + u % hc * 8;
            auto pack = [&](const float (&y)[8]) {
                return make_uint2(encode4<FMT>(times(y[0], ki), times(y[1], ki), times(y[2], ki), times(y[3], ki)),
                                  encode4<FMT>(times(y[4], ki), times(y[5], ki), times(y[6], ki), times(y[7], ki)));
            };
            *reinterpret_cast<uint2 *>(dst) = pack(x[i]);
            *reinterpret_cast<uint2 *>(dst + half) = pack(p[i]);
        }
    }
    if (lo > 0 && ks > old.x) {
        const float ratio = __fdiv_rn(old.x, ks);
        for (int u = lane; u < lo * d / 8; u += 64) {
            uint2 *w = reinterpret_cast<uint2 *>(kb) + u;
            *w = make_uint2(rescale4<FMT>(w->x, ratio), rescale4<FMT>(w->y, ratio));
        }
    }

    // V: lane's units are (four tokens, 8 dims).
    constexpr int NV = (NI + 1) / 2;
    uint8_t *vb = c.v + block * 16 * d;
    const int dc = d / 8;
    uint4 rows[NV][4];
    amax = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int u = lane + 64 * i;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int r = u / dc * 4 + t - lo;  // among the new rows
            rows[i][t] = make_uint4(0, 0, 0, 0);
            if (u < 4 * dc && r >= 0 && r < n)
                rows[i][t] = *reinterpret_cast<const uint4 *>(a.v + ((row0 + r) * c.kv_heads + head) * d + u % dc * 8);
            const uint32_t w[4] = {rows[i][t].x, rows[i][t].y, rows[i][t].z, rows[i][t].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) amax = max(amax, max(w[j] << 16 & 0x7fffffffu, w[j] & 0x7fff0000u));
        }
    }
    const float vs = cover(wave_max(amax), old.y);
    const float vi = inverse(vs);
    const bool grown = lo > 0 && vs > old.y;
    const float ratio = grown ? __fdiv_rn(old.y, vs) : 1.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int u = lane + 64 * i;
        const int t0 = u / dc * 4;
        if (u >= 4 * dc) continue;
        const bool any_new = t0 < lo + n && t0 + 4 > lo, all_new = t0 >= lo && t0 + 4 <= lo + n;
        if (!any_new && !(grown && t0 < lo)) continue;
        uint32_t *dst = reinterpret_cast<uint32_t *>(vb) + (u / dc * d + u % dc * 8);
        uint32_t w[8] = {};
        if (!all_new) {
            *reinterpret_cast<uint4 *>(w) = *reinterpret_cast<const uint4 *>(dst);
            *reinterpret_cast<uint4 *>(w + 4) = *reinterpret_cast<const uint4 *>(dst + 4);
        }
        // bytes of w that are new, and those of older rows
        uint32_t fresh = 0, older = 0;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            if (t0 + t >= lo && t0 + t < lo + n) fresh |= 0xffu << (8 * t);
            if (t0 + t < lo) older |= 0xffu << (8 * t);
        }
        float y[4][8];
#pragma unroll
        for (int t = 0; t < 4; ++t) unpack8(rows[i][t], y[t]);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t now =
                encode4<FMT>(times(y[0][j], vi), times(y[1][j], vi), times(y[2][j], vi), times(y[3][j], vi));
            uint32_t kept = w[j];
            if (grown) kept = (rescale4<FMT>(kept, ratio) & older) | (kept & ~older);
            w[j] = (now & fresh) | (kept & ~fresh);
        }
        *reinterpret_cast<uint4 *>(dst) = *reinterpret_cast<const uint4 *>(w);
        *reinterpret_cast<uint4 *>(dst + 4) = *reinterpret_cast<const uint4 *>(w + 4);
    }
    if (lane == 0) *scale_at = make_float2(ks, vs);
}

// Work item: (sequence, aligned group of four tokens, kv head, 8 dims).
template <int FMT>
__global__ __launch_bounds__(256) void gather_kernel(Kv8Cache c, int batch, int tokens, int groups,
                                                     const int32_t *first, uint16_t *k_rows, uint16_t *v_rows) {
    const int d = c.head_dim, dc = d / 8;
    const int64_t work = (int64_t)batch * groups * c.kv_heads * dc;
    const int64_t capacity = (int64_t)c.pages_per_seq << c.shift;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < work; i += (int64_t)gridDim.x * 256) {
        const int at = (int)(i % dc) * 8;
        int64_t j = i / dc;
        const int head = (int)(j % c.kv_heads);
        j /= c.kv_heads;
        const int b = (int)(j / groups);
        const int64_t start = first ? first[b] : 0;
        const int64_t t0 = ((start >> 2) + j % groups) * 4;  // rows t0 .. t0 + 3, floor division for rows < 0
        uint2 kw[4] = {};
        uint32_t vw[8] = {};
        float2 s = make_float2(0.0f, 0.0f);
        const int64_t block = t0 >= 0 && t0 < capacity ? block_of(c, b, head, t0) : -1;
        if (block >= 0) {
            s = reinterpret_cast<const float2 *>(c.scales)[block];
            const int g = (int)(t0 >> 2 & 3);
#pragma unroll
            for (int t = 0; t < 4; ++t)
                kw[t] = *reinterpret_cast<const uint2 *>(c.k + (block * 16 + g * 4 + t) * d + at);
            const uint8_t *vb = c.v + block * 16 * d + (g * d + at) * 4;
            *reinterpret_cast<uint4 *>(vw) = *reinterpret_cast<const uint4 *>(vb);
            *reinterpret_cast<uint4 *>(vw + 4) = *reinterpret_cast<const uint4 *>(vb + 16);
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int64_t r = t0 + t - start;
            if (r < 0 || r >= tokens) continue;
            uint32_t ko[4], vo[4];
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const uint32_t pair = (w < 2 ? kw[t].x : kw[t].y);
                ko[w] = pack_bf16x2(byte_value<FMT>(pair, (2 * w) & 3) * s.x, byte_value<FMT>(pair, (2 * w + 1) & 3) * s.x);
                vo[w] = pack_bf16x2(byte_value<FMT>(vw[2 * w], t) * s.y, byte_value<FMT>(vw[2 * w + 1], t) * s.y);
            }
            const int64_t dst = (((int64_t)b * tokens + r) * c.kv_heads + head) * d + at;
            *reinterpret_cast<uint4 *>(k_rows + dst) = make_uint4(ko[0], ko[1], ko[2], ko[3]);
            *reinterpret_cast<uint4 *>(v_rows + dst) = make_uint4(vo[0], vo[1], vo[2], vo[3]);
        }
    }
}

// ---- attention ---------------------------------------------------------------

constexpr int kWaves = 4;
constexpr int kTile = 32;  // tokens of a wavefront's step: two blocks
constexpr int kRows = 16;  // query rows of a workgroup: one MFMA tile

struct AttentionArgs {
    Kv8Cache cache;
    const uint16_t *q;
    uint16_t *out;
    int batch, queries, q_heads;
    int row_tiles;  // of a kv head's queries * group rows
    float scale_log2e;
    int len[kKv8Batch];
};

// A workgroup of four wavefronts takes 16 query rows of one kv head ((query,
// head of the group) pairs) over all their tokens, the wavefronts 32 tokens
// each in turn:
//   * S^T = K.Q^T on v_mfma_f32_16x16x32_bf16, 16 tokens of a block as M and
//     the rows as N.  A lane's 16 bytes of a K row widen to the A operands of
//     two MFMAs, whose 8 dims per lane group are taken from Q in that order;
//   * the scores take the block's K scale times scale * log2(e) in f32;
//   * P goes to the P.V MFMA from the accumulator where S^T left it, in BF16
//     and times the block's V scale (exact: a power of two); the row sum adds
//     the rounded P, so O / l is a convex combination of V rows;
//   * a lane's 16 bytes of V are four dims of four tokens: the B operand's
//     tokens of its lane group;
//   * the four wavefronts merge in LDS.
// DM: head_dim rounded up to 64, 128 or 256; FULL: equal to it.
template <int FMT, int DM, bool FULL>
__global__ __launch_bounds__(64 * kWaves) void attention_kernel(AttentionArgs a) {
    constexpr int KP = DM / 64;  // 16-byte pieces of a lane per block
    __shared__ float comb_ml[kWaves][kRows][2];
    __shared__ __align__(16) float comb_acc[kWaves][kRows][DM];
    const Kv8Cache &c = a.cache;
    const int d = FULL ? DM : c.head_dim;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int row16 = lane & 15, grp = lane >> 4;
    const int group = a.q_heads / c.kv_heads;
    const int rt = (int)(blockIdx.x % a.row_tiles);
    const int head = (int)(blockIdx.x / a.row_tiles % c.kv_heads);
    const int b = (int)(blockIdx.x / a.row_tiles / c.kv_heads);
    const int len = a.len[b];
    const int rows = a.queries * group;

    // Row r of a kv head is (query r / group, head r % group of the group).
    auto row_at = [&](int r) {
        return (((int64_t)b * a.queries + r / group) * a.q_heads + head * group + r % group) * d;
    };
    const int my_row = rt * kRows + row16;
    const int first_limit = len - a.queries + rt * kRows / group + 1;  // tokens that the tile's first row sees
    const int limit = my_row < rows ? len - a.queries + my_row / group + 1 : 0;
    bf16x8_t qf[KP][2];
#pragma unroll
    for (int j = 0; j < KP; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int at = j * 64 + grp * 16 + h * 8;
            qf[j][h] = bf16x8_t{};
            if (my_row < rows && (FULL || at < d))
                qf[j][h] = *reinterpret_cast<const bf16x8_t *>(a.q + row_at(my_row) + at);
        }

    float m_run = -__FLT_MAX__, l_run = 0.0f;
    floatx4_t o[KP * 4];  // O[row 4*grp+i][dim 64*(sl/4) + 4*row16 + sl%4]
#pragma unroll
    for (int sl = 0; sl < KP * 4; ++sl) o[sl] = floatx4_t{0.0f, 0.0f, 0.0f, 0.0f};

    for (int t0 = wave * kTile; t0 < len; t0 += kWaves * kTile) {
        u32x4_t k[2][KP], v[2][KP];
        float2 sc[2];
        bool whole = t0 + kTile <= first_limit;
        int tokens[2];  // of a block that any row may see
#pragma unroll
        for (int blk = 0; blk < 2; ++blk) {
            const int bt = t0 + blk * 16;
            const int64_t block = bt < len ? block_of(c, b, head, bt) : -1;
            tokens[blk] = block >= 0 ? min(16, len - bt) : 0;
            whole &= block >= 0;
            const int64_t at = max(block, (int64_t)0);
            sc[blk] = reinterpret_cast<const float2 *>(c.scales)[at];
            const uint8_t *kb = c.k + at * 16 * d + row16 * d + grp * 16;
            const uint8_t *vb = c.v + at * 16 * d + grp * d * 4 + row16 * 16;
#pragma unroll
            for (int j = 0; j < KP; ++j) {
                k[blk][j] = v[blk][j] = u32x4_t{0, 0, 0, 0};
                if (FULL || j * 64 + grp * 16 < d) k[blk][j] = *reinterpret_cast<const u32x4_t *>(kb + j * 64);
                if (FULL || j * 64 + row16 * 4 < d) v[blk][j] = *reinterpret_cast<const u32x4_t *>(vb + j * 256);
            }
        }
        floatx4_t s[2];
#pragma unroll
        for (int blk = 0; blk < 2; ++blk) {
            s[blk] = floatx4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < KP; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    s[blk] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                        widen8<FMT>(k[blk][j][2 * h], k[blk][j][2 * h + 1]), qf[j][h], s[blk], 0, 0, 0);
            const float ks = sc[blk].x * a.scale_log2e;
#pragma unroll
            for (int i = 0; i < 4; ++i) s[blk][i] *= ks;
        }
        // Tokens that a row does not see weigh nothing, whatever their bytes
        // and scales hold.
        if (!whole) {
#pragma unroll
            for (int blk = 0; blk < 2; ++blk) {
                const int at = t0 + blk * 16 + grp * 4;
                const int fill = min(max(tokens[blk] - grp * 4, 0), 4);
                const uint32_t keep = fill == 4 ? 0xffffffffu : (1u << (8 * fill)) - 1;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (i >= fill || at + i >= limit) s[blk][i] = -INFINITY;
#pragma unroll
                for (int j = 0; j < KP; ++j) v[blk][j] &= keep;
            }
        }
        float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                         fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
        mx = wave_xor_max(mx, 16);
        mx = wave_xor_max(mx, 32);
        const float m_new = fmaxf(m_run, mx);
        const float alpha = __builtin_amdgcn_exp2f(m_run - m_new);
        bf16x8_t p;
        float psum = 0.0f;
#pragma unroll
        for (int blk = 0; blk < 2; ++blk)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float pr = round_bf16(__builtin_amdgcn_exp2f(s[blk][i] - m_new));
                psum += pr;
                // a NaN scale of tokens that the row does not see stays out
                p[blk * 4 + i] = (__bf16)(s[blk][i] == -INFINITY ? 0.0f : pr * sc[blk].y);
            }
        l_run = l_run * alpha + psum;
        m_run = m_new;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float ai = __shfl(alpha, 4 * grp + i, 64);
#pragma unroll
            for (int sl = 0; sl < KP * 4; ++sl) o[sl][i] *= ai;
        }
#pragma unroll
        for (int sl = 0; sl < KP * 4; ++sl)
            o[sl] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(p, widen8<FMT>(v[0][sl / 4][sl % 4], v[1][sl / 4][sl % 4]),
                                                            o[sl], 0, 0, 0);
    }

    l_run = wave_xor_sum(l_run, 16);
    l_run = wave_xor_sum(l_run, 32);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < KP; ++j)
            *reinterpret_cast<float4 *>(&comb_acc[wave][4 * grp + i][j * 64 + row16 * 4]) =
                make_float4(o[j * 4][i], o[j * 4 + 1][i], o[j * 4 + 2][i], o[j * 4 + 3][i]);
    if (lane < kRows) {
        comb_ml[wave][lane][0] = m_run;
        comb_ml[wave][lane][1] = l_run;
    }
    __syncthreads();
    const int here = min(kRows, rows - rt * kRows);
    for (int it = tid; it < here * (d / 4); it += 64 * kWaves) {
        const int r = it / (d / 4), at = it % (d / 4) * 4;
        float m = -__FLT_MAX__;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) m = fmaxf(m, comb_ml[w][r][0]);
        float l = 0.0f;
        float4 ov = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float wt = __builtin_amdgcn_exp2f(comb_ml[w][r][0] - m);
            l = fmaf(comb_ml[w][r][1], wt, l);
            const float4 y = *reinterpret_cast<const float4 *>(&comb_acc[w][r][at]);
            ov.x = fmaf(y.x, wt, ov.x); ov.y = fmaf(y.y, wt, ov.y);
            ov.z = fmaf(y.z, wt, ov.z); ov.w = fmaf(y.w, wt, ov.w);
        }
        // a row that sees nothing is zeros
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        uint2 packed;
        packed.x = pack_bf16x2(ov.x * inv, ov.y * inv);
        packed.y = pack_bf16x2(ov.z * inv, ov.w * inv);
        *reinterpret_cast<uint2 *>(a.out + row_at(rt * kRows + r) + at) = packed;
    }
}

template <int FMT, int DM>
void launch_attention(const AttentionArgs &a, unsigned grid, hipStream_t stream) {
    if (a.cache.head_dim == DM)
        hipLaunchKernelGGL((attention_kernel<FMT, DM, true>), dim3(grid), dim3(64 * kWaves), 0, stream, a);
    else
        hipLaunchKernelGGL((attention_kernel<FMT, DM, false>), dim3(grid), dim3(64 * kWaves), 0, stream, a);
}

template <int FMT>
void launch_append(const AppendArgs &a, bool rotate, unsigned grid, hipStream_t stream) {
    const int d = a.cache.head_dim;
#define MSLIM_KV8_APPEND(NI)                                                                                  \
    if (rotate) hipLaunchKernelGGL((append_kernel<FMT, NI, true>), dim3(grid), dim3(256), 0, stream, a);     \
    else hipLaunchKernelGGL((append_kernel<FMT, NI, false>), dim3(grid), dim3(256), 0, stream, a)
    if (d <= 64) { MSLIM_KV8_APPEND(1); }
    else if (d <= 128) { MSLIM_KV8_APPEND(2); }
    else { MSLIM_KV8_APPEND(4); }
#undef MSLIM_KV8_APPEND
}

}  // namespace

namespace {
// 16-token blocks that a sequence's rows can reach, and workgroups of a block
// (four kv heads each).
int append_blocks(const Kv8AppendLaunch &l) { return (l.tokens + kKv8Block - 2) / kKv8Block + 1; }
int append_groups(const Kv8AppendLaunch &l) { return (l.cache.kv_heads + 3) / 4; }
}  // namespace

int64_t kv8_append_workgroups(const Kv8AppendLaunch &l) {
    return (int64_t)l.batch * append_blocks(l) * append_groups(l) + (l.rotate ? (int64_t)l.batch * l.tokens : 0);
}

hipError_t launch_kv8_append(const Kv8AppendLaunch &l, hipStream_t stream) {
    AppendArgs a{};
    a.cache = l.cache;
    a.q = l.q; a.k = l.k; a.v = l.v; a.q_out = l.q_out;
    a.positions = l.positions;
    a.batch = l.batch; a.tokens = l.tokens; a.q_heads = l.q_heads;
    a.blocks = append_blocks(l);
    a.kv_groups = append_groups(l);
    a.kv_workgroups = (int64_t)l.batch * a.blocks * a.kv_groups;
    a.turns = l.turns;
    const unsigned grid = (unsigned)kv8_append_workgroups(l);
    if (l.cache.format == kFormatE4m3) launch_append<kFormatE4m3>(a, l.rotate, grid, stream);
    else launch_append<kFormatInt8>(a, l.rotate, grid, stream);
    return hipGetLastError();
}

hipError_t launch_kv8_gather(const Kv8Cache &cache, int batch, int tokens, const int32_t *first, uint16_t *k_rows,
                             uint16_t *v_rows, hipStream_t stream) {
    const int groups = (tokens + 2) / 4 + 1;
    const int64_t work = (int64_t)batch * groups * cache.kv_heads * (cache.head_dim / 8);
    const unsigned grid = (unsigned)std::min<int64_t>((work + 255) / 256, 1 << 20);
    if (cache.format == kFormatE4m3)
        hipLaunchKernelGGL(gather_kernel<kFormatE4m3>, dim3(grid), dim3(256), 0, stream, cache, batch, tokens, groups,
                           first, k_rows, v_rows);
    else
        hipLaunchKernelGGL(gather_kernel<kFormatInt8>, dim3(grid), dim3(256), 0, stream, cache, batch, tokens, groups,
                           first, k_rows, v_rows);
    return hipGetLastError();
}

hipError_t launch_kv8_attention(const Kv8AttentionLaunch &l, hipStream_t stream) {
    AttentionArgs a{};
    a.cache = l.cache;
    a.q = l.q; a.out = l.out;
    a.batch = l.batch; a.queries = l.queries; a.q_heads = l.q_heads;
    const int64_t rows = (int64_t)l.queries * (l.q_heads / l.cache.kv_heads);
    a.row_tiles = (int)((rows + kRows - 1) / kRows);
    a.scale_log2e = l.scale * kLog2e;
    for (int b = 0; b < l.batch; ++b) a.len[b] = l.len[b];
    const unsigned grid = (unsigned)((int64_t)l.batch * l.cache.kv_heads * a.row_tiles);
    const int d = l.cache.head_dim;
#define MSLIM_KV8_ATTENTION(FMT)                                        \
    if (d <= 64) launch_attention<FMT, 64>(a, grid, stream);            \
    else if (d <= 128) launch_attention<FMT, 128>(a, grid, stream);     \
    else launch_attention<FMT, 256>(a, grid, stream)
    if (l.cache.format == kFormatE4m3) { MSLIM_KV8_ATTENTION(kFormatE4m3); }
    else { MSLIM_KV8_ATTENTION(kFormatInt8); }
#undef MSLIM_KV8_ATTENTION
    return hipGetLastError();
}

}  // namespace mslim
