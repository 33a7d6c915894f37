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
#include <climits>
#include <type_traits>

#include "common.hpp"
#include "kernels.hpp"
#include "kv8.hpp"

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

// Four bytes of an older scale under a larger one.
template <int FMT>
__device__ __forceinline__ uint32_t rescale4(uint32_t w, float ratio) {
    return encode4<FMT>(byte_value<FMT>(w, 0) * ratio, byte_value<FMT>(w, 1) * ratio, byte_value<FMT>(w, 2) * ratio,
                        byte_value<FMT>(w, 3) * ratio);
}

__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#pragma unroll
    for (int mask = 1; mask < 64; mask <<= 1) v = max(v, (uint32_t)__shfl_xor((int)v, mask, 64));
    return v;
}

// c and s of a rotary pair: the angle is position * turn periods in 64 bits,
// reduced to half a period there, so positions keep their full accuracy
// however far they are.  The functions are rounded to 32 bits once: the f32
// ones, a unit off now and then, moved one byte in 10^6 that a rounding apart
// from them does not.
__device__ __forceinline__ float2 turn_cs(int64_t position, double turn) {
    const double t = (double)position * turn;
    double s, c;
    sincospi(2.0 * (t - rint(t)), &s, &c);
    return make_float2((float)c, (float)s);
}

// Index of the 16-token block that holds token t (>= 0) of a sequence, or -1
// where the table names no page of the pool.  scalar: the same for the whole
// wavefront.
__device__ __forceinline__ int64_t block_of(const Kv8Cache &c, int b, int head, int64_t t, bool scalar = false) {
    const int64_t page = scalar ? scalar_page(c.table + (int64_t)b * c.pages_per_seq + (t >> c.shift))
                                : c.table[(int64_t)b * c.pages_per_seq + (t >> c.shift)];
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
    uint32_t kv_workgroups;
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
// DIM: head_dim where it is 64, 128 or 256, else 0: a step of one token is a
// chain of a few loads and sums, in which the divisions by a head_dim known at
// run time alone took 1.6 of 6.2 us.
template <int FMT, int NI, bool ROTATE, int DIM>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a) {
    __shared__ float2 cs_lds[16 * 16 * NI * 2];  // [16 rows][half <= 32 * NI]
    const Kv8Cache &c = a.cache;
    const int d = DIM ? DIM : c.head_dim, half = d / 2;
    const int hc = half / 8;  // units per head row
    const int tid = threadIdx.x;
    if (blockIdx.x >= a.kv_workgroups) {
        if constexpr (ROTATE) {
            const uint32_t r = blockIdx.x - a.kv_workgroups;  // of batch * tokens
            const int64_t row = r;
            const int64_t position = (int64_t)scalar_page(a.positions + r / (uint32_t)a.tokens) + r % (uint32_t)a.tokens;
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
    const int group = (int)(blockIdx.x % (uint32_t)a.kv_groups);
    const uint32_t bj = blockIdx.x / (uint32_t)a.kv_groups;
    const int b = (int)(bj / (uint32_t)a.blocks);
    const int64_t pos = scalar_page(a.positions + b);
    const int64_t base = ((pos >> 4) + bj % (uint32_t)a.blocks) * 16;  // first token of the block
    const int64_t capacity = (int64_t)c.pages_per_seq << c.shift;
    const int64_t lo64 = max(max(pos, base), (int64_t)0);
    const int64_t hi64 = min(min(pos + a.tokens, base + 16), capacity);
    if (base < 0 || lo64 >= hi64) return;  // uniform over the workgroup
    const int lo = (int)(lo64 - base), n = (int)(hi64 - lo64);
    const int64_t row0 = (int64_t)b * a.tokens + (lo64 - pos);  // of k and v
    const int head = group * 4 + wave;
    const bool active = head < c.kv_heads;
    const int64_t block = active ? block_of(c, b, head, base, true) : -1;
    float2 *scale_at = reinterpret_cast<float2 *>(c.scales) + max(block, (int64_t)0);

    // All loads go out before the cos and sin are computed: a step of one
    // token is a chain of them.  K: a lane's units are (row, 8 pairs); V:
    // (four tokens, 8 dims).
    constexpr int NV = (NI + 1) / 2;
    const int dc = d / 8;
    uint4 kx[NI], kp[NI], rows[NV][4];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int u = lane + 64 * i;
        if (active && u < n * hc) {
            const uint16_t *src = a.k + ((row0 + u / hc) * c.kv_heads + head) * d + u % hc * 8;
            kx[i] = *reinterpret_cast<const uint4 *>(src);
            kp[i] = *reinterpret_cast<const uint4 *>(src + half);
        }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int u = lane + 64 * i;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int r = u / dc * 4 + t - lo;  // among the new rows
            rows[i][t] = make_uint4(0, 0, 0, 0);
            if (active && u < 4 * dc && r >= 0 && r < n)
                rows[i][t] = *reinterpret_cast<const uint4 *>(a.v + ((row0 + r) * c.kv_heads + head) * d + u % dc * 8);
        }
    }
    float2 old = make_float2(0.0f, 0.0f);
    if (lo > 0) old = scalar_scales(reinterpret_cast<const float *>(scale_at));  // this wavefront alone writes it
    if constexpr (ROTATE) {
        for (int u = tid; u < n * half; u += 256)
            cs_lds[u] = turn_cs(lo64 + u / half, a.turns.turn[u % half]);
        __syncthreads();
    }
    if (block < 0) return;

    uint8_t *kb = c.k + block * 16 * d;
    float x[NI][8], p[NI][8];
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int u = lane + 64 * i;
        if (u < n * hc) {
            unpack8(kx[i], x[i]);
            unpack8(kp[i], p[i]);
            if constexpr (ROTATE) rotate8(x[i], p[i], cs_lds + u / hc * half + u % hc * 8);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                amax = max(amax, max(__float_as_uint(x[i][j]) & 0x7fffffffu, __float_as_uint(p[i][j]) & 0x7fffffffu));
        }
    }
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

    uint8_t *vb = c.v + block * 16 * d;
    amax = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const uint32_t w[4] = {rows[i][t].x, rows[i][t].y, rows[i][t].z, rows[i][t].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) amax = max(amax, max(w[j] << 16 & 0x7fffffffu, w[j] & 0x7fff0000u));
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

constexpr int kTile = 32;                // tokens of a wavefront's step: two blocks
constexpr int kCus = 256;
constexpr int kMergeParts = 16;          // parts that a merging thread loads at once
// Calls that read more than the Infinity Cache holds load K and V
// non-temporally: 538 MB 99.8 -> 92.0 us, 269 MB 53.2 -> 51.0 us, 67 MB
// 20.0 -> 22.1 us.
constexpr int64_t kStreamBytes = 200ll << 20;
// kv8_two_row_tiles
constexpr int64_t kRereadBytes = 100ll << 20;
constexpr int64_t kPairSteps = 9 * 2048;
// One row tile: workgroups of eight wavefronts, one per CU, instead of four, two
// per CU, where segments have at least this many parts: half as many to merge (8,192
// tokens, 64 parts: 19.8 -> 13.5 us; 4 x 32,768 56.5 -> 53.2 us).  With
// several segments to a workgroup the switch from one to the next stalls
// twice the wavefronts: 32 sequences of 512 .. 8,192 tokens 63 -> 68 us.
constexpr int kWideParts = 12;

struct AttentionArgs {
    Kv8Cache cache;
    const uint16_t *q;
    uint16_t *out;
    float *partial;  // [2 * workgroups][rows of a tile][head_dim + 2]: the accumulators, then (m, l)
    int *counters;   // [batch][kv_heads * row_tiles] parts done, zero between launches
    int batch, queries, q_heads;
    int row_tiles;   // of a kv head's queries * group rows
    float scale_log2e;
    // Segments (sequence, kv head, row tile) have as many chunks as their
    // sequence.  Laid end to end, workgroup w of a split launch takes `share`
    // of them (one more for the first `extra` workgroups) from first_chunk(w)
    // on, so all get the same work whatever the lengths; an unsplit launch has
    // a workgroup per segment.
    bool split, merge_launch;
    int share, extra;
    int begin[kKv8Batch + 1];  // first chunk of each sequence
    int len[kKv8Batch];
};

// Chunks of a sequence: a step of `waves` wavefronts each.
__host__ __device__ inline int chunks_of(int len, int waves) {
    return len > 0 ? (len + waves * kTile - 1) / (waves * kTile) : 1;
}

// First chunk of workgroup w, and the workgroup that takes a chunk.
__device__ __forceinline__ int first_chunk(const AttentionArgs &a, int w) { return w * a.share + min(w, a.extra); }
__device__ __forceinline__ int owner_of(const AttentionArgs &a, int chunk) {
    const int more = a.extra * (a.share + 1);  // chunks of the workgroups with one more
    return chunk < more ? chunk / (a.share + 1) : a.extra + (chunk - more) / a.share;
}

// Loads of a wavefront's step: K row pieces, V pieces and the two scales of
// both blocks.
template <int KP>
struct TileRegs {
    u32x4_t k[2][KP], v[2][KP];
    float2 scale[2];
};

// 16 bytes of the cache; a call that streams more than the caches hold loads
// them non-temporally.
template <bool STREAM>
__device__ __forceinline__ u32x4_t cache_load(const uint8_t *p) {
    if constexpr (STREAM) return __builtin_nontemporal_load(reinterpret_cast<const u32x4_t *>(p));
    else return *reinterpret_cast<const u32x4_t *>(p);
}

// Four outputs of a row with the sum l; one that sees nothing is zeros.
__device__ __forceinline__ void write_row(uint16_t *out, const float4 &o, float l) {
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    uint2 packed;
    packed.x = pack_bf16x2(o.x * inv, o.y * inv);
    packed.y = pack_bf16x2(o.z * inv, o.w * inv);
    *reinterpret_cast<uint2 *>(out) = packed;
}

// Rows [r0, r1) of a row tile (first row `row0` of the kv head, `tile_rows`
// rows in a part) from the parts that workgroups w0, w0 + 1, ... left.
// Thread -> (four outputs, every `lanes`-th part from the `from`-th on), with
// more lanes where a part's rows are fewer than the threads.  A batch of parts
// costs a round trip to the device's memory: all its loads go out before the
// first is waited for, and only the sums depend on each other.  (One part
// after another, each with its own maximum, took 11 us for 64 parts, this 7.)
template <int THREADS>
__device__ __forceinline__ void merge_parts(const AttentionArgs &a, int b, int seg, int row0, int tile_rows, int r0,
                                            int r1, int d, int w0, int parts, int tid, float2 *lane_ml,
                                            float4 *lane_sums) {
    const int group = a.q_heads / a.cache.kv_heads;
    const int head = seg / a.row_tiles;
    const int64_t slot_floats = (int64_t)tile_rows * (d + 2);
    const int items = (r1 - r0) * (d / 4);
    int lanes = 1;
    while (lanes * 2 * items <= THREADS && lanes < 8) lanes *= 2;
    const int turns = (items + THREADS - 1) / THREADS;  // 1 where lanes > 1
    for (int turn = 0; turn < turns; ++turn) {
        const int it = lanes > 1 ? tid % items : turn * THREADS + tid;
        const int from = lanes > 1 ? tid / items : 0;
        const int r = r0 + min(it, items - 1) / (d / 4), at = min(it, items - 1) % (d / 4) * 4;
        float m = -__FLT_MAX__, l = 0.0f;
        float4 ov = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        auto batch = [&](int first, auto count) __attribute__((always_inline)) {
            constexpr int K = decltype(count)::value;
            float2 ml[K], x0[K], x1[K];
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int j = min(first + k * lanes, parts - 1);
                const float *src = a.partial + (2 * (w0 + j) + (j == 0 ? 1 : 0)) * slot_floats;
                ml[k] = load_coherent2(src + tile_rows * d + r * 2);
                x0[k] = load_coherent2(src + r * d + at);
                x1[k] = load_coherent2(src + r * d + at + 2);
            }
            float m_new = m;
#pragma unroll
            for (int k = 0; k < K; ++k) m_new = fmaxf(m_new, ml[k].x);
            const float keep = __builtin_amdgcn_exp2f(m - m_new);
            l *= keep;
            ov.x *= keep; ov.y *= keep; ov.z *= keep; ov.w *= keep;
            m = m_new;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (first + k * lanes >= parts) continue;
                const float w = __builtin_amdgcn_exp2f(ml[k].x - m);
                l = fmaf(ml[k].y, w, l);
                ov.x = fmaf(x0[k].x, w, ov.x); ov.y = fmaf(x0[k].y, w, ov.y);
                ov.z = fmaf(x1[k].x, w, ov.z); ov.w = fmaf(x1[k].y, w, ov.w);
            }
        };
        for (int j = from; j < parts; j += kMergeParts * lanes) {
            const int left = (parts - j + lanes - 1) / lanes;
            if (left <= 4) batch(j, std::integral_constant<int, 4>{});
            else if (left <= 8) batch(j, std::integral_constant<int, 8>{});
            else batch(j, std::integral_constant<int, kMergeParts>{});
        }
        if (lanes > 1) {
            lane_ml[tid] = make_float2(m, l);
            lane_sums[tid] = ov;
            __syncthreads();
            if (from == 0) {
                for (int k = 1; k < lanes; ++k) {
                    const float2 y = lane_ml[k * items + it];
                    const float4 x = lane_sums[k * items + it];
                    const float m_new = fmaxf(m, y.x);
                    const float wo = __builtin_amdgcn_exp2f(m - m_new), wn = __builtin_amdgcn_exp2f(y.x - m_new);
                    l = fmaf(l, wo, y.y * wn);
                    ov.x = fmaf(ov.x, wo, x.x * wn); ov.y = fmaf(ov.y, wo, x.y * wn);
                    ov.z = fmaf(ov.z, wo, x.z * wn); ov.w = fmaf(ov.w, wo, x.w * wn);
                    m = m_new;
                }
            }
        }
        if (it < items && from == 0) {
            const int row = row0 + r;
            write_row(a.out + (((int64_t)b * a.queries + row / group) * a.q_heads + head * group + row % group) * d + at,
                      ov, l);
        }
    }
}

// The merge as a launch of its own, a workgroup per row.
__global__ __launch_bounds__(256) void merge_kernel(AttentionArgs a, int tile_rows, int waves) {
    __shared__ float2 lane_ml[256];
    __shared__ float4 lane_sums[256];
    const int segments = a.cache.kv_heads * a.row_tiles;
    const int r = (int)(blockIdx.x % tile_rows);
    const int seg = (int)(blockIdx.x / tile_rows % segments), b = (int)(blockIdx.x / tile_rows / segments);
    const int row0 = seg % a.row_tiles * tile_rows;
    const int nch = chunks_of(a.len[b], waves), begin = a.begin[b] + seg * nch;
    const int w0 = owner_of(a, begin), parts = owner_of(a, begin + nch - 1) - w0 + 1;
    if (parts == 1 || row0 + r >= a.queries * (a.q_heads / a.cache.kv_heads)) return;
    merge_parts<256>(a, b, seg, row0, tile_rows, r, r + 1, a.cache.head_dim, w0, parts, threadIdx.x, lane_ml,
                     lane_sums);
}

// A workgroup of four or eight wavefronts takes 16 * NT query rows of one kv
// head ((query, head of the group) pairs) over a run of chunks, the wavefronts
// 32 tokens each of a chunk:
//   * K and V are an HBM stream: each wavefront holds two steps in registers,
//     the next one in flight while one is computed, and reads the page numbers
//     of a step one step before its loads go out (a third step in registers
//     was 1 to 2 us slower at every size, its moves costing more than it hid);
//   * S^T = K.Q^T on v_mfma_f32_16x16x32_bf16, 16 tokens of a block as M and
//     16 rows as N.  A lane's 16 bytes of a K row widen to the A operands of
//     two MFMAs, whose 8 dims per lane group are taken from Q in that order;
//   * the scores take the block's K scale times scale * log2(e) in f32;
//   * P goes to the P.V MFMA from the accumulator where S^T left it, in BF16
//     and times the block's V scale (exact: a power of two); the row sum adds
//     the rounded P, so O / l is a convex combination of V rows;
//   * a lane's 16 bytes of V are four dims of four tokens: the B operand's
//     tokens of its lane group;
//   * the wavefronts merge in LDS, the parts of a segment that several
//     workgroups took in the one that ends last or in a launch that follows,
//     in the order of the tokens either way.
// Measured, E4M3, 64/8 heads of 128: 4 x 32,768 tokens 49.4 us, 5.4 TB/s; each
// further 269 MB 40 us, 6.7 TB/s; about 4 us are the launch, 3 the first loads
// and 4 the merge.
// DM: head_dim rounded up to 64, 128 or 256; FULL: equal to it.
template <int FMT, int DM, bool FULL, int NT, int WAVES, int WGS, bool STREAM>
__global__ __launch_bounds__(64 * WAVES, WGS) void attention_kernel(AttentionArgs a) {
    constexpr int CHUNK = WAVES * kTile;
    constexpr int KP = DM / 64;  // 16-byte pieces of a lane per block
    constexpr int ROWS = 16 * NT;
    __shared__ float comb_ml[WAVES][ROWS][2];
    __shared__ __align__(16) float comb_acc[WAVES][16][DM];
    __shared__ int last_part;
    __shared__ float2 merge_ml[64 * WAVES];
    const Kv8Cache &c = a.cache;
    const int d = FULL ? DM : c.head_dim;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int row16 = lane & 15, grp = lane >> 4;
    const int group = a.q_heads / c.kv_heads;
    const int rows = a.queries * group;
    const int segments = c.kv_heads * a.row_tiles;  // of a sequence

    // Chunks [ch, ch_end) of segment `seg` of sequence b.
    auto run = [&](int b, int seg, int ch, int ch_end) __attribute__((always_inline)) {
        const int head = seg / a.row_tiles, rt = seg % a.row_tiles;
        const int len = a.len[b], nch = chunks_of(len, WAVES);
        // Row r of a kv head is (query r / group, head r % group of the group).
        auto row_at = [&](int r) {
            return (((int64_t)b * a.queries + r / group) * a.q_heads + head * group + r % group) * d;
        };
        const int first_limit = len - a.queries + rt * ROWS / group + 1;  // tokens that the tile's first row sees
        int limit[NT];
        bf16x8_t qf[NT][KP][2];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int r = rt * ROWS + t * 16 + row16;
            limit[t] = r < rows ? len - a.queries + r / group + 1 : 0;
#pragma unroll
            for (int j = 0; j < KP; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int at = j * 64 + grp * 16 + h * 8;
                    qf[t][j][h] = bf16x8_t{};
                    if (r < rows && (FULL || at < d))
                        qf[t][j][h] = *reinterpret_cast<const bf16x8_t *>(a.q + row_at(r) + at);
                }
        }

        // Loads never branch: a block past the end repeats the last one, an
        // entry that names no page reads page 0, a piece past head_dim the
        // row's last one; what they bring is masked below.
        // no row of the tile sees more than its last one
        const int most = len - a.queries + min(rt * ROWS + ROWS - 1, rows - 1) / group + 1;
        const int t_first = ch * CHUNK + wave * kTile, t_end = min(min(len, most), ch_end * CHUNK);
        const int32_t *table = c.table + (int64_t)b * c.pages_per_seq;
        const int last = max(len - 1, 0) & ~15;
        const int in_page = (1 << c.shift) - 1;
        struct Pages {
            int p[2];
        };
        auto pages_at = [&](int t0) {
            return Pages{{scalar_page(table + (min(t0, last) >> c.shift)), scalar_page(table + (min(t0 + 16, last) >> c.shift))}};
        };
        auto known = [&](int page) { return page >= 0 && page < (int)c.pool_pages; };
        const int k_at = row16 * d + grp * 16, v_at = grp * d * 4 + row16 * 16;
        auto load_tile = [&](TileRegs<KP> &r, Pages pg, int t0) {
#pragma unroll
            for (int blk = 0; blk < 2; ++blk) {
                const int bt = min(t0 + blk * 16, last);
                const int64_t page = known(pg.p[blk]) ? pg.p[blk] : 0;
                const int64_t block = ((page * c.kv_heads + head) << (c.shift - 4)) + ((bt & in_page) >> 4);
                r.scale[blk] = scalar_scales(c.scales + block * 2);
                const uint8_t *kb = c.k + block * 16 * d, *vb = c.v + block * 16 * d;
#pragma unroll
                for (int j = 0; j < KP; ++j) {
                    r.k[blk][j] = cache_load<STREAM>(
                        kb + (FULL ? k_at + j * 64 : row16 * d + min(j * 64 + grp * 16, d - 16)));
                    r.v[blk][j] = cache_load<STREAM>(
                        vb + (FULL ? v_at + j * 256 : grp * d * 4 + min(j * 64 + row16 * 4, d - 4) * 4));
                }
            }
        };

        float m_run[NT], l_run[NT];
        floatx4_t o[NT][KP * 4];  // O[row 4*grp+i][dim 64*(sl/4) + 4*row16 + sl%4]
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            m_run[t] = -__FLT_MAX__;
            l_run[t] = 0.0f;
#pragma unroll
            for (int sl = 0; sl < KP * 4; ++sl) o[t][sl] = floatx4_t{0.0f, 0.0f, 0.0f, 0.0f};
        }

        auto compute_tile = [&](TileRegs<KP> &r, Pages pg, int t0) {
            floatx4_t s[NT][2];
#pragma unroll
            for (int blk = 0; blk < 2; ++blk) {
#pragma unroll
                for (int t = 0; t < NT; ++t) s[t][blk] = floatx4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int j = 0; j < KP; ++j)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        bf16x8_t kf = widen8<FMT>(r.k[blk][j][2 * h], r.k[blk][j][2 * h + 1]);
                        if (!FULL && j * 64 + grp * 16 >= d) kf = bf16x8_t{};
#pragma unroll
                        for (int t = 0; t < NT; ++t)
                            s[t][blk] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[t][j][h], s[t][blk], 0, 0, 0);
                    }
                const float ks = r.scale[blk].x * a.scale_log2e;
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[t][blk][i] *= ks;
            }
            // Tokens that a row does not see weigh nothing, whatever their K
            // and scales hold; V of tokens that no row sees is zeroed.
            if (t0 + kTile > first_limit || !known(pg.p[0]) || !known(pg.p[1])) {
#pragma unroll
                for (int blk = 0; blk < 2; ++blk) {
                    const int at = t0 + blk * 16 + grp * 4;
                    const int fill = known(pg.p[blk]) ? min(max(len - at, 0), 4) : 0;
                    const uint32_t keep = fill == 4 ? 0xffffffffu : (1u << (8 * fill)) - 1;
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (i >= fill || at + i >= limit[t]) s[t][blk][i] = -INFINITY;
#pragma unroll
                    for (int j = 0; j < KP; ++j) r.v[blk][j] &= keep;
                }
            }
            bf16x8_t p[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                float mx = fmaxf(fmaxf(fmaxf(s[t][0][0], s[t][0][1]), fmaxf(s[t][0][2], s[t][0][3])),
                                 fmaxf(fmaxf(s[t][1][0], s[t][1][1]), fmaxf(s[t][1][2], s[t][1][3])));
                mx = wave_xor_max(mx, 16);
                mx = wave_xor_max(mx, 32);
                const float m_new = fmaxf(m_run[t], mx);
                if (wave_any(m_new > m_run[t])) {
                    const float alpha = __builtin_amdgcn_exp2f(m_run[t] - m_new);
                    l_run[t] *= alpha;
                    m_run[t] = m_new;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float ai = __shfl(alpha, 4 * grp + i, 64);
#pragma unroll
                        for (int sl = 0; sl < KP * 4; ++sl) o[t][sl][i] *= ai;
                    }
                }
                float psum = 0.0f;
#pragma unroll
                for (int blk = 0; blk < 2; ++blk)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float x = s[t][blk][i];
                        const float pr = round_bf16(__builtin_amdgcn_exp2f(x - m_run[t]));
                        psum += pr;
                        // a NaN scale of tokens that the row does not see stays out
                        p[t][blk * 4 + i] = (__bf16)(x == -INFINITY ? 0.0f : pr * r.scale[blk].y);
                    }
                l_run[t] += psum;
            }
#pragma unroll
            for (int sl = 0; sl < KP * 4; ++sl) {
                const bf16x8_t vf = widen8<FMT>(r.v[0][sl / 4][sl % 4], r.v[1][sl / 4][sl % 4]);
#pragma unroll
                for (int t = 0; t < NT; ++t)
                    o[t][sl] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(p[t], vf, o[t][sl], 0, 0, 0);
            }
        };

        // Ring over this wavefront's steps; past the last one the loads
        // repeat it, so every turn issues the same ones.
        if (t_first < t_end) {
            const int t_last = t_first + (t_end - 1 - t_first) / CHUNK * CHUNK;
            auto step_at = [&](int i) { return min(t_first + i * CHUNK, t_last); };
            TileRegs<KP> ring[2];
            Pages pages[3];
            pages[0] = pages_at(step_at(0));
            pages[1] = pages_at(step_at(1));
            load_tile(ring[0], pages[0], step_at(0));
            for (int base = 0; t_first + base * CHUNK < t_end; base += 2) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int t0 = t_first + (base + i) * CHUNK;
                    if (t0 >= t_end) break;
                    pages[2] = pages_at(step_at(base + i + 2));
                    load_tile(ring[1 - i], pages[1], step_at(base + i + 1));
                    __builtin_amdgcn_sched_barrier(0);
                    compute_tile(ring[i], pages[0], t0);
                    pages[0] = pages[1];
                    pages[1] = pages[2];
                }
            }
        }

        const bool alone = ch == 0 && ch_end == nch;
        const int seg_begin = a.begin[b] + seg * nch;
        const int here = min(ROWS, rows - rt * ROWS);
        // Slot of a workgroup's part: its last segment, which others go on
        // with, or its first, which others have begun.
        const int64_t slot_floats = (int64_t)ROWS * (d + 2);
        auto part = [&](int w, bool begins) { return a.partial + (2 * w + (begins ? 1 : 0)) * slot_floats; };
        float *mine = a.split ? part(owner_of(a, seg_begin + ch), ch == 0) : nullptr;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            float l = wave_xor_sum(l_run[t], 16);
            l = wave_xor_sum(l, 32);
            if (t) __syncthreads();
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < KP; ++j)
                    *reinterpret_cast<float4 *>(&comb_acc[wave][4 * grp + i][j * 64 + row16 * 4]) = make_float4(
                        o[t][j * 4][i], o[t][j * 4 + 1][i], o[t][j * 4 + 2][i], o[t][j * 4 + 3][i]);
            if (lane < 16) {
                comb_ml[wave][t * 16 + lane][0] = m_run[t];
                comb_ml[wave][t * 16 + lane][1] = l;
            }
            __syncthreads();
            for (int it = tid; it < min(16, here - t * 16) * (d / 4); it += 64 * WAVES) {
                const int r = it / (d / 4), at = it % (d / 4) * 4;
                float m = -__FLT_MAX__;
#pragma unroll
                for (int w = 0; w < WAVES; ++w) m = fmaxf(m, comb_ml[w][t * 16 + r][0]);
                float lr = 0.0f;
                float4 ov = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int w = 0; w < WAVES; ++w) {
                    const float wt = __builtin_amdgcn_exp2f(comb_ml[w][t * 16 + r][0] - m);
                    lr = fmaf(comb_ml[w][t * 16 + r][1], wt, lr);
                    const float4 y = *reinterpret_cast<const float4 *>(&comb_acc[w][r][at]);
                    ov.x = fmaf(y.x, wt, ov.x); ov.y = fmaf(y.y, wt, ov.y);
                    ov.z = fmaf(y.z, wt, ov.z); ov.w = fmaf(y.w, wt, ov.w);
                }
                if (alone) {
                    write_row(a.out + row_at(rt * ROWS + t * 16 + r) + at, ov, lr);
                } else {
                    float *to = mine + (t * 16 + r) * d + at;
                    store_coherent2(to, ov.x, ov.y);
                    store_coherent2(to + 2, ov.z, ov.w);
                    if (at == 0) store_coherent2(mine + ROWS * d + (t * 16 + r) * 2, m, lr);
                }
            }
        }
        if (alone || a.merge_launch) return;
        // The parts are ordered as the BF16 decode's are: written through to
        // the device, complete before the barrier, counted, and read past the
        // XCD's own L2 by the workgroup that counts the last.
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
        const int w0 = owner_of(a, seg_begin), parts = owner_of(a, seg_begin + nch - 1) - w0 + 1;
        if (tid == 0) {
            int *counter = a.counters + (int64_t)b * segments + seg;
            const int done = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            last_part = done == parts - 1;
            if (last_part) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        if (!last_part) return;
        merge_parts<64 * WAVES>(a, b, seg, rt * ROWS, ROWS, 0, here, d, w0, parts, tid, merge_ml, reinterpret_cast<float4 *>(comb_acc));
    };

    if (!a.split) {
        const int b = (int)(blockIdx.x / segments);
        run(b, (int)(blockIdx.x % segments), 0, chunks_of(a.len[b], WAVES));
        return;
    }
    // Row tiles of one kv head read the same bytes: they go to one XCD (that of
    // workgroups x, x + 8, ...), which takes a contiguous eighth of all.
    const int grid = (int)gridDim.x;
    const int w = a.row_tiles > 1 && grid % 8 == 0 ? (int)(blockIdx.x % 8) * (grid / 8) + (int)(blockIdx.x / 8)
                                                   : (int)blockIdx.x;
    int at = first_chunk(a, w);
    const int end = first_chunk(a, w + 1);
    for (bool again = false; at < end; again = true) {
        if (again) __syncthreads();  // the LDS of the part before is free
        int b = 0;
        for (int hi = a.batch - 1; b < hi;) {
            const int mid = (b + hi + 1) >> 1;
            if (a.begin[mid] <= at) b = mid;
            else hi = mid - 1;
        }
        const int nch = chunks_of(a.len[b], WAVES);
        const int seg = (at - a.begin[b]) / nch, ch = (at - a.begin[b]) % nch;
        const int ch_end = min(nch, ch + end - at);
        run(b, seg, ch, ch_end);
        at += ch_end - ch;
    }
}

// Bytes of K and V that a launch attends to.
int64_t cache_bytes(const Kv8AttentionLaunch &l) {
    int64_t tokens = 0;
    for (int b = 0; b < l.batch; ++b) tokens += l.len[b];
    return tokens * l.cache.kv_heads * l.cache.head_dim * 2;
}

// How a launch runs.
struct Shape {
    int nt, waves;  // row tiles of 16 at once, wavefronts of a workgroup
    bool stream;
    bool merge_launch;  // parts are merged by a launch of their own
    int row_tiles;
    int64_t segments, total, workgroups;
};

template <int FMT, int DM, bool FULL>
void launch_attention(const AttentionArgs &a, const Shape &s, unsigned grid, hipStream_t stream) {
    const dim3 block(64 * s.waves);
#define MSLIM_KV8_LAUNCH(NT, WAVES, WGS, STREAM) \
    hipLaunchKernelGGL((attention_kernel<FMT, DM, FULL, NT, WAVES, WGS, STREAM>), dim3(grid), block, 0, stream, a)
    if constexpr (DM <= 128) {
        if (s.nt == 1 && s.waves == 8 && s.stream) MSLIM_KV8_LAUNCH(1, 8, 1, true);
        else if (s.nt == 1 && s.waves == 8) MSLIM_KV8_LAUNCH(1, 8, 1, false);
        else if (s.nt == 1 && s.stream) MSLIM_KV8_LAUNCH(1, 4, 2, true);
        else if (s.nt == 1) MSLIM_KV8_LAUNCH(1, 4, 2, false);
        else if (s.waves == 8 && s.stream) MSLIM_KV8_LAUNCH(2, 8, 1, true);
        else if (s.waves == 8) MSLIM_KV8_LAUNCH(2, 8, 1, false);
        else if (s.stream) MSLIM_KV8_LAUNCH(2, 4, 2, true);
        else MSLIM_KV8_LAUNCH(2, 4, 2, false);
    } else {
        if (s.nt == 1) MSLIM_KV8_LAUNCH(1, 4, 1, false);
        else MSLIM_KV8_LAUNCH(2, 4, 1, false);
    }
#undef MSLIM_KV8_LAUNCH
}

template <int FMT, int DM>
void launch_attention(const AttentionArgs &a, const Shape &s, unsigned grid, hipStream_t stream) {
    if (a.cache.head_dim == DM) launch_attention<FMT, DM, true>(a, s, grid, stream);
    else launch_attention<FMT, DM, false>(a, s, grid, stream);
}

template <int FMT>
void launch_append(const AppendArgs &a, bool rotate, unsigned grid, hipStream_t stream) {
    const int d = a.cache.head_dim;
#define MSLIM_KV8_APPEND(NI, DIM)                                                                                  \
    if (rotate) hipLaunchKernelGGL((append_kernel<FMT, NI, true, DIM>), dim3(grid), dim3(256), 0, stream, a);     \
    else hipLaunchKernelGGL((append_kernel<FMT, NI, false, DIM>), dim3(grid), dim3(256), 0, stream, a)
    if (d == 64) { MSLIM_KV8_APPEND(1, 64); }
    else if (d == 128) { MSLIM_KV8_APPEND(2, 128); }
    else if (d == 256) { MSLIM_KV8_APPEND(4, 256); }
    else if (d < 64) { MSLIM_KV8_APPEND(1, 0); }
    else if (d < 128) { MSLIM_KV8_APPEND(2, 0); }
    else { MSLIM_KV8_APPEND(4, 0); }
#undef MSLIM_KV8_APPEND
}

}  // namespace

// Whether segments (`per` of each sequence) of workgroups of `waves`
// wavefronts are as even uncut: enough for `slots` workgroups at once and none
// much longer than its share.  There is nothing to merge then: 333 queries
// after 777 tokens, groups of seven, 35.6 -> 27.7 us.
static bool even_uncut(const Kv8AttentionLaunch &l, int64_t per, int waves, int64_t slots) {
    int64_t total = 0, longest = 0;
    for (int b = 0; b < l.batch; ++b) {
        const int64_t n = chunks_of(l.len[b], waves);
        total += n * per;
        longest = std::max(longest, n);
    }
    slots = std::min(slots, total);
    return per * l.batch >= slots && 2 * slots * longest <= 3 * total;
}

// Two tiles read and widen K and V once for both: 0.9 instead of 1.2 us per 16
// rows and 32 tokens on every wavefront.  But there are half as many segments,
// and what is cut has parts twice as large.  It pays
//   * where segments fill the device, two workgroups of four wavefronts per
//     CU: 512 queries after 512 tokens, 32/8 heads, 27.2 -> 22.6 us;
//   * where caches do not serve the second reading: five queries of 48
//     sessions, 188 MB, 59 -> 52 us, of 32 ragged ones, 284 MB, 86 -> 74;
//   * where there are nine steps or more (of 16 rows) to make up for the merge
//     and workgroups of eight wavefronts take one segment each, or cut few into
//     many parts: 16 queries of 8 sessions after 8,000 tokens 61 -> 45 us, 256
//     of one after 2,500 31.6 -> 27.5; but of 4 sessions after 4,000, eight
//     steps, 21.9 and 22.3, 5 after 20,000, five steps, 20 and 24, and 333 after
//     777, 28/4 heads, 292 segments on 256 CUs, 23 and 27.
// Over 128 dims a CU holds one workgroup of four wavefronts either way.
bool kv8_two_row_tiles(const Kv8AttentionLaunch &l) {
    const int64_t rows = (int64_t)l.queries * (l.q_heads / l.cache.kv_heads);
    if (rows <= 16) return false;
    const bool wide = l.cache.head_dim > 128;
    const int64_t per = (rows + 31) / 32 * l.cache.kv_heads, segments = per * l.batch;
    if (segments >= (wide ? kCus : 2 * kCus) || cache_bytes(l) >= kRereadBytes) return true;
    return !wide && kv8_steps(l) > kPairSteps &&
           (segments <= kCus / 2 || (segments <= kCus && even_uncut(l, per, 8, kCus)));
}

double kv8_steps(const Kv8AttentionLaunch &l) {
    const int64_t tiles = ((int64_t)l.queries * (l.q_heads / l.cache.kv_heads) + 15) / 16;
    double steps = 0.0;
    for (int b = 0; b < l.batch; ++b) steps += (double)((l.len[b] - l.queries / 2 + kTile - 1) / kTile);
    return steps * (double)tiles * l.cache.kv_heads;
}

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
    a.kv_workgroups = (uint32_t)((int64_t)l.batch * a.blocks * a.kv_groups);
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

namespace {
Shape shape_of(const Kv8AttentionLaunch &l) {
    Shape s;
    s.nt = kv8_two_row_tiles(l) ? 2 : 1;
    const int64_t rows = (int64_t)l.queries * (l.q_heads / l.cache.kv_heads);
    s.row_tiles = (int)((rows + 16 * s.nt - 1) / (16 * s.nt));
    s.segments = (int64_t)l.cache.kv_heads * s.row_tiles;
    auto chunks = [&](int waves) {
        int64_t n = 0;
        for (int b = 0; b < l.batch; ++b) n += chunks_of(l.len[b], waves) * s.segments;
        return n;
    };
    const int64_t all = s.segments * l.batch;
    const bool wide = l.cache.head_dim > 128;
    s.waves = 4;
    s.total = chunks(4);
    s.workgroups = std::min<int64_t>(s.total, wide ? kCus : 2 * kCus);
    // Two row tiles: workgroups of eight wavefronts where none goes on from one
    // segment to the next, or few do: five rows of 32 sessions of 8,000 tokens
    // 109 -> 90 us, of 32 ragged ones 74 -> 86.
    const bool eight = s.nt == 2 ? all <= kCus / 2 || (all < 2 * kCus && even_uncut(l, s.segments, 8, kCus))
                                 : s.workgroups >= kWideParts * all;
    if (!wide && eight) {
        s.waves = 8;
        s.total = chunks(8);
        // no more workgroups, in eights for the XCDs, than take the longest
        // share: fewer parts in the same time (one of 20,000 tokens 17.8 ->
        // 16.7 us; of workgroups of four wavefronts, two per CU, the CU's
        // other one hides the longer shares: 32 of 100 .. 1,000 tokens 17.4
        // and 18.3)
        const int64_t share = (s.total + kCus - 1) / kCus;
        s.workgroups = std::min<int64_t>(((s.total + share - 1) / share + 7) / 8 * 8, std::min<int64_t>(s.total, kCus));
    }
    // The workgroup that ends last merges a segment's parts at about 25 GB/s,
    // one of many at that; a launch of a workgroup per row takes 2 us and
    // another for every 512 of them: eight rows of four heads after 8,000
    // tokens, 530 KB a segment, 35.3 (fused) and 19.7 us, 66 KB of one row of
    // four heads 13.5 and 12.3, 83 KB of 32 rows of each of 64 segments 22.3
    // and 27.7.
    const int64_t parts = s.workgroups / all + 1;
    const double part_kb = (double)(parts * std::min<int64_t>(rows, 16 * s.nt) * (l.cache.head_dim + 2)) * 4 / 1024;
    s.merge_launch = part_kb * 0.04 > 2.0 + (double)(all * 16 * s.nt) / 512;
    s.stream = s.row_tiles == 1 && cache_bytes(l) >= kStreamBytes;
    return s;
}
}  // namespace

Kv8AttentionPlan kv8_attention_plan(const Kv8AttentionLaunch &l) {
    const Shape s = shape_of(l);
    Kv8AttentionPlan p{};
    if (even_uncut(l, s.segments, s.waves, l.cache.head_dim > 128 || s.waves == 8 ? kCus : 2 * kCus)) return p;
    if (s.total > INT32_MAX / 2) return p;  // positions of chunks are 32 bits
    p.split = true;
    p.partial_bytes = (size_t)(2 * s.workgroups) * 16 * s.nt * (l.cache.head_dim + 2) * sizeof(float);
    p.counters = (size_t)(s.segments * l.batch);
    return p;
}

hipError_t launch_kv8_attention(const Kv8AttentionLaunch &l, hipStream_t stream) {
    const Shape shape = shape_of(l);
    AttentionArgs a{};
    a.cache = l.cache;
    a.q = l.q; a.out = l.out;
    a.partial = l.partial; a.counters = l.counters;
    a.batch = l.batch; a.queries = l.queries; a.q_heads = l.q_heads;
    a.row_tiles = shape.row_tiles;
    a.scale_log2e = l.scale * kLog2e;
    a.split = l.split;
    a.merge_launch = l.split && shape.merge_launch;
    for (int b = 0; b < l.batch; ++b) a.len[b] = l.len[b];
    if (l.split) {
        a.share = (int)(shape.total / shape.workgroups);
        a.extra = (int)(shape.total % shape.workgroups);
        for (int b = 0; b < l.batch; ++b) a.begin[b + 1] = a.begin[b] + (int)(chunks_of(l.len[b], shape.waves) * shape.segments);
    }
    const unsigned grid = (unsigned)(l.split ? shape.workgroups : shape.segments * l.batch);
    const int d = l.cache.head_dim;
#define MSLIM_KV8_ATTENTION(FMT)                                              \
    if (d <= 64) launch_attention<FMT, 64>(a, shape, grid, stream);        \
    else if (d <= 128) launch_attention<FMT, 128>(a, shape, grid, stream); \
    else launch_attention<FMT, 256>(a, shape, grid, stream)
    if (l.cache.format == kFormatE4m3) { MSLIM_KV8_ATTENTION(kFormatE4m3); }
    else { MSLIM_KV8_ATTENTION(kFormatInt8); }
#undef MSLIM_KV8_ATTENTION
    if (hipError_t err = hipGetLastError(); err != hipSuccess || !a.merge_launch) return err;
    const int tile_rows = 16 * shape.nt;
    hipLaunchKernelGGL(merge_kernel, dim3((unsigned)(shape.segments * l.batch * tile_rows)), dim3(256), 0, stream, a,
                       tile_rows, shape.waves);
    return hipGetLastError();
}

}  // namespace mslim
