// Attention of many query rows over the 8-bit paged K/V cache: prompt chunks.
#include <algorithm>
#include <climits>
#include <type_traits>

#include "common.hpp"
#include "kernels.hpp"
#include "kv8.hpp"

namespace mslim {

namespace {

constexpr int kWaves = 8;
constexpr int kRows = 32 * kWaves;  // query rows of a workgroup at most
constexpr int kBN = 64;             // keys of a tile: four blocks
constexpr int kCus = 256;
constexpr int kXcds = 8;
// The reference maximum of a row moves only when a tile's row sum under it
// exceeds 2^8.
constexpr float kLazyBound = 256.0f;

typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

// How the segments of a launch are shared out.
constexpr int kWhole = 0, kPieces = 1, kRuns = 2;

// A segment of several parts, for the merge: workgroups w0, w0 + 1, ... took
// `count` parts; 0 where there is nothing to merge.
struct Part {
    int b, head, rt, w0, count;
};

struct PrefillArgs {
    Kv8Cache cache;
    const uint16_t *q;
    uint16_t *out;
    float2 *partial;  // [2 * workgroups][wavefront][pair][64]: O, then (m, l)
    Part *parts;      // kPieces: [segments], kRuns: [workgroups]
    int batch, queries, q_heads;
    int tile_queries;  // queries of a row tile: kRows / group
    int row_tiles;
    float scale_log2e;
    // Segments (sequence, kv head, row tile) laid end to end, by mode:
    //   kWhole   a workgroup per segment;
    //   kPieces  a workgroup per piece of a segment, of `quota` tiles at most;
    //   kRuns    workgroup w takes `share` tiles (one more for the first
    //            `extra` workgroups) from first_tile(w) on.
    int mode;
    int quota, share, extra, workgroups;
    int begin[kKv8Batch + 1];   // first tile (kPieces: piece) of each sequence
    int per_head[kKv8Batch];    // tiles (kPieces: pieces) of one kv head of each sequence
    int prior[kKv8Batch];
};

// Tiles of row tile rt of a sequence: up to the last key its last row sees.
__host__ __device__ inline int tiles_of(int prior, int queries, int tile_queries, int rt) {
    const int64_t end = prior + ((int64_t)(rt + 1) * tile_queries < queries ? (int64_t)(rt + 1) * tile_queries
                                                                            : (int64_t)queries);
    return (int)((end + kBN - 1) / kBN);
}

// Of a scale that the whole wavefront shares: a scalar test.
__device__ __forceinline__ bool finite(float scale) {
    return (__builtin_amdgcn_readfirstlane(__float_as_uint(scale)) & 0x7f800000u) != 0x7f800000u;
}

// First tile of workgroup w, and the workgroup that takes a tile.
__device__ __forceinline__ int first_tile(const PrefillArgs &a, int w) { return w * a.share + min(w, a.extra); }
__device__ __forceinline__ int owner_of(const PrefillArgs &a, int tile) {
    const int more = a.extra * (a.share + 1);  // tiles of the workgroups with one more
    return tile < more ? tile / (a.share + 1) : a.extra + (tile - more) / a.share;
}
// A wavefront's share of a workgroup's part: of its last segment, which others
// go on with (begins), or of its first.
__device__ __forceinline__ float2 *part_at(const PrefillArgs &a, int w, bool begins, int wave, int pairs) {
    return a.partial + (int64_t)((2 * w + (begins ? 1 : 0)) * kWaves + wave) * pairs * 64;
}

// Bytes times a scale as BF16.  A power of two, what the append writes, is
// exact; E4M3 takes it in the conversion.
template <int FMT>
__device__ __forceinline__ void widen_scaled(const u32x4_t &w, float scale, uint4 (&out)[2]) {
    uint32_t o[8];
    if (FMT == kFormatE4m3 &&
        __builtin_expect((__builtin_amdgcn_readfirstlane(__float_as_uint(scale)) & 0x7fffffu) == 0, 1)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            o[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], scale, false));
            o[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], scale, true));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            o[2 * i] = pack_bf16x2(byte_value<FMT>(w[i], 0) * scale, byte_value<FMT>(w[i], 1) * scale);
            o[2 * i + 1] = pack_bf16x2(byte_value<FMT>(w[i], 2) * scale, byte_value<FMT>(w[i], 3) * scale);
        }
    }
    out[0] = make_uint4(o[0], o[1], o[2], o[3]);
    out[1] = make_uint4(o[4], o[5], o[6], o[7]);
}

// A workgroup of eight wavefronts takes the rows of tile_queries queries and
// all heads of one kv head's group (32 rows per wavefront) over a run of
// 64-key tiles:
//   * a tile's bytes come in registers, 16 of K and 16 of V per lane, go out
//     to LDS as BF16 once for all rows, times their block's scale (exact: a
//     power of two), one tile ahead of use, and the loads one tile ahead of
//     that;
//   * S^T = K.Q^T on v_mfma_f32_32x32x16_bf16 (keys as M, a wavefront's rows
//     as N).  The accumulator has one row per lane, in the operand layout of
//     O^T = V^T.P^T, so P stays in registers and softmax, rescale and mask are
//     per-lane operations;
//   * the V^T operand's eight keys of a dim are two runs of four: the cache
//     keeps four tokens of a dim side by side, so a fragment is two 8-byte
//     reads without a transposition;
//   * VALU work hides under MFMAs of the same wavefront only: the softmax of
//     tile j runs in the slots of P.V of tile j - 1, the widening of tile
//     j + 1 in those of Q.K of tile j;
//   * the scores take scale * log2(e) and lose the row's reference maximum in
//     one f32 FMA; P is rounded to BF16 for its product with V and the row
//     sum adds the rounded P;
//   * O is rescaled only when a tile's row sum under the reference exceeds
//     2^8 (exact: O / l has the same reference);
//   * a block whose scale is not finite enters as V zeros and K NaN: rows that
//     see it get NaN, and the masked ones, whose P is zero, do not.
template <int FMT, int DM, bool FULL>
__global__ __launch_bounds__(512, 1) void kv8_prefill_kernel(PrefillArgs a) {
    constexpr int KS = DM / 16;        // Q.K MFMA k-steps
    constexpr int MT = DM / 32;        // P.V output tiles of 32 dims
    constexpr int NS = 4 * MT;         // P.V MFMAs of a tile
    constexpr int NSLOT = DM / 8;      // 16-byte slots of a K row in LDS
    constexpr int PIECES = kBN * DM / 16;  // 16-byte pieces of a tile's K (and V) bytes: 512 or 256
    constexpr int PAIRS = MT * 8 + 1;
    __shared__ __align__(256) uint16_t k_lds[2][kBN * DM];
    __shared__ __align__(16) uint16_t v_lds[4][kBN * DM];  // [block][4][dim][4 tokens]

    const Kv8Cache &c = a.cache;
    const int d = FULL ? DM : c.head_dim;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 31, half = lane >> 5;
    const int group = a.q_heads / c.kv_heads;
    const float sc = a.scale_log2e;

    // This lane's pieces of a tile: K piece = 16 dims of a row, V piece = 4
    // dims of four tokens.  Both lie in one block, the same for the wavefront.
    // DM 64: the first four wavefronts take K, the others V.
    const bool has_k = PIECES == 512 || wave < 4, has_v = PIECES == 512 || wave >= 4;
    const int piece = tid & (PIECES - 1);
    const int my_block = __builtin_amdgcn_readfirstlane(PIECES == 512 ? wave >> 1 : wave & 3);
    const int k_row = piece / (DM / 16), k_dim = piece % (DM / 16) * 16;
    const int v_grp = piece % (DM) / (DM / 4), v_dim = piece % (DM / 4) * 4;
    const bool k_in = FULL || k_dim < d, v_in = FULL || v_dim < d;
    const int k_off = (k_row & 15) * d + min(k_dim, d - 16), v_off = (v_grp * d + min(v_dim, d - 4)) * 4;
    auto k_slot = [](int row, int slot) { return slot ^ (row & (NSLOT - 1)); };
    uint16_t *const k_to0 = &k_lds[0][k_row * DM + k_slot(k_row, k_dim / 8) * 8];
    uint16_t *const k_to1 = &k_lds[0][k_row * DM + k_slot(k_row, k_dim / 8 + 1) * 8];
    uint16_t *const v_to = &v_lds[0][((piece / DM * 4 + v_grp) * DM + v_dim) * 4];

    // Fragment addresses in stage 0; a stage and a block of rows are immediates.
    // A K fragment's slot is (2 ks + half) ^ (row % NSLOT): k-step ks flips bits
    // of the address of the first.
    const uint32_t k_from = lds_offset(k_lds) + (uint32_t)(col * DM + k_slot(col, half) * 8) * 2;
    const uint32_t v_from = lds_offset(v_lds) + (uint32_t)(half * DM + col) * 8;
    constexpr uint32_t STAGE = kBN * DM * 2;

    auto run = [&](int b, int head, int rt, int tile, int tile_end, int tiles, int w)
        __attribute__((always_inline)) {
        const int prior = a.prior[b];
        const int len = prior + a.queries;
        const int r = wave * 32 + col;  // row of the tile: (query r / group, head r % group)
        const int query = rt * a.tile_queries + r / group;
        const bool live = r < a.tile_queries * group && query < a.queries;
        const int limit = live ? prior + query + 1 : 0;
        // keys that every row of the wavefront sees
        const int common = prior + rt * a.tile_queries + wave * 32 / group + 1;
        const int64_t row_at =
            (((int64_t)b * a.queries + (live ? query : 0)) * a.q_heads + head * group + r % group) * d;
        bf16x8_t qf[KS];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const int at = ks * 16 + half * 8;
            qf[ks] = bf16x8_t{};
            if (live && (FULL || at < d)) qf[ks] = *reinterpret_cast<const bf16x8_t *>(a.q + row_at + at);
        }

        // Pages of a tile's four blocks; a block past the end repeats the last.
        const int32_t *table = c.table + (int64_t)b * c.pages_per_seq;
        const int last_block = (len - 1) & ~15;
        struct Pages {
            int p[4];
        };
        auto block_at = [&](int t, int i) { return min(t * kBN + i * 16, last_block); };
        auto pages_at = [&](int t) {
            Pages pg;
#pragma unroll
            for (int i = 0; i < 4; ++i) pg.p[i] = scalar_page(table + (block_at(t, i) >> c.shift));
            return pg;
        };
        auto known = [&](int page) { return page >= 0 && page < (int)c.pool_pages; };
        auto all_known = [&](const Pages &pg) {
            return known(pg.p[0]) && known(pg.p[1]) && known(pg.p[2]) && known(pg.p[3]);
        };
        u32x4_t k_in_regs = {}, v_in_regs = {};
        float2 scale = make_float2(0.0f, 0.0f);
        bool no_page = false;  // the loaded bytes are another page's
        auto load = [&](const Pages &pg, int t) __attribute__((always_inline)) {
            const int pick = my_block == 0 ? pg.p[0] : my_block == 1 ? pg.p[1] : my_block == 2 ? pg.p[2] : pg.p[3];
            no_page = !known(pick);
            const int64_t page = no_page ? 0 : pick;
            const int64_t block = ((page * c.kv_heads + head) << (c.shift - 4)) +
                                  ((block_at(t, my_block) & ((1 << c.shift) - 1)) >> 4);
            scale = scalar_scales(c.scales + block * 2);
            if (has_k) k_in_regs = *reinterpret_cast<const u32x4_t *>(c.k + block * 16 * d + k_off);
            if (has_v) v_in_regs = *reinterpret_cast<const u32x4_t *>(c.v + block * 16 * d + v_off);
        };
        // The loaded tile to K stage ks and V stage vs.  V bytes behind the
        // last token, or of no page, become zeros; K's are masked.
        // (Scales are the same for the wavefront, so their cases are branches.)
        auto store_k = [&](int ks) __attribute__((always_inline)) {
            if (!has_k) return;
            uint4 w[2];
            widen_scaled<FMT>(k_in ? k_in_regs : u32x4_t{0, 0, 0, 0}, scale.x, w);
            if (!finite(scale.x) || !finite(scale.y))
                w[0] = w[1] = make_uint4(0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u);
            *reinterpret_cast<uint4 *>(k_to0 + ks * kBN * DM) = w[0];
            *reinterpret_cast<uint4 *>(k_to1 + ks * kBN * DM) = w[1];
        };
        auto store_v = [&](int vs, int t) __attribute__((always_inline)) {
            if (!has_v) return;
            uint4 w[2] = {};
            if (!no_page && finite(scale.y)) {
                u32x4_t bytes = v_in ? v_in_regs : u32x4_t{0, 0, 0, 0};
                if (__builtin_expect(t * kBN + kBN > len, 0)) {
                    const int fill = min(max(len - (t * kBN + my_block * 16 + v_grp * 4), 0), 4);
                    bytes &= fill == 4 ? 0xffffffffu : (1u << (8 * fill)) - 1;
                }
                widen_scaled<FMT>(bytes, scale.y, w);
            }
            *reinterpret_cast<uint4 *>(v_to + vs * kBN * DM) = w[0];
            *reinterpret_cast<uint4 *>(v_to + vs * kBN * DM + 8) = w[1];
        };

        floatx16_t o[MT];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[mt][i] = 0.0f;
        float m_used = -__FLT_MAX__, l_run = 0.0f, alpha = 1.0f;
        bool rescale = false;
        floatx16_t s[2];
        bf16x8_t p[2][2] = {};  // [key half of 32][16 of them]

        // Scores of the tile in K stage st; `mid(n)` after MFMA n.
        auto qk = [&](int st, auto &&mid) __attribute__((always_inline)) {
            const uint32_t from = k_from + st * STAGE;
            auto frag = [&](int n) __attribute__((always_inline)) {
                return lds_read_b128((from ^ (uint32_t)(n / 2 * 32)) + n % 2 * 32 * DM * 2);
            };
            bf16x8_t kq[3];
            kq[0] = frag(0);
            kq[1] = frag(1);
#pragma unroll
            for (int n = 0; n < 2 * KS; ++n) {
                if (n + 2 < 2 * KS) kq[(n + 2) % 3] = frag(n + 2);
                __builtin_amdgcn_sched_barrier(0);
                if (n < 2) {
                    floatx16_t zero;
#pragma unroll
                    for (int i = 0; i < 16; ++i) zero[i] = 0.0f;
                    s[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kq[n], qf[0], zero, 0, 0, 0);
                } else {
                    s[n % 2] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kq[n % 3], qf[n / 2], s[n % 2], 0, 0, 0);
                }
                mid(n);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        // Key of element (kb, i) in its tile: kb * 32 + (i >> 2) * 8 + half * 4 + (i & 3).
        auto mask = [&](int t, const Pages &pg) __attribute__((always_inline)) {
            if (__builtin_expect(t * kBN + kBN > common, 0)) {
                const int most = limit - 1 - t * kBN - half * 4;
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (kb * 32 + (i >> 2) * 8 + (i & 3) > most) s[kb][i] = -INFINITY;
            }
            if (__builtin_expect(!all_known(pg), 0)) {
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (!known(pg.p[kb * 2 + i / 8])) s[kb][i] = -INFINITY;
            }
        };
        auto row_max = [&]() __attribute__((always_inline)) {
            float mx = s[0][0];
#pragma unroll
            for (int i = 1; i < 16; ++i) mx = __builtin_fmaxf(mx, s[0][i]);
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = __builtin_fmaxf(mx, s[1][i]);
            return half_pair_max(mx) * sc;
        };
        uint32_t pw[2][8];
        float psum = 0.0f;
        auto score_pair = [&](int n) __attribute__((always_inline)) {
            const int kb = n / 8, i = n % 8 * 2;
            bf16x2_t pp;
            pp[0] = (__bf16)__builtin_amdgcn_exp2f(fmaf(s[kb][i], sc, -m_used));
            pp[1] = (__bf16)__builtin_amdgcn_exp2f(fmaf(s[kb][i + 1], sc, -m_used));
            pw[kb][n % 8] = __builtin_bit_cast(uint32_t, pp);
            psum = add_bf16_pair(pp, psum);
            pin_value(pw[kb][n % 8]);
        };
        // Every p is at most its tile's row sum, so the reference stays while
        // that is within the bound; else the rows whose maximum exceeds it
        // move it and the tile's P is taken again.
        auto settle = [&]() __attribute__((always_inline)) {
            if (__builtin_expect(wave_any(!(psum <= kLazyBound)), 0)) {
                const float m_new = fmaxf(row_max(), m_used);
                alpha = __builtin_amdgcn_exp2f(m_used - m_new);
                l_run *= alpha;
                m_used = m_new;
                rescale = true;
                psum = 0.0f;
#pragma unroll
                for (int n = 0; n < 16; ++n) score_pair(n);
            }
            l_run += psum;
        };
        auto keep_p = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int t = 0; t < 2; ++t)
                    p[kb][t] = __builtin_bit_cast(
                        bf16x8_t, make_uint4(pw[kb][4 * t], pw[kb][4 * t + 1], pw[kb][4 * t + 2], pw[kb][4 * t + 3]));
        };
        // P.V of the tile in V stage st, with the softmax of the current
        // scores spread over its MFMAs where SOFTMAX.
        auto pv = [&](int st, auto softmax) __attribute__((always_inline)) {
            constexpr bool SOFTMAX = decltype(softmax)::value;
            auto frag = [&](int n) __attribute__((always_inline)) {
                const int mt = n % MT, t = n / MT;  // block of 16 keys
                const uint32_t at = v_from + st * STAGE + t * 4 * DM * 8 + mt * 32 * 8;
                const u32x2_t lo = *(const __attribute__((address_space(3))) u32x2_t *)(uintptr_t)at;
                const u32x2_t hi = *(const __attribute__((address_space(3))) u32x2_t *)(uintptr_t)(at + 2 * DM * 8);
                return __builtin_bit_cast(bf16x8_t, u32x4_t{lo[0], lo[1], hi[0], hi[1]});
            };
            if constexpr (SOFTMAX) psum = 0.0f;
            bf16x8_t vq[3];
            vq[0] = frag(0);
            vq[1] = frag(1);
#pragma unroll
            for (int n = 0; n < NS; ++n) {
                if (n + 2 < NS) vq[(n + 2) % 3] = frag(n + 2);
                __builtin_amdgcn_sched_barrier(0);
                o[n % MT] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vq[n % 3], p[n / MT / 2][n / MT % 2], o[n % MT], 0, 0, 0);
                if constexpr (SOFTMAX) {
#pragma unroll
                    for (int k = 0; k < 16; ++k)
                        if (k * NS / 16 == n) score_pair(k);
                    pin_value(psum);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        // All wavefronts' LDS accesses before it are done; global loads stay
        // in flight.
        auto barrier = [&]() __attribute__((always_inline)) {
            asm volatile("" ::: "memory");
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_waitcnt(0xF | (3 << 14) | (0x7 << 4));  // lgkmcnt 0
            raw_barrier();
            __builtin_amdgcn_sched_barrier(0);
            asm volatile("" ::: "memory");
        };

        const int last_tile = tile_end - 1;
        auto clamp = [&](int t) { return min(t, last_tile); };
        Pages pg0 = pages_at(tile), pg1 = pages_at(clamp(tile + 1)), pg2 = pages_at(clamp(tile + 2));
        load(pg0, tile);
        store_k(0);
        store_v(0, tile);
        load(pg1, clamp(tile + 1));
        barrier();
        auto apply_rescale = [&]() __attribute__((always_inline)) {
            if (!rescale) return;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[mt][i] *= alpha;
            rescale = false;
        };
        int n = 0;  // tiles done; K of tile j is in stage n % 2, V in n % 4
        // Q.K of tile j, and tile j + 1 to LDS on the way
        auto scores = [&](int j) __attribute__((always_inline)) {
            qk(n & 1, [&](int m) __attribute__((always_inline)) {
                if (m == 3) store_k(~n & 1);
                if (m == KS + 1) store_v((n + 1) & 3, clamp(j + 1));
                if (m == 2 * KS - 2) load(pg2, clamp(j + 2));
            });
            mask(j, pg0);
        };
        auto next = [&](int j) __attribute__((always_inline)) {
            pg0 = pg1;
            pg1 = pg2;
            pg2 = pages_at(clamp(j + 2));
            ++n;
            barrier();
        };
        // Softmax of the scores at hand with P.V of the tile before them; a
        // run's first has P = 0 and takes its own V.
        auto softmax_pv = [&](int before) __attribute__((always_inline)) {
            apply_rescale();
            pv(max(before, 0) & 3, std::true_type{});
            settle();
            keep_p();
        };
        for (int j = tile;;) {
            scores(j);
            softmax_pv(n - 1);
            if (++j == tile_end) break;
            next(j);
        }
        apply_rescale();
        pv(n & 3, std::false_type{});

        float l = l_run + __shfl_xor(l_run, 32, 64);
        auto write_out = [&](const floatx16_t *acc, float lsum) __attribute__((always_inline)) {
            if (!live) return;
            const float inv = lsum == 0.0f ? 0.0f : 1.0f / lsum;  // a row that sees nothing is zeros
            uint16_t *op = a.out + row_at + half * 4;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int i4 = 0; i4 < 4; ++i4) {
                    uint2 w;
                    w.x = pack_bf16x2(acc[mt][i4 * 4] * inv, acc[mt][i4 * 4 + 1] * inv);
                    w.y = pack_bf16x2(acc[mt][i4 * 4 + 2] * inv, acc[mt][i4 * 4 + 3] * inv);
                    if (FULL || mt * 32 + i4 * 8 < d) *reinterpret_cast<uint2 *>(op + mt * 32 + i4 * 8) = w;
                }
        };
        if (tile == 0 && tile_end == tiles) {
            write_out(o, l);
            return;
        }
        // A part of a segment, for the merge launch.
        float2 *mine = part_at(a, w, tile == 0, wave, PAIRS) + lane;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int i = 0; i < 8; ++i) mine[(mt * 8 + i) * 64] = make_float2(o[mt][2 * i], o[mt][2 * i + 1]);
        mine[MT * 8 * 64] = make_float2(m_used, l);
    };

    // Workgroup -> run of tiles: XCD x (workgroups x, x + 8, ...) takes a
    // contiguous eighth of all, so the kv heads that it reads stay in its L2.
    // One call of run() for all modes: a cold workgroup's time is the fetching
    // of its instructions.
    const int w = a.workgroups % kXcds || a.mode == kWhole
                      ? (int)blockIdx.x
                      : (int)(blockIdx.x % kXcds) * (a.workgroups / kXcds) + (int)(blockIdx.x / kXcds);
    int b = 0, head, rt = 0, seg_begin = 0, tiles, at, end;
    if (a.mode == kWhole) {
        rt = w % a.row_tiles;
        head = w / a.row_tiles % c.kv_heads;
        b = w / a.row_tiles / c.kv_heads;
        tiles = tiles_of(a.prior[b], a.queries, a.tile_queries, rt);
        at = 0;
        end = tiles;
    } else {
        at = a.mode == kPieces ? w : first_tile(a, w);
        for (int hi = a.batch - 1; b < hi;) {
            const int mid = (b + hi + 1) >> 1;
            if (a.begin[mid] <= at) b = mid;
            else hi = mid - 1;
        }
        head = (at - a.begin[b]) / a.per_head[b];
        seg_begin = a.begin[b] + head * a.per_head[b];
        tiles = tiles_of(a.prior[b], a.queries, a.tile_queries, 0);
        const int quota = a.mode == kPieces ? a.quota : 1;
        int pieces = (tiles + quota - 1) / quota;
        while (seg_begin + pieces <= at) {
            seg_begin += pieces;
            tiles = tiles_of(a.prior[b], a.queries, a.tile_queries, ++rt);
            pieces = (tiles + quota - 1) / quota;
        }
        if (a.mode == kPieces) {
            const int i = at - seg_begin;
            if (tid == 0 && i == 0)
                a.parts[(b * c.kv_heads + head) * a.row_tiles + rt] = Part{b, head, rt, w, pieces > 1 ? pieces : 0};
            seg_begin = 0;
            at = i * (tiles / pieces) + min(i, tiles % pieces);
            end = (i + 1) * (tiles / pieces) + min(i + 1, tiles % pieces);
        } else {
            end = first_tile(a, w + 1);
        }
    }
    Part begun = {};
    for (;;) {
        const int tile = at - seg_begin, tile_end = min(tiles, end - seg_begin);
        if (a.mode == kRuns && tile == 0 && tile_end < tiles)
            begun = Part{b, head, rt, w, owner_of(a, seg_begin + tiles - 1) - w + 1};
        run(b, head, rt, tile, tile_end, tiles, w);
        at = seg_begin + tile_end;
        if (at >= end) break;
        __syncthreads();  // the LDS of this part is free
        seg_begin += tiles;
        if (++rt == a.row_tiles) {
            rt = 0;
            if (++head == c.kv_heads) {
                head = 0;
                b = min(b + 1, a.batch - 1);
            }
        }
        tiles = tiles_of(a.prior[b], a.queries, a.tile_queries, rt);
    }
    if (a.mode == kRuns && tid == 0) a.parts[w] = begun;
}

// Merges the parts of a segment in the order of its keys: a wavefront per 32
// rows and 32 dims.  (The workgroup that ends last, alone with all rows, took
// 5 us per part of 133 KB.)
template <int MT>
__global__ __launch_bounds__(64) void merge_kernel(PrefillArgs a) {
    constexpr int PAIRS = MT * 8 + 1;
    constexpr int K = 4;  // parts whose loads go out together
    const int mt = (int)(blockIdx.x % MT), wave = (int)(blockIdx.x / MT % kWaves);
    const Part seg = a.parts[blockIdx.x / MT / kWaves];
    const int b = seg.b, head = seg.head, rt = seg.rt, w0 = seg.w0, parts = seg.count;
    if (parts == 0) return;
    const int lane = threadIdx.x;
    const int group = a.q_heads / a.cache.kv_heads, d = a.cache.head_dim;
    const int r = wave * 32 + (lane & 31), query = rt * a.tile_queries + r / group;
    if (r >= a.tile_queries * group || query >= a.queries) return;
    float m = -__FLT_MAX__, l = 0.0f;
    float2 o[8] = {};
    for (int j = 0; j < parts; j += K) {
        float2 x[K][8], ml[K];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int p = min(j + k, parts - 1);
            const float2 *from = part_at(a, w0 + p, p == 0, wave, PAIRS) + lane;
            ml[k] = from[MT * 8 * 64];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[k][i] = from[(mt * 8 + i) * 64];
        }
        float m_new = m;
#pragma unroll
        for (int k = 0; k < K; ++k) m_new = fmaxf(m_new, ml[k].x);
        const float keep = __builtin_amdgcn_exp2f(m - m_new);
        m = m_new;
        l *= keep;
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = make_float2(o[i].x * keep, o[i].y * keep);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (j + k >= parts) continue;
            const float w = __builtin_amdgcn_exp2f(ml[k].x - m);
            l = fmaf(ml[k].y, w, l);
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = make_float2(fmaf(x[k][i].x, w, o[i].x), fmaf(x[k][i].y, w, o[i].y));
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    uint16_t *op = a.out + (((int64_t)b * a.queries + query) * a.q_heads + head * group + r % group) * d + mt * 32 +
                   (lane >> 5) * 4;
#pragma unroll
    for (int i4 = 0; i4 < 4; ++i4) {
        uint2 w;
        w.x = pack_bf16x2(o[2 * i4].x * inv, o[2 * i4].y * inv);
        w.y = pack_bf16x2(o[2 * i4 + 1].x * inv, o[2 * i4 + 1].y * inv);
        if (mt * 32 + i4 * 8 < d) *reinterpret_cast<uint2 *>(op + i4 * 8) = w;
    }
}

struct Shape {
    int tile_queries, row_tiles;
    int64_t total, segments;
    int mode, quota, workgroups;
    int64_t begin[kKv8Batch + 1], per_head[kKv8Batch];
};
Shape shape_of(const Kv8AttentionLaunch &l) {
    Shape s{};
    s.tile_queries = kRows / (l.q_heads / l.cache.kv_heads);
    s.row_tiles = (l.queries + s.tile_queries - 1) / s.tile_queries;
    s.segments = (int64_t)l.batch * l.cache.kv_heads * s.row_tiles;
    // tiles (pieces of at most `quota`, where given) of all segments
    auto lay = [&](int quota) {
        for (int b = 0; b < l.batch; ++b) {
            int64_t n = 0;
            for (int rt = 0; rt < s.row_tiles; ++rt) {
                const int tiles = tiles_of(l.len[b] - l.queries, l.queries, s.tile_queries, rt);
                n += quota ? (tiles + quota - 1) / quota : tiles;
            }
            s.per_head[b] = n;
            s.begin[b + 1] = s.begin[b] + n * l.cache.kv_heads;
        }
        return s.begin[l.batch];
    };
    s.total = lay(0);
    if (s.segments <= kCus) {
        // The size of a piece with the shortest call, of those that leave no
        // more pieces than CUs: a tile takes a workgroup 2 us, a part 0.06 us
        // of the device's bandwidth (133 KB written and read) and 0.2 us in
        // the merge's chain.
        s.mode = kPieces;
        int longest = 1;
        for (int b = 0; b < l.batch; ++b)
            longest = std::max(longest, tiles_of(l.len[b] - l.queries, l.queries, s.tile_queries, s.row_tiles - 1));
        double best = 0.0;
        for (int q = (int)std::max<int64_t>(1, s.total / kCus); q <= longest; q += 1 + q / 16) {
            const int64_t pieces = lay(q);
            if (pieces > kCus) continue;
            const double cost = 2.0 * q + 0.06 * (double)pieces + 0.2 * ((longest + q - 1) / q);
            if (!s.quota || cost < best) {
                best = cost;
                s.quota = q;
            }
        }
        if (!s.quota) s.quota = longest;
        s.workgroups = (int)lay(s.quota);
    } else {
        s.mode = s.total > INT32_MAX / 2 ? kWhole : kRuns;  // positions of tiles are 32 bits
        s.workgroups = (int)std::min<int64_t>(s.total, kCus);
    }
    return s;
}

template <int FMT, int DM>
void launch(const PrefillArgs &a, unsigned grid, hipStream_t stream) {
    if (a.cache.head_dim == DM)
        hipLaunchKernelGGL((kv8_prefill_kernel<FMT, DM, true>), dim3(grid), dim3(512), 0, stream, a);
    else
        hipLaunchKernelGGL((kv8_prefill_kernel<FMT, DM, false>), dim3(grid), dim3(512), 0, stream, a);
}

}  // namespace

// The other kernel takes 16 rows and 32 tokens a step, on 2,048 wavefronts at
// once, 1.2 us each or, two row tiles at a time, 0.9 us; this one's 0.5 us per
// such step have to make up for its fixed 26 us.  E4M3: 400 queries after 1,000
// tokens, 32/8 heads, 15 steps, 32 us there and 33 here; 333 after 1,777, 28/4
// heads, 17 steps, 37 and 32; two at a time 512 after 1,024, 20 steps, 30 and
// 35; 1,024 after 256, 24 steps, 43 and 40; 256 after 4,000, 32 steps, still 38
// and 41.  Up to 64 rows a kv head most of a workgroup here would idle: 8
// queries of 32 sessions, 64/8 heads, 117 and 249 us.
bool kv8_prefill_supported(const Kv8AttentionLaunch &l) {
    const int group = l.q_heads / l.cache.kv_heads;
    const int64_t rows = (int64_t)l.queries * group;
    if (l.cache.head_dim > 128 || group > kRows || rows <= 64) return false;
    return kv8_steps(l) > (kv8_two_row_tiles(l) ? 24 : 16) * 2048;
}

namespace {
size_t part_bytes(const Kv8AttentionLaunch &l, const Shape &s) {
    const size_t pairs = (l.cache.head_dim <= 64 ? 2 : 4) * 8 + 1;
    return (size_t)(2 * s.workgroups) * kWaves * pairs * 64 * sizeof(float2);
}
size_t merges(const Shape &s) { return s.mode == kPieces ? (size_t)s.segments : (size_t)s.workgroups; }
}  // namespace

Kv8AttentionPlan kv8_prefill_plan(const Kv8AttentionLaunch &l) {
    const Shape s = shape_of(l);
    Kv8AttentionPlan p{};
    if (s.mode == kWhole) return p;
    p.split = true;
    p.partial_bytes = part_bytes(l, s) + merges(s) * sizeof(Part);
    return p;
}

hipError_t launch_kv8_prefill(const Kv8AttentionLaunch &l, hipStream_t stream) {
    const Shape s = shape_of(l);
    PrefillArgs a{};
    a.cache = l.cache;
    a.q = l.q; a.out = l.out;
    a.partial = reinterpret_cast<float2 *>(l.partial);
    a.batch = l.batch; a.queries = l.queries; a.q_heads = l.q_heads;
    a.tile_queries = s.tile_queries;
    a.row_tiles = s.row_tiles;
    a.scale_log2e = l.scale * kLog2e;
    a.mode = l.split ? s.mode : kWhole;
    a.quota = s.quota;
    a.workgroups = s.workgroups;
    a.share = (int)(s.total / s.workgroups);
    a.extra = (int)(s.total % s.workgroups);
    if (l.split) a.parts = reinterpret_cast<Part *>(reinterpret_cast<char *>(l.partial) + part_bytes(l, s));
    for (int b = 0; b < l.batch; ++b) {
        a.begin[b + 1] = (int)s.begin[b + 1];  // split launches only
        a.per_head[b] = (int)s.per_head[b];
        a.prior[b] = l.len[b] - l.queries;
    }
    const unsigned grid = (unsigned)(l.split ? s.workgroups : s.segments);
#define MSLIM_KV8_PREFILL(FMT)                                              \
    if (l.cache.head_dim <= 64) launch<FMT, 64>(a, grid, stream);           \
    else launch<FMT, 128>(a, grid, stream)
    if (l.cache.format == kFormatE4m3) { MSLIM_KV8_PREFILL(kFormatE4m3); }
    else { MSLIM_KV8_PREFILL(kFormatInt8); }
#undef MSLIM_KV8_PREFILL
    if (hipError_t err = hipGetLastError(); err != hipSuccess || !l.split) return err;
    if (s.mode == kPieces && s.workgroups == s.segments) return hipSuccess;  // nothing was split
    const unsigned merge = (unsigned)(merges(s) * kWaves);
    if (l.cache.head_dim <= 64) hipLaunchKernelGGL((merge_kernel<2>), dim3(merge * 2), dim3(64), 0, stream, a);
    else hipLaunchKernelGGL((merge_kernel<4>), dim3(merge * 4), dim3(64), 0, stream, a);
    return hipGetLastError();
}

}  // namespace mslim
