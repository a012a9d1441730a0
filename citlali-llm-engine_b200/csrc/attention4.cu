// Attention over the cache in 4 bits on the tensor cores: single tokens and short runs of tokens (bfloat16 queries, pages of 64 keys).
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(f q . k_j - m),  f = scale log2(e),  over the keys lo..pos that a row sees
//
// What bounds it: reading the cache, 9/8 byte a key's element with its value's.  A key and a value are read once for all query
// heads that share them, and for a run's tokens of one tile.  The codes go from memory to shared memory (cp.async, a ring a
// warp) and from there straight into operand registers; nothing is written back.
//
// Operands.  The keys are the rows of the product (m16n8k16, half operands, float sums) and the queries its columns: scores are
// S^T = K Q^T, 16 keys by 8 columns, and results are O^T += V^T P^T.  So eight columns cost half of what the other way round would,
// where 16 rows of queries would be padded.  A column is a pair (token of the tile, query head of the group).
//   K: lane (r, t) = (lane / 4, lane % 4) holds for the keys r and r + 8 the elements t D/4 .. (t + 1) D/4 - 1, as they lie in
//      memory: the order of the contraction is free as long as the queries have the same.
//   V: it holds for the keys 2t, 2t + 1, 2t + 8, 2t + 9 the elements r D/8 .. (r + 1) D/8 - 1; two keys' codes are laid side by side
//      (one byte permutation for four elements) so that a register's halves are two keys of one element.
//   P: the scores' registers hold (key r, columns 2t, 2t + 1); one movmatrix gives (column r, keys 2t, 2t + 1), the operand.
// Words.  A word holds eight codes c + 8.  (w & 0x000f000f) | 0x6400 is the half 1032 + c, (w & 0x00f000f0) | 0x5400 is 72 + c, and
// c s = (1032 + c) s - 1032 s is one fma whose operands and result are exact (cache4.cuh): four lop3, a shift and four fmas for
// eight elements.  s here is the byte's half, an eighth of the scale; the 8 comes back in f and in the last division.
// Queries are made halves after they were multiplied by a power of two that puts the row's largest into [2^14, 2^15): exact for every
// element above 2^-32 of that.  P is rounded to half (half a step is 2^-11 of it, an eighth of bfloat16's); all weights are 2^15 times
// what the formula says, which the division takes out again, so that those below 2^-14 of the largest are not subnormal halves.
//
// Work.  16 keys are a unit.  The units of all (sequence, key/value head, tile) are laid end to end and dealt out evenly to the
// blocks, whatever the sequences' lengths, which are read on the device: the launch depends on none and can be captured.  A block's
// share is made of pieces of one or more (sequence, head, tile); its eight warps take the piece's units in turn, and are merged in
// warp order.  A piece that is the whole goes to memory as the result, another as (m, l, O) in float, which a second kernel merges in
// the order of the keys.  So every sum has an order that the step's lengths fix.
#include "api.h"
#include "cache4.cuh"
#include "common.cuh"
#include "mma_common.cuh"

namespace citlali {
namespace c4 {

constexpr int kPage = 64, kUnitKeys = 16;
constexpr int kWarps4 = 8, kThreads4 = 32 * kWarps4;
constexpr float kWeightBits = 15.0f;
constexpr int kLeastUnits = 8;          // of a block's share: a unit a warp

struct Attention4 {
    const __nv_bfloat16* q;
    size_t q_stride;
    const uint8_t *k_codes, *k_scales, *v_codes, *v_scales;
    const int32_t* table;
    int table_stride;
    const int32_t *seq_start, *seq_slot, *seq_past;      // seq_start null: a row a sequence
    __nv_bfloat16* out;
    size_t out_stride;
    int sequences, nq, nkv, group;
    int tokens, heads, head_tiles;                       // of a tile; the tiles a group's heads are cut into
    int window;
    float scale_log2;
    float* partial;                                      // [blocks][2][columns][D + 2]
};

// What a sequence of the step asks for: `units` of 16 keys for each of `segments` (head tile of a key/value head, token tile).
struct Sequence {
    int past, fresh, row, first_unit, units, tiles, segments;
};
__device__ __forceinline__ Sequence sequence_of(const Attention4& a, int b) {
    Sequence s;
    s.past = a.seq_past[b];
    s.row = a.seq_start ? a.seq_start[b] : b;
    s.fresh = a.seq_start ? a.seq_start[b + 1] - s.row : 1;
    const int lo = a.window > 0 ? max(0, s.past - a.window + 1) : 0;
    s.first_unit = lo / kUnitKeys;
    s.units = s.fresh > 0 ? (s.past + s.fresh - 1) / kUnitKeys - s.first_unit + 1 : 0;
    s.tiles = (s.fresh + a.tokens - 1) / a.tokens;
    s.segments = s.tiles * a.nkv * a.head_tiles;
    return s;
}

// A place in the line of all units, and the piece of one segment from there to the share's end.
struct Cursor {
    long long x, base;                                   // the place, and where its sequence begins
    int b, segment, from, to;                            // units [from, to) of the sequence's segment
    Sequence s;
};
__device__ __forceinline__ bool enter(const Attention4& a, Cursor& c, long long end) {
    if (c.x >= end) return false;
    while (c.x >= c.base + (long long)c.s.segments * c.s.units) {      // ends: c.x < end <= all units
        c.base += (long long)c.s.segments * c.s.units;
        ++c.b;
        c.s = sequence_of(a, c.b);
    }
    const int off = (int)(c.x - c.base);
    c.segment = off / c.s.units;
    c.from = off - c.segment * c.s.units;
    c.to = (int)min((long long)c.s.units, c.from + (end - c.x));
    return true;
}
__device__ __forceinline__ bool next_piece(const Attention4& a, Cursor& c, long long end) {
    c.x += c.to - c.from;
    return enter(a, c, end);
}

// All lanes of a warp: the units of the step, and the share of a block of `blocks`.
__device__ __forceinline__ long long share_of(const Attention4& a, int blocks) {
    long long total = 0;
    for (int b = threadIdx.x & 31; b < a.sequences; b += 32) {
        const Sequence s = sequence_of(a, b);
        total += (long long)s.segments * s.units;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    const long long wanted = (total + kLeastUnits - 1) / kLeastUnits;
    const long long used = wanted < blocks ? (wanted > 0 ? wanted : 1) : blocks;
    return (total + used - 1) / used;
}
// All lanes of a warp: the cursor at place x (with the piece up to `end`), or false where the line ends before.  `end` is cut to the line.
__device__ __forceinline__ bool find(const Attention4& a, Cursor& c, long long x, long long& end) {
    const int lane = threadIdx.x & 31;
    long long run = 0;
    bool found = false;
    for (int b0 = 0; b0 < a.sequences; b0 += 32) {
        long long mine = 0;
        if (b0 + lane < a.sequences) {
            const Sequence s = sequence_of(a, b0 + lane);
            mine = (long long)s.segments * s.units;
        }
        long long sum = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long up = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += up;
        }
        const unsigned past = __ballot_sync(0xffffffffu, run + sum > x);
        if (!found && past) {
            const int which = __ffs(past) - 1;
            c.b = b0 + which;
            c.base = run + __shfl_sync(0xffffffffu, sum - mine, which);
            found = true;
        }
        run += __shfl_sync(0xffffffffu, sum, 31);
        if (found && run >= end) break;
    }
    if (!found) return false;
    end = min(end, run);
    c.x = x;
    c.s = sequence_of(a, c.b);
    return enter(a, c, end);
}

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ __half2 as_half2(uint32_t x) { return *reinterpret_cast<__half2*>(&x); }
__device__ __forceinline__ uint32_t as_word(__half2 x) { return *reinterpret_cast<uint32_t*>(&x); }

// A scale (or two keys' scales) as the conversion needs it.
struct Scale {
    __half2 s, low, high;                                // s, -1032 s, -72 s
    __device__ __forceinline__ explicit Scale(uint32_t two_bytes) {      // bytes 0 and 2
        s = as_half2(two_bytes << 7);
        low = __hmul2(s, __float2half2_rn(-1032.0f));
        high = __hmul2(s, __float2half2_rn(-72.0f));
    }
};
// Nibbles 0 and 4 (first), 1 and 5 (second) of w times the scale.
__device__ __forceinline__ uint32_t first_of(uint32_t w, const Scale& k) {
    return as_word(__hfma2(as_half2((w & 0x000f000fu) | 0x64006400u), k.s, k.low));
}
__device__ __forceinline__ uint32_t second_of(uint32_t w, const Scale& k) {
    return as_word(__hfma2(as_half2((w & 0x00f000f0u) | 0x54005400u), k.s, k.high));
}

template <int N>
__device__ __forceinline__ void load_words(uint32_t (&w)[N], const uint8_t* p) {
    if constexpr (N == 1) {
        w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else if constexpr (N == 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        w[0] = v.x; w[1] = v.y;
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const uint4 v = *reinterpret_cast<const uint4*>(p + 4 * i);
            w[i] = v.x; w[i + 1] = v.y; w[i + 2] = v.z; w[i + 3] = v.w;
        }
    }
}

// Sizes of a block's shared memory: the warps' rings, then where the warps are merged.
template <int D, int NT>
struct Layout {
    static constexpr int columns = 8 * NT;
    static constexpr int codes = kUnitKeys * D / 2, scales = kUnitKeys * D / kGroup, unit = 2 * (codes + scales);
    static constexpr int stages = D == 64 ? 8 : (NT == 1 ? 4 : 6);
    static constexpr int ring = kWarps4 * stages * unit;
    static constexpr int parked = kWarps4 * columns * (D + 2) * 4;
    static constexpr int bytes = ring + parked + kWarps4 * columns * 4 + columns * 8;
    static constexpr int per_sm = D == 256 ? 1 : (NT == 1 ? 2 : 1);
};

template <int D, int NT>
__global__ void __launch_bounds__(kThreads4, Layout<D, NT>::per_sm)
attention4_kernel(const __grid_constant__ Attention4 a) {
    using L = Layout<D, NT>;
    constexpr int C = L::columns, S = L::stages;
    constexpr int KW = D / 32, VW = D / 64;              // words of a key and of a value that a lane holds
    extern __shared__ __align__(16) uint8_t shared[];
    dependents_may_launch();
    wait_for_predecessor();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, r = lane >> 2, t = lane & 3;
    const long long share = share_of(a, gridDim.x);
    const long long begin = share * blockIdx.x;
    long long end = begin + share;
    Cursor c;
    if (!find(a, c, begin, end)) return;                 // (all warps alike)

    uint8_t* ring = shared + warp * (S * L::unit);
    float* parked = reinterpret_cast<float*>(shared + L::ring);                       // [warp][column][m, l, O]
    float* weight = reinterpret_cast<float*>(shared + L::ring + L::parked);           // [warp][column]
    float* whole = weight + kWarps4 * C;                                              // [column]: M, then the sum

    // the ring's own cursor, ahead of the one that computes
    Cursor f = c;
    bool more = true;
    int fetch = f.from + warp;
    auto load_next = [&](int slot) {
        while (more && fetch >= f.to) {
            more = next_piece(a, f, end);
            fetch = f.from + warp;
        }
        if (more) {
            const int unit = f.s.first_unit + fetch;
            const int head = f.segment / f.s.tiles / a.head_tiles;
            const int page = a.table[(size_t)a.seq_slot[f.b] * a.table_stride + (unit >> 2)];
            const size_t at = place(page, a.nkv, head, kPage, (unit & 3) * kUnitKeys);
            const uint32_t dst = (uint32_t)__cvta_generic_to_shared(ring + slot * L::unit);
            const uint8_t *kc = a.k_codes + at * (D / 2), *vc = a.v_codes + at * (D / 2);
            const uint8_t *ks = a.k_scales + at * (D / kGroup), *vs = a.v_scales + at * (D / kGroup);
#pragma unroll
            for (int i = 0; i < L::codes / 16; i += 32) {
                const int o = (i + lane) * 16;
                fa::cp_async16(dst + o, kc + o);
                fa::cp_async16(dst + L::codes + o, vc + o);
            }
            constexpr int each = L::scales / 16;         // 16-byte pieces of the scales of a unit's keys
            if (lane < 2 * each) {
                const int o = (lane % each) * 16;
                fa::cp_async16(dst + 2 * L::codes + lane * 16, (lane < each ? ks : vs) + o);
            }
            fetch += kWarps4;
        }
        fa::cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < S - 1; ++i) load_next(i);
    int slot = 0;

    do {
        // ---- the piece: its tile's columns and their queries
        const int tile = c.segment % c.s.tiles, part = c.segment / c.s.tiles, head_tile = part % a.head_tiles, kv = part / a.head_tiles;
        const int token0 = tile * a.tokens, tokens = min(a.tokens, c.s.fresh - token0);
        const int head0 = kv * a.group + head_tile * a.heads, heads = min(a.heads, a.group - head_tile * a.heads);
        const int used = tokens * heads;                 // columns
        const int pos0 = c.s.past + token0, last = pos0 + tokens - 1;        // of the first and the last token
        const int low0 = a.window > 0 ? max(0, pos0 - a.window + 1) : 0, low1 = a.window > 0 ? max(0, last - a.window + 1) : 0;

        uint32_t qf[NT][2 * KW][2];                      // [columns' eight][contraction step][b0, b1]
        float factor[NT][2];                             // of the columns 2t, 2t + 1
        int seen[NT][2];                                 // their tokens' positions
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int column = n * 8 + r;
            const bool on = column < used;
            const __nv_bfloat16* src = a.q + (size_t)(c.s.row + token0 + (on ? column / heads : 0)) * a.q_stride
                                       + (size_t)(head0 + (on ? column % heads : 0)) * D + t * (D / 4);
            uint4 raw[KW];
            uint32_t most = 0;
#pragma unroll
            for (int w = 0; w < KW; ++w) {
                raw[w] = on ? *reinterpret_cast<const uint4*>(src + 8 * w) : make_uint4(0, 0, 0, 0);
                const uint32_t* p = &raw[w].x;
#pragma unroll
                for (int i = 0; i < 4; ++i) most = max(most, max((p[i] & 0x7fffu) << 16, p[i] & 0x7fff0000u));
            }
            most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
            most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
            const int up = min(100, max(-113, 14 + 127 - (int)(most >> 23)));
            const float by = __int_as_float((127 + up) << 23);
#pragma unroll
            for (int w = 0; w < KW; ++w) {
                float x[8];
                const uint32_t* p = &raw[w].x;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[2 * i] = __uint_as_float(p[i] << 16) * by;
                    x[2 * i + 1] = __uint_as_float(p[i] & 0xffff0000u) * by;
                }
                qf[n][2 * w][0] = as_word(__floats2half2_rn(x[0], x[4]));
                qf[n][2 * w][1] = as_word(__floats2half2_rn(x[1], x[5]));
                qf[n][2 * w + 1][0] = as_word(__floats2half2_rn(x[2], x[6]));
                qf[n][2 * w + 1][1] = as_word(__floats2half2_rn(x[3], x[7]));
            }
            const float back = __int_as_float((127 - up) << 23) * (a.scale_log2 * kUnit);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                factor[n][j] = __shfl_sync(0xffffffffu, back, (2 * t + j) * 4);
                seen[n][j] = pos0 + min(n * 8 + 2 * t + j, used - 1) / heads;
            }
        }
        float m[NT][2], l[NT][2], o[NT][D / 16][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            m[n][0] = m[n][1] = -INFINITY;
            l[n][0] = l[n][1] = 0.0f;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.0f;
        }

        // ---- its units
        for (int u = c.from + warp; u < c.to; u += kWarps4) {
            fa::cp_async_wait<S - 2>();
            __syncwarp();                                // the unit is there for all lanes, and all are done with the one before
            load_next(slot == 0 ? S - 1 : slot - 1);
            uint8_t* at = ring + slot * L::unit;
            slot = slot + 1 == S ? 0 : slot + 1;
            const int key0 = (c.s.first_unit + u) * kUnitKeys;
            if (key0 > last || key0 + kUnitKeys <= low0) continue;        // none of the tile's tokens sees any of them
            const bool border = key0 + kUnitKeys - 1 > pos0 || key0 < low1;

            float s[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
            {
                uint32_t ka[KW], kb[KW];
                load_words<KW>(ka, at + r * (D / 2) + t * (D / 8));
                load_words<KW>(kb, at + (r + 8) * (D / 2) + t * (D / 8));
                const uint8_t* sa = at + 2 * L::codes + r * (D / kGroup) + t * (D / 64);
                const uint8_t* sb = sa + 8 * (D / kGroup);
#pragma unroll
                for (int g = 0; g < D / 64; ++g) {
                    const Scale ga(sa[g] * 0x10001u), gb(sb[g] * 0x10001u);
#pragma unroll
                    for (int w = 2 * g; w < 2 * g + 2; ++w) {
                        const uint32_t a0 = first_of(ka[w], ga), a2 = second_of(ka[w], ga), a1 = first_of(kb[w], gb), a3 = second_of(kb[w], gb);
                        const uint32_t ha = ka[w] >> 8, hb = kb[w] >> 8;
                        const uint32_t c0 = first_of(ha, ga), c2 = second_of(ha, ga), c1 = first_of(hb, gb), c3 = second_of(hb, gb);
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            mma_f16(s[n], a0, a1, a2, a3, qf[n][2 * w][0], qf[n][2 * w][1]);
                            mma_f16(s[n], c0, c1, c2, c3, qf[n][2 * w + 1][0], qf[n][2 * w + 1][1]);
                        }
                    }
                }
            }
            bool grows = false;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    s[n][j] *= factor[n][j & 1];
                    if (border) {
                        const int key = key0 + r + (j >> 1) * 8, p = seen[n][j & 1];
                        if (key > p || (a.window > 0 && key <= p - a.window)) s[n][j] = -INFINITY;
                    }
                    grows |= s[n][j] > m[n][j & 1];
                }
            }
            // The maximum only has to keep the exponentials in range: it is looked for where a score exceeds it.
            if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float most = fmaxf(m[n][j], fmaxf(s[n][j], s[n][j + 2]));
                        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 4));
                        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 8));
                        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 16));
                        const float turn = most == -INFINITY ? 1.0f : fa::fast_exp2(m[n][j] - most);
                        m[n][j] = most;
                        l[n][j] *= turn;
#pragma unroll
                        for (int i = 0; i < D / 16; ++i) { o[n][i][j] *= turn; o[n][i][j + 2] *= turn; }
                    }
            }
            uint32_t p0[NT], p1[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float e[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float to = m[n][j & 1];
                    e[j] = fa::fast_exp2(s[n][j] - (to == -INFINITY ? 0.0f : to - kWeightBits));       // a score that is no number gives none
                    l[n][j & 1] += e[j];
                }
                p0[n] = transposed(as_word(__floats2half2_rn(e[0], e[1])));
                p1[n] = transposed(as_word(__floats2half2_rn(e[2], e[3])));
            }
            uint8_t* scales = at + 2 * L::codes + L::scales;
            if (border) {
                // What a key that no token of the tile sees holds must not count: even zero times a NaN is one.  Its scales are put to zero
                // here, where they lie.  A key that is no number and that only some of the tokens see makes their results none by hand.
                constexpr int words = L::scales / 4, per_key = D / kGroup / 4;
                uint32_t w[(words + 31) / 32];
                bool none = false;
#pragma unroll
                for (int i = 0; i < (words + 31) / 32; ++i) {
                    const int at_word = i * 32 + lane, key = key0 + at_word / per_key;
                    w[i] = 0;
                    if (at_word < words && key >= low0 && key <= last) w[i] = reinterpret_cast<const uint32_t*>(scales)[at_word];
                    none |= __vcmpgeu4(w[i], 0xf8f8f8f8u) != 0;
                }
                const bool by_hand = tokens > 1 && __any_sync(0xffffffffu, none);
                if (by_hand) {
                    for (int k = 0; k < kUnitKeys; ++k)
#pragma unroll
                        for (int h = 0; h < (VW + 1) / 2; ++h) {
                            if (scales[k * (D / kGroup) + (r * (D / 8)) / kGroup + h] < 0xf8) continue;
#pragma unroll
                            for (int n = 0; n < NT; ++n)
#pragma unroll
                                for (int j = 0; j < 2; ++j) {
                                    const int key = key0 + k, p = seen[n][j];
                                    if (key > p || (a.window > 0 && key <= p - a.window)) continue;
#pragma unroll
                                    for (int i = 8 * h; i < min(8 * h + 8, D / 16); ++i) o[n][i][j] = o[n][i][j + 2] = __int_as_float(0x7fc00000);
                                }
                        }
                }
                __syncwarp();
#pragma unroll
                for (int i = 0; i < (words + 31) / 32; ++i)
                    if (i * 32 + lane < words)
                        reinterpret_cast<uint32_t*>(scales)[i * 32 + lane] = by_hand ? w[i] & ~__vcmpgeu4(w[i], 0xf8f8f8f8u) : w[i];
                __syncwarp();
            }
            uint32_t va[VW], vb[VW], vc[VW], vd[VW];
            const uint8_t* codes = at + L::codes + r * (D / 16);
            load_words<VW>(va, codes + (2 * t) * (D / 2));
            load_words<VW>(vb, codes + (2 * t + 1) * (D / 2));
            load_words<VW>(vc, codes + (2 * t + 8) * (D / 2));
            load_words<VW>(vd, codes + (2 * t + 9) * (D / 2));
#pragma unroll
            for (int h = 0; h < (VW + 1) / 2; ++h) {
                auto byte = [&](int k) { return (uint32_t)scales[k * (D / kGroup) + (r * (D / 8)) / kGroup + h]; };
                const Scale ab(byte(2 * t) | byte(2 * t + 1) << 16), cd(byte(2 * t + 8) | byte(2 * t + 9) << 16);
#pragma unroll
                for (int w = 2 * h; w < min(2 * h + 2, VW); ++w) {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const uint32_t pick = half == 0 ? 0x5410u : 0x7632u;
                        uint32_t x = __byte_perm(va[w], vb[w], pick), y = __byte_perm(vc[w], vd[w], pick);
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const uint32_t a0 = first_of(x, ab), a1 = second_of(x, ab), a2 = first_of(y, cd), a3 = second_of(y, cd);
#pragma unroll
                            for (int n = 0; n < NT; ++n) mma_f16(o[n][4 * w + 2 * half + k], a0, a1, a2, a3, p0[n], p1[n]);
                            x >>= 8;
                            y >>= 8;
                        }
                    }
                }
            }
        }

        // ---- the warps' (m, l, O), merged in warp order
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float sum = l[n][j];
                sum += __shfl_xor_sync(0xffffffffu, sum, 4);
                sum += __shfl_xor_sync(0xffffffffu, sum, 8);
                sum += __shfl_xor_sync(0xffffffffu, sum, 16);
                const int column = n * 8 + 2 * t + j;
                if (column < used) {
                    float* mine = parked + (size_t)(warp * C + column) * (D + 2);
                    if (r == 0) { mine[0] = sum == sum ? m[n][j] : 0.0f; mine[1] = sum; }     // (a sum that is no number must count)
#pragma unroll
                    for (int i = 0; i < D / 16; ++i)
                        *reinterpret_cast<float2*>(mine + 2 + r * (D / 8) + 2 * i) = make_float2(o[n][i][j], o[n][i][j + 2]);
                }
            }
        __syncthreads();
        if (tid < used) {
            float M = -INFINITY;
            for (int w = 0; w < kWarps4; ++w) M = fmaxf(M, parked[(size_t)(w * C + tid) * (D + 2)]);
            float sum = 0.0f;
            for (int w = 0; w < kWarps4; ++w) {
                const float* its = parked + (size_t)(w * C + tid) * (D + 2);
                const float by = its[0] == -INFINITY ? 0.0f : fa::fast_exp2(its[0] - M);
                weight[w * C + tid] = by;
                sum = fmaf(its[1], by, sum);
            }
            whole[2 * tid] = M;
            whole[2 * tid + 1] = sum;
        }
        __syncthreads();
        const bool all = c.from == 0 && c.to == c.s.units;
        float* part_out = a.partial + (size_t)(blockIdx.x * 2 + (c.from == 0 ? 1 : 0)) * C * (D + 2);
        for (int i = tid; i < used * D; i += kThreads4) {
            const int column = i / D, e = i % D;
            float sum = 0.0f;
#pragma unroll
            for (int w = 0; w < kWarps4; ++w) {
                sum = fmaf(parked[(size_t)(w * C + column) * (D + 2) + 2 + e], weight[w * C + column], sum);
            }
            if (all) {
                const float value = sum * (kUnit / whole[2 * column + 1]);
                a.out[(size_t)(c.s.row + token0 + column / heads) * a.out_stride + (size_t)(head0 + column % heads) * D + e] = __float2bfloat16_rn(value);
            } else {
                part_out[(size_t)column * (D + 2) + 2 + e] = sum;
                if (e < 2) part_out[(size_t)column * (D + 2) + e] = whole[2 * column + e];
            }
        }
        __syncthreads();                                 // before the next piece's warps park theirs
    } while (next_piece(a, c, end));
}

// Block i merges the segment that begins in share i and goes on behind it, if there is one: its first part is in slot 1 of block i,
// the others in slot 0 of the blocks behind.
template <int D>
__global__ void __launch_bounds__(128)
attention4_merge_kernel(const __grid_constant__ Attention4 a, int columns) {
    extern __shared__ float merge[];                     // [columns][parts]
    dependents_may_launch();
    wait_for_predecessor();
    const long long share = share_of(a, gridDim.x);
    const long long begin = share * blockIdx.x;
    long long end = begin + share;
    Cursor c;
    if (!find(a, c, begin, end)) return;
    // the segment of the share's last unit
    long long whole_end = end;
    if (!find(a, c, end - 1, whole_end)) return;
    const long long from = c.x - c.from, to = from + c.s.units;          // its place in the line
    if (from < begin || to <= end) return;               // it began earlier, or ends here
    const int parts = (int)((to - 1) / share - blockIdx.x) + 1;
    const int tile = c.segment % c.s.tiles, part = c.segment / c.s.tiles, head_tile = part % a.head_tiles, kv = part / a.head_tiles;
    const int token0 = tile * a.tokens, tokens = min(a.tokens, c.s.fresh - token0);
    const int head0 = kv * a.group + head_tile * a.heads, heads = min(a.heads, a.group - head_tile * a.heads);
    const int used = tokens * heads;
    auto its = [&](int column, int p) {
        return a.partial + ((size_t)((blockIdx.x + p) * 2 + (p == 0 ? 1 : 0)) * columns + column) * (D + 2);
    };
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int column = warp; column < used; column += 4) {
        float M = -INFINITY;
        for (int p = lane; p < parts; p += 32) M = fmaxf(M, its(column, p)[0]);
        M = warp_max(M);
        float sum = 0.0f;
        for (int p = lane; p < parts; p += 32) {
            const float* one = its(column, p);
            const float by = one[0] == -INFINITY ? 0.0f : fa::fast_exp2(one[0] - M);
            merge[column * parts + p] = by;
            sum = fmaf(one[1], by, sum);
        }
        sum = warp_sum(sum);
        __syncwarp();
        const float back = kUnit / sum;
        for (int e = lane; e < D; e += 32) {
            float value = 0.0f;
            for (int p = 0; p < parts; ++p) value = fmaf(its(column, p)[2 + e], merge[column * parts + p], value);
            a.out[(size_t)(c.s.row + token0 + column / heads) * a.out_stride + (size_t)(head0 + column % heads) * D + e]
                = __float2bfloat16_rn(value * back);
        }
    }
}

// How a step's columns are tiled.
struct Tiling {
    int wide;            // columns / 8
    int tokens, heads, head_tiles;
};
static Tiling tiling(int group, int head_dim, int max_new) {
    const int most = head_dim == 256 ? 8 : 16;
    Tiling t;
    t.head_tiles = (group + most - 1) / most;
    t.heads = (group + t.head_tiles - 1) / t.head_tiles;
    const long long wanted = (long long)t.heads * max_new;
    t.wide = most == 8 || wanted <= 8 ? 1 : 2;
    t.tokens = t.wide * 8 / t.heads;
    if (t.tokens > max_new) t.tokens = max_new;
    if (t.tokens < 1) t.tokens = 1;
    return t;
}
static int blocks_of(const Tiling& t, int head_dim) {
    return device_sm_count() * (head_dim != 256 && t.wide == 1 ? 2 : 1);
}

template <int D, int NT>
static int launch(const Attention4& a, int blocks, cudaStream_t stream) {
    auto kernel = attention4_kernel<D, NT>;
    constexpr int bytes = Layout<D, NT>::bytes;
    static_assert(bytes * Layout<D, NT>::per_sm <= 227 * 1024, "the rings and the merge fit an SM");
    if (int e = raise_shared_limit(kernel, bytes, bytes)) return e;
    launch_kernel(kernel, dim3(blocks), kThreads4, bytes, stream, a);
    if (int e = CITLALI_LAUNCH_CHECK()) return e;
    constexpr int columns = Layout<D, NT>::columns;
    const size_t weights = (size_t)columns * blocks * sizeof(float);
    if (int e = raise_shared_limit(attention4_merge_kernel<D>, weights, kRowShared)) return e;
    launch_kernel(attention4_merge_kernel<D>, dim3(blocks), 128, weights, stream, a, columns);
    return CITLALI_LAUNCH_CHECK();
}

}  // namespace c4
}  // namespace citlali

using namespace citlali;

// Whether citlali_attention4 takes this head and page size.
extern "C" int citlali_attention4_supports(int head_dim, int page_size) {
    return page_size == c4::kPage && (head_dim == 64 || head_dim == 128 || head_dim == 256);
}

extern "C" size_t citlali_attention4_scratch_floats(int nq, int nkv, int head_dim, int max_new) {
    if (nkv <= 0 || nq <= 0 || nq % nkv != 0 || max_new <= 0) return 0;
    const c4::Tiling t = c4::tiling(nq / nkv, head_dim, max_new);
    return (size_t)c4::blocks_of(t, head_dim) * 2 * (8 * t.wide) * (head_dim + 2);
}

extern "C" int citlali_attention4(const void* q, size_t q_stride, const void* k_codes, const void* k_scales, const void* v_codes,
                                  const void* v_scales, const int32_t* page_table, int page_table_stride, const int32_t* seq_start,
                                  const int32_t* seq_slot, const int32_t* seq_past, void* out, size_t out_stride, float* partial,
                                  size_t partial_floats, int sequences, int max_new, int nq, int nkv, int head_dim, int page_size,
                                  int window, float scale, cudaStream_t stream) {
    if (sequences <= 0 || max_new <= 0) return 0;
    if (!citlali_attention4_supports(head_dim, page_size) || nq <= 0 || nkv <= 0 || nq % nkv != 0 || window < 0) {
        set_last_error("attention4: no kernel for %d query heads over %d key/value heads of %d with pages of %d, window %d (head sizes 64, "
                       "128 and 256, pages of 64)", nq, nkv, head_dim, page_size, window);
        return kBadShape;
    }
    if (q_stride % 8 != 0 || ((uintptr_t)q & 15u) || (((uintptr_t)k_codes | (uintptr_t)k_scales | (uintptr_t)v_codes | (uintptr_t)v_scales) & 15u)) {
        set_last_error("attention4: query rows, codes and scales must be 16-byte aligned (row pitch %zu elements)", q_stride);
        return kBadAlignment;
    }
    const c4::Tiling t = c4::tiling(nq / nkv, head_dim, max_new);
    const int blocks = c4::blocks_of(t, head_dim);
    if (partial == nullptr || partial_floats < citlali_attention4_scratch_floats(nq, nkv, head_dim, max_new)) {
        set_last_error("attention4: the scratch holds %zu floats, too few", partial_floats);
        return kTooLarge;
    }
    const long long units = ((long long)page_table_stride * page_size + max_new) / c4::kUnitKeys + 2;
    const long long segments = ((long long)max_new + t.tokens - 1) / t.tokens * nkv * t.head_tiles;
    if (units * segments > 0x7fffffffLL) {
        set_last_error("attention4: %d new tokens of one sequence over %d pages are too many for one launch", max_new, page_table_stride);
        return kTooLarge;
    }
    c4::Attention4 a = {};
    a.q = (const __nv_bfloat16*)q; a.q_stride = q_stride;
    a.k_codes = (const uint8_t*)k_codes; a.k_scales = (const uint8_t*)k_scales;
    a.v_codes = (const uint8_t*)v_codes; a.v_scales = (const uint8_t*)v_scales;
    a.table = page_table; a.table_stride = page_table_stride;
    a.seq_start = seq_start; a.seq_slot = seq_slot; a.seq_past = seq_past;
    a.out = (__nv_bfloat16*)out; a.out_stride = out_stride;
    a.sequences = sequences; a.nq = nq; a.nkv = nkv; a.group = nq / nkv;
    a.tokens = t.tokens; a.heads = t.heads; a.head_tiles = t.head_tiles;
    a.window = window; a.scale_log2 = scale * 1.4426950408889634f; a.partial = partial;
    if (head_dim == 64) return t.wide == 1 ? c4::launch<64, 1>(a, blocks, stream) : c4::launch<64, 2>(a, blocks, stream);
    if (head_dim == 128) return t.wide == 1 ? c4::launch<128, 1>(a, blocks, stream) : c4::launch<128, 2>(a, blocks, stream);
    return c4::launch<256, 1>(a, blocks, stream);
}
