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
// element above 2^-32 of that.  P is rounded to half (half a step is 2^-11 of it, an eighth of bfloat16's); the weights are kept near
// 2^11 times what the formula says, which the division takes out again, so that only those below 2^-25 of the largest are subnormal halves.
// l, the sum of the weights, is one more product, with ones.
//
// Work.  32 keys are a unit.  The units of all segments (sequence, key/value head, tile) lie end to end on a line, a little room
// ahead of each segment for what it costs to begin one, and the line is dealt out evenly to the warps, eight neighbouring ones a
// block, whatever the sequences' lengths, which are read on the device: the launch depends on none and can be captured.  A warp that
// has a whole segment stores its result.  The parts of one that several warps share are merged by the block when its warps are done,
// in the order of the keys, and the parts of one that several blocks share go to memory as (m, l, O) in float, for a second kernel
// that merges them in the same order, or, where the caller gives counters, for the block that comes last (one sequence of 900 keys: 8.8 us,
// with the second kernel 10.0).  So every sum has an order that the step's lengths fix.
//
// Measured (single tokens, heads of 128): 64 sequences of 128 to 8,192 keys, 40 heads over 8, 170 MB, 50.7 us; 16 heads over 8: 8 of 4,096
// keys, 38 MB, 18.0, two of 40,960 30.5, one of 900 7.6.  A unit takes a warp some 4,000 clocks, sixteen warps an SM, which is 5.2 TB/s of the 6.5 there are: the integer
// pipe that picks codes apart is busy half of the time, latencies are the rest.  Some 10 us go by beside that: the launch, the first
// reads (lengths, page numbers, codes, one after another: 3), and merging what warps and blocks share (3 to 4).
#include "api.h"
#include "cache4.cuh"
#include "common.cuh"
#include "mma_common.cuh"

namespace citlali {
namespace c4 {

constexpr int kPage = 64, kUnitKeys = 32, kUnitsOfAPage = kPage / kUnitKeys;
constexpr int kWarps4 = 8, kThreads4 = 32 * kWarps4;
constexpr float kWeightBits = 11.0f, kMostBits = 15.0f;         // of the largest weight when the maximum is looked for, and before it is again
constexpr uint32_t kOnes = 0x3c003c00u;
constexpr float kNoScore = -3.402823466e+38f;
// What beginning a segment costs, in units (one of 900 keys, 64 of 128 to 8,192: 1 unit 9.4, 52.9 us; 2 8.7, 52.1; 4 7.8, 51.0).
constexpr int kRoom = 4;

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
    int most;                                            // sequences with more new tokens than this are left out
    float scale_log2;
    float* partial;                                      // [blocks][2][columns][m, l, two unused, D values]
    int32_t* arrived;                                    // [2][blocks], zero before and after: parts in memory of the segment that begins in a block, and of a group of them
};

// What a sequence of the step asks for: `units` of 32 keys for each of `segments` (head tile of a key/value head, token tile).
struct Sequence {
    int past, fresh, row, first_unit, units, tiles, segments;
    __device__ __forceinline__ uint32_t length() const { return (uint32_t)segments * (units + kRoom); }      // on the line
};
__device__ __forceinline__ Sequence sequence_of(const Attention4& a, int b) {
    Sequence s;
    s.past = a.seq_past[b];
    s.row = a.seq_start ? a.seq_start[b] : b;
    s.fresh = a.seq_start ? a.seq_start[b + 1] - s.row : 1;
    if (s.fresh > a.most) s.fresh = 0;
    const int lo = a.window > 0 ? max(0, s.past - a.window + 1) : 0;
    s.first_unit = lo / kUnitKeys;
    s.units = s.fresh > 0 ? (s.past + s.fresh - 1) / kUnitKeys - s.first_unit + 1 : 0;
    s.tiles = (s.fresh + a.tokens - 1) / a.tokens;
    s.segments = s.tiles * a.nkv * a.head_tiles;
    return s;
}
// One segment: its tile's tokens and query heads.
struct Tile {
    int token0, tokens, head0, heads, kv;
    __device__ __forceinline__ int used() const { return tokens * heads; }               // columns
};
__device__ __forceinline__ Tile tile_of(const Attention4& a, const Sequence& s, int segment) {
    Tile t;
    const int part = s.tiles == 1 ? segment : segment / s.tiles, head_tile = a.head_tiles == 1 ? 0 : part % a.head_tiles;
    t.kv = a.head_tiles == 1 ? part : part / a.head_tiles;
    t.token0 = (segment - part * s.tiles) * a.tokens;
    t.tokens = min(a.tokens, s.fresh - t.token0);
    t.head0 = t.kv * a.group + head_tile * a.heads;
    t.heads = min(a.heads, a.group - head_tile * a.heads);
    return t;
}

// A place on the line: its sequence and where that begins.
struct Place {
    uint32_t base;
    int b;
};
// All lanes of a warp: the line's length.
__device__ __forceinline__ uint32_t line_length(const Attention4& a) {
    uint32_t total = 0;
#pragma unroll 1
    for (int b = threadIdx.x & 31; b < a.sequences; b += 32) total += sequence_of(a, b).length();
    return __reduce_add_sync(0xffffffffu, total);
}
// All lanes of a warp: the sequence of place x, which is on the line.
__device__ __forceinline__ Place place_of(const Attention4& a, uint32_t x) {
    const int lane = threadIdx.x & 31;
    uint32_t run = 0;
#pragma unroll 1
    for (int b0 = 0; b0 < a.sequences; b0 += 32) {
        const uint32_t mine = b0 + lane < a.sequences ? sequence_of(a, b0 + lane).length() : 0;
        uint32_t sum = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t up = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += up;
        }
        const unsigned behind = __ballot_sync(0xffffffffu, run + sum > x);
        if (behind) {
            const int which = __ffs(behind) - 1;
            return {run + __shfl_sync(0xffffffffu, sum - mine, which), b0 + which};
        }
        run += __shfl_sync(0xffffffffu, sum, 31);
    }
    return {run, a.sequences};
}
// Units of the segment from place x to `end` (one warp's share ends there): [from, to), none if the share ends ahead of them.
struct Piece {
    int segment, from, to;
    uint32_t first;                                      // the place of the segment's unit 0
};
__device__ __forceinline__ Piece piece_of(const Sequence& s, uint32_t base, uint32_t x, uint32_t end) {
    Piece p;
    const uint32_t each = s.units + kRoom;
    p.segment = (int)((x - base) / each);
    p.first = base + p.segment * each + kRoom;
    p.from = x > p.first ? (int)(x - p.first) : 0;
    p.to = end > p.first ? min(s.units, (int)(end - p.first)) : 0;
    return p;
}
// Of a column (below 16): the token of the tile, and with it the head of the group.  Exact: column / 256 is less than 1 / heads.
__device__ __forceinline__ int token_of(int column, int heads, int inverse) { return column * inverse >> 8; }
__device__ __forceinline__ int inverse_of(int heads) { return (255 + heads) / heads; }
// How the line is dealt out: places of a warp.
__device__ __forceinline__ uint32_t places_of_a_warp(uint32_t length, int blocks) {
    return (length + blocks * kWarps4 - 1) / (blocks * kWarps4);
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

template <int N>
__device__ __forceinline__ uint32_t load_bytes(const uint8_t* p) {
    if constexpr (N == 1) return *p;
    else if constexpr (N == 2) return *reinterpret_cast<const uint16_t*>(p);
    else return *reinterpret_cast<const uint32_t*>(p);
}

// A part of a segment that its warp does not have whole, as the block's merge finds it.
struct Part {
    uint32_t first;                                      // the segment's place; ~0: there is no such part
    int units, row, head0, heads, used;
};
// A piece that a warp works on: units [from, to) of a sequence (none: the end) for a tile.
struct Job {
    Part part;
    int from, to, whole;                                 // whole: the segment has no others
    int pos0, tokens, inverse;
};

// Sizes of a block's shared memory: the warps' rings (each at least as large as what its warp parks there at the end), then what a warp
// parks of a segment that began ahead of it, the parts' descriptions, and the warps' pieces: those that are being fetched or are there.
template <int D, int NT>
struct Layout {
    static constexpr int columns = 8 * NT;
    static constexpr int codes = kUnitKeys * D / 2, scales = kUnitKeys * D / kGroup, stage = 2 * (codes + scales);
    static constexpr int parked = columns * (D + 2) * 4;
    static constexpr int stages = D == 64 ? 4 : (D == 128 && NT == 2 ? 3 : 2);
    static constexpr int jobs = 8;                       // at most one a stage, one that ends, one that was looked up, and the end
    static_assert(stages + 3 <= jobs && (jobs & (jobs - 1)) == 0, "a piece's description is read before it is written over");
    static constexpr int ring = stages * stage;
    static_assert(ring >= parked && ring % 64 == 0 && (codes + scales) % 64 == 0 && parked % 16 == 0, "a warp parks its last part in its ring");
    static constexpr int bytes = kWarps4 * (ring + parked + 2 * (int)sizeof(Part) + jobs * (int)sizeof(Job));
    static constexpr int per_sm = D == 256 ? 1 : (NT == 1 ? 2 : 1);
};

// The result of a segment from its parts in memory (`to` null), or one part from several: part 0 is in slot 1 of block `first`, part p in
// slot 0 of block first + p; `count` of them, from `from` on, `step` apart, in the order of the keys.  They are brought to shared memory (`room`
// bytes there), at most kParts at once and as many columns at a time as fit (more parts: as many as the threads have one element each
// of).  This runs once in a block, when its instructions have yet to be fetched: short loops are worth more here than unrolled ones.
constexpr int kParts = 32;
template <int D>
__device__ __forceinline__ void merge_parts(const Attention4& a, int columns, int first, int from, int step, int count, const Part& part,
                                            float* to, uint8_t* shared, int room, int threads) {
    constexpr int kRow = (D + 4) * 4;                    // bytes of a part's column
    const int inverse = inverse_of(part.heads), slot = columns * kRow, at_once = min(count, kParts);
    const int fit = min(min(part.used, room / (at_once * kRow)), count > at_once ? threads / D : part.used);
    auto its = [&](int q) {
        const int p = from + q * step;
        return reinterpret_cast<const uint8_t*>(a.partial) + (size_t)((first + p) * 2 + (p == 0)) * slot;
    };
    const uint32_t dst = (uint32_t)__cvta_generic_to_shared(shared);
#pragma unroll 1
    for (int column0 = 0; column0 < part.used; column0 += fit) {
        const int here = min(fit, part.used - column0), pieces = here * (kRow / 16);
        float M = kNoScore, sum = 0.0f, value = 0.0f;
#pragma unroll 1
        for (int q0 = 0; q0 < count; q0 += kParts) {
            const int n = min(kParts, count - q0);
            __syncthreads();                             // the room is free
#pragma unroll 1
            for (int p = threadIdx.x >> 5; p < n; p += threads >> 5)
#pragma unroll 1
                for (int k = threadIdx.x & 31; k < pieces; k += 32) fa::cp_async16(dst + (p * pieces + k) * 16, its(q0 + p) + column0 * kRow + k * 16);
            fa::cp_async_commit();
            fa::cp_async_wait<0>();
            __syncthreads();
#pragma unroll 1
            for (int i = threadIdx.x; i < here * D; i += threads) {
                const int column = i / D, e = i % D;
                if (q0 == 0) { M = kNoScore; sum = value = 0.0f; }
                const float* one = reinterpret_cast<const float*>(shared) + column * (D + 4);
                const float before = M;
#pragma unroll 4
                for (int p = 0; p < n; ++p) M = fmaxf(M, one[p * here * (D + 4)]);
                const float turn = fa::fast_exp2(before - M);
                sum *= turn;
                value *= turn;
#pragma unroll 4
                for (int p = 0; p < n; ++p) {
                    const float by = fa::fast_exp2(one[p * here * (D + 4)] - M);
                    sum = fmaf(one[p * here * (D + 4) + 1], by, sum);
                    value = fmaf(one[p * here * (D + 4) + 4 + e], by, value);
                }
                if (q0 + n < count) continue;
                if (to) {
                    float* mine = to + (column0 + column) * (D + 4);
                    mine[4 + e] = value;
                    if (e == 0) *reinterpret_cast<float2*>(mine) = make_float2(M, sum);
                } else {
                    const int token = token_of(column0 + column, part.heads, inverse), head = column0 + column - token * part.heads;
                    a.out[(size_t)(part.row + token) * a.out_stride + (size_t)(part.head0 + head) * D + e] = __float2bfloat16_rn(value * (kUnit / sum));
                }
            }
        }
    }
}

// (What runs once in a piece or a block is kept short: it waits for its instructions more than for anything else.)
template <int D, int NT>
__global__ void __launch_bounds__(kThreads4, Layout<D, NT>::per_sm)
attention4_kernel(const __grid_constant__ Attention4 a) {
    using L = Layout<D, NT>;
    constexpr int C = L::columns, S = L::stages;
    constexpr int KW = D / 32, VW = D / 64;              // words of a key and of a value that a lane holds
    constexpr int KSC = 2 * L::codes, VSC = KSC + L::scales;              // in a stage: keys' codes, values' codes, keys' scales, values' scales
    extern __shared__ __align__(128) uint8_t shared[];    // (values' codes swap halves of 64 bytes by an address bit)
    __shared__ Part pending[2];                          // what goes to memory: of a segment that began earlier, and of one that goes on
    __shared__ int4 merged[2];                           // of those: what this block merges
    dependents_may_launch();
    // (positions and page tables come from the host before the step; what other kernels write is read behind the wait)
    // (the warp's number by way of a shuffle: so the compiler knows that all lanes go the same way wherever it decides)
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), r = lane >> 2, t = lane & 3;
    const Words words;
    uint8_t* ring = shared + warp * L::ring;
    float* early = reinterpret_cast<float*>(shared + kWarps4 * L::ring + warp * L::parked);      // [column][m, l, O]
    Part* parts = reinterpret_cast<Part*>(shared + kWarps4 * (L::ring + L::parked));             // [warp][early, late]
    Job* jobs = reinterpret_cast<Job*>(parts + 2 * kWarps4) + warp * L::jobs;

    const uint32_t length = line_length(a), each = places_of_a_warp(length, gridDim.x);
    const uint32_t begin = min(length, (blockIdx.x * kWarps4 + warp) * each), end = min(length, begin + each);
    if (blockIdx.x * kWarps4 * each >= length) {         // (all warps alike)
        wait_for_predecessor();
        return;
    }
    if (lane < 2) parts[2 * warp + lane].first = ~0u;
    if (tid < 2) pending[tid].used = 0;
    Place fetch = begin < end ? place_of(a, begin) : Place{0, 0};

    // ---- the ring's way along the line, ahead of the work: a unit a call, then, where a piece ends, the next one is looked up
    uint32_t fetch_x = begin;                            // the next piece's place
    int fetch_unit = 0, fetch_end = 0, fetch_head = 0, page = 0, next_page = 0, job = 0;
    const int32_t* fetch_pages = a.table;
    // Heads of 128: a value's 64 bytes of codes fill half of the banks.  A lane reads those of the keys 2t and 2t + 1: odd t take the second
    // first, and keys whose number has bit 2 have the halves of their codes swapped, so that a half-warp's reads are of different banks.
    const uint32_t swap_to = D == 128 ? (lane >> 4 & 1) * 32 : 0;         // (16 bytes a lane, four lanes a key)
    const int odd = D == 128 ? t & 1 : 0, swap_from = D == 128 ? (t >> 1) * 32 : 0;
    const uint32_t low_pick = odd ? 0x1054u : 0x5410u, high_pick = odd ? 0x3276u : 0x7632u;
    auto load_next = [&](uint8_t* to) {
        if (fetch_unit < fetch_end) {
            const size_t at = place(page, a.nkv, fetch_head, kPage, fetch_unit % kUnitsOfAPage * kUnitKeys);
            const uint32_t dst = (uint32_t)__cvta_generic_to_shared(to) + lane * 16, dst_v = dst ^ swap_to;
            const uint8_t *kc = a.k_codes + at * (D / 2) + lane * 16, *vc = a.v_codes + at * (D / 2) + lane * 16;
#pragma unroll
            for (int i = 0; i < L::codes; i += 512) {
                fa::cp_async16(dst + i, kc + i);
                fa::cp_async16(dst_v + L::codes + i, vc + i);
            }
            constexpr int pieces = L::scales / 16;       // 16-byte pieces of the scales of a unit's keys
#pragma unroll
            for (int i = 0; i < (2 * pieces + 31) / 32; ++i) {
                const int k = i * 32 + lane;
                if (k < 2 * pieces)
                    fa::cp_async16(dst + KSC + i * 512, (k < pieces ? a.k_scales : a.v_scales) + at * (D / kGroup) + k % pieces * 16);
            }
            ++fetch_unit;
            if (fetch_unit % kUnitsOfAPage == 0) {
                page = next_page;
                if (fetch_unit + kUnitsOfAPage < fetch_end) next_page = fetch_pages[fetch_unit / kUnitsOfAPage + 1];
            }
        }
        fa::cp_async_commit();
        if (fetch_unit == fetch_end && fetch_end >= 0) { // (what it reads is there when the next unit is asked for)
            Sequence s = {};
            Piece p = {0, 0, 0, 0};
#pragma unroll 1
            while (fetch_x < end && p.to <= p.from) {
                s = sequence_of(a, fetch.b);
                if (fetch_x >= fetch.base + s.length()) {
                    fetch.base += s.length();
                    ++fetch.b;
                } else {
                    p = piece_of(s, fetch.base, fetch_x, end);
                    fetch_x = p.first + s.units;
                }
            }
            Job j = {};
            fetch_end = fetch_unit = -1;                 // the end
            if (p.to > p.from) {
                const Tile tile = tile_of(a, s, p.segment);
                fetch_head = tile.kv;
                fetch_pages = a.table + (size_t)a.seq_slot[fetch.b] * a.table_stride;
                fetch_unit = s.first_unit + p.from;
                fetch_end = s.first_unit + p.to;
                page = fetch_pages[fetch_unit / kUnitsOfAPage];
                next_page = fetch_pages[min(fetch_unit / kUnitsOfAPage + 1, (fetch_end - 1) / kUnitsOfAPage)];
                j.part = {p.first, s.units, s.row + tile.token0, tile.head0, tile.heads, tile.used()};
                j.from = fetch_unit;
                j.to = fetch_end;
                j.whole = p.from == 0 && p.to == s.units;
                j.pos0 = s.past + tile.token0;
                j.tokens = tile.tokens;
                j.inverse = inverse_of(tile.heads);
            }
            if (lane == 0) jobs[job & (L::jobs - 1)] = j;
            ++job;
        }
    };
    auto fetch_queries = [&](const Job& j) {             // into L1, a line a lane
        constexpr int lines = D * 2 / 128;
        const int column = lane / lines;
        if (column < j.part.used) {
            const int token = token_of(column, j.part.heads, j.inverse), head = column - token * j.part.heads;
            const __nv_bfloat16* p = a.q + (size_t)(j.part.row + token) * a.q_stride + (size_t)(j.part.head0 + head) * D + lane % lines * 64;
            asm volatile("prefetch.global.L1 [%0];" ::"l"(p));
        }
    };

    uint32_t qf[NT][2 * KW][2];                          // [columns' eight][contraction step][b0, b1]
    float factor[NT][2];                                 // of the columns 2t, 2t + 1
    // m: a running maximum less kWeightBits; the lowest number there is where there is none, which no sum with a score overflows to a NaN
    float m[NT][2], l[NT][4], o[NT][D / 16][4];
    bool fresh = true;                                   // no unit of the piece has counted yet
    int u = 0, stop = 0, done = 0, pos0 = 0, last = 0, heads = 1, inverse = 256, used = 1;
    uint8_t *at = ring, *free_stage = ring;
#pragma unroll 1
    for (int turn = 0;; ++turn) {
        // the first S turns only look ahead: the first piece is looked up, then S - 1 units are asked for
        if (turn == 1) wait_for_predecessor();
        if (turn >= S) {
            fa::cp_async_wait<S - 2>();
            __syncwarp();                                // the stage is there for all lanes, and all are done with the one before
        }
        const int known = job;
        load_next(free_stage);
        if (turn > 0 && (turn == 1 || job > known)) {
            __syncwarp();
            if (turn == 1) fetch_queries(jobs[0]);
            if (job > known) fetch_queries(jobs[known & (L::jobs - 1)]);
        }
        free_stage = free_stage + L::stage == ring + L::ring ? ring : free_stage + L::stage;
        if (turn < S) {
            if (turn == 0) free_stage = ring;            // (nothing was asked for)
            continue;
        }
        if (u == stop) {
            // ---- the next piece: its tile's columns and their queries
            __syncwarp();
            const Job& j = jobs[done++ & (L::jobs - 1)];
            u = j.from;
            stop = j.to;
            if (u == stop) break;
            fresh = true;
            used = j.part.used;
            heads = j.part.heads;
            inverse = j.inverse;
            pos0 = j.pos0;
            last = pos0 + j.tokens - 1;                  // positions of the first and the last token
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int column = n * 8 + r;
                const bool on = column < used;
                const int token = on ? token_of(column, heads, inverse) : 0, head = on ? column - token * heads : 0;
                const __nv_bfloat16* src = a.q + (size_t)(j.part.row + token) * a.q_stride + (size_t)(j.part.head0 + head) * D + t * (D / 4);
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
                    float y[8];
                    const uint32_t* p = &raw[w].x;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        y[2 * i] = __uint_as_float(p[i] << 16) * by;
                        y[2 * i + 1] = __uint_as_float(p[i] & 0xffff0000u) * by;
                    }
                    qf[n][2 * w][0] = as_word(__floats2half2_rn(y[0], y[4]));
                    qf[n][2 * w][1] = as_word(__floats2half2_rn(y[1], y[5]));
                    qf[n][2 * w + 1][0] = as_word(__floats2half2_rn(y[2], y[6]));
                    qf[n][2 * w + 1][1] = as_word(__floats2half2_rn(y[3], y[7]));
                }
                const float back = __int_as_float((127 - up) << 23) * (a.scale_log2 * kUnit);
#pragma unroll
                for (int k = 0; k < 2; ++k) factor[n][k] = __shfl_sync(0xffffffffu, back, (2 * t + k) * 4);
                m[n][0] = m[n][1] = kNoScore;
                l[n][0] = l[n][1] = l[n][2] = l[n][3] = 0.0f;
#pragma unroll
                for (int i = 0; i < D / 16; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.0f;
            }
        }

        // ---- a unit
        const uint8_t* const stage = at;
        at = at + L::stage == ring + L::ring ? ring : at + L::stage;
        const int key0 = u * kUnitKeys, key1 = key0 + kUnitKeys;
        const int low0 = a.window > 0 ? max(0, pos0 - a.window + 1) : 0;
        ++u;
        if (key0 <= last && key1 > low0) {               // (some of the tile's tokens see some of them)
            const bool border = key1 - 1 > pos0 || (a.window > 0 && key0 <= last - a.window);
            auto sees = [&](int column, int key) {       // whether the column's token does
                const int p = pos0 + token_of(min(column, used - 1), heads, inverse);
                return key <= p && (a.window == 0 || key > p - a.window);
            };

            float e[2][NT][4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int n = 0; n < NT; ++n) e[h][n][0] = e[h][n][1] = e[h][n][2] = e[h][n][3] = 0.0f;
                uint32_t ka[KW], kb[KW];
                const uint8_t* codes = stage + h * (L::codes / 2) + r * (D / 2) + t * (D / 8);
                load_words<KW>(ka, codes);
                load_words<KW>(kb, codes + 8 * (D / 2));
                const uint8_t* scales = stage + KSC + h * (L::scales / 2) + r * (D / kGroup) + t * (D / 64);
                const uint32_t ba = load_bytes<D / 64>(scales), bb = load_bytes<D / 64>(scales + 8 * (D / kGroup));
#pragma unroll
                for (int g = 0; g < D / 64; ++g) {
                    const Scale ga(__byte_perm(ba, 0, 0x4040 + 0x101 * g)), gb(__byte_perm(bb, 0, 0x4040 + 0x101 * g));
#pragma unroll
                    for (int w = 2 * g; w < 2 * g + 2; ++w) {
                        const uint32_t a0 = words.first_of(ka[w], ga), a2 = words.second_of(ka[w], ga), a1 = words.first_of(kb[w], gb), a3 = words.second_of(kb[w], gb);
                        const uint32_t ha = ka[w] >> 8, hb = kb[w] >> 8;
                        const uint32_t c0 = words.first_of(ha, ga), c2 = words.second_of(ha, ga), c1 = words.first_of(hb, gb), c3 = words.second_of(hb, gb);
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            mma_f16(e[h][n], a0, a1, a2, a3, qf[n][2 * w][0], qf[n][2 * w][1]);
                            mma_f16(e[h][n], c0, c1, c2, c3, qf[n][2 * w + 1][0], qf[n][2 * w + 1][1]);
                        }
                    }
                }
            }
            // w = 2^(score - m).  m only has to keep the weights in range: it is looked for where one exceeds 2^kMostBits.
            float w[2][NT][4];
            float most = -INFINITY;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    w[0][n][j] = fmaf(e[0][n][j], factor[n][j & 1], -m[n][j & 1]);
                    w[1][n][j] = fmaf(e[1][n][j], factor[n][j & 1], -m[n][j & 1]);
                    if (border) {
                        const int column = n * 8 + 2 * t + (j & 1), key = key0 + r + (j >> 1) * 8;
                        if (!sees(column, key)) w[0][n][j] = -INFINITY;
                        if (!sees(column, key + 16)) w[1][n][j] = -INFINITY;
                    }
                    most = fmaxf(most, fmaxf(w[0][n][j], w[1][n][j]));
                }
            if (__any_sync(0xffffffffu, most > kMostBits)) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float top = kNoScore;
#pragma unroll
                        for (int h = 0; h < 2; ++h)
#pragma unroll
                            for (int i = j; i < 4; i += 2)
                                if (w[h][n][i] != -INFINITY) top = fmaxf(top, e[h][n][i] * factor[n][j]);
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                        top = fmaxf(m[n][j], fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16)) - kWeightBits);
                        const float turn = fa::fast_exp2(m[n][j] - top);
                        m[n][j] = top;
                        if (!fresh) {                    // (else they are zeros)
                            l[n][j] *= turn;
#pragma unroll
                            for (int i = 0; i < D / 16; ++i) { o[n][i][j] *= turn; o[n][i][j + 2] *= turn; }
                        }
#pragma unroll
                        for (int h = 0; h < 2; ++h)
#pragma unroll
                            for (int i = j; i < 4; i += 2)
                                if (w[h][n][i] != -INFINITY) w[h][n][i] = fmaf(e[h][n][i], factor[n][j], -top);
                    }
                fresh = false;
            }
            uint32_t p[2][NT][2];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    p[h][n][0] = transposed(as_word(__floats2half2_rn(fa::fast_exp2(w[h][n][0]), fa::fast_exp2(w[h][n][1]))));
                    p[h][n][1] = transposed(as_word(__floats2half2_rn(fa::fast_exp2(w[h][n][2]), fa::fast_exp2(w[h][n][3]))));
                    mma_f16(l[n], kOnes, kOnes, kOnes, kOnes, p[h][n][0], p[h][n][1]);        // every row of the product is the columns' sums
                }
            if (border) {
                // What a key that no token of the tile sees holds must not count: even zero times a NaN is one.  Its scales are put to zero
                // here, where they lie.  A value that is no number and that only some of the tokens see becomes zero as well, and spoils
                // the sums of those that do see it.
                uint32_t* const scales = reinterpret_cast<uint32_t*>(const_cast<uint8_t*>(stage) + VSC);
                constexpr int per_key = D / kGroup / 4;
#pragma unroll 1
                for (int i = lane; i < L::scales / 4; i += 32) {
                    const int key = key0 + i / per_key;
                    uint32_t w = key >= low0 && key <= last ? scales[i] : 0;
                    const uint32_t none = __vcmpgeu4(w, 0xf8f8f8f8u);
                    const unsigned found = __ballot_sync(0xffffffffu, none != 0 && last > pos0);
                    if (last > pos0) w &= ~none;
                    scales[i] = w;
#pragma unroll 1
                    for (unsigned rest = found; rest; rest &= rest - 1) {
                        const int spoilt = key0 + (i - lane + __ffs(rest) - 1) / per_key;
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int j = 0; j < 2; ++j)
                                if (sees(n * 8 + 2 * t + j, spoilt)) l[n][j] = __int_as_float(0x7fc00000);
                    }
                }
                __syncwarp();
            }
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                uint32_t va[VW], vb[VW], vc[VW], vd[VW];
                const uint8_t* codes = stage + L::codes + half * (L::codes / 2) + ((r * (D / 16)) ^ swap_from);
                load_words<VW>(va, codes + (2 * t + odd) * (D / 2));
                load_words<VW>(vb, codes + (2 * t + 1 - odd) * (D / 2));
                load_words<VW>(vc, codes + (2 * t + 8 + odd) * (D / 2));
                load_words<VW>(vd, codes + (2 * t + 9 - odd) * (D / 2));
                const uint8_t* scales = stage + VSC + half * (L::scales / 2) + (r * (D / 8)) / kGroup;
#pragma unroll
                for (int h = 0; h < (VW + 1) / 2; ++h) {
                    auto byte = [&](int k) { return (uint32_t)scales[k * (D / kGroup) + h]; };
                    const Scale ab(byte(2 * t) | byte(2 * t + 1) << 16), cd(byte(2 * t + 8) | byte(2 * t + 9) << 16);
#pragma unroll
                    for (int w = 2 * h; w < min(2 * h + 2, VW); ++w) {
#pragma unroll
                        for (int part = 0; part < 2; ++part) {
                            const uint32_t pick = part == 0 ? low_pick : high_pick;
                            uint32_t y = __byte_perm(va[w], vb[w], pick), z = __byte_perm(vc[w], vd[w], pick);
#pragma unroll
                            for (int k = 0; k < 2; ++k) {
                                const uint32_t a0 = words.first_of(y, ab), a1 = words.second_of(y, ab), a2 = words.first_of(z, cd), a3 = words.second_of(z, cd);
#pragma unroll
                                for (int n = 0; n < NT; ++n) mma_f16(o[n][4 * w + 2 * part + k], a0, a1, a2, a3, p[half][n][0], p[half][n][1]);
                                y >>= 8;
                                z >>= 8;
                            }
                        }
                    }
                }
            }
        }

        if (u < stop) continue;

        // ---- the piece's end: the whole segment's result, or a part to merge
        __syncwarp();
        const Job& j = jobs[(done - 1) & (L::jobs - 1)];
        const bool late = !j.whole && j.part.first + j.part.units >= end;       // a part is the warp's first or its last
        if (late) {
            fa::cp_async_wait<0>();
            __syncwarp();                                // the ring is the warp's own and empty
        }
        float* parked = late ? reinterpret_cast<float*>(ring) : early;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int column = n * 8 + 2 * t + k;
                if (column >= used) continue;
                if (j.whole) {
                    const float by = kUnit / l[n][k];
                    const int token = token_of(column, heads, inverse);
                    __nv_bfloat16* dst = a.out + (size_t)(j.part.row + token) * a.out_stride + (size_t)(j.part.head0 + column - token * heads) * D + r * (D / 8);
#pragma unroll
                    for (int i = 0; i < D / 16; ++i)
                        *reinterpret_cast<uint32_t*>(dst + 2 * i) = fa::pack_bf16(o[n][i][k] * by, o[n][i][k + 2] * by);
                } else {
                    float* mine = parked + column * (D + 2);
                    if (r == 0) { mine[0] = m[n][k]; mine[1] = l[n][k]; }
#pragma unroll
                    for (int i = 0; i < D / 16; ++i)
                        *reinterpret_cast<float2*>(mine + 2 + r * (D / 8) + 2 * i) = make_float2(o[n][i][k], o[n][i][k + 2]);
                }
            }
        if (!j.whole && lane == 0) parts[2 * warp + (late ? 1 : 0)] = j.part;
    }

    // ---- the block's parts, in the order of the line: those of one segment are neighbours.  Nothing is written to shared memory any more.
    __syncthreads();
    const uint32_t block_begin = blockIdx.x * kWarps4 * each, block_end = min(length, block_begin + kWarps4 * each);
    const uint32_t mine = lane < 2 * kWarps4 ? parts[lane].first : ~0u;
#pragma unroll 1
    for (unsigned left = __ballot_sync(0xffffffffu, mine != ~0u); left;) {
        const int k0 = __ffs(left) - 1;
        const unsigned run = __ballot_sync(0xffffffffu, mine == __shfl_sync(0xffffffffu, mine, k0)) & left;
        left &= ~run;
        // one part of each of the warps w0 .. w1: their last, but for w1's, which may be its first
        const int w0 = k0 >> 1, k1 = 31 - __clz(run), count = (k1 >> 1) - w0;
        const Part part = parts[k0];
        const bool begins = part.first >= block_begin, all = begins && part.first + part.units <= block_end;
        float* part_out = a.partial + (size_t)(blockIdx.x * 2 + (begins ? 1 : 0)) * C * (D + 4);
        const float* lates = reinterpret_cast<const float*>(shared + w0 * L::ring);
        const float* final_one = reinterpret_cast<const float*>(shared + (k1 & 1 ? (k1 >> 1) * L::ring : kWarps4 * L::ring + (k1 >> 1) * L::parked));
#pragma unroll 1
        for (int i = tid; i < part.used * D; i += kThreads4) {
            const int column = i / D, element = i % D, at = column * (D + 2);
            float M = final_one[at], sum = 0.0f, value = 0.0f;
#pragma unroll 4
            for (int w = 0; w < count; ++w) M = fmaxf(M, lates[w * (L::ring / 4) + at]);
#pragma unroll 4
            for (int w = 0; w < count; ++w) {
                const float* one = lates + w * (L::ring / 4) + at;
                const float by = fa::fast_exp2(one[0] - M);
                sum = fmaf(one[1], by, sum);
                value = fmaf(one[2 + element], by, value);
            }
            const float by = fa::fast_exp2(final_one[at] - M);
            sum = fmaf(final_one[at + 1], by, sum);
            value = fmaf(final_one[at + 2 + element], by, value);
            if (all) {
                const int token = token_of(column, part.heads, inverse_of(part.heads)), head = column - token * part.heads;
                a.out[(size_t)(part.row + token) * a.out_stride + (size_t)(part.head0 + head) * D + element] = __float2bfloat16_rn(value * (kUnit / sum));
            } else {
                part_out[column * (D + 4) + 4 + element] = value;
                if (element == 0) *reinterpret_cast<float2*>(part_out + column * (D + 4)) = make_float2(M, sum);
            }
        }
        if (!all && tid == 0) pending[begins ? 1 : 0] = part;
    }
    if (a.arrived == nullptr) return;
    // The block whose part of a segment comes to memory last merges them all; nobody waits for anybody.  Parts of more than kParts blocks
    // are merged so by kParts neighbours first, into the first one's place (one sequence of 64,000 keys, 8 heads over one of 128: 24 us;
    // by one block alone, whose room held no column of all 250 parts, 960).
    const uint32_t share = kWarps4 * each;
    auto blocks_of = [&](const Part& part) { return (int)((part.first + part.units - 1) / share) - (int)(part.first / share) + 1; };
#pragma unroll 1
    for (int level = 0;; ++level) {
        __syncthreads();
        if (lane == 0 && warp < 2) {
            const Part part = pending[warp];
            int4 what = make_int4(0, 0, 0, 0);           // the segment's first block, and the parts to merge: from, step, count
            if (part.used && (level == 0 || (merged[warp].w && blocks_of(part) > kParts))) {
                const int first = (int)(part.first / share), all = blocks_of(part), own = (int)blockIdx.x - first;
                what = make_int4(first, 0, 1, all);
                int32_t* arrived = a.arrived + first;
                if (all > kParts && level == 0) {        // (counted apart: the segment's last block may be another one's first)
                    what.y = own / kParts * kParts;
                    what.w = min(kParts, all - what.y);
                    arrived += gridDim.x + what.y;
                } else if (level == 1) {
                    what.z = kParts;
                    what.w = (all + kParts - 1) / kParts;
                }
                // (a group of one block, a segment's last, is complete; its counter may be the next segment's first group's)
                if (what.w > 1) {
                    int before;                          // (ordered behind the block's writes, which the barrier has put ahead, and ahead of what is read)
                    asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(before) : "l"(arrived) : "memory");
                    if (before == what.w - 1) *arrived = 0;      // as the next call wants it
                    else what.w = 0;
                }
            }
            merged[warp] = what;
        }
        __syncthreads();
        bool more = false;                               // (for all threads alike)
#pragma unroll 1
        for (int k = 0; k < 2; ++k) {
            const Part part = pending[k];
            const int4 what = merged[k];
            if (!part.used || !what.w) continue;
            float* to = nullptr;
            if (level == 0 && blocks_of(part) > kParts) {
                to = a.partial + (size_t)((what.x + what.y) * 2 + (what.y == 0)) * C * (D + 4);
                more = true;
            }
            merge_parts<D>(a, C, what.x, what.y, what.z, what.w, part, to, shared, kWarps4 * (L::ring + L::parked), kThreads4);
        }
        if (!more) return;
    }
}

// The same as a kernel of its own, where there is nothing to count arrivals in: block i merges the segment whose unit 0 is in the share
// of block i and that goes on behind it, if there is one.
constexpr int kMergeThreads = 256, kMergeRoom = 40 * 1024;
template <int D>
__global__ void __launch_bounds__(kMergeThreads)
attention4_merge_kernel(const __grid_constant__ Attention4 a, int columns) {
    extern __shared__ __align__(16) uint8_t shared[];
    dependents_may_launch();
    const uint32_t length = line_length(a), share = places_of_a_warp(length, gridDim.x) * kWarps4;
    const uint32_t begin = blockIdx.x * share, end = begin + share;
    Place here = {0, 0};
    if (end < length) here = place_of(a, end);           // the segment that the next share begins in
    wait_for_predecessor();                              // (every block: the kernel behind this one waits for this one alone)
    if (end >= length) return;                           // nothing lies behind
    const Sequence s = sequence_of(a, here.b);
    const Piece piece = piece_of(s, here.base, end, end + 1);
    if (piece.first < begin || piece.first >= end) return;               // it began earlier, or only its room is here
    const Tile tile = tile_of(a, s, piece.segment);
    const Part part = {piece.first, s.units, s.row + tile.token0, tile.head0, tile.heads, tile.used()};
    merge_parts<D>(a, columns, blockIdx.x, 0, 1, (int)((piece.first + s.units - 1) / share - blockIdx.x) + 1, part, nullptr, shared, kMergeRoom,
                   kMergeThreads);
}

// How a step's columns are tiled: 8 at a time where a segment has no more (two blocks an SM), else 16 (one).  16 for 8 columns: one
// sequence of 900 keys 7.7 -> 8.3 us, 8 of 4,096 18.0 -> 22.8, 64 of 128 to 8,192 50.7 -> 70.0.
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
    static_assert((bytes + 1024) * Layout<D, NT>::per_sm <= 228 * 1024, "the blocks of an SM fit it");
    if (int e = raise_shared_limit(kernel, bytes, bytes)) return e;
    launch_kernel(kernel, dim3(blocks), kThreads4, bytes, stream, a);
    if (int e = CITLALI_LAUNCH_CHECK()) return e;
    if (a.arrived) return 0;
    launch_kernel(attention4_merge_kernel<D>, dim3(blocks), kMergeThreads, kMergeRoom, stream, a, Layout<D, NT>::columns);
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
    return (size_t)c4::blocks_of(t, head_dim) * 2 * (8 * t.wide) * (head_dim + 4);
}

extern "C" int citlali_attention4(const void* q, size_t q_stride, const void* k_codes, const void* k_scales, const void* v_codes,
                                  const void* v_scales, const int32_t* page_table, int page_table_stride, const int32_t* seq_start,
                                  const int32_t* seq_slot, const int32_t* seq_past, void* out, size_t out_stride, float* partial,
                                  size_t partial_floats, int32_t* arrived, size_t arrived_ints, int sequences, int max_new, int most_new, int nq, int nkv, int head_dim,
                                  int page_size, int window, float scale, cudaStream_t stream) {
    if (sequences <= 0 || max_new <= 0) return 0;
    if (!citlali_attention4_supports(head_dim, page_size) || nq <= 0 || nkv <= 0 || nq % nkv != 0 || window < 0) {
        set_last_error("attention4: no kernel for %d query heads over %d key/value heads of %d with pages of %d, window %d (head sizes 64, "
                       "128 and 256, pages of 64)", nq, nkv, head_dim, page_size, window);
        return kBadShape;
    }
    if (q_stride % 8 != 0 || out_stride % 2 != 0 || ((uintptr_t)out & 3u) ||
        (((uintptr_t)q | (uintptr_t)k_codes | (uintptr_t)k_scales | (uintptr_t)v_codes | (uintptr_t)v_scales | (uintptr_t)partial) & 15u)) {
        set_last_error("attention4: query rows, codes, scales and scratch must be 16-byte aligned, rows of results 4-byte (pitches of %zu and "
                       "%zu elements)", q_stride, out_stride);
        return kBadAlignment;
    }
    const c4::Tiling t = c4::tiling(nq / nkv, head_dim, max_new);
    const int blocks = c4::blocks_of(t, head_dim);
    if (partial == nullptr || partial_floats < citlali_attention4_scratch_floats(nq, nkv, head_dim, max_new)) {
        set_last_error("attention4: the scratch holds %zu floats, too few", partial_floats);
        return kTooLarge;
    }
    if (arrived != nullptr && arrived_ints < 2 * (size_t)blocks) {
        set_last_error("attention4: room for %zu counters, two for each of %d blocks", arrived_ints, blocks);
        return kTooLarge;
    }
    const long long units = ((long long)page_table_stride * page_size + max_new) / c4::kUnitKeys + 2 + c4::kRoom;
    const long long segments = ((long long)max_new + t.tokens - 1) / t.tokens * nkv * t.head_tiles;
    if (units * segments > 0x3fffffffLL / sequences) {             // (places on the line are 32 bits)
        set_last_error("attention4: %d sequences of up to %d new tokens over %d pages are too many for one launch", sequences, max_new,
                       page_table_stride);
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
    a.window = window; a.most = most_new > 0 ? most_new : 0x7fffffff; a.scale_log2 = scale * 1.4426950408889634f; a.partial = partial; a.arrived = arrived;
    if (head_dim == 64) return t.wide == 1 ? c4::launch<64, 1>(a, blocks, stream) : c4::launch<64, 2>(a, blocks, stream);
    if (head_dim == 128) return t.wide == 1 ? c4::launch<128, 1>(a, blocks, stream) : c4::launch<128, 2>(a, blocks, stream);
    return c4::launch<256, 1>(a, blocks, stream);
}
