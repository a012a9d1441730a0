// Log probabilities of given tokens, the entropy of a row's distribution and its likeliest tokens, from logits in one pass.
//
//   over the finite entries of a row:  m = max x,  S = sum e^(x - m),  T = sum (x - m) e^(x - m)
//   log p(token) = x_token - m - log S      entropy = log S - T / S      the `top` largest entries, the lowest index first among equals
//
// Entries that are not finite have no probability, as in sampling.cu; a row without a finite entry has none at all (log
// probabilities of minus infinity, entropy 0, ids -1).  Logits are float32 or bfloat16; all sums are float32.
//
// What bounds it: reading the logits once (1,000 rows of 151,936 float32: 107 us, 5.7 TB/s); with few rows the passes over the
// likeliest that follow (8 rows, 20 likeliest: 10.4 us, of which reading takes 2).  A cluster of 1 to 8 blocks takes a row, a block an even share of it; a thread has 16
// entries in registers and the next 16 on their way.  m, S and T are the thread's own until the end (the running maximum is looked
// at once for 16 entries).
//
// The likeliest tokens.  A share's first tiles (all of a short share) are looked at a second time, out of the caches, once a bound is
// known.  A thread remembers the largest of its tiles' maxima, which tile it was, and the second largest.  Every warp of the cluster
// names as many of its lanes' largest as there have to be for `top` numbers; the top-th of them has at least `top` entries at or above
// it, and hardly more threads that hold any: of those threads alone the warp looks through the tile again (through all of the thread's
// tiles where the second maximum
// reaches the bound too), and what it finds is sorted.  From then on a tile's entries are looked at only if one exceeds the last entry
// that still counts in any warp of the block; a warp keeps a list of what it finds, lane i the i-th largest.  (So it does from the
// start where more than 512 entries reached the first bound: many alike.)  Warps and then blocks, through distributed shared memory,
// merge their lists pairwise: the larger of a[i] and b[31 - i] are the 32 largest of both, and five exchanges sort them.
#include "api.h"
#include "common.cuh"
#include "mma_common.cuh"

namespace citlali {
namespace lp {

constexpr int kThreads = 256, kWarps = 8, kEach = 16, kMost = 32;
constexpr int kMaxCluster = 8;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kNone = 0x7fffffff;                        // no entry: behind every index

// Tiles ahead of the first bound (1,000 rows of 151,936: 4 and 8 alike, 16 4 us longer), and what the first block has room to sort.
constexpr int kWindow = 8, kFound = 512;

struct Summary { float m, s, t; };

// A float as a whole number in the same order, and back.
__device__ __forceinline__ int ordered(float v) {
    const int i = __float_as_int(v);
    return i < 0 ? i ^ 0x7fffffff : i;
}
__device__ __forceinline__ float unordered(int i) { return __int_as_float(i < 0 ? i ^ 0x7fffffff : i); }

__device__ __forceinline__ bool before(float v, int i, float w, int j) { return v > w || (v == w && i < j); }

// The summary over both.
__device__ __forceinline__ Summary joined(Summary a, Summary b) {
    const float m = fmaxf(a.m, b.m);
    if (m == -INFINITY) return a;
    // (x - m) e^(x - m) from (x - a.m) e^(x - a.m): the exponent shifts by a.m - m, and every term by as much
    const float da = fmaxf(a.m - m, -104.0f), db = fmaxf(b.m - m, -104.0f);
    const float ea = expf(da), eb = expf(db);
    return {m, a.s * ea + b.s * eb, (a.t + a.s * da) * ea + (b.t + b.s * db) * eb};
}

// A warp's list: lane i holds its i-th entry.
__device__ __forceinline__ void exchange(float& v, int& i, int distance, bool larger_first) {
    const float w = __shfl_xor_sync(0xffffffffu, v, distance);
    const int j = __shfl_xor_sync(0xffffffffu, i, distance);
    const bool low = (threadIdx.x & distance) == 0;
    if (before(w, j, v, i) == (low == larger_first)) { v = w; i = j; }
}
__device__ __forceinline__ void sort(float& v, int& i) {
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int distance = size >> 1; distance > 0; distance >>= 1) exchange(v, i, distance, (threadIdx.x & size & 31) == 0);
}
// (w, j): another list, lane i given its entry 31 - i.
__device__ __forceinline__ void merge(float& v, int& i, float w, int j) {
    if (before(w, j, v, i)) { v = w; i = j; }
#pragma unroll
    for (int distance = 16; distance > 0; distance >>= 1) exchange(v, i, distance, true);
}

__device__ __forceinline__ void load(const float* p, float (&x)[kEach]) {
#pragma unroll
    for (int k = 0; k < kEach / 4; ++k) {
        const float4 v = *(reinterpret_cast<const float4*>(p) + k * kThreads);
        x[4 * k] = v.x; x[4 * k + 1] = v.y; x[4 * k + 2] = v.z; x[4 * k + 3] = v.w;
    }
}
__device__ __forceinline__ void load(const __nv_bfloat16* p, float (&x)[kEach]) {
#pragma unroll
    for (int k = 0; k < kEach / 8; ++k) {
        const uint4 v = *(reinterpret_cast<const uint4*>(p) + k * kThreads);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) { x[8 * k + 2 * e] = __uint_as_float(w[e] << 16); x[8 * k + 2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u); }
    }
}

struct Block {                                           // what a block tells the first of its cluster
    Summary sum;
    float v[kMost];
    int i[kMost];
};

template <typename T, bool TOP>
__global__ void __launch_bounds__(kThreads, 4)
token_logprobs_kernel(const T* __restrict__ logits, const int32_t* __restrict__ tokens, float* __restrict__ logprobs,
                      float* __restrict__ entropy, int32_t* __restrict__ top_ids, float* __restrict__ top_logprobs, int vocab, int top,
                      int cluster) {
    constexpr int kVec = 16 / sizeof(T);                 // entries of a 16-byte load
    __shared__ Summary sums[kWarps];
    __shared__ float list_v[kWarps][32];
    __shared__ int list_i[kWarps][32];
    __shared__ Block blocks[kMaxCluster];
    __shared__ float found_v[TOP ? kFound : 1];
    __shared__ int found_i[TOP ? kFound : 1], found, shared_bound, named[64];
    dependents_may_launch();
    wait_for_predecessor();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const long long row = blockIdx.x / cluster;
    const int rank = blockIdx.x % cluster;
    const T* x = logits + row * vocab;

    // the row from its first 16-byte boundary on, in tiles of kThreads * kEach entries, dealt out to the cluster's blocks evenly;
    // the first block also takes the entries ahead of the boundary, the last one those behind the last whole vector
    const int lead = min(vocab, (int)((16 - ((uintptr_t)x & 15)) % 16 / sizeof(T)));
    const int vectors = (vocab - lead) / kVec, share = (vectors + cluster - 1) / cluster;
    const int first = min(vectors, rank * share), stop = min(vectors, first + share);      // this block's vectors

    Summary mine = {-INFINITY, 0.0f, 0.0f};
    float best = -INFINITY;                              // lane i: the warp's i-th largest entry
    int at = kNone;
    float bound = -INFINITY;                             // the top-th
    int bound_at = kNone;
    if (TOP && tid == 0) found = 0;
    __syncwarp();
    if (cluster > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");       // (waited for ahead of the first write to another block)

    // The largest of a thread's 16 entries, quarter by quarter.  Plus infinity is no entry (nor is a NaN, which no maximum takes).
    auto largest = [&](float (&y)[kEach], float (&quarter)[4]) {
        float most;
        auto look = [&] {
#pragma unroll
            for (int k = 0; k < 4; ++k) quarter[k] = fmaxf(fmaxf(y[4 * k], y[4 * k + 1]), fmaxf(y[4 * k + 2], y[4 * k + 3]));
            most = fmaxf(fmaxf(quarter[0], quarter[1]), fmaxf(quarter[2], quarter[3]));
        };
        look();
        if (most == INFINITY) {
#pragma unroll
            for (int e = 0; e < kEach; ++e) y[e] = y[e] == INFINITY ? -INFINITY : y[e];
            look();
        }
        return most;
    };
    auto add = [&](const float (&y)[kEach], float most) {
        if (most > mine.m) {
            const float d = fmaxf(mine.m - most, -104.0f), by = fa::fast_exp2(d * kLog2e);
            mine.t = (mine.t + mine.s * d) * by;
            mine.s *= by;
            mine.m = most;
        }
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            // 2^-150 is zero here; where the difference is no number (an entry that is none, or a thread without any yet) it is that, too
            const float u = fmaxf(y[e] - mine.m, -104.0f), p = fa::fast_exp2(u * kLog2e);
            mine.s += p;
            mine.t = fmaf(p, u, mine.t);
        }
    };
    // 16 entries a lane, `where(e)` their indices
    auto keep = [&](const float (&y)[kEach], const float (&quarter)[4], float most, auto where) {
        const float others = unordered(*(volatile int*)&shared_bound);   // (at least `top` entries of the row are at or above it)
        if (!__any_sync(0xffffffffu, most >= fmaxf(bound, others) && most > -INFINITY)) return;
        if (others > bound) { bound = others; bound_at = kNone; }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (!__any_sync(0xffffffffu, quarter[k] >= bound && quarter[k] > -INFINITY)) continue;
#pragma unroll
            for (int e = 4 * k; e < 4 * k + 4; ++e) {
                const int index = where(e);
                unsigned who = __ballot_sync(0xffffffffu, y[e] > -INFINITY && (y[e] > bound || (y[e] == bound && index < bound_at)));
                while (who) {
                    const int from = __ffs(who) - 1;
                    who &= who - 1;
                    const float v = __shfl_sync(0xffffffffu, y[e], from);
                    const int i = __shfl_sync(0xffffffffu, index, from);
                    const int rank_of = __popc(__ballot_sync(0xffffffffu, before(best, at, v, i)));
                    const float up = __shfl_up_sync(0xffffffffu, best, 1);
                    const int up_at = __shfl_up_sync(0xffffffffu, at, 1);
                    if (lane > rank_of) { best = up; at = up_at; }
                    if (lane == rank_of) { best = v; at = i; }
                }
            }
            const float last = __shfl_sync(0xffffffffu, best, top - 1);
            if (last >= bound) {
                bound = last;
                bound_at = __shfl_sync(0xffffffffu, at, top - 1);
                if (lane == 0) atomicMax(&shared_bound, ordered(bound));
            }
        }
    };

    // The share tile by tile: whole ones, then the rest, less than a tile, then the row's ends (the lead with the first block, the tail
    // with the last; a thread an entry).  `use(y, tile)` gets 16 entries a lane, minus infinity where there is none.
    constexpr int kTile = kThreads * kEach / kVec;       // vectors of a tile
    const int tiles = (stop - first) / kTile;            // whole ones
    const int tail = lead + vectors * kVec;
    const T* base = x + lead + ((long long)first + tid) * kVec;
    // A share of less than a tile goes to the threads an entry at a time, so that all have some and the warps' largest make a bound
    // (1,000 rows of 700 bfloat16 entries, five likeliest: 55 us in vectors, 15 so; longer ones lose a microsecond by it).
    const bool spread = TOP && tiles == 0;
    auto index_of = [&](int tile, int thread, int e) {   // the entry's, or -1: there is none
        if (tile <= tiles) {
            const int i = spread ? first * kVec + e * kThreads + thread : (first + tile * kTile + e / kVec * kThreads + thread) * kVec + e % kVec;
            return i < stop * kVec ? lead + i : -1;
        }
        if (e == 0 && rank == 0 && thread < lead) return thread;
        return e == 0 && rank == cluster - 1 && thread >= 32 && tail + thread - 32 < vocab ? tail + thread - 32 : -1;
    };
    auto walk = [&](int from, int to, auto use) {        // tiles from .. to - 1; to = tiles + 2: the rest and the ends too
        float y[kEach], next[kEach];
        const int whole = min(to, tiles);
        if (from < whole) load(base + (long long)from * kTile * kVec, next);
#pragma unroll 1
        for (int k = from; k < whole; ++k) {
#pragma unroll
            for (int e = 0; e < kEach; ++e) y[e] = next[e];
            if (k + 1 < whole) load(base + (long long)(k + 1) * kTile * kVec, next);
            use(y, k);
        }
        const int rest = first + tiles * kTile;
        if (to > tiles && rest < stop) {
            if (spread) {
#pragma unroll
                for (int e = 0; e < kEach; ++e) {
                    const int index = index_of(tiles, tid, e);
                    y[e] = index >= 0 ? ldf(x, index) : -INFINITY;
                }
            } else {
#pragma unroll
                for (int k = 0; k < kEach / kVec; ++k) {
                    const int vector = rest + k * kThreads + tid;
                    uint4 v = make_uint4(0, 0, 0, 0);
                    if (vector < stop) v = *reinterpret_cast<const uint4*>(x + lead + (long long)vector * kVec);
                    const T* in = reinterpret_cast<const T*>(&v);
#pragma unroll
                    for (int e = 0; e < kVec; ++e) y[k * kVec + e] = vector < stop ? ldf(in, e) : -INFINITY;
                }
            }
            use(y, tiles);
        }
        if (to > tiles && warp < 2) {
            const int odd = index_of(tiles + 1, tid, 0);
#pragma unroll
            for (int e = 0; e < kEach; ++e) y[e] = -INFINITY;
            if (odd >= 0) y[0] = ldf(x, odd);
            use(y, tiles + 1);
        }
    };

    const int window = !TOP || tiles < 2 * kWindow ? tiles + 2 : kWindow;          // tiles ahead of the first bound
    float largest_tile = -INFINITY, second_tile = -INFINITY;
    int which_tile = 0;
    walk(0, window, [&](float (&y)[kEach], int tile) {
        float quarter[4];
        const float most = largest(y, quarter);
        add(y, most);
        if (TOP && most > largest_tile) {
            second_tile = largest_tile;
            largest_tile = most;
            which_tile = tile;
        } else if (TOP) {
            second_tile = fmaxf(second_tile, most);
        }
    });
    // Into the shared memory of the cluster's block `to`, where `here` lies in this one's; all blocks meet.
    auto there = [&](const void* here, int to) {
        uint32_t remote;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"((uint32_t)__cvta_generic_to_shared(here)), "r"(to));
        return remote;
    };
    auto put = [&](const void* here, int to, uint32_t bits) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(there(here, to)), "r"(bits) : "memory"); };
    auto meet = [&] {
        if (cluster == 1) {
            __syncthreads();
            return;
        }
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    };
    if (cluster > 1) {                                   // all of the cluster's blocks are there: their memory may be written to
        __syncwarp();
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
    bool listed = false;                                 // whether warps have lists
    if constexpr (TOP) {
        // the bound: every warp's `each` largest lanes, and the top-th of all of them
        const int each = (top + kWarps * cluster - 1) / (kWarps * cluster), count = kWarps * cluster * each;        // 64 at most
        int rest = ordered(largest_tile), mine_to_tell = 0;
#pragma unroll 1
        for (int k = 0; k < each; ++k) {
            const int nth = __reduce_max_sync(0xffffffffu, rest);
            const unsigned who = __ballot_sync(0xffffffffu, rest == nth);
            if (lane == __ffs(who) - 1) rest = ordered(-INFINITY);
            if (lane % each == k) mine_to_tell = nth;
        }
        if (lane < cluster * each) put(&named[(rank * kWarps + warp) * each + lane % each], lane / each, (uint32_t)mine_to_tell);
        meet();
        int least = ordered(-INFINITY);
        {
            const int a = lane < count ? named[lane] : ordered(-INFINITY), b = lane + 32 < count ? named[lane + 32] : ordered(-INFINITY);
            int before_a = 0, before_b = 0;
#pragma unroll 4
            for (int k = 0; k < count; ++k) {
                const int v = named[k];
                before_a += v > a || (v == a && k < lane);
                before_b += v > b || (v == b && k < lane + 32);
            }
            if (lane < count && before_a == top - 1) least = a;
            if (lane + 32 < count && before_b == top - 1) least = b;
            least = __reduce_max_sync(0xffffffffu, least);
        }
        const float at_least = unordered(least);
        auto look = [&](int i) {
            if (i < 0) return;
            const float v = ldf(x, i);
            if (!(v >= at_least && fabsf(v) <= 3.402823466e+38f)) return;
            int k;
            asm volatile("atom.shared::cluster.add.s32 %0, [%1], 1;" : "=r"(k) : "r"(there(&found, 0)) : "memory");
            if (k < kFound) {
                put(&found_v[k], 0, __float_as_uint(v));
                put(&found_i[k], 0, (uint32_t)i);
            }
        };
#pragma unroll 1
        for (unsigned who = __ballot_sync(0xffffffffu, largest_tile >= at_least && largest_tile > -INFINITY); who;) {
            // two threads at a time, half a warp each
            const int one = __ffs(who) - 1;
            who &= who - 1;
            const int two = who ? __ffs(who) - 1 : -1;
            who &= who - 1;
            const int from = lane < kEach ? one : two, tile = __shfl_sync(0xffffffffu, which_tile, from & 31);
            const float second = __shfl_sync(0xffffffffu, second_tile, from & 31);           // (all lanes, also where there is no second thread)
            const bool more = from >= 0 && second >= at_least;
            if (from >= 0 && !more) look(index_of(tile, warp * 32 + from, lane % kEach));
            if (more)
#pragma unroll 4
                for (int k = 0; k < window; ++k) look(index_of(k, warp * 32 + from, lane % kEach));
        }
        meet();
        int all_found;
        asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(all_found) : "r"(there(&found, 0)) : "memory");
        listed = all_found > kFound || window < tiles + 2;
        if (tid == 0) shared_bound = least;
        if (all_found > kFound) {                        // (many alike)
            __syncthreads();
            walk(0, window, [&](float (&y)[kEach], int tile) {
                float quarter[4];
                const float most = largest(y, quarter);
                keep(y, quarter, most, [&](int e) { return index_of(tile, tid, e); });
            });
        } else if (rank == 0 && warp == 0) {
#pragma unroll 1
            for (int k = 0; k < all_found; k += 32) {
                float v = k + lane < all_found ? found_v[k + lane] : -INFINITY;
                int i = k + lane < all_found ? found_i[k + lane] : kNone;
                sort(v, i);
                merge(best, at, __shfl_sync(0xffffffffu, v, 31 - lane), __shfl_sync(0xffffffffu, i, 31 - lane));
            }
            bound = __shfl_sync(0xffffffffu, best, top - 1);
            bound_at = __shfl_sync(0xffffffffu, at, top - 1);
            if (lane == 0) shared_bound = ordered(bound);
        }
        if (listed) {
            __syncthreads();                             // (the bound is there)
            if (window < tiles + 2)
                walk(window, tiles + 2, [&](float (&y)[kEach], int tile) {
                    float quarter[4];
                    const float most = largest(y, quarter);
                    add(y, most);
                    keep(y, quarter, most, [&](int e) { return index_of(tile, tid, e); });
                });
        }
    }

    // ---- the warp's, the block's, the cluster's
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        mine = joined(mine, {__shfl_xor_sync(0xffffffffu, mine.m, o), __shfl_xor_sync(0xffffffffu, mine.s, o), __shfl_xor_sync(0xffffffffu, mine.t, o)});
    if (lane == 0) sums[warp] = mine;
    if constexpr (TOP) { list_v[warp][lane] = best; list_i[warp][lane] = at; }
    __syncthreads();
    if constexpr (TOP) {
#pragma unroll 1
        for (int half = kWarps / 2; half > 0 && listed; half >>= 1) {
            if (warp < half) {
                merge(best, at, list_v[warp + half][31 - lane], list_i[warp + half][31 - lane]);
                list_v[warp][lane] = best;
                list_i[warp][lane] = at;
            }
            __syncthreads();
        }
    }
    auto all_of = [&](Summary one, int count) {          // over the first `count` lanes (a power of two), for all lanes
#pragma unroll 1
        for (int o = count >> 1; o > 0; o >>= 1)
            one = joined(one, {__shfl_xor_sync(0xffffffffu, one.m, o), __shfl_xor_sync(0xffffffffu, one.s, o), __shfl_xor_sync(0xffffffffu, one.t, o)});
        return one;
    };
    if (warp == 0) mine = all_of(sums[lane % kWarps], kWarps);
    if (cluster > 1) {
        if (warp == 0) {                                 // to the cluster's first block
            if (lane == 0) {
                put(&blocks[rank].sum.m, 0, __float_as_uint(mine.m));
                put(&blocks[rank].sum.s, 0, __float_as_uint(mine.s));
                put(&blocks[rank].sum.t, 0, __float_as_uint(mine.t));
            }
            if (listed) {
                put(&blocks[rank].v[lane], 0, __float_as_uint(best));
                put(&blocks[rank].i[lane], 0, (uint32_t)at);
            }
        }
        meet();                                          // (and no block is gone while another looks into its memory)
        if (rank != 0) return;
        if (warp == 0) mine = all_of(blocks[lane % cluster].sum, cluster);
        if (listed) {
#pragma unroll 1
            for (int half = cluster / 2; half > 0; half >>= 1) {
                if (warp < half) {
                    best = blocks[warp].v[lane];
                    at = blocks[warp].i[lane];
                    merge(best, at, blocks[warp + half].v[31 - lane], blocks[warp + half].i[31 - lane]);
                    blocks[warp].v[lane] = best;
                    blocks[warp].i[lane] = at;
                }
                __syncthreads();
            }
        }
    }
    if (warp != 0) return;
    const float log_s = logf(mine.s);                    // (no finite entry: log 0, and m is minus infinity)
    const bool some = mine.m > -INFINITY;
    if (lane == 0) {
        entropy[row] = some ? log_s - mine.t / mine.s : 0.0f;
        if (tokens) {
            const int token = tokens[row];
            float lp = __int_as_float(0x7fc00000);       // no such token
            if (token >= 0 && token < vocab) {
                const float v = ldf(x, token);
                lp = fabsf(v) <= 3.402823466e+38f ? v - mine.m - log_s : -INFINITY;
            }
            logprobs[row] = lp;
        }
    }
    if constexpr (TOP) {
        if (lane < top) {
            top_ids[row * top + lane] = at == kNone ? -1 : at;
            top_logprobs[row * top + lane] = at == kNone ? -INFINITY : best - mine.m - log_s;
        }
    }
}

template <typename T, bool TOP>
static int launch(const void* logits, const int32_t* tokens, float* logprobs, float* entropy, int32_t* top_ids, float* top_logprobs, int rows,
                  int vocab, int top, int cluster, cudaStream_t stream) {
    launch_kernel_clustered(token_logprobs_kernel<T, TOP>, dim3((unsigned)(rows * cluster)), kThreads, 0, cluster, stream, (const T*)logits, tokens,
                            logprobs, entropy, top_ids, top_logprobs, vocab, top, cluster);
    return CITLALI_LAUNCH_CHECK();
}

}  // namespace lp
}  // namespace citlali

using namespace citlali;

extern "C" int citlali_token_logprobs(const void* logits, int dtype, const int32_t* tokens, float* logprobs, float* entropy, int32_t* top_ids,
                                      float* top_logprobs, int rows, int vocab, int top, cudaStream_t stream) {
    if (rows <= 0) return 0;
    if (vocab <= 0 || vocab > 0x7fffffff - 65536 || top < 0 || top > lp::kMost || top > vocab || rows > 0x7fffffff / lp::kMaxCluster) {
        set_last_error("token_logprobs: %d rows of %d entries, %d alternatives (at most %d, and no more than entries)", rows, vocab, top, lp::kMost);
        return kBadShape;
    }
    if ((uintptr_t)logits % (dtype == kF32 ? 4 : 2) != 0) {
        set_last_error("token_logprobs: logits are not aligned");
        return kBadAlignment;
    }
    // Blocks a row: more until there are four a multiprocessor, each with two tiles or more (float32, 151,936 entries: 8 rows 32.6 us by
    // one block, 13.7 by four, 10.4 by eight; 1,000 rows 109.5 by one, 151 by two).
    int cluster = 1;
    while (cluster < lp::kMaxCluster && rows * cluster < 4 * device_sm_count() && vocab >= 2 * cluster * lp::kThreads * lp::kEach) cluster *= 2;
    return CITLALI_DISPATCH_FLOAT(dtype, T, [&]() {
        return top > 0 ? lp::launch<T, true>(logits, tokens, logprobs, entropy, top_ids, top_logprobs, rows, vocab, top, cluster, stream)
                       : lp::launch<T, false>(logits, tokens, logprobs, entropy, top_ids, top_logprobs, rows, vocab, top, cluster, stream);
    });
}
