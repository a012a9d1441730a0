// The cache in 4 bits: appending a step's keys and values to it, with head norms and rotation on the way, and reading rows back.
//
// append does what qk_norm_rope_cache (attention_generic.cu) does for a cache of 16 or 32 bits: for every row of the projection
// [q | k | v], y = x / sqrt(mean x^2 + eps) gain on the q and k heads, pairs (i, i + rotated / 2) turned by pos inv_freq[i], then the
// queries back to memory and keys and values into the row's page, here as codes and scales (cache4.cuh).  Nothing is rounded between.
//
// The angle.  pos inv_freq[i] in 32 bits is off by up to 2^-24 of itself, 0.004 at position 65,536: as much as a bfloat16 query's own
// rounding.  The product's rounding error e is one fma away, and cos(a + e) = cos a - e sin a to 32 bits, so it is put right.
//
// What bounds it: instructions.  A group's codes are whole numbers nearest to exact quotients, some 9 instructions an element; with norm and
// rotation 30 an element of a key (2,048 rows of 16 + 8 + 8 heads of 128: 10.9 us for 30 MB, issue slots 0.65 busy; 8 rows 2.5 us).  Reading
// back is bound by what it writes (2,048 rows: 4.8 us for 11 MB; 8 rows 2.1).
#include "api.h"
#include "cache4.cuh"
#include "common.cuh"

namespace citlali {
namespace c4 {

constexpr int kThreads = 128;
constexpr int kWarps = 8;          // of the form that takes any size

__device__ __forceinline__ float2 turn_of(int pos, float f) {
    const float p = (float)pos, a = p * f, e = fmaf(p, f, -a);       // positions are below 2^24
    float sn, cs;
    sincosf(a, &sn, &cs);
    return make_float2(fmaf(-e, sn, cs), fmaf(e, cs, sn));
}

__device__ __forceinline__ void load8(const float* p, float (&f)[8]) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&f)[8]) {
    const uint4 w = *reinterpret_cast<const uint4*>(p);
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&w);
#pragma unroll
    for (int i = 0; i < 4; ++i) { const float2 v = __bfloat1622float2(h[i]); f[2 * i] = v.x; f[2 * i + 1] = v.y; }
}
__device__ __forceinline__ void store8(float* p, const float (&f)[8]) {
    *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(f[4], f[5], f[6], f[7]);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&f)[8]) {
    uint4 w;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&w);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = w;
}

// The eight values of a word of codes.
__device__ __forceinline__ void store_values(__nv_bfloat16* p, uint32_t w, float s) {
    uint32_t v[4];
    values_of(w, s, v);
    *reinterpret_cast<uint4*>(p) = make_uint4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void store_values(float* p, uint32_t w, float s) {
    uint32_t v[4];
    values_of(w, s, v);
    uint4* out = reinterpret_cast<uint4*>(p);
    out[0] = make_uint4(v[0] << 16, v[0] & 0xffff0000u, v[1] << 16, v[1] & 0xffff0000u);
    out[1] = make_uint4(v[2] << 16, v[2] & 0xffff0000u, v[3] << 16, v[3] & 0xffff0000u);
}

struct Pools {
    uint8_t *k_codes, *k_scales, *v_codes, *v_scales;
};
struct Rows {
    const int32_t *row_slot, *row_pos, *page_table;
    int page_table_stride, page_size;
};

// Eight elements of half a group (its other half is the neighbouring lane's): their word of codes and the group's byte.
__device__ __forceinline__ void put8(uint8_t* codes, uint8_t* scales, size_t at, int d, int e, const float (&x)[8], bool on) {
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) most = max(most, magnitude(x[i]));
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
    if (!on) return;
    float s;
    const int byte = scale_byte(most, s);
    *reinterpret_cast<uint32_t*>(codes + at * (d / 2) + e / 2) = codes_of(x, s);
    if (e % kGroup == 0) scales[at * (d / kGroup) + e / kGroup] = (uint8_t)byte;
}

// `lanes` = d / 16 neighbouring lanes share a head.  Lane p < rotated / 16 has elements 8p .. 8p + 7 and their partners rotated / 2
// further on; the lanes behind share the elements that are not rotated the same way.  Sizes are such that an even lane and the next
// one always hold the two halves of one group (rotated and the rest multiples of 32).
template <typename T, typename TG>
__global__ void __launch_bounds__(kThreads)
append_kernel(const T* __restrict__ qkv, T* q_out, size_t q_out_stride, const TG* __restrict__ q_gain, const TG* __restrict__ k_gain,
              const float* __restrict__ inv_freq, int rotated, const __grid_constant__ Rows rows, const __grid_constant__ Pools pools,
              int nq, int nkv, int d, float eps, int store, int heads_per_block, int lanes) {
    extern __shared__ __align__(16) float2 turns[];                  // the row's [element of a lane's eight][lane], shared by the block's heads
    dependents_may_launch();
    // positions, slots and page tables come from the host before the step: the turns and the row's place in the cache are worked
    // out while the kernel ahead (the projection) is still running
    const int row = blockIdx.x;
    const int total = nq + 2 * nkv, used = store ? total : nq;
    const int begin = blockIdx.y * heads_per_block, end = min(used, begin + heads_per_block);
    const int half = rotated >> 1;
    const int pos = rows.row_pos[row];
    if (begin < nq + nkv)
        for (int i = threadIdx.x; i < half; i += kThreads) turns[(i & 7) * (half >> 3) + (i >> 3)] = turn_of(pos, inv_freq[i]);
    int page = 0;
    if (store) page = rows.page_table[(size_t)rows.row_slot[row] * rows.page_table_stride + pos / rows.page_size];
    __syncthreads();
    wait_for_predecessor();
    const T* in = qkv + (size_t)row * total * d;
    const int part = threadIdx.x % lanes, pairs = half >> 3;
    const bool turned = part < pairs;
    const int rest = d - rotated;
    const int e0 = turned ? 8 * part : rotated + 8 * (part - pairs), e1 = e0 + (turned ? half : rest >> 1);
    const int heads_per_pass = kThreads / lanes;
    for (int h0 = begin; h0 < end; h0 += heads_per_pass) {           // the same trip count for every lane
        const int head = h0 + threadIdx.x / lanes;
        const bool on = head < end;
        float x0[8], x1[8];
        if (on) {
            load8(in + (size_t)head * d + e0, x0);
            load8(in + (size_t)head * d + e1, x1);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x0[i] = x1[i] = 0.0f;
        }
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) { ss = fmaf(x0[i], x0[i], ss); ss = fmaf(x1[i], x1[i], ss); }
        for (int o = lanes >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const bool is_q = head < nq, is_v = head >= nq + nkv;
        if (on && !is_v) {
            const TG* gain = is_q ? q_gain : k_gain;
            if (gain) {
                const float inv = rsqrtf(ss / (float)d + eps);
                float g0[8], g1[8];
                load8(gain + e0, g0);
                load8(gain + e1, g1);
#pragma unroll
                for (int i = 0; i < 8; ++i) { x0[i] = x0[i] * inv * g0[i]; x1[i] = x1[i] * inv * g1[i]; }
            }
            if (turned) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float2 t = turns[i * pairs + part];
                    const float a = x0[i], b = x1[i];
                    x0[i] = a * t.x - b * t.y;
                    x1[i] = b * t.x + a * t.y;
                }
            }
        }
        if (on && is_q) {
            T* out = q_out + (size_t)row * q_out_stride + (size_t)head * d;
            store8(out + e0, x0);
            store8(out + e1, x1);
        }
        const bool cached = on && !is_q;
        const size_t at = cached ? place(page, nkv, (head - nq) % nkv, rows.page_size, pos % rows.page_size) : 0;
        uint8_t* codes = is_v ? pools.v_codes : pools.k_codes;
        uint8_t* scales = is_v ? pools.v_scales : pools.k_scales;
        put8(codes, scales, at, d, e0, x0, cached);                  // (every lane: a group's two lanes exchange their maxima)
        put8(codes, scales, at, d, e1, x1, cached);
    }
}

// Any head size that groups divide and any even number of rotated elements: a warp a head, the head in shared memory.
template <typename T, typename TG>
__global__ void __launch_bounds__(kWarps * 32)
append_any_kernel(const T* __restrict__ qkv, T* q_out, size_t q_out_stride, const TG* __restrict__ q_gain, const TG* __restrict__ k_gain,
                  const float* __restrict__ inv_freq, int rotated, const __grid_constant__ Rows rows, const __grid_constant__ Pools pools,
                  int nq, int nkv, int d, float eps, int store) {
    extern __shared__ float shared[];                                // [kWarps][d], then the turns [rotated / 2]
    float2* turns = reinterpret_cast<float2*>(shared + kWarps * d);
    dependents_may_launch();
    const int row = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int total = nq + 2 * nkv, used = store ? total : nq;
    const int half = rotated >> 1;
    const int pos = rows.row_pos[row];
    for (int i = threadIdx.x; i < half; i += kWarps * 32) turns[i] = turn_of(pos, inv_freq[i]);
    int page = 0;
    if (store) page = rows.page_table[(size_t)rows.row_slot[row] * rows.page_table_stride + pos / rows.page_size];
    __syncthreads();
    wait_for_predecessor();
    float* y = shared + warp * d;
    for (int head = blockIdx.y * kWarps + warp; head < used; head += gridDim.y * kWarps) {
        const T* in = qkv + ((size_t)row * total + head) * d;
        const bool is_q = head < nq, is_v = head >= nq + nkv;
        const TG* gain = is_v ? nullptr : (is_q ? q_gain : k_gain);
        float ss = 0.0f;
        for (int i = lane; i < d; i += 32) {
            const float x = ldf(in, i);
            y[i] = x;
            ss = fmaf(x, x, ss);
        }
        ss = warp_sum(ss);
        __syncwarp();
        if (!is_v) {
            const float inv = gain ? rsqrtf(ss / (float)d + eps) : 1.0f;
            for (int i = lane; i < half; i += 32) {
                const float a = gain ? y[i] * inv * ldf(gain, i) : y[i], b = gain ? y[i + half] * inv * ldf(gain, i + half) : y[i + half];
                y[i] = a * turns[i].x - b * turns[i].y;
                y[i + half] = b * turns[i].x + a * turns[i].y;
            }
            if (gain)
                for (int i = rotated + lane; i < d; i += 32) y[i] = y[i] * inv * ldf(gain, i);
            __syncwarp();
        }
        if (is_q) {
            T* out = q_out + (size_t)row * q_out_stride + (size_t)head * d;
            for (int i = lane; i < d; i += 32) stf(out, i, y[i]);
        } else {
            uint8_t* codes = is_v ? pools.v_codes : pools.k_codes;
            uint8_t* scales = is_v ? pools.v_scales : pools.k_scales;
            const size_t at = place(page, nkv, (head - nq) % nkv, rows.page_size, pos % rows.page_size);
            for (int g = lane; g < d / kGroup; g += 32) {
                uint32_t most = 0;
                for (int i = 0; i < kGroup; ++i) most = max(most, magnitude(y[g * kGroup + i]));
                float s;
                scales[at * (d / kGroup) + g] = (uint8_t)scale_byte(most, s);
                for (int half = 0; half < 2; ++half) {
                    float x[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[i] = y[g * kGroup + 8 * half + i];
                    const uint32_t w = codes_of(x, s);
                    uint8_t* out = codes + at * (d / 2) + (g * kGroup) / 2 + 4 * half;       // (any alignment)
#pragma unroll
                    for (int i = 0; i < 4; ++i) out[i] = (uint8_t)(w >> (8 * i));
                }
            }
        }
        __syncwarp();
    }
}

// keys[r, h, :], values[r, h, :] = what the cache holds for position positions[r] of slot slots[r]; NaN where there is no such slot,
// position or page.  A thread a group.
template <typename TO>
__global__ void __launch_bounds__(kThreads)
read_kernel(const __grid_constant__ Rows rows, const __grid_constant__ Pools pools, TO* __restrict__ keys, TO* __restrict__ values,
            long long groups, int slots, int pages, int nkv, int d) {
    dependents_may_launch();
    wait_for_predecessor();
    const int per_head = d / kGroup;
    const long long i = (long long)blockIdx.x * kThreads + threadIdx.x;
    if (i >= groups) return;
    const bool is_v = blockIdx.y != 0;
    const int g = (int)(i % per_head), head = (int)(i / per_head % nkv);
    const long long row = i / ((long long)per_head * nkv);
    const int pos = rows.row_pos[row], slot = rows.row_slot[row], index = pos / rows.page_size;
    const bool named = slot >= 0 && slot < slots && pos >= 0 && index < rows.page_table_stride;
    const int page = named ? rows.page_table[(size_t)slot * rows.page_table_stride + index] : -1;
    uint2 w = make_uint2(0, 0);
    float s = __int_as_float(0x7fc00000);
    if (page >= 0 && page < pages) {
        const size_t at = place(page, nkv, head, rows.page_size, pos % rows.page_size);
        w = *reinterpret_cast<const uint2*>((is_v ? pools.v_codes : pools.k_codes) + at * (d / 2) + g * 8);
        s = scale_of((is_v ? pools.v_scales : pools.k_scales)[at * per_head + g]);
    }
    TO* out = (is_v ? values : keys) + ((size_t)row * nkv + head) * d + g * kGroup;
    store_values(out, w.x, s);
    store_values(out + 8, w.y, s);
}

// The pages that a run's rows see, as bfloat16 pages of their own (exact), with a page table and slots for the attention kernels of a
// cache of 16 bits: sequence b is slot b there.  A block a (page, key/value head, keys or values).  Positions that no row of the run sees become
// zeros.  A value that is no number becomes zero too, and its token's key none: a row that does not see the token gives it the
// weight zero, and zero times a NaN would reach it; a row that does see it gets a NaN from the key.  (2,048 positions of 8 heads of 128:
// 5 to 10 us with caches cold, bound by what it writes.)
struct Runs {
    const int32_t *seq_start, *seq_slot, *seq_past;
    int sequences, window;
};
constexpr int kExpandThreads = 256, kRunPage = 64;
__global__ void __launch_bounds__(kExpandThreads)
expand_kernel(const __grid_constant__ Runs runs, const int32_t* __restrict__ page_table, int page_table_stride,
              const __grid_constant__ Pools pools, __nv_bfloat16* __restrict__ keys, __nv_bfloat16* __restrict__ values,
              int32_t* __restrict__ table_out, int table_out_stride, int32_t* __restrict__ slots_out, int nkv, int d) {
    dependents_may_launch();
    const int lane = threadIdx.x & 31, head = blockIdx.y;
    // the sequence of this page: every warp finds it for itself (lists and page tables come from the host before the step)
    auto tiles_of = [&](int b, int& first) {
        const int past = runs.seq_past[b], fresh = runs.seq_start[b + 1] - runs.seq_start[b];
        first = runs.window > 0 ? max(0, past - runs.window + 1) / kRunPage & ~1 : 0;        // (the kernels read pairs of pages)
        return fresh > 0 ? (past + fresh - 1) / kRunPage - first + 1 : 0;
    };
    int b = -1, tile = 0, run = 0;
    for (int b0 = 0; b0 < runs.sequences && b < 0; b0 += 32) {
        int first, mine = b0 + lane < runs.sequences ? tiles_of(b0 + lane, first) : 0, sum = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += up;
        }
        const unsigned behind = __ballot_sync(0xffffffffu, run + sum > (int)blockIdx.x);
        if (behind) {
            const int which = __ffs(behind) - 1;
            b = b0 + which;
            tile = (int)blockIdx.x - run - __shfl_sync(0xffffffffu, sum - mine, which);
        }
        run += __shfl_sync(0xffffffffu, sum, 31);
    }
    wait_for_predecessor();
    if (b < 0) return;
    int first;
    tiles_of(b, first);
    tile += first;
    if (tile >= table_out_stride) return;
    const int past = runs.seq_past[b], last = past + runs.seq_start[b + 1] - runs.seq_start[b] - 1;
    const int low = runs.window > 0 ? max(0, past - runs.window + 1) : 0;
    if (head == 0 && blockIdx.z == 0 && threadIdx.x == 0) {
        table_out[(size_t)b * table_out_stride + tile] = blockIdx.x;
        if (tile == first) slots_out[b] = b;
    }
    const int page = page_table[(size_t)runs.seq_slot[b] * page_table_stride + tile];
    const int per_row = d / kGroup;
    const bool is_v = blockIdx.z != 0;
    const size_t from0 = place(page, nkv, head, kRunPage, 0), to0 = place(blockIdx.x, nkv, head, kRunPage, 0);
    const uint8_t* codes = (is_v ? pools.v_codes : pools.k_codes) + from0 * (d / 2);
    const uint8_t *own = (is_v ? pools.v_scales : pools.k_scales) + from0 * per_row, *others = pools.v_scales + from0 * per_row;
    __nv_bfloat16* out = (is_v ? values : keys) + to0 * d;
#pragma unroll 2
    for (int i = threadIdx.x; i < kRunPage * per_row; i += kExpandThreads) {     // (a group's row and place follow from i alone)
        const int row = i / per_row, pos = tile * kRunPage + row;
        const uint2 w = *reinterpret_cast<const uint2*>(codes + i * 8);
        const uint8_t byte = own[i];
        bool none = false;                               // of the token's values
        if (is_v) {
            none = byte >= 0xf8;
        } else if (per_row % 4 == 0) {
            for (int k = 0; k < per_row; k += 4) none |= __vcmpgeu4(*reinterpret_cast<const uint32_t*>(others + row * per_row + k), 0xf8f8f8f8u) != 0;
        } else {
            for (int k = 0; k < per_row; ++k) none |= others[row * per_row + k] >= 0xf8;
        }
        __nv_bfloat16* to = out + (size_t)i * kGroup;
        if (pos < low || pos > last) {
            reinterpret_cast<uint4*>(to)[0] = reinterpret_cast<uint4*>(to)[1] = make_uint4(0, 0, 0, 0);
            continue;
        }
        const float s = !none ? scale_of(byte) : is_v ? 0.0f : __int_as_float(0x7fc00000);
        store_values(to, w.x, s);
        store_values(to + 8, w.y, s);
    }
}

static int check_sizes(const char* what, int nkv, int d, int page_size) {
    if (d < kGroup || d % kGroup != 0 || d > 256) {
        set_last_error("%s: a cache in 4 bits takes head sizes that are multiples of %d up to 256, not %d", what, kGroup, d);
        return kBadShape;
    }
    if (nkv <= 0 || page_size <= 0) {
        set_last_error("%s: bad number of key/value heads (%d) or page size (%d)", what, nkv, page_size);
        return kBadShape;
    }
    return 0;
}

static bool aligned(const void* p, size_t bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }

template <typename T, typename TG>
static int launch_append(const T* qkv, T* q_out, size_t q_out_stride, const TG* q_gain, const TG* k_gain, const float* inv_freq, int rotated,
                         const Rows& where, const Pools& pools, int rows, int nq, int nkv, int d, float eps, int store, cudaStream_t stream) {
    const int used = store ? nq + 2 * nkv : nq, lanes = d / 16;
    const bool in_pairs = d >= 32 && (lanes & (lanes - 1)) == 0 && rotated % 32 == 0 && (d - rotated) % 32 == 0;
    const bool wide = aligned(qkv, 16) && aligned(q_out, 16) && q_out_stride * sizeof(T) % 16 == 0 && aligned(q_gain, 16)
                      && aligned(k_gain, 16) && aligned(pools.k_codes, 4) && aligned(pools.v_codes, 4);
    if (in_pairs && wide) {
        // few rows: a pass of heads a block, so that the heads spread over the SMs; many rows: a row a block, whose turns serve all heads
        // (16 + 8 + 8 heads of 128: 2,048 rows 10.9 us a row a block, some 12 by passes; 8 rows 3.3 and 2.5)
        const int pass = kThreads / lanes, blocks = rows >= 4 * device_sm_count() ? 1 : (used + pass - 1) / pass;
        const int each = blocks == 1 ? used : pass;
        launch_kernel(append_kernel<T, TG>, dim3(rows, blocks), kThreads, (size_t)(rotated / 2) * sizeof(float2), stream, qkv, q_out,
                      q_out_stride, q_gain, k_gain, inv_freq, rotated, where, pools, nq, nkv, d, eps, store, each, lanes);
    } else {
        const int blocks = rows >= 4 * device_sm_count() ? 1 : (used + kWarps - 1) / kWarps;
        launch_kernel(append_any_kernel<T, TG>, dim3(rows, blocks), kWarps * 32, (size_t)(kWarps * d + rotated) * sizeof(float), stream, qkv,
                      q_out, q_out_stride, q_gain, k_gain, inv_freq, rotated, where, pools, nq, nkv, d, eps, store);
    }
    return CITLALI_LAUNCH_CHECK();
}

}  // namespace c4
}  // namespace citlali

using namespace citlali;

extern "C" int citlali_cache4_append(const void* qkv, int dtype, void* q_out, size_t q_out_stride, const void* q_gain, const void* k_gain,
                                     int gain_dtype, const float* inv_freq, int rotary_dim, const int32_t* row_slot, const int32_t* row_pos,
                                     const int32_t* page_table, int page_table_stride, void* k_codes, void* k_scales, void* v_codes,
                                     void* v_scales, int page_size, int rows, int nq, int nkv, int head_dim, float eps, int store,
                                     cudaStream_t stream) {
    if (rows <= 0) return 0;
    if (int bad = c4::check_sizes("cache4_append", store ? nkv : 1, head_dim, page_size)) return bad;
    if (nq < 0 || nkv < 0 || nq + 2 * nkv <= 0 || (!store && nq == 0) || rotary_dim < 0 || rotary_dim % 2 != 0 || rotary_dim > head_dim) {
        set_last_error("cache4_append: bad head counts (%d, %d), or a rotated part (%d) that is odd or larger than the head (%d)", nq, nkv,
                       rotary_dim, head_dim);
        return kBadShape;
    }
    if (nq + 2 * nkv > 65535) {
        set_last_error("cache4_append: too many heads (%d)", nq + 2 * nkv);
        return kTooLarge;
    }
    const c4::Rows where = {row_slot, row_pos, page_table, page_table_stride, page_size};
    const c4::Pools pools = {(uint8_t*)k_codes, (uint8_t*)k_scales, (uint8_t*)v_codes, (uint8_t*)v_scales};
    return CITLALI_DISPATCH_FLOAT(dtype, T, [&]() {
        return CITLALI_DISPATCH_FLOAT(gain_dtype, TG, [&]() {
            return c4::launch_append<T, TG>((const T*)qkv, (T*)q_out, q_out_stride, (const TG*)q_gain, (const TG*)k_gain, inv_freq, rotary_dim,
                                            where, pools, rows, nq, nkv, head_dim, eps, store, stream);
        });
    });
}

extern "C" int citlali_cache4_read(const void* k_codes, const void* k_scales, const void* v_codes, const void* v_scales,
                                   const int32_t* page_table, int page_table_rows, int page_table_stride, int page_size, int pages,
                                   const int32_t* slots, const int32_t* positions, void* keys, void* values, int out_dtype, int rows,
                                   int nkv, int head_dim, cudaStream_t stream) {
    if (rows <= 0) return 0;
    if (int bad = c4::check_sizes("cache4_read", nkv, head_dim, page_size)) return bad;
    if (!c4::aligned(k_codes, 8) || !c4::aligned(v_codes, 8) || !c4::aligned(keys, 16) || !c4::aligned(values, 16)) {
        set_last_error("cache4_read: codes must be 8-byte and rows 16-byte aligned");
        return kBadAlignment;
    }
    const long long groups = (long long)rows * nkv * (head_dim / c4::kGroup), blocks = (groups + c4::kThreads - 1) / c4::kThreads;
    if (blocks > 0x7fffffffLL) {
        set_last_error("cache4_read: too many rows (%d)", rows);
        return kTooLarge;
    }
    const c4::Rows where = {slots, positions, page_table, page_table_stride, page_size};
    const c4::Pools pools = {(uint8_t*)k_codes, (uint8_t*)k_scales, (uint8_t*)v_codes, (uint8_t*)v_scales};
    return CITLALI_DISPATCH_FLOAT(out_dtype, TO, [&]() {
        launch_kernel(c4::read_kernel<TO>, dim3((unsigned)blocks, 2), c4::kThreads, 0, stream, where, pools, (TO*)keys, (TO*)values, groups,
                      page_table_rows, pages, nkv, head_dim);
        return CITLALI_LAUNCH_CHECK();
    });
}

extern "C" int citlali_cache4_expand(const void* k_codes, const void* k_scales, const void* v_codes, const void* v_scales,
                                     const int32_t* page_table, int page_table_stride, const int32_t* seq_start, const int32_t* seq_slot,
                                     const int32_t* seq_past, int sequences, int window, void* keys, void* values, int pages,
                                     int32_t* table_out, int table_out_stride, int32_t* slots_out, int page_size, int nkv, int head_dim,
                                     cudaStream_t stream) {
    if (sequences <= 0 || pages <= 0) return 0;
    if (int bad = c4::check_sizes("cache4_expand", nkv, head_dim, page_size)) return bad;
    if (page_size != c4::kRunPage || nkv > 65535 || window < 0) {
        set_last_error("cache4_expand: pages of %d (only of 64), %d heads, window %d", page_size, nkv, window);
        return kBadShape;
    }
    if (!c4::aligned(k_codes, 8) || !c4::aligned(v_codes, 8) || !c4::aligned(v_scales, 4) || !c4::aligned(keys, 16) || !c4::aligned(values, 16)) {
        set_last_error("cache4_expand: codes must be 8-byte, scales 4-byte and pages 16-byte aligned");
        return kBadAlignment;
    }
    const c4::Runs runs = {seq_start, seq_slot, seq_past, sequences, window};
    const c4::Pools pools = {(uint8_t*)k_codes, (uint8_t*)k_scales, (uint8_t*)v_codes, (uint8_t*)v_scales};
    launch_kernel(c4::expand_kernel, dim3(pages, nkv, 2), c4::kExpandThreads, 0, stream, runs, page_table, page_table_stride, pools,
                  (__nv_bfloat16*)keys, (__nv_bfloat16*)values, table_out, table_out_stride, slots_out, nkv, head_dim);
    return CITLALI_LAUNCH_CHECK();
}
