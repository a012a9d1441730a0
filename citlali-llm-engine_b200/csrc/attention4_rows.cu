// Attention over the cache in 4 bits, in 32-bit arithmetic, for any head size that groups divide and any page size: the 32-bit path's
// kernel, and the one for head sizes that attention4.cu does not take.
//
// A block takes (row, HB query heads that share a key/value head); its sixteen warps take 32 keys each in turn.  A lane scores one key
// for the HB heads.  For the result a key's d / 8 words of codes go to as many lanes, so that a warp works on 256 / d keys at once; the
// weights go through shared memory.  A warp keeps a running maximum and sum, and its groups of lanes a result each; all are merged in
// order.  What bounds it: the latency of a few dependent reads a turn where rows are few, and the multiply-adds where they are many.
// Measured: five rows over 40 to 1,500 keys, 12 heads over 4 of 64, 14.1 us; 64 rows over 1,000 keys, 16 heads over 4 of 128, 46.
#include "api.h"
#include "cache4.cuh"
#include "common.cuh"

namespace citlali {
namespace c4 {

constexpr int kRowWarps = 16;

// A word's eight values as floats.
__device__ __forceinline__ void floats_of(uint32_t w, float s, float (&y)[8]) {
    uint32_t v[4];
    values_of(w, s, v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        y[2 * i] = __uint_as_float(v[i] << 16);
        y[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
    }
}

// Of a block's shared memory: queries [HB][d], weights and places of the warps' keys, the parts (m, l, result) of the warps' groups of lanes.
__host__ __device__ inline int keys_at_once(int d) { return 256 / d; }
__host__ __device__ inline size_t rows_shared_bytes(int heads, int d) {
    return (size_t)heads * d * 4 + (size_t)kRowWarps * 32 * (8 + 4 * heads) + (size_t)kRowWarps * keys_at_once(d) * heads * (2 + d) * 4;
}

template <typename T, int HB>
__global__ void __launch_bounds__(kRowWarps * 32)
attention_rows_kernel(const T* __restrict__ q, size_t q_stride, const uint8_t* __restrict__ k_codes, const uint8_t* __restrict__ k_scales,
                      const uint8_t* __restrict__ v_codes, const uint8_t* __restrict__ v_scales, const int32_t* __restrict__ page_table,
                      int page_table_stride, const int32_t* __restrict__ row_slot, const int32_t* __restrict__ row_pos, T* __restrict__ out,
                      size_t out_stride, int nq, int nkv, int d, int page_size, int window, float scale) {
    extern __shared__ __align__(16) float shared[];
    dependents_may_launch();
    const int row = blockIdx.x, head0 = blockIdx.y * HB, g = head0 / (nq / nkv);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int pos = row_pos[row];                            // (positions, slots and page tables come from the host before the step)
    const int lo = window > 0 && pos - window + 1 > 0 ? pos - window + 1 : 0;
    const int32_t* pages = page_table + (size_t)row_slot[row] * page_table_stride;
    unsigned long long* places = reinterpret_cast<unsigned long long*>(shared + HB * d) + warp * 32;
    float* weights = shared + HB * d + kRowWarps * 64 + warp * 32 * HB;              // [key][HB]
    float* parked = shared + HB * d + kRowWarps * 32 * (2 + HB);
    wait_for_predecessor();
    for (int i = threadIdx.x; i < HB * d; i += kRowWarps * 32) shared[i] = ldf(q, (size_t)row * q_stride + (size_t)head0 * d + i) * scale;
    __syncthreads();

    const int words = d / 8, at_once = keys_at_once(d), group = lane / words, word = lane - group * words;
    float m[HB], l[HB], acc[HB][8];
#pragma unroll
    for (int h = 0; h < HB; ++h) {
        m[h] = -INFINITY; l[h] = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[h][e] = 0.0f;
    }
    for (int first = lo + warp * 32; first <= pos; first += kRowWarps * 32) {
        const int key = first + lane, count = min(32, pos - first + 1);
        float s[HB];
#pragma unroll
        for (int h = 0; h < HB; ++h) s[h] = -INFINITY;
        if (key <= pos) {
            const size_t at = place(pages[key / page_size], nkv, g, page_size, key % page_size);       // the key's row in the pools
            places[lane] = at;
            const uint2* codes = reinterpret_cast<const uint2*>(k_codes + at * (d / 2));
            const uint8_t* scales = k_scales + at * (d / kGroup);
#pragma unroll
            for (int h = 0; h < HB; ++h) s[h] = 0.0f;
#pragma unroll 4
            for (int i = 0; i < d / kGroup; ++i) {
                const uint2 w = codes[i];
                const float sg = scale_of(scales[i]);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    float y[8];
                    floats_of(half ? w.y : w.x, sg, y);
#pragma unroll
                    for (int h = 0; h < HB; ++h) {
                        const float4* x = reinterpret_cast<const float4*>(shared + h * d + i * kGroup + 8 * half);
                        const float4 a = x[0], b = x[1];
                        s[h] = fmaf(y[0], a.x, fmaf(y[1], a.y, fmaf(y[2], a.z, fmaf(y[3], a.w, s[h]))));
                        s[h] = fmaf(y[4], b.x, fmaf(y[5], b.y, fmaf(y[6], b.z, fmaf(y[7], b.w, s[h]))));
                    }
                }
            }
        }
#pragma unroll
        for (int h = 0; h < HB; ++h) {
            const float most = fmaxf(m[h], warp_max(s[h]));
            const float to = most == -INFINITY ? 0.0f : most;        // scores that are no numbers leave no maximum
            const float turn = expf(m[h] - to);
            s[h] = key <= pos ? expf(s[h] - to) : 0.0f;
            l[h] = l[h] * turn + s[h];
            m[h] = most;
            weights[lane * HB + h] = s[h];
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[h][e] *= turn;
        }
        __syncwarp();
        if (group < at_once) {
#pragma unroll 4
            for (int j = group; j < count; j += at_once) {
                const size_t at = places[j];
                const uint32_t w = reinterpret_cast<const uint32_t*>(v_codes + at * (d / 2))[word];
                float y[8];
                floats_of(w, scale_of(v_scales[at * (d / kGroup) + word / 2]), y);
#pragma unroll
                for (int h = 0; h < HB; ++h) {
                    const float p = weights[j * HB + h];
#pragma unroll
                    for (int e = 0; e < 8; ++e) acc[h][e] = fmaf(p, y[e], acc[h][e]);
                }
            }
        }
        __syncwarp();
    }
    const int parts = kRowWarps * at_once;
#pragma unroll
    for (int h = 0; h < HB; ++h) {
        l[h] = warp_sum(l[h]);
        if (group < at_once) {
            float* mine = parked + (size_t)((warp * at_once + group) * HB + h) * (2 + d);
            // (a sum that is no number must count; the warp's first group has the warp's sum)
            if (word == 0) { mine[0] = l[h] == l[h] ? m[h] : 0.0f; mine[1] = group == 0 ? l[h] : 0.0f; }
#pragma unroll
            for (int e = 0; e < 8; ++e) mine[2 + word * 8 + e] = acc[h][e];
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < HB * d; i += kRowWarps * 32) {
        const int h = i / d, e = i % d;
        float M = -INFINITY;
        for (int w = 0; w < parts; w += at_once) M = fmaxf(M, parked[(size_t)(w * HB + h) * (2 + d)]);
        float L = 0.0f, o = 0.0f;
        for (int w = 0; w < parts; ++w) {
            const float* its = parked + (size_t)(w * HB + h) * (2 + d);
            if (its[0] == -INFINITY) continue;               // a warp that saw no key
            const float f = expf(its[0] - M);
            L = fmaf(its[1], f, L);
            o = fmaf(its[2 + e], f, o);
        }
        stf(out, (size_t)row * out_stride + (size_t)head0 * d + i, o / L);
    }
}

template <typename T, int HB>
static int launch_rows(const void* q, size_t q_stride, const void* k_codes, const void* k_scales, const void* v_codes, const void* v_scales,
                       const int32_t* page_table, int page_table_stride, const int32_t* row_slot, const int32_t* row_pos, void* out,
                       size_t out_stride, int rows, int nq, int nkv, int d, int page_size, int window, float scale, cudaStream_t stream) {
    auto kernel = attention_rows_kernel<T, HB>;
    const size_t bytes = rows_shared_bytes(HB, d);
    if (int e = raise_shared_limit(kernel, bytes, kRowShared)) return e;
    launch_kernel(kernel, dim3(rows, nq / HB), kRowWarps * 32, bytes, stream, (const T*)q, q_stride, (const uint8_t*)k_codes,
                  (const uint8_t*)k_scales, (const uint8_t*)v_codes, (const uint8_t*)v_scales, page_table, page_table_stride, row_slot,
                  row_pos, (T*)out, out_stride, nq, nkv, d, page_size, window, scale);
    return CITLALI_LAUNCH_CHECK();
}

}  // namespace c4
}  // namespace citlali

using namespace citlali;

extern "C" int citlali_attention4_rows(const void* q, size_t q_stride, int dtype, const void* k_codes, const void* k_scales,
                                       const void* v_codes, const void* v_scales, const int32_t* page_table, int page_table_stride,
                                       const int32_t* row_slot, const int32_t* row_pos, void* out, size_t out_stride, int rows, int nq,
                                       int nkv, int head_dim, int page_size, int window, float scale, cudaStream_t stream) {
    if (rows <= 0) return 0;
    if (nq <= 0 || nkv <= 0 || nq % nkv != 0 || nq > 65535 || head_dim < c4::kGroup || head_dim % c4::kGroup != 0 || head_dim > 256
        || page_size <= 0 || window < 0) {
        set_last_error("attention4_rows: %d query heads over %d key/value heads of %d (a multiple of 16 up to 256), pages of %d, window %d",
                       nq, nkv, head_dim, page_size, window);
        return kBadShape;
    }
    if (((uintptr_t)k_codes | (uintptr_t)v_codes) & 7u) {
        set_last_error("attention4_rows: codes must be 8-byte aligned");
        return kBadAlignment;
    }
    // Heads a block: as many as share a key/value head, four at most, but fewer where a block for each keeps more multiprocessors busy.
    // (16 heads over 4 of 128: one row over 4,000 keys 43 us a head a block, 70 four; 64 rows over 1,000 77 and 46.)
    const int group = nq / nkv, widest = group % 4 == 0 ? 4 : group % 2 == 0 ? 2 : 1;
    int hb = widest;
    while (hb > 1 && (long long)rows * (nq / hb) < device_sm_count()) hb /= 2;
#define CITLALI_ROWS4(HB) return c4::launch_rows<T, HB>(q, q_stride, k_codes, k_scales, v_codes, v_scales, page_table, page_table_stride, \
                                                                  row_slot, row_pos, out, out_stride, rows, nq, nkv, head_dim, page_size, window, scale, stream)
    return CITLALI_DISPATCH_FLOAT(dtype, T, [&]() -> int {
        if (hb == 4) CITLALI_ROWS4(4);
        if (hb == 2) CITLALI_ROWS4(2);
        CITLALI_ROWS4(1);
    });
#undef CITLALI_ROWS4
}
