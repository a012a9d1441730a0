// Attention over the cache in 4 bits, in 32-bit arithmetic, for any head size that groups divide and any page size: the 32-bit path's
// kernel, and the one for head sizes that attention4.cu does not take.
//
// A block takes (row, HB query heads that share a key/value head); its eight warps take 32 keys each in turn.  A lane scores one key
// for the HB heads: sum over groups of s_g sum_e c_e q_e, the whole numbers c_e kept apart from their scale until the group is done.
// The warp keeps a running maximum, sum and result (a lane has EPL elements of the result); the eight warps' are merged in warp order.
#include "api.h"
#include "cache4.cuh"
#include "common.cuh"

namespace citlali {
namespace c4 {

constexpr int kRowWarps = 8;

template <typename T, int HB, int EPL>
__global__ void __launch_bounds__(kRowWarps * 32)
attention_rows_kernel(const T* __restrict__ q, size_t q_stride, const uint8_t* __restrict__ k_codes, const uint8_t* __restrict__ k_scales,
                      const uint8_t* __restrict__ v_codes, const uint8_t* __restrict__ v_scales, const int32_t* __restrict__ page_table,
                      int page_table_stride, const int32_t* __restrict__ row_slot, const int32_t* __restrict__ row_pos, T* __restrict__ out,
                      size_t out_stride, int nq, int nkv, int d, int page_size, int window, float scale) {
    extern __shared__ float shared[];                        // queries [HB][d], then the warps' (m, l, result) [kRowWarps][HB][2 + d]
    dependents_may_launch();
    wait_for_predecessor();
    const int row = blockIdx.x, head0 = blockIdx.y * HB, g = head0 / (nq / nkv);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int pos = row_pos[row];
    const int lo = window > 0 && pos - window + 1 > 0 ? pos - window + 1 : 0;
    const int32_t* pages = page_table + (size_t)row_slot[row] * page_table_stride;
    for (int i = threadIdx.x; i < HB * d; i += kRowWarps * 32) shared[i] = ldf(q, (size_t)row * q_stride + (size_t)head0 * d + i) * scale;
    __syncthreads();

    const int e0 = lane * EPL;
    const bool has = e0 < d;
    float m[HB], l[HB], acc[HB][EPL];
#pragma unroll
    for (int h = 0; h < HB; ++h) {
        m[h] = -INFINITY; l[h] = 0.0f;
#pragma unroll
        for (int e = 0; e < EPL; ++e) acc[h][e] = 0.0f;
    }
    for (int first = lo + warp * 32; first <= pos; first += kRowWarps * 32) {
        const int key = first + lane, count = min(32, pos - first + 1);
        size_t at = 0;                                       // the key's row in the pools
        float s[HB];
#pragma unroll
        for (int h = 0; h < HB; ++h) s[h] = -INFINITY;
        if (key <= pos) {
            at = place(pages[key / page_size], nkv, g, page_size, key % page_size);
            const uint32_t* words = reinterpret_cast<const uint32_t*>(k_codes + at * (d / 2));
            const uint8_t* scales = k_scales + at * (d / kGroup);
#pragma unroll
            for (int h = 0; h < HB; ++h) s[h] = 0.0f;
            for (int group = 0; group < d / kGroup; ++group) {
                const float sg = scale_of(scales[group]);
                float part[HB];
#pragma unroll
                for (int h = 0; h < HB; ++h) part[h] = 0.0f;
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    const uint32_t word = words[group * 2 + w];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float c = value_of(word, e, 1.0f);
#pragma unroll
                        for (int h = 0; h < HB; ++h) part[h] = fmaf(c, shared[h * d + group * kGroup + w * 8 + e], part[h]);
                    }
                }
#pragma unroll
                for (int h = 0; h < HB; ++h) s[h] = fmaf(sg, part[h], s[h]);
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
#pragma unroll
            for (int e = 0; e < EPL; ++e) acc[h][e] *= turn;
        }
        for (int j = 0; j < count; ++j) {
            const size_t there = __shfl_sync(0xffffffffu, (unsigned long long)at, j);
            float p[HB];
#pragma unroll
            for (int h = 0; h < HB; ++h) p[h] = __shfl_sync(0xffffffffu, s[h], j);
            if (!has) continue;
            const float sv = scale_of(v_scales[there * (d / kGroup) + e0 / kGroup]);
            const uint8_t* codes = v_codes + there * (d / 2) + e0 / 2;
            uint32_t word = EPL == 8 ? *reinterpret_cast<const uint32_t*>(codes) : *reinterpret_cast<const uint16_t*>(codes);
#pragma unroll
            for (int e = 0; e < EPL; ++e) {
                const float v = value_of(word, e, sv);
#pragma unroll
                for (int h = 0; h < HB; ++h) acc[h][e] = fmaf(p[h], v, acc[h][e]);
            }
        }
    }
    float* parked = shared + HB * d;
#pragma unroll
    for (int h = 0; h < HB; ++h) {
        l[h] = warp_sum(l[h]);
        float* mine = parked + (size_t)(warp * HB + h) * (2 + d);
        if (lane == 0) { mine[0] = l[h] == l[h] ? m[h] : 0.0f; mine[1] = l[h]; }        // (a sum that is no number must count)
        if (has) {
#pragma unroll
            for (int e = 0; e < EPL; ++e) mine[2 + e0 + e] = acc[h][e];
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < HB * d; i += kRowWarps * 32) {
        const int h = i / d, e = i % d;
        float M = -INFINITY;
        for (int w = 0; w < kRowWarps; ++w) M = fmaxf(M, parked[(size_t)(w * HB + h) * (2 + d)]);
        float L = 0.0f, o = 0.0f;
        for (int w = 0; w < kRowWarps; ++w) {
            const float* its = parked + (size_t)(w * HB + h) * (2 + d);
            if (its[0] == -INFINITY) continue;               // a warp that saw no key
            const float f = expf(its[0] - M);
            L = fmaf(its[1], f, L);
            o = fmaf(its[2 + e], f, o);
        }
        stf(out, (size_t)row * out_stride + (size_t)head0 * d + i, o / L);
    }
}

template <typename T, int HB, int EPL>
static int launch_rows(const void* q, size_t q_stride, const void* k_codes, const void* k_scales, const void* v_codes, const void* v_scales,
                       const int32_t* page_table, int page_table_stride, const int32_t* row_slot, const int32_t* row_pos, void* out,
                       size_t out_stride, int rows, int nq, int nkv, int d, int page_size, int window, float scale, cudaStream_t stream) {
    auto kernel = attention_rows_kernel<T, HB, EPL>;
    const size_t bytes = (size_t)HB * (d + kRowWarps * (2 + d)) * sizeof(float);
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
    if (((uintptr_t)k_codes | (uintptr_t)v_codes) & 3u) {
        set_last_error("attention4_rows: codes must be 4-byte aligned");
        return kBadAlignment;
    }
    const int group = nq / nkv, hb = group % 4 == 0 ? 4 : group % 2 == 0 ? 2 : 1;
#define CITLALI_ROWS4(HB, EPL) return c4::launch_rows<T, HB, EPL>(q, q_stride, k_codes, k_scales, v_codes, v_scales, page_table, page_table_stride, \
                                                                  row_slot, row_pos, out, out_stride, rows, nq, nkv, head_dim, page_size, window, scale, stream)
    return CITLALI_DISPATCH_FLOAT(dtype, T, [&]() -> int {
        if (head_dim <= 128) {
            if (hb == 4) CITLALI_ROWS4(4, 4);
            if (hb == 2) CITLALI_ROWS4(2, 4);
            CITLALI_ROWS4(1, 4);
        }
        if (hb == 4) CITLALI_ROWS4(4, 8);
        if (hb == 2) CITLALI_ROWS4(2, 8);
        CITLALI_ROWS4(1, 8);
    });
#undef CITLALI_ROWS4
}
