// Attention of runs of new tokens over the cache in 4 bits on the fifth-generation tensor cores (bfloat16 queries, pages of 64 keys, head
// sizes 64 and 128).
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(f q . k_j - m),  f = scale log2(e),  over the keys lo..pos that a row sees
//
// A tile is 128 rows: pairs (token, query head) of one sequence and key/value head.  A block owns a multiprocessor and has a tile and the
// pages that its tokens see, or a cluster of 2, 4 or 8 blocks shares the pages.  A page is a step, four are under way:
//   warps 8-15  put its codes back, two threads a key, warps 8-11 the even pages and 12-15 the odd ones: the codes come from memory into
//               registers a page ahead, and go to shared memory as halves c s / 8 (exact, cache4.cuh) in rows of 128 bytes with the 128-byte
//               swizzle, keys ahead of values.
//   warps 16, 17  one lane each issues the products (tcgen05.mma, 128 rows, float sums): S = Q K^T as far ahead as there is room, and
//               O += P V with P in tensor memory over the scores that it came from, and V as it was stored (its rows are the contraction).
//   warps 0-7   a thread a row, warps 0-3 the even pages and 4-7 the odd ones: the largest of 64 scores, read from tensor memory; the row's
//               reference m, which goes from page to page between the two threads of a row and only has to keep weights in range (it is
//               renewed, and O scaled, where a weight would exceed 2^15); then the weights, read again, as halves, and their sum.
// The element order.  (w & 0x000f000f) | 0x6400 is a pair (i, i + 4) of a word's eight elements, so elements lie in the order 0 4 1 5 2 6
// 3 7 in shared memory.  Queries have the same order, and results are put right on their way out.
// Queries are made halves after they were multiplied by a power of two that puts the row's largest into [2^14, 2^15): exact for every
// element above 2^-28 of that.  P is rounded to half (half a step is 2^-11 of it); the reference is such that the largest weight is 2^6 or
// more, so a half that is subnormal is off by 2^-31 of it at most.
// A value that is no number becomes zero, and its token's key none: a row that does not see the token gives it the weight zero, and zero
// times a NaN would reach it; a row that does see it gets a NaN from the key.
// A cluster's blocks leave O, m and the sum in their shared memory, and each merges an even share of the rows, always in the same order.
//
// What bounds it: a page takes 1,280 clocks, of which the products take 512 and the exponentials 512 (16 a clock); the rest is the issue
// of what puts codes back and of the softmax (issue slots half used) and the latencies between the roles.  A block spends about 4 us beside
// its pages.  With the softmax on four warps and two blocks a multiprocessor a page took 2,300 clocks a block; with one issuing lane for both
// products 2,700, since an MMA takes it 60 clocks and telling a barrier 200.  Measured (16 heads over 8 of 128): a prompt of 2,048 tokens 34 us
// (over pages made bfloat16 first: 53), eight of 512 40 (48), 64 new tokens over 32,768 56 (by the kernel for single tokens: 116).
// All waits are bounded; one that runs out reports through the error word, and the block's results are NaN.
#include "api.h"
#include "cache4.cuh"
#include "common.cuh"
#include "mma_common.cuh"
#include "tc_common.cuh"

namespace citlali {
namespace c4 {

using namespace tc;

constexpr int kRunRows = 128, kRunKeys = 64, kRunThreads = 576, kRunCluster = 8;
constexpr int kSoftWarps = 8, kLoadWarps = 8, kScoreWarp = 16;            // (and one more for the values' products)
constexpr int kStages = 4;                                           // pages under way
constexpr float kRunBits = 6.0f, kRunMost = 15.0f;                   // log2 of the largest weight when m is renewed, and above which it is
constexpr float kNothingYet = -3.402823466e+38f;
constexpr uint32_t kRunColumns = 512, kColScores = 0, kColOut = kStages * kRunKeys;         // of tensor memory; the scores of so many pages
constexpr uint32_t kRegion = kRunKeys * 128;                         // bytes of 64 keys by 64 elements

template <int D>
struct RunLayout {
    static constexpr uint32_t part = D / 64 * kRegion, stage = 2 * part;         // keys (or values) of a page, and both
    static constexpr uint32_t queries = 2 * part;                    // ahead of the stages
    static constexpr uint32_t needed = queries + kStages * stage + 1024, bytes = needed > 120 * 1024 ? needed : 120 * 1024;
    static_assert(bytes + 8192 <= 227 * 1024 && 2 * bytes > 227 * 1024, "one block fits, and no second");
    static_assert(kRunRows * D * 4 <= kStages * stage, "a block's results take the stages' place");
};

struct Runs4 {
    const __nv_bfloat16* q;
    size_t q_stride;
    const uint8_t *k_codes, *k_scales, *v_codes, *v_scales;
    const int32_t* table;
    int table_stride;
    const int32_t *seq_start, *seq_slot, *seq_past;
    __nv_bfloat16* out;
    size_t out_stride;
    int sequences, nq, nkv, group, tokens;                           // tokens: of a tile
    int least;                                                       // sequences with fewer new tokens are left out
    int window, cluster;
    float scale_log2;
    int32_t* error_flag;
};

// Four products over 16 elements of the contraction each, by the lane that has `go`.  The whole warp comes here, so that descriptors stay
// in registers that all lanes share (a page took 15 % longer with one lane alone), and what changes between the four is an addition to
// a descriptor.  A in shared memory, 32 bytes further from one to the next as B is; or in tensor memory, with B's rows the contraction.
__device__ __forceinline__ void mma_four(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate, uint32_t go) {
    asm volatile(
        "{\n.reg .pred p, yes, go;\n.reg .b64 a, b;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "setp.ne.b32 go, %5, 0;\n"
        "setp.eq.u32 yes, 0, 0;\n"
        "@go tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n"
        "add.u64 a, %1, 2;\n add.u64 b, %2, 2;\n"
        "@go tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, yes;\n"
        "add.u64 a, %1, 4;\n add.u64 b, %2, 4;\n"
        "@go tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, yes;\n"
        "add.u64 a, %1, 6;\n add.u64 b, %2, 6;\n"
        "@go tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, yes;\n}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(go) : "memory");
}
__device__ __forceinline__ void mma_four_rows(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate, uint32_t go) {
    asm volatile(
        "{\n.reg .pred p, yes, go;\n.reg .b32 a;\n.reg .b64 b;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "setp.ne.b32 go, %5, 0;\n"
        "setp.eq.u32 yes, 0, 0;\n"
        "@go tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
        "add.u32 a, %1, 8;\n add.u64 b, %2, 128;\n"
        "@go tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, yes;\n"
        "add.u32 a, %1, 16;\n add.u64 b, %2, 256;\n"
        "@go tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, yes;\n"
        "add.u32 a, %1, 24;\n add.u64 b, %2, 384;\n"
        "@go tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, yes;\n}"
        ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(go) : "memory");
}
__device__ __forceinline__ uint32_t elected() {
    uint32_t r;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.b32 %0, 1, 0, p;\n}" : "=r"(r));
    return r;
}
__device__ __forceinline__ void commit_if(uint32_t bar, uint32_t go) {
    asm volatile("{\n.reg .pred go;\nsetp.ne.b32 go, %1, 0;\n@go tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}" ::"r"(bar), "r"(go) : "memory");
}
// Half operands, float sums, M x N; the B operand's rows are N, or (`rows_are_k`) the contraction.
__host__ __device__ constexpr uint32_t instr_desc_half(int m, int n, bool rows_are_k) {
    return (1u << 4) | (rows_are_k ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// An operand of rows of 128 bytes with the 128-byte swizzle whose rows are the contraction: the next 64 of the other dimension lie
// `step` bytes further.
__device__ __forceinline__ uint64_t smem_desc_rows_are_k(uint32_t addr, uint32_t step) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | (uint64_t)((step >> 4) & 0x3FFFu) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 |
           (uint64_t)2 << 61;
}
// Columns of the thread's lane: loads (to be waited for), the waits (the registers go through them), and stores.
#define CITLALI_R32(r) "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), \
    "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), \
    "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), \
    "=r"(r[30]), "=r"(r[31])
__device__ __forceinline__ void tmem_load32(uint32_t at, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : CITLALI_R32(r) : "r"(at) : "memory");
}
__device__ __forceinline__ void tmem_wait16(uint32_t* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
                   "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]) :: "memory");
}
__device__ __forceinline__ void tmem_wait32(uint32_t* r) {
    tmem_wait16(r);
    tmem_wait16(r + 16);
}
__device__ __forceinline__ void tmem_store32(uint32_t at, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
        ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
          "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
          "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
          "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]) : "memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t at, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                   "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
#undef CITLALI_R32
__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ uint32_t packed(float low, float high) {
    const __half2 x = __floats2half2_rn(low, high);
    return *reinterpret_cast<const uint32_t*>(&x);
}
// From another block of the cluster (what it holds does not change any more).
__device__ __forceinline__ float2 load2_cluster(uint32_t at) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at));
    return v;
}
__device__ __forceinline__ float4 load4_cluster(uint32_t at) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at));
    return v;
}

// What a thread loads of a key and its value: half of either's codes and scales.
template <int D>
struct HalfKey {
    uint4 k[D / 64], v[D / 64];
    uint32_t k_scales, v_scales;                                     // D / 32 bytes
};

template <int D>
__global__ void __launch_bounds__(kRunThreads, 1)
attention4_runs_kernel(const __grid_constant__ Runs4 a) {
    using L = RunLayout<D>;
    extern __shared__ uint8_t raw[];
    __shared__ __align__(8) uint64_t q_full, k_full[kStages], v_full[kStages], v_empty[kStages], s_full[kStages], p_full[kStages], m_known[2][4];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_word;
    __shared__ float row_factor[kRunRows];                           // what takes a row's scores to powers of two
    __shared__ float row_m[kRunRows], row_l[2][kRunRows];            // the reference, and the sums of the even and the odd pages' weights
    __shared__ float2 row_sums[kRunRows];                            // (m, l)
    __shared__ float row_weights[kRunRows];                          // of the blocks' parts of this block's rows [row][block]
    __shared__ __nv_bfloat16* row_out[kRunRows];
    volatile int* abort_flag = &abort_word;
    const uint32_t queries = (smem_u32(raw) + 1023u) & ~1023u, base = queries + L::queries;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const int cluster = a.cluster, rank = (int)blockIdx.x % cluster;

    // the block's tile, the last tiles (which see the most) first; lists and page tables come from the host before the step
    int b = -1, segment = 0;
    {
        const int wanted = (int)gridDim.x / cluster - 1 - (int)blockIdx.x / cluster;
        int run = 0;
#pragma unroll 1
        for (int b0 = 0; b0 < a.sequences && b < 0; b0 += 32) {
            int mine = 0;
            if (b0 + lane < a.sequences) mine = a.seq_start[b0 + lane + 1] - a.seq_start[b0 + lane];
            mine = mine < a.least ? 0 : (mine + a.tokens - 1) / a.tokens * a.nkv;
            int sum = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += up;
            }
            const unsigned behind = __ballot_sync(0xffffffffu, run + sum > wanted);
            if (behind) {
                const int which = __ffs(behind) - 1;
                b = b0 + which;
                segment = wanted - run - __shfl_sync(0xffffffffu, sum - mine, which);
            }
            run += __shfl_sync(0xffffffffu, sum, 31);
        }
    }
    if (b < 0) {                                                     // (all of a cluster's threads alike)
        dependents_may_launch();
        wait_for_predecessor();
        return;
    }
    const int row0 = a.seq_start[b], fresh = a.seq_start[b + 1] - row0, past = a.seq_past[b];
    const int kv = segment % a.nkv, token0 = segment / a.nkv * a.tokens, tokens = min(a.tokens, fresh - token0), used = tokens * a.group;
    const int pos0 = past + token0, last = pos0 + tokens - 1;        // of the tile's first and last token
    const int first_page = a.window > 0 ? max(0, pos0 - a.window + 1) / kRunKeys : 0, all = last / kRunKeys - first_page + 1;
    const int share = (all + cluster - 1) / cluster, page0 = first_page + min(all, rank * share);
    const int pages = min(share, max(0, all - rank * share));        // this block's
    const int32_t* table = a.table + (size_t)a.seq_slot[b] * a.table_stride + page0;

    if (tid == 0) {
        abort_word = 0;
        mbar_init(smem_u32(&q_full), kSoftWarps + kLoadWarps);
        for (int i = 0; i < kStages; ++i) {
            mbar_init(smem_u32(&k_full[i]), kLoadWarps / 2);
            mbar_init(smem_u32(&v_full[i]), kLoadWarps / 2);
            mbar_init(smem_u32(&v_empty[i]), 1);
            mbar_init(smem_u32(&s_full[i]), 1);
            mbar_init(smem_u32(&p_full[i]), kSoftWarps / 2);
        }
        for (int i = 0; i < 8; ++i) mbar_init(smem_u32(&m_known[i >> 2][i & 3]), 1);
        fence_barrier_init();
        fence_async_proxy();
    }
    if (tid < kRunRows) {
        const int token = tid / a.group;
        row_out[tid] = a.out + (size_t)(row0 + token0 + token) * a.out_stride + (size_t)(kv * a.group + tid - token * a.group) * D;
    }
    if (warp == kScoreWarp) {
        tmem_alloc(smem_u32(&tmem_slot), kRunColumns);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    dependents_may_launch();                                         // only now: this block holds its tensor memory
    wait_for_predecessor();

    // ---- the first page's codes (a thread half a key and value), then the queries, by the warps of both kinds, eight rows each
    // (a quarter of a warp: eight rows of shared memory, which meet no bank twice)
    const int key = (warp & 3) * 16 + (lane & 15), half = lane >> 4, odd = warp >> 2 & 1;      // (odd: of a warp that takes the odd pages)
    auto fetch = [&](HalfKey<D>& x, int page) {
        const size_t at = place(page, a.nkv, kv, kRunKeys, key);
        const uint4 *kc = reinterpret_cast<const uint4*>(a.k_codes + at * (D / 2) + half * (D / 4)),
                    *vc = reinterpret_cast<const uint4*>(a.v_codes + at * (D / 2) + half * (D / 4));
#pragma unroll
        for (int i = 0; i < D / 64; ++i) { x.k[i] = __ldcg(kc + i); x.v[i] = __ldcg(vc + i); }
        const size_t scales = at * (D / kGroup) + half * (D / 32);
        if constexpr (D == 128) {
            x.k_scales = __ldcg(reinterpret_cast<const uint32_t*>(a.k_scales + scales));
            x.v_scales = __ldcg(reinterpret_cast<const uint32_t*>(a.v_scales + scales));
        } else {
            x.k_scales = __ldcg(reinterpret_cast<const uint16_t*>(a.k_scales + scales));
            x.v_scales = __ldcg(reinterpret_cast<const uint16_t*>(a.v_scales + scales));
        }
    };
    HalfKey<D> next = {};
    int page_after = 0;
    if (warp >= kSoftWarps && warp < kSoftWarps + kLoadWarps && pages > odd) {
        if (pages > odd + 2) page_after = table[odd + 2];
        fetch(next, table[odd]);
    }
    if (warp < kSoftWarps + kLoadWarps) {
        // D / 8 lanes a row: a lane's pieces all on their way at once, then made halves
        constexpr int lanes_of = D / 8, at_once = 32 / lanes_of;
        constexpr int rows_of = kRunRows / (kSoftWarps + kLoadWarps);
        const int piece = lane % lanes_of, first = warp * rows_of;
        auto at = [&](int r) { return queries + (piece / 8) * (kRunRows * 128) + r * 128 + (((piece & 7) ^ (r & 7)) << 4); };
        size_t from = 0;
        {
            const int r = min(first + lane % rows_of, used - 1), t = r / a.group;
            from = (size_t)(row0 + token0 + t) * a.q_stride + (size_t)(kv * a.group + r - t * a.group) * D;
        }
        uint4 its[rows_of / at_once];
#pragma unroll
        for (int i = 0; i < rows_of / at_once; ++i) {
            const int k = lane / lanes_of + i * at_once;
            const uint4* src = reinterpret_cast<const uint4*>(a.q + __shfl_sync(0xffffffffu, from, k) + 8 * piece);
            its[i] = first + k < used ? *src : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < rows_of / at_once; ++i) {
            const int k = lane / lanes_of + i * at_once;
            const uint4 in = its[i];
            uint32_t most = __vimax3_u16x2(in.x & 0x7fff7fffu, in.y & 0x7fff7fffu, __vmaxu2(in.z & 0x7fff7fffu, in.w & 0x7fff7fffu));
            most = max(most << 16, most & 0x7fff0000u);
#pragma unroll
            for (int o = 1; o < lanes_of; o <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
            const int up = min(100, max(-113, 14 + 127 - (int)(most >> 23)));
            const float by = copysignf(__int_as_float((127 + up) << 23), a.scale_log2);
            auto two = [&](uint32_t low, uint32_t high) {            // the words' lower elements, and their upper ones
                return make_uint2(packed(__uint_as_float(low << 16) * by, __uint_as_float(high << 16) * by),
                                  packed(__uint_as_float(low & 0xffff0000u) * by, __uint_as_float(high & 0xffff0000u) * by));
            };
            const uint2 even = two(in.x, in.z), odd = two(in.y, in.w);           // elements (0, 4), (1, 5) and (2, 6), (3, 7)
            st_shared_v4(at(first + k), even.x, even.y, odd.x, odd.y);
            if (piece == 0) row_factor[first + k] = __int_as_float((127 - up) << 23) * (fabsf(a.scale_log2) * kUnit);
        }
        fence_async_proxy();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&q_full));
    }

    float m = kNothingYet, l = 0.0f;                                 // of the softmax threads' rows
    const uint32_t lanes = (uint32_t)(warp & 3) * 32 << 16;
    if (warp < kSoftWarps) {
        // ---- a page's scores, weights and sum: the even pages' warps 0-3, the odd pages' warps 4-7, a thread a row
        const int quarter = warp & 3, row = tid % kRunRows, token = row / a.group;
        const bool on = row < used;
        mbar_wait(smem_u32(&q_full), 0, abort_flag, a.error_flag, 401);
        __syncwarp();
        const float factor = row_factor[row];
        const int pos = on ? pos0 + token : -1, low = a.window > 0 ? pos - a.window + 1 : 0;
#pragma unroll 1
        for (int i = odd; i < pages; i += 2) {
            const int stage = i % kStages;
            const uint32_t at_scores = tmem + lanes + kColScores + stage * kRunKeys;
            if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&s_full[stage]), i / kStages & 1u, abort_flag, a.error_flag, 402))) break;
            tc_fence_after();
            const int key0 = (page0 + i) * kRunKeys;
            // pages that some of the tile's tokens see in part (rows behind its last have queries of zeros, and are not stored)
            const bool border = key0 + kRunKeys - 1 > pos0 || (a.window > 0 && key0 <= last - a.window);
            const float by = border ? 1.0f : factor;
            uint32_t x[32];
            auto scores = [&](int c0) {
                tmem_load32(at_scores + c0, x);
                tmem_wait32(x);
                if (border) {
#pragma unroll
                    for (int c = 0; c < 32; ++c) {
                        const int at = key0 + c0 + c;
                        x[c] = __float_as_uint(at > pos || at < low ? -INFINITY : __uint_as_float(x[c]) * factor);
                    }
                }
            };
            float top = kNothingYet;
#pragma unroll 1
            for (int c0 = 0; c0 < kRunKeys; c0 += 32) {
                scores(c0);
#pragma unroll
                for (int c = 0; c < 32; ++c) top = fmaxf(top, __uint_as_float(x[c]));
            }
            top *= by;                                               // (not negative: the queries have the scale's sign)
            // the reference as the page before leaves it, and as this one does
            float before = kNothingYet;
            if (i > 0) {
                if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&m_known[odd ^ 1][quarter]), (i - 1) >> 1 & 1u, abort_flag, a.error_flag, 403))) break;
                before = row_m[row];
            }
            const bool renew = __any_sync(0xffffffffu, top - before > kRunMost);
            const float now = renew ? fmaxf(before, top - kRunBits) : before;
            row_m[row] = now;
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&m_known[odd][quarter]));
            l *= fa::fast_exp2(m - now);
            m = now;
            float sums[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
            for (int c0 = 0; c0 < kRunKeys; c0 += 32) {
                scores(c0);
#pragma unroll
                for (int c = 0; c < 16; ++c) {
                    const float u = fa::fast_exp2(fmaf(__uint_as_float(x[2 * c]), by, -m)), v = fa::fast_exp2(fmaf(__uint_as_float(x[2 * c + 1]), by, -m));
                    sums[c & 3] += u + v;
                    x[c] = packed(u, v);
                }
                tmem_store16(at_scores + c0 / 2, x);        // (over scores that have been read)
            }
            l += (sums[0] + sums[1]) + (sums[2] + sums[3]);
            if (renew && i > 0) {
                // (the product with the page before must have ended)
                if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&v_empty[(i - 1) % kStages]), (i - 1) / kStages & 1u, abort_flag, a.error_flag, 404))) break;
                tc_fence_after();
                const float turn = fa::fast_exp2(before - now);
#pragma unroll 1
                for (int c = 0; c < D; c += 32) {
                    tmem_load32(tmem + lanes + kColOut + c, x);
                    tmem_wait32(x);
#pragma unroll
                    for (int k = 0; k < 32; ++k) x[k] = __float_as_uint(__uint_as_float(x[k]) * turn);
                    tmem_store32(tmem + lanes + kColOut + c, x);
                }
            }
            tmem_store_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&p_full[stage]));
        }
        if (pages > 0) {
            const int end = pages - 1;
            if ((end & 1) != odd) mbar_wait(smem_u32(&m_known[odd ^ 1][quarter]), end >> 1 & 1u, abort_flag, a.error_flag, 405);
            const float now = row_m[row];                            // (of the last page)
            l *= fa::fast_exp2(m - now);
            if (!odd) row_sums[row].x = now;
            mbar_wait(smem_u32(&v_empty[end % kStages]), end / kStages & 1u, abort_flag, a.error_flag, 406);
        } else if (!odd) {
            row_sums[row].x = kNothingYet;
        }
        row_l[odd][row] = l;
        __syncwarp();
        tc_fence_after();
    } else if (warp < kSoftWarps + kLoadWarps) {
        // ---- a page's keys and values
        constexpr int words = D / 16;                                // of a thread's half of a key
        const Words pairs;
        // chunk c (16 bytes) of row `key` lies at c ^ (key & 7)
        auto put = [&](uint32_t region, const uint4 (&codes)[D / 64], uint32_t scales) {
            const uint32_t to = region + (D == 128 ? half * kRegion : 64u * half) + key * 128;           // (a multiple of 64)
            const uint32_t swap = (key & 7) << 4;
#pragma unroll
            for (int i = 0; i < words; ++i) {
                const uint32_t w = i % 4 == 0 ? codes[i / 4].x : i % 4 == 1 ? codes[i / 4].y : i % 4 == 2 ? codes[i / 4].z : codes[i / 4].w;
                const Scale scale(((scales >> (4 * (i & ~1))) & 0xffu) * 0x00010001u);
                st_shared_v4((to + 16 * i) ^ swap, pairs.first_of(w, scale), pairs.second_of(w, scale), pairs.first_of(w >> 8, scale),
                             pairs.second_of(w >> 8, scale));
            }
        };
#pragma unroll 1
        for (int i = odd; i < pages; i += 2) {
            const HalfKey<D> x = next;
            if (i + 2 < pages) {
                fetch(next, page_after);
                if (i + 4 < pages) page_after = table[i + 4];
            }
            const int place_of = i % kStages;
            const uint32_t stage = base + place_of * L::stage, turn = i / kStages & 1u;
            // the scores of the page that was here have come out: its keys' place is free
            if (i >= kStages && !__all_sync(0xffffffffu, mbar_wait(smem_u32(&s_full[place_of]), turn ^ 1u, abort_flag, a.error_flag, 407))) break;
            const uint32_t bad = __vcmpgeu4(x.v_scales, 0xf8f8f8f8u);
            const bool none = (bad | __shfl_xor_sync(0xffffffffu, bad, 16)) != 0;
            put(stage, x.k, none ? 0xffffffffu : x.k_scales);
            fence_async_proxy();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&k_full[place_of]));
            if (i >= kStages && !__all_sync(0xffffffffu, mbar_wait(smem_u32(&v_empty[place_of]), turn ^ 1u, abort_flag, a.error_flag, 408))) break;
            put(stage + L::part, x.v, x.v_scales & ~bad);
            fence_async_proxy();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&v_full[place_of]));
        }
    } else if (warp == kScoreWarp) {
        // ---- the scores' products
        constexpr uint32_t form = instr_desc_half(kRunRows, kRunKeys, false);
        const uint64_t asked = smem_desc_sw128(queries, 0), keys = smem_desc_sw128(base, 0);
        const uint32_t go = elected();
        if (pages > 0 && __all_sync(0xffffffffu, mbar_wait(smem_u32(&q_full), 0, abort_flag, a.error_flag, 409))) {
#pragma unroll 1
            for (int i = 0; i < pages; ++i) {
                const int stage = i % kStages;
                const uint32_t turn = i / kStages & 1u;
                // (their place held the weights of a page before, which have been multiplied with its values)
                if (i >= kStages && !__all_sync(0xffffffffu, mbar_wait(smem_u32(&v_empty[stage]), turn ^ 1u, abort_flag, a.error_flag, 410))) break;
                if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&k_full[stage]), turn, abort_flag, a.error_flag, 411))) break;
                tc_fence_after();
#pragma unroll
                for (int k = 0; k < D / 64; ++k)
                    mma_four(tmem + kColScores + stage * kRunKeys, asked + k * (kRunRows * 128 >> 4), keys + stage * (L::stage >> 4) + k * (kRegion >> 4),
                             form, k > 0, go);
                commit_if(smem_u32(&s_full[stage]), go);
            }
        }
    } else {
        // ---- the values' products
        const uint32_t go = elected();
        constexpr uint32_t form = instr_desc_half(kRunRows, D, true);
        const uint64_t vals = smem_desc_rows_are_k(base + L::part, kRegion);
#pragma unroll 1
        for (int i = 0; i < pages; ++i) {
            const int stage = i % kStages;
            const uint32_t turn = i / kStages & 1u;
            if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&v_full[stage]), turn, abort_flag, a.error_flag, 412) &&
                                             mbar_wait(smem_u32(&p_full[stage]), turn, abort_flag, a.error_flag, 413))) break;
            tc_fence_after();
            mma_four_rows(tmem + kColOut, tmem + kColScores + stage * kRunKeys, vals + stage * (L::stage >> 4), form, i > 0, go);
            commit_if(smem_u32(&v_empty[stage]), go);
        }
    }
    __syncwarp();

    // ---- the rows' parts, or their results: all pages have been read, so they take the stages' place, in 16-byte pieces that swap places so
    // that a quarter of a warp meets no bank twice
    __syncthreads();
    if (warp < kSoftWarps) {
        const int row = tid % kRunRows;
        const float sum = *abort_flag ? __int_as_float(0x7fc00000) : row_l[0][row] + row_l[1][row], by = kUnit / sum;
        if (!odd) row_sums[row].y = sum;
        // (half of the elements each)
#pragma unroll 1
        for (int c = odd * (D / 2); c < odd * (D / 2) + D / 2; c += 32) {
            uint32_t o[32];
            tmem_load32(tmem + lanes + kColOut + c, o);
            tmem_wait32(o);
            if (cluster == 1) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    float y[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) y[e] = __uint_as_float(o[8 * k + e]) * by;
                    st_shared_v4(base + row * (2 * D) + (((c / 8 + k) ^ (row & 7)) << 4), fa::pack_bf16(y[0], y[2]), fa::pack_bf16(y[4], y[6]),
                                 fa::pack_bf16(y[1], y[3]), fa::pack_bf16(y[5], y[7]));
                }
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const uint32_t to = base + (row * D << 2) + (((c / 4 + k) ^ (row & 7)) << 4);
                    if (pages > 0) st_shared_v4(to, o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
                    else st_shared_v4(to, 0, 0, 0, 0);
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kScoreWarp) {
        if (*abort_flag) __nanosleep(100000);                        // products that are still under way end meanwhile
        __syncwarp();
        tmem_dealloc(tmem, kRunColumns);
    }
    if (cluster == 1) {
#pragma unroll 4
        for (int i = tid; i < used * (D / 8); i += kRunThreads) {
            const int row = i / (D / 8), piece = i % (D / 8);
            *reinterpret_cast<uint4*>(row_out[row] + 8 * piece) = ld_shared_v4(base + row * (2 * D) + ((piece ^ (row & 7)) << 4));
        }
        return;
    }
    __syncwarp();
    cluster_sync_all();                                              // every block's parts are there
    const int rows = kRunRows / cluster, mine = rank * rows, count = min(rows, used - mine);             // this block's of them
    if (tid < kRunRows) {                                            // a thread a row and block
        const int row = tid / cluster, k = tid % cluster;
        const float2 ml = load2_cluster(cluster_addr(smem_u32(&row_sums[mine + row]), (rank + k) & (cluster - 1)));
        float M = ml.x;
#pragma unroll 1
        for (int o = 1; o < cluster; o <<= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
        const float by = fa::fast_exp2(ml.x - M);
        float sum = ml.y * by;
#pragma unroll 1
        for (int o = 1; o < cluster; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        row_weights[tid] = by * (kUnit / sum);
    }
    __syncthreads();
    // A thread a 16-byte piece of a row, from its own block's part on (all of them at one block's door would wait there): elements 0 4 1 5
    // of eight, or 2 6 3 7, which it puts right with its neighbour
    constexpr int per_pass = kRunThreads / (D / 4);                  // rows
    const int piece = tid % (D / 4);
    auto finish = [&](int row, const float (&y)[4]) {                // (all lanes)
        const uint32_t here = fa::pack_bf16(y[0], y[2]), there = fa::pack_bf16(y[1], y[3]);              // (0, 1) or (2, 3), (4, 5) or (6, 7)
        const uint32_t other = __shfl_xor_sync(0xffffffffu, piece & 1 ? here : there, 1);
        if (row < mine + count) *reinterpret_cast<uint2*>(row_out[row] + 4 * piece) = piece & 1 ? make_uint2(other, there) : make_uint2(here, other);
    };
    auto at = [&](int row) { return base + (row * D << 2) + ((piece ^ (row & 7)) << 4); };
#pragma unroll 1
    for (int i = tid / (D / 4); i - tid / (D / 4) < count; i += per_pass) {
        const int row = mine + i, known = min(i, count - 1);
        const uint32_t here = at(min(row, kRunRows - 1));
        float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
        for (int k = 0; k < cluster; ++k) {
            const float4 v = load4_cluster(cluster_addr(here, (rank + k) & (cluster - 1)));
            const float w = row_weights[known * cluster + k];
            y[0] = fmaf(v.x, w, y[0]); y[1] = fmaf(v.y, w, y[1]); y[2] = fmaf(v.z, w, y[2]); y[3] = fmaf(v.w, w, y[3]);
        }
        finish(row, y);
    }
    __syncwarp();
    cluster_sync_all();                                              // no block is gone while another reads its parts
}

template <int D>
static int launch_runs(const Runs4& a, int tiles, cudaStream_t stream) {
    auto kernel = attention4_runs_kernel<D>;
    constexpr int bytes = (int)RunLayout<D>::bytes;
    if (int e = raise_shared_limit(kernel, bytes, bytes)) return e;
    launch_kernel_clustered(kernel, dim3((unsigned)(tiles * a.cluster)), kRunThreads, bytes, a.cluster, stream, a);
    return CITLALI_LAUNCH_CHECK();
}

}  // namespace c4
}  // namespace citlali

using namespace citlali;

// The tokens of a tile; 0: the kernel does not take these sizes.
extern "C" int citlali_attention4_runs_tokens(int nq, int nkv, int head_dim, int page_size) {
    if (nq <= 0 || nkv <= 0 || nq % nkv != 0 || page_size != c4::kRunKeys || (head_dim != 64 && head_dim != 128)) return 0;
    return c4::kRunRows / (nq / nkv);
}

extern "C" int citlali_attention4_runs(const void* q, size_t q_stride, const void* k_codes, const void* k_scales, const void* v_codes,
                                       const void* v_scales, const int32_t* page_table, int page_table_stride, const int32_t* seq_start,
                                       const int32_t* seq_slot, const int32_t* seq_past, void* out, size_t out_stride, int sequences,
                                       int least_new, int tiles, int cluster, int nq, int nkv, int head_dim, int page_size, int window, float scale,
                                       int32_t* error_flag, cudaStream_t stream) {
    if (sequences <= 0 || tiles <= 0) return 0;
    const int tokens = citlali_attention4_runs_tokens(nq, nkv, head_dim, page_size);
    if (tokens == 0 || window < 0) {
        set_last_error("attention4_runs: no kernel for %d query heads over %d key/value heads of %d with pages of %d, window %d (head sizes 64 "
                       "and 128, pages of 64, at most 128 query heads a key/value head)", nq, nkv, head_dim, page_size, window);
        return kBadShape;
    }
    if (cluster < 1 || cluster > c4::kRunCluster || (cluster & (cluster - 1)) != 0 || tiles > 0x7fffffff / c4::kRunCluster) {
        set_last_error("attention4_runs: %d tiles in clusters of %d (1, 2, 4 or 8 blocks)", tiles, cluster);
        return kBadShape;
    }
    if (q_stride % 8 != 0 || out_stride % 8 != 0 ||
        (((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_codes | (uintptr_t)k_scales | (uintptr_t)v_codes | (uintptr_t)v_scales) & 15u)) {
        set_last_error("attention4_runs: query rows, results, codes and scales must be 16-byte aligned (pitches of %zu and %zu elements)", q_stride,
                       out_stride);
        return kBadAlignment;
    }
    c4::Runs4 a = {};
    a.q = (const __nv_bfloat16*)q; a.q_stride = q_stride;
    a.k_codes = (const uint8_t*)k_codes; a.k_scales = (const uint8_t*)k_scales;
    a.v_codes = (const uint8_t*)v_codes; a.v_scales = (const uint8_t*)v_scales;
    a.table = page_table; a.table_stride = page_table_stride;
    a.seq_start = seq_start; a.seq_slot = seq_slot; a.seq_past = seq_past;
    a.out = (__nv_bfloat16*)out; a.out_stride = out_stride;
    a.sequences = sequences; a.nq = nq; a.nkv = nkv; a.group = nq / nkv; a.tokens = tokens;
    a.least = least_new > 1 ? least_new : 1;
    a.window = window; a.cluster = cluster; a.scale_log2 = scale * 1.4426950408889634f;
    a.error_flag = error_flag;
    return head_dim == 64 ? c4::launch_runs<64>(a, tiles, stream) : c4::launch_runs<128>(a, tiles, stream);
}
