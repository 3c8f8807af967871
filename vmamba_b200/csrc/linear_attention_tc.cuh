// Long bf16 sequences of the linear attention on the 5th-generation tensor cores, no chunk waiting for the one in front of it: what each chunk adds to the state
// (la_gather), the states in front of the chunks by one pass over them (la_spread), and the outputs (la_outputs).  The walk of linear_attention.cu moves fewer bytes (q, k, v
// once, no state), but its chunks follow one another through barriers and some 10 instructions for each matrix instruction; here the CUDA cores do no more than
// weight the keys, decay the pairs and add up.  16 385 tokens of 16 heads of 128 x 128: la_gather 61 us (DRAM 43 % of its rate), la_spread 38 (57 %), la_outputs 65 (58 %), the walk
// 306 in all; 41 for the bytes of q, k, v and outputs alone.  What is left is the latency of each CTA's own chain, loads, weights, products, stores, with two CTAs an SM.
//
// A tile of tokens comes by TMA as rows of 64 elements with the 128-byte swizzle.  Contractions over tokens read it as an MN-major operand, those over dk as a
// K-major one, so that nothing is transposed.  dk fills 64 or 128 rows, dv 64 or 128 columns; what is missing is read as zeros.
#pragma once
#include "tc05.cuh"

namespace ss2d {

namespace {

namespace lat {

using namespace tc05;

constexpr int kThreads = 256;

// (batch, head, token, element) rows in memory
inline bool make_rows_map(CUtensorMap* m, const Rows& r, long long B, long long H, long long L, long long D, int tokens) {     // a box: 64 elements of `tokens` rows
    EncodeFn enc = encode_fn();
    if (!enc) return false;
    auto stride = [](long long s) { return (cuuint64_t)(s > 0 ? s * 2 : 16); };       // of one element any will do
    const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)L, (cuuint64_t)H, (cuuint64_t)B};
    const cuuint64_t strides[3] = {stride(r.l), stride(r.h), stride(r.b)};
    const cuuint32_t box[4] = {64, (cuuint32_t)tokens, 1, 1}, one[4] = {1, 1, 1, 1};
    return enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(r.p), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// (state, dk, dv) planes of states, `bytes_apart`
inline bool make_states_map(CUtensorMap* m, const void* p, long long n, long long bytes_apart, long long dk, long long ld, int rows) {
    EncodeFn enc = encode_fn();
    if (!enc) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)ld, (cuuint64_t)dk, (cuuint64_t)n}, strides[2] = {(cuuint64_t)ld * 2, (cuuint64_t)bytes_apart};
    const cuuint32_t box[3] = {64, (cuuint32_t)rows, 1}, one[3] = {1, 1, 1};
    return enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(p), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// (state, dk, ld) fp32, a box: 32 x 32
inline bool make_added_map(CUtensorMap* m, const void* p, long long n, long long dk, long long ld) {
    EncodeFn enc = encode_fn();
    if (!enc) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)ld, (cuuint64_t)dk, (cuuint64_t)n}, strides[2] = {(cuuint64_t)ld * 4, (cuuint64_t)(dk * ld * 4)};
    const cuuint32_t box[3] = {32, 32, 1}, one[3] = {1, 1, 1};
    return enc(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, const_cast<void*>(p), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
__device__ __forceinline__ void store_boxes_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void store_boxes_done() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, const void* src, int x, int y, int z) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];\n cp.async.bulk.commit_group;"
                 ::"l"(map), "r"(smem_u32(src)), "r"(x), "r"(y), "r"(z) : "memory");
}
__device__ __forceinline__ void tma_store_4d(const CUtensorMap* map, const void* src, int x, int y, int z, int w) {
    asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5}], [%1];\n cp.async.bulk.commit_group;"
                 ::"l"(map), "r"(smem_u32(src)), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                 ::"r"(smem_u32(dst)), "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z) : "memory");
}
__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, int x, int y, int z, int w, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
                 ::"r"(smem_u32(dst)), "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

// Cumulative sums of kTokens log decays by one warp, kTokens / 32 in a row for each lane; f(token, sum, sum of all)
template <int kTokens, typename F> __device__ __forceinline__ Cum each_decay(const float* g, long long stride, int first, int L, int lane, F&& f) {
    constexpr int N = kTokens / 32;
    Cum c[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int t = first + N * lane + i;
        c[i] = cum_of(t < L ? g[(long long)t * stride] : 0.f);
        if (i) c[i] = cum_add(c[i - 1], c[i]);
    }
    Cum s = c[N - 1];
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const Cum o = {__shfl_up_sync(0xffffffffu, s.n, off), __shfl_up_sync(0xffffffffu, s.f, off)};
        if (lane >= off) s = cum_add(o, s);
    }
    Cum before = {__shfl_up_sync(0xffffffffu, s.n, 1), __shfl_up_sync(0xffffffffu, s.f, 1)};
    if (lane == 0) before = {0.f, 0.f};
    const Cum all = {__shfl_sync(0xffffffffu, s.n, 31), __shfl_sync(0xffffffffu, s.f, 31)};
#pragma unroll
    for (int i = 0; i < N; ++i) f(N * lane + i, cum_add(before, c[i]), all);
    return all;
}

// ---- what a chunk adds to the state -------------------------------------------------------------------------------------
struct GatherArgs {
    const float* g;
    long long g_b, g_l, g_h;
    float* decay;               // (B, H, chunks): log2 of the decay over the chunk
    int H, rep, L, dk, dv, chunks;
    float scale;                // backwards
    int* error_flag;
};
template <int DK, int DV, int kTokens> struct GatherSmem {
    static constexpr int kBlock = kTokens * 128;                        // 64 columns
    static constexpr int kK = 0, kLow = kK + DK / 64 * kBlock, kNone = kLow + DK / 64 * kBlock, kV = kNone + (DK == 64 ? kBlock : 0);
    static constexpr int kEnd = kV + DV / 64 * kBlock, kTx = (DK + DV) / 64 * kBlock;
    static constexpr size_t kBytes = kEnd + kTokens * 4 + 64 + 1024;
};

// Weighted keys as three bf16 pieces, the first in place of the keys, the last in the place where the second follows it; a product of 128 x DV over the chunk's tokens for each.
// With two, 2^-17 off each, states are 2.4e-6 from 64 bits (2-norm); so they are 1e-7 to 3e-7, as with elementary fp32 operations, for 5 % of a forward call: 16 385 tokens of 16 heads of
// 128 x 128 158 -> 166 us, 2 x 4 096 82 -> 86 (training 453 -> 459); the walk, 16 x 3 136 of 12 heads of 64 x 32, 123 -> 133 (494 -> 516).
template <int DK, int DV, int kTokens, bool kBack>
__global__ void __launch_bounds__(kThreads) la_gather_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                                                             const __grid_constant__ CUtensorMap tmO, const GatherArgs a) {
    follow_previous();
    using M = GatherSmem<DK, DV, kTokens>;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* const sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    float* const w = reinterpret_cast<float*>(sm + M::kEnd);
    uint64_t* const loaded = reinterpret_cast<uint64_t*>(w + kTokens);
    uint64_t* const done = loaded + 1;
    uint32_t* const slot = reinterpret_cast<uint32_t*>(done + 1);
    volatile int* const abort_flag = reinterpret_cast<volatile int*>(slot + 1);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int c = blockIdx.x % a.chunks, bh = blockIdx.x / a.chunks, b = bh / a.H, h = bh % a.H, first = c * kTokens;
    if (tid == 0) {
        mbar_init(loaded, 1);
        mbar_init(done, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        mbar_expect_tx(loaded, M::kTx);
#pragma unroll
        for (int i = 0; i < DK / 64; ++i) tma_load_4d(sm + M::kK + i * M::kBlock, &tmK, 64 * i, first, h / a.rep, b, loaded);
#pragma unroll
        for (int i = 0; i < DV / 64; ++i) tma_load_4d(sm + M::kV + i * M::kBlock, &tmV, 64 * i, first, h, b, loaded);
    }
    if (warp == 1) { tmem_alloc(slot, DV); tmem_relinquish(); }
    if (warp == 2) {
        const Cum all = each_decay<kTokens>(a.g + b * a.g_b + h * a.g_h, a.g_l, first, a.L, lane, [&](int t, Cum s, Cum end) {
            w[t] = kBack ? a.scale * ex2_approx(s.n + s.f) : exp_diff(end, s);
        });
        if (lane == 0) a.decay[blockIdx.x] = all.n + all.f;
    }
    if constexpr (DK == 64)
        for (int i = tid; i < M::kBlock / 16; i += kThreads) reinterpret_cast<uint4*>(sm + M::kNone)[i] = make_uint4(0, 0, 0, 0);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *slot;
    bool ok = mbar_wait_prompt(loaded, 0, abort_flag);
    int commits = 0;                                                    // of the thread that issues them
    constexpr int kUnits = DK / 64 * M::kBlock / 16 / kThreads;         // 8 elements each, of a thread
    uint4 second[kUnits];
    if (ok) {
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
            const int i = tid + u * kThreads;
            uint4* const at = reinterpret_cast<uint4*>(sm + M::kK) + i;
            const float s = w[i / 8 % kTokens];
            const uint4 x = *at;
            uint32_t in[4] = {x.x, x.y, x.z, x.w}, p[3][4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float2 f = __fmul2_rn(Half2Of<__nv_bfloat16>::unpack(in[j]), splat2(s));
#pragma unroll
                for (int k = 0; k < 3; ++k) {
                    p[k][j] = Half2Of<__nv_bfloat16>::pack(f.x, f.y);
                    const float2 r = Half2Of<__nv_bfloat16>::unpack(p[k][j]);
                    f.x -= r.x; f.y -= r.y;
                }
            }
            *at = make_uint4(p[0][0], p[0][1], p[0][2], p[0][3]);
            second[u] = make_uint4(p[1][0], p[1][1], p[1][2], p[1][3]);
            *reinterpret_cast<uint4*>(sm + M::kLow + 16 * i) = make_uint4(p[2][0], p[2][1], p[2][2], p[2][3]);
        }
    }
    constexpr uint32_t idesc = instr_desc(1, true, 128, DV) | (1u << 16);
    const uint32_t base = smem_u32(sm);
    const uint64_t high = smem_desc(base + M::kK, DK == 64 ? M::kNone - M::kK : M::kBlock, 1024, kSw128);
    const uint64_t low = smem_desc(base + M::kLow, DK == 64 ? M::kNone - M::kLow : M::kBlock, 1024, kSw128);
    const uint64_t v = smem_desc(base + M::kV, M::kBlock, 1024, kSw128);
    fence_async_smem();
    __syncthreads();
    if (tid == 0 && ok) {
#pragma unroll
        for (int k = 0; k < kTokens / 16; ++k) tc_mma(tmem, low + k * 128, v + k * 128, idesc, k > 0);
        tc_commit(done);
        commits = 1;
    }
    ok = ok && mbar_wait_prompt(done, 0, abort_flag);
    __syncwarp();
    if (ok) {
#pragma unroll
        for (int u = 0; u < kUnits; ++u) *reinterpret_cast<uint4*>(sm + M::kLow + 16 * (tid + u * kThreads)) = second[u];
    }
    fence_async_smem();
    __syncthreads();
    if (tid == 0 && ok) {
#pragma unroll
        for (int k = 0; k < kTokens / 16; ++k) tc_mma(tmem, low + k * 128, v + k * 128, idesc, 1);
#pragma unroll
        for (int k = 0; k < kTokens / 16; ++k) tc_mma(tmem, high + k * 128, v + k * 128, idesc, 1);
        tc_commit(done);
        commits = 2;
    }
    ok = ok && mbar_wait_prompt(done, 1, abort_flag);
    __syncwarp();
    tc_fence_after();
    if (ok) {
        // 32 rows and 32 columns at a time through shared memory, in place of the operands, which have been read
        static_assert(M::kEnd >= 8 * 4096);
        unsigned char* const stage = sm + warp * 4096;
        const int row = 32 * (warp & 3), ld = state_row(a.dv);
#pragma unroll
        for (int q = 0; q < DV / 2; q += 32) {
            const int col = (warp >> 2) * (DV / 2) + q;
            if (row >= a.dk || col >= ld) break;
            uint32_t r[2][16];
            tmem_ld16(tmem + ((uint32_t)row << 16) + col, r[0]);
            tmem_ld16(tmem + ((uint32_t)row << 16) + col + 16, r[1]);
            tmem_ld_wait();
            if (q && lane == 0) store_boxes_read();
            __syncwarp();
#pragma unroll
            for (int u = 0; u < 8; ++u)
                *reinterpret_cast<uint4*>(stage + lane * 128 + ((u ^ (lane & 7)) << 4)) =
                    make_uint4(r[u / 4][4 * (u & 3)], r[u / 4][4 * (u & 3) + 1], r[u / 4][4 * (u & 3) + 2], r[u / 4][4 * (u & 3) + 3]);
            fence_async_smem();
            __syncwarp();
            if (lane == 0) tma_store_3d(&tmO, stage, col, row, blockIdx.x);
            __syncwarp();
        }
        if (lane == 0) store_boxes_done();
        __syncwarp();
    }
    if (tid == 0 && !ok) {
        mbar_drain(loaded, 0);
        if (commits) mbar_drain(done, commits - 1);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) { tc_fence_after(); tmem_dealloc(tmem, DV); }
    if (tid == 0 && *abort_flag) atomicExch(a.error_flag, 1);
}

// ---- states in front of the chunks --------------------------------------------------------------------------------------
struct SpreadArgs {
    const float *added, *decay; // (B, H, chunks, dk, ld), (B, H, chunks)
    const float* first;         // (B, H, dk, dv) or NULL
    float* last;                // the same, or NULL
    float* states;              // (B, H, chunks, dk, ld) or NULL: for the gradients
    __nv_bfloat16* plane;       // the same rounded, or NULL: for the outputs
    int chunks, dk, dv, ld;
    bool back;
};
// Four neighbouring elements a thread, eight chunks read ahead (sixteen: 47 us in place of 39 at 129 chunks of 16 heads of 128 x 128; two groups of four in turn: 65)
__global__ void __launch_bounds__(128) la_spread_kernel(const SpreadArgs a) {
    follow_previous();
    const int size = a.dk * a.ld, per = (size / 4 + 127) / 128, bh = blockIdx.x / per, e = 4 * (blockIdx.x % per * 128 + threadIdx.x);
    if (e >= size) return;
    const int row = e / a.ld, col = e % a.ld;
    const long long own = ((long long)bh * a.dk + row) * a.dv + col;
    float s[4] = {};
    if (a.first)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] = col + i < a.dv ? a.first[own + i] : 0.f;
    auto at = [&](int i) { return (long long)bh * a.chunks + (a.back ? a.chunks - 1 - i : i); };
    constexpr int kAhead = 8;
    for (int i0 = 0; i0 < a.chunks; i0 += kAhead) {
        float4 x[kAhead];
        float d[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
            if (i0 + i < a.chunks) {
                x[i] = *reinterpret_cast<const float4*>(a.added + at(i0 + i) * size + e);
                d[i] = a.decay[at(i0 + i)];
            }
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
            if (i0 + i < a.chunks) {
                if (a.states) *reinterpret_cast<float4*>(a.states + at(i0 + i) * size + e) = make_float4(s[0], s[1], s[2], s[3]);
                if (a.plane)
                    *reinterpret_cast<uint2*>(a.plane + at(i0 + i) * size + e) = make_uint2(Half2Of<__nv_bfloat16>::pack(s[0], s[1]), Half2Of<__nv_bfloat16>::pack(s[2], s[3]));
                const float k = ex2_approx(d[i]);
                s[0] = fmaf(k, s[0], x[i].x); s[1] = fmaf(k, s[1], x[i].y); s[2] = fmaf(k, s[2], x[i].z); s[3] = fmaf(k, s[3], x[i].w);
            }
    }
    if (a.last)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (col + i < a.dv) a.last[own + i] = s[i];
}

// ---- outputs ------------------------------------------------------------------------------------------------------------
constexpr int kTile = 128;
struct OutArgs {
    const float* g;
    long long g_b, g_l, g_h;
    int H, rep, L, dk, dv, tiles;
    int states, step;           // of a (batch, head): states in memory, and how many lie between those of two tiles
    float scale;
    int* error_flag;
};
// Two roundings to bf16 in front of the outputs' own: the pairs' weights and the state that the queries meet, one piece each.  Outputs are 1.4 times as far from 64 bits as one
// rounding (2.4e-3 for 1.7e-3, 2-norm); a second piece of both would double the products and bring 40 KB more into a CTA for what the outputs' own rounding hides.
// The pairs take the place of the keys, v that of the queries, once these have been read; with both sides of 64 v has its own place, the products with the state wait
// for the pairs to have left TMEM and take half their columns: 96 to 128 KB and 256 columns become 96 KB and 256, or 72 KB and 128, and two or three CTAs share an SM.
template <int DK, int DV> struct OutSmem {
    static constexpr bool kSmall = DK == 64 && DV == 64;
    static constexpr int kBlock = kTile * 128;
    static constexpr int kQ = 0, kV = kSmall ? kBlock : 0, kP = kV + (DV > DK ? DV : DK) / 64 * kBlock, kK = kP, kS = kP + 2 * kBlock;
    static constexpr int kEnd = kS + DV / 64 * DK * 128;
    static constexpr int kFloats = 4 * kTile + 4 * kTile;               // n, f, e, near; far of four blocks of 32 tokens
    static constexpr size_t kBytes = kEnd + kFloats * 4 + 64 + 1024;
    static constexpr int kTmem = kSmall ? 128 : 256, kAcross = kSmall ? 64 : 128;   // pairs, and in their place their products with v; products with the state
};

template <int DK, int DV>
__global__ void __launch_bounds__(kThreads, DK == 64 && DV == 64 ? 3 : 2) la_outputs_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                                                              const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmS,
                                                              const __grid_constant__ CUtensorMap tmO, const OutArgs a) {
    follow_previous();
    using M = OutSmem<DK, DV>;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* const sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    float *const dn = reinterpret_cast<float*>(sm + M::kEnd), *const df = dn + kTile, *const de = df + kTile, *const near = de + kTile, *const far = near + kTile;
    uint64_t* const bars = reinterpret_cast<uint64_t*>(far + 4 * kTile);            // q and k, states, first products, last ones, v
    uint32_t* const slot = reinterpret_cast<uint32_t*>(bars + 5);
    volatile int* const abort_flag = reinterpret_cast<volatile int*>(slot + 1);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int c = blockIdx.x % a.tiles, bh = blockIdx.x / a.tiles, b = bh / a.H, h = bh % a.H, first = c * kTile;
    if (tid == 0) {
        for (int i = 0; i < 5; ++i) mbar_init(bars + i, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        mbar_expect_tx(bars, 2 * DK / 64 * M::kBlock);
#pragma unroll
        for (int i = 0; i < DK / 64; ++i) {
            tma_load_4d(sm + M::kQ + i * M::kBlock, &tmQ, 64 * i, first, h / a.rep, b, bars);
            tma_load_4d(sm + M::kK + i * M::kBlock, &tmK, 64 * i, first, h / a.rep, b, bars);
        }
        mbar_expect_tx(bars + 1, DV / 64 * (DK * 128));
#pragma unroll
        for (int i = 0; i < DV / 64; ++i) tma_load_3d(sm + M::kS + i * DK * 128, &tmS, 64 * i, 0, bh * a.states + c * a.step, bars + 1);
        if constexpr (M::kSmall) {
            mbar_expect_tx(bars + 4, M::kBlock);
            tma_load_4d(sm + M::kV, &tmV, 0, first, h, b, bars + 4);
        }
    }
    if (warp == 1) { tmem_alloc(slot, M::kTmem); tmem_relinquish(); }
    if (warp == 2)
        each_decay<kTile>(a.g + b * a.g_b + h * a.g_h, a.g_l, first, a.L, lane, [&](int t, Cum s, Cum) { dn[t] = s.n; df[t] = s.f; de[t] = ex2_approx(s.n + s.f); });
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *slot;
    const uint32_t base = smem_u32(sm);
    bool ok = true;
    bool pending[5] = {true, true, false, false, M::kSmall};                        // barriers that something is on its way to (of the thread that sends it)
    auto with_states = [&] {                                                        // queries times the state in front
        constexpr uint32_t idesc = instr_desc(1, false, 128, DV) | (1u << 16);
        const uint64_t q = smem_desc(base + M::kQ, 16, 1024, kSw128), s = smem_desc(base + M::kS, DK * 128, 1024, kSw128);
        if (!mbar_wait_prompt(bars + 1, 0, abort_flag)) return false;
        tc_fence_after();
#pragma unroll
        for (int i = 0; i < DK / 16; ++i)
            tc_mma(tmem + M::kAcross, q + ((uint64_t)(i / 4 * M::kBlock + i % 4 * 32) >> 4), s + i * 128, idesc, i > 0);
        return true;
    };
    if (tid == 0) {
        constexpr uint32_t idesc = instr_desc(1, false, 128, 128);
        const uint64_t q = smem_desc(base + M::kQ, 16, 1024, kSw128), k = smem_desc(base + M::kK, 16, 1024, kSw128);
        ok = mbar_wait_prompt(bars, 0, abort_flag);
        if (ok) {
            tc_fence_after();
#pragma unroll
            for (int i = 0; i < DK / 16; ++i) {
                const uint64_t off = (uint64_t)(i / 4 * M::kBlock + i % 4 * 32) >> 4;
                tc_mma(tmem, q + off, k + off, idesc, i > 0);
            }
            if constexpr (!M::kSmall) ok = with_states();
            if (ok) { tc_commit(bars + 2); pending[2] = true; }
        }
    }
    // pairs of different blocks of 32 tokens: one exponential a token (as in the walk)
    for (int i = tid; i < 5 * kTile; i += kThreads) {
        const int blk = i / kTile, t = i % kTile;
        const Cum own = {dn[t], df[t]}, start = {dn[blk < 4 ? 32 * blk : t / 32 * 32], df[blk < 4 ? 32 * blk : t / 32 * 32]};
        if (blk < 4) far[i] = t < 32 * blk ? exp_diff(start, own) : 0.f;
        else near[t] = exp_diff(own, start);
    }
    __syncthreads();
    ok = ok && mbar_wait_prompt(bars + 2, 0, abort_flag);
    if constexpr (!M::kSmall)
        if (tid == 0 && ok) {                                                       // the queries have been read
            mbar_expect_tx(bars + 4, DV / 64 * M::kBlock);
#pragma unroll
            for (int i = 0; i < DV / 64; ++i) tma_load_4d(sm + M::kV + i * M::kBlock, &tmV, 64 * i, first, h, b, bars + 4);
            pending[4] = true;
        }
    __syncwarp();
    tc_fence_after();
    const int quarter = warp & 3, row = 32 * quarter + lane;
    const uint32_t lane_base = tmem + ((uint32_t)(32 * quarter) << 16);
    if (ok) {
        const Cum own = {dn[row], df[row]};
        const float nr = near[row];
#pragma unroll 1
        for (int q = 0; q < 64; q += 16) {
            const int col = 64 * (warp >> 2) + q;
            uint32_t r[16], p[8];
            if (col < 32 * quarter + 32) {                  // (by warp: the loads take all of it)
                tmem_ld16(lane_base + col, r);
                tmem_ld_wait();
                if (col < 32 * quarter) {
                    const float* const f = far + quarter * kTile + col;
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        p[j] = Half2Of<__nv_bfloat16>::pack(__uint_as_float(r[2 * j]) * (nr * f[2 * j]), __uint_as_float(r[2 * j + 1]) * (nr * f[2 * j + 1]));
                } else {
                    float x[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j) x[j] = col + j <= row ? __uint_as_float(r[j]) * exp_diff(own, Cum{dn[col + j], df[col + j]}) : 0.f;
#pragma unroll
                    for (int j = 0; j < 8; ++j) p[j] = Half2Of<__nv_bfloat16>::pack(x[2 * j], x[2 * j + 1]);
                }
            } else
#pragma unroll
                for (int j = 0; j < 8; ++j) p[j] = 0;
            unsigned char* const to = sm + M::kP + (warp >> 2) * M::kBlock + row * 128;
#pragma unroll
            for (int u = 0; u < 2; ++u)
                *reinterpret_cast<uint4*>(to + (((q / 8 + u) ^ (row & 7)) << 4)) = make_uint4(p[4 * u], p[4 * u + 1], p[4 * u + 2], p[4 * u + 3]);
        }
    }
    fence_async_smem();
    tc_fence_before();
    __syncthreads();
    if (tid == 0 && ok) {
        tc_fence_after();
        constexpr uint32_t idesc = instr_desc(1, false, 128, DV) | (1u << 16);
        const uint64_t p = smem_desc(base + M::kP, 16, 1024, kSw128), v = smem_desc(base + M::kV, M::kBlock, 1024, kSw128);
        if constexpr (M::kSmall) ok = with_states();
        ok = ok && mbar_wait_prompt(bars + 4, 0, abort_flag);
        if (ok) {
            tc_fence_after();
#pragma unroll
            for (int i = 0; i < kTile / 16; ++i) tc_mma(tmem, p + ((uint64_t)(i / 4 * M::kBlock + i % 4 * 32) >> 4), v + i * 128, idesc, i > 0);
            tc_commit(bars + 3);
            pending[3] = true;
        }
    }
    ok = ok && mbar_wait_prompt(bars + 3, 0, abort_flag);
    __syncwarp();
    tc_fence_after();
    if (ok) {
        // 32 tokens and 64 columns at a time through shared memory, where the pairs were
        const float e = a.scale * de[row];
        const int half = warp >> 2;
        unsigned char* const stage = sm + M::kP + (DV == 128 ? warp : quarter) * 4096;
#pragma unroll
        for (int q = 0; q < DV / 2; q += 16) {
            const int col = half * (DV / 2) + q;
            uint32_t x[16], y[16], w[8];
            tmem_ld16(lane_base + col, x);
            tmem_ld16(lane_base + M::kAcross + col, y);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 8; ++j)
                w[j] = Half2Of<__nv_bfloat16>::pack(fmaf(e, __uint_as_float(y[2 * j]), a.scale * __uint_as_float(x[2 * j])),
                                                    fmaf(e, __uint_as_float(y[2 * j + 1]), a.scale * __uint_as_float(x[2 * j + 1])));
            const int at = DV == 128 ? q : col;
#pragma unroll
            for (int u = 0; u < 2; ++u)
                *reinterpret_cast<uint4*>(stage + lane * 128 + (((at / 8 + u) ^ (lane & 7)) << 4)) = make_uint4(w[4 * u], w[4 * u + 1], w[4 * u + 2], w[4 * u + 3]);
        }
        fence_async_smem();
    }
    if constexpr (DV == 64) __syncthreads();                                // two warps have filled a block of 64 columns
    else __syncwarp();
    if (ok && lane == 0 && (DV == 128 || warp < 4)) {
        const int x = DV == 128 ? (warp >> 2) * 64 : 0, y = first + 32 * quarter;
        if (x < a.dv && y < a.L) tma_store_4d(&tmO, sm + M::kP + warp * 4096, x, y, h, b);
        store_boxes_done();
    }
    if (tid == 0 && !ok) {
#pragma unroll
        for (int i = 0; i < 5; ++i)
            if (pending[i]) mbar_drain(bars + i, 0);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) { tc_fence_after(); tmem_dealloc(tmem, M::kTmem); }
    if (tid == 0 && *abort_flag) atomicExch(a.error_flag, 1);
}

// ---- host ---------------------------------------------------------------------------------------------------------------
inline int* device_flag() {
    int* host = error_flag_for_current_device();
    int* dev = nullptr;
    if (!host || *host || cudaHostGetDevicePointer((void**)&dev, host, 0) != cudaSuccess) return nullptr;      // (or an earlier launch gave up on a wait)
    return dev;
}
template <int DK, int DV, int kTokens, bool kBack> int gather(const Rows& k, const Rows& v, float* added, long long B, long long G, GatherArgs a, cudaStream_t st) {
    a.error_flag = device_flag();
    if (!a.error_flag) return SS2D_ECUDA;
    CUtensorMap tk, tv, to;
    if (!make_rows_map(&tk, k, B, G, a.L, a.dk, kTokens) || !make_rows_map(&tv, v, B, a.H, a.L, a.dv, kTokens) ||
        !make_added_map(&to, added, B * a.H * a.chunks, a.dk, state_row(a.dv)))
        return SS2D_ECUDA;
    auto kern = la_gather_kernel<DK, DV, kTokens, kBack>;
    constexpr size_t smem = GatherSmem<DK, DV, kTokens>::kBytes;
    if (const int rc = allow_dynamic_smem(kern, smem)) return rc;
    launch(kern, (unsigned)(B * a.H * a.chunks), kThreads, smem, st, tk, tv, to, a);
    count_launch();
    return check_launch();
}
inline int spread(const SpreadArgs& a, long long bh, cudaStream_t st) {
    launch(la_spread_kernel, (unsigned)(bh * ((a.dk * a.ld / 4 + 127) / 128)), 128, 0, st, a);
    count_launch();
    return check_launch();
}
template <int DK, int DV> int outputs(const Rows& q, const Rows& k, const Rows& v, const Rows& o, const void* states, long long bytes_apart, long long B, long long G, OutArgs a, cudaStream_t st) {
    a.error_flag = device_flag();
    if (!a.error_flag) return SS2D_ECUDA;
    CUtensorMap tq, tk, tv, ts, to;
    if (!make_rows_map(&tq, q, B, G, a.L, a.dk, kTile) || !make_rows_map(&tk, k, B, G, a.L, a.dk, kTile) || !make_rows_map(&tv, v, B, a.H, a.L, a.dv, kTile) ||
        !make_rows_map(&to, o, B, a.H, a.L, a.dv, 32) || !make_states_map(&ts, states, B * a.H * a.states, bytes_apart, a.dk, state_row(a.dv), DK))
        return SS2D_ECUDA;
    auto kern = la_outputs_kernel<DK, DV>;
    constexpr size_t smem = OutSmem<DK, DV>::kBytes;
    if (const int rc = allow_dynamic_smem(kern, smem)) return rc;
    launch(kern, (unsigned)(B * a.H * a.tiles), kThreads, smem, st, tq, tk, tv, ts, to, a);
    count_launch();
    return check_launch();
}

}  // namespace lat

}  // namespace

}  // namespace ss2d
