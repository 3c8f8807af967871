// Products of the gated feed-forward block on the 5th-generation tensor cores, 16-bit types: C (M x N) = A (M x K) . B (N x K)^T with the block's
// epilogues on the accumulators.
//
// One persistent CTA per SM walks tiles of 128 rows.  Warp 0 brings 64 contraction elements of both operands at a time by TMA into a ring of stages, warp 1
// issues the MMAs, two groups of four warps take the accumulators of alternate tiles (TMEM holds two tiles) and write results through shared memory by TMA,
// 32 rows of 128 bytes a warp: with stores from registers, a row a lane, the load/store unit takes as long as the tile's MMAs.
// An operand is read as it lies in memory: rows of the contraction index ("MN-major") or rows of M / N ("K-major"), so that no weight and no map is
// transposed for any of the backward products.  Edges: TMA reads zeros and drops what it would write outside.
//
// Value and gate of a column come as two blocks of rows of the same operand, side by side in TMEM (EPI_GATE).  EPI_GRAD goes through two
// contractions for a tile, x . w1 for value and gate and dy . w2 for the gradient of the hidden map, and forms the gradients of value and gate from the
// three: they are computed again instead of kept, 4 more operations per weight and token in place of 16 bytes written and read per hidden element.
//
// What bounds them is the way of the operands into an SM, some 50 bytes a cycle however few of them read: a tile of 128 x 128 needs 32 KB for a step (64 of the
// contraction) that takes the tensor core 256 cycles, and gets them in 650.  Pairs of CTAs (kPair) share a tile of 256 rows, each with its own half of A's rows and of
// B's: 32 KB for 128 x 256 results, in place of 48.
//
// Rates (bf16, both launches of the forward call, GELU and biases; library products of these sizes, which leave both out, in brackets): 8 192 tokens, 1 024 channels, 4 096 hidden, a
// call at a time 155 us (148), 200 in a row 163 (171), 1 270 TFLOP/s, 0.91 of the measured sustained rate; 12 544, 512, 2 048 in a row 81 (82), 970 TFLOP/s; kernels alone 51 and 29, tensor
// pipe 54 and 58 % active, DRAM 4 and 20 %, the second one 98 tiles on 74 pairs of CTAs, two rounds for 1.3.
//
// Every wait is bounded; one that runs out raises the device's error flag (tc05.cuh), all roles leave and the TMEM is freed.
#pragma once
#include "gated_epilogue.cuh"
#include "tc05.cuh"

namespace ss2d {
namespace ptc {

using namespace tc05;

constexpr int kRows = 128, kDepth = 64;                 // tile rows; contraction elements of a stage
constexpr int kFirstEpi = 4, kEpiWarps = 8, kThreads = 32 * (kFirstEpi + kEpiWarps);

struct Args {
    int m_tiles, n_tiles, splits;
    int blocks, per_split;          // stages of the first contraction; of a split
    int blocks2;                    // EPI_GRAD: of the second one
    int M, N, second;               // second: rows of B between value and gate
    const void* bias;
    int* error_flag;
};

// kCols: TMEM columns of a tile.  EPI_GATE: half value, half gate; EPI_GRAD: a third each of value, gate and hidden gradient.
template <int EPI, int kCols, bool kPair> struct Shape {
    static constexpr int kOut = EPI == EPI_GATE ? kCols / 2 : EPI == EPI_GRAD ? kCols / 3 : kCols;       // columns of the result
    static constexpr int kB = EPI == EPI_GRAD ? 2 * kOut : kCols;                                        // rows of B of the (first) contraction
    static constexpr int kShare = kPair ? 2 : 1;                                                         // CTAs among which they are divided
    static constexpr int kABytes = kRows * kDepth * 2, kStage = kABytes + kB / kShare * kDepth * 2;
    // tiles in TMEM; of EPI_GRAD one tile's value and gate, and two tiles' hidden gradient, which the MMAs fill while the epilogue still reads the other two
    static constexpr int kBufs = kCols <= 256 ? 2 : 1;
    static constexpr int kOuts = EPI == EPI_GRAD ? 2 : 1;                                                // blocks of 32 rows that a warp stores at once
    static constexpr int kHalves = kOuts == 1 && kOut >= 128 ? 2 : 1;                                    // one is filled while the other is read
    static constexpr int kWarpStaging = kOuts * kHalves * 4096, kStaging = kEpiWarps * kWarpStaging;
    static constexpr int kBiasFloats = EPI == EPI_PART ? 0 : EPI == EPI_OUT ? kOut : kBufs == 2 ? 2 * kOut : kOut;      // of a group of epilogue warps
    static constexpr int kBias = 2 * 2 * kBiasFloats * 4;
    static constexpr int kRoom = 232448 - 1024 - 256 - kStaging - kBias, kStages = kRoom / kStage > 8 ? 8 : kRoom / kStage;
    static constexpr int kTmem = kCols > 128 ? 512 : kCols > 64 ? 256 : 128;                             // a power of two
    static constexpr int kPitch = kTmem / kBufs;
    static constexpr int kBars = kStages * kStage + kStaging, kBiasAt = kBars + 256;
    static constexpr size_t kBytes = kBiasAt + kBias + 1024;
    static_assert((EPI == EPI_GRAD) == (kBufs == 1) && (EPI != EPI_GRAD || kCols + kOut <= kTmem));
    static_assert(kCols <= kPitch && kOut % 64 == 0 && kStages >= 3 && (kB / kShare) % 64 == 0);
    static_assert(kBufs == 2 || kOut == 128, "with one tile in TMEM the two groups of epilogue warps have 64 columns each");
};

__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, const void* src, int x, int y, int z) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(map), "r"(smem_u32(src)), "r"(x), "r"(y), "r"(z) : "memory");
}
__device__ __forceinline__ void store_done() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

template <typename T, bool kAMN, bool kBMN, int EPI, int ACT, int kCols, bool kPair>
__global__ void __launch_bounds__(kThreads, 1)
product_tc05_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmA2,
                    const __grid_constant__ CUtensorMap tmB2, const __grid_constant__ CUtensorMap tmO, const __grid_constant__ CUtensorMap tmO2, const Args a) {
    follow_previous();
    using S = Shape<EPI, kCols, kPair>;
    constexpr int NS = S::kStages, NB = S::kBufs;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* const sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint64_t* const bars = reinterpret_cast<uint64_t*>(sm + S::kBars);
    uint64_t *const full = bars, *const empty = bars + NS, *const acc_full = bars + 2 * NS, *const acc_empty = acc_full + 2;
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
    volatile int* const abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = kPair ? (int)cluster_rank() : 0;
    if (threadIdx.x == 0) {
        for (int i = 0; i < NS; ++i) { mbar_init(full + i, 1); mbar_init(empty + i, 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(acc_full + i, 1); mbar_init(acc_empty + i, (NB == 2 ? 4 : 8) * S::kShare); }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        if constexpr (kPair) tmem_alloc_pair(tmem_slot, S::kTmem);
        else { tmem_alloc(tmem_slot, S::kTmem); tmem_relinquish(); }
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (kPair) cluster_sync();                 // the other CTA's barriers and TMEM are there
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const int tiles = a.m_tiles * a.n_tiles * a.splits, walker = blockIdx.x / S::kShare, walkers = gridDim.x / S::kShare;
    struct Tile { int m0, n0, split, k0, k1; };
    auto tile_at = [&](int i) {
        Tile t;
        t.n0 = i % a.n_tiles * S::kOut;
        t.m0 = (i / a.n_tiles % a.m_tiles * S::kShare + rank) * kRows;
        t.split = i / (a.n_tiles * a.m_tiles);
        t.k0 = t.split * a.per_split;
        t.k1 = min(a.blocks, t.k0 + a.per_split);
        return t;
    };

    if (warp == 0) {
        // ---------------------------------------------------------------- TMA producer
        if (lane == 0) {
            int s = 0, round = 0;
            bool ok = true;
            // the first CTA's barrier counts the bytes of both
            auto slot = [&](uint32_t bytes) -> unsigned char* {
                if (round > 0 && !mbar_wait_prompt(empty + s, (round - 1) & 1, abort_flag)) { ok = false; return nullptr; }
                if (rank == 0) mbar_expect_tx(full + s, bytes * S::kShare);
                return sm + s * S::kStage;
            };
            auto next = [&] { if (++s == NS) { s = 0; ++round; } };
            auto load = [&](unsigned char* dst, const CUtensorMap* map, int x, int y) {
                if constexpr (kPair) tma_load_2d_pair(dst, map, x, y, in_rank(full + s, 0));
                else tma_load_2d(dst, map, x, y, full + s);
            };
            constexpr int kHalf = S::kB / S::kShare;     // rows of B in this CTA
            for (int i = walker; ok && i < tiles; i += walkers) {
                const Tile t = tile_at(i);
                if constexpr (EPI == EPI_GRAD) {
                    constexpr int kHalf2 = S::kOut / S::kShare;
                    for (int k = 0; ok && k < a.blocks2; ++k) {
                        unsigned char* st = slot(S::kABytes + kHalf2 * 128);
                        if (!ok) break;
                        load(st, &tmA2, k * kDepth, t.m0);
#pragma unroll
                        for (int j = 0; j < kHalf2 / 64; ++j) load(st + S::kABytes + j * 8192, &tmB2, t.n0 + rank * kHalf2 + 64 * j, k * kDepth);
                        next();
                    }
                }
                for (int k = t.k0; k < t.k1; ++k) {
                    unsigned char* st = slot(S::kStage);
                    if (!ok) break;
                    const int k0 = k * kDepth;
                    if constexpr (kAMN) {
                        load(st, &tmA, t.m0, k0);
                        load(st + 8192, &tmA, t.m0 + 64, k0);
                    } else
                        load(st, &tmA, k0, t.m0);
                    unsigned char* b = st + S::kABytes;
                    if constexpr (EPI == EPI_GATE || EPI == EPI_GRAD) {            // value rows, gate rows; of a pair one has those and one these
                        if (rank == 0) load(b, &tmB, k0, t.n0);
                        if (!kPair || rank == 1) load(b + (kPair ? 0 : S::kOut * 128), &tmB, k0, a.second + t.n0);
                    } else if constexpr (kBMN) {
#pragma unroll
                        for (int j = 0; j < kHalf / 64; ++j) load(b + j * 8192, &tmB, t.n0 + rank * kHalf + 64 * j, k0);
                    } else
                        load(b, &tmB, k0, t.n0 + rank * kHalf);
                    next();
                }
            }
            const int last = s, rounds = round;
            // what is in flight has been read, and the other CTA's last arrivals are here, before this one leaves
            for (int j = 0; ok && j < NS; ++j) {
                if (round > 0) ok = mbar_wait_prompt(empty + s, (round - 1) & 1, abort_flag);
                next();
            }
            // or, where this CTA has given up, has arrived (of a pair the first CTA's barriers count both)
            if (!ok && rank == 0)
                for (int j = 0; j < NS; ++j) {
                    const int sent = rounds + (j < last);
                    if (sent > 0) mbar_drain(full + j, (sent - 1) & 1);
                }
        }
    } else if (warp == 1) {
        // ---------------------------------------------------------------- MMA issuer
        if (lane == 0 && rank == 0) {
            constexpr bool kDual = EPI == EPI_GRAD;
            constexpr uint32_t idesc = instr_desc(Fmt<T>::id, kAMN, kRows * S::kShare, S::kB) | ((kBMN && !kDual ? 1u : 0u) << 16);
            constexpr uint32_t idesc2 = instr_desc(Fmt<T>::id, false, kRows * S::kShare, S::kOut) | (1u << 16);
            const uint32_t base = smem_u32(sm);
            const uint64_t da0 = kAMN ? smem_desc(base, 8192, 1024, kSw128) : smem_desc(base, 16, 1024, kSw128);
            const uint64_t db0 = kBMN && !kDual ? smem_desc(base + S::kABytes, 8192, 1024, kSw128) : smem_desc(base + S::kABytes, 16, 1024, kSw128);
            const uint64_t db2 = smem_desc(base + S::kABytes, 8192, 1024, kSw128);
            constexpr uint64_t stepA = (kAMN ? 2048 : 32) >> 4, stepB = (kBMN && !kDual ? 2048 : 32) >> 4;
            auto mma = [&](uint32_t d, uint64_t x, uint64_t y, uint32_t id, uint32_t more) {
                if constexpr (kPair) tc_mma_pair(d, x, y, id, more);
                else tc_mma(d, x, y, id, more);
            };
            auto commit = [&](uint64_t* bar) {
                if constexpr (kPair) tc_commit_pair(bar);
                else tc_commit(bar);
            };
            int s = 0, round = 0, it = 0;
            bool ok = true;
            for (int i = walker; ok && i < tiles; i += walkers, ++it) {
                const Tile t = tile_at(i);
                const int buf = it % NB;
                const uint32_t acc = tmem + buf * S::kPitch;
                if constexpr (kDual)           // (the epilogue of two tiles ago has left this half: the wait below was for it, a tile ago)
                    for (int k = 0; ok && k < a.blocks2; ++k) {
                        if (!mbar_wait_prompt(full + s, round & 1, abort_flag)) { ok = false; break; }
                        tc_fence_after();
                        const uint64_t off = (uint64_t)((uint32_t)(s * S::kStage) >> 4);
#pragma unroll
                        for (int j = 0; j < kDepth / 16; ++j)
                            mma(acc + S::kB + (it & 1) * S::kOut, da0 + off + j * stepA, db2 + off + j * (2048 >> 4), idesc2, k > 0 || j > 0 ? 1u : 0u);
                        commit(empty + s);
                        if (++s == NS) { s = 0; ++round; }
                    }
                if (!ok || (it >= NB && !mbar_wait_prompt(acc_empty + buf, (it / NB - 1) & 1, abort_flag))) break;
                tc_fence_after();
                for (int k = t.k0; k < t.k1; ++k) {
                    if (!mbar_wait_prompt(full + s, round & 1, abort_flag)) { ok = false; break; }
                    tc_fence_after();
                    const uint64_t off = (uint64_t)((uint32_t)(s * S::kStage) >> 4);
#pragma unroll
                    for (int j = 0; j < kDepth / 16; ++j) mma(acc, da0 + off + j * stepA, db0 + off + j * stepB, idesc, k > t.k0 || j > 0 ? 1u : 0u);
                    commit(empty + s);
                    if (++s == NS) { s = 0; ++round; }
                }
                if (ok) commit(acc_full + buf);
            }
        }
    } else if (warp >= kFirstEpi) {
        // ---------------------------------------------------------------- epilogue: group `grp` of four warps has every second tile, or half the columns
        const int grp = (warp - kFirstEpi) >> 2, quarter = warp & 3;
        const uint32_t lane_base = tmem + ((uint32_t)(quarter * 32) << 16) + (NB == 2 ? grp * S::kPitch : 0);
        unsigned char* const staging = sm + NS * S::kStage + (warp - kFirstEpi) * S::kWarpStaging;
        int half = 0;                                                               // of the staging: where the next 32 rows go
        auto put = [&](int unit, uint4 w, int block = 0) {
            *reinterpret_cast<uint4*>(staging + (half + block) * 4096 + lane * 128 + ((unit ^ (lane & 7)) << 4)) = w;
        };
        auto ready = [&] {                                                          // what was stored from there has been read
            if (lane == 0) {
                if constexpr (S::kHalves == 2) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
                else asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            }
            __syncwarp();
        };
        auto send = [&](int x, int y, int z) {
            fence_async_smem();
            __syncwarp();
            if (lane == 0) {
                if (x < a.N && y < a.M) {
                    tma_store_3d(&tmO, staging + half * 4096, x, y, z);
                    if constexpr (S::kOuts == 2) tma_store_3d(&tmO2, staging + 4096, x, y, z);
                }
                asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            }
            half ^= S::kHalves - 1;
        };
        // biases of the tile's columns, fp32: (EPI_GATE, EPI_GRAD) value and gate.  Two buffers, so that one barrier a tile is enough.
        float* const bias_at = reinterpret_cast<float*>(sm + S::kBiasAt) + grp * 2 * S::kBiasFloats;
        constexpr int kBiasCols = EPI == EPI_OUT ? S::kBiasFloats : S::kBiasFloats / 2;
        auto fill_bias = [&](float* to, int n0) {
            const T* const bias = (const T*)a.bias;
            for (int i = threadIdx.x & 127; i < S::kBiasFloats; i += 128) {
                const int gate = i >= kBiasCols, n = n0 + i - gate * kBiasCols;
                to[i] = bias && n < a.N ? to_f<T>(bias[n + gate * a.second]) : 0.f;
            }
            asm volatile("bar.sync %0, 128;" ::"r"(1 + grp) : "memory");
        };
        int it = 0;
        for (int i = walker; i < tiles; i += walkers, ++it) {
            if (NB == 2 && (it & 1) != grp) continue;
            const Tile t = tile_at(i);
            const int m0 = t.m0 + quarter * 32, n0 = t.n0, first = NB == 2 ? 0 : 64 * grp;
            float* const bias = bias_at + (it / NB & 1) * S::kBiasFloats;
            if constexpr (EPI != EPI_PART) fill_bias(bias, n0 + first);
            if (!mbar_wait_prompt(acc_full + it % NB, (it / NB) & 1, abort_flag)) break;
            __syncwarp();
            tc_fence_after();
            if constexpr (EPI == EPI_PART) {
#pragma unroll 1
                for (int c = 0; c < S::kOut; c += 32) {
                    uint32_t r[2][16];
                    ready();
                    tmem_ld16(lane_base + c, r[0]);
                    tmem_ld16(lane_base + c + 16, r[1]);
                    tmem_ld_wait();
#pragma unroll
                    for (int q = 0; q < 2; ++q)
#pragma unroll
                        for (int u = 0; u < 4; ++u) put(4 * q + u, make_uint4(r[q][4 * u], r[q][4 * u + 1], r[q][4 * u + 2], r[q][4 * u + 3]));
                    send(n0 + c, m0, t.split);
                }
            } else {
                // 16 columns at a time; the next ones leave TMEM while these are worked on
                constexpr int kIn = EPI == EPI_OUT ? 1 : EPI == EPI_GATE ? 2 : 3;
#pragma unroll 1
                for (int c = first; c < S::kOut; c += NB == 2 ? 64 : 128) {
                    uint32_t r[2][kIn][16];
                    auto load = [&](int q) {
#pragma unroll
                        for (int j = 0; j < kIn; ++j) tmem_ld16(lane_base + (j == 2 ? 2 + (it & 1) : j) * S::kOut + c + 16 * q, r[q & 1][j]);
                    };
                    ready();
                    load(0);
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        tmem_ld_wait();
                        if (q < 3) load(q + 1);
                        const auto& x = r[q & 1];
                        const float* const b = bias + c - first + 16 * q;
                        uint32_t w[8], w2[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const int e = 2 * j;
                            const float2 v = __fadd2_rn(make_float2(__uint_as_float(x[0][e]), __uint_as_float(x[0][e + 1])), *reinterpret_cast<const float2*>(b + e));
                            if constexpr (EPI == EPI_OUT) w[j] = Half2Of<T>::pack(v.x, v.y);
                            else {
                                const float2 g = __fadd2_rn(make_float2(__uint_as_float(x[1][e]), __uint_as_float(x[1][e + 1])),
                                                            *reinterpret_cast<const float2*>(b + kBiasCols + e));
                                if constexpr (EPI == EPI_GATE) {
                                    const float2 o = __fmul2_rn(v, act_pair<ACT>(g));
                                    w[j] = Half2Of<T>::pack(o.x, o.y);
                                } else {
                                    const float2 dh = make_float2(__uint_as_float(x[kIn - 1][e]), __uint_as_float(x[kIn - 1][e + 1]));
                                    float2 act, slope;
                                    act_grad_pair<ACT>(g, act, slope);
                                    const float2 dv = __fmul2_rn(dh, act), dg = __fmul2_rn(__fmul2_rn(dh, v), slope);
                                    w[j] = Half2Of<T>::pack(dv.x, dv.y);
                                    w2[j] = Half2Of<T>::pack(dg.x, dg.y);
                                }
                            }
                        }
                        put(2 * q, make_uint4(w[0], w[1], w[2], w[3]));
                        put(2 * q + 1, make_uint4(w[4], w[5], w[6], w[7]));
                        if constexpr (EPI == EPI_GRAD) {
                            put(2 * q, make_uint4(w2[0], w2[1], w2[2], w2[3]), 1);
                            put(2 * q + 1, make_uint4(w2[4], w2[5], w2[6], w2[7]), 1);
                        }
                    }
                    send(n0 + c, m0, 0);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if constexpr (kPair) mbar_arrive_at(in_rank(acc_empty + it % NB, 0));
                else mbar_arrive(acc_empty + it % NB);
            }
        }
        if (lane == 0) store_done();
    }
    // ---------------------------------------------------------------- teardown
    tc_fence_before();
    __syncthreads();
    if constexpr (kPair) cluster_sync();
    if (warp == 1) {
        tc_fence_after();
        if constexpr (kPair) tmem_dealloc_pair(tmem, S::kTmem);
        else tmem_dealloc(tmem, S::kTmem);
    }
    if (threadIdx.x == 0 && *abort_flag) atomicExch(a.error_flag, 1);
}

// ---- host --------------------------------------------------------------------------------------------------------------
// (splits, rows, cols) of T or fp32, rows `pitch` elements apart; box: 32 rows of 128 bytes
template <typename E> bool make_out_map(CUtensorMap* m, const void* base, long long splits, long long rows, long long cols, long long pitch) {
    EncodeFn enc = encode_fn();
    if (!enc) return false;
    CUtensorMapDataType dt;
    if constexpr (sizeof(E) == 4) dt = CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
    else dt = Fmt<E>::tm;
    const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)splits};
    const cuuint64_t strides[2] = {(cuuint64_t)(pitch * (long long)sizeof(E)), (cuuint64_t)(rows * pitch * (long long)sizeof(E))};
    const cuuint32_t box[3] = {128 / sizeof(E), 32, 1}, estr[3] = {1, 1, 1};
    return enc(m, dt, 3, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// An operand in memory: rows `pitch` elements apart, of the contraction where the kernel's kAMN / kBMN says so ("MN-major"), else of M / N
struct Operand {
    const void* p;
    long long pitch;
};
struct Product {
    Operand a, b, a2, b2;
    long long M, N, K, K2;          // N: columns of the result
    long long b_rows;               // rows of B in memory (EPI_GATE, EPI_GRAD: 2 N)
    const void* bias;
    void *out, *out2;
    long long out_pitch;
    int splits, per_split;          // EPI_PART
};

inline int sm_count() {
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
    return sms;
}

template <typename T, bool kAMN, bool kBMN, int EPI, int ACT, int kCols, bool kPair> int run_product(const Product& p, cudaStream_t st) {
    using S = Shape<EPI, kCols, kPair>;
    constexpr bool kDual = EPI == EPI_GATE || EPI == EPI_GRAD;
    constexpr auto sw = CU_TENSOR_MAP_SWIZZLE_128B;
    constexpr auto l2 = CU_TENSOR_MAP_L2_PROMOTION_L2_256B;       // 5 % faster than 128 bytes: a row's next 64 elements are the next stage's
    // (in front of the maps: a thread that has made no runtime call yet, one of autograd's for instance, has no context for the driver to encode in)
    int* host_flag = error_flag_for_current_device();
    if (!host_flag || *host_flag) return SS2D_ECUDA;                            // no flag, or an earlier launch on this device gave up on a wait
    int* dev_flag = nullptr;
    if (cudaHostGetDevicePointer((void**)&dev_flag, host_flag, 0) != cudaSuccess) return SS2D_ECUDA;
    CUtensorMap ta, tb, ta2, tb2, to, to2;
    bool ok = kAMN ? make_map_pitched(&ta, Fmt<T>::tm, p.a.p, p.K, p.M, p.a.pitch, kDepth, 64, sw, l2)
                   : make_map_pitched(&ta, Fmt<T>::tm, p.a.p, p.M, p.K, p.a.pitch, kRows, kDepth, sw, l2);
    ok = ok && (kBMN && !kDual ? make_map_pitched(&tb, Fmt<T>::tm, p.b.p, p.K, p.N, p.b.pitch, kDepth, 64, sw, l2)
                               : make_map_pitched(&tb, Fmt<T>::tm, p.b.p, p.b_rows, p.K, p.b.pitch, kDual ? S::kOut : S::kB / S::kShare, kDepth, sw, l2));
    ta2 = ta; tb2 = tb;
    if constexpr (EPI == EPI_GRAD)
        ok = ok && make_map_pitched(&ta2, Fmt<T>::tm, p.a2.p, p.M, p.K2, p.a2.pitch, kRows, kDepth, sw, l2) &&
             make_map_pitched(&tb2, Fmt<T>::tm, p.b2.p, p.K2, p.N, p.b2.pitch, kDepth, 64, sw, l2);
    if constexpr (EPI == EPI_PART) ok = ok && make_out_map<float>(&to, p.out, p.splits, p.M, p.N, p.out_pitch);
    else ok = ok && make_out_map<T>(&to, p.out, 1, p.M, p.N, p.out_pitch);
    to2 = to;
    if constexpr (EPI == EPI_GRAD) ok = ok && make_out_map<T>(&to2, p.out2, 1, p.M, p.N, p.out_pitch);
    if (!ok) return SS2D_ECUDA;
    auto kern = product_tc05_kernel<T, kAMN, kBMN, EPI, ACT, kCols, kPair>;
    if (const int rc = allow_dynamic_smem(kern, S::kBytes)) return rc;
    Args a = {};
    a.m_tiles = (int)((p.M + kRows * S::kShare - 1) / (kRows * S::kShare)); a.n_tiles = (int)((p.N + S::kOut - 1) / S::kOut);
    a.splits = EPI == EPI_PART ? p.splits : 1;
    a.blocks = (int)((p.K + kDepth - 1) / kDepth); a.per_split = EPI == EPI_PART ? p.per_split : a.blocks;
    a.blocks2 = (int)((p.K2 + kDepth - 1) / kDepth);
    a.M = (int)p.M; a.N = (int)p.N; a.second = (int)p.N; a.bias = p.bias; a.error_flag = dev_flag;
    const int tiles = a.m_tiles * a.n_tiles * a.splits, sms = sm_count();
    if (!sms) return SS2D_ECUDA;
    const int walkers = tiles < sms / S::kShare ? tiles : sms / S::kShare;
    if constexpr (kPair) launch_pairs(kern, walkers * 2, kThreads, S::kBytes, st, ta, tb, ta2, tb2, to, to2, a);
    else launch(kern, walkers, kThreads, S::kBytes, st, ta, tb, ta2, tb2, to, to2, a);
    count_launch();
    return check_launch();
}

}  // namespace ptc
}  // namespace ss2d
