// Linear attention with a decay for each head:
//   S_t = exp(g_t) S_{t-1} + k_t v_t^T        (S: dk x dv, fp32)
//   o_t = scale S_t^T q_t
// walked in chunks of 64 tokens.  With G the cumulative sum of g inside a chunk (base 2 from here on), e_i = 2^G_i, w_j = 2^(G_C - G_j):
//   o_i  = scale (e_i S_in^T q_i + sum_{j <= i} 2^(G_i - G_j) (q_i . k_j) v_j)
//   S_out = 2^G_C S_in + sum_j w_j k_j v_j^T
// and for the gradients, with dS the gradient of the state behind the chunk,
//   dS_in = 2^G_C dS + scale sum_i e_i q_i do_i^T
//   dq_i  = scale (e_i S_in do_i + sum_{j <= i} D_ij (do_i . v_j) k_j),   D_ij = 2^(G_i - G_j)
//   dk_j  = w_j dS v_j + scale sum_{i >= j} D_ij (do_i . v_j) q_i
//   dv_j  = w_j dS^T k_j + scale sum_{i >= j} D_ij (q_i . k_j) do_i
//   dg_t  = what crosses the boundary in front of token t: 2^G_C <S_in, dS> + sum_{s >= t} scale e_s q_s^T S_in do_s
//           + sum_{r < t} w_r k_r^T dS v_r + sum_{r < t <= s} scale D_sr (q_s . k_r)(do_s . v_r)
// (the telescoped form q . dq - k . dk summed from the end needs no states, but its terms cancel over the whole sequence: with products of
// 16-bit operands the noise of thousands of tokens stays in every dg).
//
// Decays are differences of two numbers, an integer and a fraction, so that a chunk whose decays run to thousands loses nothing of the small
// ones behind; log decays below 2^-200 a token count as a reset (exp is 0 in fp32 long before), so -inf is one.
//
// Kernels.  la_walk: one CTA per (sequence, head, 32 or 64 columns of v, segment of chunks) walks its chunks with the state in registers and writes
// outputs and, where asked, the state in front of every chunk; the same kernel without outputs gathers the states of a segment, or the state gradients
// backwards.  la_join: states in front of the segments from those that the segments gather.  la_grad: everything else of the backward pass, one CTA per
// (sequence, group of heads, chunk), no order between them.  la_step: one token, the state read and written once.  Long bf16 sequences of wide heads take
// linear_attention_tc.cuh in place of the walk.
//
// What bounds them (B200): the walk issues some 10 instructions for each matrix instruction and its warps wait for one another at two barriers a chunk (issue 55 %, tensor
// pipe 33 %, DRAM 5 % of their rates at 16 x 784 tokens of 24 heads of 64 x 32, fp16: 75 us, 8 of them for its bytes); la_grad waits at barriers for loads of a chunk that nothing
// overlaps but the other CTA of the SM (issue 38 %, tensor pipe 20 %, DRAM 16 % at 16 x 3 136 tokens of 12 heads of 64 x 32: 268 us; when states came in two pieces, 264, of which
// 114 were loads, decays, barriers and stores, 55 the pairs, 65 the products with the states); la_step is a copy of the state (128 sequences of 16 heads of 128 x 128: 52 us, 5.2 TB/s, 0.79 of the copy rate).
#include "mma_tiles.cuh"

namespace ss2d {

namespace {

using namespace mt;

constexpr int kChunk = 64;
constexpr int kSlab = 32;           // rows of the states that the gradient kernel holds at a time
constexpr float kFloor = -200.f;    // 2^-200 is 0 in fp32

struct Rows {                       // (batch, token, head) rows of contiguous elements
    const void* p;
    long long b, l, h;
    bool vec;
};

// ---- decays of a chunk -------------------------------------------------------------------------------------------------
struct Cum { float n, f; };         // n + f, n whole, 0 <= f < 1: exact in n, 2^-25 in f
__device__ __forceinline__ Cum cum_of(float log_decay) {
    float x = log_decay * kLog2e;
    x = x < kFloor ? kFloor : x;    // (NaN stays)
    const float n = floorf(x), f = x - n;
    return f >= 1.f ? Cum{n + 1.f, 0.f} : Cum{n, f};        // (x between -2^-25 and 0: its fraction rounds up)
}
__device__ __forceinline__ Cum cum_add(Cum a, Cum b) {
    const float f = a.f + b.f, c = f >= 1.f ? 1.f : 0.f;
    return {a.n + b.n + c, f - c};
}
__device__ __forceinline__ float exp_diff(Cum a, Cum b) { return ex2_approx((a.n - b.n) + (a.f - b.f)); }

struct alignas(16) Decays {
    float n[kChunk], f[kChunk];     // cumulative sums
    float e[kChunk], w[kChunk];     // 2^G_i, 2^(G_C - G_i)
    // Pairs in different blocks of 16 tokens: 2^(G_i - G_j) = near[i] far[block of i][j], both at most 1 where decays are, G at the block's first token
    // between them: one exponential a token in place of one a pair.
    float near[kChunk], far[4][kChunk];
    float total_n, total_f, total;  // G_C, 2^G_C
    __device__ __forceinline__ Cum at(int i) const { return {n[i], f[i]}; }
};
// one warp: from the log decays of tokens 2 lane and 2 lane + 1
__device__ __forceinline__ void fill_decays(Decays& d, float g0, float g1, int lane) {
    const Cum a = cum_of(g0);
    Cum s = cum_add(a, cum_of(g1));
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const Cum o = {__shfl_up_sync(0xffffffffu, s.n, off), __shfl_up_sync(0xffffffffu, s.f, off)};
        if (lane >= off) s = cum_add(o, s);
    }
    Cum before = {__shfl_up_sync(0xffffffffu, s.n, 1), __shfl_up_sync(0xffffffffu, s.f, 1)};
    if (lane == 0) before = {0.f, 0.f};
    const Cum first = cum_add(before, a);
    const Cum all = {__shfl_sync(0xffffffffu, s.n, 31), __shfl_sync(0xffffffffu, s.f, 31)};
    d.n[2 * lane] = first.n; d.f[2 * lane] = first.f;
    d.n[2 * lane + 1] = s.n; d.f[2 * lane + 1] = s.f;
    d.e[2 * lane] = ex2_approx(first.n + first.f);
    d.e[2 * lane + 1] = ex2_approx(s.n + s.f);
    d.w[2 * lane] = exp_diff(all, first);
    d.w[2 * lane + 1] = exp_diff(all, s);
    if (lane == 0) { d.total_n = all.n; d.total_f = all.f; d.total = ex2_approx(all.n + all.f); }
#pragma unroll
    for (int b = 0; b < 4; ++b) {
        const Cum start = {__shfl_sync(0xffffffffu, first.n, 8 * b), __shfl_sync(0xffffffffu, first.f, 8 * b)};
        if (lane / 8 == b) { d.near[2 * lane] = exp_diff(first, start); d.near[2 * lane + 1] = exp_diff(s, start); }
        if (lane / 8 < b) { d.far[b][2 * lane] = exp_diff(start, first); d.far[b][2 * lane + 1] = exp_diff(start, s); }
    }
}
// a token past the end decays nothing
__device__ __forceinline__ void load_decays(float& g0, float& g1, const float* g, long long stride, int first, int L, int lane) {
    const int t = first + 2 * lane;
    g0 = t < L ? g[t * stride] : 0.f;
    g1 = t + 1 < L ? g[(t + 1) * stride] : 0.f;
}

// A state that the gradient kernel reads: rows of `state_row(dv)` elements, fp32.  What is behind dv is zero.
__host__ __device__ constexpr int state_row(int dv) { return (dv + 7) / 8 * 8; }

// ---- walking a sequence ------------------------------------------------------------------------------------------------
struct WalkArgs {
    Rows q, k, v;                   // kOut: q, k, v.  Otherwise the rows of the state's update: k (forwards) or q (backwards), and v or do
    const float* g;
    long long g_b, g_l, g_h;
    const float* start;             // (B, H, segments, dk, dv) or NULL: zeros
    float* end;                     // the same, or NULL
    float* end_decay;               // (B, H, segments): log2 of the decay over the segment, or NULL
    float* states;                  // (B, H, chunks) states (above): in front of every chunk (walking backwards: behind it), or NULL
    void* o;                        // (B, L, H, dv)
    int H, rep, L, dk, dv, chunks, per_segment, segments, pairs;
    float scale;
};

template <typename T, int DK, int DVT> struct WalkSmem {
    using P = typename Plane<T>::type;
    static constexpr int kLdK = DK + 8, kLdV = DVT + 8;
    static constexpr int kQ = kChunk * kLdK, kV = kChunk * kLdV;       // elements
    static constexpr size_t stage(bool out) { return ((out ? 2 : 1) * kQ + kV) * sizeof(T); }
    static constexpr size_t plane(bool out) { return out ? DK * kLdV * sizeof(P) : 0; }
    static constexpr size_t bytes(bool out) { return 2 * stage(out) + plane(out) + 2 * sizeof(Decays); }
};

// Four warps.  Outputs: a warp has 16 tokens.  State: a warp has DK / 4 of its rows, in accumulators, DK / 64 blocks of 16 (one for two warps at DK = 32).
template <typename T, int DK, int DVT, bool kOut, bool kBack>
__global__ void __launch_bounds__(128) la_walk_kernel(const WalkArgs a) {
    follow_previous();
    using M = WalkSmem<T, DK, DVT>;
    using P = typename M::P;
    extern __shared__ __align__(16) unsigned char smem[];
    constexpr int kBlocks = (DK + 63) / 64, NT = DVT / 8;
    T* const stage0 = reinterpret_cast<T*>(smem);
    P* const plane = reinterpret_cast<P*>(smem + 2 * M::stage(kOut));
    Decays* const decays = reinterpret_cast<Decays*>(smem + 2 * M::stage(kOut) + M::plane(kOut));
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gq = lane >> 2, t = lane & 3;
    const int slices = (a.dv + DVT - 1) / DVT, slice = blockIdx.x % slices, bh = blockIdx.x / slices, seg = blockIdx.y;
    const int v0 = slice * DVT, dv = min(DVT, a.dv - v0), b = bh / a.H, h = bh % a.H;
    const int c0 = seg * a.per_segment, c1 = min(a.chunks, c0 + a.per_segment);
    const T* const q = (const T*)a.q.p + b * a.q.b + (h / a.rep) * a.q.h;
    const T* const k = (const T*)a.k.p + b * a.k.b + (h / a.rep) * a.k.h;
    const T* const v = (const T*)a.v.p + b * a.v.b + h * a.v.h + v0;
    const float* const g = a.g + b * a.g_b + h * a.g_h;
    const long long state_size = (long long)a.dk * a.dv;

    float S[kBlocks][NT][4];
    const int m_first = warp * 16;                         // first row of the warp's block 0; the next one is 64 rows on
    const bool holds = DK >= 64 || warp < DK / 16;
    auto for_state = [&](auto&& f) {                       // f(row, column, first of two accumulators)
#pragma unroll
        for (int m = 0; m < kBlocks; ++m)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int r = 0; r < 2; ++r) f(m_first + 64 * m + gq + 8 * r, 8 * n + 2 * t, S[m][n] + 2 * r);
    };
    {
        const float* s0 = a.start ? a.start + ((long long)bh * a.segments + seg) * state_size + v0 : nullptr;
        for_state([&](int row, int col, float* s) {
            const bool in = s0 && holds && row < a.dk;
            s[0] = in && col < dv ? s0[(long long)row * a.dv + col] : 0.f;
            s[1] = in && col + 1 < dv ? s0[(long long)row * a.dv + col + 1] : 0.f;
        });
    }
    auto put_plane = [&] {
        if constexpr (kOut)
            if (holds) for_state([&](int row, int col, float* s) { put2<T, 1>(plane + row * M::kLdV + col, 0, s[0], s[1]); });
    };
    auto write_state = [&](float* to) {
        if (holds)
            for_state([&](int row, int col, float* s) {
                if (row >= a.dk) return;
                float* p = to + (long long)row * a.dv + v0 + col;
                if (a.pairs && col + 1 < dv) *reinterpret_cast<float2*>(p) = make_float2(s[0], s[1]);
                else {
                    if (col < dv) p[0] = s[0];
                    if (col + 1 < dv) p[1] = s[1];
                }
            });
    };
    auto keep_state = [&](long long which) {
        const int ld = state_row(a.dv);
        float* const to = a.states + which * a.dk * ld + v0;
        if (holds)
            for_state([&](int row, int col, float* s) {
                if (row < a.dk && v0 + col < ld) *reinterpret_cast<float2*>(to + row * ld + col) = make_float2(s[0], s[1]);
            });
    };
    auto fetch = [&](int c, int buf) {
        T* s = stage0 + buf * ((kOut ? 2 : 1) * M::kQ + M::kV);
        const int first = c * kChunk, rows = min(kChunk, a.L - first);
        fetch_rows<T, kChunk, DK>(s, M::kLdK, k + (long long)first * a.k.l, a.k.l, rows, a.dk, a.k.vec, tid, 128);
        fetch_rows<T, kChunk, DVT>(s + M::kQ, M::kLdV, v + (long long)first * a.v.l, a.v.l, rows, dv, a.v.vec, tid, 128);
        if constexpr (kOut) fetch_rows<T, kChunk, DK>(s + M::kQ + M::kV, M::kLdK, q + (long long)first * a.q.l, a.q.l, rows, a.dk, a.q.vec, tid, 128);
        commit_copies();
    };

    const int n = c1 - c0;
    auto chunk_at = [&](int i) { return kBack ? c1 - 1 - i : c0 + i; };
    float g0 = 0.f, g1 = 0.f;
    auto next_decays = [&](int i) {                        // by warp 0, which has the fewest pairs: chunk i's, and the loads for the one behind it
        if (warp == 0 && i < n) {
            fill_decays(decays[i & 1], g0, g1, lane);
            if (i + 1 < n) load_decays(g0, g1, g, a.g_l, chunk_at(i + 1) * kChunk, a.L, lane);
        }
    };
    fetch(chunk_at(0), 0);
    if (warp == 0) load_decays(g0, g1, g, a.g_l, chunk_at(0) * kChunk, a.L, lane);
    next_decays(0);
    put_plane();
    Cum over = {0.f, 0.f};
    for (int i = 0; i < n; ++i) {
        const int c = chunk_at(i), buf = i & 1;
        Decays& d = decays[buf];
        wait_copies();
        __syncthreads();
        if (i + 1 < n) fetch(chunk_at(i + 1), buf ^ 1);
        next_decays(i + 1);
        if (a.states) keep_state((long long)bh * a.chunks + c);
        const T* sk = stage0 + buf * ((kOut ? 2 : 1) * M::kQ + M::kV);
        const T* sv = sk + M::kQ;
        if constexpr (kOut) {
            const T* sq = sv + M::kV;
            const int r0 = warp * 16;
            float p[8][4] = {}, o[NT][4] = {};
#pragma unroll
            for (int k0 = 0; k0 < DK; k0 += 16) {
                const OpA<T> qa = load_a<false>(sq, M::kLdK, r0, k0, lane);
#pragma unroll
                for (int j = 0; j < 8; j += 2)
                    if (j <= 2 * warp) {                   // keys up to the warp's last token
                        OpB<T> b0, b1;
                        load_b2<false>(b0, b1, sk, M::kLdK, 8 * j, k0, lane);
                        mma_exact(p[j], qa, b0);
                        mma_exact(p[j + 1], qa, b1);
                    }
#pragma unroll
                for (int j = 0; j < NT; j += 2) mma_plane2<T, 1, true>(o[j], o[j + 1], qa, plane, 0, M::kLdV, 8 * j, k0, lane);
            }
            const Cum lo = d.at(r0 + gq), hi = d.at(r0 + gq + 8);
            const float el = d.e[r0 + gq], eh = d.e[r0 + gq + 8], nl = d.near[r0 + gq], nh = d.near[r0 + gq + 8];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                o[j][0] *= el; o[j][1] *= el; o[j][2] *= eh; o[j][3] *= eh;
            }
#pragma unroll
            for (int j = 0; j < 8; j += 2)
                if (j <= 2 * warp) {
                    float x[8];
                    if (j < 2 * warp) {
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            const float2 f = *reinterpret_cast<const float2*>(d.far[warp] + 8 * (j + u) + 2 * t);
                            x[4 * u] = p[j + u][0] * (nl * f.x); x[4 * u + 1] = p[j + u][1] * (nl * f.y);
                            x[4 * u + 2] = p[j + u][2] * (nh * f.x); x[4 * u + 3] = p[j + u][3] * (nh * f.y);
                        }
                    } else {
#pragma unroll
                        for (int u = 0; u < 2; ++u)
#pragma unroll
                            for (int s = 0; s < 2; ++s) {
                                const int col = 8 * (j + u) + 2 * t + s;
                                const Cum at = d.at(col);
                                x[4 * u + s] = col <= r0 + gq ? p[j + u][s] * exp_diff(lo, at) : 0.f;
                                x[4 * u + 2 + s] = col <= r0 + gq + 8 ? p[j + u][2 + s] * exp_diff(hi, at) : 0.f;
                            }
                    }
                    const Derived<T, 1> pd = derive<T, 1>(x);
#pragma unroll
                    for (int u = 0; u < NT; u += 2) {
                        OpB<T> b0, b1;
                        load_b2<true>(b0, b1, sv, M::kLdV, 8 * u, 8 * j, lane);
                        mma_derived<T, 1>(o[u], pd, b0);
                        mma_derived<T, 1>(o[u + 1], pd, b1);
                    }
                }
            T* const out = (T*)a.o + ((long long)b * a.L + c * kChunk) * a.H * a.dv + (long long)h * a.dv + v0;
            const int rows = min(kChunk, a.L - c * kChunk);
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int row = r0 + gq + 8 * r;
                if (row < rows) {
                    T* to = out + (long long)row * a.H * a.dv;
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        const int col = 8 * j + 2 * t;
                        const float y[2] = {a.scale * o[j][2 * r], a.scale * o[j][2 * r + 1]};
                        if (a.pairs && col + 1 < dv) Vec<T, 2>::store(to + col, y);
                        else {
                            if (col < dv) to[col] = from_f<T>(y[0]);
                            if (col + 1 < dv) to[col + 1] = from_f<T>(y[1]);
                        }
                    }
                }
            }
            __syncthreads();                               // the plane has been read
        }
        // state: rows of k^T weighted by what is left of them at the end of the chunk (backwards: of q^T by what reaches them)
        const float keep = d.total;
        if (holds) {
            // a chunk's products are summed on their own: tensor cores cut sums off towards zero, which a state of thousands of tokens would collect
#pragma unroll
            for (int m = 0; m < kBlocks; ++m) {
                float add[NT][4] = {};
#pragma unroll
                for (int k0 = 0; k0 < kChunk; k0 += 16) {
                    const float* w = kBack ? d.e : d.w;
                    float ws[4] = {w[k0 + 2 * t], w[k0 + 2 * t + 1], w[k0 + 8 + 2 * t], w[k0 + 9 + 2 * t]};
                    if constexpr (kBack) {
#pragma unroll
                        for (int s = 0; s < 4; ++s) ws[s] *= a.scale;
                    }
                    float x[8];
                    values(load_a<true>(sk, M::kLdK, m_first + 64 * m, k0, lane), x);
#pragma unroll
                    for (int s = 0; s < 8; ++s) x[s] *= ws[(s & 1) + 2 * (s >> 2)];
                    // the state is an fp32 result: three pieces of bf16, two of tf32
                    constexpr int kPieces = std::is_same<T, __nv_bfloat16>::value ? 3 : 2;
                    const Derived<T, kPieces> kd = derive<T, kPieces>(x);
#pragma unroll
                    for (int j = 0; j < NT; j += 2) {
                        OpB<T> b0, b1;
                        load_b2<true>(b0, b1, sv, M::kLdV, 8 * j, k0, lane);
                        mma_derived<T, kPieces>(add[j], kd, b0);
                        mma_derived<T, kPieces>(add[j + 1], kd, b1);
                    }
                }
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int s = 0; s < 4; ++s) S[m][j][s] = fmaf(keep, S[m][j][s], add[j][s]);
            }
        }
        put_plane();
        over = cum_add(over, {d.total_n, d.total_f});
    }
    if (a.end) write_state(a.end + ((long long)bh * a.segments + seg) * state_size);
    if (a.end_decay && slice == 0 && tid == 0) a.end_decay[(long long)bh * a.segments + seg] = over.n + over.f;
}

// ---- states in front of the segments -----------------------------------------------------------------------------------
struct JoinArgs {
    const float* first;             // (B, H, dk, dv) or NULL
    float* part;                    // (B, H, segments, dk, dv): what the segments gather; becomes the state that each starts from
    const float* decay;             // (B, H, segments)
    float* last;                    // (B, H, dk, dv) or NULL
    long long size;                 // dk dv
    int segments;
    bool back;
};
__global__ void __launch_bounds__(256) la_join_kernel(const JoinArgs a) {
    follow_previous();
    const long long blocks = (a.size + 255) / 256, bh = blockIdx.x / blocks, e = blockIdx.x % blocks * 256 + threadIdx.x;
    if (e >= a.size) return;
    float s = a.first ? a.first[bh * a.size + e] : 0.f;
    constexpr int kAhead = 8;               // what several segments have gathered, read side by side
    for (int i0 = 0; i0 < a.segments; i0 += kAhead) {
        float x[kAhead], d[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
            if (i0 + i < a.segments) {
                const long long at = bh * a.segments + (a.back ? a.segments - 1 - i0 - i : i0 + i);
                x[i] = a.part[at * a.size + e];
                d[i] = a.decay[at];
            }
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
            if (i0 + i < a.segments) {
                const long long at = bh * a.segments + (a.back ? a.segments - 1 - i0 - i : i0 + i);
                a.part[at * a.size + e] = s;
                s = fmaf(ex2_approx(d[i]), s, x[i]);
            }
    }
    if (a.last) a.last[bh * a.size + e] = s;
}

// ---- gradients of a chunk ----------------------------------------------------------------------------------------------
struct GradArgs {
    Rows q, k, v, dy;
    const float* g;
    long long g_b, g_l, g_h;
    const float *states, *dstates;  // (B, H, chunks) states: in front of the chunk; gradient of the state behind it
    void *dq, *dk_, *dv_;           // dense
    float* dg;                      // (B, L, H)
    int G, rep, L, dk, dv, chunks, pairs_k, pairs_v;
    float scale;
};

template <typename T, int DK, int DV> struct GradShape {
    using P = typename Plane<T>::type;
    static constexpr bool kSplit = Plane<T>::kSplit;
    static constexpr int kPlanes = kSplit ? 3 : 1;
    static constexpr int kGroups = DK == 128 || DV == 128 ? 3 : 2;      // groups of four warps: dq; dk and dv, apart where both would not stay in registers
    static constexpr int kThreads = 128 * kGroups, kSlabs = DK / kSlab;
    static constexpr int kLdK = DK + 8, kLdV = DV + 8, kLdP = kChunk + 8;
    static constexpr int kK = kChunk * kLdK, kV = kChunk * kLdV, kPair = kChunk * kLdP, kPlane = kSlab * kLdV;
    static constexpr size_t kRowBytes = (2 * kK + 2 * kV) * sizeof(T), kPairBytes = 2 * kPair * sizeof(P), kSlabBytes = 2 * kPlanes * kPlane * sizeof(P);
    static constexpr size_t kSums = (3 + 4 + 2) * kChunk * sizeof(float) + 64;
    static constexpr size_t kWaitBytes = kSplit ? 2 * kSlab * DV * sizeof(float) : 0;       // beside bf16: a slab in fp32, on its way into pieces
    static constexpr size_t kFixed = kRowBytes + kPairBytes + kWaitBytes + sizeof(Decays) + kSums;
    static constexpr int kStages = kSplit || kSlabs == 1 || kFixed + 2 * kSlabBytes > 232448 ? 1 : 2;
    static constexpr size_t kBytes = kFixed + kStages * kSlabBytes;
    static constexpr int kResident = 2 * (kBytes + 1024) <= 233472 && kGroups == 2 ? 2 : 1;
    static_assert(kBytes <= 232448);
};

// Pairs first: the 16 x 16 blocks of the lower triangle go round the warps, each gives decayed q . k and do . v, their sums by row and column, and both as operands in
// shared memory.  Then a group of warps has dq, 16 queries a warp, another dk and dv, 16 keys a warp; the states pass in slabs of 32 rows, beside bf16 in three pieces: the gradients of
// the decays are fp32 results, sums over products with both states whose terms cancel (of two pieces 2e-6 to 4e-6 from 64 bits, of three 3e-7 to 5e-7, as of elementary fp32 operations; training of 2 x 4 096
// tokens of 16 heads of 128 x 128 459 -> 502 us, of 16 x 3 136 of 12 heads of 64 x 32 522 -> 518).  Heads that share
// their keys follow one another with dq and dk in accumulators.
template <typename T, int DK, int DV>
__global__ void __launch_bounds__(GradShape<T, DK, DV>::kThreads, GradShape<T, DK, DV>::kResident) la_grad_kernel(const GradArgs a) {
    follow_previous();
    using M = GradShape<T, DK, DV>;
    using P = typename M::P;
    constexpr int kLdK = M::kLdK, kLdV = M::kLdV, kLdP = M::kLdP, kThreads = M::kThreads, kGroups = M::kGroups;
    extern __shared__ __align__(16) unsigned char smem[];
    T *const sq = reinterpret_cast<T*>(smem), *const sk = sq + M::kK, *const sv = sk + M::kK, *const sy = sv + M::kV;
    P *const s_w = reinterpret_cast<P*>(smem + M::kRowBytes), *const s_a = s_w + M::kPair, *const slabs = s_a + M::kPair;
    float* const waiting = reinterpret_cast<float*>(smem + M::kRowBytes + M::kPairBytes + M::kStages * M::kSlabBytes);
    Decays& d = *reinterpret_cast<Decays*>(smem + M::kRowBytes + M::kPairBytes + M::kStages * M::kSlabBytes + M::kWaitBytes);
    float *const row_sum = reinterpret_cast<float*>(&d + 1), *const col_sum = row_sum + 3 * kChunk, *const into = col_sum + 4 * kChunk, *const from = into + kChunk,
                *const cross = from + kChunk;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gq = lane >> 2, t = lane & 3;
    const int group = warp >> 2, w4 = warp & 3, r0 = 16 * w4;
    const int c = blockIdx.x % a.chunks, bg = blockIdx.x / a.chunks, b = bg / a.G, grp = bg % a.G, H = a.G * a.rep;
    const int first = c * kChunk, rows = min(kChunk, a.L - first);
    const int ld = state_row(a.dv), n_slabs = (a.dk + kSlab - 1) / kSlab;
    auto src = [&](const Rows& r, int head) { return (const T*)r.p + b * r.b + (long long)first * r.l + head * r.h; };
    // what the group computes for its rows (queries for dq, keys for dk and dv); dq and dk of all heads, dv of one
    const bool has_dq = group == 0, has_dk = group == 1, has_dv = group == kGroups - 1;
    // dq or dk in blocks of 8 columns, and behind them dv; in their place where the groups of warps are three and none has both
    constexpr int kDv = kGroups == 3 ? 0 : DK / 8;
    float acc_all[(kGroups == 3 ? (DK > DV ? DK : DV) / 8 : DK / 8 + DV / 8)][4] = {};
    fetch_rows<T, kChunk, DK>(sq, kLdK, src(a.q, grp), a.q.l, rows, a.dk, a.q.vec, tid, kThreads);
    fetch_rows<T, kChunk, DK>(sk, kLdK, src(a.k, grp), a.k.l, rows, a.dk, a.k.vec, tid, kThreads);
    for (int hh = 0; hh < a.rep; ++hh) {
        const int h = grp * a.rep + hh;
        if (hh) __syncthreads();
        fetch_rows<T, kChunk, DV>(sv, kLdV, src(a.v, h), a.v.l, rows, a.dv, a.v.vec, tid, kThreads);
        fetch_rows<T, kChunk, DV>(sy, kLdV, src(a.dy, h), a.dy.l, rows, a.dv, a.dy.vec, tid, kThreads);
        const long long at = ((long long)(b * H + h) * a.chunks + c) * a.dk * ld;
        auto fetch_slab = [&](int s) {
            if (s < n_slabs) {
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    const float* g = (p ? a.dstates : a.states) + at + s * kSlab * ld;
                    if constexpr (M::kSplit) fetch_rows<float, kSlab, DV>(waiting + p * kSlab * DV, DV, g, ld, a.dk - s * kSlab, ld, true, tid, kThreads);
                    else fetch_rows<float, kSlab, DV>(slabs + ((s % M::kStages) * 2 + p) * M::kPlane, kLdV, g, ld, a.dk - s * kSlab, ld, true, tid, kThreads);
                }
            }
            commit_copies();
        };
        float both = 0.f;                                  // <S, dS>, this thread's share
        auto take_slab = [&]() {                           // beside bf16: what has waited, into pieces
            for (int i = tid; i < kSlab * DV / 2; i += kThreads) {
                const int row = i / (DV / 2), col = i % (DV / 2) * 2;
                const float2 x = *reinterpret_cast<const float2*>(waiting + row * DV + col), y = *reinterpret_cast<const float2*>(waiting + (kSlab + row) * DV + col);
                both = fmaf(x.x, y.x, fmaf(x.y, y.y, both));
                put2<T, 3>(slabs + row * kLdV + col, M::kPlane, x.x, x.y);
                put2<T, 3>(slabs + M::kPlanes * M::kPlane + row * kLdV + col, M::kPlane, y.x, y.y);
            }
        };
        fetch_slab(0);
        if constexpr (M::kStages == 2) fetch_slab(1);
        if (warp == 0) {
            float g0, g1;
            load_decays(g0, g1, a.g + b * a.g_b + h * a.g_h, a.g_l, first, a.L, lane);
            fill_decays(d, g0, g1, lane);
        }
        wait_copies<M::kStages - 1>();
        __syncthreads();
        if constexpr (M::kSplit) take_slab();
        {
            float sum[2] = {0.f, 0.f};
            const Cum own[2] = {d.at(r0 + gq), d.at(r0 + gq + 8)};
            const float near[2] = {a.scale * d.near[r0 + gq], a.scale * d.near[r0 + gq + 8]};
            for (int cb = group; cb <= w4; cb += kGroups) {
                float qk[2][4] = {}, yv[2][4] = {};
#pragma unroll
                for (int k0 = 0; k0 < DK; k0 += 16) {
                    OpB<T> b0, b1;
                    const OpA<T> x = load_a<false>(sq, kLdK, r0, k0, lane);
                    load_b2<false>(b0, b1, sk, kLdK, 16 * cb, k0, lane);
                    mma_exact(qk[0], x, b0);
                    mma_exact(qk[1], x, b1);
                }
#pragma unroll
                for (int k0 = 0; k0 < DV; k0 += 16) {
                    OpB<T> b0, b1;
                    const OpA<T> x = load_a<false>(sy, kLdV, r0, k0, lane);
                    load_b2<false>(b0, b1, sv, kLdV, 16 * cb, k0, lane);
                    mma_exact(yv[0], x, b0);
                    mma_exact(yv[1], x, b1);
                }
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    float col[2] = {0.f, 0.f};
                    const int n = 16 * cb + 8 * u + 2 * t;
                    const float2 far = *reinterpret_cast<const float2*>(d.far[w4] + n);
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const int m = r0 + gq + 8 * r;
                        float x[2], y[2];
#pragma unroll
                        for (int s = 0; s < 2; ++s) {
                            const float D = cb < w4 ? near[r] * (s ? far.y : far.x) : n + s <= m ? a.scale * exp_diff(own[r], d.at(n + s)) : 0.f;
                            x[s] = D * qk[u][2 * r + s];
                            y[s] = D * yv[u][2 * r + s];
                            // the pair of a token with itself crosses nothing
                            const float w = n + s < m ? x[s] * yv[u][2 * r + s] : 0.f;
                            sum[r] += w;
                            col[s] += w;
                        }
                        put2<T, 1>(s_w + m * kLdP + n, 0, x[0], x[1]);
                        put2<T, 1>(s_a + m * kLdP + n, 0, y[0], y[1]);
                    }
#pragma unroll
                    for (int s = 0; s < 2; ++s) {
#pragma unroll
                        for (int off = 4; off < 32; off <<= 1) col[s] += __shfl_xor_sync(0xffffffffu, col[s], off);
                        if (gq == 0) col_sum[w4 * kChunk + n + s] = col[s];
                    }
                }
            }
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 1);
                sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 2);
                if (t == 0) row_sum[group * kChunk + r0 + gq + 8 * r] = sum[r];
            }
        }
        __syncthreads();
        const float wl = (has_dq ? a.scale * d.e[r0 + gq] : d.w[r0 + gq]), wh = (has_dq ? a.scale * d.e[r0 + gq + 8] : d.w[r0 + gq + 8]);
        float (*const total)[4] = acc_all, (*const dv)[4] = acc_all + kDv;
        if (has_dv) {
#pragma unroll
            for (int j = 0; j < DV / 8; ++j)
#pragma unroll
                for (int s = 0; s < 4; ++s) dv[j][s] = 0.f;
        }
        float through[2] = {0.f, 0.f};
        const T *const X = has_dq ? sy : sv, *const Own = has_dq ? sq : sk, *const Other = has_dq ? sk : sq;
#pragma unroll
        for (int s = 0; s < M::kSlabs; ++s) {
            if (s < n_slabs) {
                const int m0 = s * kSlab;
                if (s) {
                    wait_copies<M::kStages - 1>();
                    __syncthreads();
                    if constexpr (M::kSplit) {
                        take_slab();
                        __syncthreads();
                    }
                }
                if constexpr (M::kSplit) fetch_slab(s + 1);
                const P *const s_in = slabs + (s % M::kStages) * (2 * M::kPlanes * M::kPlane), *const s_out = s_in + M::kPlanes * M::kPlane;
                if constexpr (!M::kSplit)
                    for (int i = tid; i < kSlab * DV / 2; i += kThreads) {
                        const int at = i / (DV / 2) * kLdV + i % (DV / 2) * 2;
                        both = fmaf(s_in[at], s_out[at], fmaf(s_in[at + 1], s_out[at + 1], both));
                    }
                if (has_dq || has_dk) {
                    const P* const S = has_dq ? s_in : s_out;
                    float acc[4][4] = {};
#pragma unroll
                    for (int k0 = 0; k0 < DV; k0 += 16) {
                        const OpA<T> x = load_a<false>(X, kLdV, r0, k0, lane);
#pragma unroll
                        for (int j = 0; j < 4; j += 2) mma_plane2<T, M::kSplit ? 3 : 2, false>(acc[j], acc[j + 1], x, S, M::kPlane, kLdV, 8 * j, k0, lane);
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int r = 0; r < 2; ++r) {
                            const T* p = Own + (r0 + gq + 8 * r) * kLdK + m0 + 8 * j + 2 * t;
                            through[r] = fmaf(to_f<T>(p[0]), acc[j][2 * r], fmaf(to_f<T>(p[1]), acc[j][2 * r + 1], through[r]));
                            total[4 * s + j][2 * r] = fmaf(r ? wh : wl, acc[j][2 * r], total[4 * s + j][2 * r]);
                            total[4 * s + j][2 * r + 1] = fmaf(r ? wh : wl, acc[j][2 * r + 1], total[4 * s + j][2 * r + 1]);
                        }
                    for (int kb = has_dq ? 0 : w4; kb <= (has_dq ? w4 : 3); ++kb) {
                        const OpA<P> x = has_dq ? load_a<false>(s_a, kLdP, r0, 16 * kb, lane) : load_a<true>(s_a, kLdP, r0, 16 * kb, lane);
#pragma unroll
                        for (int u = 0; u < 4; u += 2) {
                            OpB<T> b0, b1;
                            load_b2<true>(b0, b1, Other, kLdK, m0 + 8 * u, 16 * kb, lane);
                            mma_plane_a<T>(total[4 * s + u], x, b0);
                            mma_plane_a<T>(total[4 * s + u + 1], x, b1);
                        }
                    }
                }
                if (has_dv) {
#pragma unroll
                    for (int k0 = 0; k0 < kSlab; k0 += 16) {
                        const OpA<T> x = load_a<false>(sk, kLdK, r0, m0 + k0, lane);
#pragma unroll
                        for (int j = 0; j < DV / 8; j += 2) mma_plane2<T, 1, true>(dv[j], dv[j + 1], x, s_out, M::kPlane, kLdV, 8 * j, k0, lane);
                    }
                }
                if constexpr (!M::kSplit) {
                    if (s + M::kStages < M::kSlabs) {
                        __syncthreads();
                        fetch_slab(s + M::kStages);
                    } else if constexpr (M::kStages == 2)
                        commit_copies();                   // keeps the count of groups behind a slab
                }
            }
        }
        if (has_dv) {
            const float vl = d.w[r0 + gq], vh = d.w[r0 + gq + 8];
#pragma unroll
            for (int j = 0; j < DV / 8; ++j) {
                dv[j][0] *= vl; dv[j][1] *= vl; dv[j][2] *= vh; dv[j][3] *= vh;
            }
            for (int kb = w4; kb < 4; ++kb) {
                const OpA<P> x = load_a<true>(s_w, kLdP, r0, 16 * kb, lane);
#pragma unroll
                for (int u = 0; u < DV / 8; u += 2) {
                    OpB<T> b0, b1;
                    load_b2<true>(b0, b1, sy, kLdV, 8 * u, 16 * kb, lane);
                    mma_plane_a<T>(dv[u], x, b0);
                    mma_plane_a<T>(dv[u + 1], x, b1);
                }
            }
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int row = r0 + gq + 8 * r;
                if (row >= rows) continue;
                T* to = (T*)a.dv_ + (((long long)b * a.L + first + row) * H + h) * a.dv;
#pragma unroll
                for (int j = 0; j < DV / 8; ++j) {
                    const int col = 8 * j + 2 * t;
                    const float y[2] = {dv[j][2 * r], dv[j][2 * r + 1]};
                    if (a.pairs_v && col + 1 < a.dv) Vec<T, 2>::store(to + col, y);
                    else {
                        if (col < a.dv) to[col] = from_f<T>(y[0]);
                        if (col + 1 < a.dv) to[col + 1] = from_f<T>(y[1]);
                    }
                }
            }
        }
        if (has_dq || has_dk) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                through[r] *= r ? wh : wl;
                through[r] += __shfl_xor_sync(0xffffffffu, through[r], 1);
                through[r] += __shfl_xor_sync(0xffffffffu, through[r], 2);
                if (t == 0) (has_dq ? into : from)[r0 + gq + 8 * r] = through[r];
            }
        }
#pragma unroll
        for (int off = 16; off; off >>= 1) both += __shfl_xor_sync(0xffffffffu, both, off);
        if (lane == 0) cross[warp] = both;
        __syncthreads();
        if (warp == 0) {
            // tokens 2 lane and 2 lane + 1: suffix sums of what reaches them from in front, prefix sums of what leaves them
            float x = 0.f, in[2], out[2];
            for (int i = 0; i < 4 * kGroups; ++i) x += cross[i];
            x *= d.total;
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const int i = 2 * lane + s;
                in[s] = into[i];
                out[s] = from[i];
                float pairs = 0.f;
                for (int p = 0; p < kGroups; ++p) pairs += row_sum[p * kChunk + i];
                for (int r = i / 16; r < 4; ++r) pairs -= col_sum[r * kChunk + i];
                in[s] += pairs;
            }
            float suffix = in[0] + in[1], prefix = out[0] + out[1];
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const float u = __shfl_down_sync(0xffffffffu, suffix, off), v = __shfl_up_sync(0xffffffffu, prefix, off);
                if (lane + off < 32) suffix += u;
                if (lane >= off) prefix += v;
            }
            const float after = __shfl_down_sync(0xffffffffu, suffix, 1), before = __shfl_up_sync(0xffffffffu, prefix, 1);
            const float s1 = in[1] + (lane < 31 ? after : 0.f), p0 = lane ? before : 0.f;
            const float y[2] = {x + s1 + in[0] + p0, x + s1 + p0 + out[0]};
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const int i = 2 * lane + s;
                // nothing crosses a reset; the pairs in front of it and behind it have cancelled to rounding only
                // (neighbouring sums may have been added up in other orders, one of them with a carry more)
                const bool reset = d.n[i] - (i ? d.n[i - 1] : 0.f) <= kFloor + 1.f;
                if (i < rows) a.dg[((long long)b * a.L + first + i) * H + h] = reset ? 0.f : y[s];
            }
        }
    }
    if (has_dq || has_dk) {
        T* const out = (T*)(has_dq ? a.dq : a.dk_);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int row = r0 + gq + 8 * r;
            if (row >= rows) continue;
            T* const to = out + (((long long)b * a.L + first + row) * a.G + grp) * a.dk;
#pragma unroll
            for (int s = 0; s < M::kSlabs; ++s)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int col = s * kSlab + 8 * j + 2 * t;
                    const float y[2] = {acc_all[4 * s + j][2 * r], acc_all[4 * s + j][2 * r + 1]};
                    if (a.pairs_k && col + 1 < a.dk) Vec<T, 2>::store(to + col, y);
                    else {
                        if (col < a.dk) to[col] = from_f<T>(y[0]);
                        if (col + 1 < a.dk) to[col + 1] = from_f<T>(y[1]);
                    }
                }
        }
    }
}

// ---- one token ---------------------------------------------------------------------------------------------------------
struct StepArgs {
    const void *q, *k, *v;
    const float* g;
    const float* state;
    float* state_out;
    void* o;                        // (B, H, dv)
    long long q_b, q_h, k_b, k_h, v_b, v_h, g_b, g_h, s_b, so_b;
    int H, rep, dk, dv;
    float scale;
};
constexpr int kStepThreads = 256, kMostRow = 128;

// A CTA has one head's state.  Threads stand on kVec neighbouring columns each and take every n-th row.
template <typename T, int kVec>
__global__ void __launch_bounds__(kStepThreads) la_step_kernel(const StepArgs a) {
    follow_previous();
    __shared__ float sq[kMostRow], sk[kMostRow];
    __shared__ __align__(16) float part[kStepThreads * kVec];
    const int tid = threadIdx.x, b = blockIdx.x / a.H, h = blockIdx.x % a.H;
    const T* q = (const T*)a.q + b * a.q_b + (h / a.rep) * a.q_h;
    const T* k = (const T*)a.k + b * a.k_b + (h / a.rep) * a.k_h;
    for (int i = tid; i < a.dk; i += kStepThreads) { sq[i] = a.scale * to_f<T>(q[i]); sk[i] = to_f<T>(k[i]); }
    const float keep = expf(a.g[b * a.g_b + h * a.g_h]);
    const int across = (a.dv + kVec - 1) / kVec, down = kStepThreads / across, col = tid % across, row0 = tid / across;
    const bool live = row0 < down;
    float v[kVec], o[kVec] = {};
#pragma unroll
    for (int i = 0; i < kVec; ++i) v[i] = to_f<T>(((const T*)a.v + b * a.v_b + h * a.v_h)[col * kVec + i]);
    __syncthreads();
    const long long first = (long long)h * a.dk * a.dv + col * kVec;
    const float* s = a.state + b * a.s_b + first;
    float* to = a.state_out + b * a.so_b + first;
    if (live) {
#pragma unroll 8
        for (int r = row0; r < a.dk; r += down) {
            float x[kVec];
            Vec<float, kVec>::load(s + (long long)r * a.dv, x);
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
                x[i] = fmaf(keep, x[i], sk[r] * v[i]);
                o[i] = fmaf(sq[r], x[i], o[i]);
            }
            Vec<float, kVec>::store(to + (long long)r * a.dv, x);
        }
    }
#pragma unroll
    for (int i = 0; i < kVec; ++i) part[tid * kVec + i] = o[i];
    __syncthreads();
    T* out = (T*)a.o + (long long)blockIdx.x * a.dv;
    for (int i = tid; i < a.dv; i += kStepThreads) {
        float x = 0.f;
        for (int r = 0; r < down; ++r) x += part[r * across * kVec + i];
        out[i] = from_f<T>(x);
    }
}

}  // namespace

}  // namespace ss2d

#include "linear_attention_tc.cuh"

namespace ss2d {

namespace {

// ---- host --------------------------------------------------------------------------------------------------------------
constexpr int kMostWidth = 128;

int check_common(const ss2d_linear_attention_params& p) {
    if (!p.q || !p.k || !p.v || !p.log_decay) return SS2D_EINVAL_NULL;
    if (!dtype_ok(p.dtype)) return SS2D_EINVAL_DTYPE;
    if (p.batch <= 0 || p.seqlen <= 0 || p.n_groups <= 0 || p.heads <= 0 || p.heads % p.n_groups || p.dk <= 0 || p.dv <= 0) return SS2D_EINVAL_SHAPE;
    if (p.dk > kMostWidth || p.dv > kMostWidth) return SS2D_ENOTSUP;
    // grids of (sequence, head, 256 elements of a state) and of (sequence, group, chunk)
    if (p.seqlen > 0x7fffffc0LL || p.batch > 0x7fffffffLL / 64 / p.heads || p.batch * p.n_groups > 0x7fffffffLL / ((p.seqlen + kChunk - 1) / kChunk)) return SS2D_ENOTSUP;
    for (int64_t s : {p.q_batch_stride, p.q_token_stride, p.q_head_stride, p.k_batch_stride, p.k_token_stride, p.k_head_stride, p.v_batch_stride,
                      p.v_token_stride, p.v_head_stride, p.decay_batch_stride, p.decay_token_stride, p.decay_head_stride})
        if (s < 0) return SS2D_EINVAL_STRIDE;
    const size_t e = dtype_size(p.dtype);
    if (!aligned_to(p.q, e) || !aligned_to(p.k, e) || !aligned_to(p.v, e) || !aligned_to(p.log_decay, 4)) return SS2D_EINVAL_ALIGN;
    return SS2D_OK;
}

Rows rows_of(const void* p, int64_t b, int64_t l, int64_t h, int dtype) {
    const int64_t per = 16 / (int64_t)dtype_size(dtype);
    return {p, b, l, h, aligned_to(p, 16) && b % per == 0 && l % per == 0 && h % per == 0};
}
long long chunks_of(const ss2d_linear_attention_params& p) { return (p.seqlen + kChunk - 1) / kChunk; }

// Columns of v of a walking CTA: 64, but 32 where derived operands in fp32 (all types but bf16) beside 128 rows of 64 columns of state would not stay in registers.  fp16, us with 64 / 32,
// forward, then a training step: 4 096 tokens of 16 heads of 128 x 128 175 / 163, 551 / 551; 16 x 784 of 24 heads of 128 x 64 283 / 254, 1 090 / 1 049, of 128 x 128 544 / 478, 2 030 / 2 028;
// 64 x 200 of 8 heads of 128 x 64 123 / 113, 453 / 446; 4 x 1 000 of 16 heads of 96 x 80 174 / 106, 478 / 371.
template <typename T, int DK> constexpr bool kWideSlices = std::is_same<T, __nv_bfloat16>::value || DK <= 64;
int slice_of(const ss2d_linear_attention_params& p) { return p.dv <= 32 || (p.dtype != SS2D_BF16 && p.dk > 64) ? 32 : 64; }

// Segments of a sequence: where sequences, heads and slices leave room on the chip, sequences are cut, and each segment's own state is gathered by a
// walk of its own first.  As many as are resident at once (two CTAs an SM with 128 rows of state, four with fewer): one more round of few CTAs would take as
// long as all others.  us with 1 / 2 / 3 / 4 / 8 / 9 / 12 segments (the one that the rule takes in brackets), bf16: 16 385 tokens of 16 heads of 128 x 128, forward 1 311 / 1 000 / 675 / 515 /
// 343 / 306 / 433 (9); 2 x 4 096 tokens, training 859 / 755 / 703 / 607 / 622 / 622 / 648 (4); 16 x 3 136 tokens of 12 heads of 64 x 32, training 566 / 570 / 517 / 540 / 531 / 529 / 531 (3);
// 16 x 784 tokens of 24 heads, fp16, forward 80 / 122 / 120 / 116 / 118 / 118 / 118 (1).
long long room_of(const ss2d_linear_attention_params& p) {
    return 148 * (p.dk > 64 ? 2 : 4) / (p.batch * p.heads * ((p.dv + slice_of(p) - 1) / slice_of(p)));
}
int segments_of(const ss2d_linear_attention_params& p) {
    const long long chunks = chunks_of(p), room = room_of(p);
    if (room < 2 || chunks < 8) return 1;
    const long long seg = room < chunks / 2 ? room : chunks / 2, per = (chunks + seg - 1) / seg;
    return (int)((chunks + per - 1) / per);
}
long long segment_bytes(const ss2d_linear_attention_params& p) {
    const long long seg = segments_of(p);
    return seg == 1 ? 0 : 4 * p.batch * p.heads * seg * (p.dk * p.dv + 4);
}
long long states_bytes(const ss2d_linear_attention_params& p) { return 4 * p.batch * p.heads * chunks_of(p) * p.dk * state_row((int)p.dv); }

template <typename F> int for_type(int dtype, F&& f) {
    switch (dtype) {
        case SS2D_F32: return f((float)0);
        case SS2D_F16: return f(__half());
        default: return f(__nv_bfloat16());
    }
}
template <typename F> int for_dk(int64_t dk, F&& f) {
    if (dk <= 32) return f(std::integral_constant<int, 32>());
    if (dk <= 64) return f(std::integral_constant<int, 64>());
    return f(std::integral_constant<int, 128>());
}

template <typename T, int DK, int DVT, bool kOut, bool kBack> int launch_walk(const WalkArgs& a, long long bh, cudaStream_t st) {
    auto kern = la_walk_kernel<T, DK, DVT, kOut, kBack>;
    const size_t smem = WalkSmem<T, DK, DVT>::bytes(kOut);
    if (const int rc = allow_dynamic_smem(kern, smem)) return rc;
    launch(kern, dim3((unsigned)(bh * ((a.dv + DVT - 1) / DVT)), a.segments), 128, smem, st, a);
    count_launch();
    return check_launch();
}

// One pass over the sequences: gathers the segments' states first where there are several.  `first` and `last`: states before and behind the whole walk
template <typename T, int DK, int DVT, bool kOut, bool kBack>
int walk(WalkArgs a, const float* first, float* last, void* workspace, long long bh, cudaStream_t st) {
    const int seg = a.segments;
    if (seg == 1) {
        a.per_segment = a.chunks;
        a.start = first; a.end = last;
        return launch_walk<T, DK, DVT, kOut, kBack>(a, bh, st);
    }
    float* part = (float*)workspace;
    float* decay = part + bh * seg * a.dk * a.dv;
    a.per_segment = (a.chunks + seg - 1) / seg;
    WalkArgs g = a;
    if constexpr (kOut) g.q = Rows{};
    g.states = nullptr; g.start = nullptr; g.end = part; g.end_decay = decay;
    if (const int rc = launch_walk<T, DK, DVT, false, kBack>(g, bh, st)) return rc;
    JoinArgs j = {first, part, decay, last, (long long)a.dk * a.dv, seg, kBack};
    launch(la_join_kernel, (unsigned)(bh * ((j.size + 255) / 256)), 256, 0, st, j);
    count_launch();
    if (const int rc = check_launch()) return rc;
    a.start = part; a.end = nullptr;
    return launch_walk<T, DK, DVT, kOut, kBack>(a, bh, st);
}

WalkArgs walk_args(const ss2d_linear_attention_params& p) {
    WalkArgs a = {};
    a.g = (const float*)p.log_decay;
    a.g_b = p.decay_batch_stride; a.g_l = p.decay_token_stride; a.g_h = p.decay_head_stride;
    a.H = (int)p.heads; a.rep = (int)(p.heads / p.n_groups); a.L = (int)p.seqlen; a.dk = (int)p.dk; a.dv = (int)p.dv;
    a.chunks = (int)chunks_of(p); a.segments = segments_of(p); a.scale = p.scale;
    a.pairs = p.dv % 2 == 0;
    return a;
}

// ---- long bf16 sequences on the tensor cores of linear_attention_tc.cuh ---------------------------------------------------
// By the shape; the workspace follows it.  The walk moves less and is one launch where it need not be cut; these kernels win where a walk would be cut (room for
// twice its CTAs), and with wide heads from 8 chunks on.  us of the walk / these, forward, then a training step: 4 096 tokens of 16 heads of 128 x 128 97 / 48, 323 / 254,
// of 64 x 64 43 / 33, 124 / 111, of 64 x 32 32 / 32, 93 / 95; 16 x 3 136 of 12 heads of 128 x 128 624 / 341, 2 345 / 2 095, of 128 x 64 322 / 257, 1 480 / 1 401, of 64 x 64
// 224 / 177, 785 / 754, of 64 x 32 142 / 159, 572 / 596; 16 x 784 of 24 heads of 128 x 64 174 / 152, 779 / 752, of 64 x 64 119 / 108, 388 / 412; 64 x 200 of 8 heads of 128 x 128
// 116 / 101, 462 / 474, of 128 x 64 60 / 71, 296 / 311.
constexpr int kLongChunks = 4;
bool tc_shape(const ss2d_linear_attention_params& p) {
    const long long chunks = chunks_of(p);
    if (p.dtype != SS2D_BF16 || p.dk % 8 || p.dv % 8 || chunks < kLongChunks || p.batch * p.heads > 0x7fffffffLL / chunks) return false;
    if (p.dk > 64 || p.dv > 64) return room_of(p) >= 2 || chunks >= 8 || (p.dk > 64 && p.dv > 64);
    return p.dk > 32 && p.dv > 32 && room_of(p) >= 2;
}
// by strides and alignment: rows that TMA can read
bool tc_rows(const Rows& r, long long B, long long L, long long H) {
    return r.vec && (B == 1 || r.b > 0) && (L == 1 || r.l > 0) && (H == 1 || r.h > 0) && r.b < 1LL << 38 && r.l < 1LL << 38 && r.h < 1LL << 38;
}
struct TcPlan { long long chunks, decay, added, states, total; };
TcPlan tc_plan(const ss2d_linear_attention_params& p, bool train, bool back) {
    TcPlan t = {};
    if (!tc_shape(p)) return t;
    auto up = [](long long n) { return (n + 255) / 256 * 256; };
    const long long bh = p.batch * p.heads, size = p.dk * state_row((int)p.dv);
    t.chunks = train ? chunks_of(p) : (p.seqlen + lat::kTile - 1) / lat::kTile;
    t.decay = up(4 * bh * t.chunks);
    t.added = up(4 * bh * t.chunks * size);
    t.states = back ? 0 : up(2 * bh * t.chunks * size);         // in bf16, for the outputs; the gradients read those in fp32
    t.total = t.decay + t.added + t.states;
    return t;
}
template <typename F> int for_tc(const ss2d_linear_attention_params& p, F&& f) {
    auto with = [&](auto dk) {
        return p.dv <= 64 ? f(dk, std::integral_constant<int, 64>()) : f(dk, std::integral_constant<int, 128>());
    };
    return p.dk <= 64 ? with(std::integral_constant<int, 64>()) : with(std::integral_constant<int, 128>());
}
// the states in front of all chunks (backwards: the gradients behind them), `k` and `v` as in WalkArgs
template <bool kBack> int tc_states(const ss2d_linear_attention_params& p, const WalkArgs& w, const TcPlan& plan, bool train, const float* first, float* last, float* states,
                                    __nv_bfloat16* plane, char* ws, cudaStream_t st) {
    float* const added = (float*)(ws + plan.decay);
    lat::GatherArgs g = {w.g, w.g_b, w.g_l, w.g_h, (float*)ws, w.H, w.rep, w.L, w.dk, w.dv, (int)plan.chunks, w.scale, nullptr};
    const int rc = for_tc(p, [&](auto dk, auto dv) {
        constexpr int DK = decltype(dk)::value, DV = decltype(dv)::value;
        if constexpr (!kBack)
            if (!train) return lat::gather<DK, DV, lat::kTile, false>(w.k, w.v, added, p.batch, p.n_groups, g, st);
        return lat::gather<DK, DV, kChunk, kBack>(w.k, w.v, added, p.batch, p.n_groups, g, st);
    });
    if (rc != SS2D_OK) return rc;
    return lat::spread({added, g.decay, first, last, states, plane, g.chunks, w.dk, w.dv, state_row(w.dv), kBack}, p.batch * p.heads, st);
}
int tc_forward(const ss2d_linear_attention_params& p, const WalkArgs& w, cudaStream_t st) {
    const bool train = p.chunk_states != nullptr;
    const TcPlan plan = tc_plan(p, train, false);
    char* const ws = (char*)p.workspace;
    __nv_bfloat16* const plane = (__nv_bfloat16*)(ws + plan.decay + plan.added);
    if (const int rc = tc_states<false>(p, w, plan, train, (const float*)p.initial_state, (float*)p.final_state, (float*)p.chunk_states, plane, ws, st)) return rc;
    lat::OutArgs o = {w.g, w.g_b, w.g_l, w.g_h, w.H, w.rep, w.L, w.dk, w.dv, (int)((p.seqlen + lat::kTile - 1) / lat::kTile), (int)plan.chunks,
                      train ? lat::kTile / kChunk : 1, w.scale, nullptr};
    const Rows out = rows_of(p.out, p.seqlen * p.heads * p.dv, p.heads * p.dv, p.dv, p.dtype);
    return for_tc(p, [&](auto dk, auto dv) {
        return lat::outputs<decltype(dk)::value, decltype(dv)::value>(w.q, w.k, w.v, out, plane, 2LL * w.dk * state_row(w.dv), p.batch, p.n_groups, o, st);
    });
}
long long fwd_workspace(const ss2d_linear_attention_params& p) {
    const long long walk = segment_bytes(p), tc = tc_plan(p, p.chunk_states != nullptr, false).total;
    return walk > tc ? walk : tc;
}

}  // namespace

long long linear_attention_states_bytes(const ss2d_linear_attention_params* p) {
    if (!p || check_common(*p) != SS2D_OK) return -1;
    return states_bytes(*p);
}

long long linear_attention_workspace_bytes(const ss2d_linear_attention_params* p) {
    if (!p || check_common(*p) != SS2D_OK) return -1;
    return fwd_workspace(*p);
}

int linear_attention_fwd(const ss2d_linear_attention_params* p, cudaStream_t st) {
    if (!p) return SS2D_EINVAL_NULL;
    if (const int rc = check_common(*p)) return rc;
    if (!p->out) return SS2D_EINVAL_NULL;
    if (!aligned_to(p->out, 2 * dtype_size(p->dtype)) || !aligned_to(p->initial_state, 4) || !aligned_to(p->final_state, 8) || !aligned_to(p->chunk_states, 16))
        return SS2D_EINVAL_ALIGN;
    const long long need = fwd_workspace(*p), bh = p->batch * p->heads;
    if (need && (!p->workspace || p->workspace_bytes < need || !aligned_to(p->workspace, 16))) return SS2D_EWORKSPACE;
    WalkArgs a = walk_args(*p);
    a.q = rows_of(p->q, p->q_batch_stride, p->q_token_stride, p->q_head_stride, p->dtype);
    a.k = rows_of(p->k, p->k_batch_stride, p->k_token_stride, p->k_head_stride, p->dtype);
    a.v = rows_of(p->v, p->v_batch_stride, p->v_token_stride, p->v_head_stride, p->dtype);
    a.o = p->out;
    a.states = (float*)p->chunk_states;
    if (tc_shape(*p) && aligned_to(p->out, 16) && tc_rows(a.q, p->batch, p->seqlen, p->n_groups) && tc_rows(a.k, p->batch, p->seqlen, p->n_groups) &&
        tc_rows(a.v, p->batch, p->seqlen, p->heads))
        return tc_forward(*p, a, st);
    return for_type(p->dtype, [&](auto z) {
        return for_dk(p->dk, [&](auto n) {
            using T = decltype(z);
            constexpr int DK = decltype(n)::value;
            const float* first = (const float*)p->initial_state;
            float* last = (float*)p->final_state;
            if constexpr (kWideSlices<T, DK>)
                if (slice_of(*p) == 64) return walk<T, DK, 64, true, false>(a, first, last, p->workspace, bh, st);
            return walk<T, DK, 32, true, false>(a, first, last, p->workspace, bh, st);
        });
    });
}

namespace {
struct BwdPlan { long long segments, dstates, total; };
BwdPlan bwd_plan(const ss2d_linear_attention_params& p) {
    BwdPlan b = {};
    const long long walk = (segment_bytes(p) + 255) / 256 * 256, tc = tc_plan(p, true, true).total;
    b.segments = walk > tc ? walk : tc;
    b.dstates = states_bytes(p);
    b.total = b.segments + b.dstates;
    return b;
}
template <typename T, int DK, int DV> int launch_grad(const GradArgs& a, long long groups, cudaStream_t st) {
    auto kern = la_grad_kernel<T, DK, DV>;
    constexpr size_t smem = GradShape<T, DK, DV>::kBytes;
    if (const int rc = allow_dynamic_smem(kern, smem)) return rc;
    launch(kern, (unsigned)(groups * a.chunks), GradShape<T, DK, DV>::kThreads, smem, st, a);
    count_launch();
    return check_launch();
}
}  // namespace

long long linear_attention_bwd_workspace_bytes(const ss2d_linear_attention_bwd_params* p) {
    if (!p || check_common(p->fwd) != SS2D_OK) return -1;
    return bwd_plan(p->fwd).total;
}

int linear_attention_bwd(const ss2d_linear_attention_bwd_params* p, cudaStream_t st) {
    if (!p) return SS2D_EINVAL_NULL;
    const ss2d_linear_attention_params& f = p->fwd;
    if (const int rc = check_common(f)) return rc;
    if (!f.chunk_states || !p->dout || !p->dq || !p->dk || !p->dv || !p->dlog_decay) return SS2D_EINVAL_NULL;
    if (p->dout_batch_stride < 0 || p->dout_token_stride < 0 || p->dout_head_stride < 0) return SS2D_EINVAL_STRIDE;
    const size_t e = dtype_size(f.dtype);
    if (!aligned_to(p->dout, e) || !aligned_to(p->dq, 2 * e) || !aligned_to(p->dk, 2 * e) || !aligned_to(p->dv, 2 * e) || !aligned_to(p->dlog_decay, 4) ||
        !aligned_to(f.chunk_states, 16) || !aligned_to(p->dfinal_state, 4) || !aligned_to(p->dinitial_state, 8))
        return SS2D_EINVAL_ALIGN;
    const BwdPlan plan = bwd_plan(f);
    if (!p->workspace || p->workspace_bytes < plan.total || !aligned_to(p->workspace, 16)) return SS2D_EWORKSPACE;
    const long long bh = f.batch * f.heads;
    char* ws = (char*)p->workspace;
    float* dstates = (float*)(ws + plan.segments);
    WalkArgs w = walk_args(f);
    w.k = rows_of(f.q, f.q_batch_stride, f.q_token_stride, f.q_head_stride, f.dtype);
    w.v = rows_of(p->dout, p->dout_batch_stride, p->dout_token_stride, p->dout_head_stride, f.dtype);
    w.states = dstates;
    GradArgs a = {};
    a.q = w.k; a.dy = w.v;
    a.k = rows_of(f.k, f.k_batch_stride, f.k_token_stride, f.k_head_stride, f.dtype);
    a.v = rows_of(f.v, f.v_batch_stride, f.v_token_stride, f.v_head_stride, f.dtype);
    a.g = w.g; a.g_b = w.g_b; a.g_l = w.g_l; a.g_h = w.g_h;
    a.states = (const float*)f.chunk_states; a.dstates = dstates;
    a.dq = p->dq; a.dk_ = p->dk; a.dv_ = p->dv; a.dg = (float*)p->dlog_decay;
    a.G = (int)f.n_groups; a.rep = w.rep; a.L = w.L; a.dk = w.dk; a.dv = w.dv; a.chunks = w.chunks; a.scale = f.scale;
    a.pairs_k = a.dk % 2 == 0; a.pairs_v = a.dv % 2 == 0;
    const float* first = (const float*)p->dfinal_state;
    float* last = (float*)p->dinitial_state;
    const bool tc = tc_shape(f) && tc_rows(w.k, f.batch, f.seqlen, f.n_groups) && tc_rows(w.v, f.batch, f.seqlen, f.heads);
    if (tc)
        if (const int rc = tc_states<true>(f, w, tc_plan(f, true, true), true, first, last, dstates, nullptr, ws, st)) return rc;
    return for_type(f.dtype, [&](auto z) {
        using T = decltype(z);
        return for_dk(f.dk, [&](auto n) {
            constexpr int DK = decltype(n)::value;
            int rc = SS2D_OK;
            bool wide = false;
            if constexpr (kWideSlices<T, DK>) {
                wide = slice_of(f) == 64;
                if (wide && !tc) rc = walk<T, DK, 64, false, true>(w, first, last, ws, bh, st);
            }
            if (!wide && !tc) rc = walk<T, DK, 32, false, true>(w, first, last, ws, bh, st);
            if (rc != SS2D_OK) return rc;
            const long long groups = f.batch * f.n_groups;
            return f.dv <= 32 ? launch_grad<T, DK, 32>(a, groups, st) : f.dv <= 64 ? launch_grad<T, DK, 64>(a, groups, st) : launch_grad<T, DK, 128>(a, groups, st);
        });
    });
}

int linear_attention_step(const ss2d_linear_attention_step_params* p, cudaStream_t st) {
    if (!p || !p->q || !p->k || !p->v || !p->log_decay || !p->state || !p->state_out || !p->out) return SS2D_EINVAL_NULL;
    if (!dtype_ok(p->dtype)) return SS2D_EINVAL_DTYPE;
    if (p->batch <= 0 || p->n_groups <= 0 || p->heads <= 0 || p->heads % p->n_groups || p->dk <= 0 || p->dv <= 0) return SS2D_EINVAL_SHAPE;
    if (p->dk > kMostWidth || p->dv > kMostWidth || p->batch > 0x7fffffffLL / p->heads) return SS2D_ENOTSUP;
    const int64_t size = p->heads * p->dk * p->dv;
    for (int64_t s : {p->q_batch_stride, p->q_head_stride, p->k_batch_stride, p->k_head_stride, p->v_batch_stride, p->v_head_stride,
                      p->decay_batch_stride, p->decay_head_stride})
        if (s < 0) return SS2D_EINVAL_STRIDE;
    if (p->state_batch_stride < size || p->state_out_batch_stride < size) return SS2D_EINVAL_STRIDE;
    const size_t e = dtype_size(p->dtype);
    if (!aligned_to(p->q, e) || !aligned_to(p->k, e) || !aligned_to(p->v, e) || !aligned_to(p->out, e) || !aligned_to(p->log_decay, 4) ||
        !aligned_to(p->state, 4) || !aligned_to(p->state_out, 4))
        return SS2D_EINVAL_ALIGN;
    StepArgs a = {p->q, p->k, p->v, (const float*)p->log_decay, (const float*)p->state, (float*)p->state_out, p->out,
                  p->q_batch_stride, p->q_head_stride, p->k_batch_stride, p->k_head_stride, p->v_batch_stride, p->v_head_stride,
                  p->decay_batch_stride, p->decay_head_stride, p->state_batch_stride, p->state_out_batch_stride,
                  (int)p->heads, (int)(p->heads / p->n_groups), (int)p->dk, (int)p->dv, p->scale};
    const bool vec = p->dv % 4 == 0 && p->state_batch_stride % 4 == 0 && p->state_out_batch_stride % 4 == 0 && aligned_to(p->state, 16) && aligned_to(p->state_out, 16);
    return for_type(p->dtype, [&](auto z) {
        using T = decltype(z);
        const unsigned grid = (unsigned)(p->batch * p->heads);
        if (vec) launch(la_step_kernel<T, 4>, grid, kStepThreads, 0, st, a);
        else launch(la_step_kernel<T, 1>, grid, kStepThreads, 0, st, a);
        count_launch();
        return check_launch();
    });
}

}  // namespace ss2d
