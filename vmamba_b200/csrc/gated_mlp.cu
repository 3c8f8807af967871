// Gated feed-forward block:  h = (x Wv^T + bv) * act(x Wg^T + bg),  y = h W2^T + b2, and its backward pass
//   dh = dy W2;  dv = dh act(g);  dg = dh v act'(g);  dx = [dv dg] W1;  dW1 = [dv dg]^T x;  dW2 = dy^T h;  db1, db2 the column sums.
// The two projections run as one product whose tile holds the same columns of value and gate, so that activation and product happen on its
// accumulators; in the backward pass dh never leaves them either.  Nothing but x and h is kept for it: v and g are computed again, in fp32.
#include "gated_epilogue.cuh"
#include "mma_tiles.cuh"
#include "product_tc05.cuh"

namespace ss2d {

namespace {

using namespace mt;

// ---- products of any types, strides and sizes ---------------------------------------------------------------------------
// C (M x N) = A (M x K) . B (N x K)^T, rows of K (or of M / N, kAK / kBK: "stored by K") contiguous, lda / ldb elements apart.
struct ProductArgs {
    const void *a, *b;
    long long lda, ldb;
    int M, N, K;
    bool veca, vecb;
    int second;             // EPI_GATE: rows of B between a column's value and its gate
    int per_split;          // contraction elements of a split (a multiple of the step)
    EpiArgs e;
};
// fp32 and what TMA cannot read.  1 001 tokens of 192 channels, 768 hidden, fp32: 26 us for value and gate, of which three tf32 products for each would take 10 at 512
// multiplications a cycle and SM.  Taking operands apart once for all their products and reading them in pairs changed nothing (25 us).
constexpr int kTile = 64, kStep = 32, kRing = 3;

template <typename T, bool kAK, bool kBK, int EPI> struct ProductSmem {
    static constexpr int kLdA = kAK ? kTile + 8 : kStep + 8, kLdB = kBK ? kTile + 8 : kStep + 8;
    static constexpr int kA = (kAK ? kStep : kTile) * kLdA, kB = (kBK ? kStep : kTile) * kLdB;
    static constexpr int kNB = EPI == EPI_GATE ? 2 : 1;
    static constexpr int kStage = kA + kNB * kB;
    static constexpr size_t kBytes = (size_t)kRing * kStage * sizeof(T);
};

// Four warps of 32 x 32.  A ring of three stages keeps two steps of loads in flight.
template <typename T, bool kAK, bool kBK, int EPI, int ACT>
__global__ void __launch_bounds__(128) product_kernel(const ProductArgs p) {
    follow_previous();
    using S = ProductSmem<T, kAK, kBK, EPI>;
    extern __shared__ __align__(16) unsigned char smem[];
    T* const ring = reinterpret_cast<T*>(smem);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int m0 = blockIdx.y * kTile, n0 = blockIdx.x * kTile, wm = (warp >> 1) * 32, wn = (warp & 1) * 32;
    const int k_begin = blockIdx.z * p.per_split, k_end = min(p.K, k_begin + p.per_split);
    const int steps = (k_end - k_begin + kStep - 1) / kStep;
    auto fetch = [&](int i) {
        if (i < steps) {
            T* s = ring + (i % kRing) * S::kStage;
            const int k = k_begin + i * kStep;
            const T *a = (const T*)p.a, *b = (const T*)p.b;
            if constexpr (kAK) fetch_rows<T, kStep, kTile>(s, S::kLdA, a + (long long)k * p.lda + m0, p.lda, k_end - k, p.M - m0, p.veca, tid, 128);
            else fetch_rows<T, kTile, kStep>(s, S::kLdA, a + (long long)m0 * p.lda + k, p.lda, p.M - m0, k_end - k, p.veca, tid, 128);
#pragma unroll
            for (int j = 0; j < S::kNB; ++j) {
                T* to = s + S::kA + j * S::kB;
                if constexpr (kBK) fetch_rows<T, kStep, kTile>(to, S::kLdB, b + (long long)k * p.ldb + n0, p.ldb, k_end - k, p.N - n0, p.vecb, tid, 128);
                else fetch_rows<T, kTile, kStep>(to, S::kLdB, b + (long long)(n0 + j * p.second) * p.ldb + k, p.ldb, p.N - n0, k_end - k, p.vecb, tid, 128);
            }
        }
        commit_copies();
    };
    float acc[S::kNB][2][4][4] = {};
    fetch(0);
    fetch(1);
    for (int i = 0; i < steps; ++i) {
        wait_copies<1>();
        __syncthreads();
        fetch(i + 2);
        const T* s = ring + (i % kRing) * S::kStage;
        // Tensor cores cut their sums off instead of rounding them, always towards zero: over hundreds of steps that adds up in fp32 results.  A
        // step's products are summed on their own and added with ordinary additions there.
        float now[S::kNB][2][4][4] = {};
        auto& to = [&]() -> auto& { if constexpr (sizeof(T) == 4) return now; else return acc; }();
#pragma unroll
        for (int k0 = 0; k0 < kStep; k0 += 16) {
            OpA<T> a[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) a[u] = load_a<kAK>(s, S::kLdA, wm + 16 * u, k0, lane);
#pragma unroll
            for (int j = 0; j < S::kNB; ++j)
#pragma unroll
                for (int n = 0; n < 4; n += 2) {
                    OpB<T> b0, b1;
                    load_b2<kBK>(b0, b1, s + S::kA + j * S::kB, S::kLdB, wn + 8 * n, k0, lane);
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        mma_exact<false>(to[j][u][n], a[u], b0);
                        mma_exact<false>(to[j][u][n + 1], a[u], b1);
                    }
                }
        }
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int j = 0; j < S::kNB * 32; ++j) (&acc[0][0][0][0])[j] += (&now[0][0][0][0])[j];
        }
    }
    wait_copies();
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const long long m = m0 + wm + 16 * u + 8 * r + (lane >> 2);
            if (m >= p.M) continue;
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const float x[2] = {acc[0][u][n][2 * r], acc[0][u][n][2 * r + 1]};
                const float y[2] = {acc[S::kNB - 1][u][n][2 * r], acc[S::kNB - 1][u][n][2 * r + 1]};
                finish_pair<T, EPI, ACT>(p.e, m, n0 + wn + 8 * n + 2 * (lane & 3), p.N, x, y, (long long)blockIdx.z * p.M + m);
            }
        }
}

// ---- few tokens ---------------------------------------------------------------------------------------------------------
// Up to 16 tokens of 16-bit types: the weights' way from memory is the whole time, and every SM has to take part in it.  A CTA has kRows rows of the weights (of value and
// gate alike), its eight warps every eighth 32 elements of them, straight from memory into the A operand of mma.sync: a lane reads 16 bytes, 8 contraction elements in a row,
// and the products take them in that order (the tokens' elements come the same way).  The warps' sums meet in shared memory.  us of both launches in a
// graph, eight sets of weights in turn, with 1 / 8 / 16 tokens, and of the tensor-core kernels with 33: 768 channels and 2 048 hidden 9.2 / 9.1 / 11.9, 16.1; 384 and 1 536 5.5 / 5.9 / 8.9, 14.1;
// 1 024 and 4 096, more than L2 holds, 18 / 19 / 24, 19.
constexpr int kFew = 16;
struct FewArgs {
    const void *x, *w, *bias;
    void* out;
    long long ldx, second;      // second: rows between value and gate
    int M, N, K;
};
template <typename T, int kTiles, int kRows, int EPI, int ACT>
__global__ void __launch_bounds__(256) few_tokens_kernel(const FewArgs a) {
    follow_previous();
    constexpr int kMats = EPI == EPI_GATE ? 2 : 1, kBlocks = kRows / 8;
    __shared__ float sums[8][kMats][kTiles][kRows][9];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3, n0 = blockIdx.x * kRows;
    float acc[kMats][kTiles][4] = {};
    const T *const x = (const T*)a.x, *const w = (const T*)a.w;
    constexpr int kAhead = 16 / (kMats * kBlocks);          // 16 loads of weights on their way
#pragma unroll kAhead
    for (int k = warp * 32 + 8 * t; k < (a.K + 31) / 32 * 32; k += 256) {
        const uint4 none = make_uint4(0, 0, 0, 0);
        uint4 wr[kMats][2], xr[kTiles];
#pragma unroll
        for (int m = 0; m < kMats; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int row = n0 + g + 8 * h;
                wr[m][h] = h < kBlocks && k < a.K && row < a.N ? *reinterpret_cast<const uint4*>(w + (row + m * a.second) * a.K + k) : none;
            }
#pragma unroll
        for (int i = 0; i < kTiles; ++i)
            xr[i] = k < a.K && 8 * i + g < a.M ? *reinterpret_cast<const uint4*>(x + (8 * i + g) * a.ldx + k) : none;
#pragma unroll
        for (int m = 0; m < kMats; ++m) {
            const uint32_t lo[4] = {wr[m][0].x, wr[m][1].x, wr[m][0].y, wr[m][1].y}, hi[4] = {wr[m][0].z, wr[m][1].z, wr[m][0].w, wr[m][1].w};
#pragma unroll
            for (int i = 0; i < kTiles; ++i) {
                const uint32_t b0[2] = {xr[i].x, xr[i].y}, b1[2] = {xr[i].z, xr[i].w};
                MmaK16<T>::run(acc[m][i], lo, b0);
                MmaK16<T>::run(acc[m][i], hi, b1);
            }
        }
    }
#pragma unroll
    for (int m = 0; m < kMats; ++m)
#pragma unroll
        for (int i = 0; i < kTiles; ++i)
#pragma unroll
            for (int j = 0; j < 2 * kBlocks; ++j) sums[warp][m][i][g + 8 * (j >> 1)][2 * t + (j & 1)] = acc[m][i][j];
    __syncthreads();
    for (int i = tid; i < kRows * 8 * kTiles; i += 256) {
        const int row = i % kRows, token = i / kRows, n = n0 + row;
        if (n >= a.N || token >= a.M) continue;
        float y[kMats];
#pragma unroll
        for (int m = 0; m < kMats; ++m) {
            y[m] = a.bias ? to_f<T>(((const T*)a.bias)[n + m * a.second]) : 0.f;
            for (int v = 0; v < 8; ++v) y[m] += sums[v][m][token / 8][row][token % 8];
        }
        if constexpr (EPI == EPI_GATE) y[0] *= gate_act<ACT>(y[1]);
        ((T*)a.out)[(long long)token * a.N + n] = from_f<T>(y[0]);
    }
}

// ---- sums ---------------------------------------------------------------------------------------------------------------
// Column sums of two (rows, cols) matrices (the second may have none) over spans of rows, fp32: part[span][cols of both].  A warp has 32 kVec columns, eight warps
// every eighth row.
constexpr int kSpan = 128;
struct SumArgs {
    const void* a[2];
    long long ld[2], rows;
    int cols[2], blocks;        // CTAs of the first matrix
    float* part;
    void* out[2];
    int spans;
};
template <typename T, int kVec> __global__ void __launch_bounds__(256) column_sums_kernel(const SumArgs s) {
    follow_previous();
    __shared__ __align__(16) float sums[8][32 * kVec];
    const int which = (int)blockIdx.x >= s.blocks, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int c0 = ((int)blockIdx.x - which * s.blocks) * 32 * kVec, c = c0 + lane * kVec, cols = s.cols[which];
    const T* const a = (const T*)s.a[which];
    const long long ld = s.ld[which], r0 = (long long)blockIdx.y * kSpan, r1 = r0 + kSpan < s.rows ? r0 + kSpan : s.rows;
    float x[kVec] = {};
    if (c < cols) {
#pragma unroll 8
        for (long long r = r0 + warp; r < r1; r += 8) {
            float y[kVec];
            Vec<T, kVec>::load(a + r * ld + c, y);
#pragma unroll
            for (int i = 0; i < kVec; ++i) x[i] += y[i];
        }
    }
#pragma unroll
    for (int i = 0; i < kVec; ++i) sums[warp][lane * kVec + i] = x[i];
    __syncthreads();
    for (int i = threadIdx.x; i < 32 * kVec && c0 + i < cols; i += 256) {
        float y = 0.f;
        for (int w = 0; w < 8; ++w) y += sums[w][i];
        s.part[(long long)blockIdx.y * (s.cols[0] + s.cols[1]) + which * s.cols[0] + c0 + i] = y;
    }
}
template <typename T> __global__ void __launch_bounds__(256) add_columns_kernel(const SumArgs s) {
    follow_previous();
    const int i = blockIdx.x * 256 + threadIdx.x, n = s.cols[0] + s.cols[1];
    if (i >= n) return;
    float x = 0.f;
#pragma unroll 8
    for (int p = 0; p < s.spans; ++p) x += s.part[(long long)p * n + i];
    const int which = i >= s.cols[0];
    ((T*)s.out[which])[i - which * s.cols[0]] = from_f<T>(x);
}
// out[i] = sum over parts, in order
// (+ bias of the column, rows of `cols`)
template <typename T, int kVec> __global__ void __launch_bounds__(256) add_parts_kernel(const float* part, T* out, long long n, int parts, const T* bias, int cols) {
    follow_previous();
    const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * kVec;
    if (i >= n) return;
    float x[kVec] = {};
    if (bias) Vec<T, kVec>::load(bias + i % cols, x);
#pragma unroll 4
    for (int p = 0; p < parts; ++p) {
        float y[kVec];
        Vec<float, kVec>::load(part + p * n + i, y);
#pragma unroll
        for (int j = 0; j < kVec; ++j) x[j] += y[j];
    }
    Vec<T, kVec>::store(out + i, x);
}

// ---- host ---------------------------------------------------------------------------------------------------------------
template <typename T, bool kAK, bool kBK, int EPI, int ACT> int launch_product(const ProductArgs& p, int splits, cudaStream_t st) {
    auto kern = product_kernel<T, kAK, kBK, EPI, ACT>;
    const size_t smem = ProductSmem<T, kAK, kBK, EPI>::kBytes;
    if (const int rc = allow_dynamic_smem(kern, smem)) return rc;
    launch(kern, dim3((p.N + kTile - 1) / kTile, (p.M + kTile - 1) / kTile, splits), 128, smem, st, p);
    count_launch();
    return check_launch();
}
template <typename T> bool vec_rows(const void* p, long long ld) { return aligned_to(p, 16) && ld % (16 / (long long)sizeof(T)) == 0; }
template <typename T> ProductArgs product_args(const void* a, long long lda, const void* b, long long ldb, long long M, long long N, long long K) {
    ProductArgs p = {};
    p.a = a; p.b = b; p.lda = lda; p.ldb = ldb; p.M = (int)M; p.N = (int)N; p.K = (int)K;
    p.veca = vec_rows<T>(a, lda); p.vecb = vec_rows<T>(b, ldb);
    p.per_split = (p.K + kStep - 1) / kStep * kStep;
    return p;
}
// Splits of a contraction whose result has few tiles: enough for two CTAs an SM, each with 4 steps at least
int splits_of(long long M, long long N, long long K) {
    const long long tiles = ((M + kTile - 1) / kTile) * ((N + kTile - 1) / kTile), steps = (K + kStep - 1) / kStep;
    long long s = (2 * 148 + tiles - 1) / tiles;
    if (s > steps / 4) s = steps / 4;
    return s < 1 ? 1 : s > 64 ? 64 : (int)s;
}
template <typename T> int add_parts(const float* part, void* out, long long n, int parts, const void* bias, long long cols, cudaStream_t st) {
    if (cols % 4 == 0 && n % 4 == 0 && aligned_to(out, 4 * sizeof(T)) && aligned_to(bias, 4 * sizeof(T)))
        launch(add_parts_kernel<T, 4>, (unsigned)((n / 4 + 255) / 256), 256, 0, st, part, (T*)out, n, parts, (const T*)bias, (int)cols);
    else launch(add_parts_kernel<T, 1>, (unsigned)((n + 255) / 256), 256, 0, st, part, (T*)out, n, parts, (const T*)bias, (int)cols);
    count_launch();
    return check_launch();
}
// out (M x N, dense) = A B^T (+ bias)
template <typename T, bool kAK, bool kBK>
int product(const void* a, long long lda, const void* b, long long ldb, long long M, long long N, long long K, const void* bias, void* out, float* part, cudaStream_t st) {
    ProductArgs p = product_args<T>(a, lda, b, ldb, M, N, K);
    p.e.pairs = N % 2 == 0;
    const int want = splits_of(M, N, K);
    p.per_split = (p.K + want - 1) / want;
    p.per_split = (p.per_split + kStep - 1) / kStep * kStep;
    const int splits = (p.K + p.per_split - 1) / p.per_split;
    if (splits == 1) {
        p.e.bias = bias; p.e.out = out; p.e.ld = N;
        return launch_product<T, kAK, kBK, EPI_OUT, ACT_NONE>(p, 1, st);
    }
    p.e.part = part;
    if (const int rc = launch_product<T, kAK, kBK, EPI_PART, ACT_NONE>(p, splits, st)) return rc;
    return add_parts<T>(part, out, M * N, splits, bias, N, st);
}
template <typename T> int column_sums(SumArgs s, cudaStream_t st) {
    s.spans = (int)((s.rows + kSpan - 1) / kSpan);
    constexpr int kMost = 16 / (int)sizeof(T);
    bool vec = true;
    for (int i = 0; i < 2; ++i) vec = vec && (!s.cols[i] || (aligned_to(s.a[i], 16) && s.ld[i] % kMost == 0 && s.cols[i] % kMost == 0));
    const int per = 32 * (vec ? kMost : 1);
    s.blocks = (s.cols[0] + per - 1) / per;
    const dim3 grid(s.blocks + (s.cols[1] + per - 1) / per, s.spans);
    if (vec) launch(column_sums_kernel<T, kMost>, grid, 256, 0, st, s);
    else launch(column_sums_kernel<T, 1>, grid, 256, 0, st, s);
    count_launch();
    if (const int rc = check_launch()) return rc;
    launch(add_columns_kernel<T>, (unsigned)((s.cols[0] + s.cols[1] + 255) / 256), 256, 0, st, s);
    count_launch();
    return check_launch();
}

int check_common(const ss2d_gated_mlp_params& p) {
    if (!p.x || !p.w1 || !p.w2) return SS2D_EINVAL_NULL;
    if (!dtype_ok(p.dtype)) return SS2D_EINVAL_DTYPE;
    if (p.act != ACT_GELU && p.act != ACT_SILU) return SS2D_ENOTSUP;
    if (p.tokens <= 0 || p.channels <= 0 || p.hidden <= 0 || p.outputs <= 0) return SS2D_EINVAL_SHAPE;
    if (p.x_row_stride < p.channels) return SS2D_EINVAL_STRIDE;
    // grids of 64-row tiles in y, sizes in 32 bits
    if (p.tokens > 65535LL * kTile || p.channels > 65535 * kTile || p.hidden > 32767 * kTile || p.outputs > 65535 * kTile) return SS2D_ENOTSUP;
    const size_t e = dtype_size(p.dtype);
    for (const void* q : {p.x, p.w1, p.w2, p.b1, p.b2})
        if (!aligned_to(q, e)) return SS2D_EINVAL_ALIGN;
    return SS2D_OK;
}

template <typename T, int ACT> int plain_forward(const ss2d_gated_mlp_params& p, cudaStream_t st) {
    ProductArgs a = product_args<T>(p.x, p.x_row_stride, p.w1, p.channels, p.tokens, p.hidden, p.channels);
    a.second = (int)p.hidden;
    a.e.bias = p.b1; a.e.out = p.h; a.e.ld = p.hidden; a.e.hidden = (int)p.hidden; a.e.pairs = p.hidden % 2 == 0;
    if (const int rc = launch_product<T, false, false, EPI_GATE, ACT>(a, 1, st)) return rc;
    return product<T, false, false>(p.h, p.hidden, p.w2, p.hidden, p.tokens, p.outputs, p.hidden, p.b2, p.y, (float*)p.workspace, st);
}

// 16-bit operands whose rows TMA can read: the tensor-core kernels.
bool tc_fits(const ss2d_gated_mlp_params& p) {
    if (p.dtype == SS2D_F32 || p.channels % 8 || p.hidden % 8 || p.outputs % 8 || p.x_row_stride % 8) return false;
    for (const void* q : {p.x, p.w1, p.w2, p.b1, p.b2})
        if (!aligned_to(q, 16)) return false;
    return true;
}

bool tc_forward_fits(const ss2d_gated_mlp_params& p) { return tc_fits(p) && aligned_to(p.y, 16); }

// Tiles of the tensor-core kernels: 128 x 128, 128 x 256 (in TMEM; EPI_GATE gives half as many columns) by one CTA, 256 x 256 by two.
enum Form { kNarrow, kWide, kPair, kForms };
constexpr int kFormRows[kForms] = {128, 128, 256}, kFormCols[kForms] = {128, 256, 256}, kFormCtas[kForms] = {1, 1, 2};
// Cycles that a step of 64 of the contraction takes them, measured with all SMs at it (kernel times in us of h / y / dx of 16 384 tokens, 1 024 channels and 2 728 hidden: 201 / 122 / 195,
// 138 / 112 / 167, 126 / 85 / 137; of 6 272, 384 and 1 536: 24.0 / 12.4 / 19.6, 19.3 / 15.3 / 22.8, 23.7 / 15.1 / 22.2: rounds of tiles over the SMs decide there).
constexpr double kFormStep[kForms] = {660, 950, 800};

struct Plan { int form, splits, per_split; };
// The fewest cycles: rounds of tiles, their steps, and a fixed part for filling the ring and the last tile's epilogue.  A contraction is split, if it may be, where there
// are few tiles: the partial sums are written and read again (8 bytes an element and split at about 3 300 bytes a cycle) by a launch of its own.
Plan plan_of(long long M, long long N, long long K, bool gate, bool may_split) {
    const long long steps = (K + ptc::kDepth - 1) / ptc::kDepth;
    Plan best = {0, 1, (int)steps};
    double least = 1e30;
    for (int f = 0; f < kForms; ++f) {
        const long long out = gate ? kFormCols[f] / 2 : kFormCols[f], at_once = 148 / kFormCtas[f];
        const long long tiles = ((M + kFormRows[f] - 1) / kFormRows[f]) * ((N + out - 1) / out);
        for (long long s = 1; s <= (may_split ? 64 : 1) && s <= steps; ++s) {
            if (s > 1 && 4500.0 + 8.0 * s * M * N / 3300.0 >= least) break;          // (what the parts alone cost: more of them are no better)
            const long long per = (steps + s - 1) / s, splits = (steps + per - 1) / per;
            const double t = (double)((tiles * splits + at_once - 1) / at_once) * per * kFormStep[f] + (splits > 1 ? 4500.0 + 8.0 * splits * M * N / 3300.0 : 0.0);
            if (t < least) { least = t; best = {f, (int)splits, (int)per}; }
        }
    }
    return best;
}
// Gradients of value and gate: tiles of 128 columns by one CTA, or by two of 256 rows, whose steps are shorter by what those of the forward products are: whichever takes
// fewer rounds by them
bool grad_by_pairs(long long tokens, long long hidden) {
    const long long n = (hidden + 127) / 128, one = ((tokens + 127) / 128 * n + 147) / 148, two = ((tokens + 255) / 256 * n + 73) / 74;
    return two * kFormStep[kPair] < one * kFormStep[kWide];
}
long long part_elements(long long M, long long N, long long K) {
    const Plan w = plan_of(M, N, K, false, true);
    return w.splits > 1 ? w.splits * M * N : 0;
}
template <typename T, bool kAMN, bool kBMN, int EPI, int ACT> int run_form(int form, const ptc::Product& p, cudaStream_t st) {
    switch (form) {
        case kNarrow: return ptc::run_product<T, kAMN, kBMN, EPI, ACT, 128, false>(p, st);
        case kWide: return ptc::run_product<T, kAMN, kBMN, EPI, ACT, 256, false>(p, st);
        default: return ptc::run_product<T, kAMN, kBMN, EPI, ACT, 256, true>(p, st);
    }
}
// out (M x N, dense) = A B^T (+ bias)
template <typename T, bool kAMN, bool kBMN> int tc_product(ptc::Operand a, ptc::Operand b, long long M, long long N, long long K, const void* bias, void* out, float* part, cudaStream_t st) {
    const Plan w = plan_of(M, N, K, false, true);
    ptc::Product p = {};
    p.a = a; p.b = b;
    p.M = M; p.N = N; p.K = K; p.b_rows = N; p.out_pitch = N;
    if (w.splits == 1) {
        p.bias = bias; p.out = out;
        return run_form<T, kAMN, kBMN, EPI_OUT, ACT_NONE>(w.form, p, st);
    }
    p.out = part; p.splits = w.splits; p.per_split = w.per_split;
    if (const int rc = run_form<T, kAMN, kBMN, EPI_PART, ACT_NONE>(w.form, p, st)) return rc;
    return add_parts<T>(part, out, M * N, w.splits, bias, N, st);
}

template <typename T, int EPI, int ACT> int launch_few(const FewArgs& a, cudaStream_t st) {
    auto go = [&](auto tiles, auto rows) {
        constexpr int kTiles = decltype(tiles)::value, kRows = decltype(rows)::value;
        launch(few_tokens_kernel<T, kTiles, kRows, EPI, ACT>, (a.N + kRows - 1) / kRows, 256, 0, st, a);
        count_launch();
        return check_launch();
    };
    auto with = [&](auto tiles) {       // rows of a CTA: 16, or 8 where that leaves SMs without one
        return (a.N + 15) / 16 < 148 ? go(tiles, std::integral_constant<int, 8>()) : go(tiles, std::integral_constant<int, 16>());
    };
    return a.M <= 8 ? with(std::integral_constant<int, 1>()) : with(std::integral_constant<int, 2>());
}
template <typename T, int ACT> int few_forward(const ss2d_gated_mlp_params& p, cudaStream_t st) {
    if (const int rc = launch_few<T, EPI_GATE, ACT>({p.x, p.w1, p.b1, p.h, p.x_row_stride, p.hidden, (int)p.tokens, (int)p.hidden, (int)p.channels}, st)) return rc;
    return launch_few<T, EPI_OUT, ACT_NONE>({p.h, p.w2, p.b2, p.y, p.hidden, 0, (int)p.tokens, (int)p.outputs, (int)p.hidden}, st);
}

template <typename T, int ACT> int tc_forward(const ss2d_gated_mlp_params& p, cudaStream_t st) {
    if (p.tokens <= kFew) return few_forward<T, ACT>(p, st);
    ptc::Product a = {};
    a.a = {p.x, p.x_row_stride}; a.b = {p.w1, p.channels};
    a.M = p.tokens; a.N = p.hidden; a.K = p.channels; a.b_rows = 2 * p.hidden;
    a.bias = p.b1; a.out = p.h; a.out_pitch = p.hidden;
    if (const int rc = run_form<T, false, false, EPI_GATE, ACT>(plan_of(a.M, a.N, a.K, true, false).form, a, st)) return rc;
    return tc_product<T, false, false>({p.h, p.hidden}, {p.w2, p.hidden}, p.tokens, p.outputs, p.hidden, p.b2, p.y, (float*)p.workspace, st);
}
// of either kind of kernel: which one takes a call also depends on where its tensors start
long long fwd_workspace(const ss2d_gated_mlp_params& p) {
    const long long s = splits_of(p.tokens, p.outputs, p.hidden), plain = s > 1 ? s * p.tokens * p.outputs : 0;
    const long long tc = p.dtype == SS2D_F32 || p.tokens <= kFew ? 0 : part_elements(p.tokens, p.outputs, p.hidden);
    return 4 * (plain > tc ? plain : tc);
}

// The same for the backward call's own tensors: what its workspace holds follows from it.
bool tc_fits(const ss2d_gated_mlp_bwd_params& p) {
    if (!tc_fits(p.fwd) || !p.dy || p.dy_row_stride % 8) return false;
    for (const void* q : {p.dy, (const void*)p.dx, (const void*)p.dw1, (const void*)p.dw2})
        if (!aligned_to(q, 16)) return false;
    return true;
}
struct BwdPlan { bool tc; long long dz, part, pre, total; };
BwdPlan bwd_plan(const ss2d_gated_mlp_bwd_params& b) {
    const ss2d_gated_mlp_params& p = b.fwd;
    auto up = [](long long n) { return (n + 255) / 256 * 256; };
    BwdPlan w;
    w.tc = tc_fits(b);
    w.dz = up(2 * p.tokens * p.hidden * (long long)dtype_size(p.dtype));
    const long long spans = (p.tokens + kSpan - 1) / kSpan;
    long long most = spans * (2 * p.hidden + p.outputs);
    const long long M1 = 2 * p.hidden, N1 = p.channels, M2 = p.outputs, N2 = p.hidden;
    auto parts = [&](long long M, long long N, long long K) { return w.tc ? part_elements(M, N, K) : splits_of(M, N, K) * M * N; };
    for (long long n : {parts(M1, N1, p.tokens), parts(M2, N2, p.tokens), parts(p.tokens, p.channels, M1)})
        if (n > most) most = n;
    w.part = up(4 * most);
    w.pre = w.tc ? 0 : up(8 * p.tokens * p.hidden);           // the tensor-core kernels have value and gate in TMEM
    w.total = w.dz + w.part + w.pre;
    return w;
}

template <typename T, int ACT> int backward(const ss2d_gated_mlp_bwd_params& p, const BwdPlan& plan, cudaStream_t st) {
    const ss2d_gated_mlp_params& f = p.fwd;
    char* const ws = (char*)p.workspace;
    void* const dz = ws;
    float *const part = (float*)(ws + plan.dz), *const pre = (float*)(ws + plan.dz + plan.part);
    const long long H = f.hidden, H2 = 2 * H;
    const bool tc = plan.tc;
    if (p.dx || p.dw1 || p.db1) {
        if constexpr (sizeof(T) == 2)
            if (tc) {
                ptc::Product a = {};
                a.a = {f.x, f.x_row_stride}; a.b = {f.w1, f.channels}; a.a2 = {p.dy, p.dy_row_stride}; a.b2 = {f.w2, H};
                a.M = f.tokens; a.N = H; a.K = f.channels; a.K2 = f.outputs; a.b_rows = H2; a.bias = f.b1;
                a.out = dz; a.out2 = (T*)dz + H; a.out_pitch = H2;
                if (const int rc = grad_by_pairs(f.tokens, H) ? ptc::run_product<T, false, true, EPI_GRAD, ACT, 384, true>(a, st)
                                                              : ptc::run_product<T, false, true, EPI_GRAD, ACT, 384, false>(a, st)) return rc;
            }
        if (!tc) {
            ProductArgs g = product_args<T>(f.x, f.x_row_stride, f.w1, f.channels, f.tokens, H, f.channels);
            g.second = (int)H;
            g.e.bias = f.b1; g.e.hidden = (int)H; g.e.pre = pre; g.e.pairs = H % 2 == 0;
            if (const int rc = launch_product<T, false, false, EPI_GATE, ACT>(g, 1, st)) return rc;
            ProductArgs a = product_args<T>(p.dy, p.dy_row_stride, f.w2, H, f.tokens, H, f.outputs);
            a.e.out = dz; a.e.ld = H2; a.e.hidden = (int)H; a.e.pre = pre; a.e.pairs = H % 2 == 0;
            if (const int rc = launch_product<T, false, true, EPI_GRAD, ACT>(a, 1, st)) return rc;
        }
    }
    if (p.dx) {
        if constexpr (sizeof(T) == 2)
            if (tc) {
                if (const int rc = tc_product<T, false, true>({dz, H2}, {f.w1, f.channels}, f.tokens, f.channels, H2, nullptr, p.dx, part, st)) return rc;
            }
        if (!tc) {
            if (const int rc = product<T, false, true>(dz, H2, f.w1, f.channels, f.tokens, f.channels, H2, nullptr, p.dx, part, st)) return rc;
        }
    }
    auto weight = [&](const void* a, long long lda, const void* b, long long ldb, long long M, long long N, void* out) {
        if constexpr (sizeof(T) == 2)
            if (tc) return tc_product<T, true, true>({a, lda}, {b, ldb}, M, N, f.tokens, nullptr, out, part, st);
        return product<T, true, true>(a, lda, b, ldb, M, N, f.tokens, nullptr, out, part, st);
    };
    if (p.dw1)
        if (const int rc = weight(dz, H2, f.x, f.x_row_stride, H2, f.channels, p.dw1)) return rc;
    if (p.dw2)
        if (const int rc = weight(p.dy, p.dy_row_stride, f.h, H, f.outputs, H, p.dw2)) return rc;
    if (p.db1 || p.db2) {
        SumArgs sums = {};
        int n = 0;
        auto add = [&](const void* m, long long ld, long long cols, void* out) {
            sums.a[n] = m; sums.ld[n] = ld; sums.cols[n] = (int)cols; sums.out[n++] = out;
        };
        if (p.db1) add(dz, H2, H2, p.db1);
        if (p.db2) add(p.dy, p.dy_row_stride, f.outputs, p.db2);
        sums.rows = f.tokens; sums.part = part;
        if (const int rc = column_sums<T>(sums, st)) return rc;
    }
    return SS2D_OK;
}

template <typename F> int for_type_act(int dtype, int act, F&& f) {
    auto with = [&](auto z) {
        return act == ACT_GELU ? f(z, std::integral_constant<int, ACT_GELU>()) : f(z, std::integral_constant<int, ACT_SILU>());
    };
    switch (dtype) {
        case SS2D_F32: return with((float)0);
        case SS2D_F16: return with(__half());
        default: return with(__nv_bfloat16());
    }
}

}  // namespace

int gated_mlp_fwd(const ss2d_gated_mlp_params* p, cudaStream_t st) {
    if (!p) return SS2D_EINVAL_NULL;
    if (const int rc = check_common(*p)) return rc;
    if (!p->h || !p->y) return SS2D_EINVAL_NULL;
    if (!aligned_to(p->h, 16) || !aligned_to(p->y, 2 * dtype_size(p->dtype))) return SS2D_EINVAL_ALIGN;
    const long long need = fwd_workspace(*p);
    if (need && (!p->workspace || p->workspace_bytes < need || !aligned_to(p->workspace, 16))) return SS2D_EWORKSPACE;
    return for_type_act(p->dtype, p->act, [&](auto z, auto act) {
        using T = decltype(z);
        constexpr int A = decltype(act)::value;
        if constexpr (sizeof(T) == 2)
            if (tc_forward_fits(*p)) return tc_forward<T, A>(*p, st);
        return plain_forward<T, A>(*p, st);
    });
}

long long gated_mlp_workspace_bytes(const ss2d_gated_mlp_params* p) {
    if (!p || check_common(*p) != SS2D_OK) return -1;
    return fwd_workspace(*p);
}

long long gated_mlp_bwd_workspace_bytes(const ss2d_gated_mlp_bwd_params* p) {
    if (!p || check_common(p->fwd) != SS2D_OK) return -1;
    return bwd_plan(*p).total;
}

int gated_mlp_kernel(const ss2d_gated_mlp_bwd_params* p, int product) {
    if (!p) return SS2D_EINVAL_NULL;
    const ss2d_gated_mlp_params& f = p->fwd;
    if (const int rc = check_common(f)) return rc;
    const long long sizes[6][3] = {{f.tokens, f.hidden, f.channels}, {f.tokens, f.outputs, f.hidden}, {f.tokens, f.hidden, f.outputs}, {f.tokens, f.channels, 2 * f.hidden},
                                   {2 * f.hidden, f.channels, f.tokens}, {f.outputs, f.hidden, f.tokens}};
    if (product < 0 || product > 5) return SS2D_EINVAL_SHAPE;
    const auto& [M, N, K] = sizes[product];
    const bool one = product == 0 || product == 2;                                // nothing is split in front of an activation
    if (!(product < 2 ? tc_forward_fits(f) : tc_fits(*p))) {
        const long long want = one ? 1 : splits_of(M, N, K), per = ((K + want - 1) / want + kStep - 1) / kStep * kStep;
        return SS2D_GATED_MLP_PLAIN + 16 * (int)((K + per - 1) / per);
    }
    if (product < 2 && f.tokens <= kFew) return SS2D_GATED_MLP_FEW + 16;
    if (product == 2) return (grad_by_pairs(M, N) ? SS2D_GATED_MLP_PAIR : SS2D_GATED_MLP_WIDE) + 16;
    const Plan w = plan_of(M, N, K, product == 0, !one);
    return SS2D_GATED_MLP_NARROW + w.form + 16 * w.splits;
}

int gated_mlp_bwd(const ss2d_gated_mlp_bwd_params* p, cudaStream_t st) {
    if (!p) return SS2D_EINVAL_NULL;
    const ss2d_gated_mlp_params& f = p->fwd;
    if (const int rc = check_common(f)) return rc;
    if (!p->dy || !f.h) return SS2D_EINVAL_NULL;
    if (p->dy_row_stride < f.outputs) return SS2D_EINVAL_STRIDE;
    const size_t e = dtype_size(f.dtype);
    if (!aligned_to(p->dy, e) || !aligned_to(f.h, 16)) return SS2D_EINVAL_ALIGN;
    for (const void* q : {p->dx, p->dw1, p->dw2, p->db1, p->db2})
        if (!aligned_to(q, 2 * e)) return SS2D_EINVAL_ALIGN;
    const BwdPlan plan = bwd_plan(*p);
    if (!p->workspace || p->workspace_bytes < plan.total || !aligned_to(p->workspace, 16)) return SS2D_EWORKSPACE;
    return for_type_act(f.dtype, f.act, [&](auto z, auto act) { return backward<decltype(z), decltype(act)::value>(*p, plan, st); });
}

}  // namespace ss2d
