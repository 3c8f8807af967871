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
                        mma_exact(to[j][u][n], a[u], b0);
                        mma_exact(to[j][u][n + 1], a[u], b1);
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

// ---- sums ---------------------------------------------------------------------------------------------------------------
// Column sums of a (rows, cols) matrix over spans of rows, fp32: part[span][col]
constexpr int kSpan = 256;
template <typename T> __global__ void __launch_bounds__(256) column_sums_kernel(const T* a, long long ld, long long rows, int cols, float* part) {
    follow_previous();
    __shared__ float s[8][32];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5, c = blockIdx.x * 32 + tx;
    const long long r0 = (long long)blockIdx.y * kSpan, r1 = r0 + kSpan < rows ? r0 + kSpan : rows;
    float x = 0.f;
    if (c < cols)
        for (long long r = r0 + ty; r < r1; r += 8) x += to_f<T>(a[r * ld + c]);
    s[ty][tx] = x;
    __syncthreads();
    if (ty == 0 && c < cols) {
        for (int i = 1; i < 8; ++i) x += s[i][tx];
        part[(long long)blockIdx.y * cols + c] = x;
    }
}
// out[i] = sum over parts, in order
template <typename T> __global__ void __launch_bounds__(256) add_parts_kernel(const float* part, T* out, long long n, int parts) {
    follow_previous();
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    float x = 0.f;
    for (int p = 0; p < parts; ++p) x += part[p * n + i];
    out[i] = from_f<T>(x);
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
// Splits of a contraction over the tokens whose result has few tiles: enough for two CTAs an SM, each with 8 steps at least
int splits_of(long long M, long long N, long long K) {
    const long long tiles = ((M + kTile - 1) / kTile) * ((N + kTile - 1) / kTile), steps = (K + kStep - 1) / kStep;
    long long s = (2 * 148 + tiles - 1) / tiles;
    if (s > steps / 8) s = steps / 8;
    return s < 1 ? 1 : s > 64 ? 64 : (int)s;
}
template <typename T> int add_parts(const float* part, void* out, long long n, int parts, cudaStream_t st) {
    launch(add_parts_kernel<T>, (unsigned)((n + 255) / 256), 256, 0, st, part, (T*)out, n, parts);
    count_launch();
    return check_launch();
}
// out (M x N) = A^T B over K tokens, rows of A and B contiguous
template <typename T> int weight_gradient(const void* a, long long lda, const void* b, long long ldb, long long M, long long N, long long K, void* out, float* part, cudaStream_t st) {
    ProductArgs p = product_args<T>(a, lda, b, ldb, M, N, K);
    p.e.pairs = N % 2 == 0;
    const int want = splits_of(M, N, K);
    p.per_split = (p.K + want - 1) / want;
    p.per_split = (p.per_split + kStep - 1) / kStep * kStep;
    const int splits = (p.K + p.per_split - 1) / p.per_split;
    if (splits == 1) {
        p.e.out = out; p.e.ld = N;
        return launch_product<T, true, true, EPI_OUT, ACT_NONE>(p, 1, st);
    }
    p.e.part = part;
    if (const int rc = launch_product<T, true, true, EPI_PART, ACT_NONE>(p, splits, st)) return rc;
    return add_parts<T>(part, out, M * N, splits, st);
}
template <typename T> int column_sums(const void* a, long long ld, long long rows, int cols, void* out, float* part, cudaStream_t st) {
    const long long spans = (rows + kSpan - 1) / kSpan;
    launch(column_sums_kernel<T>, dim3((cols + 31) / 32, (unsigned)spans), 256, 0, st, (const T*)a, ld, rows, cols, part);
    count_launch();
    if (const int rc = check_launch()) return rc;
    return add_parts<T>(part, out, cols, (int)spans, st);
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
    ProductArgs b = product_args<T>(p.h, p.hidden, p.w2, p.hidden, p.tokens, p.outputs, p.hidden);
    b.e.bias = p.b2; b.e.out = p.y; b.e.ld = p.outputs; b.e.pairs = p.outputs % 2 == 0;
    return launch_product<T, false, false, EPI_OUT, ACT_NONE>(b, 1, st);
}

struct BwdPlan { long long dz, part, pre, total; };

// 16-bit operands whose rows TMA can read: the tensor-core kernels.
bool tc_fits(const ss2d_gated_mlp_params& p) {
    if (p.dtype == SS2D_F32 || p.channels % 8 || p.hidden % 8 || p.outputs % 8 || p.x_row_stride % 8) return false;
    for (const void* q : {p.x, p.w1, p.w2, p.b1, p.b2})
        if (!aligned_to(q, 16)) return false;
    return true;
}

// Time of a tensor-core product in cycles, for the choice among its tiles: rounds of tiles over the SMs, each as long as its MMAs (a step of 64 of the contraction
// takes as many cycles as it has columns, and no fewer than 128 columns' worth) and a fixed part for filling the ring and the last tile's epilogue.
double tc_cycles(long long tiles, long long steps, int columns) {
    const long long rounds = (tiles + 147) / 148;
    return (double)rounds * steps * (columns < 128 ? 128 : columns) + 1500.0;
}
long long tc_tiles(long long M, long long N, int out) { return ((M + ptc::kRows - 1) / ptc::kRows) * ((N + out - 1) / out); }

template <typename T, int ACT> int tc_forward(const ss2d_gated_mlp_params& p, cudaStream_t st) {
    ptc::Product a = {};
    a.a = {p.x, p.x_row_stride}; a.b = {p.w1, p.channels};
    a.M = p.tokens; a.N = p.hidden; a.K = p.channels; a.b_rows = 2 * p.hidden;
    a.bias = p.b1; a.out = p.h; a.out_pitch = p.hidden;
    const long long steps = (p.channels + ptc::kDepth - 1) / ptc::kDepth;
    const bool wide = tc_cycles(tc_tiles(a.M, a.N, 128), steps, 256) <= tc_cycles(tc_tiles(a.M, a.N, 64), steps, 128);
    if (const int rc = wide ? ptc::run_product<T, false, false, EPI_GATE, ACT, 256>(a, st) : ptc::run_product<T, false, false, EPI_GATE, ACT, 128>(a, st)) return rc;
    ptc::Product b = {};
    b.a = {p.h, p.hidden}; b.b = {p.w2, p.hidden};
    b.M = p.tokens; b.N = p.outputs; b.K = p.hidden; b.b_rows = p.outputs;
    b.bias = p.b2; b.out = p.y; b.out_pitch = p.outputs;
    const long long steps2 = (p.hidden + ptc::kDepth - 1) / ptc::kDepth;
    const bool wide2 = tc_cycles(tc_tiles(b.M, b.N, 256), steps2, 256) <= tc_cycles(tc_tiles(b.M, b.N, 128), steps2, 128);
    return wide2 ? ptc::run_product<T, false, false, EPI_OUT, ACT_NONE, 256>(b, st) : ptc::run_product<T, false, false, EPI_OUT, ACT_NONE, 128>(b, st);
}

// Splits of a weight gradient's contraction over the tokens, and its tile: the fewest cycles, with the partial sums' way to memory and back (8 bytes an element
// and split at about 3 300 bytes a cycle)
struct WeightPlan { int splits, per_split; bool wide; };
WeightPlan tc_weight_plan(long long M, long long N, long long K) {
    const long long steps = (K + ptc::kDepth - 1) / ptc::kDepth;
    WeightPlan best = {1, (int)steps, false};
    double least = 1e30;
    for (int wide = 0; wide < 2; ++wide)
        for (long long s = 1; s <= 64 && s <= steps; ++s) {
            const long long per = (steps + s - 1) / s, splits = (steps + per - 1) / per;
            const double t = tc_cycles(tc_tiles(M, N, wide ? 256 : 128) * splits, per, wide ? 256 : 128) + (splits > 1 ? 3000.0 + 8.0 * splits * M * N / 3300.0 : 0.0);
            if (t < least) { least = t; best = {(int)splits, (int)per, wide != 0}; }
        }
    return best;
}
template <typename T> int tc_weight_gradient(const void* a, long long lda, const void* b, long long ldb, long long M, long long N, long long K, void* out, float* part, cudaStream_t st) {
    const WeightPlan w = tc_weight_plan(M, N, K);
    ptc::Product p = {};
    p.a = {a, lda}; p.b = {b, ldb};
    p.M = M; p.N = N; p.K = K; p.b_rows = N; p.out_pitch = N;
    if (w.splits == 1) {
        p.out = out;
        return w.wide ? ptc::run_product<T, true, true, EPI_OUT, ACT_NONE, 256>(p, st) : ptc::run_product<T, true, true, EPI_OUT, ACT_NONE, 128>(p, st);
    }
    p.out = part; p.splits = w.splits; p.per_split = w.per_split;
    if (const int rc = w.wide ? ptc::run_product<T, true, true, EPI_PART, ACT_NONE, 256>(p, st) : ptc::run_product<T, true, true, EPI_PART, ACT_NONE, 128>(p, st)) return rc;
    return add_parts<T>(part, out, M * N, w.splits, st);
}

BwdPlan bwd_plan(const ss2d_gated_mlp_params& p) {
    auto up = [](long long n) { return (n + 255) / 256 * 256; };
    BwdPlan b;
    b.dz = up(2 * p.tokens * p.hidden * (long long)dtype_size(p.dtype));
    const long long spans = (p.tokens + kSpan - 1) / kSpan;
    long long most = spans * (2 * p.hidden > p.outputs ? 2 * p.hidden : p.outputs);
    const long long M1 = 2 * p.hidden, N1 = p.channels, M2 = p.outputs, N2 = p.hidden;
    for (long long n : {splits_of(M1, N1, p.tokens) * M1 * N1, splits_of(M2, N2, p.tokens) * M2 * N2, tc_weight_plan(M1, N1, p.tokens).splits * M1 * N1,
                        tc_weight_plan(M2, N2, p.tokens).splits * M2 * N2})
        if (n > most) most = n;
    b.part = up(4 * most);
    b.pre = up(8 * p.tokens * p.hidden);                      // of calls that the tensor-core kernels do not take, wherever their tensors start
    b.total = b.dz + b.part + b.pre;
    return b;
}

template <typename T, int ACT> int backward(const ss2d_gated_mlp_bwd_params& p, cudaStream_t st) {
    const ss2d_gated_mlp_params& f = p.fwd;
    const BwdPlan plan = bwd_plan(f);
    char* const ws = (char*)p.workspace;
    void* const dz = ws;
    float *const part = (float*)(ws + plan.dz), *const pre = (float*)(ws + plan.dz + plan.part);
    const long long H = f.hidden, H2 = 2 * H;
    bool tc = false;
    if constexpr (sizeof(T) == 2) {
        tc = tc_fits(f) && p.dy_row_stride % 8 == 0;
        for (const void* q : {p.dy, (const void*)p.dx, (const void*)p.dw1, (const void*)p.dw2}) tc = tc && aligned_to(q, 16);
    }
    if (p.dx || p.dw1 || p.db1) {
        if constexpr (sizeof(T) == 2)
            if (tc) {
                ptc::Product a = {};
                a.a = {f.x, f.x_row_stride}; a.b = {f.w1, f.channels}; a.a2 = {p.dy, p.dy_row_stride}; a.b2 = {f.w2, H};
                a.M = f.tokens; a.N = H; a.K = f.channels; a.K2 = f.outputs; a.b_rows = H2; a.bias = f.b1;
                a.out = dz; a.out2 = (T*)dz + H; a.out_pitch = H2;
                if (const int rc = ptc::run_product<T, false, true, EPI_GRAD, ACT, 192>(a, st)) return rc;
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
                ptc::Product a = {};
                a.a = {dz, H2}; a.b = {f.w1, f.channels};
                a.M = f.tokens; a.N = f.channels; a.K = H2; a.b_rows = f.channels; a.out = p.dx; a.out_pitch = f.channels;
                const long long steps = (H2 + ptc::kDepth - 1) / ptc::kDepth;
                const bool wide = tc_cycles(tc_tiles(a.M, a.N, 256), steps, 256) <= tc_cycles(tc_tiles(a.M, a.N, 128), steps, 128);
                if (const int rc = wide ? ptc::run_product<T, false, true, EPI_OUT, ACT_NONE, 256>(a, st) : ptc::run_product<T, false, true, EPI_OUT, ACT_NONE, 128>(a, st)) return rc;
            }
        if (!tc) {
            ProductArgs a = product_args<T>(dz, H2, f.w1, f.channels, f.tokens, f.channels, H2);
            a.e.out = p.dx; a.e.ld = f.channels; a.e.pairs = f.channels % 2 == 0;
            if (const int rc = launch_product<T, false, true, EPI_OUT, ACT_NONE>(a, 1, st)) return rc;
        }
    }
    auto weight = [&](const void* a, long long lda, const void* b, long long ldb, long long M, long long N, void* out) {
        if constexpr (sizeof(T) == 2)
            if (tc) return tc_weight_gradient<T>(a, lda, b, ldb, M, N, f.tokens, out, part, st);
        return weight_gradient<T>(a, lda, b, ldb, M, N, f.tokens, out, part, st);
    };
    if (p.dw1)
        if (const int rc = weight(dz, H2, f.x, f.x_row_stride, H2, f.channels, p.dw1)) return rc;
    if (p.dw2)
        if (const int rc = weight(p.dy, p.dy_row_stride, f.h, H, f.outputs, H, p.dw2)) return rc;
    if (p.db1)
        if (const int rc = column_sums<T>(dz, H2, f.tokens, (int)H2, p.db1, part, st)) return rc;
    if (p.db2)
        if (const int rc = column_sums<T>(p.dy, p.dy_row_stride, f.tokens, (int)f.outputs, p.db2, part, st)) return rc;
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
    return for_type_act(p->dtype, p->act, [&](auto z, auto act) {
        using T = decltype(z);
        constexpr int A = decltype(act)::value;
        if constexpr (sizeof(T) == 2)
            if (tc_fits(*p) && aligned_to(p->y, 16)) return tc_forward<T, A>(*p, st);
        return plain_forward<T, A>(*p, st);
    });
}

long long gated_mlp_bwd_workspace_bytes(const ss2d_gated_mlp_bwd_params* p) {
    if (!p || check_common(p->fwd) != SS2D_OK) return -1;
    return bwd_plan(p->fwd).total;
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
    if (!p->workspace || p->workspace_bytes < bwd_plan(f).total || !aligned_to(p->workspace, 16)) return SS2D_EWORKSPACE;
    return for_type_act(f.dtype, f.act, [&](auto z, auto act) { return backward<decltype(z), decltype(act)::value>(*p, st); });
}

}  // namespace ss2d
