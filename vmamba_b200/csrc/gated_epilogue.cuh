// What follows the products of the gated feed-forward block, for accumulators of any kernel: value and gate to hidden, the gradients of both, biases.
#pragma once
#include <type_traits>

#include "activations.cuh"

namespace ss2d {

enum Epilogue { EPI_OUT = 0, EPI_GATE = 1, EPI_GRAD = 2, EPI_PART = 3 };

struct EpiArgs {
    const void* bias;       // of the block's type or NULL: one for each output column (EPI_GATE: 2 hidden, values first)
    void* out;              // EPI_OUT: (rows, cols); EPI_GATE: hidden (rows, hidden) or NULL; EPI_GRAD: gradients of value and gate (rows, 2 hidden)
    float* pre;             // values and gates in front of the product, (rows, 2 hidden), fp32.  EPI_GATE: written unless NULL; EPI_GRAD: read
    float* part;            // EPI_PART: (splits, rows, cols)
    long long ld;           // elements between rows of `out`
    int hidden;
    bool pairs;             // two neighbouring columns may be stored at once
};

// Activation of the gate and its derivative, to fp32's accuracy relative to the value itself: sigmoid and Phi as products with an exponential of -|g| or -g^2 / 2 on
// the negative side, where 1/2 - 1/2 tanh and 1/2 + 1/2 erf would leave no digits of them.
template <int ACT> __device__ __forceinline__ void gate_act_grad(float g, float& a, float& da) {
    if constexpr (ACT == ACT_GELU) {
        const float phi = normcdff(g), h = g * g, rest = h < 1e8f ? fmaf(g, g, -h) : 0.f;       // g^2 in two pieces: an exponent's rounding is the result's
        a = g * phi;
        da = fmaf(g * 0.3989422804014327f, expf(-0.5f * h) * fmaf(-0.5f, rest, 1.0f), phi);
    } else {
        const float e = expf(-fabsf(g)), r = 1.0f / (1.0f + e), s = g < 0.f ? e * r : r, other = g < 0.f ? r : e * r;
        a = g * s;
        da = s * fmaf(g, other, 1.0f);
    }
}
template <int ACT> __device__ __forceinline__ float gate_act(float g) {
    if constexpr (ACT == ACT_GELU) return g * normcdff(g);
    else {
        const float e = expf(-fabsf(g));
        return g * ((g < 0.f ? e : 1.0f) / (1.0f + e));
    }
}

// The same on pairs, for 16-bit types, within 2^-16 of the value for every gate whose activation is a normal number.
// Phi(-a) = exp(-a^2 / 2) R(a), R(a) = erfcx(a / sqrt 2) / 2 as t P(t), t = 1 / (1 + 0.3075 a), P of degree 5: the mapping of Shepherd and Laframboise (1981), fitted to 3.8e-6
// relative on 0 <= a <= 13.5, where fp32's exponential ends (own fit, reweighted least squares).  Two transcendentals a gate.  Before: a polynomial for erf, 3.5e-5 off, which was
// all of the value from a gate of -4.3 on, and a tanh for bf16's sigmoid, 2^-12 off, most of it at -8.  What that costs (us of a forward call, before / now, bf16): 12 544 tokens, 512 channels,
// 2 048 hidden GELU 81 / 85, SiLU 79 / 83; 8 192, 1 024, 4 096 153 / 157, 151 / 153.  (One reciprocal for both of a pair: 87, 83, 157, 153.)
__device__ __forceinline__ float fast_rcp(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float2 below(float2 g, float2 x, float2 y) { return make_float2(g.x < 0.f ? x.x : y.x, g.y < 0.f ? x.y : y.y); }
// Phi(g) and exp(-g^2 / 2)
__device__ __forceinline__ void normal_cdf_pair(float2 g, float2& phi, float2& bell) {
    const float2 a = make_float2(fabsf(g.x), fabsf(g.y)), d = __ffma2_rn(a, splat2(0.3075f), splat2(1.0f));
    const float2 t = make_float2(fast_rcp(d.x), fast_rcp(d.y)), e = __fmul2_rn(__fmul2_rn(g, g), splat2(-0.5f * kLog2e));
    bell = make_float2(ex2_approx(e.x), ex2_approx(e.y));
    float2 p = splat2(-7.584733516e-02f);
    p = __ffma2_rn(p, t, splat2(1.920761615e-01f));
    p = __ffma2_rn(p, t, splat2(4.935927223e-03f));
    p = __ffma2_rn(p, t, splat2(1.374342889e-01f));
    p = __ffma2_rn(p, t, splat2(1.184579805e-01f));
    p = __ffma2_rn(p, t, splat2(1.229414865e-01f));
    const float2 tail = __fmul2_rn(bell, __fmul2_rn(t, p));
    phi = below(g, tail, __ffma2_rn(tail, splat2(-1.0f), splat2(1.0f)));
}
// sigmoid(g) and sigmoid(-g)
__device__ __forceinline__ void sigmoid_pair(float2 g, float2& s, float2& other) {
    const float2 e = make_float2(ex2_approx(-kLog2e * fabsf(g.x)), ex2_approx(-kLog2e * fabsf(g.y))), d = __fadd2_rn(e, splat2(1.0f));
    const float2 r = make_float2(fast_rcp(d.x), fast_rcp(d.y)), er = __fmul2_rn(e, r);
    s = below(g, er, r);
    other = below(g, r, er);
}
template <int ACT> __device__ __forceinline__ float2 act_pair(float2 g) {
    float2 phi, more;
    if constexpr (ACT == ACT_GELU) normal_cdf_pair(g, phi, more);
    else sigmoid_pair(g, phi, more);
    return __fmul2_rn(g, phi);
}
template <int ACT> __device__ __forceinline__ void act_grad_pair(float2 g, float2& a, float2& da) {
    float2 phi, more;
    if constexpr (ACT == ACT_GELU) {
        normal_cdf_pair(g, phi, more);
        da = __ffma2_rn(__fmul2_rn(g, splat2(0.3989422804014327f)), more, phi);
    } else {
        sigmoid_pair(g, phi, more);
        da = __fmul2_rn(phi, __ffma2_rn(g, more, splat2(1.0f)));
    }
    a = __fmul2_rn(g, phi);
}

template <typename T> __device__ __forceinline__ void store_pair(T* p, float a, float b, bool both, bool pairs) {
    if (both && pairs) {
        const float v[2] = {a, b};
        Vec<T, 2>::store(p, v);
    } else {
        p[0] = from_f<T>(a);
        if (both) p[1] = from_f<T>(b);
    }
}

// Two neighbouring columns n, n + 1 of row m: x are the accumulators (of the value), y those of the gate (EPI_GATE alone)
template <typename T, int EPI, int ACT>
__device__ __forceinline__ void finish_pair(const EpiArgs& e, long long m, int n, int cols, const float (&x)[2], const float (&y)[2], long long part_row) {
    if (n >= cols) return;
    const bool both = n + 1 < cols;
    if constexpr (EPI == EPI_PART) {
        float* p = e.part + part_row * cols + n;
        store_pair<float>(p, x[0], x[1], both, e.pairs);
    } else if constexpr (EPI == EPI_OUT) {
        float b[2] = {0.f, 0.f};
        if (e.bias) { b[0] = to_f<T>(((const T*)e.bias)[n]); if (both) b[1] = to_f<T>(((const T*)e.bias)[n + 1]); }
        store_pair<T>((T*)e.out + m * e.ld + n, x[0] + b[0], x[1] + b[1], both, e.pairs);
    } else if constexpr (EPI == EPI_GATE) {
        float v[2] = {x[0], x[1]}, g[2] = {y[0], y[1]};
        if (e.bias) {
            const T* b = (const T*)e.bias + n;
            v[0] += to_f<T>(b[0]); g[0] += to_f<T>(b[e.hidden]);
            if (both) { v[1] += to_f<T>(b[1]); g[1] += to_f<T>(b[e.hidden + 1]); }
        }
        if (e.pre) {
            float* p = e.pre + m * 2 * e.hidden + n;
            store_pair<float>(p, v[0], v[1], both, e.pairs);
            store_pair<float>(p + e.hidden, g[0], g[1], both, e.pairs);
        }
        if (e.out) store_pair<T>((T*)e.out + m * e.ld + n, v[0] * gate_act<ACT>(g[0]), v[1] * gate_act<ACT>(g[1]), both, e.pairs);
    } else {
        const float* p = e.pre + m * 2 * e.hidden + n;
        float v[2], g[2] = {0.f, 0.f}, a[2], da[2];
        v[0] = p[0]; g[0] = p[e.hidden];
        v[1] = both ? p[1] : 0.f;
        if (both) g[1] = p[e.hidden + 1];
#pragma unroll
        for (int i = 0; i < 2; ++i) gate_act_grad<ACT>(g[i], a[i], da[i]);
        T* o = (T*)e.out + m * e.ld + n;
        store_pair<T>(o, x[0] * a[0], x[1] * a[1], both, e.pairs);
        store_pair<T>(o + e.hidden, x[0] * v[0] * da[0], x[1] * v[1] * da[1], both, e.pairs);
    }
}

}  // namespace ss2d
