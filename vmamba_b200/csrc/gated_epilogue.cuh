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

// activation of the gate and its derivative, to fp32's accuracy (the sums that follow them round far more for 16-bit types, but not for fp32)
template <int ACT> __device__ __forceinline__ float gate_act(float g) {
    if constexpr (ACT == ACT_GELU) return 0.5f * g * (1.0f + erff(g * 0.70710678118654752f));
    else return g * __fdividef(1.0f, 1.0f + __expf(-g));
}
template <int ACT> __device__ __forceinline__ void gate_act_grad(float g, float& a, float& da) {
    if constexpr (ACT == ACT_GELU) {
        const float phi = 0.5f * (1.0f + erff(g * 0.70710678118654752f));
        a = g * phi;
        da = fmaf(g * 0.3989422804014327f, __expf(-0.5f * g * g), phi);
    } else {
        const float s = __fdividef(1.0f, 1.0f + __expf(-g));
        a = g * s;
        da = s * fmaf(g, 1.0f - s, 1.0f);
    }
}

// The same on pairs, for 16-bit types: gelu by a polynomial on the FMA pipe (error 3.5e-5), sigmoid through tanh.approx (2^-11 of tanh) where the
// result is rounded to bf16, through an exponential and a division beside fp16.
template <typename T> __device__ __forceinline__ float2 sigmoid_pair(float2 g) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        const float2 h = __fmul2_rn(g, splat2(0.5f));
        float2 t;
        asm("tanh.approx.f32 %0, %1;" : "=f"(t.x) : "f"(h.x));
        asm("tanh.approx.f32 %0, %1;" : "=f"(t.y) : "f"(h.y));
        return __ffma2_rn(t, splat2(0.5f), splat2(0.5f));
    } else
        return make_float2(__fdividef(1.0f, 1.0f + __expf(-g.x)), __fdividef(1.0f, 1.0f + __expf(-g.y)));
}
template <typename T, int ACT> __device__ __forceinline__ float2 act_pair(float2 g) {
    if constexpr (ACT == ACT_GELU) return __fmul2_rn(g, normal_cdf_pair(g));
    else return __fmul2_rn(g, sigmoid_pair<T>(g));
}
template <typename T, int ACT> __device__ __forceinline__ void act_grad_pair(float2 g, float2& a, float2& da) {
    if constexpr (ACT == ACT_GELU) {
        const float2 phi = normal_cdf_pair(g);
        const float2 e = __fmul2_rn(__fmul2_rn(g, g), splat2(-0.5f * kLog2e));
        a = __fmul2_rn(g, phi);
        da = __ffma2_rn(__fmul2_rn(g, splat2(0.3989422804014327f)), make_float2(ex2_approx(e.x), ex2_approx(e.y)), phi);
    } else {
        const float2 s = sigmoid_pair<T>(g);
        a = __fmul2_rn(g, s);
        da = __ffma2_rn(a, __ffma2_rn(s, splat2(-1.0f), splat2(1.0f)), s);
    }
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
