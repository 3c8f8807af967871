// Warp-level matrix products out of shared memory for fp32, fp16 and bf16 operands: one interface over mma.sync forms, 16 contraction
// elements a step, fp32 accumulators.
//
// Two kinds of operand.  What is read as the caller's type is exact: 16-bit elements go to the 16-bit form as they are, fp32 ones are taken as
// the sum of two tf32 halves, three products for one (22 bits; the product of the low halves, 2^-22 at most, is left out).  What a kernel has
// computed in fp32 ("derived") is rounded for the product, into `kParts` pieces of the form's type: one where the result is a 16-bit map whose own rounding is
// as large, as many as fp32 has where an fp32 result follows: three of bf16, two of tf32.  A derived operand beside fp16 goes as tf32 and not as fp16: the same 11 bits, but fp32's range
// (a state sums over the tokens and has no bound of fp16).
//
// The contraction order of the tf32 form is permuted in pairs (element 2t of 8 in place of t, 2t + 1 in place of t + 4, t the lane's quad
// position), for both operands alike.  It makes every form's accumulator layout its own A layout, 8 elements a lane in the order
//   (g, 2t) (g, 2t+1) (g+8, 2t) (g+8, 2t+1)  and the same 8 columns on,          g = lane / 4, t = lane % 4.
#pragma once
#include <type_traits>

#include "common.cuh"

namespace ss2d {
namespace mt {

__device__ __forceinline__ void mma_tf32(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t to_tf32(float v) {
    uint32_t r;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(v));
    return r;
}
template <bool kTrans> __device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], const void* p) {
    const uint32_t a = (uint32_t)__cvta_generic_to_shared(p);
    if constexpr (kTrans)
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
    else
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}

// Operands of one step: A 16 x 16, B 16 x 8.  16-bit: packed pairs; fp32: values in the order above (B: k = 2t, 2t+1, 8+2t, 9+2t of column g).
template <typename T> struct OpA { uint32_t r[4]; };
template <> struct OpA<float> { float v[8]; };
template <typename T> struct OpB { uint32_t r[2]; };
template <> struct OpB<float> { float v[4]; };

// kStoredK: shared memory holds rows of the contraction index ([k][m]) instead of rows of m ([m][k])
template <bool kStoredK, typename T> __device__ __forceinline__ OpA<T> load_a(const T* s, int ld, int m0, int k0, int lane) {
    OpA<T> o;
    if constexpr (sizeof(T) == 2) {
        if constexpr (kStoredK) ldmatrix4<true>(o.r, s + (k0 + (lane & 7) + ((lane >> 4) << 3)) * ld + m0 + (((lane >> 3) & 1) << 3));
        else ldmatrix4<false>(o.r, s + (m0 + (lane & 15)) * ld + k0 + ((lane >> 4) << 3));
    } else {
        const int g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int row = 0; row < 2; ++row)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int m = m0 + g + 8 * row, k = k0 + 8 * h + 2 * t + j;
                    o.v[4 * h + 2 * row + j] = kStoredK ? s[k * ld + m] : s[m * ld + k];
                }
    }
    return o;
}
// two B operands, columns n0 .. n0+7 and n0+8 .. n0+15.  kStoredK: rows of the contraction index ([k][n]), else rows of n ([n][k])
template <bool kStoredK, typename T> __device__ __forceinline__ void load_b2(OpB<T>& b0, OpB<T>& b1, const T* s, int ld, int n0, int k0, int lane) {
    if constexpr (sizeof(T) == 2) {
        uint32_t r[4];
        if constexpr (kStoredK) ldmatrix4<true>(r, s + (k0 + (lane & 15)) * ld + n0 + ((lane >> 4) << 3));
        else ldmatrix4<false>(r, s + (n0 + (lane & 7) + ((lane >> 4) << 3)) * ld + k0 + (((lane >> 3) & 1) << 3));
        b0.r[0] = r[0]; b0.r[1] = r[1]; b1.r[0] = r[2]; b1.r[1] = r[3];
    } else {
        const int g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int k = k0 + (j >> 1) * 8 + 2 * t + (j & 1);
            b0.v[j] = kStoredK ? s[k * ld + n0 + g] : s[(n0 + g) * ld + k];
            b1.v[j] = kStoredK ? s[k * ld + n0 + 8 + g] : s[(n0 + 8 + g) * ld + k];
        }
    }
}

template <typename T> __device__ __forceinline__ void values(const OpA<T>& a, float (&v)[8]) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {           // registers: (g, k 0-7) (g+8, k 0-7) (g, k 8-15) (g+8, k 8-15)
            const float2 f = Half2Of<T>::unpack(a.r[i]);
            v[2 * i] = f.x; v[2 * i + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = a.v[i];
    }
}
template <typename T> __device__ __forceinline__ void values(const OpB<T>& b, float (&v)[4]) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float2 f = Half2Of<T>::unpack(b.r[i]);
            v[2 * i] = f.x; v[2 * i + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = b.v[i];
    }
}

// fp32 values as tf32 pieces: kA of a and kB of b (1 or 2); the product of two second pieces is left out.
// kApart: a step's products are summed on their own and join the others by ordinary additions, as tensor cores cut their sums off instead of rounding them, always towards zero.  For
// fp32 results; not where a caller adds up few steps apart itself.  Linear attention in fp32, against 64 bits: gradients 9e-7 to 1.1e-6 -> 4e-7 to 5e-7, outputs 8e-7 -> 5e-7 (elementary fp32
// operations 2e-7); training of 4 x 1 001 tokens of 8 heads of 32 x 64 128 -> 130 us, of 2 x 4 096 of 16 heads of 128 x 128 2 051 -> 2 251.
template <int kA, int kB, bool kApart = (kA > 1 && kB > 1)> __device__ __forceinline__ void mma_values(float (&c)[4], const float (&a)[8], const float (&b)[4]) {
    float own[4] = {};
    auto& to = [&]() -> auto& { if constexpr (kApart) return own; else return c; }();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const float* x = a + 4 * h;
        uint32_t ah[4], bh[2];
#pragma unroll
        for (int i = 0; i < 4; ++i) ah[i] = to_tf32(x[i]);
#pragma unroll
        for (int i = 0; i < 2; ++i) bh[i] = to_tf32(b[2 * h + i]);
        if constexpr (kA > 1) {
            uint32_t al[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) al[i] = to_tf32(x[i] - __uint_as_float(ah[i]));
            mma_tf32(to, al[0], al[2], al[1], al[3], bh[0], bh[1]);
        }
        if constexpr (kB > 1) {
            uint32_t bl[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) bl[i] = to_tf32(b[2 * h + i] - __uint_as_float(bh[i]));
            mma_tf32(to, ah[0], ah[2], ah[1], ah[3], bl[0], bl[1]);
        }
        mma_tf32(to, ah[0], ah[2], ah[1], ah[3], bh[0], bh[1]);
    }
    if constexpr (kApart) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c[i] += own[i];
    }
}

// exact times exact
template <bool kApart = true, typename T> __device__ __forceinline__ void mma_exact(float (&c)[4], const OpA<T>& a, const OpB<T>& b) {
    if constexpr (sizeof(T) == 2) MmaK16<T>::run(c, a.r, b.r);
    else mma_values<2, 2, kApart>(c, a.v, b.v);
}

// A derived operand in the pieces that its products take
template <typename T, int kParts> struct Derived { float v[8]; };
template <int kParts> struct Derived<__nv_bfloat16, kParts> { uint32_t r[kParts][4]; };
template <typename T, int kParts> __device__ __forceinline__ Derived<T, kParts> derive(const float (&v)[8]) {
    Derived<T, kParts> d;
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        float rest[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) rest[i] = v[i];
#pragma unroll
        for (int p = 0; p < kParts; ++p)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                d.r[p][i] = Half2Of<T>::pack(rest[2 * i], rest[2 * i + 1]);
                if (p + 1 < kParts) {
                    const float2 f = Half2Of<T>::unpack(d.r[p][i]);
                    rest[2 * i] -= f.x; rest[2 * i + 1] -= f.y;
                }
            }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) d.v[i] = v[i];
    }
    return d;
}
// derived times exact
template <typename T, int kParts> __device__ __forceinline__ void mma_derived(float (&c)[4], const Derived<T, kParts>& a, const OpB<T>& b) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
#pragma unroll
        for (int p = kParts - 1; p >= 0; --p) MmaK16<T>::run(c, a.r[p], b.r);
    } else {
        float w[4];
        values(b, w);
        if constexpr (sizeof(T) == 4) mma_values<2, 2, false>(c, a.v, w);
        else mma_values<kParts, 1>(c, a.v, w);
    }
}

// A derived matrix in shared memory: bf16 planes of its pieces beside bf16, fp32 beside the others
template <typename T> struct Plane { using type = float; static constexpr bool kSplit = false; };
template <> struct Plane<__nv_bfloat16> { using type = __nv_bfloat16; static constexpr bool kSplit = true; };
// c0, c1 += exact A times columns n0 .. n0+15 of it; `plane`: elements between two pieces
template <typename T, int kParts, bool kStoredK>
__device__ __forceinline__ void mma_plane2(float (&c0)[4], float (&c1)[4], const OpA<T>& a, const typename Plane<T>::type* s, int plane, int ld, int n0, int k0, int lane) {
    if constexpr (Plane<T>::kSplit) {
#pragma unroll
        for (int p = kParts - 1; p >= 0; --p) {
            OpB<T> b0, b1;
            load_b2<kStoredK>(b0, b1, s + p * plane, ld, n0, k0, lane);
            MmaK16<T>::run(c0, a.r, b0.r);
            MmaK16<T>::run(c1, a.r, b1.r);
        }
    } else {
        OpB<float> b0, b1;
        load_b2<kStoredK>(b0, b1, s, ld, n0, k0, lane);
        float v[8];
        values(a, v);
        constexpr int kA = sizeof(T) == 4 ? 2 : 1, kB = sizeof(T) == 4 ? 2 : kParts;
        mma_values<kA, kB>(c0, v, b0.v);
        mma_values<kA, kB>(c1, v, b1.v);
    }
}
// derived A out of shared memory (one piece) times exact
template <typename T> __device__ __forceinline__ void mma_plane_a(float (&c)[4], const OpA<typename Plane<T>::type>& a, const OpB<T>& b) {
    if constexpr (Plane<T>::kSplit) MmaK16<T>::run(c, a.r, b.r);
    else {
        float w[4];
        values(b, w);
        mma_values<sizeof(T) == 4 ? 2 : 1, sizeof(T) == 4 ? 2 : 1>(c, a.v, w);
    }
}
// two neighbouring values into the planes
template <typename T, int kParts> __device__ __forceinline__ void put2(typename Plane<T>::type* s, int plane, float a, float b) {
    if constexpr (Plane<T>::kSplit) {
#pragma unroll
        for (int p = 0; p < kParts; ++p) {
            const uint32_t w = Half2Of<__nv_bfloat16>::pack(a, b);
            *reinterpret_cast<uint32_t*>(s + p * plane) = w;
            const float2 f = Half2Of<__nv_bfloat16>::unpack(w);
            a -= f.x; b -= f.y;
        }
    } else {
        *reinterpret_cast<float2*>(s) = make_float2(a, b);
    }
}

// `kRows` x `kCols` elements of row-major global memory, rows `stride` elements apart, into shared memory; rows from `rows` on and columns
// from `cols` on come as zeros.  vec: rows start on 16 bytes (copies are asynchronous then: cp.async.wait before use).
template <typename T, int kRows, int kCols>
__device__ __forceinline__ void fetch_rows(T* dst, int ld, const T* src, long long stride, int rows, int cols, bool vec, int tid, int threads) {
    if (vec) {
        constexpr int E = 16 / (int)sizeof(T), P = kCols / E;
        for (int i = tid; i < kRows * P; i += threads) {
            const int r = i / P, c = (i % P) * E;
            const int left = r < rows ? (cols - c) * (int)sizeof(T) : 0, n = left < 0 ? 0 : left > 16 ? 16 : left;
            const T* p = n > 0 ? src + r * stride + c : src;
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst + r * ld + c)), "l"(p), "r"(n) : "memory");
        }
    } else {
        for (int i = tid; i < kRows * kCols; i += threads) {
            const int r = i / kCols, c = i % kCols;
            dst[r * ld + c] = r < rows && c < cols ? src[r * stride + c] : from_f<T>(0.f);
        }
    }
}
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft = 0> __device__ __forceinline__ void wait_copies() { asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory"); }

}  // namespace mt
}  // namespace ss2d
