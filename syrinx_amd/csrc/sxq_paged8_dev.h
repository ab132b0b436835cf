// sxq_paged8_dev.h -- the 8-bit cache's codes, and its queries, as operands of the matrix cores.
#pragma once
#include "sxq_paged_dev.h"

namespace sxq {
namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

// ---- codes as matrix operands ------------------------------------------------------------
// Both codes are exact in bf16 (int8: seven bits and a sign; e4m3: four bits) and in f16.
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));

template <typename C, typename M>
struct Operand;
template <>
struct Operand<E4M3, __bf16> {
    // elements 2 hi and 2 hi + 1 of w
    template <bool HI>
    static SXQ_DEV uint32_t two(uint32_t w) {
        return __builtin_bit_cast(uint32_t, (v2bf)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HI));
    }
    static SXQ_DEV v4u eight(uint32_t a, uint32_t b) { return (v4u){two<false>(a), two<true>(a), two<false>(b), two<true>(b)}; }
    // out[c]: byte c of a (lower half) and of b
    static SXQ_DEV void columns(uint32_t a, uint32_t b, uint32_t* out) {
        const uint32_t lo = __builtin_amdgcn_perm(b, a, 0x05010400), hi = __builtin_amdgcn_perm(b, a, 0x07030602);
        out[0] = two<false>(lo), out[1] = two<true>(lo), out[2] = two<false>(hi), out[3] = two<true>(hi);
    }
};
template <>
struct Operand<E4M3, _Float16> {
    template <bool HI>
    static SXQ_DEV uint32_t two(uint32_t w) {
        return __builtin_bit_cast(uint32_t, (v2h)__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HI));
    }
    static SXQ_DEV v4u eight(uint32_t a, uint32_t b) { return (v4u){two<false>(a), two<true>(a), two<false>(b), two<true>(b)}; }
};
template <>
struct Operand<I8, __bf16> {
    template <int E>
    static SXQ_DEV uint32_t bits(uint32_t w) {
        return __float_as_uint((float)(int8_t)(w >> (8 * E)));
    }
    // (the upper halves of two f32, exact)
    static SXQ_DEV uint32_t pack(uint32_t lo, uint32_t hi) { return __builtin_amdgcn_perm(hi, lo, 0x07060302); }
    static SXQ_DEV v4u eight(uint32_t a, uint32_t b) {
        return (v4u){pack(bits<0>(a), bits<1>(a)), pack(bits<2>(a), bits<3>(a)), pack(bits<0>(b), bits<1>(b)), pack(bits<2>(b), bits<3>(b))};
    }
    static SXQ_DEV void columns(uint32_t a, uint32_t b, uint32_t* out) {
        out[0] = pack(bits<0>(a), bits<0>(b)), out[1] = pack(bits<1>(a), bits<1>(b));
        out[2] = pack(bits<2>(a), bits<2>(b)), out[3] = pack(bits<3>(a), bits<3>(b));
    }
};
template <>
struct Operand<I8, _Float16> {
    // 0x6400 | b is 1024 + b: with the code's sign bit turned, b - 128 is the code
    static SXQ_DEV uint32_t two(uint32_t w, uint32_t sel) {
        const v2h v = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, w, sel));
        return __builtin_bit_cast(uint32_t, v - (v2h){(_Float16)1152.0f, (_Float16)1152.0f});
    }
    static SXQ_DEV v4u eight(uint32_t a, uint32_t b) {
        a ^= 0x80808080u, b ^= 0x80808080u;
        return (v4u){two(a, 0x04010400), two(a, 0x04030402), two(b, 0x04010400), two(b, 0x04030402)};
    }
};

// A query's matrix type, and into how many bf16 parts its elements and the weights are cut.
template <typename TQ>
struct Query {
    typedef TQ M;
    static constexpr int kQP = 1, kWP = 2;
};
template <>
struct Query<float> {
    typedef __bf16 M;
    static constexpr int kQP = 3, kWP = 3;
};
template <typename M>
struct Vec8;
template <>
struct Vec8<__bf16> {
    typedef v8bf T;
};
template <>
struct Vec8<_Float16> {
    typedef v8h T;
};

// Eight elements of a query as QP operands of 8 (parts of an f32 element sum to it exactly; what
// passes bf16's range is infinite, its further parts zero).
template <typename TQ, int QP>
SXQ_DEV void query_parts(const TQ* src, bool in, v4u (&out)[QP]) {
    if constexpr (QP == 1) {
        const v4u v = *(const v4u*)src;
#pragma unroll
        for (int e = 0; e < 4; ++e) out[0][e] = in ? v[e] : 0;
    } else {
        float f[8];
        *(v4f*)f = *(const v4f*)src;
        *(v4f*)(f + 4) = *(const v4f*)(src + 4);
#pragma unroll
        for (int q = 0; q < QP; ++q) {
            v8bf part;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                part[e] = (__bf16)(in ? f[e] : 0.0f);
                const float p = (float)part[e];
                f[e] = fabsf(p) < INFINITY ? f[e] - p : p == p ? 0.0f : p;
            }
            out[q] = __builtin_bit_cast(v4u, part);
        }
    }
}

}  // namespace
}  // namespace sxq
