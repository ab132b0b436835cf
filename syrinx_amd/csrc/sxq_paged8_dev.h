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

// A query's matrix type, and into how many parts its elements are cut: an f32 row, times the power of two
// that takes its largest element to 2^14 .. 2^15, into two of f16 (off by at most 2^-22 of the element, or
// 2^-39 of the row's largest).
template <typename TQ>
struct Query {
    typedef TQ M;
    static constexpr int kQP = 1;
};
template <>
struct Query<float> {
    typedef _Float16 M;
    static constexpr int kQP = 2;
};
// What a row's products with a block's codes are to be multiplied by: the row's factor times the keys'
// scale; of an f32 row never too large or too small for an f32 (its power of two and a scale may be 2^200
// together, or 2^-200): infinity times a product of zero, or zero times an infinite one, would be NaN.
template <typename TQ>
SXQ_DEV float score_factor(float row, float scale) {
    const float f = row * scale;
    if constexpr (Query<TQ>::kQP == 1) return f;
    else return __builtin_copysignf(__builtin_amdgcn_fmed3f(fabsf(f), 0x1p-126f, 0x1.fffffep127f), f);
}
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

// The operands of one lane's share of a row, N times eight elements from q + cols[i] on (in[i]: within the
// head), and what the row's products are to be multiplied by.  all_lanes takes a lane's largest to the
// row's.
template <typename TQ, int N, typename V8, typename Reduce>
SXQ_DEV float load_query(const TQ* q, const int (&cols)[N], const bool (&in)[N], V8 (&out)[Query<TQ>::kQP][N], Reduce all_lanes) {
    if constexpr (Query<TQ>::kQP == 1) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            v4u v = *(const v4u*)(q + (in[i] ? cols[i] : 0));
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = in[i] ? v[e] : 0;
            out[0][i] = __builtin_bit_cast(V8, v);
        }
        return 1.0f;
    } else {
        float f[N][8], most = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const TQ* src = q + (in[i] ? cols[i] : 0);
            *(v4f*)f[i] = *(const v4f*)src;
            *(v4f*)(f[i] + 4) = *(const v4f*)(src + 4);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                f[i][e] = in[i] ? f[i][e] : 0.0f;
                const float a = fabsf(f[i][e]);
                most = a < INFINITY ? fmaxf(most, a) : most;
            }
        }
        most = all_lanes(most);
        // 2^(14 - E) of the largest, 2^E and up (E at least -112, which 2^126 takes to 2^14)
        const int up = 14 - max((int)(__float_as_uint(most) >> 23) - 127, -112);
        const float by = __uint_as_float((uint32_t)(up + 127) << 23);
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float v = f[i][e] * by;
                const _Float16 hi = (_Float16)v;
                out[0][i][e] = hi;
                const float rest = v - (float)hi;
                out[1][i][e] = (_Float16)(rest == rest ? rest : 0.0f);  // (an infinity has none)
            }
        return __uint_as_float((uint32_t)(127 - up) << 23);
    }
}

}  // namespace
}  // namespace sxq
