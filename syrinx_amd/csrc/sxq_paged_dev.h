// sxq_paged_dev.h -- device helpers that the paged cache's kernels share: searches in offsets,
// vectors of four elements as f32, and the codes of 8-bit pages.
#pragma once
#include "sxq_paged_launch.h"

namespace sxq {

// The last i with first[i] <= j, over n ascending firsts (first[0] <= j); for U values of j at
// once, so that the steps' LDS (or L2) reads overlap.
template <int U>
SXQ_DEV void owners(const int* first, int n, const int (&j)[U], int (&i)[U]) {
#pragma unroll
    for (int u = 0; u < U; ++u) i[u] = 0;
    for (int step = n > 1 ? 1 << (31 - __builtin_clz(n - 1)) : 0; step; step >>= 1)
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i[u] + step < n && first[i[u] + step] <= j[u]) i[u] += step;
}
SXQ_DEV int owner(const int* first, int n, int j) {
    const int jj[1] = {j};
    int i[1];
    owners(first, n, jj, i);
    return i[0];
}

// The same by a whole wave for one j: 64 offsets a step.
SXQ_DEV int wave_owner(const int* first, int n, int j) {
    const int lane = threadIdx.x & 63;
    int lo = 0;
    while (n > 1) {
        const int step = (n + 63) / 64, at = lane * step;
        const int k = __builtin_popcountll(__ballot(at < n && first[lo + min(at, n - 1)] <= j)) - 1;
        lo += k * step;
        n = min(step, n - k * step);
    }
    return lo;
}

// Four consecutive elements as f32, at any element's alignment, and back.
template <typename T>
SXQ_DEV void load4(const T* p, float* f) {
    typedef T v4 __attribute__((ext_vector_type(4), aligned(sizeof(T))));
    const v4 v = *(const v4*)p;
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = to_f32(v[e]);
}
template <typename T>
SXQ_DEV void store4(T* p, const float* f) {
    typedef T v4 __attribute__((ext_vector_type(4), aligned(sizeof(T))));
    v4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = from_f32<T>(f[e]);
    *(v4*)p = v;
}

// ---- 8-bit codes ---------------------------------------------------------------------------
struct I8 {
    static constexpr bool kNan = false;
    static constexpr float kTop = 127.0f;
    static constexpr int kTopExp = 6;           // 127 = 1.984375 * 2^6
    static constexpr uint32_t kTopMant = 0x7E0000u;
    // Four codes, byte e of the result the code of x[e] (already divided by the scale): nearest,
    // ties to even; beyond the largest code, the largest; NaN as 0.
    static SXQ_DEV uint32_t pack(const float* x) {
        uint32_t b[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float c = __builtin_amdgcn_fmed3f(x[e], -kTop, kTop);
            b[e] = (uint32_t)(int)rintf(x[e] == x[e] ? c : 0.0f);
        }
        return __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[3], b[2], 0x0C0C0400), __builtin_amdgcn_perm(b[1], b[0], 0x0C0C0400),
                                     0x05040100);
    }
    static SXQ_DEV void unpack(uint32_t w, float* x) {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = (float)(int8_t)(w >> (8 * e));
    }
};
struct E4M3 {
    static constexpr bool kNan = true;
    static constexpr float kTop = 448.0f;
    static constexpr int kTopExp = 8;           // 448 = 1.75 * 2^8
    static constexpr uint32_t kTopMant = 0x600000u;
    // as I8::pack; NaN as the code's NaN
    static SXQ_DEV uint32_t pack(const float* x) {
        float c[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            c[e] = __builtin_amdgcn_fmed3f(x[e], -kTop, kTop);
            c[e] = x[e] == x[e] ? c[e] : x[e];
        }
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(c[0], c[1], 0, false);
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c[2], c[3], w, true);
    }
    static SXQ_DEV void unpack(uint32_t w, float* x) {
        typedef float f2 __attribute__((ext_vector_type(2)));
        const f2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
        x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
    }
};
constexpr int kMinScaleExp = -100;
// The smallest 2^e, e >= kMinScaleExp, with amax <= C::kTop * 2^e; amax finite, 0 or more.  With
// amax = f 2^E, 1 <= f < 2: e = E - kTopExp, one more where f passes the top's own fraction.
template <typename C>
SXQ_DEV float block_scale(float amax) {
    const uint32_t u = __float_as_uint(amax);
    const int e = max((int)(u >> 23) - 127 - C::kTopExp + ((u & 0x7FFFFFu) > C::kTopMant ? 1 : 0), kMinScaleExp);
    return __uint_as_float((uint32_t)(e + 127) << 23);
}

}  // namespace sxq
