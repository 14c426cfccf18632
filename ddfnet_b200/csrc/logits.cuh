// What the kernels over rows of logits share (top_logits.cu, distill.cu): a row as 16-byte granules,
// the running maximum and sum of a softmax, and their combination over a block.
//
// A row of V elements starts at any element.  It is read as whole aligned 16-byte granules; the elements
// of the first and last granule that lie outside the row are masked.  (A granule never straddles two
// allocations, so the masked elements are readable.)
//
// Sums of exponentials are kept in base 2 and relative to the largest element m: with c = log2(e) / T the
// summand is 2^((x - m) c).  The difference comes first: (x c) - (m c) would overflow for masks of float's
// lowest value, and round at the size of m c instead of at the size of the difference.
#pragma once

#include "common.cuh"

namespace ddf {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kMaxTop = 256;  // entries of a row's list of top logits: one thread of a block each

__device__ __forceinline__ float neg_inf() { return __int_as_float(0xff800000); }

// Larger of two, NaN if either is (fmaxf drops NaN).
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

template <typename T> struct Granule {
    static constexpr int N = 16 / (int)sizeof(T);
    static __device__ __forceinline__ void get(const uint4& g, float (&x)[N]) {
        const uint32_t w[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = Word<T>::get(w[i / Word<T>::EPW], i % Word<T>::EPW);
    }
    static __device__ __forceinline__ uint4 put(const float (&x)[N]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[i] = Word<T>::put(x[i * Word<T>::EPW], x[i * Word<T>::EPW + Word<T>::EPW - 1]);
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};

// A run of `len` elements of a row as granules: element i of the run is element (i + phase) of the granules.
template <typename T> struct Run {
    const char* base;  // of the first granule
    int phase, len, granules;
    __device__ __forceinline__ Run(const T* p, int len_) : len(len_) {
        const unsigned long long a = reinterpret_cast<unsigned long long>(p);
        base = reinterpret_cast<const char*>(a & ~15ull);
        phase = (int)(a & 15ull) / (int)sizeof(T);
        granules = (phase + len + Granule<T>::N - 1) / Granule<T>::N;
    }
    __device__ __forceinline__ uint4 load(int g) const { return ld_granule(base + (long long)g * 16); }
    // Bits of granule g's elements that lie outside the run.
    __device__ __forceinline__ uint32_t outside(int g) const {
        constexpr int N = Granule<T>::N;
        uint32_t m = 0;
        if (g == 0) m = (1u << phase) - 1u;
        const int end = phase + len - g * N;  // elements up to the run's end
        if (end < N) m |= ((1u << N) - 1u) & ~((1u << (end < 0 ? 0 : end)) - 1u);
        return m;
    }
};

// Sum of 2^((x - m) c) over the elements x so far, m the largest of them.  Nothing yet, or nothing above
// -inf: m = -inf, s = 0, and `ref`, which stands for m in differences, 0.  A NaN or +inf makes s NaN for good.
struct Online {
    float m, ref, s;
    static __device__ __forceinline__ Online none() { return Online{neg_inf(), 0.f, 0.f}; }
    __device__ __forceinline__ void raise(float x, float c) {
        s = m == neg_inf() ? 0.f : s * ex2((ref - x) * c);
        m = ref = x;
    }
    // `most` is the largest of x[], or NaN if one is.  Masked elements are -inf.
    template <int N> __device__ __forceinline__ void add(const float (&x)[N], float most, float c) {
        if (!(most <= m)) raise(most, c);
        const unsigned long long r2 = f2_pack(-ref, -ref), c2 = f2_pack(c, c);
        float t0 = 0.f, t1 = 0.f;
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            float a, b;
            f2_unpack(f2_mul(f2_add(f2_pack(x[i], x[i + 1]), r2), c2), a, b);
            t0 += ex2(a);
            t1 += ex2(b);
        }
        s += t0 + t1;
    }
    __device__ __forceinline__ void merge(const Online& o, float c) {
        if (o.s == 0.f) return;
        if (s == 0.f) {
            *this = o;
        } else if (!(o.m <= m)) {
            s = o.s + s * ex2((ref - o.ref) * c);
            m = o.m;
            ref = o.ref;
        } else {
            s += o.s * ex2((o.ref - ref) * c);
        }
    }
};

__device__ __forceinline__ Online warp_merge(Online o, float c) {
#pragma unroll
    for (int d = 16; d; d >>= 1) {
        Online p;
        p.m = __shfl_xor_sync(~0u, o.m, d);
        p.ref = __shfl_xor_sync(~0u, o.ref, d);
        p.s = __shfl_xor_sync(~0u, o.s, d);
        o.merge(p, c);
    }
    return o;
}

// Over the block; every thread gets the result.  `room`: one Online for each warp.
template <int WARPS> __device__ __forceinline__ Online block_merge(Online o, float c, Online* room) {
    o = warp_merge(o, c);
    if ((threadIdx.x & 31) == 0) room[threadIdx.x >> 5] = o;
    __syncthreads();
    Online all = Online::none();
#pragma unroll
    for (int w = 0; w < WARPS; ++w) all.merge(room[w], c);
    return all;
}

__device__ __forceinline__ float warp_max_nan(float v) {
#pragma unroll
    for (int d = 16; d; d >>= 1) v = max_nan(v, __shfl_xor_sync(~0u, v, d));
    return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(~0u, v, d);
    return v;
}

}  // namespace ddf
