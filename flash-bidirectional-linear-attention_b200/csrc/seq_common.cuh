// Device helpers shared by the sequence operators beside the attention passes: rotary positions
// (rotary.cu), the short causal convolution (causal_conv.cu) and the selective scan
// (selective_scan.cu).
#pragma once

#include "fbla_common.cuh"

namespace fbla {
namespace seq {

// ---- V consecutive elements in one access ---------------------------------------------------------
// The caller has made sure that the address is a multiple of V elements.
template <int BYTES> struct Raw;
template <> struct Raw<2> { using type = unsigned short; };
template <> struct Raw<4> { using type = unsigned int; };
template <> struct Raw<8> { using type = uint2; };
template <> struct Raw<16> { using type = uint4; };

template <typename T, int V> struct Pack {
    static constexpr int kBytes = (int)sizeof(T) * V;
    static constexpr int kWord = kBytes > 16 ? 16 : kBytes;     // one access is 16 bytes at most
    static constexpr int kWords = kBytes / kWord;
    using R = typename Raw<kWord>::type;
    union {
        R r[kWords];
        T e[V];
    };
    __device__ __forceinline__ Pack() {}
    __device__ __forceinline__ void load(const T* p) {
#pragma unroll
        for (int i = 0; i < kWords; ++i) r[i] = reinterpret_cast<const R*>(p)[i];
    }
    // Streaming: read once, so L1 need not keep it.
    __device__ __forceinline__ void load_stream(const T* p) {
#pragma unroll
        for (int i = 0; i < kWords; ++i) r[i] = __ldcs(reinterpret_cast<const R*>(p) + i);
    }
    __device__ __forceinline__ void store(T* p) const {
#pragma unroll
        for (int i = 0; i < kWords; ++i) reinterpret_cast<R*>(p)[i] = r[i];
    }
    __device__ __forceinline__ void store_stream(T* p) const {
#pragma unroll
        for (int i = 0; i < kWords; ++i) __stcs(reinterpret_cast<R*>(p) + i, r[i]);
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < V; ++i) e[i] = from_f<T>(0.f);
    }
    __device__ __forceinline__ float get(int i) const { return to_f<T>(e[i]); }
    __device__ __forceinline__ void set(int i, float x) { e[i] = from_f<T>(x); }
};

// ---- elementary functions -------------------------------------------------------------------------
// The library is compiled with approximate division and exponentials; where an error of a few units
// in the last place would show in an fp32 result these are used instead.

// e^x to about one unit in the last place: x = n ln2 + r with |r| <= ln2 / 2 (ln2 in two parts after Cody
// and Waite), Taylor of degree 7 for e^r (next term (0.3466)^8 / 8! = 5e-9), times 2^n in two factors so
// that neither leaves the range.
__device__ __forceinline__ float exp_full(float x) {
    x = fminf(fmaxf(x, -104.f), 89.f);      // below: 0 in fp32; above: infinity
    const float n = rintf(x * 1.44269504f);
    float r = fmaf(n, -0.693359375f, x);    // ln2 = 0.693359375 - 2.12194440e-4 (the first is exact in 10 bits)
    r = fmaf(n, 2.12194440e-4f, r);
    float p = 1.f / 5040.f;
    p = fmaf(p, r, 1.f / 720.f);
    p = fmaf(p, r, 1.f / 120.f);
    p = fmaf(p, r, 1.f / 24.f);
    p = fmaf(p, r, 1.f / 6.f);
    p = fmaf(p, r, 0.5f);
    p = fmaf(p, r, 1.f);
    p = fmaf(p, r, 1.f);
    const int k = (int)n, k1 = k >> 1;
    return p * __int_as_float((k1 + 127) << 23) * __int_as_float((k - k1 + 127) << 23);
}

// A NaN goes through fminf / fmaxf as the other operand: keep it.
__device__ __forceinline__ float exp_of(float x) { return x != x ? x : exp_full(x); }

// 1 / (1 + e^-x); for 16-bit results the approximate exponential (2^-22 relative) is far below the rounding.
template <typename T> __device__ __forceinline__ float sigmoid(float x) { return __fdividef(1.f, 1.f + __expf(-x)); }
template <> __device__ __forceinline__ float sigmoid<float>(float x) { return __frcp_rn(1.f + exp_of(-x)); }

// ---- packed sequences -----------------------------------------------------------------------------
// Sequence s owns tokens [cu[s], cu[s+1]).
struct SeqSpan {
    int s;              // sequence of a token, -1 when no sequence owns it
    int64_t lo, hi;     // its first token and its end
};

// Only compares with cu and indexes inside it, whatever it holds.
__device__ __forceinline__ SeqSpan seq_of(const int32_t* cu, int n, int64_t t) {
    int a = 0, b = n + 1;           // first index with cu[i] > t lies in [a, b]
    while (a < b) {
        const int m = (a + b) >> 1;
        if ((int64_t)cu[m] > t) b = m; else a = m + 1;
    }
    SeqSpan r;
    if (a == 0 || a > n) {          // before the first sequence, or behind the last
        r.s = -1;
        r.lo = t;
        r.hi = a == 0 ? (int64_t)cu[0] : INT64_MAX;
    } else {
        r.s = a - 1;
        r.lo = cu[a - 1] > 0 ? cu[a - 1] : 0;
        r.hi = cu[a];
    }
    return r;
}

// ---- sums over rows -------------------------------------------------------------------------------
// out[i] = sum over r of in[r * n + i], rows in order: how per-block partial sums become one gradient
// with the same bits on every run.
cudaError_t sum_rows(const float* in, int64_t rows, int64_t n, int out_dtype, void* out, cudaStream_t st);

inline bool aligned_to(const void* p, int64_t bytes) { return (reinterpret_cast<uintptr_t>(p) % (uintptr_t)bytes) == 0; }

}  // namespace seq
}  // namespace fbla
