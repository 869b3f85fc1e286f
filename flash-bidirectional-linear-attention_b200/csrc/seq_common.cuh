// Device helpers shared by the sequence operators beside the attention passes: rotary positions
// (rotary.cu), the short causal convolution (causal_conv.cu) and the selective scan
// (selective_scan.cu).
#pragma once

#include "fbla_common.cuh"
#include "tc_kernels.cuh"

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


// Two fp32 values in one 64-bit register: one instruction for two multiply-adds.  The rate of the multiply-add
// units is the same (128 per clock and SM measured either way), half of the issue slots are left to others.
struct F2 {
    unsigned long long v;
    __device__ __forceinline__ F2() {}
    __device__ __forceinline__ F2(float x, float y) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y)); }
    __device__ __forceinline__ explicit F2(float x) : F2(x, x) {}
    __device__ __forceinline__ void get(float& x, float& y) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
    __device__ __forceinline__ float x() const { float a, b; get(a, b); return a; }
    __device__ __forceinline__ float y() const { float a, b; get(a, b); return b; }
};
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
    F2 r;
    asm("fma.rn.ftz.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
    F2 r;
    asm("mul.rn.ftz.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float rcp(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// 1 / (1 + e^-x).  16-bit results: by the special functions, off by at most 2^-21 absolute and, for x > -16, 2^-19 relative.
// With u = 2^-24: e^-x has the relative error of ex2.approx (4 u) and of its argument (1.3 |x| u), the result that times
// 1 - sigmoid (at most 1.1 u absolute for every x), and the sum and rcp.approx add 3 u.  Far below their rounding.
template <typename T> __device__ __forceinline__ float sigmoid(float x) { return rcp(1.f + ex2(x * -1.44269504f)); }
template <> __device__ __forceinline__ float sigmoid<float>(float x) { return __frcp_rn(1.f + exp_of(-x)); }

// log(1 + e^v) of two values: max(v, 0) + log1p(w) with w = e^-|v| in (0, 1], and log1p(w) = 2 atanh(w / (2 + w))
// as its series in s = w / (2 + w) <= 1/3 (the first term left out is s^14 / 15 = 1.4e-8 relative).  e^-|v| is the
// special function unit's 2^x; what rounding |v| log2(e) loses (2^-24 of up to 150) comes back as a factor.
// About 3 units in the last place.
__device__ __forceinline__ F2 softplus2(float v0, float v1) {
    const F2 m(!(v0 <= 0.f) ? v0 : 0.f, !(v1 <= 0.f) ? v1 : 0.f);      // a NaN stays
    const F2 a(fminf(fabsf(v0), 104.f), fminf(fabsf(v1), 104.f));      // e^-104 is 0 in fp32
    const F2 x = mul2(a, F2(1.44269504f));
    F2 lost = fma2(a, F2(-1.44269504f), x);
    lost = fma2(a, F2(-1.92596299e-8f), lost);
    const F2 e(ex2(-x.x()), ex2(-x.y()));
    const F2 w = fma2(mul2(e, F2(0.69314718f)), lost, e);
    const F2 den = fma2(w, F2(1.f), F2(2.f));
    const F2 s = mul2(w, F2(rcp(den.x()), rcp(den.y()))), t = mul2(s, s);
    F2 p(2.f / 13.f);
    p = fma2(p, t, F2(2.f / 11.f));
    p = fma2(p, t, F2(2.f / 9.f));
    p = fma2(p, t, F2(2.f / 7.f));
    p = fma2(p, t, F2(2.f / 5.f));
    p = fma2(p, t, F2(2.f / 3.f));
    p = fma2(p, t, F2(2.f));
    return fma2(p, s, m);
}
__device__ __forceinline__ float softplus(float v) { return softplus2(v, 0.f).x(); }

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

// ---- host side ------------------------------------------------------------------------------------

// Like every launching call: not after another one gave up a bounded wait, whose results may be what this one is given.
inline int check_device_status() {
    const int site = fbla::tc_device_status();
    if (site == 0) return FBLA_OK;
    return fbla::api_fail(FBLA_ERR_DEVICE, "a kernel gave up a bounded wait (site %d); results are invalid", site);
}

inline bool aligned_to(const void* p, int64_t bytes) { return (reinterpret_cast<uintptr_t>(p) % (uintptr_t)bytes) == 0; }

}  // namespace seq
}  // namespace fbla
