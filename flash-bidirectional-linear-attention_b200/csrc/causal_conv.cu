// Short causal convolution over tokens, one filter of W taps per channel:
//
//   p[t,c] = bias[c] + sum_j w[c,j] x[t-W+1+j, c],     y = p  or  y = p sigmoid(p)
//
// Tokens before a sequence come from its initial state (the last W-1 inputs of what went before) or are
// zero.  Gradients, with g = dy y'(p):
//   dx[t] = sum_j w[j] g[t+W-1-j],   dw[j] = sum_t g[t] x[t-W+1+j],   dbias = sum_t g[t]
//
// What bounds it: HBM (forward one read and one write, backward two reads and one write).  Channels are
// the contiguous dimension, so a thread owns V channels and walks along the tokens with the last W-1
// inputs (and, backward, the last W-1 gradients) in registers: x is read once, plus W-1 tokens per run.
// Tokens go by in groups of four, and the groups to come are on their way (Ring below).  Measured at
// B8-T4096-C2048, 4 taps, silu, bf16: forward 53 us (5.1 TB/s), backward 109 us and 7 for the sum of the weight
// gradient (3.5 TB/s); with one load in flight per thread 124 and 298, with a group's loads in registers, where the
// compiler decides what is waited for together, 66 and 214.
// Two channels share the packed fp32 instructions: in plain ones the arithmetic (W products per element forward,
// 3 W + 1 backward, a sigmoid) takes as long as the memory.  The weight gradient is summed in registers over a
// thread's run, in shared memory over the runs of a block, and then over the blocks by a kernel of its own: no atomics,
// the same bits on every run.
#include <type_traits>

#include "seq_common.cuh"

namespace {

using fbla::from_f;
using fbla::to_f;
using fbla::seq::F2;
using fbla::seq::fma2;
using fbla::seq::mul2;
using fbla::seq::Pack;
using fbla::seq::seq_of;
using fbla::seq::SeqSpan;

struct ConvParams {
    int batch, channels, silu, w32, num_seqs;
    int64_t len;
    int64_t xs[2], gs[2];       // batch and token strides of x and of dy, in elements
    const int32_t* cu;
    int run;                    // tokens a thread walks over
    const void *w, *bias;       // w (channels, W), bias (channels) or NULL; fp32 when w32, else the type of x
};

__device__ __forceinline__ SeqSpan span_of(const ConvParams& p, int64_t b, int64_t t) {
    if (p.cu != nullptr) return seq_of(p.cu, p.num_seqs, t);
    SeqSpan s;
    s.s = (int)b;
    s.lo = 0;
    s.hi = p.len;
    return s;
}

// V channels as pairs; with one channel the second half of the pair is idle
template <int V> struct Lanes {
    static constexpr int P = (V + 1) / 2;
    F2 v[P];
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < P; ++i) v[i] = F2(0.f);
    }
    template <typename T> __device__ __forceinline__ void from(const Pack<T, V>& p) {
#pragma unroll
        for (int i = 0; i < P; ++i) v[i] = F2(p.get(2 * i), 2 * i + 1 < V ? p.get(2 * i + 1 < V ? 2 * i + 1 : 0) : 0.f);
    }
    template <typename T> __device__ __forceinline__ void to(Pack<T, V>& p) const {
#pragma unroll
        for (int i = 0; i < P; ++i) {
            p.set(2 * i, v[i].x());
            if (2 * i + 1 < V) p.set(2 * i + 1 < V ? 2 * i + 1 : 0, v[i].y());
        }
    }
};

// Input of token u (which may lie before its sequence: initial state, or zero), V channels from c.
template <typename T, int W, int V>
__device__ __forceinline__ Lanes<V> input_of(const ConvParams& p, const T* x, const T* init, const SeqSpan& s, int64_t b, int64_t u, int c) {
    Pack<T, V> v;
    if (u >= s.lo && s.s >= 0) {
        v.load(x + b * p.xs[0] + u * p.xs[1] + c);
    } else if (init != nullptr && s.s >= 0) {
        v.load(init + ((int64_t)s.s * (W - 1) + (W - 1 + (u - s.lo))) * p.channels + c);
    } else {
        v.zero();
    }
    Lanes<V> r;
    r.from(v);
    return r;
}

template <typename T> __device__ __forceinline__ F2 sigmoid2(F2 x) {
    return F2(fbla::seq::sigmoid<T>(x.x()), fbla::seq::sigmoid<T>(x.y()));
}
template <typename T, bool SILU> __device__ __forceinline__ F2 activate(F2 x) { return SILU ? mul2(x, sigmoid2<T>(x)) : x; }

// dy times the slope of the activation at x: silu'(x) = s (1 + x (1 - s)), s = sigmoid(x)
template <typename T, bool SILU> __device__ __forceinline__ F2 pre_grad(F2 dy, F2 x) {
    if (!SILU) return dy;
    const F2 s = sigmoid2<T>(x);
    return mul2(mul2(dy, s), fma2(x, fma2(s, F2(-1.f), F2(1.f)), F2(1.f)));
}

constexpr int U = 4;            // tokens of a group
constexpr int kStages = 3;      // groups in the ring

// A thread's own tokens on their way from global memory: asynchronous copies into a ring of groups in shared
// memory, two groups ahead.  A slot is written and read by one thread only, so nothing but that thread's own wait
// orders it.  Copies are of 4 bytes or more; the one 2-byte case (odd channel counts of the 16-bit types) keeps
// the next group in registers.
template <typename T, int V> struct Ring {
    static constexpr int kBytes = (int)sizeof(T) * V;
    static constexpr bool kAsync = kBytes >= 4;
    static constexpr int kAhead = kAsync ? kStages - 1 : 1;
    static constexpr int kThreadBytes = kAsync ? kStages * U * kBytes : 0;
    const T* base;
    int64_t stride;
    uint32_t at;                // shared address of this thread's first slot
    Pack<T, V> regs[kAsync ? 1 : U];
    __device__ __forceinline__ Ring(const T* b, int64_t s, unsigned char* smem) : base(b), stride(s) {
        at = (uint32_t)__cvta_generic_to_shared(smem) + (threadIdx.y * blockDim.x + threadIdx.x) * kBytes;
    }
    __device__ __forceinline__ uint32_t slot(int stage, int k) const { return at + (stage * U + k) * 256 * kBytes; }
    // Tokens t .. t + U - 1 into `stage`, zeros from `end` on.
    __device__ __forceinline__ void fetch(int stage, int64_t t, int64_t end) {
        if constexpr (kAsync) {
#pragma unroll
            for (int k = 0; k < U; ++k) {
                const bool in = t + k < end;
                asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(slot(stage, k)),
                             "l"(base + (in ? t + k : 0) * stride), "n"(kBytes), "r"(in ? kBytes : 0) : "memory");
            }
        } else {
#pragma unroll
            for (int k = 0; k < U; ++k) {
                regs[k].zero();
                if (t + k < end) regs[k].load(base + (t + k) * stride);
            }
        }
    }
    __device__ __forceinline__ Pack<T, V> get(int stage, int k) const {
        Pack<T, V> r;
        if constexpr (!kAsync) {
            r = regs[k];
        } else if constexpr (kBytes == 4) {
            asm volatile("ld.shared.b32 %0, [%1];" : "=r"(*reinterpret_cast<uint32_t*>(&r)) : "r"(slot(stage, k)) : "memory");
        } else if constexpr (kBytes == 8) {
            uint32_t* w = reinterpret_cast<uint32_t*>(&r);
            asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(slot(stage, k)) : "memory");
        } else {
            uint32_t* w = reinterpret_cast<uint32_t*>(&r);
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                         : "r"(slot(stage, k)) : "memory");
        }
        return r;
    }
};
__device__ __forceinline__ void ring_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void ring_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Parameters of V channels
template <int W, int V> struct Filter {
    Lanes<V> w[W], bias;
    template <typename WT> __device__ __forceinline__ void load_as(const WT* wp, const WT* bp, int c) {
        Pack<WT, V> k[W], b;                // (V, W) consecutive elements
#pragma unroll
        for (int j = 0; j < W; ++j) k[j].load(wp + (int64_t)c * W + j * V);
        if (bp != nullptr) b.load(bp + c);
        else b.zero();
        bias.from(b);
#pragma unroll
        for (int j = 0; j < W; ++j) {
            Pack<WT, V> t;
#pragma unroll
            for (int i = 0; i < V; ++i) t.e[i] = k[(i * W + j) / V].e[(i * W + j) % V];
            w[j].from(t);
        }
    }
    template <typename T> __device__ __forceinline__ void load(const ConvParams& p, int c) {
        if (p.w32) load_as((const float*)p.w, (const float*)p.bias, c);
        else load_as((const T*)p.w, (const T*)p.bias, c);
    }
};

// A thread walks over its run piece by piece, a piece being the run's tokens of one sequence.
template <typename T, int W, int V, bool SILU>
__global__ void __launch_bounds__(256, 3) conv_fwd_kernel(const ConvParams p, const T* __restrict__ x, const T* __restrict__ init,
                                                          T* __restrict__ y) {
    constexpr int P = Lanes<V>::P;
    const int c = (blockIdx.x * blockDim.x + threadIdx.x) * V;
    const int64_t b = blockIdx.z;
    const int64_t t0 = ((int64_t)blockIdx.y * blockDim.y + threadIdx.y) * p.run;
    if (c >= p.channels || t0 >= p.len) return;
    const int64_t t1 = min(p.len, t0 + p.run);
    const T* xb = x + b * p.xs[0] + c;
    T* yb = y + b * p.len * p.channels + c;
    Filter<W, V> f;
    f.template load<T>(p, c);
    extern __shared__ __align__(16) unsigned char smem[];
    Ring<T, V> rx(xb, p.xs[1], smem);
    for (int64_t a = t0; a < t1;) {
        const SeqSpan s = span_of(p, b, a);
        const int64_t end = min(t1, s.hi);
        if (s.s < 0) {
            Pack<T, V> none;
            none.zero();
            for (; a < end; ++a) none.store(yb + a * p.channels);
            continue;
        }
#pragma unroll
        for (int i = 0; i < Ring<T, V>::kAhead; ++i) {
            rx.fetch(i, a + i * U, end);
            ring_commit();
        }
        Lanes<V> in[W - 1 + U];         // the last W-1 inputs, then the group's
#pragma unroll
        for (int j = 0; j < W - 1; ++j) in[j] = input_of<T, W, V>(p, x, init, s, b, a - (W - 1) + j, c);
        for (int stage = 0; a < end; a += U) {
            ring_wait<Ring<T, V>::kAhead - 1>();
#pragma unroll
            for (int k = 0; k < U; ++k) in[W - 1 + k].from(rx.get(stage, k));
            const int into = stage == 0 ? kStages - 1 : stage - 1;      // the slot read before this one
            rx.fetch(into, a + Ring<T, V>::kAhead * U, end);
            ring_commit();
            stage = stage == kStages - 1 ? 0 : stage + 1;
#pragma unroll
            for (int k = 0; k < U; ++k) {
                Lanes<V> o = f.bias;
#pragma unroll
                for (int i = 0; i < P; ++i) {
#pragma unroll
                    for (int j = 0; j < W; ++j) o.v[i] = fma2(f.w[j].v[i], in[k + j].v[i], o.v[i]);
                    o.v[i] = activate<T, SILU>(o.v[i]);
                }
                Pack<T, V> out;
                o.to(out);
                if (a + k < end) out.store(yb + (a + k) * p.channels);
            }
#pragma unroll
            for (int j = 0; j < W - 1; ++j) in[j] = in[j + U];
        }
        ring_wait<0>();                 // the zeros behind the piece's end: the next piece starts the ring anew
        a = end;
    }
}

// Last W-1 inputs of every sequence: row r is the input of token end - (W-1) + r.
template <typename T, int W>
__global__ void __launch_bounds__(256) conv_final_kernel(const ConvParams p, const T* __restrict__ x, const T* __restrict__ init,
                                                         T* __restrict__ fin) {
    const int c = blockIdx.x * blockDim.x + threadIdx.x;
    if (c >= p.channels) return;
    const int r = blockIdx.y;
    const int64_t q = blockIdx.z;
    const int64_t lo = p.cu != nullptr ? p.cu[q] : 0, hi = p.cu != nullptr ? p.cu[q + 1] : p.len;
    const int64_t b = p.cu != nullptr ? 0 : q;
    const int64_t u = hi - (W - 1) + r;
    T v = from_f<T>(0.f);
    if (u >= lo && u >= 0 && u < p.len) v = x[b * p.xs[0] + u * p.xs[1] + c];
    else if (u < lo && init != nullptr && W - 1 + (u - lo) >= 0) v = init[(q * (W - 1) + (W - 1 + (u - lo))) * p.channels + c];
    fin[(q * (W - 1) + r) * p.channels + c] = v;
}

// dx, and per block the sums for dw and dbias (part: [block of tokens][W + 1][channels]).
// The gradient g of a token reaches back to the W-1 inputs before it, so a piece is walked W-1 tokens beyond its
// end: those belong to the next run, or are zero where the sequence ends; only their g is needed here.
template <typename T, int W, int V, bool SILU>
__global__ void __launch_bounds__(256, 2) conv_bwd_kernel(const ConvParams p, const T* __restrict__ x, const T* __restrict__ init,
                                                          const T* __restrict__ dy, const T* __restrict__ dfin, T* __restrict__ dx,
                                                          float* __restrict__ part) {
    constexpr int P = Lanes<V>::P;
    extern __shared__ __align__(16) unsigned char smem[];       // the rings of x and dy; then the block's sums
    const int c = (blockIdx.x * blockDim.x + threadIdx.x) * V;
    const int64_t b = blockIdx.z;
    const int64_t t0 = ((int64_t)blockIdx.y * blockDim.y + threadIdx.y) * p.run;
    Lanes<V> dw[W], db;
    db.zero();
#pragma unroll
    for (int j = 0; j < W; ++j) dw[j].zero();
    if (c < p.channels && t0 < p.len) {
        const int64_t t1 = min(p.len, t0 + p.run);
        const T* xb = x + b * p.xs[0] + c;
        const T* gb = dy + b * p.gs[0] + c;
        T* ob = dx + b * p.len * p.channels + c;
        Filter<W, V> f;
        f.template load<T>(p, c);
        Ring<T, V> rx(xb, p.xs[1], smem), rg(gb, p.gs[1], smem + 256 * Ring<T, V>::kThreadBytes);
        for (int64_t a = t0; a < t1;) {
            const SeqSpan s = span_of(p, b, a);
            const int64_t end = min(t1, s.hi);
            if (s.s < 0) {
                Pack<T, V> none;
                none.zero();
                for (; a < end; ++a) none.store(ob + a * p.channels);
                continue;
            }
            const int64_t from = a, reach = min(min(p.len, s.hi), end + (W - 1));    // tokens whose g is needed
#pragma unroll
            for (int i = 0; i < Ring<T, V>::kAhead; ++i) {
                rx.fetch(i, a + i * U, reach);
                rg.fetch(i, a + i * U, reach);
                ring_commit();
            }
            Lanes<V> in[W - 1 + U], g[W - 1 + U];       // inputs and gradients of tokens a - (W-1) ..
#pragma unroll
            for (int j = 0; j < W - 1; ++j) {
                in[j] = input_of<T, W, V>(p, x, init, s, b, a - (W - 1) + j, c);
                g[j].zero();
            }
            int stage = 0;
            // One group.  INNER: its tokens are all the piece's own, and so are the W-1 before them.
            auto group = [&](auto inner) {
                constexpr bool INNER = decltype(inner)::value;
                ring_wait<Ring<T, V>::kAhead - 1>();
                Pack<T, V> pg[U];
#pragma unroll
                for (int k = 0; k < U; ++k) {
                    in[W - 1 + k].from(rx.get(stage, k));
                    pg[k] = rg.get(stage, k);
                }
                const int into = stage == 0 ? kStages - 1 : stage - 1;      // the slot read before this one
                rx.fetch(into, a + Ring<T, V>::kAhead * U, reach);
                rg.fetch(into, a + Ring<T, V>::kAhead * U, reach);
                ring_commit();
                stage = stage == kStages - 1 ? 0 : stage + 1;
#pragma unroll
                for (int k = 0; k < U; ++k) {
                    Lanes<V> d;
                    d.from(pg[k]);
                    const bool own = INNER || a + k < end, has = INNER || a + k < reach;
#pragma unroll
                    for (int i = 0; i < P; ++i) {
                        F2 o = f.bias.v[i];
#pragma unroll
                        for (int j = 0; j < W; ++j) o = fma2(f.w[j].v[i], in[k + j].v[i], o);
                        const F2 v = has ? pre_grad<T, SILU>(d.v[i], o) : F2(0.f);
                        g[W - 1 + k].v[i] = v;
                        if (own) {
                            db.v[i] = fma2(v, F2(1.f), db.v[i]);
#pragma unroll
                            for (int j = 0; j < W; ++j) dw[j].v[i] = fma2(v, in[k + j].v[i], dw[j].v[i]);
                        }
                    }
                    const int64_t u = a + k - (W - 1);  // all that u reaches is there: token u + m saw it through tap W-1-m
                    if (INNER || (u >= from && u < end)) {
                        Lanes<V> o;
#pragma unroll
                        for (int i = 0; i < P; ++i) {
                            o.v[i] = mul2(f.w[W - 1].v[i], g[k].v[i]);
#pragma unroll
                            for (int m = 1; m < W; ++m) o.v[i] = fma2(f.w[W - 1 - m].v[i], g[k + m].v[i], o.v[i]);
                        }
                        if (!INNER && dfin != nullptr && u >= s.hi - (W - 1)) {
                            Pack<T, V> q;
                            q.load(dfin + ((int64_t)s.s * (W - 1) + (u - (s.hi - (W - 1)))) * p.channels + c);
                            Lanes<V> r;
                            r.from(q);
#pragma unroll
                            for (int i = 0; i < P; ++i) o.v[i] = fma2(r.v[i], F2(1.f), o.v[i]);
                        }
                        Pack<T, V> out;
                        o.to(out);
                        out.store(ob + u * p.channels);
                    }
                }
#pragma unroll
                for (int j = 0; j < W - 1; ++j) {
                    in[j] = in[j + U];
                    g[j] = g[j + U];
                }
            };
            for (; a < end + (W - 1); a += U) {
                if (a + U <= end && a >= from + (W - 1)) group(std::true_type());
                else group(std::false_type());
            }
            ring_wait<0>();             // the zeros behind the piece's reach: the next piece starts the rings anew
            a = end;
        }
    }
    __syncthreads();
    float* red = reinterpret_cast<float*>(smem);        // [blockDim.y][W + 1][blockDim.x * V]
    const int width = blockDim.x * V;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        float* r = red + (int64_t)threadIdx.y * (W + 1) * width + threadIdx.x * V + i;
#pragma unroll
        for (int j = 0; j < W; ++j) r[j * width] = i & 1 ? dw[j].v[i / 2].y() : dw[j].v[i / 2].x();
        r[W * width] = i & 1 ? db.v[i / 2].y() : db.v[i / 2].x();
    }
    __syncthreads();
    const int64_t row = ((int64_t)b * gridDim.y + blockIdx.y) * (W + 1);
    for (int e = threadIdx.y * blockDim.x + threadIdx.x; e < (W + 1) * width; e += blockDim.x * blockDim.y) {
        float sum = 0.f;
        for (int yy = 0; yy < (int)blockDim.y; ++yy) sum += red[(int64_t)yy * (W + 1) * width + e];
        const int j = e / width, cc = blockIdx.x * width + e % width;
        if (cc < p.channels) part[(row + j) * p.channels + cc] = sum;
    }
}

// Gradient of the initial states: row r stands for token lo - (W-1) + r.  dw of the first tokens already
// counted these inputs in conv_bwd_kernel.
template <typename T, int W>
__global__ void __launch_bounds__(256) conv_init_grad_kernel(const ConvParams p, const T* __restrict__ x, const T* __restrict__ init,
                                                             const T* __restrict__ dy, const T* __restrict__ dfin,
                                                             T* __restrict__ dinit) {
    const int c = blockIdx.x * blockDim.x + threadIdx.x;
    if (c >= p.channels) return;
    const int64_t q = blockIdx.y;
    SeqSpan s;
    s.s = (int)q;
    s.lo = p.cu != nullptr ? p.cu[q] : 0;
    s.hi = p.cu != nullptr ? p.cu[q + 1] : p.len;
    if (s.lo < 0) s.lo = 0;
    if (s.hi > p.len) s.hi = p.len;
    if (s.hi < s.lo) s.hi = s.lo;
    const int64_t b = p.cu != nullptr ? 0 : q;
    Filter<W, 1> f;
    f.template load<T>(p, c);
    float acc[W - 1];
#pragma unroll
    for (int r = 0; r < W - 1; ++r) {
        acc[r] = 0.f;
        const int64_t u = s.lo - (W - 1) + r;       // the state's own way into the final state of a short sequence
        if (dfin != nullptr && u >= s.hi - (W - 1)) acc[r] = to_f<T>(dfin[(q * (W - 1) + (u - (s.hi - (W - 1)))) * p.channels + c]);
    }
    for (int n = 0; n < W - 1; ++n) {
        const int64_t t = s.lo + n;
        if (t >= s.hi) break;
        F2 o = f.bias.v[0];
#pragma unroll
        for (int j = 0; j < W; ++j) o = fma2(f.w[j].v[0], input_of<T, W, 1>(p, x, init, s, b, t - (W - 1) + j, c).v[0], o);
        const F2 dv(to_f<T>(dy[b * p.gs[0] + t * p.gs[1] + c]), 0.f);
        const float g = (p.silu ? pre_grad<T, true>(dv, o) : dv).x();
#pragma unroll
        for (int r = 0; r < W - 1; ++r)             // tap j of token lo + n is row j + n
#pragma unroll
            for (int m = 0; m <= r; ++m)
                if (m == n) acc[r] = fmaf(f.w[r - m].v[0].x(), g, acc[r]);
    }
#pragma unroll
    for (int r = 0; r < W - 1; ++r) dinit[(q * (W - 1) + r) * p.channels + c] = from_f<T>(acc[r]);
}

// part [rows][W + 1][channels] -> dw (channels, W) and dbias (channels): every eighth row in order, then the
// eight sums in order.
template <int W, typename OT>
__global__ void __launch_bounds__(256) conv_weight_grad_kernel(const float* __restrict__ part, int64_t rows, int channels,
                                                               OT* __restrict__ dw, OT* __restrict__ db) {
    __shared__ float sums[8][32];
    const int64_t i = (int64_t)blockIdx.x * 32 + threadIdx.x, n = (int64_t)channels * (W + 1);
    float s = 0.f;
    if (i < n) {
#pragma unroll 4
        for (int64_t r = threadIdx.y; r < rows; r += 8) s += part[r * n + i];
    }
    sums[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.y != 0 || i >= n) return;
    s = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) s += sums[k][threadIdx.x];
    const int j = (int)(i / channels), c = (int)(i - (int64_t)j * channels);
    if (j < W) dw[(int64_t)c * W + j] = from_f<OT>(s);
    else if (db != nullptr) db[c] = from_f<OT>(s);
}

// One token per row; the history is shifted in place.
template <typename T, int W, int V>
__global__ void __launch_bounds__(128) conv_step_kernel(const ConvParams p, const T* __restrict__ x, T* __restrict__ state,
                                                        T* __restrict__ y) {
    const int c = (blockIdx.x * blockDim.x + threadIdx.x) * V;
    if (c >= p.channels) return;
    const int64_t b = blockIdx.y;
    T* h = state + b * (W - 1) * p.channels + c;
    Pack<T, V> in, old[W - 1], out;
    in.load(x + b * p.xs[0] + c);
#pragma unroll
    for (int j = 0; j < W - 1; ++j) old[j].load(h + (int64_t)j * p.channels);
    Filter<W, V> f;
    f.template load<T>(p, c);
    Lanes<V> o = f.bias, v;
#pragma unroll
    for (int j = 0; j < W; ++j) {
        v.from(j < W - 1 ? old[j < W - 1 ? j : 0] : in);
#pragma unroll
        for (int i = 0; i < Lanes<V>::P; ++i) o.v[i] = fma2(f.w[j].v[i], v.v[i], o.v[i]);
    }
    if (p.silu) {
#pragma unroll
        for (int i = 0; i < Lanes<V>::P; ++i) o.v[i] = activate<T, true>(o.v[i]);
    }
    o.to(out);
#pragma unroll
    for (int j = 0; j + 1 < W - 1; ++j) old[j + 1].store(h + (int64_t)j * p.channels);
    in.store(h + (int64_t)(W - 2) * p.channels);
    out.store(y + b * p.channels + c);
}

// ---- host side ------------------------------------------------------------------------------------

struct Shape {
    int vx, ty, run;        // threads along channels, runs per block, tokens per run
    int64_t blocks_t;       // blocks along the tokens
};

// Longer runs read fewer halo tokens and have fewer groups at their edges, shorter ones give more threads.  At
// B8-T4096-C2048 runs of 64 tokens against 32: forward 55 us against 60, backward 108 against 125.  With fewer than
// about four warps per scheduler the latency of a run's loads shows instead, so runs shrink until there are 148 * 1024
// threads or four tokens are left.
Shape shape_of(const ConvParams& p, int v) {
    Shape s;
    const int nv = (p.channels + v - 1) / v;
    s.vx = nv >= 64 ? 64 : (nv >= 32 ? 32 : 16);
    s.ty = 256 / s.vx;
    s.run = 64;
    const int64_t per_token = (int64_t)p.batch * nv;
    while (s.run > 4 && per_token * ((p.len + s.run - 1) / s.run) < 148LL * 1024) s.run /= 2;
    while (p.len > 65535LL * s.run * s.ty) s.run *= 2;      // blocks along one grid dimension
    s.blocks_t = (p.len + (int64_t)s.run * s.ty - 1) / ((int64_t)s.run * s.ty);
    return s;
}

// Packs of v elements: every row on a boundary, the parameters too.
bool vec_ok(const ConvParams& p, int v, int elem, const void* const* ptrs, int n) {
    const int wide = p.w32 ? 4 * v : elem * v;
    bool ok = fbla::seq::aligned_to(p.w, wide > 16 ? 16 : wide) && fbla::seq::aligned_to(p.bias, wide > 16 ? 16 : wide);
    ok = ok && p.channels % v == 0 && p.xs[0] % v == 0 && p.xs[1] % v == 0 && p.gs[0] % v == 0 && p.gs[1] % v == 0;
    for (int i = 0; i < n; ++i) ok = ok && fbla::seq::aligned_to(ptrs[i], (int64_t)v * elem);
    return ok;
}

int resolve(const fbla_conv_problem* p, ConvParams* r) {
    using fbla::api_fail;
    if (p == nullptr) return api_fail(FBLA_ERR_INVALID, "problem is NULL");
    if (p->dtype != FBLA_F32 && p->dtype != FBLA_BF16 && p->dtype != FBLA_F16)
        return api_fail(FBLA_ERR_INVALID, "dtype %d is not one of FBLA_F32/FBLA_BF16/FBLA_F16", p->dtype);
    if (p->weight_dtype != FBLA_F32 && p->weight_dtype != p->dtype)
        return api_fail(FBLA_ERR_INVALID, "weight_dtype %d is neither fp32 nor the type of x", p->weight_dtype);
    if (p->width < 2 || p->width > 4) return api_fail(FBLA_ERR_UNSUPPORTED, "width=%d must be in [2, 4]", p->width);
    if (p->batch < 0 || p->batch > 65535 || p->channels < 1 || p->seq_len < 0)
        return api_fail(FBLA_ERR_INVALID, "batch=%d (at most 65535), channels=%d, seq_len=%lld", p->batch, p->channels, (long long)p->seq_len);
    if (p->cu_seqlens != nullptr && (p->num_seqs < 1 || p->num_seqs > 65535 || p->batch != 1))
        return api_fail(FBLA_ERR_INVALID, "packed sequences: num_seqs=%d must be in [1, 65535] and batch=%d be 1", p->num_seqs, p->batch);
    if (p->seq_len > (1LL << 31) - 1) return api_fail(FBLA_ERR_UNSUPPORTED, "seq_len=%lld", (long long)p->seq_len);
    r->batch = p->batch;
    r->channels = p->channels;
    r->silu = p->silu != 0;
    r->w32 = p->weight_dtype == FBLA_F32;
    r->num_seqs = p->cu_seqlens != nullptr ? p->num_seqs : p->batch;
    r->len = p->seq_len;
    const int64_t size[2] = {p->batch, p->seq_len};
    for (int i = 0; i < 2; ++i) {       // the stride of a dimension of one element is not used, whatever it is
        r->xs[i] = size[i] > 1 ? p->x_stride[i] : 0;
        r->gs[i] = size[i] > 1 ? p->dy_stride[i] : 0;
    }
    r->cu = p->cu_seqlens;
    r->run = 1;
    return FBLA_OK;
}

dim3 token_grid(const ConvParams& p, const Shape& s, int v) {
    return dim3((unsigned)(((p.channels + v - 1) / v + s.vx - 1) / s.vx), (unsigned)s.blocks_t, (unsigned)p.batch);
}

template <typename T, int W, int V>
cudaError_t launch_fwd(ConvParams p, const T* x, const T* init, T* y, cudaStream_t st) {
    const Shape s = shape_of(p, V);
    p.run = s.run;
    const size_t smem = 256 * Ring<T, V>::kThreadBytes;
    static_assert(256 * Ring<T, V>::kThreadBytes <= 48 * 1024, "the ring fits without asking for more");
    if (p.silu) conv_fwd_kernel<T, W, V, true><<<token_grid(p, s, V), dim3(s.vx, s.ty), smem, st>>>(p, x, init, y);
    else conv_fwd_kernel<T, W, V, false><<<token_grid(p, s, V), dim3(s.vx, s.ty), smem, st>>>(p, x, init, y);
    fbla::note_launches(1);
    return cudaGetLastError();
}

template <typename T, int W>
cudaError_t run_fwd(const ConvParams& p, const T* x, const T* init, T* y, T* fin, cudaStream_t st) {
    constexpr int V = 4;
    const void* ptrs[3] = {x, init, y};
    if (p.len > 0 && p.batch > 0) {
        cudaError_t e;
        if (vec_ok(p, V, sizeof(T), ptrs, 3)) e = launch_fwd<T, W, V>(p, x, init, y, st);
        else if (vec_ok(p, 2, sizeof(T), ptrs, 3)) e = launch_fwd<T, W, 2>(p, x, init, y, st);
        else e = launch_fwd<T, W, 1>(p, x, init, y, st);
        if (e != cudaSuccess) return e;
    }
    if (fin != nullptr && p.num_seqs > 0) {
        conv_final_kernel<T, W><<<dim3((p.channels + 255) / 256, W - 1, p.num_seqs), 256, 0, st>>>(p, x, init, fin);
        fbla::note_launches(1);
    }
    return cudaGetLastError();
}

template <typename T, int W, int V>
cudaError_t launch_bwd(ConvParams p, const T* x, const T* init, const T* dy, const T* dfin, T* dx, float* part, cudaStream_t st) {
    const Shape s = shape_of(p, V);
    p.run = s.run;
    const int rings = 2 * 256 * Ring<T, V>::kThreadBytes, sums = s.ty * (W + 1) * s.vx * V * (int)sizeof(float);
    const int smem = rings > sums ? rings : sums;
    static_assert(2 * 256 * Ring<T, V>::kThreadBytes <= 48 * 1024 && 256 * (W + 1) * V * sizeof(float) <= 48 * 1024,
                  "rings and sums fit without asking for more");
    if (p.silu) conv_bwd_kernel<T, W, V, true><<<token_grid(p, s, V), dim3(s.vx, s.ty), smem, st>>>(p, x, init, dy, dfin, dx, part);
    else conv_bwd_kernel<T, W, V, false><<<token_grid(p, s, V), dim3(s.vx, s.ty), smem, st>>>(p, x, init, dy, dfin, dx, part);
    fbla::note_launches(1);
    return cudaGetLastError();
}

template <typename T> constexpr int bwd_v() { return sizeof(T) == 2 ? 4 : 2; }

template <typename T, int W>
cudaError_t run_bwd(const ConvParams& p, const T* x, const T* init, const T* dy, const T* dfin, T* dx, void* dw, void* db, T* dinit,
                    float* ws, cudaStream_t st) {
    constexpr int V = bwd_v<T>();
    const void* ptrs[5] = {x, init, dy, dfin, dx};
    int64_t rows = 0;
    if (p.len > 0 && p.batch > 0) {
        const int v = vec_ok(p, V, sizeof(T), ptrs, 5) ? V : vec_ok(p, 2, sizeof(T), ptrs, 5) ? 2 : 1;
        const cudaError_t e = v == V ? launch_bwd<T, W, V>(p, x, init, dy, dfin, dx, ws, st)
                            : v == 2 ? launch_bwd<T, W, 2>(p, x, init, dy, dfin, dx, ws, st)
                                     : launch_bwd<T, W, 1>(p, x, init, dy, dfin, dx, ws, st);
        if (e != cudaSuccess) return e;
        rows = shape_of(p, v).blocks_t * p.batch;
    }
    const unsigned blocks = (unsigned)(((int64_t)p.channels * (W + 1) + 31) / 32);
    if (p.w32) conv_weight_grad_kernel<W, float><<<blocks, dim3(32, 8), 0, st>>>(ws, rows, p.channels, (float*)dw, (float*)db);
    else conv_weight_grad_kernel<W, T><<<blocks, dim3(32, 8), 0, st>>>(ws, rows, p.channels, (T*)dw, (T*)db);
    fbla::note_launches(1);
    if (dinit != nullptr && p.num_seqs > 0) {
        conv_init_grad_kernel<T, W><<<dim3((p.channels + 255) / 256, p.num_seqs), 256, 0, st>>>(p, x, init, dy, dfin, dinit);
        fbla::note_launches(1);
    }
    return cudaGetLastError();
}

template <typename T, int W>
cudaError_t run_step(const ConvParams& p, const T* x, T* state, T* y, cudaStream_t st) {
    constexpr int V = 16 / (int)sizeof(T) / 2;
    const void* ptrs[3] = {x, state, y};
    if (vec_ok(p, V, sizeof(T), ptrs, 3))
        conv_step_kernel<T, W, V><<<dim3((p.channels / V + 127) / 128, p.batch), 128, 0, st>>>(p, x, state, y);
    else
        conv_step_kernel<T, W, 1><<<dim3((p.channels + 127) / 128, p.batch), 128, 0, st>>>(p, x, state, y);
    fbla::note_launches(1);
    return cudaGetLastError();
}

// Calls f with the element type and the width as types.
template <int W> struct Taps { static constexpr int value = W; };
template <typename F> cudaError_t with_width(int width, F f) {
    return width == 2 ? f(Taps<2>()) : width == 3 ? f(Taps<3>()) : f(Taps<4>());
}
template <typename F> cudaError_t with_type(int dtype, F f) {
    return dtype == FBLA_F32 ? f((float*)nullptr) : dtype == FBLA_BF16 ? f((__nv_bfloat16*)nullptr) : f((__half*)nullptr);
}

int finish(cudaError_t e, const char* what) {
    return e == cudaSuccess ? FBLA_OK : fbla::api_fail(FBLA_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

}  // namespace

extern "C" {

int64_t fbla_causal_conv_workspace_bytes(const fbla_conv_problem* p) {
    ConvParams r;
    if (resolve(p, &r) != FBLA_OK) return -1;
    int64_t most = 0;           // kernels of different widths cut the tokens differently
    for (int v = 1; v <= 4; v *= 2) {
        const int64_t blocks = shape_of(r, v).blocks_t;
        most = blocks > most ? blocks : most;
    }
    return most * r.batch * (p->width + 1) * (int64_t)r.channels * (int64_t)sizeof(float);
}

int fbla_causal_conv_fwd(const fbla_conv_problem* p, const void* x, const void* w, const void* bias, const void* initial_state,
                         void* y, void* final_state, fbla_stream_t stream) {
    using fbla::api_fail;
    ConvParams r;
    if (int rc = resolve(p, &r)) return rc;
    if (w == nullptr) return api_fail(FBLA_ERR_INVALID, "w is NULL");
    if (r.batch > 0 && r.len > 0 && (x == nullptr || y == nullptr)) return api_fail(FBLA_ERR_INVALID, "x or y is NULL");
    r.w = w;
    r.bias = bias;
    r.gs[0] = r.gs[1] = 0;
    if (int rc = fbla::seq::check_device_status()) return rc;
    return finish(with_type(p->dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        return with_width(p->width, [&](auto k) {
            return run_fwd<T, decltype(k)::value>(r, (const T*)x, (const T*)initial_state, (T*)y, (T*)final_state, (cudaStream_t)stream);
        });
    }), "causal convolution");
}

int fbla_causal_conv_bwd(const fbla_conv_problem* p, const void* x, const void* w, const void* bias, const void* initial_state,
                         const void* dy, const void* d_final_state, void* dx, void* dw, void* dbias, void* d_initial_state,
                         void* workspace, size_t workspace_bytes, fbla_stream_t stream) {
    using fbla::api_fail;
    ConvParams r;
    if (int rc = resolve(p, &r)) return rc;
    if (w == nullptr || dw == nullptr) return api_fail(FBLA_ERR_INVALID, "w or dw is NULL");
    if (r.batch > 0 && r.len > 0 && (x == nullptr || dy == nullptr || dx == nullptr))
        return api_fail(FBLA_ERR_INVALID, "x, dy or dx is NULL");
    const int64_t need = fbla_causal_conv_workspace_bytes(p);
    if (need > 0 && (workspace == nullptr || (int64_t)workspace_bytes < need))
        return api_fail(FBLA_ERR_WORKSPACE, "workspace of %lld bytes needed, %lld given", (long long)need,
                        (long long)(workspace ? workspace_bytes : 0));
    r.w = w;
    r.bias = bias;
    if (int rc = fbla::seq::check_device_status()) return rc;
    return finish(with_type(p->dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        return with_width(p->width, [&](auto k) {
            return run_bwd<T, decltype(k)::value>(r, (const T*)x, (const T*)initial_state, (const T*)dy, (const T*)d_final_state, (T*)dx,
                                                  dw, dbias, (T*)d_initial_state, (float*)workspace, (cudaStream_t)stream);
        });
    }), "causal convolution backward");
}

int fbla_causal_conv_step(const fbla_conv_problem* p, const void* x, const void* w, const void* bias, void* state, void* y,
                          fbla_stream_t stream) {
    using fbla::api_fail;
    ConvParams r;
    if (int rc = resolve(p, &r)) return rc;
    if (r.cu != nullptr) return api_fail(FBLA_ERR_INVALID, "cu_seqlens given to the single-token step");
    if (r.batch == 0) return FBLA_OK;
    if (x == nullptr || w == nullptr || state == nullptr || y == nullptr)
        return api_fail(FBLA_ERR_INVALID, "x, w, state or y is NULL");
    r.w = w;
    r.bias = bias;
    r.xs[1] = r.gs[0] = r.gs[1] = 0;
    if (int rc = fbla::seq::check_device_status()) return rc;
    return finish(with_type(p->dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        return with_width(p->width, [&](auto k) {
            return run_step<T, decltype(k)::value>(r, (const T*)x, (T*)state, (T*)y, (cudaStream_t)stream);
        });
    }), "causal convolution step");
}

}  // extern "C"
