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
// Tokens go by in groups of four, and the next group's loads are on their way while one is worked on: with
// one load in flight per thread a B8-T4096-C2048 forward took 124 us and the backward 298.
// The weight gradient is summed in registers over a thread's run, in shared memory over the runs of a
// block, and then over the blocks by a kernel of its own: no atomics, the same bits on every run.
#include <type_traits>

#include "seq_common.cuh"

namespace fbla {
namespace seq {

namespace {
template <typename OT>
__global__ void __launch_bounds__(256) sum_rows_kernel(const float* __restrict__ in, int64_t rows, int64_t n, OT* __restrict__ out) {
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= n) return;
    float s = 0.f;
    for (int64_t r = 0; r < rows; ++r) s += in[r * n + i];
    out[i] = from_f<OT>(s);
}
}  // namespace

cudaError_t sum_rows(const float* in, int64_t rows, int64_t n, int out_dtype, void* out, cudaStream_t st) {
    if (n == 0) return cudaSuccess;
    const int64_t blocks = (n + 255) / 256;
    if (blocks > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
    if (out_dtype == FBLA_F32) sum_rows_kernel<float><<<(unsigned)blocks, 256, 0, st>>>(in, rows, n, (float*)out);
    else if (out_dtype == FBLA_BF16) sum_rows_kernel<__nv_bfloat16><<<(unsigned)blocks, 256, 0, st>>>(in, rows, n, (__nv_bfloat16*)out);
    else sum_rows_kernel<__half><<<(unsigned)blocks, 256, 0, st>>>(in, rows, n, (__half*)out);
    note_launches(1);
    return cudaGetLastError();
}

}  // namespace seq
}  // namespace fbla

namespace {

using fbla::from_f;
using fbla::to_f;
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

template <typename T> __device__ __forceinline__ float param(const ConvParams& p, const void* base, int64_t i) {
    return p.w32 ? reinterpret_cast<const float*>(base)[i] : to_f<T>(reinterpret_cast<const T*>(base)[i]);
}

__device__ __forceinline__ SeqSpan span_of(const ConvParams& p, int64_t b, int64_t t) {
    if (p.cu != nullptr) return seq_of(p.cu, p.num_seqs, t);
    SeqSpan s;
    s.s = (int)b;
    s.lo = 0;
    s.hi = p.len;
    return s;
}

// Input of token u (which may lie before its sequence: initial state, or zero), V channels from c.
template <typename T, int W, int V>
__device__ __forceinline__ void input_of(const ConvParams& p, const T* x, const T* init, const SeqSpan& s, int64_t b, int64_t u,
                                         int c, float (&out)[V]) {
    Pack<T, V> v;
    if (u >= s.lo && s.s >= 0) {
        v.load(x + b * p.xs[0] + u * p.xs[1] + c);
    } else if (init != nullptr && s.s >= 0) {
        v.load(init + ((int64_t)s.s * (W - 1) + (W - 1 + (u - s.lo))) * p.channels + c);
    } else {
        v.zero();
    }
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = v.get(i);
}

template <typename T> __device__ __forceinline__ float activate(float x, int silu) {
    return silu ? x * fbla::seq::sigmoid<T>(x) : x;
}

// dy times the slope of the activation at p
template <typename T> __device__ __forceinline__ float pre_grad(float dy, float x, int silu) {
    if (!silu) return dy;
    const float sg = fbla::seq::sigmoid<T>(x);
    return dy * sg * fmaf(x, 1.f - sg, 1.f);
}

constexpr int U = 4;            // tokens of a group

template <typename T, int V> __device__ __forceinline__ void load_group(const T* base, int64_t stride, int64_t t, int64_t end, Pack<T, V> (&v)[U]) {
#pragma unroll
    for (int k = 0; k < U; ++k)
        if (t + k < end) v[k].load(base + (t + k) * stride);
}

// Parameters of V channels
template <typename T, int W, int V> struct Filter {
    float w[W][V], bias[V];
    __device__ __forceinline__ void load(const ConvParams& p, int c) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            bias[i] = p.bias != nullptr ? param<T>(p, p.bias, c + i) : 0.f;
#pragma unroll
            for (int j = 0; j < W; ++j) w[j][i] = param<T>(p, p.w, (int64_t)(c + i) * W + j);
        }
    }
};

// A thread walks over its run piece by piece, a piece being the run's tokens of one sequence.
template <typename T, int W, int V>
__global__ void __launch_bounds__(256) conv_fwd_kernel(const ConvParams p, const T* __restrict__ x, const T* __restrict__ init,
                                                       T* __restrict__ y) {
    const int c = (blockIdx.x * blockDim.x + threadIdx.x) * V;
    const int64_t b = blockIdx.z;
    const int64_t t0 = ((int64_t)blockIdx.y * blockDim.y + threadIdx.y) * p.run;
    if (c >= p.channels || t0 >= p.len) return;
    const int64_t t1 = min(p.len, t0 + p.run);
    const T* xb = x + b * p.xs[0] + c;
    T* yb = y + b * p.len * p.channels + c;
    Filter<T, W, V> f;
    f.load(p, c);
    for (int64_t a = t0; a < t1;) {
        const SeqSpan s = span_of(p, b, a);
        const int64_t end = min(t1, s.hi);
        if (s.s < 0) {
            Pack<T, V> none;
            none.zero();
            for (; a < end; ++a) none.store(yb + a * p.channels);
            continue;
        }
        Pack<T, V> next[U];
        load_group<T, V>(xb, p.xs[1], a, end, next);
        float in[W - 1 + U][V];         // the last W-1 inputs, then the group's
#pragma unroll
        for (int j = 0; j < W - 1; ++j) input_of<T, W, V>(p, x, init, s, b, a - (W - 1) + j, c, in[j]);
        for (; a < end; a += U) {
#pragma unroll
            for (int k = 0; k < U; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) in[W - 1 + k][i] = next[k].get(i);
            load_group<T, V>(xb, p.xs[1], a + U, end, next);
#pragma unroll
            for (int k = 0; k < U; ++k) {
                Pack<T, V> out;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    float o = f.bias[i];
#pragma unroll
                    for (int j = 0; j < W; ++j) o = fmaf(f.w[j][i], in[k + j][i], o);
                    out.set(i, activate<T>(o, p.silu));
                }
                if (a + k < end) out.store(yb + (a + k) * p.channels);
            }
#pragma unroll
            for (int j = 0; j < W - 1; ++j)
#pragma unroll
                for (int i = 0; i < V; ++i) in[j][i] = in[j + U][i];
        }
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
template <typename T, int W, int V>
__global__ void __launch_bounds__(256, 2) conv_bwd_kernel(const ConvParams p, const T* __restrict__ x, const T* __restrict__ init,
                                                          const T* __restrict__ dy, const T* __restrict__ dfin, T* __restrict__ dx,
                                                          float* __restrict__ part) {
    extern __shared__ float red[];              // [blockDim.y][W + 1][blockDim.x * V]
    const int c = (blockIdx.x * blockDim.x + threadIdx.x) * V;
    const int64_t b = blockIdx.z;
    const int64_t t0 = ((int64_t)blockIdx.y * blockDim.y + threadIdx.y) * p.run;
    float dw[W][V], db[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        db[i] = 0.f;
#pragma unroll
        for (int j = 0; j < W; ++j) dw[j][i] = 0.f;
    }
    if (c < p.channels && t0 < p.len) {
        const int64_t t1 = min(p.len, t0 + p.run);
        const T* xb = x + b * p.xs[0] + c;
        const T* gb = dy + b * p.gs[0] + c;
        T* db_out = dx + b * p.len * p.channels + c;
        Filter<T, W, V> f;
        f.load(p, c);
        for (int64_t a = t0; a < t1;) {
            const SeqSpan s = span_of(p, b, a);
            const int64_t end = min(t1, s.hi);
            if (s.s < 0) {
                Pack<T, V> none;
                none.zero();
                for (; a < end; ++a) none.store(db_out + a * p.channels);
                continue;
            }
            const int64_t from = a, reach = min(min(p.len, s.hi), end + (W - 1));    // tokens whose g is needed
            Pack<T, V> nx[U], ng[U];
            load_group<T, V>(xb, p.xs[1], a, reach, nx);
            load_group<T, V>(gb, p.gs[1], a, reach, ng);
            float in[W - 1 + U][V], g[W - 1 + U][V];    // inputs and gradients of tokens a - (W-1) ..
#pragma unroll
            for (int j = 0; j < W - 1; ++j) {
                input_of<T, W, V>(p, x, init, s, b, a - (W - 1) + j, c, in[j]);
#pragma unroll
                for (int i = 0; i < V; ++i) g[j][i] = 0.f;
            }
            for (; a < end + (W - 1); a += U) {
                float d[U][V];
#pragma unroll
                for (int k = 0; k < U; ++k)
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        in[W - 1 + k][i] = nx[k].get(i);
                        d[k][i] = ng[k].get(i);
                    }
                load_group<T, V>(xb, p.xs[1], a + U, reach, nx);
                load_group<T, V>(gb, p.gs[1], a + U, reach, ng);
                const bool inner = a + U <= end;        // all four tokens are the piece's own
#pragma unroll
                for (int k = 0; k < U; ++k) {
                    const bool own = inner || a + k < end, has = inner || a + k < reach;
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        float o = f.bias[i];
#pragma unroll
                        for (int j = 0; j < W; ++j) o = fmaf(f.w[j][i], in[k + j][i], o);
                        const float v = has ? pre_grad<T>(d[k][i], o, p.silu) : 0.f;
                        g[W - 1 + k][i] = v;
                        if (own) {
                            db[i] += v;
#pragma unroll
                            for (int j = 0; j < W; ++j) dw[j][i] = fmaf(v, in[k + j][i], dw[j][i]);
                        }
                    }
                    const int64_t u = a + k - (W - 1);  // all that u reaches is there: token u + m saw it through tap W-1-m
                    if (u >= from && u < end) {
                        float o[V];
#pragma unroll
                        for (int i = 0; i < V; ++i) {
                            o[i] = 0.f;
#pragma unroll
                            for (int m = 0; m < W; ++m) o[i] = fmaf(f.w[W - 1 - m][i], g[k + m][i], o[i]);
                        }
                        if (dfin != nullptr && u >= s.hi - (W - 1)) {
                            const T* q = dfin + ((int64_t)s.s * (W - 1) + (u - (s.hi - (W - 1)))) * p.channels + c;
#pragma unroll
                            for (int i = 0; i < V; ++i) o[i] += to_f<T>(q[i]);
                        }
                        Pack<T, V> out;
#pragma unroll
                        for (int i = 0; i < V; ++i) out.set(i, o[i]);
                        out.store(db_out + u * p.channels);
                    }
                }
#pragma unroll
                for (int j = 0; j < W - 1; ++j)
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        in[j][i] = in[j + U][i];
                        g[j][i] = g[j + U][i];
                    }
            }
            a = end;
        }
    }
    const int width = blockDim.x * V;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        float* r = red + (int64_t)threadIdx.y * (W + 1) * width + threadIdx.x * V + i;
#pragma unroll
        for (int j = 0; j < W; ++j) r[j * width] = dw[j][i];
        r[W * width] = db[i];
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
    float w[W], acc[W - 1], win[W][1];
    const float bias = p.bias != nullptr ? param<T>(p, p.bias, c) : 0.f;
#pragma unroll
    for (int j = 0; j < W; ++j) w[j] = param<T>(p, p.w, (int64_t)c * W + j);
#pragma unroll
    for (int r = 0; r < W - 1; ++r) {
        acc[r] = 0.f;
        const int64_t u = s.lo - (W - 1) + r;       // the state's own way into the final state of a short sequence
        if (dfin != nullptr && u >= s.hi - (W - 1)) acc[r] = to_f<T>(dfin[(q * (W - 1) + (u - (s.hi - (W - 1)))) * p.channels + c]);
    }
    for (int n = 0; n < W - 1; ++n) {
        const int64_t t = s.lo + n;
        if (t >= s.hi) break;
        float a = bias;
#pragma unroll
        for (int j = 0; j < W; ++j) {
            input_of<T, W, 1>(p, x, init, s, b, t - (W - 1) + j, c, win[j]);
            a = fmaf(w[j], win[j][0], a);
        }
        const float g = pre_grad<T>(to_f<T>(dy[b * p.gs[0] + t * p.gs[1] + c]), a, p.silu);
#pragma unroll
        for (int r = 0; r < W - 1; ++r)             // tap j of token lo + n is row j + n
            if (r - n >= 0) acc[r] = fmaf(w[r - n], g, acc[r]);
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
#pragma unroll
    for (int i = 0; i < V; ++i) {
        float a = p.bias != nullptr ? param<T>(p, p.bias, c + i) : 0.f;
#pragma unroll
        for (int j = 0; j < W; ++j) a = fmaf(param<T>(p, p.w, (int64_t)(c + i) * W + j), (j < W - 1 ? old[j].get(i) : in.get(i)), a);
        out.set(i, activate<T>(a, p.silu));
    }
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

// Longer runs read fewer halo tokens, shorter ones give more threads.  A run of 32 costs (W-1)/32 = 9 %
// more reads (mostly from L2); with fewer than about four warps per scheduler the latency of a run's
// loads shows instead, so runs shrink until there are 148 * 1024 threads or four tokens are left.
Shape shape_of(const ConvParams& p, int v) {
    Shape s;
    const int nv = (p.channels + v - 1) / v;
    s.vx = nv >= 64 ? 64 : (nv >= 32 ? 32 : 16);
    s.ty = 256 / s.vx;
    s.run = 32;
    const int64_t per_token = (int64_t)p.batch * nv;
    while (s.run > 4 && per_token * ((p.len + s.run - 1) / s.run) < 148LL * 1024) s.run /= 2;
    while (p.len > 65535LL * s.run * s.ty) s.run *= 2;      // blocks along one grid dimension
    s.blocks_t = (p.len + (int64_t)s.run * s.ty - 1) / ((int64_t)s.run * s.ty);
    return s;
}

bool vec_ok(const ConvParams& p, int v, int elem, const void* const* ptrs, int n) {
    bool ok = p.channels % v == 0 && p.xs[0] % v == 0 && p.xs[1] % v == 0 && p.gs[0] % v == 0 && p.gs[1] % v == 0;
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
    for (int i = 0; i < 2; ++i) {
        r->xs[i] = p->x_stride[i];
        r->gs[i] = p->dy_stride[i];
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
    conv_fwd_kernel<T, W, V><<<token_grid(p, s, V), dim3(s.vx, s.ty), 0, st>>>(p, x, init, y);
    fbla::note_launches(1);
    return cudaGetLastError();
}

template <typename T, int W>
cudaError_t run_fwd(const ConvParams& p, const T* x, const T* init, T* y, T* fin, cudaStream_t st) {
    constexpr int V = 16 / (int)sizeof(T);
    const void* ptrs[3] = {x, init, y};
    if (p.len > 0 && p.batch > 0) {
        const cudaError_t e = vec_ok(p, V, sizeof(T), ptrs, 3) ? launch_fwd<T, W, V>(p, x, init, y, st) : launch_fwd<T, W, 1>(p, x, init, y, st);
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
    const size_t smem = (size_t)s.ty * (W + 1) * s.vx * V * sizeof(float);
    conv_bwd_kernel<T, W, V><<<token_grid(p, s, V), dim3(s.vx, s.ty), smem, st>>>(p, x, init, dy, dfin, dx, part);
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
        const bool vec = vec_ok(p, V, sizeof(T), ptrs, 5);
        const cudaError_t e = vec ? launch_bwd<T, W, V>(p, x, init, dy, dfin, dx, ws, st) : launch_bwd<T, W, 1>(p, x, init, dy, dfin, dx, ws, st);
        if (e != cudaSuccess) return e;
        rows = shape_of(p, vec ? V : 1).blocks_t * p.batch;
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
    // the scalar and the vector kernel cut the tokens differently: the larger of the two
    const int v = p->dtype == FBLA_F32 ? bwd_v<float>() : bwd_v<__half>();
    const int64_t a = shape_of(r, 1).blocks_t, b = shape_of(r, v).blocks_t;
    return (a > b ? a : b) * r.batch * (p->width + 1) * (int64_t)r.channels * (int64_t)sizeof(float);
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
    return finish(with_type(p->dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        return with_width(p->width, [&](auto k) {
            return run_step<T, decltype(k)::value>(r, (const T*)x, (T*)state, (T*)y, (cudaStream_t)stream);
        });
    }), "causal convolution step");
}

}  // extern "C"
