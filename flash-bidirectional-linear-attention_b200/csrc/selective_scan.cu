// Selective state space scan: per channel c a state of N numbers that decays and is fed token by token.
//
//   d = dt + dt_bias (softplus'd when asked),   a_n = exp(d A[c,n])
//   h_n <- a_n h_n + d x B[t,n],   s = sum_n C[t,n] h_n,   y = (s + D x) * z sigmoid(z)
//
// Backward, with e = dy z sigmoid(z) and G_t = e C_t + a_{t+1} G_{t+1}:
//   dC = e h, dB = d x G (both summed over the channels of a group), r = a h_{t-1} G,
//   dd = sum_n A r + x sum_n G B,  dx = d sum_n G B + D e,  dA += d r
//
// What bounds it: N exponentials per (token, channel) against 8 bytes of HBM traffic, so the special
// function unit (16 per clock and SM) and the issue slots, not memory.  Everything is fp32; a decay close
// to 1 is where an error of the exponential would add up over the steps that a state remembers, so those
// come from a polynomial that is exact at 0 (see decay()).
//
// Layout: four lanes share a channel, each holding N/4 states in registers, so a warp owns 8 channels and
// a CTA 64; the tokens go by in tiles whose x, dt (turned into d and d x once per channel, not once per
// lane) and B, C are staged in shared memory.  The sum over the four lanes is a transposed butterfly over
// four tokens: three shuffles for four results.
// A CTA walks over one segment of the tokens.  With few channels the tokens are cut into several
// segments: a first pass forms each segment's own end state (from zero) and its total decay, which is
// exp(A sum d); the main pass starts from the combination of the segments before it.  The backward pass
// does the same from the other end.
#include <cfloat>
#include <type_traits>

#include "seq_common.cuh"

namespace {

using fbla::from_f;
using fbla::to_f;
using fbla::seq::Pack;
using fbla::seq::seq_of;

constexpr int kCB = 64;             // channels of a CTA
constexpr int kThreads = 4 * kCB;
constexpr int kWarps = kThreads / 32;
constexpr int kPad = kCB + 8;       // row of a per-token, per-channel float array: the four lanes of a channel write
                                    // four rows at once, 8 banks apart

struct ScanParams {
    int batch, channels, states, groups, softplus, num_seqs;
    int segs;
    int64_t len, seg_len;
    int64_t xs[2], ds[2], zs[2], gs[2];     // batch, token strides of x, dt, z, dy
    int64_t bs[3], cs[3];                   // batch, token, group strides of B, C
    const int32_t* cu;
    const float *A, *D, *bias;
    int vec;                                // x, dt, z, dy, y can be read and written in packs
};

// Tokens of a tile: bounded by the shared memory that the sums over channels take in the backward pass.
template <int NS> struct Tile {
    static constexpr int kNP = 4 * NS;                  // states held, the last ones zero when N is smaller
    static constexpr int kTok = NS >= 8 ? 16 : 32;
    static constexpr int kSub = NS >= 8 ? 4 : 8;        // tokens whose decays and states the backward keeps in registers
    static constexpr int kVPT = kCB * kTok / kThreads;  // channels of a thread when it loads or stores a tile
    static constexpr int kTPR = kThreads / kTok;        // threads per token then
};

// 2^x for the decay of a state, x = d A log2(e).  |x| < 1/4: Taylor polynomial of degree 5 (next term
// (x ln2)^6 / 6! < 4e-8), 1 exactly at 0, error of the order of one rounding: a state with such a decay
// remembers many steps and a systematic error would add up over them.  Elsewhere the special function
// unit's 2^-22 is good enough, as the state forgets it within a few steps.
__device__ __forceinline__ float decay(float x) {
    float p = 1.3333558e-3f;                // ln2^5 / 5!
    p = fmaf(p, x, 9.6181291e-3f);          // ln2^4 / 4!
    p = fmaf(p, x, 5.5504109e-2f);          // ln2^3 / 3!
    p = fmaf(p, x, 0.24022651f);            // ln2^2 / 2!
    p = fmaf(p, x, 0.69314718f);            // ln2
    p = fmaf(p, x, 1.f);
    return fabsf(x) < 0.25f ? p : exp2f(x);
}

__device__ __forceinline__ float softplus(float v) { return v > 20.f ? v : log1pf(fbla::seq::exp_of(v)); }

// NS consecutive floats at a 4*NS-byte boundary
template <int NS> __device__ __forceinline__ void load_ns(const float* p, float (&v)[NS]) {
    Pack<float, NS> k;
    k.load(p);
#pragma unroll
    for (int i = 0; i < NS; ++i) v[i] = k.e[i];
}
template <int NS> __device__ __forceinline__ void store_ns(float* p, const float (&v)[NS]) {
    Pack<float, NS> k;
#pragma unroll
    for (int i = 0; i < NS; ++i) k.e[i] = v[i];
    k.store(p);
}
// Lane's states of a caller's (.., channels, N) tensor; the ones behind N are zero.
template <int NS> __device__ __forceinline__ void load_user(const float* row, int n0, int N, float (&v)[NS]) {
    if (N == 4 * NS) {
        load_ns<NS>(row + n0, v);
    } else {
#pragma unroll
        for (int i = 0; i < NS; ++i) v[i] = n0 + i < N ? row[n0 + i] : 0.f;
    }
}
template <int NS> __device__ __forceinline__ void store_user(float* row, int n0, int N, const float (&v)[NS]) {
    if (N == 4 * NS) {
        store_ns<NS>(row + n0, v);
    } else {
#pragma unroll
        for (int i = 0; i < NS; ++i)
            if (n0 + i < N) row[n0 + i] = v[i];
    }
}

// Where this CTA and lane stand.
template <int NS> struct Place {
    int64_t b;
    int seg, group, c0, cend;   // c0: first channel of the CTA, cend: end of its group
    int tile_in_group;
    int warp, lane, q, cl, c;   // q: which states, cl / c: the lane's channel in the CTA / at all
    bool live;
    __device__ __forceinline__ Place(const ScanParams& p) {
        const int cpg = p.channels / p.groups, tpg = (cpg + kCB - 1) / kCB;
        b = blockIdx.z;
        seg = blockIdx.y;
        group = blockIdx.x / tpg;
        tile_in_group = blockIdx.x - group * tpg;
        c0 = group * cpg + tile_in_group * kCB;
        cend = (group + 1) * cpg;
        warp = threadIdx.x >> 5;
        lane = threadIdx.x & 31;
        q = lane & 3;
        cl = warp * 8 + (lane >> 2);
        c = c0 + cl;
        live = c < cend;
    }
};

// Packed sequences: what happens at a token of the tile.
struct Marks {
    int first[32], last[32], inside[32];    // sequence that begins / ends here (-1: none); owned by a sequence at all
};

__device__ __forceinline__ void fill_marks(const ScanParams& p, Marks* m, int64_t t0, int n, int64_t end) {
    if ((int)threadIdx.x < n) {
        const int64_t t = t0 + threadIdx.x;
        int f = -1, l = -1, in = 0;
        if (t < end) {
            const auto s = seq_of(p.cu, p.num_seqs, t);
            if (s.s >= 0) {
                in = 1;
                f = t == s.lo ? s.s : -1;
                l = t == s.hi - 1 ? s.s : -1;
            }
        }
        m->first[threadIdx.x] = f;
        m->last[threadIdx.x] = l;
        m->inside[threadIdx.x] = in;
    }
}

// The state that token `tt` of the tile continues from: that of the token before it, unless a sequence begins.
template <int NS, bool VARLEN>
__device__ __forceinline__ void state_before(const ScanParams& p, const Place<NS>& at, const Marks& m, int tt, const float* init,
                                             const float (&h)[NS], float (&hp)[NS]) {
    const int f = VARLEN ? m.first[tt] : -1;
#pragma unroll
    for (int i = 0; i < NS; ++i) hp[i] = VARLEN && f >= 0 ? 0.f : h[i];
    if (VARLEN && f >= 0 && init != nullptr && at.live)
        load_user<NS>(init + ((int64_t)f * p.channels + at.c) * p.states, at.q * NS, p.states, hp);
}

// V elements of one token's row from channel c, zeros behind cend.
template <typename T, int V>
__device__ __forceinline__ void load_row(const T* row, int c, int cend, bool vec, float (&out)[V]) {
    if (vec && c + V <= cend) {
        Pack<T, V> k;
        k.load(row + c);
#pragma unroll
        for (int i = 0; i < V; ++i) out[i] = k.get(i);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) out[i] = c + i < cend ? to_f<T>(row[c + i]) : 0.f;
    }
}
template <typename T, int V>
__device__ __forceinline__ void store_row(T* row, int c, int cend, bool vec, const float (&v)[V]) {
    if (vec && c + V <= cend) {
        Pack<T, V> k;
#pragma unroll
        for (int i = 0; i < V; ++i) k.set(i, v[i]);
        k.store(row + c);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (c + i < cend) row[c + i] = from_f<T>(v[i]);
    }
}

// One of B, C for the tokens [t0, t0 + kTok) into dst[token][kNP]; zeros behind N, behind `end`, and for
// tokens of no sequence.
template <typename T, int NS, bool VARLEN>
__device__ __forceinline__ void stage_bc(const T* src, const int64_t (&st)[3], const ScanParams& p, const Place<NS>& at, int64_t t0,
                                         int64_t end, const Marks* m, float* dst) {
    using L = Tile<NS>;
    const T* base = src + at.b * st[0] + at.group * st[2];
    for (int i = threadIdx.x; i < L::kTok * L::kNP; i += kThreads) {
        const int t = i / L::kNP, n = i % L::kNP;
        bool ok = n < p.states && t0 + t < end;
        if (VARLEN) ok = ok && m->inside[t];
        dst[i] = ok ? to_f<T>(base[(t0 + t) * st[1] + n]) : 0.f;
    }
}

// Lane q of the four gets the sum over them of v[q].
__device__ __forceinline__ float sum4(const float (&v)[4], int q) {
    const bool odd = q & 1, high = q & 2;
    float a = odd ? v[1] : v[0], b = odd ? v[3] : v[2];
    a += __shfl_xor_sync(0xffffffffu, odd ? v[0] : v[1], 1);
    b += __shfl_xor_sync(0xffffffffu, odd ? v[2] : v[3], 1);
    return (high ? b : a) + __shfl_xor_sync(0xffffffffu, high ? a : b, 2);
}

// Workspace of the segmented passes: [batch][segs][channels][kNP] states, then [batch][segs][channels] sums of d.
template <int NS> __device__ __forceinline__ int64_t seg_at(const ScanParams& p, int64_t b, int seg, int c) {
    return (b * p.segs + seg) * p.channels + c;
}

template <typename T, int NS> struct FwdSmem {
    using L = Tile<NS>;
    float2 dx[L::kTok][kCB];            // (d, d x)
    float B[L::kTok * L::kNP], C[L::kTok * L::kNP];
    float y[L::kTok][kPad];
    Marks marks;
};

// LOCAL: end state of the segment from zero, and the sum of d (infinite when a sequence begins inside, so
// that nothing from before gets through).  Otherwise the outputs.
template <typename T, int NS, bool VARLEN, bool LOCAL>
__global__ void __launch_bounds__(kThreads) scan_fwd_kernel(const ScanParams p, const T* __restrict__ x, const T* __restrict__ dt,
                                                            const T* __restrict__ Bm, const T* __restrict__ Cm,
                                                            const T* __restrict__ z, const float* __restrict__ init,
                                                            T* __restrict__ y, float* __restrict__ fin, float* __restrict__ ckpt,
                                                            float* __restrict__ seg_h, float* __restrict__ seg_d) {
    using L = Tile<NS>;
    extern __shared__ __align__(16) unsigned char raw_smem[];
    FwdSmem<T, NS>& sm = *reinterpret_cast<FwdSmem<T, NS>*>(raw_smem);
    const Place<NS> at(p);
    if (LOCAL && at.seg == p.segs - 1) return;      // nothing comes behind it
    const int N = p.states, n0 = at.q * NS;
    const int64_t t0 = at.seg * p.seg_len, t1 = min(p.len, t0 + p.seg_len);

    float A2[NS], h[NS], sum_d = 0.f;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        A2[i] = at.live && n0 + i < N ? p.A[(int64_t)at.c * N + n0 + i] * 1.44269504f : 0.f;
        h[i] = 0.f;
    }
    if (!LOCAL && at.live) {
        if (!VARLEN && init != nullptr) load_user<NS>(init + (at.b * p.channels + at.c) * N, n0, N, h);
        for (int j = 0; j < at.seg; ++j) {
            const int64_t k = seg_at<NS>(p, at.b, j, at.c);
            const float sd = seg_d[k];
            float own[NS];
            load_ns<NS>(seg_h + k * L::kNP + n0, own);
#pragma unroll
            for (int i = 0; i < NS; ++i) h[i] = sd == INFINITY ? own[i] : fmaf(decay(sd * A2[i]), h[i], own[i]);
        }
    }
    const int row = threadIdx.x / L::kTPR, col = (threadIdx.x % L::kTPR) * L::kVPT;     // when loading or storing
    const int64_t ntiles = (p.len + L::kTok - 1) / L::kTok;

    for (int64_t tb = t0; tb < t1; tb += L::kTok) {
        if (VARLEN) {
            fill_marks(p, &sm.marks, tb, L::kTok, t1);
            __syncthreads();
        }
        const int64_t t = tb + row;
        bool ok = t < t1;
        if (VARLEN) ok = ok && sm.marks.inside[row];
        float xv[L::kVPT], dv[L::kVPT];
        if (ok) {
            load_row<T, L::kVPT>(x + at.b * p.xs[0] + t * p.xs[1], at.c0 + col, at.cend, p.vec, xv);
            load_row<T, L::kVPT>(dt + at.b * p.ds[0] + t * p.ds[1], at.c0 + col, at.cend, p.vec, dv);
#pragma unroll
            for (int i = 0; i < L::kVPT; ++i) {
                if (p.bias != nullptr && at.c0 + col + i < at.cend) dv[i] += p.bias[at.c0 + col + i];
                if (p.softplus) dv[i] = softplus(dv[i]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < L::kVPT; ++i) xv[i] = dv[i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < L::kVPT; ++i) sm.dx[row][col + i] = make_float2(dv[i], dv[i] * xv[i]);
        stage_bc<T, NS, VARLEN>(Bm, p.bs, p, at, tb, t1, &sm.marks, sm.B);
        if (!LOCAL) stage_bc<T, NS, VARLEN>(Cm, p.cs, p, at, tb, t1, &sm.marks, sm.C);
        __syncthreads();

        if (!LOCAL && ckpt != nullptr && at.live)
            store_ns<NS>(ckpt + (((at.b * ntiles + tb / L::kTok) * p.channels + at.c) * L::kNP + n0), h);
#pragma unroll 2
        for (int tt = 0; tt < L::kTok; tt += 4) {
            float ys[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float2 v = sm.dx[tt + k][at.cl];
                float Bv[NS], Cv[NS];
                load_ns<NS>(sm.B + (tt + k) * L::kNP + n0, Bv);
                if (!LOCAL) load_ns<NS>(sm.C + (tt + k) * L::kNP + n0, Cv);
                float hp[NS];
                state_before<NS, VARLEN>(p, at, sm.marks, tt + k, init, h, hp);
                if (LOCAL) sum_d += VARLEN && sm.marks.first[tt + k] >= 0 ? INFINITY : v.x;
                float acc = 0.f;
#pragma unroll
                for (int i = 0; i < NS; ++i) {
                    h[i] = fmaf(decay(v.x * A2[i]), hp[i], v.y * Bv[i]);
                    if (!LOCAL) acc = fmaf(Cv[i], h[i], acc);
                }
                ys[k] = acc;
                if (VARLEN && !LOCAL && fin != nullptr) {
                    const int l = sm.marks.last[tt + k];
                    if (l >= 0 && at.live) store_user<NS>(fin + ((int64_t)l * p.channels + at.c) * N, n0, N, h);
                }
            }
            if (!LOCAL) sm.y[tt + at.q][at.cl] = sum4(ys, at.q);
        }
        __syncthreads();
        if (!LOCAL && t < t1) {
            float out[L::kVPT], zv[L::kVPT];
            if (z != nullptr) load_row<T, L::kVPT>(z + at.b * p.zs[0] + t * p.zs[1], at.c0 + col, at.cend, p.vec, zv);
#pragma unroll
            for (int i = 0; i < L::kVPT; ++i) {
                float s = sm.y[row][col + i];
                if (p.D != nullptr && at.c0 + col + i < at.cend) s = fmaf(p.D[at.c0 + col + i], xv[i], s);
                if (z != nullptr) s *= zv[i] * fbla::seq::sigmoid<T>(zv[i]);
                out[i] = ok ? s : 0.f;
            }
            store_row<T, L::kVPT>(y + (at.b * p.len + t) * p.channels, at.c0 + col, at.cend, p.vec, out);
        }
    }
    if (!at.live) return;
    if (LOCAL) {
        const int64_t k = seg_at<NS>(p, at.b, at.seg, at.c);
        store_ns<NS>(seg_h + k * L::kNP + n0, h);
        if (at.q == 0) seg_d[k] = sum_d;
    } else if (!VARLEN && fin != nullptr && at.seg == p.segs - 1) {
        store_user<NS>(fin + (at.b * p.channels + at.c) * N, n0, N, h);
    }
}

// to[s] = from[s] (or 0) for the sequences without a token: nothing else writes their final state, or the
// gradient of their initial state.
__global__ void __launch_bounds__(256) scan_empty_kernel(const ScanParams p, const float* __restrict__ from, float* __restrict__ to) {
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x, n = (int64_t)p.channels * p.states;
    if (i >= n) return;
    const int64_t s = blockIdx.y;
    const int64_t tokens = p.cu != nullptr ? (int64_t)p.cu[s + 1] - p.cu[s] : p.len;
    if (tokens <= 0) to[s * n + i] = from != nullptr ? from[s * n + i] : 0.f;
}

template <typename T, int NS> struct BwdSmem {
    using L = Tile<NS>;
    float4 v[L::kTok][kCB];                         // (d, d x, e, -)
    float B[L::kTok * L::kNP], C[L::kTok * L::kNP];
    float start[L::kTok / L::kSub][kThreads][NS];   // each thread's states at the starts of the sub-tiles
    float gB[L::kTok][kPad], rA[L::kTok][kPad], y[L::kTok][kPad];
    float dbc[kWarps][L::kTok][2 * L::kNP];         // per warp: sums of dB, dC over its eight channels
    float dD[kThreads][L::kVPT], db[kThreads][L::kVPT];
    Marks marks;
};

// What a thread loads of a tile in the backward passes: d and the slope of d, x, e, and what dz needs.
template <typename T, int V> struct BwdRow {
    float x[V], d[V], slope[V], e[V], dy[V], zv[V];
};

template <typename T, int NS>
__device__ __forceinline__ void load_bwd_row(const ScanParams& p, const Place<NS>& at, const T* x, const T* dt, const T* z, const T* dy,
                                             int64_t t, int col, bool ok, BwdRow<T, Tile<NS>::kVPT>& r) {
    constexpr int V = Tile<NS>::kVPT;
    const int c = at.c0 + col;
#pragma unroll
    for (int i = 0; i < V; ++i) r.x[i] = r.d[i] = r.slope[i] = r.e[i] = r.dy[i] = r.zv[i] = 0.f;
    if (!ok) return;
    if (x != nullptr) load_row<T, V>(x + at.b * p.xs[0] + t * p.xs[1], c, at.cend, p.vec, r.x);
    load_row<T, V>(dt + at.b * p.ds[0] + t * p.ds[1], c, at.cend, p.vec, r.d);
    load_row<T, V>(dy + at.b * p.gs[0] + t * p.gs[1], c, at.cend, p.vec, r.dy);
    if (z != nullptr) load_row<T, V>(z + at.b * p.zs[0] + t * p.zs[1], c, at.cend, p.vec, r.zv);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        if (p.bias != nullptr && c + i < at.cend) r.d[i] += p.bias[c + i];
        r.slope[i] = 1.f;
        if (p.softplus) {
            r.slope[i] = r.d[i] > 20.f ? 1.f : fbla::seq::sigmoid<float>(r.d[i]);
            r.d[i] = softplus(r.d[i]);
        }
        r.e[i] = z != nullptr ? r.dy[i] * r.zv[i] * fbla::seq::sigmoid<float>(r.zv[i]) : r.dy[i];
    }
}

template <typename T, int NS> struct BwdLocalSmem {
    using L = Tile<NS>;
    float2 v[L::kTok][kCB];             // (d, e)
    float C[L::kTok * L::kNP];
    Marks marks;
};

// What a segment passes to the one before it, from zero: a G of its first token.  seg_d as in the forward.
template <typename T, int NS, bool VARLEN>
__global__ void __launch_bounds__(kThreads) scan_bwd_local_kernel(const ScanParams p, const T* __restrict__ dt, const T* __restrict__ Cm,
                                                                  const T* __restrict__ z, const T* __restrict__ dy,
                                                                  const float* __restrict__ dfin, float* __restrict__ seg_g,
                                                                  float* __restrict__ seg_d) {
    using L = Tile<NS>;
    extern __shared__ __align__(16) unsigned char raw_smem[];
    BwdLocalSmem<T, NS>& sm = *reinterpret_cast<BwdLocalSmem<T, NS>*>(raw_smem);
    const Place<NS> at(p);
    if (at.seg == 0) return;            // nothing comes before it
    const int N = p.states, n0 = at.q * NS;
    const int64_t t0 = at.seg * p.seg_len, t1 = min(p.len, t0 + p.seg_len);
    float A2[NS], g[NS], sum_d = 0.f;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        A2[i] = at.live && n0 + i < N ? p.A[(int64_t)at.c * N + n0 + i] * 1.44269504f : 0.f;
        g[i] = 0.f;
    }
    if (!VARLEN && dfin != nullptr && at.live && at.seg == p.segs - 1) load_user<NS>(dfin + (at.b * p.channels + at.c) * N, n0, N, g);
    const int row = threadIdx.x / L::kTPR, col = (threadIdx.x % L::kTPR) * L::kVPT;
    for (int64_t tb = t0 + (t1 - 1 - t0) / L::kTok * L::kTok; tb >= t0; tb -= L::kTok) {
        __syncthreads();
        if (VARLEN) {
            fill_marks(p, &sm.marks, tb, L::kTok, t1);
            __syncthreads();
        }
        const int64_t t = tb + row;
        bool ok = t < t1;
        if (VARLEN) ok = ok && sm.marks.inside[row];
        BwdRow<T, L::kVPT> r;
        load_bwd_row<T, NS>(p, at, nullptr, dt, z, dy, t, col, ok, r);
#pragma unroll
        for (int i = 0; i < L::kVPT; ++i) sm.v[row][col + i] = make_float2(r.d[i], r.e[i]);
        stage_bc<T, NS, VARLEN>(Cm, p.cs, p, at, tb, t1, &sm.marks, sm.C);
        __syncthreads();
        for (int tt = L::kTok - 1; tt >= 0; --tt) {
            const float2 v = sm.v[tt][at.cl];
            float Cv[NS];
            load_ns<NS>(sm.C + tt * L::kNP + n0, Cv);
            if (VARLEN && dfin != nullptr) {
                const int l = sm.marks.last[tt];
                if (l >= 0 && at.live) load_user<NS>(dfin + ((int64_t)l * p.channels + at.c) * N, n0, N, g);
            }
            sum_d += v.x;
#pragma unroll
            for (int i = 0; i < NS; ++i) g[i] = decay(v.x * A2[i]) * fmaf(v.y, Cv[i], g[i]);
            if (VARLEN && sm.marks.first[tt] >= 0) {
                sum_d = INFINITY;
#pragma unroll
                for (int i = 0; i < NS; ++i) g[i] = 0.f;
            }
        }
    }
    if (!at.live) return;
    const int64_t k = seg_at<NS>(p, at.b, at.seg, at.c);
    store_ns<NS>(seg_g + k * L::kNP + n0, g);
    if (at.q == 0) seg_d[k] = sum_d;
}

// Sums over the eight channels of a warp (lane bits 2, 3, 4) of the M values each lane holds: halving
// exchanges while there is something to halve.  Returns the index of the first value the lane ends with;
// max(1, M / 8) of them are left in v[0 ..].
template <int M> __device__ __forceinline__ int sum8(float (&v)[M], int lane) {
    int first = 0, m = M;
#pragma unroll
    for (int mask = 16; mask >= 4; mask >>= 1) {
        const bool up = lane & mask;
        if (m > 1) {
            m >>= 1;
#pragma unroll
            for (int i = 0; i < M / 2; ++i) {
                if (i < m) {
                    const float give = up ? v[i] : v[i + m], keep = up ? v[i + m] : v[i];
                    v[i] = keep + __shfl_xor_sync(0xffffffffu, give, mask);
                }
            }
            if (up) first += m;
        } else {
            v[0] += __shfl_xor_sync(0xffffffffu, v[0], mask);
        }
    }
    return first;
}

// All gradients of one segment.  part_bc: [channel tile of the group][batch][token][group][2][kNP] sums over the
// CTA's channels; part_A [batch][segs][channels][N], part_D / part_bias [batch][segs][channels].
template <typename T, int NS, bool VARLEN>
__global__ void __launch_bounds__(kThreads, 2) scan_bwd_kernel(
    const ScanParams p, const T* __restrict__ x, const T* __restrict__ dt, const T* __restrict__ Bm, const T* __restrict__ Cm,
    const T* __restrict__ z, const float* __restrict__ init, const T* __restrict__ dy, const float* __restrict__ dfin,
    const float* __restrict__ ckpt, const float* __restrict__ seg_g, const float* __restrict__ seg_d, T* __restrict__ dx,
    T* __restrict__ ddt, T* __restrict__ dz, float* __restrict__ dinit, float* __restrict__ part_bc, float* __restrict__ part_A,
    float* __restrict__ part_D, float* __restrict__ part_bias) {
    using L = Tile<NS>;
    constexpr int K = L::kSub;
    extern __shared__ __align__(16) unsigned char raw_smem[];
    BwdSmem<T, NS>& sm = *reinterpret_cast<BwdSmem<T, NS>*>(raw_smem);
    const Place<NS> at(p);
    const int N = p.states, n0 = at.q * NS;
    const int64_t t0 = at.seg * p.seg_len, t1 = min(p.len, t0 + p.seg_len);
    const int64_t ntiles = (p.len + L::kTok - 1) / L::kTok;

    float A[NS], g[NS], dA[NS];         // g: a G of the token behind
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        A[i] = at.live && n0 + i < N ? p.A[(int64_t)at.c * N + n0 + i] : 0.f;
        g[i] = dA[i] = 0.f;
    }
    if (at.live) {
        if (!VARLEN && dfin != nullptr && at.seg == p.segs - 1) load_user<NS>(dfin + (at.b * p.channels + at.c) * N, n0, N, g);
        for (int j = p.segs - 1; j > at.seg; --j) {
            const int64_t k = seg_at<NS>(p, at.b, j, at.c);
            const float sd = seg_d[k];
            float own[NS];
            load_ns<NS>(seg_g + k * L::kNP + n0, own);
#pragma unroll
            for (int i = 0; i < NS; ++i) g[i] = sd == INFINITY ? own[i] : fmaf(decay(sd * A[i] * 1.44269504f), g[i], own[i]);
        }
    }
    const int row = threadIdx.x / L::kTPR, col = (threadIdx.x % L::kTPR) * L::kVPT;
#pragma unroll
    for (int i = 0; i < L::kVPT; ++i) sm.dD[threadIdx.x][i] = sm.db[threadIdx.x][i] = 0.f;

    for (int64_t tb = t0 + (t1 - 1 - t0) / L::kTok * L::kTok; tb >= t0; tb -= L::kTok) {
        __syncthreads();
        if (VARLEN) {
            fill_marks(p, &sm.marks, tb, L::kTok, t1);
            __syncthreads();
        }
        const int64_t t = tb + row;
        bool ok = t < t1;
        if (VARLEN) ok = ok && sm.marks.inside[row];
        {
            BwdRow<T, L::kVPT> r;
            load_bwd_row<T, NS>(p, at, x, dt, z, dy, t, col, ok, r);
#pragma unroll
            for (int i = 0; i < L::kVPT; ++i) sm.v[row][col + i] = make_float4(r.d[i], r.d[i] * r.x[i], r.e[i], 0.f);
        }
        stage_bc<T, NS, VARLEN>(Bm, p.bs, p, at, tb, t1, &sm.marks, sm.B);
        stage_bc<T, NS, VARLEN>(Cm, p.cs, p, at, tb, t1, &sm.marks, sm.C);
        __syncthreads();

        // forward again: the states at the starts of the sub-tiles
        float h[NS];
#pragma unroll
        for (int i = 0; i < NS; ++i) h[i] = 0.f;
        if (at.live) load_ns<NS>(ckpt + (((at.b * ntiles + tb / L::kTok) * p.channels + at.c) * L::kNP + n0), h);
#pragma unroll 1
        for (int sub = 0; sub < L::kTok / K; ++sub) {
            store_ns<NS>(sm.start[sub][threadIdx.x], h);
            if (sub == L::kTok / K - 1) break;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int tt = sub * K + k;
                const float2 v = *reinterpret_cast<const float2*>(&sm.v[tt][at.cl]);
                float Bv[NS];
                load_ns<NS>(sm.B + tt * L::kNP + n0, Bv);
                float hp[NS];
                state_before<NS, VARLEN>(p, at, sm.marks, tt, init, h, hp);
#pragma unroll
                for (int i = 0; i < NS; ++i) h[i] = fmaf(decay(v.x * (A[i] * 1.44269504f)), hp[i], v.y * Bv[i]);
            }
        }
#pragma unroll 1
        for (int sub = L::kTok / K - 1; sub >= 0; --sub) {
            float a[K][NS], hs[K + 1][NS];
            load_ns<NS>(sm.start[sub][threadIdx.x], hs[0]);
            float ys[K], gb[K], ra[K];
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int tt = sub * K + k;
                const float2 v = *reinterpret_cast<const float2*>(&sm.v[tt][at.cl]);
                float Bv[NS], Cv[NS];
                load_ns<NS>(sm.B + tt * L::kNP + n0, Bv);
                load_ns<NS>(sm.C + tt * L::kNP + n0, Cv);
                float hp[NS];
                state_before<NS, VARLEN>(p, at, sm.marks, tt, init, hs[k], hp);
                float acc = 0.f;
#pragma unroll
                for (int i = 0; i < NS; ++i) {
                    a[k][i] = decay(v.x * (A[i] * 1.44269504f));
                    hs[k + 1][i] = fmaf(a[k][i], hp[i], v.y * Bv[i]);
                    acc = fmaf(Cv[i], hs[k + 1][i], acc);
                }
                ys[k] = acc;
            }
#pragma unroll
            for (int k = K - 1; k >= 0; --k) {
                const int tt = sub * K + k;
                const float4 v = sm.v[tt][at.cl];
                float Bv[NS], Cv[NS], bc[2 * NS];
                load_ns<NS>(sm.B + tt * L::kNP + n0, Bv);
                load_ns<NS>(sm.C + tt * L::kNP + n0, Cv);
                if (VARLEN && dfin != nullptr) {
                    const int l = sm.marks.last[tt];
                    if (l >= 0 && at.live) load_user<NS>(dfin + ((int64_t)l * p.channels + at.c) * N, n0, N, g);
                }
                float hp[NS];
                state_before<NS, VARLEN>(p, at, sm.marks, tt, init, hs[k], hp);
                gb[k] = ra[k] = 0.f;
#pragma unroll
                for (int i = 0; i < NS; ++i) {
                    const float G = fmaf(v.z, Cv[i], g[i]);
                    bc[i] = v.y * G;
                    bc[NS + i] = v.z * hs[k + 1][i];
                    gb[k] = fmaf(G, Bv[i], gb[k]);
                    g[i] = a[k][i] * G;
                    const float r = g[i] * hp[i];
                    ra[k] = fmaf(r, A[i], ra[k]);
                    dA[i] = fmaf(v.x, r, dA[i]);
                }
                if (VARLEN) {
                    const int f = sm.marks.first[tt];
                    if (f >= 0) {
                        if (dinit != nullptr && at.live) store_user<NS>(dinit + ((int64_t)f * p.channels + at.c) * N, n0, N, g);
#pragma unroll
                        for (int i = 0; i < NS; ++i) g[i] = 0.f;
                    }
                }
                const int first = sum8<2 * NS>(bc, at.lane);
                constexpr int LEFT = 2 * NS >= 8 ? 2 * NS / 8 : 1;
#pragma unroll
                for (int i = 0; i < LEFT; ++i) {
                    const int w = first + i;            // dB of state n0 + w, or dC of state n0 + w - NS
                    sm.dbc[at.warp][tt][(w < NS ? n0 + w : L::kNP + n0 + w - NS)] = bc[i];
                }
            }
#pragma unroll
            for (int k = 0; k < K; k += 4) {
                const int tt = sub * K + k + at.q;
                const float y4[4] = {ys[k], ys[k + 1], ys[k + 2], ys[k + 3]}, g4[4] = {gb[k], gb[k + 1], gb[k + 2], gb[k + 3]},
                            r4[4] = {ra[k], ra[k + 1], ra[k + 2], ra[k + 3]};
                sm.y[tt][at.cl] = sum4(y4, at.q);
                sm.gB[tt][at.cl] = sum4(g4, at.q);
                sm.rA[tt][at.cl] = sum4(r4, at.q);
            }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < L::kTok * 2 * L::kNP; i += kThreads) {
            const int tt = i / (2 * L::kNP), w = i % (2 * L::kNP);
            if (tb + tt >= t1) continue;
            float s = 0.f;
#pragma unroll
            for (int k = 0; k < kWarps; ++k) s += sm.dbc[k][tt][w];
            part_bc[((((int64_t)at.tile_in_group * p.batch + at.b) * p.len + tb + tt) * p.groups + at.group) * (2 * L::kNP) + w] = s;
        }
        if (t < t1) {
            BwdRow<T, L::kVPT> r;
            load_bwd_row<T, NS>(p, at, x, dt, z, dy, t, col, ok, r);
            float ox[L::kVPT], od[L::kVPT], oz[L::kVPT];
#pragma unroll
            for (int i = 0; i < L::kVPT; ++i) {
                const int c = at.c0 + col + i;
                const float D = p.D != nullptr && c < at.cend ? p.D[c] : 0.f;
                const float gB = sm.gB[row][col + i];
                ox[i] = ok ? fmaf(r.d[i], gB, D * r.e[i]) : 0.f;
                od[i] = ok ? r.slope[i] * fmaf(r.x[i], gB, sm.rA[row][col + i]) : 0.f;
                if (z != nullptr) {
                    const float sg = fbla::seq::sigmoid<float>(r.zv[i]);
                    oz[i] = ok ? r.dy[i] * fmaf(D, r.x[i], sm.y[row][col + i]) * sg * (1.f + r.zv[i] * (1.f - sg)) : 0.f;
                }
                sm.dD[threadIdx.x][i] += r.e[i] * r.x[i];
                sm.db[threadIdx.x][i] += od[i];
            }
            const int64_t o = (at.b * p.len + t) * p.channels;
            store_row<T, L::kVPT>(dx + o, at.c0 + col, at.cend, p.vec, ox);
            store_row<T, L::kVPT>(ddt + o, at.c0 + col, at.cend, p.vec, od);
            if (z != nullptr) store_row<T, L::kVPT>(dz + o, at.c0 + col, at.cend, p.vec, oz);
        }
    }
    __syncthreads();
    const int64_t bs = at.b * p.segs + at.seg;
    if ((int)threadIdx.x < kCB && at.c0 + (int)threadIdx.x < at.cend) {
        const int k = threadIdx.x / L::kVPT, i = threadIdx.x % L::kVPT;
        float sD = 0.f, sb = 0.f;
        for (int r = 0; r < L::kTok; ++r) {
            sD += sm.dD[r * L::kTPR + k][i];
            sb += sm.db[r * L::kTPR + k][i];
        }
        part_D[bs * p.channels + at.c0 + threadIdx.x] = sD;
        part_bias[bs * p.channels + at.c0 + threadIdx.x] = sb;
    }
    if (!at.live) return;
    store_user<NS>(part_A + (bs * p.channels + at.c) * N, n0, N, dA);
    if (!VARLEN && dinit != nullptr && at.seg == 0) store_user<NS>(dinit + (at.b * p.channels + at.c) * N, n0, N, g);
}

// dB, dC (batch, token, group, N) from the channel tiles' sums, tiles in order.
template <typename T, int NP>
__global__ void __launch_bounds__(256) scan_bc_kernel(const float* __restrict__ part, int tiles, int64_t rows, int N, T* __restrict__ dB,
                                                      T* __restrict__ dC) {
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= rows * 2 * NP) return;
    const int64_t r = i / (2 * NP);
    const int w = (int)(i % (2 * NP)), n = w % NP;
    if (n >= N) return;
    float s = 0.f;
    for (int k = 0; k < tiles; ++k) s += part[k * rows * 2 * NP + i];
    (w < NP ? dB : dC)[r * N + n] = from_f<T>(s);
}

// One token per row, the state updated in place.
template <typename T, int NS>
__global__ void __launch_bounds__(kThreads) scan_step_kernel(const ScanParams p, const T* __restrict__ x, const T* __restrict__ dt,
                                                             const T* __restrict__ Bm, const T* __restrict__ Cm,
                                                             const T* __restrict__ z, float* __restrict__ state, T* __restrict__ y) {
    const Place<NS> at(p);
    const int N = p.states, n0 = at.q * NS;
    float acc = 0.f, xv = 0.f;
    if (at.live) {
        float* hp = state + (at.b * p.channels + at.c) * N;
        float h[NS], A[NS], Bv[NS], Cv[NS];
        load_user<NS>(hp, n0, N, h);
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            const bool in = n0 + i < N;
            A[i] = in ? p.A[(int64_t)at.c * N + n0 + i] : 0.f;
            Bv[i] = in ? to_f<T>(Bm[at.b * p.bs[0] + at.group * p.bs[2] + n0 + i]) : 0.f;
            Cv[i] = in ? to_f<T>(Cm[at.b * p.cs[0] + at.group * p.cs[2] + n0 + i]) : 0.f;
        }
        xv = to_f<T>(x[at.b * p.xs[0] + at.c]);
        float d = to_f<T>(dt[at.b * p.ds[0] + at.c]);
        if (p.bias != nullptr) d += p.bias[at.c];
        if (p.softplus) d = softplus(d);
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            h[i] = fmaf(decay(d * (A[i] * 1.44269504f)), h[i], d * xv * Bv[i]);
            acc = fmaf(Cv[i], h[i], acc);
        }
        store_user<NS>(hp, n0, N, h);
    }
    acc += __shfl_xor_sync(0xffffffffu, acc, 1);
    acc += __shfl_xor_sync(0xffffffffu, acc, 2);
    if (at.live && at.q == 0) {
        if (p.D != nullptr) acc = fmaf(p.D[at.c], xv, acc);
        if (z != nullptr) {
            const float zv = to_f<T>(z[at.b * p.zs[0] + at.c]);
            acc *= zv * fbla::seq::sigmoid<T>(zv);
        }
        y[at.b * p.channels + at.c] = from_f<T>(acc);
    }
}

// ---- host side ------------------------------------------------------------------------------------

int ns_of(int N) { return N <= 4 ? 1 : N <= 8 ? 2 : N <= 16 ? 4 : 8; }
int np_of(int N) { return 4 * ns_of(N); }
int tok_of(int N) { return ns_of(N) >= 8 ? 16 : 32; }
int tiles_per_group(const ScanParams& p) { return (p.channels / p.groups + kCB - 1) / kCB; }

// One CTA walks a whole sequence unless that leaves SMs without work: then the tokens are cut so that
// about two CTAs per SM exist.  A segment is at least four tiles: its local pass and the combination of the
// segments before it have to stay small beside it.
void cut(ScanParams& p) {
    const int tok = tok_of(p.states);
    const int64_t ctas = (int64_t)p.batch * p.groups * tiles_per_group(p), tiles = (p.len + tok - 1) / tok;
    int64_t segs = ctas > 0 ? (2 * 148 + ctas - 1) / ctas : 1;
    if (segs > tiles / 4) segs = tiles / 4;
    if (segs < 1 || ctas >= 148) segs = 1;
    const int64_t per = segs > 0 ? (tiles + segs - 1) / segs : 1;
    p.seg_len = (per > 0 ? per : 1) * tok;
    p.segs = p.len > 0 ? (int)((p.len + p.seg_len - 1) / p.seg_len) : 1;
}

int64_t seg_floats(const ScanParams& p) { return p.segs > 1 ? (int64_t)p.batch * p.segs * p.channels * (np_of(p.states) + 1) : 0; }

int resolve(const fbla_scan_problem* p, ScanParams* r) {
    using fbla::api_fail;
    if (p == nullptr) return api_fail(FBLA_ERR_INVALID, "problem is NULL");
    if (p->dtype != FBLA_F32 && p->dtype != FBLA_BF16 && p->dtype != FBLA_F16)
        return api_fail(FBLA_ERR_INVALID, "dtype %d is not one of FBLA_F32/FBLA_BF16/FBLA_F16", p->dtype);
    if (p->states < 1 || p->states > 32) return api_fail(FBLA_ERR_UNSUPPORTED, "states=%d must be in [1, 32]", p->states);
    if (p->batch < 0 || p->batch > 65535 || p->channels < 1 || p->seq_len < 0)
        return api_fail(FBLA_ERR_INVALID, "batch=%d (at most 65535), channels=%d, seq_len=%lld", p->batch, p->channels, (long long)p->seq_len);
    if (p->groups < 1 || p->channels % p->groups != 0)
        return api_fail(FBLA_ERR_INVALID, "groups=%d must divide channels=%d", p->groups, p->channels);
    if (p->cu_seqlens != nullptr && (p->num_seqs < 1 || p->num_seqs > 65535 || p->batch != 1))
        return api_fail(FBLA_ERR_INVALID, "packed sequences: num_seqs=%d must be in [1, 65535] and batch=%d be 1", p->num_seqs, p->batch);
    if (p->seq_len > (1LL << 31) - 1) return api_fail(FBLA_ERR_UNSUPPORTED, "seq_len=%lld", (long long)p->seq_len);
    r->batch = p->batch;
    r->channels = p->channels;
    r->states = p->states;
    r->groups = p->groups;
    r->softplus = p->softplus != 0;
    r->num_seqs = p->cu_seqlens != nullptr ? p->num_seqs : p->batch;
    r->len = p->seq_len;
    for (int i = 0; i < 2; ++i) {
        r->xs[i] = p->x_stride[i];
        r->ds[i] = p->dt_stride[i];
        r->zs[i] = p->z_stride[i];
        r->gs[i] = p->dy_stride[i];
    }
    for (int i = 0; i < 3; ++i) {
        r->bs[i] = p->b_stride[i];
        r->cs[i] = p->c_stride[i];
    }
    r->cu = p->cu_seqlens;
    r->A = r->D = r->bias = nullptr;
    r->vec = 0;
    cut(*r);
    return FBLA_OK;
}

// Packs of 8 (4 for states above 16) elements: every row and every CTA's first channel on a boundary.
bool can_vec(const ScanParams& p, int elem, bool z, bool dy, std::initializer_list<const void*> ptrs) {
    const int v = tok_of(p.states) == 16 ? 4 : 8;
    const int64_t bytes = v * elem > 16 ? 16 : v * elem;
    bool ok = (p.channels / p.groups) % v == 0 && p.xs[0] % v == 0 && p.xs[1] % v == 0 && p.ds[0] % v == 0 && p.ds[1] % v == 0;
    if (z) ok = ok && p.zs[0] % v == 0 && p.zs[1] % v == 0;
    if (dy) ok = ok && p.gs[0] % v == 0 && p.gs[1] % v == 0;
    for (const void* q : ptrs) ok = ok && fbla::seq::aligned_to(q, bytes);
    return ok;
}

template <typename Kernel> cudaError_t allow_smem(Kernel k, size_t bytes) {
    return bytes > 48 * 1024 ? cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) : cudaSuccess;
}

struct ScanTensors {
    const void *x, *dt, *B, *C, *z, *dy;
    const float *init, *dfin;
    void *y, *dx, *ddt, *dB, *dC, *dz;
    float *fin, *ckpt, *dA, *dD, *dbias, *dinit, *ws;
};

dim3 scan_grid(const ScanParams& p) { return dim3((unsigned)(p.groups * tiles_per_group(p)), (unsigned)p.segs, (unsigned)p.batch); }

cudaError_t fill_empty(const ScanParams& p, const float* from, float* to, cudaStream_t st) {
    if (to == nullptr || p.num_seqs == 0 || (p.cu == nullptr && p.len > 0)) return cudaSuccess;
    const int64_t n = (int64_t)p.channels * p.states;
    scan_empty_kernel<<<dim3((unsigned)((n + 255) / 256), (unsigned)p.num_seqs), 256, 0, st>>>(p, from, to);
    fbla::note_launches(1);
    return cudaGetLastError();
}

template <typename T, int NS, bool VARLEN> cudaError_t run_fwd(const ScanParams& p, const ScanTensors& a, cudaStream_t st) {
    if (cudaError_t e = fill_empty(p, a.init, a.fin, st)) return e;
    if (p.len == 0 || p.batch == 0) return cudaSuccess;
    using S = FwdSmem<T, NS>;
    float* seg_h = a.ws;
    float* seg_d = p.segs > 1 ? a.ws + (int64_t)p.batch * p.segs * p.channels * Tile<NS>::kNP : nullptr;
    if (p.segs > 1) {
        auto k = scan_fwd_kernel<T, NS, VARLEN, true>;
        if (cudaError_t e = allow_smem(k, sizeof(S))) return e;
        k<<<scan_grid(p), kThreads, sizeof(S), st>>>(p, (const T*)a.x, (const T*)a.dt, (const T*)a.B, (const T*)a.C, nullptr, a.init, nullptr,
                                                     nullptr, nullptr, seg_h, seg_d);
        fbla::note_launches(1);
    }
    auto k = scan_fwd_kernel<T, NS, VARLEN, false>;
    if (cudaError_t e = allow_smem(k, sizeof(S))) return e;
    k<<<scan_grid(p), kThreads, sizeof(S), st>>>(p, (const T*)a.x, (const T*)a.dt, (const T*)a.B, (const T*)a.C, (const T*)a.z, a.init,
                                                 (T*)a.y, a.fin, a.ckpt, seg_h, seg_d);
    fbla::note_launches(1);
    return cudaGetLastError();
}

// Floats of the backward's workspace in front of the segment states.
struct BwdLayout {
    int64_t A, D, bias, bc, seg, total;
};
BwdLayout bwd_layout(const ScanParams& p) {
    const int64_t bsc = (int64_t)p.batch * p.segs * p.channels;
    auto up = [](int64_t v) { return (v + 3) / 4 * 4; };
    BwdLayout l;
    l.A = 0;
    l.D = l.A + up(bsc * p.states);
    l.bias = l.D + up(bsc);
    l.bc = l.bias + up(bsc);
    l.seg = l.bc + (int64_t)tiles_per_group(p) * p.batch * p.len * p.groups * 2 * np_of(p.states);
    l.total = l.seg + seg_floats(p);
    return l;
}

template <typename T, int NS, bool VARLEN> cudaError_t run_bwd(const ScanParams& p, const ScanTensors& a, cudaStream_t st) {
    if (cudaError_t e = fill_empty(p, a.dfin, a.dinit, st)) return e;
    const BwdLayout l = bwd_layout(p);
    const bool any = p.len > 0 && p.batch > 0;
    const int64_t rows = any ? (int64_t)p.batch * p.segs : 0;
    if (any) {
        float* seg_g = a.ws + l.seg;
        float* seg_d = seg_g + (int64_t)p.batch * p.segs * p.channels * Tile<NS>::kNP;
        if (p.segs > 1) {
            auto k = scan_bwd_local_kernel<T, NS, VARLEN>;
            using S = BwdLocalSmem<T, NS>;
            if (cudaError_t e = allow_smem(k, sizeof(S))) return e;
            k<<<scan_grid(p), kThreads, sizeof(S), st>>>(p, (const T*)a.dt, (const T*)a.C, (const T*)a.z, (const T*)a.dy, a.dfin, seg_g, seg_d);
            fbla::note_launches(1);
        }
        auto k = scan_bwd_kernel<T, NS, VARLEN>;
        using S = BwdSmem<T, NS>;
        if (cudaError_t e = allow_smem(k, sizeof(S))) return e;
        k<<<scan_grid(p), kThreads, sizeof(S), st>>>(p, (const T*)a.x, (const T*)a.dt, (const T*)a.B, (const T*)a.C, (const T*)a.z, a.init,
                                                     (const T*)a.dy, a.dfin, a.ckpt, seg_g, seg_d, (T*)a.dx, (T*)a.ddt, (T*)a.dz, a.dinit,
                                                     a.ws + l.bc, a.ws + l.A, a.ws + l.D, a.ws + l.bias);
        fbla::note_launches(1);
        if (cudaError_t e = cudaGetLastError()) return e;
        const int64_t tok = (int64_t)p.batch * p.len * p.groups, n = tok * 2 * Tile<NS>::kNP;
        scan_bc_kernel<T, Tile<NS>::kNP><<<(unsigned)((n + 255) / 256), 256, 0, st>>>(a.ws + l.bc, tiles_per_group(p), tok, p.states,
                                                                                     (T*)a.dB, (T*)a.dC);
        fbla::note_launches(1);
    }
    if (cudaError_t e = fbla::seq::sum_rows(a.ws + l.A, rows, (int64_t)p.channels * p.states, FBLA_F32, a.dA, st)) return e;
    if (a.dD != nullptr)
        if (cudaError_t e = fbla::seq::sum_rows(a.ws + l.D, rows, p.channels, FBLA_F32, a.dD, st)) return e;
    if (a.dbias != nullptr)
        if (cudaError_t e = fbla::seq::sum_rows(a.ws + l.bias, rows, p.channels, FBLA_F32, a.dbias, st)) return e;
    return cudaGetLastError();
}

template <typename T, int NS> cudaError_t run_step(const ScanParams& p, const ScanTensors& a, cudaStream_t st) {
    scan_step_kernel<T, NS><<<scan_grid(p), kThreads, 0, st>>>(p, (const T*)a.x, (const T*)a.dt, (const T*)a.B, (const T*)a.C, (const T*)a.z,
                                                               a.fin, (T*)a.y);
    fbla::note_launches(1);
    return cudaGetLastError();
}

template <int V> struct Num { static constexpr int value = V; };
// Calls f with (element type, states per lane).
template <typename F> cudaError_t with_shape(int dtype, int N, F f) {
    auto inner = [&](auto* t) {
        switch (ns_of(N)) {
            case 1: return f(t, Num<1>());
            case 2: return f(t, Num<2>());
            case 4: return f(t, Num<4>());
            default: return f(t, Num<8>());
        }
    };
    return dtype == FBLA_F32 ? inner((float*)nullptr) : dtype == FBLA_BF16 ? inner((__nv_bfloat16*)nullptr) : inner((__half*)nullptr);
}

int finish(cudaError_t e, const char* what) {
    return e == cudaSuccess ? FBLA_OK : fbla::api_fail(FBLA_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

int check_states(std::initializer_list<const void*> ptrs) {
    for (const void* q : ptrs)
        if (!fbla::seq::aligned_to(q, 16)) return fbla::api_fail(FBLA_ERR_INVALID, "states and workspaces must be 16-byte aligned");
    return FBLA_OK;
}

int check_ws(int64_t need, const void* ws, size_t have) {
    if (need > 0 && (ws == nullptr || (int64_t)have < need))
        return fbla::api_fail(FBLA_ERR_WORKSPACE, "workspace of %lld bytes needed, %lld given", (long long)need, (long long)(ws ? have : 0));
    return FBLA_OK;
}

}  // namespace

extern "C" {

int64_t fbla_selective_scan_checkpoint_floats(const fbla_scan_problem* p) {
    ScanParams r;
    if (resolve(p, &r) != FBLA_OK) return -1;
    const int tok = tok_of(r.states);
    return (int64_t)r.batch * ((r.len + tok - 1) / tok) * r.channels * np_of(r.states);
}

int64_t fbla_selective_scan_workspace_bytes(const fbla_scan_problem* p, int backward) {
    ScanParams r;
    if (resolve(p, &r) != FBLA_OK) return -1;
    return (backward ? bwd_layout(r).total : seg_floats(r)) * (int64_t)sizeof(float);
}

int fbla_selective_scan_fwd(const fbla_scan_problem* p, const void* x, const void* dt, const float* A, const void* B, const void* C,
                            const float* D, const void* z, const float* dt_bias, const float* initial_state, void* y, float* final_state,
                            float* checkpoints, void* workspace, size_t workspace_bytes, fbla_stream_t stream) {
    using fbla::api_fail;
    ScanParams r;
    if (int rc = resolve(p, &r)) return rc;
    if (A == nullptr) return api_fail(FBLA_ERR_INVALID, "A is NULL");
    if (r.batch > 0 && r.len > 0 && (x == nullptr || dt == nullptr || B == nullptr || C == nullptr || y == nullptr))
        return api_fail(FBLA_ERR_INVALID, "x, dt, B, C or y is NULL");
    if (int rc = check_ws(seg_floats(r) * (int64_t)sizeof(float), workspace, workspace_bytes)) return rc;
    if (int rc = check_states({initial_state, final_state, checkpoints, workspace})) return rc;
    r.A = A;
    r.D = D;
    r.bias = dt_bias;
    r.vec = can_vec(r, p->dtype == FBLA_F32 ? 4 : 2, z != nullptr, false, {x, dt, z, y});
    ScanTensors a = {};
    a.x = x; a.dt = dt; a.B = B; a.C = C; a.z = z; a.init = initial_state; a.y = y; a.fin = final_state; a.ckpt = checkpoints;
    a.ws = (float*)workspace;
    return finish(with_shape(p->dtype, r.states, [&](auto* t, auto n) {
        using T = std::remove_pointer_t<decltype(t)>;
        return r.cu != nullptr ? run_fwd<T, decltype(n)::value, true>(r, a, (cudaStream_t)stream)
                               : run_fwd<T, decltype(n)::value, false>(r, a, (cudaStream_t)stream);
    }), "selective scan");
}

int fbla_selective_scan_bwd(const fbla_scan_problem* p, const void* x, const void* dt, const float* A, const void* B, const void* C,
                            const float* D, const void* z, const float* dt_bias, const float* initial_state, const float* checkpoints,
                            const void* dy, const float* d_final_state, void* dx, void* ddt, float* dA, void* dB, void* dC, float* dD,
                            void* dz, float* d_dt_bias, float* d_initial_state, void* workspace, size_t workspace_bytes,
                            fbla_stream_t stream) {
    using fbla::api_fail;
    ScanParams r;
    if (int rc = resolve(p, &r)) return rc;
    if (A == nullptr || dA == nullptr) return api_fail(FBLA_ERR_INVALID, "A or dA is NULL");
    if (r.batch > 0 && r.len > 0 && (x == nullptr || dt == nullptr || B == nullptr || C == nullptr || dy == nullptr || dx == nullptr ||
                                     ddt == nullptr || dB == nullptr || dC == nullptr || checkpoints == nullptr))
        return api_fail(FBLA_ERR_INVALID, "x, dt, B, C, dy, their gradients or checkpoints is NULL");
    if ((z == nullptr) != (dz == nullptr)) return api_fail(FBLA_ERR_INVALID, "dz goes with z");
    if (int rc = check_ws(bwd_layout(r).total * (int64_t)sizeof(float), workspace, workspace_bytes)) return rc;
    if (int rc = check_states({initial_state, d_final_state, d_initial_state, checkpoints, workspace})) return rc;
    r.A = A;
    r.D = D;
    r.bias = dt_bias;
    r.vec = can_vec(r, p->dtype == FBLA_F32 ? 4 : 2, z != nullptr, true, {x, dt, z, dy, dx, ddt, dz});
    ScanTensors a = {};
    a.x = x; a.dt = dt; a.B = B; a.C = C; a.z = z; a.dy = dy; a.init = initial_state; a.dfin = d_final_state;
    a.dx = dx; a.ddt = ddt; a.dB = dB; a.dC = dC; a.dz = dz; a.ckpt = const_cast<float*>(checkpoints);
    a.dA = dA; a.dD = dD; a.dbias = d_dt_bias; a.dinit = d_initial_state; a.ws = (float*)workspace;
    return finish(with_shape(p->dtype, r.states, [&](auto* t, auto n) {
        using T = std::remove_pointer_t<decltype(t)>;
        return r.cu != nullptr ? run_bwd<T, decltype(n)::value, true>(r, a, (cudaStream_t)stream)
                               : run_bwd<T, decltype(n)::value, false>(r, a, (cudaStream_t)stream);
    }), "selective scan backward");
}

int fbla_selective_scan_step(const fbla_scan_problem* p, const void* x, const void* dt, const float* A, const void* B, const void* C,
                             const float* D, const void* z, const float* dt_bias, float* state, void* y, fbla_stream_t stream) {
    using fbla::api_fail;
    ScanParams r;
    if (int rc = resolve(p, &r)) return rc;
    if (r.cu != nullptr) return api_fail(FBLA_ERR_INVALID, "cu_seqlens given to the single-token step");
    if (r.batch == 0) return FBLA_OK;
    if (x == nullptr || dt == nullptr || A == nullptr || B == nullptr || C == nullptr || state == nullptr || y == nullptr)
        return api_fail(FBLA_ERR_INVALID, "x, dt, A, B, C, state or y is NULL");
    if (int rc = check_states({state})) return rc;
    r.A = A;
    r.D = D;
    r.bias = dt_bias;
    r.segs = 1;
    ScanTensors a = {};
    a.x = x; a.dt = dt; a.B = B; a.C = C; a.z = z; a.fin = state; a.y = y;
    return finish(with_shape(p->dtype, r.states, [&](auto* t, auto n) {
        using T = std::remove_pointer_t<decltype(t)>;
        return run_step<T, decltype(n)::value>(r, a, (cudaStream_t)stream);
    }), "selective scan step");
}

}  // extern "C"
