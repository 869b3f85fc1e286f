// Selective state space scan: per channel c a state of N numbers that decays and is fed token by token.
//
//   d = dt + dt_bias (softplus'd when asked),   a_n = exp(d A[c,n])
//   h_n <- a_n h_n + d x B[t,n],   s = sum_n C[t,n] h_n,   y = (s + D x) * z sigmoid(z)
//
// Backward, with e = dy z sigmoid(z) and G_t = e C_t + a_{t+1} G_{t+1}:
//   dC = e h, dB = d x G (both summed over the channels of a group), r = a h_{t-1} G,
//   dd = sum_n A r + x sum_n G B,  dx = d sum_n G B + D e,  dA += d r
//
// What bounds it: N exponentials per (token, channel) against 8 bytes of HBM traffic, so arithmetic, not memory.
// Everything is fp32; a decay close to 1 is where an error of the exponential would add up over the steps that a
// state remembers, so those come from a polynomial that is exact at 0 (see decay2()).
// Measured at B8-T4096-C2048, 16 states, bf16: forward 692 us, backward 2022 us.  Forward, on an SM with three CTAs:
// special function unit 58 % busy, multiply-add units 56 %, issue slots 62 %, 1.1 stall cycles of fixed latency per
// issue: no unit is at its limit, and more warps (four CTAs, 128 registers) or unrolling gave nothing.  The special
// function unit alone (16 + 4 operations per token and channel, 16 per clock and SM) would take 290 us forward.
//
// Layout: four lanes share two channels, each lane holding N/4 states of both in registers, so a warp owns 16
// channels and a CTA of four warps 64; the tokens go by in tiles whose x, dt (turned into d and d x once per
// channel, not once per lane) and B, C are staged in shared memory.  Two channels per lane because what a lane
// reads of B and C counts: shared memory delivers 128 bytes per clock to the registers of an SM whether lanes
// read the same address or not, and with one channel per lane those reads took as long as the arithmetic.  The
// sum over the four lanes is a transposed butterfly over four tokens: three shuffles for four results.
// A CTA walks over one segment of the tokens.  With few channels the tokens are cut into several
// segments: a first pass forms each segment's own end state (from zero) and its total decay, which is
// exp(A sum d); the main pass starts from the combination of the segments before it.  The backward pass
// does the same from the other end.
#pragma once

#include <type_traits>

#include "seq_common.cuh"

namespace fbla {
namespace scan {

using fbla::seq::Pack;
using fbla::seq::seq_of;
using fbla::seq::ex2;
using fbla::seq::F2;
using fbla::seq::fma2;
using fbla::seq::mul2;

constexpr int kCB = 64;                 // channels of a CTA
constexpr int kThreads = 2 * kCB;       // four lanes for two channels
constexpr int kWarps = kThreads / 32;
constexpr int kRow4 = kCB / 2 + 4;      // row of 16-byte slots (two channels each): 64 bytes of padding
constexpr int kRow2 = kCB / 2 + 4;      // row of 8-byte slots: 32 bytes of padding

struct ScanParams {
    int batch, channels, states, groups, softplus, num_seqs;
    int segs;
    int64_t len, seg_len;
    int64_t xs[2], ds[2], zs[2], gs[2];     // batch, token strides of x, dt, z, dy
    int64_t bs[3], cs[3];                   // batch, token, group strides of B, C
    const int32_t* cu;
    const float *A, *D, *bias;
    int vec;                                // x, dt, z, dy, y can be read and written in packs
    int wide_A;                             // A can be read in packs: no states behind N, and its address on a boundary
};

// Tokens of a tile: bounded by the shared memory that the sums over channels take in the backward pass.
template <int NS> struct Tile {
    static constexpr int kNP = 4 * NS;                  // states held, the last ones zero when N is smaller
    static constexpr int kTok = NS >= 8 ? 16 : 32;
    static constexpr int kSub = NS >= 8 ? 4 : 8;        // tokens whose decays and states the backward keeps in registers
    static constexpr int kVPT = kCB * kTok / kThreads;  // channels of a thread when it loads or stores a tile
    static constexpr int kTPR = kThreads / kTok;        // threads per token then
};

// 2^x for the decays of two states, x = d A log2(e).
// For x in [-5/64, 0]: 1 + x (ln2 + x (c1 + x c2)), c1 and c2 chosen by minimising the largest error of (2^x - 1) / x
// over that range with ln2 held fixed: 1.5e-8 at most, a quarter of a rounding, and relative to the steps that a
// state with such a decay remembers (1 / (x ln2)) an error of the state of 2.7e-7 at most and none for x -> 0.
// Elsewhere the special function unit: measured on B200 it is off by -2e-8 on average between -0.25 and 0 and by
// -5e-8 below, which over the 18 steps or fewer that such a state remembers is 4e-7.  Over the thousands of steps
// of a slow state an error that always has the same sign would be the largest of all, so it is not used there.
// (A negative x not below -5/64 is, read as an integer, not above that of -5/64.)
__device__ __forceinline__ F2 decay2(F2 x) {
    F2 p(5.4470904e-2f);
    p = fma2(p, x, F2(0.24020165f));
    p = fma2(p, x, F2(0.69314718f));
    p = fma2(p, x, F2(1.f));
    float x0, x1, p0, p1;
    x.get(x0, x1);
    p.get(p0, p1);
    asm("{ .reg .pred q; setp.gt.s32 q, %1, 0xBDA00000; @q ex2.approx.ftz.f32 %0, %2; }" : "+f"(p0) : "r"(__float_as_int(x0)), "f"(x0));
    asm("{ .reg .pred q; setp.gt.s32 q, %1, 0xBDA00000; @q ex2.approx.ftz.f32 %0, %2; }" : "+f"(p1) : "r"(__float_as_int(x1)), "f"(x1));
    return F2(p0, p1);
}

// A lane's NS states as pairs
template <int NS> struct States {
    F2 v[NS / 2];
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < NS / 2; ++i) v[i] = F2(0.f);
    }
    // NS floats at p, aligned to 4 * NS bytes.  With `swap` the two halves change places (see sum_channels).
    __device__ __forceinline__ void load(const float* p, bool swap = false) {
        if constexpr (NS == 2) {
            v[0].v = *reinterpret_cast<const unsigned long long*>(p);
        } else {
            const float *lo = p + (swap ? NS / 2 : 0), *hi = p + (swap ? 0 : NS / 2);
#pragma unroll
            for (int i = 0; i < NS / 4; ++i) {
                v[i].v = reinterpret_cast<const unsigned long long*>(lo)[i];
                v[NS / 4 + i].v = reinterpret_cast<const unsigned long long*>(hi)[i];
            }
        }
    }
    __device__ __forceinline__ void store(float* p, bool swap = false) const {
        if constexpr (NS == 2) {
            *reinterpret_cast<unsigned long long*>(p) = v[0].v;
        } else {
            float *lo = p + (swap ? NS / 2 : 0), *hi = p + (swap ? 0 : NS / 2);
#pragma unroll
            for (int i = 0; i < NS / 4; ++i) {
                reinterpret_cast<unsigned long long*>(lo)[i] = v[i].v;
                reinterpret_cast<unsigned long long*>(hi)[i] = v[NS / 4 + i].v;
            }
        }
    }
    // The same in one piece, of 16 bytes where there are as many
    __device__ __forceinline__ void load_wide(const float* p) {
        if constexpr (NS == 2) {
            load(p);
        } else {
#pragma unroll
            for (int i = 0; i < NS / 4; ++i) {
                const ulonglong2 w = reinterpret_cast<const ulonglong2*>(p)[i];
                v[2 * i].v = w.x;
                v[2 * i + 1].v = w.y;
            }
        }
    }
    __device__ __forceinline__ void store_wide(float* p) const {
        if constexpr (NS == 2) {
            store(p);
        } else {
#pragma unroll
            for (int i = 0; i < NS / 4; ++i) reinterpret_cast<ulonglong2*>(p)[i] = make_ulonglong2(v[2 * i].v, v[2 * i + 1].v);
        }
    }
    // A caller's (.., channels, N) tensor; the states behind N are zero.  `wide`: in packs, which wants N = 4 NS and the
    // tensor on a 16-byte boundary.
    __device__ __forceinline__ void load_user(const float* row, int n0, int N, bool swap, bool wide) {
        if (wide) {
            load(row + n0, swap);
        } else {
#pragma unroll
            for (int i = 0; i < NS / 2; ++i) {
                const int n = n0 + (swap && NS > 2 ? (2 * i) ^ (NS / 2) : 2 * i);
                v[i] = F2(n < N ? row[n] : 0.f, n + 1 < N ? row[n + 1] : 0.f);
            }
        }
    }
    // States: the entry points have checked their addresses.
    __device__ __forceinline__ void load_user(const float* row, int n0, int N, bool swap) { load_user(row, n0, N, swap, N == 4 * NS); }
    __device__ __forceinline__ void store_user(float* row, int n0, int N, bool swap) const {
        if (N == 4 * NS) {
            store(row + n0, swap);
        } else {
#pragma unroll
            for (int i = 0; i < NS / 2; ++i) {
                const int n = n0 + (swap && NS > 2 ? (2 * i) ^ (NS / 2) : 2 * i);
                if (n < N) row[n] = v[i].x();
                if (n + 1 < N) row[n + 1] = v[i].y();
            }
        }
    }
    __device__ __forceinline__ void load_user(const float* row, int n0, int N) {
        if (N == 4 * NS) load_wide(row + n0);
        else load_user(row, n0, N, false);
    }
    __device__ __forceinline__ void store_user(float* row, int n0, int N) const {
        if (N == 4 * NS) store_wide(row + n0);
        else store_user(row, n0, N, false);
    }
};

// Where this CTA and lane stand.
template <int NS> struct Place {
    using L = Tile<NS>;
    int64_t b;
    int seg, group, c0, cend;   // c0: first channel of the CTA, cend: end of its group
    int tile_in_group;
    int warp, lane, q;          // q: which states the lane holds
    int slot, c;                // the lane's two channels: their slot in a row of shared memory, the number of the first
    bool live[2];
    bool swap;                  // the lane holds the halves of its states the other way round (backward pass)
    __device__ __forceinline__ explicit Place(const ScanParams& p, bool exchange = false) {
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
        slot = warp * 8 + (lane >> 2);
        c = c0 + (slot % L::kTPR) * L::kVPT + slot / L::kTPR * 2;
        live[0] = c < cend;
        live[1] = c + 1 < cend;
        swap = exchange && (lane & 16) != 0;
    }
    // When a tile is loaded or stored a thread has kVPT consecutive channels of one token; the channels 2 i and
    // 2 i + 1 of them lie at slot(i): threads next to each other write next to each other, and so read the lanes
    // of a warp.
    __device__ __forceinline__ static int row() { return threadIdx.x / L::kTPR; }
    __device__ __forceinline__ static int col() { return threadIdx.x % L::kTPR * L::kVPT; }
    __device__ __forceinline__ static int slot_of(int i) { return i * L::kTPR + threadIdx.x % L::kTPR; }
};

// Packed sequences: what happens at a token of the tile.
struct Marks {
    int first[32], last[32], inside[32];    // sequence that begins / ends here (-1: none); owned by a sequence at all
};

// Returns (to all threads, as a barrier) whether a sequence begins or ends in the tile: most tiles of longer
// sequences have no such token and take the path without looking.
__device__ __forceinline__ bool fill_marks(const ScanParams& p, Marks* m, int64_t t0, int n, int64_t end) {
    int f = -1, l = -1, in = 0;
    if ((int)threadIdx.x < n) {
        const int64_t t = t0 + threadIdx.x;
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
    return __syncthreads_or(f >= 0 || l >= 0) != 0;
}

// The state that token `tt` of the tile continues from: that of the token before it, unless a sequence begins.
template <int NS, bool VARLEN>
__device__ __forceinline__ States<NS> state_before(const ScanParams& p, const Place<NS>& at, const Marks& m, int tt, const float* init,
                                                   const States<NS>& h, int ch) {
    States<NS> r = h;
    if (VARLEN) {
        const int f = m.first[tt];
        if (f >= 0) {
            r.zero();
            if (init != nullptr && at.live[ch]) r.load_user(init + ((int64_t)f * p.channels + at.c + ch) * p.states, at.q * NS, p.states, at.swap);
        }
    }
    return r;
}

// A thread's share of a tile of x and the like: kVPT channels of one token, zeros behind the CTA's channels.
// Where rows start on boundaries it is read as it is.  Otherwise (channel counts or offsets that are no multiple of
// eight) a warp reads its tokens' rows channel next to channel, 32 at a time, and settle() hands the elements to their
// owners through the warp's part of `scratch` (kTok * kCB elements): read by their owners they would be 16 requests
// of 32 sectors each.
template <typename T, int NS, bool VEC> struct Share {
    using L = Tile<NS>;
    static constexpr int V = L::kVPT, kRows = L::kTok / kWarps;
    static_assert(2 * kRows == V, "a warp's rows, 32 channels at a time");
    Pack<T, V> v;
    // `base`: the tensor at this row of the batch; tokens tb .. of which those before `end` exist
    __device__ __forceinline__ void fetch(const T* base, int64_t stride, const Place<NS>& at, int64_t tb, int64_t end) {
        if constexpr (VEC) {
            const int c = at.c0 + at.col();
            const int64_t t = tb + at.row();
            if (t >= end) return;           // whoever reads it asks whether the token exists
            if (c + V <= at.cend) {
                v.load(base + t * stride + c);
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) v.e[i] = c + i < at.cend ? base[t * stride + c + i] : from_f<T>(0.f);
            }
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int64_t t = tb + at.warp * kRows + i / 2;
                const int c = at.c0 + at.lane + (i & 1) * 32;
                v.e[i] = t < end && c < at.cend ? base[t * stride + c] : from_f<T>(0.f);
            }
        }
    }
    __device__ __forceinline__ void settle(const Place<NS>& at, void* scratch) {
        if constexpr (VEC) return;
        T* s = reinterpret_cast<T*>(scratch) + at.warp * kRows * kCB;
        __syncwarp();
#pragma unroll
        for (int i = 0; i < V; ++i) s[i / 2 * kCB + at.lane + (i & 1) * 32] = v.e[i];
        __syncwarp();
        v.load(s + (at.row() - at.warp * kRows) * kCB + at.col());
    }
    __device__ __forceinline__ float get(int i) const { return v.get(i); }
};
// The way back; rows of `stride` elements.  All lanes of a warp take part.
template <typename T, int NS, bool VEC>
__device__ __forceinline__ void store_share(const float (&o)[Tile<NS>::kVPT], T* base, int64_t stride, const Place<NS>& at,
                                            int64_t tb, int64_t end, void* scratch) {
    using Sh = Share<T, NS, VEC>;
    constexpr int V = Sh::V;
    Pack<T, V> k;
#pragma unroll
    for (int i = 0; i < V; ++i) k.set(i, o[i]);
    if constexpr (VEC) {
        const int c = at.c0 + at.col();
        const int64_t t = tb + at.row();
        if (t >= end) return;
        if (c + V <= at.cend) {
            k.store(base + t * stride + c);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (c + i < at.cend) base[t * stride + c + i] = k.e[i];
        }
    } else {
        T* s = reinterpret_cast<T*>(scratch) + at.warp * Sh::kRows * kCB;
        __syncwarp();
        k.store(s + (at.row() - at.warp * Sh::kRows) * kCB + at.col());
        __syncwarp();
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int64_t t = tb + at.warp * Sh::kRows + i / 2;
            const int c = at.c0 + at.lane + (i & 1) * 32;
            if (t < end && c < at.cend) base[t * stride + c] = s[i / 2 * kCB + at.lane + (i & 1) * 32];
        }
    }
}

// A thread's share of B (or C) of a tile: loaded while the tile before is worked on, then put in place.  Zeros
// behind N, behind `end`, and for tokens of no sequence.
template <typename T, int NS> struct BCShare {
    using L = Tile<NS>;
    static constexpr int kEach = L::kTok * L::kNP / kThreads;
    T v[kEach];
    __device__ __forceinline__ void load(const T* src, const int64_t (&st)[3], const ScanParams& p, const Place<NS>& at, int64_t t0,
                                         int64_t end) {
        const T* base = src + at.b * st[0] + at.group * st[2];
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            const int i = threadIdx.x + k * kThreads, t = i / L::kNP, n = i % L::kNP;
            v[k] = n < p.states && t0 + t < end ? base[(t0 + t) * st[1] + n] : from_f<T>(0.f);
        }
    }
    // `swapped`: a second copy with the halves of each lane's states exchanged
    template <bool VARLEN> __device__ __forceinline__ void put(float* dst, const Marks& m, float* swapped = nullptr) const {
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            const int i = threadIdx.x + k * kThreads;
            const float x = !VARLEN || m.inside[i / L::kNP] ? to_f<T>(v[k]) : 0.f;
            dst[i] = x;
            if (swapped != nullptr) swapped[i ^ (NS / 2)] = x;
        }
    }
};

// Step sizes of two channels, from dt + bias
__device__ __forceinline__ F2 step2(const ScanParams& p, float r0, float r1) {
    return p.softplus ? fbla::seq::softplus2(r0, r1) : F2(r0, r1);
}

// Lane q of the four gets the sum over them of v[q].
__device__ __forceinline__ float sum4(const float (&v)[4], int q) {
    const bool odd = q & 1, high = q & 2;
    float a = odd ? v[1] : v[0], b = odd ? v[3] : v[2];
    a += __shfl_xor_sync(0xffffffffu, odd ? v[0] : v[1], 1);
    b += __shfl_xor_sync(0xffffffffu, odd ? v[2] : v[3], 1);
    return (high ? b : a) + __shfl_xor_sync(0xffffffffu, high ? a : b, 2);
}

// A log2(e) of the lane's two channels
template <int NS> __device__ __forceinline__ void load_rates(const ScanParams& p, const Place<NS>& at, States<NS> (&A2)[2]) {
#pragma unroll
    for (int ch = 0; ch < 2; ++ch) {
        A2[ch].zero();
        if (at.live[ch]) A2[ch].load_user(p.A + (int64_t)(at.c + ch) * p.states, at.q * NS, p.states, at.swap, p.wide_A != 0);
#pragma unroll
        for (int i = 0; i < NS / 2; ++i) A2[ch].v[i] = mul2(A2[ch].v[i], F2(1.44269504f));
    }
}

// Workspace of the segmented passes: [batch][segs][channels][kNP] states, then [batch][segs][channels] sums of d.
template <int NS> __device__ __forceinline__ int64_t seg_at(const ScanParams& p, int64_t b, int seg, int c) {
    return (b * p.segs + seg) * p.channels + c;
}

// own + 2^x v, where 2^x is the decay of a whole segment and `near` the same in one product: far from 1 it can leave
// fp32's range although its product with a state does not (e^128 times a state that is still zero; e^-128 times 1e30),
// and is then applied in three factors, which reach from 2^-378 to 2^378; beyond, the product is out of range as well.
// The factors themselves are neither zero nor infinite, so a state that is stays it, as it does token by token.  No
// branch: with one, the next segments' loads wait for it (26 of them: 10 us).
__device__ __forceinline__ float add_decayed(float x, float v, float own, float near) {
    const float t = ex2(fminf(fmaxf(x * (1.f / 3.f), -126.f), 126.f));
    const float far = fmaf(v * t * t, t, own);
    return fabsf(x) > 126.f ? far : near;
}

// v <- own state of segment j + (its decay) v, for the lane's two channels
template <int NS>
__device__ __forceinline__ void add_segment(const ScanParams& p, const Place<NS>& at, int j, const float* seg_v, const float* seg_d,
                                            const States<NS> (&A2)[2], States<NS> (&v)[2]) {
#pragma unroll
    for (int ch = 0; ch < 2; ++ch) {
        if (!at.live[ch]) continue;
        const int64_t k = seg_at<NS>(p, at.b, j, at.c + ch);
        const float sd = seg_d[k];
        States<NS> own;
        own.load(seg_v + k * Tile<NS>::kNP + at.q * NS, at.swap);
#pragma unroll
        for (int i = 0; i < NS / 2; ++i) {
            const F2 x = mul2(F2(sd), A2[ch].v[i]), w = v[ch].v[i], o = own.v[i], near = fma2(decay2(x), w, o);
            const F2 r(add_decayed(x.x(), w.x(), o.x(), near.x()), add_decayed(x.y(), w.y(), o.y(), near.y()));
            v[ch].v[i] = sd == INFINITY ? o : r;
        }
    }
}

template <typename T, int NS> struct FwdSmem {
    using L = Tile<NS>;
    T scratch[L::kTok * kCB];
    float4 dx[L::kTok][kRow4];          // per two channels (d, d x, d, d x)
    float B[L::kTok * L::kNP], C[L::kTok * L::kNP];
    float2 y[L::kTok][kRow2];
    float2 D[kCB / 2], bias[kCB / 2];   // by slot
    Marks marks;
};

template <int NS> __device__ __forceinline__ void load_per_channel(const ScanParams& p, const Place<NS>& at, const float* src, float2* dst) {
    if (at.row() != 0) return;
    const int c = at.c0 + at.col();
#pragma unroll
    for (int i = 0; i < Tile<NS>::kVPT / 2; ++i) {
        const int k = c + 2 * i;
        dst[at.slot_of(i)] = make_float2(src != nullptr && k < at.cend ? src[k] : 0.f, src != nullptr && k + 1 < at.cend ? src[k + 1] : 0.f);
    }
}

// LOCAL: end state of the segment from zero, and the sum of d (infinite when a sequence begins inside, so
// that nothing from before gets through).  Otherwise the outputs.  What the next tile needs from global memory
// is on its way while a tile is worked on.
template <typename T, int NS, bool VARLEN, bool VEC, bool LOCAL>
__global__ void __launch_bounds__(kThreads, 3) scan_fwd_kernel(const ScanParams p, const T* __restrict__ x, const T* __restrict__ dt,
                                                               const T* __restrict__ Bm, const T* __restrict__ Cm,
                                                               const T* __restrict__ z, const float* __restrict__ init,
                                                               T* __restrict__ y, float* __restrict__ fin, float* __restrict__ ckpt,
                                                               float* __restrict__ seg_h, float* __restrict__ seg_d) {
    using L = Tile<NS>;
    constexpr int V = L::kVPT;
    extern __shared__ __align__(16) unsigned char raw_smem[];
    FwdSmem<T, NS>& sm = *reinterpret_cast<FwdSmem<T, NS>*>(raw_smem);
    const Place<NS> at(p);
    if (LOCAL && at.seg == p.segs - 1) return;      // nothing comes behind it
    const int N = p.states, n0 = at.q * NS;
    const int64_t t0 = at.seg * p.seg_len, t1 = min(p.len, t0 + p.seg_len);

    States<NS> A2[2], h[2];
    float sum_d[2] = {0.f, 0.f};
    load_rates<NS>(p, at, A2);
#pragma unroll
    for (int ch = 0; ch < 2; ++ch) {
        h[ch].zero();
        if (!LOCAL && !VARLEN && init != nullptr && at.live[ch]) h[ch].load_user(init + (at.b * p.channels + at.c + ch) * N, n0, N);
    }
    if (!LOCAL)
        for (int j = 0; j < at.seg; ++j) add_segment<NS>(p, at, j, seg_h, seg_d, A2, h);
    const int row = at.row();           // when loading or storing
    load_per_channel<NS>(p, at, p.D, sm.D);
    load_per_channel<NS>(p, at, p.bias, sm.bias);
    const int64_t ntiles = (p.len + L::kTok - 1) / L::kTok;

    Share<T, NS, VEC> px, pd;
    BCShare<T, NS> pB, pC;
    auto fetch = [&](int64_t tb) {
        px.fetch(x + at.b * p.xs[0], p.xs[1], at, tb, t1);
        pd.fetch(dt + at.b * p.ds[0], p.ds[1], at, tb, t1);
        pB.load(Bm, p.bs, p, at, tb, t1);
        if (!LOCAL) pC.load(Cm, p.cs, p, at, tb, t1);
    };
    fetch(t0);
    __syncthreads();
    for (int64_t tb = t0; tb < t1; tb += L::kTok) {
        const bool marked = VARLEN && fill_marks(p, &sm.marks, tb, L::kTok, t1);
        bool ok = tb + row < t1;
        if (VARLEN) ok = ok && sm.marks.inside[row];
        px.settle(at, sm.scratch);
        pd.settle(at, sm.scratch);
        Share<T, NS, VEC> cx, cz;
        cx.v.zero();
        if (ok) cx = px;
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            const float2 bias = sm.bias[at.slot_of(i)];
            const F2 d = ok ? step2(p, pd.get(2 * i) + bias.x, pd.get(2 * i + 1) + bias.y) : F2(0.f);
            const F2 u = mul2(d, F2(cx.get(2 * i), cx.get(2 * i + 1)));
            sm.dx[row][at.slot_of(i)] = make_float4(d.x(), u.x(), d.y(), u.y());
        }
        pB.template put<VARLEN>(sm.B, sm.marks);
        if (!LOCAL) pC.template put<VARLEN>(sm.C, sm.marks);
        __syncthreads();

        if (tb + L::kTok < t1) fetch(tb + L::kTok);
        if (!LOCAL) {
            if (z != nullptr) cz.fetch(z + at.b * p.zs[0], p.zs[1], at, tb, t1);
#pragma unroll
            for (int ch = 0; ch < 2; ++ch)
                if (ckpt != nullptr && at.live[ch])
                    h[ch].store_wide(ckpt + (((at.b * ntiles + tb / L::kTok) * p.channels + at.c + ch) * L::kNP + n0));
        }
        auto work = [&](auto marks) {
            constexpr bool MARKED = decltype(marks)::value;
#pragma unroll 1
            for (int tt = 0; tt < L::kTok; tt += 4) {
                float ys[2][4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float4 v = sm.dx[tt + k][at.slot];
                    States<NS> Bv, Cv;
                    Bv.load_wide(sm.B + (tt + k) * L::kNP + n0);
                    if (!LOCAL) Cv.load_wide(sm.C + (tt + k) * L::kNP + n0);
#pragma unroll
                    for (int ch = 0; ch < 2; ++ch) {
                        const float d = ch ? v.z : v.x;
                        const F2 d2(d), dx2(ch ? v.w : v.y);
                        h[ch] = state_before<NS, MARKED>(p, at, sm.marks, tt + k, init, h[ch], ch);
                        // (not added: what a sequence before it made of the sum ends here)
                        if (LOCAL) sum_d[ch] = MARKED && sm.marks.first[tt + k] >= 0 ? INFINITY : sum_d[ch] + d;
                        F2 s2(0.f);
#pragma unroll
                        for (int i = 0; i < NS / 2; ++i) {
                            h[ch].v[i] = fma2(decay2(mul2(d2, A2[ch].v[i])), h[ch].v[i], mul2(dx2, Bv.v[i]));
                            if (!LOCAL) s2 = i == 0 ? mul2(Cv.v[i], h[ch].v[i]) : fma2(Cv.v[i], h[ch].v[i], s2);
                        }
                        ys[ch][k] = s2.x() + s2.y();
                        if (MARKED && !LOCAL && fin != nullptr) {
                            const int l = sm.marks.last[tt + k];
                            if (l >= 0 && at.live[ch]) h[ch].store_user(fin + ((int64_t)l * p.channels + at.c + ch) * N, n0, N);
                        }
                    }
                }
                if (!LOCAL) {
                    const float y0 = sum4(ys[0], at.q), y1 = sum4(ys[1], at.q);
                    sm.y[tt + at.q][at.slot] = make_float2(y0, y1);
                }
            }
        };
        if (marked) work(std::integral_constant<bool, VARLEN>());
        else work(std::false_type());
        __syncthreads();
        if (!LOCAL) {
            if (z != nullptr) cz.settle(at, sm.scratch);
            float out[V];
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
                const float2 s = sm.y[row][at.slot_of(i)], D = sm.D[at.slot_of(i)];
                out[2 * i] = fmaf(D.x, cx.get(2 * i), s.x);
                out[2 * i + 1] = fmaf(D.y, cx.get(2 * i + 1), s.y);
            }
#pragma unroll
            for (int i = 0; i < V; ++i) {
                if (z != nullptr) out[i] *= cz.get(i) * fbla::seq::sigmoid<T>(cz.get(i));
                if (!ok) out[i] = 0.f;
            }
            store_share<T, NS, VEC>(out, y + at.b * p.len * p.channels, p.channels, at, tb, t1, sm.scratch);
        }
    }
#pragma unroll
    for (int ch = 0; ch < 2; ++ch) {
        if (!at.live[ch]) continue;
        if (LOCAL) {
            const int64_t k = seg_at<NS>(p, at.b, at.seg, at.c + ch);
            h[ch].store(seg_h + k * L::kNP + n0);
            if (at.q == 0) seg_d[k] = sum_d[ch];
        } else if (!VARLEN && fin != nullptr && at.seg == p.segs - 1) {
            h[ch].store_user(fin + (at.b * p.channels + at.c + ch) * N, n0, N);
        }
    }
}

// to[s] = from[s] (or 0) for the sequences without a token: nothing else writes their final state, or the
// gradient of their initial state.
static __global__ void __launch_bounds__(256) scan_empty_kernel(const ScanParams p, const float* __restrict__ from, float* __restrict__ to) {
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x, n = (int64_t)p.channels * p.states;
    if (i >= n) return;
    const int64_t s = blockIdx.y;
    const int64_t tokens = p.cu != nullptr ? (int64_t)p.cu[s + 1] - p.cu[s] : p.len;
    if (tokens <= 0) to[s * n + i] = from != nullptr ? from[s * n + i] : 0.f;
}

// What a thread loads of a tile in the backward passes, as it stands in memory.
template <typename T, int NS, bool VEC> struct BwdShare {
    Share<T, NS, VEC> x, dt, z, dy;
    __device__ __forceinline__ void fetch(const ScanParams& p, const Place<NS>& at, const T* xp, const T* dtp, const T* zp, const T* dyp,
                                          int64_t tb, int64_t end) {
        if (xp != nullptr) x.fetch(xp + at.b * p.xs[0], p.xs[1], at, tb, end);
        dt.fetch(dtp + at.b * p.ds[0], p.ds[1], at, tb, end);
        dy.fetch(dyp + at.b * p.gs[0], p.gs[1], at, tb, end);
        if (zp != nullptr) z.fetch(zp + at.b * p.zs[0], p.zs[1], at, tb, end);
    }
    __device__ __forceinline__ void settle(const Place<NS>& at, bool with_x, bool gated, void* scratch) {
        if (with_x) x.settle(at, scratch);
        dt.settle(at, scratch);
        dy.settle(at, scratch);
        if (gated) z.settle(at, scratch);
    }
    // e = dy silu(z)
    __device__ __forceinline__ float e(int i, bool gated) const {
        const float g = dy.get(i);
        return gated ? g * z.get(i) * fbla::seq::sigmoid<T>(z.get(i)) : g;
    }
    // and dy silu'(z), what dz is of the ungated output
    __device__ __forceinline__ float e(int i, bool gated, float& slope) const {
        const float g = dy.get(i);
        slope = 0.f;
        if (!gated) return g;
        const float zv = z.get(i), gate = fbla::seq::sigmoid<T>(zv), gg = g * gate;
        slope = gg * fmaf(zv, 1.f - gate, 1.f);
        return gg * zv;
    }
};

template <typename T, int NS> struct BwdLocalSmem {
    using L = Tile<NS>;
    T scratch[L::kTok * kCB];
    float4 v[L::kTok][kRow4];           // per two channels (d, e, d, e)
    float C[L::kTok * L::kNP];
    float2 bias[kCB / 2];
    Marks marks;
};

// What a segment passes to the one before it, from zero: a G of its first token.  seg_d as in the forward.
template <typename T, int NS, bool VARLEN, bool VEC>
__global__ void __launch_bounds__(kThreads, 3) scan_bwd_local_kernel(const ScanParams p, const T* __restrict__ dt, const T* __restrict__ Cm,
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
    States<NS> A2[2], g[2];
    float sum_d[2] = {0.f, 0.f};
    load_rates<NS>(p, at, A2);
#pragma unroll
    for (int ch = 0; ch < 2; ++ch) {
        g[ch].zero();
        if (!VARLEN && dfin != nullptr && at.live[ch] && at.seg == p.segs - 1)
            g[ch].load_user(dfin + (at.b * p.channels + at.c + ch) * N, n0, N);
    }
    load_per_channel<NS>(p, at, p.bias, sm.bias);
    const int row = at.row();
    BwdShare<T, NS, VEC> next;
    BCShare<T, NS> pC;
    auto fetch = [&](int64_t tb) {
        next.fetch(p, at, nullptr, dt, z, dy, tb, t1);
        pC.load(Cm, p.cs, p, at, tb, t1);
    };
    const int64_t tlast = t0 + (t1 - 1 - t0) / L::kTok * L::kTok;
    fetch(tlast);
    for (int64_t tb = tlast; tb >= t0; tb -= L::kTok) {
        __syncthreads();
        const bool marked = VARLEN && fill_marks(p, &sm.marks, tb, L::kTok, t1);
        bool ok = tb + row < t1;
        if (VARLEN) ok = ok && sm.marks.inside[row];
        next.settle(at, false, z != nullptr, sm.scratch);
#pragma unroll
        for (int i = 0; i < L::kVPT / 2; ++i) {
            const float2 bias = sm.bias[at.slot_of(i)];
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            if (ok) {
                const F2 d = step2(p, next.dt.get(2 * i) + bias.x, next.dt.get(2 * i + 1) + bias.y);
                v = make_float4(d.x(), next.e(2 * i, z != nullptr), d.y(), next.e(2 * i + 1, z != nullptr));
            }
            sm.v[row][at.slot_of(i)] = v;
        }
        pC.template put<VARLEN>(sm.C, sm.marks);
        __syncthreads();
        if (tb > t0) fetch(tb - L::kTok);
        auto work = [&](auto marks) {
            constexpr bool MARKED = decltype(marks)::value;
#pragma unroll 4
            for (int tt = L::kTok - 1; tt >= 0; --tt) {
                const float4 v = sm.v[tt][at.slot];
                States<NS> Cv;
                Cv.load(sm.C + tt * L::kNP + n0);
#pragma unroll
                for (int ch = 0; ch < 2; ++ch) {
                    const F2 d2(ch ? v.z : v.x), e2(ch ? v.w : v.y);
                    if (MARKED && dfin != nullptr) {
                        const int l = sm.marks.last[tt];
                        if (l >= 0 && at.live[ch]) g[ch].load_user(dfin + ((int64_t)l * p.channels + at.c + ch) * N, n0, N);
                    }
                    sum_d[ch] += d2.x();
#pragma unroll
                    for (int i = 0; i < NS / 2; ++i) g[ch].v[i] = mul2(decay2(mul2(d2, A2[ch].v[i])), fma2(e2, Cv.v[i], g[ch].v[i]));
                    if (MARKED && sm.marks.first[tt] >= 0) {
                        sum_d[ch] = INFINITY;
                        g[ch].zero();
                    }
                }
            }
        };
        if (marked) work(std::integral_constant<bool, VARLEN>());
        else work(std::false_type());
    }
#pragma unroll
    for (int ch = 0; ch < 2; ++ch) {
        if (!at.live[ch]) continue;
        const int64_t k = seg_at<NS>(p, at.b, at.seg, at.c + ch);
        g[ch].store(seg_g + k * L::kNP + n0);
        if (at.q == 0) seg_d[k] = sum_d[ch];
    }
}

__device__ __forceinline__ F2 add2(F2 a, F2 b) {
    F2 r;
    asm("add.rn.ftz.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ F2 shfl2(F2 a, int mask) {
    return F2(__shfl_xor_sync(0xffffffffu, a.x(), mask), __shfl_xor_sync(0xffffffffu, a.y(), mask));
}
__device__ __forceinline__ F2 pick(bool first, F2 a, F2 b) { return F2(first ? a.x() : b.x(), first ? a.y() : b.y()); }

// Sums of dB and dC over the channels of a warp (lane bits 4, 3 and 2), by exchanges that halve what a lane holds:
// first the halves of its states -- lanes with bit 4 hold them the other way round, so that every lane gives away its
// second half and nothing has to be selected --, then dB against dC, then one of two pairs (of two values with four
// states).  out: what is left, for consecutive columns of [dB | dC] from the returned one on.
template <int NS> __device__ __forceinline__ int sum_channels(const F2 (&dB)[NS / 2], const F2 (&dC)[NS / 2], int lane, float (&out)[NS >= 8 ? 2 : 1]) {
    const bool b4 = lane & 16, b3 = lane & 8, b2 = lane & 4;
    const int n0 = (lane & 3) * NS;
    if constexpr (NS == 2) {
        F2 v = add2(pick(!b4, dB[0], dC[0]), shfl2(pick(b4, dB[0], dC[0]), 16));
        const float give = b3 ? v.x() : v.y(), keep = b3 ? v.y() : v.x();
        out[0] = keep + __shfl_xor_sync(0xffffffffu, give, 8);
        out[0] += __shfl_xor_sync(0xffffffffu, out[0], 4);
        return (b4 ? Tile<NS>::kNP : 0) + n0 + (b3 ? 1 : 0);
    } else {
        constexpr int H = NS / 4;
        F2 v[H];
#pragma unroll
        for (int i = 0; i < H; ++i) {
            const F2 b = add2(dB[i], shfl2(dB[H + i], 16)), c = add2(dC[i], shfl2(dC[H + i], 16));
            v[i] = add2(pick(!b3, b, c), shfl2(pick(b3, b, c), 8));
        }
        const int col = (b3 ? Tile<NS>::kNP : 0) + n0 + (b4 ? NS / 2 : 0);
        if constexpr (NS == 4) {
            const float give = b2 ? v[0].x() : v[0].y(), keep = b2 ? v[0].y() : v[0].x();
            out[0] = keep + __shfl_xor_sync(0xffffffffu, give, 4);
            return col + (b2 ? 1 : 0);
        } else {
            const F2 r = add2(pick(!b2, v[0], v[1]), shfl2(pick(b2, v[0], v[1]), 4));
            r.get(out[0], out[1]);
            return col + (b2 ? 2 : 0);
        }
    }
}

template <int NS> struct BwdSmem {
    using L = Tile<NS>;
    static constexpr int kSubs = L::kTok / L::kSub;
    static_assert(kSubs * 2 * kThreads * NS >= L::kTok * kCB, "`start` also serves as the loads' scratch");
    float4 dx[L::kTok][kRow4];                      // per two channels (d, d x, d, d x); behind its reverse pass sum A r for d x
    float2 e[L::kTok][kRow2];                       // dy silu(z)
    float2 slope[L::kTok][kRow2];                   // dy silu'(z)
    float2 y[L::kTok][kRow2];                       // s = sum C h
    float2 gB[L::kTok][kRow2];                      // sum G B
    float B[2][L::kTok * L::kNP], C[2][L::kTok * L::kNP];       // the second with the halves of the states exchanged
    float start[kSubs][2][kThreads][NS];            // each thread's states at the starts of the sub-tiles
    float dbc[kWarps][L::kTok][2 * L::kNP];         // per warp: sums of dB, dC over its channels
    float4 acc[L::kVPT / 2][kThreads];              // each thread's sums for dD (two channels) and dbias
    float2 D[kCB / 2], bias[kCB / 2];
    Marks marks;
};

__device__ __forceinline__ void prefetch(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

// All gradients of one segment, tile after tile from its end.  In a tile the states are formed again from the
// checkpoint, first up to the starts of its sub-tiles; then sub-tile after sub-tile, from the last one, with
// the decays and states of its tokens in registers, the reverse recurrence.
// part_bc: [channel tile of the group][batch][token][group][2][kNP] sums over the CTA's channels;
// part_A [batch][segs][channels][N], part_D / part_bias [batch][segs][channels].
template <typename T, int NS, bool VARLEN, bool VEC>
__global__ void __launch_bounds__(kThreads, 2) scan_bwd_kernel(
    const ScanParams p, const T* __restrict__ x, const T* __restrict__ dt, const T* __restrict__ Bm, const T* __restrict__ Cm,
    const T* __restrict__ z, const float* __restrict__ init, const T* __restrict__ dy, const float* __restrict__ dfin,
    const float* __restrict__ ckpt, const float* __restrict__ seg_g, const float* __restrict__ seg_d, T* __restrict__ dx,
    T* __restrict__ ddt, T* __restrict__ dz, float* __restrict__ dinit, float* __restrict__ part_bc, float* __restrict__ part_A,
    float* __restrict__ part_D, float* __restrict__ part_bias) {
    using L = Tile<NS>;
    constexpr int K = L::kSub, V = L::kVPT, P = NS / 2;
    extern __shared__ __align__(16) unsigned char raw_smem[];
    BwdSmem<NS>& sm = *reinterpret_cast<BwdSmem<NS>*>(raw_smem);
    const Place<NS> at(p, NS > 2);
    const int N = p.states, n0 = at.q * NS;
    const int64_t t0 = at.seg * p.seg_len, t1 = min(p.len, t0 + p.seg_len);
    const int64_t ntiles = (p.len + L::kTok - 1) / L::kTok;

    // A2 = A log2(e); the sum with A itself is formed with A2 and scaled back once
    States<NS> A2[2], g[2], dA[2];      // g: a G of the token behind
    load_rates<NS>(p, at, A2);
#pragma unroll
    for (int ch = 0; ch < 2; ++ch) {
        g[ch].zero();
        dA[ch].zero();
        if (!VARLEN && dfin != nullptr && at.live[ch] && at.seg == p.segs - 1)
            g[ch].load_user(dfin + (at.b * p.channels + at.c + ch) * N, n0, N, at.swap);
    }
    for (int j = p.segs - 1; j > at.seg; --j) add_segment<NS>(p, at, j, seg_g, seg_d, A2, g);
    const int row = at.row();
    const float *sB = sm.B[at.swap] + n0, *sC = sm.C[at.swap] + n0;     // the lane's states of token 0
    load_per_channel<NS>(p, at, p.D, sm.D);
    load_per_channel<NS>(p, at, p.bias, sm.bias);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) sm.acc[i][threadIdx.x] = make_float4(0.f, 0.f, 0.f, 0.f);

    for (int64_t tb = t0 + (t1 - 1 - t0) / L::kTok * L::kTok; tb >= t0; tb -= L::kTok) {
        __syncthreads();
        const bool marked = VARLEN && fill_marks(p, &sm.marks, tb, L::kTok, t1);
        const int64_t t = tb + row;
        bool ok = t < t1;
        if (VARLEN) ok = ok && sm.marks.inside[row];
        void* scratch = sm.start;       // free outside the passes
        States<NS> h[2];
#pragma unroll
        for (int ch = 0; ch < 2; ++ch) {
            h[ch].zero();
            if (at.live[ch]) h[ch].load(ckpt + (((at.b * ntiles + tb / L::kTok) * p.channels + at.c + ch) * L::kNP + n0), at.swap);
        }
        {
            BwdShare<T, NS, VEC> in;
            in.fetch(p, at, x, dt, z, dy, tb, t1);
            BCShare<T, NS> bc;
            bc.load(Bm, p.bs, p, at, tb, t1);
            bc.template put<VARLEN>(sm.B[0], sm.marks, NS > 2 ? sm.B[1] : nullptr);
            bc.load(Cm, p.cs, p, at, tb, t1);
            bc.template put<VARLEN>(sm.C[0], sm.marks, NS > 2 ? sm.C[1] : nullptr);
            in.settle(at, true, z != nullptr, scratch);
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
                const int s = at.slot_of(i);
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                float2 e = make_float2(0.f, 0.f), slope = e;
                if (ok) {
                    const float2 bias = sm.bias[s];
                    const float x0 = in.x.get(2 * i), x1 = in.x.get(2 * i + 1);
                    const F2 d = step2(p, in.dt.get(2 * i) + bias.x, in.dt.get(2 * i + 1) + bias.y);
                    const F2 u = mul2(d, F2(x0, x1));
                    v = make_float4(d.x(), u.x(), d.y(), u.y());
                    e.x = in.e(2 * i, z != nullptr, slope.x);
                    e.y = in.e(2 * i + 1, z != nullptr, slope.y);
                    float2& sum = *reinterpret_cast<float2*>(&sm.acc[i][threadIdx.x].x);
                    sum = make_float2(fmaf(e.x, x0, sum.x), fmaf(e.y, x1, sum.y));
                }
                sm.dx[row][s] = v;
                sm.e[row][s] = e;
                if (z != nullptr) sm.slope[row][s] = slope;
            }
        }
        __syncthreads();
        if (tb > t0) {                  // the tile before this one, on its way to L2
            const int64_t u = t - L::kTok;
            const int c = at.c0 + at.col();
            if (c < at.cend) {
                prefetch(x + at.b * p.xs[0] + u * p.xs[1] + c);
                prefetch(dt + at.b * p.ds[0] + u * p.ds[1] + c);
                prefetch(dy + at.b * p.gs[0] + u * p.gs[1] + c);
                if (z != nullptr) prefetch(z + at.b * p.zs[0] + u * p.zs[1] + c);
            }
        }

        auto work = [&](auto marks) {
            constexpr bool MARKED = decltype(marks)::value;
#pragma unroll 1
            for (int sub = 0; sub < BwdSmem<NS>::kSubs; ++sub) {
#pragma unroll
                for (int ch = 0; ch < 2; ++ch) h[ch].store_wide(sm.start[sub][ch][threadIdx.x]);
                if (sub == BwdSmem<NS>::kSubs - 1) break;
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    const int tt = sub * K + k;
                    const float4 v = sm.dx[tt][at.slot];
                    States<NS> Bv;
                    Bv.load_wide(sB + tt * L::kNP);
#pragma unroll
                    for (int ch = 0; ch < 2; ++ch) {
                        const F2 d2(ch ? v.z : v.x), dx2(ch ? v.w : v.y);
                        h[ch] = state_before<NS, MARKED>(p, at, sm.marks, tt, init, h[ch], ch);
#pragma unroll
                        for (int i = 0; i < P; ++i) h[ch].v[i] = fma2(decay2(mul2(d2, A2[ch].v[i])), h[ch].v[i], mul2(dx2, Bv.v[i]));
                    }
                }
            }
#pragma unroll 1
            for (int sub = BwdSmem<NS>::kSubs - 1; sub >= 0; --sub) {
                States<NS> a[2][K], hs[2][K + 1];
#pragma unroll
                for (int ch = 0; ch < 2; ++ch) hs[ch][0].load_wide(sm.start[sub][ch][threadIdx.x]);
#pragma unroll
                for (int k0 = 0; k0 < K; k0 += 4) {
                    float ys[2][4];
#pragma unroll
                    for (int k = k0; k < k0 + 4; ++k) {
                        const int tt = sub * K + k;
                        const float4 v = sm.dx[tt][at.slot];
                        States<NS> Bv, Cv;
                        Bv.load_wide(sB + tt * L::kNP);
                        Cv.load_wide(sC + tt * L::kNP);
#pragma unroll
                        for (int ch = 0; ch < 2; ++ch) {
                            const F2 d2(ch ? v.z : v.x), dx2(ch ? v.w : v.y);
                            const States<NS> hp = state_before<NS, MARKED>(p, at, sm.marks, tt, init, hs[ch][k], ch);
                            F2 s2(0.f);
#pragma unroll
                            for (int i = 0; i < P; ++i) {
                                a[ch][k].v[i] = decay2(mul2(d2, A2[ch].v[i]));
                                hs[ch][k + 1].v[i] = fma2(a[ch][k].v[i], hp.v[i], mul2(dx2, Bv.v[i]));
                                s2 = i == 0 ? mul2(Cv.v[i], hs[ch][k + 1].v[i]) : fma2(Cv.v[i], hs[ch][k + 1].v[i], s2);
                            }
                            ys[ch][k - k0] = s2.x() + s2.y();
                        }
                    }
                    const float y0 = sum4(ys[0], at.q), y1 = sum4(ys[1], at.q);
                    sm.y[sub * K + k0 + at.q][at.slot] = make_float2(y0, y1);
                }
#pragma unroll
                for (int k0 = K - 4; k0 >= 0; k0 -= 4) {
                    float gb[2][4], ra[2][4];
#pragma unroll
                    for (int k = k0 + 3; k >= k0; --k) {
                        const int tt = sub * K + k;
                        const float4 v = sm.dx[tt][at.slot];
                        const float2 e = sm.e[tt][at.slot];
                        States<NS> Bv, Cv;
                        Bv.load_wide(sB + tt * L::kNP);
                        Cv.load_wide(sC + tt * L::kNP);
                        F2 dB[P], dC[P];
#pragma unroll
                        for (int ch = 0; ch < 2; ++ch) {
                            const F2 d2(ch ? v.z : v.x), dx2(ch ? v.w : v.y), e2(ch ? e.y : e.x);
                            if (MARKED && dfin != nullptr) {
                                const int l = sm.marks.last[tt];
                                if (l >= 0 && at.live[ch]) g[ch].load_user(dfin + ((int64_t)l * p.channels + at.c + ch) * N, n0, N, at.swap);
                            }
                            const States<NS> hp = state_before<NS, MARKED>(p, at, sm.marks, tt, init, hs[ch][k], ch);
                            F2 gb2(0.f), ra2(0.f);
#pragma unroll
                            for (int i = 0; i < P; ++i) {
                                const F2 G = fma2(e2, Cv.v[i], g[ch].v[i]);
                                dB[i] = ch == 0 ? mul2(dx2, G) : fma2(dx2, G, dB[i]);
                                dC[i] = ch == 0 ? mul2(e2, hs[ch][k + 1].v[i]) : fma2(e2, hs[ch][k + 1].v[i], dC[i]);
                                gb2 = i == 0 ? mul2(G, Bv.v[i]) : fma2(G, Bv.v[i], gb2);
                                g[ch].v[i] = mul2(a[ch][k].v[i], G);
                                const F2 r = mul2(g[ch].v[i], hp.v[i]);
                                ra2 = i == 0 ? mul2(r, A2[ch].v[i]) : fma2(r, A2[ch].v[i], ra2);
                                dA[ch].v[i] = fma2(d2, r, dA[ch].v[i]);
                            }
                            gb[ch][k - k0] = gb2.x() + gb2.y();
                            ra[ch][k - k0] = ra2.x() + ra2.y();
                            if (MARKED) {
                                const int f = sm.marks.first[tt];
                                if (f >= 0) {
                                    if (dinit != nullptr && at.live[ch]) g[ch].store_user(dinit + ((int64_t)f * p.channels + at.c + ch) * N, n0, N, at.swap);
                                    g[ch].zero();
                                }
                            }
                        }
                        float sums[NS >= 8 ? 2 : 1];
                        const int col = sum_channels<NS>(dB, dC, at.lane, sums);
                        if constexpr (NS >= 8) *reinterpret_cast<float2*>(&sm.dbc[at.warp][tt][col]) = make_float2(sums[0], sums[1]);
                        else sm.dbc[at.warp][tt][col] = sums[0];
                    }
                    const float g0 = sum4(gb[0], at.q), g1 = sum4(gb[1], at.q), r0 = sum4(ra[0], at.q), r1 = sum4(ra[1], at.q);
                    __syncwarp();               // the four lanes of a channel are done with its d x of these tokens
                    const int tt = sub * K + k0 + at.q;
                    sm.gB[tt][at.slot] = make_float2(g0, g1);
                    sm.dx[tt][at.slot].y = r0 * 0.69314718f;
                    sm.dx[tt][at.slot].w = r1 * 0.69314718f;
                }
            }
        };
        if (marked) work(std::integral_constant<bool, VARLEN>());
        else work(std::false_type());
        __syncthreads();
        for (int i = threadIdx.x; i < L::kTok * 2 * L::kNP; i += kThreads) {
            const int tt = i / (2 * L::kNP), w = i % (2 * L::kNP);
            if (tb + tt >= t1) continue;
            float s = 0.f;
#pragma unroll
            for (int k = 0; k < kWarps; ++k) s += sm.dbc[k][tt][w];
            // behind the last sequence its state still stands, and may be infinite: 0 times it is not 0
            if (VARLEN && !sm.marks.inside[tt]) s = 0.f;
            part_bc[((((int64_t)at.tile_in_group * p.batch + at.b) * p.len + tb + tt) * p.groups + at.group) * (2 * L::kNP) + w] = s;
        }
        if (!VEC || t < t1) {           // without packs all lanes of a warp take part in its loads and stores
            Share<T, NS, VEC> xv, dtv;
            xv.fetch(x + at.b * p.xs[0], p.xs[1], at, tb, t1);
            dtv.fetch(dt + at.b * p.ds[0], p.ds[1], at, tb, t1);
            xv.settle(at, scratch);
            dtv.settle(at, scratch);
            float ox[V], od[V], oz[V];
#pragma unroll
            for (int i = 0; i < V; i += 2) {
                const int s = at.slot_of(i / 2);
                const float4 v = sm.dx[row][s];             // d, sum A r
                const float2 e = sm.e[row][s], gB = sm.gB[row][s], D = sm.D[s], bias = sm.bias[s];
                const float x0 = xv.get(i), x1 = xv.get(i + 1);
                ox[i] = fmaf(v.x, gB.x, D.x * e.x);
                ox[i + 1] = fmaf(v.z, gB.y, D.y * e.y);
                od[i] = fmaf(x0, gB.x, v.y);
                od[i + 1] = fmaf(x1, gB.y, v.w);
                if (p.softplus) {
                    const float r0 = dtv.get(i) + bias.x, r1 = dtv.get(i + 1) + bias.y;
                    od[i] *= r0 > 20.f ? 1.f : fbla::seq::sigmoid<T>(r0);
                    od[i + 1] *= r1 > 20.f ? 1.f : fbla::seq::sigmoid<T>(r1);
                }
                if (z != nullptr) {
                    const float2 slope = sm.slope[row][s], y2 = sm.y[row][s];
                    oz[i] = slope.x * fmaf(D.x, x0, y2.x);
                    oz[i + 1] = slope.y * fmaf(D.y, x1, y2.y);
                }
                if (!ok) ox[i] = ox[i + 1] = od[i] = od[i + 1] = oz[i] = oz[i + 1] = 0.f;
                float2& sum = *reinterpret_cast<float2*>(&sm.acc[i / 2][threadIdx.x].z);
                sum = make_float2(sum.x + od[i], sum.y + od[i + 1]);
            }
            const int64_t o = at.b * p.len * p.channels;
            store_share<T, NS, VEC>(ox, dx + o, p.channels, at, tb, t1, scratch);
            store_share<T, NS, VEC>(od, ddt + o, p.channels, at, tb, t1, scratch);
            if (z != nullptr) store_share<T, NS, VEC>(oz, dz + o, p.channels, at, tb, t1, scratch);
        }
    }
    __syncthreads();
    const int64_t bs = at.b * p.segs + at.seg;
    if ((int)threadIdx.x < kCB && at.c0 + (int)threadIdx.x < at.cend) {
        const int k = threadIdx.x / V, i = threadIdx.x % V;
        float sD = 0.f, sb = 0.f;
        for (int r = 0; r < L::kTok; ++r) {
            const float4 v = sm.acc[i / 2][r * L::kTPR + k];
            sD += i & 1 ? v.y : v.x;
            sb += i & 1 ? v.w : v.z;
        }
        part_D[bs * p.channels + at.c0 + threadIdx.x] = sD;
        part_bias[bs * p.channels + at.c0 + threadIdx.x] = sb;
    }
#pragma unroll
    for (int ch = 0; ch < 2; ++ch) {
        if (!at.live[ch]) continue;
        dA[ch].store_user(part_A + (bs * p.channels + at.c + ch) * N, n0, N, at.swap);
        if (!VARLEN && dinit != nullptr && at.seg == 0) g[ch].store_user(dinit + (at.b * p.channels + at.c + ch) * N, n0, N, at.swap);
    }
}

// What follows the backward pass, in one launch: dB, dC (batch, token, group, N) from the channel tiles' sums, and dA, dD
// and d_dt_bias from the segments', all in order.  The first `bc_blocks` blocks do the former.
struct SumParams {
    const float *bc, *A, *D, *bias;
    float *dA, *dD, *dbias;
    int64_t bc_rows, seg_rows, bc_blocks;
    int tiles, channels, states;
};
template <typename T, int NP>
__global__ void __launch_bounds__(256) scan_sums_kernel(const SumParams p, T* __restrict__ dB, T* __restrict__ dC) {
    if ((int64_t)blockIdx.x < p.bc_blocks) {
        const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
        if (i >= p.bc_rows * 2 * NP) return;
        const int64_t r = i / (2 * NP);
        const int w = (int)(i % (2 * NP)), n = w % NP;
        if (n >= p.states) return;
        float s = 0.f;
#pragma unroll 4
        for (int k = 0; k < p.tiles; ++k) s += p.bc[k * p.bc_rows * 2 * NP + i];
        (w < NP ? dB : dC)[r * p.states + n] = from_f<T>(s);
        return;
    }
    const int64_t nA = (int64_t)p.channels * p.states, i = ((int64_t)blockIdx.x - p.bc_blocks) * 256 + threadIdx.x;
    const float* in;
    float* out;
    int64_t n, at;
    if (i < nA) {
        in = p.A, out = p.dA, n = nA, at = i;
    } else {
        at = i - nA, n = p.channels;
        if (at < n) {
            in = p.D, out = p.dD;
        } else {
            at -= n;
            in = p.bias, out = p.dbias;
        }
        if (at >= n || out == nullptr) return;
    }
    float s = 0.f;
#pragma unroll 4
    for (int64_t r = 0; r < p.seg_rows; ++r) s += in[r * n + at];
    out[at] = s;
}

// One token per row, the state updated in place.  Four lanes per channel: a state is read and written once, 16 bytes
// per lane where N allows, and that traffic is what bounds it (8 N bytes per channel against 8 of everything else).
constexpr int kStepChannels = 32;
template <typename T, int NS>
__global__ void __launch_bounds__(4 * kStepChannels) scan_step_kernel(const ScanParams p, const T* __restrict__ x, const T* __restrict__ dt,
                                                                      const T* __restrict__ Bm, const T* __restrict__ Cm,
                                                                      const T* __restrict__ z, float* __restrict__ state, T* __restrict__ y) {
    const int64_t b = blockIdx.y;
    const int c = blockIdx.x * kStepChannels + threadIdx.x / 4, q = threadIdx.x & 3, N = p.states, n0 = q * NS;
    const bool live = c < p.channels;
    float acc = 0.f, xv = 0.f;
    if (live) {
        float* hp = state + (b * p.channels + c) * N;
        const int group = c / (p.channels / p.groups);
        States<NS> h, A;
        h.load_user(hp, n0, N);
        if (p.wide_A) A.load_wide(p.A + (int64_t)c * N + n0);
        else A.load_user(p.A + (int64_t)c * N, n0, N, false, false);
        const T* Bp = Bm + b * p.bs[0] + group * p.bs[2];
        const T* Cp = Cm + b * p.cs[0] + group * p.cs[2];
        xv = to_f<T>(x[b * p.xs[0] + c]);
        float d = to_f<T>(dt[b * p.ds[0] + c]);
        if (p.bias != nullptr) d += p.bias[c];
        if (p.softplus) d = fbla::seq::softplus(d);
        Pack<T, NS> Bv, Cv;
        if (p.vec) {                    // N is 4 NS and the rows of B and C start on boundaries
            Bv.load(Bp + n0);
            Cv.load(Cp + n0);
        } else {
#pragma unroll
            for (int i = 0; i < NS; ++i) {
                Bv.e[i] = n0 + i < N ? Bp[n0 + i] : from_f<T>(0.f);
                Cv.e[i] = n0 + i < N ? Cp[n0 + i] : from_f<T>(0.f);
            }
        }
        F2 s2(0.f);
#pragma unroll
        for (int i = 0; i < NS / 2; ++i) {
            const F2 a = decay2(mul2(F2(d), mul2(A.v[i], F2(1.44269504f))));
            h.v[i] = fma2(a, h.v[i], mul2(F2(d * xv), F2(Bv.get(2 * i), Bv.get(2 * i + 1))));
            s2 = fma2(F2(Cv.get(2 * i), Cv.get(2 * i + 1)), h.v[i], s2);
        }
        acc = s2.x() + s2.y();
        h.store_user(hp, n0, N);
    }
    acc += __shfl_xor_sync(0xffffffffu, acc, 1);
    acc += __shfl_xor_sync(0xffffffffu, acc, 2);
    if (live && q == 0) {
        if (p.D != nullptr) acc = fmaf(p.D[c], xv, acc);
        if (z != nullptr) {
            const float zv = to_f<T>(z[b * p.zs[0] + c]);
            acc *= zv * fbla::seq::sigmoid<T>(zv);
        }
        y[b * p.channels + c] = from_f<T>(acc);
    }
}

// ---- launches --------------------------------------------------------------------------------------

inline int ns_of(int N) { return N <= 8 ? 2 : N <= 16 ? 4 : 8; }
inline int np_of(int N) { return 4 * ns_of(N); }
inline int tok_of(int N) { return ns_of(N) >= 8 ? 16 : 32; }
inline int tiles_per_group(const ScanParams& p) { return (p.channels / p.groups + kCB - 1) / kCB; }

inline int64_t seg_floats(const ScanParams& p) { return p.segs > 1 ? (int64_t)p.batch * p.segs * p.channels * (np_of(p.states) + 1) : 0; }

template <typename Kernel> cudaError_t allow_smem(Kernel k, size_t bytes) {
    return bytes > 48 * 1024 ? cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) : cudaSuccess;
}

struct ScanTensors {
    const void *x, *dt, *B, *C, *z, *dy;
    const float *init, *dfin;
    void *y, *dx, *ddt, *dB, *dC, *dz;
    float *fin, *ckpt, *dA, *dD, *dbias, *dinit, *ws;
};

inline dim3 scan_grid(const ScanParams& p) { return dim3((unsigned)(p.groups * tiles_per_group(p)), (unsigned)p.segs, (unsigned)p.batch); }

inline cudaError_t fill_empty(const ScanParams& p, const float* from, float* to, cudaStream_t st) {
    if (to == nullptr || p.num_seqs == 0 || (p.cu == nullptr && p.len > 0)) return cudaSuccess;
    const int64_t n = (int64_t)p.channels * p.states;
    scan_empty_kernel<<<dim3((unsigned)((n + 255) / 256), (unsigned)p.num_seqs), 256, 0, st>>>(p, from, to);
    fbla::note_launches(1);
    return cudaGetLastError();
}

template <typename T, int NS, bool VARLEN, bool VEC> cudaError_t run_fwd(const ScanParams& p, const ScanTensors& a, cudaStream_t st) {
    if (cudaError_t e = fill_empty(p, a.init, a.fin, st)) return e;
    if (p.len == 0 || p.batch == 0) return cudaSuccess;
    using S = FwdSmem<T, NS>;
    float* seg_h = a.ws;
    float* seg_d = p.segs > 1 ? a.ws + (int64_t)p.batch * p.segs * p.channels * Tile<NS>::kNP : nullptr;
    if (p.segs > 1) {
        auto k = scan_fwd_kernel<T, NS, VARLEN, VEC, true>;
        if (cudaError_t e = allow_smem(k, sizeof(S))) return e;
        k<<<scan_grid(p), kThreads, sizeof(S), st>>>(p, (const T*)a.x, (const T*)a.dt, (const T*)a.B, (const T*)a.C, nullptr, a.init, nullptr,
                                                     nullptr, nullptr, seg_h, seg_d);
        fbla::note_launches(1);
    }
    auto k = scan_fwd_kernel<T, NS, VARLEN, VEC, false>;
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
inline BwdLayout bwd_layout(const ScanParams& p) {
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

template <typename T, int NS, bool VARLEN, bool VEC> cudaError_t run_bwd(const ScanParams& p, const ScanTensors& a, cudaStream_t st) {
    if (cudaError_t e = fill_empty(p, a.dfin, a.dinit, st)) return e;
    const BwdLayout l = bwd_layout(p);
    const bool any = p.len > 0 && p.batch > 0;
    const int64_t rows = any ? (int64_t)p.batch * p.segs : 0;
    if (any) {
        float* seg_g = a.ws + l.seg;
        float* seg_d = seg_g + (int64_t)p.batch * p.segs * p.channels * Tile<NS>::kNP;
        if (p.segs > 1) {
            auto k = scan_bwd_local_kernel<T, NS, VARLEN, VEC>;
            using S = BwdLocalSmem<T, NS>;
            if (cudaError_t e = allow_smem(k, sizeof(S))) return e;
            k<<<scan_grid(p), kThreads, sizeof(S), st>>>(p, (const T*)a.dt, (const T*)a.C, (const T*)a.z, (const T*)a.dy, a.dfin, seg_g, seg_d);
            fbla::note_launches(1);
        }
        auto k = scan_bwd_kernel<T, NS, VARLEN, VEC>;
        using S = BwdSmem<NS>;
        if (cudaError_t e = allow_smem(k, sizeof(S))) return e;
        k<<<scan_grid(p), kThreads, sizeof(S), st>>>(p, (const T*)a.x, (const T*)a.dt, (const T*)a.B, (const T*)a.C, (const T*)a.z, a.init,
                                                     (const T*)a.dy, a.dfin, a.ckpt, seg_g, seg_d, (T*)a.dx, (T*)a.ddt, (T*)a.dz, a.dinit,
                                                     a.ws + l.bc, a.ws + l.A, a.ws + l.D, a.ws + l.bias);
        fbla::note_launches(1);
        if (cudaError_t e = cudaGetLastError()) return e;
    }
    SumParams q;
    q.bc = a.ws + l.bc;
    q.A = a.ws + l.A;
    q.D = a.ws + l.D;
    q.bias = a.ws + l.bias;
    q.dA = a.dA;
    q.dD = a.dD;
    q.dbias = a.dbias;
    q.bc_rows = any ? (int64_t)p.batch * p.len * p.groups : 0;
    q.seg_rows = rows;
    q.bc_blocks = (q.bc_rows * 2 * Tile<NS>::kNP + 255) / 256;
    q.tiles = tiles_per_group(p);
    q.channels = p.channels;
    q.states = p.states;
    const int64_t blocks = q.bc_blocks + ((int64_t)p.channels * (p.states + 2) + 255) / 256;
    if (blocks > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
    scan_sums_kernel<T, Tile<NS>::kNP><<<(unsigned)blocks, 256, 0, st>>>(q, (T*)a.dB, (T*)a.dC);
    fbla::note_launches(1);
    return cudaGetLastError();
}

template <typename T, int NS> cudaError_t run_step(const ScanParams& p, const ScanTensors& a, cudaStream_t st) {
    const dim3 grid((unsigned)((p.channels + kStepChannels - 1) / kStepChannels), (unsigned)p.batch);
    scan_step_kernel<T, NS><<<grid, 4 * kStepChannels, 0, st>>>(p, (const T*)a.x, (const T*)a.dt, (const T*)a.B, (const T*)a.C, (const T*)a.z,
                                                               a.fin, (T*)a.y);
    fbla::note_launches(1);
    return cudaGetLastError();
}


// What one element type brings along (one source file each): the launches for every number of states, packed or not,
// aligned or not.
template <typename T> struct Launcher {
    static cudaError_t fwd(const ScanParams& p, const ScanTensors& a, cudaStream_t st);
    static cudaError_t bwd(const ScanParams& p, const ScanTensors& a, cudaStream_t st);
    static cudaError_t step(const ScanParams& p, const ScanTensors& a, cudaStream_t st);
};


template <int V> struct Num { static constexpr int value = V; };
template <typename F> cudaError_t with_states(int N, F f) {
    switch (ns_of(N)) {
        case 2: return f(Num<2>());
        case 4: return f(Num<4>());
        default: return f(Num<8>());
    }
}
template <typename T> cudaError_t Launcher<T>::fwd(const ScanParams& p, const ScanTensors& a, cudaStream_t st) {
    return with_states(p.states, [&](auto n) {
        constexpr int NS = decltype(n)::value;
        if (p.cu != nullptr) return p.vec ? run_fwd<T, NS, true, true>(p, a, st) : run_fwd<T, NS, true, false>(p, a, st);
        return p.vec ? run_fwd<T, NS, false, true>(p, a, st) : run_fwd<T, NS, false, false>(p, a, st);
    });
}
template <typename T> cudaError_t Launcher<T>::bwd(const ScanParams& p, const ScanTensors& a, cudaStream_t st) {
    return with_states(p.states, [&](auto n) {
        constexpr int NS = decltype(n)::value;
        if (p.cu != nullptr) return p.vec ? run_bwd<T, NS, true, true>(p, a, st) : run_bwd<T, NS, true, false>(p, a, st);
        return p.vec ? run_bwd<T, NS, false, true>(p, a, st) : run_bwd<T, NS, false, false>(p, a, st);
    });
}
template <typename T> cudaError_t Launcher<T>::step(const ScanParams& p, const ScanTensors& a, cudaStream_t st) {
    return with_states(p.states, [&](auto n) { return run_step<T, decltype(n)::value>(p, a, st); });
}

}  // namespace scan
}  // namespace fbla
