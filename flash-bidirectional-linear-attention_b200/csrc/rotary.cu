// Rotary positions: pairs of features of q and k turned by an angle that grows with the position.
//
//   (x0, x1) -> factor * (x0 cos a - x1 sin a,  x0 sin a + x1 cos a),   a = position * freq[pair]
//
// The gradient is the same call with -a (the matrix is a multiple of a rotation).  Features behind the
// rotated ones are copied.
//
// What bounds it: HBM, one read and one write of q and k.  The angle of a (token, pair) is the same for
// all heads, so a thread owns a few pairs of one token, forms their sines once and walks over the heads,
// four at a time so that eight loads are in flight.  Angles are reduced in 64 bits (a position of 1e6
// leaves only 2^-4 of a turn in fp32 products).
// Measured on B200, bf16: q and k of B8-H16-L32768-D64, forward and backward 652 us, 6.6 TB/s, the rate of a
// copy; B2-L8192 with 32 + 8 heads of 128, forward 61 us, 5.5 TB/s.
#include <cmath>

#include "seq_common.cuh"

namespace {

using fbla::seq::Pack;
using fbla::seq::seq_of;

struct RotaryParams {
    int batch, hq, hk, dim, pairs, axes, interleaved, num_seqs;
    int heads_per_thread;
    int64_t len;
    int64_t qs[3], ks[3], qos[3], kos[3];   // batch, head, token strides in elements
    const void* positions;
    int positions32;
    int64_t pos_b, pos_t;
    int64_t offset;
    const int32_t* cu;
    const double* freqs;
    float factor, sign;
};

// Sine and cosine of an angle in turns, reduced to half a turn in 64 bits: adding and taking away 1.5 * 2^52 rounds
// to the nearest integer.  fp32 results: to two units in the last place; 16-bit ones: the special function unit's, off by
// at most 2^-20 absolute (documented 2^-21.2 on [-pi, pi], and up to 5 2^-24 from rounding f and its product with 2 pi),
// far below their rounding (forming them otherwise costs more than a dozen heads' products).
template <typename T> __device__ __forceinline__ void sincos_turns(double turns, float& s, float& c) {
    const double whole = __dadd_rn(__dadd_rn(turns, 6755399441055744.0), -6755399441055744.0);
    const float f = (float)(turns - whole);
    if (sizeof(T) == 4) {
        sincospif(2.f * f, &s, &c);
    } else {
        s = __sinf(f * 6.28318531f);
        c = __cosf(f * 6.28318531f);
    }
}

// Slots of one token: PAIRED = two runs of V features whose elements pair up (half layout, and V = 1 for
// interleaved pairs at odd alignments); otherwise one run of V features holding V/2 interleaved pairs.
template <typename T, int V, bool PAIRED>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryParams p, const T* __restrict__ q, const T* __restrict__ k,
                                                     T* __restrict__ qo, T* __restrict__ ko) {
    constexpr int NP = PAIRED ? V : V / 2;          // pairs of a slot
    const int rot_slots = PAIRED ? p.pairs / V : p.dim / V;
    const int slots = PAIRED ? rot_slots + (p.dim - 2 * p.pairs) / V : rot_slots;
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= (int64_t)p.batch * p.len * slots) return;
    const int64_t tok = i / slots;
    const int slot = (int)(i - tok * slots);
    const int64_t b = tok / p.len, t = tok - b * p.len;
    const bool copy = PAIRED && slot >= rot_slots;

    int64_t start = 0;
    bool outside = false;
    if (p.cu != nullptr) {
        const auto s = seq_of(p.cu, p.num_seqs, t);
        outside = s.s < 0;                          // tokens of no sequence come out as zeros
        start = s.lo;
    }
    float cs[NP], sn[NP];
    if (!copy) {
        const int pair0 = PAIRED ? slot * V : slot * NP;
        const int per_axis = p.pairs / p.axes;
        auto position = [&](int axis) {
            if (p.positions == nullptr) return (double)(t - start + p.offset);
            const int64_t at = b * p.pos_b + t * p.pos_t + axis;
            return p.positions32 ? (double)reinterpret_cast<const int32_t*>(p.positions)[at]
                                 : (double)reinterpret_cast<const int64_t*>(p.positions)[at];
        };
        int axis = pair0 / per_axis;
        double pos = pair0 < p.pairs ? position(axis) * 0.15915494309189533577 : 0.0;
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            const int pr = pair0 + j;
            cs[j] = 1.f;
            sn[j] = 0.f;
            if (pr < p.pairs) {
                if (p.axes > 1 && pr >= (axis + 1) * per_axis) pos = position(++axis) * 0.15915494309189533577;
                float s, c;
                sincos_turns<T>(pos * p.freqs[pr], s, c);
                cs[j] = c * p.factor;
                sn[j] = s * p.factor * p.sign;
            }
        }
    }
    int fa, fb;                                     // first feature of the two runs
    if (PAIRED) {
        if (copy) {
            fa = 2 * p.pairs + (slot - rot_slots) * V;
            fb = fa;
        } else {
            fa = p.interleaved ? 2 * slot : slot * V;
            fb = p.interleaved ? fa + 1 : fa + p.pairs;
        }
    } else {
        fa = fb = slot * V;
    }

    const int heads = p.hq + p.hk;
    const int h0 = blockIdx.y * p.heads_per_thread, h1 = min(heads, h0 + p.heads_per_thread);
    constexpr int U = 4;
    for (int h = h0; h < h1; h += U) {
        Pack<T, V> a[U], c[U];
        T *oa[U], *ob[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int hh = h + u;
            if (hh < h1) {
                const bool isq = hh < p.hq;
                const int hl = isq ? hh : hh - p.hq;
                const T* src = isq ? q + b * p.qs[0] + hl * p.qs[1] + t * p.qs[2] : k + b * p.ks[0] + hl * p.ks[1] + t * p.ks[2];
                T* dst = isq ? qo + b * p.qos[0] + hl * p.qos[1] + t * p.qos[2] : ko + b * p.kos[0] + hl * p.kos[1] + t * p.kos[2];
                oa[u] = dst + fa;
                ob[u] = dst + fb;
                a[u].load_stream(src + fa);
                if (PAIRED && !copy) c[u].load_stream(src + fb);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (h + u >= h1) continue;
            if (outside) {
                a[u].zero();
                if (PAIRED) c[u].zero();
            } else if (PAIRED) {
                if (!copy) {
#pragma unroll
                    for (int j = 0; j < NP; ++j) {
                        const float x0 = a[u].get(j), x1 = c[u].get(j);
                        a[u].set(j, x0 * cs[j] - x1 * sn[j]);
                        c[u].set(j, x0 * sn[j] + x1 * cs[j]);
                    }
                }
            } else {
#pragma unroll
                for (int j = 0; j < NP; ++j) {
                    const float x0 = a[u].get(2 * j), x1 = a[u].get(2 * j + 1);
                    if (fa + 2 * j < 2 * p.pairs) {
                        a[u].set(2 * j, x0 * cs[j] - x1 * sn[j]);
                        a[u].set(2 * j + 1, x0 * sn[j] + x1 * cs[j]);
                    }
                }
            }
            a[u].store_stream(oa[u]);
            if (PAIRED && !copy) c[u].store_stream(ob[u]);
        }
    }
}

template <typename T, int V, bool PAIRED>
cudaError_t launch(RotaryParams p, const void* q, const void* k, void* qo, void* ko, cudaStream_t st) {
    const int slots = PAIRED ? p.pairs / V + (p.dim - 2 * p.pairs) / V : p.dim / V;
    const int64_t n = (int64_t)p.batch * p.len * slots;
    const int heads = p.hq + p.hk;
    // Few tokens: spread the heads over threads too (a thread that walks 32 heads in a row waits for memory eight
    // times); otherwise one thread does all heads of its slot, since the way to its sines (position, frequency, 64-bit
    // product) is a fixed latency: 40 heads of 128 at 16384 tokens 61 us, halved 64, in quarters 70.
    int per = heads;
    while (per > 4 && n * ((heads + per - 1) / per) < 148LL * 512) per = (per + 1) / 2;
    p.heads_per_thread = per;
    const int threads = 256;
    const int64_t blocks = (n + threads - 1) / threads;
    if (blocks > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
    const dim3 grid((unsigned)blocks, (unsigned)((heads + per - 1) / per));
    rotary_kernel<T, V, PAIRED><<<grid, threads, 0, st>>>(p, (const T*)q, (const T*)k, (T*)qo, (T*)ko);
    fbla::note_launches(1);
    return cudaGetLastError();
}

// The widest access that the feature counts, the strides and the addresses allow.
template <typename T>
cudaError_t dispatch(const RotaryParams& p, const void* q, const void* k, void* qo, void* ko, cudaStream_t st) {
    auto fits = [&](int v) {
        const int64_t bytes = (int64_t)v * sizeof(T) > 16 ? 16 : (int64_t)v * sizeof(T);
        bool ok = p.dim % v == 0 && (p.interleaved || (p.pairs % v == 0));
        const int64_t size[3] = {p.batch, p.hq, p.len}, size_k[3] = {p.batch, p.hk, p.len};     // a stride of one element is not used
        for (int i = 0; i < 3; ++i) {
            ok = ok && (size[i] == 1 || (p.qs[i] % v == 0 && p.qos[i] % v == 0));
            ok = ok && (p.hk == 0 || size_k[i] == 1 || (p.ks[i] % v == 0 && p.kos[i] % v == 0));
        }
        ok = ok && fbla::seq::aligned_to(q, bytes) && fbla::seq::aligned_to(qo, bytes);
        return ok && (p.hk == 0 || (fbla::seq::aligned_to(k, bytes) && fbla::seq::aligned_to(ko, bytes)));
    };
    constexpr int VMAX = 16 / (int)sizeof(T);
    if (p.interleaved) {
        if (fits(VMAX)) return launch<T, VMAX, false>(p, q, k, qo, ko, st);
        if (fits(2)) return launch<T, 2, false>(p, q, k, qo, ko, st);
        return launch<T, 1, true>(p, q, k, qo, ko, st);
    }
    if (fits(VMAX)) return launch<T, VMAX, true>(p, q, k, qo, ko, st);
    if (VMAX > 4 && fits(4)) return launch<T, 4, true>(p, q, k, qo, ko, st);
    if (fits(2)) return launch<T, 2, true>(p, q, k, qo, ko, st);
    return launch<T, 1, true>(p, q, k, qo, ko, st);
}

}  // namespace

extern "C" int fbla_rotary(const fbla_rotary_problem* p, const void* q, const void* k, void* q_out, void* k_out,
                           fbla_stream_t stream) {
    using fbla::api_fail;
    if (p == nullptr) return api_fail(FBLA_ERR_INVALID, "problem is NULL");
    if (p->dtype != FBLA_F32 && p->dtype != FBLA_BF16 && p->dtype != FBLA_F16)
        return api_fail(FBLA_ERR_INVALID, "dtype %d is not one of FBLA_F32/FBLA_BF16/FBLA_F16", p->dtype);
    if (p->batch < 0 || p->seq_len < 0 || p->heads_q < 1 || p->heads_k < 0 || p->dim < 2)
        return api_fail(FBLA_ERR_INVALID, "batch=%d, seq_len=%lld, heads %d / %d, dim=%d", p->batch, (long long)p->seq_len,
                        p->heads_q, p->heads_k, p->dim);
    if (p->pairs < 1 || 2 * (int64_t)p->pairs > p->dim)
        return api_fail(FBLA_ERR_INVALID, "pairs=%d must be in [1, dim / 2], dim=%d", p->pairs, p->dim);
    if (p->axes < 1 || p->pairs % p->axes != 0)
        return api_fail(FBLA_ERR_INVALID, "axes=%d must divide pairs=%d", p->axes, p->pairs);
    if (p->axes > 1 && p->positions == nullptr)
        return api_fail(FBLA_ERR_INVALID, "positions on %d axes have to be given", p->axes);
    if (p->freqs == nullptr) return api_fail(FBLA_ERR_INVALID, "freqs is NULL");
    if (p->cu_seqlens != nullptr && (p->num_seqs < 1 || p->batch != 1))
        return api_fail(FBLA_ERR_INVALID, "packed sequences: num_seqs=%d must be positive and batch=%d be 1", p->num_seqs, p->batch);
    if (p->batch == 0 || p->seq_len == 0) return FBLA_OK;
    if (q == nullptr || q_out == nullptr) return api_fail(FBLA_ERR_INVALID, "q or q_out is NULL");
    if (p->heads_k > 0 && (k == nullptr || k_out == nullptr)) return api_fail(FBLA_ERR_INVALID, "k or k_out is NULL");
    if (int rc = fbla::seq::check_device_status()) return rc;
    RotaryParams r;
    r.batch = p->batch;
    r.hq = p->heads_q;
    r.hk = p->heads_k;
    r.dim = p->dim;
    r.pairs = p->pairs;
    r.axes = p->axes;
    r.interleaved = p->interleaved != 0;
    r.num_seqs = p->num_seqs;
    r.heads_per_thread = 1;
    r.len = p->seq_len;
    for (int i = 0; i < 3; ++i) {
        r.qs[i] = p->q_stride[i];
        r.ks[i] = p->k_stride[i];
        r.qos[i] = p->q_out_stride[i];
        r.kos[i] = p->k_out_stride[i];
    }
    r.positions = p->positions;
    r.positions32 = p->positions32 != 0;
    r.pos_b = p->pos_stride[0];
    r.pos_t = p->pos_stride[1];
    r.offset = p->offset;
    r.cu = p->cu_seqlens;
    r.freqs = p->freqs;
    r.factor = p->factor;
    r.sign = p->inverse ? -1.f : 1.f;
    const cudaStream_t st = (cudaStream_t)stream;
    cudaError_t e;
    if (p->dtype == FBLA_F32) e = dispatch<float>(r, q, k, q_out, k_out, st);
    else if (p->dtype == FBLA_BF16) e = dispatch<__nv_bfloat16>(r, q, k, q_out, k_out, st);
    else e = dispatch<__half>(r, q, k, q_out, k_out, st);
    return e == cudaSuccess ? FBLA_OK : api_fail(FBLA_ERR_CUDA, "rotary: %s", cudaGetErrorString(e));
}
