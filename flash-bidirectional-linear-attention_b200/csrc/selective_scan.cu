// The C ABI of the selective scan: argument checks, how a problem is cut into segments, and the choice of kernels.
// The kernels are in selective_scan_kernels.cuh, compiled for one element type per source file.
#include <initializer_list>

#include "selective_scan_kernels.cuh"

extern template struct fbla::scan::Launcher<float>;
extern template struct fbla::scan::Launcher<__nv_bfloat16>;
extern template struct fbla::scan::Launcher<__half>;

namespace {

using namespace fbla::scan;

// One CTA walks a whole sequence unless that leaves SMs without work: with fewer CTAs than SMs the tokens are cut
// into segments, as many as fill the places for CTAs (three per SM forward, two backward: registers) in one round, or
// in two or three where that leaves fewer of them empty.  B1-T8192-C4096 forward, 64 CTAs: 3 segments 711 us, 6 (one
// round, 86 %) 562, 7 (a second round of four CTAs) 587, 13 (two rounds, 94 %) 519; B1-T16384-C1024 backward, 16 CTAs:
// 9 segments 962 us, 18 (97 %) 626, 23 823.  Not from 148 CTAs on: the local pass costs more than half of the main
// one (8 rows of 2048 channels, 256 CTAs, forward: 1 segment 701 us, 2 segments 1028).
// A segment is at least four tiles: its local pass and the combination of the segments before it have to stay small.
void cut(ScanParams& p, bool backward) {
    const int tok = tok_of(p.states);
    const int64_t ctas = (int64_t)p.batch * p.groups * tiles_per_group(p), tiles = (p.len + tok - 1) / tok;
    const int64_t places = 148 * (backward ? 2 : 3);
    int64_t segs = 1;
    if (ctas > 0 && ctas < 148) {
        double fullest = 0.0;
        for (int64_t rounds = 1; rounds <= 3 && fullest < 0.93; ++rounds) {
            const int64_t n = places * rounds / ctas;
            const double full = (double)(n * ctas) / (double)(places * rounds);
            if (n >= 1 && full > fullest + 0.02) {
                fullest = full;
                segs = n;
            }
        }
    }
    if (segs > tiles / 4) segs = tiles / 4;
    if (segs < 1) segs = 1;
    const int64_t per = (tiles + segs - 1) / segs;
    p.seg_len = (per > 0 ? per : 1) * tok;
    p.segs = p.len > 0 ? (int)((p.len + p.seg_len - 1) / p.seg_len) : 1;
}

int resolve(const fbla_scan_problem* p, bool backward, ScanParams* r) {
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
    const int64_t size[2] = {p->batch, p->seq_len};
    for (int i = 0; i < 2; ++i) {       // the stride of a dimension of one element is not used, whatever it is
        r->xs[i] = size[i] > 1 ? p->x_stride[i] : 0;
        r->ds[i] = size[i] > 1 ? p->dt_stride[i] : 0;
        r->zs[i] = size[i] > 1 ? p->z_stride[i] : 0;
        r->gs[i] = size[i] > 1 ? p->dy_stride[i] : 0;
    }
    for (int i = 0; i < 3; ++i) {
        r->bs[i] = p->b_stride[i];
        r->cs[i] = p->c_stride[i];
    }
    r->cu = p->cu_seqlens;
    r->A = r->D = r->bias = nullptr;
    r->vec = r->wide_A = 0;
    cut(*r, backward);
    return FBLA_OK;
}

// Packs of a multiple of 8 elements: every row and every CTA's first channel on a boundary.
bool can_vec(const ScanParams& p, int elem, bool z, bool dy, std::initializer_list<const void*> ptrs) {
    const int v = 8;        // 16 bytes of the 16-bit types; an fp32 pack is two accesses
    const int64_t bytes = v * elem > 16 ? 16 : v * elem;
    bool ok = (p.channels / p.groups) % v == 0 && p.xs[0] % v == 0 && p.xs[1] % v == 0 && p.ds[0] % v == 0 && p.ds[1] % v == 0;
    if (z) ok = ok && p.zs[0] % v == 0 && p.zs[1] % v == 0;
    if (dy) ok = ok && p.gs[0] % v == 0 && p.gs[1] % v == 0;
    for (const void* q : ptrs) ok = ok && fbla::seq::aligned_to(q, bytes);
    return ok;
}

// A comes from a parameter and may lie anywhere, unlike the states: packs only where its address allows them.
void set_rates(ScanParams& p, const float* A) {
    p.A = A;
    p.wide_A = p.states == np_of(p.states) && fbla::seq::aligned_to(A, 16);
}

template <typename F> cudaError_t with_type(int dtype, F f) {
    return dtype == FBLA_F32 ? f((float*)nullptr) : dtype == FBLA_BF16 ? f((__nv_bfloat16*)nullptr) : f((__half*)nullptr);
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
    if (resolve(p, false, &r) != FBLA_OK) return -1;
    const int tok = tok_of(r.states);
    return (int64_t)r.batch * ((r.len + tok - 1) / tok) * r.channels * np_of(r.states);
}

int64_t fbla_selective_scan_workspace_bytes(const fbla_scan_problem* p, int backward) {
    ScanParams r;
    if (resolve(p, backward != 0, &r) != FBLA_OK) return -1;
    return (backward ? bwd_layout(r).total : seg_floats(r)) * (int64_t)sizeof(float);
}

int fbla_selective_scan_fwd(const fbla_scan_problem* p, const void* x, const void* dt, const float* A, const void* B, const void* C,
                            const float* D, const void* z, const float* dt_bias, const float* initial_state, void* y, float* final_state,
                            float* checkpoints, void* workspace, size_t workspace_bytes, fbla_stream_t stream) {
    using fbla::api_fail;
    ScanParams r;
    if (int rc = resolve(p, false, &r)) return rc;
    if (A == nullptr) return api_fail(FBLA_ERR_INVALID, "A is NULL");
    if (r.batch > 0 && r.len > 0 && (x == nullptr || dt == nullptr || B == nullptr || C == nullptr || y == nullptr))
        return api_fail(FBLA_ERR_INVALID, "x, dt, B, C or y is NULL");
    if (int rc = check_ws(seg_floats(r) * (int64_t)sizeof(float), workspace, workspace_bytes)) return rc;
    if (int rc = check_states({initial_state, final_state, checkpoints, workspace})) return rc;
    set_rates(r, A);
    r.D = D;
    r.bias = dt_bias;
    r.vec = can_vec(r, p->dtype == FBLA_F32 ? 4 : 2, z != nullptr, false, {x, dt, z, y});
    ScanTensors a = {};
    a.x = x; a.dt = dt; a.B = B; a.C = C; a.z = z; a.init = initial_state; a.y = y; a.fin = final_state; a.ckpt = checkpoints;
    a.ws = (float*)workspace;
    if (int rc = fbla::seq::check_device_status()) return rc;
    return finish(with_type(p->dtype, [&](auto* t) { return Launcher<std::remove_pointer_t<decltype(t)>>::fwd(r, a, (cudaStream_t)stream); }),
                  "selective scan");
}

int fbla_selective_scan_bwd(const fbla_scan_problem* p, const void* x, const void* dt, const float* A, const void* B, const void* C,
                            const float* D, const void* z, const float* dt_bias, const float* initial_state, const float* checkpoints,
                            const void* dy, const float* d_final_state, void* dx, void* ddt, float* dA, void* dB, void* dC, float* dD,
                            void* dz, float* d_dt_bias, float* d_initial_state, void* workspace, size_t workspace_bytes,
                            fbla_stream_t stream) {
    using fbla::api_fail;
    ScanParams r;
    if (int rc = resolve(p, true, &r)) return rc;
    if (A == nullptr || dA == nullptr) return api_fail(FBLA_ERR_INVALID, "A or dA is NULL");
    if (r.batch > 0 && r.len > 0 && (x == nullptr || dt == nullptr || B == nullptr || C == nullptr || dy == nullptr || dx == nullptr ||
                                     ddt == nullptr || dB == nullptr || dC == nullptr || checkpoints == nullptr))
        return api_fail(FBLA_ERR_INVALID, "x, dt, B, C, dy, their gradients or checkpoints is NULL");
    if ((z == nullptr) != (dz == nullptr)) return api_fail(FBLA_ERR_INVALID, "dz goes with z");
    if (int rc = check_ws(bwd_layout(r).total * (int64_t)sizeof(float), workspace, workspace_bytes)) return rc;
    if (int rc = check_states({initial_state, d_final_state, d_initial_state, checkpoints, workspace})) return rc;
    set_rates(r, A);
    r.D = D;
    r.bias = dt_bias;
    r.vec = can_vec(r, p->dtype == FBLA_F32 ? 4 : 2, z != nullptr, true, {x, dt, z, dy, dx, ddt, dz});
    ScanTensors a = {};
    a.x = x; a.dt = dt; a.B = B; a.C = C; a.z = z; a.dy = dy; a.init = initial_state; a.dfin = d_final_state;
    a.dx = dx; a.ddt = ddt; a.dB = dB; a.dC = dC; a.dz = dz; a.ckpt = const_cast<float*>(checkpoints);
    a.dA = dA; a.dD = dD; a.dbias = d_dt_bias; a.dinit = d_initial_state; a.ws = (float*)workspace;
    if (int rc = fbla::seq::check_device_status()) return rc;
    return finish(with_type(p->dtype, [&](auto* t) { return Launcher<std::remove_pointer_t<decltype(t)>>::bwd(r, a, (cudaStream_t)stream); }),
                  "selective scan backward");
}

int fbla_selective_scan_step(const fbla_scan_problem* p, const void* x, const void* dt, const float* A, const void* B, const void* C,
                             const float* D, const void* z, const float* dt_bias, float* state, void* y, fbla_stream_t stream) {
    using fbla::api_fail;
    ScanParams r;
    if (int rc = resolve(p, false, &r)) return rc;
    if (r.cu != nullptr) return api_fail(FBLA_ERR_INVALID, "cu_seqlens given to the single-token step");
    if (r.batch == 0) return FBLA_OK;
    if (x == nullptr || dt == nullptr || A == nullptr || B == nullptr || C == nullptr || state == nullptr || y == nullptr)
        return api_fail(FBLA_ERR_INVALID, "x, dt, A, B, C, state or y is NULL");
    if (int rc = check_states({state})) return rc;
    set_rates(r, A);
    r.D = D;
    r.bias = dt_bias;
    r.segs = 1;
    const int ns = ns_of(r.states), elem = p->dtype == FBLA_F32 ? 4 : 2;
    r.vec = r.states == 4 * ns && fbla::seq::aligned_to(B, ns * elem > 16 ? 16 : ns * elem) &&
            fbla::seq::aligned_to(C, ns * elem > 16 ? 16 : ns * elem);
    for (int i = 0; i < 3; i += 2) r.vec = r.vec && r.bs[i] % ns == 0 && r.cs[i] % ns == 0;
    ScanTensors a = {};
    a.x = x; a.dt = dt; a.B = B; a.C = C; a.z = z; a.fin = state; a.y = y;
    if (int rc = fbla::seq::check_device_status()) return rc;
    return finish(with_type(p->dtype, [&](auto* t) { return Launcher<std::remove_pointer_t<decltype(t)>>::step(r, a, (cudaStream_t)stream); }),
                  "selective scan step");
}

}  // extern "C"
