// pma_capi.cu -- the extern "C" entry points declared in include/pma.h:
// argument validation on the host, planning (kernel, chunk, segments) and launch.
#include <atomic>
#include <cstring>
#include <mutex>

#include "fp8.cuh"
#include "prefill.cuh"
#include "recurrence.cuh"
#include "sampling.cuh"
#include "tc_common.cuh"

using namespace pma;

namespace {

struct DevInfo {
    int sms = 0;
    int major = 0;
    bool valid = false;
};

thread_local int g_last_cuda_error = 0;

// The caller's fault word (pma_set_fault_word) and the test hook's wait limit
// (pma_test_expire_waits): read by every launch of a kernel with bounded waits.
std::atomic<int *> g_fault_word{nullptr};
std::atomic<unsigned long long> g_test_wait_ns{0};

}  // namespace

// PMA_ERR_CUDA with the cause remembered for pma_last_cuda_error() (also used by prefill_static.cu).
int pma::cuda_fail(cudaError_t e) {
    g_last_cuda_error = (int)e;
    return PMA_ERR_CUDA;
}

namespace {

inline int d_ok(const DevInfo &d) { return d.major == 10 ? PMA_OK : PMA_ERR_DEVICE; }

constexpr int kMaxDevices = 64;
DevInfo g_dev[kMaxDevices];
std::mutex g_dev_mu;

int device_info(DevInfo *out) {
    int dev = 0;
    cudaError_t ce = cudaGetDevice(&dev);
    if (ce != cudaSuccess) return cuda_fail(ce);
    if (dev < 0 || dev >= kMaxDevices) return PMA_ERR_DEVICE;
    std::lock_guard<std::mutex> lk(g_dev_mu);
    if (!g_dev[dev].valid) {
        DevInfo d;
        if ((ce = cudaDeviceGetAttribute(&d.sms, cudaDevAttrMultiProcessorCount, dev)) != cudaSuccess)
            return cuda_fail(ce);
        if ((ce = cudaDeviceGetAttribute(&d.major, cudaDevAttrComputeCapabilityMajor, dev)) != cudaSuccess)
            return cuda_fail(ce);
        d.valid = true;
        g_dev[dev] = d;
    }
    *out = g_dev[dev];
    return d_ok(*out);
}

bool supported_d(int D) { return D == 16 || D == 32 || D == 64 || D == 128; }
bool supported_dtype(int t) { return t == PMA_F32 || t == PMA_BF16; }
size_t esize(int t) { return t == PMA_F32 ? 4 : 2; }

// Each row of D elements must start on a 16-byte boundary (vector loads, TMA).
int check_seq(const pma_seq_tensor *t, bool use_l, bool empty = false) {
    if (!t) return PMA_ERR_ARGUMENT;
    if (!t->data) return empty ? (supported_dtype(t->dtype) ? PMA_OK : PMA_ERR_DTYPE) : PMA_ERR_ARGUMENT;
    if (!supported_dtype(t->dtype)) return PMA_ERR_DTYPE;
    const int64_t step = 16 / (int64_t)esize(t->dtype);
    if (reinterpret_cast<uintptr_t>(t->data) % 16) return PMA_ERR_LAYOUT;
    if (t->stride_b % step || t->stride_h % step || (use_l && t->stride_l % step)) return PMA_ERR_LAYOUT;
    if (t->stride_b < 0 || t->stride_h < 0 || (use_l && t->stride_l < 0)) return PMA_ERR_LAYOUT;
    return PMA_OK;
}

int check_state(const pma_state *s) {
    if (!s || !s->S0 || !s->S1 || !s->S2 || !s->Z0 || !s->Z1 || !s->Z2) return PMA_ERR_ARGUMENT;
    const uintptr_t a[6] = {(uintptr_t)s->S0, (uintptr_t)s->S1, (uintptr_t)s->S2,
                            (uintptr_t)s->Z1, (uintptr_t)s->Z2, 0};
    for (int i = 0; i < 6; ++i)
        if (a[i] % 16) return PMA_ERR_LAYOUT;
    if ((uintptr_t)s->Z0 % 4) return PMA_ERR_LAYOUT;
    return PMA_OK;
}

Seq seq_of(const pma_seq_tensor *t) { return Seq{t->data, t->stride_b, t->stride_h, t->stride_l}; }
SeqOut seqout_of(const pma_seq_tensor *t) {
    return t ? SeqOut{t->data, t->stride_b, t->stride_h, t->stride_l} : SeqOut{nullptr, 0, 0, 0};
}
StateRef user_ref(const pma_state *s) {
    StateRef r{};
    if (s) r.user = *s;
    r.packed = nullptr;
    r.slots = 1;
    return r;
}
StateRef packed_ref(float *ws, int slots) {
    StateRef r{};
    r.packed = ws;
    r.slots = slots;
    return r;
}

struct Plan {
    bool tc = false;
    int chunk = 64;
    int nseg = 1;
    int seg_len = 0;
    size_t ws_bytes = 0;
};

// A [B, L, C] array of the recurrence: elements on their own boundary, strides not negative, the
// dtype of `like`.
int check_blc(const pma_seq_tensor *t, const pma_seq_tensor *like, bool empty) {
    if (!t || !like) return PMA_ERR_ARGUMENT;
    if (!supported_dtype(t->dtype) || t->dtype != like->dtype) return PMA_ERR_DTYPE;
    if (!t->data) return empty ? PMA_OK : PMA_ERR_ARGUMENT;
    if (reinterpret_cast<uintptr_t>(t->data) % esize(t->dtype) || t->stride_b < 0 || t->stride_l < 0)
        return PMA_ERR_LAYOUT;
    return PMA_OK;
}
Blc blc_of(const pma_seq_tensor *t) { return t ? Blc{t->data, t->stride_b, t->stride_l} : Blc{nullptr, 0, 0}; }

// Workspace of the recurrence: [256 B: counter, abort flag][states][runs][partial bias sums].
// A sequence of one tile needs no words.
struct ScanWs {
    int chunks;
    size_t nwords, runs_at, part_at;
    static ScanWs of(int B, int L, int C) {
        ScanWs w;
        w.chunks = scan_chunks(L);
        w.nwords = (size_t)B * w.chunks * C;
        const bool one = w.chunks <= 1;
        w.runs_at = one ? 0 : (256 + 4 * w.nwords + 255) / 256 * 256;
        w.part_at = one ? 0 : (w.runs_at + 8 * w.nwords + 255) / 256 * 256;
        return w;
    }
    size_t bytes(bool backward) const { return part_at + (backward ? 4 * nwords : 0); }
    uint32_t *incl(void *ws) const { return reinterpret_cast<uint32_t *>((char *)ws + 256); }
    float *part(void *ws) const { return reinterpret_cast<float *>((char *)ws + part_at); }
    // Every word unwritten (all ones), the counter and the abort flag at -1.
    cudaError_t arm(ScanParams &p, void *ws, bool needed, cudaStream_t st) const {
        if (chunks <= 1) return cudaSuccess;
        p.counter = reinterpret_cast<int *>(ws);
        p.incl = incl(ws);
        p.agg = reinterpret_cast<unsigned long long *>((char *)ws + runs_at);
        return needed ? cudaMemsetAsync(ws, 0xff, part_at, st) : cudaSuccess;
    }
};

ScanParams scan_params(int B, int L, int C, const pma_seq_tensor *x, const pma_seq_tensor *f,
                       const pma_seq_tensor *gate, const float *bias, const float *h0, const uint8_t *reset) {
    ScanParams p{};
    p.B = B;
    p.L = L;
    p.C = C;
    p.chunks = scan_chunks(L);
    p.x = blc_of(x);
    p.f = blc_of(f);
    p.gate = blc_of(gate);
    p.bias = bias;
    p.h0 = h0;
    p.reset = reset;
    p.fault = g_fault_word.load(std::memory_order_acquire);
    p.wait_ns = 2000000000ull;  // as the tensor-core kernels: 2 s per wait
    p.test_wait_ns = g_test_wait_ns.load(std::memory_order_acquire);
    return p;
}

// Rows of e4m3 bytes for a tensor map: 16-byte base and stride.
int check_e4m3(const void *q, int64_t stride, int K) {
    if (!q) return PMA_ERR_ARGUMENT;
    if (stride < K || (uintptr_t)q % 16 || stride % 16) return PMA_ERR_LAYOUT;
    return PMA_OK;
}
// The [M, K] or [N, K] input of a quantisation.
int check_dense(const void *x, int64_t stride, int dtype, int rows, int K) {
    if (!supported_dtype(dtype)) return PMA_ERR_DTYPE;
    if (!x || (rows > 1 && stride < K)) return PMA_ERR_ARGUMENT;
    return (uintptr_t)x % esize(dtype) ? PMA_ERR_LAYOUT : PMA_OK;
}

// Workspace of pma_fp8_linear: e4m3 rows of round16(K) bytes, then the scales [ceil(K/128), M].
struct Fp8Ws {
    int64_t stride;
    size_t scale_at, bytes;
    static Fp8Ws of(int M, int K) {
        Fp8Ws w;
        w.stride = ((int64_t)K + 15) / 16 * 16;
        w.scale_at = ((size_t)M * w.stride + 255) / 256 * 256;
        w.bytes = w.scale_at + (size_t)M * ((K + FP8_BLOCK - 1) / FP8_BLOCK) * 4;
        return w;
    }
};

int fp8_product(int M, int N, int K, const Fp8Rows &x, const Fp8Rows &w, void *y, int64_t ys, int ydt, int sms,
                bool after_quantize, cudaStream_t st) {
    Fp8Params p{};
    p.M = M;
    p.N = N;
    p.K = K;
    p.x = x;
    p.w = w;
    p.y = y;
    p.ys = ys;
    p.y_f32 = ydt == PMA_F32;
    p.fault = g_fault_word.load(std::memory_order_acquire);
    p.test_wait_ns = g_test_wait_ns.load(std::memory_order_acquire);
    const cudaError_t e = launch_fp8_matmul(p, sms, after_quantize, st);
    return e == cudaSuccess ? PMA_OK : cuda_fail(e);
}

bool bf16_exact(float f) {
    uint32_t u;
    memcpy(&u, &f, 4);
    return (u & 0xffffu) == 0;
}

// D = 128 runs on tensor cores when the kernel needs no LayerNorm pass (`pro` null: no prologue).
bool tc128_plan(int D, int dtype, const Prologue *pro) {
    if (D != 128 || !tc128_supported(dtype)) return false;
    return !pro || (!pro->qw && !pro->kw && (pro->q_scale == 1.0f || bf16_exact(pro->q_scale)));
}

Plan make_plan(int B, int H, int L, int D, int dtype, int sms, const Prologue *pro) {
    Plan p;
    p.tc = tc_supported(D, dtype) || tc128_plan(D, dtype, pro);
    p.chunk = p.tc ? TC_CHUNK : simt_chunk(D);
    const long BH = (long)B * H;
    const int nchunks = (L + p.chunk - 1) / p.chunk;
    // CTAs resident per SM: SIMT D<=64 fits two; D=128 and the tensor-core kernel one.
    const long slots = (long)sms * ((!p.tc && D <= 64) ? 2 : 1);
    // Split sequences into segments only when B*H leaves SMs idle, and only into as
    // many as fit one wave (a partial second wave costs more than the idle SMs).
    int nseg = 1;
    if (BH > 0 && BH * 2 <= slots) nseg = (int)(slots / BH);
    if (nseg > nchunks) nseg = nchunks;
    if (nseg < 1) nseg = 1;
    const int seg_chunks = (nchunks + nseg - 1) / nseg;
    p.nseg = seg_chunks > 0 ? (nchunks + seg_chunks - 1) / seg_chunks : 1;
    p.seg_len = seg_chunks * p.chunk;
    p.ws_bytes = p.tc ? WS_HEADER : 0;
    if (p.nseg > 1) p.ws_bytes = WS_HEADER + (size_t)BH * p.nseg * slot_floats(D) * sizeof(float);
    return p;
}

// pma_prologue -> kernel view; NULL is the identity (no GQA, no norm, scale 1).
int prologue_of(const pma_prologue *pp, int H, Prologue *out) {
    Prologue r{1, 1.0f, nullptr, nullptr, nullptr, nullptr, 1e-5f};
    if (pp) {
        if (pp->kv_groups < 1 || H % pp->kv_groups) return PMA_ERR_ARGUMENT;
        if (!(pp->norm_eps >= 0.0f) || pp->q_scale != pp->q_scale) return PMA_ERR_ARGUMENT;
        const float *ptrs[4] = {pp->q_norm_weight, pp->q_norm_bias, pp->k_norm_weight, pp->k_norm_bias};
        for (const float *f : ptrs)
            if (reinterpret_cast<uintptr_t>(f) % 4) return PMA_ERR_LAYOUT;
        r.groups = pp->kv_groups;
        r.q_scale = pp->q_scale;
        r.qw = pp->q_norm_weight;
        r.qb = pp->q_norm_weight ? pp->q_norm_bias : nullptr;
        r.kw = pp->k_norm_weight;
        r.kb = pp->k_norm_weight ? pp->k_norm_bias : nullptr;
        r.ln_eps = pp->norm_eps;
    }
    *out = r;
    return PMA_OK;
}

int prefill_impl(int B, int H, int L, int D, const pma_seq_tensor *q, const pma_seq_tensor *k,
                 const pma_seq_tensor *v, const pma_prologue *prologue, const float *lambda,
                 int64_t lambda_stride_b, const pma_state *state_in, const pma_state *state_out, float eps,
                 const pma_seq_tensor *y, void *workspace, size_t workspace_bytes, pma_stream_t stream,
                 bool resume = false);
int decode_impl(int N, int H, int D, const pma_seq_tensor *q, const pma_seq_tensor *k, const pma_seq_tensor *v,
                const pma_prologue *prologue, const float *lambda, int64_t lambda_stride_n, const int32_t *rows,
                int pool_rows, const pma_state *state_in, const pma_state *state_out, float eps,
                const pma_seq_tensor *y, pma_stream_t stream, const float *k_head_scale = nullptr,
                bool selective = false);

// Tensor-core path: which inputs the QK-norm pass rewrites, and the workspace beyond the plan's.
struct ProPass {
    bool q = false, k = false;
    size_t q_off = 0, k_off = 0, total = 0;  // byte offsets of the copies in the workspace; total bytes
};

ProPass pro_pass(const Plan &pl, const Prologue &pro, int B, int H, int L, bool want_y) {
    ProPass r;
    r.total = pl.ws_bytes;
    if (!pl.tc) return r;  // the CUDA-core kernel folds the prologue into its loads
    r.q = want_y && (pro.qw != nullptr || (pro.q_scale != 1.0f && !bf16_exact(pro.q_scale)));
    r.k = pro.kw != nullptr;
    size_t off = (pl.ws_bytes + 255) / 256 * 256;
    if (r.q) {
        r.q_off = off;
        off += (size_t)B * H * L * 64 * 2;
    }
    if (r.k) {
        off = (off + 255) / 256 * 256;
        r.k_off = off;
        off += (size_t)B * (H / pro.groups) * L * 64 * 2;
    }
    if (r.q || r.k) r.total = off;
    return r;
}

// Tensor-core path: the QK-norm pass for q and / or k (pro_pass says which) into the workspace;
// the core then reads the normalised rows and keeps the GQA map and a bf16-exact q scale.
cudaError_t run_prologue_passes(const ProPass &pp, const Prologue &pro, PrefillParams &p, int B, int H, int L,
                                void *workspace, bool want_y, int sms, cudaStream_t st) {
    char *wsb = reinterpret_cast<char *>(workspace);
    const int hkv = H / pro.groups;
    cudaError_t e;
    if (pp.q) {
        if ((e = launch_qk_norm(p.q, B, H, L, pro.qw, pro.qb, pro.ln_eps, pro.q_scale, wsb + pp.q_off, sms, st)) !=
            cudaSuccess)
            return e;
        p.q = Seq{wsb + pp.q_off, (int64_t)H * L * 64, (int64_t)L * 64, 64};
        p.pro.q_scale = 1.0f;
    }
    if (pp.k) {
        if ((e = launch_qk_norm(p.k, B, hkv, L, pro.kw, pro.kb, pro.ln_eps, 1.0f, wsb + pp.k_off, sms, st)) !=
            cudaSuccess)
            return e;
        p.k = Seq{wsb + pp.k_off, (int64_t)hkv * L * 64, (int64_t)L * 64, 64};
    }
    p.pro.qw = p.pro.qb = p.pro.kw = p.pro.kb = nullptr;
    if (!want_y) p.pro.q_scale = 1.0f;
    return cudaSuccess;
}

// The selective prefill's plan: one segment per head-state (its per-token decay has no per-head
// carry factor for the segment prefix); tensor cores for bf16 at D = 64.
Plan selective_plan(int L, int D, int dtype) {
    Plan p;
    p.tc = tc_supported(D, dtype);
    p.chunk = p.tc ? TC_CHUNK : simt_chunk(D);
    p.nseg = 1;
    p.seg_len = ((L + p.chunk - 1) / p.chunk) * p.chunk;
    p.ws_bytes = p.tc ? WS_HEADER : 0;
    return p;
}

cudaError_t launch_prefill(const Plan &pl, const PrefillParams &p, int D, int idt, int ydt, dim3 grid,
                           cudaStream_t st) {
    if (!pl.tc) return launch_prefill_simt(p, D, idt, ydt, grid, st);
    return D == 128 ? launch_prefill_tc128(p, ydt, grid, st) : launch_prefill_tc(p, ydt, grid, st);
}

}  // namespace

extern "C" {

int pma_version(void) { return PMA_ABI_VERSION; }

const char *pma_status_string(int status) {
    switch (status) {
        case PMA_OK: return "ok";
        case PMA_ERR_ARGUMENT: return "invalid argument (null pointer or negative size)";
        case PMA_ERR_HEAD_DIM: return "unsupported head_dim (supported: 16, 32, 64, 128)";
        case PMA_ERR_DTYPE: return "unsupported dtype (float32 or bfloat16)";
        case PMA_ERR_LAYOUT: return "unsupported layout (rows must start on 16-byte boundaries, head dim contiguous)";
        case PMA_ERR_WORKSPACE: return "workspace missing or too small";
        case PMA_ERR_CUDA: return "CUDA runtime error";
        case PMA_ERR_DEVICE: return "current device is not sm_100 (B200 class)";
        default: return "unknown status";
    }
}

int pma_last_cuda_error(void) { return g_last_cuda_error; }

void pma_set_fault_word(int *word) { g_fault_word.store(word); }

void pma_test_expire_waits(unsigned long long limit_ns) { g_test_wait_ns.store(limit_ns); }

const char *pma_cuda_error_string(int cuda_error) { return cudaGetErrorString((cudaError_t)cuda_error); }

size_t pma_state_floats(int D) { return D > 0 ? state_floats(D) : 0; }

int pma_supported_head_dims(int dtype, int *dims, int cap) {
    static const int all[4] = {16, 32, 64, 128};
    if (!supported_dtype(dtype)) return 0;
    for (int i = 0; i < 4 && i < cap; ++i)
        if (dims) dims[i] = all[i];
    return 4;
}

size_t pma_prefill_workspace_bytes(int B, int H, int L, int D, int dtype) {
    if (B <= 0 || H <= 0 || L <= 0 || !supported_d(D) || !supported_dtype(dtype)) return 0;
    DevInfo di;
    if (device_info(&di) != PMA_OK) return 0;
    return make_plan(B, H, L, D, dtype, di.sms, nullptr).ws_bytes;
}

size_t pma_prefill_ex_workspace_bytes(int B, int H, int L, int D, int dtype, const pma_prologue *prologue) {
    if (B <= 0 || H <= 0 || L <= 0 || !supported_d(D) || !supported_dtype(dtype)) return 0;
    Prologue pro;
    if (prologue_of(prologue, H, &pro) != PMA_OK) return 0;
    DevInfo di;
    if (device_info(&di) != PMA_OK) return 0;
    return pro_pass(make_plan(B, H, L, D, dtype, di.sms, &pro), pro, B, H, L, true).total;
}

int pma_prefill(int B, int H, int L, int D, const pma_seq_tensor *q, const pma_seq_tensor *k,
                const pma_seq_tensor *v, const float *lambda, int64_t lambda_stride_b, const pma_state *state_in,
                const pma_state *state_out, float eps, const pma_seq_tensor *y, void *workspace,
                size_t workspace_bytes, pma_stream_t stream) {
    return prefill_impl(B, H, L, D, q, k, v, nullptr, lambda, lambda_stride_b, state_in, state_out, eps, y,
                        workspace, workspace_bytes, stream);
}

int pma_prefill_ex(int B, int H, int L, int D, const pma_seq_tensor *q, const pma_seq_tensor *k,
                   const pma_seq_tensor *v, const pma_prologue *prologue, const float *lambda,
                   int64_t lambda_stride_b, const pma_state *state_in, const pma_state *state_out, float eps,
                   const pma_seq_tensor *y, void *workspace, size_t workspace_bytes, pma_stream_t stream) {
    return prefill_impl(B, H, L, D, q, k, v, prologue, lambda, lambda_stride_b, state_in, state_out, eps, y,
                        workspace, workspace_bytes, stream);
}

int pma_prefill_resume(int B, int H, int L, int D, const pma_seq_tensor *q, const pma_seq_tensor *k,
                       const pma_seq_tensor *v, const float *lambda, int64_t lambda_stride_b,
                       const pma_state *state_in, const pma_state *state_out, float eps, const pma_seq_tensor *y,
                       void *workspace, size_t workspace_bytes, pma_stream_t stream) {
    if (!y) return PMA_ERR_ARGUMENT;  // the output pass is what this entry runs
    return prefill_impl(B, H, L, D, q, k, v, nullptr, lambda, lambda_stride_b, state_in, state_out, eps, y,
                        workspace, workspace_bytes, stream, true);
}

int pma_decode_step(int N, int H, int D, const pma_seq_tensor *q, const pma_seq_tensor *k, const pma_seq_tensor *v,
                    const float *lambda, int64_t lambda_stride_n, const pma_state *state_in,
                    const pma_state *state_out, float eps, const pma_seq_tensor *y, pma_stream_t stream) {
    return decode_impl(N, H, D, q, k, v, nullptr, lambda, lambda_stride_n, nullptr, 0, state_in, state_out, eps, y,
                       stream);
}

int pma_decode_step_rows(int N, int H, int D, const pma_seq_tensor *q, const pma_seq_tensor *k,
                         const pma_seq_tensor *v, const float *lambda, int64_t lambda_stride_n, const int32_t *rows,
                         int pool_rows, const pma_state *pool_in, const pma_state *pool_out, float eps,
                         const pma_seq_tensor *y, pma_stream_t stream) {
    if (N > 0 && !rows) return PMA_ERR_ARGUMENT;
    return decode_impl(N, H, D, q, k, v, nullptr, lambda, lambda_stride_n, rows, pool_rows, pool_in, pool_out, eps,
                       y, stream);
}

int pma_decode_step_ex(int N, int H, int D, const pma_seq_tensor *q, const pma_seq_tensor *k,
                       const pma_seq_tensor *v, const pma_prologue *prologue, const float *lambda,
                       int64_t lambda_stride_n, const int32_t *rows, int pool_rows, const pma_state *state_in,
                       const pma_state *state_out, float eps, const pma_seq_tensor *y, pma_stream_t stream) {
    return decode_impl(N, H, D, q, k, v, prologue, lambda, lambda_stride_n, rows, pool_rows, state_in, state_out,
                       eps, y, stream);
}

}  // extern "C"

namespace {

int prefill_impl(int B, int H, int L, int D, const pma_seq_tensor *q, const pma_seq_tensor *k,
                 const pma_seq_tensor *v, const pma_prologue *prologue, const float *lambda,
                 int64_t lambda_stride_b, const pma_state *state_in, const pma_state *state_out, float eps,
                 const pma_seq_tensor *y, void *workspace, size_t workspace_bytes, pma_stream_t stream,
                 bool resume) {
    if (B < 0 || H <= 0 || L < 0 || !lambda || lambda_stride_b < 0) return PMA_ERR_ARGUMENT;
    if (!supported_d(D)) return PMA_ERR_HEAD_DIM;
    int rc;
    Prologue pro;
    if ((rc = prologue_of(prologue, H, &pro))) return rc;
    const bool empty = (L == 0 || B == 0);  // no element is touched: null data is fine
    if ((rc = check_seq(q, true, empty)) || (rc = check_seq(k, true, empty)) || (rc = check_seq(v, true, empty)))
        return rc;
    if (q->dtype != k->dtype || q->dtype != v->dtype) return PMA_ERR_DTYPE;
    if (y && (rc = check_seq(y, true, empty))) return rc;
    if (state_in && (rc = check_state(state_in))) return rc;
    if (state_out && (rc = check_state(state_out))) return rc;
    DevInfo di;
    if ((rc = device_info(&di))) return rc;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const int BH = B * H;
    if (BH == 0) return PMA_OK;

    if (L == 0) {  // nothing consumed: final state = incoming state
        if (!state_out) return PMA_OK;
        const size_t DD = (size_t)D * D;
        float *dst[6] = {state_out->S0, state_out->S1, state_out->S2, state_out->Z0, state_out->Z1, state_out->Z2};
        const float *src[6] = {state_in ? state_in->S0 : nullptr, state_in ? state_in->S1 : nullptr,
                               state_in ? state_in->S2 : nullptr, state_in ? state_in->Z0 : nullptr,
                               state_in ? state_in->Z1 : nullptr, state_in ? state_in->Z2 : nullptr};
        const size_t n[6] = {BH * (size_t)D, BH * DD, BH * DD, (size_t)BH, BH * (size_t)D, BH * (size_t)D};
        for (int i = 0; i < 6; ++i) {
            cudaError_t e = src[i] ? (src[i] == dst[i] ? cudaSuccess
                                                        : cudaMemcpyAsync(dst[i], src[i], n[i] * 4,
                                                                          cudaMemcpyDeviceToDevice, st))
                                   : cudaMemsetAsync(dst[i], 0, n[i] * 4, st);
            if (e != cudaSuccess) return cuda_fail(e);
        }
        return PMA_OK;
    }

    const Plan pl = make_plan(B, H, L, D, q->dtype, di.sms, &pro);
    const ProPass pp = pro_pass(pl, pro, B, H, L, y != nullptr);
    if (pp.total && (!workspace || workspace_bytes < pp.total)) return PMA_ERR_WORKSPACE;
    if (pp.total && reinterpret_cast<uintptr_t>(workspace) % 16) return PMA_ERR_WORKSPACE;
    if (!y && !state_out) return PMA_OK;  // nothing requested
    const int ydt = y ? y->dtype : PMA_F32;

    PrefillParams p{};
    p.B = B;
    p.H = H;
    p.L = L;
    p.seg_len = pl.seg_len;
    p.q = seq_of(q);
    p.k = seq_of(k);
    p.v = seq_of(v);
    p.pro = pro;
    cudaError_t e;
    if (pl.tc && (e = run_prologue_passes(pp, pro, p, B, H, L, workspace, y != nullptr, di.sms, st)) != cudaSuccess)
        return cuda_fail(e);
    p.y = seqout_of(y);
    p.lambda = lambda;
    p.lam_sb = lambda_stride_b;
    p.eps = eps;
    p.status = nullptr;
    p.fault = g_fault_word.load();
    p.test_wait_ns = g_test_wait_ns.load();

    if (pl.ws_bytes) {  // clear the status word the tensor-core kernel reports timeouts in
        p.status = reinterpret_cast<int *>(workspace);
        if ((e = cudaMemsetAsync(p.status, 0, sizeof(int), st)) != cudaSuccess) return cuda_fail(e);
    }
    if (pl.nseg == 1) {
        p.in = user_ref(state_in);
        p.out = user_ref(state_out);
        p.state_only = 0;
        e = launch_prefill(pl, p, D, q->dtype, ydt, dim3(BH, 1), st);
        return e == cudaSuccess ? PMA_OK : cuda_fail(e);
    }

    float *ws = reinterpret_cast<float *>(reinterpret_cast<char *>(workspace) + WS_HEADER);
    if (resume) {
        // the workspace holds the state entering every segment from a zero start (left there by a
        // state-only call with the same plan): shift them to state_in, then the full pass
        if (state_in && (e = launch_segment_resume(BH, H, D, pl.nseg, pl.seg_len, ws, user_ref(state_in), lambda,
                                                   lambda_stride_b, st)) != cudaSuccess)
            return cuda_fail(e);
        p.in = packed_ref(ws, pl.nseg);
        p.out = user_ref(state_out);
        p.state_only = 0;
        e = launch_prefill(pl, p, D, q->dtype, ydt, dim3(BH, pl.nseg), st);
        return e == cudaSuccess ? PMA_OK : cuda_fail(e);
    }
    // 1. each segment's own state from zero (the last one only when no y is wanted)
    PrefillParams ps = p;
    ps.y = SeqOut{nullptr, 0, 0, 0};
    ps.in = user_ref(nullptr);
    ps.out = packed_ref(ws, pl.nseg);
    ps.state_only = 1;
    const int nstate = y ? pl.nseg - 1 : pl.nseg;
    e = launch_prefill(pl, ps, D, q->dtype, ydt, dim3(BH, nstate), st);
    if (e != cudaSuccess) return cuda_fail(e);
    // 2. in-place prefix: state entering every segment (and the final state if no y)
    e = launch_segment_prefix(BH, H, D, pl.nseg, pl.seg_len, L, ws, user_ref(state_in),
                              y ? user_ref(nullptr) : user_ref(state_out), lambda, lambda_stride_b, st);
    if (e != cudaSuccess) return cuda_fail(e);
    if (!y) return PMA_OK;
    // 3. full pass, every segment starting from its carried state
    p.in = packed_ref(ws, pl.nseg);
    p.out = user_ref(state_out);
    p.state_only = 0;
    e = launch_prefill(pl, p, D, q->dtype, ydt, dim3(BH, pl.nseg), st);
    return e == cudaSuccess ? PMA_OK : cuda_fail(e);
}

int decode_impl(int N, int H, int D, const pma_seq_tensor *q, const pma_seq_tensor *k, const pma_seq_tensor *v,
                const pma_prologue *prologue, const float *lambda, int64_t lambda_stride_n, const int32_t *rows,
                int pool_rows, const pma_state *state_in, const pma_state *state_out, float eps,
                const pma_seq_tensor *y, pma_stream_t stream, const float *k_head_scale, bool selective) {
    if (N < 0 || H <= 0 || !lambda || lambda_stride_n < 0 || pool_rows < 0) return PMA_ERR_ARGUMENT;
    if (!supported_d(D)) return PMA_ERR_HEAD_DIM;
    int rc;
    Prologue pro;
    if ((rc = prologue_of(prologue, H, &pro))) return rc;
    const bool empty = N == 0;
    if ((rc = check_seq(q, false, empty)) || (rc = check_seq(k, false, empty)) || (rc = check_seq(v, false, empty)) ||
        (rc = check_seq(y, false, empty)))
        return rc;
    if (q->dtype != k->dtype || q->dtype != v->dtype) return PMA_ERR_DTYPE;
    if ((rc = check_state(state_in)) || (rc = check_state(state_out))) return rc;
    DevInfo di;
    if ((rc = device_info(&di))) return rc;
    if (N == 0) return PMA_OK;
    if ((long)N * H > (1L << 30) || (long)pool_rows * H > (1L << 30)) return PMA_ERR_ARGUMENT;
    DecodeParams p{};
    p.N = N;
    p.H = H;
    p.q = seq_of(q);
    p.k = seq_of(k);
    p.v = seq_of(v);
    p.pro = pro;
    p.y = seqout_of(y);
    p.lambda = lambda;
    p.lam_sn = lambda_stride_n;
    p.in = *state_in;
    p.out = *state_out;
    p.eps = eps;
    p.rows = rows;
    p.pool_rows = rows ? pool_rows : 0;
    p.k_head_scale = k_head_scale;
    p.log_lambda = selective ? 1 : 0;
    p.half_sq = selective ? 1 : 0;
    cudaError_t e = launch_decode(p, D, q->dtype, y->dtype, reinterpret_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? PMA_OK : cuda_fail(e);
}

}  // namespace

extern "C" {

int pma_delta_prefill(int B, int H, int L, int D, const pma_seq_tensor *q, const pma_seq_tensor *k,
                      const pma_seq_tensor *v, const float *beta, const float *alpha, const float *lambda,
                      int64_t lambda_stride_b, int chunk, float lyapunov_bound, float norm_eps,
                      const float *state_in, float *state_out, const pma_seq_tensor *y, void *workspace,
                      size_t workspace_bytes, pma_stream_t stream) {
    if (B < 0 || H <= 0 || L < 0 || !lambda || lambda_stride_b < 0 || !(norm_eps > 0.0f)) return PMA_ERR_ARGUMENT;
    if (D != 16 && D != 32 && D != 64) return PMA_ERR_HEAD_DIM;
    if (chunk != 32 && chunk != 64) return PMA_ERR_ARGUMENT;
    if (!y && !state_out) return PMA_ERR_ARGUMENT;
    int rc;
    const bool empty = (L == 0 || B == 0);
    if ((rc = check_seq(q, true, empty)) || (rc = check_seq(k, true, empty)) || (rc = check_seq(v, true, empty)))
        return rc;
    if (q->dtype != k->dtype || q->dtype != v->dtype) return PMA_ERR_DTYPE;
    if (y && (rc = check_seq(y, true, empty))) return rc;
    if (!empty && !beta) return PMA_ERR_ARGUMENT;
    if ((uintptr_t)state_in % 16 || (uintptr_t)state_out % 16) return PMA_ERR_LAYOUT;
    DevInfo di;
    if ((rc = device_info(&di))) return rc;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const size_t sbytes = (size_t)B * H * D * 2 * D * sizeof(float);
    if (B == 0) return PMA_OK;
    if (L == 0) {
        if (!state_out) return PMA_OK;
        cudaError_t e = state_in ? (state_in == state_out ? cudaSuccess
                                                          : cudaMemcpyAsync(state_out, state_in, sbytes,
                                                                            cudaMemcpyDeviceToDevice, st))
                                 : cudaMemsetAsync(state_out, 0, sbytes, st);
        return e == cudaSuccess ? PMA_OK : cuda_fail(e);
    }
    DeltaParams p{};
    p.B = B;
    p.H = H;
    p.L = L;
    p.q = seq_of(q);
    p.k = seq_of(k);
    p.v = seq_of(v);
    p.y = seqout_of(y);
    p.beta = beta;
    p.alpha = alpha;
    p.lambda = lambda;
    p.lam_sb = lambda_stride_b;
    p.bound = lyapunov_bound;
    p.norm_eps = norm_eps;
    p.state_in = state_in;
    p.state_out = state_out;
    p.fault = g_fault_word.load();
    p.test_wait_ns = g_test_wait_ns.load();
    const int ydt = y ? y->dtype : PMA_F32;
    cudaError_t e;
    if (delta_tc_supported(D, chunk, q->dtype)) {
        if (workspace && workspace_bytes) {
            const int window = delta_wy_window(B, H, L, workspace_bytes);
            if (window == 0) return PMA_ERR_WORKSPACE;
            if ((uintptr_t)workspace % 256) return PMA_ERR_LAYOUT;
            e = launch_delta_prefill_wy(p, ydt, workspace, window, st);
        } else {
            e = launch_delta_prefill_tc(p, ydt, st);
        }
    } else {
        e = launch_delta_prefill(p, D, chunk, q->dtype, ydt, st);
    }
    return e == cudaSuccess ? PMA_OK : cuda_fail(e);
}

size_t pma_delta_prefill_workspace_bytes(int B, int H, int L, int D, int chunk, int dtype) {
    if (!delta_tc_supported(D, chunk, dtype)) return 0;
    return delta_wy_workspace_bytes(B, H, L);
}

int pma_delta_decode_step(int N, int H, int D, const pma_seq_tensor *q, const pma_seq_tensor *k,
                          const pma_seq_tensor *v, const float *beta, const float *alpha, float lyapunov_bound,
                          float norm_eps, const float *state_in, float *state_out, const pma_seq_tensor *y,
                          pma_stream_t stream) {
    if (N < 0 || H <= 0 || !(norm_eps > 0.0f)) return PMA_ERR_ARGUMENT;
    if (D != 16 && D != 32 && D != 64) return PMA_ERR_HEAD_DIM;
    int rc;
    const bool empty = N == 0;
    if ((rc = check_seq(q, false, empty)) || (rc = check_seq(k, false, empty)) || (rc = check_seq(v, false, empty)) ||
        (rc = check_seq(y, false, empty)))
        return rc;
    if (q->dtype != k->dtype || q->dtype != v->dtype) return PMA_ERR_DTYPE;
    if (!empty && (!beta || !alpha || !state_in || !state_out)) return PMA_ERR_ARGUMENT;
    if ((uintptr_t)state_in % 16 || (uintptr_t)state_out % 16) return PMA_ERR_LAYOUT;
    DevInfo di;
    if ((rc = device_info(&di))) return rc;
    if (N == 0) return PMA_OK;
    if ((long)N * H > (1L << 30)) return PMA_ERR_ARGUMENT;
    DeltaStepParams p{};
    p.N = N;
    p.H = H;
    p.q = seq_of(q);
    p.k = seq_of(k);
    p.v = seq_of(v);
    p.y = seqout_of(y);
    p.beta = beta;
    p.alpha = alpha;
    p.bound = lyapunov_bound;
    p.norm_eps = norm_eps;
    p.state_in = state_in;
    p.state_out = state_out;
    cudaError_t e = launch_delta_step(p, D, q->dtype, y->dtype, reinterpret_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? PMA_OK : cuda_fail(e);
}

size_t pma_selective_prefill_workspace_bytes(int B, int H, int L, int D, int dtype, const pma_prologue *prologue) {
    if (B <= 0 || H <= 0 || L <= 0 || !supported_d(D) || !supported_dtype(dtype)) return 0;
    Prologue pro;
    if (prologue_of(prologue, H, &pro) != PMA_OK) return 0;
    return pro_pass(selective_plan(L, D, dtype), pro, B, H, L, true).total;
}

int pma_selective_prefill(int B, int H, int L, int D, const pma_seq_tensor *q, const pma_seq_tensor *k,
                          const pma_seq_tensor *v, const pma_prologue *prologue, const float *log_decay,
                          const float *beta, const pma_state *state_in, const pma_state *state_out, float eps,
                          const pma_seq_tensor *y, void *workspace, size_t workspace_bytes, pma_stream_t stream) {
    if (B < 0 || H <= 0 || L < 0 || !beta || (L > 0 && B > 0 && !log_decay)) return PMA_ERR_ARGUMENT;
    if (!supported_d(D)) return PMA_ERR_HEAD_DIM;
    int rc;
    Prologue pro;
    if ((rc = prologue_of(prologue, H, &pro))) return rc;
    const bool empty = (L == 0 || B == 0);
    if ((rc = check_seq(q, true, empty)) || (rc = check_seq(k, true, empty)) || (rc = check_seq(v, true, empty)))
        return rc;
    if (q->dtype != k->dtype || q->dtype != v->dtype) return PMA_ERR_DTYPE;
    if (y && (rc = check_seq(y, true, empty))) return rc;
    if (state_in && (rc = check_state(state_in))) return rc;
    if (state_out && (rc = check_state(state_out))) return rc;
    if (!y && !state_out) return PMA_OK;
    DevInfo di;
    if ((rc = device_info(&di))) return rc;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const int BH = B * H;
    if (BH == 0) return PMA_OK;
    if (L == 0) {  // the state passes through unchanged (same layout in and out)
        if (!state_out) return PMA_OK;
        const size_t DD = (size_t)D * D;
        float *dst[6] = {state_out->S0, state_out->S1, state_out->S2, state_out->Z0, state_out->Z1, state_out->Z2};
        const float *src[6] = {state_in ? state_in->S0 : nullptr, state_in ? state_in->S1 : nullptr,
                               state_in ? state_in->S2 : nullptr, state_in ? state_in->Z0 : nullptr,
                               state_in ? state_in->Z1 : nullptr, state_in ? state_in->Z2 : nullptr};
        const size_t n[6] = {BH * (size_t)D, BH * DD, BH * DD, (size_t)BH, BH * (size_t)D, BH * (size_t)D};
        for (int i = 0; i < 6; ++i) {
            cudaError_t e = src[i] ? (src[i] == dst[i] ? cudaSuccess
                                                        : cudaMemcpyAsync(dst[i], src[i], n[i] * 4,
                                                                          cudaMemcpyDeviceToDevice, st))
                                   : cudaMemsetAsync(dst[i], 0, n[i] * 4, st);
            if (e != cudaSuccess) return cuda_fail(e);
        }
        return PMA_OK;
    }
    const Plan pl = selective_plan(L, D, q->dtype);
    const ProPass pp = pro_pass(pl, pro, B, H, L, y != nullptr);
    if (pp.total && (!workspace || workspace_bytes < pp.total)) return PMA_ERR_WORKSPACE;
    if (pp.total && reinterpret_cast<uintptr_t>(workspace) % 16) return PMA_ERR_WORKSPACE;
    PrefillParams p{};
    p.B = B;
    p.H = H;
    p.L = L;
    p.seg_len = pl.seg_len;
    p.q = seq_of(q);
    p.k = seq_of(k);
    p.v = seq_of(v);
    p.pro = pro;
    p.y = seqout_of(y);
    p.lambda = beta;  // not read on the per-token path; any valid pointer
    p.lam_sb = 0;
    p.in = user_ref(state_in);
    p.out = user_ref(state_out);
    p.eps = eps;
    p.state_only = 0;
    p.status = nullptr;
    p.fault = g_fault_word.load();
    p.test_wait_ns = g_test_wait_ns.load();
    p.logdecay = log_decay;
    p.k_head_scale = beta;
    p.half_sq = 1;
    cudaError_t e;
    if (pl.tc) {
        p.status = reinterpret_cast<int *>(workspace);
        if ((e = cudaMemsetAsync(p.status, 0, sizeof(int), st)) != cudaSuccess) return cuda_fail(e);
        if ((e = run_prologue_passes(pp, pro, p, B, H, L, workspace, y != nullptr, di.sms, st)) != cudaSuccess)
            return cuda_fail(e);
        e = launch_prefill_tc(p, y ? y->dtype : PMA_F32, dim3(BH, 1), st);
    } else {
        e = launch_prefill_simt(p, D, q->dtype, y ? y->dtype : PMA_F32, dim3(BH, 1), st);
    }
    return e == cudaSuccess ? PMA_OK : cuda_fail(e);
}

int pma_selective_decode_step(int N, int H, int D, const pma_seq_tensor *q, const pma_seq_tensor *k,
                              const pma_seq_tensor *v, const pma_prologue *prologue, const float *log_decay,
                              const float *beta, const int32_t *rows, int pool_rows, const pma_state *state_in,
                              const pma_state *state_out, float eps, const pma_seq_tensor *y,
                              pma_stream_t stream) {
    if (!beta) return PMA_ERR_ARGUMENT;
    return decode_impl(N, H, D, q, k, v, prologue, log_decay, H, rows, pool_rows, state_in, state_out, eps, y,
                       stream, beta, true);
}

int pma_swiglu(int64_t rows, int inter, const void *gate, int64_t gate_stride, const void *up, int64_t up_stride,
               void *out, int64_t out_stride, int dtype, pma_stream_t stream) {
    if (rows < 0 || inter <= 0 || gate_stride < inter || up_stride < inter || out_stride < inter)
        return PMA_ERR_ARGUMENT;
    if (!supported_dtype(dtype)) return PMA_ERR_DTYPE;
    if (rows == 0) return PMA_OK;
    if (!gate || !up || !out) return PMA_ERR_ARGUMENT;
    int rc;
    DevInfo di;
    if ((rc = device_info(&di))) return rc;
    cudaError_t e = launch_swiglu(dtype, gate, gate_stride, up, up_stride, out, out_stride, rows, inter, di.sms,
                                  reinterpret_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? PMA_OK : cuda_fail(e);
}

size_t pma_gated_scan_workspace_bytes(int B, int L, int C) {
    return B <= 0 || L <= 0 || C <= 0 ? 0 : ScanWs::of(B, L, C).bytes(false);
}
size_t pma_gated_scan_backward_workspace_bytes(int B, int L, int C) {
    return B <= 0 || L <= 0 || C <= 0 ? 0 : ScanWs::of(B, L, C).bytes(true);
}

int pma_gated_scan(int B, int L, int C, const pma_seq_tensor *x, const pma_seq_tensor *f, const pma_seq_tensor *gate,
                   const float *bias, const float *h0, const uint8_t *reset, const pma_seq_tensor *y, float *h_last,
                   void *workspace, size_t workspace_bytes, pma_stream_t stream) {
    if (B < 0 || L < 0 || C <= 0) return PMA_ERR_ARGUMENT;
    int rc;
    const bool empty = B == 0 || L == 0;
    if ((rc = check_blc(x, x, empty)) || (rc = check_blc(f, x, empty)) || (gate && (rc = check_blc(gate, x, empty))) ||
        (rc = check_blc(y, x, empty)))
        return rc;
    if (!empty && h_last && h_last == h0) return PMA_ERR_ARGUMENT;  // every warp of the first tiles reads h0
    DevInfo di;
    if ((rc = device_info(&di))) return rc;
    if (B == 0) return PMA_OK;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    cudaError_t e;
    if (L == 0) {  // the state passes through
        if (!h_last || h_last == h0) return PMA_OK;
        const size_t n = (size_t)B * C * sizeof(float);
        e = h0 ? cudaMemcpyAsync(h_last, h0, n, cudaMemcpyDeviceToDevice, st) : cudaMemsetAsync(h_last, 0, n, st);
        return e == cudaSuccess ? PMA_OK : cuda_fail(e);
    }
    const ScanWs w = ScanWs::of(B, L, C);
    if (workspace_bytes < w.bytes(false) || (w.bytes(false) && (!workspace || (uintptr_t)workspace % 256)))
        return PMA_ERR_WORKSPACE;
    ScanParams p = scan_params(B, L, C, x, f, gate, bias, h0, reset);
    p.y = blc_of(y);
    p.h_last = h_last;
    const bool words = !scan_by_cluster(B, L, C, x->dtype, di.sms);
    if ((e = w.arm(p, workspace, words, st)) != cudaSuccess) return cuda_fail(e);
    e = launch_gated_scan(p, x->dtype, di.sms, st);
    return e == cudaSuccess ? PMA_OK : cuda_fail(e);
}

int pma_gated_scan_backward(int B, int L, int C, const pma_seq_tensor *x, const pma_seq_tensor *f,
                            const pma_seq_tensor *gate, const float *bias, const float *h0, const uint8_t *reset,
                            const pma_seq_tensor *dy, const float *dh_last, const pma_seq_tensor *dx,
                            const pma_seq_tensor *df, const pma_seq_tensor *dgate, float *dbias, float *dh0,
                            const void *forward_ws, size_t forward_ws_bytes, void *workspace, size_t workspace_bytes,
                            pma_stream_t stream) {
    if (B < 0 || L < 0 || C <= 0 || (gate == nullptr) != (dgate == nullptr)) return PMA_ERR_ARGUMENT;
    int rc;
    const bool empty = B == 0 || L == 0;
    for (const pma_seq_tensor *t : {x, f, dy, dx, df})
        if ((rc = check_blc(t, x, empty))) return rc;
    if (gate && ((rc = check_blc(gate, x, empty)) || (rc = check_blc(dgate, x, empty)))) return rc;
    if (!empty && dh0 && (dh0 == dh_last || dh0 == h0)) return PMA_ERR_ARGUMENT;
    DevInfo di;
    if ((rc = device_info(&di))) return rc;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    cudaError_t e;
    if (empty) {
        if (dbias && (e = cudaMemsetAsync(dbias, 0, (size_t)C * sizeof(float), st)) != cudaSuccess) return cuda_fail(e);
        if (!dh0 || B == 0 || dh0 == dh_last) return PMA_OK;
        const size_t n = (size_t)B * C * sizeof(float);
        e = dh_last ? cudaMemcpyAsync(dh0, dh_last, n, cudaMemcpyDeviceToDevice, st) : cudaMemsetAsync(dh0, 0, n, st);
        return e == cudaSuccess ? PMA_OK : cuda_fail(e);
    }
    const ScanWs w = ScanWs::of(B, L, C);
    if (forward_ws_bytes < w.bytes(false) || (w.bytes(false) && (!forward_ws || (uintptr_t)forward_ws % 256)))
        return PMA_ERR_WORKSPACE;
    if (workspace_bytes < w.bytes(true) || !workspace || (uintptr_t)workspace % 256) return PMA_ERR_WORKSPACE;
    ScanParams p = scan_params(B, L, C, x, f, gate, bias, h0, reset);
    p.dy = blc_of(dy);
    p.dh_last = dh_last;
    p.dx = blc_of(dx);
    p.df = blc_of(df);
    p.dgate = blc_of(dgate);
    p.dh0 = dh0;
    p.states = w.nwords && w.chunks > 1 ? w.incl(const_cast<void *>(forward_ws)) : nullptr;
    p.dbias_part = dbias ? w.part(workspace) : nullptr;
    const bool words = !scan_by_cluster(B, L, C, x->dtype, di.sms);
    if ((e = w.arm(p, workspace, words, st)) != cudaSuccess) return cuda_fail(e);
    e = launch_gated_scan_backward(p, x->dtype, dbias, di.sms, st);
    return e == cudaSuccess ? PMA_OK : cuda_fail(e);
}

int pma_gated_scan_step(int N, int C, const pma_seq_tensor *x, const pma_seq_tensor *f, const pma_seq_tensor *gate,
                        const float *bias, const float *h_in, float *h_out, const int32_t *rows, int pool_rows,
                        const pma_seq_tensor *y, pma_stream_t stream) {
    if (N < 0 || C <= 0 || (rows && pool_rows < 0)) return PMA_ERR_ARGUMENT;
    int rc;
    if ((rc = check_blc(x, x, N == 0)) || (rc = check_blc(f, x, N == 0)) || (gate && (rc = check_blc(gate, x, N == 0))) ||
        (rc = check_blc(y, x, N == 0)))
        return rc;
    if (N && (!h_in || !h_out)) return PMA_ERR_ARGUMENT;
    DevInfo di;
    if ((rc = device_info(&di))) return rc;
    if (N == 0) return PMA_OK;
    ScanStepParams p{};
    p.N = N;
    p.C = C;
    p.x = blc_of(x);
    p.f = blc_of(f);
    p.gate = blc_of(gate);
    p.y = blc_of(y);
    p.bias = bias;
    p.h_in = h_in;
    p.h_out = h_out;
    p.rows = rows;
    p.pool_rows = pool_rows;
    cudaError_t e = launch_gated_scan_step(p, x->dtype, reinterpret_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? PMA_OK : cuda_fail(e);
}

int pma_sample(int B, int V, const void *logits, int64_t row_stride, int dtype, const float *u,
               const float *temperature, float temperature_value, const int32_t *top_k, int top_k_value,
               const float *top_p, float top_p_value, const float *min_p, float min_p_value, int64_t *tokens,
               float *logprobs, pma_stream_t stream) {
    if (B < 0 || B > (1 << 27) || V <= 0 || V > SAMPLE_MAX_V || row_stride < 0 || (B > 1 && row_stride < V))
        return PMA_ERR_ARGUMENT;
    if (!supported_dtype(dtype)) return PMA_ERR_DTYPE;
    if (B == 0) return PMA_OK;
    if (!logits || !u || !tokens) return PMA_ERR_ARGUMENT;
    if (reinterpret_cast<uintptr_t>(logits) % esize(dtype)) return PMA_ERR_LAYOUT;
    int rc;
    DevInfo di;
    if ((rc = device_info(&di))) return rc;
    SampleParams p{};
    p.B = B;
    p.V = V;
    p.logits = logits;
    p.stride = row_stride;
    p.u = u;
    p.temperature = {temperature, temperature_value};
    p.top_k = {top_k, top_k_value};
    p.top_p = {top_p, top_p_value};
    p.min_p = {min_p, min_p_value};
    p.token = tokens;
    p.logprob = logprobs;
    cudaError_t e = launch_sample(p, dtype, di.sms, reinterpret_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? PMA_OK : cuda_fail(e);
}

int pma_fp8_quantize(int M, int K, const void *x, int64_t x_stride, int dtype, void *q, int64_t q_stride, float *scale,
                     int64_t scale_stride_m, int64_t scale_stride_k, pma_stream_t stream) {
    if (M < 0 || K <= 0 || scale_stride_m < 0 || scale_stride_k < 0) return PMA_ERR_ARGUMENT;
    if (M == 0) return PMA_OK;
    int rc;
    if ((rc = check_dense(x, x_stride, dtype, M, K)) || (rc = check_e4m3(q, q_stride, K))) return rc;
    if (!scale) return PMA_ERR_ARGUMENT;
    DevInfo di;
    if ((rc = device_info(&di))) return rc;
    const cudaError_t e = launch_fp8_quantize(x, x_stride, dtype, M, K, static_cast<uint8_t *>(q), q_stride, scale,
                                              scale_stride_m, scale_stride_k, di.sms, reinterpret_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? PMA_OK : cuda_fail(e);
}

int pma_fp8_quantize_weight(int N, int K, const void *w, int64_t w_stride, int dtype, void *q, int64_t q_stride,
                            float *scale, pma_stream_t stream) {
    if (N < 0 || K <= 0) return PMA_ERR_ARGUMENT;
    if (N == 0) return PMA_OK;
    int rc;
    if ((rc = check_dense(w, w_stride, dtype, N, K)) || (rc = check_e4m3(q, q_stride, K))) return rc;
    if (!scale) return PMA_ERR_ARGUMENT;
    DevInfo di;
    if ((rc = device_info(&di))) return rc;
    const cudaError_t e = launch_fp8_quantize_weight(w, w_stride, dtype, N, K, static_cast<uint8_t *>(q), q_stride,
                                                     scale, reinterpret_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? PMA_OK : cuda_fail(e);
}

static int fp8_matmul_impl(int M, int N, int K, const void *xq, int64_t xq_stride, const float *x_scale,
                           int64_t x_scale_stride_m, int64_t x_scale_stride_k, const void *wq, int64_t wq_stride,
                           const float *w_scale, int64_t w_scale_stride, void *y, int64_t y_stride, int y_dtype,
                           bool after_quantize, pma_stream_t stream) {
    if (M < 0 || N <= 0 || K <= 0 || x_scale_stride_m < 0 || x_scale_stride_k < 0) return PMA_ERR_ARGUMENT;
    if (!supported_dtype(y_dtype)) return PMA_ERR_DTYPE;
    if (M == 0) return PMA_OK;
    int rc;
    if ((rc = check_e4m3(xq, xq_stride, K)) || (rc = check_e4m3(wq, wq_stride, K))) return rc;
    const int blocks = (K + FP8_BLOCK - 1) / FP8_BLOCK;
    if (!x_scale || !w_scale || w_scale_stride < blocks || !y || (M > 1 && y_stride < N)) return PMA_ERR_ARGUMENT;
    if ((uintptr_t)y % esize(y_dtype)) return PMA_ERR_LAYOUT;
    DevInfo di;
    if ((rc = device_info(&di))) return rc;
    return fp8_product(M, N, K, {static_cast<const uint8_t *>(xq), xq_stride, x_scale, x_scale_stride_m, x_scale_stride_k},
                       {static_cast<const uint8_t *>(wq), wq_stride, w_scale, w_scale_stride, 1}, y, y_stride, y_dtype,
                       di.sms, after_quantize, reinterpret_cast<cudaStream_t>(stream));
}

int pma_fp8_matmul(int M, int N, int K, const void *xq, int64_t xq_stride, const float *x_scale,
                   int64_t x_scale_stride_m, int64_t x_scale_stride_k, const void *wq, int64_t wq_stride,
                   const float *w_scale, int64_t w_scale_stride, void *y, int64_t y_stride, int y_dtype,
                   pma_stream_t stream) {
    return fp8_matmul_impl(M, N, K, xq, xq_stride, x_scale, x_scale_stride_m, x_scale_stride_k, wq, wq_stride, w_scale,
                           w_scale_stride, y, y_stride, y_dtype, false, stream);
}

size_t pma_fp8_linear_workspace_bytes(int M, int K) { return M <= 0 || K <= 0 ? 0 : Fp8Ws::of(M, K).bytes; }

int pma_fp8_linear(int M, int N, int K, const void *x, int64_t x_stride, int x_dtype, const void *wq, int64_t wq_stride,
                   const float *w_scale, int64_t w_scale_stride, void *y, int64_t y_stride, int y_dtype,
                   void *workspace, size_t workspace_bytes, pma_stream_t stream) {
    if (M < 0 || N <= 0 || K <= 0) return PMA_ERR_ARGUMENT;
    if (M == 0) return PMA_OK;
    const Fp8Ws w = Fp8Ws::of(M, K);
    if (workspace_bytes < w.bytes || !workspace || (uintptr_t)workspace % 256) return PMA_ERR_WORKSPACE;
    float *scale = reinterpret_cast<float *>((char *)workspace + w.scale_at);
    const int rc = pma_fp8_quantize(M, K, x, x_stride, x_dtype, workspace, w.stride, scale, 1, M, stream);
    return rc ? rc
              : fp8_matmul_impl(M, N, K, workspace, w.stride, scale, 1, M, wq, wq_stride, w_scale, w_scale_stride, y,
                                y_stride, y_dtype, true, stream);
}

int pma_state_combine(int B, int H, int D, const float *lambda, int64_t lambda_stride_b, int64_t len,
                      const pma_state *T, const pma_state *P, pma_stream_t stream) {
    if (B < 0 || H <= 0 || !lambda || lambda_stride_b < 0 || len < 0) return PMA_ERR_ARGUMENT;
    if (!supported_d(D)) return PMA_ERR_HEAD_DIM;
    int rc;
    if ((rc = check_state(T)) || (rc = check_state(P))) return rc;
    DevInfo di;
    if ((rc = device_info(&di))) return rc;
    if (B == 0) return PMA_OK;
    cudaError_t e = launch_state_combine(B, H, D, lambda, lambda_stride_b, len, *T, *P,
                                         reinterpret_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? PMA_OK : cuda_fail(e);
}

}  // extern "C"
