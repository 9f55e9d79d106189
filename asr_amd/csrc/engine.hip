// libasr_amd.so -- handle, weight store, workspaces, encoder / beam-search orchestration and the
// C ABI of include/asr_amd.h.  One handle = one GPU.  Reference citations are relative to
// /root/reference/transformer/.
#include "asr_common.h"
#include "../../include/asr_amd.h"
#include "ops_common.h"

#include <math.h>
#include <stdio.h>
#include <string.h>

#include <algorithm>
#include <deque>
#include <map>
#include <memory>
#include <new>
#include <mutex>
#include <string>
#include <vector>

namespace {

std::string g_create_error;

// ---- scratch of the allocation-free entry point (asr_op_input_norm_timing_noalloc) ----------------------------
// The per-utterance partial sums of the input layer norm (rowops.hip: 2 x 64 doubles per utterance) live in this
// file-scope device array instead of a hipMalloc'ed buffer.  In host code the array's NAME is only a stand-in (passing
// it to a kernel compiles and then faults the GPU): asr_create resolves its device address once per device, with that
// device current, by hipGetSymbolAddress, and host code uses that pointer everywhere.  Every GPU the library runs on
// holds its own 1 MiB copy until the process ends.
constexpr int NOALLOC_MAX_UTTS = 1024;
constexpr int NOALLOC_DOUBLES_PER_UTT = 128;
constexpr int MAX_DEVICES = 64;
constexpr int MAX_VIEWS = 4;        // sub-batches a beam search may run as (asr_config.sub_batches)
// Handles that share the GPU choose the K-slices of their decode-row GEMMs independently of the row count from this many beam
// rows up (decode_splits, logit_split_for): a whole batch and a joint decode of two or more of them then sum in the same order,
// which is what lets asr_amd.model pair whole batches with bit-identical hypotheses (PAIR_MIN_ROWS there is this number).
// 448 = 45 utterances at beam 10: BASELINE config 5's 50-utterance batches count as whole.
constexpr int WHOLE_BATCH_ROWS_DEFAULT = 448;
static int whole_batch_rows()
{
    static const int v = [] { const char* e = getenv("ASR_AMD_WHOLE_ROWS"); const int x = e ? atoi(e) : 0; return x > 0 ? x : WHOLE_BATCH_ROWS_DEFAULT; }();   // (development)
    return v;
}
static __device__ __align__(256) double g_norm_scratch[NOALLOC_MAX_UTTS * NOALLOC_DOUBLES_PER_UTT];
double* g_norm_scratch_ptr[MAX_DEVICES] = {};      // device address of g_norm_scratch on device d (null: not resolved yet)
std::mutex g_norm_scratch_mu[MAX_DEVICES];         // held while a device's entry is resolved (asr_create) and, by the allocation-free
                                                   // entry point, from its launch to the end of its wait: handles of one GPU on
                                                   // several host threads (EnginePool) take turns on that GPU's one array

// The packed weights of one checkpoint on one GPU.  Handles of one GPU may share a store (asr_share_weights): the planes are
// read-only once asr_finalize_weights has returned, so an EnginePool of four handles holds them once instead of four times.
struct WeightStore {
    int device = 0;
    std::vector<void*> allocs;
    int64_t bytes = 0;
    ~WeightStore()
    {
        if (allocs.empty()) return;
        (void)hipSetDevice(device);
        for (void* p : allocs) (void)hipFree(p);
    }
};

struct HostTensor {
    std::vector<float> data;
    std::vector<int64_t> shape;
};

struct ProfClass {
    const char* name;
    double ms = 0.0;
    int64_t launches = 0;
    double flops = 0.0, bytes = 0.0;
};

struct EncBlock {
    float *wqkv, *bqkv, *wo, *bo, *ln0s, *ln0b, *w1, *b1, *w2, *b2, *ln1s, *ln1b;
};
struct DecBlock {
    float *wqkv, *bqkv, *wo, *bo, *ln0s, *ln0b;
    float *wq, *bq, *wkv, *bkv, *wco, *bco, *ln1s, *ln1b;
    float *w1, *b1, *w2, *b2, *ln2s, *ln2b;
};

}  // namespace

struct asr_handle {
    asr_config cfg;
    int H = 0, heads = 0, L = 0, V = 0, D = 0, F = 0, K = 0;
    bool glu = false;
    int ff_epi = EPI_RELU;
    int nprod = 0;                      // 0: exact f32 MFMA GEMMs; 13: fp16x3, 6 / 3 / 1: bf16 planes (gemm_split.hip)
    int nprod_active = 0;               // = nprod, except while a call is repeated on the bf16x6 kernels (13 -> 6)
    int32_t* range_flag = nullptr;      // device: set by an fp16x3 GEMM that met an activation outside fp16's range
    int64_t range_retries = 0;          // calls repeated on the bf16x6 kernels so far
    bool weights_out_of_range = false;  // single-kernel probes: the caller's weight operand did not fit fp16
    bool kv_bf16 = false;               // precision bf16: K/V caches (self and cross) stored as bf16 (attention.hip KV16)
    // a joint decode of groups with different T (asr_decode_groups), for the duration of the call: per-utterance key
    // counts and first-key row offsets of the cross attention (device, [n]) and the keys of all utterances together
    const int32_t* grp_t = nullptr;
    const int32_t* grp_off = nullptr;
    double grp_rows = 0.0;
    int32_t* grp_buf = nullptr;         // device home of those arrays and of the per-utterance loop limits: [3][grp_cap]
    size_t grp_cap = 0;
    int logit_split = 1;                // K slices of the logits GEMM (their slabs are summed by the top-k kernel)
    int logit_split_shared = 2;         // ... of handles that share the GPU, from whole_batch_rows() beam rows (env ASR_AMD_LOGIT_SPLIT_SHARED: development)
    float* emb_gemm = nullptr;          // logits operand when tied: = emb (f32 mode) or its bf16 planes
    hipStream_t stream = nullptr;
    mutable std::string err;
    std::map<std::string, HostTensor> staged;
    bool finalized = false;

    std::map<void*, size_t> allocs;     // everything hipMalloc'ed through dev_alloc -> bytes (the handle's own: caches, workspaces)
    int64_t dev_bytes = 0;
    std::shared_ptr<WeightStore> wstore;    // the weights (asr_finalize_weights fills one; asr_share_weights adopts another handle's)
    bool wstore_filling = false;        // dev_alloc books into the store (only while asr_finalize_weights uploads)
    bool wstore_owner = false;          // this handle created the store: asr_device_bytes counts it here and nowhere else

    // weights
    float *w_src = nullptr, *b_src = nullptr, *in_gamma = nullptr, *in_beta = nullptr;
    float *emb = nullptr, *softmax_w = nullptr;
    std::vector<EncBlock> enc;
    std::vector<DecBlock> dec;
    float* pe = nullptr;
    int pe_rows = 0;

    // encoder workspaces (capacity in rows = n*t)
    size_t cap_rows = 0;
    int cap_n = 0, cap_t = 0;
    float *xin = nullptr, *x0 = nullptr, *x1 = nullptr, *x2 = nullptr, *x3 = nullptr, *qkv = nullptr, *hid = nullptr;
    int32_t *pad = nullptr, *pad2 = nullptr;
    double* norm_scratch = nullptr;
    std::vector<float*> cross_k, cross_v;

    // decoder workspaces (capacity in rows = n*K)
    int cap_dec_n = 0;
    float *y0 = nullptr, *z1 = nullptr, *z2 = nullptr, *dctx = nullptr, *part = nullptr, *dhid = nullptr, *logits = nullptr;
    float* cand_scores = nullptr;
    int32_t* cand_tokens = nullptr;
    std::vector<float*> kcache, vcache;
    BeamState beam{};
    int32_t* done_host = nullptr;       // pinned, [MAX_VIEWS][max_target_length + 8]
    std::vector<hipEvent_t> step_events;    // [MAX_VIEWS][8]
    // The beam search of a batch may run as two independent halves (utterances are independent) on two streams,
    // so that the launch gaps and tails of one half's kernels are filled by the other's (ASR_AMD_SUBBATCH=1 disables)
    hipStream_t xstream[3] = {nullptr, nullptr, nullptr};   // streams of sub-batches 1..3 (sub-batch 0 runs on `stream`)
    hipEvent_t fork_ev = nullptr;
    std::string twice;                  // ASR_AMD_DOUBLE (measurement aid): decode kernel class that is launched twice
    bool shared_gpu = false;            // asr_config.shared_gpu: other handles keep the GPU busy, prefer fewer K-slices
    int use_graph = -1;                 // steps 2.. of the beam search replayed from a captured HIP graph: 1 always, 0 never,
                                        // -1 from 320 beam rows up (the sub-batch regime, where the host issues 100 000 launches a
                                        // second without it); env ASR_AMD_GRAPH
    int sub_batches = 0;                // 0 = automatic (two halves from 320 rows), 1 = never, 2..4 = that many parts whenever n allows

    // profile
    int profile = 0;
    std::vector<ProfClass> prof;
    double prof_overhead_ms = 0.0;     // elapsed time of an event pair with nothing between (calibrated by asr_set_profile)
    hipEvent_t pe0 = nullptr, pe1 = nullptr;
    // profile mode 2 (brackets left in the queue, no host wait per kernel: the durations kernels have in the running
    // pipeline, the other sub-batch's kernels beside them): a pool of events and the brackets not yet read back
    struct ProfPending { int cls; hipEvent_t e0, e1; };
    std::vector<hipEvent_t> prof_free;
    std::deque<ProfPending> prof_pending;
    int32_t* live_host = nullptr;      // pinned [steps + 2][n]: live-row counts per step (what self-attention streamed)
    size_t live_host_cap = 0;
    int live_host_n = 0;
};

namespace {

#define HIP_TRY(h, expr)                                                                              \
    do {                                                                                              \
        hipError_t e__ = (expr);                                                                      \
        if (e__ != hipSuccess) {                                                                      \
            (h)->err = std::string(#expr) + ": " + hipGetErrorString(e__);                            \
            return ASR_ERR_HIP;                                                                       \
        }                                                                                             \
    } while (0)

int fail(asr_handle* h, int code, const std::string& msg)
{
    h->err = msg;
    return code;
}

// Blocking copy on the handle's own stream.  (The plain hipMemcpy runs on the legacy stream, which the runtime ties to
// every other stream of the process: it is refused while ANOTHER handle's thread is capturing its decode step into a graph,
// and it is a meeting point of handles that should run free of each other.)
hipError_t copy_blocking(asr_handle* h, void* dst, const void* src, size_t bytes, hipMemcpyKind kind, hipStream_t stream = nullptr)
{
    if (!stream) stream = h->stream;
    const hipError_t e = hipMemcpyAsync(dst, src, bytes, kind, stream);
    return e != hipSuccess ? e : hipStreamSynchronize(stream);
}

int dev_alloc(asr_handle* h, void** p, size_t bytes)
{
    if (bytes == 0) bytes = 16;
    HIP_TRY(h, hipMalloc(p, bytes));
    if (h->wstore_filling && h->wstore) {
        h->wstore->allocs.push_back(*p);
        h->wstore->bytes += (int64_t)bytes;
        return ASR_OK;
    }
    h->allocs[*p] = bytes;
    h->dev_bytes += (int64_t)bytes;
    return ASR_OK;
}

void dev_free(asr_handle* h, void* p)
{
    if (!p) return;
    auto it = h->allocs.find(p);
    if (it != h->allocs.end()) { h->dev_bytes -= (int64_t)it->second; h->allocs.erase(it); }
    (void)hipFree(p);
}

template <typename T>
int dev_alloc_t(asr_handle* h, T** p, size_t count)
{
    return dev_alloc(h, reinterpret_cast<void**>(p), count * sizeof(T));
}

// ---- profile brackets -----------------------------------------------------------------------
hipEvent_t prof_event(asr_handle* h)
{
    hipEvent_t e = nullptr;
    if (!h->prof_free.empty()) { e = h->prof_free.back(); h->prof_free.pop_back(); }
    else if (hipEventCreate(&e) != hipSuccess) e = nullptr;
    return e;
}

// reads back the brackets of profile mode 2 in launch order; wait = false stops at the first one still in flight
void prof_drain(asr_handle* h, bool wait)
{
    while (!h->prof_pending.empty()) {
        const asr_handle::ProfPending p = h->prof_pending.front();
        if (wait) (void)hipEventSynchronize(p.e1);
        else if (hipEventQuery(p.e1) != hipSuccess) break;
        float ms = 0.f;
        if (hipEventElapsedTime(&ms, p.e0, p.e1) == hipSuccess && p.cls < (int)h->prof.size())
            h->prof[p.cls].ms += std::max(0.0, (double)ms - h->prof_overhead_ms);
        h->prof_free.push_back(p.e0);
        h->prof_free.push_back(p.e1);
        h->prof_pending.pop_front();
    }
}

struct ProfScope {
    asr_handle* h;
    int cls = -1;
    hipStream_t st;
    hipEvent_t e0 = nullptr, e1 = nullptr;
    // `stream` = the stream the bracketed kernel is launched on (a half batch's kernels run on their own stream)
    ProfScope(asr_handle* h_, const char* name, double flops, double bytes, hipStream_t stream = nullptr) : h(h_), st(stream ? stream : h_->stream)
    {
        if (!h->profile) return;
        for (size_t i = 0; i < h->prof.size(); ++i)
            if (h->prof[i].name == name || strcmp(h->prof[i].name, name) == 0) { cls = (int)i; break; }
        if (cls < 0) {
            h->prof.push_back(ProfClass{name});
            cls = (int)h->prof.size() - 1;
        }
        ProfClass& pc = h->prof[cls];
        pc.flops += flops;
        pc.bytes += bytes;
        pc.launches += 1;
        if (h->profile == 2) {
            e0 = prof_event(h); e1 = prof_event(h);
            if (e0 && e1) (void)hipEventRecord(e0, st);
        } else {
            (void)hipEventRecord(h->pe0, st);
        }
    }
    ~ProfScope()
    {
        if (cls < 0) return;
        if (h->profile == 2) {
            if (e0 && e1) {
                (void)hipEventRecord(e1, st);
                h->prof_pending.push_back(asr_handle::ProfPending{cls, e0, e1});
            }
            return;
        }
        (void)hipEventRecord(h->pe1, st);
        (void)hipEventSynchronize(h->pe1);
        float ms = 0.f;
        (void)hipEventElapsedTime(&ms, h->pe0, h->pe1);
        h->prof[cls].ms += std::max(0.0, (double)ms - h->prof_overhead_ms);    // minus what an EMPTY event pair measures
    }
};

// bf16-plane kernels need whole 32-deep k-tiles; a GEMM whose K is not a multiple of 32 (no layer of the reference
// configs; the single-kernel probes allow it) runs on the exact-f32 kernel in every precision mode.  Uploads and
// launches both decide by this function, so the operand format always matches the kernel.
inline int gemm_nprod(const asr_handle* h, int K) { return (K & 31) ? 0 : h->nprod_active; }
// In fp16x3 mode (nprod 13) every plane-format operand holds both formats, [fp16 planes | bf16x6 planes], so that a call
// whose activations leave fp16's range can be repeated on the bf16x6 kernels without touching the weights again.
inline bool dual_format(const asr_handle* h, int K) { return h->nprod == 13 && !(K & 31); }
inline size_t plane_elems(const asr_handle* h, int n, int k)
{
    if (dual_format(h, k)) return gemm_split_weight_elems(n, k, 2) + gemm_split_weight_elems(n, k, 3);
    return gemm_split_weight_elems(n, k, gemm_split_planes(h->nprod));
}
// packs `w` [n][k] into `out` (plane_elems() uint16 values); false: a weight does not fit fp16 (fp16x3 mode only)
inline bool pack_planes(const asr_handle* h, const float* w, int n, int k, uint16_t* out)
{
    if (!dual_format(h, k)) return gemm_split_weights_host(w, n, k, h->nprod, out);
    const bool ok = gemm_split_weights_host(w, n, k, 13, out);
    gemm_split_weights_host(w, n, k, 6, out + gemm_split_weight_elems(n, k, 2));
    return ok;
}

// Tile of the split GEMM for this handle: handles that share the GPU (asr_config.shared_gpu) do not take the 96 x 256 tile -
// it exists to get a whole-batch launch through the chip in ONE round of workgroups, at the price of 5 % padded rows, and
// with other handles' kernels in the queue there are no idle rounds to avoid (four steps in flight, same box: 203.0 -> 201.7 ms).
inline int split_tile_for(const asr_handle* h, int M, int N, int K, int split_k, int epilogue)
{
    static const int forced = getenv("ASR_AMD_DECODE_TILE") ? atoi(getenv("ASR_AMD_DECODE_TILE")) : 0;   // development: 2, 6 or 9 for the decode rows
    if (forced && M <= 4096) return forced;
    const int t = gemm_split_pick_tile(M, N, K, split_k, epilogue);
    // One-product mode (bf16) with handles sharing the GPU, two whole batches per call (1000+ beam rows): a k-tile's side work
    // (loads, A staging, fragment reads) outweighs its four matrix instructions at 64 rows, so 128 x 256 tiles - the same side
    // work for eight.  Same box, four handles x two steps: 104.7 -> 103.3 ms per step (config 5: 132.0 -> 131.0); the three-product
    // mode loses 7 % with it (its k-tiles are matrix-bound and fewer workgroups balance worse).
    if (h->nprod_active == 1 && h->shared_gpu && M >= 1000 && M <= 4096 && t == 9) return 10;
    return (t == 6 && h->shared_gpu) ? 9 : t;
}

// Measurement aid (ASR_AMD_DOUBLE=glu|proj|qkv|ffn2|logits|self|cross|ln|topk|encoder): the decode-step kernels of that class are launched
// twice - every one of them is idempotent (same inputs, same outputs) - so the change in step time is what that class costs
// with everything else as it is (the costs add up to the step).  1 launch when unset.
// Arithmetic of the many-query attention kernels (attention.hip launch_mha) for this handle's current mode: the dense layers'
// fp16x3 / bf16 product schemes, or the exact-f32 matrix instruction (f32, f32_bf16x6, bf16x3, and an fp16x3 call that is being
// repeated after a range flag).  ASR_AMD_MHA_EXACT=1: development (always exact).
inline int mha_mode(const asr_handle* h)
{
    static const bool exact = getenv("ASR_AMD_MHA_EXACT") && atoi(getenv("ASR_AMD_MHA_EXACT")) != 0;
    if (exact) return 0;
    return h->nprod_active == 13 ? 13 : (h->nprod_active == 1 ? 1 : 0);
}
inline bool self_exact()                  // ASR_AMD_SELF_EXACT=1 (development): decode self-attention on the exact-f32 instruction in every mode
{
    static const bool v = getenv("ASR_AMD_SELF_EXACT") && atoi(getenv("ASR_AMD_SELF_EXACT")) != 0;
    return v;
}
inline int launches_of(const asr_handle* h, const char* cls) { return (!h->twice.empty() && h->twice == cls) ? 2 : 1; }

const char* gemm_class_name(const asr_handle* h, int nprod, int M, int N, int K, int epilogue, int split_k)
{
    static std::map<std::string, std::string> interned;           // stable c_str() for ProfClass::name
    static std::mutex interned_mu;                                // handles on other GPUs / other host threads share it
    const int tile = nprod == 0 ? gemm_f32_pick_tile(M, N, split_k, epilogue) : split_tile_for(h, M, N, K, split_k, epilogue);
    std::string n = nprod == 0 ? "gemm_f32_nt" : nprod == 13 ? "gemm_f16x3_nt" : nprod == 6 ? "gemm_bf16x6_nt" : nprod == 3 ? "gemm_bf16x3_nt" : "gemm_bf16_nt";
    if (nprod) n += tile == 1 ? "<128,128," : tile == 5 ? "<160,128," : tile == 6 ? "<96,256," : tile == 10 ? "<128,256," : tile == 7 || tile == 9 ? "<64,256," : "<64,128,";
    else n += tile == 1 ? "<128,128," : tile == 4 ? "<128,64," : "<64,64,";
    n += epilogue == EPI_GLU ? "GLU>" : epilogue == EPI_PARTIAL ? "PARTIAL>" : epilogue == EPI_BIAS ? "BIAS>" : "ACT>";
    std::lock_guard<std::mutex> lock(interned_mu);
    auto it = interned.find(n);
    if (it == interned.end()) it = interned.emplace(n, n).first;
    return it->second.c_str();
}

int gemm(asr_handle* h, const float* A, const float* W, const float* bias, float* C, int M, int N, int K, int epilogue,
         int split_k, hipStream_t stream = nullptr)
{
    if (!stream) stream = h->stream;
    GemmArgs a{};
    a.A = A; a.W = W; a.Wp = reinterpret_cast<const uint16_t*>(W); a.bias = bias; a.C = C;
    a.M = M; a.N = N; a.K = K;
    a.lda = K; a.ldw = K;
    a.ldc = (epilogue == EPI_GLU) ? N / 2 : N;
    a.split_k = split_k;
    a.epilogue = epilogue;
    const double nout = (epilogue == EPI_GLU) ? N / 2.0 : (double)N * split_k;
    const int nprod = gemm_nprod(h, K);
    if (nprod == 6 && dual_format(h, K)) a.Wp += gemm_split_weight_elems(N, K, 2);        // the bf16x6 copy (a repeated call)
    a.range_flag = nprod == 13 ? h->range_flag : nullptr;
    const double wbytes = nprod ? 2.0 * gemm_split_planes(nprod) : 4.0;
    ProfScope ps(h, h->profile ? gemm_class_name(h, nprod, M, N, K, epilogue, split_k) : "", 2.0 * M * N * (double)K,
                 4.0 * ((double)M * K + (double)M * nout) + wbytes * (double)N * K, stream);
    const char* cls = M > 4096 ? "" : epilogue == EPI_GLU ? "glu" : K == h->F ? "ffn2" : N == 3 * h->H ? "qkv" : N == h->V ? "logits" :
                      (N == h->H && K == h->H) ? "proj" : "";
    for (int rep = launches_of(h, cls); rep > 1; --rep)
        if (nprod) HIP_TRY(h, launch_gemm_split(a, nprod, split_tile_for(h, M, N, K, split_k, epilogue), stream));
    if (nprod) HIP_TRY(h, launch_gemm_split(a, nprod, split_tile_for(h, M, N, K, split_k, epilogue), stream));
    else HIP_TRY(h, launch_gemm_f32(a, 0, stream));
    return ASR_OK;
}

// ---- timing signal table (third_party/tensor2tensor/common_attention.py:28-69), evaluated with
// correctly rounded float32 elementary functions in the graph's op order -----------------------
std::vector<float> timing_table(int rows, int channels)
{
    std::vector<float> t((size_t)rows * channels, 0.f);
    const int nts = channels / 2;
    const float inc = (float)log(1.0e5 / 1.0) / ((float)nts - 1.0f);
    std::vector<float> inv(nts);
    for (int j = 0; j < nts; ++j) inv[j] = 1.0f * (float)exp((double)((float)j * -inc));
    for (int p = 0; p < rows; ++p)
        for (int j = 0; j < nts; ++j) {
            const float st = (float)p * inv[j];
            t[(size_t)p * channels + j] = (float)sin((double)st);
            t[(size_t)p * channels + nts + j] = (float)cos((double)st);
        }
    return t;
}

int ensure_pe(asr_handle* h, int rows)
{
    if (rows <= h->pe_rows) return ASR_OK;
    rows = std::max(rows, 512);
    if (h->pe) dev_free(h, h->pe);
    h->pe = nullptr;
    std::vector<float> t = timing_table(rows, h->H);
    int rc = dev_alloc_t(h, &h->pe, t.size());
    if (rc) return rc;
    HIP_TRY(h, copy_blocking(h, h->pe, t.data(), t.size() * sizeof(float), hipMemcpyHostToDevice));
    h->pe_rows = rows;
    return ASR_OK;
}

// ---- variable table -----------------------------------------------------------------
struct VarSpec { std::string name; std::vector<int64_t> shape; };

std::vector<VarSpec> required_vars(const asr_handle* h)
{
    const int64_t H = h->H, D = h->D, V = h->V, F = h->F;
    std::vector<VarSpec> v;
    auto add = [&](const std::string& n, std::vector<int64_t> s) { v.push_back({n, std::move(s)}); };
    add("encoder/src_change/kernel", {H, D});
    add("encoder/src_change/bias", {H});
    add("encoder/LayerNorm/beta", {H});
    add("encoder/LayerNorm/gamma", {H});
    auto ffn = [&](const std::string& p) {
        if (h->glu) {
            add(p + "/ff_hidden/dense/arg1/kernel", {F, H}); add(p + "/ff_hidden/dense/arg1/bias", {F});
            add(p + "/ff_hidden/dense/arg2/kernel", {F, H}); add(p + "/ff_hidden/dense/arg2/bias", {F});
        } else {
            add(p + "/ff_hidden/dense/kernel", {F, H}); add(p + "/ff_hidden/dense/bias", {F});
        }
        add(p + "/ff_hidden/dense_1/kernel", {H, F}); add(p + "/ff_hidden/dense_1/bias", {H});
    };
    auto ln = [&](const std::string& p, const char* n) {
        add(p + "/" + n + "/layer_norm_scale", {H}); add(p + "/" + n + "/layer_norm_bias", {H});
    };
    for (int i = 0; i < h->L; ++i) {
        const std::string p = "encoder/block_" + std::to_string(i);
        add(p + "/encoder_self_attention/qkv_transform/kernel", {3 * H, H});
        add(p + "/encoder_self_attention/qkv_transform/bias", {3 * H});
        add(p + "/encoder_self_attention/output_transform/kernel", {H, H});
        add(p + "/encoder_self_attention/output_transform/bias", {H});
        ffn(p); ln(p, "layer_norm"); ln(p, "layer_norm_1");
    }
    add("decoder/dst_embedding/kernel", {V, H});
    if (!h->cfg.tie_embedding_and_softmax) add("decoder/softmax/kernel", {V, H});
    for (int i = 0; i < h->L; ++i) {
        const std::string p = "decoder/block_" + std::to_string(i);
        add(p + "/decoder_self_attention/qkv_transform/kernel", {3 * H, H});
        add(p + "/decoder_self_attention/qkv_transform/bias", {3 * H});
        add(p + "/decoder_self_attention/output_transform/kernel", {H, H});
        add(p + "/decoder_self_attention/output_transform/bias", {H});
        add(p + "/decoder_vanilla_attention/q_transform/kernel", {H, H});
        add(p + "/decoder_vanilla_attention/q_transform/bias", {H});
        add(p + "/decoder_vanilla_attention/kv_transform/kernel", {2 * H, H});
        add(p + "/decoder_vanilla_attention/kv_transform/bias", {2 * H});
        add(p + "/decoder_vanilla_attention/output_transform/kernel", {H, H});
        add(p + "/decoder_vanilla_attention/output_transform/bias", {H});
        ffn(p); ln(p, "layer_norm"); ln(p, "layer_norm_1"); ln(p, "layer_norm_2");
    }
    return v;
}

bool is_ignored_var(const std::string& n)
{
    auto ends_with = [&](const char* s) { const size_t l = strlen(s); return n.size() >= l && n.compare(n.size() - l, l, s) == 0; };
    return ends_with("/Adam") || ends_with("/Adam_1") || n == "beta1_power" || n == "beta2_power" ||
           n.compare(0, 11, "global_step") == 0;
}

int upload(asr_handle* h, const std::string& name, float** dst)
{
    const HostTensor& t = h->staged.at(name);
    int rc = dev_alloc_t(h, dst, t.data.size());
    if (rc) return rc;
    HIP_TRY(h, copy_blocking(h, *dst, t.data.data(), t.data.size() * sizeof(float), hipMemcpyHostToDevice));
    return ASR_OK;
}

// a GEMM operand: f32 [N][K] as is, or split into bf16 planes [planes][N][K] (gemm_split.hip)
int upload_gemm_host(asr_handle* h, const float* w, int n, int k, float** dst)
{
    const size_t count = (size_t)n * k;
    if (gemm_nprod(h, k) == 0) {
        int rc = dev_alloc_t(h, dst, count);
        if (rc) return rc;
        HIP_TRY(h, copy_blocking(h, *dst, w, count * sizeof(float), hipMemcpyHostToDevice));
        return ASR_OK;
    }
    std::vector<uint16_t> planes(plane_elems(h, n, k));
    if (!pack_planes(h, w, n, k, planes.data())) return fail(h, ASR_ERR_WEIGHTS, "a weight does not fit fp16 (precision f32_f16x3)");
    uint16_t* d = nullptr;
    int rc = dev_alloc_t(h, &d, planes.size());
    if (rc) return rc;
    HIP_TRY(h, copy_blocking(h, d, planes.data(), planes.size() * sizeof(uint16_t), hipMemcpyHostToDevice));
    *dst = reinterpret_cast<float*>(d);
    return ASR_OK;
}

int upload_gemm(asr_handle* h, const std::string& name, float** dst)
{
    const HostTensor& t = h->staged.at(name);
    if (t.shape.size() != 2) return fail(h, ASR_ERR_ARG, "GEMM operand is not a matrix");
    return upload_gemm_host(h, t.data.data(), (int)t.shape[0], (int)t.shape[1], dst);
}

// ff_hidden first dense: GLU weights packed [2F][H] per 32 rows: 16 value rows | 16 gate rows
int upload_ffn1(asr_handle* h, const std::string& p, float** w, float** b)
{
    if (!h->glu) {
        int rc = upload_gemm(h, p + "/ff_hidden/dense/kernel", w);
        if (rc) return rc;
        return upload(h, p + "/ff_hidden/dense/bias", b);
    }
    const HostTensor& w1 = h->staged.at(p + "/ff_hidden/dense/arg1/kernel");
    const HostTensor& w2 = h->staged.at(p + "/ff_hidden/dense/arg2/kernel");
    const HostTensor& b1 = h->staged.at(p + "/ff_hidden/dense/arg1/bias");
    const HostTensor& b2 = h->staged.at(p + "/ff_hidden/dense/arg2/bias");
    const int F = h->F, H = h->H;
    std::vector<float> wp((size_t)2 * F * H), bp((size_t)2 * F);
    for (int g = 0; g < F / 16; ++g)
        for (int r = 0; r < 16; ++r) {
            memcpy(&wp[((size_t)g * 32 + r) * H], &w1.data[((size_t)g * 16 + r) * H], (size_t)H * sizeof(float));
            memcpy(&wp[((size_t)g * 32 + 16 + r) * H], &w2.data[((size_t)g * 16 + r) * H], (size_t)H * sizeof(float));
            bp[(size_t)g * 32 + r] = b1.data[(size_t)g * 16 + r];
            bp[(size_t)g * 32 + 16 + r] = b2.data[(size_t)g * 16 + r];
        }
    int rc = upload_gemm_host(h, wp.data(), 2 * F, H, w);
    if (rc) return rc;
    rc = dev_alloc_t(h, b, bp.size());
    if (rc) return rc;
    HIP_TRY(h, copy_blocking(h, *b, bp.data(), bp.size() * sizeof(float), hipMemcpyHostToDevice));
    return ASR_OK;
}

// ---- workspaces -------------------------------------------------------------------------------
int ensure_encoder_rows(asr_handle* h, int n, size_t rows);
int ensure_encoder_capacity(asr_handle* h, int n, int t) { return ensure_encoder_rows(h, n, (size_t)n * t); }
int ensure_encoder_rows(asr_handle* h, int n, size_t rows)
{
    if (rows <= h->cap_rows && n <= h->cap_n) return ASR_OK;
    const size_t nrows = std::max(rows, h->cap_rows);
    const int nn = std::max(n, h->cap_n);
    float** bufs[] = {&h->xin, &h->x0, &h->x1, &h->x2, &h->x3, &h->qkv, &h->hid};
    for (auto b : bufs) { dev_free(h, *b); *b = nullptr; }
    dev_free(h, h->pad); dev_free(h, h->pad2); dev_free(h, h->norm_scratch);
    h->pad = h->pad2 = nullptr; h->norm_scratch = nullptr;
    for (auto p : h->cross_k) dev_free(h, p);
    for (auto p : h->cross_v) dev_free(h, p);
    h->cross_k.assign(h->L, nullptr);
    h->cross_v.assign(h->L, nullptr);
    const size_t H = h->H;
    int rc = 0;
    rc |= dev_alloc_t(h, &h->xin, nrows * (size_t)h->D);
    rc |= dev_alloc_t(h, &h->x0, nrows * H);
    rc |= dev_alloc_t(h, &h->x1, nrows * H);
    rc |= dev_alloc_t(h, &h->x2, nrows * H);
    rc |= dev_alloc_t(h, &h->x3, nrows * H);
    rc |= dev_alloc_t(h, &h->qkv, nrows * 3 * H);
    rc |= dev_alloc_t(h, &h->hid, nrows * (size_t)h->F);
    rc |= dev_alloc_t(h, &h->pad, nrows);
    rc |= dev_alloc_t(h, &h->pad2, nrows + ASR_XATT_SLACK_ROWS);
    rc |= dev_alloc_t(h, &h->norm_scratch, input_norm_scratch_doubles(nn, 0, 0));
    for (int l = 0; l < h->L && !rc; ++l) {
        const size_t kv_floats = (nrows * H + ASR_XATT_SLACK_ROWS * 64) / (h->kv_bf16 ? 2 : 1);      // bf16: two values a float
        rc |= dev_alloc_t(h, &h->cross_k[l], kv_floats);
        rc |= dev_alloc_t(h, &h->cross_v[l], kv_floats);
    }
    if (rc) return ASR_ERR_HIP;
    h->cap_rows = nrows; h->cap_n = nn;
    return ASR_OK;
}

int decode_splits(const asr_handle* h, int R, int* s_qkv, int* s_proj, int* s_ffn2)
{
    *s_qkv = gemm_pick_split_k(R, 3 * h->H, h->H, gemm_nprod(h, h->H));
    *s_proj = gemm_pick_split_k(R, h->H, h->H, gemm_nprod(h, h->H));
    *s_ffn2 = gemm_pick_split_k(R, h->H, h->F, gemm_nprod(h, h->F));
    // Other handles' kernels fill the chip (asr_config.shared_gpu): what counts then is bytes, not how well one kernel covers
    // 256 CUs alone, and every K-slice is one more slab written and read.  Measured with four handles on 64-utterance batches
    // (ms per batch): 2,2,8 (the values above) 212.3; 1,1,1 219.4; 1,1,2 204.8; 1,1,4 205.3; 1,2,4 206.5; 2,2,4 208.4; 1,1,8 208.8.
    // Ten-utterance batches lose with fewer slices (1377 -> 1160 audio-s/s): only for whole-batch row counts.
    // One-product mode (bf16), same sweep: 1,1,2 125.9; 1,1,4 122.2; 1,2,4 123.7; 2,2,4 126.0; 2,2,8 128.9; 1,1,1 132.0.
    // Round 3, two whole batches per call (1280 rows), bf16: 1,1,2 103.5 ms per step; 1,1,4 105.3; 1,1,1 104.2 - two slices in every mode
    // (three-product mode at 1280 rows: 1,1,2 187.5; 1,1,1 187.9; 1,1,4 189.9).
    if (h->shared_gpu && R >= whole_batch_rows()) { *s_qkv = 1; *s_proj = 1; *s_ffn2 = 2; }
    if (const char* e = getenv("ASR_AMD_SPLITS")) {                  // development: "qkv,proj,ffn2"
        int a = 0, b = 0, c = 0;
        if (sscanf(e, "%d,%d,%d", &a, &b, &c) == 3 && a >= 1 && b >= 1 && c >= 1 && a <= ASR_MAX_SPLITK && b <= ASR_MAX_SPLITK &&
            c <= ASR_MAX_SPLITK) { *s_qkv = a; *s_proj = b; *s_ffn2 = c; }
    }
    return 0;
}

// K-slices of the logits GEMM for R beam rows (their slabs are summed by the soft-max / top-k kernel): at most two.  Handles that
// share the GPU run whole-batch row counts unsplit like the other projections (every slab is written and read once more, and
// the XCD partition of gemm_split.hip already keeps the weight reads to one XCD each); ASR_AMD_LOGIT_SPLIT pins it (development).
int logit_split_for(const asr_handle* h, int R)
{
    if (const char* e = getenv("ASR_AMD_LOGIT_SPLIT")) { const int v = atoi(e); if (v == 1 || v == 2) return v; }
    if (h->shared_gpu && R >= whole_batch_rows()) return h->logit_split_shared;
    return std::min(2, gemm_pick_split_k(R, h->V, h->H, gemm_nprod(h, h->H)));
}

int ensure_decoder_capacity(asr_handle* h, int n)
{
    if (n <= h->cap_dec_n) return ASR_OK;
    const size_t R = (size_t)n * h->K, H = h->H;
    const int width = h->cfg.max_target_length + 2;
    float** bufs[] = {&h->y0, &h->z1, &h->z2, &h->dctx, &h->part, &h->dhid, &h->logits, &h->cand_scores};
    for (auto b : bufs) { dev_free(h, *b); *b = nullptr; }
    dev_free(h, h->cand_tokens); h->cand_tokens = nullptr;
    for (auto p : h->kcache) dev_free(h, p);
    for (auto p : h->vcache) dev_free(h, p);
    h->kcache.assign(h->L, nullptr);
    h->vcache.assign(h->L, nullptr);
    void* bs[] = {h->beam.scores[0], h->beam.scores[1], h->beam.finished[0], h->beam.finished[1], h->beam.preds[0],
                  h->beam.preds[1], h->beam.anc[0], h->beam.anc[1], h->beam.pos, h->beam.tokens, h->beam.parents,
                  h->beam.live, h->beam.live_cnt};
    for (auto p : bs) dev_free(h, p);
    h->beam = BeamState{};

    int rc = 0;
    rc |= dev_alloc_t(h, &h->y0, R * H);
    rc |= dev_alloc_t(h, &h->z1, R * H);
    rc |= dev_alloc_t(h, &h->z2, R * H);
    rc |= dev_alloc_t(h, &h->dctx, R * H);
    rc |= dev_alloc_t(h, &h->part, (size_t)ASR_MAX_SPLITK * R * 3 * H);
    rc |= dev_alloc_t(h, &h->dhid, R * (size_t)h->F);
    h->logit_split = logit_split_for(h, (int)R);                                                          // <= 2 slabs of logits
    rc |= dev_alloc_t(h, &h->logits, 2 * R * (size_t)h->V);
    rc |= dev_alloc_t(h, &h->cand_scores, R * (size_t)h->K);
    rc |= dev_alloc_t(h, &h->cand_tokens, R * (size_t)h->K);
    for (int l = 0; l < h->L && !rc; ++l) {
        rc |= dev_alloc_t(h, &h->kcache[l], R * width * H / (h->kv_bf16 ? 2 : 1));
        rc |= dev_alloc_t(h, &h->vcache[l], R * width * H / (h->kv_bf16 ? 2 : 1));
    }
    for (int i = 0; i < 2 && !rc; ++i) {
        rc |= dev_alloc_t(h, &h->beam.scores[i], R);
        rc |= dev_alloc_t(h, &h->beam.finished[i], R);
        rc |= dev_alloc_t(h, &h->beam.preds[i], R * width);
        rc |= dev_alloc_t(h, &h->beam.anc[i], R * width);
    }
    rc |= dev_alloc_t(h, &h->beam.pos, 16);              // pos / done / unfinished of up to MAX_VIEWS sub-batches, 4 ints each
    rc |= dev_alloc_t(h, &h->beam.tokens, R);
    rc |= dev_alloc_t(h, &h->beam.parents, R);
    rc |= dev_alloc_t(h, &h->beam.live, R * width);
    rc |= dev_alloc_t(h, &h->beam.live_cnt, (size_t)n);
    if (rc) return ASR_ERR_HIP;
    h->beam.done = h->beam.pos + 1;
    h->beam.unfinished = h->beam.pos + 2;
    h->beam.width = width;
    h->cap_dec_n = n;
    return ASR_OK;
}

// ---- encoder (model.py:444-490) ----------------------------------------------------------------
// X_dev [n, t, D] -> h->x0 [n*t, H] (encoder output), h->pad / h->pad2 [n*t]
// Groups of utterances padded to different T, decoded as ONE beam search (asr_decode_groups): X_dev holds group after group.
struct Groups {
    int count = 0;
    const int32_t* n = nullptr;        // host [count]
    const int32_t* t = nullptr;        // host [count]
    const int32_t *d_t = nullptr, *d_off = nullptr, *d_limit = nullptr;     // device [sum n]: per utterance
    int t_max = 0;
    size_t rows = 0;                   // sum n[g] * t[g]
};

// With `gr`: the rows of all groups go through the row-wise kernels (GEMMs, residual + layer norm, padding flags) together;
// what depends on a group's own T - the input layer norm over (T, H) (model.py:453), the attention over its own keys - is
// launched group by group on that group's rows.  (n, t) are then unused.
int run_encoder(asr_handle* h, const float* X_dev, int n, int t, const Groups* gr = nullptr)
{
    const int M = gr ? (int)gr->rows : n * t, H = h->H, F = h->F;
    int32_t* pad2_dst = h->pad2;
    if (gr) t = gr->t_max;
    int rc = ensure_pe(h, std::max(t, h->cfg.max_target_length + 2));
    if (rc) return rc;
    hipStream_t s = h->stream;
    {
        ProfScope ps(h, "pad_mask", 0, 4.0 * M * (h->D + 1));
        HIP_TRY(h, launch_pad_mask(X_dev, M, h->D, h->pad, s));
    }
    rc = gemm(h, X_dev, h->w_src, h->b_src, h->x1, M, H, h->D, EPI_BIAS, 1);                        // :451
    if (rc) return rc;
    {
        ProfScope ps(h, "input_norm_timing", 0, 4.0 * M * H * 4.0);
        if (gr) {
            size_t row0 = 0;
            for (int g = 0; g < gr->count; ++g) {
                HIP_TRY(h, launch_input_norm_timing(h->x1 + row0 * H, h->in_gamma, h->in_beta, h->pe, gr->n[g], gr->t[g], H, h->norm_scratch,
                                                    h->x0 + row0 * H, s));
                row0 += (size_t)gr->n[g] * gr->t[g];
            }
        } else {
            HIP_TRY(h, launch_input_norm_timing(h->x1, h->in_gamma, h->in_beta, h->pe, n, t, H, h->norm_scratch, h->x0, s));   // :453,456
        }
    }
    for (int l = 0; l < h->L; ++l) {
        const EncBlock& b = h->enc[l];
        const bool last = (l == h->L - 1);
        rc = gemm(h, h->x0, b.wqkv, b.bqkv, h->qkv, M, 3 * H, H, EPI_BIAS, 1);                      // utils.py:612
        if (rc) return rc;
        {
            double tt = (double)n * t * t;
            if (gr) { tt = 0.0; for (int g = 0; g < gr->count; ++g) tt += (double)gr->n[g] * gr->t[g] * gr->t[g]; }
            ProfScope ps(h, "encoder_attention", 4.0 * tt * H, 4.0 * M * 4.0 * H);
            if (gr) {
                size_t row0 = 0;
                for (int g = 0; g < gr->count; ++g) {
                    HIP_TRY(h, launch_encoder_attention(h->qkv + row0 * 3 * H, h->pad + row0, gr->n[g], gr->t[g], h->heads, h->x1 + row0 * H, mha_mode(h), h->range_flag, s));
                    row0 += (size_t)gr->n[g] * gr->t[g];
                }
            } else {
                HIP_TRY(h, launch_encoder_attention(h->qkv, h->pad, n, t, h->heads, h->x1, mha_mode(h), h->range_flag, s));     // utils.py:624-631
            }
        }
        rc = gemm(h, h->x1, b.wo, nullptr, h->x2, M, H, H, EPI_PARTIAL, 1);                         // utils.py:632
        if (rc) return rc;
        {
            ProfScope ps(h, "add_layer_norm", 0, 4.0 * M * H * 3.0);
            HIP_TRY(h, launch_add_layer_norm(h->x0, h->x2, 1, 0, b.bo, b.ln0s, b.ln0b, nullptr, nullptr, M, H, h->x3, s));   // model.py:466
        }
        rc = gemm(h, h->x3, b.w1, b.b1, h->hid, M, h->glu ? 2 * F : F, H, h->glu ? EPI_GLU : h->ff_epi, 1);   // utils.py:566
        if (rc) return rc;
        rc = gemm(h, h->hid, b.w2, nullptr, h->x2, M, H, F, EPI_PARTIAL, 1);                        // utils.py:567
        if (rc) return rc;
        {
            ProfScope ps(h, "add_layer_norm", 0, 4.0 * M * H * 3.0);
            HIP_TRY(h, launch_add_layer_norm(h->x3, h->x2, 1, 0, b.b2, b.ln1s, b.ln1b, last ? h->pad : nullptr,
                                             last ? pad2_dst : nullptr, M, H, h->x0, s));           // model.py:481,489
        }
    }
    return ASR_OK;
}

// cross-attention K/V of every decoder block, once per utterance (instead of once per step per beam)
int run_cross_kv(asr_handle* h, int n, int t, const Groups* gr = nullptr)
{
    const int M = gr ? (int)gr->rows : n * t, H = h->H;
    const size_t esz = h->kv_bf16 ? 2 : 4;
    for (int l = 0; l < h->L; ++l) {
        int rc = gemm(h, h->x0, h->dec[l].wkv, h->dec[l].bkv, h->qkv, M, 2 * H, H, EPI_BIAS, 1);   // utils.py:618
        if (rc) return rc;
        ProfScope ps(h, "pack_cross_kv", 0, 4.0 * M * 4.0 * H);
        int32_t* rf = h->nprod_active == 13 ? h->range_flag : nullptr;
        if (gr) {                                                     // every group's [n][heads][t][64] behind the groups before it
            size_t row0 = 0;
            for (int g = 0; g < gr->count; ++g) {
                HIP_TRY(h, launch_pack_cross_kv(h->qkv + row0 * 2 * H, gr->n[g], gr->t[g], h->heads,
                                                reinterpret_cast<char*>(h->cross_k[l]) + row0 * H * esz,
                                                reinterpret_cast<char*>(h->cross_v[l]) + row0 * H * esz, h->kv_bf16 ? 1 : 0, rf, h->stream));
                row0 += (size_t)gr->n[g] * gr->t[g];
            }
        } else {
            HIP_TRY(h, launch_pack_cross_kv(h->qkv, n, t, h->heads, h->cross_k[l], h->cross_v[l], h->kv_bf16 ? 1 : 0, rf, h->stream));
        }
    }
    return ASR_OK;
}

// A contiguous run of utterances of the batch that is beam-searched on its own stream with its own loop state:
// every buffer of the handle indexed by row or utterance, offset to the run's first one.
struct DecView {
    int n0 = 0, n = 0, idx = 0;
    hipStream_t stream = nullptr;
    float *y0, *z1, *z2, *dctx, *part, *dhid, *logits, *cand_scores;
    int32_t* cand_tokens;
    const int32_t* pad2;
    size_t cache_off = 0, cross_off = 0;
    BeamState beam{};
    int32_t* done_host = nullptr;
    hipEvent_t* events = nullptr;
};

DecView make_view(asr_handle* h, int idx, int n0, int nv, int t, hipStream_t stream)
{
    const size_t K = h->K, H = h->H, r0 = (size_t)n0 * K, width = h->beam.width;
    DecView v;
    v.n0 = n0; v.n = nv; v.idx = idx; v.stream = stream;
    v.y0 = h->y0 + r0 * H; v.z1 = h->z1 + r0 * H; v.z2 = h->z2 + r0 * H; v.dctx = h->dctx + r0 * H;
    v.part = h->part + (size_t)ASR_MAX_SPLITK * r0 * 3 * H;          // slabs of a view are contiguous, stride = its own rows
    v.dhid = h->dhid + r0 * (size_t)h->F;
    v.logits = h->logits + 2 * r0 * (size_t)h->V;
    v.cand_scores = h->cand_scores + r0 * K;
    v.cand_tokens = h->cand_tokens + r0 * K;
    v.pad2 = h->pad2 + (size_t)n0 * t;
    v.cache_off = r0 * width * H;                                    // [u][heads][width][K][64]
    v.cross_off = (size_t)n0 * t * H;                                // [u][heads][t][64]
    v.beam = h->beam;
    for (int i = 0; i < 2; ++i) {
        v.beam.scores[i] += r0; v.beam.finished[i] += r0; v.beam.preds[i] += r0 * width; v.beam.anc[i] += r0 * width;
    }
    v.beam.live += r0 * width; v.beam.live_cnt += n0;
    v.beam.tokens += r0; v.beam.parents += r0;
    v.beam.pos = h->beam.pos + 4 * idx; v.beam.done = v.beam.pos + 1; v.beam.unfinished = v.beam.pos + 2;
    v.done_host = h->done_host + (size_t)idx * (h->cfg.max_target_length + 8);
    v.events = h->step_events.data() + 8 * idx;
    return v;
}

// One decode step (model.py:270-303 with decoder_with_caching_impl :559-633 restated on a K/V cache), in pieces: head
// (embedding), per block an attention half and a feed-forward half, tail (logits, soft-max/top-k, pruning).
struct StepCtx {
    int n, R, s_qkv, s_proj, s_ffn2, step;
    size_t RH;
};

StepCtx step_ctx(const asr_handle* h, const DecView& v)
{
    StepCtx c;
    c.n = v.n; c.R = v.n * h->K; c.RH = (size_t)c.R * h->H;
    decode_splits(h, c.R, &c.s_qkv, &c.s_proj, &c.s_ffn2);
    return c;
}

int step_head(asr_handle* h, const DecView& v, const StepCtx& c)
{
    const float mult = h->cfg.scale_embedding ? (float)sqrt((double)h->H) : 1.0f;
    const BeamState& st = v.beam;
    ProfScope ps(h, "embed_pe", 0, 4.0 * c.R * h->H * 3.0, v.stream);
    HIP_TRY(h, launch_embed_pe(h->emb, st.preds[0], st.preds[1], st.width, st.pos, h->pe, mult, c.R, h->H, v.y0, st.done, v.stream));
    return ASR_OK;
}

// self-attention + cross-attention sub-layers of block l (model.py:588-616): y0 -> z2
int step_attention_half(asr_handle* h, const DecView& v, const StepCtx& c, int l, int t)
{
    const int n = c.n, R = c.R, H = h->H, K = h->K;
    const size_t RH = c.RH;
    hipStream_t s = v.stream;
    const BeamState& st = v.beam;
    const DecBlock& b = h->dec[l];
    int rc = gemm(h, v.y0, b.wqkv, nullptr, v.part, R, 3 * H, H, EPI_PARTIAL, c.s_qkv, s);
    if (rc) return rc;
    {
        SelfAttnArgs a{};
        a.qkv = v.part; a.nsplit = c.s_qkv; a.split_stride = 3 * RH; a.bias = b.bqkv;
        const size_t esz = h->kv_bf16 ? 2 : 4;                       // bytes per cached value
        a.kcache = reinterpret_cast<char*>(h->kcache[l]) + v.cache_off * esz; a.vcache = reinterpret_cast<char*>(h->vcache[l]) + v.cache_off * esz;
        a.kv_bf16 = h->kv_bf16 ? 1 : 0;
        a.f16x3 = (h->nprod_active == 13 && !h->kv_bf16 && !self_exact()) ? 1 : 0;
        a.range_flag = a.f16x3 ? h->range_flag : nullptr;
        a.anc0 = st.anc[0]; a.anc1 = st.anc[1]; a.live = st.live; a.live_cnt = st.live_cnt; a.pos = st.pos; a.done = st.done;
        a.ctx = v.dctx; a.b = n; a.k = K; a.heads = h->heads; a.width = st.width;
        a.lds_stride = std::min(st.width, st.limit + 2);
        // bytes here: the q/k/v slabs in, the new K/V rows and the context out; the history it streams (the utterances'
        // LIVE rows) is added by decode_core from the live counts of the steps that ran
        ProfScope ps(h, "decoder_self_attention", 0, 4.0 * R * 3.0 * H * c.s_qkv + 2.0 * R * H * (double)esz + 4.0 * R * H, s);
        for (int rep = launches_of(h, "self"); rep > 0; --rep) HIP_TRY(h, launch_decoder_self_attention(a, s));
    }
    rc = gemm(h, v.dctx, b.wo, nullptr, v.part, R, H, H, EPI_PARTIAL, c.s_proj, s);
    if (rc) return rc;
    {
        ProfScope ps(h, "add_layer_norm(dec)", 0, 4.0 * R * H * (2.0 + c.s_proj), s);
        for (int rep = launches_of(h, "ln"); rep > 0; --rep) HIP_TRY(h, launch_add_layer_norm_done(v.y0, v.part, c.s_proj, RH, b.bo, b.ln0s, b.ln0b, nullptr, nullptr, R, H,
                                              v.z1, st.done, s));
    }
    rc = gemm(h, v.z1, b.wq, nullptr, v.part, R, H, H, EPI_PARTIAL, c.s_proj, s);
    if (rc) return rc;
    {
        CrossAttnArgs a{};
        a.qpart = v.part; a.nsplit = c.s_proj; a.split_stride = RH; a.qbias = b.bq;
        const size_t esz = h->kv_bf16 ? 2 : 4;
        a.kc = reinterpret_cast<const char*>(h->cross_k[l]) + v.cross_off * esz; a.v = reinterpret_cast<const char*>(h->cross_v[l]) + v.cross_off * esz;
        a.kv_bf16 = h->kv_bf16 ? 1 : 0;
        // default mode: the attention products on the fp16 matrix pipe like the GEMMs' (three per multiply); a repeated call
        // (nprod_active 6) and the other modes keep the exact-f32 matrix instruction
        a.f16x3 = (h->nprod_active == 13 && !h->kv_bf16) ? 1 : 0;
        a.range_flag = a.f16x3 ? h->range_flag : nullptr;
        a.pad2 = v.pad2; a.done = st.done;
        a.ctx = v.dctx; a.b = n; a.k = K; a.heads = h->heads; a.t = t;
        a.t_arr = h->grp_t; a.row_off = h->grp_off;
        const double keys = h->grp_t ? h->grp_rows : (double)n * t;                       // keys of all utterances of the view
        ProfScope ps(h, "decoder_cross_attention", 4.0 * K * keys * H, (h->kv_bf16 ? 2.0 : 4.0) * 2.0 * keys * H, s);
        for (int rep = launches_of(h, "cross"); rep > 0; --rep) HIP_TRY(h, launch_decoder_cross_attention(a, s));
    }
    rc = gemm(h, v.dctx, b.wco, nullptr, v.part, R, H, H, EPI_PARTIAL, c.s_proj, s);
    if (rc) return rc;
    {
        ProfScope ps(h, "add_layer_norm(dec)", 0, 4.0 * R * H * (2.0 + c.s_proj), s);
        for (int rep = launches_of(h, "ln"); rep > 0; --rep) HIP_TRY(h, launch_add_layer_norm_done(v.z1, v.part, c.s_proj, RH, b.bco, b.ln1s, b.ln1b, nullptr, nullptr, R, H,
                                              v.z2, st.done, s));
    }
    return ASR_OK;
}

// feed-forward sub-layer of block l (model.py:619-627): z2 -> y0
int step_ffn_half(asr_handle* h, const DecView& v, const StepCtx& c, int l)
{
    const int R = c.R, H = h->H, F = h->F;
    hipStream_t s = v.stream;
    const DecBlock& b = h->dec[l];
    int rc = gemm(h, v.z2, b.w1, b.b1, v.dhid, R, h->glu ? 2 * F : F, H, h->glu ? EPI_GLU : h->ff_epi, 1, s);
    if (rc) return rc;
    rc = gemm(h, v.dhid, b.w2, nullptr, v.part, R, H, F, EPI_PARTIAL, c.s_ffn2, s);
    if (rc) return rc;
    ProfScope ps(h, "add_layer_norm(dec)", 0, 4.0 * R * H * (2.0 + c.s_ffn2), s);
    for (int rep = launches_of(h, "ln"); rep > 0; --rep) HIP_TRY(h, launch_add_layer_norm_done(v.z2, v.part, c.s_ffn2, c.RH, b.b2, b.ln2s, b.ln2b, nullptr, nullptr, R, H,
                                          v.y0, v.beam.done, s));
    return ASR_OK;
}

int step_tail(asr_handle* h, const DecView& v, const StepCtx& c)
{
    const int R = c.R, H = h->H, K = h->K;
    hipStream_t s = v.stream;
    const BeamState& st = v.beam;
    const float* wout = h->cfg.tie_embedding_and_softmax ? h->emb_gemm : h->softmax_w;
    const int s_log = logit_split_for(h, R);                                                                 // <= 2 slabs of logits
    int rc = gemm(h, v.y0, wout, nullptr, v.logits, R, h->V, H, EPI_PARTIAL, s_log, s);             // model.py:341 (no bias)
    if (rc) return rc;
    {
        ProfScope ps(h, "log_softmax_topk", 0, 4.0 * R * (double)h->V * s_log, s);
        for (int rep = launches_of(h, "topk"); rep > 0; --rep)
            HIP_TRY(h, launch_log_softmax_topk(v.logits, s_log, (size_t)R * h->V, R, h->V, K, v.cand_scores, v.cand_tokens, st.done, s));   // :345-346
    }
    {
        ProfScope ps(h, "beam_step", 0, 4.0 * R * H * 3.0, s);          // embedding row + timing row in, next decoder input out
        const float mult = h->cfg.scale_embedding ? (float)sqrt((double)h->H) : 1.0f;
        HIP_TRY(h, launch_beam_step(st, v.cand_scores, v.cand_tokens, c.n, K, h->emb, h->pe, mult, H, v.y0, s));   // :280-301, :569-576
    }
    return ASR_OK;
}

int run_view_step(asr_handle* h, const DecView& v, int t, int step)
{
    StepCtx c = step_ctx(h, v);
    c.step = step;
    if (h->profile && h->live_host && (size_t)(step + 1) * h->live_host_n <= h->live_host_cap)
        HIP_TRY(h, hipMemcpyAsync(h->live_host + (size_t)step * h->live_host_n + v.n0, v.beam.live_cnt, (size_t)v.n * sizeof(int32_t),
                                  hipMemcpyDeviceToHost, v.stream));
    int rc = step == 1 ? step_head(h, v, c) : ASR_OK;               // later steps: beam_step_kernel wrote the decoder input
    if (rc) return rc;
    for (int l = 0; l < h->L; ++l) {
        if ((rc = step_attention_half(h, v, c, l, t))) return rc;
        if ((rc = step_ffn_half(h, v, c, l))) return rc;
    }
    return step_tail(h, v, c);
}

// Steps 2.. of a view launch the same kernels with the same arguments (the step index, the double-buffer parity and the
// loop state live on the device), so the step is captured once per call into a HIP graph and replayed: one host call
// per step and view instead of 70, and the queue holds the whole step when its first kernel starts.
int capture_view_step(asr_handle* h, const DecView& v, int t, hipGraphExec_t* out)
{
    // One capture at a time in the process, and in the mode that leaves other threads' calls alone: other handles (other
    // host threads) go on allocating, copying and synchronising on their own streams while this one records its step.
    static std::mutex capture_mu;
    std::lock_guard<std::mutex> lock(capture_mu);
    HIP_TRY(h, hipStreamBeginCapture(v.stream, hipStreamCaptureModeRelaxed));
    const int rc = run_view_step(h, v, t, 2);
    hipGraph_t g = nullptr;
    const hipError_t e = hipStreamEndCapture(v.stream, &g);
    if (rc || e != hipSuccess) {
        if (g) (void)hipGraphDestroy(g);
        return rc ? rc : fail(h, ASR_ERR_HIP, std::string("hipStreamEndCapture: ") + hipGetErrorString(e));
    }
    const hipError_t e2 = hipGraphInstantiate(out, g, nullptr, nullptr, 0);
    (void)hipGraphDestroy(g);
    if (e2 != hipSuccess) return fail(h, ASR_ERR_HIP, std::string("hipGraphInstantiate: ") + hipGetErrorString(e2));
    return ASR_OK;
}

struct StepGraphs {                                                  // one per view, destroyed when the call returns
    hipGraphExec_t g[MAX_VIEWS] = {nullptr, nullptr, nullptr, nullptr};
    bool disabled = false;                                           // a capture failed: direct launches for the rest of the call
    ~StepGraphs() { for (auto x : g) if (x) (void)hipGraphExecDestroy(x); }
};

// One step of every active view.  Two views run free of each other on their two streams: what was measured
// (rocprofv3 kernel trace of both queues) is that two kernels that share the CUs each take about the sum of their solo
// times - also an HBM-bound attention kernel beside a matrix-bound GEMM - so forcing the views half a block apart with
// events (tried: -12 %) buys nothing; the gain of two views (+3.3 %) is the launch gaps and tails they fill for each other.
int run_decode_step(asr_handle* h, DecView* views, const bool* active, int nviews, int t, int step, StepGraphs* graphs)
{
    for (int vi = 0; vi < nviews; ++vi) {
        if (!active[vi]) continue;
        const DecView& v = views[vi];
        if (graphs && !graphs->disabled && step >= 2) {
            if (!graphs->g[vi] && capture_view_step(h, v, t, &graphs->g[vi]) != ASR_OK) {
                graphs->g[vi] = nullptr;
                graphs->disabled = true;                             // (a real launch error shows again below)
                (void)hipGetLastError();
            }
            if (graphs->g[vi]) {
                HIP_TRY(h, hipGraphLaunch(graphs->g[vi], v.stream));
                continue;
            }
        }
        const int rc = run_view_step(h, v, t, step);
        if (rc) return rc;
    }
    return ASR_OK;
}

// `len` = steps this run of utterances took, `ylen` >= len = row length of Y (columns len.. are padded with 3: what
// further steps of a finished search append)
void finalize_host(const int32_t* preds, const float* scores, int n, int K, int width, int len, float alpha, int32_t* Y, int ylen)
{
    for (int u = 0; u < n; ++u) {
        int best = 0;
        float bestv = -INFINITY;
        for (int k = 0; k < K; ++k) {
            const int32_t* p = preds + (size_t)(u * K + k) * width;
            int cnt = 0;
            for (int j = 0; j <= len; ++j) cnt += (p[j] != 3);
            const float lp = powf((5.0f + (float)cnt) / 6.0f, alpha);
            const float v = scores[u * K + k] / lp;
            if (k == 0 || v > bestv) { bestv = v; best = k; }
        }
        const int32_t* p = preds + (size_t)(u * K + best) * width;
        for (int j = 0; j < len; ++j) Y[(size_t)u * ylen + j] = p[1 + j];
        for (int j = len; j < ylen; ++j) Y[(size_t)u * ylen + j] = 3;
    }
}

struct TraceOut { int steps = 0; float* logits = nullptr; float* scores = nullptr; int32_t* tokens = nullptr; int32_t* parents = nullptr; };

// X_dev [n,t,D] on device (already stacked) -> Y host
int decode_core(asr_handle* h, const float* X_dev, int n, int t, int32_t* Y, int64_t y_capacity, int32_t* len_out,
                const TraceOut* tr, const Groups* gr = nullptr)
{
    struct GroupScope {                // the handle's per-call group state never outlives the call
        asr_handle* h;
        ~GroupScope() { h->grp_t = h->grp_off = nullptr; h->grp_rows = 0.0; h->beam.limit_u = nullptr; }
    } group_scope{h};
    if (!h->finalized) return fail(h, ASR_ERR_STATE, "asr_finalize_weights has not succeeded on this handle");
    if (n == 0) { *len_out = 0; return ASR_OK; }                                                    // model.py:184-187
    int rc = ensure_decoder_capacity(h, n);
    if (rc) return rc;
    for (int rep = launches_of(h, "encoder"); rep > 0; --rep) {     // (encoder + cross K/V of the batch: idempotent as a whole)
        // with groups: every group keeps ITS T wherever T is part of the arithmetic, its cross K / V and padding flags are laid
        // out behind the groups before it
        rc = run_encoder(h, X_dev, n, t, gr);
        if (rc) return rc;
        rc = run_cross_kv(h, n, t, gr);
        if (rc) return rc;
    }
    const int K = h->K, R = n * K;
    if (gr) {
        t = gr->t_max;                                              // the joint loop runs as long as the longest group's
        h->grp_t = gr->d_t; h->grp_off = gr->d_off; h->grp_rows = (double)gr->rows;
        h->beam.limit_u = gr->d_limit;
    }
    h->beam.limit = std::min(t + 50, (int)h->cfg.max_target_length);                                // :310 (Q7)
    const int max_steps = h->beam.limit + 1;
    if (h->profile && !tr) {
        const size_t need = (size_t)(max_steps + 2) * n;
        if (need > h->live_host_cap) {
            if (h->live_host) (void)hipHostFree(h->live_host);
            h->live_host = nullptr; h->live_host_cap = 0;
            HIP_TRY(h, hipHostMalloc(reinterpret_cast<void**>(&h->live_host), need * sizeof(int32_t), 0));
            h->live_host_cap = need;
        }
        h->live_host_n = n;
    } else {
        h->live_host_n = 0;
    }
    // Utterances are independent, so the search may run as two halves with their own loop state on two streams
    // (kernels of one half fill the launch gaps and tails of the other's).  The joint loop of the reference ends
    // when every utterance has finished: a half that ends earlier is padded with 3, which is what further steps
    // append to finished beams (model.py:253) without changing their order or scores.
    int nviews = h->sub_batches >= 2 ? std::min(h->sub_batches, n) : (h->sub_batches == 0 && R >= 320 ? 2 : 1);   // auto: each half still fills the GPU
    if (tr || gr) nviews = 1;                       // (profile mode keeps the parts: its brackets time the shapes the timed passes launch)
    DecView views[MAX_VIEWS];
    for (int vi = 0, n0 = 0; vi < nviews; ++vi) {   // the first n % nviews parts get one utterance more
        const int nv = n / nviews + (vi < n % nviews ? 1 : 0);
        if (vi > 0 && !h->xstream[vi - 1]) HIP_TRY(h, hipStreamCreateWithFlags(&h->xstream[vi - 1], hipStreamNonBlocking));
        views[vi] = make_view(h, vi, n0, nv, t, vi == 0 ? h->stream : h->xstream[vi - 1]);
        n0 += nv;
    }
    if (nviews > 1) {
        HIP_TRY(h, hipEventRecord(h->fork_ev, h->stream));                                          // encoder + cross K/V done
        for (int vi = 1; vi < nviews; ++vi) HIP_TRY(h, hipStreamWaitEvent(views[vi].stream, h->fork_ev, 0));
    }
    for (int v = 0; v < nviews; ++v) HIP_TRY(h, launch_beam_init(views[v].beam, views[v].n, K, views[v].stream));
    constexpr int LOOKAHEAD = 3;
    StepGraphs graphs;
    const bool use_graph = (h->use_graph < 0 ? R >= 320 : h->use_graph != 0) && !h->profile && !tr;
    bool ended[MAX_VIEWS];
    for (int vi = 0; vi < MAX_VIEWS; ++vi) ended[vi] = vi >= nviews;
    auto all_ended = [&]() { for (int vi = 0; vi < nviews; ++vi) if (!ended[vi]) return false; return true; };
    for (int s = 1; s <= max_steps && !all_ended(); ++s) {
        bool active[MAX_VIEWS];
        for (int vi = 0; vi < MAX_VIEWS; ++vi) active[vi] = !ended[vi];
        rc = run_decode_step(h, views, active, nviews, t, s, use_graph ? &graphs : nullptr);
        if (rc) return rc;
        if (tr && s <= tr->steps) {
            const int buf = s & 1;
            HIP_TRY(h, hipStreamSynchronize(h->stream));
            int32_t posd[2];
            HIP_TRY(h, copy_blocking(h, posd, h->beam.pos, sizeof(posd), hipMemcpyDeviceToHost));
            if (posd[0] == s) {                                                                     // the step really ran
                if (tr->logits) {
                    float* dst = tr->logits + (size_t)(s - 1) * R * h->V;
                    const size_t cnt = (size_t)R * h->V;
                    HIP_TRY(h, copy_blocking(h, dst, h->logits, cnt * 4, hipMemcpyDeviceToHost));
                    if (logit_split_for(h, R) > 1) {            // second K slice, added in slab order like the top-k kernel does
                        std::vector<float> slab(cnt);
                        HIP_TRY(h, copy_blocking(h, slab.data(), h->logits + cnt, cnt * 4, hipMemcpyDeviceToHost));
                        for (size_t i = 0; i < cnt; ++i) dst[i] += slab[i];
                    }
                }
                if (tr->scores) HIP_TRY(h, copy_blocking(h, tr->scores + (size_t)(s - 1) * R, h->beam.scores[buf], (size_t)R * 4, hipMemcpyDeviceToHost));
                if (tr->tokens) HIP_TRY(h, copy_blocking(h, tr->tokens + (size_t)(s - 1) * R, h->beam.tokens, (size_t)R * 4, hipMemcpyDeviceToHost));
                if (tr->parents) HIP_TRY(h, copy_blocking(h, tr->parents + (size_t)(s - 1) * R, h->beam.parents, (size_t)R * 4, hipMemcpyDeviceToHost));
            }
        }
        for (int vi = 0; vi < nviews; ++vi) {
            DecView& v = views[vi];
            if (!active[vi]) continue;
            HIP_TRY(h, hipMemcpyAsync(&v.done_host[s], v.beam.done, sizeof(int32_t), hipMemcpyDeviceToHost, v.stream));
            HIP_TRY(h, hipEventRecord(v.events[s % 8], v.stream));
            if (s > LOOKAHEAD) {
                const int c = s - LOOKAHEAD;
                HIP_TRY(h, hipEventSynchronize(v.events[c % 8]));
                if (v.done_host[c]) ended[vi] = true;
            }
        }
        if (h->profile == 2) prof_drain(h, false);
    }
    int lens[MAX_VIEWS] = {0, 0, 0, 0};
    for (int vi = 0; vi < nviews; ++vi) {
        HIP_TRY(h, hipStreamSynchronize(views[vi].stream));
        int32_t posd[2] = {0, 0};
        HIP_TRY(h, copy_blocking(h, posd, views[vi].beam.pos, sizeof(posd), hipMemcpyDeviceToHost, views[vi].stream));
        lens[vi] = posd[0];
        if (!posd[1] || lens[vi] < 1 || lens[vi] > max_steps)
            return fail(h, ASR_ERR_HIP, "beam search loop ended in an inconsistent state");
    }
    if (h->profile == 2) prof_drain(h, true);
    if (h->profile && h->live_host_n == n) {                       // what self-attention streamed: the live rows of every step taken
        double live = 0.0;
        for (int vi = 0; vi < nviews; ++vi)
            for (int s = 1; s <= lens[vi]; ++s)
                for (int u = 0; u < views[vi].n; ++u) live += h->live_host[(size_t)s * n + views[vi].n0 + u];
        for (auto& pc : h->prof)
            if (strcmp(pc.name, "decoder_self_attention") == 0) {
                pc.bytes += h->L * live * 2.0 * h->H * (h->kv_bf16 ? 2.0 : 4.0);
                pc.flops += h->L * live * 4.0 * K * h->H;
            }
    }
    const int len = *std::max_element(lens, lens + MAX_VIEWS);
    if ((int64_t)n * len > y_capacity) return fail(h, ASR_ERR_CAPACITY, "Y too small: need n * " + std::to_string(len) + " int32");
    const int width = h->beam.width;
    for (int vi = 0; vi < nviews; ++vi) {
        const DecView& v = views[vi];
        const int buf = lens[vi] & 1, rv = v.n * K;
        std::vector<int32_t> preds((size_t)rv * width);
        std::vector<float> scores(rv);
        HIP_TRY(h, copy_blocking(h, preds.data(), v.beam.preds[buf], preds.size() * 4, hipMemcpyDeviceToHost, v.stream));
        HIP_TRY(h, copy_blocking(h, scores.data(), v.beam.scores[buf], scores.size() * 4, hipMemcpyDeviceToHost, v.stream));
        finalize_host(preds.data(), scores.data(), v.n, K, width, lens[vi], h->cfg.lp_alpha, Y + (size_t)v.n0 * len, len);
    }
    *len_out = len;
    return ASR_OK;
}

int check_xshape(asr_handle* h, int n, int t, int d)
{
    if (n < 0 || t < 0 || d != h->D) return fail(h, ASR_ERR_ARG, "X must be [n, t, input_dim=" + std::to_string(h->D) + "]");
    if (n > 0 && t < 1) return fail(h, ASR_ERR_ARG, "t must be >= 1");
    if (self_attention_lds_bytes(h->K, std::min(t + 50, (int)h->cfg.max_target_length) + 2) > 150 * 1024)
        return fail(h, ASR_ERR_ARG, "min(t + 50, max_target_length) * beam_size exceeds the self-attention LDS budget");
    return ASR_OK;
}

int set_device(asr_handle* h)
{
    HIP_TRY(h, hipSetDevice(h->cfg.device));
    return ASR_OK;
}

struct TmpBufs {
    std::vector<void*> p;
    ~TmpBufs() { for (void* q : p) (void)hipFree(q); }
    template <typename T>
    hipError_t up(T** d, const T* src, size_t count, hipStream_t s)
    {
        hipError_t e = hipMalloc(reinterpret_cast<void**>(d), std::max<size_t>(count * sizeof(T), 16));
        if (e != hipSuccess) return e;
        p.push_back(*d);
        if (src) e = hipMemcpyAsync(*d, src, count * sizeof(T), hipMemcpyHostToDevice, s);
        return e;
    }
    // a GEMM weight operand in the handle's precision mode (f32, or bf16 planes)
    int up_gemm(asr_handle* h, float** d, const float* w, int n, int k, hipStream_t s)
    {
        if (gemm_nprod(h, k) == 0) { HIP_TRY(h, up(d, w, (size_t)n * k, s)); return ASR_OK; }
        std::vector<uint16_t> planes(plane_elems(h, n, k));
        if (!pack_planes(h, w, n, k, planes.data())) h->weights_out_of_range = true;     // checked by the caller's retry wrapper
        uint16_t* dp = nullptr;
        HIP_TRY(h, up(&dp, planes.data(), planes.size(), s));
        HIP_TRY(h, hipStreamSynchronize(s));                   // `planes` is a local
        *d = reinterpret_cast<float*>(dp);
        return ASR_OK;
    }
};

// copies `in_count` floats up, runs `launch(din, dout)`, copies `out_count` floats back
template <typename F>
int fea_roundtrip(asr_handle* h, const float* in, size_t in_count, float* out, size_t out_count, F launch)
{
    TmpBufs tb;
    float *din = nullptr, *dout = nullptr;
    hipStream_t s = h->stream;
    HIP_TRY(h, tb.up(&din, in, in_count, s));
    HIP_TRY(h, tb.up(&dout, static_cast<const float*>(nullptr), out_count, s));
    HIP_TRY(h, launch(din, dout, tb, s));
    HIP_TRY(h, hipMemcpyAsync(out, dout, out_count * sizeof(float), hipMemcpyDeviceToHost, s));
    HIP_TRY(h, hipStreamSynchronize(s));
    return ASR_OK;
}

// fp16x3 mode: run a call; if one of its GEMMs met an activation (or, for the single-kernel probes, a weight) outside
// fp16's range, discard the result and repeat the whole call on the bf16x6 kernels (same accuracy, no range limit).
template <typename F>
int with_range_retry(asr_handle* h, F&& run)
{
    h->weights_out_of_range = false;
    int rc = run();
    if (rc != ASR_OK || h->nprod != 13 || h->nprod_active != 13) return rc;
    int32_t flag = 0;
    HIP_TRY(h, copy_blocking(h, &flag, h->range_flag, sizeof(flag), hipMemcpyDeviceToHost));
    if (!flag && !h->weights_out_of_range) return ASR_OK;
    HIP_TRY(h, hipMemsetAsync(h->range_flag, 0, sizeof(flag), h->stream));
    HIP_TRY(h, hipStreamSynchronize(h->stream));
    h->range_retries += 1;
    h->nprod_active = 6;
    rc = run();
    h->nprod_active = 13;
    return rc;
}

}  // namespace

// =================================================================================================
// C ABI
// =================================================================================================
// device buffers of one call, released on return
struct CallBufs {
    asr_handle* h;
    std::vector<void*> p;
    ~CallBufs() { for (void* q : p) dev_free(h, q); }
    template <typename T> int get(T** out, size_t count)
    {
        int r = dev_alloc_t(h, out, count);
        if (!r) p.push_back(*out);
        return r;
    }
};

extern "C" {

int asr_device_count(void)
{
    int n = 0;
    if (hipGetDeviceCount(&n) != hipSuccess) return 0;
    return n;
}

int asr_create(const asr_config* cfg, asr_handle** out)
{
    if (!cfg || !out) { g_create_error = "null argument"; return ASR_ERR_ARG; }
    *out = nullptr;
    auto bad = [&](const std::string& m) { g_create_error = m; return (int)ASR_ERR_ARG; };
    if (cfg->hidden_units <= 0 || cfg->num_heads <= 0 || cfg->hidden_units != cfg->num_heads * ASR_D_HEAD)
        return bad("hidden_units / num_heads must be 64");
    if (cfg->hidden_units > 2048 || (cfg->hidden_units & 63)) return bad("hidden_units must be a multiple of 64, <= 2048");
    if (cfg->input_dim <= 0 || (cfg->input_dim & 3)) return bad("input_dim must be a positive multiple of 4");
    if (cfg->num_blocks < 1) return bad("num_blocks must be >= 1");
    if (cfg->beam_size < 1 || cfg->beam_size > ASR_MAX_BEAM) return bad("beam_size must be in 1..32");
    if (cfg->dst_vocab_size < cfg->beam_size || cfg->dst_vocab_size < 4 || (size_t)cfg->dst_vocab_size * 4 > 150 * 1024)
        return bad("dst_vocab_size must be in [max(4, beam_size), 38400]");
    if (cfg->max_target_length < 1 || cfg->max_target_length > 4000) return bad("max_target_length must be in 1..4000");
    if (cfg->ff_activation < ASR_FF_RELU || cfg->ff_activation > ASR_FF_SWISH) return bad("unknown ff_activation");
    if (cfg->precision < ASR_PRECISION_F32 || cfg->precision > ASR_PRECISION_F32_F16X3) return bad("unknown precision");
    if (cfg->sub_batches < 0 || cfg->sub_batches > MAX_VIEWS) return bad("sub_batches must be 0 (default) or 1..4");
    if (cfg->shared_gpu != 0 && cfg->shared_gpu != 1) return bad("shared_gpu must be 0 or 1");
    if (cfg->reserved[0]) return bad("reserved fields must be zero");
    int ndev = 0;
    if (hipGetDeviceCount(&ndev) != hipSuccess || ndev < 1) { g_create_error = "no HIP device visible (libasr_amd needs an MI355X)"; return ASR_ERR_HIP; }
    if (cfg->device < 0 || cfg->device >= ndev || cfg->device >= MAX_DEVICES) return bad("device ordinal out of range");

    asr_handle* h = new asr_handle();
    h->cfg = *cfg;
    h->H = cfg->hidden_units; h->heads = cfg->num_heads; h->L = cfg->num_blocks; h->V = cfg->dst_vocab_size;
    h->D = cfg->input_dim; h->F = 4 * cfg->hidden_units; h->K = cfg->beam_size;
    h->glu = cfg->ff_activation == ASR_FF_GLU;
    h->nprod = cfg->precision == ASR_PRECISION_F32_BF16X6 ? 6 : cfg->precision == ASR_PRECISION_BF16X3 ? 3
             : cfg->precision == ASR_PRECISION_BF16 ? 1 : cfg->precision == ASR_PRECISION_F32_F16X3 ? 13 : 0;
    h->nprod_active = h->nprod;
    h->kv_bf16 = cfg->precision == ASR_PRECISION_BF16;
    switch (cfg->ff_activation) {
        case ASR_FF_SIGMOID: h->ff_epi = EPI_SIGMOID; break;
        case ASR_FF_TANH: h->ff_epi = EPI_TANH; break;
        case ASR_FF_SWISH: h->ff_epi = EPI_SWISH; break;
        default: h->ff_epi = EPI_RELU; break;
    }
    auto hip_fail = [&](hipError_t e, const char* what) {
        g_create_error = std::string(what) + ": " + hipGetErrorString(e);
        asr_destroy(h);
        return (int)ASR_ERR_HIP;
    };
    hipError_t e;
    if ((e = hipSetDevice(cfg->device)) != hipSuccess) return hip_fail(e, "hipSetDevice");
    {                                                       // once per device, with that device current
        std::lock_guard<std::mutex> lock(g_norm_scratch_mu[cfg->device]);
        double* p = g_norm_scratch_ptr[cfg->device];
        if (!p) {
            if ((e = hipGetSymbolAddress(reinterpret_cast<void**>(&p), HIP_SYMBOL(g_norm_scratch))) != hipSuccess)
                return hip_fail(e, "hipGetSymbolAddress(g_norm_scratch)");
            if (!p) return hip_fail(hipErrorInvalidSymbol, "hipGetSymbolAddress(g_norm_scratch)");
            g_norm_scratch_ptr[cfg->device] = p;
        }
    }
    if ((e = hipStreamCreateWithFlags(&h->stream, hipStreamNonBlocking)) != hipSuccess) return hip_fail(e, "hipStreamCreate");
    if ((e = hipMalloc(reinterpret_cast<void**>(&h->range_flag), 16)) != hipSuccess) return hip_fail(e, "hipMalloc");
    // first work on the stream here, at creation: the runtime binds a stream to one of the process's hardware queues when it
    // is first used, and handles that are first used at the same moment from several host threads were seen to end up on
    // one queue (their kernels then never overlap)
    if ((e = hipMemsetAsync(h->range_flag, 0, 16, h->stream)) != hipSuccess) return hip_fail(e, "hipMemsetAsync");
    if ((e = hipStreamSynchronize(h->stream)) != hipSuccess) return hip_fail(e, "hipStreamSynchronize");
    if ((e = hipEventCreate(&h->pe0)) != hipSuccess) return hip_fail(e, "hipEventCreate");
    if ((e = hipEventCreate(&h->pe1)) != hipSuccess) return hip_fail(e, "hipEventCreate");
    // (the streams of sub-batches 1..3 are created when a call first runs that many parts: a process has few hardware
    //  queues - 4 by default - and streams share them in creation order, so a handle that runs whole batches should hold one)
    if ((e = hipEventCreateWithFlags(&h->fork_ev, hipEventDisableTiming)) != hipSuccess) return hip_fail(e, "hipEventCreate");
    h->shared_gpu = cfg->shared_gpu != 0;
    if (const char* tw = getenv("ASR_AMD_DOUBLE")) h->twice = tw;
    if (const char* ls = getenv("ASR_AMD_LOGIT_SPLIT_SHARED")) { const int v = atoi(ls); if (v == 1 || v == 2) h->logit_split_shared = v; }
    if (cfg->sub_batches) h->sub_batches = cfg->sub_batches;
    else if (const char* sb = getenv("ASR_AMD_SUBBATCH")) h->sub_batches = std::max(0, std::min(MAX_VIEWS, atoi(sb)));
    if (const char* gr = getenv("ASR_AMD_GRAPH")) h->use_graph = atoi(gr) != 0 ? 1 : 0;
    h->step_events.resize(8 * MAX_VIEWS);
    for (auto& ev : h->step_events)
        if ((e = hipEventCreateWithFlags(&ev, hipEventDisableTiming)) != hipSuccess) return hip_fail(e, "hipEventCreate");
    if ((e = hipHostMalloc(reinterpret_cast<void**>(&h->done_host), (size_t)MAX_VIEWS * (cfg->max_target_length + 8) * sizeof(int32_t), 0)) != hipSuccess)
        return hip_fail(e, "hipHostMalloc");
    h->cross_k.assign(h->L, nullptr); h->cross_v.assign(h->L, nullptr);
    h->kcache.assign(h->L, nullptr); h->vcache.assign(h->L, nullptr);
    // the timing-signal table exists from here on (the allocation-free entry point cannot build or grow it)
    if (ensure_pe(h, cfg->max_target_length + 2) != ASR_OK) {
        g_create_error = "timing table: " + h->err;
        asr_destroy(h);
        return ASR_ERR_HIP;
    }
    *out = h;
    return ASR_OK;
}

void asr_destroy(asr_handle* h)
{
    if (!h) return;
    (void)hipSetDevice(h->cfg.device);
    if (h->stream) (void)hipStreamSynchronize(h->stream);
    for (auto xs : h->xstream) if (xs) (void)hipStreamSynchronize(xs);
    for (auto& kv : h->allocs) (void)hipFree(kv.first);
    if (h->range_flag) (void)hipFree(h->range_flag);
    if (h->done_host) (void)hipHostFree(h->done_host);
    for (auto ev : h->step_events) if (ev) (void)hipEventDestroy(ev);
    for (auto& p : h->prof_pending) { (void)hipEventDestroy(p.e0); (void)hipEventDestroy(p.e1); }
    for (hipEvent_t e : h->prof_free) (void)hipEventDestroy(e);
    if (h->live_host) (void)hipHostFree(h->live_host);
    if (h->pe0) (void)hipEventDestroy(h->pe0);
    if (h->pe1) (void)hipEventDestroy(h->pe1);
    if (h->fork_ev) (void)hipEventDestroy(h->fork_ev);
    for (auto xs : h->xstream) if (xs) (void)hipStreamDestroy(xs);
    if (h->stream) (void)hipStreamDestroy(h->stream);
    delete h;
}

const char* asr_last_error(const asr_handle* h) { return h ? h->err.c_str() : g_create_error.c_str(); }

int asr_load_tensor(asr_handle* h, const char* name, const float* data, const int64_t* shape, int32_t ndim)
{
    if (!h || !name || !data || !shape || ndim < 0 || ndim > 4) return h ? fail(h, ASR_ERR_ARG, "bad argument") : ASR_ERR_ARG;
    if (h->finalized) return fail(h, ASR_ERR_STATE, "weights already finalized");
    const std::string n(name);
    if (is_ignored_var(n)) return ASR_OK;
    for (const VarSpec& v : required_vars(h)) {
        if (v.name != n) continue;
        std::vector<int64_t> s(shape, shape + ndim);
        if (s != v.shape) {
            std::string m = "shape mismatch for " + n + ": got [";
            for (auto x : s) m += std::to_string(x) + ",";
            m += "] want [";
            for (auto x : v.shape) m += std::to_string(x) + ",";
            return fail(h, ASR_ERR_WEIGHTS, m + "]");
        }
        size_t cnt = 1;
        for (auto x : s) cnt *= (size_t)x;
        HostTensor t;
        t.shape = s;
        t.data.assign(data, data + cnt);
        h->staged[n] = std::move(t);
        return ASR_OK;
    }
    return fail(h, ASR_ERR_WEIGHTS, "variable not in the inference graph: " + n);
}

int asr_finalize_weights(asr_handle* h)
{
    if (!h) return ASR_ERR_ARG;
    if (h->finalized) return ASR_OK;
    int rc = set_device(h);
    if (rc) return rc;
    std::string missing;
    int nmiss = 0;
    for (const VarSpec& v : required_vars(h))
        if (!h->staged.count(v.name)) { if (nmiss++ < 12) missing += "\n  " + v.name; }
    if (nmiss) return fail(h, ASR_ERR_WEIGHTS, std::to_string(nmiss) + " variable(s) missing:" + missing + (nmiss > 12 ? "\n  ..." : ""));
    if (h->nprod == 13) {
        // fp16x3 needs every GEMM weight inside fp16's range and no weight row below 2^-10 throughout (gemm_split.hip); a
        // checkpoint that is not runs on the bf16x6 kernels instead (same accuracy).
        bool fits = true;
        for (const auto& kv : h->staged) {
            const HostTensor& t = kv.second;
            if (t.shape.size() != 2) continue;                          // GEMM operands are the matrices
            const size_t rows = (size_t)t.shape[0], cols = (size_t)t.shape[1];
            for (size_t r = 0; r < rows && fits; ++r) {
                float rmax = 0.f;
                bool finite = true;
                for (size_t c = 0; c < cols; ++c) {
                    const float a = fabsf(t.data[r * cols + c]);
                    if (!(a < 65504.0f)) finite = false;
                    rmax = fmaxf(rmax, a);
                }
                if (!finite || (rmax > 0.f && rmax < 0.0009765625f)) fits = false;
            }
        }
        if (!fits) h->nprod = h->nprod_active = 6;
    }
    // everything uploaded from here to the end of the variable table goes into the handle's weight store
    h->wstore = std::make_shared<WeightStore>();
    h->wstore->device = h->cfg.device;
    h->wstore_owner = true;
    struct Filling { asr_handle* h; ~Filling() { h->wstore_filling = false; } } filling{h};
    h->wstore_filling = true;
    if ((rc = upload_gemm(h, "encoder/src_change/kernel", &h->w_src))) return rc;
    if ((rc = upload(h, "encoder/src_change/bias", &h->b_src))) return rc;
    if ((rc = upload(h, "encoder/LayerNorm/gamma", &h->in_gamma))) return rc;
    if ((rc = upload(h, "encoder/LayerNorm/beta", &h->in_beta))) return rc;
    if ((rc = upload(h, "decoder/dst_embedding/kernel", &h->emb))) return rc;          // f32: the embedding lookup
    if (!h->cfg.tie_embedding_and_softmax) {
        if ((rc = upload_gemm(h, "decoder/softmax/kernel", &h->softmax_w))) return rc;
    } else if (gemm_nprod(h, h->H)) {
        if ((rc = upload_gemm(h, "decoder/dst_embedding/kernel", &h->emb_gemm))) return rc;
    } else {
        h->emb_gemm = h->emb;
    }
    h->enc.resize(h->L);
    h->dec.resize(h->L);
    for (int i = 0; i < h->L; ++i) {
        const std::string p = "encoder/block_" + std::to_string(i);
        EncBlock& b = h->enc[i];
        if ((rc = upload_gemm(h, p + "/encoder_self_attention/qkv_transform/kernel", &b.wqkv))) return rc;
        if ((rc = upload(h, p + "/encoder_self_attention/qkv_transform/bias", &b.bqkv))) return rc;
        if ((rc = upload_gemm(h, p + "/encoder_self_attention/output_transform/kernel", &b.wo))) return rc;
        if ((rc = upload(h, p + "/encoder_self_attention/output_transform/bias", &b.bo))) return rc;
        if ((rc = upload(h, p + "/layer_norm/layer_norm_scale", &b.ln0s))) return rc;
        if ((rc = upload(h, p + "/layer_norm/layer_norm_bias", &b.ln0b))) return rc;
        if ((rc = upload_ffn1(h, p, &b.w1, &b.b1))) return rc;
        if ((rc = upload_gemm(h, p + "/ff_hidden/dense_1/kernel", &b.w2))) return rc;
        if ((rc = upload(h, p + "/ff_hidden/dense_1/bias", &b.b2))) return rc;
        if ((rc = upload(h, p + "/layer_norm_1/layer_norm_scale", &b.ln1s))) return rc;
        if ((rc = upload(h, p + "/layer_norm_1/layer_norm_bias", &b.ln1b))) return rc;
    }
    for (int i = 0; i < h->L; ++i) {
        const std::string p = "decoder/block_" + std::to_string(i);
        DecBlock& b = h->dec[i];
        if ((rc = upload_gemm(h, p + "/decoder_self_attention/qkv_transform/kernel", &b.wqkv))) return rc;
        if ((rc = upload(h, p + "/decoder_self_attention/qkv_transform/bias", &b.bqkv))) return rc;
        if ((rc = upload_gemm(h, p + "/decoder_self_attention/output_transform/kernel", &b.wo))) return rc;
        if ((rc = upload(h, p + "/decoder_self_attention/output_transform/bias", &b.bo))) return rc;
        if ((rc = upload(h, p + "/layer_norm/layer_norm_scale", &b.ln0s))) return rc;
        if ((rc = upload(h, p + "/layer_norm/layer_norm_bias", &b.ln0b))) return rc;
        if ((rc = upload_gemm(h, p + "/decoder_vanilla_attention/q_transform/kernel", &b.wq))) return rc;
        if ((rc = upload(h, p + "/decoder_vanilla_attention/q_transform/bias", &b.bq))) return rc;
        if ((rc = upload_gemm(h, p + "/decoder_vanilla_attention/kv_transform/kernel", &b.wkv))) return rc;
        if ((rc = upload(h, p + "/decoder_vanilla_attention/kv_transform/bias", &b.bkv))) return rc;
        if ((rc = upload_gemm(h, p + "/decoder_vanilla_attention/output_transform/kernel", &b.wco))) return rc;
        if ((rc = upload(h, p + "/decoder_vanilla_attention/output_transform/bias", &b.bco))) return rc;
        if ((rc = upload(h, p + "/layer_norm_1/layer_norm_scale", &b.ln1s))) return rc;
        if ((rc = upload(h, p + "/layer_norm_1/layer_norm_bias", &b.ln1b))) return rc;
        if ((rc = upload_ffn1(h, p, &b.w1, &b.b1))) return rc;
        if ((rc = upload_gemm(h, p + "/ff_hidden/dense_1/kernel", &b.w2))) return rc;
        if ((rc = upload(h, p + "/ff_hidden/dense_1/bias", &b.b2))) return rc;
        if ((rc = upload(h, p + "/layer_norm_2/layer_norm_scale", &b.ln2s))) return rc;
        if ((rc = upload(h, p + "/layer_norm_2/layer_norm_bias", &b.ln2b))) return rc;
    }
    h->wstore_filling = false;
    h->staged.clear();
    if ((rc = ensure_pe(h, h->cfg.max_target_length + 2))) return rc;
    h->finalized = true;
    return ASR_OK;
}

// The handles of one GPU share one copy of the packed weights (include/asr_amd.h): `h` adopts the store `from` filled.
int asr_share_weights(asr_handle* h, asr_handle* from)
{
    if (!h || !from || h == from) return h ? fail(h, ASR_ERR_ARG, "asr_share_weights needs two different handles") : ASR_ERR_ARG;
    if (h->finalized) return fail(h, ASR_ERR_STATE, "weights already finalized");
    if (!from->finalized || !from->wstore) return fail(h, ASR_ERR_STATE, "the other handle holds no finalized weights");
    const asr_config &a = h->cfg, &b = from->cfg;
    if (a.device != b.device) return fail(h, ASR_ERR_ARG, "handles of different GPUs cannot share weights");
    if (a.input_dim != b.input_dim || a.hidden_units != b.hidden_units || a.num_heads != b.num_heads || a.num_blocks != b.num_blocks ||
        a.dst_vocab_size != b.dst_vocab_size || a.ff_activation != b.ff_activation ||
        (a.tie_embedding_and_softmax != 0) != (b.tie_embedding_and_softmax != 0) || a.precision != b.precision)
        return fail(h, ASR_ERR_ARG, "handles with different model shapes or precision modes cannot share weights");
    h->wstore = from->wstore;
    h->wstore_owner = false;
    h->nprod = from->nprod;                                 // (a checkpoint outside fp16's range has moved the owner to bf16x6)
    h->nprod_active = h->nprod;
    h->w_src = from->w_src; h->b_src = from->b_src; h->in_gamma = from->in_gamma; h->in_beta = from->in_beta;
    h->emb = from->emb; h->softmax_w = from->softmax_w; h->emb_gemm = from->emb_gemm;
    h->enc = from->enc; h->dec = from->dec;
    h->staged.clear();
    int rc = set_device(h);
    if (rc) return rc;
    if ((rc = ensure_pe(h, h->cfg.max_target_length + 2))) return rc;
    h->finalized = true;
    return ASR_OK;
}

// Regime of the calls that follow (include/asr_amd.h): what asr_config.shared_gpu / sub_batches set at creation.
int asr_set_sharing(asr_handle* h, int32_t shared_gpu, int32_t sub_batches)
{
    if (!h) return ASR_ERR_ARG;
    if ((shared_gpu != 0 && shared_gpu != 1) || sub_batches < 0 || sub_batches > MAX_VIEWS)
        return fail(h, ASR_ERR_ARG, "shared_gpu must be 0 or 1, sub_batches 0 (automatic) or 1..4");
    h->shared_gpu = shared_gpu != 0;
    h->sub_batches = sub_batches;
    return ASR_OK;
}

static int asr_decode_dev_once(asr_handle* h, const float* X_dev, int32_t n, int32_t t, int32_t d, int32_t raw_frames, int32_t raw_dim,
                   int32_t left, int32_t right, int32_t sub, int32_t* Y, int64_t y_capacity, int32_t* len_out)
{
    if (!h || !len_out || (n > 0 && (!X_dev || !Y))) return h ? fail(h, ASR_ERR_ARG, "null argument") : ASR_ERR_ARG;
    int rc = set_device(h);
    if (rc) return rc;
    if (raw_frames > 0) {
        if (sub < 1 || left < 0 || right < 0 || raw_dim < 1) return fail(h, ASR_ERR_ARG, "bad frame-stacking parameters");
        t = (raw_frames + sub - 1) / sub;
        d = raw_dim * (left + right + 1);
    }
    if ((rc = check_xshape(h, n, t, d))) return rc;
    if (n == 0) { *len_out = 0; return ASR_OK; }
    if ((rc = ensure_encoder_capacity(h, n, t))) return rc;
    const float* X = X_dev;
    if (raw_frames > 0) {
        ProfScope ps(h, "frame_stack", 0, 4.0 * n * ((double)raw_frames * raw_dim + (double)t * d));
        HIP_TRY(h, launch_frame_stack(X_dev, n, raw_frames, raw_dim, left, right, sub, h->xin, h->stream));
        X = h->xin;
    }
    return decode_core(h, X, n, t, Y, y_capacity, len_out, nullptr);
}

int asr_decode_dev(asr_handle* h, const float* X_dev, int32_t n, int32_t t, int32_t d, int32_t raw_frames, int32_t raw_dim,
                   int32_t left, int32_t right, int32_t sub, int32_t* Y, int64_t y_capacity, int32_t* len_out)
{
    if (!h) return ASR_ERR_ARG;
    return with_range_retry(h, [&]() { return asr_decode_dev_once(h, X_dev, n, t, d, raw_frames, raw_dim, left, right, sub, Y, y_capacity, len_out); });
}

static int asr_decode_trace_once(asr_handle* h, const float* X, int32_t n, int32_t t, int32_t d, int32_t* Y, int64_t y_capacity,
                     int32_t* len_out, int32_t trace_steps, float* logits, float* scores, int32_t* tokens, int32_t* parents)
{
    if (!h || !len_out || (n > 0 && (!X || !Y))) return h ? fail(h, ASR_ERR_ARG, "null argument") : ASR_ERR_ARG;
    int rc = set_device(h);
    if (rc) return rc;
    if ((rc = check_xshape(h, n, t, d))) return rc;
    if (n == 0) { *len_out = 0; return ASR_OK; }
    if ((rc = ensure_encoder_capacity(h, n, t))) return rc;
    HIP_TRY(h, hipMemcpyAsync(h->xin, X, (size_t)n * t * d * sizeof(float), hipMemcpyHostToDevice, h->stream));
    TraceOut tr;
    tr.steps = trace_steps; tr.logits = logits; tr.scores = scores; tr.tokens = tokens; tr.parents = parents;
    return decode_core(h, h->xin, n, t, Y, y_capacity, len_out, trace_steps > 0 ? &tr : nullptr);
}

int asr_decode_trace(asr_handle* h, const float* X, int32_t n, int32_t t, int32_t d, int32_t* Y, int64_t y_capacity,
                     int32_t* len_out, int32_t trace_steps, float* logits, float* scores, int32_t* tokens, int32_t* parents)
{
    if (!h) return ASR_ERR_ARG;
    return with_range_retry(h, [&]() { return asr_decode_trace_once(h, X, n, t, d, Y, y_capacity, len_out, trace_steps, logits, scores, tokens, parents); });
}

int asr_decode(asr_handle* h, const float* X, int32_t n, int32_t t, int32_t d, int32_t* Y, int64_t y_capacity, int32_t* len_out)
{
    return asr_decode_trace(h, X, n, t, d, Y, y_capacity, len_out, 0, nullptr, nullptr, nullptr, nullptr);
}

static int asr_decode_groups_once(asr_handle* h, const float* X, int32_t n_groups, const int32_t* n_g, const int32_t* t_g, int32_t d,
                                  int32_t* Y, int64_t y_capacity, int32_t* len_out)
{
    if (!h || !len_out || !X || !Y || !n_g || !t_g || n_groups < 1 || n_groups > 4096)
        return h ? fail(h, ASR_ERR_ARG, "null argument or group count outside 1..4096") : ASR_ERR_ARG;
    int rc = set_device(h);
    if (rc) return rc;
    Groups gr;
    gr.count = n_groups; gr.n = n_g; gr.t = t_g;
    int64_t n = 0;
    for (int g = 0; g < n_groups; ++g) {
        if (n_g[g] < 1 || t_g[g] < 1) return fail(h, ASR_ERR_ARG, "every group needs n >= 1 utterances of t >= 1 frames");
        n += n_g[g];
        gr.rows += (size_t)n_g[g] * t_g[g];
        gr.t_max = std::max(gr.t_max, (int)t_g[g]);
    }
    if (n > (1 << 20) || gr.rows > ((size_t)1 << 31) - 64) return fail(h, ASR_ERR_ARG, "too many utterances or frames in one call");
    if ((rc = check_xshape(h, (int)n, gr.t_max, d))) return rc;
    if ((rc = ensure_encoder_rows(h, (int)n, gr.rows))) return rc;
    std::vector<int32_t> ut(n), uoff(n), ulim(n);
    {
        size_t row0 = 0, u = 0;
        for (int g = 0; g < n_groups; ++g) {
            for (int i = 0; i < n_g[g]; ++i, ++u) {
                ut[u] = t_g[g];
                uoff[u] = (int32_t)(row0 + (size_t)i * t_g[g]);
                ulim[u] = std::min(t_g[g] + 50, (int)h->cfg.max_target_length);                 // model.py:310 with the group's T
            }
            row0 += (size_t)n_g[g] * t_g[g];
        }
    }
    if ((size_t)n > h->grp_cap) {                                  // kept by the handle: no allocation per call (a free would wait
        dev_free(h, h->grp_buf);                                   // for the other handles' kernels too)
        h->grp_buf = nullptr; h->grp_cap = 0;
        const size_t cap = std::max<size_t>((size_t)n, 256);
        if (dev_alloc_t(h, &h->grp_buf, 3 * cap)) return ASR_ERR_HIP;
        h->grp_cap = cap;
    }
    int32_t *dt = h->grp_buf, *doff = h->grp_buf + h->grp_cap, *dlim = h->grp_buf + 2 * h->grp_cap;
    // (the host vectors outlive the copies: decode_core has waited for the stream when it returns)
    HIP_TRY(h, hipMemcpyAsync(dt, ut.data(), (size_t)n * sizeof(int32_t), hipMemcpyHostToDevice, h->stream));
    HIP_TRY(h, hipMemcpyAsync(doff, uoff.data(), (size_t)n * sizeof(int32_t), hipMemcpyHostToDevice, h->stream));
    HIP_TRY(h, hipMemcpyAsync(dlim, ulim.data(), (size_t)n * sizeof(int32_t), hipMemcpyHostToDevice, h->stream));
    gr.d_t = dt; gr.d_off = doff; gr.d_limit = dlim;
    HIP_TRY(h, hipMemcpyAsync(h->xin, X, gr.rows * (size_t)d * sizeof(float), hipMemcpyHostToDevice, h->stream));
    return decode_core(h, h->xin, (int)n, gr.t_max, Y, y_capacity, len_out, nullptr, &gr);
}

int asr_decode_groups(asr_handle* h, const float* X, int32_t n_groups, const int32_t* n_g, const int32_t* t_g, int32_t d, int32_t* Y,
                      int64_t y_capacity, int32_t* len_out)
{
    if (!h) return ASR_ERR_ARG;
    return with_range_retry(h, [&]() { return asr_decode_groups_once(h, X, n_groups, n_g, t_g, d, Y, y_capacity, len_out); });
}

// Encoder and teacher-forced decoder_impl on shift_right(Y) (model.py:171,492-557): logits [n * ty, V] of every target position, queued on the
// handle's stream; *dY: the targets on the device
static int teacher_forced_logits(asr_handle* h, const float* X, int32_t n, int32_t t, int32_t d, const int32_t* Y, int32_t ty, CallBufs& tmp,
                                 float** logits, int32_t** dY)
{
    int rc;
    if ((rc = ensure_encoder_capacity(h, n, t))) return rc;
    if ((rc = ensure_pe(h, std::max(t, ty)))) return rc;
    hipStream_t s = h->stream;
    const int H = h->H, F = h->F, M = n * t, Md = n * ty;
    const size_t MH = (size_t)Md * H;
    float *y0, *z1, *z2, *ctx, *part, *qkv, *kv, *hid;
    if ((rc = tmp.get(dY, (size_t)Md))) return rc;
    if ((rc = tmp.get(&y0, MH)) || (rc = tmp.get(&z1, MH)) || (rc = tmp.get(&z2, MH)) || (rc = tmp.get(&ctx, MH)) || (rc = tmp.get(&part, MH)) ||
        (rc = tmp.get(&qkv, 3 * MH)) || (rc = tmp.get(&kv, (size_t)M * 2 * H)) || (rc = tmp.get(&hid, (size_t)Md * F)) ||
        (rc = tmp.get(logits, (size_t)Md * h->V)))
        return rc;
    HIP_TRY(h, hipMemcpyAsync(h->xin, X, (size_t)M * d * sizeof(float), hipMemcpyHostToDevice, s));
    HIP_TRY(h, hipMemcpyAsync(*dY, Y, (size_t)Md * sizeof(int32_t), hipMemcpyHostToDevice, s));
    if ((rc = run_encoder(h, h->xin, n, t))) return rc;                         // -> h->x0, h->pad2
    const float mult = h->cfg.scale_embedding ? (float)sqrt((double)H) : 1.0f;
    HIP_TRY(h, launch_embed_shifted(h->emb, *dY, Md, ty, h->V, h->pe, mult, H, y0, s));            // model.py:500-508
    for (int l = 0; l < h->L; ++l) {
        const DecBlock& b = h->dec[l];
        if ((rc = gemm(h, y0, b.wqkv, b.bqkv, qkv, Md, 3 * H, H, EPI_BIAS, 1))) return rc;
        HIP_TRY(h, launch_mha(qkv, 3 * H, qkv + H, 3 * H, qkv + 2 * H, 3 * H, nullptr, 1, n, ty, ty, h->heads, ctx, mha_mode(h), h->range_flag, s));   // :516-529
        if ((rc = gemm(h, ctx, b.wo, nullptr, part, Md, H, H, EPI_PARTIAL, 1))) return rc;
        HIP_TRY(h, launch_add_layer_norm(y0, part, 1, 0, b.bo, b.ln0s, b.ln0b, nullptr, nullptr, Md, H, z1, s));
        if ((rc = gemm(h, z1, b.wq, b.bq, part, Md, H, H, EPI_BIAS, 1))) return rc;
        if ((rc = gemm(h, h->x0, b.wkv, b.bkv, kv, M, 2 * H, H, EPI_BIAS, 1))) return rc;
        HIP_TRY(h, launch_mha(part, H, kv, 2 * H, kv + H, 2 * H, h->pad2, 0, n, ty, t, h->heads, ctx, mha_mode(h), h->range_flag, s));              // :532-544
        if ((rc = gemm(h, ctx, b.wco, nullptr, part, Md, H, H, EPI_PARTIAL, 1))) return rc;
        HIP_TRY(h, launch_add_layer_norm(z1, part, 1, 0, b.bco, b.ln1s, b.ln1b, nullptr, nullptr, Md, H, z2, s));
        if ((rc = gemm(h, z2, b.w1, b.b1, hid, Md, h->glu ? 2 * F : F, H, h->glu ? EPI_GLU : h->ff_epi, 1))) return rc;
        if ((rc = gemm(h, hid, b.w2, nullptr, part, Md, H, F, EPI_PARTIAL, 1))) return rc;
        HIP_TRY(h, launch_add_layer_norm(z2, part, 1, 0, b.b2, b.ln2s, b.ln2b, nullptr, nullptr, Md, H, y0, s));        // :547-555
    }
    const float* wout = h->cfg.tie_embedding_and_softmax ? h->emb_gemm : h->softmax_w;
    if ((rc = gemm(h, y0, wout, nullptr, *logits, Md, h->V, H, EPI_BIAS, 1))) return rc;            // :353-355
    return ASR_OK;
}

// Replaces Evaluator.loss (evaluate.py:49-50): sess.run(model.loss_sum) for one tower = the teacher-forced logits and test_loss (model.py:350-360).
static int asr_loss_once(asr_handle* h, const float* X, int32_t n, int32_t t, int32_t d, const int32_t* Y, int32_t ty, double* loss_sum)
{
    if (!h || !loss_sum || (n > 0 && (!X || !Y))) return h ? fail(h, ASR_ERR_ARG, "null argument") : ASR_ERR_ARG;
    *loss_sum = 0.0;
    if (!h->finalized) return fail(h, ASR_ERR_STATE, "asr_finalize_weights has not succeeded on this handle");
    int rc = set_device(h);
    if (rc) return rc;
    if ((rc = check_xshape(h, n, t, d))) return rc;
    if (n == 0) return ASR_OK;                                                  // model.py:184-187: loss 0.0
    if (ty < 1 || ty > 16384) return fail(h, ASR_ERR_ARG, "target length must be in 1..16384");
    CallBufs tmp{h, {}};
    float *logits = nullptr, *rowl = nullptr;
    int32_t* dY = nullptr;
    if ((rc = teacher_forced_logits(h, X, n, t, d, Y, ty, tmp, &logits, &dY))) return rc;
    const int Md = n * ty;
    if ((rc = tmp.get(&rowl, (size_t)Md))) return rc;
    hipStream_t s = h->stream;
    HIP_TRY(h, launch_xent_rows(logits, dY, Md, h->V, rowl, s));
    std::vector<float> rl((size_t)Md);
    HIP_TRY(h, hipMemcpyAsync(rl.data(), rowl, rl.size() * sizeof(float), hipMemcpyDeviceToHost, s));
    HIP_TRY(h, hipStreamSynchronize(s));
    double acc = 0.0;
    for (float v : rl) acc += (double)v;
    *loss_sum = acc;
    return ASR_OK;
}

int asr_loss(asr_handle* h, const float* X, int32_t n, int32_t t, int32_t d, const int32_t* Y, int32_t ty, double* loss_sum)
{
    if (!h) return ASR_ERR_ARG;
    return with_range_retry(h, [&]() { return asr_loss_once(h, X, n, t, d, Y, ty, loss_sum); });
}

// Token by token: the teacher-forced logits and token_logprobs (ops_rows.hip) on them.
static int asr_score_once(asr_handle* h, const float* X, int32_t n, int32_t t, int32_t d, const int32_t* Y, int32_t ty, int32_t top, float* logprob,
                          float* entropy, float* top_logprobs, int32_t* top_tokens)
{
    if (n > 0 && (!X || !Y || !logprob || !entropy || (top > 0 && (!top_logprobs || !top_tokens)))) return fail(h, ASR_ERR_ARG, "null argument");
    if (!h->finalized) return fail(h, ASR_ERR_STATE, "asr_finalize_weights has not succeeded on this handle");
    int rc = set_device(h);
    if (rc) return rc;
    if ((rc = check_xshape(h, n, t, d))) return rc;
    if (top < 0 || top > 32 || top > h->V) return fail(h, ASR_ERR_ARG, "top must be in 0..min(32, dst_vocab_size)");
    if (n == 0) return ASR_OK;
    if (ty < 1 || ty > 16384) return fail(h, ASR_ERR_ARG, "target length must be in 1..16384");
    const size_t Md = (size_t)n * ty;
    std::vector<int32_t> tokens(Y, Y + Md);                                     // (outlives the device buffers, whose release waits for the copies)
    CallBufs tmp{h, {}};
    for (int32_t& v : tokens)
        if (v == 0) v = -1;                                                     // padding: "no token"
    float *logits = nullptr, *dlp, *dh, *dtl = nullptr;
    int32_t *dY = nullptr, *dtok, *dtt = nullptr;
    if ((rc = teacher_forced_logits(h, X, n, t, d, Y, ty, tmp, &logits, &dY))) return rc;
    if ((rc = tmp.get(&dtok, Md)) || (rc = tmp.get(&dlp, Md)) || (rc = tmp.get(&dh, Md))) return rc;
    if (top > 0 && ((rc = tmp.get(&dtl, Md * top)) || (rc = tmp.get(&dtt, Md * top)))) return rc;
    hipStream_t s = h->stream;
    HIP_TRY(h, hipMemcpyAsync(dtok, tokens.data(), Md * sizeof(int32_t), hipMemcpyHostToDevice, s));
    asr_token_logprobs_args a{};
    a.logits = logits; a.tokens = dtok; a.logprob = dlp; a.entropy = dh; a.top_logprobs = dtl; a.top_tokens = dtt;
    a.rows = (int64_t)Md; a.row_stride = h->V; a.vocab = h->V; a.top = top; a.dtype = ASR_F32; a.token_bytes = 4;
    if ((rc = ops_token_logprobs(a, s))) return fail(h, rc, asr_ops_last_error());
    HIP_TRY(h, hipMemcpyAsync(logprob, dlp, Md * sizeof(float), hipMemcpyDeviceToHost, s));
    HIP_TRY(h, hipMemcpyAsync(entropy, dh, Md * sizeof(float), hipMemcpyDeviceToHost, s));
    if (top > 0) {
        HIP_TRY(h, hipMemcpyAsync(top_logprobs, dtl, Md * top * sizeof(float), hipMemcpyDeviceToHost, s));
        HIP_TRY(h, hipMemcpyAsync(top_tokens, dtt, Md * top * sizeof(int32_t), hipMemcpyDeviceToHost, s));
    }
    HIP_TRY(h, hipStreamSynchronize(s));
    return ASR_OK;
}

int asr_score(asr_handle* h, const float* X, int32_t n, int32_t t, int32_t d, const int32_t* Y, int32_t ty, int32_t top, float* logprob, float* entropy,
              float* top_logprobs, int32_t* top_tokens)
{
    if (!h) return ASR_ERR_ARG;
    try {
        return with_range_retry(h, [&]() { return asr_score_once(h, X, n, t, d, Y, ty, top, logprob, entropy, top_logprobs, top_tokens); });
    } catch (const std::bad_alloc&) {
        return fail(h, ASR_ERR_CAPACITY, "out of memory");
    }
}

int asr_stack_frames(asr_handle* h, const float* feats, int32_t n_frames, int32_t dim, int32_t left, int32_t right, int32_t sub,
                     float* out)
{
    if (!h || !feats || !out || n_frames < 1 || dim < 1 || left < 0 || right < 0 || sub < 1)
        return h ? fail(h, ASR_ERR_ARG, "bad argument") : ASR_ERR_ARG;
    int rc = set_device(h);
    if (rc) return rc;
    const int t = (n_frames + sub - 1) / sub, w = dim * (left + right + 1);
    float *din = nullptr, *dout = nullptr;
    HIP_TRY(h, hipMalloc(reinterpret_cast<void**>(&din), (size_t)n_frames * dim * 4));
    hipError_t e = hipMalloc(reinterpret_cast<void**>(&dout), (size_t)t * w * 4);
    if (e == hipSuccess) e = hipMemcpyAsync(din, feats, (size_t)n_frames * dim * 4, hipMemcpyHostToDevice, h->stream);
    if (e == hipSuccess) e = launch_frame_stack(din, 1, n_frames, dim, left, right, sub, dout, h->stream);
    if (e == hipSuccess) e = hipMemcpyAsync(out, dout, (size_t)t * w * 4, hipMemcpyDeviceToHost, h->stream);
    if (e == hipSuccess) e = hipStreamSynchronize(h->stream);
    (void)hipFree(din);
    if (dout) (void)hipFree(dout);
    HIP_TRY(h, e);
    return ASR_OK;
}

// ---- feature front end (third_party/feat_convert/io/fea.py), one utterance per call, host buffers -------------
int asr_fea_add_delt(asr_handle* h, const float* feats, int32_t n_frames, int32_t dim, float* out)
{
    if (!h || !feats || !out || n_frames < 1 || dim < 1) return h ? fail(h, ASR_ERR_ARG, "bad argument") : ASR_ERR_ARG;
    int rc = set_device(h);
    if (rc) return rc;
    const size_t cnt = (size_t)n_frames * dim;
    return fea_roundtrip(h, feats, cnt, out, 3 * cnt, [&](float* din, float* dout, TmpBufs&, hipStream_t s) {
        return launch_fea_add_delt(din, n_frames, dim, dout, s);
    });
}

int asr_fea_cmvn_global(asr_handle* h, const float* feats, int32_t n_frames, int32_t dim, const float* mean, const float* var,
                        float* out)
{
    if (!h || !feats || !out || !mean || !var || n_frames < 1 || dim < 1)
        return h ? fail(h, ASR_ERR_ARG, "bad argument") : ASR_ERR_ARG;
    int rc = set_device(h);
    if (rc) return rc;
    const size_t cnt = (size_t)n_frames * dim;
    return fea_roundtrip(h, feats, cnt, out, cnt, [&](float* din, float* dout, TmpBufs& tb, hipStream_t s) {
        float *dm = nullptr, *dv = nullptr;
        hipError_t e = tb.up(&dm, mean, (size_t)dim, s);
        if (e == hipSuccess) e = tb.up(&dv, var, (size_t)dim, s);
        if (e == hipSuccess) e = launch_fea_cmvn_global(din, dm, dv, n_frames, dim, dout, s);
        return e;
    });
}

int asr_fea_cmvn_utt(asr_handle* h, const float* feats, int32_t n_frames, int32_t dim, float* out)
{
    if (!h || !feats || !out || n_frames < 1 || dim < 1) return h ? fail(h, ASR_ERR_ARG, "bad argument") : ASR_ERR_ARG;
    int rc = set_device(h);
    if (rc) return rc;
    const size_t cnt = (size_t)n_frames * dim;
    return fea_roundtrip(h, feats, cnt, out, cnt, [&](float* din, float* dout, TmpBufs&, hipStream_t s) {
        return launch_fea_cmvn_utt(din, n_frames, dim, dout, s);
    });
}

int asr_fea_splice(asr_handle* h, const float* feats, int32_t n_frames, int32_t dim, int32_t left, int32_t right, int32_t sub,
                   int32_t offset, int32_t edge, float* out)
{
    if (!h || !feats || !out || n_frames < 1 || dim < 1 || left < 0 || right < 0 || sub < 1 || offset < 0 || offset >= n_frames ||
        (edge != 0 && edge != 1))
        return h ? fail(h, ASR_ERR_ARG, "bad argument") : ASR_ERR_ARG;
    int rc = set_device(h);
    if (rc) return rc;
    const size_t t_out = (size_t)(n_frames - offset + sub - 1) / sub;
    return fea_roundtrip(h, feats, (size_t)n_frames * dim, out, t_out * dim * (left + right + 1),
                         [&](float* din, float* dout, TmpBufs&, hipStream_t s) {
                             return launch_fea_splice(din, n_frames, dim, left, right, sub, offset, edge, dout, s);
                         });
}

static int asr_encode_once(asr_handle* h, const float* X, int32_t n, int32_t t, int32_t d, float* enc_out, int32_t* pad_out)
{
    if (!h || !X || !enc_out) return h ? fail(h, ASR_ERR_ARG, "null argument") : ASR_ERR_ARG;
    if (!h->finalized) return fail(h, ASR_ERR_STATE, "asr_finalize_weights has not succeeded on this handle");
    int rc = set_device(h);
    if (rc) return rc;
    if ((rc = check_xshape(h, n, t, d))) return rc;
    if (n == 0) return ASR_OK;
    if ((rc = ensure_encoder_capacity(h, n, t))) return rc;
    HIP_TRY(h, hipMemcpyAsync(h->xin, X, (size_t)n * t * d * sizeof(float), hipMemcpyHostToDevice, h->stream));
    if ((rc = run_encoder(h, h->xin, n, t))) return rc;
    HIP_TRY(h, hipMemcpyAsync(enc_out, h->x0, (size_t)n * t * h->H * sizeof(float), hipMemcpyDeviceToHost, h->stream));
    if (pad_out) HIP_TRY(h, hipMemcpyAsync(pad_out, h->pad, (size_t)n * t * sizeof(int32_t), hipMemcpyDeviceToHost, h->stream));
    HIP_TRY(h, hipStreamSynchronize(h->stream));
    return ASR_OK;
}

int asr_encode(asr_handle* h, const float* X, int32_t n, int32_t t, int32_t d, float* enc_out, int32_t* pad_out)
{
    if (!h) return ASR_ERR_ARG;
    return with_range_retry(h, [&]() { return asr_encode_once(h, X, n, t, d, enc_out, pad_out); });
}

// ---- single-kernel probes ----------------------------------------------------------------------

static int asr_op_dense_once(asr_handle* h, const float* x, const float* w, const float* bias, int32_t m, int32_t n, int32_t k, int32_t split_k,
                 float* y)
{
    if (!h || !x || !w || !y || m < 1 || n < 1 || k < 4 || (k & 3) || split_k < 1 || split_k > ASR_MAX_SPLITK)
        return h ? fail(h, ASR_ERR_ARG, "bad argument") : ASR_ERR_ARG;
    int rc = set_device(h);
    if (rc) return rc;
    TmpBufs tb;
    float *dx, *dw, *db = nullptr, *dy, *dpart = nullptr;
    hipStream_t s = h->stream;
    HIP_TRY(h, tb.up(&dx, x, (size_t)m * k, s));
    if ((rc = tb.up_gemm(h, &dw, w, n, k, s))) return rc;
    if (bias) HIP_TRY(h, tb.up(&db, bias, (size_t)n, s));
    HIP_TRY(h, tb.up<float>(&dy, nullptr, (size_t)m * n, s));
    if (split_k == 1) {
        if ((rc = gemm(h, dx, dw, db, dy, m, n, k, EPI_BIAS, 1))) return rc;
    } else {
        // split-K slabs, reduced in slab order by a trivial host loop (the product path reduces them inside
        // the consumer kernels; see asr_op_add_layer_norm for that path)
        HIP_TRY(h, tb.up<float>(&dpart, nullptr, (size_t)split_k * m * n, s));
        if ((rc = gemm(h, dx, dw, nullptr, dpart, m, n, k, EPI_PARTIAL, split_k))) return rc;
        std::vector<float> part((size_t)split_k * m * n);
        HIP_TRY(h, hipMemcpyAsync(part.data(), dpart, part.size() * 4, hipMemcpyDeviceToHost, s));
        HIP_TRY(h, hipStreamSynchronize(s));
        for (size_t i = 0; i < (size_t)m * n; ++i) {
            float acc = 0.f;
            for (int z = 0; z < split_k; ++z) acc += part[(size_t)z * m * n + i];
            y[i] = acc + (bias ? bias[i % n] : 0.f);
        }
        return ASR_OK;
    }
    HIP_TRY(h, hipMemcpyAsync(y, dy, (size_t)m * n * 4, hipMemcpyDeviceToHost, s));
    HIP_TRY(h, hipStreamSynchronize(s));
    return ASR_OK;
}

int asr_op_dense(asr_handle* h, const float* x, const float* w, const float* bias, int32_t m, int32_t n, int32_t k, int32_t split_k,
                 float* y)
{
    if (!h) return ASR_ERR_ARG;
    return with_range_retry(h, [&]() { return asr_op_dense_once(h, x, w, bias, m, n, k, split_k, y); });
}

static int asr_op_dense_glu_once(asr_handle* h, const float* x, const float* w1, const float* b1, const float* w2, const float* b2, int32_t m,
                     int32_t n, int32_t k, float* y)
{
    if (!h || !x || !w1 || !w2 || !y || m < 1 || n < 16 || (n & 15) || k < 4 || (k & 3))
        return h ? fail(h, ASR_ERR_ARG, "bad argument (n must be a multiple of 16)") : ASR_ERR_ARG;
    int rc = set_device(h);
    if (rc) return rc;
    std::vector<float> wp((size_t)2 * n * k), bp((size_t)2 * n, 0.f);
    for (int g = 0; g < n / 16; ++g)
        for (int r = 0; r < 16; ++r) {
            memcpy(&wp[((size_t)g * 32 + r) * k], &w1[((size_t)g * 16 + r) * k], (size_t)k * 4);
            memcpy(&wp[((size_t)g * 32 + 16 + r) * k], &w2[((size_t)g * 16 + r) * k], (size_t)k * 4);
            if (b1) bp[(size_t)g * 32 + r] = b1[(size_t)g * 16 + r];
            if (b2) bp[(size_t)g * 32 + 16 + r] = b2[(size_t)g * 16 + r];
        }
    TmpBufs tb;
    float *dx, *dw, *db, *dy;
    hipStream_t s = h->stream;
    HIP_TRY(h, tb.up(&dx, x, (size_t)m * k, s));
    if ((rc = tb.up_gemm(h, &dw, wp.data(), 2 * n, k, s))) return rc;
    HIP_TRY(h, tb.up(&db, bp.data(), bp.size(), s));
    HIP_TRY(h, tb.up<float>(&dy, nullptr, (size_t)m * n, s));
    if ((rc = gemm(h, dx, dw, db, dy, m, 2 * n, k, EPI_GLU, 1))) return rc;
    HIP_TRY(h, hipMemcpyAsync(y, dy, (size_t)m * n * 4, hipMemcpyDeviceToHost, s));
    HIP_TRY(h, hipStreamSynchronize(s));
    return ASR_OK;
}

int asr_op_dense_glu(asr_handle* h, const float* x, const float* w1, const float* b1, const float* w2, const float* b2, int32_t m,
                     int32_t n, int32_t k, float* y)
{
    if (!h) return ASR_ERR_ARG;
    return with_range_retry(h, [&]() { return asr_op_dense_glu_once(h, x, w1, b1, w2, b2, m, n, k, y); });
}

int asr_op_add_layer_norm(asr_handle* h, const float* x, const float* delta, const float* dbias, const float* scale, const float* bias,
                          int32_t rows, int32_t hidden, float* y)
{
    if (!h || !x || !delta || !scale || !bias || !y || rows < 1 || hidden < 4 || (hidden & 3) || hidden > 2048)
        return h ? fail(h, ASR_ERR_ARG, "bad argument") : ASR_ERR_ARG;
    int rc = set_device(h);
    if (rc) return rc;
    TmpBufs tb;
    float *dx, *dd, *db = nullptr, *ds, *dbi, *dy;
    hipStream_t s = h->stream;
    const size_t cnt = (size_t)rows * hidden;
    HIP_TRY(h, tb.up(&dx, x, cnt, s));
    HIP_TRY(h, tb.up(&dd, delta, cnt, s));
    if (dbias) HIP_TRY(h, tb.up(&db, dbias, (size_t)hidden, s));
    HIP_TRY(h, tb.up(&ds, scale, (size_t)hidden, s));
    HIP_TRY(h, tb.up(&dbi, bias, (size_t)hidden, s));
    HIP_TRY(h, tb.up<float>(&dy, nullptr, cnt, s));
    HIP_TRY(h, launch_add_layer_norm(dx, dd, 1, 0, db, ds, dbi, nullptr, nullptr, rows, hidden, dy, s));
    HIP_TRY(h, hipMemcpyAsync(y, dy, cnt * 4, hipMemcpyDeviceToHost, s));
    HIP_TRY(h, hipStreamSynchronize(s));
    return ASR_OK;
}

int asr_op_embedding(asr_handle* h, const float* emb, const int32_t* tokens, int32_t rows, int32_t vocab, int32_t hidden,
                     int32_t position, int32_t scale, float* y)
{
    if (!h || !emb || !tokens || !y || rows < 1 || vocab < 1 || hidden != h->H || position < 0)
        return h ? fail(h, ASR_ERR_ARG, "bad argument (hidden must equal the handle's hidden_units, position >= 0)") : ASR_ERR_ARG;
    for (int r = 0; r < rows; ++r)
        if (tokens[r] < 0 || tokens[r] >= vocab) return fail(h, ASR_ERR_ARG, "token id outside [0, vocab)");
    int rc = set_device(h);
    if (rc) return rc;
    if ((rc = ensure_pe(h, position + 1))) return rc;
    // the decode step's own kernel: it takes the token of row r from column `pos` of the prediction table of parity pos & 1
    const int stride = position + 1;
    std::vector<int32_t> preds((size_t)rows * stride, 3);
    for (int r = 0; r < rows; ++r) preds[(size_t)r * stride + position] = tokens[r];
    const int32_t scalars[2] = {position, 0};                        // pos, done
    TmpBufs tb;
    float *de, *dy;
    int32_t *dp, *dsc;
    hipStream_t s = h->stream;
    HIP_TRY(h, tb.up(&de, emb, (size_t)vocab * hidden, s));
    HIP_TRY(h, tb.up(&dp, preds.data(), preds.size(), s));
    HIP_TRY(h, tb.up(&dsc, scalars, (size_t)2, s));
    HIP_TRY(h, tb.up<float>(&dy, nullptr, (size_t)rows * hidden, s));
    const float mult = scale ? (float)sqrt((double)hidden) : 1.0f;
    HIP_TRY(h, launch_embed_pe(de, dp, dp, stride, dsc, h->pe, mult, rows, hidden, dy, dsc + 1, s));
    HIP_TRY(h, hipMemcpyAsync(y, dy, (size_t)rows * hidden * 4, hipMemcpyDeviceToHost, s));
    HIP_TRY(h, hipStreamSynchronize(s));
    return ASR_OK;
}

int asr_op_pack_cross_kv(asr_handle* h, const float* kv, int32_t n, int32_t t, int32_t heads, int32_t as_bf16, void* k, void* v)
{
    if (!h || !kv || !k || !v || n < 1 || t < 1 || heads < 1 || heads > 64)
        return h ? fail(h, ASR_ERR_ARG, "bad argument") : ASR_ERR_ARG;
    int rc = set_device(h);
    if (rc) return rc;
    const size_t hidden = (size_t)heads * ASR_D_HEAD, cnt = (size_t)n * t * hidden, esz = as_bf16 ? 2 : 4;
    TmpBufs tb;
    float* dkv;
    char *dk, *dv;
    hipStream_t s = h->stream;
    HIP_TRY(h, tb.up(&dkv, kv, cnt * 2, s));
    HIP_TRY(h, tb.up<char>(&dk, nullptr, cnt * esz, s));
    HIP_TRY(h, tb.up<char>(&dv, nullptr, cnt * esz, s));
    HIP_TRY(h, launch_pack_cross_kv(dkv, n, t, heads, dk, dv, as_bf16 ? 1 : 0, nullptr, s));
    HIP_TRY(h, hipMemcpyAsync(k, dk, cnt * esz, hipMemcpyDeviceToHost, s));
    HIP_TRY(h, hipMemcpyAsync(v, dv, cnt * esz, hipMemcpyDeviceToHost, s));
    HIP_TRY(h, hipStreamSynchronize(s));
    return ASR_OK;
}

int asr_op_decoder_cross_attention(asr_handle* h, const float* q, const float* qbias, const float* kv, const int32_t* pad, int32_t n,
                                   int32_t t, int32_t heads, int32_t beams, int32_t variant, float* ctx, int32_t* range_flag)
{
    if (!h || !q || !qbias || !kv || !pad || !ctx || n < 1 || t < 1 || heads < 1 || heads > 64 || beams < 1 || beams > ASR_MAX_BEAM ||
        variant < 0 || variant > 2)
        return h ? fail(h, ASR_ERR_ARG, "bad argument") : ASR_ERR_ARG;
    int rc = set_device(h);
    if (rc) return rc;
    const size_t hidden = (size_t)heads * ASR_D_HEAD, rows = (size_t)n * t, cnt = rows * hidden, R = (size_t)n * beams;
    const size_t esz = variant == 2 ? 2 : 4, slack = (size_t)ASR_XATT_SLACK_ROWS * 64;
    TmpBufs tb;
    float *dq, *db, *dkv, *dctx;
    char *dk, *dv;
    int32_t *dpad, *dflags;
    hipStream_t s = h->stream;
    HIP_TRY(h, tb.up(&dq, q, R * hidden, s));
    HIP_TRY(h, tb.up(&db, qbias, hidden, s));
    HIP_TRY(h, tb.up(&dkv, kv, cnt * 2, s));
    HIP_TRY(h, tb.up<char>(&dk, nullptr, (cnt + slack) * esz, s));
    HIP_TRY(h, tb.up<char>(&dv, nullptr, (cnt + slack) * esz, s));
    HIP_TRY(h, tb.up<int32_t>(&dpad, nullptr, rows + ASR_XATT_SLACK_ROWS, s));
    HIP_TRY(h, tb.up<int32_t>(&dflags, nullptr, 2, s));                          // [0] done = 0, [1] range flag
    HIP_TRY(h, tb.up<float>(&dctx, nullptr, R * hidden, s));
    HIP_TRY(h, hipMemsetAsync(dflags, 0, 2 * sizeof(int32_t), s));
    HIP_TRY(h, hipMemsetAsync(dpad, 0, (rows + ASR_XATT_SLACK_ROWS) * sizeof(int32_t), s));
    HIP_TRY(h, hipMemcpyAsync(dpad, pad, rows * sizeof(int32_t), hipMemcpyHostToDevice, s));
    HIP_TRY(h, launch_pack_cross_kv(dkv, n, t, heads, dk, dv, variant == 2 ? 1 : 0, variant == 1 ? dflags + 1 : nullptr, s));
    CrossAttnArgs a{};
    a.qpart = dq; a.nsplit = 1; a.split_stride = 0; a.qbias = db;
    a.kc = dk; a.v = dv; a.kv_bf16 = variant == 2 ? 1 : 0;
    a.f16x3 = variant == 1 ? 1 : 0; a.range_flag = variant == 1 ? dflags + 1 : nullptr;
    a.pad2 = dpad; a.done = dflags; a.ctx = dctx; a.b = n; a.k = beams; a.heads = heads; a.t = t;
    HIP_TRY(h, launch_decoder_cross_attention(a, s));
    int32_t flags[2] = {0, 0};
    HIP_TRY(h, hipMemcpyAsync(ctx, dctx, R * hidden * sizeof(float), hipMemcpyDeviceToHost, s));
    HIP_TRY(h, hipMemcpyAsync(flags, dflags, sizeof(flags), hipMemcpyDeviceToHost, s));
    HIP_TRY(h, hipStreamSynchronize(s));
    if (range_flag) *range_flag = flags[1];
    return ASR_OK;
}

int asr_op_decoder_self_attention(asr_handle* h, const float* qkv, const float* bias, const float* hist_k, const float* hist_v,
                                  const int32_t* anc, int32_t n, int32_t pos, int32_t heads, int32_t beams, int32_t kv_bf16, float* ctx)
{
    if (!h || !qkv || !bias || !ctx || n < 1 || pos < 0 || pos > 4096 || heads < 1 || heads > 64 || beams < 1 || beams > ASR_MAX_BEAM ||
        (pos > 0 && (!hist_k || !hist_v || !anc)))
        return h ? fail(h, ASR_ERR_ARG, "bad argument") : ASR_ERR_ARG;
    const int K = beams, width = std::max(pos + 1, 2);
    if (kv_bf16 < 0 || kv_bf16 > 2) return fail(h, ASR_ERR_ARG, "variant must be 0 (float32), 1 (bf16 caches) or 2 (float32 caches, fp16x3 products)");
    const bool f16x3 = kv_bf16 == 2;
    if (f16x3) kv_bf16 = 0;
    const size_t hidden = (size_t)heads * ASR_D_HEAD, R = (size_t)n * K, esz = kv_bf16 ? 2 : 4;
    if (self_attention_lds_bytes(K, width) > 150 * 1024) return fail(h, ASR_ERR_CAPACITY, "beams x positions beyond the kernel's LDS tables");
    for (size_t i = 0; i < (size_t)n * K * pos; ++i)
        if (anc[i] < 0 || anc[i] >= K) return fail(h, ASR_ERR_ARG, "ancestor slot outside [0, beams)");
    int rc = set_device(h);
    if (rc) return rc;
    // host images of what the engine keeps on the device: head-major caches [n][heads][width][K][64], ancestry [n][K][width],
    // live rows (position << 5 | slot) of each utterance = the (position, slot) pairs some beam's ancestry names
    const size_t cache_elems = (size_t)n * heads * width * K * 64;
    std::vector<char> kc(cache_elems * esz, 0), vc(cache_elems * esz, 0);
    auto put = [&](std::vector<char>& dst, size_t idx, float x) {
        if (kv_bf16) {
            uint32_t u; memcpy(&u, &x, 4);
            const uint16_t b = (uint16_t)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);       // round to nearest even (finite inputs)
            memcpy(&dst[idx * 2], &b, 2);
        } else memcpy(&dst[idx * 4], &x, 4);
    };
    for (int u = 0; u < n; ++u)
        for (int j = 0; j < pos; ++j)
            for (int sl = 0; sl < K; ++sl)
                for (int hd = 0; hd < heads; ++hd)
                    for (int d = 0; d < 64; ++d) {
                        const size_t src = (((size_t)u * pos + j) * K + sl) * hidden + hd * 64 + d;
                        const size_t dst = ((((size_t)u * heads + hd) * width + j) * K + sl) * 64 + d;
                        put(kc, dst, hist_k[src]); put(vc, dst, hist_v[src]);
                    }
    std::vector<int32_t> anc_w((size_t)n * K * width, 0), live((size_t)n * K * width, 0), live_cnt(n, 0);
    // the live list in the order beam_step_kernel writes it: by position, and within a position by ascending slot
    for (int u = 0; u < n; ++u)
        for (int j = 0; j < pos; ++j) {
            uint32_t mask = 0;
            for (int b = 0; b < K; ++b) {
                const int sl = anc[((size_t)u * K + b) * pos + j];
                anc_w[((size_t)u * K + b) * width + j] = sl;
                mask |= 1u << sl;
            }
            for (int sl = 0; sl < 32; ++sl)
                if (mask & (1u << sl)) live[(size_t)u * K * width + live_cnt[u]++] = (j << 5) | sl;
        }
    TmpBufs tb;
    float *dqkv, *dbias, *dctx;
    char *dk, *dv;
    int32_t *danc, *dlive, *dcnt, *dflags;
    hipStream_t s = h->stream;
    HIP_TRY(h, tb.up(&dqkv, qkv, R * 3 * hidden, s));
    HIP_TRY(h, tb.up(&dbias, bias, 3 * hidden, s));
    HIP_TRY(h, tb.up(&dk, kc.data(), kc.size(), s));
    HIP_TRY(h, tb.up(&dv, vc.data(), vc.size(), s));
    HIP_TRY(h, tb.up(&danc, anc_w.data(), anc_w.size(), s));
    HIP_TRY(h, tb.up(&dlive, live.data(), live.size(), s));
    HIP_TRY(h, tb.up(&dcnt, live_cnt.data(), live_cnt.size(), s));
    const int32_t flags[2] = {pos, 0};                                            // [0] position, [1] done = 0
    HIP_TRY(h, tb.up(&dflags, flags, 2, s));
    HIP_TRY(h, tb.up<float>(&dctx, nullptr, R * hidden, s));
    SelfAttnArgs a{};
    a.qkv = dqkv; a.nsplit = 1; a.split_stride = 0; a.bias = dbias;
    a.kcache = dk; a.vcache = dv; a.kv_bf16 = kv_bf16 ? 1 : 0; a.f16x3 = f16x3 ? 1 : 0; a.range_flag = nullptr;
    a.anc0 = danc; a.anc1 = danc; a.live = dlive; a.live_cnt = dcnt; a.pos = dflags; a.done = dflags + 1;
    a.ctx = dctx; a.b = n; a.k = K; a.heads = heads; a.width = width; a.lds_stride = width;
    HIP_TRY(h, launch_decoder_self_attention(a, s));
    HIP_TRY(h, hipMemcpyAsync(ctx, dctx, R * hidden * sizeof(float), hipMemcpyDeviceToHost, s));
    HIP_TRY(h, hipStreamSynchronize(s));
    return ASR_OK;
}

int asr_op_input_norm_timing(asr_handle* h, const float* x, const float* gamma, const float* beta, int32_t n, int32_t t, int32_t hidden,
                             float* y)
{
    if (!h || !x || !gamma || !beta || !y || n < 1 || t < 1 || hidden != h->H)
        return h ? fail(h, ASR_ERR_ARG, "bad argument (hidden must equal the handle's hidden_units)") : ASR_ERR_ARG;
    int rc = set_device(h);
    if (rc) return rc;
    if ((rc = ensure_pe(h, t))) return rc;
    TmpBufs tb;
    float *dx, *dg, *db, *dy;
    double* dscr;
    hipStream_t s = h->stream;
    const size_t cnt = (size_t)n * t * hidden;
    HIP_TRY(h, tb.up(&dx, x, cnt, s));
    HIP_TRY(h, tb.up(&dg, gamma, (size_t)hidden, s));
    HIP_TRY(h, tb.up(&db, beta, (size_t)hidden, s));
    HIP_TRY(h, tb.up<float>(&dy, nullptr, cnt, s));
    HIP_TRY(h, tb.up<double>(&dscr, nullptr, input_norm_scratch_doubles(n, t, hidden), s));
    HIP_TRY(h, launch_input_norm_timing(dx, dg, db, h->pe, n, t, hidden, dscr, dy, s));
    HIP_TRY(h, hipMemcpyAsync(y, dy, cnt * 4, hipMemcpyDeviceToHost, s));
    HIP_TRY(h, hipStreamSynchronize(s));
    return ASR_OK;
}

// Allocation-free variant of asr_op_input_norm_timing (include/asr_amd.h): inputs and output are DEVICE pointers of this
// handle's GPU, the partial-sum scratch is the file-scope g_norm_scratch array (through the pointer asr_create resolved),
// the timing table is the one the handle already holds.  No hipMalloc / hipFree / allocating call on any path.
int asr_op_input_norm_timing_noalloc(asr_handle* h, const float* x_dev, const float* gamma_dev, const float* beta_dev, int32_t n, int32_t t,
                                     int32_t hidden, float* y_dev)
{
    if (!h) return ASR_ERR_ARG;
    if (!x_dev || !gamma_dev || !beta_dev || !y_dev || n < 1 || t < 1 || hidden != h->H)
        return fail(h, ASR_ERR_ARG, "bad argument (hidden must equal the handle's hidden_units)");
    if (n > NOALLOC_MAX_UTTS)
        return fail(h, ASR_ERR_CAPACITY, "asr_op_input_norm_timing_noalloc: n = " + std::to_string(n) + " exceeds the static scratch (" +
                                             std::to_string(NOALLOC_MAX_UTTS) + " utterances per call)");
    if (t > h->pe_rows)
        return fail(h, ASR_ERR_CAPACITY, "asr_op_input_norm_timing_noalloc: t = " + std::to_string(t) + " exceeds the handle's timing table (" +
                                             std::to_string(h->pe_rows) + " positions; this entry point cannot grow it)");
    if ((reinterpret_cast<uintptr_t>(x_dev) | reinterpret_cast<uintptr_t>(gamma_dev) | reinterpret_cast<uintptr_t>(beta_dev) |
         reinterpret_cast<uintptr_t>(y_dev)) & 15)
        return fail(h, ASR_ERR_ARG, "device pointers must be 16-byte aligned");
    int rc = set_device(h);
    if (rc) return rc;
    // a host pointer here would fault the GPU: every pointer must be device memory of this handle's device
    const void* ptrs[4] = {x_dev, gamma_dev, beta_dev, y_dev};
    for (const void* q : ptrs) {
        hipPointerAttribute_t at{};
        if (hipPointerGetAttributes(&at, q) != hipSuccess || (at.type != hipMemoryTypeDevice && at.type != hipMemoryTypeManaged) ||
            (at.type == hipMemoryTypeDevice && at.device != h->cfg.device)) {
            (void)hipGetLastError();
            return fail(h, ASR_ERR_ARG, "asr_op_input_norm_timing_noalloc takes device pointers of the handle's GPU");
        }
    }
    double* scratch = g_norm_scratch_ptr[h->cfg.device];
    if (!scratch) return fail(h, ASR_ERR_STATE, "static scratch was not resolved on this device");
    static_assert(NOALLOC_DOUBLES_PER_UTT == 128, "rowops.hip: 2 x 64 partial sums per utterance");
    if (input_norm_scratch_doubles(n, t, hidden) > (size_t)NOALLOC_MAX_UTTS * NOALLOC_DOUBLES_PER_UTT)
        return fail(h, ASR_ERR_CAPACITY, "static scratch too small");
    // Nothing in the scratch has to start at zero: the first statistics kernel writes every slot the later ones read
    // (rowops.hip input_norm_stats_kernel), so the previous call's contents are simply overwritten.
    // One array per GPU: handles of that GPU on other host threads wait here for their turn (the call blocks anyway).
    std::lock_guard<std::mutex> lock(g_norm_scratch_mu[h->cfg.device]);
    HIP_TRY(h, launch_input_norm_timing(x_dev, gamma_dev, beta_dev, h->pe, n, t, hidden, scratch, y_dev, h->stream));
    HIP_TRY(h, hipStreamSynchronize(h->stream));
    return ASR_OK;
}

static int asr_op_encoder_attention_once(asr_handle* h, const float* qkv, const int32_t* pad, int32_t n, int32_t t, float* ctx)
{
    int rc = set_device(h);
    if (rc) return rc;
    TmpBufs tb;
    float *dq, *dc;
    int32_t* dp;
    hipStream_t s = h->stream;
    const size_t rows = (size_t)n * t;
    HIP_TRY(h, tb.up(&dq, qkv, rows * 3 * h->H, s));
    HIP_TRY(h, tb.up(&dp, pad, rows, s));
    HIP_TRY(h, tb.up<float>(&dc, nullptr, rows * h->H, s));
    HIP_TRY(h, launch_encoder_attention(dq, dp, n, t, h->heads, dc, mha_mode(h), h->range_flag, s));
    HIP_TRY(h, hipMemcpyAsync(ctx, dc, rows * h->H * 4, hipMemcpyDeviceToHost, s));
    HIP_TRY(h, hipStreamSynchronize(s));
    return ASR_OK;
}

int asr_op_encoder_attention(asr_handle* h, const float* qkv, const int32_t* pad, int32_t n, int32_t t, float* ctx)
{
    if (!h || !qkv || !pad || !ctx || n < 1 || t < 1) return h ? fail(h, ASR_ERR_ARG, "bad argument") : ASR_ERR_ARG;
    // (fp16x3 mode: q, k or v outside fp16's range -> repeated on the exact-f32 matrix instruction, like a whole decode)
    return with_range_retry(h, [&]() { return asr_op_encoder_attention_once(h, qkv, pad, n, t, ctx); });
}

int asr_op_log_softmax_topk(asr_handle* h, const float* logits, int32_t rows, int32_t vocab, int32_t k, float* values, int32_t* indices)
{
    if (!h || !logits || !values || !indices || rows < 1 || vocab < 1 || k < 1 || k > vocab || k > ASR_MAX_BEAM)
        return h ? fail(h, ASR_ERR_ARG, "bad argument") : ASR_ERR_ARG;
    int rc = set_device(h);
    if (rc) return rc;
    TmpBufs tb;
    float *dl, *dv;
    int32_t* di;
    hipStream_t s = h->stream;
    HIP_TRY(h, tb.up(&dl, logits, (size_t)rows * vocab, s));
    HIP_TRY(h, tb.up<float>(&dv, nullptr, (size_t)rows * k, s));
    HIP_TRY(h, tb.up<int32_t>(&di, nullptr, (size_t)rows * k, s));
    HIP_TRY(h, launch_log_softmax_topk(dl, 1, 0, rows, vocab, k, dv, di, nullptr, s));
    HIP_TRY(h, hipMemcpyAsync(values, dv, (size_t)rows * k * 4, hipMemcpyDeviceToHost, s));
    HIP_TRY(h, hipMemcpyAsync(indices, di, (size_t)rows * k * 4, hipMemcpyDeviceToHost, s));
    HIP_TRY(h, hipStreamSynchronize(s));
    return ASR_OK;
}

int asr_op_beam_step(asr_handle* h, const float* scores, const int32_t* finished, const float* cand_scores, const int32_t* cand_tokens,
                     int32_t b, int32_t k, float* new_scores, int32_t* tokens, int32_t* parents, int32_t* finished_out)
{
    if (!h || !scores || !finished || !cand_scores || !cand_tokens || !new_scores || !tokens || !parents || !finished_out || b < 1 ||
        k < 1 || k > ASR_MAX_BEAM)
        return h ? fail(h, ASR_ERR_ARG, "bad argument") : ASR_ERR_ARG;
    int rc = set_device(h);
    if (rc) return rc;
    TmpBufs tb;
    float *ds, *dcs, *dns;
    int32_t *df, *dct, *dt, *dp, *dfo;
    hipStream_t s = h->stream;
    const size_t R = (size_t)b * k;
    HIP_TRY(h, tb.up(&ds, scores, R, s));
    HIP_TRY(h, tb.up(&df, finished, R, s));
    HIP_TRY(h, tb.up(&dcs, cand_scores, R * k, s));
    HIP_TRY(h, tb.up(&dct, cand_tokens, R * k, s));
    HIP_TRY(h, tb.up<float>(&dns, nullptr, R, s));
    HIP_TRY(h, tb.up<int32_t>(&dt, nullptr, R, s));
    HIP_TRY(h, tb.up<int32_t>(&dp, nullptr, R, s));
    HIP_TRY(h, tb.up<int32_t>(&dfo, nullptr, R, s));
    HIP_TRY(h, launch_beam_prune(ds, df, dcs, dct, b, k, dns, dt, dp, dfo, s));
    HIP_TRY(h, hipMemcpyAsync(new_scores, dns, R * 4, hipMemcpyDeviceToHost, s));
    HIP_TRY(h, hipMemcpyAsync(tokens, dt, R * 4, hipMemcpyDeviceToHost, s));
    HIP_TRY(h, hipMemcpyAsync(parents, dp, R * 4, hipMemcpyDeviceToHost, s));
    HIP_TRY(h, hipMemcpyAsync(finished_out, dfo, R * 4, hipMemcpyDeviceToHost, s));
    HIP_TRY(h, hipStreamSynchronize(s));
    return ASR_OK;
}

// ---- instrumentation ---------------------------------------------------------------------------
int asr_set_profile(asr_handle* h, int32_t mode)
{
    if (!h) return ASR_ERR_ARG;
    if (h->profile == 2) prof_drain(h, true);
    h->profile = mode == 2 ? 2 : mode ? 1 : 0;
    if (mode) {
        h->prof.clear();
        // An event pair brackets the kernel AND the completion signalling of its own two markers; calibrate that
        // part on an empty pair (median of 33) so that per-kernel times agree with rocprofv3's dispatch durations.
        int rc = set_device(h);
        if (rc) return rc;
        std::vector<float> v;
        if (h->profile == 2) {                                     // pairs queued back to back, as the brackets of this mode are
            std::vector<hipEvent_t> ev;
            for (int i = 0; i < 66; ++i) ev.push_back(prof_event(h));
            for (hipEvent_t e : ev) if (!e) return fail(h, ASR_ERR_HIP, "hipEventCreate failed");
            for (int i = 0; i < 66; ++i) HIP_TRY(h, hipEventRecord(ev[i], h->stream));
            HIP_TRY(h, hipEventSynchronize(ev[65]));
            for (int i = 0; i < 66; i += 2) {
                float ms = 0.f;
                HIP_TRY(h, hipEventElapsedTime(&ms, ev[i], ev[i + 1]));
                v.push_back(ms);
            }
            for (hipEvent_t e : ev) h->prof_free.push_back(e);
        }
        for (int i = 0; i < 33 && h->profile == 1; ++i) {
            HIP_TRY(h, hipEventRecord(h->pe0, h->stream));
            HIP_TRY(h, hipEventRecord(h->pe1, h->stream));
            HIP_TRY(h, hipEventSynchronize(h->pe1));
            float ms = 0.f;
            HIP_TRY(h, hipEventElapsedTime(&ms, h->pe0, h->pe1));
            v.push_back(ms);
        }
        std::sort(v.begin(), v.end());
        h->prof_overhead_ms = v[v.size() / 2];
    }
    return ASR_OK;
}

int asr_get_profile(asr_handle* h, int32_t cap, const char** names, double* ms, int64_t* launches, double* flops, double* bytes,
                    int32_t* n_out)
{
    if (!h || !n_out) return ASR_ERR_ARG;
    if (h->profile == 2 && set_device(h) == ASR_OK) prof_drain(h, true);
    int n = std::min<int>(cap, (int)h->prof.size());
    int64_t total = 0;
    for (int i = 0; i < n; ++i) {
        if (names) names[i] = h->prof[i].name;
        if (ms) ms[i] = h->prof[i].ms;
        if (launches) launches[i] = h->prof[i].launches;
        if (flops) flops[i] = h->prof[i].flops;
        if (bytes) bytes[i] = h->prof[i].bytes;
        total += h->prof[i].launches;
    }
    if (n < cap && n > 0) {                                        // what was subtracted, as a pseudo class
        if (names) names[n] = "(event_pair_overhead)";
        if (ms) ms[n] = h->prof_overhead_ms * (double)total;
        if (launches) launches[n] = total;
        if (flops) flops[n] = 0.0;
        if (bytes) bytes[n] = 0.0;
        ++n;
    }
    *n_out = n;
    return ASR_OK;
}

int64_t asr_device_bytes(const asr_handle* h)
{
    if (!h) return 0;
    return h->dev_bytes + ((h->wstore && h->wstore_owner) ? h->wstore->bytes : 0);
}

int64_t asr_range_retries(const asr_handle* h) { return h ? h->range_retries : 0; }

// crc32c (Castagnoli), slicing-by-8 on the host: the tensor / block checksum of TF-V2 checkpoints
uint32_t asr_crc32c(const void* data, int64_t n, uint32_t crc)
{
    static uint32_t T[8][256];
    static std::once_flag init;
    std::call_once(init, [] {
        for (uint32_t i = 0; i < 256; ++i) {
            uint32_t c = i;
            for (int k = 0; k < 8; ++k) c = (c & 1) ? (c >> 1) ^ 0x82F63B78u : c >> 1;
            T[0][i] = c;
        }
        for (uint32_t i = 0; i < 256; ++i)
            for (int s = 1; s < 8; ++s) T[s][i] = (T[s - 1][i] >> 8) ^ T[0][T[s - 1][i] & 0xFF];
    });
    const uint8_t* p = static_cast<const uint8_t*>(data);
    uint32_t c = ~crc;
    while (n >= 8) {
        uint32_t lo, hi;
        memcpy(&lo, p, 4);
        memcpy(&hi, p + 4, 4);
        lo ^= c;
        c = T[7][lo & 0xFF] ^ T[6][(lo >> 8) & 0xFF] ^ T[5][(lo >> 16) & 0xFF] ^ T[4][lo >> 24] ^
            T[3][hi & 0xFF] ^ T[2][(hi >> 8) & 0xFF] ^ T[1][(hi >> 16) & 0xFF] ^ T[0][hi >> 24];
        p += 8; n -= 8;
    }
    while (n-- > 0) c = T[0][(c ^ *p++) & 0xFF] ^ (c >> 8);
    return ~c;
}

}  // extern "C"
