// Operators on device memory, row by row: log probabilities of given tokens with entropy and alternatives, and the writer of the
// 8-bit K/V cache.  C entry points: include/asr_amd.h.
#include "ops_common.h"

#include <stdarg.h>
#include <stdio.h>

namespace {

thread_local char g_ops_error[256] = "";

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr float LOG2E = 1.44269504088896340736f;
constexpr float NEG_INF = -__builtin_inff();

}  // namespace

int ops_fail(int code, const char* fmt, ...)
{
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_ops_error, sizeof g_ops_error, fmt, ap);
    va_end(ap);
    return code;
}

int ops_launched(const char* what, hipError_t e)
{
    if (e == hipSuccess) return ASR_OK;
    (void)hipGetLastError();
    return ops_fail(ASR_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}

namespace {

// ---- token_logprobs ----------------------------------------------------------------------------------------------------
// One workgroup per row, one pass over its logits: every thread keeps the running maximum m, S = sum e^(x-m) and T = sum e^(x-m) (x-m) of its
// strip (rescaled when the maximum of a group of loads beats m), the workgroup joins them, and
//     log p(t) = x_t - m - ln S,      H = ln S - T / S
// (both terms of H are >= 0: nothing cancels).  The difference x - m is taken before the factor log2(e), so that large logits lose nothing.
// The alternatives come without a second pass over the row: the strips' maxima are joined to 64 groups', a bound that the maxima of at least `top` and
// hardly more groups reach is found by bisection over them (one wave, a ballot a step); only the strips whose own maximum reaches it are read again
// (by the whole workgroup, from the cache), what reaches the bound is collected (usually little more than `top` values) and ranked.  Where that does not fit the list - masked rows of fewer than `top` admitted
// tokens, equal logits, the likeliest tokens all in a few strips - the alternatives are taken one by one instead.

__device__ inline float bf16_lo(uint32_t u) { return __uint_as_float(u << 16); }
__device__ inline float bf16_hi(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }

template <int DT> struct Elem;
template <> struct Elem<ASR_F32> {
    typedef float T;
    static constexpr int PER = 4;
    static constexpr uint32_t NONE = 0xff800000u;              // -infinity in every place of a word
    static __device__ float one(const float* p) { return *p; }
    static __device__ void unpack(const u32x4& r, float* x)
    {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(r[i]);
    }
};
template <> struct Elem<ASR_BF16> {
    typedef uint16_t T;
    static constexpr int PER = 8;
    static constexpr uint32_t NONE = 0xff80ff80u;
    static __device__ float one(const uint16_t* p) { return __uint_as_float((uint32_t)*p << 16); }
    static __device__ void unpack(const u32x4& r, float* x)
    {
#pragma unroll
        for (int i = 0; i < 4; ++i) { x[2 * i] = bf16_lo(r[i]); x[2 * i + 1] = bf16_hi(r[i]); }
    }
};
template <> struct Elem<ASR_F16> {
    typedef _Float16 T;
    static constexpr int PER = 8;
    static constexpr uint32_t NONE = 0xfc00fc00u;
    static __device__ float one(const _Float16* p) { return (float)*p; }
    static __device__ void unpack(const u32x4& r, float* x)
    {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int i = 0; i < 4; ++i) { const uint32_t w = r[i]; const h2 v = __builtin_bit_cast(h2, w); x[2 * i] = (float)v[0]; x[2 * i + 1] = (float)v[1]; }
    }
};

// order of logits as unsigned numbers: -0 counts as +0, NaN above everything
__device__ inline uint32_t ordered(float x)
{
    if (x != x) return 0xffffffffu;
    const uint32_t b = __float_as_uint(x + 0.0f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ inline float unordered(uint32_t o)
{
    if (o == 0xffffffffu) return __builtin_nanf("");
    return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}
// (logit, token) as one key: the larger logit first, the lower token among equals; 0 = none
__device__ inline uint64_t key_of(float x, int idx) { return ((uint64_t)ordered(x) << 32) | (uint32_t)~idx; }

struct Stats { float m, s, t; };

__device__ inline float base_of(float m) { return m == NEG_INF ? 0.0f : m; }      // (a strip without an admitted token: e^(-inf - 0) = 0)

// a's sums brought to the maximum m (m >= a.m).  A difference of -infinity belongs to sums of 0: it is held finite so that 0 stays 0.
__device__ inline Stats at_max(const Stats& a, float m)
{
    const float d = fmaxf(base_of(a.m) - base_of(m), -1e30f);
    const float f = a.m == NEG_INF ? (a.s == a.s ? 0.0f : a.s) : __builtin_amdgcn_exp2f(d * LOG2E);
    Stats r;
    r.m = m;
    r.s = a.m == NEG_INF ? f : a.s * f;
    r.t = a.m == NEG_INF ? f : (a.t + a.s * d) * f;
    return r;
}

// maximum / sum over a wave: rotations inside rows of 16 lanes, then the rows
template <int CTRL> __device__ inline float rotated(float x)
{
    return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), CTRL, 0xf, 0xf, true));
}
template <typename F> __device__ inline float row_reduce(float x, F f)
{
    x = f(x, rotated<0x128>(x));
    x = f(x, rotated<0x124>(x));
    x = f(x, rotated<0x122>(x));
    return f(x, rotated<0x121>(x));
}
template <typename F> __device__ inline float wave_reduce(float x, F f)
{
    x = row_reduce(x, f);
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = f(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return f(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
struct Max { __device__ float operator()(float a, float b) const { return fmaxf(a, b); } };
struct Sum { __device__ float operator()(float a, float b) const { return a + b; } };

template <int N> __device__ inline void add_group(Stats& st, const float* x)
{
    float gm = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) gm = fmaxf(gm, x[i]);
    if (gm > st.m) st = at_max(st, gm);
    const float m = base_of(st.m);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float d = x[i] - m;
        const float e = __builtin_amdgcn_exp2f(d * LOG2E);
        st.s += e;
        st.t = fmaf(e, fmaxf(d, -1e30f), st.t);
    }
}

// chunks c, c + NT, ... (N of them, those below `chunks`) of a row: loaded together, then added
template <int DT, int NT, int N> __device__ inline void add_chunks(Stats& st, const u32x4* v, int c, int chunks)
{
    constexpr int PER = Elem<DT>::PER;
    u32x4 raw[N];
#pragma unroll
    for (int u = 0; u < N; ++u) {
        raw[u] = u32x4{Elem<DT>::NONE, Elem<DT>::NONE, Elem<DT>::NONE, Elem<DT>::NONE};
        if (c + u * NT < chunks) raw[u] = v[c + u * NT];
    }
    float x[N * PER];
#pragma unroll
    for (int u = 0; u < N; ++u) Elem<DT>::unpack(raw[u], x + u * PER);
    add_group<N * PER>(st, x);
}

__device__ inline uint64_t shfl_max_u64(uint64_t v)
{
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        const uint64_t w = __shfl_xor((unsigned long long)v, o, 64);
        v = w > v ? w : v;
    }
    return v;
}

// Every element of thread `tid`'s strip, f(x, index): the head up to the first 16-byte boundary, 16-byte chunks tid, tid + NT, ..., the tail
template <int DT, int NT, typename F> __device__ inline void for_strip(const typename Elem<DT>::T* row, int vocab, int head, int tid, F f)
{
    constexpr int PER = Elem<DT>::PER;
    const int chunks = (vocab - head) / PER, body = head + chunks * PER;
    if (tid < head) f(Elem<DT>::one(row + tid), tid);
    const u32x4* v = reinterpret_cast<const u32x4*>(row + head);
    for (int c = tid; c < chunks; c += NT) {
        float x[PER];
        Elem<DT>::unpack(v[c], x);
#pragma unroll
        for (int i = 0; i < PER; ++i) f(x[i], head + c * PER + i);
    }
    if (tid < vocab - body) f(Elem<DT>::one(row + body + tid), body + tid);
}

struct TokenLogprobsArgs {
    const void* logits;
    const void* tokens;
    float *logprob, *entropy, *top_logprobs;
    int32_t* top_tokens;
    int64_t rows, row_stride;
    int vocab, top, token_bytes;
};

constexpr int MAX_TOP = 32;
constexpr int MAX_CANDIDATES = 512;
constexpr int MAX_GRID = 1 << 20;        // workgroups; further rows are taken in turn

template <int DT, int NT> __global__ __launch_bounds__(NT) void token_logprobs_kernel(TokenLogprobsArgs a)
{
    typedef typename Elem<DT>::T T;
    constexpr int PER = Elem<DT>::PER, NW = NT / 64;
    __shared__ float red[3][NW];
    __shared__ uint64_t wkey[NW], cand[MAX_CANDIDATES];
    constexpr int GS = NT / 64;                                          // threads of a group; 64 groups
    __shared__ uint32_t group_max[64], bound;
    __shared__ uint16_t strips[NT];
    __shared__ int n_strips, n_cand;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* row = static_cast<const T*>(a.logits) + r * a.row_stride;
        const int head = min(a.vocab, (int)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / (int)sizeof(T));
        const int chunks = (a.vocab - head) / PER, body = head + chunks * PER;
        // asked for first: the token's own logit and what lies outside the 16-byte chunks
        const int64_t token = a.token_bytes == 8 ? static_cast<const int64_t*>(a.tokens)[r] : (int64_t) static_cast<const int32_t*>(a.tokens)[r];
        const bool in = token >= 0 && token < a.vocab;
        const float x_token = Elem<DT>::one(row + (in ? token : 0));
        float ends[2] = {NEG_INF, NEG_INF};
        if (tid < head) ends[0] = Elem<DT>::one(row + tid);
        if (tid < a.vocab - body) ends[1] = Elem<DT>::one(row + body + tid);
        const u32x4* v = reinterpret_cast<const u32x4*>(row + head);
        Stats st{NEG_INF, 0.0f, 0.0f};
        int c0 = 0;
        for (; chunks - c0 > 2 * NT; c0 += 4 * NT) add_chunks<DT, NT, 4>(st, v, c0 + tid, chunks);
        if (chunks - c0 > NT) add_chunks<DT, NT, 2>(st, v, c0 + tid, chunks);
        else if (chunks > c0) add_chunks<DT, NT, 1>(st, v, c0 + tid, chunks);
        add_group<2>(st, ends);
        // the waves' sums under the waves' maxima, then the workgroup's
        Stats w = at_max(st, wave_reduce(st.m, Max()));
        w.s = wave_reduce(w.s, Sum());
        w.t = wave_reduce(w.t, Sum());
        if (lane == 0) { red[0][wave] = w.m; red[1][wave] = w.s; red[2][wave] = w.t; }
        float gm = st.m;
#pragma unroll
        for (int o = 1; o < GS; o *= 2) gm = fmaxf(gm, __shfl_xor(gm, o, 64));
        if (tid % GS == 0) group_max[tid / GS] = ordered(gm);
        __syncthreads();
        const int l16 = lane & 15;                                       // every 16 lanes join the (at most 16) waves' sums
        w = l16 < NW ? Stats{red[0][l16], red[1][l16], red[2][l16]} : Stats{NEG_INF, 0.0f, 0.0f};
        Stats all = at_max(w, row_reduce(w.m, Max()));
        all.s = row_reduce(all.s, Sum());
        all.t = row_reduce(all.t, Sum());
        const bool none = all.m == NEG_INF && all.s == 0.0f;             // every token is masked out
        const float m = base_of(all.m), log_s = logf(all.s);
        if (tid == 0) {
            const float lp = token < 0 ? 0.0f : !in ? __builtin_nanf("") : none ? NEG_INF : (x_token - m) - log_s;
            a.logprob[r] = lp;
            a.entropy[r] = none ? 0.0f : log_s - all.t / all.s;
        }
        if (a.top > 0) {
            if (wave == 0) {
                const uint32_t mine = group_max[lane];
                uint32_t thr = 0;
                for (uint32_t bit = 0x80000000u; bit; bit >>= 1) {
                    const int n = __popcll(__ballot(mine >= (thr | bit)));
                    if (n >= a.top) {
                        thr |= bit;
                        if (n <= a.top + 2) break;
                    }
                }
                if (lane == 0) { bound = thr; n_strips = 0; n_cand = 0; }
            }
            __syncthreads();
            const uint32_t thr = bound;
            if (ordered(st.m) >= thr) strips[atomicAdd(&n_strips, 1)] = (uint16_t)tid;
            __syncthreads();
            const auto collect = [&](float x, int i) {
                if (ordered(x) >= thr) {
                    const int at = atomicAdd(&n_cand, 1);
                    if (at < MAX_CANDIDATES) cand[at] = key_of(x, i);
                }
            };
            const int per_strip = (chunks + NT - 1) / NT, total = n_strips * per_strip;
            for (int i = tid; i < total; i += NT) {
                const int c = strips[i / per_strip] + i % per_strip * NT;
                if (c < chunks) {
                    float x[PER];
                    Elem<DT>::unpack(v[c], x);
#pragma unroll
                    for (int j = 0; j < PER; ++j) collect(x[j], head + c * PER + j);
                }
            }
            if (tid < head) collect(ends[0], tid);
            if (tid < a.vocab - body) collect(ends[1], body + tid);
            __syncthreads();
            const int found = n_cand;
            if (found <= MAX_CANDIDATES) {
                for (int i = tid; i < found; i += NT) {
                    const uint64_t key = cand[i];
                    int rank = 0;
                    for (int j = 0; j < found; ++j) rank += cand[j] > key;
                    if (rank < a.top) {
                        a.top_tokens[r * a.top + rank] = (int32_t) ~(uint32_t)key;
                        a.top_logprobs[r * a.top + rank] = none ? NEG_INF : (unordered((uint32_t)(key >> 32)) - m) - log_s;
                    }
                }
            } else {
                // One alternative a round: the workgroup's largest key; its owner then looks for the next one of its strip.
                uint64_t mine = 0;
                for_strip<DT, NT>(row, a.vocab, head, tid, [&](float x, int i) { const uint64_t k = key_of(x, i); mine = k > mine ? k : mine; });
                for (int j = 0; j < a.top; ++j) {
                    const uint64_t best = shfl_max_u64(mine);
                    if (lane == 0) wkey[wave] = best;
                    __syncthreads();
                    uint64_t win = wkey[0];
#pragma unroll
                    for (int i = 1; i < NW; ++i) win = wkey[i] > win ? wkey[i] : win;
                    __syncthreads();
                    if (tid == 0) {
                        a.top_tokens[r * a.top + j] = (int32_t) ~(uint32_t)win;
                        a.top_logprobs[r * a.top + j] = none ? NEG_INF : (unordered((uint32_t)(win >> 32)) - m) - log_s;
                    }
                    if (mine == win && j + 1 < a.top) {
                        uint64_t next = 0;
                        for_strip<DT, NT>(row, a.vocab, head, tid, [&](float x, int i) {
                            const uint64_t k = key_of(x, i);
                            next = (k < win && k > next) ? k : next;
                        });
                        mine = next;
                    }
                }
            }
        }
        __syncthreads();                                             // (the next row uses red again)
    }
}

template <int DT> hipError_t run_token_logprobs(const TokenLogprobsArgs& k, hipStream_t s)
{
    const dim3 grid((uint32_t)(k.rows < MAX_GRID ? k.rows : MAX_GRID));
    // Few long rows: a row's loads wait for one another, so more threads share it (64 x 28444 bf16: 9.2 us with 256 threads, 7.5 with 1024; with 1024
    // rows 19 and 29: there the rows fill the chip, and a wider workgroup only has more to join)
    if (k.rows <= 256 && k.vocab / Elem<DT>::PER >= 2048) return ops_launch(token_logprobs_kernel<DT, 1024>, grid, dim3(1024), s, k);
    // Short rows: one wave has a few loads for each thread and meets nobody, and its 64 strips are the groups of the bound - spread over 256 threads they fill so
    // few groups that most of the row becomes candidates (2991 x 197 f32, top 13: 36 us with 256 threads, 7.3 with 64; 3000 x 2000 bf16, top 10: 13.4 and 9;
    // 100 x 1000 bf16, top 32: 56 and 8.7; 10 x 1000 f32: 5.5 and 5.4).  Longer ones too where there are
    // rows enough for every wave (20000 x 3000 bf16: 62 and 32; 3000 x 7000: 16.4 and 14.7; but 200 x 4000: 6.4 and 7.7)
    if (k.vocab / Elem<DT>::PER <= (k.rows >= 1024 ? 1024 : 256)) return ops_launch(token_logprobs_kernel<DT, 64>, grid, dim3(64), s, k);
    return ops_launch(token_logprobs_kernel<DT, 256>, grid, dim3(256), s, k);
}

}  // namespace

int ops_token_logprobs(const asr_token_logprobs_args& a, hipStream_t s)
{
    if (a.rows < 0) return ops_fail(ASR_ERR_ARG, "token_logprobs: negative rows");
    if (a.vocab < 1 || a.vocab > (1 << 30)) return ops_fail(ASR_ERR_ARG, "token_logprobs: vocab must be in 1..2^30");
    if (a.top < 0 || a.top > MAX_TOP || a.top > a.vocab) return ops_fail(ASR_ERR_ARG, "token_logprobs: top must be in 0..min(%d, vocab)", MAX_TOP);
    if (!ops_dtype_ok(a.dtype)) return ops_fail(ASR_ERR_ARG, "token_logprobs: unknown dtype %d", a.dtype);
    if (a.token_bytes != 4 && a.token_bytes != 8) return ops_fail(ASR_ERR_ARG, "token_logprobs: token_bytes must be 4 or 8");
    if (a.rows > 1 && a.row_stride < 0) return ops_fail(ASR_ERR_ARG, "token_logprobs: negative row stride");
    if (a.rows == 0) return ASR_OK;
    if (!a.logits || !a.tokens || !a.logprob || !a.entropy || (a.top > 0 && (!a.top_logprobs || !a.top_tokens)))
        return ops_fail(ASR_ERR_ARG, "token_logprobs: null argument");
    if (reinterpret_cast<uintptr_t>(a.logits) % ops_dtype_size(a.dtype)) return ops_fail(ASR_ERR_ARG, "token_logprobs: logits are not aligned to their type");
    const TokenLogprobsArgs k{a.logits, a.tokens, a.logprob, a.entropy, a.top_logprobs, a.top_tokens, a.rows, a.row_stride, a.vocab, a.top, a.token_bytes};
    return ops_launched("token_logprobs", a.dtype == ASR_F32 ? run_token_logprobs<ASR_F32>(k, s)
                                          : a.dtype == ASR_BF16 ? run_token_logprobs<ASR_BF16>(k, s) : run_token_logprobs<ASR_F16>(k, s));
}

namespace {

// ---- kv8_append --------------------------------------------------------------------------------------------------------
// One workgroup per (64-token block that may get tokens, sequence and head, K or V): the new tokens' magnitudes -> the block's
// exponent -> codes.  The scale is 2^e with the smallest e that keeps the magnitudes within 448 = 1.75 * 2^8, found in the bits of the largest one;
// dividing by a power of two is exact, so a value is rounded once.  Moving bytes bounds it: each new value is read once, into registers, each code written
// once.  Neighbouring workgroups take the heads of the same tokens, which lie side by side in the projection's output.
constexpr int KV8_MIN_EXP = -100;

__device__ inline int kv8_exponent(uint32_t magnitude)          // of a finite float's bits without sign
{
    const int p = (int)(magnitude >> 23) - 127;                 // amax = 1.f * 2^p (subnormals: far below the smallest exponent)
    const int e = (magnitude & 0x7fffffu) <= 0x600000u ? p - 8 : p - 7;
    return max(e, KV8_MIN_EXP);
}
__device__ inline float pow2f(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }      // -126 <= e <= 127

// the largest code under a scale of 2^e: 448, but under 2^120, which only magnitudes from 1.75 * 2^127 need, 256 would already stand for 2^128
__device__ inline float kv8_most(int e) { return e < 120 ? 448.0f : 240.0f; }
// four e4m3 codes of x * inv: infinities saturate (a code conversion of anything beyond 464 would give NaN), NaN passes
__device__ inline float kv8_clamp(float x, float most) { return x != x ? x : __builtin_amdgcn_fmed3f(x, -most, most); }
__device__ inline uint32_t kv8_codes(float x0, float x1, float x2, float x3, float most)
{
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(kv8_clamp(x0, most), kv8_clamp(x1, most), 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(kv8_clamp(x2, most), kv8_clamp(x3, most), r, true);
}

struct Kv8AppendArgs {
    const void* x[2];                    // k, v
    uint8_t* cache[2];
    float* scale[2];
    const int32_t *lens, *counts;
    int64_t stride[2][3];
    int64_t cache_stride[2];
    int new_tokens, kv_heads, d, capacity;
};

// NT threads, each with up to ITEMS 16-byte loads of the block's new tokens
template <int DT, int NT, int ITEMS> __global__ __launch_bounds__(NT) void kv8_append_kernel(Kv8AppendArgs a)
{
    typedef typename Elem<DT>::T T;
    constexpr int PER = Elem<DT>::PER, NW = NT / 64;
    __shared__ uint32_t top_bits[NW];
    const int which = (int)blockIdx.x >= a.kv_heads, h = blockIdx.x - (which ? a.kv_heads : 0), b = blockIdx.z;
    const int held = a.lens[b];
    if (held < 0 || held >= a.capacity) return;
    const int count = a.counts ? min(a.counts[b], a.new_tokens) : a.new_tokens;
    const int end = (int)min((int64_t)a.capacity, (int64_t)held + count);        // positions held .. end get tokens
    const int block = held / ASR_KV8_BLOCK + blockIdx.y;
    if (block >= a.capacity / ASR_KV8_BLOCK) return;
    const int first = block * ASR_KV8_BLOCK;
    const int lo = max(held, first), hi = min(end, first + ASR_KV8_BLOCK);
    if (lo >= hi) return;
    const int tid = threadIdx.x, per_row = a.d / PER, items = (hi - lo) * per_row;
    const T* x = static_cast<const T*>(a.x[which]) + (int64_t)b * a.stride[which][0] + (int64_t)h * a.stride[which][2] + (int64_t)(lo - held) * a.stride[which][1];
    uint8_t* codes = a.cache[which] + (int64_t)b * a.cache_stride[0] + (int64_t)h * a.cache_stride[1] + (int64_t)first * a.d;
    float* scale = a.scale[which] + ((int64_t)b * a.kv_heads + h) * (a.capacity / ASR_KV8_BLOCK) + block;
    const float was = *scale;

    u32x4 raw[ITEMS];
#pragma unroll
    for (int u = 0; u < ITEMS; ++u) {
        const int i = tid + u * NT, t = i / per_row, c = i - t * per_row;
        raw[u] = i < items ? *reinterpret_cast<const u32x4*>(x + (int64_t)t * a.stride[which][1] + c * PER) : u32x4{};
    }
    uint32_t most = 0;
#pragma unroll
    for (int u = 0; u < ITEMS; ++u) {
        float y[PER];
        Elem<DT>::unpack(raw[u], y);
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const uint32_t m = __float_as_uint(y[j]) & 0x7fffffffu;
            most = max(most, m < 0x7f800000u ? m : 0u);
        }
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) most = max(most, (uint32_t)__shfl_xor((int)most, o, 64));
    if (NW > 1) {
        if ((tid & 63) == 0) top_bits[tid >> 6] = most;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NW; ++i) most = max(most, top_bits[i]);
    }
    int e = kv8_exponent(most);
    if (held > first) {                                              // the block holds older tokens: its scale only grows
        const int e_was = min(max((int)(__float_as_uint(was) >> 23) - 127, KV8_MIN_EXP), 120);
        if (e > e_was) {
            // the older tokens under the new scale (a power of two lower: exact unless a code becomes subnormal)
            const float f = pow2f(max(e_was - e, -126));
            uint32_t* old = reinterpret_cast<uint32_t*>(codes);
            for (int i = tid; i < (held - first) * a.d / 4; i += NT) {
                const uint32_t c = old[i];
                typedef float f32x2 __attribute__((ext_vector_type(2)));
                const f32x2 p = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false), q = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
                old[i] = kv8_codes(p[0] * f, p[1] * f, q[0] * f, q[1] * f, kv8_most(e));
            }
        }
        e = max(e, e_was);
    }
    const float inv = pow2f(-e), largest = kv8_most(e);
    uint8_t* to = codes + (lo - first) * a.d;
#pragma unroll
    for (int u = 0; u < ITEMS; ++u) {
        const int i = tid + u * NT;                                  // (the new tokens' codes are dense)
        if (i >= items) continue;
        float y[PER];
        Elem<DT>::unpack(raw[u], y);
        uint32_t w[PER / 4];
#pragma unroll
        for (int j = 0; j < PER / 4; ++j) w[j] = kv8_codes(y[4 * j] * inv, y[4 * j + 1] * inv, y[4 * j + 2] * inv, y[4 * j + 3] * inv, largest);
        uint32_t* out = reinterpret_cast<uint32_t*>(to + i * PER);
#pragma unroll
        for (int j = 0; j < PER / 4; ++j) out[j] = w[j];
    }
    if (tid == 0) *scale = pow2f(e);                                 // (every thread of a wider workgroup has read the old one: the barrier above)
}

template <int DT> hipError_t run_kv8_append(const Kv8AppendArgs& k, dim3 grid, hipStream_t s)
{
    constexpr int PER = Elem<DT>::PER;
    // a few tokens: one wave holds a block's share (64 sequences, one token, 16 heads: 4.7 us with four waves)
    if ((int64_t)k.new_tokens * k.d <= 64 * PER) return ops_launch(kv8_append_kernel<DT, 64, 1>, grid, dim3(64), s, k);
    if (k.d <= 64) return ops_launch(kv8_append_kernel<DT, 256, 64 * 64 / PER / 256>, grid, dim3(256), s, k);
    return ops_launch(kv8_append_kernel<DT, 256, 64 * 128 / PER / 256>, grid, dim3(256), s, k);
}

}  // namespace

extern "C" {

const char* asr_ops_last_error(void) { return g_ops_error; }

int asr_token_logprobs(const asr_token_logprobs_args* a, void* stream)
{
    if (!a) return ops_fail(ASR_ERR_ARG, "null argument");
    return ops_token_logprobs(*a, static_cast<hipStream_t>(stream));
}

int asr_kv8_append(const asr_kv8_append_args* a, void* stream)
{
    if (!a) return ops_fail(ASR_ERR_ARG, "null argument");
    if (a->n < 0 || a->new_tokens < 0 || a->kv_heads < 1 || a->capacity < 0) return ops_fail(ASR_ERR_ARG, "kv8_append: bad sizes");
    if (a->d < 16 || a->d > 128 || a->d % 16) return ops_fail(ASR_ERR_ARG, "kv8_append: d must be a multiple of 16 in 16..128");
    if (a->capacity % ASR_KV8_BLOCK) return ops_fail(ASR_ERR_ARG, "kv8_append: the capacity must be a multiple of %d tokens", ASR_KV8_BLOCK);
    if (!ops_dtype_ok(a->dtype)) return ops_fail(ASR_ERR_ARG, "kv8_append: unknown dtype %d", a->dtype);
    if (a->n == 0 || a->new_tokens == 0 || a->capacity == 0) return ASR_OK;
    if (!a->k || !a->v || !a->k_cache || !a->v_cache || !a->k_scale || !a->v_scale || !a->lens) return ops_fail(ASR_ERR_ARG, "kv8_append: null argument");
    if (!ops_rows16(a->k, a->k_stride, a->n, a->new_tokens, a->kv_heads, a->dtype) || !ops_rows16(a->v, a->v_stride, a->n, a->new_tokens, a->kv_heads, a->dtype))
        return ops_fail(ASR_ERR_ARG, "kv8_append: rows of k and v must start on 16 bytes");
    if (((reinterpret_cast<uintptr_t>(a->k_cache) | reinterpret_cast<uintptr_t>(a->v_cache)) & 15) || a->cache_stride[0] % 16 || a->cache_stride[1] % 16)
        return ops_fail(ASR_ERR_ARG, "kv8_append: cache rows must start on 16 bytes");
    // blocks that new_tokens tokens can touch, wherever the first one falls
    const int64_t touched = ((int64_t)a->new_tokens + ASR_KV8_BLOCK - 2) / ASR_KV8_BLOCK + 1;
    const int64_t blocks = touched < a->capacity / ASR_KV8_BLOCK ? touched : a->capacity / ASR_KV8_BLOCK;
    if (a->n > 65535 || a->kv_heads > (1 << 20) || blocks > 65535)
        return ops_fail(ASR_ERR_ARG, "kv8_append: at most 65535 sequences, 2^20 heads and 65535 blocks of tokens a call");
    if (a->k_cache == a->v_cache || a->k_scale == a->v_scale) return ops_fail(ASR_ERR_ARG, "kv8_append: keys and values need caches and scales of their own");
    Kv8AppendArgs k{};
    k.x[0] = a->k; k.x[1] = a->v;
    k.cache[0] = a->k_cache; k.cache[1] = a->v_cache;
    k.scale[0] = a->k_scale; k.scale[1] = a->v_scale;
    k.lens = a->lens; k.counts = a->counts;
    for (int i = 0; i < 3; ++i) { k.stride[0][i] = a->k_stride[i]; k.stride[1][i] = a->v_stride[i]; }
    k.cache_stride[0] = a->cache_stride[0]; k.cache_stride[1] = a->cache_stride[1];
    k.new_tokens = a->new_tokens; k.kv_heads = a->kv_heads; k.d = a->d; k.capacity = a->capacity;
    const dim3 grid(2 * a->kv_heads, (uint32_t)blocks, a->n);
    hipStream_t s = static_cast<hipStream_t>(stream);
    return ops_launched("kv8_append", a->dtype == ASR_F32 ? run_kv8_append<ASR_F32>(k, grid, s)
                                      : a->dtype == ASR_BF16 ? run_kv8_append<ASR_BF16>(k, grid, s) : run_kv8_append<ASR_F16>(k, grid, s));
}

}  // extern "C"
