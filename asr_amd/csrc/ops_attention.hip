// Attention operators on device memory: over the states of another sequence, and over the 8-bit K/V cache.  C entry points:
// include/asr_amd.h.
//
// With G = heads / kv_heads, the rows r = i * G + g of one (sequence, K/V head) share its keys and values:
//     S = c q K^T,   P = e^(S - m),   out = P V / l,   m = running row maximum, l = running row sum of P
// taken over tiles of keys in one pass (when m grows, what was summed is scaled by e^(m_old - m_new)).  Everything is computed transposed:
// S^T = K q^T leaves a query row in each lane of 16 (its statistics are then per-lane values and need no exchange but over the four lane
// groups), and O^T = V^T P^T takes the probabilities straight from the accumulators as its second operand: the order of keys inside a tile is
// free, so tile row m is given the key that puts eight consecutive keys of one lane group where the next product wants them.
#include "ops_common.h"

#include <math.h>

namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr float LOG2E = 1.44269504088896340736f;
constexpr float NEG_INF = -__builtin_inff();

enum { KV_F32 = ASR_F32, KV_BF16 = ASR_BF16, KV_F16 = ASR_F16, KV_E4M3 = 3 };

struct AttnArgs {
    const char *q, *k, *v;
    char* out;
    const float *k_scale, *v_scale;      // KV_E4M3
    const int32_t *lens, *counts;        // counts (KV_E4M3): a sequence's own queries, its first ones; null: all tq
    const uint8_t* pad;
    float* ws;                           // nsplit > 1: per (split, sequence, K/V head, row): m, l, then O [d]
    int64_t q_stride[3], out_stride[3], k_stride[3], v_stride[3];        // bytes; of n, t, head
    int64_t pad_stride, scale_stride;    // scale_stride: floats of one (sequence, head)
    int n, tq, tk, kv_heads, group, d, causal;
    int rows, tiles, nsplit;             // rows = tq * group of one (sequence, K/V head); tiles of rows
    float c;                             // scale * log2(e): powers of two instead of e
};

// a place in GPU memory: where pointers are chosen between, the compiler no longer sees that they are none of LDS and takes slower loads
typedef const __attribute__((address_space(1))) char* mem;
template <typename T> __device__ inline T load_as(mem p) { return *(const __attribute__((address_space(1))) T*)p; }

__device__ inline uint32_t pack_bf16(float a, float b)
{
    bf16x2 r;
    r[0] = (__bf16)a;
    r[1] = (__bf16)b;
    return __builtin_bit_cast(uint32_t, r);
}
__device__ inline uint32_t pack_f16(float a, float b)
{
    f16x2 r;
    r[0] = (_Float16)a;
    r[1] = (_Float16)b;
    return __builtin_bit_cast(uint32_t, r);
}
template <bool F16> __device__ inline uint32_t pack16(float a, float b) { return F16 ? pack_f16(a, b) : pack_bf16(a, b); }
template <bool F16> __device__ inline f32x2 unpack16(uint32_t u)
{
    f32x2 r;
    if (F16) {
        const f16x2 h = __builtin_bit_cast(f16x2, u);
        r[0] = (float)h[0];
        r[1] = (float)h[1];
    } else {
        r[0] = __uint_as_float(u << 16);
        r[1] = __uint_as_float(u & 0xffff0000u);
    }
    return r;
}
template <bool F16> __device__ inline f32x4 mfma16(const u32x4& a, const u32x4& b, const f32x4& c)
{
    if (F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
// two e4m3 codes (the low or the high half of a word) times a power of two: exact in bf16
template <bool HI> __device__ inline uint32_t codes_bf16(uint32_t w, float scale)
{
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, scale, HI));
}

// all ones in the bytes of w that are NaN codes (all seven bits below the sign set)
__device__ inline uint32_t nan_codes(uint32_t w)
{
    const uint32_t top = ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
    return top | (top - (top >> 7));
}

// all ones where bit `at` of `bits` is set; x there, else -infinity (two instructions a value)
__device__ inline uint32_t spread_bit(uint32_t bits, int at) { return (uint32_t)((int32_t)(bits << (31 - at)) >> 31); }
__device__ inline float admit(float x, uint32_t ones) { return __uint_as_float((__float_as_uint(x) & ones) | (0xff800000u & ~ones)); }

// maximum / sum over the four 16-lane groups of a wave
__device__ inline float groups_max(float x)
{
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ inline float groups_sum(float x)
{
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// P = 2^(score - m).  m follows a row's maximum (in powers of two) only when that grows by more than SLACK: P is at most 2^SLACK then, its rounding is relative as before, and
// nearly all tiles skip the scaling of the sums.  It starts finite, so that no difference with it is NaN.  A float16 P is relative down to 2^-14 and 0 below 2^-25: there m stays
// LIFT below the maximum that it follows, so that the largest P of a row is 2^7 to 2^15 and keys 22 nats below it still count (a largest one of 1 lost those 17 nats below).
constexpr float SLACK = 8.0f, LIFT16 = 7.0f, NO_MAX = -3.0e38f;
// a b rounded, never one operation with what is added to it
__device__ inline float product(float a, float b)
{
#pragma clang fp contract(off)
    return a * b;
}
__device__ inline float rescale(float m_old, float m_new) { return __builtin_amdgcn_exp2f(m_old - m_new); }

// An infinity in an admitted V: a term of P that is 0, or of the other sign than the first, makes NaN of it, as does scaling what was summed by 0, and the cut of a float32 one.
// Where a sum is NaN though the row's P are finite, its columns of V are looked through again (bit i for column i of what a lane has): with one sign of infinity the
// sum is that, with both or with NaN it is NaN.
struct Seen {
    uint32_t up = 0, down = 0, nan = 0;
    template <int KVT> __device__ inline void add(mem p, int bit)
    {
        constexpr uint32_t INF = KVT == KV_F32 ? 0x7f800000u : KVT == KV_F16 ? 0x7c00u : 0x7f80u, SIGN = KVT == KV_F32 ? 0x80000000u : 0x8000u;
        uint32_t x;
        if constexpr (KVT == KV_F32) x = load_as<uint32_t>(p);
        else x = load_as<uint16_t>(p);
        const uint32_t size = x & ~SIGN;
        up |= (uint32_t)(x == INF) << bit;
        down |= (uint32_t)(x == (INF | SIGN)) << bit;
        nan |= (uint32_t)(size > INF) << bit;
    }
    __device__ inline float instead_of(float sum, int bit) const
    {
        const bool u = up >> bit & 1, d = down >> bit & 1, n = nan >> bit & 1;
        return n || (u && d) ? __builtin_nanf("") : u ? __builtin_inff() : d ? -__builtin_inff() : sum;
    }
};
// x f, but an infinite x stays what it is where f is 0
__device__ inline float scaled(float x, float f) { return __builtin_fabsf(x) == __builtin_inff() ? x : x * f; }
__device__ inline f32x4 scaled(const f32x4& x, float f) { return f32x4{scaled(x[0], f), scaled(x[1], f), scaled(x[2], f), scaled(x[3], f)}; }

__device__ inline int keys_of(const AttnArgs& a, int b) { return a.lens ? min(max(a.lens[b], 0), a.tk) : a.tk; }

// Workgroup `id` -> (sequence, K/V head), and what is left of id for its row tile and share, `per` of them for each.  Consecutive workgroups go round the
// eight XCDs, each with an L2 of its own: all workgroups of one (sequence, head) go to one XCD, next to each other, so that its keys are read into one
// L2 once; an XCD gets another head of each sequence (the same head's rows, a power of two apart where the heads of a token lie side by side, share a few of
// the L2's channels).  Eight sequences, eight heads of 128, 24 row tiles, probabilities of one term: 328 us with the tiles next to each other, 368 with the heads.
__device__ inline int place_of(int nbh, int per, int64_t& id)
{
    int bh;
    if (nbh % 8) {
        bh = (int)(id / per);
        id %= per;
    } else {
        const int xcd = (int)(id % 8), j = (int)(id / 8 / per);
        bh = 8 * j + ((xcd - j) & 7);
        id = id / 8 % per;
    }
    return bh;
}

// the queries that sequence b has; those behind them are computed like its last one and given zeros
template <bool CODES> __device__ inline int queries_of(const AttnArgs& a, int b) { return CODES && a.counts ? min(max(a.counts[b], 0), a.tq) : a.tq; }

// The sequence that is number `at` when the longest come first (at itself where that would not matter or take too long): the last workgroups of a launch
// are then short ones (16 x 200 queries over 1500 states of half to full length: 45.2 -> 43.1 us; 64 x 80 over caches of up to 2048 of 8 heads: 61.5 -> 57; one token over 64
// such caches of 16 heads: 45.7 -> 42.9).  Finding it
// costs up to half a microsecond a workgroup, too much for few rows over short keys (64 x 10 queries over 334 states: 15.5 -> 16.4 us).
__device__ inline int longest_first(const AttnArgs& a, int at)
{
    if (!a.lens || a.n < 2 || a.n > 64 || a.tk >= 1 << 25) return at;
    const int lane = threadIdx.x & 63, key = lane < a.n ? keys_of(a, lane) * 64 + 63 - lane : -1;
    int before = 0;
    for (int j = 0; j < a.n; j += 8)
#pragma unroll
        for (int i = 0; i < 8; ++i) before += __builtin_amdgcn_readlane(key, (j + i) & 63) > key;
    return __builtin_ctzll(__ballot(lane < a.n && before == at));
}

// ---- few rows: the waves of a workgroup share the keys ------------------------------------------------------------------
// A workgroup has one tile of 16 NQ rows of one (sequence, K/V head) and one share of its keys; its four waves take 32 keys at a time in turn,
// straight from memory into registers in the operands' own order (no LDS in the loop), and join their sums in LDS at the end.  The next chunk's
// keys are loaded as soon as the scores have been taken from this one's, the next values behind the output.  K and V are read once by each row
// tile: bound by those bytes while there are few rows.  QT: type of q and out, KVT: of K and V.
// Terms: 16-bit K / V are exact factors; q enters as QTERMS 16-bit terms (bf16 codes: f16 = 2, f32 = 3 bf16 terms lose nothing) and
// P as PTERMS (two: 2^-17 of it lost, of float16 2^-22 or 2^-32 of the row's largest, whichever is more; three: nothing), which costs matrix instructions that a loop waiting for memory has to spare.
// float32 K / V are cut into three bf16 terms as well (8 + 8 + 8 bits: exact), and of the nine products the six above 2^-24 are taken: the 16-bit matrix
// pipe is 16 times the float32 one, which besides shares its units with the vector instructions (50 x 61 queries over 1000 states of 16 heads:
// 133 us on the float32 instruction, 108 so).
template <int QT, int KVT, int DP, int NQ> struct Few {
    static constexpr bool MATH32 = KVT == KV_F32, F16 = KVT == KV_F16, CODES = KVT == KV_E4M3;
    static constexpr int QTERMS = QT == ASR_F32 ? 3 : CODES && QT == ASR_F16 ? 2 : 1;
    static constexpr int PTERMS = QT == ASR_F32 ? 3 : 2, KTERMS = MATH32 ? 3 : 1;
    static constexpr int KVB = KVT == KV_F32 ? 4 : CODES ? 1 : 2;         // bytes of a K / V value
    static constexpr int QB = QT == ASR_F32 ? 4 : 2;
    static constexpr int KW = DP / 4 * KVB / 4;                             // words of a key row in one lane (a quarter of it)
    static constexpr int VW = DP / 16 * KVB / 4;                            // words of a value row in one lane (a sixteenth)
    typedef uint32_t VRow __attribute__((ext_vector_type(VW)));
    static constexpr int NO = DP / 16;                                      // 16 x 16 output tiles of one row tile
};

constexpr int FEW_WAVES = 4;

// eight float32 values as three bf16 vectors that add up to them: the upper half of each, of what is left, and of what is left then (exact; an infinite value
// leaves NaN)
__device__ inline void cut(const uint32_t (&x)[8], u32x4 (&t)[3])
{
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t a = x[2 * j], b = x[2 * j + 1];
        const float a1 = __uint_as_float(a) - __uint_as_float(a & 0xffff0000u), b1 = __uint_as_float(b) - __uint_as_float(b & 0xffff0000u);
        const uint32_t a1u = __float_as_uint(a1), b1u = __float_as_uint(b1);
        const float a2 = a1 - __uint_as_float(a1u & 0xffff0000u), b2 = b1 - __uint_as_float(b1u & 0xffff0000u);
        t[0][j] = __builtin_amdgcn_perm(b, a, 0x07060302u);
        t[1][j] = __builtin_amdgcn_perm(b1u, a1u, 0x07060302u);
        t[2][j] = __builtin_amdgcn_perm(__float_as_uint(b2), __float_as_uint(a2), 0x07060302u);
    }
}
// eight float16 values as two bf16 vectors that add up to them
__device__ inline void cut_f16(const u32x4& x, u32x4 (&t)[2])
{
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const f32x2 y = unpack16<true>(x[j]);
        const uint32_t hi = pack_bf16(y[0], y[1]);
        const f32x2 z = unpack16<false>(hi);
        t[0][j] = hi;
        t[1][j] = pack_bf16(y[0] - z[0], y[1] - z[1]);
    }
}
// c + a b over bf16 terms of a and b, those above 2^-24 of the product, the smallest first
template <bool F16, int NA, int NB> __device__ inline f32x4 mfma_terms(const u32x4 (&a)[NA], const u32x4 (&b)[NB], f32x4 c)
{
#pragma unroll
    for (int sum = NA + NB - 2 < 2 ? NA + NB - 2 : 2; sum >= 0; --sum)
#pragma unroll
        for (int i = NA - 1; i >= 0; --i)
            if (sum - i >= 0 && sum - i < NB) c = mfma16<F16>(a[i], b[sum - i], c);
    return c;
}

// the place in a row of value j (0 .. DP/4) of lane group g's quarter of it
template <int KVT> __device__ constexpr int quarter_at(int g, int j)
{
    return KVT == KV_F32 ? 16 * (j >> 2) + 4 * g + (j & 3) : KVT == KV_E4M3 ? 64 * (j >> 4) + 16 * g + (j & 15) : 32 * (j >> 3) + 8 * g + (j & 7);
}

// (two workgroups on a compute unit but where float32 rows of 128 need all registers)
template <int QT, int KVT, int DP, int NQ, bool FULL> __global__ __launch_bounds__(64 * FEW_WAVES, KVT == KV_F32 && DP == 128 && NQ == 2 ? 1 : 2)
void attention_few_kernel(AttnArgs a)
{
    typedef Few<QT, KVT, DP, NQ> F;
    constexpr int PITCH = DP + 4;
    __shared__ float s_m[FEW_WAVES][16 * NQ], s_l[FEW_WAVES][16 * NQ];
    __shared__ __align__(16) float s_o[FEW_WAVES][16 * NQ][PITCH];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), x16 = lane & 15, g = lane >> 4;
    int64_t id = blockIdx.x;
    const int place = place_of(a.n * a.kv_heads, a.tiles * a.nsplit, id);
    const int split = (int)(id % a.nsplit), tile = (int)(id / a.nsplit);
    const int b = a.tk >= 1024 ? longest_first(a, place / a.kv_heads) : place / a.kv_heads, h = place % a.kv_heads, bh = b * a.kv_heads + h;
    const int len = keys_of(a, b), row0 = tile * 16 * NQ, tq = queries_of<F::CODES>(a, b);

    // this tile's keys: all of them, or in a causal call what its last row sees; none without queries
    int last_key = len;
    if (a.causal) last_key = min(len, max(0, len - tq + min(min(row0 + 16 * NQ - 1, a.rows - 1) / a.group, tq - 1) + 1));
    if (row0 / a.group >= tq) last_key = 0;
    const int chunks = (last_key + 31) / 32, share = (chunks + a.nsplit - 1) / a.nsplit;
    const int chunk0 = split * share, chunk1 = min(chunks, chunk0 + share);

    // q in the second operand's layout: lane x16 holds row x16, lane group g its quarter of the row
    u32x4 qf[NQ][DP / 32][F::QTERMS];
    int lim[NQ];
#pragma unroll
    for (int t = 0; t < NQ; ++t) {
        const int r = row0 + 16 * t + x16, rc = min(r, a.rows - 1);
        lim[t] = a.causal ? len - tq + min(rc / a.group, tq - 1) + 1 : len;
        const char* qp = a.q + (int64_t)b * a.q_stride[0] + (int64_t)(rc / a.group) * a.q_stride[1] + (int64_t)(h * a.group + rc % a.group) * a.q_stride[2];
#pragma unroll
        for (int u = 0; u < DP / 32; ++u) {
            // eight values: consecutive, or (float32 K) four and four
            const int at = quarter_at<KVT>(g, 8 * u), at2 = quarter_at<KVT>(g, 8 * u + 4);
            const bool in = at < a.d && r < a.rows, in2 = at2 < a.d && r < a.rows;
            if constexpr (F::QTERMS == 1) qf[t][u][0] = in ? *reinterpret_cast<const u32x4*>(qp + 2 * at) : u32x4{};
            else if constexpr (QT == ASR_F32) {
                const u32x4 lo = in ? *reinterpret_cast<const u32x4*>(qp + 4 * at) : u32x4{}, hi = in2 ? *reinterpret_cast<const u32x4*>(qp + 4 * at2) : u32x4{};
                const uint32_t x[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
                cut(x, qf[t][u]);
            } else {
                cut_f16(in ? *reinterpret_cast<const u32x4*>(qp + 2 * at) : u32x4{}, qf[t][u]);
            }
        }
    }

    const int first_lim = a.causal ? len - tq + row0 / a.group + 1 : 0x7fffffff;         // every row of this tile sees the keys below it

    f32x4 o[NQ][F::NO];
    float m[NQ], l[NQ];
#pragma unroll
    for (int t = 0; t < NQ; ++t) {
        m[t] = NO_MAX;
        l[t] = 0.0f;
#pragma unroll
        for (int i = 0; i < F::NO; ++i) o[t][i] = f32x4{};
    }
    const char* kb = a.k + (int64_t)b * a.k_stride[0] + (int64_t)h * a.k_stride[2];
    const char* vb = a.v + (int64_t)b * a.v_stride[0] + (int64_t)h * a.v_stride[2];
    const float *ksc = nullptr, *vsc = nullptr;
    if constexpr (F::CODES) {
        ksc = a.k_scale + (int64_t)bh * a.scale_stride;
        vsc = a.v_scale + (int64_t)bh * a.scale_stride;
    }
    const uint8_t* pad = a.pad ? a.pad + (int64_t)b * a.pad_stride : nullptr;

    // K: tile t2's row x16 is key 8 (x16 / 4) + 4 t2 + x16 % 4 of a chunk; V: lane group g has keys 8 g .. 8 g + 7, lane x16 a sixteenth of each row.
    // Keys past the end are read from the last one; values past d are zeros (K) or not used (V).
    const int k_row = 8 * (x16 >> 2) + (x16 & 3), v_row = 8 * g;
    const int v_at = F::MATH32 ? 4 * x16 : DP / 16 * x16;
    const mem kp = (mem)(kb + (uint64_t)k_row * (uint64_t)a.k_stride[1]);
    const mem vp = (mem)(vb + (uint64_t)v_row * (uint64_t)a.v_stride[1] + (FULL || v_at < a.d ? v_at * F::KVB : 0));
    u32x4 kr[2][F::KW / 4];                        // (vectors as they are loaded: taken apart into words here, pairs of them were given one register)
    typename F::VRow vr[8];
    uint32_t flag = 0;
    float ks = 1.0f, vs = 1.0f;
    const auto load_k = [&](int c0) __attribute__((always_inline)) {
        if (pad) flag = c0 + (lane & 31) < len ? pad[c0 + (lane & 31)] : 0;
        if constexpr (F::CODES) ks = ksc[c0 / ASR_KV8_BLOCK];
        mem p[2];
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2) p[t2] = kp + (c0 + 4 * t2) * a.k_stride[1];
        if (c0 + 32 > len) {
            asm volatile("");                                                  // (a branch: products of 64 bits in the last chunk only)
#pragma unroll
            for (int t2 = 0; t2 < 2; ++t2) p[t2] += (int64_t)min(0, len - 1 - (c0 + 4 * t2 + k_row)) * a.k_stride[1];
        }
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2)
#pragma unroll
            for (int w = 0; w < F::KW; w += 4) {
                const int at = quarter_at<KVT>(g, w * 4 / F::KVB);
                kr[t2][w / 4] = load_as<u32x4>(p[t2] + (FULL || at < a.d ? at * F::KVB : 0));
                if (!FULL && at >= a.d) kr[t2][w / 4] = u32x4{};
            }
    };
    const auto load_v = [&](int c0) __attribute__((always_inline)) {
        if constexpr (F::CODES) vs = vsc[c0 / ASR_KV8_BLOCK];
        mem p[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) p[j] = vp + (c0 + j) * a.v_stride[1];
        if (c0 + 32 > len) {
            asm volatile("");
#pragma unroll
            for (int j = 0; j < 8; ++j) p[j] += (int64_t)min(0, len - 1 - (c0 + j + v_row)) * a.v_stride[1];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if constexpr (F::MATH32) {
#pragma unroll
                for (int u = 0; u < DP / 64; ++u) {
                    const u32x4 x = load_as<u32x4>(p[j] + (FULL || 64 * u + v_at < a.d ? 256 * u : 0));
#pragma unroll
                    for (int w = 0; w < 4; ++w) vr[j][4 * u + w] = x[w];
                }
            } else vr[j] = load_as<typename F::VRow>(p[j]);
        }
    };

    constexpr float LIFT = F::F16 ? LIFT16 : 0.0f;
    uint64_t nan_seen = 0;
    int chunk = chunk0 + wave;
    if (chunk < chunk1) {
        load_k(32 * chunk);
        load_v(32 * chunk);
    }
    for (; chunk < chunk1; chunk += FEW_WAVES) {
        const int c0 = chunk * 32;
        const bool more = chunk + FEW_WAVES < chunk1;
        // one admitted-bit per key of the chunk, the same for the whole wave
        const uint32_t mask = (uint32_t)__ballot(c0 + (lane & 31) < len && flag == 0);
        const uint32_t mine = mask >> (8 * g);                                 // bits 0 .. 7: keys 8 g .. 8 g + 7
        // S^T
        f32x4 s[NQ][2];
#pragma unroll
        for (int t = 0; t < NQ; ++t) s[t][0] = s[t][1] = f32x4{};
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2) {
#pragma unroll
            for (int u = 0; u < DP / 32; ++u) {
                u32x4 kf[F::KTERMS];
                if constexpr (F::MATH32) {
                    const u32x4 &lo = kr[t2][2 * u], &hi = kr[t2][2 * u + 1];
                    const uint32_t x[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
                    cut(x, kf);
                } else if constexpr (F::CODES) {
                    const uint32_t lo = kr[t2][u / 2][2 * (u & 1)], hi = kr[t2][u / 2][2 * (u & 1) + 1];
                    kf[0] = u32x4{codes_bf16<false>(lo, ks), codes_bf16<true>(lo, ks), codes_bf16<false>(hi, ks), codes_bf16<true>(hi, ks)};
                } else kf[0] = kr[t2][u];
#pragma unroll
                for (int t = 0; t < NQ; ++t) s[t][t2] = mfma_terms<F::F16>(kf, qf[t][u], s[t][t2]);
            }
        }
        if (more) load_k(c0 + 32 * FEW_WAVES);

        // soft-max step; p[t][4 t2 + i] belongs to key 8 g + 4 t2 + i
        float p[NQ][8];
#pragma unroll
        for (int t = 0; t < NQ; ++t) {
#pragma unroll
            for (int j = 0; j < 8; ++j) p[t][j] = product(s[t][j >> 2][j & 3], a.c);
            if (mask != 0xffffffffu) {
                asm volatile("");                                              // (a branch, not selects in every chunk)
#pragma unroll
                for (int j = 0; j < 8; ++j) p[t][j] = admit(p[t][j], spread_bit(mine, j));
            }
            if (c0 + 32 > first_lim) {                                         // (causal calls)
                asm volatile("");
#pragma unroll
                for (int j = 0; j < 8; ++j) p[t][j] = c0 + 8 * g + j < lim[t] ? p[t][j] : NEG_INF;
            }
            float top = p[t][0];
#pragma unroll
            for (int j = 1; j < 8; ++j) top = fmaxf(top, p[t][j]);
            top = groups_max(top);
            if (__ballot(top - m[t] > SLACK + LIFT)) {                         // (the difference: exact where m + SLACK would be rounded)
                const float grown = fmaxf(m[t], top - LIFT), f = rescale(m[t], grown);
                m[t] = grown;
                l[t] *= f;
#pragma unroll
                for (int i = 0; i < F::NO; ++i) o[t][i] *= f;
            }
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                p[t][j] = __builtin_amdgcn_exp2f(p[t][j] - m[t]);
                sum += p[t][j];
            }
            l[t] += sum;
        }

        // O^T += V^T P^T; what is not admitted may hold anything: P = 0 meets V = 0
        if (mask != 0xffffffffu) {
#pragma unroll
            for (int j = 0; j < 8; ++j) vr[j] &= spread_bit(mine, j);
        }
        // What a causal call hides from some of the rows may be NaN as well: such values are taken as 0 and looked up again at the end
        if constexpr (F::CODES) {
            if (c0 + 32 > first_lim) {
                uint32_t any = 0;
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int w = 0; w < F::VW; ++w) {
                        const uint32_t x = nan_codes(vr[j][w]);
                        any |= x;
                        vr[j][w] &= ~x;
                    }
                nan_seen |= __ballot(any != 0);
            }
        }
        u32x4 pf[NQ][F::PTERMS];
#pragma unroll
        for (int t = 0; t < NQ; ++t)
#pragma unroll
            for (int term = 0; term < F::PTERMS; ++term)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t w = pack16<F::F16>(p[t][2 * j], p[t][2 * j + 1]);
                    pf[t][term][j] = w;
                    const f32x2 y = unpack16<F::F16>(w);
                    p[t][2 * j] -= y[0];
                    p[t][2 * j + 1] -= y[1];
                }
#pragma unroll
        for (int i = 0; i < F::NO; ++i) {
            u32x4 vf[F::KTERMS];
            if constexpr (F::MATH32) {
                const uint32_t x[8] = {vr[0][i], vr[1][i], vr[2][i], vr[3][i], vr[4][i], vr[5][i], vr[6][i], vr[7][i]};
                cut(x, vf);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if constexpr (F::CODES) {
                        const uint32_t two = __builtin_amdgcn_perm(vr[2 * j + 1][i >> 2], vr[2 * j][i >> 2], i & 2 ? 0x07030602u : 0x05010400u);
                        vf[0][j] = i & 1 ? codes_bf16<true>(two, vs) : codes_bf16<false>(two, vs);
                    } else {
                        vf[0][j] = __builtin_amdgcn_perm(vr[2 * j + 1][i >> 1], vr[2 * j][i >> 1], i & 1 ? 0x07060302u : 0x05040100u);
                    }
                }
            }
#pragma unroll
            for (int t = 0; t < NQ; ++t) o[t][i] = mfma_terms<F::F16>(vf, pf[t], o[t][i]);
        }
        if (more) load_v(c0 + 32 * FEW_WAVES);
    }

    if constexpr (F::CODES) {
        if (nan_seen) {
            // where a row sees a NaN its sum is one (this wave's chunks; a lane has DP / 16 columns from DP / 16 (4 g + j) on)
            for (int c = chunk0 + wave; c < chunk1; c += FEW_WAVES)
                for (int key = 32 * c; 32 * c + 32 > first_lim && key < min(32 * c + 32, len); ++key)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int w = 0; w < F::VW; ++w) {
                            const int at = DP / 16 * (4 * g + j) + 4 * w;
                            const uint32_t x = at < a.d ? nan_codes(load_as<uint32_t>((mem)vb + (int64_t)key * a.v_stride[1] + at)) : 0u;
#pragma unroll
                            for (int e = 0; e < 4; ++e)
#pragma unroll
                                for (int t = 0; t < NQ; ++t) o[t][4 * w + e][j] = key < lim[t] && (x >> (8 * e)) & 1 ? __builtin_nanf("") : o[t][4 * w + e][j];
                        }
        }
    }

    // join the waves
#pragma unroll
    for (int t = 0; t < NQ; ++t) {
        const float sum = groups_sum(l[t]);
        if (g == 0) {
            s_m[wave][16 * t + x16] = m[t];
            s_l[wave][16 * t + x16] = sum;
        }
#pragma unroll
        for (int i = 0; i < F::NO; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int at = F::MATH32 ? 64 * (i >> 2) + 4 * (4 * g + j) + (i & 3) : DP / 16 * (4 * g + j) + i;
                s_o[wave][16 * t + x16][at] = o[t][i][j];
            }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < 16 * NQ * (DP / 4); e += 64 * FEW_WAVES) {
        const int rr = e / (DP / 4), at = e % (DP / 4) * 4, r = row0 + rr;
        if (r >= a.rows || at >= a.d) continue;
        float top = s_m[0][rr];
#pragma unroll
        for (int w = 1; w < FEW_WAVES; ++w) top = fmaxf(top, s_m[w][rr]);
        float sum = 0.0f;
        f32x4 acc{};
#pragma unroll
        for (int w = 0; w < FEW_WAVES; ++w) {
            const float f = rescale(s_m[w][rr], top);
            sum += s_l[w][rr] * f;
            acc += *reinterpret_cast<const f32x4*>(&s_o[w][rr][at]) * f;
        }
        if constexpr (!F::CODES) {
            const float all = acc[0] + acc[1] + acc[2] + acc[3];
            if (all != all && sum < __builtin_inff()) {
                Seen seen;
                for (int key = 32 * chunk0; key < min(32 * chunk1, len); ++key) {
                    if (pad && pad[key]) continue;
                    const mem p = (mem)vb + (int64_t)key * a.v_stride[1] + at * F::KVB;
#pragma unroll
                    for (int i = 0; i < 4; ++i) seen.add<KVT>(p + i * F::KVB, i);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[i] = seen.instead_of(acc[i], i);
            }
        }
        if (r / a.group >= tq) {
            sum = 0.0f;
            acc = f32x4{};
        }
        if (a.nsplit > 1) {
            float* ws = a.ws + (((int64_t)split * a.n * a.kv_heads + bh) * a.rows + r) * (a.d + 4);
            if (at == 0) { ws[0] = top; ws[1] = sum; }
            *reinterpret_cast<f32x4*>(ws + 4 + at) = acc;
        } else {
            acc = sum == 0.0f ? f32x4{} : acc * (1.0f / sum);
            char* op = a.out + (int64_t)b * a.out_stride[0] + (int64_t)(r / a.group) * a.out_stride[1] +
                       (int64_t)(h * a.group + r % a.group) * a.out_stride[2] + at * F::QB;
            if constexpr (QT == ASR_F32) *reinterpret_cast<f32x4*>(op) = acc;
            else {
                u32x2 w;
                w[0] = pack16<QT == ASR_F16>(acc[0], acc[1]);
                w[1] = pack16<QT == ASR_F16>(acc[2], acc[3]);
                *reinterpret_cast<u32x2*>(op) = w;
            }
        }
    }
}

// ---- many rows: the waves of a workgroup share tiles of keys in LDS ------------------------------------------------------
// 16-bit products only, the probabilities as two terms like those of few rows (codes with a float16 q: q as two bf16 terms too, which keep its bits).  One term would
// save a third of the products and round every probability to 8 bits: as much error as the result's own rounding adds (8 x 768 queries of 32 heads over 4001 states of 8
// heads of 128: 450 us and 0.0017 of the result with two, 328 us and 0.0023 with one).  A workgroup has 128 rows (NR = 1) or 256, 32 NR for each of its four waves, and walks over tiles of 64 keys that it stages into LDS
// (K three buffers, V two: the next tiles' loads are in flight while this one is used, one barrier a tile; codes become bf16 on the way, times their block's
// scale).  32 x 32 x 16 products: S^T = K q^T has a row in each lane of 32 and lane half; O^T = V^T P^T takes V^T from LDS with the transposing read
// (four keys of one column a lane) and P^T straight from the accumulators: what a term lacks is exact in float32 and becomes the next one.
// The 16-byte chunks of a row are permuted by its number (K: chunk ^ row % 16, V: chunk ^ 4 (row % 4), by pairs of rows where rows are half
// as long): both kinds of read then meet every bank evenly.  Rows of 16-bit values as long as the tile go from memory to LDS directly.
// What bounds it: instructions.  A tile is 48 products (1536 cycles of the matrix pipe) and some 300 vector instructions a wave and row tile; products of one
// wave run beside the vector instructions of both waves of a SIMD, but a wave alone issues only every 7 cycles.
constexpr int MANY_WAVES = 4, MANY_ROWS = 32 * MANY_WAVES, MANY_KEYS = 64;               // (MANY_ROWS: for each row tile of a wave)

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

template <bool F16> __device__ inline f32x16 mfma32(const u32x4& a, const u32x4& b, const f32x16& c)
{
    if (F16) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ inline u32x2 lds_read_transposed(const __attribute__((address_space(3))) char* p)
{
    const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
    return __builtin_bit_cast(u32x2, x);
}
// 16 bytes a lane from memory to LDS, the wave's 1024 in lane order from `lds` on; done when the wave has waited for its memory operations.  (The
// builtin would have every later LDS read wait for it, as the compiler cannot tell the buffers apart.  The place in LDS is an operand in m0, so the compiler sets that
// register and knows what is in it; its read needs a wait state.)
__device__ inline uint32_t lds_at(char* p) { return __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)p); }
__device__ inline void load_to_lds(mem p, uint32_t at)
{
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(p), "{m0}"(at) : "memory");
}
__device__ inline void wait_for_memory() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory"); }
__device__ inline float halves_max(float x)
{
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ inline float halves_sum(float x)
{
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// dot product of two 16-bit pairs with (1, 1), added to c: the sum of two probabilities as they are multiplied
template <bool F16> __device__ inline float pair_sum(uint32_t w, float c)
{
    if (F16) return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, w), f16x2{(_Float16)1.0f, (_Float16)1.0f}, c, false);
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w), bf16x2{(__bf16)1.0f, (__bf16)1.0f}, c, false);
}

template <int QT, int KVT, int DP, int NR, bool FULL> __global__ __launch_bounds__(64 * MANY_WAVES, 2) void attention_many_kernel(AttnArgs a)
{
    constexpr bool F16 = KVT == KV_F16, CODES = KVT == KV_E4M3;
    constexpr bool DIRECT = FULL && !CODES;
    constexpr int QTERMS = CODES && QT == ASR_F16 ? 2 : 1, PTERMS = 2;             // 16-bit terms of a value of q, of a probability
    constexpr int PITCH = DP * 2, PAIR = 128 / DP;
    constexpr int ROW_LOADS = DP / (CODES ? 16 : 8);                            // 16-byte loads of a key row
    constexpr int LOADS = MANY_KEYS * ROW_LOADS / (64 * MANY_WAVES);              // of a thread, for K and for V
    constexpr int LOAD_ROWS = 64 * MANY_WAVES / ROW_LOADS;                        // rows from one load of a thread to its next (a multiple of 16)
    __shared__ __align__(16) char s_kv[5][MANY_KEYS * PITCH];
    char(*const s_k)[MANY_KEYS * PITCH] = s_kv, (*const s_v)[MANY_KEYS * PITCH] = s_kv + 3;
    const auto turn_k = [](int row) { return (row / PAIR) & (DP / 8 - 1); };                 // of a row's 16-byte chunks
    const auto turn_v = [](int row) { return PAIR == 1 ? 4 * (row & 3) : 4 * ((row >> 1) & 1); };
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), x32 = lane & 31, half = lane >> 5;

    int64_t id = blockIdx.x;
    const int place = place_of(a.n * a.kv_heads, a.tiles * a.nsplit, id);
    const int split = (int)(id % a.nsplit), tile = a.tiles - 1 - (int)(id / a.nsplit);   // (causal: the longest rows first)
    const int b = longest_first(a, place / a.kv_heads), h = place % a.kv_heads, bh = b * a.kv_heads + h;
    const int len = keys_of(a, b), row0 = tile * MANY_ROWS * NR, wave_row0 = row0 + 32 * NR * wave, tq = queries_of<CODES>(a, b);
    int last_key = len;
    if (a.causal) last_key = min(len, max(0, len - tq + min(min(row0 + MANY_ROWS * NR - 1, a.rows - 1) / a.group, tq - 1) + 1));
    if (row0 / a.group >= tq) last_key = 0;
    const int first_lim = a.causal ? len - tq + row0 / a.group + 1 : 0x7fffffff;         // every row of this workgroup sees the keys below it
    const int all_tiles = (last_key + MANY_KEYS - 1) / MANY_KEYS, share = (all_tiles + a.nsplit - 1) / a.nsplit;
    const int t0 = split * share, t1 = min(all_tiles, t0 + share);

    // q as second operand (a negative factor is moved into it: exact)
    const float c = fmaxf(fabsf(a.c), 1e-37f);                                        // (a factor of 0 must leave -infinity what it is)
    u32x4 qf[NR][DP / 16][QTERMS];
    int lim[NR];                                                                      // this lane's rows see keys below it
#pragma unroll
    for (int t = 0; t < NR; ++t) {
        const int r = wave_row0 + 32 * t + x32, rc = min(r, a.rows - 1);
        const char* qp = a.q + (int64_t)b * a.q_stride[0] + (int64_t)(rc / a.group) * a.q_stride[1] + (int64_t)(h * a.group + rc % a.group) * a.q_stride[2];
#pragma unroll
        for (int u = 0; u < DP / 16; ++u) {
            const int at = 16 * u + 8 * half;
            u32x4 w = at < a.d && r < a.rows ? *reinterpret_cast<const u32x4*>(qp + 2 * at) : u32x4{};
            if (a.c < 0) w ^= 0x80008000u;
            if constexpr (QTERMS == 2) cut_f16(w, qf[t][u]);
            else qf[t][u][0] = w;
        }
        lim[t] = a.causal ? len - tq + min(rc / a.group, tq - 1) + 1 : len;
    }
    const int wave_first = a.causal ? len - tq + min(min(wave_row0, a.rows - 1) / a.group, tq - 1) + 1 : 0x7fffffff;      // every row of this wave sees keys below it

    const char* kb = a.k + (int64_t)b * a.k_stride[0] + (int64_t)h * a.k_stride[2];
    const char* vb = a.v + (int64_t)b * a.v_stride[0] + (int64_t)h * a.v_stride[2];
    const float* ksc = CODES ? a.k_scale + (int64_t)bh * a.scale_stride : nullptr;
    const float* vsc = CODES ? a.v_scale + (int64_t)bh * a.scale_stride : nullptr;
    const uint8_t* pad = a.pad ? a.pad + (int64_t)b * a.pad_stride : nullptr;

    // this thread's place in a tile: row and 16-byte load of it
    const int my_row = tid / ROW_LOADS, my_load = tid % ROW_LOADS;
    const int k_at = DIRECT ? (my_load ^ turn_k(my_row)) * 16 : my_load * 16, v_at = DIRECT ? (my_load ^ turn_v(my_row)) * 16 : my_load * 16;
    const bool in = FULL || my_load * 16 < a.d * (CODES ? 1 : 2);
    const mem kp = (mem)(kb + (uint64_t)my_row * (uint64_t)a.k_stride[1] + (in ? k_at : 0));
    const mem vp = (mem)(vb + (uint64_t)my_row * (uint64_t)a.v_stride[1] + (in ? v_at : 0));

    const int64_t k_step = LOAD_ROWS * a.k_stride[1], v_step = LOAD_ROWS * a.v_stride[1];

    u32x4 kr[DIRECT ? 1 : LOADS], vr[DIRECT ? 1 : LOADS];
    float ks = 1.0f, vs = 1.0f;
    // one bit for each admitted key of tile t, from this lane's flag of it (asked for a tile ahead: waiting for it costs as much as half a tile)
    const auto flag_of = [&](int t) __attribute__((always_inline)) {
        const int key = t * MANY_KEYS + lane;
        return pad && key < len ? (uint32_t)pad[key] : 0u;
    };
    const auto admitted = [&](int t, uint32_t flag) __attribute__((always_inline)) {
        if (!pad && (t + 1) * MANY_KEYS <= len) return ~(uint64_t)0;
        return (uint64_t)__ballot(t * MANY_KEYS + lane < len && flag == 0);
    };
    // where this thread's loads of tile t of K or V come from (p: its first row's place in that tile); keys past the end are read from the last one
    const auto aim = [&](int t, mem p, int64_t stride, int64_t step, mem (&x)[LOADS]) __attribute__((always_inline)) {
        const int c0 = t * MANY_KEYS;
#pragma unroll
        for (int u = 0; u < LOADS; ++u) x[u] = u ? x[u - 1] + step : p;
        if (c0 + MANY_KEYS > len) {
            asm volatile("");                                                       // (a branch: products of 64 bits in the last tile only)
#pragma unroll
            for (int u = 0; u < LOADS; ++u) x[u] += (int64_t)min(0, len - 1 - (c0 + u * LOAD_ROWS + my_row)) * stride;
        }
    };
    // ... load u of them, to registers or LDS
    const auto load = [&](const mem (&x)[LOADS], int u, u32x4* regs, uint32_t lds) __attribute__((always_inline)) {
        if constexpr (DIRECT) load_to_lds(x[u], lds + u * MANY_WAVES * 1024);
        else regs[u] = load_as<u32x4>(x[u]);
    };
    const uint32_t my_lds = lds_at(s_k[0]) + wave * 1024, tile_bytes = MANY_KEYS * PITCH;                       // where this wave's loads of K go, of V behind them
    const auto k_lds = [&](int buf) { return my_lds + buf * tile_bytes; };
    const auto v_lds = [&](int t) { return my_lds + (3 + (t & 1)) * tile_bytes; };
    // fetched registers into LDS (the caller waits and meets the other waves afterwards)
    const auto put = [&](u32x4* regs, char* lds, float scale, auto turn) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < LOADS; ++u) {
            char* row = lds + (my_row + u * LOAD_ROWS) * PITCH;
            if (!in) regs[u] = u32x4{};
            if constexpr (CODES) {
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    u32x4 x;
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        x[2 * j] = codes_bf16<false>(regs[u][2 * w + j], scale);
                        x[2 * j + 1] = codes_bf16<true>(regs[u][2 * w + j], scale);
                    }
                    *reinterpret_cast<u32x4*>(row + ((2 * my_load + w) ^ turn(my_row)) * 16) = x;
                }
            } else *reinterpret_cast<u32x4*>(row + (my_load ^ turn(my_row)) * 16) = regs[u];
        }
    };
    const auto put_k = [&](int buf) __attribute__((always_inline)) {
        if constexpr (!DIRECT) put(kr, s_k[buf], ks, turn_k);
    };
    // what is not admitted may hold anything: V = 0 meets P = 0.  What a causal call hides from some of the rows may be NaN as well: such values
    // are taken as 0 and looked up again at the end.
    uint64_t nan_seen = 0;
    const auto put_v = [&](int t, uint64_t mask) __attribute__((always_inline)) {
        if constexpr (DIRECT) {
            if (mask == ~0ull) return;
            wait_for_memory();                                                      // (a thread clears what its own loads brought)
#pragma unroll
            for (int u = 0; u < LOADS; ++u)
                if (!((mask >> (my_row + u * LOAD_ROWS)) & 1)) *reinterpret_cast<u32x4*>(&s_v[t & 1][(tid + u * 64 * MANY_WAVES) * 16]) = u32x4{};
        } else {
            if (mask != ~0ull) {
#pragma unroll
                for (int u = 0; u < LOADS; ++u)
                    if (!((mask >> (my_row + u * LOAD_ROWS)) & 1)) vr[u] = u32x4{};
            }
            if constexpr (CODES) {
                if ((t + 1) * MANY_KEYS > first_lim) {
                    uint32_t any = 0;
#pragma unroll
                    for (int u = 0; u < LOADS; ++u)
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            const uint32_t x = in ? nan_codes(vr[u][w]) : 0u;
                            any |= x;
                            vr[u][w] &= ~x;
                        }
                    nan_seen |= __ballot(any != 0);
                }
            }
            put(vr, s_v[t & 1], vs, turn_v);
        }
    };
    const auto meet = [&]() __attribute__((always_inline)) {
        wait_for_memory();
        __syncthreads();
    };

    // where the reads of a tile go: K row x32 of a half, 16-byte chunk 2 u + half of it; V: lane group lane / 16 reads four keys, 4 half + 0 .. 3, of columns
    // 16 (group % 2) + 0 .. 15, its lane i key i / 4 and four columns from 4 (i % 4)
    const int k_read = x32 * PITCH + 16 * (half ^ turn_k(x32)), v_row = 4 * half + ((lane & 15) >> 2);
    const int v_read = v_row * PITCH + 8 * (lane & 1) + 16 * ((2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ turn_v(v_row));
    f32x16 o[NR][DP / 32];
    float m[NR], l[NR], top[NR];
#pragma unroll
    for (int t = 0; t < NR; ++t) {
        m[t] = NO_MAX;
        l[t] = 0.0f;
#pragma unroll
        for (int i = 0; i < DP / 32; ++i) o[t][i] = f32x16{};
    }
    uint64_t mask = 0;
    constexpr int AHEAD = 4, N = DP / 16;                                            // N products of a half's scores, and of its output, for each row tile
    u32x4 kf[N];                                                                     // of the next half's scores, AHEAD of them read beforehand

    // LDS addresses of the reads, renewed when a tile is first read (its halves differ by a constant in the instruction)
    typedef const __attribute__((address_space(3))) char* lds_mem;
    const lds_mem kv_lds = (lds_mem)s_kv[0];
    lds_mem kf_at[N], vf_at[N / 2];
    const auto k_frag = [&](int buf, int sub, int u) __attribute__((always_inline)) {
        if (sub == 0) {
            kf_at[u] = kv_lds + buf * (MANY_KEYS * PITCH) + (k_read ^ (32 * u));
            asm volatile("" : "+v"(kf_at[u]));
        }
        return *(const __attribute__((address_space(3))) u32x4*)(kf_at[u] + 32 * sub * PITCH);
    };
    const auto score = [&](const u32x4& k, int r, int u, f32x16& s) __attribute__((always_inline)) {
        if (u == 0) s = f32x16{};
#pragma unroll
        for (int term = QTERMS - 1; term >= 0; --term) s = mfma32<F16>(k, qf[r][u][term], s);
    };
    const auto most = [&](const f32x16& s) __attribute__((always_inline)) {
        float x = s[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) x = fmaxf(x, s[i]);
        return halves_max(x);
    };
    // The exponentials take fma(s, c, -m) with m a rounded product: none is above that of the maximum but by half a step of m.  Where that step is more than a few hundredths (FAR) scores
    // are multiplied, rounded like m, and m subtracted: their steps would otherwise pass the range of P.
    constexpr float LIFT = F16 ? LIFT16 : 0.0f, FAR = 0x1p20f;
    uint64_t far = 0, grow = 0;                                                      // the lanes whose rows' m is that far; ... or whose maximum has grown
    const auto grown_by = [&](int r) __attribute__((always_inline)) { return fmaf(top[r], c, -m[r]); };
    const auto grows = [&]() __attribute__((always_inline)) {
        bool x = grown_by(0) > SLACK + LIFT;
        if (NR > 1) x |= grown_by(NR - 1) > SLACK + LIFT;
        return __ballot(x) | far;
    };
    // soft-max and output of half `sub` of tile t from its scores s with their maxima `top`, and the scores of the half behind it.  The products are laid out
    // as slots, one for each, and between them, in the order in which it is to be issued (the compiler left to itself puts all products on one
    // side): the LDS reads AHEAD products before their own; the exponentials, over the slots of the scores and of the output's first half, whose probabilities
    // the second half multiplies - each value a stage further a slot later, so that none waits for the one before; the maxima of the new scores; and
    // the next tiles' loads, one a slot (all at once they fill the memory pipe's queue and the wave waits).
    const auto step = [&](int t, int sub, f32x16 (&s)[NR], int next_buf, int buf_after, f32x16 (&next)[NR], auto bring) __attribute__((always_inline)) {
        const int c0 = t * MANY_KEYS + 32 * sub;
        const uint32_t bits = (uint32_t)(mask >> (32 * sub));
        if (bits != ~0u || c0 + 32 > wave_first) {
            asm volatile("");                                                       // (a branch, not 16 selects in every step)
            const uint32_t mine = bits >> (4 * half);
#pragma unroll
            for (int r = 0; r < NR; ++r) {
#pragma unroll
                for (int i = 0; i < 16; ++i) s[r][i] = admit(s[r][i], spread_bit(mine, 8 * (i >> 2) + (i & 3)));
                if (c0 + 32 > wave_first) {                                         // (causal calls)
                    asm volatile("");
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[r][i] = c0 + 8 * (i >> 2) + 4 * half + (i & 3) < lim[r] ? s[r][i] : NEG_INF;
                }
                top[r] = most(s[r]);
            }
            grow = grows();
        }
        float factor = c;
        if (grow) {
            bool is_far = false;
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                const float t = product(top[r], c), grown = fmaxf(grown_by(r), t - m[r]) > SLACK + LIFT ? t - LIFT : m[r], f = rescale(m[r], grown);
                m[r] = grown;
                is_far |= fabsf(grown) > FAR && grown != NO_MAX;
                l[r] *= f;
#pragma unroll
                for (int i = 0; i < DP / 32; ++i)
#pragma unroll
                    for (int j = 0; j < 16; ++j) o[r][i][j] *= f;
            }
            far = __ballot(is_far);
            if (far) {
                factor = 1.0f;
#pragma unroll
                for (int r = 0; r < NR; ++r)
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[r][i] = product(s[r][i], c);
            }
        }
        const auto v_frag = [&](int q) __attribute__((always_inline)) {
            const int i = q % (N / 2);
            if (sub == 0 && q < N / 2) {
                vf_at[i] = kv_lds + (3 + (t & 1)) * (MANY_KEYS * PITCH) + (v_read ^ (64 * i));
                asm volatile("" : "+v"(vf_at[i]));
            }
            const lds_mem p = vf_at[i] + (32 * sub + 16 * (q / (N / 2))) * PITCH;
            const u32x2 lo = lds_read_transposed(p), hi = lds_read_transposed(p + 8 * PITCH);
            return u32x4{lo[0], lo[1], hi[0], hi[1]};
        };
        constexpr int SLOTS = N * NR, VALUES = 16 * NR, FROM = SLOTS / 4 < 2 ? 1 : SLOTS / 2 - 2 < 2 ? SLOTS / 2 - 2 : 2;
        u32x4 vf[N];
        float x[NR][16], most_of[NR][2];
        uint32_t pf[PTERMS][NR][8];
        // value e in the order in which they are needed: the first 16 keys' of every row tile, then the others'
        const auto row_of = [](int e) { return e / 8 % NR; };
        const auto key_of = [](int e) { return 8 * (e / (8 * NR)) + e % 8; };
        // values whose exponential is taken by the end of slot w: all before the output's second half
        const auto taken = [](int w) { return w < 0 ? 0 : VALUES * (w + 1) >= VALUES * (SLOTS * 3 / 2 - 1) ? VALUES : (VALUES * (w + 1) + SLOTS * 3 / 2 - 2) / (SLOTS * 3 / 2 - 1); };
        const auto begin = [&](int e) __attribute__((always_inline)) { x[row_of(e)][key_of(e)] = fmaf(s[row_of(e)][key_of(e)], factor, -m[row_of(e)]); };
        const auto between = [&](int w) __attribute__((always_inline)) {
            if (w >= SLOTS * 3 / 2) return;
#pragma unroll
            for (int e = taken(w); e < taken(w + 1); ++e) begin(e);
#pragma unroll
            for (int e = taken(w - 1); e < taken(w); ++e) x[row_of(e)][key_of(e)] = __builtin_amdgcn_exp2f(x[row_of(e)][key_of(e)]);
#pragma unroll
            for (int i = taken(w - 2) / 2; i < taken(w - 1) / 2; ++i) {
                const int r = row_of(2 * i), j = key_of(2 * i);
                const uint32_t w = pack16<F16>(x[r][j], x[r][j + 1]);
                const f32x2 y = unpack16<F16>(w);
                const uint32_t rest = pack16<F16>(x[r][j] - y[0], x[r][j + 1] - y[1]);
                pf[0][r][j / 2] = w;
                pf[1][r][j / 2] = rest;
                l[r] = pair_sum<F16>(rest, pair_sum<F16>(w, l[r]));
            }
        };
#pragma unroll
        for (int e = 0; e < taken(0); ++e) begin(e);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int w = 0; w < SLOTS; ++w) {
            const int u = w / NR, r = w % NR;
            if (r == 0) {
                if (u + AHEAD < N) kf[u + AHEAD] = k_frag(next_buf, sub ^ 1, u + AHEAD);
                else vf[u + AHEAD - N] = v_frag(u + AHEAD - N);
            }
            score(kf[u], r, u, next[r]);
            bring(w);
            __builtin_amdgcn_sched_barrier(0);
            between(w);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int w = 0; w < SLOTS; ++w) {
            const int q = w / NR, r = w % NR, k16 = q / (N / 2), i = q % (N / 2);
            if (r == 0) {
                if (q + AHEAD < N) vf[q + AHEAD] = v_frag(q + AHEAD);
                else kf[q + AHEAD - N] = k_frag(buf_after, sub, q + AHEAD - N);
            }
#pragma unroll
            for (int term = PTERMS - 1; term >= 0; --term) {
                const uint32_t* x = pf[term][r] + 4 * k16;
                o[r][i] = mfma32<F16>(vf[q], u32x4{x[0], x[1], x[2], x[3]}, o[r][i]);
            }
            bring(SLOTS + w);
            __builtin_amdgcn_sched_barrier(0);
            between(SLOTS + w);
            if (w >= FROM && w < FROM + SLOTS / 2) {
#pragma unroll
                for (int e = VALUES * (w - FROM) / (SLOTS / 2); e < VALUES * (w + 1 - FROM) / (SLOTS / 2); e += 2) {
                    float(&y)[2] = most_of[e / 16];
                    const f32x16& z = next[e / 16];
                    if (e % 16 == 0) y[0] = z[0], y[1] = z[1];
                    else if (e % 4 == 0) y[0] = fmaxf(fmaxf(y[0], z[e % 16]), z[e % 16 + 1]);
                    else y[1] = fmaxf(fmaxf(y[1], z[e % 16]), z[e % 16 + 1]);
                }
#pragma unroll
                for (int r = 0; r < NR; ++r)
                    if (VALUES * (w + 1 - FROM) / (SLOTS / 2) > 16 * r + 3 && VALUES * (w - FROM) / (SLOTS / 2) < 16 * (r + 1))
                        asm volatile("" : "+v"(most_of[r][0]), "+v"(most_of[r][1]));                  // (here, not behind the last product)
            }
            if (w == FROM + SLOTS / 2) {
#pragma unroll
                for (int r = 0; r < NR; ++r) {
                    top[r] = halves_max(fmaxf(most_of[r][0], most_of[r][1]));
                    asm volatile("" : "+v"(top[r]));
                }
            }
            if (w == SLOTS - 1) grow = grows();
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    if (t0 < t1) {
        f32x16 sa[NR], sb[NR];
        mem from[LOADS], v_places[LOADS];
        int now = 0, behind = 1, fetched = 2;                                           // K buffers of tiles t, t + 1, t + 2
        mask = admitted(t0, flag_of(t0));
        // this thread's first row of the tile that is loaded next
        mem k_from = kp + (int64_t)t0 * MANY_KEYS * a.k_stride[1], v_from = vp + (int64_t)t0 * MANY_KEYS * a.v_stride[1];
        const int64_t k_tile = MANY_KEYS * a.k_stride[1], v_tile = MANY_KEYS * a.v_stride[1];
        const auto bring_k = [&](int t, int buf) __attribute__((always_inline)) {
            aim(t, k_from, a.k_stride[1], k_step, from);
            if constexpr (CODES) ks = ksc[t];
#pragma unroll
            for (int u = 0; u < LOADS; ++u) load(from, u, kr, k_lds(buf));
            put_k(buf);
        };
        bring_k(t0, now);
        aim(t0, v_from, a.v_stride[1], v_step, from);
        if constexpr (CODES) vs = vsc[t0];
#pragma unroll
        for (int u = 0; u < LOADS; ++u) load(from, u, vr, v_lds(t0));
        put_v(t0, mask);
        if (t0 + 1 < t1) {
            k_from += k_tile;
            bring_k(t0 + 1, behind);
        }
        meet();
#pragma unroll
        for (int r = 0; r < NR; ++r) {
#pragma unroll
            for (int u = 0; u < N; ++u) score(k_frag(now, 0, u), r, u, sa[r]);
            top[r] = most(sa[r]);
        }
        grow = grows();
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) kf[u] = k_frag(now, 1, u);
        for (int t = t0; t < t1; ++t) {
            // (behind the last tile the last one is loaded again, and scores are taken of what LDS holds: neither is used)
            const int tk = min(t + 2, t1 - 1), tv = min(t + 1, t1 - 1);
            const uint32_t next_flag = flag_of(tv);
            if (t + 2 < t1) k_from += k_tile;
            if (t + 1 < t1) v_from += v_tile;
            aim(tk, k_from, a.k_stride[1], k_step, from);
            aim(tv, v_from, a.v_stride[1], v_step, v_places);
            if constexpr (CODES) {
                ks = ksc[tk];
                vs = vsc[tv];
            }
            step(t, 0, sa, now, behind, sb, [&](int w) __attribute__((always_inline)) {
                if (w % NR) return;
                if (w / NR < LOADS) load(v_places, w / NR, vr, v_lds(t + 1));
                else if (w / NR < 2 * LOADS) load(from, w / NR - LOADS, kr, k_lds(fetched));
            });
            step(t, 1, sb, behind, behind, sa, [](int) {});
            if (t + 1 < t1) {
                put_k(fetched);
                mask = admitted(t + 1, next_flag);
                put_v(t + 1, mask);
                meet();
                const int free = now;
                now = behind;
                behind = fetched;
                fetched = free;
            }
        }
        wait_for_memory();                                                              // (no load into LDS may outlive its workgroup)
        if constexpr (!CODES) {
            bool lost = false;
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                f32x4 z{};
#pragma unroll
                for (int i = 0; i < DP / 32; ++i)
#pragma unroll
                    for (int j = 0; j < 16; ++j) z[j & 3] = fmaf(o[r][i][j], 0.0f, z[j & 3]);
                z[0] += z[1] + z[2] + z[3];
                lost |= z[0] != z[0] && halves_sum(l[r]) < __builtin_inff();
            }
            if (__ballot(lost)) {
                Seen seen[DP / 32];
                for (int key = t0 * MANY_KEYS; key < min(t1 * MANY_KEYS, len); ++key) {
                    if (pad && pad[key]) continue;
                    const mem p = (mem)vb + (int64_t)key * a.v_stride[1];
#pragma unroll
                    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            const int at = 32 * i + 8 * (j >> 2) + 4 * half + (j & 3);
                            if (at < a.d) seen[i].template add<KVT>(p + 2 * at, j);
                        }
                }
#pragma unroll
                for (int r = 0; r < NR; ++r)
#pragma unroll
                    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
                        for (int j = 0; j < 16; ++j) o[r][i][j] = seen[i].instead_of(o[r][i][j], j);
            }
        }
        if constexpr (CODES) {
            if (a.causal) {
                uint32_t* waves = reinterpret_cast<uint32_t*>(s_k);                     // (LDS is full: two workgroups share it)
                __syncthreads();
                if (lane == 0) waves[wave] = nan_seen != 0;
                __syncthreads();
                if (waves[0] | waves[1] | waves[2] | waves[3]) {
                    // where this lane's row sees a NaN its sum is one
                    for (int key = max(t0, first_lim >> 6) * MANY_KEYS; key < min(t1 * MANY_KEYS, len); ++key)
#pragma unroll
                        for (int i = 0; i < DP / 32; ++i)
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const int at = 32 * i + 8 * j + 4 * half;
                                const uint32_t x = at < a.d ? nan_codes(load_as<uint32_t>((mem)vb + (int64_t)key * a.v_stride[1] + at)) : 0u;
#pragma unroll
                                for (int e = 0; e < 4; ++e)
#pragma unroll
                                    for (int r = 0; r < NR; ++r)
                                        o[r][i][4 * j + e] = key < lim[r] && (x >> (8 * e)) & 1 ? __builtin_nanf("") : o[r][i][4 * j + e];
                            }
                }
            }
        }
    }

#pragma unroll
    for (int t = 0; t < NR; ++t) {
        const int r = wave_row0 + 32 * t + x32;
        float sum = halves_sum(l[t]);
        if (r >= a.rows) continue;
        if (CODES && r / a.group >= tq) {
            sum = 0.0f;
#pragma unroll
            for (int i = 0; i < DP / 32; ++i) o[t][i] = f32x16{};
        }
        if (a.nsplit > 1) {
            float* ws = a.ws + (((int64_t)split * a.n * a.kv_heads + bh) * a.rows + r) * (a.d + 4);
            if (half == 0) { ws[0] = m[t]; ws[1] = sum; }
#pragma unroll
            for (int i = 0; i < DP / 32; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int at = 32 * i + 8 * j + 4 * half;
                    if (at < a.d) *reinterpret_cast<f32x4*>(ws + 4 + at) = f32x4{o[t][i][4 * j], o[t][i][4 * j + 1], o[t][i][4 * j + 2], o[t][i][4 * j + 3]};
                }
            continue;
        }
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        char* op = a.out + (int64_t)b * a.out_stride[0] + (int64_t)(r / a.group) * a.out_stride[1] + (int64_t)(h * a.group + r % a.group) * a.out_stride[2];
#pragma unroll
        for (int i = 0; i < DP / 32; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int at = 32 * i + 8 * j + 4 * half;
                if (at >= a.d) continue;
                u32x2 w;
                w[0] = pack16<QT == ASR_F16>(o[t][i][4 * j] * inv, o[t][i][4 * j + 1] * inv);
                w[1] = pack16<QT == ASR_F16>(o[t][i][4 * j + 2] * inv, o[t][i][4 * j + 3] * inv);
                *reinterpret_cast<u32x2*>(op + 2 * at) = w;
            }
    }
}

// Joins the shares of a long key axis.  A row has 32 G threads: four values each, every G-th share (a row's shares are far apart, so the loads of many
// have to be in flight: with one thread for all 64 shares of a row this took 35 us of a 50 us call), then the G sums in LDS.
template <int QT, int G> __global__ __launch_bounds__(256) void attention_join_kernel(AttnArgs a)
{
    constexpr int ROWS = 8 / G;
    __shared__ __align__(16) float s_acc[ROWS][G][32][4];
    __shared__ float s_sum[ROWS][G];
    const int lane = threadIdx.x & 31, g = threadIdx.x / 32 % G, slot = threadIdx.x / (32 * G), at = 4 * lane;
    const int64_t rows = (int64_t)a.n * a.kv_heads * a.rows, split_stride = rows * (a.d + 4);
    for (int64_t row0 = (int64_t)blockIdx.x * ROWS; row0 < rows; row0 += (int64_t)gridDim.x * ROWS) {
        const int64_t row = row0 + slot < rows ? row0 + slot : rows - 1;
        const float* ws = a.ws + row * (a.d + 4);
        float top = NO_MAX;
        for (int s = lane; s < a.nsplit; s += 32) top = fmaxf(top, ws[s * split_stride]);
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 32));
        float sum = 0.0f;
        f32x4 acc{};
#pragma unroll 4
        for (int s = g; s < a.nsplit; s += G) {
            const float* p = ws + s * split_stride;
            const float f = rescale(p[0], top);
            sum += p[1] * f;
            acc += scaled(*reinterpret_cast<const f32x4*>(p + 4 + (at < a.d ? at : 0)), f);
        }
        *reinterpret_cast<f32x4*>(s_acc[slot][g][lane]) = acc;
        if (lane == 0) s_sum[slot][g] = sum;
        __syncthreads();
        if (g == 0 && at < a.d && row0 + slot < rows) {
#pragma unroll
            for (int i = 1; i < G; ++i) {
                acc += *reinterpret_cast<const f32x4*>(s_acc[slot][i][lane]);
                sum += s_sum[slot][i];
            }
            acc = sum == 0.0f ? f32x4{} : acc * (1.0f / sum);
            const int r = (int)(row % a.rows), bh = (int)(row / a.rows), b = bh / a.kv_heads, h = bh % a.kv_heads;
            char* op = a.out + (int64_t)b * a.out_stride[0] + (int64_t)(r / a.group) * a.out_stride[1] +
                       (int64_t)(h * a.group + r % a.group) * a.out_stride[2] + at * (QT == ASR_F32 ? 4 : 2);
            if constexpr (QT == ASR_F32) *reinterpret_cast<f32x4*>(op) = acc;
            else {
                u32x2 w;
                w[0] = pack16<QT == ASR_F16>(acc[0], acc[1]);
                w[1] = pack16<QT == ASR_F16>(acc[2], acc[3]);
                *reinterpret_cast<u32x2*>(op) = w;
            }
        }
        __syncthreads();
    }
}

// ---- the choice of kernel -----------------------------------------------------------------------------------------------
struct Plan {
    int rows, tiles, nq, nsplit;
    bool many;
    int64_t ws_bytes;
};

// terms: 16-bit terms of a value of q; 3: float32
Plan plan_of(int64_t n, int64_t tq, int64_t tk, int64_t heads, int64_t kv_heads, int64_t d, int terms)
{
    Plan p{};
    p.rows = (int)(tq * (heads / kv_heads));
    // us of few rows and of many: 50 x 16 heads of 64 over 1000 states, 64 rows: 50.7 and 56, 80: 67 and 58; 8 x 16 of them, 64: 14.4 and 22, 128: 18 and 23; 16 x 8 heads of 128
    // over 2000, 33: 40 and 36, 64: 42 and 39, 80: 52 and 41; 2 x 8 of them over 4096, 64: 15.8 and 18.5, 96: 21.4 and 20.4; over codes 8 x 8 heads of 128 and 4096 tokens, 64: 33 and
    // 33, 80: 40 and 35; 32 x 16 of 64 and 1024, 64: 23 and 32, 80: 32 and 32; the same with float16 queries, 64: 30 and 35, 80: 37 and 33
    p.many = terms < 3 && p.rows > 64;
    if (p.many) {
        // two row tiles a wave where its registers hold them and workgroups of twice the rows still give every compute unit two, without many idle rows (8 x 512
        // queries of 32 heads over 4096 states of 8 heads of 64: 230 us with one, 220 with two, though those spill eleven registers, over codes 22; heads of 128 would leave one
        // wave a SIMD)
        const int64_t tiles = (p.rows + MANY_ROWS - 1) / MANY_ROWS;
        p.nq = terms == 1 && d == 64 && (tiles % 2 == 0 || tiles >= 8) && n * kv_heads * ((tiles + 1) / 2) >= 512 ? 2 : 1;
        p.tiles = (int)((tiles + p.nq - 1) / p.nq);
        // shares of at least eight tiles, with few workgroups of four where there are twelve (joining them is a launch: 4 x 100 queries of 16 heads over 1000 states,
        // 64 workgroups, 22.8 us with eight and 18.8 with four; 2 x 100 over 1500, 32 workgroups, 22.8 and 16.3; 4 x 80 of 8 heads of 128 over 1000, 29 and 19.6; 8 x 100 over
        // 800, 128 workgroups, 19.7 and 23.8)
        const int64_t wgs = n * kv_heads * p.tiles, most = wgs <= 64 && tk >= 12 * MANY_KEYS ? tk / (MANY_KEYS * 4) : tk / (MANY_KEYS * 8);
        int64_t split = wgs > 0 ? 512 / wgs : 1;
        if (split > most) split = most;
        if (split > 16) split = 16;
        p.nsplit = split < 1 ? 1 : (int)split;
        p.ws_bytes = p.nsplit > 1 ? (int64_t)p.nsplit * n * kv_heads * p.rows * (d + 4) * 4 : 0;
        return p;
    }
    p.nq = p.rows > 16 ? 2 : 1;
    p.tiles = (p.rows + 16 * p.nq - 1) / (16 * p.nq);
    // shares of the key axis: enough workgroups for the chip (three for each of 256 compute units: 16 x 4 queries over 4096 f32 keys 41 us with one, 31 with
    // two, 29 with three), each with at least four chunks of 32 keys for each wave, or two where a few workgroups have a short axis (one token over 1000 f32 states,
    // 16 workgroups: 17 us and 12.2 with two; 14 x 25 over 832 bf16 tokens, 70: 12.9 and 11.6; but 8 x 10 over 600, 128: 8.5 and 10.2; 7 x 29 x 8 over 4587: 28.7 and 34)
    const int64_t wgs = n * kv_heads * p.tiles, most = tk / (FEW_WAVES * 32 * (wgs <= 80 && tk <= 2048 ? 2 : 4));
    int64_t split = wgs > 0 ? (768 + wgs - 1) / wgs : 1;
    if (split > most) split = most;
    if (split > 64) split = 64;
    p.nsplit = split < 1 ? 1 : (int)split;
    p.ws_bytes = p.nsplit > 1 ? (int64_t)p.nsplit * n * kv_heads * p.rows * (d + 4) * 4 : 0;
    return p;
}

template <int QT, int KVT> hipError_t launch_few(const AttnArgs& a, int nq, hipStream_t s)
{
    const dim3 grid((uint32_t)((int64_t)a.n * a.kv_heads * a.nsplit * a.tiles)), block(64 * FEW_WAVES);
    if (a.d == 64) return nq == 1 ? ops_launch(attention_few_kernel<QT, KVT, 64, 1, true>, grid, block, s, a) : ops_launch(attention_few_kernel<QT, KVT, 64, 2, true>, grid, block, s, a);
    if (a.d == 128) return nq == 1 ? ops_launch(attention_few_kernel<QT, KVT, 128, 1, true>, grid, block, s, a) : ops_launch(attention_few_kernel<QT, KVT, 128, 2, true>, grid, block, s, a);
    if (a.d < 64) return nq == 1 ? ops_launch(attention_few_kernel<QT, KVT, 64, 1, false>, grid, block, s, a) : ops_launch(attention_few_kernel<QT, KVT, 64, 2, false>, grid, block, s, a);
    return nq == 1 ? ops_launch(attention_few_kernel<QT, KVT, 128, 1, false>, grid, block, s, a) : ops_launch(attention_few_kernel<QT, KVT, 128, 2, false>, grid, block, s, a);
}

template <int QT, int KVT> hipError_t launch_many(const AttnArgs& a, int nr, hipStream_t s)
{
    const dim3 grid((uint32_t)((int64_t)a.n * a.kv_heads * a.nsplit * a.tiles)), block(64 * MANY_WAVES);
    if constexpr (!(QT == ASR_F16 && KVT == KV_E4M3))
        if (a.d == 64 && nr == 2) return ops_launch(attention_many_kernel<QT, KVT, 64, 2, true>, grid, block, s, a);
    if (a.d == 64) return ops_launch(attention_many_kernel<QT, KVT, 64, 1, true>, grid, block, s, a);
    if (a.d == 128) return ops_launch(attention_many_kernel<QT, KVT, 128, 1, true>, grid, block, s, a);
    return a.d < 64 ? ops_launch(attention_many_kernel<QT, KVT, 64, 1, false>, grid, block, s, a) : ops_launch(attention_many_kernel<QT, KVT, 128, 1, false>, grid, block, s, a);
}

template <int QT> hipError_t launch_join(const AttnArgs& a, hipStream_t s)
{
    const int64_t rows = (int64_t)a.n * a.kv_heads * a.rows, blocks = a.nsplit >= 8 ? rows : (rows + 3) / 4;
    const dim3 grid((uint32_t)(blocks < 65536 ? blocks : 65536)), block(256);
    return a.nsplit >= 8 ? ops_launch(attention_join_kernel<QT, 8>, grid, block, s, a) : ops_launch(attention_join_kernel<QT, 2>, grid, block, s, a);
}

template <int QT, int KVT> int attend(const char* what, AttnArgs& a, const Plan& p, void* ws, int64_t ws_bytes, hipStream_t s)
{
    a.rows = p.rows;
    a.tiles = p.tiles;
    a.nsplit = p.nsplit;
    if (p.ws_bytes > 0) {
        if (!ws || ws_bytes < p.ws_bytes) return ops_fail(ASR_ERR_CAPACITY, "%s: the workspace must hold %lld bytes", what, (long long)p.ws_bytes);
        if (reinterpret_cast<uintptr_t>(ws) & 15) return ops_fail(ASR_ERR_ARG, "%s: the workspace must be 16-byte aligned", what);
        a.ws = static_cast<float*>(ws);
    }
    hipError_t e;
    if constexpr (QT != ASR_F32) e = p.many ? launch_many<QT, KVT>(a, p.nq, s) : launch_few<QT, KVT>(a, p.nq, s);
    else e = launch_few<QT, KVT>(a, p.nq, s);
    if (e == hipSuccess && p.nsplit > 1) e = launch_join<QT>(a, s);
    return ops_launched(what, e);
}

// what both operators ask of their sizes; null: fine
const char* bad_sizes(int64_t n, int64_t tq, int64_t tk, int64_t heads, int64_t kv_heads, int64_t d, int64_t d_step)
{
    if (n < 0 || tq < 0 || tk < 0) return "negative sizes";
    if (heads < 1 || kv_heads < 1 || heads % kv_heads) return "heads must be a multiple of kv_heads";
    if (d < d_step || d > 128 || d % d_step) return d_step == 8 ? "d must be a multiple of 8 in 8..128" : "d must be a multiple of 16 in 16..128";
    if (tk > 0x7fffffff - 64 || tq * heads > 0x7fffffff / 2) return "too many query rows or keys";
    const int64_t rows = tq * (heads / kv_heads);
    // workgroups of 256 threads in one grid dimension, whatever the split
    if (n * kv_heads > (1 << 22) || n * kv_heads * ((rows + 15) / 16) > (1 << 22)) return "too many sequences, heads and query rows for one call";
    return nullptr;
}

bool nonnegative(const int64_t* s) { return s[0] >= 0 && s[1] >= 0 && s[2] >= 0; }

}  // namespace

extern "C" {

int64_t asr_cross_attention_workspace(int32_t n, int32_t tq, int32_t tk, int32_t heads, int32_t kv_heads, int32_t d, int32_t dtype)
{
    if (bad_sizes(n, tq, tk, heads, kv_heads, d, 8) || !ops_dtype_ok(dtype)) return 0;
    return plan_of(n, tq, tk, heads, kv_heads, d, dtype == ASR_F32 ? 3 : 1).ws_bytes;
}

int asr_cross_attention(const asr_cross_attention_args* a, void* stream)
{
    if (!a) return ops_fail(ASR_ERR_ARG, "null argument");
    if (const char* why = bad_sizes(a->n, a->tq, a->tk, a->heads, a->kv_heads, a->d, 8)) return ops_fail(ASR_ERR_ARG, "cross_attention: %s", why);
    if (!ops_dtype_ok(a->dtype)) return ops_fail(ASR_ERR_ARG, "cross_attention: unknown dtype %d", a->dtype);
    if (!isfinite(a->scale * LOG2E)) return ops_fail(ASR_ERR_ARG, "cross_attention: the scale must be finite");
    if (a->n == 0 || a->tq == 0) return ASR_OK;
    if (!a->q || !a->out || (a->tk > 0 && (!a->k || !a->v))) return ops_fail(ASR_ERR_ARG, "cross_attention: null argument");
    if (!nonnegative(a->q_stride) || !nonnegative(a->k_stride) || !nonnegative(a->v_stride) || !nonnegative(a->out_stride) || a->pad_stride < 0)
        return ops_fail(ASR_ERR_ARG, "cross_attention: negative stride");
    if (!ops_rows16(a->q, a->q_stride, a->n, a->tq, a->heads, a->dtype) || !ops_rows16(a->out, a->out_stride, a->n, a->tq, a->heads, a->dtype) ||
        (a->tk > 0 && (!ops_rows16(a->k, a->k_stride, a->n, a->tk, a->kv_heads, a->dtype) ||
                       !ops_rows16(a->v, a->v_stride, a->n, a->tk, a->kv_heads, a->dtype))))
        return ops_fail(ASR_ERR_ARG, "cross_attention: every row of q, k, v and out must start on 16 bytes");
    AttnArgs x{};
    const int64_t size = ops_dtype_size(a->dtype);
    x.q = static_cast<const char*>(a->q); x.k = static_cast<const char*>(a->k); x.v = static_cast<const char*>(a->v);
    x.out = static_cast<char*>(a->out);
    x.lens = a->lens; x.pad = a->pad; x.pad_stride = a->pad_stride;
    for (int i = 0; i < 3; ++i) {
        x.q_stride[i] = a->q_stride[i] * size; x.out_stride[i] = a->out_stride[i] * size;
        x.k_stride[i] = a->k_stride[i] * size; x.v_stride[i] = a->v_stride[i] * size;
    }
    x.n = a->n; x.tq = a->tq; x.tk = a->tk; x.kv_heads = a->kv_heads; x.group = a->heads / a->kv_heads; x.d = a->d;
    x.c = a->scale * LOG2E;
    const Plan p = plan_of(a->n, a->tq, a->tk, a->heads, a->kv_heads, a->d, a->dtype == ASR_F32 ? 3 : 1);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (a->dtype == ASR_F32) return attend<ASR_F32, KV_F32>("cross_attention", x, p, a->workspace, a->workspace_bytes, s);
    if (a->dtype == ASR_BF16) return attend<ASR_BF16, KV_BF16>("cross_attention", x, p, a->workspace, a->workspace_bytes, s);
    return attend<ASR_F16, KV_F16>("cross_attention", x, p, a->workspace, a->workspace_bytes, s);
}

int64_t asr_kv8_attention_workspace(int32_t n, int32_t tq, int32_t capacity, int32_t heads, int32_t kv_heads, int32_t d, int32_t dtype)
{
    if (bad_sizes(n, tq, capacity, heads, kv_heads, d, 16) || !ops_dtype_ok(dtype)) return 0;
    return plan_of(n, tq, capacity, heads, kv_heads, d, dtype == ASR_F32 ? 3 : dtype == ASR_F16 ? 2 : 1).ws_bytes;
}

int asr_kv8_attention_counts(const asr_kv8_attention_args* a, const int32_t* counts, void* stream)
{
    if (!a) return ops_fail(ASR_ERR_ARG, "null argument");
    if (const char* why = bad_sizes(a->n, a->tq, a->capacity, a->heads, a->kv_heads, a->d, 16)) return ops_fail(ASR_ERR_ARG, "kv8_attention: %s", why);
    if (a->capacity % ASR_KV8_BLOCK) return ops_fail(ASR_ERR_ARG, "kv8_attention: the capacity must be a multiple of %d tokens", ASR_KV8_BLOCK);
    if (!ops_dtype_ok(a->dtype)) return ops_fail(ASR_ERR_ARG, "kv8_attention: unknown dtype %d", a->dtype);
    if (!isfinite(a->scale * LOG2E)) return ops_fail(ASR_ERR_ARG, "kv8_attention: the scale must be finite");
    if (a->n == 0 || a->tq == 0) return ASR_OK;
    if (!a->q || !a->out || !a->lens || (a->capacity > 0 && (!a->k_cache || !a->v_cache || !a->k_scale || !a->v_scale)))
        return ops_fail(ASR_ERR_ARG, "kv8_attention: null argument");
    if (!nonnegative(a->q_stride) || !nonnegative(a->out_stride) || a->cache_stride[0] < 0 || a->cache_stride[1] < 0)
        return ops_fail(ASR_ERR_ARG, "kv8_attention: negative stride");
    if (!ops_rows16(a->q, a->q_stride, a->n, a->tq, a->heads, a->dtype) || !ops_rows16(a->out, a->out_stride, a->n, a->tq, a->heads, a->dtype))
        return ops_fail(ASR_ERR_ARG, "kv8_attention: every row of q and out must start on 16 bytes");
    if (((reinterpret_cast<uintptr_t>(a->k_cache) | reinterpret_cast<uintptr_t>(a->v_cache)) & 15) || a->cache_stride[0] % 16 || a->cache_stride[1] % 16)
        return ops_fail(ASR_ERR_ARG, "kv8_attention: cache rows must start on 16 bytes");
    AttnArgs x{};
    const int64_t size = ops_dtype_size(a->dtype);
    x.q = static_cast<const char*>(a->q); x.out = static_cast<char*>(a->out);
    x.k = reinterpret_cast<const char*>(a->k_cache); x.v = reinterpret_cast<const char*>(a->v_cache);
    x.k_scale = a->k_scale; x.v_scale = a->v_scale; x.scale_stride = a->capacity / ASR_KV8_BLOCK;
    x.lens = a->lens; x.counts = counts;
    for (int i = 0; i < 3; ++i) { x.q_stride[i] = a->q_stride[i] * size; x.out_stride[i] = a->out_stride[i] * size; }
    x.k_stride[0] = x.v_stride[0] = a->cache_stride[0];
    x.k_stride[1] = x.v_stride[1] = a->d;
    x.k_stride[2] = x.v_stride[2] = a->cache_stride[1];
    x.n = a->n; x.tq = a->tq; x.tk = a->capacity; x.kv_heads = a->kv_heads; x.group = a->heads / a->kv_heads; x.d = a->d;
    x.causal = a->causal ? 1 : 0;
    x.c = a->scale * LOG2E;
    const Plan p = plan_of(a->n, a->tq, a->capacity, a->heads, a->kv_heads, a->d, a->dtype == ASR_F32 ? 3 : a->dtype == ASR_F16 ? 2 : 1);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (a->dtype == ASR_F32) return attend<ASR_F32, KV_E4M3>("kv8_attention", x, p, a->workspace, a->workspace_bytes, s);
    if (a->dtype == ASR_BF16) return attend<ASR_BF16, KV_E4M3>("kv8_attention", x, p, a->workspace, a->workspace_bytes, s);
    return attend<ASR_F16, KV_E4M3>("kv8_attention", x, p, a->workspace, a->workspace_bytes, s);
}

int asr_kv8_attention(const asr_kv8_attention_args* a, void* stream) { return asr_kv8_attention_counts(a, nullptr, stream); }

}  // extern "C"
