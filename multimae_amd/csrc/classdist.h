// Class distributions: log probabilities of given classes with entropy and top alternatives (forward and backward), and
// distillation from a teacher's top classes (loss and gradient).
//
// logits hold `outer` samples of `classes` x `inner` values: class j of position (b, i) is at b * ld + j * inner + i, so
// rows [N, C] are inner = 1 and class maps [B, C, H, W] are inner = H * W.  With x = z / T, m = max x, s = sum exp(x - m):
//   log p_j = x_j - m - log s,   H = -sum p_j log p_j (terms of p = 0 are 0)
//   d/dz_j (gl log p_y + gh H) = (gl ([j = y] - p_j) - gh p_j (log p_j + H)) / T
// Everything between the loads and the stores is fp32.  Exponentials are the bare base-2 instruction, which gives 0 for results below
// 2^-126: probabilities and gradients that fp32 would hold as subnormal numbers are 0.
#pragma once
#include "common.h"

#include <math.h>

namespace classdist {

constexpr int MAX_TOP = 64;  // classes a call ranks or takes: one lane of a wave each
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

typedef _Float16 f16;

// 16 bytes of a row: VEC elements.  Loads and stores take any alignment of the element type.
struct __attribute__((may_alias)) Piece { uint32_t w[4]; };
__device__ __forceinline__ void clear_halves(Piece& q, uint32_t f, uint32_t fill) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t m = ((0u - (f >> (2 * e) & 1u)) & 0xffffu) | ((0u - (f >> (2 * e + 1) & 1u)) & 0xffff0000u);
        q.w[e] = (q.w[e] & ~m) | (fill & m);
    }
}
// KEY_BITS: leading bits of ordered(v) that tell all values of the type apart
struct F32 {
    typedef float E;
    static constexpr int VEC = 4, KEY_BITS = 32;
    static constexpr uint32_t NEG_INF = 0xff800000u;  // as a word of a piece
    static __device__ __forceinline__ float up(float v) { return v; }
    static __device__ __forceinline__ float down(float v) { return v; }
    static __device__ __forceinline__ float get(const Piece& q, int e) { return __uint_as_float(q.w[e]); }
    static __device__ __forceinline__ void put(Piece& q, int e, float v) { q.w[e] = __float_as_uint(v); }
    static __device__ __forceinline__ void clear(Piece& q, uint32_t f) {  // -inf into the elements whose bits are set
#pragma unroll
        for (int e = 0; e < 4; ++e) q.w[e] = f >> e & 1 ? NEG_INF : q.w[e];
    }
    static __device__ __forceinline__ Piece pack(const float (&v)[4]) { return {__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])}; }
};
struct B16 {
    typedef bf16 E;
    static constexpr int VEC = 8, KEY_BITS = 16;
    static constexpr uint32_t NEG_INF = 0xff80ff80u;
    static __device__ __forceinline__ float up(bf16 v) { return (float)v; }
    static __device__ __forceinline__ bf16 down(float v) { return (bf16)v; }
    static __device__ __forceinline__ float get(const Piece& q, int e) { return __uint_as_float(e & 1 ? q.w[e >> 1] & 0xffff0000u : q.w[e >> 1] << 16); }
    static __device__ __forceinline__ void put(Piece& q, int e, float v) {
        const uint32_t b = __builtin_bit_cast(uint16_t, (bf16)v);
        q.w[e >> 1] = e & 1 ? (q.w[e >> 1] & 0xffffu) | b << 16 : (q.w[e >> 1] & 0xffff0000u) | b;
    }
    static __device__ __forceinline__ void clear(Piece& q, uint32_t f) { clear_halves(q, f, NEG_INF); }
    static __device__ __forceinline__ Piece pack(const float (&v)[8]) {
        typedef __attribute__((ext_vector_type(8))) bf16 V;
        V r;
#pragma unroll
        for (int e = 0; e < 8; ++e) r[e] = (bf16)v[e];
        return __builtin_bit_cast(Piece, r);
    }
};
struct H16 {
    typedef f16 E;
    static constexpr int VEC = 8, KEY_BITS = 20;  // sign, 8 exponent bits of fp32, 10 mantissa bits (and one spare)
    static constexpr uint32_t NEG_INF = 0xfc00fc00u;
    static __device__ __forceinline__ float up(f16 v) { return (float)v; }
    static __device__ __forceinline__ f16 down(float v) { return (f16)v; }
    static __device__ __forceinline__ float get(const Piece& q, int e) {
        return (float)__builtin_bit_cast(f16, (uint16_t)(e & 1 ? q.w[e >> 1] >> 16 : q.w[e >> 1]));
    }
    static __device__ __forceinline__ void put(Piece& q, int e, float v) {
        const uint32_t b = __builtin_bit_cast(uint16_t, (f16)v);
        q.w[e >> 1] = e & 1 ? (q.w[e >> 1] & 0xffffu) | b << 16 : (q.w[e >> 1] & 0xffff0000u) | b;
    }
    static __device__ __forceinline__ void clear(Piece& q, uint32_t f) { clear_halves(q, f, NEG_INF); }
    static __device__ __forceinline__ Piece pack(const float (&v)[8]) {
        typedef __attribute__((ext_vector_type(8))) f16 V;
        V r;
#pragma unroll
        for (int e = 0; e < 8; ++e) r[e] = (f16)v[e];
        return __builtin_bit_cast(Piece, r);
    }
};
template <class T> __device__ __forceinline__ Piece load_piece(const typename T::E* p) {
    Piece q;
    __builtin_memcpy(&q, p, 16);
    return q;
}
template <class T> __device__ __forceinline__ void store_piece(typename T::E* p, const Piece& q) { __builtin_memcpy(p, &q, 16); }

__device__ __forceinline__ float exp2_(float v) { return __builtin_amdgcn_exp2f(v); }
__device__ __forceinline__ float log2_(float v) { return __builtin_amdgcn_logf(v); }

// Rank of (value, class) as one integer: larger first, NaN as +inf, -0 = +0, equal values by the lower class.
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    if (v != v) return 0xff800000u;
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ uint64_t rank_key(float v, uint32_t cls) { return (uint64_t)ordered(v) << 32 | (0xffffffffu - cls); }
__device__ __forceinline__ float key_value(uint64_t key) {
    const uint32_t u = (uint32_t)(key >> 32);
    return __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u);
}
__device__ __forceinline__ uint32_t key_class(uint64_t key) { return 0xffffffffu - (uint32_t)key; }

// The largest key of a wave, in every lane: along the rows of 16 lanes and from row to row without the LDS's exchanges.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t max_with(uint64_t v) {  // lanes without a partner keep their own
    const uint32_t lo = (uint32_t)v, hi = (uint32_t)(v >> 32);
    const uint64_t w = (uint64_t)(uint32_t)__builtin_amdgcn_update_dpp((int)hi, (int)hi, CTRL, ROWS, 0xf, false) << 32 |
                       (uint32_t)__builtin_amdgcn_update_dpp((int)lo, (int)lo, CTRL, ROWS, 0xf, false);
    return w > v ? w : v;
}
__device__ __forceinline__ uint64_t wave_max_key(uint64_t v) {
    v = max_with<0x111, 0xf>(v);  // from 1, 2, 4 and 8 lanes below in the row
    v = max_with<0x112, 0xf>(v);
    v = max_with<0x114, 0xf>(v);
    v = max_with<0x118, 0xf>(v);
    v = max_with<0x142, 0xa>(v);  // the last lane of rows 0 and 2 to the rows above them
    v = max_with<0x143, 0xc>(v);  // lane 31 to the upper half
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), 63) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

__device__ __forceinline__ float load_any(const void* p, int dtype, long i) {
    if (dtype == MMAE_DT_F32) return ((const float*)p)[i];
    if (dtype == MMAE_DT_BF16) return (float)((const bf16*)p)[i];
    return (float)((const f16*)p)[i];
}
__device__ __forceinline__ long load_class(const void* p, int bytes, long i) {
    return bytes == 8 ? (long)((const int64_t*)p)[i] : (long)((const int32_t*)p)[i];
}

__device__ __forceinline__ float finite_ref(float m) { return m == -INFINITY ? 0.f : m; }
// Where d stands beside 2^d it is bounded below, as 0 * -inf would be NaN: at -128, since the exponential instruction gives 0 below -126
// (and a bound of -10^4 times a large gradient left fp32).
__device__ __forceinline__ float bounded(float d) { return fmaxf(d, -128.f); }

struct Geometry {
    const void* logits;
    long ld;
    int outer, classes, inner;
    float c, inv_t;  // log2(e) / T, 1 / T
    // log p of logit z, formed in natural units: a finite lowest logit times log2(e) would leave the range of fp32
    __device__ __forceinline__ float log_p(float z, float m, float l2) const { return (z - m) * inv_t - l2 * LN2; }
};

// Sums in the base-2 domain against a reference exponent R: s = sum 2^(z c - R), t = sum (z c - R) 2^(z c - R), m = max z.
// z c - R is one fused multiply-add without intermediate overflow.  R = m c, held to +-FAR, is a rounded number, and the multiply-add
// sees what the rounding lost as a whole: up to FAR = 2^24 that is at most 1/2, a factor between 2^-1/2 and 2^1/2 that s, t and every
// term have in common, and R is the same number wherever it is used, so it cancels.  (At 2^33 it would be up to 2^8: s of 0 or
// infinity.)  Sums of values that all lie below -FAR, classes that are switched off, are 0 beside any other; a row whose maximum lies
// beyond FAR (every class left is one of those) has its sums formed anew from (z - m) c, and so has the mass of the classes that a
// teacher does not keep where their maximum does.
constexpr float FAR = 16777216.f;
struct Sums { float m, R, s, t; };
__device__ __forceinline__ float reference_exponent(float m, float c) { return __builtin_amdgcn_fmed3f(m * c, -FAR, FAR); }
__device__ __forceinline__ Sums join(const Sums& a, const Sums& b) {
    const float R = fmaxf(a.R, b.R), da = a.R - R, db = b.R - R, fa = exp2_(da), fb = exp2_(db);
    return {fmaxf(a.m, b.m), R, a.s * fa + b.s * fb, fa * (a.t + bounded(da) * a.s) + fb * (b.t + bounded(db) * b.s)};
}
__device__ __forceinline__ Sums wave_sums(Sums v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = join(v, {__shfl_xor(v.m, o, 64), __shfl_xor(v.R, o, 64), __shfl_xor(v.s, o, 64), __shfl_xor(v.t, o, 64)});
    return v;
}
__device__ __forceinline__ bool is_far(float m, float c) { return fabsf(m) < INFINITY && fabsf(m * c) > FAR; }

// log p of one logit, in natural units.  l2 = log2 of the sum (+inf: nothing left).
__device__ __forceinline__ float row_log_p(const Geometry& g, float z, float m, float l2) {
    const float d = __builtin_fmaf(z, g.c, -reference_exponent(m, g.c)) - l2;
    // the lowest finite values leave the base-2 range before they leave the natural one
    return is_far(m, g.c) || (d == -INFINITY && z != -INFINITY) ? g.log_p(z, m, l2) : d * LN2;
}

struct LogProbArgs {
    Geometry g;
    const int64_t* target;
    int k;
    float *log_prob, *entropy, *row_max, *row_log_sum, *top_log_prob;
    int64_t* top_class;
};

struct LogProbBwdArgs {
    Geometry g;
    const int64_t* target;
    const float *entropy, *row_max, *row_log_sum, *d_log_prob, *d_entropy;
    void* d_logits;  // contiguous
};

// ---- distillation ----------------------------------------------------------------------------------------------------
// q_i: the teacher's probabilities of the kept classes c_i, from its logits (softmax over the kept ones of value / T) or from
// its log probabilities (exp value; the rest r = 1 - sum q is one more outcome).  Per position
//   l = sum_i q_i (log q_i - log p_{c_i})  [+ r (log r - log P), P = the student's probability of all classes not kept]
//   dl/dx_j = p_j Q - sum_{i: c_i = j} q_i  [- r p_j / P where j is not kept],   Q = sum q [+ r]
// loss = T^2 * sum_p w_p l_p.  Padding (a class outside [0, C)) is left out; a class listed twice counts twice.  Where no
// mass is left outside the kept classes (P = 0) the rest's term is left out; a position whose logits are all -inf has no
// gradient.
struct DistillArgs {
    Geometry g;
    const void *top_class, *top_value;
    int class_bytes, value_dtype, k, log_probs;
    const int64_t* mask;
    int W, patch, tok_w, tokens;  // map geometry of the mask
    float weight;                 // without a mask: T^2 / positions
    float temperature;
    const float *count, *valid;   // with a mask: masked tokens per sample, samples that have any
    const float* upstream;        // gradient arriving at the loss (device scalar) or NULL
    int skip_unit;                // do nothing where it is 1
    float* part;                  // weighted loss per position
    void* d_logits;
};

// What one position's loss counts (T^2 included).
__device__ __forceinline__ float position_weight(const DistillArgs& a, long p) {
    if (!a.mask) return a.weight;
    const int b = (int)(p / a.g.inner), i = (int)(p % a.g.inner);
    const int tok = a.tokens == 1 ? 0 : (i / a.W / a.patch) * a.tok_w + (i % a.W) / a.patch;
    if (a.mask[(long)b * a.tokens + tok] == 0) return 0.f;
    return a.temperature * a.temperature / ((a.tokens == 1 ? 1.f : a.count[b]) * (float)(a.patch * a.patch) * a.valid[0]);
}

// One wave: lane i < k holds kept class i; returns class (-1 for padding), q, log q and the totals over the wave.
struct Kept { int cls; float q, lq; float total, rest; };
__device__ __forceinline__ void read_kept(const DistillArgs& a, long p, int lane, int& cls, float& value) {
    const long at = (p / a.g.inner) * a.k * (long)a.g.inner + p % a.g.inner + (long)lane * a.g.inner;
    cls = -1;
    value = -INFINITY;
    if (lane < a.k) {
        const long c = load_class(a.top_class, a.class_bytes, at);
        const float v = load_any(a.top_value, a.value_dtype, at);
        if (c >= 0 && c < a.g.classes) {
            cls = (int)c;
            value = v;
        }
    }
}
// exp v with the product's rounding put back: relative error of the exponential instruction, not of v.
__device__ __forceinline__ float exp_(float v) {
    const float d = v * LOG2E, lost = __builtin_fmaf(v, LOG2E, -d) + v * 1.9259629e-8f;  // log2(e) - LOG2E
    const float x = exp2_(d);
    return fabsf(d) < 1e4f ? __builtin_fmaf(x, lost * LN2, x) : x;
}
// The lane's share of the teacher's distribution; SUMS: the totals over the wave too (in 64 bits where the rest is what a sum
// near 1 leaves), else those of logits only.
template <bool SUMS = true>
__device__ __forceinline__ Kept kept_share(const DistillArgs& a, int cls, float v) {
    Kept e = {cls, 0.f, 0.f, 0.f, 0.f};
    if (a.log_probs) {
        e.lq = v;
        e.q = cls >= 0 ? exp_(v) : 0.f;
        if (SUMS) {
            double t = cls >= 0 ? exp((double)v) : 0.0;
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) t += __shfl_xor(t, o, 64);
            e.rest = t != t ? (float)t : fmaxf((float)(1.0 - t), 0.f);
            e.total = (float)t;
        }
    } else {
        const float m = finite_ref(wave_max(v)), c = LOG2E * a.g.inv_t;
        const float d = (v - m) * c, x = cls >= 0 ? exp2_(d) : 0.f, s = wave_sum(x);
        e.q = s > 0.f || s != s ? x / s : 0.f;
        e.lq = (v - m) * a.g.inv_t - log2_(s) * LN2;
        e.total = s > 0.f ? 1.f : (s != s ? s : 0.f);
    }
    return e;
}
__device__ __forceinline__ Kept load_kept(const DistillArgs& a, long p, int lane) {
    int cls;
    float v;
    read_kept(a, p, lane, cls, v);
    return kept_share(a, cls, v);
}

// ---- maps: a lane per position ------------------------------------------------------------------------------------------
constexpr int POS = 64;  // positions of a tile: one wave

// Reads a position's kept entries in groups, every load of a group on its way before the first is used: take(i, class or -1, value).
template <class F>
__device__ __forceinline__ void read_entries(const DistillArgs& a, long at, bool live, F take) {
    constexpr int G = 8;
    for (int i0 = 0; i0 < a.k; i0 += G) {
        long cls[G];
        float v[G];
#pragma unroll
        for (int u = 0; u < G; ++u) {
            const long e = at + (long)(i0 + u < a.k ? i0 + u : a.k - 1) * a.g.inner;
            cls[u] = load_class(a.top_class, a.class_bytes, e);
            v[u] = load_any(a.top_value, a.value_dtype, e);
        }
#pragma unroll
        for (int u = 0; u < G; ++u)
            if (i0 + u < a.k) {
                const bool in = live && cls[u] >= 0 && cls[u] < a.g.classes;
                take(i0 + u, in ? (int)cls[u] : -1, in ? v[u] : -INFINITY);
            }
    }
}

// Adds the exponentials of N logits to a lane's running sums.
template <int N, bool ENTROPY>
__device__ __forceinline__ void add_logits(Sums& v, const float (&x)[N], float c) {
    float m = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) m = fmaxf(m, x[i]);
    if (m > v.m) {
        v.m = m;
        const float R = reference_exponent(m, c), d = v.R - R, f = exp2_(d);
        if (ENTROPY) v.t = f * (v.t + bounded(d) * v.s);
        v.s *= f;
        v.R = R;
    }
    float s = 0.f, t = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float d = __builtin_fmaf(x[i], c, -v.R), e = exp2_(d);
        s += e;
        if (ENTROPY) t = __builtin_fmaf(e, bounded(d), t);
    }
    v.s += s;
    if (ENTROPY) v.t += t;
}

// A lane per position, its k kept values at q[i * POS]: their probabilities in place; total: their sum, left: what it leaves of 1,
// loss: sum q log q.
__device__ __forceinline__ void shares_of_log_probs(float* q, int k, float& total, float& left, float& loss) {
    double sum = 0.0;  // 64 bits: the rest is what a sum near 1 leaves
    for (int i = 0; i < k; ++i) {
        const float x = q[i * POS], e = expf(x);
        sum += exp((double)x);
        if (e != 0.f) loss += e * x;
        q[i * POS] = e;
    }
    total = (float)sum;
    left = sum != sum ? total : fmaxf((float)(1.0 - sum), 0.f);
}
__device__ __forceinline__ void shares_of_logits(float* q, int k, float m, float c, float inv_t, float& total, float& loss) {
    m = finite_ref(m);  // (the largest)
    float sum = 0.f;
    for (int i = 0; i < k; ++i) {
        const float d = q[i * POS] - m, e = exp2_(d * c);
        sum += e;
        if (e != 0.f) loss += e * d;
        q[i * POS] = e;
    }
    const float inv = sum != 0.f ? 1.f / sum : 0.f;
    for (int i = 0; i < k; ++i) q[i * POS] *= inv;
    total = sum > 0.f ? 1.f : (sum != sum ? sum : 0.f);
    loss = sum != 0.f ? loss * inv * inv_t - log2_(sum) * LN2 : 0.f;
}

// A launch holds fewer than 2^32 threads.
inline int fits_grid(const char* name, long blocks, int threads) {
    MMAE_REQUIRE(blocks * threads <= 0xffffffffL, MMAE_ESHAPE, "%s: %ld workgroups of %d threads are more than one launch holds", name, blocks, threads);
    return MMAE_OK;
}
#define REQUIRE_GRID(name, blocks, threads)                          \
    do {                                                             \
        const int rc__ = fits_grid(name, (long)(blocks), threads);   \
        if (rc__ != MMAE_OK) return rc__;                            \
    } while (0)

#define BY_DTYPE(dtype, CALL)            \
    do {                                 \
        if ((dtype) == MMAE_DT_F32) { CALL(F32); } \
        else if ((dtype) == MMAE_DT_BF16) { CALL(B16); } \
        else { CALL(H16); }              \
    } while (0)

// classdist_rows.hip: rows, inner = 1
size_t log_probs_rows_workspace(int rows, int classes, int top_k);
int log_probs_rows(int dtype, const LogProbArgs& a, void* workspace, hipStream_t stream);
int log_probs_bwd_rows(int dtype, const LogProbBwdArgs& a, hipStream_t stream);
size_t distill_rows_workspace(int rows, int classes);
int distill_rows(int dtype, const DistillArgs& a, void* workspace, bool again, hipStream_t stream);  // again: the workspace is an earlier call's
// Maps, inner > 1, whose classes are worked on in slices (count 1: all at once).  A slice leaves its sums and its k best keys (0: none)
// of every position, sums[slice][position] and keys[slice][i][position].
struct MapSlices { int count, width; Sums* sums; uint64_t* keys; };
inline int map_tiles(int inner) { return inner / POS + (inner % POS != 0); }
inline long map_blocks(const Geometry& g) { return (long)g.outer * map_tiles(g.inner); }
// classdist_maps.hip
int log_probs_map(int dtype, const LogProbArgs& a, const MapSlices& slices, hipStream_t stream);
int log_probs_bwd_map(int dtype, const LogProbBwdArgs& a, hipStream_t stream);
int distill_map(int dtype, const DistillArgs& a, hipStream_t stream);
// classdist_slices.hip
MapSlices log_probs_map_slices(int dtype, int classes, int top_k);  // (without buffers)
MapSlices distill_map_slices(int dtype, int classes);
size_t log_probs_slices_workspace(const MapSlices& s, int outer, int inner, int top_k);
int log_probs_slices(int dtype, const LogProbArgs& a, MapSlices s, void* workspace, hipStream_t stream);
size_t distill_slices_workspace(const MapSlices& s, int outer, int inner, int k);
int distill_slices(int dtype, const DistillArgs& a, const MapSlices& s, void* workspace, bool again, hipStream_t stream);

}  // namespace classdist
