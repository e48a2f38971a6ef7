// Class distributions: log probabilities of given classes with entropy and top alternatives (forward and backward), and
// distillation from a teacher's top classes (loss and gradient).
//
// logits hold `outer` samples of `classes` x `inner` values: class j of position (b, i) is at b * ld + j * inner + i, so
// rows [N, C] are inner = 1 and class maps [B, C, H, W] are inner = H * W.  With x = z / T, m = max x, s = sum exp(x - m):
//   log p_j = x_j - m - log s,   H = -sum p_j log p_j (terms of p = 0 are 0)
//   d/dz_j (gl log p_y + gh H) = (gl ([j = y] - p_j) - gh p_j (log p_j + H)) / T
// Everything between the loads and the stores is fp32; exponentials are taken of differences (z - m) * log2(e) / T, formed
// before scaling, so that logits of the type's lowest value (a mask) stay finite differences where a whole row has them.
#include "common.h"

#include <math.h>

namespace {

constexpr int MAX_TOP = 64;  // classes a call ranks or takes: one lane of a wave each
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

typedef _Float16 f16;

struct F32 {
    typedef float E;
    static __device__ __forceinline__ float up(float v) { return v; }
    static __device__ __forceinline__ float down(float v) { return v; }
};
struct B16 {
    typedef bf16 E;
    static __device__ __forceinline__ float up(bf16 v) { return (float)v; }
    static __device__ __forceinline__ bf16 down(float v) { return (bf16)v; }
};
struct H16 {
    typedef f16 E;
    static __device__ __forceinline__ float up(f16 v) { return (float)v; }
    static __device__ __forceinline__ f16 down(float v) { return (f16)v; }
};

__device__ __forceinline__ float exp2_(float v) { return __builtin_amdgcn_exp2f(v); }
__device__ __forceinline__ float log2_(float v) { return __builtin_amdgcn_logf(v); }

// Rank of (value, class) as one integer: larger first, NaN above everything, -0 = +0, equal values by the lower class.
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    if (v != v) return 0xffffffffu;
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ uint64_t rank_key(float v, uint32_t cls) { return (uint64_t)ordered(v) << 32 | (0xffffffffu - cls); }

__device__ __forceinline__ float load_any(const void* p, int dtype, long i) {
    if (dtype == MMAE_DT_F32) return ((const float*)p)[i];
    if (dtype == MMAE_DT_BF16) return (float)((const bf16*)p)[i];
    return (float)((const f16*)p)[i];
}
__device__ __forceinline__ long load_class(const void* p, int bytes, long i) {
    return bytes == 8 ? (long)((const int64_t*)p)[i] : (long)((const int32_t*)p)[i];
}

// (m, s, t): maximum, sum of 2^d and sum of d 2^d with d = (z - m) * c.  d is bounded below in t, where 0 * -inf would be NaN.
struct Stats { float m, s, t; };
__device__ __forceinline__ float finite_ref(float m) { return m == -INFINITY ? 0.f : m; }
__device__ __forceinline__ float bounded(float d) { return fmaxf(d, -10000.f); }
__device__ __forceinline__ Stats join(const Stats& a, const Stats& b, float c) {
    const float m = fmaxf(a.m, b.m), r = finite_ref(m);
    const float da = (a.m - r) * c, db = (b.m - r) * c;
    const float fa = exp2_(da), fb = exp2_(db);
    return {m, a.s * fa + b.s * fb, fa * (a.t + bounded(da) * a.s) + fb * (b.t + bounded(db) * b.s)};
}

struct Geometry {
    const void* logits;
    long ld;
    int outer, classes, inner;
    float c, inv_t;  // log2(e) / T, 1 / T
    // log p of logit z, formed in natural units: a finite lowest logit times log2(e) would leave the range of fp32
    __device__ __forceinline__ float log_p(float z, float m, float l2) const { return (z - m) * inv_t - l2 * LN2; }
    __device__ __forceinline__ long base(long p) const { return inner == 1 ? p * ld : (p / inner) * ld + p % inner; }
};

__device__ Stats block_stats(Stats v, float c, Stats* red) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const Stats w = {__shfl_xor(v.m, o, 64), __shfl_xor(v.s, o, 64), __shfl_xor(v.t, o, 64)};
        v = join(v, w, c);
    }
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, nw = (blockDim.x + 63) >> 6;
    __syncthreads();
    if (lane == 0) red[w] = v;
    __syncthreads();
    Stats r = red[0];
    for (int i = 1; i < nw; ++i) r = join(r, red[i], c);
    return r;
}

// ---- log probabilities, one workgroup per position -------------------------------------------------------------------
struct LogProbArgs {
    Geometry g;
    const int64_t* target;
    int k;
    float *log_prob, *entropy, *row_max, *row_log_sum, *top_log_prob;
    int64_t* top_class;
};

template <class T>
__global__ __launch_bounds__(256) void log_probs_kernel(LogProbArgs a) {
    __shared__ Stats red[4];
    __shared__ uint64_t best[4];
    const typename T::E* z = (const typename T::E*)a.g.logits;
    const long p = blockIdx.x, base = a.g.base(p), cs = a.g.inner;
    const int C = a.g.classes;
    const float c = a.g.c;
    Stats v = {-INFINITY, 0.f, 0.f};
    for (int j = threadIdx.x; j < C; j += 256) v.m = fmaxf(v.m, T::up(z[base + j * cs]));
    const float r = finite_ref(v.m);
    for (int j = threadIdx.x; j < C; j += 256) {
        const float d = (T::up(z[base + j * cs]) - r) * c, e = exp2_(d);
        v.s += e;
        v.t += e * bounded(d);
    }
    v = block_stats(v, c, red);
    const bool empty = v.m == -INFINITY && v.s == 0.f;
    const float l2 = empty ? INFINITY : log2_(v.s), m = finite_ref(v.m);  // +inf: every log probability is -inf
    if (threadIdx.x == 0) {
        const long y = a.target[p];
        a.log_prob[p] = y >= 0 && y < C ? a.g.log_p(T::up(z[base + y * cs]), m, l2) : 0.f;
        a.entropy[p] = empty ? 0.f : (l2 - v.t / v.s) * LN2;
        a.row_max[p] = m;
        a.row_log_sum[p] = l2;
    }
    const long at = (p / a.g.inner) * a.k * cs + p % a.g.inner;
    uint64_t last = ~0ull;
    for (int i = 0; i < a.k; ++i) {  // the largest key below the last one found
        uint64_t top = 0;
        for (int j = threadIdx.x; j < C; j += 256) {
            const uint64_t key = rank_key(T::up(z[base + j * cs]), j);
            if (key < last && key > top) top = key;
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            const uint64_t w = __shfl_xor((unsigned long long)top, o, 64);
            top = w > top ? w : top;
        }
        __syncthreads();
        if ((threadIdx.x & 63) == 0) best[threadIdx.x >> 6] = top;
        __syncthreads();
        for (int w = 0; w < 4; ++w) top = best[w] > top ? best[w] : top;
        last = top;
        if (threadIdx.x == 0) {
            const uint32_t j = 0xffffffffu - (uint32_t)top;
            a.top_class[at + i * cs] = j;
            a.top_log_prob[at + i * cs] = a.g.log_p(T::up(z[base + j * cs]), m, l2);
        }
    }
}

struct LogProbBwdArgs {
    Geometry g;
    const int64_t* target;
    const float *entropy, *row_max, *row_log_sum, *d_log_prob, *d_entropy;
    void* d_logits;  // contiguous
};

template <class T>
__global__ __launch_bounds__(256) void log_probs_bwd_kernel(LogProbBwdArgs a) {
    const typename T::E* z = (const typename T::E*)a.g.logits;
    typename T::E* dz = (typename T::E*)a.d_logits;
    const long p = blockIdx.x, base = a.g.base(p), cs = a.g.inner;
    const int C = a.g.classes;
    const long out = a.g.inner == 1 ? p * C : (p / a.g.inner) * C * cs + p % a.g.inner;
    const float m = a.row_max[p], l2 = a.row_log_sum[p], c = a.g.c;
    const long y = a.target[p];
    const float gl = a.d_log_prob && y >= 0 && y < C && l2 != INFINITY ? a.d_log_prob[p] * a.g.inv_t : 0.f;
    const float gh = a.d_entropy ? a.d_entropy[p] * a.g.inv_t : 0.f, h = a.entropy[p];
    for (int j = threadIdx.x; j < C; j += 256) {
        const float lp2 = (T::up(z[base + j * cs]) - m) * c - l2;
        const float q = exp2_(lp2);
        dz[out + j * cs] = T::down((j == y ? gl : 0.f) - q * (gl + gh * (bounded(lp2) * LN2 + h)));
    }
}

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
    return a.temperature * a.temperature / (a.count[b] * (float)(a.patch * a.patch) * a.valid[0]);
}

// One wave: lane i < k holds kept class i; returns class (-1 for padding), q, log q and the totals over the wave.
struct Kept { int cls; float q, lq; float total, rest; };
__device__ __forceinline__ Kept load_kept(const DistillArgs& a, long p, int lane) {
    const long at = (p / a.g.inner) * a.k * (long)a.g.inner + p % a.g.inner + (long)lane * a.g.inner;
    Kept e = {-1, 0.f, 0.f, 0.f, 0.f};
    float v = -INFINITY;
    if (lane < a.k) {
        const long cls = load_class(a.top_class, a.class_bytes, at);
        if (cls >= 0 && cls < a.g.classes) {
            e.cls = (int)cls;
            v = load_any(a.top_value, a.value_dtype, at);
        }
    }
    if (a.log_probs) {
        e.lq = v;
        e.q = e.cls >= 0 ? expf(v) : 0.f;
        double t = e.cls >= 0 ? exp((double)v) : 0.0;  // 64 bits: the rest is what a sum near 1 leaves
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) t += __shfl_xor(t, o, 64);
        e.rest = t != t ? (float)t : fmaxf((float)(1.0 - t), 0.f);
        e.total = (float)t;
    } else {
        const float m = finite_ref(wave_max(v)), c = LOG2E * a.g.inv_t;
        const float d = (v - m) * c, x = e.cls >= 0 ? exp2_(d) : 0.f, s = wave_sum(x);
        e.q = s > 0.f || s != s ? x / s : 0.f;
        e.lq = (v - m) * a.g.inv_t - log2_(s) * LN2;
        e.total = s > 0.f ? 1.f : (s != s ? s : 0.f);
    }
    return e;
}

template <class T>
__global__ __launch_bounds__(256) void distill_kernel(DistillArgs a) {
    __shared__ Stats red[4];
    __shared__ int s_cls[MAX_TOP];
    __shared__ float s_q[MAX_TOP], s_l[1], s_tot[2];
    if (a.upstream && a.skip_unit && a.upstream[0] == 1.f) return;
    const typename T::E* z = (const typename T::E*)a.g.logits;
    const long p = blockIdx.x, base = a.g.base(p), cs = a.g.inner;
    const int C = a.g.classes, lane = threadIdx.x & 63;
    const float c = a.g.c, w = position_weight(a, p);
    typename T::E* dz = (typename T::E*)a.d_logits;
    const long out = a.g.inner == 1 ? p * C : (p / a.g.inner) * C * cs + p % a.g.inner;
    if (w == 0.f) {
        if (dz) for (int j = threadIdx.x; j < C; j += 256) dz[out + j * cs] = T::down(0.f);
        if (threadIdx.x == 0 && a.part) a.part[p] = 0.f;
        return;
    }
    Kept e = {};
    if (threadIdx.x < 64) {
        e = load_kept(a, p, lane);
        s_cls[lane] = e.cls;
        s_q[lane] = e.q;
        if (lane == 0) { s_tot[0] = e.total; s_tot[1] = e.rest; }
    }
    __syncthreads();
    Stats v = {-INFINITY, 0.f, 0.f}, u = {-INFINITY, 0.f, 0.f};  // all classes; the ones not kept
    for (int j = threadIdx.x; j < C; j += 256) {
        const float x = T::up(z[base + j * cs]);
        bool kept = !a.log_probs;
        for (int i = 0; i < a.k && !kept; ++i) kept = s_cls[i] == j;
        v = join(v, Stats{x, x == -INFINITY ? 0.f : 1.f, 0.f}, c);
        if (!kept) u = join(u, Stats{x, x == -INFINITY ? 0.f : 1.f, 0.f}, c);
    }
    v = block_stats(v, c, red);
    u = block_stats(u, c, red);
    const bool empty = v.m == -INFINITY && v.s == 0.f;
    const float m = finite_ref(v.m), l2 = empty ? 0.f : log2_(v.s);
    const float um = finite_ref(u.m), ul2 = log2_(u.s);
    const float rest = u.s != 0.f ? s_tot[1] : 0.f, Q = s_tot[0] + rest;
    if (threadIdx.x < 64 && a.part) {
        float l = 0.f;
        if (e.q != 0.f) l = e.q * (e.lq - a.g.log_p(T::up(z[base + e.cls * cs]), m, l2));
        l = wave_sum(l);
        if (rest != 0.f) l += rest * ((log2_(rest) - (ul2 - l2)) * LN2 - (um - m) * a.g.inv_t);
        if (lane == 0) a.part[p] = w * l;
    }
    if (!dz) return;
    const float gs = empty ? 0.f : w * a.g.inv_t * (a.upstream ? a.upstream[0] : 1.f);
    for (int j = threadIdx.x; j < C; j += 256) {
        const float x = T::up(z[base + j * cs]);
        float q = 0.f;
        bool kept = false;
        for (int i = 0; i < a.k; ++i)
            if (s_cls[i] == j) { q += s_q[i]; kept = true; }
        float d = exp2_((x - m) * c - l2) * Q - q;
        if (!kept && rest != 0.f) d -= rest * exp2_((x - um) * c - ul2);
        dz[out + j * cs] = T::down(gs * d);
    }
}

// Masked tokens per sample; then the number of samples that have any.
__global__ __launch_bounds__(64) void distill_count_kernel(const int64_t* mask, int outer, int tokens, float* count) {
    const int b = blockIdx.x;
    int n = 0;
    for (int i = threadIdx.x; i < tokens; i += 64) n += mask[(long)b * tokens + i] != 0;
    const float s = wave_sum((float)n);
    if (threadIdx.x == 0) count[b] = s;
}
__global__ __launch_bounds__(1024) void distill_valid_kernel(const float* count, int outer, float* valid) {
    __shared__ float red[16];
    float n = 0.f;
    for (int b = threadIdx.x; b < outer; b += 1024) n += count[b] > 0.f ? 1.f : 0.f;
    n = block_sum(n, red);
    if (threadIdx.x == 0) valid[0] = n;
}
// The parts added in a fixed order, in 64 bits.
__global__ __launch_bounds__(1024) void distill_sum_kernel(const float* part, long n, float* loss) {
    __shared__ double red[16];
    double s = 0.0;
    for (long i = threadIdx.x; i < n; i += 1024) s += (double)part[i];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 16; ++w) s += red[w];
        loss[0] = (float)s;
    }
}

int check_logits(const char* name, const void* logits, int dtype, int outer, int classes, int inner, long ld, float temperature) {
    MMAE_REQUIRE(logits, MMAE_EINVAL, "%s: null pointer", name);
    MMAE_REQUIRE(dtype >= MMAE_DT_F32 && dtype <= MMAE_DT_F16, MMAE_EINVAL, "%s: dtype code %d", name, dtype);
    MMAE_REQUIRE(outer > 0 && classes > 0 && inner > 0, MMAE_ESHAPE, "%s: empty input (%d x %d x %d)", name, outer, classes, inner);
    MMAE_REQUIRE((long)outer * inner <= 0x7fffffffL, MMAE_ESHAPE, "%s: %d x %d positions are more than 2^31 - 1", name, outer, inner);
    MMAE_REQUIRE(ld >= (long)classes * inner, MMAE_ESHAPE, "%s: samples %ld elements apart hold %d x %d values", name, ld, classes, inner);
    MMAE_REQUIRE(temperature > 0.f && temperature < INFINITY, MMAE_EINVAL, "%s: temperature %g is not positive and finite", name, temperature);
    return MMAE_OK;
}

#define BY_DTYPE(dtype, CALL)            \
    do {                                 \
        if ((dtype) == MMAE_DT_F32) { CALL(F32); } \
        else if ((dtype) == MMAE_DT_BF16) { CALL(B16); } \
        else { CALL(H16); }              \
    } while (0)

}  // namespace

extern "C" size_t mmae_class_log_probs_workspace_bytes(int outer, int classes, int inner, int top_k) { return 0; }

extern "C" int mmae_class_log_probs(const void* logits, int dtype, int outer, int classes, int inner, long ld, const int64_t* target,
                                    int top_k, float temperature, float* log_prob, float* entropy, float* row_max,
                                    float* row_log_sum, float* top_log_prob, int64_t* top_class, void* workspace,
                                    size_t workspace_bytes, hipStream_t stream) {
    const int rc = check_logits("class_log_probs", logits, dtype, outer, classes, inner, ld, temperature);
    if (rc != MMAE_OK) return rc;
    MMAE_REQUIRE(target && log_prob && entropy && row_max && row_log_sum && (!top_k || (top_log_prob && top_class)), MMAE_EINVAL,
                 "class_log_probs: null pointer");
    MMAE_REQUIRE(top_k >= 0 && top_k <= MAX_TOP && top_k <= classes, MMAE_ESHAPE,
                 "class_log_probs: %d top classes of %d (at most %d)", top_k, classes, MAX_TOP);
    LogProbArgs a = {{logits, ld, outer, classes, inner, LOG2E / temperature, 1.f / temperature}, target, top_k, log_prob, entropy, row_max,
                     row_log_sum, top_log_prob, top_class};
#define CALL(T) hipLaunchKernelGGL(log_probs_kernel<T>, dim3(outer * inner), dim3(256), 0, stream, a)
    BY_DTYPE(dtype, CALL);
#undef CALL
    MMAE_CHECK_LAUNCH("class_log_probs");
    return MMAE_OK;
}

extern "C" int mmae_class_log_probs_bwd(const void* logits, int dtype, int outer, int classes, int inner, long ld,
                                        const int64_t* target, float temperature, const float* entropy, const float* row_max,
                                        const float* row_log_sum, const float* d_log_prob, const float* d_entropy, void* d_logits,
                                        hipStream_t stream) {
    const int rc = check_logits("class_log_probs_bwd", logits, dtype, outer, classes, inner, ld, temperature);
    if (rc != MMAE_OK) return rc;
    MMAE_REQUIRE(target && entropy && row_max && row_log_sum && d_logits, MMAE_EINVAL, "class_log_probs_bwd: null pointer");
    LogProbBwdArgs a = {{logits, ld, outer, classes, inner, LOG2E / temperature, 1.f / temperature}, target, entropy, row_max, row_log_sum,
                        d_log_prob, d_entropy, d_logits};
#define CALL(T) hipLaunchKernelGGL(log_probs_bwd_kernel<T>, dim3(outer * inner), dim3(256), 0, stream, a)
    BY_DTYPE(dtype, CALL);
#undef CALL
    MMAE_CHECK_LAUNCH("class_log_probs_bwd");
    return MMAE_OK;
}

extern "C" size_t mmae_distill_workspace_bytes(int outer, int classes, int inner, int k) {
    return sizeof(float) * (4 + (size_t)outer + (size_t)outer * inner);
}

extern "C" int mmae_distill(const void* logits, int dtype, int outer, int classes, int inner, long ld, const void* top_class,
                            int class_bytes, const void* top_value, int value_dtype, int k, int kind, float temperature,
                            const int64_t* mask, int width, int patch, const float* upstream, int skip_unit, float* loss,
                            void* d_logits, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    const int rc = check_logits("distill", logits, dtype, outer, classes, inner, ld, temperature);
    if (rc != MMAE_OK) return rc;
    MMAE_REQUIRE(top_class && top_value && workspace && (loss || d_logits), MMAE_EINVAL, "distill: null pointer");
    MMAE_REQUIRE(class_bytes == 4 || class_bytes == 8, MMAE_EINVAL, "distill: classes of %d bytes", class_bytes);
    MMAE_REQUIRE(value_dtype >= MMAE_DT_F32 && value_dtype <= MMAE_DT_F16, MMAE_EINVAL, "distill: value dtype code %d", value_dtype);
    MMAE_REQUIRE(k >= 1 && k <= MAX_TOP, MMAE_ESHAPE, "distill: %d kept classes, between 1 and %d are taken", k, MAX_TOP);
    MMAE_REQUIRE(kind == 0 || kind == 1, MMAE_EINVAL, "distill: kind %d not in {0 (logits), 1 (log probabilities)}", kind);
    MMAE_REQUIRE(!mask || (width >= 1 && patch >= 1 && inner % width == 0 && width % patch == 0 && inner / width % patch == 0), MMAE_ESHAPE,
                 "distill: %d positions in rows of %d are not whole patches of %d", inner, width, patch);
    MMAE_REQUIRE(workspace_bytes >= mmae_distill_workspace_bytes(outer, classes, inner, k), MMAE_EWORKSPACE, "distill: workspace too small");
    float* ws = (float*)workspace;
    DistillArgs a = {{logits, ld, outer, classes, inner, LOG2E / temperature, 1.f / temperature}, top_class, top_value, class_bytes, value_dtype, k, kind, mask};
    a.W = width; a.patch = mask ? patch : 1;
    a.tok_w = mask ? width / patch : 1;
    a.tokens = mask ? a.tok_w * (inner / width / patch) : 1;
    a.temperature = temperature;
    a.weight = (float)((double)temperature * temperature / ((double)outer * inner));
    a.valid = ws; a.count = ws + 4; a.part = loss ? ws + 4 + outer : nullptr;
    a.upstream = upstream; a.skip_unit = skip_unit; a.d_logits = d_logits;
    if (mask) {
        hipLaunchKernelGGL(distill_count_kernel, dim3(outer), dim3(64), 0, stream, mask, outer, a.tokens, ws + 4);
        MMAE_CHECK_LAUNCH("distill_count");
        hipLaunchKernelGGL(distill_valid_kernel, dim3(1), dim3(1024), 0, stream, ws + 4, outer, ws);
        MMAE_CHECK_LAUNCH("distill_valid");
    }
#define CALL(T) hipLaunchKernelGGL(distill_kernel<T>, dim3(outer * inner), dim3(256), 0, stream, a)
    BY_DTYPE(dtype, CALL);
#undef CALL
    MMAE_CHECK_LAUNCH("distill");
    if (loss) {
        hipLaunchKernelGGL(distill_sum_kernel, dim3(1), dim3(1024), 0, stream, a.part, (long)outer * inner, loss);
        MMAE_CHECK_LAUNCH("distill_sum");
    }
    return MMAE_OK;
}
