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

// 16 bytes of a row: VEC elements.  Loads and stores take any alignment of the element type.
struct Piece { uint32_t w[4]; };
// KEY_BITS: leading bits of ordered(v) that tell all values of the type apart
struct F32 {
    typedef float E;
    static constexpr int VEC = 4, KEY_BITS = 32;
    static constexpr uint32_t NEG_INF = 0xff800000u;  // as a word of a piece
    static __device__ __forceinline__ float up(float v) { return v; }
    static __device__ __forceinline__ float down(float v) { return v; }
    static __device__ __forceinline__ float get(const Piece& q, int e) { return __uint_as_float(q.w[e]); }
    static __device__ __forceinline__ void put(Piece& q, int e, float v) { q.w[e] = __float_as_uint(v); }
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

// Rank of (value, class) as one integer: larger first, NaN above everything, -0 = +0, equal values by the lower class.
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    if (v != v) return 0xffffffffu;
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ uint64_t rank_key(float v, uint32_t cls) { return (uint64_t)ordered(v) << 32 | (0xffffffffu - cls); }
__device__ __forceinline__ float key_value(uint64_t key) {  // (NaN stays NaN)
    const uint32_t u = (uint32_t)(key >> 32);
    return __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u);
}
__device__ __forceinline__ uint32_t key_class(uint64_t key) { return 0xffffffffu - (uint32_t)key; }

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

// ---- rows: one pass over a row, or a slice of it --------------------------------------------------------------------
// Sums in the base-2 domain against a reference exponent R: s = sum 2^(z c - R), t = sum (z c - R) 2^(z c - R), m = max z.
// z c - R is one fused multiply-add without intermediate overflow; R = m c, held to +-FAR, is the same rounded number wherever
// it is used, so its rounding cancels.  Beyond FAR (every class left at the type's lowest value, say) the row's sums are
// formed anew from (z - m) c.
constexpr float FAR = 1e38f;
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
template <int NT>
__device__ Sums block_sums(Sums v, Sums* red) {
    v = wave_sums(v);
    if (NT == 64) return v;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    Sums r = red[0];
    for (int i = 1; i < NT / 64; ++i) r = join(r, red[i]);
    return r;
}
__device__ __forceinline__ bool is_far(float m, float c) { return fabsf(m) < INFINITY && fabsf(m * c) > FAR; }

// The sums of a whole row by (z - m) c, for the rows beyond FAR.
template <class T, int NT>
__device__ __noinline__ Sums far_sums(const typename T::E* z, int C, float m, float c, Sums* red) {
    Sums v = {m, 0.f, 0.f, 0.f};
    for (int j = threadIdx.x; j < C; j += NT) {
        const float d = (T::up(z[j]) - m) * c, e = exp2_(d);
        v.s += e;
        v.t += e * bounded(d);
    }
    return block_sums<NT>(v, red);
}

// log p of one logit, in natural units.  l2 = log2 of the sum (+inf: nothing left).
__device__ __forceinline__ float row_log_p(const Geometry& g, float z, float m, float l2) {
    const float d = __builtin_fmaf(z, g.c, -reference_exponent(m, g.c)) - l2;
    // the lowest finite values leave the base-2 range before they leave the natural one
    return is_far(m, g.c) || (d == -INFINITY && z != -INFINITY) ? g.log_p(z, m, l2) : d * LN2;
}

template <class T, int NT, int NV>
__device__ __forceinline__ void load_tile(Piece (&q)[NV], const typename T::E* z, int base, int end) {
    constexpr int VEC = T::VEC;
    if (base + NT * NV * VEC <= end) {
#pragma unroll
        for (int i = 0; i < NV; ++i) q[i] = load_piece<T>(z + base + (i * NT + threadIdx.x) * VEC);
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int j = base + (i * NT + threadIdx.x) * VEC;
            if (j + VEC <= end) {
                q[i] = load_piece<T>(z + j);
            } else {
                q[i] = {T::NEG_INF, T::NEG_INF, T::NEG_INF, T::NEG_INF};
#pragma unroll
                for (int e = 0; e < VEC; ++e)
                    if (j + e < end) T::put(q[i], e, T::up(z[j + e]));
            }
        }
    }
}

// Most keys a tile can append: the list's own, and those above the k-th largest of the threads' maxima, which belong to
// fewer than k threads.
template <int EPT> constexpr int list_room() { return MAX_TOP + (MAX_TOP - 1) * EPT; }

template <int ROOM, int NT>
struct TopList {
    uint64_t keys[ROOM];    // sorted up to `have` between tiles, appended behind it
    uint64_t sorted[MAX_TOP];
    float maxima[NT];
    int count, wave_count[NT / 64];
};

// ordered() of the k-th largest of the NT maxima, searched bit by bit: each wave looks at all maxima and counts by ballots, so
// no wave waits for another.
template <class T, int NT>
__device__ __forceinline__ uint32_t kth_maximum(const float* maxima, int k) {
    const int lane = threadIdx.x & 63;
    uint32_t key[NT / 64];
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) key[i] = ordered(maxima[i * 64 + lane]);
    uint32_t at = 0;
    for (int b = 31; b >= 32 - T::KEY_BITS; --b) {
        const uint32_t next = at | 1u << b;
        int n = 0;
#pragma unroll
        for (int i = 0; i < NT / 64; ++i) n += __popcll(__ballot(key[i] >= next));
        if (n >= k) at = next;
    }
    return at & 0x80000000u ? at : at | ((1ull << (32 - T::KEY_BITS)) - 1);  // (negative values are inverted, their later bits are set)
}

// Ranks the `n` keys of the list and keeps the first k, sorted.  Returns the value a further key has to exceed.
template <int NT, class L>
__device__ float keep_best(L& list, int n, int k) {
    for (int i = threadIdx.x; i < n; i += NT) {
        const uint64_t key = list.keys[i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += list.keys[j] > key;
        if (rank < k) list.sorted[rank] = key;
    }
    __syncthreads();
    const int have = n < k ? n : k;
    for (int i = threadIdx.x; i < have; i += NT) list.keys[i] = list.sorted[i];
    if (threadIdx.x == 0) list.count = have;
    __syncthreads();
    return have < k ? -INFINITY : key_value(list.keys[k - 1]);
}

// Takes a tile's elements into the list.  floor: the value a key has to exceed (the k-th best so far: an equal one has a
// higher class), -inf with `open` while the list holds fewer than k.
template <class T, int NT, int NV, class L>
__device__ __forceinline__ void take_tile(L& list, const Piece (&q)[NV], float tile_max, int base, int end, int k, float& floor, bool& open) {
    constexpr int VEC = T::VEC, ROOM = sizeof(list.keys) / 8;
    const int above = NT == 64 ? __popcll(__ballot(open || tile_max > floor)) : __syncthreads_count(open || tile_max > floor);
    if (above == 0) return;
    const int have = list.count;
    float least = floor;     // take values above this one ...
    bool equals = open;      // ... and equal to it
    if (above >= k) {        // else fewer than k threads hold values above the floor: they all fit
        list.maxima[threadIdx.x] = tile_max;
        __syncthreads();
        const uint32_t kth = kth_maximum<T, NT>(list.maxima, k);
        const float v = key_value((uint64_t)kth << 32);
        if (open || v > floor) { least = v; equals = true; }
    }
    if (NT != 64) __syncthreads();  // (list.count is read)
    if (tile_max > least || (equals && tile_max == least)) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float v = T::get(q[i], e);
                const int j = base + (i * NT + threadIdx.x) * VEC + e;
                if ((v > least || (equals && v == least)) && j < end) {
                    const int n = atomicAdd(&list.count, 1);
                    if (n < ROOM) list.keys[n] = rank_key(v, j);
                }
            }
    }
    __syncthreads();
    int n = list.count;
    if (n > ROOM) {
        // More equal values than the list holds: the greater ones (fewer than k threads have any), then the equal ones of
        // the lowest classes, piece by piece in the order of classes.
        __syncthreads();
        if (threadIdx.x == 0) list.count = have;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float v = T::get(q[i], e);
                if (v > least) {
                    const int n = atomicAdd(&list.count, 1);
                    if (n < ROOM) list.keys[n] = rank_key(v, base + (i * NT + threadIdx.x) * VEC + e);
                }
            }
        __syncthreads();
        n = list.count < ROOM ? list.count : ROOM;
        int left = k < ROOM - n ? k : ROOM - n;  // equal values taken: k cover every need, keep_best cuts
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int j = base + (i * NT + threadIdx.x) * VEC;
            int mine = 0;
#pragma unroll
            for (int e = 0; e < VEC; ++e) mine += T::get(q[i], e) == least && j + e < end;
            int before = mine;  // inclusive prefix over the wave, then over the waves
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int w = __shfl_up(before, o, 64);
                if ((int)(threadIdx.x & 63) >= o) before += w;
            }
            __syncthreads();
            if ((threadIdx.x & 63) == 63) list.wave_count[threadIdx.x >> 6] = before;
            __syncthreads();
            int all = 0;
            before -= mine;
            for (int w = 0; w < NT / 64; ++w) {
                if (w < (int)(threadIdx.x >> 6)) before += list.wave_count[w];
                all += list.wave_count[w];
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                if (T::get(q[i], e) == least && j + e < end) {
                    if (before < left) list.keys[n + before] = rank_key(least, j + e);
                    ++before;
                }
            n += all < left ? all : left;
            left -= all < left ? all : left;
        }
        __syncthreads();
    }
    floor = keep_best<NT>(list, n, k);
    open = list.count < k;
}

// The k best of z[first, end) by k scans, for slices that hold NaN (which compare with nothing).
template <class T, int NT, class L>
__device__ __noinline__ void scan_top(L& list, const typename T::E* z, int first, int end, int k) {
    uint64_t last = ~0ull;
    const int n = end - first < k ? end - first : k;
    for (int i = 0; i < n; ++i) {
        uint64_t top = 0;
        for (int j = first + threadIdx.x; j < end; j += NT) {
            const uint64_t key = rank_key(T::up(z[j]), j);
            if (key < last && key > top) top = key;
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            const uint64_t w = __shfl_xor((unsigned long long)top, o, 64);
            top = w > top ? w : top;
        }
        __syncthreads();
        if ((threadIdx.x & 63) == 0) list.sorted[threadIdx.x >> 6] = top;
        __syncthreads();
        for (int w = 0; w < NT / 64; ++w) top = list.sorted[w] > top ? list.sorted[w] : top;
        last = top;
        if (threadIdx.x == 0) list.keys[i] = top;
    }
    __syncthreads();
    if (threadIdx.x == 0) list.count = n;
    __syncthreads();
}

// A row's results from its sums and its sorted best keys (keys[i], i < k); the threads of one wave.
template <class T, int NT>
__device__ __forceinline__ void finish_row(const LogProbArgs& a, long p, const typename T::E* z, Sums v, const uint64_t* keys, Sums* red) {
    const float c = a.g.c;
    if (is_far(v.m, c)) v = far_sums<T, NT>(z, a.g.classes, v.m, c, red);
    if (v.m == INFINITY) v.s = __builtin_nanf("");
    const bool empty = v.m == -INFINITY && v.s == 0.f;
    const float l2 = empty ? INFINITY : log2_(v.s);
    if (threadIdx.x == 0) {
        const long y = a.target[p];
        a.log_prob[p] = y >= 0 && y < a.g.classes ? row_log_p(a.g, T::up(z[y]), v.m, l2) : 0.f;
        a.entropy[p] = empty ? 0.f : (l2 - v.t / v.s) * LN2;
        a.row_max[p] = v.m;
        a.row_log_sum[p] = l2;
    }
    if ((int)threadIdx.x < a.k) {
        const uint64_t key = keys[threadIdx.x];
        a.top_class[p * a.k + threadIdx.x] = key_class(key);
        a.top_log_prob[p * a.k + threadIdx.x] = row_log_p(a.g, key_value(key), v.m, l2);
    }
}

// What a slice leaves for the join: its sums, then its k keys (0 where it holds fewer classes).
__host__ __device__ inline size_t slice_bytes(int k) { return sizeof(Sums) + sizeof(uint64_t) * (size_t)k; }

template <class T, int NT, int NV, bool TOP>
__global__ __launch_bounds__(NT) void log_probs_rows_kernel(LogProbArgs a, int slices, int slice_tiles, char* parts) {
    constexpr int VEC = T::VEC, TILE = NT * NV * VEC, ROOM = TOP ? list_room<NV * VEC>() : 1;
    __shared__ Sums red[NT / 64];
    __shared__ TopList<ROOM, NT> list;
    const long p = blockIdx.x / slices;
    const int slice = blockIdx.x % slices;
    const typename T::E* z = (const typename T::E*)a.g.logits + p * a.g.ld;
    const int C = a.g.classes, first = slice * slice_tiles * TILE;
    const int end = first + slice_tiles * TILE < C ? first + slice_tiles * TILE : C;
    const float c = a.g.c;
    Sums v = {-INFINITY, -FAR, 0.f, 0.f};
    float floor = -INFINITY;
    bool open = true;
    if (TOP) {
        if (threadIdx.x == 0) list.count = 0;
        __syncthreads();
    }
    Piece q[NV], next[NV];
    load_tile<T, NT, NV>(q, z, first, end);
    for (int base = first;;) {
        const bool more = base + TILE < end;
        if (more) load_tile<T, NT, NV>(next, z, base + TILE, end);
        float m = T::get(q[0], 0);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < VEC; ++e) m = fmaxf(m, T::get(q[i], e));
        if (m > v.m) {
            v.m = m;
            const float R = reference_exponent(m, c), d = v.R - R, f = exp2_(d);
            v.t = f * (v.t + bounded(d) * v.s);
            v.s *= f;
            v.R = R;
        }
        float s = 0.f, t = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float d = __builtin_fmaf(T::get(q[i], e), c, -v.R), x = exp2_(d);
                s += x;
                t = __builtin_fmaf(x, bounded(d), t);
            }
        v.s += s;
        v.t += t;
        if (TOP) take_tile<T, NT, NV>(list, q, m, base, end, a.k, floor, open);
        if (!more) break;
        base += TILE;
#pragma unroll
        for (int i = 0; i < NV; ++i) q[i] = next[i];
    }
    v = block_sums<NT>(v, red);
    if (TOP && v.s != v.s) scan_top<T, NT>(list, z, first, end, a.k);
    if (slices == 1) {
        finish_row<T, NT>(a, p, z, v, list.keys, red);
        return;
    }
    char* out = parts + (size_t)blockIdx.x * slice_bytes(a.k);
    if (threadIdx.x == 0) *(Sums*)out = v;
    if (TOP && (int)threadIdx.x < a.k) ((uint64_t*)(out + sizeof(Sums)))[threadIdx.x] = (int)threadIdx.x < list.count ? list.keys[threadIdx.x] : 0;
}

// Joins the slices of a row: one wave per row, lane i walks slice i's sorted keys.
constexpr int MAX_SLICES = 64;
template <class T>
__global__ __launch_bounds__(64) void log_probs_join_kernel(LogProbArgs a, int slices, const char* parts) {
    extern __shared__ uint64_t s_keys[];  // [slices][k], then the k best
    __shared__ Sums red[1];
    const long p = blockIdx.x;
    const int lane = threadIdx.x, k = a.k;
    const char* part = parts + (size_t)p * slices * slice_bytes(k);
    Sums v = {-INFINITY, -FAR, 0.f, 0.f};
    if (lane < slices) v = *(const Sums*)(part + lane * slice_bytes(k));
    for (int i = lane; i < slices * k; i += 64) s_keys[i] = ((const uint64_t*)(part + (i / k) * slice_bytes(k) + sizeof(Sums)))[i % k];
    v = wave_sums(v);
    __syncthreads();
    int at = 0;
    uint64_t head = lane < slices && k ? s_keys[lane * k] : 0;
    for (int i = 0; i < k; ++i) {
        uint64_t top = head;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            const uint64_t w = __shfl_xor((unsigned long long)top, o, 64);
            top = w > top ? w : top;
        }
        if (head == top && top) {  // keys are unique: one lane
            ++at;
            head = at < k ? s_keys[lane * k + at] : 0;
        }
        if (lane == 0) s_keys[slices * k + i] = top;
    }
    __syncthreads();
    finish_row<T, 64>(a, p, (const typename T::E*)a.g.logits + p * a.g.ld, v, s_keys + slices * k, red);
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

// Rows, forward: a tile per workgroup.  -(gl + gh (log p + H)) p is p (A + B log2 p).
template <class T, int NT, int NV>
__global__ __launch_bounds__(NT) void log_probs_bwd_rows_kernel(LogProbBwdArgs a, int tiles) {
    constexpr int VEC = T::VEC, TILE = NT * NV * VEC;
    const long p = blockIdx.x / tiles;
    const int base = (blockIdx.x % tiles) * TILE, C = a.g.classes;
    const typename T::E* z = (const typename T::E*)a.g.logits + p * a.g.ld;
    typename T::E* dz = (typename T::E*)a.d_logits + p * C;
    Piece q[NV];
    load_tile<T, NT, NV>(q, z, base, C);
    const float m = a.row_max[p], l2 = a.row_log_sum[p], c = a.g.c;
    const long y = a.target[p];
    const float gl = a.d_log_prob && y >= 0 && y < C && l2 != INFINITY ? a.d_log_prob[p] * a.g.inv_t : 0.f;
    const float gh = a.d_entropy ? a.d_entropy[p] * a.g.inv_t : 0.f;
    const float A = -(gl + gh * a.entropy[p]), B = -gh * LN2;
    const int at = y >= 0 && y < C ? (int)y : -VEC;
    const bool far = is_far(m, c);
    const float R = far ? 0.f : reference_exponent(m, c);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int j = base + (i * NT + threadIdx.x) * VEC;
        if (j >= C) break;
        float o[VEC];
        const bool named = (unsigned)(at - j) < (unsigned)VEC;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const float x = T::get(q[i], e);
            const float d = (far ? (x - m) * c : __builtin_fmaf(x, c, -R)) - l2, w = exp2_(d);
            float g = w * __builtin_fmaf(B, bounded(d), A);
            o[e] = named && at - j == e ? g + gl : g;
        }
        if (j + VEC <= C) {
            store_piece<T>(dz + j, T::pack(o));
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                if (j + e < C) dz[j + e] = T::down(o[e]);
        }
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
    return a.temperature * a.temperature / ((a.tokens == 1 ? 1.f : a.count[b]) * (float)(a.patch * a.patch) * a.valid[0]);
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

// One position, any layout, by a whole workgroup: class after class from memory, differences (z - m) c.
template <class T, int NT>
__device__ void distill_position(const DistillArgs& a, long p, float w, Stats* red, int* s_cls, float* s_q, float* s_tot) {
    const typename T::E* z = (const typename T::E*)a.g.logits;
    const long base = a.g.base(p), cs = a.g.inner;
    const int C = a.g.classes, lane = threadIdx.x & 63;
    const float c = a.g.c;
    typename T::E* dz = (typename T::E*)a.d_logits;
    const long out = a.g.inner == 1 ? p * C : (p / a.g.inner) * C * cs + p % a.g.inner;
    Kept e = {};
    __syncthreads();
    if (threadIdx.x < 64) {
        e = load_kept(a, p, lane);
        s_cls[lane] = e.cls;
        s_q[lane] = e.q;
        if (lane == 0) { s_tot[0] = e.total; s_tot[1] = e.rest; }
    }
    __syncthreads();
    Stats v = {-INFINITY, 0.f, 0.f}, u = {-INFINITY, 0.f, 0.f};  // all classes; the ones not kept
    for (int j = threadIdx.x; j < C; j += NT) {
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
    for (int j = threadIdx.x; j < C; j += NT) {
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

template <class T>
__global__ __launch_bounds__(256) void distill_kernel(DistillArgs a) {
    __shared__ Stats red[4];
    __shared__ int s_cls[MAX_TOP];
    __shared__ float s_q[MAX_TOP], s_tot[2];
    if (a.upstream && a.skip_unit && a.upstream[0] == 1.f) return;
    const long p = blockIdx.x, cs = a.g.inner;
    const float w = position_weight(a, p);
    if (w == 0.f) {
        typename T::E* dz = (typename T::E*)a.d_logits + (p / cs) * a.g.classes * cs + p % cs;
        if (a.d_logits) for (int j = threadIdx.x; j < a.g.classes; j += 256) dz[j * cs] = T::down(0.f);
        if (threadIdx.x == 0 && a.part) a.part[p] = 0.f;
        return;
    }
    distill_position<T, 256>(a, p, w, red, s_cls, s_q, s_tot);
}

// ---- distillation of rows -------------------------------------------------------------------------------------------
// The sums over a row leave the kept classes out (their logits become -inf in the registers); what they add comes from their
// k logits.  So P, the mass outside, is a sum of its own and not a difference, and the gradient of every other class is one
// factor F times its exponential:  gs (Q 2^(R' - R) / s - r / s'),  s' and R' the sums outside, s and R those of the whole row.
struct KeptLane {  // what one wave knows of its lane's kept class
    Kept e;
    float z;         // the student's logit
    float q_class;   // the class's whole share of q (it may be listed twice)
    bool first;      // no earlier lane lists the class
};
template <class T>
__device__ __forceinline__ KeptLane load_kept_lane(const DistillArgs& a, long p, const typename T::E* z, int lane) {
    KeptLane l;
    l.e = load_kept(a, p, lane);
    l.z = l.e.cls >= 0 ? T::up(z[l.e.cls]) : -INFINITY;
    l.q_class = 0.f;
    l.first = l.e.cls >= 0;
    for (int i = 0; i < a.k; ++i) {
        const int cls = __shfl(l.e.cls, i, 64);
        const float q = __shfl(l.e.q, i, 64);
        if (cls == l.e.cls) {
            l.q_class += q;
            if (i < lane) l.first = false;
        }
    }
    return l;
}

struct RowResult { Sums all; float factor, ref; };  // factor F, R'
// One wave: the row from the sums outside the kept classes.  Writes the row's loss, returns the lane's class gradient in d.
template <class T>
__device__ __forceinline__ RowResult join_row(const DistillArgs& a, long p, float w, const KeptLane& l, const Sums& rest, float& d, int lane, bool write) {
    const float c = a.g.c;
    Sums v = {-INFINITY, -FAR, 0.f, 0.f};
    if (l.first) {
        v.m = l.z == l.z ? l.z : -INFINITY;
        v.R = reference_exponent(v.m, c);
        v.s = exp2_(__builtin_fmaf(l.z, c, -v.R));
    }
    v = join(wave_sums(v), rest);
    if (v.m == INFINITY) v.s = __builtin_nanf("");
    const bool empty = v.m == -INFINITY && v.s == 0.f;
    const float l2 = empty ? INFINITY : log2_(v.s);
    const float r = rest.s != 0.f ? l.e.rest : 0.f, Q = l.e.total + r;
    const float gs = empty ? 0.f : w * a.g.inv_t * (a.upstream ? a.upstream[0] : 1.f);
    if (write && a.part) {
        float x = l.e.q != 0.f ? l.e.q * (l.e.lq - row_log_p(a.g, l.z, v.m, l2)) : 0.f;
        x = wave_sum(x);
        if (r != 0.f) x += r * (log2_(r) - ((rest.R - v.R) + log2_(rest.s) - l2)) * LN2;
        if (lane == 0) a.part[p] = w * x;
    }
    d = gs * (exp2_(__builtin_fmaf(l.z, c, -v.R) - l2) * Q - l.q_class);
    return {v, gs * (Q * exp2_(rest.R - v.R - l2) - (r != 0.f ? r / rest.s : 0.f)), rest.R};
}

template <class T, int NT>
__device__ __forceinline__ void zero_row(typename T::E* dz, int first, int end) {
    for (int j = first + (int)threadIdx.x * T::VEC; j < end; j += NT * T::VEC) {
        if (j + T::VEC <= end) store_piece<T>(dz + j, Piece{});
        else for (int e = j; e < end; ++e) dz[e] = T::down(0.f);
    }
}

template <class T, int NT, int NV>
__device__ __forceinline__ Sums tile_sums(const Piece (&q)[NV], float c) {  // one thread's
    Sums v = {T::get(q[0], 0), 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < T::VEC; ++e) v.m = fmaxf(v.m, T::get(q[i], e));
    if (v.m != v.m) v.m = -INFINITY;
    v.R = reference_exponent(v.m, c);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < T::VEC; ++e) s += exp2_(__builtin_fmaf(T::get(q[i], e), c, -v.R));
        v.s += s;
    }
    return v;
}

// A row held in the registers of one workgroup: read once, its gradient written once.
template <class T, int NT, int NV>
__global__ __launch_bounds__(NT) void distill_rows_kernel(DistillArgs a) {
    constexpr int VEC = T::VEC;
    __shared__ __align__(16) uint32_t flags[NT * NV / 4];  // a byte per piece: which of its elements are kept classes
    __shared__ Sums red[NT / 64];
    __shared__ Stats red_far[NT / 64];
    __shared__ int s_cls[MAX_TOP];
    __shared__ float s_d[MAX_TOP], s_row[4];
    if (a.upstream && a.skip_unit && a.upstream[0] == 1.f) return;
    const long p = blockIdx.x;
    const int C = a.g.classes, lane = threadIdx.x & 63;
    const typename T::E* z = (const typename T::E*)a.g.logits + p * a.g.ld;
    typename T::E* dz = (typename T::E*)a.d_logits + p * C;
    const float w = position_weight(a, p), c = a.g.c;
    if (w == 0.f) {
        if (a.d_logits) zero_row<T, NT>(dz, 0, C);
        if (threadIdx.x == 0 && a.part) a.part[p] = 0.f;
        return;
    }
    Piece q[NV];
    load_tile<T, NT, NV>(q, z, 0, C);
    for (int i = threadIdx.x; i < NT * NV / 4; i += NT) flags[i] = 0;
    __syncthreads();
    KeptLane l;
    if (threadIdx.x < 64) {
        l = load_kept_lane<T>(a, p, z, lane);
        s_cls[lane] = l.e.cls;
        if (l.e.cls >= 0) atomicOr(&flags[l.e.cls / VEC / 4], 1u << (l.e.cls / VEC % 4 * 8 + l.e.cls % VEC));
    }
    __syncthreads();
    const uint8_t* flag = (const uint8_t*)flags;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const uint32_t f = flag[i * NT + threadIdx.x];
        if (f) {
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                if (f >> e & 1) T::put(q[i], e, -INFINITY);
        }
    }
    const Sums rest = block_sums<NT>(tile_sums<T, NT, NV>(q, c), red);
    if (threadIdx.x < 64) {
        float d;
        const RowResult row = join_row<T>(a, p, w, l, rest, d, lane, true);
        s_d[lane] = d;
        if (lane == 0) { s_row[0] = row.factor; s_row[1] = row.ref; s_row[2] = row.all.m; }
    }
    __syncthreads();
    if (is_far(s_row[2], c)) {
        distill_position<T, NT>(a, p, w, red_far, s_cls, s_d, s_row);
        return;
    }
    if (!a.d_logits) return;
    const float F = s_row[0], R = s_row[1];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int j = (i * NT + threadIdx.x) * VEC;
        if (j >= C) break;
        float o[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) o[e] = F * exp2_(__builtin_fmaf(T::get(q[i], e), c, -R));
        const uint32_t f = flag[i * NT + threadIdx.x];
        if (f)
            for (int k = 0; k < a.k; ++k) {
                const int at = s_cls[k] - j;
#pragma unroll
                for (int e = 0; e < VEC; ++e) o[e] = at == e ? s_d[k] : o[e];
            }
        if (j + VEC <= C) {
            store_piece<T>(dz + j, T::pack(o));
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                if (j + e < C) dz[j + e] = T::down(o[e]);
        }
    }
}

// Calls put(i, e, lane) for every kept class inside a tile: lane holds the class, i and e name the piece and element of the
// thread that is asked about.  Uniform over the wave but for `mine`.
template <class T, int NT, int NV, class F>
__device__ __forceinline__ void each_kept(int cls, int base, int end, F put) {
    uint64_t in = __ballot(cls >= base && cls < end && cls < base + NT * NV * T::VEC);
    while (in) {
        const int k = __builtin_ctzll(in);
        in &= in - 1;
        const int off = __shfl(cls, k, 64) - base, piece = off / T::VEC;
        if (piece % NT == (int)threadIdx.x) put(piece / NT, off % T::VEC, k);
    }
}

// Few or long rows, first pass: the sums outside the kept classes, a slice per workgroup.
template <class T, int NT, int NV>
__global__ __launch_bounds__(NT) void distill_slices_kernel(DistillArgs a, int slices, int slice_tiles, Sums* parts) {
    constexpr int VEC = T::VEC, TILE = NT * NV * VEC;
    __shared__ Sums red[NT / 64];
    if (a.upstream && a.skip_unit && a.upstream[0] == 1.f) return;
    const long p = blockIdx.x / slices;
    if (position_weight(a, p) == 0.f) return;
    const int C = a.g.classes, lane = threadIdx.x & 63, first = blockIdx.x % slices * slice_tiles * TILE;
    const int end = first + slice_tiles * TILE < C ? first + slice_tiles * TILE : C;
    const typename T::E* z = (const typename T::E*)a.g.logits + p * a.g.ld;
    const long cls64 = lane < a.k ? load_class(a.top_class, a.class_bytes, p * a.k + lane) : -1;
    const int cls = cls64 >= 0 && cls64 < C ? (int)cls64 : -1;
    Sums v = {-INFINITY, -FAR, 0.f, 0.f};
    Piece q[NV], next[NV];
    load_tile<T, NT, NV>(q, z, first, end);
    for (int base = first;;) {
        const bool more = base + TILE < end;
        if (more) load_tile<T, NT, NV>(next, z, base + TILE, end);
        each_kept<T, NT, NV>(cls, base, end, [&](int pi, int pe, int) {
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int e = 0; e < VEC; ++e)
                    if (i == pi && e == pe) T::put(q[i], e, -INFINITY);
        });
        v = join(v, tile_sums<T, NT, NV>(q, a.g.c));
        if (!more) break;
        base += TILE;
#pragma unroll
        for (int i = 0; i < NV; ++i) q[i] = next[i];
    }
    v = block_sums<NT>(v, red);
    if (threadIdx.x == 0) parts[blockIdx.x] = v;
}

// Second pass: the gradient, a tile per workgroup; the first tile's workgroup writes the row's loss.
template <class T, int NT, int NV>
__global__ __launch_bounds__(NT) void distill_tiles_kernel(DistillArgs a, int tiles, int slices, const Sums* parts) {
    constexpr int VEC = T::VEC, TILE = NT * NV * VEC;
    __shared__ Stats red_far[NT / 64];
    __shared__ int s_cls[MAX_TOP];
    __shared__ float s_d[MAX_TOP], s_row[4];
    if (a.upstream && a.skip_unit && a.upstream[0] == 1.f) return;
    const long p = blockIdx.x / tiles;
    const int tile = blockIdx.x % tiles, base = tile * TILE, C = a.g.classes, lane = threadIdx.x & 63;
    const typename T::E* z = (const typename T::E*)a.g.logits + p * a.g.ld;
    typename T::E* dz = (typename T::E*)a.d_logits + p * C;
    const float w = position_weight(a, p), c = a.g.c;
    if (w == 0.f) {
        if (a.d_logits) zero_row<T, NT>(dz, base, base + TILE < C ? base + TILE : C);
        if (tile == 0 && threadIdx.x == 0 && a.part) a.part[p] = 0.f;
        return;
    }
    Piece q[NV];
    if (a.d_logits) load_tile<T, NT, NV>(q, z, base, C);
    if (threadIdx.x < 64) {
        Sums rest = {-INFINITY, -FAR, 0.f, 0.f};
        if (lane < slices) rest = parts[p * slices + lane];
        rest = wave_sums(rest);
        const KeptLane l = load_kept_lane<T>(a, p, z, lane);
        float d;
        const RowResult row = join_row<T>(a, p, w, l, rest, d, lane, tile == 0);
        s_cls[lane] = l.e.cls;
        s_d[lane] = d;
        if (lane == 0) { s_row[0] = row.factor; s_row[1] = row.ref; s_row[2] = row.all.m; }
    }
    __syncthreads();
    if (is_far(s_row[2], c)) {
        if (tile == 0) distill_position<T, NT>(a, p, w, red_far, s_cls, s_d, s_row);
        return;
    }
    if (!a.d_logits) return;
    const float F = s_row[0], R = s_row[1];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        float o[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) o[e] = F * exp2_(__builtin_fmaf(T::get(q[i], e), c, -R));
        q[i] = T::pack(o);
    }
    each_kept<T, NT, NV>(s_cls[lane], base, C, [&](int pi, int pe, int k) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                if (i == pi && e == pe) T::put(q[i], e, s_d[k]);
    });
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int j = base + (i * NT + threadIdx.x) * VEC;
        if (j + VEC <= C) {
            store_piece<T>(dz + j, q[i]);
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                if (j + e < C) dz[j + e] = T::down(T::get(q[i], e));
        }
    }
}

// Masked tokens per sample; then the number of samples that have any (of rows, and of samples of one token: from the mask).
__global__ __launch_bounds__(64) void distill_count_kernel(const int64_t* mask, int outer, int tokens, float* count) {
    const int b = blockIdx.x;
    int n = 0;
    for (int i = threadIdx.x; i < tokens; i += 64) n += mask[(long)b * tokens + i] != 0;
    const float s = wave_sum((float)n);
    if (threadIdx.x == 0) count[b] = s;
}
__global__ __launch_bounds__(1024) void distill_valid_kernel(const float* count, const int64_t* mask, int outer, float* valid) {
    __shared__ float red[16];
    float n = 0.f;  // (whole numbers: exact in any order up to 2^24 per thread)
    for (int b = threadIdx.x; b < outer; b += 1024) n += (mask ? mask[b] != 0 : count[b] > 0.f) ? 1.f : 0.f;
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
    MMAE_REQUIRE(classes <= 1 << 30, MMAE_ESHAPE, "%s: %d classes", name, classes);
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

// Tiles of the row kernels: 32 elements a thread; one wave up to 2048 classes, four beyond.
constexpr int SHORT_ROW = 2048, ROW_TILE = 8192;
// Workgroups a row is split into: enough for every CU to hold eight, at least a tile each.
static int row_slices(int rows, int classes) {
    if (classes <= SHORT_ROW) return 1;
    const int tiles = (classes + ROW_TILE - 1) / ROW_TILE, want = (2048 + rows - 1) / rows;
    int n = want < tiles ? want : tiles;
    if (n > MAX_SLICES) n = MAX_SLICES;
    const int per = (tiles + n - 1) / n;
    return (tiles + per - 1) / per;  // (no slice is empty)
}

extern "C" size_t mmae_class_log_probs_workspace_bytes(int outer, int classes, int inner, int top_k) {
    if (inner != 1 || outer < 1 || top_k < 0) return 0;
    const int n = row_slices(outer, classes);
    return n == 1 ? 0 : (size_t)outer * n * slice_bytes(top_k);
}

template <class T>
static void launch_log_probs_rows(const LogProbArgs& a, void* workspace, hipStream_t stream) {
    constexpr int NV = 32 / T::VEC;
    const int rows = a.g.outer, n = row_slices(rows, a.g.classes);
#define ROWS(NT, TOP, tiles) hipLaunchKernelGGL((log_probs_rows_kernel<T, NT, NV, TOP>), dim3((unsigned)rows * n), dim3(NT), 0, stream, a, n, tiles, (char*)workspace)
    if (a.g.classes <= SHORT_ROW) {
        if (a.k) ROWS(64, true, 1); else ROWS(64, false, 1);
        return;
    }
    const int tiles = (a.g.classes + ROW_TILE - 1) / ROW_TILE, per = (tiles + n - 1) / n;
    if (a.k) ROWS(256, true, per); else ROWS(256, false, per);
#undef ROWS
    if (n > 1) hipLaunchKernelGGL(log_probs_join_kernel<T>, dim3(rows), dim3(64), sizeof(uint64_t) * (size_t)(n + 1) * a.k, stream, a, n, (const char*)workspace);
}

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
    MMAE_REQUIRE(workspace_bytes >= mmae_class_log_probs_workspace_bytes(outer, classes, inner, top_k) && (workspace || !workspace_bytes),
                 MMAE_EWORKSPACE, "class_log_probs: workspace too small");
    if (inner == 1) {
#define CALL(T) launch_log_probs_rows<T>(a, workspace, stream)
        BY_DTYPE(dtype, CALL);
#undef CALL
    } else {
#define CALL(T) hipLaunchKernelGGL(log_probs_kernel<T>, dim3(outer * inner), dim3(256), 0, stream, a)
        BY_DTYPE(dtype, CALL);
#undef CALL
    }
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
    if (inner == 1) {
        const int tile = classes <= SHORT_ROW ? SHORT_ROW : ROW_TILE, tiles = (classes + tile - 1) / tile;
        MMAE_REQUIRE((long)outer * tiles <= 0x7fffffffL, MMAE_ESHAPE, "class_log_probs_bwd: %d rows of %d classes", outer, classes);
#define CALL(T)                                                                                                                   \
    if (classes <= SHORT_ROW) hipLaunchKernelGGL((log_probs_bwd_rows_kernel<T, 64, 32 / T::VEC>), dim3((unsigned)outer * tiles), dim3(64), 0, stream, a, tiles); \
    else hipLaunchKernelGGL((log_probs_bwd_rows_kernel<T, 256, 32 / T::VEC>), dim3((unsigned)outer * tiles), dim3(256), 0, stream, a, tiles)
        BY_DTYPE(dtype, CALL);
#undef CALL
    } else {
#define CALL(T) hipLaunchKernelGGL(log_probs_bwd_kernel<T>, dim3(outer * inner), dim3(256), 0, stream, a)
        BY_DTYPE(dtype, CALL);
#undef CALL
    }
    MMAE_CHECK_LAUNCH("class_log_probs_bwd");
    return MMAE_OK;
}

// Rows held in registers where a workgroup takes them; in two passes over slices where there are too few rows for the card or
// they are longer.
template <class T> constexpr int longest_held_row() { return T::VEC == 8 ? 131072 : 65536; }
static bool held_rows(int rows, int classes, int dtype) {
    if (classes <= ROW_TILE) return true;
    return rows >= 256 && classes <= (dtype == MMAE_DT_F32 ? longest_held_row<F32>() : longest_held_row<B16>());
}
static size_t distill_floats(int outer, int inner) { return (4 + (size_t)outer + (size_t)outer * inner + 3) / 4 * 4; }

extern "C" size_t mmae_distill_workspace_bytes(int outer, int classes, int inner, int k) {
    if (outer < 1 || inner < 1) return 0;
    const size_t parts = inner == 1 ? sizeof(Sums) * (size_t)outer * row_slices(outer, classes) : 0;
    return sizeof(float) * distill_floats(outer, inner) + parts;
}

template <class T>
static void launch_distill_rows(const DistillArgs& a, int dtype, Sums* parts, hipStream_t stream) {
    const int rows = a.g.outer, C = a.g.classes;
    constexpr int V = T::VEC;
#define HELD(NT, EPT) hipLaunchKernelGGL((distill_rows_kernel<T, NT, EPT / V>), dim3(rows), dim3(NT), 0, stream, a)
    if (held_rows(rows, C, dtype)) {
        if (C <= 2048) HELD(64, 32);
        else if (C <= 8192) HELD(256, 32);
        else if (C <= 16384) HELD(512, 32);
        else if (C <= 32768) HELD(1024, 32);
        else if (C <= 65536) HELD(1024, 64);
        else if constexpr (V == 8) HELD(1024, 128);
        return;
    }
#undef HELD
    const int tiles = (C + ROW_TILE - 1) / ROW_TILE, n = row_slices(rows, C), per = (tiles + n - 1) / n;
    hipLaunchKernelGGL((distill_slices_kernel<T, 256, 32 / V>), dim3((unsigned)rows * n), dim3(256), 0, stream, a, n, per, parts);
    hipLaunchKernelGGL((distill_tiles_kernel<T, 256, 32 / V>), dim3((unsigned)rows * (a.d_logits ? tiles : 1)), dim3(256), 0, stream, a,
                       a.d_logits ? tiles : 1, n, (const Sums*)parts);
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
        if (a.tokens > 1) {
            hipLaunchKernelGGL(distill_count_kernel, dim3(outer), dim3(64), 0, stream, mask, outer, a.tokens, ws + 4);
            MMAE_CHECK_LAUNCH("distill_count");
        }
        hipLaunchKernelGGL(distill_valid_kernel, dim3(1), dim3(1024), 0, stream, ws + 4, a.tokens > 1 ? nullptr : mask, outer, ws);
        MMAE_CHECK_LAUNCH("distill_valid");
    }
    if (inner == 1) {
        MMAE_REQUIRE((long)outer * ((classes + ROW_TILE - 1) / ROW_TILE) <= 0x7fffffffL, MMAE_ESHAPE, "distill: %d rows of %d classes", outer, classes);
        Sums* parts = (Sums*)(ws + distill_floats(outer, inner));
#define CALL(T) launch_distill_rows<T>(a, dtype, parts, stream)
        BY_DTYPE(dtype, CALL);
#undef CALL
    } else {
#define CALL(T) hipLaunchKernelGGL(distill_kernel<T>, dim3(outer * inner), dim3(256), 0, stream, a)
        BY_DTYPE(dtype, CALL);
#undef CALL
    }
    MMAE_CHECK_LAUNCH("distill");
    if (loss) {
        hipLaunchKernelGGL(distill_sum_kernel, dim3(1), dim3(1024), 0, stream, a.part, (long)outer * inner, loss);
        MMAE_CHECK_LAUNCH("distill_sum");
    }
    return MMAE_OK;
}
