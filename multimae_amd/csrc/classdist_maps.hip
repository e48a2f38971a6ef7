// Class distributions over maps [B, C, inner]: the classes of 64 positions in a wave's registers or a workgroup's LDS, a lane per
// position.
//
// A class's 64 positions are 128 or 256 contiguous bytes, read and written in 16-byte pieces; in the LDS class c of position i is
// tile[c * 64 + i], which every lane reads without a conflict and at any class.  The waves of a workgroup share the classes.
#include "classdist.h"

namespace classdist {
namespace {

constexpr int LDS_BYTES = 160 * 1024;
constexpr uint32_t NONE = 0xffffffffu;

template <class T>
__device__ __forceinline__ Piece load_positions(const typename T::E* z, int px, int n) {  // px .. px + VEC of n
    if (px + T::VEC <= n) return load_piece<T>(z + px);
    Piece q = {};
#pragma unroll
    for (int e = 0; e < T::VEC; ++e)
        if (px + e < n) T::put(q, e, T::up(z[px + e]));
    return q;
}
template <class T>
__device__ __forceinline__ void store_positions(typename T::E* z, int px, int n, const Piece& q) {
    if (px + T::VEC <= n) {
        store_piece<T>(z + px, q);
    } else {
#pragma unroll
        for (int e = 0; e < T::VEC; ++e)
            if (px + e < n) z[px + e] = T::down(T::get(q, e));
    }
}

// z: the tile's first position in class 0; n positions of it exist.
template <class T>
__device__ __forceinline__ void load_map_tile(typename T::E* tile, const typename T::E* z, int C, int inner, int n) {
    constexpr int PPR = POS / T::VEC, U = 8;
    const int pieces = C * PPR, step = blockDim.x;
    for (int at = threadIdx.x; at < pieces; at += step * U) {
        Piece q[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int id = at + u * step;
            if (id < pieces) q[u] = load_positions<T>(z + (long)(id / PPR) * inner, id % PPR * T::VEC, n);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int id = at + u * step;
            if (id < pieces) *(Piece*)(tile + (size_t)id * T::VEC) = q[u];
        }
    }
}

// ---- log probabilities ----------------------------------------------------------------------------------------------
// One pass makes the sums and each lane's K best values: a sorted list takes a value with one median of three per slot.
// The waves' lists are joined (the larger ends of two sorted lists, sorted again by halving strides).  A second pass finds
// the classes: those that reach the k-th best value wait in a short queue per lane and go to the slot their rank names;
// equal values share a run of slots, which atomic minima keep in the order of classes whatever wave comes first.
//
// The 16-bit types leave the low bits of an fp32 number free: there a value carries its class along, so that the sorted list is
// the answer and the second pass falls away.
//
// 256 x 150 x 56 x 56: fp32 113 us (4.3 TB/s), with 8 alternatives 283 us; 167 x 255 x 56 x 56 bf16 72 and 186 us: the lists'
// arithmetic and, fp32, the second pass (the vector ALU is busy in 86 % of the cycles, without a list in 88 %).
constexpr int QUEUE = 16;
constexpr int CODE_BITS = 12;                   // of a carried class: the mantissa bits that bf16 (16) and f16 (13) leave
constexpr uint32_t CODES = (1u << CODE_BITS) - 1, CARRIED_INF = 0x7f800000u - (1u << CODE_BITS);  // above the largest finite value of both
template <class T> constexpr bool carries() { return sizeof(typename T::E) == 2; }

// As fp32 numbers, larger values come first and equal ones by the lower class; +-inf (and NaN, as +inf) stay finite.
__device__ __forceinline__ float carry(float v, uint32_t cls) {
    const float big = __uint_as_float(CARRIED_INF);
    const uint32_t b = __float_as_uint(__builtin_amdgcn_fmed3f(v + 0.0f, -big, big));
    const uint32_t negative = (uint32_t)((int32_t)b >> 31);
    return __uint_as_float(b | ((negative & CODES) ^ (CODES ^ cls)));
}
__device__ __forceinline__ uint32_t carried_class(float key) {
    const uint32_t b = __float_as_uint(key), negative = (uint32_t)((int32_t)b >> 31);
    return (b ^ (negative & CODES) ^ CODES) & CODES;
}
__device__ __forceinline__ float carried_value(float key) {
    const uint32_t b = __float_as_uint(key) & ~CODES;
    return (b & 0x7fffffffu) == CARRIED_INF ? __uint_as_float((b & 0x80000000u) | 0x7f800000u) : __uint_as_float(b);
}

template <int K>
__device__ __forceinline__ void list_add(float (&a)[K], float x) {
#pragma unroll
    for (int i = K - 1; i > 0; --i) a[i] = __builtin_amdgcn_fmed3f(a[i - 1], a[i], x);
    a[0] = fmaxf(a[0], x);
}

// (a list of 64 takes more registers than 16 waves leave a lane)
__host__ __device__ constexpr int most_waves(int slots) { return slots == 64 ? 8 : 16; }
__host__ __device__ inline int list_slots(int k) { return k == 0 ? 0 : k <= 4 ? 4 : k <= 8 ? 8 : k <= 16 ? 16 : k <= 32 ? 32 : 64; }
// Bytes behind the tile: the waves' sums; their lists, later their queues; the slots.
inline int log_probs_map_bytes(int element, int classes, int k, int waves) {
    const bool second = k && element == 4;  // queues and slots
    const int lists = waves * POS * list_slots(k) * 4, queues = second ? waves * POS * QUEUE * 2 : 0;
    return (classes * POS * element + 15) / 16 * 16 + waves * POS * (int)sizeof(Sums) + (lists > queues ? lists : queues) + (second ? k * POS * 4 : 0);
}

template <class T, int K>
__global__ __launch_bounds__(64 * most_waves(K)) void log_probs_map_kernel(LogProbArgs a, int tiles, MapSlices sl) {
    extern __shared__ __align__(16) char smem[];
    const int slice = blockIdx.x / tiles % sl.count, first = slice * sl.width, C = a.g.classes - first < sl.width ? a.g.classes - first : sl.width;
    const int inner = a.g.inner, k = a.k, waves = blockDim.x / 64, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    typename T::E* tile = (typename T::E*)smem;
    Sums* s_sums = (Sums*)(smem + (C * POS * sizeof(typename T::E) + 15) / 16 * 16);
    float* s_list = (float*)(s_sums + waves * POS);
    uint16_t* s_queue = (uint16_t*)s_list;
    constexpr int REGION = K * 4 > QUEUE * 2 ? K * 4 : QUEUE * 2;
    uint32_t* s_slot = (uint32_t*)((char*)s_list + (K ? waves * POS * REGION : 0));
    const int b = blockIdx.x / tiles / sl.count, i0 = blockIdx.x % tiles * POS, n = inner - i0 < POS ? inner - i0 : POS;
    const typename T::E* z = (const typename T::E*)a.g.logits + b * a.g.ld + (long)first * inner + i0;
    const long positions = (long)a.g.outer * inner;
    const bool whole = sl.count == 1;
    const float c = a.g.c;
    load_map_tile<T>(tile, z, C, inner, n);
    if (!carries<T>())
        for (int i = threadIdx.x; i < k * POS; i += blockDim.x) s_slot[i] = NONE;
    __syncthreads();

    const int c0 = (int)((long)C * wave / waves), c1 = (int)((long)C * (wave + 1) / waves);
    Sums v = {-INFINITY, -FAR, 0.f, 0.f};
    float best[K ? K : 1];
#pragma unroll
    for (int i = 0; i < K; ++i) best[i] = -INFINITY;
    for (int j = c0; j < c1; j += 8) {
        float x[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) x[u] = j + u < c1 ? T::up(tile[(j + u) * POS + lane]) : -INFINITY;
        add_logits<8, true>(v, x, c);
        if constexpr (K > 0) {
#pragma unroll
            for (int u = 0; u < 8; ++u) list_add(best, carries<T>() ? (j + u < c1 ? carry(x[u], j + u) : -INFINITY) : x[u]);
        }
    }
    if constexpr (K > 0) {
        if (__any(v.s != v.s)) {  // NaN ranks as +inf: written so into the tile, the wave's lists anew
#pragma unroll
            for (int i = 0; i < K; ++i) best[i] = -INFINITY;
            for (int j = c0; j < c1; ++j) {
                float x = T::up(tile[j * POS + lane]);
                if (x != x) {
                    x = INFINITY;
                    tile[j * POS + lane] = T::down(x);
                }
                list_add(best, carries<T>() ? carry(x, j) : x);
            }
        }
    }
    s_sums[wave * POS + lane] = v;
    if constexpr (K > 0) {
#pragma unroll
        for (int i = 0; i < K; ++i) s_list[(wave * K + i) * POS + lane] = best[i];
    }
    __syncthreads();
    v = s_sums[lane];
    for (int w = 1; w < waves; ++w) v = join(v, s_sums[w * POS + lane]);
    const long p = (long)b * inner + i0 + lane;
    if (!whole && wave == 0 && lane < n) sl.sums[slice * positions + p] = v;
    const bool far = whole && is_far(v.m, c) && v.s == v.s;
    if (__any(far)) {
        float s = 0.f, t = 0.f;
        for (int j = 0; j < C; ++j) {
            const float d = (T::up(tile[j * POS + lane]) - v.m) * c, e = exp2_(d);
            s += e;
            t += e * bounded(d);
        }
        if (far) { v.s = s; v.t = t; }
    }
    if (v.m == INFINITY) v.s = __builtin_nanf("");
    const bool empty = v.m == -INFINITY && v.s == 0.f;
    const float l2 = empty ? INFINITY : log2_(v.s);
    if (whole && wave == 0 && lane < n) {
        const long y = a.target[p];
        a.log_prob[p] = y >= 0 && y < C ? row_log_p(a.g, T::up(tile[y * POS + lane]), v.m, l2) : 0.f;
        a.entropy[p] = empty ? 0.f : (l2 - v.t / v.s) * LN2;
        if (a.row_max) {
            a.row_max[p] = v.m;
            a.row_log_sum[p] = l2;
        }
    }
    if constexpr (K > 0) {
#pragma unroll
        for (int i = 0; i < K; ++i) best[i] = s_list[i * POS + lane];
        for (int w = 1; w < waves; ++w) {
#pragma unroll
            for (int i = 0; i < K; ++i) best[i] = fmaxf(best[i], s_list[(w * K + K - 1 - i) * POS + lane]);
#pragma unroll
            for (int o = K / 2; o > 0; o >>= 1)
#pragma unroll
                for (int i = 0; i < K; ++i)
                    if (!(i & o)) {
                        const float hi = fmaxf(best[i], best[i + o]), lo = fminf(best[i], best[i + o]);
                        best[i] = hi;
                        best[i + o] = lo;
                    }
        }
        if constexpr (carries<T>()) {
            if (lane < n) {
#pragma unroll
                for (int i = 0; i < K; ++i)
                    if (i < k && i % waves == wave) {
                        const long at = ((long)b * k + i) * inner + i0 + lane;
                        const int cls = carried_class(best[i]);
                        const float x = carried_value(best[i]);
                        if (whole) {
                            a.top_class[at] = cls;
                            a.top_log_prob[at] = row_log_p(a.g, x, v.m, l2);
                        } else {
                            sl.keys[((long)slice * k + i) * positions + p] = i < C ? rank_key(x, first + cls) : 0;
                        }
                    }
            }
            return;
        }
        float least = best[0];  // the k-th best
#pragma unroll
        for (int i = 1; i < K; ++i) least = i == k - 1 ? best[i] : least;
        __syncthreads();  // the lists are read: their room is the queues' now
        uint16_t* queue = s_queue + wave * QUEUE * POS + lane;
        int queued = 0;
        auto drain = [&]() {
            for (int i = 0; __any(i < queued); ++i)
                if (i < queued) {
                    uint32_t cls = queue[i * POS];
                    const float x = T::up(tile[cls * POS + lane]);
                    int rank = 0, end = 0;
#pragma unroll
                    for (int r = 0; r < K; ++r) {
                        rank += best[r] > x;
                        end += best[r] >= x;
                    }
                    if (end > k) end = k;
                    for (int s = rank; s < end && cls != NONE; ++s) {
                        const uint32_t old = atomicMin(&s_slot[s * POS + lane], cls);
                        cls = old > cls ? old : cls;
                    }
                }
            queued = 0;
        };
        for (int j = c0; j < c1; j += 8) {
            float x[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) x[u] = T::up(tile[(j + u < c1 ? j + u : c1 - 1) * POS + lane]);
            if (__any(queued > QUEUE - 8)) drain();
#pragma unroll
            for (int u = 0; u < 8; ++u) {  // (written in any case: most classes are wanted by some lane)
                queue[queued * POS] = j + u;
                queued += lane < n && j + u < c1 && x[u] >= least;
            }
        }
        drain();
        __syncthreads();
        if (lane < n)
            for (int i = wave; i < k; i += waves) {
                const uint32_t cls = s_slot[i * POS + lane];
                const long at = ((long)b * k + i) * inner + i0 + lane;
                if (whole) {
                    a.top_class[at] = cls;
                    a.top_log_prob[at] = row_log_p(a.g, T::up(tile[cls * POS + lane]), v.m, l2);
                } else {
                    sl.keys[((long)slice * k + i) * positions + p] = i < C ? rank_key(T::up(tile[cls * POS + lane]), first + cls) : 0;
                }
            }
    }
}

// ---- log probabilities, backward: a thread's piece of positions stays the same from class to class ---------------------
// HBM bounds it: 32 x 133 x 96 x 96 bf16 31 us (5.1 TB/s).
template <class T>
__global__ __launch_bounds__(256) void log_probs_bwd_map_kernel(LogProbBwdArgs a, int tiles, int splits) {
    constexpr int VEC = T::VEC, PPR = POS / VEC, ROWS = 256 / PPR, U = 4, IGNORED = -2;
    __shared__ float s_ref[POS], s_l2[POS], s_A[POS], s_B[POS], s_gl[POS];
    __shared__ int s_at[POS], s_is_far[POS], s_far;
    const int C = a.g.classes, inner = a.g.inner, tid = threadIdx.x;
    const int t = blockIdx.x / splits, split = blockIdx.x % splits;
    const int b = t / tiles, i0 = t % tiles * POS, n = inner - i0 < POS ? inner - i0 : POS;
    const typename T::E* z = (const typename T::E*)a.g.logits + b * a.g.ld + i0;
    typename T::E* dz = (typename T::E*)a.d_logits + (long)b * C * inner + i0;
    const float c = a.g.c;
    if (tid < POS) {
        const long p = (long)b * inner + i0 + (tid < n ? tid : 0);
        const float m = a.row_max[p], l2 = a.row_log_sum[p];
        const long y = a.target[p];
        const bool named = y >= 0 && y < C;
        const float gl = a.d_log_prob && named && l2 != INFINITY ? a.d_log_prob[p] * a.g.inv_t : 0.f;
        const float gh = a.d_entropy ? a.d_entropy[p] * a.g.inv_t : 0.f;
        const bool far = is_far(m, c);
        s_ref[tid] = far ? m : reference_exponent(m, c);
        s_l2[tid] = l2;
        s_A[tid] = -(gl + gh * a.entropy[p]);
        s_B[tid] = -gh * LN2;
        s_gl[tid] = gl;
        s_at[tid] = named ? (int)y : gh == 0.f ? IGNORED : -1;
        s_is_far[tid] = far;
        const bool any = __any(far);
        if (tid == 0) s_far = any;
    }
    __syncthreads();
    const int px = tid % PPR * VEC;
    if (px >= n) return;
    float ref[VEC], l2[VEC], A[VEC], B[VEC], gl[VEC];
    int at[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        ref[e] = s_ref[px + e]; l2[e] = s_l2[px + e]; A[e] = s_A[px + e]; B[e] = s_B[px + e]; gl[e] = s_gl[px + e]; at[e] = s_at[px + e];
    }
    const bool any_far = s_far;
    const int c0 = (int)((long)C * split / splits), c1 = (int)((long)C * (split + 1) / splits);
    for (int j = c0 + tid / PPR; j < c1; j += ROWS * U) {
        Piece q[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (j + u * ROWS < c1) q[u] = load_positions<T>(z + (long)(j + u * ROWS) * inner, px, n);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int cls = j + u * ROWS;
            if (cls >= c1) break;
            float o[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float x = T::get(q[u], e);
                float d = __builtin_fmaf(x, c, -ref[e]);
                if (any_far && s_is_far[px + e]) d = (x - ref[e]) * c;
                d -= l2[e];
                const float g = exp2_(d) * __builtin_fmaf(B[e], bounded(d), A[e]);
                o[e] = cls == at[e] ? g + gl[e] : at[e] == IGNORED ? 0.f : g;  // (ignored: whatever the logits are)
            }
            store_positions<T>(dz + (long)cls * inner, px, n, T::pack(o));
        }
    }
}

// ---- distillation ---------------------------------------------------------------------------------------------------
// Wave 0 prepares the kept classes, a lane per position: each class once (an entry listed again adds its q to the entry whose
// number the tile's element holds last), the student's logits beside them, and -inf in the tile where the sums leave them out.
// After the sums the tile's logits become the gradient in place, the kept classes get theirs, and the tile is stored.  167 x 255 x
// 56 x 56 fp32, 8 kept classes: 268 us (4.0 TB/s).
inline int distill_map_bytes(int element, int classes, int k, int waves) {
    return (classes * POS * element + 15) / 16 * 16 + waves * POS * (int)sizeof(Sums) + 3 * k * POS * 4 + 2 * POS * 4;
}

template <class T> struct Bits { typedef uint16_t U; };  // an element as a whole number
template <> struct Bits<F32> { typedef uint32_t U; };

template <class T, bool REST>
__global__ __launch_bounds__(1024) void distill_map_kernel(DistillArgs a, int tiles) {
    extern __shared__ __align__(16) char smem[];
    __shared__ uint64_t s_far;
    if (a.upstream && a.skip_unit && a.upstream[0] == 1.f) return;
    typedef typename T::E E;
    typedef typename Bits<T>::U U;
    constexpr int VEC = T::VEC, PPR = POS / VEC;
    const int C = a.g.classes, inner = a.g.inner, k = a.k, waves = blockDim.x / 64, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    E* tile = (E*)smem;
    Sums* s_sums = (Sums*)(smem + (C * POS * sizeof(E) + 15) / 16 * 16);
    int* s_cls = (int*)(s_sums + waves * POS);   // [k][POS]: the class, -1 for padding and for entries listed before
    float* s_q = (float*)(s_cls + k * POS);      // its share of q, later its gradient
    float* s_z = s_q + k * POS;                  // the student's logit
    float *s_F = s_z + k * POS, *s_R = s_F + POS;
    const int b = blockIdx.x / tiles, i0 = blockIdx.x % tiles * POS, n = inner - i0 < POS ? inner - i0 : POS;
    const E* z = (const E*)a.g.logits + b * a.g.ld + i0;
    E* dz = (E*)a.d_logits + (long)b * C * inner + i0;
    const long p = (long)b * inner + i0 + lane;
    const float c = a.g.c, w = lane < n ? position_weight(a, p) : 0.f;
    if (!__any(w != 0.f)) {  // (the same in every wave)
        if (a.d_logits)
            for (int id = threadIdx.x; id < C * PPR; id += blockDim.x) store_positions<T>(dz + (long)(id / PPR) * inner, id % PPR * VEC, n, Piece{});
        if (threadIdx.x == 0 && a.part) a.part[blockIdx.x] = 0.f;
        return;
    }
    load_map_tile<T>(tile, z, C, inner, n);
    float total = 0.f, left = 0.f, loss = 0.f;  // sum of q, what it leaves, the position's loss
    if (wave == 0) {
        const long at = (long)b * k * inner + i0 + (lane < n ? lane : 0);
        float m = -INFINITY;
        read_entries(a, at, lane < n, [&](int i, int cls, float x) {
            s_cls[i * POS + lane] = cls;
            s_q[i * POS + lane] = x;
            m = fmaxf(m, x);
        });
        if (REST) shares_of_log_probs(s_q + lane, k, total, left, loss);
        else shares_of_logits(s_q + lane, k, m, c, a.g.inv_t, total, loss);
    }
    __syncthreads();
    if (wave == 0) {
        for (int i = 0; i < k; ++i) {
            const int cls = s_cls[i * POS + lane];
            s_z[i * POS + lane] = cls >= 0 ? T::up(tile[cls * POS + lane]) : -INFINITY;
        }
        for (int i = 0; i < k; ++i) {
            const int cls = s_cls[i * POS + lane];
            if (cls >= 0) tile[cls * POS + lane] = __builtin_bit_cast(E, (U)i);
        }
        for (int i = 0; i < k; ++i) {
            const int cls = s_cls[i * POS + lane];
            if (cls < 0) continue;
            const int last = __builtin_bit_cast(U, tile[cls * POS + lane]);
            if (last != i) {
                s_q[last * POS + lane] += s_q[i * POS + lane];
                s_cls[i * POS + lane] = -1;
            }
        }
        for (int i = 0; i < k; ++i) {
            const int cls = s_cls[i * POS + lane];
            if (cls >= 0) tile[cls * POS + lane] = T::down(REST ? -INFINITY : s_z[i * POS + lane]);
        }
    }
    __syncthreads();
    const int c0 = (int)((long)C * wave / waves), c1 = (int)((long)C * (wave + 1) / waves);
    Sums v = {-INFINITY, -FAR, 0.f, 0.f};
    for (int j = c0; j < c1; j += 8) {
        float x[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) x[u] = j + u < c1 ? T::up(tile[(j + u) * POS + lane]) : -INFINITY;
        add_logits<8, false>(v, x, c);
    }
    s_sums[wave * POS + lane] = v;
    __syncthreads();
    Sums rest = {};
    bool far = false;
    if (wave == 0) {
        rest = s_sums[lane];
        for (int i = 1; i < waves; ++i) rest = join(rest, s_sums[i * POS + lane]);
        v = rest;  // the whole position
        if (REST)
            for (int i = 0; i < k; ++i)
                if (s_cls[i * POS + lane] >= 0) {
                    const float x[1] = {s_z[i * POS + lane]};
                    add_logits<1, false>(v, x, c);
                }
        if (v.m == INFINITY) v.s = __builtin_nanf("");
        const bool empty = v.m == -INFINITY && v.s == 0.f;
        const float l2 = empty ? INFINITY : log2_(v.s);
        const float r = REST && rest.s != 0.f ? left : 0.f, Q = total + r;
        const float gs = empty ? 0.f : w * a.g.inv_t * (a.upstream ? a.upstream[0] : 1.f);
        far = w != 0.f && (is_far(v.m, c) || (REST && is_far(rest.m, c)));
        const uint64_t fars = __ballot(far);
        const float share_log_q = loss;
        for (int i = 0; i < k; ++i) {
            const int cls = s_cls[i * POS + lane];
            if (cls < 0 || far) continue;
            const float q = s_q[i * POS + lane], x = s_z[i * POS + lane];
            if (q != 0.f) loss -= q * row_log_p(a.g, x, v.m, l2);
            s_q[i * POS + lane] = w != 0.f ? gs * (exp2_(__builtin_fmaf(x, c, -v.R) - l2) * Q - q) : 0.f;
        }
        if (r != 0.f) loss += r * (log2_(r) - ((rest.R - v.R) + log2_(rest.s) - l2)) * LN2;
        const float sum = wave_sum(w != 0.f && !far ? w * loss : 0.f);
        if (lane == 0) {
            s_far = fars;
            if (a.part) a.part[blockIdx.x] = sum;
        }
        loss = share_log_q;
        s_F[lane] = w != 0.f ? gs * (Q * exp2_(rest.R - v.R - l2) - (r != 0.f ? r / rest.s : 0.f)) : 0.f;
        s_R[lane] = far ? (rest.m == -INFINITY ? finite_ref(v.m) : rest.m) : rest.R;
    }
    __syncthreads();
    const uint64_t fars = s_far;
    if (fars) {  // positions beyond FAR: the sums anew, by differences to the maximum of the tile's classes, which R holds there
        const float um = s_R[lane];
        float s = 0.f;
        for (int j = c0; j < c1; ++j) s += exp2_((T::up(tile[j * POS + lane]) - um) * c);
        s_sums[wave * POS + lane].s = s;
        __syncthreads();
        if (wave == 0) {
            for (int i = 1; i < waves; ++i) s += s_sums[i * POS + lane].s;
            const float m = finite_ref(v.m), apart = (um - m) * c;
            float all = s * exp2_(apart);
            if (REST)
                for (int i = 0; i < k; ++i)
                    if (s_cls[i * POS + lane] >= 0) all += exp2_((s_z[i * POS + lane] - m) * c);
            if (v.m == INFINITY) all = __builtin_nanf("");
            const float l2 = log2_(all), r = REST && s != 0.f ? left : 0.f, Q = total + r;  // (not empty: a maximum is finite)
            const float gs = w * a.g.inv_t * (a.upstream ? a.upstream[0] : 1.f);
            for (int i = 0; i < k; ++i) {
                if (s_cls[i * POS + lane] < 0 || !far) continue;
                const float q = s_q[i * POS + lane], x = s_z[i * POS + lane];
                if (q != 0.f) loss -= q * a.g.log_p(x, m, l2);
                s_q[i * POS + lane] = gs * (exp2_((x - m) * c - l2) * Q - q);
            }
            if (r != 0.f) loss += r * ((log2_(r) - (log2_(s) - l2)) * LN2 - (um - m) * a.g.inv_t);
            loss = wave_sum(far ? w * loss : 0.f);
            if (lane == 0 && a.part) a.part[blockIdx.x] += loss;
            if (far) s_F[lane] = gs * (Q * exp2_(apart - l2) - (r != 0.f ? r / s : 0.f));
        }
        __syncthreads();
    }
    if (a.d_logits) {
        const int px = threadIdx.x % PPR * VEC;  // (the workgroup's size is a multiple of PPR)
        float F[VEC], R[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) { F[e] = s_F[px + e]; R[e] = s_R[px + e]; }
        for (int id = threadIdx.x; id < C * PPR; id += blockDim.x) {
            const Piece q = *(const Piece*)(tile + (size_t)id * VEC);
            float o[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) {  // (outside the loss a logit may be anything)
                const float x = T::get(q, e);
                float d = __builtin_fmaf(x, c, -R[e]);
                if (fars && (fars >> (px + e) & 1)) d = (x - R[e]) * c;
                o[e] = F[e] != 0.f ? F[e] * exp2_(d) : 0.f;
            }
            *(Piece*)(tile + (size_t)id * VEC) = T::pack(o);
        }
        __syncthreads();
        for (int i = wave; i < k; i += waves) {
            const int cls = s_cls[i * POS + lane];
            if (cls >= 0) tile[cls * POS + lane] = T::down(s_q[i * POS + lane]);
        }
        __syncthreads();
        for (int id = threadIdx.x; id < C * PPR; id += blockDim.x)
            store_positions<T>(dz + (long)(id / PPR) * inner, id % PPR * VEC, n, *(const Piece*)(tile + (size_t)id * VEC));
    }
}

// ---- many positions, up to 136 classes: a wave per tile, the logits in its registers ------------------------------------
// The tile in the LDS bounds the maps' kernels above by latency: 34 KiB of 133 fp32 classes leave three workgroups on a CU,
// each in one phase at a time.  Held in registers the same tile takes no LDS and no other wave: 12 waves a CU that wait for
// nobody: 256 x 133 x 56 x 56 fp32 with 8 alternatives 119 us (4.4 TB/s with the outputs), in the LDS 276 us; bf16 91 and 127 us, where
// the vector ALU is busy in 74 % of the cycles (32 x 133 x 96 x 96 with 4: 38 us, 52 %; a lane loads two bytes, and 28 bytes a lane of
// the 16-bit kernels' registers are spilled under the bound of three waves a SIMD).
// CP: classes held (the first MIN of them exist).
constexpr int REG_CLASSES = 136, REG_TOP = 16;

// Class after class of a map: a uniform address that one scalar addition moves on, and the lane's offset beside it (as vector
// addresses, 136 classes would take the registers).
template <class E> using Global = __attribute__((address_space(1))) E;
template <class E>
__device__ __forceinline__ void step(Global<E>*& row, int inner) {
    row += inner;
    asm volatile("" : "+s"(row));
}
template <class T, int CP, int MIN>
__device__ __forceinline__ void load_classes(float (&x)[CP], const typename T::E* z, unsigned px, int C, int inner) {
    typedef typename T::E E;
    Global<const E>* row = (Global<const E>*)z;
    E raw[CP];  // (all of them on their way before the first is converted)
#pragma unroll
    for (int j = 0; j < CP; ++j) {  // (behind the last class: the last one again; under a branch each load would be waited for)
        raw[j] = row[px];
        step(row, j + 1 < MIN || j + 1 < C ? inner : 0);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < CP; ++j) {
        x[j] = T::up(raw[j]);
        if (j >= MIN && j >= C) x[j] = -INFINITY;
        if (sizeof(E) == 2) asm("" : "+v"(x[j]));  // (one register a class from here on: not the 16 bits and the fp32 value)
    }
}
template <int CP>
__device__ __forceinline__ float max_of(const float (&x)[CP]) {
    static_assert(CP % 2 == 0, "in pairs");
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < CP; j += 2) asm("v_max3_f32 %0, %1, %2, %3" : "=v"(m) : "v"(m), "v"(x[j]), "v"(x[j + 1]));  // (fmaxf quiets each operand first)
    return m;
}

template <class T, int CP, int MIN, int K>
__global__ __launch_bounds__(64, 3) void log_probs_map_regs_kernel(LogProbArgs a, int tiles) {
    constexpr int PLACES = K && !carries<T>() ? K + 4 : 0;  // of the queue: values and classes; the place behind it takes the overflow
    __shared__ float s_x[PLACES ? (PLACES + 1) * POS : 1];
    __shared__ uint32_t s_c[PLACES ? (PLACES + 1) * POS : 1], s_slot[PLACES ? K * POS : 1];
    const int C = a.g.classes, inner = a.g.inner, k = a.k, lane = threadIdx.x;
    const int b = blockIdx.x / tiles, i0 = blockIdx.x % tiles * POS, n = inner - i0 < POS ? inner - i0 : POS;
    const unsigned px = lane < n ? lane : 0;
    const typename T::E* z = (const typename T::E*)a.g.logits + b * a.g.ld + i0;
    const long p = (long)b * inner + i0 + px;
    const float c = a.g.c;
    const long target = a.target[p];
    const int y = target >= 0 && target < C ? (int)target : -1;
    float x[CP];
    load_classes<T, CP, MIN>(x, z, px, C, inner);
    const float named = T::up(z[(long)(y < 0 ? 0 : y) * inner + px]);
    const float m = max_of(x), R = reference_exponent(m, c);
    float s = 0.f, t = 0.f;
#pragma unroll
    for (int j = 0; j < CP; j += 8) {
        float s8 = 0.f, t8 = 0.f;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const float d = __builtin_fmaf(x[j + u], c, -R), e = exp2_(d);
            s8 += e;
            t8 = __builtin_fmaf(e, bounded(d), t8);
        }
        s += s8;
        t += t8;
    }
    const bool nan = s != s;
    if (__any(is_far(m, c) && !nan)) {
        float fs = 0.f, ft = 0.f;
#pragma unroll
        for (int j = 0; j < CP; ++j) {
            const float d = (x[j] - m) * c, e = exp2_(d);
            fs += e;
            ft += e * bounded(d);
        }
        if (is_far(m, c) && !nan) { s = fs; t = ft; }
    }
    if (m == INFINITY) s = __builtin_nanf("");
    const bool empty = m == -INFINITY && s == 0.f;
    const float l2 = empty ? INFINITY : log2_(s);
    if (lane < n) {
        a.log_prob[p] = y >= 0 ? row_log_p(a.g, named, m, l2) : 0.f;
        a.entropy[p] = empty ? 0.f : (l2 - t / s) * LN2;
        if (a.row_max) {
            a.row_max[p] = m;
            a.row_log_sum[p] = l2;
        }
    }
    if constexpr (K > 0) {
        const bool any_nan = __any(nan);
        if (any_nan) {  // NaN ranks as +inf
#pragma unroll
            for (int j = 0; j < CP; ++j) x[j] = x[j] != x[j] ? INFINITY : x[j];
        }
        float best[K];
#pragma unroll
        for (int i = 0; i < K; ++i) best[i] = -INFINITY;
        if constexpr (carries<T>()) {
#pragma unroll
            for (int j = 0; j < CP; ++j) {  // (behind the last class: -inf of a higher class, which ranks behind all others)
                list_add(best, carry(x[j], j));
                if (j % 8 == 7) {  // (the list stands here: put off, it would keep all keys beside the values)
#pragma unroll
                    for (int i = 0; i < K; ++i) asm volatile("" : "+v"(best[i]));
                }
            }
            if (lane < n) {
#pragma unroll
                for (int i = 0; i < K; ++i)
                    if (i < k) {
                        const long at = ((long)b * k + i) * inner + i0 + lane;
                        a.top_class[at] = carried_class(best[i]);
                        a.top_log_prob[at] = row_log_p(a.g, carried_value(best[i]), m, l2);
                    }
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < K; ++i) s_slot[i * POS + lane] = NONE;
#pragma unroll
        for (int j = 0; j < CP; ++j) list_add(best, x[j]);
        float least = best[0];
#pragma unroll
        for (int i = 1; i < K; ++i) least = i == k - 1 ? best[i] : least;
        int queued = 0;
        auto drain = [&]() {
            for (int i = 0; __any(i < queued); ++i)
                if (i < queued) {
                    const float v = s_x[i * POS + lane];
                    uint32_t cls = s_c[i * POS + lane];
                    int rank = 0, end = 0;
#pragma unroll
                    for (int r = 0; r < K; ++r) {
                        rank += best[r] > v;
                        end += best[r] >= v;
                    }
                    if (end > k) end = k;
                    for (int q = rank; q < end && cls != NONE; ++q) {  // equal values: the lower class first
                        const uint32_t old = s_slot[q * POS + lane];
                        if (cls < old) {
                            s_slot[q * POS + lane] = cls;
                            cls = old;
                        }
                    }
                }
            queued = 0;
        };
#pragma unroll
        for (int j = 0; j < CP; ++j)
            if (x[j] >= least && (j < MIN || j < C)) {
                const int at = (queued < PLACES ? queued : PLACES) * POS + lane;
                s_x[at] = x[j];
                s_c[at] = j;
                ++queued;
            }
        if (__any(queued > PLACES)) {  // many equal values: class after class, a full queue emptied at once
            queued = 0;
            for (int j = 0; j < C; ++j) {
                float v = T::up(z[(long)j * inner + px]);
                if (v != v) v = INFINITY;
                if (v >= least) {
                    s_x[queued * POS + lane] = v;
                    s_c[queued++ * POS + lane] = j;
                }
                if (__any(queued == PLACES)) drain();
            }
        }
        drain();
        if (lane < n) {
#pragma unroll
            for (int i = 0; i < K; ++i)
                if (i < k) {
                    const long at = ((long)b * k + i) * inner + i0 + lane;
                    a.top_class[at] = s_slot[i * POS + lane];
                    a.top_log_prob[at] = row_log_p(a.g, best[i], m, l2);
                }
        }
    }
}

// Distillation.  The kept classes of a position are bits of a mask; a kept class has a place in the LDS, the number of kept
// classes below it, which a walk over the classes counts along.  So its logit gets there and its gradient back without a
// load or store of its own, each of which would move a line per position.  256 x 133 x 56 x 56, 8 kept classes: fp32 197 us
// (4.7 TB/s with the kept classes), with the teacher's log probabilities 204 us; in the LDS 242 and 261 us.  bf16 152 and 160 us (LDS 171
// and 182): neither HBM (3.0 - 3.2 TB/s) nor the vector ALU (39 and 49 % of the cycles) is full; there are as many loads and stores as in
// fp32, of two bytes a lane, and two waves a SIMD to cover them.
template <class T, int CP, int MIN, bool REST>
__global__ __launch_bounds__(64, 2) void distill_map_regs_kernel(DistillArgs a, int tiles) {
    constexpr int WORDS = (CP + 31) / 32;
    extern __shared__ __align__(16) char smem[];
    if (a.upstream && a.skip_unit && a.upstream[0] == 1.f) return;
    typedef typename T::E E;
    const int C = a.g.classes, inner = a.g.inner, k = a.k, lane = threadIdx.x;
    int* s_cls = (int*)smem + lane;        // [k][POS], entry by entry: the class or -1, later with its place << 16
    float* s_q = (float*)smem + k * POS + lane;      // the entry's q
    float* s_z = s_q + k * POS;            // [k + 1][POS], place by place: the student's logit
    float* s_d = s_z + (k + 1) * POS;      // the class's share of q, then its gradient
    const int b = blockIdx.x / tiles, i0 = blockIdx.x % tiles * POS, n = inner - i0 < POS ? inner - i0 : POS;
    const unsigned px = lane < n ? lane : 0;
    const E* z = (const E*)a.g.logits + b * a.g.ld + i0;
    E* dz = (E*)a.d_logits + (long)b * C * inner + i0;
    const float c = a.g.c, w = lane < n ? position_weight(a, (long)b * inner + i0 + lane) : 0.f;
    const bool write = a.d_logits && lane < n;
    if (!__any(w != 0.f)) {
        if (write)
            for (int j = 0; j < C; ++j) dz[(long)j * inner + px] = T::down(0.f);
        if (lane == 0 && a.part) a.part[blockIdx.x] = 0.f;
        return;
    }
    float top = -INFINITY;
    uint32_t kept[WORDS] = {};
    read_entries(a, (long)b * k * inner + i0 + px, true, [&](int i, int cls, float v) {
        s_cls[i * POS] = cls;
        s_q[i * POS] = v;
        s_d[i * POS] = 0.f;
        top = fmaxf(top, v);
#pragma unroll
        for (int u = 0; u < WORDS; ++u) kept[u] |= cls >= 0 && cls / 32 == u ? 1u << cls % 32 : 0u;
    });
    float x[CP];
    load_classes<T, CP, MIN>(x, z, px, C, inner);
    float total, left = 0.f, loss = 0.f;  // sum of q, what it leaves, the position's loss
    if (REST) {
        double sum = 0.0;  // 64 bits: the rest is what a sum near 1 leaves
#pragma unroll 1
        for (int i = 0; i < k; ++i) {
            const float v = s_q[i * POS], q = exp_(v);
            sum += exp((double)v);
            if (q != 0.f) loss += q * v;
            s_q[i * POS] = q;
        }
        total = (float)sum;
        left = sum != sum ? total : fmaxf((float)(1.0 - sum), 0.f);
    } else {
        top = finite_ref(top);
        float sum = 0.f;
#pragma unroll 1
        for (int i = 0; i < k; ++i) {
            const float d = s_q[i * POS] - top, q = exp2_(d * c);
            sum += q;
            if (q != 0.f) loss += q * d;
            s_q[i * POS] = q;
        }
        const float inv = sum != 0.f ? 1.f / sum : 0.f;
#pragma unroll 1
        for (int i = 0; i < k; ++i) s_q[i * POS] *= inv;
        total = sum > 0.f ? 1.f : (sum != sum ? sum : 0.f);
        loss = sum != 0.f ? loss * inv * a.g.inv_t - log2_(sum) * LN2 : 0.f;
    }
    int places = 0;
#pragma unroll
    for (int u = 0; u < WORDS; ++u) places += __popc(kept[u]);
#pragma unroll 1
    for (int i = 0; i < k; ++i) {
        const int cls = s_cls[i * POS];
        if (cls < 0) continue;
        int place = 0;
#pragma unroll
        for (int u = 0; u < WORDS; ++u) place += __popc(kept[u] & (cls / 32 > u ? ~0u : cls / 32 == u ? (1u << cls % 32) - 1 : 0u));
        s_cls[i * POS] = cls | place << 16;
        s_d[place * POS] += s_q[i * POS];
    }
    {
        float* at = s_z;  // every class is written, a kept one moves on: what stands at a place is the kept class's
#pragma unroll
        for (int j = 0; j < CP; ++j) {
            const uint32_t bit = kept[j / 32] >> j % 32 & 1;
            *at = x[j];
            at += bit * POS;
            if (REST) x[j] = bit ? -INFINITY : x[j];
        }
    }
    Sums rest = {max_of(x), 0.f, 0.f, 0.f};
    rest.R = reference_exponent(rest.m, c);
#pragma unroll
    for (int j = 0; j < CP; j += 8) {
        float s8 = 0.f;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            x[j + u] = exp2_(__builtin_fmaf(x[j + u], c, -rest.R));
            s8 += x[j + u];
        }
        rest.s += s8;
    }
    Sums v = rest;  // the whole position
    if (REST)
#pragma unroll 1
        for (int i = 0; i < places; ++i) {
            const float one[1] = {s_z[i * POS]};
            add_logits<1, false>(v, one, c);
        }
    // A wave with a position beyond FAR goes by differences to the two maxima, class after class from memory.
    if (__any(is_far(v.m, c) || (REST && is_far(rest.m, c)))) {
        const float m = finite_ref(v.m), rest_m = finite_ref(rest.m);
        auto each = [&](auto take) {  // (class, logit, whether it is kept)
            for (int j0 = 0; j0 < C; j0 += 8) {
                float one[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) one[u] = T::up(z[(long)(j0 + u < C ? j0 + u : C - 1) * inner + px]);
                uint32_t word = kept[0];
#pragma unroll
                for (int u = 1; u < WORDS; ++u) word = j0 / 32 == u ? kept[u] : word;
#pragma unroll
                for (int u = 0; u < 8; ++u)
                    if (j0 + u < C) take(j0 + u, one[u], word >> ((j0 + u) & 31) & 1);
            }
        };
        float all = 0.f, out = 0.f;
        each([&](int, float one, uint32_t is_kept) {
            all += exp2_((one - m) * c);
            if (REST && !is_kept) out += exp2_((one - rest_m) * c);
        });
        if (v.m == INFINITY) all = __builtin_nanf("");
        const bool empty = v.m == -INFINITY && all == 0.f;
        const float l2 = empty ? 0.f : log2_(all), out_l2 = log2_(out), r = out != 0.f ? left : 0.f, Q = total + r;
        const float gs = empty ? 0.f : w * a.g.inv_t * (a.upstream ? a.upstream[0] : 1.f);
#pragma unroll 1
        for (int i = 0; i < places; ++i) {
            const float q = s_d[i * POS], zk = s_z[i * POS];
            if (q != 0.f) loss -= q * a.g.log_p(zk, m, l2);
            s_d[i * POS] = w != 0.f ? gs * (exp2_((zk - m) * c - l2) * Q - q) : 0.f;
        }
        if (r != 0.f) loss += r * ((log2_(r) - (out_l2 - l2)) * LN2 - (rest_m - m) * a.g.inv_t);
        loss = wave_sum(w != 0.f ? w * loss : 0.f);
        if (lane == 0 && a.part) a.part[blockIdx.x] = loss;
        if (!write) return;
        each([&](int j, float one, uint32_t) {
            const float d = exp2_((one - m) * c - l2) * Q - (r != 0.f ? r * exp2_((one - rest_m) * c - out_l2) : 0.f);
            dz[(long)j * inner + px] = T::down(w != 0.f ? gs * d : 0.f);  // (outside the loss a logit may be anything)
        });
        for (int i = 0; i < k; ++i)
            if (s_cls[i * POS] >= 0) dz[(long)(s_cls[i * POS] & 0xffff) * inner + px] = T::down(s_d[(s_cls[i * POS] >> 16) * POS]);
        return;
    }
    if (v.m == INFINITY) v.s = __builtin_nanf("");
    const bool empty = v.m == -INFINITY && v.s == 0.f;
    const float l2 = empty ? INFINITY : log2_(v.s);
    const float r = REST && rest.s != 0.f ? left : 0.f, Q = total + r;
    const float gs = empty ? 0.f : w * a.g.inv_t * (a.upstream ? a.upstream[0] : 1.f);
#pragma unroll 1
    for (int i = 0; i < places; ++i) {
        const float q = s_d[i * POS], zk = s_z[i * POS];
        if (q != 0.f) loss -= q * row_log_p(a.g, zk, v.m, l2);
        s_d[i * POS] = w != 0.f ? gs * (exp2_(__builtin_fmaf(zk, c, -v.R) - l2) * Q - q) : 0.f;
    }
    if (r != 0.f) loss += r * (log2_(r) - ((rest.R - v.R) + log2_(rest.s) - l2)) * LN2;
    loss = wave_sum(w != 0.f ? w * loss : 0.f);
    if (lane == 0 && a.part) a.part[blockIdx.x] = loss;
    if (!write) return;
    const float F = w != 0.f ? gs * (Q * exp2_(rest.R - v.R - l2) - (r != 0.f ? r / rest.s : 0.f)) : 0.f;
    Global<E>* row = (Global<E>*)dz;
    const float* at = s_d;
#pragma unroll
    for (int u = 0; u < WORDS; ++u) asm volatile("" : "+v"(kept[u]));  // (the walk anew: its addresses kept would take a register a class)
#pragma unroll
    for (int j0 = 0; j0 < CP; j0 += 8) {  // (eight places asked for at once)
        float place[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            place[u] = *at;
            at += (kept[(j0 + u) / 32] >> (j0 + u) % 32 & 1) * POS;
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int j = j0 + u;
            float d = F != 0.f ? F * x[j] : 0.f;  // (outside the loss a logit may be anything)
            d = kept[j / 32] >> j % 32 & 1 ? place[u] : d;
            if (j < MIN || j < C) row[px] = T::down(d);
            step(row, inner);
        }
    }
}

// Waves of a workgroup: enough that the workgroups whose tiles fit a CU bring 16, more where the map has few tiles.
int map_waves(long tiles, int bytes, int classes) {
    const int on_cu = LDS_BYTES / bytes < 1 ? 1 : LDS_BYTES / bytes;
    int waves = 1;
    while (waves < 16 && waves * 16 <= classes && (waves * on_cu < 16 || tiles * waves < 2048)) waves *= 2;
    return waves;
}

int allow_lds(const void* kernel, int bytes, const char* name) {
    const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    MMAE_REQUIRE(e == hipSuccess, MMAE_ELAUNCH, "%s: %d bytes of LDS refused: %s", name, bytes, hipGetErrorString(e));
    return MMAE_OK;
}

constexpr int DISTILL_STATIC = 1024;  // the distillation kernel's fixed arrays (an upper bound)

// The largest number of waves that map_waves may ask for and that fits.
template <class F>
int fitting_waves(long tiles, int classes, F bytes, int room, int most) {
    int waves = map_waves(tiles, bytes(4), classes);
    if (waves > most) waves = most;
    while (waves > 1 && bytes(waves) > room) waves /= 2;
    return waves;
}

template <class T, int K>
int launch_log_probs_map(const LogProbArgs& a, const MapSlices& s, hipStream_t stream) {
    const int tiles = map_tiles(a.g.inner), C = s.width, k = a.k;
    const long all = (long)a.g.outer * tiles * s.count;
    const int waves = fitting_waves(all, C, [&](int w) { return log_probs_map_bytes(sizeof(typename T::E), C, k, w); }, LDS_BYTES, most_waves(K));
    const int bytes = log_probs_map_bytes(sizeof(typename T::E), C, k, waves);
    if (bytes > 65536) {
        const int rc = allow_lds((const void*)log_probs_map_kernel<T, K>, bytes, "class_log_probs");
        if (rc != MMAE_OK) return rc;
    }
    REQUIRE_GRID("class_log_probs", all, 64 * waves);
    hipLaunchKernelGGL((log_probs_map_kernel<T, K>), dim3((unsigned)all), dim3(64 * waves), bytes, stream, a, tiles, s);
    return MMAE_OK;
}
// The register kernels take what fits them.  Distillation alone shares a tile of a small map among the waves of a workgroup: its
// walk over the classes is longer (8 x 133 x 56 x 56 fp32, 392 tiles: 22.5 us in registers, 20 us in the LDS; 784 tiles: 26.5
// and 34.9 us).
constexpr long REG_TILES = 512;
bool in_registers(int classes, int k) { return classes <= REG_CLASSES && k <= REG_TOP; }

#define BY_CLASSES(C, CALL)             \
    do {                                \
        if ((C) <= 32) CALL(32, 0);     \
        else if ((C) <= 64) CALL(64, 32); \
        else if ((C) <= 104) CALL(104, 64); \
        else CALL(136, 104);            \
    } while (0)

template <class T>
int launch_log_probs_map(const LogProbArgs& a, const MapSlices& s, hipStream_t stream) {
    const int tiles = map_tiles(a.g.inner);
    const long all = (long)a.g.outer * tiles;
    if (in_registers(a.g.classes, a.k)) {
        REQUIRE_GRID("class_log_probs", all, 64);
#define CALL(CP, MIN)                                                                                                              \
    do {                                                                                                                           \
        if (a.k == 0) hipLaunchKernelGGL((log_probs_map_regs_kernel<T, CP, MIN, 0>), dim3((unsigned)all), dim3(64), 0, stream, a, tiles); \
        else if (a.k <= 4) hipLaunchKernelGGL((log_probs_map_regs_kernel<T, CP, MIN, 4>), dim3((unsigned)all), dim3(64), 0, stream, a, tiles); \
        else if (a.k <= 8) hipLaunchKernelGGL((log_probs_map_regs_kernel<T, CP, MIN, 8>), dim3((unsigned)all), dim3(64), 0, stream, a, tiles); \
        else hipLaunchKernelGGL((log_probs_map_regs_kernel<T, CP, MIN, 16>), dim3((unsigned)all), dim3(64), 0, stream, a, tiles);     \
    } while (0)
        BY_CLASSES(a.g.classes, CALL);
#undef CALL
        return MMAE_OK;
    }
    switch (list_slots(a.k)) {
        case 0: return launch_log_probs_map<T, 0>(a, s, stream);
        case 4: return launch_log_probs_map<T, 4>(a, s, stream);
        case 8: return launch_log_probs_map<T, 8>(a, s, stream);
        case 16: return launch_log_probs_map<T, 16>(a, s, stream);
        case 32: return launch_log_probs_map<T, 32>(a, s, stream);
        default: return launch_log_probs_map<T, 64>(a, s, stream);
    }
}

template <class T, bool REST>
int launch_distill_map(const DistillArgs& a, hipStream_t stream) {
    const int tiles = map_tiles(a.g.inner), C = a.g.classes, k = a.k;
    const long all = (long)a.g.outer * tiles;
    if (all >= REG_TILES && in_registers(C, k)) {
        REQUIRE_GRID("distill", all, 64);
#define CALL(CP, MIN) hipLaunchKernelGGL((distill_map_regs_kernel<T, CP, MIN, REST>), dim3((unsigned)all), dim3(64), (4 * k + 2) * POS * 4, stream, a, tiles)
        BY_CLASSES(C, CALL);
#undef CALL
        return MMAE_OK;
    }
    const int waves = fitting_waves((long)a.g.outer * tiles, C, [&](int w) { return distill_map_bytes(sizeof(typename T::E), C, k, w); },
                                    LDS_BYTES - DISTILL_STATIC, 16);
    const int bytes = distill_map_bytes(sizeof(typename T::E), C, k, waves);
    if (bytes > 65536 - DISTILL_STATIC) {
        const int rc = allow_lds((const void*)distill_map_kernel<T, REST>, bytes, "distill");
        if (rc != MMAE_OK) return rc;
    }
    REQUIRE_GRID("distill", all, 64 * waves);
    hipLaunchKernelGGL((distill_map_kernel<T, REST>), dim3((unsigned)((long)a.g.outer * tiles)), dim3(64 * waves), bytes, stream, a, tiles);
    return MMAE_OK;
}

}  // namespace

int log_probs_map(int dtype, const LogProbArgs& a, const MapSlices& s, hipStream_t stream) {
    return dtype == MMAE_DT_F32 ? launch_log_probs_map<F32>(a, s, stream)
                                : dtype == MMAE_DT_BF16 ? launch_log_probs_map<B16>(a, s, stream) : launch_log_probs_map<H16>(a, s, stream);
}

int log_probs_bwd_map(int dtype, const LogProbBwdArgs& a, hipStream_t stream) {
    const int tiles = map_tiles(a.g.inner);
    const long all = (long)a.g.outer * tiles;
    int splits = 1;  // workgroups that share a tile's classes, where there are few tiles
    while (splits < 16 && all * splits < 2048 && splits * 64 < a.g.classes) splits *= 2;
    REQUIRE_GRID("class_log_probs_bwd", all * splits, 256);
#define CALL(T) hipLaunchKernelGGL(log_probs_bwd_map_kernel<T>, dim3((unsigned)(all * splits)), dim3(256), 0, stream, a, tiles, splits)
    BY_DTYPE(dtype, CALL);
#undef CALL
    return MMAE_OK;
}

int distill_map(int dtype, const DistillArgs& a, hipStream_t stream) {
    int rc = MMAE_OK;
#define CALL(T) rc = a.log_probs ? launch_distill_map<T, true>(a, stream) : launch_distill_map<T, false>(a, stream)
    BY_DTYPE(dtype, CALL);
#undef CALL
    return rc;
}

}  // namespace classdist
