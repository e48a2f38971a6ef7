// Class distributions over rows [N, C]: a row, or a slice of it, per workgroup.
#include "classdist.h"

namespace classdist {
namespace {

// ---- log probabilities: one pass over a row, or a slice of it -------------------------------------------------------
// A thread keeps a maximum and the sums s, t against it, rescaled when it grows; H = log2 s - t / s.  HBM bounds it: 4096 x 150016
// bf16 214 us (5.7 TB/s), with 8 alternatives 224 - 238 us, where the vector ALU is busy too (87 % of the cycles); 2047 x 50001 fp32 with 8
// 83 us (4.9 TB/s).  In the first 20 ms of work after an idle card such launches take up to 330 us, until its clocks have settled.
// Short rows with alternatives are bounded by the list's barriers and searches (8192 x 5000 bf16: 20 us without, 59 us with 8); 16-bit
// rows that begin at odd elements load 16 bytes across lines (4095 x 64007: 116 us, x 64008: 101 us).
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

template <class T, int NT, int NV>
__device__ __forceinline__ void load_full_tile(Piece (&q)[NV], const typename T::E* z, int base) {
#pragma unroll
    for (int i = 0; i < NV; ++i) q[i] = load_piece<T>(z + base + (i * NT + threadIdx.x) * T::VEC);
}
// The tile at `base` of a row's first `end` classes, -inf behind them: read without a branch and inside the row (pieces behind
// the end as the last whole one; loads under conditions wait for each other), then mended: the piece that the end cuts is shifted.
template <class T, int NT, int NV>
__device__ __forceinline__ void mend_tile(Piece (&q)[NV], int base, int end) {
    constexpr int VEC = T::VEC;
    if (base + NT * NV * VEC <= end) return;
    const Piece none = {T::NEG_INF, T::NEG_INF, T::NEG_INF, T::NEG_INF};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int n = end - (base + (int)(i * NT + threadIdx.x) * VEC);
        if (n <= 0) {
            q[i] = none;
        } else if (n < VEC) {
            typedef unsigned __int128 W;
            const int bits = (VEC - n) * (int)sizeof(typename T::E) * 8;
            q[i] = __builtin_bit_cast(Piece, __builtin_bit_cast(W, q[i]) >> bits | __builtin_bit_cast(W, none) << (128 - bits));
        }
    }
}
template <class T, int NT>
__device__ __forceinline__ Piece load_inside(const typename T::E* z, int i, int base, int end) {
    const int j = base + (i * NT + (int)threadIdx.x) * T::VEC;
    return load_piece<T>(z + (j + T::VEC <= end ? j : end - T::VEC));
}
template <class T, int NT, int NV>
__device__ __forceinline__ void load_tile(Piece (&q)[NV], const typename T::E* z, int base, int end) {
    constexpr int VEC = T::VEC;
    if (base + NT * NV * VEC <= end) {
        load_full_tile<T, NT, NV>(q, z, base);
    } else if (end >= VEC) {
#pragma unroll
        for (int i = 0; i < NV; ++i) q[i] = load_inside<T, NT>(z, i, base, end);
        mend_tile<T, NT, NV>(q, base, end);
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i) q[i] = {T::NEG_INF, T::NEG_INF, T::NEG_INF, T::NEG_INF};
        if (threadIdx.x == 0 && base == 0) {
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                if (e < end) T::put(q[0], e, T::up(z[e]));
        }
    }
}

// max(a, b, c) as one instruction: through fmaxf each operand that comes from memory bits is quieted first, one more each.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}
template <class T, int NV>
__device__ __forceinline__ float tile_max(const Piece (&q)[NV]) {
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < T::VEC; e += 2) m = max3(m, T::get(q[i], e), T::get(q[i], e + 1));
    return m;
}

// The list of best keys: sorted and cut to k when it grows past SOFT, so the floor that a value has to exceed (the k-th best at
// that time) follows slowly and most tiles only append.  A tile appends at most the values above the k-th largest of the
// threads' maxima, which belong to fewer than k threads (and equal ones, which have a way of their own).
constexpr int SOFT = 2 * MAX_TOP;
template <int EPT, int NT>
struct TopList {
    static constexpr int ROOM = SOFT + (MAX_TOP - 1) * EPT;
    uint64_t keys[ROOM];
    uint64_t sorted[MAX_TOP];
    float maxima[NT];
    int count, wave_count[NT / 64];
    int added[3];  // keys appended by a tile; in turn, so that one barrier a tile is enough
};
struct ListState {  // the same in every thread
    int have, turn;
    float floor;
    bool open;  // no floor yet: fewer than k keys
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

// ordered() of the k-th largest element of one wave's tile: the bound that the maxima give leaves up to 5 k values above it where
// k is near the number of lanes that hold any (1024 x 1000 bf16, 64 alternatives: 16 us instead of 119).
template <class T, int NV>
__device__ __forceinline__ uint32_t kth_element(const Piece (&q)[NV], int k) {
    uint32_t at = 0;
    for (int b = 31; b >= 32 - T::KEY_BITS; --b) {
        const uint32_t next = at | 1u << b;
        // (the later bits are those of the least value that begins so; what lies beyond the infinities is NaN, no element reaches it)
        const float least = key_value((uint64_t)(next & 0x80000000u ? next : next | ((1ull << (32 - T::KEY_BITS)) - 1)) << 32);
        int n = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < T::VEC; ++e) n += __popcll(__ballot(T::get(q[i], e) >= least));
        if (n >= k) at = next;
    }
    at = at & 0x80000000u ? at : at | ((1ull << (32 - T::KEY_BITS)) - 1);
    return at < 0x007fffffu ? 0x007fffffu : at;  // (-inf)
}

// Ranks the keys of the list and keeps the first k, sorted.
template <int NT, class L>
__device__ __forceinline__ void keep_best(L& list, ListState& st, int k) {
    const int n = st.have;
    for (int i = threadIdx.x; i < n; i += NT) {
        const uint64_t key = list.keys[i];
        int rank = 0;
#pragma unroll 8
        for (int j = 0; j < n; ++j) rank += list.keys[j] > key;
        if (rank < k) list.sorted[rank] = key;
    }
    __syncthreads();
    st.have = n < k ? n : k;
    for (int i = threadIdx.x; i < st.have; i += NT) list.keys[i] = list.sorted[i];
    if (threadIdx.x == 0) list.count = st.have;
    __syncthreads();
    st.open = st.have < k;
    st.floor = st.open ? -INFINITY : key_value(list.keys[k - 1]);
}

// A tile that opens the list, or holds more values above the floor than the list has room for.
template <class T, int NT, int NV, class L>
__device__ __forceinline__ void take_crowded_tile(L& list, const Piece (&q)[NV], float tile_max, int base, int end, int k, ListState& st) {
    constexpr int VEC = T::VEC;
    __syncthreads();
    list.maxima[threadIdx.x] = tile_max;
    if (threadIdx.x == 0) list.count = st.have;
    __syncthreads();
    uint32_t bound;
    if (NT == 64 && 2 * k > (end - base < 64 * VEC ? (end - base) / VEC : 64)) bound = kth_element<T, NV>(q, k);
    else bound = kth_maximum<T, NT>(list.maxima, k);
    const float v = key_value((uint64_t)bound << 32);
    const bool equals = st.open || v > st.floor;  // values equal to the bound are wanted too
    const float least = equals ? v : st.floor;
    if (tile_max > least || (equals && tile_max == least)) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float x = T::get(q[i], e);
                const int j = base + (i * NT + threadIdx.x) * VEC + e;
                if ((x > least || (equals && x == least)) && j < end) {
                    const int n = atomicAdd(&list.count, 1);
                    if (n < L::ROOM) list.keys[n] = rank_key(x, j);
                }
            }
    }
    __syncthreads();
    int n = list.count;
    if (n > L::ROOM) {
        // More equal values than the list holds: the greater ones (fewer than k threads have any), then the equal ones of
        // the lowest classes, piece by piece in the order of classes.
        __syncthreads();
        if (threadIdx.x == 0) list.count = st.have;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float x = T::get(q[i], e);
                if (x > least) {
                    const int n = atomicAdd(&list.count, 1);
                    if (n < L::ROOM) list.keys[n] = rank_key(x, base + (i * NT + threadIdx.x) * VEC + e);
                }
            }
        __syncthreads();
        n = list.count < L::ROOM ? list.count : L::ROOM;
        int left = k < L::ROOM - n ? k : L::ROOM - n;  // equal values taken: k cover every need, keep_best cuts
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
    st.have = n;
    keep_best<NT>(list, st, k);
}

// Takes a tile's elements into the list.
template <class T, int NT, int NV, class L>
__device__ __forceinline__ void take_tile(L& list, const Piece (&q)[NV], float tile_max, int base, int end, int k, ListState& st) {
    constexpr int VEC = T::VEC;
    bool crowded = st.open;
    if (!crowded) {
        if (tile_max > st.floor) {
            int mine = 0;
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float x = T::get(q[i], e);
                    if (x > st.floor) {  // (behind the end: -inf)
                        const int n = atomicAdd(&list.count, 1);
                        if (n < L::ROOM) list.keys[n] = rank_key(x, base + (i * NT + threadIdx.x) * VEC + e);
                        ++mine;
                    }
                }
            atomicAdd(&list.added[st.turn], mine);
        }
        __syncthreads();
        const int added = list.added[st.turn], clear = st.turn == 0 ? 2 : st.turn - 1;
        if (threadIdx.x == 0) list.added[clear] = 0;  // last read before this barrier, next used after the next one
        st.turn = st.turn == 2 ? 0 : st.turn + 1;
        crowded = st.have + added > L::ROOM;
        if (!crowded) {
            st.have += added;
            if (st.have > SOFT) keep_best<NT>(list, st, k);
        }
    }
    if (crowded) take_crowded_tile<T, NT, NV>(list, q, tile_max, base, end, k, st);
}

// The k best of z[first, end) by k scans, for slices that hold NaN (which compare with nothing).
template <class T, int NT, class L>
__device__ __noinline__ void scan_top(L& list, const typename T::E* z, int first, int end, int k) {
    __syncthreads();
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

// The logit of the given class, asked for before the row is read: two loads that depend on each other.
template <class T>
__device__ __forceinline__ float named_logit(const LogProbArgs& a, long p, const typename T::E* z) {
    const long y = a.target[p];
    return T::up(z[y >= 0 && y < a.g.classes ? y : 0]);
}

// A row's results from its sums and its sorted best keys (keys[i], i < k); the threads of one wave.
template <class T, int NT>
__device__ __forceinline__ void finish_row(const LogProbArgs& a, long p, const typename T::E* z, Sums v, const uint64_t* keys, Sums* red, float named) {
    const float c = a.g.c;
    if (is_far(v.m, c)) v = far_sums<T, NT>(z, a.g.classes, v.m, c, red);
    if (v.m == INFINITY) v.s = __builtin_nanf("");
    const bool empty = v.m == -INFINITY && v.s == 0.f;
    const float l2 = empty ? INFINITY : log2_(v.s);
    if (threadIdx.x == 0) {
        const long y = a.target[p];
        a.log_prob[p] = y >= 0 && y < a.g.classes ? row_log_p(a.g, named, v.m, l2) : 0.f;
        a.entropy[p] = empty ? 0.f : (l2 - v.t / v.s) * LN2;
        if (a.row_max) {
            a.row_max[p] = v.m;
            a.row_log_sum[p] = l2;
        }
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
    constexpr int VEC = T::VEC, TILE = NT * NV * VEC;
    __shared__ Sums red[NT / 64];
    __shared__ TopList<NV * VEC, NT> list;
    const long p = blockIdx.x / slices;
    const int slice = blockIdx.x % slices;
    const typename T::E* z = (const typename T::E*)a.g.logits + p * a.g.ld;
    const int C = a.g.classes, first = slice * slice_tiles * TILE;
    const int end = first + slice_tiles * TILE < C ? first + slice_tiles * TILE : C;
    const float c = a.g.c;
    const float named = slices == 1 ? named_logit<T>(a, p, z) : 0.f;
    Sums v = {-INFINITY, -FAR, 0.f, 0.f};
    ListState st = {0, 0, -INFINITY, true};
    if (TOP) {
        if (threadIdx.x < 3) list.added[threadIdx.x] = 0;
    }
    auto process = [&](const Piece (&q)[NV], int base) {
        const float m = tile_max<T, NV>(q);
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
        if (TOP) take_tile<T, NT, NV>(list, q, m, base, end, a.k, st);
    };
    // Whole tiles, the next one on its way while one is worked on (the last asks for itself again: a load that depended on
    // a branch would be waited for at once); then what is left of the slice.
    Piece q[NV], next[NV];
    const int whole = first + (end - first) / TILE * TILE;
    if (whole > first) {
        load_full_tile<T, NT, NV>(q, z, first);
        for (int base = first; base < whole; base += TILE) {
            load_full_tile<T, NT, NV>(next, z, base + TILE < whole ? base + TILE : base);
            process(q, base);
#pragma unroll
            for (int i = 0; i < NV; ++i) q[i] = next[i];
        }
    }
    if (whole < end) {
        load_tile<T, NT, NV>(q, z, whole, end);
        process(q, whole);
    }
    if (TOP && st.have > a.k) keep_best<NT>(list, st, a.k);
    v = block_sums<NT>(v, red);
    if (TOP && v.s != v.s) scan_top<T, NT>(list, z, first, end, a.k);
    if (slices == 1) {
        finish_row<T, NT>(a, p, z, v, list.keys, red, named);
        return;
    }
    char* out = parts + (size_t)blockIdx.x * slice_bytes(a.k);
    if (threadIdx.x == 0) *(Sums*)out = v;
    if (TOP && (int)threadIdx.x < a.k) ((uint64_t*)(out + sizeof(Sums)))[threadIdx.x] = (int)threadIdx.x < list.count ? list.keys[threadIdx.x] : 0;
}

// Joins the slices of a row: four waves fetch the keys, then one goes on: lane i walks slice i's sorted keys.  Latency: the fetch, and
// k largest of the lanes' heads (24 x 131072 bf16, 32 slices of 20 alternatives: 7 us after 9 us of the slices; fetched by one wave, and
// the largest found by exchanges through the LDS, 5 us more).
constexpr int MAX_SLICES = 64, JOIN_NT = 256;
template <class T>
__global__ __launch_bounds__(JOIN_NT) void log_probs_join_kernel(LogProbArgs a, int slices, const char* parts) {
    extern __shared__ uint64_t s_keys[];  // [slices][k], then the k best
    __shared__ Sums red[1];
    const long p = blockIdx.x;
    const int lane = threadIdx.x & 63, k = a.k;
    const char* part = parts + (size_t)p * slices * slice_bytes(k);
    const typename T::E* z = (const typename T::E*)a.g.logits + p * a.g.ld;
    const float named = named_logit<T>(a, p, z);
    Sums v = {-INFINITY, -FAR, 0.f, 0.f};
    if (lane < slices) v = *(const Sums*)(part + lane * slice_bytes(k));
    constexpr int U = 4;  // (64 slices of 16 alternatives on their way at once)
    for (int i0 = threadIdx.x; i0 < slices * k; i0 += U * JOIN_NT) {
        uint64_t key[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * JOIN_NT < slices * k ? i0 + u * JOIN_NT : slices * k - 1;
            key[u] = ((const uint64_t*)(part + (i / k) * slice_bytes(k) + sizeof(Sums)))[i % k];
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i0 + u * JOIN_NT < slices * k) s_keys[i0 + u * JOIN_NT] = key[u];
    }
    __syncthreads();
    if (threadIdx.x >= 64) return;
    v = wave_sums(v);
    int at = 0;
    uint64_t head = lane < slices && k ? s_keys[lane * k] : 0;
    for (int i = 0; i < k; ++i) {
        const uint64_t top = wave_max_key(head);
        if (head == top && top) {  // keys are unique: one lane
            ++at;
            head = at < k ? s_keys[lane * k + at] : 0;
        }
        if (lane == 0) s_keys[slices * k + i] = top;
    }
    __syncthreads();
    finish_row<T, 64>(a, p, z, v, s_keys + slices * k, red, named);
}

template <class T, int NT>
__device__ __forceinline__ void zero_row(typename T::E* dz, int first, int end) {
    for (int j = first + (int)threadIdx.x * T::VEC; j < end; j += NT * T::VEC) {
        if (j + T::VEC <= end) store_piece<T>(dz + j, Piece{});
        else for (int e = j; e < end; ++e) dz[e] = T::down(0.f);
    }
}

// Rows, backward: a tile per workgroup.  gl 1[j = y] - (gl + gh (log p + H)) p, the second term as p (A + B log2 p).  HBM bounds it: 4095
// x 64000 bf16 199 us (5.3 TB/s).
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
    if (at < 0 && gh == 0.f) {  // an ignored row: whatever its logits are
        zero_row<T, NT>(dz, base, C - base < TILE ? C : base + TILE);
        return;
    }
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
template <class T, bool SUMS = true>
__device__ __forceinline__ KeptLane kept_lane(const DistillArgs& a, int cls, float value, const typename T::E* z, int lane, bool repeats) {
    KeptLane l;
    l.z = cls >= 0 ? T::up(z[cls]) : -INFINITY;
    l.e = kept_share<SUMS>(a, cls, value);
    l.q_class = l.e.q;
    l.first = cls >= 0;
    if (repeats) {
        l.q_class = 0.f;
        for (int i = 0; i < a.k; ++i) {
            const int other = __shfl(cls, i, 64);
            const float q = __shfl(l.e.q, i, 64);
            if (other == cls) {
                l.q_class += q;
                if (i < lane) l.first = false;
            }
        }
    }
    return l;
}

struct RowResult { float factor, ref; bool far; };  // factor F, R'; beyond FAR: to be formed anew
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
    return {gs * (Q * exp2_(rest.R - v.R - l2) - (r != 0.f ? r / rest.s : 0.f)), rest.R, is_far(v.m, c) || (a.log_probs && is_far(rest.m, c))};
}

template <class T>
__device__ __forceinline__ Piece load_some(const typename T::E* z, int n) {  // the first n elements
    if (n == T::VEC) return load_piece<T>(z);
    Piece q = {};
#pragma unroll
    for (int e = 0; e < T::VEC; ++e)
        if (e < n) T::put(q, e, T::up(z[e]));
    return q;
}
// A row beyond FAR, or whose classes that are not kept are, by a whole workgroup and differences to the two maxima: three passes over
// memory.  A bit per class modulo 1024 says which classes to look for among the kept ones.  Returns the row's weighted loss (in the first
// wave).  4096 x 32000 bf16, only the 8 kept classes not switched off: 624 us (140 us within FAR).
struct FarRoom { uint32_t bits[32]; float red[2][16]; };
template <class T>
__device__ __forceinline__ float far_row(const DistillArgs& a, long p, float w, FarRoom& room, int* s_cls, float* s_q, float* s_tot) {
    const int C = a.g.classes, lane = threadIdx.x & 63, nw = blockDim.x >> 6;
    const float c = a.g.c;
    const typename T::E* z = (const typename T::E*)a.g.logits + p * a.g.ld;
    typename T::E* dz = (typename T::E*)a.d_logits + p * C;
    Kept e = {};
    __syncthreads();
    if (threadIdx.x < 64) {
        e = load_kept(a, p, lane);
        s_cls[lane] = e.cls;
        s_q[lane] = e.q;
        if (lane == 0) { s_tot[0] = e.total; s_tot[1] = e.rest; }
        if (lane < 32) room.bits[lane] = 0;
        if (e.cls >= 0) atomicOr(&room.bits[e.cls >> 5 & 31], 1u << (e.cls & 31));
    }
    __syncthreads();
    auto maybe = [&](int j) __attribute__((always_inline)) { return (room.bits[j >> 5 & 31] >> (j & 31) & 1) != 0; };
    auto kept = [&](int j) __attribute__((always_inline)) {
        if (!maybe(j)) return false;
        for (int i = 0; i < a.k; ++i)
            if (s_cls[i] == j) return true;
        return false;
    };
    const int first = threadIdx.x * T::VEC, step = blockDim.x * T::VEC;
    float m = -INFINITY, um = -INFINITY;  // of all classes; of those not kept
    for (int j = first; j < C; j += step) {
        const int n = C - j < T::VEC ? C - j : T::VEC;
        const Piece q = load_some<T>(z + j, n);
#pragma unroll
        for (int i = 0; i < T::VEC; ++i) {
            const float x = i < n ? T::get(q, i) : -INFINITY;
            m = fmaxf(m, x);
            if (a.log_probs && !kept(j + i)) um = fmaxf(um, x);
        }
    }
    m = wave_max(m);
    um = wave_max(um);
    if (lane == 0) { room.red[0][threadIdx.x >> 6] = m; room.red[1][threadIdx.x >> 6] = um; }
    __syncthreads();
    for (int i = 0; i < nw; ++i) { m = fmaxf(m, room.red[0][i]); um = fmaxf(um, room.red[1][i]); }
    const bool nothing = m == -INFINITY;
    m = finite_ref(m);
    um = finite_ref(um);
    float s = 0.f, us = 0.f;
    for (int j = first; j < C; j += step) {
        const int n = C - j < T::VEC ? C - j : T::VEC;
        const Piece q = load_some<T>(z + j, n);
#pragma unroll
        for (int i = 0; i < T::VEC; ++i) {
            const float x = i < n ? T::get(q, i) : -INFINITY;
            s += exp2_((x - m) * c);
            if (a.log_probs && !kept(j + i)) us += exp2_((x - um) * c);
        }
    }
    s = block_sum(s, room.red[0]);
    us = block_sum(us, room.red[1]);
    const bool empty = nothing && s == 0.f;
    const float l2 = empty ? 0.f : log2_(s), ul2 = log2_(us);
    const float rest = us != 0.f ? s_tot[1] : 0.f, Q = s_tot[0] + rest;
    float l = 0.f;
    if (threadIdx.x < 64) {
        if (e.q != 0.f) l = e.q * (e.lq - a.g.log_p(T::up(z[e.cls]), m, l2));
        l = wave_sum(l);
        if (rest != 0.f) l += rest * ((log2_(rest) - (ul2 - l2)) * LN2 - (um - m) * a.g.inv_t);
        l *= w;
    }
    if (!a.d_logits) return l;
    const float gs = empty ? 0.f : w * a.g.inv_t * (a.upstream ? a.upstream[0] : 1.f);
    for (int j = first; j < C; j += step) {
        const int n = C - j < T::VEC ? C - j : T::VEC;
        const Piece q = load_some<T>(z + j, n);
        float o[T::VEC];
#pragma unroll
        for (int i = 0; i < T::VEC; ++i) {
            const float x = T::get(q, i);
            float share = 0.f;
            bool is_kept = false;
            if (maybe(j + i))
                for (int e = 0; e < a.k; ++e)
                    if (s_cls[e] == j + i) { share += s_q[e]; is_kept = true; }
            float d = exp2_((x - m) * c - l2) * Q - share;
            if (!is_kept && rest != 0.f) d -= rest * exp2_((x - um) * c - ul2);
            o[i] = gs * d;
        }
        if (n == T::VEC) store_piece<T>(dz + j, T::pack(o));
        else
#pragma unroll
            for (int i = 0; i < T::VEC; ++i)
                if (i < n) dz[j + i] = T::down(o[i]);
    }
    return l;
}

// The pieces stay as they were read: elements unpacked for one phase and kept for the next would hold twice the registers.
template <int NV>
__device__ __forceinline__ void keep_packed(Piece (&q)[NV]) {
#pragma unroll
    for (int i = 0; i < NV; ++i) asm volatile("" : "+v"(q[i].w[0]), "+v"(q[i].w[1]), "+v"(q[i].w[2]), "+v"(q[i].w[3]));
}

template <class T, int NT, int NV>
__device__ __forceinline__ Sums tile_sums(Piece (&q)[NV], float c) {  // one thread's
    Sums v = {tile_max<T, NV>(q), 0.f, 0.f, 0.f};
    v.R = reference_exponent(v.m, c);
    if (NV > 8) keep_packed<NV>(q);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < T::VEC; ++e) s += exp2_(__builtin_fmaf(T::get(q[i], e), c, -v.R));
        v.s += s;
    }
    return v;
}

__device__ __forceinline__ float uniform(float v) { return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(v))); }

// A row held in the registers of one workgroup: read once, its gradient written once.  Several workgroups a CU overlap one row's
// loads with another's stores: 8192 x 32000 fp32 414 us (5.1 TB/s).  The bound on the registers (64) keeps eight waves on a SIMD.
template <class T, int NT, int NV>
__global__ __launch_bounds__(NT, 8) void distill_rows_kernel(DistillArgs a) {
    constexpr int VEC = T::VEC;
    __shared__ __align__(16) uint32_t flags[NT * NV / 4];  // a byte per piece: which of its elements are kept classes
    __shared__ Sums red[NT / 64];
    __shared__ FarRoom far_room;
    __shared__ int s_cls[MAX_TOP];
    __shared__ float s_d[MAX_TOP], s_row[2];
    __shared__ int s_far;
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
    int cls = -1;
    float value = -INFINITY;
    if (threadIdx.x < 64) read_kept(a, p, lane, cls, value);
    Piece q[NV];
    load_tile<T, NT, NV>(q, z, 0, C);
    for (int i = threadIdx.x; i < NT * NV / 4; i += NT) flags[i] = 0;
    __syncthreads();
    KeptLane l;
    if (threadIdx.x < 64) {
        bool again = false;
        if (cls >= 0) {
            const uint32_t bit = 1u << (cls / VEC % 4 * 8 + cls % VEC);
            again = atomicOr(&flags[cls / VEC / 4], bit) & bit;
        }
        s_cls[lane] = cls;
        l = kept_lane<T>(a, cls, value, z, lane, __any(again));
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
    const Sums own = tile_sums<T, NT, NV>(q, c);
    keep_packed<NV>(q);
    const Sums rest = block_sums<NT>(own, red);
    if (threadIdx.x < 64) {
        float d;
        const RowResult row = join_row<T>(a, p, w, l, rest, d, lane, true);
        s_d[lane] = d;
        if (lane == 0) { s_row[0] = row.factor; s_row[1] = row.ref; s_far = row.far; }
    }
    __syncthreads();
    if (s_far) {
        const float x = far_row<T>(a, p, w, far_room, s_cls, s_d, s_row);
        if (threadIdx.x == 0 && a.part) a.part[p] = x;
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

// Many rows, and long ones, of which a CU holds one or two: a workgroup takes row after row, and while the pieces of one row's
// gradient leave, the next row's come into the registers they free, so that reading and writing overlap; the sums in between do
// not (4096 x 128000 bf16 500 us, 4.2 TB/s; 4095 x 64000 232 us, 4.5 TB/s).  Every piece but the last
// begins at a multiple of NT * VEC elements and the last one ends with the row, so that a piece is a uniform address and the
// thread's own offset.  The elements that the last piece shares with the one before are -inf in the last one,
// which writes its zeros first.
template <class T, int NT>
struct LongRow {
    static constexpr int VEC = T::VEC, SPAN = NT * VEC;
    int C, last;  // classes (at least SPAN); the piece that ends with the row
    __device__ __forceinline__ explicit LongRow(int classes) : C(classes), last((classes - 1) / SPAN) {}
    // (the pieces' starts are a few scalar instructions; kept from row to row they would take the registers)
    __device__ __forceinline__ LongRow again() const {
        LongRow r = *this;
        r.C = __builtin_amdgcn_readfirstlane(C);
        r.last = __builtin_amdgcn_readfirstlane(last);
        asm volatile("" : "+s"(r.C), "+s"(r.last));
        return r;
    }
    __device__ __forceinline__ int start(int i) const { return i < last ? i * SPAN : C - SPAN; }
    __device__ __forceinline__ uint32_t shared() const {  // bits of the thread's elements of the last piece that the one before holds
        const int n = last * SPAN - (C - SPAN + (int)threadIdx.x * VEC);
        return n <= 0 ? 0u : n >= VEC ? 0xffu : (1u << n) - 1;
    }
    __device__ __forceinline__ int place(int cls) const {  // the class's element, counted piece by piece and thread by thread
        const int piece = cls / SPAN;
        return piece * SPAN + cls - start(piece);
    }
    __device__ __forceinline__ Piece load(const typename T::E* z, int i) const { return load_piece<T>(z + start(i) + (unsigned)(threadIdx.x * VEC)); }
};

// What goes from kernel to kernel with a long row: the teacher's totals, made before (in 64 bits, whose constants would take
// registers from the pieces), and whether the row, or what the teacher does not keep of it, is beyond FAR.
struct RowNote { float total, rest; int far, unused; };
static_assert(sizeof(RowNote) == sizeof(Sums), "both live in the rows' workspace");
__global__ __launch_bounds__(64) void distill_notes_kernel(DistillArgs a, RowNote* notes) {
    const long p = blockIdx.x;
    const Kept e = load_kept(a, p, threadIdx.x);
    if (threadIdx.x == 0) notes[p] = {e.total, e.rest, 0, 0};
}

// The next row in the loss from `p` on, the rows outside it zeroed; `rows` behind the last.
template <class T, int NT>
__device__ __forceinline__ int next_row(const DistillArgs& a, int p, float& w) {
    const int rows = a.g.outer, C = a.g.classes;
    for (; p < rows; p += gridDim.x) {
        w = uniform(position_weight(a, p));
        if (w != 0.f) break;
        zero_row<T, NT>((typename T::E*)a.d_logits + (long)p * C, 0, C);
        if (threadIdx.x == 0 && a.part) a.part[p] = 0.f;
    }
    return p;
}

// Waves per SIMD that the registers of NV pieces a thread leave, and the workgroups of a CU.
constexpr int long_waves(int NT, int NV) { return NT == 256 ? (NV <= 4 ? 5 : 4) : NV <= 16 ? 4 : 2; }
constexpr int long_groups(int NT, int NV) { return long_waves(NT, NV) * 256 / NT; }

template <class T, int NT, int NV>
__global__ __launch_bounds__(NT, long_waves(NT, NV)) void distill_long_rows_kernel(DistillArgs a, RowNote* notes) {
    constexpr int VEC = T::VEC;
    __shared__ __align__(16) uint32_t flags[NT * NV / 4];  // a byte per piece: which of its elements are kept classes
    __shared__ Sums red[NT / 64];
    __shared__ int s_cls[MAX_TOP];
    __shared__ float s_d[MAX_TOP], s_row[2];
    if (a.upstream && a.skip_unit && a.upstream[0] == 1.f) return;
    const int C = a.g.classes, lane = threadIdx.x & 63, rows = a.g.outer;
    const float c = a.g.c;
    const LongRow<T, NT> row_at(C);
    const uint8_t* flag = (const uint8_t*)flags;
    for (int i = threadIdx.x; i < NT * NV / 4; i += NT) flags[i] = 0;
    __syncthreads();
    float w = 0.f;
    int p = next_row<T, NT>(a, blockIdx.x, w);
    if (p >= rows) return;
    int cls = -1;
    float value = -INFINITY;
    if (threadIdx.x < 64) read_kept(a, p, lane, cls, value);
    const typename T::E* z = (const typename T::E*)a.g.logits + (long)p * a.g.ld;
    Piece q[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) q[i] = row_at.load(z, i);
    while (p < rows) {
        float next_w = 0.f;
        const int next = next_row<T, NT>(a, p + gridDim.x, next_w);
        const typename T::E* next_z = (const typename T::E*)a.g.logits + (long)(next < rows ? next : p) * a.g.ld;  // (at the end: once more)
        int word = 0;
        KeptLane l;
        if (threadIdx.x < 64) {
            bool again = false;
            if (cls >= 0) {
                const int place = row_at.place(cls), byte = place / VEC;
                const uint32_t bit = 1u << (byte % 4 * 8 + place % VEC);
                word = byte / 4;
                again = atomicOr(&flags[word], bit) & bit;
            }
            s_cls[lane] = cls;
            l = kept_lane<T, false>(a, cls, value, z, lane, __any(again));
            if (a.log_probs) {
                l.e.total = notes[p].total;
                l.e.rest = notes[p].rest;
            }
        }
        __syncthreads();
        const int last = row_at.last;
        const uint32_t shared = row_at.shared();
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            uint32_t f = flag[i * NT + threadIdx.x];
            if (i >= last) f = i > last ? 0xffu : f | shared;
            if (__any(f != 0)) T::clear(q[i], f);
            __builtin_amdgcn_sched_barrier(0);
        }
        const Sums own = tile_sums<T, NT, NV>(q, c);
        keep_packed<NV>(q);
        const Sums rest = block_sums<NT>(own, red);
        if (threadIdx.x < 64) {
            float d;
            const RowResult row = join_row<T>(a, p, w, l, rest, d, lane, true);
            s_d[lane] = d;
            if (lane == 0) {
                s_row[0] = row.factor;
                s_row[1] = row.ref;
                if (row.far) notes[p].far = 1;
            }
        }
        int next_cls = -1;
        float next_value = -INFINITY;
        if (threadIdx.x < 64 && next < rows) read_kept(a, next, lane, next_cls, next_value);
        __syncthreads();
        typename T::E* dz = (typename T::E*)a.d_logits + (long)p * C;
        const float F = s_row[0], R = s_row[1];
#pragma unroll
        for (int i = NV - 1; i >= 0; --i) {
            const LongRow<T, NT> at = row_at.again();
            float o[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) o[e] = F * exp2_(__builtin_fmaf(T::get(q[i], e), c, -R));
            if (i <= at.last) store_piece<T>(dz + at.start(i) + (unsigned)(threadIdx.x * VEC), T::pack(o));
            q[i] = at.load(next_z, i);
            if (i == at.last) __syncthreads();  // (the shared elements: the piece before writes them after this one's zeros)
            __builtin_amdgcn_sched_barrier(0);  // (moved up, the loads would hold a second row's registers)
        }
        __syncthreads();
        if (cls >= 0) {  // the first wave: over the pieces' values there; it marks the next row's classes, too
            flags[word] = 0;
            dz[cls] = T::down(s_d[lane]);
        }
        p = next; w = next_w; z = next_z; cls = next_cls; value = next_value;
    }
}

// The rows that distill_long_rows_kernel found beyond FAR, anew (a kernel of its own: what it keeps would take registers from the
// long rows' pieces).
template <class T>
__global__ __launch_bounds__(256) void distill_far_rows_kernel(DistillArgs a, const RowNote* notes) {
    __shared__ FarRoom room;
    __shared__ int s_cls[MAX_TOP];
    __shared__ float s_q[MAX_TOP], s_tot[2];
    if (a.upstream && a.skip_unit && a.upstream[0] == 1.f) return;
    const long p = blockIdx.x;
    if (!notes[p].far) return;
    const float x = far_row<T>(a, p, position_weight(a, p), room, s_cls, s_q, s_tot);
    if (threadIdx.x == 0 && a.part) a.part[p] = x;
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

// Few or long rows, first pass: the sums outside the kept classes, a slice per workgroup.  Few rows are latency: 16 x 32000 bf16
// takes 7 us here and 9 us in the second pass; 64 x 128001 21 us together.
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
    int cls;
    float value;
    read_kept(a, p, lane, cls, value);
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
__global__ __launch_bounds__(NT, 8) void distill_tiles_kernel(DistillArgs a, int tiles, int slices, const Sums* parts) {
    constexpr int VEC = T::VEC, TILE = NT * NV * VEC;
    __shared__ FarRoom far_room;
    __shared__ int s_cls[MAX_TOP];
    __shared__ float s_d[MAX_TOP], s_row[2];
    __shared__ int s_far;
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
        int cls;
        float value;
        read_kept(a, p, lane, cls, value);
        const KeptLane l = kept_lane<T>(a, cls, value, z, lane, true);
        float d;
        const RowResult row = join_row<T>(a, p, w, l, rest, d, lane, tile == 0);
        s_cls[lane] = l.e.cls;
        s_d[lane] = d;
        if (lane == 0) { s_row[0] = row.factor; s_row[1] = row.ref; s_far = row.far; }
    }
    __syncthreads();
    if (s_far) {
        if (tile == 0) {
            const float x = far_row<T>(a, p, w, far_room, s_cls, s_d, s_row);
            if (threadIdx.x == 0 && a.part) a.part[p] = x;
        }
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

constexpr int CUS = 256;
constexpr int SHORT_ROW = 2048;  // up to here a row is one wave's
// Elements of a tile, a workgroup of 256 threads: in the log probabilities' forward pass, which holds a second tile on its way,
// 16 a thread (8 alternatives, 4096 x 150016 bf16 and 2047 x 50001 fp32: 238 and 88 us; 8 a thread 252 and 92, 32 a thread 240 and 97;
// 512 threads, which wait for each other at the lists' barriers, 337 and 149; all of them after 200 launches), 32 elsewhere.
constexpr int LP_NT = 256, LP_EPT = 16, LP_TILE = LP_NT * LP_EPT, ROW_TILE = 8192;
// Workgroups a row is split into, and the tiles of each: enough for every CU to hold eight, at least a tile each, none empty.
struct Split { int slices, tiles; };
Split split_row(int rows, int classes, int tile) {
    const int tiles = (classes + tile - 1) / tile, want = rows < 8 * CUS ? (8 * CUS + rows - 1) / rows : 1;
    int n = want < tiles ? want : tiles;
    if (n > MAX_SLICES) n = MAX_SLICES;
    const int per = (tiles + n - 1) / n;
    return {(tiles + per - 1) / per, per};
}
// A row of the log probabilities' forward pass is one wave's, which waits for no other, up to SHORT_ROW classes, and where every CU
// has eight rows up to 8192 (bf16, 4096 x 5000: 12 us, a workgroup of four waves 20; 8192 x 8000: 28 and 37).  The list of
// alternatives is where one wave is slow: up to 4096 with 16 of them (4096 x 4000, 8 alternatives: 23 and 27 us; 20 alternatives 32 and
// 29 us).  Beyond 4096 a wave would gain with 8 alternatives (4096 x 6000: 32 and 35 us, 8192 x 5000: 46 and 59 us); what it does with
// other lists there is not measured.
bool one_wave(int rows, int classes, int k) { return classes <= (rows < 8 * CUS || k > 16 ? SHORT_ROW : k ? 4096 : 8192); }
Split log_probs_split(int rows, int classes, int k) {
    return one_wave(rows, classes, k) ? Split{1, (classes + 64 * LP_EPT - 1) / (64 * LP_EPT)} : split_row(rows, classes, LP_TILE);
}
int row_slices(int rows, int classes) { return split_row(rows, classes, ROW_TILE).slices; }

template <class T>
static void launch_log_probs_rows(const LogProbArgs& a, void* workspace, hipStream_t stream) {
    constexpr int NV = LP_EPT / T::VEC;
    const int rows = a.g.outer;
    const Split d = log_probs_split(rows, a.g.classes, a.k);
#define ROWS(NT, TOP) \
    hipLaunchKernelGGL((log_probs_rows_kernel<T, NT, NV, TOP>), dim3((unsigned)rows * d.slices), dim3(NT), 0, stream, a, d.slices, d.tiles, (char*)workspace)
    if (one_wave(rows, a.g.classes, a.k)) {
        if (a.k) ROWS(64, true); else ROWS(64, false);
        return;
    }
    if (a.k) ROWS(LP_NT, true); else ROWS(LP_NT, false);
#undef ROWS
    if (d.slices > 1)
        hipLaunchKernelGGL(log_probs_join_kernel<T>, dim3(rows), dim3(JOIN_NT), sizeof(uint64_t) * (size_t)(d.slices + 1) * a.k, stream, a, d.slices, (const char*)workspace);
}

// Three ways.  Many rows are walked, each workgroup holding one and the next one on its way.  Fewer rows, and fp32 ones, if short, are
// held by one workgroup each; few and long ones are cut into slices and read twice, the second time mostly from the caches.
// Walked against held, logits and gradients from HBM: 16-bit rows of 2049 - 32768 classes come out even where there are many (bf16,
// 16384 x 4000: 103 us both; 4096 x 16000: 75 us both; 4096 x 32000: 135 and 137 us), gain at 4096 x 8000 (44 and 47 us) and lose at
// 16384 x 8000 (137 and 129 us); from 256 to 2047 rows held is ahead below 16000 classes (1024 x 4000: 17 and 24 us, two launches less;
// 1024 x 32000: 44 and 42 us).  fp32 rows of up to 4096 classes are held (4096 x 4000: 40 and 42 us; 65536 x 4000: 418 and 474 us).  A row
// of more than 32768 classes takes half a CU or all of it, and no second workgroup covers its loads: walked from one row per CU on
// (against slices, bf16 1024 x 128000: 152 and 170 us, 256 x 64000: 27 and 28 us; fp32 1024 x 50000: 116 and 122 us, but
// 256 x 50000: 38 and 32 us).  Held against slices: 256 x 16000 bf16 17 and 21 us, 1024 x 32000 fp32 56 and 68 us.  Rows beyond the
// registers are sliced however many they are: 4096 x 200000 bf16 941 us, 2048 x 100000 fp32 468 us (3.5 TB/s of the logits and the
// gradient, which the second reading of the logits is added to).
bool walked_rows(int rows, int classes, int dtype) {
    if (dtype == MMAE_DT_F32) return classes > 32768 && classes <= 65536 && rows >= CUS;
    return classes > SHORT_ROW && classes <= 131072 && rows >= (classes > 32768 ? CUS : 8 * CUS);
}
bool held_rows(int rows, int classes) { return classes <= ROW_TILE || (rows >= 256 && classes <= 32768); }

template <class T>
static void launch_distill_rows(const DistillArgs& a, int dtype, Sums* parts, bool again, hipStream_t stream) {
    const int rows = a.g.outer, C = a.g.classes;
    constexpr int V = T::VEC;
#define HELD(NT, EPT) hipLaunchKernelGGL((distill_rows_kernel<T, NT, EPT / V>), dim3(rows), dim3(NT), 0, stream, a)
#define LONG(NT, NV)                                                                                                           \
    do {                                                                                                                       \
        RowNote* notes = (RowNote*)parts;                                                                                      \
        const int groups = CUS * long_groups(NT, NV);                                                                          \
        if (!again) hipLaunchKernelGGL(distill_notes_kernel, dim3(rows), dim3(64), 0, stream, a, notes);                         \
        hipLaunchKernelGGL((distill_long_rows_kernel<T, NT, NV>), dim3(rows < groups ? rows : groups), dim3(NT), 0, stream, a, notes); \
        hipLaunchKernelGGL((distill_far_rows_kernel<T>), dim3(rows), dim3(256), 0, stream, a, (const RowNote*)notes);            \
        return;                                                                                                                \
    } while (0)
    if (a.d_logits && walked_rows(rows, C, dtype)) {
        if constexpr (V == 8) {
            if (C <= 4096) LONG(256, 2);
            else if (C <= 8192) LONG(256, 4);
            else if (C <= 16384) LONG(256, 8);
            else if (C <= 32768) LONG(512, 8);
            else if (C <= 49152) LONG(512, 12);
            else if (C <= 65536) LONG(512, 16);
            else if (C <= 81920) LONG(512, 20);
            else if (C <= 98304) LONG(512, 24);
            else if (C <= 114688) LONG(512, 28);
            else LONG(512, 32);
        } else {
            if (C <= 49152) LONG(512, 24);
            else LONG(512, 32);
        }
    }
    if (held_rows(rows, C)) {
        if (C <= 2048) HELD(64, 32);
        else if (C <= 8192) HELD(256, 32);
        else if (C <= 16384) HELD(512, 32);
        else HELD(1024, 32);
        return;
    }
#undef HELD
#undef LONG
    const int tiles = (C + ROW_TILE - 1) / ROW_TILE;
    const Split d = split_row(rows, C, ROW_TILE);
    if (!again) hipLaunchKernelGGL((distill_slices_kernel<T, 256, 32 / V>), dim3((unsigned)rows * d.slices), dim3(256), 0, stream, a, d.slices, d.tiles, parts);
    hipLaunchKernelGGL((distill_tiles_kernel<T, 256, 32 / V>), dim3((unsigned)rows * (a.d_logits ? tiles : 1)), dim3(256), 0, stream, a,
                       a.d_logits ? tiles : 1, d.slices, (const Sums*)parts);
}

}  // namespace

size_t log_probs_rows_workspace(int rows, int classes, int top_k) {
    const int n = log_probs_split(rows, classes, top_k).slices;
    return n == 1 ? 0 : (size_t)rows * n * slice_bytes(top_k);
}

int log_probs_rows(int dtype, const LogProbArgs& a, void* workspace, hipStream_t stream) {
    const int slices = log_probs_split(a.g.outer, a.g.classes, a.k).slices;
    REQUIRE_GRID("class_log_probs", (long)a.g.outer * slices, one_wave(a.g.outer, a.g.classes, a.k) ? 64 : LP_NT);
#define CALL(T) launch_log_probs_rows<T>(a, workspace, stream)
    BY_DTYPE(dtype, CALL);
#undef CALL
    return MMAE_OK;
}

int log_probs_bwd_rows(int dtype, const LogProbBwdArgs& a, hipStream_t stream) {
    const int C = a.g.classes, tile = C <= SHORT_ROW ? SHORT_ROW : ROW_TILE, tiles = (C + tile - 1) / tile;
    REQUIRE_GRID("class_log_probs_bwd", (long)a.g.outer * tiles, C <= SHORT_ROW ? 64 : 256);
    const unsigned grid = (unsigned)a.g.outer * tiles;
#define CALL(T)                                                                                                                    \
    if (C <= SHORT_ROW) hipLaunchKernelGGL((log_probs_bwd_rows_kernel<T, 64, 32 / T::VEC>), dim3(grid), dim3(64), 0, stream, a, tiles); \
    else hipLaunchKernelGGL((log_probs_bwd_rows_kernel<T, 256, 32 / T::VEC>), dim3(grid), dim3(256), 0, stream, a, tiles)
    BY_DTYPE(dtype, CALL);
#undef CALL
    return MMAE_OK;
}

size_t distill_rows_workspace(int rows, int classes) { return sizeof(Sums) * (size_t)rows * row_slices(rows, classes); }

int distill_rows(int dtype, const DistillArgs& a, void* workspace, bool again, hipStream_t stream) {
    const int C = a.g.classes;
    REQUIRE_GRID("distill", (long)a.g.outer * ((C + ROW_TILE - 1) / ROW_TILE), C <= SHORT_ROW ? 64 : C <= ROW_TILE ? 256 : 1024);
#define CALL(T) launch_distill_rows<T>(a, dtype, (Sums*)workspace, again, stream)
    BY_DTYPE(dtype, CALL);
#undef CALL
    return MMAE_OK;
}

}  // namespace classdist
