// Class distributions over maps [B, C, inner] of more classes than a workgroup's LDS holds well: slices of the classes, whose sums
// (and best classes) are joined per position.  Read once for the log probabilities, twice for distillation with its gradient.
//
// A wave's load is one class of 64 neighbouring positions.  The log probabilities' lists of best classes are joined by a lane per
// position where the slices are few, by a wave per position where they are many.  131 x 1000 x 32 x 32 fp32 (537 MB): log
// probabilities 118 us (4.6 TB/s), with 8 alternatives 313 us, where the lists bound them (the vector ALU is busy in 91 % of the cycles),
// distillation with its gradient 438 us (three passes, 3.7 TB/s); a workgroup per position, which reads a line for each of its logits,
// takes 1270, 9121 and 4030 us.  Maps of few positions a sample (2 x 2) leave most lanes idle.
#include "classdist.h"

namespace classdist {
namespace {

constexpr int U = 8;  // loads on their way

// The slices' sums of one position.
__device__ __forceinline__ Sums join_slices(const Sums* sums, int count, long positions) {
    Sums v = {-INFINITY, -FAR, 0.f, 0.f};
    for (int s0 = 0; s0 < count; s0 += U) {
        Sums x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) x[u] = sums[(s0 + u < count ? s0 + u : count - 1) * positions];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (s0 + u < count) v = join(v, x[u]);
    }
    return v;
}

// A lane per position: joins the sums and walks the slices' sorted keys, each into the list of the best so far (in the LDS, sorted)
// as long as they reach it.
template <class T>
__global__ __launch_bounds__(64) void log_probs_map_join_kernel(LogProbArgs a, int tiles, MapSlices sl) {
    extern __shared__ uint64_t s_best[];  // [k][POS]
    const int inner = a.g.inner, k = a.k, lane = threadIdx.x;
    const int b = blockIdx.x / tiles, i0 = blockIdx.x % tiles * POS, n = inner - i0 < POS ? inner - i0 : POS;
    if (lane >= n) return;
    const long positions = (long)a.g.outer * inner, p = (long)b * inner + i0 + lane;
    const typename T::E* z = (const typename T::E*)a.g.logits + b * a.g.ld + i0 + lane;
    const float c = a.g.c;
    const long y = a.target[p];
    const bool named = y >= 0 && y < a.g.classes;
    const float zy = T::up(z[(named ? y : 0) * inner]);
    Sums v = join_slices(sl.sums + p, sl.count, positions);
    if (is_far(v.m, c) && v.s == v.s) {
        v.s = v.t = 0.f;
        for (int j = 0; j < a.g.classes; ++j) {
            const float d = (T::up(z[(long)j * inner]) - v.m) * c, e = exp2_(d);
            v.s += e;
            v.t += e * bounded(d);
        }
    }
    if (v.m == INFINITY) v.s = __builtin_nanf("");
    const bool empty = v.m == -INFINITY && v.s == 0.f;
    const float l2 = empty ? INFINITY : log2_(v.s);
    a.log_prob[p] = named ? row_log_p(a.g, zy, v.m, l2) : 0.f;
    a.entropy[p] = empty ? 0.f : (l2 - v.t / v.s) * LN2;
    if (a.row_max) {
        a.row_max[p] = v.m;
        a.row_log_sum[p] = l2;
    }
    if (!k) return;
    uint64_t* best = s_best + lane;
    const uint64_t* keys = sl.keys + p;
    for (int i = 0; i < k; ++i) best[i * POS] = keys[i * positions];  // the first slice's are sorted already
    uint64_t worst = best[(k - 1) * POS];
    for (int s = 1; s < sl.count; ++s) {
        const uint64_t* from = keys + (long)s * k * positions;
        bool more = true;
        for (int i0 = 0; i0 < k && more; i0 += U) {
            uint64_t key[U];
#pragma unroll
            for (int u = 0; u < U; ++u) key[u] = from[(i0 + u < k ? i0 + u : k - 1) * positions];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                more = more && i0 + u < k && key[u] > worst;
                if (more) {
                    int j = k - 1;
                    for (; j > 0; --j) {
                        const uint64_t above = best[(j - 1) * POS];
                        if (above > key[u]) break;
                        best[j * POS] = above;
                    }
                    best[j * POS] = key[u];
                    worst = best[(k - 1) * POS];
                }
            }
        }
    }
    for (int i = 0; i < k; ++i) {
        const uint64_t key = best[i * POS];
        const long at = ((long)b * k + i) * inner + i0 + lane;
        a.top_class[at] = key_class(key);
        a.top_log_prob[at] = row_log_p(a.g, key_value(key), v.m, l2);
    }
}

// The same with a wave per position, a lane per slice: k times the largest of the lanes' heads, whose lane takes its next key.  The
// last lane holds the best of the slices before, 63 at a time.  Each key costs six exchanges instead of insertions that wait for
// each other: 16 x 32000 x 16 x 16 bf16, 63 slices, with 8 alternatives 202 us (338 by lanes), with 64 719 us (2351).  4
// slices fill 4 lanes only (131 x 1000 x 32 x 32 fp32 with 8: 742 us instead of 569); from 8 to 16 both take the same.
template <class T>
__global__ __launch_bounds__(256) void log_probs_map_merge_kernel(LogProbArgs a, MapSlices sl) {
    const int inner = a.g.inner, k = a.k, lane = threadIdx.x & 63;
    const long positions = (long)a.g.outer * inner, p = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (p >= positions) return;
    const long b = p / inner, i0 = p % inner;
    const typename T::E* z = (const typename T::E*)a.g.logits + b * a.g.ld + i0;
    const float c = a.g.c;
    const long y = a.target[p];
    const bool named = y >= 0 && y < a.g.classes;
    const float zy = T::up(z[(named ? y : 0) * inner]);
    Sums v = {-INFINITY, -FAR, 0.f, 0.f};
    for (int s = lane; s < sl.count; s += 64) v = join(v, sl.sums[s * positions + p]);
    v = wave_sums(v);
    if (is_far(v.m, c) && v.s == v.s) {
        float s = 0.f, t = 0.f;
        for (int j = lane; j < a.g.classes; j += 64) {
            const float d = (T::up(z[(long)j * inner]) - v.m) * c, e = exp2_(d);
            s += e;
            t += e * bounded(d);
        }
        v.s = wave_sum(s);
        v.t = wave_sum(t);
    }
    if (v.m == INFINITY) v.s = __builtin_nanf("");
    const bool empty = v.m == -INFINITY && v.s == 0.f;
    const float l2 = empty ? INFINITY : log2_(v.s);
    if (lane == 0) {
        a.log_prob[p] = named ? row_log_p(a.g, zy, v.m, l2) : 0.f;
        a.entropy[p] = empty ? 0.f : (l2 - v.t / v.s) * LN2;
        if (a.row_max) {
            a.row_max[p] = v.m;
            a.row_log_sum[p] = l2;
        }
    }
    uint64_t best = 0;  // lane i: the i-th best of the slices so far
    for (int s0 = 0; s0 < sl.count; s0 += 63) {
        const bool slice = lane < 63 && s0 + lane < sl.count;
        const uint64_t* keys = sl.keys + (long)(slice ? s0 + lane : 0) * k * positions + p;
        uint64_t head = keys[0], next = keys[k > 1 ? positions : 0], fresh = 0;
        if (!slice || k == 1) next = 0;
        if (!slice) head = 0;
        const uint64_t first = __shfl((unsigned long long)best, 0, 64);
        if (lane == 63) head = first;
        int at = 0;  // of the lane's head
        for (int i = 0; i < k; ++i) {
            const uint64_t top = wave_max_key(head);
            if (lane == i) fresh = top;
            if (!top) break;
            const bool mine = head == top;  // keys are unique: one lane
            if (mine) ++at;
            const uint64_t follow = __shfl((unsigned long long)best, __shfl(at, 63, 64) & 63, 64);
            if (mine) {
                head = next;
                if (lane == 63) head = at < k ? follow : 0;
                else next = at + 1 < k ? keys[(at + 1) * positions] : 0;
            }
        }
        best = fresh;
    }
    if (lane < k) {
        const long at = (b * k + lane) * inner + i0;
        a.top_class[at] = key_class(best);
        a.top_log_prob[at] = row_log_p(a.g, key_value(best), v.m, l2);
    }
}

// ---- distillation -------------------------------------------------------------------------------------------------------
// First the sums over the classes that are not kept, a bit per class and position of the slice says which are; then a lane per
// position joins them, adds the kept classes and leaves the factors of the gradient; then the gradient, slice by slice.
constexpr int SLICE_BYTES = 64 * 1024, MOST_WIDTH = SLICE_BYTES / (POS * 2);  // a CU holds two such tiles

struct SliceNotes {  // per position: gradient = F 2^(x c - R) where not kept (2^((x - m) c) where m is a number: beyond FAR); the kept classes' beside
    float *F, *R, *m;
    int* cls;   // [k][positions], -1: none
    float* g;
};

__device__ __forceinline__ bool skip_call(const DistillArgs& a) { return a.upstream && a.skip_unit && a.upstream[0] == 1.f; }

template <class T>
__global__ __launch_bounds__(256) void distill_map_sums_kernel(DistillArgs a, int tiles, int count, int width, Sums* sums) {
    __shared__ uint32_t kept[MOST_WIDTH * 2];
    __shared__ Sums part[4 * POS];
    const int slice = blockIdx.x / tiles % count, first = slice * width, C = a.g.classes - first < width ? a.g.classes - first : width;
    const int b = blockIdx.x / tiles / count, i0 = blockIdx.x % tiles * POS, inner = a.g.inner, n = inner - i0 < POS ? inner - i0 : POS;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = i0 + (lane < n ? lane : n - 1);
    const long p = (long)b * inner + i;
    const float w = position_weight(a, p), c = a.g.c;
    if (!__any(w != 0.f)) return;  // (the same in every wave)
    for (int j = threadIdx.x; j < 2 * C; j += 256) kept[j] = 0;
    __syncthreads();
    for (int e = wave; e < a.k; e += 4) {
        const long cls = load_class(a.top_class, a.class_bytes, ((long)b * a.k + e) * inner + i) - first;
        if (cls >= 0 && cls < C && lane < n) atomicOr(&kept[cls * 2 + (lane >> 5)], 1u << (lane & 31));
    }
    __syncthreads();
    const typename T::E* z = (const typename T::E*)a.g.logits + b * a.g.ld + (long)first * inner + i;
    const int c0 = C * wave / 4, c1 = C * (wave + 1) / 4;
    Sums v = {-INFINITY, -FAR, 0.f, 0.f};
    for (int j = c0; j < c1; j += U) {
        float x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) x[u] = T::up(z[(long)(j + u < c1 ? j + u : c1 - 1) * inner]);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool in = j + u < c1 && !(kept[(j + u < c1 ? j + u : c1 - 1) * 2 + (lane >> 5)] >> (lane & 31) & 1);
            x[u] = in ? x[u] : -INFINITY;
        }
        add_logits<U, false>(v, x, c);
    }
    part[threadIdx.x] = v;
    __syncthreads();
    if (wave == 0 && lane < n) {
        for (int o = 1; o < 4; ++o) v = join(v, part[o * POS + lane]);
        sums[(long)slice * a.g.outer * inner + p] = v;
    }
}

template <class T>
__global__ __launch_bounds__(64) void distill_map_join_kernel(DistillArgs a, int tiles, int count, const Sums* sums, SliceNotes notes) {
    extern __shared__ int s_cls[];  // [k][POS], then q (later the gradient) and the student's logits alike
    if (skip_call(a)) return;
    const int inner = a.g.inner, k = a.k, lane = threadIdx.x;
    const int b = blockIdx.x / tiles, i0 = blockIdx.x % tiles * POS, n = inner - i0 < POS ? inner - i0 : POS;
    const int i = i0 + (lane < n ? lane : n - 1);
    const long positions = (long)a.g.outer * inner, p = (long)b * inner + i;
    const float c = a.g.c, w = lane < n ? position_weight(a, p) : 0.f;
    const uint64_t live = __ballot(w != 0.f);
    if (!live) {
        if (lane == 0 && a.part) a.part[blockIdx.x] = 0.f;
        return;
    }
    const typename T::E* z = (const typename T::E*)a.g.logits + b * a.g.ld + i;
    float* s_q = (float*)s_cls + k * POS;
    float* s_z = s_q + k * POS;
    float m = -INFINITY, total = 0.f, left = 0.f, loss = 0.f;
    read_entries(a, (long)b * k * inner + i, w != 0.f, [&](int e, int cls, float x) {
        s_cls[e * POS + lane] = cls;
        s_q[e * POS + lane] = x;
        s_z[e * POS + lane] = cls >= 0 ? T::up(z[(long)cls * inner]) : -INFINITY;
        m = fmaxf(m, x);
    });
    if (a.log_probs) shares_of_log_probs(s_q + lane, k, total, left, loss);
    else shares_of_logits(s_q + lane, k, m, c, a.g.inv_t, total, loss);
    for (int e = 1; e < k; ++e) {  // an entry listed before adds its q to that one
        const int cls = s_cls[e * POS + lane];
        for (int o = 0; o < e && cls >= 0; ++o)
            if (s_cls[o * POS + lane] == cls) {
                s_q[o * POS + lane] += s_q[e * POS + lane];
                s_cls[e * POS + lane] = -1;
                break;
            }
    }
    Sums rest = join_slices(sums + p, count, positions);
    Sums v = rest;
    for (int e = 0; e < k; ++e)
        if (s_cls[e * POS + lane] >= 0) {
            const float x[1] = {s_z[e * POS + lane]};
            add_logits<1, false>(v, x, c);
        }
    // Beyond FAR, of all classes or of those not kept: the sums anew, by differences to the latter's maximum, class after class from memory.
    const bool far = w != 0.f && (is_far(v.m, c) || (a.log_probs && is_far(rest.m, c)));
    const float top = finite_ref(v.m), rest_m = rest.m == -INFINITY ? top : rest.m, apart = (rest_m - top) * c;
    if (__any(far)) {
        float s = 0.f;
        for (int j0 = 0; j0 < a.g.classes; j0 += U) {
            float x[U];
#pragma unroll
            for (int u = 0; u < U; ++u) x[u] = T::up(z[(long)(j0 + u < a.g.classes ? j0 + u : a.g.classes - 1) * inner]);
            uint32_t out = a.g.classes - j0 < U ? (1u << (a.g.classes - j0)) - 1 : (1u << U) - 1;
            for (int e = 0; e < k; ++e) {
                const unsigned at = s_cls[e * POS + lane] - j0;
                out &= ~(at < U ? 1u << at : 0u);
            }
            float s8 = 0.f;
#pragma unroll
            for (int u = 0; u < U; ++u) s8 += out >> u & 1 ? exp2_((x[u] - rest_m) * c) : 0.f;
            s += s8;
        }
        float all = s * exp2_(apart);
        for (int e = 0; e < k; ++e)
            if (s_cls[e * POS + lane] >= 0) all += exp2_((s_z[e * POS + lane] - top) * c);
        if (far) { rest.s = s; v.s = all; }
    }
    if (v.m == INFINITY) v.s = __builtin_nanf("");
    const bool empty = v.m == -INFINITY && v.s == 0.f;
    const float l2 = empty ? INFINITY : log2_(v.s);
    const float r = a.log_probs && rest.s != 0.f ? left : 0.f, Q = total + r;
    const float gs = empty ? 0.f : w * a.g.inv_t * (a.upstream ? a.upstream[0] : 1.f);
    for (int e = 0; e < k; ++e) {
        const int cls = s_cls[e * POS + lane];
        const float q = s_q[e * POS + lane], x = s_z[e * POS + lane];
        if (cls >= 0 && q != 0.f) loss -= q * (far ? a.g.log_p(x, top, l2) : row_log_p(a.g, x, v.m, l2));
        if (a.d_logits && lane < n) {
            notes.cls[e * positions + p] = w != 0.f ? cls : -1;
            notes.g[e * positions + p] = gs * (exp2_((far ? (x - top) * c : __builtin_fmaf(x, c, -v.R)) - l2) * Q - q);
        }
    }
    if (r != 0.f) loss += far ? r * ((log2_(r) - (log2_(rest.s) - l2)) * LN2 - (rest_m - top) * a.g.inv_t) : r * (log2_(r) - ((rest.R - v.R) + log2_(rest.s) - l2)) * LN2;
    loss = wave_sum(w != 0.f ? w * loss : 0.f);
    if (a.d_logits && lane < n) {
        notes.F[p] = w != 0.f ? gs * (Q * exp2_((far ? apart : rest.R - v.R) - l2) - (r != 0.f ? r / rest.s : 0.f)) : 0.f;
        notes.R[p] = rest.R;
        notes.m[p] = far ? rest_m : __builtin_nanf("");
    }
    if (lane == 0 && a.part) a.part[blockIdx.x] = loss;
}

template <class T>
__global__ __launch_bounds__(256) void distill_map_gradient_kernel(DistillArgs a, int tiles, int count, int width, SliceNotes notes) {
    if (skip_call(a)) return;
    const int slice = blockIdx.x / tiles % count, first = slice * width, C = a.g.classes - first < width ? a.g.classes - first : width;
    const int b = blockIdx.x / tiles / count, i0 = blockIdx.x % tiles * POS, inner = a.g.inner, n = inner - i0 < POS ? inner - i0 : POS;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = i0 + (lane < n ? lane : n - 1);
    const long p = (long)b * inner + i, positions = (long)a.g.outer * inner;
    const float w = position_weight(a, p), c = a.g.c;
    const bool any = __any(w != 0.f);  // (the same in every wave; else the notes are not written)
    const float F = any ? notes.F[p] : 0.f, R = any ? notes.R[p] : 0.f, m = any ? notes.m[p] : __builtin_nanf("");
    const bool mine = lane < n, far = m == m, any_far = __any(far);
    const typename T::E* z = (const typename T::E*)a.g.logits + b * a.g.ld + (long)first * inner + i;
    typename T::E* dz = (typename T::E*)a.d_logits + ((long)b * a.g.classes + first) * inner + i;
    const int c0 = C * wave / 4, c1 = C * (wave + 1) / 4;
    for (int j = c0; j < c1; j += U) {
        float x[U];
        if (any) {
#pragma unroll
            for (int u = 0; u < U; ++u) x[u] = T::up(z[(long)(j + u < c1 ? j + u : c1 - 1) * inner]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (mine && j + u < c1) {
                float d = any ? __builtin_fmaf(x[u], c, -R) : 0.f;
                if (any_far && far) d = (x[u] - m) * c;
                dz[(long)(j + u) * inner] = T::down(any && F != 0.f ? F * exp2_(d) : 0.f);
            }
    }
    if (!any) return;
    __syncthreads();
    for (int e = wave; e < a.k; e += 4) {
        const int cls = notes.cls[e * positions + p];
        const float g = notes.g[e * positions + p];
        if (mine && cls >= first && cls < first + C) dz[(long)(cls - first) * inner] = T::down(g);
    }
}

SliceNotes slice_notes(char* at, long positions, int k) {
    float* f = (float*)at;
    return {f, f + positions, f + 2 * positions, (int*)(f + 3 * positions), f + (3 + k) * positions};
}

}  // namespace

static MapSlices map_slices(int dtype, int classes, int whole, int slice) {
    const int bytes = POS * (dtype == MMAE_DT_F32 ? 4 : 2), most = slice / bytes;
    const int count = (long)classes * bytes <= whole ? 1 : (classes + most - 1) / most, width = (classes + count - 1) / count;
    return {(classes + width - 1) / width, width, nullptr, nullptr};
}
// Whole up to a tile of 80 KiB where slices cost more than they overlap: distillation, which reads them twice (109 x 300 x 64 x 64
// fp32: 431 us whole, 541 us sliced), and long lists of alternatives (64: 1878 and 3765 us; none: 192 and 127 us).  Short lists
// gain by more and smaller workgroups on a CU (8 alternatives, 131 x 1000 x 32 x 32: fp32 392 us with slices of 64 KiB, 314 us
// of 48, 360 us of 32; bf16 252 us of 64, 196 us of 48, 213 us of 32, but with 16 488, 410 and 327 us).
constexpr int WHOLE_BYTES = 80 * 1024;
MapSlices log_probs_map_slices(int dtype, int classes, int top_k) {
    if (top_k > 16) return map_slices(dtype, classes, WHOLE_BYTES, SLICE_BYTES);
    const int most = !top_k ? SLICE_BYTES : dtype == MMAE_DT_F32 ? 48 * 1024 : 32 * 1024;
    return map_slices(dtype, classes, most, most);
}
MapSlices distill_map_slices(int dtype, int classes) { return map_slices(dtype, classes, WHOLE_BYTES, SLICE_BYTES); }

size_t log_probs_slices_workspace(const MapSlices& s, int outer, int inner, int top_k) {
    return s.count == 1 ? 0 : (size_t)outer * inner * s.count * (sizeof(Sums) + sizeof(uint64_t) * (size_t)top_k);
}

constexpr int FEW_SLICES = 8;  // up to here a lane per position joins the lists, beyond a wave
int log_probs_slices(int dtype, const LogProbArgs& a, MapSlices s, void* workspace, hipStream_t stream) {
    s.sums = (Sums*)workspace;
    s.keys = (uint64_t*)(s.sums + (size_t)a.g.outer * a.g.inner * s.count);
    const int rc = log_probs_map(dtype, a, s, stream);
    if (rc != MMAE_OK || s.count == 1) return rc;
    const int tiles = map_tiles(a.g.inner);
    const long waves = ((long)a.g.outer * a.g.inner + 3) / 4;
    if (a.k && s.count > FEW_SLICES) {
        REQUIRE_GRID("class_log_probs", waves, 256);
#define CALL(T) hipLaunchKernelGGL(log_probs_map_merge_kernel<T>, dim3((unsigned)waves), dim3(256), 0, stream, a, s)
        BY_DTYPE(dtype, CALL);
#undef CALL
        return MMAE_OK;
    }
#define CALL(T) hipLaunchKernelGGL(log_probs_map_join_kernel<T>, dim3((unsigned)map_blocks(a.g)), dim3(64), a.k * POS * sizeof(uint64_t), stream, a, tiles, s)
    BY_DTYPE(dtype, CALL);
#undef CALL
    return MMAE_OK;
}

size_t distill_slices_workspace(const MapSlices& s, int outer, int inner, int k) {
    return s.count == 1 ? 0 : (size_t)outer * inner * (s.count * sizeof(Sums) + (3 + 2 * (size_t)k) * sizeof(float));
}

int distill_slices(int dtype, const DistillArgs& a, const MapSlices& s, void* workspace, bool again, hipStream_t stream) {
    const int tiles = map_tiles(a.g.inner);
    const long all = map_blocks(a.g), positions = (long)a.g.outer * a.g.inner;
    REQUIRE_GRID("distill", all * s.count, 256);
    Sums* sums = (Sums*)workspace;
    const SliceNotes notes = slice_notes((char*)(sums + positions * s.count), positions, a.k);
#define CALL(T)                                                                                                                          \
    do {                                                                                                                                 \
        if (!again) hipLaunchKernelGGL(distill_map_sums_kernel<T>, dim3((unsigned)(all * s.count)), dim3(256), 0, stream, a, tiles, s.count, s.width, sums); \
        hipLaunchKernelGGL(distill_map_join_kernel<T>, dim3((unsigned)all), dim3(64), 3 * a.k * POS * 4, stream, a, tiles, s.count, (const Sums*)sums, notes); \
        if (a.d_logits)                                                                                                                  \
            hipLaunchKernelGGL(distill_map_gradient_kernel<T>, dim3((unsigned)(all * s.count)), dim3(256), 0, stream, a, tiles, s.count, s.width, notes); \
    } while (0)
    BY_DTYPE(dtype, CALL);
#undef CALL
    return MMAE_OK;
}

}  // namespace classdist
