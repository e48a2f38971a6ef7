// Class distributions: entry points and the mask's counts.
#include "classdist.h"

#include <float.h>

namespace classdist {
namespace {

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

// Sizes that the launches take (the products below stay inside their types); a workspace is asked for before they are looked at.
constexpr int MOST_CLASSES = 1 << 30;
constexpr long MOST_POSITIONS = 0x7fffffc0L;
bool sizes_taken(int outer, int classes, int inner, int k) {
    return outer > 0 && classes > 0 && inner > 0 && classes <= MOST_CLASSES && (long)outer * inner <= MOST_POSITIONS && k >= 0 && k <= MAX_TOP;
}
int check_logits(const char* name, const void* logits, int dtype, int outer, int classes, int inner, long ld, float temperature) {
    MMAE_REQUIRE(logits, MMAE_EINVAL, "%s: null pointer", name);
    MMAE_REQUIRE(dtype >= MMAE_DT_F32 && dtype <= MMAE_DT_F16, MMAE_EINVAL, "%s: dtype code %d", name, dtype);
    MMAE_REQUIRE(outer > 0 && classes > 0 && inner > 0, MMAE_ESHAPE, "%s: empty input (%d x %d x %d)", name, outer, classes, inner);
    MMAE_REQUIRE(classes <= MOST_CLASSES, MMAE_ESHAPE, "%s: %d classes", name, classes);
    MMAE_REQUIRE((long)outer * inner <= MOST_POSITIONS, MMAE_ESHAPE, "%s: %d x %d positions are more than 2^31 - 64", name, outer, inner);
    MMAE_REQUIRE(ld >= (long)classes * inner, MMAE_ESHAPE, "%s: samples %ld elements apart hold %d x %d values", name, ld, classes, inner);
    MMAE_REQUIRE(temperature > 0.f && temperature < INFINITY && LOG2E / temperature < INFINITY, MMAE_EINVAL,
                 "%s: temperature %g is not positive and finite, with a finite reciprocal", name, temperature);
    return MMAE_OK;
}

}  // namespace
}  // namespace classdist

using namespace classdist;

extern "C" size_t mmae_class_log_probs_workspace_bytes(int dtype, int outer, int classes, int inner, int top_k) {
    if (!sizes_taken(outer, classes, inner, top_k)) return 0;
    return inner == 1 ? log_probs_rows_workspace(outer, classes, top_k) : log_probs_slices_workspace(log_probs_map_slices(dtype, classes, top_k), outer, inner, top_k);
}

extern "C" int mmae_class_log_probs(const void* logits, int dtype, int outer, int classes, int inner, long ld, const int64_t* target,
                                    int top_k, float temperature, float* log_prob, float* entropy, float* row_max,
                                    float* row_log_sum, float* top_log_prob, int64_t* top_class, void* workspace,
                                    size_t workspace_bytes, hipStream_t stream) {
    const int rc = check_logits("class_log_probs", logits, dtype, outer, classes, inner, ld, temperature);
    if (rc != MMAE_OK) return rc;
    MMAE_REQUIRE(target && log_prob && entropy && !row_max == !row_log_sum && (!top_k || (top_log_prob && top_class)), MMAE_EINVAL,
                 "class_log_probs: null pointer");
    MMAE_REQUIRE(top_k >= 0 && top_k <= MAX_TOP && top_k <= classes, MMAE_ESHAPE,
                 "class_log_probs: %d top classes of %d (at most %d)", top_k, classes, MAX_TOP);
    LogProbArgs a = {{logits, ld, outer, classes, inner, LOG2E / temperature, 1.f / temperature}, target, top_k, log_prob, entropy, row_max,
                     row_log_sum, top_log_prob, top_class};
    MMAE_REQUIRE(workspace_bytes >= mmae_class_log_probs_workspace_bytes(dtype, outer, classes, inner, top_k) && (workspace || !workspace_bytes),
                 MMAE_EWORKSPACE, "class_log_probs: workspace too small");
    const int r = inner == 1 ? log_probs_rows(dtype, a, workspace, stream) : log_probs_slices(dtype, a, log_probs_map_slices(dtype, classes, top_k), workspace, stream);
    if (r != MMAE_OK) return r;
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
    const int r = inner == 1 ? log_probs_bwd_rows(dtype, a, stream) : log_probs_bwd_map(dtype, a, stream);
    if (r != MMAE_OK) return r;
    MMAE_CHECK_LAUNCH("class_log_probs_bwd");
    return MMAE_OK;
}

// Parts of the loss that are added at the end: one per row, or per tile of a map.
static long distill_parts(int outer, int inner) { return inner == 1 ? outer : (long)outer * map_tiles(inner); }
static size_t distill_floats(int outer, long parts) { return (4 + (size_t)outer + (size_t)parts + 3) / 4 * 4; }

extern "C" size_t mmae_distill_workspace_bytes(int dtype, int outer, int classes, int inner, int k) {
    if (!sizes_taken(outer, classes, inner, k)) return 0;
    return sizeof(float) * distill_floats(outer, distill_parts(outer, inner)) +
           (inner == 1 ? distill_rows_workspace(outer, classes) : distill_slices_workspace(distill_map_slices(dtype, classes), outer, inner, k));
}

extern "C" int mmae_distill(const void* logits, int dtype, int outer, int classes, int inner, long ld, const void* top_class,
                            int class_bytes, const void* top_value, int value_dtype, int k, int kind, float temperature,
                            const int64_t* mask, int width, int patch, const float* upstream, int again, int skip_unit, float* loss,
                            void* d_logits, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    const int rc = check_logits("distill", logits, dtype, outer, classes, inner, ld, temperature);
    if (rc != MMAE_OK) return rc;
    MMAE_REQUIRE(top_class && top_value && workspace && (loss || d_logits), MMAE_EINVAL, "distill: null pointer");
    const double square = (double)temperature * temperature;  // (no position weighs less than one of all)
    MMAE_REQUIRE(square <= FLT_MAX && square / ((double)outer * inner) >= FLT_MIN, MMAE_EINVAL, "distill: the square of temperature %g, or its share of %d x %d positions, is not held in fp32",
                 temperature, outer, inner);
    MMAE_REQUIRE(class_bytes == 4 || class_bytes == 8, MMAE_EINVAL, "distill: classes of %d bytes", class_bytes);
    MMAE_REQUIRE(value_dtype >= MMAE_DT_F32 && value_dtype <= MMAE_DT_F16, MMAE_EINVAL, "distill: value dtype code %d", value_dtype);
    MMAE_REQUIRE(k >= 1 && k <= MAX_TOP, MMAE_ESHAPE, "distill: %d kept classes, between 1 and %d are taken", k, MAX_TOP);
    MMAE_REQUIRE(kind == 0 || kind == 1, MMAE_EINVAL, "distill: kind %d not in {0 (logits), 1 (log probabilities)}", kind);
    MMAE_REQUIRE(!mask || (width >= 1 && patch >= 1 && inner % width == 0 && width % patch == 0 && inner / width % patch == 0), MMAE_ESHAPE,
                 "distill: %d positions in rows of %d are not whole patches of %d", inner, width, patch);
    MMAE_REQUIRE(workspace_bytes >= mmae_distill_workspace_bytes(dtype, outer, classes, inner, k), MMAE_EWORKSPACE, "distill: workspace too small");
    MMAE_REQUIRE(!again || !loss, MMAE_EINVAL, "distill: the loss comes from the first call");
    REQUIRE_GRID("distill", outer, 64);  // (the count of masked positions)
    float* ws = (float*)workspace;
    DistillArgs a = {{logits, ld, outer, classes, inner, LOG2E / temperature, 1.f / temperature}, top_class, top_value, class_bytes, value_dtype, k, kind, mask};
    a.W = width; a.patch = mask ? patch : 1;
    a.tok_w = mask ? width / patch : 1;
    a.tokens = mask ? a.tok_w * (inner / width / patch) : 1;
    a.temperature = temperature;
    a.weight = (float)(square / ((double)outer * inner));
    a.valid = ws; a.count = ws + 4; a.part = loss ? ws + 4 + outer : nullptr;
    a.upstream = upstream; a.skip_unit = skip_unit; a.d_logits = d_logits;
    if (mask && !again) {
        if (a.tokens > 1) {
            hipLaunchKernelGGL(distill_count_kernel, dim3(outer), dim3(64), 0, stream, mask, outer, a.tokens, ws + 4);
            MMAE_CHECK_LAUNCH("distill_count");
        }
        hipLaunchKernelGGL(distill_valid_kernel, dim3(1), dim3(1024), 0, stream, ws + 4, a.tokens > 1 ? nullptr : mask, outer, ws);
        MMAE_CHECK_LAUNCH("distill_valid");
    }
    const long parts = distill_parts(outer, inner);
    void* room = ws + distill_floats(outer, parts);
    const MapSlices s = distill_map_slices(dtype, classes);
    const int r = inner == 1 ? distill_rows(dtype, a, room, again, stream)
                             : s.count == 1 ? distill_map(dtype, a, stream) : distill_slices(dtype, a, s, room, again, stream);
    if (r != MMAE_OK) return r;
    MMAE_CHECK_LAUNCH("distill");
    if (loss) {
        hipLaunchKernelGGL(distill_sum_kernel, dim3(1), dim3(1024), 0, stream, a.part, parts, loss);
        MMAE_CHECK_LAUNCH("distill_sum");
    }
    return MMAE_OK;
}
