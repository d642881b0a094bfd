// clip_api.cu -- C entry points of the global gradient norm and clipping
// (declared in include/fpemu.h).
#include <cuda_runtime.h>

#include <algorithm>
#include <vector>

#include "clip_kernels.cuh"
#include "fpemu_host.h"

using namespace fpemu;

namespace {

constexpr int kSmallTable = 32, kLargeTable = 512;

int clip_grid(const DevInfo& d, int64_t chunks) { return (int)std::min<int64_t>(chunks, (int64_t)d.sms * 4); }

// Elements of a chunk: enough chunks for every block where there are elements enough.
int chunk_size(const DevInfo& d, int64_t count, const int64_t* numel) {
    int64_t all = 0;
    for (int64_t i = 0; i < count; ++i) all += numel[i];
    const int64_t even = all / ((int64_t)d.sms * 4);
    int size = kClipChunkMin;
    while (size < kClipChunkMax && size < even) size *= 2;
    return size;
}

constexpr int64_t kTypeSize[4] = {8, 4, 2, 2};  // by FPEMU_DT_ code

// The scaling kernel's blocks read and write in any order, so no output may meet
// another output, or an input that is not its own.
int clip_check_overlap(int64_t count, const void* const* src, void* const* dst, const int64_t* numel,
                       const int32_t* dtype) {
    struct Range {
        uintptr_t lo, hi;
        int64_t tensor;
        bool output;
    };
    try {
        std::vector<Range> r;
        r.reserve((size_t)count * 2);
        for (int64_t i = 0; i < count; ++i) {
            if (numel[i] == 0) continue;
            const uintptr_t s = reinterpret_cast<uintptr_t>(src[i]), o = reinterpret_cast<uintptr_t>(dst[i]);
            const uintptr_t bytes = (uintptr_t)(numel[i] * kTypeSize[dtype[i]]);
            r.push_back({o, o + bytes, i, true});
            if (s != o) r.push_back({s, s + bytes, i, false});
        }
        std::sort(r.begin(), r.end(), [](const Range& a, const Range& b) { return a.lo < b.lo; });
        // Furthest end so far of the outputs, and of everything: inputs may overlap each other.
        uintptr_t out_end = 0, any_end = 0;
        for (const Range& x : r) {
            if (x.lo < (x.output ? any_end : out_end))
                return fail(FPEMU_ERR_INVALID, "clip_grads: the output of a tensor overlaps another tensor (tensor %lld)",
                            (long long)x.tensor);
            any_end = std::max(any_end, x.hi);
            if (x.output) out_end = std::max(out_end, x.hi);
        }
    } catch (...) {
        return fail(FPEMU_ERR_INVALID, "clip_grads: out of host memory for %lld tensors", (long long)count);
    }
    return FPEMU_OK;
}

int clip_check(int64_t count, const void* const* src, void* const* dst, const int64_t* numel, const int32_t* dtype) {
    if (count < 0 || (count > 0 && (src == nullptr || numel == nullptr || dtype == nullptr)))
        return fail(FPEMU_ERR_INVALID, "clip_grads: bad tensor list");
    for (int64_t i = 0; i < count; ++i) {
        if (numel[i] < 0 || (numel[i] > 0 && (src[i] == nullptr || (dst != nullptr && dst[i] == nullptr))))
            return fail(FPEMU_ERR_INVALID, "clip_grads: tensor %lld has a null pointer or a negative size", (long long)i);
        if (dtype[i] < FPEMU_DT_F64 || dtype[i] > FPEMU_DT_BF16)
            return fail(FPEMU_ERR_INVALID, "clip_grads: tensor %lld has unknown dtype code %d", (long long)i, dtype[i]);
        const uintptr_t at = reinterpret_cast<uintptr_t>(src[i]) | (dst ? reinterpret_cast<uintptr_t>(dst[i]) : 0);
        if (numel[i] > 0 && at % kTypeSize[dtype[i]] != 0)
            return fail(FPEMU_ERR_INVALID, "clip_grads: tensor %lld is not aligned to its elements", (long long)i);
    }
    return dst == nullptr ? FPEMU_OK : clip_check_overlap(count, src, dst, numel, dtype);
}

// Fills the table with the next tensors that hold anything; returns where the list goes on.
template <int N>
int64_t fill(ClipTable<N>& t, int64_t from, int64_t count, const void* const* src, void* const* dst,
             const int64_t* numel, const int32_t* dtype, int size) {
    t.count = 0;
    t.chunk_size = size;
    int64_t chunk = 0;
    for (; from < count && t.count < N; ++from) {
        if (numel[from] == 0) continue;
        const int i = t.count++;
        t.src[i] = src[from];
        t.dst[i] = dst ? dst[from] : nullptr;
        t.numel[i] = numel[from];
        t.dtype[i] = (uint8_t)dtype[from];
        t.chunk[i] = chunk;
        chunk += (numel[from] + size - 1) / size;
    }
    t.chunk[t.count] = chunk;
    return from;
}

template <int N, int P>
int clip_run(const DevInfo& d, int64_t count, const void* const* src, void* const* dst, const int64_t* numel,
             const int32_t* dtype, double max_norm, void* norm, int norm_f64, double* partial, cudaStream_t st) {
    ClipTable<N> t;
    const int size = chunk_size(d, count, numel);
    int partials = 0;
    for (int64_t from = 0; from < count;) {
        from = fill(t, from, count, src, dst, numel, dtype, size);
        const int grid = clip_grid(d, t.chunk[t.count]);
        if (grid == 0) continue;
        norm_partial_kernel<N, P><<<grid, kClipThreads, 0, st>>>(t, partial + (int64_t)partials * kClipSums);
        FPEMU_CUDA(cudaGetLastError());
        partials += grid;
    }
    if (dst == nullptr || partials == 0) {
        norm_join_kernel<P><<<1, kClipThreads, 0, st>>>(partial, partials, norm, norm_f64);
        FPEMU_CUDA(cudaGetLastError());
        return FPEMU_OK;
    }
    for (int64_t from = 0; from < count;) {
        from = fill(t, from, count, src, dst, numel, dtype, size);
        const int grid = clip_grid(d, t.chunk[t.count]);
        if (grid == 0) continue;
        clip_scale_kernel<N, P><<<grid, kClipThreads, 0, st>>>(t, partial, partials, max_norm, norm, norm_f64);
        FPEMU_CUDA(cudaGetLastError());
        norm = nullptr;  // written by the first launch
    }
    return FPEMU_OK;
}

}  // namespace

extern "C" {

size_t fpemu_clip_workspace_size(int64_t count) {
    DevInfo d;
    if (count < 0 || device_info(&d) != FPEMU_OK) return 0;
    const int64_t launches = count / kLargeTable + 1;
    return (size_t)(launches * d.sms * 4 * kClipSums) * sizeof(double);
}

int fpemu_clip_grads(int64_t count, const void* const* src, void* const* dst, const int64_t* numel,
                     const int32_t* dtype, int norm_type, double max_norm, void* norm, int norm_f64, void* workspace,
                     size_t workspace_bytes, void* stream) {
    DevInfo d;
    FPEMU_TRY(clip_check(count, src, dst, numel, dtype));
    if (norm_type < 0 || norm_type > 2)
        return fail(FPEMU_ERR_INVALID, "clip_grads: norm_type %d (1, 2, or 0 for the largest magnitude)", norm_type);
    if (dst != nullptr && !(max_norm >= 0)) return fail(FPEMU_ERR_INVALID, "clip_grads: max_norm %g", max_norm);
    if (norm == nullptr || reinterpret_cast<uintptr_t>(norm) % (norm_f64 ? 8 : 4) != 0)
        return fail(FPEMU_ERR_INVALID, "clip_grads: null or misaligned norm");
    FPEMU_TRY(device_info(&d));
    if (workspace == nullptr || workspace_bytes < fpemu_clip_workspace_size(count) ||
        reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
        return fail(FPEMU_ERR_WORKSPACE, "clip_grads: need %zu bytes of 16-byte aligned workspace, got %zu",
                    fpemu_clip_workspace_size(count), workspace_bytes);
    double* partial = static_cast<double*>(workspace);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
#define FPEMU_CLIP(N, P) clip_run<N, P>(d, count, src, dst, numel, dtype, max_norm, norm, norm_f64, partial, st)
    if (count <= kSmallTable)
        return norm_type == 2 ? FPEMU_CLIP(kSmallTable, 2) : norm_type == 1 ? FPEMU_CLIP(kSmallTable, 1)
                                                                           : FPEMU_CLIP(kSmallTable, 0);
    return norm_type == 2 ? FPEMU_CLIP(kLargeTable, 2) : norm_type == 1 ? FPEMU_CLIP(kLargeTable, 1)
                                                                       : FPEMU_CLIP(kLargeTable, 0);
#undef FPEMU_CLIP
}

}  // extern "C"
