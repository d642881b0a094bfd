// adapter_api.cu -- C entry points of the low-rank adapter operators
// (declared in include/fpemu.h).
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <initializer_list>
#include <type_traits>

#include "adapter_few.cuh"
#include "adapter_tiles.cuh"
#include "fpemu_host.h"

using namespace fpemu;

namespace {

int element_size(int dtype) {
    switch (dtype) {
        case FPEMU_DT_F64: return 8;
        case FPEMU_DT_F32: return 4;
        case FPEMU_DT_F16: return 2;
        case FPEMU_DT_BF16: return 2;
        default: return 0;
    }
}

int check_sizes(const char* what, int dtype, int64_t rows, int64_t k, int64_t n, int64_t rank, int64_t adapters) {
    if (element_size(dtype) == 0) return fail(FPEMU_ERR_INVALID, "%s: unknown dtype code %d", what, dtype);
    if (rows < 0 || rows > FPEMU_ADAPTER_MAX_ROWS || k < 0 || n < 0)
        return fail(FPEMU_ERR_INVALID, "%s: bad sizes rows=%lld k=%lld n=%lld", what, (long long)rows, (long long)k,
                    (long long)n);
    if (k >= 1 << 30 || n >= 1 << 30)
        return fail(FPEMU_ERR_UNSUPPORTED, "%s: k=%lld n=%lld: below 2^30", what, (long long)k, (long long)n);
    if (rank < 1 || rank > FPEMU_ADAPTER_MAX_RANK)
        return fail(FPEMU_ERR_UNSUPPORTED, "%s: rank %lld outside [1, %d]", what, (long long)rank,
                    FPEMU_ADAPTER_MAX_RANK);
    if (adapters < 1 || adapters > FPEMU_ADAPTER_MAX_COUNT)
        return fail(FPEMU_ERR_UNSUPPORTED, "%s: %lld adapters outside [1, %d]", what, (long long)adapters,
                    FPEMU_ADAPTER_MAX_COUNT);
    return FPEMU_OK;
}

// Whether one of the addresses is no multiple of `size` (a power of two).
bool misplaced(int size, std::initializer_list<const void*> pointers) {
    uintptr_t all = 0;
    for (const void* p : pointers) all |= reinterpret_cast<uintptr_t>(p);
    return all % size != 0;
}

// Lets a kernel use `bytes` of dynamic shared memory, once per kernel and device.
template <auto* KERNEL>
int allow_shared(int bytes) {
    static std::atomic<uint64_t> done{0};
    int dev = 0;
    FPEMU_CUDA(cudaGetDevice(&dev));
    const uint64_t bit = 1ull << (dev & 63);
    if (!(done.load(std::memory_order_relaxed) & bit)) {
        FPEMU_CUDA(cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
        done.fetch_or(bit, std::memory_order_relaxed);
    }
    return FPEMU_OK;
}

template <typename T, int RP>
int launch_few_rank(const AdapterParams& P, const DevInfo& d, cudaStream_t st) {
    auto kern = adapter_few_kernel<T, RP>;
    using Tile = FewTile<T, RP>;
    if (Tile::kSmem > 48 * 1024) FPEMU_TRY((allow_shared<adapter_few_kernel<T, RP>>(Tile::kSmem)));
    // Groups of eight rows of one adapter, of none, or with a bad id: never more than this.
    const int64_t units = std::min<int64_t>(P.rows, P.rows / kGroupRows + P.adapters + 2);
    // The largest cluster with which all blocks are on the device at once (200 rows of 24 adapters,
    // 4096 x 4096 bfloat16, rank 16: 10.6 us with 4 blocks, 16.7 with 8 that are not; 250 rows with an
    // adapter each: 24.5 with 1, 29.5 with 2.  100 rows with one each, rank 64 and 128: 32 and 59 us so, 39
    // and 82 with twice and four times the blocks; float64 101 and 219, 113 and 251).
    int cluster = 8;
    while (cluster > 1 && units * cluster > d.sms * Tile::kBlocks) cluster /= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(units * cluster));
    cfg.blockDim = dim3(kFewThreads);
    cfg.dynamicSmemBytes = Tile::kSmem;
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = cluster;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    FPEMU_CUDA(cudaLaunchKernelEx(&cfg, kern, P));
    return FPEMU_OK;
}

template <typename T>
int launch_few(const AdapterParams& P, const DevInfo& d, cudaStream_t st) {
    if (P.r <= 16) return launch_few_rank<T, 16>(P, d, st);
    if (P.r <= 32) return launch_few_rank<T, 32>(P, d, st);
    if (P.r <= 64) return launch_few_rank<T, 64>(P, d, st);
    return launch_few_rank<T, 128>(P, d, st);
}

int padded_rank(int64_t r) { return r <= 16 ? 16 : r <= 32 ? 32 : r <= 64 ? 64 : 128; }

constexpr int kMostBlocks = 2;  // of a tile kernel on an SM

template <typename T>
constexpr CUtensorMapDataType map_type() {
    return sizeof(T) == 8 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT64
           : sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
           : std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
}

template <typename T>
bool map_ok(const void* p, int64_t stride) {
    return p != nullptr && reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride > 0 && stride * (int64_t)sizeof(T) % 16 == 0 &&
           stride < (int64_t(1) << 36);
}

// Rows of `length` elements in boxes of a slot's rows by 128 bytes.
template <typename T>
bool make_row_map(CUtensorMap* map, const void* p, int64_t stride, int64_t length, int64_t rows) {
    auto enc = tensor_map_encoder();
    if (enc == nullptr || !map_ok<T>(p, stride) || stride < length) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)length, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)stride * sizeof(T)};
    const cuuint32_t box[2] = {128 / (cuuint32_t)sizeof(T), kSlotRows}, step[2] = {1, 1};
    return enc(map, map_type<T>(), 2, const_cast<void*>(p), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// All adapters' weights as (inner, outer / turns, turns, adapter): element `turns` i + p of the outer
// dimension is (i, p), so that a box can hold them in the order of p.
template <typename T>
bool make_weight_map(CUtensorMap* map, const void* p, int64_t row, int64_t adapter, int64_t inner, int64_t outer,
                     int64_t adapters, int turns, int inner_box, int outer_box) {
    auto enc = tensor_map_encoder();
    if (adapters == 1) adapter = row;  // unused, but it has to be a stride
    if (enc == nullptr || !map_ok<T>(p, row) || !map_ok<T>(p, adapter) || outer % turns != 0) return false;
    const cuuint64_t e = sizeof(T);
    const cuuint64_t dims[4] = {(cuuint64_t)inner, (cuuint64_t)(outer / turns), (cuuint64_t)turns, (cuuint64_t)adapters};
    const cuuint64_t strides[3] = {(cuuint64_t)(turns * row) * e, (cuuint64_t)row * e, (cuuint64_t)adapter * e};
    const cuuint32_t box[4] = {(cuuint32_t)inner_box, (cuuint32_t)outer_box, (cuuint32_t)turns, 1}, step[4] = {1, 1, 1, 1};
    const int bytes = inner_box * (int)e;
    return enc(map, map_type<T>(), 4, const_cast<void*>(p), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
               bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : bytes == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, bool TR, int RP>
int launch_tiles_rank(AdapterParams& P, const DevInfo& d, cudaStream_t st) {
    using Tile = AdapterTile<T, TR, RP>;
    static_assert(Tile::kBlocks <= kMostBlocks, "the workspace holds a part of every block");
    auto shrink = adapter_shrink_kernel<T, TR, RP>;
    auto expand = adapter_expand_kernel<T, TR, RP>;
    FPEMU_TRY((allow_shared<adapter_shrink_kernel<T, TR, RP>>(Tile::kSmem)));
    FPEMU_TRY((allow_shared<adapter_expand_kernel<T, TR, RP>>(Tile::kSmem)));
    const int64_t slots = plan_slots(P.rows, P.adapters);
    auto grid = [&](int64_t length) {
        const int64_t chunks = std::max<int64_t>((length + Tile::KC - 1) / Tile::KC, 1);
        return (int)std::min<int64_t>((int64_t)d.sms * Tile::kBlocks, slots * chunks);
    };
    // Each product's rows and weights by TMA where they are aligned for it (few strides are not).
    CUtensorMap maps[4] = {};
    constexpr int inner = Tile::kInner / (int)sizeof(T);
    auto weights = [&](CUtensorMap* map, const void* w, int64_t row, int64_t adapter, int64_t length, bool by_long, int turns) {
        return by_long ? make_weight_map<T>(map, w, row, adapter, P.r, length, P.adapters, turns, inner, Tile::KC / turns)
                       : make_weight_map<T>(map, w, row, adapter, length, P.r, P.adapters, 1, Tile::KC, RP);
    };
    P.budget_ns = wait_budget_ns();
    P.stall = test_stall_idx();
    P.tma1 = P.tma2 = 0;
    if (P.k > 0 && make_row_map<T>(&maps[0], P.x, P.x_row, P.k, P.rows)) P.tma1 |= kTmaRows;
    if (P.k > 0 && weights(&maps[1], P.w1, P.w1_row, P.w1_adapter, P.k, TR, 1)) P.tma1 |= kTmaWeights;
    if (P.n > 0 && make_row_map<T>(&maps[2], P.base, P.base_row, P.n, P.rows)) P.tma2 |= kTmaRows;
    if (P.n > 0 && weights(&maps[3], P.w2, P.w2_row, P.w2_adapter, P.n, !TR, TR ? 1 : Tile::NT)) P.tma2 |= kTmaWeights;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(kTileThreads + kCopyThreads);
    cfg.dynamicSmemBytes = Tile::kSmem;
    cfg.stream = st;
    P.shrink_grid = grid(P.k);
    cfg.gridDim = dim3((unsigned)P.shrink_grid);
    if (P.k > 0) FPEMU_CUDA(cudaLaunchKernelEx(&cfg, shrink, P, maps[0], maps[1]));
    // The second kernel's blocks start as the first one's end, and wait for it before they read u.
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = P.k > 0 ? 1 : 0;
    cfg.gridDim = dim3((unsigned)grid(P.n));
    FPEMU_CUDA(cudaLaunchKernelEx(&cfg, expand, P, maps[2], maps[3]));
    return FPEMU_OK;
}

template <typename T, bool TR>
int launch_tiles(AdapterParams& P, const DevInfo& d, cudaStream_t st) {
    if (P.r <= 16) return launch_tiles_rank<T, TR, 16>(P, d, st);
    if (P.r <= 32) return launch_tiles_rank<T, TR, 32>(P, d, st);
    if (P.r <= 64) return launch_tiles_rank<T, TR, 64>(P, d, st);
    return launch_tiles_rank<T, TR, 128>(P, d, st);
}

template <typename T, int RP>
int launch_grad_rank(AdapterGradParams& P, size_t parts_bytes, const DevInfo& d, cudaStream_t st) {
    using Tile = AdapterGradTile<T, RP>;
    auto kern = adapter_grad_kernel<T, RP>;
    FPEMU_TRY((allow_shared<adapter_grad_kernel<T, RP>>(Tile::kSmem)));
    int64_t blocks[2];
    for (int i = 0; i < 2; ++i) blocks[i] = P.side[i].grad ? (P.side[i].cols + Tile::COLS - 1) / Tile::COLS : 0;
    if (blocks[0] + blocks[1] == 0) return FPEMU_OK;
    // Parts of an adapter's rows, by the average adapter (an uneven batch waits for its longest): as many as
    // make five blocks an SM (two to six fit, by type and rank; 16384 rows of 4 adapters, 4096 x 4096
    // bfloat16, rank 32, middle in two parts: 96 us in 512 blocks, 117 in 1024); twice that while a part
    // is long enough for its start not to count, since an SM's last blocks weigh less then (the same in
    // float64: 315 us in 1024 blocks, 377 in 512).
    const int64_t all = (blocks[0] + blocks[1]) * P.adapters, each = P.rows / P.adapters;
    int cluster = 1;
    while (cluster < kGradCluster && each > cluster * 4 * Tile::KT &&
           all * cluster * 2 <= d.sms * (each >= cluster * 128 * Tile::KT ? 10 : 5))
        cluster *= 2;
    // Segments of 8 chunks a block or more, as many as the device holds and the workspace has room for
    // (bfloat16, one adapter, middle in two parts, with the second kernel and without segments: 20000 rows,
    // 512 -> 512, rank 16, 22 us and 62; a million rows, 32 -> 32, rank 8, 118 and 2670; in three parts with
    // segments 25 and 163).
    int64_t segments = 1;
    if (cluster == kGradCluster && P.parts != nullptr)
        segments = std::max<int64_t>(1, std::min({d.sms * 5 / (all * cluster), each / (cluster * 8 * Tile::KT),
                                                  (int64_t)(parts_bytes / (grad_values(P, 2) * sizeof(typename Tile::Acc)))}));
    P.first_blocks = blocks[0] * cluster;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((blocks[0] + blocks[1]) * cluster), (unsigned)P.adapters, (unsigned)segments);
    cfg.blockDim = dim3(kGradThreads);
    cfg.dynamicSmemBytes = Tile::kSmem;
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = cluster;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    FPEMU_CUDA(cudaLaunchKernelEx(&cfg, kern, P));
    if (segments > 1) {
        const int64_t grid = std::min<int64_t>((grad_values(P, 2) + 255) / 256, d.sms * 8);
        adapter_grad_join_kernel<T><<<(unsigned)grid, 256, 0, st>>>(P, (int)segments);
        FPEMU_CUDA(cudaGetLastError());
    }
    return FPEMU_OK;
}

template <typename T>
int launch_grad(AdapterGradParams& P, size_t parts_bytes, const DevInfo& d, cudaStream_t st) {
    if (P.r <= 16) return launch_grad_rank<T, 16>(P, parts_bytes, d, st);
    if (P.r <= 32) return launch_grad_rank<T, 32>(P, parts_bytes, d, st);
    if (P.r <= 64) return launch_grad_rank<T, 64>(P, parts_bytes, d, st);
    return launch_grad_rank<T, 128>(P, parts_bytes, d, st);
}

size_t workspace_size(const DevInfo& d, int dtype, int64_t rows, int64_t rank, int64_t adapters) {
    // A part for every block of the first kernel and every slot, one of which begins or ends with each.
    return (size_t)(plan_slots(rows, adapters) + (int64_t)d.sms * kMostBlocks) * kSlotRows * padded_rank(rank) *
           (dtype == FPEMU_DT_F64 ? 8 : 4);
}

int check_workspace(const char* what, int dtype, int64_t rows, int64_t rank, int64_t adapters, const void* workspace,
                    size_t bytes) {
    DevInfo d;
    FPEMU_TRY(device_info(&d));
    const size_t need = workspace_size(d, dtype, rows, rank, adapters);
    if (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 16 != 0 || bytes < need)
        return fail(FPEMU_ERR_WORKSPACE, "%s: need %zu bytes of 16-byte aligned workspace, got %zu", what, need, bytes);
    return FPEMU_OK;
}

template <typename F>
int with_type(int dtype, F&& f) {
    switch (dtype) {
        case FPEMU_DT_F64: return f((double*)nullptr);
        case FPEMU_DT_F32: return f((float*)nullptr);
        case FPEMU_DT_F16: return f((__half*)nullptr);
        default: return f((__nv_bfloat16*)nullptr);
    }
}

}  // namespace

extern "C" {

int64_t fpemu_adapter_plan_size(int64_t rows, int64_t adapters) {
    if (rows < 0 || rows > FPEMU_ADAPTER_MAX_ROWS || adapters < 1 || adapters > FPEMU_ADAPTER_MAX_COUNT) return 0;
    return plan_words(rows, adapters) * 4;
}

int fpemu_adapter_plan(const void* index, int index_bytes, int64_t rows, int64_t adapters, void* plan,
                       size_t plan_bytes, void* stream) {
    DevInfo d;
    FPEMU_TRY(check_sizes("adapter_plan", FPEMU_DT_F64, rows, 0, 0, 1, adapters));
    if (index_bytes != 4 && index_bytes != 8)
        return fail(FPEMU_ERR_INVALID, "adapter_plan: index of %d-byte elements", index_bytes);
    if (plan == nullptr || plan_bytes < (size_t)plan_words(rows, adapters) * 4 ||
        reinterpret_cast<uintptr_t>(plan) % 16 != 0)
        return fail(FPEMU_ERR_WORKSPACE, "adapter_plan: need %lld bytes, 16-byte aligned",
                    (long long)plan_words(rows, adapters) * 4);
    if (rows > 0 && index == nullptr) return fail(FPEMU_ERR_INVALID, "adapter_plan: null index");
    if (misplaced(index_bytes, {index})) return fail(FPEMU_ERR_INVALID, "adapter_plan: misaligned index");
    FPEMU_TRY(device_info(&d));
    ErrorSink sink;
    FPEMU_TRY(error_sink(&sink));
    adapter_plan_kernel<<<(unsigned)(adapters + 2), 1024, 0, static_cast<cudaStream_t>(stream)>>>(
        index, index_bytes == 8, rows, (int)adapters, static_cast<int32_t*>(plan), sink);
    FPEMU_CUDA(cudaGetLastError());
    adapter_pack_kernel<<<1, 1024, 0, static_cast<cudaStream_t>(stream)>>>(rows, (int)adapters,
                                                                            static_cast<int32_t*>(plan));
    FPEMU_CUDA(cudaGetLastError());
    return FPEMU_OK;
}

size_t fpemu_adapter_workspace_size(int dtype, int64_t rows, int64_t rank, int64_t adapters) {
    DevInfo d;
    if (check_sizes("adapter_workspace_size", dtype, rows, 0, 0, rank, adapters) != FPEMU_OK || device_info(&d) != FPEMU_OK)
        return 0;
    return workspace_size(d, dtype, rows, rank, adapters);
}

int fpemu_adapter_matmul(int dtype, int64_t rows, int64_t k, int64_t n, int64_t rank, int64_t adapters,
                         const void* x, int64_t x_row, const void* A, int64_t A_adapter, int64_t A_row,
                         const void* B, int64_t B_adapter, int64_t B_row, const void* base, int64_t base_row, void* y,
                         int64_t y_row, const double* scales, double scale, const void* index, int index_bytes,
                         const void* plan, void* u, void* workspace, size_t workspace_bytes, void* stream) {
    DevInfo d;
    FPEMU_TRY(check_sizes("adapter_matmul", dtype, rows, k, n, rank, adapters));
    if (rows == 0) return FPEMU_OK;
    if ((k > 0 && (x == nullptr || A == nullptr)) || (n > 0 && (B == nullptr || y == nullptr)))
        return fail(FPEMU_ERR_INVALID, "adapter_matmul: null matrix pointer");
    if (x_row < 0 || base_row < 0 || A_adapter < 0 || B_adapter < 0 || A_row < 0 || B_row < 0 || (y_row < n && rows > 1))
        return fail(FPEMU_ERR_INVALID, "adapter_matmul: negative stride or output rows that overlap");
    if (plan == nullptr && (rows > FPEMU_ADAPTER_FEW_ROWS || index == nullptr || (index_bytes != 4 && index_bytes != 8)))
        return fail(FPEMU_ERR_INVALID, "adapter_matmul: %lld rows need a plan, few rows an index of 4 or 8 bytes",
                    (long long)rows);
    const int size = element_size(dtype);
    if (misplaced(size, {x, A, B, base, y}) || misplaced(8, {scales}) || misplaced(size == 8 ? 8 : 4, {u}) ||
        misplaced(16, {plan}) || (plan == nullptr && misplaced(index_bytes, {index})))
        return fail(FPEMU_ERR_INVALID, "adapter_matmul: a pointer is not aligned to its elements (the plan to 16 bytes)");
    FPEMU_TRY(device_info(&d));
    if (plan != nullptr) FPEMU_TRY(check_workspace("adapter_matmul", dtype, rows, rank, adapters, workspace, workspace_bytes));
    AdapterParams P = {};
    P.rows = rows, P.k = k, P.n = n, P.r = (int)rank, P.adapters = (int)adapters;
    P.x = x, P.x_row = x_row;
    P.w1 = A, P.w1_adapter = A_adapter, P.w1_row = A_row;
    P.w2 = B, P.w2_adapter = B_adapter, P.w2_row = B_row;
    P.base = base, P.base_row = base_row, P.y = y, P.y_row = y_row;
    P.scales = scales, P.scale = scale;
    P.index = index, P.index_wide = index_bytes == 8, P.plan = static_cast<const int32_t*>(plan);
    P.u = u, P.u_row = middle_row((int)rank), P.parts = workspace;
    FPEMU_TRY(error_sink(&P.sink));
    return with_type(dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        return P.plan ? launch_tiles<T, false>(P, d, st) : launch_few<T>(P, d, st);
    });
}

int fpemu_capture_id(void* stream, uint64_t* id) {
    if (id == nullptr) return fail(FPEMU_ERR_INVALID, "capture_id: id is null");
    cudaStreamCaptureStatus status;
    unsigned long long number = 0;
    FPEMU_CUDA(cudaStreamGetCaptureInfo(static_cast<cudaStream_t>(stream), &status, &number));
    *id = status == cudaStreamCaptureStatusNone ? 0 : number;
    return FPEMU_OK;
}

int fpemu_adapter_backward(int dtype, int64_t rows, int64_t k, int64_t n, int64_t rank, int64_t adapters,
                           const void* x, int64_t x_row, const void* A, int64_t A_adapter, int64_t A_row,
                           const void* B, int64_t B_adapter, int64_t B_row, const void* dy, int64_t dy_row,
                           const double* scales, double scale, const void* plan, const void* u, void* v, void* dx,
                           void* dA, void* dB, void* workspace, size_t workspace_bytes, void* stream) {
    DevInfo d;
    FPEMU_TRY(check_sizes("adapter_backward", dtype, rows, k, n, rank, adapters));
    if (plan == nullptr || (rows > 0 && ((k > 0 && dA && !x) || (n > 0 && !dy) || (k > 0 && dx && !A) ||
                                         (n > 0 && (dx || dA) && !B) || (dB && !u) || ((dx || dA) && !v))))
        return fail(FPEMU_ERR_INVALID, "adapter_backward: null pointer");
    if ((reinterpret_cast<uintptr_t>(u) | reinterpret_cast<uintptr_t>(v)) % 16 != 0)
        return fail(FPEMU_ERR_INVALID, "adapter_backward: u and v start on a 16-byte boundary");
    if (x_row < 0 || dy_row < 0 || A_adapter < 0 || B_adapter < 0 || A_row < 0 || B_row < 0)
        return fail(FPEMU_ERR_INVALID, "adapter_backward: negative stride");
    if (misplaced(element_size(dtype), {x, A, B, dy, dx, dA, dB}) || misplaced(8, {scales}) || misplaced(16, {plan}))
        return fail(FPEMU_ERR_INVALID, "adapter_backward: a pointer is not aligned to its elements (the plan to 16 bytes)");
    FPEMU_TRY(device_info(&d));
    if (dx || dA) FPEMU_TRY(check_workspace("adapter_backward", dtype, rows, rank, adapters, workspace, workspace_bytes));
    return with_type(dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        if (rows > 0 && (dx || dA)) {  // v = s dy B, dx = v A: the forward product with the factors' roles exchanged
            AdapterParams P = {};
            P.rows = rows, P.k = n, P.n = dx ? k : 0, P.r = (int)rank, P.adapters = (int)adapters;
            P.x = dy, P.x_row = dy_row;
            P.w1 = B, P.w1_adapter = B_adapter, P.w1_row = B_row;
            P.w2 = A, P.w2_adapter = A_adapter, P.w2_row = A_row;
            P.y = dx, P.y_row = k;
            P.scales = scales, P.scale = scale;
            P.plan = static_cast<const int32_t*>(plan);
            P.u = v, P.u_row = middle_row((int)rank), P.parts = workspace;
            FPEMU_TRY(error_sink(&P.sink));
            const int status = launch_tiles<T, true>(P, d, st);
            if (status != FPEMU_OK) return status;
        }
        AdapterGradParams G = {};
        G.rows = rows, G.r = (int)rank, G.p_row = middle_row((int)rank), G.adapters = (int)adapters;
        G.plan = static_cast<const int32_t*>(plan);
        G.side[0] = AdapterGradSide{v, x, x_row, k, dA, 0};
        G.side[1] = AdapterGradSide{u, dy, dy_row, n, dB, 1};
        if (dx || dA) G.parts = workspace;  // the products before have been through with it
        return launch_grad<T>(G, workspace_bytes, d, st);
    });
}

}  // extern "C"
