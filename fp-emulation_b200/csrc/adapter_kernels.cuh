// adapter_kernels.cuh -- low-rank adapters of many requests beside a shared
// projection: for every row t with adapter i = index[t],
//
//     u_t = s_i * A_i x_t        (r values)
//     y_t = base_t + B_i u_t
//
// and the sums of the backward pass over the rows of each adapter.
#pragma once

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <limits.h>
#include <stdint.h>

#include <type_traits>

#include "fpemu_error.cuh"

namespace fpemu {

namespace cg = cooperative_groups;

constexpr int kAdapterMaxRank = 128;
constexpr int kSlotRows = 64;      // rows of one adapter that a slot of the plan holds
constexpr int kFewRows = 256;      // up to here the forward kernel groups the rows itself

// Sums are held in float for 16- and 32-bit data and in double for float64.
template <typename T>
struct AccOf {
    using type = float;
};
template <>
struct AccOf<double> {
    using type = double;
};

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ double widen(double v) { return v; }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T narrow(typename AccOf<T>::type v);
template <>
__device__ __forceinline__ float narrow<float>(float v) { return v; }
template <>
__device__ __forceinline__ double narrow<double>(double v) { return v; }
template <>
__device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Two neighbours at a time (one conversion for 16-bit types).
__device__ __forceinline__ float2 widen2(const float* v) { return make_float2(v[0], v[1]); }
__device__ __forceinline__ double2 widen2(const double* v) { return make_double2(v[0], v[1]); }
__device__ __forceinline__ float2 widen2(const __half* v) { return __half22float2(*reinterpret_cast<const __half2*>(v)); }
__device__ __forceinline__ float2 widen2(const __nv_bfloat16* v) {
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(v));
}
__device__ __forceinline__ void narrow2(float* v, float a, float b) { v[0] = a, v[1] = b; }
__device__ __forceinline__ void narrow2(double* v, double a, double b) { v[0] = a, v[1] = b; }
__device__ __forceinline__ void narrow2(__half* v, float a, float b) {
    *reinterpret_cast<__half2*>(v) = __floats2half2_rn(a, b);
}
__device__ __forceinline__ void narrow2(__nv_bfloat16* v, float a, float b) {
    *reinterpret_cast<__nv_bfloat162*>(v) = __floats2bfloat162_rn(a, b);
}

// One slot of the plan: up to kSlotRows rows of one adapter (class `cls`:
// an adapter, `adapters` for rows without one, `adapters + 1` for bad ids).
struct AdapterSlot {
    int cls, start, count, unused;
};

// The plan: int32 words [0, adapters + 3) are the first position of each class
// in `perm` (classes in order; the last word is the number of rows); then
// (16-byte aligned) the classes' slots, in which a class begins at
// start/kSlotRows + class -- ranges of two classes never meet because
// ceil(c/S) <= (start + c)/S - start/S + 1 -- and some stay empty; then the slots
// that hold rows, those of adapters from the front and the others from the back,
// and how many there are of each; then perm, the rows sorted by class and in their
// own order within one.
__host__ __device__ __forceinline__ int64_t plan_slots(int64_t rows, int64_t adapters) {
    return rows / kSlotRows + adapters + 2;
}
__host__ __device__ __forceinline__ int64_t plan_slot_word(int64_t adapters) { return (adapters + 3 + 3) / 4 * 4; }
__host__ __device__ __forceinline__ int64_t plan_busy_word(int64_t rows, int64_t adapters) {
    return plan_slot_word(adapters) + 4 * plan_slots(rows, adapters);
}
__host__ __device__ __forceinline__ int64_t plan_header_word(int64_t rows, int64_t adapters) {
    return plan_busy_word(rows, adapters) + 4 * plan_slots(rows, adapters);
}
__host__ __device__ __forceinline__ int64_t plan_perm_word(int64_t rows, int64_t adapters) {
    return plan_header_word(rows, adapters) + 4;
}
__host__ __device__ __forceinline__ int64_t plan_words(int64_t rows, int64_t adapters) {
    return plan_perm_word(rows, adapters) + rows;
}

// Elements of a row of the middle (u and v): 16-byte units of 4 floats or 2 doubles.
__host__ __device__ __forceinline__ int middle_row(int r) { return (r + 3) / 4 * 4; }

__device__ __forceinline__ int row_class(const void* index, int wide, int64_t t, int adapters) {
    const int64_t id = wide ? static_cast<const int64_t*>(index)[t] : (int64_t) static_cast<const int32_t*>(index)[t];
    return id == -1 ? adapters : (id < 0 || id >= adapters) ? adapters + 1 : (int)id;
}

// One block per class.  Each warp counts the class's rows, and those of smaller
// classes, in its own stretch of the index; a scan over the warps' counts gives
// every warp its first position, and a second walk writes the rows in order.
// No atomics: the order is that of the rows.  Every block reads the whole index, which
// stays in the L2: rows x adapters, once for all layers (16384 rows of 64 adapters 7 us, of
// 1000 41 us, of 65000 2.4 ms; a million rows of 64 224 us).
__global__ void __launch_bounds__(1024) adapter_plan_kernel(const void* index, int wide, int64_t rows, int adapters,
                                                            int32_t* plan, ErrorSink sink) {
    __shared__ int own_count[32], below_count[32];
    const int cls = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t stretch = ((rows + 31) / 32 + 31) / 32 * 32;
    const int64_t t0 = warp * stretch, t1 = t0 + stretch < rows ? t0 + stretch : rows;
    constexpr int U = 8;  // ids a thread has in flight
    auto ids = [&](int64_t b, int (&c)[U]) {
        if (b + 32 * U <= t1) {  // all loads before the first use (a million rows: 222 us against 362; 16384: 6.5, 7.6)
            auto load = [&](const auto* p) {
                std::remove_cv_t<std::remove_pointer_t<decltype(p)>> v[U];
#pragma unroll
                for (int u = 0; u < U; ++u) v[u] = p[b + u * 32 + lane];
#pragma unroll
                for (int u = 0; u < U; ++u) c[u] = v[u] >= 0 && v[u] < adapters ? (int)v[u] : adapters + (v[u] != -1);
            };
            if (wide)
                load(static_cast<const int64_t*>(index));
            else
                load(static_cast<const int32_t*>(index));
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t t = b + u * 32 + lane;
                c[u] = t < t1 ? row_class(index, wide, t, adapters) : INT_MAX;
            }
        }
    };
    int own = 0, below = 0;
    for (int64_t b = t0; b < t1; b += 32 * U) {
        int c[U];
        ids(b, c);
#pragma unroll
        for (int u = 0; u < U; ++u) own += c[u] == cls, below += c[u] < cls;
    }
    own = __reduce_add_sync(0xffffffffu, own);
    below = __reduce_add_sync(0xffffffffu, below);
    if (lane == 0) own_count[warp] = own, below_count[warp] = below;
    __syncthreads();
    int start = 0, total = 0, at = 0;
    for (int w = 0; w < 32; ++w) {
        start += below_count[w];
        if (w == warp) at = total;
        total += own_count[w];
    }
    int32_t* perm = plan + plan_perm_word(rows, adapters);
    at += start;
    for (int64_t b = t0; b < t1; b += 32 * U) {
        int c[U];
        ids(b, c);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const unsigned m = __ballot_sync(0xffffffffu, c[u] == cls);
            if (c[u] == cls) perm[at + __popc(m & ((1u << lane) - 1))] = (int32_t)(b + u * 32 + lane);
            at += __popc(m);
        }
    }
    const int64_t s0 = start / kSlotRows + cls, s1 = (start + total) / kSlotRows + cls + 1;
    AdapterSlot* slots = reinterpret_cast<AdapterSlot*>(plan + plan_slot_word(adapters));
    for (int64_t s = s0 + threadIdx.x; s < s1; s += blockDim.x) {
        const int64_t first = (s - s0) * kSlotRows;
        const int64_t left = total - first;
        slots[s] = AdapterSlot{cls, (int)(start + first), (int)(left < 0 ? 0 : left < kSlotRows ? left : kSlotRows), 0};
    }
    __syncthreads();  // perm is written: the first bad row may be another warp's
    if (threadIdx.x == 0) {
        plan[cls] = start;
        if (cls == adapters + 1) {
            plan[adapters + 2] = (int32_t)rows;
            if (total > 0) report_error(sink.dev, sink.host, FPEMU_ERR_INVALID, kWhereAdapterIndex, perm[start]);
        }
    }
}

// The slots that hold rows, one block.
__global__ void __launch_bounds__(1024) adapter_pack_kernel(int64_t rows, int adapters, int32_t* plan) {
    __shared__ int counts[2][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t slots = plan_slots(rows, adapters);
    const AdapterSlot* from = reinterpret_cast<const AdapterSlot*>(plan + plan_slot_word(adapters));
    AdapterSlot* to = reinterpret_cast<AdapterSlot*>(plan + plan_busy_word(rows, adapters));
    int done[2] = {0, 0};  // adapters' slots, others
    for (int64_t first = 0; first < slots; first += 1024) {
        const int64_t i = first + threadIdx.x;
        const AdapterSlot s = i < slots ? from[i] : AdapterSlot{0, 0, 0, 0};
        const bool kind[2] = {s.count > 0 && s.cls < adapters, s.count > 0 && s.cls >= adapters};
        unsigned m[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            m[h] = __ballot_sync(0xffffffffu, kind[h]);
            if (lane == 0) counts[h][warp] = __popc(m[h]);
        }
        __syncthreads();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            int at = done[h] + __popc(m[h] & ((1u << lane) - 1));
            for (int w = 0; w < 32; ++w) {
                if (w < warp) at += counts[h][w];
                done[h] += counts[h][w];
            }
            if (kind[h]) to[h ? slots - 1 - at : at] = s;
        }
        __syncthreads();
    }
    if (threadIdx.x < 2) plan[plan_header_word(rows, adapters) + threadIdx.x] = done[threadIdx.x];
}

constexpr int kTmaRows = 1, kTmaWeights = 2;

struct AdapterParams {
    int64_t rows, k, n;
    int r, adapters;
    const void* x;      // [rows, k]
    int64_t x_row;
    const void* w1;     // forward A [adapters, r, k]; transposed B [adapters, k, r]
    int64_t w1_adapter, w1_row;
    const void* w2;     // forward B [adapters, n, r]; transposed A [adapters, r, n]
    int64_t w2_adapter, w2_row;
    const void* base;   // [rows, n] or null
    int64_t base_row;
    void* y;            // [rows, n]
    int64_t y_row;
    const double* scales;  // one per adapter, or null: `scale` for all
    double scale;
    const void* index;
    int index_wide;
    const int32_t* plan;  // null: the kernel groups the (few) rows itself
    void* u;              // [rows, u_row], kept for the gradients, or null
    int u_row;
    void* parts;          // with a plan: the first product's partial sums
    int shrink_grid;      // blocks that leave them
    uint64_t budget_ns;   // of a wait
    int stall;            // chunk at which the first block's copying warps stop (failure tests), or -1
    int tma1, tma2;       // which maps there are for the first and the second product
    ErrorSink sink;
};

__device__ __forceinline__ const AdapterSlot* plan_busy(const AdapterParams& P) {
    return reinterpret_cast<const AdapterSlot*>(P.plan + plan_busy_word(P.rows, P.adapters));
}
__device__ __forceinline__ const int32_t* plan_perm(const AdapterParams& P) {
    return P.plan + plan_perm_word(P.rows, P.adapters);
}

}  // namespace fpemu
