// clip_kernels.cuh -- the global norm over many tensors and their scaling.
//
//     N = (sum |g|^p)^(1/p) over every element of every tensor, p = 1, 2 or inf
//     c = min(1, max_norm / (N + 1e-6)),  g' = c * g
//
// One kernel leaves a partial sum per block, a second one joins them (every
// block the same sums in the same order) and scales.  Every element enters the
// sums as a double; the blocks and their order depend on the sizes alone, so
// results repeat.
//
// Bound by the bytes: the norm reads every element once, the scaling reads and
// writes it (what the norm read last from the L2).  Measured, 285 M bfloat16 values
// in 38 tensors: norm 110 us, 5.2 TB/s (doubles made from the bits instead of by
// conversions, 16 a clock and SM: no faster); scaling 181 us, 6.3 TB/s.  219 MB of mixed types in bounds: 41 us
// for the norm, and 5 us to see that nothing is to be scaled.  Eight small tensors:
// 3 us each, of a call that takes 25-40 on the host.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "fpemu_internal.h"

namespace fpemu {

constexpr int kClipThreads = 256;
constexpr int kClipChunkMin = 1024;    // elements of one tensor that a block takes at a time,
constexpr int kClipChunkMax = 16384;   // by how many there are for every block
constexpr int kClipSums = 3;           // doubles a block leaves (see NormSum)

// Up to N tensors, passed in the launch's parameters: no copy of a pointer table.
template <int N>
struct ClipTable {
    const void* src[N];
    void* dst[N];
    int64_t numel[N];
    int64_t chunk[N + 1];  // first chunk of each tensor, then their number
    uint8_t dtype[N];
    int count;
    int chunk_size;
};

// p = 2: squares of doubles leave the range long before their norm does, so
// values above 2^490 are summed scaled by 2^-600 and values below 2^-490
// scaled by 2^600, apart from the others (2^40 squares of 2^490 stay finite).
// p = 1 and inf use the first sum alone.
struct NormSum {
    double mid = 0, big = 0, small = 0;

    template <int P>
    __device__ __forceinline__ void add_wide(double v) {
        const double a = fabs(v);
        if (P == 2) {
            if (a > 0x1p490) big = fma(a * 0x1p-600, a * 0x1p-600, big);
            else if (a < 0x1p-490) small = fma(a * 0x1p600, a * 0x1p600, small);
            else mid = fma(a, a, mid);  // NaN too
        } else if (P == 1) {
            mid += a;
        } else {
            mid = (a > mid || isnan(a)) ? a : mid;  // a NaN stays
        }
    }
    // Floats, halves and bfloat16: their squares are well inside the range of doubles.
    template <int P>
    __device__ __forceinline__ void add(float v) {
        const double a = (double)fabsf(v);
        if (P == 2) mid = fma(a, a, mid);
        else if (P == 1) mid += a;
        else mid = (a > mid || isnan(a)) ? a : mid;
    }
    template <int P>
    __device__ __forceinline__ void add(double v) { add_wide<P>(v); }
    template <int P>
    __device__ __forceinline__ void join(double m, double b, double s) {
        if (P == 0) mid = (m > mid || isnan(m)) ? m : mid;
        else mid += m, big += b, small += s;
    }
    template <int P>
    __device__ __forceinline__ double norm() const {
        if (P != 2) return mid;
        if (isnan(mid) || isnan(big)) return mid + big;
        if (big > 0) return sqrt(big + mid * 0x1p-600 * 0x1p-600) * 0x1p600;
        if (mid > 0) return sqrt(mid + small * 0x1p-600 * 0x1p-600);
        return sqrt(small) * 0x1p-600;
    }
};

__device__ __forceinline__ float clip_widen(float v) { return v; }
__device__ __forceinline__ double clip_widen(double v) { return v; }
__device__ __forceinline__ float clip_widen(__half v) { return __half2float(v); }
__device__ __forceinline__ float clip_widen(__nv_bfloat16 v) { return __bfloat162float(v); }

// The factor as one double, and as two floats whose sum it is: but for 2^-48 of it, as long as it is
// above 2^-100.  TINY: below that a float loses digits and then all of them, and the product is one
// of doubles.
struct ClipFactor {
    double c;
    float hi, lo;
};
template <bool TINY>
__device__ __forceinline__ double clip_scale(double v, const ClipFactor& f) { return v * f.c; }
// The product with the float pair rounds once (but for 2^-48), as the product with the double would.
template <bool TINY>
__device__ __forceinline__ float clip_scale(float v, const ClipFactor& f) {
    return TINY ? (float)((double)v * f.c) : fmaf(v, f.hi, v * f.lo);
}
template <bool TINY>
__device__ __forceinline__ __half clip_scale(__half v, const ClipFactor& f) {
    return TINY ? __double2half((double)__half2float(v) * f.c) : __float2half_rn(__half2float(v) * f.hi);
}
template <bool TINY>
__device__ __forceinline__ __nv_bfloat16 clip_scale(__nv_bfloat16 v, const ClipFactor& f) {
    return TINY ? __double2bfloat16((double)__bfloat162float(v) * f.c) : __float2bfloat16_rn(__bfloat162float(v) * f.hi);
}

// Block-wide join of the threads' sums, in a fixed order; thread 0 has the result.
template <int P>
__device__ NormSum block_join(NormSum v) {
    __shared__ double part[kClipThreads / 32][kClipSums];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const double m = __shfl_xor_sync(0xffffffffu, v.mid, o);
        const double b = __shfl_xor_sync(0xffffffffu, v.big, o), s = __shfl_xor_sync(0xffffffffu, v.small, o);
        v.join<P>(m, b, s);
    }
    __syncthreads();
    if (lane == 0) part[warp][0] = v.mid, part[warp][1] = v.big, part[warp][2] = v.small;
    __syncthreads();
    NormSum t;
    for (int w = 0; w < kClipThreads / 32; ++w) t.join<P>(part[w][0], part[w][1], part[w][2]);
    return t;
}

// Elements of type T before the first 16-byte boundary.
template <typename T>
__device__ __forceinline__ int clip_head(const void* p, int n) {
    const int h = ((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / sizeof(T);
    return h < n ? h : n;
}

template <typename T, int P>
__device__ __forceinline__ void add_vector(const uint4& raw, NormSum (&s)[2]) {
    const T* v = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int e = 0; e < (int)(16 / sizeof(T)); ++e) s[e & 1].template add<P>(clip_widen(v[e]));
}

template <typename T, int P>
__device__ void chunk_norm(const T* p, int n, NormSum& sum) {
    constexpr int V = 16 / sizeof(T), U = 4;
    const int head = clip_head<T>(p, n), vecs = (n - head) / V;
    NormSum s[2];
    const uint4* q = reinterpret_cast<const uint4*>(p + head);
    int i = threadIdx.x;
    for (; i + (U - 1) * kClipThreads < vecs; i += U * kClipThreads) {
        uint4 raw[U];
#pragma unroll
        for (int u = 0; u < U; ++u) raw[u] = q[i + u * kClipThreads];
#pragma unroll
        for (int u = 0; u < U; ++u) add_vector<T, P>(raw[u], s);
    }
    for (; i < vecs; i += kClipThreads) add_vector<T, P>(q[i], s);
    if (threadIdx.x < head) s[0].template add<P>(clip_widen(p[threadIdx.x]));
    const int t = head + vecs * V + threadIdx.x;
    if (t < n) s[0].template add<P>(clip_widen(p[t]));
    sum.join<P>(s[0].mid, s[0].big, s[0].small);
    sum.join<P>(s[1].mid, s[1].big, s[1].small);
}

template <bool TINY, typename T>
__device__ void chunk_scale(const T* p, T* o, int n, const ClipFactor& f) {
    constexpr int V = 16 / sizeof(T), U = 4;
    const bool same = ((reinterpret_cast<uintptr_t>(p) ^ reinterpret_cast<uintptr_t>(o)) & 15) == 0;
    const int head = same ? clip_head<T>(p, n) : 0, vecs = same ? (n - head) / V : 0;
    const uint4* q = reinterpret_cast<const uint4*>(p + head);
    uint4* w = reinterpret_cast<uint4*>(o + head);
    auto scaled = [&](uint4 raw) {
        T* v = reinterpret_cast<T*>(&raw);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = clip_scale<TINY>(v[e], f);
        return raw;
    };
    int i = threadIdx.x;
    for (; i + (U - 1) * kClipThreads < vecs; i += U * kClipThreads) {
        uint4 raw[U];
#pragma unroll
        for (int u = 0; u < U; ++u) raw[u] = __ldcs(q + i + u * kClipThreads);
#pragma unroll
        for (int u = 0; u < U; ++u) __stcs(w + i + u * kClipThreads, scaled(raw[u]));
    }
    for (; i < vecs; i += kClipThreads) __stcs(w + i, scaled(__ldcs(q + i)));
    if (threadIdx.x < head) o[threadIdx.x] = clip_scale<TINY>(p[threadIdx.x], f);
    for (int t = head + vecs * V + threadIdx.x; t < n; t += kClipThreads) o[t] = clip_scale<TINY>(p[t], f);
}

// Calls f(tensor, first element, elements) for this block's share of the chunks,
// first to last or, BACK, last to first: what the norm's pass read last is still in
// the L2 when the scaling begins with it.
template <bool BACK, int N, typename F>
__device__ __forceinline__ void for_chunks(const ClipTable<N>& t, F&& f) {
    const int64_t chunks = t.chunk[t.count];
    const int64_t begin = chunks * blockIdx.x / gridDim.x, end = chunks * (blockIdx.x + 1) / gridDim.x;
    const int64_t from = BACK ? end - 1 : begin;
    int i = 0, hi = t.count - 1;
    while (i < hi) {
        const int mid = (i + hi + 1) / 2;
        if (t.chunk[mid] <= from) i = mid;
        else hi = mid - 1;
    }
    for (int64_t n = 0; n < end - begin; ++n) {
        const int64_t c = BACK ? end - 1 - n : begin + n;
        if (BACK) while (c < t.chunk[i]) --i;
        else while (c >= t.chunk[i + 1]) ++i;
        const int64_t at = (c - t.chunk[i]) * t.chunk_size, left = t.numel[i] - at;
        f(i, at, (int)(left < t.chunk_size ? left : t.chunk_size));
    }
}

template <int N, int P>
__global__ void __launch_bounds__(kClipThreads) norm_partial_kernel(const __grid_constant__ ClipTable<N> t,
                                                                    double* partial) {
    NormSum sum;
    for_chunks<false>(t, [&](int i, int64_t at, int n) {
        const void* p = t.src[i];
        switch (t.dtype[i]) {
            case FPEMU_DT_F64:
                chunk_norm<double, P>(static_cast<const double*>(p) + at, n, sum);
                break;
            case FPEMU_DT_F32: chunk_norm<float, P>(static_cast<const float*>(p) + at, n, sum); break;
            case FPEMU_DT_F16: chunk_norm<__half, P>(static_cast<const __half*>(p) + at, n, sum); break;
            default: chunk_norm<__nv_bfloat16, P>(static_cast<const __nv_bfloat16*>(p) + at, n, sum);
        }
    });
    sum = block_join<P>(sum);
    if (threadIdx.x == 0) {
        double* o = partial + (int64_t)blockIdx.x * kClipSums;
        o[0] = sum.mid, o[1] = sum.big, o[2] = sum.small;
    }
}

template <int P>
__device__ double joined_norm(const double* partial, int partials) {
    NormSum sum;
    for (int i = threadIdx.x; i < partials; i += kClipThreads)
        sum.join<P>(partial[i * kClipSums], partial[i * kClipSums + 1], partial[i * kClipSums + 2]);
    return block_join<P>(sum).template norm<P>();
}

__device__ __forceinline__ void store_norm(double norm, void* out, int out_f64) {
    if (out_f64) *static_cast<double*>(out) = norm;
    else *static_cast<float*>(out) = (float)norm;
}

template <int P>
__global__ void __launch_bounds__(kClipThreads) norm_join_kernel(const double* partial, int partials, void* out,
                                                                 int out_f64) {
    const double norm = joined_norm<P>(partial, partials);
    if (threadIdx.x == 0) store_norm(norm, out, out_f64);
}

// A tensor scaled in place by exactly 1 is left alone: the product would be itself.
template <int N, int P>
__global__ void __launch_bounds__(kClipThreads) clip_scale_kernel(const __grid_constant__ ClipTable<N> t,
                                                                  const double* partial, int partials,
                                                                  double max_norm, void* out, int out_f64) {
    const double norm = joined_norm<P>(partial, partials);
    if (out != nullptr && blockIdx.x == 0 && threadIdx.x == 0) store_norm(norm, out, out_f64);
    ClipFactor f;
    const double c = max_norm / (norm + 1e-6);
    f.c = c > 1.0 ? 1.0 : c;  // NaN stays
    f.hi = (float)f.c;
    f.lo = (float)(f.c - (double)f.hi);
    const bool tiny = f.c < 0x1p-100 && f.c > 0;
    for_chunks<true>(t, [&](int i, int64_t at, int n) {
        if (t.src[i] == t.dst[i] && f.c == 1.0) return;
        auto scale = [&](auto type) {
            using T = decltype(type);
            const T* p = static_cast<const T*>(t.src[i]) + at;
            T* o = static_cast<T*>(t.dst[i]) + at;
            if (tiny && sizeof(T) < 8) chunk_scale<true>(p, o, n, f);
            else chunk_scale<false>(p, o, n, f);
        };
        switch (t.dtype[i]) {
            case FPEMU_DT_F64: scale(double()); break;
            case FPEMU_DT_F32: scale(float()); break;
            case FPEMU_DT_F16: scale(__half()); break;
            default: scale(__nv_bfloat16());
        }
    });
}

}  // namespace fpemu
