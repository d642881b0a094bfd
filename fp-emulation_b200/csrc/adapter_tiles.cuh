// adapter_tiles.cuh -- the adapter products of long batches on the tensor cores.
//
// A cluster of blocks takes one slot of the plan, up to 64 rows of one adapter.
// The blocks share the length k of the first product and the columns n of the
// second one; every element of x, base and y passes through one block, once.
// The chunks of both products (64 rows by 128 bytes of x and W1, then of base
// and W2) go through one ring of asynchronous copies, so the second product's
// first chunks arrive while the blocks exchange the rank-long middle.
//
// What a chunk costs: the rank is small, so both products are bound by the
// bytes of x, base and y for float64 up to rank 16 and for 16-bit data up to
// rank 64; mma.sync reaches 37 TFLOP/s for f64 (the device's whole rate), 545
// for 16-bit and 273 for tf32 data, which is enough there.
#pragma once

#include "adapter_kernels.cuh"

namespace fpemu {

constexpr int kTileThreads = 128;  // four warps of 16 rows

__device__ __forceinline__ uint32_t shared_address(const void* p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// 16 bytes of a tile: `avail` elements from src, zeros after them.
template <typename T>
__device__ __forceinline__ void fetch16(uint8_t* dst, const T* src, const T* safe, int avail, bool vec) {
    constexpr int V = 16 / sizeof(T);
    if (vec) {
        copy16(shared_address(dst), avail > 0 ? src : safe, avail * (int)sizeof(T));
    } else {
        alignas(16) T v[V];
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = i < avail ? src[i] : T(0.0f);
        *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<uint4*>(v);
    }
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}

template <typename T>
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                     "{%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                     "{%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f64(double (&c)[4], double a0, double a1, double b) {
    asm volatile("mma.sync.aligned.m16n8k4.row.col.f64.f64.f64.f64 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};"
                 : "+d"(c[0]), "+d"(c[1]), "+d"(c[2]), "+d"(c[3]) : "d"(a0), "d"(a1), "d"(b));
}

// A float as two tf32 parts: hi is x rounded to 10 bits after the point, lo the
// first bits of the rest.  A product of two floats takes three of the four partial
// products; what it loses is 2^-20 of it at most.  An infinite or NaN x is in lo,
// with a finite hi, so that a zero lo of the other factor meets no infinity.
struct Tf32Pair {
    uint32_t hi, lo;
};
__device__ __forceinline__ Tf32Pair tf32_split(float x) {
    const float top = __uint_as_float(0x7f7fe000u);  // the largest tf32 value
    Tf32Pair p;
    p.hi = (__float_as_uint(fmaxf(fminf(x, top), -top)) + 0x1000u) & 0xffffe000u;
    p.lo = __float_as_uint(x - __uint_as_float(p.hi)) & 0xffffe000u;
    return p;
}

// The same for two neighbouring values as pairs of 16-bit parts (16 bits of bfloat16, 22 of halves).
template <typename T>
__device__ __forceinline__ void split16(float x, float y, uint32_t& hi, uint32_t& lo) {
    if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(x, y);
        const float2 f = __half22float2(h);
        const __half2 l = __floats2half2_rn(fminf(x - f.x, 65504.f), fminf(y - f.y, 65504.f));
        hi = *reinterpret_cast<const uint32_t*>(&h);
        lo = *reinterpret_cast<const uint32_t*>(&l);
    } else {  // cut, not rounded: a finite value stays finite
        const uint32_t a = __float_as_uint(x) & 0xffff0000u, b = __float_as_uint(y) & 0xffff0000u;
        const __nv_bfloat162 l = __floats2bfloat162_rn(fminf(x - __uint_as_float(a), 1e38f),
                                                       fminf(y - __uint_as_float(b), 1e38f));
        hi = (a >> 16) | b;
        lo = *reinterpret_cast<const uint32_t*>(&l);
    }
}

// Tiles in shared memory.  "Rank-major" weights have a row for each rank and
// 128 bytes along the long dimension, "long-major" ones a row for each of its
// elements and the rank along it.  The pitches keep the warps' fragment loads
// free of bank conflicts: odd numbers of 16-byte units for ldmatrix; 4 (mod 16)
// 8-byte units for f64; for f32, 4 or 8 (mod 32) words as the fragment runs
// along the row or across rows.
template <typename T, bool TR, int RP>
struct AdapterTile {
    using Acc = typename AccOf<T>::type;
    static constexpr int E = sizeof(T), V = 16 / E;
    static constexpr int KC = 128 / E;
    static constexpr int kPitchX = E == 8 ? 160 : 144;
    static constexpr int kPitchRank = E == 8 || (E == 4 && TR) ? 160 : 144;
    static constexpr int kPitchLong = E == 8 ? (RP + 4) * 8 : E == 4 ? (RP + (TR ? 8 : 4)) * 4 : RP * 2 + 16;
    static constexpr int kRankBytes = RP * kPitchRank, kLongBytes = KC * kPitchLong;
    static constexpr int kStageX = kSlotRows * kPitchX;
    static constexpr int kStage = kStageX + (kRankBytes > kLongBytes ? kRankBytes : kLongBytes);
    static constexpr int kStages = RP <= 32 ? 4 : 3;
    static constexpr int kPitchU = E == 2 ? RP + 8 : RP + 4;  // elements of Acc
    static constexpr int kSmem = kStages * kStage + kSlotRows * kPitchU * (int)sizeof(Acc);
};

// Rows without an adapter or with a bad id, this block's share of the columns.
template <typename T>
__device__ void plain_rows(const AdapterParams& P, const int* list, int count, bool bad, int64_t n0, int64_t n1) {
    constexpr int V = 16 / sizeof(T);
    if (!bad && P.base == P.y && P.base_row == P.y_row) return;
    const T* base = static_cast<const T*>(P.base);
    T* y = static_cast<T*>(P.y);
    const bool vec = !bad && ((reinterpret_cast<uintptr_t>(base) | reinterpret_cast<uintptr_t>(y)) & 15) == 0 &&
                     (P.base_row * sizeof(T)) % 16 == 0 && (P.y_row * sizeof(T)) % 16 == 0;
    for (int i = 0; i < count; ++i) {
        const int64_t row = list[i];
        int64_t c = n0;
        if (vec) {
            const int64_t vecs = (n1 - n0) / V;
            for (int64_t v = threadIdx.x; v < vecs; v += blockDim.x)
                *reinterpret_cast<uint4*>(y + row * P.y_row + n0 + v * V) =
                    base ? *reinterpret_cast<const uint4*>(base + row * P.base_row + n0 + v * V) : uint4{0, 0, 0, 0};
            c += vecs * V;
        }
        if (c < n1) plain_row<T>(P, row, bad, c, n1);
    }
}

template <typename T, bool TR, int RP>
__global__ void __launch_bounds__(kTileThreads) adapter_tile_kernel(AdapterParams P) {
    using Tile = AdapterTile<T, TR, RP>;
    using Acc = typename Tile::Acc;
    constexpr int E = Tile::E, V = Tile::V, KC = Tile::KC, S = Tile::kStages;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ int list[kSlotRows];
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, q = lane & 3;
    const int cr = (int)cluster.block_rank(), cs = (int)cluster.num_blocks();
    const AdapterSlot slot =
        reinterpret_cast<const AdapterSlot*>(P.plan + plan_slot_word(P.adapters))[blockIdx.x / cs];
    const int count = slot.count;
    if (count == 0) return;
    if (tid < kSlotRows)
        list[tid] = (P.plan + plan_perm_word(P.rows, P.adapters))[slot.start + (tid < count ? tid : 0)];
    __syncthreads();
    const int64_t kshare = (P.k + (int64_t)KC * cs - 1) / ((int64_t)KC * cs) * KC;
    const int64_t nshare = (P.n + (int64_t)KC * cs - 1) / ((int64_t)KC * cs) * KC;
    const int64_t k0 = cr * kshare < P.k ? cr * kshare : P.k, k1 = k0 + kshare < P.k ? k0 + kshare : P.k;
    const int64_t n0 = cr * nshare < P.n ? cr * nshare : P.n, n1 = n0 + nshare < P.n ? n0 + nshare : P.n;
    if (slot.cls >= P.adapters) {
        plain_rows<T>(P, list, count, slot.cls != P.adapters, n0, n1);
        return;
    }
    const int nk = (int)((k1 - k0 + KC - 1) / KC), total = nk + (int)((n1 - n0 + KC - 1) / KC);
    const T* w1 = static_cast<const T*>(P.w1) + slot.cls * P.w1_adapter;
    const T* w2 = static_cast<const T*>(P.w2) + slot.cls * P.w2_adapter;
    const T* x = static_cast<const T*>(P.x);
    const T* base = static_cast<const T*>(P.base);
    T* y = static_cast<T*>(P.y);
    auto aligned = [](const void* p, int64_t stride) {
        return ((reinterpret_cast<uintptr_t>(p) | (uintptr_t)(stride * E)) & 15) == 0;
    };
    const bool vec_x = aligned(x, P.x_row), vec_w1 = aligned(w1, P.w1_row), vec_w2 = aligned(w2, P.w2_row);
    const bool vec_base = aligned(base, P.base_row), vec_y = aligned(y, P.y_row);

    auto clamp = [](int64_t v) { return v < 0 ? 0 : v > V ? V : (int)v; };
    auto fetch_rows = [&](uint8_t* st, const T* src, int64_t stride, int64_t c0, int64_t c1, bool vec) {
#pragma unroll
        for (int i = 0; i < kSlotRows / 16; ++i) {
            const int row = tid / 8 + 16 * i;
            const int64_t c = c0 + (tid % 8) * V;
            fetch16(st + row * Tile::kPitchX + (tid % 8) * 16, src + list[row] * stride + c, src,
                    row < count ? clamp(c1 - c) : 0, vec);
        }
    };
    auto fetch_rank = [&](uint8_t* st, const T* w, int64_t stride, int64_t c0, int64_t c1, bool vec) {
#pragma unroll
        for (int i = 0; i < RP * 8 / kTileThreads; ++i) {
            const int j = tid / 8 + 16 * i;
            const int64_t c = c0 + (tid % 8) * V;
            fetch16(st + j * Tile::kPitchRank + (tid % 8) * 16, w + j * stride + c, w, j < P.r ? clamp(c1 - c) : 0, vec);
        }
    };
    auto fetch_long = [&](uint8_t* st, const T* w, int64_t stride, int64_t c0, int64_t c1, bool vec) {
        constexpr int per = RP * E / 16;
#pragma unroll
        for (int i = 0; i < (KC * per + kTileThreads - 1) / kTileThreads; ++i) {
            const int idx = tid + i * kTileThreads, l = idx / per, j = idx % per * V;
            if (KC * per % kTileThreads == 0 || idx < KC * per)
                fetch16(st + l * Tile::kPitchLong + j * E, w + (c0 + l) * stride + j, w,
                        c0 + l < c1 ? clamp(P.r - j) : 0, vec);
        }
    };
    auto fetch = [&](int c) {
        uint8_t* st = smem + c % S * Tile::kStage;
        if (c < nk) {
            const int64_t c0 = k0 + (int64_t)c * KC;
            fetch_rows(st, x, P.x_row, c0, k1, vec_x);
            if (TR) fetch_long(st + Tile::kStageX, w1, P.w1_row, c0, k1, vec_w1);
            else fetch_rank(st + Tile::kStageX, w1, P.w1_row, c0, k1, vec_w1);
        } else {
            const int64_t c0 = n0 + (int64_t)(c - nk) * KC;
            if (base) fetch_rows(st, base, P.base_row, c0, n1, vec_base);
            if (TR) fetch_rank(st + Tile::kStageX, w2, P.w2_row, c0, n1, vec_w2);
            else fetch_long(st + Tile::kStageX, w2, P.w2_row, c0, n1, vec_w2);
        }
    };

    Acc* us = reinterpret_cast<Acc*>(smem + S * Tile::kStage);
    Acc acc[RP / 8][4] = {};
    // The middle as this thread's part of the left operand: 16-bit data split in
    // two and, for halves, scaled by a power of two per row; f32 and f64 plain.
    uint32_t uh[E == 2 ? RP / 16 : 1][4], ul[E == 2 ? RP / 16 : 1][4];
    Acc uf[E == 2 ? 1 : RP / (E == 4 ? 8 : 4)][E == 4 ? 4 : 2];
    float back[2] = {1.f, 1.f};
    const bool busy = warp * 16 < count;

    auto exchange = [&]() {
        Acc* own = us + warp * 16 * Tile::kPitchU;
#pragma unroll
        for (int t = 0; t < RP / 8; ++t) {
            own[g * Tile::kPitchU + t * 8 + 2 * q] = acc[t][0];
            own[g * Tile::kPitchU + t * 8 + 2 * q + 1] = acc[t][1];
            own[(g + 8) * Tile::kPitchU + t * 8 + 2 * q] = acc[t][2];
            own[(g + 8) * Tile::kPitchU + t * 8 + 2 * q + 1] = acc[t][3];
        }
        cluster.sync();
        const Acc s = (Acc)(P.scales ? P.scales[slot.cls] : P.scale);
        const Acc* parts[8];
#pragma unroll
        for (int b = 0; b < 8; ++b) parts[b] = b < cs ? cluster.map_shared_rank(own, b) : nullptr;
        auto at = [&](int row, int j) {
            Acc v = 0;
#pragma unroll
            for (int b = 0; b < 8; ++b)
                if (b < cs) v += parts[b][row * Tile::kPitchU + j];
            return j < P.r ? v * s : Acc(0);  // past the rank, an infinite x met a zero: NaN
        };
        auto keep = [&](int row, int j, Acc v) {
            if (P.u && cr == 0 && j < P.r && warp * 16 + row < count)
                static_cast<Acc*>(P.u)[(int64_t)list[warp * 16 + row] * P.u_row + j] = v;
        };
        if (busy) {
            if constexpr (E == 2) {
                float v[RP / 16][8];
                float top[2] = {0.f, 0.f};
#pragma unroll
                for (int t = 0; t < RP / 16; ++t)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {  // a0..a3 of two: rows g, g + 8, then columns + 8
                        const int row = g + (e >> 1 & 1) * 8, j = t * 16 + 2 * q + (e & 1) + (e >> 2) * 8;
                        v[t][e] = at(row, j);
                        keep(row, j, v[t][e]);
                        top[e >> 1 & 1] = fmaxf(top[e >> 1 & 1], fabsf(v[t][e]));
                    }
                float down[2] = {1.f, 1.f};
                if constexpr (std::is_same<T, __half>::value) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
                        top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
                        const int e = (int)(__float_as_uint(top[h]) >> 23);  // 0 and 255 stay unscaled
                        if (e > 0 && e < 254) {
                            down[h] = __uint_as_float((254 - e) << 23);
                            back[h] = __uint_as_float(e << 23);
                        }
                    }
                }
#pragma unroll
                for (int t = 0; t < RP / 16; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        split16<T>(v[t][2 * e] * down[e & 1], v[t][2 * e + 1] * down[e & 1], uh[t][e], ul[t][e]);
            } else if constexpr (E == 4) {
#pragma unroll
                for (int t = 0; t < RP / 8; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int row = g + (e & 1) * 8, j = t * 8 + q + (e >> 1) * 4;
                        uf[t][e] = at(row, j);
                        keep(row, j, uf[t][e]);
                    }
            } else {
#pragma unroll
                for (int t = 0; t < RP / 4; ++t)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        uf[t][e] = at(g + e * 8, t * 4 + q);
                        keep(g + e * 8, t * 4 + q, uf[t][e]);
                    }
            }
        }
    };

    auto shrink = [&](const uint8_t* st) {
        const uint8_t* wt = st + Tile::kStageX;
        if constexpr (E == 2) {
            const uint32_t xa = shared_address(st) + (warp * 16 + (lane & 15)) * Tile::kPitchX + (lane >> 4) * 16;
            const uint32_t wa = shared_address(wt) +
                                (TR ? (lane & 15) * Tile::kPitchLong + (lane >> 4) * 16
                                    : ((lane & 7) + (lane >> 4) * 8) * Tile::kPitchRank + (lane >> 3 & 1) * 16);
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
                uint32_t a[4], b[4];
                ldsm4(a, xa + ks * 32);
#pragma unroll
                for (int p = 0; p < RP / 16; ++p) {
                    if (TR) ldsm4t(b, wa + ks * 16 * Tile::kPitchLong + p * 32);
                    else ldsm4(b, wa + p * 16 * Tile::kPitchRank + ks * 32);
                    mma16<T>(acc[2 * p], a, b[0], b[1]);
                    mma16<T>(acc[2 * p + 1], a, b[2], b[3]);
                }
            }
        } else if constexpr (E == 4) {
            // The tensor cores' sums run over one chunk; chunks are added in registers, rounded to nearest.
            float sum[RP / 8][4] = {};
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
                uint32_t ah[4], al[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const Tf32Pair p = tf32_split(*reinterpret_cast<const float*>(
                        st + (warp * 16 + g + (e & 1) * 8) * Tile::kPitchX + (ks * 8 + q + (e >> 1) * 4) * 4));
                    ah[e] = p.hi, al[e] = p.lo;
                }
#pragma unroll
                for (int t = 0; t < RP / 8; ++t) {
                    Tf32Pair b[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int kk = ks * 8 + q + e * 4, j = t * 8 + g;
                        b[e] = tf32_split(*reinterpret_cast<const float*>(
                            wt + (TR ? kk * Tile::kPitchLong + j * 4 : j * Tile::kPitchRank + kk * 4)));
                    }
                    mma_tf32(sum[t], ah, b[0].lo, b[1].lo);
                    mma_tf32(sum[t], al, b[0].hi, b[1].hi);
                    mma_tf32(sum[t], ah, b[0].hi, b[1].hi);
                }
            }
#pragma unroll
            for (int t = 0; t < RP / 8; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[t][e] += sum[t][e];
        } else {
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
                const uint8_t* xa = st + (warp * 16 + g) * Tile::kPitchX + (ks * 4 + q) * 8;
                const double a0 = *reinterpret_cast<const double*>(xa);
                const double a1 = *reinterpret_cast<const double*>(xa + 8 * Tile::kPitchX);
#pragma unroll
                for (int t = 0; t < RP / 8; ++t) {
                    const int kk = ks * 4 + q, j = t * 8 + g;
                    mma_f64(acc[t], a0, a1, *reinterpret_cast<const double*>(
                        wt + (TR ? kk * Tile::kPitchLong + j * 8 : j * Tile::kPitchRank + kk * 8)));
                }
            }
        }
    };

    // Two neighbouring results of rows g and g + 8 at column `col` of the chunk: base plus the
    // product, rounded once, left where base was.
    auto finish = [&](uint8_t* st, int col, Acc c0, Acc c1, Acc c2, Acc c3) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            T* o = reinterpret_cast<T*>(st + (warp * 16 + g + h * 8) * Tile::kPitchX) + col;
            Acc a = h ? c2 : c0, b = h ? c3 : c1;
            if constexpr (std::is_same<T, __half>::value) a *= back[h], b *= back[h];
            if (base) a += widen(o[0]), b += widen(o[1]);
            alignas(16) T v[2] = {narrow<T>(a), narrow<T>(b)};
            if constexpr (E == 2) *reinterpret_cast<uint32_t*>(o) = *reinterpret_cast<uint32_t*>(v);
            else if constexpr (E == 4) *reinterpret_cast<uint2*>(o) = *reinterpret_cast<uint2*>(v);
            else *reinterpret_cast<uint4*>(o) = *reinterpret_cast<uint4*>(v);
        }
    };

    auto expand = [&](uint8_t* st, int64_t c0) {
        const uint8_t* wt = st + Tile::kStageX;
        if constexpr (E == 2) {
            const uint32_t wa = shared_address(wt) +
                                (TR ? (lane & 15) * Tile::kPitchRank + (lane >> 4) * 16
                                    : ((lane & 7) + (lane >> 4) * 8) * Tile::kPitchLong + (lane >> 3 & 1) * 16);
#pragma unroll
            for (int p = 0; p < KC / 16; ++p) {
                float c[2][4] = {};
#pragma unroll
                for (int t = 0; t < RP / 16; ++t) {
                    uint32_t b[4];
                    if (TR) ldsm4t(b, wa + t * 16 * Tile::kPitchRank + p * 32);
                    else ldsm4(b, wa + p * 16 * Tile::kPitchLong + t * 32);
                    mma16<T>(c[0], ul[t], b[0], b[1]);
                    mma16<T>(c[1], ul[t], b[2], b[3]);
                    mma16<T>(c[0], uh[t], b[0], b[1]);
                    mma16<T>(c[1], uh[t], b[2], b[3]);
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) finish(st, p * 16 + h * 8 + 2 * q, c[h][0], c[h][1], c[h][2], c[h][3]);
            }
        } else if constexpr (E == 4) {
            float c[KC / 8][4] = {};
#pragma unroll
            for (int t = 0; t < RP / 8; ++t) {
                uint32_t ah[4], al[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const Tf32Pair p = tf32_split(uf[t][e]);
                    ah[e] = p.hi, al[e] = p.lo;
                }
#pragma unroll
                for (int p = 0; p < KC / 8; ++p) {
                    Tf32Pair b[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int j = t * 8 + q + e * 4, l = p * 8 + g;
                        b[e] = tf32_split(*reinterpret_cast<const float*>(
                            wt + (TR ? j * Tile::kPitchRank + l * 4 : l * Tile::kPitchLong + j * 4)));
                    }
                    mma_tf32(c[p], ah, b[0].lo, b[1].lo);
                    mma_tf32(c[p], al, b[0].hi, b[1].hi);
                    mma_tf32(c[p], ah, b[0].hi, b[1].hi);
                }
            }
#pragma unroll
            for (int p = 0; p < KC / 8; ++p) finish(st, p * 8 + 2 * q, c[p][0], c[p][1], c[p][2], c[p][3]);
        } else {
            double c[KC / 8][4] = {};
#pragma unroll
            for (int t = 0; t < RP / 4; ++t)
#pragma unroll
                for (int p = 0; p < KC / 8; ++p) {
                    const int j = t * 4 + q, l = p * 8 + g;
                    mma_f64(c[p], uf[t][0], uf[t][1], *reinterpret_cast<const double*>(
                        wt + (TR ? j * Tile::kPitchRank + l * 8 : l * Tile::kPitchLong + j * 8)));
                }
#pragma unroll
            for (int p = 0; p < KC / 8; ++p) finish(st, p * 8 + 2 * q, c[p][0], c[p][1], c[p][2], c[p][3]);
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // 8 lanes a row, 16 bytes each
            const int row = warp * 16 + i * 4 + lane / 8;
            const int64_t c = c0 + (lane % 8) * V;
            const int avail = row < count ? clamp(n1 - c) : 0;
            const uint8_t* src = st + row * Tile::kPitchX + (lane % 8) * 16;
            T* dst = y + list[row] * P.y_row + c;
            if (vec_y && avail == V) {
                *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(src);
            } else {
                for (int e = 0; e < avail; ++e) dst[e] = reinterpret_cast<const T*>(src)[e];
            }
        }
    };

#pragma unroll
    for (int c = 0; c < S - 1; ++c) {
        if (c < total) fetch(c);
        copy_commit();
    }
    for (int c = 0; c < total; ++c) {
        copy_wait<S - 2>();
        __syncthreads();  // chunk c has arrived for all; chunk c - 1's buffer is free
        if (c + S - 1 < total) fetch(c + S - 1);
        copy_commit();
        uint8_t* st = smem + c % S * Tile::kStage;
        if (c < nk) {
            if (busy) shrink(st);
        } else {
            if (c == nk) exchange();
            if (busy) expand(st, n0 + (int64_t)(c - nk) * KC);
        }
    }
    if (total == nk) exchange();
    cluster.sync();  // no block leaves while another may read its partial sums
}

// Gradients of the factors: grad[i][j][c] = sum over the rows t of adapter i of
// p[t][j] * q[t][c], dA from (v, x) and dB from (u, dy), in one launch.
//
// A block holds a stretch of columns and all of the rank in registers and walks
// the adapter's rows, so q is read once and p (rank values a row) by every block
// of columns.  Where that gives too few blocks, a cluster splits the rows into
// consecutive parts, whose sums meet in the blocks' order.
struct AdapterGradSide {
    const void* p;  // [rows, p_row] of the sums' type
    const void* q;  // [rows, cols]
    int64_t q_row, cols;
    void* grad;     // [adapters, r, cols] or, by_column, [adapters, cols, r]
    int by_column;
};
struct AdapterGradParams {
    AdapterGradSide side[2];
    int64_t first_blocks;  // blocks of side 0; the others are side 1's
    int64_t rows;
    int r, p_row, adapters;
    const int32_t* plan;
};

template <typename T, int RP>
struct AdapterGradTile {
    using Acc = typename AccOf<T>::type;
    static constexpr int E = sizeof(T), V = 16 / E;
    static constexpr int MT = E == 2 && RP < 128 ? 2 : 1;     // 16-column tiles a warp holds
    static constexpr int COLS = 64 * MT;
    static constexpr int KT = E == 8 ? 16 : 32;               // rows of a chunk
    static constexpr int kPitchQ = COLS * E + (E == 2 ? 16 : 32);
    static constexpr int kPitchP = (RP + (E == 4 ? 8 : 4)) * (int)sizeof(Acc);
    static constexpr int kStage = KT * (kPitchQ + kPitchP);
    static constexpr int kStages = RP <= 64 ? 4 : 3;
    static constexpr int kPitchD = RP + 1;                    // the block's sums, after the rows
    static constexpr int kJoin = COLS * kPitchD * (int)sizeof(Acc);
    static constexpr int kSmem = kStages * kStage > kJoin ? kStages * kStage : kJoin;
    static constexpr int kFlush = E == 2 ? 8 : 1;             // chunks that the tensor cores sum by themselves
};

template <typename T, int RP>
__global__ void __launch_bounds__(kTileThreads) adapter_grad_kernel(const __grid_constant__ AdapterGradParams P) {
    using Tile = AdapterGradTile<T, RP>;
    using Acc = typename Tile::Acc;
    constexpr int E = Tile::E, V = Tile::V, KT = Tile::KT, S = Tile::kStages, MT = Tile::MT, COLS = Tile::COLS;
    extern __shared__ __align__(16) uint8_t smem[];
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, q = lane & 3;
    const int cr = (int)cluster.block_rank(), cs = (int)cluster.num_blocks();
    const bool second = blockIdx.x >= P.first_blocks;
    const AdapterGradSide& side = P.side[second];
    const int64_t c0 = (blockIdx.x - (second ? P.first_blocks : 0)) / cs * COLS;
    const int cls = blockIdx.y;
    const int start = P.plan[cls], rows = P.plan[cls + 1] - start;
    const int32_t* perm = P.plan + plan_perm_word(P.rows, P.adapters) + start;
    const int share = (rows + KT * cs - 1) / (KT * cs) * KT;
    const int t0 = cr * share < rows ? cr * share : rows, t1 = t0 + share < rows ? t0 + share : rows;
    const int chunks = (t1 - t0 + KT - 1) / KT;
    const T* qs = static_cast<const T*>(side.q);
    const Acc* ps = static_cast<const Acc*>(side.p);
    const bool vec = ((reinterpret_cast<uintptr_t>(qs) | (uintptr_t)(side.q_row * E)) & 15) == 0;

    // Row ids of a thread's copies, one chunk ahead of the copies themselves.
    constexpr int QU = COLS / V, QI = KT * QU / kTileThreads;          // 16-byte units of a q row; copies a thread
    constexpr int PV = 16 / (int)sizeof(Acc), PU = RP / PV, PI = KT * PU / kTileThreads;
    int q_id[QI], p_id[PI];
    auto ids = [&](int c) {
#pragma unroll
        for (int i = 0; i < QI; ++i) {
            const int t = t0 + c * KT + (tid + i * kTileThreads) / QU;
            q_id[i] = t < t1 ? perm[t] : -1;
        }
#pragma unroll
        for (int i = 0; i < PI; ++i) {
            const int t = t0 + c * KT + (tid + i * kTileThreads) / PU;
            p_id[i] = t < t1 ? perm[t] : -1;
        }
    };
    auto fetch = [&](int c) {
        uint8_t* st = smem + c % S * Tile::kStage;
#pragma unroll
        for (int i = 0; i < QI; ++i) {
            const int u = tid + i * kTileThreads;
            const int64_t col = c0 + u % QU * V, left = side.cols - col;
            const int avail = q_id[i] < 0 || left < 0 ? 0 : left > V ? V : (int)left;
            fetch16(st + u / QU * Tile::kPitchQ + u % QU * 16, qs + q_id[i] * side.q_row + col, qs, avail, vec);
        }
#pragma unroll
        for (int i = 0; i < PI; ++i) {
            const int u = tid + i * kTileThreads, j = u % PU * PV;
            const int avail = p_id[i] < 0 || j >= P.p_row ? 0 : PV;  // p_row is a multiple of PV
            fetch16(st + KT * Tile::kPitchQ + u / PU * Tile::kPitchP + u % PU * 16,
                    ps + (int64_t)p_id[i] * P.p_row + j, ps, avail, true);
        }
    };

    Acc acc[MT][RP / 8][4] = {}, sum[E == 8 ? 1 : MT][E == 8 ? 1 : RP / 8][4] = {};
    auto flush = [&]() {
        if constexpr (E != 8) {
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int t = 0; t < RP / 8; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[m][t][e] += sum[m][t][e], sum[m][t][e] = 0;
        }
    };
    auto compute = [&](const uint8_t* st) {
        const uint8_t* pt = st + KT * Tile::kPitchQ;
        auto p_at = [&](int row, int j) {
            return *reinterpret_cast<const Acc*>(pt + row * Tile::kPitchP + j * (int)sizeof(Acc));
        };
        if constexpr (E == 2) {
            const uint32_t qa = shared_address(st) + ((lane & 7) + (lane >> 4) * 8) * Tile::kPitchQ +
                                (warp * 16 * MT + (lane >> 3 & 1) * 8) * 2;
#pragma unroll
            for (int ks = 0; ks < KT / 16; ++ks) {
                uint32_t a[MT][4];
#pragma unroll
                for (int m = 0; m < MT; ++m) ldsm4t(a[m], qa + ks * 16 * Tile::kPitchQ + m * 32);
                if constexpr (std::is_same<T, __nv_bfloat16>::value) {
#pragma unroll
                    for (int t = 0; t < RP / 8; ++t) {
                        uint32_t hi[2], lo[2];
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int row = ks * 16 + 2 * q + e * 8, j = t * 8 + g;
                            split16<T>(p_at(row, j), p_at(row + 1, j), hi[e], lo[e]);
                        }
#pragma unroll
                        for (int m = 0; m < MT; ++m) {
                            mma16<T>(sum[m][t], a[m], lo[0], lo[1]);
                            mma16<T>(sum[m][t], a[m], hi[0], hi[1]);
                        }
                    }
                } else {
                    // A half is a tf32 value as it is; the middle, whose range is a float's, is split
                    // in two.  The order of rows within the sum is free: rows 2q and 2q + 1 stand
                    // where the instruction has q and q + 4.
                    uint32_t w[MT][2][4];
#pragma unroll
                    for (int m = 0; m < MT; ++m)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&a[m][e]));
                            w[m][e >> 1][e & 1] = __float_as_uint(f.x);
                            w[m][e >> 1][(e & 1) + 2] = __float_as_uint(f.y);
                        }
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int t = 0; t < RP / 8; ++t) {
                            const int row = ks * 16 + h * 8 + 2 * q, j = t * 8 + g;
                            const Tf32Pair b0 = tf32_split(p_at(row, j)), b1 = tf32_split(p_at(row + 1, j));
#pragma unroll
                            for (int m = 0; m < MT; ++m) {
                                mma_tf32(sum[m][t], w[m][h], b0.lo, b1.lo);
                                mma_tf32(sum[m][t], w[m][h], b0.hi, b1.hi);
                            }
                        }
                }
            }
        } else if constexpr (E == 4) {
#pragma unroll
            for (int ks = 0; ks < KT / 8; ++ks) {
                uint32_t ah[4], al[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const Tf32Pair p = tf32_split(*reinterpret_cast<const float*>(
                        st + (ks * 8 + q + (e >> 1) * 4) * Tile::kPitchQ + (warp * 16 + g + (e & 1) * 8) * 4));
                    ah[e] = p.hi, al[e] = p.lo;
                }
#pragma unroll
                for (int t = 0; t < RP / 8; ++t) {
                    const Tf32Pair b0 = tf32_split(p_at(ks * 8 + q, t * 8 + g));
                    const Tf32Pair b1 = tf32_split(p_at(ks * 8 + q + 4, t * 8 + g));
                    mma_tf32(sum[0][t], ah, b0.lo, b1.lo);
                    mma_tf32(sum[0][t], al, b0.hi, b1.hi);
                    mma_tf32(sum[0][t], ah, b0.hi, b1.hi);
                }
            }
        } else {
#pragma unroll
            for (int ks = 0; ks < KT / 4; ++ks) {
                const uint8_t* qa = st + (ks * 4 + q) * Tile::kPitchQ + (warp * 16 + g) * 8;
                const double a0 = *reinterpret_cast<const double*>(qa), a1 = *reinterpret_cast<const double*>(qa + 64);
#pragma unroll
                for (int t = 0; t < RP / 8; ++t) mma_f64(acc[0][t], a0, a1, p_at(ks * 4 + q, t * 8 + g));
            }
        }
    };

    ids(0);
#pragma unroll
    for (int c = 0; c < S - 1; ++c) {
        if (c < chunks) {
            fetch(c);
            ids(c + 1);
        }
        copy_commit();
    }
    for (int c = 0; c < chunks; ++c) {
        copy_wait<S - 2>();
        __syncthreads();
        if (c + S - 1 < chunks) {
            fetch(c + S - 1);
            ids(c + S);
        }
        copy_commit();
        compute(smem + c % S * Tile::kStage);
        if (c % Tile::kFlush == Tile::kFlush - 1) flush();
    }
    flush();
    copy_wait<0>();
    __syncthreads();
    Acc* mine = reinterpret_cast<Acc*>(smem);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int t = 0; t < RP / 8; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                mine[((warp * MT + m) * 16 + g + (e >> 1) * 8) * Tile::kPitchD + t * 8 + 2 * q + (e & 1)] = acc[m][t][e];
    cluster.sync();
    const Acc* parts[8];
#pragma unroll
    for (int b = 0; b < 8; ++b) parts[b] = b < cs ? cluster.map_shared_rank(mine, b) : nullptr;
    const int cols = side.cols - c0 < COLS ? (int)(side.cols - c0) : COLS, own = COLS / cs;
    const int first = cr * own, last = first + own < cols ? first + own : cols;
    T* grad = static_cast<T*>(side.grad) + (int64_t)cls * P.r * side.cols;
    const int many = last > first ? (last - first) * P.r : 0;
    for (int i = tid; i < many; i += kTileThreads) {
        const int c = first + (side.by_column ? i / P.r : i % (last - first));
        const int j = side.by_column ? i % P.r : i / (last - first);
        Acc v = 0;
#pragma unroll
        for (int b = 0; b < 8; ++b)
            if (b < cs) v += parts[b][c * Tile::kPitchD + j];
        grad[side.by_column ? (c0 + c) * P.r + j : j * side.cols + c0 + c] = narrow<T>(v);
    }
    cluster.sync();
}

}  // namespace fpemu
