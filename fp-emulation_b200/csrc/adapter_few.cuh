// adapter_few.cuh -- the adapter products of a few rows (single tokens, small
// batches), where the weights are what there is to read.
//
// A cluster of blocks takes up to eight rows of one adapter and shares the
// lengths k and n.  Weights and rows go from memory straight into the operands
// of mma.sync: the order of k inside a sum is free, so a thread's 16 contiguous
// bytes of a weight row and of an input row stand for the same slots, and no
// value passes through shared memory.  Eight rows fill the narrow side of the
// instruction; in the second product the sixteen rows of its wide side hold the
// eight rows twice, as the high and the low part of the middle.  A bfloat16 middle
// has a third part, in an instruction of its own: two parts hold 16 of a float's 24
// bits, which moved three results in a thousand to a neighbouring bfloat16.
//
// Measured (kernel alone, cold L2), 4096 -> 4096, rank 16: 32 rows with an adapter
// each, bfloat16, 10.1 us (its 9 MB take 1.4 at the copy rate), float64 15.4 (5.6);
// 200 rows of 24 adapters, 11.3 (1.7) and 19.0 (6.9); 7 us for any tiny call.  What is left is latency, a few microseconds each for finding
// the rows, the two streams of loads and the two meetings of the cluster; the call's
// host side takes 15 us.  Fetching the weights ahead into the L2 changed nothing.
#pragma once

#include "adapter_tiles.cuh"

namespace fpemu {

constexpr int kFewThreads = 256;
constexpr int kGroupRows = 8;

__device__ __forceinline__ void mma_f64_8(double (&c)[2], double a, double b) {
    asm volatile("mma.sync.aligned.m8n8k4.row.col.f64.f64.f64.f64 {%0,%1}, {%2}, {%3}, {%0,%1};"
                 : "+d"(c[0]), "+d"(c[1]) : "d"(a), "d"(b));
}

// 16 bytes of a row: `avail` elements, zeros after them.  Vec: the row is aligned and
// `avail` is a whole 16 bytes or none; the load is predicated, not branched around, so
// that a thread's loads leave together.  (Not through the read-only path: base may be
// y itself.)
template <bool Vec, typename T>
__device__ __forceinline__ uint4 load16(const T* p, int avail) {
    constexpr int V = 16 / sizeof(T);
    if constexpr (Vec) {
        uint4 v;
        asm("{\n.reg .pred p;\nsetp.gt.s32 p, %5, 0;\nmov.b32 %0, 0;\nmov.b32 %1, 0;\nmov.b32 %2, 0;\nmov.b32 %3, 0;\n"
            "@p ld.global.v4.u32 {%0,%1,%2,%3}, [%4];\n}"
            : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w)
            : "l"(p), "r"(avail));
        return v;
    }
    alignas(16) T v[V];
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = i < avail ? p[i] : T(0.0f);
    return *reinterpret_cast<uint4*>(v);
}

// Joins the blocks' parts of N sums: each block takes its share of them, adds
// the parts in the blocks' order, and stores done(e, sum) to every block (each block
// adding up all of them itself took 0.7 us a block more, one load after another).  A
// cluster barrier before makes the parts visible, one after the results; after
// that no block reads or writes another's memory.
template <int N, typename Acc, typename At, typename Done>
__device__ __forceinline__ void join_parts(cg::cluster_group& cluster, int cr, int cs, Acc* part, Acc* out, At at,
                                           Done done) {
    for (int i = threadIdx.x; i < N / cs; i += blockDim.x) {
        const int e = cr * (N / cs) + i, o = at(e);
        Acc p[8];
#pragma unroll
        for (int b = 0; b < 8; ++b)  // all loads in flight before the first addition
            if (b < cs) p[b] = *cluster.map_shared_rank(part + o, b);
        Acc v = p[0];
#pragma unroll
        for (int b = 1; b < 8; ++b)
            if (b < cs) v += p[b];
        v = done(e, v);
#pragma unroll
        for (int b = 0; b < 8; ++b)
            if (b < cs) *cluster.map_shared_rank(out + o, b) = v;
    }
}

template <typename T, int RP>
struct FewTile {
    using Acc = typename AccOf<T>::type;
    static constexpr int E = sizeof(T), V = 16 / E, KS = 4 * V;     // elements of k a warp takes at a step
    static constexpr int MR = E == 8 ? 8 : 16;                      // ranks of an instruction
    static constexpr int RT = RP / MR, PA = E == 8 ? 2 : 4;         // rank tiles; sums a thread holds of one
    static constexpr int UN = RP <= 16 ? 4 : RP <= 32 ? 2 : 1;  // steps with their loads in flight together
    static constexpr int JS = (RP + KS - 1) / KS;                   // 16-byte steps along the rank
    static constexpr int UG = E == 8 && RP <= 16 ? 4 : JS * V >= 16 ? 1 : JS * V >= 8 ? 2 : 4;  // column groups, likewise
    static constexpr int kWarps = kFewThreads / 32;
    static constexpr int kSmem = (kWarps + 2) * RP * kGroupRows * (int)sizeof(Acc);
    // An SM's blocks, by registers (three with 80 registers each spill: 32 rows, bfloat16, 10.4 us for 9.7).
    static constexpr int kBlocks = RP <= 64 ? 2 : 1;
};

template <typename T, int RP>
__global__ void __launch_bounds__(kFewThreads, FewTile<T, RP>::kBlocks) adapter_few_kernel(const __grid_constant__ AdapterParams P) {
    using Tile = FewTile<T, RP>;
    using Acc = typename Tile::Acc;
    constexpr int E = Tile::E, V = Tile::V, KS = Tile::KS, RT = Tile::RT, MR = Tile::MR, UN = Tile::UN, JS = Tile::JS;
    constexpr int W = Tile::kWarps;
    extern __shared__ __align__(16) uint8_t smem[];
    Acc* red = reinterpret_cast<Acc*>(smem);           // [warp][rank][row]
    Acc* part = red + W * RP * kGroupRows;             // [rank][row], read by the cluster
    Acc* us = part + RP * kGroupRows;                  // [rank][row], the cluster's sums
    __shared__ __align__(16) int ids[kFewRows];
    __shared__ unsigned leaders[W];
    __shared__ int list[kGroupRows], lead[2];
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, q = lane & 3;
    const int cr = (int)cluster.block_rank(), cs = (int)cluster.num_blocks();
    const int rows = (int)P.rows, unit = blockIdx.x / cs;

    // Rows of a class in groups of eight, by the rows' order; this cluster's group is the one whose
    // first row is the unit-th of all groups' first rows.
    const int mine = tid < rows ? row_class(P.index, P.index_wide, tid, P.adapters) : -1;
    ids[tid] = mine;
    __syncthreads();
    int rank = 0;
    for (int t = 0; t < tid; t += 4) {
        const int4 v = *reinterpret_cast<const int4*>(ids + t);
        rank += (v.x == mine) + (v.y == mine && t + 1 < tid) + (v.z == mine && t + 2 < tid) + (v.w == mine && t + 3 < tid);
    }
    const bool leader = tid < rows && rank % kGroupRows == 0;
    const unsigned ballot = __ballot_sync(0xffffffffu, leader);
    if (lane == 0) leaders[warp] = ballot;
    __syncthreads();
    int before = __popc(ballot & ((1u << lane) - 1)), groups = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
        if (w < warp) before += __popc(leaders[w]);
        groups += __popc(leaders[w]);
    }
    if (unit >= groups) return;
    if (leader && before == unit) lead[0] = mine, lead[1] = rank;
    __syncthreads();
    const int cls = lead[0], place = rank - lead[1];
    const bool in = tid < rows && mine == cls && place >= 0 && place < kGroupRows;
    if (in) list[place] = tid;
    const int count = __syncthreads_count(in);

    const int k = (int)P.k, n = (int)P.n;
    const int kshare = (k + KS * cs - 1) / (KS * cs) * KS, nshare = (n + KS * cs - 1) / (KS * cs) * KS;
    const int k0 = min(cr * kshare, k), n0 = min(cr * nshare, n);
    const int k1 = min(k0 + kshare, k), n1 = min(n0 + nshare, n);
    if (cls >= P.adapters) {
        if (cls > P.adapters && cr == 0 && tid == 0)
            report_error(P.sink.dev, P.sink.host, FPEMU_ERR_INVALID, kWhereAdapterIndex, list[0]);
        plain_rows<T>(P, list, count, cls != P.adapters, n0, n1);
        return;
    }
    const T* w1 = static_cast<const T*>(P.w1) + cls * P.w1_adapter;
    const T* w2 = static_cast<const T*>(P.w2) + cls * P.w2_adapter;
    const int64_t row = list[g < count ? g : 0];
    const T* xp = static_cast<const T*>(P.x) + row * P.x_row;
    const T* base = P.base ? static_cast<const T*>(P.base) + row * P.base_row : nullptr;
    T* y = static_cast<T*>(P.y) + row * P.y_row;
    auto aligned = [](const void* p, int64_t stride) {
        return ((reinterpret_cast<uintptr_t>(p) | (uintptr_t)(stride * E)) & 15) == 0;
    };
    const bool vec_x = aligned(P.x, P.x_row), vec_w1 = aligned(w1, P.w1_row), vec_w2 = aligned(w2, P.w2_row);
    const bool vec_y = aligned(P.y, P.y_row), vec_base = aligned(P.base, P.base_row);

    // The second product's weights start towards the L2 now.
    if (P.w2_row == P.r) {
        const char* from = reinterpret_cast<const char*>(w2 + (int64_t)n0 * P.r);
        const int64_t bytes = (int64_t)(n1 - n0) * P.r * E;
        for (int64_t at = (int64_t)tid * 128; at < bytes; at += kFewThreads * 128)
            asm volatile("prefetch.global.L2 [%0];" ::"l"(from + at));
    }

    Acc acc[RT][Tile::PA] = {};
    // The tensor cores' adders truncate: after some instructions (FL rounds of loads) their sums of
    // floats go to this thread's places in `red`, rounded there (65536 values of one sign, one block,
    // float32: 9e-5 off without).
    constexpr int FL = E == 4 ? 1 : 32 / UN;
    bool more = false;
    auto flush = [&]() {
        if constexpr (E != 8) {
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float2* o = reinterpret_cast<float2*>(&red[(warp * RP + t * MR + h * 8 + g) * kGroupRows + 2 * q]);
                    const float2 old = more ? *o : make_float2(0.f, 0.f);
                    *o = make_float2(old.x + acc[t][2 * h], old.y + acc[t][2 * h + 1]);
                    acc[t][2 * h] = acc[t][2 * h + 1] = 0;
                }
            more = true;
        }
    };
    auto add_up = [&](auto vec) {
        int rounds = 0;
        for (int c = k0 + warp * KS; c < k1; c += W * KS * UN) {
            uint4 xv[UN], wv[UN][RT][MR / 8];
#pragma unroll
            for (int u = 0; u < UN; ++u) {
                const int at = c + u * W * KS + q * V, avail = k1 - at;
                xv[u] = load16<vec>(xp + at, avail);
#pragma unroll
                for (int t = 0; t < RT; ++t)
#pragma unroll
                    for (int h = 0; h < MR / 8; ++h) {
                        const int j = t * MR + h * 8 + g;
                        wv[u][t][h] = load16<vec>(w1 + j * P.w1_row + at, j < P.r ? avail : 0);
                    }
            }
#pragma unroll
            for (int u = 0; u < UN; ++u) {
                const uint32_t* xr = reinterpret_cast<const uint32_t*>(&xv[u]);
#pragma unroll
                for (int t = 0; t < RT; ++t) {
                    if constexpr (E == 8) {
                        const double* xd = reinterpret_cast<const double*>(&xv[u]);
                        const double* wd = reinterpret_cast<const double*>(&wv[u][t][0]);
                        mma_f64_8(acc[t], wd[0], xd[0]);
                        mma_f64_8(acc[t], wd[1], xd[1]);
                    } else {
                        const uint32_t* wa = reinterpret_cast<const uint32_t*>(&wv[u][t][0]);
                        const uint32_t* wb = reinterpret_cast<const uint32_t*>(&wv[u][t][MR / 8 - 1]);
#pragma unroll
                        for (int m = 0; m < 2; ++m) {
                            if constexpr (E == 2) {
                                const uint32_t a[4] = {wa[2 * m], wb[2 * m], wa[2 * m + 1], wb[2 * m + 1]};
                                mma16<T>(acc[t], a, xr[2 * m], xr[2 * m + 1]);
                            } else {
                                const Tf32Pair p0 = tf32_split(__uint_as_float(wa[2 * m]));
                                const Tf32Pair p1 = tf32_split(__uint_as_float(wb[2 * m]));
                                const Tf32Pair p2 = tf32_split(__uint_as_float(wa[2 * m + 1]));
                                const Tf32Pair p3 = tf32_split(__uint_as_float(wb[2 * m + 1]));
                                const Tf32Pair b0 = tf32_split(__uint_as_float(xr[2 * m]));
                                const Tf32Pair b1 = tf32_split(__uint_as_float(xr[2 * m + 1]));
                                const uint32_t hi[4] = {p0.hi, p1.hi, p2.hi, p3.hi}, lo[4] = {p0.lo, p1.lo, p2.lo, p3.lo};
                                mma_tf32(acc[t], hi, b0.lo, b1.lo);
                                mma_tf32(acc[t], lo, b0.hi, b1.hi);
                                mma_tf32(acc[t], hi, b0.hi, b1.hi);
                            }
                        }
                    }
                }
            }
            if (E != 8 && ++rounds % FL == 0) flush();
        }
    };
    if (vec_x && vec_w1 && k % V == 0)
        add_up(std::true_type{});
    else
        add_up(std::false_type{});
    // The second product's loads: UG groups of KS columns of this warp, their weights and base.
    constexpr int NT = V / 2;  // 8-column tiles of a group; a thread's results are 16 bytes of neighbours
    constexpr int UG = Tile::UG;
    uint4 w2v[UG][NT][JS], held[UG];
    auto load_groups = [&](int first, auto vec) {
#pragma unroll
        for (int u = 0; u < UG; ++u) {
            const int c0 = first + u * W * KS;
#pragma unroll
            for (int p = 0; p < NT; ++p)
#pragma unroll
                for (int t = 0; t < JS; ++t) {
                    const int c = c0 + g / 2 * V + 2 * p + g % 2, j = t * KS + q * V;
                    w2v[u][p][t] = load16<vec>(w2 + c * P.w2_row + j, c < n1 ? P.r - j : 0);
                }
            const int avail = g < count ? n1 - c0 - q * V : 0;
            held[u] = load16<vec>(base + c0 + q * V, base ? avail : 0);
        }
    };
    const bool vec2 = vec_w2 && vec_base && P.r % V == 0 && n % V == 0;
    auto load_second = [&](int first) {
        if (vec2)
            load_groups(first, std::true_type{});
        else
            load_groups(first, std::false_type{});
    };
    load_second(n0 + warp * KS);  // its first loads cross the exchange of the middle

    if constexpr (E == 8) {
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e) red[(warp * RP + t * MR + g) * kGroupRows + 2 * q + e] = acc[t][e];
    } else {
        flush();
    }
    __syncthreads();
    for (int i = tid; i < RP * kGroupRows; i += kFewThreads) {
        Acc v = red[i];
#pragma unroll
        for (int w = 1; w < W; ++w) v += red[w * RP * kGroupRows + i];
        part[i] = v;
    }
    cluster.sync();
    const Acc s = (Acc)(P.scales ? P.scales[cls] : P.scale);
    join_parts<RP * kGroupRows>(cluster, cr, cs, part, us, [](int e) { return e; }, [&](int e, Acc v) {
        const int j = e / kGroupRows, r = e % kGroupRows;
        v = j < P.r ? v * s : Acc(0);
        if (P.u && j < P.r && r < count) static_cast<Acc*>(P.u)[(int64_t)list[r] * P.u_row + j] = v;
        return v;
    });
    cluster.sync();

    // The middle as the left operand: rows g; where there are sixteen, rows g + 8 hold the low parts.
    constexpr int UA = E == 8 ? 2 : E == 4 ? 8 : 8;
    using Part = typename std::conditional<E == 8, double, uint32_t>::type;
    constexpr bool kThird = std::is_same<T, __nv_bfloat16>::value;
    Part ua[JS][UA];
    uint32_t third[kThird ? JS : 1][4];
    float down = 1.f, back = 1.f;
    if constexpr (E == 2 && std::is_same<T, __half>::value) {
        float top = 0.f;
        for (int j = q; j < RP; j += 4) top = HalfScale::larger(top, us[j * kGroupRows + g]);
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const HalfScale s(top);
        down = s.down, back = s.back;
    }
#pragma unroll
    for (int t = 0; t < JS; ++t) {
        const int j0 = t * KS + q * V;
        auto at = [&](int i) { return RP % KS == 0 || j0 + i < RP ? us[(j0 + i) * kGroupRows + g] : Acc(0); };
        if constexpr (E == 8) {
            ua[t][0] = at(0), ua[t][1] = at(1);
        } else if constexpr (E == 4) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const Tf32Pair p = tf32_split(at(i));
                ua[t][2 * i] = p.hi, ua[t][2 * i + 1] = p.lo;
            }
        } else if constexpr (kThird) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t p[3];
                split_bf16(at(2 * i), at(2 * i + 1), p);
                ua[t][2 * i] = p[0], ua[t][2 * i + 1] = p[1], third[t][i] = p[2];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                split_half(at(2 * i) * down, at(2 * i + 1) * down, ua[t][2 * i], ua[t][2 * i + 1]);
        }
    }
    for (int first = n0 + warp * KS; first < n1; first += W * KS * UG) {
        if (first != n0 + warp * KS) load_second(first);
#pragma unroll
        for (int u = 0; u < UG; ++u) {
            const int col = first + u * W * KS + q * V, avail = g < count ? n1 - col : 0;
            T* v = reinterpret_cast<T*>(&held[u]);
#pragma unroll
            for (int p = 0; p < NT; ++p) {
                Acc r0, r1;
                if constexpr (E == 8) {
                    double c[2] = {};
#pragma unroll
                    for (int t = 0; t < JS; ++t) {
                        const double* wd = reinterpret_cast<const double*>(&w2v[u][p][t]);
                        mma_f64_8(c, ua[t][0], wd[0]);
                        mma_f64_8(c, ua[t][1], wd[1]);
                    }
                    r0 = c[0], r1 = c[1];
                } else {
                    float c[4] = {};
#pragma unroll
                    for (int t = 0; t < JS; ++t) {
                        const uint32_t* wr = reinterpret_cast<const uint32_t*>(&w2v[u][p][t]);
#pragma unroll
                        for (int m = 0; m < 2; ++m) {
                            const uint32_t a[4] = {ua[t][4 * m], ua[t][4 * m + 1], ua[t][4 * m + 2], ua[t][4 * m + 3]};
                            if constexpr (E == 2) {
                                if constexpr (kThird) {
                                    const uint32_t rest[4] = {third[t][2 * m], 0, third[t][2 * m + 1], 0};
                                    mma16<T>(c, rest, wr[2 * m], wr[2 * m + 1]);
                                }
                                mma16<T>(c, a, wr[2 * m], wr[2 * m + 1]);
                            } else {
                                const Tf32Pair b0 = tf32_split(__uint_as_float(wr[2 * m]));
                                const Tf32Pair b1 = tf32_split(__uint_as_float(wr[2 * m + 1]));
                                // Low parts meet high ones alone: an infinite middle is all in its low part.
                                const uint32_t high[4] = {a[0], 0, a[2], 0};
                                mma_tf32(c, high, b0.lo, b1.lo);
                                mma_tf32(c, a, b0.hi, b1.hi);
                            }
                        }
                    }
                    r0 = (c[2] + c[0]) * back, r1 = (c[3] + c[1]) * back;
                }
                if (base) r0 += widen(v[2 * p]), r1 += widen(v[2 * p + 1]);
                v[2 * p] = narrow<T>(r0), v[2 * p + 1] = narrow<T>(r1);
            }
            if (vec_y && avail >= V) {
                *reinterpret_cast<uint4*>(y + col) = held[u];
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e)
                    if (e < avail) y[col + e] = v[e];
            }
        }
    }
}

}  // namespace fpemu
