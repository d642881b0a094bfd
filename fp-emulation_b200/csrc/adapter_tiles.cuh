// adapter_tiles.cuh -- the adapter products of long batches on the tensor cores.
//
// Two kernels: u = s W1 x (k long, rank wide), then y = base + W2 u.  Their work
// is a list of chunks, 64 rows of one adapter (a slot of the plan) by 128 bytes
// along k or n, dealt out in equal consecutive stretches to as many blocks as the
// device holds, whatever the adapters' shares of the batch.  A block streams its
// stretch through one ring of asynchronous copies without a pause from slot to
// slot.  A slot whose k is divided between blocks leaves partial sums in the
// workspace, which the second kernel adds in the blocks' order.  x, base and y
// pass through one block once; u and its parts are a rank wide and stay in the L2.
//
// What bounds them: the bytes of x, base and y, as long as the rank is small --
// float64 up to rank 16 or so (mma.sync f64 reaches 37 TFLOP/s, the device's whole
// rate), 16-bit data up to rank 64 (545 TFLOP/s; tf32, for floats, 273).  Measured:
//   float64, 16384 x 4096 -> 4096, rank 16, 8 adapters in runs: 307 us, 5.3 TB/s of
//     algorithmic bytes, 0.81 of the measured copy rate (107 us for u, 5.0 TB/s);
//   half, 16384 x 4096 -> 8192, rank 64, 16 adapters: 215 us, 3.2 TB/s.  There the
//     second kernel (172 us) is bound by what a computing warp does for a chunk:
//     without its matrix instructions it takes 119 us, its copies alone 80.
// One kernel for both products, in clusters that exchanged the middle through
// distributed shared memory, was no faster (330 us for the float64 case): its blocks'
// shares came in whole slots, and 256 of them on 148 SMs left a seventh of the device idle.
#pragma once

#include <cuda.h>

#include "adapter_kernels.cuh"
#include "fpemu_barrier.cuh"

namespace fpemu {

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

template <int B>
__device__ __forceinline__ void copy_small(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(B), "r"(bytes) : "memory");
}

// How an operand's rows may be copied: 16 bytes at a time; 4 (floats and even
// pairs of 16-bit values) or 8 (doubles); or, 0, 16-bit values at odd places, one
// by one through registers.
template <typename T>
__device__ __forceinline__ int copy_unit(const void* p, int64_t stride) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(p) | (uintptr_t)(stride * (int64_t)sizeof(T));
    return (a & 15) == 0 ? 16 : sizeof(T) >= 4 ? (int)sizeof(T) : (a & 3) == 0 ? 4 : 0;
}

template <typename T>
__device__ __forceinline__ int copy_unit2(const void* p, int64_t row, int64_t adapter) {
    const int a = copy_unit<T>(p, row), b = copy_unit<T>(p, adapter);
    return a < b ? a : b;
}

// 16 bytes of a tile: `avail` elements from src, zeros after them.  What is not
// available is not read.
template <typename T>
__device__ __forceinline__ void fetch16(uint8_t* dst, const T* src, int avail, int unit) {
    constexpr int E = sizeof(T), V = 16 / E, B = E == 8 ? 8 : 4;
    if (unit == 16) {
        copy16(shared_address(dst), src, avail * E);
    } else if (unit != 0) {
#pragma unroll
        for (int i = 0; i < 16 / B; ++i) {
            const int left = avail * E - i * B;
            copy_small<B>(shared_address(dst) + i * B, src + i * (B / E), left < 0 ? 0 : left < B ? left : B);
        }
    } else if (E == 2) {
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
// products; what it loses is 2^-21 of it at most (lo x lo, and the last bit of a lo that
// has twelve).  An infinite or NaN x is in lo,
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

// What a row of the middle is multiplied by for halves, and its reciprocal: powers of two that put
// the row's largest finite magnitude `top` between 2^14 and 2^15.  The values down to 2^-17 of it then
// keep 22 bits, those down to 2^-28 at least 11, as many as a half (below 2^-112 nothing of
// a row is left in a half).
struct HalfScale {
    float down = 1.f, back = 1.f;
    __device__ __forceinline__ explicit HalfScale(float top) {
        const uint32_t e = __float_as_uint(top) >> 23;
        if (e >= 15) down = __uint_as_float((268 - e) << 23), back = __uint_as_float((e - 14) << 23);
    }
    // The largest finite magnitude so far.
    static __device__ __forceinline__ float larger(float top, float v) {
        return fabsf(v) < __int_as_float(0x7f800000) ? fmaxf(top, fabsf(v)) : top;
    }
};

// Two neighbouring floats as two halves each, 22 bits of them.
__device__ __forceinline__ void split_half(float x, float y, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(fminf(x - f.x, 65504.f), fminf(y - f.y, 65504.f));
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
}

// Two neighbouring floats as three bfloat16 parts each, largest first, which hold all of their 24
// bits: every part is cut, not rounded, so that a finite value stays finite and the rest is exact.
// The parts have one sign; those after an infinite one are finite.
__device__ __forceinline__ void split_bf16(float x, float y, uint32_t (&p)[3]) {
    constexpr uint32_t keep = 0xffff0000u;
    auto rest = [](float v) {  // of an infinite v the difference is NaN
        const float r = fabsf(v - __uint_as_float(__float_as_uint(v) & keep));
        return copysignf(fminf(r, 1e38f), v);
    };
    const float x1 = rest(x), y1 = rest(y);
    const float x2 = x1 - __uint_as_float(__float_as_uint(x1) & keep), y2 = y1 - __uint_as_float(__float_as_uint(y1) & keep);
    auto pack = [](float a, float b) { return __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632); };
    p[0] = pack(x, y), p[1] = pack(x1, y1), p[2] = pack(x2, y2);
}

constexpr int kTileThreads = 256;      // eight warps that compute
constexpr int kCopyThreads = 64;       // and two that copy

// Tiles in shared memory, as TMA writes them with 128-byte swizzle: rows of 128
// bytes whose 16-byte units change places by the row.  "Rank-major" weights have a
// row for each rank and 128 bytes along the long dimension.  "Long-major" ones have
// a row for each of its elements and the rank along it, in sub-tiles of at most 128
// bytes of rank (narrower rows have the narrower swizzles).  A warp's fragment loads
// are free of bank conflicts, but for weights read across their rows by f32 and f64.
__device__ __forceinline__ uint32_t tile_at(int row, int byte) { return row * 128 + (byte ^ (row & 7) << 4); }

template <typename T, bool TR, int RP>
struct AdapterTile {
    using Acc = typename AccOf<T>::type;
    static constexpr int E = sizeof(T), V = 16 / E;
    static constexpr int KC = 128 / E;                             // elements of a chunk along k or n
    static constexpr int kStageX = kSlotRows * 128, kStage = kStageX + RP * 128;
    static constexpr int kInner = RP * E < 128 ? RP * E : 128;     // bytes of a long-major row
    static constexpr int kSubs = RP * E / kInner;
    static constexpr int kPitchU = E == 2 ? RP + 8 : RP + 4;       // elements of Acc
    static constexpr int kMiddle = kSlotRows * kPitchU * (int)sizeof(Acc);
    // Two blocks an SM where the registers for a rank's sums allow it, and as many chunks in flight as fit.
    static constexpr int kBlocks = RP * E <= 128 ? 2 : 1;
    static constexpr int kFit = ((kBlocks == 2 ? 108000 : 220000) - kMiddle) / kStage;
    static constexpr int kStages = kFit < 8 ? kFit : 8;
    static constexpr int kSmem = kStages * kStage + kMiddle + 1024;  // and room to align
    static_assert(kStages >= 3, "the copies of a chunk overlap the work on others");
    static __device__ __forceinline__ uint32_t long_at(int row, int byte) {
        const int sub = byte / kInner, in = byte % kInner;
        const int turn = kInner == 128 ? row & 7 : kInner == 64 ? row >> 1 & 3 : row >> 2 & 1;
        return sub * (KC * kInner) + row * kInner + (in ^ turn << 4);
    }
    // The results of a warp's two rows are 16 bytes of neighbouring columns for each thread: column
    // NT i + p of a chunk stands where the instruction has column i of its tile p.  Long-major weights of
    // the second product are laid out in that order; 16-bit rank-major ones (read transposed, eight
    // neighbours at a time) are not, and their results go through the tile instead.
    static constexpr int NT = V / 2;
    static constexpr bool kDirect = !(TR && E == 2);
    static __device__ __forceinline__ int at(int c) { return c % NT * 16 + c / NT; }
};

// Rows without an adapter (base, or 0) or with an id that is none (NaN, so that a
// wrong index never looks like a result), this block's share of the columns.
template <typename T>
__device__ void plain_rows(const AdapterParams& P, const int* list, int count, bool bad, int n0, int n1) {
    using Acc = typename AccOf<T>::type;
    constexpr int V = 16 / (int)sizeof(T);
    if ((!bad && P.base == P.y && P.base_row == P.y_row) || n1 <= n0) return;
    const T* base = static_cast<const T*>(P.base);
    T* y = static_cast<T*>(P.y);
    const T fill = narrow<T>(bad ? (Acc)__longlong_as_double(0x7ff8000000000000ll) : (Acc)0);
    const bool vec = !bad && base && copy_unit<T>(base, P.base_row) == 16 && copy_unit<T>(y, P.y_row) == 16;
    constexpr int warps = kTileThreads / 32;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, len = n1 - n0;
    const int whole = vec ? len / V * V : 0;  // of a row, copied 16 bytes at a time
    for (int first = warp; first < count; first += 8 * warps) {
        // Eight rows of a warp with their loads in flight together.
        auto columns = [&](auto unit, int from, int to, int step) {
            using U = decltype(unit);
            for (int c = from; c < to; c += step) {
                U v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int t = first + i * warps;
                    if (t < count && !bad && base) v[i] = *reinterpret_cast<const U*>(base + list[t] * P.base_row + n0 + c);
                    else if constexpr (std::is_same<U, T>::value) v[i] = fill;
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int t = first + i * warps;
                    if (t < count) *reinterpret_cast<U*>(y + list[t] * P.y_row + n0 + c) = v[i];
                }
            }
        };
        columns(uint4{}, lane * V, whole, 32 * V);
        columns(T(0.0f), whole + lane, len, 32);
    }
}

// 64 gathered rows by 128 bytes: a copying thread's 16 bytes of every eighth row.
template <typename T>
struct RowTile {
    static constexpr int V = 16 / (int)sizeof(T), KC = 8 * V, N = kSlotRows * 8 / kCopyThreads;
    const T* p[N];
    int count;
    __device__ __forceinline__ void aim(int t, const T* src, int64_t stride, const int* list, int rows, int64_t c0) {
#pragma unroll
        for (int i = 0; i < N; ++i) p[i] = src + list[t / 8 + 8 * i] * stride + c0 + t % 8 * V;
        count = rows;
    }
    // `left` elements of the rows are there; moves on to the next chunk.
    __device__ __forceinline__ void fetch(int t, uint8_t* st, int left, int unit) {
        const int here = left - t % 8 * V, avail = here < 0 ? 0 : here > V ? V : here;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            fetch16(st + tile_at(t / 8 + 8 * i, t % 8 * 16), p[i], t / 8 + 8 * i < count ? avail : 0, unit);
            p[i] += KC;
        }
    }
};

// The weights of a chunk: LONG, a row of the rank for each of KC elements (in the
// order of the results where PLACED), or RP rows of KC elements.
template <typename T, typename Tile, int RP, bool LONG, bool PLACED>
struct WeightTile {
    static constexpr int E = sizeof(T), V = 16 / E, KC = 8 * V;
    static constexpr int UPR = LONG ? RP * E / 16 : 8, SKIP = kCopyThreads / UPR, N = RP / 8;
    const T* p;
    __device__ __forceinline__ void aim(int t, const T* w, int64_t stride, int64_t c0) {
        p = w + (t / UPR + (LONG ? c0 : 0)) * stride + t % UPR * V + (LONG ? 0 : c0);
    }
    __device__ __forceinline__ void fetch(int t, uint8_t* wt, int64_t stride, int r, int left, int unit) {
        const int l = t / UPR, j = t % UPR * V, here = LONG ? r - j : left - j;
        const int avail = here < 0 ? 0 : here > V ? V : here;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int row = l + i * SKIP;
            fetch16(wt + (LONG ? Tile::long_at(PLACED ? Tile::at(row) : row, j * E) : tile_at(row, j * E)),
                    p + i * SKIP * stride, (LONG ? row < left : row < r) ? avail : 0, unit);
        }
        p += LONG ? KC * stride : KC;
    }
};

// TMA: a box of consecutive rows, or of the weights' map (see make_weight_map).
// What lies outside the maps is zero.  (Rows that do not follow one another are
// copied by the threads: TMA's gather of four rows by 128 bytes took some 50 cycles
// an instruction on an SM, 2.9 TB/s in all, where two warps' copies reach 4.2.)
__device__ __forceinline__ void tma_box2(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
                 " [%0], [%1, {%3, %4}], [%2];" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)),
                 "r"(smem_u32(bar)), "r"(c0), "r"(c1) : "memory");
}
__device__ __forceinline__ void tma_box4(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c3) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
                 " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)),
                 "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(0), "r"(c3) : "memory");
}

template <int ID, int N>
__device__ __forceinline__ void named_barrier() {
    asm volatile("bar.sync %0, %1;" ::"n"(ID), "n"(N) : "memory");
}
// Meets the N threads of barrier ID and says whether every one of them came with `yes`.
template <int ID, int N>
__device__ __forceinline__ bool agreed_barrier(bool yes) {
    uint32_t all;
    asm volatile("{\n.reg .pred p, q;\nsetp.ne.u32 p, %1, 0;\nbar.red.and.pred q, %2, %3, p;\nselp.u32 %0, 1, 0, q;\n}"
                 : "=r"(all) : "r"((uint32_t)yes), "n"(ID), "n"(N) : "memory");
    return all != 0;
}
constexpr int kCopyBarrier = 1, kWorkBarrier = 2;

// A warp's wait: it runs out for all lanes or for none (each has a clock of its own, and
// what follows a wait takes the whole warp).
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, uint64_t budget_ns) {
    const uint32_t a = smem_u32(bar);
    if (__all_sync(0xffffffffu, mbar_try_wait(a, parity))) return true;
    const uint64_t t0 = global_ns();
    for (uint32_t i = 1;; ++i) {
        if (__all_sync(0xffffffffu, mbar_try_wait(a, parity))) return true;
        if ((i & 255u) == 0u && __any_sync(0xffffffffu, global_ns() - t0 > budget_ns)) return false;
    }
}

// The ring of chunks: a buffer is full when TMA's bytes and every copying thread's
// copies have arrived (and what they wrote themselves is visible), and free again
// when each of the eight computing warps has left it.  So a warp runs ahead of
// another by as many chunks as there are buffers, and loads, products and stores
// overlap.  Waits are bounded (FPEMU_WAIT_BUDGET_MS): when one runs out, the error
// is recorded and what could not be finished becomes NaN.  A warp gives up as a whole;
// the others find out at their own next wait, so until then it still meets them at
// every barrier that they pass.
template <int S>
struct ChunkRing {
    uint64_t full[S], empty[S];
    volatile int failed;  // a computing warp's wait ran out
    __device__ __forceinline__ void init() {
        if (threadIdx.x == 0) {
            failed = 0;
#pragma unroll
            for (int i = 0; i < S; ++i)
                mbar_init(&full[i], 2 * kCopyThreads), mbar_init(&empty[i], kTileThreads / 32);
            fence_barrier_init();
        }
        __syncthreads();
    }
    // One chunk: the threads' copies, and what thread 0 asks of TMA (`bytes` in all).  Every copying thread
    // arrives twice, when its copies have landed and for what it wrote itself.
    template <typename Copies, typename Tma>
    __device__ __forceinline__ void copied_after(int s, int t, uint32_t bytes, Copies copies, Tma tma) {
        if (t == 0 && bytes > 0) {
            mbar_arrive_expect_tx(&full[s], bytes);
            tma();
        }
        copies();
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(shared_address(&full[s])) : "memory");
        if (t > 0 || bytes == 0) mbar_arrive(&full[s]);
    }
    __device__ __forceinline__ void left(int s) {
        __syncwarp();
        if ((threadIdx.x & 31) == 0) mbar_arrive(&empty[s]);
    }
};

// The slots of a block's stretch, for the copying threads: rows and record of the
// slot that is being fetched and of those behind it that are still being computed,
// with the loads of the next ones under way.
struct SlotFeed {
    static constexpr int kRing = 16;  // a chunk in flight each, at most
    int (*list)[kSlotRows];   // [kRing], shared
    AdapterSlot* rec;         // [kRing], shared
    const AdapterSlot* slots;
    const int32_t* perm;
    int busy, t;              // slots; this thread, of kCopyThreads
    int slot;                 // the one that enter() makes current next
    AdapterSlot next, after;
    int id;
    __device__ __forceinline__ int load_id(const AdapterSlot& s) { return perm[s.start + (t < s.count ? t : 0)]; }
    __device__ __forceinline__ AdapterSlot load(int i) const { return slots[i < busy ? i : busy - 1]; }
    __device__ __forceinline__ void begin(int first) {
        slot = first;
        next = load(first), after = load(first + 1);
        id = load_id(next);
    }
    // All copying threads; `now` becomes the slot whose rows are in list[(slot - 1) % kRing].  False,
    // for both warps, if one of them comes without `ok`.
    __device__ __forceinline__ bool enter(bool ok, AdapterSlot& now) {
        const int at = slot % kRing;
        list[at][t] = id;
        if (t == 0) rec[at] = next;
        if (!agreed_barrier<kCopyBarrier, kCopyThreads>(ok)) return false;
        now = next;
        next = after;
        id = load_id(next);
        ++slot;
        after = load(slot + 1);
        return true;
    }
};

// What a kernel streams: gathered rows (or none) and weights, `length` elements long.
struct StreamParams {
    const void *rows, *w;
    int64_t row_stride, w_adapter, w_row;
    int length, rank;
    const CUtensorMap *row_map, *w_map;
    int tma;  // kTmaRows, kTmaWeights: which maps there are
    uint64_t budget_ns;
    int stall;
};

// The copying warps of a block: its chunks from `at` of slot `slot` on.  Weights,
// and the rows of a slot that follow one another in memory, come by TMA where
// pointers and strides are multiples of 16 bytes (rows past the slot's are then some
// other slot's: no result meets them).  The rest is copied by the threads, 16 bytes
// at a time, 4 or 8, or single values, whatever the alignment.
template <typename T, typename Tile, int RP, bool LONG, bool PLACED>
__device__ __forceinline__ void stream_chunks(const StreamParams& q, ChunkRing<Tile::kStages>& ring, uint8_t* smem,
                                              int (*list)[kSlotRows], AdapterSlot* rec, const AdapterSlot* slots,
                                              const int32_t* perm, int busy, int slot, int at, int per, int chunks,
                                              ErrorSink sink) {
    constexpr int S = Tile::kStages, KC = Tile::KC, kNT = PLACED ? Tile::NT : 1;
    const int t = threadIdx.x - kTileThreads;
    const T* rows = static_cast<const T*>(q.rows);
    const T* w = static_cast<const T*>(q.w);
    const bool tma_w = q.tma & kTmaWeights;
    RowTile<T> xt;
    WeightTile<T, Tile, RP, LONG, PLACED> wt;
    const int unit_rows = copy_unit<T>(rows, q.row_stride), unit_w = copy_unit2<T>(w, q.w_row, q.w_adapter);
    SlotFeed feed{list, rec, slots, perm, busy, t};
    if (chunks > 0) feed.begin(slot);
    int stage = 0, cls = 0, first = 0, asked = 0;  // chunks whose copies this warp has asked for
    uint32_t round = 1;
    bool box = true, ok = true;
    int fenced = 0;  // up to this chunk, buffers may hold rows that the threads copied
    for (int c = 0; c < chunks; ++c) {
        if (ok && blockIdx.x == 0 && c == q.stall) ok = false;
        if (ok && c >= S && !warp_wait(&ring.empty[stage], round, q.budget_ns)) {
            report_error(sink.dev, sink.host, FPEMU_ERR_TIMEOUT, kWaitAdapterEmpty, c);
            ok = false;
        }
        if (c == 0 || at == 0) {
            AdapterSlot s;
            if (!feed.enter(ok, s)) break;
            const int* ids = list[(feed.slot - 1) % SlotFeed::kRing];
            cls = s.cls, first = ids[0];
            const bool before = box;
            box = (q.tma & kTmaRows) && ids[s.count - 1] - first == s.count - 1;
            if (box && !before) fenced = c + S;
            if (rows && !box) xt.aim(t, rows, q.row_stride, ids, s.count, (int64_t)at * KC);
            if (!tma_w) wt.aim(t, w + s.cls * q.w_adapter, q.w_row, (int64_t)at * KC);
        }
        uint8_t* st = smem + stage * Tile::kStage;
        if (ok) ring.copied_after(stage, t, (rows && box ? Tile::kStageX : 0) + (tma_w ? RP * 128 : 0), [&]() {
            if (rows && !box) xt.fetch(t, st, q.length - at * KC, unit_rows);
            if (!tma_w) wt.fetch(t, st + Tile::kStageX, q.w_row, q.rank, q.length - at * KC, unit_w);
        }, [&]() {
            const uint32_t to = shared_address(st);
            // The threads' copies were ordinary writes; TMA's to the same place come after them.
            if (c < fenced) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            if (rows && box) tma_box2(to, q.row_map, &ring.full[stage], at * KC, first);
            if (tma_w) {
                if (LONG)
#pragma unroll
                    for (int b = 0; b < Tile::kSubs; ++b)
                        tma_box4(to + Tile::kStageX + b * (KC * Tile::kInner), q.w_map, &ring.full[stage],
                                 b * (Tile::kInner / Tile::E), at * (KC / kNT), cls);
                else tma_box4(to + Tile::kStageX, q.w_map, &ring.full[stage], at * KC, 0, cls);
            }
        });
        asked += ok;
        if (++at == per) at = 0;
        if (++stage == S) stage = 0, round ^= 1;
    }
    copy_commit();
    copy_wait<0>();
    // Given up: what TMA has under way has to land before the block may end.  (A chunk that the other
    // warp gave up never becomes full; its wait is the time that the copies have.)
    if (asked < chunks)
        for (int i = asked < S ? 0 : asked - S; i < asked; ++i)
            if (!warp_wait(&ring.full[i % S], i / S & 1, q.budget_ns)) break;
}

// Block b of `blocks` takes chunks [total b / blocks, total (b + 1) / blocks).  A
// stretch is an eighth of a slot at least, so that a slot has few parts.
struct ChunkShare {
    int64_t total;
    int blocks;
    __device__ __forceinline__ ChunkShare(int busy, int per, int grid) {
        total = (int64_t)busy * per;
        const int64_t most = total / ((per + 7) / 8);
        blocks = (int)(most < grid ? (most > 0 ? most : 1) : grid);
    }
    __device__ __forceinline__ int64_t first(int b) const { return total * b / blocks; }
    __device__ __forceinline__ int owner(int64_t chunk) const { return (int)(((chunk + 1) * blocks - 1) / total); }
};

// u: eight warps, RG groups of rows by KW parts of every chunk's k; a warp holds
// its rows' sums over its parts for the whole rank, and the KW sums are added when
// the block leaves the slot.  (The warps of a group read each x once; with all of k
// and half of the rank for each they would read it twice, and the loads from shared
// memory would bind the kernel.)
template <typename T, bool TR, int RP>
__global__ void __launch_bounds__(kTileThreads + kCopyThreads, AdapterTile<T, TR, RP>::kBlocks)
    adapter_shrink_kernel(const __grid_constant__ AdapterParams P, const __grid_constant__ CUtensorMap row_map,
                          const __grid_constant__ CUtensorMap w_map) {
    using Tile = AdapterTile<T, TR, RP>;
    using Acc = typename Tile::Acc;
    constexpr int E = Tile::E, KC = Tile::KC, S = Tile::kStages;
    constexpr int MT = RP < (E == 4 ? 32 : 128) ? 2 : 1, RG = 4 / MT, KW = 8 / RG, NT = RP / 8;
    // Chunks that the tensor cores sum by themselves.  Their adders truncate, which moves a sum of one
    // sign by some 2^-25 an instruction: floats are flushed into registers, and 16-bit data, for
    // which there are none left, into the slot's part in the workspace.
    constexpr int FLUSH = 4, HOLD = E == 2 ? 64 : INT_MAX;
    extern __shared__ uint8_t raw[];
    uint8_t* smem = raw + ((1024 - (shared_address(raw) & 1023)) & 1023);  // the swizzles repeat every 1024 bytes
    __shared__ int list[SlotFeed::kRing][kSlotRows];
    __shared__ AdapterSlot rec[SlotFeed::kRing];
    __shared__ ChunkRing<S> ring;
    cudaTriggerProgrammaticLaunchCompletion();
    const int tid = threadIdx.x, lane = tid & 31, g = lane >> 2, q = lane & 3;
    const int rows0 = (tid >> 5) % RG * 16 * MT, kw = (tid >> 5) / RG;
    const int busy = P.plan[plan_header_word(P.rows, P.adapters)];
    const int k = (int)P.k, per = (k + KC - 1) / KC;
    if (busy == 0) return;
    const ChunkShare share(busy, per, gridDim.x);
    if ((int)blockIdx.x >= share.blocks) return;
    const int64_t begin = share.first(blockIdx.x);
    const int chunks = (int)(share.first(blockIdx.x + 1) - begin);
    ring.init();
    if (tid >= kTileThreads) {
        const StreamParams q{P.x, P.w1, P.x_row, P.w1_adapter, P.w1_row, k, P.r, &row_map, &w_map, P.tma1, P.budget_ns, P.stall};
        stream_chunks<T, Tile, RP, TR, false>(q, ring, smem, list, rec, plan_busy(P), plan_perm(P), busy,
                                              (int)(begin / per), (int)(begin % per), per, chunks, P.sink);
        return;
    }

    Acc acc[MT][NT][4] = {}, sum[E == 4 ? MT : 1][E == 4 ? NT : 1][4] = {};
    auto flush = [&]() {
        if constexpr (E == 4) {
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[m][t][e] += sum[m][t][e], sum[m][t][e] = 0;
        }
    };
    auto shrink = [&](const uint8_t* st) {
        const uint8_t* ws = st + Tile::kStageX;
#pragma unroll
        for (int i = 0; i < 4 / KW; ++i) {
            const int ks = kw * (4 / KW) + i;
            if constexpr (E == 2) {
                const uint32_t xa = shared_address(st) + tile_at(rows0 + (lane & 15), ks * 32 + (lane >> 4) * 16);
                uint32_t a[MT][4];
#pragma unroll
                for (int m = 0; m < MT; ++m) ldsm4(a[m], xa + m * 16 * 128);
#pragma unroll
                for (int p = 0; p < RP / 16; ++p) {
                    uint32_t b[4];
                    if (TR) ldsm4t(b, shared_address(ws) + Tile::long_at(ks * 16 + (lane & 15), p * 32 + (lane >> 4) * 16));
                    else ldsm4(b, shared_address(ws) + tile_at(p * 16 + (lane & 7) + (lane >> 4) * 8, ks * 32 + (lane >> 3 & 1) * 16));
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        mma16<T>(acc[m][2 * p], a[m], b[0], b[1]);
                        mma16<T>(acc[m][2 * p + 1], a[m], b[2], b[3]);
                    }
                }
            } else if constexpr (E == 4) {
                uint32_t ah[MT][4], al[MT][4];
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const Tf32Pair p = tf32_split(*reinterpret_cast<const float*>(
                            st + tile_at(rows0 + m * 16 + g + (e & 1) * 8, (ks * 8 + q + (e >> 1) * 4) * 4)));
                        ah[m][e] = p.hi, al[m][e] = p.lo;
                    }
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    Tf32Pair b[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int kk = ks * 8 + q + e * 4, j = t * 8 + g;
                        b[e] = tf32_split(*reinterpret_cast<const float*>(
                            ws + (TR ? Tile::long_at(kk, j * 4) : tile_at(j, kk * 4))));
                    }
#pragma unroll
                    for (int m = 0; m < MT; ++m) mma_tf32(sum[m][t], ah[m], b[0].lo, b[1].lo);
#pragma unroll
                    for (int m = 0; m < MT; ++m) mma_tf32(sum[m][t], al[m], b[0].hi, b[1].hi);
#pragma unroll
                    for (int m = 0; m < MT; ++m) mma_tf32(sum[m][t], ah[m], b[0].hi, b[1].hi);
                }
            } else {
                // The order of k is free: this one puts the four threads of a row into different banks.
                const int kk = (q >> 1) * 8 + ks * 2 + (q & 1);
                double a[MT][2];
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        a[m][h] = *reinterpret_cast<const double*>(
                            st + tile_at(rows0 + m * 16 + h * 8 + g, kk * 8));
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const int j = t * 8 + g;
                    const double b = *reinterpret_cast<const double*>(ws + (TR ? Tile::long_at(kk, j * 8) : tile_at(j, kk * 8)));
#pragma unroll
                    for (int m = 0; m < MT; ++m) mma_f64(acc[m][t], a[m][0], a[m][1], b);
                }
            }
        }
    };
    // The block's sums of a slot to the workspace: the parts of k one after the other.
    Acc* red = reinterpret_cast<Acc*>(smem + S * Tile::kStage);
    auto leave = [&](int64_t part, bool more) {  // `more`: adds to what the block left there before
        flush();
        named_barrier<kWorkBarrier, kTileThreads>();  // every warp has read the last slot's sums
        for (int p = 0; p < KW; ++p) {
            if (kw == p) {
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            Acc* o = red + (rows0 + m * 16 + g + (e >> 1) * 8) * Tile::kPitchU + t * 8 + 2 * q + (e & 1);
                            *o = p ? *o + acc[m][t][e] : acc[m][t][e];
                            acc[m][t][e] = 0;
                        }
            }
            named_barrier<kWorkBarrier, kTileThreads>();
        }
        Acc* out = static_cast<Acc*>(P.parts) + part * (kSlotRows * RP);
        const bool ok = !ring.failed;  // else some warp's part is missing: the rows become NaN
        if (more) {
            for (int i = tid; i < kSlotRows * RP; i += kTileThreads) red[i / RP * Tile::kPitchU + i % RP] += out[i];
        }
        for (int i = tid; i < kSlotRows * RP; i += kTileThreads)
            out[i] = ok ? red[i / RP * Tile::kPitchU + i % RP] : (Acc)__longlong_as_double(0x7ff8000000000000ll);
    };

    int at = (int)(begin % per), slot = (int)(begin / per), stage = 0, held = 0;
    uint32_t round = 0;
    bool ok = true, more = false;
    for (int c = 0; c < chunks; ++c) {
        if (ok && !warp_wait(&ring.full[stage], round, P.budget_ns)) {
            report_error(P.sink.dev, P.sink.host, FPEMU_ERR_TIMEOUT, kWaitAdapterFull, c);
            ring.failed = 1;
            ok = false;
        }
        if (ok && rows0 < rec[slot % SlotFeed::kRing].count) shrink(smem + stage * Tile::kStage);
        ring.left(stage);
        if (++stage == S) stage = 0, round ^= 1;
        if (c % FLUSH == FLUSH - 1) flush();
        ++at, ++held;
        if (at == per || c + 1 == chunks || held == HOLD) {
            leave((int64_t)blockIdx.x + slot, more);
            held = 0, more = at < per;
            if (at == per) at = 0, ++slot;
        }
    }
}

// y: eight warps, four groups of 16 rows by the halves of every chunk's columns.
template <typename T, bool TR, int RP>
__global__ void __launch_bounds__(kTileThreads + kCopyThreads, AdapterTile<T, TR, RP>::kBlocks)
    adapter_expand_kernel(const __grid_constant__ AdapterParams P, const __grid_constant__ CUtensorMap row_map,
                          const __grid_constant__ CUtensorMap w_map) {
    using Tile = AdapterTile<T, TR, RP>;
    using Acc = typename Tile::Acc;
    constexpr int E = Tile::E, V = Tile::V, KC = Tile::KC, S = Tile::kStages;
    extern __shared__ uint8_t raw[];
    uint8_t* smem = raw + ((1024 - (shared_address(raw) & 1023)) & 1023);  // the swizzles repeat every 1024 bytes
    __shared__ int list[SlotFeed::kRing][kSlotRows];
    __shared__ AdapterSlot rec[SlotFeed::kRing];
    __shared__ ChunkRing<S> ring;
    __shared__ int plain[kSlotRows];  // rows without an adapter, apart from the copying warps' lists
    const int tid = threadIdx.x, lane = tid & 31, g = lane >> 2, q = lane & 3;
    const int rows0 = (tid >> 5 & 3) * 16, half = tid >> 7;
    const int32_t* header = P.plan + plan_header_word(P.rows, P.adapters);
    const int busy = header[0], idle = header[1];
    const int n = (int)P.n, per = n > 0 ? (n + KC - 1) / KC : 1;  // without columns, for u alone
    const T* base = static_cast<const T*>(P.base);
    const bool vec_y = copy_unit<T>(P.y, P.y_row) == 16;
    const ChunkShare share(busy > 0 ? busy : 1, per, gridDim.x);
    const bool here = busy > 0 && (int)blockIdx.x < share.blocks;
    const int64_t begin = here ? share.first(blockIdx.x) : 0;
    const int chunks = here ? (int)(share.first(blockIdx.x + 1) - begin) : 0;
    const int kper = ((int)P.k + KC - 1) / KC;
    const ChunkShare kshare(busy > 0 ? busy : 1, kper > 0 ? kper : 1, P.shrink_grid);
    ring.init();
    // Rows without an adapter, an eighth of the columns at a time, by the threads that compute.
    constexpr int kParts = 8;
    const int width = (n + kParts * V - 1) / (kParts * V) * V;
    if (tid >= kTileThreads) {
        const StreamParams q{P.base, P.w2, P.base_row, P.w2_adapter, P.w2_row, n, P.r, &row_map, &w_map, P.tma2, P.budget_ns, P.stall};
        stream_chunks<T, Tile, RP, !TR, !TR>(q, ring, smem, list, rec, plan_busy(P), plan_perm(P), busy,
                                             (int)(begin / per), (int)(begin % per), per, chunks, P.sink);
        cudaGridDependencySynchronize();
        return;
    }

    // f64: the rank that step t of this thread stands for (any order will do; this one spreads the banks).
    auto rank_of = [&](int t) { return t / 4 * 16 + (q >> 1) * 8 + t % 4 * 2 + (q & 1); };
    Acc* us = reinterpret_cast<Acc*>(smem + S * Tile::kStage);
    // The middle as this thread's part of the left operand: halves in two parts,
    // scaled by a power of two per row; bfloat16 in three; f32 and f64 plain.
    constexpr bool kThird = std::is_same<T, __nv_bfloat16>::value;
    uint32_t uh[E == 2 ? RP / 16 : 1][4], ul[E == 2 ? RP / 16 : 1][4], um[kThird ? RP / 16 : 1][4];
    Acc uf[E == 2 ? 1 : RP / (E == 4 ? 8 : 4)][E == 4 ? 4 : 2];
    float back[2];
    T* yp[2];
    bool ok = true;
    auto take_slot = [&](int slot, int at) {
        const AdapterSlot& now = rec[slot % SlotFeed::kRing];
        const int* rows = list[slot % SlotFeed::kRing];
        const Acc s = (Acc)(P.scales ? P.scales[now.cls] : P.scale);
        const int b0 = kper ? kshare.owner((int64_t)slot * kper) : 0;
        const int b1 = kper ? kshare.owner((int64_t)(slot + 1) * kper - 1) : -1;
        const Acc* parts = static_cast<const Acc*>(P.parts) + (int64_t)(b0 + slot) * (kSlotRows * RP);
        named_barrier<kWorkBarrier, kTileThreads>();  // every warp has read the last slot's middle
#pragma unroll 4
        for (int i = tid; i < kSlotRows * RP; i += kTileThreads) {
            Acc v = 0;
            for (int b = 0; b <= b1 - b0; ++b) v += __ldcg(parts + (int64_t)b * (kSlotRows * RP) + i);
            const int row = i / RP, r = i % RP;
            v = r < P.r ? v * s : Acc(0);  // past the rank, an infinite x met a zero: NaN
            us[row * Tile::kPitchU + r] = v;
            if (P.u && at == 0 && r < P.r && row < now.count)
                static_cast<Acc*>(P.u)[(int64_t)rows[row] * P.u_row + r] = v;
        }
        named_barrier<kWorkBarrier, kTileThreads>();
        const Acc* from = us + (rows0 + g) * Tile::kPitchU;
        if constexpr (E == 2) {
            float v[RP / 16][8];  // a0..a3 of two: rows g, g + 8, then columns + 8
#pragma unroll
            for (int t = 0; t < RP / 16; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 f = *reinterpret_cast<const float2*>(
                        from + (e & 1) * 8 * Tile::kPitchU + t * 16 + 2 * q + (e >> 1) * 8);
                    v[t][2 * e] = f.x, v[t][2 * e + 1] = f.y;
                }
            float down[2] = {1.f, 1.f};
            if constexpr (std::is_same<T, __half>::value) {
                float top[2] = {0.f, 0.f};
#pragma unroll
                for (int t = 0; t < RP / 16; ++t)
#pragma unroll
                    for (int e = 0; e < 8; ++e) top[e >> 1 & 1] = HalfScale::larger(top[e >> 1 & 1], v[t][e]);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
                    top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
                    const HalfScale s(top[h]);
                    down[h] = s.down, back[h] = s.back;
                }
            }
#pragma unroll
            for (int t = 0; t < RP / 16; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if constexpr (kThird) {
                        uint32_t part[3];
                        split_bf16(v[t][2 * e], v[t][2 * e + 1], part);
                        uh[t][e] = part[0], um[t][e] = part[1], ul[t][e] = part[2];
                    } else {
                        split_half(v[t][2 * e] * down[e & 1], v[t][2 * e + 1] * down[e & 1], uh[t][e], ul[t][e]);
                    }
                }
        } else {
            constexpr int step = E == 4 ? 8 : 4;  // a0, a1 of rows g, g + 8; f32 two more, four columns on
#pragma unroll
            for (int t = 0; t < RP / step; ++t)
#pragma unroll
                for (int e = 0; e < step / 2; ++e)
                    uf[t][e] = from[(e & 1) * 8 * Tile::kPitchU + (E == 8 ? rank_of(t) : t * step + q + (e >> 1) * 4)];
        }
        // This thread's rows of y at its 16 bytes of the warp's group of columns.
#pragma unroll
        for (int h = 0; h < 2; ++h)
            yp[h] = static_cast<T*>(P.y) + rows[rows0 + g + h * 8] * P.y_row + (int64_t)at * KC + half * (KC / 2) + q * V;
    };

    // 16-bit weights: where this thread's loads of a chunk start, from the chunk's buffer.
    uint32_t w_at[E == 2 ? (TR ? 2 : RP / 16) : 1];
    if constexpr (E == 2) {
        if constexpr (TR) {
#pragma unroll
            for (int p = 0; p < 2; ++p) w_at[p] = tile_at(lane & 15, (half * 32 + p * 16 + (lane >> 4) * 8) * 2);
        } else {
#pragma unroll
            for (int t = 0; t < RP / 16; ++t)
                w_at[t] = Tile::long_at((lane >> 4) * 16 + half * 8 + (lane & 7), t * 32 + (lane >> 3 & 1) * 16);
        }
    }
    auto expand = [&](uint8_t* st, int left, const int* rows, int count) {
        constexpr int NT = Tile::NT;  // 8-column tiles of the warp's half chunk
        const uint8_t* wt = st + Tile::kStageX;
        Acc c[NT][4] = {};
        if constexpr (E == 2) {
            const uint32_t w0 = shared_address(wt);
#pragma unroll
            for (int t = 0; t < RP / 16; ++t) {
                uint32_t b[2][4];
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    if (TR) ldsm4t(b[p], w0 + w_at[p] + t * 16 * 128);
                    else ldsm4(b[p], w0 + w_at[t] + p * 32 * Tile::kInner);
                }
#pragma unroll
                for (int p = 0; p < 4; ++p) mma16<T>(c[p], ul[t], b[p / 2][p % 2 * 2], b[p / 2][p % 2 * 2 + 1]);
#pragma unroll
                for (int p = 0; p < 4; ++p)
                    if constexpr (kThird) mma16<T>(c[p], um[t], b[p / 2][p % 2 * 2], b[p / 2][p % 2 * 2 + 1]);
#pragma unroll
                for (int p = 0; p < 4; ++p) mma16<T>(c[p], uh[t], b[p / 2][p % 2 * 2], b[p / 2][p % 2 * 2 + 1]);
            }
        } else if constexpr (E == 4) {
            float rest[NT][4] = {};
#pragma unroll
            for (int t = 0; t < RP / 8; ++t) {
                uint32_t ah[4], al[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const Tf32Pair p = tf32_split(uf[t][e]);
                    ah[e] = p.hi, al[e] = p.lo;
                }
#pragma unroll
                for (int p = 0; p < NT; ++p) {
                    Tf32Pair b[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int j = t * 8 + q + e * 4;
                        b[e] = tf32_split(*reinterpret_cast<const float*>(
                            wt + (TR ? tile_at(j, (half * 16 + NT * g + p) * 4) : Tile::long_at(p * 16 + half * 8 + g, j * 4))));
                    }
                    mma_tf32(rest[p], ah, b[0].lo, b[1].lo);
                    mma_tf32(c[p], ah, b[0].hi, b[1].hi);
                    mma_tf32(rest[p], al, b[0].hi, b[1].hi);
                }
            }
#pragma unroll
            for (int p = 0; p < NT; ++p)
#pragma unroll
                for (int e = 0; e < 4; ++e) c[p][e] += rest[p][e];
        } else {
            double odd[4] = {};
#pragma unroll
            for (int t = 0; t < RP / 4; ++t) {
                const int j = rank_of(t), l = half * 8 + g;
                mma_f64(t % 2 ? odd : c[0], uf[t][0], uf[t][1], *reinterpret_cast<const double*>(
                    wt + (TR ? tile_at(j, l * 8) : Tile::long_at(l, j * 8))));
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) c[0][e] += odd[e];
        }
        if constexpr (!Tile::kDirect) {
            // Through the tile: pairs of columns in, 16 bytes of a row out; base waits in the tile meanwhile.
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int p = 0; p < NT; ++p) {
                    T* o = reinterpret_cast<T*>(st + tile_at(rows0 + g + h * 8, half * 64 + p * 16 + 4 * q));
                    alignas(4) T v[2];
                    float a = c[p][2 * h], b = c[p][2 * h + 1];
                    if constexpr (std::is_same<T, __half>::value) a *= back[h], b *= back[h];
                    if (base) {
                        const float2 old = widen2(o);
                        a += old.x, b += old.y;
                    }
                    narrow2(v, a, b);
                    *reinterpret_cast<uint32_t*>(o) = *reinterpret_cast<uint32_t*>(v);
                }
            __syncwarp();
        }
        const bool whole = vec_y && left >= KC;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            alignas(16) T v[V];
            uint8_t* tile = st + tile_at(rows0 + g + h * 8, half * 64 + q * 16);
            if (!Tile::kDirect || base) *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(tile);
            if constexpr (Tile::kDirect) {
                Acc r[V];  // element NT b + p is column b of tile p
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    r[e] = c[e % NT][2 * h + e / NT];
                    if constexpr (std::is_same<T, __half>::value) r[e] *= back[h];
                }
#pragma unroll
                for (int e = 0; e < V; e += 2) {
                    if (base) {
                        const auto old = widen2(v + e);
                        r[e] += old.x, r[e + 1] += old.y;
                    }
                    narrow2(v + e, r[e], r[e + 1]);
                }
            }
            if (whole) {
                if (rows0 + g + h * 8 < count) *reinterpret_cast<uint4*>(yp[h]) = *reinterpret_cast<uint4*>(v);
            } else {
                *reinterpret_cast<uint4*>(tile) = *reinterpret_cast<uint4*>(v);
            }
            yp[h] += KC;
        }
        if (!whole) {  // element by element, neighbouring lanes on neighbouring columns
            constexpr int H = KC / 2;
            __syncwarp();
#pragma unroll 4
            for (int i = lane; i < 16 * H; i += 32) {
                const int row = rows0 + i / H, col = half * H + i % H;
                if (row < count && col < left)
                    static_cast<T*>(P.y)[rows[row] * P.y_row + n - left + col] =
                        *reinterpret_cast<const T*>(st + tile_at(row, col * E));
            }
        }
        // The tile was written here and is next written by TMA.
        if (!Tile::kDirect || !whole) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    };

    // This thread's share of a middle that take_slot did not get to.
    auto lose_middle = [&](const AdapterSlot& s) {
        for (int i = tid; i < kSlotRows * RP; i += kTileThreads)
            if (i / RP < s.count && i % RP < P.r)
                static_cast<Acc*>(P.u)[(int64_t)plan_perm(P)[s.start + i / RP] * P.u_row + i % RP] =
                    (Acc)__longlong_as_double(0x7ff8000000000000ll);
    };

    cudaGridDependencySynchronize();  // the parts of u are there
    int at = (int)(begin % per), slot = (int)(begin / per), stage = 0;
    uint32_t round = 0;
    for (int c = 0; c < chunks; ++c) {
        if (ok && !warp_wait(&ring.full[stage], round, P.budget_ns)) {
            report_error(P.sink.dev, P.sink.host, FPEMU_ERR_TIMEOUT, kWaitAdapterFull, c);
            ring.failed = 1;
            ok = false;
        }
        if (c == 0 || at == 0) {
            if (ok) {
                take_slot(slot, at);
            } else {  // a warp that has given up still meets the others, as often as in take_slot
                named_barrier<kWorkBarrier, kTileThreads>();
                named_barrier<kWorkBarrier, kTileThreads>();
                if (P.u && at == 0) lose_middle(plan_busy(P)[slot]);
            }
            ok = __all_sync(0xffffffffu, ok && !ring.failed);  // else a warp's share of the middle is missing
        }
        if (!ok) {  // what is left becomes NaN
            const AdapterSlot s = plan_busy(P)[slot];
            const T nan = narrow<T>((Acc)__longlong_as_double(0x7ff8000000000000ll));
            for (int i = lane; i < 16 * (KC / 2); i += 32) {
                const int row = rows0 + i / (KC / 2), col = at * KC + half * (KC / 2) + i % (KC / 2);
                if (row < s.count && col < n) static_cast<T*>(P.y)[plan_perm(P)[s.start + row] * P.y_row + col] = nan;
            }
            if (++at == per) at = 0, ++slot;
            continue;
        }
        const int count = rec[slot % SlotFeed::kRing].count;
        if (rows0 < count) expand(smem + stage * Tile::kStage, n - at * KC, list[slot % SlotFeed::kRing], count);
        ring.left(stage);
        if (++stage == S) stage = 0, round ^= 1;
        if (++at == per) at = 0, ++slot;
    }
    const AdapterSlot* last = plan_busy(P) + plan_slots(P.rows, P.adapters) - 1;
    for (int i = blockIdx.x; i < idle * kParts; i += gridDim.x) {
        const AdapterSlot s = last[-(i / kParts)];
        named_barrier<kWorkBarrier, kTileThreads>();
        if (tid < s.count) plain[tid] = plan_perm(P)[s.start + tid];
        named_barrier<kWorkBarrier, kTileThreads>();
        plain_rows<T>(P, plain, s.count, s.cls != P.adapters, min(i % kParts * width, n), min((i % kParts + 1) * width, n));
    }
}

// Gradients of the factors: grad[i][j][c] = sum over the rows t of adapter i of
// p[t][j] * q[t][c], dA from (v, x) and dB from (u, dy), in one launch.
//
// A block holds a stretch of columns and all of the rank in registers and walks
// the adapter's rows, so q is read once and p (rank values a row) by every block
// of columns.  Where that gives too few blocks, a cluster splits the rows into
// consecutive parts, whose sums meet in the blocks' order; where a cluster of eight is
// still too little, the rows come in segments, a cluster each, whose sums meet in the
// forward pass's workspace.
//
// Bound by the bytes of x and dy on paper; measured, 16384 x 4096 bfloat16, rank 32,
// four adapters: 126 us for the 268 MB of both, 2.1 TB/s, with the warps waiting for
// their loads from shared memory and for one another in turn (with p in two parts, 16
// bits of it, 96 us); a million rows, 32
// columns to 32, rank 8, one adapter: 157 us for 192 MB.  The ring of the products, with two
// copying warps, was no faster here and slower for rows in any order (3333 x 1024
// bfloat16 rank 20, p in two parts: 35 us against 18), whose copies two warps cannot issue fast enough.
constexpr int kGradThreads = 128;
constexpr int kGradCluster = 8;  // the most blocks whose sums meet in a cluster

struct AdapterGradSide {
    const void* p;  // [rows, p_row], as the products left it
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
    void* parts;  // with several segments of the rows: their sums, laid out like the gradients
};

// The values of the first `sides` gradients that are wanted.
__host__ __device__ inline int64_t grad_values(const AdapterGradParams& P, int sides) {
    int64_t v = 0;
    for (int i = 0; i < sides; ++i) v += P.side[i].grad ? (int64_t)P.adapters * P.r * P.side[i].cols : 0;
    return v;
}

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
    static constexpr int kStages = 3;  // a fourth leaves room for fewer blocks: 3333 x 1023 -> 515 floats, 24 us for 20
    static constexpr int kPitchD = RP + 1;                    // the block's sums, after the rows
    static constexpr int kJoin = COLS * kPitchD * (int)sizeof(Acc);
    // bfloat16: p as three parts, split where it was copied to, a pair of rows to a word.  The first
    // parts of rows 2 j and 2 j + 1 take row 2 j's place, the second ones row 2 j + 1's; the third
    // ones have a place of their own, for two chunks.
    static constexpr bool kPairs = std::is_same<T, __nv_bfloat16>::value;
    static constexpr int kPitchL = (RP + 8) * 4, kThird = kPairs ? KT / 2 * kPitchL : 0;
    static constexpr int kRing = kStages * kStage + 2 * kThird;
    static constexpr int kSmem = kRing > kJoin ? kRing : kJoin;
    // Chunks that the (truncating) tensor cores sum by themselves: of 16-bit data 4 (8 moved a fifth
    // more results to a neighbouring bfloat16, in 125 us for 126).
    static constexpr int kFlush = E == 2 ? 4 : 1;
};

template <typename T, int RP>
__global__ void __launch_bounds__(kGradThreads) adapter_grad_kernel(const __grid_constant__ AdapterGradParams P) {
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
    const int ways = cs * (int)gridDim.z, way = (int)blockIdx.z * cs + cr;
    const int share = (int)(((int64_t)rows + KT * ways - 1) / (KT * ways) * KT);
    const int t0 = (int64_t)way * share < rows ? way * share : rows, t1 = t0 + share < rows ? t0 + share : rows;
    const int chunks = (t1 - t0 + KT - 1) / KT;
    const T* qs = static_cast<const T*>(side.q);
    const Acc* ps = static_cast<const Acc*>(side.p);
    const int vec = copy_unit<T>(qs, side.q_row);

    // A thread's copies of a chunk: 16 bytes of QI rows of q, 16 of PI rows of p, each at one place along
    // the row.  Every warp reads the chunk's row ids, one chunk ahead of the copies that need them.
    constexpr int QU = COLS / V, QI = KT * QU / kGradThreads, QS = kGradThreads / QU;
    constexpr int PV = 16 / (int)sizeof(Acc), PU = RP / PV, PS = kGradThreads / PU;
    constexpr int PI = KT * PU <= kGradThreads && Tile::kPairs ? 2 : KT * PU / kGradThreads;
    // The row of p of a thread's copy i; in pairs, of the first half of the threads alone for the smallest rank.
    auto p_row_of = [&](int i) { return Tile::kPairs ? tid / PU * 2 + i % 2 + i / 2 * 2 * PS : tid / PU + i * PS; };
    const int64_t col = c0 + tid % QU * V, cols_left = side.cols - col;
    const int q_avail = cols_left < 0 ? 0 : cols_left > V ? V : (int)cols_left;
    const int p_bytes = tid % PU * PV < P.p_row ? 16 : 0;  // p_row is a multiple of PV
    const Acc* pc = ps + tid % PU * PV;
    int id = 0;
    auto ids = [&](int c) {
        const int t = t0 + c * KT + lane;
        id = lane < KT && t < t1 ? perm[t] : -1;
    };
    auto fetch = [&](int c) {
        uint8_t* st = smem + c % S * Tile::kStage;
#pragma unroll
        for (int i = 0; i < QI; ++i) {
            const int r = __shfl_sync(0xffffffffu, id, tid / QU + i * QS);
            fetch16(st + (tid / QU + i * QS) * Tile::kPitchQ + tid % QU * 16, qs + r * side.q_row + col,
                    r < 0 ? 0 : q_avail, vec);
        }
#pragma unroll
        for (int i = 0; i < PI; ++i) {
            const int row = p_row_of(i), r = __shfl_sync(0xffffffffu, id, row & 31);
            if (row < KT)
                copy16(shared_address(st + KT * Tile::kPitchQ + row * Tile::kPitchP + tid % PU * 16),
                       pc + (int64_t)r * P.p_row, r < 0 ? 0 : p_bytes);
        }
    };
    // A chunk's p in parts: each thread what it copied itself, before the others look at it.  (Every
    // warp splitting the operands that it loads: 147 us in the training case above for 126.)
    auto split = [&](int c) {
        if constexpr (Tile::kPairs) {
            uint8_t* pt = smem + c % S * Tile::kStage + KT * Tile::kPitchQ + tid % PU * 16;
            uint8_t* third = smem + S * Tile::kStage + (c & 1) * Tile::kThird + tid % PU * 16;
#pragma unroll
            for (int i = 0; i < PI; i += 2) {
                const int row = p_row_of(i);
                if (row >= KT) break;
                alignas(16) float a[4], b[4];
                uint32_t part[4][3];
                *reinterpret_cast<float4*>(a) = *reinterpret_cast<const float4*>(pt + row * Tile::kPitchP);
                *reinterpret_cast<float4*>(b) = *reinterpret_cast<const float4*>(pt + (row + 1) * Tile::kPitchP);
#pragma unroll
                for (int e = 0; e < 4; ++e) split_bf16(a[e], b[e], part[e]);
                auto store = [&](uint8_t* to, int k) {
                    *reinterpret_cast<uint4*>(to) = make_uint4(part[0][k], part[1][k], part[2][k], part[3][k]);
                };
                store(pt + row * Tile::kPitchP, 0);
                store(pt + (row + 1) * Tile::kPitchP, 1);
                store(third + row / 2 * Tile::kPitchL, 2);
            }
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
    auto compute = [&](int chunk) {
        const uint8_t *st = smem + chunk % S * Tile::kStage, *pt = st + KT * Tile::kPitchQ;
        const uint8_t* third = smem + S * Tile::kStage + (chunk & 1) * Tile::kThird;
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
                // Two 8-rank tiles at a time: rank 2 n + t of 16 stands where the instruction has column n of
                // tile t, so that one 8-byte load serves both.
#pragma unroll
                for (int t = 0; t < RP / 16; ++t) {
                    if constexpr (Tile::kPairs) {
                        uint2 w[3][2];  // part; rows 2 q and 2 q + 1, then 8 on; .x for tile 2 t, .y for 2 t + 1
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const int pair = ks * 8 + i * 4 + q, at = (t * 16 + 2 * g) * 4;
                            w[0][i] = *reinterpret_cast<const uint2*>(pt + 2 * pair * Tile::kPitchP + at);
                            w[1][i] = *reinterpret_cast<const uint2*>(pt + (2 * pair + 1) * Tile::kPitchP + at);
                            w[2][i] = *reinterpret_cast<const uint2*>(third + pair * Tile::kPitchL + at);
                        }
#pragma unroll
                        for (int i = 2; i >= 0; --i)
#pragma unroll
                            for (int m = 0; m < MT; ++m) {
                                mma16<T>(sum[m][2 * t], a[m], w[i][0].x, w[i][1].x);
                                mma16<T>(sum[m][2 * t + 1], a[m], w[i][0].y, w[i][1].y);
                            }
                    } else {
                        uint2 w[2][2];  // rows 2 q, 2 q + 1, then 8 on; .x for tile 2 t, .y for 2 t + 1
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            w[e >> 1][e & 1] = *reinterpret_cast<const uint2*>(
                                pt + (ks * 16 + 2 * q + (e >> 1) * 8 + (e & 1)) * Tile::kPitchP + (t * 16 + 2 * g) * 4);
                        // A half is a tf32 value as it is; the middle, whose range is a float's, is split in two.
                        // The order of rows within the sum is free: rows 2q and 2q + 1 stand where the
                        // instruction has q and q + 4.
#pragma unroll
                        for (int k8 = 0; k8 < 2; ++k8)
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const Tf32Pair b0 = tf32_split(__uint_as_float(h ? w[k8][0].y : w[k8][0].x));
                                const Tf32Pair b1 = tf32_split(__uint_as_float(h ? w[k8][1].y : w[k8][1].x));
#pragma unroll
                                for (int m = 0; m < MT; ++m) {
                                    const float2 f0 = __half22float2(*reinterpret_cast<const __half2*>(&a[m][2 * k8]));
                                    const float2 f1 = __half22float2(*reinterpret_cast<const __half2*>(&a[m][2 * k8 + 1]));
                                    const uint32_t x[4] = {__float_as_uint(f0.x), __float_as_uint(f1.x),
                                                           __float_as_uint(f0.y), __float_as_uint(f1.y)};
                                    mma_tf32(sum[m][2 * t + h], x, b0.lo, b1.lo);
                                    mma_tf32(sum[m][2 * t + h], x, b0.hi, b1.hi);
                                }
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
        split(c);
        __syncthreads();
        if (c + S - 1 < chunks) {
            fetch(c + S - 1);
            ids(c + S);
        }
        copy_commit();
        compute(c);
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
                mine[((warp * MT + m) * 16 + g + (e >> 1) * 8) * Tile::kPitchD +
                     (E == 2 ? t / 2 * 16 + 2 * (2 * q + (e & 1)) + t % 2 : t * 8 + 2 * q + (e & 1))] = acc[m][t][e];
    cluster.sync();
    const Acc* parts[kGradCluster];
#pragma unroll
    for (int b = 0; b < kGradCluster; ++b) parts[b] = b < cs ? cluster.map_shared_rank(mine, b) : nullptr;
    const int cols = side.cols - c0 < COLS ? (int)(side.cols - c0) : COLS, own = COLS / cs;
    const int first = cr * own, last = first + own < cols ? first + own : cols;
    const int64_t at = (int64_t)cls * P.r * side.cols;
    T* grad = static_cast<T*>(side.grad) + at;
    Acc* part = nullptr;
    if (gridDim.z > 1)
        part = static_cast<Acc*>(P.parts) + grad_values(P, 2) * blockIdx.z + (second ? grad_values(P, 1) : 0) + at;
    const int many = last > first ? (last - first) * P.r : 0;
    for (int i = tid; i < many; i += kGradThreads) {
        const int c = first + (side.by_column ? i / P.r : i % (last - first));
        const int j = side.by_column ? i % P.r : i / (last - first);
        Acc v = 0;
#pragma unroll
        for (int b = 0; b < kGradCluster; ++b)
            if (b < cs) v += parts[b][c * Tile::kPitchD + j];
        const int64_t o = side.by_column ? (c0 + c) * P.r + j : j * side.cols + c0 + c;
        if (part)
            part[o] = v;
        else
            grad[o] = narrow<T>(v);
    }
    cluster.sync();
}

// Adds the segments' sums in their order.
template <typename T>
__global__ void __launch_bounds__(256) adapter_grad_join_kernel(const __grid_constant__ AdapterGradParams P, int segments) {
    using Acc = typename AccOf<T>::type;
    const int64_t first = grad_values(P, 1), all = grad_values(P, 2);
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < all; i += (int64_t)gridDim.x * blockDim.x) {
        const Acc* p = static_cast<const Acc*>(P.parts) + i;
        Acc v = 0;
#pragma unroll 8
        for (int s = 0; s < segments; ++s) v += p[s * all];
        static_cast<T*>(P.side[i >= first].grad)[i >= first ? i - first : i] = narrow<T>(v);
    }
}

}  // namespace fpemu
