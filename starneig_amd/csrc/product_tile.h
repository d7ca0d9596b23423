// The tile of the grouped and the 8-bit products: BM x BN outputs of one workgroup from the matrix cores, operands through LDS.
//
// A k-tile is 128 bytes of the inner index (64 numbers of 16 bits, 128 of 8).  An operand lies in memory with the inner index
// contiguous ("K": weights of a forward product, tokens) or with the outer index contiguous (weights of an input
// gradient, both operands of a weight gradient); LDS holds a straight copy of what is contiguous, in 16-byte chunks:
//   K:  [outer][8 chunks of inner],          chunk c of row r at place c ^ swizzle_k(r); fragments by ds_read_b128
//   MN: [64 inner rows][outer / 8 chunks],   chunk c of row k at place c ^ swizzle_mn(k); fragments by ds_read_b64_tr_b16, which
//       hands lane i of 16 the four numbers of its column out of four rows
// Both leave the fragment reads without bank conflicts.
//
// Outer index of lane i of a fragment: the four fragments t of 64 rows interleave, row = 16 (i >> 2) + 4 t + (i & 3).  The accumulators of the four
// fragments then hold 16 consecutive rows of a column per lane, and a column's 64 rows are stored as whole lines.
#pragma once
#include "product_types.h"

namespace sn {

typedef short s16x4 __attribute__((ext_vector_type(4)));

// How an operand is brought into LDS: DIRECT = buffer loads that write LDS themselves (16-byte aligned columns, whole chunks), no registers and
// no LDS instructions; STAGED = through registers, any alignment and any extent.
enum Feed { DIRECT, STAGED };

template <typename T, int ROWS, bool K, int THREADS>
struct Operand {
    static constexpr int EL = 16 / (int)sizeof(T);          // numbers a chunk
    static constexpr int KT = 128 / (int)sizeof(T);         // inner terms a k-tile
    static constexpr int BYTES = ROWS * 128;
    static constexpr int LOADS = ROWS * 8 / THREADS;        // chunks a thread brings
    static constexpr int CR = ROWS / EL;                    // MN: chunks a row

    static __device__ __forceinline__ int swizzle_k(int r) { return (r & 3) | (r >> 2 & 4); }
    static __device__ __forceinline__ int swizzle_mn(int k) { return (k & 1) | (k & 2) << 2; }

    // outer and inner position, inside the tile, of the chunk that goes to place e
    static __device__ __forceinline__ void chunk(int e, int &outer, int &inner)
    {
        if (K) { outer = e >> 3; inner = ((e & 7) ^ swizzle_k(outer)) * EL; }
        else   { inner = e / CR; outer = ((e % CR) ^ swizzle_mn(inner)) * EL; }
    }

    // fragment t of the 64 rows from `row0`, 64 bytes of inner index number `half`
    static __device__ __forceinline__ i32x4 fragment(char const *lds, int row0, int t, int half)
    {
        int const lane = threadIdx.x & 63, i = lane & 15, q = lane >> 4;
        if constexpr (K) {
            int const r = row0 + 16 * (i >> 2) + 4 * t + (i & 3), c = half * 4 + q;
            return *(i32x4 const *)(lds + r * 128 + ((c ^ swizzle_k(r)) << 4));
        } else {
            // lane 4 j + c of the 16 names four numbers of row j: rows 16 c + 4 t ...; it gets column i = 4 c' + e of all four
            int const j = i >> 2, c = i & 3;
            u32x2 part[2];
            #pragma unroll
            for (int h = 0; h < 2; h++) {
                int const k = half * 32 + 8 * q + 4 * h + j, outer = row0 + 16 * c + 4 * t;
                char const *const at = lds + k * (ROWS * 2) + (((outer >> 3) ^ swizzle_mn(k)) << 4) + (outer & 4) * 2;
                part[h] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(at)));
            }
            return (i32x4){(int)part[0].x, (int)part[0].y, (int)part[1].x, (int)part[1].y};
        }
    }
};

// One operand of one tile on its way into LDS.  `base`: its element (outer 0, inner 0) of the tile; `outers`: how many outer positions
// exist from there (may exceed ROWS); `k`: inner terms in all; `ld`: distance of the positions that are not contiguous.
template <typename T, int ROWS, bool K, int THREADS, Feed FEED> struct Stream;

template <typename T, int ROWS, bool K, int THREADS>
struct Stream<T, ROWS, K, THREADS, DIRECT> {
    using O = Operand<T, ROWS, K, THREADS>;
    T const *base;
    long step;                      // MN: numbers between k-tiles
    int k;
    unsigned at[O::LOADS];          // byte offsets of the thread's chunks; beyond the buffer where there is nothing to read
    int inner[K ? 1 : O::LOADS];

    __device__ __forceinline__ Stream(T const *base_, int outers, int k_, long ld) : base(base_), step(ld * O::KT), k(k_)
    {
        #pragma unroll
        for (int s = 0; s < O::LOADS; s++) {
            int outer, in;
            O::chunk(s * THREADS + threadIdx.x, outer, in);
            if (K) { at[s] = outer < outers ? (unsigned)(outer * (int)(ld * sizeof(T)) + in * (int)sizeof(T)) : 0x80000000u; inner[0] = in; }
            else   { at[s] = outer < outers ? (unsigned)(in * (int)(ld * sizeof(T)) + outer * (int)sizeof(T)) : 0x80000000u; inner[K ? 0 : s] = in; }
        }
    }
    // starts bringing k-tile kt to `lds`.  Offsets from 2^31 on read zeros (the buffer's length is 2^31 - 1): positions past the outer
    // end, and inner chunks past k.
    __device__ __forceinline__ void fetch(char *lds, int kt) const
    {
        T const *const from = K ? base + (long)kt * O::KT : base + kt * step;
        __amdgpu_buffer_rsrc_t const r = __builtin_amdgcn_make_buffer_rsrc((void *)from, 0, 0x7fffffff, 0x00020000);
        int const left = k - kt * O::KT;
        #pragma unroll
        for (int s = 0; s < O::LOADS; s++) {
            unsigned v = at[s];
            if (left < O::KT) v = inner[K ? 0 : s] < left ? v : 0x80000000u;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void *)(lds + (s * THREADS + (int)(threadIdx.x & ~63u)) * 16),
                16, (int)v, 0, 0, 0);
        }
    }
    __device__ __forceinline__ void put(char *) const {}
};

template <typename T, int ROWS, bool K, int THREADS>
struct Stream<T, ROWS, K, THREADS, STAGED> {
    using O = Operand<T, ROWS, K, THREADS>;
    T const *base;
    long ld;
    int outers, k;
    i32x4 held[O::LOADS];

    __device__ __forceinline__ Stream(T const *base_, int outers_, int k_, long ld_) : base(base_), ld(ld_), outers(outers_), k(k_) {}

    __device__ __forceinline__ void fetch(char *, int kt)
    {
        int const left = k - kt * O::KT;
        T const *const from = K ? base + (long)kt * O::KT : base + (long)kt * O::KT * ld;
        #pragma unroll
        for (int s = 0; s < O::LOADS; s++) {
            int outer, inner;
            O::chunk(s * THREADS + threadIdx.x, outer, inner);
            // (whole chunks by one load from wherever they start; a chunk that the end cuts, number by number)
            bool const whole = K ? inner + O::EL <= left && outer < outers : outer + O::EL <= outers && inner < left;
            T const *const p = K ? from + outer * ld + inner : from + inner * ld + outer;
            i32x4 v = {0, 0, 0, 0};
            if (whole) __builtin_memcpy(&v, p, 16);
            else {
                int const rest = K ? (outer < outers ? left - inner : 0) : (inner < left ? outers - outer : 0);
                T one[O::EL];
                #pragma unroll
                for (int e = 0; e < O::EL; e++) one[e] = e < rest ? p[e] : (T)0;
                __builtin_memcpy(&v, one, 16);
            }
            held[s] = v;
        }
    }
    __device__ __forceinline__ void put(char *lds) const
    {
        #pragma unroll
        for (int s = 0; s < O::LOADS; s++) *(i32x4 *)(lds + (s * THREADS + threadIdx.x) * 16) = held[s];
    }
};

template <typename T, int BM_, int BN_, int WAVES_M_, int WAVES_N_, bool AK_, bool BK_, Feed FEED_>
struct ProductTile {
    static constexpr int BM = BM_, BN = BN_, WAVES_M = WAVES_M_, WAVES_N = WAVES_N_, THREADS = 64 * WAVES_M * WAVES_N;
    static constexpr int MB = BM / WAVES_M / 64, NB = BN / WAVES_N / 64;     // 64 x 64 blocks a wave
    typedef typename Mfma<T>::Acc Acc;
    using OA = Operand<T, BM, AK_, THREADS>;
    using OB = Operand<T, BN, BK_, THREADS>;
    static constexpr int STAGE = OA::BYTES + OB::BYTES, LDS_BYTES = 2 * STAGE;
    static constexpr int KT = OA::KT;
    static constexpr bool A_K = AK_;

    Acc acc[MB][4][NB][4];

    __device__ __forceinline__ void multiply(char const *lds)
    {
        int const wave = threadIdx.x >> 6, m0 = wave % WAVES_M * (BM / WAVES_M), n0 = wave / WAVES_M * (BN / WAVES_N);
        #pragma unroll
        for (int half = 0; half < 2; half++) {
            // (one half's fragments at a time: without it both are loaded first, and the 256 x 256 tile spills)
            if (half) __builtin_amdgcn_sched_barrier(0);
            i32x4 a[MB][4], b[NB][4];
            #pragma unroll
            for (int y = 0; y < NB; y++)
                #pragma unroll
                for (int t = 0; t < 4; t++) b[y][t] = OB::fragment(lds + OA::BYTES, n0 + 64 * y, t, half);
            #pragma unroll
            for (int x = 0; x < MB; x++)
                #pragma unroll
                for (int t = 0; t < 4; t++) a[x][t] = OA::fragment(lds, m0 + 64 * x, t, half);
            #pragma unroll
            for (int x = 0; x < MB; x++)
                #pragma unroll
                for (int t = 0; t < 4; t++)
                    #pragma unroll
                    for (int y = 0; y < NB; y++)
                        #pragma unroll
                        for (int u = 0; u < 4; u++) acc[x][t][y][u] = Mfma<T>::mul(a[x][t], b[y][u], acc[x][t][y][u]);
        }
    }

    // acc = sum over the k inner terms; rows / cols: outputs that exist from the tile's corner on
    __device__ __forceinline__ void run(T const *A, long lda, int rows, T const *B, long ldb, int cols, int k, char *lds)
    {
        Stream<T, BM, AK_, THREADS, FEED_> a(A, rows, k, lda);
        Stream<T, BN, BK_, THREADS, FEED_> b(B, cols, k, ldb);
        #pragma unroll
        for (int x = 0; x < MB; x++)
            #pragma unroll
            for (int t = 0; t < 4; t++)
                #pragma unroll
                for (int y = 0; y < NB; y++)
                    #pragma unroll
                    for (int u = 0; u < 4; u++) acc[x][t][y][u] = Acc{};
        int const tiles = (k + KT - 1) / KT;
        if (tiles == 0) return;
        a.fetch(lds, 0); b.fetch(lds + OA::BYTES, 0);
        a.put(lds); b.put(lds + OA::BYTES);
        landed();
        int now = 0;
        for (int kt = 0; kt < tiles; kt++) {
            // (past the last k-tile the fetch reads nothing and leaves zeros)
            int const next = now ^ STAGE;
            a.fetch(lds + next, kt + 1); b.fetch(lds + next + OA::BYTES, kt + 1);
            multiply(lds + now);
            a.put(lds + next); b.put(lds + next + OA::BYTES);
            landed();
            now = next;
        }
    }

    // every wave's part of the next k-tile is in LDS, and every wave is done with this one's
    static __device__ __forceinline__ void landed()
    {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    }

    // f(row, column, 16 accumulators of consecutive rows) for every column of the lane's; rows and columns count from the tile's corner
    template <typename F>
    __device__ __forceinline__ void each(F &&f)
    {
        int const lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, q = lane >> 4;
        int const m0 = wave % WAVES_M * (BM / WAVES_M), n0 = wave / WAVES_M * (BN / WAVES_N);
        #pragma unroll
        for (int x = 0; x < MB; x++)
            #pragma unroll
            for (int y = 0; y < NB; y++)
                #pragma unroll
                for (int u = 0; u < 4; u++) {
                    auto const v = [&](int r) { return acc[x][r >> 2][y][u][r & 3]; };
                    f(m0 + 64 * x + 16 * q, n0 + 64 * y + 16 * (i >> 2) + 4 * u + (i & 3), v);
                }
    }
};

// 16 consecutive numbers of a column, `rows` of which exist; value(r) gives them
template <typename D, typename V>
__device__ __forceinline__ void store16(D *to, int rows, bool aligned, V &&value)
{
    constexpr int EL = 16 / (int)sizeof(D);
    if (rows >= 16 && aligned) {
        #pragma unroll
        for (int c = 0; c < 16 / EL; c++) {
            D one[EL];
            #pragma unroll
            for (int e = 0; e < EL; e++) one[e] = (D)value(c * EL + e);
            i32x4 v;
            __builtin_memcpy(&v, one, 16);
            *(i32x4 *)(to + c * EL) = v;
        }
        return;
    }
    #pragma unroll
    for (int r = 0; r < 16; r++)
        if (r < rows) to[r] = (D)value(r);
}

} // namespace sn
