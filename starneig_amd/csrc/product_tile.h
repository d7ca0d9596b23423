// The tile of the grouped and the 8-bit products: BM x BN outputs of one workgroup from the matrix cores, operands through LDS.
//
// A k-tile is 128 bytes of the inner index (64 numbers of 16 bits, 128 of 8): a cache line.  An operand lies in memory with the inner index
// contiguous ("K": weights of a forward product, tokens) or with the outer index contiguous ("MN": weights of an input
// gradient, both operands of a weight gradient); LDS holds a straight copy of what is contiguous, in 16-byte chunks:
//   K:  [outer][8 chunks of inner],          chunk c of row r at place c ^ swizzle_k(r); fragments by ds_read_b128
//   MN: [64 inner rows][outer / 8 chunks],   chunk c of row k at place c ^ swizzle_mn(k); fragments by ds_read_b64_tr_b16, which
//       hands lane i of 16 the four numbers of its column out of four rows
// Both leave the fragment reads without bank conflicts.
//
// The two fragments t of 64 rows interleave.  K: lane i holds row 8 (i >> 2) + 4 t + (i & 3), so that the accumulators of the two hold eight
// consecutive rows of a column per lane.  MN: row 32 t + i, whose reads touch every bank; four consecutive rows per lane.
#pragma once
#include "product_types.h"

namespace sn {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) char lds_char;
typedef __attribute__((address_space(3))) i32x4 lds_i32x4;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// How an operand is brought into LDS: DIRECT = buffer loads that write LDS themselves (columns aligned to 4 bytes), no registers and
// no LDS instructions; STAGED = through registers, any alignment.
enum Feed { DIRECT, STAGED };

// A buffer of `bytes` bytes from `p` on: loads from offsets beyond it give zeros.
__device__ __forceinline__ i32x4 buffer(void const *p, int bytes)
{
    unsigned long long const at = (unsigned long long)p;
    return (i32x4){__builtin_amdgcn_readfirstlane((int)at), __builtin_amdgcn_readfirstlane((int)(at >> 32) & 0xffff), bytes, 0x00020000};
}
// 16 bytes a lane from `offset` of the buffer into LDS: the wave's from `to` (the same in all lanes) on, in the lanes' order.  In assembly: with the
// builtin the compiler waits for all loads before the next transposing LDS read, which it takes to read what they write; here the
// barriers order them.  The compiler does not look inside, so the five wait states are here that a load needs behind a vector
// instruction (v_readfirstlane) that has written one of its scalar registers, and the one behind m0.  m0 is named as written, so that no
// value of the compiler's own is taken to outlast the statement (it warns that it never allocates m0, which holds).
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void load_to_lds(i32x4 buffer, unsigned offset, int to)
{
    i32x4 const b = {uniform(buffer.x), uniform(buffer.y), uniform(buffer.z), uniform(buffer.w)};
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" :: "s"(uniform(to)), "v"(offset), "s"(b) : "m0", "memory");
}
#pragma clang diagnostic pop
// threadIdx.x for what is computed once a tile: the compiler must not compute it before the loops and hold it in registers meanwhile
__device__ __forceinline__ int thread_now() { int t = threadIdx.x; asm volatile("" : "+v"(t)); return t; }
// number of the wave, of the threads that share a tile
__device__ __forceinline__ int wave_number() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

// THREADS: how many bring the operand together, the workgroup's or a wave's
template <typename T, int ROWS, bool K, int THREADS>
struct Operand {
    static constexpr int EL = 16 / (int)sizeof(T);          // numbers a chunk
    static constexpr int KT = 128 / (int)sizeof(T);         // inner terms a k-tile
    static constexpr int BYTES = ROWS * 128;
    static constexpr int LOADS = ROWS * 8 / THREADS;        // chunks a thread brings
    static constexpr int CR = ROWS / EL;                    // MN: chunks a row

    // (ds_read_b128 serves 16 lanes at a time: 0-3, 12-15, 20-27; 4-11, 16-19, 28-31; and so on; ds_read_b64_tr_b16 32)
    static __host__ __device__ __forceinline__ int swizzle_k(int r) { return sizeof(T) == 8 ? r >> 1 & 7 : (r >> 1 & 1) | (r >> 3 & 6); }
    static __host__ __device__ __forceinline__ int swizzle_mn(int k) { return sizeof(T) == 8 ? 0 : CR >= 16 ? (k & 3) << 2 : (k & 2) << 1; }

    // row of lane i of fragment t of 64 rows
    static __device__ __forceinline__ int row(int i, int t) { return K ? 8 * (i >> 2) + 4 * t + (i & 3) : 32 * t + i; }

    // outer and inner position, inside the tile, of the chunk that goes to place e
    static __host__ __device__ __forceinline__ void chunk(int e, int &outer, int &inner)
    {
        if (K) { outer = e >> 3; inner = ((e & 7) ^ swizzle_k(outer)) * EL; }
        else   { inner = e / CR; outer = ((e % CR) ^ swizzle_mn(inner)) * EL; }
    }

    // K, a k-tile in LDS of which `left` inner terms exist: zeroes those behind them in the chunk that k cuts (it brought whatever lay there)
    static __device__ __forceinline__ void trim(lds_char *lds, int left)
    {
        i32x4 mask;
        #pragma unroll
        for (int w = 0; w < 4; w++) {
            int const bits = min(max(left % EL * 8 * (int)sizeof(T) - 32 * w, 0), 32);
            mask[w] = bits == 32 ? -1 : (int)((1u << bits) - 1);
        }
        for (int r = thread_now() % THREADS; r < ROWS; r += THREADS) {
            lds_i32x4 *const at = (lds_i32x4 *)(lds + r * 128 + ((left / EL ^ swizzle_k(r)) << 4));
            *at = *at & mask;
        }
    }

    // fp64: the fragments t of 32 rows from `row0` for two instructions e, which take the inner terms 8 half + 2 q + e of the lanes with q = lane >> 4: two
    // 16-byte reads, of two inner terms (K) or of the two fragments' rows (MN) each
    static __device__ __forceinline__ int double_row(int i, int t) { return K ? 16 * t + i : 2 * i + t; }
    static __device__ __forceinline__ void doubles(lds_char const *lds, int row0, int half, double (&f)[2][2])
    {
        typedef double d2 __attribute__((ext_vector_type(2)));
        typedef __attribute__((address_space(3))) d2 lds_d2;
        int const lane = threadIdx.x & 63, i = lane & 15, q = lane >> 4;
        #pragma unroll
        for (int x = 0; x < 2; x++) {
            int const r = row0 + 16 * x + i, k = 8 * half + 2 * q + x;
            d2 const v = *(lds_d2 const *)(K ? lds + r * 128 + ((4 * half + q ^ swizzle_k(r)) << 4) : lds + k * (ROWS * 8) + (row0 / 2 + i) * 16);
            (K ? f[0][x] : f[x][0]) = v.x;
            (K ? f[1][x] : f[x][1]) = v.y;
        }
    }

    // fragment t of the 64 rows from `row0`, 32 bytes of inner index number `step` of 4
    static __device__ __forceinline__ i32x4 fragment(lds_char const *lds, int row0, int t, int step)
    {
        int const lane = threadIdx.x & 63, q = lane >> 5;
        if constexpr (K) {
            int const r = row(lane & 31, t);
            return *(lds_i32x4 const *)(lds + (row0 + r) * 128 + (((2 * step + q) ^ swizzle_k(r)) << 4));
        } else {
            // lane 4 j + c of 16 names four numbers of row j of four; it gets its own column's of all four rows
            int const j = lane >> 2 & 3, c = lane & 3, outer = row0 + row((lane & 16) + 4 * c, t);
            u32x2 part[2];
            #pragma unroll
            for (int h = 0; h < 2; h++) {
                int const k = 16 * step + 8 * q + 4 * h + j;
                lds_char const *const at = lds + k * (ROWS * 2) + (((outer >> 3) ^ swizzle_mn(k)) << 4) + (outer & 4) * 2;
                part[h] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)at));
            }
            return (i32x4){(int)part[0].x, (int)part[0].y, (int)part[1].x, (int)part[1].y};
        }
    }
};

// One operand on its way into LDS, tile after tile.  set(): `base`: its element (outer 0, inner 0) of the tile; `outers`: how many outer positions
// exist from there (may exceed ROWS); `k`: inner terms in all; `ld`: distance of the positions that are not contiguous.
template <typename T, int ROWS, bool K, int THREADS, Feed FEED> struct Stream;

template <typename T, int ROWS, bool K, int THREADS>
struct Stream<T, ROWS, K, THREADS, DIRECT> {
    using O = Operand<T, ROWS, K, THREADS>;
    T const *base;
    long step;                      // MN: numbers between k-tiles
    int k, ld, outers;
    unsigned at[O::LOADS];          // byte offsets of the thread's chunks

    // Which bytes a k-tile's loads read; the tests compute them on the host.  Offsets from 2^31 on read zeros.
    static constexpr unsigned NOTHING = 0x80000000u;
    // Where chunk e of a tile lies: nowhere if it is past the outer end.
    static __host__ __device__ __forceinline__ unsigned offset(int e, int outers, int ld)
    {
        int outer, inner;
        O::chunk(e, outer, inner);
        return outer < outers ? (unsigned)(((K ? outer : inner) * ld + (K ? inner : outer)) * (int)sizeof(T)) : NOTHING;
    }
    // Whether chunk e lies behind the `left` inner terms that there are from this k-tile's first on.
    static __host__ __device__ __forceinline__ bool behind(int e, int left)
    {
        int outer, inner;
        O::chunk(e, outer, inner);
        return inner >= left;
    }
    // The bytes of the buffer: up to the last word of the operand (words, four bytes: the hardware tests each), where a chunk may reach it.  In the
    // last k-tile that is a chunk that starts in front of the end; MN, where a chunk is wider than the leading dimension, also one of the rows in front
    // of them, which covers the next rows' numbers: up to EL rows.  Behind the last k-tile, and without outer positions, the buffer is empty.
    static constexpr int REACH = K ? O::KT : O::KT + O::EL, WHOLE = 0x7fffffff;
    static __host__ __device__ __forceinline__ int bytes(int left, int outers, int ld)
    {
        if (left > REACH) return WHOLE;
        if (left <= 0 || outers <= 0) return 0;
        int const rows = outers < ROWS ? outers : ROWS, wide = outers < ROWS + O::EL ? outers : ROWS + O::EL;
        return (K ? (rows - 1) * ld + left : (left - 1) * ld + wide) * (int)sizeof(T) + 3 & ~3;
    }

    __device__ __forceinline__ void set(T const *base_, int outers_, int k_, long ld_)
    {
        base = base_; k = k_; ld = (int)ld_; outers = outers_; step = ld_ * O::KT;
        int const thread = thread_now() % THREADS;
        #pragma unroll
        for (int s = 0; s < O::LOADS; s++) at[s] = offset(s * THREADS + thread, outers, ld);
    }
    // Loads 0 ... LOADS - 1 of k-tile kt to `lds`, after begin(kt); k-tiles are fetched in order.
    i32x4 from;
    __device__ __forceinline__ void begin(int kt)
    {
        int const left = k - kt * O::KT;
        int size = WHOLE;
        if (left <= REACH) {            // (one branch in all other k-tiles)
            size = bytes(left, outers, ld);
            if (left <= O::KT) {
                int const thread = thread_now() % THREADS;
                #pragma unroll
                for (int s = 0; s < O::LOADS; s++)
                    if (behind(s * THREADS + thread, left)) at[s] = NOTHING;
            }
        }
        from = buffer(K ? base + (long)kt * O::KT : base + kt * step, size);
    }
    __device__ __forceinline__ void load(int lds, int s) const { load_to_lds(from, at[s], lds + wave_number() % (THREADS / 64) * 1024 + s * THREADS * 16); }
    __device__ __forceinline__ void fetch(int lds, int kt)
    {
        begin(kt);
        #pragma unroll
        for (int s = 0; s < O::LOADS; s++) load(lds, s);
    }
};

// 16 bytes of global memory from any address
__device__ __forceinline__ i32x4 load16(void const *p)
{
    typedef int any_i32x4 __attribute__((ext_vector_type(4), aligned(1)));
    return *(__attribute__((address_space(1))) any_i32x4 const *)p;
}

// v moved down by `bits`, zeros from above
__device__ __forceinline__ i32x4 moved_down(i32x4 v, int bits)
{
    typedef unsigned long long u64x2 __attribute__((ext_vector_type(2)));
    u64x2 w = __builtin_bit_cast(u64x2, v);
    if (bits >= 64) { w.x = w.y; w.y = 0; bits -= 64; }
    if (bits >= 64) w.x = 0;
    else if (bits > 0) { w.x = w.x >> bits | w.y << (64 - bits); w.y >>= bits; }
    return __builtin_bit_cast(i32x4, w);
}

// Every load is of a whole chunk inside the operand: positions that are not there read others in their place, and a chunk that the end
// cuts is read from where it ends there (the operand has a chunk of contiguous numbers at least).  put() moves such a chunk to its place and
// zeroes what has to be zero: the inner terms past k.  (Outer positions past the end only meet outputs that are not stored.)
template <typename T, int ROWS, bool K, int THREADS>
struct Stream<T, ROWS, K, THREADS, STAGED> {
    using O = Operand<T, ROWS, K, THREADS>;
    T const *base;
    long ld;
    int outers, k;
    i32x4 held[2][O::LOADS];        // two k-tiles

    __device__ __forceinline__ void set(T const *base_, int outers_, int k_, long ld_) { base = base_; ld = ld_; outers = outers_; k = k_; }

    __device__ __forceinline__ void fetch(int set, int kt)
    {
        #pragma unroll
        for (int s = 0; s < O::LOADS; s++) {
            int outer, inner;
            O::chunk(s * THREADS + (int)threadIdx.x % THREADS, outer, inner);
            inner += kt * O::KT;
            held[set][s] = load16(K ? base + min(outer, outers - 1) * ld + min(inner, k - O::EL)
                                    : base + min(inner, k - 1) * ld + min(outer, outers - O::EL));
        }
    }
    __device__ __forceinline__ void put(lds_char *lds, int set, int kt) const
    {
        bool const cut = (kt + 1) * O::KT > k || (!K && outers < ROWS);
        #pragma unroll
        for (int s = 0; s < O::LOADS; s++) {
            i32x4 v = held[set][s];
            if (cut) {
                int outer, inner;
                O::chunk(s * THREADS + (int)threadIdx.x % THREADS, outer, inner);
                inner += kt * O::KT;
                int const over = K ? inner - (k - O::EL) : outer - (outers - O::EL);
                if (over > 0) v = moved_down(v, min(over, O::EL) * 8 * (int)sizeof(T));
                if (!K && inner >= k) v = (i32x4){0, 0, 0, 0};
            }
            *(lds_i32x4 *)(lds + (s * THREADS + (int)threadIdx.x % THREADS) * 16) = v;
        }
    }
};

// What a tile is the product of.  rows / cols: outputs that exist from its corner on, which is (r0, c0); k: inner terms.
template <typename T>
struct Plan {
    T const *A, *B;
    long lda, ldb;
    int rows, cols, k, r0, c0;
};

// WAVES_K > 1: so many waves, each by itself, with a part of the inner index and of LDS; their sums are added up in their order.
template <typename T, int BM_, int BN_, int WAVES_M_, int WAVES_N_, bool AK_, bool BK_, Feed FEED_, int WAVES_K_ = 1>
struct ProductTile {
    static constexpr int BM = BM_, BN = BN_, WAVES_M = WAVES_M_, WAVES_N = WAVES_N_, WAVES_K = WAVES_K_, SHARE = 64 * WAVES_M * WAVES_N, THREADS = SHARE * WAVES_K;
    static_assert(WAVES_K == 1 || SHARE == 64, "each wave by itself");
    static constexpr int MB = BM / WAVES_M / 64, NB = BN / WAVES_N / 64;     // 64 x 64 blocks a wave
    static_assert(BM == BN, "the places in LDS are of one size");
    typedef typename Mfma<T>::Acc Acc;
    using OA = Operand<T, BM, AK_, SHARE>;
    using OB = Operand<T, BN, BK_, SHARE>;
    static constexpr int PLACE = OA::BYTES, PLACES = FEED_ == DIRECT ? 5 : 4, RING = PLACES * PLACE, LDS_BYTES = RING * WAVES_K;
    static constexpr int KT = OA::KT;
    static constexpr bool A_K = AK_;
    static constexpr int PER_SIMD = MB * NB > 2 || WAVES_K > 1 ? 1 : 2;     // waves

    Acc acc[MB][2][NB][2];

    // the operands of half a k-tile in registers
    struct Fragments { i32x4 a[2][MB][2], b[2][NB][2]; };

    static constexpr int READS = 4 * (MB + NB), PRODUCTS = 8 * MB * NB;         // of half a k-tile
    static __device__ __forceinline__ void read(Fragments &f, lds_char const *la, lds_char const *lb, int half, int r)
    {
        int const wave = wave_number() % (SHARE / 64), m0 = wave % WAVES_M * (BM / WAVES_M), n0 = wave / WAVES_M * (BN / WAVES_N);
        int const s = r / (2 * (MB + NB)), i = r % (2 * (MB + NB)), x = i / 2 - NB, y = i / 2, t = i % 2;
        if (y < NB) f.b[s][y][t] = OB::fragment(lb, n0 + 64 * y, t, 2 * half + s);
        else        f.a[s][x][t] = OA::fragment(la, m0 + 64 * x, t, 2 * half + s);
    }
    __device__ __forceinline__ void multiply(Fragments const &f, int p)
    {
        int const s = p / (PRODUCTS / 2), i = p % (PRODUCTS / 2), x = i / (4 * NB), t = i / (2 * NB) % 2, y = i / 2 % NB, u = i % 2;
        acc[x][t][y][u] = Mfma<T>::mul(f.a[s][x][t], f.b[s][y][u], acc[x][t][y][u]);
    }
    // The products of f's half k-tile, and between them, evenly, the reads of the next one into g and the loads of a whole one: a wave issues in order,
    // and loads in a bunch would hold the products behind them up for as long as the address units need for all of them.
    template <typename S>
    __device__ __forceinline__ void turn(Fragments const &f, Fragments &g, lds_char const *la, lds_char const *lb, int half, S &stream, int place)
    {
        constexpr int LOADS = S::O::LOADS;
        #pragma unroll
        for (int p = 0; p < PRODUCTS; p++) {
            #pragma unroll
            for (int r = 0; r < READS; r++) if (r * PRODUCTS / READS == p) read(g, la, lb, half, r);
            if (p == 0) __builtin_amdgcn_s_setprio(1);
            multiply(f, p);
            #pragma unroll
            for (int l = 0; l < LOADS; l++) if ((2 * l + 1) * PRODUCTS / (2 * LOADS) == p) stream.load(place, l);
            __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_setprio(0);
    }
    // All but the last LOADS loads of every wave have landed, and every wave has read what it has asked LDS for.
    // (STAGED: nothing but LDS is waited for; the compiler waits for the registers.  A wave by itself meets nobody.)
    template <int LOADS>
    static __device__ __forceinline__ void meet()
    {
        if constexpr (FEED_ == STAGED) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        else asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" :: "n"(LOADS) : "memory");
        if constexpr (WAVES_K == 1) asm volatile("s_barrier" ::: "memory");
    }

    Stream<T, BM, AK_, SHARE, FEED_> a;
    Stream<T, BN, BK_, SHARE, FEED_> b;
    Fragments f[FEED_ == DIRECT ? 2 : 1];
    int now;

    // DIRECT: k-tiles of a tile, at least the two that are fetched ahead (what is past k is zero)
    static __device__ __forceinline__ int tiles_of(int k) { int const t = (k + KT - 1) / KT; return FEED_ == DIRECT ? max(t, 2) : t; }
    static __device__ __forceinline__ int after(int place, int n) { place += n * PLACE; return place >= RING ? place - RING : place; }
    __device__ __forceinline__ void set_a(Plan<T> const &p) { a.set(p.A, p.rows, p.k, p.lda); }
    __device__ __forceinline__ void set_b(Plan<T> const &p) { b.set(p.B, p.cols, p.k, p.ldb); }

    // The k-tile whose chunks are cut by k, -1: none
    static __device__ __forceinline__ int cut_tile(int k) { return (AK_ || BK_) && k % OA::EL != 0 ? k / KT : -1; }
    __device__ __forceinline__ void trim(lds_char *lds, int place, int k)
    {
        if (AK_) OA::trim(lds + place, k % KT);
        if (BK_) OB::trim(lds + after(place, 1), k % KT);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if constexpr (WAVES_K == 1) asm volatile("s_barrier" ::: "memory");
    }

    // before the first tile
    __device__ __forceinline__ void start(Plan<T> const &p, char *shared)
    {
        lds_char *const lds = (lds_char *)shared;
        set_a(p); set_b(p);
        if constexpr (FEED_ == DIRECT) {
            int const lds0 = __builtin_amdgcn_readfirstlane((int)(unsigned long long)lds);
            a.fetch(lds0, 0); b.fetch(lds0 + PLACE, 0); a.fetch(lds0 + 2 * PLACE, 1); b.fetch(lds0 + 3 * PLACE, 1);
            meet<OA::LOADS + OB::LOADS>();
            if (cut_tile(p.k) == 0) trim(lds, 0, p.k);
            #pragma unroll
            for (int r = 0; r < READS; r++) read(f[0], lds, lds + PLACE, 0, r);
            now = 0;
        }
    }

    // acc = the tile p; where `next` is another, its loads have begun when this one's products end (otherwise it is empty: k = 0)
    __device__ __forceinline__ void run(Plan<T> const &p, Plan<T> const &next, char *shared)
    {
        lds_char *const lds = (lds_char *)shared;
        #pragma unroll
        for (int x = 0; x < MB; x++)
            #pragma unroll
            for (int t = 0; t < 2; t++)
                #pragma unroll
                for (int y = 0; y < NB; y++)
                    #pragma unroll
                    for (int u = 0; u < 2; u++) acc[x][t][y][u] = Acc{};
        int const tiles = tiles_of(p.k);
        if constexpr (FEED_ == DIRECT) {
            int const lds0 = __builtin_amdgcn_readfirstlane((int)(unsigned long long)lds), cut = cut_tile(p.k);
            for (int kt = 0; kt < tiles; kt++) {
                int const place = after(now, 2), ahead = kt + 2 < tiles ? kt + 2 : kt + 2 - tiles;
                if (kt + 2 == tiles) set_a(next);
                a.begin(ahead);
                turn(f[0], f[1], lds + now, lds + after(now, 1), 1, a, lds0 + after(now, 4));
                // the next k-tile is there, and no wave reads this one's places any more
                meet<OA::LOADS>();
                // (kt + 1 == tiles: the next tile's first)
                if (kt + 1 == cut) trim(lds, place, p.k);
                if (kt + 1 == tiles && cut_tile(next.k) == 0) trim(lds, place, next.k);
                if (kt + 2 == tiles) set_b(next);
                b.begin(ahead);
                turn(f[1], f[0], lds + place, lds + after(place, 1), 0, b, lds0 + now);
                now = place;
            }
        } else {
            if (tiles == 0) return;
            a.fetch(0, 0); b.fetch(0, 0);
            a.fetch(1, 1); b.fetch(1, 1);
            a.put(lds, 0, 0); b.put(lds + PLACE, 0, 0);
            for (int kt = 0; kt < tiles; kt += 2) {
                #pragma unroll
                for (int p = 0; p < 2; p++) {
                    lds_char *const here = lds + p * 2 * PLACE, *const there = lds + (p ^ 1) * 2 * PLACE;
                    meet<0>();
                    a.fetch(p, kt + p + 2); b.fetch(p, kt + p + 2);
                    if (kt + p < tiles) {
                        #pragma unroll
                        for (int half = 0; half < 2; half++) {
                            #pragma unroll
                            for (int r = 0; r < READS; r++) read(f[0], here, here + PLACE, half, r);
                            #pragma unroll
                            for (int q = 0; q < PRODUCTS; q++) multiply(f[0], q);
                        }
                        a.put(there, p ^ 1, kt + p + 1); b.put(there + PLACE, p ^ 1, kt + p + 1);
                    }
                }
            }
        }
    }

    // All tiles of a workgroup: get(turn, plan) makes the plan of its tile number `turn` (`there` false: there is none), done(plan, what get gave)
    // stores it.  WAVES_K > 1: one tile.
    template <typename G, typename E>
    __device__ __forceinline__ void all(char *shared, G &&get, E &&done)
    {
        Plan<T> p;
        auto keep = get(0, p);
        if (!keep.there) return;
        if constexpr (WAVES_K > 1) {
            Plan<T> mine = p;
            int const part = ((p.k + KT - 1) / KT + WAVES_K - 1) / WAVES_K * KT, k0 = min(wave_number() * part, p.k);
            mine.A = uniform(p.A + k0 * (AK_ ? 1L : p.lda)); mine.B = uniform(p.B + k0 * (BK_ ? 1L : p.ldb));
            mine.k = uniform(min(part, p.k - k0));
            Plan<T> none = mine;
            none.k = 0; none.rows = none.cols = 0;
            char *const ring = shared + wave_number() * RING;
            // (STAGED: the chunk that k cuts is read from where it ends there, in front of the part if that is shorter)
            start(mine, ring);
            run(mine, none, ring);
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            add_up((lds_char *)shared);
            done(p, keep);
            return;
        }
        start(p, shared);
        for (int turn = 1;; turn++) {
            Plan<T> next = p;
            auto const more = get(turn, next);
            if (!more.there) { next.k = 0; next.rows = next.cols = 0; }
            next.A = uniform(next.A); next.B = uniform(next.B);
            next.rows = uniform(next.rows); next.cols = uniform(next.cols); next.k = uniform(next.k); next.r0 = uniform(next.r0); next.c0 = uniform(next.c0);
            run(p, next, shared);
            // (STAGED: other waves may still read what this one is about to overwrite)
            if constexpr (FEED_ == STAGED) asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            done(p, keep);
            if (!more.there) break;
            p = next; keep = more;
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            if constexpr (FEED_ != DIRECT) { set_a(p); set_b(p); }
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }

    // WAVES_K = 4: wave w is left with the sums of registers 4 w ... 4 w + 3 of every accumulator, in registers 0 ... 3
    __device__ __forceinline__ void add_up(lds_char *lds)
    {
        static_assert(WAVES_K == 1 || (WAVES_K == 4 && MB == 1 && NB == 1), "four times four registers");
        typedef typename Mfma<T>::Acc16 Four;
        typedef __attribute__((address_space(3))) Four lds_four;
        lds_four *const all = (lds_four *)lds;          // [wave that summed][wave that takes][2 t + u][lane]
        int const lane = threadIdx.x & 63, wave = wave_number();
        #pragma unroll
        for (int g = 0; g < 4; g++)
            #pragma unroll
            for (int i = 0; i < 4; i++) {
                auto const &v = acc[0][i >> 1][0][i & 1];
                all[((wave * 4 + g) * 4 + i) * 64 + lane] = Four{v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]};
            }
        __syncthreads();
        #pragma unroll
        for (int i = 0; i < 4; i++) {
            Four sum = all[(wave * 4 + i) * 64 + lane];
            #pragma unroll
            for (int w = 1; w < 4; w++) sum += all[((w * 4 + wave) * 4 + i) * 64 + lane];
            #pragma unroll
            for (int r = 0; r < 4; r++) acc[0][i >> 1][0][i & 1][r] = sum[r];
        }
    }

    // The tile as numbers of type S, value(x, t, y, u, r) of register r of acc[x][t][y][u]: out.put(row, column, the numbers of 16 bytes from that row on), which
    // count from the tile's corner.  Each wave turns its accumulators round through 4 KB of LDS (the place
    // of the last k-tile's B, which nobody reads any more), so that every store is of whole 128-byte lines: stored as they lie in the registers, 32
    // bytes a line at a time, 24 gradients 720 x 1336 in fp32 over 2784 columns took 46 us instead of 28.  WAVES_K > 1: four rows at a time, as the registers hold them.
    template <typename S, typename V, typename O>
    __device__ __forceinline__ void store(char *shared, V &&value, O const &out)
    {
        int const lane = thread_now() & 63, wave = wave_number() % (SHARE / 64), j = lane & 31, q = lane >> 5;
        int const m0 = wave % WAVES_M * (BM / WAVES_M), n0 = wave / WAVES_M * (BN / WAVES_N);
        if constexpr (WAVES_K > 1) {
            int const g = wave_number();
            #pragma unroll
            for (int u = 0; u < 2; u++)
                #pragma unroll
                for (int t = 0; t < 2; t++) {
                    int const row = OA::row(8 * g + 4 * q, t), col = OB::row(j, u);
                    S v[4];
                    #pragma unroll
                    for (int r = 0; r < 4; r++) v[r] = value(0, t, 0, u, r);
                    out.template put<false>(row, col, v);
                }
            return;
        }
        // (a tile that is all there has no tests between its stores)
        if (O::FREE && out.rows() >= BM && out.cols() >= BN) turn_round<S, true>(shared, value, out, lane, wave, m0, n0);
        else turn_round<S, false>(shared, value, out, lane, wave, m0, n0);
    }
    template <typename S, bool WHOLE, typename V, typename O>
    __device__ __forceinline__ void turn_round(char *shared, V &&value, O const &out, int lane, int wave, int m0, int n0)
    {
        constexpr int EL = 16 / (int)sizeof(S);
        typedef __attribute__((address_space(3))) u32x2 lds_u32x2;
        int const j = lane & 31, q = lane >> 5;
        lds_char *const lds = (lds_char *)shared + (FEED_ == DIRECT ? after(now, 4) : 0) + wave * 4096;
        lds_char *const mine = lds + j * 128, *const theirs = lds + (lane >> 3) * 128;
        #pragma unroll
        for (int x = 0; x < MB; x++)
            #pragma unroll
            for (int y = 0; y < NB; y++)
                #pragma unroll
                for (int u = 0; u < 2; u++)
                    #pragma unroll
                    for (int half = 0; half < (int)sizeof(S) / 2; half++) {
                        #pragma unroll
                        for (int t = 0; t < 2; t++)
                            #pragma unroll
                            for (int g = 0; g < 4; g++) {
                                // four rows from `row` on; the half of 32 rows that they are in
                                int const row = OA::row(8 * g, t) + (AK_ ? 8 : 4) * q;
                                if (sizeof(S) == 4 && (AK_ ? g >> 1 : t) != half) continue;
                                S v[4];
                                #pragma unroll
                                for (int r = 0; r < 4; r++) v[r] = value(x, t, y, u, 4 * g + r);
                                int const byte = (row - (sizeof(S) == 4 ? 32 * half : 0)) * (int)sizeof(S);
                                lds_char *const to = mine + (((byte >> 4) ^ (j >> 1 & 7)) << 4) + (byte & 8);
                                if constexpr (sizeof(S) == 4) { i32x4 w; __builtin_memcpy(&w, v, 16); *(lds_i32x4 *)to = w; }
                                else { u32x2 w; __builtin_memcpy(&w, v, 8); *(lds_u32x2 *)to = w; }
                            }
                        i32x4 w[4];
                        #pragma unroll
                        for (int i = 0; i < 4; i++) w[i] = *(lds_i32x4 const *)(theirs + i * 1024 + (((lane & 7) ^ (((lane >> 3) + 8 * i) >> 1 & 7)) << 4));
                        #pragma unroll
                        for (int i = 0; i < 4; i++) {
                            S v[EL];
                            __builtin_memcpy(v, &w[i], 16);
                            out.template put<WHOLE>(m0 + 64 * x + 32 * half + (lane & 7) * EL, n0 + 64 * y + OB::row((lane >> 3) + 8 * i, u), v);
                        }
                    }
    }
};

// 64 x 64 outputs in fp64, four waves of 32 x 32.  A k-tile is 16 inner terms; LDS holds three of both operands, fed directly, so that a k-tile's loads
// have two k-tiles' time, and there is one barrier a k-tile; three workgroups a compute unit hide what is left.  Like in the
// library's dgemm, sums of 256 terms are added up in their turn.
template <bool AK, bool BK>
struct DoubleTile {
    static constexpr int SIZE = 64, THREADS = 256, FLUSH = 16;
    using SA = Stream<double, SIZE, AK, THREADS, DIRECT>;
    using SB = Stream<double, SIZE, BK, THREADS, DIRECT>;
    using OA = typename SA::O;
    using OB = typename SB::O;
    static constexpr int KT = OA::KT, PLACE = OA::BYTES, PAIR = 2 * PLACE, LDS_BYTES = 3 * PAIR;
    typedef double d4 __attribute__((ext_vector_type(4)));

    d4 sum[2][2];           // [columns][rows]: lane l, register r: row l & 15, column (l >> 4) + 4 r of the fragments'

    // p.k may be 0
    __device__ __forceinline__ void run(Plan<double> const &p, char *shared)
    {
        lds_char *const lds = (lds_char *)shared;
        int const wave = wave_number(), m0 = wave % 2 * 32, n0 = wave / 2 * 32;
        int const lds0 = uniform((int)(unsigned long long)lds), tiles = (p.k + KT - 1) / KT, cut = (AK || BK) && p.k % OA::EL != 0 ? p.k / KT : -1;
        SA a;
        SB b;
        a.set(p.A, p.rows, p.k, p.lda); b.set(p.B, p.cols, p.k, p.ldb);
        #pragma unroll
        for (int i = 0; i < 2; i++) { a.fetch(lds0 + i * PAIR, i); b.fetch(lds0 + i * PAIR + PLACE, i); }
        d4 acc[2][2];
        #pragma unroll
        for (int c = 0; c < 2; c++)
            #pragma unroll
            for (int r = 0; r < 2; r++) acc[c][r] = sum[c][r] = d4{0.0, 0.0, 0.0, 0.0};
        int now = 0;
        for (int kt = 0; kt < tiles; kt++) {
            // this k-tile is there, and every wave has read the one before, whose place the next loads take
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"(OA::LOADS + OB::LOADS) : "memory");
            if (kt == cut) {
                if (AK) OA::trim(lds + now, p.k % KT);
                if (BK) OB::trim(lds + now + PLACE, p.k % KT);
                asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            }
            int const free = now == 0 ? 2 * PAIR : now - PAIR;
            a.fetch(lds0 + free, kt + 2); b.fetch(lds0 + free + PLACE, kt + 2);
            double fa[2][2][2], fb[2][2][2];
            #pragma unroll
            for (int h = 0; h < 2; h++) { OA::doubles(lds + now, m0, h, fa[h]); OB::doubles(lds + now + PLACE, n0, h, fb[h]); }
            #pragma unroll
            for (int h = 0; h < 2; h++) {
                __builtin_amdgcn_sched_barrier(0);
                #pragma unroll
                for (int e = 0; e < 2; e++)
                    #pragma unroll
                    for (int c = 0; c < 2; c++)
                        #pragma unroll
                        for (int r = 0; r < 2; r++) acc[c][r] = __builtin_amdgcn_mfma_f64_16x16x4f64(fb[h][e][c], fa[h][e][r], acc[c][r], 0, 0, 0);
            }
            if ((kt + 1) % FLUSH == 0)
                #pragma unroll
                for (int c = 0; c < 2; c++)
                    #pragma unroll
                    for (int r = 0; r < 2; r++) { sum[c][r] += acc[c][r]; acc[c][r] = d4{0.0, 0.0, 0.0, 0.0}; }
            now = now == 2 * PAIR ? 0 : now + PAIR;
        }
        #pragma unroll
        for (int c = 0; c < 2; c++)
            #pragma unroll
            for (int r = 0; r < 2; r++) sum[c][r] += acc[c][r];
        // (what was fetched past the end is zeros that nobody reads, but it must have landed before LDS is another workgroup's)
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    // C = sums + beta C, of which rows x cols exist
    __device__ __forceinline__ void store(double beta, double *C, long ldc, int rows, int cols) const
    {
        int const lane = threadIdx.x & 63, wave = wave_number(), m0 = wave % 2 * 32, n0 = wave / 2 * 32;
        #pragma unroll
        for (int c = 0; c < 2; c++)
            #pragma unroll
            for (int i = 0; i < 4; i++) {
                int const col = n0 + OB::double_row((lane >> 4) + 4 * i, c);
                #pragma unroll
                for (int r = 0; r < 2; r++) {
                    int const row = m0 + OA::double_row(lane & 15, r);
                    double *const to = C + col * ldc + row;
                    if (col < cols && row < rows) *to = beta == 0.0 ? sum[c][r][i] : fma(beta, *to, sum[c][r][i]);
                }
            }
    }
};

// N consecutive numbers of a column, `rows` of which exist (WHOLE: all).  (Wide stores at any alignment)
template <bool WHOLE, int N, typename D>
__device__ __forceinline__ void store_run(D *to, int rows, D const (&v)[N])
{
    if (WHOLE || rows >= N) __builtin_memcpy(to, v, sizeof v);
    else
        #pragma unroll
        for (int r = 0; r < N; r++)
            if (r < rows) to[r] = v[r];
}

} // namespace sn
