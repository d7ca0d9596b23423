// Matrix products over ragged groups of columns: C_g = op(A_g) B_g and D_g = X_g Y_g^T + beta D_g, where group g owns the
// columns [offsets[g], offsets[g + 1]) of B and C (of X and Y) and a matrix of its own; the first also in 8-bit integers with scales.
#include "product_tile.h"
#include "dgemm_tile.h"
#include "products.h"
#include <algorithm>
#include <cmath>
#include <type_traits>

namespace sn {

#ifdef SN_TEST_HOOKS
static int forced_tile = 0, forced_slices = 0;         // a test's choice in place of the rules' (0: theirs)
#else
static constexpr int forced_tile = 0, forced_slices = 0;
#endif

// a tile's place in the matrices
struct Place { Span s; bool there; };

// Where a tile goes: high x wide numbers from `to` on exist.  put: WHOLE, without a look at these.
template <typename D>
struct Columns {
    static constexpr bool FREE = true;          // worth code of its own without the tests
    D *to;
    long ld;
    int high, wide;
    __device__ __forceinline__ int rows() const { return high; }
    __device__ __forceinline__ int cols() const { return wide; }
    template <bool WHOLE, int N> __device__ __forceinline__ void put(int r, int c, D const (&v)[N]) const
    {
        if (WHOLE || c < wide) store_run<WHOLE>(to + c * ld + r, high - r, v);
    }
};
// The same for sums in fp32 that are added to beta times what is there.
template <typename D>
struct Added : Columns<D> {
    static constexpr bool FREE = false;
    float beta;
    template <bool WHOLE> __device__ __forceinline__ void put(int r, int c, float const (&v)[4]) const
    {
        if (!WHOLE && c >= this->wide) return;
        D *const at = this->to + c * this->ld + r;
        D sum[4];
        if (WHOLE || r + 4 <= this->high) __builtin_memcpy(sum, at, sizeof sum);
        else
            #pragma unroll
            for (int e = 0; e < 4; e++) sum[e] = r + e < this->high ? at[e] : (D)0.f;
        #pragma unroll
        for (int e = 0; e < 4; e++) sum[e] = (D)(v[e] + beta * (float)sum[e]);
        store_run<WHOLE>(at, this->high - r, sum);
    }
};

template <typename T, typename P>
__global__ __launch_bounds__(P::THREADS, P::PER_SIMD)
void grouped_gemm_kernel(int groups, int m, int n, int k, int const *__restrict__ offsets, T const *__restrict__ A, long lda, long strideA,
    T const *__restrict__ B, long ldb, T *__restrict__ C, long ldc)
{
    __shared__ __attribute__((aligned(16))) char lds[P::LDS_BYTES];
    int const rows = (m + P::BM - 1) / P::BM;
    Pieces pieces(offsets, groups, n, P::BN);
    P tile;
    tile.all(lds, [&](int turn, Plan<T> &p) {
        int const t = tile_of_workgroup(rows * pieces.total, turn);
        if (t < 0) return Place{Span{}, false};
        int row, piece;
        row_and_column(t, rows, pieces.total, row, piece);
        Span const s = pieces.at(piece);
        int const r0 = row * P::BM;
        p = Plan<T>{A + s.group * strideA + r0 * (P::A_K ? lda : 1L), B + s.begin * ldb, lda, ldb, m - r0, s.end - s.begin, s.empty() ? 0 : k, r0, 0};
        return Place{s, true};
    }, [&](Plan<T> const &p, Place const &at) {
        tile.template store<T>(lds, [&](int x, int t, int y, int u, int r) { return (T)tile.acc[x][t][y][u][r]; },
            Columns<T>{C + at.s.begin * ldc + p.r0, ldc, p.rows, p.cols});
    });
}

// One item is a tile of one group over one of `slices` runs of its columns.  The items lie in the order of their lengths, and the workgroups take them
// to and fro (0 1 2 ... 2 1 0), which evens out what each has to do.  With several slices `out` has a plane of all groups' outputs (m x n without gaps)
// for each slice, and grouped_outer_sum_kernel adds them up in the slices' order.
template <typename T, typename D, typename P>
__global__ __launch_bounds__(P::THREADS, P::PER_SIMD)
void grouped_outer_kernel(int groups, int m, int n, int k, int slices, int const *__restrict__ offsets, T const *__restrict__ X, long ldx,
    T const *__restrict__ Y, long ldy, float beta, D *__restrict__ out, long ldd, long strideD)
{
    __shared__ __attribute__((aligned(16))) char lds[P::LDS_BYTES];
    int const rows = (m + P::BM - 1) / P::BM, cols = (n + P::BN - 1) / P::BN, each = rows * cols, items = groups * slices * each;
    Longest order(offsets, groups, k);
    P tile;
    struct Item { int group, slice; bool there; };
    tile.all(lds, [&](int turn, Plan<T> &p) {
        int const here = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
        unsigned const i = turn * gridDim.x + (turn & 1 ? gridDim.x - 1 - here : here);
        if (i >= (unsigned)items) return Item{0, 0, false};
        Span const s = order.at(i / (unsigned)(each * slices));
        int const in = i % (unsigned)(each * slices), slice = (unsigned)in / (unsigned)each;
        int row, col;
        row_and_column(in - slice * each, rows, cols, row, col);
        int const length = s.end - s.begin, part = slices == 1 ? length : ((length + slices - 1) / slices + P::KT - 1) / P::KT * P::KT;
        int const begin = s.begin + (int)min((long)slice * part, (long)length), end = min(begin + part, s.end);
        int const r0 = row * P::BM, c0 = col * P::BN;
        p = Plan<T>{X + begin * ldx + r0, Y + begin * ldy + c0, ldx, ldy, m - r0, n - c0, end - begin, r0, c0};
        return Item{s.group, slice, true};
    }, [&](Plan<T> const &p, Item const &at) {
        Columns<D> const to{out + ((long)at.slice * groups + at.group) * strideD + p.c0 * ldd + p.r0, ldd, p.rows, p.cols};
        if (beta == 0.f) tile.template store<D>(lds, [&](int x, int t, int y, int u, int r) { return (D)tile.acc[x][t][y][u][r]; }, to);
        else tile.template store<float>(lds, [&](int x, int t, int y, int u, int r) { return tile.acc[x][t][y][u][r]; }, Added<D>{to, beta});
    });
}

// PARTS threads an output, each with a run of the slices, eight of them in flight; the runs' sums in their order.  (1 thread with one load at a time: 64 planes of
// 64 x 64 in fp64 took 18 us, with 8 threads 3.9 us; 4 planes of 512 x 512 in fp32 take 3.9 us either way.)
template <typename S, typename D, int PARTS>
__global__ __launch_bounds__(256)
void grouped_outer_sum_kernel(int groups, int m, int n, int slices, S const *__restrict__ planes, S beta, D *__restrict__ out, long ldd, long strideD)
{
    constexpr int WIDE = 256 / PARTS;
    __shared__ S part[PARTS][WIDE];
    long const all = (long)groups * n * m;
    int const mine = threadIdx.x % WIDE, p = threadIdx.x / WIDE, each = (slices + PARTS - 1) / PARTS, end = min((p + 1) * each, slices);
    for (long e0 = (long)blockIdx.x * WIDE; e0 < all; e0 += (long)gridDim.x * WIDE) {
        long const e = e0 + mine;
        S sum = 0;
        if (e < all)
            for (int s = p * each; s < end; s += 8) {
                S v[8];
                #pragma unroll
                for (int i = 0; i < 8; i++) v[i] = s + i < end ? planes[(s + i) * all + e] : (S)0;
                #pragma unroll
                for (int i = 0; i < 8; i++) sum += v[i];
            }
        if (PARTS > 1) {
            part[p][mine] = sum;
            __syncthreads();
            if (p == 0)
                #pragma unroll
                for (int i = 1; i < PARTS; i++) sum += part[i][mine];
            __syncthreads();
        }
        if (p == 0 && e < all) {
            long const column = e / m;
            D *const to = out + column / n * strideD + column % n * ldd + e % m;
            *to = (D)(beta == 0 ? sum : sum + beta * (S)*to);
        }
    }
}

// The scaling is three roundings to fp32 and one to the result's type: the empty statement keeps the compiler from fusing the
// second product with the conversion to fp16, whose one rounding would depend on the type of the result.
__device__ __forceinline__ float scaled(int sum, float row, float col)
{
    float v = (float)sum * row * col;
    asm("" : "+v"(v));
    return v;
}

template <typename D>
struct Scaled : Columns<D> {
    float const *row, *col;
    template <bool WHOLE> __device__ __forceinline__ void put(int r, int c, int const (&v)[4]) const
    {
        if (!WHOLE && c >= this->wide) return;
        float const scale = col[c];
        D d[4];
        #pragma unroll
        for (int e = 0; e < 4; e++) d[e] = (D)scaled(v[e], row[WHOLE ? r + e : min(r + e, this->high - 1)], scale);
        store_run<WHOLE>(this->to + c * this->ld + r, this->high - r, d);
    }
};

template <typename D, typename P>
__global__ __launch_bounds__(P::THREADS, P::PER_SIMD)
void gemm_i8_kernel(int groups, int m, int n, int k, int const *__restrict__ offsets, signed char const *__restrict__ A, long lda, long strideA,
    float const *__restrict__ scaleA, long strideS, signed char const *__restrict__ B, long ldb, float const *__restrict__ scaleB, D *__restrict__ C, long ldc)
{
    __shared__ __attribute__((aligned(16))) char lds[P::LDS_BYTES];
    typedef signed char T;
    int const rows = (m + P::BM - 1) / P::BM;
    Pieces pieces(offsets, groups, n, P::BN);
    P tile;
    tile.all(lds, [&](int turn, Plan<T> &p) {
        int const t = tile_of_workgroup(rows * pieces.total, turn);
        if (t < 0) return Place{Span{}, false};
        int row, piece;
        row_and_column(t, rows, pieces.total, row, piece);
        Span const s = pieces.at(piece);
        int const r0 = row * P::BM;
        p = Plan<T>{A + s.group * strideA + r0 * lda, B + s.begin * ldb, lda, ldb, m - r0, s.end - s.begin, s.empty() ? 0 : k, r0, 0};
        return Place{s, true};
    }, [&](Plan<T> const &p, Place const &at) {
        tile.template store<int>(lds, [&](int x, int t, int y, int u, int r) { return tile.acc[x][t][y][u][r]; },
            Scaled<D>{{C + at.s.begin * ldc + p.r0, ldc, p.rows, p.cols}, scaleA + at.s.group * strideS + p.r0, scaleB + at.s.begin});
    });
}

// Too few contiguous numbers for a 16-byte load (fewer than 8 rows or inner terms of 16 bits, 16 of 8): one wave an output, its lanes
// stride over the inner index.  Element (r, i) of an operand is at r * rs + i * is.
template <typename T, typename S>
__device__ __forceinline__ S narrow_sum(T const *__restrict__ a, long ais, T const *__restrict__ b, long bis, int k)
{
    S sum = 0;
    for (int i = threadIdx.x & 63; i < k; i += 64) sum += (S)a[i * ais] * (S)b[i * bis];
    #pragma unroll
    for (int d = 32; d > 0; d /= 2) sum += __shfl_xor(sum, d);
    return sum;
}

template <typename T, typename D>
__global__ __launch_bounds__(256)
void grouped_gemm_narrow_kernel(int groups, int m, int n, int k, int const *__restrict__ offsets, T const *__restrict__ A, long ars, long ais, long strideA,
    float const *__restrict__ scaleA, long strideS, T const *__restrict__ B, long ldb, float const *__restrict__ scaleB, D *__restrict__ C, long ldc)
{
    Pieces pieces(offsets, groups, n, 4);
    if ((int)blockIdx.x >= pieces.total) return;
    Span const s = pieces.at(blockIdx.x);
    int const c = s.begin + (threadIdx.x >> 6);
    if (c >= s.end) return;
    for (int r = blockIdx.y; r < m; r += gridDim.y) {
        T const *const a = A + s.group * strideA + r * ars, *const b = B + c * ldb;
        D v;
        if constexpr (sizeof(T) == 1) v = (D)scaled(narrow_sum<T, int>(a, ais, b, 1, k), scaleA[s.group * strideS + r], scaleB[c]);
        else v = (D)narrow_sum<T, float>(a, ais, b, 1, k);
        if ((threadIdx.x & 63) == 0) C[c * ldc + r] = v;
    }
}

template <typename T, typename D>
__global__ __launch_bounds__(256)
void grouped_outer_narrow_kernel(int m, int n, int k, int const *__restrict__ offsets, T const *__restrict__ X, long ldx,
    T const *__restrict__ Y, long ldy, float beta, D *__restrict__ out, long ldd, long strideD)
{
    Span const s = whole_group(offsets, k, blockIdx.z);
    for (long e = blockIdx.x * 4 + (threadIdx.x >> 6); e < (long)m * n; e += gridDim.x * 4) {
        long const r = e % m, c = e / m;
        float v = narrow_sum<T, float>(X + s.begin * ldx + r, ldx, Y + s.begin * ldy + c, ldy, s.end - s.begin);
        D *const to = out + s.group * strideD + c * ldd + r;
        if (beta != 0.f) v += beta * (float)*to;
        if ((threadIdx.x & 63) == 0) *to = (D)v;
    }
}

// Few columns a group (a token or a batch of them while text is generated): the matrix is read once, as fast as memory gives it, and nothing
// else counts.  A workgroup takes 16 rows of A_g and up to 16 columns; its eight waves cut the inner index into eight runs, load their operands
// straight into the matrix instructions' registers, eight 16-byte loads of A in flight a lane, and add up their
// sums through LDS in the waves' order.  Only for A with the inner index contiguous.  Any alignment: the chunk that k cuts is
// read from where it ends at k, and what of it the chunk before held is zeroed, in both operands alike.
// One token through 8 of 64 matrices 1024 x 2048 in bf16: 9 us, 3.7 TB/s; 4096 x 4096 in 8 bits: 5.3 us, 3.2 TB/s.
template <typename T, typename Out>
__device__ __forceinline__ void few_columns_tile(T const *__restrict__ A, long lda, int rows, T const *__restrict__ B, long ldb, int cols, int k, Out &&out)
{
    constexpr int EL = 16 / (int)sizeof(T), WAVES = 8, U = 8;
    typedef typename Mfma<T>::Acc16 Acc;
    __shared__ __attribute__((aligned(16))) Acc sums[WAVES][64];
    int const lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, q = lane >> 4;
    int const steps = (k + 4 * EL - 1) / (4 * EL), run = (steps + WAVES - 1) / WAVES;
    int const first = min(wave * run, steps), end = min(first + run, steps);
    T const *const a = A + min(i, rows - 1) * lda;          // (a row or column that is not there: another's, and its result is not stored)
    T const *const b = B + min(i, cols - 1) * ldb;
    Acc acc = {};
    // chunk q of step s: entirely below k in all but the last step
    int s = first;
    for (; s + U <= min(end, k / (4 * EL)); s += U) {
        i32x4 va[U], vb[U];
        #pragma unroll
        for (int u = 0; u < U; u++) va[u] = load16(a + ((s + u) * 4 + q) * EL);
        #pragma unroll
        for (int u = 0; u < U; u++) vb[u] = load16(b + ((s + u) * 4 + q) * EL);
        #pragma unroll
        for (int u = 0; u < U; u++) acc = Mfma<T>::mul16(va[u], vb[u], acc);
    }
    if (s < end) {
        i32x4 va[U], vb[U];
        int skip[U];
        #pragma unroll
        for (int u = 0; u < U; u++) {
            int const at = ((s + u) * 4 + q) * EL, from = min(at, k - EL);
            skip[u] = s + u < end ? min(at - from, EL) : EL;
            va[u] = load16(a + from);
            vb[u] = load16(b + from);
        }
        #pragma unroll
        for (int u = 0; u < U; u++) {
            i32x4 mask;
            #pragma unroll
            for (int w = 0; w < 4; w++) {
                int const bits = min(max(skip[u] * 8 * (int)sizeof(T) - 32 * w, 0), 32);
                mask[w] = bits == 32 ? 0 : (int)(0xffffffffu << bits);
            }
            va[u] &= mask;
            acc = Mfma<T>::mul16(va[u], vb[u] & mask, acc);
        }
    }
    sums[wave][lane] = acc;
    __syncthreads();
    // lane l, register r of a sum is row 4 (l >> 4) + r, column l & 15
    if (threadIdx.x < 256) {
        int const row = threadIdx.x & 15, col = threadIdx.x >> 4, l = (row >> 2) * 16 + col;
        auto sum = sums[0][l][row & 3];
        #pragma unroll
        for (int w = 1; w < WAVES; w++) sum += sums[w][l][row & 3];
        if (row < rows && col < cols) out(row, col, sum);
    }
}

template <typename T>
__global__ __launch_bounds__(512)
void grouped_gemm_few_kernel(int groups, int m, int n, int k, int const *__restrict__ offsets, T const *__restrict__ A, long lda, long strideA,
    T const *__restrict__ B, long ldb, T *__restrict__ C, long ldc)
{
    Pieces pieces(offsets, groups, n, 16);
    int const t = tile_of_workgroup((m + 15) / 16 * pieces.total, 0);
    if (t < 0) return;
    Span const s = pieces.at((unsigned)t % (unsigned)pieces.total);
    if (s.empty()) return;
    int const row = (unsigned)t / (unsigned)pieces.total;
    int const r0 = row * 16;
    few_columns_tile<T>(A + s.group * strideA + r0 * lda, lda, m - r0, B + s.begin * ldb, ldb, s.end - s.begin, k,
        [&](int r, int c, float sum) { C[(s.begin + c) * ldc + r0 + r] = (T)sum; });
}

// fp64: one piece of a group a workgroup; the tile rows of a piece side by side, so that its columns come from memory once.
// (24 matrices 312 x 312, 40000 columns: 154 us, 51 TFLOP/s, with the tile of dgemm 172 us; 20000 columns, 8 matrices 1024 x 1024: 705 us, 60 TFLOP/s, 762 us)
// FAST: operands that can be fed directly; others by the tile of the library's own dgemm.
template <bool TA, bool FAST>
__global__ __launch_bounds__(256, FAST ? 3 : 2)
void grouped_dgemm_kernel(int groups, int m, int n, int k, int const *__restrict__ offsets, double const *__restrict__ A, int lda, long strideA,
    double const *__restrict__ B, int ldb, double *__restrict__ C, int ldc)
{
    Pieces pieces(offsets, groups, n, 64);
    int const rows = (m + 63) / 64, t = tile_of_workgroup(rows * pieces.total, 0);
    if (t < 0) return;
    int const row = (unsigned)t % (unsigned)rows;
    Span const s = pieces.at((unsigned)t / (unsigned)rows);
    if (s.empty()) return;
    if constexpr (FAST) {
        __shared__ __attribute__((aligned(16))) char lds[DoubleTile<TA, true>::LDS_BYTES];
        long const r0 = row * 64;
        DoubleTile<TA, true> tile;
        tile.run(Plan<double>{A + s.group * strideA + r0 * (TA ? lda : 1), B + (long)s.begin * ldb, lda, ldb, m - row * 64, s.end - s.begin, k, 0, 0}, lds);
        tile.store(0.0, C + (long)s.begin * ldc + r0, ldc, m - row * 64, s.end - s.begin);
    } else          // (k > 0: this tile reads its operands' last inner term)
        gemm_tile<64, 64, 16, TA, false, 16>(m, s.end - s.begin, k, 1.0, A + s.group * strideA, lda, B + (size_t)s.begin * ldb, ldb,
            0.0, C + (size_t)s.begin * ldc, ldc, row, 0);
}

// fp64, too few 64 x 64 tiles to fill the chip: 16 x 16 outputs a workgroup, whose eight waves cut the inner index into eight runs, straight from memory; eight
// steps of eight inner terms (8 s + 2 q + e for the lanes with q = lane >> 4, two instructions e) in flight.  Sums of 64 terms, added up in their turn.
template <bool TA>
__global__ __launch_bounds__(512)
void grouped_dgemm_few_kernel(int groups, int m, int n, int k, int const *__restrict__ offsets, double const *__restrict__ A, long lda, long strideA,
    double const *__restrict__ B, long ldb, double *__restrict__ C, long ldc)
{
    typedef double d2 __attribute__((ext_vector_type(2)));
    typedef double d4 __attribute__((ext_vector_type(4)));
    constexpr int WAVES = 8, U = 8;
    __shared__ d4 sums[WAVES][64];
    Pieces pieces(offsets, groups, n, 16);
    int const t = tile_of_workgroup((m + 15) / 16 * pieces.total, 0);
    if (t < 0) return;
    Span const p = pieces.at((unsigned)t % (unsigned)pieces.total);
    if (p.empty()) return;
    int const r0 = (unsigned)t / (unsigned)pieces.total * 16, rows = m - r0, cols = p.end - p.begin;
    int const lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, q = lane >> 4;
    int const steps = (k + 7) / 8, run = (steps + WAVES - 1) / WAVES, first = min(wave * run, steps), end = min(first + run, steps);
    // (a row or column that is not there: another's, and its result is not stored)
    double const *const a = A + p.group * strideA + (r0 + min(i, rows - 1)) * (TA ? lda : 1L), *const b = B + (p.begin + min(i, cols - 1)) * ldb;
    d4 sum = {0.0, 0.0, 0.0, 0.0};
    for (int s = first; s < end; s += U) {
        d2 va[U], vb[U];
        if (s + U <= min(end, k / 8)) {
            #pragma unroll
            for (int u = 0; u < U; u++) {
                long const at = (s + u) * 8L + 2 * q;
                if (TA) va[u] = __builtin_bit_cast(d2, load16(a + at));
                else va[u] = d2{a[at * lda], a[(at + 1) * lda]};
                vb[u] = __builtin_bit_cast(d2, load16(b + at));
            }
        } else {
            #pragma unroll
            for (int u = 0; u < U; u++)
                #pragma unroll
                for (int e = 0; e < 2; e++) {
                    int const at = (s + u) * 8 + 2 * q + e;
                    long const from = min(at, k - 1);
                    double const x = a[from * (TA ? 1L : lda)], y = b[from];
                    bool const there = s + u < end && at < k;
                    va[u][e] = there ? x : 0.0; vb[u][e] = there ? y : 0.0;
                }
        }
        d4 acc = {0.0, 0.0, 0.0, 0.0};
        #pragma unroll
        for (int u = 0; u < U; u++)
            #pragma unroll
            for (int e = 0; e < 2; e++) acc = __builtin_amdgcn_mfma_f64_16x16x4f64(va[u][e], vb[u][e], acc, 0, 0, 0);
        sum += acc;
    }
    sums[wave][lane] = sum;
    __syncthreads();
    // lane l, register r of a sum is row (l >> 4) + 4 r, column l & 15
    if (threadIdx.x < 256) {
        int const row = threadIdx.x & 15, col = threadIdx.x >> 4, l = (row & 3) * 16 + col;
        double v = sums[0][l][row >> 2];
        #pragma unroll
        for (int w = 1; w < WAVES; w++) v += sums[w][l][row >> 2];
        if (row < rows && col < cols) C[(p.begin + col) * ldc + r0 + row] = v;
    }
}

// (cut into slices of the columns like the others: see grouped_outer_kernel)
template <bool FAST>
__global__ __launch_bounds__(256, FAST ? 3 : 2)
void grouped_douter_kernel(int groups, int m, int n, int k, int slices, int const *__restrict__ offsets, double const *__restrict__ X, int ldx,
    double const *__restrict__ Y, int ldy, double beta, double *__restrict__ D, int ldd, long strideD)
{
    int const rows = (m + 63) / 64, cols = (n + 63) / 64, each = rows * cols, t = tile_of_workgroup(groups * slices * each, 0);
    if (t < 0) return;
    int const in = (unsigned)t % (unsigned)(each * slices), slice = (unsigned)in / (unsigned)each, tile = in - slice * each;
    int const row = (unsigned)tile % (unsigned)rows, col = (unsigned)tile / (unsigned)rows;
    Span const s = whole_group(offsets, k, (unsigned)t / (unsigned)(each * slices));
    int const length = s.end - s.begin, part = slices == 1 ? length : ((length + slices - 1) / slices + 15) / 16 * 16;
    int const begin = s.begin + (int)min((long)slice * part, (long)length), end = min(begin + part, s.end);
    double *const to = D + ((long)slice * groups + s.group) * strideD;
    if constexpr (FAST) {
        __shared__ __attribute__((aligned(16))) char lds[DoubleTile<false, false>::LDS_BYTES];
        int const r0 = row * 64, c0 = col * 64;
        DoubleTile<false, false> one;
        one.run(Plan<double>{X + (long)begin * ldx + r0, Y + (long)begin * ldy + c0, ldx, ldy, m - r0, n - c0, end - begin, 0, 0}, lds);
        one.store(beta, to + (long)c0 * ldd + r0, ldd, m - r0, n - c0);
    } else if (begin == end) {
        for (int e = threadIdx.x; e < 64 * 64; e += 256) {
            int const r = row * 64 + e % 64, c = col * 64 + e / 64;
            if (r < m && c < n) { double *const p = to + (size_t)c * ldd + r; *p = beta == 0.0 ? 0.0 : beta * *p; }
        }
    } else
        gemm_tile<64, 64, 16, false, true, 16>(m, n, end - begin, 1.0, X + (size_t)begin * ldx, ldx, Y + (size_t)begin * ldy, ldy,
            beta, to, ldd, row, col);
}

// Whether an operand can be fed directly: columns aligned to 4 bytes, positions within a tile below 2^31 bytes (256 columns of up to 4 MB).
static bool direct(void const *p, long ld, long stride, int size)
{
    return (uintptr_t)p % 4 == 0 && ld * size % 4 == 0 && stride * size % 4 == 0 && ld * size <= 1 << 22;
}

template <bool TA>
static hipError_t dgemm_launch(hipStream_t s, int groups, int m, int n, int k, int const *offsets, double const *A, int lda, long strideA,
    double const *B, int ldb, double *C, int ldc)
{
    long const tiles = most_pieces(groups, n, 64) * ((m + 63) / 64);
    if (tiles >= 1L << 31) return hipErrorInvalidConfiguration;
    // In us, fitted to 1 ... 640 columns, 426 ... 1152 rows and 300 ... 4096 inner terms; elsewhere an extrapolation.  1 column, 768 x 2624: 19 us (tiles of 64: 117 us); 64 columns, 512 x 512: 10 us
    // (26 us); 576 columns, 512 x 4096: 143 us (180 us); 512 columns, 512 x 300: 21 us (17 us)
    long const small = most_pieces(groups, n, 16) * ((m + 15) / 16);
    if (k > 0 && !forced_tile && 10 + 3.4e-5 * small * k < 6 + 0.0425 * k * std::max(1.0, tiles / 256.0) && small < 1L << 22)
        return launch_kernel(grouped_dgemm_few_kernel<TA>, dim3((unsigned)roundup(small, 8)), 512, s, 0,
            groups, m, n, k, offsets, A, (long)lda, strideA, B, (long)ldb, C, (long)ldc);
    bool const fast = k == 0 || (direct(A, lda, strideA, 8) && direct(B, ldb, 0, 8));
    return launch_kernel(fast ? grouped_dgemm_kernel<TA, true> : grouped_dgemm_kernel<TA, false>, dim3((unsigned)roundup(tiles, 8)), 256, s,
        fast ? 0 : GemmCfg<64, 64, 16, TA, false>::LDS_BYTES, groups, m, n, k, offsets, A, lda, strideA, B, ldb, C, ldc);
}

// Workgroups for so many equal tiles: no more than the chip holds at once, each with a run of tiles, so that the loads of the next tile
// begin while the last one's products end.
template <typename P>
static unsigned resident(long tiles)
{
    return (unsigned)(P::WAVES_K > 1 ? roundup(tiles, 8) : std::min<long>(roundup(tiles, 8), 256 * (163840 / P::LDS_BYTES)));
}

// What a launch takes, in us, fitted to launches of 64 ... 65536 columns, 1 ... 32 groups, 64 ... 4096 rows and 256 ... 8192 inner terms: rounds of the
// workgroups that the chip holds at once, each of so many k-tiles and what it takes to begin and to store a tile.  A k-tile takes as long as the
// memory's latency while few workgroups run, as long as the matrix cores need when they fill the chip.  (Measured with 16-bit numbers; a k-tile of 8-bit ones has
// as many bytes, takes as many instructions, and is taken for as long.)
//   tile  64: four waves cut the inner index, for products of few outputs;   200 columns, 512 x 8192:  26 us (128: 74 us)
//   tile 128: two workgroups a compute unit;                                2048 columns, 4096 x 4096: 73 us (64: 124 us, 256: 89 us)
//   tile 256: the fewest reads a product;                                   4096 columns, 4096 x 4096: 120 us (128: 143 us)
static double tile_time(int tile, bool fast, double workgroups, double ktiles)
{
    double const w = std::max(1.0, workgroups), rounds = std::max(1.0, std::ceil(w / (tile == 128 ? 512 : 256) - 0.01));
    if (tile == 64) return rounds * ((fast ? 0.66 : 1.1) * std::ceil(ktiles / 4) + (fast ? 4.9 : 8.6));
    if (tile == 128) return w <= 256 ? (fast ? 0.62 : 0.9) * ktiles + 6 : rounds * ((fast ? 1.05 : 1.3) * ktiles + 6);
    return rounds * ((1.1 + 0.65 * std::min(1.0, w / 256)) * ktiles + 8);
}
// The tile of a product.  The host does not know the groups' lengths: it counts the pieces that exponentially distributed ones of this mean have.
static int product_tile(bool fast, int groups, int m, int n, int ktiles)
{
    if (forced_tile) return forced_tile;
    int best = 64;
    double least = 0;
    for (int tile : {64, 128, 256}) {
        if (tile == 256 && !fast) continue;
        // (and a tenth more of what exceeds one a group: a last round of hardly any tiles costs as much as a full one)
        double const some = std::min(groups, n), expected = some / (1 - std::exp(-tile * some / n));
        double const pieces = groups == 1 ? (n + tile - 1) / tile : expected + 0.1 * (expected - some);
        double const time = tile_time(tile, fast, pieces * ((m + tile - 1) / tile), ktiles);
        if (tile == 64 || time < least) { best = tile; least = time; }
    }
    return best;
}
// Few columns a group on average, and too few 64 x 64 tiles to fill the chip: 16 columns, 4096 x 4096: 11 us, in tiles of 64 15 us; 256 columns of 32
// groups, 2048 x 1408: 62 us, in tiles of 128 36 us.
static bool few_columns(int groups, int m, int n) { return !forced_tile && (long)n <= 16L * groups && most_pieces(groups, n, 64) * ((m + 63) / 64) < 256; }

template <typename T, typename P>
static hipError_t gemm_tiles(hipStream_t s, int groups, int m, int n, int k, int const *offsets, void const *A, int lda, long strideA,
    void const *B, int ldb, void *C, int ldc)
{
    long const tiles = most_pieces(groups, n, P::BN) * ((m + P::BM - 1) / P::BM);
    if (tiles >= 1L << 31) return hipErrorInvalidConfiguration;
    return launch_kernel(grouped_gemm_kernel<T, P>, dim3(resident<P>(tiles)), P::THREADS, s, 0,
        groups, m, n, k, offsets, (T const *)A, (long)lda, strideA, (T const *)B, (long)ldb, (T *)C, (long)ldc);
}

template <typename T, bool TA>
static hipError_t gemm_launch(hipStream_t s, int groups, int m, int n, int k, int const *offsets, void const *A, int lda, long strideA,
    void const *B, int ldb, void *C, int ldc)
{
    if (TA && k >= 8 && few_columns(groups, m, n)) {
        return launch_kernel(grouped_gemm_few_kernel<T>, dim3((unsigned)roundup(most_pieces(groups, n, 16) * ((m + 15) / 16), 8)), 512, s, 0,
            groups, m, n, k, offsets, (T const *)A, (long)lda, strideA, (T const *)B, (long)ldb, (T *)C, (long)ldc);
    }
    bool const fast = direct(A, lda, strideA, sizeof(T)) && direct(B, ldb, 0, sizeof(T));
    if (!fast && (k < 8 || (!TA && m < 8)))
        return launch_kernel(grouped_gemm_narrow_kernel<T, T>, dim3((unsigned)most_pieces(groups, n, 4), std::min(m, 65535)), 256, s, 0, groups, m, n, k, offsets,
            (T const *)A, TA ? (long)lda : 1L, TA ? 1L : (long)lda, strideA, (float const *)nullptr, 0L, (T const *)B, (long)ldb, (float const *)nullptr, (T *)C, (long)ldc);
    int const tile = product_tile(fast, groups, m, n, (k + 63) / 64);
    auto const launch = fast ? tile == 256 ? gemm_tiles<T, ProductTile<T, 256, 256, 2, 4, TA, true, DIRECT>> : tile == 128 ? gemm_tiles<T, ProductTile<T, 128, 128, 2, 2, TA, true, DIRECT>>
            : gemm_tiles<T, ProductTile<T, 64, 64, 1, 1, TA, true, DIRECT, 4>>
        : tile == 128 ? gemm_tiles<T, ProductTile<T, 128, 128, 2, 2, TA, true, STAGED>> : gemm_tiles<T, ProductTile<T, 64, 64, 1, 1, TA, true, STAGED, 4>>;
    return launch(s, groups, m, n, k, offsets, A, lda, strideA, B, ldb, C, ldc);
}

hipError_t grouped_gemm(hipStream_t s, ProductType type, bool transA, int groups, int m, int n, int k, int const *offsets,
    void const *A, int lda, long strideA, void const *B, int ldb, void *C, int ldc)
{
    if (type == PRODUCT_BF16) return (transA ? gemm_launch<__bf16, true> : gemm_launch<__bf16, false>)(s, groups, m, n, k, offsets, A, lda, strideA, B, ldb, C, ldc);
    if (type == PRODUCT_F16) return (transA ? gemm_launch<_Float16, true> : gemm_launch<_Float16, false>)(s, groups, m, n, k, offsets, A, lda, strideA, B, ldb, C, ldc);
    auto const launch = transA ? dgemm_launch<true> : dgemm_launch<false>;
    return launch(s, groups, m, n, k, offsets, (double const *)A, lda, strideA, (double const *)B, ldb, (double *)C, ldc);
}

// A weight gradient's tile and the slices that its columns are cut into: with slices there is a plane to write and read for each, and a second launch.
struct Cut { int tile, slices; };
static double outer_time(Cut c, bool fast, long groups, long m, long n, long k)
{
    long const items = groups * ((m + c.tile - 1) / c.tile) * ((n + c.tile - 1) / c.tile) * c.slices;
    return tile_time(c.tile, fast, items, (double)k / groups / c.slices / 64) + (c.slices > 1 ? 3 + c.slices * (double)groups * m * n * 8 / 4e6 : 0);
}
static Cut outer_cut(bool fast, long groups, long m, long n, long k, int most_slices = 64)
{
    Cut best = {128, 1};
    if (forced_tile) return Cut{forced_tile, std::min(forced_slices, most_slices)};
    for (int tile : {256, 128, 64})
        for (int slices : {1, 2, 4, 8, 16, 32, 64}) {
            Cut const c = {tile, slices};
            if (slices > most_slices || (tile == 256 && !fast) || (slices > 1 && k / groups / slices < 64)) continue;
            if (outer_time(c, fast, groups, m, n, k) < outer_time(best, fast, groups, m, n, k)) best = c;
        }
    return best;
}

template <typename T, typename D, typename P>
static hipError_t outer_tiles(hipStream_t s, int slices, int groups, int m, int n, int k, int const *offsets, void const *X, int ldx, void const *Y, int ldy,
    double beta, void *out, int ldd, long strideD)
{
    long const items = (long)groups * slices * ((m + P::BM - 1) / P::BM) * ((n + P::BN - 1) / P::BN);
    if (items >= 1L << 31) return hipErrorInvalidConfiguration;
    return launch_kernel(grouped_outer_kernel<T, D, P>, dim3(resident<P>(items)), P::THREADS, s, 0,
        groups, m, n, k, slices, offsets, (T const *)X, (long)ldx, (T const *)Y, (long)ldy, (float)beta, (D *)out, (long)ldd, strideD);
}

template <typename S, typename D>
static hipError_t outer_sum(hipStream_t s, int slices, int groups, int m, int n, void const *work, double beta, void *out, int ldd, long strideD)
{
    int const wide = slices > 4 ? 32 : 256;
    return launch_kernel(slices > 4 ? grouped_outer_sum_kernel<S, D, 8> : grouped_outer_sum_kernel<S, D, 1>,
        dim3((unsigned)std::min(((long)groups * m * n + wide - 1) / wide, 16384L)), 256, s, 0, groups, m, n, slices, (S const *)work, (S)beta, (D *)out, (long)ldd, strideD);
}

template <typename T, typename D>
static hipError_t outer_launch(hipStream_t s, int groups, int m, int n, int k, int const *offsets, void const *X, int ldx, void const *Y, int ldy,
    double beta, void *out, int ldd, long strideD, void *work, long work_size)
{
    bool const fast = direct(X, ldx, 0, sizeof(T)) && direct(Y, ldy, 0, sizeof(T));
    if (!fast && (m < 8 || n < 8))
        return launch_kernel(grouped_outer_narrow_kernel<T, D>, dim3((unsigned)std::min((long)m * n / 4 + 1, 16384L), 1, groups), 256, s, 0,
            m, n, k, offsets, (T const *)X, (long)ldx, (T const *)Y, (long)ldy, (float)beta, (D *)out, (long)ldd, strideD);
    Cut c = outer_cut(fast, groups, m, n, k);
    long const plane = (long)groups * m * n * 4;
    // (the tile that is best with slices need not be without: 36501 columns, 1050 x 666: 256 with 16 slices, 64 with
    // one, which takes 168 us instead of 665)
    if (c.slices > 1 && (work == nullptr || work_size < c.slices * plane)) c = outer_cut(fast, groups, m, n, k, 1);
    auto const go = [&](auto *to, int ld, long stride, double b) {
        typedef std::remove_pointer_t<decltype(to)> O;
        auto const launch = c.tile == 256 ? outer_tiles<T, O, ProductTile<T, 256, 256, 2, 4, false, false, DIRECT>>
            : c.tile == 128 ? fast ? outer_tiles<T, O, ProductTile<T, 128, 128, 2, 2, false, false, DIRECT>> : outer_tiles<T, O, ProductTile<T, 128, 128, 2, 2, false, false, STAGED>>
            : fast ? outer_tiles<T, O, ProductTile<T, 64, 64, 1, 1, false, false, DIRECT, 4>> : outer_tiles<T, O, ProductTile<T, 64, 64, 1, 1, false, false, STAGED, 4>>;
        return launch(s, c.slices, groups, m, n, k, offsets, X, ldx, Y, ldy, b, to, ld, stride);
    };
    if (c.slices == 1) return go((D *)out, ldd, strideD, beta);
    hipError_t const e = go((float *)work, m, (long)m * n, 0.0);
    if (e != hipSuccess) return e;
    return outer_sum<float, D>(s, c.slices, groups, m, n, work, beta, out, ldd, strideD);
}

// fp64: as many slices as fill the chip's three workgroups a compute unit, of 256 columns at least
static int douter_slices(long groups, long m, long n, long k)
{
    if (forced_tile) return forced_slices;
    long const tiles = groups * ((m + 63) / 64) * ((n + 63) / 64);
    return (int)std::max(1L, std::min({768 / tiles, k / groups / 256, 64L}));
}

long grouped_outer_work_size(ProductType type, int groups, int m, int n, int k)
{
    if (type == PRODUCT_F64) { int const slices = douter_slices(groups, m, n, k); return slices > 1 ? (long)slices * groups * m * n * 8 : 0; }
    // (whichever way the operands are aligned)
    int const slices = std::max(outer_cut(true, groups, m, n, k).slices, outer_cut(false, groups, m, n, k).slices);
    return slices > 1 ? (long)slices * groups * m * n * 4 : 0;
}

hipError_t grouped_outer(hipStream_t s, ProductType type, ProductType typeD, int groups, int m, int n, int k, int const *offsets,
    void const *X, int ldx, void const *Y, int ldy, double beta, void *D, int ldd, long strideD, void *work, long work_size)
{
    if (type == PRODUCT_F64) {
        int const slices = work != nullptr && work_size >= grouped_outer_work_size(type, groups, m, n, k) ? douter_slices(groups, m, n, k) : 1;
        long const tiles = (long)groups * slices * ((m + 63) / 64) * ((n + 63) / 64);
        if (tiles >= 1L << 31) return hipErrorInvalidConfiguration;
        bool const fast = direct(X, ldx, 0, 8) && direct(Y, ldy, 0, 8);
        hipError_t const e = launch_kernel(fast ? grouped_douter_kernel<true> : grouped_douter_kernel<false>, dim3((unsigned)roundup(tiles, 8)), 256, s,
            fast ? 0 : GemmCfg<64, 64, 16, false, true>::LDS_BYTES,
            groups, m, n, k, slices, offsets, (double const *)X, ldx, (double const *)Y, ldy, slices > 1 ? 0.0 : beta,
            slices > 1 ? (double *)work : (double *)D, slices > 1 ? m : ldd, slices > 1 ? (long)m * n : strideD);
        if (e != hipSuccess || slices == 1) return e;
        return outer_sum<double, double>(s, slices, groups, m, n, work, beta, D, ldd, strideD);
    }
    bool const wide = typeD == PRODUCT_F32;
    auto const launch = type == PRODUCT_BF16 ? (wide ? outer_launch<__bf16, float> : outer_launch<__bf16, __bf16>)
                                             : (wide ? outer_launch<_Float16, float> : outer_launch<_Float16, _Float16>);
    return launch(s, groups, m, n, k, offsets, X, ldx, Y, ldy, beta, D, ldd, strideD, work, work_size);
}

// ---- 8-bit integers ----------------------------------------------------------------------------------------------

template <typename D>
__global__ __launch_bounds__(512)
void gemm_i8_few_kernel(int groups, int m, int n, int k, int const *__restrict__ offsets, signed char const *__restrict__ A, long lda, long strideA,
    float const *__restrict__ scaleA, long strideS, signed char const *__restrict__ B, long ldb, float const *__restrict__ scaleB, D *__restrict__ C, long ldc)
{
    Pieces pieces(offsets, groups, n, 16);
    int const t = tile_of_workgroup((m + 15) / 16 * pieces.total, 0);
    if (t < 0) return;
    Span const s = pieces.at((unsigned)t % (unsigned)pieces.total);
    if (s.empty()) return;
    int const row = (unsigned)t / (unsigned)pieces.total;
    int const r0 = row * 16;
    float const *const sa = scaleA + s.group * strideS + r0;
    few_columns_tile<signed char>(A + s.group * strideA + r0 * lda, lda, m - r0, B + s.begin * ldb, ldb, s.end - s.begin, k,
        [&](int r, int c, int sum) { C[(s.begin + c) * ldc + r0 + r] = (D)scaled(sum, sa[r], scaleB[s.begin + c]); });
}

template <typename D, typename P>
static hipError_t gemm_i8_tiles(hipStream_t s, int groups, int m, int n, int k, int const *offsets, signed char const *A, int lda, long strideA,
    float const *scaleA, long strideS, signed char const *B, int ldb, float const *scaleB, void *C, int ldc)
{
    long const tiles = most_pieces(groups, n, P::BN) * ((m + P::BM - 1) / P::BM);
    if (tiles >= 1L << 31) return hipErrorInvalidConfiguration;
    return launch_kernel(gemm_i8_kernel<D, P>, dim3(resident<P>(tiles)), P::THREADS, s, 0,
        groups, m, n, k, offsets, A, (long)lda, strideA, scaleA, strideS, B, (long)ldb, scaleB, (D *)C, (long)ldc);
}

template <typename D>
static hipError_t gemm_i8_launch(hipStream_t s, int groups, int m, int n, int k, int const *offsets, signed char const *A, int lda, long strideA,
    float const *scaleA, long strideS, signed char const *B, int ldb, float const *scaleB, void *C, int ldc)
{
    if (k >= 16 && few_columns(groups, m, n)) {
        return launch_kernel(gemm_i8_few_kernel<D>, dim3((unsigned)roundup(most_pieces(groups, n, 16) * ((m + 15) / 16), 8)), 512, s, 0,
            groups, m, n, k, offsets, A, (long)lda, strideA, scaleA, strideS, B, (long)ldb, scaleB, (D *)C, (long)ldc);
    }
    bool const fast = direct(A, lda, strideA, 1) && direct(B, ldb, 0, 1);
    if (!fast && k < 16)
        return launch_kernel(grouped_gemm_narrow_kernel<signed char, D>, dim3((unsigned)most_pieces(groups, n, 4), std::min(m, 65535)), 256, s, 0, groups, m, n, k, offsets,
            A, (long)lda, 1L, strideA, scaleA, strideS, B, (long)ldb, scaleB, (D *)C, (long)ldc);
    typedef signed char T;
    int const tile = product_tile(fast, groups, m, n, (k + 127) / 128);
    auto const launch = fast ? tile == 256 ? gemm_i8_tiles<D, ProductTile<T, 256, 256, 2, 4, true, true, DIRECT>> : tile == 128 ? gemm_i8_tiles<D, ProductTile<T, 128, 128, 2, 2, true, true, DIRECT>>
            : gemm_i8_tiles<D, ProductTile<T, 64, 64, 1, 1, true, true, DIRECT, 4>>
        : tile == 128 ? gemm_i8_tiles<D, ProductTile<T, 128, 128, 2, 2, true, true, STAGED>> : gemm_i8_tiles<D, ProductTile<T, 64, 64, 1, 1, true, true, STAGED, 4>>;
    return launch(s, groups, m, n, k, offsets, A, lda, strideA, scaleA, strideS, B, ldb, scaleB, C, ldc);
}

hipError_t gemm_i8(hipStream_t s, ProductType typeC, int groups, int m, int n, int k, int const *offsets, signed char const *A, int lda, long strideA,
    float const *scaleA, long strideS, signed char const *B, int ldb, float const *scaleB, void *C, int ldc)
{
    auto const launch = typeC == PRODUCT_BF16 ? gemm_i8_launch<__bf16> : typeC == PRODUCT_F16 ? gemm_i8_launch<_Float16> : gemm_i8_launch<float>;
    return launch(s, groups, m, n, k, offsets, A, lda, strideA, scaleA, strideS, B, ldb, scaleB, C, ldc);
}

// q = rint(x / s), s = max |x| / 127 of the column, in IEEE fp32 steps: a plain program in fp32 finds the same numbers.
// A column is read once and waits in registers for its maximum, which is taken over the numbers' bits (without the sign they order
// as integers, NaN above infinity above all others).  The quotient is x times the rounded reciprocal of s and two corrections
// by its remainder: the first leaves it within one unit, and from there the second rounds correctly (Markstein's theorem
// on division by multiply-add); a third of the compiler's full division.  Adding 3 * 2^22 rounds to an integer, halves to even, whose low
// byte is then q.
// 8192 columns of 4096 bf16 numbers: 18 - 19 us, 5.4 TB/s of reads and writes.
template <typename T> struct Eight;         // eight numbers as they lie in memory
template <> struct Eight<float> {
    u32x4 v[2];
    __device__ __forceinline__ unsigned top() const
    {
        unsigned t = 0;
        #pragma unroll
        for (int i = 0; i < 8; i++) t = max(t, v[i >> 2][i & 3] & 0x7fffffffu);
        return t;
    }
    __device__ __forceinline__ float at(int i) const { return __uint_as_float(v[i >> 2][i & 3]); }
    static __device__ __forceinline__ float value(unsigned top) { return __uint_as_float(top); }
};
template <typename T> struct EightHalves {
    u32x4 v;
    __device__ __forceinline__ unsigned top() const
    {
        typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
        u16x2 t = {0, 0};
        #pragma unroll
        for (int i = 0; i < 4; i++) t = __builtin_elementwise_max(t, __builtin_bit_cast(u16x2, v[i] & 0x7fff7fffu));
        return max(t.x, t.y);
    }
    __device__ __forceinline__ float at(int i) const { return value(i & 1 ? v[i >> 1] >> 16 : v[i >> 1] & 0xffff); }
    static __device__ __forceinline__ float value(unsigned bits) { return (float)__builtin_bit_cast(T, (unsigned short)bits); }
};
template <> struct Eight<__bf16> : EightHalves<__bf16> {};
template <> struct Eight<_Float16> : EightHalves<_Float16> {};

template <typename T>
__device__ __forceinline__ Eight<T> load_eight(T const *__restrict__ x, int i, int k)
{
    Eight<T> e;
    if (i + 8 <= k) __builtin_memcpy(&e, x + i, sizeof e);
    else {
        T one[8];
        #pragma unroll
        for (int j = 0; j < 8; j++) one[j] = i + j < k ? x[i + j] : (T)0;
        __builtin_memcpy(&e, one, sizeof e);
    }
    return e;
}

struct Divisor { float s, inverse; bool simple; };

template <typename T>
__device__ __forceinline__ void store_eight(signed char *__restrict__ q, int i, int k, Eight<T> const &e, Divisor const &d)
{
    unsigned low[8];
    #pragma unroll
    for (int j = 0; j < 8; j++) {
        float const x = e.at(j);
        float v;
        if (d.simple) {
            v = x * d.inverse;
            v = fmaf(fmaf(-v, d.s, x), d.inverse, v);
            v = fmaf(fmaf(-v, d.s, x), d.inverse, v);
        } else
            v = d.s > 0.f && d.s < INFINITY ? fminf(fmaxf(x / d.s, -127.f), 127.f) : 0.f;       // (also where s is a NaN)
        low[j] = __float_as_uint(v + 12582912.f);
    }
    u32x2 const w = {(low[0] & 255) | (low[1] & 255) << 8 | (low[2] & 255) << 16 | low[3] << 24, (low[4] & 255) | (low[5] & 255) << 8 | (low[6] & 255) << 16 | low[7] << 24};
    if (i + 8 <= k) __builtin_memcpy(q + i, &w, 8);
    else
        #pragma unroll
        for (int j = 0; j < 8; j++)
            if (i + j < k) q[i + j] = (signed char)(w[j >> 2] >> (j & 3) * 8);
}

// WAVES waves a column; HELD: eights a thread keeps in registers (0: the column is longer than that, and is read twice)
template <typename T, int WAVES, int HELD>
__global__ __launch_bounds__(WAVES < 4 ? 256 : 64 * WAVES)
void quantize_i8_kernel(int k, int n, T const *__restrict__ X, long ldx, signed char *__restrict__ Q, long ldq, float *__restrict__ scale)
{
    constexpr int COLUMNS = WAVES < 4 ? 4 / WAVES : 1, T_COL = 64 * WAVES;
    __shared__ unsigned part[COLUMNS * WAVES];
    int const me = threadIdx.x % T_COL;
    long const c = (long)blockIdx.x * COLUMNS + threadIdx.x / T_COL;
    bool const mine = c < n;
    T const *const x = X + (mine ? c : 0) * ldx;
    signed char *const q = Q + (mine ? c : 0) * ldq;
    int const end = mine ? k : 0;
    Eight<T> held[HELD ? HELD : 1];
    unsigned top = 0;
    if (HELD) {
        #pragma unroll
        for (int h = 0; h < HELD; h++) held[h] = load_eight(x, (h * T_COL + me) * 8, end);
        #pragma unroll
        for (int h = 0; h < HELD; h++) top = max(top, held[h].top());
    } else
        for (int i = me * 8; i < end; i += T_COL * 8) top = max(top, load_eight(x, i, end).top());
    #pragma unroll
    for (int d = 32; d > 0; d /= 2) top = max(top, (unsigned)__shfl_xor((int)top, d));
    if (WAVES > 1) {
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
        __syncthreads();
        #pragma unroll
        for (int w = 0; w < WAVES; w++) top = max(top, part[threadIdx.x / T_COL * WAVES + w]);
    }
    Divisor d;
    d.s = Eight<T>::value(top) / 127.f;
    d.inverse = 1.f / d.s;
    d.simple = d.s > 0x1p-100f && d.s < 0x1p100f;       // neither the reciprocal nor a remainder that counts leaves the normal range
    if (mine && me == 0) scale[c] = d.s;
    if (HELD) {
        #pragma unroll
        for (int h = 0; h < HELD; h++) store_eight(q, (h * T_COL + me) * 8, end, held[h], d);
    } else
        for (int i = me * 8; i < end; i += T_COL * 8) store_eight(q, i, end, load_eight(x, i, end), d);
}

template <typename T>
static hipError_t quantize_launch(hipStream_t s, int k, int n, void const *X, int ldx, signed char *Q, int ldq, float *scale)
{
    auto const go = [&](auto kernel, int columns, int threads) {
        return launch_kernel(kernel, dim3((n + columns - 1) / columns), threads, s, 0, k, n, (T const *)X, (long)ldx, Q, (long)ldq, scale);
    };
    // the fewest threads that hold a column in 4 eights each; one workgroup a column from 2048 numbers on
    if (k <= 512 * 2) return go(quantize_i8_kernel<T, 1, 2>, 4, 256);
    if (k <= 512 * 4) return go(quantize_i8_kernel<T, 1, 4>, 4, 256);
    if (k <= 2048 * 2) return go(quantize_i8_kernel<T, 4, 2>, 1, 256);
    if (k <= 2048 * 4) return go(quantize_i8_kernel<T, 4, 4>, 1, 256);
    if (k <= 8192 * 4) return go(quantize_i8_kernel<T, 16, 4>, 1, 1024);
    return go(quantize_i8_kernel<T, 16, 0>, 1, 1024);
}

hipError_t quantize_i8(hipStream_t s, ProductType type, int k, int n, void const *X, int ldx, signed char *Q, int ldq, float *scale)
{
    auto const launch = type == PRODUCT_BF16 ? quantize_launch<__bf16> : type == PRODUCT_F16 ? quantize_launch<_Float16> : quantize_launch<float>;
    return launch(s, k, n, X, ldx, Q, ldq, scale);
}

} // namespace sn

#ifdef SN_TEST_HOOKS   // compiled into libstarneig_amd_test.so only (csrc/Makefile), never into the product library
namespace {
// The bytes that the direct loads of an operand read past its last word, at most over all k-tiles (0: none).  Every word of a chunk is
// read whose four bytes lie in front of the buffer's end.
template <typename T, int ROWS, bool K>
long reads_past(int outers, int k, int ld)
{
    using S = sn::Stream<T, ROWS, K, 256, sn::DIRECT>;
    using O = typename S::O;
    long const end = ((K ? (long)(outers - 1) * ld + k : (long)(k - 1) * ld + outers) * (long)sizeof(T) + 3) / 4 * 4;
    long past = 0;
    for (int kt = 0; kt < (k + O::KT - 1) / O::KT + 2; kt++) {
        int const left = k - kt * O::KT;
        unsigned const bytes = (unsigned)S::bytes(left, outers, ld);
        long const base = (K ? (long)kt * O::KT : (long)kt * O::KT * ld) * (long)sizeof(T);
        for (int e = 0; e < ROWS * 8; e++) {
            if (left <= O::KT && left > 0 && S::behind(e, left)) continue;
            for (int w = 0; w < 4; w++) {
                unsigned long const at = (unsigned long)S::offset(e, outers, ld) + 4 * w;
                if (at + 4 <= bytes && base + (long)at + 4 - end > past) past = base + (long)at + 4 - end;
            }
        }
    }
    return past;
}
template <typename T>
long reads_past(int tile, bool inner_contiguous, int outers, int k, int ld)
{
    auto const f = tile == 64 ? inner_contiguous ? reads_past<T, 64, true> : reads_past<T, 64, false>
        : tile == 128 ? inner_contiguous ? reads_past<T, 128, true> : reads_past<T, 128, false>
        : inner_contiguous ? reads_past<T, 256, true> : reads_past<T, 256, false>;
    return f(outers, k, ld);
}
}
// size: bytes of a number
extern "C" __attribute__((visibility("default")))
long sn_internal_product_reads_past(int size, int tile, int inner_contiguous, int outers, int k, int ld)
{
    return size == 1 ? reads_past<signed char>(tile, true, outers, k, ld) : size == 2 ? reads_past<__bf16>(tile, inner_contiguous, outers, k, ld)
        : inner_contiguous ? reads_past<double, 64, true>(outers, k, ld) : reads_past<double, 64, false>(outers, k, ld);
}
// From here on the offsets of more than 64 groups are looked up `ints` behind those that the pieces are counted from (as if they had changed meanwhile).
extern "C" __attribute__((visibility("default")))
int sn_internal_product_later_offsets(int ints) { return (int)hipMemcpyToSymbol(HIP_SYMBOL(sn::test_later_offsets), &ints, sizeof ints); }
// The tile and the slices of a gradient with aligned or other columns, with scratch memory for so many slices or none (most_slices 1): slices * 1000 + tile
extern "C" __attribute__((visibility("default")))
int sn_internal_product_outer_cut(int aligned, int groups, int m, int n, int k, int most_slices)
{
    sn::Cut const c = sn::outer_cut(aligned, groups, m, n, k, most_slices);
    return c.slices * 1000 + c.tile;
}
// What the rules take a gradient's launch for, in us
extern "C" __attribute__((visibility("default")))
double sn_internal_product_outer_time(int tile, int slices, int aligned, int groups, int m, int n, int k)
{ return sn::outer_time(sn::Cut{tile, slices}, aligned, groups, m, n, k); }
// From here on products by tiles of this size (64, 128, 256 where columns are aligned), sums over columns in this many slices (at least 1);
// 0: as the rules have it.
extern "C" __attribute__((visibility("default")))
void sn_internal_product_force(int tile, int slices) { sn::forced_tile = tile; sn::forced_slices = slices; }
#endif  // SN_TEST_HOOKS
