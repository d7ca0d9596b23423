// Matrix products over ragged groups of columns: C_g = op(A_g) B_g and D_g = X_g Y_g^T + beta D_g, where group g owns the
// columns [offsets[g], offsets[g + 1]) of B and C (of X and Y) and a matrix of its own; the first also in 8-bit integers with scales.
#include "product_tile.h"
#include "dgemm_tile.h"
#include "products.h"

namespace sn {

template <typename T, typename P>
__global__ __launch_bounds__(P::THREADS, 2)
void grouped_gemm_kernel(int groups, int m, int n, int k, int const *__restrict__ offsets, T const *__restrict__ A, long lda, long strideA,
    T const *__restrict__ B, long ldb, T *__restrict__ C, long ldc, bool aligned)
{
    __shared__ __attribute__((aligned(16))) char lds[P::LDS_BYTES];
    int const rows = (m + P::BM - 1) / P::BM;
    int row = 0;
    Span const s = find_piece(offsets, groups, n, P::BN, [&](int pieces) {
        long const t = tile_of_workgroup((long)rows * pieces);
        int piece = -1;
        if (t >= 0) row_and_column(t, rows, pieces, row, piece);
        return piece;
    });
    if (s.group < 0) return;
    int const r0 = row * P::BM;
    P tile;
    tile.run(A + s.group * strideA + r0 * (P::A_K ? lda : 1L), lda, m - r0, B + s.begin * ldb, ldb, s.end - s.begin, k, lds);
    tile.each([&](int r, int c, auto &&value) {
        if (s.begin + c < s.end) store16(C + (s.begin + c) * ldc + r0 + r, m - r0 - r, aligned, value);
    });
}

template <typename T, typename D, typename P>
__global__ __launch_bounds__(P::THREADS, 2)
void grouped_outer_kernel(int groups, int m, int n, int k, int const *__restrict__ offsets, T const *__restrict__ X, long ldx,
    T const *__restrict__ Y, long ldy, float beta, D *__restrict__ out, long ldd, long strideD, bool aligned)
{
    __shared__ __attribute__((aligned(16))) char lds[P::LDS_BYTES];
    int const rows = (m + P::BM - 1) / P::BM, cols = (n + P::BN - 1) / P::BN;
    long const t = tile_of_workgroup((long)groups * rows * cols);
    if (t < 0) return;
    int row, col;
    row_and_column(t % ((long)rows * cols), rows, cols, row, col);
    Span const s = whole_group(offsets, k, (int)(t / ((long)rows * cols)));
    int const r0 = row * P::BM, c0 = col * P::BN;
    P tile;
    tile.run(X + s.begin * ldx + r0, ldx, m - r0, Y + s.begin * ldy + c0, ldy, n - c0, s.end - s.begin, lds);
    D *const to = out + s.group * strideD;
    tile.each([&](int r, int c, auto &&value) {
        if (c0 + c >= n) return;
        D *const at = to + (c0 + c) * ldd + r0 + r;
        int const left = m - r0 - r;
        if (beta != 0.f) {
            // (all old values are asked for before any is overwritten)
            float old[16];
            #pragma unroll
            for (int e = 0; e < 16; e++) old[e] = e < left ? (float)at[e] : 0.f;
            store16(at, left, aligned, [&](int e) { return value(e) + beta * old[e]; });
        } else
            store16(at, left, aligned, value);
    });
}

// fp64: the tile of the library's own dgemm, one piece of a group a workgroup
template <bool TA>
__global__ __launch_bounds__(256, 2)
void grouped_dgemm_kernel(int groups, int m, int n, int k, int const *__restrict__ offsets, double const *__restrict__ A, int lda, long strideA,
    double const *__restrict__ B, int ldb, double *__restrict__ C, int ldc)
{
    Span const s = find_piece(offsets, groups, n, 64, [](int) { return (int)blockIdx.x; });
    if (s.group < 0) return;
    if (k == 0) {           // (the tile reads its operands' last inner term: there must be one)
        for (int e = threadIdx.x; e < 64 * 64; e += 256) {
            int const r = blockIdx.y * 64 + e % 64, c = s.begin + e / 64;
            if (r < m && c < s.end) C[(size_t)c * ldc + r] = 0.0;
        }
        return;
    }
    gemm_tile<64, 64, 16, TA, false, 16>(m, s.end - s.begin, k, 1.0, A + s.group * strideA, lda, B + (size_t)s.begin * ldb, ldb,
        0.0, C + (size_t)s.begin * ldc, ldc, blockIdx.y, 0);
}

__global__ __launch_bounds__(256, 2)
void grouped_douter_kernel(int m, int n, int k, int const *__restrict__ offsets, double const *__restrict__ X, int ldx,
    double const *__restrict__ Y, int ldy, double beta, double *__restrict__ D, int ldd, long strideD)
{
    Span const s = whole_group(offsets, k, blockIdx.z);
    double *const to = D + s.group * strideD;
    if (s.begin == s.end) {
        for (int e = threadIdx.x; e < 64 * 64; e += 256) {
            int const r = blockIdx.x * 64 + e % 64, c = blockIdx.y * 64 + e / 64;
            if (r < m && c < n) { double *const p = to + (size_t)c * ldd + r; *p = beta == 0.0 ? 0.0 : beta * *p; }
        }
        return;
    }
    gemm_tile<64, 64, 16, false, true, 16>(m, n, s.end - s.begin, 1.0, X + (size_t)s.begin * ldx, ldx, Y + (size_t)s.begin * ldy, ldy,
        beta, to, ldd, blockIdx.x, blockIdx.y);
}

template <bool TA>
static hipError_t dgemm_launch(hipStream_t s, int groups, int m, int n, int k, int const *offsets, double const *A, int lda, long strideA,
    double const *B, int ldb, double *C, int ldc)
{
    return launch_kernel(grouped_dgemm_kernel<TA>, dim3((unsigned)most_pieces(groups, n, 64), (m + 63) / 64), 256, s,
        GemmCfg<64, 64, 16, TA, false>::LDS_BYTES, groups, m, n, k, offsets, A, lda, strideA, B, ldb, C, ldc);
}

// Whether an operand can be fed directly: 16-byte aligned columns of whole chunks, positions within a tile below 2^31 bytes
// (256 columns of up to 4 MB).
static bool direct(void const *p, long ld, long stride, int contiguous, int size)
{
    return (uintptr_t)p % 16 == 0 && ld * size % 16 == 0 && stride * size % 16 == 0 && (long)contiguous * size % 16 == 0 && ld * size <= 1 << 22;
}

template <typename T, typename P>
static hipError_t gemm_tiles(hipStream_t s, int groups, int m, int n, int k, int const *offsets, void const *A, int lda, long strideA,
    void const *B, int ldb, void *C, int ldc)
{
    long const tiles = most_pieces(groups, n, P::BN) * ((m + P::BM - 1) / P::BM);
    bool const aligned = (uintptr_t)C % 16 == 0 && (long)ldc * sizeof(T) % 16 == 0;
    return launch_kernel(grouped_gemm_kernel<T, P>, dim3((unsigned)roundup(tiles, 8)), P::THREADS, s, 0,
        groups, m, n, k, offsets, (T const *)A, (long)lda, strideA, (T const *)B, (long)ldb, (T *)C, (long)ldc, aligned);
}

template <typename T, bool TA>
static hipError_t gemm_launch(hipStream_t s, int groups, int m, int n, int k, int const *offsets, void const *A, int lda, long strideA,
    void const *B, int ldb, void *C, int ldc)
{
    bool const fast = direct(A, lda, strideA, TA ? k : m, sizeof(T)) && direct(B, ldb, 0, k, sizeof(T));
    // (the large tile where it leaves no compute unit idle)
    if (most_pieces(groups, n, 256) * ((m + 255) / 256) >= 256)
    return (fast ? gemm_tiles<T, ProductTile<T, 256, 256, 2, 4, TA, true, DIRECT>> : gemm_tiles<T, ProductTile<T, 128, 128, 2, 2, TA, true, STAGED>>)
        (s, groups, m, n, k, offsets, A, lda, strideA, B, ldb, C, ldc);
    return (fast ? gemm_tiles<T, ProductTile<T, 128, 128, 2, 2, TA, true, DIRECT>> : gemm_tiles<T, ProductTile<T, 128, 128, 2, 2, TA, true, STAGED>>)
        (s, groups, m, n, k, offsets, A, lda, strideA, B, ldb, C, ldc);
}

hipError_t grouped_gemm(hipStream_t s, ProductType type, bool transA, int groups, int m, int n, int k, int const *offsets,
    void const *A, int lda, long strideA, void const *B, int ldb, void *C, int ldc)
{
    if (type == PRODUCT_BF16) return (transA ? gemm_launch<__bf16, true> : gemm_launch<__bf16, false>)(s, groups, m, n, k, offsets, A, lda, strideA, B, ldb, C, ldc);
    if (type == PRODUCT_F16) return (transA ? gemm_launch<_Float16, true> : gemm_launch<_Float16, false>)(s, groups, m, n, k, offsets, A, lda, strideA, B, ldb, C, ldc);
    auto const launch = transA ? dgemm_launch<true> : dgemm_launch<false>;
    return launch(s, groups, m, n, k, offsets, (double const *)A, lda, strideA, (double const *)B, ldb, (double *)C, ldc);
}

template <typename T, typename D, typename P>
static hipError_t outer_tiles(hipStream_t s, int groups, int m, int n, int k, int const *offsets, void const *X, int ldx, void const *Y, int ldy,
    double beta, void *out, int ldd, long strideD)
{
    long const tiles = (long)groups * ((m + P::BM - 1) / P::BM) * ((n + P::BN - 1) / P::BN);
    bool const aligned = (uintptr_t)out % 16 == 0 && (long)ldd * sizeof(D) % 16 == 0 && strideD * (long)sizeof(D) % 16 == 0;
    return launch_kernel(grouped_outer_kernel<T, D, P>, dim3((unsigned)roundup(tiles, 8)), P::THREADS, s, 0,
        groups, m, n, k, offsets, (T const *)X, (long)ldx, (T const *)Y, (long)ldy, (float)beta, (D *)out, (long)ldd, strideD, aligned);
}

template <typename T, typename D>
static hipError_t outer_launch(hipStream_t s, int groups, int m, int n, int k, int const *offsets, void const *X, int ldx, void const *Y, int ldy,
    double beta, void *out, int ldd, long strideD)
{
    bool const fast = direct(X, ldx, 0, m, sizeof(T)) && direct(Y, ldy, 0, n, sizeof(T));
    // (the large tile where it leaves no compute unit idle)
    if ((long)groups * ((m + 255) / 256) * ((n + 255) / 256) >= 256)
    return (fast ? outer_tiles<T, D, ProductTile<T, 256, 256, 2, 4, false, false, DIRECT>> : outer_tiles<T, D, ProductTile<T, 128, 128, 2, 2, false, false, STAGED>>)
        (s, groups, m, n, k, offsets, X, ldx, Y, ldy, beta, out, ldd, strideD);
    return (fast ? outer_tiles<T, D, ProductTile<T, 128, 128, 2, 2, false, false, DIRECT>> : outer_tiles<T, D, ProductTile<T, 128, 128, 2, 2, false, false, STAGED>>)
        (s, groups, m, n, k, offsets, X, ldx, Y, ldy, beta, out, ldd, strideD);
}

hipError_t grouped_outer(hipStream_t s, ProductType type, ProductType typeD, int groups, int m, int n, int k, int const *offsets,
    void const *X, int ldx, void const *Y, int ldy, double beta, void *D, int ldd, long strideD)
{
    if (type == PRODUCT_F64)
        return launch_kernel(grouped_douter_kernel, dim3((m + 63) / 64, (n + 63) / 64, groups), 256, s, GemmCfg<64, 64, 16, false, true>::LDS_BYTES,
            m, n, k, offsets, (double const *)X, ldx, (double const *)Y, ldy, beta, (double *)D, ldd, strideD);
    bool const wide = typeD == PRODUCT_F32;
    auto const launch = type == PRODUCT_BF16 ? (wide ? outer_launch<__bf16, float> : outer_launch<__bf16, __bf16>)
                                             : (wide ? outer_launch<_Float16, float> : outer_launch<_Float16, _Float16>);
    return launch(s, groups, m, n, k, offsets, X, ldx, Y, ldy, beta, D, ldd, strideD);
}

// ---- 8-bit integers ----------------------------------------------------------------------------------------------

// The scaling is three roundings to fp32 and one to the result's type: the empty statement keeps the compiler from fusing the
// second product with the conversion to fp16, whose one rounding would depend on the type of the result.
__device__ __forceinline__ float scaled(int sum, float row, float col)
{
    float v = (float)sum * row * col;
    asm("" : "+v"(v));
    return v;
}

template <typename D, typename P>
__global__ __launch_bounds__(P::THREADS, 2)
void gemm_i8_kernel(int groups, int m, int n, int k, int const *__restrict__ offsets, signed char const *__restrict__ A, long lda, long strideA,
    float const *__restrict__ scaleA, long strideS, signed char const *__restrict__ B, long ldb, float const *__restrict__ scaleB, D *__restrict__ C, long ldc, bool aligned)
{
    __shared__ __attribute__((aligned(16))) char lds[P::LDS_BYTES];
    int const rows = (m + P::BM - 1) / P::BM;
    int row = 0;
    auto const which = [&](int pieces) {
        long const t = tile_of_workgroup((long)rows * pieces);
        int piece = -1;
        if (t >= 0) row_and_column(t, rows, pieces, row, piece);
        return piece;
    };
    Span s;
    if (offsets) s = find_piece(offsets, groups, n, P::BN, which);
    else {
        int const piece = which((n + P::BN - 1) / P::BN);
        s = Span{piece < 0 ? -1 : 0, piece * P::BN, min(n, piece * P::BN + P::BN)};
    }
    if (s.group < 0) return;
    int const r0 = row * P::BM;
    P tile;
    tile.run(A + s.group * strideA + r0 * lda, lda, m - r0, B + s.begin * ldb, ldb, s.end - s.begin, k, lds);
    float const *const sa = scaleA + s.group * strideS + r0;
    tile.each([&](int r, int c, auto &&value) {
        if (s.begin + c >= s.end) return;
        float const col = scaleB[s.begin + c];
        int const left = m - r0 - r;
        store16(C + (s.begin + c) * ldc + r0 + r, left, aligned, [&](int e) { return scaled(value(e), e < left ? sa[r + e] : 0.f, col); });
    });
}

template <typename D, typename P>
static hipError_t gemm_i8_tiles(hipStream_t s, int groups, int m, int n, int k, int const *offsets, signed char const *A, int lda, long strideA,
    float const *scaleA, long strideS, signed char const *B, int ldb, float const *scaleB, void *C, int ldc)
{
    long const tiles = most_pieces(groups, n, P::BN) * ((m + P::BM - 1) / P::BM);
    bool const aligned = (uintptr_t)C % 16 == 0 && (long)ldc * sizeof(D) % 16 == 0;
    return launch_kernel(gemm_i8_kernel<D, P>, dim3((unsigned)roundup(tiles, 8)), P::THREADS, s, 0,
        groups, m, n, k, offsets, A, (long)lda, strideA, scaleA, strideS, B, (long)ldb, scaleB, (D *)C, (long)ldc, aligned);
}

template <typename D>
static hipError_t gemm_i8_launch(hipStream_t s, int groups, int m, int n, int k, int const *offsets, signed char const *A, int lda, long strideA,
    float const *scaleA, long strideS, signed char const *B, int ldb, float const *scaleB, void *C, int ldc)
{
    bool const fast = direct(A, lda, strideA, k, 1) && direct(B, ldb, 0, k, 1);
    typedef signed char T;
    // (the large tile where it leaves no compute unit idle)
    if (most_pieces(groups, n, 256) * ((m + 255) / 256) >= 256)
    return (fast ? gemm_i8_tiles<D, ProductTile<T, 256, 256, 2, 4, true, true, DIRECT>> : gemm_i8_tiles<D, ProductTile<T, 128, 128, 2, 2, true, true, STAGED>>)
        (s, groups, m, n, k, offsets, A, lda, strideA, scaleA, strideS, B, ldb, scaleB, C, ldc);
    return (fast ? gemm_i8_tiles<D, ProductTile<T, 128, 128, 2, 2, true, true, DIRECT>> : gemm_i8_tiles<D, ProductTile<T, 128, 128, 2, 2, true, true, STAGED>>)
        (s, groups, m, n, k, offsets, A, lda, strideA, scaleA, strideS, B, ldb, scaleB, C, ldc);
}

hipError_t gemm_i8(hipStream_t s, ProductType typeC, int groups, int m, int n, int k, int const *offsets, signed char const *A, int lda, long strideA,
    float const *scaleA, long strideS, signed char const *B, int ldb, float const *scaleB, void *C, int ldc)
{
    auto const launch = typeC == PRODUCT_BF16 ? gemm_i8_launch<__bf16> : typeC == PRODUCT_F16 ? gemm_i8_launch<_Float16> : gemm_i8_launch<float>;
    return launch(s, groups, m, n, k, offsets, A, lda, strideA, scaleA, strideS, B, ldb, scaleB, C, ldc);
}

// q = rint(x / s), s = max |x| / 127 of the column, in IEEE fp32 steps (the division is rounded correctly: |q| <= 127 always, and
// a plain program in fp32 finds the same numbers).
template <typename T>
__global__ __launch_bounds__(256)
void quantize_i8_kernel(int k, T const *__restrict__ X, long ldx, signed char *__restrict__ Q, long ldq, float *__restrict__ scale)
{
    __shared__ float part[4];
    T const *const x = X + blockIdx.x * ldx;
    signed char *const q = Q + blockIdx.x * ldq;
    float top = 0.f;
    for (int i = threadIdx.x; i < k; i += 256) {
        float const a = fabsf((float)x[i]);
        top = a > top || a != a ? a : top;      // a NaN stays
    }
    for (int d = 32; d > 0; d /= 2) { float const o = __shfl_xor(top, d); top = o > top || o != o ? o : top; }
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
    __syncthreads();
    top = part[0];
    for (int w = 1; w < 4; w++) top = part[w] > top || part[w] != part[w] ? part[w] : top;
    float const s = top / 127.f;
    if (threadIdx.x == 0) scale[blockIdx.x] = s;
    for (int i = threadIdx.x; i < k; i += 256) {
        float const v = s > 0.f && s < INFINITY ? rintf((float)x[i] / s) : 0.f;
        q[i] = (signed char)(int)fminf(fmaxf(v, -127.f), 127.f);
    }
}

hipError_t quantize_i8(hipStream_t s, ProductType type, int k, int n, void const *X, int ldx, signed char *Q, int ldq, float *scale)
{
    if (type == PRODUCT_BF16) return launch_kernel(quantize_i8_kernel<__bf16>, dim3(n), 256, s, 0, k, (__bf16 const *)X, (long)ldx, Q, (long)ldq, scale);
    if (type == PRODUCT_F16) return launch_kernel(quantize_i8_kernel<_Float16>, dim3(n), 256, s, 0, k, (_Float16 const *)X, (long)ldx, Q, (long)ldq, scale);
    return launch_kernel(quantize_i8_kernel<float>, dim3(n), 256, s, 0, k, (float const *)X, (long)ldx, Q, (long)ldq, scale);
}

} // namespace sn
