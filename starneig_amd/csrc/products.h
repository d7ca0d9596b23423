// Grouped and 8-bit matrix products (products.hip): host interface.  All calls enqueue on `s` and
// return the launch's error; arguments are checked by the callers in capi.hip.
#pragma once
#include "common.h"

namespace sn {

// starneig_amd_type_t of include/starneig_amd.h
enum ProductType { PRODUCT_F64 = 0, PRODUCT_F32 = 1, PRODUCT_BF16 = 2, PRODUCT_F16 = 3 };

// C(:, c) = op(A_g) B(:, c) for the columns c of group g; offsets: groups + 1 numbers on the device
hipError_t grouped_gemm(hipStream_t s, ProductType type, bool transA, int groups, int m, int n, int k, int const *offsets,
    void const *A, int lda, long strideA, void const *B, int ldb, void *C, int ldc);
// D_g = X_g Y_g^T + beta D_g over the columns of group g; k columns in all
hipError_t grouped_outer(hipStream_t s, ProductType type, ProductType typeD, int groups, int m, int n, int k, int const *offsets,
    void const *X, int ldx, void const *Y, int ldy, double beta, void *D, int ldd, long strideD, void *work, long work_size);
// bytes of `work` with which it is fastest (0: none; with less it runs without)
long grouped_outer_work_size(ProductType type, int groups, int m, int n, int k);
// C(r, c) = scaleA_g(r) scaleB(c) sum_i A_g(i, r) B(i, c); offsets NULL: one group of all columns
hipError_t gemm_i8(hipStream_t s, ProductType typeC, int groups, int m, int n, int k, int const *offsets, signed char const *A, int lda, long strideA,
    float const *scaleA, long strideS, signed char const *B, int ldb, float const *scaleB, void *C, int ldc);
// Q(:, c) = rint(X(:, c) / scale(c)), scale(c) = max |X(:, c)| / 127
hipError_t quantize_i8(hipStream_t s, ProductType type, int k, int n, void const *X, int ldx, signed char *Q, int ldq, float *scale);

} // namespace sn
