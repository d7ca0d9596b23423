// Element types, matrix instructions and the walk over ragged groups of columns, shared by the grouped and the
// 8-bit products (products.hip).
#pragma once
#include "common.h"

namespace sn {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// One matrix instruction multiplies 16 x 64 bytes by 64 bytes x 16: lane l holds the 16 bytes
// A[i = l & 15][bytes 16 (l >> 4) ...], B[same bytes][j = l & 15] and D[i = 4 (l >> 4) + reg][j = l & 15].
// The order of the inner index within the 64 bytes is free as long as both operands use the same one.
template <typename T> struct Mfma;
template <> struct Mfma<__bf16> {
    typedef f32x4 Acc;
    static __device__ __forceinline__ Acc mul(i32x4 a, i32x4 b, Acc c)
    { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0); }
};
template <> struct Mfma<_Float16> {
    typedef f32x4 Acc;
    static __device__ __forceinline__ Acc mul(i32x4 a, i32x4 b, Acc c)
    { return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0); }
};
template <> struct Mfma<signed char> {
    typedef i32x4 Acc;
    static __device__ __forceinline__ Acc mul(i32x4 a, i32x4 b, Acc c)
    { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }
};

// The columns [begin, end) of a group, or of the piece of a group that a workgroup takes.
struct Span { int group, begin, end; };

// Offsets come from the device (a router's prefix sums) and are not trusted: each is clamped to [0, n] and to its
// predecessors' maximum, so that the groups are disjoint and inside the matrix whatever the array holds.
//
// The groups are cut into pieces of at most `width` columns, in the groups' order; which(number of pieces) names the piece
// that the caller wants (negative: none).  Every wave walks by itself, 64 groups at a time: a prefix maximum for
// the offsets and a prefix sum for the pieces, no shared memory and no barrier.
template <typename F>
__device__ __forceinline__ Span find_piece(int const *__restrict__ offsets, int groups, int n, int width, F &&which)
{
    int const lane = threadIdx.x & 63;
    int begin, first, count, end, carry, before;
    auto const start = [&]() { carry = min(max(offsets[0], 0), n); before = 0; };
    auto const walk = [&](int g0) {
        int const g = g0 + lane;
        end = g < groups ? min(max(offsets[g + 1], 0), n) : 0;
        end = max(end, carry);
        #pragma unroll
        for (int d = 1; d < 64; d *= 2) { int const o = __shfl_up(end, d); if (lane >= d) end = max(end, o); }
        begin = __shfl_up(end, 1);
        if (lane == 0) begin = carry;
        count = (end - begin + width - 1) / width;
        int sum = count;
        #pragma unroll
        for (int d = 1; d < 64; d *= 2) { int const o = __shfl_up(sum, d); if (lane >= d) sum += o; }
        first = before + sum - count;
        before += __builtin_amdgcn_readlane(sum, 63);
        carry = __builtin_amdgcn_readlane(end, 63);
    };
    start();
    for (int g0 = 0; g0 < groups; g0 += 64) walk(g0);
    int const piece = which(before);
    if (piece < 0 || piece >= before) return Span{-1, 0, 0};
    if (groups > 64) start();
    for (int g0 = 0;; g0 += 64) {
        if (groups > 64) walk(g0);
        unsigned long long const here = __ballot(piece >= first && piece < first + count);
        if (here) {
            int const l = __ffsll(here) - 1;
            Span s;
            s.group = g0 + l;
            s.begin = __builtin_amdgcn_readlane(begin, l) + (piece - __builtin_amdgcn_readlane(first, l)) * width;
            s.end = min(s.begin + width, __builtin_amdgcn_readlane(end, l));
            return s;
        }
    }
}

// The columns of one group.
__device__ __forceinline__ Span whole_group(int const *__restrict__ offsets, int n, int group)
{
    int const lane = threadIdx.x & 63;
    int top = 0;
    for (int g0 = 0; g0 <= group; g0 += 64)
        if (g0 + lane <= group) top = max(top, min(max(offsets[g0 + lane], 0), n));
    #pragma unroll
    for (int d = 32; d > 0; d /= 2) top = max(top, __shfl_xor(top, d));
    top = __builtin_amdgcn_readfirstlane(top);
    int const end = __builtin_amdgcn_readfirstlane(max(min(max(offsets[group + 1], 0), n), top));
    return Span{group, top, end};
}

// The most pieces of `width` columns that `groups` groups of together n columns can have: each group that has a column
// adds at most width - 1 columns of rounding.
static inline long most_pieces(int groups, int n, int width)
{
    long const some = groups < n ? groups : n;
    return ((long)n + some * (width - 1)) / width;
}

// Workgroup `id` of a grid of at least roundup(tiles, 8) workgroups -> tile: workgroups go round the 8 XCDs, and each XCD gets a
// run of neighbouring tiles, whose operands its own L2 then holds.  Negative: no tile.
__device__ __forceinline__ long tile_of_workgroup(long tiles)
{
    long const each = (tiles + 7) / 8, at = blockIdx.x >> 3, t = (blockIdx.x & 7) * each + at;
    return at < each && t < tiles ? t : -1;
}
// Tiles in bands of 8 tile rows, column by column within the band: the 32 workgroups of an XCD hold 8 + 4 operand panels.
__device__ __forceinline__ void row_and_column(long t, int rows, int cols, int &row, int &col)
{
    long const band = t / (8L * cols), in = t % (8L * cols);
    int const first = (int)band * 8, high = min(rows - first, 8);
    row = first + (int)(in % high); col = (int)(in / high);
}

// hipLaunchKernel with the error of this launch alone as its result (hipGetLastError would hand out, and clear,
// an earlier call's).
template <typename... P, typename... A>
static inline hipError_t launch_kernel(void (*kernel)(P...), dim3 grid, int threads, hipStream_t s, int lds, A... args)
{
    if (grid.x == 0 || grid.y == 0 || grid.z == 0) return hipSuccess;
    if ((unsigned long long)grid.x * threads >= 1ULL << 32 || grid.y > 65535 || grid.z > 65535) return hipErrorInvalidConfiguration;
    return [&](P... p) {
        void *at[] = {(void *)&p...};
        return hipLaunchKernel((void const *)kernel, grid, dim3(threads), at, lds, s);
    }(args...);
}

} // namespace sn
