// Element types, matrix instructions and the walk over ragged groups of columns, shared by the grouped and the
// 8-bit products (products.hip).
#pragma once
#include "common.h"

namespace sn {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// The matrix instructions.  mul: 32 x 32 bytes by 32 bytes x 32, lane l holds the 16 bytes A[i = l & 31][bytes 16 (l >> 5) ...],
// B[same bytes][j = l & 31] and D[i = 8 (r >> 2) + 4 (l >> 5) + (r & 3)][j = l & 31].  (The products of a 16 x 16 instruction cost the
// same time, but its operands are read from the registers twice as often: more power, and with it a lower clock.)
// mul16: 16 x 64 bytes by 64 bytes x 16, the 16 bytes A[i = l & 15][bytes 16 (l >> 4) ...] and D[i = 4 (l >> 4) + r][j = l & 15].
// The order of the inner index within these bytes is free as long as both operands use the same one.
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
template <typename T> struct Mfma;
template <> struct Mfma<__bf16> {
    typedef f32x16 Acc;
    typedef f32x4 Acc16;
    static __device__ __forceinline__ Acc mul(i32x4 a, i32x4 b, Acc c)
    { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0); }
    static __device__ __forceinline__ Acc16 mul16(i32x4 a, i32x4 b, Acc16 c)
    { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0); }
};
template <> struct Mfma<_Float16> {
    typedef f32x16 Acc;
    typedef f32x4 Acc16;
    static __device__ __forceinline__ Acc mul(i32x4 a, i32x4 b, Acc c)
    { return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0); }
    static __device__ __forceinline__ Acc16 mul16(i32x4 a, i32x4 b, Acc16 c)
    { return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0); }
};
template <> struct Mfma<signed char> {
    typedef i32x16 Acc;
    typedef i32x4 Acc16;
    static __device__ __forceinline__ Acc mul(i32x4 a, i32x4 b, Acc c) { return __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ Acc16 mul16(i32x4 a, i32x4 b, Acc16 c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }
};

// The columns [begin, end) of a group, or of the piece of a group that a workgroup takes.
struct Span
{
    int group, begin, end;
    __device__ __forceinline__ bool empty() const { return begin >= end; }
};

#ifdef SN_TEST_HOOKS
__device__ int test_later_offsets;      // where the offsets are that more than 64 groups are walked over again, behind those that were counted
#endif

// Offsets come from the device (a router's prefix sums) and are not trusted: each is clamped to [0, n] and to its
// predecessors' maximum, so that the groups are disjoint and inside the matrix whatever the array holds.
//
// Prefix sum / prefix maximum of non-negative numbers over the lanes, and the number of the lane before (lane 0: `first`), by the
// cross-lane operands of vector instructions (a shuffle through LDS takes ten times as long, and six of them wait for each other).
template <int CTRL, int ROWS> __device__ __forceinline__ int from_lane(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false); }
__device__ __forceinline__ int prefix_sum(int v)
{
    v += from_lane<0x111, 0xf>(v); v += from_lane<0x112, 0xf>(v); v += from_lane<0x114, 0xf>(v); v += from_lane<0x118, 0xf>(v);
    v += from_lane<0x142, 0xa>(v); v += from_lane<0x143, 0xc>(v);
    return v;
}
__device__ __forceinline__ int prefix_max(int v)
{
    v = max(v, from_lane<0x111, 0xf>(v)); v = max(v, from_lane<0x112, 0xf>(v)); v = max(v, from_lane<0x114, 0xf>(v)); v = max(v, from_lane<0x118, 0xf>(v));
    v = max(v, from_lane<0x142, 0xa>(v)); v = max(v, from_lane<0x143, 0xc>(v));
    return v;
}
__device__ __forceinline__ int lane_before(int v, int first) { return __builtin_amdgcn_update_dpp(first, v, 0x138, 0xf, 0xf, false); }

// The groups cut into pieces of at most `width` columns, in the groups' order.  Every wave walks by itself, 64 groups at a time: a prefix
// maximum for the offsets and a prefix sum for the pieces, no shared memory and no barrier; up to 64 groups
// stay in the lanes, so that a further piece is found without another walk.
struct Pieces {
    int const *offsets;
    int groups, n, width;
    int total;                              // pieces
    int begin, end, first;                  // of the lane's group: its columns, its first piece
    int carry, before;

    __device__ __forceinline__ Pieces(int const *offsets_, int groups_, int n_, int width_) : offsets(offsets_), groups(groups_), n(n_), width(width_)
    {
        start();
        for (int g0 = 0; g0 < groups; g0 += 64) walk(g0);
        total = before;
#ifdef SN_TEST_HOOKS
        if (groups > 64) offsets += test_later_offsets;
#endif
    }
    __device__ __forceinline__ int offset(int g) const { return offsets ? min(max(offsets[g], 0), n) : g ? n : 0; }     // (none: one group of all columns)
    __device__ __forceinline__ void start() { carry = __builtin_amdgcn_readfirstlane(offset(0)); before = 0; }
    __device__ __forceinline__ void walk(int g0)
    {
        int const lane = threadIdx.x & 63, g = g0 + lane;
        end = g < groups ? offset(g + 1) : 0;
        end = max(end, carry);
        end = prefix_max(end);
        begin = lane_before(end, carry);
        int const count = ((unsigned)(end - begin) + width - 1) / (unsigned)width, sum = prefix_sum(count);
        first = before + sum - count;
        before += __builtin_amdgcn_readlane(sum, 63);
        carry = __builtin_amdgcn_readlane(end, 63);
    }
    // Piece number `piece` < total.  Empty where the offsets of more than 64 groups have changed meanwhile, which they must not; the callers
    // take it for no work, so that nothing is read or written outside the matrices.
    __device__ __forceinline__ Span at(int piece)
    {
        if (groups > 64) start();
        for (int g0 = 0; g0 < groups; g0 += 64) {
            if (groups > 64) walk(g0);
            unsigned long long const here = __ballot(piece >= first && (long)(piece - first) * width < end - begin);
            if (here) {
                int const l = __ffsll(here) - 1;
                Span s;
                s.group = g0 + l;
                s.begin = __builtin_amdgcn_readlane(begin, l) + (piece - __builtin_amdgcn_readlane(first, l)) * width;
                s.end = s.begin + min(width, __builtin_amdgcn_readlane(end, l) - s.begin);
                return s;
            }
        }
        return Span{0, 0, 0};
    }
};

// The columns of one group.
__device__ __forceinline__ Span whole_group(int const *__restrict__ offsets, int n, int group)
{
    int const lane = threadIdx.x & 63;
    int top = 0;
    for (int g0 = 0; g0 <= group; g0 += 64)
        if (g0 + lane <= group) top = max(top, min(max(offsets[g0 + lane], 0), n));
    top = __builtin_amdgcn_readlane(prefix_max(top), 63);
    int const end = __builtin_amdgcn_readfirstlane(max(min(max(offsets[group + 1], 0), n), top));
    return Span{group, top, end};
}

// The groups with the longest first (up to 64 groups; more stay in their own order).
struct Longest {
    int const *offsets;
    int groups, n;
    int begin, end, rank;                   // of the lane's group

    __device__ __forceinline__ Longest(int const *offsets_, int groups_, int n_) : offsets(offsets_), groups(groups_), n(n_)
    {
        if (groups > 64) return;
        int const lane = threadIdx.x & 63;
        int const before = __builtin_amdgcn_readfirstlane(min(max(offsets[0], 0), n));
        end = max(lane < groups ? min(max(offsets[lane + 1], 0), n) : 0, before);
        end = prefix_max(end);
        begin = lane_before(end, before);
        int const length = end - begin;
        rank = lane < groups ? 0 : 64;
        for (int g = 0; g < groups; g++) {
            int const other = __builtin_amdgcn_readlane(length, g);
            rank += lane < groups && (other > length || (other == length && g < lane));
        }
    }
    __device__ __forceinline__ Span at(int place)
    {
        if (groups > 64) return whole_group(offsets, n, place);
        int const l = __ffsll((unsigned long long)__ballot(rank == place)) - 1;
        return Span{l, __builtin_amdgcn_readlane(begin, l), __builtin_amdgcn_readlane(end, l)};
    }
};

// The most pieces of `width` columns that `groups` groups of together n columns can have: each group that has a column
// adds at most width - 1 columns of rounding.
static inline long most_pieces(int groups, int n, int width)
{
    long const some = groups < n ? groups : n;
    return ((long)n + some * (width - 1)) / width;
}

// Tile number `turn` of the workgroup, of a grid of a multiple of 8 workgroups: workgroups go round the 8 XCDs, and each XCD gets a
// run of neighbouring tiles, whose operands its own L2 then holds.  Negative: no more tiles.
__device__ __forceinline__ int tile_of_workgroup(int tiles, int turn)
{
    unsigned const each = ((unsigned)tiles + 7) / 8, at = (blockIdx.x >> 3) + (unsigned)turn * (gridDim.x >> 3), t = (blockIdx.x & 7) * each + at;
    return at < each && t < (unsigned)tiles ? (int)t : -1;
}
// Tiles in bands of 8 tile rows, column by column within the band: the 32 workgroups of an XCD hold 8 + 4 operand panels.
__device__ __forceinline__ void row_and_column(int t, int rows, int cols, int &row, int &col)
{
    int const band = (unsigned)t / (8u * cols), in = t - band * 8 * cols, first = band * 8, high = min(rows - first, 8);
    row = first + (unsigned)in % (unsigned)high; col = (unsigned)in / (unsigned)high;
}
// the same value in all lanes, in a scalar register
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ long uniform(long v)
{ return (long)((unsigned long)(unsigned)uniform((int)v) | (unsigned long)(unsigned)uniform((int)(v >> 32)) << 32); }
template <typename P> __device__ __forceinline__ P *uniform(P *p) { return (P *)uniform((long)p); }

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
