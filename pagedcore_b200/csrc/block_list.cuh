// A decode batch as the split attention kernels over quantised caches walk it: the rows'
// block tables form one flat list, and a CTA works on a contiguous piece of it.
//
// Args holds batch, capacity and error_flag, and gives prefix_at(row) and length_at(row).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "pagedkv.h"
#include "ptx.cuh"

namespace pkv {

// The batch's block count, from the device so that a captured launch serves changing batches.
template <typename Args>
__device__ __forceinline__ int total_blocks(const Args &a) {
    const int total = a.prefix_at(a.batch);
    if (total >= 0 && total <= a.capacity) return total;
    atomicOr(a.error_flag, PKV_DEVICE_BAD_BLOCK);
    return 0;
}

// Whether row `row` breaks the order of the list: it begins at block 0 and no row ends
// before it begins.  Such a list is reported, and no partial is written where the plan has
// no room for one.
__device__ __forceinline__ bool out_of_order(int row, int first, int last) {
    return last < first || (row == 0 && first != 0);
}

// Rows of the block list: where each begins and ends.  32 rows from `base` in registers.
struct Rows {
    int base, first, last, length;
};

template <typename Args>
__device__ __forceinline__ Rows load_rows(const Args &a, int base, int lane) {
    const int r = base + lane;
    if (r >= a.batch) return Rows{base, INT32_MAX, INT32_MAX, 0};
    return Rows{base, a.prefix_at(r), a.prefix_at(r + 1), a.length_at(r)};
}

// The first row at or after `row` that has blocks past `block`, with its window.
template <typename Args>
__device__ __forceinline__ int advance_row(const Args &a, Rows &w, int row, int block, int lane) {
    while (true) {
        if (row - w.base >= 32) w = load_rows(a, row, lane);
        const unsigned past = __ballot_sync(0xffffffffu, w.base + lane >= row && w.last > block);
        if (past != 0) return w.base + __ffs(past) - 1;
        row = w.base + 32;
    }
}

// Over the eight lanes that differ in lane / 4.
__device__ __forceinline__ float max8(float v) {
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
    return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
}

__device__ __forceinline__ float sum8(float v) {
    v += __shfl_xor_sync(0xffffffffu, v, 4);
    v += __shfl_xor_sync(0xffffffffu, v, 8);
    return v + __shfl_xor_sync(0xffffffffu, v, 16);
}

// Partial results of a head joined: maximum, normaliser and four dims of the sum.
struct Merge {
    float M, L, A[4];

    __device__ __forceinline__ void add(float m, float l, const float4 &v) {
        const float top = fmaxf(M, m);
        const float x = exp2_approx(M - top), y = exp2_approx(m - top);
        M = top;
        L = fmaf(L, x, l * y);
        A[0] = fmaf(A[0], x, v.x * y);
        A[1] = fmaf(A[1], x, v.y * y);
        A[2] = fmaf(A[2], x, v.z * y);
        A[3] = fmaf(A[3], x, v.w * y);
    }
};

}  // namespace pkv
