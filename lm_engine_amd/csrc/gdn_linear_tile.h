// LDS tiles of 64 rows for the bf16 kernels of linear attention: how rows get there and how fragments of
// v_mfma_f32_32x32x16_bf16 are read from them.
#pragma once

#include "gdn_linear_common.h"

namespace gdn {

constexpr int LC = 64;  // tokens of a chunk

// 16-byte granule g of row r of an LDS tile lies at granule g ^ key(r): 8 lanes that read one granule of 8 consecutive rows, or of
// rows {0 - 3, 8 - 11} (the swapped order), and 16 lanes that read two neighbouring granules of 4 rows (the transposing read), then
// touch every bank once.
__device__ __forceinline__ int tile_key(int r) { return ((r & 3) << 1) | (((r >> 2) ^ (r >> 3)) & 1); }

template <int LD>
__device__ __forceinline__ bf16x8 tile_row8(const bf16_t* m, int row, int granule) {
    return *reinterpret_cast<const bf16x8*>(m + row * LD + ((granule ^ tile_key(row)) << 3));
}

// lane i of a 16-lane group: rows row0 .. row0 + 3 of column col0 + sigma(i), sigma the swap of bits 2 and 3
template <int LD>
__device__ __forceinline__ bf16x4 tile_tr4(const bf16_t* m, int row0, int col0, int l16) {
    const int q = l16 & 3, row = row0 + (l16 >> 2);
    const int col = col0 + 4 * (((q & 1) << 1) | (q >> 1));
    const bf16_t* p = m + row * LD + (((col >> 3) ^ tile_key(row)) << 3) + (col & 7);
    const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
    return __builtin_bit_cast(bf16x4, v);
}

// A operand: row m = column col0 + swap(m) of the tile, reduction index = rows row0 + 0 .. 15
template <int LD>
__device__ __forceinline__ bf16x8 tile_tr8(const bf16_t* m, int row0, int col0, int lane) {
    const int r = row0 + 8 * (lane >> 5), c = col0 + 16 * ((lane >> 4) & 1), l16 = lane & 15;
    const bf16x4 lo = tile_tr4<LD>(m, r, c, l16), hi = tile_tr4<LD>(m, r + 4, c, l16);
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// A thread's share of the rows of one role: granules of 8 columns, ITERS rows apart by STEP.
template <int COLS, int NT>
struct Stream {
    static constexpr int GRANULES = COLS / 8, STEP = NT / GRANULES, ITERS = LC / STEP;
    static_assert(NT % GRANULES == 0 && LC % STEP == 0, "whole rows");
    const bf16_t* p;    // this thread's granule of the chunk's first row
    int64_t row;        // elements from a row to the next one of the walk
    int r0;
    bool in_columns;
    bf16x8 v[ITERS];

    __device__ __forceinline__ Stream(const LinearRole& role, int b, int h, int64_t token, bool reverse, int c0, int columns, int tid) {
        r0 = tid / GRANULES;
        const int c = (tid % GRANULES) * 8;
        in_columns = c < columns;
        row = reverse ? -role.stride_t : role.stride_t;
        p = static_cast<const bf16_t*>(role.p) + b * role.stride_b + (h / role.div) * role.stride_h + token * role.stride_t + c0 + c + r0 * row;
    }
    __device__ __forceinline__ void load(int rows) {  // of the chunk; the rest is zero
#pragma unroll
        for (int i = 0; i < ITERS; i++) {
            bf16x8 x = {};
            if (in_columns && r0 + i * STEP < rows) x = *reinterpret_cast<const bf16x8*>(p + (int64_t)(i * STEP) * row);
            v[i] = x;
        }
        p += LC * row;
    }
    __device__ __forceinline__ void store(bf16_t* tile) const {
        const int g = threadIdx.x % GRANULES;
#pragma unroll
        for (int i = 0; i < ITERS; i++) {
            const int r = r0 + i * STEP;
            *reinterpret_cast<bf16x8*>(tile + r * COLS + ((g ^ tile_key(r)) << 3)) = v[i];
        }
    }
};

}  // namespace gdn
