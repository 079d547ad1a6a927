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

// Where a lane of v_mfma_f32_32x32x16_bf16 reads a tile of LD columns.  The key of a row is that of the row 16 further on, and a step
// of 64 columns changes no bit that the key touches; within 64 columns a step is one of bits that are exclusive-ored anyway.  So three
// offsets do for a whole tile.
template <int LD>
struct TileLane {
    int row, swapped, pair;

    __device__ __forceinline__ TileLane(int lane) {
        const int l32 = lane & 31, half = lane >> 5, q = lane & 3;
        row = l32 * LD + ((half ^ tile_key(l32)) << 3);
        swapped = slice_col(l32) * LD + ((half ^ tile_key(slice_col(l32))) << 3);
        const int r = 8 * half + ((lane & 15) >> 2), c = 16 * ((lane >> 4) & 1) + 4 * (((q & 1) << 1) | (q >> 1));
        pair = r * LD + (((c >> 3) ^ tile_key(r)) << 3) + (c & 7);
    }
    // x where it is used, rather than what follows from x in registers over a whole walk
    __device__ __forceinline__ void recompute() { asm volatile("" : "+v"(row), "+v"(swapped), "+v"(pair)); }
    // 8 columns 16 s + 8 half .. of row row0 + l32; row0 a multiple of 32
    __device__ __forceinline__ bf16x8 fragment(const bf16_t* tile, int row0, int s) const {
        return *reinterpret_cast<const bf16x8*>(tile + (row ^ (16 * (s & 3))) + row0 * LD + (s >> 2) * 64);
    }
    // ... of row row0 + swap(l32)
    __device__ __forceinline__ bf16x8 swapped_fragment(const bf16_t* tile, int row0, int s) const {
        return *reinterpret_cast<const bf16x8*>(tile + (swapped ^ (16 * (s & 3))) + row0 * LD + (s >> 2) * 64);
    }
    // rows 16 s + 8 half .. + 7 of column 32 t + swap(l32)
    __device__ __forceinline__ bf16x8 transposed(const bf16_t* tile, int s, int t) const {
        const bf16_t* const p = tile + 16 * s * LD + (t >> 1) * 64;
        const int at = pair ^ (32 * (t & 1));
        const bf16x4 lo = read(p + at), hi = read(p + (at ^ 8) + 4 * LD);
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
    static __device__ __forceinline__ bf16x4 read(const bf16_t* p) {
        const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
        return __builtin_bit_cast(bf16x4, v);
    }
};

// A thread's share of the rows of one role: granules of 8 columns, ITERS rows apart by STEP.  Addresses are a base that the whole
// workgroup shares, advanced chunk by chunk, and 32 bits of the thread's own (the host checks the strides).  What lies past
// the last row or column is read from the chunk's first row and column instead, and zero by the time it is in LDS: a chunk of no row
// must not be fetched.
template <int COLS, int NT>
struct Stream {
    static constexpr int GRANULES = COLS / 8, STEP = NT / GRANULES, ITERS = LC / STEP;
    static_assert(NT % GRANULES == 0 && LC % STEP == 0, "whole rows");
    const char* base;
    int64_t chunk_bytes, step_bytes;
    uint32_t offset, first;
    int r0;
    bool in_columns;

    // `token`: the first of the walk, uniform over the workgroup
    __device__ __forceinline__ Stream(const LinearRole& role, int b, int h, int64_t token, bool reverse, int c0, int columns, int tid) {
        r0 = tid / GRANULES;
        const int c = (tid % GRANULES) * 8;
        in_columns = c < columns;
        const int64_t row_bytes = role.stride_t * 2;
        const int64_t lowest = reverse ? token - (LC - 1) : token;  // of the first chunk's 64 rows in memory
        base = static_cast<const char*>(role.p) + 2 * (b * role.stride_b + (h / role.div) * role.stride_h + c0) + lowest * row_bytes;
        offset = (uint32_t)((reverse ? LC - 1 - r0 : r0) * row_bytes) + 2 * c;
        first = reverse ? (uint32_t)((LC - 1) * row_bytes) : 0;
        chunk_bytes = (reverse ? -LC : LC) * row_bytes;
        step_bytes = (reverse ? -STEP : STEP) * row_bytes;
    }
    __device__ __forceinline__ bool there(int i, int rows) const { return in_columns && r0 + i * STEP < rows; }
    // the next chunk, all of it, or (`whole` false) the `rows` rows and the columns that there are
    __device__ __forceinline__ void fetch(bf16x8 (&v)[ITERS], int rows, bool whole) {
        if (whole) {
#pragma unroll
            for (int i = 0; i < ITERS; i++) v[i] = *reinterpret_cast<const bf16x8*>(base + i * step_bytes + offset);
        } else {
#pragma unroll
            for (int i = 0; i < ITERS; i++) {
                // (an address of the chunk's, whichever: the first row's)
                v[i] = *reinterpret_cast<const bf16x8*>(base + (there(i, rows) ? offset + (uint32_t)(i * step_bytes) : first));
            }
        }
        base += chunk_bytes;
    }
    template <int LD = COLS>
    __device__ __forceinline__ void stage(bf16_t* tile, const bf16x8 (&v)[ITERS], int rows, bool whole) const {
        bf16_t* const at = tile + r0 * LD + ((threadIdx.x % GRANULES ^ tile_key(r0)) << 3);  // (STEP rows on: the same key)
#pragma unroll
        for (int i = 0; i < ITERS; i++) {
            const int r = r0 + i * STEP;
            const bf16x8 zero = {};
            bf16_t* const to = STEP % 16 == 0 ? at + i * STEP * LD : tile + r * LD + ((threadIdx.x % GRANULES ^ tile_key(r)) << 3);
            *reinterpret_cast<bf16x8*>(to) = whole || there(i, rows) ? v[i] : zero;
        }
    }
};

}  // namespace gdn
