// LDS tiles of 64 rows for the bf16 kernels of linear attention: how rows get there and how fragments of
// v_mfma_f32_32x32x16_bf16 are read from them.
#pragma once

#include "gdn_linear_common.h"

namespace gdn {

constexpr int LC = 64;  // tokens of a chunk

// 16-byte granule g of row r of an LDS tile of LD columns lies at granule g ^ key(r).  LDS has 64 banks of 4 bytes; a read of 16 bytes
// per lane takes 16 lanes at a time, the transposing read of 8 bytes 32.  With this key one granule of 16 consecutive rows, and 4
// neighbouring granules of 4 consecutive rows, touch every bank once.  (Rows of LD = 64 or 192 columns are odd multiples of half the
// banks: the row's lowest bit is in the address already.)
template <int LD>
__device__ __forceinline__ constexpr int tile_key(int r) {
    return LD % 128 == 0 ? ((r & 3) << 2) | ((r >> 2) & 3) : ((r & 2) << 1) | ((r >> 2) & 3);
}

// Where a lane of v_mfma_f32_32x32x16_bf16 reads a tile of LD columns.  The key of a row is that of the row 16 further on, a step of
// PERIOD columns changes no bit that the key touches, and smaller steps are ones of bits that are exclusive-ored anyway.  So three
// offsets do for a whole tile.
template <int LD>
struct TileLane {
    static constexpr int PERIOD = LD % 128 == 0 ? 128 : 64;
    int row, swapped, pair;

    __device__ __forceinline__ TileLane(int lane) {
        const int l32 = lane & 31, half = lane >> 5, q = lane & 3;
        row = l32 * LD + ((half ^ tile_key<LD>(l32)) << 3);
        swapped = slice_col(l32) * LD + ((half ^ tile_key<LD>(slice_col(l32))) << 3);
        const int r = 8 * half + ((lane & 15) >> 2), c = 16 * ((lane >> 4) & 1) + 4 * (((q & 1) << 1) | (q >> 1));
        pair = r * LD + (((c >> 3) ^ tile_key<LD>(r)) << 3) + (c & 7);
    }
    // x where it is used, rather than what follows from x in registers over a whole walk
    __device__ __forceinline__ void recompute() { asm volatile("" : "+v"(row), "+v"(swapped), "+v"(pair)); }
    // 8 columns 16 s + 8 half .. of row row0 + l32; row0 a multiple of 32
    __device__ __forceinline__ bf16x8 fragment(const bf16_t* tile, int row0, int s) const {
        return *reinterpret_cast<const bf16x8*>(tile + (row ^ (16 * s % PERIOD)) + row0 * LD + 16 * s / PERIOD * PERIOD);
    }
    // ... of row row0 + swap(l32)
    __device__ __forceinline__ bf16x8 swapped_fragment(const bf16_t* tile, int row0, int s) const {
        return *reinterpret_cast<const bf16x8*>(tile + (swapped ^ (16 * s % PERIOD)) + row0 * LD + 16 * s / PERIOD * PERIOD);
    }
    // rows 16 s + 8 half .. + 7 of column 32 t + swap(l32)
    __device__ __forceinline__ bf16x8 transposed(const bf16_t* tile, int s, int t) const {
        const bf16_t* const p = tile + 16 * s * LD + 32 * t / PERIOD * PERIOD;
        const int at = pair ^ (32 * t % PERIOD);
        // 4 rows on, the key's lowest bit is the other
        const bf16x4 lo = read(p + at), hi = read(p + (at ^ 8) + 4 * LD);
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
    // 4 rows of 16 columns: lane i of a 16-lane group gets column i of them; lanes 4 r .. 4 r + 3 address row r, 4 columns each
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
    // chunk c, all of it, or (`whole` false) the `rows` rows and the columns that there are; past the caches, which rows that are read once
    // gain nothing from (with the outputs' stores: 255 -> 245 us at 32768 packed tokens, 369 -> 352 training on 4 x 4096)
    __device__ __forceinline__ void fetch_chunk(int c, bf16x8 (&v)[ITERS], int rows, bool whole) const {
        const char* const from = base + c * chunk_bytes;
        if (whole) {
#pragma unroll
            for (int i = 0; i < ITERS; i++) v[i] = __builtin_nontemporal_load(reinterpret_cast<const bf16x8*>(from + i * step_bytes + offset));
        } else {
#pragma unroll
            for (int i = 0; i < ITERS; i++) {
                // (else an address of the chunk's, whichever: the first row's; by bits, a choice between the two members goes through memory)
                const uint32_t here = there(i, rows) ? ~0u : 0u;
                v[i] = *reinterpret_cast<const bf16x8*>(from + (((offset + (uint32_t)(i * step_bytes)) & here) | (first & ~here)));
            }
        }
    }
    // the next chunk
    __device__ __forceinline__ void fetch(bf16x8 (&v)[ITERS], int rows, bool whole) {
        fetch_chunk(0, v, rows, whole);
        base += chunk_bytes;
    }
    template <int LD = COLS>
    __device__ __forceinline__ void stage(bf16_t* tile, const bf16x8 (&v)[ITERS], int rows, bool whole) const {
        bf16_t* const at = tile + r0 * LD + ((threadIdx.x % GRANULES ^ tile_key<LD>(r0)) << 3);  // (STEP rows on: the same key)
#pragma unroll
        for (int i = 0; i < ITERS; i++) {
            const int r = r0 + i * STEP;
            const bf16x8 zero = {};
            bf16_t* const to = STEP % 16 == 0 ? at + i * STEP * LD : tile + r * LD + ((threadIdx.x % GRANULES ^ tile_key<LD>(r)) << 3);
            *reinterpret_cast<bf16x8*>(to) = whole || there(i, rows) ? v[i] : zero;
        }
    }
};

}  // namespace gdn
