// Partial softmax results over parts of a row's keys, joined: o = sum_s w_s o_s / sum_s w_s l_s with w_s = 2^(m_s - max m).
#pragma once

#include "gdn_common.h"

namespace gdn {

constexpr int JOIN_MOST = 128;  // parts

// One row by 256 threads: `part_m` [parts, rows, 2] has m and l, `part_o` [parts, rows, D] the sums.  All parts' loads are on their way at once:
// a thread has four columns of every 256 / (D / 4)th part.  True for the threads that then have columns col .. col + 3 of the row.
// (A part of no key has the lowest m and zeros.)
__device__ __forceinline__ bool join_row(const float* part_o, const float* part_m, int64_t rows, int64_t at, int parts, int D, float& m, float& l, f32x4& o, int& col) {
    __shared__ float weights[JOIN_MOST], shared_m[2], shared_l[2];
    __shared__ f32x4 shared_o[256];
    const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE;
    float own_m = -3.402823466e38f, own_l = 0.f;
    if ((int)threadIdx.x < parts) {
        const f32x2 x = *reinterpret_cast<const f32x2*>(part_m + 2 * (threadIdx.x * rows + at));
        own_m = x.x, own_l = x.y;
    }
    float top = own_m;
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, WAVE));
    if (lane == 0 && wave < 2) shared_m[wave] = top;
    __syncthreads();
    m = fmaxf(shared_m[0], shared_m[1]);
    const float weight = __builtin_amdgcn_exp2f(own_m - m);
    if ((int)threadIdx.x < parts) weights[threadIdx.x] = weight;
    own_l = wave_sum(weight * own_l);
    if (lane == 0 && wave < 2) shared_l[wave] = own_l;
    int quads = 4;
    while (4 * quads < D) quads *= 2;
    const int groups = 256 / quads, group = threadIdx.x / quads;
    col = 4 * (threadIdx.x % quads);
    __syncthreads();
    l = shared_l[0] + shared_l[1];
    o = f32x4{0.f, 0.f, 0.f, 0.f};
    if (col < D) {
#pragma unroll 8
        for (int s = group; s < parts; s += groups) o += *reinterpret_cast<const f32x4*>(part_o + (s * rows + at) * D + col) * weights[s];
    }
    shared_o[threadIdx.x] = o;
    __syncthreads();
    if (group != 0 || col >= D) return false;
    for (int g = 1; g < groups; g++) o += shared_o[g * quads + col / 4];
    return true;
}

}  // namespace gdn
