// Softmax attention over a window in fp32, forward and backward (gdn_window_attention.h): the walks of the bf16 kernels on
// v_mfma_f32_16x16x4_f32, 16 rows (or keys) to a wave and tiles of 32 keys (or rows).  An accumulator's register r of lane (n, g) is row
// 4 g + r of column n, and the fp32 product takes its operand one row of four lanes at a time: register r goes on as it is, against rows
// 4 g + r of the other operand, whichever way round that one is read.
// The weights are 2^(c s - m) / l with the m and l of the forward, kept as two numbers: as one, log2 of the sum, their rounding would come back
// relative in every weight (4e-7 at 16).
#include <algorithm>

#include "gdn_launch.h"
#include "gdn_window_attention.h"

namespace gdn {

namespace {

__device__ __forceinline__ f32x4 mma4(float a, float b, const f32x4& c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

constexpr int TILE = 32;

// rows of 4 columns more than they have: 16 rows, or 16 columns of every fourth row, touch all banks once
template <int DP>
struct Tile {
    static constexpr int LD = DP + 4, ITERS = TILE * DP / 4 / 256;
};

template <int DP>
struct Fetched {
    f32x4 v[Tile<DP>::ITERS];
};

// `offset(row)`: elements from base; rows past `count` and columns past D are zeros
template <int DP, typename Offset>
__device__ __forceinline__ void fetch(const float* base, const Offset& offset, int count, int D, Fetched<DP>& f) {
#pragma unroll
    for (int i = 0; i < Tile<DP>::ITERS; i++) {
        const int at = threadIdx.x + 256 * i, row = at / (DP / 4), col = 4 * (at % (DP / 4));
        const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
        f.v[i] = row < count && col < D ? *reinterpret_cast<const f32x4*>(base + offset(row) + col) : zero;
    }
}
template <int DP>
__device__ __forceinline__ void stage(float* tile, const Fetched<DP>& f) {
#pragma unroll
    for (int i = 0; i < Tile<DP>::ITERS; i++) {
        const int at = threadIdx.x + 256 * i, row = at / (DP / 4), col = 4 * (at % (DP / 4));
        *reinterpret_cast<f32x4*>(tile + row * Tile<DP>::LD + col) = f.v[i];
    }
}

// columns 4 s + g of a row in memory
template <int DP>
__device__ __forceinline__ void load_row(const float* row, int D, int g, bool there, float (&f)[DP / 4]) {
#pragma unroll
    for (int s = 0; s < DP / 4; s++) f[s] = there && 4 * s < D ? row[4 * s + g] : 0.f;
}

// sum over columns of (rows 16 x + lane & 15 of the tile) times a row held as load_row has it
template <int DP>
__device__ __forceinline__ f32x4 scores(const float* tile, int x, int lane, const float (&f)[DP / 4]) {
    const float* const row = tile + (16 * x + (lane & 15)) * Tile<DP>::LD + (lane >> 4);
    f32x4 a = {0.f, 0.f, 0.f, 0.f}, b = a;
#pragma unroll
    for (int s = 0; s < DP / 4; s += 2) a = mma4(row[4 * s], f[s], a), b = mma4(row[4 * s + 4], f[s + 1], b);
    return a + b;
}
// acc[t] += columns 16 t + .. of the tile's rows 16 x .. + 15, weighted by w
template <int DP>
__device__ __forceinline__ void add_rows(const float* tile, int x, int lane, const f32x4& w, f32x4 (&acc)[DP / 16]) {
#pragma unroll
    for (int r = 0; r < 4; r++) {
        const float* const row = tile + (16 * x + 4 * (lane >> 4) + r) * Tile<DP>::LD + (lane & 15);
#pragma unroll
        for (int t = 0; t < DP / 16; t++) acc[t] = mma4(row[16 * t], w[r], acc[t]);
    }
}
template <int DP>
__device__ __forceinline__ void store_row(float* row, int D, int g, const f32x4 (&acc)[DP / 16], float by) {
#pragma unroll
    for (int t = 0; t < DP / 16; t++) {
        const int c = 16 * t + 4 * g;
        if (c < D) *reinterpret_cast<f32x4*>(row + c) = acc[t] * by;
    }
}

__device__ __forceinline__ float over_groups(float x, bool largest) {
#pragma unroll
    for (int off = 16; off <= 32; off <<= 1) {
        const float y = __shfl_xor(x, off, WAVE);
        x = largest ? fmaxf(x, y) : x + y;
    }
    return x;
}

// What the two walks over keys have in common: where a workgroup's rows and tiles are.
struct KeyWalk {
    int b, hk, lane, wave, g, r0, row, r, t, head;
    RowView view;
    WaveView w, all;
    int sink_tiles, tiles;
    __device__ __forceinline__ bool begin(const WindowParams& p, int (&bounds)[4][6]) {
        int pair, block;
        if (!work_item(p, blockIdx.x, pair, block)) return false;
        block = p.blocks - 1 - block;
        b = pair / p.HK, hk = pair - b * p.HK;
        lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), g = lane >> 4;
        r0 = block * WINDOW_ROWS_F32, row = r0 + 16 * wave + (lane & 15), r = min(row, p.rows - 1);
        t = r / p.G, head = hk * p.G + (r - t * p.G);
        view = row_view(p, b, r);
        w = wave_view(view);
        all = join_waves<4>(w, bounds, wave, lane);
        all.sink_end = min(all.sink_end, all.lo);
        sink_tiles = all.sink_end > all.sink ? (all.sink_end - all.sink + TILE - 1) / TILE : 0;
        tiles = sink_tiles + (all.end > all.lo ? (all.end - all.lo + TILE - 1) / TILE : 0);
        return true;
    }
    __device__ __forceinline__ void tile_at(int i, int& j0, int& count) const {
        const bool s = i < sink_tiles;
        j0 = s ? all.sink + TILE * i : all.lo + TILE * (i - sink_tiles);
        count = min((s ? all.sink_end : all.end) - j0, TILE);
    }
    __device__ __forceinline__ bool seen_by_all(int i, int j0) const { return i >= sink_tiles && j0 >= all.full_lo && j0 + TILE <= all.full_end; }
};

template <int DP>
__global__ __launch_bounds__(256, DP <= 64 ? 2 : 1) void window_fwd_f32_kernel(const WindowParams p) {
    __shared__ __attribute__((aligned(16))) float kt[TILE * Tile<DP>::LD], vt[TILE * Tile<DP>::LD];
    __shared__ int bounds[4][6];
    KeyWalk x;
    if (!x.begin(p, bounds)) return;
    float q[DP / 4];
    load_row<DP>(static_cast<const float*>(p.q.p) + x.b * p.q.b + x.t * p.q.t + x.head * p.q.h, p.D, x.g, true, q);
    if (p.negative)
#pragma unroll
        for (int s = 0; s < DP / 4; s++) q[s] = -q[s];
    int first = 0, last = x.tiles;
    if (p.splits > 1) {
        const int each = (last + p.splits - 1) / p.splits;
        first = min((int)blockIdx.y * each, last), last = min(first + each, last);
    }
    const float* const kb = static_cast<const float*>(p.k.p) + x.b * p.k.b + x.hk * p.k.h;
    const float* const vb = static_cast<const float*>(p.v.p) + x.b * p.v.b + x.hk * p.v.h;
    Fetched<DP> kf, vf;
    auto fetch_tile = [&](int i) {
        int j0, count;
        x.tile_at(i, j0, count);
        fetch<DP>(kb, [&](int row) { return (j0 + row) * p.k.t; }, count, p.D, kf);
        fetch<DP>(vb, [&](int row) { return (j0 + row) * p.v.t; }, count, p.D, vf);
    };
    f32x4 o[DP / 16] = {};
    float m = LOWEST, l = 0.f;
    bool taken_out = false;
    if (first < last) fetch_tile(first);
    for (int i = first; i < last; i++) {
        int j0, count;
        x.tile_at(i, j0, count);
        if (!x.seen_by_all(i, j0)) {  // (as in the bf16 kernel: 0 times what is not finite)
            bool found = false;
#pragma unroll
            for (int y = 0; y < Tile<DP>::ITERS; y++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (!(fabsf(vf.v[y][e]) < __builtin_inff())) vf.v[y][e] = 0.f, found = true;
            taken_out |= __syncthreads_or(found) != 0;
        } else {
            __syncthreads();
        }
        stage<DP>(kt, kf);
        stage<DP>(vt, vf);
        __syncthreads();
        if (i + 1 < last) fetch_tile(i + 1);
        TileView own(x.view, i >= x.sink_tiles, x.all.sink_end);
        if (i < x.sink_tiles) own.first = own.span, own.st = own.from;
        f32x4 s[2];
        float top = -__builtin_inff();
#pragma unroll
        for (int y = 0; y < 2; y++) {
            s[y] = scores<DP>(kt, y, x.lane, q);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (!own.sees_mixed(j0 + 16 * y + 4 * x.g + e)) s[y][e] = -__builtin_inff();
                else top = fmaxf(top, s[y][e] * p.c);
            }
        }
        top = over_groups(top, true);
        const float next = fmaxf(m, top), alpha = __builtin_amdgcn_exp2f(m - next);
        m = next;
        float sum = 0.f;
#pragma unroll
        for (int y = 0; y < 2; y++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                s[y][e] = s[y][e] == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(__builtin_fmaf(s[y][e], p.c, -m));
                sum += s[y][e];
            }
        l = l * alpha + sum;
#pragma unroll
        for (int z = 0; z < DP / 16; z++) o[z] *= alpha;
#pragma unroll
        for (int y = 0; y < 2; y++) add_rows<DP>(vt, y, x.lane, s[y], o);
    }
    l = over_groups(l, false);
    const int64_t part = (((int64_t)blockIdx.y * p.B + x.b) * p.HK + x.hk) * p.rows + x.r0;
    if (x.row < p.rows) {
        if (p.splits > 1) {
            const int64_t at = part + x.row - x.r0;
            if (x.g == 0) p.part_m[2 * at] = m, p.part_m[2 * at + 1] = l;
            store_row<DP>(p.part_o + at * p.D, p.D, x.g, o, 1.f);
        } else {
            const int64_t head = ((int64_t)x.b * p.T + x.t) * p.H + x.head;
            const float by = l == 0.f ? 0.f : 1.f / l;
            if (p.lse != nullptr && x.g == 0) p.lse[2 * head] = l == 0.f ? 0.f : m, p.lse[2 * head + 1] = by;
            store_row<DP>(static_cast<float*>(const_cast<void*>(p.o.p)) + x.b * p.o.b + x.t * p.o.t + x.head * p.o.h, p.D, x.g, o, by);
        }
    }
    if (taken_out) add_taken_out<float>(p, x.b, x.hk, x.r0, WINDOW_ROWS_F32, x.all, first, last, x.sink_tiles, [&](int i, int& j0, int& count) { x.tile_at(i, j0, count); }, part);
}

template <int DP>
__global__ __launch_bounds__(256, 1) void window_dq_f32_kernel(const WindowParams p) {
    __shared__ __attribute__((aligned(16))) float kt[TILE * Tile<DP>::LD], vt[TILE * Tile<DP>::LD];
    __shared__ int bounds[4][6];
    KeyWalk x;
    if (!x.begin(p, bounds)) return;
    float q[DP / 4], d[DP / 4];
    load_row<DP>(static_cast<const float*>(p.q.p) + x.b * p.q.b + x.t * p.q.t + x.head * p.q.h, p.D, x.g, true, q);
    load_row<DP>(static_cast<const float*>(p.dout.p) + x.b * p.dout.b + x.t * p.dout.t + x.head * p.dout.h, p.D, x.g, true, d);
    const int64_t scalar = ((int64_t)x.b * p.T + x.t) * p.H + x.head;
    float delta = 0.f;
    {
        const float* const o = static_cast<const float*>(p.o.p) + x.b * p.o.b + x.t * p.o.t + x.head * p.o.h;
#pragma unroll
        for (int s = 0; s < DP / 4; s++) delta += 4 * s < p.D ? o[4 * s + x.g] * d[s] : 0.f;
        delta = over_groups(delta, false);
        if (x.g == 0 && x.row < p.rows) p.delta[scalar] = delta;
    }
    const float m = p.lse[2 * scalar], by = p.lse[2 * scalar + 1], c = p.negative ? -p.c : p.c;
    const float* const kb = static_cast<const float*>(p.k.p) + x.b * p.k.b + x.hk * p.k.h;
    const float* const vb = static_cast<const float*>(p.v.p) + x.b * p.v.b + x.hk * p.v.h;
    Fetched<DP> kf, vf;
    auto fetch_tile = [&](int i) {
        int j0, count;
        x.tile_at(i, j0, count);
        fetch<DP>(kb, [&](int row) { return (j0 + row) * p.k.t; }, count, p.D, kf);
        fetch<DP>(vb, [&](int row) { return (j0 + row) * p.v.t; }, count, p.D, vf);
    };
    f32x4 dq[DP / 16] = {};
    if (x.tiles > 0) fetch_tile(0);
    for (int i = 0; i < x.tiles; i++) {
        int j0, count;
        x.tile_at(i, j0, count);
        __syncthreads();
        stage<DP>(kt, kf);
        stage<DP>(vt, vf);
        __syncthreads();
        if (i + 1 < x.tiles) fetch_tile(i + 1);
        TileView own(x.view, i >= x.sink_tiles, x.all.sink_end);
        if (i < x.sink_tiles) own.first = own.span, own.st = own.from;
#pragma unroll
        for (int y = 0; y < 2; y++) {
            f32x4 s = scores<DP>(kt, y, x.lane, q);
            const f32x4 dw = scores<DP>(vt, y, x.lane, d);
#pragma unroll
            for (int e = 0; e < 4; e++)
                s[e] = own.sees_mixed(j0 + 16 * y + 4 * x.g + e) ? __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], c, -m)) * by * (dw[e] - delta) : 0.f;
            add_rows<DP>(kt, y, x.lane, s, dq);
        }
    }
    if (x.row < p.rows) store_row<DP>(static_cast<float*>(const_cast<void*>(p.dq.p)) + x.b * p.dq.b + x.t * p.dq.t + x.head * p.dq.h, p.D, x.g, dq, p.scale);
}

template <int DP>
__global__ __launch_bounds__(256, 1) void window_dkv_f32_kernel(const WindowParams p) {
    __shared__ __attribute__((aligned(16))) float qt[TILE * Tile<DP>::LD], dt[TILE * Tile<DP>::LD];
    __shared__ __attribute__((aligned(16))) float row_m[TILE], row_by[TILE], row_delta[TILE];
    __shared__ __attribute__((aligned(16))) int row_at[TILE];
    __shared__ int bounds[4][6];
    int pair, block;
    if (!work_item(p, blockIdx.x, pair, block)) return;
    const int b = pair / p.HK, hk = pair - b * p.HK;
    const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), g = lane >> 4;
    const int j = block * WINDOW_KEYS_F32 + 16 * wave + (lane & 15);
    int st = 0, en = 0, n, from = 1 << 30, upto = -1;
    if (j < p.S) {
        sequence_at(p, b, j, st, en, n);
        if (en > st) {
            from = max(j, p.S - p.T), upto = p.window == 0 || p.window >= en - j || j - st < p.sinks ? en - 1 : j + p.window - 1;
            if (upto < from) from = 1 << 30, upto = -1;
        }
    }
    WaveView w;
    w.lo = wave_min(from), w.end = wave_max(upto) + 1, w.sink = w.sink_end = w.full_lo = w.full_end = 0;
    const WaveView all = join_waves<4>(w, bounds, wave, lane);
    const int offset = p.S - p.T;
    const bool any = all.end > all.lo;
    const int r0 = any ? (all.lo - offset) * p.G : 0, r1 = any ? (all.end - offset) * p.G : 0;

    float k[DP / 4], v[DP / 4];
    load_row<DP>(static_cast<const float*>(p.k.p) + b * p.k.b + min(j, p.S - 1) * p.k.t + hk * p.k.h, p.D, g, j < p.S, k);
    load_row<DP>(static_cast<const float*>(p.v.p) + b * p.v.b + min(j, p.S - 1) * p.v.t + hk * p.v.h, p.D, g, j < p.S, v);
    const float* const qb = static_cast<const float*>(p.q.p) + b * p.q.b + hk * p.G * p.q.h;
    const float* const db = static_cast<const float*>(p.dout.p) + b * p.dout.b + hk * p.G * p.dout.h;
    const float c = p.negative ? -p.c : p.c;
    Fetched<DP> qf, df;
    auto fetch_tile = [&](int first) {
        const int count = min(TILE, r1 - first);
        fetch<DP>(qb, [&](int row) { const int r = first + row, t = r / p.G; return t * p.q.t + (r - t * p.G) * p.q.h; }, count, p.D, qf);
        fetch<DP>(db, [&](int row) { const int r = first + row, t = r / p.G; return t * p.dout.t + (r - t * p.G) * p.dout.h; }, count, p.D, df);
    };
    f32x4 dk[DP / 16] = {}, dv[DP / 16] = {};
    if (r0 < r1) fetch_tile(r0);
    for (int first = r0; first < r1; first += TILE) {
        __syncthreads();
        stage<DP>(qt, qf);
        stage<DP>(dt, df);
        if (threadIdx.x < TILE) {
            const int r = first + (int)threadIdx.x, t = min(r, r1 - 1) / p.G;
            const int64_t scalar = ((int64_t)b * p.T + t) * p.H + hk * p.G + (min(r, r1 - 1) - t * p.G);
            row_m[threadIdx.x] = p.lse[2 * scalar], row_by[threadIdx.x] = p.lse[2 * scalar + 1], row_delta[threadIdx.x] = p.delta[scalar];
            row_at[threadIdx.x] = r < r1 ? t + offset : -1;
        }
        __syncthreads();
        if (first + TILE < r1) fetch_tile(first + TILE);
#pragma unroll
        for (int y = 0; y < 2; y++) {
            f32x4 s = scores<DP>(qt, y, lane, k), dw = scores<DP>(dt, y, lane, v);
            const int at = 16 * y + 4 * g;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const bool seen = row_at[at + e] >= from && row_at[at + e] <= upto;
                const float weight = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], c, -row_m[at + e])) * row_by[at + e];
                dw[e] = seen ? weight * (dw[e] - row_delta[at + e]) : 0.f;
                s[e] = seen ? weight : 0.f;
            }
            add_rows<DP>(dt, y, lane, s, dv);
            add_rows<DP>(qt, y, lane, dw, dk);
        }
    }
    if (j >= p.S) return;
    store_row<DP>(static_cast<float*>(const_cast<void*>(p.dk.p)) + b * p.dk.b + j * p.dk.t + hk * p.dk.h, p.D, g, dk, p.scale);
    store_row<DP>(static_cast<float*>(const_cast<void*>(p.dv.p)) + b * p.dv.b + j * p.dv.t + hk * p.dv.h, p.D, g, dv, 1.f);
}

dim3 grid_of(const WindowParams& p) { return dim3((unsigned)(((int64_t)p.B * p.HK * p.blocks + 7) / 8 * 8), p.splits); }

template <int DP>
int launch_bwd(const WindowParams& p, hipStream_t stream) {
    WindowParams r = p, k = p;
    r.blocks = (p.rows + WINDOW_ROWS_F32 - 1) / WINDOW_ROWS_F32, k.blocks = (p.S + WINDOW_KEYS_F32 - 1) / WINDOW_KEYS_F32;
    hipLaunchKernelGGL((window_dq_f32_kernel<DP>), grid_of(r), dim3(256), 0, stream, r);
    if (const int e = (int)hipGetLastError(); e != 0) return e;
    hipLaunchKernelGGL((window_dkv_f32_kernel<DP>), grid_of(k), dim3(256), 0, stream, k);
    return (int)hipGetLastError();
}

}  // namespace

int launch_window_fwd_f32(const WindowParams& p, hipStream_t stream) {
    if (p.D <= 64) hipLaunchKernelGGL((window_fwd_f32_kernel<64>), grid_of(p), dim3(256), 0, stream, p);
    else if (p.D <= 128) hipLaunchKernelGGL((window_fwd_f32_kernel<128>), grid_of(p), dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((window_fwd_f32_kernel<256>), grid_of(p), dim3(256), 0, stream, p);
    if (const int e = (int)hipGetLastError(); e != 0) return e;
    return p.splits > 1 ? launch_window_combine(p, GDN_F32, stream) : GDN_OK;
}

int launch_window_bwd_f32(const WindowParams& p, hipStream_t stream) {
    if (p.D <= 64) return launch_bwd<64>(p, stream);
    if (p.D <= 128) return launch_bwd<128>(p, stream);
    return launch_bwd<256>(p, stream);
}

}  // namespace gdn
