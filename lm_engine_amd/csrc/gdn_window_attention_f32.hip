// Softmax attention over a window in fp32, forward and backward (gdn_window_attention.h): the walks of the bf16 kernels on
// v_mfma_f32_16x16x4_f32, 16 rows (or keys) to a wave and tiles of 16 keys (or rows).  An accumulator's register r of lane (n, g) is row
// 4 g + r of column n, and the fp32 product takes its operand one row of four lanes at a time: register r goes on as it is, against rows
// 4 g + r of the other operand.
// Four waves share 16 rows (or keys): each takes every fourth tile, and they add up in LDS at the end.  Small calls are what this type is used for,
// and with 64 rows to a workgroup they leave the chip empty: forward and backward at 1 x 256 tokens, 2 heads of 64, window 100 took 22 + 66 us,
// now 8 + 20; 1 x 2048, 16 heads of 128 over 4, all keys 292 + 2160 us, now 227 + 890 (54 TFLOP/s, of the 154 of a large product).  At
// 4 x 4096, 16 heads of 128, window 1024, where the chip is full anyway, 64 rows on one tile in LDS were faster forward, 1340 us against 1565, and
// slower backward, 9700 against 5200 with 4 first keys that every row sees.
// Operands come straight from memory, without barriers, 16 bytes to a lane: a sum over columns may take them in any order (step
// 4 u + e: column 16 u + 4 g + e in lane group g of both operands), and so may the columns of a result (accumulator e of lane n: column
// 4 n + e of each 64).  The forward needs each tile in one form; a tile that is needed in both is loaded once and turned in LDS by its wave
// (loaded twice: backward at the large size 5.8 ms instead of 5.1).  The next tile is asked for as soon as this one's registers are free.
// The weights are 2^(c s - m) / l with the m and l of the forward, kept as two numbers: as one, log2 of the sum, their rounding would come back
// relative in every weight (4e-7 at 16).
#include <algorithm>

#include "gdn_launch.h"
#include "gdn_window_attention.h"

namespace gdn {

namespace {

__device__ __forceinline__ f32x4 mma4(float a, float b, const f32x4& c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

constexpr int TILE = 16;

// columns 16 u + 4 g .. + 3 of a row
template <int DP>
struct Across {
    f32x4 v[DP / 16];
    __device__ __forceinline__ void load(const float* row, int D, int g) {
#pragma unroll
        for (int u = 0; u < DP / 16; u++) {
            const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
            v[u] = 16 * u + 4 * g < D ? *reinterpret_cast<const f32x4*>(row + 16 * u + 4 * g) : zero;
        }
    }
};
// columns 64 c + 4 n .. + 3 of rows 4 g + r
template <int DP>
struct Down {
    f32x4 v[4][DP / 64];
    template <typename RowAt>
    __device__ __forceinline__ void load(const RowAt& row_at, int D, int n, int g) {
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const float* const row = row_at(4 * g + r);
#pragma unroll
            for (int c = 0; c < DP / 64; c++) {
                const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
                v[r][c] = 64 * c + 4 * n < D ? *reinterpret_cast<const f32x4*>(row + 64 * c + 4 * n) : zero;
            }
        }
    }
};
// row 4 g + r of x (a tile), column n of y
template <int DP>
__device__ __forceinline__ f32x4 scores(const Across<DP>& x, const Across<DP>& y) {
    f32x4 a = {0.f, 0.f, 0.f, 0.f}, b = a;
#pragma unroll
    for (int u = 0; u < DP / 16; u++)
#pragma unroll
        for (int e = 0; e < 4; e += 2) a = mma4(x.v[u][e], y.v[u][e], a), b = mma4(x.v[u][e + 1], y.v[u][e + 1], b);
    return a + b;
}
// Sums over a tile's rows, weighted: acc[c][e] of lane (n, g), register r: column 64 c + 16 g + 4 r + e of row n.
template <int DP>
struct Sums {
    f32x4 acc[DP / 64][4];
    __device__ __forceinline__ Sums() {
#pragma unroll
        for (int c = 0; c < DP / 64; c++)
#pragma unroll
            for (int e = 0; e < 4; e++) acc[c][e] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    __device__ __forceinline__ void add(const Down<DP>& x, const f32x4& w) {
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int c = 0; c < DP / 64; c++)
#pragma unroll
                for (int e = 0; e < 4; e++) acc[c][e] = mma4(x.v[r][c][e], w[r], acc[c][e]);
    }
    __device__ __forceinline__ void scale(float by) {
#pragma unroll
        for (int c = 0; c < DP / 64; c++)
#pragma unroll
            for (int e = 0; e < 4; e++) acc[c][e] *= by;
    }
    __device__ __forceinline__ void store(float* row, int D, int g, float by) const {
#pragma unroll
        for (int c = 0; c < DP / 64; c++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int at = 64 * c + 16 * g + 4 * r;
                if (at < D) *reinterpret_cast<f32x4*>(row + at) = f32x4{acc[c][0][r] * by, acc[c][1][r] * by, acc[c][2][r] * by, acc[c][3][r] * by};
            }
    }
};
// 16 rows of each of four waves in LDS: a tile that a wave turns (stored as it came, read in the other form), or the waves' sums over the same rows,
// added in the waves' order.
template <int DP>
struct Rows {
    static constexpr int LD = DP + 4;
    float rows[4][16][LD];
    __device__ __forceinline__ void put(const Across<DP>& x, int wave, int n, int g) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int u = 0; u < DP / 16; u++) *reinterpret_cast<f32x4*>(&rows[wave][n][16 * u + 4 * g]) = x.v[u];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    __device__ __forceinline__ void get(Down<DP>& x, int wave, int n, int g) const {
        x.load([&](int y) { return rows[wave][y]; }, DP, n, g);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    __device__ __forceinline__ void put(const Sums<DP>& s, int wave, int n, int g, float by) { s.store(rows[wave][n], DP, g, by); }
    template <typename Store>
    __device__ __forceinline__ void take(const Store& store, int D) const {
#pragma unroll
        for (int i = 0; i < DP / 64; i++) {
            const int at = threadIdx.x + 256 * i, row = at / (DP / 4), col = 4 * (at % (DP / 4));
            f32x4 sum = *reinterpret_cast<const f32x4*>(&rows[0][row][col]);
#pragma unroll
            for (int w = 1; w < 4; w++) sum += *reinterpret_cast<const f32x4*>(&rows[w][row][col]);
            if (col < D) store(row, col, sum);
        }
    }
};

__device__ __forceinline__ float over_groups(float x, bool largest) {
#pragma unroll
    for (int off = 16; off <= 32; off <<= 1) {
        const float y = __shfl_xor(x, off, WAVE);
        x = largest ? fmaxf(x, y) : x + y;
    }
    return x;
}

// What the two walks over keys have in common: where a wave's rows and tiles are.
struct KeyWalk {
    int b, hk, lane, wave, n, g, r0, row, r, t, head;
    RowView view;
    WaveView all;
    int sink_tiles, tiles;
    __device__ __forceinline__ void begin(const WindowParams& p) {
        int pair, block;
        work_item(p, blockIdx.x, pair, block);
        block = p.blocks - 1 - block;
        b = pair / p.HK, hk = pair - b * p.HK;
        lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), n = lane & 15, g = lane >> 4;
        r0 = block * WINDOW_ROWS_F32, row = r0 + n, r = min(row, p.rows - 1);
        t = r / p.G, head = hk * p.G + (r - t * p.G);
        view = row_view(p, b, r);
        all = wave_view(view);
        all.sink_end = min(all.sink_end, all.lo);
        sink_tiles = all.sink_end > all.sink ? (all.sink_end - all.sink + TILE - 1) / TILE : 0;
        tiles = sink_tiles + (all.end > all.lo ? (all.end - all.lo + TILE - 1) / TILE : 0);
    }
    __device__ __forceinline__ void tile_at(int i, int& j0, int& count) const {
        const bool s = i < sink_tiles;
        j0 = s ? all.sink + TILE * i : all.lo + TILE * (i - sink_tiles);
        count = min((s ? all.sink_end : all.end) - j0, TILE);
    }
    __device__ __forceinline__ TileView seen(int i) const {
        TileView own(view, i >= sink_tiles, all.sink_end);
        if (i < sink_tiles) own.first = own.span, own.st = own.from;
        return own;
    }
    __device__ __forceinline__ bool seen_by_all(int i, int j0) const { return i >= sink_tiles && j0 >= all.full_lo && j0 + TILE <= all.full_end; }
    // keys past a tile's last one are that one again, without weight
    template <int DP>
    __device__ __forceinline__ void across(const WindowRows& x, int i, int D, Across<DP>& f) const {
        int j0, count;
        tile_at(i, j0, count);
        f.load(static_cast<const float*>(x.p) + b * x.b + hk * x.h + (j0 + min(n, count - 1)) * x.t, D, g);
    }
    template <int DP>
    __device__ __forceinline__ void down(const WindowRows& x, int i, int D, Down<DP>& f) const {
        int j0, count;
        tile_at(i, j0, count);
        const float* const base = static_cast<const float*>(x.p) + b * x.b + hk * x.h + j0 * x.t;
        f.load([&](int y) { return base + min(y, count - 1) * x.t; }, D, n, g);
    }
    __device__ __forceinline__ float* place(const WindowRows& x, int of_row, const WindowParams& p) const {
        const int tt = of_row / p.G, hh = hk * p.G + (of_row - tt * p.G);
        return static_cast<float*>(const_cast<void*>(x.p)) + b * x.b + tt * x.t + hh * x.h;
    }
};

template <int DP>
__global__ __launch_bounds__(256, DP <= 128 ? 2 : 1) void window_fwd_f32_kernel(const WindowParams p) {
    KeyWalk x;
    x.begin(p);
    Across<DP> q;
    q.load(x.place(p.q, x.r, p), p.D, x.g);
    if (p.negative)
#pragma unroll
        for (int u = 0; u < DP / 16; u++) q.v[u] = -q.v[u];
    int first = 0, last = x.tiles;
    if (p.splits > 1) {
        const int each = (last + p.splits - 1) / p.splits;
        first = min((int)blockIdx.y * each, last), last = min(first + each, last);
    }
    Across<DP> k;
    Down<DP> v;
    Sums<DP> o;
    float m = LOWEST, l = 0.f;
    bool taken_out = false;
    int i = first + x.wave;
    if (i < last) x.across(p.k, i, p.D, k), x.down(p.v, i, p.D, v);
    for (; i < last; i += 4) {
        int j0, count;
        x.tile_at(i, j0, count);
        f32x4 s = scores<DP>(k, q);
        if (i + 4 < last) x.across(p.k, i + 4, p.D, k);
        float top = -__builtin_inff();
        const TileView own = x.seen(i);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if (!own.sees_mixed(j0 + 4 * x.g + e)) s[e] = -__builtin_inff();
            else top = fmaxf(top, s[e] * p.c);
        }
        top = over_groups(top, true);
        const float next = fmaxf(m, top), alpha = __builtin_amdgcn_exp2f(m - next);
        m = next;
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            s[e] = s[e] == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], p.c, -m));
            sum += s[e];
        }
        l = l * alpha + sum;
        o.scale(alpha);
        if (!x.seen_by_all(i, j0)) {  // (as in the bf16 kernel: 0 times what is not finite)
            bool found = false;
#pragma unroll
            for (int y = 0; y < 4; y++)
#pragma unroll
                for (int c = 0; c < DP / 64; c++)
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (!(fabsf(v.v[y][c][e]) < __builtin_inff())) v.v[y][c][e] = 0.f, found = true;
            taken_out |= __ballot(found) != 0;
        }
        o.add(v, s);
        if (i + 4 < last) x.down(p.v, i + 4, p.D, v);
    }
    l = over_groups(l, false);
    const int64_t part = (((int64_t)blockIdx.y * p.B + x.b) * p.HK + x.hk) * p.rows + x.r0;
    __shared__ __attribute__((aligned(16))) Rows<DP> rows;
    __shared__ float tops[4][16], sums[4][16];
    if (x.g == 0) tops[x.wave][x.n] = m;
    __syncthreads();
    m = fmaxf(fmaxf(tops[0][x.n], tops[1][x.n]), fmaxf(tops[2][x.n], tops[3][x.n]));
    const float by = __builtin_amdgcn_exp2f(tops[x.wave][x.n] - m);
    if (x.g == 0) sums[x.wave][x.n] = l * by;
    rows.put(o, x.wave, x.n, x.g, by);
    __syncthreads();
    auto total = [&](int row) { return sums[0][row] + sums[1][row] + sums[2][row] + sums[3][row]; };
    auto inverse = [](float sum) { return sum == 0.f ? 0.f : 1.f / sum; };
    rows.take(
        [&](int row, int col, const f32x4& sum) {
            if (x.r0 + row >= p.rows) return;
            if (p.splits > 1) *reinterpret_cast<f32x4*>(p.part_o + (part + row) * p.D + col) = sum;
            else *reinterpret_cast<f32x4*>(x.place(p.o, x.r0 + row, p) + col) = sum * inverse(total(row));
        },
        p.D);
    if (x.row < p.rows && threadIdx.x < 16) {
        l = total(x.n);
        const int64_t scalar = ((int64_t)x.b * p.T + x.t) * p.H + x.head;
        if (p.splits > 1) p.part_m[2 * (part + x.n)] = m, p.part_m[2 * (part + x.n) + 1] = l;
        else if (p.lse != nullptr) p.lse[2 * scalar] = l == 0.f ? 0.f : m, p.lse[2 * scalar + 1] = inverse(l);
    }
    if (__syncthreads_or(taken_out))
        add_taken_out<float>(p, x.b, x.hk, x.r0, WINDOW_ROWS_F32, x.all, first, last, x.sink_tiles, TILE, [&](int y, int& j0, int& count) { x.tile_at(y, j0, count); }, part);
}

template <int DP>
__global__ __launch_bounds__(256, DP <= 128 ? 2 : 1) void window_dq_f32_kernel(const WindowParams p) {
    __shared__ __attribute__((aligned(16))) Rows<DP> rows;
    KeyWalk x;
    x.begin(p);
    Across<DP> q, d, k, v;
    q.load(x.place(p.q, x.r, p), p.D, x.g);
    d.load(x.place(p.dout, x.r, p), p.D, x.g);
    int i = x.wave;
    if (i < x.tiles) x.across(p.k, i, p.D, k), x.across(p.v, i, p.D, v);
    const int64_t scalar = ((int64_t)x.b * p.T + x.t) * p.H + x.head;
    float delta = 0.f;
    {
        Across<DP> o;
        o.load(x.place(p.o, x.r, p), p.D, x.g);
#pragma unroll
        for (int u = 0; u < DP / 16; u++)
#pragma unroll
            for (int e = 0; e < 4; e++) delta += o.v[u][e] * d.v[u][e];
        delta = over_groups(delta, false);
        if (x.g == 0 && x.row < p.rows && x.wave == 0) p.delta[scalar] = delta;
    }
    const float m = p.lse[2 * scalar], by = p.lse[2 * scalar + 1], c = p.negative ? -p.c : p.c;
    Sums<DP> dq;
    for (; i < x.tiles; i += 4) {
        int j0, count;
        x.tile_at(i, j0, count);
        rows.put(k, x.wave, x.n, x.g);
        f32x4 s = scores<DP>(k, q);
        const f32x4 dw = scores<DP>(v, d);
        if (i + 4 < x.tiles) x.across(p.k, i + 4, p.D, k), x.across(p.v, i + 4, p.D, v);
        Down<DP> kd;
        rows.get(kd, x.wave, x.n, x.g);
        const TileView own = x.seen(i);
#pragma unroll
        for (int e = 0; e < 4; e++)
            s[e] = own.sees_mixed(j0 + 4 * x.g + e) ? __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], c, -m)) * by * (dw[e] - delta) : 0.f;
        dq.add(kd, s);
    }
    rows.put(dq, x.wave, x.n, x.g, p.scale);
    __syncthreads();
    rows.take(
        [&](int row, int col, const f32x4& sum) {
            if (x.r0 + row < p.rows) *reinterpret_cast<f32x4*>(x.place(p.dq, x.r0 + row, p) + col) = sum;
        },
        p.D);
}

template <int DP>
__global__ __launch_bounds__(256, DP <= 128 ? 2 : 1) void window_dkv_f32_kernel(const WindowParams p) {
    __shared__ __attribute__((aligned(16))) Rows<DP> q_rows, d_rows;
    int pair, block;
    work_item(p, blockIdx.x, pair, block);
    const int b = pair / p.HK, hk = pair - b * p.HK;
    const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), n = lane & 15, g = lane >> 4;
    const int j0 = WINDOW_KEYS_F32 * block, j = j0 + n;
    int st = 0, en = 0, number, from = 1 << 30, upto = -1;
    if (j < p.S) {
        sequence_at(p, b, j, st, en, number);
        if (en > st) {
            from = max(j, p.S - p.T), upto = p.window == 0 || p.window >= en - j || j - st < p.sinks ? en - 1 : j + p.window - 1;
            if (upto < from) from = 1 << 30, upto = -1;
        }
    }
    const int lo = wave_min(from), end = wave_max(upto) + 1, offset = p.S - p.T;
    const int r0 = end > lo ? (lo - offset) * p.G : 0, r1 = end > lo ? (end - offset) * p.G : 0;

    Across<DP> k, v, q, d;
    k.load(static_cast<const float*>(p.k.p) + b * p.k.b + min(j, p.S - 1) * p.k.t + hk * p.k.h, p.D, g);
    v.load(static_cast<const float*>(p.v.p) + b * p.v.b + min(j, p.S - 1) * p.v.t + hk * p.v.h, p.D, g);
    const float* const qb = static_cast<const float*>(p.q.p) + b * p.q.b + hk * p.G * p.q.h;
    const float* const db = static_cast<const float*>(p.dout.p) + b * p.dout.b + hk * p.G * p.dout.h;
    const float c = p.negative ? -p.c : p.c;
    float row_m, row_by, row_delta;
    int row_at;
    auto load = [&](int first) {
        const int r = min(first + n, r1 - 1), t = r / p.G, h = r - t * p.G;
        const int64_t scalar = ((int64_t)b * p.T + t) * p.H + hk * p.G + h;
        row_m = p.lse[2 * scalar], row_by = p.lse[2 * scalar + 1], row_delta = p.delta[scalar];
        row_at = first + n < r1 ? t + offset : -1;
        q.load(qb + t * p.q.t + h * p.q.h, p.D, g);
        d.load(db + t * p.dout.t + h * p.dout.h, p.D, g);
    };
    Sums<DP> dk, dv;
    int first = r0 + TILE * wave;
    if (first < r1) load(first);
    for (; first < r1; first += 4 * TILE) {
        q_rows.put(q, wave, n, g);
        d_rows.put(d, wave, n, g);
        f32x4 s = scores<DP>(q, k), dw = scores<DP>(d, v);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int of = 4 * g + e, at = __shfl(row_at, of, WAVE);
            const float delta = __shfl(row_delta, of, WAVE);  // (by all lanes, seen or not)
            const float weight = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], c, -__shfl(row_m, of, WAVE))) * __shfl(row_by, of, WAVE);
            const bool seen = at >= from && at <= upto;
            dw[e] = seen ? weight * (dw[e] - delta) : 0.f;
            s[e] = seen ? weight : 0.f;
        }
        if (first + 4 * TILE < r1) load(first + 4 * TILE);
        Down<DP> x;
        d_rows.get(x, wave, n, g);
        dv.add(x, s);
        q_rows.get(x, wave, n, g);
        dk.add(x, dw);
    }
    q_rows.put(dk, wave, n, g, p.scale);
    d_rows.put(dv, wave, n, g, 1.f);
    __syncthreads();
    auto store = [&](const Rows<DP>& rows, const WindowRows& x) {
        float* const base = static_cast<float*>(const_cast<void*>(x.p)) + b * x.b + hk * x.h;
        rows.take(
            [&](int row, int col, const f32x4& sum) {
                if (j0 + row < p.S) *reinterpret_cast<f32x4*>(base + (j0 + row) * x.t + col) = sum;
            },
            p.D);
    };
    store(q_rows, p.dk);
    store(d_rows, p.dv);
}

dim3 grid_of(const WindowParams& p) { return dim3((unsigned)((int64_t)p.B * p.HK * p.blocks), p.splits); }

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
