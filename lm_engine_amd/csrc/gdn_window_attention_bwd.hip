// Softmax attention over a window, backward, bf16 (gdn_window_attention.h).  With w = 2^(c q.k - lse), per row and key:
//     delta = sum o do,   ds = w (do . v - delta),   dq = scale sum_j ds k_j,   dk_j = scale sum_rows ds q,   dv_j = sum_rows w do
// Two passes over the scores, each with its own sums in registers and nothing added up in memory, so that results do not depend on an order:
// window_dq_kernel goes over the keys of 128 rows, as the forward does, window_dkv_kernel over the rows of 128 keys (of all heads that share
// them).  Scores are formed the way round that makes them operands as they lie: with a lane a row (S^T = K Q^T) for dq^T += K^T ds^T,
// with a lane a key (S = Q K^T) for dv^T += do^T w and dk^T += q^T ds.
// A sequence's first keys are seen by all of its rows: those beyond the window are shared out over many workgroups (window_first_keys, the
// same walk), whose parts the keys' own workgroup adds to its sums.
#include <algorithm>

#include "gdn_launch.h"
#include "gdn_window_attention.h"

namespace gdn {

namespace {

template <int DP>
__global__ __launch_bounds__(256, DP <= 128 ? 2 : 1) void window_dq_kernel(const WindowParams p) {
    constexpr int KS = DP / 16, DT = DP / 32;
    using Loads = TileLoads<DP>;
    __shared__ __attribute__((aligned(1024))) bf16_t tiles[2][2][64 * DP];
    int pair, block;
    if (!work_item(p, blockIdx.x, pair, block)) return;
    block = p.blocks - 1 - block;
    const int b = pair / p.HK, hk = pair - b * p.HK;
    const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), half = lane >> 5;
    const int row = block * WINDOW_ROWS + 32 * wave + (lane & 31), r = min(row, p.rows - 1);
    const int t = p.G == 1 ? r : r / p.G, head = hk * p.G + (r - t * p.G);
    const int64_t scalar = ((int64_t)b * p.T + t) * p.H + head;

    bf16x8 q[KS], d[KS];
    load_row_fragments<DP>(static_cast<const bf16_t*>(p.q.p) + b * p.q.b + t * p.q.t + head * p.q.h, p.D, half, true, q);
    load_row_fragments<DP>(static_cast<const bf16_t*>(p.dout.p) + b * p.dout.b + t * p.dout.t + head * p.dout.h, p.D, half, true, d);
    float delta = 0.f;
    {
        bf16x8 o[KS];
        load_row_fragments<DP>(static_cast<const bf16_t*>(p.o.p) + b * p.o.b + t * p.o.t + head * p.o.h, p.D, half, true, o);
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int e = 0; e < 8; e++) delta += (float)o[s][e] * (float)d[s][e];
        delta += other_half(delta);
        if (half == 0 && row < p.rows) p.delta[scalar] = delta;
    }
    const float lse = p.lse[scalar], c = p.negative ? -p.c : p.c;

    const RowView view = row_view(p, b, r);
    const WaveView w = wave_view(view);
    __shared__ int bounds[4][6];
    const WaveView all = join_waves<4>(w, bounds, wave, lane);
    const int lo = all.lo, end = all.end, sink = all.sink, sink_end = min(all.sink_end, lo);
    const int sink_tiles = sink_end > sink ? (sink_end - sink + 63) / 64 : 0, near_tiles = end > lo ? (end - lo + 63) / 64 : 0;
    const int tile_count = sink_tiles + near_tiles;

    const char* const kb = reinterpret_cast<const char*>(static_cast<const bf16_t*>(p.k.p) + b * p.k.b + hk * p.k.h);
    const char* const vb = reinterpret_cast<const char*>(static_cast<const bf16_t*>(p.v.p) + b * p.v.b + hk * p.v.h);
    const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)&tiles[0][0][0];
    auto tile_at = [&](int i, int& j0, int& count) {
        const bool s = i < sink_tiles;
        j0 = s ? sink + 64 * i : lo + 64 * (i - sink_tiles);
        count = min((s ? sink_end : end) - j0, 64);
    };
    auto load_tile = [&](int i) {
        int j0, count;
        tile_at(i, j0, count);
        const char *const k0 = kb + (int64_t)j0 * p.k.t * 2, *const v0 = vb + (int64_t)j0 * p.v.t * 2;
        const uint32_t to = lds + (i & 1) * 2 * 64 * DP * 2;
#pragma unroll
        for (int x = 0; x < Loads::ITERS; x++) {
            const int kr = Loads::row(wave, lane, x), col = Loads::column(wave, lane, x);
            const bool there = kr < count && col < p.D;
            Loads::load(k0, there ? (uint32_t)(kr * (int)p.k.t + col) * 2 : PAST, to, wave, x);
            Loads::load(v0, there ? (uint32_t)(kr * (int)p.v.t + col) * 2 : PAST, to + 64 * DP * 2, wave, x);
        }
    };

    const TileReader<DP> reader(lane);
    f32x16 dq[DT] = {};
    if (tile_count > 0) load_tile(0);
    for (int i = 0; i < tile_count; i++) {
        loads_done();
        __syncthreads();
        if (i + 1 < tile_count) load_tile(i + 1);
        int j0, count;
        tile_at(i, j0, count);
        const bf16_t *const kt = tiles[i & 1][0], *const vt = tiles[i & 1][1];
        const bool near = i >= sink_tiles, full = near && j0 >= w.full_lo && j0 + 64 <= w.full_end;
        if (!w.meets(j0, count)) continue;
        const TileView own(view, near, sink_end);
#pragma unroll
        for (int x = 0; x < 2; x++) {
            f32x16 s = {}, dw = {};
#pragma unroll
            for (int y = 0; y < KS; y++) s = mma(reader.across(kt, 32 * x, y), q[y], s);
#pragma unroll
            for (int y = 0; y < KS; y++) dw = mma(reader.across(vt, 32 * x, y), d[y], dw);
#pragma unroll
            for (int e = 0; e < 16; e++) s[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], c, -lse)) * (dw[e] - delta);
            if (!full) {
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    const int j = j0 + 32 * x + acc_row(e, half);
                    if (!own.sees(j)) s[e] = 0.f;
                }
            }
#pragma unroll
            for (int y = 0; y < 2; y++) {
                const bf16x8 ds = pack8(s, y);
#pragma unroll
                for (int z = 0; z < DT; z++) dq[z] = mma(reader.down(kt, 2 * x + y, z), ds, dq[z]);
            }
        }
    }
    if (row >= p.rows) return;
    store_transposed<DP>(static_cast<bf16_t*>(const_cast<void*>(p.dq.p)) + b * p.dq.b + t * p.dq.t + head * p.dq.h, p.D, half, dq, p.scale);
}

// Gradients of 128 keys, 32 to a wave.  FIRST: of the keys of a sequence that all of its rows see, from one part of the rows that do
// not have them in their window; blockIdx.x goes over (sequence, head of k and v, block of 128 such keys, part).
template <int DP, bool FIRST>
__global__ __launch_bounds__(256, DP <= 64 ? 2 : 1) void window_dkv_kernel(const WindowParams p) {
    constexpr int KS = DP / 16, DT = DP / 32;
    using Loads = TileLoads<DP>;
    __shared__ __attribute__((aligned(1024))) bf16_t tiles[2][2][64 * DP];
    __shared__ __attribute__((aligned(16))) float row_lse[2][64], row_delta[2][64];
    __shared__ __attribute__((aligned(16))) int row_at[2][64];
    const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), half = lane >> 5;
    int b, hk, n = 0, piece = 0, key0, keys;  // key0: of the workgroup
    int64_t slot = 0;
    if constexpr (FIRST) {
        const int key_blocks = p.first_keys / WINDOW_KEYS;
        int x = blockIdx.x;
        piece = x % p.pieces, x /= p.pieces;
        const int kblock = x % key_blocks;
        x /= key_blocks;
        hk = x % p.HK, n = x / p.HK;
        b = p.cu != nullptr && !p.padded ? 0 : n;
        int st, len;
        if (p.cu == nullptr) st = 0, len = p.S;
        else if (p.padded) len = min(max(p.cu[n + 1] - p.cu[n], 0), p.S), st = p.S - len;
        else packed_bounds(p.cu, n, p.S, st, len);
        key0 = st + kblock * WINDOW_KEYS, keys = min(WINDOW_KEYS, min(p.sinks, len) - kblock * WINDOW_KEYS);
        slot = (((int64_t)n * p.HK + hk) * p.pieces + piece) * p.first_keys + kblock * WINDOW_KEYS;
    } else {
        int pair, block;
        if (!work_item(p, blockIdx.x, pair, block)) return;
        b = pair / p.HK, hk = pair - b * p.HK;
        key0 = block * WINDOW_KEYS, keys = min(WINDOW_KEYS, p.S - key0);
    }
    // this lane's key, and the positions that see it: [from, upto]
    const int own = 32 * wave + (lane & 31), j = key0 + own;
    int st = 0, en = 0, sequence = 0, from = 1 << 30, upto = -1;
    if (own < keys) {
        sequence_at(p, b, j, st, en, sequence);
        if (en > st) {
            const bool first = j - st < p.sinks;
            if constexpr (FIRST) from = p.window < en - j ? j + p.window : 1 << 30, upto = from < en ? en - 1 : -1;
            else from = j, upto = p.window == 0 || p.window >= en - j || (first && p.pieces == 0) ? en - 1 : j + p.window - 1;
            from = max(from, p.S - p.T);  // (positions in front of the queries)
            if (upto < from) from = 1 << 30, upto = -1;
        }
    }
    WaveView w;
    w.lo = wave_min(from), w.end = wave_max(upto) + 1, w.full_lo = wave_max(from), w.full_end = upto < 0 ? 0 : upto + 1;
    w.full_end = wave_min(w.full_end), w.sink = w.sink_end = 0;
    __shared__ int bounds[4][6];
    const WaveView all = join_waves<4>(w, bounds, wave, lane);
    const int offset = p.S - p.T;
    int a0 = all.lo, a1 = all.end;  // positions whose rows are walked over
    if (a1 <= a0) a0 = a1 = offset;
    if constexpr (FIRST) {
        const int each = (int)(((int64_t)a1 - a0 + p.pieces - 1) / p.pieces);
        const int64_t begin = a0 + (int64_t)piece * each;
        a1 = (int)min((int64_t)a1, begin + each), a0 = (int)min((int64_t)a1, begin);
    }
    const int r0 = (a0 - offset) * p.G, r1 = (a1 - offset) * p.G;
    const int tile_count = (r1 - r0 + 63) / 64;

    bf16x8 k[KS], v[KS];
    {
        const bool there = own < keys;
        const int at = there ? j : key0 < p.S ? key0 : 0;
        load_row_fragments<DP>(static_cast<const bf16_t*>(p.k.p) + b * p.k.b + at * p.k.t + hk * p.k.h, p.D, half, there, k);
        load_row_fragments<DP>(static_cast<const bf16_t*>(p.v.p) + b * p.v.b + at * p.v.t + hk * p.v.h, p.D, half, there, v);
    }

    const char* const qb = reinterpret_cast<const char*>(static_cast<const bf16_t*>(p.q.p) + b * p.q.b + hk * p.G * p.q.h);
    const char* const db = reinterpret_cast<const char*>(static_cast<const bf16_t*>(p.dout.p) + b * p.dout.b + hk * p.G * p.dout.h);
    const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)&tiles[0][0][0];
    float lse_next = 0.f, delta_next = 0.f;
    int at_next = 0;
    auto load_tile = [&](int i) {
        const int first = r0 + 64 * i, count = min(64, r1 - first);
        const int t0 = p.G == 1 ? first : first / p.G, g0 = first - t0 * p.G;
        const char *const q0 = qb + (int64_t)t0 * p.q.t * 2, *const d0 = db + (int64_t)t0 * p.dout.t * 2;
        const uint32_t to = lds + (i & 1) * 2 * 64 * DP * 2;
#pragma unroll
        for (int x = 0; x < Loads::ITERS; x++) {
            const int rr = Loads::row(wave, lane, x), col = Loads::column(wave, lane, x);
            int tt, g;
            split_rows(p, g0 + rr, tt, g);
            const bool there = rr < count && col < p.D;
            Loads::load(q0, there ? (uint32_t)(tt * (int)p.q.t + g * (int)p.q.h + col) * 2 : PAST, to, wave, x);
            Loads::load(d0, there ? (uint32_t)(tt * (int)p.dout.t + g * (int)p.dout.h + col) * 2 : PAST, to + 64 * DP * 2, wave, x);
        }
        if (wave == 0) {
            int tt, g;
            split_rows(p, g0 + lane, tt, g);
            const bool there = lane < count;
            const int64_t scalar = ((int64_t)b * p.T + t0 + (there ? tt : 0)) * p.H + hk * p.G + (there ? g : 0);
            lse_next = there ? p.lse[scalar] : __builtin_inff(), delta_next = there ? p.delta[scalar] : 0.f;
            at_next = there ? t0 + tt + offset : -1;
        }
    };
    auto stage_scalars = [&](int i) {
        if (wave == 0) row_lse[i & 1][lane] = lse_next, row_delta[i & 1][lane] = delta_next, row_at[i & 1][lane] = at_next;
    };

    const TileReader<DP> reader(lane);
    const float c = p.negative ? -p.c : p.c;
    f32x16 dk[DT] = {}, dv[DT] = {};
    if (tile_count > 0) load_tile(0);
    for (int i = 0; i < tile_count; i++) {
        loads_done();
        stage_scalars(i);
        __syncthreads();
        if (i + 1 < tile_count) load_tile(i + 1);
        const int first = r0 + 64 * i, count = min(64, r1 - first);
        const int p0 = (p.G == 1 ? first : first / p.G) + offset, p1 = (p.G == 1 ? first + count - 1 : (first + count - 1) / p.G) + offset;  // positions
        if (!(p0 < w.end && p1 >= w.lo)) continue;
        const bool full = p0 >= w.full_lo && p1 < w.full_end && count == 64;
        const bf16_t *const qt = tiles[i & 1][0], *const dt = tiles[i & 1][1];
#pragma unroll
        for (int x = 0; x < 2; x++) {
            f32x16 s = {}, dw = {};
#pragma unroll
            for (int y = 0; y < KS; y++) s = mma(reader.across(qt, 32 * x, y), k[y], s);
#pragma unroll
            for (int y = 0; y < KS; y++) dw = mma(reader.across(dt, 32 * x, y), v[y], dw);
#pragma unroll
            for (int y = 0; y < 4; y++) {
                const f32x4 lse = *reinterpret_cast<const f32x4*>(&row_lse[i & 1][32 * x + 8 * y + 4 * half]);
                const f32x4 delta = *reinterpret_cast<const f32x4*>(&row_delta[i & 1][32 * x + 8 * y + 4 * half]);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float weight = __builtin_amdgcn_exp2f(__builtin_fmaf(s[4 * y + e], c, -lse[e]));
                    dw[4 * y + e] = weight * (dw[4 * y + e] - delta[e]);
                    s[4 * y + e] = weight;
                }
                if (!full) {
                    const i32x4 at = *reinterpret_cast<const i32x4*>(&row_at[i & 1][32 * x + 8 * y + 4 * half]);
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (at[e] < from || at[e] > upto) s[4 * y + e] = dw[4 * y + e] = 0.f;
                }
            }
#pragma unroll
            for (int y = 0; y < 2; y++) {
                const bf16x8 weights = pack8(s, y), ds = pack8(dw, y);
#pragma unroll
                for (int z = 0; z < DT; z++) dv[z] = mma(reader.down(dt, 2 * x + y, z), weights, dv[z]);
#pragma unroll
                for (int z = 0; z < DT; z++) dk[z] = mma(reader.down(qt, 2 * x + y, z), ds, dk[z]);
            }
        }
    }
    if constexpr (FIRST) {
        if (own >= keys) return;
        float* const to = p.part_dk + (slot + own) * 2 * p.D;
#pragma unroll
        for (int z = 0; z < DT; z++)
#pragma unroll
            for (int y = 0; y < 4; y++) {
                const int col = 32 * z + 8 * y + 4 * half;
                if (col >= p.D) continue;
                *reinterpret_cast<f32x4*>(to + col) = f32x4{dk[z][4 * y], dk[z][4 * y + 1], dk[z][4 * y + 2], dk[z][4 * y + 3]};
                *reinterpret_cast<f32x4*>(to + p.D + col) = f32x4{dv[z][4 * y], dv[z][4 * y + 1], dv[z][4 * y + 2], dv[z][4 * y + 3]};
            }
    } else {
        if (own >= keys) return;
        if (p.pieces > 0 && en > st && j - st < p.sinks) {
            const float* const parts = p.part_dk + ((((int64_t)sequence * p.HK + hk) * p.pieces) * p.first_keys + (j - st)) * 2 * p.D;
            for (int x = 0; x < p.pieces; x++) {
                const float* const part = parts + (int64_t)x * p.first_keys * 2 * p.D;
#pragma unroll
                for (int z = 0; z < DT; z++)
#pragma unroll
                    for (int y = 0; y < 4; y++) {
                        const int col = 32 * z + 8 * y + 4 * half;
                        if (col >= p.D) continue;
                        const f32x4 a = *reinterpret_cast<const f32x4*>(part + col), d = *reinterpret_cast<const f32x4*>(part + p.D + col);
#pragma unroll
                        for (int e = 0; e < 4; e++) dk[z][4 * y + e] += a[e], dv[z][4 * y + e] += d[e];
                    }
            }
        }
        store_transposed<DP>(static_cast<bf16_t*>(const_cast<void*>(p.dk.p)) + b * p.dk.b + j * p.dk.t + hk * p.dk.h, p.D, half, dk, p.scale);
        store_transposed<DP>(static_cast<bf16_t*>(const_cast<void*>(p.dv.p)) + b * p.dv.b + j * p.dv.t + hk * p.dv.h, p.D, half, dv, 1.f);
    }
}

template <int DP>
int launch_bwd(const WindowParams& p, hipStream_t stream) {
    WindowParams r = p, k = p;
    r.blocks = (p.rows + WINDOW_ROWS - 1) / WINDOW_ROWS, k.blocks = (p.S + WINDOW_KEYS - 1) / WINDOW_KEYS;
    const auto grid = [&](const WindowParams& x) { return dim3((unsigned)(((int64_t)p.B * p.HK * x.blocks + 7) / 8 * 8)); };
    hipLaunchKernelGGL((window_dq_kernel<DP>), grid(r), dim3(256), 0, stream, r);
    if (const int e = (int)hipGetLastError(); e != 0) return e;
    if (p.pieces > 0) {
        hipLaunchKernelGGL((window_dkv_kernel<DP, true>), dim3((unsigned)((int64_t)p.N * p.HK * (p.first_keys / WINDOW_KEYS) * p.pieces)), dim3(256), 0, stream, k);
        if (const int e = (int)hipGetLastError(); e != 0) return e;
    }
    hipLaunchKernelGGL((window_dkv_kernel<DP, false>), grid(k), dim3(256), 0, stream, k);
    return (int)hipGetLastError();
}

}  // namespace

int launch_window_bwd(const WindowParams& p, hipStream_t stream) {
    if (p.D <= 64) return launch_bwd<64>(p, stream);
    if (p.D <= 128) return launch_bwd<128>(p, stream);
    return launch_bwd<256>(p, stream);
}

}  // namespace gdn
