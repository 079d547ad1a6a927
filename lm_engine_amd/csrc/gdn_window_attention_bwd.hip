// Softmax attention over a window, backward, bf16 (gdn_window_attention.h).  With w = 2^(c q.k - lse), per row and key:
//     delta = sum o do,   ds = w (do . v - delta),   dq = scale sum_j ds k_j,   dk_j = scale sum_rows ds q,   dv_j = sum_rows w do
// Two passes over the scores, each with its own sums in registers and nothing added up in memory, so that results do not depend on an order:
// window_dq_kernel goes over the keys of 128 rows, as the forward does, window_dkv_kernel over the rows of 128 keys (of all heads that share
// them).  Scores are formed the way round that makes them operands as they lie: with a lane a row (S^T = K Q^T) for dq^T += K^T ds^T,
// with a lane a key (S = Q K^T) for dv^T += do^T w and dk^T += q^T ds.
// A sequence's first keys are seen by all of its rows: those beyond the window are shared out over many workgroups, in a launch of their own, and
// the parts joined by another.  Where there are few blocks of keys, the rows of each are cut into shares, joined in the same way.
// Rounding: w and ds become bf16 for the second product of each pass, at most half a step (2^-8) of the value; everything else is fp32.  delta from the
// output as it is stored, rounded and made of rounded weights, is off by some 1e-3 of its terms, which goes into dq times the row's weighted mean of
// the keys, and into dk times the queries.  But sum_j ds_j = 0: what that sum is short of zero is delta's error.  window_dq_kernel forms it, takes its
// part out of dq (see there), and leaves the exact delta for dk.  In rms: dq 2.2e-3, dk 2.4e-3, of which 1.7e-3 are their own rounding (1200 tokens,
// 64 columns); keys, queries and values with a mean as large as their spread: dq 2.3e-3 (1.0e-2 with delta from the output); 0.3 to 0.98 of a row's
// weight on one key eight times as long as the others: 2.1e-3 down to 1.7e-3 (256 columns, with two walks: 2.3e-3 to 2.5e-3).
// Bound by the matrix unit together with the exponentials and the products' operands from LDS: at 4 x 4096 tokens, 16 heads of 128 over 2, window
// 1024 and 4 first keys dq takes 266 us (its four products at 900 TFLOP/s), the keys' 302 to 309 (740), the first keys' 26 and 5 to join them.  With 64
// columns, where a score has half the products but the same exponential, 930 and 810 TFLOP/s (4 x 4096, 16 heads, all keys) beside 1000 and 860 with 128.
#include <algorithm>

#include "gdn_launch.h"
#include "gdn_window_attention.h"

namespace gdn {

namespace {

// sum + the eight values' sum
__device__ __forceinline__ float sum8(const bf16x8& x, float sum) {
    const bf16x2 one = {(bf16_t)1.f, (bf16_t)1.f};
#pragma unroll
    for (int e = 0; e < 4; e++) sum = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{x[2 * e], x[2 * e + 1]}, one, sum, false);
    return sum;
}

// Gradients of 128 rows, 32 to a wave.  delta is first formed from the output, and off by r; since the weights of a row add up to 1, r = sum_j ds_j.
// Up to 128 columns sum_j w_j k_j is carried beside dq, and r times it taken off in the end.  Both products take operands in bf16; r is there
// the quotient of their own sums, as they are rounded, so that the coefficients that the keys are left with add up to zero: where one key has nearly
// all of a row's weight, its coefficient is as good as the others', however small they are.  That is a fourth product to each tile.  At 128 columns
// there are registers for it with do's rows in LDS and tiles of 32 keys: backward, at 4 x 4096 tokens, 16 heads of 128 over 2, window 1024, 600 us (710
// with two walks, 557 with neither); 64 columns, 16 heads, all keys 620 (780 and 577).
// Above 128 columns the registers are short of it by far, and a walk of its own over the keys, without the third product, forms the exact delta
// before: 8 x 4096 tokens, 2 heads of 256 over one, window 1024, 710 us (1087 with the product and what it spills, 640 with neither).
template <int DP>
__global__ __launch_bounds__(256, DP <= 128 ? 2 : 1) void window_dq_kernel(const WindowParams p) {
    constexpr int KS = DP / 16, DT = DP / 32, KEYS = DP == 128 ? 32 : 64;
    constexpr bool OWN = DP != 128, TWICE = DP > 128;  // rows of do in registers; two walks
    using Loads = TileLoads<DP, KEYS / 4>;
    using RowLoads = TileLoads<DP, 32>;
    static_assert(row_offsets_fit(KEYS, false) && row_offsets_fit(32, true));
    __shared__ __attribute__((aligned(1024))) bf16_t tiles[2][2][KEYS * DP];
    __shared__ __attribute__((aligned(1024))) bf16_t do_rows[OWN ? 1 : WINDOW_ROWS * DP];
    int pair, block;
    work_item(p, blockIdx.x, pair, block);
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
    }
    const float lse = p.lse[scalar], c = p.negative ? -p.c : p.c;

    const RowView view = row_view(p, b, r);
    const WaveView w = wave_view(view);
    __shared__ int bounds[4][6];
    const WaveView all = join_waves<4>(w, bounds, wave, lane);
    const int lo = all.lo, end = all.end, sink = all.sink, sink_end = min(all.sink_end, lo);
    const int sink_tiles = sink_end > sink ? (sink_end - sink + KEYS - 1) / KEYS : 0, near_tiles = end > lo ? (end - lo + KEYS - 1) / KEYS : 0;
    const int tile_count = sink_tiles + near_tiles;

    const char* const kb = reinterpret_cast<const char*>(static_cast<const bf16_t*>(p.k.p) + b * p.k.b + hk * p.k.h);
    const char* const vb = reinterpret_cast<const char*>(static_cast<const bf16_t*>(p.v.p) + b * p.v.b + hk * p.v.h);
    const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)&tiles[0][0][0];
    auto tile_at = [&](int i, int& j0, int& count) {
        const bool s = i < sink_tiles;
        j0 = s ? sink + KEYS * i : lo + KEYS * (i - sink_tiles);
        count = min((s ? sink_end : end) - j0, KEYS);
    };
    auto load_tile = [&](int i, int buffer) {
        int j0, count;
        tile_at(i, j0, count);
        const char *const k0 = kb + (int64_t)j0 * p.k.t * 2, *const v0 = vb + (int64_t)j0 * p.v.t * 2;
        const uint32_t to = lds + buffer * 2 * KEYS * DP * 2;
#pragma unroll
        for (int x = 0; x < Loads::ITERS; x++) {
            const int kr = Loads::row(wave, lane, x), col = Loads::column(wave, lane, x);
            const bool there = kr < count && col < p.D;
            Loads::load(k0, there ? (uint32_t)(kr * (int)p.k.t + col) * 2 : PAST, to, wave, x);
            Loads::load(v0, there ? (uint32_t)(kr * (int)p.v.t + col) * 2 : PAST, to + KEYS * DP * 2, wave, x);
        }
    };

    TileReader<DP> reader(lane);
    f32x16 dq[DT] = {}, wk[TWICE ? 1 : DT] = {};
    float rest = 0.f, ds_sum = 0.f, w_sum = 0.f;  // the sum of ds; of ds and the weights as they are rounded
    int step = TWICE ? -tile_count : 0;
    if (!OWN && tile_count > 0) {  // a wave's own rows, which it reads behind the loads_done of its first tile
        const int first = block * WINDOW_ROWS + 32 * wave, t0 = p.G == 1 ? first : first / p.G, g0 = first - t0 * p.G;
        const char* const d0 = reinterpret_cast<const char*>(static_cast<const bf16_t*>(p.dout.p) + b * p.dout.b + hk * p.G * p.dout.h + t0 * p.dout.t);
        const uint32_t to = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)&do_rows[0];
#pragma unroll
        for (int x = 0; x < RowLoads::ITERS; x++) {
            const int rr = RowLoads::row(0, lane, x), col = RowLoads::column(0, lane, x);
            int tt, g;
            split_rows(p, g0 + rr, tt, g);
            RowLoads::load(d0, first + rr < p.rows && col < p.D ? (uint32_t)(tt * (int)p.dout.t + g * (int)p.dout.h + col) * 2 : PAST, to, wave, x);
        }
    }
    if (tile_count > 0) load_tile(0, step & 1);
    for (; step < tile_count; step++) {
        if (TWICE && step == 0) delta += rest + other_half(rest), rest = 0.f;
        const int i = step < 0 ? step + tile_count : step;
        loads_done();
        __syncthreads();
        reader.recompute();
        if (step + 1 < tile_count) load_tile(i + 1 == tile_count ? 0 : i + 1, (step + 1) & 1);
        int j0, count;
        tile_at(i, j0, count);
        const bf16_t *const kt = tiles[step & 1][0], *const vt = tiles[step & 1][1];
        const bool near = i >= sink_tiles, full = near && j0 >= w.full_lo && j0 + KEYS <= w.full_end;
        if (!w.meets(j0, count)) continue;
        const TileView own(view, near, sink_end);
#pragma unroll
        for (int x = 0; x < KEYS / 32; x++) {
            f32x16 s = {}, dw = {};
#pragma unroll
            for (int y = 0; y < KS; y++) s = mma(reader.across(kt, 32 * x, y), q[y], s);
            if constexpr (!OWN) __builtin_amdgcn_sched_barrier(0);  // (registers: operands of one product at a time)
#pragma unroll
            for (int y = 0; y < KS; y++) dw = mma(reader.across(vt, 32 * x, y), OWN ? d[y] : reader.across(do_rows, 32 * wave, y), dw);
#pragma unroll
            for (int e = 0; e < 16; e++) s[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], c, -lse)), dw[e] = s[e] * (dw[e] - delta);
            if (!full) {
                stay_a_branch();
                if (!(near && j0 < all.sink_end)) {
#pragma unroll
                    for (int e = 0; e < 16; e++)
                        if (!own.sees(j0 + 32 * x + acc_row(e, half))) s[e] = dw[e] = 0.f;
                } else {
#pragma unroll
                    for (int e = 0; e < 16; e++)
                        if (!own.sees_mixed(j0 + 32 * x + acc_row(e, half))) s[e] = dw[e] = 0.f;
                }
            }
#pragma unroll
            for (int e = 0; e < 16; e++) rest += dw[e];
            if (TWICE && step < 0) continue;
#pragma unroll
            for (int y = 0; y < 2; y++) {
                const bf16x8 ds = pack8(dw, y);
                if constexpr (TWICE) {
#pragma unroll
                    for (int z = 0; z < DT; z++) dq[z] = mma(reader.down(kt, 2 * x + y, z), ds, dq[z]);
                } else {
                    const bf16x8 weights = pack8(s, y);
                    ds_sum = sum8(ds, ds_sum), w_sum = sum8(weights, w_sum);
#pragma unroll
                    for (int z = 0; z < DT; z++) {
                        const bf16x8 k = reader.down(kt, 2 * x + y, z);
                        dq[z] = mma(k, ds, dq[z]), wk[z] = mma(k, weights, wk[z]);
                    }
                }
            }
        }
    }
    delta += rest + other_half(rest);
    if constexpr (!TWICE) {
        ds_sum += other_half(ds_sum), w_sum += other_half(w_sum);
        const float by = w_sum == 0.f ? 0.f : ds_sum / w_sum;
#pragma unroll
        for (int z = 0; z < DT; z++)
#pragma unroll
            for (int e = 0; e < 16; e++) dq[z][e] = __builtin_fmaf(wk[z][e], -by, dq[z][e]);
    }
    int last = row;
    asm volatile("" : "+v"(last));  // (what follows from it is formed anew, rather than kept in registers over the walk)
    if (last >= p.rows) return;
    const int last_t = p.G == 1 ? last : last / p.G, last_head = hk * p.G + (last - last_t * p.G);
    if (half == 0) p.delta[((int64_t)b * p.T + last_t) * p.H + last_head] = delta;
    store_transposed<DP>(static_cast<bf16_t*>(const_cast<void*>(p.dq.p)) + b * p.dq.b + last_t * p.dq.t + last_head * p.dq.h, p.D, half, dq, p.scale);
}

// Gradients of KEYS keys.  The keys and values lie in LDS for the whole walk, so that a wave's registers are its sums': two waves on a SIMD, one
// of which has products to do while the other waits (with keys and values in registers, and one wave, the walk took 560 us instead of 330 at
// 4 x 4096 tokens, 16 heads of 128 over 2, window 1024).
// A wave has 32 keys and 32 rows of each tile; the waves that share keys add up at the end.  Above 128 columns, where the sums of both
// gradients would not fit into its registers, a wave has one of them, and scores are formed twice (ROLES 2).
// Not FIRST: all keys, and the rows that have them in their window; 128 keys (64) and tiles of 64 rows (32), the next one on its way.
// FIRST: the keys of a sequence that all of its rows see, 32 of them, and of those rows that do not have them in their window one part, in tiles of
// 256 rows (64): (sequence, head of k and v, block of such keys, part).  Both leave their sums for such keys to window_first_keys_kernel.
template <int DP, bool FIRST, bool SHARED>
__global__ __launch_bounds__(DP == 128 ? 512 : 256, DP == 64 ? 3 : DP == 128 ? 2 : 1) void window_dkv_kernel(const WindowParams p) {
    constexpr int KS = DP / 16, DT = DP / 32, KEYS = FIRST ? WINDOW_FIRST_KEYS : window_keys(DP), ROLES = DP <= 128 ? 1 : 2, WAVES = DP == 128 ? 8 : 4;
    constexpr int KEY_WAVES = KEYS / 32, ROW_WAVES = WAVES / ROLES / KEY_WAVES, ROWS = 32 * ROW_WAVES, BUFFERS = FIRST ? 1 : 2;
    using Loads = TileLoads<DP, ROWS / WAVES>;
    using KeyLoads = TileLoads<DP, 16>;
    static_assert(row_offsets_fit(ROWS / WAVES, true) && row_offsets_fit(KEYS, false));  // (all of a tile's rows: FROM_WAVE)
    __shared__ __attribute__((aligned(1024))) bf16_t lds_tiles[2 * KEYS * DP + BUFFERS * 2 * ROWS * DP];  // keys, values; rows of q, of do
    __shared__ __attribute__((aligned(16))) float row_lse[BUFFERS][ROWS], row_delta[BUFFERS][ROWS];
    __shared__ __attribute__((aligned(16))) int row_at[BUFFERS][ROWS];
    __shared__ int bounds[WAVES][6];
    const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), half = lane >> 5;
    const int key_wave = wave % KEY_WAVES, row_wave = wave / KEY_WAVES % ROW_WAVES, role = wave / KEY_WAVES / ROW_WAVES;  // role 0: dk (and dv), 1: dv
    int b, hk, n = 0, piece = p.pieces + (SHARED ? (int)blockIdx.y : 0), key0, keys;  // key0: of the workgroup
    if constexpr (FIRST) {
        const int key_blocks = p.first_keys / KEYS;
        int x = blockIdx.x;
        piece = x % p.pieces, x /= p.pieces;
        const int kblock = x % key_blocks;
        x /= key_blocks;
        hk = x % p.HK, n = x / p.HK;
        b = p.cu != nullptr && !p.padded ? 0 : n;
        int st, len;
        sequence_of(p, n, st, len);
        key0 = st + kblock * KEYS, keys = min(KEYS, min(p.sinks, len) - kblock * KEYS);
    } else {
        int pair, block;
        work_item(p, blockIdx.x, pair, block);
        b = pair / p.HK, hk = pair - b * p.HK;
        key0 = block * KEYS, keys = min(KEYS, p.S - key0);
    }
    // this lane's key, and the positions that see it: [from, upto]
    const int own = 32 * key_wave + (lane & 31), j = key0 + own;
    int st = 0, en = 0, from = 1 << 30, upto = -1;
    if (own < keys) {
        int sequence;
        sequence_at(p, b, j, st, en, sequence);
        if (!FIRST) n = sequence;
        if (en > st) {
            if (FIRST) from = p.window < en - j ? j + p.window : 1 << 30, upto = from < en ? en - 1 : -1;
            else from = j, upto = p.window == 0 || p.window >= en - j || (p.pieces == 0 && j - st < p.sinks) ? en - 1 : j + p.window - 1;
            from = max(from, p.S - p.T);  // (positions in front of the queries)
            if (upto < from) from = 1 << 30, upto = -1;
        }
    }
    WaveView w;
    w.lo = wave_min(from), w.end = wave_max(upto) + 1, w.full_lo = wave_max(from), w.full_end = wave_min(upto) + 1, w.sink = w.sink_end = 0;
    const WaveView all = join_waves<WAVES>(w, bounds, wave, lane);
    const int offset = p.S - p.T;
    int a0 = all.lo, a1 = all.end;  // positions whose rows are walked over
    if (a1 <= a0) a0 = a1 = offset;
    if constexpr (FIRST) {
        const int each = (a1 - a0 + p.pieces - 1) / p.pieces;
        a0 = min(a1, a0 + piece * each), a1 = min(a1, a0 + each);
    }
    int r0 = (a0 - offset) * p.G, r1 = (a1 - offset) * p.G;
    if constexpr (SHARED) {
        const int each = ((r1 - r0 + ROWS - 1) / ROWS + p.shares - 1) / p.shares * ROWS;
        r0 = min(r1, r0 + (int)blockIdx.y * each), r1 = min(r1, r0 + each);
    }
    const int tile_count = (r1 - r0 + ROWS - 1) / ROWS;

    const char* const qb = reinterpret_cast<const char*>(static_cast<const bf16_t*>(p.q.p) + b * p.q.b + hk * p.G * p.q.h);
    const char* const db = reinterpret_cast<const char*>(static_cast<const bf16_t*>(p.dout.p) + b * p.dout.b + hk * p.G * p.dout.h);
    bf16_t *const kt = lds_tiles, *const vt = kt + KEYS * DP, *const rows = vt + KEYS * DP;
    const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)&lds_tiles[0];
    {
        const char* const k0 = reinterpret_cast<const char*>(static_cast<const bf16_t*>(p.k.p) + b * p.k.b + hk * p.k.h + (keys > 0 ? key0 : 0) * p.k.t);
        const char* const v0 = reinterpret_cast<const char*>(static_cast<const bf16_t*>(p.v.p) + b * p.v.b + hk * p.v.h + (keys > 0 ? key0 : 0) * p.v.t);
        if (tile_count > 0 && wave < KEYS / 16) {  // (the walk's first tile waits for them)
#pragma unroll
            for (int x = 0; x < KeyLoads::ITERS; x++) {
                const int kr = KeyLoads::row(wave, lane, x), col = KeyLoads::column(wave, lane, x);
                const bool there = kr < keys && col < p.D;
                KeyLoads::load(k0, there ? (uint32_t)(kr * (int)p.k.t + col) * 2 : PAST, lds, wave, x);
                KeyLoads::load(v0, there ? (uint32_t)(kr * (int)p.v.t + col) * 2 : PAST, lds + KEYS * DP * 2, wave, x);
            }
        }
    }
    float lse_next = 0.f, delta_next = 0.f;
    int at_next = 0;
    auto load_tile = [&](int i) {
        const int first = r0 + ROWS * i, count = min(ROWS, r1 - first);
        const int t0 = p.G == 1 ? first : first / p.G, g0 = first - t0 * p.G;
        // Where the bytes of a whole tile's rows (256 tokens) would pass what the offsets hold, they go from the wave's first row on.  (Everywhere: 328
        // us instead of 302 at 4 x 4096 tokens, 16 heads of 128 over 2, window 1024.)
        constexpr bool FROM_WAVE = !row_offsets_fit(ROWS, true);
        const int base_row = FROM_WAVE ? Loads::row(wave, 0, 0) : 0;
        int t1 = 0, g1 = g0;
        if constexpr (FROM_WAVE) split_rows(p, g0 + base_row, t1, g1);
        const char *const q0 = qb + (int64_t)(t0 + t1) * p.q.t * 2, *const d0 = db + (int64_t)(t0 + t1) * p.dout.t * 2;
        const uint32_t to = lds + (2 * KEYS + (i % BUFFERS) * 2 * ROWS) * DP * 2;
#pragma unroll
        for (int x = 0; x < Loads::ITERS; x++) {
            const int rr = Loads::row(wave, lane, x), col = Loads::column(wave, lane, x);
            int tt, g;
            split_rows(p, g1 + rr - base_row, tt, g);
            const bool there = rr < count && col < p.D;
            Loads::load(q0, there ? (uint32_t)(tt * (int)p.q.t + g * (int)p.q.h + col) * 2 : PAST, to, wave, x);
            Loads::load(d0, there ? (uint32_t)(tt * (int)p.dout.t + g * (int)p.dout.h + col) * 2 : PAST, to + ROWS * DP * 2, wave, x);
        }
        if (threadIdx.x < ROWS) {
            int tt, g;
            split_rows(p, g0 + (int)threadIdx.x, tt, g);
            const bool there = (int)threadIdx.x < count;
            const int64_t scalar = ((int64_t)b * p.T + t0 + (there ? tt : 0)) * p.H + hk * p.G + (there ? g : 0);
            lse_next = there ? p.lse[scalar] : __builtin_inff(), delta_next = there ? p.delta[scalar] : 0.f;
            at_next = there ? t0 + tt + offset : -1;
        }
    };

    TileReader<DP> reader(lane);
    const float c = p.negative ? -p.c : p.c;
    f32x16 dk[DT] = {}, dv[ROLES == 1 ? DT : 1] = {};  // (two roles: dk is the one gradient that there is)
    // `full`: every row of the tile sees every key of the wave
    auto add_tile = [&](int i, bool full) {
        reader.recompute();
        const bf16_t *const qt = rows + (i % BUFFERS) * 2 * ROWS * DP, *const dt = qt + ROWS * DP;
        const int at0 = 32 * row_wave + 4 * half;
        const bf16_t *const qx = qt + 32 * row_wave * DP, *const dx = dt + 32 * row_wave * DP;
        f32x16 s = {}, dw = {};
#pragma unroll
        for (int y = 0; y < KS; y++) {
            s = mma(reader.across(qx, 0, y), reader.across(kt + 32 * key_wave * DP, 0, y), s);
            if (ROLES == 1 || role == 0) dw = mma(reader.across(dx, 0, y), reader.across(vt + 32 * key_wave * DP, 0, y), dw);
        }
#pragma unroll
        for (int y = 0; y < 4; y++) {
            const f32x4 lse = *reinterpret_cast<const f32x4*>(&row_lse[i % BUFFERS][at0 + 8 * y]);
            const f32x4 delta = *reinterpret_cast<const f32x4*>(&row_delta[i % BUFFERS][at0 + 8 * y]);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                s[4 * y + e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[4 * y + e], c, -lse[e]));
                dw[4 * y + e] = s[4 * y + e] * (dw[4 * y + e] - delta[e]);
            }
        }
        if (!full) {
            stay_a_branch();
#pragma unroll
            for (int y = 0; y < 4; y++) {
                const i32x4 at = *reinterpret_cast<const i32x4*>(&row_at[i % BUFFERS][at0 + 8 * y]);
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (at[e] < from || at[e] > upto) s[4 * y + e] = dw[4 * y + e] = 0.f;
            }
        }
        if constexpr (ROLES == 1) {
#pragma unroll
            for (int y = 0; y < 2; y++) {
                const bf16x8 weights = pack8(s, y), ds = pack8(dw, y);
#pragma unroll
                for (int z = 0; z < DT; z++) dv[z] = mma(reader.down(dx, y, z), weights, dv[z]);
#pragma unroll
                for (int z = 0; z < DT; z++) dk[z] = mma(reader.down(qx, y, z), ds, dk[z]);
            }
        } else {
            const bf16_t* const from_rows = role == 0 ? qx : dx;
#pragma unroll
            for (int y = 0; y < 2; y++) {
                const bf16x8 by = role == 0 ? pack8(dw, y) : pack8(s, y);
#pragma unroll
                for (int z = 0; z < DT; z++) dk[z] = mma(reader.down(from_rows, y, z), by, dk[z]);
            }
        }
    };
    if (tile_count > 0) load_tile(0);
    for (int i = 0; i < tile_count; i++) {
        loads_done();
        if (threadIdx.x < ROWS) row_lse[i % BUFFERS][threadIdx.x] = lse_next, row_delta[i % BUFFERS][threadIdx.x] = delta_next, row_at[i % BUFFERS][threadIdx.x] = at_next;
        __syncthreads();
        if (BUFFERS == 2 && i + 1 < tile_count) load_tile(i + 1);
        const int first = r0 + ROWS * i, count = min(ROWS, r1 - first);
        const int p0 = (p.G == 1 ? first : first / p.G) + offset, p1 = (p.G == 1 ? first + count - 1 : (first + count - 1) / p.G) + offset;  // positions
        if (p0 < w.end && p1 >= w.lo) add_tile(i, p0 >= w.full_lo && p1 < w.full_end && count == ROWS);
        if (BUFFERS == 1 && i + 1 < tile_count) {
            __syncthreads();
            load_tile(i + 1);
        }
    }
    // the waves that share keys, half of them to the other half
    if constexpr (ROW_WAVES > 1) {
        constexpr int TENSORS = ROLES == 1 ? 2 : 1, PIECES = TENSORS * DT * 4;  // f32x4 of a lane
        static_assert(ROW_WAVES / 2 * KEY_WAVES * ROLES * PIECES * 64 * 16 <= sizeof(lds_tiles), "the sums fit");
        loads_done();
#pragma unroll
        for (int h = ROW_WAVES / 2; h >= 1; h /= 2) {
            f32x4* const shared = reinterpret_cast<f32x4*>(lds_tiles) + ((row_wave % h) * KEY_WAVES * ROLES + role * KEY_WAVES + key_wave) * PIECES * 64 + lane;
            __syncthreads();
            if (row_wave >= h && row_wave < 2 * h) {
#pragma unroll
                for (int z = 0; z < DT; z++)
#pragma unroll
                    for (int y = 0; y < 4; y++) {
                        shared[(4 * z + y) * 64] = f32x4{dk[z][4 * y], dk[z][4 * y + 1], dk[z][4 * y + 2], dk[z][4 * y + 3]};
                        if constexpr (ROLES == 1) shared[(4 * (DT + z) + y) * 64] = f32x4{dv[z][4 * y], dv[z][4 * y + 1], dv[z][4 * y + 2], dv[z][4 * y + 3]};
                    }
            }
            __syncthreads();
            if (row_wave < h) {
#pragma unroll
                for (int z = 0; z < DT; z++)
#pragma unroll
                    for (int y = 0; y < 4; y++) {
                        const f32x4 a = shared[(4 * z + y) * 64];
#pragma unroll
                        for (int e = 0; e < 4; e++) dk[z][4 * y + e] += a[e];
                        if constexpr (ROLES == 1) {
                            const f32x4 d = shared[(4 * (DT + z) + y) * 64];
#pragma unroll
                            for (int e = 0; e < 4; e++) dv[z][4 * y + e] += d[e];
                        }
                    }
            }
        }
        if (row_wave > 0) return;
    }
    if (own >= keys) return;
    const bool to_parts = p.pieces > 0 && en > st && j - st < p.sinks;
    float* const part = p.part_dk + (to_parts ? ((((int64_t)n * p.HK + hk) * (p.pieces + p.shares) + piece) * p.first_keys + (j - st)) * 2 * p.D : 0);
    auto leave = [&](const f32x16 (&sums)[DT], bool value) {
        const WindowRows& out = value ? p.dv : p.dk;
        if (!FIRST && !SHARED && !to_parts) store_transposed<DP>(static_cast<bf16_t*>(const_cast<void*>(out.p)) + b * out.b + j * out.t + hk * out.h, p.D, half, sums, value ? 1.f : p.scale);
        if (!SHARED && !to_parts) return;
        float* const to = (to_parts ? part : p.part_all + ((((int64_t)blockIdx.y * p.B + b) * p.HK + hk) * p.S + j) * 2 * p.D) + (value ? p.D : 0);
#pragma unroll
        for (int z = 0; z < DT; z++)
#pragma unroll
            for (int y = 0; y < 4; y++) {
                const int col = 32 * z + 8 * y + 4 * half;
                if (col < p.D) *reinterpret_cast<f32x4*>(to + col) = f32x4{sums[z][4 * y], sums[z][4 * y + 1], sums[z][4 * y + 2], sums[z][4 * y + 3]};
            }
    };
    if constexpr (ROLES == 1) {
        leave(dk, false);
        leave(dv, true);
    } else {
        leave(dk, role == 1);
    }
}

// The parts of a sequence's first keys joined, in their order: a workgroup a key, the parts shared out over its threads' groups.
__global__ __launch_bounds__(256) void window_first_keys_kernel(const WindowParams p) {
    __shared__ f32x4 shared[256];
    int x = blockIdx.x;
    const int i = x % p.sinks;
    x /= p.sinks;
    const int hk = x % p.HK, n = x / p.HK, b = p.cu != nullptr && !p.padded ? 0 : n;
    int st, len;
    sequence_of(p, n, st, len);
    if (i >= len) return;
    const int quads = 2 * p.D / 4, groups = max(1, 256 / quads), group = threadIdx.x / quads, at = threadIdx.x - group * quads;  // 2 D <= 512 numbers a part
    const float* const from = p.part_dk + (((int64_t)n * p.HK + hk) * (p.pieces + p.shares) * p.first_keys + i) * 2 * p.D + 4 * at;
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    if (group < groups) {
#pragma unroll 8
        for (int y = group; y < p.pieces + p.shares; y += groups) sum += *reinterpret_cast<const f32x4*>(from + (int64_t)y * p.first_keys * 2 * p.D);
    }
    shared[threadIdx.x] = sum;
    __syncthreads();
    if (group != 0) return;
    for (int y = 1; y < groups; y++) sum += shared[y * quads + at];
    const int col = 4 * at;
    if (col < p.D) store4<bf16_t>(static_cast<bf16_t*>(const_cast<void*>(p.dk.p)) + b * p.dk.b + (st + i) * p.dk.t + hk * p.dk.h + col, sum * p.scale);
    else store4<bf16_t>(static_cast<bf16_t*>(const_cast<void*>(p.dv.p)) + b * p.dv.b + (st + i) * p.dv.t + hk * p.dv.h + col - p.D, sum);
}

// The shares of the other keys joined, in their order: a thread four columns.
__global__ __launch_bounds__(256) void window_shares_kernel(const WindowParams p) {
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x, keys = (int64_t)p.B * p.HK * p.S;
    const int quads = 2 * p.D / 4;
    const int64_t key = at / quads;
    if (key >= keys) return;
    const int64_t pair = key / p.S;
    const int col = 4 * (int)(at - key * quads), j = (int)(key - pair * p.S), b = (int)(pair / p.HK), hk = (int)(pair - (int64_t)b * p.HK);
    if (p.pieces > 0) {
        int st, en, n;
        sequence_at(p, b, j, st, en, n);
        if (en > st && j - st < p.sinks) return;
    }
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int y = 0; y < p.shares; y++) sum += *reinterpret_cast<const f32x4*>(p.part_all + (y * keys + key) * 2 * p.D + col);
    if (col < p.D) store4<bf16_t>(static_cast<bf16_t*>(const_cast<void*>(p.dk.p)) + b * p.dk.b + j * p.dk.t + hk * p.dk.h + col, sum * p.scale);
    else store4<bf16_t>(static_cast<bf16_t*>(const_cast<void*>(p.dv.p)) + b * p.dv.b + j * p.dv.t + hk * p.dv.h + col - p.D, sum);
}

template <int DP>
int launch_bwd(const WindowParams& p, hipStream_t stream) {
    WindowParams r = p, k = p;
    r.blocks = (p.rows + WINDOW_ROWS - 1) / WINDOW_ROWS, k.blocks = (p.S + window_keys(DP) - 1) / window_keys(DP);
    const auto grid = [&](const WindowParams& x) { return dim3((unsigned)((int64_t)p.B * p.HK * x.blocks)); };
    hipLaunchKernelGGL((window_dq_kernel<DP>), grid(r), dim3(256), 0, stream, r);
    if (const int e = (int)hipGetLastError(); e != 0) return e;
    const dim3 threads(DP == 128 ? 512 : 256);
    if (p.pieces > 0) {
        hipLaunchKernelGGL((window_dkv_kernel<DP, true, false>), dim3((unsigned)((int64_t)p.N * p.HK * (p.first_keys / WINDOW_FIRST_KEYS) * p.pieces)), threads, 0, stream, k);
        if (const int e = (int)hipGetLastError(); e != 0) return e;
    }
    if (p.shares > 1) hipLaunchKernelGGL((window_dkv_kernel<DP, false, true>), dim3(grid(k).x, p.shares), threads, 0, stream, k);
    else hipLaunchKernelGGL((window_dkv_kernel<DP, false, false>), grid(k), threads, 0, stream, k);
    if (const int e = (int)hipGetLastError(); e != 0) return e;
    if (p.shares > 1) {
        const int64_t quads = (int64_t)p.B * p.HK * p.S * (2 * p.D / 4);
        hipLaunchKernelGGL(window_shares_kernel, dim3((unsigned)((quads + 255) / 256)), dim3(256), 0, stream, k);
        if (const int e = (int)hipGetLastError(); e != 0) return e;
    }
    if (p.pieces == 0) return GDN_OK;
    hipLaunchKernelGGL(window_first_keys_kernel, dim3((unsigned)((int64_t)p.N * p.HK * p.sinks)), dim3(256), 0, stream, k);
    return (int)hipGetLastError();
}

}  // namespace

int launch_window_bwd(const WindowParams& p, hipStream_t stream) {
    if (p.D <= 64) return launch_bwd<64>(p, stream);
    if (p.D <= 128) return launch_bwd<128>(p, stream);
    return launch_bwd<256>(p, stream);
}

}  // namespace gdn
