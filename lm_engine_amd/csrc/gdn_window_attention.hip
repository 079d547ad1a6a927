// Softmax attention over a window, forward, bf16 (include/gdn_attention_hip.h, gdn_window_attention.h).
//
// A workgroup has 128 rows, 32 to a wave, and walks over the keys that they see in tiles of 64.  Scores are formed as S^T = K Q^T, so that a
// lane holds one row: its maximum and sum need one exchange between lanes, and P^T is the next product's operand O^T += V^T P^T as it
// lies in registers.  Keys and values go from memory into LDS without registers, the next tile while this one is worked on.
// Softmax in one pass: weights are 2^(c s - m), m the largest c s that was met when it last passed the reference by 8 (2^8 is no harm
// to fp32 sums, and bf16 rounds relative to the weight), so that the outputs are seldom rescaled.
// Rounding: the weights become bf16 for the second product, at most half a step (2^-8) of each, 1.7e-3 rms of the output's norm; their sum l is of the
// weights before that.  Everything else is fp32 up to the output's own rounding.
// Bound by the matrix unit and the exponentials beside it: 4 x 4096 tokens, 16 heads of 128 over 2, window 1024 and 4 first keys 157 us
// (770 TFLOP/s; a large library product reaches 1165), over 16 and all keys 302 (910).  128 rows and four waves, two workgroups to a compute unit: 256 rows and
// eight waves took 178 instead of 158 us.  With 64 columns, where the exponentials alone take twice the products' time, 700 TFLOP/s.  Small calls
// are bound by latency, 8 to 14 us: a launch's instructions come from L2 once, and one workgroup after the other finds the same.
#include <algorithm>

#include "gdn_join.h"
#include "gdn_launch.h"
#include "gdn_window_attention.h"

namespace gdn {

namespace {

// zeros in the place of what is not finite; whether there was any
__device__ __forceinline__ bool make_finite(bf16x8& x) {
    i32x4 w = __builtin_bit_cast(i32x4, x);
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 4; e++) bad |= (w[e] & 0x7f80) == 0x7f80 || (w[e] & 0x7f800000) == 0x7f800000;
    if (!bad) return false;
#pragma unroll
    for (int e = 0; e < 4; e++) w[e] = ((w[e] & 0x7f80) == 0x7f80 ? 0 : w[e] & 0xffff) | ((w[e] & 0x7f800000) == 0x7f800000 ? 0 : w[e] & 0xffff0000);
    x = __builtin_bit_cast(bf16x8, w);
    return true;
}

template <int DP>
__global__ __launch_bounds__(256, DP <= 128 ? 2 : 1) void window_fwd_kernel(const WindowParams p) {
    constexpr int KS = DP / 16, DT = DP / 32;
    using Loads = TileLoads<DP>;
    static_assert(row_offsets_fit(64, false));
    __shared__ __attribute__((aligned(1024))) bf16_t tiles[2][2][64 * DP];  // keys, values; tiles in turn
    int pair, block;
    work_item(p, blockIdx.x, pair, block);
    block = p.blocks - 1 - block;  // the rows that see most keys first
    const int b = pair / p.HK, hk = pair - b * p.HK;
    const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), half = lane >> 5;
    const int r0 = block * WINDOW_ROWS;
    const int row = r0 + 32 * wave + (lane & 31), r = min(row, p.rows - 1);  // (past the end: the last row once more, and not stored)
    const int t = p.G == 1 ? r : r / p.G, g = r - t * p.G;

    bf16x8 q[KS];
    load_row_fragments<DP>(static_cast<const bf16_t*>(p.q.p) + b * p.q.b + t * p.q.t + (hk * p.G + g) * p.q.h, p.D, half, true, q);
    if (p.negative)
#pragma unroll
        for (int s = 0; s < KS; s++) q[s] = -q[s];

    const RowView view = row_view(p, b, r);
    // keys that the workgroup needs: [lo, end) and the first ones of its first row's sequence, [sink, sink_end)
    const WaveView w = wave_view(view);
    __shared__ int bounds[4][6];
    const WaveView all = join_waves<4>(w, bounds, wave, lane);
    const int lo = all.lo, end = all.end, sink = all.sink, sink_end = min(all.sink_end, lo);

    const int sink_tiles = sink_end > sink ? (sink_end - sink + 63) / 64 : 0, near_tiles = end > lo ? (end - lo + 63) / 64 : 0;
    int first_tile = 0, last_tile = sink_tiles + near_tiles;
    if (p.splits > 1) {
        const int each = (last_tile + p.splits - 1) / p.splits;
        first_tile = min((int)blockIdx.y * each, last_tile), last_tile = min(first_tile + each, last_tile);
    }

    const char* const kb = reinterpret_cast<const char*>(static_cast<const bf16_t*>(p.k.p) + b * p.k.b + hk * p.k.h);
    const char* const vb = reinterpret_cast<const char*>(static_cast<const bf16_t*>(p.v.p) + b * p.v.b + hk * p.v.h);
    const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)&tiles[0][0][0];
    auto tile_at = [&](int i, int& j0, int& count) {
        const bool s = i < sink_tiles;
        j0 = s ? sink + 64 * i : lo + 64 * (i - sink_tiles);
        count = min((s ? sink_end : end) - j0, 64);
    };
    const int row0 = Loads::row(wave, lane, 0);
    const uint32_t place = 2 * Loads::column(wave, lane, 0), key_bytes = (uint32_t)(row0 * (int)p.k.t) * 2, value_bytes = (uint32_t)(row0 * (int)p.v.t) * 2;
    // keys and values of tile i, into the half of their buffer that i's parity names
    using Request = TileRequest<DP>;
    auto keys_of = [&](int i) {
        int j0, count;
        tile_at(i, j0, count);
        if (i >= last_tile) j0 = 0, count = 0;
        return Request{kb + (int64_t)j0 * p.k.t * 2, (int)p.k.t, count, p.D, lds + (i & 1) * 64 * DP * 2, key_bytes, place, row0};
    };
    auto values_of = [&](int i) {
        int j0, count;
        tile_at(i, j0, count);
        return Request{vb + (int64_t)j0 * p.v.t * 2, (int)p.v.t, count, p.D, lds + (2 + (i & 1)) * 64 * DP * 2, value_bytes, place, row0};
    };

    TileReader<DP> reader(lane);
    f32x16 o[DT], s_even[2], s_odd[2];
    float m, l;
    bool careful = false, taken_out = false;
    auto scores = [&](int i, f32x16 (&to)[2]) {
        const bf16_t* const kt = tiles[0][i & 1];
#pragma unroll
        for (int y = 0; y < KS; y++)
#pragma unroll
            for (int x = 0; x < 2; x++) to[x] = mma(reader.across(kt, 32 * x, y), q[y], y == 0 ? f32x16{} : to[x]);
    };
    // Tile i, whose scores are in s; NEXT: the next one's scores are formed beside its weights, where the matrix unit would have nothing to do
    auto step = [&](int i, f32x16 (&s)[2], f32x16 (&s_next)[2], auto next) {
        int j0, count;
        tile_at(i, j0, count);
        const bool near = i >= sink_tiles, full = near && j0 >= w.full_lo && j0 + 64 <= w.full_end;
        if (careful && !(near && j0 >= all.full_lo && j0 + 64 <= all.full_end)) {
            bf16x8* const v8 = reinterpret_cast<bf16x8*>(tiles[1][i & 1]);
            bool found = false;
#pragma unroll
            for (int x = 0; x < 64 * DP / 8 / 256; x++) {
                bf16x8 v = v8[threadIdx.x + 256 * x];
                if (make_finite(v)) v8[threadIdx.x + 256 * x] = v, found = true;
            }
            taken_out |= __syncthreads_or(found) != 0;
        }
        Request keys, values;
        if constexpr (next()) keys = keys_of(i + 2), values = values_of(i + 1);
        if (!w.meets(j0, count)) {
            if constexpr (next()) {
                keys.all(wave), values.all(wave);
                scores(i + 1, s_next);
            }
            return;
        }
        float c = p.c;
        if (!full) {
            stay_a_branch();
            const TileView own(view, near, sink_end);
            c = 1.f;
            if (!(near && j0 < all.sink_end)) {
#pragma unroll
                for (int x = 0; x < 2; x++)
#pragma unroll
                    for (int e = 0; e < 16; e++) s[x][e] = own.sees(j0 + 32 * x + acc_row(e, half)) ? s[x][e] * p.c : -__builtin_inff();
            } else {
#pragma unroll
                for (int x = 0; x < 2; x++)
#pragma unroll
                    for (int e = 0; e < 16; e++) s[x][e] = own.sees_mixed(j0 + 32 * x + acc_row(e, half)) ? s[x][e] * p.c : -__builtin_inff();
            }
        }
        float top = s[0][0];
#pragma unroll
        for (int x = 0; x < 2; x++)
#pragma unroll
            for (int e = 0; e < 16; e++) top = fmaxf(top, s[x][e]);
        top = fmaxf(top, other_half(top)) * c;
        if (__builtin_amdgcn_ballot_w64(top > m + 8.f) != 0) {
            const float reference = fmaxf(m, top), alpha = __builtin_amdgcn_exp2f(m - reference);
            m = reference;
            l *= alpha;
#pragma unroll
            for (int x = 0; x < DT; x++) o[x] *= alpha;
        }
        // Products one after the other, each with the reading of the operand for the one four further on, its share of the weights' arithmetic
        // and of the loads of the tiles to come, in this order (the compiler's own has every product wait for its operand).
        constexpr int AHEAD = 2, QK = 2 * KS, PV = 4 * DT, EACH = 32 / QK;
        const bf16_t *const kt = tiles[0][(i + 1) & 1], *const vt = tiles[1][i & 1];
        __builtin_amdgcn_s_setprio(1);  // before the wave that is between its products
        bf16x8 ahead[AHEAD], weights[4];
        float sum = 0.f;
        auto fetch = [&](int k) {  // product k's operand: of keys, then of values
            return k < QK ? reader.across(kt, 32 * (k & 1), k >> 1) : reader.down(vt, (k - QK) / DT, (k - QK) % DT);
        };
        constexpr int BEGIN = next() ? 0 : QK;
#pragma unroll
        for (int k = 0; k < AHEAD; k++) ahead[k] = fetch(BEGIN + k);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int k = 0; k < QK; k++) {
            if constexpr (next()) {
                s_next[k & 1] = mma(ahead[k % AHEAD], q[k >> 1], k < 2 ? f32x16{} : s_next[k & 1]);
                ahead[k % AHEAD] = fetch(k + AHEAD);
                if (k % 2 == 0) k < QK / 2 ? values.piece(wave, k / 2) : keys.piece(wave, (k - QK / 2) / 2);
            }
#pragma unroll
            for (int e = EACH * k; e < EACH * (k + 1); e++) {
                s[e >> 4][e & 15] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e >> 4][e & 15], c, -m));
                sum += s[e >> 4][e & 15];
                if (e % 8 == 7) weights[e >> 3] = pack8(s[e >> 4], e >> 3 & 1);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        l += sum;
        __builtin_amdgcn_s_setprio(2);
#pragma unroll
        for (int k = 0; k < PV; k++) {
            o[k % DT] = mma(ahead[k % AHEAD], weights[k / DT], o[k % DT]);
            if (k + AHEAD < PV) ahead[k % AHEAD] = fetch(QK + k + AHEAD);
            __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_setprio(0);
    };
    for (;;) {
        m = LOWEST, l = 0.f;
#pragma unroll
        for (int x = 0; x < DT; x++) o[x] = f32x16{};
        if (first_tile >= last_tile) break;
        keys_of(first_tile).all(wave);
        if constexpr (DP <= 128) {  // scores of the next tile beside this one's weights: 316 us instead of 347 at 4 x 4096, 16 heads of 128, all keys
            loads_done();
            __syncthreads();
            values_of(first_tile).all(wave);
            keys_of(first_tile + 1).all(wave);
            scores(first_tile, s_even);
            // here: the scores of tile i are in s, its values and the keys of the next one have been asked for
            int i = first_tile;
            auto advance = [&]() {
                loads_done();
                __syncthreads();
                reader.recompute();
            };
            for (; i + 2 < last_tile; i++) {
                advance();
                step(i, s_even, s_odd, std::true_type{});
                i++;
                advance();
                step(i, s_odd, s_even, std::true_type{});
            }
            if (i + 1 < last_tile) {
                advance();
                step(i, s_even, s_odd, std::true_type{});
                s_even[0] = s_odd[0], s_even[1] = s_odd[1];
            }
            advance();
            step(last_tile - 1, s_even, s_odd, std::false_type{});
        } else {  // (the next tile's scores find no registers)
            values_of(first_tile).all(wave);
            for (int i = first_tile; i < last_tile; i++) {
                loads_done();
                __syncthreads();
                if (i + 1 < last_tile) keys_of(i + 1).all(wave), values_of(i + 1).all(wave);
                scores(i, s_even);
                step(i, s_even, s_odd, std::false_type{});
            }
        }
        if (careful) break;
        // 0 times a value that is not finite must not reach the rows that do not see it.  Where a result is not finite, the walk is
        // taken once more, without such values in tiles that some row does not see all of; they go to the rows that see them in the end.
        float zero = 0.f;
#pragma unroll
        for (int x = 0; x < DT; x++)
#pragma unroll
            for (int e = 0; e < 16; e++) zero = __builtin_fmaf(o[x][e], 0.f, zero);
        if (!__syncthreads_or(zero != 0.f)) break;
        careful = true;
    }

    l += other_half(l);
    const int64_t part = (((int64_t)blockIdx.y * p.B + b) * p.HK + hk) * p.rows + r0;
    bf16_t* const out = static_cast<bf16_t*>(const_cast<void*>(p.o.p)) + b * p.o.b + hk * p.G * p.o.h;
    if (row < p.rows) {
        if (p.splits > 1) {
            const int64_t at = part + row - r0;
            if (half == 0) p.part_m[2 * at] = m, p.part_m[2 * at + 1] = l;
            float* const to = p.part_o + at * p.D;
#pragma unroll
            for (int x = 0; x < DT; x++)
#pragma unroll
                for (int y = 0; y < 4; y++) {
                    const int c = 32 * x + 8 * y + 4 * half;
                    if (c < p.D) *reinterpret_cast<f32x4*>(to + c) = f32x4{o[x][4 * y], o[x][4 * y + 1], o[x][4 * y + 2], o[x][4 * y + 3]};
                }
        } else {
            if (p.lse != nullptr && half == 0) p.lse[((int64_t)b * p.T + t) * p.H + hk * p.G + g] = l == 0.f ? __builtin_inff() : m + log2f(l);
            store_transposed<DP>(out + t * p.o.t + g * p.o.h, p.D, half, o, l == 0.f ? 0.f : 1.f / l);
        }
    }
    if (!taken_out) return;
    add_taken_out<bf16_t>(p, b, hk, r0, WINDOW_ROWS, all, first_tile, last_tile, sink_tiles, 64, tile_at, part);
}

// The parts of a row joined: a workgroup a row.
template <typename T>
__global__ __launch_bounds__(256) void window_combine_kernel(const WindowParams p) {
    const int64_t at = blockIdx.x;
    float m, l;
    f32x4 o;
    int col;
    if (!join_row(p.part_o, p.part_m, (int64_t)p.B * p.HK * p.rows, at, p.splits, p.D, m, l, o, col)) return;
    const int64_t pair = at / p.rows;
    const int r = (int)(at - pair * p.rows), b = (int)(pair / p.HK), hk = (int)(pair - (int64_t)b * p.HK), t = r / p.G, g = r - t * p.G;
    if (p.lse != nullptr && col == 0) {
        const int64_t head = ((int64_t)b * p.T + t) * p.H + hk * p.G + g;
        if constexpr (sizeof(T) == 2) p.lse[head] = l == 0.f ? __builtin_inff() : m + log2f(l);
        else p.lse[2 * head] = l == 0.f ? 0.f : m, p.lse[2 * head + 1] = l == 0.f ? 0.f : 1.f / l;
    }
    store4<T>(static_cast<T*>(const_cast<void*>(p.o.p)) + b * p.o.b + t * p.o.t + (hk * p.G + g) * p.o.h + col, o * (l == 0.f ? 0.f : 1.f / l));
}

}  // namespace

int launch_window_fwd(const WindowParams& p, hipStream_t stream) {
    const dim3 grid((unsigned)((int64_t)p.B * p.HK * p.blocks), p.splits);
    if (p.D <= 64) hipLaunchKernelGGL((window_fwd_kernel<64>), grid, dim3(256), 0, stream, p);
    else if (p.D <= 128) hipLaunchKernelGGL((window_fwd_kernel<128>), grid, dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((window_fwd_kernel<256>), grid, dim3(256), 0, stream, p);
    if (const int e = (int)hipGetLastError(); e != 0) return e;
    return p.splits > 1 ? launch_window_combine(p, GDN_BF16, stream) : GDN_OK;
}

int launch_window_combine(const WindowParams& p, int dtype, hipStream_t stream) {
    const dim3 grid((unsigned)((int64_t)p.B * p.HK * p.rows));
    if (dtype == GDN_BF16) hipLaunchKernelGGL((window_combine_kernel<bf16_t>), grid, dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((window_combine_kernel<float>), grid, dim3(256), 0, stream, p);
    return (int)hipGetLastError();
}

}  // namespace gdn
