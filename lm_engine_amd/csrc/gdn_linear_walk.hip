// Linear attention with a decay for each head, bf16: a workgroup walks a segment of a sequence in chunks of 64 tokens.
//
// A wave holds the state of 32 columns of the value dim and all keys in accumulator registers, fp32, for the whole segment.  Per
// chunk (x, y, z: 64 rows each, in LDS; v_mfma_f32_32x32x16_bf16 throughout):
//     P^T = y x^T, masked and decayed          3 tiles of 32 x 32, each formed by one wave, handed round through LDS
//     out^T = (S^T x^T) w^{i + a} + z^T P^T    the state's registers are the left operand as they are, P^T and z^T fragments
//     S = w^n S + y^T (w^{n - a - j} z)        y^T and z^T by transposing LDS reads
// Rows of an accumulator tile are numbered so that registers 8 s .. 8 s + 7 of a lane are 8 consecutive rows (bits 2 and 3 of the row
// index swapped, by the order in which the left operand's rows are read): they are then a fragment of the next product, and outputs
// leave in 16-byte pieces.  The next chunk's rows are on their way in registers meanwhile.
//
// 32 columns to a wave, so that a fragment of x or y feeds as many columns as a product takes, and the four waves of 128 columns share the
// rows of x and y: 16 columns to a wave read LDS twice as often and were slower.  Bound by memory and LDS together: 32768 packed tokens,
// 16 heads of 128, 11 sequences: the states' pass 94 us (268 MB of rows, 2.9 TB/s, its three-part products beside them; with two parts the
// forward of one sequence takes 190 us instead of 202), their sums 18, the walk 168 (536 MB of rows, 3.2 TB/s); in the backward of 4 x 4096
// tokens 31 (two parts), 11 and 62 us.
#include <algorithm>

#include "gdn_launch.h"
#include "gdn_linear_tile.h"

namespace gdn {

namespace {

// Order of the instructions of a region that reads LDS fragments for matrix products: AHEAD reads, then PER reads to every STEP
// products.  Left alone, the scheduler waits for every read in front of its product.
template <int AHEAD, int STEPS, int STEP, int PER>
__device__ __forceinline__ void reads_ahead() {
    __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);
#pragma unroll
    for (int i = 0; i < STEPS; i++) {
        __builtin_amdgcn_sched_group_barrier(0x008, STEP, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, PER, 0);
    }
}

// Where the value dim has 64 columns or fewer two of the four waves have none, and two waves to a workgroup take as long: 4 x 4096 tokens
// of 16 heads of 64, the backward 157 us against 156.
constexpr int WALK_WAVES = WALK_COLUMNS / 32;

// What a walk is for, and in how many bf16 parts the decayed rows of z go into the state (the rows of y are exact).  Three hold all 24
// bits of an fp32 product: where the state is a result.  Two, 16 bits and more, where it only goes on into outputs, which round it to
// 8 as an operand: with one the state would carry as much error as that rounding adds.
enum class Walk {
    outputs,        // two parts; a segment of several, its state given
    outputs_state,  // three parts; the only segment, its state a result
    sums,           // as outputs, partial outputs in fp32 (LinearParams::sums)
    states,         // the segments' own states, two parts
    exact_states,   // ... three parts
};

template <int KD, Walk MODE>
__global__ __launch_bounds__(64 * WALK_WAVES, KD <= 128 ? 2 : 1) void linear_walk_kernel(const LinearParams p) {
    constexpr int NW = WALK_WAVES, NT = 64 * NW, VC = WALK_COLUMNS, KT = KD / 32;
    constexpr bool STATES_ONLY = MODE == Walk::states || MODE == Walk::exact_states, SUMS = MODE == Walk::sums;
    constexpr int PARTS = MODE == Walk::outputs_state || MODE == Walk::exact_states ? 3 : 2;
    __shared__ __align__(16) bf16_t sx[STATES_ONLY ? 8 : LC * KD];
    __shared__ __align__(16) bf16_t sy[LC * KD];
    __shared__ __align__(16) bf16_t sz[LC * VC];
    __shared__ __align__(16) bf16_t sp[STATES_ONLY ? 8 : 6 * 512];  // fragments of P^T
    __shared__ __align__(16) float sw[LC];                          // us w^{n - a - j}
    __shared__ __align__(16) bf16_t so[STATES_ONLY || SUMS ? 8 : LC * VC];  // the chunk's output, to leave in whole rows
    // ps w^{row - key} over a tile of P, in the order of its accumulator: on the diagonal, below it
    __shared__ __align__(16) f32x4 sdecay[STATES_ONLY ? 1 : 2][4][64];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l32 = lane & 31, half = lane >> 5;
    // blocks are dealt round the 8 XCDs: the blocks of one XCD get neighbouring places, so that those that read the same rows
    // (columns of the value dim, heads that share keys) meet in its L2
    const unsigned per_xcd = (gridDim.x + 7) / 8;
    const unsigned id = blockIdx.x % 8 * per_xcd + blockIdx.x / 8;
    const int slices = (p.V + VC - 1) / VC;
    if (id >= (unsigned)p.slots * p.H * slices) return;
    const int slice = id % slices, h = id / slices % p.H, slot = id / slices / p.H;
    const int c0 = slice * VC, columns = min(VC, p.V - c0);

    if constexpr (!STATES_ONLY)
        if (p.zero && p.cu != nullptr) linear_zero_gaps<bf16_t>(p, slot, h, c0, columns, tid, NT);
    LinearSegment sg;
    if (!linear_find(p, slot, sg, lane)) return;
    const int segments = linear_segments(sg.len, p.seg);
    const bool last = sg.s == segments - 1;
    if (MODE == Walk::states && last) return;  // nothing starts from it
    const int walked = sg.s * p.seg, total = min(p.seg, sg.len - walked);
    const int64_t token = p.reverse ? (int64_t)sg.t0 + sg.len - 1 - walked : (int64_t)sg.t0 + walked;  // the first of the walk
    const float g = linear_log2(p.g, h);
    const int a = p.a;

    Stream<KD, NT> ys(p.y, sg.b, h, token, p.reverse, 0, p.K, tid);
    Stream<VC, NT> zs(p.z, sg.b, h, token, p.reverse, c0, columns, tid);
    Stream<KD, NT> xs(STATES_ONLY ? p.y : p.x, sg.b, h, token, p.reverse, 0, p.K, tid);
    bf16x8 ry[Stream<KD, NT>::ITERS], rz[Stream<VC, NT>::ITERS], rx[STATES_ONLY ? 1 : Stream<KD, NT>::ITERS];
    const bool whole_rows = p.K == KD && columns == VC;
    auto fetch = [&](int left) __attribute__((always_inline)) {  // the next chunk's rows, on their way into registers
        const bool all = left >= LC && whole_rows;
        ys.fetch(ry, left, all), zs.fetch(rz, left, all);
        if constexpr (!STATES_ONLY) xs.fetch(rx, left, all);
    };
    if (total > 0) fetch(total);  // (a segment without tokens has no row to read)

    // the state: keys 32 kt + 16 (r / 8) + 8 half + r % 8 in register r of S[kt], column c0 + 32 wave + swap(l32)
    const int64_t chain = (int64_t)sg.n * p.H + h, cells = p.cells;
    const int my_v = c0 + 32 * wave + slice_col(l32);
    f32x16 S[KT];
    auto for_cells = [&](auto&& f) __attribute__((always_inline)) {
        if (my_v >= p.V) return;
#pragma unroll
        for (int kt = 0; kt < KT; kt++)
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const int key = 32 * kt + 16 * (r >> 3) + 8 * half + (r & 7);
                if (key < p.K) f(kt, r, (int64_t)key * p.state_k + (int64_t)my_v * p.state_v);
            }
    };
#pragma unroll
    for (int kt = 0; kt < KT; kt++) S[kt] = f32x16{};
    // in the registers' own order a state is 4 keys to a lane and 1 KiB to a wave at a time
    const int64_t own = ((int64_t)slot * p.H + h) * p.local_cells + (int64_t)(slice * NW + wave) * KT * 1024 + 4 * lane;
    if (!STATES_ONLY && sg.s > 0) {
        if (p.local_keys == 0) {
            const float* const from = p.local + ((int64_t)slot * p.H + h) * p.local_cells;
            for_cells([&](int kt, int r, int64_t at) __attribute__((always_inline)) { S[kt][r] = from[at]; });
        } else if (p.local_swapped) {
            const float* const from = p.local + ((int64_t)slot * p.H + h) * p.local_cells;
#pragma unroll
            for (int kt = 0; kt < KT; kt++)
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int key = 32 * kt + 16 * (r >> 3) + 8 * half + (r & 7);
                    if (key < p.K && my_v < p.V) S[kt][r] = from[linear_fragment(p.local_keys, my_v, key + p.local_first)];
                }
        } else {
#pragma unroll
            for (int kt = 0; kt < KT; kt++)
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const f32x4 x = *reinterpret_cast<const f32x4*>(p.local + own + (4 * kt + q) * 256);
#pragma unroll
                    for (int r = 0; r < 4; r++) S[kt][4 * q + r] = x[r];
                }
        }
    } else if (!STATES_ONLY && p.init != nullptr) {
        const float* const from = p.init + chain * cells;
        for_cells([&](int kt, int r, int64_t at) __attribute__((always_inline)) { S[kt][r] = from[at]; });
    }

    constexpr int TILES = 3;  // of P: (key tile, row tile) (0, 0), (0, 1), (1, 1)
    float row_weight[2];
    if constexpr (!STATES_ONLY) {
        for (int i = wave; i < 8; i += NW) {
            f32x4 w;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int distance = 32 * (i >> 2) + l32 - (16 * (i >> 1 & 1) + 8 * half + 4 * (i & 1) + r);
                w[r] = distance >= 0 ? p.ps * linear_power(g, distance) : 0.f;
            }
            sdecay[i >> 2][i & 3][lane] = w;
        }
#pragma unroll
        for (int i = 0; i < 2; i++) row_weight[i] = p.os * linear_power(g, 32 * i + l32 + a);
    }
    if (tid < LC) sw[tid] = p.us * linear_power(g, LC - a - tid);
    // A chunk's factor is one number: its rounding, up to 2^-25, comes back with every chunk of the segment, 1e-6 of the state after 32.  (In two
    // parts, as a segment's: 1 x 65536 tokens 1347 us instead of 1285, the decay's gradient a third longer.)
    const float whole = linear_power(g, LC);
    TileLane<KD> tile(lane);
    TileLane<VC> ztile(lane);

    // outputs, addressed as the streams are
    using Out = Stream<VC, NT>;
    const LinearRole out_role = {p.out, p.out_stride_b, p.out_stride_t, p.out_stride_h, 1};
    Out os(out_role, sg.b, h, token, p.reverse, c0, columns, tid);
    auto leave = [&](int rows) __attribute__((always_inline)) {  // the output in LDS, rows as they lie in memory
        char* const to = const_cast<char*>(os.base);
#pragma unroll
        for (int i = 0; i < Out::ITERS; i++) {
            const int r = os.r0 + i * Out::STEP;
            if (os.there(i, rows))
                __builtin_nontemporal_store(*reinterpret_cast<const bf16x8*>(so + r * VC + ((tid % Out::GRANULES ^ tile_key<VC>(r)) << 3)), reinterpret_cast<bf16x8*>(to + i * os.step_bytes + os.offset));
        }
        os.base += os.chunk_bytes;
    };
    const int col = c0 + 32 * wave + 8 * half;
    float* const sums = SUMS ? p.sums + ((int64_t)sg.b * p.T + token) * p.H * p.V + (int64_t)h * p.V : nullptr;
    const int64_t sums_row = (p.reverse ? -1 : 1) * (int64_t)p.H * p.V;

    const int chunks = (total + LC - 1) / LC;
    for (int c = 0; c < chunks; c++) {
        const int rows = min(LC, total - c * LC);
        __syncthreads();  // the tiles of the chunk before are read, its output is in LDS
        if (rows < LC && tid < LC) sw[tid] = p.us * linear_power(g, max(rows - a - tid, 0));
        if (rows == LC && whole_rows) {
            ys.stage(sy, ry, rows, true), zs.stage(sz, rz, rows, true);
            if constexpr (!STATES_ONLY) xs.stage(sx, rx, rows, true);
        } else {
            ys.stage(sy, ry, rows, false), zs.stage(sz, rz, rows, false);
            if constexpr (!STATES_ONLY) xs.stage(sx, rx, rows, false);
        }
        // (behind the wait for the rows, which stores in front of it would be part of)
        if constexpr (!STATES_ONLY && !SUMS)
            if (c > 0) leave(LC);
        __syncthreads();
        if (c + 1 < chunks) fetch(total - (c + 1) * LC);
        tile.recompute(), ztile.recompute();

        if constexpr (!STATES_ONLY) {
            for (int t = wave; t < TILES; t += NW) {
                const int jt = t == 2, it = t >= 1;
                const bf16_t *const yt = sy + 32 * jt * KD, *const xt = sx + 32 * it * KD;
                f32x16 acc = {};
#pragma unroll
                for (int s = 0; s < KD / 16; s++) acc = mfma32_bf16(tile.swapped_fragment(yt, 0, s), tile.fragment(xt, 0, s), acc);
                reads_ahead<8, KD / 16, 1, 2>();
                // selected, not multiplied away: a row before the key takes nothing of it, whatever its product is
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const f32x4 w = sdecay[t == 1][q][lane];
#pragma unroll
                    for (int r = 4 * q; r < 4 * q + 4; r++) acc[r] = t != 1 && l32 < 16 * (r >> 3) + 8 * half + (r & 7) ? 0.f : acc[r] * w[r & 3];
                }
                *reinterpret_cast<bf16x8*>(sp + (2 * t + 0) * 512 + lane * 8) = pack8_16(acc, 0, 1.f);
                *reinterpret_cast<bf16x8*>(sp + (2 * t + 1) * 512 + lane * 8) = pack8_16(acc, 1, 1.f);
            }
            __builtin_amdgcn_sched_barrier(0);
            f32x16 O[2] = {};
#pragma unroll
            for (int s = 0; s < KD / 16; s++) {
                const bf16x8 sf = pack8_16(S[s >> 1], s & 1, 1.f);  // the state as an operand: its one rounding to bf16 for the output
#pragma unroll
                for (int i = 0; i < 2; i++) O[i] = mfma32_bf16(sf, tile.fragment(sx, 32 * i, s), O[i]);
            }
            reads_ahead<8, KD / 16, 2, 2>();
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int r = 0; r < 16; r++) O[i][r] *= row_weight[i];
            __syncthreads();  // P is there
            bf16x8 zf[4];
#pragma unroll
            for (int s = 0; s < 4; s++) zf[s] = ztile.transposed(sz, s, wave);
#pragma unroll
            for (int t = 0; t < TILES; t++)
#pragma unroll
                for (int s = 0; s < 2; s++)
                    O[t >= 1] = mfma32_bf16(zf[2 * (t == 2) + s], *reinterpret_cast<const bf16x8*>(sp + (2 * t + s) * 512 + lane * 8), O[t >= 1]);
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int row = 32 * i + l32;
#pragma unroll
                for (int s = 0; s < 2; s++) {
                    if constexpr (SUMS) {
                        if (row >= rows || col + 16 * s >= p.V) continue;
                        f32x4* const at = reinterpret_cast<f32x4*>(sums + (int64_t)(c * LC + row) * sums_row + col + 16 * s);
#pragma unroll
                        for (int e = 0; e < 8; e++)
                            if (p.sums_in) O[i][8 * s + e] += at[e >> 2][e & 3];
                        if (p.sums_out) {
#pragma unroll
                            for (int e = 0; e < 2; e++) at[e] = f32x4{O[i][8 * s + 4 * e], O[i][8 * s + 4 * e + 1], O[i][8 * s + 4 * e + 2], O[i][8 * s + 4 * e + 3]};
                            continue;
                        }
                        const int64_t token_row = token + (p.reverse ? -1 : 1) * (int64_t)(c * LC + row);
                        bf16_t* const out = static_cast<bf16_t*>(p.out) + sg.b * p.out_stride_b + h * p.out_stride_h + token_row * p.out_stride_t;
                        *reinterpret_cast<bf16x8*>(out + col + 16 * s) = pack8_16(O[i], s, 1.f);
                    } else {
                        *reinterpret_cast<bf16x8*>(so + row * VC + (((4 * wave + 2 * s + half) ^ tile_key<VC>(row)) << 3)) = pack8_16(O[i], s, 1.f);
                    }
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        bf16x8 part[4][PARTS];
#pragma unroll
        for (int s = 0; s < 4; s++) {
            const bf16x8 z = ztile.transposed(sz, s, wave);
            const float* const weights = sw + 16 * s + 8 * half;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                float x = (float)z[e] * weights[e];
#pragma unroll
                for (int u = 0; u < PARTS; u++) part[s][u][e] = (bf16_t)x, x -= (float)part[s][u][e];
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        const float shrink = rows < LC ? linear_power(g, rows) : whole;
#pragma unroll
        for (int kt = 0; kt < KT; kt++)
#pragma unroll
            for (int r = 0; r < 16; r++) S[kt][r] *= shrink;
#pragma unroll
        for (int kt = 0; kt < KT; kt++)
#pragma unroll
            for (int s = 0; s < 4; s++) {
                const bf16x8 yt = tile.transposed(sy, s, kt);
#pragma unroll
                for (int u = 0; u < PARTS; u++) S[kt] = mfma32_bf16(yt, part[s][u], S[kt]);
            }
        reads_ahead<8, 4 * KT, PARTS, 2>();
        __builtin_amdgcn_sched_barrier(0);
    }

    if constexpr (!STATES_ONLY && !SUMS) {
        if (chunks > 0) {
            __syncthreads();
            leave(total - (chunks - 1) * LC);
        }
    }
    if constexpr (STATES_ONLY) {
#pragma unroll
        for (int kt = 0; kt < KT; kt++)
#pragma unroll
            for (int q = 0; q < 4; q++) *reinterpret_cast<f32x4*>(p.local + own + (4 * kt + q) * 256) = f32x4{S[kt][4 * q], S[kt][4 * q + 1], S[kt][4 * q + 2], S[kt][4 * q + 3]};
    } else if (MODE == Walk::outputs_state && p.fin != nullptr) {
        float* const to = p.fin + chain * cells;
        for_cells([&](int kt, int r, int64_t at) __attribute__((always_inline)) { to[at] = S[kt][r]; });
    }
}

// From the segments' own states (slots 0 .. of a sequence) to what every segment but the first starts from, and to what the sequence ends
// with where that is a result (then the last segment's own state is there as well).  A thread has 4 cells of a (sequence, head); the
// states lie contiguous, and those of a sequence H states apart.
__global__ __launch_bounds__(256) void linear_combine_kernel(const LinearParams p) {
    const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    const int h = blockIdx.y;
    // the 4 cells in init and fin: a step of `apart`, `there` of them (in the registers' order the last keys and columns are padding)
    int64_t cell = at, apart = 1;
    bool there = at < p.cells;
    if (p.local_keys != 0) {
        const int lane = at / 4 % 64, q = at / 256 % 4, kt = at / 1024 % (p.local_keys / 32), v = (int)(at / 1024 / (p.local_keys / 32)) * 32 + slice_col(lane & 31);
        const int key = 32 * kt + 16 * (q >> 1) + 8 * (lane >> 5) + 4 * (q & 1);  // (a multiple of 4, as K is of 8)
        there = key < p.K && v < p.V;
        cell = (int64_t)key * p.state_k + (int64_t)v * p.state_v, apart = p.state_k;
    }
    for (int n = blockIdx.z; n < p.N; n += gridDim.z) {
        int b, t0, len;
        linear_bounds(p, n, b, t0, len);
        const int segments = linear_segments(len, p.seg);
        if (segments == 1 && p.fin == nullptr) continue;
        int slot0 = n * p.nseg;
        if (p.nseg == 0) {
            LinearSegment none;
            linear_find_packed(p, -1, none, threadIdx.x & 63, n, &slot0);
        }
        if (slot0 + segments > p.slots || at >= p.local_cells) continue;
        const float g = p.g == nullptr ? 0.f : p.g[h];
        const LinearFactor whole = linear_factor(g, p.seg);
        float* local = p.local + ((int64_t)slot0 * p.H + h) * p.local_cells + at;
        const int64_t next = (int64_t)p.H * p.local_cells, chain = ((int64_t)n * p.H + h) * p.cells + cell;
        f32x4 carry = {0.f, 0.f, 0.f, 0.f};
        if (p.init != nullptr && there) {
#pragma unroll
            for (int e = 0; e < 4; e++) carry[e] = p.init[chain + e * apart];
        }
        f32x4 own = *reinterpret_cast<const f32x4*>(local);
        for (int s = 1; s < segments; s++) {
            f32x4 following = {0.f, 0.f, 0.f, 0.f};
            if (s + 1 < segments || p.fin != nullptr) following = *reinterpret_cast<const f32x4*>(local + s * next);
            carry = whole(carry) + own;
            *reinterpret_cast<f32x4*>(local + s * next) = carry;
            own = following;
        }
        if (p.fin != nullptr && there) {  // behind the last segment, whose tokens are `rest`
            carry = linear_factor(g, len - (segments - 1) * p.seg)(carry) + own;
#pragma unroll
            for (int e = 0; e < 4; e++) p.fin[chain + e * apart] = carry[e];
        }
    }
}

template <int KD>
int launch(const LinearParams& p, bool states_only, hipStream_t stream) {
    const int64_t blocks = (int64_t)p.slots * p.H * ((p.V + WALK_COLUMNS - 1) / WALK_COLUMNS);
    if (blocks > 0xfffff000ll / (64 * WALK_WAVES)) return GDN_ERR_UNSUPPORTED;  // (a launch holds at most 2^32 - 1 threads)
    const dim3 grid((unsigned)((blocks + 7) / 8 * 8)), threads(64 * WALK_WAVES);
    if (states_only && p.fin != nullptr) hipLaunchKernelGGL((linear_walk_kernel<KD, Walk::exact_states>), grid, threads, 0, stream, p);
    else if (states_only) hipLaunchKernelGGL((linear_walk_kernel<KD, Walk::states>), grid, threads, 0, stream, p);
    else if (p.sums != nullptr) hipLaunchKernelGGL((linear_walk_kernel<KD, Walk::sums>), grid, threads, 0, stream, p);
    else if (p.fin != nullptr) hipLaunchKernelGGL((linear_walk_kernel<KD, Walk::outputs_state>), grid, threads, 0, stream, p);
    else hipLaunchKernelGGL((linear_walk_kernel<KD, Walk::outputs>), grid, threads, 0, stream, p);
    return (int)hipGetLastError();
}

}  // namespace

int linear_walk_keys(int K) { return K <= 64 ? 64 : K <= 128 ? 128 : 256; }

int launch_linear_walk(const LinearParams& p, bool states_only, hipStream_t stream) {
    if (p.K <= 64) return launch<64>(p, states_only, stream);
    if (p.K <= 128) return launch<128>(p, states_only, stream);
    return launch<256>(p, states_only, stream);
}

int launch_linear_combine(const LinearParams& p, hipStream_t stream) {
    hipLaunchKernelGGL(linear_combine_kernel, dim3((unsigned)((p.local_cells + 1023) / 1024), (unsigned)p.H, (unsigned)std::min(p.N, 32768)), dim3(256), 0, stream, p);
    return (int)hipGetLastError();
}

}  // namespace gdn
