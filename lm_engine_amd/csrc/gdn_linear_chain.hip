// Linear attention with a decay for each head, forward, bf16, up to 128 keys: a workgroup of twelve waves walks a whole sequence in
// chunks of 64 tokens, for 32 columns of the value dim.
//
// The state's columns are independent of each other, so a (sequence, head) is split over its columns, and no state goes through
// memory: q, k, v are read once and the output is written once (the workgroups of one pair are neighbours on an XCD and meet in its L2
// for the rows of x and y).  What a chunk then costs is the time from one state to the next, so the work is dealt out to three groups
// of four waves that meet at one barrier a chunk, in interval c:
//     P waves    P_c^T = y x^T, decayed, masked: the 10 tiles of 16 x 16 that hold anything        (v_mfma_f32_16x16x32_bf16)
//     S waves    S_{c+1} = w^n S_c + y^T (w^{n - a - j} z): tiles of 32 keys x 32 columns          (v_mfma_f32_32x32x16_bf16)
//     O waves    out_{c-1}^T = ... + z^T P_{c-1}^T, stored; then out_c^T = (S_c^T x^T) w^{i + a}: 16 rows each
// P, and the state as bf16 fragments, go round through LDS.  Rows are on their way in registers two chunks ahead, in LDS one chunk
// ahead; the P waves bring in x and z (and its decayed rows, in two or three bf16 parts), the S waves y.  The O waves load nothing: the
// compiler's wait for rows would be one for their stores.
//
// Measured at 4 sequences of 4096 tokens, 16 heads, K = V = 128, which is one workgroup to a compute unit: 77 us, with a final state
// 80 to 91 (two registers spilled), 1.25 us a chunk, of which some 0.9 us are the S waves' own work and the rest the barrier and the other
// groups.  Their eight or twelve products are no more than 0.11 to 0.16 us of that (32 cycles of the matrix unit each); what takes the time is
// that one thing waits for the other: operand reads that begin behind the barrier, the products, the state's rounding and its way to LDS.
// 268 MB in and out are 51 us at a large copy's rate.  With the tiles of P on the diagonal formed by the O waves, 83; with 64 columns to a
// workgroup registers spill.
#include <algorithm>

#include "gdn_launch.h"
#include "gdn_linear_tile.h"

namespace gdn {

namespace {

// Where a lane of v_mfma_f32_16x16x32_bf16 reads a tile of LD columns; as TileLane.
template <int LD>
struct TileLane16 {
    static constexpr int PERIOD = TileLane<LD>::PERIOD;
    int row, pair;

    __device__ __forceinline__ TileLane16(int lane) {
        const int l16 = lane & 15, g4 = lane >> 4, r = 4 * g4 + (l16 >> 2);
        row = l16 * LD + ((g4 ^ tile_key<LD>(l16)) << 3);
        pair = r * LD + (((l16 & 3) ^ tile_key<LD>(r)) << 3);
    }
    // 8 columns 32 b + 8 g4 .. of row l16
    __device__ __forceinline__ bf16x8 fragment(const bf16_t* tile, int b) const {
        return *reinterpret_cast<const bf16x8*>(tile + (row ^ (32 * b % PERIOD)) + 32 * b / PERIOD * PERIOD);
    }
    // lane i of a 16-lane group: rows row0 + 4 g4 .. + 3 and row0 + 16 + 4 g4 .. + 3 of column 32 b + 4 u + 8 (i / 4) + i % 4
    __device__ __forceinline__ bf16x8 transposed(const bf16_t* tile, int row0, int b, int u) const {
        const bf16_t* const p = tile + (pair ^ (32 * b % PERIOD)) + row0 * LD + 32 * b / PERIOD * PERIOD + 4 * u;
        return __builtin_shufflevector(TileLane<LD>::read(p), TileLane<LD>::read(p + 16 * LD), 0, 1, 2, 3, 4, 5, 6, 7);
    }
};

// rows row0 + 8 half .. + 7 of column 32 b + 4 (lane / 16 % 2) + 8 (lane % 16 / 4) + lane % 4: the state's columns, see `column`
template <int LD>
struct TileColumns {
    static constexpr int PERIOD = TileLane<LD>::PERIOD;
    int pair;
    __device__ __forceinline__ TileColumns(int lane) {
        const int r = 8 * (lane >> 5) + ((lane & 15) >> 2);
        pair = r * LD + (((lane & 3) ^ tile_key<LD>(r)) << 3) + 4 * ((lane >> 4) & 1);
    }
    __device__ __forceinline__ bf16x8 transposed(const bf16_t* tile, int row0, int b) const {
        const bf16_t* const p = tile + row0 * LD + 32 * b / PERIOD * PERIOD;
        const int at = pair ^ (32 * b % PERIOD);
        // 4 rows on, the key's lowest bit is the other
        return __builtin_shufflevector(TileLane<LD>::read(p + at), TileLane<LD>::read(p + (at ^ 8) + 4 * LD), 0, 1, 2, 3, 4, 5, 6, 7);
    }
};

template <int KD>
struct ChainShape {
    static constexpr int THREADS = 768, GROUP = 256, VC = 32, KT = KD / 32;
    static constexpr int ZLD = 128;  // z, then the parts of its decayed rows
    static constexpr int XY = LC * KD, Z = LC * ZLD, SF = KD * VC, PF = 10 * 256;  // elements
    static constexpr int LDS_BYTES = 2 * 2 * (2 * XY + Z + SF + PF);
};

template <int KD, bool EXACT>
__global__ __launch_bounds__(768) void linear_chain_kernel(const LinearParams p) {
    using Shape = ChainShape<KD>;
    constexpr int GROUP = Shape::GROUP, VC = Shape::VC, ZLD = Shape::ZLD, KT = Shape::KT;
    constexpr int PARTS = EXACT ? 3 : 2;  // of a decayed row of z, as in linear_walk_kernel
    extern __shared__ __align__(16) bf16_t lds[];  // everything twice
    bf16_t* const tx = lds;
    bf16_t* const ty = tx + 2 * Shape::XY;
    bf16_t* const tz = ty + 2 * Shape::XY;
    bf16_t* const ts = tz + 2 * Shape::Z;   // [KT][4 octets of keys][32 columns][8 keys]
    bf16_t* const tp = ts + 2 * Shape::SF;  // tiles of P^T, rows 16 it, keys 16 jt, at it (it + 1) / 2 + jt

    const int tid = threadIdx.x % GROUP, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int group = wave >> 2, w4 = wave & 3, l32 = lane & 31, half = lane >> 5, l16 = lane & 15, g4 = lane >> 4;
    const unsigned per_xcd = (gridDim.x + 7) / 8;  // neighbouring places to the blocks of one XCD
    const unsigned id = blockIdx.x % 8 * per_xcd + blockIdx.x / 8;
    const int slices = (p.V + VC - 1) / VC;
    if (id >= (unsigned)p.slots * p.H * slices) return;
    const int slice = id % slices, h = id / slices % p.H, slot = id / slices / p.H;
    const int c0 = slice * VC, columns = min(VC, p.V - c0);
    if (p.zero && p.cu != nullptr) linear_zero_gaps<bf16_t>(p, slot, h, c0, columns, threadIdx.x, Shape::THREADS);
    LinearSegment sg;
    if (!linear_find(p, slot, sg, lane)) return;  // (one segment to a sequence)
    const int total = sg.len;
    const int64_t token = sg.t0;
    const float g = linear_log2(p.g, h);
    const int a = p.a, chunks = (total + LC - 1) / LC;
    const int64_t chain = (int64_t)sg.n * p.H + h;

    // Chunk c computed in interval c, staged in LDS in interval c - 1, fetched in interval c - 3 (or in front): registers of two chunks.
    // Every interval fetches, the last ones the last chunk again: the wait for rows counts what was asked for behind them, and has to
    // be the same however it was come to.
    using Even = std::integral_constant<int, 0>;
    using Odd = std::integral_constant<int, 1>;
    auto run = [&](auto&& fetch, auto&& stage, auto&& begin, auto&& interval) __attribute__((always_inline)) {
        begin();
        if (chunks == 0) return;
        fetch(0, Even{});
        fetch(min(1, chunks - 1), Odd{});
        stage(0, Even{}, 0);
        fetch(min(2, chunks - 1), Even{});
        __syncthreads();
        int c = 0;
        for (; c + 1 < chunks; c += 2) {
            stage(c + 1, Odd{}, 1);
            fetch(min(c + 3, chunks - 1), Odd{});
            interval(c, Even{});
            __syncthreads();
            stage(min(c + 2, chunks - 1), Even{}, 0);
            fetch(min(c + 4, chunks - 1), Even{});
            interval(c + 1, Odd{});
            __syncthreads();
        }
        if (c < chunks) {
            interval(c, Even{});
            __syncthreads();
        }
    };

    if (group == 0) {
        Stream<KD, GROUP> xs(p.x, sg.b, h, token, 0, 0, p.K, tid);
        bf16x8 rx[2][Stream<KD, GROUP>::ITERS];
        const bool whole_rows = p.K == KD;
        const TileLane16<KD> tile(lane);
        Stream<VC, GROUP> zs(p.z, sg.b, h, token, 0, c0, columns, tid);
        constexpr int ZI = Stream<VC, GROUP>::ITERS;
        bf16x8 rz[2][ZI];
        const bool all_columns = columns == VC;
        float z_weight[ZI];
#pragma unroll
        for (int i = 0; i < ZI; i++) z_weight[i] = p.us * linear_power(g, LC - a - (zs.r0 + i * Stream<VC, GROUP>::STEP));
        // row tile 3: keys 0, 1, 2 | row tile 2: keys 0, 1, 2 | row tile 1: keys 0, 1 | row tile 3: keys 3, and row tile 0: keys 0
        const int it = w4 == 0 ? 3 : w4 == 1 ? 2 : w4 == 2 ? 1 : 3, jt = w4 == 3 ? 3 : 0;
        const int last_it = w4 == 3 ? 0 : it, last_jt = w4 == 3 ? 0 : it < 2 ? 1 : 2;  // the one that is done last
        auto decayed = [&](int tiles, int r) __attribute__((always_inline)) {  // row - key: 16 tiles + ...
            const int d = 16 * tiles + l16 - 4 * g4 - r;
            return d < 0 ? 0.f : p.ps * linear_power(g, d);
        };
        f32x4 decay[3];
#pragma unroll
        for (int r = 0; r < 4; r++) decay[0][r] = decayed(it - jt, r), decay[1][r] = decayed(it - 1, r), decay[2][r] = decayed(last_it - last_jt, r);
        run([&](int c, auto set) __attribute__((always_inline)) {
                constexpr int R = decltype(set)::value;
                const int rows = total - c * LC;
                xs.fetch_chunk(c, rx[R], rows, rows >= LC && whole_rows);
                zs.fetch_chunk(c, rz[R], rows, rows >= LC && all_columns);
            },
            [&](int c, auto set, int buf) __attribute__((always_inline)) {
                constexpr int R = decltype(set)::value;
                const int rows = total - c * LC;
                if (rows >= LC && whole_rows) xs.stage(tx + buf * Shape::XY, rx[R], rows, true);
                else xs.stage(tx + buf * Shape::XY, rx[R], rows, false);
#pragma unroll
                for (int i = 0; i < ZI; i++) {
                    const int r = zs.r0 + i * Stream<VC, GROUP>::STEP;
                    bf16x8 x = rz[R][i], part[PARTS];
                    float w = z_weight[i];
                    if (rows < LC || !all_columns) {
                        const bf16x8 zero = {};
                        if (!zs.there(i, rows)) x = zero;
                        w = p.us * linear_power(g, max(min(rows, LC) - a - r, 0));
                    }
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        float z = (float)x[e] * w;
#pragma unroll
                        for (int u = 0; u < PARTS; u++) part[u][e] = (bf16_t)z, z -= (float)part[u][e];
                    }
                    bf16_t* const to = tz + buf * Shape::Z + r * ZLD;
                    const int g = tid % Stream<VC, GROUP>::GRANULES, key = tile_key<ZLD>(r);
                    *reinterpret_cast<bf16x8*>(to + ((g ^ key) << 3)) = x;
#pragma unroll
                    for (int u = 0; u < PARTS; u++) *reinterpret_cast<bf16x8*>(to + (((4 + 4 * u + g) ^ key) << 3)) = part[u];
                }
            },
            [] {},
            [&](int, auto buf) __attribute__((always_inline)) {
                constexpr int B = decltype(buf)::value;
                const bf16_t *const x = tx + B * Shape::XY, *const y = ty + B * Shape::XY;
                bf16x8 xf[KT], yf[2][KT];
#pragma unroll
                for (int k = 0; k < KT; k++) xf[k] = tile.fragment(x + 16 * it * KD, k), yf[0][k] = tile.fragment(y + 16 * jt * KD, k);
#pragma unroll
                for (int k = 0; k < KT; k++) yf[1][k] = tile.fragment(y + 16 * (w4 < 2 ? 1 : last_jt) * KD, k);
                auto form = [&](const bf16x8* ys, int t, int i, int j) __attribute__((always_inline)) {
                    f32x4 P = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int k = 0; k < KT; k++) P = mfma_bf16(ys[k], xf[k], P);
                    // selected, not multiplied away: a row before the key takes nothing of it, whatever its product is
#pragma unroll
                    for (int r = 0; r < 4; r++) P[r] = i == j && 4 * g4 + r > l16 ? 0.f : P[r] * decay[t][r];
                    store4<bf16_t>(tp + B * Shape::PF + (i * (i + 1) / 2 + j) * 256 + lane * 4, P);
                };
                form(yf[0], 0, it, jt);
                if (w4 == 3) {
#pragma unroll
                    for (int k = 0; k < KT; k++) xf[k] = tile.fragment(x, k);
                }
                if (w4 < 2) {
#pragma unroll
                    for (int k = 0; k < KT; k++) yf[0][k] = tile.fragment(y + 16 * last_jt * KD, k);
                    form(yf[1], 1, it, 1);
                    form(yf[0], 2, last_it, last_jt);
                } else {
                    form(yf[1], 2, last_it, last_jt);
                }
            });
        return;
    }

    if (group == 1) {
        Stream<KD, GROUP> ys(p.y, sg.b, h, token, 0, 0, p.K, tid);
        bf16x8 ry[2][Stream<KD, GROUP>::ITERS];
        const bool whole_rows = p.K == KD;
        const TileLane<KD> tile(lane);
        const TileColumns<ZLD> ztile(lane);
        const float whole = linear_power(g, LC);
        const int column = 8 * (l16 >> 2) + 4 * ((lane >> 4) & 1) + (lane & 3);  // of this lane, in 32
        // keys 32 w4 + 16 (r / 8) + 8 half + r % 8 in register r (64 keys: two of the waves have nothing to do)
        f32x16 S = {};
        const bool mine = w4 < KT;
        auto for_cells = [&](auto&& f) __attribute__((always_inline)) {
            const int v = c0 + column;
            if (!mine || v >= p.V) return;
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const int key = 32 * w4 + 16 * (r >> 3) + 8 * half + (r & 7);
                if (key < p.K) f(r, (int64_t)key * p.state_k + (int64_t)v * p.state_v);
            }
        };
        auto publish = [&](int buf) __attribute__((always_inline)) {  // the state as an operand: its one rounding to bf16 for the output
            if (!mine) return;
#pragma unroll
            for (int s = 0; s < 2; s++)
                *reinterpret_cast<bf16x8*>(ts + buf * Shape::SF + ((w4 * 4 + 2 * s + half) * 32 + l32) * 8) = pack8_16(S, s, 1.f);
        };
        run([&](int c, auto set) __attribute__((always_inline)) {
                const int rows = total - c * LC;
                ys.fetch_chunk(c, ry[decltype(set)::value], rows, rows >= LC && whole_rows);
            },
            [&](int c, auto set, int buf) __attribute__((always_inline)) {
                const int rows = total - c * LC;
                if (rows >= LC && whole_rows) ys.stage(ty + buf * Shape::XY, ry[decltype(set)::value], rows, true);
                else ys.stage(ty + buf * Shape::XY, ry[decltype(set)::value], rows, false);
            },
            [&]() __attribute__((always_inline)) {
                if (p.init != nullptr) {
                    const float* const from = p.init + chain * p.cells;
                    for_cells([&](int r, int64_t at) __attribute__((always_inline)) { S[r] = from[at]; });
                }
                publish(0);
            },
            [&](int c, auto buf) __attribute__((always_inline)) {
                constexpr int B = decltype(buf)::value;
                const int rows = total - c * LC;
                const bf16_t *const y = ty + B * Shape::XY, *const z = tz + B * Shape::Z;
                const float shrink = rows < LC ? linear_power(g, rows) : whole;
                if (mine) {
                    bf16x8 yt[4], zt[4];
#pragma unroll
                    for (int s = 0; s < 4; s++) yt[s] = tile.transposed(y, s, w4), zt[s] = ztile.transposed(z, 16 * s, 1);
                    f32x16 low = {};
#pragma unroll
                    for (int r = 0; r < 16; r++) S[r] *= shrink;
#pragma unroll
                    for (int u = 0; u < PARTS; u++)
#pragma unroll
                        for (int s = 0; s < 4; s++) {
                            f32x16& to = u == 0 ? S : low;
                            to = mfma32_bf16(yt[s], zt[s], to);
                            if (u + 1 < PARTS) zt[s] = ztile.transposed(z, 16 * s, u + 2);
                        }
                    // all reads of the first products first, then theirs and the next part's reads: left alone, the scheduler waits for
                    // every read in front of its product
                    __builtin_amdgcn_sched_group_barrier(0x100, 16, 0);
#pragma unroll
                    for (int i = 0; i < 4 * PARTS; i++) {
                        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                        if (i < 4 * PARTS - 4) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
                    }
#pragma unroll
                    for (int r = 0; r < 16; r++) S[r] += low[r];
                }
                publish(1 - B);
            });
        if (p.fin != nullptr) {
            float* const to = p.fin + chain * p.cells;
            for_cells([&](int r, int64_t at) __attribute__((always_inline)) { to[at] = S[r]; });
        }
        return;
    }

    const TileLane16<KD> tile(lane);
    const TileLane16<ZLD> ztile(lane);
    const int row = 16 * w4 + l16;  // this lane's row of a chunk
    const float row_weight = p.os * linear_power(g, row + a);
    char* out = static_cast<char*>(p.out) + 2 * (sg.b * p.out_stride_b + h * p.out_stride_h) + token * p.out_stride_t * 2;
    const int64_t out_row = 2 * p.out_stride_t;
    const int col = c0 + 8 * g4;
    f32x4 O[2];
    bf16x8 zf[2][2];
    const int first = w4 * (w4 + 1) / 2;  // of this row tile's tiles of P^T; those behind the diagonal are none
    bf16x4 part[4];
    auto read_parts = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < 4; t++) part[t] = *reinterpret_cast<const bf16x4*>(tp + buf * Shape::PF + (first + min(t, w4)) * 256 + lane * 4);
    };
    // out_c is complete: add what lies inside the chunk, store
    auto finish = [&](int c) __attribute__((always_inline)) {
        const bf16x4 zero = {};
#pragma unroll
        for (int t = 1; t < 4; t++) part[t] = t > w4 ? zero : part[t];
        const bf16x8 P[2] = {__builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7), __builtin_shufflevector(part[2], part[3], 0, 1, 2, 3, 4, 5, 6, 7)};
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int u = 0; u < 2; u++) O[u] = mfma_bf16(zf[s][u], P[s], O[u]);
        if (row < total - c * LC && col < p.V) *reinterpret_cast<bf16x8*>(out + (int64_t)(c * LC + row) * out_row + 2 * col) = pack8(O[0], O[1]);
    };
    run([](int, auto) {}, [](int, auto, int) {}, [] {},
        [&](int c, auto buf) __attribute__((always_inline)) {
            constexpr int B = decltype(buf)::value;
            const bf16_t* const x = tx + B * Shape::XY + 16 * w4 * KD;
            const bf16_t *const z = tz + B * Shape::Z, *const sf = ts + B * Shape::SF + (g4 * 32 + l16) * 8;
            bf16x8 xf[KT], state[KT][2];
            read_parts(1 - B);
#pragma unroll
            for (int k = 0; k < KT; k++) xf[k] = tile.fragment(x, k);
#pragma unroll
            for (int k = 0; k < KT; k++)
#pragma unroll
                for (int u = 0; u < 2; u++) state[k][u] = *reinterpret_cast<const bf16x8*>(sf + (k * 128 + 16 * u) * 8);
            __builtin_amdgcn_sched_barrier(0);  // all reads under way
            if (c > 0) finish(c - 1);
            O[0] = O[1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < KT; k++)
#pragma unroll
                for (int u = 0; u < 2; u++) O[u] = mfma_bf16(state[k][u], xf[k], O[u]);
#pragma unroll
            for (int s = 0; s < 2; s++)
#pragma unroll
                for (int u = 0; u < 2; u++) zf[s][u] = ztile.transposed(z, 32 * s, 0, u);
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int r = 0; r < 4; r++) O[u][r] *= row_weight;
        });
    if (chunks > 0) {
        read_parts((chunks - 1) & 1);
        finish(chunks - 1);
    }
}

template <int KD>
int launch(const LinearParams& p, hipStream_t stream) {
    const int64_t blocks = (int64_t)p.slots * p.H * ((p.V + 31) / 32);
    if (blocks > 0xfffff000ll / 768) return GDN_ERR_UNSUPPORTED;  // (a launch holds at most 2^32 - 1 threads)
    constexpr int bytes = ChainShape<KD>::LDS_BYTES;
    static_assert(bytes <= 160 * 1024, "LDS of a compute unit");
    auto* const kernel = p.fin != nullptr ? linear_chain_kernel<KD, true> : linear_chain_kernel<KD, false>;
    if (const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes); e != hipSuccess) return (int)e;
    hipLaunchKernelGGL(kernel, dim3((unsigned)((blocks + 7) / 8 * 8)), dim3(768), bytes, stream, p);
    return (int)hipGetLastError();
}

}  // namespace

int launch_linear_chain(const LinearParams& p, hipStream_t stream) { return p.K <= 64 ? launch<64>(p, stream) : launch<128>(p, stream); }

}  // namespace gdn
