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
#include <algorithm>

#include "gdn_launch.h"
#include "gdn_linear_tile.h"

namespace gdn {

namespace {

template <int KD, int NW, bool STATES_ONLY>
__global__ __launch_bounds__(64 * NW, KD <= 128 ? NW / 2 : NW / 4 > 0 ? NW / 4 : 1) void linear_walk_kernel(const LinearParams p) {
    constexpr int NT = 64 * NW, VC = 32 * NW, KT = KD / 32;
    __shared__ __align__(16) bf16_t sx[STATES_ONLY ? 8 : LC * KD];
    __shared__ __align__(16) bf16_t sy[LC * KD];
    __shared__ __align__(16) bf16_t sz[LC * VC];
    __shared__ __align__(16) bf16_t sp[STATES_ONLY ? 8 : 6 * 512];
    __shared__ __align__(16) float sw[LC];  // us w^{n - a - j}

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l32 = lane & 31, half = lane >> 5;
    // blocks are dealt round the 8 XCDs: the blocks of one XCD get neighbouring places, so that those that read the same rows
    // (columns of the value dim, heads that share keys) meet in its L2
    const unsigned per_xcd = (gridDim.x + 7) / 8;
    const unsigned id = blockIdx.x % 8 * per_xcd + blockIdx.x / 8;
    const int slices = (p.V + VC - 1) / VC;
    if (id >= (unsigned)p.slots * p.H * slices) return;
    const int slice = id % slices, h = id / slices % p.H, slot = id / slices / p.H;
    const int c0 = slice * VC, columns = min(VC, p.V - c0);

    if constexpr (!STATES_ONLY)
        if (p.zero && (p.cu != nullptr)) linear_zero_gaps<bf16_t, 8>(p, slot, h, c0, columns, tid, NT);
    LinearSegment sg;
    if (!linear_find(p, slot, sg, lane)) return;
    const int segments = linear_segments(sg.len, p.seg);
    const bool last = sg.s == segments - 1;
    if (STATES_ONLY && last) return;  // nothing starts from it
    const int walked = sg.s * p.seg, total = min(p.seg, sg.len - walked);
    const int64_t token = p.reverse ? (int64_t)sg.t0 + sg.len - 1 - walked : (int64_t)sg.t0 + walked;  // the first of the walk
    const float g = p.g == nullptr ? 0.f : p.g[h];
    const int a = p.a;

    Stream<KD, NT> ys(p.y, sg.b, h, token, p.reverse, 0, p.K, tid);
    Stream<VC, NT> zs(p.z, sg.b, h, token, p.reverse, c0, columns, tid);
    Stream<KD, NT> xs(STATES_ONLY ? p.y : p.x, sg.b, h, token, p.reverse, 0, p.K, tid);

    const int64_t chain = (int64_t)sg.n * p.H + h, cells = p.cells;
    const int my_v = c0 + 32 * wave + slice_col(l32);  // the state's column of this lane
    auto state_at = [&](int kt, int r) { return (int64_t)(32 * kt + 16 * (r >> 3) + 8 * half + (r & 7)) * p.state_k + (int64_t)my_v * p.state_v; };
    auto state_key = [&](int kt, int r) { return 32 * kt + 16 * (r >> 3) + 8 * half + (r & 7); };
    f32x16 S[KT];
#pragma unroll
    for (int kt = 0; kt < KT; kt++) S[kt] = f32x16{};
    const float* from = nullptr;
    if (!STATES_ONLY) from = sg.s > 0 ? p.local + ((int64_t)slot * p.H + h) * cells : p.init == nullptr ? nullptr : p.init + chain * cells;
    if (from != nullptr && my_v < p.V) {
#pragma unroll
        for (int kt = 0; kt < KT; kt++)
#pragma unroll
            for (int r = 0; r < 16; r++)
                if (state_key(kt, r) < p.K) S[kt][r] = from[state_at(kt, r)];
    }

    // the wave's tile of P: (key tile, row tile) (0, 0), (0, 1), (1, 1); on the diagonal rows before the key get nothing
    constexpr int TILES = 3;
    f32x16 decay = {};
    if constexpr (!STATES_ONLY) {
        const int t = wave;  // NW = 2: wave 0 has both tiles on the diagonal
        const int ji = t == 1 ? -32 : 0;
#pragma unroll
        for (int r = 0; r < 16; r++) {
            const int distance = l32 - (16 * (r >> 3) + 8 * half + (r & 7)) - ji;
            decay[r] = distance >= 0 ? p.ps * linear_power(g, distance) : 0.f;
        }
    }
    float row_weight[2];
#pragma unroll
    for (int i = 0; i < 2; i++) row_weight[i] = p.os * linear_power(g, 32 * i + l32 + a);

    // outputs: this lane's row of the chunk's first 32, its 8 columns
    bf16_t* out = static_cast<bf16_t*>(p.out) + sg.b * p.out_stride_b + h * p.out_stride_h + token * p.out_stride_t;
    const int64_t out_row = p.reverse ? -p.out_stride_t : p.out_stride_t;
    float* sums = p.sums == nullptr ? nullptr : p.sums + ((int64_t)sg.b * p.T + token) * p.H * p.V + (int64_t)h * p.V;
    const int64_t sums_row = (p.reverse ? -1 : 1) * (int64_t)p.H * p.V;

    const int chunks = (total + LC - 1) / LC;
    ys.load(total), zs.load(total);
    if constexpr (!STATES_ONLY) xs.load(total);
    for (int c = 0; c < chunks; c++) {
        const int rows = min(LC, total - c * LC);
        __syncthreads();  // the tiles of the chunk before are read
        if (c == 0 || rows < LC) {
            if (tid < LC) sw[tid] = p.us * linear_power(g, max(rows - a - tid, 0));
        }
        ys.store(sy), zs.store(sz);
        if constexpr (!STATES_ONLY) xs.store(sx);
        __syncthreads();
        if (c + 1 < chunks) {
            const int left = total - (c + 1) * LC;
            ys.load(left), zs.load(left);
            if constexpr (!STATES_ONLY) xs.load(left);
        }
        bf16x8 zf[4];
#pragma unroll
        for (int s = 0; s < 4; s++) zf[s] = tile_tr8<VC>(sz, 16 * s, 32 * wave, lane);

        if constexpr (!STATES_ONLY) {
            for (int t = wave; t < TILES; t += NW) {
                const int jt = t == 2, it = t >= 1;
                f32x16 acc = {};
#pragma unroll
                for (int s = 0; s < KD / 16; s++)
                    acc = mfma32_bf16(tile_row8<KD>(sy, 32 * jt + slice_col(l32), 2 * s + half), tile_row8<KD>(sx, 32 * it + l32, 2 * s + half), acc);
                // selected, not multiplied away: a row before the key takes nothing of it, whatever its product is
#pragma unroll
                for (int r = 0; r < 16; r++) acc[r] = t != 1 && l32 < 16 * (r >> 3) + 8 * half + (r & 7) ? 0.f : acc[r] * decay[r];
                *reinterpret_cast<bf16x8*>(sp + (2 * t + 0) * 512 + lane * 8) = pack8_16(acc, 0, 1.f);
                *reinterpret_cast<bf16x8*>(sp + (2 * t + 1) * 512 + lane * 8) = pack8_16(acc, 1, 1.f);
            }
            f32x16 O[2] = {};
#pragma unroll
            for (int kt = 0; kt < KT; kt++)
#pragma unroll
                for (int s = 0; s < 2; s++) {
                    const bf16x8 sf = pack8_16(S[kt], s, 1.f);  // the state as an operand: its one rounding to bf16 for the output
#pragma unroll
                    for (int i = 0; i < 2; i++) O[i] = mfma32_bf16(sf, tile_row8<KD>(sx, 32 * i + l32, 4 * kt + 2 * s + half), O[i]);
                }
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int r = 0; r < 16; r++) O[i][r] *= row_weight[i];
            __syncthreads();  // P is there
#pragma unroll
            for (int t = 0; t < TILES; t++)
#pragma unroll
                for (int s = 0; s < 2; s++)
                    O[t >= 1] = mfma32_bf16(zf[2 * (t == 2) + s], *reinterpret_cast<const bf16x8*>(sp + (2 * t + s) * 512 + lane * 8), O[t >= 1]);
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int row = 32 * i + l32;
                if (row < rows) {
#pragma unroll
                    for (int s = 0; s < 2; s++) {
                        const int col = c0 + 32 * wave + 16 * s + 8 * half;
                        if (col >= p.V) continue;
                        if (sums != nullptr) {
                            float* at = sums + (c * LC + row) * sums_row + col;
#pragma unroll
                            for (int e = 0; e < 8; e++) {
                                if (p.sums_in) O[i][8 * s + e] += at[e];
                                if (p.sums_out) at[e] = O[i][8 * s + e];
                            }
                            if (p.sums_out) continue;
                        }
                        *reinterpret_cast<bf16x8*>(out + (c * LC + row) * out_row + col) = pack8_16(O[i], s, 1.f);
                    }
                }
            }
        }
        // The state's own sums are kept to fp32 accuracy: the decayed rows of z go in as two bf16 parts, high and low (16 bits and
        // more together), the rows of y are exact.
        bf16x8 hi[4], lo[4];
#pragma unroll
        for (int s = 0; s < 4; s++) {
            const float* weights = sw + 16 * s + 8 * half;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float z = (float)zf[s][e] * weights[e];
                hi[s][e] = (bf16_t)z;
                lo[s][e] = (bf16_t)(z - (float)hi[s][e]);
            }
        }
        const float whole = linear_power(g, rows);
#pragma unroll
        for (int kt = 0; kt < KT; kt++) {
#pragma unroll
            for (int r = 0; r < 16; r++) S[kt][r] *= whole;
#pragma unroll
            for (int s = 0; s < 4; s++) {
                const bf16x8 yt = tile_tr8<KD>(sy, 16 * s, 32 * kt, lane);
                S[kt] = mfma32_bf16(yt, hi[s], S[kt]);
                S[kt] = mfma32_bf16(yt, lo[s], S[kt]);
            }
        }
    }
    float* to = nullptr;
    if constexpr (STATES_ONLY) to = p.local + ((int64_t)slot * p.H + h) * cells;
    else if (last && p.fin != nullptr) to = p.fin + chain * cells;
    if (to != nullptr && my_v < p.V) {
#pragma unroll
        for (int kt = 0; kt < KT; kt++)
#pragma unroll
            for (int r = 0; r < 16; r++)
                if (state_key(kt, r) < p.K) to[state_at(kt, r)] = S[kt][r];
    }
}

// From the segments' own states (slots 0 .. of a sequence) to what every segment but the first starts from.  A thread has 4 cells
// of a (sequence, head); the states lie contiguous, and those of a sequence H states apart.
__global__ __launch_bounds__(256) void linear_combine_kernel(const LinearParams p) {
    const int64_t cells = p.cells;
    const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    const int h = blockIdx.y;
    for (int n = blockIdx.z; n < p.N; n += gridDim.z) {
        int b, t0, len;
        linear_bounds(p, n, b, t0, len);
        const int segments = linear_segments(len, p.seg);
        if (segments == 1) continue;
        int slot0 = n * p.nseg;
        if (p.nseg == 0) {
            LinearSegment none;
            linear_find_packed(p, -1, none, threadIdx.x & 63, n, &slot0);
        }
        if (slot0 + segments > p.slots || at >= cells) continue;
        const float whole = linear_power(p.g == nullptr ? 0.f : p.g[h], p.seg);
        float* local = p.local + ((int64_t)slot0 * p.H + h) * cells + at;
        const int64_t next = (int64_t)p.H * cells;
        f32x4 carry = {0.f, 0.f, 0.f, 0.f};
        if (p.init != nullptr) carry = *reinterpret_cast<const f32x4*>(p.init + ((int64_t)n * p.H + h) * cells + at);
        f32x4 own = *reinterpret_cast<const f32x4*>(local);
        for (int s = 1; s < segments; s++) {
            f32x4 following = {0.f, 0.f, 0.f, 0.f};
            if (s + 1 < segments) following = *reinterpret_cast<const f32x4*>(local + s * next);
            carry = carry * whole + own;
            *reinterpret_cast<f32x4*>(local + s * next) = carry;
            own = following;
        }
    }
}

template <int KD, int NW>
int launch(const LinearParams& p, bool states_only, hipStream_t stream) {
    const int64_t blocks = (int64_t)p.slots * p.H * ((p.V + 32 * NW - 1) / (32 * NW));
    if (blocks > 0xfffff000ll / (64 * NW)) return GDN_ERR_UNSUPPORTED;  // (a launch holds at most 2^32 - 1 threads)
    const dim3 grid((unsigned)((blocks + 7) / 8 * 8)), threads(64 * NW);
    if (states_only) hipLaunchKernelGGL((linear_walk_kernel<KD, NW, true>), grid, threads, 0, stream, p);
    else hipLaunchKernelGGL((linear_walk_kernel<KD, NW, false>), grid, threads, 0, stream, p);
    return (int)hipGetLastError();
}

}  // namespace

int linear_walk_columns(int V) { return V <= 64 ? 64 : 128; }

int launch_linear_walk(const LinearParams& p, bool states_only, hipStream_t stream) {
    const bool narrow = linear_walk_columns(p.V) == 64;
    if (p.K <= 64) return narrow ? launch<64, 2>(p, states_only, stream) : launch<64, 4>(p, states_only, stream);
    if (p.K <= 128) return narrow ? launch<128, 2>(p, states_only, stream) : launch<128, 4>(p, states_only, stream);
    return narrow ? launch<256, 2>(p, states_only, stream) : launch<256, 4>(p, states_only, stream);
}

int launch_linear_combine(const LinearParams& p, hipStream_t stream) {
    hipLaunchKernelGGL(linear_combine_kernel, dim3((unsigned)((p.cells + 1023) / 1024), (unsigned)p.H, (unsigned)std::min(p.N, 32768)), dim3(256), 0, stream, p);
    return (int)hipGetLastError();
}

}  // namespace gdn
