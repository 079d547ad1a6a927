// Linear attention with a decay for each head: the derivative with respect to the log-decay g[h], over all sequences.
//
// The state's derivative U = dS / dg is carried along with the state, forward in time: per token U_t = w (U_{t-1} + S_{t-1}), and
//     dg = sum_t scale do_t . (U_t^T q_t) + <dht, U_T>
// No difference of large sums anywhere (the other way, sums of t (q_t . dq_t - k_t . dk_t), loses a digit with every factor of 10 of
// the length).  Per chunk of n tokens, i and j from 0:
//     dg += scale ( <G', S> + <G, U> + sum_{j <= i} (i - j) w^{i - j} (q_i . k_j) (do_i . v_j) ),   G = sum_i w^{i+1} q_i do_i^T,
//     G' = sum_i (i + 1) w^{i+1} q_i do_i^T;   U = w^n (U + n S) + sum_j (n - 1 - j) w^{n-1-j} k_j v_j^T,   S as ever
// bf16: on the matrix units, decayed rows in three bf16 parts (as the walk's states), S and U only ever as fp32: dg is good to fp32 sums
// of such terms, 1e-5.  A workgroup leaves one number per segment, head and columns; the sums over them are one more launch, in order.
// No prefetch here: where the keys number 64 at most two workgroups to a compute unit cover each other's loads.  Bound by latency and
// LDS: 6 left-padded rows of 1500 tokens, 16 heads of 64: the states and their derivatives 27 us, their sums 7, the dots 40, dg 5.
// S and U of all keys are one wave's: with 128 keys they and the fragments fill all its registers (4 x 4096 tokens, 16 heads of 128: 242 us of
// 596, forward and backward).  With 256 keys they do not fit, and the kernels live in scratch: the dots spill some 850 registers, the states
// some 100 (2 heads of 256 x 512: 557 us of 1141).  With 64 keys and four waves, which two workgroups to a unit hold to 256 registers, the
// dots spill some 95.
#include <algorithm>
#include <cfloat>

#include "gdn_launch.h"
#include "gdn_linear_tile.h"

namespace gdn {

namespace {

// sum over a workgroup, in thread 0
template <int THREADS>
__device__ __forceinline__ float block_sum(float x, float* shared) {
    x = wave_sum(x);
    __syncthreads();
    if (threadIdx.x % WAVE == 0) shared[threadIdx.x / WAVE] = x;
    __syncthreads();
    x = 0.f;
#pragma unroll
    for (int i = 0; i < THREADS / WAVE; i++) x += shared[i];
    return x;
}

template <int KD, int NW, bool STATES_ONLY>
__global__ __launch_bounds__(64 * NW, KD <= 64 ? NW / 2 : 1) void linear_tangent_kernel(const LinearParams p) {
    constexpr int NT = 64 * NW, VC = 32 * NW, KT = KD / 32;
    __shared__ __align__(16) bf16_t sq[STATES_ONLY ? 8 : LC * KD];
    __shared__ __align__(16) bf16_t sk[LC * KD];
    __shared__ __align__(16) bf16_t sv[LC * VC];
    __shared__ __align__(16) bf16_t sd[STATES_ONLY ? 8 : LC * VC];
    __shared__ __align__(16) float sw[4][LC];  // weights of rows: of v for S and U, of do for G and G'
    __shared__ float shared[NW];

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l32 = lane & 31, half = lane >> 5;
    const int slices = (p.V + VC - 1) / VC;
    const unsigned id = blockIdx.x;
    const int slice = id % slices, h = id / slices % p.H, slot = id / slices / p.H;
    const int c0 = slice * VC, columns = min(VC, p.V - c0);
    float* const dot = STATES_ONLY ? nullptr : p.dots + ((int64_t)slot * slices + slice) * p.H + h;
    LinearSegment sg;
    if (!linear_find(p, slot, sg, lane)) {
        if (!STATES_ONLY && tid == 0) *dot = 0.f;
        return;
    }
    const bool last = sg.s == linear_segments(sg.len, p.seg) - 1;
    if (STATES_ONLY && last) return;
    const int walked = sg.s * p.seg, total = min(p.seg, sg.len - walked);
    const int64_t token = (int64_t)sg.t0 + walked;
    const float g = linear_log2(p.g, h);

    Stream<KD, NT> ks(p.y, sg.b, h, token, false, 0, p.K, tid), qs(STATES_ONLY ? p.y : p.x, sg.b, h, token, false, 0, p.K, tid);
    Stream<VC, NT> vs(p.z, sg.b, h, token, false, c0, columns, tid), ds(STATES_ONLY ? p.z : p.d, sg.b, h, token, false, c0, columns, tid);

    const int64_t chain = (int64_t)sg.n * p.H + h, cells = p.cells, own = ((int64_t)slot * p.H + h) * cells;
    const int my_v = c0 + 32 * wave + slice_col(l32);
    auto key = [&](int kt, int r) { return 32 * kt + 16 * (r >> 3) + 8 * half + (r & 7); };
    f32x16 S[KT], U[KT];
#pragma unroll
    for (int kt = 0; kt < KT; kt++) S[kt] = f32x16{}, U[kt] = f32x16{};
    auto for_cells = [&](auto&& f) {
        if (my_v >= p.V) return;
#pragma unroll
        for (int kt = 0; kt < KT; kt++)
#pragma unroll
            for (int r = 0; r < 16; r++)
                if (key(kt, r) < p.K) f(kt, r, (int64_t)key(kt, r) * p.V + my_v);
    };
    if constexpr (!STATES_ONLY) {
        if (sg.s > 0) for_cells([&](int kt, int r, int64_t at) { S[kt][r] = p.local[own + at], U[kt][r] = p.local_slope[own + at]; });
        else if (p.init != nullptr) for_cells([&](int kt, int r, int64_t at) { S[kt][r] = p.init[chain * cells + at]; });
    }

    const TileLane<KD> tile(lane);
    const TileLane<VC> ztile(lane);
    // B fragments (reduction over rows, column = this lane's) of a tile's columns of this wave, weighted, in three parts
    auto weighted = [&](const bf16_t* rows_of, const float* weights, bf16x8 (&part)[3][4]) {
#pragma unroll
        for (int s = 0; s < 4; s++) {
            const bf16x8 rows = ztile.transposed(rows_of, s, wave);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                float x = (float)rows[e] * weights[16 * s + 8 * half + e];
#pragma unroll
                for (int u = 0; u < 3; u++) part[u][s][e] = (bf16_t)x, x -= (float)part[u][s][e];
            }
        }
    };
    auto product = [&](const bf16_t* rows_of, int kt, const bf16x8 (&part)[3][4], f32x16 acc) {
#pragma unroll
        for (int s = 0; s < 4; s++) {
            const bf16x8 a = tile.transposed(rows_of, s, kt);
#pragma unroll
            for (int u = 0; u < 3; u++) acc = mfma32_bf16(a, part[u][s], acc);
        }
        return acc;
    };

    float sum = 0.f;
    const int chunks = (total + LC - 1) / LC;
    for (int c = 0; c < chunks; c++) {
        const int rows = min(LC, total - c * LC);
        bf16x8 rk[Stream<KD, NT>::ITERS], rv[Stream<VC, NT>::ITERS], rq[STATES_ONLY ? 1 : Stream<KD, NT>::ITERS], rd[STATES_ONLY ? 1 : Stream<VC, NT>::ITERS];
        ks.fetch(rk, rows, false), vs.fetch(rv, rows, false);
        if constexpr (!STATES_ONLY) qs.fetch(rq, rows, false), ds.fetch(rd, rows, false);
        __syncthreads();  // the tiles of the chunk before are read
        if (tid < LC) {
            const int left = max(rows - 1 - tid, 0);
            const float w = linear_power(g, left);
            sw[0][tid] = w, sw[1][tid] = (float)left * w;
            if constexpr (!STATES_ONLY) {
                const int from_start = min(tid + 1, rows);  // (behind the last row there are zeros: no power that could overflow where the rows' own do not)
                const float forward = p.os * linear_power(g, from_start);
                sw[2][tid] = forward, sw[3][tid] = (float)from_start * forward;
            }
        }
        ks.stage(sk, rk, rows, false), vs.stage(sv, rv, rows, false);
        if constexpr (!STATES_ONLY) qs.stage(sq, rq, rows, false), ds.stage(sd, rd, rows, false);
        __syncthreads();
        bf16x8 part[3][4];
        if constexpr (!STATES_ONLY) {
            weighted(sd, sw[3], part);
#pragma unroll
            for (int kt = 0; kt < KT; kt++) {
                const f32x16 G = product(sq, kt, part, f32x16{});
#pragma unroll
                for (int r = 0; r < 16; r++) sum += G[r] * S[kt][r];
            }
            weighted(sd, sw[2], part);
#pragma unroll
            for (int kt = 0; kt < KT; kt++) {
                const f32x16 G = product(sq, kt, part, f32x16{});
#pragma unroll
                for (int r = 0; r < 16; r++) sum += G[r] * U[kt][r];
            }
            // inside the chunk: this wave's columns of do . v, all keys of q . k; rows i, keys j
#pragma unroll
            for (int t = 0; t < 3; t++) {
                const int jt = t == 2, it = t >= 1;
                f32x16 A = {}, B = {};
#pragma unroll
                for (int s = 0; s < KD / 16; s++)
                    A = mfma32_bf16(tile.fragment(sk, 32 * jt, s), tile.fragment(sq, 32 * it, s), A);
#pragma unroll
                for (int s = 0; s < 2; s++)
                    B = mfma32_bf16(ztile.fragment(sv, 32 * jt, 2 * wave + s), ztile.fragment(sd, 32 * it, 2 * wave + s), B);
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int distance = 32 * it + l32 - (32 * jt + 8 * (r >> 2) + 4 * half + (r & 3));
                    // (finite: the products of missing rows are zeros; cut off at `rows` instead, it would be formed anew in every chunk,
                    // 4 x 4096 tokens of 16 heads of 128 611 us forward and backward instead of 573)
                    const float weight = __builtin_amdgcn_fmed3f(p.ps * (float)distance * linear_power(g, distance), -FLT_MAX, FLT_MAX);
                    if (distance > 0) sum += A[r] * B[r] * weight;
                }
            }
        }
        const float whole = linear_power(g, rows);
#pragma unroll
        for (int kt = 0; kt < KT; kt++)
#pragma unroll
            for (int r = 0; r < 16; r++) {
                U[kt][r] = whole * (U[kt][r] + (float)rows * S[kt][r]);
                S[kt][r] *= whole;
            }
        weighted(sv, sw[1], part);
#pragma unroll
        for (int kt = 0; kt < KT; kt++) U[kt] = product(sk, kt, part, U[kt]);
        weighted(sv, sw[0], part);
#pragma unroll
        for (int kt = 0; kt < KT; kt++) S[kt] = product(sk, kt, part, S[kt]);
    }
    if constexpr (STATES_ONLY) {
        for_cells([&](int kt, int r, int64_t at) { p.local[own + at] = S[kt][r], p.local_slope[own + at] = U[kt][r]; });
    } else {
        if (last && p.init_grad != nullptr) for_cells([&](int kt, int r, int64_t at) { sum += p.init_grad[chain * cells + at] * U[kt][r]; });
        sum = block_sum<NT>(sum, shared);
        if (tid == 0) *dot = sum;
    }
}

// The same token by token in fp32: a workgroup has 32 columns, a thread 4 of them and KR keys, as in linear_tokens_kernel.
template <int KR, bool STATES_ONLY>
__global__ __launch_bounds__(256) void linear_tangent_tokens_kernel(const LinearParams p) {
    constexpr int VL = 8, GROUPS = 256 / VL, KP = GROUPS * KR, VC = 4 * VL, TB = 16;
    __shared__ __align__(16) float sq[STATES_ONLY ? 1 : TB][KP];
    __shared__ __align__(16) float sk[TB][KP];
    __shared__ __align__(16) float sv[TB][VC];
    __shared__ __align__(16) float sd[STATES_ONLY ? 1 : TB][VC];
    __shared__ float shared[4];

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int slices = (p.V + VC - 1) / VC;
    const unsigned id = blockIdx.x;
    const int slice = id % slices, h = id / slices % p.H, slot = id / slices / p.H;
    const int c0 = slice * VC, columns = min(VC, p.V - c0);
    float* const dot = STATES_ONLY ? nullptr : p.dots + ((int64_t)slot * slices + slice) * p.H + h;
    LinearSegment sg;
    if (!linear_find(p, slot, sg, lane)) {
        if (!STATES_ONLY && tid == 0) *dot = 0.f;
        return;
    }
    const bool last = sg.s == linear_segments(sg.len, p.seg) - 1;
    if (STATES_ONLY && last) return;
    const int walked = sg.s * p.seg, total = min(p.seg, sg.len - walked);
    const int64_t token = (int64_t)sg.t0 + walked;
    const LinearFactor w(p.g[h]);

    const int group = wave * (64 / VL) + lane / VL, col = 4 * (lane % VL);
    const bool mine = col < columns;
    const int64_t chain = (int64_t)sg.n * p.H + h, cells = p.cells, own = ((int64_t)slot * p.H + h) * cells;
    auto key = [&](int r) { return r * GROUPS + group; };
    auto at = [&](const float* base, int r) { return reinterpret_cast<const f32x4*>(base + (int64_t)key(r) * p.V + c0 + col); };
    f32x4 S[KR], U[KR];
#pragma unroll
    for (int r = 0; r < KR; r++) {
        S[r] = U[r] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (STATES_ONLY || !mine || key(r) >= p.K) continue;
        if (sg.s > 0) S[r] = *at(p.local + own, r), U[r] = *at(p.local_slope + own, r);
        else if (p.init != nullptr) S[r] = *at(p.init + chain * cells, r);
    }
    auto role = [&](const LinearRole& x) { return static_cast<const float*>(x.p) + sg.b * x.stride_b + (h / x.div) * x.stride_h + token * x.stride_t; };
    const float *const pk = role(p.y), *const pv = role(p.z), *const pq = role(STATES_ONLY ? p.y : p.x), *const pd = role(STATES_ONLY ? p.z : p.d);

    float sum = 0.f;
    const f32x4 none = {0.f, 0.f, 0.f, 0.f};
    for (int first = 0; first < total; first += TB) {
        const int n = min(TB, total - first);
        if (first > 0) __syncthreads();
        for (int i = tid; i < n * (KP / 4); i += 256) {
            const int t = i / (KP / 4), k = (i - t * (KP / 4)) * 4;
            const int64_t row = first + t;
            *reinterpret_cast<f32x4*>(&sk[t][k]) = k < p.K ? load4<float>(pk + row * p.y.stride_t + k) : none;
            if constexpr (!STATES_ONLY) *reinterpret_cast<f32x4*>(&sq[t][k]) = k < p.K ? load4<float>(pq + row * p.x.stride_t + k) * p.os : none;
        }
        for (int i = tid; i < n * VL; i += 256) {
            const int t = i / VL, c = (i - t * VL) * 4;
            const int64_t row = first + t;
            *reinterpret_cast<f32x4*>(&sv[t][c]) = c < columns ? load4<float>(pv + row * p.z.stride_t + c0 + c) : none;
            if constexpr (!STATES_ONLY) *reinterpret_cast<f32x4*>(&sd[t][c]) = c < columns ? load4<float>(pd + row * p.d.stride_t + c0 + c) : none;
        }
        __syncthreads();
        auto walk = [&](auto shrunk) __attribute__((always_inline)) {
            for (int t = 0; t < n; t++) {
                const f32x4 v = *reinterpret_cast<const f32x4*>(&sv[t][col]);
                f32x4 o = none;
#pragma unroll
                for (int r = 0; r < KR; r++) {
                    U[r] = shrunk(U[r] + S[r]);
                    S[r] = shrunk(S[r]) + v * sk[t][key(r)];
                    if constexpr (!STATES_ONLY) o += U[r] * sq[t][key(r)];
                }
                if constexpr (!STATES_ONLY) {
                    const f32x4 d = *reinterpret_cast<const f32x4*>(&sd[t][col]);
                    sum += o[0] * d[0] + o[1] * d[1] + o[2] * d[2] + o[3] * d[3];
                }
            }
        };
        // (one operation each: with both parts multiplied 4 x 1024 tokens of 16 heads of 128 take 5 % longer, forward and backward)
        if (w.kept == 1.f) walk([&](f32x4 s) { return s * w.rest + s; });
        else walk([&](f32x4 s) { return s * w.rest; });
    }
    if constexpr (STATES_ONLY) {
#pragma unroll
        for (int r = 0; r < KR; r++)
            if (mine && key(r) < p.K) {
                *const_cast<f32x4*>(at(p.local + own, r)) = S[r];
                *const_cast<f32x4*>(at(p.local_slope + own, r)) = U[r];
            }
    } else {
#pragma unroll
        for (int r = 0; r < KR; r++)
            if (last && p.init_grad != nullptr && mine && key(r) < p.K) {
                const f32x4 x = *at(p.init_grad + chain * cells, r) * U[r];
                sum += x[0] + x[1] + x[2] + x[3];
            }
        sum = block_sum<256>(sum, shared);
        if (tid == 0) *dot = sum;
    }
}

// as linear_combine_kernel, state and derivative together
__global__ __launch_bounds__(256) void linear_tangent_combine_kernel(const LinearParams p) {
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
        if (slot0 + segments > p.slots || at >= p.cells) continue;
        const LinearFactor whole = linear_factor(p.g[h], p.seg);
        const float tokens = (float)p.seg;
        const int64_t first = ((int64_t)slot0 * p.H + h) * p.cells + at, next = (int64_t)p.H * p.cells;
        auto cell = [&](float* base, int s) { return reinterpret_cast<f32x4*>(base + first + s * next); };
        f32x4 S = {0.f, 0.f, 0.f, 0.f}, U = S;
        if (p.init != nullptr) S = *reinterpret_cast<const f32x4*>(p.init + ((int64_t)n * p.H + h) * p.cells + at);
        f32x4 own_S = *cell(p.local, 0), own_U = *cell(p.local_slope, 0);
        for (int s = 1; s < segments; s++) {
            f32x4 next_S = {0.f, 0.f, 0.f, 0.f}, next_U = next_S;
            if (s + 1 < segments) next_S = *cell(p.local, s), next_U = *cell(p.local_slope, s);
            U = whole(U + S * tokens) + own_U;
            S = whole(S) + own_S;
            *cell(p.local, s) = S, *cell(p.local_slope, s) = U;
            own_S = next_S, own_U = next_U;
        }
    }
}

__global__ __launch_bounds__(256) void linear_tangent_sum_kernel(const float* dots, int count, int H, float* dg) {
    __shared__ float shared[4];
    const int h = blockIdx.x;
    float sum = 0.f;
    for (int i = threadIdx.x; i < count; i += 256) sum += dots[(int64_t)i * H + h];
    sum = block_sum<256>(sum, shared);
    if (threadIdx.x == 0) dg[h] = sum;
}

template <int KD, int NW>
void launch(const LinearParams& p, bool states_only, unsigned blocks, hipStream_t stream) {
    if (states_only) hipLaunchKernelGGL((linear_tangent_kernel<KD, NW, true>), dim3(blocks), dim3(64 * NW), 0, stream, p);
    else hipLaunchKernelGGL((linear_tangent_kernel<KD, NW, false>), dim3(blocks), dim3(64 * NW), 0, stream, p);
}
template <int KR>
void launch_tokens(const LinearParams& p, bool states_only, unsigned blocks, hipStream_t stream) {
    if (states_only) hipLaunchKernelGGL((linear_tangent_tokens_kernel<KR, true>), dim3(blocks), dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((linear_tangent_tokens_kernel<KR, false>), dim3(blocks), dim3(256), 0, stream, p);
}

void run_one(const LinearParams& p, int dtype, bool states_only, unsigned blocks, hipStream_t stream) {
    if (dtype == GDN_F32) {
        if (p.K <= 64) return launch_tokens<2>(p, states_only, blocks, stream);
        if (p.K <= 128) return launch_tokens<4>(p, states_only, blocks, stream);
        return launch_tokens<8>(p, states_only, blocks, stream);
    }
    // Two waves have all columns of a value dim up to 64, and twice the workgroups fit: 4 x 4096 tokens, heads of 64 x 64 (16) 281 us, forward and
    // backward, with four waves 339, of 128 x 64 402 | 490, of 256 x 64 (8) 859 | 907, of 64 x 32 269 | 332.
    const bool narrow = p.V <= 64;
    if (p.K <= 64) return narrow ? launch<64, 2>(p, states_only, blocks, stream) : launch<64, 4>(p, states_only, blocks, stream);
    if (p.K <= 128) return narrow ? launch<128, 2>(p, states_only, blocks, stream) : launch<128, 4>(p, states_only, blocks, stream);
    return narrow ? launch<256, 2>(p, states_only, blocks, stream) : launch<256, 4>(p, states_only, blocks, stream);
}

}  // namespace

int linear_tangent_columns(int dtype, int V) { return dtype == GDN_F32 ? 32 : V <= 64 ? 64 : 128; }

int launch_linear_tangent(const LinearParams& p, int dtype, bool several, float* dg, hipStream_t stream) {
    const int columns = linear_tangent_columns(dtype, p.V);
    const int64_t slices = (p.V + columns - 1) / columns, blocks = p.slots * slices * p.H;
    if (blocks > 0xfffff000ll / 256) return GDN_ERR_UNSUPPORTED;
    if (several) {
        run_one(p, dtype, true, (unsigned)blocks, stream);
        if (const hipError_t e = hipGetLastError(); e != hipSuccess) return (int)e;
        hipLaunchKernelGGL(linear_tangent_combine_kernel, dim3((unsigned)((p.cells + 1023) / 1024), (unsigned)p.H, (unsigned)std::min(p.N, 32768)), dim3(256), 0, stream, p);
        if (const hipError_t e = hipGetLastError(); e != hipSuccess) return (int)e;
    }
    run_one(p, dtype, false, (unsigned)blocks, stream);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return (int)e;
    hipLaunchKernelGGL(linear_tangent_sum_kernel, dim3((unsigned)p.H), dim3(256), 0, stream, p.dots, (int)(p.slots * slices), p.H, dg);
    return (int)hipGetLastError();
}

}  // namespace gdn
