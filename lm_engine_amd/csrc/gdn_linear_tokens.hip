// Linear attention with a decay for each head, token by token in fp32: decoding (one token, or a few, per state) and the exact path
// of fp32 inputs.  The recurrence and its roles: gdn_linear_common.h.
//
// A workgroup has 4 VL columns of the value dim and all keys of one (segment, head).  A thread has 4 columns of KR keys in a row, in
// registers: on a single token it reads and writes 16-byte pieces, 16 VL bytes of a state row at a time, and the state passes through it
// once, past the caches.  Tokens are taken TB at a time through LDS; per token a lane adds up its keys, the lanes of a wave their
// groups by shuffles, and the four waves' sums meet in LDS behind the TB.
// Bound by memory on one token: 256 states of 32 heads, K = V = 128, 1.07 GB to and fro: 178 us, 6.0 TB/s (203 through the caches; at 128
// states, which they hold from call to call, 93 against 78: a model's other layers would not leave them there).  On many tokens by the
// chain from one token to the next: 0.36 us a token in the smallest calls, 4 x 1024 tokens of 16 heads of 128 in fp32 299 us (280 with a
// token's factor as one number).
#include <algorithm>

#include "gdn_launch.h"
#include "gdn_linear_common.h"

namespace gdn {

namespace {

// TB: tokens of a batch
template <typename T, int KR, int VL, int TB, bool STATES_ONLY>
__global__ __launch_bounds__(256) void linear_tokens_kernel(const LinearParams p) {
    constexpr int GROUPS = 256 / VL, KP = GROUPS * KR, VC = 4 * VL;
    __shared__ __align__(16) float sx[STATES_ONLY ? 1 : TB][KP];
    __shared__ __align__(16) float sy[TB][KP];
    __shared__ __align__(16) float sz[TB][VC];
    __shared__ __align__(16) float part[STATES_ONLY ? 1 : 4][TB][VC];

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const unsigned per_xcd = (gridDim.x + 7) / 8;  // as in linear_walk_kernel
    const unsigned id = blockIdx.x % 8 * per_xcd + blockIdx.x / 8;
    const int slices = (p.V + VC - 1) / VC;
    if (id >= (unsigned)p.slots * p.H * slices) return;
    const int slice = id % slices, h = id / slices % p.H, slot = id / slices / p.H;
    const int c0 = slice * VC, columns = min(VC, p.V - c0);
    if constexpr (!STATES_ONLY)
        if (p.zero && p.cu != nullptr) linear_zero_gaps<T>(p, slot, h, c0, columns, tid, 256);
    LinearSegment sg;
    if (!linear_find(p, slot, sg, lane)) return;
    const bool last = sg.s == linear_segments(sg.len, p.seg) - 1;
    if (STATES_ONLY && last && p.fin == nullptr) return;  // nothing starts from it
    const int walked = sg.s * p.seg, total = min(p.seg, sg.len - walked);
    const int64_t token = p.reverse ? (int64_t)sg.t0 + sg.len - 1 - walked : (int64_t)sg.t0 + walked;
    const LinearFactor factor(p.g == nullptr ? 0.f : p.g[h]), none(0.f);  // of a token

    const int vl = lane % VL, group = wave * (64 / VL) + lane / VL;
    const int col = 4 * vl;
    const bool mine = col < columns;
    const int64_t chain = (int64_t)sg.n * p.H + h, cells = p.cells;
    auto key = [&](int r) { return group * KR + r; };
    auto state_at = [&](int r) { return (int64_t)key(r) * p.state_k + (int64_t)(c0 + col) * p.state_v; };
    f32x4 S[KR];
#pragma unroll
    for (int r = 0; r < KR; r++) S[r] = f32x4{0.f, 0.f, 0.f, 0.f};
    const float* from = nullptr;
    if (!STATES_ONLY) from = sg.s > 0 ? p.local + ((int64_t)slot * p.H + h) * p.local_cells : p.init == nullptr ? nullptr : p.init + chain * cells;
    if (from != nullptr && mine) {
        if (p.state_v == 1) {
#pragma unroll
            for (int r = 0; r < KR; r++)
                if (key(r) < p.K) S[r] = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(from + state_at(r)));
        } else {
            for (int r = 0; r < KR; r++)
                for (int e = 0; e < 4; e++)
                    if (key(r) < p.K) S[r][e] = from[state_at(r) + (int64_t)e * p.state_v];
        }
    }

    const int64_t step = p.reverse ? -1 : 1;
    auto role = [&](const LinearRole& x) { return static_cast<const T*>(x.p) + sg.b * x.stride_b + (h / x.div) * x.stride_h + token * x.stride_t; };
    const T* const px = role(STATES_ONLY ? p.y : p.x);
    const T* const py = role(p.y);
    const T* const pz = role(p.z);
    T* const out = static_cast<T*>(p.out) + sg.b * p.out_stride_b + h * p.out_stride_h + token * p.out_stride_t;
    float* const sums = p.sums == nullptr ? nullptr : p.sums + ((int64_t)sg.b * p.T + token) * p.H * p.V + (int64_t)h * p.V;

    for (int first = 0; first < total; first += TB) {
        const int n = min(TB, total - first);
        if (first > 0) __syncthreads();
        for (int i = tid; i < n * (KP / 4); i += 256) {
            const int t = i / (KP / 4), k = (i - t * (KP / 4)) * 4;
            f32x4 x = {0.f, 0.f, 0.f, 0.f}, y = x;
            if (k < p.K) {
                y = load4<T>(py + (first + t) * step * p.y.stride_t + k);
                if constexpr (!STATES_ONLY) x = load4<T>(px + (first + t) * step * p.x.stride_t + k);
            }
            *reinterpret_cast<f32x4*>(&sy[t][k]) = y * p.us;
            if constexpr (!STATES_ONLY) *reinterpret_cast<f32x4*>(&sx[t][k]) = x;
        }
        for (int i = tid; i < n * VL; i += 256) {
            const int t = i / VL, c = (i - t * VL) * 4;
            f32x4 z = {0.f, 0.f, 0.f, 0.f};
            if (c < columns) z = load4<T>(pz + (first + t) * step * p.z.stride_t + c0 + c);
            *reinterpret_cast<f32x4*>(&sz[t][c]) = z;
        }
        __syncthreads();
        for (int t = 0; t < n; t++) {
            const LinearFactor w = p.a == 1 || first + t > 0 ? factor : none;  // a = 0: the state decays behind a token, not in front of it
            const f32x4 z = *reinterpret_cast<const f32x4*>(&sz[t][col]);
            f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int r = 0; r < KR; r++) {
                S[r] = w(S[r]) + z * sy[t][key(r)];
                if constexpr (!STATES_ONLY) o += S[r] * sx[t][key(r)];
            }
            if constexpr (!STATES_ONLY) {
#pragma unroll
                for (int off = VL; off < 64; off <<= 1)
#pragma unroll
                    for (int e = 0; e < 4; e++) o[e] += __shfl_xor(o[e], off, WAVE);
                if (lane < VL) *reinterpret_cast<f32x4*>(&part[wave][t][col]) = o;
            }
        }
        if constexpr (!STATES_ONLY) {
            __syncthreads();
            for (int i = tid; i < n * VL; i += 256) {
                const int t = i / VL, c = (i - t * VL) * 4;
                if (c >= columns) continue;
                f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int v = 0; v < 4; v++) o += *reinterpret_cast<const f32x4*>(&part[v][t][c]);
                o = o * p.os;
                if (sums != nullptr) {
                    f32x4* const at = reinterpret_cast<f32x4*>(sums + (first + t) * step * p.H * p.V + c0 + c);
                    if (p.sums_in) o += *at;
                    if (p.sums_out) {
                        *at = o;
                        continue;
                    }
                }
                store4<T>(out + (first + t) * step * p.out_stride_t + c0 + c, o);
            }
        }
    }
    if (p.a == 0 && total > 0) {
#pragma unroll
        for (int r = 0; r < KR; r++) S[r] = factor(S[r]);
    }
    float* to = nullptr;
    if constexpr (STATES_ONLY) to = p.local + ((int64_t)slot * p.H + h) * p.local_cells;
    else if (last && p.fin != nullptr) to = p.fin + chain * cells;
    if (to != nullptr && mine) {
#pragma unroll
        for (int r = 0; r < KR; r++)
            if (key(r) < p.K) {
                if (p.state_v == 1) __builtin_nontemporal_store(S[r], reinterpret_cast<f32x4*>(to + state_at(r)));
                else
                    for (int e = 0; e < 4; e++) to[state_at(r) + (int64_t)e * p.state_v] = S[r][e];
            }
    }
}

// blocks of 4 VL columns
template <int VL>
bool grid_of(const LinearParams& p, dim3& grid) {
    const int64_t blocks = (int64_t)p.slots * p.H * ((p.V + 4 * VL - 1) / (4 * VL));
    grid = dim3((unsigned)((blocks + 7) / 8 * 8));
    return blocks <= 0xfffff000ll / 256;  // (a launch holds at most 2^32 - 1 threads)
}

template <typename T, int KR, int VL>
int launch(const LinearParams& p, hipStream_t stream) {
    dim3 grid;
    if (!grid_of<VL>(p, grid)) return GDN_ERR_UNSUPPORTED;
    // room for one token where there is no second, so that more workgroups fit a unit: 64 states of 32 heads 49.5 us against 51.4, 32 24.5
    // against 25.5, 256 179 either way
    if (p.T == 1) hipLaunchKernelGGL((linear_tokens_kernel<T, KR, VL, 1, false>), grid, dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((linear_tokens_kernel<T, KR, VL, 16, false>), grid, dim3(256), 0, stream, p);
    return (int)hipGetLastError();
}

template <typename T>
int launch_of(const LinearParams& p, int columns, hipStream_t stream) {
    if (columns == 32) {
        if (p.K <= 64) return launch<T, 2, 8>(p, stream);
        if (p.K <= 128) return launch<T, 4, 8>(p, stream);
        return launch<T, 8, 8>(p, stream);
    }
    if (p.K <= 64) return launch<T, 8, 32>(p, stream);
    if (p.K <= 128) return launch<T, 16, 32>(p, stream);
    return launch<T, 32, 32>(p, stream);
}

template <int KR>
int launch_states(const LinearParams& p, hipStream_t stream) {
    dim3 grid;
    if (!grid_of<8>(p, grid)) return GDN_ERR_UNSUPPORTED;
    hipLaunchKernelGGL((linear_tokens_kernel<float, KR, 8, 16, true>), grid, dim3(256), 0, stream, p);
    return (int)hipGetLastError();
}

// Gradients of shared heads of q and k, added up and rounded once: a thread has 4 columns of one head.  Bound by memory: group fp32 rows
// for each one written.
template <typename T>
__global__ __launch_bounds__(256) void linear_fold_kernel(const LinearFold p) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= p.pieces) return;
    const int per_head = p.D / 4;
    const int64_t row = i / per_head, token = row / p.heads;  // token and head; b and t
    const int c = (int)(i - row * per_head) * 4;
    const float* const in = p.in + row * p.group * p.D + c;
    f32x4 sum = *reinterpret_cast<const f32x4*>(in);
    for (int j = 1; j < p.group; j++) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(in + (int64_t)j * p.D);
#pragma unroll
        for (int e = 0; e < 4; e++) sum[e] += x[e];
    }
    const int64_t b = token / p.T;
    store4<T>(static_cast<T*>(p.out) + b * p.stride_b + (token - b * p.T) * p.stride_t + (row - token * p.heads) * p.stride_h + c, sum);
}

}  // namespace

// 128 columns to a workgroup where they make one to every unit (16 states of 32 heads 11.0 us, with 32 columns 14.1), else 32: more of them
int linear_tokens_columns(int64_t chains, int V, int cus) { return V >= 128 && chains * ((V + 127) / 128) >= cus ? 128 : 32; }

int launch_linear_tokens(const LinearParams& p, int dtype, int columns, hipStream_t stream) {
    return dtype == GDN_BF16 ? launch_of<bf16_t>(p, columns, stream) : launch_of<float>(p, columns, stream);
}

int launch_linear_token_states(const LinearParams& p, hipStream_t stream) {
    if (p.K <= 64) return launch_states<2>(p, stream);
    return p.K <= 128 ? launch_states<4>(p, stream) : launch_states<8>(p, stream);
}

int launch_linear_fold(const LinearFold& p, int dtype, hipStream_t stream) {
    const int64_t blocks = (p.pieces + 255) / 256;
    if (blocks > 0xfffff000ll / 256) return GDN_ERR_UNSUPPORTED;  // (a launch holds at most 2^32 - 1 threads)
    if (dtype == GDN_BF16) hipLaunchKernelGGL(linear_fold_kernel<bf16_t>, dim3((unsigned)blocks), dim3(256), 0, stream, p);
    else hipLaunchKernelGGL(linear_fold_kernel<float>, dim3((unsigned)blocks), dim3(256), 0, stream, p);
    return (int)hipGetLastError();
}

}  // namespace gdn
