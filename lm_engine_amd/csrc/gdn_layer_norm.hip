// Layer norm over the rows of a matrix, forward and backward (include/gdn_linear_hip.h):
//     xh = (x - mean) r,  r = 1 / sqrt(var + eps);   y = xh w + b
//     u = dy w;  dx = r (u - mean(u) - xh mean(u xh));   dw = sum_rows dy xh;   db = sum_rows dy
// A row is held in registers by TPR threads, PER elements each: x (and dy) are read once, the mean first, then the squares of what is
// left of it, in fp32.  The backward forms mean and r again from the row that it reads anyway, so the forward keeps nothing.
// Workgroups walk the rows, the next one on its way where there are registers for it; weight, bias and the backward's sums of dw and db
// stay in registers, and every workgroup leaves one partial row of each, added up in a fixed order.
// Bound by memory: 16384 rows of 2048, bf16: forward 25 to 29 us, 134 MB at 4.7 to 5.3 TB/s; backward 42 us, 201 MB at 4.8, and 4 for the
// sums over the partial rows.  Rows that 16-byte pieces do not fit are read in single elements: 16384 of 2049 57 us, forward and backward 154 (71
// at 2048), of 777 17 and 46 (776: 15 and 43), of 2048 at an odd address 27 and 271.  Above 8192 the backward of 1024 threads, 128 registers
// each, spills 39 to 51 of them: 2048 rows of 16384 189 us, forward and backward, where 4096 of 8192 take 93.  Two
// workgroups to a compute unit: with eight, and every thread reading its parameters for two rows, the forward took 51 us; a prefetch
// takes the backward past 256 registers, and to 72 us.
#include <algorithm>
#include <type_traits>

#include "gdn_common.h"
#include "gdn_launch.h"
#include "gdn_linear_hip.h"

namespace gdn {

namespace {

struct NormRows {
    const void *x, *dy, *weight, *bias;
    void *y, *dx;
    float *dw, *db;
    int64_t x_stride, y_stride, dy_stride, dx_stride, rows;
    int D, w_bf16;
    float eps;
};

// The elements of a row that thread t of its TPR threads has: pieces of 16 bytes, TPR pieces apart; where the row cannot be read in
// such pieces, single elements TPR apart.
template <typename T, bool VEC, int TPR, int PER>
struct Layout {
    static constexpr int E = VEC ? 16 / (int)sizeof(T) : 1;
    static __device__ __forceinline__ int index(int i, int t) { return (i / E * TPR + t) * E + i % E; }

    using Piece = std::conditional_t<!VEC, T, std::conditional_t<sizeof(T) == 2, bf16x8, f32x4>>;
    struct Row {
        Piece piece[PER / E];
    };
    // Every thread reads, past the row's end its last piece again: nothing but the loads themselves stands between them.
    static __device__ __forceinline__ void fetch(const T* row, int D, int t, Row& x) {
#pragma unroll
        for (int i = 0; i < PER; i += E) x.piece[i / E] = *reinterpret_cast<const Piece*>(row + min(index(i, t), D - E));
    }
    // as fp32, zeros past D
    static __device__ __forceinline__ void widen(const Row& x, int D, int t, float (&v)[PER]) {
#pragma unroll
        for (int i = 0; i < PER; i += E) {
            const bool there = index(i, t) < D;
#pragma unroll
            for (int e = 0; e < E; e++) {
                if constexpr (VEC) v[i + e] = there ? (float)x.piece[i / E][e] : 0.f;
                else v[i] = there ? (float)x.piece[i] : 0.f;
            }
        }
    }
    static __device__ __forceinline__ void store(T* row, int D, int t, const float (&v)[PER]) {
#pragma unroll
        for (int i = 0; i < PER; i += E) {
            const int at = index(i, t);
            if (at >= D) continue;
            if constexpr (VEC && sizeof(T) == 2) {
                bf16x8 x;
#pragma unroll
                for (int e = 0; e < E; e++) x[e] = (bf16_t)v[i + e];
                *reinterpret_cast<bf16x8*>(row + at) = x;
            } else if constexpr (VEC) {
                *reinterpret_cast<f32x4*>(row + at) = f32x4{v[i], v[i + 1], v[i + 2], v[i + 3]};
            } else {
                row[at] = (T)v[i];
            }
        }
    }
    // weight or bias, in pieces of four where they lie so that they can be read like this; `otherwise` where there is none
    static __device__ __forceinline__ void parameter(const void* p, int bf16, int D, int t, float otherwise, float (&v)[PER]) {
        if (p == nullptr) {
#pragma unroll
            for (int i = 0; i < PER; i++) v[i] = otherwise;
            return;
        }
        if (VEC && reinterpret_cast<uintptr_t>(p) % (bf16 ? 8 : 16) == 0) {
            constexpr int Q = VEC ? 4 : 1;
#pragma unroll
            for (int i = 0; i < PER; i += Q) {
                const int at = min(index(i, t), D - Q);
#pragma unroll
                for (int e = 0; e < Q; e++)
                    v[i + e] = bf16 ? (float)(*reinterpret_cast<const bf16x4*>(static_cast<const bf16_t*>(p) + at))[e]
                                    : (*reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + at))[e];
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int at = min(index(i, t), D - 1);
            v[i] = bf16 ? (float)static_cast<const bf16_t*>(p)[at] : static_cast<const float*>(p)[at];
        }
    }
};

template <int TPR>
__device__ __forceinline__ float row_sum(float x, float* shared) {
#pragma unroll
    for (int off = 1; off < (TPR < WAVE ? TPR : WAVE); off <<= 1) x += __shfl_xor(x, off, WAVE);
    if constexpr (TPR > WAVE) {  // the whole workgroup has one row
        __syncthreads();
        if (threadIdx.x % WAVE == 0) shared[threadIdx.x / WAVE] = x;
        __syncthreads();
        x = 0.f;
#pragma unroll
        for (int i = 0; i < TPR / WAVE; i++) x += shared[i];
    }
    return x;
}

// mean and 1 / sqrt(var + eps) of the row in v, whose entries past D are zero
template <typename L, int TPR, int PER>
__device__ __forceinline__ void row_statistics(const float (&v)[PER], int D, float eps, int t, float* shared, float& mean, float& r) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < PER; i++) sum += v[i];
    mean = row_sum<TPR>(sum, shared) / (float)D;
    float squares = 0.f;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const float d = L::index(i, t) < D ? v[i] - mean : 0.f;
        squares += d * d;
    }
    r = 1.f / sqrtf(row_sum<TPR>(squares, shared) / (float)D + eps);
}

template <typename T, bool VEC, int TPR, int PER>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void layer_norm_fwd_kernel(const NormRows p) {
    using L = Layout<T, VEC, TPR, PER>;
    constexpr int THREADS = TPR > 256 ? TPR : 256, RPB = THREADS / TPR;
    __shared__ float shared[THREADS / WAVE];
    const int t = threadIdx.x % TPR;
    float w[PER], b[PER];
    L::parameter(p.weight, p.w_bf16, p.D, t, 1.f, w);
    L::parameter(p.bias, p.w_bf16, p.D, t, 0.f, b);
    const int64_t step = (int64_t)gridDim.x * RPB, last = p.rows - 1;
    int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR;
    auto fetch = [&](int64_t r, typename L::Row& x) { L::fetch(static_cast<const T*>(p.x) + min(r, last) * p.x_stride, p.D, t, x); };
    constexpr bool AHEAD = VEC && TPR <= 256;  // the next row is on its way, where there are registers for it
    typename L::Row next;
    if (AHEAD) fetch(row, next);
    // (a group of threads without a row walks along on the last one: the sums cross lanes)
    for (int64_t first = (int64_t)blockIdx.x * RPB; first < p.rows; first += step, row += step) {
        float v[PER], mean, r;
        if (!AHEAD) fetch(row, next);
        L::widen(next, p.D, t, v);
        if (AHEAD) fetch(row + step, next);
        row_statistics<L, TPR>(v, p.D, p.eps, t, shared, mean, r);
#pragma unroll
        for (int i = 0; i < PER; i++) v[i] = (v[i] - mean) * r * w[i] + b[i];
        if (row < p.rows) L::store(static_cast<T*>(p.y) + row * p.y_stride, p.D, t, v);
    }
}

template <typename T, bool VEC, int TPR, int PER>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void layer_norm_bwd_kernel(const NormRows p) {
    using L = Layout<T, VEC, TPR, PER>;
    constexpr int THREADS = TPR > 256 ? TPR : 256, RPB = THREADS / TPR;
    __shared__ float shared[THREADS / WAVE];
    const int t = threadIdx.x % TPR;
    float w[PER], dw[PER] = {}, db[PER] = {};
    L::parameter(p.weight, p.w_bf16, p.D, t, 1.f, w);
    const int64_t step = (int64_t)gridDim.x * RPB, last = p.rows - 1;
    int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR;
    auto fetch = [&](int64_t r, typename L::Row& x, typename L::Row& d) {
        L::fetch(static_cast<const T*>(p.x) + min(r, last) * p.x_stride, p.D, t, x);
        L::fetch(static_cast<const T*>(p.dy) + min(r, last) * p.dy_stride, p.D, t, d);
    };
    constexpr bool AHEAD = VEC && TPR <= 256 && PER <= 16;
    typename L::Row next, next_dy;
    if (AHEAD) fetch(row, next, next_dy);
    for (int64_t first = (int64_t)blockIdx.x * RPB; first < p.rows; first += step, row += step) {
        const bool live = row < p.rows;
        float v[PER], u[PER], mean, r;
        if (!AHEAD) fetch(row, next, next_dy);
        L::widen(next, p.D, t, v);
        L::widen(next_dy, live ? p.D : 0, t, u);
        if (AHEAD) fetch(row + step, next, next_dy);
        row_statistics<L, TPR>(v, p.D, p.eps, t, shared, mean, r);
        float sum = 0.f, product = 0.f;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            v[i] = L::index(i, t) < p.D ? (v[i] - mean) * r : 0.f;  // xh
            dw[i] += u[i] * v[i], db[i] += u[i];                    // (a thread without a row has u = 0)
            u[i] *= w[i];
            sum += u[i], product += u[i] * v[i];
        }
        sum = row_sum<TPR>(sum, shared) / (float)p.D;
        product = row_sum<TPR>(product, shared) / (float)p.D;
#pragma unroll
        for (int i = 0; i < PER; i++) v[i] = r * (u[i] - sum - v[i] * product);
        if (live) L::store(static_cast<T*>(p.dx) + row * p.dx_stride, p.D, t, v);
    }
    float* const out[2] = {p.dw, p.db};
    if constexpr (TPR >= 256) {
#pragma unroll
        for (int j = 0; j < 2; j++)
            if (out[j] != nullptr) {
#pragma unroll
                for (int i = 0; i < PER; i++) {
                    const int at = L::index(i, t);
                    if (at < p.D) out[j][(int64_t)blockIdx.x * p.D + at] = j == 0 ? dw[i] : db[i];
                }
            }
    } else {
        // rows of the workgroup: lanes by shuffles, then the waves one after the other through LDS
        __shared__ float total[TPR * PER];
#pragma unroll
        for (int j = 0; j < 2; j++) {
            if (out[j] == nullptr) continue;
#pragma unroll
            for (int wave = 0; wave < THREADS / WAVE; wave++) {
                if ((int)threadIdx.x / WAVE == wave) {
#pragma unroll
                    for (int i = 0; i < PER; i++) {
                        float x = j == 0 ? dw[i] : db[i];
#pragma unroll
                        for (int off = TPR; off < WAVE; off <<= 1) x += __shfl_xor(x, off, WAVE);
                        if ((int)threadIdx.x % WAVE < TPR) total[i * TPR + t] = wave == 0 ? x : total[i * TPR + t] + x;
                    }
                }
                __syncthreads();
            }
            if ((int)threadIdx.x < TPR) {
#pragma unroll
                for (int i = 0; i < PER; i++) {
                    const int at = L::index(i, t);
                    if (at < p.D) out[j][(int64_t)blockIdx.x * p.D + at] = total[i * TPR + t];
                }
            }
            __syncthreads();
        }
    }
}

// Threads to a row, by D: 8 elements each up to a wave (512), then 16 and 32, then a workgroup of 256 or 1024.
int threads_per_row(int D) { return D <= 64 ? 8 : D <= 128 ? 16 : D <= 256 ? 32 : D <= 2048 ? 64 : D <= 8192 ? 256 : 1024; }
int rows_per_block(int D) { return std::max(1, 256 / threads_per_row(D)); }
int64_t blocks_for(int64_t rows, int D, int per_unit) {
    return std::min<int64_t>((rows + rows_per_block(D) - 1) / rows_per_block(D), (int64_t)per_unit * compute_units());
}
int backward_blocks(int64_t rows, int D) { return (int)blocks_for(rows, D, 2); }

template <bool BACKWARD, typename T, bool VEC, int TPR, int PER>
int launch_one(const NormRows& p, hipStream_t stream) {
    const dim3 threads(TPR > 256 ? TPR : 256);
    if constexpr (BACKWARD) hipLaunchKernelGGL((layer_norm_bwd_kernel<T, VEC, TPR, PER>), dim3((unsigned)backward_blocks(p.rows, p.D)), threads, 0, stream, p);
    else hipLaunchKernelGGL((layer_norm_fwd_kernel<T, VEC, TPR, PER>), dim3((unsigned)blocks_for(p.rows, p.D, 2)), threads, 0, stream, p);
    return (int)hipGetLastError();
}

template <bool BACKWARD, typename T, bool VEC>
int launch_of(const NormRows& p, hipStream_t stream) {
    if (p.D <= 64) return launch_one<BACKWARD, T, VEC, 8, 8>(p, stream);
    if (p.D <= 128) return launch_one<BACKWARD, T, VEC, 16, 8>(p, stream);
    if (p.D <= 256) return launch_one<BACKWARD, T, VEC, 32, 8>(p, stream);
    if (p.D <= 512) return launch_one<BACKWARD, T, VEC, 64, 8>(p, stream);
    if (p.D <= 1024) return launch_one<BACKWARD, T, VEC, 64, 16>(p, stream);
    if (p.D <= 2048) return launch_one<BACKWARD, T, VEC, 64, 32>(p, stream);
    if (p.D <= 4096) return launch_one<BACKWARD, T, VEC, 256, 16>(p, stream);
    if (p.D <= 8192) return launch_one<BACKWARD, T, VEC, 256, 32>(p, stream);
    return launch_one<BACKWARD, T, VEC, 1024, 16>(p, stream);
}

template <bool BACKWARD>
int launch_norm(const NormRows& p, int dtype, bool vec, hipStream_t stream) {
    if (dtype == GDN_BF16) return vec ? launch_of<BACKWARD, bf16_t, true>(p, stream) : launch_of<BACKWARD, bf16_t, false>(p, stream);
    return vec ? launch_of<BACKWARD, float, true>(p, stream) : launch_of<BACKWARD, float, false>(p, stream);
}

bool at_multiple(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// rows readable in 16-byte pieces
bool in_pieces(const void* p, int64_t stride, int64_t rows, int dtype) {
    return at_multiple(p, 16) && (rows == 1 || stride % (dtype == GDN_BF16 ? 8 : 4) == 0);
}

int check_rows_of(const void* p, int64_t stride, int64_t rows, int D, int dtype) {
    if (p == nullptr) return GDN_ERR_NULL;
    if (rows > 1 && stride < 0) return GDN_ERR_SHAPE;
    if (!at_multiple(p, dtype == GDN_BF16 ? 2 : 4)) return GDN_ERR_ALIGN;
    return GDN_OK;
}

int check_sizes(int64_t rows, int D, int dtype, int w_dtype) {
    if (rows <= 0 || D <= 0) return GDN_ERR_SHAPE;
    if (D > GDN_LAYER_NORM_MAX_D || rows > (int64_t)1 << 40) return GDN_ERR_UNSUPPORTED;
    if ((dtype != GDN_BF16 && dtype != GDN_F32) || (w_dtype != GDN_BF16 && w_dtype != GDN_F32)) return GDN_ERR_UNSUPPORTED;
    return GDN_OK;
}

}  // namespace
}  // namespace gdn

using namespace gdn;

extern "C" int gdn_layer_norm_fwd(const gdn_layer_norm_args* a, void* stream) {
    if (a == nullptr) return GDN_ERR_NULL;
    if (const int e = check_sizes(a->rows, a->D, a->dtype, a->w_dtype); e != GDN_OK) return e;
    if (const int e = check_rows_of(a->x, a->x_stride, a->rows, a->D, a->dtype); e != GDN_OK) return e;
    if (const int e = check_rows_of(a->y, a->y_stride, a->rows, a->D, a->dtype); e != GDN_OK) return e;
    if (a->rows > 1 && a->y_stride < a->D) return GDN_ERR_SHAPE;
    const size_t w_size = a->w_dtype == GDN_BF16 ? 2 : 4;
    if (!at_multiple(a->weight, w_size) || !at_multiple(a->bias, w_size)) return GDN_ERR_ALIGN;
    NormRows p{};
    p.x = a->x, p.weight = a->weight, p.bias = a->bias, p.y = a->y;
    p.x_stride = a->x_stride, p.y_stride = a->y_stride, p.rows = a->rows;
    p.D = a->D, p.w_bf16 = a->w_dtype == GDN_BF16, p.eps = a->eps;
    const bool vec = a->D % (a->dtype == GDN_BF16 ? 8 : 4) == 0 && in_pieces(a->x, a->x_stride, a->rows, a->dtype) && in_pieces(a->y, a->y_stride, a->rows, a->dtype);
    return launch_norm<false>(p, a->dtype, vec, static_cast<hipStream_t>(stream));
}

extern "C" int gdn_layer_norm_partial_blocks(int64_t rows, int32_t D, int32_t dtype) {
    if (check_sizes(rows, D, dtype, GDN_F32) != GDN_OK) return 0;
    return backward_blocks(rows, D);
}

extern "C" int gdn_layer_norm_bwd(const gdn_layer_norm_bwd_args* a, void* stream) {
    if (a == nullptr) return GDN_ERR_NULL;
    if (const int e = check_sizes(a->rows, a->D, a->dtype, a->w_dtype); e != GDN_OK) return e;
    if (const int e = check_rows_of(a->x, a->x_stride, a->rows, a->D, a->dtype); e != GDN_OK) return e;
    if (const int e = check_rows_of(a->dy, a->dy_stride, a->rows, a->D, a->dtype); e != GDN_OK) return e;
    if (const int e = check_rows_of(a->dx, a->dx_stride, a->rows, a->D, a->dtype); e != GDN_OK) return e;
    if (a->rows > 1 && a->dx_stride < a->D) return GDN_ERR_SHAPE;
    if (!at_multiple(a->weight, a->w_dtype == GDN_BF16 ? 2 : 4) || !at_multiple(a->dweight_partial, 4) || !at_multiple(a->dbias_partial, 4)) return GDN_ERR_ALIGN;
    if ((a->dweight_partial != nullptr || a->dbias_partial != nullptr) && a->partial_blocks != backward_blocks(a->rows, a->D)) return GDN_ERR_WORKSPACE;
    NormRows p{};
    p.x = a->x, p.dy = a->dy, p.weight = a->weight, p.dx = a->dx, p.dw = a->dweight_partial, p.db = a->dbias_partial;
    p.x_stride = a->x_stride, p.dy_stride = a->dy_stride, p.dx_stride = a->dx_stride, p.rows = a->rows;
    p.D = a->D, p.w_bf16 = a->w_dtype == GDN_BF16, p.eps = a->eps;
    const bool vec = a->D % (a->dtype == GDN_BF16 ? 8 : 4) == 0 && in_pieces(a->x, a->x_stride, a->rows, a->dtype) && in_pieces(a->dy, a->dy_stride, a->rows, a->dtype)
                     && in_pieces(a->dx, a->dx_stride, a->rows, a->dtype);
    return launch_norm<true>(p, a->dtype, vec, static_cast<hipStream_t>(stream));
}
