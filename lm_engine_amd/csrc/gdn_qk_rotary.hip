// RMS norm of every head of q and k and the rotation by position, forward and backward (include/gdn_attention_hip.h).  Per row x [D]:
//     u = x r,  r = 1 / sqrt(mean(x^2) + eps),  n = u w;   (y_lo, y_hi) = (n_lo cos - n_hi sin, n_hi cos + n_lo sin)
//     dn = the inverse rotation of dy;   dw = sum_rows dn u;   du = dn w;   dx = r (du - u mean(u du))
// A row is held by L threads, one chunk each: VEC elements of the rotated dims' first half and the VEC they are rotated with, so that no
// element crosses lanes; the dims that are not rotated are halved in the same way.  q and k are one list of heads, one launch.
// Bound by memory: 4 x 4096 tokens, 16 heads of q and 2 of k of 128, bf16: forward 29 us, 151 MB at 5.1 TB/s (39 with stores through the caches),
// backward 52 us, 226 MB at 4.4 TB/s, and 4 for the sums over the partial rows.  Single tokens of 53 sequences: 4.8 us.
#include <algorithm>

#include "gdn_attention_hip.h"
#include "gdn_common.h"
#include "gdn_launch.h"

namespace gdn {

namespace {

struct RotaryParams {
    const void *x[2], *w[2], *dy[2];
    void *y[2], *dx[2];
    float* dw[2];
    int64_t x_b[2], x_t[2], x_h[2], dy_b[2], dy_t[2], dy_h[2];
    const float *cos, *sin;
    const int32_t* pos;
    int64_t pos_b;
    int heads[2];
    int T, D, R, table_rows, slices, w_bf16;
    uint32_t units;  // (token, slice of the heads)
    int bwd_slices[2];
    uint32_t bwd_units[2];
    float eps;
};

template <int VEC>
struct Vec {
    float v[VEC];
};

template <typename T, int VEC>
struct Piece {
    typedef __attribute__((ext_vector_type(VEC))) T type;
};

template <typename T, int VEC>
__device__ __forceinline__ Vec<VEC> widen(const typename Piece<T, VEC>::type& x) {
    Vec<VEC> r;
#pragma unroll
    for (int e = 0; e < VEC; e++) r.v[e] = (float)x[e];
    return r;
}

template <typename T, int VEC>
__device__ __forceinline__ void store(T* to, const Vec<VEC>& x) {
    typename Piece<T, VEC>::type r;
#pragma unroll
    for (int e = 0; e < VEC; e++) r[e] = (T)x.v[e];
    __builtin_nontemporal_store(r, reinterpret_cast<typename Piece<T, VEC>::type*>(to));
}

template <int VEC>
__device__ __forceinline__ Vec<VEC> weight_at(const void* w, int bf16, int at) {
    Vec<VEC> r;
#pragma unroll
    for (int e = 0; e < VEC; e++) r.v[e] = w == nullptr ? 1.f : bf16 ? (float)static_cast<const bf16_t*>(w)[at + e] : static_cast<const float*>(w)[at + e];
    return r;
}

template <int L>
__device__ __forceinline__ float group_sum(float x) {
#pragma unroll
    for (int off = 1; off < L; off <<= 1) x += __shfl_xor(x, off, WAVE);
    return x;
}

// What a thread has of every row: where its two pieces lie, and their angle.
template <int VEC>
struct Chunk {
    int lo, hi;
    bool there, rotated;
    __device__ __forceinline__ Chunk(const RotaryParams& p, int t) {
        const int turned = p.R / 2 / VEC;
        there = t < p.D / 2 / VEC;
        rotated = t < turned;
        lo = rotated ? t * VEC : p.R + (t - turned) * VEC;
        hi = lo + (rotated ? p.R : p.D - p.R) / 2;
        if (!there) lo = hi = 0;  // (an address that exists)
    }
    __device__ __forceinline__ void angle(const RotaryParams& p, int b, int t, Vec<VEC>& c, Vec<VEC>& s) const {
        const int at = p.pos == nullptr ? t : p.pos[b * p.pos_b + t];
        const bool known = at >= 0 && at < p.table_rows;
        const int64_t row = (int64_t)(known ? at : 0) * (p.R / 2) + (rotated ? lo : 0);
#pragma unroll
        for (int e = 0; e < VEC; e += 4) {
            const f32x4 a = *reinterpret_cast<const f32x4*>(p.cos + row + e), d = *reinterpret_cast<const f32x4*>(p.sin + row + e);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                c.v[e + i] = known ? (rotated ? a[i] : 1.f) : __builtin_nanf("");
                s.v[e + i] = known ? (rotated ? d[i] : 0.f) : __builtin_nanf("");
            }
        }
    }
};

template <typename T, int VEC>
struct Row {
    typename Piece<T, VEC>::type lo, hi;
    __device__ __forceinline__ void fetch(const T* row, const Chunk<VEC>& c) {
        lo = *reinterpret_cast<const typename Piece<T, VEC>::type*>(row + c.lo);
        hi = *reinterpret_cast<const typename Piece<T, VEC>::type*>(row + c.hi);
    }
};

__device__ __forceinline__ void unit_of(const RotaryParams& p, uint32_t unit, int& b, int& t, int& slice) {
    const uint32_t token = unit / (uint32_t)p.slices;
    slice = (int)(unit - token * (uint32_t)p.slices);
    b = (int)(token / (uint32_t)p.T);
    t = (int)(token - (uint32_t)b * (uint32_t)p.T);
}

// head `h` of the joint list: which tensor, which of its heads
__device__ __forceinline__ int64_t row_at(const int64_t (&sb)[2], const int64_t (&st)[2], const int64_t (&sh)[2], int b, int t, int which, int head) {
    return b * (which ? sb[1] : sb[0]) + t * (which ? st[1] : st[0]) + head * (which ? sh[1] : sh[0]);
}

template <typename T, int VEC, int L>
__global__ __launch_bounds__(256) void rotary_fwd_kernel(const RotaryParams p) {
    constexpr int GROUPS = 256 / L;
    const int lane = threadIdx.x % L;
    const Chunk<VEC> c(p, lane);
    const uint32_t unit = min(blockIdx.x * (uint32_t)GROUPS + threadIdx.x / L, p.units - 1);  // (past the end: the last one once more)
    int b, t, slice;
    unit_of(p, unit, b, t, slice);
    const int all = p.heads[0] + p.heads[1];
    auto source = [&](int h) {
        const int which = h >= p.heads[0];
        return static_cast<const T*>(which ? p.x[1] : p.x[0]) + row_at(p.x_b, p.x_t, p.x_h, b, t, which, which ? h - p.heads[0] : h);
    };
    Row<T, VEC> next;
    next.fetch(source(slice), c);
    Vec<VEC> cs, sn;
    c.angle(p, b, t, cs, sn);
    const Vec<VEC> wq_lo = weight_at<VEC>(p.w[0], p.w_bf16, c.lo), wq_hi = weight_at<VEC>(p.w[0], p.w_bf16, c.hi);
    const Vec<VEC> wk_lo = weight_at<VEC>(p.w[1], p.w_bf16, c.lo), wk_hi = weight_at<VEC>(p.w[1], p.w_bf16, c.hi);
    const float over = 1.f / (float)p.D;
    for (int h = slice; h < all; h += p.slices) {
        const Vec<VEC> lo = widen<T, VEC>(next.lo), hi = widen<T, VEC>(next.hi);
        if (h + p.slices < all) next.fetch(source(h + p.slices), c);
        float squares = 0.f;
#pragma unroll
        for (int e = 0; e < VEC; e++) squares += lo.v[e] * lo.v[e] + hi.v[e] * hi.v[e];
        const float r = 1.f / sqrtf(group_sum<L>(c.there ? squares : 0.f) * over + p.eps);
        const bool key = h >= p.heads[0];
        Vec<VEC> a, d;
#pragma unroll
        for (int e = 0; e < VEC; e++) {
            const float n_lo = lo.v[e] * r * (key ? wk_lo.v[e] : wq_lo.v[e]), n_hi = hi.v[e] * r * (key ? wk_hi.v[e] : wq_hi.v[e]);
            a.v[e] = n_lo * cs.v[e] - n_hi * sn.v[e];
            d.v[e] = n_hi * cs.v[e] + n_lo * sn.v[e];
        }
        if (c.there) {
            const int64_t token = (int64_t)b * p.T + t;
            T* const to = static_cast<T*>(key ? p.y[1] : p.y[0]) + (token * (key ? p.heads[1] : p.heads[0]) + (key ? h - p.heads[0] : h)) * p.D;
            store<T, VEC>(to + c.lo, a);
            store<T, VEC>(to + c.hi, d);
        }
    }
}

// q first, then k, so that one set of weights and of their gradients is in registers.
template <typename T, int VEC, int L>
__global__ __launch_bounds__(256, 4) void rotary_bwd_kernel(const RotaryParams p) {
    constexpr int GROUPS = 256 / L;
    __shared__ float total[L * 2 * VEC];
    const int lane = threadIdx.x % L;
    const Chunk<VEC> c(p, lane);
    const float over = 1.f / (float)p.D;
    for (int which = 0; which < 2; which++) {
        const int heads = p.heads[which], slices = p.bwd_slices[which];
        const int64_t x_b = p.x_b[which], x_t = p.x_t[which], x_h = p.x_h[which], dy_b = p.dy_b[which], dy_t = p.dy_t[which], dy_h = p.dy_h[which];
        const T *const xs = static_cast<const T*>(p.x[which]), *const dys = static_cast<const T*>(p.dy[which]);
        const Vec<VEC> w_lo = weight_at<VEC>(p.w[which], p.w_bf16, c.lo), w_hi = weight_at<VEC>(p.w[which], p.w_bf16, c.hi);
        float dw[2 * VEC] = {};
        const uint32_t units = p.bwd_units[which];
        // (the lanes of a group walk together, groups of a wave need not: nothing crosses groups before the end)
        for (uint32_t unit = blockIdx.x * (uint32_t)GROUPS + threadIdx.x / L; unit < units; unit += gridDim.x * (uint32_t)GROUPS) {
            const uint32_t token = unit / (uint32_t)slices;
            const int slice = (int)(unit - token * (uint32_t)slices), b = (int)(token / (uint32_t)p.T), t = (int)(token - (uint32_t)b * (uint32_t)p.T);
            const T *x_row = xs + b * x_b + t * x_t + slice * x_h, *dy_row = dys + b * dy_b + t * dy_t + slice * dy_h;
            T* to = static_cast<T*>(p.dx[which]) + ((int64_t)token * heads + slice) * p.D;
            Row<T, VEC> next, next_dy;
            next.fetch(x_row, c), next_dy.fetch(dy_row, c);
            Vec<VEC> cs, sn;
            c.angle(p, b, t, cs, sn);
            for (int h = slice; h < heads; h += slices) {
                Vec<VEC> lo = widen<T, VEC>(next.lo), hi = widen<T, VEC>(next.hi);
                const Vec<VEC> dy_lo = widen<T, VEC>(next_dy.lo), dy_hi = widen<T, VEC>(next_dy.hi);
                if (h + slices < heads) {
                    x_row += slices * x_h, dy_row += slices * dy_h;
                    next.fetch(x_row, c), next_dy.fetch(dy_row, c);
                }
                float squares = 0.f;
#pragma unroll
                for (int e = 0; e < VEC; e++) squares += lo.v[e] * lo.v[e] + hi.v[e] * hi.v[e];
                const float r = 1.f / sqrtf(group_sum<L>(c.there ? squares : 0.f) * over + p.eps);
                float product = 0.f;
                Vec<VEC> du_lo, du_hi;
#pragma unroll
                for (int e = 0; e < VEC; e++) {
                    const float dn_lo = dy_lo.v[e] * cs.v[e] + dy_hi.v[e] * sn.v[e], dn_hi = dy_hi.v[e] * cs.v[e] - dy_lo.v[e] * sn.v[e];
                    lo.v[e] *= r, hi.v[e] *= r;
                    dw[e] += dn_lo * lo.v[e], dw[VEC + e] += dn_hi * hi.v[e];
                    du_lo.v[e] = dn_lo * w_lo.v[e], du_hi.v[e] = dn_hi * w_hi.v[e];
                    product += du_lo.v[e] * lo.v[e] + du_hi.v[e] * hi.v[e];
                }
                product = group_sum<L>(c.there ? product : 0.f) * over;
#pragma unroll
                for (int e = 0; e < VEC; e++) {
                    du_lo.v[e] = r * (du_lo.v[e] - lo.v[e] * product);
                    du_hi.v[e] = r * (du_hi.v[e] - hi.v[e] * product);
                }
                if (c.there) {
                    store<T, VEC>(to + c.lo, du_lo);
                    store<T, VEC>(to + c.hi, du_hi);
                }
                to += (int64_t)slices * p.D;
            }
        }
        if (p.dw[which] == nullptr) continue;
        // the workgroup's rows: a wave's groups by shuffles, then the waves one after the other through LDS
#pragma unroll
        for (int wave = 0; wave < 256 / WAVE; wave++) {
            if ((int)threadIdx.x / WAVE == wave) {
#pragma unroll
                for (int e = 0; e < 2 * VEC; e++) {
                    float x = dw[e];
#pragma unroll
                    for (int off = L; off < WAVE; off <<= 1) x += __shfl_xor(x, off, WAVE);
                    if ((int)threadIdx.x % WAVE < L) total[lane * 2 * VEC + e] = wave == 0 ? x : total[lane * 2 * VEC + e] + x;
                }
            }
            __syncthreads();
        }
        if (threadIdx.x < L && c.there) {
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                p.dw[which][(int64_t)blockIdx.x * p.D + c.lo + e] = total[lane * 2 * VEC + e];
                p.dw[which][(int64_t)blockIdx.x * p.D + c.hi + e] = total[lane * 2 * VEC + VEC + e];
            }
        }
        __syncthreads();
    }
}

// elements of a piece: 16 bytes, or 8 where the halves do not begin at multiples of 16
int piece_of(const gdn_qk_rotary_args& a) { return a.dtype == GDN_BF16 && a.R % 16 == 0 && a.D % 16 == 0 ? 8 : 4; }
int lanes_of(const gdn_qk_rotary_args& a, int piece) {
    int L = 4;
    while (L * 2 * piece < a.D) L *= 2;
    return L;
}

// Heads of a token that one group of threads has: as many as leave the chip full, 8 at most (4 x 4096 tokens, 16 and 2 heads of 128: with 1 79 us,
// with 2 49, 4 31, 8 29, 16 33, the first two with stores through the caches).
int slices_of(const gdn_qk_rotary_args& a) {
    const int64_t rows = (int64_t)a.B * a.T * (a.heads[0] + a.heads[1]), groups = (int64_t)compute_units() * 16 * (WAVE / lanes_of(a, piece_of(a)));
    const int64_t each = std::min<int64_t>(std::max<int64_t>(rows / groups, 1), 8);
    return (int)((a.heads[0] + a.heads[1] + each - 1) / each);
}

int64_t units_of(const gdn_qk_rotary_args& a) { return (int64_t)a.B * a.T * slices_of(a); }

// The same in the backward, which goes over q and k one after the other, in pieces of four elements: with eight it has 152 registers, and three
// workgroups to a compute unit (4 x 4096 tokens, 16 and 2 heads of 128: 60 us in that many, 53 with pieces of four and four of them).
int bwd_slices_of(const gdn_qk_rotary_args& a, int which) {
    const int64_t rows = (int64_t)a.B * a.T * a.heads[which], groups = (int64_t)compute_units() * 16 * (WAVE / lanes_of(a, 4));
    const int64_t each = std::min<int64_t>(std::max<int64_t>(rows / groups, 1), 4);
    return (int)((a.heads[which] + each - 1) / each);
}
int64_t bwd_units_of(const gdn_qk_rotary_args& a, int which) { return (int64_t)a.B * a.T * bwd_slices_of(a, which); }

int check_rotary(const gdn_qk_rotary_args& a) {
    if (a.B <= 0 || a.T <= 0 || a.heads[0] <= 0 || a.heads[1] <= 0 || a.D <= 0 || a.R <= 0 || a.table_rows <= 0) return GDN_ERR_SHAPE;
    if (a.D % 8 != 0 || a.R % 8 != 0 || a.R > a.D || a.D > GDN_QK_ROTARY_MAX_D) return GDN_ERR_UNSUPPORTED;
    if ((a.dtype != GDN_BF16 && a.dtype != GDN_F32) || (a.w_dtype != GDN_BF16 && a.w_dtype != GDN_F32)) return GDN_ERR_UNSUPPORTED;
    if (a.heads[0] > 1 << 20 || a.heads[1] > 1 << 20 || (int64_t)a.B * a.T > INT32_MAX / (a.heads[0] + a.heads[1])) return GDN_ERR_UNSUPPORTED;  // rows in 32 bits
    return GDN_OK;
}

bool on(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

int check_rotary_rows(const void* p, int64_t b, int64_t t, int64_t h, int dtype) {
    const int64_t vec = dtype == GDN_BF16 ? 8 : 4;
    if (p == nullptr) return GDN_ERR_NULL;
    return on(p, 16) && b % vec == 0 && t % vec == 0 && h % vec == 0 ? GDN_OK : GDN_ERR_ALIGN;
}

int check_rotary_inputs(const gdn_qk_rotary_args& a) {
    if (const int e = check_rotary(a); e != GDN_OK) return e;
    if (a.cos == nullptr || a.sin == nullptr) return GDN_ERR_NULL;
    for (int i = 0; i < 2; i++) {
        if (const int e = check_rotary_rows(a.x[i], a.x_stride_b[i], a.x_stride_t[i], a.x_stride_h[i], a.dtype); e != GDN_OK) return e;
        if (!on(a.weight[i], a.w_dtype == GDN_BF16 ? 2 : 4)) return GDN_ERR_ALIGN;
    }
    return on(a.cos, 16) && on(a.sin, 16) && on(a.pos, 4) ? GDN_OK : GDN_ERR_ALIGN;
}

RotaryParams params_of(const gdn_qk_rotary_args& a) {
    RotaryParams p{};
    for (int i = 0; i < 2; i++) {
        p.x[i] = a.x[i], p.w[i] = a.weight[i], p.y[i] = a.y[i], p.heads[i] = a.heads[i];
        p.x_b[i] = a.x_stride_b[i], p.x_t[i] = a.x_stride_t[i], p.x_h[i] = a.x_stride_h[i];
    }
    p.cos = a.cos, p.sin = a.sin, p.pos = a.pos, p.pos_b = a.pos_stride_b;
    p.T = a.T, p.D = a.D, p.R = a.R, p.table_rows = a.table_rows, p.eps = a.eps, p.w_bf16 = a.w_dtype == GDN_BF16;
    p.slices = slices_of(a), p.units = (uint32_t)units_of(a);
    return p;
}

int blocks_of_bwd(const gdn_qk_rotary_args& a) {
    const int64_t groups = 256 / lanes_of(a, 4);
    return (int)std::min<int64_t>((std::max(bwd_units_of(a, 0), bwd_units_of(a, 1)) + groups - 1) / groups, 4 * compute_units());
}

template <bool BACKWARD, typename T, int VEC, int L>
int launch_one(const RotaryParams& p, int blocks, hipStream_t stream) {
    if constexpr (BACKWARD) hipLaunchKernelGGL((rotary_bwd_kernel<T, VEC, L>), dim3(blocks), dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((rotary_fwd_kernel<T, VEC, L>), dim3((p.units + 256 / L - 1) / (256 / L)), dim3(256), 0, stream, p);
    return (int)hipGetLastError();
}

template <bool BACKWARD, typename T, int VEC>
int launch_lanes(const RotaryParams& p, int lanes, int blocks, hipStream_t stream) {
    if (lanes == 4) return launch_one<BACKWARD, T, VEC, 4>(p, blocks, stream);
    if (lanes == 8) return launch_one<BACKWARD, T, VEC, 8>(p, blocks, stream);
    if (lanes == 16) return launch_one<BACKWARD, T, VEC, 16>(p, blocks, stream);
    if (lanes == 32) return launch_one<BACKWARD, T, VEC, 32>(p, blocks, stream);
    if constexpr (VEC == 4) return launch_one<BACKWARD, T, VEC, 64>(p, blocks, stream);
    return GDN_ERR_UNSUPPORTED;
}

template <bool BACKWARD>
int launch_rotary(const gdn_qk_rotary_args& a, const RotaryParams& p, int blocks, hipStream_t stream) {
    const int piece = BACKWARD ? 4 : piece_of(a), lanes = lanes_of(a, piece);
    if (a.dtype == GDN_F32) return launch_lanes<BACKWARD, float, 4>(p, lanes, blocks, stream);
    if constexpr (!BACKWARD)
        if (piece == 8) return launch_lanes<BACKWARD, bf16_t, 8>(p, lanes, blocks, stream);
    return launch_lanes<BACKWARD, bf16_t, 4>(p, lanes, blocks, stream);
}

}  // namespace
}  // namespace gdn

using namespace gdn;

extern "C" int gdn_qk_norm_rotary_fwd(const gdn_qk_rotary_args* a, void* stream) {
    if (a == nullptr) return GDN_ERR_NULL;
    if (const int e = check_rotary_inputs(*a); e != GDN_OK) return e;
    for (int i = 0; i < 2; i++) {
        if (a->y[i] == nullptr) return GDN_ERR_NULL;
        if (!on(a->y[i], 16)) return GDN_ERR_ALIGN;
    }
    return launch_rotary<false>(*a, params_of(*a), 0, static_cast<hipStream_t>(stream));
}

extern "C" int gdn_qk_rotary_partial_blocks(const gdn_qk_rotary_args* a) { return a == nullptr || check_rotary(*a) != GDN_OK ? 0 : blocks_of_bwd(*a); }

extern "C" int gdn_qk_norm_rotary_bwd(const gdn_qk_rotary_bwd_args* b, void* stream) {
    if (b == nullptr) return GDN_ERR_NULL;
    const gdn_qk_rotary_args& a = b->fwd;
    if (const int e = check_rotary_inputs(a); e != GDN_OK) return e;
    RotaryParams p = params_of(a);
    for (int i = 0; i < 2; i++) {
        if (const int e = check_rotary_rows(b->dy[i], b->dy_stride_b[i], b->dy_stride_t[i], b->dy_stride_h[i], a.dtype); e != GDN_OK) return e;
        if (b->dx[i] == nullptr) return GDN_ERR_NULL;
        if (!on(b->dx[i], 16) || !on(b->dweight_partial[i], 4)) return GDN_ERR_ALIGN;
        p.dy[i] = b->dy[i], p.dx[i] = b->dx[i], p.dw[i] = b->dweight_partial[i];
        p.bwd_slices[i] = bwd_slices_of(a, i), p.bwd_units[i] = (uint32_t)bwd_units_of(a, i);
        p.dy_b[i] = b->dy_stride_b[i], p.dy_t[i] = b->dy_stride_t[i], p.dy_h[i] = b->dy_stride_h[i];
    }
    if ((p.dw[0] != nullptr || p.dw[1] != nullptr) && b->partial_blocks != blocks_of_bwd(a)) return GDN_ERR_WORKSPACE;
    return launch_rotary<true>(a, p, blocks_of_bwd(a), static_cast<hipStream_t>(stream));
}
