// Linear attention with a decay for each head: what its kernels share.
//
// All passes of the operator are one recurrence in three roles, x (asks), y (is stored under) and z (is stored), walked forward or
// backward in time.  With walk index i (token i from the front, or from the back), w = e^g, S [K, V]:
//     out_i = os w^{i + a} S0^T x_i + ps sum_{j <= i} w^{i - j} (x_i . y_j) z_j         S' = w^n S0 + us sum_j w^{n - a - j} y_j z_j^T
//     o  = (x, y, z) = (q, k, v)    forward,  a = 1, os = ps = scale, us = 1
//     dq =             (do, v, k)   forward,  a = 1, os = ps = scale, us = 1      state: the transpose of the forward's
//     dk =             (v, do, q)   backward, a = 0, os = 1, ps = us = scale      state: the transpose of R, below
//     dv =             (k, q, do)   backward, a = 0, os = 1, ps = us = scale      state: R = dL/dS at the last token of what is behind
// No power of w has a negative exponent anywhere, so no decay, however fast, overflows.
#pragma once

#include "gdn_chunk32_common.h"
#include "gdn_linear_hip.h"

namespace gdn {

// One walk.  Roles and their tensors [B, T, heads, .]; value head h reads head h / div of a tensor whose heads are shared.
struct LinearRole {
    const void* p;
    int64_t stride_b, stride_t, stride_h;
    int div;
};

struct LinearParams {
    LinearRole x, y, z;
    void* out;
    int64_t out_stride_b, out_stride_t, out_stride_h;
    const float* g;       // [H] or NULL
    const float* init;    // [N, H] states or NULL: what the walk starts from
    float* fin;           // [N, H] states or NULL: what it ends with (several segments: for the states' launches, not for the walk)
    float* local;         // [slots, H] states: of a segment's own tokens, then (linear_combine_kernel) what the segment starts from
    int state_k, state_v;  // element (key k, value v) of a state is at k * state_k + v * state_v
    int64_t cells;         // of a state
    // Layout of `local`.  local_keys 0: as init and fin.  Else in the order of the bf16 walk's registers (linear_fragment), padded to
    // local_keys keys and whole workgroups of columns; local_swapped: written by a walk whose keys are this one's columns, and whose
    // column local_first is this one's first key.
    int local_keys, local_swapped, local_first;
    int64_t local_cells;
    const int32_t* cu;
    int padded;           // cu: prefix sums of the valid lengths of left-padded rows
    int B, T, H, N, K, V;  // K, V: of the roles (key dim, value dim)
    int seg;              // tokens of a segment
    int nseg;             // segments per row (batches, left-padded rows); 0: packed
    int slots;            // segments there is room for
    int chain;            // the walk is the one over whole sequences (host only)
    int reverse, a;
    float os, ps, us;
    int zero;             // zeros at tokens of no sequence
    float* sums;          // fp32 [B, T, H, V] contiguous or NULL: outputs of a key dim that is walked in pieces, of heads that are added up
    int sums_in, sums_out;  // add what is there; leave the result there instead of rounding it to out
    int sums_only;          // out is not written: tokens of no sequence have their zeros in sums
    // the derivative with respect to the log-decay (gdn_linear_tangent.hip)
    LinearRole d;            // gradient of the output
    const float* init_grad;  // of the final state, or NULL
    float* local_slope;      // as local, of the state's derivative
    float* dots;             // [slots * slices, H]
};

// Segment `s` (in walk order) of sequence n: row b, first token t0, sequence length.
struct LinearSegment {
    int n = 0, s = 0, b = 0, t0 = 0, len = 0;
};

__device__ __forceinline__ int linear_segments(int len, int seg) { return max(1, (len + seg - 1) / seg); }

__device__ __forceinline__ void linear_bounds(const LinearParams& p, int n, int& b, int& t0, int& len) {
    if (p.nseg == 0) {
        b = 0;
        packed_bounds(p.cu, n, p.T, t0, len);
        return;
    }
    b = n;
    len = p.padded ? min(max(p.cu[n + 1] - p.cu[n], 0), p.T) : p.T;
    t0 = p.T - len;
}

// The first slot of packed sequence n when `slot` < 0, else the segment that `slot` holds (false: none).  A wave adds up the
// sequences' segments 64 at a time; every addition is capped, so that a malformed prefix cannot overflow.
__device__ __forceinline__ bool linear_find_packed(const LinearParams& p, int slot, LinearSegment& out, int lane, int first_of = -1, int* first_slot = nullptr) {
    int base = 0;
    for (int n0 = 0; n0 < p.N; n0 += WAVE) {
        const int n = n0 + lane;
        int t0 = 0, len = 0;
        if (n < p.N) packed_bounds(p.cu, n, p.T, t0, len);
        const int count = n < p.N ? linear_segments(len, p.seg) : 0;
        int upto = min(count, 1 << 24);
#pragma unroll
        for (int d = 1; d < WAVE; d <<= 1) {
            const int y = __shfl_up(upto, d, WAVE);
            if (lane >= d) upto = min(upto + y, 1 << 30);
        }
        if (first_slot != nullptr) {
            if (first_of < n0 + WAVE) {
                *first_slot = min(base + __shfl(upto - count, first_of - n0, WAVE), 1 << 30);
                return true;
            }
        } else {
            const uint64_t past = __builtin_amdgcn_ballot_w64(n < p.N && base + upto > slot);
            if (past != 0) {
                const int f = __builtin_ctzll(past);
                out.n = n0 + f, out.b = 0;
                out.s = slot - (base + __shfl(upto - count, f, WAVE));
                out.t0 = __shfl(t0, f, WAVE);
                out.len = __shfl(len, f, WAVE);
                return true;
            }
        }
        base = min(base + __shfl(upto, WAVE - 1, WAVE), 1 << 30);
    }
    return false;
}

// (the same in all lanes, and said so: addresses built on it stay in scalar registers)
__device__ __forceinline__ bool linear_find(const LinearParams& p, int slot, LinearSegment& out, int lane) {
    if (p.nseg == 0) {
        const bool found = linear_find_packed(p, slot, out, lane);
        out.n = __builtin_amdgcn_readfirstlane(out.n), out.s = __builtin_amdgcn_readfirstlane(out.s), out.b = 0;
        out.t0 = __builtin_amdgcn_readfirstlane(out.t0), out.len = __builtin_amdgcn_readfirstlane(out.len);
        return found;
    }
    out.n = slot / p.nseg;
    out.s = slot - out.n * p.nseg;
    if (out.n >= p.N) return false;
    linear_bounds(p, out.n, out.b, out.t0, out.len);
    return out.s < linear_segments(out.len, p.seg);
}

// The tokens of no sequence that slot `slot` looks after: [first, first + count) of row b, twice (in front of a sequence, behind the
// last one).  Every slot has the tokens at its own place in the rows, so that the zeros are written by all of them.
struct LinearGaps {
    int b, first[2], count[2];
};
__device__ __forceinline__ LinearGaps linear_gaps(const LinearParams& p, int slot) {
    LinearGaps gap;
    int row_slot = slot, begin, end;
    gap.b = 0;
    if (p.nseg == 0) {
        begin = min(max(p.cu[0], 0), p.T), end = min(max(p.cu[p.N], begin), p.T);
    } else {
        gap.b = slot / p.nseg, row_slot = slot - gap.b * p.nseg;
        if (gap.b >= p.B) gap.b = 0, row_slot = 1 << 30;
        const int len = p.padded ? min(max(p.cu[gap.b + 1] - p.cu[gap.b], 0), p.T) : p.T;
        begin = p.T - len, end = p.T;
    }
    const int64_t at = (int64_t)row_slot * p.seg;
    const int lo = (int)min(at, (int64_t)p.T), hi = (int)min(at + p.seg, (int64_t)p.T);
    gap.first[0] = lo, gap.count[0] = max(0, min(hi, begin) - lo);
    gap.first[1] = max(lo, end), gap.count[1] = max(0, hi - max(lo, end));
    return gap;
}

// zeros at those tokens, columns [c0, c0 + width) of head h; T_out has 16-byte pieces of VEC elements, width a multiple of VEC
template <typename T_out, int VEC>
__device__ __forceinline__ void linear_zero_rows(const LinearParams& p, void* to, int64_t stride_b, int64_t stride_t, int64_t stride_h, int slot, int h, int c0,
                                                 int width, int tid, int threads) {
    const LinearGaps gap = linear_gaps(p, slot);
    T_out* const out = static_cast<T_out*>(to) + gap.b * stride_b + h * stride_h + c0;
    const int pieces = width / VEC;
    for (int side = 0; side < 2; side++)
        for (int64_t i = tid; i < (int64_t)gap.count[side] * pieces; i += threads) {
            const int row = (int)(i / pieces), c = (int)(i - (int64_t)row * pieces) * VEC;
            f32x4 zero = {0.f, 0.f, 0.f, 0.f};
            *reinterpret_cast<f32x4*>(out + (int64_t)(gap.first[side] + row) * stride_t + c) = zero;
        }
}
template <typename T_out>
__device__ __forceinline__ void linear_zero_gaps(const LinearParams& p, int slot, int h, int c0, int width, int tid, int threads) {
    if (p.sums_only) linear_zero_rows<float, 4>(p, p.sums, (int64_t)p.T * p.H * p.V, (int64_t)p.H * p.V, p.V, slot, h, c0, width, tid, threads);
    else linear_zero_rows<T_out, 16 / sizeof(T_out)>(p, p.out, p.out_stride_b, p.out_stride_t, p.out_stride_h, slot, h, c0, width, tid, threads);
}

// log2 of a token's factor, from the natural logarithm that callers give; w^n from it, 1 for n = 0 also where the state forgets at once
// (-inf).  One rounding in each: relative to w^n an error of some |n g| 2^-24, as exp(g n) in fp32 has.
__device__ __forceinline__ float linear_log2(const float* g, int h) { return g == nullptr ? 0.f : g[h] * 1.4426950408889634f; }
__device__ __forceinline__ float linear_power(float g2, int n) { return n == 0 ? 1.f : __builtin_amdgcn_exp2f(g2 * (float)n); }

// A factor w = e^x that is applied again and again, as kept + rest: 1 and w - 1 where the state lasts, exact to 2^-24 of what it takes away
// then.  As one number its rounding, up to 2^-25, would come back with every application that the state remembers.
struct LinearFactor {
    float kept, rest;
    __device__ __forceinline__ explicit LinearFactor(float x) : kept(x > -0.5f ? 1.f : 0.f), rest(x > -0.5f ? expm1f(x) : expf(x)) {}
    template <typename T>
    __device__ __forceinline__ T operator()(T s) const {
        return s * rest + s * kept;
    }
};
// ... of n tokens; 1 for none also where the state forgets at once (-inf)
__device__ __forceinline__ LinearFactor linear_factor(float g, int n) { return LinearFactor(n == 0 ? 0.f : g * (float)n); }

// Where cell (key, v) lies in a state that the bf16 walk has written: [32 columns][32 keys][4 registers of 4][64 lanes][4 keys].
__device__ __forceinline__ int64_t linear_fragment(int keys, int key, int v) {
    const int r = 8 * (key >> 4 & 1) + (key & 7), lane = 32 * (key >> 3 & 1) + slice_col(v & 31);
    return ((((int64_t)(v >> 5) * (keys >> 5) + (key >> 5)) * 4 + (r >> 2)) * 64 + lane) * 4 + (r & 3);
}

// launches, gdn_linear_walk.hip and gdn_linear_tokens.hip; `states_only`, token_states (fp32): the segments' own states into p.local
int launch_linear_walk(const LinearParams& p, bool states_only, hipStream_t stream);
// gdn_linear_tokens.hip: fp32 [B, T, heads group, D], each group's rows added up, to rows of dtype
struct LinearFold {
    const float* in;
    void* out;
    int64_t stride_b, stride_t, stride_h;  // of out
    int64_t pieces;                        // of 4 columns, over all of out
    int T, heads, group, D;
};
int launch_linear_fold(const LinearFold& p, int dtype, hipStream_t stream);
int launch_linear_chain(const LinearParams& p, hipStream_t stream);  // gdn_linear_chain.hip: forward, bf16, up to 128 keys, whole sequences
int launch_linear_tokens(const LinearParams& p, int dtype, int columns, hipStream_t stream);
int launch_linear_token_states(const LinearParams& p, hipStream_t stream);
int linear_walk_keys(int K);            // keys that the bf16 walk is built for
constexpr int WALK_COLUMNS = 128;       // of the value dim that a workgroup of the bf16 walk has
int linear_tokens_columns(int64_t chains, int V, int cus);  // of the token kernel
int launch_linear_combine(const LinearParams& p, hipStream_t stream);
// gdn_linear_tangent.hip: p.dots, and dg [H] from them; with several segments their states first, p.local and p.local_slope
int launch_linear_tangent(const LinearParams& p, int dtype, bool several, float* dg, hipStream_t stream);
int linear_tangent_columns(int dtype, int V);

}  // namespace gdn
