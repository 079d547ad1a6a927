// C ABI of linear attention with a decay for each head (include/gdn_linear_hip.h): argument checks, how long sequences are cut, and
// the walks that make up a call.  What lives on the device (cu_seqlens) is clamped by the kernels.
#include <algorithm>

#include "gdn_launch.h"
#include "gdn_linear_common.h"

namespace gdn {

namespace {

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

int check_rows(const void* p, int64_t b, int64_t t, int64_t h, int dtype) {
    const int64_t vec = dtype == GDN_BF16 ? 8 : 4;
    if (p == nullptr) return GDN_ERR_NULL;
    if (!aligned16(p) || b % vec != 0 || t % vec != 0 || h % vec != 0) return GDN_ERR_ALIGN;
    if (t < 0 || t > 1 << 24) return GDN_ERR_UNSUPPORTED;  // the bytes of a chunk of 64 tokens are counted in 32 bits, without a sign
    return GDN_OK;
}

int check_shape(const gdn_linear_attn_args& a) {
    if (a.B <= 0 || a.T <= 0 || a.H <= 0 || a.K <= 0 || a.V <= 0 || a.N <= 0) return GDN_ERR_SHAPE;
    if (a.qk_heads < 0 || (a.qk_heads > 0 && a.H % a.qk_heads != 0)) return GDN_ERR_SHAPE;
    const bool padded = (a.flags & GDN_FLAG_LEFT_PADDED) != 0;
    if (padded && a.cu_seqlens == nullptr) return GDN_ERR_NULL;
    if (a.cu_seqlens != nullptr && !padded) {
        if (a.B != 1) return GDN_ERR_VARLEN;
    } else if (a.N != a.B) {
        return GDN_ERR_SHAPE;
    }
    if (a.dtype != GDN_BF16 && a.dtype != GDN_F32) return GDN_ERR_UNSUPPORTED;
    if (a.K % 8 != 0 || a.K > 256 || a.V % 8 != 0) return GDN_ERR_UNSUPPORTED;
    if (a.flags & ~(GDN_FLAG_LEFT_PADDED | GDN_FLAG_ZERO_PADDING)) return GDN_ERR_UNSUPPORTED;
    // sizes that the kernels hold in 32 bits: token indexes, heads (a grid dimension), cells of a state
    if (a.T > 1 << 30 || a.H > 65535 || a.V > 1 << 20) return GDN_ERR_UNSUPPORTED;
    return GDN_OK;
}

int check_inputs(const gdn_linear_attn_args& a) {
    int e;
    if ((e = check_rows(a.q, a.q_stride_b, a.q_stride_t, a.q_stride_h, a.dtype)) != GDN_OK) return e;
    if ((e = check_rows(a.k, a.k_stride_b, a.k_stride_t, a.k_stride_h, a.dtype)) != GDN_OK) return e;
    if ((e = check_rows(a.v, a.v_stride_b, a.v_stride_t, a.v_stride_h, a.dtype)) != GDN_OK) return e;
    if (!aligned16(a.h0) || !aligned16(a.ht)) return GDN_ERR_ALIGN;
    if (reinterpret_cast<uintptr_t>(a.g) % 4 != 0 || reinterpret_cast<uintptr_t>(a.cu_seqlens) % 4 != 0) return GDN_ERR_ALIGN;
    return GDN_OK;
}

// How the sequences are cut: `seg` tokens to a segment.
struct Cut {
    int seg, nseg, slots;
    bool chain;    // bf16: whole sequences, split over the columns of the value dim (gdn_linear_chain.hip)
    bool several;  // a sequence may have more than one segment: their states come first
};

// Workgroups that a launch should have (`wanted`), and the shortest segment that is worth another one.
Cut cut_sequences(const gdn_linear_attn_args& a, int64_t slices, int64_t wanted, int shortest) {
    const bool packed = a.cu_seqlens != nullptr && !(a.flags & GDN_FLAG_LEFT_PADDED);
    const int64_t tokens = (int64_t)a.B * a.T, work = a.H * slices;
    int64_t seg = (tokens * work + wanted - 1) / wanted;
    seg = std::max<int64_t>((seg + 63) / 64 * 64, shortest);
    Cut c;
    c.chain = false;
    if (seg >= a.T) {
        c.seg = (a.T + 63) / 64 * 64, c.nseg = packed ? 0 : 1, c.slots = a.N, c.several = false;
        return c;
    }
    if (packed) {
        c.seg = (int)seg, c.nseg = 0, c.slots = a.T / c.seg + a.N;
    } else {
        const int64_t n = (a.T + seg - 1) / seg;
        c.seg = (int)(((a.T + n - 1) / n + 63) / 64 * 64);
        c.nseg = (a.T + c.seg - 1) / c.seg;
        c.slots = a.N * c.nseg;
    }
    c.several = true;
    return c;
}

// The walk runs two workgroups to a compute unit (one where the keys number more than 128), and as many are wanted: half as many or twice as
// many, forward and backward, 4 x 4096 tokens of 16 heads of 128 371 | 349 | 414 us, 6 x 1500 of 16 / 8 heads of 64 186 | 156 | 173; forward, 32768
// of 16 heads of 128 235 | 201 | 230, 65536 of 32 heads of 128 x 256 1548 | 1309 | 1317; 4 x 4096 of 2 heads of 256 x 512 1005 | 585 | 512 (which
// twice as many would suit).  No segment under 128 tokens: 777 tokens of 2 heads of 256 x 512 38 us, with 64 41, with 256 51.
// fp32 walks of 256 threads, four to a unit, no segment under 64 tokens: forward and backward, half | as it is | twice as many, 4 x 1024 tokens of
// 16 heads of 128 1308 | 1093 | 1079 us, 1 x 2048 681 | 592 | 605; 256 tokens of 2 heads of 64 135 us, with segments of 128 231.
Cut cut_segments(const gdn_linear_attn_args& a) {
    const int width = a.dtype == GDN_BF16 ? WALK_COLUMNS : 32, cus = compute_units();
    const int64_t slices = (a.V + width - 1) / width;
    if (a.dtype == GDN_BF16) return cut_sequences(a, slices, a.K <= 128 ? 2 * cus : cus, 128);
    return cut_sequences(a, slices, 4 * cus, 64);
}

// The forward in bf16: where segments would take three launches, a walk over whole sequences, 32 columns to a workgroup and one
// workgroup to a compute unit, may be faster.  It takes 6 us and 1.25 us a chunk (0.8 up to 64 keys) of the longest sequence, for each
// round of workgroups; the segments 30 us and 18 ns (7) for every chunk of 64 rows and 128 columns.  Measured, whole sequences against
// segments, us, with 16 heads of 128: 4 x 1024 tokens 28 | 50, 4 x 2048 46 | 67, 8 x 4096 190 | 202, 2 x 4096 75 | 69,
// 1 x 2048 40 | 37, 1 x 4096 72 | 52; 1 x 65536 with 32 heads and V = 256 1320 | 1297; 16 heads of 64: 16 x 1024 39 | 63, 4 x 4096 60 | 64.
// It errs where a second round of workgroups is half empty (6 x 2048 tokens of 16 heads of 128, 88 | 107).
// In the backward, where the states serve two walks, the two were level (370 us at 4 x 4096 tokens), and it has segments alone.  How
// long the longest of packed sequences is lives on the device: it may have nearly all tokens (11 of them in 32768 tokens: 404 | 257).
Cut cut_forward(const gdn_linear_attn_args& a) {
    const Cut segments = cut_segments(a);
    if (a.dtype != GDN_BF16 || a.K > 128 || !segments.several) return segments;
    const int64_t chunks = (a.T + 63) / 64, cus = compute_units();
    const int64_t rounds = ((int64_t)a.N * a.H * ((a.V + 31) / 32) + cus - 1) / cus;
    const int64_t blocks = (int64_t)a.B * a.H * chunks * ((a.V + 127) / 128);
    if (rounds * (6000 + (a.K <= 64 ? 800 : 1250) * chunks) >= 30000 + (a.K <= 64 ? 7 : 18) * blocks) return segments;  // ns
    Cut c;
    c.seg = (a.T + 63) / 64 * 64, c.nseg = a.cu_seqlens != nullptr && !(a.flags & GDN_FLAG_LEFT_PADDED) ? 0 : 1;
    c.slots = a.N, c.chain = true, c.several = false;
    return c;
}

// cells of a state between the launches: bf16 in the order of the walk's registers (whole workgroups), fp32 as it is
int64_t local_cells(int dtype, int K, int V) {
    if (dtype != GDN_BF16) return (int64_t)K * V;
    return (int64_t)linear_walk_keys(K) * ((V + WALK_COLUMNS - 1) / WALK_COLUMNS * WALK_COLUMNS);
}

uint64_t states_bytes(const gdn_linear_attn_args& a, const Cut& c, int64_t cells) {
    return c.several ? ((uint64_t)c.slots * a.H * cells * 4 + 255) / 256 * 256 : 0;
}

// what every walk over these sequences has in common
LinearParams base_params(const gdn_linear_attn_args& a, const Cut& c) {
    LinearParams p{};
    p.g = a.g;
    p.cu = a.cu_seqlens;
    p.padded = (a.flags & GDN_FLAG_LEFT_PADDED) != 0;
    p.B = a.B, p.T = a.T, p.H = a.H, p.N = a.N;
    p.cells = (int64_t)a.K * a.V;
    p.seg = c.seg, p.nseg = c.nseg, p.slots = c.slots, p.chain = c.chain;
    p.zero = (a.flags & GDN_FLAG_ZERO_PADDING) != 0;
    return p;
}

int heads_shared(const gdn_linear_attn_args& a) { return a.qk_heads == 0 ? 1 : a.H / a.qk_heads; }

struct Roles {
    LinearRole q, k, v;
};
Roles roles_of(const gdn_linear_attn_args& a) {
    const int div = heads_shared(a);
    return {{a.q, a.q_stride_b, a.q_stride_t, a.q_stride_h, div},
            {a.k, a.k_stride_b, a.k_stride_t, a.k_stride_h, div},
            {a.v, a.v_stride_b, a.v_stride_t, a.v_stride_h, 1}};
}

// S [K, V] as it lies: keys are the first index
void natural(LinearParams& p, int K, int V) { p.K = K, p.V = V, p.state_k = V, p.state_v = 1; }

int run(const LinearParams& p, int dtype, bool states_only, hipStream_t stream) {
    if (p.chain) return launch_linear_chain(p, stream);
    if (dtype == GDN_BF16) return launch_linear_walk(p, states_only, stream);
    return states_only ? launch_linear_token_states(p, stream) : launch_linear_tokens(p, dtype, 32, stream);
}

// the states that the segments start from, into p.local: their own, then the sums, and p.fin
int run_states(LinearParams& p, int dtype, hipStream_t stream) {
    p.local_cells = local_cells(dtype, p.K, p.V);
    p.local_keys = dtype == GDN_BF16 ? linear_walk_keys(p.K) : 0;
    if (const int e = run(p, dtype, true, stream); e != GDN_OK) return e;
    return launch_linear_combine(p, stream);
}

const void* offset(const void* p, int64_t elements, int dtype) { return static_cast<const char*>(p) + elements * (dtype == GDN_BF16 ? 2 : 4); }

constexpr int KEYS = 256;  // of a walk at most

// outputs of dq and dk in fp32: where their keys, the value dim, are walked in pieces, and where value heads share a head of q and k
uint64_t sums_bytes(const gdn_linear_attn_args& a) {
    return a.V > KEYS || heads_shared(a) > 1 ? ((uint64_t)a.B * a.T * a.H * a.K * 4 + 255) / 256 * 256 : 0;
}

uint64_t dots_bytes(const gdn_linear_attn_args& a, const Cut& c) {
    const int columns = linear_tangent_columns(a.dtype, a.V);
    return ((uint64_t)c.slots * ((a.V + columns - 1) / columns) * a.H * 4 + 255) / 256 * 256;
}

// The backward's workspace: states that the segments start from (the forward's, their gradients, with dg the derivatives), partial
// outputs, the parts of dg.
struct BackwardSpace {
    uint64_t forward, gradients, slope, sums, dots;
    bool own_orientation;  // the forward's states are written with the value dim as keys, as dq reads them
    BackwardSpace(const gdn_linear_attn_args& a, const Cut& c, bool dg) {
        own_orientation = a.dtype == GDN_BF16 && !dg;
        const int64_t natural_cells = (int64_t)a.K * a.V;
        forward = states_bytes(a, c, own_orientation ? local_cells(a.dtype, std::min(a.V, KEYS), a.K) : natural_cells);
        gradients = states_bytes(a, c, local_cells(a.dtype, a.K, a.V));
        slope = dg ? states_bytes(a, c, natural_cells) : 0;
        sums = sums_bytes(a);
        dots = dg ? dots_bytes(a, c) : 0;
    }
    uint64_t total() const { return forward + gradients + slope + sums + dots; }
};

// dq or dk: a walk whose keys are the value dim, 256 of them at a time; p.x, p.y, p.z and the states are set for all of them.
// own_states: the states that the segments start from are formed here, in p.local, 256 keys after 256 keys as well
int run_transposed(LinearParams p, const gdn_linear_attn_args& a, bool own_states, float* sums, hipStream_t stream) {
    const LinearParams whole = p;
    for (int first = 0; first < a.V; first += KEYS) {
        p.K = std::min(KEYS, a.V - first), p.V = a.K;
        p.state_k = 1, p.state_v = a.V;
        p.x.p = offset(whole.x.p, first, a.dtype), p.y.p = offset(whole.y.p, first, a.dtype);
        p.init = whole.init == nullptr ? nullptr : whole.init + first;
        p.sums = sums;
        p.sums_in = first > 0, p.sums_only = heads_shared(a) > 1, p.sums_out = p.sums_only || first + KEYS < a.V;
        if (p.sums_only) p.zero = 1;  // (all rows of sums are added up)
        if (own_states) {
            if (const int e = run_states(p, a.dtype, stream); e != GDN_OK) return e;
        } else if (p.local != nullptr && p.local_keys != 0) {
            p.local_swapped = 1, p.local_first = first;
        } else if (p.local != nullptr) {
            p.local = whole.local + first;
        }
        if (const int e = run(p, a.dtype, false, stream); e != GDN_OK) return e;
    }
    if (!p.sums_only) return GDN_OK;
    LinearFold f;
    f.in = sums, f.out = p.out, f.stride_b = p.out_stride_b, f.stride_t = p.out_stride_t, f.stride_h = p.out_stride_h;
    f.T = a.T, f.heads = a.qk_heads, f.group = heads_shared(a), f.D = a.K;
    f.pieces = (int64_t)a.B * a.T * a.qk_heads * (a.K / 4);
    return launch_linear_fold(f, a.dtype, stream);
}

}  // namespace
}  // namespace gdn

using namespace gdn;

extern "C" int gdn_linear_abi_version(void) { return GDN_LINEAR_ABI_VERSION; }

extern "C" uint64_t gdn_linear_attn_workspace_bytes(const gdn_linear_attn_args* a) {
    if (a == nullptr || check_shape(*a) != GDN_OK) return 0;
    return states_bytes(*a, cut_forward(*a), local_cells(a->dtype, a->K, a->V));
}

extern "C" int gdn_linear_attn_chunk_fwd(const gdn_linear_attn_args* args, void* stream) {
    if (args == nullptr) return GDN_ERR_NULL;
    const gdn_linear_attn_args& a = *args;
    if (const int e = check_shape(a); e != GDN_OK) return e;
    if (const int e = check_inputs(a); e != GDN_OK) return e;
    if (const int e = check_rows(a.o, a.o_stride_b, a.o_stride_t, a.o_stride_h, a.dtype); e != GDN_OK) return e;
    if (a.h0 != nullptr && a.ht == a.h0) return GDN_ERR_UNSUPPORTED;
    const Cut c = cut_forward(a);
    if (c.several && (a.workspace == nullptr || a.workspace_bytes < states_bytes(a, c, local_cells(a.dtype, a.K, a.V)))) return GDN_ERR_WORKSPACE;
    if (c.several && !aligned16(a.workspace)) return GDN_ERR_ALIGN;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const Roles r = roles_of(a);
    LinearParams p = base_params(a, c);
    natural(p, a.K, a.V);
    p.x = r.q, p.y = r.k, p.z = r.v;
    p.out = a.o, p.out_stride_b = a.o_stride_b, p.out_stride_t = a.o_stride_t, p.out_stride_h = a.o_stride_h;
    p.init = a.h0, p.fin = a.ht;
    p.reverse = 0, p.a = 1, p.os = p.ps = a.scale, p.us = 1.f;
    if (c.several) {
        p.local = static_cast<float*>(a.workspace);
        if (const int e = run_states(p, a.dtype, st); e != GDN_OK) return e;
        p.fin = nullptr;
    }
    return run(p, a.dtype, false, st);
}

extern "C" int gdn_linear_attn_recurrent_fwd(const gdn_linear_attn_args* args, void* stream) {
    if (args == nullptr) return GDN_ERR_NULL;
    const gdn_linear_attn_args& a = *args;
    if (const int e = check_shape(a); e != GDN_OK) return e;
    if (const int e = check_inputs(a); e != GDN_OK) return e;
    if (const int e = check_rows(a.o, a.o_stride_b, a.o_stride_t, a.o_stride_h, a.dtype); e != GDN_OK) return e;
    const Roles r = roles_of(a);
    Cut c;
    c.seg = (a.T + 63) / 64 * 64, c.nseg = a.cu_seqlens != nullptr && !(a.flags & GDN_FLAG_LEFT_PADDED) ? 0 : 1, c.slots = a.N, c.chain = false, c.several = false;
    LinearParams p = base_params(a, c);
    natural(p, a.K, a.V);
    p.x = r.q, p.y = r.k, p.z = r.v;
    p.out = a.o, p.out_stride_b = a.o_stride_b, p.out_stride_t = a.o_stride_t, p.out_stride_h = a.o_stride_h;
    p.init = a.h0, p.fin = a.ht;
    p.reverse = 0, p.a = 1, p.os = p.ps = a.scale, p.us = 1.f;
    return launch_linear_tokens(p, a.dtype, linear_tokens_columns((int64_t)a.N * a.H, a.V, compute_units()), static_cast<hipStream_t>(stream));
}

extern "C" uint64_t gdn_linear_attn_bwd_workspace_bytes(const gdn_linear_attn_bwd_args* b) {
    if (b == nullptr || check_shape(b->fwd) != GDN_OK) return 0;
    const gdn_linear_attn_args& a = b->fwd;
    return BackwardSpace(a, cut_segments(a), b->dg != nullptr).total();
}

extern "C" int gdn_linear_attn_bwd(const gdn_linear_attn_bwd_args* args, void* stream) {
    if (args == nullptr) return GDN_ERR_NULL;
    const gdn_linear_attn_bwd_args& b = *args;
    const gdn_linear_attn_args& a = b.fwd;
    if (const int e = check_shape(a); e != GDN_OK) return e;
    if (const int e = check_inputs(a); e != GDN_OK) return e;
    if (const int e = check_rows(b.dout, b.dout_stride_b, b.dout_stride_t, b.dout_stride_h, a.dtype); e != GDN_OK) return e;
    if (const int e = check_rows(b.dq, b.dq_stride_b, b.dq_stride_t, b.dq_stride_h, a.dtype); e != GDN_OK) return e;
    if (const int e = check_rows(b.dk, b.dk_stride_b, b.dk_stride_t, b.dk_stride_h, a.dtype); e != GDN_OK) return e;
    if (const int e = check_rows(b.dv, b.dv_stride_b, b.dv_stride_t, b.dv_stride_h, a.dtype); e != GDN_OK) return e;
    if (!aligned16(b.dht) || !aligned16(b.dh0)) return GDN_ERR_ALIGN;
    if (b.dg != nullptr && a.g == nullptr) return GDN_ERR_NULL;
    const Cut c = cut_segments(a);
    const BackwardSpace space(a, c, b.dg != nullptr);
    if (space.total() > 0) {
        if (b.workspace == nullptr || b.workspace_bytes < space.total()) return GDN_ERR_WORKSPACE;
        if (!aligned16(b.workspace)) return GDN_ERR_ALIGN;
    }
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const Roles r = roles_of(a);
    const LinearRole d = {b.dout, b.dout_stride_b, b.dout_stride_t, b.dout_stride_h, 1};
    char* const ws = static_cast<char*>(b.workspace);
    float* const gradients_at = reinterpret_cast<float*>(ws + space.forward);
    float* const sums_at = space.sums == 0 ? nullptr : reinterpret_cast<float*>(ws + space.forward + space.gradients + space.slope);

    LinearParams s = base_params(a, c);  // of the forward's states
    natural(s, a.K, a.V);
    s.x = r.q, s.y = r.k, s.z = r.v;
    s.init = a.h0;
    s.reverse = 0, s.a = 1, s.os = s.ps = a.scale, s.us = 1.f;
    LinearParams t = s;  // of their gradients
    t.x = r.k, t.y = r.q, t.z = d;
    t.init = b.dht;
    t.reverse = 1, t.a = 0, t.os = 1.f, t.ps = t.us = a.scale;
    if (b.dg != nullptr) {  // (which leaves the states that the segments start from as well)
        LinearParams u = s;
        u.d = d, u.init_grad = b.dht;
        if (c.several) u.local = reinterpret_cast<float*>(ws), u.local_slope = gradients_at + space.gradients / 4;
        u.dots = reinterpret_cast<float*>(ws + space.forward + space.gradients + space.slope + space.sums);
        if (const int e = launch_linear_tangent(u, a.dtype, c.several, b.dg, st); e != GDN_OK) return e;
    }
    if (c.several) {
        s.local = reinterpret_cast<float*>(ws), t.local = gradients_at;
        s.local_cells = (int64_t)a.K * a.V;  // (natural, as the tangent's launch leaves them)
        if (b.dg == nullptr && !space.own_orientation)
            if (const int e = run_states(s, a.dtype, st); e != GDN_OK) return e;
        t.fin = b.dh0;
        if (const int e = run_states(t, a.dtype, st); e != GDN_OK) return e;
    }
    t.out = b.dv, t.out_stride_b = b.dv_stride_b, t.out_stride_t = b.dv_stride_t, t.out_stride_h = b.dv_stride_h;
    t.fin = c.several ? nullptr : b.dh0;
    if (const int e = run(t, a.dtype, false, st); e != GDN_OK) return e;
    LinearParams k = t;
    k.x = r.v, k.y = d, k.z = r.q;
    k.out = b.dk, k.out_stride_b = b.dk_stride_b, k.out_stride_t = b.dk_stride_t, k.out_stride_h = b.dk_stride_h;
    k.fin = nullptr;
    if (const int e = run_transposed(k, a, false, sums_at, st); e != GDN_OK) return e;
    LinearParams q = s;
    q.x = d, q.y = r.v, q.z = r.k;
    q.out = b.dq, q.out_stride_b = b.dq_stride_b, q.out_stride_t = b.dq_stride_t, q.out_stride_h = b.dq_stride_h;
    q.fin = nullptr;
    return run_transposed(q, a, c.several && space.own_orientation, sums_at, st);
}
