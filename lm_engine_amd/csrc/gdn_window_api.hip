// C ABI of softmax attention over a window (include/gdn_attention_hip.h): argument checks, and how a call is cut.  What lives on the device
// (cu_seqlens) is clamped by the kernels.
#include <algorithm>
#include <cmath>

#include "gdn_join.h"
#include "gdn_launch.h"
#include "gdn_window_attention.h"

namespace gdn {

namespace {

bool on16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

int check_rows(const void* p, int64_t b, int64_t t, int64_t h, int heads, int dtype) {
    const int64_t vec = dtype == GDN_BF16 ? 8 : 4;
    if (p == nullptr) return GDN_ERR_NULL;
    if (!on16(p) || b % vec != 0 || t % vec != 0 || h % vec != 0) return GDN_ERR_ALIGN;
    // the bytes from a base to the rows that a wave loads, or to 128 keys, are counted in 31 bits (row_offsets_fit, at each kernel's tiles)
    if (t < 0 || t > MOST_APART || h < 0 || h > MOST_HEADS / heads) return GDN_ERR_UNSUPPORTED;
    return GDN_OK;
}

int check_shape(const gdn_window_attn_args& a) {
    if (a.B <= 0 || a.T <= 0 || a.S <= 0 || a.H <= 0 || a.HK <= 0 || a.D <= 0 || a.N <= 0 || a.H % a.HK != 0) return GDN_ERR_SHAPE;
    if (a.window < 0 || a.sinks < 0) return GDN_ERR_SHAPE;
    const bool padded = (a.flags & GDN_FLAG_LEFT_PADDED) != 0;
    if (padded && a.cu_seqlens == nullptr) return GDN_ERR_NULL;
    if (a.cu_seqlens != nullptr && a.T != a.S) return GDN_ERR_SHAPE;
    if (a.cu_seqlens != nullptr && !padded) {
        if (a.B != 1) return GDN_ERR_VARLEN;
    } else if (a.N != a.B) {
        return GDN_ERR_SHAPE;
    }
    if (a.dtype != GDN_BF16 && a.dtype != GDN_F32) return GDN_ERR_UNSUPPORTED;
    if (a.D % 8 != 0 || a.D > 256 || (a.flags & ~GDN_FLAG_LEFT_PADDED)) return GDN_ERR_UNSUPPORTED;
    // what the kernels hold in 32 bits: positions with a window's length on top, rows of a head of k and v, work items
    const int64_t rows = (int64_t)a.T * (a.H / a.HK);
    if (a.S >= 1 << 29 || rows >= 1 << 30 || a.N > 1 << 28) return GDN_ERR_UNSUPPORTED;
    if ((int64_t)a.B * a.HK * ((std::max<int64_t>(rows, a.S) + 15) / 16) >= 1 << 30) return GDN_ERR_UNSUPPORTED;
    return GDN_OK;
}

// (rows of a tile are taken apart into tokens and heads)
bool backward_fits(const gdn_window_attn_args& a) { return a.dtype != GDN_BF16 || a.H / a.HK <= MOST_GROUP; }

int check_inputs(const gdn_window_attn_args& a) {
    int e;
    if ((e = check_rows(a.q, a.q_stride_b, a.q_stride_t, a.q_stride_h, a.H, a.dtype)) != GDN_OK) return e;
    if ((e = check_rows(a.k, a.k_stride_b, a.k_stride_t, a.k_stride_h, a.HK, a.dtype)) != GDN_OK) return e;
    if ((e = check_rows(a.v, a.v_stride_b, a.v_stride_t, a.v_stride_h, a.HK, a.dtype)) != GDN_OK) return e;
    if ((e = check_rows(a.o, a.o_stride_b, a.o_stride_t, a.o_stride_h, a.H, a.dtype)) != GDN_OK) return e;
    if (reinterpret_cast<uintptr_t>(a.lse) % 4 != 0 || reinterpret_cast<uintptr_t>(a.cu_seqlens) % 4 != 0) return GDN_ERR_ALIGN;
    return GDN_OK;
}

WindowParams params_of(const gdn_window_attn_args& a) {
    WindowParams p{};
    p.q = {a.q, a.q_stride_b, a.q_stride_t, a.q_stride_h};
    p.k = {a.k, a.k_stride_b, a.k_stride_t, a.k_stride_h};
    p.v = {a.v, a.v_stride_b, a.v_stride_t, a.v_stride_h};
    p.o = {a.o, a.o_stride_b, a.o_stride_t, a.o_stride_h};
    p.lse = a.lse, p.cu = a.cu_seqlens, p.padded = (a.flags & GDN_FLAG_LEFT_PADDED) != 0;
    p.B = a.B, p.T = a.T, p.S = a.S, p.H = a.H, p.HK = a.HK, p.G = a.H / a.HK, p.D = a.D, p.N = a.N;
    p.rows = a.T * p.G, p.by_g = (uint32_t)((((uint64_t)1 << 32) + p.G - 1) / p.G);
    p.window = a.window >= a.S ? 0 : a.window, p.sinks = p.window == 0 ? 0 : std::min(a.sinks, a.S);
    p.scale = a.scale, p.negative = a.scale < 0, p.c = std::fabs(a.scale) * 1.4426950408889634f;
    p.splits = 1;
    return p;
}

// Parts that the keys of a block of rows are cut into: until two workgroups a compute unit are there, none of them under 128 keys, and whole below
// 384.  The joining launch costs 4.5 us, 64 keys one (bf16, 128 columns): 1 x 300 tokens of 4 heads over one take 14.4 us whole and 16.1 in two
// parts, 1 x 777 of 2 over one with a window of 512 21.2 whole, 19.8 in two and 17.8 in four (256 columns: 39.7, 30.6, 25.7, still falling at the last of
// them; parts under 128 keys were not measured).
int splits_of(const gdn_window_attn_args& a) {
    const int64_t rows = (int64_t)a.T * (a.H / a.HK), edge = a.dtype == GDN_BF16 ? WINDOW_ROWS : WINDOW_ROWS_F32;
    const int64_t groups = (int64_t)a.B * a.HK * ((rows + edge - 1) / edge);
    const int64_t tokens = (edge + a.H / a.HK - 1) / (a.H / a.HK);
    const int64_t keys = a.window == 0 ? a.S : std::min<int64_t>(a.S, (int64_t)a.window + tokens + a.sinks);
    if (keys < 384) return 1;
    return (int)std::max<int64_t>(1, std::min<int64_t>({2 * compute_units() / groups, keys / 128, JOIN_MOST}));
}

uint64_t part_o_bytes(const gdn_window_attn_args& a, int splits) {
    return splits <= 1 ? 0 : ((uint64_t)splits * a.B * a.T * a.H * a.D * 4 + 255) / 256 * 256;
}
uint64_t workspace_of(const gdn_window_attn_args& a) {
    const int splits = splits_of(a);
    return splits <= 1 ? 0 : part_o_bytes(a, splits) + (uint64_t)splits * a.B * a.T * a.H * 8;
}

// The parts in which rows beyond the window are shared out for a sequence's first keys: about one workgroup a compute unit in all, 256 rows or
// more to each.  (Half or twice as many: backward 617 us each instead of 611 at 4 x 4096, 16 heads of 128 over 2, window 1024, 4 first keys.)
int pieces_of(const WindowParams& p, int dtype) {
    // (first keys of more places than there are tokens: sequences of which most are first keys, which the blocks' own walks take as they come)
    if (dtype != GDN_BF16 || p.sinks == 0 || (int64_t)p.N * p.sinks > (int64_t)p.B * p.S) return 0;
    const int64_t blocks = (int64_t)p.N * p.HK * ((p.sinks + WINDOW_FIRST_KEYS - 1) / WINDOW_FIRST_KEYS), rows = (int64_t)p.T * p.G;
    return (int)std::max<int64_t>(1, std::min<int64_t>(compute_units() / blocks, (rows + 255) / 256));
}
int first_keys_of(const WindowParams& p) { return (p.sinks + WINDOW_FIRST_KEYS - 1) / WINDOW_FIRST_KEYS * WINDOW_FIRST_KEYS; }

// The shares that the rows of a block of keys are cut into, where few heads of k and v leave fewer blocks than the chip has room for: with a window
// one workgroup to a compute unit (up to 64 columns three), without one twice that (four), since then blocks have from all rows to none;
// 4 tiles of rows or more to each.  Backward in us, whole and shared: 1 x 4096, 16 heads of 128 over 2, window 512 215 and 117 (4 shares; 2: 146, 8:
// 131); the same with 64 columns 136 and 72 (6; 2: 90, 8: 80); 4 x 4096 of them without a window 1536 and 1190 (2; 4: 1209); 1 x 777, 4 heads of 128
// over one, window 512 114 and 51 (8 tiles or more to each: 57).  What it costs: the sums once more in fp32, and a launch of about 4 us.
int shares_of(const WindowParams& p, int dtype) {
    if (dtype != GDN_BF16) return 1;
    const int64_t blocks = (int64_t)p.B * p.HK * ((p.S + window_keys(p.D) - 1) / window_keys(p.D));
    const int64_t tokens = p.window == 0 ? p.T : std::min(p.T, p.window + window_keys(p.D)), least = p.D > 128 ? 128 : 256;
    const int64_t wanted = (p.D <= 64 ? p.window == 0 ? 4 : 3 : p.window == 0 ? 2 : 1) * compute_units();
    return (int)std::max<int64_t>(1, std::min<int64_t>({wanted / blocks, tokens * p.G / least, 16}));
}
uint64_t shares_bytes(const WindowParams& p, int shares) { return shares <= 1 ? 0 : (uint64_t)shares * p.B * p.HK * p.S * 2 * p.D * 4; }

uint64_t delta_bytes(const gdn_window_attn_args& a) { return ((uint64_t)a.B * a.T * a.H * 4 + 255) / 256 * 256; }
uint64_t backward_bytes(const gdn_window_attn_args& a, const WindowParams& p) {
    const int pieces = pieces_of(p, a.dtype), shares = shares_of(p, a.dtype);
    const uint64_t first = pieces == 0 ? 0 : (uint64_t)p.N * p.HK * (pieces + shares) * first_keys_of(p) * 2 * p.D * 4;
    return delta_bytes(a) + shares_bytes(p, shares) + first;
}

}  // namespace
}  // namespace gdn

using namespace gdn;

extern "C" int gdn_attention_abi_version(void) { return GDN_ATTENTION_ABI_VERSION; }

extern "C" uint64_t gdn_window_attn_workspace_bytes(const gdn_window_attn_args* a) { return a == nullptr || check_shape(*a) != GDN_OK ? 0 : workspace_of(*a); }

extern "C" int gdn_window_attn_fwd(const gdn_window_attn_args* args, void* stream) {
    if (args == nullptr) return GDN_ERR_NULL;
    const gdn_window_attn_args& a = *args;
    if (const int e = check_shape(a); e != GDN_OK) return e;
    if (const int e = check_inputs(a); e != GDN_OK) return e;
    WindowParams p = params_of(a);
    p.splits = splits_of(a);
    if (p.splits > 1) {
        if (a.workspace == nullptr || a.workspace_bytes < workspace_of(a)) return GDN_ERR_WORKSPACE;
        if (!on16(a.workspace)) return GDN_ERR_ALIGN;
        p.part_o = static_cast<float*>(a.workspace);
        p.part_m = reinterpret_cast<float*>(static_cast<char*>(a.workspace) + part_o_bytes(a, p.splits));
    }
    const int edge = a.dtype == GDN_BF16 ? WINDOW_ROWS : WINDOW_ROWS_F32;
    p.blocks = (p.rows + edge - 1) / edge;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    return a.dtype == GDN_BF16 ? launch_window_fwd(p, st) : launch_window_fwd_f32(p, st);
}

extern "C" uint64_t gdn_window_attn_bwd_workspace_bytes(const gdn_window_attn_bwd_args* b) {
    return b == nullptr || check_shape(b->fwd) != GDN_OK || !backward_fits(b->fwd) ? 0 : backward_bytes(b->fwd, params_of(b->fwd));
}

extern "C" int gdn_window_attn_bwd(const gdn_window_attn_bwd_args* args, void* stream) {
    if (args == nullptr) return GDN_ERR_NULL;
    const gdn_window_attn_bwd_args& b = *args;
    const gdn_window_attn_args& a = b.fwd;
    if (const int e = check_shape(a); e != GDN_OK) return e;
    if (!backward_fits(a)) return GDN_ERR_UNSUPPORTED;
    if (const int e = check_inputs(a); e != GDN_OK) return e;
    if (a.lse == nullptr) return GDN_ERR_NULL;
    if (const int e = check_rows(b.dout, b.dout_stride_b, b.dout_stride_t, b.dout_stride_h, a.H, a.dtype); e != GDN_OK) return e;
    if (const int e = check_rows(b.dq, b.dq_stride_b, b.dq_stride_t, b.dq_stride_h, a.H, a.dtype); e != GDN_OK) return e;
    if (const int e = check_rows(b.dk, b.dk_stride_b, b.dk_stride_t, b.dk_stride_h, a.HK, a.dtype); e != GDN_OK) return e;
    if (const int e = check_rows(b.dv, b.dv_stride_b, b.dv_stride_t, b.dv_stride_h, a.HK, a.dtype); e != GDN_OK) return e;
    WindowParams p = params_of(a);
    if (pieces_of(p, a.dtype) > 0 && (uint64_t)p.N * p.HK * first_keys_of(p) > INT32_MAX) return GDN_ERR_UNSUPPORTED;  // a workgroup each, in the join
    if (b.workspace == nullptr || b.workspace_bytes < backward_bytes(a, p)) return GDN_ERR_WORKSPACE;
    if (!on16(b.workspace)) return GDN_ERR_ALIGN;
    p.dout = {b.dout, b.dout_stride_b, b.dout_stride_t, b.dout_stride_h};
    p.dq = {b.dq, b.dq_stride_b, b.dq_stride_t, b.dq_stride_h};
    p.dk = {b.dk, b.dk_stride_b, b.dk_stride_t, b.dk_stride_h};
    p.dv = {b.dv, b.dv_stride_b, b.dv_stride_t, b.dv_stride_h};
    p.delta = static_cast<float*>(b.workspace);
    p.pieces = pieces_of(p, a.dtype), p.first_keys = first_keys_of(p);
    p.shares = shares_of(p, a.dtype);
    p.part_all = reinterpret_cast<float*>(static_cast<char*>(b.workspace) + delta_bytes(a));
    p.part_dk = reinterpret_cast<float*>(static_cast<char*>(b.workspace) + delta_bytes(a) + shares_bytes(p, p.shares));
    const hipStream_t st = static_cast<hipStream_t>(stream);
    return a.dtype == GDN_BF16 ? launch_window_bwd(p, st) : launch_window_bwd_f32(p, st);
}
