// Attention of a few tokens per sequence over the paged cache in 8 bits (include/gdn_attention_hip.h, gdn_paged_cache.h).
//
// A workgroup has the rows (query heads of all new tokens that share a head of keys and values, 16 of them) of one sequence and one part of
// its keys; its four waves take chunks of 64 keys in turn, and their results are joined in LDS, the parts' by a second launch.
// Nothing of the cache goes through LDS: the products are S^T = K Q^T and O^T += V^T P^T on v_mfma_f32_16x16x32_bf16, whose sums over columns
// and keys may run in any order, so a lane reads 16 bytes at a time of either as they lie.  Lane (i, g) has
//     of K   key 16 (i / 4) + 4 x + i % 4 in product x, columns 64 u + 16 g .. + 15 as the operands of two products
//     of S^T row i, keys 16 g .. + 15   (4 x + r in register r of product x)
//     of V   column 16 t + i, keys 16 g .. + 15: the 16 tokens of a column that the cache holds together
// so that all 16 keys of a lane lie in one page.  Codes become bf16 with their page's scale in one instruction per pair, exactly.
// Bound by memory where there is work: 256 sequences of 4096 keys on average, 32 query heads over 4 of 128, 227 us, the codes at 4.8 TB/s.
// One token of a few sequences is bound by latency, 8 us and 2.5 to join the parts: a chain of table, scales and codes, each behind the last.
// Rounding: weights become bf16 for the second product (half a step, 2^-8 of each, at most; up to 1.7e-3 rms of the output's norm); everything else is
// fp32 up to the output's own rounding.
#include <algorithm>
#include <cmath>

#include "gdn_join.h"
#include "gdn_launch.h"
#include "gdn_paged_cache.h"

namespace gdn {

namespace {

constexpr float LOWEST = -3.402823466e38f;
constexpr int CHUNK = 64, ROWS = 16;

struct AttendParams {
    gdn_paged_cache c;
    const bf16_t* q;
    bf16_t* o;
    const int32_t* lengths;
    int64_t q_b, q_t, q_h, o_b, o_t, o_h;
    int T, G, rows, row_tiles, window, sinks, negative, splits;
    float scale;     // |scale| log2(e)
    float* part_o;   // [splits, N, HK, rows, D]
    float* part_m;   // [splits, N, HK, rows, 2]
};

__device__ __forceinline__ f32x4 mma16(const bf16x8& a, const bf16x8& b, const f32x4& c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// eight codes (two words) as bf16, times 2^e of `scale`
__device__ __forceinline__ bf16x8 widen(unsigned lo, unsigned hi, float scale) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
    return bf16x8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// bytes of NaN codes to zeros; whether there was one
__device__ __forceinline__ bool make_finite(u32x4& v) {
    unsigned any = 0;
#pragma unroll
    for (int w = 0; w < 4; w++) {
        const unsigned nan = ((v[w] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
        any |= nan;
        v[w] &= ~((nan >> 7) * 0xffu);
    }
    return any != 0;
}

__device__ __forceinline__ int lanes_min(int x) {
#pragma unroll
    for (int off = 8; off >= 1; off >>= 1) x = min(x, __shfl_xor(x, off, WAVE));
    return __builtin_amdgcn_readfirstlane(x);
}

// What row `r` of sequence n sees: keys [lo, a] and [0, sk); a < lo: none.
struct View {
    int a, lo, sk;
};
__device__ __forceinline__ View view_of(const AttendParams& p, int length, int r) {
    View v;
    const int t = p.G == 1 ? r : r / p.G;
    v.a = length - p.T + t;
    if (v.a < 0) v.a = -1, v.lo = 1 << 30, v.sk = 0;
    else v.lo = p.window == 0 ? 0 : max(0, v.a - p.window + 1), v.sk = min(p.sinks, v.lo);
    return v;
}
__device__ __forceinline__ bool sees(const View& v, int j) { return j <= v.a && (j >= v.lo || j < v.sk); }

template <int DP>
struct KeyPieces {
    u32x4 v[4][DP / 64];
};

template <int DP>
__global__ __launch_bounds__(256, DP <= 128 ? 2 : 1) void cache_attn_kernel(const AttendParams p) {
    constexpr int U = DP / 64, DT = DP / 16;
    const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), i16 = lane & 15, g = lane >> 4;
    int x = blockIdx.x;
    const int tile = x % p.row_tiles;
    x /= p.row_tiles;
    const int hk = x % p.c.HK, n = x / p.c.HK, split = blockIdx.y;
    const int P = p.c.P, D = p.c.D;
    const int length = min(max(p.lengths[n], 0), p.c.table_pages * P);
    const int row = ROWS * tile + i16, r = min(row, p.rows - 1), t = p.G == 1 ? r : r / p.G, head = hk * p.G + (r - t * p.G);

    bf16x8 q[2 * U];
    {
        const bf16_t* const from = p.q + n * p.q_b + t * p.q_t + head * p.q_h;
#pragma unroll
        for (int s = 0; s < 2 * U; s++) {
            const int col = 64 * (s >> 1) + 16 * g + 8 * (s & 1);
            const bf16x8 zero = {};
            q[s] = col < D ? *reinterpret_cast<const bf16x8*>(from + col) : zero;
            if (p.negative) q[s] = -q[s];
        }
    }
    const View view = view_of(p, length, r);
    const int lo = lanes_min(view.lo), end = -lanes_min(-view.a) + 1, full_lo = -lanes_min(-view.lo), full_end = lanes_min(view.a) + 1;
    const int near = lo & ~(CHUNK - 1), sink_end = min(-lanes_min(-view.sk), near);
    const int sink_chunks = (sink_end + CHUNK - 1) / CHUNK, chunks = sink_chunks + (end > lo ? (end - near + CHUNK - 1) / CHUNK : 0);
    const int each = (chunks + p.splits - 1) / p.splits, first = min(split * each, chunks), last = min(first + each, chunks);
    auto chunk_at = [&](int i) { return i < sink_chunks ? CHUNK * i : near + CHUNK * (i - sink_chunks); };

    const int64_t page_bytes = (int64_t)p.c.HK * P * D, head_bytes = (int64_t)hk * P * D;
    const char *const kb = static_cast<const char*>(p.c.k_codes) + head_bytes, *const vb = static_cast<const char*>(p.c.v_codes) + head_bytes;
    // the page of the 16 keys at `at`, and where they lie in it; a page that is not there: page 0 is read, and `known` is false
    auto page_at = [&](int at, int& page, int& place) {
        const int index = at / P;
        page = at < length ? cache_page(p.c, n, index) : 0;
        place = at - index * P;
        const bool known = page >= 0;
        page = max(page, 0);
        return known;
    };

    f32x4 o[DT] = {};
    float m = LOWEST, l = 0.f;
    bool taken_out = false;
    KeyPieces<DP> keys;
    float k_scale = 1.f;
    auto fetch_keys = [&](int c0) {
        int page, place;
        page_at(c0 + 16 * (i16 >> 2), page, place);
        k_scale = power_of_two(cache_scale(p.c.k_scales, (int64_t)page * p.c.HK + hk));
        const char* const from = kb + page * page_bytes + (int64_t)(place + (i16 & 3)) * D + 16 * g;
#pragma unroll
        for (int y = 0; y < 4; y++)
#pragma unroll
            for (int u = 0; u < U; u++) {
                const u32x4 zero = {0, 0, 0, 0};
                keys.v[y][u] = 64 * u + 16 * g < D ? *reinterpret_cast<const u32x4*>(from + 4 * y * D + 64 * u) : zero;
            }
    };
    if (first + wave < last) fetch_keys(chunk_at(first + wave));
    for (int i = first + wave; i < last; i += 4) {
        const int c0 = chunk_at(i);
        int page, place;
        const bool known = page_at(c0 + 16 * g, page, place);
        const float v_scale = power_of_two(cache_scale(p.c.v_scales, (int64_t)page * p.c.HK + hk));
        u32x4 values[DT];
        {
            const char* const from = vb + page * page_bytes + (int64_t)place * D + 16 * i16;
#pragma unroll
            for (int z = 0; z < DT; z++) {
                const u32x4 zero = {0, 0, 0, 0};
                values[z] = 16 * z < D ? *reinterpret_cast<const u32x4*>(from + 256 * z) : zero;
            }
        }
        f32x4 s[4];
#pragma unroll
        for (int y = 0; y < 4; y++) {
            f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int u = 0; u < U; u++) {
                acc = mma16(widen(keys.v[y][u][0], keys.v[y][u][1], k_scale), q[2 * u], acc);
                acc = mma16(widen(keys.v[y][u][2], keys.v[y][u][3], k_scale), q[2 * u + 1], acc);
            }
            s[y] = acc;
        }
        if (i + 4 < last) fetch_keys(chunk_at(i + 4));
        // (every page of a chunk that all rows see is below the length, and looked up)
        const bool full = i >= sink_chunks && c0 >= full_lo && c0 + CHUNK <= full_end && __builtin_amdgcn_ballot_w64(!known) == 0;
        float scale = p.scale;
        if (!full) {
            // (first keys end where the near ones begin)
            View own = view;
            if (i < sink_chunks) own.lo = 1 << 30, own.sk = min(view.sk, sink_end);
            scale = 1.f;
#pragma unroll
            for (int y = 0; y < 4; y++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    s[y][e] = sees(own, c0 + 16 * g + 4 * y + e) ? (known ? s[y][e] * p.scale : __builtin_nanf("")) : -__builtin_inff();
            bool found = false;
#pragma unroll
            for (int z = 0; z < DT; z++) found |= make_finite(values[z]);
            taken_out |= found;
        }
        float top = s[0][0];
#pragma unroll
        for (int y = 0; y < 4; y++)
#pragma unroll
            for (int e = 0; e < 4; e++) top = fmaxf(top, s[y][e]);
        top = fmaxf(top, __shfl_xor(top, 16, WAVE));
        top = fmaxf(top, __shfl_xor(top, 32, WAVE)) * scale;
        if (__builtin_amdgcn_ballot_w64(top > m + 8.f) != 0) {  // (as in gdn_window_attention.hip)
            const float next = fmaxf(m, top), alpha = __builtin_amdgcn_exp2f(m - next);
            m = next;
            l *= alpha;
#pragma unroll
            for (int z = 0; z < DT; z++) o[z] *= alpha;
        }
#pragma unroll
        for (int y = 0; y < 4; y++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                s[y][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[y][e], scale, -m));
                l += s[y][e];
            }
#pragma unroll
        for (int y = 0; y < 2; y++) {
            bf16x8 w;
#pragma unroll
            for (int e = 0; e < 8; e++) w[e] = (bf16_t)s[2 * y + (e >> 2)][e & 3];
#pragma unroll
            for (int z = 0; z < DT; z++) o[z] = mma16(widen(values[z][2 * y], values[z][2 * y + 1], v_scale), w, o[z]);
        }
    }
    l += __shfl_xor(l, 16, WAVE);
    l += __shfl_xor(l, 32, WAVE);

    // the waves' results: o [wave][row][column], lane (i16, g) has columns 16 z + 4 g .. + 3
    __shared__ __attribute__((aligned(16))) float shared_o[4][ROWS][DP + 4];
    __shared__ float shared_m[4][ROWS], shared_l[4][ROWS];
    if (g == 0) shared_m[wave][i16] = m, shared_l[wave][i16] = l;
#pragma unroll
    for (int z = 0; z < DT; z++) *reinterpret_cast<f32x4*>(&shared_o[wave][i16][16 * z + 4 * g]) = o[z];
    taken_out = __syncthreads_or(taken_out) != 0;
    const int out_row = threadIdx.x / 16, at = ROWS * tile + out_row;  // 16 threads a row
    if (at >= p.rows) return;
    float best = LOWEST, sum = 0.f, weight[4];
#pragma unroll
    for (int w = 0; w < 4; w++) best = fmaxf(best, shared_m[w][out_row]);
#pragma unroll
    for (int w = 0; w < 4; w++) {
        weight[w] = __builtin_amdgcn_exp2f(shared_m[w][out_row] - best);
        sum += weight[w] * shared_l[w][out_row];
    }
    const int out_t = p.G == 1 ? at : at / p.G;
    bf16_t* const to = p.o + n * p.o_b + out_t * p.o_t + (hk * p.G + at - out_t * p.G) * p.o_h;
    const int64_t part = (((int64_t)split * p.c.N + n) * p.c.HK + hk) * p.rows + at;
    const float by = sum == 0.f ? 0.f : 1.f / sum;
    const View own = view_of(p, length, at);
    if (p.splits > 1 && threadIdx.x % 16 == 0) p.part_m[2 * part] = best, p.part_m[2 * part + 1] = sum;
    for (int col = 4 * (threadIdx.x % 16); col < D; col += 64) {
        f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; w++) y += *reinterpret_cast<const f32x4*>(&shared_o[w][out_row][col]) * weight[w];
        if (taken_out) {
            // NaN codes that were taken out of chunks that not all rows see, for the rows that see them
            for (int i = first; i < last; i++) {
                const int c0 = chunk_at(i);
                if (i >= sink_chunks && c0 >= full_lo && c0 + CHUNK <= full_end) continue;
                for (int j = c0; j < min(i < sink_chunks ? min(c0 + CHUNK, sink_end) : c0 + CHUNK, own.a + 1); j++) {
                    if (!sees(own, j)) continue;
                    int page, place;
                    page_at(j, page, place);
                    const uint8_t* const codes = reinterpret_cast<const uint8_t*>(vb) + page * page_bytes + ((int64_t)(place / 16) * D + col) * 16 + place % 16;
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if ((codes[16 * e] & 0x7f) == 0x7f) y[e] = __builtin_nanf("");
                }
            }
        }
        if (p.splits > 1) *reinterpret_cast<f32x4*>(p.part_o + part * D + col) = y;
        else store4<bf16_t>(to + col, y * by);
    }
}

// The parts of a row joined: a workgroup a row.
__global__ __launch_bounds__(256) void cache_join_kernel(const AttendParams p) {
    const int64_t at = blockIdx.x;
    float m, l;
    f32x4 o;
    int col;
    if (!join_row(p.part_o, p.part_m, (int64_t)p.c.N * p.c.HK * p.rows, at, p.splits, p.c.D, m, l, o, col)) return;
    const int64_t pair = at / p.rows;
    const int r = (int)(at - pair * p.rows), n = (int)(pair / p.c.HK), hk = (int)(pair - (int64_t)n * p.c.HK), t = r / p.G;
    store4<bf16_t>(p.o + n * p.o_b + t * p.o_t + (hk * p.G + r - t * p.G) * p.o_h + col, o * (l == 0.f ? 0.f : 1.f / l));
}

int check_attend(const gdn_cache_attn_args& a) {
    if (const int e = check_cache(a.cache); e != GDN_OK) return e;
    if (a.T <= 0 || a.H <= 0 || a.H % a.cache.HK != 0 || a.window < 0 || a.sinks < 0) return GDN_ERR_SHAPE;
    const int64_t rows = (int64_t)a.T * (a.H / a.cache.HK);
    if (rows > INT32_MAX / 2 || (int64_t)a.cache.N * a.cache.HK * ((rows + ROWS - 1) / ROWS) > INT32_MAX / 2) return GDN_ERR_UNSUPPORTED;
    return GDN_OK;
}

// Parts of a sequence's keys: until there are two workgroups to a compute unit, none of them under four chunks (one for each wave), and whole
// below twelve.  Measured with 16 heads of 128 over 2, in us, for one workgroup to a compute unit, two and four: 32 sequences of 4096 keys 21.0,
// 19.8, 22.5; 64 of 2048 (over 8 heads) 42.3, 42.2, 49.6.  For parts of eight chunks, four and two: one sequence of 4096 keys 12.5, 10.7, 10.8; 8 of
// 4096 12.7, 11.1, 12.9.  The joining launch is 2.5 of it: 4 sequences of 600 keys take 8.3 us whole and 10.6 in two parts, one of 1024 13.1
// whole and 10.3 in four.
int splits_of(const gdn_cache_attn_args& a) {
    const int64_t groups = (int64_t)a.cache.N * a.cache.HK * (((int64_t)a.T * (a.H / a.cache.HK) + ROWS - 1) / ROWS);
    const int64_t room = (int64_t)a.cache.table_pages * a.cache.P, keys = a.window == 0 ? room : std::min<int64_t>(room, (int64_t)a.window + a.T + a.sinks + CHUNK);
    if (keys < 12 * CHUNK) return 1;
    return (int)std::max<int64_t>(1, std::min<int64_t>({2 * compute_units() / groups, keys / (4 * CHUNK), JOIN_MOST}));
}
uint64_t part_o_bytes(const gdn_cache_attn_args& a, int splits) { return ((uint64_t)splits * a.cache.N * a.T * a.H * a.cache.D * 4 + 255) / 256 * 256; }
uint64_t attend_bytes(const gdn_cache_attn_args& a) {
    const int splits = splits_of(a);
    return splits <= 1 ? 0 : part_o_bytes(a, splits) + (uint64_t)splits * a.cache.N * a.T * a.H * 8;
}

int check_query_rows(const void* p, int64_t b, int64_t t, int64_t h) {
    if (p == nullptr) return GDN_ERR_NULL;
    return cache_aligned(p, 16) && b % 8 == 0 && t % 8 == 0 && h % 8 == 0 ? GDN_OK : GDN_ERR_ALIGN;
}

}  // namespace
}  // namespace gdn

using namespace gdn;

extern "C" uint64_t gdn_cache_attn_workspace_bytes(const gdn_cache_attn_args* a) { return a == nullptr || check_attend(*a) != GDN_OK ? 0 : attend_bytes(*a); }

extern "C" int gdn_cache_attn(const gdn_cache_attn_args* args, void* stream) {
    if (args == nullptr) return GDN_ERR_NULL;
    const gdn_cache_attn_args& a = *args;
    if (const int e = check_attend(a); e != GDN_OK) return e;
    if (const int e = check_cache_pointers(a.cache); e != GDN_OK) return e;
    if (const int e = check_query_rows(a.q, a.q_stride_b, a.q_stride_t, a.q_stride_h); e != GDN_OK) return e;
    if (const int e = check_query_rows(a.o, a.o_stride_b, a.o_stride_t, a.o_stride_h); e != GDN_OK) return e;
    if (a.lengths == nullptr) return GDN_ERR_NULL;
    if (!cache_aligned(a.lengths, 4)) return GDN_ERR_ALIGN;
    AttendParams p{};
    p.c = a.cache, p.q = static_cast<const bf16_t*>(a.q), p.o = static_cast<bf16_t*>(a.o), p.lengths = a.lengths;
    p.q_b = a.q_stride_b, p.q_t = a.q_stride_t, p.q_h = a.q_stride_h, p.o_b = a.o_stride_b, p.o_t = a.o_stride_t, p.o_h = a.o_stride_h;
    p.T = a.T, p.G = a.H / a.cache.HK, p.rows = a.T * p.G, p.row_tiles = (p.rows + ROWS - 1) / ROWS;
    const int64_t room = (int64_t)a.cache.table_pages * a.cache.P;
    p.window = a.window >= room ? 0 : a.window, p.sinks = p.window == 0 ? 0 : a.sinks;
    p.negative = a.scale < 0, p.scale = std::fabs(a.scale) * 1.4426950408889634f;
    p.splits = splits_of(a);
    if (p.splits > 1) {
        if (a.workspace == nullptr || a.workspace_bytes < attend_bytes(a)) return GDN_ERR_WORKSPACE;
        if (!cache_aligned(a.workspace, 16)) return GDN_ERR_ALIGN;
        p.part_o = static_cast<float*>(a.workspace);
        p.part_m = reinterpret_cast<float*>(static_cast<char*>(a.workspace) + part_o_bytes(a, p.splits));
    }
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const dim3 grid((unsigned)(a.cache.N * a.cache.HK * p.row_tiles), p.splits);
    if (a.cache.D <= 64) hipLaunchKernelGGL((cache_attn_kernel<64>), grid, dim3(256), 0, st, p);
    else if (a.cache.D <= 128) hipLaunchKernelGGL((cache_attn_kernel<128>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((cache_attn_kernel<256>), grid, dim3(256), 0, st, p);
    if (const int e = (int)hipGetLastError(); e != 0 || p.splits == 1) return e;
    hipLaunchKernelGGL(cache_join_kernel, dim3((unsigned)((int64_t)a.cache.N * a.cache.HK * p.rows)), dim3(256), 0, st, p);
    return (int)hipGetLastError();
}
