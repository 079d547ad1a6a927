// The paged cache in 8 bits: writing new tokens, and reading back what it holds (include/gdn_attention_hip.h, gdn_paged_cache.h).
// A workgroup has one head of one touched page, of the keys or of the values.  A thread's task is 16 tokens of 8 columns, which it
// holds in registers from the one reading to the stores: a piece of 16 bytes (fp32: two) of each row comes in; keys leave as 8 codes of
// each row, values as 16 tokens' codes of each column.
// A page's scale 2^e is the smallest with which its largest magnitude is at most 448, and grows with its tokens: older codes then move by whole
// exponents, which is exact but where they reach e4m3's smallest one.  A code is off by at most half a step, 2^-4 of the value: the choice of the
// format.
// Bound by memory: 8 prompts of up to 4001 tokens, 8 heads of 128, bf16: written in 50 us (197 MB, 3.9 TB/s: reads and writes mixed, with
// pages that end inside prompts), read back in 35 (227 MB, most of the codes
// still in the last cache).  A token of each of 256 sequences, 8 heads of 128: 6 us, latency.
#include <algorithm>

#include "gdn_launch.h"
#include "gdn_paged_cache.h"

namespace gdn {

namespace {

struct WriteParams {
    gdn_paged_cache c;
    const void *x[2];
    int64_t b[2], t[2], h[2];
    const int32_t *start, *cu;
    int B, T, padded, each;  // each: pages that a row's tokens can lie in (0: packed sequences, which are looked up)
};

// One thread's 16 tokens x 8 columns.
struct Block {
    float v[16][8];
};

// Eight columns of a row, as they are in memory; rows of new tokens are read once, past the caches.
template <typename T>
struct RowPiece;
template <>
struct RowPiece<bf16_t> {
    bf16x8 x = {};
    __device__ __forceinline__ void load(const bf16_t* p) { x = __builtin_nontemporal_load(reinterpret_cast<const bf16x8*>(p)); }
    __device__ __forceinline__ float operator[](int e) const { return (float)x[e]; }
};
template <>
struct RowPiece<float> {
    f32x4 x = {0.f, 0.f, 0.f, 0.f}, y = {0.f, 0.f, 0.f, 0.f};
    __device__ __forceinline__ void load(const float* p) {
        x = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(p)), y = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(p + 4));
    }
    __device__ __forceinline__ float operator[](int e) const { return e < 4 ? x[e & 3] : y[e & 3]; }
};

// pages that the tokens [start, start + len) of a sequence lie in; what lies in front of position 0 or past the table is cut off before
__device__ __forceinline__ int pages_of(int start, int len, int P) { return len > 0 ? (start + len - 1) / P - start / P + 1 : 0; }

// A sequence's new tokens: `start` the position of the first, `first` its place in the row (b), after the cut.
struct NewTokens {
    int b, first, start, len;
};
__device__ __forceinline__ NewTokens new_tokens(const WriteParams& p, int n) {
    NewTokens s;
    if (p.cu == nullptr) {
        s.b = n, s.first = 0, s.len = p.T;
    } else if (p.padded) {
        s.b = n, s.len = min(max(p.cu[n + 1] - p.cu[n], 0), p.T), s.first = p.T - s.len;
    } else {
        s.b = 0;
        packed_bounds(p.cu, n, p.T, s.first, s.len);
    }
    const int64_t start = p.start[n], end = min(start + s.len, (int64_t)p.c.table_pages * p.c.P);
    const int dropped = (int)min(max(-start, (int64_t)0), (int64_t)s.len);
    s.first += dropped;
    s.start = (int)max(start, (int64_t)0);
    s.len = (int)max(min(end - s.start, (int64_t)s.len), (int64_t)0);
    if (start > end) s.len = 0;
    return s;
}

// which sequence's which page `slot` is, for packed sequences: their pages are counted 64 sequences at a time
__device__ __forceinline__ bool find_page(const WriteParams& p, int slot, int& n, int& nth) {
    const int lane = threadIdx.x % WAVE;
    int base = 0;
    for (int n0 = 0; n0 < p.c.N; n0 += WAVE) {
        int count = 0;
        if (n0 + lane < p.c.N) {
            const NewTokens s = new_tokens(p, n0 + lane);
            count = pages_of(s.start, s.len, p.c.P);
        }
        int upto = min(count, 1 << 24);
#pragma unroll
        for (int d = 1; d < WAVE; d <<= 1) {
            const int y = __shfl_up(upto, d, WAVE);
            if (lane >= d) upto = min(upto + y, 1 << 30);
        }
        const uint64_t past = __builtin_amdgcn_ballot_w64(base + upto > slot);
        if (past != 0) {
            const int f = __builtin_ctzll(past);
            n = n0 + f, nth = slot - (base + __shfl(upto - count, f, WAVE));
            return true;
        }
        base = min(base + __shfl(upto, WAVE - 1, WAVE), 1 << 30);
    }
    return false;
}

template <typename T>
__global__ __launch_bounds__(256) void cache_write_kernel(const WriteParams p) {
    const int slot = blockIdx.x / p.c.HK, h = blockIdx.x - slot * p.c.HK, value = blockIdx.y, P = p.c.P, D = p.c.D;
    int n, nth;
    if (p.each > 0) n = slot / p.each, nth = slot - n * p.each;
    else if (!find_page(p, slot, n, nth)) return;
    const NewTokens s = new_tokens(p, n);
    const int index = s.start / P + nth;
    if (nth >= pages_of(s.start, s.len, P)) return;
    const int page = cache_page(p.c, n, index);
    if (page < 0) return;
    const int o0 = max(s.start - index * P, 0), o1 = min(s.start + s.len - index * P, P);  // places of the page that are written
    const int64_t head = (int64_t)page * p.c.HK + h;
    uint8_t* const codes = static_cast<uint8_t*>(value ? p.c.v_codes : p.c.k_codes) + head * P * D;
    uint8_t* const scales = value ? p.c.v_scales : p.c.k_scales;
    // the row that would lie at place 0 of the page
    const T* const rows = static_cast<const T*>(value ? p.x[1] : p.x[0]) + s.b * (value ? p.b[1] : p.b[0]) + h * (value ? p.h[1] : p.h[0]);
    const int64_t stride = value ? p.t[1] : p.t[0], row0 = (int64_t)s.first + (index * P - s.start);

    const int columns = D / 8, tasks = P / 16 * columns;
    auto load = [&](int task, RowPiece<T> (&x)[16]) {
        const int g = task / columns, c = task - g * columns;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const int o = 16 * g + i;
            x[i] = RowPiece<T>();
            if (o >= o0 && o < o1) x[i].load(rows + (row0 + o) * stride + 8 * c);
        }
    };
    RowPiece<T> x[16];
    float top = 0.f;
    const int threads = blockDim.x;
    for (int task = threadIdx.x; task < tasks; task += threads) {
        load(task, x);
#pragma unroll
        for (int i = 0; i < 16; i++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float a = fabsf(x[i][e]);
                top = fmaxf(top, a < __builtin_inff() ? a : 0.f);
            }
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, WAVE));
    __shared__ float tops[4];
    if (threads > WAVE) {
        if (threadIdx.x % WAVE == 0) tops[threadIdx.x / WAVE] = top;
        __syncthreads();
        for (int w = 0; w < threads / WAVE; w++) top = fmaxf(top, tops[w]);
    }
    int e = cache_exponent(top);
    const int before = cache_scale(scales, head);
    if (o0 > 0) e = max(e, before);
    const bool again = o0 > 0 && e > before;  // what the page held is rounded to its new scale
    const float by = power_of_two(-e), shift = power_of_two(max(before - e, -126));
    __syncthreads();  // (the old scale has been read by all)
    if (threadIdx.x == 0) scales[head] = (uint8_t)(e + 127);

    auto rescale = [&](unsigned w) {
        const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
        return cache_codes(lo.x * shift, lo.y * shift, hi.x * shift, hi.y * shift);
    };
    auto one = [&](float v) { return fabsf(v) < __builtin_inff() ? v * by : __builtin_nanf(""); };
    for (int task = threadIdx.x; task < tasks; task += threads) {
        const int g = task / columns, c = task - g * columns;
        if (16 * g >= o1 || (!again && 16 * g + 16 <= o0)) continue;
        if (tasks > threads) load(task, x);
        if (value) {
            u32x4* const to = reinterpret_cast<u32x4*>(codes) + g * D + 8 * c;
            const bool whole = 16 * g >= o0 && 16 * g + 16 <= o1;
#pragma unroll
            for (int d = 0; d < 8; d++) {
                u32x4 out;
                if (!whole) out = to[d];
#pragma unroll
                for (int w = 0; w < 4; w++) {
                    const unsigned fresh = cache_codes(one(x[4 * w][d]), one(x[4 * w + 1][d]), one(x[4 * w + 2][d]), one(x[4 * w + 3][d]));
                    if (whole) {
                        out[w] = fresh;
                        continue;
                    }
                    const unsigned held = out[w], older = again ? rescale(held) : held;
                    unsigned r = 0;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int o = 16 * g + 4 * w + i;
                        r |= (o < o0 ? older : o < o1 ? fresh : held) & (0xffu << (8 * i));
                    }
                    out[w] = r;
                }
                to[d] = out;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const int o = 16 * g + i;
                u32x2* const to = reinterpret_cast<u32x2*>(codes + (int64_t)o * D + 8 * c);
                if (o >= o0 && o < o1) {
                    u32x2 out;
                    out.x = cache_codes(one(x[i][0]), one(x[i][1]), one(x[i][2]), one(x[i][3]));
                    out.y = cache_codes(one(x[i][4]), one(x[i][5]), one(x[i][6]), one(x[i][7]));
                    *to = out;
                } else if (again && o < o0) {
                    u32x2 out = *to;
                    out.x = rescale(out.x), out.y = rescale(out.y);
                    *to = out;
                }
            }
        }
    }
}

// A few new tokens per sequence: a group of L lanes, eight columns each, has one head of one touched page, keys or values, and goes over its new
// rows; nothing of the page is read but the scale, unless that grows (by the page's workgroup of cache_write_kernel a token of 256 sequences took
// 16.7 us, now 6.2).  Values leave code by code (16 bytes apart).
template <typename T, int L>
__global__ __launch_bounds__(256) void cache_append_kernel(const WriteParams p) {
    const int P = p.c.P, D = p.c.D, lane = threadIdx.x % L;
    const int64_t unit = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L, slot = unit / (2 * p.c.HK);
    const int rest = (int)(unit - slot * 2 * p.c.HK), value = rest & 1, h = rest >> 1;
    const int n = (int)(slot / p.each), nth = (int)(slot - (int64_t)n * p.each), col = 8 * lane;
    if (n >= p.c.N) return;
    const NewTokens s = new_tokens(p, n);
    const int index = s.start / P + nth;
    if (nth >= pages_of(s.start, s.len, P)) return;
    const int page = cache_page(p.c, n, index);
    const int o0 = max(s.start - index * P, 0), o1 = min(s.start + s.len - index * P, P);
    const T* const rows = static_cast<const T*>(value ? p.x[1] : p.x[0]) + s.b * (value ? p.b[1] : p.b[0]) + h * (value ? p.h[1] : p.h[0]) + col;
    const int64_t stride = value ? p.t[1] : p.t[0], row0 = (int64_t)s.first + (index * P - s.start);
    const bool there = col < D;
    RowPiece<T> first;
    float top = 0.f;
    for (int o = o1 - 1; o >= o0; o--) {
        first = RowPiece<T>();
        if (there) first.load(rows + (row0 + o) * stride);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float a = fabsf(first[e]);
            top = fmaxf(top, a < __builtin_inff() ? a : 0.f);
        }
    }
#pragma unroll
    for (int off = L / 2; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, WAVE));
    if (page < 0) return;
    const int64_t head = (int64_t)page * p.c.HK + h;
    uint8_t* const codes = static_cast<uint8_t*>(value ? p.c.v_codes : p.c.k_codes) + head * P * D;
    uint8_t* const scales = value ? p.c.v_scales : p.c.k_scales;
    int e = cache_exponent(top);
    if (o0 > 0) {
        const int before = cache_scale(scales, head);
        if (e > before) {
            const float shift = power_of_two(max(before - e, -126));
            auto rescale = [&](unsigned w) {
                const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
                return cache_codes(lo.x * shift, lo.y * shift, hi.x * shift, hi.y * shift);
            };
            if (there && value) {
                for (int g = 0; 16 * g < o0; g++) {
                    uint8_t* const from = codes + ((int64_t)g * D + col) * 16;
                    for (int x = 0; x < 32; x++) {  // four tokens of a column; those from o0 on are written anew, or hold nothing
                        unsigned* const to = reinterpret_cast<unsigned*>(from) + x;
                        const int held = min(o0 - 16 * g - 4 * (x & 3), 4);
                        const unsigned keep = held >= 4 ? ~0u : held <= 0 ? 0 : (1u << (8 * held)) - 1, w = *to;
                        *to = (rescale(w) & keep) | (w & ~keep);
                    }
                }
            } else if (there) {
                for (int o = 0; o < o0; o++) {
                    u32x2* const to = reinterpret_cast<u32x2*>(codes + (int64_t)o * D + col);
                    u32x2 w = *to;
                    w.x = rescale(w.x), w.y = rescale(w.y);
                    *to = w;
                }
            }
        }
        e = max(e, before);
    }
    if (lane == 0) scales[head] = (uint8_t)(e + 127);
    if (!there) return;
    const float by = power_of_two(-e);
    auto one = [&](float v) { return fabsf(v) < __builtin_inff() ? v * by : __builtin_nanf(""); };
    for (int o = o0; o < o1; o++) {
        RowPiece<T> x = first;
        if (o > o0) x.load(rows + (row0 + o) * stride);
        const unsigned lo = cache_codes(one(x[0]), one(x[1]), one(x[2]), one(x[3])), hi = cache_codes(one(x[4]), one(x[5]), one(x[6]), one(x[7]));
        if (value) {
            uint8_t* const to = codes + ((int64_t)(o / 16) * D + col) * 16 + o % 16;
#pragma unroll
            for (int i = 0; i < 4; i++) to[16 * i] = (uint8_t)(lo >> (8 * i)), to[16 * (i + 4)] = (uint8_t)(hi >> (8 * i));
        } else {
            u32x2 out;
            out.x = lo, out.y = hi;
            *reinterpret_cast<u32x2*>(codes + (int64_t)o * D + col) = out;
        }
    }
}

struct ReadParams {
    gdn_paged_cache c;
    void* out[2];
    const int32_t* lengths;
    int T, each;
};

template <typename T>
__device__ __forceinline__ void store_row(T* p, const float (&v)[8]) {
    if constexpr (sizeof(T) == 2) {
        bf16x8 x;
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = (bf16_t)v[e];
        __builtin_nontemporal_store(x, reinterpret_cast<bf16x8*>(p));
    } else {
        __builtin_nontemporal_store(f32x4{v[0], v[1], v[2], v[3]}, reinterpret_cast<f32x4*>(p));
        __builtin_nontemporal_store(f32x4{v[4], v[5], v[6], v[7]}, reinterpret_cast<f32x4*>(p + 4));
    }
}

template <typename T>
__global__ __launch_bounds__(256) void cache_read_kernel(const ReadParams p) {
    const int value = blockIdx.z, h = blockIdx.y, P = p.c.P, D = p.c.D;
    const int n = blockIdx.x / p.each, index = blockIdx.x - n * p.each;
    const int length = min(p.lengths[n], p.T), first = index * P;
    const int page = first < length ? cache_page(p.c, n, index) : -1;
    const int64_t head = (int64_t)max(page, 0) * p.c.HK + h;
    const uint8_t* const codes = static_cast<const uint8_t*>(value ? p.c.v_codes : p.c.k_codes) + head * P * D;
    const float by = page < 0 ? __builtin_nanf("") : power_of_two(cache_scale(value ? p.c.v_scales : p.c.k_scales, head));
    T* const out = static_cast<T*>(value ? p.out[1] : p.out[0]) + ((int64_t)n * p.T * p.c.HK + h) * D;
    const int columns = D / 8, tasks = P / 16 * columns;
    for (int task = threadIdx.x; task < tasks; task += blockDim.x) {
        const int g = task / columns, c = task - g * columns;
        Block x;
        if (value) {
            u32x4 in[8];
#pragma unroll
            for (int d = 0; d < 8; d++) in[d] = *(reinterpret_cast<const u32x4*>(codes) + g * D + 8 * c + d);
#pragma unroll
            for (int d = 0; d < 8; d++)
#pragma unroll
                for (int w = 0; w < 4; w++) {
                    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)in[d][w], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)in[d][w], true);
                    x.v[4 * w][d] = lo.x, x.v[4 * w + 1][d] = lo.y, x.v[4 * w + 2][d] = hi.x, x.v[4 * w + 3][d] = hi.y;
                }
        } else {
            u32x2 in[16];
#pragma unroll
            for (int i = 0; i < 16; i++) in[i] = *reinterpret_cast<const u32x2*>(codes + (int64_t)(16 * g + i) * D + 8 * c);
#pragma unroll
            for (int i = 0; i < 16; i++)
#pragma unroll
                for (int w = 0; w < 2; w++) {
                    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)in[i][w], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)in[i][w], true);
                    x.v[i][4 * w] = lo.x, x.v[i][4 * w + 1] = lo.y, x.v[i][4 * w + 2] = hi.x, x.v[i][4 * w + 3] = hi.y;
                }
        }
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const int t = first + 16 * g + i;
            if (t >= p.T) continue;
            const bool there = t < length;
#pragma unroll
            for (int e = 0; e < 8; e++) x.v[i][e] = there ? x.v[i][e] * by : 0.f;
            store_row<T>(out + (int64_t)t * p.c.HK * D + 8 * c, x.v[i]);
        }
    }
}

// Up to here rows of tokens go by cache_append_kernel, past it by cache_write_kernel.  Both, in us, at 64 sequences, 2 heads of 128, bf16: a token each
// 4.1 and 10.9, 4 tokens 5.9 and 11.2, 8 8.9 and 11.5, 16 12.4 and 11.8, 32 20.2 and 11.8; 4 sequences, 8 heads, 16 tokens 18.7 and 11.2.
constexpr int APPEND_TOKENS = 8;

int threads_for(int P, int D) { return std::min(256, (P / 16 * (D / 8) + WAVE - 1) / WAVE * WAVE); }

int check_rows16(const void* p, int64_t b, int64_t t, int64_t h, int dtype) {
    const int64_t vec = dtype == GDN_BF16 ? 8 : 4;
    if (p == nullptr) return GDN_ERR_NULL;
    return cache_aligned(p, 16) && b % vec == 0 && t % vec == 0 && h % vec == 0 ? GDN_OK : GDN_ERR_ALIGN;
}

}  // namespace
}  // namespace gdn

using namespace gdn;

extern "C" int gdn_cache_write(const gdn_cache_write_args* a, void* stream) {
    if (a == nullptr) return GDN_ERR_NULL;
    if (const int e = check_cache(a->cache); e != GDN_OK) return e;
    if (a->B <= 0 || a->T <= 0) return GDN_ERR_SHAPE;
    const bool padded = (a->flags & GDN_FLAG_LEFT_PADDED) != 0;
    if (padded && a->cu_seqlens == nullptr) return GDN_ERR_NULL;
    if (a->cu_seqlens != nullptr && !padded) {
        if (a->B != 1) return GDN_ERR_VARLEN;
    } else if (a->cache.N != a->B) {
        return GDN_ERR_SHAPE;
    }
    if ((a->dtype != GDN_BF16 && a->dtype != GDN_F32) || (a->flags & ~GDN_FLAG_LEFT_PADDED) || a->T > 1 << 30) return GDN_ERR_UNSUPPORTED;
    if (const int e = check_cache_pointers(a->cache); e != GDN_OK) return e;
    if (const int e = check_rows16(a->k, a->k_stride_b, a->k_stride_t, a->k_stride_h, a->dtype); e != GDN_OK) return e;
    if (const int e = check_rows16(a->v, a->v_stride_b, a->v_stride_t, a->v_stride_h, a->dtype); e != GDN_OK) return e;
    if (a->start == nullptr) return GDN_ERR_NULL;
    if (!cache_aligned(a->start, 4) || !cache_aligned(a->cu_seqlens, 4)) return GDN_ERR_ALIGN;
    WriteParams p{};
    p.c = a->cache;
    p.x[0] = a->k, p.b[0] = a->k_stride_b, p.t[0] = a->k_stride_t, p.h[0] = a->k_stride_h;
    p.x[1] = a->v, p.b[1] = a->v_stride_b, p.t[1] = a->v_stride_t, p.h[1] = a->v_stride_h;
    p.start = a->start, p.cu = a->cu_seqlens, p.B = a->B, p.T = a->T, p.padded = padded;
    const int P = a->cache.P;
    const bool packed = a->cu_seqlens != nullptr && !padded;
    p.each = packed ? 0 : std::min((int)(((int64_t)a->T + P - 2) / P + 1), a->cache.table_pages);
    // packed: sequences of a token or more touch at most (tokens - 1) / P + 2 pages each
    const int64_t slots = packed ? (int64_t)a->T / P + 2 * (int64_t)std::min(a->cache.N, a->T) : (int64_t)a->cache.N * p.each;
    if (slots > INT32_MAX) return GDN_ERR_UNSUPPORTED;
    if (!packed && a->T <= APPEND_TOKENS) {
        const int lanes = a->cache.D <= 64 ? 8 : a->cache.D <= 128 ? 16 : 32;
        const int64_t groups = slots * a->cache.HK * 2, blocks = (groups + 256 / lanes - 1) / (256 / lanes);
        if (blocks > INT32_MAX) return GDN_ERR_UNSUPPORTED;
        const hipStream_t st = static_cast<hipStream_t>(stream);
        const auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), 0, st, p); };
        if (a->dtype == GDN_BF16) lanes == 8 ? go(cache_append_kernel<bf16_t, 8>) : lanes == 16 ? go(cache_append_kernel<bf16_t, 16>) : go(cache_append_kernel<bf16_t, 32>);
        else lanes == 8 ? go(cache_append_kernel<float, 8>) : lanes == 16 ? go(cache_append_kernel<float, 16>) : go(cache_append_kernel<float, 32>);
        return (int)hipGetLastError();
    }
    if (slots * a->cache.HK > INT32_MAX) return GDN_ERR_UNSUPPORTED;
    const dim3 grid((unsigned)(slots * a->cache.HK), 2), block(threads_for(P, a->cache.D));
    if (a->dtype == GDN_BF16) hipLaunchKernelGGL((cache_write_kernel<bf16_t>), grid, block, 0, static_cast<hipStream_t>(stream), p);
    else hipLaunchKernelGGL((cache_write_kernel<float>), grid, block, 0, static_cast<hipStream_t>(stream), p);
    return (int)hipGetLastError();
}

extern "C" int gdn_cache_read(const gdn_cache_read_args* a, void* stream) {
    if (a == nullptr) return GDN_ERR_NULL;
    if (const int e = check_cache(a->cache); e != GDN_OK) return e;
    if (a->T <= 0) return GDN_ERR_SHAPE;
    if ((a->dtype != GDN_BF16 && a->dtype != GDN_F32) || a->T > (int64_t)a->cache.table_pages * a->cache.P) return GDN_ERR_UNSUPPORTED;
    if (const int e = check_cache_pointers(a->cache); e != GDN_OK) return e;
    if (a->k == nullptr || a->v == nullptr || a->lengths == nullptr) return GDN_ERR_NULL;
    if (!cache_aligned(a->k, 16) || !cache_aligned(a->v, 16) || !cache_aligned(a->lengths, 4)) return GDN_ERR_ALIGN;
    ReadParams p{};
    p.c = a->cache, p.out[0] = a->k, p.out[1] = a->v, p.lengths = a->lengths, p.T = a->T;
    p.each = (a->T - 1) / a->cache.P + 1;
    const int64_t slots = (int64_t)a->cache.N * p.each;
    if (slots > INT32_MAX) return GDN_ERR_UNSUPPORTED;
    const dim3 grid((unsigned)slots, a->cache.HK, 2), block(threads_for(a->cache.P, a->cache.D));
    if (a->dtype == GDN_BF16) hipLaunchKernelGGL((cache_read_kernel<bf16_t>), grid, block, 0, static_cast<hipStream_t>(stream), p);
    else hipLaunchKernelGGL((cache_read_kernel<float>), grid, block, 0, static_cast<hipStream_t>(stream), p);
    return (int)hipGetLastError();
}
