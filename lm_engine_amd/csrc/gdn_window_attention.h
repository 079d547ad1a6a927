// Softmax attention over a window: what its kernels share (include/gdn_attention_hip.h has the definition).
//
// Rows.  A row is one query head of one token; the query heads that share a head of k and v are the rows t G + g of one matrix, so that a tile
// of keys serves all of them and the gradients of a shared head add up where they are formed.  Query t stands at key position
// a = t + S - T.  What row and key see of each other are intervals:
//     row at a, of a sequence that begins at st:     keys [max(st, a - W + 1), a] and [st, st + sinks), up to a
//     key j of a sequence [st, en):                  positions [j, min(en, j + W) - 1], and up to en - 1 if j < st + sinks
// so that no tile needs more than two comparisons per element, and most need none.
#pragma once

#include "gdn_attention_hip.h"
#include "gdn_linear_tile.h"

namespace gdn {

struct WindowRows {  // a tensor [B, T, heads, D], strides in elements
    const void* p;
    int64_t b, t, h;
};

struct WindowParams {
    WindowRows q, k, v, o, dout, dq, dk, dv;
    float* lse;    // [B, T, H]; fp32 [B, T, H, 2]
    float* delta;  // [B, T, H]: sum over D of o do
    const int32_t* cu;
    int padded;
    int B, T, S, H, HK, G, D, N;
    int rows;         // T G
    uint32_t by_g;    // ceil(2^32 / G), for split_rows
    int window, sinks;  // window 0: every key
    float scale, c;   // c = |scale| log2(e)
    int negative;     // of scale
    int blocks;       // of rows (or keys), per pair of batch row and head
    // keys cut into `splits` parts, each with its own partial result
    int splits;
    float* part_o;    // [splits, B, HK, rows, D]
    float* part_m;    // [splits, B, HK, rows, 2]: reference exponent, sum
    // gradients of a sequence's first keys from rows that see them beyond the window, in `pieces` parts per sequence
    int pieces, first_keys;  // first_keys: sinks, in whole blocks
    float* part_dk;   // [N, HK, pieces + shares, first_keys, 2, D]; the last parts are from the rows that have them in their window
    // the rows of a block of keys cut into `shares`
    int shares;
    float* part_all;  // [shares, B, HK, S, 2, D]
};

// n / G and the rest, for n < G + 256.  by_g is less than 1 / G too large in units of 2^32 / G, so that n by_g / 2^32 is n / G rounded down as long as
// n G < 2^32: the backward refuses more heads to one.
constexpr int MOST_GROUP = 65280;
static_assert((uint64_t)MOST_GROUP * (MOST_GROUP + 256) < (uint64_t)1 << 32);
__device__ __forceinline__ void split_rows(const WindowParams& p, int n, int& t, int& g) {
    t = p.G == 1 ? n : (int)__umulhi((unsigned)n, p.by_g);
    g = n - t * p.G;
}

// The sequence [st, en) of key position `at` in batch row b: empty (en = st) where the position belongs to none; and its number.
__device__ __forceinline__ void sequence_at(const WindowParams& p, int b, int at, int& st, int& en, int& n) {
    n = b;
    if (p.cu == nullptr) {
        st = 0, en = p.S;
    } else if (p.padded) {
        st = p.S - min(max(p.cu[b + 1] - p.cu[b], 0), p.S), en = p.S;
    } else {
        int lo = 0, hi = p.N + 1;  // the first entry past `at`
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (p.cu[mid] <= at) lo = mid + 1;
            else hi = mid;
        }
        n = lo - 1;
        if (lo == 0 || lo > p.N) {
            st = en = 0, n = 0;
            return;
        }
        packed_bounds(p.cu, n, p.S, st, en);
        en += st;
    }
    if (at < st || at >= en) en = st;
}

// sequence n's first position and length
__device__ __forceinline__ void sequence_of(const WindowParams& p, int n, int& st, int& len) {
    if (p.cu == nullptr) st = 0, len = p.S;
    else if (p.padded) len = min(max(p.cu[n + 1] - p.cu[n], 0), p.S), st = p.S - len;
    else packed_bounds(p.cu, n, p.S, st, len);
}

// What a row sees: keys [lo, a] and [st, sk); a < lo: none.
struct RowView {
    int a, lo, st, sk;
};
__device__ __forceinline__ RowView row_view(const WindowParams& p, int b, int r) {
    RowView v;
    const int t = p.G == 1 ? r : r / p.G;
    v.a = t + p.S - p.T;
    int en, n;
    sequence_at(p, b, v.a, v.st, en, n);
    if (v.a < 0 || en <= v.st) v.a = -1, v.lo = 1 << 30, v.st = v.sk = 0;
    else v.lo = p.window == 0 ? v.st : max(v.st, v.a - p.window + 1), v.sk = min(v.st + min(p.sinks, p.S - v.st), v.lo);
    return v;
}

template <int CTRL>
__device__ __forceinline__ int lane_moved(int x) {
    return __builtin_amdgcn_update_dpp(0, x, CTRL, 0xF, 0xF, false);
}
// (over neighbours by moves within rows of 16 lanes, then rows, then halves: five of these took 2000 cycles by way of LDS, at the head of every kernel)
__device__ __forceinline__ int wave_min(int x) {
    x = min(x, lane_moved<0xB1>(x));   // lane l ^ 1
    x = min(x, lane_moved<0x4E>(x));   // l ^ 2
    x = min(x, lane_moved<0x141>(x));  // the other four of eight
    x = min(x, lane_moved<0x128>(x));  // eight lanes on in the row
    const auto rows = __builtin_amdgcn_permlane16_swap((unsigned)x, (unsigned)x, false, false);
    x = min((int)rows[0], (int)rows[1]);
    const auto halves = __builtin_amdgcn_permlane32_swap((unsigned)x, (unsigned)x, false, false);
    return __builtin_amdgcn_readfirstlane(min((int)halves[0], (int)halves[1]));
}
__device__ __forceinline__ int wave_max(int x) { return -wave_min(-x); }

// The keys of a tile that a row sees: an interval of the keys near it, or of the first keys (which end at `sink_end`, where the near ones
// begin); where first keys lie among near ones (`mixed`, the same for the workgroup) also those.
struct TileView {
    int from, st;
    unsigned span, first;
    __device__ __forceinline__ TileView(const RowView& v, bool near, int sink_end)
        : from(near ? v.lo : v.st), st(v.st), span(near ? max(v.a + 1 - v.lo, 0) : max(min(v.sk, sink_end) - v.st, 0)), first(max(v.sk - v.st, 0)) {}
    __device__ __forceinline__ bool sees(int j) const { return (unsigned)(j - from) < span; }
    __device__ __forceinline__ bool sees_mixed(int j) const { return sees(j) || (unsigned)(j - st) < first; }
};

// What a wave's rows see: keys from [lo, end) and [sink, sink_end), all of them those of [full_lo, full_end).
struct WaveView {
    int lo, end, sink, sink_end, full_lo, full_end;
    // whether one of the rows may see one of `count` keys (a row's first keys may lie among the near ones of others)
    __device__ __forceinline__ bool meets(int j0, int count) const { return (j0 < end && j0 + count > lo) || (j0 < sink_end && j0 + count > sink); }
};
__device__ __forceinline__ WaveView wave_view(const RowView& v) {
    WaveView w;
    w.lo = wave_min(v.lo), w.end = wave_max(v.a) + 1, w.full_lo = wave_max(v.lo), w.full_end = wave_min(v.a) + 1;
    w.sink = wave_min(v.sk > v.st ? v.st : 1 << 30), w.sink_end = wave_max(v.sk > v.st ? v.sk : 0);
    return w;
}
template <int WAVES>
__device__ __forceinline__ WaveView join_waves(const WaveView& w, int (&shared)[WAVES][6], int wave, int lane) {
    if (lane == 0) shared[wave][0] = w.lo, shared[wave][1] = w.end, shared[wave][2] = w.sink, shared[wave][3] = w.sink_end, shared[wave][4] = w.full_lo, shared[wave][5] = w.full_end;
    __syncthreads();
    WaveView r = w;
#pragma unroll
    for (int i = 0; i < WAVES; i++) {
        r.lo = min(r.lo, shared[i][0]), r.end = max(r.end, shared[i][1]), r.sink = min(r.sink, shared[i][2]), r.sink_end = max(r.sink_end, shared[i][3]);
        r.full_lo = max(r.full_lo, shared[i][4]), r.full_end = min(r.full_end, shared[i][5]);
    }
    r.lo = __builtin_amdgcn_readfirstlane(r.lo), r.end = __builtin_amdgcn_readfirstlane(r.end), r.sink = __builtin_amdgcn_readfirstlane(r.sink);
    r.sink_end = __builtin_amdgcn_readfirstlane(r.sink_end), r.full_lo = __builtin_amdgcn_readfirstlane(r.full_lo), r.full_end = __builtin_amdgcn_readfirstlane(r.full_end);
    return r;
}

// Workgroup x's pair of (batch row, kv head) and block: the pairs one after the other, then the next block.  (Neighbouring blocks, which share keys, on
// one of the eight XCDs instead: 157 us as before with 8 pairs and a window; without one 1054 instead of 851 us backward with 6 pairs, where
// an XCD's blocks are then all long or all short.)
__device__ __forceinline__ void work_item(const WindowParams& p, int x, int& pair, int& block) {
    const int pairs = p.B * p.HK;
    block = x / pairs, pair = x - block * pairs;
}

// A tile of rows of DP columns (WROWS a wave) on its way into LDS, without registers in between: a wave's instruction fills 1 KB, the lanes' 16 bytes
// one behind the other, so the granules are swapped (tile_key) where they are read.  What lies past the rows or columns that there are is
// read past the buffer's end, which gives zeros.
typedef __attribute__((ext_vector_type(4))) int i32x4;
constexpr uint32_t PAST = 0x80000000u;
// What rows may lie apart, in elements: one token and the next, and the heads of a token in all (gdn_window_api.hip refuses more).
constexpr int64_t MOST_APART = 1 << 23, MOST_HEADS = 1 << 28;
// whether the bytes from one base to every column of `rows` rows (tokens, or heads of as many tokens and one more begun) stay below PAST
constexpr bool row_offsets_fit(int rows, bool heads) { return ((rows - (heads ? 0 : 1)) * MOST_APART + (heads ? MOST_HEADS : 0) + 256) * 2 < PAST; }
template <int DP, int WROWS = 16>
struct TileLoads {
    static constexpr int GRANULES = DP / 8, RPI = 64 / GRANULES, ITERS = WROWS / RPI;
    static_assert(GRANULES <= 64 && WROWS % RPI == 0, "a wave loads WROWS rows");
    static __device__ __forceinline__ int row(int wave, int lane, int i) { return WROWS * wave + RPI * i + lane / GRANULES; }
    static __device__ __forceinline__ int column(int wave, int lane, int i) { return 8 * (lane % GRANULES ^ tile_key<DP>(row(wave, lane, i))); }
    // `to`: LDS address of the tile; offset (and `more`, the same in all lanes) in bytes from `base`
    static __device__ __forceinline__ void load(const void* base, uint32_t offset, uint32_t to, int wave, int i, int more = 0) {
        const uint64_t a = reinterpret_cast<uint64_t>(base);
        i32x4 r;
        r[0] = __builtin_amdgcn_readfirstlane((int)(uint32_t)a), r[1] = __builtin_amdgcn_readfirstlane((int)(uint32_t)(a >> 32) & 0xffff);
        r[2] = (int)PAST, r[3] = 0x00020000;
        const int at = __builtin_amdgcn_readfirstlane((int)(to + (WROWS * wave + RPI * i) * DP * 2));
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(at), "v"(offset), "s"(r), "s"(more) : "memory");
    }
};
// A tile whose rows lie `stride` elements apart, asked for in ITERS pieces, to be spread over the work on another one: a load takes the wave's
// time until the compute unit's address path has taken it, and eight waves ask at once (800 cycles a tile in one go).
template <int DP, int WROWS = 16>
struct TileRequest {
    using Loads = TileLoads<DP, WROWS>;
    const char* base;
    int stride, count, columns;
    uint32_t to, row_bytes, place;
    int row0;
    // row RPI i on, the granule's place is the first one's with some bits turned
    __device__ __forceinline__ void piece(int wave, int i) const {
        const uint32_t at = place ^ (16 * tile_key<DP>(Loads::RPI * i));
        Loads::load(base, row0 + Loads::RPI * i < count && (int)at < 2 * columns ? at + row_bytes : PAST, to, wave, i, Loads::RPI * i * stride * 2);
    }
    __device__ __forceinline__ void all(int wave) const {
#pragma unroll
        for (int i = 0; i < Loads::ITERS; i++) piece(wave, i);
    }
};
// everything that this wave has asked for is in LDS
__device__ __forceinline__ void loads_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// Operand fragments of v_mfma_f32_32x32x16_bf16 from such a tile.
template <int DP>
struct TileReader {
    int row, pair;
    __device__ __forceinline__ TileReader(int lane) {
        const int l32 = lane & 31, half = lane >> 5;
        row = l32 * DP + ((half ^ tile_key<DP>(l32)) << 3);
        const int r = 4 * half + ((lane & 15) >> 2), c = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
        pair = r * DP + (((c >> 3) ^ tile_key<DP>(r)) << 3) + (c & 7);
    }
    static constexpr int PERIOD = TileLane<DP>::PERIOD;
    // x where it is used, rather than what follows from x in registers over a whole walk
    __device__ __forceinline__ void recompute() { asm volatile("" : "+v"(row), "+v"(pair)); }
    // columns 16 s + 8 half .. + 7 of row row0 + (lane & 31); row0 a multiple of 32
    __device__ __forceinline__ bf16x8 across(const bf16_t* tile, int row0, int s) const {
        return *reinterpret_cast<const bf16x8*>(tile + (row ^ (16 * s % PERIOD)) + row0 * DP + 16 * s / PERIOD * PERIOD);
    }
    // rows 16 s + 4 half + {0 .. 3, 8 .. 11} of column 32 t + (lane & 31): the order in which a lane holds 8 rows of an accumulator, so that
    // one goes on as an operand as it is
    __device__ __forceinline__ bf16x8 down(const bf16_t* tile, int s, int t) const {
        const bf16_t* const p = tile + 16 * s * DP + 32 * t / PERIOD * PERIOD;
        const int at = pair ^ (32 * t % PERIOD);
        const bf16x4 lo = TileLane<DP>::read(p + at), hi = TileLane<DP>::read(p + (at ^ 16) + 8 * DP);  // (8 rows on, the key's second bit is the other)
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
};

__device__ __forceinline__ f32x16 mma(const bf16x8& a, const bf16x8& b, const f32x16& c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }

// x of the lane 32 further (or back)
__device__ __forceinline__ float other_half(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
    return __builtin_bit_cast(float, (threadIdx.x & 32) ? r[0] : r[1]);
}

__device__ __forceinline__ bf16x8 pack8(const f32x16& d, int s) {
    bf16x8 r;
#pragma unroll
    for (int e = 0; e < 8; e++) r[e] = (bf16_t)d[8 * s + e];
    return r;
}

// 8 columns 16 s + 8 half of a row in memory, zeros past D
template <int DP>
__device__ __forceinline__ void load_row_fragments(const bf16_t* row, int D, int half, bool there, bf16x8 (&f)[DP / 16]) {
#pragma unroll
    for (int s = 0; s < DP / 16; s++) {
        const int c = 16 * s + 8 * half;
        const bf16x8 zero = {};
        f[s] = there && c < D ? *reinterpret_cast<const bf16x8*>(row + c) : zero;
    }
}

// In a branch that few tiles take: without it the compiler turns the branch into selects that all of them pay for.
__device__ __forceinline__ void stay_a_branch() { asm volatile(""); }

// row of accumulator register r: (r & 3) + 8 (r >> 2) + 4 half
__device__ __forceinline__ constexpr int acc_row(int r, int half) { return (r & 3) + 8 * (r >> 2) + 4 * half; }

// columns [0, D) of a row from a transposed accumulator [DP, rows], this lane's row
template <int DP>
__device__ __forceinline__ void store_transposed(bf16_t* row, int D, int half, const f32x16 (&acc)[DP / 32], float by) {
#pragma unroll
    for (int t = 0; t < DP / 32; t++)
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const int c = 32 * t + 8 * q + 4 * half;
            if (c < D) store4<bf16_t>(row + c, f32x4{acc[t][4 * q] * by, acc[t][4 * q + 1] * by, acc[t][4 * q + 2] * by, acc[t][4 * q + 3] * by});
        }
}

constexpr float LOWEST = -3.402823466e38f;

// What a forward took out of tiles that not all of its rows see (values that are not finite), added to the results of the rows that see it: a
// few threads a row, behind the stores of the whole workgroup.  An infinite value stays what it is under any weight, and NaN too.  `width`: keys of
// a whole tile, by which the walk tells which tiles all rows see all of; a last tile that ends with the keys is not one of them.
template <typename T, typename TileAt>
__device__ __forceinline__ void add_taken_out(const WindowParams& p, int b, int hk, int r0, int rows, const WaveView& all, int first_tile, int last_tile, int sink_tiles,
                                           int width, const TileAt& tile_at, int64_t part) {
    __syncthreads();
    const int each = (int)blockDim.x / rows, own = r0 + (int)threadIdx.x / each;
    if (own >= p.rows) return;
    const RowView v = row_view(p, b, own);
    const int t = p.G == 1 ? own : own / p.G, g = own - t * p.G;
    T* const out = static_cast<T*>(const_cast<void*>(p.o.p)) + b * p.o.b + t * p.o.t + (hk * p.G + g) * p.o.h;
    for (int i = first_tile; i < last_tile; i++) {
        int j0, count;
        tile_at(i, j0, count);
        if (i >= sink_tiles && j0 >= all.full_lo && j0 + width <= all.full_end) continue;
        for (int j = max(j0, v.st); j < j0 + count && j <= v.a; j++) {
            if (j < v.lo && j >= v.sk) continue;
            const T* const value = static_cast<const T*>(p.v.p) + b * p.v.b + j * p.v.t + hk * p.v.h;
            for (int d = threadIdx.x % each; d < p.D; d += each) {
                const float x = (float)value[d];
                if (fabsf(x) < __builtin_inff()) continue;
                if (p.splits > 1) p.part_o[(part + own - r0) * p.D + d] += x;
                else out[d] = (T)((float)out[d] + x);
            }
        }
    }
}

int launch_window_fwd(const WindowParams& p, hipStream_t stream);           // bf16, gdn_window_attention.hip
int launch_window_bwd(const WindowParams& p, hipStream_t stream);           // bf16, gdn_window_attention_bwd.hip
int launch_window_fwd_f32(const WindowParams& p, hipStream_t stream);       // gdn_window_attention_f32.hip
int launch_window_bwd_f32(const WindowParams& p, hipStream_t stream);
int launch_window_combine(const WindowParams& p, int dtype, hipStream_t stream);
constexpr int WINDOW_ROWS = 128;      // of a workgroup, bf16
constexpr int window_keys(int D) { return D > 64 && D <= 128 ? 128 : 64; }  // of a workgroup of the keys' gradients, bf16
constexpr int WINDOW_FIRST_KEYS = 32;  // of a workgroup of a sequence's first keys
constexpr int WINDOW_ROWS_F32 = 16;
constexpr int WINDOW_KEYS_F32 = 16;

}  // namespace gdn
