// ft_hip_attn.hip -- attention of a batch's newest tokens over a quantised cache
// (ft_hip_attention): each sequence over a prefix that all share and over its
// own tokens. The cache's layout is ft_kv.hpp's.
//
//   out = sum_j softmax_j(scale q . k_j) v_j,  k_j = dk_j K_j, v_j = dv_j V_j  (K, V of 8 bits, a scale a row)
//
// In steps of 32 tokens a wavefront holds 16 columns, each a query on one key
// head: S^T = K Q^T leaves a lane with 8 tokens of its column, from which the
// softmax makes the operand of out^T += V^T P^T without moving anything between
// lanes. The scales are rows' scales and stay out of the products: dk_j times
// the score, dv_j times the weight. Running maximum and sum, f32 accumulators.
//
// Bits. K and V are whole numbers or codes that f16 holds exactly. A query row
// is scaled by a power of two and split into f16 values whose sum it is: one for
// f16 and bf16, two for f32 (22 bits). The weights p_j dv_j are f16 likewise:
// one where the output is of 16 bits, two where it is f32. f32 rows of a
// head come as 8 columns with the first halves and 8 with the second (MODE
// PACK), which costs no further products, or, if there are more rows, as two
// products each (SPLIT).
//
// Split. The batch's own tokens are one line of steps, sequence by sequence and
// head by head, cut into equal lengths, one a wavefront: no sequence is longer
// than another for it, and a single long one is worked on by the whole device.
// What it leaves of a row that it has not seen whole goes to the workspace and
// k_attn_merge joins the pieces. The prefix is a line of its own, cut likewise
// into a piece for each workgroup that the own tokens leave: its four wavefronts
// take 16 rows or more each, whichever sequence they belong to, on tiles that they
// widen once for all of them in LDS. By wavefronts alone, each widening for itself,
// 64 queries behind 32768 tokens took 167 us for 118.
//
// What bounds it (an MI355X that copies 5.1 TB/s and multiplies 1110 TFLOP/s in
// f16), in us a call, and of the own and joining kernels in a profiled run:
// one sequence of 131071 tokens on 8 heads of 128, 277 MB, 62 (53 + 8.4): the
// cache's bytes, 5.2 TB/s in the first, then the joining of 256 pieces a row.
// 64 sequences of up to 4096 on 8 heads of 256, f32, 82 (75 + 6): bytes and the
// widening beside them. One of 777, 12.6 (9.7 + 4.7): two launches, and in each
// reads that wait for each other (lengths, pages, tokens, queries). 64 queries of
// 16 heads of 256 behind 8192, f32, 54 (48 + 8.8): 34 of it do not grow with the
// prefix (21 for each further 8192 tokens), starts, pieces and their joining.
// 256 queries of 64 heads of 128 behind 16390, 252 (265 + 19 at a profiled run's
// clock), where the products alone are 125: the softmax's vector instructions,
// which a wavefront's products do not hide, and rows of a few hundred own tokens.

#include "ft_device.hpp"
#include "ft_kv.hpp"
#include "ft_overlap.hpp"
#include "ft_runtime.hpp"
#include "ft_wave.hpp"

#include <cfloat>
#include <cmath>

using namespace ft;

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float float2_ __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr int STEP = 32;  // tokens of a step, two tiles
constexpr int THREADS = 256, WAVES = THREADS / 64;
constexpr int MAX_SEQS = FT_ATTN_MAX_SEQS;
constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.693147180559945309417f;

enum { HALF, PACK, SPLIT };

// Workgroups at most, two on each CU: a third leaves 168 registers, and the prefix's loop spills (256 queries behind 16390 283
// us for 261). With two, forms that are not among the timed ones spill as well: f32 heads of 256 with more than 8 rows (43 to
// 53 registers), 16-bit heads of 64 behind a prefix (24, i8 60) and f32 heads of 128 behind one (22 to 28).
constexpr int BLOCKS = 512;

// Where the parts of a call lie, in the workspace and else.
struct AttnArgs {
    const void* q;
    int64_t q_stride;
    void* out;
    int64_t out_stride;
    float* lse;
    const uint8_t* cache;
    const int32_t* tables;
    int64_t table_stride;
    const int32_t* lens;
    const int32_t* prefix;
    const int32_t* prefix_len;
    int prefix_pages, table_pages, n_pages, page_shift;
    int n_seqs, n_q, kv_heads, group, type;
    int row_tiles;   // tiles of a sequence's rows on a head
    int pre_tiles, pre_nt;  // tiles of the batch's rows on a head, and of a wavefront's
    int window;
    float scale;     // times log2 e
    // workspace: a word of how many pieces the prefix is cut into, descriptors of the own items, pieces
    int32_t* head;   // [0]: workgroups that the prefix is cut for
    int2* items;
    float* own;      // pieces of own rows: `piece` floats each
    float* pre;      // pieces of prefix rows: 16 rows each
    int own_waves;   // at most
    int rows;        // of an own piece
};

// Floats of a piece of `rows` rows: the rows' averages, then their maxima and sums. An odd number of rows leaves the next piece
// between two vectors' places.
__host__ __device__ __forceinline__ int64_t piece_floats(int rows, int D) { return (int64_t)rows * (D + 2); }

// At the head of a branch that few waves take: keeps the compiler from doing its work always and choosing afterwards.
__device__ __forceinline__ void rare() { asm volatile(""); }
__device__ __forceinline__ int clampi(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }
__device__ __forceinline__ int uni(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Largest of the lanes l, l ^ 16, l ^ 32, l ^ 48, in each.
__device__ __forceinline__ float max_groups(float v) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float sum_groups(float v) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
// The lane 8 on in the row of 16.
__device__ __forceinline__ float other8(float v) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x128, 0xF, 0xF, false));
}

// Four bytes of the cache as f16.
template <int CT>
__device__ __forceinline__ void widen4(uint32_t w, half2& a, half2& b) {
    if constexpr (CT == FT_KV_I8) {  // 0x6400 | byte is 1024 + byte
        const half2 off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
        a = __builtin_bit_cast(half2, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) + off;
        b = __builtin_bit_cast(half2, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) + off;
    } else {
        a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false);
        b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true);
    }
}
template <int CT>
__device__ __forceinline__ half8 widen8(uint32_t lo, uint32_t hi) {
    half2 a, b, c, d;
    widen4<CT>(lo, a, b);
    widen4<CT>(hi, c, d);
    return half8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// Eight keys' dimensions. Where q is of 16 bits, i8's byte q + 128 as it is makes a subnormal f16 of (q + 128) 2^-24,
// which the products take exactly; what the 128 adds to a sum of products is the same for all keys, and the sum starts
// from less than 0 by it (Attend::from). f32 queries take the keys without the 128: its part of a sum is several times the
// rest and so are the roundings, and their first halves' and second halves' products leave time for the widening (64
// sequences of up to 4096 tokens 82 us with the 128, 75 without).
template <int CT, bool F32>
__device__ __forceinline__ half8 widen_k(uint32_t lo, uint32_t hi) {
    if constexpr (CT == FT_KV_I8 && !F32) {
        const u32x4 w = {__builtin_amdgcn_perm(0, lo, 0x0C010C00u), __builtin_amdgcn_perm(0, lo, 0x0C030C02u),
                         __builtin_amdgcn_perm(0, hi, 0x0C010C00u), __builtin_amdgcn_perm(0, hi, 0x0C030C02u)};
        return __builtin_bit_cast(half8, w);
    } else {
        return widen8<CT>(lo, hi);
    }
}

__device__ __forceinline__ f32x4 mfma(half8 a, half8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// Vectors at any address of their element type: the loads and stores of global
// memory take it.
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned u32x2_any __attribute__((ext_vector_type(2), aligned(2)));

// Eight consecutive values of a query as f32.
template <bool F32>
__device__ __forceinline__ void load_q8(const void* q, int64_t at, bool f16, float* x) {
    if constexpr (F32) {
        const f32x4_any* p = reinterpret_cast<const f32x4_any*>(static_cast<const float*>(q) + at);
        const f32x4 a = p[0], b = p[1];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
    } else {
        const u32x4 a = *reinterpret_cast<const u32x4_any*>(static_cast<const uint16_t*>(q) + at);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t lo = a[i] & 0xFFFF, hi = a[i] >> 16;
            x[2 * i] = f16 ? h2f((uint16_t)lo) : __uint_as_float(lo << 16);
            x[2 * i + 1] = f16 ? h2f((uint16_t)hi) : __uint_as_float(a[i] & 0xFFFF0000u);
        }
    }
}

__device__ __forceinline__ uint16_t narrow(float v, bool f16) {
    const uint32_t w = __float_as_uint(v);
    if (f16) return f2h(v);
    return (w & 0x7FFFFFFFu) > 0x7F800000u ? (uint16_t)(w >> 16 | 0x40) : (uint16_t)((w + 0x7FFF + (w >> 16 & 1)) >> 16);
}
template <bool F32>
__device__ __forceinline__ void store_out(void* out, int64_t at, bool f16, f32x4 v) {
    if constexpr (F32) {
        *reinterpret_cast<f32x4_any*>(static_cast<float*>(out) + at) = v;
    } else {
        u32x2_any w;
        w[0] = narrow(v[0], f16) | (uint32_t)narrow(v[1], f16) << 16;
        w[1] = narrow(v[2], f16) | (uint32_t)narrow(v[3], f16) << 16;
        *reinterpret_cast<u32x2_any*>(static_cast<uint16_t*>(out) + at) = w;
    }
}

// Which query a column of a wavefront holds.
struct Column {
    int seq, t, head;  // t: which of the sequence's new tokens
    bool live;         // there is such a row, and its query is no padding
};

// Where the tiles of a list of pages lie, 64 tiles at a time, a lane each.
template <int D>
struct Tiles64 {
    int first, end;     // the tile of lane 0; the list's tiles end before this one
    uint64_t in_cache;  // a bit for each lane whose tile is in the cache and before the end
    int lo, hi;         // the lane's tile's address, a tile of page 0's in place of one that is not in the cache
    int raw, raw_next;  // its page's number, and that of 64 tiles on
    const int32_t* ids;
    int n;
    __device__ __forceinline__ int fetch(const AttnArgs& a, int from) const {
        const int at = (from + (int)(threadIdx.x & 63)) >> (a.page_shift - 4);
        return ids[at < n ? at : n - 1];
    }
    // Has the pages' numbers fetched; settle() waits for them.
    __device__ __forceinline__ void open(const AttnArgs& a, const int32_t* pages, int count, int tile, int end_) {
        ids = pages, n = count, first = tile, end = end_;
        raw = fetch(a, tile), raw_next = fetch(a, tile + 64);
    }
    __device__ __forceinline__ void settle(const AttnArgs& a, int head) {
        const int tile = first + (threadIdx.x & 63), mask = (1 << (a.page_shift - 4)) - 1;
        const bool good = (unsigned)raw < (unsigned)a.n_pages && tile < end;
        const uint64_t at = reinterpret_cast<uint64_t>(a.cache) + (tile & mask) * (16 * D) +
                            ((int64_t)(good ? raw : 0) * a.kv_heads + head) * kv_block_bytes((int64_t)1 << a.page_shift, D);
        lo = (int)at, hi = (int)(at >> 32), in_cache = __ballot(good);
    }
    // To the tiles from `tile` on, which is an even number from the first.
    __device__ __forceinline__ void reach(const AttnArgs& a, int head, int tile) {
        if (tile - first < 64) return;
        rare();
        first += 64;
        raw = raw_next;
        raw_next = fetch(a, first + 64);
        settle(a, head);
    }
    __device__ __forceinline__ const uint8_t* at(int tile) const {
        const uint32_t l = __builtin_amdgcn_readlane(lo, tile - first), h = __builtin_amdgcn_readlane(hi, tile - first);
        return reinterpret_cast<const uint8_t*>((uint64_t)h << 32 | l);
    }
    __device__ __forceinline__ bool has(int tile) const { return in_cache >> (tile - first) & 1; }
};

// From a tile's keys to its scales, or with D = 1 more than there is to its values' and theirs.
__device__ __forceinline__ int64_t to_scales(const AttnArgs& a, int D, int tile) {
    const int in = tile & ((1 << (a.page_shift - 4)) - 1);
    return ((int64_t)(2 * D) << a.page_shift) - in * (16 * D - 64);
}

// Two tiles of a head's tokens, on their way.
template <int ND>
struct Step {
    static constexpr int D = 64 * ND;
    static constexpr bool FAR = false;
    static constexpr int BATCH = 2;  // operands that are taken at a time
    u32x4 k[2][ND], v[2][ND];
    f32x4 dk[2], dv[2];

    // Where the tiles `tile` and `tile` + 1 of a list lie.
    struct Aim {
        const uint8_t* at[2];
        int64_t scales[2];
        bool has[2];
        int lane16, lane64;
        __device__ __forceinline__ void to(const AttnArgs& a, Tiles64<D>& p, int head, int tile) {
            p.reach(a, head, tile);
            const int lane = threadIdx.x & 63;
            lane16 = lane * 16, lane64 = lane >> 4 << 4;
#pragma unroll
            for (int x = 0; x < 2; ++x) at[x] = p.at(tile + x), has[x] = p.has(tile + x), scales[x] = to_scales(a, D, tile + x);
        }
        // What is loaded next is of no use: all lanes load the same.
        __device__ __forceinline__ void nowhere() { lane16 = lane64 = 0; }
    };
    // Operands of the products: keys 64 c + 16 g + 8 h on of tile x, values 64 c + 4 r + j of both tiles.
    template <int CT, bool F32>
    __device__ __forceinline__ half8 key(int x, int c, int h) const { return widen_k<CT, F32>(k[x][c][2 * h], k[x][c][2 * h + 1]); }
    template <int CT>
    __device__ __forceinline__ half8 value(int c, int j) const { return widen8<CT>(v[0][c][j], v[1][c][j]); }
    __device__ __forceinline__ f32x4 key_scale(int x) const { return dk[x]; }
    __device__ __forceinline__ f32x4 value_scale(int x) const { return dv[x]; }
    // Tile x has tokens of the list in the bytes of `keep` alone: what the others hold may be codes and scales that are
    // NaN, whose 0 fold is NaN.
    __device__ __forceinline__ void clear(int x, uint32_t keep) {
#pragma unroll
        for (int c = 0; c < ND; ++c) v[x][c] &= keep;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (!(keep >> (8 * i) & 1)) dv[x][i] = 0.0f;
    }

    __device__ __forceinline__ void load_k(const Aim& m) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
#pragma unroll
            for (int c = 0; c < ND; ++c) k[x][c] = *reinterpret_cast<const u32x4*>(m.at[x] + c * 1024 + m.lane16);
            dk[x] = *reinterpret_cast<const f32x4*>(m.at[x] + m.scales[x] + m.lane64);
        }
    }
    __device__ __forceinline__ void load_v(const AttnArgs& a, const Aim& m) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const uint8_t* p = m.at[x] + ((int64_t)D << a.page_shift);
#pragma unroll
            for (int c = 0; c < ND; ++c) v[x][c] = *reinterpret_cast<const u32x4*>(p + c * 1024 + m.lane16);
            dv[x] = *reinterpret_cast<const f32x4*>(m.at[x] + m.scales[x] + (4 << a.page_shift) + m.lane64);
        }
    }
};

// A wavefront's NT times 16 columns (PACK: 8 rows). EACH: a lane's columns may see different tokens, and each has a unit of
// its own, so that values that one does not see cost it no bits. With one for all, which the prefix takes where there is no
// window, 256 queries behind 16390 tokens are 253 us, with one each 262.
template <int CT, int ND, int MODE, int NT, bool EACH>
struct Attend {
    static constexpr int D = 64 * ND;
    static constexpr int PARTS = MODE == SPLIT ? 2 : 1;
    static constexpr bool F32 = MODE != HALF;
    static constexpr int UNITS = EACH ? NT : 1;
    half8 q[NT][PARTS][2 * ND];
    f32x4 acc[NT][4 * ND];
    float base[NT], l[NT];  // the maximum that weights are taken against, and their sum
    float limit[NT];        // over the base: scores above it raise the base; -FLT_MAX while there is none
    float from[NT];         // what a column's sums of products start from
    float fac[NT];          // of a column's products
    float unit[UNITS];      // the weights' unit: the values' largest scale so far as a power of two, over 2^8
    int lo[NT], hi[NT];     // tokens that the column sees
    int all_lo, all_hi;     // that every column sees
    int tokens;             // that the list of pages holds

    // The columns' queries, each in units of a power of two that its largest value gives: one that is no number, or far
    // larger, is no other's concern.
    __device__ __forceinline__ void load(const AttnArgs& a, const Column (&c)[NT]) {
        const int g = (threadIdx.x & 63) >> 4;
        const float second = MODE == PACK && (threadIdx.x & 8) ? -1.0f : 0.0f;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int64_t at = ((int64_t)c[n].seq * a.n_q + c[n].t) * a.q_stride + (int64_t)c[n].head * D + 16 * g;
            float x[2 * ND][8], top = 0.0f;
#pragma unroll
            for (int i = 0; i < 2 * ND; ++i) load_q8<F32>(a.q, at + (i >> 1) * 64 + (i & 1) * 8, a.type == FT_TYPE_F16, x[i]);
#pragma unroll
            for (int i = 0; i < 2 * ND; ++i)
#pragma unroll
                for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[i][e]));
            top = max_groups(top);
            const int e2 = clampi(__float_as_int(top) >> 23, 14, 254);
            const float up = __int_as_float((267 - e2) << 23);  // the largest comes to lie in [2^13, 2^14)
            fac[n] = a.scale * __int_as_float((e2 - 13) << 23) * (CT == FT_KV_I8 && !F32 ? 0x1p24f : 1.0f);
#pragma unroll
            for (int i = 0; i < 2 * ND; ++i)
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    const float2_ v = {x[i][e] * up, x[i][e + 1] * up};
                    const half2 h = __builtin_convertvector(v, half2);
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        q[n][0][i][e + u] = MODE == PACK ? (_Float16)fmaf(second, (float)h[u], v[u]) : h[u];
                        if constexpr (MODE == SPLIT) q[n][PARTS - 1][i][e + u] = (_Float16)fmaf(-1.0f, (float)h[u], v[u]);
                    }
                }
            // keys come as (q + 128) 2^-24 (widen_k): what the 128 is worth, by products with it
            f32x4 worth = {0.0f, 0.0f, 0.0f, 0.0f};
            if constexpr (CT == FT_KV_I8 && !F32) {
                const u32x4 k = {0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u};  // f16 of -128 2^-24
                const half8 minus = __builtin_bit_cast(half8, k);
#pragma unroll
                for (int p = 0; p < PARTS; ++p)
#pragma unroll
                    for (int i = 0; i < 2 * ND; ++i) worth = mfma(minus, q[n][p][i], worth);
            }
            from[n] = worth[0];
#pragma unroll
            for (int i = 0; i < 4 * ND; ++i) acc[n][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            base[n] = 0.0f, l[n] = 0.0f, limit[n] = -FLT_MAX;
        }
#pragma unroll
        for (int n = 0; n < UNITS; ++n) unit[n] = 0x1p-126f;  // p dv is exact to 2^-151 at least: f32 itself has no finer steps than 2^-149
    }

    // The columns' scores of a step less their bases; the keys and their scales are free afterwards.
    template <class Tiles>
    __device__ __forceinline__ void scores(const Tiles& t, f32x4 (&s)[NT][2]) const {
#pragma unroll
        for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = f32x4{from[n], from[n], from[n], from[n]};
#pragma unroll
        for (int i = 0; i < 4 * ND; i += Tiles::BATCH) {
            constexpr int BATCH = Tiles::BATCH;
            half8 k[BATCH];
#pragma unroll
            for (int u = 0; u < BATCH; ++u) k[u] = t.template key<CT, F32>(i + u & 1, (i + u) >> 2, (i + u) >> 1 & 1);
            if constexpr (Tiles::FAR) __builtin_amdgcn_sched_barrier(0);  // read together, not each where it is used
#pragma unroll
            for (int u = 0; u < BATCH; ++u)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int p = 0; p < PARTS; ++p)
                        s[n][i + u & 1] = mfma(k[u], q[n][p][(i + u) >> 1], s[n][i + u & 1]);
        }
        const f32x4 dk[2] = {t.key_scale(0), t.key_scale(1)};
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const f32x4 d = dk[x] * fac[n];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (MODE == PACK) s[n][x][i] += other8(s[n][x][i]);
                    s[n][x][i] = fmaf(s[n][x][i], d[i], -base[n]);
                }
            }
    }

    // Weights of a step at token `at` from its scores, and their sums with the values.
    template <class Tiles>
    __device__ __forceinline__ void weigh(Tiles& t, f32x4 (&s)[NT][2], const bool (&has)[2], int at) {
        const int lane = threadIdx.x & 63, g = lane >> 4;
        const bool whole = has[0] && has[1] && at >= all_lo && at + STEP <= all_hi;
        constexpr int BATCH = Tiles::BATCH;
        half8 w[NT][PARTS], v[BATCH];
        float vt[UNITS];  // the largest scale of values that a lane's columns see of its tokens
        if constexpr (Tiles::FAR) {  // the first values are on their way while the weights are made
#pragma unroll
            for (int u = 0; u < BATCH; ++u) v[u] = t.template value<CT>(u >> 2, u & 3);
            __builtin_amdgcn_sched_barrier(0);
        }
        if (!whole) {
            rare();
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                uint32_t keep = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int j = at + 16 * x + 4 * g + i;
                    const bool in = has[x] && j < tokens;
                    if (in) keep |= 255u << (8 * i);
#pragma unroll
                    for (int n = 0; n < NT; ++n)
                        if (!in || j < lo[n] || j >= hi[n]) s[n][x][i] = -INFINITY;
                }
                t.clear(x, keep);
            }
#pragma unroll
            for (int n = 0; n < (EACH ? NT : 0); ++n) {
                vt[n] = 0.0f;
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const f32x4 d = t.value_scale(x);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (s[n][x][i] != -INFINITY) vt[n] = fmaxf(vt[n], d[i]);
                }
            }
        }
        const f32x4 dv[2] = {t.value_scale(0), t.value_scale(1)};
        // a lane's own scores say enough: the base is raised where any of them is far above it
        float top[NT];
        bool grows = false;
        const float largest = fmaxf(fmaxf(fmaxf(dv[0][0], dv[0][1]), fmaxf(dv[0][2], dv[0][3])),
                                    fmaxf(fmaxf(dv[1][0], dv[1][1]), fmaxf(dv[1][2], dv[1][3])));
        if (whole || !EACH) {
#pragma unroll
            for (int n = 0; n < UNITS; ++n) vt[n] = largest;
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            top[n] = fmaxf(fmaxf(fmaxf(s[n][0][0], s[n][0][1]), fmaxf(s[n][0][2], s[n][0][3])),
                           fmaxf(fmaxf(s[n][1][0], s[n][1][1]), fmaxf(s[n][1][2], s[n][1][3])));
            grows |= top[n] > limit[n];
            if (n < UNITS) grows |= vt[n] > unit[n] * 256.0f;
        }
        if (__any(grows)) rescale(s, top, vt);
        f32x4 in_units[2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const float second = MODE == PACK && (lane & 8) ? 1.0f : 0.0f;
            if (n < UNITS) in_units[0] = dv[0] * inverse(unit[n]), in_units[1] = dv[1] * inverse(unit[n]);
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int i = 0; i < 4; i += 2) {
                    float2_ v;
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float p = __builtin_amdgcn_exp2f(s[n][x][i + e]);
                        l[n] += p;
                        v[e] = p * in_units[x][i + e];
                        // the product as rounded, or hi would round it once and lo be the rest of another hi
                        if constexpr (F32) asm("" : "+v"(v[e]));
                    }
                    const half2 h = __builtin_convertvector(v, half2);
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        w[n][0][4 * x + i + e] = MODE == PACK ? (_Float16)fmaf(-second, (float)h[e], v[e]) : h[e];
                        if constexpr (MODE == SPLIT) w[n][PARTS - 1][4 * x + i + e] = (_Float16)(v[e] - (float)h[e]);
                    }
                }
        }
        if (!whole) {  // 0 times a scale that is NaN, of a token that the column does not see
            rare();
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (s[n][x][i] == -INFINITY) {
#pragma unroll
                            for (int p = 0; p < PARTS; ++p) w[n][p][4 * x + i] = (_Float16)0.0f;
                        }
        }
#pragma unroll
        for (int i = 0; i < 4 * ND; i += BATCH) {
            if (!Tiles::FAR || i > 0) {
#pragma unroll
                for (int u = 0; u < BATCH; ++u) v[u] = t.template value<CT>((i + u) >> 2, (i + u) & 3);
            }
            if constexpr (Tiles::FAR) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int u = 0; u < BATCH; ++u)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int p = 0; p < PARTS; ++p) acc[n][i + u] = mfma(v[u], w[n][p], acc[n][i + u]);
        }
    }

    // A larger maximum, or a larger scale of values.
    __device__ __forceinline__ void rescale(f32x4 (&s)[NT][2], const float (&top)[NT], const float (&vt)[UNITS]) {
        float g = 1.0f;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            if (n < UNITS) {
                const float most = max_groups(vt[n]);
                g = 1.0f;
                if (most > unit[n] * 256.0f) {
                    const float to = __int_as_float((min((__float_as_int(most) >> 23) + 1, 254) - 8) << 23);
                    g = unit[n] * inverse(to);
                    unit[n] = to;
                }
            }
            float f = g;
            const float up = max_groups(top[n]);
            if (up > limit[n]) {  // by its own scores alone: a row's bits are the same whatever its neighbours are
                const float d = __builtin_amdgcn_exp2f(-up);
                if (limit[n] > 0.0f) f *= d, l[n] *= d;  // else there is nothing yet
                limit[n] = 6.0f;
                base[n] += up;
#pragma unroll
                for (int i = 0; i < 4; ++i) s[n][0][i] -= up, s[n][1][i] -= up;
            }
#pragma unroll
            for (int i = 0; i < 4 * ND; ++i) acc[n][i] *= f;
        }
    }
    __device__ __forceinline__ float unit_of(int n) const { return unit[n < UNITS ? n : 0]; }
    // 1 / v of a power of two from 2^-126 to 2^126.
    __device__ __forceinline__ static float inverse(float v) { return __int_as_float(0x7F000000 - __float_as_int(v)); }
    // The maximum that a column's sums are taken against.
    __device__ __forceinline__ float top_of(int n) const { return limit[n] > 0.0f ? base[n] : -INFINITY; }

    // Sums over the lanes that share a column.
    __device__ __forceinline__ void finish(int n, bool live) {
        l[n] = sum_groups(l[n]);
        if (!live) l[n] = 0.0f;
        if constexpr (MODE == PACK) {
#pragma unroll
            for (int i = 0; i < 4 * ND; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[n][i][e] += other8(acc[n][i][e]);
        }
    }
    // Four of the lane's values: dimensions 64 c + 16 g + 4 i on.
    __device__ __forceinline__ f32x4 values(int n, int c, int i, float f) const {
        return f32x4{acc[n][4 * c][i], acc[n][4 * c + 1][i], acc[n][4 * c + 2][i], acc[n][4 * c + 3][i]} * f;
    }
    // A piece is an average, which is no larger than the values: their sum may leave f32's range.
    __device__ __forceinline__ void to_piece(int n, float* piece, int rows, int col) const {
        const int g = (threadIdx.x & 63) >> 4;
        const float f = unit_of(n) * __builtin_amdgcn_rcpf(l[n]);  // within 2^-23; no number where nothing is seen, which is passed over
#pragma unroll
        for (int c = 0; c < ND; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<f32x4_any*>(piece + (int64_t)col * D + 64 * c + 16 * g + 4 * i) = values(n, c, i, f);
        if (g == 0) {
            piece[(int64_t)rows * D + col] = top_of(n);
            piece[(int64_t)rows * D + rows + col] = l[n];
        }
    }
    __device__ __forceinline__ void to_out(int n, const AttnArgs& a, const Column& c) const {
        const int g = (threadIdx.x & 63) >> 4;
        const int64_t row = (int64_t)c.seq * a.n_q + c.t;
        const bool some = l[n] > 0.0f || l[n] != l[n];
        const float f = some ? unit_of(n) / l[n] : 0.0f;
#pragma unroll
        for (int i = 0; i < ND; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                store_out<F32>(a.out, row * a.out_stride + (int64_t)c.head * D + 64 * i + 16 * g + 4 * e, a.type == FT_TYPE_F16,
                               some ? values(n, i, e, f) : f32x4{0.0f, 0.0f, 0.0f, 0.0f});
        if (a.lse && g == 0)
            a.lse[row * a.kv_heads * a.group + c.head] = some ? (top_of(n) + __builtin_amdgcn_logf(l[n])) * LN2 : -INFINITY;
    }
};

// A sequence's own tokens: their number, the first tile that a query sees and the steps from there.
struct Own {
    int len, tile0, steps;
};
__device__ __forceinline__ Own own_of(const AttnArgs& a, int len) {
    Own o;
    const int64_t most = (int64_t)a.table_pages << a.page_shift;
    o.len = len < 0 ? 0 : len > most ? (int)most : len;
    const int first = max(0, o.len - a.n_q);  // the first query's place
    o.tile0 = a.window ? max(0, first - a.window + 1) >> 4 : 0;
    o.steps = max(1, ((o.len + 15) / 16 - o.tile0 + 1) / 2);
    return o;
}

// Sum over the workgroup of what lanes before hold, and the total.
__device__ __forceinline__ int block_scan(int v, int* part, int* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int upto = wave_scan(v);
    __syncthreads();
    if (lane == 63) part[wave] = upto;
    __syncthreads();
    int before = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        if (w < wave) before += part[w];
        sum += part[w];
    }
    *total = sum;
    return before + upto - v;
}

// A line of n steps cut into w pieces, the first n % w of them a step longer.
struct Cuts {
    unsigned each, longer;
    __device__ __forceinline__ Cuts(unsigned n, unsigned w) : each(n / w), longer(n - n / w * w) {}
    __device__ __forceinline__ unsigned begin(unsigned i) const { return i * each + min(i, longer); }
    __device__ __forceinline__ unsigned of(unsigned step) const {  // the piece that holds a step
        const unsigned head = longer * (each + 1);
        return step < head ? step / (each + 1) : longer + (step - head) / max(each, 1u);
    }
};

// What the start and the end of an item cost a wavefront, in steps: each item counts as so many steps more, which come
// first. 64 sequences of up to 4096 tokens 87 us, with 1 89 to 93, with 8 91; 256 of up to 300 28.5, 32 and 29.5.
constexpr int START = 2;

// A wavefront's own steps at least, where there are more than FEW_STEPS in all. One sequence of 4096 tokens on 8 heads 17.0
// us, with 1 step 19.1, with 4 19.4; 8 of up to 4096 23.3, 26.1 and 21.9. One of 777 12.6, with 2 steps 13.9.
constexpr int MIN_STEPS = 2;
constexpr int FEW_STEPS = 1024;

// A prefix step of a workgroup in steps of a wavefront, by which the workgroups are dealt. 64 queries' 16 heads behind 8192
// tokens 55.2 us, at 3 56.5, at 6 60.2; 32 queries' 64 heads behind 16390 with 2000 own tokens 63.4, 66.5 and 69.5; 16 behind
// 32768 59.8, 59.9 and 69.2. 256 queries of 64 heads: 248, 250, 333.
constexpr float PRE_COST = 4.0f;

// The prefix as the batch sees it: its tokens, its first tile that a query may see and the steps from there.
struct Prefix {
    int len, tile0, steps;
};
__device__ __forceinline__ Prefix prefix_of(const AttnArgs& a) {
    Prefix p;
    const int64_t most = (int64_t)a.prefix_pages << a.page_shift;
    const int len = a.prefix_len[0];
    p.len = len < 0 ? 0 : len > most ? (int)most : len;
    p.tile0 = a.window ? max(0, p.len - a.window + 1) >> 4 : 0;  // the first query's place is not before the prefix's end
    p.steps = ((p.len + 15) / 16 - p.tile0 + 1) / 2;
    return p;
}

// Workgroup `b` of `n` so that neighbours are on one die's L2 (workgroups go to the 8 dies in turn).
__device__ __forceinline__ int near_block(int b, int n) {
    const int each = n >> 3;
    return b < each * 8 ? (b & 7) * each + (b >> 3) : b;
}

__device__ __forceinline__ int least_of_wave(int v) {
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) v = min(v, __shfl_xor(v, s));
    return uni(v);
}

// Tiles of 16 rows that a wavefront takes of the prefix, as many as its registers hold.
constexpr int pre_columns(int nd, bool f32) { return nd == 4 ? 1 : nd == 2 ? 2 : f32 ? 2 : 4; }

// Two tiles of the prefix in LDS, as the products take them.
template <int ND>
struct Wide {
    static constexpr bool FAR = true;  // LDS: a batch of operands is read before the first is used
    static constexpr int BATCH = ND == 1 ? 4 : 8;
    half8 k[2][ND][2][64], v[ND][4][64];
    f32x4 dk[2][4], dv[2][4];
    int has[2];
    template <int CT, bool F32>
    __device__ __forceinline__ half8 key(int x, int c, int h) const { return k[x][c][h][threadIdx.x & 63]; }
    template <int CT>
    __device__ __forceinline__ half8 value(int c, int j) const { return v[c][j][threadIdx.x & 63]; }
    __device__ __forceinline__ f32x4 key_scale(int x) const { return dk[x][(threadIdx.x & 63) >> 4]; }
    __device__ __forceinline__ f32x4 value_scale(int x) const { return dv[x][(threadIdx.x & 63) >> 4]; }
    __device__ __forceinline__ void clear(int, uint32_t) const {}  // done where they were widened
};

// A wavefront's share of two tiles on their way: the keys (waves 0 and 1) or values (2 and 3) of one of them.
template <int CT, int ND, bool F32>
struct Share {
    static constexpr int D = 64 * ND;
    u32x4 raw[ND];
    float scale;
    int tile;
    bool has;
    __device__ __forceinline__ void load(const AttnArgs& a, Tiles64<D>& p, int head, int at, bool some) {
        const int wave = uni(threadIdx.x >> 6), lane = threadIdx.x & 63;
        p.reach(a, head, at);
        tile = at + (wave & 1);
        has = some && p.has(tile);
        const uint8_t* keys = p.at(tile);
        const uint8_t* from = keys + ((int64_t)(wave >> 1) * D << a.page_shift) + (some ? lane * 16 : 0);
#pragma unroll
        for (int c = 0; c < ND; ++c) raw[c] = *reinterpret_cast<const u32x4*>(from + c * 1024);
        scale = *reinterpret_cast<const float*>(keys + to_scales(a, D, tile) + ((wave >> 1) * 4 << a.page_shift) + (lane & 15) * 4);
    }
    __device__ __forceinline__ void widen(Wide<ND>& to, int tokens) {
        const int wave = uni(threadIdx.x >> 6), lane = threadIdx.x & 63, x = wave & 1;
        if (wave < 2) {
#pragma unroll
            for (int c = 0; c < ND; ++c)
#pragma unroll
                for (int h = 0; h < 2; ++h) to.k[x][c][h][lane] = widen_k<CT, F32>(raw[c][2 * h], raw[c][2 * h + 1]);
            if (lane < 16) reinterpret_cast<float*>(to.dk[x])[lane] = scale;
            if (lane == 0) to.has[x] = has;
            return;
        }
        if (!has || tile * 16 + 16 > tokens) {  // Step::clear
            rare();
            uint32_t keep = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (has && tile * 16 + (lane >> 4) * 4 + i < tokens) keep |= 255u << (8 * i);
#pragma unroll
            for (int c = 0; c < ND; ++c) raw[c] &= keep;
            if (!has || tile * 16 + (lane & 15) >= tokens) scale = 0.0f;
        }
#pragma unroll
        for (int c = 0; c < ND; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                half2 w[2];
                widen4<CT>(raw[c][j], w[0], w[1]);
                reinterpret_cast<uint2*>(&to.v[c][j][lane])[x] = make_uint2(__builtin_bit_cast(uint32_t, w[0]), __builtin_bit_cast(uint32_t, w[1]));
            }
        if (lane < 16) reinterpret_cast<float*>(to.dv[x])[lane] = scale;
    }
};

// Prefix rows: the lines of WAVES NT tiles of 16 rows on a head, one after the other, are cut into a piece for each
// workgroup. Its wavefronts share the widening: each step's tiles lie in LDS while the next one's are widened beside them.
template <int CT, int ND, int MODE, int NT, bool EACH>
__device__ __forceinline__ void attend_prefix(const AttnArgs& a, const Prefix& pre, int b, int blocks, Wide<ND>* wide, int* part) {
    const int lane = threadIdx.x & 63, col = lane & 15, wave = uni(threadIdx.x >> 6);
    const int groups = (a.pre_tiles + NT * WAVES - 1) / (NT * WAVES);
    const Cuts by((unsigned)pre.steps * (unsigned)(a.kv_heads * groups), (unsigned)blocks);
    unsigned pos = by.begin(b);
    const unsigned stop = by.begin(b + 1);
    while (pos < stop) {
        const int line = uni((int)(pos / (unsigned)pre.steps)), head = line / groups, tile = (line % groups * WAVES + wave) * NT;
        int s0 = (int)pos - line * pre.steps, s1 = min(pre.steps, s0 + (int)(stop - pos));
        pos += s1 - s0;
        Tiles64<64 * ND> tiles;
        tiles.open(a, a.prefix, a.prefix_pages, pre.tile0 + 2 * s0, (pre.len + 15) / 16);
        Attend<CT, ND, MODE, NT, EACH> w;
        Column c[NT];
        int least = pre.len, most_lo = 0;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int r = (tile + n) * 16 + col;
            const bool row = r < a.n_seqs * a.n_q * a.group;
            const int token = row ? r / a.group : 0;
            c[n].seq = token / a.n_q, c[n].t = token % a.n_q, c[n].head = head * a.group + (row ? r % a.group : 0);
            const int at = own_of(a, a.lens[c[n].seq]).len - a.n_q + c[n].t;
            c[n].live = row && at >= 0;
            const int lo = EACH && a.window ? max(0, pre.len + at - a.window + 1) : 0;
            w.lo[n] = c[n].live ? lo : INT32_MIN, w.hi[n] = pre.len;  // one without a query sees all, to no effect
            if (c[n].live) least = min(least, lo), most_lo = max(most_lo, lo);
        }
        w.tokens = w.all_hi = pre.len, w.all_lo = EACH && a.window ? -least_of_wave(-most_lo) : 0;
        if (EACH && a.window) {  // the steps before the first column's first token are nobody's
            least = least_of_wave(least);
            __syncthreads();
            if (lane == 0) part[wave] = least;
            __syncthreads();
#pragma unroll
            for (int v = 0; v < WAVES; ++v) least = min(least, part[v]);
            const int skip = uni(clampi((least / 16 - pre.tile0) / 2, s0, s1));
            if (skip > s0) s0 = skip, tiles.open(a, a.prefix, a.prefix_pages, pre.tile0 + 2 * s0, (pre.len + 15) / 16);
        }
        const int first = pre.tile0 + 2 * s0;
        tiles.settle(a, head);
        Share<CT, ND, MODE != HALF> share;
        share.load(a, tiles, head, first, s0 < s1);
        w.load(a, c);
        __syncthreads();  // the last piece's tiles are done with
        share.widen(wide[0], pre.len);
        share.load(a, tiles, head, first + 2, s0 + 1 < s1);
        const bool mine = tile < a.pre_tiles;
        for (int s = s0; s < s1; ++s) {
            const int at = pre.tile0 + 2 * s, now = (s - s0) & 1;
            __syncthreads();
            share.widen(wide[now ^ 1], pre.len);
            share.load(a, tiles, head, at + 4, s + 2 < s1);
            if (mine) {
                const bool has[2] = {uni(wide[now].has[0]) != 0, uni(wide[now].has[1]) != 0};
                f32x4 sc[NT][2];
                w.scores(wide[now], sc);
                w.weigh(wide[now], sc, has, at * 16);
            }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            if (tile + n >= a.pre_tiles) continue;
            w.finish(n, c[n].live);
            w.to_piece(n, a.pre + ((int64_t)(b + line) * (WAVES * NT) + wave * NT + n) * piece_floats(16, 64 * ND), 16, col);
        }
    }
}

template <int CT, int ND, int MODE, bool PRE>
__global__ __launch_bounds__(THREADS, 2) void k_attn(AttnArgs a) {
    constexpr int COLS = MODE == PACK ? 8 : 16;
    // the prefix's tiles lie where the lengths were
    constexpr int LENS = (2 * MAX_SEQS + 1) * 4, POOL = PRE && (int)sizeof(Wide<ND>[2]) > LENS ? (int)sizeof(Wide<ND>[2]) : LENS;
    __shared__ __attribute__((aligned(16))) char pool[POOL];
    __shared__ int part[WAVES];
    int *const cum = reinterpret_cast<int*>(pool), *const lens = cum + MAX_SEQS + 1;
    const int t = threadIdx.x, lane = t & 63, col = lane & 15;
    // the steps before each sequence
    int before = 0;
    for (int i0 = 0; i0 < a.n_seqs; i0 += THREADS) {
        const int i = i0 + t;
        int total;
        const int len = i < a.n_seqs ? a.lens[i] : 0;
        const int x = block_scan(i < a.n_seqs ? own_of(a, len).steps + START : 0, part, &total);
        if (i < a.n_seqs) cum[i] = before + x, lens[i] = len;
        before += total;
    }
    if (t == 0) cum[a.n_seqs] = before;
    __syncthreads();
    const unsigned lines = a.kv_heads * a.row_tiles;  // items of a sequence
    const unsigned T = before * lines;
    int n_own = (a.own_waves + WAVES - 1) / WAVES;
    bool alone = true;  // the own tokens are all that is seen
    if constexpr (PRE) {
        constexpr int NT = pre_columns(ND, MODE != HALF);
        const Prefix pre = prefix_of(a);
        if (pre.steps > 0) {
            alone = false;
            // the workgroups are dealt by the steps; a prefix step is worth PRE_COST own ones
            const int blocks = gridDim.x, groups = a.kv_heads * ((a.pre_tiles + NT * WAVES - 1) / (NT * WAVES));
            const float work = (float)pre.steps * (float)groups * PRE_COST, all = work + (float)T;
            n_own = min(n_own, clampi((int)((float)T / all * (float)blocks + 0.5f), 1, blocks - 1));
            const int n_pre = min(blocks - n_own, (pre.steps + 1) / 2 * groups);
            if ((int)blockIdx.x >= n_own) {
                const int b = near_block(blockIdx.x - n_own, blocks - n_own);
                if (b == 0 && t == 0) a.head[0] = n_pre;
                __syncthreads();
                if (b >= n_pre) return;
                constexpr int M = MODE == PACK ? SPLIT : MODE;
                Wide<ND>* const wide = reinterpret_cast<Wide<ND>*>(pool);
                if (NT > 1 && a.window)
                    attend_prefix<CT, ND, M, NT, true>(a, pre, b, n_pre, wide, part);
                else
                    attend_prefix<CT, ND, M, NT, NT == 1>(a, pre, b, n_pre, wide, part);
                return;
            }
        } else if (blockIdx.x == 0 && t == 0) {
            a.head[0] = 0;
        }
    }
    const unsigned me = uni(blockIdx.x * WAVES + (t >> 6));
    const unsigned want = T <= FEW_STEPS ? T : (T + MIN_STEPS - 1) / MIN_STEPS;
    const unsigned W = min(want, (unsigned)min(a.own_waves, n_own * WAVES));
    if (me >= W) return;
    const Cuts by(T, W);
    const unsigned begin = by.begin(me), end = by.begin(me + 1);
    // the item that holds the wave's first step
    int seq, line, s0;
    {
        const int u = (int)(begin / lines);
        int i = 0, j = a.n_seqs;
        while (j - i > 1) {
            const int mid = (i + j) >> 1;
            if (cum[mid] <= u)
                i = mid;
            else
                j = mid;
        }
        seq = uni(i);
        const unsigned in = begin - cum[seq] * lines, steps = cum[seq + 1] - cum[seq];
        line = uni((int)(in / steps)), s0 = uni((int)(in % steps)) - START;
    }
    unsigned pos = begin + max(-s0, 0);  // the start of an item is its first step's wave's
    if (pos >= end) return;
    s0 = max(s0, 0);
    Own o = own_of(a, uni(lens[seq]));
    Tiles64<64 * ND> tiles;
    tiles.open(a, a.tables + seq * a.table_stride, a.table_pages, o.tile0 + 2 * s0, (o.len + 15) / 16);
    tiles.settle(a, line % a.kv_heads);
    Step<ND> st;
    typename Step<ND>::Aim aim;
    aim.to(a, tiles, line % a.kv_heads, o.tile0 + 2 * s0);
    st.load_k(aim);
    st.load_v(a, aim);
    bool first = true;
    while (true) {
        const int head = line % a.kv_heads, tile = line / a.kv_heads;
        const int s1 = min(o.steps, s0 + (int)(end - pos));
        // the item behind this one: its pages are on their way while this one is worked on
        const unsigned then = pos + (s1 - s0) + START;
        const bool follows = then < end;
        int seq2 = seq, line2 = line + 1;
        Own o2 = o;
        Tiles64<64 * ND> tiles2 = tiles;
        if (follows) {
            if (line2 == (int)lines) {
                seq2 = seq + 1, line2 = 0;
                o2 = own_of(a, uni(lens[seq2]));
            }
            tiles2.open(a, a.tables + seq2 * a.table_stride, a.table_pages, o2.tile0, (o2.len + 15) / 16);
        }
        Column cs[1], &c = cs[0];
        const int mine = MODE == PACK ? col & 7 : col;
        const int rows = a.n_q * a.group, r = tile * COLS + mine;
        const bool row = r < rows;
        c.seq = seq, c.t = row ? r / a.group : 0, c.head = head * a.group + (row ? r % a.group : 0);
        const int place = o.len - a.n_q + c.t;
        c.live = row && place >= 0;
        Attend<CT, ND, MODE, 1, true> w;
        w.load(a, cs);
        w.lo[0] = c.live && a.window ? max(0, place - a.window + 1) : 0;
        w.hi[0] = c.live ? place + 1 : o.len;  // one without a query sees all, to no effect
        w.tokens = o.len;
        {  // of the tile's first and last live row
            const int first = max((tile * COLS) / a.group, a.n_q - o.len), at_end = min((tile * COLS + COLS - 1) / a.group, a.n_q - 1);
            w.all_hi = uni(o.len - a.n_q + first + 1);
            w.all_lo = a.window ? uni(max(0, o.len - a.n_q + at_end - a.window + 1)) : 0;
        }
        int at = o.tile0 + 2 * s0;
        for (int s = s0; s < s1; ++s) {
            const bool has[2] = {aim.has[0], aim.has[1]};
            if (s + 1 < s1) {
                aim.to(a, tiles, head, at + 2);
            } else if (follows) {
                tiles = tiles2;
                tiles.settle(a, line2 % a.kv_heads);
                aim.to(a, tiles, line2 % a.kv_heads, o2.tile0);
            } else {
                aim.nowhere();
            }
            f32x4 sc[1][2];
            if (o.len > 0) w.scores(st, sc);
            st.load_k(aim);
            if (o.len > 0) w.weigh(st, sc, has, at * 16);
            st.load_v(a, aim);
            at += 2;
        }
        // what other wavefronts have of the item
        const unsigned item_at = cum[seq] * lines + line * (o.steps + START) + START;
        const int fw = (int)by.of(item_at), lw = (int)by.of(item_at + o.steps - 1);
        const int64_t id = (int64_t)seq * lines + line;
        const bool direct = fw == lw && alone;
        // a piece is its wave's first (slot 2 w) or its last (2 w + 1); of a whole item with a prefix, the item's
        const int64_t slot = fw == lw ? 2 * (int64_t)a.own_waves + id : first ? 2 * (int64_t)me : 2 * (int64_t)me + 1;
        if (s0 == 0 && lane == 0)
            a.items[id] = direct ? make_int2(0, 0) : make_int2((int)slot, (lw - fw + 1) << 16 | fw);
        w.finish(0, c.live);
        if (!(MODE == PACK && col >= 8) && row) {
            if (direct)
                w.to_out(0, a, c);
            else
                w.to_piece(0, a.own + slot * piece_floats(a.rows, 64 * ND), a.rows, mine);
        }
        if (!follows) return;
        pos = then, seq = seq2, line = line2, s0 = 0, o = o2, first = false;
    }
}

// Joins the pieces of the own items' rows, TEAM threads a row. The pieces' maxima and sums, a lane each, and the first
// eight pieces' values for each thread are on their way together.
template <int ND, int TEAM>
__global__ __launch_bounds__(TEAM < 256 ? 256 : TEAM) void k_attn_merge(AttnArgs a, int cols) {
    constexpr bool ALL = TEAM >= 256;          // the workgroup's one row
    constexpr int D = 64 * ND, LANES = D / 4;  // lanes that hold a piece's values
    constexpr int MERGE_WAVES = ALL ? TEAM / 64 : 4;
    constexpr int MOST = ALL ? 1024 : 256;  // pieces of a round
    constexpr int SLICES = TEAM / LANES;
    __shared__ float factor[ALL ? 1 : MERGE_WAVES][MOST];
    __shared__ f32x4 sums[ALL ? TEAM : 1];
    __shared__ float red[2][MERGE_WAVES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, t = ALL ? threadIdx.x : lane;
    const int lines = a.kv_heads * a.row_tiles;
    const int64_t id = blockIdx.x;
    const int y = ALL ? blockIdx.y : blockIdx.y * MERGE_WAVES + wave;  // the row in its tile
    const int2 it = a.items[id];
    const int n_pre = a.prefix ? a.head[0] : 0;
    const int own = it.y >> 16, fw = it.y & 0xFFFF;
    if (own == 0) return;  // written where it was made
    const int seq = (int)(id / lines), item = (int)(id % lines);
    const int head = item % a.kv_heads, tile = item / a.kv_heads;
    const int r = tile * cols + y;
    if (y >= a.rows || r >= a.n_q * a.group) return;
    const int all = (seq * a.n_q + r / a.group) * a.group + r % a.group;  // the row among the batch's
    const int64_t own_floats = piece_floats(a.rows, D), pre_floats = piece_floats(16, D);
    // the prefix's pieces of the row's line
    int n = own;
    const float* pre = nullptr;
    const int width = WAVES * a.pre_nt;  // tiles of a line
    if (n_pre > 0) {
        const Prefix p = prefix_of(a);
        const int groups = (a.pre_tiles + width - 1) / width, line = head * groups + (all >> 4) / width;
        const Cuts by((unsigned)p.steps * (unsigned)(a.kv_heads * groups), (unsigned)n_pre);
        const int first = (int)by.of((unsigned)line * p.steps);
        n += (int)by.of((unsigned)line * p.steps + p.steps - 1) - first + 1;
        pre = a.pre + ((int64_t)(first + line) * width + (all >> 4) % width) * pre_floats;
    }
    const auto piece = [&](int i) {
        return i < own ? a.own + (i == 0 ? (int64_t)it.x : 2 * (int64_t)(fw + i)) * own_floats
                       : pre + (int64_t)(i - own) * width * pre_floats;
    };
    float* const fs = factor[ALL ? 0 : wave];
    // what is in a round of pieces joins what was before it: more rounds than one only where pieces are very many
    float M = -INFINITY, L = 0.0f;
    f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int i0 = 0; i0 < n; i0 += MOST) {
        if (ALL && i0) __syncthreads();
        const int k = min(n - i0, MOST), at = (t % LANES) * 4;
        const auto fetch = [&](f32x4 (&v)[8], int from) {  // eight pieces at once
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int j = min(from + u * SLICES, k - 1);
                v[u] = *reinterpret_cast<const f32x4_any*>(piece(i0 + j) + (int64_t)(i0 + j < own ? y : all & 15) * D + at);
            }
        };
        f32x4 v[8];
        fetch(v, t / LANES);
        float top = M;
        for (int i = t; i < k; i += TEAM) {
            const float* p = piece(i0 + i);
            const int rows = i0 + i < own ? a.rows : 16, row = i0 + i < own ? y : all & 15;
            const float m = p[(int64_t)rows * D + row], l = p[(int64_t)rows * D + rows + row];
            fs[i] = l == 0.0f ? -INFINITY : m;  // nothing seen
            if (l != 0.0f) top = fmaxf(top, m);
        }
        top = wave_max(top);
        if (ALL) {
            __syncthreads();
            if (lane == 0) red[0][wave] = top;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < MERGE_WAVES; ++w) top = fmaxf(top, red[0][w]);
        }
        const float f = M == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(M - top);
        M = top;
        float sum = 0.0f;
        for (int i = t; i < k; i += TEAM) {
            const float* p = piece(i0 + i);
            const int rows = i0 + i < own ? a.rows : 16, row = i0 + i < own ? y : all & 15;
            const float l = p[(int64_t)rows * D + rows + row];
            const float e = l * __builtin_amdgcn_exp2f(fs[i] - M);
            fs[i] = l == 0.0f ? -1.0f : e;  // nothing seen: its average may be no number, which is nobody's
            if (l != 0.0f) sum += e;
        }
        sum = (float)wave_sum((double)sum);
        if (ALL) {
            if (lane == 0) red[1][wave] = sum;
            __syncthreads();
            sum = 0.0f;
#pragma unroll
            for (int w = 0; w < MERGE_WAVES; ++w) sum += red[1][w];
        }
        // x is the average of what was joined so far
        const float was = L * f;
        L = was + sum;
        const float part = L == 0.0f ? 0.0f : 1.0f / L;
        x *= was * part;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the lanes read each other's factors
        for (int i = t / LANES; i < k; i += 8 * SLICES) {
            if (i >= 8 * SLICES) fetch(v, i);
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int j = i + u * SLICES;
                const float e = j < k ? fs[j] * part : -1.0f;
                if (!(e < 0.0f)) x += v[u] * e;  // a weight of 0 too: no number among what is seen shows, whatever its weight
            }
        }
    }
    // the slices' sums
    if (ALL) {
        sums[threadIdx.x] = x;
        __syncthreads();
        if (threadIdx.x >= LANES) return;
#pragma unroll
        for (int w = 1; w < SLICES; ++w) x += sums[w * LANES + threadIdx.x];
    } else {
#pragma unroll
        for (int s = LANES; s < 64; s <<= 1)
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] += __shfl_xor(x[e], s);
        if (lane >= LANES) return;
    }
    const bool some = L > 0.0f || L != L;
    const int64_t token = (int64_t)seq * a.n_q + r / a.group;
    const int qh = head * a.group + r % a.group;
    const f32x4 v = some ? x : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const int64_t to = token * a.out_stride + (int64_t)qh * D + 4 * (t % LANES);
    if (a.type == FT_TYPE_F32)
        store_out<true>(a.out, to, false, v);
    else
        store_out<false>(a.out, to, a.type == FT_TYPE_F16, v);
    if (a.lse && t == 0) a.lse[token * a.kv_heads * a.group + qh] = some ? (M + __builtin_amdgcn_logf(L)) * LN2 : -INFINITY;
}

// Threads that join a row: a wavefront where the rows fill the device or have few pieces, four where the device would be
// empty (one sequence of 777 tokens 12.6 us of both kernels, by a wavefront 15.8; 8 of up to 4096 23.1 and 30.0; but 2048 rows
// behind 16390 tokens 66.5 and 64.3, and one sequence of 97, of few pieces, 12.3 and 12.0), sixteen for a handful of rows of
// many pieces (one sequence of 20000 30.7, by four 36.9; 16 rows of 32 pieces 13.5 by sixteen and 12.6 by
// four; 1024 rows of over 64 67.0 and 56.5).
constexpr int PER_WAVE = 16, PER_FOUR = 64;        // pieces
constexpr int ROWS_FOUR = 1024, ROWS_SIXTEEN = 256;

// What a call's sizes make of it.
struct Sizes {
    int cols, rows, row_tiles, pre_tiles, pre_nt, waves;
    int64_t items;
    size_t at_items, at_own, at_pre, bytes;
};

bool sizes_of(Sizes& z, bool f32, int64_t n_seqs, int64_t n_q, int64_t n_heads, int64_t kv_heads, int64_t D) {
    if (n_seqs < 0 || n_seqs > MAX_SEQS || n_q < 1 || n_q > 64 || kv_heads < 1 || kv_heads > 256 ||
        n_heads < kv_heads || n_heads > 4096 || n_heads % kv_heads || (D != 64 && D != 128 && D != 256))
        return false;
    const int64_t rows = n_q * (n_heads / kv_heads);
    z.cols = f32 && rows <= 8 ? 8 : 16;
    z.rows = (int)(rows < z.cols ? rows : z.cols);
    z.row_tiles = (int)((rows + z.cols - 1) / z.cols);
    const int64_t pre_tiles = (n_seqs * rows + 15) / 16;
    z.items = n_seqs * kv_heads * z.row_tiles;
    if (z.items > 1 << 24 || kv_heads * pre_tiles > 1 << 20) return false;
    z.pre_tiles = (int)pre_tiles;
    z.waves = BLOCKS * WAVES;
    z.pre_nt = pre_columns((int)D / 64, f32);
    const auto up = [](size_t v) { return (v + 255) / 256 * 256; };
    z.at_items = 256;
    z.at_own = z.at_items + up((size_t)z.items * 8);
    z.at_pre = z.at_own + up((size_t)(2 * z.waves + z.items) * piece_floats(z.rows, (int)D) * 4);
    // pieces of the prefix: a line's for each workgroup, and one more wherever a line begins in one
    const int64_t width = WAVES * z.pre_nt, lines = kv_heads * ((pre_tiles + width - 1) / width);
    z.bytes = z.at_pre + up((size_t)(BLOCKS + lines) * width * piece_floats(16, (int)D) * 4);
    return true;
}

template <int CT, int ND, int MODE>
void launch_attn(const AttnArgs& a, const Sizes& z, hipStream_t s) {
    const unsigned own = (unsigned)((a.own_waves + WAVES - 1) / WAVES);
    if (a.prefix)
        hipLaunchKernelGGL((k_attn<CT, ND, MODE, true>), dim3(BLOCKS), dim3(THREADS), 0, s, a);
    else
        hipLaunchKernelGGL((k_attn<CT, ND, MODE, false>), dim3(own), dim3(THREADS), 0, s, a);
    // a row's pieces at most, where they are dealt evenly
    const int64_t pieces = a.own_waves / z.items + (a.prefix ? 2 * BLOCKS * z.pre_nt * WAVES / (a.kv_heads * z.pre_tiles) : 0) + 2;
    const auto rows = dim3((unsigned)z.items, (unsigned)z.rows);
    if (pieces > PER_FOUR && z.items * z.rows <= ROWS_SIXTEEN)
        hipLaunchKernelGGL((k_attn_merge<ND, 1024>), rows, dim3(1024), 0, s, a, z.cols);
    else if (pieces > PER_WAVE && z.items * z.rows <= ROWS_FOUR)
        hipLaunchKernelGGL((k_attn_merge<ND, 256>), rows, dim3(256), 0, s, a, z.cols);
    else
        hipLaunchKernelGGL((k_attn_merge<ND, 64>), dim3((unsigned)z.items, (unsigned)((z.rows + 3) / 4)), dim3(256), 0, s, a, z.cols);
}

template <int CT, int ND>
void launch_mode(const AttnArgs& a, const Sizes& z, hipStream_t s) {
    if (a.type != FT_TYPE_F32)
        launch_attn<CT, ND, HALF>(a, z, s);
    else if (z.cols == 8)
        launch_attn<CT, ND, PACK>(a, z, s);
    else
        launch_attn<CT, ND, SPLIT>(a, z, s);
}

template <int CT>
void launch_dim(const AttnArgs& a, const Sizes& z, int64_t D, hipStream_t s) {
    if (D == 64)
        launch_mode<CT, 1>(a, z, s);
    else if (D == 128)
        launch_mode<CT, 2>(a, z, s);
    else
        launch_mode<CT, 4>(a, z, s);
}

}  // namespace

extern "C" size_t ft_hip_attention_workspace_bytes(int64_t n_seqs, int64_t n_q, int64_t n_heads, int64_t n_kv_heads,
                                                   int64_t head_dim) {
    Sizes f, h;
    if (!sizes_of(f, true, n_seqs, n_q, n_heads, n_kv_heads, head_dim) ||
        !sizes_of(h, false, n_seqs, n_q, n_heads, n_kv_heads, head_dim))
        return 0;
    return f.bytes > h.bytes ? f.bytes : h.bytes;
}

extern "C" int ft_hip_attention(ft_hip_ctx* ctx, void* stream, const void* q, int64_t q_stride, int q_type,
                                const void* cache, int cache_type, int64_t n_pages, int64_t page_tokens,
                                int64_t n_kv_heads, int64_t head_dim, const int32_t* tables, int64_t table_stride,
                                int64_t table_pages, const int32_t* lens, const int32_t* prefix, int64_t prefix_pages,
                                const int32_t* prefix_len, int64_t n_seqs, int64_t n_q, int64_t n_heads, float scale,
                                int64_t window, void* out, int64_t out_stride, float* lse, void* workspace,
                                size_t workspace_bytes) {
    clear_error();
    if (!kv_dims_fit(page_tokens, n_kv_heads, head_dim))
        return fail(FT_HIP_E_SHAPE, "attention: page_tokens=%lld (16 to 256, a power of two), n_kv_heads=%lld (1 to 256) or head_dim=%lld (64, 128, 256)",
                    (long long)page_tokens, (long long)n_kv_heads, (long long)head_dim);
    if (!kv_pages_fit(n_pages, page_tokens))
        return fail(FT_HIP_E_SHAPE, "attention: n_pages=%lld not in [1, 2^31 tokens]", (long long)n_pages);
    if (q_type != FT_TYPE_F32 && q_type != FT_TYPE_F16 && q_type != FT_TYPE_BF16)
        return fail(FT_HIP_E_INVALID, "attention: q_type=%d is no FT_TYPE", q_type);
    if (cache_type != FT_KV_I8 && cache_type != FT_KV_E4M3)
        return fail(FT_HIP_E_INVALID, "attention: cache_type=%d is no FT_KV", cache_type);
    if (n_seqs < 0 || n_seqs > MAX_SEQS)
        return fail(FT_HIP_E_SHAPE, "attention: n_seqs=%lld not in [0, %d]", (long long)n_seqs, MAX_SEQS);
    if (n_q < 1 || n_q > 64) return fail(FT_HIP_E_SHAPE, "attention: n_q=%lld not in [1, 64]", (long long)n_q);
    if (n_heads < 1 || n_heads > 4096 || n_heads % n_kv_heads)
        return fail(FT_HIP_E_SHAPE, "attention: n_heads=%lld not in [1, 4096] or no multiple of n_kv_heads=%lld", (long long)n_heads,
                    (long long)n_kv_heads);
    Sizes z;
    if (!sizes_of(z, q_type == FT_TYPE_F32, n_seqs, n_q, n_heads, n_kv_heads, head_dim))
        return fail(FT_HIP_E_SHAPE, "attention: n_seqs=%lld of n_q=%lld queries on n_heads=%lld are too many for one call", (long long)n_seqs,
                    (long long)n_q, (long long)n_heads);
    if (table_pages < 1 || table_pages > INT32_MAX / page_tokens)
        return fail(FT_HIP_E_SHAPE, "attention: table_pages=%lld not in [1, 2^31 tokens]", (long long)table_pages);
    const int64_t cap_steps = z.items * (table_pages * page_tokens / STEP + 2 + START);
    if (cap_steps >= (int64_t)1 << 31)
        return fail(FT_HIP_E_SHAPE, "attention: n_seqs=%lld tables of table_pages=%lld are too many for one call", (long long)n_seqs,
                    (long long)table_pages);
    if (table_stride < table_pages || table_stride > (int64_t)1 << 36)
        return fail(FT_HIP_E_SHAPE, "attention: table_stride out of range");
    if (prefix_pages < 0 || prefix_pages > INT32_MAX / page_tokens || (prefix && prefix_pages < 1))
        return fail(FT_HIP_E_SHAPE, "attention: prefix_pages=%lld not in [1, 2^31 tokens]", (long long)prefix_pages);
    const int64_t tokens_most = (int64_t)(prefix ? prefix_pages : 0) + table_pages;
    if (prefix && z.pre_tiles * n_kv_heads * (prefix_pages * page_tokens / STEP + 2) >= (int64_t)1 << 31)
        return fail(FT_HIP_E_SHAPE, "attention: n_seqs=%lld behind prefix_pages=%lld are too many for one call", (long long)n_seqs,
                    (long long)prefix_pages);
    if (tokens_most > INT32_MAX / page_tokens)
        return fail(FT_HIP_E_SHAPE, "attention: prefix_pages=%lld and table_pages=%lld pass 2^31 tokens", (long long)prefix_pages,
                    (long long)table_pages);
    if (window < 0 || window > INT32_MAX) return fail(FT_HIP_E_SHAPE, "attention: window=%lld not in [0, 2^31)", (long long)window);
    if (!std::isfinite(scale)) return fail(FT_HIP_E_SHAPE, "attention: scale is not finite");
    const int64_t width = n_heads * head_dim, size = q_type == FT_TYPE_F32 ? 4 : 2;
    if (q_stride < width || q_stride > (int64_t)1 << 36 || out_stride < width || out_stride > (int64_t)1 << 36)
        return fail(FT_HIP_E_SHAPE, "attention: q_stride or out_stride out of range");
    if (!aligned(q, size) || !aligned(out, size) || !aligned(cache, 16) || !aligned(tables, 4) || !aligned(lens, 4) ||
        !aligned(prefix, 4) || !aligned(prefix_len, 4) || !aligned(lse, 4) || !aligned(workspace, 16))
        return fail(FT_HIP_E_SHAPE, "attention: a pointer is not aligned to its type (cache and workspace: 16 bytes)");
    // one size for every type
    const size_t need = ft_hip_attention_workspace_bytes(n_seqs, n_q, n_heads, n_kv_heads, head_dim);
    if (need == 0 || workspace_bytes < need)
        return fail(FT_HIP_E_SHAPE, "attention: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    if (!ctx) return fail(FT_HIP_E_INVALID, "attention: null argument");
    if (n_seqs == 0) return FT_HIP_OK;  // an empty tensor has no address
    if (!q || !cache || !tables || !lens || !out || !workspace || (prefix && !prefix_len))
        return fail(FT_HIP_E_INVALID, "attention: null argument");
    const int64_t rows = n_seqs * n_q;
    const Span sq{q, rows, q_stride * size, width * size}, so{out, rows, out_stride * size, width * size},
        sl{lse, 1, 0, rows * n_heads * 4}, sw{workspace, 1, 0, (int64_t)need};
    const Span in[] = {sq,
                       {cache, 1, 0, n_pages * n_kv_heads * kv_block_bytes(page_tokens, head_dim)},
                       {tables, n_seqs, table_stride * 4, table_pages * 4},
                       {lens, 1, 0, n_seqs * 4},
                       {prefix, 1, 0, prefix_pages * 4},
                       {prefix_len, 1, 0, 4}};
    for (const Span& i : in)
        if (overlap(so, i) || overlap(sl, i) || overlap(sw, i))
            return fail(FT_HIP_E_SHAPE, "attention: out, lse or the workspace overlaps an input");
    if (overlap(so, sl) || overlap(so, sw) || overlap(sl, sw))
        return fail(FT_HIP_E_SHAPE, "attention: out, lse and the workspace overlap each other");
    int shift = 4;
    while (1 << shift < page_tokens) ++shift;
    char* const ws = static_cast<char*>(workspace);
    AttnArgs a;
    a.q = q, a.q_stride = q_stride, a.out = out, a.out_stride = out_stride, a.lse = lse;
    a.cache = static_cast<const uint8_t*>(cache), a.tables = tables, a.table_stride = table_stride, a.lens = lens;
    a.prefix = prefix, a.prefix_len = prefix_len, a.prefix_pages = (int)prefix_pages;
    a.table_pages = (int)table_pages, a.n_pages = (int)n_pages, a.page_shift = shift;
    a.n_seqs = (int)n_seqs, a.n_q = (int)n_q, a.kv_heads = (int)n_kv_heads, a.group = (int)(n_heads / n_kv_heads), a.type = q_type;
    a.row_tiles = z.row_tiles, a.pre_tiles = z.pre_tiles, a.pre_nt = z.pre_nt, a.rows = z.rows, a.window = (int)window;
    a.scale = scale * LOG2E;
    a.head = reinterpret_cast<int32_t*>(ws), a.items = reinterpret_cast<int2*>(ws + z.at_items);
    a.own = reinterpret_cast<float*>(ws + z.at_own), a.pre = reinterpret_cast<float*>(ws + z.at_pre);
    a.own_waves = (int)(cap_steps < z.waves ? cap_steps : z.waves);
    DeviceGuard on(ctx->device);
    if (!on.ok) return fail(FT_HIP_E_DEVICE, "attention: device %d cannot be made current", ctx->device);
    if (cache_type == FT_KV_I8)
        launch_dim<FT_KV_I8>(a, z, head_dim, static_cast<hipStream_t>(stream));
    else
        launch_dim<FT_KV_E4M3>(a, z, head_dim, static_cast<hipStream_t>(stream));
    return launch_status("attention");
}
