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
// k_attn_merge joins the pieces. The prefix is a line of its own, of which a
// wavefront takes a piece for 16 rows, whichever sequence they belong to: read
// once per 16 rows of the batch, and by neighbours at the same time.

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
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr int STEP = 32;  // tokens of a step, two tiles
constexpr int THREADS = 256, WAVES = THREADS / 64;
constexpr int MAX_SEQS = FT_ATTN_MAX_SEQS;
constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.693147180559945309417f;

enum { HALF, PACK, SPLIT };

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
    int pre_tiles;   // tiles of the batch's rows on a head
    int window;
    float scale;     // times log2 e
    float pre_cost;  // of a prefix step, in own ones
    // workspace: a word of how many pieces the prefix is cut into, descriptors of the own items, pieces
    int32_t* head;
    int2* items;
    float* own;      // pieces of own rows: `piece` floats each
    float* pre;      // pieces of prefix rows: 16 rows each
    int own_waves;   // at most
    int rows;        // of an own piece
};

// Floats of a piece of `rows` rows: the rows' values, then their maxima and sums.
__host__ __device__ __forceinline__ int64_t piece_floats(int rows, int D) { return (int64_t)rows * (D + 2); }

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

// The pages of a run of tiles, 64 tiles at a time, a lane each; -1 for one that is not in the cache.
struct Pages {
    int first, now, next;  // first: the tile of lane 0
    const int32_t* ids;
    int n;
    __device__ __forceinline__ int list(const AttnArgs& a, int from) const {
        const int at = (from + (int)(threadIdx.x & 63)) >> (a.page_shift - 4);
        const int id = ids[at < n ? at : n - 1];
        return (unsigned)id < (unsigned)a.n_pages ? id : -1;
    }
    __device__ __forceinline__ void open(const AttnArgs& a, const int32_t* pages, int count, int tile) {
        ids = pages, n = count, first = tile;
        now = list(a, tile), next = list(a, tile + 64);
    }
    // To the tiles from `tile` on, which is an even number from the first.
    __device__ __forceinline__ void reach(const AttnArgs& a, int tile) {
        if (tile - first < 64) return;
        first += 64;
        now = next;
        next = list(a, first + 64);
    }
    __device__ __forceinline__ int page(int tile) const { return __builtin_amdgcn_readlane(now, tile - first); }
};

// Two tiles of a head's tokens, on their way.
template <int ND>
struct Step {
    static constexpr int D = 64 * ND;
    u32x4 k[2][ND], v[2][ND];
    f32x4 dk[2], dv[2];

    // Where the tiles `tile` and `tile` + 1 of a list lie that ends before tile `end`.
    struct Aim {
        int page[2];
        const uint8_t* block[2];
        int in[2], lane16, lane64;
        // some: there are such tiles; if not, what is loaded is of no use, and all lanes load the same
        __device__ __forceinline__ void at(const AttnArgs& a, Pages& p, int head, int tile, int end, bool some) {
            p.reach(a, tile);
            const int mask = (1 << (a.page_shift - 4)) - 1, lane = threadIdx.x & 63;
            page[0] = some ? p.page(tile) : -1, page[1] = some && tile + 1 < end ? p.page(tile + 1) : -1;
            lane16 = some ? lane * 16 : 0, lane64 = some ? lane >> 4 << 4 : 0;
#pragma unroll
            for (int x = 0; x < 2; ++x) {  // instead of a page that is not there the first
                block[x] = a.cache + ((int64_t)max(page[x], 0) * a.kv_heads + head) * kv_block_bytes((int64_t)1 << a.page_shift, D);
                in[x] = (tile + x) & mask;
            }
        }
    };
    __device__ __forceinline__ void load_k(const AttnArgs& a, const Aim& m) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const uint8_t* p = m.block[x] + m.in[x] * (16 * D);
#pragma unroll
            for (int c = 0; c < ND; ++c) k[x][c] = *reinterpret_cast<const u32x4*>(p + c * 1024 + m.lane16);
            dk[x] = *reinterpret_cast<const f32x4*>(m.block[x] + ((int64_t)(2 * D) << a.page_shift) + m.in[x] * 64 + m.lane64);
        }
    }
    __device__ __forceinline__ void load_v(const AttnArgs& a, const Aim& m) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const uint8_t* p = m.block[x] + ((int64_t)D << a.page_shift) + m.in[x] * (16 * D);
#pragma unroll
            for (int c = 0; c < ND; ++c) v[x][c] = *reinterpret_cast<const u32x4*>(p + c * 1024 + m.lane16);
            dv[x] = *reinterpret_cast<const f32x4*>(m.block[x] + ((int64_t)(2 * D + 4) << a.page_shift) + m.in[x] * 64 + m.lane64);
        }
    }
};

// A wavefront's NT times 16 columns (PACK: 8 rows).
template <int CT, int ND, int MODE, int NT>
struct Attend {
    static constexpr int D = 64 * ND;
    static constexpr int PARTS = MODE == SPLIT ? 2 : 1;
    static constexpr bool F32 = MODE != HALF;
    half8 q[NT][PARTS][2 * ND];
    f32x4 acc[NT][4 * ND];
    float m[NT], base[NT], l[NT], fac[NT];
    float unit, inv_unit;  // the weights' unit: the values' largest scale so far as a power of two, over 2^8
    int lo[NT], hi[NT];    // tokens that the column sees
    int all_lo, all_hi;    // that every column sees
    int tokens;            // that the list of pages holds

    __device__ __forceinline__ void load(const AttnArgs& a, int n, const Column& c) {
        const int g = (threadIdx.x & 63) >> 4;
        float x[2 * ND][8], top = 0.0f;
        const int64_t at = ((int64_t)c.seq * a.n_q + c.t) * a.q_stride + (int64_t)c.head * D + 16 * g;
#pragma unroll
        for (int i = 0; i < 2 * ND; ++i) load_q8<F32>(a.q, at + (i >> 1) * 64 + (i & 1) * 8, a.type == FT_TYPE_F16, x[i]);
#pragma unroll
        for (int i = 0; i < 2 * ND; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[i][e]));
        top = max_groups(top);
        const int e2 = max(__float_as_int(top) >> 23, 10);
        const float up = __int_as_float((263 - e2) << 23);  // the row's largest comes to lie in [2^9, 2^10)
        fac[n] = a.scale * __int_as_float((e2 - 9) << 23);
        const float second = MODE == PACK && (threadIdx.x & 8) ? 1.0f : 0.0f;
#pragma unroll
        for (int i = 0; i < 2 * ND; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float v = x[i][e] * up;
                const _Float16 h = (_Float16)v;
                if constexpr (MODE == SPLIT) q[n][PARTS - 1][i][e] = (_Float16)(v - (float)h);
                q[n][0][i][e] = MODE == PACK ? (_Float16)(v - second * (float)h) : h;
            }
#pragma unroll
        for (int i = 0; i < 4 * ND; ++i) acc[n][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        m[n] = -INFINITY, base[n] = 0.0f, l[n] = 0.0f, unit = 0x1p-100f, inv_unit = 0x1p100f;
    }

    // The columns' scores of a step; the keys and their scales are free afterwards.
    __device__ __forceinline__ void scores(const Step<ND>& t, f32x4 (&s)[NT][2]) const {
#pragma unroll
        for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < ND; ++c)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const half8 k = widen8<CT>(t.k[x][c][2 * h], t.k[x][c][2 * h + 1]);
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int p = 0; p < PARTS; ++p) s[n][x] = mfma(k, q[n][p][2 * c + h], s[n][x]);
                }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                if constexpr (MODE == PACK) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[n][x][i] += other8(s[n][x][i]);
                }
                s[n][x] *= t.dk[x] * fac[n];
            }
    }

    // Weights of a step at token `at` from its scores, and their sums with the values.
    __device__ __forceinline__ void weigh(Step<ND>& t, f32x4 (&s)[NT][2], const int (&page)[2], int at) {
        const int lane = threadIdx.x & 63, g = lane >> 4;
        const bool whole = page[0] >= 0 && page[1] >= 0 && at >= all_lo && at + STEP <= all_hi;
        half8 w[NT][PARTS];
        float top[NT];
        f32x4 dv[2] = {t.dv[0], t.dv[1]};
        bool grows = false;
        if (!whole) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                uint32_t keep = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int j = at + 16 * x + 4 * g + i;
                    // tokens that the list does not hold may have codes and scales that are NaN, whose 0 fold is NaN
                    const bool in = page[x] >= 0 && j < tokens;
                    if (in) keep |= 255u << (8 * i);
                    if (!in) dv[x][i] = 0.0f;
#pragma unroll
                    for (int n = 0; n < NT; ++n)
                        if (!in || j < lo[n] || j >= hi[n]) s[n][x][i] = -INFINITY;
                }
#pragma unroll
                for (int c = 0; c < ND; ++c) t.v[x][c] &= keep;
            }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            top[n] = fmaxf(fmaxf(fmaxf(s[n][0][0], s[n][0][1]), fmaxf(s[n][0][2], s[n][0][3])),
                           fmaxf(fmaxf(s[n][1][0], s[n][1][1]), fmaxf(s[n][1][2], s[n][1][3])));
            top[n] = max_groups(top[n]);
            grows |= top[n] > m[n] + 6.0f;
        }
        const float vt = fmaxf(fmaxf(fmaxf(dv[0][0], dv[0][1]), fmaxf(dv[0][2], dv[0][3])),
                               fmaxf(fmaxf(dv[1][0], dv[1][1]), fmaxf(dv[1][2], dv[1][3])));
        if (__any(grows || vt > unit * 256.0f)) rescale(top, vt);
#pragma unroll
        for (int x = 0; x < 2; ++x) dv[x] *= inv_unit;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const float second = MODE == PACK && (lane & 8) ? 1.0f : 0.0f;
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float p = __builtin_amdgcn_exp2f(s[n][x][i] - base[n]);
                    l[n] += p;
                    float v = p * dv[x][i];
                    // a scale that is NaN, of a token that the column does not see
                    if (!whole && s[n][x][i] == -INFINITY) v = 0.0f;
                    const _Float16 h = (_Float16)v;
                    w[n][0][4 * x + i] = MODE == PACK ? (_Float16)(v - second * (float)h) : h;
                    if constexpr (MODE == SPLIT) w[n][PARTS - 1][4 * x + i] = (_Float16)(v - (float)h);
                }
        }
#pragma unroll
        for (int c = 0; c < ND; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const half8 v = widen8<CT>(t.v[0][c][j], t.v[1][c][j]);
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int p = 0; p < PARTS; ++p) acc[n][4 * c + j] = mfma(v, w[n][p], acc[n][4 * c + j]);
            }
    }

    // A larger maximum, or a larger scale of values.
    __device__ __forceinline__ void rescale(const float (&top)[NT], float vt) {
        float g = 1.0f;
        const float most = wave_max(vt);
        if (most > unit * 256.0f) {
            const int e = clampi((__float_as_int(most) >> 23) + 1, 30, 254);
            const float to = __int_as_float((e - 8) << 23);
            inv_unit = __int_as_float((254 - (e - 8)) << 23);
            g = unit * inv_unit;
            unit = to;
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            float f = g;
            if (top[n] > m[n]) {
                const float d = __builtin_amdgcn_exp2f(m[n] - top[n]);
                f *= d;
                l[n] *= d;
                m[n] = base[n] = top[n];
            }
#pragma unroll
            for (int i = 0; i < 4 * ND; ++i) acc[n][i] *= f;
        }
    }

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
    __device__ __forceinline__ void to_piece(int n, float* piece, int rows, int col) const {
        const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
        for (int c = 0; c < ND; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<f32x4*>(piece + (int64_t)col * D + 64 * c + 16 * g + 4 * i) = values(n, c, i, unit);
        if (g == 0) {
            piece[(int64_t)rows * D + col] = m[n];
            piece[(int64_t)rows * D + rows + col] = l[n];
        }
    }
    __device__ __forceinline__ void to_out(int n, const AttnArgs& a, const Column& c) const {
        const int g = (threadIdx.x & 63) >> 4;
        const int64_t row = (int64_t)c.seq * a.n_q + c.t;
        const bool some = l[n] > 0.0f || l[n] != l[n];
        const float f = some ? unit / l[n] : 0.0f;
#pragma unroll
        for (int i = 0; i < ND; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                store_out<F32>(a.out, row * a.out_stride + (int64_t)c.head * D + 64 * i + 16 * g + 4 * e, a.type == FT_TYPE_F16,
                               some ? values(n, i, e, f) : f32x4{0.0f, 0.0f, 0.0f, 0.0f});
        if (a.lse && g == 0)
            a.lse[row * a.kv_heads * a.group + c.head] = some ? (m[n] + __builtin_amdgcn_logf(l[n])) * LN2 : -INFINITY;
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
// first.
constexpr int start_of(int nd) { return 4 / nd; }

constexpr int MIN_STEPS = 2;  // of a wavefront's own steps, where there are more than FEW_STEPS in all
constexpr int FEW_STEPS = 1024;

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
constexpr int pre_columns(int nd, bool f32) { return f32 ? (nd <= 2 ? 2 : 1) : 4 / nd; }

// Prefix rows: a wavefront takes a piece of the prefix for NT tiles of 16 rows.
template <int CT, int ND, int MODE, int NT>
__device__ __forceinline__ void attend_prefix(const AttnArgs& a, const Prefix& pre, int cuts, int x0, int stride) {
    const int lane = threadIdx.x & 63, col = lane & 15;
    const int groups = (a.pre_tiles + NT - 1) / NT;
    for (int x = x0; x < cuts * a.kv_heads * groups; x += stride) {
        const int tile = uni(x % groups) * NT, seg = x / groups;
        const int head = uni(seg / cuts), cut = uni(seg % cuts);
        const Cuts by((unsigned)pre.steps, (unsigned)cuts);
        int s0 = (int)by.begin(cut), s1 = (int)by.begin(cut + 1);
        Pages pages;
        pages.open(a, a.prefix, a.prefix_pages, pre.tile0 + 2 * s0);
        Attend<CT, ND, MODE, NT> w;
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
            const int lo = a.window ? max(0, pre.len + at - a.window + 1) : 0;
            w.lo[n] = c[n].live ? lo : INT32_MIN, w.hi[n] = pre.len;  // one without a query sees all, to no effect
            if (c[n].live) least = min(least, lo), most_lo = max(most_lo, lo);
        }
        w.tokens = w.all_hi = pre.len, w.all_lo = -least_of_wave(-most_lo);
        // the steps before the first column's first token are nobody's
        const int skip = (least_of_wave(least) / 16 - pre.tile0) / 2;
        if (skip > s0) s0 = min(skip, s1), pages.open(a, a.prefix, a.prefix_pages, pre.tile0 + 2 * s0);
        Step<ND> t;
        typename Step<ND>::Aim aim;
        const int end = (pre.len + 15) / 16;
        int at = pre.tile0 + 2 * s0;
        aim.at(a, pages, head, at, end, s0 < s1);
        t.load_k(a, aim);
        t.load_v(a, aim);
#pragma unroll
        for (int n = 0; n < NT; ++n) w.load(a, n, c[n]);
        for (int s = s0; s < s1; ++s) {
            f32x4 sc[NT][2];
            const int page[2] = {aim.page[0], aim.page[1]};
            aim.at(a, pages, head, at + 2, end, s + 1 < s1);
            w.scores(t, sc);
            t.load_k(a, aim);
            w.weigh(t, sc, page, at * 16);
            t.load_v(a, aim);
            at += 2;
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            w.finish(n, c[n].live);
            if (tile + n < a.pre_tiles)
                w.to_piece(n, a.pre + ((int64_t)seg * a.pre_tiles + tile + n) * piece_floats(16, 64 * ND), 16, col);
        }
    }
}

template <int CT, int ND, int MODE, bool PRE>
__global__ __launch_bounds__(THREADS, 2) void k_attn(AttnArgs a) {
    constexpr int COLS = MODE == PACK ? 8 : 16, START = start_of(ND);
    __shared__ int cum[MAX_SEQS + 1], lens[MAX_SEQS];
    __shared__ int part[WAVES];
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
    int n_own = (a.own_waves + WAVES - 1) / WAVES, cuts = 0;
    if constexpr (PRE) {
        constexpr int NT = pre_columns(ND, MODE != HALF);
        const Prefix pre = prefix_of(a);
        if (pre.steps > 0) {
            // the workgroups are dealt by the steps; a prefix step is worth PRE_COST own ones
            const unsigned groups = a.kv_heads * ((a.pre_tiles + NT - 1) / NT);
            const float work = (float)pre.steps * (float)groups * a.pre_cost, all = work + (float)T;
            const int blocks = gridDim.x;
            n_own = min(n_own, clampi((int)((float)T / all * (float)blocks + 0.5f), 1, blocks - 1));
            const int n_pre = blocks - n_own;
            cuts = clampi((int)((unsigned)n_pre * WAVES / groups), 1, (pre.steps + MIN_STEPS - 1) / MIN_STEPS);
            if ((int)blockIdx.x >= n_own) {
                if ((int)blockIdx.x == n_own && t == 0) a.head[0] = cuts;
                const int b = near_block(blockIdx.x - n_own, n_pre);
                attend_prefix<CT, ND, MODE == PACK ? SPLIT : MODE, NT>(a, pre, cuts, uni(b * WAVES + (t >> 6)), n_pre * WAVES);
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
    Pages pages;
    pages.open(a, a.tables + seq * a.table_stride, a.table_pages, o.tile0 + 2 * s0);
    Step<ND> st;
    typename Step<ND>::Aim aim;
    aim.at(a, pages, line % a.kv_heads, o.tile0 + 2 * s0, (o.len + 15) / 16, o.len > 0);
    st.load_k(a, aim);
    st.load_v(a, aim);
    bool first = true;
    while (true) {
        const int head = line % a.kv_heads, tile = line / a.kv_heads;
        const int s1 = min(o.steps, s0 + (int)(end - pos)), last = (o.len + 15) / 16;
        // the item behind this one: its pages are on their way while this one is worked on
        const unsigned then = pos + (s1 - s0) + START;
        const bool follows = then < end;
        int seq2 = seq, line2 = line + 1;
        Own o2 = o;
        Pages pages2 = pages;
        if (follows) {
            if (line2 == (int)lines) {
                seq2 = seq + 1, line2 = 0;
                o2 = own_of(a, uni(lens[seq2]));
            }
            pages2.open(a, a.tables + seq2 * a.table_stride, a.table_pages, o2.tile0);
        }
        Column c;
        const int mine = MODE == PACK ? col & 7 : col;
        const int rows = a.n_q * a.group, r = tile * COLS + mine;
        const bool row = r < rows;
        c.seq = seq, c.t = row ? r / a.group : 0, c.head = head * a.group + (row ? r % a.group : 0);
        const int place = o.len - a.n_q + c.t;
        c.live = row && place >= 0;
        Attend<CT, ND, MODE, 1> w;
        w.load(a, 0, c);
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
            const int page[2] = {aim.page[0], aim.page[1]};
            if (s + 1 < s1) {
                aim.at(a, pages, head, at + 2, last, true);
            } else {
                pages = pages2;
                aim.at(a, pages, line2 % a.kv_heads, follows ? o2.tile0 : pages.first, (o2.len + 15) / 16, follows && o2.len > 0);
            }
            f32x4 sc[1][2];
            w.scores(st, sc);
            st.load_k(a, aim);
            if (o.len > 0) w.weigh(st, sc, page, at * 16);
            st.load_v(a, aim);
            at += 2;
        }
        // what other wavefronts have of the item
        const unsigned item_at = cum[seq] * lines + line * (o.steps + START) + START;
        const int fw = (int)by.of(item_at), lw = (int)by.of(item_at + o.steps - 1);
        const int64_t id = (int64_t)seq * lines + line;
        const bool direct = fw == lw && cuts == 0;
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

// Joins the pieces of the own items' rows: a wavefront a row, or with ALL the
// whole workgroup. First the pieces' maxima and sums, a lane each, then their
// values, several pieces at a time.
template <int ND, bool ALL>
__global__ __launch_bounds__(ALL ? 1024 : 256) void k_attn_merge(AttnArgs a, int cols) {
    constexpr int D = 64 * ND, LANES = D / 4;  // lanes that hold a piece's values
    constexpr int MERGE_WAVES = ALL ? 16 : 4;
    constexpr int MOST = ALL ? 1024 : 256;  // pieces of a round
    constexpr int TEAM = ALL ? 1024 : 64, SLICES = TEAM / LANES;
    __shared__ float factor[ALL ? 1 : MERGE_WAVES][MOST];
    __shared__ f32x4 sums[ALL ? TEAM : 1];
    __shared__ float red[2][MERGE_WAVES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, t = ALL ? threadIdx.x : lane;
    const int lines = a.kv_heads * a.row_tiles;
    const int64_t id = blockIdx.x;
    const int y = ALL ? blockIdx.y : blockIdx.y * MERGE_WAVES + wave;  // the row in its tile
    const int2 it = a.items[id];
    const int cuts = a.prefix ? a.head[0] : 0;
    const int own = it.y >> 16, fw = it.y & 0xFFFF;
    if (own == 0) return;  // written where it was made
    const int seq = (int)(id / lines), item = (int)(id % lines);
    const int head = item % a.kv_heads, tile = item / a.kv_heads;
    const int r = tile * cols + y;
    if (y >= a.rows || r >= a.n_q * a.group) return;
    const int all = (seq * a.n_q + r / a.group) * a.group + r % a.group;  // the row among the batch's
    const int64_t own_floats = piece_floats(a.rows, D), pre_floats = piece_floats(16, D);
    const int n = own + cuts;
    const auto piece = [&](int i) {
        return i < own ? a.own + (i == 0 ? (int64_t)it.x : 2 * (int64_t)(fw + i)) * own_floats
                       : a.pre + ((int64_t)(head * cuts + i - own) * a.pre_tiles + (all >> 4)) * pre_floats;
    };
    float* const fs = factor[ALL ? 0 : wave];
    // what is in a round of pieces joins what was before it: more rounds than one only where pieces are very many
    float M = -INFINITY, L = 0.0f;
    f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int i0 = 0; i0 < n; i0 += MOST) {
        if (ALL && i0) __syncthreads();
        const int k = min(n - i0, MOST);
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
            const float e = l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(fs[i] - M);
            fs[i] = e;
            sum += l * e;
        }
        sum = (float)wave_sum((double)sum);
        if (ALL) {
            if (lane == 0) red[1][wave] = sum;
            __syncthreads();
            sum = 0.0f;
#pragma unroll
            for (int w = 0; w < MERGE_WAVES; ++w) sum += red[1][w];
        }
        L = L * f + sum;
        x *= f;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the lanes read each other's factors
        const int at = (t % LANES) * 4;
        for (int i = t / LANES; i < k; i += 8 * SLICES) {  // eight pieces at once on their way
            f32x4 v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int j = min(i + u * SLICES, k - 1);
                v[u] = *reinterpret_cast<const f32x4*>(piece(i0 + j) + (int64_t)(i0 + j < own ? y : all & 15) * D + at);
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int j = i + u * SLICES;
                const float e = j < k ? fs[j] : 0.0f;
                if (e != 0.0f) x += v[u] * e;  // what was seen by nobody may be no number
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
    const f32x4 v = some ? x * (1.0f / L) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const int64_t to = token * a.out_stride + (int64_t)qh * D + 4 * (t % LANES);
    if (a.type == FT_TYPE_F32)
        store_out<true>(a.out, to, false, v);
    else
        store_out<false>(a.out, to, a.type == FT_TYPE_F16, v);
    if (a.lse && t == 0) a.lse[token * a.kv_heads * a.group + qh] = some ? (M + __builtin_amdgcn_logf(L)) * LN2 : -INFINITY;
}

// What a call's sizes make of it.
struct Sizes {
    int cols, rows, row_tiles, pre_tiles;
    int64_t items, lines_pre;
    size_t at_items, at_own, at_pre, bytes;
};
// Workgroups: two on each CU.
constexpr int BLOCKS = 512, OWN_WAVES = BLOCKS * WAVES;

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
    z.lines_pre = kv_heads * pre_tiles;
    if (z.items > 1 << 24 || z.lines_pre > 1 << 24) return false;
    z.pre_tiles = (int)pre_tiles;
    const auto up = [](size_t v) { return (v + 255) / 256 * 256; };
    z.at_items = 256;
    z.at_own = z.at_items + up((size_t)z.items * 8);
    z.at_pre = z.at_own + up((size_t)(2 * OWN_WAVES + z.items) * piece_floats(z.rows, (int)D) * 4);
    // pieces of the prefix: one for each of a wavefront's tiles, or for each line where there are more of those
    const int64_t pieces = (int64_t)OWN_WAVES * pre_columns((int)D / 64, f32);
    z.bytes = z.at_pre + up((size_t)(z.lines_pre > pieces ? z.lines_pre : pieces) * piece_floats(16, (int)D) * 4);
    return true;
}

template <int CT, int ND, int MODE>
void launch_attn(const AttnArgs& a, const Sizes& z, hipStream_t s) {
    const unsigned own = (unsigned)((a.own_waves + WAVES - 1) / WAVES);
    if (a.prefix)
        hipLaunchKernelGGL((k_attn<CT, ND, MODE, true>), dim3(BLOCKS), dim3(THREADS), 0, s, a);
    else
        hipLaunchKernelGGL((k_attn<CT, ND, MODE, false>), dim3(own), dim3(THREADS), 0, s, a);
    if (z.items * z.rows > 256)  // rows enough for a wavefront each
        hipLaunchKernelGGL((k_attn_merge<ND, false>), dim3((unsigned)z.items, (unsigned)((z.rows + 3) / 4)), dim3(256), 0, s, a,
                           z.cols);
    else
        hipLaunchKernelGGL((k_attn_merge<ND, true>), dim3((unsigned)z.items, (unsigned)z.rows), dim3(1024), 0, s, a, z.cols);
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

extern "C" int ft_hip_attention(ft_hip_ctx* ctx, void* stream, const void* q, int64_t q_stride, int type,
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
    if (type != FT_TYPE_F32 && type != FT_TYPE_F16 && type != FT_TYPE_BF16)
        return fail(FT_HIP_E_INVALID, "attention: type=%d is no FT_TYPE", type);
    if (cache_type != FT_KV_I8 && cache_type != FT_KV_E4M3)
        return fail(FT_HIP_E_INVALID, "attention: cache_type=%d is no FT_KV", cache_type);
    if (n_seqs < 0 || n_seqs > MAX_SEQS)
        return fail(FT_HIP_E_SHAPE, "attention: n_seqs=%lld not in [0, %d]", (long long)n_seqs, MAX_SEQS);
    if (n_q < 1 || n_q > 64) return fail(FT_HIP_E_SHAPE, "attention: n_q=%lld not in [1, 64]", (long long)n_q);
    if (n_heads < 1 || n_heads > 4096 || n_heads % n_kv_heads)
        return fail(FT_HIP_E_SHAPE, "attention: n_heads=%lld not in [1, 4096] or no multiple of n_kv_heads=%lld", (long long)n_heads,
                    (long long)n_kv_heads);
    Sizes z;
    if (!sizes_of(z, type == FT_TYPE_F32, n_seqs, n_q, n_heads, n_kv_heads, head_dim))
        return fail(FT_HIP_E_SHAPE, "attention: n_seqs=%lld of n_q=%lld queries on n_heads=%lld are too many for one call", (long long)n_seqs,
                    (long long)n_q, (long long)n_heads);
    if (table_pages < 1 || table_pages > INT32_MAX / page_tokens)
        return fail(FT_HIP_E_SHAPE, "attention: table_pages=%lld not in [1, 2^31 tokens]", (long long)table_pages);
    const int64_t cap_steps = z.items * (table_pages * page_tokens / STEP + 2 + start_of((int)head_dim / 64));
    if (cap_steps >= (int64_t)1 << 31)
        return fail(FT_HIP_E_SHAPE, "attention: n_seqs=%lld tables of table_pages=%lld are too many for one call", (long long)n_seqs,
                    (long long)table_pages);
    if (table_stride < table_pages || table_stride > (int64_t)1 << 36)
        return fail(FT_HIP_E_SHAPE, "attention: table_stride out of range");
    if (prefix_pages < 0 || prefix_pages > INT32_MAX / page_tokens || (prefix && prefix_pages < 1))
        return fail(FT_HIP_E_SHAPE, "attention: prefix_pages=%lld not in [1, 2^31 tokens]", (long long)prefix_pages);
    const int64_t tokens_most = (int64_t)(prefix ? prefix_pages : 0) + table_pages;
    if (tokens_most > INT32_MAX / page_tokens)
        return fail(FT_HIP_E_SHAPE, "attention: prefix_pages=%lld and table_pages=%lld pass 2^31 tokens", (long long)prefix_pages,
                    (long long)table_pages);
    if (window < 0 || window > INT32_MAX) return fail(FT_HIP_E_SHAPE, "attention: window=%lld not in [0, 2^31)", (long long)window);
    if (!std::isfinite(scale)) return fail(FT_HIP_E_SHAPE, "attention: scale is not finite");
    const int64_t width = n_heads * head_dim, size = type == FT_TYPE_F32 ? 4 : 2;
    if (q_stride < width || q_stride > (int64_t)1 << 36 || out_stride < width || out_stride > (int64_t)1 << 36)
        return fail(FT_HIP_E_SHAPE, "attention: q_stride or out_stride out of range");
    if (!aligned(q, size) || !aligned(out, size) || !aligned(cache, 16) || !aligned(tables, 4) || !aligned(lens, 4) ||
        !aligned(prefix, 4) || !aligned(prefix_len, 4) || !aligned(lse, 4) || !aligned(workspace, 16))
        return fail(FT_HIP_E_SHAPE, "attention: a pointer is not aligned to its type (cache and workspace: 16 bytes)");
    if (workspace_bytes < z.bytes)
        return fail(FT_HIP_E_SHAPE, "attention: workspace of %zu bytes, %zu needed", workspace_bytes, z.bytes);
    if (!ctx) return fail(FT_HIP_E_INVALID, "attention: null argument");
    if (n_seqs == 0) return FT_HIP_OK;  // an empty tensor has no address
    if (!q || !cache || !tables || !lens || !out || !workspace || (prefix && !prefix_len))
        return fail(FT_HIP_E_INVALID, "attention: null argument");
    const int64_t rows = n_seqs * n_q;
    const Span sq{q, rows, q_stride * size, width * size}, so{out, rows, out_stride * size, width * size},
        sl{lse, 1, 0, rows * n_heads * 4}, sw{workspace, 1, 0, (int64_t)z.bytes};
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
    a.n_seqs = (int)n_seqs, a.n_q = (int)n_q, a.kv_heads = (int)n_kv_heads, a.group = (int)(n_heads / n_kv_heads), a.type = type;
    a.row_tiles = z.row_tiles, a.pre_tiles = z.pre_tiles, a.rows = z.rows, a.window = (int)window;
    a.scale = scale * LOG2E;
    a.pre_cost = 1.0f;
    a.head = reinterpret_cast<int32_t*>(ws), a.items = reinterpret_cast<int2*>(ws + z.at_items);
    a.own = reinterpret_cast<float*>(ws + z.at_own), a.pre = reinterpret_cast<float*>(ws + z.at_pre);
    a.own_waves = (int)(cap_steps < OWN_WAVES ? cap_steps : OWN_WAVES);
    DeviceGuard on(ctx->device);
    if (!on.ok) return fail(FT_HIP_E_DEVICE, "attention: device %d cannot be made current", ctx->device);
    if (cache_type == FT_KV_I8)
        launch_dim<FT_KV_I8>(a, z, head_dim, static_cast<hipStream_t>(stream));
    else
        launch_dim<FT_KV_E4M3>(a, z, head_dim, static_cast<hipStream_t>(stream));
    return launch_status("attention");
}
