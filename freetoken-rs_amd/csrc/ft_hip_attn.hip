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
    bool q_vec, out_vec;
    // workspace: a word of how many pieces the prefix is cut into, descriptors of the own items, pieces
    int32_t* head;
    int2* items;
    float* own;      // pieces of own rows: `piece` floats each
    float* pre;      // pieces of prefix rows: 16 rows each
    int own_waves, pre_waves;  // at most
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

// Eight consecutive values of a query as f32.
__device__ __forceinline__ void load_q8(const void* q, int64_t at, int type, bool vec, float* x) {
    if (type == FT_TYPE_F32) {
        const float* p = static_cast<const float*>(q) + at;
        if (vec) {
            const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
            x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = p[i];
        }
        return;
    }
    const uint16_t* p = static_cast<const uint16_t*>(q) + at;
    uint16_t b[8];
    if (vec) {
        const uint4 a = *reinterpret_cast<const uint4*>(p);
        __builtin_memcpy(b, &a, 16);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) b[i] = p[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = type == FT_TYPE_F16 ? h2f(b[i]) : __uint_as_float((uint32_t)b[i] << 16);
}

__device__ __forceinline__ void store_out(void* out, int64_t at, int type, bool vec, f32x4 v) {
    if (type == FT_TYPE_F32) {
        float* p = static_cast<float*>(out) + at;
        if (vec) {
            *reinterpret_cast<f32x4*>(p) = v;
        } else {
            p[0] = v[0], p[1] = v[1], p[2] = v[2], p[3] = v[3];
        }
        return;
    }
    uint16_t* p = static_cast<uint16_t*>(out) + at;
    uint16_t b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t w = __float_as_uint(v[i]);
        b[i] = type == FT_TYPE_F16                      ? f2h(v[i])
               : (w & 0x7FFFFFFFu) > 0x7F800000u ? (uint16_t)(w >> 16 | 0x40)
                                                        : (uint16_t)((w + 0x7FFF + (w >> 16 & 1)) >> 16);
    }
    if (vec)
        *reinterpret_cast<uint2*>(p) = make_uint2(b[0] | (uint32_t)b[1] << 16, b[2] | (uint32_t)b[3] << 16);
    else
        p[0] = b[0], p[1] = b[1], p[2] = b[2], p[3] = b[3];
}

// Which query a column of a wavefront holds.
struct Column {
    int seq, t, head;  // t: which of the sequence's new tokens
    bool live;         // there is such a row, and its query is no padding
    bool row;          // there is such a row
};

// A wavefront's columns over some of a list of pages.
template <int CT, int ND, int MODE>
struct Attend {
    static constexpr int D = 64 * ND, BLOCK16 = 16 * D;
    static constexpr int PARTS = MODE == SPLIT ? 2 : 1;
    half8 q[PARTS][2 * ND];
    f32x4 acc[4 * ND];
    float m, base, l, fac;
    float unit, inv_unit;  // the weights' unit: the values' largest scale so far as a power of two, over 2^8
    int lo, hi;            // tokens that the column sees
    int all_lo, all_hi;    // that every column sees
    int tokens;            // that the list of pages holds

    // The lane's column's query. vec: rows start on 16 bytes.
    __device__ __forceinline__ void load(const AttnArgs& a, const Column& c) {
        const int g = (threadIdx.x & 63) >> 4;
        float x[2 * ND][8], top = 0.0f;
        const int64_t at = ((int64_t)c.seq * a.n_q + c.t) * a.q_stride + (int64_t)c.head * D + 16 * g;
#pragma unroll
        for (int i = 0; i < 2 * ND; ++i) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[i][e] = 0.0f;
            if (c.live) load_q8(a.q, at + (i >> 1) * 64 + (i & 1) * 8, a.type, a.q_vec, x[i]);
        }
#pragma unroll
        for (int i = 0; i < 2 * ND; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[i][e]));
        top = max_groups(top);
        const int e2 = max(__float_as_int(top) >> 23, 10);
        const float up = __int_as_float((263 - e2) << 23);  // the row's largest comes to lie in [2^9, 2^10)
        fac = a.scale * __int_as_float((e2 - 9) << 23);
        const bool second = MODE == PACK && (threadIdx.x & 8);
#pragma unroll
        for (int i = 0; i < 2 * ND; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float v = x[i][e] * up;
                const _Float16 h = (_Float16)v;
                if constexpr (MODE == SPLIT) q[PARTS - 1][i][e] = (_Float16)(v - (float)h);
                q[0][i][e] = MODE == PACK && second ? (_Float16)(v - (float)h) : h;
            }
#pragma unroll
        for (int i = 0; i < 4 * ND; ++i) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        m = -INFINITY, base = 0.0f, l = 0.0f, unit = 0x1p-100f, inv_unit = 0x1p100f;
    }

    // Tokens that the lane's column sees: [from, to) of n; one without a query sees all n, to no effect (what lies
    // behind them may hold any scale, and the largest is the wavefront's unit).
    __device__ __forceinline__ void see(int from, int to, bool live, int n) {
        lo = live ? from : INT32_MIN, hi = live ? to : n, tokens = n;
        int x = lo, y = hi;
#pragma unroll
        for (int s = 1; s < 64; s <<= 1) {
            x = max(x, __shfl_xor(x, s));
            y = min(y, __shfl_xor(y, s));
        }
        all_lo = uni(x), all_hi = uni(y);
    }

    struct Tile {
        u32x4 k[ND], v[ND];
        f32x4 dk, dv;
    };

    __device__ __forceinline__ const uint8_t* block_of(const AttnArgs& a, int page, int head) const {
        const int at = page < 0 ? 0 : page;
        return a.cache + ((int64_t)at * a.kv_heads + head) * kv_block_bytes((int64_t)1 << a.page_shift, D);
    }
    __device__ __forceinline__ void load_k(const AttnArgs& a, const uint8_t* block, int tile, Tile& t) const {
        const int lane = threadIdx.x & 63;
        const uint8_t* p = block + tile * BLOCK16;
#pragma unroll
        for (int c = 0; c < ND; ++c) t.k[c] = *reinterpret_cast<const u32x4*>(p + c * 1024 + lane * 16);
        t.dk = *reinterpret_cast<const f32x4*>(block + ((int64_t)(2 * D) << a.page_shift) + tile * 64 + (lane >> 4) * 16);
    }
    __device__ __forceinline__ void load_v(const AttnArgs& a, const uint8_t* block, int tile, Tile& t) const {
        const int lane = threadIdx.x & 63;
        const uint8_t* p = block + ((int64_t)D << a.page_shift) + tile * BLOCK16;
#pragma unroll
        for (int c = 0; c < ND; ++c) t.v[c] = *reinterpret_cast<const u32x4*>(p + c * 1024 + lane * 16);
        t.dv = *reinterpret_cast<const f32x4*>(block + ((int64_t)(2 * D + 4) << a.page_shift) + tile * 64 + (lane >> 4) * 16);
    }

    __device__ __forceinline__ f32x4 scores(const Tile& t) const {
        f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < ND; ++c) {
            const half8 a = widen8<CT>(t.k[c][0], t.k[c][1]), b = widen8<CT>(t.k[c][2], t.k[c][3]);
#pragma unroll
            for (int p = 0; p < PARTS; ++p) {
                s = mfma(a, q[p][2 * c], s);
                s = mfma(b, q[p][2 * c + 1], s);
            }
        }
        return s;
    }

    // The steps [s0, s1) of a list of pages; step s is tiles 2 s and 2 s + 1 from tile0 on, up to tile `end`.
    __device__ void run(const AttnArgs& a, const int32_t* pages, int n_list, int head, int tile0, int end, int s0, int s1) {
        if (s0 >= s1) return;
        const int lane = threadIdx.x & 63, g = lane >> 4;
        const int per = a.page_shift - 4, in_page = (1 << per) - 1;
        // the pages of 64 tiles at a time, a lane each
        int first = tile0 + 2 * s0;
        const auto list = [&](int from) {
            const int at = (from + lane) >> per;
            const int id = pages[at < n_list ? at : n_list - 1];
            return (unsigned)id < (unsigned)a.n_pages ? id : -1;
        };
        int now = list(first), next = list(first + 64);
        const auto page_of = [&](int tile) {  // -1: none
            const int i = tile - first;
            const int id = i < 64 ? __builtin_amdgcn_readlane(now, i) : __builtin_amdgcn_readlane(next, i - 64);
            return tile < end ? id : -1;
        };
        Tile A, B;
        int ta = first, pa = page_of(ta), pb = page_of(ta + 1);
        {
            const uint8_t *ba = block_of(a, pa, head), *bb = block_of(a, pb < 0 ? pa : pb, head);
            load_k(a, ba, ta & in_page, A);
            load_k(a, bb, (ta + 1) & in_page, B);
            load_v(a, ba, ta & in_page, A);
            load_v(a, bb, (ta + 1) & in_page, B);
        }
        for (int s = s0; s < s1; ++s) {
            const int tn = ta + 2;
            const bool more = s + 1 < s1;
            int na = pa, nb = pb;
            if (more) na = page_of(tn), nb = page_of(tn + 1);
            const uint8_t *ba = block_of(a, na, head), *bb = block_of(a, nb < 0 ? na : nb, head);
            f32x4 sa = scores(A), sb = scores(B);
            const f32x4 ka = A.dk * fac, kb = B.dk * fac;
            if (more) {
                load_k(a, ba, tn & in_page, A);
                load_k(a, bb, (tn + 1) & in_page, B);
            }
            if constexpr (MODE == PACK) {
#pragma unroll
                for (int i = 0; i < 4; ++i) sa[i] += other8(sa[i]), sb[i] += other8(sb[i]);
            }
            sa *= ka, sb *= kb;
            const int at = ta * 16;
            f32x4 da = A.dv, db = B.dv;
            const bool whole = pa >= 0 && pb >= 0 && at >= all_lo && at + STEP <= all_hi;
            if (!whole) {  // 0 times a scale that is NaN would be NaN
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int ja = at + 4 * g + i, jb = ja + 16;
                    if (pa < 0 || ja < lo || ja >= hi) sa[i] = -INFINITY, da[i] = 0.0f;
                    if (pb < 0 || jb < lo || jb >= hi) sb[i] = -INFINITY, db[i] = 0.0f;
                }
                // tokens that were never written may hold codes that are NaN
                clear(A, pa, at + 4 * g);
                clear(B, pb, at + 16 + 4 * g);
            }
            float top = fmaxf(fmaxf(fmaxf(sa[0], sa[1]), fmaxf(sa[2], sa[3])), fmaxf(fmaxf(sb[0], sb[1]), fmaxf(sb[2], sb[3])));
            top = max_groups(top);
            const float vt = fmaxf(fmaxf(fmaxf(da[0], da[1]), fmaxf(da[2], da[3])), fmaxf(fmaxf(db[0], db[1]), fmaxf(db[2], db[3])));
            if (__any(top > m + 6.0f || vt > unit * 256.0f)) rescale(top, vt);
            f32x4 wa, wb;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                wa[i] = __builtin_amdgcn_exp2f(sa[i] - base), wb[i] = __builtin_amdgcn_exp2f(sb[i] - base);
                l += wa[i] + wb[i];
            }
            wa *= da * inv_unit, wb *= db * inv_unit;
            half8 w[PARTS];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const _Float16 x = (_Float16)wa[i], y = (_Float16)wb[i];
                const _Float16 x2 = (_Float16)(wa[i] - (float)x), y2 = (_Float16)(wb[i] - (float)y);
                const bool second = MODE == PACK && (lane & 8);
                w[0][i] = second ? x2 : x, w[0][4 + i] = second ? y2 : y;
                if constexpr (MODE == SPLIT) w[PARTS - 1][i] = x2, w[PARTS - 1][4 + i] = y2;
            }
#pragma unroll
            for (int c = 0; c < ND; ++c)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const half8 v = widen8<CT>(A.v[c][j], B.v[c][j]);
#pragma unroll
                    for (int p = 0; p < PARTS; ++p) acc[4 * c + j] = mfma(v, w[p], acc[4 * c + j]);
                }
            if (more) {
                load_v(a, ba, tn & in_page, A);
                load_v(a, bb, (tn + 1) & in_page, B);
            }
            pa = na, pb = nb, ta = tn;
            if (ta - first >= 64) {
                first += 64;
                now = next;
                next = list(first + 64);
            }
        }
    }

    // Values of the four tokens from `at` on, where the list has no such tokens: 0.
    __device__ __forceinline__ void clear(Tile& t, int page, int at) const {
        uint32_t keep = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (page >= 0 && at + i < tokens) keep |= 255u << (8 * i);
#pragma unroll
        for (int c = 0; c < ND; ++c) t.v[c] &= keep;
    }

    // A larger maximum, or a larger scale of values.
    __device__ __forceinline__ void rescale(float top, float vt) {
        float f = 1.0f;
        if (top > m) {
            f = __builtin_amdgcn_exp2f(m - top);
            m = top;
            l *= f;
            base = top;
        }
        const float most = wave_max(vt);
        if (most > unit * 256.0f) {
            const int e = clampi((__float_as_int(most) >> 23) + 1, 30, 254);
            const float to = __int_as_float((e - 8) << 23);
            f *= unit * (1.0f / to);
            unit = to;
            inv_unit = 1.0f / to;
        }
#pragma unroll
        for (int i = 0; i < 4 * ND; ++i) acc[i] *= f;
    }

    // Sums over the lanes that share a column.
    __device__ __forceinline__ void finish(bool live) {
        l = sum_groups(l);
        if (!live) l = 0.0f;
        if constexpr (MODE == PACK) {
#pragma unroll
            for (int i = 0; i < 4 * ND; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][e] += other8(acc[i][e]);
        }
    }
    // Four of the lane's values: dimensions 64 c + 16 g + 4 i on.
    __device__ __forceinline__ f32x4 values(int c, int i, float f) const {
        return f32x4{acc[4 * c][i], acc[4 * c + 1][i], acc[4 * c + 2][i], acc[4 * c + 3][i]} * f;
    }
    __device__ __forceinline__ void to_piece(float* piece, int rows, int col) const {
        const int g = (threadIdx.x & 63) >> 4;
        if (col >= rows) return;
#pragma unroll
        for (int c = 0; c < ND; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<f32x4*>(piece + (int64_t)col * D + 64 * c + 16 * g + 4 * i) = values(c, i, unit);
        if (g == 0) {
            piece[(int64_t)rows * D + col] = m;
            piece[(int64_t)rows * D + rows + col] = l;
        }
    }
    __device__ __forceinline__ void to_out(const AttnArgs& a, const Column& c) const {
        const int g = (threadIdx.x & 63) >> 4;
        const int64_t row = (int64_t)c.seq * a.n_q + c.t;
        const bool some = l > 0.0f || l != l;
        const float f = some ? unit / l : 0.0f;
#pragma unroll
        for (int i = 0; i < ND; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                store_out(a.out, row * a.out_stride + (int64_t)c.head * D + 64 * i + 16 * g + 4 * e, a.type, a.out_vec,
                          some ? values(i, e, f) : f32x4{0.0f, 0.0f, 0.0f, 0.0f});
        if (a.lse && g == 0)
            a.lse[row * a.kv_heads * a.group + c.head] = some ? (m + __builtin_amdgcn_logf(l)) * LN2 : -INFINITY;
    }
};

// A sequence's own tokens: their number, the first tile that a query sees and the steps from there.
struct Own {
    int len, tile0, steps;
};
__device__ __forceinline__ Own own_of(const AttnArgs& a, int seq) {
    Own o;
    const int64_t most = (int64_t)a.table_pages << a.page_shift;
    const int len = a.lens[seq];
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

// How the waves are dealt, from the lengths: the same in every workgroup.
struct Deal {
    int64_t own_steps;   // of all own items
    int own_waves;       // that take part
    int pre_lo, pre_len; // the prefix's first tile that a query may see, its tokens
    int pre_steps, cuts; // cuts: pieces of the prefix
};

constexpr int MIN_STEPS = 2;  // of a wavefront's own steps, where there are enough

__device__ __forceinline__ Deal deal(const AttnArgs& a, int64_t own_steps) {
    Deal d;
    d.own_steps = own_steps;
    d.pre_len = 0, d.pre_lo = 0, d.pre_steps = 0, d.cuts = 0;
    if (a.prefix) {
        const int64_t most = (int64_t)a.prefix_pages << a.page_shift;
        const int len = a.prefix_len[0];
        d.pre_len = len < 0 ? 0 : len > most ? (int)most : len;
        // the first query's place is not before the prefix's end
        d.pre_lo = a.window ? max(0, d.pre_len - a.window + 1) >> 4 : 0;
        d.pre_steps = ((d.pre_len + 15) / 16 - d.pre_lo + 1) / 2;
        if (d.pre_steps > 0) {
            const int lines = a.kv_heads * a.pre_tiles;
            d.cuts = clampi(a.pre_waves / lines, 1, (d.pre_steps + MIN_STEPS - 1) / MIN_STEPS);
        }
    }
    const int64_t want = (own_steps + MIN_STEPS - 1) / MIN_STEPS;
    d.own_waves = want < a.own_waves ? (int)want : a.own_waves;
    return d;
}

// Workgroup `b` of `n` so that neighbours are on one die's L2 (workgroups go to the 8 dies in turn).
__device__ __forceinline__ int near_block(int b, int n) {
    const int each = n >> 3;
    return b < each * 8 ? (b & 7) * each + (b >> 3) : b;
}

template <int CT, int ND, int MODE, bool PRE>
__global__ __launch_bounds__(THREADS, ND == 4 ? 2 : 3) void k_attn(AttnArgs a) {
    constexpr int COLS = MODE == PACK ? 8 : 16;
    __shared__ int cum[MAX_SEQS + 1];
    __shared__ int part[WAVES];
    const int t = threadIdx.x, lane = t & 63, col = lane & 15;
    // the steps before each sequence
    int before = 0;
    for (int i0 = 0; i0 < a.n_seqs; i0 += THREADS) {
        const int i = i0 + t;
        int total;
        const int x = block_scan(i < a.n_seqs ? own_of(a, i).steps : 0, part, &total);
        if (i < a.n_seqs) cum[i] = before + x;
        before += total;
    }
    if (t == 0) cum[a.n_seqs] = before;
    __syncthreads();
    const int lines = a.kv_heads * a.row_tiles;  // items of a sequence
    const Deal d = deal(a, (int64_t)before * lines);
    const int n_own = (a.own_waves + WAVES - 1) / WAVES;
    int b = blockIdx.x;
    if (PRE && b >= n_own) {
        if (b == n_own && t == 0) a.head[0] = d.cuts;
        b = near_block(b - n_own, gridDim.x - n_own);
        constexpr int PM = MODE == PACK ? SPLIT : MODE;
        for (int x = uni(b * WAVES + (t >> 6)); x < d.cuts * a.kv_heads * a.pre_tiles; x += (gridDim.x - n_own) * WAVES) {
            const int tile = x % a.pre_tiles, seg = x / a.pre_tiles;
            const int head = seg / d.cuts, cut = seg % d.cuts;
            Column c;
            const int r = tile * 16 + col;
            c.row = r < a.n_seqs * a.n_q * a.group;
            const int token = c.row ? r / a.group : 0;
            c.seq = token / a.n_q, c.t = token % a.n_q, c.head = head * a.group + (c.row ? r % a.group : 0);
            const Own o = own_of(a, c.seq);
            const int at = o.len - a.n_q + c.t;
            c.live = c.row && at >= 0;
            const int lo = c.live ? (a.window ? max(0, d.pre_len + at - a.window + 1) : 0) : d.pre_len;
            Attend<CT, ND, PM> w;
            w.load(a, c);
            w.see(lo, d.pre_len, c.live, d.pre_len);
            int s0 = (int)((int64_t)d.pre_steps * cut / d.cuts), s1 = (int)((int64_t)d.pre_steps * (cut + 1) / d.cuts);
            int least = lo;  // of all columns: the steps before it are nobody's
#pragma unroll
            for (int s = 1; s < 64; s <<= 1) least = min(least, __shfl_xor(least, s));
            s0 = max(s0, (uni(least) / 16 - d.pre_lo) / 2);
            w.run(a, a.prefix, a.prefix_pages, head, d.pre_lo, (d.pre_len + 15) / 16, s0, s1);
            w.finish(c.live);
            w.to_piece(a.pre + (int64_t)x * piece_floats(16, 64 * ND), 16, col);
        }
        return;
    }
    const int me = uni(b * WAVES + (t >> 6));
    if (me >= d.own_waves) return;
    const int64_t T = d.own_steps, W = d.own_waves;
    const int64_t begin = me * T / W, end = (me + 1) * T / W;
    int64_t pos = begin;
    while (pos < end) {
        // the sequence whose steps hold pos
        const int u = (int)(pos / lines);
        int i = 0, j = a.n_seqs;
        while (j - i > 1) {
            const int mid = (i + j) >> 1;
            if (cum[mid] <= u)
                i = mid;
            else
                j = mid;
        }
        const int seq = uni(i);
        const Own o = own_of(a, seq);
        const int64_t seq_at = (int64_t)cum[seq] * lines;
        const int in = (int)(pos - seq_at), item = uni(in / o.steps), s0 = uni(in % o.steps);
        const int s1 = (int)(end - pos < o.steps - s0 ? s0 + (end - pos) : o.steps);
        const int head = item % a.kv_heads, tile = item / a.kv_heads;
        const int64_t item_at = seq_at + (int64_t)item * o.steps;
        const int fw = (int)(((item_at + 1) * W - 1) / T), lw = (int)(((item_at + o.steps) * W - 1) / T);
        const int64_t id = (int64_t)seq * lines + item;
        const bool direct = fw == lw && d.cuts == 0;
        // a piece is its wave's first (slot 2 w) or its last (2 w + 1); of a whole item with a prefix, the item's
        const int64_t slot = fw == lw ? 2 * (int64_t)a.own_waves + id : pos == begin ? 2 * (int64_t)me : 2 * (int64_t)me + 1;
        if (s0 == 0 && lane == 0)
            a.items[id] = direct ? make_int2(0, 0) : make_int2((int)slot, (lw - fw + 1) << 16 | fw);
        Column c;
        const int mine = MODE == PACK ? col & 7 : col;
        const int r = tile * COLS + mine;
        c.row = r < a.n_q * a.group;
        c.seq = seq, c.t = c.row ? r / a.group : 0, c.head = head * a.group + (c.row ? r % a.group : 0);
        const int at = o.len - a.n_q + c.t;
        c.live = c.row && at >= 0;
        Attend<CT, ND, MODE> w;
        w.load(a, c);
        w.see(a.window ? max(0, at - a.window + 1) : 0, at + 1, c.live, o.len);
        if (o.len > 0)
            w.run(a, a.tables + seq * a.table_stride, a.table_pages, head, o.tile0, (o.len + 15) / 16, s0, s1);
        w.finish(c.live);
        if (!(MODE == PACK && col >= 8) && c.row) {
            if (direct)
                w.to_out(a, c);
            else
                w.to_piece(a.own + slot * piece_floats(a.rows, 64 * ND), a.rows, mine);
        }
        pos += s1 - s0;
    }
}

// A workgroup joins the pieces of one row of an own item; a wavefront takes every eighth piece.
constexpr int MERGE_WAVES = 8;

template <int ND>
__global__ __launch_bounds__(MERGE_WAVES * 64) void k_attn_merge(AttnArgs a, int cols) {
    constexpr int D = 64 * ND;
    __shared__ float part[MERGE_WAVES][D], ms[MERGE_WAVES], ls[MERGE_WAVES];
    const int lines = a.kv_heads * a.row_tiles;
    const int64_t id = blockIdx.x;
    const int2 it = a.items[id];
    const int cuts = a.prefix ? a.head[0] : 0;
    const int own = it.y >> 16, fw = it.y & 0xFFFF;
    if (own == 0) return;  // written where it was made
    const int seq = (int)(id / lines), item = (int)(id % lines);
    const int head = item % a.kv_heads, tile = item / a.kv_heads;
    const int r = tile * cols + blockIdx.y;
    if (r >= a.n_q * a.group) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int all = (seq * a.n_q + r / a.group) * a.group + r % a.group;  // the row among the batch's
    const int64_t own_floats = piece_floats(a.rows, D), pre_floats = piece_floats(16, D);
    const auto piece = [&](int i, int* row, int* rows) {
        if (i < own) {
            *row = (int)blockIdx.y, *rows = a.rows;
            return a.own + (i == 0 ? (int64_t)it.x : 2 * (int64_t)(fw + i)) * own_floats;
        }
        *row = all & 15, *rows = 16;
        return a.pre + ((int64_t)(head * cuts + i - own) * a.pre_tiles + (all >> 4)) * pre_floats;
    };
    float m = -INFINITY, l = 0.0f;
    float x[ND] = {};
    for (int i = wave; i < own + cuts; i += MERGE_WAVES) {
        int row, rows;
        const float* p = piece(i, &row, &rows);
        const float pm = p[(int64_t)rows * D + row], pl = p[(int64_t)rows * D + rows + row];
        float v[ND];
#pragma unroll
        for (int c = 0; c < ND; ++c) v[c] = p[(int64_t)row * D + 64 * c + lane];
        if (pl == 0.0f) continue;  // nothing seen
        const float to = fmaxf(m, pm);
        const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - to), h = __builtin_amdgcn_exp2f(pm - to);
        l = l * f + pl * h;
#pragma unroll
        for (int c = 0; c < ND; ++c) x[c] = x[c] * f + v[c] * h;
        m = to;
    }
#pragma unroll
    for (int c = 0; c < ND; ++c) part[wave][64 * c + lane] = x[c];
    if (lane == 0) ms[wave] = m, ls[wave] = l;
    __syncthreads();
    if (threadIdx.x >= D) return;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < MERGE_WAVES; ++w) M = fmaxf(M, ms[w]);
    float L = 0.0f, X = 0.0f;
#pragma unroll
    for (int w = 0; w < MERGE_WAVES; ++w) {
        if (ls[w] == 0.0f) continue;
        const float f = __builtin_amdgcn_exp2f(ms[w] - M);
        L += ls[w] * f;
        X += part[w][threadIdx.x] * f;
    }
    const bool some = L > 0.0f || L != L;
    const int64_t token = (int64_t)seq * a.n_q + r / a.group;
    const int qh = head * a.group + r % a.group;
    const float v = some ? X / L : 0.0f;
    const int64_t at = token * a.out_stride + (int64_t)qh * D + threadIdx.x;
    if (a.type == FT_TYPE_F32) {
        static_cast<float*>(a.out)[at] = v;
    } else if (a.type == FT_TYPE_F16) {
        static_cast<uint16_t*>(a.out)[at] = f2h(v);
    } else {
        const uint32_t w = __float_as_uint(v);
        static_cast<uint16_t*>(a.out)[at] =
            (w & 0x7FFFFFFFu) > 0x7F800000u ? (uint16_t)(w >> 16 | 0x40) : (uint16_t)((w + 0x7FFF + (w >> 16 & 1)) >> 16);
    }
    if (a.lse && threadIdx.x == 0)
        a.lse[token * a.kv_heads * a.group + qh] = some ? (M + __builtin_amdgcn_logf(L)) * LN2 : -INFINITY;
}

// What a call's sizes make of it.
struct Sizes {
    int cols, rows, row_tiles, pre_tiles;
    int64_t items, lines_pre;
    size_t at_items, at_own, at_pre, bytes;
};
// Workgroups: two on each CU for the own tokens, two for the prefix.
constexpr int OWN_WAVES = 512 * WAVES, PRE_WAVES = 512 * WAVES;

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
    z.bytes = z.at_pre + up((size_t)(z.lines_pre > PRE_WAVES ? z.lines_pre : PRE_WAVES) * piece_floats(16, (int)D) * 4);
    return true;
}

template <int CT, int ND, int MODE>
void launch_attn(const AttnArgs& a, const Sizes& z, hipStream_t s) {
    const unsigned own = (unsigned)((a.own_waves + WAVES - 1) / WAVES);
    if (a.prefix) {
        const int64_t most = z.lines_pre > PRE_WAVES ? z.lines_pre : PRE_WAVES;
        const unsigned pre = (unsigned)((most < PRE_WAVES ? most : PRE_WAVES) / WAVES);
        hipLaunchKernelGGL((k_attn<CT, ND, MODE, true>), dim3(own + pre), dim3(THREADS), 0, s, a);
    } else {
        hipLaunchKernelGGL((k_attn<CT, ND, MODE, false>), dim3(own), dim3(THREADS), 0, s, a);
    }
    hipLaunchKernelGGL(k_attn_merge<ND>, dim3((unsigned)z.items, (unsigned)z.rows), dim3(MERGE_WAVES * 64), 0, s, a, z.cols);
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
    const int64_t cap_steps = z.items * (table_pages * page_tokens / STEP + 2);
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
    a.q_vec = aligned(q, 16) && q_stride * size % 16 == 0;
    a.out_vec = aligned(out, 4 * size) && out_stride % 4 == 0;
    a.head = reinterpret_cast<int32_t*>(ws), a.items = reinterpret_cast<int2*>(ws + z.at_items);
    a.own = reinterpret_cast<float*>(ws + z.at_own), a.pre = reinterpret_cast<float*>(ws + z.at_pre);
    const int64_t want = (cap_steps + MIN_STEPS - 1) / MIN_STEPS;
    a.own_waves = (int)(want < OWN_WAVES ? want : OWN_WAVES), a.pre_waves = PRE_WAVES;
    DeviceGuard on(ctx->device);
    if (!on.ok) return fail(FT_HIP_E_DEVICE, "attention: device %d cannot be made current", ctx->device);
    if (cache_type == FT_KV_I8)
        launch_dim<FT_KV_I8>(a, z, head_dim, static_cast<hipStream_t>(stream));
    else
        launch_dim<FT_KV_E4M3>(a, z, head_dim, static_cast<hipStream_t>(stream));
    return launch_status("attention");
}
