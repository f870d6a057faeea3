// ft_hip_kv.hip -- keys and values quantised into the pages of a cache
// (ft_hip_kv_write) and read back (ft_hip_kv_read); the layout is ft_kv.hpp's.
//
// Per token and head, a = max |x| of its D values:
//   i8    q = round half away(127 x / a), d = f32(a / 127), the byte is q + 128
//   e4m3  d = 2^e, the smallest with a / d <= 448 (e >= -126), the byte is the
//         code nearest to x / d, halves to even
// i8's quotient is rounded as the real number, as add_rmsnorm's quants are: with
// x = U 2^i and a = A 2^j of 24-bit whole U and A it differs from a half by
// nothing or by more than 2^-32 of itself; it is taken in f64 with 127 / a a
// little enlarged (1 + 2^-44), so that a half comes out above the half and any
// other stays on its side. e4m3's scale is a power of two because then x / d is
// exact and the conversion is the only rounding; a code's relative error is the
// same at any scale, and the range below the largest shrinks by one bit at most.
// The byte of i8 is q + 128 because the products take it apart as the low byte
// of an f16 of 1024 + q + 128.
//
// A wavefront takes four tokens of a head's keys, or of its values: 16 lanes a
// token, eight values a lane (four of f32, and where heads have 64). Values of
// four tokens that stand side by side in one group of the cache change places over
// lanes and are stored as words; others byte by byte. Of many rows (MANY) a
// wavefront takes four parts, all of them on their way at once.
//
// What bounds it: bytes, at 5.1 TB/s of a large copy. 32768 tokens of 8 heads of 256
// from e4m3 to bf16, 405 MB, 85 us, 4.8 TB/s (a head a wavefront and four values a
// lane 107 us). 16387 tokens of 8 heads of 128 written from bf16, 102 MB, 24 us. A few
// hundred rows are 3 us of a launch and two dependent reads.

#include "ft_device.hpp"
#include "ft_kv.hpp"
#include "ft_overlap.hpp"
#include "ft_runtime.hpp"
#include "ft_wave.hpp"

#include <cfloat>
#include <cmath>

using namespace ft;

namespace {

// Tokens times heads from which a wavefront takes four parts. 16387 tokens of 8 heads: written (128 values, from bf16) 23.1 us,
// by one part 28.5; read (256, to bf16) 49.0 and 54.0. 4096 tokens: 8.8 and 8.3, 14.4 and 11.9; 512: 3.8 and 2.8, 6.7 and 4.0.
constexpr int64_t MANY = 65536;

struct KvArgs {
    const void *k, *v;  // rows to write, or to read into
    int64_t k_stride, v_stride;
    const int32_t* slots;
    uint8_t* cache;
    int n, heads, page_shift;
    unsigned n_slots;
};

// W values as they lie, and what they are.
template <int TYPE, int W>
struct Some {
    static constexpr int WORDS = TYPE == FT_TYPE_F32 ? W : W / 2;
    uint32_t w[WORDS];
    __device__ __forceinline__ void load(const void* base, int64_t at, bool vec) {
        if (vec) {
            typedef uint32_t vector __attribute__((ext_vector_type(WORDS)));
            const vector a = *reinterpret_cast<const vector*>(static_cast<const char*>(base) + at * (TYPE == FT_TYPE_F32 ? 4 : 2));
#pragma unroll
            for (int i = 0; i < WORDS; ++i) w[i] = a[i];
        } else if constexpr (TYPE == FT_TYPE_F32) {
#pragma unroll
            for (int i = 0; i < WORDS; ++i) w[i] = static_cast<const uint32_t*>(base)[at + i];
        } else {
            const uint16_t* p = static_cast<const uint16_t*>(base) + at;
#pragma unroll
            for (int i = 0; i < WORDS; ++i) w[i] = p[2 * i] | (uint32_t)p[2 * i + 1] << 16;
        }
    }
    __device__ __forceinline__ float value(int i) const {
        if constexpr (TYPE == FT_TYPE_F32) return __uint_as_float(w[i]);
        const uint16_t b = (uint16_t)(w[i >> 1] >> (i & 1) * 16);
        return TYPE == FT_TYPE_F16 ? h2f(b) : __uint_as_float((uint32_t)b << 16);
    }
};

__device__ __forceinline__ uint16_t narrow(float v, int type) {
    if (type == FT_TYPE_F16) return f2h(v);
    const uint32_t b = __float_as_uint(v);
    if ((b & 0x7FFFFFFFu) > 0x7F800000u) return (uint16_t)(b >> 16 | 0x40);  // NaN
    return (uint16_t)((b + 0x7FFF + (b >> 16 & 1)) >> 16);
}

template <int TYPE, int W>
__device__ __forceinline__ void store_some(void* base, int64_t at, bool vec, const float* v) {
    constexpr int WORDS = Some<TYPE, W>::WORDS;
    uint32_t w[WORDS];
#pragma unroll
    for (int i = 0; i < WORDS; ++i) {
        if constexpr (TYPE == FT_TYPE_F32)
            w[i] = __float_as_uint(v[i]);
        else
            w[i] = narrow(v[2 * i], TYPE) | (uint32_t)narrow(v[2 * i + 1], TYPE) << 16;
    }
    char* const p = static_cast<char*>(base) + at * (TYPE == FT_TYPE_F32 ? 4 : 2);
    if (vec) {
        typedef uint32_t vector __attribute__((ext_vector_type(WORDS)));
        vector a;
#pragma unroll
        for (int i = 0; i < WORDS; ++i) a[i] = w[i];
        *reinterpret_cast<vector*>(p) = a;
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i) {
            if constexpr (TYPE == FT_TYPE_F32)
                reinterpret_cast<uint32_t*>(p)[i] = w[i];
            else
                reinterpret_cast<uint16_t*>(p)[i] = (uint16_t)(w[i >> 1] >> (i & 1) * 16);
        }
    }
}

// Lane (token g, r) holds four values' bytes of token g; afterwards lane (g, r)
// holds the four tokens' bytes of value g, and the other way round.
__device__ __forceinline__ uint32_t swap_tokens(uint32_t w, int g) {
    const uint32_t o = __shfl_xor((int)w, 32);
    w = g & 2 ? __builtin_amdgcn_perm(w, o, 0x07060302) : __builtin_amdgcn_perm(o, w, 0x05040100);
    const uint32_t p = __shfl_xor((int)w, 16);
    return g & 1 ? __builtin_amdgcn_perm(w, p, 0x07030501) : __builtin_amdgcn_perm(p, w, 0x06020400);
}

// Where a wavefront's four tokens lie.
struct Place {
    int idx;        // the token's index in the call
    int slot;       // its place in the cache, or -1
    bool together;  // the four stand in one group of the cache, in order
    int64_t page;   // where its page begins
    int o;          // its place in the page
};

// The groups of four are laid so that those of the first token's run meet the cache's.
__device__ __forceinline__ Place place_of(const KvArgs& a, int group, int dim, int g) {
    const int first = a.slots[0];
    Place p;
    p.idx = 4 * group - (first > 0 ? first & 3 : 0) + g;
    const int slot = p.idx >= 0 && p.idx < a.n ? a.slots[p.idx] : -1;
    p.slot = (unsigned)slot < a.n_slots ? slot : -1;
    const int at0 = __builtin_amdgcn_readfirstlane(p.slot);  // of token 0
    p.together = at0 >= 0 && (at0 & 3) == 0 && __all(p.slot == at0 + g);
    p.page = (int64_t)(p.slot >> a.page_shift) * a.heads * kv_block_bytes((int64_t)1 << a.page_shift, dim);
    p.o = p.slot & ((1 << a.page_shift) - 1);
    return p;
}

// Where in a block's keys dimension `dim` of the token at `o` lies, and in its values.
template <int ND>
__device__ __forceinline__ int key_at(int o, int dim) {
    return (o >> 4) * (1024 * ND) + (dim >> 4) * 256 + (o & 15) * 16 + (dim & 15);
}
template <int ND>
__device__ __forceinline__ int value_at(int o, int dim) {
    return (o >> 4) * (1024 * ND) + (dim >> 6) * 1024 + (o >> 2 & 3) * 256 + (dim & 63) * 4 + (o & 3);
}

// A lane's W values' bytes, words of four. Values of four tokens side by side change places over the lanes: lane g then
// holds the four tokens' bytes of W / 4 of the values, those from its g's on.
template <int W>
__device__ __forceinline__ void spread(uint32_t (&w)[W / 4], int g) {
    if constexpr (W == 8) {  // even and odd values apart
        const uint32_t even = __builtin_amdgcn_perm(w[1], w[0], 0x06040200), odd = __builtin_amdgcn_perm(w[1], w[0], 0x07050301);
        w[0] = swap_tokens(even, g), w[1] = swap_tokens(odd, g);
    } else {
        w[0] = swap_tokens(w[0], g);
    }
}
template <int W>
__device__ __forceinline__ void gather(uint32_t (&w)[W / 4], int g) {
    if constexpr (W == 8) {
        const uint32_t even = swap_tokens(w[0], g), odd = swap_tokens(w[1], g);
        w[0] = __builtin_amdgcn_perm(odd, even, 0x05010400), w[1] = __builtin_amdgcn_perm(odd, even, 0x07030602);
    } else {
        w[0] = swap_tokens(w[0], g);
    }
}
template <int W>
__device__ __forceinline__ void put(uint8_t* p, const uint32_t (&w)[W / 4]) {
    if constexpr (W == 8)
        *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else
        *reinterpret_cast<uint32_t*>(p) = w[0];
}
template <int W>
__device__ __forceinline__ void take(const uint8_t* p, uint32_t (&w)[W / 4]) {
    if constexpr (W == 8) {
        const uint2 a = *reinterpret_cast<const uint2*>(p);
        w[0] = a.x, w[1] = a.y;
    } else {
        w[0] = *reinterpret_cast<const uint32_t*>(p);
    }
}

// A wavefront per group of four tokens and R of the 2 * heads parts, a head's keys or values each, which are all on
// their way before the first is worked on; 16 lanes a token, W values a lane in each round. Four groups make a workgroup;
// the workgroups of one group's parts follow each other, so that those running at once touch whole rows and all of the
// memory's channels (32768 tokens of 8 heads of 256 read 107 us with the tokens first, 85 so).
template <int CT, int TYPE, int ND, int R, int W>
__global__ __launch_bounds__(256) void k_kv_write(KvArgs a, bool vec) {
    constexpr int D = 64 * ND, NR = D / (16 * W);
    const int lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
    const int parts = (2 * a.heads + R - 1) / R, group = blockIdx.x / parts, part0 = (blockIdx.x - group * parts) * R;
    const Place p = place_of(a, group * 4 + (threadIdx.x >> 6), D, g);
    const bool live = p.slot >= 0;
    Some<TYPE, W> raw[R][NR];
#pragma unroll
    for (int u = 0; u < R; ++u) {
        const int part = part0 + u;
        if (R > 1 && part >= 2 * a.heads) break;
        const int64_t from = (int64_t)p.idx * (part & 1 ? a.v_stride : a.k_stride) + (part >> 1) * D + W * r;
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            raw[u][i] = Some<TYPE, W>{};
            if (live) raw[u][i].load(part & 1 ? a.v : a.k, from + 16 * W * i, vec);
        }
    }
#pragma unroll
    for (int u = 0; u < R; ++u) {
        const int part = part0 + u, head = part >> 1;
        const bool value = part & 1;
        if (R > 1 && part >= 2 * a.heads) break;
        float x[NR][W], top = 0.0f;
#pragma unroll
        for (int i = 0; i < NR; ++i)
#pragma unroll
            for (int e = 0; e < W; ++e) {
                x[i][e] = raw[u][i].value(e);
                // NaN counts as inf: the maximum then says that the row is no numbers
                top = fmaxf(top, fabsf(x[i][e]) <= FLT_MAX ? fabsf(x[i][e]) : INFINITY);
            }
        top = row_max16(top);
        const bool bad = top == INFINITY;
        float d = 0.0f;
        uint32_t word[NR][W / 4];
        if constexpr (CT == FT_KV_I8) {
            const double of = top > 0.0f && !bad ? 127.0 / (double)top * (1.0 + 0x1p-44) : 0.0;
            d = (float)((double)top / 127.0);
#pragma unroll
            for (int i = 0; i < NR; ++i)
#pragma unroll
                for (int e = 0; e < W; e += 4) {
                    // the sum's last bit is 1: its low half is the nearest whole number
                    const auto q = [&](float v) { return (uint32_t)(int)__double_as_longlong(fma((double)(bad ? 0.0f : v), of, 0x1.8p52 + 128.0)); };
                    word[i][e / 4] = (q(x[i][e]) & 255) | (q(x[i][e + 1]) & 255) << 8 | (q(x[i][e + 2]) & 255) << 16 | q(x[i][e + 3]) << 24;
                }
        } else {
            const int bits = __float_as_int(top);
            const int e2 = max((bits >> 23) - 127 - 8 + ((bits & 0x7FFFFF) > 0x600000 ? 1 : 0), -126);
            const float inv = __int_as_float((127 - e2) << 23);
            if (top > 0.0f) d = __int_as_float((127 + e2) << 23);
#pragma unroll
            for (int i = 0; i < NR; ++i)
#pragma unroll
                for (int e = 0; e < W; e += 4) {
                    const auto y = [&](float v) { return bad ? 0.0f : v * inv; };
                    const int w = __builtin_amdgcn_cvt_pk_fp8_f32(y(x[i][e]), y(x[i][e + 1]), 0, false);
                    word[i][e / 4] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y(x[i][e + 2]), y(x[i][e + 3]), w, true);
                }
        }
        if (bad) d = __int_as_float(0x7FC00000);
        uint8_t* const block = a.cache + p.page + head * kv_block_bytes((int64_t)1 << a.page_shift, D);
        uint8_t* const rows = block + (value ? (int64_t)D << a.page_shift : 0);
        if (live && r == 0)
            reinterpret_cast<float*>(block + ((int64_t)(2 * D) << a.page_shift))[(value ? 1 << a.page_shift : 0) + p.o] = d;
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            const int dim = 16 * W * i + W * r;
            if (!value) {
                if (live) put<W>(rows + key_at<ND>(p.o, dim), word[i]);
            } else if (p.together) {
                spread<W>(word[i], g);
                put<W>(rows + value_at<ND>(p.o & ~3, dim + W / 4 * g), word[i]);
            } else if (live) {
#pragma unroll
                for (int e = 0; e < W; ++e) rows[value_at<ND>(p.o, dim + e)] = (uint8_t)(word[i][e >> 2] >> (8 * (e & 3)));
            }
        }
    }
}

template <int CT, int TYPE, int ND, int R, int W>
__global__ __launch_bounds__(256) void k_kv_read(KvArgs a, bool vec) {
    constexpr int D = 64 * ND, NR = D / (16 * W);
    const int lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
    const int parts = (2 * a.heads + R - 1) / R, group = blockIdx.x / parts, part0 = (blockIdx.x - group * parts) * R;
    const Place p = place_of(a, group * 4 + (threadIdx.x >> 6), D, g);
    const bool live = p.slot >= 0;
    uint32_t word[R][NR][W / 4];
    float d[R];
#pragma unroll
    for (int u = 0; u < R; ++u) {
        const int part = part0 + u;
        const bool value = part & 1;
        if (R > 1 && part >= 2 * a.heads) break;
        const uint8_t* const block = a.cache + p.page + (part >> 1) * kv_block_bytes((int64_t)1 << a.page_shift, D);
        const uint8_t* const rows = block + (value ? (int64_t)D << a.page_shift : 0);
        d[u] = 0.0f;
        if (live) d[u] = reinterpret_cast<const float*>(block + ((int64_t)(2 * D) << a.page_shift))[(value ? 1 << a.page_shift : 0) + p.o];
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            const int dim = 16 * W * i + W * r;
#pragma unroll
            for (int e = 0; e < W / 4; ++e) word[u][i][e] = 0;
            if (!live) continue;
            if (!value) {
                take<W>(rows + key_at<ND>(p.o, dim), word[u][i]);
            } else if (p.together) {
                take<W>(rows + value_at<ND>(p.o & ~3, dim + W / 4 * g), word[u][i]);
            } else {
#pragma unroll
                for (int e = 0; e < W; ++e) word[u][i][e >> 2] |= (uint32_t)rows[value_at<ND>(p.o, dim + e)] << (8 * (e & 3));
            }
        }
    }
#pragma unroll
    for (int u = 0; u < R; ++u) {
        const int part = part0 + u;
        const bool value = part & 1;
        if (R > 1 && part >= 2 * a.heads) break;
        const int64_t to = (int64_t)p.idx * (value ? a.v_stride : a.k_stride) + (part >> 1) * D + W * r;
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            if (value && p.together) gather<W>(word[u][i], g);
            float v[W];
#pragma unroll
            for (int e = 0; e < W; ++e) {
                const uint32_t w = word[u][i][e >> 2];
                float q;
                if constexpr (CT == FT_KV_I8)
                    q = (float)(int)(w >> (8 * (e & 3)) & 255) - 128.0f;
                else
                    q = (e & 3) == 0   ? __builtin_amdgcn_cvt_f32_fp8((int)w, 0)
                        : (e & 3) == 1 ? __builtin_amdgcn_cvt_f32_fp8((int)w, 1)
                        : (e & 3) == 2 ? __builtin_amdgcn_cvt_f32_fp8((int)w, 2)
                                       : __builtin_amdgcn_cvt_f32_fp8((int)w, 3);
                v[e] = q * d[u];
                if constexpr (TYPE == FT_TYPE_F16) asm("" : "+v"(v[e]));  // as rounded to f32, not once to f16 in an instruction
            }
            if (live) store_some<TYPE, W>(const_cast<void*>(value ? a.v : a.k), to + 16 * W * i, vec, v);
        }
    }
}

template <bool WRITE, int CT, int TYPE, int ND, int R>
void launch_parts(const KvArgs& a, bool vec, hipStream_t s) {
    // a group more than the tokens need: the first may begin up to three tokens before the first token
    const dim3 grid((unsigned)(((int64_t)a.n + 3 + 15) / 16 * ((2 * a.heads + R - 1) / R)));
    // 16 bytes of a row a lane, as far as the heads have them
    constexpr int W = TYPE == FT_TYPE_F32 || ND == 1 ? 4 : 8;
    if (WRITE)
        hipLaunchKernelGGL((k_kv_write<CT, TYPE, ND, R, W>), grid, dim3(256), 0, s, a, vec);
    else
        hipLaunchKernelGGL((k_kv_read<CT, TYPE, ND, R, W>), grid, dim3(256), 0, s, a, vec);
}

template <bool WRITE, int CT, int TYPE>
void launch_nd(const KvArgs& a, int nd, bool vec, hipStream_t s) {
    const auto go = [&](auto ND) {
        constexpr int N = decltype(ND)::value;
        // many tokens: several parts a wavefront
        if ((int64_t)a.n * a.heads >= MANY)
            launch_parts<WRITE, CT, TYPE, N, 4>(a, vec, s);
        else
            launch_parts<WRITE, CT, TYPE, N, 1>(a, vec, s);
    };
    if (nd == 1)
        go(std::integral_constant<int, 1>{});
    else if (nd == 2)
        go(std::integral_constant<int, 2>{});
    else
        go(std::integral_constant<int, 4>{});
}

template <bool WRITE>
void launch_kv(const KvArgs& a, int cache_type, int type, int nd, bool vec, hipStream_t s) {
    if (cache_type == FT_KV_I8) {
        if (type == FT_TYPE_F32)
            launch_nd<WRITE, FT_KV_I8, FT_TYPE_F32>(a, nd, vec, s);
        else if (type == FT_TYPE_F16)
            launch_nd<WRITE, FT_KV_I8, FT_TYPE_F16>(a, nd, vec, s);
        else
            launch_nd<WRITE, FT_KV_I8, FT_TYPE_BF16>(a, nd, vec, s);
    } else {
        if (type == FT_TYPE_F32)
            launch_nd<WRITE, FT_KV_E4M3, FT_TYPE_F32>(a, nd, vec, s);
        else if (type == FT_TYPE_F16)
            launch_nd<WRITE, FT_KV_E4M3, FT_TYPE_F16>(a, nd, vec, s);
        else
            launch_nd<WRITE, FT_KV_E4M3, FT_TYPE_BF16>(a, nd, vec, s);
    }
}

// What both entry points check and do; rows: the tensors beside the cache.
template <bool WRITE>
int kv_call(const char* what, ft_hip_ctx* ctx, void* stream, const void* k, int64_t k_stride, const void* v,
            int64_t v_stride, int row_type, const int32_t* slots, const void* cache, int cache_type, int64_t n_pages,
            int64_t page_tokens, int64_t n_heads, int64_t head_dim, int64_t n) {
    clear_error();
    if (!kv_dims_fit(page_tokens, n_heads, head_dim))
        return fail(FT_HIP_E_SHAPE, "%s: page_tokens=%lld (16 to 256, a power of two), n_heads=%lld (1 to 256) or head_dim=%lld (64, 128, 256)",
                    what, (long long)page_tokens, (long long)n_heads, (long long)head_dim);
    if (!kv_pages_fit(n_pages, page_tokens))
        return fail(FT_HIP_E_SHAPE, "%s: n_pages=%lld not in [1, 2^31 tokens]", what, (long long)n_pages);
    if (n < 0 || n > 1 << 20) return fail(FT_HIP_E_SHAPE, "%s: n=%lld not in [0, 2^20]", what, (long long)n);
    if (row_type != FT_TYPE_F32 && row_type != FT_TYPE_F16 && row_type != FT_TYPE_BF16)
        return fail(FT_HIP_E_INVALID, "%s: row_type=%d is no FT_TYPE", what, row_type);
    if (cache_type != FT_KV_I8 && cache_type != FT_KV_E4M3)
        return fail(FT_HIP_E_INVALID, "%s: cache_type=%d is no FT_KV", what, cache_type);
    const int64_t width = n_heads * head_dim, most = (int64_t)1 << 36;
    if (k_stride < width || k_stride > most || v_stride < width || v_stride > most)
        return fail(FT_HIP_E_SHAPE, "%s: k_stride or v_stride out of range", what);
    const int64_t size = row_type == FT_TYPE_F32 ? 4 : 2;
    if (!aligned(k, size) || !aligned(v, size) || !aligned(slots, 4) || !aligned(cache, 16))
        return fail(FT_HIP_E_SHAPE, "%s: a pointer is not aligned to its type (cache: 16 bytes)", what);
    if (!ctx) return fail(FT_HIP_E_INVALID, "%s: null argument", what);
    if (n == 0) return FT_HIP_OK;  // an empty tensor has no address
    if (!k || !v || !slots || !cache) return fail(FT_HIP_E_INVALID, "%s: null argument", what);
    const Span sk{k, n, k_stride * size, width * size}, sv{v, n, v_stride * size, width * size}, ss{slots, 1, 0, n * 4},
        sc{cache, 1, 0, n_pages * n_heads * kv_block_bytes(page_tokens, head_dim)};
    if (overlap(sc, sk) || overlap(sc, sv) || overlap(sc, ss))
        return fail(FT_HIP_E_SHAPE, "%s: the cache overlaps another argument", what);
    if (!WRITE && (overlap(sk, sv) || overlap(sk, ss) || overlap(sv, ss)))
        return fail(FT_HIP_E_SHAPE, "%s: k or v overlaps another argument", what);
    int shift = 4;
    while (1 << shift < page_tokens) ++shift;
    const KvArgs a{k, v, k_stride, v_stride, slots, static_cast<uint8_t*>(const_cast<void*>(cache)), (int)n,
                   (int)n_heads, shift, (unsigned)(n_pages * page_tokens)};
    // 16 bytes of a row at a time where every row starts on them
    const bool vec = aligned(k, 16) && aligned(v, 16) && k_stride * size % 16 == 0 && v_stride * size % 16 == 0;
    DeviceGuard on(ctx->device);
    if (!on.ok) return fail(FT_HIP_E_DEVICE, "%s: device %d cannot be made current", what, ctx->device);
    launch_kv<WRITE>(a, cache_type, row_type, (int)head_dim / 64, vec, static_cast<hipStream_t>(stream));
    return launch_status(what);
}

}  // namespace

extern "C" int64_t ft_hip_kv_page_bytes(int64_t page_tokens, int64_t n_heads, int64_t head_dim) {
    return kv_dims_fit(page_tokens, n_heads, head_dim) ? n_heads * kv_block_bytes(page_tokens, head_dim) : -1;
}

extern "C" int ft_hip_kv_write(ft_hip_ctx* ctx, void* stream, const void* k, int64_t k_stride, const void* v,
                               int64_t v_stride, int row_type, const int32_t* slots, void* cache, int cache_type,
                               int64_t n_pages, int64_t page_tokens, int64_t n_heads, int64_t head_dim, int64_t n) {
    return kv_call<true>("kv_write", ctx, stream, k, k_stride, v, v_stride, row_type, slots, cache, cache_type, n_pages,
                         page_tokens, n_heads, head_dim, n);
}

extern "C" int ft_hip_kv_read(ft_hip_ctx* ctx, void* stream, const void* cache, int cache_type, int64_t n_pages,
                              int64_t page_tokens, int64_t n_heads, int64_t head_dim, const int32_t* slots, void* k,
                              int64_t k_stride, void* v, int64_t v_stride, int row_type, int64_t n) {
    return kv_call<false>("kv_read", ctx, stream, k, k_stride, v, v_stride, row_type, slots, cache, cache_type, n_pages,
                          page_tokens, n_heads, head_dim, n);
}
