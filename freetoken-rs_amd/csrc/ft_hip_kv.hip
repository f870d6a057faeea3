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
// token, four values a lane in each of D / 64 rounds. Values of four tokens that
// stand side by side in one group of the cache change places over lanes and are
// stored as words; others are stored byte by byte.

#include "ft_device.hpp"
#include "ft_kv.hpp"
#include "ft_overlap.hpp"
#include "ft_runtime.hpp"
#include "ft_wave.hpp"

#include <cfloat>
#include <cmath>

using namespace ft;

namespace {

struct KvArgs {
    const void *k, *v;  // rows to write, or to read into
    int64_t k_stride, v_stride;
    const int32_t* slots;
    uint8_t* cache;
    int n, heads, page_shift;
    unsigned n_slots;
};

__device__ __forceinline__ float4 load4(const void* base, int64_t at, int type, bool vec) {
    if (type == FT_TYPE_F32) {
        const float* p = static_cast<const float*>(base) + at;
        if (vec) return *reinterpret_cast<const float4*>(p);
        return make_float4(p[0], p[1], p[2], p[3]);
    }
    const uint16_t* p = static_cast<const uint16_t*>(base) + at;
    uint16_t b[4];
    if (vec) {
        const uint2 a = *reinterpret_cast<const uint2*>(p);
        b[0] = (uint16_t)a.x, b[1] = (uint16_t)(a.x >> 16), b[2] = (uint16_t)a.y, b[3] = (uint16_t)(a.y >> 16);
    } else {
        b[0] = p[0], b[1] = p[1], b[2] = p[2], b[3] = p[3];
    }
    const auto wide = [&](uint16_t v) { return type == FT_TYPE_F16 ? h2f(v) : __uint_as_float((uint32_t)v << 16); };
    return make_float4(wide(b[0]), wide(b[1]), wide(b[2]), wide(b[3]));
}

__device__ __forceinline__ uint16_t narrow(float v, int type) {
    if (type == FT_TYPE_F16) return f2h(v);
    const uint32_t b = __float_as_uint(v);
    if ((b & 0x7FFFFFFFu) > 0x7F800000u) return (uint16_t)(b >> 16 | 0x40);  // NaN
    return (uint16_t)((b + 0x7FFF + (b >> 16 & 1)) >> 16);
}

__device__ __forceinline__ void store4(void* base, int64_t at, int type, bool vec, const float* v) {
    if (type == FT_TYPE_F32) {
        float* p = static_cast<float*>(base) + at;
        if (vec) {
            *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
            return;
        }
        for (int i = 0; i < 4; ++i) p[i] = v[i];
        return;
    }
    uint16_t* p = static_cast<uint16_t*>(base) + at;
    uint16_t b[4];
    for (int i = 0; i < 4; ++i) b[i] = narrow(v[i], type);
    if (vec) {
        *reinterpret_cast<uint2*>(p) = make_uint2(b[0] | (uint32_t)b[1] << 16, b[2] | (uint32_t)b[3] << 16);
        return;
    }
    for (int i = 0; i < 4; ++i) p[i] = b[i];
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
    uint8_t* block; // its head's block
    int o;          // its place in the page
};

// The groups of four are laid so that those of the first token's run meet the cache's.
__device__ __forceinline__ Place place_of(const KvArgs& a, int group, int head, int dim, int g) {
    const int first = a.slots[0];
    Place p;
    p.idx = 4 * group - (first > 0 ? first & 3 : 0) + g;
    const int slot = p.idx >= 0 && p.idx < a.n ? a.slots[p.idx] : -1;
    p.slot = (unsigned)slot < a.n_slots ? slot : -1;
    const int at0 = __builtin_amdgcn_readfirstlane(p.slot);  // of token 0
    p.together = at0 >= 0 && (at0 & 3) == 0 && __all(p.slot == at0 + g);
    const int page = p.slot >> a.page_shift;
    p.o = p.slot & ((1 << a.page_shift) - 1);
    p.block = a.cache + ((int64_t)page * a.heads + head) * kv_block_bytes((int64_t)1 << a.page_shift, dim);
    return p;
}

// A value's word or byte (token t of its group) in a block's keys or values.
template <int ND>
__device__ __forceinline__ int key_at(int o, int i, int r) {
    return (o >> 4) * (1024 * ND) + (4 * i + (r >> 2)) * 256 + (o & 15) * 16 + (r & 3) * 4;
}
template <int ND>
__device__ __forceinline__ int value_at(int o, int i, int dim) {
    return (o >> 4) * (1024 * ND) + i * 1024 + (o >> 2 & 3) * 256 + dim * 4 + (o & 3);
}

// grid: (groups of 16 tokens, 2 * heads); a wavefront per group of four
template <int CT, int TYPE, int ND>
__global__ __launch_bounds__(256) void k_kv_write(KvArgs a, bool vec) {
    constexpr int D = 64 * ND;
    const int lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
    const int head = blockIdx.y >> 1;
    const bool value = blockIdx.y & 1;
    const Place p = place_of(a, blockIdx.x * 4 + (threadIdx.x >> 6), head, D, g);
    const bool live = p.slot >= 0;
    float4 x[ND];
    float top = 0.0f;
    const int64_t from = (int64_t)p.idx * (value ? a.v_stride : a.k_stride) + head * D + 4 * r;
#pragma unroll
    for (int i = 0; i < ND; ++i) {
        x[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (live) x[i] = load4(value ? a.v : a.k, from + 64 * i, TYPE, vec);
        // NaN counts as inf: the maximum then says that the row is no numbers
        const auto size = [](float v) { return fabsf(v) <= FLT_MAX ? fabsf(v) : INFINITY; };
        top = fmaxf(fmaxf(fmaxf(top, size(x[i].x)), fmaxf(size(x[i].y), size(x[i].z))), size(x[i].w));
    }
    top = row_max16(top);
    const bool bad = top == INFINITY;
    float d = 0.0f;
    uint32_t word[ND];
    if constexpr (CT == FT_KV_I8) {
        const double of = top > 0.0f && !bad ? 127.0 / (double)top * (1.0 + 0x1p-44) : 0.0;
        d = (float)((double)top / 127.0);
#pragma unroll
        for (int i = 0; i < ND; ++i) {
            // the sum's last bit is 1: its low half is the nearest whole number
            const auto q = [&](float v) { return (uint32_t)(int)__double_as_longlong(fma((double)(bad ? 0.0f : v), of, 0x1.8p52 + 128.0)); };
            word[i] = (q(x[i].x) & 255) | (q(x[i].y) & 255) << 8 | (q(x[i].z) & 255) << 16 | q(x[i].w) << 24;
        }
    } else {
        const int bits = __float_as_int(top);
        const int e = max((bits >> 23) - 127 - 8 + ((bits & 0x7FFFFF) > 0x600000 ? 1 : 0), -126);
        const float inv = __int_as_float((127 - e) << 23);
        if (top > 0.0f) d = __int_as_float((127 + e) << 23);
#pragma unroll
        for (int i = 0; i < ND; ++i) {
            const auto y = [&](float v) { return bad ? 0.0f : v * inv; };
            int w = __builtin_amdgcn_cvt_pk_fp8_f32(y(x[i].x), y(x[i].y), 0, false);
            word[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y(x[i].z), y(x[i].w), w, true);
        }
    }
    if (bad) d = __int_as_float(0x7FC00000);
    uint8_t* const rows = p.block + (value ? (int64_t)D << a.page_shift : 0);
    if (live && r == 0) reinterpret_cast<float*>(p.block + ((int64_t)(2 * D) << a.page_shift))[(value ? 1 << a.page_shift : 0) + p.o] = d;
    if (!value) {
        if (!live) return;
#pragma unroll
        for (int i = 0; i < ND; ++i) *reinterpret_cast<uint32_t*>(rows + key_at<ND>(p.o, i, r)) = word[i];
    } else if (p.together) {
#pragma unroll
        for (int i = 0; i < ND; ++i)
            *reinterpret_cast<uint32_t*>(rows + value_at<ND>(p.o & ~3, i, 4 * r + g)) = swap_tokens(word[i], g);
    } else if (live) {
#pragma unroll
        for (int i = 0; i < ND; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) rows[value_at<ND>(p.o, i, 4 * r + e)] = (uint8_t)(word[i] >> (8 * e));
    }
}

template <int CT, int TYPE, int ND>
__global__ __launch_bounds__(256) void k_kv_read(KvArgs a, bool vec) {
    constexpr int D = 64 * ND;
    const int lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
    const int head = blockIdx.y >> 1;
    const bool value = blockIdx.y & 1;
    const Place p = place_of(a, blockIdx.x * 4 + (threadIdx.x >> 6), head, D, g);
    const bool live = p.slot >= 0;
    const uint8_t* const rows = p.block + (value ? (int64_t)D << a.page_shift : 0);
    uint32_t word[ND];
    float d = 0.0f;
    if (live) d = reinterpret_cast<const float*>(p.block + ((int64_t)(2 * D) << a.page_shift))[(value ? 1 << a.page_shift : 0) + p.o];
    if (!value) {
        if (!live) return;
#pragma unroll
        for (int i = 0; i < ND; ++i) word[i] = *reinterpret_cast<const uint32_t*>(rows + key_at<ND>(p.o, i, r));
    } else if (p.together) {
#pragma unroll
        for (int i = 0; i < ND; ++i) word[i] = *reinterpret_cast<const uint32_t*>(rows + value_at<ND>(p.o & ~3, i, 4 * r + g));
#pragma unroll
        for (int i = 0; i < ND; ++i) word[i] = swap_tokens(word[i], g);
    } else {
        if (!live) return;
#pragma unroll
        for (int i = 0; i < ND; ++i) {
            word[i] = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) word[i] |= (uint32_t)rows[value_at<ND>(p.o, i, 4 * r + e)] << (8 * e);
        }
    }
    const int64_t to = (int64_t)p.idx * (value ? a.v_stride : a.k_stride) + head * D + 4 * r;
#pragma unroll
    for (int i = 0; i < ND; ++i) {
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float q;
            if constexpr (CT == FT_KV_I8)
                q = (float)(int)(word[i] >> (8 * e) & 255) - 128.0f;
            else
                q = e == 0   ? __builtin_amdgcn_cvt_f32_fp8((int)word[i], 0)
                    : e == 1 ? __builtin_amdgcn_cvt_f32_fp8((int)word[i], 1)
                    : e == 2 ? __builtin_amdgcn_cvt_f32_fp8((int)word[i], 2)
                             : __builtin_amdgcn_cvt_f32_fp8((int)word[i], 3);
            v[e] = q * d;
        }
        store4(const_cast<void*>(value ? a.v : a.k), to + 64 * i, TYPE, vec, v);
    }
}

template <bool WRITE, int CT, int TYPE>
void launch_nd(const KvArgs& a, int nd, bool vec, dim3 grid, hipStream_t s) {
    const auto go = [&](auto ND) {
        constexpr int N = decltype(ND)::value;
        if (WRITE)
            hipLaunchKernelGGL((k_kv_write<CT, TYPE, N>), grid, dim3(256), 0, s, a, vec);
        else
            hipLaunchKernelGGL((k_kv_read<CT, TYPE, N>), grid, dim3(256), 0, s, a, vec);
    };
    if (nd == 1)
        go(std::integral_constant<int, 1>{});
    else if (nd == 2)
        go(std::integral_constant<int, 2>{});
    else
        go(std::integral_constant<int, 4>{});
}

template <bool WRITE>
void launch_kv(const KvArgs& a, int cache_type, int type, int head_dim, bool vec, hipStream_t s) {
    // a group more than the tokens need: the first may begin up to three tokens before the first token
    const dim3 grid((unsigned)(((int64_t)a.n + 3 + 15) / 16), (unsigned)(2 * a.heads));
    const int nd = head_dim / 64;
    if (cache_type == FT_KV_I8) {
        if (type == FT_TYPE_F32)
            launch_nd<WRITE, FT_KV_I8, FT_TYPE_F32>(a, nd, vec, grid, s);
        else if (type == FT_TYPE_F16)
            launch_nd<WRITE, FT_KV_I8, FT_TYPE_F16>(a, nd, vec, grid, s);
        else
            launch_nd<WRITE, FT_KV_I8, FT_TYPE_BF16>(a, nd, vec, grid, s);
    } else {
        if (type == FT_TYPE_F32)
            launch_nd<WRITE, FT_KV_E4M3, FT_TYPE_F32>(a, nd, vec, grid, s);
        else if (type == FT_TYPE_F16)
            launch_nd<WRITE, FT_KV_E4M3, FT_TYPE_F16>(a, nd, vec, grid, s);
        else
            launch_nd<WRITE, FT_KV_E4M3, FT_TYPE_BF16>(a, nd, vec, grid, s);
    }
}

// What both entry points check and do; rows: the tensors beside the cache.
template <bool WRITE>
int kv_call(const char* what, ft_hip_ctx* ctx, void* stream, const void* k, int64_t k_stride, const void* v,
            int64_t v_stride, int type, const int32_t* slots, const void* cache, int cache_type, int64_t n_pages,
            int64_t page_tokens, int64_t n_heads, int64_t head_dim, int64_t n) {
    clear_error();
    if (!kv_dims_fit(page_tokens, n_heads, head_dim))
        return fail(FT_HIP_E_SHAPE, "%s: page_tokens=%lld (16 to 256, a power of two), n_heads=%lld (1 to 256) or head_dim=%lld (64, 128, 256)",
                    what, (long long)page_tokens, (long long)n_heads, (long long)head_dim);
    if (!kv_pages_fit(n_pages, page_tokens))
        return fail(FT_HIP_E_SHAPE, "%s: n_pages=%lld not in [1, 2^31 tokens]", what, (long long)n_pages);
    if (n < 0 || n > 1 << 24) return fail(FT_HIP_E_SHAPE, "%s: n=%lld not in [0, 2^24]", what, (long long)n);
    if (type != FT_TYPE_F32 && type != FT_TYPE_F16 && type != FT_TYPE_BF16)
        return fail(FT_HIP_E_INVALID, "%s: type=%d is no FT_TYPE", what, type);
    if (cache_type != FT_KV_I8 && cache_type != FT_KV_E4M3)
        return fail(FT_HIP_E_INVALID, "%s: cache_type=%d is no FT_KV", what, cache_type);
    const int64_t width = n_heads * head_dim, most = (int64_t)1 << 36;
    if (k_stride < width || k_stride > most || v_stride < width || v_stride > most)
        return fail(FT_HIP_E_SHAPE, "%s: k_stride or v_stride out of range", what);
    const int64_t size = type == FT_TYPE_F32 ? 4 : 2;
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
    // four values at a time where every row starts on them
    const bool vec = aligned(k, 4 * size) && aligned(v, 4 * size) && k_stride % 4 == 0 && v_stride % 4 == 0;
    DeviceGuard on(ctx->device);
    if (!on.ok) return fail(FT_HIP_E_DEVICE, "%s: device %d cannot be made current", what, ctx->device);
    launch_kv<WRITE>(a, cache_type, type, (int)head_dim, vec, static_cast<hipStream_t>(stream));
    return launch_status(what);
}

}  // namespace

extern "C" int64_t ft_hip_kv_page_bytes(int64_t page_tokens, int64_t n_heads, int64_t head_dim) {
    return kv_dims_fit(page_tokens, n_heads, head_dim) ? n_heads * kv_block_bytes(page_tokens, head_dim) : -1;
}

extern "C" int ft_hip_kv_write(ft_hip_ctx* ctx, void* stream, const void* k, int64_t k_stride, const void* v,
                               int64_t v_stride, int type, const int32_t* slots, void* cache, int cache_type,
                               int64_t n_pages, int64_t page_tokens, int64_t n_heads, int64_t head_dim, int64_t n) {
    return kv_call<true>("kv_write", ctx, stream, k, k_stride, v, v_stride, type, slots, cache, cache_type, n_pages,
                         page_tokens, n_heads, head_dim, n);
}

extern "C" int ft_hip_kv_read(ft_hip_ctx* ctx, void* stream, const void* cache, int cache_type, int64_t n_pages,
                              int64_t page_tokens, int64_t n_heads, int64_t head_dim, const int32_t* slots, void* k,
                              int64_t k_stride, void* v, int64_t v_stride, int type, int64_t n) {
    return kv_call<false>("kv_read", ctx, stream, k, k_stride, v, v_stride, type, slots, cache, cache_type, n_pages,
                          page_tokens, n_heads, head_dim, n);
}
