// ft_hip_norm.hip -- the residual addition and RMS norm in front of a section,
// with the q8 blocks that its q4 GEMVs take, in one pass over the rows
// (ft_hip_add_rmsnorm).
//
//   h   = residual + x,  or with the branch's own norm  residual + x / rms(x) * x_w
//   inv = 1 / sqrt(mean(h * h) + eps),  y = h * inv * w
//   q8  : u = f32(h * w); per 32 values a = max |u|, q = round half away(127 u / a), d = a * inv / 127
//
// The quants are those of u, before the row's scale: 127 u / a is the same
// quotient for y, and taken from u it depends on 32 values instead of on the
// last bit of a sum over the row. The quotient is rounded as the real number:
// with u = U 2^i and a = A 2^j of 24-bit whole U and A, i <= j, it differs from
// a half by |254 U - odd A 2^(j-i)| / (2 A 2^(j-i)): not at all, or by at least
// 1 / (2 A 2^(j-i)), which is the quotient over 254 U and so over 2^-32 of it.
// It is taken as u times 127 / a * (1 + 2^-44), in f64 off by less than 2^-45
// of itself besides: a half comes out above the half, any other stays on its
// side, and the nearest whole number is the one sought.
//
// Bound by memory: x, the residual, h, y and the blocks each move once; the
// row stays in registers between its sum and its outputs. Sums and scales are
// f64 (its rate is f32's here), h and y are rounded to f32 once.
//
// Measured, kernel alone, hidden 2816, f32 in, h and q8 out: 1 row 2.4 us, 64
// rows 3.4, 777 rows 7.2, 16384 rows 104 (5.9 TB/s; a copy of 256 MiB runs at
// 5.0). Up to some hundred rows the time is a launch and one round trip.

#include "ft_device.hpp"
#include "ft_overlap.hpp"
#include "ft_runtime.hpp"
#include "ft_wave.hpp"

#include <cfloat>
#include <cmath>

using namespace ft;

namespace {

struct NormArgs {
    const void* x;
    int64_t x_stride;
    const float* x_w;
    const float* residual;
    int64_t r_stride;
    float* h;
    int64_t h_stride;
    const float* w;
    float* y;
    int64_t y_stride;
    uint8_t* q8;
    int hidden;
    double eps, per_value;  // per_value: 1 / hidden
};

// V consecutive values (V = 4: one aligned vector access, V = 1: any address)
template <int V>
struct Vals {
    float v[V];
};

template <int V>
__device__ __forceinline__ Vals<V> load_f32(const float* p) {
    Vals<V> r;
    if constexpr (V == 4) {
        const float4 a = *reinterpret_cast<const float4*>(p);
        r.v[0] = a.x, r.v[1] = a.y, r.v[2] = a.z, r.v[3] = a.w;
    } else {
        r.v[0] = *p;
    }
    return r;
}

template <int V, int TYPE>
__device__ __forceinline__ Vals<V> load_typed(const void* base, int64_t at) {
    if constexpr (TYPE == FT_TYPE_F32) {
        return load_f32<V>(static_cast<const float*>(base) + at);
    } else {
        uint16_t b[V];
        const uint16_t* p = static_cast<const uint16_t*>(base) + at;
        if constexpr (V == 4) {
            const uint2 a = *reinterpret_cast<const uint2*>(p);
            b[0] = (uint16_t)a.x, b[1] = (uint16_t)(a.x >> 16), b[2] = (uint16_t)a.y, b[3] = (uint16_t)(a.y >> 16);
        } else {
            b[0] = *p;
        }
        Vals<V> r;
#pragma unroll
        for (int i = 0; i < V; ++i) r.v[i] = TYPE == FT_TYPE_F16 ? h2f(b[i]) : __uint_as_float((uint32_t)b[i] << 16);
        return r;
    }
}

template <int V>
__device__ __forceinline__ void store_f32(float* p, const Vals<V>& r) {
    if constexpr (V == 4)
        *reinterpret_cast<float4*>(p) = make_float4(r.v[0], r.v[1], r.v[2], r.v[3]);
    else
        *p = r.v[0];
}

// Sum over the workgroup, the same bits in every thread and on every run: the
// waves' sums in order.
__device__ __forceinline__ double row_sum(double v, double* red) {
    v = wave_sum(v);
    const int waves = blockDim.x >> 6, lane = threadIdx.x & 63;
    if (waves == 1) return v;
    if (lane == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return wave_sum(lane < waves ? red[lane] : 0.0);
}

// 1 / x and 1 / sqrt(x) to an ulp or two of f64: the instruction's 24 bits and
// two Newton steps (IEEE division and square root take about 60 instructions
// between them). x positive, and for rsqrt 0 gives inf or NaN, inf gives 0.
__device__ __forceinline__ double recip(double x) {
    double y = __builtin_amdgcn_rcp(x);
    y = fma(fma(-x, y, 1.0), y, y);
    return fma(fma(-x, y, 1.0), y, y);
}
__device__ __forceinline__ double rsqrt_of(double x) {
    if (x > 0x1p1000) return 0.0;  // of f32 values: inf
    double y = __builtin_amdgcn_rsq(x);
    y = fma(fma(-x * y, y, 1.0), 0.5 * y, y);
    return fma(fma(-x * y, y, 1.0), 0.5 * y, y);
}

// One q8 block per group of 32 / V lanes.
template <int V>
__device__ __forceinline__ void quantize_u(const Vals<V>& u, double inv, uint8_t* blk, int part) {
    float a = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) a = fmaxf(a, fabsf(u.v[i]));  // NaN is skipped
    if constexpr (V == 4) {  // 8 lanes: quad, then the half-row's other quad
        a = fmaxf(a, quad_xor1(a));
        a = fmaxf(a, quad_xor2(a));
        a = fmaxf(a, dpp_f<0x141>(a));
    } else {
        a = half_max32(a);
    }
    const double r = a > 0.0f && a < INFINITY ? recip((double)a) * (127.0 * (1.0 + 0x1p-44)) : 0.0;
    const float most = fminf(a, FLT_MAX);
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const float v = fabsf(u.v[i]) <= most ? u.v[i] : 0.0f;  // NaN and inf: quant 0
        // the sum's last bit is 1: its low half is the nearest whole number
        const int q = (int)__double_as_longlong(fma((double)v, r, 0x1.8p52));
        word |= (uint32_t)(uint8_t)q << (8 * i);
    }
    int qsum = V == 4 ? __builtin_amdgcn_sdot4((int)word, 0x01010101, 0, false) : (int)(int8_t)word;
    if constexpr (V == 4) {
        qsum += quad_xor1i(qsum);
        qsum += quad_xor2i(qsum);
        qsum += dpp_i<0x141>(qsum);
        reinterpret_cast<uint32_t*>(blk)[2 + part] = word;
    } else {
        qsum = half_sum32(qsum);
        blk[8 + part] = (uint8_t)word;
    }
    if (part == 0) {
        reinterpret_cast<float*>(blk)[0] = a > 0.0f ? (float)((double)a * inv * (1.0 / 127.0)) : 0.0f;
        reinterpret_cast<int*>(blk)[1] = qsum;
    }
}

// A workgroup per row; thread t holds the values (i * threads + t) * V .. + V
// of it for i < NV. Lanes past the row's end hold zeros; hidden is a multiple
// of 32 where q8 is written, so that a block's lanes are all inside the row
// or all outside.
template <int TYPE, int V, int NV>
__global__ __launch_bounds__(1024) void k_add_rmsnorm(NormArgs a) {
    __shared__ double red[2][16];
    const int64_t row = blockIdx.x;
    const int t = threadIdx.x, step = blockDim.x * V;
    const auto zero = [](Vals<V>& r) {
#pragma unroll
        for (int e = 0; e < V; ++e) r.v[e] = 0.0f;
    };
    // all that the row's sums do not decide is loaded at once
    Vals<V> h[NV], r[NV], xw[NV], w[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = i * step + t * V;
        if (c >= a.hidden) {
            zero(h[i]);
            continue;
        }
        h[i] = load_typed<V, TYPE>(a.x, row * a.x_stride + c);
        if (a.residual) r[i] = load_f32<V>(a.residual + row * a.r_stride + c);
        if (a.x_w) xw[i] = load_f32<V>(a.x_w + c);
        if (a.w) w[i] = load_f32<V>(a.w + c);
    }
    if (a.x_w) {
        double ss = 0.0;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) ss = fma((double)h[i].v[e], (double)h[i].v[e], ss);
        const double inv = rsqrt_of(fma(row_sum(ss, red[0]), a.per_value, a.eps));
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (i * step + t * V >= a.hidden) continue;
#pragma unroll
            for (int e = 0; e < V; ++e)
                h[i].v[e] = (float)fma((double)h[i].v[e] * inv, (double)xw[i].v[e],
                                       a.residual ? (double)r[i].v[e] : 0.0);
        }
    } else if (a.residual) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (i * step + t * V >= a.hidden) continue;
#pragma unroll
            for (int e = 0; e < V; ++e) h[i].v[e] = r[i].v[e] + h[i].v[e];
        }
    }
    double ss = 0.0;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) ss = fma((double)h[i].v[e], (double)h[i].v[e], ss);
    const double inv = rsqrt_of(fma(row_sum(ss, red[1]), a.per_value, a.eps));
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = i * step + t * V;
        if (c >= a.hidden) continue;
        if (a.h) store_f32<V>(a.h + row * a.h_stride + c, h[i]);
        if (!a.w) {
#pragma unroll
            for (int e = 0; e < V; ++e) w[i].v[e] = 1.0f;
        }
        if (a.y) {
            Vals<V> y;
#pragma unroll
            for (int e = 0; e < V; ++e) y.v[e] = (float)((double)h[i].v[e] * inv * (double)w[i].v[e]);
            store_f32<V>(a.y + row * a.y_stride + c, y);
        }
        if (a.q8) {
            Vals<V> u;
#pragma unroll
            for (int e = 0; e < V; ++e) u.v[e] = h[i].v[e] * w[i].v[e];
            quantize_u<V>(u, inv, a.q8 + (row * (a.hidden >> 5) + (c >> 5)) * Q8_BLK, (c & 31) / V);
        }
    }
}

template <int TYPE>
void launch_norm(const NormArgs& a, int64_t n, int64_t few, bool vec, void* stream) {
    const dim3 grid((unsigned)n);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (!vec) {
        const int threads = a.hidden >= 1024 ? 1024 : (a.hidden + 63) / 64 * 64;
        hipLaunchKernelGGL((k_add_rmsnorm<TYPE, 1, 16>), grid, dim3(threads), 0, s, a);
        return;
    }
    // few rows: as many threads on a row as it has vectors; many: four vectors a thread, so that what a wave does once
    // a row (two sums, two square roots) is shared by more values. Hidden 2816: 64 rows 3.4 us against 4.0, 256 rows
    // 4.0 against 4.5; 777 rows 7.7 against 7.0, 16384 rows 115 against 104.
    const int vecs = a.hidden / 4, wide = (vecs + 63) / 64 * 64;
    if (n <= few && vecs <= 1024)
        hipLaunchKernelGGL((k_add_rmsnorm<TYPE, 4, 1>), grid, dim3(wide), 0, s, a);
    else
        hipLaunchKernelGGL((k_add_rmsnorm<TYPE, 4, 4>), grid, dim3((vecs + 255) / 256 * 64), 0, s, a);
}

}  // namespace

extern "C" int ft_hip_add_rmsnorm(ft_hip_ctx* ctx, void* stream, const void* x, int x_type, int64_t x_stride,
                                  const float* x_w, const float* residual, int64_t residual_stride, float* h,
                                  int64_t h_stride, const float* w, float eps, float* y, int64_t y_stride, void* q8,
                                  int64_t hidden, int64_t n) {
    clear_error();
    if (hidden <= 0 || hidden > 16384)
        return fail(FT_HIP_E_SHAPE, "add_rmsnorm: hidden=%lld not in [1, 16384]", (long long)hidden);
    if (q8 && hidden % 32)
        return fail(FT_HIP_E_SHAPE, "add_rmsnorm: hidden=%lld must be a multiple of 32 for q8", (long long)hidden);
    if (n < 0 || n > 4194303)  // a workgroup of up to 1024 threads per row, fewer than 2^32 in all
        return fail(FT_HIP_E_SHAPE, "add_rmsnorm: n=%lld not in [0, 4194303]", (long long)n);
    if (x_type != FT_TYPE_F32 && x_type != FT_TYPE_F16 && x_type != FT_TYPE_BF16)
        return fail(FT_HIP_E_INVALID, "add_rmsnorm: x_type=%d is no FT_TYPE", x_type);
    if (!(eps >= 0.0f) || std::isinf(eps)) return fail(FT_HIP_E_SHAPE, "add_rmsnorm: eps is not a number >= 0");
    const int64_t most = INT64_MAX / 4 / (n > 0 ? n : 1);
    if (x_stride < hidden || x_stride > most) return fail(FT_HIP_E_SHAPE, "add_rmsnorm: x_stride out of range");
    if (residual && (residual_stride < hidden || residual_stride > most))
        return fail(FT_HIP_E_SHAPE, "add_rmsnorm: residual_stride out of range");
    if (h && (h_stride < hidden || h_stride > most)) return fail(FT_HIP_E_SHAPE, "add_rmsnorm: h_stride out of range");
    if (y && (y_stride < hidden || y_stride > most)) return fail(FT_HIP_E_SHAPE, "add_rmsnorm: y_stride out of range");
    const unsigned size = x_type == FT_TYPE_F32 ? 4 : 2;
    if (!aligned(x, size) || !aligned(x_w, 4) || !aligned(residual, 4) || !aligned(h, 4) || !aligned(w, 4) ||
        !aligned(y, 4) || !aligned(q8, 4))
        return fail(FT_HIP_E_SHAPE, "add_rmsnorm: a pointer is not aligned to its type (q8: 4 bytes)");
    if (!ctx) return fail(FT_HIP_E_INVALID, "add_rmsnorm: null argument");
    if (n == 0) return FT_HIP_OK;  // an empty tensor has no address
    if (!x) return fail(FT_HIP_E_INVALID, "add_rmsnorm: null argument");
    if (!h && !y && !q8) return fail(FT_HIP_E_INVALID, "add_rmsnorm: no output (h, y and q8 are null)");
    // A thread writes the places that it has read, and no others: h or y may lie on an input's rows, on all of them with
    // the same stride; any other overlap would mix rows, or blocks with what they are made of.
    const auto f32 = [&](const float* p, int64_t stride) { return Span{p, n, stride * 4, hidden * 4}; };
    const Span sx{x, n, x_stride * size, hidden * size}, sr = f32(residual, residual_stride), sh = f32(h, h_stride),
        sy = f32(y, y_stride), sq{q8, 1, 0, n * (hidden / 32) * Q8_BLK}, sw{w, 1, 0, hidden * 4}, sxw{x_w, 1, 0, hidden * 4};
    const auto mixes = [&](const Span& out, const Span& in) {
        return overlap(out, in) && !(out.at == in.at && out.bytes == in.bytes && (n == 1 || out.stride == in.stride));
    };
    for (const Span& out : {sh, sy})
        if (mixes(out, sx) || mixes(out, sr) || overlap(out, sw) || overlap(out, sxw) || overlap(out, sq))
            return fail(FT_HIP_E_SHAPE, "add_rmsnorm: h or y overlaps an input other than row on row, a weight or q8");
    if (overlap(sh, sy)) return fail(FT_HIP_E_SHAPE, "add_rmsnorm: h and y overlap");
    if (overlap(sq, sx) || overlap(sq, sr) || overlap(sq, sw) || overlap(sq, sxw))
        return fail(FT_HIP_E_SHAPE, "add_rmsnorm: q8 overlaps an input");
    const NormArgs a{x, x_stride, x_w, residual, residual_stride, h, h_stride, w, y, y_stride,
                     static_cast<uint8_t*>(q8), (int)hidden, (double)eps, 1.0 / (double)hidden};
    // vectors of 4 where every row starts on one; else value by value
    const bool vec = hidden % 4 == 0 && aligned(x, 4 * size) && x_stride % 4 == 0 && aligned(x_w, 16) &&
                     aligned(w, 16) && aligned(residual, 16) && (!residual || residual_stride % 4 == 0) && aligned(h, 16) &&
                     (!h || h_stride % 4 == 0) && aligned(y, 16) && (!y || y_stride % 4 == 0);
    DeviceGuard on(ctx->device);
    if (!on.ok) return fail(FT_HIP_E_DEVICE, "add_rmsnorm: device %d cannot be made current", ctx->device);
    if (x_type == FT_TYPE_F32)
        launch_norm<FT_TYPE_F32>(a, n, ctx->num_cus, vec, stream);
    else if (x_type == FT_TYPE_F16)
        launch_norm<FT_TYPE_F16>(a, n, ctx->num_cus, vec, stream);
    else
        launch_norm<FT_TYPE_BF16>(a, n, ctx->num_cus, vec, stream);
    return launch_status("add_rmsnorm");
}
