// ft_hip_route.hip -- experts chosen from router logits by softmax or sigmoid
// scores, with a selection bias, groups of experts, renormalised and scaled
// weights (ft_hip_route_experts).
//
// Per token: s = softmax(l) or sigmoid(l) over its experts, c = s + bias. With
// groups, a group's score is its best c or the sum of its best two, and only
// the best top_groups groups stay open. The top_k experts by c are chosen,
// equal ones by the lower index, and weighted by s.
//
// Which of two experts comes first is decided on f64 scores (f64 runs at
// f32's rate here): an f32 exp's last bit would swap near-equal experts in
// some of a prompt's thousands of tokens.
//
// A token's experts lie over the 64 lanes of a wave, expert lane + 64 j in
// slot j; every selection is a maximum over the wave.

#include "ft_device.hpp"
#include "ft_runtime.hpp"

#include <cmath>

using namespace ft;

namespace {

constexpr int MAX_GROUPS = 64;

struct RouteArgs {
    const float* logits;
    int64_t stride;
    const float* bias;
    const float* escale;
    int32_t* ids;
    float* wts;
    int sigmoid, n_groups, group_size, top_groups, group_rank, renorm;
    double scale;
    int E, k;
    int64_t n;
};

__device__ __forceinline__ double shfl_xor_f64(double v, int m) {
    const long long b = __double_as_longlong(v);
    const int lo = __shfl_xor((int)b, m), hi = __shfl_xor((int)(b >> 32), m);
    return __longlong_as_double(((long long)hi << 32) | (uint32_t)lo);
}
__device__ __forceinline__ double shfl_f64(double v, int l) {
    const long long b = __double_as_longlong(v);
    const int lo = __shfl((int)b, l), hi = __shfl((int)(b >> 32), l);
    return __longlong_as_double(((long long)hi << 32) | (uint32_t)lo);
}

// LDS written by a wave is read by its other lanes after this.
__device__ __forceinline__ void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
    __builtin_amdgcn_wave_barrier();
}

template <int VPL>
__global__ __launch_bounds__(256) void k_route_experts(RouteArgs a) {
    extern __shared__ double lds[];  // with groups: per wave its token's c
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t token = (int64_t)blockIdx.x * 4 + wave;
    if (token >= a.n) return;  // whole waves; no workgroup barrier below
    const float* row = a.logits + token * a.stride;
    const double none = -(double)INFINITY;

    float l[VPL];
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
        const int e = lane + 64 * j;
        l[j] = e < a.E ? row[e] : -INFINITY;
        m = fmaxf(m, l[j]);  // NaN is skipped
    }
    double s[VPL], c[VPL];
    if (a.sigmoid) {
#pragma unroll
        for (int j = 0; j < VPL; ++j) s[j] = 1.0 / (1.0 + exp(-(double)l[j]));
    } else {
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) m = fmaxf(m, __shfl_xor(m, o));
        double sum = 0.0;
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
            s[j] = l[j] == m ? 1.0 : exp((double)l[j] - (double)m);  // several +inf share
            sum += l[j] > -INFINITY ? s[j] : 0.0;
        }
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) sum += shfl_xor_f64(sum, o);
#pragma unroll
        for (int j = 0; j < VPL; ++j) s[j] = s[j] / sum;
    }
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
        const int e = lane + 64 * j;
        c[j] = s[j] + (a.bias && e < a.E ? (double)a.bias[e] : 0.0);
        if (!(l[j] > -INFINITY) || !(c[j] == c[j])) c[j] = none;  // -inf, NaN: never chosen
    }

    if (a.n_groups > 1) {
        double* w = lds + wave * a.E;
#pragma unroll
        for (int j = 0; j < VPL; ++j)
            if (lane + 64 * j < a.E) w[lane + 64 * j] = c[j];
        wave_lds_fence();
        // the group's two best, by lane g < n_groups
        double b1 = none, b2 = none;
        if (lane < a.n_groups)
            for (int i = 0; i < a.group_size; ++i) {
                const double v = w[lane * a.group_size + i];
                b2 = fmax(b2, fmin(b1, v));
                b1 = fmax(b1, v);
            }
        const double gs = a.group_rank == 2 && b2 > none ? b1 + b2 : b1;
        // open: fewer than top_groups groups are ahead of it
        int ahead = 0;
        for (int g = 0; g < a.n_groups; ++g) {
            const double o = shfl_f64(gs, g);
            ahead += o > gs || (o == gs && g < lane);
        }
        const uint64_t open = __ballot(lane < a.n_groups && ahead < a.top_groups);
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
            const int e = lane + 64 * j;
            if (e < a.E && !((open >> (e / a.group_size)) & 1)) c[j] = none;
        }
    }

    int id = 0;
    double wt = 0.0;  // lane r holds the r-th chosen
    for (int r = 0; r < a.k; ++r) {
        double bc = none;
        int bi = 0x7FFFFFFF;
#pragma unroll
        for (int j = 0; j < VPL; ++j)
            if (c[j] > bc) {
                bc = c[j];
                bi = lane + 64 * j;
            }
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const double oc = shfl_xor_f64(bc, o);
            const int oi = __shfl_xor(bi, o);
            if (oc > bc || (oc == bc && oi < bi)) {
                bc = oc;
                bi = oi;
            }
        }
        if (bi == 0x7FFFFFFF) break;  // none left (uniform)
        double sv = 0.0;
#pragma unroll
        for (int j = 0; j < VPL; ++j)
            if (bi == lane + 64 * j) {
                c[j] = none;
                sv = s[j];
            }
        sv = shfl_f64(sv, bi & 63);
        if (lane == r) {
            id = bi;
            wt = sv;
        }
    }
    if (a.renorm) {
        double sum = wt;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) sum += shfl_xor_f64(sum, o);
        wt = sum > 0.0 ? wt / sum : 0.0;
    }
    if (lane < a.k) {
        a.ids[token * a.k + lane] = id;
        a.wts[token * a.k + lane] = (float)(wt * a.scale * (a.escale ? (double)a.escale[id] : 1.0));
    }
}

}  // namespace

extern "C" int ft_hip_route_experts(ft_hip_ctx* ctx, void* stream, const float* logits, int64_t logits_stride,
                                    const float* bias, const float* expert_scale, int score, int64_t n_groups,
                                    int64_t top_groups, int group_rank, int renorm, float scale, int32_t* ids,
                                    float* wts, int64_t n_experts, int64_t top_k, int64_t n_seqs) {
    clear_error();
    const long long E = n_experts, G = n_groups;
    if (E <= 0 || E > 1024) return fail(FT_HIP_E_SHAPE, "route_experts: n_experts=%lld not in [1, 1024]", E);
    if (G <= 0 || G > MAX_GROUPS || E % G)
        return fail(FT_HIP_E_SHAPE, "route_experts: n_groups=%lld not in [1, %d] or no divisor of %lld experts", G, MAX_GROUPS, E);
    if (top_groups <= 0 || top_groups > G)
        return fail(FT_HIP_E_SHAPE, "route_experts: top_groups=%lld not in [1, %lld]", (long long)top_groups, G);
    if (top_k <= 0 || top_k > 32 || top_k > top_groups * (E / G))
        return fail(FT_HIP_E_SHAPE, "route_experts: top_k=%lld not in [1, 32] or more than the open groups hold", (long long)top_k);
    if (group_rank != 1 && group_rank != 2)
        return fail(FT_HIP_E_SHAPE, "route_experts: group_rank=%d is not 1 or 2", group_rank);
    if (score != FT_SCORE_SOFTMAX && score != FT_SCORE_SIGMOID)
        return fail(FT_HIP_E_INVALID, "route_experts: score=%d is no FT_SCORE", score);
    if (renorm != 0 && renorm != 1) return fail(FT_HIP_E_SHAPE, "route_experts: renorm=%d is not 0 or 1", renorm);
    if (!std::isfinite(scale)) return fail(FT_HIP_E_SHAPE, "route_experts: scale is not finite");
    if (n_seqs < 0 || n_seqs > (1 << 24))
        return fail(FT_HIP_E_SHAPE, "route_experts: n_seqs=%lld not in [0, 2^24]", (long long)n_seqs);
    if (logits_stride < E || logits_stride > (int64_t)1 << 36)
        return fail(FT_HIP_E_SHAPE, "route_experts: logits_stride out of range");
    if (!ctx || !logits || !ids || !wts) return fail(FT_HIP_E_INVALID, "route_experts: null argument");
    if (n_seqs == 0) return FT_HIP_OK;
    const RouteArgs a{logits, logits_stride, bias, expert_scale, ids, wts, score == FT_SCORE_SIGMOID, (int)G,
                      (int)(E / G), (int)top_groups, group_rank, renorm, (double)scale, (int)E, (int)top_k, n_seqs};
    DeviceGuard on(ctx->device);
    if (!on.ok) return fail(FT_HIP_E_DEVICE, "route_experts: device %d cannot be made current", ctx->device);
    const dim3 grid((unsigned)((n_seqs + 3) / 4)), block(256);
    const size_t lds = G > 1 ? 4 * (size_t)E * sizeof(double) : 0;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (E <= 64)
        hipLaunchKernelGGL(k_route_experts<1>, grid, block, lds, s, a);
    else if (E <= 128)
        hipLaunchKernelGGL(k_route_experts<2>, grid, block, lds, s, a);
    else if (E <= 256)
        hipLaunchKernelGGL(k_route_experts<4>, grid, block, lds, s, a);
    else if (E <= 512)
        hipLaunchKernelGGL(k_route_experts<8>, grid, block, lds, s, a);
    else
        hipLaunchKernelGGL(k_route_experts<16>, grid, block, lds, s, a);
    return launch_status("route_experts");
}
