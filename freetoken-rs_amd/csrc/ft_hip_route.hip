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
// SUB lanes of a wave share a token (64 / SUB tokens a wave), each with VPL
// consecutive experts, sorted in registers once; the next expert is then the
// largest of the lanes' first ones, and its lane moves up its next. Lanes hold
// rising experts, so that among equal ones the lowest lane has the lowest.
//
// Bound by instructions: a wave of 64 lanes with four experts each runs about
// 670. Measured, kernel alone: 16384 tokens over 256 experts in 8 groups, 8 chosen,
// 23.5 us (the instructions of 16 waves a SIMD are 18 of these, the 18 MB of
// traffic 2.2); 5003 tokens over 128 experts 7.4 us; 64 tokens 6.2 and one 4.6,
// which is a launch and the chain of a single wave's selections.

#include "ft_device.hpp"
#include "ft_overlap.hpp"
#include "ft_runtime.hpp"
#include "ft_wave.hpp"

#include <algorithm>
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
    int n;
    bool vec;  // rows start on 16 bytes and E is a multiple of 4
};

// Exchanges within the SUB lanes of a token: step 0..log2(SUB)-1 of a
// butterfly, in which mirrors stand for the wider exchanges inside a row.
template <int STEP>
__device__ __forceinline__ void partner(int v, int& a, int& b) {
    if constexpr (STEP < 4) {
        a = v;
        b = dpp_i<STEP == 0 ? 0xB1 : STEP == 1 ? 0x4E : STEP == 2 ? 0x141 : 0x140>(v);
    } else {
        const auto s = STEP == 4 ? __builtin_amdgcn_permlane16_swap(v, v, false, false)
                                 : __builtin_amdgcn_permlane32_swap(v, v, false, false);
        a = s[0];
        b = s[1];
    }
}
template <int STEP>
__device__ __forceinline__ void partner(double v, double& a, double& b) {
    const long long x = __double_as_longlong(v);
    int al, bl, ah, bh;
    partner<STEP>((int)x, al, bl);
    partner<STEP>((int)(x >> 32), ah, bh);
    a = __longlong_as_double(((long long)ah << 32) | (uint32_t)al);
    b = __longlong_as_double(((long long)bh << 32) | (uint32_t)bl);
}
// Sum over the first P of a token's lanes (the others hold 0) or over aligned
// runs of P, P a power of two up to SUB.
template <int SUB, int STEP = 0, typename T>
__device__ __forceinline__ T sub_sum(T v, int P = SUB) {
    if constexpr (1 << STEP < SUB) {
        if (1 << STEP < P) {
            T a, b;
            partner<STEP>(v, a, b);
            v = a + b;
        }
        return sub_sum<SUB, STEP + 1>(v, P);
    }
    return v;
}
template <int SUB, int STEP = 0>
__device__ __forceinline__ float sub_max(float v) {
    if constexpr (1 << STEP < SUB) {
        int a, b;
        partner<STEP>(__float_as_int(v), a, b);
        return sub_max<SUB, STEP + 1>(fmaxf(__int_as_float(a), __int_as_float(b)));
    }
    return v;
}
template <int SUB>
__device__ __forceinline__ uint32_t sub_max(uint32_t v) {
    v = row_max16<(SUB < 16)>(v);
    if constexpr (SUB >= 32) {
        int a, b;
        partner<4>((int)v, a, b);
        v = max((uint32_t)a, (uint32_t)b);
    }
    if constexpr (SUB >= 64) {
        int a, b;
        partner<5>((int)v, a, b);
        v = max((uint32_t)a, (uint32_t)b);
    }
    return v;
}
// Of values that are no NaN: without the maximum with itself that fmax takes
// first of a value from memory. The wait is for a DPP move of the result.
__device__ __forceinline__ double max_of(double a, double b) {
    double r;
    asm("v_max_f64 %0, %1, %2\n\ts_nop 1" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
__device__ __forceinline__ double min_of(double a, double b) {
    double r;
    asm("v_min_f64 %0, %1, %2\n\ts_nop 1" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
// The two largest of P lanes' pairs (P a power of two up to SUB).
template <int SUB, int STEP = 0>
__device__ __forceinline__ void sub_top2(double& b1, double& b2, int P) {
    if constexpr (1 << STEP < SUB) {
        if (1 << STEP < P) {
            double a1, c1, a2, c2;
            partner<STEP>(b1, a1, c1);
            partner<STEP>(b2, a2, c2);
            b1 = max_of(a1, c1);
            b2 = max_of(min_of(a1, c1), max_of(a2, c2));
        }
        sub_top2<SUB, STEP + 1>(b1, b2, P);
    }
}

// exp(x) for x in [-745, 700], to 2^-51: x = n ln 2 + r by the sum with
// 1.5 * 2^52, whose low half is n; the series of exp(r), |r| <= ln 2 / 2, to
// r^12 (the next term is below 2^-52).
__device__ __forceinline__ double exp_series(double x) {
    const double t = fma(x, 1.4426950408889634074, 0x1.8p52), n = t - 0x1.8p52;
    double r = fma(n, -0x1.62e42fefap-1, x);  // ln 2 to 34 bits: n times it is exact
    r = fma(n, -0x1.cf79abc9e3b3ap-40, r);    // and the rest of it
    double p = scalar(1.0 / 479001600);
    p = fma(p, r, scalar(1.0 / 39916800));
    p = fma(p, r, scalar(1.0 / 3628800));
    p = fma(p, r, scalar(1.0 / 362880));
    p = fma(p, r, scalar(1.0 / 40320));
    p = fma(p, r, scalar(1.0 / 5040));
    p = fma(p, r, scalar(1.0 / 720));
    p = fma(p, r, scalar(1.0 / 120));
    p = fma(p, r, scalar(1.0 / 24));
    p = fma(p, r, scalar(1.0 / 6));
    p = fma(fma(fma(p, r, 0.5), r, 1.0), r, 1.0);
    return ldexp(p, (int)__double_as_longlong(t));
}
__device__ __forceinline__ double recip(double x) {  // of x in [1e-290, 1e305]
    double y = __builtin_amdgcn_rcp(x);
    y = fma(fma(-x, y, 1.0), y, y);
    return fma(fma(-x, y, 1.0), y, y);
}

// A key that rises with c, its last bits (`bits`) replaced by `place`; 0: not to be chosen.
__device__ __forceinline__ uint64_t key_of(double c, bool ok, uint32_t bits, uint32_t place) {
    const uint64_t b = (uint64_t)__double_as_longlong(c);
    const uint64_t key = ((b ^ ((uint64_t)((int64_t)b >> 63) | 0x8000000000000000ull)) & ~(uint64_t)bits) | place;
    return ok ? key : 0;
}

// N keys by falling size (odd-even merge sort).
template <int N>
__device__ __forceinline__ void sort_falling(uint64_t key[N]) {
#pragma unroll
    for (int p = 1; p < N; p <<= 1)
#pragma unroll
        for (int k = p; k >= 1; k >>= 1)
#pragma unroll
            for (int j = k % p; j + k < N; j += 2 * k)
#pragma unroll
                for (int i = 0; i < k; ++i)
                    if (i + j + k < N && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
                        const uint64_t x = key[i + j], y = key[i + j + k];
                        key[i + j] = y > x ? y : x;
                        key[i + j + k] = y > x ? x : y;
                    }
}

template <int SUB, int VPL>
__global__ __launch_bounds__(256) void k_route_experts(RouteArgs a) {
    extern __shared__ double lds[];  // with groups: per wave its tokens' c
    __shared__ int chosen[256];
    constexpr int TOKENS = 64 / SUB;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sub = lane & (SUB - 1), first = lane & ~(SUB - 1);
    const int wanted = ((int)blockIdx.x * 4 + wave) * TOKENS + lane / SUB;
    const int token = min(wanted, a.n - 1);  // past the last: computed again, not stored
    const float* row = a.logits + token * a.stride;
    const double none = -(double)INFINITY;

    float l[VPL];
    if (a.vec) {
#pragma unroll
        for (int j = 0; j < VPL; j += 4) {
            const int e = sub * VPL + j;
            const float4 x = *reinterpret_cast<const float4*>(row + (e < a.E ? e : 0));
            const bool in = e < a.E;
            l[j] = in ? x.x : -INFINITY, l[j + 1] = in ? x.y : -INFINITY;
            l[j + 2] = in ? x.z : -INFINITY, l[j + 3] = in ? x.w : -INFINITY;
        }
    } else {
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
            const int e = sub * VPL + j;
            const float x = row[e < a.E ? e : 0];
            l[j] = e < a.E ? x : -INFINITY;
        }
    }
    float bias[VPL];
#pragma unroll
    for (int j = 0; j < VPL; ++j) bias[j] = a.bias ? a.bias[min(sub * VPL + j, a.E - 1)] : 0.0f;
    double s[VPL], sum = 0.0;
    float m = -INFINITY;
    if (a.sigmoid) {
#pragma unroll
        for (int j = 0; j < VPL; ++j) s[j] = recip(1.0 + exp_series(fmin(fmax(-(double)l[j], -700.0), 700.0)));
    } else {
#pragma unroll
        for (int j = 0; j < VPL; ++j) m = fmaxf(m, l[j]);  // NaN is skipped
        m = sub_max<SUB>(m);
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
            s[j] = l[j] == m ? 1.0 : exp_series(fmax((double)l[j] - (double)m, -745.0));  // several +inf share
            sum += l[j] > -INFINITY ? s[j] : 0.0;
        }
        sum = sub_sum<SUB>(sum);
        const double per = recip(fmax(sum, 1.0));
#pragma unroll
        for (int j = 0; j < VPL; ++j) s[j] *= per;
    }
    // a key's last bits are the expert's place in its lane, the first the largest: c of a lane that differ by less than
    // 2^-48 of themselves count as equal
    uint64_t key[VPL];
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
        const double c = s[j] + (double)bias[j];
        const bool ok = l[j] > -INFINITY && c > none;  // -inf, NaN: never chosen
        key[j] = key_of(c, ok, VPL - 1, VPL - 1 - j);
        s[j] = ok ? c : none;
    }

    if (a.n_groups > 1) {
        double* w = lds + (wave * 64 + first) * VPL;
#pragma unroll
        for (int j = 0; j < VPL; ++j) w[sub * VPL + j] = s[j];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");  // read by the wave's other lanes below
        __builtin_amdgcn_wave_barrier();
        // P lanes to a group: its two best
        const int P = SUB >> (32 - __clz(a.n_groups - 1)), g = sub / P;
        double b1 = none, b2 = none;
        if (g < a.n_groups)
            for (int i = sub & (P - 1); i < a.group_size; i += P) {
                const double v = w[g * a.group_size + i];
                b2 = max_of(b2, min_of(b1, v));
                b1 = max_of(b1, v);
            }
        sub_top2<SUB>(b1, b2, P);
        const double gs = a.group_rank == 2 && b2 > none ? b1 + b2 : b1;
        // open: fewer than top_groups groups are ahead of it; its lanes ask a part of the others each
        int ahead = 0;
        for (int o = sub & (P - 1); o - (sub & (P - 1)) < a.n_groups; o += P) {
            const long long x = __double_as_longlong(gs);
            const int from = first + min(o, a.n_groups - 1) * P;
            const int lo = __shfl((int)x, from), hi = __shfl((int)(x >> 32), from);
            const double v = __longlong_as_double(((long long)hi << 32) | (uint32_t)lo);
            ahead += o < a.n_groups && (v > gs || (v == gs && o < g));
        }
        ahead = sub_sum<SUB>(ahead, P);
        const uint64_t open = __ballot(ahead < a.top_groups) >> first;
        // e / group_size by a product, for e * group_size < 2^20
        const uint32_t per = ((1u << 20) + a.group_size - 1) / a.group_size;
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
            const uint32_t of = __umul24(sub * VPL + j, per) >> 20;
            if (!((open >> min(of * P, 63u)) & 1)) key[j] = 0;
        }
    }

    sort_falling<VPL>(key);
    int* out = chosen + wave * 64 + first;
    int found = 0;
    for (int r = 0; r < a.k; ++r) {
        const uint32_t top = sub_max<SUB>((uint32_t)(key[0] >> 32));
        const bool here = (uint32_t)(key[0] >> 32) == top && top;
        constexpr uint64_t MINE = ~0ull >> (64 - SUB);
        uint64_t set = __ballot(here) >> first & MINE;
        if (__ballot(__popcll(set) > 1)) {  // equal upper halves: rare
            const uint32_t own = here ? (uint32_t)key[0] | (VPL - 1) : 0u, low = sub_max<SUB>(own);
            set = __ballot(here && own == low) >> first & MINE;  // of equal c the lowest lane's
        }
        found += set != 0;  // 0: none left for this token
        if (sub == __ffsll((unsigned long long)set) - 1) {
            out[r] = sub * VPL + (VPL - 1) - (int)((uint32_t)key[0] & (VPL - 1));
#pragma unroll
            for (int j = 0; j + 1 < VPL; ++j) key[j] = key[j + 1];
            key[VPL - 1] = 0;
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
    __builtin_amdgcn_wave_barrier();
    int e = 0;
    double wt = 0.0;  // lane r holds the r-th chosen
    if (sub < found) {
        e = out[sub];
        const double x = row[e];
        // as above; where that is far out, by the full functions, which end in 0
        if (a.sigmoid)
            wt = x > -700.0 ? recip(1.0 + exp_series(fmax(-x, -700.0))) : 1.0 / (1.0 + exp(-x));
        else
            wt = x == (double)m ? 1.0 / sum
                                : (x - (double)m > -700.0 ? exp_series(x - (double)m) : exp(x - (double)m)) * recip(sum);
    }
    if (a.renorm) {
        const double total = sub_sum<SUB>(wt, 1 << (32 - __clz(max(a.k - 1, 0))));
        wt = total > 1e-290 ? wt * recip(total) : total > 0.0 ? wt / total : 0.0;
    }
    if (sub < a.k && wanted < a.n) {
        a.ids[(int64_t)token * a.k + sub] = e;
        a.wts[(int64_t)token * a.k + sub] = (float)(wt * a.scale * (a.escale ? (double)a.escale[e] : 1.0));
    }
}

template <int SUB, int VPL>
void launch_route(const RouteArgs& a, void* stream) {
    constexpr int TOKENS = 4 * (64 / SUB);
    const size_t lds = a.n_groups > 1 ? 256 * VPL * sizeof(double) : 0;
    hipLaunchKernelGGL((k_route_experts<SUB, VPL>), dim3((unsigned)((a.n + TOKENS - 1) / TOKENS)), dim3(256), lds,
                       static_cast<hipStream_t>(stream), a);
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
        return fail(FT_HIP_E_SHAPE, "route_experts: n_groups=%lld not in [1, %d] or no divisor of %lld experts", G,
                    MAX_GROUPS, E);
    if (top_groups <= 0 || top_groups > G)
        return fail(FT_HIP_E_SHAPE, "route_experts: top_groups=%lld not in [1, %lld]", (long long)top_groups, G);
    if (top_k <= 0 || top_k > 32 || top_k > top_groups * (E / G))
        return fail(FT_HIP_E_SHAPE, "route_experts: top_k=%lld not in [1, 32] or more than the open groups hold",
                    (long long)top_k);
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
    if (!aligned(logits, 4) || !aligned(bias, 4) || !aligned(expert_scale, 4) || !aligned(ids, 4) || !aligned(wts, 4))
        return fail(FT_HIP_E_SHAPE, "route_experts: a pointer is not aligned to 4 bytes");
    if (!ctx) return fail(FT_HIP_E_INVALID, "route_experts: null argument");
    if (n_seqs == 0) return FT_HIP_OK;  // an empty tensor has no address
    if (!logits || !ids || !wts) return fail(FT_HIP_E_INVALID, "route_experts: null argument");
    const Span in_l{logits, n_seqs, logits_stride * 4, E * 4}, in_b{bias, 1, 0, E * 4}, in_s{expert_scale, 1, 0, E * 4},
        out_i{ids, 1, 0, n_seqs * top_k * 4}, out_w{wts, 1, 0, n_seqs * top_k * 4};
    for (const Span& out : {out_i, out_w})
        if (overlap(out, in_l) || overlap(out, in_b) || overlap(out, in_s))
            return fail(FT_HIP_E_SHAPE, "route_experts: ids or wts overlap an input");
    if (overlap(out_i, out_w)) return fail(FT_HIP_E_SHAPE, "route_experts: ids and wts overlap");
    const RouteArgs a{logits, logits_stride, bias, expert_scale, ids, wts, score == FT_SCORE_SIGMOID, (int)G,
                      (int)(E / G), (int)top_groups, group_rank, renorm, (double)scale, (int)E, (int)top_k, (int)n_seqs,
                      aligned(logits, 16) && logits_stride % 4 == 0 && E % 4 == 0};
    DeviceGuard on(ctx->device);
    if (!on.ok) return fail(FT_HIP_E_DEVICE, "route_experts: device %d cannot be made current", ctx->device);
    // As few lanes to a token as hold its experts four to a lane, and one lane each for its groups and its choices.
    // (Eight to a lane need a fifth fewer instructions, but each wave's chain of selections is longer: 16384 tokens
    // over 256 experts 24.9 us against 23.5, 5003 over 128 8.6 against 7.4.)
    const int64_t lanes = std::max({(E + 3) / 4, G, (long long)top_k});
    if (lanes <= 8)
        launch_route<8, 4>(a, stream);
    else if (lanes <= 16)
        launch_route<16, 4>(a, stream);
    else if (lanes <= 32)
        launch_route<32, 4>(a, stream);
    else if (E <= 256)
        launch_route<64, 4>(a, stream);
    else if (E <= 512)
        launch_route<64, 8>(a, stream);
    else
        launch_route<64, 16>(a, stream);
    return launch_status("route_experts");
}
