// ft_hip_sample.hip -- a token drawn from each row of logits with
// temperature, top-k, top-p and min-p from a given random number
// (ft_hip_sample_tokens).
//
// Per row, with M the largest logit: e_i = exp((l_i - M) / T). Logits falling
// (equal ones by rising index) are the order; kept are its first top_k, of
// these the shortest prefix whose e sum to top_p of theirs, of these the e of
// at least min_p. The token is the first kept index, in index order, at which
// the running sum of e passes u times the kept sum.
//
// Where a running sum passes a limit is decided in f64: over a vocabulary's
// hundreds of thousands of terms f32 sums would move the border by whole
// tokens. Sums are made in a fixed order, and where many threads add to one
// counter it holds whole numbers, so a row's result is the same on every run.

#include "ft_device.hpp"
#include "ft_runtime.hpp"

#include <cmath>

using namespace ft;

namespace {

constexpr int ROW_THREADS = 1024, ROW_WAVES = ROW_THREADS / 64;
constexpr int FIX = 42;  // fraction bits of a weight <= 1: 2^21 of them stay below 2^63

struct SampleArgs {
    const void* logits;
    int64_t stride;
    int V;
    const float* temperature;
    const int32_t* top_k;
    const float* top_p;
    const float* min_p;
    const float* u;
    int32_t* tokens;
    float* logprobs;
};

// A row's settings, with what is out of range brought into it.
struct Row {
    double inv_t, p, m, u;
    int k;
    bool greedy;
};

__device__ __forceinline__ Row row_of(const SampleArgs& a, int64_t r) {
    Row s;
    const float t = a.temperature ? a.temperature[r] : 1.0f;
    s.greedy = !(t > 0.0f);
    s.inv_t = s.greedy ? 1.0 : 1.0 / (double)t;
    const int k = a.top_k ? a.top_k[r] : 0;
    s.k = k > 0 && k < a.V ? k : a.V;
    const float p = a.top_p ? a.top_p[r] : 1.0f;
    s.p = p < 1.0f ? fmax((double)p, 0.0) : 1.0;  // NaN: off
    const float m = a.min_p ? a.min_p[r] : 0.0f;
    s.m = m > 0.0f ? fmin((double)m, 1.0) : 0.0;  // NaN: off
    const float u = a.u[r];
    s.u = u > 0.0f ? fmin((double)u, 1.0) : 0.0;
    return s;
}

template <int TYPE>
__device__ __forceinline__ float logit(const void* row, int i) {
    if constexpr (TYPE == FT_TYPE_F32) return static_cast<const float*>(row)[i];
    const uint16_t b = static_cast<const uint16_t*>(row)[i];
    return TYPE == FT_TYPE_F16 ? h2f(b) : __uint_as_float((uint32_t)b << 16);
}

// Logits as whole numbers in the same order; -0 is +0.
__device__ __forceinline__ uint32_t key_of(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

// exp((l - at) / T) for l <= at; one of several +inf is as good as another.
__device__ __forceinline__ double weight(float l, float at, double inv_t) {
    return l == at ? 1.0 : at == INFINITY ? 0.0 : exp(((double)l - (double)at) * inv_t);
}

__device__ __forceinline__ double shfl_f64(double v, int l) {
    const long long b = __double_as_longlong(v);
    const int lo = __shfl((int)b, l), hi = __shfl((int)(b >> 32), l);
    return __longlong_as_double(((long long)hi << 32) | (uint32_t)lo);
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) v += shfl_f64(v, (threadIdx.x & 63) ^ o);
    return v;
}
// Sum of lanes 0..lane.
__device__ __forceinline__ double wave_scan(double v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double x = shfl_f64(v, lane >= o ? lane - o : lane);
        if (lane >= o) v += x;
    }
    return v;
}
__device__ __forceinline__ int wave_scan_i(int v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int x = __shfl(v, lane >= o ? lane - o : lane);
        if (lane >= o) v += x;
    }
    return v;
}

struct RowLds {
    uint64_t w[1024];
    uint32_t n[1024];
    double part[ROW_WAVES];
    int parti[ROW_WAVES];
    int pick;
    double at, at_w;
    int at_n;
};

// Where the order is cut: the first `ties` values equal to key and all above.
struct Cut {
    uint32_t key;
    int ties, of;   // of: how many values equal key
    double before;  // their sum above key
    double e;       // one of key's
};

// First place of the order at which the count (by_count) or the sum reaches
// the target: the key range [lo, hi] is counted into up to 1024 equal pieces,
// the piece that reaches it is the next range, until a piece is one key. A
// piece's weights are summed as whole numbers relative to its upper edge, so
// that the sum has about FIX bits wherever it lies.
template <int TYPE>
__device__ Cut find_cut(const void* row, int V, const Row& s, float M, bool by_count, bool sums, double target,
                        RowLds& l) {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    uint32_t hi = key_of(M), lo = M == INFINITY ? hi : key_of(-INFINITY) + 1;
    int base_n = 0;
    double base_w = 0.0;
    for (;;) {
        const uint32_t width = hi - lo;
        const int shift = width < 1024u ? 0 : 22 - __clz(width);
        l.n[t] = 0;
        l.w[t] = 0;
        if (t == 0) l.pick = 1024;
        __syncthreads();
        for (int i = t; i < V; i += ROW_THREADS) {
            const float v = logit<TYPE>(row, i);
            const uint32_t k = key_of(v);
            if (!(v > -INFINITY) || k < lo || k > hi) continue;
            const uint32_t b = (hi - k) >> shift;
            atomicAdd(&l.n[b], 1u);
            if (sums) {
                const double e = weight(v, of_key(hi - (b << shift)), s.inv_t);
                atomicAdd((unsigned long long*)&l.w[b], (unsigned long long)(e * (double)(1ull << FIX) + 0.5));
            }
        }
        __syncthreads();
        const int own_n = (int)l.n[t];
        const uint64_t last = (uint64_t)t << shift;
        const double own_w = own_n && sums ? (double)l.w[t] * (1.0 / (double)(1ull << FIX)) *
                                                 weight(of_key(hi - (uint32_t)last), M, s.inv_t)
                                           : 0.0;
        const double scan_w = wave_scan(own_w);
        const int scan_n = wave_scan_i(own_n);
        if (lane == 63) {
            l.part[wave] = scan_w;
            l.parti[wave] = scan_n;
        }
        __syncthreads();
        double cum_w = base_w;
        int cum_n = base_n;
        for (int i = 0; i < wave; ++i) {
            cum_w += l.part[i];
            cum_n += l.parti[i];
        }
        const double prev_w = cum_w + (scan_w - own_w);
        const int prev_n = cum_n + scan_n - own_n;
        cum_w += scan_w;
        cum_n += scan_n;
        const bool there = own_n && (by_count ? (double)cum_n >= target : cum_w >= target);
        if (there) atomicMin(&l.pick, t);
        __syncthreads();
        if (l.pick == 1024) {  // a rounding below the target: the last piece that holds anything
            __syncthreads();
            if (t == 0) l.pick = -1;
            __syncthreads();
            if (own_n) atomicMax(&l.pick, t);
            __syncthreads();
        }
        const int b = l.pick;
        if (t == b) {
            l.at = prev_w;
            l.at_w = own_w;
            l.at_n = prev_n;
        }
        __syncthreads();
        base_w = l.at;
        base_n = l.at_n;
        const int here = (int)l.n[b];
        hi -= (uint32_t)b << shift;
        if (shift == 0) {
            Cut c{hi, here, here, base_w, weight(of_key(hi), M, s.inv_t)};
            if (by_count) {
                c.ties = min(here, max(1, (int)target - base_n));
            } else if (c.e > 0.0) {  // the fewest with before + ties * e >= target
                int m = (int)fmin((double)here, fmax(1.0, ceil((target - base_w) / c.e)));
                if (m > 1 && base_w + (m - 1) * c.e >= target) --m;
                if (m < here && base_w + m * c.e < target) ++m;
                c.ties = m;
            }
            __syncthreads();
            return c;
        }
        const uint32_t span = (1u << shift) - 1;
        if (hi - lo > span) lo = hi - span;
        __syncthreads();
    }
}

// One workgroup takes a row from memory as often as it needs it: right for
// every case, for any number of kept or equal values.
template <int TYPE>
__device__ void sample_streaming(const SampleArgs& a, int64_t r, const Row& s, RowLds& l) {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, V = a.V;
    const void* row = static_cast<const char*>(a.logits) + r * a.stride * (TYPE == FT_TYPE_F32 ? 4 : 2);
    float M = -INFINITY;
    for (int i = t; i < V; i += ROW_THREADS) M = fmaxf(M, logit<TYPE>(row, i));  // NaN is skipped
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) M = fmaxf(M, __shfl_xor(M, o));
    if (lane == 0) l.part[wave] = M;
    if (t == 0) l.pick = 0x7FFFFFFF;
    __syncthreads();
    for (int i = 0; i < ROW_WAVES; ++i) M = fmaxf(M, (float)l.part[i]);
    __syncthreads();
    if (M == -INFINITY) {  // nothing can be drawn
        if (t == 0) {
            a.tokens[r] = -1;
            if (a.logprobs) a.logprobs[r] = NAN;
        }
        return;
    }
    if (s.greedy) {
        for (int i = t; i < V; i += ROW_THREADS)
            if (logit<TYPE>(row, i) == M) {
                atomicMin(&l.pick, i);
                break;
            }
        __syncthreads();
        if (t == 0) {
            a.tokens[r] = l.pick;
            if (a.logprobs) a.logprobs[r] = 0.0f;
        }
        return;
    }
    Cut cut{0, 0x7FFFFFFF, 0x7FFFFFFF, 0.0, 0.0};
    const bool by_p = s.p < 1.0;
    if (s.k < V) cut = find_cut<TYPE>(row, V, s, M, true, by_p, (double)s.k, l);
    if (by_p) {
        double z;
        if (s.k < V) {
            z = cut.before + cut.ties * cut.e;
        } else {
            z = 0.0;
            for (int i = t; i < V; i += ROW_THREADS) {
                const float v = logit<TYPE>(row, i);
                if (v > -INFINITY) z += weight(v, M, s.inv_t);
            }
            z = wave_sum(z);
            if (lane == 0) l.part[wave] = z;
            __syncthreads();
            z = 0.0;
            for (int i = 0; i < ROW_WAVES; ++i) z += l.part[i];
            __syncthreads();
        }
        const Cut c = find_cut<TYPE>(row, V, s, M, false, true, s.p * z, l);
        if (c.key > cut.key || (c.key == cut.key && c.ties < cut.ties)) cut = c;
    }
    // of the values equal to the cut's key, those up to index tie_end are kept
    int tie_end = V;
    if (cut.ties < cut.of) {
        int seen = 0;
        for (int base = 0; base < V; base += ROW_THREADS) {
            const int i = base + t;
            const float v = i < V ? logit<TYPE>(row, i) : -INFINITY;
            const bool tie = v > -INFINITY && key_of(v) == cut.key;
            const uint64_t set = __ballot(tie);
            if (lane == 0) l.parti[wave] = __popcll(set);
            __syncthreads();
            int rank = seen;
            for (int w = 0; w < ROW_WAVES; ++w) {
                if (w < wave) rank += l.parti[w];
                seen += l.parti[w];
            }
            if (tie && rank + __popcll(set & ((2ull << lane) - 1)) == cut.ties) l.pick = i;
            __syncthreads();
            if (seen >= cut.ties) break;
        }
        tie_end = l.pick;
        __syncthreads();
    }
    const auto kept = [&](int i) {
        const float v = logit<TYPE>(row, i);
        if (!(v > -INFINITY)) return 0.0;
        const uint32_t k = key_of(v);
        if (k < cut.key || (k == cut.key && i > tie_end)) return 0.0;
        const double e = weight(v, M, s.inv_t);
        return e >= s.m ? e : 0.0;
    };
    // the range that holds the token, a sixteenth of the last each time
    int lo = 0, len = V;
    double before = 0.0, total = 0.0, goal = 0.0;
    while (len > 64) {
        const int piece = ((len + ROW_WAVES - 1) / ROW_WAVES + 63) / 64 * 64;
        const int b0 = lo + wave * piece, b1 = min(lo + len, b0 + piece);
        double z = 0.0;
        for (int i = b0 + lane; i < b1; i += 64) z += kept(i);
        z = wave_sum(z);
        if (lane == 0) l.part[wave] = z;
        __syncthreads();
        if (len == V) {
            for (int i = 0; i < ROW_WAVES; ++i) total += l.part[i];
            goal = s.u * total;
        }
        int at = -1, some = 0;
        double cum = before, at_before = before, some_before = before;
        for (int i = 0; i < ROW_WAVES; ++i) {
            const double z = l.part[i];
            if (z > 0.0) {
                some = i;
                some_before = cum;
            }
            if (at < 0 && cum + z > goal) {
                at = i;
                at_before = cum;
            }
            cum += z;
        }
        if (at < 0) {  // u at 1, or a rounding: the last that holds anything
            at = some;
            at_before = some_before;
        }
        before = at_before;
        len = min(piece, lo + len - (lo + at * piece));
        lo += at * piece;
        __syncthreads();
    }
    if (wave) return;
    const double e = lane < len ? kept(lo + lane) : 0.0;
    const double cum = wave_scan(e);
    if (V <= 64) {
        total = shfl_f64(cum, 63);
        goal = s.u * total;
    }
    const uint64_t over = __ballot(e > 0.0 && before + cum > goal), any = __ballot(e > 0.0);
    const int at = over ? __ffsll((unsigned long long)over) - 1 : 63 - __clzll((long long)any);
    if (lane == at) {
        a.tokens[r] = lo + lane;
        if (a.logprobs) a.logprobs[r] = (float)log(e / total);
    }
}

template <int TYPE>
__global__ __launch_bounds__(ROW_THREADS) void k_sample_rows(SampleArgs a) {
    __shared__ RowLds l;
    const int64_t r = blockIdx.x;
    sample_streaming<TYPE>(a, r, row_of(a, r), l);
}

}  // namespace

extern "C" size_t ft_hip_sample_tokens_workspace_bytes(int64_t vocab, int64_t n) {
    if (vocab <= 0 || vocab > FT_SAMPLE_MAX_VOCAB || n < 0 || n > FT_SAMPLE_MAX_ROWS) return 0;
    return 256;
}

extern "C" int ft_hip_sample_tokens(ft_hip_ctx* ctx, void* stream, const void* logits, int logits_type,
                                    int64_t logits_stride, int64_t vocab, int64_t n, const float* temperature,
                                    const int32_t* top_k, const float* top_p, const float* min_p, const float* u,
                                    int32_t* tokens, float* logprobs, void* workspace, size_t workspace_bytes) {
    clear_error();
    if (vocab <= 0 || vocab > FT_SAMPLE_MAX_VOCAB)
        return fail(FT_HIP_E_SHAPE, "sample_tokens: vocab=%lld not in [1, %d]", (long long)vocab, FT_SAMPLE_MAX_VOCAB);
    if (n < 0 || n > FT_SAMPLE_MAX_ROWS)
        return fail(FT_HIP_E_SHAPE, "sample_tokens: n=%lld not in [0, %d]", (long long)n, FT_SAMPLE_MAX_ROWS);
    if (logits_type != FT_TYPE_F32 && logits_type != FT_TYPE_F16 && logits_type != FT_TYPE_BF16)
        return fail(FT_HIP_E_INVALID, "sample_tokens: logits_type=%d is no FT_TYPE", logits_type);
    if (logits_stride < vocab || logits_stride > (int64_t)1 << 40)
        return fail(FT_HIP_E_SHAPE, "sample_tokens: logits_stride out of range");
    if (reinterpret_cast<uintptr_t>(logits) % (logits_type == FT_TYPE_F32 ? 4 : 2))
        return fail(FT_HIP_E_SHAPE, "sample_tokens: logits are not aligned to their type");
    if (reinterpret_cast<uintptr_t>(workspace) % 16)
        return fail(FT_HIP_E_SHAPE, "sample_tokens: workspace must be 16-byte aligned");
    const size_t need = ft_hip_sample_tokens_workspace_bytes(vocab, n);
    if (workspace_bytes < need)
        return fail(FT_HIP_E_SHAPE, "sample_tokens: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    if (!ctx || !logits || !u || !tokens || !workspace) return fail(FT_HIP_E_INVALID, "sample_tokens: null argument");
    if (n == 0) return FT_HIP_OK;
    const SampleArgs a{logits, logits_stride, (int)vocab, temperature, top_k, top_p, min_p, u, tokens, logprobs};
    DeviceGuard on(ctx->device);
    if (!on.ok) return fail(FT_HIP_E_DEVICE, "sample_tokens: device %d cannot be made current", ctx->device);
    const dim3 grid((unsigned)n), block(ROW_THREADS);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (logits_type == FT_TYPE_F32)
        hipLaunchKernelGGL(k_sample_rows<FT_TYPE_F32>, grid, block, 0, s, a);
    else if (logits_type == FT_TYPE_F16)
        hipLaunchKernelGGL(k_sample_rows<FT_TYPE_F16>, grid, block, 0, s, a);
    else
        hipLaunchKernelGGL(k_sample_rows<FT_TYPE_BF16>, grid, block, 0, s, a);
    return launch_status("sample_tokens");
}
