// ft_hip_logits.hip -- penalties for repeated tokens, biases and a grammar's
// mask on rows of logits, in front of the draw (ft_hip_adjust_logits).
//
// Per row and token v, c its occurrences in the row's history:
//   x = l;  c > 0: x = (x > 0 ? x / repetition : x * repetition) - (presence + frequency c)
//   x += the row's biases for v, in their order;  masked: x = -inf
//
// A workgroup takes a chunk of a row. Its logits are on their way while it goes
// through the history and the biases and keeps what falls into the chunk: counts
// in LDS (whole numbers, whose sum no order changes) and the biased tokens as a
// list with a bit a token. Then each logit moves once. Bound by memory: a row is
// read and written once in f32; the history comes from L2 once per chunk.

#include "ft_device.hpp"
#include "ft_overlap.hpp"
#include "ft_runtime.hpp"

#include <cmath>

using namespace ft;

namespace {

struct LogitArgs {
    const void* logits;
    int64_t stride;
    float* out;
    int64_t out_stride;
    int V;
    const int32_t* history;
    int64_t h_stride;
    int h_max;
    const int32_t* h_len;
    const float *repetition, *presence, *frequency;
    const int32_t* bias_ids;
    const float* bias;
    int n_bias;
    const uint32_t* mask;
    int64_t mask_stride;
    bool vec;
};

constexpr int MAX_BIAS = FT_ADJUST_MAX_BIAS;

template <int TYPE>
__device__ __forceinline__ float4 four(const LogitArgs& a, int64_t row, int v) {
    float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if constexpr (TYPE == FT_TYPE_F32) {
        const float* p = static_cast<const float*>(a.logits) + row * a.stride + v;
        if (a.vec && v + 4 <= a.V) return *reinterpret_cast<const float4*>(p);
        for (int i = 0; i < 4; ++i)
            if (v + i < a.V) x[i] = p[i];
    } else {
        const uint16_t* p = static_cast<const uint16_t*>(a.logits) + row * a.stride + v;
        uint16_t b[4] = {0, 0, 0, 0};
        if (a.vec && v + 4 <= a.V) {
            const uint2 w = *reinterpret_cast<const uint2*>(p);
            b[0] = (uint16_t)w.x, b[1] = (uint16_t)(w.x >> 16), b[2] = (uint16_t)w.y, b[3] = (uint16_t)(w.y >> 16);
        } else {
            for (int i = 0; i < 4; ++i)
                if (v + i < a.V) b[i] = p[i];
        }
        for (int i = 0; i < 4; ++i) x[i] = TYPE == FT_TYPE_F16 ? h2f(b[i]) : __uint_as_float((uint32_t)b[i] << 16);
    }
    return make_float4(x[0], x[1], x[2], x[3]);
}

// CHUNK tokens of a row by THREADS threads, four at a time
template <int TYPE, int CHUNK, int THREADS>
__global__ __launch_bounds__(THREADS) void k_adjust(LogitArgs a) {
    constexpr int EACH = CHUNK / 4 / THREADS;
    // what is not given takes no LDS: more workgroups on a CU
    extern __shared__ __attribute__((aligned(16))) uint32_t lds[];
    uint32_t* const count = lds;
    uint32_t* const biased = lds + (a.history ? CHUNK : 0);
    int* const list_at = reinterpret_cast<int*>(biased + CHUNK / 32);
    int* const list_i = list_at + a.n_bias;
    float* const list_add = reinterpret_cast<float*>(list_i + a.n_bias);
    __shared__ int listed, again;
    const int t = threadIdx.x, v0 = blockIdx.x * CHUNK;
    const int64_t row = blockIdx.y;
    float4 x[EACH];
    uint32_t bits[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const int v = v0 + (i * THREADS + t) * 4;
        x[i] = v < a.V ? four<TYPE>(a, row, v) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        bits[i] = 15;
        if (a.mask && v < a.V) bits[i] = a.mask[row * a.mask_stride + (v >> 5)] >> (v & 31);
    }
    // the lists' first entries are on their way as well
    const int32_t* const h = a.history + row * a.h_stride;
    const int32_t* const ids = a.bias_ids + row * a.n_bias;
    const float* const adds = a.bias + row * a.n_bias;
    int len = 0, id[8], bias_id = -1;
    float bias = 0.0f;
    if (a.history) {
        len = a.h_len ? a.h_len[row] : a.h_max;
#pragma unroll
        for (int u = 0; u < 8; ++u) id[u] = u * THREADS + t < a.h_max ? h[u * THREADS + t] : -1;
        for (int i = t; i < CHUNK / 4; i += THREADS) reinterpret_cast<uint4*>(count)[i] = make_uint4(0, 0, 0, 0);
    }
    if (a.n_bias) {
        if (t < a.n_bias) bias_id = ids[t], bias = adds[t];
        for (int i = t; i < CHUNK / 32; i += THREADS) biased[i] = 0;
        if (t == 0) listed = 0, again = 0;
    }
    __syncthreads();
    if (a.history) {
        len = len < a.h_max ? len : a.h_max;
        for (int i0 = 0; i0 < len; i0 += 8 * THREADS) {
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const unsigned at = (unsigned)id[u] - (unsigned)v0;
                if (i0 + u * THREADS + t < len && at < CHUNK && id[u] >= 0) atomicAdd(&count[at], 1u);
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int i = i0 + (8 + u) * THREADS + t;
                id[u] = i < len ? h[i] : -1;
            }
        }
    }
    if (a.n_bias) {
        for (int i = t; i < a.n_bias; i += THREADS) {
            const unsigned at = (unsigned)bias_id - (unsigned)v0;
            if (at < CHUNK && bias_id >= 0) {
                const int k = atomicAdd(&listed, 1);
                list_at[k] = (int)at, list_add[k] = bias, list_i[k] = i;
                if (atomicOr(&biased[at >> 5], 1u << (at & 31)) >> (at & 31) & 1) again = 1;
            }
            if (i + THREADS < a.n_bias) bias_id = ids[i + THREADS], bias = adds[i + THREADS];
        }
        __syncthreads();
        if (again) {  // a token more than once: its first entry adds them all, in their order
            constexpr int OWN = MAX_BIAS / THREADS;
            float sum[OWN];
            bool first[OWN];
#pragma unroll
            for (int u = 0; u < OWN; ++u) {
                const int k = t + u * THREADS;
                first[u] = false, sum[u] = 0.0f;
                if (k >= listed) continue;
                const int at = list_at[k], i0 = list_i[k];
                first[u] = true;
                for (int j = 0; j < listed; ++j)
                    if (list_at[j] == at && list_i[j] < i0) first[u] = false;
                if (!first[u]) continue;
                sum[u] = list_add[k];
                for (int i = i0 + 1; i < a.n_bias; ++i)
                    if (ids[i] == v0 + at) sum[u] += adds[i];
            }
            __syncthreads();
#pragma unroll
            for (int u = 0; u < OWN; ++u) {
                const int k = t + u * THREADS;
                if (k >= listed) continue;
                list_add[k] = sum[u];
                if (!first[u]) list_at[k] = -1;
            }
        }
    }
    __syncthreads();
    const float rep = a.repetition ? a.repetition[row] : 1.0f, pres = a.presence ? a.presence[row] : 0.0f,
                freq = a.frequency ? a.frequency[row] : 0.0f;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const int at = (i * THREADS + t) * 4, v = v0 + at;
        if (v >= a.V) continue;
        float y[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
        if (a.history) {
            const uint4 n = *reinterpret_cast<const uint4*>(&count[at]);
            const uint32_t c[4] = {n.x, n.y, n.z, n.w};
            if (n.x | n.y | n.z | n.w) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (c[e] == 0) continue;
                    if (a.repetition) y[e] = y[e] > 0.0f ? y[e] / rep : y[e] * rep;
                    y[e] -= pres + freq * (float)c[e];
                }
            }
        }
        if (a.n_bias) {
            const uint32_t b = biased[at >> 5] >> (at & 31) & 15;
            if (b) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (!(b >> e & 1)) continue;
                    for (int k = 0; k < listed; ++k)
                        if (list_at[k] == at + e) y[e] += list_add[k];
                }
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (!(bits[i] >> e & 1)) y[e] = -INFINITY;
        float* p = a.out + row * a.out_stride + v;
        if (a.vec && v + 4 <= a.V) {
            *reinterpret_cast<float4*>(p) = make_float4(y[0], y[1], y[2], y[3]);
        } else {
            for (int e = 0; e < 4; ++e)
                if (v + e < a.V) p[e] = y[e];
        }
    }
}

template <int TYPE, int CHUNK, int THREADS>
void launch_chunks(const LogitArgs& a, int64_t n, hipStream_t s) {
    const size_t lds = (a.history ? CHUNK * 4 : 0) + (a.n_bias ? CHUNK / 8 + a.n_bias * 12 : 0);
    hipLaunchKernelGGL((k_adjust<TYPE, CHUNK, THREADS>), dim3((unsigned)((a.V + CHUNK - 1) / CHUNK), (unsigned)n), dim3(THREADS), lds, s, a);
}

// Chunks as long as there are enough of them: each goes through the whole history. 64 rows of 262144 with 6000 tokens and
// 100 biases 32.1 us, in chunks of 8192 37.2 and of 4096 37.5; 12 rows 11.3, 10.0 and 9.8.
template <int TYPE>
void launch_adjust(const LogitArgs& a, int64_t n, hipStream_t s) {
    const int64_t values = (int64_t)a.V * n;
    if (values < 1 << 20)
        launch_chunks<TYPE, 2048, 256>(a, n, s);
    else if (values < 1 << 23)
        launch_chunks<TYPE, 4096, 512>(a, n, s);
    else
        launch_chunks<TYPE, 16384, 1024>(a, n, s);
}

}  // namespace

extern "C" int ft_hip_adjust_logits(ft_hip_ctx* ctx, void* stream, const void* logits, int logits_type,
                                    int64_t logits_stride, int64_t vocab, int64_t n, const int32_t* history,
                                    int64_t history_stride, int64_t history_max, const int32_t* history_len,
                                    const float* repetition, const float* presence, const float* frequency,
                                    const int32_t* bias_ids, const float* bias, int64_t n_bias, const uint32_t* mask,
                                    int64_t mask_stride, float* out, int64_t out_stride) {
    clear_error();
    if (vocab <= 0 || vocab > FT_SAMPLE_MAX_VOCAB)
        return fail(FT_HIP_E_SHAPE, "adjust_logits: vocab=%lld not in [1, %d]", (long long)vocab, FT_SAMPLE_MAX_VOCAB);
    if (n < 0 || n > FT_SAMPLE_MAX_ROWS)
        return fail(FT_HIP_E_SHAPE, "adjust_logits: n=%lld not in [0, %d]", (long long)n, FT_SAMPLE_MAX_ROWS);
    if (logits_type != FT_TYPE_F32 && logits_type != FT_TYPE_F16 && logits_type != FT_TYPE_BF16)
        return fail(FT_HIP_E_INVALID, "adjust_logits: logits_type=%d is no FT_TYPE", logits_type);
    const int64_t most = (int64_t)1 << 40, words = (vocab + 31) / 32;
    if (logits_stride < vocab || logits_stride > most || out_stride < vocab || out_stride > most)
        return fail(FT_HIP_E_SHAPE, "adjust_logits: logits_stride or out_stride out of range");
    if (history && (history_max < 1 || history_max > 1 << 24 || history_stride < history_max || history_stride > most))
        return fail(FT_HIP_E_SHAPE, "adjust_logits: history_max=%lld not in [1, 2^24] or history_stride out of range",
                    (long long)history_max);
    if (n_bias < 0 || n_bias > MAX_BIAS)
        return fail(FT_HIP_E_SHAPE, "adjust_logits: n_bias=%lld not in [0, %d]", (long long)n_bias, MAX_BIAS);
    if (mask && (mask_stride < words || mask_stride > most))
        return fail(FT_HIP_E_SHAPE, "adjust_logits: mask_stride out of range");
    const int64_t size = logits_type == FT_TYPE_F32 ? 4 : 2;
    if (!aligned(logits, size) || !aligned(out, 4) || !aligned(history, 4) || !aligned(history_len, 4) ||
        !aligned(repetition, 4) || !aligned(presence, 4) || !aligned(frequency, 4) || !aligned(bias_ids, 4) ||
        !aligned(bias, 4) || !aligned(mask, 4))
        return fail(FT_HIP_E_SHAPE, "adjust_logits: a pointer is not aligned to its type");
    if (!ctx) return fail(FT_HIP_E_INVALID, "adjust_logits: null argument");
    if (n == 0) return FT_HIP_OK;  // an empty tensor has no address
    if (!logits || !out || (n_bias && (!bias_ids || !bias))) return fail(FT_HIP_E_INVALID, "adjust_logits: null argument");
    // a thread writes the places that it has read: out may be the logits themselves
    const Span so{out, n, out_stride * 4, vocab * 4}, sl{logits, n, logits_stride * size, vocab * size};
    if (overlap(so, sl) && !(out == logits && size == 4 && (n == 1 || out_stride == logits_stride)))
        return fail(FT_HIP_E_SHAPE, "adjust_logits: out overlaps the logits other than row on row");
    const auto row4 = [&](const void* p, int64_t each) { return Span{p, 1, 0, n * each * 4}; };
    const Span in[] = {{history, n, history_stride * 4, history_max * 4}, row4(history_len, 1), row4(repetition, 1),
                       row4(presence, 1), row4(frequency, 1), row4(bias_ids, n_bias), row4(bias, n_bias),
                       {mask, n, mask_stride * 4, words * 4}};
    for (const Span& i : in)
        if (overlap(so, i)) return fail(FT_HIP_E_SHAPE, "adjust_logits: out overlaps an input");
    LogitArgs a;
    a.logits = logits, a.stride = logits_stride, a.out = out, a.out_stride = out_stride, a.V = (int)vocab;
    a.history = history, a.h_stride = history_stride, a.h_max = (int)history_max, a.h_len = history_len;
    a.repetition = repetition, a.presence = presence, a.frequency = frequency;
    a.bias_ids = bias_ids, a.bias = bias, a.n_bias = (int)n_bias, a.mask = mask, a.mask_stride = mask_stride;
    a.vec = aligned(logits, 4 * size) && logits_stride % 4 == 0 && aligned(out, 16) && out_stride % 4 == 0;
    DeviceGuard on(ctx->device);
    if (!on.ok) return fail(FT_HIP_E_DEVICE, "adjust_logits: device %d cannot be made current", ctx->device);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (logits_type == FT_TYPE_F32)
        launch_adjust<FT_TYPE_F32>(a, n, s);
    else if (logits_type == FT_TYPE_F16)
        launch_adjust<FT_TYPE_F16>(a, n, s);
    else
        launch_adjust<FT_TYPE_BF16>(a, n, s);
    return launch_status("adjust_logits");
}
