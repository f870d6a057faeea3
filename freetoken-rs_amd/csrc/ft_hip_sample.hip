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
//
// Rows of up to 8192 logits are one launch, longer ones a scan by many
// workgroups and a finish by one per row; what bounds each, and its times
// (kernels alone, f32 logits), stand beside it.

#include "ft_device.hpp"
#include "ft_overlap.hpp"
#include "ft_runtime.hpp"
#include "ft_wave.hpp"

#include <cfloat>
#include <cmath>

using namespace ft;

namespace {

constexpr int ROW_THREADS = 1024, ROW_WAVES = ROW_THREADS / 64;
constexpr int FIX = 42;     // fraction bits of a weight <= 1: 2^21 of them stay below 2^63
// values of a row that a workgroup keeps in LDS: the most, with what a finish keeps beside them, that its 160 KB hold
// (one workgroup a CU). With 4096 64 rows of 8000 go through scan and finish, top-k 64 with top-p 18.2 us against 10.8,
// neither 21.5 against 12.7, while 64 rows of 262144 with top-p take 91 against 97.
constexpr int LIST = 8192;
// values that are ranked by comparing all with all, four a lane of the wave that sums them: a row of 262144 with top-k
// 64 and top-p 18.5 us, by counting as longer lists 23.9; where nothing but min_p cuts, 9.4 against 8.1 (64 rows of 2000)
constexpr int FEW = 256;
constexpr int SEG = 64;     // values whose maximum the scan leaves
constexpr int MAX_SEGS = FT_SAMPLE_MAX_VOCAB / SEG;
constexpr int MAX_CHUNKS = FT_SAMPLE_MAX_VOCAB / 8192;

// e is counted in steps of 2^(1/8): BINS of them reach 2^-64 below a chunk's
// largest, beyond which 2^21 values weigh less than 2^-43 of it (more of them
// would not fit the finish's LDS). A value's e over its step's middle is in
// [2^-1/16, 2^1/16); a bin's word holds the number of values above bit 47 and
// below it their sum over OFFSET in units of 2^-FRAC (8192 times 0.107 * 2^35
// is far below 2^47). The chunk's largest value itself is in no bin: how often
// it occurs is counted apart, so that equal largest logits weigh the same whole
// number everywhere.
constexpr int BINS = 512, FRAC = 35;
constexpr double OFFSET = 0.9375;

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
    int given;  // HAS_*
};
enum { HAS_T = 1, HAS_K = 2, HAS_P = 4, HAS_M = 8 };

// A row's settings, with what is out of range brought into it.
struct Row {
    double inv_t, p, m, u;
    int k;
    bool greedy;
};

// The settings that are not given come as `u`, so that all are loaded at once.
__device__ __forceinline__ Row row_of(const SampleArgs& a, int64_t r) {
    const float t_in = a.temperature[r], p_in = a.top_p[r], m_in = a.min_p[r], u = a.u[r];
    const int k_in = a.top_k[r];
    const float t = a.given & HAS_T ? t_in : 1.0f, p = a.given & HAS_P ? p_in : 1.0f, m = a.given & HAS_M ? m_in : 0.0f;
    const int k = a.given & HAS_K ? k_in : 0;
    Row s;
    s.greedy = !(t > 0.0f);
    // T = inf as 2^200: exp of any two f32 values' distance over it is 1, and -inf over it is -inf
    s.inv_t = s.greedy ? 1.0 : fmax(1.0 / (double)t, 0x1p-200);
    s.k = k > 0 && k < a.V ? k : a.V;
    s.p = p < 1.0f ? fmax((double)p, 0.0) : 1.0;  // NaN: off
    s.m = m > 0.0f ? fmin((double)m, 1.0) : 0.0;  // NaN: off
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

// What a workgroup that finishes a row keeps in LDS.
struct RowLds {
    uint64_t w[1024];
    uint32_t n[1024];
    double part[ROW_WAVES];
    int parti[ROW_WAVES];
    int pick;
    uint32_t key_hi, key_lo;  // init_range
    double at, at_w;
    int at_n;
    float v[LIST];  // values taken from the row, by rising index
    int i[LIST];
};

template <int TYPE>
__device__ __forceinline__ const void* row_at(const SampleArgs& a, int64_t r) {
    return static_cast<const char*>(a.logits) + r * a.stride * (TYPE == FT_TYPE_F32 ? 4 : 2);
}

// The values that a step of a row's work goes through, by rising index.
template <int TYPE>
struct WholeRow {
    const void* row;
    int V;
    __device__ __forceinline__ int size() const { return V; }
    __device__ __forceinline__ float value(int at) const { return logit<TYPE>(row, at); }
    __device__ __forceinline__ int index(int at) const { return at; }
};
struct List {
    const float* v;
    const int* i;
    int n;
    __device__ __forceinline__ int size() const { return n; }
    __device__ __forceinline__ float value(int at) const { return v[at]; }
    __device__ __forceinline__ int index(int at) const { return i[at]; }
};

// Where the order is cut: kept are all keys above `key` and the values equal to it up to index `end`.
struct Cut {
    uint32_t key;
    int ties, of;   // of the `of` values equal to key the first `ties` are kept
    int end;        // index of the last of these
    double before;  // sum of e above key
    double e;       // one of key's
};

// First place of the order at which the count (by_count) or the sum reaches
// the target, among the source's keys in [lo, hi]; base_n values of sum base_w
// are ahead of them. The range is counted into up to 1024 equal pieces, the
// piece that reaches the target is the next range, until a piece is one key. A
// piece's weights are summed as whole numbers relative to its upper edge: each
// is off by at most half a unit, 2^-43 of the edge, so a sum over n values by
// n 2^-43 of the largest's weight (a list's 9.3e-10, a whole row's 2.4e-7).
template <typename SRC>
__device__ Cut find_cut(const SRC& src, uint32_t lo, uint32_t hi, int base_n, double base_w, const Row& s, float M,
                        bool by_count, bool sums, double target, RowLds& l) {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, size = src.size();
    for (;;) {
        const uint32_t width = hi - lo;
        const int shift = width < 1024u ? 0 : 22 - __clz(width);
        l.n[t] = 0;
        l.w[t] = 0;
        if (t == 0) l.pick = 1024;
        __syncthreads();
        for (int i = t; i < size; i += ROW_THREADS) {
            const float v = src.value(i);
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
        const int scan_n = wave_scan(own_n);
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
        if (l.pick == 1024) {  // fewer values than asked for, or a rounding below the target: the last that holds any
            __syncthreads();
            if (t == 0) l.pick = -1;
            __syncthreads();
            if (own_n) atomicMax(&l.pick, t);
            __syncthreads();
        }
        const int b = l.pick;
        if (b < 0) return Cut{0, 1, 1, 0x7FFFFFFF, 0.0, 0.0};  // no value in the range: no cut
        if (t == b) {
            l.at = prev_w;
            l.at_n = prev_n;
            l.at_w = own_w;
        }
        __syncthreads();
        base_w = l.at;
        base_n = l.at_n;
        const int here = (int)l.n[b];
        hi -= (uint32_t)b << shift;
        if (here == 1 && shift) {  // the only value of its piece: kept, and all above the piece's end
            const uint32_t span = (1u << shift) - 1;
            const Cut c{hi - lo > span ? hi - span : lo, 1, 1, 0x7FFFFFFF, base_w, l.at_w};
            __syncthreads();
            return c;
        }
        if (shift == 0) {
            Cut c{hi, here, here, 0x7FFFFFFF, base_w, weight(of_key(hi), M, s.inv_t)};
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

// The index of the last value equal to the cut's key that is kept.
template <typename SRC>
__device__ void find_end(const SRC& src, Cut& cut, RowLds& l) {
    if (cut.ties >= cut.of) return;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, size = src.size();
    int seen = 0;
    for (int base = 0; base < size && seen < cut.ties; base += ROW_THREADS) {
        const float v = base + t < size ? src.value(base + t) : -INFINITY;
        const bool tie = v > -INFINITY && key_of(v) == cut.key;
        const uint64_t set = __ballot(tie);
        if (lane == 0) l.parti[wave] = __popcll(set);
        __syncthreads();
        int rank = seen;
        for (int w = 0; w < ROW_WAVES; ++w) {
            if (w < wave) rank += l.parti[w];
            seen += l.parti[w];
        }
        if (tie && rank + wave_below(set) + 1 == cut.ties) l.pick = src.index(base + t);
        __syncthreads();
    }
    cut.end = l.pick;
    __syncthreads();
}

// e of a value if it is kept, else 0.
__device__ __forceinline__ double kept(float v, int index, const Cut& cut, const Row& s, float M) {
    if (!(v > -INFINITY)) return 0.0;
    const uint32_t k = key_of(v);
    if (k < cut.key || (k == cut.key && index > cut.end)) return 0.0;
    const double e = weight(v, M, s.inv_t);
    return e >= s.m ? e : 0.0;
}

// Place of the first sum that passes `goal`, `base` before them, and the sum
// before it; where none does the last place that adds anything. A wave's work:
// v, its lanes' sums in order. -1: none adds anything.
__device__ __forceinline__ int pick_lane(double own, double base, double goal, double* before, bool* passed,
                                         double* after) {
    const double scan = wave_scan(own), cum = base + scan;
    const uint64_t over = __ballot(own > 0.0 && cum > goal), any = __ballot(own > 0.0);
    *after = wave_lane(cum, 63);
    *passed = over != 0;
    if (!any) return -1;
    const int at = over ? __ffsll((unsigned long long)over) - 1 : 63 - __clzll((long long)any);
    *before = at ? wave_lane(cum, at - 1) : base;
    return at;
}

// The draw among the source's places [lo, lo + len), ahead of which the kept
// sum is `before`; total < 0: [lo, lo + len) is all, and its sum the total.
// Sixteenths of the range are summed, the one that holds the token is the next
// range, down to a wave's 64 places.
template <typename SRC>
__device__ void draw(const SampleArgs& a, int64_t r, const SRC& src, int lo, int len, double before, double total,
                     const Cut& cut, const Row& s, float M, RowLds& l) {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    while (len > 64) {
        const int piece = ((len + ROW_WAVES - 1) / ROW_WAVES + 63) / 64 * 64;
        const int b0 = lo + wave * piece, b1 = min(lo + len, b0 + piece);
        double z = 0.0;
        for (int i = b0 + lane; i < b1; i += 64) z += kept(src.value(i), src.index(i), cut, s, M);
        z = wave_sum(z);
        if (lane == 0) l.part[wave] = z;
        __syncthreads();
        if (total < 0.0) {
            total = 0.0;
            for (int i = 0; i < ROW_WAVES; ++i) total += l.part[i];
        }
        double here = before, after;
        bool passed;
        const double part = lane < ROW_WAVES ? l.part[lane] : 0.0;
        const int at = max(0, pick_lane(part, before, s.u * total, &here, &passed, &after));
        before = here;
        len = min(piece, len - at * piece);
        lo += at * piece;
        __syncthreads();
    }
    if (wave) return;
    const int i = lo + lane;
    const double e = lane < len ? kept(src.value(i), src.index(i), cut, s, M) : 0.0;
    const double cum = wave_scan(e);
    if (total < 0.0) total = wave_lane(cum, 63);
    const uint64_t over = __ballot(e > 0.0 && before + cum > s.u * total), any = __ballot(e > 0.0);
    const int at = over ? __ffsll((unsigned long long)over) - 1 : 63 - __clzll((long long)any);
    if (lane == at) {
        a.tokens[r] = src.index(i);
        if (a.logprobs) a.logprobs[r] = (float)log(e / total);
    }
}

// Sum over the workgroup, the same in every thread.
__device__ __forceinline__ double block_sum(double z, RowLds& l) {
    z = wave_sum(z);
    if ((threadIdx.x & 63) == 0) l.part[threadIdx.x >> 6] = z;
    __syncthreads();
    z = 0.0;
    for (int i = 0; i < ROW_WAVES; ++i) z += l.part[i];
    __syncthreads();
    return z;
}
__device__ __forceinline__ void answer(const SampleArgs& a, int64_t r, int token, float logprob) {
    if (threadIdx.x == 0) {
        a.tokens[r] = token;
        if (a.logprobs) a.logprobs[r] = logprob;
    }
}

// The largest and the smallest value above -inf over the workgroup (-inf and
// anything where there is none). init_range before, and a barrier between.
__device__ __forceinline__ void init_range(RowLds& l) {
    if (threadIdx.x == 0) {
        l.key_hi = 0;
        l.key_lo = 0xFFFFFFFFu;
    }
}
__device__ __forceinline__ void block_range(float& hi, float& lo, RowLds& l) {
    hi = wave_max(hi);
    lo = -wave_max(-lo);
    if ((threadIdx.x & 63) == 0 && hi > -INFINITY) {
        atomicMax(&l.key_hi, key_of(hi));
        atomicMin(&l.key_lo, key_of(lo));
    }
    __syncthreads();
    hi = l.key_hi ? of_key(l.key_hi) : -INFINITY;
    lo = of_key(l.key_lo);
    __syncthreads();
}

// A row from all of its values, streamed: right for every case, with any
// number of kept or equal values. M > -inf.
template <int TYPE>
__device__ __attribute__((noinline)) void sample_streaming(const SampleArgs& a, int64_t r, const Row& s, float M,
                                                           RowLds& l) {
    const WholeRow<TYPE> src{row_at<TYPE>(a, r), a.V};
    const int t = threadIdx.x;
    const uint32_t hi = key_of(M), lo = M == INFINITY ? hi : key_of(-INFINITY) + 1;
    const bool by_p = s.p < 1.0;
    Cut cut{0, 1, 1, 0x7FFFFFFF, 0.0, 0.0};
    double z = 0.0;
    if (s.k < a.V) {
        cut = find_cut(src, lo, hi, 0, 0.0, s, M, true, by_p, (double)s.k, l);
        z = cut.before + cut.ties * cut.e;
    } else if (by_p) {
        for (int i = t; i < a.V; i += ROW_THREADS) {
            const float v = src.value(i);
            if (v > -INFINITY) z += weight(v, M, s.inv_t);
        }
        z = block_sum(z, l);
    }
    if (by_p) {
        const Cut c = find_cut(src, lo, hi, 0, 0.0, s, M, false, true, s.p * z, l);
        if (c.key > cut.key || (c.key == cut.key && c.ties < cut.ties)) cut = c;
    }
    find_end(src, cut, l);
    draw(a, r, src, 0, a.V, 0.0, -1.0, cut, s, M, l);
}

// A row whose kept values are all in the list, of at most FEW values: each is
// ranked by comparing it with all others; a wave then sums e over the ranks for
// the cuts and over the indices for the draw, four places a lane. rest: the sum
// of e outside the list that top_p is also a share of (without top-k).
__device__ __forceinline__ void sample_few(const SampleArgs& a, int64_t r, int n, double rest, const Row& s, float M,
                                           RowLds& l) {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, at = t & (FEW - 1);
    const float v = at < n ? l.v[at] : -INFINITY;
    const bool ok = v > -INFINITY;
    const uint64_t key = ((uint64_t)(ok ? key_of(v) : 0u) << 32) | (uint32_t)~at;
    if (t < FEW) {
        l.w[t] = key;
        l.n[t] = 0;
    }
    __syncthreads();
    int ahead = 0;
    const int j0 = wave / (FEW / 64) * (FEW * FEW / ROW_THREADS);  // a quarter of the others
#pragma unroll 8
    for (int j = 0; j < FEW * FEW / ROW_THREADS; ++j) ahead += l.w[j0 + j] > key;
    atomicAdd(&l.n[at], (uint32_t)ahead);
    __syncthreads();
    double* by_rank = reinterpret_cast<double*>(l.w);
    double* by_index = by_rank + FEW;
    if (t < FEW) {
        const double e = ok ? weight(v, M, s.inv_t) : 0.0;
        by_rank[l.n[t]] = e;
        by_index[t] = e;
    }
    __syncthreads();
    if (wave) return;
    double e[4], z = 0.0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        e[i] = 4 * lane + i < s.k ? by_rank[4 * lane + i] : 0.0;
        z += e[i];
    }
    const double scan = wave_scan(z), goal = s.p * (wave_lane(scan, 63) + rest);
    double cum = wave_lane_before(scan, 0.0);
    int kept_n = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // cum: the sum before this one
        kept_n += e[i] > 0.0 && e[i] >= s.m && (4 * lane + i == 0 || s.p >= 1.0 || cum < goal);
        cum += e[i];
    }
    kept_n = wave_sum(kept_n);
    double own = 0.0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        e[i] = (int)l.n[4 * lane + i] < kept_n ? by_index[4 * lane + i] : 0.0;
        own += e[i];
    }
    const double total = wave_sum(own), draw = s.u * total;
    double before, after;
    bool passed;
    const int p = pick_lane(own, 0.0, draw, &before, &passed, &after);
    if (lane != p) return;
    int i = -1;
    double had = 0.0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (e[j] > 0.0 && (i < 0 || !(before > draw))) {  // to the first that passes, or the last
            i = j;
            had = e[j];
        }
        before += e[j];
    }
    a.tokens[r] = l.i[4 * lane + i];
    if (a.logprobs) a.logprobs[r] = (float)log(had / total);
}

// A row whose kept values are all in the list.
__device__ __forceinline__ void sample_list(const SampleArgs& a, int64_t r, int n, double rest, const Row& s, float M,
                                            RowLds& l) {
    if (n <= FEW) return sample_few(a, r, n, rest, s, M, l);
    const int t = threadIdx.x;
    const List list{l.v, l.i, n};
    init_range(l);
    float x = -INFINITY, y = INFINITY;
    __syncthreads();
    for (int i = t; i < n; i += ROW_THREADS)
        if (l.v[i] > -INFINITY) {
            x = fmaxf(x, l.v[i]);
            y = fminf(y, l.v[i]);
        }
    block_range(x, y, l);
    const uint32_t hi = key_of(x), lo = x == INFINITY ? hi : key_of(y);
    const bool by_k = s.k < n, by_p = s.p < 1.0;
    Cut cut{0, 1, 1, 0x7FFFFFFF, 0.0, 0.0};
    double z = 0.0;
    if (by_p && !by_k) {
        for (int i = t; i < n; i += ROW_THREADS)
            if (l.v[i] > -INFINITY) z += weight(l.v[i], M, s.inv_t);
        z = block_sum(z, l) + rest;
    }
#pragma unroll 1
    for (int step = by_k ? 0 : 1; step < (by_p ? 2 : 1); ++step) {
        const Cut c = find_cut(list, lo, hi, 0, 0.0, s, M, step == 0, by_p, step == 0 ? (double)s.k : s.p * z, l);
        if (step == 0) z = c.before + c.ties * c.e;
        if (c.key > cut.key || (c.key == cut.key && c.ties < cut.ties)) cut = c;
    }
    find_end(list, cut, l);
    draw(a, r, list, 0, n, 0.0, -1.0, cut, s, M, l);
}

// The sum of the waves' counts before this wave's, and of all.
__device__ __forceinline__ void waves_before(const int* counts, int& before, int& all) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int own = lane < ROW_WAVES ? counts[lane] : 0, scan = wave_scan(own);
    before = wave_lane(scan - own, wave);
    all = wave_lane(scan, 63);
}

// A value that at least k of the row's values reach, from the maxima of parts
// of it (lowest: the smallest of these above -inf, or less): k parts have one
// each. -inf if fewer than k parts hold any. Counted in 256 pieces of the key
// range, and again in the piece that reaches k while that holds many more, or
// more than `most`: a range that goes below 0 has pieces of whole binades. l.n
// is 0 on entry.
template <typename PARTS>
__device__ __forceinline__ float reached_by(int k, int most, const PARTS& parts, float lowest, float M, RowLds& l) {
    const int lane = threadIdx.x & 63;
    uint32_t hi = key_of(M), lo = key_of(lowest);
    int base = 0;
#pragma unroll 1
    for (uint32_t* counts = l.n;; counts += 256) {
        const uint32_t width = hi - lo;
        const int shift = width < 256u ? 0 : 24 - __clz(width);
        parts.each([&](float m, int) {
            const uint32_t q = key_of(m);
            if (m > -INFINITY && q >= lo && q <= hi) atomicAdd(&counts[(hi - q) >> shift], 1u);
        });
        __syncthreads();
        int own[4], sum = 0;  // bins 4 lane ..
#pragma unroll
        for (int i = 0; i < 4; ++i) sum += own[i] = (int)counts[4 * lane + i];
        const int scan = base + wave_scan(sum);
        const uint64_t set = __ballot(scan >= k);
        if (!set) return -INFINITY;
        const int at = __ffsll((unsigned long long)set) - 1;
        int b = 0, before = scan - sum;
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (b == i && before + own[i] < k) {
                before += own[i];
                ++b;
            }
        const int here = b == 0 ? own[0] : b == 1 ? own[1] : b == 2 ? own[2] : own[3];
        b = 4 * at + wave_lane(b, at);
        base = wave_lane(before, at);
        const int through = base + wave_lane(here, at);
        const uint64_t under = (((uint64_t)b + 1) << shift) - 1;
        lo = under >= width ? lo : hi - (uint32_t)under;
        hi -= (uint32_t)b << shift;
        if (shift == 0 || through <= min(k + k / 2 + 32, most) || counts == l.n + 768) return of_key(lo);
    }
}

// A thread's part of a row, by its maximum.
struct Part {
    float max;
    template <typename F>
    __device__ __forceinline__ void each(const F& fn) const {
        fn(max, 0);
    }
};

// A little less than the value whose e is x: what is below has less for sure.
__device__ __forceinline__ float value_below(double x, const Row& s, float M) {
    const double d = log(x) / s.inv_t, v = (double)M + d - 1e-6 * (fabs((double)M) + fabs(d));
    return v > -(double)FLT_MAX ? (float)v : -INFINITY;  // also where inf meets -inf
}

// Rows of at most LIST values, one launch: in registers, a run of 512 to a
// wave; those that may be kept go into the list. Bound by the chain of steps of
// one workgroup, most of them the instructions' first fetch and a barrier: 64
// rows of 8000 take 10.9 us with top-k 64 and top-p, 22.7 with top-p, 12.9 with
// neither, where scan and finish take 19.5, 25.9 and 21.5; a row of 2000 9.2,
// 11.7 and 8.5.
template <int TYPE>
__global__ __launch_bounds__(ROW_THREADS) void k_sample_rows(SampleArgs a) {
    __shared__ RowLds l;
    constexpr int N = LIST / ROW_THREADS;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, first = wave * 64 * N + lane;
    const int64_t r = blockIdx.x;
    const void* row = row_at<TYPE>(a, r);
    float v[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const int i = first + 64 * j;
        const float x = logit<TYPE>(row, i < a.V ? i : 0);
        v[j] = i < a.V && x > -INFINITY ? x : -INFINITY;  // NaN too
    }
    init_range(l);
    if (t == 0) l.pick = 0x7FFFFFFF;
    l.n[t] = 0;
    const Row s = row_of(a, r);
    __syncthreads();
    float top = -INFINITY;  // of the thread's
#pragma unroll
    for (int j = 0; j < N; ++j) top = fmaxf(top, v[j]);
    float M = top, lowest = top > -INFINITY ? top : INFINITY;
    block_range(M, lowest, l);
    if (M == -INFINITY) return answer(a, r, -1, NAN);
    if (s.greedy) {
#pragma unroll
        for (int j = N - 1; j >= 0; --j)
            if (v[j] == M) atomicMin(&l.pick, first + 64 * j);
        __syncthreads();
        return answer(a, r, l.pick, 0.0f);
    }
    const bool by_k = s.k < a.V, by_p = s.p < 1.0;
    float from = -INFINITY;
    if (by_k && s.k <= ROW_THREADS) from = reached_by(s.k, ROW_THREADS, Part{top}, lowest, M, l);
    if (by_p && !by_k) {  // those of less than (1 - p) z / V are together less than the (1 - p) z that top_p leaves out
        double z = 0.0;
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (v[j] > -INFINITY) z += weight(v[j], M, s.inv_t);
        from = value_below((1.0 - s.p) * (1.0 - 1e-9) * block_sum(z, l) / a.V, s, M);
    }
    if (s.m > 0.0 && !by_p) from = fmaxf(from, value_below(s.m, s, M));
    from = fmaxf(from, -FLT_MAX);
    double rest = 0.0;
    int got = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        got += __popcll(__ballot(v[j] >= from));
        if (by_p && !by_k && v[j] > -INFINITY && v[j] < from) rest += weight(v[j], M, s.inv_t);
    }
    if (lane == 0) l.parti[wave] = got;
    __syncthreads();
    int at, n;
    waves_before(l.parti, at, n);
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const uint64_t set = __ballot(v[j] >= from);
        const int to = at + wave_below(set);
        if (v[j] >= from) {
            l.v[to] = v[j];
            l.i[to] = first + 64 * j;
        }
        at += __popcll(set);
    }
    rest = block_sum(rest, l);  // its barriers also close the list
    sample_list(a, r, n, rest, s, M, l);
}

// ---- longer rows: a scan by many workgroups, then one that finishes the row ----

// What the scan says of a chunk (a workgroup's values).
struct Chunk {
    double sum;    // of the binned e, over the middle of the largest's step
    double far;    // of e further than the bins below the largest, over the largest's
    float max;
    uint32_t top;  // how many values equal it
};

// The scan's results, per row: every segment's maximum, the chunks, their bins.
struct Scan {
    char* base;
    int64_t row_bytes;
    int chunk, chunks, segs;
    int most_k;        // the largest top-k that the segments' maxima decide
    int most_reached;  // and how many of them the value that bounds it may leave
    __host__ __device__ static int64_t up16(int64_t v) { return (v + 15) / 16 * 16; }
    __host__ __device__ int64_t at_info() const { return up16((int64_t)segs * 4); }
    __host__ __device__ int64_t at_bins() const { return at_info() + up16((int64_t)chunks * sizeof(Chunk)); }
    __host__ __device__ int64_t bytes() const { return at_bins() + (int64_t)chunks * BINS * 8; }
    __device__ float* seg(int i) const { return reinterpret_cast<float*>(base + i * row_bytes); }
    __device__ Chunk* info(int i) const { return reinterpret_cast<Chunk*>(base + i * row_bytes + at_info()); }
    __device__ uint64_t* bins(int i) const { return reinterpret_cast<uint64_t*>(base + i * row_bytes + at_bins()); }
};

// Whether a row is decided by its segments' maxima: the largest value alone,
// or a top-k that they bound by a list that fits (else the scan fills the bins).
__device__ __forceinline__ bool by_maxima(const Row& s, const Scan& w) { return s.greedy || s.k <= w.most_k; }

// A value's place in steps of e (per_unit: the step of 2^(1/8) per unit of the
// logit), and its step, the nearest whole number: by the sum with MAGIC, whose
// last bit is 1; further out, where the steps of f32 are many of these, by rint.
constexpr double MAGIC = 0x1.8p52, NEAR = 0x1p50;
__device__ __forceinline__ double per_unit(const Row& s) { return s.inv_t * (8.0 * 1.4426950408889634074); }
__device__ __forceinline__ double step_of(float v, double unit) {
    const double y = (double)v * unit;
    return fabs(y) < NEAR ? fma((double)v, unit, MAGIC) - MAGIC : rint(y);
}
// Steps below the largest's (g: step_of(M)); BINS: that or more.
__device__ __forceinline__ int bin_of(float v, float M, double g, double unit) {
    if (v == M) return 0;
    const double d = g - step_of(v, unit);
    return d < (double)BINS ? (int)d : BINS;
}
// The largest's place over the middle of its step, in steps.
__device__ __forceinline__ double over_step(float M, double g, double unit) {
    const double d = fma((double)M, unit, -g);
    return fabs(d) <= 0.5 ? d : 0.0;  // inf - inf: 0
}
__device__ __forceinline__ double bin_sum(uint64_t word) {
    return (double)(uint32_t)(word >> 47) * OFFSET +
           (double)(word & ((1ull << 47) - 1)) * (1.0 / (double)(1ull << FRAC));
}

// Four values from an aligned place of a row.
template <int TYPE>
__device__ __forceinline__ void load4(const void* row, int i, float v[4]) {
    if constexpr (TYPE == FT_TYPE_F32) {
        const float4 x = *reinterpret_cast<const float4*>(static_cast<const float*>(row) + i);
        v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
    } else {
        const uint2 x = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(row) + i);
        const uint16_t b[4] = {(uint16_t)x.x, (uint16_t)(x.x >> 16), (uint16_t)x.y, (uint16_t)(x.y >> 16)};
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = TYPE == FT_TYPE_F16 ? h2f(b[e]) : __uint_as_float((uint32_t)b[e] << 16);
    }
}
// From any place; -inf past the end.
template <int TYPE>
__device__ __forceinline__ void load4(const void* row, int i, int V, bool vec, float v[4]) {
    if (vec && i + 4 <= V) return load4<TYPE>(row, i, v);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = i + e < V ? logit<TYPE>(row, i + e) : -INFINITY;
}
template <int TYPE>
__device__ __forceinline__ bool vec_row(const void* row) {
    return (reinterpret_cast<uintptr_t>(row) & (TYPE == FT_TYPE_F32 ? 15 : 7)) == 0;
}

// Workgroup (c, row): chunk c of the row in registers, VECS times four values
// a thread; one pass over memory. With bins to fill it is bound by instructions,
// about 33 a value, most in f64, and an LDS atomic: 256 rows of 262144 take 72 us
// (3.7 TB/s), 64 rows 25, one 6.2. Where the segments' maxima decide, by memory:
// 64 rows 11.7 us (5.7 TB/s, in part from the caches), one 3.2.
template <int TYPE, int VECS>
__global__ __launch_bounds__(1024) void k_sample_scan(SampleArgs a, Scan w, int64_t row0) {
    __shared__ uint64_t bins[BINS];
    __shared__ double part[16], part2[16];
    __shared__ uint32_t top_n;
    const int t = threadIdx.x, T = blockDim.x, lane = t & 63, wave = t >> 6, waves = T >> 6, c = blockIdx.x;
    const int64_t r = row0 + blockIdx.y;
    const void* row = row_at<TYPE>(a, r);
    const bool vec = vec_row<TYPE>(row);
    float v[VECS][4];
    if (vec && (c + 1) * w.chunk <= a.V) {  // one branch for all loads: a branch at each would wait for each
#pragma unroll
        for (int i = 0; i < VECS; ++i) load4<TYPE>(row, c * w.chunk + (i * T + t) * 4, v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < VECS; ++i) load4<TYPE>(row, c * w.chunk + (i * T + t) * 4, a.V, vec, v[i]);
    }
    const Row s = row_of(a, r);
    float m = -INFINITY;
    float* seg = w.seg(blockIdx.y);
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
        const float x = row_max16(fmaxf(fmaxf(fmaxf(v[i][0], v[i][1]), fmaxf(v[i][2], v[i][3])), -INFINITY));
        const int at = (c * w.chunk + (i * T + t) * 4) / SEG;
        if ((lane & 15) == 0 && at < w.segs) seg[at] = x;
        m = fmaxf(m, x);
    }
    if (by_maxima(s, w)) return;
    m = wave_max(m);
    if (lane == 0) part[wave] = m;
    for (int b = t; b < BINS; b += T) bins[b] = 0;
    if (t == 0) top_n = 0;
    __syncthreads();
    for (int i = 0; i < waves; ++i) m = fmaxf(m, (float)part[i]);
    __syncthreads();
    const double unit = per_unit(s), g = step_of(m, unit);
    double far = 0.0;
    // the bins hold the values from `low` on: the smallest on one of the first BINS steps
    float low = m;
    if (fabs(g) < NEAR) {
        low = (float)fmax((g - BINS + 0.5) / unit, -(double)FLT_MAX);
        if (step_of(low, unit) <= g - BINS) low = of_key(key_of(low) + 1);
        const float less = of_key(key_of(low) - 1);
        if (less >= -FLT_MAX && step_of(less, unit) > g - BINS) low = less;
    }
    const float under = of_key(key_of(low) - 1);  // what is up to here is beyond them
    bool beyond = false;
    int top = 0;
#pragma unroll
    for (int i = 0; i < VECS; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) top += __popcll(__ballot(v[i][e] == m));
    // a value's word: (2^(q / 8) - OFFSET) 2^FRAC by the series to q^5 (|q| <= 1/2: what is left is under a third of a
    // unit), whose sum with 2^52 has it in its low half, as the sum with MAGIC has the step: conversions of f64 are
    // slow. The constants are kept in scalar registers: as literals each would cost two moves per use.
    const double L = 0.08664339756999316, U = (double)(1ull << FRAC);  // ln 2 / 8
    const double c0 = scalar((1.0 - OFFSET) * U + 0x1p52), c1 = scalar(L * U), c2 = scalar(L * L / 2 * U),
                 c3 = scalar(L * L * L / 6 * U), c4 = scalar(L * L * L * L / 24 * U),
                 c5 = scalar(L * L * L * L * L / 120 * U);
    const int g_low = (int)__double_as_longlong(g + MAGIC);
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
        uint32_t word[4];
        int bin[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const double x = v[i][e], n = fma(x, unit, MAGIC), q = fma(x, unit, -(n - MAGIC));
            word[e] = (uint32_t)__double_as_longlong(
                fma(fma(fma(fma(fma(q, c5, c4), q, c3), q, c2), q, c1), q, c0));
            bin[e] = g_low - (int)__double_as_longlong(n);
            asm("" : "+v"(word[e]), "+v"(bin[e]));  // four chains side by side, not each under its mask
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float x = v[i][e];
            if (x >= low && x < m) atomicAdd((unsigned long long*)&bins[bin[e]], (1ull << 47) + word[e]);
            beyond |= x == __builtin_amdgcn_fmed3f(x, -FLT_MAX, under);
        }
    }
    if (__ballot(beyond)) {  // far below the largest: few in most rows, from the caches again
#pragma unroll 1
        for (int i = 0; i < VECS; ++i) {
            float x[4];
            load4<TYPE>(row, c * w.chunk + (i * T + t) * 4, a.V, vec, x);
            for (int e = 0; e < 4; ++e)
                if (x[e] < low && x[e] > -INFINITY) far += weight(x[e], m, s.inv_t);
        }
    }
    if (lane == 0) atomicAdd(&top_n, (uint32_t)top);
    __syncthreads();
    // the chunk's sums, its bins in their order
    double z = 0.0;
    uint64_t* out = w.bins(blockIdx.y) + (int64_t)c * BINS;
    double scale = exp2(t * -0.125);
    for (int b = t; b < BINS; b += T) {
        const uint64_t word = bins[b];
        out[b] = word;
        z += bin_sum(word) * scale;
        scale = ldexp(scale, -T / 8);
    }
    z = wave_sum(z);
    far = wave_sum(far);
    if (lane == 0) {
        part[wave] = z;
        part2[wave] = far;
    }
    __syncthreads();
    if (t == 0) {
        Chunk k{0.0, 0.0, m, m > -INFINITY ? top_n : 0};
        for (int i = 0; i < waves; ++i) {
            k.sum += part[i];
            k.far += part2[i];
        }
        w.info(blockIdx.y)[c] = k;
    }
}

// What k_sample_finish keeps beside RowLds.
struct FinishLds {
    double cum_w[BINS], scale[BINS];
    int cum_n[BINS];
    double sums[MAX_CHUNKS], top_w[MAX_CHUNKS];  // the chunks' kept e, and that of their largest values
    uint64_t top_f[MAX_CHUNKS];                  // one such e as a bin holds it
    uint32_t top[MAX_CHUNKS];                    // how many these are
    int off[MAX_CHUNKS];                         // and their bin
    uint16_t open[MAX_SEGS];
    int cut_lo, cut_hi;
};

constexpr int SEGS_HELD = 4;  // segments' maxima that a thread keeps

// A wave's segments: a run of `per`, 64 at a time; the first SEGS_HELD times are in registers.
struct Segs {
    const float* p;
    int segs, per, s0;
    float held[SEGS_HELD];
    __device__ __forceinline__ void load(const float* seg, int n) {
        p = seg;
        segs = n;
        per = ((n + ROW_WAVES - 1) / ROW_WAVES + 63) / 64 * 64;
        s0 = (threadIdx.x >> 6) * per + (threadIdx.x & 63);
#pragma unroll
        for (int j = 0; j < SEGS_HELD; ++j) held[j] = j * 64 < per && s0 + j * 64 < segs ? p[s0 + j * 64] : -INFINITY;
    }
    // fn(segment's maximum (-inf past the end), its number) for each of the thread's, all of a wave's lanes together
    template <typename F>
    __device__ __forceinline__ void each(const F& fn) const {
#pragma unroll
        for (int j = 0; j < SEGS_HELD; ++j)
            if (j * 64 < per) fn(held[j], s0 + j * 64);
        for (int j = SEGS_HELD; j * 64 < per; ++j) fn(s0 + j * 64 < segs ? p[s0 + j * 64] : -INFINITY, s0 + j * 64);
    }
};

// The row's values in [from, to], by rising index, into the list, from the
// segments whose maximum is at least `from`. Returns how many there are; more
// than LIST: not all were taken.
template <int TYPE>
__device__ __forceinline__ int gather(const void* row, int V, const Segs& segs, float from, float to, RowLds& l,
                                      FinishLds& f) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const bool vec = vec_row<TYPE>(row);
    from = fmaxf(from, -FLT_MAX);
    // the open segments' numbers, in order
    int mine = 0;
    segs.each([&](float m, int) { mine += __popcll(__ballot(m >= from)); });
    if (lane == 0) l.parti[wave] = mine;
    __syncthreads();
    int at, count;
    waves_before(l.parti, at, count);
    segs.each([&](float m, int k) {
        const bool in = m >= from;
        const uint64_t set = __ballot(in);
        if (in) f.open[at + wave_below(set)] = (uint16_t)k;
        at += __popcll(set);
    });
    __syncthreads();
    // rounds of up to 8 times 4 segments a wave, the next round's loads ahead: the waves' runs of a round lie one after
    // the other
    float ahead[8][4];
    int ahead_i[8];
    const auto load = [&](int base) {
        const int now = min(count - base, ROW_WAVES * 32), per = (now + ROW_WAVES * 4 - 1) / (ROW_WAVES * 4);
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            if (u >= per) break;
            const int k = (wave * per + u) * 4 + (lane >> 4);
            ahead_i[u] = k < now ? f.open[base + k] * SEG + (lane & 15) * 4 : V;
            load4<TYPE>(row, ahead_i[u], V, vec, ahead[u]);
        }
        return per;
    };
    int n = 0, next = load(0);
    for (int base = 0; base < count && n <= LIST; base += ROW_WAVES * 32) {
        float v[8][4];
        int first[8];
        const int per = next;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            if (u >= per) break;
            first[u] = ahead_i[u];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[u][e] = ahead[u][e];
        }
        if (base + ROW_WAVES * 32 < count) next = load(base + ROW_WAVES * 32);
        uint32_t mask = 0;  // bit 4 u + e
        int own[3] = {0, 0, 0};  // how many by u, 10 bits each
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            if (u >= per) break;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                mask |= v[u][e] == __builtin_amdgcn_fmed3f(v[u][e], from, to) ? 1u << (4 * u + e) : 0u;
            own[u / 3] |= __popc(mask >> (4 * u)) << (10 * (u % 3));
        }
        int lower[3], all[3], got = 0;
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            const int scan = wave_scan(own[i]);
            lower[i] = scan - own[i];
            all[i] = wave_lane(scan, 63);
            got += (all[i] & 1023) + (all[i] >> 10 & 1023) + (all[i] >> 20);
        }
        __syncthreads();  // the last round's counts are read
        if (lane == 0) l.parti[wave] = got;
        __syncthreads();
        int put, more;
        waves_before(l.parti, put, more);
        put += n;
        n += more;
        if (got == 0) continue;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            if (u >= per) break;
            int at = put + (lower[u / 3] >> (10 * (u % 3)) & 1023);
            put += all[u / 3] >> (10 * (u % 3)) & 1023;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (mask >> (4 * u + e) & 1) {
                    if (at < LIST) {
                        l.v[at] = v[u][e];
                        l.i[at] = first[u] + e;
                    }
                    ++at;
                }
        }
    }
    __syncthreads();
    return n;
}

// The smallest value whose bin is at most b (b < BINS), found 64 keys at a time.
__device__ __forceinline__ float lowest_in(int b, float M, double g, double unit) {
    if (M == INFINITY) return M;
    const int lane = threadIdx.x & 63;
    uint32_t lo = key_of(-INFINITY) + 1, hi = key_of(M);  // hi is in; the answer is in [lo, hi]
    while (lo < hi) {
        const uint32_t step = (hi - lo) / 64 + 1;
        const uint64_t k = (uint64_t)lo + (uint64_t)lane * step;
        const bool in = k >= hi || bin_of(of_key((uint32_t)k), M, g, unit) <= b;
        const uint64_t set = __ballot(in);  // a run of lanes to the last, or none
        const int first = set ? __ffsll((unsigned long long)set) - 1 : 64;
        const uint64_t up = (uint64_t)lo + (uint64_t)first * step;
        if (first > 0) lo = lo + (uint32_t)(first - 1) * step + 1;
        if (up < hi) hi = (uint32_t)up;
        if (first == 0) break;
    }
    return of_key(hi);
}

// Sum of `n` values in LDS, the same in every wave.
__device__ __forceinline__ double sum_of(const double* v, int n) {
    double z = 0.0;
    for (int i = threadIdx.x & 63; i < n; i += 64) z += v[i];
    return wave_sum(z);
}

// The chunk that holds the token, among `n` kept sums; the same in every wave.
__device__ __forceinline__ int pick_chunk(const double* sums, int n, double u, double* before, double* total) {
    const int lane = threadIdx.x & 63;
    *total = sum_of(sums, n);
    double base = 0.0;
    int some = 0;
    bool passed = false;
    for (int i = 0; i < n && !passed; i += 64) {
        double here, after;
        const int at = pick_lane(i + lane < n ? sums[i + lane] : 0.0, base, u * *total, &here, &passed, &after);
        if (at >= 0) {
            some = i + at;
            *before = here;
        }
        base = after;
    }
    return some;
}

// How many of the n rising numbers are below x, found 64 places at a time.
__device__ __forceinline__ int run_end(const int* v, int n, int x) {
    const int lane = threadIdx.x & 63;
    int lo = 0, hi = n;  // the answer is in [lo, hi]
    while (lo < hi) {
        const int step = (hi - lo) / 64 + 1, at = lo + lane * step;
        const uint64_t below = __ballot(at < hi && v[at] < x);  // a run from lane 0, or none
        const int many = __popcll(below);
        hi = min(hi, lo + many * step);
        if (many) lo += (many - 1) * step + 1;
    }
    return lo;
}

// The rest of a row after the scan, by one workgroup:
//  - top_k up to Scan::most_k: the values that k segments' maxima reach are a
//    little more than k and contain the top k; they go into the list, which
//    decides alone.
//  - else the bins say on which step of e the order is cut. If all from there
//    up fit the list, it decides alone; if not, the list holds the steps on
//    which the cut lies, the bins what is above, and the token's chunk is read
//    again for the draw.
//  - where neither fits the list, the row is streamed: more than LIST values on
//    the step of the cut (equal ones, or a flat row: 262144 normal values of sd
//    1 put some 8750 on the step of top-p 0.9), top_k with top_p where more than LIST
//    reach top_k's step, a top_k by maxima that lie in an order (the largest in
//    few of the segments).
// Bound by the chain of one workgroup's steps (its 162 KB of LDS leave a CU one):
// about 4 us until the first data is there, then the list's making and its cuts.
// A row of 262144: 14.7 us with top-k 64 and top-p; 57 with top-p alone where
// the cut lies among thousands (64 rows 71, 256 rows 76 to 84), of which reading
// its open segments again is 25 to 36; streamed 0.3 to 1.4 ms, a row of 2^21 3
// to 10.
template <int TYPE>
__global__ __launch_bounds__(ROW_THREADS) void k_sample_finish(SampleArgs a, Scan w, int64_t row0) {
    __shared__ RowLds l;
    __shared__ FinishLds f;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, V = a.V, chunks = w.chunks;
    const int64_t r = row0 + blockIdx.x;
    Segs segs;
    segs.load(w.seg(blockIdx.x), w.segs);
    init_range(l);
    if (t == 0) l.pick = 0x7FFFFFFF;
    l.n[t] = 0;
    const Row s = row_of(a, r);
    __syncthreads();
    const void* row = row_at<TYPE>(a, r);
    float M = -INFINITY, lowest = INFINITY;
    segs.each([&](float m, int) {
        M = fmaxf(M, m);
        if (m > -INFINITY) lowest = fminf(lowest, m);
    });
    block_range(M, lowest, l);
    if (M == -INFINITY) return answer(a, r, -1, NAN);
    if (s.greedy) {
        segs.each([&](float m, int k) {
            if (m == M) atomicMin(&l.pick, k);
        });
        __syncthreads();
        if (wave) return;
        const int i = l.pick * SEG + lane;
        const uint64_t set = __ballot(i < V && logit<TYPE>(row, i) == M);
        return answer(a, r, l.pick * SEG + __ffsll((unsigned long long)set) - 1, 0.0f);
    }
    const bool by_k = s.k < V, by_p = s.p < 1.0;
    float from, to = INFINITY;
    int first = 0, last = BINS;  // the bins in the list
    bool all = true;             // the list holds all from the largest on
    bool too_many = false;       // for the list
    double rest = 0.0, goal = 0.0;
    const double unit = per_unit(s), g = step_of(M, unit), ref = over_step(M, g, unit);
    const uint64_t* bins = w.bins(blockIdx.x);
    if (by_maxima(s, w)) {
        from = reached_by(s.k, w.most_reached, segs, lowest, M, l);
        if (s.m > 0.0 && !by_p) from = fmaxf(from, value_below(s.m, s, M));  // without top_p no sum needs the others
    } else {
        double far = 0.0;
        for (int c = t; c < chunks; c += ROW_THREADS) {
            const Chunk k = w.info(blockIdx.x)[c];
            const bool some = k.max > -INFINITY;
            const double e = some ? weight(k.max, M, s.inv_t) : 0.0;
            const double below = k.max == M ? 0.0 : g - step_of(k.max, unit);  // of its step under the largest's
            f.off[c] = some ? bin_of(k.max, M, g, unit) : BINS;
            f.top[c] = k.top;
            const double over = fmax(e * exp2((f.off[c] + ref) * 0.125) - OFFSET, 0.0);
            f.top_f[c] = some && k.max < INFINITY && f.off[c] < BINS
                             ? (uint64_t)fma(over, (double)(1ull << FRAC), 0.5)
                             : 0;
            f.top_w[c] = k.top * e;
            f.sums[c] = e > 0.0 ? f.top_w[c] + k.far * e + k.sum * exp2((below + ref) * -0.125) : 0.0;
            far += k.far * e;
        }
        __syncthreads();
        if (!by_k && !by_p && s.m == 0.0) {
            double before, total;
            const int c = pick_chunk(f.sums, chunks, s.u, &before, &total);
            return draw(a, r, WholeRow<TYPE>{row, V}, c * w.chunk, min(w.chunk, V - c * w.chunk), before, total,
                        Cut{0, 1, 1, 0x7FFFFFFF, 0.0, 0.0}, s, M, l);
        }
        // the chunks' bins as the row's: whole numbers, in any order
        {
            const int b = t & (BINS - 1);
            uint64_t frac = 0;
            uint32_t n = 0;
#pragma unroll 8
            for (int c = t / BINS; c < chunks; c += ROW_THREADS / BINS) {
                const int j = b - f.off[c];
                const uint64_t x = j >= 0 ? bins[(int64_t)c * BINS + j] : 0;
                n += (uint32_t)(x >> 47) + (j == 0 ? f.top[c] : 0);
                frac += (x & ((1ull << 47) - 1)) + (j == 0 ? f.top[c] * f.top_f[c] : 0);
            }
            l.n[t] = n;
            l.w[t] = frac;
        }
        if (t == 0) f.cut_lo = f.cut_hi = BINS;
        __syncthreads();
        // the bins' running sums, and the steps on which top_k or top_p may cut (sums are right to 1e-9)
        double own_w = 0.0;
        int own_n = 0;
        if (t < BINS) {
            f.scale[t] = exp2((t + ref) * -0.125);  // a step's middle over the largest e
            own_n = (int)(l.n[t] + l.n[t + BINS]);
            own_w = (own_n * OFFSET + (double)(l.w[t] + l.w[t + BINS]) * (1.0 / (double)(1ull << FRAC))) * f.scale[t];
        }
        const double scan_w = wave_scan(own_w);
        const int scan_n = wave_scan(own_n);
        if (lane == 63) {
            l.part[wave] = scan_w;
            l.parti[wave] = scan_n;
        }
        const double z = sum_of(f.sums, chunks);
        goal = s.p * z;
        __syncthreads();
        if (t < BINS) {
            int n, every;
            waves_before(l.parti, n, every);
            const double part = lane < ROW_WAVES ? l.part[lane] : 0.0, parts = wave_scan(part);
            const int up = __builtin_amdgcn_readfirstlane(wave);
            const double c = scan_w + (up ? wave_lane(parts, up - 1) : 0.0);
            n += scan_n;
            f.cum_w[t] = c;
            f.cum_n[t] = n;
            const uint64_t lo = __ballot(by_k ? n >= s.k : by_p && c >= goal * (1.0 - 1e-9));
            const uint64_t hi = __ballot(by_k ? n >= s.k : by_p && c >= goal * (1.0 + 1e-9));
            if (lane == 0 && lo) atomicMin(&f.cut_lo, t + __ffsll((unsigned long long)lo) - 1);
            if (lane == 0 && hi) atomicMin(&f.cut_hi, t + __ffsll((unsigned long long)hi) - 1);
        }
        __syncthreads();
        // and min_p: its place below the largest's step, in steps
        int min_lo = BINS, min_hi = BINS;
        if (s.m > 0.0 && !(by_k && by_p)) {  // top_p's share is of all the top k
            const double x = log(s.m) * (-8.0 * 1.4426950408889634074) - ref;
            if (x < (double)BINS - 2) {
                min_lo = (int)fmax(0.0, rint(x - 1e-6));
                min_hi = (int)fmax(0.0, rint(x + 1e-6));
            }
        }
        last = min(f.cut_hi, min_hi);
        all = last >= BINS || f.cum_n[last] <= LIST;
        first = all ? 0 : min(f.cut_lo, min_lo);
        if (last >= BINS || f.cum_n[last] - (first ? f.cum_n[first - 1] : 0) > LIST) too_many = true;
        if (by_k && by_p && !all) too_many = true;  // two cuts: only the list decides both
        if (by_p && !by_k && all) {
            double x = far;
            if (t > last) x += own_w;
            rest = block_sum(x, l);
        }
        from = too_many ? M : lowest_in(last, M, g, unit);
        if (first && !too_many) {
            const uint32_t k = key_of(lowest_in(first - 1, M, g, unit));
            to = of_key(k == key_of(0.0f) ? k - 2 : k - 1);  // below 0 comes no -0
        }
    }
    const int n = too_many ? LIST + 1 : gather<TYPE>(row, V, segs, from, to, l, f);
    if (n > LIST) return sample_streaming<TYPE>(a, r, s, M, l);
    if (all) return sample_list(a, r, n, rest, s, M, l);
    Cut cut{0, 1, 1, 0x7FFFFFFF, 0.0, 0.0};
    if (n > 0 && f.cut_lo <= last) {
        init_range(l);
        __syncthreads();
        float x = -INFINITY, y = INFINITY;
        for (int i = t; i < n; i += ROW_THREADS) {
            x = fmaxf(x, l.v[i]);
            y = fminf(y, l.v[i]);
        }
        block_range(x, y, l);
        cut = find_cut(List{l.v, l.i, n}, key_of(y), key_of(x), first ? f.cum_n[first - 1] : 0,
                       first ? f.cum_w[first - 1] : 0.0, s, M, by_k, by_p, by_k ? (double)s.k : goal, l);
        find_end(List{l.v, l.i, n}, cut, l);
    }
    __syncthreads();
    for (int c = wave; c < chunks; c += ROW_WAVES) {  // the chunks' kept sums
        double x = 0.0;
        for (int b = lane; b < first; b += 64) {
            const int j = b - f.off[c];
            if (j >= 0) x += bin_sum(bins[(int64_t)c * BINS + j]) * f.scale[b];
        }
        if (lane == 0 && f.off[c] < first) x += f.top_w[c];
        const int i1 = run_end(l.i, n, (c + 1) * w.chunk);
        for (int i = run_end(l.i, n, c * w.chunk) + lane; i < i1; i += 64) x += kept(l.v[i], l.i[i], cut, s, M);
        x = wave_sum(x);
        if (lane == 0) f.sums[c] = x;
    }
    __syncthreads();
    double before, total;
    const int c = pick_chunk(f.sums, chunks, s.u, &before, &total);
    draw(a, r, WholeRow<TYPE>{row, V}, c * w.chunk, min(w.chunk, V - c * w.chunk), before, total, cut, s, M, l);
}

// Rows whose scan the workspace holds, 148 KB each at 262144: two to a CU in the finish. 1024 rows of 32003 with top-k 64
// and top-p 103 us; with 256 rows at a time 116, with all 1024 93 and twice the workspace.
constexpr int SCAN_ROWS = 512;

// A chunk of 8192 values by 1024 threads, where all chunks at once leave the
// device half empty, or by 256 threads with four times the values each, which
// share a chunk's fixed steps: a row of 262144 6.2 us against 7.2, 8 rows of
// 151936 6.3 against 7.4; 32 rows of 262144 18.4 against 15.7, 256 rows 114
// against 71.
bool wide_scan(int64_t vocab, int64_t n) { return vocab * n < (int64_t)1024 * 8192; }

// Where values lie in no order, those that k of the segments' maxima reach are -segs ln(1 - k / segs) in number: the k
// for which they take a share of the list (a list that overflows is streamed).
int parts_for(int segs, double share) { return (int)(segs * (1.0 - exp(-share * LIST / segs))); }

// The largest top-k that the maxima decide takes 5/6 of the list, and is 7/8 of the segments at most: from there on the
// list is far longer than k. Scan and finish, logits of sd 2.5, by maxima against by bins: 64 rows of 262144 (limit
// 3322), top-k 64 28.9 us against 47.1, 3000 64 against 73; 256 rows, 3000 101 against 125, and past the limit 3481 392
// against 134; a row of 2^21 (limit 6162), 6000 99 against 124, 8192 3126 against 162; 64 rows of 131072 (limit 1792),
// 1740 46.5 against 52.0, 2048 248 against 56.
int most_k_of(int segs) {
    const int fits = parts_for(segs, 5.0 / 6.0), most = segs / 8 * 7;
    return fits < most ? fits : most;
}

Scan scan_of(int64_t vocab, int64_t n, void* workspace) {
    Scan w;
    w.base = static_cast<char*>(workspace);
    w.chunk = 8192;
    w.chunks = (int)((vocab + w.chunk - 1) / w.chunk);
    w.segs = (int)((vocab + SEG - 1) / SEG);
    w.most_k = most_k_of(w.segs);
    w.most_reached = parts_for(w.segs, 0.95);
    w.row_bytes = Scan::up16(w.bytes());
    return w;
}

template <int TYPE>
void launch_sample(const SampleArgs& a, int64_t n, void* workspace, void* stream) {
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (a.V <= LIST) {
        hipLaunchKernelGGL(k_sample_rows<TYPE>, dim3((unsigned)n), dim3(ROW_THREADS), 0, s, a);
        return;
    }
    const int64_t rows = n < SCAN_ROWS ? n : SCAN_ROWS;
    const Scan w = scan_of(a.V, rows, workspace);
    for (int64_t r = 0; r < n; r += rows) {
        const unsigned now = (unsigned)(n - r < rows ? n - r : rows);
        const dim3 grid((unsigned)w.chunks, now);
        if (wide_scan(a.V, rows))
            hipLaunchKernelGGL((k_sample_scan<TYPE, 2>), grid, dim3(1024), 0, s, a, w, r);
        else
            hipLaunchKernelGGL((k_sample_scan<TYPE, 8>), grid, dim3(256), 0, s, a, w, r);
        hipLaunchKernelGGL(k_sample_finish<TYPE>, dim3(now), dim3(ROW_THREADS), 0, s, a, w, r);
    }
}

}  // namespace

extern "C" size_t ft_hip_sample_tokens_workspace_bytes(int64_t vocab, int64_t n) {
    if (vocab <= 0 || vocab > FT_SAMPLE_MAX_VOCAB || n < 0 || n > FT_SAMPLE_MAX_ROWS) return 0;
    const int64_t rows = n < SCAN_ROWS ? n : SCAN_ROWS;
    return vocab <= LIST || n == 0 ? 256 : (size_t)(rows * scan_of(vocab, rows, nullptr).row_bytes);
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
    if (!aligned(logits, logits_type == FT_TYPE_F32 ? 4 : 2))
        return fail(FT_HIP_E_SHAPE, "sample_tokens: logits are not aligned to their type");
    if (!aligned(temperature, 4) || !aligned(top_k, 4) || !aligned(top_p, 4) || !aligned(min_p, 4) || !aligned(u, 4) ||
        !aligned(tokens, 4) || !aligned(logprobs, 4))
        return fail(FT_HIP_E_SHAPE, "sample_tokens: a row's settings or outputs are not aligned to 4 bytes");
    if (!aligned(workspace, 16))
        return fail(FT_HIP_E_SHAPE, "sample_tokens: workspace must be 16-byte aligned");
    const size_t need = ft_hip_sample_tokens_workspace_bytes(vocab, n);
    if (workspace_bytes < need)
        return fail(FT_HIP_E_SHAPE, "sample_tokens: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    if (!ctx) return fail(FT_HIP_E_INVALID, "sample_tokens: null argument");
    if (n == 0) return FT_HIP_OK;  // an empty tensor has no address
    if (!logits || !u || !tokens || !workspace) return fail(FT_HIP_E_INVALID, "sample_tokens: null argument");
    // a row's settings are read before its outputs are written, and no other row's are: an output may be one of them
    const int64_t size = logits_type == FT_TYPE_F32 ? 4 : 2;
    const auto row4 = [&](const void* p) { return Span{p, 1, 0, n * 4}; };
    const Span rows{logits, n, logits_stride * size, vocab * size}, ws{workspace, 1, 0, (int64_t)need},
        tok = row4(tokens), lp = row4(logprobs), settings[] = {row4(temperature), row4(top_k), row4(top_p), row4(min_p),
                                                               row4(u)};
    if (overlap(tok, rows) || overlap(lp, rows) || overlap(tok, lp))
        return fail(FT_HIP_E_SHAPE, "sample_tokens: tokens or logprobs overlap the logits or each other");
    if (overlap(ws, rows) || overlap(ws, tok) || overlap(ws, lp))
        return fail(FT_HIP_E_SHAPE, "sample_tokens: the workspace overlaps the logits or an output");
    for (const Span& in : settings)
        if (overlap(ws, in) || (overlap(tok, in) && tok.at != in.at) || (overlap(lp, in) && lp.at != in.at))
            return fail(FT_HIP_E_SHAPE, "sample_tokens: the workspace or an output overlaps a row's settings");
    const int given = (temperature ? HAS_T : 0) | (top_k ? HAS_K : 0) | (top_p ? HAS_P : 0) | (min_p ? HAS_M : 0);
    const SampleArgs a{logits, logits_stride, (int)vocab, temperature ? temperature : u,
                       top_k ? top_k : reinterpret_cast<const int32_t*>(u), top_p ? top_p : u, min_p ? min_p : u, u,
                       tokens, logprobs, given};
    DeviceGuard on(ctx->device);
    if (!on.ok) return fail(FT_HIP_E_DEVICE, "sample_tokens: device %d cannot be made current", ctx->device);
    if (logits_type == FT_TYPE_F32)
        launch_sample<FT_TYPE_F32>(a, n, workspace, stream);
    else if (logits_type == FT_TYPE_F16)
        launch_sample<FT_TYPE_F16>(a, n, workspace, stream);
    else
        launch_sample<FT_TYPE_BF16>(a, n, workspace, stream);
    return launch_status("sample_tokens");
}
