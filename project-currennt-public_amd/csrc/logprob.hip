// Log probabilities of given tokens with the entropy of their distribution, the most probable alternatives, and the gradient.
//
//   z = scale * logit,   lse = log sum_v exp z_v,   logp_v = z_v - lse,   H = - sum_v p_v logp_v
//   err_v = scale * (g * ([v = token] - p_v) - h * p_v * (logp_v + H))       g, h: errors of the token's logp and of the entropy
//
// One pass over the logits: a lane keeps the running maximum m of its logits, s = sum 2^t and w = sum t 2^t with t = (x - m) * scale *
// log2(e), and brings them to a new maximum once in up to 32 logits; then lse = scale * m + log s and H = log s - ln 2 * w / s.  The
// difference to the maximum is formed before it is scaled, so the rows of a mask of the type's lowest value stay exact.  All sums are fp32.
#include "elements.hpp"

#include <algorithm>
#include <cmath>

namespace cnt {
namespace {

constexpr int kMostTop = 64;
constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.693147180559945309f;
constexpr float kMinusInfinity = -__builtin_inff();

struct RowArgs {
    const void *logits;
    long stride;
    const int *tokens;
    long N;
    int V, K;
    int parts, part;  // workgroups that share a row, logits of each
    float scale;
    float *logp, *lse, *entropy, *top_logp;
    int *top_tokens;
    float *part_stats, *part_values;  // of a shared row: three statistics, K values, K tokens per part
    int *part_tokens;
    const float *logp_err, *entropy_err;
    void *err;
    long err_stride;
};

// ----- a wave's view of a row: chunks of NV vectors of W logits per lane -----------------------------------------------------
template <typename T, int NV>
struct Chunk {
    static constexpr int W = kWide<T>, COUNT = NV * W, SPAN = 64 * COUNT;
    float x[COUNT];
};
// logits begin .. begin + SPAN of a row, those from `end` on are -inf
template <typename T, int NV>
__device__ __forceinline__ void load_chunk(const T *row, int begin, int end, int lane, Chunk<T, NV> &c) {
    constexpr int W = Chunk<T, NV>::W;
    const bool whole = begin + Chunk<T, NV>::SPAN <= end;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int at = begin + (j * 64 + lane) * W;
        float v[W];
        if (whole) fetch_elements<T, W>(row + at, v);
        else fetch_some<T, W>(row + at, max(0, min(W, end - at)), v, kMinusInfinity);
#pragma unroll
        for (int i = 0; i < W; ++i) c.x[j * W + i] = v[i];
    }
}

// ----- statistics ------------------------------------------------------------------------------------------------------------
struct Stats {
    float m, s, w;
};
__device__ __forceinline__ void begin_stats(Stats &a) {
    a.m = kMinusInfinity;
    a.s = a.w = 0.0f;
}
// t of a logit that is -inf is -inf, and its share of w is 0 and not 0 * -inf
__device__ __forceinline__ float at_least(float t) { return fmaxf(t, -1000.0f); }
// brings the sums from their maximum to `m`, which is not below it (ref: m, 0 for -inf)
__device__ __forceinline__ void shift_stats(Stats &a, float m, float ref, float c) {
    const float shift = a.s == 0.0f ? 0.0f : (a.m - ref) * c;
    const float f = __builtin_amdgcn_exp2f(shift);
    a.w = (a.w + a.s * at_least(shift)) * f;
    a.s *= f;
    a.m = m;
}
template <typename T, int NV>
__device__ __forceinline__ void fold(Stats &a, const Chunk<T, NV> &x, float c) {
    float m = a.m;
#pragma unroll
    for (int i = 0; i < Chunk<T, NV>::COUNT; ++i) m = fmaxf(m, x.x[i]);
    const float ref = m == kMinusInfinity ? 0.0f : m;
    shift_stats(a, m, ref, c);
#pragma unroll
    for (int i = 0; i < Chunk<T, NV>::COUNT; ++i) {
        const float t = (x.x[i] - ref) * c, e = __builtin_amdgcn_exp2f(t);
        a.s += e;
        a.w = __builtin_fmaf(e, at_least(t), a.w);
    }
}
__device__ __forceinline__ Stats join(Stats a, Stats b, float c) {
    const float m = fmaxf(a.m, b.m), ref = m == kMinusInfinity ? 0.0f : m;
    shift_stats(a, m, ref, c);
    shift_stats(b, m, ref, c);
    a.s += b.s;
    a.w += b.w;
    return a;
}
__device__ __forceinline__ Stats join_lanes(Stats a, float c) {
    for (int o = 32; o > 0; o >>= 1) {
        const Stats b = {__shfl_xor(a.m, o), __shfl_xor(a.s, o), __shfl_xor(a.w, o)};
        a = join(a, b, c);
    }
    return a;
}

// ----- the best K of a row, in the first K lanes of a wave ----------------------------------------------------------------------
// Order: the larger logit, the lower token where two are equal.  NaN is never among them.
struct Best {
    float value;
    int token, count;  // count: entries in the list, the same in every lane
    float least;       // value of the last one of a full list, the same in every lane
};
__device__ __forceinline__ void begin_best(Best &b) {
    b.value = b.least = __builtin_nanf("");
    b.token = -1;
    b.count = 0;
}
__device__ __forceinline__ float of_lane(float v, int lane) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), lane)); }
// puts an entry to place `rank` < K; the others from there on move one lane up
__device__ __forceinline__ void insert(Best &b, float value, int token, int rank, int K, int lane) {
    const float below_value = __shfl_up(b.value, 1);
    const int below_token = __shfl_up(b.token, 1);
    b.value = lane == rank ? value : lane > rank ? below_value : b.value;
    b.token = lane == rank ? token : lane > rank ? below_token : b.token;
    b.count = min(b.count + 1, K);
    b.least = of_lane(b.value, K - 1);
}
__device__ __forceinline__ float wave_max(float v) {
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return of_lane(v, 0);
}
// A chunk's logits that belong into the list, largest first: at most K rounds, each of which takes one logit out of the chunk (c is used
// up).  Most chunks of a long row end in the first test.  Tokens of later chunks are higher, so an equal logit goes behind.
template <typename T, int NV>
__device__ __forceinline__ void take_best(Best &b, Chunk<T, NV> &c, int begin, int end, int K, int lane) {
    constexpr int W = Chunk<T, NV>::W;
    float top[NV], best = __builtin_nanf("");
    if (begin + Chunk<T, NV>::SPAN > end) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < W; ++i)
                if (begin + (j * 64 + lane) * W + i >= end) c.x[j * W + i] = __builtin_nanf("");
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        top[j] = c.x[j * W];
#pragma unroll
        for (int i = 1; i < W; ++i) top[j] = fmaxf(top[j], c.x[j * W + i]);
        best = fmaxf(best, top[j]);
    }
    // one more round than the list has places would find nothing: the list's last entry is then not below the chunk's largest
    while (true) {
        const bool full = b.count == K;
        if (full && __ballot(best > b.least) == 0) break;
        const float m = wave_max(best);
        if (m != m) break;
        unsigned long long holders = 0;
        int vec = 0;
#pragma unroll
        for (int j = NV - 1; j >= 0; --j) {
            const unsigned long long h = __ballot(top[j] == m);
            if (h) {
                holders = h;
                vec = j;
            }
        }
        const int owner = __builtin_ctzll(holders);
        int at = 0;
        best = __builtin_nanf("");
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            if (j == vec) {
#pragma unroll
                for (int i = W - 1; i >= 0; --i) at = c.x[j * W + i] == m ? i : at;
                at = __builtin_amdgcn_readlane(at, owner);
                float t = __builtin_nanf("");
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    if (lane == owner && i == at) c.x[j * W + i] = __builtin_nanf("");
                    t = fmaxf(t, c.x[j * W + i]);
                }
                top[j] = t;
            }
            best = fmaxf(best, top[j]);
        }
        const int rank = __popcll(__ballot(b.value >= m));
        insert(b, m, begin + (vec * 64 + owner) * W + at, rank, K, lane);
    }
}
// entries of another list, largest first, in lanes 0 .. K - 1 of (value, token); token -1: none
__device__ __forceinline__ void merge_best(Best &b, float value, int token, int K, int lane) {
    for (int k = 0; k < K; ++k) {
        const float v = of_lane(value, k);
        const int t = __builtin_amdgcn_readlane(token, k);
        if (t < 0) break;
        const int rank = __popcll(__ballot(b.token >= 0 && lane < K && (b.value > v || (b.value == v && b.token < t))));
        if (rank >= K) break;
        insert(b, v, t, rank, K, lane);
    }
}

// ----- results of a row --------------------------------------------------------------------------------------------------------
__device__ __forceinline__ float logp_of(float x, const Stats &a, float scale, float log_s) {
    // a row whose mask leaves nothing has no probabilities: all are 0
    return a.m == kMinusInfinity && a.s == 0.0f ? kMinusInfinity : (x - a.m) * scale - log_s;
}
__device__ __forceinline__ float entropy_of(const Stats &a, float log_s) {
    return a.m == kMinusInfinity && a.s == 0.0f ? 0.0f : log_s - kLn2 * (a.w / a.s);
}
template <typename T>
__device__ __forceinline__ void write_results(const RowArgs &a, long n, const Stats &s, const Best &b, int lane) {
    const float log_s = logf(s.s);
    const T *row = static_cast<const T *>(a.logits) + n * a.stride;
    if (lane == 0) {
        if (a.logp) {
            const int token = a.tokens ? a.tokens[n] : -1;
            a.logp[n] = token >= 0 && token < a.V ? logp_of((float)row[token], s, a.scale, log_s) : 0.0f;
        }
        if (a.lse) a.lse[n] = s.m * a.scale + log_s;
        if (a.entropy) a.entropy[n] = entropy_of(s, log_s);
    }
    if (lane < a.K) {
        if (a.top_logp) a.top_logp[n * a.K + lane] = b.token < 0 ? __builtin_nanf("") : logp_of(b.value, s, a.scale, log_s);
        if (a.top_tokens) a.top_tokens[n * a.K + lane] = b.token;
    }
}

// A row, or a part of one, by WAVES waves of a workgroup of four: their chunks alternate.
template <typename T, int NV, int WAVES, bool TOP>
__global__ __launch_bounds__(256) void logprob_kernel(const RowArgs a) {
    constexpr int SPAN = Chunk<T, NV>::SPAN;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long n = WAVES == 1 ? (long)blockIdx.x * 4 + wave : (long)blockIdx.x;
    if (n >= a.N) return;  // (a workgroup of one row never)
    const float c = a.scale * kLog2e;
    const T *row = static_cast<const T *>(a.logits) + n * a.stride;
    const int begin = WAVES == 1 ? 0 : (int)blockIdx.y * a.part, end = WAVES == 1 ? a.V : min(a.V, begin + a.part);
    Stats s;
    Best b;
    begin_stats(s);
    begin_best(b);
    for (int at = begin + (WAVES == 1 ? 0 : wave * SPAN); at < end; at += WAVES * SPAN) {
        Chunk<T, NV> x;
        load_chunk(row, at, end, lane, x);
        fold(s, x, c);
        if (TOP) take_best(b, x, at, end, a.K, lane);
    }
    s = join_lanes(s, c);
    if (WAVES > 1) {
        __shared__ Stats stats[4];
        __shared__ float values[4][kMostTop];
        __shared__ int tokens[4][kMostTop];
        if (lane == 0) stats[wave] = s;
        if (TOP) {
            values[wave][lane] = b.value;
            tokens[wave][lane] = lane < b.count ? b.token : -1;
        }
        __syncthreads();
        if (wave != 0) return;
#pragma unroll
        for (int w = 1; w < WAVES; ++w) {
            s = join(s, stats[w], c);
            if (TOP) merge_best(b, values[w][lane], tokens[w][lane], a.K, lane);
        }
        if (a.parts > 1) {
            const long p = n * a.parts + blockIdx.y;
            if (lane == 0) {
                a.part_stats[p * 3] = s.m;
                a.part_stats[p * 3 + 1] = s.s;
                a.part_stats[p * 3 + 2] = s.w;
            }
            if (TOP && lane < a.K) {
                a.part_values[p * a.K + lane] = b.value;
                a.part_tokens[p * a.K + lane] = b.token;
            }
            return;
        }
    }
    write_results<T>(a, n, s, b, lane);
}

// the parts of a row, by a wave
template <typename T>
__global__ __launch_bounds__(64) void logprob_join_kernel(const RowArgs a) {
    const long n = blockIdx.x;
    const int lane = threadIdx.x;
    const float c = a.scale * kLog2e;
    Stats s;
    Best b;
    begin_stats(s);
    begin_best(b);
    const long p = n * a.parts;
    if (lane < a.parts) s = {a.part_stats[(p + lane) * 3], a.part_stats[(p + lane) * 3 + 1], a.part_stats[(p + lane) * 3 + 2]};
    s = join_lanes(s, c);
    if (a.K > 0)
        for (int i = 0; i < a.parts; ++i) {
            const long at = (p + i) * a.K + lane;
            merge_best(b, lane < a.K ? a.part_values[at] : 0.0f, lane < a.K ? a.part_tokens[at] : -1, a.K, lane);
        }
    write_results<T>(a, n, s, b, lane);
}

// ----- gradient ----------------------------------------------------------------------------------------------------------------
// err = p * (first + second * t), t = log2 p, and `given` more at the token
struct Slopes {
    float first, second, given;
    int token;
};
__device__ __forceinline__ Slopes slopes_of(const RowArgs &a, long n, float lse, float entropy) {
    int token = a.tokens ? a.tokens[n] : -1;
    if (token >= a.V || token < 0) token = -1;
    const float g = a.logp_err && token >= 0 ? a.logp_err[n] : 0.0f, h = a.entropy_err ? a.entropy_err[n] : 0.0f;
    Slopes s;
    s.first = -a.scale * (h == 0.0f ? g : g + h * entropy);
    s.second = -a.scale * h * kLn2;
    s.given = a.scale * g;
    s.token = lse == kMinusInfinity ? -1 : token;  // nothing to choose from: no gradient
    if (lse != lse) s.first = lse;
    return s;
}
template <typename T, int NV>
__device__ __forceinline__ void put_gradient(T *row, int begin, int end, int lane, const Slopes &s, const Chunk<T, NV> &t) {
    constexpr int W = Chunk<T, NV>::W;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int at = begin + (j * 64 + lane) * W;
        float v[W];
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const float u = at_least(t.x[j * W + i]);
            v[i] = __builtin_amdgcn_exp2f(u) * __builtin_fmaf(s.second, u, s.first);
        }
        if ((unsigned)(s.token - at) < (unsigned)W) {
#pragma unroll
            for (int i = 0; i < W; ++i) v[i] += s.token - at == i ? s.given : 0.0f;
        }
        put_some<T, W>(row + at, max(0, min(W, end - at)), v);
    }
}

// from saved statistics: blockIdx.x the row, blockIdx.y a stretch of it
template <typename T, int NV>
__global__ __launch_bounds__(256) void logprob_gradient_kernel(const RowArgs a) {
    constexpr int SPAN = Chunk<T, NV>::SPAN;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long n = blockIdx.x;
    const float lse = a.lse[n];
    const Slopes s = slopes_of(a, n, lse, a.entropy ? a.entropy[n] : 0.0f);
    const T *row = static_cast<const T *>(a.logits) + n * a.stride;
    T *to = static_cast<T *>(a.err) + n * a.err_stride;
    const float ref = lse == kMinusInfinity ? 0.0f : lse;
    for (int at = (blockIdx.y * 4 + wave) * SPAN; at < a.V; at += gridDim.y * 4 * SPAN) {
        Chunk<T, NV> x;
        load_chunk(row, at, a.V, lane, x);
#pragma unroll
        for (int i = 0; i < Chunk<T, NV>::COUNT; ++i) x.x[i] = (x.x[i] * a.scale - ref) * kLog2e;
        put_gradient(to, at, a.V, lane, s, x);
    }
}

// statistics and gradient of a row by WAVES waves of a workgroup of four
template <typename T, int NV, int WAVES>
__global__ __launch_bounds__(256) void logprob_error_kernel(const RowArgs a) {
    constexpr int SPAN = Chunk<T, NV>::SPAN;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long n = WAVES == 1 ? (long)blockIdx.x * 4 + wave : (long)blockIdx.x;
    if (n >= a.N) return;
    const float c = a.scale * kLog2e;
    const T *row = static_cast<const T *>(a.logits) + n * a.stride;
    T *to = static_cast<T *>(a.err) + n * a.err_stride;
    const int first = WAVES == 1 ? 0 : wave * SPAN;
    Stats s;
    Best none;
    begin_stats(s);
    begin_best(none);
    Chunk<T, NV> x;
    for (int at = first; at < a.V; at += WAVES * SPAN) {
        load_chunk(row, at, a.V, lane, x);
        fold(s, x, c);
    }
    s = join_lanes(s, c);
    if (WAVES > 1) {
        __shared__ Stats stats[4];
        if (lane == 0) stats[wave] = s;
        __syncthreads();
        s = stats[0];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) s = join(s, stats[w], c);
    }
    if (WAVES == 1 || wave == 0) write_results<T>(a, n, s, none, lane);
    // the errors may take the logits' place: the token's logit has been read before any of the workgroup's errors is written
    if (WAVES > 1) __syncthreads();
    const float log_s = logf(s.s), log2_s = log_s * kLog2e;
    const Slopes slopes = slopes_of(a, n, s.m * a.scale + log_s, entropy_of(s, log_s));
    const float ref = s.m == kMinusInfinity ? 0.0f : s.m;
    for (int at = first; at < a.V; at += WAVES * SPAN) {
        if (WAVES > 1) load_chunk(row, at, a.V, lane, x);
#pragma unroll
        for (int i = 0; i < Chunk<T, NV>::COUNT; ++i) x.x[i] = (x.x[i] - ref) * c - log2_s;
        put_gradient(to, at, a.V, lane, slopes, x);
    }
}

// ----- launches ------------------------------------------------------------------------------------------------------------------
// Logits of a wave's chunk: 32 per lane.  A row that fits into one is a wave's.
constexpr int kSpan = 64 * 32;
// Parts of a row: enough workgroups for the card where there are few rows, each with a chunk per wave at least, as many as a wave can join.
int parts_of(long N, int V) {
    if (V <= kSpan || N == 0 || N >= 512) return 1;
    return (int)std::min({64L, (V + 4L * kSpan - 1) / (4 * kSpan), (1023 + N) / N});
}

template <typename T, int NV, int WAVES>
void launch_rows(hipStream_t stream, const RowArgs &a) {
    const dim3 grid((unsigned)(WAVES == 1 ? (a.N + 3) / 4 : a.N), (unsigned)a.parts), block(256);
    if (a.K > 0) hipLaunchKernelGGL((logprob_kernel<T, NV, WAVES, true>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((logprob_kernel<T, NV, WAVES, false>), grid, block, 0, stream, a);
    if (a.parts > 1) hipLaunchKernelGGL(logprob_join_kernel<T>, dim3((unsigned)a.N), dim3(64), 0, stream, a);
}

size_t scratch_of(long N, int V, int K) {
    const int parts = parts_of(N, V);
    return parts == 1 ? 0 : (size_t)N * parts * (3 + 2 * (size_t)K) * sizeof(float);
}
// where a shared row's statistics and lists are
void lay_out(RowArgs &a, void *scratch) {
    const size_t p = (size_t)a.N * a.parts;
    a.part_stats = static_cast<float *>(scratch);
    a.part_values = a.part_stats + p * 3;
    a.part_tokens = reinterpret_cast<int *>(a.part_values + p * a.K);
    // a part is a whole number of its waves' rounds
    a.part = ((a.V + a.parts - 1) / a.parts + 4 * kSpan - 1) / (4 * kSpan) * (4 * kSpan);
}

int forward(hipStream_t stream, int type, RowArgs &a, void *scratch) {
    a.parts = parts_of(a.N, a.V);
    lay_out(a, scratch);
    with_type(type, [&](auto t) {
        using T = typename decltype(t)::type;
        constexpr int NV = 32 / kWide<T>;
        if (a.V <= 64 * kWide<T>) launch_rows<T, 1, 1>(stream, a);
        else if (a.V <= kSpan) launch_rows<T, NV, 1>(stream, a);
        else launch_rows<T, NV, 4>(stream, a);
    });
    CNT_HIP(hipGetLastError());
    return CNT_OK;
}

int gradient(hipStream_t stream, int type, const RowArgs &a) {
    const dim3 grid((unsigned)a.N, (unsigned)std::min(1024L, (a.V + 4L * kSpan - 1) / (4 * kSpan)));
    with_type(type, [&](auto t) {
        using T = typename decltype(t)::type;
        hipLaunchKernelGGL((logprob_gradient_kernel<T, 32 / kWide<T>>), grid, dim3(256), 0, stream, a);
    });
    CNT_HIP(hipGetLastError());
    return CNT_OK;
}

// what every call asks of its rows
int check_rows(const char *who, long N, int V, int type, const void *logits, long stride, float scale) {
    CNT_REQUIRE(N >= 0 && V > 0 && V <= 1 << 30 && N < 1L << 24, "%s: bad sizes", who);
    CNT_REQUIRE(known_type(type), "%s: unknown element type %d", who, type);
    CNT_REQUIRE(stride >= 0, "%s: negative stride", who);
    CNT_REQUIRE(N == 0 || logits, "%s: null argument", who);
    CNT_REQUIRE(scale > 0 && std::isfinite(scale), "%s: the scale has to be positive and finite", who);
    return CNT_OK;
}
int check_scratch(const char *who, long N, int V, int K, const void *scratch, size_t bytes) {
    const size_t need = scratch_of(N, V, K);
    CNT_REQUIRE(need == 0 || (scratch && bytes >= need), "%s: %zu bytes of scratch memory, %zu are needed", who, bytes, need);
    CNT_REQUIRE(need == 0 || reinterpret_cast<uintptr_t>(scratch) % 4 == 0, "%s: the scratch memory is not aligned to 4 bytes", who);
    return CNT_OK;
}

}  // namespace
}  // namespace cnt

extern "C" {

long cnt_logprob_scratch(long N, int V, int K) {
    if (N < 0 || V <= 0 || K < 0 || K > cnt::kMostTop) return -1;
    return (long)cnt::scratch_of(N, V, K);
}

int cnt_logprob_forward(void *stream_, long N, int V, int type, const void *logits, long stride, float scale, const int *tokens,
                        float *logp, float *lse, float *entropy, int K, float *top_logp, int *top_tokens, void *scratch,
                        size_t scratch_bytes) {
    using namespace cnt;
    CNT_TRY(check_rows("logprob_forward", N, V, type, logits, stride, scale));
    CNT_REQUIRE(K >= 0 && K <= kMostTop && K <= V, "logprob_forward: %d alternatives, up to %d and up to the number of tokens are possible",
                K, kMostTop);
    CNT_REQUIRE(K == 0 || N == 0 || top_logp || top_tokens, "logprob_forward: alternatives without a place for them");
    CNT_REQUIRE(!logp || tokens || N == 0, "logprob_forward: log probabilities of which tokens?");
    CNT_TRY(check_scratch("logprob_forward", N, V, K, scratch, scratch_bytes));
    if (N == 0) return CNT_OK;
    RowArgs a = {};
    a.logits = logits; a.stride = stride; a.tokens = tokens; a.N = N; a.V = V; a.K = K; a.scale = scale;
    a.logp = logp; a.lse = lse; a.entropy = entropy; a.top_logp = top_logp; a.top_tokens = top_tokens;
    ProfileScope prof(static_cast<hipStream_t>(stream_), "logprob_forward");
    return forward(static_cast<hipStream_t>(stream_), type, a, scratch);
}

int cnt_logprob_backward(void *stream_, long N, int V, int type, const void *logits, long stride, float scale, const int *tokens,
                         const float *lse, const float *entropy, const float *logp_err, const float *entropy_err, void *err,
                         long err_stride) {
    using namespace cnt;
    CNT_TRY(check_rows("logprob_backward", N, V, type, logits, stride, scale));
    CNT_REQUIRE(err_stride >= V, "logprob_backward: rows of the errors overlap");
    CNT_REQUIRE(N == 0 || (lse && err), "logprob_backward: null argument");
    CNT_REQUIRE(!entropy_err || entropy || N == 0, "logprob_backward: errors of entropies without the entropies");
    CNT_REQUIRE(!logp_err || tokens || N == 0, "logprob_backward: errors of log probabilities of which tokens?");
    if (N == 0) return CNT_OK;
    RowArgs a = {};
    a.logits = logits; a.stride = stride; a.tokens = tokens; a.N = N; a.V = V; a.scale = scale;
    a.lse = const_cast<float *>(lse); a.entropy = const_cast<float *>(entropy);
    a.logp_err = logp_err; a.entropy_err = entropy_err; a.err = err; a.err_stride = err_stride;
    ProfileScope prof(static_cast<hipStream_t>(stream_), "logprob_backward");
    return gradient(static_cast<hipStream_t>(stream_), type, a);
}

int cnt_logprob_error_backward(void *stream_, long N, int V, int type, const void *logits, long stride, float scale, const int *tokens,
                               const float *logp_err, const float *entropy_err, float *logp, float *lse, float *entropy, void *err,
                               long err_stride, void *scratch, size_t scratch_bytes) {
    using namespace cnt;
    CNT_TRY(check_rows("logprob_error_backward", N, V, type, logits, stride, scale));
    CNT_REQUIRE(err_stride >= V, "logprob_error_backward: rows of the errors overlap");
    CNT_REQUIRE(N == 0 || (err && lse && entropy), "logprob_error_backward: null argument");
    CNT_REQUIRE((!logp_err && !logp) || tokens || N == 0, "logprob_error_backward: log probabilities of which tokens?");
    CNT_TRY(check_scratch("logprob_error_backward", N, V, 0, scratch, scratch_bytes));
    if (N == 0) return CNT_OK;
    RowArgs a = {};
    a.logits = logits; a.stride = stride; a.tokens = tokens; a.N = N; a.V = V; a.scale = scale;
    a.logp = logp; a.lse = lse; a.entropy = entropy;
    a.logp_err = logp_err; a.entropy_err = entropy_err; a.err = err; a.err_stride = err_stride;
    hipStream_t stream = static_cast<hipStream_t>(stream_);
    ProfileScope prof(stream, "logprob_error_backward");
    if (parts_of(N, V) > 1) {  // few long rows: shared out among workgroups
        CNT_TRY(forward(stream, type, a, scratch));
        return gradient(stream, type, a);
    }
    with_type(type, [&](auto t) {
        using T = typename decltype(t)::type;
        constexpr int NV = 32 / kWide<T>;
        const dim3 few((unsigned)((N + 3) / 4)), many((unsigned)N), block(256);
        if (V <= 64 * kWide<T>) hipLaunchKernelGGL((logprob_error_kernel<T, 1, 1>), few, block, 0, stream, a);
        else if (V <= kSpan) hipLaunchKernelGGL((logprob_error_kernel<T, NV, 1>), few, block, 0, stream, a);
        else hipLaunchKernelGGL((logprob_error_kernel<T, NV, 4>), many, block, 0, stream, a);
    });
    CNT_HIP(hipGetLastError());
    return CNT_OK;
}

}  // extern "C"
