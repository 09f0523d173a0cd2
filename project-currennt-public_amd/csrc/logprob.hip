// Log probabilities of given tokens with the entropy of their distribution, the most probable alternatives, and the gradient.
//
//   z = scale * logit,   lse = log sum_v exp z_v,   logp_v = z_v - lse,   H = - sum_v p_v logp_v
//   err_v = scale * (g * ([v = token] - p_v) - h * p_v * (logp_v + H))       g, h: errors of the token's logp and of the entropy
//
// One pass over the logits: a lane keeps the running maximum m of its logits, s = sum 2^t and w = sum t 2^t with t = (x - m) * scale *
// log2(e), and brings them to a new maximum once in 16 logits (32 in the longest rows' errors); then lse = scale * m + log s and H = log s - ln 2 * w / s.  The
// difference to the maximum is formed before it is scaled, so the rows of a mask of the type's lowest value stay exact
// (but for the gradient from a saved log sum, which is rounded to 32 bits).  All sums are fp32.
#include "elements.hpp"

#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>

namespace cnt {
namespace {

constexpr int kMostTop = 64, kMostJoined = 1024;
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
    float *part_stats, *part_values;  // of a shared row: three statistics, K values, K tokens per part; joined: maximum and log s in the first part's place
    int *part_tokens;
    const float *logp_err, *entropy_err;
    void *err;
    long err_stride;
};

// ----- sums and maxima over the lanes that share a row: 16 (a row of the data-parallel permutations) or a wave ----------------
template <int ROTATE>
__device__ __forceinline__ int rotated(int v) { return __builtin_amdgcn_update_dpp(v, v, 0x120 + ROTATE, 0xf, 0xf, false); }
template <int ROTATE>
__device__ __forceinline__ unsigned rotated(unsigned v) { return (unsigned)rotated<ROTATE>((int)v); }
template <int ROTATE>
__device__ __forceinline__ float rotated(float v) { return __int_as_float(rotated<ROTATE>(__float_as_int(v))); }
__device__ __forceinline__ float of_lane(float v, int lane) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane)); }
template <int LANES, typename V, typename F>
__device__ __forceinline__ V over_lanes(V v, F f) {
    v = f(v, rotated<8>(v));
    v = f(v, rotated<4>(v));
    v = f(v, rotated<2>(v));
    v = f(v, rotated<1>(v));
    if (LANES == 16) return v;
    auto at = [&](int lane) {
        if constexpr (std::is_integral<V>::value) return (V)__builtin_amdgcn_readlane((int)v, lane);
        else return of_lane(v, lane);
    };
    return f(f(at(0), at(16)), f(at(32), at(48)));
}
template <int LANES>
__device__ __forceinline__ float max_of(float v) { return over_lanes<LANES>(v, [](float a, float b) { return fmaxf(a, b); }); }
template <int LANES>
__device__ __forceinline__ float sum_of(float v) { return over_lanes<LANES>(v, [](float a, float b) { return a + b; }); }
template <int LANES>
__device__ __forceinline__ int min_of(int v) { return over_lanes<LANES>(v, [](int a, int b) { return a < b ? a : b; }); }

// ----- a wave's view of a row: chunks of NV vectors of W logits per lane -----------------------------------------------------
template <typename T, int NV>
struct Chunk {
    static constexpr int W = kWide<T>, COUNT = NV * W, SPAN = 64 * COUNT;
    float x[COUNT];
};
// Logits of a row are dealt to threads in vectors from a cache line's begin on, `lead` logits before the row's first one, if the row begins inside a
// line: 16-byte accesses that do not begin at 16 bytes took a fifth longer (2047 rows of 100003 16-bit logits: 97 us for 84).
template <typename T>
__device__ __forceinline__ int lead_of(const T *row) { return (int)(reinterpret_cast<uintptr_t>(row) % 128 / sizeof(T)); }
// W logits from `at` on, those before the row and from `end` on are `rest`
template <bool ONCE, typename T, int W>
__device__ __forceinline__ void fetch_within(const T *row, int at, int end, float (&v)[W], float rest) {
    if (at >= 0 && at + W <= end) {
        fetch_elements<T, W, ONCE>(row + at, v);
        return;
    }
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] = at + i >= 0 && at + i < end ? (float)row[at + i] : rest;
}
template <typename T, int W>
__device__ __forceinline__ void put_within(T *row, int at, int end, const float (&v)[W]) {
    if (at >= 0 && at + W <= end) {
        put_elements<T, W, true>(row + at, v);
        return;
    }
#pragma unroll
    for (int i = 0; i < W; ++i)
        if (at + i >= 0 && at + i < end) row[at + i] = (T)v[i];
}
// 16 bytes of a row as they stand in memory.  values<USE>(): the logits in 32 bits, converted anew for every USE: from expressions that it knows to be
// the same the compiler keeps one use's 32-bit values for the next, which takes twice the registers of 16-bit logits.
template <int USE>
__device__ __forceinline__ void halves(unsigned x, float &low, float &high, __bf16) {
    asm("v_lshlrev_b32 %0, 16, %1 ; %2" : "=v"(low) : "v"(x), "i"(USE));
    asm("v_and_b32 %0, 0xffff0000, %1 ; %2" : "=v"(high) : "v"(x), "i"(USE));
}
template <int USE>
__device__ __forceinline__ void halves(unsigned x, float &low, float &high, _Float16) {
    asm("v_cvt_f32_f16 %0, %1 ; %2" : "=v"(low) : "v"(x), "i"(USE));
    asm("v_cvt_f32_f16_sdwa %0, %1 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:WORD_1 ; %2" : "=v"(high) : "v"(x), "i"(USE));
}
template <typename T>
struct Raw {
    typedef unsigned words __attribute__((ext_vector_type(4), aligned(2)));
    words x;
    // (a vector that is not there is never looked at)
    __device__ __forceinline__ void load(const T *p, bool whole) {
        x = words{0u, 0u, 0u, 0u};
        if (whole) x = __builtin_nontemporal_load(reinterpret_cast<const words *>(p));
    }
    // The logits from `at` on that are within 0 .. end, the others are -inf: whole vectors by the first of these, the rest by the second, which a lane
    // calls for all of its vectors behind the first, so that one's loads do not wait for another's.
    template <bool ONCE>
    __device__ __forceinline__ void load_within(const T *row, int at, int end) {
        constexpr unsigned nothing = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __bf16>::value ? 0xff80ff80u : 0xfc00fc00u;
        x = words{nothing, nothing, nothing, nothing};
        const auto *from = reinterpret_cast<const words *>(row + at);
        if (at >= 0 && at + kWide<T> <= end) x = ONCE ? __builtin_nontemporal_load(from) : *from;
    }
    __device__ __forceinline__ void load_edge(const T *row, int at, int end) {
        if (at >= end || at + kWide<T> <= 0 || (at >= 0 && at + kWide<T> <= end)) return;
#pragma unroll
        for (int i = 0; i < kWide<T>; ++i) {
            if (at + i < 0 || at + i >= end) continue;
            if constexpr (sizeof(T) == 4) {
                x[i] = reinterpret_cast<const unsigned *>(row)[at + i];
            } else {
                const unsigned one = reinterpret_cast<const unsigned short *>(row)[at + i];
                x[i / 2] = i % 2 ? (x[i / 2] & 0xffffu) | one << 16 : (x[i / 2] & 0xffff0000u) | one;
            }
        }
    }
    template <int USE>
    __device__ __forceinline__ void values(float (&v)[kWide<T>]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) v[i] = __uint_as_float(x[i]);
            else halves<USE>(x[i], v[2 * i], v[2 * i + 1], T());
        }
    }
};

// a whole chunk as it stands in memory
template <typename T, int NV>
struct RawChunk {
    Raw<T> part[NV];
    __device__ __forceinline__ void load(const T *chunk, int lane) {
#pragma unroll
        for (int j = 0; j < NV; ++j) part[j].load(chunk + (j * 64 + lane) * kWide<T>, true);
    }
    template <bool ONCE>
    __device__ __forceinline__ void load_within(const T *row, int begin, int end, int lane) {
#pragma unroll
        for (int j = 0; j < NV; ++j) part[j].template load_within<ONCE>(row, begin + (j * 64 + lane) * kWide<T>, end);
#pragma unroll
        for (int j = 0; j < NV; ++j) part[j].load_edge(row, begin + (j * 64 + lane) * kWide<T>, end);
    }
    __device__ __forceinline__ void values(Chunk<T, NV> &c) const {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            float v[kWide<T>];
            part[j].template values<0>(v);
#pragma unroll
            for (int i = 0; i < kWide<T>; ++i) c.x[j * kWide<T> + i] = v[i];
        }
    }
};

// logits begin .. begin + SPAN of a row, those outside of 0 .. end are -inf
template <bool ONCE, typename T, int NV>
__device__ __forceinline__ void load_chunk(const T *row, int begin, int end, int lane, Chunk<T, NV> &c) {
    RawChunk<T, NV> x;
    x.template load_within<ONCE>(row, begin, end, lane);
    x.values(c);
}

// up to here r - m * c is below 2^-4
constexpr float kMostFused = 1 << 20;

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
// (hands back the lane's largest of the chunk; NaN are no numbers to it)
template <typename T, int NV>
__device__ __forceinline__ float fold(Stats &a, const Chunk<T, NV> &x, float c) {
    float largest = x.x[0];
#pragma unroll
    for (int i = 1; i < Chunk<T, NV>::COUNT; ++i) largest = fmaxf(largest, x.x[i]);
    const float m = fmaxf(a.m, largest), ref = m == kMinusInfinity ? 0.0f : m;
    shift_stats(a, m, ref, c);
#pragma unroll
    for (int i = 0; i < Chunk<T, NV>::COUNT; ++i) {
        const float t = (x.x[i] - ref) * c, e = __builtin_amdgcn_exp2f(t);
        a.s += e;
        a.w = __builtin_fmaf(e, at_least(t), a.w);
    }
    return largest;
}
// t as one fused operation, x * c - r with r = m * c rounded, for 16-bit logits, where instructions and memory bound a pass about equally.  All
// of a chunk's terms are off by the same factor 2^(r - m * c) then, which is known exactly and taken out of the chunk's sums.
template <typename T, int NV>
__device__ __forceinline__ float fold_fused(Stats &a, const Chunk<T, NV> &x, float c) {
    float largest = x.x[0];
#pragma unroll
    for (int i = 1; i < Chunk<T, NV>::COUNT; ++i) largest = fmaxf(largest, x.x[i]);
    const float m = fmaxf(a.m, largest), ref = m == kMinusInfinity ? 0.0f : m, r = ref * c;
    if (__ballot(!(fabsf(r) <= kMostFused))) return fold(a, x, c);
    shift_stats(a, m, ref, c);
    const float off = __builtin_fmaf(ref, c, -r);  // m * c - r
    float s = 0.0f, w = 0.0f;
#pragma unroll
    for (int i = 0; i < Chunk<T, NV>::COUNT; ++i) {
        const float t = __builtin_fmaf(x.x[i], c, -r), e = __builtin_amdgcn_exp2f(t);
        s += e;
        w = __builtin_fmaf(e, at_least(t), w);
    }
    const float f = __builtin_amdgcn_exp2f(-off);
    a.s = __builtin_fmaf(s, f, a.s);
    a.w = __builtin_fmaf(w - s * off, f, a.w);
    return largest;
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
    const float m = max_of<64>(a.m);
    shift_stats(a, m, m == kMinusInfinity ? 0.0f : m, c);
    a.s = sum_of<64>(a.s);
    a.w = sum_of<64>(a.w);
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
// puts an entry to place `rank` < K; the others from there on move one lane up
__device__ __forceinline__ void insert(Best &b, float value, int token, int rank, int K, int lane) {
    const float below_value = __shfl_up(b.value, 1);
    const int below_token = __shfl_up(b.token, 1);
    b.value = lane == rank ? value : lane > rank ? below_value : b.value;
    b.token = lane == rank ? token : lane > rank ? below_token : b.token;
    b.count = min(b.count + 1, K);
    b.least = of_lane(b.value, K - 1);
}
// A chunk's logits that belong into the list, largest first: at most K rounds, each of which takes one logit out of the chunk (c is used
// up).  Most chunks of a long row end in the first test.  Tokens of later chunks are higher, so an equal logit goes behind.
template <typename T, int NV>
__device__ __forceinline__ void take_best(Best &b, Chunk<T, NV> &c, int begin, int end, int K, int lane) {
    constexpr int W = Chunk<T, NV>::W;
    float top[NV], best = __builtin_nanf("");
    if (begin < 0 || begin + Chunk<T, NV>::SPAN > end) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < W; ++i)
                if (begin + (j * 64 + lane) * W + i < 0 || begin + (j * 64 + lane) * W + i >= end) c.x[j * W + i] = __builtin_nanf("");
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
        const float m = max_of<64>(best);
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
// The given token's logit, read in two steps that a kernel has in front of its work (behind it, values and gradient of 32000 rows of 1024 in fp32
// took 48.0 us, 46.4 so).
struct Given {
    int token;  // -1: none, or nobody asks
    float logit;
};
__device__ __forceinline__ int given_token(const RowArgs &a, long n) {
    const int token = a.logp && a.tokens ? a.tokens[n] : -1;
    return token < a.V ? token : -1;
}
template <typename T>
__device__ __forceinline__ Given given_logit(const T *row, int token) { return {token, token >= 0 ? (float)row[token] : 0.0f}; }
// by one lane
__device__ __forceinline__ void write_stats(const RowArgs &a, long n, const Given &g, const Stats &s, float log_s) {
    if (a.logp) a.logp[n] = g.token >= 0 ? logp_of(g.logit, s, a.scale, log_s) : 0.0f;
    if (a.lse) a.lse[n] = s.m * a.scale + log_s;
    if (a.entropy) a.entropy[n] = entropy_of(s, log_s);
}
// alternative `rank` of a row; token -1: there is none
__device__ __forceinline__ void write_top(const RowArgs &a, long n, int rank, float value, int token, const Stats &s, float log_s) {
    if (a.top_logp) a.top_logp[n * a.K + rank] = token < 0 ? __builtin_nanf("") : logp_of(value, s, a.scale, log_s);
    if (a.top_tokens) a.top_tokens[n * a.K + rank] = token;
}

// whole numbers in the order of floats, -0 the same as 0; no number is 0
__device__ __forceinline__ unsigned ordered(float v) {
    const unsigned u = __float_as_uint(v + 0.0f);
    return u ^ ((unsigned)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float of_ordered(unsigned k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }

// ----- short rows: LANES lanes hold a row, COUNT logits each ---------------------------------------------------------------------
// The row is read once and stays in registers, so the maximum is known before the first exponential.  16 lanes per row and not a wave
// where they can hold it: a row's steps across lanes and the rounds of its alternatives are then taken for four rows at a time.
template <typename T, int COUNT, int LANES>
struct ShortRow {
    static constexpr int W = kWide<T>, NV = COUNT / W;
    float x[COUNT];
    static __device__ __forceinline__ int index(int i, int l) { return (i / W * LANES + l) * W + i % W; }
    __device__ __forceinline__ void load(const T *row, int V, int l) {
        Raw<T> part[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j) part[j].template load_within<true>(row, index(j * W, l), V);
        if (V % W) {
#pragma unroll
            for (int j = 0; j < NV; ++j) part[j].load_edge(row, index(j * W, l), V);
        }
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            float v[W];
            part[j].template values<0>(v);
#pragma unroll
            for (int i = 0; i < W; ++i) x[j * W + i] = v[i];
        }
    }
    __device__ __forceinline__ float largest() const {
        float m = x[0];
#pragma unroll
        for (int i = 1; i < COUNT; ++i) m = fmaxf(m, x[i]);
        return m;
    }
    __device__ __forceinline__ Stats stats(float c) const {
        const float m = max_of<LANES>(largest());
        Stats a = {m == m ? m : kMinusInfinity, 0.0f, 0.0f};  // (all NaN)
        const float ref = a.m == kMinusInfinity ? 0.0f : a.m;
#pragma unroll
        for (int i = 0; i < COUNT; ++i) {
            const float t = (x[i] - ref) * c, e = __builtin_amdgcn_exp2f(t);
            a.s += e;
            a.w = __builtin_fmaf(e, at_least(t), a.w);
        }
        a.s = sum_of<LANES>(a.s);
        a.w = sum_of<LANES>(a.w);
        return a;
    }
};

template <typename T, int COUNT, int LANES, bool TOP>
__global__ __launch_bounds__(256) void logprob_short_kernel(const RowArgs a) {
    const int l = threadIdx.x % LANES;
    const long n = (long)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    const bool here = n < a.N;  // (whole groups of lanes)
    const T *row = static_cast<const T *>(a.logits) + (here ? n : 0) * a.stride;
    const int token = here && l == 0 ? given_token(a, n) : -1;
    ShortRow<T, COUNT, LANES> x;
    x.load(row, here ? a.V : 0, l);
    const Given given = given_logit(row, token);
    const Stats s = x.stats(a.scale * kLog2e);
    const float log_s = logf(s.s);
    if (here && l == 0) write_stats(a, n, given, s, log_s);
    if (!TOP) return;
    // K rounds: the largest of what is left, the lowest token where several hold it.  As whole numbers in the order of the logits: their maxima
    // take one instruction per step across lanes.  What is taken, NaN and what is behind the row is 0, which no number is.
    unsigned key[COUNT];
#pragma unroll
    for (int i = 0; i < COUNT; ++i) key[i] = ordered(x.x[i]);
    if (a.V < COUNT * LANES || __ballot(s.s != s.s)) {
#pragma unroll
        for (int i = 0; i < COUNT; ++i) key[i] = x.index(i, l) < a.V && x.x[i] == x.x[i] ? key[i] : 0u;
    }
    unsigned kept = 0;  // result number k stays with lane k % LANES until all lanes have one
    int kept_token = -1;
    for (int k = 0; k < a.K; ++k) {
        unsigned best = key[0];
#pragma unroll
        for (int i = 1; i < COUNT; ++i) best = max(best, key[i]);
        const unsigned most = over_lanes<LANES>(best, [](unsigned p, unsigned q) { return max(p, q); });
        int at = 0;
        bool first[COUNT], seen = false;  // the first of the lane's that hold it
#pragma unroll
        for (int i = 0; i < COUNT; ++i) {
            first[i] = key[i] == most && !seen;
            seen = seen || first[i];
            at = first[i] ? i : at;
        }
        const int own = seen ? x.index(at, l) : INT_MAX, token = min_of<LANES>(own);
        const bool mine = k % LANES == l, last = k + 1 == a.K;
        kept = mine ? most : kept;
        kept_token = mine ? token : kept_token;
        if (here && (last || k % LANES == LANES - 1) && l <= k % LANES)
            write_top(a, n, k / LANES * LANES + l, of_ordered(kept), kept ? kept_token : -1, s, log_s);
        if (last) break;
        const bool owner = own == token;
#pragma unroll
        for (int i = 0; i < COUNT; ++i) key[i] = owner && first[i] ? 0u : key[i];
    }
}

// ----- long rows: a workgroup of one or four waves for a row or a part of one ------------------------------------------------------------
// The best K without keeping them up to date on the way, which at K = 16 took longer than everything else (2047 rows of 100003: 200 us, of
// which a list per wave 130): a lane remembers the largest logit of its best two chunks, and of which chunks, and that of its third.  The
// K-th largest of the lanes' largest is a bound that K logits reach.  Read again are the remembered chunks that reach it, their lane's logits
// only, some 16 K or 32 K of them, and all of a lane whose third chunk reaches it too.  Where ties or sorted rows make that too
// many, the row is read once more with lists.
struct Cells {
    float first, second, third;
    int first_at, second_at;
};
__device__ __forceinline__ void remember(Cells &c, float largest, int at) {
    const bool a = largest > c.first, b = largest > c.second;
    c.third = b ? c.second : fmaxf(c.third, largest);
    c.second_at = a ? c.first_at : b ? at : c.second_at;
    c.second = a ? c.first : b ? largest : c.second;
    c.first_at = a ? at : c.first_at;
    c.first = a ? largest : c.first;
}
// A bound that at least K of a wave's keys reach, and no more than K + kSlack but for equal ones: keys up to COUNT per lane, `entries` in all; 0: there
// are fewer, keys of 0 being none.  Bit by bit between the first and the last that not all keys have in common.
constexpr int kSlack = 8;
template <int COUNT>
__device__ __forceinline__ unsigned bound_of(const unsigned (&key)[COUNT], int entries, int K) {
    unsigned all = ~0u, any = 0;
#pragma unroll
    for (int q = 0; q < COUNT; ++q)
        if (q * 64 < entries) {
            all &= key[q];
            any |= key[q];
        }
    all = over_lanes<64>((int)all, [](int a, int b) { return a & b; });
    any = over_lanes<64>((int)any, [](int a, int b) { return a | b; });
    const unsigned differ = any & ~all;
    const int top = differ ? 31 - __builtin_clz(differ) : -1, last = differ ? __builtin_ctz(differ) : 0;
    unsigned t = top < 0 ? all : all & ~((2u << top) - 1);
    for (int bit = top; bit >= last; --bit) {
        const unsigned more = t | 1u << bit;
        int count = 0;
#pragma unroll
        for (int q = 0; q < COUNT; ++q)
            if (q * 64 < entries) count += __popcll(__ballot(key[q] >= more));
        if (count >= K) t = more;
        if (count >= K && count <= K + kSlack) break;
    }
    return t;
}

// Lanes all of whose chunks are read again (2100 rows of 9000 bf16 logits, K = 16, up to 16 19.3 us, 64 19.5, one lane 39.0; 512 of 131072, K = 32
// 33.4, 33.6 and 104.8).
constexpr int kMostWhole = 16;
template <int WAVES>
struct Shared {
    static constexpr int THREADS = 64 * WAVES, CELLS = WAVES == 1 ? 128 : THREADS, CANDIDATES = WAVES == 1 ? 256 : 512;
    Stats stats[WAVES];
    float first[THREADS], second[THREADS], third[THREADS];
    int first_at[THREADS], second_at[THREADS];
    int cell_lane[CELLS], cell_at[CELLS];
    int whole[kMostWhole];  // lanes (with their waves) all of whose chunks are read again
    unsigned least;
    int cells, wholes, candidates;
    float value[CANDIDATES];
    int token[CANDIDATES];
};

// entry i of a list, at its rank if that is among the first K: f(rank)
template <typename F>
__device__ __forceinline__ void rank_entry(const float *value, const int *token, int count, int i, int K, F f) {
    const float v = value[i];
    const int t = token[i];
    int rank = 0;
    for (int k = 0; k < count; ++k) rank += value[k] > v || (value[k] == v && token[k] < t);
    if (rank < K) f(rank, v, t);
}

// (registers for eight workgroups of a compute unit: with seven, 2047 rows with alternatives took two rounds of the card)
template <typename T, int NV, int WAVES, bool TOP>
__global__ __launch_bounds__(64 * WAVES, 8) void logprob_kernel(const RowArgs a) {
    using X = Chunk<T, NV>;
    using Sh = Shared<WAVES>;
    constexpr int SPAN = X::SPAN, W = X::W, THREADS = 64 * WAVES;
    __shared__ Sh sh;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long n = blockIdx.x;
    const float c = a.scale * kLog2e;
    const T *row = static_cast<const T *>(a.logits) + n * a.stride;
    const int begin = (int)blockIdx.y * a.part - lead_of(row), end = min(a.V, begin + a.part);
    const bool shared_row = a.parts > 1;
    const Given given = given_logit(row, shared_row || threadIdx.x > 0 ? -1 : given_token(a, n));
    Stats s;
    begin_stats(s);
    Cells cells = {kMinusInfinity, kMinusInfinity, kMinusInfinity, -1, -1};
    auto take = [&](const X &x, int at) {
        const float largest = sizeof(T) == 2 ? fold_fused(s, x, c) : fold(s, x, c);
        if (TOP) remember(cells, largest, at);
    };
    // the first chunk, if the row begins within it; whole ones, each asked for while the one before is worked on; the rest of the last one
    auto take_part = [&](int at) {
        X x;
        load_chunk<true>(row, at, end, lane, x);
        take(x, at);
    };
    int at = begin + wave * SPAN;
    if (at < 0) {
        take_part(at);
        at += WAVES * SPAN;
    }
    if (at + SPAN <= end) {
        RawChunk<T, NV> next;
        next.load(row + at, lane);
        while (true) {
            RawChunk<T, NV> now = next;
            const int here = at;
            at += WAVES * SPAN;
            if (at + SPAN <= end) next.load(row + at, lane);
            X x;
            now.values(x);
            take(x, here);
            if (at + SPAN > end) break;
        }
    }
    if (at < end) take_part(at);
    s = join_lanes(s, c);
    if (lane == 0) sh.stats[wave] = s;
    if (TOP) {
        sh.first[threadIdx.x] = cells.first;
        sh.second[threadIdx.x] = cells.second;
        sh.first_at[threadIdx.x] = cells.first_at;
        sh.second_at[threadIdx.x] = cells.second_at;
        sh.third[threadIdx.x] = cells.third;
    }
    __syncthreads();
    s = sh.stats[0];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) s = join(s, sh.stats[w], c);
    const float log_s = logf(s.s);
    const long p = n * a.parts + blockIdx.y;
    if (threadIdx.x == 0) {
        if (shared_row) {
            a.part_stats[p * 3] = s.m;
            a.part_stats[p * 3 + 1] = s.s;
            a.part_stats[p * 3 + 2] = s.w;
        } else {
            write_stats(a, n, given, s, log_s);
        }
    }
    if (!TOP) return;
    auto put = [&](int rank, float value, int token) {
        if (shared_row) {
            a.part_values[p * a.K + rank] = value;
            a.part_tokens[p * a.K + rank] = token;
        } else {
            write_top(a, n, rank, value, token, s, log_s);
        }
    };
    if (wave == 0) {
        unsigned key[WAVES];
#pragma unroll
        for (int w = 0; w < WAVES; ++w) key[w] = ordered(sh.first[w * 64 + lane]);
        const unsigned least = bound_of<WAVES>(key, THREADS, a.K);
        int wholes = 0, count = 0;
#pragma unroll
        for (int q = 0; q < 3 * WAVES; ++q) {  // third, first, second
            const int from = q % WAVES * 64 + lane;
            const bool whole = ordered(sh.third[from]) >= least;
            const bool in = q < WAVES ? whole : !whole && ordered(q < 2 * WAVES ? sh.first[from] : sh.second[from]) >= least;
            const unsigned long long b = __ballot(in);
            const int place = (q < WAVES ? wholes : count) + __popcll(b & ((1ull << lane) - 1));
            if (q < WAVES) {
                if (in && place < kMostWhole) sh.whole[place] = from;
                wholes += __popcll(b);
            } else {
                if (in && place < Sh::CELLS) {
                    sh.cell_lane[place] = lane;
                    sh.cell_at[place] = q < 2 * WAVES ? sh.first_at[from] : sh.second_at[from];
                }
                count += __popcll(b);
            }
        }
        if (lane == 0) {
            sh.least = least;
            sh.cells = wholes <= kMostWhole && count <= Sh::CELLS ? count : -1;
            sh.wholes = wholes;
            sh.candidates = 0;
        }
    }
    __syncthreads();
    const int n_cells = sh.cells;
    bool listed = n_cells < 0;
    if (!listed) {
        const unsigned least = sh.least;
        auto look = [&](int chunk, int of, int vec) {
            const int first = chunk + (vec * 64 + of) * W;
            float v[W];
            fetch_within<false>(row, first, end, v, __builtin_nanf(""));
#pragma unroll
            for (int q = 0; q < W; ++q) {
                if (v[q] == v[q] && ordered(v[q]) >= least) {
                    const int place = atomicAdd(&sh.candidates, 1);
                    if (place < Sh::CANDIDATES) {
                        sh.value[place] = v[q];
                        sh.token[place] = first + q;
                    }
                }
            }
        };
        for (int i = threadIdx.x; i < n_cells * NV; i += THREADS) look(sh.cell_at[i / NV], sh.cell_lane[i / NV], i % NV);
        const int rounds = (end - begin + WAVES * SPAN - 1) / (WAVES * SPAN), each = rounds * NV;
        for (int i = threadIdx.x; i < sh.wholes * each; i += THREADS) {
            const int from = sh.whole[i / each], of = from & 63, in = i % each;
            look(begin + (in / NV * WAVES + from / 64) * SPAN, of, in % NV);
        }
        __syncthreads();
        listed = sh.candidates > Sh::CANDIDATES;
        const int candidates = sh.candidates;
        for (int i = threadIdx.x; !listed && i < candidates; i += THREADS) rank_entry(sh.value, sh.token, candidates, i, a.K, put);
    }
    if (!listed) return;
    // the row again, with a list per wave
    Best b;
    begin_best(b);
    for (int at = begin + wave * SPAN; at < end; at += WAVES * SPAN) {
        X x;
        load_chunk<false>(row, at, end, lane, x);
        take_best(b, x, at, end, a.K, lane);
    }
    __syncthreads();
    float *values = sh.first;  // 64 of each wave
    int *tokens = sh.first_at;
    values[threadIdx.x] = b.value;
    tokens[threadIdx.x] = lane < b.count ? b.token : -1;
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int w = 1; w < WAVES; ++w) merge_best(b, values[w * 64 + lane], tokens[w * 64 + lane], a.K, lane);
    if (lane < a.K) put(lane, b.value, lane < b.count ? b.token : -1);
}

// The parts of a row, by a wave: up to Q * 64 alternatives of all parts.
template <typename T, int Q>
__global__ __launch_bounds__(64) void logprob_join_kernel(const RowArgs a) {
    __shared__ float value[Q * 64];
    __shared__ int token[Q * 64];
    const long n = blockIdx.x;
    const int lane = threadIdx.x;
    const float c = a.scale * kLog2e;
    Stats s;
    begin_stats(s);
    const long p = n * a.parts;
    const int given_one = given_token(a, n);
    if (lane < a.parts) s = {a.part_stats[(p + lane) * 3], a.part_stats[(p + lane) * 3 + 1], a.part_stats[(p + lane) * 3 + 2]};
    float v[Q];
    int t[Q];
    const int entries = a.parts * a.K;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        const int i = q * 64 + lane;
        v[q] = i < entries ? a.part_values[p * a.K + i] : 0.0f;
        t[q] = i < entries ? a.part_tokens[p * a.K + i] : -1;
    }
    const Given given = given_logit(static_cast<const T *>(a.logits) + n * a.stride, given_one);
    s = join_lanes(s, c);
    const float log_s = logf(s.s);
    if (lane == 0) {
        write_stats(a, n, given, s, log_s);
        // for the errors of the joint call (all lanes' statistics have been read: they are in these two)
        a.part_stats[p * 3] = s.m;
        a.part_stats[p * 3 + 1] = log_s;
    }
    if (a.K == 0) return;
    unsigned key[Q];
#pragma unroll
    for (int q = 0; q < Q; ++q) key[q] = t[q] >= 0 ? ordered(v[q]) : 0u;
    const unsigned least = max(1u, bound_of<Q>(key, entries, a.K));
    int count = 0;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        const unsigned long long b = __ballot(key[q] >= least);
        const int place = count + __popcll(b & ((1ull << lane) - 1));
        if (key[q] >= least) {
            value[place] = v[q];
            token[place] = t[q];
        }
        count += __popcll(b);
    }
    __syncthreads();
    for (int i = lane; i < count; i += 64)
        rank_entry(value, token, count, i, a.K, [&](int rank, float x, int y) { write_top(a, n, rank, x, y, s, log_s); });
    for (int i = count + lane; i < a.K; i += 64) write_top(a, n, i, 0.0f, -1, s, log_s);  // NaN took the others' places
}

// ----- gradient ----------------------------------------------------------------------------------------------------------------
// err = p * (first + second * t), t = log2 p, and `given` more at the token
struct Slopes {
    float first, second, given;
    int token;
};
// sum: log s of a row, or its saved log sum: -inf where there is nothing to choose from, NaN where there are no numbers.  (The log sum of a
// row whose maximum is known says neither: it may be beyond 32 bits.)
__device__ __forceinline__ Slopes slopes_of(const RowArgs &a, long n, float sum, float entropy) {
    int token = a.tokens ? a.tokens[n] : -1;
    if (token >= a.V || token < 0) token = -1;
    const float error = a.logp_err ? a.logp_err[n] : 0.0f;  // (not waiting for the token)
    const float g = token >= 0 ? error : 0.0f, h = a.entropy_err ? a.entropy_err[n] : 0.0f;
    Slopes s;
    s.first = -a.scale * (h == 0.0f ? g : g + h * entropy);
    s.second = -a.scale * h * kLn2;
    s.given = a.scale * g;
    s.token = sum == kMinusInfinity ? -1 : token;  // nothing to choose from: no gradient
    if (sum != sum) s.first = sum;
    return s;
}
// the given token's own error, if it is one of W from logit `at` on
template <int W>
__device__ __forceinline__ void add_given(int at, const Slopes &s, float (&v)[W]) {
    if ((unsigned)(s.token - at) < (unsigned)W) {
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] += s.token - at == i ? s.given : 0.0f;
    }
}
// W errors of a row from logit `at` on in the place of log2 of the probabilities
template <int W>
__device__ __forceinline__ void errors_of(int at, const Slopes &s, float (&t)[W]) {
#pragma unroll
    for (int i = 0; i < W; ++i) {
        // (a saved log sum in 32 bits may be off by more than 128: no probability is above 1)
        const float u = __builtin_amdgcn_fmed3f(t[i], -1000.0f, 0.0f);
        t[i] = __builtin_amdgcn_exp2f(u) * __builtin_fmaf(s.second, u, s.first);
    }
    add_given<W>(at, s, t);
}
template <typename T, int W>
__device__ __forceinline__ void put_errors(T *row, int at, int end, const Slopes &s, float (&t)[W]) {
    errors_of<W>(at, s, t);
    put_within(row, at, end, t);
}
template <typename T, int NV>
__device__ __forceinline__ void put_gradient(T *row, int begin, int end, int lane, const Slopes &s, const Chunk<T, NV> &t) {
    constexpr int W = Chunk<T, NV>::W;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        float v[W];
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] = t.x[j * W + i];
        put_errors<T, W>(row, begin + (j * 64 + lane) * W, end, s, v);
    }
}

// From saved statistics, `parts` waves for a row, neighbouring ones for neighbouring stretches (rows of 32000 16-bit logits dealt row by row
// instead: 75 us for 3001; workgroups that have one row each: 55 us for
// 6517 of 9819, 47 so).  A wave has one chunk but in very long rows.
// JOINED: the rows of a joint call that are shared out, from their maximum and log s apart, as the other forms of that call have them: rows far from zero
// have a log sum that 32 bits round by more than its logits differ (a row of the type's lowest value: p = 1 for 1 / V).  Four rows of 131072 bf16 13.6 us
// in all three launches, 13.7 from the log sum; 511 of 140001 76.3 and 76.2.
template <typename T, int NV, bool JOINED>
__global__ __launch_bounds__(256) void logprob_gradient_kernel(const RowArgs a, int forward_parts) {
    constexpr int SPAN = Chunk<T, NV>::SPAN, W = kWide<T>;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const unsigned id = blockIdx.x * 4 + wave;
    const long n = id / (unsigned)a.parts;
    const int stretch = id % (unsigned)a.parts;
    if (n >= a.N) return;
    const T *row = static_cast<const T *>(a.logits) + n * a.stride;
    T *to = static_cast<T *>(a.err) + n * a.err_stride;
    const float *joined = JOINED ? a.part_stats + n * forward_parts * 3 : nullptr;
    const float c = a.scale * kLog2e;
    auto errors = [&](float (&t)[W], int at, float ref, float log2_s, const Slopes &s) {
#pragma unroll
        for (int i = 0; i < W; ++i) t[i] = JOINED ? (t[i] - ref) * c - log2_s : __builtin_fmaf(t[i], a.scale, -ref) * kLog2e;
        errors_of<W>(at, s, t);
    };
    for (int at = stretch * SPAN - lead_of(row); at < a.V; at += a.parts * SPAN) {
        const bool whole = at >= 0 && at + SPAN <= a.V;
        RawChunk<T, NV> x;  // (asked for in front of the row's values)
        if (whole) x.load(row + at, lane);
        else x.template load_within<true>(row, at, a.V, lane);
        const float base = JOINED ? joined[0] : a.lse[n], sum = JOINED ? joined[1] : base, ref = base == kMinusInfinity ? 0.0f : base;
        const Slopes s = slopes_of(a, n, sum, a.entropy ? a.entropy[n] : 0.0f);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int first = at + (j * 64 + lane) * W;
            float t[W];
            x.part[j].template values<0>(t);
            errors(t, first, ref, sum * kLog2e, s);
            if (whole) put_elements<T, W, true>(to + first, t);
            else put_within(to, first, a.V, t);
        }
    }
}

// The same for rows that a wave or 16 lanes hold (a workgroup for each of 38270 rows of 41 16-bit logits: 57 us).
template <typename T, int COUNT, int LANES>
__global__ __launch_bounds__(256) void logprob_short_gradient_kernel(const RowArgs a) {
    using X = ShortRow<T, COUNT, LANES>;
    constexpr int W = X::W;
    const int l = threadIdx.x % LANES;
    const long n = (long)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    if (n >= a.N) return;
    X x;
    x.load(static_cast<const T *>(a.logits) + n * a.stride, a.V, l);
    const float lse = a.lse[n], ref = lse == kMinusInfinity ? 0.0f : lse;
    const Slopes slopes = slopes_of(a, n, lse, a.entropy ? a.entropy[n] : 0.0f);
    T *to = static_cast<T *>(a.err) + n * a.err_stride;
#pragma unroll
    for (int j = 0; j < X::NV; ++j) {
        float t[W];
#pragma unroll
        for (int i = 0; i < W; ++i) t[i] = __builtin_fmaf(x.x[j * W + i], a.scale, -ref) * kLog2e;
        put_errors<T, W>(to, (j * LANES + l) * W, a.V, slopes, t);
    }
}

template <typename T, int COUNT, int LANES>
__global__ __launch_bounds__(256) void logprob_short_error_kernel(const RowArgs a) {
    using X = ShortRow<T, COUNT, LANES>;
    constexpr int W = X::W;
    const int l = threadIdx.x % LANES;
    const long n = (long)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    const bool here = n < a.N;
    const float c = a.scale * kLog2e;
    const T *row = static_cast<const T *>(a.logits) + (here ? n : 0) * a.stride;
    const int token = here && l == 0 ? given_token(a, n) : -1;
    X x;
    x.load(row, here ? a.V : 0, l);
    const Given given = given_logit(row, token);
    const Stats s = x.stats(c);
    if (!here) return;
    const float log_s = logf(s.s), log2_s = log_s * kLog2e;
    if (l == 0) write_stats(a, n, given, s, log_s);
    const Slopes slopes = slopes_of(a, n, log_s, entropy_of(s, log_s));
    const float ref = s.m == kMinusInfinity ? 0.0f : s.m;
    T *to = static_cast<T *>(a.err) + n * a.err_stride;
#pragma unroll
    for (int j = 0; j < X::NV; ++j) {
        float t[W];
#pragma unroll
        for (int i = 0; i < W; ++i) t[i] = (x.x[j * W + i] - ref) * c - log2_s;
        put_errors<T, W>(to, (j * LANES + l) * W, a.V, slopes, t);
    }
}

// A long row that a workgroup of THREADS holds in registers, NV vectors per thread: read once, written once.  GROUPS: workgroups that a compute
// unit has registers for, so that one's loads and stores go on while another computes.
template <typename T, int NV, int THREADS, int GROUPS>
__global__ __launch_bounds__(THREADS, GROUPS * THREADS / 256) void logprob_held_error_kernel(const RowArgs a) {
    constexpr int W = kWide<T>, WAVES = THREADS / 64;
    __shared__ float maxima[WAVES], sums[WAVES], means[WAVES], given;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long n = blockIdx.x;
    const float c = a.scale * kLog2e;
    const T *row = static_cast<const T *>(a.logits) + n * a.stride;
    T *to = static_cast<T *>(a.err) + n * a.err_stride;
    const int token = a.tokens ? __builtin_amdgcn_readfirstlane(a.tokens[n]) : -1;
    // the row's whole vectors; what stands in front of and behind them, a logit for each of the first threads of two waves
    const int lead = lead_of(row);
    Raw<T> x[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int at = (j * THREADS + (int)threadIdx.x) * W - lead;
        x[j].load(row + at, at >= 0 && at + W <= a.V);
    }
    const int front = (W - lead % W) % W;
    int other = wave == 0 && lane < front ? lane : -1;
    if (wave == 1 && lane < (a.V - front) % W) other = front + (a.V - front) / W * W + lane;
    const float rest = other >= 0 ? (float)row[other] : kMinusInfinity;
    // The vectors one after another: quick(j, at, v) for those that all threads have, if `use_quick`, else slow(j, at, v) for those that the row
    // fills.  Both questions are the whole wave's: in front of single instructions they took a fifth of the kernel's time.
    auto for_vectors = [&](auto use, bool use_quick, auto quick, auto slow) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int first = j * THREADS * W - lead, at = first + (int)threadIdx.x * W;
            float v[W];
            if (use_quick && first >= 0 && first + THREADS * W <= a.V) {
                x[j].template values<use.value>(v);
                quick(j, at, v);
            } else if (at >= 0 && at + W <= a.V) {
                x[j].template values<use.value>(v);
                slow(j, at, v);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    float m = rest, low = 0.0f;
    auto look = [&](int, int, const float (&v)[W]) {
#pragma unroll
        for (int i = 0; i < W; ++i) {
            m = fmaxf(m, v[i]);
            low = fminf(low, v[i]);
        }
    };
    for_vectors(std::integral_constant<int, 1>(), true, look, look);
    m = max_of<64>(m);
    if (lane == 0) maxima[wave] = m;
    // the errors may take the logits' place: the given token's logit is kept before any of them is written
    if (threadIdx.x == 0 && token >= 0 && token < a.V) given = (float)row[token];
    __syncthreads();
    const int w = lane % 16;  // every 16 lanes add the waves up
    m = of_lane(max_of<16>(w < WAVES ? maxima[w] : kMinusInfinity), 0);
    m = m == m ? m : kMinusInfinity;  // (all NaN)
    const float ref = m == kMinusInfinity ? 0.0f : m, r = ref * c;
    // (see fold_fused; the whole workgroup has one maximum here)
    const bool fused = sizeof(T) == 2 && fabsf(r) <= kMostFused;
    const float off = fused ? __builtin_fmaf(ref, c, -r) : 0.0f;
    const float t_rest = fused ? __builtin_fmaf(rest, c, -r) : (rest - ref) * c, e_rest = __builtin_amdgcn_exp2f(t_rest);
    Stats s = {m, e_rest, e_rest * at_least(t_rest)};
    // Logits whose t is -inf, which have to be kept from 0 * -inf, are looked for once: most waves have none.
    const bool ruled_out = __ballot((low - ref) * c < -1e38f) != 0;
    for_vectors(std::integral_constant<int, 2>(), !ruled_out && (sizeof(T) == 4 || fused),
        [&](int, int, const float (&v)[W]) {
#pragma unroll
            for (int i = 0; i < W; ++i) {
                const float t = sizeof(T) == 2 ? __builtin_fmaf(v[i], c, -r) : (v[i] - ref) * c, e = __builtin_amdgcn_exp2f(t);
                s.s += e;
                s.w = __builtin_fmaf(e, t, s.w);
            }
        },
        [&](int, int, const float (&v)[W]) {
#pragma unroll
            for (int i = 0; i < W; ++i) {
                const float t = fused ? __builtin_fmaf(v[i], c, -r) : (v[i] - ref) * c, e = __builtin_amdgcn_exp2f(t);
                s.s += e;
                s.w = __builtin_fmaf(e, at_least(t), s.w);
            }
        });
    s.s = sum_of<64>(s.s);
    s.w = sum_of<64>(s.w);
    if (lane == 0) {
        sums[wave] = s.s;
        means[wave] = s.w;
    }
    __syncthreads();
    s.s = of_lane(sum_of<16>(w < WAVES ? sums[w] : 0.0f), 0);
    s.w = of_lane(sum_of<16>(w < WAVES ? means[w] : 0.0f), 0);
    if (fused) {
        const float f = __builtin_amdgcn_exp2f(-off);
        s.w = (s.w - s.s * off) * f;
        s.s *= f;
    }
    const float log_s = logf(s.s), log2_s = log_s * kLog2e, entropy = entropy_of(s, log_s), lse = s.m * a.scale + log_s;
    if (threadIdx.x == 0) {
        if (a.logp) a.logp[n] = token >= 0 && token < a.V ? logp_of(given, s, a.scale, log_s) : 0.0f;
        a.lse[n] = lse;
        a.entropy[n] = entropy;
    }
    const Slopes slopes = slopes_of(a, n, log_s, entropy);
    // 16-bit errors take log2 p = x * c - z from one operation: below 64 z is rounded by 2^-18, the results by 2^-9 or 2^-12
    const float z = r + (log2_s + off);
    const int holder = (slopes.token + lead) / (THREADS * W);
    // second * t, which has no bound on t here, has to be a number where the probability is 0: far masks, large scales, large errors
    const bool numbers = __ballot(!(fabsf(slopes.second) * ((ref - low) * c + log2_s) < 1e38f)) == 0;
    for_vectors(std::integral_constant<int, 3>(), !ruled_out && numbers && (sizeof(T) == 4 || (fused && fabsf(z) <= 64.0f)),
        [&](int j, int at, float (&t)[W]) {
#pragma unroll
            for (int i = 0; i < W; ++i) {
                t[i] = sizeof(T) == 2 ? __builtin_fmaf(t[i], c, -z) : (t[i] - ref) * c - log2_s;
                t[i] = __builtin_amdgcn_exp2f(t[i]) * __builtin_fmaf(slopes.second, t[i], slopes.first);
            }
            if (j == holder) add_given<W>(at, slopes, t);
            put_elements<T, W, true>(to + at, t);
        },
        [&](int, int at, float (&t)[W]) {
#pragma unroll
            for (int i = 0; i < W; ++i) t[i] = (t[i] - ref) * c - log2_s;
            errors_of<W>(at, slopes, t);
            put_elements<T, W, true>(to + at, t);
        });
    if (other >= 0) {
        float t[1] = {(rest - ref) * c - log2_s};
        errors_of<1>(other, slopes, t);
        to[other] = (T)t[0];
    }
}

// Longer rows: a workgroup of 16 waves reads the row twice, the second time mostly from the caches.
template <typename T, int NV>
__global__ __launch_bounds__(1024) void logprob_long_error_kernel(const RowArgs a) {
    constexpr int SPAN = Chunk<T, NV>::SPAN, WAVES = 16;
    __shared__ Stats stats[WAVES];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long n = blockIdx.x;
    const float c = a.scale * kLog2e;
    const T *row = static_cast<const T *>(a.logits) + n * a.stride;
    T *to = static_cast<T *>(a.err) + n * a.err_stride;
    const Given given = given_logit(row, threadIdx.x == 0 ? given_token(a, n) : -1);
    Stats s;
    begin_stats(s);
    Chunk<T, NV> x;
    for (int at = wave * SPAN - lead_of(row); at < a.V; at += WAVES * SPAN) {
        load_chunk<false>(row, at, a.V, lane, x);
        fold(s, x, c);
    }
    s = join_lanes(s, c);
    if (lane == 0) stats[wave] = s;
    __syncthreads();
    s = stats[0];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) s = join(s, stats[w], c);
    const float log_s = logf(s.s), log2_s = log_s * kLog2e;
    if (threadIdx.x == 0) write_stats(a, n, given, s, log_s);
    __syncthreads();  // the errors may take the logits' place: the given token's logit has been read
    const Slopes slopes = slopes_of(a, n, log_s, entropy_of(s, log_s));
    const float ref = s.m == kMinusInfinity ? 0.0f : s.m;
    for (int at = wave * SPAN - lead_of(row); at < a.V; at += WAVES * SPAN) {
        load_chunk<true>(row, at, a.V, lane, x);
#pragma unroll
        for (int i = 0; i < Chunk<T, NV>::COUNT; ++i) x.x[i] = (x.x[i] - ref) * c - log2_s;
        put_gradient(to, at, a.V, lane, slopes, x);
    }
}

// ----- launches ------------------------------------------------------------------------------------------------------------------
// A row of this many logits has room in the registers of a wave.
constexpr int kSpan = 64 * 32;
// Logits of a long row that a workgroup takes at a time: 16 for every lane.
constexpr int kChunk = 16, kRound = 256 * kChunk;
// Bytes of a row that the largest workgroup's registers hold with its errors' work.
constexpr int kMostHeld = 1024 * 16 * 16;

// Which kernel takes the rows; measured on 32000 rows of up to 1000 logits, 20000 of 1975, 16384 of 3000 and 8192 of 10000, us:
//   a row in registers, K rounds (HELD) against a wave that streams a row (WAVE): 500 logits, K = 8 34 / 47, 16 55 / 52, 32 96 / 66;
//   1000, K = 2 31 / 43, 8 58 / 48, 32 183 / 70; 1975, K = 1 37 / 35, 4 50 / 38, 32 217 / 57; 256, K = 16 31 / 41, 64 100 / 359
//   four waves for a row (GROUP) against WAVE: 1975, K = 64 161 / 326 (HELD 415); 3000, K = 0 29 / 23, 16 80 / 38, 64 123 / 278; 10000,
//   K = 16 56 / 41, 64 78 / 266; 4096 rows of 30000, K = 16 55 / 53
// A wave bounds its alternatives by 64 lanes, four by 256: beyond 32 alternatives too many logits reach a wave's bound.
enum Form { HELD, WAVE, GROUP };
constexpr int kWaveTop = 32;
Form form_of(long N, int V, int K) {
    const bool wave = K <= kWaveTop;
    if (V <= 256) return HELD;
    if (V <= 512) return K > 16 && wave ? WAVE : HELD;
    if (V <= 1024) return K >= 8 && wave ? WAVE : HELD;
    if (V <= kSpan) return K <= 1 ? HELD : wave ? WAVE : GROUP;
    return N >= 2048 && V <= 16384 && wave ? WAVE : GROUP;
}
// Parts of a row: enough workgroups for the card where there are few rows, each with a chunk per wave at least, as many as a wave can join.
// From 512 rows on a workgroup has a row (bf16, K = 8, in parts / one each: 200 rows of 100003 21.1 us / -, 300 24.5 / 25.6, 400 27.7 / 26.4, 700 36.7 /
// 31.8, 1000 46.6 / 39.3; 300 rows of 20000 16.5 / 11.2, 511 18.5 / 11.8, 700 19.4 / 13.0).
int parts_of(long N, int V, int K) {
    if (V <= kSpan || N == 0 || N >= 512) return 1;
    return (int)std::min({64L, (V + kRound - 1L) / kRound, (1023 + N) / N, K > 0 ? (long)kMostJoined / K : 64L});
}

// f(COUNT, LANES) for a short row
template <typename F>
void with_lanes(int V, F f) {
    using std::integral_constant;
    if (V <= 128) f(integral_constant<int, 8>(), integral_constant<int, 16>());
    else if (V <= 256) f(integral_constant<int, 16>(), integral_constant<int, 16>());
    else if (V <= 512) f(integral_constant<int, 32>(), integral_constant<int, 16>());
    else if (V <= 1024) f(integral_constant<int, 16>(), integral_constant<int, 64>());
    else f(integral_constant<int, 32>(), integral_constant<int, 64>());
}

// The same for a row's values and errors, which have no alternatives to look for: up to twice as long where there are many 16-bit ones (20000 rows of
// 4000 fp16 logits 62 us, 77 by a workgroup for each; 400 of bf16 5.9 and 5.4; 20000 of 4001 fp32 logits 118 and 108).
template <typename T>
int most_in_wave(long N) { return sizeof(T) == 2 && N >= 2048 ? 2 * kSpan : kSpan; }
template <typename T, typename F>
void with_error_lanes(int V, F f) {
    using std::integral_constant;
    if constexpr (sizeof(T) == 2) {
        if (V > kSpan) {
            f(integral_constant<int, 64>(), integral_constant<int, 64>());
            return;
        }
    }
    with_lanes(V, f);
}

// Whether a row's values and errors are shared out among workgroups, in three launches: rows that no workgroup's registers hold, and the longest of
// very few (one of 64000 fp32 logits 8.7 us, 10.5 by one workgroup; of 32000 8.8 and 6.8; 150 of 64000 25 and 18).
bool shared_errors(long N, int V, int type) {
    return parts_of(N, V, 0) > 1 && (V > kMostHeld / (int)element_size(type) - 128 || (V > 48 * 1024 && N < 64));
}

size_t scratch_of(long N, int V, int K) {
    const int parts = parts_of(N, V, K);
    return parts == 1 ? 0 : (size_t)N * parts * (3 + 2 * (size_t)K) * sizeof(float);
}
// where a shared row's statistics and lists are
void lay_out(RowArgs &a, void *scratch) {
    const size_t p = (size_t)a.N * a.parts;
    a.part_stats = static_cast<float *>(scratch);
    a.part_values = a.part_stats + p * 3;
    a.part_tokens = reinterpret_cast<int *>(a.part_values + p * a.K);
    // a part is a whole number of its waves' rounds
    a.part = ((a.V + 63 + a.parts - 1) / a.parts + kRound - 1) / kRound * kRound;
}

int forward(hipStream_t stream, int type, RowArgs &a, void *scratch) {
    a.parts = parts_of(a.N, a.V, a.K);
    lay_out(a, scratch);
    with_type(type, [&](auto t) {
        using T = typename decltype(t)::type;
        const Form form = form_of(a.N, a.V, a.K);
        if (form == HELD) {
            with_lanes(a.V, [&](auto count, auto lanes) {
                constexpr int COUNT = decltype(count)::value, LANES = decltype(lanes)::value;
                const dim3 grid((unsigned)((a.N + 256 / LANES - 1) / (256 / LANES)));
                auto kernel = a.K > 0 ? logprob_short_kernel<T, COUNT, LANES, true> : logprob_short_kernel<T, COUNT, LANES, false>;
                hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, a);
            });
        } else {
            constexpr int NV = kChunk / kWide<T>;
            auto four = a.K > 0 ? logprob_kernel<T, NV, 4, true> : logprob_kernel<T, NV, 4, false>;
            auto one = a.K > 0 ? logprob_kernel<T, NV, 1, true> : logprob_kernel<T, NV, 1, false>;
            const dim3 grid((unsigned)a.N, (unsigned)a.parts);
            if (form == WAVE) hipLaunchKernelGGL(one, grid, dim3(64), 0, stream, a);
            else hipLaunchKernelGGL(four, grid, dim3(256), 0, stream, a);
            auto joined = a.parts * a.K <= 256 ? logprob_join_kernel<T, 4> : logprob_join_kernel<T, kMostJoined / 64>;
            if (a.parts > 1) hipLaunchKernelGGL(joined, dim3((unsigned)a.N), dim3(64), 0, stream, a);
        }
    });
    CNT_HIP(hipGetLastError());
    return CNT_OK;
}

// forward_parts: of a joint call, the parts of a row whose statistics the forward launches have left in scratch; else 0
int gradient(hipStream_t stream, int type, RowArgs &a, int forward_parts) {
    a.parts = (int)std::min({4096L, ((1L << 26) - 4) / a.N, (a.V + 63L + kSpan - 1) / kSpan});
    with_type(type, [&](auto t) {
        using T = typename decltype(t)::type;
        if (a.V <= kSpan) {  // (none of a joint call's shared rows)
            with_lanes(a.V, [&](auto count, auto lanes) {
                constexpr int COUNT = decltype(count)::value, LANES = decltype(lanes)::value;
                const dim3 grid((unsigned)((a.N + 256 / LANES - 1) / (256 / LANES)));
                hipLaunchKernelGGL((logprob_short_gradient_kernel<T, COUNT, LANES>), grid, dim3(256), 0, stream, a);
            });
            return;
        }
        auto kernel = forward_parts ? logprob_gradient_kernel<T, 32 / kWide<T>, true> : logprob_gradient_kernel<T, 32 / kWide<T>, false>;
        hipLaunchKernelGGL(kernel, dim3((unsigned)((a.N * a.parts + 3) / 4)), dim3(256), 0, stream, a, forward_parts);
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
    CNT_REQUIRE(scale >= 1e-30f && scale <= 1e30f, "%s: the scale has to be within 1e-30 .. 1e30", who);
    return CNT_OK;
}
// the errors' rows, which may be the logits' own places and overlap them in no other way
int check_errors(const char *who, long N, int V, int type, const void *logits, long stride, const void *err, long err_stride) {
    CNT_REQUIRE(err_stride >= V, "%s: rows of the errors overlap", who);
    if (N == 0) return CNT_OK;
    const uintptr_t size = element_size(type), from = reinterpret_cast<uintptr_t>(logits), to = reinterpret_cast<uintptr_t>(err);
    const uintptr_t from_end = from + ((N - 1) * stride + V) * size, to_end = to + ((N - 1) * err_stride + V) * size;
    CNT_REQUIRE(from_end <= to || to_end <= from || (from == to && (stride == err_stride || N == 1)),
                "%s: the errors overlap the logits without being in their places", who);
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
    CNT_REQUIRE(N == 0 || (lse && err), "logprob_backward: null argument");
    CNT_TRY(check_errors("logprob_backward", N, V, type, logits, stride, err, err_stride));
    CNT_REQUIRE(!entropy_err || entropy || N == 0, "logprob_backward: errors of entropies without the entropies");
    CNT_REQUIRE(!logp_err || tokens || N == 0, "logprob_backward: errors of log probabilities of which tokens?");
    if (N == 0) return CNT_OK;
    RowArgs a = {};
    a.logits = logits; a.stride = stride; a.tokens = tokens; a.N = N; a.V = V; a.scale = scale;
    a.lse = const_cast<float *>(lse); a.entropy = const_cast<float *>(entropy);
    a.logp_err = logp_err; a.entropy_err = entropy_err; a.err = err; a.err_stride = err_stride;
    ProfileScope prof(static_cast<hipStream_t>(stream_), "logprob_backward");
    return gradient(static_cast<hipStream_t>(stream_), type, a, 0);
}

int cnt_logprob_error_backward(void *stream_, long N, int V, int type, const void *logits, long stride, float scale, const int *tokens,
                               const float *logp_err, const float *entropy_err, float *logp, float *lse, float *entropy, void *err,
                               long err_stride, void *scratch, size_t scratch_bytes) {
    using namespace cnt;
    CNT_TRY(check_rows("logprob_error_backward", N, V, type, logits, stride, scale));
    CNT_REQUIRE(N == 0 || (err && lse && entropy), "logprob_error_backward: null argument");
    CNT_TRY(check_errors("logprob_error_backward", N, V, type, logits, stride, err, err_stride));
    CNT_REQUIRE((!logp_err && !logp) || tokens || N == 0, "logprob_error_backward: log probabilities of which tokens?");
    CNT_TRY(check_scratch("logprob_error_backward", N, V, 0, scratch, scratch_bytes));
    if (N == 0) return CNT_OK;
    RowArgs a = {};
    a.logits = logits; a.stride = stride; a.tokens = tokens; a.N = N; a.V = V; a.scale = scale;
    a.logp = logp; a.lse = lse; a.entropy = entropy;
    a.logp_err = logp_err; a.entropy_err = entropy_err; a.err = err; a.err_stride = err_stride;
    // a launch has fewer than 2^32 threads: 1024 for a row beyond 64 KB, 512 beyond 32 KB (less what it may begin by inside a cache line)
    const long row_bytes = V * (long)element_size(type) + 128;
    CNT_REQUIRE(N < 1L << (row_bytes > 1 << 16 ? 22 : row_bytes > 1 << 15 ? 23 : 24), "logprob_error_backward: too many rows of this length");
    hipStream_t stream = static_cast<hipStream_t>(stream_);
    ProfileScope prof(stream, "logprob_error_backward");
    if (shared_errors(N, V, type)) {
        CNT_TRY(forward(stream, type, a, scratch));
        return gradient(stream, type, a, a.parts);
    }
    with_type(type, [&](auto t) {
        using T = typename decltype(t)::type;
        constexpr int W = kWide<T>;
        const dim3 rows((unsigned)N);
        // what rows may begin inside a cache line by (lead_of)
        const bool lines = reinterpret_cast<uintptr_t>(logits) % 128 == 0 && (stride * (long)sizeof(T) % 128 == 0 || N == 1);
        const int lead = lines ? 0 : 127 / (int)sizeof(T);
        if (V <= most_in_wave<T>(N)) {
            with_error_lanes<T>(V, [&](auto count, auto lanes) {
                constexpr int COUNT = decltype(count)::value, LANES = decltype(lanes)::value;
                const dim3 grid((unsigned)((N + 256 / LANES - 1) / (256 / LANES)));
                hipLaunchKernelGGL((logprob_short_error_kernel<T, COUNT, LANES>), grid, dim3(256), 0, stream, a);
            });
        } else if (V <= 256 * 4 * W - lead) {
            hipLaunchKernelGGL((logprob_held_error_kernel<T, 4, 256, 4>), rows, dim3(256), 0, stream, a);
        } else if (V <= 256 * 8 * W - lead) {
            hipLaunchKernelGGL((logprob_held_error_kernel<T, 8, 256, 4>), rows, dim3(256), 0, stream, a);
        } else if (V <= 512 * 8 * W - lead) {
            hipLaunchKernelGGL((logprob_held_error_kernel<T, 8, 512, 3>), rows, dim3(512), 0, stream, a);
        } else if (V <= 1024 * 8 * W - lead) {
            hipLaunchKernelGGL((logprob_held_error_kernel<T, 8, 1024, 2>), rows, dim3(1024), 0, stream, a);
        } else if (V <= 1024 * 16 * W - lead) {
            hipLaunchKernelGGL((logprob_held_error_kernel<T, 16, 1024, 1>), rows, dim3(1024), 0, stream, a);
        } else {
            hipLaunchKernelGGL((logprob_long_error_kernel<T, 32 / W>), rows, dim3(1024), 0, stream, a);
        }
    });
    CNT_HIP(hipGetLastError());
    return CNT_OK;
}

}  // extern "C"
