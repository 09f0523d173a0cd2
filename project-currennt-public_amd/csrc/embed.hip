// Rows of a table looked up by token and scaled, and the table's gradient.
//
//   out[n] = scale * table[token[n]]                       (zero where slot n has no token)
//   grad[v] = scale * sum over the slots n of token v of err[n]    (+ what grad held, if asked)
//
// Both move rows and are bounded by memory; small gradients by launches that wait for each other.  A gradient's sums are formed in 32 bits, in an
// order that the tokens alone determine, without atomics and without clearing the table first.  Three ways:
//   up to 128 slots: every workgroup looks for its rows' slots among all of them
//   slabs of 512 slots, sorted and added up by a workgroup each, for small and middle tables and lists
//   else a stable counting sort of the slots by token (one or two passes of at most ten bits, three beyond 2^20 rows), which makes a token's slots
//   neighbours; a run that covers whole pieces of the sorted list (tokens are as skewed as in any text) is added up piece by piece first
#include "elements.hpp"

#include <algorithm>
#include <cmath>

namespace cnt {
namespace {

// ----- lookup ---------------------------------------------------------------------------------------------------------------
struct LookupArgs {
    const void *table;
    void *out;
    const int *tokens;
    long N, table_stride, out_stride;
    int V, D, lanes, lead;  // threads that share a row; values by which its rows may begin behind a line's begin
    float scale;
};

constexpr int kSlotsPerThread = 4, kLine = 128;

// A thread has the same columns of several slots, whose tokens and then rows it asks for together.  The output's rows are dealt to threads in vectors
// from a cache line's begin on; not LINES: rows that begin inside a line (33222 rows of 1204, bf16 to fp32, 36 us, dealt from the rows' begins 44; the
// questions that this asks are spared for the others, 16 rows of 4096 4.4 us and 6.2).
template <typename T, typename O, bool LINES>
__global__ __launch_bounds__(256) void embed_lookup_kernel(const LookupArgs a) {
    constexpr int W = kBoth<T, O>, U = kSlotsPerThread;
    const int rows = 256 / a.lanes;
    const long n = (long)blockIdx.x * (rows * U) + threadIdx.x / a.lanes;
    const bool whole = a.D >= W;
    bool held[U];
    const T *from[U];
    O *to[U];
    int lead[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int token = n + u * rows < a.N ? a.tokens[n + u * rows] : -1;
        held[u] = token >= 0 && token < a.V;
        from[u] = static_cast<const T *>(a.table) + (held[u] ? token : 0) * a.table_stride;
        to[u] = static_cast<O *>(a.out) + (n + u * rows) * a.out_stride;
        lead[u] = LINES ? 0 : (int)(reinterpret_cast<uintptr_t>(to[u]) % kLine / sizeof(O));
    }
    for (int k = (threadIdx.x % a.lanes) * W; k < a.D + a.lead; k += a.lanes * W) {
        Vector<T, W> x[U];
        if (LINES) {
            const Columns c = columns_of<W>(k, a.D);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                x[u].clear();
                if (held[u]) x[u].load(from[u], c);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (n + u * rows >= a.N) break;
                float v[W];
#pragma unroll
                for (int q = 0; q < W; ++q) v[q] = x[u].value(q) * (held[u] ? a.scale : 0.0f);
                put_columns<O, W, true>(to[u], c, v);
            }
            continue;
        }
        int at[U];  // the column read first: a row's first and last vectors are read where the row has whole ones
        bool in[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int d = k - lead[u];
            in[u] = d < a.D && d + W > 0 && n + u * rows < a.N;
            at[u] = max(0, whole ? min(d, a.D - W) : d);
            x[u].clear();
            if (in[u] && held[u]) x[u].load(from[u], Columns{at[u], min(W, a.D - at[u]), 0, whole});
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (!in[u]) continue;
            const int d = k - lead[u];
            float v[W];
#pragma unroll
            for (int q = 0; q < W; ++q) v[q] = x[u].value(q) * (held[u] ? a.scale : 0.0f);
            if (at[u] == d && whole) {
                put_elements<O, W, true>(to[u] + d, v);
                continue;
            }
#pragma unroll
            for (int q = 0; q < W; ++q)
                if (at[u] + q >= d && at[u] + q < min(d + W, a.D)) to[u][at[u] + q] = (O)v[q];
        }
    }
}

// ----- sort of the slots by token ---------------------------------------------------------------------------------------------
constexpr int kMostBits = 10, kMostBins = 1 << kMostBits, kMostSortBlocks = 512, kSortThreads = 1024, kSortWaves = kSortThreads / 64;
// Up to here every workgroup counts the whole list's digits for itself, which takes about as long as a launch of its own for the counts, and less in
// short lists (gradient of 65536 x 128 in bf16, counted by every workgroup / by a launch: 8000 slots 31.5 us / 33.1, 16384 37.0 / 36.1, 30000
// 41.6 / 39.6; 45000 48.1 / 41.1, 120000 76.7 / 53.3).
constexpr long kCountedTwice = 32768;
constexpr int kFillVectors = 4;
// Tables that are filled on the way, bytes per launch.  Filled / not, us: 65536 x 1024 fp32 from 16384 slots 65.9 / 75.0, 30000 x 768 from 8192
// 37.8 / 38.7; tables of 16 to 40 MB are up to two us slower so (8192 x 512 from 20000 34.3 / 33.3, 20000 x 512 from 16384 35.7 / 33.8).
// 24, 32, 48, 64 and 80 MB per launch: 65536 x 1024 fp32 from 16384 slots 71.0, 68.7, 66.1, 63.4 and 65.0, from 8192 61.8, 59.7, 56.4, 55.6 and
// 60.1; 131072 x 512 bf16 from 16384 42.0, 42.2, 44.6, 44.8 and 46.3; 131072 x 1024 bf16 from 4000 59.1, 56.5, 52.3, 52.6 and 59.3.
constexpr size_t kFillFrom = 16 << 20, kFillBytes = 48 << 20;

// Scratch of a gradient, which is enough for shorter lists as well: two lists of (token, slot), counts of every block and digit, the number of slots with a token, where the rows' runs
// begin, partial sums.
struct SortPlan {
    int bits, passes, block, blocks, piece;  // slots per block, blocks; piece: entries of the sorted list that are added up together
    bool counted;                            // the counts are made by a launch of their own
    size_t keys[2], slots[2], counts, total, starts, partial, bytes;
};
SortPlan sort_plan(long V, int D, long N) {
    SortPlan p = {};
    int all = 0;
    while ((1L << all) < V) ++all;
    p.passes = std::max(1, (all + kMostBits - 1) / kMostBits);
    p.bits = std::max(1, (all + p.passes - 1) / p.passes);
    p.block = (int)((std::max(1L, (N + kMostSortBlocks - 1) / kMostSortBlocks) + kSortThreads - 1) / kSortThreads * kSortThreads);
    p.blocks = (int)std::max(1L, (N + p.block - 1) / p.block);
    p.counted = N > kCountedTwice;
    // partial sums of pieces: about as many entries in a piece as pieces in the longest runs
    p.piece = 32;
    while (64L * p.piece * p.piece < N) p.piece *= 2;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    const size_t list = (size_t)N * sizeof(int);
    p.keys[0] = take(list); p.slots[0] = take(list);
    p.keys[1] = p.passes > 1 ? take(list) : 0; p.slots[1] = p.passes > 1 ? take(list) : 0;
    p.counts = take(p.counted ? (size_t)std::min<long>(kMostSortBlocks, (N + kSortThreads - 1) / kSortThreads) * (1 << p.bits) * sizeof(int) : 0);
    p.total = take(sizeof(int));
    p.starts = take(((size_t)V + 1) * sizeof(int));
    // (a list that has pieces of half the length has up to 64 p^2 entries in them, p being that half)
    p.partial = take((size_t)std::max(N / p.piece, p.piece > 32 ? 32L * p.piece : 0L) * D * sizeof(float));
    p.bytes = at;
    return p;
}

// Zeros for a stretch of the table's gradient, from workgroups behind those of a launch that leaves most of the card idle.
struct Fill {
    char *to;
    long vectors;  // of 16 bytes
};
template <int THREADS>
__device__ __forceinline__ void fill_zeros(const Fill &f, int block) {
    typedef unsigned four __attribute__((ext_vector_type(4), aligned(2)));
    const long first = (long)block * (THREADS * kFillVectors) + threadIdx.x;
#pragma unroll
    for (int u = 0; u < kFillVectors; ++u)
        if (first + u * THREADS < f.vectors) __builtin_nontemporal_store(four{0u, 0u, 0u, 0u}, reinterpret_cast<four *>(f.to) + first + u * THREADS);
}
unsigned fill_blocks(const Fill &f, int threads) { return (unsigned)((f.vectors + threads * kFillVectors - 1) / (threads * kFillVectors)); }

struct SortArgs {
    const int *keys, *slots;  // the list before the pass; first pass: keys are the tokens, slots NULL
    int *keys_out, *slots_out, *counts, *total;
    int N, V, shift, bits, block, blocks;
    Fill fill;
};

// First pass: a slot without a token has no place in the list.  Later ones: `total` entries are in it.
template <bool FIRST>
__device__ __forceinline__ int entries(const SortArgs &a) { return FIRST ? a.N : *a.total; }
template <bool FIRST>
__device__ __forceinline__ bool listed(const SortArgs &a, int key) { return !FIRST || (unsigned)key < (unsigned)a.V; }

// how often every digit occurs among entries begin .. end, added to bins
template <bool FIRST>
__device__ __forceinline__ void count_digits(const SortArgs &a, int begin, int end, int first, int step, int *bins) {
    constexpr int U = 8;  // loads in flight
    // (whole waves go round, so that all lanes take part in the ballots)
    for (int i = begin + first; i - (int)(threadIdx.x & 63) < end; i += U * step) {
        int key[U];
#pragma unroll
        for (int u = 0; u < U; ++u) key[u] = i + u * step < end ? a.keys[i + u * step] : -1;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool in = FIRST ? (unsigned)key[u] < (unsigned)a.V : key[u] >= 0;
            const int digit = (key[u] >> a.shift) & ((1 << a.bits) - 1);
            if (FIRST) {
                if (in) atomicAdd(&bins[digit], 1);
                continue;
            }
            // Upper digits: that of the wave's first entry is counted at once.  Half of all tokens have the same one, and additions to
            // one address go one by one (second pass of 16384 tokens of 65536: 12.4 us so, 9.4 us with a count; the first one's 7.4 and 9.6).
            const unsigned long long all = __ballot(in);
            if (all) {
                const int common = __builtin_amdgcn_readlane(digit, __builtin_ctzll(all));
                const unsigned long long same = __ballot(in && digit == common);
                if ((threadIdx.x & 63) == __builtin_ctzll(same)) atomicAdd(&bins[common], (int)__popcll(same));
                if (in && digit != common) atomicAdd(&bins[digit], 1);
            }
        }
    }
}

template <bool FIRST>
__global__ __launch_bounds__(kSortThreads) void token_count_kernel(const SortArgs a) {
    __shared__ int bins[kMostBins];
    const int n_bins = 1 << a.bits, n = entries<FIRST>(a), d = threadIdx.x;
    bins[d] = 0;
    __syncthreads();
    const int begin = min(n, (int)blockIdx.x * a.block);
    count_digits<FIRST>(a, begin, min(n, begin + a.block), d, kSortThreads, bins);
    __syncthreads();
    if (d < n_bins) a.counts[blockIdx.x * n_bins + d] = bins[d];
}

// Puts a block's entries to their places, a thread per digit and entry.  COUNTED: every block adds the blocks' counts up for itself, which
// saves a launch; else it counts the whole list.
template <bool FIRST, bool COUNTED>
__global__ __launch_bounds__(kSortThreads) void token_place_kernel(const SortArgs a) {
    static_assert(kSortThreads == kMostBins, "a thread per digit");
    __shared__ int next[kSortWaves][kMostBins];  // counts of a wave's entries, then the next place for every wave and digit
    __shared__ int earlier[kMostBins], others[kMostBins];
    __shared__ int wave_totals[kSortWaves];
    if ((int)blockIdx.x >= a.blocks) {
        fill_zeros<kSortThreads>(a.fill, blockIdx.x - a.blocks);
        return;
    }
    const int n_bins = 1 << a.bits, n = entries<FIRST>(a), d = threadIdx.x, lane = d & 63, wave = d >> 6;
    if (d < n_bins) {
#pragma unroll
        for (int w = 0; w < kSortWaves; ++w) next[w][d] = 0;
        earlier[d] = others[d] = 0;
    }
    __syncthreads();
    const int block_begin = min(n, (int)blockIdx.x * a.block), block_end = min(n, block_begin + a.block);
    const int share = a.block / kSortWaves, begin = min(n, block_begin + wave * share), end = min(n, begin + share);
    count_digits<FIRST>(a, begin, end, lane, 64, next[wave]);
    int before = 0, all = 0;
    if (COUNTED) {
        if (d < n_bins) {
#pragma unroll 8
            for (int b = 0; b < a.blocks; ++b) {
                const int c = a.counts[b * n_bins + d];
                all += c;
                before += b < (int)blockIdx.x ? c : 0;
            }
        }
    } else {
        count_digits<FIRST>(a, 0, block_begin, d, kSortThreads, earlier);
        count_digits<FIRST>(a, block_end, n, d, kSortThreads, others);
    }
    __syncthreads();
    if (!COUNTED && d < n_bins) {
        before = earlier[d];
        all = before + others[d];
#pragma unroll
        for (int w = 0; w < kSortWaves; ++w) all += next[w][d];
    }
    // places of the digits
    int upto = all;
    for (int o = 1; o < 64; o *= 2) {
        const int other = __shfl_up(upto, o);
        if (lane >= o) upto += other;
    }
    if (lane == 63) wave_totals[wave] = upto;
    __syncthreads();
    int at = upto - all;
    for (int w = 0; w < wave; ++w) at += wave_totals[w];
    if (FIRST && blockIdx.x == 0 && d == kSortThreads - 1) *a.total = at + all;
    at += before;
    if (d < n_bins) {
#pragma unroll
        for (int w = 0; w < kSortWaves; ++w) {
            const int c = next[w][d];
            next[w][d] = at;
            at += c;
        }
    }
    __syncthreads();
    // In steps of 64 entries, in order: lanes of one digit find each other by one ballot per bit.  Every lane reads its digit's
    // next place before the first lane of the digit moves it on (the accesses of one wave to LDS are performed in order).
    volatile int *mine = next[wave];
    for (int i0 = begin; i0 < end; i0 += 64) {
        const int i = i0 + lane;
        const int key = i < end ? a.keys[i] : -1;
        const bool in = i < end && listed<FIRST>(a, key);
        const int digit = in ? (key >> a.shift) & (n_bins - 1) : 0;
        unsigned long long same = __ballot(in);
        for (int bit = 0; bit < a.bits; ++bit) {
            const bool set = (digit >> bit) & 1;
            const unsigned long long b = __ballot(set);
            same &= set ? b : ~b;
        }
        const int rank = __popcll(same & ((1ull << lane) - 1));
        const int place = mine[digit] + rank;
        __builtin_amdgcn_wave_barrier();
        if (in && rank == 0) mine[digit] = place + __popcll(same);
        __builtin_amdgcn_wave_barrier();
        if (in) {
            a.keys_out[place] = key;
            a.slots_out[place] = FIRST ? i : a.slots[i];
        }
    }
}

// Whether rows of the gradient are written past the caches: rows of whole lines (53665 of 512 fp32 zeros 21.1 us, 21.8 through the caches), and tables
// that the last-level cache has no room for (65536 rows of 1000 from 16384 slots 76 us and 86).  Other rows share lines, which are written twice
// past the caches (53665 of 458: 28 us, 17 through them).
inline bool past_caches(const void *grad, int V, int D, long stride, int type) {
    const long row = stride * (long)element_size(type);
    return (reinterpret_cast<uintptr_t>(grad) % 128 == 0 && row % 128 == 0) || V * (long)D * (long)element_size(type) > 128L << 20;
}
// columns c of a row of the gradient
template <typename G, int W>
__device__ __forceinline__ void put_sums(G *row, const Columns &c, const float (&sum)[W], float scale, int accumulate, int once) {
    if (c.count <= 0) return;
    float v[W];
#pragma unroll
    for (int q = 0; q < W; ++q) v[q] = sum[q] * scale;
    if (accumulate) {
        Vector<G, W> old;
        old.clear();
        old.load(row, c);
#pragma unroll
        for (int q = 0; q < W; ++q) v[q] = old.value(q) + sum[q] * scale;
    }
    if (once) put_columns<G, W, true>(row, c, v);
    else put_columns<G, W, false>(row, c, v);
}

// ----- sums of the runs -------------------------------------------------------------------------------------------------------
constexpr int kWindow = 16, kZeroRows = 4;

struct SumArgs {
    const int *keys, *slots, *total;
    const void *err;
    void *grad;
    int *starts;  // V + 1: where the rows' runs begin in the sorted list
    float *partial;
    long err_stride, grad_stride;
    int V, D, lanes, piece, accumulate;
    int tiles;         // of `lanes` threads' columns in a row; neighbouring workgroups have neighbouring ones
    int by_rows, searched, once;
    int first_blocks, run_blocks;  // workgroups of a launch's first and second kind, in front of those of the third
    int pieces;
    int filled;  // rows, the first ones, that hold zeros already
    Fill fill;
    float scale;
};

// Sum of every step-th of the entries begin .. end and begin2 .. end2 of the sorted list, from number `first` on, by the
// `lanes` threads of a group: every thread has one of the next slots, which go round the group, so that a slot is waited for once in
// `lanes` entries.
template <typename E, int W>
__device__ __forceinline__ void add_entries(const SumArgs &a, int begin, int end, int begin2, int end2, int first, int step, const Columns &c,
                                            float (&sum)[W]) {
    constexpr int U = 8;  // rows in flight
    const E *err = static_cast<const E *>(a.err);
    const int x = threadIdx.x % a.lanes, n1 = end - begin, n = n1 + end2 - begin2;
    for (int i = first; i < n; i += a.lanes * step) {
        const int e = i + x * step;
        const int mine = e < n ? a.slots[e < n1 ? begin + e : begin2 + e - n1] : 0;
        const int rows = min(a.lanes, (n - i + step - 1) / step);
        for (int k = 0; k < rows; k += U) {
            Vector<E, W> v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int slot = __shfl(mine, k + u, a.lanes);
                v[u].clear();
                if (k + u < rows && c.count > 0) v[u].load(err + slot * a.err_stride, c);
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int q = 0; q < W; ++q) sum[q] += v[u].value(q);
        }
    }
}

// the sums of a workgroup's groups, in the first group
template <int W>
__device__ __forceinline__ void join_groups(int lanes, float (&sum)[W]) {
    __shared__ float parts[256 * W];
    const int x = threadIdx.x % lanes, g = threadIdx.x / lanes, groups = 256 / lanes;
    __syncthreads();
#pragma unroll
    for (int q = 0; q < W; ++q) parts[(g * W + q) * lanes + x] = sum[q];
    __syncthreads();
    if (g == 0)
        for (int o = 1; o < groups; ++o)
#pragma unroll
            for (int q = 0; q < W; ++q) sum[q] += parts[(o * W + q) * lanes + x];
}

// Where the runs of the rows key(i - 1) + 1 .. key(i) begin: at entry i.  A wave for 64 entries; long gaps between two keys are filled
// by the whole wave.
__device__ __forceinline__ void find_starts(const SumArgs &a) {
    const int lane = threadIdx.x & 63, n = *a.total;
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    int from = 0, to = -1;  // rows whose runs begin at entry i
    if (i <= n) {
        from = i == 0 ? 0 : a.keys[i - 1] + 1;
        to = i == n ? a.V : a.keys[i];
    }
    unsigned long long far = __ballot(to - from >= 64);
    if (to - from < 64)
        for (int v = from; v <= to; ++v) a.starts[v] = (int)i;
    for (; far; far &= far - 1) {
        const int owner = __builtin_ctzll(far), first = __builtin_amdgcn_readlane(from, owner), last = __builtin_amdgcn_readlane(to, owner);
        const int entry = __builtin_amdgcn_readlane((int)i, owner);
        for (long v = (long)first + lane; v <= last; v += 64) a.starts[v] = entry;
    }
}

// The same for one row per thread, by bisection.
__device__ __forceinline__ void search_starts(const SumArgs &a) {
    const long v = (long)blockIdx.x * 256 + threadIdx.x;
    if (v > a.V) return;
    int begin = 0;
    for (int rest = *a.total; rest > 0;) {
        const int half = rest / 2;
        const bool above = a.keys[begin + half] < v;
        begin = above ? begin + half + 1 : begin;
        rest = above ? rest - half - 1 : half;
    }
    a.starts[v] = begin;
}

// First workgroups: where the runs begin.  Then sums of the pieces of the sorted list that lie within one run.  Then zeros.
// blockIdx.y: the columns.
template <typename E, int W>
__global__ __launch_bounds__(256) void embed_pieces_kernel(const SumArgs a) {
    if ((int)blockIdx.x < a.first_blocks) {
        if (blockIdx.y == 0) a.searched ? search_starts(a) : find_starts(a);
        return;
    }
    if ((int)blockIdx.x >= a.first_blocks + a.pieces) {
        if (blockIdx.y == 0) fill_zeros<256>(a.fill, blockIdx.x - a.first_blocks - a.pieces);
        return;
    }
    const int piece = blockIdx.x - a.first_blocks, begin = piece * a.piece, end = begin + a.piece;
    if (end > *a.total || a.keys[begin] != a.keys[end - 1]) return;
    const int x = threadIdx.x % a.lanes, g = threadIdx.x / a.lanes;
    const Columns c = columns_of<W>((blockIdx.y * a.lanes + x) * W, a.D);
    float sum[W] = {};
    add_entries<E, W>(a, begin, end, 0, 0, g, 256 / a.lanes, c, sum);
    join_groups<W>(a.lanes, sum);
    if (g == 0) put_sums(a.partial + (size_t)piece * a.D, c, sum, 1.0f, 0, 0);
}

template <typename G, int W>
__device__ __forceinline__ void write_row(const SumArgs &a, int row, const Columns &c, const float (&sum)[W]) {
    put_sums(static_cast<G *>(a.grad) + row * a.grad_stride, c, sum, a.scale, a.accumulate, a.once);
}

// The rows of the runs that begin at entries from .. from + kWindow of the sorted list and hold no first entry of a piece, by a group of threads:
// it goes through the list, eight rows of errors in flight, and writes a row where its run ends.
template <typename E, typename G, int W>
__device__ __forceinline__ void sum_short_runs(const SumArgs &a, int from, const Columns &c) {
    constexpr int U = 8;
    const int n = *a.total, x = threadIdx.x % a.lanes;
    if (from >= n) return;
    // from `stop` on, runs are others'; so is the run that holds the entry in front, or the first one of a piece
    const int stop = min(n, (from / a.piece + 1) * a.piece), behind = min(from + kWindow, stop);
    const int skipped = a.keys[from % a.piece == 0 ? from : from - 1], last = a.keys[behind - 1];
    if (last == skipped) return;
    const E *err = static_cast<const E *>(a.err);
    int current = skipped;
    float sum[W] = {};
    for (int i0 = from; i0 < stop; i0 += a.lanes) {
        const int mine = i0 + x < stop ? a.keys[i0 + x] : skipped, my_slot = i0 + x < stop ? a.slots[i0 + x] : 0;
        const int here = min(a.lanes, stop - i0);
        for (int k = 0; k < here; k += U) {
            Vector<E, W> v[U];
            int key[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                key[u] = __shfl(mine, k + u, a.lanes);
                const int slot = __shfl(my_slot, k + u, a.lanes);
                const bool needed = k + u < here && key[u] != skipped && (i0 + k + u < behind || key[u] == last);
                v[u].clear();
                if (needed && c.count > 0) v[u].load(err + slot * a.err_stride, c);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (k + u >= here) break;
                if (key[u] != current) {
                    if (current != skipped) write_row<G, W>(a, current, c, sum);
                    if (i0 + k + u >= behind) return;
                    current = key[u];
#pragma unroll
                    for (int q = 0; q < W; ++q) sum[q] = 0.0f;
                }
#pragma unroll
                for (int q = 0; q < W; ++q) sum[q] += v[u].value(q);
            }
        }
    }
    if (stop == n || a.keys[stop] != current) write_row<G, W>(a, current, c, sum);
}

// First workgroups: rows whose run holds the first entry of a piece, by all groups of the workgroup of the first such piece; whole pieces go
// by their sums.  Then the other runs, a group of `lanes` threads for those that begin in kWindow entries, and zeros for the rows
// without entries, kZeroRows for a group; or, by_rows, a row for each group in place of both.
template <typename E, typename G, int W>
__global__ __launch_bounds__(256) void embed_rows_kernel(const SumArgs a) {
    const int groups = 256 / a.lanes, x = threadIdx.x % a.lanes, g = threadIdx.x / a.lanes;
    const int block = blockIdx.x / a.tiles;
    const Columns c = columns_of<W>(((int)blockIdx.x % a.tiles * a.lanes + x) * W, a.D);
    float sum[W] = {};
    if (block < a.first_blocks) {
        const int here = block * a.piece;
        if (here >= *a.total) return;
        const int row = a.keys[here], begin = a.starts[row], end = a.starts[row + 1];
        if (here - begin >= a.piece) return;
        const int whole = end / a.piece * a.piece;  // >= here
        if (c.count > 0) {
#pragma unroll 8
            for (int p = block + g; p < whole / a.piece; p += groups) {
                Vector<float, W> v;
                v.clear();
                v.load(a.partial + (size_t)p * a.D, c);
#pragma unroll
                for (int q = 0; q < W; ++q) sum[q] += v.value(q);
            }
        }
        add_entries<E, W>(a, begin, here, whole, end, g, groups, c, sum);
        join_groups<W>(a.lanes, sum);
        if (g == 0) write_row<G, W>(a, row, c, sum);
        return;
    }
    if (block < a.first_blocks + a.run_blocks) {
        sum_short_runs<E, G, W>(a, ((block - a.first_blocks) * groups + g) * kWindow, c);
        return;
    }
    if (a.by_rows) {
        const long row = (long)(block - a.first_blocks) * groups + g;
        if (row >= a.V) return;
        const int begin = a.starts[row], end = a.starts[row + 1];
        // the first workgroups', or nothing to write
        if (end > begin ? (end - 1) / a.piece * a.piece >= begin : a.accumulate || row < a.filled) return;
        add_entries<E, W>(a, begin, end, 0, 0, 0, 1, c, sum);
        write_row<G, W>(a, (int)row, c, sum);
        return;
    }
    const long first = a.filled + ((long)(block - a.first_blocks - a.run_blocks) * groups + g) * kZeroRows;
    int bounds[kZeroRows + 1];
#pragma unroll
    for (int r = 0; r <= kZeroRows; ++r) bounds[r] = a.starts[min((long)a.V, first + r)];
#pragma unroll
    for (int r = 0; r < kZeroRows; ++r)
        if (first + r < a.V && bounds[r] == bounds[r + 1]) write_row<G, W>(a, (int)(first + r), c, sum);
}

// ----- few slots ---------------------------------------------------------------------------------------------------------
// Every workgroup looks through all tokens for those of its rows, which it keeps in the order of their slots; a group of threads has kept its
// row's errors added up in that order.  One launch: 5 slots of 708 rows 13.5 us by the sorted list.
constexpr int kFewSlots = 128;

struct FewArgs {
    const int *tokens;
    const void *err;
    void *grad;
    long err_stride, grad_stride;
    int N, V, D, lanes, tiles, accumulate, once;
    float scale;
};

template <typename E, typename G, int W, int R>
__global__ __launch_bounds__(256) void embed_few_kernel(const FewArgs a) {
    constexpr int U = 8;
    __shared__ int rows[kFewSlots], slots[kFewSlots], counts[2];
    const int groups = 256 / a.lanes, x = threadIdx.x % a.lanes, g = threadIdx.x / a.lanes, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int block = blockIdx.x / a.tiles;
    const Columns c = columns_of<W>(((int)blockIdx.x % a.tiles * a.lanes + x) * W, a.D);
    // the workgroup's rows, `step` apart: frequent tokens are neighbours in most vocabularies
    const int first = block * groups, step = (int)(gridDim.x / a.tiles) * groups;
    const int token = (int)threadIdx.x < a.N ? a.tokens[threadIdx.x] : -1;
    const bool mine = token >= first && token < a.V && (token - first) % step < groups;
    const unsigned long long in = __ballot(mine);
    if (wave < 2 && lane == 0) counts[wave] = __popcll(in);
    __syncthreads();
    const int found = counts[0] + counts[1];
    if (mine) {
        const int place = (wave ? counts[0] : 0) + __popcll(in & ((1ull << lane) - 1));
        rows[place] = token;
        slots[place] = threadIdx.x;
    }
    __syncthreads();
    const E *err = static_cast<const E *>(a.err);
    const unsigned long long group = a.lanes == 64 ? ~0ull : (1ull << a.lanes) - 1;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const long row = first + (long)r * step + g;
        float sum[W] = {};
        bool any = false;
        for (int i = 0; i < found; i += a.lanes) {
            // those of the group's row among the next entries, a bit for each, eight rows of errors in flight
            unsigned long long own = __ballot(i + x < found && rows[i + x] == row) >> (lane - lane % a.lanes) & group;
            any = any || own;
            while (own) {
                Vector<E, W> v[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    v[u].clear();
                    if (own && c.count > 0) v[u].load(err + slots[i + __builtin_ctzll(own)] * a.err_stride, c);
                    own &= own - 1;
                }
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int q = 0; q < W; ++q) sum[q] += v[u].value(q);
            }
        }
        if (row >= a.V || (a.accumulate && !any)) continue;
        put_sums(static_cast<G *>(a.grad) + row * a.grad_stride, c, sum, a.scale, a.accumulate, a.once);
    }
}

template <typename E, typename G>
int sum_few(hipStream_t stream, const FewArgs &args) {
    constexpr int W = kBoth<E, G>;
    FewArgs a = args;
    a.lanes = std::max(8, std::min(64, power_of_two_from((a.D + W - 1) / W)));
    a.tiles = (int)((a.D + (long)a.lanes * W - 1) / (a.lanes * W));
    // eight rows for a group where there are enough of them for the card
    const long groups = 256 / a.lanes, blocks = (a.V + groups - 1) / groups * a.tiles;
    const bool many = blocks >= 8192;
    auto kernel = many ? embed_few_kernel<E, G, W, 8> : embed_few_kernel<E, G, W, 1>;
    const long each = groups * (many ? 8 : 1);
    hipLaunchKernelGGL(kernel, dim3((unsigned)((a.V + each - 1) / each * a.tiles)), dim3(256), 0, stream, a);
    CNT_HIP(hipGetLastError());
    return CNT_OK;
}

// ----- slabs of the list ------------------------------------------------------------------------------------------------------------------
// A workgroup sorts the slots of a slab that belong to its rows in LDS and adds their errors up.  One slab's sums are the gradient itself; those
// of several are left in the place of their first slot and added up, in order, by a second launch, which goes by an index of the rows' runs; or, where
// a slab has two places for every row, in the row's (256 x 64 from 32000 slots 16.7 us, by the index 17.6; 31 x 8 from 260000 41.9 and 46.0; half empty, 509 x 746 from 6737 26 and 19).
constexpr unsigned short kNoRun = 0xffff;
constexpr int kSlab = 512, kSlabRows = 1024, kSlabWaves = kSlab / 64, kSlabLanes = 16;
// Against the sorted list, fp32, us.  One slab: 1000 x 64 from 300 slots 7.0 / 18.2, 100000 x 64 from 500 10.7 / 22.1, 50000 x 458 from 300 24.6 / 28.7;
// beyond 65536 x 1024 from 500 54 / 47 (the zeros, in rows of 256 bytes here).
constexpr long kOneSlabValues = 1 << 25;
// Several: 256 x 64 from 32000 16.7 / 23.3, 1000 x 64 from 2000 10.8 / 15.3, 1665 x 594 from 943 13.5 / 21.4, 46356 x 13 from 7743 19.4 / 29.5, 2261 x 132
// from 17980 19.4 / 30.9, 3992 x 1135 from 3826 25.3 / 29.5; beyond 19473 x 367 from 4492 36 / 28, 577 x 801 from 26051 44 / 36, 100 x 2048 from
// 16000 41 / 36.
// More errors where little is left of them: 51 x 767 from 25518 35.5 / 40.1, 20 x 512 from 30000 21.4 / 41.1.
constexpr long kSlabValues = 1 << 24, kSlabJoined = 5 << 23, kFewJoined = 1 << 21;  // errors; values of all slabs' tables
constexpr int kMostSlabs = 512;  // (31 x 8 from 260000 41 / 42, from 1000000 141 / 72)

struct SlabArgs {
    const int *tokens;
    const void *err;
    void *out;              // the gradient, or the runs' sums of all slabs
    unsigned short *index;  // of several slabs: the first slot of every row's run in every slab, kNoRun where there is none
    long err_stride, out_stride;
    int N, V, D, bits, lanes, tiles, parts, accumulate, once;  // parts: workgroups that share a slab's rows
    int dense;  // every row has its own place in a slab and needs no index
    float scale;
};

template <typename E, typename G, int W>
__global__ __launch_bounds__(kSlab) void embed_slab_kernel(const SlabArgs a) {
    constexpr int U = kSlabLanes;  // entries of a group of threads at most: all of its errors are in flight together
    static_assert(kSlabRows == 2 * kSlab, "two rows per thread in the scan");
    union Words {
        unsigned short one[kSlabWaves][kSlabRows];
        unsigned two[kSlabWaves][kSlab];
        uint4 all[kSlabWaves * kSlabRows / 8];
    };
    __shared__ Words before;  // entries of a row in 64 slots, then in all 64 slots in front of them
    __shared__ int starts[kSlabRows + 1];
    __shared__ unsigned list[kSlab];  // row and slot
    __shared__ int totals[kSlabWaves];
    __shared__ float heads[kSlab * W];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int tile = blockIdx.x % a.tiles, part = blockIdx.x / a.tiles % a.parts, slab = blockIdx.x / (a.tiles * a.parts);
    const int base = slab * kSlab, slot = base + (int)threadIdx.x;
    // the workgroup's rows
    const int low = (int)((long)a.V * part / a.parts), rows = (int)((long)a.V * (part + 1) / a.parts) - low;
    const int token = slot < a.N ? a.tokens[slot] : -1, row_of = token >= low && token < low + rows ? token - low : -1;
    for (int k = threadIdx.x; k < kSlabWaves * kSlabRows / 8; k += kSlab) before.all[k] = uint4{0u, 0u, 0u, 0u};
    __syncthreads();
    // lanes of one row find each other by one ballot per bit
    const bool in = row_of >= 0;
    unsigned long long same = __ballot(in);
    for (int bit = 0; bit < a.bits; ++bit) {
        const bool set = (row_of >> bit) & 1;
        const unsigned long long b = __ballot(set);
        same &= set ? b : ~b;
    }
    const int rank = __popcll(same & ((1ull << lane) - 1));
    if (in && rank == 0) before.one[wave][row_of] = (unsigned short)__popcll(same);
    __syncthreads();
    unsigned both = 0;  // of rows 2 * thread and 2 * thread + 1, side by side
#pragma unroll
    for (int h = 0; h < kSlabWaves; ++h) {
        const unsigned c = before.two[h][threadIdx.x];
        before.two[h][threadIdx.x] = both;
        both += c;
    }
    const int all = (int)((both & 0xffff) + (both >> 16));
    int upto = all;
    for (int o = 1; o < 64; o *= 2) {
        const int other = __shfl_up(upto, o);
        if (lane >= o) upto += other;
    }
    if (lane == 63) totals[wave] = upto;
    __syncthreads();
    int at = upto - all;
#pragma unroll
    for (int w = 0; w < kSlabWaves; ++w) at += w < wave ? totals[w] : 0;
    starts[2 * threadIdx.x] = at;
    starts[2 * threadIdx.x + 1] = at + (int)(both & 0xffff);
    if (threadIdx.x == kSlab - 1) starts[kSlabRows] = at + all;
    __syncthreads();
    if (in) list[starts[row_of] + before.one[wave][row_of] + rank] = (unsigned)row_of << 16 | threadIdx.x;
    __syncthreads();
    // Groups of threads have equal shares of the list.  A run that began in another's share is left to the group where it began.
    const int n = starts[kSlabRows];
    const int groups = kSlab / a.lanes, x = threadIdx.x % a.lanes, g = threadIdx.x / a.lanes;
    const Columns c = columns_of<W>((tile * a.lanes + x) * W, a.D);
    const E *err = static_cast<const E *>(a.err) + base * a.err_stride;
    auto write = [&](int row, const float (&total)[W]) {
        const int to = a.dense ? base + low + row : a.index ? base + (int)(list[starts[row]] & 0xffff) : low + row;
        put_sums(static_cast<G *>(a.out) + to * a.out_stride, c, total, a.scale, a.accumulate, a.once);
    };
    const int share = (n + groups - 1) / groups, begin = min(n, g * share), end = min(n, begin + share);
    const int others = begin > 0 && begin < end && list[begin] >> 16 == list[begin - 1] >> 16 ? (int)(list[begin] >> 16) : -1;
    Vector<E, W> v[U];
    int key[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const unsigned entry = begin + u < end ? list[begin + u] : ~0u;
        key[u] = begin + u < end ? (int)(entry >> 16) : -1;
        v[u].clear();
        if (begin + u < end && c.count > 0) v[u].load(err + (int)(entry & 0xffff) * a.err_stride, c);
    }
    int current = -1;
    float sum[W] = {};
    auto keep = [&]() {
#pragma unroll
        for (int q = 0; q < W; ++q) heads[(g * W + q) * a.lanes + x] = sum[q];
    };
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (key[u] < 0) break;
        if (key[u] != current) {
            if (current >= 0 && current == others) keep();
            else if (current >= 0) write(current, sum);
            current = key[u];
#pragma unroll
            for (int q = 0; q < W; ++q) sum[q] = 0.0f;
        }
#pragma unroll
        for (int q = 0; q < W; ++q) sum[q] += v[u].value(q);
    }
    if (current >= 0 && current == others) keep();
    __syncthreads();
    if (current >= 0 && current != others) {
        for (int o = g + 1; o * share < n && (int)(list[o * share] >> 16) == current; ++o) {
#pragma unroll
            for (int q = 0; q < W; ++q) sum[q] += heads[(o * W + q) * a.lanes + x];
        }
        write(current, sum);
    }
    if (a.index ? a.dense : !a.accumulate) {
#pragma unroll
        for (int q = 0; q < W; ++q) sum[q] = 0.0f;
#pragma unroll 8
        for (int row = g; row < rows; row += groups)
            if (starts[row] == starts[row + 1]) write(row, sum);
    }
    if (a.index && !a.dense && tile == 0)
        for (int row = threadIdx.x; row < rows; row += kSlab)
            a.index[(long)slab * a.V + low + row] = starts[row] < starts[row + 1] ? (unsigned short)list[starts[row]] : kNoRun;
}

struct JoinArgs {
    const float *sums;
    const unsigned short *index;
    void *grad;
    long grad_stride;
    int slabs, V, D, vectors, split, dense, accumulate, once;  // vectors of a row; split: waves that share a row's slabs, 1 or 4
    float scale;
};

// The rows' runs of all slabs, W columns per thread; U slabs in flight (5000 x 8 from 65000 slots, by sixteens 24.9 us, by
// eights 26.0; 30000 x 128 from 1000 18.7 and 15.5).
template <typename G, int U>
__global__ __launch_bounds__(256) void embed_slab_join_kernel(const JoinArgs a) {
    constexpr int W = kBoth<float, G>;
    __shared__ float sums[3][W][64];
    __shared__ int found[3][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, part = wave % a.split, each = (a.slabs + a.split - 1) / a.split;
    const unsigned i = (blockIdx.x * (4 / a.split) + wave / a.split) * 64 + lane, row = i / (unsigned)a.vectors;
    Columns c = columns_of<W>((int)(i - row * a.vectors) * W, a.D);
    if (row >= (unsigned)a.V) c.count = 0;
    const int begin = min(a.slabs, part * each), end = min(a.slabs, begin + each);
    float sum[W] = {};
    int any = 0;
    for (int s = begin; s < end; s += U) {
        int run[U];
        Vector<float, W> v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) run[u] = s + u >= end || c.count <= 0 ? kNoRun : a.dense ? (int)row : a.index[(long)(s + u) * a.V + row];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            v[u].clear();
            if (run[u] != kNoRun) v[u].load(a.sums + ((long)(s + u) * kSlab + run[u]) * a.D, c);
            any |= run[u] != kNoRun;
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int q = 0; q < W; ++q) sum[q] += v[u].value(q);
    }
    if (a.split > 1) {
        if (wave > 0) {
#pragma unroll
            for (int q = 0; q < W; ++q) sums[wave - 1][q][lane] = sum[q];
            found[wave - 1][lane] = any;
        }
        __syncthreads();
        if (wave > 0) return;
#pragma unroll
        for (int o = 0; o < 3; ++o) {
            any |= found[o][lane];
#pragma unroll
            for (int q = 0; q < W; ++q) sum[q] += sums[o][q][lane];
        }
    }
    if (row >= (unsigned)a.V || (a.accumulate && !any)) return;
    put_sums(static_cast<G *>(a.grad) + (long)row * a.grad_stride, c, sum, a.scale, a.accumulate, a.once);
}

// Scratch of a gradient by slabs: their runs' sums, where these are.
struct SlabPlan {
    int slabs;  // 0: by the sorted list
    size_t index;
};
SlabPlan slab_plan(int V, int D, long N) {
    SlabPlan p = {};
    const long slabs = (N + kSlab - 1) / kSlab;
    if (N <= kFewSlots) return p;
    if (slabs > kMostSlabs) return p;
    if (slabs > 1 ? slabs * V * D > (N * D > kSlabValues ? kFewJoined : kSlabJoined) || N * D > 2 * kSlabValues : (long)V * D > kOneSlabValues) return p;
    p.slabs = (int)slabs;
    p.index = (size_t)slabs * kSlab * D * sizeof(float);
    return p;
}

size_t gradient_scratch(int V, int D, long N) {
    // as many slabs as this list or a shorter one may have
    const long slabs = std::min({(N + kSlab - 1) / kSlab, (long)kMostSlabs, kSlabJoined / ((long)V * D), 2 * kSlabValues / D / kSlab + 1});
    return std::max(sort_plan(V, D, N).bytes, slabs > 1 ? (size_t)slabs * (kSlab * (size_t)D * sizeof(float) + V * sizeof(unsigned short)) : 0);
}

template <typename E, typename G>
int sum_slab(hipStream_t stream, const SlabArgs &args, int slabs) {
    constexpr int W = kBoth<E, G>;
    SlabArgs a = args;
    a.lanes = std::max(8, std::min(kSlabLanes, power_of_two_from((a.D + W - 1) / W)));  // (4: 31 rows of 8, 30000 slots 13.3 us, 11.9 with 8)
    a.tiles = (int)((a.D + (long)a.lanes * W - 1) / (a.lanes * W));
    // A workgroup for every compute unit, if its part has 32 rows (256 x 64 from 32000 slots, 512 workgroups 15.5 us; 1000 x 64 from 300, one 11.2;
    // 131072 x 8 from 500, 1024 11.3).
    const long most = std::max<long>((a.V + kSlabRows - 1) / kSlabRows, 256 / ((long)slabs * a.tiles));
    a.parts = (int)std::max(1L, std::min<long>((a.V + 31) / 32, most));
    while ((long)a.parts << a.bits < a.V) ++a.bits;
    hipLaunchKernelGGL((embed_slab_kernel<E, G, W>), dim3((unsigned)((long)slabs * a.tiles * a.parts)), dim3(kSlab), 0, stream, a);
    CNT_HIP(hipGetLastError());
    return CNT_OK;
}

// What a launch has workgroups for, 2^24 of 256 threads: rows of 256 columns take the most, a fourth of one for each.
bool gradient_sizes(int V, int D, long N) {
    return V > 0 && V <= 1 << 23 && D > 0 && D <= 1 << 21 && N >= 0 && N <= 1L << 30 && std::max<long>(V, N) * D <= 1L << 33;
}

// threads that share a row, W columns each
void share_columns(SumArgs &a, int W) {
    a.lanes = std::max(8, std::min(64, power_of_two_from((a.D + W - 1) / W)));  // (eight: as many rows are in flight)
    a.tiles = (int)((a.D + (long)a.lanes * W - 1) / (a.lanes * W));
}

template <typename E, typename G>
int sum_runs(hipStream_t stream, const SumArgs &args, long N) {
    SumArgs a = args;
    const long pieces = N / a.piece, starters = (N + a.piece - 1) / a.piece;
    {
        constexpr int W = kWide<E>;
        share_columns(a, W);
        // Few entries for the rows: gaps of hundreds of rows are not left to a wave each (100003 x 400 from 600 slots: 65 us for the gradient, 36 so).
        a.searched = a.V / 4 > N;
        a.first_blocks = (int)((a.searched ? a.V : N) / 256 + 1);
        a.pieces = (int)pieces;
        hipLaunchKernelGGL((embed_pieces_kernel<E, W>), dim3((unsigned)(a.first_blocks + pieces) + fill_blocks(a.fill, 256), (unsigned)a.tiles), dim3(256), 0,
                           stream, a);
        CNT_HIP(hipGetLastError());
    }
    constexpr int W = kBoth<E, G>;
    share_columns(a, W);
    // Few rows: a group's time is that of one run, and no rows are left to go through for their zeros (577 x 801 from 26051 slots 36 us, 41 by windows of
    // the list).  Many rows: most are without entries, and the runs' groups are those of the list (65536 x 1024 from 16384 67 us, 96 by rows).
    a.by_rows = a.V <= N;
    const long groups = 256 / a.lanes, windows = a.by_rows ? 0 : (N + kWindow - 1) / kWindow;
    const long others = a.by_rows ? a.V : a.accumulate ? 0 : (a.V - a.filled + kZeroRows - 1) / kZeroRows;
    a.first_blocks = (int)starters;
    a.run_blocks = (int)((windows + groups - 1) / groups);
    const long blocks = (a.first_blocks + a.run_blocks + (others + groups - 1) / groups) * a.tiles;
    if (blocks > 0) hipLaunchKernelGGL((embed_rows_kernel<E, G, W>), dim3((unsigned)blocks), dim3(256), 0, stream, a);
    CNT_HIP(hipGetLastError());
    return CNT_OK;
}

}  // namespace
}  // namespace cnt

extern "C" {

int cnt_embed_forward(void *stream_, int V, int D, long N, int table_type, const void *table, long table_stride, const int *tokens,
                      float scale, int out_type, void *out, long out_stride) {
    using namespace cnt;
    CNT_REQUIRE(V > 0 && D > 0 && D <= 1 << 30 && N >= 0, "embed_forward: bad sizes");
    CNT_REQUIRE(known_type(table_type) && known_type(out_type), "embed_forward: unknown element type");
    CNT_REQUIRE(table_stride >= 0 && out_stride >= D, "embed_forward: rows of the output overlap, or a negative stride");
    CNT_REQUIRE(table && (N == 0 || (tokens && out)), "embed_forward: null argument");
    CNT_REQUIRE(std::isfinite(scale), "embed_forward: the scale has to be finite");
    if (N == 0) return CNT_OK;
    const int wide = table_type == CNT_F32 || out_type == CNT_F32 ? 4 : 8;
    const long size = (long)element_size(out_type);
    const bool lines = reinterpret_cast<uintptr_t>(out) % kLine == 0 && (N == 1 || out_stride * size % kLine == 0);
    const int lead = lines ? 0 : kLine / (int)size - 1;
    LookupArgs a = {table, out, tokens, N, table_stride, out_stride, V, D, std::min(256, power_of_two_from((D + lead + wide - 1) / wide)), lead, scale};
    const long slots = 256 / a.lanes * kSlotsPerThread, blocks = (N + slots - 1) / slots;
    CNT_REQUIRE(blocks < 1L << 24, "embed_forward: too many slots");
    hipStream_t stream = static_cast<hipStream_t>(stream_);
    ProfileScope prof(stream, "embed_forward");
    with_type(table_type, [&](auto t) {
        with_type(out_type, [&](auto o) {
            using T = typename decltype(t)::type;
            using O = typename decltype(o)::type;
            auto kernel = lines ? embed_lookup_kernel<T, O, true> : embed_lookup_kernel<T, O, false>;
            hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), 0, stream, a);
        });
    });
    CNT_HIP(hipGetLastError());
    return CNT_OK;
}

long cnt_embed_scratch(int V, int D, long N) {
    if (!cnt::gradient_sizes(V, D, N)) return -1;
    return (long)cnt::gradient_scratch(V, D, N);
}

int cnt_embed_backward(void *stream_, int V, int D, long N, const int *tokens, float scale, int err_type, const void *err,
                       long err_stride, int grad_type, void *grad, long grad_stride, int accumulate, void *scratch,
                       size_t scratch_bytes) {
    using namespace cnt;
    CNT_REQUIRE(gradient_sizes(V, D, N), "embed_backward: bad sizes");
    CNT_REQUIRE(known_type(err_type) && known_type(grad_type), "embed_backward: unknown element type");
    CNT_REQUIRE(err_stride >= 0 && grad_stride >= D, "embed_backward: rows of the gradient overlap, or a negative stride");
    CNT_REQUIRE(std::isfinite(scale), "embed_backward: the scale has to be finite");
    const SlabPlan slabs = slab_plan(V, D, N);
    const SortPlan plan = sort_plan(V, D, N);
    const size_t need = gradient_scratch(V, D, N);
    CNT_REQUIRE(grad && scratch && (N == 0 || (tokens && err)), "embed_backward: null argument");
    CNT_REQUIRE(scratch_bytes >= need, "embed_backward: %zu bytes of scratch memory, %zu are needed", scratch_bytes, need);
    CNT_REQUIRE(reinterpret_cast<uintptr_t>(scratch) % 16 == 0, "embed_backward: the scratch memory is not aligned to 16 bytes");
    hipStream_t stream = static_cast<hipStream_t>(stream_);
    ProfileScope prof(stream, "embed_backward");
    int status = CNT_OK;
    const bool once = past_caches(grad, V, D, grad_stride, grad_type);
    if (N <= kFewSlots) {
        FewArgs few = {tokens, err, grad, err_stride, grad_stride, (int)N, V, D, 0, 0, accumulate, once, scale};
        with_type(err_type, [&](auto e) {
            with_type(grad_type, [&](auto g) { status = sum_few<typename decltype(e)::type, typename decltype(g)::type>(stream, few); });
        });
        return status;
    }
    char *mem = static_cast<char *>(scratch);
    if (slabs.slabs == 1) {
        SlabArgs s = {tokens, err, grad, nullptr, err_stride, grad_stride, (int)N, V, D, 0, 0, 0, 0, accumulate, once, 0, scale};
        with_type(err_type, [&](auto e) {
            with_type(grad_type, [&](auto g) { status = sum_slab<typename decltype(e)::type, typename decltype(g)::type>(stream, s, 1); });
        });
        return status;
    }
    if (slabs.slabs) {
        auto *index = reinterpret_cast<unsigned short *>(mem + slabs.index);
        const int dense = V <= kSlab / 2 && !accumulate;
        SlabArgs s = {tokens, err, mem, index, err_stride, D, (int)N, V, D, 0, 0, 0, 0, 0, 0, dense, 1.0f};
        with_type(err_type, [&](auto e) { status = sum_slab<typename decltype(e)::type, float>(stream, s, slabs.slabs); });
        CNT_TRY(status);
        with_type(grad_type, [&](auto g) {
            using G = typename decltype(g)::type;
            constexpr int W = kBoth<float, G>;
            const int vectors = (D + W - 1) / W;
            const long waves = ((long)V * vectors + 63) / 64;
            JoinArgs j = {reinterpret_cast<const float *>(mem), index, grad, grad_stride, slabs.slabs, V, D, vectors, waves < 2048 ? 4 : 1, dense,
                          accumulate, once, scale};
            auto kernel = slabs.slabs > 8 * j.split ? embed_slab_join_kernel<G, 16> : embed_slab_join_kernel<G, 8>;
            hipLaunchKernelGGL(kernel, dim3((unsigned)((waves * j.split + 3) / 4)), dim3(256), 0, stream, j);
        });
        CNT_HIP(hipGetLastError());
        return CNT_OK;
    }
    auto ints = [&](size_t at) { return reinterpret_cast<int *>(mem + at); };
    SortArgs s = {};
    s.counts = ints(plan.counts); s.total = ints(plan.total);
    s.N = (int)N; s.V = V; s.bits = plan.bits; s.block = plan.block; s.blocks = plan.blocks;
    // The sort and the search for runs leave most of the card idle: they bring zeros for the first rows with them, what the card writes in their
    // time (gradient of 65536 x 1024 in fp32: 73 us without).  Sixteen rows at a time are whole vectors in every type.
    const size_t row_bytes = (size_t)D * element_size(grad_type);
    const bool fills = !accumulate && grad_stride == D && (size_t)V * row_bytes >= kFillFrom;
    long filled = 0;
    auto next_fill = [&]() {
        Fill f = {};
        if (!fills) return f;
        const long rows = std::min<long>(V - filled, (long)(kFillBytes / row_bytes)) / 16 * 16;
        f.to = static_cast<char *>(grad) + (size_t)filled * row_bytes;
        f.vectors = rows * (long)row_bytes / 16;
        filled += rows;
        return f;
    };
    for (int pass = 0; pass < plan.passes; ++pass) {
        const int to = pass & 1;
        s.keys = pass ? ints(plan.keys[1 - to]) : tokens;
        s.slots = pass ? ints(plan.slots[1 - to]) : nullptr;
        s.keys_out = ints(plan.keys[to]); s.slots_out = ints(plan.slots[to]);
        s.shift = pass * plan.bits;
        s.fill = next_fill();
        const dim3 grid((unsigned)plan.blocks), block(kSortThreads);
        auto count = pass == 0 ? token_count_kernel<true> : token_count_kernel<false>;
        auto place = plan.counted ? (pass == 0 ? token_place_kernel<true, true> : token_place_kernel<false, true>)
                                  : (pass == 0 ? token_place_kernel<true, false> : token_place_kernel<false, false>);
        if (plan.counted) {
            hipLaunchKernelGGL(count, grid, block, 0, stream, s);
            CNT_HIP(hipGetLastError());
        }
        hipLaunchKernelGGL(place, dim3(plan.blocks + fill_blocks(s.fill, kSortThreads)), block, 0, stream, s);
        CNT_HIP(hipGetLastError());
    }
    const int last = (plan.passes - 1) & 1;
    SumArgs a = {};
    a.keys = ints(plan.keys[last]); a.slots = ints(plan.slots[last]); a.total = s.total;
    a.starts = ints(plan.starts);
    a.err = err; a.grad = grad; a.partial = reinterpret_cast<float *>(mem + plan.partial);
    a.err_stride = err_stride; a.grad_stride = grad_stride;
    a.V = V; a.D = D; a.piece = plan.piece; a.accumulate = accumulate; a.scale = scale;
    a.once = once;
    a.fill = next_fill();
    a.filled = (int)filled;
    with_type(err_type, [&](auto e) {
        with_type(grad_type, [&](auto g) { status = sum_runs<typename decltype(e)::type, typename decltype(g)::type>(stream, a, N); });
    });
    return status;
}

}  // extern "C"
