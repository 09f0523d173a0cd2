// Norm of all gradients of a model together, and the gradients scaled down to a norm.
//
//   norm = sqrt(sum g^2),   c = norm > max_norm ? max_norm / norm : 1,   out = c * g
//
// Two launches whatever the number of tensors.  The list is cut into pieces of at most 4 KB when the set is made, a wave takes a piece at a
// time, and a workgroup leaves one sum; the second launch adds the workgroups' sums up again in every workgroup (16 KB from the L2) and
// scales.  Squares are formed and added in 64 bits: an fp32 square overflows from 1.8e19 on, and the 64-bit rate is far from what
// bounds a pass, which is memory.  Nothing is added in an order that depends on time, so a result is the same every time.
#include "elements.hpp"

#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

namespace cnt {
namespace {

struct Piece {
    const void *in;
    void *out;
    int n, type;
};
constexpr int kPieceBytes = 4096, kMostBlocks = 2048, kLineBytes = 128;

// f(offset, elements) for the vectors of a lane in a piece: all of a whole piece's accesses are asked for together
template <typename T, bool ONCE, typename F>
__device__ __forceinline__ void for_vectors(const T *p, int n, int lane, F f) {
    constexpr int N = kWide<T>, V = kPieceBytes / 16 / 64;
    if (n == V * 64 * N) {
        float v[V][N];
#pragma unroll
        for (int u = 0; u < V; ++u) fetch_elements<T, N, ONCE>(p + (u * 64 + lane) * N, v[u]);
#pragma unroll
        for (int u = 0; u < V; ++u) f((u * 64 + lane) * N, v[u]);
        return;
    }
    const int whole = n / N;
    for (int i = lane; i < whole; i += 64) {
        float v[N];
        fetch_elements<T, N, ONCE>(p + i * N, v);
        f(i * N, v);
    }
}

template <typename T>
__device__ __forceinline__ double squares(const T *p, int n, int lane) {
    constexpr int N = kWide<T>;
    double sum[N];
#pragma unroll
    for (int q = 0; q < N; ++q) sum[q] = 0.0;
    for_vectors<T, false>(p, n, lane, [&](int, const float (&v)[N]) {
#pragma unroll
        for (int q = 0; q < N; ++q) sum[q] = __builtin_fma((double)v[q], (double)v[q], sum[q]);
    });
    if (lane < n % N) {
        const double v = (double)(float)p[n / N * N + lane];
        sum[0] = __builtin_fma(v, v, sum[0]);
    }
    double s = 0.0;
#pragma unroll
    for (int q = 0; q < N; ++q) s += sum[q];
    return s;
}

__device__ __forceinline__ double block_sum(double v) {
    __shared__ double part[4];
    v = wave_sum_64(v);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    return (part[0] + part[1]) + (part[2] + part[3]);
}

__global__ __launch_bounds__(256) void gradient_squares_kernel(const Piece *__restrict__ pieces, int count, double *__restrict__ sums) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    double s = 0.0;
    for (int i = blockIdx.x * 4 + wave; i < count; i += gridDim.x * 4) {
        const Piece p = pieces[i];
        if (p.type == CNT_F32) s += squares(static_cast<const float *>(p.in), p.n, lane);
        else if (p.type == CNT_BF16) s += squares(static_cast<const __bf16 *>(p.in), p.n, lane);
        else s += squares(static_cast<const _Float16 *>(p.in), p.n, lane);
    }
    s = block_sum(s);
    if (threadIdx.x == 0) sums[blockIdx.x] = s;
}

// The factor, by all threads of a workgroup; the first workgroup's first thread writes norm and factor down.  A norm that is no finite number in
// the 32 bits in which it is reported gives the factor 0, so that whoever looks at either decides the same.
__device__ __forceinline__ float clip_factor(const double *__restrict__ sums, int count, float max_norm, float *__restrict__ result) {
    double s = 0.0;
    for (int i = threadIdx.x; i < count; i += 256) s += sums[i];
    s = block_sum(s);
    const double norm = sqrt(s);
    const float factor = !((float)norm <= 3.402823466e38f) ? 0.0f : norm > (double)max_norm ? (float)((double)max_norm / norm) : 1.0f;
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        result[0] = (float)norm;
        result[1] = factor;
    }
    return factor;
}

__global__ __launch_bounds__(256) void gradient_norm_kernel(const double *__restrict__ sums, int count, float max_norm,
                                                            float *__restrict__ result) {
    clip_factor(sums, count, max_norm, result);
}

template <typename T>
__device__ __forceinline__ void scaled(const T *in, T *out, int n, int lane, float factor) {
    constexpr int N = kWide<T>;
    for_vectors<T, true>(in, n, lane, [&](int at, float (&v)[N]) {
#pragma unroll
        for (int q = 0; q < N; ++q) v[q] = factor == 0.0f ? 0.0f : v[q] * factor;
        put_elements<T, N, true>(out + at, v);
    });
    if (lane < n % N) {
        const int at = n / N * N + lane;
        out[at] = (T)(factor == 0.0f ? 0.0f : (float)in[at] * factor);
    }
}

// Last pieces first: they are what the caches still hold of the first launch's reads.
__global__ __launch_bounds__(256) void gradient_scale_kernel(const Piece *pieces, int count, const double *__restrict__ sums, int blocks,
                                                             float max_norm, float *__restrict__ result) {
    const float factor = clip_factor(sums, blocks, max_norm, result);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (int i = blockIdx.x * 4 + wave; i < count; i += gridDim.x * 4) {
        const Piece p = pieces[count - 1 - i];
        if (factor == 1.0f && p.in == p.out) continue;
        if (p.type == CNT_F32) scaled(static_cast<const float *>(p.in), static_cast<float *>(p.out), p.n, lane, factor);
        else if (p.type == CNT_BF16) scaled(static_cast<const __bf16 *>(p.in), static_cast<__bf16 *>(p.out), p.n, lane, factor);
        else scaled(static_cast<const _Float16 *>(p.in), static_cast<_Float16 *>(p.out), p.n, lane, factor);
    }
}

}  // namespace
}  // namespace cnt

struct cnt_gradients {
    cnt::Piece *pieces = nullptr;
    double *sums = nullptr;
    int count = 0, blocks = 1;
};

namespace {
int sum_squares(cnt_gradients *set, hipStream_t stream) {
    hipLaunchKernelGGL(cnt::gradient_squares_kernel, dim3(set->blocks), dim3(256), 0, stream, set->pieces, set->count, set->sums);
    CNT_HIP(hipGetLastError());
    return CNT_OK;
}
}  // namespace

extern "C" {

int cnt_gradients_destroy(cnt_gradients *set) {
    if (!set) return CNT_OK;
    if (set->pieces) (void)hipFree(set->pieces);
    if (set->sums) (void)hipFree(set->sums);
    delete set;
    return CNT_OK;
}

int cnt_gradients_create(int count, const void *const *gradients, void *const *clipped, const long *sizes, const int *types,
                         cnt_gradients **out) {
    using namespace cnt;
    CNT_REQUIRE(out, "gradients_create: null argument");
    *out = nullptr;
    CNT_REQUIRE(count >= 0 && (count == 0 || (gradients && sizes && types)), "gradients_create: bad argument");
    try {
        std::vector<Piece> pieces;
        for (int i = 0; i < count; ++i) {
            CNT_REQUIRE(known_type(types[i]), "gradients_create: unknown element type %d of tensor %d", types[i], i);
            CNT_REQUIRE(sizes[i] >= 0, "gradients_create: negative size of tensor %d", i);
            CNT_REQUIRE(sizes[i] == 0 || (gradients[i] && (!clipped || clipped[i])), "gradients_create: null pointer of tensor %d", i);
            const size_t size = element_size(types[i]);
            const long step = kPieceBytes / (long)size;
            const char *in = static_cast<const char *>(gradients[i]);
            char *to = clipped ? static_cast<char *>(clipped[i]) : const_cast<char *>(in);
            CNT_REQUIRE(reinterpret_cast<uintptr_t>(in) % size == 0 && reinterpret_cast<uintptr_t>(to) % size == 0,
                        "gradients_create: tensor %d is not aligned to its elements", i);
            CNT_REQUIRE(sizes[i] / step + (long)pieces.size() < 0x7fffffffL - 8192, "gradients_create: too many elements");
            // a tensor that begins inside a cache line: its first piece ends with the line, so that the others read whole lines
            long n = step;
            if (reinterpret_cast<uintptr_t>(in) % kLineBytes) n = (long)((kLineBytes - reinterpret_cast<uintptr_t>(in) % kLineBytes) / size);
            for (long at = 0; at < sizes[i]; at += n, n = step)
                pieces.push_back({in + at * (long)size, to + at * (long)size, (int)std::min(n, sizes[i] - at), types[i]});
        }
        // What is written may be its own tensor's gradient and nothing else of the list: another order of the waves would give other results.
        struct Span {
            uintptr_t begin, end;
            int tensor, writes;
        };
        std::vector<Span> spans;
        for (int i = 0; i < count; ++i) {
            const uintptr_t bytes = (uintptr_t)sizes[i] * element_size(types[i]), in = reinterpret_cast<uintptr_t>(gradients[i]);
            const uintptr_t to = clipped ? reinterpret_cast<uintptr_t>(clipped[i]) : in;
            if (bytes == 0) continue;
            spans.push_back({to, to + bytes, i, 1});
            if (to != in) spans.push_back({in, in + bytes, i, 0});
        }
        std::sort(spans.begin(), spans.end(), [](const Span &a, const Span &b) { return a.begin < b.begin; });
        const Span *written = nullptr, *any = nullptr;  // those that reach furthest so far
        for (const Span &s : spans) {
            const Span *other = s.writes ? any : written;
            CNT_REQUIRE(!other || other->end <= s.begin, "gradients_create: tensors %d and %d overlap where one is written", other->tensor, s.tensor);
            if (s.writes && (!written || written->end < s.end)) written = &s;
            if (!any || any->end < s.end) any = &s;
        }
        cnt_gradients *set = new cnt_gradients;
        set->count = (int)pieces.size();
        set->blocks = std::max(1, std::min((set->count + 3) / 4, kMostBlocks));
        auto fill = [&]() -> int {
            CNT_HIP(hipMalloc((void **)&set->sums, (size_t)set->blocks * sizeof(double)));
            if (set->count == 0) return CNT_OK;
            CNT_HIP(hipMalloc((void **)&set->pieces, pieces.size() * sizeof(Piece)));
            CNT_HIP(hipMemcpy(set->pieces, pieces.data(), pieces.size() * sizeof(Piece), hipMemcpyHostToDevice));
            return CNT_OK;
        };
        const int status = fill();
        if (status != CNT_OK) {
            cnt_gradients_destroy(set);
            return status;
        }
        *out = set;
        return CNT_OK;
    } catch (const std::exception &) {
        set_error("gradients_create: out of host memory");
        return CNT_ERR_STATE;
    }
}

int cnt_opt_grad_norm(cnt_gradients *set, void *stream_, float max_norm, float *result) {
    using namespace cnt;
    CNT_REQUIRE(set && result, "opt_grad_norm: null argument");
    CNT_REQUIRE(max_norm > 0, "opt_grad_norm: the largest norm has to be positive");
    hipStream_t stream = static_cast<hipStream_t>(stream_);
    ProfileScope prof(stream, "opt_grad_norm");
    CNT_TRY(sum_squares(set, stream));
    hipLaunchKernelGGL(gradient_norm_kernel, dim3(1), dim3(256), 0, stream, set->sums, set->blocks, max_norm, result);
    CNT_HIP(hipGetLastError());
    return CNT_OK;
}

int cnt_opt_clip(cnt_gradients *set, void *stream_, float max_norm, float *result) {
    using namespace cnt;
    CNT_REQUIRE(set && result, "opt_clip: null argument");
    CNT_REQUIRE(max_norm > 0, "opt_clip: the largest norm has to be positive");
    hipStream_t stream = static_cast<hipStream_t>(stream_);
    ProfileScope prof(stream, "opt_clip");
    CNT_TRY(sum_squares(set, stream));
    hipLaunchKernelGGL(gradient_scale_kernel, dim3(set->blocks), dim3(256), 0, stream, set->pieces, set->count, set->sums, set->blocks,
                       max_norm, result);
    CNT_HIP(hipGetLastError());
    return CNT_OK;
}

}  // extern "C"
