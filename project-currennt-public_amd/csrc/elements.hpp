// Elements of 32 and 16 bits: what the operators over symbols read and write.  All of them compute in 32 bits and round a result once.
#pragma once

#include "common.hpp"

namespace cnt {

inline bool known_type(int type) { return type == CNT_F32 || type == CNT_BF16 || type == CNT_F16; }
inline size_t element_size(int type) { return type == CNT_F32 ? 4 : 2; }

template <typename T>
struct Tag {
    using type = T;
};
// f(Tag<T>()) for the element type T that `type` names; the caller has checked it
template <typename F>
inline void with_type(int type, F f) {
    if (type == CNT_F32) f(Tag<float>());
    else if (type == CNT_BF16) f(Tag<__bf16>());
    else f(Tag<_Float16>());
}

// N neighbouring elements at any address that an element may have: rows of odd lengths begin anywhere, and the hardware takes 16-byte
// accesses at any address.
template <typename T, int N>
struct Packed {
    typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};
// ONCE: data that is not read again soon, or not at all, goes past the caches (512 MB: reads 6.3 -> 6.9 TB/s, copies 5.6 -> 6.2).
template <typename T, int N, bool ONCE = false>
__device__ __forceinline__ void fetch_elements(const T *p, float (&v)[N]) {
    const auto *from = reinterpret_cast<const typename Packed<T, N>::type *>(p);
    const typename Packed<T, N>::type x = ONCE ? __builtin_nontemporal_load(from) : *from;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (float)x[i];
}
template <typename T, int N, bool ONCE = false>
__device__ __forceinline__ void put_elements(T *p, const float (&v)[N]) {
    typename Packed<T, N>::type x;
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = (T)v[i];
    auto *to = reinterpret_cast<typename Packed<T, N>::type *>(p);
    if (ONCE) __builtin_nontemporal_store(x, to);
    else *to = x;
}
// A thread's columns of a row of D values: `count` from `column` on.  The last ones of a row are read `back` values earlier, so that a row of at least
// W values is read in whole vectors; a vector's first `back` values are another thread's then.
struct Columns {
    int column, count, back;
    bool whole;
};
template <int W>
__device__ __forceinline__ Columns columns_of(int column, int D) {
    const int count = max(0, min(W, D - column));
    return {column, count, D >= W && count > 0 ? W - count : 0, D >= W};
}
// W values as they stand in memory.  Conversions wait for what they convert: vectors that are to be in flight together are all asked for in front of
// them (gradient of 2261 x 132 from 17980 slots, bf16 to fp16, with the conversion behind every load: 43 us).
template <typename T, int W>
struct Vector {
    typename Packed<T, W>::type x;
    __device__ __forceinline__ void clear() { x = typename Packed<T, W>::type(0); }
    // (row: where the row begins)
    __device__ __forceinline__ void load(const T *row, const Columns &c) {
        if (c.whole) {
            x = *reinterpret_cast<const typename Packed<T, W>::type *>(row + c.column - c.back);
            return;
        }
#pragma unroll
        for (int i = 0; i < W; ++i)
            if (i < c.count) x[i] = row[c.column + i];
    }
    __device__ __forceinline__ float value(int i) const { return (float)x[i]; }
};
template <typename T, int W, bool ONCE>
__device__ __forceinline__ void put_columns(T *row, const Columns &c, const float (&v)[W]) {
    if (c.count == W) {
        put_elements<T, W, ONCE>(row + c.column, v);
        return;
    }
#pragma unroll
    for (int i = 0; i < W; ++i)
        if (i >= c.back && i - c.back < c.count) row[c.column + i - c.back] = (T)v[i];
}

// elements of a 16-byte access
template <typename T>
constexpr int kWide = 16 / (int)sizeof(T);

// elements per thread of a row that is read as T and written as O: neither access is wider than 16 bytes, so that a wave's accesses have no
// gaps (gradient of 65536 x 1024 from bf16 to fp32, two stores of 16 bytes 32 apart per thread: 159 us for its last launch, past the caches)
template <typename T, typename O>
constexpr int kBoth = kWide<T> < kWide<O> ? kWide<T> : kWide<O>;

inline int power_of_two_from(long n) {
    int p = 1;
    while (p < n) p *= 2;
    return p;
}

}  // namespace cnt
