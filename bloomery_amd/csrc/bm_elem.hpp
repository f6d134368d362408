// Rows of f32, f16 or bf16 values: loads into f32, stores with one rounding to nearest even. Global memory takes unaligned vector
// accesses on this target, so eight values are one or two 16-byte requests whatever the row's alignment (the element's own is all
// that is asked for).
#ifndef BM_ELEM_HPP
#define BM_ELEM_HPP

#include "bm_stream.hpp"

namespace bmk {

constexpr int kElemF32 = 0, kElemF16 = 1, kElemBF16 = 30; // ggml's numbers

template <int ET>
struct Elem;
template <>
struct Elem<kElemF32> {
    typedef float T;
};
template <>
struct Elem<kElemF16> {
    typedef _Float16 T;
};
template <>
struct Elem<kElemBF16> {
    typedef __bf16 T;
};
inline int elem_bytes(int et) { return et == kElemF32 ? 4 : 2; }

template <int ET, int N>
struct ElemVec {
    typename Elem<ET>::T v[N];
};

template <int ET, int N>
__device__ __forceinline__ void elem_load(const void *base, size_t at, float (&out)[N]) {
    ElemVec<ET, N> r;
    __builtin_memcpy(&r, static_cast<const typename Elem<ET>::T *>(base) + at, sizeof r);
#pragma unroll
    for (int i = 0; i < N; i++) out[i] = (float)r.v[i];
}
template <int ET, int N>
__device__ __forceinline__ void elem_store(void *base, size_t at, const float (&in)[N]) {
    ElemVec<ET, N> r;
#pragma unroll
    for (int i = 0; i < N; i++) r.v[i] = (typename Elem<ET>::T)in[i];
    __builtin_memcpy(static_cast<typename Elem<ET>::T *>(base) + at, &r, sizeof r);
}
template <int ET>
__device__ __forceinline__ float elem_load1(const void *base, size_t at) {
    return (float)static_cast<const typename Elem<ET>::T *>(base)[at];
}
template <int ET>
__device__ __forceinline__ void elem_store1(void *base, size_t at, float v) {
    static_cast<typename Elem<ET>::T *>(base)[at] = (typename Elem<ET>::T)v;
}
// N values from `at` on, of which the first `have` (1 .. N) are there; the others are zero, and not read.
template <int ET, int N>
__device__ __forceinline__ void elem_load_some(const void *base, size_t at, u32 have, float (&out)[N]) {
    if (have >= (u32)N) return elem_load<ET, N>(base, at, out);
#pragma unroll
    for (int i = 0; i < N; i++) out[i] = (u32)i < have ? elem_load1<ET>(base, at + i) : 0.0f;
}
template <int ET, int N>
__device__ __forceinline__ void elem_store_some(void *base, size_t at, u32 have, const float (&in)[N]) {
    if (have >= (u32)N) return elem_store<ET, N>(base, at, in);
#pragma unroll
    for (int i = 0; i < N; i++)
        if ((u32)i < have) elem_store1<ET>(base, at + i, in[i]);
}

// Sum over a wave, in every lane, in a fixed order.
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d, 64);
    return v;
}

} // namespace bmk

#endif // BM_ELEM_HPP
