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

// A value rounded to an element. The f32 value is made to stand first: a product that meets the conversion to f16 directly would become one
// instruction with one rounding (v_fma_mix), and the value would depend on what the compiler saw.
template <int ET>
__device__ __forceinline__ typename Elem<ET>::T elem_of(float v) {
    if constexpr (ET == kElemF16) __asm__("" : "+v"(v));
    return (typename Elem<ET>::T)v;
}

// Elements of a 16-byte piece, and a piece as f32.
template <int ET>
constexpr int kElemPiece = ET == kElemF32 ? 4 : 8;
template <int ET>
__device__ __forceinline__ void elem_unpack(uint4 p, float (&out)[kElemPiece<ET>]) {
    const u32 w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (ET == kElemF32) {
            out[i] = bm_bits_f32(w[i]);
        } else if constexpr (ET == kElemBF16) {
            out[2 * i] = bm_bits_f32(w[i] << 16);
            out[2 * i + 1] = bm_bits_f32(w[i] & 0xffff0000u);
        } else {
            out[2 * i] = bm_half_to_f32(w[i] & 0xffffu);
            out[2 * i + 1] = bm_half_to_f32(w[i] >> 16);
        }
    }
}
template <int ET>
__device__ __forceinline__ uint4 elem_pack(const float (&in)[kElemPiece<ET>]) {
    typename Elem<ET>::T t[kElemPiece<ET>];
#pragma unroll
    for (int i = 0; i < kElemPiece<ET>; i++) t[i] = elem_of<ET>(in[i]);
    uint4 p;
    __builtin_memcpy(&p, t, 16);
    return p;
}
template <int ET>
__device__ __forceinline__ uint4 elem_piece(const void *base, size_t at) {
    return bm_ld16u(reinterpret_cast<const uint8_t *>(static_cast<const typename Elem<ET>::T *>(base) + at));
}
template <int ET>
__device__ __forceinline__ void elem_piece_store(void *base, size_t at, uint4 p) {
    __builtin_memcpy(static_cast<typename Elem<ET>::T *>(base) + at, &p, 16);
}
template <int ET>
__device__ __forceinline__ float elem_load1(const void *base, size_t at) {
    return (float)static_cast<const typename Elem<ET>::T *>(base)[at];
}
template <int ET>
__device__ __forceinline__ void elem_store1(void *base, size_t at, float v) {
    static_cast<typename Elem<ET>::T *>(base)[at] = elem_of<ET>(v);
}
// Keeps the compiler from making one of the two ways to the same elements (whole pieces, single ones): it would take the pieces apart.
__device__ __forceinline__ size_t elem_apart(size_t at) {
    u32 zero = 0;
    __asm__("" : "+v"(zero));
    return at + zero;
}
// N values (whole pieces, or half a one) from `at` on, of which the first `have` (1 .. N) are there; the others are zero, and not read.
template <int ET, int N>
__device__ __forceinline__ void elem_load_some(const void *base, size_t at, u32 have, float (&out)[N]) {
    constexpr int V = kElemPiece<ET>;
    static_assert(N % V == 0, "whole pieces");
    if (have >= (u32)N) {
#pragma unroll
        for (int i = 0; i < N; i += V) {
            float v[V];
            elem_unpack<ET>(elem_piece<ET>(base, at + i), v);
#pragma unroll
            for (int j = 0; j < V; j++) out[i + j] = v[j];
        }
        return;
    }
    at = elem_apart(at);
#pragma unroll
    for (int i = 0; i < N; i++) out[i] = (u32)i < have ? elem_load1<ET>(base, at + i) : 0.0f;
}
template <int ET, int N>
__device__ __forceinline__ void elem_store_some(void *base, size_t at, u32 have, const float (&in)[N]) {
    constexpr int V = kElemPiece<ET>;
    if (have >= (u32)N) {
        if constexpr (N % V == 0) {
#pragma unroll
            for (int i = 0; i < N; i += V) {
                float v[V];
#pragma unroll
                for (int j = 0; j < V; j++) v[j] = in[i + j];
                elem_piece_store<ET>(base, at + i, elem_pack<ET>(v));
            }
        } else {
            static_assert(2 * N == V, "half a piece");
            typename Elem<ET>::T t[N];
#pragma unroll
            for (int j = 0; j < N; j++) t[j] = elem_of<ET>(in[j]);
            __builtin_memcpy(static_cast<typename Elem<ET>::T *>(base) + at, t, sizeof t);
        }
        return;
    }
    at = elem_apart(at);
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
