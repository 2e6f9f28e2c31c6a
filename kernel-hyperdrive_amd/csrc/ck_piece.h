// N consecutive elements of a row held by one lane ("a piece"; N a multiple of the 16-byte packet's elements), loaded and
// stored as whole packets, element by element where the row ends inside the piece.
#pragma once

#include "ck_device.h"

namespace ck {

// Non-temporal access to any 4-, 8- or 16-byte POD at any element's address: one instruction too (global memory takes
// unaligned addresses), a little slower where it crosses a cache line.  Rows of an odd length are full of such addresses:
// RMSNorm of 3000 x 5001 bf16 element by element took 58 us forward and 62 us backward.
template <int BYTES>
struct RawAnywhere {
    typedef uint32_t type __attribute__((ext_vector_type(BYTES / 4), aligned(1)));
};
template <>
struct RawAnywhere<4> {
    typedef uint32_t type __attribute__((aligned(1)));
};
template <typename P>
__device__ __forceinline__ P nt_load_anywhere(const void* p) {
    typedef typename RawAnywhere<sizeof(P)>::type R;
    R raw = __builtin_nontemporal_load(reinterpret_cast<const R*>(p));
    P out;
    __builtin_memcpy(&out, &raw, sizeof(P));
    return out;
}
template <typename P>
__device__ __forceinline__ void nt_store_anywhere(const P& v, void* p) {
    typedef typename RawAnywhere<sizeof(P)>::type R;
    R raw;
    __builtin_memcpy(&raw, &v, sizeof(P));
    __builtin_nontemporal_store(raw, reinterpret_cast<R*>(p));
}

template <typename T, int N>
struct Piece {
    static_assert(N % T::kVec == 0, "whole packets");
    VPack<T, T::kVec> p[N / T::kVec];
    __device__ __forceinline__ void set(int j, typename T::storage_t s) { p[j / T::kVec].v[j % T::kVec] = s; }
    __device__ __forceinline__ typename T::storage_t& at(int j) { return p[j / T::kVec].v[j % T::kVec]; }
    __device__ __forceinline__ const typename T::storage_t& at(int j) const { return p[j / T::kVec].v[j % T::kVec]; }
    __device__ __forceinline__ float up(int j) const { return T::up(at(j)); }
    __device__ __forceinline__ void put(int j, float f) { at(j) = T::down(f); }  // rounded
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int j = 0; j < N; ++j) put(j, 0.f);
    }
};

// the first n elements from src, zeros behind them; VEC: n is N and src 16-byte aligned.  STREAM: touched once (non-temporal)
template <typename T, int N, bool VEC, bool STREAM = true>
__device__ __forceinline__ Piece<T, N> load_piece(const typename T::storage_t* src, int n) {
    typedef VPack<T, T::kVec> P;
    Piece<T, N> out;
    if (VEC) {
#pragma unroll
        for (int i = 0; i < N / T::kVec; ++i) {
            const P* p = reinterpret_cast<const P*>(src) + i;
            out.p[i] = STREAM ? nt_load(p) : *p;
        }
    } else if (n >= N) {
#pragma unroll
        for (int i = 0; i < N / T::kVec; ++i) out.p[i] = nt_load_anywhere<P>(src + i * T::kVec);
    } else {
        out.clear();
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (j < n) out.at(j) = src[j];
    }
    return out;
}
template <typename T, int N, bool VEC>
__device__ __forceinline__ void store_piece(const Piece<T, N>& v, typename T::storage_t* dst, int n) {
    typedef VPack<T, T::kVec> P;
    if (VEC) {
#pragma unroll
        for (int i = 0; i < N / T::kVec; ++i) nt_store(v.p[i], reinterpret_cast<P*>(dst) + i);
    } else if (n >= N) {
#pragma unroll
        for (int i = 0; i < N / T::kVec; ++i) nt_store_anywhere(v.p[i], dst + i * T::kVec);
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (j < n) dst[j] = v.at(j);
    }
}

}  // namespace ck
