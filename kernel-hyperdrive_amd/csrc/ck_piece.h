// Eight consecutive elements of a row held by one lane ("a piece"): 16 bytes of a 16-bit type, 32 of fp32, loaded and stored
// as whole packets where alignment allows, element by element where it does not or the row ends inside the piece.
#pragma once

#include "ck_device.h"

namespace ck {

constexpr int kPiece = 8;

template <typename T>
struct Piece {
    VPack<T, T::kVec> p[kPiece / T::kVec];
    __device__ __forceinline__ void set(int j, typename T::storage_t s) { p[j / T::kVec].v[j % T::kVec] = s; }
    __device__ __forceinline__ typename T::storage_t& at(int j) { return p[j / T::kVec].v[j % T::kVec]; }
    __device__ __forceinline__ const typename T::storage_t& at(int j) const { return p[j / T::kVec].v[j % T::kVec]; }
    __device__ __forceinline__ float up(int j) const { return T::up(at(j)); }
    __device__ __forceinline__ void put(int j, float f) { at(j) = T::down(f); }  // rounded
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int j = 0; j < kPiece; ++j) put(j, 0.f);
    }
};

// the first n elements from src, zeros behind them; VEC: n is 8 and src 16-byte aligned.  STREAM: touched once (non-temporal)
template <typename T, bool VEC, bool STREAM = true>
__device__ __forceinline__ Piece<T> load_piece(const typename T::storage_t* src, int n) {
    typedef VPack<T, T::kVec> P;
    Piece<T> out;
    if (VEC) {
#pragma unroll
        for (int i = 0; i < kPiece / T::kVec; ++i) {
            const P* p = reinterpret_cast<const P*>(src) + i;
            out.p[i] = STREAM ? nt_load(p) : *p;
        }
    } else {
        out.clear();
#pragma unroll
        for (int j = 0; j < kPiece; ++j)
            if (j < n) out.at(j) = src[j];
    }
    return out;
}
template <typename T, bool VEC>
__device__ __forceinline__ void store_piece(const Piece<T>& v, typename T::storage_t* dst, int n) {
    typedef VPack<T, T::kVec> P;
    if (VEC) {
#pragma unroll
        for (int i = 0; i < kPiece / T::kVec; ++i) nt_store(v.p[i], reinterpret_cast<P*>(dst) + i);
    } else {
#pragma unroll
        for (int j = 0; j < kPiece; ++j)
            if (j < n) dst[j] = v.at(j);
    }
}

}  // namespace ck
