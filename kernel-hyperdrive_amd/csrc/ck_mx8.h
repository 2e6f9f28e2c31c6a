// The 8-bit form activations are kept in between forward and backward: MXINT8 of the OCP microscaling formats.
//
// A block is 32 consecutive elements of a row (the last block of a row may be shorter).  It has one scale byte b and an
// int8 code q in [-127, 127] per element; the element stands for  q * 2^(b - 133)  (the format's element step 2^-6 times
// its scale 2^(b - 127)).  b is the smallest exponent for which the block's largest magnitude rounds to at most 127
// steps: with u the bits of that magnitude as an fp32,  b = (u + 0x10000) >> 23  - the addend carries into the exponent
// exactly when the mantissa is 255/128 or more, i.e. 127.5 steps.  b is at least 7 (steps are normal fp32 numbers) and at
// most 254; 255 marks a block that holds a NaN or an infinity and stands for 32 NaNs.
// Scaling by a power of two is exact, so the only rounding is the one to whole steps (to nearest, ties to even: half a
// step, 1/254 .. 1/127 of the block's largest magnitude), codes depend on nothing but the values, and q * 2^(b - 133) has seven
// magnitude bits: it is exact in fp32 and bf16, and in fp16 up to that type's range.
//
// Four neighbouring lanes (a quad) hold a block, eight elements ("a piece") each: 16 bytes of a 16-bit type, 8 bytes of
// codes.  The block's largest magnitude takes two register exchanges inside the quad.
#pragma once

#include "ck_piece.h"

namespace ck {

constexpr int kMxBlock = 32;
constexpr int kMxPiece = kPiece;
constexpr int kMxQuad = kMxBlock / kMxPiece;

__device__ __forceinline__ uint32_t mx_bits(float f) { return __builtin_bit_cast(uint32_t, f); }
__device__ __forceinline__ float mx_float(uint32_t u) { return __builtin_bit_cast(float, u); }

// largest of the quad's four values, in all of its lanes (quad_perm 1 0 3 2, then 2 3 0 1)
__device__ __forceinline__ uint32_t quad_max(uint32_t u) {
    const uint32_t a = (uint32_t)__builtin_amdgcn_mov_dpp((int)u, 0xB1, 0xF, 0xF, true);
    u = u > a ? u : a;
    const uint32_t b = (uint32_t)__builtin_amdgcn_mov_dpp((int)u, 0x4E, 0xF, 0xF, true);
    return u > b ? u : b;
}

// ---- pieces in 8 bits ----------------------------------------------------------------------------------------------
struct alignas(8) MxCodes {
    uint32_t w[2];
};

template <bool VEC>
__device__ __forceinline__ MxCodes load_codes(const int8_t* src, int n) {
    MxCodes c;
    if (VEC) {
        c = nt_load(reinterpret_cast<const MxCodes*>(src));
    } else {
        c.w[0] = c.w[1] = 0;
#pragma unroll
        for (int j = 0; j < kMxPiece; ++j)
            if (j < n) c.w[j / 4] |= (uint32_t)(uint8_t)src[j] << (8 * (j % 4));
    }
    return c;
}
template <bool VEC>
__device__ __forceinline__ void store_codes(const MxCodes& c, int8_t* dst, int n) {
    if (VEC) {
        nt_store(c, reinterpret_cast<MxCodes*>(dst));
    } else {
#pragma unroll
        for (int j = 0; j < kMxPiece; ++j)
            if (j < n) dst[j] = (int8_t)(c.w[j / 4] >> (8 * (j % 4)));
    }
}

// codes of this lane's piece and the scale byte of its block.  All four lanes of the quad take part; elements behind a
// row's end are zeros.
__device__ __forceinline__ MxCodes mx_encode(const float (&values)[kMxPiece], uint32_t& scale) {
    uint32_t u = 0;
#pragma unroll
    for (int j = 0; j < kMxPiece; ++j) {
        const uint32_t m = mx_bits(values[j]) & 0x7fffffffu;
        u = u > m ? u : m;
    }
    u = quad_max(u);
    uint32_t b = (u + 0x10000u) >> 23;
    b = b < 7u ? 7u : (b > 254u ? 254u : b);
    const float inverse = mx_float((260u - b) << 23);
    float v[kMxPiece];
#pragma unroll
    for (int j = 0; j < kMxPiece; ++j) v[j] = values[j];
    if (u >= 0x7f7f0000u) {
        // rare: not finite, or so close to fp32's end that the largest value rounds to 128 steps of the last exponent
        const bool finite = u < 0x7f800000u;
        const float limit = 127.f * mx_float((254u - 6u) << 23);
#pragma unroll
        for (int j = 0; j < kMxPiece; ++j) v[j] = finite ? fminf(fmaxf(v[j], -limit), limit) : 0.f;
        b = finite ? b : 255u;
    }
    scale = b;
    MxCodes c;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        uint32_t q[4];
        // 1.5 * 2^23 as addend: the sum is rounded to a whole number, whose two's complement is in its low bits
#pragma unroll
        for (int j = 0; j < 4; ++j) q[j] = mx_bits(fmaf(v[4 * i + j], inverse, 12582912.f)) & 0xffu;
        c.w[i] = q[0] | q[1] << 8 | q[2] << 16 | q[3] << 24;
    }
    return c;
}

// the step a scale byte stands for; NaN for 255
__device__ __forceinline__ float mx_step(uint32_t scale) {
    return mx_float(scale >= 255u ? 0x7fc00000u : ((scale < 7u ? 7u : scale) - 6u) << 23);
}
// the values a piece of codes stands for
__device__ __forceinline__ void mx_decode(const MxCodes& c, float step, float (&v)[kMxPiece]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t biased = c.w[i] ^ 0x80808080u;  // q + 128: unsigned bytes convert in one instruction
#pragma unroll
        for (int j = 0; j < 4; ++j) v[4 * i + j] = ((float)((biased >> (8 * j)) & 0xffu) - 128.f) * step;
    }
}

// ---- pieces of a matrix ----------------------------------------------------------------------------------------------
// p / d for p < 2^31 without a division
struct FastDiv {
    uint32_t mul, shift;
    __device__ __forceinline__ uint32_t operator()(uint32_t p) const {
        return (uint32_t)(((uint64_t)p * mul >> 32) + p) >> shift;
    }
};
static inline FastDiv fast_div(uint32_t d) {
    uint32_t shift = 0;
    while (((uint64_t)1 << shift) < d) ++shift;
    FastDiv f;
    f.mul = (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << shift) - d)) / d + 1);
    f.shift = shift;
    return f;
}

// How the pieces of a [rows, h] matrix are found from their number.  kMxFlat: h is a multiple of 32 and the rows are
// dense, so the pieces are one run and nothing is divided; kMxRows: h a multiple of 8; kMxAny: any h and alignment,
// element by element.
enum { kMxFlat = 0, kMxRows = 1, kMxAny = 2 };

struct MxShape {
    uint32_t total;     // pieces, the padding of rows to whole blocks included (fewer than 2^31)
    uint32_t per_row;   // pieces of one row: 4 * blocks
    int64_t h;          // elements of one row
    FastDiv div;        // by per_row
};
struct MxAt {
    int64_t row;
    int64_t col;    // first element of the piece in its row
    int64_t block;  // block of the row
    int n;          // elements of the piece that exist: 0 .. 8
};
template <int MODE>
__device__ __forceinline__ MxAt mx_at(const MxShape& s, uint32_t p) {
    MxAt a;
    if (MODE == kMxFlat) {
        a.row = 0;
        a.col = (int64_t)p * kMxPiece;
        a.block = p / kMxQuad;
        a.n = kMxPiece;
    } else {
        const uint32_t row = s.div(p), in_row = p - row * s.per_row;
        a.row = row;
        a.col = (int64_t)in_row * kMxPiece;
        a.block = in_row / kMxQuad;
        const int64_t left = s.h - a.col;
        a.n = left >= kMxPiece ? kMxPiece : (left > 0 ? (int)left : 0);
    }
    return a;
}
// whether piece p has elements to move
template <int MODE>
__device__ __forceinline__ bool mx_has(const MxShape& s, uint32_t p, const MxAt& a) {
    return p < s.total && (MODE == kMxFlat || a.n > 0);
}

static inline int64_t mx_blocks(int64_t h) { return (h + kMxBlock - 1) / kMxBlock; }
// false where the pieces cannot be numbered in 31 bits
static inline bool mx_shape(int64_t rows, int64_t h, MxShape* s) {
    const int64_t per_row = mx_blocks(h) * kMxQuad;
    if (per_row > 0x7fffffff || rows > 0x7fffffff || per_row * rows > 0x7fffffff) return false;
    s->total = (uint32_t)(per_row * rows);
    s->per_row = (uint32_t)per_row;
    s->h = h;
    s->div = fast_div((uint32_t)per_row);
    return true;
}

}  // namespace ck
