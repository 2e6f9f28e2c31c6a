// The 8-bit form activations are kept in between forward and backward: MXINT8 of the OCP microscaling formats.
//
// A block is 32 consecutive elements of a row (the last block of a row may be shorter).  It has one scale byte b and an
// int8 code q in [-127, 127] per element; the element stands for  q * 2^(b - 133)  (the format's element step 2^-6 times
// its scale 2^(b - 127)).  b is the smallest exponent for which the block's largest magnitude rounds to at most 127
// steps: with u the bits of that magnitude as an fp32,  b = (u + 0x10000) >> 23  - the addend carries into the exponent
// exactly when the mantissa is 255/128 or more, i.e. 127.5 steps.  A written b is at least 7 (steps are normal fp32 numbers) and at
// most 254, smaller ones are read as well; 255 marks a block that holds a NaN or an infinity and stands for 32 NaNs.
// Scaling by a power of two is exact, so the only rounding is the one to whole steps (to nearest, ties to even: half a
// step, 1/254 .. 1/127 of the block's largest magnitude), codes depend on nothing but the values, and q * 2^(b - 133) has seven
// magnitude bits: it is exact in fp32 and bf16, and in fp16 between that type's subnormal numbers and its largest.
//
// A lane holds one 16-byte packet of a block ("a piece"): eight elements of a 16-bit type, four of fp32, with as many bytes of
// codes.  So four or eight neighbouring lanes hold a block, every load and store of a wave is one run of memory, and the
// block's largest magnitude takes two or three register exchanges.  (fp32 in pieces of eight, two packets a lane, read and
// wrote every second 16 bytes per instruction: 45 instead of 33 us to read 8192 x 4096 back.)
#pragma once

#include "ck_piece.h"

namespace ck {

constexpr int kMxBlock = 32;
template <typename T>
constexpr int kMxPiece = T::kVec;               // elements of a piece
template <typename T>
constexpr int kMxLanes = kMxBlock / T::kVec;    // lanes, and pieces, of a block

__device__ __forceinline__ uint32_t mx_bits(float f) { return __builtin_bit_cast(uint32_t, f); }
__device__ __forceinline__ float mx_float(uint32_t u) { return __builtin_bit_cast(float, u); }

// largest value of the LANES (4 or 8) neighbouring lanes that hold a block, in all of them: quad_perm 1 0 3 2, then 2 3 0 1;
// behind those the quads are uniform, and the mirror image of eight lanes brings the other quad's value
template <int LANES>
__device__ __forceinline__ uint32_t mx_lanes_max(uint32_t u) {
    const uint32_t a = (uint32_t)__builtin_amdgcn_mov_dpp((int)u, 0xB1, 0xF, 0xF, true);
    u = u > a ? u : a;
    const uint32_t b = (uint32_t)__builtin_amdgcn_mov_dpp((int)u, 0x4E, 0xF, 0xF, true);
    u = u > b ? u : b;
    if (LANES == 8) {
        const uint32_t c = (uint32_t)__builtin_amdgcn_mov_dpp((int)u, 0x141, 0xF, 0xF, true);
        u = u > c ? u : c;
    }
    return u;
}

// ---- pieces in 8 bits ----------------------------------------------------------------------------------------------
template <int N>
struct alignas(N) MxCodes {
    uint32_t w[N / 4];
};

template <int N, bool VEC>
__device__ __forceinline__ MxCodes<N> load_codes(const int8_t* src, int n) {
    MxCodes<N> c;
    if (VEC) {
        c = nt_load(reinterpret_cast<const MxCodes<N>*>(src));
    } else if (n >= N) {
        c = nt_load_anywhere<MxCodes<N>>(src);
    } else {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) c.w[i] = 0;
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (j < n) c.w[j / 4] |= (uint32_t)(uint8_t)src[j] << (8 * (j % 4));
    }
    return c;
}
template <int N, bool VEC>
__device__ __forceinline__ void store_codes(const MxCodes<N>& c, int8_t* dst, int n) {
    if (VEC) {
        nt_store(c, reinterpret_cast<MxCodes<N>*>(dst));
    } else if (n >= N) {
        nt_store_anywhere(c, dst);
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (j < n) dst[j] = (int8_t)(c.w[j / 4] >> (8 * (j % 4)));
    }
}

// whole steps, packed: with 1.5 * 2^23 added the sum is rounded to a whole number, whose two's complement is in its low bits
template <int N>
__device__ __forceinline__ MxCodes<N> mx_round(const float (&v)[N], float inverse) {
    MxCodes<N> c;
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
        uint32_t q[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) q[j] = mx_bits(fmaf(v[4 * i + j], inverse, 12582912.f)) & 0xffu;
        c.w[i] = q[0] | q[1] << 8 | q[2] << 16 | q[3] << 24;
    }
    return c;
}

// codes of this lane's piece and the scale byte of its block.  All lanes of the block take part; elements behind a row's
// end are zeros.
template <int N>
__device__ __forceinline__ MxCodes<N> mx_encode(const float (&values)[N], uint32_t& scale) {
    uint32_t u = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const uint32_t m = mx_bits(values[j]) & 0x7fffffffu;
        u = u > m ? u : m;
    }
    u = mx_lanes_max<kMxBlock / N>(u);
    uint32_t b = (u + 0x10000u) >> 23;
    b = b < 7u ? 7u : (b > 254u ? 254u : b);
    scale = b;
    MxCodes<N> c = mx_round(values, mx_float((260u - b) << 23));
    if (u >= 0x7f7f0000u) {
        // rare: not finite, or so close to fp32's end that the largest value rounds to 128 steps of the last exponent
        if (u < 0x7f800000u) {
            const float limit = 127.f * mx_float((254u - 6u) << 23);
            float v[N];
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] = fminf(fmaxf(values[j], -limit), limit);
            c = mx_round(v, mx_float((260u - 254u) << 23));
        } else {
            scale = 255u;
            c = MxCodes<N>{};
        }
    }
    return c;
}

// the step 2^(scale - 133) a scale byte stands for; NaN for 255.  mx_encode writes none below 7, whose steps are subnormal
// numbers (2^-127 .. 2^-133, exact as well), but codes and scales can come from elsewhere.  (One instruction scales a number
// by a power of two, subnormal results included; putting the bits together by cases cost SwiGLU's backward 46.7 us
// instead of 44.5 at 24576 x 2 x 1408 bf16.)
__device__ __forceinline__ float mx_step(uint32_t scale) {
    return scale >= 255u ? mx_float(0x7fc00000u) : ldexpf(1.f, (int)scale - 133);
}
// the same for a byte that mx_encode wrote and nobody else: RMSNorm's backward, whose rows are kept together with their
// 1 / rms.  (There the general form costs 36.3 us instead of 32.6 for odd rows, 3000 x 5001 bf16.)
__device__ __forceinline__ float mx_step_kept(uint32_t scale) {
    return mx_float(scale >= 255u ? 0x7fc00000u : ((scale < 7u ? 7u : scale) - 6u) << 23);
}
// the codes as numbers (one conversion each, the byte picked and sign-extended on the way), and the values they stand for
template <int N>
__device__ __forceinline__ float mx_code(const MxCodes<N>& c, int j) {
    return (float)(int8_t)(c.w[j / 4] >> (8 * (j % 4)));
}
template <int N>
__device__ __forceinline__ void mx_decode(const MxCodes<N>& c, float step, float (&v)[N]) {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = mx_code(c, j) * step;
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
// dense, so the pieces are one run and nothing is divided; kMxRows: h a multiple of the piece; kMxAny: any h and
// alignment.
enum { kMxFlat = 0, kMxRows = 1, kMxAny = 2 };

struct MxShape {
    uint32_t total;     // pieces, the padding of rows to whole blocks included (fewer than 2^31)
    uint32_t per_row;   // pieces of one row: whole blocks
    int64_t h;          // elements of one row
    FastDiv div;        // by per_row
};
struct MxAt {
    int64_t row;
    int64_t col;    // first element of the piece in its row
    int64_t block;  // block of the row
    int n;          // elements of the piece that exist
};
template <int N, int MODE>
__device__ __forceinline__ MxAt mx_at(const MxShape& s, uint32_t p) {
    MxAt a;
    if (MODE == kMxFlat) {
        a.row = 0;
        a.col = (int64_t)p * N;
        a.block = p / (kMxBlock / N);
        a.n = N;
    } else {
        const uint32_t row = s.div(p), in_row = p - row * s.per_row;
        a.row = row;
        a.col = (int64_t)in_row * N;
        a.block = in_row / (kMxBlock / N);
        const int64_t left = s.h - a.col;
        a.n = left >= N ? N : (left > 0 ? (int)left : 0);
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
static inline bool mx_shape(int64_t rows, int64_t h, int piece, MxShape* s) {
    const int64_t per_row = mx_blocks(h) * (kMxBlock / piece);
    if (per_row > 0x7fffffff || rows > 0x7fffffff || per_row * rows > 0x7fffffff) return false;
    s->total = (uint32_t)(per_row * rows);
    s->per_row = (uint32_t)per_row;
    s->h = h;
    s->div = fast_div((uint32_t)per_row);
    return true;
}

}  // namespace ck
