// Activations in 8 bits (ck_mx8.h) for gfx950: writing and reading them, SwiGLU forward with its inputs kept in 8 bits and
// its backward from them, and the routing weights' gradient from expert outputs kept in 8 bits.
// HBM-bound streaming kernels in the manner of swiglu.hip: a lane moves 16-byte pieces, several in flight, fp32
// math, one rounding on store.
#include "ck_mx8.h"

namespace ck {

constexpr int kMxThreads = 256;
// Pieces per lane of the two that move one tensor; the SwiGLU kernels move two or three and take one.  16384 x 4096 bf16:
// quantize 35.5 / 32.5 / 34.8 us with 1 / 2 / 4 pieces, dequantize 33.5 / 33.7 / 34.7; SwiGLU backward 85.0 / 87.3 with 1 / 2.
constexpr int kMxUnroll = 2;

template <typename T, int MODE>
__global__ void __launch_bounds__(kMxThreads)
    mx8_quantize_kernel(const typename T::storage_t* __restrict__ x, int8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                        MxShape shape) {
    constexpr int N = kMxPiece<T>, LANES = kMxLanes<T>;
    constexpr bool VEC = MODE != kMxAny;
    const int64_t blocks = shape.per_row / LANES;
    const uint32_t base = blockIdx.x * (kMxThreads * kMxUnroll) + threadIdx.x;
    Piece<T, N> in[kMxUnroll];
#pragma unroll
    for (int i = 0; i < kMxUnroll; ++i) {
        const uint32_t p = base + i * kMxThreads;
        const MxAt a = mx_at<N, MODE>(shape, p);
        if (mx_has<MODE>(shape, p, a)) in[i] = load_piece<T, N, VEC>(x + a.row * shape.h + a.col, a.n);
        else in[i].clear();
    }
#pragma unroll
    for (int i = 0; i < kMxUnroll; ++i) {
        const uint32_t p = base + i * kMxThreads;
        const MxAt a = mx_at<N, MODE>(shape, p);
        float v[N];
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = in[i].up(j);
        uint32_t scale;
        const MxCodes<N> c = mx_encode(v, scale);
        if (mx_has<MODE>(shape, p, a)) {
            store_codes<N, VEC>(c, codes + a.row * shape.h + a.col, a.n);
            if (threadIdx.x % LANES == 0) scales[a.row * blocks + a.block] = (uint8_t)scale;
        }
    }
}

// What a kept value becomes in its storage type: itself, but that a block near fp16's end may stand for a value beyond it
// (65504 is kept as 64 steps of 1024), which becomes the largest finite number.
template <typename T>
__device__ __forceinline__ float mx_limit(float v) {
    return v;
}
template <>
__device__ __forceinline__ float mx_limit<F16>(float v) {
    return v > 65504.f ? 65504.f : (v < -65504.f ? -65504.f : v);  // (a NaN fails both comparisons)
}

template <typename T, int MODE>
__global__ void __launch_bounds__(kMxThreads)
    mx8_dequantize_kernel(const int8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                          typename T::storage_t* __restrict__ out, MxShape shape) {
    constexpr int N = kMxPiece<T>, LANES = kMxLanes<T>;
    constexpr bool VEC = MODE != kMxAny;
    const int64_t blocks = shape.per_row / LANES;
    const uint32_t base = blockIdx.x * (kMxThreads * kMxUnroll) + threadIdx.x;
    MxCodes<N> in[kMxUnroll];
    uint32_t scale[kMxUnroll];
#pragma unroll
    for (int i = 0; i < kMxUnroll; ++i) {
        const uint32_t p = base + i * kMxThreads;
        const MxAt a = mx_at<N, MODE>(shape, p);
        in[i] = MxCodes<N>{};
        scale[i] = 7;
        if (mx_has<MODE>(shape, p, a)) {
            in[i] = load_codes<N, VEC>(codes + a.row * shape.h + a.col, a.n);
            scale[i] = scales[a.row * blocks + a.block];
        }
    }
#pragma unroll
    for (int i = 0; i < kMxUnroll; ++i) {
        const uint32_t p = base + i * kMxThreads;
        const MxAt a = mx_at<N, MODE>(shape, p);
        if (mx_has<MODE>(shape, p, a)) {
            const float step = mx_step(scale[i]);
            Piece<T, N> o;
#pragma unroll
            for (int j = 0; j < N; ++j) o.put(j, mx_limit<T>(mx_code(in[i], j) * step));
            store_piece<T, N, VEC>(o, out + a.row * shape.h + a.col, a.n);
        }
    }
}

// ---- SwiGLU ----------------------------------------------------------------------------------------------------------
// gate, up: rows of h elements ld apart (one tensor each, or the halves of one); codes and scales likewise, with distances
// of their own.
struct MxStrides {
    int64_t x, codes, scales;
};

template <typename T, int MODE>
__global__ void __launch_bounds__(kMxThreads)
    swiglu_fwd_mx8_kernel(const typename T::storage_t* __restrict__ gate, const typename T::storage_t* __restrict__ up,
                          typename T::storage_t* __restrict__ out, int8_t* __restrict__ gate_codes,
                          int8_t* __restrict__ up_codes, uint8_t* __restrict__ gate_scales, uint8_t* __restrict__ up_scales,
                          MxStrides ld, MxShape shape) {
    constexpr int N = kMxPiece<T>, LANES = kMxLanes<T>;
    constexpr bool VEC = MODE != kMxAny;
    const uint32_t p = blockIdx.x * kMxThreads + threadIdx.x;
    const MxAt a = mx_at<N, MODE>(shape, p);
    const bool has = mx_has<MODE>(shape, p, a);
    Piece<T, N> g, u, y;
    if (has) {
        g = load_piece<T, N, VEC>(gate + a.row * ld.x + a.col, a.n);
        u = load_piece<T, N, VEC>(up + a.row * ld.x + a.col, a.n);
    } else {
        g.clear();
        u.clear();
    }
    float gv[N], uv[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
        gv[j] = g.up(j);
        uv[j] = u.up(j);
        y.put(j, swiglu_fwd_1<T>(gv[j], uv[j]));
    }
    uint32_t gs, us;
    const MxCodes<N> gc = mx_encode(gv, gs), uc = mx_encode(uv, us);
    if (has) {
        store_piece<T, N, VEC>(y, out + a.row * shape.h + a.col, a.n);
        store_codes<N, VEC>(gc, gate_codes + a.row * ld.codes + a.col, a.n);
        store_codes<N, VEC>(uc, up_codes + a.row * ld.codes + a.col, a.n);
        if (threadIdx.x % LANES == 0) {
            gate_scales[a.row * ld.scales + a.block] = (uint8_t)gs;
            up_scales[a.row * ld.scales + a.block] = (uint8_t)us;
        }
    }
}

// ACT: also writes the activation the kept inputs give (for the next product's weight gradient)
template <typename T, int MODE, bool ACT>
__global__ void __launch_bounds__(kMxThreads)
    swiglu_bwd_mx8_kernel(const int8_t* __restrict__ gate_codes, const int8_t* __restrict__ up_codes,
                          const uint8_t* __restrict__ gate_scales, const uint8_t* __restrict__ up_scales,
                          const typename T::storage_t* __restrict__ dy, typename T::storage_t* __restrict__ dgate,
                          typename T::storage_t* __restrict__ dup, typename T::storage_t* __restrict__ act, MxStrides ld,
                          MxShape shape) {
    constexpr int N = kMxPiece<T>;
    constexpr bool VEC = MODE != kMxAny;
    const uint32_t p = blockIdx.x * kMxThreads + threadIdx.x;
    const MxAt a = mx_at<N, MODE>(shape, p);
    if (!mx_has<MODE>(shape, p, a)) return;
    const MxCodes<N> gc = load_codes<N, VEC>(gate_codes + a.row * ld.codes + a.col, a.n);
    const MxCodes<N> uc = load_codes<N, VEC>(up_codes + a.row * ld.codes + a.col, a.n);
    const float gs = mx_step(gate_scales[a.row * ld.scales + a.block]), us = mx_step(up_scales[a.row * ld.scales + a.block]);
    const Piece<T, N> d = load_piece<T, N, VEC>(dy + a.row * shape.h + a.col, a.n);
    Piece<T, N> og, ou, oa;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const float g = mx_code(gc, j) * gs, u = mx_code(uc, j) * us, dy1 = d.up(j);
        const float s = sigmoidf_<T>(g), gsig = g * s;
        og.put(j, dy1 * u * (s + gsig * (1.0f - s)));
        ou.put(j, dy1 * gsig);
        if (ACT) oa.put(j, u * gsig);
    }
    store_piece<T, N, VEC>(og, dgate + a.row * ld.x + a.col, a.n);
    store_piece<T, N, VEC>(ou, dup + a.row * ld.x + a.col, a.n);
    if (ACT) store_piece<T, N, VEC>(oa, act + a.row * shape.h + a.col, a.n);
}

// ---- routing weights' gradient: d_gates[t, s] = <expert output s of token t (kept in 8 bits), grad_out[t]> ------------------
// one wavefront per token, as in moe_combine.hip
template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
    combine_bwd_gates_mx8_kernel(const int8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                 const typename T::storage_t* __restrict__ grad_out,
                                 typename T::storage_t* __restrict__ d_gates, int64_t tokens, int k, int64_t H) {
    constexpr int N = kMxPiece<T>;
    const int64_t t = (int64_t)blockIdx.x * 4 + threadIdx.x / CK_WAVE;
    if (t >= tokens) return;
    const int lane = lane_id();
    const int64_t blocks = (H + kMxBlock - 1) / kMxBlock;
    const int64_t pieces = (H + N - 1) / N;
    const typename T::storage_t* dy = grad_out + t * H;
    for (int s = 0; s < k; ++s) {
        const int64_t row = t * k + s;
        float acc = 0.f;
        for (int64_t p = lane; p < pieces; p += CK_WAVE) {
            const int64_t left = H - p * N;
            const int n = left >= N ? N : (int)left;
            const MxCodes<N> c = load_codes<N, VEC>(codes + row * H + p * N, n);
            const float step = mx_step(scales[row * blocks + p / (kMxBlock / N)]);
            const Piece<T, N> b = load_piece<T, N, VEC, false>(dy + p * N, n);  // (re-read per slot: stays in the caches)
            float v[N];
            mx_decode(c, step, v);
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (VEC || j < n) acc += v[j] * b.up(j);
        }
        acc = wave_sum(acc);
        if (lane == 0) d_gates[row] = T::down(acc);
    }
}

}  // namespace ck

// ---- host side ---------------------------------------------------------------------------------------------------------
static int mx_piece(int dtype) { return dtype == CK_F32 ? 4 : 8; }
static bool aligned8(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 7u) == 0; }

// kMxRows wherever every row starts on a whole packet, kMxFlat where the rows are one run besides
static int mx_mode(int64_t h, int piece, bool aligned, bool dense) {
    if (!aligned || h % piece != 0) return ck::kMxAny;
    return dense && h % ck::kMxBlock == 0 ? ck::kMxFlat : ck::kMxRows;
}

#define CK_MX_MODE(mode, ...)                              \
    if ((mode) == ck::kMxFlat) {                           \
        constexpr int MODE = ck::kMxFlat;                  \
        __VA_ARGS__;                                       \
    } else if ((mode) == ck::kMxRows) {                    \
        constexpr int MODE = ck::kMxRows;                  \
        __VA_ARGS__;                                       \
    } else {                                               \
        constexpr int MODE = ck::kMxAny;                   \
        __VA_ARGS__;                                       \
    }

static dim3 mx_grid(const ck::MxShape& s, int unroll) {
    return dim3((unsigned)ck_ceil_div((int64_t)s.total, (int64_t)ck::kMxThreads * unroll));
}
static bool mx_dtype(int dtype) { return dtype == CK_F32 || dtype == CK_F16 || dtype == CK_BF16; }

extern "C" int ck_mx8_quantize(const void* x, void* codes, void* scales, int64_t rows, int64_t H, int dtype, void* stream) {
    if (rows < 0 || H < 0) return CK_ERR_SHAPE;
    if (!mx_dtype(dtype)) return CK_ERR_DTYPE;
    if (rows == 0 || H == 0) return CK_OK;
    if (!x || !codes || !scales) return CK_ERR_NULL;
    if (!ck_aligned_elem(x, dtype)) return CK_ERR_ALIGN;
    ck::MxShape shape;
    if (!ck::mx_shape(rows, H, mx_piece(dtype), &shape)) return CK_ERR_SHAPE;
    hipStream_t s = (hipStream_t)stream;
    const int mode = mx_mode(H, mx_piece(dtype), ck_aligned16(x) && aligned8(codes), true);
    CK_DISPATCH_DTYPE(dtype, {
        typedef typename T::storage_t S;
        CK_MX_MODE(mode, {
            hipLaunchKernelGGL((ck::mx8_quantize_kernel<T, MODE>), mx_grid(shape, ck::kMxUnroll), dim3(ck::kMxThreads), 0, s,
                               (const S*)x, (int8_t*)codes, (uint8_t*)scales, shape);
        });
    });
    return ck_launch_status();
}

extern "C" int ck_mx8_dequantize(const void* codes, const void* scales, void* output, int64_t rows, int64_t H, int dtype,
                                 void* stream) {
    if (rows < 0 || H < 0) return CK_ERR_SHAPE;
    if (!mx_dtype(dtype)) return CK_ERR_DTYPE;
    if (rows == 0 || H == 0) return CK_OK;
    if (!codes || !scales || !output) return CK_ERR_NULL;
    if (!ck_aligned_elem(output, dtype)) return CK_ERR_ALIGN;
    ck::MxShape shape;
    if (!ck::mx_shape(rows, H, mx_piece(dtype), &shape)) return CK_ERR_SHAPE;
    hipStream_t s = (hipStream_t)stream;
    const int mode = mx_mode(H, mx_piece(dtype), ck_aligned16(output) && aligned8(codes), true);
    CK_DISPATCH_DTYPE(dtype, {
        typedef typename T::storage_t S;
        CK_MX_MODE(mode, {
            hipLaunchKernelGGL((ck::mx8_dequantize_kernel<T, MODE>), mx_grid(shape, ck::kMxUnroll), dim3(ck::kMxThreads), 0, s,
                               (const int8_t*)codes, (const uint8_t*)scales, (S*)output, shape);
        });
    });
    return ck_launch_status();
}

extern "C" int ck_swiglu_forward_mx8(const void* gate, const void* up, int64_t ldx, void* output, void* gate_codes,
                                     void* up_codes, int64_t ldc, void* gate_scales, void* up_scales, int64_t lds,
                                     int64_t rows, int64_t H, int dtype, void* stream) {
    if (rows < 0 || H < 0 || ldx < H || ldc < H || lds < ck::mx_blocks(H)) return CK_ERR_SHAPE;
    if (!mx_dtype(dtype)) return CK_ERR_DTYPE;
    if (rows == 0 || H == 0) return CK_OK;
    if (!gate || !up || !output || !gate_codes || !up_codes || !gate_scales || !up_scales) return CK_ERR_NULL;
    if (!ck_aligned_elem(gate, dtype) || !ck_aligned_elem(up, dtype) || !ck_aligned_elem(output, dtype)) return CK_ERR_ALIGN;
    ck::MxShape shape;
    if (!ck::mx_shape(rows, H, mx_piece(dtype), &shape)) return CK_ERR_SHAPE;
    hipStream_t s = (hipStream_t)stream;
    const bool aligned = ck_aligned16(gate) && ck_aligned16(up) && ck_aligned16(output) && aligned8(gate_codes) &&
                         aligned8(up_codes) && ldx % mx_piece(dtype) == 0 && ldc % mx_piece(dtype) == 0;
    const bool dense = ldx == H && ldc == H && lds == ck::mx_blocks(H);
    const int mode = mx_mode(H, mx_piece(dtype), aligned, dense);
    const ck::MxStrides ld = {ldx, ldc, lds};
    CK_DISPATCH_DTYPE(dtype, {
        typedef typename T::storage_t S;
        CK_MX_MODE(mode, {
            hipLaunchKernelGGL((ck::swiglu_fwd_mx8_kernel<T, MODE>), mx_grid(shape, 1), dim3(ck::kMxThreads), 0, s,
                               (const S*)gate, (const S*)up, (S*)output, (int8_t*)gate_codes, (int8_t*)up_codes,
                               (uint8_t*)gate_scales, (uint8_t*)up_scales, ld, shape);
        });
    });
    return ck_launch_status();
}

extern "C" int ck_swiglu_backward_mx8(const void* gate_codes, const void* up_codes, int64_t ldc, const void* gate_scales,
                                      const void* up_scales, int64_t lds, const void* output_grad, void* gate_grad,
                                      void* up_grad, int64_t ldx, void* activation, int64_t rows, int64_t H, int dtype,
                                      void* stream) {
    if (rows < 0 || H < 0 || ldx < H || ldc < H || lds < ck::mx_blocks(H)) return CK_ERR_SHAPE;
    if (!mx_dtype(dtype)) return CK_ERR_DTYPE;
    if (rows == 0 || H == 0) return CK_OK;
    if (!gate_codes || !up_codes || !gate_scales || !up_scales || !output_grad || !gate_grad || !up_grad) return CK_ERR_NULL;
    if (!ck_aligned_elem(output_grad, dtype) || !ck_aligned_elem(gate_grad, dtype) || !ck_aligned_elem(up_grad, dtype) ||
        !ck_aligned_elem(activation, dtype))
        return CK_ERR_ALIGN;
    ck::MxShape shape;
    if (!ck::mx_shape(rows, H, mx_piece(dtype), &shape)) return CK_ERR_SHAPE;
    hipStream_t s = (hipStream_t)stream;
    const bool aligned = ck_aligned16(output_grad) && ck_aligned16(gate_grad) && ck_aligned16(up_grad) &&
                         ck_aligned16(activation) && aligned8(gate_codes) && aligned8(up_codes) &&
                         ldx % mx_piece(dtype) == 0 && ldc % mx_piece(dtype) == 0;
    const bool dense = ldx == H && ldc == H && lds == ck::mx_blocks(H);
    const int mode = mx_mode(H, mx_piece(dtype), aligned, dense);
    const ck::MxStrides ld = {ldx, ldc, lds};
    CK_DISPATCH_DTYPE(dtype, {
        typedef typename T::storage_t S;
        CK_MX_MODE(mode, {
            if (activation)
                hipLaunchKernelGGL((ck::swiglu_bwd_mx8_kernel<T, MODE, true>), mx_grid(shape, 1), dim3(ck::kMxThreads), 0, s,
                                   (const int8_t*)gate_codes, (const int8_t*)up_codes, (const uint8_t*)gate_scales,
                                   (const uint8_t*)up_scales, (const S*)output_grad, (S*)gate_grad, (S*)up_grad,
                                   (S*)activation, ld, shape);
            else
                hipLaunchKernelGGL((ck::swiglu_bwd_mx8_kernel<T, MODE, false>), mx_grid(shape, 1), dim3(ck::kMxThreads), 0,
                                   s, (const int8_t*)gate_codes, (const int8_t*)up_codes, (const uint8_t*)gate_scales,
                                   (const uint8_t*)up_scales, (const S*)output_grad, (S*)gate_grad, (S*)up_grad,
                                   (S*)nullptr, ld, shape);
        });
    });
    return ck_launch_status();
}

extern "C" int ck_moe_combine_backward_gates_mx8(const void* codes, const void* scales, const void* grad_out, void* d_gates,
                                                 int64_t tokens, int64_t k, int64_t H, int dtype, void* stream) {
    if (tokens < 0 || k <= 0 || H < 0 || k > 0x7fffffff) return CK_ERR_SHAPE;
    if (!mx_dtype(dtype)) return CK_ERR_DTYPE;
    if (tokens == 0) return CK_OK;
    if (!d_gates || (H > 0 && (!codes || !scales || !grad_out))) return CK_ERR_NULL;
    if (!ck_aligned_elem(grad_out, dtype) || !ck_aligned_elem(d_gates, dtype)) return CK_ERR_ALIGN;
    const int64_t grid = ck_ceil_div(tokens, 4);
    if (grid > 0x7fffffff) return CK_ERR_SHAPE;
    hipStream_t s = (hipStream_t)stream;
    const bool vec = aligned8(codes) && ck_aligned16(grad_out) && H % mx_piece(dtype) == 0;
    CK_DISPATCH_DTYPE(dtype, {
        typedef typename T::storage_t S;
        if (vec)
            hipLaunchKernelGGL((ck::combine_bwd_gates_mx8_kernel<T, true>), dim3((unsigned)grid), dim3(256), 0, s,
                               (const int8_t*)codes, (const uint8_t*)scales, (const S*)grad_out, (S*)d_gates, tokens, (int)k, H);
        else
            hipLaunchKernelGGL((ck::combine_bwd_gates_mx8_kernel<T, false>), dim3((unsigned)grid), dim3(256), 0, s,
                               (const int8_t*)codes, (const uint8_t*)scales, (const S*)grad_out, (S*)d_gates, tokens, (int)k, H);
    });
    return ck_launch_status();
}
