// RMSNorm that keeps its input in 8 bits (ck_mx8.h) for the backward, for gfx950.
//   forward : s = x (+ residual, rounded);  r = 1 / sqrt(mean s^2 + eps);  y = s r w;  writes y, r, the 8-bit form of s
//             (and s itself with a residual)
//   backward: with s^ the kept row:  dx = r (dy w - s^ r^2 mean(dy w s^)) (+ the sum's own gradient),  dw = sum dy s^ r
// The row (forward: as read; backward: codes and dy) stays in the registers of a team of TPR lanes, so it is read once;
// row sums are wave64 shuffles, wider teams meet through LDS.  A lane holds pieces of eight elements, lane t the pieces
// t, t + TPR, ..: the four lanes of a quad hold one block.  Backward: every team walks rows and keeps its share of dw in
// fp32 registers; a workgroup writes one partial row, a second launch adds the partial rows up.  No atomics.
#include "ck_mx8.h"

namespace ck {

constexpr int kMxMaxPieces = 8;  // of a lane

template <int TPR>
__device__ __forceinline__ float mx_team_sum(float v, float* red) {
    v = wave_sum(v);
    if (TPR > CK_WAVE) {
        __syncthreads();  // the previous use of `red`
        if (lane_id() == 0) red[threadIdx.x / CK_WAVE] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int w = 0; w < TPR / CK_WAVE; ++w) v += red[w];
    }
    return v;
}

__device__ __forceinline__ int mx_piece_size(int H, int p) {
    const int left = H - p * kMxPiece;
    return left >= kMxPiece ? kMxPiece : (left > 0 ? left : 0);
}

// one row per team; NP pieces a lane at most
template <typename T, int TPR, int NP, bool RES, bool VEC>
__global__ void __launch_bounds__(TPR > 256 ? TPR : 256)
    rmsnorm_fwd_mx8_kernel(const typename T::storage_t* __restrict__ x, const typename T::storage_t* __restrict__ res,
                           const typename T::storage_t* __restrict__ w, typename T::storage_t* __restrict__ y,
                           typename T::storage_t* __restrict__ res_out, int8_t* __restrict__ codes,
                           uint8_t* __restrict__ scales, float* __restrict__ rstd_out, int64_t B, int H, float eps) {
    __shared__ float red[16];
    const int t = threadIdx.x % TPR;
    const int64_t row = (int64_t)blockIdx.x * (blockDim.x / TPR) + threadIdx.x / TPR;
    if (row >= B) return;  // (a whole team; with TPR > 64 the workgroup is one team)
    const int blocks = (H + kMxBlock - 1) / kMxBlock;
    const typename T::storage_t* xr = x + row * H;
    Piece<T> v[NP], r[RES ? NP : 1];
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int p = t + i * TPR, n = mx_piece_size(H, p);
        if (n > 0) {
            v[i] = load_piece<T, VEC>(xr + p * kMxPiece, n);
            if (RES) r[RES ? i : 0] = load_piece<T, VEC>(res + row * H + p * kMxPiece, n);
        } else {
            v[i].clear();
            if (RES) r[RES ? i : 0].clear();
        }
    }
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
#pragma unroll
        for (int j = 0; j < kMxPiece; ++j) {
            // the sum is rounded to the storage type first: that value is the new residual and the row normalised
            if (RES) v[i].put(j, v[i].up(j) + r[RES ? i : 0].up(j));
            const float f = v[i].up(j);
            ss += f * f;
        }
    }
    ss = mx_team_sum<TPR>(ss, red);
    const float rstd = rsqrtf(ss / (float)H + eps);
    if (t == 0) rstd_out[row] = rstd;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int p = t + i * TPR, n = mx_piece_size(H, p);
        float f[kMxPiece];
#pragma unroll
        for (int j = 0; j < kMxPiece; ++j) f[j] = v[i].up(j);
        uint32_t scale;
        const MxCodes c = mx_encode(f, scale);
        if (n > 0) {
            Piece<T> o;
            if (w != nullptr) {
                const Piece<T> wv = load_piece<T, VEC, false>(w + p * kMxPiece, n);
#pragma unroll
                for (int j = 0; j < kMxPiece; ++j) o.put(j, f[j] * rstd * wv.up(j));
            } else {
#pragma unroll
                for (int j = 0; j < kMxPiece; ++j) o.put(j, f[j] * rstd);
            }
            store_piece<T, VEC>(o, y + row * H + p * kMxPiece, n);
            if (RES) store_piece<T, VEC>(v[i], res_out + row * H + p * kMxPiece, n);
            store_codes<VEC>(c, codes + row * H + p * kMxPiece, n);
            if (t % kMxQuad == 0) scales[row * blocks + p / kMxQuad] = (uint8_t)scale;
        }
    }
}

// Teams walk rows.  dy and the weight are kept in registers with the codes, except by the 1024-lane team, whose lanes have
// 128 registers: it reads dy and the weight twice, the second time from the cache.
template <typename T, int TPR, int NP, bool HAS_W, bool VEC>
__global__ void __launch_bounds__(TPR > 256 ? TPR : 256)
    rmsnorm_bwd_mx8_kernel(const int8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                           const typename T::storage_t* __restrict__ w, const typename T::storage_t* __restrict__ dy,
                           const float* __restrict__ rstd_in, const typename T::storage_t* __restrict__ dsum,
                           typename T::storage_t* __restrict__ dx, float* __restrict__ dw_partial, int64_t B, int H) {
    constexpr bool LEAN = TPR == 1024;
    constexpr int KEEP = LEAN ? 1 : NP;
    __shared__ float red[16];
    const int teams_per_block = blockDim.x / TPR;
    const int t = threadIdx.x % TPR;
    const int64_t team = (int64_t)blockIdx.x * teams_per_block + threadIdx.x / TPR;
    const int64_t num_teams = (int64_t)gridDim.x * teams_per_block;
    const int blocks = (H + kMxBlock - 1) / kMxBlock;
    const float inv_h = 1.f / (float)H;

    Piece<T> wv[HAS_W ? KEEP : 1];
    float dw[HAS_W ? NP : 1][kMxPiece];
    if (HAS_W) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int p = t + i * TPR, n = mx_piece_size(H, p);
            if (!LEAN) {
                if (n > 0) wv[LEAN ? 0 : i] = load_piece<T, VEC, false>(w + p * kMxPiece, n);
                else wv[LEAN ? 0 : i].clear();
            }
#pragma unroll
            for (int j = 0; j < kMxPiece; ++j) dw[i][j] = 0.f;
        }
    }
    for (int64_t row = team; row < B; row += num_teams) {
        const typename T::storage_t* gr = dy + row * H;
        const float rstd = rstd_in[row];
        MxCodes c[NP];
        uint32_t scale[NP];
        Piece<T> g[KEEP];
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int p = t + i * TPR, n = mx_piece_size(H, p);
            c[i].w[0] = c[i].w[1] = 0;
            scale[i] = 7;
            if (!LEAN) g[LEAN ? 0 : i].clear();
            if (n > 0) {
                c[i] = load_codes<VEC>(codes + row * H + p * kMxPiece, n);
                scale[i] = scales[row * blocks + p / kMxQuad];
                if (!LEAN) g[LEAN ? 0 : i] = load_piece<T, VEC>(gr + p * kMxPiece, n);
            }
        }
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int p = t + i * TPR, n = mx_piece_size(H, p);
            if (n > 0) {
                float f[kMxPiece];
                mx_decode(c[i], mx_step(scale[i]), f);
                const Piece<T> gp = LEAN ? load_piece<T, VEC, false>(gr + p * kMxPiece, n) : g[LEAN ? 0 : i];
                Piece<T> wp;
                if (HAS_W) wp = LEAN ? load_piece<T, VEC, false>(w + p * kMxPiece, n) : wv[LEAN ? 0 : i];
#pragma unroll
                for (int j = 0; j < kMxPiece; ++j) {
                    if (!VEC && j >= n) continue;  // (a block that stands for NaNs must not reach past the row)
                    dot += gp.up(j) * (HAS_W ? wp.up(j) : 1.f) * f[j];
                }
            }
        }
        dot = mx_team_sum<TPR>(dot, red);
        const float k = rstd * rstd * rstd * inv_h * dot;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int p = t + i * TPR, n = mx_piece_size(H, p);
            if (n > 0) {
                float f[kMxPiece];
                mx_decode(c[i], mx_step(scale[i]), f);
                const Piece<T> gp = LEAN ? load_piece<T, VEC, false>(gr + p * kMxPiece, n) : g[LEAN ? 0 : i];
                Piece<T> wp, sp, o;
                if (HAS_W) wp = LEAN ? load_piece<T, VEC, false>(w + p * kMxPiece, n) : wv[LEAN ? 0 : i];
                if (dsum != nullptr) sp = load_piece<T, VEC>(dsum + row * H + p * kMxPiece, n);
#pragma unroll
                for (int j = 0; j < kMxPiece; ++j) {
                    const float d = gp.up(j);
                    if (HAS_W && (VEC || j < n)) dw[HAS_W ? i : 0][j] += d * (f[j] * rstd);
                    float out = rstd * (HAS_W ? d * wp.up(j) : d) - k * f[j];
                    if (dsum != nullptr) out += sp.up(j);
                    o.put(j, out);
                }
                store_piece<T, VEC>(o, dx + row * H + p * kMxPiece, n);
            }
        }
    }
    if (HAS_W) {
        // one partial row per workgroup; the four teams of a 256-lane workgroup are added up in LDS, in their order
        const int padded = blocks * kMxBlock;
        constexpr int kTeams = TPR == 64 ? 4 : 1;
        constexpr int kCols = TPR == 64 ? 64 * NP * kMxPiece : 4;
        __shared__ float comb[kTeams * kCols];
        float* out = kTeams > 1 ? comb + (threadIdx.x / TPR) * kCols : dw_partial + (int64_t)blockIdx.x * padded;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int p = t + i * TPR;
            if (p < blocks * kMxQuad) {
#pragma unroll
                for (int j = 0; j < kMxPiece; j += 4)
                    *reinterpret_cast<float4*>(out + p * kMxPiece + j) = make_float4(
                        dw[HAS_W ? i : 0][j], dw[HAS_W ? i : 0][j + 1], dw[HAS_W ? i : 0][j + 2], dw[HAS_W ? i : 0][j + 3]);
            }
        }
        if (kTeams > 1) {
            __syncthreads();
            float* row = dw_partial + (int64_t)blockIdx.x * padded;
            for (int col = threadIdx.x * 4; col < padded; col += blockDim.x * 4) {
                float4 a = *reinterpret_cast<const float4*>(comb + col);
#pragma unroll
                for (int m = 1; m < kTeams; ++m) {
                    const float4 b = *reinterpret_cast<const float4*>(comb + m * kCols + col);
                    a.x += b.x;
                    a.y += b.y;
                    a.z += b.z;
                    a.w += b.w;
                }
                *reinterpret_cast<float4*>(row + col) = a;
            }
        }
    }
}

// dw[col] = sum of the partial rows, in a fixed order: a workgroup owns 16 columns, 64 groups of rows by 4 column quads
template <typename T>
__global__ void __launch_bounds__(256)
    rmsnorm_dw_mx8_kernel(const float* __restrict__ partial, typename T::storage_t* __restrict__ dw, int parts, int H,
                          int padded) {
    __shared__ float4 waves[4][4];
    const int quad = threadIdx.x & 3;
    const int col = blockIdx.x * 16 + quad * 4;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    if (col < padded) {
        for (int r = threadIdx.x >> 2; r < parts; r += 64) {
            const float4 v = *reinterpret_cast<const float4*>(partial + (int64_t)r * padded + col);
            acc.x += v.x;
            acc.y += v.y;
            acc.z += v.z;
            acc.w += v.w;
        }
    }
#pragma unroll
    for (int off = 4; off < CK_WAVE; off <<= 1) {
        acc.x += __shfl_xor(acc.x, off, CK_WAVE);
        acc.y += __shfl_xor(acc.y, off, CK_WAVE);
        acc.z += __shfl_xor(acc.z, off, CK_WAVE);
        acc.w += __shfl_xor(acc.w, off, CK_WAVE);
    }
    if (lane_id() < 4) waves[threadIdx.x / CK_WAVE][quad] = acc;
    __syncthreads();
    if (threadIdx.x < 4) {
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            const float4 v = waves[m][quad];
            sum[0] += v.x;
            sum[1] += v.y;
            sum[2] += v.z;
            sum[3] += v.w;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (col + j < H) dw[col + j] = T::down(sum[j]);
    }
}

}  // namespace ck

// ---- host side ---------------------------------------------------------------------------------------------------------
namespace {

constexpr int64_t kMxMaxRow = 65536;

// lanes per row, and pieces per lane of the narrowest instantiation that holds it
int mx_tpr(int64_t H) {
    const int64_t pieces = ck::mx_blocks(H) * ck::kMxQuad;
    return pieces <= 64 * ck::kMxMaxPieces ? 64 : (pieces <= 256 * ck::kMxMaxPieces ? 256 : 1024);
}
int mx_pieces(int64_t H, int tpr) {
    const int64_t pieces = ck::mx_blocks(H) * ck::kMxQuad;
    for (int np : {1, 2, 4})
        if (pieces <= (int64_t)np * tpr) return np;
    return 8;
}

int mx_cu_count() {
    static int cached[64] = {0};
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
    if (cached[dev] == 0) {
        int n = 0;
        if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) n = 256;
        cached[dev] = n;
    }
    return cached[dev];
}

// workgroups of the backward: each writes one partial row of dw
int mx_bwd_blocks(int64_t B, int64_t H) {
    const int tpr = mx_tpr(H);
    const int64_t need = ck_ceil_div(B, tpr == 64 ? 4 : 1);
    const int64_t most = (int64_t)mx_cu_count() * (tpr == 64 && mx_pieces(H, tpr) <= 4 ? 2 : 1);
    return (int)(need < most ? need : most);
}

struct MxFwd {
    const void *x, *res, *w;
    void *y, *res_out, *codes, *scales;
    float* rstd;
    int64_t B;
    int H;
    float eps;
};
template <typename T, int TPR, int NP, bool RES, bool VEC>
void mx_launch_fwd(hipStream_t s, const MxFwd& a) {
    typedef typename T::storage_t S;
    constexpr int block = TPR > 256 ? TPR : 256;
    hipLaunchKernelGGL((ck::rmsnorm_fwd_mx8_kernel<T, TPR, NP, RES, VEC>), dim3((unsigned)ck_ceil_div(a.B, block / TPR)),
                       dim3(block), 0, s, (const S*)a.x, (const S*)a.res, (const S*)a.w, (S*)a.y, (S*)a.res_out,
                       (int8_t*)a.codes, (uint8_t*)a.scales, a.rstd, a.B, a.H, a.eps);
}
template <typename T, bool RES>
void mx_dispatch_fwd(hipStream_t s, const MxFwd& a, bool vec) {
    const int tpr = mx_tpr(a.H), np = mx_pieces(a.H, tpr);
    if (!vec) {
        if (tpr == 64) mx_launch_fwd<T, 64, 8, RES, false>(s, a);
        else if (tpr == 256) mx_launch_fwd<T, 256, 8, RES, false>(s, a);
        else mx_launch_fwd<T, 1024, 8, RES, false>(s, a);
    } else if (tpr == 64) {
        if (np == 1) mx_launch_fwd<T, 64, 1, RES, true>(s, a);
        else if (np == 2) mx_launch_fwd<T, 64, 2, RES, true>(s, a);
        else if (np == 4) mx_launch_fwd<T, 64, 4, RES, true>(s, a);
        else mx_launch_fwd<T, 64, 8, RES, true>(s, a);
    } else if (tpr == 256) {
        if (np <= 4) mx_launch_fwd<T, 256, 4, RES, true>(s, a);
        else mx_launch_fwd<T, 256, 8, RES, true>(s, a);
    } else {
        mx_launch_fwd<T, 1024, 8, RES, true>(s, a);
    }
}

struct MxBwd {
    const void *codes, *scales, *w, *dy, *dsum;
    const float* rstd;
    void *dx, *ws;
    int64_t B;
    int H;
};
template <typename T, int TPR, int NP, bool W, bool VEC>
void mx_launch_bwd(hipStream_t s, const MxBwd& a) {
    typedef typename T::storage_t S;
    constexpr int block = TPR > 256 ? TPR : 256;
    hipLaunchKernelGGL((ck::rmsnorm_bwd_mx8_kernel<T, TPR, NP, W, VEC>), dim3((unsigned)mx_bwd_blocks(a.B, a.H)), dim3(block),
                       0, s, (const int8_t*)a.codes, (const uint8_t*)a.scales, (const S*)a.w, (const S*)a.dy, a.rstd,
                       (const S*)a.dsum, (S*)a.dx, (float*)a.ws, a.B, a.H);
}
template <typename T, bool W>
void mx_dispatch_bwd(hipStream_t s, const MxBwd& a, bool vec) {
    const int tpr = mx_tpr(a.H), np = mx_pieces(a.H, tpr);
    if (!vec) {
        if (tpr == 64) mx_launch_bwd<T, 64, 8, W, false>(s, a);
        else if (tpr == 256) mx_launch_bwd<T, 256, 8, W, false>(s, a);
        else mx_launch_bwd<T, 1024, 8, W, false>(s, a);
    } else if (tpr == 64) {
        if (np == 1) mx_launch_bwd<T, 64, 1, W, true>(s, a);
        else if (np == 2) mx_launch_bwd<T, 64, 2, W, true>(s, a);
        else if (np == 4) mx_launch_bwd<T, 64, 4, W, true>(s, a);
        else mx_launch_bwd<T, 64, 8, W, true>(s, a);
    } else if (tpr == 256) {
        if (np <= 4) mx_launch_bwd<T, 256, 4, W, true>(s, a);
        else mx_launch_bwd<T, 256, 8, W, true>(s, a);
    } else {
        mx_launch_bwd<T, 1024, 8, W, true>(s, a);
    }
}

bool mx_rows_dtype(int dtype) { return dtype == CK_F32 || dtype == CK_F16 || dtype == CK_BF16; }
bool mx_aligned8(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 7u) == 0; }

}  // namespace

extern "C" int ck_rmsnorm_forward_mx8(const void* x, const void* residual, const void* weight, void* output,
                                      void* residual_out, void* codes, void* scales, float* rstd, int64_t B, int64_t H,
                                      float eps, int dtype, void* stream) {
    if (B < 0 || H < 0 || H > kMxMaxRow) return CK_ERR_SHAPE;
    if (!mx_rows_dtype(dtype)) return CK_ERR_DTYPE;
    if (B == 0 || H == 0) return CK_OK;
    if (B > 0x7fffffff) return CK_ERR_SHAPE;
    if (!x || !output || !codes || !scales || !rstd || (residual && !residual_out)) return CK_ERR_NULL;
    const void* ptrs[5] = {x, residual, weight, output, residual_out};
    bool vec = H % ck::kMxPiece == 0 && mx_aligned8(codes);
    for (const void* p : ptrs) {
        if (!ck_aligned_elem(p, dtype)) return CK_ERR_ALIGN;
        vec = vec && ck_aligned16(p);
    }
    if (reinterpret_cast<uintptr_t>(rstd) & 3u) return CK_ERR_ALIGN;
    const MxFwd a = {x, residual, weight, output, residual_out, codes, scales, rstd, B, (int)H, eps};
    hipStream_t s = (hipStream_t)stream;
    CK_DISPATCH_DTYPE(dtype, {
        if (residual) mx_dispatch_fwd<T, true>(s, a, vec);
        else mx_dispatch_fwd<T, false>(s, a, vec);
    });
    return ck_launch_status();
}

extern "C" int64_t ck_rmsnorm_backward_mx8_workspace_size(int64_t B, int64_t H) {
    if (B <= 0 || H <= 0 || H > kMxMaxRow) return 0;
    return (int64_t)mx_bwd_blocks(B, H) * ck::mx_blocks(H) * ck::kMxBlock * 4;
}

extern "C" int ck_rmsnorm_backward_mx8(const void* codes, const void* scales, const void* weight, const void* output_grad,
                                       const float* rstd, const void* sum_grad, void* x_grad, void* weight_grad,
                                       void* workspace, int64_t workspace_bytes, int64_t B, int64_t H, int dtype,
                                       void* stream) {
    if (B < 0 || H < 0 || H > kMxMaxRow) return CK_ERR_SHAPE;
    if (!mx_rows_dtype(dtype)) return CK_ERR_DTYPE;
    hipStream_t s = (hipStream_t)stream;
    if (H == 0) return CK_OK;
    if (weight && !weight_grad) return CK_ERR_NULL;
    if (weight && (!ck_aligned_elem(weight, dtype) || !ck_aligned_elem(weight_grad, dtype))) return CK_ERR_ALIGN;
    const int padded = (int)(ck::mx_blocks(H) * ck::kMxBlock);
    int parts = 0;
    if (B > 0) {
        if (!codes || !scales || !output_grad || !rstd || !x_grad) return CK_ERR_NULL;
        const void* ptrs[4] = {weight, output_grad, sum_grad, x_grad};
        bool vec = H % ck::kMxPiece == 0 && mx_aligned8(codes);
        for (const void* p : ptrs) {
            if (!ck_aligned_elem(p, dtype)) return CK_ERR_ALIGN;
            vec = vec && ck_aligned16(p);
        }
        if (reinterpret_cast<uintptr_t>(rstd) & 3u) return CK_ERR_ALIGN;
        if (weight && (!workspace || !ck_aligned16(workspace) ||
                       workspace_bytes < ck_rmsnorm_backward_mx8_workspace_size(B, H)))
            return CK_ERR_WORKSPACE;
        parts = mx_bwd_blocks(B, H);
        const MxBwd a = {codes, scales, weight, output_grad, sum_grad, rstd, x_grad, workspace, B, (int)H};
        CK_DISPATCH_DTYPE(dtype, {
            if (weight) mx_dispatch_bwd<T, true>(s, a, vec);
            else mx_dispatch_bwd<T, false>(s, a, vec);
        });
    }
    if (weight) {
        // (an empty batch still defines dweight = 0: no partial rows)
        CK_DISPATCH_DTYPE(dtype, {
            typedef typename T::storage_t S;
            hipLaunchKernelGGL((ck::rmsnorm_dw_mx8_kernel<T>), dim3((unsigned)ck_ceil_div(H, 16)), dim3(256), 0, s,
                               (const float*)workspace, (S*)weight_grad, parts, (int)H, padded);
        });
    }
    return ck_launch_status();
}
