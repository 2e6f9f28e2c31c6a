// RMSNorm that keeps its input in 8 bits (ck_mx8.h) for the backward, for gfx950.
//   forward : s = x (+ residual, rounded);  r = 1 / sqrt(mean s^2 + eps);  y = s r w;  writes y, r, the 8-bit form of s
//             (and s itself with a residual)
//   backward: with s^ the kept row:  dx = r (dy w - s^ r^2 mean(dy w s^)) (+ the sum's own gradient),  dw = sum dy s^ r
// The row (forward: as read; backward: codes and dy) stays in the registers of a team of TPR lanes, so it is read once;
// row sums are register exchanges, wider teams meet through LDS.  Lane t holds the 16-byte pieces t, t + TPR, ..: neighbouring
// lanes hold a block.  Backward: every team walks rows and keeps its share of dw in
// fp32 registers; a workgroup writes one partial row, a second launch adds the partial rows up.  No atomics.
#include "ck_mx8.h"

namespace ck {

template <int V>
struct Int {
    static constexpr int value = V;
};

// The backward's launch: workgroups a compute unit holds, and rows a team has in flight, by element size and team width.
// Measured at 16384 x 4096 bf16 (and 8192 x 4096 fp32): three workgroups with one row in flight 69.1 us, two rows 69.4, three
// rows 69.0 but 120 registers; four workgroups 71-79 (more partial rows of dw to write and add); fp32 with two
// workgroups and two rows 57.8, three and one 58.7.
constexpr int mx_bwd_residency(int bytes, int tpr) {
    const int most = bytes == 4 ? 2 : 3;
    return tpr == 1024 ? 1 : (tpr == 512 ? (most + 1) / 2 : most);
}
constexpr int mx_bwd_depth(int bytes, int tpr) { return bytes == 4 && tpr < 1024 ? 2 : 1; }

// Sum over the wave, in all lanes: register exchanges up to sixteen lanes (quad_perm 1 0 3 2 and 2 3 0 1, then the mirror
// images of eight and sixteen, the quads and eights being uniform by then), scalar reads of the four sixteens.  A chain of
// shuffles is six trips through the LDS unit, which every row waits for (backward of 16384 x 4096 bf16 69.7 -> 68.6 us).
__device__ __forceinline__ float mx_wave_sum(float v) {
    auto moved = [](float f, auto ctrl) __attribute__((always_inline)) {
        return mx_float((uint32_t)__builtin_amdgcn_mov_dpp((int)mx_bits(f), decltype(ctrl)::value, 0xF, 0xF, true));
    };
    v += moved(v, Int<0xB1>());
    v += moved(v, Int<0x4E>());
    v += moved(v, Int<0x141>());
    v += moved(v, Int<0x140>());
    auto lane = [&](int l) __attribute__((always_inline)) {
        return mx_float((uint32_t)__builtin_amdgcn_readlane((int)mx_bits(v), l));
    };
    return (lane(0) + lane(16)) + (lane(32) + lane(48));
}

// sum over the TPR lanes of a team, in all of them.  Teams wider than a wave meet at one barrier (every thread of the
// workgroup comes here); `red` holds a float per wave, and two uses in a row take different ones.
template <int TPR>
__device__ __forceinline__ float mx_team_sum(float v, float* red) {
    v = mx_wave_sum(v);
    if (TPR > CK_WAVE) {
        const int wave = threadIdx.x / CK_WAVE;
        if (lane_id() == 0) red[wave] = v;
        __syncthreads();
        const int first = wave / (TPR / CK_WAVE) * (TPR / CK_WAVE);
        v = 0.f;
#pragma unroll
        for (int w = 0; w < TPR / CK_WAVE; ++w) v += red[first + w];
    }
    return v;
}

// Makes the compiler forget what it knows about a packed register set: values widened from it before this point are not
// kept alive in place of the packed form.
template <typename P>
__device__ __forceinline__ void forget(P& p) {
    uint32_t* w = reinterpret_cast<uint32_t*>(&p);
#pragma unroll
    for (int i = 0; i < (int)(sizeof(P) / 4); ++i) asm volatile("" : "+v"(w[i]));
}

// elements of piece p that exist
template <int N>
__device__ __forceinline__ int mx_piece_size(int H, int p) {
    const int left = H - p * N;
    return left >= N ? N : (left > 0 ? left : 0);
}

// one row per team; UNITS units of eight elements a lane at most
template <typename T, int TPR, int UNITS, bool RES, bool VEC>
__global__ void __launch_bounds__(TPR > 256 ? TPR : 256)
    rmsnorm_fwd_mx8_kernel(const typename T::storage_t* __restrict__ x, const typename T::storage_t* __restrict__ res,
                           const typename T::storage_t* __restrict__ w, typename T::storage_t* __restrict__ y,
                           typename T::storage_t* __restrict__ res_out, int8_t* __restrict__ codes,
                           uint8_t* __restrict__ scales, float* __restrict__ rstd_out, int64_t B, int H, float eps) {
    constexpr int N = kMxPiece<T>, NP = UNITS * 8 / N;
    __shared__ float red[16];
    const int t = threadIdx.x % TPR;
    const int64_t row = (int64_t)blockIdx.x * (blockDim.x / TPR) + threadIdx.x / TPR;
    const bool live = row < B;
    const int blocks = (H + kMxBlock - 1) / kMxBlock;
    const typename T::storage_t* xr = x + row * H;
    Piece<T, N> v[NP], r[RES ? NP : 1];
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int p = t + i * TPR, n = mx_piece_size<N>(H, p);
        if (live && n > 0) {
            v[i] = load_piece<T, N, VEC>(xr + p * N, n);
            if (RES) r[RES ? i : 0] = load_piece<T, N, VEC>(res + row * H + p * N, n);
        } else {
            v[i].clear();
            if (RES) r[RES ? i : 0].clear();
        }
    }
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            // the sum is rounded to the storage type first: that value is the new residual and the row normalised
            if (RES) v[i].put(j, v[i].up(j) + r[RES ? i : 0].up(j));
            const float f = v[i].up(j);
            ss += f * f;
        }
    }
    ss = mx_team_sum<TPR>(ss, red);
    const float rstd = rsqrtf(ss / (float)H + eps);
    if (live && t == 0) rstd_out[row] = rstd;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int p = t + i * TPR, n = mx_piece_size<N>(H, p);
        float f[N];
#pragma unroll
        for (int j = 0; j < N; ++j) f[j] = v[i].up(j);
        uint32_t scale;
        const MxCodes<N> c = mx_encode(f, scale);
        if (live && n > 0) {
            Piece<T, N> o;
            if (w != nullptr) {
                const Piece<T, N> wv = load_piece<T, N, VEC, false>(w + p * N, n);
#pragma unroll
                for (int j = 0; j < N; ++j) o.put(j, f[j] * rstd * wv.up(j));
            } else {
#pragma unroll
                for (int j = 0; j < N; ++j) o.put(j, f[j] * rstd);
            }
            store_piece<T, N, VEC>(o, y + row * H + p * N, n);
            if (RES) store_piece<T, N, VEC>(v[i], res_out + row * H + p * N, n);
            store_codes<N, VEC>(c, codes + row * H + p * N, n);
            if (t % kMxLanes<T> == 0) scales[row * blocks + p / kMxLanes<T>] = (uint8_t)scale;
        }
    }
}

// Rows are dealt round-robin to the teams.
// With q the codes and e the step of a block:  dx = r (dy w) - (r^2 mean(dy w s^) (r e)) q,  dw += (dy e r) q  - the steps are
// folded into factors of a piece, so the kept row costs one conversion an element and no multiplication of its own.
template <typename T, int TPR, int UNITS, bool HAS_W, bool DSUM, bool VEC>
__global__ void __launch_bounds__(TPR > 256 ? TPR : 256, mx_bwd_residency(sizeof(typename T::storage_t), TPR))
    rmsnorm_bwd_mx8_kernel(const int8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                           const typename T::storage_t* __restrict__ w, const typename T::storage_t* __restrict__ dy,
                           const float* __restrict__ rstd_in, const typename T::storage_t* __restrict__ dsum,
                           typename T::storage_t* __restrict__ dx, float* __restrict__ dw_partial, int64_t B, int H) {
    constexpr int N = kMxPiece<T>, NP = UNITS * 8 / N;
    constexpr int THREADS = TPR > 256 ? TPR : 256, TEAMS = THREADS / TPR;
    // A lane of the 1024-lane team has 128 registers.  Where its sums of dw and a row leave no room beside each other, nothing
    // of the row is kept: it is read twice, the second time from the cache.
    constexpr bool LEAN = TPR == 1024 && UNITS * sizeof(typename T::storage_t) > 8;
    constexpr int KEEP = LEAN ? 1 : NP;
    __shared__ float red[2][THREADS / CK_WAVE];
    const int t = threadIdx.x % TPR, team = threadIdx.x / TPR;
    const int blocks = (H + kMxBlock - 1) / kMxBlock;
    const float inv_h = 1.f / (float)H;

    struct Row {
        MxCodes<N> c[KEEP];
        uint32_t scale[KEEP];
        Piece<T, N> g[KEEP], s[DSUM ? KEEP : 1];
        float rstd;
    };
    // piece i of a row into place k of a Row
    auto fetch_piece = [&](int64_t row, int i, int k, Row& r) __attribute__((always_inline)) {
        const int p = t + i * TPR, n = mx_piece_size<N>(H, p);
        r.c[k] = MxCodes<N>{};
        r.scale[k] = 7;
        r.g[k].clear();
        if (row < B && n > 0) {
            r.c[k] = load_codes<N, VEC>(codes + row * H + p * N, n);
            r.scale[k] = scales[row * blocks + p / kMxLanes<T>];
            r.g[k] = load_piece<T, N, VEC, !LEAN>(dy + row * H + p * N, n);
            if (DSUM) r.s[DSUM ? k : 0] = load_piece<T, N, VEC, !LEAN>(dsum + row * H + p * N, n);
        }
    };
    auto fetch = [&](int64_t row, Row& r) __attribute__((always_inline)) {
        r.rstd = row < B ? rstd_in[row] : 0.f;
        if (!LEAN) {
#pragma unroll
            for (int i = 0; i < NP; ++i) fetch_piece(row, i, LEAN ? 0 : i, r);
        }
    };

    Piece<T, N> wv[HAS_W ? KEEP : 1];
    float dw[HAS_W ? NP : 1][N];
    if (HAS_W) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int p = t + i * TPR, n = mx_piece_size<N>(H, p);
            if (!LEAN) {
                wv[LEAN ? 0 : i].clear();
                if (n > 0) wv[LEAN ? 0 : i] = load_piece<T, N, VEC, false>(w + p * N, n);
            }
#pragma unroll
            for (int j = 0; j < N; ++j) dw[i][j] = 0.f;
        }
    }
    auto work = [&](int64_t row, Row& cur, int turn) __attribute__((always_inline)) {
        const bool live = row < B;
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int p = t + i * TPR, n = mx_piece_size<N>(H, p), at = LEAN ? 0 : i;
            if (live && n > 0) {
                if (LEAN) fetch_piece(row, i, 0, cur);
                Piece<T, N> wp;
                if (HAS_W) wp = LEAN ? load_piece<T, N, VEC, false>(w + p * N, n) : wv[HAS_W ? at : 0];
                float part = 0.f;
#pragma unroll
                for (int j = 0; j < N; ++j)
                    part += (HAS_W ? cur.g[at].up(j) * wp.up(j) : cur.g[at].up(j)) * mx_code(cur.c[at], j);
                dot += part * mx_step_kept(cur.scale[at]);
            }
            __builtin_amdgcn_sched_barrier(0);  // one piece at a time: widened values do not pile up in registers
        }
        if (!LEAN) {
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                const int at = LEAN ? 0 : i;
                forget(cur.g[at]);
                forget(cur.c[at]);
                if (HAS_W) forget(wv[HAS_W ? at : 0]);
            }
        }
        dot = mx_team_sum<TPR>(dot, red[turn]);
        // (the factors in this order: r^3 by itself leaves fp32's range at rows of 2^43 and of 2^-43)
        const float rstd = cur.rstd, k = rstd * (rstd * dot) * inv_h;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int p = t + i * TPR, n = mx_piece_size<N>(H, p), at = LEAN ? 0 : i;
            if (live && n > 0) {
                if (LEAN) fetch_piece(row, i, 0, cur);
                Piece<T, N> wp, o;
                if (HAS_W) wp = LEAN ? load_piece<T, N, VEC, false>(w + p * N, n) : wv[HAS_W ? at : 0];
                const float e = mx_step_kept(cur.scale[at]), er = e * rstd, ke = k * er;
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const float d = cur.g[at].up(j), q = mx_code(cur.c[at], j);
                    if (HAS_W) dw[HAS_W ? i : 0][j] += d * er * q;
                    float out = rstd * (HAS_W ? d * wp.up(j) : d) - ke * q;
                    if (DSUM) out += cur.s[DSUM ? at : 0].up(j);
                    o.put(j, out);
                }
                store_piece<T, N, VEC>(o, dx + row * H + p * N, n);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    const int64_t step = (int64_t)gridDim.x * TEAMS;
    int64_t first = (int64_t)blockIdx.x * TEAMS, row = first + team;
    // rows in flight while one is worked on; a row's place is filled again as soon as it is done with
    constexpr int DEPTH = LEAN ? 1 : mx_bwd_depth(sizeof(typename T::storage_t), TPR);
    Row buf[DEPTH];
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) fetch(row + d * step, buf[d]);
    int turn = 0;
    while (first < B) {
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            if (first < B) {
                work(row, buf[d], turn);
                turn ^= 1;
                fetch(row + DEPTH * step, buf[d]);
            }
            first += step;
            row += step;
        }
    }
    if (HAS_W) {
        // one partial row per workgroup; its teams are added up in LDS, in their order
        const int padded = blocks * kMxBlock;
        constexpr int kCols = TEAMS > 1 ? TPR * NP * N : 4;
        __shared__ float comb[TEAMS * kCols];
        float* out = TEAMS > 1 ? comb + team * kCols : dw_partial + (int64_t)blockIdx.x * padded;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int p = t + i * TPR;
            if (p < blocks * kMxLanes<T>) {
#pragma unroll
                for (int j = 0; j < N; j += 4)
                    *reinterpret_cast<float4*>(out + p * N + j) = make_float4(
                        dw[HAS_W ? i : 0][j], dw[HAS_W ? i : 0][j + 1], dw[HAS_W ? i : 0][j + 2], dw[HAS_W ? i : 0][j + 3]);
            }
        }
        if (TEAMS > 1) {
            __syncthreads();
            float* sum = dw_partial + (int64_t)blockIdx.x * padded;
            for (int col = threadIdx.x * 4; col < padded; col += THREADS * 4) {
                float4 a = *reinterpret_cast<const float4*>(comb + col);
#pragma unroll
                for (int m = 1; m < TEAMS; ++m) {
                    const float4 b = *reinterpret_cast<const float4*>(comb + m * kCols + col);
                    a.x += b.x;
                    a.y += b.y;
                    a.z += b.z;
                    a.w += b.w;
                }
                *reinterpret_cast<float4*>(sum + col) = a;
            }
        }
    }
}

// dw[col] = sum of the partial rows, in a fixed order: a workgroup owns 32 columns (a cache line of each partial row), 8 column
// quads by 128 groups of rows.  768 partial rows of 4096: 4.6 us, and 5.6 with 16 columns, where every line is fetched twice.
template <typename T>
__global__ void __launch_bounds__(1024)
    rmsnorm_dw_mx8_kernel(const float* __restrict__ partial, typename T::storage_t* __restrict__ dw, int parts, int H,
                          int padded) {
    __shared__ float4 waves[16][8];
    const int quad = threadIdx.x & 7;
    const int col = blockIdx.x * 32 + quad * 4;  // (rows are padded to a multiple of 32)
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int r = threadIdx.x >> 3; r < parts; r += 128) {
        const float4 v = *reinterpret_cast<const float4*>(partial + (int64_t)r * padded + col);
        acc.x += v.x;
        acc.y += v.y;
        acc.z += v.z;
        acc.w += v.w;
    }
#pragma unroll
    for (int off = 8; off < CK_WAVE; off <<= 1) {
        acc.x += __shfl_xor(acc.x, off, CK_WAVE);
        acc.y += __shfl_xor(acc.y, off, CK_WAVE);
        acc.z += __shfl_xor(acc.z, off, CK_WAVE);
        acc.w += __shfl_xor(acc.w, off, CK_WAVE);
    }
    if (lane_id() < 8) waves[threadIdx.x / CK_WAVE][quad] = acc;
    __syncthreads();
    if (threadIdx.x < 8) {
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int m = 0; m < 16; ++m) {
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

// units of eight elements in a row
int64_t mx_row_units(int64_t H) { return ck::mx_blocks(H) * 4; }

// Lanes per row, both ways: two units a lane (more only beyond 16384 elements).  Few registers keep many waves resident:
// forward 59.5 us at 16384 x 4096 bf16, against 59.8 with four units a lane and 66.1 with a wave per row.
int mx_tpr(int64_t H) {
    const int64_t units = mx_row_units(H);
    for (int tpr : {64, 128, 256, 512})
        if (units <= (int64_t)tpr * 2) return tpr;
    return 1024;
}
// the team the backward's launch takes: those of 128 and 512 lanes only for aligned rows
int mx_bwd_tpr(int64_t H, bool vec) {
    const int tpr = mx_tpr(H);
    return vec ? tpr : (tpr == 128 ? 256 : (tpr == 512 ? 1024 : tpr));
}
// the fewest units a lane has to hold, of those compiled
int mx_units(int64_t H, int tpr) {
    const int64_t units = mx_row_units(H);
    for (int n : {1, 2, 4})
        if (units <= (int64_t)n * tpr) return n;
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
int mx_bwd_blocks(int64_t B, int64_t H, int dtype, bool vec) {
    const int tpr = mx_bwd_tpr(H, vec);
    const int64_t need = ck_ceil_div(B, tpr < 256 ? 256 / tpr : 1);
    const int64_t most = (int64_t)mx_cu_count() * ck::mx_bwd_residency(dtype == CK_F32 ? 4 : 2, tpr);
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
template <typename T, int TPR, int UNITS, bool RES, bool VEC>
void mx_launch_fwd(hipStream_t s, const MxFwd& a) {
    typedef typename T::storage_t S;
    constexpr int block = TPR > 256 ? TPR : 256;
    // a launch has fewer than 2^32 lanes: rows beyond take further ones (2^30 lanes' rows of any length are whole packets)
    constexpr int64_t most = ((int64_t)1 << 30) / TPR;
    const int64_t blocks = (a.H + ck::kMxBlock - 1) / ck::kMxBlock;
    for (int64_t row = 0; row < a.B; row += most) {
        const int64_t rows = a.B - row < most ? a.B - row : most, at = row * a.H;
        hipLaunchKernelGGL((ck::rmsnorm_fwd_mx8_kernel<T, TPR, UNITS, RES, VEC>), dim3((unsigned)ck_ceil_div(rows, block / TPR)),
                           dim3(block), 0, s, (const S*)a.x + at, RES ? (const S*)a.res + at : (const S*)nullptr, (const S*)a.w,
                           (S*)a.y + at, RES ? (S*)a.res_out + at : (S*)nullptr, (int8_t*)a.codes + at,
                           (uint8_t*)a.scales + row * blocks, a.rstd + row, rows, a.H, a.eps);
    }
}
// teams of 128 and 512 lanes only where alignment lets them be fast: rows read element by element take the next wider one
template <typename T, bool RES, bool VEC>
void mx_dispatch_fwd(hipStream_t s, const MxFwd& a) {
    const int tpr = mx_tpr(a.H), units = mx_units(a.H, tpr);
    if (VEC && tpr == 64 && units == 1) mx_launch_fwd<T, 64, VEC ? 1 : 2, RES, VEC>(s, a);
    else if (tpr == 64) mx_launch_fwd<T, 64, 2, RES, VEC>(s, a);
    else if (VEC && tpr == 128) mx_launch_fwd<T, VEC ? 128 : 256, 2, RES, VEC>(s, a);
    else if (tpr <= 256) mx_launch_fwd<T, 256, 2, RES, VEC>(s, a);
    else if (VEC && tpr == 512) mx_launch_fwd<T, VEC ? 512 : 1024, 2, RES, VEC>(s, a);
    else if (units <= 2) mx_launch_fwd<T, 1024, 2, RES, VEC>(s, a);
    else if (units == 4) mx_launch_fwd<T, 1024, 4, RES, VEC>(s, a);
    else mx_launch_fwd<T, 1024, 8, RES, VEC>(s, a);
}

struct MxBwd {
    const void *codes, *scales, *w, *dy, *dsum;
    const float* rstd;
    void *dx, *ws;
    int64_t B;
    int H, blocks;
};
template <typename T, int TPR, int UNITS, bool W, bool D, bool VEC>
void mx_launch_bwd(hipStream_t s, const MxBwd& a) {
    typedef typename T::storage_t S;
    hipLaunchKernelGGL((ck::rmsnorm_bwd_mx8_kernel<T, TPR, UNITS, W, D, VEC>), dim3((unsigned)a.blocks), dim3(TPR > 256 ? TPR : 256),
                       0, s, (const int8_t*)a.codes, (const uint8_t*)a.scales, (const S*)a.w, (const S*)a.dy, a.rstd,
                       (const S*)a.dsum, (S*)a.dx, (float*)a.ws, a.B, a.H);
}
template <typename T, bool W, bool D, bool VEC>
void mx_dispatch_bwd_as(hipStream_t s, const MxBwd& a) {
    const int tpr = mx_bwd_tpr(a.H, VEC), units = mx_units(a.H, tpr);
    if (VEC && tpr == 64 && units == 1) mx_launch_bwd<T, 64, VEC ? 1 : 2, W, D, VEC>(s, a);
    else if (tpr == 64) mx_launch_bwd<T, 64, 2, W, D, VEC>(s, a);
    else if (VEC && tpr == 128) mx_launch_bwd<T, VEC ? 128 : 256, 2, W, D, VEC>(s, a);
    else if (tpr == 256) mx_launch_bwd<T, 256, 2, W, D, VEC>(s, a);
    else if (VEC && tpr == 512) mx_launch_bwd<T, VEC ? 512 : 1024, 2, W, D, VEC>(s, a);
    else if (units <= 2) mx_launch_bwd<T, 1024, 2, W, D, VEC>(s, a);
    else if (units == 4) mx_launch_bwd<T, 1024, 4, W, D, VEC>(s, a);
    else mx_launch_bwd<T, 1024, 8, W, D, VEC>(s, a);
}
template <typename T, bool W, bool VEC>
void mx_dispatch_bwd(hipStream_t s, const MxBwd& a) {
    if (a.dsum) mx_dispatch_bwd_as<T, W, true, VEC>(s, a);
    else mx_dispatch_bwd_as<T, W, false, VEC>(s, a);
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
    bool vec = H % (dtype == CK_F32 ? 4 : 8) == 0 && mx_aligned8(codes);
    for (const void* p : ptrs) {
        if (!ck_aligned_elem(p, dtype)) return CK_ERR_ALIGN;
        vec = vec && ck_aligned16(p);
    }
    if (reinterpret_cast<uintptr_t>(rstd) & 3u) return CK_ERR_ALIGN;
    const MxFwd a = {x, residual, weight, output, residual_out, codes, scales, rstd, B, (int)H, eps};
    hipStream_t s = (hipStream_t)stream;
    CK_DISPATCH_DTYPE(dtype, {
        if (residual && vec) mx_dispatch_fwd<T, true, true>(s, a);
        else if (residual) mx_dispatch_fwd<T, true, false>(s, a);
        else if (vec) mx_dispatch_fwd<T, false, true>(s, a);
        else mx_dispatch_fwd<T, false, false>(s, a);
    });
    return ck_launch_status();
}

extern "C" int64_t ck_rmsnorm_backward_mx8_workspace_size(int64_t B, int64_t H, int dtype) {
    if (B <= 0 || H <= 0 || H > kMxMaxRow) return 0;
    // (whichever way the operands turn out to be aligned)
    const int a = mx_bwd_blocks(B, H, dtype, true), b = mx_bwd_blocks(B, H, dtype, false);
    return (int64_t)(a > b ? a : b) * ck::mx_blocks(H) * ck::kMxBlock * 4;
}

extern "C" int ck_rmsnorm_backward_mx8(const void* codes, const void* scales, const void* weight, const void* output_grad,
                                       const float* rstd, const void* sum_grad, void* x_grad, void* weight_grad,
                                       void* workspace, int64_t workspace_bytes, int64_t B, int64_t H, int dtype,
                                       void* stream) {
    if (B < 0 || H < 0 || H > kMxMaxRow) return CK_ERR_SHAPE;
    if (!mx_rows_dtype(dtype)) return CK_ERR_DTYPE;
    hipStream_t s = (hipStream_t)stream;
    if (H == 0 || (B == 0 && !weight)) return CK_OK;
    if (weight && !weight_grad) return CK_ERR_NULL;
    if (weight && (!ck_aligned_elem(weight, dtype) || !ck_aligned_elem(weight_grad, dtype))) return CK_ERR_ALIGN;
    const int padded = (int)(ck::mx_blocks(H) * ck::kMxBlock);
    int parts = 0;
    if (B > 0) {
        if (!codes || !scales || !output_grad || !rstd || !x_grad) return CK_ERR_NULL;
        const void* ptrs[4] = {weight, output_grad, sum_grad, x_grad};
        bool vec = H % (dtype == CK_F32 ? 4 : 8) == 0 && mx_aligned8(codes);
        for (const void* p : ptrs) {
            if (!ck_aligned_elem(p, dtype)) return CK_ERR_ALIGN;
            vec = vec && ck_aligned16(p);
        }
        if (reinterpret_cast<uintptr_t>(rstd) & 3u) return CK_ERR_ALIGN;
        if (weight && (!workspace || !ck_aligned16(workspace) ||
                       workspace_bytes < ck_rmsnorm_backward_mx8_workspace_size(B, H, dtype)))
            return CK_ERR_WORKSPACE;
        parts = mx_bwd_blocks(B, H, dtype, vec);
        const MxBwd a = {codes, scales, weight, output_grad, sum_grad, rstd, x_grad, workspace, B, (int)H, parts};
        CK_DISPATCH_DTYPE(dtype, {
            if (weight && vec) mx_dispatch_bwd<T, true, true>(s, a);
            else if (weight) mx_dispatch_bwd<T, true, false>(s, a);
            else if (vec) mx_dispatch_bwd<T, false, true>(s, a);
            else mx_dispatch_bwd<T, false, false>(s, a);
        });
    }
    if (weight) {
        // (an empty batch still defines dweight = 0: no partial rows)
        CK_DISPATCH_DTYPE(dtype, {
            typedef typename T::storage_t S;
            hipLaunchKernelGGL((ck::rmsnorm_dw_mx8_kernel<T>), dim3((unsigned)ck_ceil_div(H, 32)), dim3(1024), 0, s,
                               (const float*)workspace, (S*)weight_grad, parts, (int)H, padded);
        });
    }
    return ck_launch_status();
}
