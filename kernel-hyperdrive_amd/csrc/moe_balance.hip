// Balance loss, z-loss and per-expert counts of an MoE router, forward and backward, for gfx950.
//   p_te = softmax over the experts of token t's logits,  lse_t = their log-sum-exp,  m_t = 1 for a token that counts
//   c_e  = how often a counting token selected expert e,  N = sum m,  f_e = c_e / (N k),  P_e = sum_t m_t p_te / N
//   balance = E sum_e f_e P_e          z = sum_t m_t lse_t^2 / N
//   d logits_te = m_t p_te [ g_b E / N (f_e - sum_j f_j p_tj) + g_z 2 / N lse_t ]
// Bound by latency up to some thousand tokens and by HBM beyond: one pass over the logits each way, ten flops an element.
// A token's row is held by LPT lanes (a power of two), eight neighbouring experts each, so row maxima and sums are
// LPT-lane shuffles and a lane's eight probability sums stay in registers over all tokens its wave walks.  Workgroups
// write partial sums; a second launch of one workgroup adds them up in a fixed order (no floating-point atomics; the
// counts are whole numbers).  Few tokens take one workgroup that finishes by itself.
// f_e - sum f p cancels when the load is balanced.  The probabilities sum to one, so any constant may be taken off f
// first: f_e - mean f = (E c_e - sum c) / (N k E) comes from whole numbers and loses nothing.  The forward leaves E / N times
// that for every expert, and 1 / N behind them, for the backward (`shares`).
#include "ck_piece.h"

namespace ck {

constexpr int kBalanceMaxExperts = 1024;
constexpr int kPiece = 8;  // experts a lane holds side by side

// Combines a value over the LPT neighbouring lanes that hold a token's row, in all of them.  Up to sixteen lanes by register
// exchanges (quad_perm 1 0 3 2, quad_perm 2 3 0 1; behind those the quads are uniform, so the mirror images of eight and of
// sixteen lanes bring the other half's value), beyond by shuffles.
template <int CTRL>
__device__ __forceinline__ float lanes_moved(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true));
}
template <int LPT, typename F>
__device__ __forceinline__ float group_reduce(float v, F&& op) {
    if (LPT >= 2) v = op(v, lanes_moved<0xB1>(v));
    if (LPT >= 4) v = op(v, lanes_moved<0x4E>(v));
    if (LPT >= 8) v = op(v, lanes_moved<0x141>(v));
    if (LPT >= 16) v = op(v, lanes_moved<0x140>(v));
    if (LPT >= 32) v = op(v, __shfl_xor(v, 16, CK_WAVE));
    if (LPT >= 64) v = op(v, __shfl_xor(v, 32, CK_WAVE));
    return v;
}
template <int LPT>
__device__ __forceinline__ float group_max(float v) {
    return group_reduce<LPT>(v, [](float a, float b) { return fmaxf(a, b); });
}
template <int LPT>
__device__ __forceinline__ float group_sum(float v) {
    return group_reduce<LPT>(v, [](float a, float b) { return a + b; });
}

// exp(x) for x <= 0, -inf or NaN: 2^(x log2 e), the product's rounding error kept and applied to first order, so that the
// result is as good at -80 as at -1.  (Below -200, where 2^.. is 0, x counts as -200: -inf has no rounding error.)
__device__ __forceinline__ float exp_nonpositive(float x) {
    x = x < -200.f ? -200.f : x;
    const float log2e = 1.44269504f, log2e_rest = 1.92596299e-8f;  // log2 e = their sum to 48 bits
    const float hi = x * log2e;
    const float lo = fmaf(x, log2e, -hi) + x * log2e_rest;
    const float e = __builtin_amdgcn_exp2f(hi);
    return fmaf(e, lo * 0.693147181f, e);
}
__device__ __forceinline__ double wave_sum_d(double v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, CK_WAVE);
    return v;
}

// experts a piece that starts at column `col` holds
__device__ __forceinline__ int piece_size(int E, int col) {
    const int left = E - col;
    return left >= kPiece ? kPiece : (left > 0 ? left : 0);
}

// lowest finite value of a storage type: what a mask writes where -inf is not wanted
template <typename T>
__device__ __forceinline__ float lowest_of();
template <>
__device__ __forceinline__ float lowest_of<F32>() { return -__FLT_MAX__; }
template <>
__device__ __forceinline__ float lowest_of<F16>() { return -65504.f; }
template <>
__device__ __forceinline__ float lowest_of<BF16>() { return -3.3895313892515355e38f; }

// Probabilities of one token from its logits, in place (columns beyond a piece's size become 0), and its log-sum-exp.  A row whose mask
// left nothing - -inf or the type's lowest value throughout - has no probabilities and counts as lse 0 (every exponential
// below is then 0); a NaN, or +inf, makes the row NaN.
template <typename T, int LPT, int CHUNKS, bool VEC>
__device__ __forceinline__ float token_softmax(float (&v)[CHUNKS][kPiece], const int (&size)[CHUNKS]) {
    const float none = -__builtin_inff();
    float top = none;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
        for (int j = 0; j < kPiece; ++j) {
            // (aligned rows have whole pieces or none)
            if (VEC ? size[c] == 0 : j >= size[c]) v[c][j] = none;
            top = fmaxf(top, v[c][j]);
        }
    top = group_max<LPT>(top);
    if (top <= lowest_of<T>()) top = 0.f;
    float sum = 0.f;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
        for (int j = 0; j < kPiece; ++j) {
            v[c][j] = exp_nonpositive(v[c][j] - top);
            sum += v[c][j];
        }
    sum = group_sum<LPT>(sum);
    const bool empty = sum == 0.f;
    const float inverse = empty ? 0.f : 1.f / sum;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
        for (int j = 0; j < kPiece; ++j) v[c][j] *= inverse;
    return empty ? 0.f : top + logf(sum);
}

// losses from the summed columns; all threads of the workgroup call it.  Thread e (< E) brings expert e's sums.
struct BalanceOut {
    float *balance, *z, *shares;
    int* counts;
};
template <int WAVES>
__device__ __forceinline__ void balance_finish(double prob, int count, double z, int tokens, int E, int k, BalanceOut out) {
    __shared__ double sums[WAVES][2];
    __shared__ int totals[WAVES][2];
    const int e = threadIdx.x, wave = e / CK_WAVE;
    const bool mine = e < E;
    const double cross = wave_sum_d(mine ? prob * (double)count : 0.0);
    z = wave_sum_d(z);
    const int selections = wave_sum_i(mine ? count : 0);
    tokens = wave_sum_i(tokens);
    if (lane_id() == 0) {
        sums[wave][0] = cross;
        sums[wave][1] = z;
        totals[wave][0] = tokens;
        totals[wave][1] = selections;
    }
    __syncthreads();
    double c = 0.0, zz = 0.0;
    int n = 0, total = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        c += sums[w][0];
        zz += sums[w][1];
        n += totals[w][0];
        total += totals[w][1];
    }
    const double per_token = n > 0 ? 1.0 / (double)n : 0.0, scale = per_token * per_token / (double)k;
    if (mine) {
        out.counts[e] = count;
        out.shares[e] = (float)(scale * (double)((long long)E * count - total));
    }
    if (threadIdx.x == 0) {
        *out.balance = (float)((double)E * c * scale);
        *out.z = (float)(zz * per_token);
        out.shares[E] = (float)per_token;
    }
}

// Partial sums of `per_block` consecutive tokens per workgroup: prob and count [G][E padded to 4], z [G], tokens [G]; ALONE: the only
// workgroup, which writes the results.
template <typename T, int LPT, int CHUNKS, int WAVES, bool VEC, bool ALONE>
__global__ void __launch_bounds__(WAVES * CK_WAVE)
    balance_fwd_kernel(const typename T::storage_t* __restrict__ logits, int64_t ld, const int64_t* __restrict__ selected,
                       const uint8_t* __restrict__ mask, int64_t tokens, int E, int k, int64_t per_block,
                       float* __restrict__ prob_partial, int* __restrict__ count_partial, float* __restrict__ z_partial,
                       int* __restrict__ token_partial, BalanceOut out) {
    constexpr int COLS = LPT * kPiece * CHUNKS;
    constexpr int TPW = CK_WAVE / LPT;  // tokens a wave holds at once
    __shared__ float prob[WAVES][COLS];
    __shared__ int count[COLS];
    __shared__ float z_wave[WAVES];
    __shared__ int n_wave[WAVES];
    const int wave = threadIdx.x / CK_WAVE, lane = lane_id(), first = (lane % LPT) * kPiece;
    const int64_t t0 = (int64_t)blockIdx.x * per_block;
    const int64_t t1 = t0 + per_block < tokens ? t0 + per_block : tokens;
    int size[CHUNKS];
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) size[c] = piece_size(E, first + c * LPT * kPiece);
    // a turn's rows: requested first, worked on after the next turn's are on their way
    struct Rows {
        Piece<T, kPiece> row[CHUNKS];
        bool real;
    };
    auto fetch = [&](int64_t base, Rows& r) __attribute__((always_inline)) {
        const int64_t t = base + lane / LPT;
        r.real = t < t1 && (mask == nullptr || mask[t] != 0);
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            r.row[c].clear();
            if (r.real && size[c] > 0)
                r.row[c] = load_piece<T, kPiece, VEC, false>(logits + t * ld + first + c * LPT * kPiece, size[c]);
        }
    };
    int64_t base = t0 + wave * TPW;
    Rows cur, next;
    fetch(base, cur);
    for (int e = threadIdx.x; e < COLS; e += WAVES * CK_WAVE) count[e] = 0;
    __syncthreads();

    for (int64_t i = t0 * k + threadIdx.x; i < t1 * k; i += WAVES * CK_WAVE) {
        const int64_t id = selected[i];
        if (id >= 0 && id < E && (mask == nullptr || mask[t0 + (uint32_t)(i - t0 * k) / (uint32_t)k] != 0))
            atomicAdd(&count[id], 1);
    }

    float acc[CHUNKS][kPiece];
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
        for (int j = 0; j < kPiece; ++j) acc[c][j] = 0.f;
    float z = 0.f;
    int n = 0;
    for (; base < t1; base += WAVES * TPW) {
        fetch(base + WAVES * TPW, next);
        float v[CHUNKS][kPiece];
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
            for (int j = 0; j < kPiece; ++j) v[c][j] = cur.row[c].up(j);
        const float lse = token_softmax<T, LPT, CHUNKS, VEC>(v, size);
        if (cur.real) {
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
                for (int j = 0; j < kPiece; ++j) acc[c][j] += v[c][j];
            if (lane % LPT == 0) {
                z += lse * lse;
                n += 1;
            }
        }
        cur = next;
    }
    // the wave's token groups, then the waves
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
        for (int j = 0; j < kPiece; ++j) {
#pragma unroll
            for (int off = LPT; off < CK_WAVE; off <<= 1) acc[c][j] += __shfl_xor(acc[c][j], off, CK_WAVE);
            if (lane < LPT) prob[wave][c * LPT * kPiece + first + j] = acc[c][j];
        }
    z = wave_sum(z);
    n = wave_sum_i(n);
    if (lane == 0) {
        z_wave[wave] = z;
        n_wave[wave] = n;
    }
    __syncthreads();
    if (ALONE) {
        double p = 0.0, zz = 0.0;
        int c = 0, nn = 0;
        if ((int)threadIdx.x < E) {
#pragma unroll
            for (int w = 0; w < WAVES; ++w) p += (double)prob[w][threadIdx.x];
            c = count[threadIdx.x];
        }
        if (threadIdx.x < WAVES) {
            zz = (double)z_wave[threadIdx.x];
            nn = n_wave[threadIdx.x];
        }
        balance_finish<WAVES>(p, c, zz, nn, E, k, out);
    } else {
        // (columns up to the next multiple of four: a piece's columns beyond E hold zeros)
        const int padded = (E + 3) & ~3;
        for (int e = threadIdx.x; e < padded; e += WAVES * CK_WAVE) {
            float p = 0.f;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) p += prob[w][e];
            prob_partial[(int64_t)blockIdx.x * padded + e] = p;
            count_partial[(int64_t)blockIdx.x * padded + e] = count[e];
        }
        if (threadIdx.x == 0) {
            float zz = 0.f;
            int nn = 0;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                zz += z_wave[w];
                nn += n_wave[w];
            }
            z_partial[blockIdx.x] = zz;
            token_partial[blockIdx.x] = nn;
        }
    }
}

// One workgroup adds the partial sums of `parts` workgroups up.  A thread owns four columns (rows of partial sums are padded
// to `padded`, a multiple of four) and every `1024 / quads`-th row, with `quads` a power of two >= padded / 4; lanes of a
// wave that own the same columns meet by shuffles, waves in LDS.
__global__ void __launch_bounds__(1024)
    balance_sum_kernel(const float* __restrict__ prob_partial, const int* __restrict__ count_partial,
                       const float* __restrict__ z_partial, const int* __restrict__ token_partial, int parts, int E,
                       int padded, int k, int quads, BalanceOut out) {
    __shared__ float prob[4096];  // [places][4 * quads]: 16 waves, or fewer rows of more than 64 quads
    __shared__ int count[4096];
    const int quad = threadIdx.x & (quads - 1), group = threadIdx.x / quads, groups = 1024 / quads;
    float p[4] = {0.f, 0.f, 0.f, 0.f};
    int c[4] = {0, 0, 0, 0};
    if (quad * 4 < padded) {
#pragma unroll 4
        for (int r = group; r < parts; r += groups) {
            const float4 pv = *reinterpret_cast<const float4*>(prob_partial + (int64_t)r * padded + quad * 4);
            const int4 cv = *reinterpret_cast<const int4*>(count_partial + (int64_t)r * padded + quad * 4);
            p[0] += pv.x;
            p[1] += pv.y;
            p[2] += pv.z;
            p[3] += pv.w;
            c[0] += cv.x;
            c[1] += cv.y;
            c[2] += cv.z;
            c[3] += cv.w;
        }
    }
    double z = 0.0;
    int n = 0;
    for (int r = threadIdx.x; r < parts; r += 1024) {
        z += (double)z_partial[r];
        n += token_partial[r];
    }
    for (int off = quads; off < CK_WAVE; off <<= 1) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            p[j] += __shfl_xor(p[j], off, CK_WAVE);
            c[j] += __shfl_xor(c[j], off, CK_WAVE);
        }
    }
    const int place = quads < CK_WAVE ? (int)threadIdx.x / CK_WAVE : group;
    const int places = quads < CK_WAVE ? 1024 / CK_WAVE : groups;
    if (quads >= CK_WAVE || lane_id() < quads) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            prob[place * 4 * quads + quad * 4 + j] = p[j];
            count[place * 4 * quads + quad * 4 + j] = c[j];
        }
    }
    __syncthreads();
    double total = 0.0;
    int hits = 0;
    if ((int)threadIdx.x < E) {
        for (int g = 0; g < places; ++g) {
            total += (double)prob[g * 4 * quads + threadIdx.x];
            hits += count[g * 4 * quads + threadIdx.x];
        }
    }
    balance_finish<16>(total, hits, z, n, E, k, out);
}

template <typename T, int LPT, int CHUNKS, bool VEC>
__global__ void __launch_bounds__(256)
    balance_bwd_kernel(const typename T::storage_t* __restrict__ logits, int64_t ld, const uint8_t* __restrict__ mask,
                       const float* __restrict__ shares, const float* __restrict__ balance_grad,
                       const float* __restrict__ z_grad, typename T::storage_t* __restrict__ d_logits, int64_t tokens, int E) {
    constexpr int TPW = CK_WAVE / LPT;
    const int lane = lane_id(), first = (lane % LPT) * kPiece;
    const int64_t wave = (int64_t)blockIdx.x * 4 + threadIdx.x / CK_WAVE, waves = (int64_t)gridDim.x * 4;
    const float g_b = balance_grad != nullptr ? *balance_grad : 0.f;
    const float z_scale = z_grad != nullptr ? 2.f * *z_grad * shares[E] : 0.f;
    int size[CHUNKS];
    float a[CHUNKS][kPiece];
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
        size[c] = piece_size(E, first + c * LPT * kPiece);
#pragma unroll
        for (int j = 0; j < kPiece; ++j) {
            const int e = first + c * LPT * kPiece + j;
            a[c][j] = e < E ? g_b * shares[e] : 0.f;
        }
    }
    for (int64_t base = wave * TPW; base < tokens; base += waves * TPW) {
        const int64_t t = base + lane / LPT;
        const bool real = t < tokens && (mask == nullptr || mask[t] != 0);
        float v[CHUNKS][kPiece];
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            Piece<T, kPiece> row;
            row.clear();
            if (real && size[c] > 0)
                row = load_piece<T, kPiece, VEC, false>(logits + t * ld + first + c * LPT * kPiece, size[c]);
#pragma unroll
            for (int j = 0; j < kPiece; ++j) v[c][j] = row.up(j);
        }
        const float lse = token_softmax<T, LPT, CHUNKS, VEC>(v, size);
        float inner = 0.f;
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
            for (int j = 0; j < kPiece; ++j) inner += a[c][j] * v[c][j];
        inner = group_sum<LPT>(inner);
        const float shift = z_scale * lse - inner;
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            Piece<T, kPiece> o;
#pragma unroll
            for (int j = 0; j < kPiece; ++j) o.put(j, real ? v[c][j] * (a[c][j] + shift) : 0.f);
            if (t < tokens && size[c] > 0)
                store_piece<T, kPiece, VEC>(o, d_logits + t * E + first + c * LPT * kPiece, size[c]);
        }
    }
}

}  // namespace ck

// ---- host side ---------------------------------------------------------------------------------------------------------
namespace {

int balance_lanes(int64_t E) {
    int lanes = 1;
    while (lanes < 64 && lanes * ck::kPiece < E) lanes *= 2;
    return lanes;
}
// Tokens sixteen waves hold at once
int64_t balance_turn(int64_t E) { return 16 * (64 / balance_lanes(E)); }
// Workgroups of the forward: a turn each, up to one per compute unit, and no more than 128 K pairs for the workgroup that
// adds them up.  Measured (both launches): 65521 x 160 fp32 24.3 us, with twice the workgroups 27.0, with half 32.3.  One
// workgroup alone takes up to four turns: 4096 x 8 bf16 11.2 us, against 12.1 in two launches; beyond, the two launches win
// (8192 x 8: 12.3 against 18.6).
int64_t balance_parts(int64_t tokens, int64_t E) {
    if (tokens <= 4 * balance_turn(E)) return 1;
    const int64_t wanted = ck_ceil_div(tokens, balance_turn(E));
    const int64_t most = 131072 / E < 256 ? 131072 / E : 256;
    return wanted < most ? wanted : most;
}
int64_t balance_padded(int64_t E) { return (E + 3) / 4 * 4; }
int64_t balance_workspace(int64_t parts, int64_t E) { return parts == 1 ? 0 : parts * (balance_padded(E) + 1) * 8; }

struct BalanceArgs {
    const void* logits;
    int64_t ld;
    const int64_t* selected;
    const uint8_t* mask;
    int64_t tokens;
    int E, k;
    int64_t parts, per_block;
    float *prob, *z;
    int *count, *n;
    ck::BalanceOut out;
};
template <typename T, int LPT, int CHUNKS, bool VEC>
void balance_launch_fwd(hipStream_t s, const BalanceArgs& a) {
    typedef typename T::storage_t S;
    if (a.parts == 1)
        hipLaunchKernelGGL((ck::balance_fwd_kernel<T, LPT, CHUNKS, 16, VEC, true>), dim3(1), dim3(1024), 0, s,
                           (const S*)a.logits, a.ld, a.selected, a.mask, a.tokens, a.E, a.k, a.tokens, (float*)nullptr,
                           (int*)nullptr, (float*)nullptr, (int*)nullptr, a.out);
    else
        hipLaunchKernelGGL((ck::balance_fwd_kernel<T, LPT, CHUNKS, 16, VEC, false>), dim3((unsigned)a.parts), dim3(1024), 0, s,
                           (const S*)a.logits, a.ld, a.selected, a.mask, a.tokens, a.E, a.k, a.per_block, a.prob, a.count,
                           a.z, a.n, a.out);
}
struct BalanceBwd {
    const void* logits;
    int64_t ld;
    const uint8_t* mask;
    const float *shares, *balance_grad, *z_grad;
    void* d_logits;
    int64_t tokens;
    int E;
};
template <typename T, int LPT, int CHUNKS, bool VEC>
void balance_launch_bwd(hipStream_t s, const BalanceBwd& a) {
    typedef typename T::storage_t S;
    // (a wave reads the experts' shares once for all its turns.  fp32, 1024 / 2048 workgroups: 65521 x 160 19.2 / 18.7 us,
    // 65536 x 256 29.1 / 32.7, 30000 x 200 11.9 / 15.1; 8192 x 1000 bf16 15.7 / 21.3)
    const int64_t need = ck_ceil_div(a.tokens, 4 * (64 / LPT));
    hipLaunchKernelGGL((ck::balance_bwd_kernel<T, LPT, CHUNKS, VEC>), dim3((unsigned)(need < 1024 ? need : 1024)), dim3(256),
                       0, s, (const S*)a.logits, a.ld, a.mask, a.shares, a.balance_grad, a.z_grad, (S*)a.d_logits, a.tokens, a.E);
}

#define CK_BALANCE_LANES(E, ...)                                                    \
    switch (balance_lanes(E)) {                                                     \
        case 1: { constexpr int LPT = 1, CHUNKS = 1; __VA_ARGS__; } break;          \
        case 2: { constexpr int LPT = 2, CHUNKS = 1; __VA_ARGS__; } break;          \
        case 4: { constexpr int LPT = 4, CHUNKS = 1; __VA_ARGS__; } break;          \
        case 8: { constexpr int LPT = 8, CHUNKS = 1; __VA_ARGS__; } break;          \
        case 16: { constexpr int LPT = 16, CHUNKS = 1; __VA_ARGS__; } break;        \
        case 32: { constexpr int LPT = 32, CHUNKS = 1; __VA_ARGS__; } break;        \
        default:                                                                    \
            if ((E) <= 512) {                                                       \
                constexpr int LPT = 64, CHUNKS = 1;                                 \
                __VA_ARGS__;                                                        \
            } else {                                                                \
                constexpr int LPT = 64, CHUNKS = 2;                                 \
                __VA_ARGS__;                                                        \
            }                                                                       \
    }

bool balance_shape(int64_t tokens, int64_t E, int64_t k) {
    return tokens >= 0 && E >= 1 && E <= ck::kBalanceMaxExperts && k >= 1 && k <= E && tokens <= 0x7fffffff / k;
}

}  // namespace

extern "C" int64_t ck_moe_balance_loss_workspace_size(int64_t tokens, int64_t E) {
    if (tokens <= 0 || E < 1 || E > ck::kBalanceMaxExperts) return 0;
    const int64_t parts = balance_parts(tokens, E);
    return balance_workspace(parts, E);
}

extern "C" int ck_moe_balance_loss_forward(const void* logits, int64_t ld, const int64_t* selected, const void* mask,
                                           float* balance, float* z, int* counts, float* shares, void* workspace,
                                           int64_t workspace_bytes, int64_t tokens, int64_t E, int64_t k, int dtype,
                                           void* stream) {
    if (!balance_shape(tokens, E, k) || ld < E) return CK_ERR_SHAPE;
    if (dtype != CK_F32 && dtype != CK_F16 && dtype != CK_BF16) return CK_ERR_DTYPE;
    if (!balance || !z || !counts || !shares || (tokens > 0 && (!logits || !selected))) return CK_ERR_NULL;
    if (!ck_aligned_elem(logits, dtype)) return CK_ERR_ALIGN;
    const int64_t parts = balance_parts(tokens, E);
    const int64_t need = balance_workspace(parts, E);
    if (need > 0 && (!workspace || !ck_aligned16(workspace) || workspace_bytes < need)) return CK_ERR_WORKSPACE;
    BalanceArgs a;
    a.logits = logits;
    a.ld = ld;
    a.selected = selected;
    a.mask = (const uint8_t*)mask;
    a.tokens = tokens;
    a.E = (int)E;
    a.k = (int)k;
    a.parts = parts;
    a.per_block = ck_ceil_div(tokens, parts);
    a.prob = (float*)workspace;
    const int64_t cells = parts * balance_padded(E);
    a.count = (int*)workspace + cells;
    a.z = (float*)workspace + 2 * cells;
    a.n = (int*)workspace + 2 * cells + parts;
    a.out = {balance, z, shares, counts};
    hipStream_t s = (hipStream_t)stream;
    const bool vec = E % ck::kPiece == 0 && ld % ck::kPiece == 0 && ck_aligned16(logits);
    CK_DISPATCH_DTYPE(dtype, {
        CK_BALANCE_LANES(E, {
            if (vec) balance_launch_fwd<T, LPT, CHUNKS, true>(s, a);
            else balance_launch_fwd<T, LPT, CHUNKS, false>(s, a);
        });
    });
    if (parts > 1) {
        int quads = 1;
        while (quads * 4 < E) quads *= 2;
        hipLaunchKernelGGL((ck::balance_sum_kernel), dim3(1), dim3(1024), 0, s, a.prob, a.count, a.z, a.n, (int)parts, a.E,
                           (int)balance_padded(E), a.k, quads, a.out);
    }
    return ck_launch_status();
}

extern "C" int ck_moe_balance_loss_backward(const void* logits, int64_t ld, const void* mask, const float* shares,
                                            const float* balance_grad, const float* z_grad, void* d_logits, int64_t tokens,
                                            int64_t E, int dtype, void* stream) {
    if (!balance_shape(tokens, E, 1) || ld < E) return CK_ERR_SHAPE;
    if (dtype != CK_F32 && dtype != CK_F16 && dtype != CK_BF16) return CK_ERR_DTYPE;
    if (tokens == 0) return CK_OK;
    if (!logits || !shares || !d_logits) return CK_ERR_NULL;
    if (!ck_aligned_elem(logits, dtype) || !ck_aligned_elem(d_logits, dtype)) return CK_ERR_ALIGN;
    const BalanceBwd a = {logits, ld, (const uint8_t*)mask, shares, balance_grad, z_grad, d_logits, tokens, (int)E};
    hipStream_t s = (hipStream_t)stream;
    const bool vec = E % ck::kPiece == 0 && ld % ck::kPiece == 0 && ck_aligned16(logits) && ck_aligned16(d_logits);
    CK_DISPATCH_DTYPE(dtype, {
        CK_BALANCE_LANES(E, {
            if (vec) balance_launch_bwd<T, LPT, CHUNKS, true>(s, a);
            else balance_launch_bwd<T, LPT, CHUNKS, false>(s, a);
        });
    });
    return ck_launch_status();
}
