// Gated linear unit, forward and backward.
//
//   w [2F, K], rows 0..F-1 the gate's and F..2F-1 the value's
//   g = x Wg^T + bg;  u = x Wu^T + bu;  y = silu(g) u
//   dg = dy u silu'(g);  du = dy silu(g);  dp = [dg du]
//   dx = dp W;  dW = dp^T x;  db = sum over rows of dp
//
// Four products of one tiled kernel. The first two share their main loop: a
// block's columns are as many gate columns as value columns of the same
// indexes, so each lane ends with g and u of the same elements, and the
// activation, the product and (backward) dp are written from the accumulators.
// The backward pass computes g and u again in place of keeping them: nothing
// but the inputs lives between the passes, and g and u are never rounded.

#include "gated_common.h"

namespace {

using f4 = __attribute__((ext_vector_type(4))) float;
using bf8 = __attribute__((ext_vector_type(8))) __bf16;

constexpr int TILE = 64, DEPTH = 32;

// What the matrix instruction takes of a lane: KL values of consecutive k, of
// the row (or column) lane % 16, at k = (lane / 16) * KL.
template <typename E> struct Mfma;
template <> struct Mfma<bf16> {
    static constexpr int STEP = 32, KL = 8;
    static DEV_INLINE f4 mul(const bf16* a, const bf16* b, f4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(*reinterpret_cast<const bf8*>(a),
                                                       *reinterpret_cast<const bf8*>(b), c, 0, 0, 0);
    }
};
template <> struct Mfma<float> {
    static constexpr int STEP = 4, KL = 1;
    static DEV_INLINE f4 mul(const float* a, const float* b, f4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x4f32(*a, *b, c, 0, 0, 0);
    }
};

enum class End { GATED, GATED_GRAD, PLAIN, PART };

// C(m, n) = sum over k of A(m, k) B(n, k); A and B have strides for both axes.
template <typename E>
struct Args {
    const E *a, *b;
    int64_t am, ak, bn, bk;
    int M, N, K;       // GATED*: N is F
    const E* bias;     // [2F] or null
    const E* dy;       // [M, F]
    E* out;            // GATED: y [M, F]; GATED_GRAD: dp [M, 2F]; PLAIN: [M, N]
    float* part;       // GATED_GRAD: [blocks of rows, 2F] or null; PART: [splits, M, N]
    int per_split;     // k of one split
};

template <typename E, End END>
__global__ void __launch_bounds__(256)
product_kernel(Args<E> p) {
    constexpr bool GATED = END == End::GATED || END == End::GATED_GRAD;
    constexpr int PAD = 16 / sizeof(E), STEP = Mfma<E>::STEP, KL = Mfma<E>::KL;
    constexpr int COLS = GATED ? TILE / 2 : TILE;  // columns of the result a block
    __shared__ __attribute__((aligned(16))) E as[TILE][DEPTH + PAD], bs[TILE][DEPTH + PAD];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int m0 = blockIdx.y * TILE, n0 = blockIdx.x * COLS;
    const int k_lo = blockIdx.z * p.per_split;
    const int k_hi = k_lo + p.per_split < p.K ? k_lo + p.per_split : p.K;
    // wave (wm, wn): rows wm * 32.., and columns wn * 32.. of the plain forms, or
    // gate columns wn * 16.. with their value columns of the gated ones
    const int wm = wave >> 1, wn = wave & 1;
    f4 acc[2][2] = {};
    for (int k0 = k_lo; k0 < k_hi; k0 += DEPTH) {
        __syncthreads();
        for (int e = threadIdx.x; e < TILE * DEPTH; e += 256) {
            // neighbours in the axis that lies together in memory
            const int am = p.ak == 1 ? e / DEPTH : e % TILE, ak = p.ak == 1 ? e % DEPTH : e / TILE;
            const int m = m0 + am, ka = k0 + ak;
            as[am][ak] = m < p.M && ka < k_hi ? p.a[m * p.am + ka * p.ak] : from_f<E>(0.0f);
            const int bn = p.bk == 1 ? e / DEPTH : e % TILE, bk = p.bk == 1 ? e % DEPTH : e / TILE;
            const int col = n0 + (GATED ? bn % COLS : bn), kb = k0 + bk;
            const int64_t row = GATED && bn >= COLS ? (int64_t)col + p.N : col;
            bs[bn][bk] = col < p.N && kb < k_hi ? p.b[row * p.bn + kb * p.bk] : from_f<E>(0.0f);
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < DEPTH; k += STEP) {
            const int at = k + (lane >> 4) * KL;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int r = wm * 32 + i * 16 + (lane & 15);
                    const int c = (GATED ? j * COLS + wn * 16 : wn * 32 + j * 16) + (lane & 15);
                    acc[i][j] = Mfma<E>::mul(&as[r][at], &bs[c][at], acc[i][j]);
                }
        }
    }
    // an accumulator's element q is at row (lane / 16) * 4 + q, column lane % 16
    if constexpr (GATED) {
        __shared__ float sums[2][2][COLS];
        const int col = n0 + wn * 16 + (lane & 15);
        float sg = 0.0f, su = 0.0f;
        if (col < p.N) {
            const float bg = p.bias ? to_f(p.bias[col]) : 0.0f;
            const float bu = p.bias ? to_f(p.bias[p.N + col]) : 0.0f;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int row = m0 + wm * 32 + i * 16 + (lane >> 4) * 4 + q;
                    if (row >= p.M) continue;
                    const float g = acc[i][0][q] + bg, u = acc[i][1][q] + bu;
                    float val, grad;
                    silu_grad(g, val, grad);
                    if (END == End::GATED) {
                        p.out[(int64_t)row * p.N + col] = from_f<E>(val * u);
                    } else {
                        const float d = to_f(p.dy[(int64_t)row * p.N + col]);
                        const float dg = d * u * grad, du = d * val;
                        p.out[(int64_t)row * 2 * p.N + col] = from_f<E>(dg);
                        p.out[(int64_t)row * 2 * p.N + p.N + col] = from_f<E>(du);
                        sg += dg;
                        su += du;
                    }
                }
        }
        if (END == End::GATED_GRAD && p.part) {
            sg += __shfl_xor(sg, 16, 64); sg += __shfl_xor(sg, 32, 64);
            su += __shfl_xor(su, 16, 64); su += __shfl_xor(su, 32, 64);
            if (lane < 16) {
                sums[wm][0][wn * 16 + lane] = sg;
                sums[wm][1][wn * 16 + lane] = su;
            }
            __syncthreads();
            const int c = threadIdx.x % COLS, which = threadIdx.x / COLS;
            if (which < 2 && n0 + c < p.N)
                p.part[(int64_t)blockIdx.y * 2 * p.N + which * (int64_t)p.N + n0 + c] =
                    sums[0][which][c] + sums[1][which][c];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int row = m0 + wm * 32 + i * 16 + (lane >> 4) * 4 + q;
                    const int col = n0 + wn * 32 + j * 16 + (lane & 15);
                    if (row >= p.M || col >= p.N) continue;
                    const int64_t at = (int64_t)row * p.N + col;
                    if (END == End::PLAIN) p.out[at] = from_f<E>(acc[i][j][q]);
                    else p.part[blockIdx.z * (int64_t)p.M * p.N + at] = acc[i][j][q];
                }
    }
}

// out = sum over the splits of part, in their order.
template <typename E>
__global__ void __launch_bounds__(256)
join_splits_kernel(const float* __restrict__ part, E* __restrict__ out, int64_t n, int splits) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    float s = 0.0f;
    for (int z = 0; z < splits; ++z) s += part[z * n + i];
    out[i] = from_f<E>(s);
}

int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

template <typename E>
int fwd(const void* x, const void* w, const void* bias, void* y, int M, int K, int F,
        hipStream_t st) {
    if ((int64_t)M * F == 0) return 0;
    Args<E> p{};
    p.a = (const E*)x; p.am = K; p.ak = 1;
    p.b = (const E*)w; p.bn = K; p.bk = 1;
    p.M = M; p.N = F; p.K = K; p.per_split = K;
    p.bias = (const E*)bias; p.out = (E*)y;
    product_kernel<E, End::GATED>
        <<<dim3(ceil_div(F, TILE / 2), ceil_div(M, TILE)), 256, 0, st>>>(p);
    LSTM_CHECK_LAUNCH();
    return 0;
}

template <typename E>
int bwd(const void* x, const void* w, const void* bias, const void* dy, void* dp, void* dx,
        void* dw, void* db, float* part_db, float* part_dw, int M, int K, int F, int splits,
        hipStream_t st) {
    if ((int64_t)M * F != 0) {
        Args<E> p{};
        p.a = (const E*)x; p.am = K; p.ak = 1;
        p.b = (const E*)w; p.bn = K; p.bk = 1;
        p.M = M; p.N = F; p.K = K; p.per_split = K;
        p.bias = (const E*)bias; p.dy = (const E*)dy; p.out = (E*)dp; p.part = db ? part_db : nullptr;
        product_kernel<E, End::GATED_GRAD>
            <<<dim3(ceil_div(F, TILE / 2), ceil_div(M, TILE)), 256, 0, st>>>(p);
        LSTM_CHECK_LAUNCH();
    }
    if (db) {
        column_sum_kernel<E><<<ceil_div(2 * F, 64), 1024, 0, st>>>(
            part_db, (E*)db, ceil_div(M, TILE), 2 * F);
        LSTM_CHECK_LAUNCH();
    }
    if (dx && (int64_t)M * K != 0) {
        Args<E> p{};
        p.a = (const E*)dp; p.am = 2 * (int64_t)F; p.ak = 1;
        p.b = (const E*)w; p.bn = 1; p.bk = K;
        p.M = M; p.N = K; p.K = 2 * F; p.per_split = 2 * F;
        p.out = (E*)dx;
        product_kernel<E, End::PLAIN>
            <<<dim3(ceil_div(K, TILE), ceil_div(M, TILE)), 256, 0, st>>>(p);
        LSTM_CHECK_LAUNCH();
    }
    if (dw && (int64_t)F * K != 0) {
        Args<E> p{};
        p.a = (const E*)dp; p.am = 1; p.ak = 2 * (int64_t)F;
        p.b = (const E*)x; p.bn = 1; p.bk = K;
        p.M = 2 * F; p.N = K; p.K = M;
        p.per_split = ceil_div(ceil_div(M > 0 ? M : 1, splits), DEPTH) * DEPTH;
        p.part = part_dw;
        product_kernel<E, End::PART>
            <<<dim3(ceil_div(K, TILE), ceil_div(2 * F, TILE), splits), 256, 0, st>>>(p);
        LSTM_CHECK_LAUNCH();
        const int64_t n = (int64_t)2 * F * K;
        join_splits_kernel<E><<<ceil_div(n, 256), 256, 0, st>>>(part_dw, (E*)dw, n, splits);
        LSTM_CHECK_LAUNCH();
    }
    return 0;
}

}  // namespace

extern "C" int launch_gated_linear_fwd(int is_bf16, const void* x, const void* w,
                                       const void* bias, void* y, int M, int K, int F,
                                       hipStream_t st) {
    return is_bf16 ? fwd<bf16>(x, w, bias, y, M, K, F, st)
                   : fwd<float>(x, w, bias, y, M, K, F, st);
}

// Rows of 2F partial sums for db, and splits of 2F * K partial sums for dw.
extern "C" int gated_linear_bias_parts(int M) { return ceil_div(M, TILE); }
extern "C" int gated_linear_splits(int M, int K, int F) {
    const int64_t tiles = (int64_t)ceil_div(2 * F, TILE) * ceil_div(K, TILE);
    const int64_t want = ceil_div(1024, tiles > 0 ? tiles : 1), most = ceil_div(M, 8 * DEPTH);
    return (int)(want < most ? (want > 0 ? want : 1) : (most > 0 ? most : 1));
}

extern "C" int launch_gated_linear_bwd(int is_bf16, const void* x, const void* w,
                                       const void* bias, const void* dy, void* dp, void* dx,
                                       void* dw, void* db, float* part_db, float* part_dw,
                                       int M, int K, int F, int splits, hipStream_t st) {
    return is_bf16 ? bwd<bf16>(x, w, bias, dy, dp, dx, dw, db, part_db, part_dw, M, K, F, splits, st)
                   : bwd<float>(x, w, bias, dy, dp, dx, dw, db, part_db, part_dw, M, K, F, splits, st);
}
