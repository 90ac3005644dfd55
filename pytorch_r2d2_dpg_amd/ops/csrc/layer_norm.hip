// Layer norm over the last axis, forward and backward.
//
//   s = x + r;  n = (s - mean(s)) * rstd;  y = n w + b
//   g = dy w;   dx = rstd (g - mean(g) - n mean(g n)) + ds
//   dw = sum over rows of dy n;  db = sum over rows of dy
//
// Memory bound: about ten operations an element. A row lives in the registers
// of its threads between the sums over it, so each input is read once. bf16 with a
// residual, on the MI355X: 32768 rows of 4096 take 183 us forward, 277 backward
// and 8 for the weight's sums, 5.9 and 4.9 TB/s, where a copy of 2 GiB reaches
// 4.9; 20480 rows of 512, which the last level of cache holds, 17, 22 and 4 us.
// Rows outside of 256 to 8192 elements are far from that: those of up to 256 leave
// lanes of their wave idle (1048576 of 64: 283 and 703 us, 1.9 and 0.95 TB/s), those
// past 8192, and those shorter than a load, are read element by element and three
// times (16384 of 8192: 184, 294 and 13 us; of 8200: 491, 1174 and 245; 4300000 of 3
// without a residual: 802, 1123 and 2592).

#include "gated_common.h"

#include <algorithm>

namespace {

template <typename E> constexpr int RUN = 16 / (int)sizeof(E);  // one load of a lane

// Sums of two values over the TPR threads of a row, the same in each of them.
// `turn` alternates between two places in LDS: one barrier a sum.
template <int TPR>
DEV_INLINE void row_sums(float& a, float& b, float2 (*lds)[16], int& turn) {
    a = wave_sum(a);
    b = wave_sum(b);
    if constexpr (TPR > 64) {
        constexpr int W = TPR / 64;
        if ((threadIdx.x & 63) == 0) lds[turn][threadIdx.x >> 6] = make_float2(a, b);
        __syncthreads();
        a = b = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            a += lds[turn][w].x;
            b += lds[turn][w].y;
        }
        turn ^= 1;
    }
}

// A thread's share of a row: run k starts at element at[k], and its elements
// from skip[k] on are the thread's own. A row's last run starts early, so that
// it is whole too; what it shares with the run before it is computed in both,
// stored twice with one value, and summed in one. A run past the row is all
// skipped. Needs dim >= RUN.
template <typename E, int TPR, int NV>
struct Share {
    int at[NV], skip[NV];
    DEV_INLINE explicit Share(int dim) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = ((int)(threadIdx.x % TPR) + k * TPR) * RUN<E>;
            at[k] = c < dim - RUN<E> ? c : dim - RUN<E>;
            skip[k] = c - at[k];
        }
    }
};

// A run as it lies in memory.
template <typename E>
struct Raw {
    E v[RUN<E>];
    DEV_INLINE void load(const E* p) { load_run<E, RUN<E>>(p, RUN<E>, v); }
    DEV_INLINE float operator[](int i) const { return to_f(v[i]); }
};

// Threads of a block: four rows of a wave each, or one row, whose waves meet at
// barriers.
constexpr int block_of(int tpr) { return tpr > 64 ? tpr : 256; }

// Rows blockIdx, blockIdx + gridDim, ... of ROWS each, TPR threads and NV runs a
// thread to a row. The weights stay in registers, and a row's loads go out
// before the row in front of it is reduced. The mean comes off before squaring:
// the variance of a row far from zero does not cancel.
template <typename E, int TPR, int NV, bool FUSED>
__global__ void __launch_bounds__(block_of(TPR))
norm_fwd_kernel(const E* __restrict__ x, const E* __restrict__ res,
                const E* __restrict__ w, const E* __restrict__ b,
                E* __restrict__ y, E* __restrict__ s_out,
                int64_t rows, int dim, float eps) {
    constexpr int R = RUN<E>, ROWS = block_of(TPR) / TPR;
    __shared__ float2 lds[2][16];
    const Share<E, TPR, NV> my(dim);
    Raw<E> wr[NV], br[NV], xr[NV], rr[NV];
    int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / TPR;
    const auto fetch = [&](int64_t row) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            xr[k].load(x + row * dim + my.at[k]);
            if (FUSED) rr[k].load(res + row * dim + my.at[k]);
        }
    };
    if (row < rows) fetch(row);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        wr[k].load(w + my.at[k]);
        if (b) br[k].load(b + my.at[k]);
    }
    int turn = 0;
    // a block of one row at a time leaves the loop as one
    for (; row < rows; row += (int64_t)gridDim.x * ROWS) {
        float v[NV][R], sum = 0.0f, sq = 0.0f, none = 0.0f;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
#pragma unroll
            for (int i = 0; i < R; ++i) {
                v[k][i] = xr[k][i] + (FUSED ? rr[k][i] : 0.0f);
                sum += i >= my.skip[k] ? v[k][i] : 0.0f;
            }
            if (FUSED && my.skip[k] < R) {
                E so[R];
#pragma unroll
                for (int i = 0; i < R; ++i) so[i] = from_f<E>(v[k][i]);
                store_run<E, R>(s_out + row * dim + my.at[k], R, so);
            }
        }
        const int64_t next = row + (int64_t)gridDim.x * ROWS;
        if (next < rows) fetch(next);
        row_sums<TPR>(sum, none, lds, turn);
        const float mean = sum / dim;
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int i = 0; i < R; ++i) {
                v[k][i] -= mean;
                sq += i >= my.skip[k] ? v[k][i] * v[k][i] : 0.0f;
            }
        row_sums<TPR>(sq, none, lds, turn);
        const float rstd = 1.0f / sqrtf(sq / dim + eps);
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            if (my.skip[k] >= R) continue;
            E out[R];
#pragma unroll
            for (int i = 0; i < R; ++i)
                out[i] = from_f<E>(v[k][i] * rstd * wr[k][i] + (b ? br[k][i] : 0.0f));
            store_run<E, R>(y + row * dim + my.at[k], R, out);
        }
    }
}

// The same walk. A thread's columns stay the same from row to row, so the
// weight's gradient sums up in registers and leaves once a block, as a row of
// part [gridDim][2][dim].
//
// s is summed again from x and r, not read back as the forward pass rounded it:
// in bf16 that rounding alone would add half again to the error of dw. The mean
// and rstd come from the same registers. The sums join in two rounds: those of
// s and g, then those of (s - mean)^2 and g (s - mean).
template <typename E, int TPR, int NV, bool FUSED>
__global__ void __launch_bounds__(block_of(TPR))
norm_bwd_kernel(const E* __restrict__ x, const E* __restrict__ res,
                const E* __restrict__ w, const E* __restrict__ dy,
                const E* __restrict__ ds, E* __restrict__ dx,
                float* __restrict__ part, int64_t rows, int dim, float eps) {
    constexpr int R = RUN<E>, ROWS = block_of(TPR) / TPR;
    __shared__ float2 lds[2][16];
    const Share<E, TPR, NV> my(dim);
    Raw<E> wr[NV], xr[NV], rr[NV], dr[NV], pr[NV];
    float dw[NV][R] = {}, db[NV][R] = {};
    const int sub = threadIdx.x / TPR, tid = threadIdx.x % TPR;
    int64_t row = (int64_t)blockIdx.x * ROWS + sub;
    const auto fetch = [&](int64_t row) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            xr[k].load(x + row * dim + my.at[k]);
            if (FUSED) rr[k].load(res + row * dim + my.at[k]);
            dr[k].load(dy + row * dim + my.at[k]);
        }
    };
    if (row < rows) fetch(row);
#pragma unroll
    for (int k = 0; k < NV; ++k) wr[k].load(w + my.at[k]);
    int turn = 0;
    for (; row < rows; row += (int64_t)gridDim.x * ROWS) {
        float n[NV][R], d[NV][R], sum = 0.0f, sg = 0.0f, sq = 0.0f, sgn = 0.0f;
        if (FUSED && ds)
#pragma unroll
            for (int k = 0; k < NV; ++k) pr[k].load(ds + row * dim + my.at[k]);
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int i = 0; i < R; ++i) {
                n[k][i] = xr[k][i] + (FUSED ? rr[k][i] : 0.0f);
                d[k][i] = dr[k][i];
                const bool own = i >= my.skip[k];
                sum += own ? n[k][i] : 0.0f;
                sg += own ? d[k][i] * wr[k][i] : 0.0f;
                db[k][i] += own ? d[k][i] : 0.0f;
            }
        const int64_t next = row + (int64_t)gridDim.x * ROWS;
        if (next < rows) fetch(next);
        row_sums<TPR>(sum, sg, lds, turn);
        const float mean = sum / dim;
        sg /= dim;
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const bool own = i >= my.skip[k];
                n[k][i] -= mean;
                sq += own ? n[k][i] * n[k][i] : 0.0f;
                sgn += own ? d[k][i] * wr[k][i] * n[k][i] : 0.0f;
            }
        row_sums<TPR>(sq, sgn, lds, turn);
        const float rstd = 1.0f / sqrtf(sq / dim + eps);
        sgn *= rstd / dim;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            E out[R];
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const float m = n[k][i] * rstd;
                dw[k][i] += i >= my.skip[k] ? d[k][i] * m : 0.0f;
                out[i] = from_f<E>((d[k][i] * wr[k][i] - sg - m * sgn) * rstd +
                                   (FUSED && ds ? pr[k][i] : 0.0f));
            }
            if (my.skip[k] < R) store_run<E, R>(dx + row * dim + my.at[k], R, out);
        }
    }
    // the block's ROWS rows of sums into one
    __shared__ float acc[ROWS > 1 ? ROWS : 1][ROWS > 1 ? 2 * TPR * R : 1];
    float* pw = part + (int64_t)blockIdx.x * 2 * dim;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        if constexpr (ROWS > 1) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < R; ++i) {
                acc[sub][tid * R + i] = dw[k][i];
                acc[sub][TPR * R + tid * R + i] = db[k][i];
            }
            __syncthreads();
            if (sub == 0) {
#pragma unroll
                for (int i = 0; i < R; ++i)
                    for (int q = 1; q < ROWS; ++q) {
                        dw[k][i] += acc[q][tid * R + i];
                        db[k][i] += acc[q][TPR * R + tid * R + i];
                    }
            }
        }
        if (sub == 0)
#pragma unroll
            for (int i = 0; i < R; ++i)
                if (i >= my.skip[k]) {
                    pw[my.at[k] + i] = dw[k][i];
                    pw[dim + my.at[k] + i] = db[k][i];
                }
    }
}

// Rows too long for registers, by 1024 threads, or shorter than a run, by a wave:
// the row is read again for each sum over it.
template <typename E, int TPR>
__global__ void __launch_bounds__(TPR)
norm_fwd_long_kernel(const E* __restrict__ x, const E* __restrict__ res,
                     const E* __restrict__ w, const E* __restrict__ b,
                     E* __restrict__ y, E* __restrict__ s_out, int64_t rows, int dim,
                     float eps) {
    __shared__ float2 lds[2][16];
    int turn = 0;
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const E* xr = x + row * dim;
        const E* rr = res ? res + row * dim : nullptr;
        float sum = 0.0f;
        for (int c = threadIdx.x; c < dim; c += TPR) {
            const float v = to_f(xr[c]) + (rr ? to_f(rr[c]) : 0.0f);
            if (rr) s_out[row * dim + c] = from_f<E>(v);
            sum += v;
        }
        float sq = 0.0f, none = 0.0f;
        row_sums<TPR>(sum, none, lds, turn);
        const float mean = sum / dim;
        for (int c = threadIdx.x; c < dim; c += TPR) {
            const float d = to_f(xr[c]) + (rr ? to_f(rr[c]) : 0.0f) - mean;
            sq += d * d;
        }
        row_sums<TPR>(sq, none, lds, turn);
        const float rstd = 1.0f / sqrtf(sq / dim + eps);
        for (int c = threadIdx.x; c < dim; c += TPR) {
            const float v = to_f(xr[c]) + (rr ? to_f(rr[c]) : 0.0f);
            y[row * dim + c] = from_f<E>((v - mean) * rstd * to_f(w[c]) +
                                         (b ? to_f(b[c]) : 0.0f));
        }
    }
}

// The row's gradient, and its mean and rstd for the weight's, which is left to
// norm_dw_long_kernel.
template <typename E, int TPR>
__global__ void __launch_bounds__(TPR)
norm_bwd_long_kernel(const E* __restrict__ x, const E* __restrict__ res,
                     const E* __restrict__ w, float* __restrict__ stats, const E* __restrict__ dy,
                     const E* __restrict__ ds, E* __restrict__ dx, int64_t rows, int dim,
                     float eps) {
    __shared__ float2 lds[2][16];
    int turn = 0;
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const E *xr = x + row * dim, *rr = res ? res + row * dim : nullptr, *dr = dy + row * dim;
        float sum = 0.0f, sg = 0.0f, sq = 0.0f, sgn = 0.0f;
        for (int c = threadIdx.x; c < dim; c += TPR) {
            sum += to_f(xr[c]) + (rr ? to_f(rr[c]) : 0.0f);
            sg += to_f(dr[c]) * to_f(w[c]);
        }
        row_sums<TPR>(sum, sg, lds, turn);
        const float mean = sum / dim;
        sg /= dim;
        for (int c = threadIdx.x; c < dim; c += TPR) {
            const float n = to_f(xr[c]) + (rr ? to_f(rr[c]) : 0.0f) - mean;
            sq += n * n;
            sgn += to_f(dr[c]) * to_f(w[c]) * n;
        }
        row_sums<TPR>(sq, sgn, lds, turn);
        const float rstd = 1.0f / sqrtf(sq / dim + eps);
        sgn *= rstd / dim;
        if (threadIdx.x == 0) {
            stats[2 * row] = mean;
            stats[2 * row + 1] = rstd;
        }
        for (int c = threadIdx.x; c < dim; c += TPR) {
            const float g = to_f(dr[c]) * to_f(w[c]);
            const float n = (to_f(xr[c]) + (rr ? to_f(rr[c]) : 0.0f) - mean) * rstd;
            dx[row * dim + c] = from_f<E>((g - sg - n * sgn) * rstd +
                                          (ds ? to_f(ds[row * dim + c]) : 0.0f));
        }
    }
}

template <typename E>
__global__ void __launch_bounds__(256)
norm_dw_long_kernel(const E* __restrict__ x, const E* __restrict__ res,
                    const float* __restrict__ stats, const E* __restrict__ dy, float* __restrict__ part,
                    int64_t rows, int dim) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= dim) return;
    float dw = 0.0f, db = 0.0f;
    for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
        const float d = to_f(dy[row * dim + c]);
        const float v = to_f(x[row * dim + c]) + (res ? to_f(res[row * dim + c]) : 0.0f);
        dw += d * (v - stats[2 * row]) * stats[2 * row + 1];
        db += d;
    }
    part[((int64_t)blockIdx.y * 2) * dim + c] = dw;
    part[((int64_t)blockIdx.y * 2 + 1) * dim + c] = db;
}

template <typename E>
__global__ void __launch_bounds__(1024)
column_sum_kernel(const float* __restrict__ part, E* __restrict__ out, int rows, int cols) {
    sum_columns<E>(part, out, rows, cols, blockIdx.x);
}

// By the runs of a row, the smallest group of threads that holds it with two
// runs a thread: in bf16 more leave the registers of one wave a SIMD. 0 threads:
// longer than 8192 elements, or shorter than a run. 512 threads end there in bf16;
// fp32, whose runs are half as long, takes four of them to the same length. No
// shape of 1024 threads, which would go on to 16384, has been built.
struct Shape {
    int threads, runs;
};
template <typename E>
Shape shape_of(int dim) {
    const int runs = (dim + RUN<E> - 1) / RUN<E>;
    if (dim < RUN<E>) return {0, 0};
    if (runs <= 64) return {64, 1};
    for (int t : {64, 128, 256, 512})
        if (runs <= t * 2) return {t, 2};
    if (sizeof(E) == 4 && runs <= 512 * 4) return {512, 4};
    return {0, 0};
}

template <typename E, typename F>
void with_shape(int dim, bool fused, F&& f) {
    const Shape p = shape_of<E>(dim);
    const auto go = [&](auto t, auto n) {
        if (p.threads != t || p.runs != n) return;
        fused ? f(t, n, std::true_type()) : f(t, n, std::false_type());
    };
    go(std::integral_constant<int, 64>(), std::integral_constant<int, 1>());
    go(std::integral_constant<int, 64>(), std::integral_constant<int, 2>());
    go(std::integral_constant<int, 128>(), std::integral_constant<int, 2>());
    go(std::integral_constant<int, 256>(), std::integral_constant<int, 2>());
    go(std::integral_constant<int, 512>(), std::integral_constant<int, 2>());
    if constexpr (sizeof(E) == 4)
        go(std::integral_constant<int, 512>(), std::integral_constant<int, 4>());
}

template <typename E, typename F>
void with_long(int dim, F&& f) {
    if (dim < RUN<E>) f(std::integral_constant<int, 64>());
    else f(std::integral_constant<int, 1024>());
}
// A launch has less than 2^32 threads.
constexpr int64_t LONG_BLOCKS = 1 << 20;

// Blocks of a launch: enough to fill the card several times over, and few
// enough that each keeps its weights for several rows. Backward each one leaves a
// row of sums as well, which column_sum_kernel has to read.
constexpr int FWD_BLOCKS = 2048, BWD_BLOCKS = 512;

int blocks_of(int64_t rows, int threads, int64_t most) {
    const int each = block_of(threads) / threads;
    const int64_t need = (rows + each - 1) / each;
    return (int)(need < most ? need : most);
}

template <typename E>
int fwd(const void* x, const void* res, const void* w, const void* b, void* y,
        void* s, int64_t rows, int dim, float eps, hipStream_t st) {
    if (rows == 0) return 0;
    if (shape_of<E>(dim).threads == 0)
        with_long<E>(dim, [&](auto t) {
            constexpr int T = decltype(t)::value;
            norm_fwd_long_kernel<E, T><<<(int)std::min(rows, LONG_BLOCKS), T, 0, st>>>(
                (const E*)x, (const E*)res, (const E*)w, (const E*)b, (E*)y, (E*)s, rows, dim,
                eps);
        });
    else
        with_shape<E>(dim, res != nullptr, [&](auto t, auto n, auto fused) {
            constexpr int T = decltype(t)::value, N = decltype(n)::value;
            norm_fwd_kernel<E, T, N, decltype(fused)::value>
                <<<blocks_of(rows, T, FWD_BLOCKS), block_of(T), 0, st>>>(
                    (const E*)x, (const E*)res, (const E*)w, (const E*)b, (E*)y,
                    (E*)s, rows, dim, eps);
        });
    LSTM_CHECK_LAUNCH();
    return 0;
}

template <typename E>
int bwd(const void* x, const void* res, const void* w, const void* dy, const void* ds, void* dx,
        float* part, float* stats, void* dwb, int64_t rows, int dim, int parts, float eps, hipStream_t st) {
    if (rows == 0) {
        parts = 0;
    } else if (shape_of<E>(dim).threads == 0) {
        with_long<E>(dim, [&](auto t) {
            constexpr int T = decltype(t)::value;
            norm_bwd_long_kernel<E, T><<<(int)std::min(rows, LONG_BLOCKS), T, 0, st>>>(
                (const E*)x, (const E*)res, (const E*)w, stats, (const E*)dy, (const E*)ds,
                (E*)dx, rows, dim, eps);
        });
        LSTM_CHECK_LAUNCH();
        norm_dw_long_kernel<E><<<dim3((dim + 255) / 256, parts), 256, 0, st>>>(
            (const E*)x, (const E*)res, stats, (const E*)dy, part, rows, dim);
    } else {
        with_shape<E>(dim, res != nullptr, [&](auto t, auto n, auto fused) {
            constexpr int T = decltype(t)::value, N = decltype(n)::value;
            norm_bwd_kernel<E, T, N, decltype(fused)::value><<<parts, block_of(T), 0, st>>>(
                (const E*)x, (const E*)res, (const E*)w, (const E*)dy, (const E*)ds, (E*)dx, part,
                rows, dim, eps);
        });
    }
    LSTM_CHECK_LAUNCH();
    column_sum_kernel<E><<<column_blocks(2 * dim), 1024, 0, st>>>(part, (E*)dwb, parts, 2 * dim);
    LSTM_CHECK_LAUNCH();
    return 0;
}

}  // namespace

extern "C" int launch_norm_fwd(int is_bf16, const void* x, const void* res, const void* w,
                               const void* b, void* y, void* s, int64_t rows, int dim,
                               float eps, hipStream_t st) {
    return is_bf16 ? fwd<bf16>(x, res, w, b, y, s, rows, dim, eps, st)
                   : fwd<float>(x, res, w, b, y, s, rows, dim, eps, st);
}

// Rows of partial sums that launch_norm_bwd writes (`part` has 2 * dim floats
// for each), and floats of `stats`, which only the rows past registers need.
extern "C" int norm_bwd_parts(int is_bf16, int64_t rows, int dim) {
    const Shape p = is_bf16 ? shape_of<bf16>(dim) : shape_of<float>(dim);
    return blocks_of(rows, p.threads ? p.threads : 1024, BWD_BLOCKS);
}

extern "C" int64_t norm_bwd_stats(int is_bf16, int64_t rows, int dim) {
    const Shape p = is_bf16 ? shape_of<bf16>(dim) : shape_of<float>(dim);
    return p.threads ? 0 : 2 * rows;
}

extern "C" int launch_norm_bwd(int is_bf16, const void* x, const void* res, const void* w,
                               const void* dy, const void* ds, void* dx, float* part,
                               float* stats, void* dwb, int64_t rows, int dim, int parts,
                               float eps, hipStream_t st) {
    return is_bf16
        ? bwd<bf16>(x, res, w, dy, ds, dx, part, stats, dwb, rows, dim, parts, eps, st)
        : bwd<float>(x, res, w, dy, ds, dx, part, stats, dwb, rows, dim, parts, eps, st);
}
