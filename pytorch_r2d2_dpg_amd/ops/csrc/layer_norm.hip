// Layer norm over the last axis, forward and backward.
//
//   s = x + r;  n = (s - mean(s)) * rstd;  y = n w + b
//   g = dy w;   dx = rstd (g - mean(g) - n mean(g n)) + ds
//   dw = sum over rows of dy n;  db = sum over rows of dy
//
// Memory bound: about ten operations an element. A row lives in the registers
// of its threads between the sums over it, so each input is read once.

#include "gated_common.h"

namespace {

constexpr int BYTES = 16;  // one load of a lane

template <typename E> constexpr int RUN = BYTES / (int)sizeof(E);

// Sum over the TPR threads of a row; the same value in each of them.
template <int TPR>
DEV_INLINE float row_sum(float v, float* lds) {
    v = wave_sum(v);
    if constexpr (TPR > 64) {
        constexpr int W = TPR / 64;
        __syncthreads();  // the last sum's readers are done
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) v += lds[w];
    }
    return v;
}

// A row of `dim` elements over TPR threads, NV runs each: thread i holds the
// runs i, i + TPR, ... The mean comes off before squaring: the variance of a
// row far from zero does not cancel.
template <typename E, int TPR, int NV>
__global__ void __launch_bounds__(TPR > 256 ? TPR : 256)
norm_fwd_kernel(const E* __restrict__ x, const E* __restrict__ res,
                const E* __restrict__ w, const E* __restrict__ b,
                E* __restrict__ y, E* __restrict__ s_out,
                int64_t rows, int dim, float eps) {
    constexpr int R = RUN<E>;
    constexpr int ROWS = TPR > 256 ? 1 : 256 / TPR;
    __shared__ float lds[16];
    const int tid = threadIdx.x % TPR;
    const int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / TPR;
    if (row >= rows) return;  // TPR >= 256: a block is one row, none diverges
    const E* xr = x + row * dim;
    float v[NV][R];
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int c = (tid + k * TPR) * R, have = dim - c;
        E in[R];
        if (have > 0) {
            load_run<E, R>(xr + c, have, in);
#pragma unroll
            for (int i = 0; i < R; ++i) v[k][i] = to_f(in[i]);
            if (res) {
                load_run<E, R>(res + row * dim + c, have, in);
                E so[R];
#pragma unroll
                for (int i = 0; i < R; ++i) {
                    v[k][i] += to_f(in[i]);
                    so[i] = from_f<E>(v[k][i]);
                }
                store_run<E, R>(s_out + row * dim + c, have, so);
            }
        } else {
#pragma unroll
            for (int i = 0; i < R; ++i) v[k][i] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < R; ++i) sum += v[k][i];
    }
    const float mean = row_sum<TPR>(sum, lds) / dim;
    float sq = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const float d = v[k][i] - mean;
            if ((tid + k * TPR) * R + i < dim) sq += d * d;
        }
    const float rstd = 1.0f / sqrtf(row_sum<TPR>(sq, lds) / dim + eps);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int c = (tid + k * TPR) * R, have = dim - c;
        if (have <= 0) continue;
        E win[R], bin[R], out[R];
        load_run<E, R>(w + c, have, win);
        if (b) load_run<E, R>(b + c, have, bin);
#pragma unroll
        for (int i = 0; i < R; ++i)
            out[i] = from_f<E>((v[k][i] - mean) * rstd * to_f(win[i]) +
                               (b ? to_f(bin[i]) : 0.0f));
        store_run<E, R>(y + row * dim + c, have, out);
    }
}

// Rows blockIdx, blockIdx + gridDim, ... of ROWS each; a thread's columns stay
// the same from row to row, so the weight's gradient sums up in registers and
// leaves once a block, as a row of part [gridDim][2][dim].
//
// s is summed again from x and r, not read back as the forward pass rounded it:
// in bf16 that rounding alone would add half again to the error of dw. The mean
// and rstd come from the same registers. The sums join in two rounds: those of
// s and g, then those of (s - mean)^2 and g (s - mean).
template <typename E, int TPR, int NV>
__global__ void __launch_bounds__(TPR > 256 ? TPR : 256)
norm_bwd_kernel(const E* __restrict__ x, const E* __restrict__ res,
                const E* __restrict__ w, const E* __restrict__ dy,
                const E* __restrict__ ds, E* __restrict__ dx,
                float* __restrict__ part, int64_t rows, int dim, float eps) {
    constexpr int R = RUN<E>;
    constexpr int ROWS = TPR > 256 ? 1 : 256 / TPR;
    __shared__ float lds[16];
    const int tid = threadIdx.x % TPR, sub = threadIdx.x / TPR;
    float dw[NV][R] = {}, db[NV][R] = {};
    for (int64_t row = (int64_t)blockIdx.x * ROWS + sub; row < rows;
         row += (int64_t)gridDim.x * ROWS) {
        float n[NV][R], d[NV][R], g[NV][R];
        float sum = 0.0f, sg = 0.0f;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (tid + k * TPR) * R, have = dim - c;
            E xin[R], rin[R], din[R], win[R];
            if (have > 0) {
                load_run<E, R>(x + row * dim + c, have, xin);
                if (res) load_run<E, R>(res + row * dim + c, have, rin);
                load_run<E, R>(dy + row * dim + c, have, din);
                load_run<E, R>(w + c, have, win);
            }
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const bool real = i < have;
                n[k][i] = real ? to_f(xin[i]) + (res ? to_f(rin[i]) : 0.0f) : 0.0f;
                d[k][i] = real ? to_f(din[i]) : 0.0f;
                g[k][i] = real ? d[k][i] * to_f(win[i]) : 0.0f;
                sum += n[k][i];
                sg += g[k][i];
            }
        }
        const float mean = row_sum<TPR>(sum, lds) / dim;
        sg = row_sum<TPR>(sg, lds) / dim;
        float sq = 0.0f, sgn = 0.0f;
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int i = 0; i < R; ++i) {
                n[k][i] = (tid + k * TPR) * R + i < dim ? n[k][i] - mean : 0.0f;
                sq += n[k][i] * n[k][i];
                sgn += g[k][i] * n[k][i];
            }
        const float rstd = 1.0f / sqrtf(row_sum<TPR>(sq, lds) / dim + eps);
        sgn = row_sum<TPR>(sgn, lds) * rstd / dim;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (tid + k * TPR) * R, have = dim - c;
            if (have <= 0) continue;
            E out[R], pass[R];
            if (ds) load_run<E, R>(ds + row * dim + c, have, pass);
#pragma unroll
            for (int i = 0; i < R; ++i) {
                n[k][i] *= rstd;
                dw[k][i] += d[k][i] * n[k][i];
                db[k][i] += d[k][i];
                out[i] = from_f<E>((g[k][i] - sg - n[k][i] * sgn) * rstd +
                                   (ds ? to_f(pass[i]) : 0.0f));
            }
            store_run<E, R>(dx + row * dim + c, have, out);
        }
    }
    // the block's ROWS rows of sums into one
    __shared__ float acc[ROWS > 1 ? ROWS : 1][ROWS > 1 ? 2 * TPR * R : 1];
    float* pw = part + (int64_t)blockIdx.x * 2 * dim;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int c = (tid + k * TPR) * R, have = dim - c;
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
        if (sub == 0 && have > 0) {
            store_run<float, R>(pw + c, have, dw[k]);
            store_run<float, R>(pw + dim + c, have, db[k]);
        }
    }
}

// Rows too long for registers: the row is read again for each sum over it.
template <typename E>
__global__ void __launch_bounds__(1024)
norm_fwd_long_kernel(const E* __restrict__ x, const E* __restrict__ res,
                     const E* __restrict__ w, const E* __restrict__ b,
                     E* __restrict__ y, E* __restrict__ s_out, int dim, float eps) {
    __shared__ float lds[16];
    const int64_t row = blockIdx.x;
    const E* xr = x + row * dim;
    const E* rr = res ? res + row * dim : nullptr;
    float sum = 0.0f;
    for (int c = threadIdx.x; c < dim; c += 1024) {
        const float v = to_f(xr[c]) + (rr ? to_f(rr[c]) : 0.0f);
        if (rr) s_out[row * dim + c] = from_f<E>(v);
        sum += v;
    }
    const float mean = row_sum<1024>(sum, lds) / dim;
    float sq = 0.0f;
    for (int c = threadIdx.x; c < dim; c += 1024) {
        const float d = to_f(xr[c]) + (rr ? to_f(rr[c]) : 0.0f) - mean;
        sq += d * d;
    }
    const float rstd = 1.0f / sqrtf(row_sum<1024>(sq, lds) / dim + eps);
    for (int c = threadIdx.x; c < dim; c += 1024) {
        const float v = to_f(xr[c]) + (rr ? to_f(rr[c]) : 0.0f);
        y[row * dim + c] = from_f<E>((v - mean) * rstd * to_f(w[c]) +
                                     (b ? to_f(b[c]) : 0.0f));
    }
}

// The row's gradient, and its mean and rstd for the weight's, which is left to
// norm_dw_long_kernel.
template <typename E>
__global__ void __launch_bounds__(1024)
norm_bwd_long_kernel(const E* __restrict__ x, const E* __restrict__ res,
                     const E* __restrict__ w, float* __restrict__ stats, const E* __restrict__ dy,
                     const E* __restrict__ ds, E* __restrict__ dx, int dim, float eps) {
    __shared__ float lds[16];
    const int64_t row = blockIdx.x;
    const E *xr = x + row * dim, *rr = res ? res + row * dim : nullptr, *dr = dy + row * dim;
    float sum = 0.0f, sg = 0.0f, sq = 0.0f, sgn = 0.0f;
    for (int c = threadIdx.x; c < dim; c += 1024) {
        sum += to_f(xr[c]) + (rr ? to_f(rr[c]) : 0.0f);
        sg += to_f(dr[c]) * to_f(w[c]);
    }
    const float mean = row_sum<1024>(sum, lds) / dim;
    sg = row_sum<1024>(sg, lds) / dim;
    for (int c = threadIdx.x; c < dim; c += 1024) {
        const float n = to_f(xr[c]) + (rr ? to_f(rr[c]) : 0.0f) - mean;
        sq += n * n;
        sgn += to_f(dr[c]) * to_f(w[c]) * n;
    }
    const float rstd = 1.0f / sqrtf(row_sum<1024>(sq, lds) / dim + eps);
    sgn = row_sum<1024>(sgn, lds) * rstd / dim;
    if (threadIdx.x == 0) {
        stats[2 * row] = mean;
        stats[2 * row + 1] = rstd;
    }
    for (int c = threadIdx.x; c < dim; c += 1024) {
        const float g = to_f(dr[c]) * to_f(w[c]);
        const float n = (to_f(xr[c]) + (rr ? to_f(rr[c]) : 0.0f) - mean) * rstd;
        dx[row * dim + c] = from_f<E>((g - sg - n * sgn) * rstd +
                                      (ds ? to_f(ds[row * dim + c]) : 0.0f));
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

// Runs of a row, and by them the smallest group of threads that holds it: a
// wave up to 4 runs a lane, then 256 and 1024 threads. 0: too long.
struct Shape {
    int threads, runs;
};
template <typename E>
Shape shape_of(int dim) {
    const int runs = (dim + RUN<E> - 1) / RUN<E>;
    for (int t : {64, 256, 1024})
        for (int nv : {1, 2, 4})
            if (runs <= t * nv) return {t, nv};
    return {0, 0};
}

template <typename E, typename F>
void with_shape(int dim, F&& f) {
    const Shape p = shape_of<E>(dim);
#define CASE(T, N) \
    if (p.threads == T && p.runs == N) \
    return f(std::integral_constant<int, T>(), std::integral_constant<int, N>())
    CASE(64, 1); CASE(64, 2); CASE(64, 4);
    CASE(256, 2); CASE(256, 4);
    CASE(1024, 2); CASE(1024, 4);
#undef CASE
}

template <typename E>
int fwd(const void* x, const void* res, const void* w, const void* b, void* y,
        void* s, int64_t rows, int dim, float eps, hipStream_t st) {
    if (rows == 0) return 0;
    if (shape_of<E>(dim).threads == 0)
        norm_fwd_long_kernel<E><<<dim3((unsigned)rows), 1024, 0, st>>>(
            (const E*)x, (const E*)res, (const E*)w, (const E*)b, (E*)y, (E*)s,
            dim, eps);
    else
        with_shape<E>(dim, [&](auto t, auto n) {
            constexpr int T = decltype(t)::value, N = decltype(n)::value;
            constexpr int ROWS = T > 256 ? 1 : 256 / T;
            norm_fwd_kernel<E, T, N>
                <<<dim3((unsigned)((rows + ROWS - 1) / ROWS)), T > 256 ? T : 256, 0, st>>>(
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
        norm_bwd_long_kernel<E><<<dim3((unsigned)rows), 1024, 0, st>>>(
            (const E*)x, (const E*)res, (const E*)w, stats, (const E*)dy, (const E*)ds, (E*)dx, dim,
            eps);
        LSTM_CHECK_LAUNCH();
        norm_dw_long_kernel<E><<<dim3((dim + 255) / 256, parts), 256, 0, st>>>(
            (const E*)x, (const E*)res, stats, (const E*)dy, part, rows, dim);
    } else {
        with_shape<E>(dim, [&](auto t, auto n) {
            constexpr int T = decltype(t)::value, N = decltype(n)::value;
            norm_bwd_kernel<E, T, N><<<parts, T > 256 ? T : 256, 0, st>>>(
                (const E*)x, (const E*)res, (const E*)w, (const E*)dy, (const E*)ds, (E*)dx, part,
                rows, dim, eps);
        });
    }
    LSTM_CHECK_LAUNCH();
    column_sum_kernel<E><<<(2 * dim + 63) / 64, 1024, 0, st>>>(part, (E*)dwb, parts, 2 * dim);
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
    const int64_t groups = p.threads == 64 ? (rows + 3) / 4 : rows;
    return (int)(groups < 512 ? groups : 512);
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
