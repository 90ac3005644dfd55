// Gated linear recurrence over time, forward and backward.
//
//   gates [T, B, 3H] = (f, v, o);   a = sigma(f)
//   h_t = a_t h_{t-1} + (1 - a_t) v_t;   y_t = h_t silu(o_t)
//   G_t = dy_t silu(o_t) + a_{t+1} G_{t+1}   (G past the end: dhT)
//   df = G (h_{t-1} - v) a (1 - a);  dv = G (1 - a);  do = dy h silu'(o);  dh0 = a_1 G_1
//
// Each step is an affine map of the state, so runs of steps compose: a wave
// holds CHUNK steps of its channels in registers and reduces them to one map
// (A, H): h -> A h + H. The block's waves, which hold consecutive chunks, apply
// each other's maps through LDS and then walk their own steps with the state
// that they start from: every input is read once and time runs in parallel.
// Where the channels are too few to fill the card, time is split over blocks
// as well: one launch reduces each segment to its map, and the next walks.
//
// The forward pass keeps the state that each chunk starts from, in 32 bits,
// 1/CHUNK of the steps: the backward pass walks the chunk again from it in
// place of reading every state back.
//
// Steps at or past a sequence's length are the identity map with y = 0: the
// state passes through whatever their gates hold.

#include "gated_common.h"

namespace {

constexpr int CHUNK = 16;  // steps of a wave, and between two kept states
constexpr int MAX_WAVES = 8;

template <typename E>
struct Args {
    const E* gates;    // [T, B, 3H]
    const float* h0;   // [B, H] or null: zeros
    const int* lengths;  // [B] or null: all T
    E* y;              // [T, B, H]
    float* hT;         // [B, H]
    float* kept;       // [chunks, B, H] or null
    const E* dy;       // [T, B, H]
    const float* dhT;  // [B, H] or null: zeros
    E* dgates;         // [T, B, 3H]
    float* dh0;        // [B, H]
    float2* maps;      // [segments, B, H]: (A, H) of a segment
    int T, B, H, segments, passes;  // a segment is `passes` times the block's waves chunks long
};

// A lane's channels: the pair (c, c + 1) of a row b; the last of an odd H alone.
struct Lane {
    int b, c, n, len;  // n: 0 past the end, else 1 or 2
};

template <typename E>
DEV_INLINE Lane lane_of(const Args<E>& p) {
    const int pairs = (p.H + 1) / 2;
    const int64_t u = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63);
    Lane q{0, 0, 0, 0};
    if (u < (int64_t)pairs * p.B) {
        q.b = (int)(u / pairs);
        q.c = 2 * (int)(u - (int64_t)q.b * pairs);
        q.n = q.c + 1 < p.H ? 2 : 1;
        q.len = p.T;
        if (p.lengths) {
            const int len = p.lengths[q.b];
            q.len = len < 0 ? 0 : len > p.T ? p.T : len;
        }
    }
    return q;
}

template <typename E>
DEV_INLINE void load2(const E* p, int n, E (&out)[2]) {
    load_run<E, 2>(p, n, out);
}

DEV_INLINE void load_state(const float* p, const Lane& q, int H, float (&h)[2]) {
    h[0] = h[1] = 0.0f;
    if (p && q.n) load_run<float, 2>(p + (int64_t)q.b * H + q.c, q.n, h);
}

DEV_INLINE void store_state(float* p, const Lane& q, int H, const float (&h)[2]) {
    if (q.n) store_run<float, 2>(p + (int64_t)q.b * H + q.c, q.n, h);
}

// The waves' maps meet in LDS. `carry` is the state before the block's first
// wave on entry and after its last one on return; `mine` is what this wave
// starts from. BACK: the order of the waves is reversed.
template <bool BACK>
DEV_INLINE void join_waves(float2 (*slots)[MAX_WAVES][64][2], int& turn, int wave, int waves,
                           const float (&A)[2], const float (&Hl)[2],
                           float (&carry)[2], float (&mine)[2]) {
    const int lane = threadIdx.x & 63;
    auto& slot = slots[turn];  // two in turn: one barrier a pass
    turn ^= 1;
#pragma unroll
    for (int i = 0; i < 2; ++i) slot[wave][lane][i] = make_float2(A[i], Hl[i]);
    __syncthreads();
    for (int k = 0; k < waves; ++k) {
        const int w = BACK ? waves - 1 - k : k;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (w == wave) mine[i] = carry[i];
            const float2 m = slot[w][lane][i];
            carry[i] = m.x * carry[i] + m.y;
        }
    }
}

// The state that a segment starts from: the maps before it, in order.
template <bool BACK, typename E>
DEV_INLINE void join_segments(const Args<E>& p, const Lane& q, int seg, float (&carry)[2]) {
    if (!q.n) return;
    const int64_t n = (int64_t)p.B * p.H, at = (int64_t)q.b * p.H + q.c;
    if (BACK) {
        for (int s = p.segments - 1; s > seg; --s)
            for (int i = 0; i < q.n; ++i) {
                const float2 m = p.maps[s * n + at + i];
                carry[i] = m.x * carry[i] + m.y;
            }
    } else {
        for (int s = 0; s < seg; ++s)
            for (int i = 0; i < q.n; ++i) {
                const float2 m = p.maps[s * n + at + i];
                carry[i] = m.x * carry[i] + m.y;
            }
    }
}

// ONLY_MAP: leave the segment's map and write nothing else.
template <typename E, bool ONLY_MAP>
__global__ void __launch_bounds__(64 * MAX_WAVES)
recurrence_fwd_kernel(Args<E> p) {
    __shared__ float2 slots[2][MAX_WAVES][64][2];
    const int wave = threadIdx.x >> 6, waves = blockDim.x >> 6, seg = blockIdx.y;
    const Lane q = lane_of(p);
    const int64_t step = (int64_t)p.B * p.H;
    const int64_t at = (int64_t)q.b * p.H + q.c;
    float carry[2] = {0.0f, 0.0f}, total[2] = {1.0f, 1.0f};
    if (!ONLY_MAP) {
        load_state(p.h0, q, p.H, carry);
        join_segments<false>(p, q, seg, carry);
    }
    int turn = 0;
    for (int pass = 0; pass < p.passes; ++pass) {
        const int chunk = (seg * p.passes + pass) * waves + wave;
        const int t0 = chunk * CHUNK;
        float a[CHUNK][2], b[CHUNK][2];
        E o[CHUNK][2];
#pragma unroll
        for (int k = 0; k < CHUNK; ++k) {
            const int t = t0 + k;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                a[k][i] = 1.0f;
                b[k][i] = 0.0f;
                o[k][i] = from_f<E>(0.0f);
            }
            if (t < q.len) {  // len is 0 for a lane past the end
                const E* g = p.gates + 3 * (int64_t)t * step + 3 * (int64_t)q.b * p.H + q.c;
                E f[2], v[2];
                load2(g, q.n, f);
                load2(g + p.H, q.n, v);
                if (!ONLY_MAP) load2(g + 2 * (int64_t)p.H, q.n, o[k]);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float keep;
                    sigmoid_pair(to_f(f[i]), a[k][i], keep);
                    b[k][i] = keep * to_f(v[i]);
                }
            }
        }
        float A[2] = {1.0f, 1.0f}, Hl[2] = {0.0f, 0.0f}, h[2];
#pragma unroll
        for (int k = 0; k < CHUNK; ++k)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                Hl[i] = a[k][i] * Hl[i] + b[k][i];
                A[i] *= a[k][i];
            }
        if (waves > 1) {
            join_waves<false>(slots, turn, wave, waves, A, Hl, carry, h);
            if (ONLY_MAP)  // the product of the A stands in the same slots
                for (int w = 0; w < waves; ++w)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        total[i] *= slots[turn ^ 1][w][threadIdx.x & 63][i].x;
        } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                h[i] = carry[i];
                carry[i] = A[i] * carry[i] + Hl[i];
                total[i] *= A[i];
            }
        }
        if (ONLY_MAP) continue;
        if (p.kept && t0 < p.T && q.n)
            store_run<float, 2>(p.kept + chunk * step + at, q.n, h);
#pragma unroll
        for (int k = 0; k < CHUNK; ++k) {
            const int t = t0 + k;
            if (t >= p.T) break;
            E out[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                h[i] = a[k][i] * h[i] + b[k][i];
                float val, grad;
                silu_grad(to_f(o[k][i]), val, grad);
                out[i] = from_f<E>(t < q.len ? h[i] * val : 0.0f);
            }
            if (q.n) store_run<E, 2>(p.y + t * step + at, q.n, out);
        }
    }
    if (ONLY_MAP) {
        if (wave == 0)
            for (int i = 0; i < q.n; ++i)
                p.maps[seg * step + at + i] = make_float2(total[i], carry[i]);
    } else if (wave == 0 && seg == p.segments - 1) {
        store_state(p.hT, q, p.H, carry);
    }
}

// R_t = a_t G_t is what step t hands to step t - 1, and the map of a step is
// R -> a (R + p) with p = dy silu(o).
template <typename E, bool ONLY_MAP>
__global__ void __launch_bounds__(64 * MAX_WAVES)
recurrence_bwd_kernel(Args<E> p) {
    __shared__ float2 slots[2][MAX_WAVES][64][2];
    const int wave = threadIdx.x >> 6, waves = blockDim.x >> 6, seg = blockIdx.y;
    const Lane q = lane_of(p);
    const int64_t step = (int64_t)p.B * p.H;
    const int64_t at = (int64_t)q.b * p.H + q.c;
    float carry[2] = {0.0f, 0.0f}, total[2] = {1.0f, 1.0f};
    if (!ONLY_MAP) {
        load_state(p.dhT, q, p.H, carry);
        join_segments<true>(p, q, seg, carry);
    }
    int turn = 0;
    for (int pass = p.passes - 1; pass >= 0; --pass) {
        const int chunk = (seg * p.passes + pass) * waves + wave;
        const int t0 = chunk * CHUNK;
        // Of a and 1 - a the smaller is held, with the sign saying which: the
        // other follows without cancelling, in half the registers.
        float m[CHUNK][2], before[CHUNK][2], g[CHUNK][2];
        E v[CHUNK][2];
        float h[2] = {0.0f, 0.0f};
        if (!ONLY_MAP && t0 < p.T && q.n) load_run<float, 2>(p.kept + chunk * step + at, q.n, h);
#pragma unroll
        for (int k = 0; k < CHUNK; ++k) {
            const int t = t0 + k;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                m[k][i] = -0.0f;  // a = 1
                g[k][i] = 0.0f;
                before[k][i] = 0.0f;
                v[k][i] = from_f<E>(0.0f);
            }
            E dout[2] = {from_f<E>(0.0f), from_f<E>(0.0f)};
            const int64_t gate = 3 * (int64_t)t * step + 3 * (int64_t)q.b * p.H + q.c;
            if (t < q.len) {
                const E* gp = p.gates + gate;
                E f[2], o[2], dy[2];
                load2(gp, q.n, f);
                if (!ONLY_MAP) load2(gp + p.H, q.n, v[k]);
                load2(gp + 2 * (int64_t)p.H, q.n, o);
                load2(p.dy + t * step + at, q.n, dy);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float a, keep, val, grad;
                    sigmoid_pair(to_f(f[i]), a, keep);
                    silu_grad(to_f(o[i]), val, grad);
                    m[k][i] = a <= keep ? a : -keep;
                    g[k][i] = to_f(dy[i]) * val;
                    if (!ONLY_MAP) {
                        before[k][i] = h[i];
                        h[i] = a * h[i] + keep * to_f(v[k][i]);
                        dout[i] = from_f<E>(to_f(dy[i]) * h[i] * grad);
                    }
                }
            }
            if (!ONLY_MAP && t < p.T && q.n)
                store_run<E, 2>(p.dgates + gate + 2 * (int64_t)p.H, q.n, dout);
        }
        float A[2] = {1.0f, 1.0f}, Rl[2] = {0.0f, 0.0f}, R[2];
#pragma unroll
        for (int k = CHUNK - 1; k >= 0; --k)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float a = __builtin_signbit(m[k][i]) ? 1.0f + m[k][i] : m[k][i];
                Rl[i] = a * (Rl[i] + g[k][i]);
                A[i] *= a;
            }
        if (waves > 1) {
            join_waves<true>(slots, turn, wave, waves, A, Rl, carry, R);
            if (ONLY_MAP)
                for (int w = 0; w < waves; ++w)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        total[i] *= slots[turn ^ 1][w][threadIdx.x & 63][i].x;
        } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                R[i] = carry[i];
                carry[i] = A[i] * carry[i] + Rl[i];
                total[i] *= A[i];
            }
        }
        if (ONLY_MAP) continue;
#pragma unroll
        for (int k = CHUNK - 1; k >= 0; --k) {
            const int t = t0 + k;
            if (t >= p.T) continue;
            E df[2], dv[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const bool neg = __builtin_signbit(m[k][i]);
                const float a = neg ? 1.0f + m[k][i] : m[k][i];
                const float keep = neg ? -m[k][i] : 1.0f - m[k][i];
                const float G = R[i] + g[k][i];
                R[i] = a * G;
                const bool real = t < q.len;
                df[i] = from_f<E>(real ? R[i] * keep * (before[k][i] - to_f(v[k][i])) : 0.0f);
                dv[i] = from_f<E>(real ? G * keep : 0.0f);
            }
            if (q.n) {
                E* gp = p.dgates + 3 * (int64_t)t * step + 3 * (int64_t)q.b * p.H + q.c;
                store_run<E, 2>(gp, q.n, df);
                store_run<E, 2>(gp + p.H, q.n, dv);
            }
        }
    }
    if (ONLY_MAP) {
        if (wave == 0)
            for (int i = 0; i < q.n; ++i)
                p.maps[seg * step + at + i] = make_float2(total[i], carry[i]);
    } else if (wave == 0 && seg == 0) {
        store_state(p.dh0, q, p.H, carry);
    }
}

// How time is laid over waves and blocks. A block takes up to MAX_WAVES chunks
// of its 64 lanes' channels at a time; where that leaves the card's 1024 SIMDs
// without a wave each, the chunks are dealt out to `segments` blocks.
struct Plan {
    int waves, segments, passes;
};

Plan plan_of(int T, int B, int H) {
    const int chunks = T > 0 ? (T + CHUNK - 1) / CHUNK : 1;
    const int64_t tiles = ((int64_t)B * ((H + 1) / 2) + 63) / 64;
    int passes = (chunks + MAX_WAVES - 1) / MAX_WAVES;
    const int waves = (chunks + passes - 1) / passes;
    int segments = 1;
    if (passes > 1 && tiles * waves < 1024) {
        const int64_t want = (1024 + tiles * waves - 1) / (tiles * waves);
        segments = (int)(want < passes ? want : passes);
        passes = (passes + segments - 1) / segments;
        segments = ((chunks + waves - 1) / waves + passes - 1) / passes;
    }
    return {waves, segments, passes};
}

template <typename E>
int run(Args<E> p, bool back, hipStream_t st) {
    if ((int64_t)p.B * p.H == 0) return 0;
    const Plan plan = plan_of(p.T, p.B, p.H);
    p.segments = plan.segments;
    p.passes = plan.passes;
    const int64_t tiles = ((int64_t)p.B * ((p.H + 1) / 2) + 63) / 64;
    const dim3 grid((unsigned)tiles, plan.segments), block(64 * plan.waves);
    if (plan.segments > 1) {
        if (!p.maps) return -1;
        if (back) recurrence_bwd_kernel<E, true><<<grid, block, 0, st>>>(p);
        else recurrence_fwd_kernel<E, true><<<grid, block, 0, st>>>(p);
        LSTM_CHECK_LAUNCH();
    }
    if (back) recurrence_bwd_kernel<E, false><<<grid, block, 0, st>>>(p);
    else recurrence_fwd_kernel<E, false><<<grid, block, 0, st>>>(p);
    LSTM_CHECK_LAUNCH();
    return 0;
}

template <typename E>
int fwd(const void* gates, const float* h0, const int* lengths, void* y, float* hT, float* kept,
        float* maps, int T, int B, int H, hipStream_t st) {
    Args<E> p{};
    p.gates = (const E*)gates; p.h0 = h0; p.lengths = lengths; p.y = (E*)y; p.hT = hT;
    p.kept = kept; p.maps = (float2*)maps; p.T = T; p.B = B; p.H = H;
    return run<E>(p, false, st);
}

template <typename E>
int bwd(const void* gates, const float* kept, const int* lengths, const void* dy,
        const float* dhT, void* dgates, float* dh0, float* maps, int T, int B, int H,
        hipStream_t st) {
    Args<E> p{};
    p.gates = (const E*)gates; p.kept = const_cast<float*>(kept); p.lengths = lengths;
    p.dy = (const E*)dy; p.dhT = dhT; p.dgates = (E*)dgates; p.dh0 = dh0;
    p.maps = (float2*)maps; p.T = T; p.B = B; p.H = H;
    return run<E>(p, true, st);
}

}  // namespace

// Steps between two kept states, and floats of workspace for the segments' maps.
extern "C" int recurrence_chunk() { return CHUNK; }
extern "C" int64_t recurrence_maps(int T, int B, int H) {
    const Plan p = plan_of(T, B, H);
    return p.segments > 1 ? (int64_t)p.segments * B * H * 2 : 0;
}

extern "C" int launch_recurrence_fwd(int is_bf16, const void* gates, const float* h0,
                                     const int* lengths, void* y, float* hT, float* kept,
                                     float* maps, int T, int B, int H, hipStream_t st) {
    return is_bf16 ? fwd<bf16>(gates, h0, lengths, y, hT, kept, maps, T, B, H, st)
                   : fwd<float>(gates, h0, lengths, y, hT, kept, maps, T, B, H, st);
}

extern "C" int launch_recurrence_bwd(int is_bf16, const void* gates, const float* kept,
                                     const int* lengths, const void* dy, const float* dhT,
                                     void* dgates, float* dh0, float* maps, int T, int B, int H,
                                     hipStream_t st) {
    return is_bf16 ? bwd<bf16>(gates, kept, lengths, dy, dhT, dgates, dh0, maps, T, B, H, st)
                   : bwd<float>(gates, kept, lengths, dy, dhT, dgates, dh0, maps, T, B, H, st);
}
