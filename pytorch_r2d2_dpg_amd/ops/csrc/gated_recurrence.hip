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
// Bound by memory: 80 steps of 256 rows of 512 in bf16 take 20 us forward and
// 30 us backward on the MI355X, 4.5 and 5.1 TB/s, where a copy of 2 GiB reaches
// 4.9. Where the channels are too few to fill the card, time is split over blocks
// as well: one launch reduces each segment to its map, and the next walks. The
// gates are read twice then: 16384 steps of 4 rows take 40 + 57 and 49 + 95 us.
// Blocks that wait for the maps of the segments before theirs, and join them in
// their fixed order, could read them once; that is not done.
//
// The forward pass keeps the state that each chunk starts from, in 32 bits,
// 1/CHUNK of the steps: the backward pass walks the chunk again from it in
// place of reading every state back.
//
// Steps at or past a sequence's length are the identity map with y = 0: the
// state passes through whatever their gates hold.

#include "gated_common.h"

namespace {

constexpr int CHUNK = 8;  // steps of a wave, and between two kept states
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
// A lane past the end has n = 0 and reads what the last one does.
struct Lane {
    int b, c, n, len;
};

template <typename E>
DEV_INLINE Lane lane_of(const Args<E>& p) {
    const int pairs = (p.H + 1) / 2;
    const int64_t units = (int64_t)pairs * p.B;
    int64_t u = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63);
    const bool in = u < units;
    if (!in) u = units - 1;
    Lane q;
    q.b = (int)(u / pairs);
    q.c = 2 * (int)(u - (int64_t)q.b * pairs);
    q.n = !in ? 0 : q.c + 1 < p.H ? 2 : 1;
    q.len = p.T;
    if (p.lengths) {
        const int len = p.lengths[q.b];
        q.len = len < 0 ? 0 : len > p.T ? p.T : len;
    }
    return q;
}

// A wave's pointer, kept in scalar registers: left to itself the compiler adds
// the lane's place to it once and then walks 64-bit addresses in every lane.
template <typename T>
using Global = __attribute__((address_space(1))) T*;
template <typename T>
DEV_INLINE Global<T> place(Global<char> p, unsigned bytes) {
#ifdef __HIP_DEVICE_COMPILE__
    asm volatile("" : "+s"(p), "+v"(bytes));
#endif
    return (Global<T>)(p + bytes);
}

// The bits of an element, and of two of them at any element's address.
template <typename E> struct Bits;
template <> struct Bits<bf16> {
    typedef unsigned short One;
    typedef unsigned Pair __attribute__((aligned(2)));
};
template <> struct Bits<float> {
    typedef unsigned One;
    typedef unsigned long long Pair __attribute__((aligned(4)));
};

// Two elements of a step: `p` is the same for the whole wave, `at` the lane's
// place in a step, which has less than 2^30 elements: its bytes stay in 32 bits.
// Without a branch, which would keep the loads behind it waiting: `second` is 0
// where a lane has one channel.
template <bool EVEN, typename E>
DEV_INLINE Two<E> load2(const E* p, unsigned at, unsigned second) {
    using B = Bits<E>;
    const Global<char> c = (Global<char>)p;
    typename B::Pair v;
    if constexpr (EVEN) {
        v = *place<const typename B::Pair>(c, at * (unsigned)sizeof(E));
    } else {
        const typename B::One lo = *place<const typename B::One>(c, at * (unsigned)sizeof(E));
        const typename B::One hi =
            *place<const typename B::One>(c, (at + second) * (unsigned)sizeof(E));
        v = lo | (typename B::Pair)hi << 8 * sizeof(E);
    }
    return __builtin_bit_cast(Two<E>, v);
}

template <bool EVEN, typename E>
DEV_INLINE void store2(E* p, unsigned at, int n, float a, float b) {
    using B = Bits<E>;
    const auto v = __builtin_bit_cast(typename B::Pair, Two<E>::of(a, b));
    const Global<char> c = (Global<char>)p;
    if constexpr (EVEN) {
        if (n) *place<typename B::Pair>(c, at * (unsigned)sizeof(E)) = v;
    } else {
        if (n) *place<typename B::One>(c, at * (unsigned)sizeof(E)) = (typename B::One)v;
        if (n > 1)
            *place<typename B::One>(c, (at + 1) * (unsigned)sizeof(E)) =
                (typename B::One)(v >> 8 * sizeof(E));
    }
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

// The state that a segment starts from: the maps before it, in order. The
// block's waves compose an equal share of them each, and join those.
template <bool BACK, typename E>
DEV_INLINE void join_segments(const Args<E>& p, float2 (*slots)[MAX_WAVES][64][2], int& turn,
                              int wave, int waves, unsigned at, unsigned second, int seg,
                              float (&carry)[2]) {
    const int64_t n = (int64_t)p.B * p.H;
    const int count = BACK ? p.segments - 1 - seg : seg;  // the same for the whole block
    if (count == 0) return;
    const int share = (count + waves - 1) / waves;
    const int rank = BACK ? waves - 1 - wave : wave;  // waves join from the last one on
    const int lo = rank * share, hi = lo + share < count ? lo + share : count;
    float A[2] = {1.0f, 1.0f}, Hl[2] = {0.0f, 0.0f}, mine[2];
    for (int s0 = lo; s0 < hi; s0 += 8) {
        float2 m[8][2];
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (s0 + k < hi) {
                const int s = BACK ? p.segments - 1 - (s0 + k) : s0 + k;
                m[k][0] = p.maps[s * n + at];
                m[k][1] = p.maps[s * n + at + second];
            }
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (s0 + k < hi)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    A[i] *= m[k][i].x;
                    Hl[i] = m[k][i].x * Hl[i] + m[k][i].y;
                }
    }
    join_waves<BACK>(slots, turn, wave, waves, A, Hl, carry, mine);
}

// ONLY_MAP: leave the segment's map and write nothing else.
template <typename E, bool EVEN, bool ONLY_MAP>
__global__ void __launch_bounds__(64 * MAX_WAVES)
recurrence_fwd_kernel(Args<E> p) {
    __shared__ float2 slots[2][MAX_WAVES][64][2];
    // the wave's own, in scalar registers: its steps, their addresses and branches
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int waves = blockDim.x >> 6, seg = blockIdx.y;
    const Lane q = lane_of(p);
    const unsigned second = q.c + 1 < p.H;
    const int64_t step = (int64_t)p.B * p.H;
    const unsigned at = (unsigned)q.b * p.H + q.c, gate_at = 3u * q.b * p.H + q.c;
    float carry[2] = {0.0f, 0.0f}, total[2] = {1.0f, 1.0f};
    int turn = 0;
    if (!ONLY_MAP) {
        if (p.h0) {
            const Two<float> s = load2<EVEN>(p.h0, at, second);
            carry[0] = s[0];
            carry[1] = s[1];
        }
        join_segments<false>(p, slots, turn, wave, waves, at, second, seg, carry);
    }
    // A chunk's loads go out together (the branches are the wave's, not a lane's),
    // and before the chunk in front of it is joined and written.
    Two<E> f[CHUNK], v[CHUNK], o[CHUNK];
    const auto fetch = [&](int chunk) {
        const int t0 = chunk * CHUNK;
        const E* g = p.gates + t0 * step * 3;
#pragma unroll
        for (int k = 0; k < CHUNK; ++k, g += 3 * step)
            if (t0 + k < p.T) {
                f[k] = load2<EVEN>(g, gate_at, second);
                v[k] = load2<EVEN>(g + p.H, gate_at, second);
                if (!ONLY_MAP) o[k] = load2<EVEN>(g + 2 * (int64_t)p.H, gate_at, second);
            }
    };
    if (p.passes) fetch(seg * p.passes * waves + wave);
    for (int pass = 0; pass < p.passes; ++pass) {
        const int chunk = (seg * p.passes + pass) * waves + wave;
        const int t0 = chunk * CHUNK;
        float a[CHUNK][2], b[CHUNK][2], silu[CHUNK][2];
        float A[2] = {1.0f, 1.0f}, Hl[2] = {0.0f, 0.0f}, h[2];
#pragma unroll
        for (int k = 0; k < CHUNK; ++k)
            if (t0 + k < p.T) {
                const bool real = t0 + k < q.len;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float pos, neg, grad;
                    sigmoid_pair(f[k][i], pos, neg);
                    a[k][i] = real ? pos : 1.0f;
                    b[k][i] = real ? neg * v[k][i] : 0.0f;
                    if (!ONLY_MAP) silu_grad(o[k][i], silu[k][i], grad);
                    Hl[i] = a[k][i] * Hl[i] + b[k][i];
                    A[i] *= a[k][i];
                }
            }
        if (pass + 1 < p.passes) fetch(chunk + waves);
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
        if (p.kept && t0 < p.T) store2<EVEN>(p.kept + chunk * step, at, q.n, h[0], h[1]);
        E* to = p.y + t0 * step;
#pragma unroll
        for (int k = 0; k < CHUNK; ++k, to += step)
            if (t0 + k < p.T) {
                const bool real = t0 + k < q.len;
                float out[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    h[i] = a[k][i] * h[i] + b[k][i];
                    out[i] = real ? h[i] * silu[k][i] : 0.0f;
                }
                store2<EVEN>(to, at, q.n, out[0], out[1]);
            }
    }
    if (wave != 0) return;
    if (ONLY_MAP) {
        for (int i = 0; i < q.n; ++i)
            p.maps[seg * step + at + i] = make_float2(total[i], carry[i]);
    } else if (seg == p.segments - 1) {
        store2<EVEN>(p.hT, at, q.n, carry[0], carry[1]);
    }
}

// R_t = a_t G_t is what step t hands to step t - 1, and the map of a step is
// R -> a (R + p) with p = dy silu(o).
template <typename E, bool EVEN, bool ONLY_MAP>
__global__ void __launch_bounds__(64 * MAX_WAVES)
recurrence_bwd_kernel(Args<E> p) {
    __shared__ float2 slots[2][MAX_WAVES][64][2];
    // the wave's own, in scalar registers: its steps, their addresses and branches
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int waves = blockDim.x >> 6, seg = blockIdx.y;
    const Lane q = lane_of(p);
    const unsigned second = q.c + 1 < p.H;
    const int64_t step = (int64_t)p.B * p.H;
    const unsigned at = (unsigned)q.b * p.H + q.c, gate_at = 3u * q.b * p.H + q.c;
    float carry[2] = {0.0f, 0.0f}, total[2] = {1.0f, 1.0f};
    int turn = 0;
    if (!ONLY_MAP) {
        if (p.dhT) {
            const Two<float> s = load2<EVEN>(p.dhT, at, second);
            carry[0] = s[0];
            carry[1] = s[1];
        }
        join_segments<true>(p, slots, turn, wave, waves, at, second, seg, carry);
    }
    Two<E> f[CHUNK], v[CHUNK], o[CHUNK], dy[CHUNK];
    Two<float> kept{};
    const auto fetch = [&](int chunk) {
        const int t0 = chunk * CHUNK;
        if (!ONLY_MAP && t0 < p.T) kept = load2<EVEN>(p.kept + chunk * step, at, second);
        const E *g = p.gates + t0 * step * 3, *d = p.dy + t0 * step;
#pragma unroll
        for (int k = 0; k < CHUNK; ++k, g += 3 * step, d += step)
            if (t0 + k < p.T) {
                f[k] = load2<EVEN>(g, gate_at, second);
                if (!ONLY_MAP) v[k] = load2<EVEN>(g + p.H, gate_at, second);
                o[k] = load2<EVEN>(g + 2 * (int64_t)p.H, gate_at, second);
                dy[k] = load2<EVEN>(d, at, second);
            }
    };
    if (p.passes) fetch(((seg + 1) * p.passes - 1) * waves + wave);
    for (int pass = p.passes - 1; pass >= 0; --pass) {
        const int chunk = (seg * p.passes + pass) * waves + wave;
        const int t0 = chunk * CHUNK;
        // Of a and 1 - a the smaller is held, with the sign saying which: the
        // other follows without cancelling, in half the registers. dist is
        // h_{t-1} - v, g is dy silu(o).
        float m[CHUNK][2], dist[CHUNK][2], g[CHUNK][2], h[2] = {kept[0], kept[1]};
        E* to = p.dgates + t0 * step * 3;
#pragma unroll
        for (int k = 0; k < CHUNK; ++k, to += 3 * step)
            if (t0 + k < p.T) {
                const bool real = t0 + k < q.len;
                float out[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float a, keep, val, grad;
                    sigmoid_pair(f[k][i], a, keep);
                    silu_grad(o[k][i], val, grad);
                    m[k][i] = real ? (a <= keep ? a : -keep) : -0.0f;  // a pad: a = 1
                    g[k][i] = real ? dy[k][i] * val : 0.0f;
                    if (!ONLY_MAP) {
                        dist[k][i] = h[i] - v[k][i];
                        h[i] = real ? a * h[i] + keep * v[k][i] : h[i];
                        out[i] = real ? dy[k][i] * h[i] * grad : 0.0f;
                    }
                }
                if (!ONLY_MAP)
                    store2<EVEN>(to + 2 * (int64_t)p.H, gate_at, q.n, out[0], out[1]);
            }
        if (pass > 0) fetch(chunk - waves);
        float A[2] = {1.0f, 1.0f}, Rl[2] = {0.0f, 0.0f}, R[2];
#pragma unroll
        for (int k = CHUNK - 1; k >= 0; --k)
            if (t0 + k < p.T)
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
            to -= 3 * step;
            if (t0 + k < p.T) {
                const bool real = t0 + k < q.len;
                float df[2], dv[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const bool neg = __builtin_signbit(m[k][i]);
                    const float a = neg ? 1.0f + m[k][i] : m[k][i];
                    const float keep = neg ? -m[k][i] : 1.0f - m[k][i];
                    const float G = R[i] + g[k][i];
                    R[i] = a * G;
                    df[i] = real ? R[i] * keep * dist[k][i] : 0.0f;
                    dv[i] = real ? G * keep : 0.0f;
                }
                store2<EVEN>(to, gate_at, q.n, df[0], df[1]);
                store2<EVEN>(to + p.H, gate_at, q.n, dv[0], dv[1]);
            }
        }
    }
    if (wave != 0) return;
    if (ONLY_MAP) {
        for (int i = 0; i < q.n; ++i)
            p.maps[seg * step + at + i] = make_float2(total[i], carry[i]);
    } else if (seg == 0) {
        store2<EVEN>(p.dh0, at, q.n, carry[0], carry[1]);
    }
}

// How time is laid over waves and blocks; a tile is 64 lanes' channels. Four
// waves a SIMD hide the memory's latency, so a block has the 4 to 8 waves that
// bring the launch to WAVES. Measured in bf16, H = 512, forward and backward, side
// by side when the rule was made: 1024 tiles of 80 steps 20 and 36 us with 4
// waves, 21 and 46 with 5; 256 tiles
// of 200 steps 16 and 26 with 7, 20 and 32 with 4. Where 8 waves leave the card
// half empty and take three passes or more, the chunks are dealt out to
// `segments` blocks of 4 waves: 64 tiles of 256 steps take 11 and 17 us in 8
// segments, 15 and 23 in one; of 128 steps 9 and 13 either way. These were even H;
// the rule is the same for odd ones, whose lanes take two loads a pair.
struct Plan {
    int waves, segments, passes;
};

constexpr int WAVES = 4096;

Plan plan_of(int T, int B, int H) {
    const int64_t tiles = ((int64_t)B * ((H + 1) / 2) + 63) / 64;
    if (T == 0 || tiles == 0) return {1, 1, 0};  // the state alone, or nothing
    const int chunks = (T + CHUNK - 1) / CHUNK;
    const int64_t most = WAVES / tiles;
    int waves = most < 4 ? 4 : most < MAX_WAVES ? (int)most : MAX_WAVES;
    int passes = (chunks + waves - 1) / waves;
    if (tiles * waves * 2 > WAVES || passes < 3) return {(chunks + passes - 1) / passes, 1, passes};
    waves = 4;
    passes = (chunks + waves - 1) / waves;
    const int64_t want = (WAVES + tiles * waves - 1) / (tiles * waves);
    const int segments = (int)(want < passes ? want : passes);
    const int each = (passes + segments - 1) / segments;
    return {waves, (passes + each - 1) / each, each};
}

template <typename E>
int run(Args<E> p, bool back, hipStream_t st) {
    if ((int64_t)p.B * p.H == 0) return 0;
    const Plan plan = plan_of(p.T, p.B, p.H);
    p.segments = plan.segments;
    p.passes = plan.passes;
    const int64_t tiles = ((int64_t)p.B * ((p.H + 1) / 2) + 63) / 64;
    const dim3 grid((unsigned)tiles, plan.segments), block(64 * plan.waves);
    const auto go = [&](auto even, auto only_map) {
        constexpr bool EVEN = decltype(even)::value, MAP = decltype(only_map)::value;
        if (back) recurrence_bwd_kernel<E, EVEN, MAP><<<grid, block, 0, st>>>(p);
        else recurrence_fwd_kernel<E, EVEN, MAP><<<grid, block, 0, st>>>(p);
        return hipGetLastError() == hipSuccess;
    };
    const std::true_type yes;
    const std::false_type no;
    if (plan.segments > 1) {
        if (!p.maps) return -1;
        if (!(p.H % 2 ? go(no, yes) : go(yes, yes))) return -3;
    }
    return (p.H % 2 ? go(no, no) : go(yes, no)) ? 0 : -3;
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
