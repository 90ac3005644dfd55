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
// but the inputs lives between the passes, and g and u are never rounded. dp is
// rounded to the type, as the matrix instructions of the next products take it: in
// bf16 a second rounding of half a step behind dx and dW, whose error (of the norm,
// against 64 bits) is 0.0023 with it and 0.0017 without. db sums dp unrounded.
//
// Bound by the matrix instructions where the sizes are large: in a training pass
// 16384 x 2048 x 4096 (M, K, F) in bf16 takes 471 us forward, and 526, 437 and 411
// for dp, dx and dW on the MI355X (rocprofv3, medians), 1170, 1050, 1260 and 1340
// TFLOP/s, where a library's plain product of 8192^3 reaches 1358. What is left goes
// to LDS and, for dp, which reads dy and writes 2F columns, to the memory at the end
// of each tile, and to the 23 registers a thread that its largest tile's end spills.
// fp32 4000 x 2000 x 4000 takes 920 to 958 us a product, 134 to 139 of 153 TFLOP/s.
// Keeping g and u would save the second of the four products and cost 2F columns of
// 32 bits in memory, 537 MB at the large size: it was not taken.

#include "gated_common.h"

namespace {

using f4 = __attribute__((ext_vector_type(4))) float;
using bf8 = __attribute__((ext_vector_type(8))) __bf16;
using s4 = __attribute__((ext_vector_type(4))) short;
using u4 = __attribute__((ext_vector_type(4))) unsigned int;
#define LDS_PTR(T) __attribute__((address_space(3))) T*

// Tiles are handled in pieces of 16 bytes: PIECE elements.
template <typename E> constexpr int PIECE = 16 / (int)sizeof(E);
// k of one stage of a tile: 64 bytes of it, as much as the matrix instructions
// take of a lane's piece.
template <typename E> constexpr int DEPTH = 64 / (int)sizeof(E);

// Reads as zeros wherever a piece lies past the operand's end.
__device__ const u4 nothing = {0, 0, 0, 0};

// A lane's piece holds k = 4 groups of PIECE, group lane / 16, of one row (or
// column) lane % 16. bf16 takes the piece in one instruction; fp32 in four of
// k = 4, the s-th taking element s of every group.
DEV_INLINE f4 mul(bf16, u4 a, u4 b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, a),
                                                   __builtin_bit_cast(bf8, b), c, 0, 0, 0);
}
DEV_INLINE f4 mul(float, u4 a, u4 b, f4 c) {
    const f4 x = __builtin_bit_cast(f4, a), y = __builtin_bit_cast(f4, b);
#pragma unroll
    for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[s], y[s], c, 0, 0, 0);
    return c;
}

// 16 bytes a lane from memory to LDS, lane l's to to[l]: from a wave's address
// and a lane's offset, or from a lane's address. The caller waits: the compiler,
// which would know of the builtin's loads, has every transposing read wait for
// all of them, also those of the stages to come (600 us in place of 440 for
// 8192 x 2048 x 16384). The reads of LDS keep their distance by wait_and_meet,
// which no memory access and no other asm crosses.
DEV_INLINE void load_to_lds(const void* base, unsigned bytes, unsigned to) {
#ifdef __HIP_DEVICE_COMPILE__
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                 :
                 : "s"(to), "v"(bytes), "s"((__attribute__((address_space(1))) const void*)base)
                 : "m0");
#endif
}
DEV_INLINE void load_to_lds(const void* p, unsigned to) {
#ifdef __HIP_DEVICE_COMPILE__
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
                 :
                 : "s"(to), "v"((__attribute__((address_space(1))) const void*)p)
                 : "m0");
#endif
}

// How an operand lies in memory: k together (rows of it are the result's rows or
// columns), or the result's index together (rows of it are k).
enum class Lie { K, INDEX };

// One operand's stages of SPAN indexes by DEPTH k, in LDS as the operand lies in
// memory, the pieces permuted so that the lanes that read together meet
// different banks: by the place of the row in its fragment where k lies
// together; else by the 8 rows of k (bf16, pairs of pieces) or the 4 (fp32,
// fours of pieces) that one cycle of 64 banks takes values of.
// JUMP: a fragment's 16 indexes are four runs of 4, 4 * JUMP apart; JUMP of
// them, 4 apart, cover 16 * JUMP indexes, and a lane's accumulators 4 * JUMP
// neighbours of the result, which it stores in one piece.
template <typename E, Lie LIE, int SPAN, int THREADS, bool DIRECT, int JUMP>
struct Operand {
    static constexpr int P = PIECE<E>, PIECES = SPAN * 4;
    // Every thread takes part in every round, so that each wave has as many loads
    // under way: ROOM pieces of a stage, the last ones without use.
    static constexpr int ROUNDS = (PIECES + THREADS - 1) / THREADS, ROOM = ROUNDS * THREADS;
    static constexpr int ROW = LIE == Lie::K ? 4 : SPAN / P;  // pieces of a row in LDS
    static constexpr int KEPT = (ROW & -ROW) - 1;  // bits that may turn without leaving it

    const E* base;        // the tile's first index and k
    int64_t pitch;
    int inside;           // indexes of the tile that exist, K: 1 at least
    int half, other;      // K: indexes from `half` on lie `other` rows further
    unsigned at[ROUNDS];  // this thread's pieces: elements from base on, at k = 0
    u4 held[DIRECT ? 1 : 3][ROUNDS];  // stages on their way through registers

    static DEV_INLINE int swizzle(int row, int piece) {
        const int run = row / (4 * JUMP);
        return LIE == Lie::K    ? piece ^ ((run & 1) << 1 | (run >> 1 & 1))
               : sizeof(E) == 2 ? piece ^ (((row & 3) | (row >> 1 & 4)) << 1 & KEPT)
                                : piece ^ ((row >> 2 & 3) << 2 & KEPT);
    }

    // A thread's row of the stage in LDS, and its piece of that row in memory.
    static DEV_INLINE int row_of(int r) { return (r * THREADS + (int)threadIdx.x) % PIECES / ROW; }
    static DEV_INLINE int piece_of(int r) {
        return swizzle(row_of(r), (r * THREADS + (int)threadIdx.x) % PIECES % ROW);
    }

    // From the index `first` on, `count` of them in all. From the tile's `half` on
    // K's indexes are those of its first half, `other` rows further. Indexes past
    // the end read the last ones: nothing of theirs is stored.
    DEV_INLINE void start(const E* p, int64_t pitch_, int first, int count, int half, int other) {
        pitch = pitch_;
        base = p + (LIE == Lie::K ? first * pitch : first);
        inside = count - first;
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) {
            const int row = row_of(r);
            if constexpr (LIE == Lie::K) {
                int i = row % half;
                if (i >= inside) i = inside - 1;
                at[r] = (unsigned)((i + (row >= half ? (int64_t)other : 0)) * pitch) + piece_of(r) * P;
            } else {
                const int i = piece_of(r) * P;
                const int last = (inside - 1) / P * P;  // piece
                at[r] = (unsigned)(row * pitch) + (i < last ? i : last);
            }
        }
    }

    // Elements of a piece that exist in the stage at k0.
    DEV_INLINE int left(int r, int k0, int k_hi) const {
        if constexpr (LIE == Lie::K) return k_hi - k0 - piece_of(r) * P;
        else return k0 + row_of(r) >= k_hi ? 0 : DIRECT ? P : inside - piece_of(r) * P;
    }

    // Every piece of the stage can be read whole. Unaligned ones may pass a row's
    // end, into the next row: their values past it belong to results that are not
    // stored.
    DEV_INLINE bool whole(int k0, int k_hi) const {
        if (LIE == Lie::K || DIRECT || SPAN <= inside) return k0 + DEPTH<E> <= k_hi;
        return k0 + DEPTH<E> < k_hi && pitch >= P;
    }

    // One round of a whole stage.
    DEV_INLINE void fetch_round(int r, unsigned stage, int k0) const {
        const unsigned to = stage + __builtin_amdgcn_readfirstlane(threadIdx.x) * 16;
        load_to_lds(base + (LIE == Lie::K ? k0 : k0 * pitch), at[r] * (unsigned)sizeof(E),
                    to + r * THREADS * 16);
    }

    // A stage straight to LDS. Aligned pitches: a piece exists whole or not at all.
    DEV_INLINE void fetch(unsigned stage, int k0, int k_hi) const {
        const E* p = base + (LIE == Lie::K ? k0 : k0 * pitch);
        const unsigned to = stage + __builtin_amdgcn_readfirstlane(threadIdx.x) * 16;
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r)
            load_to_lds(left(r, k0, k_hi) > 0 ? (const void*)(p + at[r]) : &nothing,
                        to + r * THREADS * 16);
    }

    // A stage by way of registers, element by element where it is not WHOLE.
    template <bool WHOLE>
    DEV_INLINE void hold(int set, int k0, int k_hi) {
        const E* p = base + (LIE == Lie::K ? k0 : k0 * pitch);
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) {
            E v[P];
            load_run<E, P>(p + at[r], WHOLE ? P : left(r, k0, k_hi), v);
            held[set][r] = __builtin_bit_cast(u4, v);
        }
    }
    DEV_INLINE void settle(int set, u4* stage) const {
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) stage[r * THREADS + threadIdx.x] = held[set][r];
    }

    // The piece of the matrix instructions for the 16 indexes of the fragment that
    // starts at `first`.
    static DEV_INLINE u4 read(const u4* stage, int first) {
        const int lane = threadIdx.x & 63, group = lane >> 4;
        if constexpr (LIE == Lie::K) {
            const int row = first + (lane >> 2 & 3) * 4 * JUMP + (lane & 3);
            return stage[row * 4 + swizzle(row, group)];
        } else if constexpr (sizeof(E) == 2) {
            // 16 lanes read 4 k by 16 indexes, 8 bytes each, and get back the 4 k
            // of one index each
            s4 v[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int row = group * 8 + h * 4 + ((lane & 15) >> 2);
                const int i = first + (lane & 3) * 4;
                const char* p = (const char*)(stage + row * ROW + swizzle(row, i / P)) + (i % P) * 2;
                v[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_PTR(s4))p);
            }
            return __builtin_bit_cast(u4, v);
        } else {
            const int i = first + (lane & 15);
            u4 out;
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const int row = group * 4 + s;
                out[s] = reinterpret_cast<const unsigned*>(stage + row * ROW + swizzle(row, i / P))[i % P];
            }
            return out;
        }
    }
};

enum class End { GATED, GATED_GRAD, PLAIN, PART };

// C(m, n) = sum over k of A(m, k) B(n, k).
template <typename E>
struct Args {
    const E *a, *b;
    int64_t pitch_a, pitch_b;
    int M, N, K;        // GATED*: N is F
    const E* bias;      // [2F] or null
    const E* dy;        // [M, F]
    E* out;             // GATED: y [M, F]; GATED_GRAD: dp [M, 2F]; PLAIN: [M, N]
    float* part;        // GATED_GRAD: [tiles of M, 2F] or null; PART: [splits, M, N]
    int tiles_m, tiles_n, per_split;
};

// Blocks go round the 8 XCDs by their index. Each XCD, which has an L2 of its
// own, gets a run of tiles, in patches of 8 rows of tiles: those in flight
// share their operands.
DEV_INLINE void tile_of(int id, int tiles_m, int tiles_n, int& tm, int& tn) {
    const int total = tiles_m * tiles_n, q = total / 8, r = total % 8;
    const int xcd = id % 8, i = id / 8;
    const int t = xcd * q + (xcd < r ? xcd : r) + i;
    const int patch = t / (8 * tiles_n), first = patch * 8;
    const int rows = tiles_m - first < 8 ? tiles_m - first : 8;
    const int in = t - patch * 8 * tiles_n;
    tm = first + in % rows;
    tn = in / rows;
}

// BM x BN of a result by WM x WN waves, with STAGES of the operands in LDS, of 64
// bytes a row. A fifth one fits with the largest tile and with four blocks of the
// smallest, whose few rows wait for the weights from memory. Side by side when it was
// chosen, each kernel alone in a loop: 16384 x 2048 x 4096 forward 436 us, 457 with two
// stages of 128 bytes; 16 x 2048 x 4096 11.5 us, 15.2 with four stages. Between these
// tiles it gained nothing.
template <int BM_, int BN_, int WM_, int WN_, int STAGES_ = 4>
struct Tile {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, THREADS = 64 * WM * WN;
    static constexpr int STAGES = STAGES_;
    static_assert(STAGES == 4 || STAGES == 5, "the waits count one or two stages under way");
    static constexpr int MI = BM / WM / 16, NI = BN / WN / 16;
    static_assert(MI * WM * 16 == BM && NI * WN * 16 == BN, "whole fragments");
};

template <typename E, int N, bool INSIDE>
DEV_INLINE void load_piece(const E* p, int have, E (&v)[N]) {
    if constexpr (INSIDE) have = N;
    load_run<E, N>(p, have, v);
}
template <typename E, int N, bool INSIDE>
DEV_INLINE void store_piece(E* p, int have, const E (&v)[N]) {
    if constexpr (INSIDE) have = N;
    store_run<E, N>(p, have, v);
}

template <typename E, typename T, End END, bool INSIDE>
DEV_INLINE void finish(const Args<E>& p, const f4 (&acc)[T::MI][T::NI], int tm, int m0, int n0,
                       void* lds) {
    constexpr bool GATED = END == End::GATED || END == End::GATED_GRAD;
    constexpr int HALF = T::BN / 2;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wm = wave / T::WN, wn = wave % T::WN;
    const int row0 = m0 + wm * T::MI * 16 + (lane & 15);
    if constexpr (GATED) {
        constexpr int NB = T::NI / 2, C = 4 * NB;
        const int in = wn * NB * 16 + (lane >> 4) * C, col = n0 + in, have = p.N - col;
        float bg[C] = {}, bu[C] = {}, sg[C] = {}, su[C] = {};
        if (p.bias) {
            E g[C], u[C];
            load_piece<E, C, INSIDE>(p.bias + col, have, g);
            load_piece<E, C, INSIDE>(p.bias + p.N + col, have, u);
#pragma unroll
            for (int c = 0; c < C; ++c) {
                bg[c] = to_f(g[c]);
                bu[c] = to_f(u[c]);
            }
        }
        // dy of all rows is on its way before the first is used
        E d[END == End::GATED_GRAD ? T::MI : 1][C];
        if (END == End::GATED_GRAD) {
#pragma unroll
            for (int i = 0; i < T::MI; ++i) {
                const int row = row0 + i * 16;
                load_piece<E, C, INSIDE>(p.dy + (int64_t)row * p.N + col, row < p.M ? have : 0, d[i]);
            }
#ifdef __HIP_DEVICE_COMPILE__
            __builtin_amdgcn_sched_barrier(0);
#endif
        }
#pragma unroll
        for (int i = 0; i < T::MI; ++i) {
            const int row = row0 + i * 16;
            if (!INSIDE && (row >= p.M || have <= 0)) continue;
            E out[C], out2[C];
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const float g = acc[i][c / 4][c % 4] + bg[c];
                const float u = acc[i][c / 4 + NB][c % 4] + bu[c];
                float val, grad;
                silu_grad(g, val, grad);
                if (END == End::GATED) {
                    out[c] = from_f<E>(val * u);
                } else {
                    const float dg = to_f(d[i][c]) * u * grad, du = to_f(d[i][c]) * val;
                    out[c] = from_f<E>(dg);
                    out2[c] = from_f<E>(du);
                    sg[c] += dg;
                    su[c] += du;
                }
            }
            if (END == End::GATED) {
                store_piece<E, C, INSIDE>(p.out + (int64_t)row * p.N + col, have, out);
            } else {
                E* to = p.out + (int64_t)row * 2 * p.N + col;
                store_piece<E, C, INSIDE>(to, have, out);
                store_piece<E, C, INSIDE>(to + p.N, have, out2);
            }
        }
        if (END == End::GATED_GRAD && p.part) {
            float* sums = reinterpret_cast<float*>(lds);  // [WM][2][HALF]
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const float a = row_sum16(sg[c]), b = row_sum16(su[c]);
                if ((lane & 15) == 0) {
                    sums[(wm * 2) * HALF + in + c] = a;
                    sums[(wm * 2 + 1) * HALF + in + c] = b;
                }
            }
            __syncthreads();
            for (int c = threadIdx.x; c < 2 * HALF; c += T::THREADS) {
                const int which = c / HALF, at = c % HALF;
                float s = 0.0f;
#pragma unroll
                for (int w = 0; w < T::WM; ++w) s += sums[(w * 2 + which) * HALF + at];
                if (n0 + at < p.N)
                    p.part[(int64_t)tm * 2 * p.N + which * (int64_t)p.N + n0 + at] = s;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < T::MI; ++i) {
            const int row = row0 + i * 16;
            if (!INSIDE && row >= p.M) continue;
#pragma unroll
            for (int j = 0; j < T::NI; ++j) {
                const int col = n0 + (wn * T::NI + j) * 16 + (lane >> 4) * 4, have = p.N - col;
                if (!INSIDE && have <= 0) continue;
                const int64_t at = (int64_t)row * p.N + col;
                const float v[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
                if (END == End::PLAIN) {
                    E out[4];
#pragma unroll
                    for (int q = 0; q < 4; ++q) out[q] = from_f<E>(v[q]);
                    store_piece<E, 4, INSIDE>(p.out + at, have, out);
                } else {
                    store_piece<float, 4, INSIDE>(
                        p.part + blockIdx.z * (int64_t)p.M * p.N + at, have, v);
                }
            }
        }
    }
}

// Waits until at most `loads` of this wave's loads and none of its LDS reads are
// under way, then for the other waves.
template <int LOADS>
DEV_INLINE void wait_and_meet() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((LOADS & 15) | (LOADS >> 4) << 14 | 7 << 4);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

template <typename E, typename T, Lie LA, Lie LB, End END, bool DIRECT>
__global__ void __launch_bounds__(T::THREADS)
product_kernel(Args<E> p) {
    constexpr bool GATED = END == End::GATED || END == End::GATED_GRAD;
    constexpr int HALF = T::BN / 2, COLS = GATED ? HALF : T::BN;  // of the result a block
    constexpr int NB = GATED ? T::NI / 2 : T::NI;  // a wave's fragments side by side
    constexpr int BD = DEPTH<E>;
    using A = Operand<E, LA, T::BM, T::THREADS, DIRECT, 1>;
    using B = Operand<E, LB, T::BN, T::THREADS, DIRECT, GATED ? NB : 1>;
    __shared__ u4 lds[T::STAGES][A::ROOM + B::ROOM];
    const int wave = threadIdx.x >> 6;
    const int wm = wave / T::WN, wn = wave % T::WN;
    int tm, tn;
    tile_of(blockIdx.x, p.tiles_m, p.tiles_n, tm, tn);
    const int m0 = tm * T::BM, n0 = tn * COLS;
    const int k_lo = blockIdx.z * p.per_split;
    const int k_hi = k_lo + p.per_split < p.K ? k_lo + p.per_split : p.K;

    A a;
    B b;
    a.start(p.a, p.pitch_a, m0, p.M, T::BM, 0);
    b.start(p.b, p.pitch_b, n0, p.N, GATED ? HALF : T::BN, GATED ? p.N : 0);
    constexpr int STAGES = T::STAGES;
    const unsigned lds_at = (unsigned)(uintptr_t)(LDS_PTR(u4))&lds[0][0];
    const auto fetch = [&](int place, int k0) {
        const unsigned to = lds_at + place * (A::ROOM + B::ROOM) * 16;
        a.fetch(to, k0, k_hi);
        b.fetch(to + A::ROOM * 16, k0, k_hi);
    };
    const auto hold = [&](int set, int k0, auto whole) {
        constexpr bool WHOLE = decltype(whole)::value;
        if (!WHOLE && k0 >= k_hi) return;
        a.template hold<WHOLE>(set, k0, k_hi);
        b.template hold<WHOLE>(set, k0, k_hi);
    };
    const auto settle = [&](int set, int place) {
        a.settle(set, lds[place]);
        b.settle(set, lds[place] + A::ROOM);
    };
    // Fragments in registers: those of b of two stages, of a the next AHEAD + 1.
    constexpr int RING = T::MI < 4 ? T::MI : 2 * T::MI % 4 == 0 ? 4 : 5, AHEAD = RING - 1;
    static_assert(2 * T::MI % RING == 0, "a turn of the loop ends where it began");
    static_assert(T::NI <= T::MI, "b's fragments are read beside a's");
    u4 af[RING], bf[2][T::NI];
    const auto read_b = [&](int set, int j, int place) {
        // gated: the wave's first half of columns are gates, then their values
        const int first = GATED ? (j / NB) * HALF + wn * NB * 16 + j % NB * 4
                                : (wn * NB + j) * 16;
        bf[set][j] = B::read(lds[place] + A::ROOM, first);
    };
    const auto read_a = [&](int slot, int i, int place) {
        af[slot] = A::read(lds[place], (wm * T::MI + i) * 16);
    };
    // LDS instructions of a fragment, matrix instructions of a product.
    constexpr int RA = LA == Lie::K ? 1 : sizeof(E) == 2 ? 2 : 4;
    constexpr int RB = LB == Lie::K ? 1 : sizeof(E) == 2 ? 2 : 4;
    constexpr int EACH = sizeof(E) == 2 ? 1 : 4;

    f4 acc[T::MI][T::NI] = {};
    // Stage t lies in place t % STAGES. While its products run, row of fragments by
    // row, its last fragments and its successor's first are read: the successor has
    // landed when the waves meet at its beginning, and the place of the stage
    // before it is free for the one STAGES - 1 on.
    constexpr int LOADS = DIRECT ? A::ROUNDS + B::ROUNDS : 0;
    const auto read_first = [&] {
#pragma unroll
        for (int j = 0; j < T::NI; ++j) read_b(0, j, 0);
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) read_a(i, i, 0);
    };
    int place = 0;  // of the stage whose products run
    // Two stages from k0 on. SPREAD: all that they wait for and fetch exists whole,
    // and is fetched a round at a time between the products: all at once the loads
    // hold up the waves until the memory has taken them. By way of registers a
    // stage is fetched three ahead and settles in LDS one ahead; without a branch
    // on the way, behind which the compiler would wait for all loads.
    const auto two_stages = [&](int k0, auto spread) {
        constexpr bool SPREAD = decltype(spread)::value;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int at = k0 + s * BD, far = at + (STAGES - 1) * BD;
            if (!SPREAD && at >= k_hi) break;
            const int after = place + 1 < STAGES ? place + 1 : 0;
            const int before = place > 0 ? place - 1 : STAGES - 1;
            const unsigned to = lds_at + before * (A::ROOM + B::ROOM) * 16;
            if constexpr (!DIRECT) {
                if (SPREAD || at + BD < k_hi) settle(s, after);
                wait_and_meet<63>();
                hold(s, at + 3 * BD, spread);
            } else if (SPREAD || far - BD < k_hi) {
                wait_and_meet<(STAGES - 3) * LOADS>();
            } else if (STAGES > 4 && far - 2 * BD < k_hi) {
                wait_and_meet<LOADS>();  // of the STAGES - 3 stages that may be on their way one is
            } else {
                wait_and_meet<0>();
            }
            if constexpr (DIRECT && !SPREAD)
                if (far < k_hi) fetch(before, far);
#pragma unroll
            for (int i = 0; i < T::MI; ++i) {
                const int now = s * T::MI + i, next = i + AHEAD;
                read_a((now + AHEAD) % RING, next % T::MI, next < T::MI ? place : after);
                if (i < T::NI) read_b((s + 1) & 1, i, after);
                if constexpr (SPREAD && DIRECT)
#pragma unroll
                    for (int n = i * LOADS / T::MI; n < (i + 1) * LOADS / T::MI; ++n) {
                        if (n < A::ROUNDS) a.fetch_round(n, to, far);
                        else b.fetch_round(n - A::ROUNDS, to + A::ROOM * 16, far);
                    }
#pragma unroll
                for (int j = 0; j < T::NI; ++j)
                    acc[i][j] = mul(E(), bf[s & 1][j], af[now % RING], acc[i][j]);
#ifdef __HIP_DEVICE_COMPILE__
                __builtin_amdgcn_sched_group_barrier(0x100, RA, 0);
                if (i < T::NI) __builtin_amdgcn_sched_group_barrier(0x100, RB, 0);
                __builtin_amdgcn_sched_group_barrier(0x008, T::NI * EACH, 0);
#endif
            }
            place = after;
        }
    };
    // The first stages, then pairs of them as long as the second one fetches a
    // whole stage, then the last ones.
    constexpr int FAR = DIRECT ? STAGES - 1 : 3;
    const int last = a.whole(k_lo, k_hi) && b.whole(k_lo, k_hi) ? k_hi - (FAR + 2) * BD - !DIRECT
                                                                : k_lo - 1;
    int k0 = k_lo;
    const auto main_loop = [&] {
#pragma unroll 1
        for (; k0 <= last; k0 += 2 * BD) two_stages(k0, std::true_type());
    };
    if constexpr (DIRECT) {
        if (k_lo < k_hi) {
#pragma unroll
            for (int s = 0; s < STAGES - 1; ++s)
                if (k_lo + s * BD < k_hi) fetch(s, k_lo + s * BD);
            if (k_lo + (STAGES - 2) * BD >= k_hi) wait_and_meet<0>();
            else wait_and_meet<(STAGES - 2) * LOADS>();
            read_first();
            main_loop();
        }
    } else {
        const auto begin = [&](auto whole) {
            hold(2, k_lo, whole);
            hold(0, k_lo + BD, whole);
            hold(1, k_lo + 2 * BD, whole);
            settle(2, 0);
            wait_and_meet<63>();
            read_first();
        };
        if (k_lo <= last) {
            begin(std::true_type());
            main_loop();
        } else if (k_lo < k_hi) {
            begin(std::false_type());
        }
    }
#pragma unroll 1
    for (; k0 < k_hi; k0 += 2 * BD) two_stages(k0, std::false_type());
    wait_and_meet<0>();  // nothing is on its way into LDS any more

    // Fragment j's accumulator holds row lane % 16 and, as its element q, column
    // (lane / 16) * 4 * JUMP + 4 j + q. Tiles inside the result are stored
    // without looking at each piece.
    if (m0 + T::BM <= p.M && n0 + COLS <= p.N)
        finish<E, T, END, true>(p, acc, tm, m0, n0, lds);
    else
        finish<E, T, END, false>(p, acc, tm, m0, n0, lds);
}

// out[i] = sum over the splits of part [splits, n], in a fixed order.
template <typename E>
struct Splits {
    const float* part;
    E* out;
    int64_t n;
    int splits;  // 1: the product has written the result itself
    // Groups of a block's threads, which add every GROUPS-th split of the same
    // results. Four where the results are few and their splits many: 128 x 64 of 64
    // splits take 10 us with the product, 18 with one group, but 2048 x 512 of 8
    // take 58 in place of 55. The border lies between these two, which alone were
    // measured.
    __host__ __device__ bool grouped() const { return splits >= 8 && n <= 1 << 19; }
    int blocks() const {
        const int each = grouped() ? 1024 : 4096;
        return splits > 1 ? (int)((n + each - 1) / each) : 0;
    }
};

template <typename E, int GROUPS>
DEV_INLINE void join_splits(const Splits<E>& q, int block) {
    constexpr int THREADS = 1024 / GROUPS;
    const int group = threadIdx.x / THREADS, in = threadIdx.x % THREADS;
    const int64_t i = ((int64_t)block * THREADS + in) * 4, left = q.n - i;
    const int have = left < 0 ? 0 : left < 4 ? (int)left : 4;
    f4 s = {};
    float v[8][4];
    for (int z0 = group; z0 < q.splits; z0 += 8 * GROUPS) {
#pragma unroll
        for (int z = 0; z < 8; ++z)
            if (z0 + GROUPS * z < q.splits)
                load_run<float, 4>(q.part + (z0 + GROUPS * z) * q.n + i, have, v[z]);
#pragma unroll
        for (int z = 0; z < 8; ++z)
            if (z0 + GROUPS * z < q.splits) s += f4{v[z][0], v[z][1], v[z][2], v[z][3]};
    }
    if constexpr (GROUPS > 1) {
        __shared__ f4 sums[GROUPS][THREADS];
        sums[group][in] = s;
        __syncthreads();
        if (group) return;
#pragma unroll
        for (int g = 1; g < GROUPS; ++g) s += sums[g][in];
    }
    E o[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] = from_f<E>(s[k]);
    store_run<E, 4>(q.out + i, have, o);
}
template <typename E>
DEV_INLINE void join_splits(const Splits<E>& q, int block) {
    if (q.grouped()) join_splits<E, 4>(q, block);
    else join_splits<E, 1>(q, block);
}

// What the products of the backward pass leave in parts, in one launch: three
// would take a small batch longer than their work.
template <typename E>
__global__ void __launch_bounds__(1024)
join_kernel(Splits<E> dx, int dx_blocks, Splits<E> dw, int dw_blocks,
            const float* __restrict__ part_db, E* __restrict__ db, int rows, int cols) {
    int block = blockIdx.x;
    if (block < dx_blocks) return join_splits(dx, block);
    block -= dx_blocks;
    if (block < dw_blocks) return join_splits(dw, block);
    sum_columns<E>(part_db, db, rows, cols, block - dw_blocks);
}

int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// The tiles that a product may be cut into: how many blocks of one share a CU,
// what the CU reaches with them in a long product (TFLOP/s), and the time that
// one block alone takes for a step of DEPTH, which it spends waiting (us); all
// measured with stages that go straight to LDS. By way of registers a product takes
// up to half as long again as they say.
struct Rate {
    int blocks;
    double tflops, alone;
};
template <typename E, typename F>
void each_tile(F&& f) {
    if constexpr (sizeof(E) == 2) {
        f(Tile<256, 256, 2, 4, 5>(), Rate{1, 4.9, 0});
        f(Tile<192, 256, 2, 4>(), Rate{1, 4.7, 0});
        f(Tile<160, 256, 2, 4>(), Rate{1, 4.5, 0});
        f(Tile<128, 256, 2, 4>(), Rate{1, 4.3, 0});
        f(Tile<128, 128, 2, 2>(), Rate{2, 3.5, 0.4});
        f(Tile<64, 64, 2, 2, 5>(), Rate{4, 2.0, 0.25});
    } else {
        f(Tile<128, 128, 2, 2>(), Rate{2, 0.5, 1.1});
        f(Tile<64, 64, 2, 2>(), Rate{4, 0.47, 0.38});
    }
}

// How a product is cut: which tile, and into how many splits of k, whose sums
// join_kernel adds.
struct Cut {
    int bm, bn, splits;
};

// The cut with the least estimated time: what the fullest CU does, plus the
// splits' way through memory. `wide` is N, or 2F where gate and value columns
// share a tile.
template <typename E>
Cut cut_of(int64_t m, int64_t wide, int64_t k, bool may_split) {
    constexpr int64_t CUS = 256;
    Cut best{0, 0, 1};
    double least = 0;
    if (m < 1) m = 1;  // sums over no rows, for one
    if (wide < 1) wide = 1;
    each_tile<E>([&](auto tile, Rate rate) {
        using T = decltype(tile);
        const int64_t tiles = (int64_t)ceil_div(m, T::BM) * ceil_div(wide, T::BN);
        const int64_t steps = ceil_div(k, DEPTH<E>);
        for (int64_t splits = 1; splits <= 64; splits *= 2) {
            if (splits > 1 && (!may_split || steps < 2 * splits)) break;
            const int64_t mine = (tiles * splits + CUS - 1) / CUS;  // a CU's blocks
            const int64_t together = mine < rate.blocks ? mine : rate.blocks;
            const double shared = together * 2.0 * T::BM * T::BN * DEPTH<E> / rate.tflops * 1e-6;
            const double step = shared > rate.alone ? shared : rate.alone;
            const int64_t rounds = (mine + together - 1) / together;
            double us = rounds * (ceil_div(steps, splits) * step + 1.5 + T::BM * T::BN / 32768.0);
            if (splits > 1) us += 3.0 + splits * m * wide * 8 / 6e6;
            if (best.bm == 0 || us < least) {
                least = us;
                best = {T::BM, T::BN, (int)splits};
            }
        }
    });
    return best;
}

template <typename E, typename T, Lie LA, Lie LB, End END>
int launch(Args<E> p, int splits, hipStream_t st) {
    constexpr bool GATED = END == End::GATED || END == End::GATED_GRAD;
    p.tiles_m = ceil_div(p.M, T::BM);
    p.tiles_n = ceil_div(p.N, GATED ? T::BN / 2 : T::BN);
    p.per_split = ceil_div(ceil_div(p.K > 0 ? p.K : 1, splits), DEPTH<E>) * DEPTH<E>;
    const dim3 grid(p.tiles_m * p.tiles_n, 1, splits);
    const auto whole = [](const void* q, int64_t pitch) {
        return (uintptr_t)q % 16 == 0 && pitch % PIECE<E> == 0;
    };
    if (whole(p.a, p.pitch_a) && whole(p.b, p.pitch_b))
        product_kernel<E, T, LA, LB, END, true><<<grid, T::THREADS, 0, st>>>(p);
    else
        product_kernel<E, T, LA, LB, END, false><<<grid, T::THREADS, 0, st>>>(p);
    LSTM_CHECK_LAUNCH();
    return 0;
}

template <typename E, Lie LA, Lie LB, End END>
int product(const Args<E>& p, Cut cut, hipStream_t st) {
    int rc = -1;
    each_tile<E>([&](auto tile, Rate) {
        using T = decltype(tile);
        if (T::BM == cut.bm && T::BN == cut.bn) rc = launch<E, T, LA, LB, END>(p, cut.splits, st);
    });
    return rc;
}

// A plain product to `out`, in one piece or in splits, for the join, through its part.
template <typename E, Lie LA, Lie LB>
int plain(Args<E> p, Cut cut, const Splits<E>& to, hipStream_t st) {
    p.out = to.out;
    p.part = const_cast<float*>(to.part);
    return to.splits == 1 ? product<E, LA, LB, End::PLAIN>(p, cut, st)
                          : product<E, LA, LB, End::PART>(p, cut, st);
}

template <typename E> Cut cut_gated(int M, int K, int F) {
    return cut_of<E>(M, 2 * (int64_t)F, K, false);
}
template <typename E> Cut cut_dx(int M, int K, int F) {
    return cut_of<E>(M, K, 2 * (int64_t)F, true);
}
template <typename E> Cut cut_dw(int M, int K, int F) {
    return cut_of<E>(2 * (int64_t)F, K, M, true);
}

template <typename E>
int fwd(const void* x, const void* w, const void* bias, void* y, int M, int K, int F,
        hipStream_t st) {
    if ((int64_t)M * F == 0) return 0;
    Args<E> p{};
    p.a = (const E*)x; p.pitch_a = K;
    p.b = (const E*)w; p.pitch_b = K;
    p.M = M; p.N = F; p.K = K;
    p.bias = (const E*)bias; p.out = (E*)y;
    return product<E, Lie::K, Lie::K, End::GATED>(p, cut_gated<E>(M, K, F), st);
}

// Rows of 2F partial sums for db.
template <typename E>
int bias_parts(int M, int K, int F) {
    return ceil_div(M, cut_gated<E>(M, K, F).bm);
}

// The splits of dx and dw, whose partial sums lie one behind the other.
template <typename E>
void splits_of(int M, int K, int F, E* dx, E* dw, const float* part, Splits<E>& x, Splits<E>& w) {
    x = {part, dx, (int64_t)M * K, dx ? cut_dx<E>(M, K, F).splits : 1};
    const int64_t before = x.splits > 1 ? x.splits * x.n : 0;
    w = {part + before, dw, 2 * (int64_t)F * K, dw ? cut_dw<E>(M, K, F).splits : 1};
}

// Floats of those partial sums.
template <typename E>
int64_t split_sums(int M, int K, int F, bool dx, bool dw) {
    const int64_t x = dx ? cut_dx<E>(M, K, F).splits : 1, w = dw ? cut_dw<E>(M, K, F).splits : 1;
    return (x > 1 ? x * M * K : 0) + (w > 1 ? w * 2 * F * K : 0);
}

template <typename E>
int bwd(const void* x, const void* w, const void* bias, const void* dy, void* dp, void* dx,
        void* dw, void* db, float* part_db, float* part, int M, int K, int F, hipStream_t st) {
    int rc = 0;
    if ((int64_t)M * F != 0) {
        Args<E> p{};
        p.a = (const E*)x; p.pitch_a = K;
        p.b = (const E*)w; p.pitch_b = K;
        p.M = M; p.N = F; p.K = K;
        p.bias = (const E*)bias; p.dy = (const E*)dy; p.out = (E*)dp; p.part = db ? part_db : nullptr;
        rc = product<E, Lie::K, Lie::K, End::GATED_GRAD>(p, cut_gated<E>(M, K, F), st);
        if (rc) return rc;
    }
    Splits<E> sx, sw;
    splits_of<E>(M, K, F, (E*)dx, (E*)dw, part, sx, sw);
    if (dx && sx.n) {
        Args<E> p{};
        p.a = (const E*)dp; p.pitch_a = 2 * (int64_t)F;
        p.b = (const E*)w; p.pitch_b = K;
        p.M = M; p.N = K; p.K = 2 * F;
        rc = plain<E, Lie::K, Lie::INDEX>(p, cut_dx<E>(M, K, F), sx, st);
        if (rc) return rc;
    }
    if (dw && sw.n) {
        Args<E> p{};
        p.a = (const E*)dp; p.pitch_a = 2 * (int64_t)F;
        p.b = (const E*)x; p.pitch_b = K;
        p.M = 2 * F; p.N = K; p.K = M;
        rc = plain<E, Lie::INDEX, Lie::INDEX>(p, cut_dw<E>(M, K, F), sw, st);
        if (rc) return rc;
    }
    const int bx = sx.blocks(), bw = sw.blocks(), bb = db ? column_blocks(2 * F) : 0;
    if (bx + bw + bb == 0) return 0;
    join_kernel<E><<<bx + bw + bb, 1024, 0, st>>>(sx, bx, sw, bw, part_db, (E*)db,
                                                  bias_parts<E>(M, K, F), 2 * F);
    LSTM_CHECK_LAUNCH();
    return 0;
}

}  // namespace

extern "C" int launch_gated_linear_fwd(int is_bf16, const void* x, const void* w,
                                       const void* bias, void* y, int M, int K, int F,
                                       hipStream_t st) {
    return is_bf16 ? fwd<bf16>(x, w, bias, y, M, K, F, st)
                   : fwd<float>(x, w, bias, y, M, K, F, st);
}

// How the product `which` is cut: 0 y's and dp's, 1 dx's, 2 dw's.
extern "C" void gated_linear_cut(int is_bf16, int which, int M, int K, int F, int* bm, int* bn,
                                 int* splits) {
    const auto of = [&](auto e) {
        using E = decltype(e);
        return which == 0 ? cut_gated<E>(M, K, F) : which == 1 ? cut_dx<E>(M, K, F) : cut_dw<E>(M, K, F);
    };
    const Cut cut = is_bf16 ? of(bf16()) : of(float());
    *bm = cut.bm;
    *bn = cut.bn;
    *splits = cut.splits;
}

extern "C" int gated_linear_bias_parts(int is_bf16, int M, int K, int F) {
    return is_bf16 ? bias_parts<bf16>(M, K, F) : bias_parts<float>(M, K, F);
}
extern "C" int64_t gated_linear_split_sums(int is_bf16, int M, int K, int F, int dx, int dw) {
    return is_bf16 ? split_sums<bf16>(M, K, F, dx, dw) : split_sums<float>(M, K, F, dx, dw);
}

extern "C" int launch_gated_linear_bwd(int is_bf16, const void* x, const void* w,
                                       const void* bias, const void* dy, void* dp, void* dx,
                                       void* dw, void* db, float* part_db, float* part,
                                       int M, int K, int F, hipStream_t st) {
    return is_bf16 ? bwd<bf16>(x, w, bias, dy, dp, dx, dw, db, part_db, part, M, K, F, st)
                   : bwd<float>(x, w, bias, dy, dp, dx, dw, db, part_db, part, M, K, F, st);
}
