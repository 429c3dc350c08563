// pm_decay.h — K14: linear attention with a decay for each head, its kernels.
//
// For one head, with log-decays g:   S_t = e^{g_t} S_{t-1} + k_t v_t^T,   o_t = scale S_t^T q_t.
//
// One pass serves the forward and every gradient.  It walks a sequence in chunks of C tokens with
// roles Q, K, V; with G the sums of the log-decays inside the chunk and S the state before it
//     A[i][j] = e^{G_i - G_j} (Q_i . K_j)   for j <= i
//     O_i = e^{G_i} S^T Q_i + sum_j A[i][j] V_j,      S <- e^{G_C} S + sum_j e^{G_C - G_j} K_j V_j^T
//   forward   Q, K, V = q, k, v      O = o    S = the state
//   gq        Q, K, V = go, v, k     O = gq   S = the state, transposed
//   gk        Q, K, V = v, go, q     O = gk   S = the state's gradient, transposed   } from the last
//   gv        Q, K, V = k, q, go     O = gv   S = the state's gradient               } token to the first
// Walking backwards, token t is entered with the log-decay of token t + 1 (none at the end), and the
// first token's own is applied to the last state.  In a group of query heads that share a key head,
// the first two run once per query head, the others sum over the group's heads inside a chunk.
//
// Products run on bf16 MFMA.  A value of more than 8 bits is a sum of bf16 planes (the value rounded, what
// that leaves rounded, ...), a product of two such sums the products of their planes down to the last
// plane's size.  bf16 inputs are one plane and exact; next to them
//   the decayed V, which sums into states      three planes (2^-25 relative; two, 2^-17, in the backward's
//     passes alone took 556 us where three take 580, with the forward)
//   the state in passes that leave parts of the gates' gradient, which is fp32    three (two: 580 for 599 us,
//     and the gradient 3.0e-6 off in the 2-norm where it is 3.7e-7)
//   A and the state in what comes out          two (2^-17).  What comes out in bf16 is then as if it were
//     rounded once, and in fp32 nearly so; one part (2^-8 of each term) took 128 us where two take 135 at
//     B4 T4096 H16 D128, forward, and 536 for 556 with the backward, and was 1.4 times one rounding off
// fp32 inputs and everything next to them are three.  On this card six such bf16 products take 6/16 of
// the time of the fp32 MFMA.
//
// Log-decays are summed in 64 bits, and kept as a multiple of 2^-10 and a rest, so that a
// difference G_i - G_j has fp32's relative error also where both are large (behind a closed gate).
#pragma once

#include <algorithm>
#include <type_traits>

#include "pm_cdna4.h"
#include "pm_decay_args.h"

namespace pm {
namespace {

template <int P>
struct DecayShape {
    static constexpr int C = P == 1 ? 64 : 32;   // tokens of a chunk (three planes of 64 would not fit LDS)
    static constexpr int PA = P == 1 ? 2 : 3;    // planes of A, and of the state in what comes out
    static constexpr int MT = C / 16;            // 16-token tiles
    static constexpr int TRI = MT * (MT + 1) / 2;  // lower 16x16 tiles of A
    static constexpr int BLK = P == 1 ? 6 : 2;   // packed operand blocks of A (qblk)
};

constexpr double kLog2e = 1.4426950408889634;

// ---- planes -----------------------------------------------------------------------------------

// Eight floats as N planes of packed bf16 (plane n holds what the planes before it leave).
template <int N>
__device__ __forceinline__ void split8(const float (&x)[8], u32x4_t (&p)[N]) {
    float r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = x[i];
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned w = pack2(r[2 * i], r[2 * i + 1]);
            p[n][i] = w;
            if (n + 1 < N) {
                r[2 * i] -= __uint_as_float(w << 16);
                r[2 * i + 1] -= __uint_as_float(w & 0xffff0000u);
            }
        }
}
template <int N>
__device__ __forceinline__ void split4(f32x4_t x, u32x2_t (&p)[N]) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
        p[n] = cvt4(x);
        if (n + 1 < N) x -= widen4(p[n]);
    }
}
// acc += X Y over the planes' products that count.
template <int NX, int NY>
__device__ __forceinline__ f32x4_t mfma_planes(const u32x4_t (&x)[NX], const u32x4_t (&y)[NY], f32x4_t acc) {
    constexpr int N = NX > NY ? NX : NY;
#pragma unroll
    for (int s = N - 1; s >= 0; --s)  // the small products first
#pragma unroll
        for (int i = 0; i < NX; ++i) {
            const int j = s - i;
            if (j >= 0 && j < NY)
                acc = mfma32(__builtin_bit_cast(bf16x8_t, x[i]), __builtin_bit_cast(bf16x8_t, y[j]), acc);
        }
    return acc;
}

// ---- loads from global memory -----------------------------------------------------------------

// Eight elements of a row as they are in memory (P 1: bf16, P 3: fp32).
template <int P>
struct Raw8 {
    static constexpr int W = P == 1 ? 4 : 8;
    using E = typename std::conditional<P == 1, uint16_t, float>::type;
    uint32_t w[W];
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < W; ++i) w[i] = 0;
    }
    // all eight, at any alignment of the elements
    __device__ __forceinline__ void load(const void* p) { __builtin_memcpy(w, p, sizeof w); }
    // the first n (at most 8) of p, zeros behind them
    __device__ __forceinline__ void load(const E* p, int n) {
        if (n >= 8) {
            load(p);
            return;
        }
        zero();
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) {
                if constexpr (P == 1) w[i / 2] |= static_cast<uint32_t>(p[i]) << (16 * (i % 2));
                else w[i] = __float_as_uint(p[i]);
            }
    }
    // elements n.. moved to the front, zeros behind them
    __device__ __forceinline__ void drop(int n) {
        if (n >= 8) zero();
#pragma unroll
        for (int s = 1; s < 8; s *= 2)
            if (n & s)
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    const int by = P == 1 ? s / 2 : s;
                    if (P == 1 && s == 1) w[i] = w[i] >> 16 | (i + 1 < W ? w[i + 1 < W ? i + 1 : 0] << 16 : 0u);
                    else w[i] = i + by < W ? w[i + by < W ? i + by : 0] : 0u;
                }
    }
    __device__ __forceinline__ void planes(u32x4_t (&p)[P]) const {
        if constexpr (P == 1) {
#pragma unroll
            for (int i = 0; i < 4; ++i) p[0][i] = w[i];
        } else {
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(w[i]);
            split8<P>(x, p);
        }
    }
};

// ---- LDS tiles --------------------------------------------------------------------------------

// A token-major tile of Q or K, DK bf16 a row: the 16-byte chunk c of row r is at chunk c ^ kf(r)
// (pm_cdna4.h's tables: 16 rows' operand reads fall into different banks).
template <int DK>
__device__ __forceinline__ int kf(int r) {
    return DK == 64 ? kq_f<64>(r) : kq_f<128>(r);
}
template <int DK>
__device__ __forceinline__ u32x4_t op_row(const uint16_t* m, int row, int kb, int g) {
    return *reinterpret_cast<const u32x4_t*>(m + row * DK + 8 * ((4 * kb + g) ^ kf<DK>(row)));
}
// The V tile, NT bf16 a row.  128: as K's.  64 (8 chunks): rows r and r + 1 lie in different halves of
// the banks, the four pairs of rows r, r + 2, r + 4, r + 6 in different quarters of a half for any pair
// of chunks.
template <int NT>
__device__ __forceinline__ int vf(int r) {
    return NT == 64 ? 2 * ((r >> 1) & 3) : kq_f<128>(r);
}

// Transposed reads, waited for in the same block: N 8-byte reads from addr + the offsets.
template <int O0, int O1>
__device__ __forceinline__ void tr2(unsigned addr, u32x2_t& a, u32x2_t& b) {
    __asm__ volatile("ds_read_b64_tr_b16 %0, %2 offset:%3\n\tds_read_b64_tr_b16 %1, %2 offset:%4\n\t"
                     "s_waitcnt lgkmcnt(0)"
                     : "=&v"(a), "=&v"(b) : "v"(addr), "n"(O0), "n"(O1) : "memory");
}
template <int O0, int O1, int O2, int O3, int O4, int O5, int O6, int O7>
__device__ __forceinline__ void tr8(unsigned addr, u32x2_t (&r)[8]) {
    __asm__ volatile("ds_read_b64_tr_b16 %0, %8 offset:%9\n\tds_read_b64_tr_b16 %1, %8 offset:%10\n\t"
                     "ds_read_b64_tr_b16 %2, %8 offset:%11\n\tds_read_b64_tr_b16 %3, %8 offset:%12\n\t"
                     "ds_read_b64_tr_b16 %4, %8 offset:%13\n\tds_read_b64_tr_b16 %5, %8 offset:%14\n\t"
                     "ds_read_b64_tr_b16 %6, %8 offset:%15\n\tds_read_b64_tr_b16 %7, %8 offset:%16\n\t"
                     "s_waitcnt lgkmcnt(0)"
                     : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(r[4]), "=&v"(r[5]), "=&v"(r[6]),
                       "=&v"(r[7])
                     : "v"(addr), "n"(O0), "n"(O1), "n"(O2), "n"(O3), "n"(O4), "n"(O5), "n"(O6), "n"(O7)
                     : "memory");
}
template <int O0, int O1, int O2, int O3>
__device__ __forceinline__ void tr4(unsigned addr, u32x2_t& a, u32x2_t& b, u32x2_t& c, u32x2_t& d) {
    __asm__ volatile("ds_read_b64_tr_b16 %0, %4 offset:%5\n\tds_read_b64_tr_b16 %1, %4 offset:%6\n\t"
                     "ds_read_b64_tr_b16 %2, %4 offset:%7\n\tds_read_b64_tr_b16 %3, %4 offset:%8\n\t"
                     "s_waitcnt lgkmcnt(0)"
                     : "=&v"(a), "=&v"(b), "=&v"(c), "=&v"(d)
                     : "v"(addr), "n"(O0), "n"(O1), "n"(O2), "n"(O3) : "memory");
}
__device__ __forceinline__ u32x4_t join(u32x2_t a, u32x2_t b) {
    const u32x4_t r = {a.x, a.y, b.x, b.y};
    return r;
}

// The larger halves of two pairs, as unsigned numbers.
__device__ __forceinline__ uint32_t max_halves(uint32_t a, uint32_t b) {
    typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, a), __builtin_bit_cast(u16x2_t, b)));
}

// The same number, as one the compiler knows nothing of: what is computed from it is computed where it is
// used, not ahead of the loop, where it would take a register (or scratch memory, whose loads wait for
// the rows that are on their way: the backward of B4 T4096 H16 D128 takes 549 us without, 467 so).
__device__ __forceinline__ int fresh(int x) {
    __asm__ volatile("" : "+v"(x));
    return x;
}

// ---- log-decays -------------------------------------------------------------------------------

template <int CTRL, int ROW_MASK>
__device__ __forceinline__ double dpp_add_f64(double x) {
    const int lo = __builtin_amdgcn_update_dpp(0, __double2loint(x), CTRL, ROW_MASK, 0xF, false);
    const int hi = __builtin_amdgcn_update_dpp(0, __double2hiint(x), CTRL, ROW_MASK, 0xF, false);
    return x + __hiloint2double(hi, lo);
}
// Inclusive prefix sum over the wave's lanes, as wave_prefix_sum.
__device__ __forceinline__ double wave_prefix_f64(double x) {
    x = dpp_add_f64<0x111, 0xF>(x);
    x = dpp_add_f64<0x112, 0xF>(x);
    x = dpp_add_f64<0x114, 0xF>(x);
    x = dpp_add_f64<0x118, 0xF>(x);
    x = dpp_add_f64<0x142, 0xA>(x);
    return dpp_add_f64<0x143, 0xC>(x);
}
// A log-decay in units of log 2, within +-200 (2^-200 is 0 in fp32 and 2^200 infinite; a chunk's sum
// stays below 2^14); NaN stays NaN.
__device__ __forceinline__ double log2_decay(float g) {
    const double x = g * kLog2e;
    return x < -200.0 ? -200.0 : x > 200.0 ? 200.0 : x;
}
__device__ __forceinline__ float2 split_log(double x) {
    const float hi = static_cast<float>(rint(x * 1024.0) * (1.0 / 1024.0));
    return make_float2(hi, static_cast<float>(x - hi));
}
__device__ __forceinline__ float exp2_diff(float2 a, float2 b) {
    return exp2_hw((a.x - b.x) + (a.y - b.y));
}
__device__ __forceinline__ float exp2_f64(double x) {
    return exp2_hw(static_cast<float>(x));
}

// ---- the pass ---------------------------------------------------------------------------------
//
// A workgroup walks through one span of a sequence for one head (or a group of heads that share their
// K and V, or their Q), NT = 64 CT columns of the state: wave w keeps 16 CT of them for all DK rows in
// accumulators, 16 CT columns of O for the chunk, and a quarter of A's tiles, which the waves exchange
// through LDS.  Two column tiles a wave (DK >= 128) halve the LDS reads of Q and K^T per product, which
// bound the kernel with one (forward of B4 T4096 H16 D128: 156 us with one, LDS at 220 KB a chunk and 64
// columns, 135 with two).
// The next chunk's rows are loaded into registers while this one's products run.

// What a launch of decay_pass does besides its outputs.
enum { kPassPlain = 0, kPassPart = 1, kPassState = 2 };

template <int DK>
struct DecayTile {
    static constexpr int CT = DK >= 128 ? 2 : 1, NT = 64 * CT;
};

template <int P, int DK, int KIND>
__global__ __launch_bounds__(256, KIND == kPassState || DK < 256 ? 2 : 1) void decay_pass(DecayPasses passes) {
    using Sh = DecayShape<P>;
    constexpr int C = Sh::C, PA = Sh::PA, MT = Sh::MT, KB = DK / 32, MD = DK / 16;
    constexpr int CT = DecayTile<DK>::CT, NT = DecayTile<DK>::NT;
    constexpr int UQ = C * DK / 2048, UV = C * NT / 2048;  // 8-element units per thread
    constexpr int RQ = 2048 / DK, RV = 2048 / NT;          // rows between a thread's units
    constexpr bool OUT = KIND != kPassState, AUX = KIND == kPassPart;
    constexpr int PS = AUX ? 3 : PA;  // planes of the state as a factor
    constexpr int CS = AUX ? 1 : CT;  // column tiles whose planes are held at once (three of both spill 32 registers)
    constexpr int PC = 3;  // planes of the decayed V, which sums into the state
    using E = typename std::conditional<P == 1, uint16_t, float>::type;

    __shared__ __attribute__((aligned(16))) uint16_t sq[OUT ? P * C * DK : 8];
    __shared__ __attribute__((aligned(16))) uint16_t sk[P * C * DK];
    __shared__ __attribute__((aligned(16))) uint16_t sv[P * C * NT];
    __shared__ __attribute__((aligned(16))) uint16_t sa[OUT ? PA * Sh::BLK * 512 : 8];
    __shared__ float2 sg[2][C];                  // the sums G, split
    __shared__ float s_into[2][C], s_out[2][C];  // e^{G_i} and e^{G_C - G_j}, with their scales
    __shared__ double s_total[2];
    __shared__ float s_part[AUX ? 4 : 1][AUX ? C : 1];

    const int t = threadIdx.x, lane = t & 63, l16 = lane & 15, lg = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(t >> 6);

    // workgroups of one head's passes and column tiles are 8 apart: on one XCD, they share its L2's lines
    const unsigned id = blockIdx.x, rest = id >> 3, n_tiles = passes.pass[0].n_tiles;
    const DecayPass& a = passes.pass[rest % passes.n];
    const int tile = static_cast<int>(rest / passes.n % n_tiles);
    const int64_t unit = static_cast<int64_t>(rest / passes.n / n_tiles) * 8 + (id & 7);
    const int groups = OUT ? a.HO / a.n_dst : a.HS;  // head groups (the states' pass: one per state)
    if (unit >= static_cast<int64_t>(a.n_slots_grid) * groups) return;
    const int slot_id = static_cast<int>(unit / groups), hg = static_cast<int>(unit % groups);
    const int ho0 = OUT ? hg * a.n_dst : hg;
    const int hs = OUT ? ho0 / (a.HO / a.HS) : hg;   // the state's head
    const int n_src = a.HK / a.HS, n_dst = OUT ? a.n_dst : 1, n_m = n_src * n_dst;
    const int n0 = tile * NT;

    // the sequence and this workgroup's span of it
    int seq, order;
    int64_t start = 0, rows0 = 0;
    int len = a.T;
    const E *qp = static_cast<const E*>(a.q), *kp = static_cast<const E*>(a.k), *vp = static_cast<const E*>(a.v);
    const E* xp = static_cast<const E*>(a.aux);
    const float* gp = a.g + hs;
    if (a.cu) {
        const int2 so = a.slot_table[slot_id];
        seq = so.x, order = so.y;
        if (seq < 0) return;
        const int z0 = min(max(a.cu[seq], 0), a.T), z1 = min(max(a.cu[seq + 1], 0), a.T);
        start = rows0 = z0;
        len = max(z1 - z0, 0);
    } else {
        seq = slot_id / a.n_spans, order = slot_id % a.n_spans;
        qp += seq * a.q_sb, kp += seq * a.k_sb, vp += seq * a.v_sb, gp += seq * a.g_sb, xp += seq * a.x_sb;
        rows0 = static_cast<int64_t>(seq) * a.T;
    }
    const int n_spans = spans_of(len, a.span);
    // (the last span's share is not wanted; where malformed offsets overlap, a next slot may be missing)
    if (!OUT && (order + 1 >= n_spans || slot_id + 1 >= a.n_slots_grid)) return;
    const int my_span = a.reverse ? n_spans - 1 - order : order;
    const int c_begin = my_span * a.span;  // first token, relative to the sequence
    const int c_end = span_end(c_begin, a.span, len);
    const int n_chunks = (c_end - c_begin + C - 1) / C;
    const int64_t state_pair = static_cast<int64_t>(seq) * a.HS + hs;

    // ---- the state before the span.  Tile ct of wave w: columns n(ct, l16), rows s_row_d(md, 4 lg + r);
    // two tiles take turns every 4 columns, so that a lane's outputs of both are 8 columns in a row
    int n_col[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
        n_col[ct] = n0 + (CT == 1 ? 16 * w + l16 : 32 * w + 8 * (l16 >> 2) + 4 * ct + (l16 & 3));
    f32x4_t S[CT][MD];
    int64_t slot_pair = state_pair;
    bool stored = true;
    if (a.slots) {
        const int slot = a.slots[seq];
        stored = slot >= 0 && slot < a.n_slots;
        slot_pair = static_cast<int64_t>(stored ? slot : 0) * a.HS + hs;
        if (OUT && !stored && a.bad_slot && t == 0) *a.bad_slot = 1;
    }
    {
        const float* from = nullptr;
        int64_t row = a.s_row, col = a.s_col;
        if (OUT && a.span_state) {
            from = a.span_state + (static_cast<int64_t>(slot_id) * a.HS + hs) * a.D * a.D;
            row = a.u_row, col = a.u_col;
        } else if (OUT && a.s0 && (stored || a.s0_gathered)) {
            from = a.s0 + (a.s0_gathered ? state_pair : slot_pair) * a.D * a.D;
        }
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
#pragma unroll
            for (int md = 0; md < MD; ++md) {
                S[ct][md] = f32x4_t{0.f, 0.f, 0.f, 0.f};
                if (!from) continue;
                const int d0 = s_row_d(md, 4 * lg);
                const float* p = from + d0 * row + n_col[ct] * col;
                if (row == 1 && a.D % 4 == 0) {
                    if (d0 < a.D && n_col[ct] < a.D) __builtin_memcpy(&S[ct][md], p, 16);
                } else {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (d0 + r < a.D && n_col[ct] < a.D) S[ct][md][r] = p[r * row];
                }
            }
    }

    // halves of A's blocks that no tile covers
    if (OUT && w == 0)
#pragma unroll
        for (int p = 0; p < PA; ++p)
#pragma unroll
            for (int i = 0; i < MT; i += 2) zero_upper_half(sa + p * Sh::BLK * 512, qblk(i, i >> 1), lane);

    // ---- loads of one step (a chunk and one of its heads) into registers.  Every lane loads, from a row
    // and columns that are there, and what is not to be seen is cut off on the way to LDS: with branches
    // around the loads the compiler merges registers behind them, and so waits for what was to arrive
    // while the products run (22,000 cycles a chunk instead of 13,000).
    const int row_q = t / (DK / 8), col_q = 8 * (t % (DK / 8)), row_v = t / (NT / 8), col_v = n0 + 8 * (t % (NT / 8));
    const int at_q = max(min(col_q, a.D - 8), 0), at_v = max(min(col_v, a.D - 8), 0);
    const uint32_t q_sb = a.q_st * sizeof(E), k_sb = a.k_st * sizeof(E), v_sb = a.v_st * sizeof(E);  // (64 of them fit)
    const bool tiny = a.D < 8;  // (rows too short for such a load: element by element, later)
    Raw8<P> rq[OUT ? UQ : 1], rk[UQ], rv[UV];
    auto chunk_at = [&](int c, int& first, int& cnt) {  // tokens relative to the sequence
        const int k = a.reverse ? n_chunks - 1 - c : c;
        first = c_begin + k * C;
        cnt = min(C, c_end - first);
    };
    struct Src {
        const E *q, *k, *v;  // the chunk's first token in memory
    };
    qp += start * a.q_st + ho0 * a.q_sh;
    kp += start * a.k_st + static_cast<int64_t>(hs) * n_src * a.k_sh;
    vp += start * a.v_st + static_cast<int64_t>(hs) * n_src * a.v_sh;
    auto source = [&](int first, int m) {
        const int mq = n_dst > 1 ? m : 0, mk = n_dst > 1 ? 0 : m;
        return Src{qp + first * a.q_st + mq * a.q_sh, kp + first * a.k_st + mk * a.k_sh,
                   vp + first * a.v_st + mk * a.v_sh};
    };
    auto token_of = [&](int row, int cnt) { return a.reverse ? cnt - 1 - row : row; };
    auto fetch = [&](int c, int m) {
        // (registers that a step does not load are cleared, so that none is kept from step to step)
        if (tiny || c >= n_chunks || (n_dst > 1 && m > 0)) {
#pragma unroll
            for (int i = 0; i < UQ; ++i) rk[i].zero();
#pragma unroll
            for (int i = 0; i < UV; ++i) rv[i].zero();
        }
        if (!OUT || tiny || c >= n_chunks || (n_dst == 1 && m > 0)) {
#pragma unroll
            for (int i = 0; i < UQ; ++i) rq[OUT ? i : 0].zero();
        }
        if (tiny || c >= n_chunks) return;
        int first, cnt;
        chunk_at(c, first, cnt);
        const Src src = source(first, m);
        if (n_dst == 1 || m == 0) {
#pragma unroll
            for (int i = 0; i < UQ; ++i) {
                const uint32_t tok = token_of(min(row_q + i * RQ, cnt - 1), cnt);
                rk[i].load(reinterpret_cast<const char*>(src.k) + (tok * k_sb + static_cast<uint32_t>(at_q * sizeof(E))));
            }
#pragma unroll
            for (int i = 0; i < UV; ++i) {
                const uint32_t tok = token_of(min(row_v + i * RV, cnt - 1), cnt);
                rv[i].load(reinterpret_cast<const char*>(src.v) + (tok * v_sb + static_cast<uint32_t>(at_v * sizeof(E))));
            }
        }
        if (OUT && (n_dst > 1 || m == 0))
#pragma unroll
            for (int i = 0; i < UQ; ++i) {
                const uint32_t tok = token_of(min(row_q + i * RQ, cnt - 1), cnt);
                rq[OUT ? i : 0].load(reinterpret_cast<const char*>(src.q) +
                                     (tok * q_sb + static_cast<uint32_t>(at_q * sizeof(E))));
            }
    };
    // one of them on its way to LDS
    auto cut = [&](Raw8<P>& x, int row, int cnt, int col, int at, const E* p, int64_t st) {
        if (tiny && row < cnt) x.load(p + token_of(row, cnt) * st + col, a.D - col);
        if (row >= cnt || col >= a.D) x.zero();
        else if (!tiny && col != at) x.drop(col - at);
    };
    // wave 0 has the log-decays: chunk c's are loaded and summed while chunk c - 1 runs
    auto load_g = [&](int c) {  // (a value that is there; sum_g takes it for what it is)
        int first, cnt;
        chunk_at(min(c, n_chunks - 1), first, cnt);
        const int tok = a.reverse ? first + cnt - t : first + t;  // (backwards: the token after)
        return gp[(start + max(min(tok, len - 1), 0)) * a.g_st];
    };
    auto sum_g = [&](int c, float rg) {
        int first, cnt;
        chunk_at(min(c, n_chunks - 1), first, cnt);
        const int buf = c & 1;
        const bool there = t < cnt && (a.reverse ? first + cnt - t : first + t) < len;
        const double G = wave_prefix_f64(there ? log2_decay(rg) : 0.0);
        const double last = __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(G), 63),
                                             __builtin_amdgcn_readlane(__double2loint(G), 63));
        const int i = fresh(t);
        if (i < C) {
            sg[buf][i] = split_log(G);
            s_into[buf][i] = exp2_f64(G) * a.into_scale;
            s_out[buf][i] = exp2_f64(last - G) * a.out_scale;
        }
        if (t == 0) s_total[buf] = last;
    };

    f32x4_t O[CT][MT];
    double log_total = 0.0;
    fetch(0, 0);
    if (w == 0 && n_chunks > 0) sum_g(0, load_g(0));
    for (int c = 0, m = 0; c < n_chunks;) {
        const int buf = c & 1, m_next = m + 1 < n_m ? m + 1 : 0, c_next = m_next ? c : c + 1;
        const bool first_m = m == 0, last_m = m == n_m - 1, dst = n_dst > 1;
        int first, cnt;
        chunk_at(c, first, cnt);
        const int ho = ho0 + (dst ? m : 0);
        // ---- registers to LDS
        const bool whole = cnt == C && a.D == DK;
        Src src{};
        if (!whole) src = source(first, m);
        if (!dst || first_m) {
#pragma unroll
            for (int i = 0; i < UQ; ++i) {
                const int row = row_q + i * RQ, ch = (t % (DK / 8)) ^ kf<DK>(row);
                if (!whole) cut(rk[i], row, cnt, col_q, at_q, src.k, a.k_st);
                u32x4_t p[P];
                rk[i].planes(p);
#pragma unroll
                for (int x = 0; x < P; ++x) *reinterpret_cast<u32x4_t*>(sk + x * C * DK + row * DK + 8 * ch) = p[x];
            }
#pragma unroll
            for (int i = 0; i < UV; ++i) {
                const int row = row_v + i * RV, ch = (t % (NT / 8)) ^ vf<NT>(row);
                if (!whole) cut(rv[i], row, cnt, col_v, at_v, src.v, a.v_st);
                u32x4_t p[P];
                rv[i].planes(p);
#pragma unroll
                for (int x = 0; x < P; ++x) *reinterpret_cast<u32x4_t*>(sv + x * C * NT + row * NT + 8 * ch) = p[x];
            }
        }
        if (OUT && (dst || first_m))
#pragma unroll
            for (int i = 0; i < UQ; ++i) {
                const int row = row_q + i * RQ, ch = (t % (DK / 8)) ^ kf<DK>(row);
                if (!whole) cut(rq[OUT ? i : 0], row, cnt, col_q, at_q, src.q, a.q_st);
                u32x4_t p[P];
                rq[OUT ? i : 0].planes(p);
#pragma unroll
                for (int x = 0; x < P; ++x) *reinterpret_cast<u32x4_t*>(sq + x * C * DK + row * DK + 8 * ch) = p[x];
            }
        lds_barrier();
        const float rg = load_g(c + 1);  // (by every wave: a branch around it would wait; summed below)
        if (!OUT) fetch(c_next, m_next);

        const double chunk_log = s_total[buf];
        // ---- A's tiles of the wave's 16 source tokens and, from the same rows of Q, the state's part of
        // the outputs (in a chunk's later heads of a group with shared Q: A alone)
        f32x4_t A[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) A[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        if (dst || first_m) {
            if (OUT) {
                constexpr int XN = 4 * CT;  // a lane's columns in a row
                uint32_t aux[AUX ? MT : 1][P == 1 ? XN / 2 : XN];  // as they are in memory
                const int x_col = n0 + (CT == 1 ? 16 * w + 4 * lg : 32 * w + 8 * lg);
                const bool x_wide = a.D % XN == 0;
                const E* x_p = xp + (start + first) * a.x_st + static_cast<int64_t>(ho) * a.x_sh;
                const bool parts = AUX && a.part;
                if (parts && x_wide)
                    // (rows and columns that are not there: some that are, since their O is 0)
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
                        const uint32_t tok = token_of(min(16 * i + (fresh(t) & 15), cnt - 1), cnt);
                        __builtin_memcpy(aux[AUX ? i : 0],
                                         reinterpret_cast<const char*>(x_p) +
                                             (tok * static_cast<uint32_t>(a.x_st * sizeof(E)) +
                                              static_cast<uint32_t>(min(x_col, a.D - XN) * sizeof(E))),
                                         sizeof aux[0]);
                    }
#pragma unroll
                for (int ct = 0; ct < CT; ++ct)
#pragma unroll
                    for (int i = 0; i < MT; ++i) O[ct][i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) {
                    u32x4_t so[CS][PS], qo[MT][P], ko[P];
#pragma unroll
                    for (int i = 0; i < MT; ++i)
#pragma unroll
                        for (int p = 0; p < P; ++p) qo[i][p] = op_row<DK>(sq + p * C * DK, 16 * i + l16, kb, lg);
#pragma unroll
                    for (int p = 0; p < P; ++p) ko[p] = op_row<DK>(sk + p * C * DK, 16 * (w % MT) + l16, kb, lg);
                    auto split_state = [&](int c0) {
#pragma unroll
                        for (int ct = 0; ct < CS; ++ct) {
                            const f32x4_t s0 = S[c0 + ct][2 * kb], s1 = S[c0 + ct][2 * kb + 1];
                            const float s8[8] = {s0[0], s0[1], s0[2], s0[3], s1[0], s1[1], s1[2], s1[3]};
                            split8<PS>(s8, so[ct]);
                        }
                    };
                    if (!AUX) split_state(0);
#pragma unroll
                    for (int x = P - 1; x >= 0; --x)
#pragma unroll
                        for (int p = 0; p < P; ++p)
                            if (x - p >= 0)
#pragma unroll
                                for (int i = 0; i < MT; ++i)
                                    A[i] = mfma32(__builtin_bit_cast(bf16x8_t, ko[x - p]),
                                                  __builtin_bit_cast(bf16x8_t, qo[i][p]), A[i]);
#pragma unroll
                    for (int c0 = 0; c0 < CT; c0 += CS) {
                        if (AUX) split_state(c0);
#pragma unroll
                        for (int x = PS - 1; x >= 0; --x)  // (the small products first, all tiles of one before the next)
#pragma unroll
                            for (int p = 0; p < P; ++p)
                                if (x - p >= 0)
#pragma unroll
                                    for (int ct = 0; ct < CS; ++ct)
#pragma unroll
                                        for (int i = 0; i < MT; ++i)
                                            O[c0 + ct][i] = mfma32(__builtin_bit_cast(bf16x8_t, so[ct][x - p]),
                                                                   __builtin_bit_cast(bf16x8_t, qo[i][p]), O[c0 + ct][i]);
                    }
                }
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    const float e = s_into[buf][16 * i + (fresh(t) & 15)];
#pragma unroll
                    for (int ct = 0; ct < CT; ++ct) O[ct][i] *= e;
                }
                if (parts && !x_wide)
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
                        const int row = 16 * i + (fresh(t) & 15), left = row < cnt ? a.D - x_col : 0;
                        const E* x = x_p + token_of(min(row, cnt - 1), cnt) * a.x_st + x_col;
#pragma unroll
                        for (int r = 0; r < XN; ++r) {
                            if constexpr (P == 1) {
                                const uint32_t v = r < left ? x[r] : 0;
                                aux[AUX ? i : 0][r / 2] = r % 2 ? aux[AUX ? i : 0][r / 2] | v << 16 : v;
                            } else {
                                aux[AUX ? i : 0][r] = r < left ? __float_as_uint(x[r]) : 0u;
                            }
                        }
                    }
                if (parts) {
                    // each token's product of that part with the row of `aux` (q for gq, k for gk)
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
                        float sum = 0.f;
#pragma unroll
                        for (int r = 0; r < XN; ++r) {
                            const uint32_t v = P == 1 ? (r % 2 ? aux[AUX ? i : 0][r / 2] & 0xffff0000u : aux[AUX ? i : 0][r / 2] << 16) : aux[AUX ? i : 0][r % (P == 1 ? 1 : XN)];
                            sum += __uint_as_float(v) * O[r / 4][i][r % 4];
                        }
                        sum += __shfl_xor(sum, 16);
                        sum += __shfl_xor(sum, 32);
                        if (lg == 0) s_part[AUX ? w : 0][AUX ? 16 * i + (fresh(t) & 15) : 0] = sum;
                    }
                }
            }
        }
        if (OUT) {
            if (!dst && !first_m)
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) {
                    u32x4_t qo[MT][P], ko[P];
#pragma unroll
                    for (int p = 0; p < P; ++p) {
                        ko[p] = op_row<DK>(sk + p * C * DK, 16 * (w % MT) + l16, kb, lg);
#pragma unroll
                        for (int i = 0; i < MT; ++i) qo[i][p] = op_row<DK>(sq + p * C * DK, 16 * i + l16, kb, lg);
                    }
#pragma unroll
                    for (int x = P - 1; x >= 0; --x)
#pragma unroll
                        for (int p = 0; p < P; ++p)
                            if (x - p >= 0)
#pragma unroll
                                for (int i = 0; i < MT; ++i)
                                    A[i] = mfma32(__builtin_bit_cast(bf16x8_t, ko[x - p]),
                                                  __builtin_bit_cast(bf16x8_t, qo[i][p]), A[i]);
                }
            // as packed operands: lane (lg, l16) has A[16 i + l16][16 w + 4 lg + r]
            float2 gj[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) gj[r] = sg[buf][16 * (w % MT) + 4 * lg + r];
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                if (i < w) continue;  // (above the diagonal)
                const float2 gi = sg[buf][16 * i + (fresh(t) & 15)];
                f32x4_t x;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    x[r] = A[i][r] * (exp2_diff(gi, gj[r]) * a.a_scale);
                    if (i == w && 4 * lg + r > l16) x[r] = 0.f;
                }
                u32x2_t ap[PA];
                split4<PA>(x, ap);
                const int blk = i < 2 ? i : 2 * i - 2 + (w >> 1);  // (qblk)
#pragma unroll
                for (int p = 0; p < PA; ++p)
                    *reinterpret_cast<u32x2_t*>(sa + (p * Sh::BLK + blk) * 512 + (fresh(t) & 63) * 8 + 4 * (w & 1)) = ap[p];
            }
        }
        if (OUT && w == 0 && first_m) sum_g(c + 1, rg);
        if (first_m) log_total += chunk_log;
        const bool update = !dst || last_m;
        if (dst ? last_m : first_m) {
            const float e = exp2_f64(chunk_log);
#pragma unroll
            for (int ct = 0; ct < CT; ++ct)
#pragma unroll
                for (int md = 0; md < MD; ++md) S[ct][md] *= e;
        }
        // ---- V, and the state
        u32x4_t vo[MT / 2][CT][P];
        const int j4 = (lane >> 2) & 3, cc = lane & 3, row_t = 4 * lg + j4;  // of the transposed reads
#pragma unroll
        for (int kb = 0; kb < MT / 2; ++kb) {
            // V of tokens 32 kb + {4 lg + [0, 4), 16 + 4 lg + [0, 4)}, columns n(ct, l16)
            const unsigned va = lds_addr(sv + (32 * kb + row_t) * NT +
                                         (CT == 1 ? 8 * ((2 * w + (cc >> 1)) ^ vf<NT>(row_t)) + 4 * (cc & 1)
                                                  : 8 * ((4 * w + cc) ^ vf<NT>(row_t))));
            constexpr int R16 = 16 * NT * 2, VP = C * NT * 2;
            f32x4_t x0[CT], x1[CT];
            auto take = [&](int p, u32x2_t lo0, u32x2_t hi0, u32x2_t lo1, u32x2_t hi1) {
                vo[kb][0][p] = join(lo0, hi0);
                x0[0] = p == P - 1 ? widen4(lo0) : x0[0] + widen4(lo0);
                x1[0] = p == P - 1 ? widen4(hi0) : x1[0] + widen4(hi0);
                if (CT == 2) {
                    vo[kb][CT - 1][p] = join(lo1, hi1);
                    x0[CT - 1] = p == P - 1 ? widen4(lo1) : x0[CT - 1] + widen4(lo1);
                    x1[CT - 1] = p == P - 1 ? widen4(hi1) : x1[CT - 1] + widen4(hi1);
                }
            };
            u32x2_t b0, b1, b2 = {0u, 0u}, b3 = {0u, 0u};
            if constexpr (P == 3) {  // (the smallest parts first)
                if constexpr (CT == 1) tr2<2 * VP, 2 * VP + R16>(va, b0, b1);
                else tr4<2 * VP, 2 * VP + R16, 2 * VP + 8, 2 * VP + 8 + R16>(va, b0, b1, b2, b3);
                take(2 % P, b0, b1, b2, b3);
                if constexpr (CT == 1) tr2<VP, VP + R16>(va, b0, b1);
                else tr4<VP, VP + R16, VP + 8, VP + 8 + R16>(va, b0, b1, b2, b3);
                take(1 % P, b0, b1, b2, b3);
            }
            if constexpr (CT == 1) tr2<0, R16>(va, b0, b1);
            else tr4<0, R16, 8, 8 + R16>(va, b0, b1, b2, b3);
            take(0, b0, b1, b2, b3);
            if (!update) continue;
            u32x4_t wo[CT][PC];
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
                float v8[8];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    v8[r] = x0[ct][r] * s_out[buf][32 * kb + 4 * lg + r];
                    v8[4 + r] = x1[ct][r] * s_out[buf][32 * kb + 16 + 4 * lg + r];
                }
                split8<PC>(v8, wo[ct]);
            }
#pragma unroll
            for (int d32 = 0; d32 < KB; ++d32) {
                // K^T: rows 32 d32 + 8 .. (s_row_d of tiles 2 d32 and 2 d32 + 1), the same tokens
                const unsigned ka = lds_addr(sk + (32 * kb + row_t) * DK + 8 * ((4 * d32 + cc) ^ kf<DK>(row_t)));
                constexpr int K16 = 16 * DK * 2, KP = C * DK * 2;
                u32x4_t ko[2][P];
                u32x2_t a0, a1;
                tr4<0, K16, 8, 8 + K16>(ka, a0, a1, b0, b1);
                ko[0][0] = join(a0, a1), ko[1][0] = join(b0, b1);
                if constexpr (P == 3) {
                    u32x2_t x[8];
                    tr8<KP, KP + K16, KP + 8, KP + 8 + K16, 2 * KP, 2 * KP + K16, 2 * KP + 8, 2 * KP + 8 + K16>(ka, x);
                    ko[0][1] = join(x[0], x[1]), ko[1][1] = join(x[2], x[3]);
                    ko[0][2] = join(x[4], x[5]), ko[1][2] = join(x[6], x[7]);
                }
#pragma unroll
                for (int x = PC - 1; x >= 0; --x)
#pragma unroll
                    for (int p = 0; p < P; ++p)
                        if (x - p >= 0)
#pragma unroll
                            for (int ct = 0; ct < CT; ++ct)
#pragma unroll
                                for (int h = 0; h < 2; ++h)
                                    S[ct][2 * d32 + h] = mfma32(__builtin_bit_cast(bf16x8_t, ko[h][p]),
                                                                __builtin_bit_cast(bf16x8_t, wo[ct][x - p]),
                                                                S[ct][2 * d32 + h]);
            }
        }
        // ---- infinities and NaN of V stay out of A V, where A's zeros would carry them to tokens before theirs:
        // zeros go in their place, and from its first such token on a column comes out as NaN.  (No cost but
        // for the test; without its weight in the compiler's favour 24 us of the training step's 568 went
        // into registers that the branch takes.)
        if (OUT) {
            uint32_t most = 0;
#pragma unroll
            for (int kb = 0; kb < MT / 2; ++kb)
#pragma unroll
                for (int ct = 0; ct < CT; ++ct)
#pragma unroll
                    for (int x = 0; x < 4; ++x) most = max_halves(most, vo[kb][ct][0][x] & 0x7fff7fffu);
            if (__builtin_expect(__any((most & 0xffffu) >= 0x7f80u || most >= 0x7f800000u), 0)) {
#pragma unroll
                for (int ct = 0; ct < CT; ++ct) {
                    int from = C;  // the first such token of the lane's column
                    const int tok = 4 * (fresh(t) >> 4 & 3);
#pragma unroll
                    for (int kb = MT / 2 - 1; kb >= 0; --kb)
#pragma unroll
                        for (int x = 3; x >= 0; --x) {
                            const uint32_t v = vo[kb][ct][0][x] & 0x7fff7fffu;
                            const bool hi = v >= 0x7f800000u, lo = (v & 0xffffu) >= 0x7f80u;
                            from = hi ? tok + (32 * kb + 8 * (x / 2) * 2 + 2 * (x % 2) + 1) : from;
                            from = lo ? tok + (32 * kb + 8 * (x / 2) * 2 + 2 * (x % 2)) : from;
                            const uint32_t keep = (hi ? 0u : 0xffff0000u) | (lo ? 0u : 0xffffu);
#pragma unroll
                            for (int p = 0; p < P; ++p) vo[kb][ct][p][x] &= keep;
                        }
                    from = min(from, __shfl_xor(from, 16));
                    from = min(from, __shfl_xor(from, 32));
                    const int row = fresh(t) & 15;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int x = __shfl(from, tok + r) - row;
#pragma unroll
                        for (int i = 0; i < MT; ++i) O[ct][i][r] = 16 * i >= x ? __builtin_nanf("") : O[ct][i][r];
                    }
                }
            }
        }
        // (the next step's loads: after the products that need every register, before the wait for the other
        // waves; 179 us here, 184 before the state's products, 186 before all of them, 182 after A V, at B32
        // T1024 H16 D128.  A states' pass has registers to spare and asks before its products.)
        if (OUT) fetch(c_next, m_next);
        if (!OUT && w == 0 && first_m) sum_g(c + 1, rg);
        // (from here on nothing reads the chunk's rows or log-decays: the next ones may come in; A is
        // written again only after the barrier that follows them)
        lds_barrier();
        // ---- A V
        if (OUT)
#pragma unroll
            for (int kb = 0; kb < MT / 2; ++kb) {
                u32x4_t ao[MT][PA];
#pragma unroll
                for (int i = 2 * kb; i < MT; ++i)
#pragma unroll
                    for (int p = 0; p < PA; ++p)
                        ao[i][p] = *reinterpret_cast<const u32x4_t*>(sa + (p * Sh::BLK + qblk(i, kb)) * 512 + lane * 8);
#pragma unroll
                for (int x = PA - 1; x >= 0; --x)
#pragma unroll
                    for (int p = 0; p < P; ++p)
                        if (x - p >= 0)
#pragma unroll
                            for (int ct = 0; ct < CT; ++ct)
#pragma unroll
                                for (int i = 2 * kb; i < MT; ++i)
                                    O[ct][i] = mfma32(__builtin_bit_cast(bf16x8_t, vo[kb][ct][p]),
                                                      __builtin_bit_cast(bf16x8_t, ao[i][x - p]), O[ct][i]);
            }
        // ---- outputs
        if (OUT && (dst || last_m)) {
            const int col = n0 + (CT == 1 ? 16 * w + 4 * lg : 32 * w + 8 * lg), left = a.D - col;
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const int row = 16 * i + (fresh(t) & 15);
                if (row >= cnt || left <= 0) continue;
                const int64_t at = ((rows0 + first + token_of(row, cnt)) * a.HO + ho) * a.D + col;
                float v[4 * CT];
#pragma unroll
                for (int r = 0; r < 4 * CT; ++r) v[r] = O[r / 4][i][r % 4];
                if (a.out_bf16) {
                    uint16_t* o = static_cast<uint16_t*>(a.o) + at;
                    uint32_t p[2 * CT];
#pragma unroll
                    for (int r = 0; r < 2 * CT; ++r) p[r] = pack2(v[2 * r], v[2 * r + 1]);
                    if (left >= 4 * CT) __builtin_memcpy(o, p, sizeof p);
                    else
#pragma unroll
                        for (int r = 0; r < 4 * CT; ++r)
                            if (r < left) o[r] = static_cast<uint16_t>(p[r / 2] >> (16 * (r & 1)));
                } else {
                    float* o = static_cast<float*>(a.o) + at;
                    if (left >= 4 * CT) __builtin_memcpy(o, v, sizeof v);
                    else
#pragma unroll
                        for (int r = 0; r < 4 * CT; ++r)
                            if (r < left) o[r] = v[r];
                }
            }
        }
        if constexpr (AUX)
            if (a.part && (dst || first_m) && t < cnt) {
                const int i = fresh(t);
                const int64_t tok = rows0 + first + token_of(i, cnt);
                a.part[(static_cast<int64_t>(tile) * a.HO + ho) * a.n_rows + tok] =
                    (s_part[0][i] + s_part[1][i]) + (s_part[2][i] + s_part[3][i]);
            }
        c = c_next, m = m_next;
    }

    // ---- the state after the span
    float* to = nullptr;
    int64_t row = a.s_row, col = a.s_col;
    float e = 1.f;
    if (!OUT) {  // (the next span's place: the scan over spans turns shares into states)
        to = a.span_state + (static_cast<int64_t>(slot_id + 1) * a.HS + hs) * a.D * a.D;
        row = a.u_row, col = a.u_col;
        if (tile == 0 && t == 0) a.span_log[static_cast<int64_t>(slot_id + 1) * a.HS + hs] = log_total;
    } else if (a.s_out && order == n_spans - 1 && ho0 % (a.HO / a.HS) == 0 && stored) {
        to = a.s_out + slot_pair * a.D * a.D;
        if (a.reverse && len > 0) e = exp2_f64(log2_decay(gp[start * a.g_st]));
    }
    if (to)
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
#pragma unroll
            for (int md = 0; md < MD; ++md) {
                const int d0 = s_row_d(md, 4 * lg);
                float* p = to + d0 * row + n_col[ct] * col;
                S[ct][md] *= e;
                if (row == 1 && a.D % 4 == 0) {
                    if (d0 < a.D && n_col[ct] < a.D) __builtin_memcpy(p, &S[ct][md], 16);
                } else {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (d0 + r < a.D && n_col[ct] < a.D) p[r * row] = S[ct][md][r];
                }
            }
}

// ---- dL/dg ------------------------------------------------------------------------------------
//
// dL/dg_t sums, over all pairs of a token j < t and a token i >= t, what j contributes through i
// (and what the first state and the last state's gradient add).  Per chunk: pairs inside it from
// the products (q_i . k_j)(go_i . v_j) e^{G_i - G_j}; pairs with j before it or i behind it from the
// two passes' products r_i, c_j; pairs around the whole chunk from the gradient at its span's first
// token, e^g <the state before it, the gradient of the state behind it>, which is handed on from chunk
// to chunk: no sum is taken as a difference of others over more than a span's 512 tokens.
//
// This kernel has the pairs inside chunks, one wave a chunk, from all four tensors once more.  (With
// q's rows as a fourth tile of gq's pass instead, whose registers are full, that pass took 146 us
// longer at B4 T4096 H16 D128.)  WIDE: D is a multiple of 8, rows load without tests.
template <int P, bool WIDE>
__global__ __launch_bounds__(256, P == 1 ? 2 : 3) void decay_near(DecayNear a) {
    using Sh = DecayShape<P>;
    using E = typename Raw8<P>::E;
    constexpr int C = Sh::C, MT = Sh::MT, W = 4;
    __shared__ float sp[W][C][C + 1];
    __shared__ float2 sg[W][C];
    const int t = threadIdx.x, lane = t & 63, l16 = lane & 15, lg = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(t >> 6);
    const int n_blocks = (a.T + W * C - 1) / (W * C);
    const int64_t id = blockIdx.x;
    const int hq = static_cast<int>(id % a.Hq), h = hq / (a.Hq / a.H);
    const int64_t b = id / a.Hq / n_blocks;
    const int first = (static_cast<int>(id / a.Hq % n_blocks) * W + w) * C;
    const int cnt = min(C, a.T - first);  // (may be <= 0 for the last waves)

    const double x = lane < cnt ? log2_decay(a.g[b * a.g_sb + (first + lane) * a.g_st + h]) : 0.0;
    const double sum = wave_prefix_f64(x);
    if (lane < C) sg[w][lane] = split_log(sum);
    f32x4_t x1[Sh::TRI], x2[Sh::TRI];
#pragma unroll
    for (int i = 0; i < Sh::TRI; ++i) x1[i] = x2[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    if (cnt > 0) {
        const E* kp = static_cast<const E*>(a.k) + b * a.k_sb + first * a.k_st + h * a.k_sh;
        const E* vp = static_cast<const E*>(a.v) + b * a.v_sb + first * a.v_st + h * a.v_sh;
        const E* qp = static_cast<const E*>(a.q) + b * a.q_sb + first * a.q_st + hq * a.q_sh;
        const E* op = static_cast<const E*>(a.go) + b * a.go_sb + first * a.go_st + hq * a.go_sh;
        for (int c0 = 0; c0 < a.D; c0 += 32) {
            const int col = c0 + 8 * lg;
            // (rows and columns that are there, cleared afterwards where they stand for others)
            auto ask = [&](Raw8<P>(&r)[MT], const E* p, int64_t st) {
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    const E* at = p + min(16 * i + l16, cnt - 1) * st;
                    if constexpr (WIDE) r[i].load(at + min(col, a.D - 8));
                    else r[i].load(at + col, max(a.D - col, 0));
                }
            };
            auto ready = [&](Raw8<P>(&r)[MT], u32x4_t(&x)[MT][P]) {
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    if (16 * i + l16 >= cnt || col >= a.D) r[i].zero();
                    r[i].planes(x[i]);
                }
            };
            Raw8<P> r1[MT], r2[MT], r3[MT], r4[MT];
            ask(r1, kp, a.k_st);
            ask(r2, qp, a.q_st);
            ask(r3, vp, a.v_st);
            ask(r4, op, a.go_st);
            u32x4_t src[MT][P], dst[MT][P];
            ready(r1, src);
            ready(r2, dst);
#pragma unroll
            for (int i = 0, n = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j <= i; ++j, ++n) x1[n] = mfma_planes<P, P>(src[j], dst[i], x1[n]);
            ready(r3, src);
            ready(r4, dst);
#pragma unroll
            for (int i = 0, n = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j <= i; ++j, ++n) x2[n] = mfma_planes<P, P>(src[j], dst[i], x2[n]);
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0, n = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j <= i; ++j, ++n) {
            const int row = 16 * i + l16;
            const float2 gi = sg[w][row];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int col = 16 * j + 4 * lg + k;
                sp[w][row][col] = col < row ? x1[n][k] * x2[n][k] * exp2_diff(gi, sg[w][col]) : 0.f;
            }
        }
    __syncthreads();
    if (lane < C) {  // row by row: the sums over j < t, sixteen reads in flight
        float run = 0.f;
        for (int j = 0; j < C; j += 16) {
            float p[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) p[k] = sp[w][lane][j + k];
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                sp[w][lane][j + k] = run;
                run += j + k < lane ? p[k] : 0.f;  // (above the diagonal there may be anything)
            }
        }
    }
    __syncthreads();
    float near = 0.f;
    if (lane < C)
#pragma unroll 16
        for (int i = 0; i < C; ++i) near += i >= lane ? sp[w][i][lane] : 0.f;
    if (lane < cnt) a.near[hq * a.n_rows + b * a.T + first + lane] = a.scale * near;
}

template <int P, int DK>
hipError_t launch_pass(const DecayPasses& a, int kind, hipStream_t st) {
    int64_t units = 0;
    for (int i = 0; i < a.n; ++i) {
        const DecayPass& x = a.pass[i];
        units = std::max(units, static_cast<int64_t>(x.n_slots_grid) * (kind == kPassState ? x.HS : x.HO / x.n_dst));
    }
    const dim3 grid(static_cast<unsigned>((units + 7) / 8 * 8 * a.pass[0].n_tiles * a.n));
    switch (kind) {
        case kPassPlain: hipLaunchKernelGGL((decay_pass<P, DK, kPassPlain>), grid, dim3(256), 0, st, a); break;
        case kPassPart: hipLaunchKernelGGL((decay_pass<P, DK, kPassPart>), grid, dim3(256), 0, st, a); break;
        default: hipLaunchKernelGGL((decay_pass<P, DK, kPassState>), grid, dim3(256), 0, st, a); break;
    }
    return hipGetLastError();
}

template <int P>
hipError_t run_pass(const DecayPasses& a, int kind, hipStream_t st) {
    const int D = a.pass[0].D;
    if (D <= 64) return launch_pass<P, 64>(a, kind, st);
    if (D <= 128) return launch_pass<P, 128>(a, kind, st);
    return launch_pass<P, 256>(a, kind, st);
}

template <int P>
hipError_t run_near(const DecayNear& a, hipStream_t st) {
    const int64_t n = static_cast<int64_t>(a.B) * a.Hq * ((a.T + 4 * DecayShape<P>::C - 1) / (4 * DecayShape<P>::C));
    const dim3 grid(static_cast<unsigned>(n));
    if (a.D % 8 == 0) hipLaunchKernelGGL((decay_near<P, true>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((decay_near<P, false>), grid, dim3(256), 0, st, a);
    return hipGetLastError();
}

}  // namespace
}  // namespace pm
