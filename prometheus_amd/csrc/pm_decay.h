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
// Products run on bf16 MFMA.  A value of more than 8 bits is a sum of bf16 planes (hi, next, ...),
// a product of two such sums the products of their planes down to the last plane's size: bf16 inputs
// are one plane and exact; A, S and the decayed V are two planes next to them (a relative error of
// 2^-17 at most, against 2^-9 with one: fp32 states and the gates' gradients need it); fp32 inputs
// and everything else next to them are three (2^-25).  On this card six such bf16 products take 6/16
// of the time of the fp32 MFMA.
//
// Log-decays are summed in 64 bits, and kept as a multiple of 2^-10 and a rest, so that a
// difference G_i - G_j has fp32's relative error also where both are large (behind a closed gate).
#pragma once

#include <type_traits>

#include "pm_cdna4.h"
#include "pm_decay_args.h"

namespace pm {
namespace {

template <int P>
struct DecayShape {
    static constexpr int C = P == 1 ? 64 : 32;   // tokens of a chunk (three planes of 64 would not fit LDS)
    static constexpr int PC = P == 1 ? 2 : 3;    // planes of computed operands
    static constexpr int MT = C / 16;            // 16-token tiles
    static constexpr int TRI = MT * (MT + 1) / 2;  // lower 16x16 tiles of A
    static constexpr int BLK = P == 1 ? 6 : 2;   // packed operand blocks of A (qblk)
};

constexpr int kDecayCols = 64;  // columns of the state per workgroup: 16 per wave
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

// Eight elements of a row as they are in memory (P 1: bf16, P 3: fp32), zeros past `n` of them.
template <int P>
struct Raw8 {
    uint32_t w[P == 1 ? 4 : 8];
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < (P == 1 ? 4 : 8); ++i) w[i] = 0;
    }
    __device__ __forceinline__ void load(const void* base, int64_t at, int n) {
        using E = typename std::conditional<P == 1, uint16_t, float>::type;
        const E* p = static_cast<const E*>(base) + at;
        if (n >= 8) {
            __builtin_memcpy(w, p, sizeof w);  // (any alignment of the elements)
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
// The V tile, 64 bf16 (8 chunks) a row: rows r and r + 1 lie in different halves of the banks, the
// four pairs of rows r, r + 2, r + 4, r + 6 in different quarters of a half for any pair of chunks.
__device__ __forceinline__ int vf(int r) { return 2 * ((r >> 1) & 3); }

// Transposed reads, waited for in the same block: N 8-byte reads from addr + the offsets.
template <int O0, int O1>
__device__ __forceinline__ void tr2(unsigned addr, u32x2_t& a, u32x2_t& b) {
    __asm__ volatile("ds_read_b64_tr_b16 %0, %2 offset:%3\n\tds_read_b64_tr_b16 %1, %2 offset:%4\n\t"
                     "s_waitcnt lgkmcnt(0)"
                     : "=&v"(a), "=&v"(b) : "v"(addr), "n"(O0), "n"(O1) : "memory");
}
template <int O0, int O1, int O2, int O3>
__device__ __forceinline__ void tr4(unsigned addr, u32x2_t& a, u32x2_t& b, u32x2_t& c, u32x2_t& d) {
    __asm__ volatile("ds_read_b64_tr_b16 %0, %4 offset:%5\n\tds_read_b64_tr_b16 %1, %4 offset:%6\n\t"
                     "ds_read_b64_tr_b16 %2, %4 offset:%7\n\tds_read_b64_tr_b16 %3, %4 offset:%8\n\t"
                     "s_waitcnt lgkmcnt(0)"
                     : "=&v"(a), "=&v"(b), "=&v"(c), "=&v"(d)
                     : "v"(addr), "n"(O0), "n"(O1), "n"(O2), "n"(O3) : "memory");
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
__device__ __forceinline__ u32x4_t join(u32x2_t a, u32x2_t b) {
    const u32x4_t r = {a.x, a.y, b.x, b.y};
    return r;
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

// (i, j) of lower tile number x: 0 (0,0), 1 (1,0), 2 (1,1), 3 (2,0), ...
__device__ __forceinline__ void tri_tile(int x, int& i, int& j) {
    i = x >= 6 ? 3 : x >= 3 ? 2 : x >= 1 ? 1 : 0;
    j = x - i * (i + 1) / 2;
}

// ---- the pass ---------------------------------------------------------------------------------

// What a launch of decay_pass does besides its outputs.
enum { kPassPlain = 0, kPassGq = 1, kPassGk = 2, kPassState = 3 };

template <int P, int DK, int KIND>
__global__ __launch_bounds__(256, 1) void decay_pass(DecayPass a) {
    using Sh = DecayShape<P>;
    constexpr int C = Sh::C, PC = Sh::PC, MT = Sh::MT, KB = DK / 32, MD = DK / 16;
    constexpr int UQ = C * DK / 8 / 256, UV = C * kDecayCols / 8 / 256;  // 8-element units per thread
    constexpr bool OUT = KIND != kPassState, AUX = KIND == kPassGq || KIND == kPassGk;

    __shared__ __attribute__((aligned(16))) uint16_t sq[OUT ? P * C * DK : 8];
    __shared__ __attribute__((aligned(16))) uint16_t sk[P * C * DK];
    __shared__ __attribute__((aligned(16))) uint16_t sv[P * C * kDecayCols];
    __shared__ __attribute__((aligned(16))) uint16_t sa[OUT ? PC * Sh::BLK * 512 : 8];
    __shared__ float2 sg[C];              // the sums G, split
    __shared__ float s_into[C], s_out[C];  // e^{G_i} and e^{G_C - G_j}, with their scales
    __shared__ double s_total;
    __shared__ float s_part[AUX ? 4 : 1][AUX ? C : 1];
    __shared__ float s_dot[4];

    const int t = threadIdx.x, lane = t & 63, w = t >> 6, l16 = lane & 15, lg = lane >> 4;

    // workgroups of one head's column tiles are 8 apart: on one XCD, they share its L2's lines
    const unsigned id = blockIdx.x, rest = id >> 3;
    const int tile = static_cast<int>(rest % a.n_tiles);
    const int64_t pair = static_cast<int64_t>(rest / a.n_tiles) * 8 + (id & 7);
    const int HO = KIND == kPassState ? a.HS : a.HO;  // (the states' pass runs once per state)
    if (pair >= static_cast<int64_t>(a.n_seqs) * HO) return;
    const int seq = static_cast<int>(pair / HO), ho = static_cast<int>(pair % HO);
    const int hs = ho / (HO / a.HS);                   // the state's head
    const int n_src = a.HK / a.HS;
    const int n0 = tile * kDecayCols;

    // the sequence and this workgroup's span of it
    int64_t start = 0, rows0 = 0;
    int len = a.T;
    int64_t qb = 0, kb_ = 0, vb = 0, gb = 0, xb = 0;
    if (a.cu) {
        const int z0 = min(max(a.cu[seq], 0), a.T), z1 = min(max(a.cu[seq + 1], 0), a.T);
        start = z0;
        len = max(z1 - z0, 0);
        rows0 = z0;
    } else {
        qb = seq * a.q_sb, kb_ = seq * a.k_sb, vb = seq * a.v_sb, gb = seq * a.g_sb, xb = seq * a.x_sb;
        rows0 = static_cast<int64_t>(seq) * a.T;
    }
    const int n_spans = max((len + a.span - 1) / a.span, 1), order = blockIdx.y;
    if (order >= n_spans || (KIND == kPassState && order + 1 >= n_spans)) return;
    const int my_span = a.reverse ? n_spans - 1 - order : order;
    const int c_begin = my_span * a.span;                    // first token, relative to the sequence
    const int c_end = min(c_begin + a.span, len);
    const int n_chunks = (c_end - c_begin + C - 1) / C;

    const int64_t state_pair = static_cast<int64_t>(seq) * a.HS + hs;
    const int64_t frag = static_cast<int64_t>(MD) * 256;     // float4s of a workgroup's part of a state
    // ---- the state before the span
    f32x4_t S[MD];
#pragma unroll
    for (int md = 0; md < MD; ++md) S[md] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    const int n = n0 + 16 * w + l16;                         // this lane's column
    int64_t slot_pair = state_pair;
    bool stored = true;
    if (a.slots) {
        const int slot = a.slots[seq];
        stored = slot >= 0 && slot < a.n_slots;
        slot_pair = static_cast<int64_t>(stored ? slot : 0) * a.HS + hs;
        if (!stored && a.bad_slot && t == 0) *a.bad_slot = 1;
    }
    if (KIND != kPassState) {
        if (a.s0 && (stored || a.s0_gathered)) {
            const float* s0 = a.s0 + (a.s0_gathered ? state_pair : slot_pair) * a.D * a.D;
#pragma unroll
            for (int md = 0; md < MD; ++md)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int d = s_row_d(md, 4 * lg + r);
                    if (d < a.D && n < a.D) S[md][r] = s0[static_cast<int64_t>(d) * a.s_row + static_cast<int64_t>(n) * a.s_col];
                }
        }
        for (int s = 0; s < order; ++s) {
            const int64_t at = state_pair * a.n_spans + s;
            const float e = exp2_f64(a.span_log[at]);
            const f32x4_t* u = reinterpret_cast<const f32x4_t*>(a.span_state) + (at * a.n_tiles + tile) * frag;
#pragma unroll
            for (int md = 0; md < MD; ++md) S[md] = e * S[md] + u[(w * MD + md) * 64 + lane];
        }
    }

    // halves of A's blocks that no tile covers
    if (OUT && w == 0)
#pragma unroll
        for (int p = 0; p < PC; ++p)
#pragma unroll
            for (int i = 0; i < MT; i += 2) zero_upper_half(sa + p * Sh::BLK * 512, qblk(i, i >> 1), lane);

    // ---- loads of one step (a chunk and one of its source heads) into registers
    Raw8<P> rq[OUT ? UQ : 1], rk[UQ], rv[UV];
    float rg = 0.f;
    const int n_steps = n_chunks * n_src;
    auto chunk_at = [&](int c, int& first, int& cnt) {  // tokens relative to the sequence
        const int k = a.reverse ? n_chunks - 1 - c : c;
        first = c_begin + k * C;
        cnt = min(C, c_end - first);
    };
    auto fetch = [&](int step) {
        int first, cnt;
        chunk_at(step / n_src, first, cnt);
        const int m = step % n_src;
        const int64_t kh = static_cast<int64_t>(hs) * (a.HK / a.HS) + m;  // the source head
#pragma unroll
        for (int i = 0; i < UQ; ++i) {
            const int u = t + 256 * i, row = u / (DK / 8), col = 8 * (u % (DK / 8));
            const int64_t tok = start + (a.reverse ? first + cnt - 1 - row : first + row);
            const bool in = row < cnt && col < a.D;
            if (in) {
                rk[i].load(a.k, kb_ + tok * a.k_st + kh * a.k_sh + col, a.D - col);
                if (OUT) rq[i].load(a.q, qb + tok * a.q_st + static_cast<int64_t>(ho) * a.q_sh + col, a.D - col);
            } else {
                rk[i].zero();
                if (OUT) rq[i].zero();
            }
        }
#pragma unroll
        for (int i = 0; i < UV; ++i) {
            const int u = t + 256 * i, row = u >> 3, col = n0 + 8 * (u & 7);
            const int64_t tok = start + (a.reverse ? first + cnt - 1 - row : first + row);
            if (row < cnt && col < a.D) rv[i].load(a.v, vb + tok * a.v_st + kh * a.v_sh + col, a.D - col);
            else rv[i].zero();
        }
        if (t < C && m == 0) {
            rg = 0.f;
            if (t < cnt) {
                const int tok = a.reverse ? first + cnt - t : first + t;  // (backwards: the token after)
                if (tok < len) rg = a.g[gb + (start + tok) * a.g_st + hs];
            }
        }
    };

    f32x4_t O[MT];
    double log_total = 0.0;
    if (n_steps > 0) fetch(0);
    for (int step = 0; step < n_steps; ++step) {
        const int c = step / n_src, m = step % n_src;
        int first, cnt;
        chunk_at(c, first, cnt);
        // ---- registers to LDS
#pragma unroll
        for (int i = 0; i < UQ; ++i) {
            const int u = t + 256 * i, row = u / (DK / 8), ch = (u % (DK / 8)) ^ kf<DK>(row);
            u32x4_t p[P];
            rk[i].planes(p);
#pragma unroll
            for (int x = 0; x < P; ++x) *reinterpret_cast<u32x4_t*>(sk + x * C * DK + row * DK + 8 * ch) = p[x];
            if (OUT) {
                rq[i].planes(p);
#pragma unroll
                for (int x = 0; x < P; ++x) *reinterpret_cast<u32x4_t*>(sq + x * C * DK + row * DK + 8 * ch) = p[x];
            }
        }
#pragma unroll
        for (int i = 0; i < UV; ++i) {
            const int u = t + 256 * i, row = u >> 3, ch = (u & 7) ^ vf(row);
            u32x4_t p[P];
            rv[i].planes(p);
#pragma unroll
            for (int x = 0; x < P; ++x)
                *reinterpret_cast<u32x4_t*>(sv + x * C * kDecayCols + row * kDecayCols + 8 * ch) = p[x];
        }
        if (w == 0 && m == 0) {
            const double G = wave_prefix_f64(t < C ? log2_decay(rg) : 0.0);
            const double last = __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(G), 63),
                                                 __builtin_amdgcn_readlane(__double2loint(G), 63));
            if (t < C) {
                sg[t] = split_log(G);
                s_into[t] = exp2_f64(G) * a.into_scale;
                s_out[t] = exp2_f64(last - G) * a.out_scale;
            }
            if (t == 0) s_total = last;
        }
        lds_barrier();
        if (step + 1 < n_steps) fetch(step + 1);

        // ---- A, lower tiles, as packed operands
        if (OUT) {
            for (int x = w; x < Sh::TRI; x += 4) {
                int i, j;
                tri_tile(x, i, j);
                f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) {
                    u32x4_t ko[P], qo[P];
#pragma unroll
                    for (int p = 0; p < P; ++p) {
                        ko[p] = op_row<DK>(sk + p * C * DK, 16 * j + l16, kb, lg);
                        qo[p] = op_row<DK>(sq + p * C * DK, 16 * i + l16, kb, lg);
                    }
                    acc = mfma_planes<P, P>(ko, qo, acc);
                }
                const int row = 16 * i + l16;
                const float2 gi = sg[row];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int col = 16 * j + 4 * lg + r;
                    acc[r] = col <= row ? acc[r] * (exp2_diff(gi, sg[col]) * a.a_scale) : 0.f;
                }
                u32x2_t ap[PC];
                split4<PC>(acc, ap);
#pragma unroll
                for (int p = 0; p < PC; ++p)
                    *reinterpret_cast<u32x2_t*>(sa + (p * Sh::BLK + qblk(i, j >> 1)) * 512 + lane * 8 + 4 * (j & 1)) =
                        ap[p];
            }
            lds_barrier();
        }

        const double chunk_log = s_total;
        if (m == 0) {
            // ---- the state's part of the outputs
            if (OUT) {
#pragma unroll
                for (int i = 0; i < MT; ++i) O[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) {
                    u32x4_t so[PC];
                    const float s8[8] = {S[2 * kb][0], S[2 * kb][1], S[2 * kb][2], S[2 * kb][3],
                                         S[2 * kb + 1][0], S[2 * kb + 1][1], S[2 * kb + 1][2], S[2 * kb + 1][3]};
                    split8<PC>(s8, so);
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
                        u32x4_t qo[P];
#pragma unroll
                        for (int p = 0; p < P; ++p) qo[p] = op_row<DK>(sq + p * C * DK, 16 * i + l16, kb, lg);
                        O[i] = mfma_planes<PC, P>(so, qo, O[i]);
                    }
                }
#pragma unroll
                for (int i = 0; i < MT; ++i) O[i] *= s_into[16 * i + l16];
            }
            if (KIND == kPassGq && (first / C) % a.keep == 0 && ho % (HO / a.HS) == 0) {
                f32x4_t* kept = reinterpret_cast<f32x4_t*>(a.kept) +
                                ((state_pair * a.n_keep + first / C / a.keep) * a.n_tiles + tile) * frag;
#pragma unroll
                for (int md = 0; md < MD; ++md) kept[(w * MD + md) * 64 + lane] = S[md];
            }
            if constexpr (AUX) {
                // each token's product of that part with the row of `aux` (q for gq, k for gk)
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    const int row = 16 * i + l16, col = n0 + 16 * w + 4 * lg;
                    float sum = 0.f;
                    if (row < cnt) {
                        const int64_t tok = start + (a.reverse ? first + cnt - 1 - row : first + row);
                        const int64_t at = xb + tok * a.x_st + static_cast<int64_t>(ho) * a.x_sh + col;
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (col + r < a.D) {
                                const float x = P == 1 ? bf16_to_f32(static_cast<const uint16_t*>(a.aux)[at + r])
                                                       : static_cast<const float*>(a.aux)[at + r];
                                sum += x * O[i][r];
                            }
                    }
                    sum += __shfl_xor(sum, 16);
                    sum += __shfl_xor(sum, 32);
                    if (lg == 0) s_part[w][row] = sum;
                }
            }
            const float e = exp2_f64(chunk_log);
#pragma unroll
            for (int md = 0; md < MD; ++md) S[md] *= e;
            log_total += chunk_log;
        }
        // ---- A V, and the state
#pragma unroll
        for (int kb = 0; kb < MT / 2; ++kb) {
            // V of tokens 32 kb + {4 lg + [0, 4), 16 + 4 lg + [0, 4)}, column 16 w + l16
            const int j4 = (lane >> 2) & 3, cc = lane & 3, row = 4 * lg + j4;
            const unsigned va = lds_addr(sv + (32 * kb + row) * kDecayCols +
                                         8 * ((2 * w + (cc >> 1)) ^ vf(row)) + 4 * (cc & 1));
            constexpr int R16 = 16 * kDecayCols * 2, VP = C * kDecayCols * 2;
            u32x4_t vo[P];
            f32x4_t x0 = {0.f, 0.f, 0.f, 0.f}, x1 = x0;
            if constexpr (P == 1) {
                u32x2_t lo, hi;
                tr2<0, R16>(va, lo, hi);
                vo[0] = join(lo, hi);
                x0 = widen4(lo), x1 = widen4(hi);
            } else {
                u32x2_t lo[3], hi[3];
                tr2<0, R16>(va, lo[0], hi[0]);
                tr2<VP, VP + R16>(va, lo[1], hi[1]);
                tr2<2 * VP, 2 * VP + R16>(va, lo[2], hi[2]);
#pragma unroll
                for (int p = 2; p >= 0; --p) {
                    vo[p] = join(lo[p], hi[p]);
                    x0 += widen4(lo[p]), x1 += widen4(hi[p]);
                }
            }
            if (OUT) {
#pragma unroll
                for (int i = 2 * kb; i < MT; ++i) {
                    u32x4_t ao[PC];
#pragma unroll
                    for (int p = 0; p < PC; ++p)
                        ao[p] = *reinterpret_cast<const u32x4_t*>(sa + (p * Sh::BLK + qblk(i, kb)) * 512 + lane * 8);
                    O[i] = mfma_planes<P, PC>(vo, ao, O[i]);
                }
            }
            float v8[8];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                v8[r] = x0[r] * s_out[32 * kb + 4 * lg + r];
                v8[4 + r] = x1[r] * s_out[32 * kb + 16 + 4 * lg + r];
            }
            u32x4_t wo[PC];
            split8<PC>(v8, wo);
#pragma unroll
            for (int d32 = 0; d32 < KB; ++d32) {
                // K^T: rows 32 d32 + 8 .. (s_row_d of tiles 2 d32 and 2 d32 + 1), the same tokens
                const unsigned ka = lds_addr(sk + (32 * kb + row) * DK + 8 * ((4 * d32 + cc) ^ kf<DK>(row)));
                constexpr int K16 = 16 * DK * 2, KP = C * DK * 2;
                u32x4_t k0[P], k1[P];
                u32x2_t a0, a1, b0, b1;
                tr4<0, K16, 8, 8 + K16>(ka, a0, a1, b0, b1);
                k0[0] = join(a0, a1), k1[0] = join(b0, b1);
                if constexpr (P == 3) {
                    tr4<KP, KP + K16, KP + 8, KP + 8 + K16>(ka, a0, a1, b0, b1);
                    k0[1] = join(a0, a1), k1[1] = join(b0, b1);
                    tr4<2 * KP, 2 * KP + K16, 2 * KP + 8, 2 * KP + 8 + K16>(ka, a0, a1, b0, b1);
                    k0[2] = join(a0, a1), k1[2] = join(b0, b1);
                }
                S[2 * d32] = mfma_planes<P, PC>(k0, wo, S[2 * d32]);
                S[2 * d32 + 1] = mfma_planes<P, PC>(k1, wo, S[2 * d32 + 1]);
            }
        }
        // ---- outputs
        if (OUT && m == n_src - 1) {
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const int row = 16 * i + l16, col = n0 + 16 * w + 4 * lg;
                if (row >= cnt || col >= a.D) continue;
                const int64_t tok = rows0 + (a.reverse ? first + cnt - 1 - row : first + row);
                const int64_t at = (tok * HO + ho) * a.D + col;
                const int left = a.D - col;
                if (a.out_bf16) {
                    uint16_t* o = static_cast<uint16_t*>(a.o) + at;
                    const u32x2_t v = cvt4(O[i]);
                    if (left >= 4) __builtin_memcpy(o, &v, 8);
                    else
                        for (int r = 0; r < left; ++r) o[r] = static_cast<uint16_t>((r < 2 ? v.x : v.y) >> (16 * (r & 1)));
                } else {
                    float* o = static_cast<float*>(a.o) + at;
                    if (left >= 4) __builtin_memcpy(o, &O[i], 16);
                    else
                        for (int r = 0; r < left; ++r) o[r] = O[i][r];
                }
            }
            if (KIND == kPassGk && (first / C) % a.keep == 0) {
                // dL/dg of the chunk's first token: e^g <the state before it, the gradient after it>
                const f32x4_t* kept = reinterpret_cast<const f32x4_t*>(a.kept) +
                                      ((state_pair * a.n_keep + first / C / a.keep) * a.n_tiles + tile) * frag;
                float dot = 0.f;
#pragma unroll
                for (int md = 0; md < MD; ++md) {
                    const f32x4_t x = kept[(w * MD + md) * 64 + lane] * S[md];
                    dot += (x[0] + x[1]) + (x[2] + x[3]);
                }
                dot = wave_sum_row3(dot);
                if (lane == 63) s_dot[w] = dot;
            }
        }
        lds_barrier();
        if constexpr (AUX)
            if (m == 0 && t < cnt) {
                const int64_t tok = rows0 + (a.reverse ? first + cnt - 1 - t : first + t);
                a.part[(static_cast<int64_t>(tile) * a.n_rows + tok) * HO + ho] =
                    (s_part[0][t] + s_part[1][t]) + (s_part[2][t] + s_part[3][t]);
            }
        if (KIND == kPassGk && m == n_src - 1 && t == 0 && (first / C) % a.keep == 0) {
            const float e = exp2_f64(log2_decay(a.g[gb + (start + first) * a.g_st + hs]));
            a.cross[(state_pair * a.n_keep + first / C / a.keep) * a.n_tiles + tile] =
                e * ((s_dot[0] + s_dot[1]) + (s_dot[2] + s_dot[3]));
        }
    }

    // ---- the state after the span
    if (KIND == kPassState) {
        const int64_t at = state_pair * a.n_spans + order;
        f32x4_t* u = reinterpret_cast<f32x4_t*>(a.span_state) + (at * a.n_tiles + tile) * frag;
#pragma unroll
        for (int md = 0; md < MD; ++md) u[(w * MD + md) * 64 + lane] = S[md];
        if (tile == 0 && t == 0) a.span_log[at] = log_total;
    } else if (a.s_out && order == n_spans - 1 && ho % (HO / a.HS) == 0 && stored) {
        float e = 1.f;
        if (a.reverse && len > 0) e = exp2_f64(log2_decay(a.g[gb + start * a.g_st + hs]));
        float* so = a.s_out + slot_pair * a.D * a.D;
#pragma unroll
        for (int md = 0; md < MD; ++md)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int d = s_row_d(md, 4 * lg + r);
                if (d < a.D && n < a.D) so[static_cast<int64_t>(d) * a.s_row + static_cast<int64_t>(n) * a.s_col] = e * S[md][r];
            }
    }
}

// ---- dL/dg ------------------------------------------------------------------------------------
//
// dL/dg_t sums, over all pairs of a token j < t and a token i >= t, what j contributes through i
// (and what the first state and the last state's gradient add).  Per chunk: pairs inside it from
// the products (q_i . k_j)(go_i . v_j) e^{G_i - G_j}; pairs with j before it or i behind it from the
// two passes' products r_i, c_j; pairs around the whole chunk from the directly computed gradient at
// every `keep` chunks' first token.  No sum is taken as a difference of others over more than those
// 256 tokens.  One wave a chunk, one workgroup `keep` chunks (256 tokens).
template <int P>
__global__ __launch_bounds__(P == 1 ? 256 : 512) void decay_gate_grad(DecayGateGrad a) {
    using Sh = DecayShape<P>;
    constexpr int C = Sh::C, MT = Sh::MT, W = 256 / C;  // (W: chunks, waves)
    __shared__ float sp[W][C][C + 1];
    __shared__ float2 sg[W][C];
    __shared__ float s_r[W][C], s_c[W][C + 1], s_sum[W];
    const int t = threadIdx.x, lane = t & 63, w = t >> 6, l16 = lane & 15, lg = lane >> 4;
    const int G = a.Hq / a.H;
    const int64_t id = blockIdx.x;
    const int h = static_cast<int>(id % a.H);
    const int ks = static_cast<int>(id / a.H % a.n_keep);
    const int64_t b = id / a.H / a.n_keep, pair = b * a.H + h;
    const int first = (ks * W + w) * C, cnt = min(C, a.T - first);  // (may be <= 0 for the last waves)

    const double x = lane < cnt ? log2_decay(a.g[b * a.g_sb + (first + lane) * a.g_st + h]) : 0.0;
    const double sum = wave_prefix_f64(x);
    if (lane < C) sg[w][lane] = split_log(sum);

    f32x4_t acc[Sh::TRI];
#pragma unroll
    for (int i = 0; i < Sh::TRI; ++i) acc[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    for (int m = 0; m < G; ++m) {
        const int64_t hq = static_cast<int64_t>(h) * G + m;
        f32x4_t x1[Sh::TRI], x2[Sh::TRI];
#pragma unroll
        for (int i = 0; i < Sh::TRI; ++i) x1[i] = x2[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        for (int col = 8 * lg; col - 8 * lg < a.D; col += 32) {
            auto rows = [&](const void* p, int64_t sb, int64_t st, int64_t sh, int64_t head, u32x4_t(&op)[MT][P]) {
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    Raw8<P> r;
                    const int row = 16 * i + l16;
                    if (row < cnt && col < a.D) r.load(p, b * sb + (first + row) * st + head * sh + col, a.D - col);
                    else r.zero();
                    r.planes(op[i]);
                }
            };
            u32x4_t src[MT][P], dst[MT][P];
            rows(a.k, a.k_sb, a.k_st, a.k_sh, h, src);
            rows(a.q, a.q_sb, a.q_st, a.q_sh, hq, dst);
#pragma unroll
            for (int i = 0, n = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j <= i; ++j, ++n) x1[n] = mfma_planes<P, P>(src[j], dst[i], x1[n]);
            rows(a.v, a.v_sb, a.v_st, a.v_sh, h, src);
            rows(a.go, a.go_sb, a.go_st, a.go_sh, hq, dst);
#pragma unroll
            for (int i = 0, n = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j <= i; ++j, ++n) x2[n] = mfma_planes<P, P>(src[j], dst[i], x2[n]);
        }
#pragma unroll
        for (int i = 0; i < Sh::TRI; ++i) acc[i] += x1[i] * x2[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0, n = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j <= i; ++j, ++n) {
            const int row = 16 * i + l16;
            const float2 gi = sg[w][row];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int col = 16 * j + 4 * lg + r;
                sp[w][row][col] = col < row ? acc[n][r] * exp2_diff(gi, sg[w][col]) : 0.f;
            }
        }
    // r from the last token to the first (lane l: row C - 1 - l), c from the first to the last
    float r = 0.f, c = 0.f;
    const int back = C - 1 - lane;
    if (back >= 0 && back < cnt)
        for (int x = 0; x < a.n_tiles; ++x)
            for (int m = 0; m < G; ++m)
                r += a.r_part[(static_cast<int64_t>(x) * a.n_rows + b * a.T + first + back) * a.Hq + h * G + m];
    if (lane < cnt)
        for (int x = 0; x < a.n_tiles; ++x)
            c += a.c_part[(static_cast<int64_t>(x) * a.n_rows + b * a.T + first + lane) * a.H + h];
    r = wave_prefix_sum(r);
    c = wave_prefix_sum(c);
    if (lane < C) {
        s_r[w][back] = r;      // the sum over tokens from `back` on
        s_c[w][lane + 1] = c;  // the sum over tokens before lane + 1
    }
    if (lane == 0) s_c[w][0] = 0.f;
    __syncthreads();
    if (lane < C) {  // row by row: the sums over j < t
        float run = 0.f;
        for (int j = 0; j <= lane; ++j) {
            const float p = sp[w][lane][j];
            sp[w][lane][j] = run;
            run += p;
        }
    }
    __syncthreads();
    float dg = 0.f;
    if (lane < C)
        for (int i = lane; i < C; ++i) dg += sp[w][i][lane];
    float around = 0.f;
    for (int x = 0; x < a.n_tiles; ++x) around += a.cross[(pair * a.n_keep + ks) * a.n_tiles + x];
    for (int i = 0; i < w; ++i) around += s_c[i][C] - s_r[i][0];
    if (lane < cnt) {
        // (the chunk's first token: the gradient handed on, without taking r's sum out and in again)
        dg = lane == 0 ? around : a.scale * dg + s_r[w][lane] + s_c[w][lane] + (around - s_r[w][0]);
        if (a.gg) a.gg[(b * a.T + first + lane) * a.H + h] = dg;
    } else {
        dg = 0.f;
    }
    if (a.gg_part) {
        const float total = wave_sum_row3(dg);
        if (lane == 63) s_sum[w] = total;
        __syncthreads();
        if (t == 0) {
            float s = 0.f;
            for (int i = 0; i < W; ++i) s += s_sum[i];
            a.gg_part[(b * a.n_keep + ks) * a.H + h] = s;
        }
    }
}

template <int P, int DK>
hipError_t launch_pass(const DecayPass& a, int kind, int n_spans, hipStream_t st) {
    const int heads = kind == kPassState ? a.HS : a.HO;
    const int64_t pairs = static_cast<int64_t>(a.n_seqs) * heads;
    const dim3 grid(static_cast<unsigned>((pairs + 7) / 8 * 8 * a.n_tiles), static_cast<unsigned>(n_spans));
    switch (kind) {
        case kPassPlain: hipLaunchKernelGGL((decay_pass<P, DK, kPassPlain>), grid, dim3(256), 0, st, a); break;
        case kPassGq: hipLaunchKernelGGL((decay_pass<P, DK, kPassGq>), grid, dim3(256), 0, st, a); break;
        case kPassGk: hipLaunchKernelGGL((decay_pass<P, DK, kPassGk>), grid, dim3(256), 0, st, a); break;
        default: hipLaunchKernelGGL((decay_pass<P, DK, kPassState>), grid, dim3(256), 0, st, a); break;
    }
    return hipGetLastError();
}

// One pass: the states of all spans but the last where there are several, then the outputs.
template <int P>
hipError_t run_pass(const DecayPass& a, int kind, hipStream_t st) {
    auto go = [&](int what, int spans) {
        if (a.D <= 64) return launch_pass<P, 64>(a, what, spans, st);
        if (a.D <= 128) return launch_pass<P, 128>(a, what, spans, st);
        return launch_pass<P, 256>(a, what, spans, st);
    };
    if (a.n_spans > 1)
        if (hipError_t e = go(kPassState, a.n_spans - 1); e != hipSuccess) return e;
    return go(kind, a.n_spans);
}

template <int P>
hipError_t run_gate_grad(const DecayGateGrad& a, hipStream_t st) {
    const int64_t n = static_cast<int64_t>(a.B) * a.H * a.n_keep;
    hipLaunchKernelGGL((decay_gate_grad<P>), dim3(static_cast<unsigned>(n)), dim3(P == 1 ? 256 : 512), 0, st, a);
    return hipGetLastError();
}

}  // namespace
}  // namespace pm
