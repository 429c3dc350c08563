// decay_attention.hip — K14: linear attention with a decay for each head.  The passes for bf16 inputs
// (pm_decay.h has their mathematics), the single token, and how calls are cut into workgroups.

#include <algorithm>
#include <type_traits>

#include "pm_decay.h"
#include "pm_internal.h"
#include "pm_vec.h"

namespace pm {

hipError_t decay_pass_bf16(const DecayPass& a, int kind, hipStream_t st) { return run_pass<1>(a, kind, st); }
hipError_t decay_gate_grad_bf16(const DecayGateGrad& a, hipStream_t st) { return run_gate_grad<1>(a, st); }

namespace {

// The states of n sequences from their slots (zeros for a slot outside the pool), in order.
__global__ __launch_bounds__(256) void gather_states(const float* pool, const int32_t* slots, int n_slots, float* to,
                                                     int64_t size) {
    const int slot = slots ? slots[blockIdx.y] : static_cast<int>(blockIdx.y);
    const bool there = !slots || (slot >= 0 && slot < n_slots);
    const float* from = pool + (there ? slot : 0) * size;
    float* out = to + blockIdx.y * size;
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < size; i += gridDim.x * 256ll) out[i] = there ? from[i] : 0.f;
}

// gg[h] = the sum of its n parts, in 64 bits, in an order that does not change
__global__ __launch_bounds__(256) void sum_gate_parts(const float* part, float* gg, int64_t n, int H) {
    __shared__ double s[256];
    double sum = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += 256) sum += part[i * H + blockIdx.x];
    s[threadIdx.x] = sum;
    for (int m = 128; m > 0; m >>= 1) {
        __syncthreads();
        if (static_cast<int>(threadIdx.x) < m) s[threadIdx.x] += s[threadIdx.x + m];
    }
    if (threadIdx.x == 0) gg[blockIdx.x] = static_cast<float>(s[0]);
}

struct Plan {
    int n_tiles, span, n_spans;
};

// Workgroups: one per sequence, output head and 64 columns of the state, or, where these are fewer
// than two for every CU, as many again along the sequence as make it two (spans of at least 512
// tokens: a span costs a state written and read, as much as 128 tokens' q, k, v and o).
Plan plan(int n_seqs, int T, int HO, int D) {
    Plan p{(D + kDecayCols - 1) / kDecayCols, max(T, 1), 1};
    const int64_t groups = static_cast<int64_t>(n_seqs) * HO * p.n_tiles;
    const int64_t want = groups > 0 ? (512 + groups - 1) / groups : 1;
    if (want > 1 && T > 512) {
        const int64_t per = std::max<int64_t>((T + want - 1) / want, 512);
        p.span = static_cast<int>((per + kDecayKeep - 1) / kDecayKeep * kDecayKeep);
        p.n_spans = (T + p.span - 1) / p.span;
    }
    return p;
}

size_t up(size_t n) { return (n + 255) / 256 * 256; }
int padded(int D) { return D <= 64 ? 64 : D <= 128 ? 128 : 256; }
// Bytes of one state's accumulators: n_tiles workgroups of (padded D) x 64 floats.
size_t frag_bytes(const Plan& p, int D) { return static_cast<size_t>(p.n_tiles) * padded(D) * kDecayCols * 4; }

struct FwdWs {
    size_t gathered, span_state, span_log, bytes;
};
FwdWs fwd_ws(int n_seqs, int T, int Hq, int H, int D, bool in_place) {
    const Plan p = plan(n_seqs, T, Hq, D);
    const size_t states = static_cast<size_t>(n_seqs) * H;
    FwdWs w{};
    // several workgroups read a first state that another one may already have replaced
    if (in_place && (p.n_spans > 1 || Hq > H)) w.bytes += up(states * D * D * 4);
    w.span_state = w.bytes;
    if (p.n_spans > 1) w.bytes += up(states * p.n_spans * frag_bytes(p, D));
    w.span_log = w.bytes;
    if (p.n_spans > 1) w.bytes += up(states * p.n_spans * 8);
    return w;
}

struct BwdWs {
    size_t span_state, span_log, kept, cross, r_part, c_part, gg_part, bytes;
};
BwdWs bwd_ws(int B, int T, int Hq, int H, int D, bool gates) {
    const Plan pq = plan(B, T, Hq, D), pk = plan(B, T, H, D);
    const size_t states = static_cast<size_t>(B) * H, spans = max(pq.n_spans, pk.n_spans);
    const size_t keep = (T + kDecayKeep - 1) / kDecayKeep, rows = static_cast<size_t>(B) * T;
    BwdWs w{};
    auto take = [&](size_t n) {
        const size_t at = w.bytes;
        w.bytes += up(n);
        return at;
    };
    w.span_state = take(spans > 1 ? states * spans * frag_bytes(pq, D) : 0);
    w.span_log = take(spans > 1 ? states * spans * 8 : 0);
    if (gates) {
        w.kept = take(states * keep * frag_bytes(pq, D));
        w.cross = take(states * keep * pq.n_tiles * 4);
        w.r_part = take(pq.n_tiles * rows * Hq * 4);
        w.c_part = take(pq.n_tiles * rows * H * 4);
        w.gg_part = take(states * keep * 4);
    }
    return w;
}

template <typename T>
T* at(void* base, size_t off) {
    return reinterpret_cast<T*>(static_cast<char*>(base) + off);
}

}  // namespace

size_t decay_attn_ws_bytes(int n_seqs, int T, int Hq, int H, int D, bool in_place) {
    return fwd_ws(n_seqs, T, Hq, H, D, in_place).bytes;
}
size_t decay_attn_bwd_ws_bytes(int B, int T, int Hq, int H, int D, bool gates) {
    return bwd_ws(B, T, Hq, H, D, gates).bytes;
}
int64_t decay_attn_groups(int n_seqs, int T, int Hq, int D) {
    const Plan p = plan(n_seqs, T, Hq, D);
    return (static_cast<int64_t>(n_seqs) * Hq + 7) / 8 * 8 * p.n_tiles;
}
int decay_attn_spans(int n_seqs, int T, int Hq, int D) { return plan(n_seqs, T, Hq, D).n_spans; }

hipError_t launch_decay_attn(const DecayAttnArgs& a, hipStream_t st) {
    if (a.cu && a.cu_flag)
        if (hipError_t e = launch_varlen_check(a.cu, a.n_seqs, a.T, a.cu_flag, st); e != hipSuccess) return e;
    const Plan p = plan(a.n_seqs, a.T, a.Hq, a.D);
    const bool in_place = a.s0 && a.s0 == a.s_out;
    const FwdWs w = fwd_ws(a.n_seqs, a.T, a.Hq, a.H, a.D, in_place);
    DecayPass x{};
    x.q = a.q, x.k = a.k, x.v = a.v;
    x.q_sb = a.strides[0], x.q_st = a.strides[1], x.q_sh = a.strides[2];
    x.k_sb = a.strides[3], x.k_st = a.strides[4], x.k_sh = a.strides[5];
    x.v_sb = a.strides[6], x.v_st = a.strides[7], x.v_sh = a.strides[8];
    x.g = a.g, x.g_sb = a.g_sb, x.g_st = a.g_st;
    x.cu = a.cu;
    x.s0 = a.s0, x.s_out = a.s_out, x.s_row = a.D, x.s_col = 1;
    x.slots = a.slots, x.n_slots = a.n_slots, x.bad_slot = a.bad_slot;
    if (in_place && (p.n_spans > 1 || a.Hq > a.H)) {
        const int64_t size = static_cast<int64_t>(a.H) * a.D * a.D;
        float* to = at<float>(a.workspace, w.gathered);
        for (int b0 = 0; b0 < a.n_seqs; b0 += 65535) {
            const int n = min(65535, a.n_seqs - b0);
            const dim3 grid(static_cast<unsigned>(std::min<int64_t>((size + 1023) / 1024, 256)), static_cast<unsigned>(n));
            hipLaunchKernelGGL(gather_states, grid, dim3(256), 0, st, a.slots ? a.s0 : a.s0 + b0 * size,
                               a.slots ? a.slots + b0 : nullptr, a.n_slots, to + b0 * size, size);
            if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
        }
        x.s0 = to;
        x.s0_gathered = true;
    }
    x.o = a.o, x.out_bf16 = a.out_bf16;
    x.n_seqs = a.n_seqs, x.T = a.T, x.HO = a.Hq, x.HK = x.HS = a.H, x.D = a.D;
    x.n_tiles = p.n_tiles, x.span = p.span, x.n_spans = p.n_spans;
    x.span_state = at<float>(a.workspace, w.span_state);
    x.span_log = at<double>(a.workspace, w.span_log);
    x.a_scale = x.into_scale = a.scale, x.out_scale = 1.f;
    return a.bf16 ? decay_pass_bf16(x, 0, st) : decay_pass_f32(x, 0, st);
}

hipError_t launch_decay_attn_bwd(const DecayAttnBwdArgs& a, hipStream_t st) {
    const bool gates = a.gg != nullptr;
    const Plan pq = plan(a.B, a.T, a.Hq, a.D), pk = plan(a.B, a.T, a.H, a.D);
    const BwdWs w = bwd_ws(a.B, a.T, a.Hq, a.H, a.D, gates);
    struct Role {
        const void* p;
        const int64_t* s;
    };
    const int64_t go_strides[3] = {static_cast<int64_t>(a.T) * a.Hq * a.D, static_cast<int64_t>(a.Hq) * a.D, a.D};
    const Role q{a.q, a.strides}, k{a.k, a.strides + 3}, v{a.v, a.strides + 6}, go{a.go, go_strides};
    auto run = [&](Role Q, Role K, Role V, Role aux, int HO, int HK, const Plan& p, bool reverse, bool transposed,
                   const float* s0, float* s_out, void* o, float* part, int kind) {
        DecayPass x{};
        x.q = Q.p, x.q_sb = Q.s[0], x.q_st = Q.s[1], x.q_sh = Q.s[2];
        x.k = K.p, x.k_sb = K.s[0], x.k_st = K.s[1], x.k_sh = K.s[2];
        x.v = V.p, x.v_sb = V.s[0], x.v_st = V.s[1], x.v_sh = V.s[2];
        x.aux = aux.p, x.x_sb = aux.s[0], x.x_st = aux.s[1], x.x_sh = aux.s[2];
        x.g = a.g, x.g_sb = a.g_sb, x.g_st = a.g_st;
        x.s0 = s0, x.s_out = s_out;
        x.s_row = transposed ? 1 : a.D, x.s_col = transposed ? a.D : 1;
        x.o = o, x.out_bf16 = a.bf16, x.reverse = reverse;
        x.n_seqs = a.B, x.T = a.T, x.HO = HO, x.HK = HK, x.HS = a.H, x.D = a.D;
        x.n_tiles = p.n_tiles, x.span = p.span, x.n_spans = p.n_spans;
        x.span_state = at<float>(a.workspace, w.span_state);
        x.span_log = at<double>(a.workspace, w.span_log);
        x.a_scale = a.scale, x.into_scale = reverse ? 1.f : a.scale, x.out_scale = reverse ? a.scale : 1.f;
        x.part = part;
        x.n_rows = static_cast<int64_t>(a.B) * a.T;
        x.kept = at<float>(a.workspace, w.kept), x.cross = at<float>(a.workspace, w.cross);
        x.keep = kDecayKeep / (a.bf16 ? 64 : 32), x.n_keep = (a.T + kDecayKeep - 1) / kDecayKeep;
        return a.bf16 ? decay_pass_bf16(x, kind, st) : decay_pass_f32(x, kind, st);
    };
    float* r_part = at<float>(a.workspace, w.r_part);
    float* c_part = at<float>(a.workspace, w.c_part);
    if (hipError_t e = run(go, v, k, q, a.Hq, a.H, pq, false, true, a.s0, nullptr, a.gq, r_part, gates ? 1 : 0);
        e != hipSuccess)
        return e;
    if (hipError_t e = run(k, q, go, k, a.H, a.Hq, pk, true, false, a.gs, a.gs0, a.gv, nullptr, 0); e != hipSuccess)
        return e;
    if (hipError_t e = run(v, go, q, k, a.H, a.Hq, pk, true, true, a.gs, nullptr, a.gk, c_part, gates ? 2 : 0);
        e != hipSuccess)
        return e;
    if (!gates) return hipSuccess;
    const bool constant = a.g_sb == 0 && a.g_st == 0;
    if (a.T > 0) {
        DecayGateGrad x{};
        x.q = q.p, x.q_sb = q.s[0], x.q_st = q.s[1], x.q_sh = q.s[2];
        x.k = k.p, x.k_sb = k.s[0], x.k_st = k.s[1], x.k_sh = k.s[2];
        x.v = v.p, x.v_sb = v.s[0], x.v_st = v.s[1], x.v_sh = v.s[2];
        x.go = go.p, x.go_sb = go.s[0], x.go_st = go.s[1], x.go_sh = go.s[2];
        x.g = a.g, x.g_sb = a.g_sb, x.g_st = a.g_st;
        x.r_part = r_part, x.c_part = c_part, x.cross = at<float>(a.workspace, w.cross);
        x.gg = constant ? nullptr : a.gg, x.gg_part = constant ? at<float>(a.workspace, w.gg_part) : nullptr;
        x.n_rows = static_cast<int64_t>(a.B) * a.T;
        x.B = a.B, x.T = a.T, x.Hq = a.Hq, x.H = a.H, x.D = a.D;
        x.n_tiles = pq.n_tiles, x.n_keep = (a.T + kDecayKeep - 1) / kDecayKeep;
        x.scale = a.scale;
        if (hipError_t e = a.bf16 ? decay_gate_grad_bf16(x, st) : decay_gate_grad_f32(x, st); e != hipSuccess) return e;
    }
    if (constant) {
        const int64_t n = static_cast<int64_t>(a.B) * ((a.T + kDecayKeep - 1) / kDecayKeep);
        hipLaunchKernelGGL(sum_gate_parts, dim3(static_cast<unsigned>(a.H)), dim3(256), 0, st,
                           at<float>(a.workspace, w.gg_part), a.gg, n, a.H);
        return hipGetLastError();
    }
    return hipSuccess;
}

// ---- one token --------------------------------------------------------------------------------
//
// S = e^g S + k v^T in place, o = scale S^T q for the group's query heads: the state is read and
// written once, 16 bytes a lane (K3's mapping), and everything else is small beside it.  CG column
// groups of 4, 256 / CG row groups.  More than 4 query heads take the new state from the caches
// again, 4 at a time.
namespace {

template <int CG, typename E>
__global__ __launch_bounds__(256) void decay_step(DecayAttnStepArgs a, int b0) {
    constexpr int RG = 256 / CG, GB = 4;
    __shared__ float sk[256], sq[GB][256], red[GB][4][4 * CG];
    const int h = blockIdx.x, b = b0 + blockIdx.y, t = threadIdx.x, cg = t % CG, rg = t / CG, lane = t & 63, w = t >> 6;
    const int G = a.Hq / a.H, D = a.D, col = 4 * cg;
    const auto* q = static_cast<const E*>(a.q) + b * a.strides[0];
    const auto* k = static_cast<const E*>(a.k) + b * a.strides[2] + h * a.strides[3];
    const auto* v = static_cast<const E*>(a.v) + b * a.strides[4] + h * a.strides[5];
    auto out = [&](int m, int d, float x) {
        const int64_t at = (static_cast<int64_t>(b) * a.Hq + static_cast<int64_t>(h) * G + m) * D + d;
        if (a.out_bf16) static_cast<uint16_t*>(a.o)[at] = f32_to_bf16(x);
        else static_cast<float*>(a.o)[at] = x;
    };
    int64_t row = b;
    if (a.slots) {
        const int slot = a.slots[b];
        if (slot < 0 || slot >= a.n_slots) {  // padding
            for (int i = t; i < G * D; i += 256) out(i / D, i % D, 0.f);
            return;
        }
        row = slot;
    }
    float* s = a.s + (row * a.H + h) * D * D;
    const float e = expf(a.g[b * a.g_sb + h]);
    f32x4_t vv = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int r = 0; r < 4; ++r)
        if (col + r < D) vv[r] = to_f32(v[col + r]);
    const int left = D - col;
    for (int m0 = 0; m0 < G; m0 += GB) {
        const int gn = min(GB, G - m0);
        __syncthreads();
        if (t < D) {
            sk[t] = to_f32(k[t]);
#pragma unroll
            for (int m = 0; m < GB; ++m)
                sq[m][t] = m < gn ? to_f32(q[(static_cast<int64_t>(h) * G + m0 + m) * a.strides[1] + t]) : 0.f;
        }
        __syncthreads();
        f32x4_t acc[GB];
#pragma unroll
        for (int m = 0; m < GB; ++m) acc[m] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        if (left > 0) {
#pragma unroll 8
            for (int d = rg; d < D; d += RG) {
                float* p = s + static_cast<int64_t>(d) * D + col;
                f32x4_t x = {0.f, 0.f, 0.f, 0.f};
                if (left >= 4) __builtin_memcpy(&x, p, 16);
                else
                    for (int r = 0; r < left; ++r) x[r] = p[r];
                if (m0 == 0) {
                    x = e * x + sk[d] * vv;
                    if (left >= 4) __builtin_memcpy(p, &x, 16);
                    else
                        for (int r = 0; r < left; ++r) p[r] = x[r];
                }
#pragma unroll
                for (int m = 0; m < GB; ++m) acc[m] += sq[m][d] * x;
            }
        }
#pragma unroll
        for (int m = 0; m < GB; ++m) {
            if (m >= gn) break;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float x = acc[m][r];
                for (int z = CG; z < 64; z <<= 1) x += __shfl_xor(x, z);
                if (lane < CG) red[m][w][4 * cg + r] = x;
            }
        }
        __syncthreads();
        // (CG 64: every wave holds other rows of all columns too)
        for (int i = t; i < gn * D; i += 256) {
            const int m = i / D, d = i % D;
            out(m0 + m, d, a.scale * ((red[m][0][d] + red[m][1][d]) + (red[m][2][d] + red[m][3][d])));
        }
    }
}

template <typename E>
hipError_t step_types(const DecayAttnStepArgs& a, hipStream_t st) {
    for (int b0 = 0; b0 < a.B; b0 += 65535) {
        const dim3 grid(static_cast<unsigned>(a.H), static_cast<unsigned>(min(65535, a.B - b0)));
        if (a.D <= 32) hipLaunchKernelGGL((decay_step<8, E>), grid, dim3(256), 0, st, a, b0);
        else if (a.D <= 64) hipLaunchKernelGGL((decay_step<16, E>), grid, dim3(256), 0, st, a, b0);
        else if (a.D <= 128) hipLaunchKernelGGL((decay_step<32, E>), grid, dim3(256), 0, st, a, b0);
        else hipLaunchKernelGGL((decay_step<64, E>), grid, dim3(256), 0, st, a, b0);
        if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace

hipError_t launch_decay_attn_step(const DecayAttnStepArgs& a, hipStream_t st) {
    return a.bf16 ? step_types<uint16_t>(a, st) : step_types<float>(a, st);
}

}  // namespace pm
