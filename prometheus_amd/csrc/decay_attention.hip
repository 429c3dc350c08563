// decay_attention.hip — K14: linear attention with a decay for each head.  The passes for bf16 inputs
// (pm_decay.h has their mathematics), the single token, and how calls are cut into workgroups.

#include <algorithm>
#include <utility>

#include "pm_decay.h"
#include "pm_internal.h"
#include "pm_vec.h"

namespace pm {

hipError_t decay_pass_bf16(const DecayPasses& a, int kind, hipStream_t st) { return run_pass<1>(a, kind, st); }
hipError_t decay_near_bf16(const DecayNear& a, hipStream_t st) { return run_near<1>(a, st); }

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

// The gates' gradient (pm_decay.h) from near, r and c: a workgroup takes a span, each of its four waves a
// chunk at a time.
__global__ __launch_bounds__(256) void gate_grad(DecayGateGrad a) {
    constexpr int W = 4;
    __shared__ float s_r[W][64], s_c[W][65], s_sum[W];
    const int t = threadIdx.x, lane = t & 63, w = t >> 6, C = a.chunk, G = a.Hq / a.H;
    const int64_t id = blockIdx.x;
    const int h = static_cast<int>(id % a.H);
    const int span = static_cast<int>(id / a.H % a.n_spans);
    const int64_t b = id / a.H / a.n_spans;
    const int begin = span * a.span, end = span_end(begin, a.span, a.T);

    // the gradient at the span's first token
    float around = 0.f;
    {
        const int64_t size = static_cast<int64_t>(a.D) * a.D;
        const float *x = nullptr, *y = nullptr;
        if (span > 0) {
            x = a.ahead + ((b * a.n_spans + span) * a.H + h) * size;
            y = a.back + ((b * a.n_spans + a.n_spans - span) * a.H + h) * size;
        } else if (a.s0) {
            x = a.s0 + (b * a.H + h) * size;
            y = a.gs0 + (b * a.H + h) * size;  // (with the first token's decay already)
        }
        if (x) {
            f32x4_t dot[4] = {};
            const int quads = static_cast<int>(size / 4);
            auto quad = [&](int i, int j) {
                f32x4_t u, v;
                __builtin_memcpy(&u, x + 4 * i, 16);
                __builtin_memcpy(&v, y + 4 * i, 16);
                dot[j] += u * v;
            };
            int i = t;
            for (; i + 768 < quads; i += 1024) {
#pragma unroll
                for (int j = 0; j < 4; ++j) quad(i + 256 * j, j);
            }
            for (; i < quads; i += 256) quad(i, 0);
            if (t < size % 4) dot[0][0] += x[4 * quads + t] * y[4 * quads + t];
            dot[0] = (dot[0] + dot[1]) + (dot[2] + dot[3]);
            const float sum = wave_sum_row3((dot[0][0] + dot[0][1]) + (dot[0][2] + dot[0][3]));
            if (lane == 63) s_sum[w] = sum;
            __syncthreads();
            around = (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]);
            if (span > 0) around *= exp2_f64(log2_decay(a.g[b * a.g_sb + begin * a.g_st + h]));
        }
    }
    float total = 0.f;
    for (int base = begin; base < end; base += W * C) {
        const int first = base + w * C, cnt = min(C, end - first);  // (may be <= 0 for the last waves)
        // r from the last token to the first (lane l: row C - 1 - l), c from the first to the last
        float r = 0.f, c = 0.f, near = 0.f;
        const int back = C - 1 - lane;
        const int64_t row = b * a.T + first;
        if (lane < cnt)
            for (int m = 0; m < G; ++m) near += a.near[(static_cast<int64_t>(h) * G + m) * a.n_rows + row + lane];
        for (int y = 0; y < a.n_tiles; ++y) {
            if (back >= 0 && back < cnt)
                for (int m = 0; m < G; ++m)
                    r += a.r_part[(static_cast<int64_t>(y) * a.Hq + h * G + m) * a.n_rows + row + back];
            if (lane < cnt) c += a.c_part[(static_cast<int64_t>(y) * a.H + h) * a.n_rows + row + lane];
        }
        r = wave_prefix_sum(r);
        c = wave_prefix_sum(c);
        __syncthreads();  // (the chunks before are done with LDS)
        if (lane < C) {
            s_r[w][back] = r;      // the sum over tokens from `back` on
            s_c[w][lane + 1] = c;  // the sum over tokens before lane + 1
        }
        if (lane == 0) s_c[w][0] = 0.f;
        __syncthreads();
        float here = around, dg = 0.f;  // `here`: at this wave's first token
        for (int i = 0; i < w; ++i) here += s_c[i][C] - s_r[i][0];
        for (int i = 0; i < W; ++i) around += s_c[i][C] - s_r[i][0];
        if (lane < cnt) {
            // (the chunk's first token: the gradient handed on, without taking r's sum out and in again)
            dg = lane == 0 ? here : near + s_r[w][lane] + s_c[w][lane] + (here - s_r[w][0]);
            if (a.gg) a.gg[(row + lane) * a.H + h] = dg;
        }
        total += dg;
    }
    if (a.gg_part) {
        total = wave_sum_row3(total);
        __syncthreads();
        if (lane == 63) s_sum[w] = total;
        __syncthreads();
        if (t == 0) a.gg_part[(b * a.n_spans + span) * a.H + h] = (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]);
    }
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

// Packed calls: which sequence and span of it each slot of the grid is, each sequence's first slot, and
// the check of the offsets (launch_varlen_check's bits).  One workgroup; every thread counts the spans of
// its own run of sequences, then writes their slots.  Slots past the last are (-1, 0); where malformed
// offsets overlap, those that would not fit are left out.
__global__ __launch_bounds__(1024) void assign_slots(const int32_t* cu, int n_seqs, int T, int span, int n_slots,
                                                     int2* table, int* first_slot, int32_t* flag) {
    __shared__ int sums[1024];
    const int t = threadIdx.x, per = (n_seqs + 1023) / 1024, i0 = min(t * per, n_seqs), i1 = min(i0 + per, n_seqs);
    auto spans = [&](int i) {
        const int z0 = min(max(cu[i], 0), T), z1 = min(max(cu[i + 1], 0), T);
        return spans_of(z1 - z0, span);
    };
    int n = 0, bits = 0;
    for (int i = i0; i < i1; ++i) {
        n = min(n + spans(i), n_slots);
        if (cu[i + 1] < cu[i]) bits |= 4;
        if (cu[i + 1] < 0 || cu[i + 1] > T) bits |= 8;
    }
    if (t == 0 && cu[0] != 0) bits |= cu[0] < 0 || cu[0] > T ? 9 : 1;
    if (t == 0 && cu[n_seqs] != T) bits |= 2;
    if (bits && flag) atomicOr(flag, bits);
    sums[t] = n;
    for (int m = 1; m < 1024; m <<= 1) {
        __syncthreads();
        const int x = t >= m ? sums[t - m] : 0;
        __syncthreads();
        sums[t] = min(sums[t] + x, n_slots);
    }
    __syncthreads();
    int at = t > 0 ? sums[t - 1] : 0;
    for (int i = i0; i < i1; ++i) {
        const int k = spans(i);
        first_slot[i] = at;
        for (int j = 0; j < k && at < n_slots; ++j, ++at) table[at] = make_int2(i, j);
    }
    for (int j = sums[1023] + t; j < n_slots; j += 1024) table[j] = make_int2(-1, 0);
}

// States before the spans from each span's own share: S = e^G S + U, span after span, V elements of a
// state to a thread (4 where a state's size allows it).  The shares do not wait for each other: 128
// bytes a thread are asked for ahead.
template <int V>
__global__ __launch_bounds__(256) void scan_spans(DecayPasses passes, const int* first_slot) {
    typedef float vec __attribute__((ext_vector_type(V)));
    constexpr int AHEAD = V == 1 ? 32 : 8;
    const DecayPass& a = passes.pass[blockIdx.z % passes.n];
    const int64_t pair = blockIdx.y + static_cast<int64_t>(blockIdx.z / passes.n) * 65535;
    if (pair >= static_cast<int64_t>(a.n_seqs) * a.HS) return;
    const int seq = static_cast<int>(pair / a.HS), h = static_cast<int>(pair % a.HS);
    const int size = a.D * a.D, e = (blockIdx.x * 256 + threadIdx.x) * V;
    if (e >= size) return;
    int len = a.T, slot = seq * a.n_spans;
    if (a.cu) {
        len = max(min(max(a.cu[seq + 1], 0), a.T) - min(max(a.cu[seq], 0), a.T), 0);
        slot = first_slot[seq];
    }
    const int n = min(spans_of(len, a.span), a.n_slots_grid - slot);
    vec S = {};
    if (a.s0) {
        int64_t from = seq;
        bool there = true;
        if (a.slots && !a.s0_gathered) {
            from = a.slots[seq];
            there = from >= 0 && from < a.n_slots;
        }
        if (there) __builtin_memcpy(&S, a.s0 + (from * a.HS + h) * size + e, sizeof S);
    }
    float* u = a.span_state + (static_cast<int64_t>(slot) * a.HS + h) * size + e;
    const double* log = a.span_log + static_cast<int64_t>(slot) * a.HS + h;
    const int64_t step = static_cast<int64_t>(a.HS) * size;
    if (n > 0) __builtin_memcpy(u, &S, sizeof S);
    for (int i = 1; i < n; i += AHEAD) {
        vec x[AHEAD];
        float g[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {  // (past the last: the last again; a branch would wait for each)
            const int64_t from = min(i + j, n - 1);
            __builtin_memcpy(&x[j], u + from * step, sizeof S);
            g[j] = exp2_f64(log[from * a.HS]);
        }
#pragma unroll
        for (int j = 0; j < AHEAD; ++j)
            if (i + j < n) {
                S = g[j] * S + x[j];
                __builtin_memcpy(u + (i + j) * step, &S, sizeof S);
            }
    }
}

constexpr int kMinSpan = 64;

struct Plan {
    int n_tiles, n_dst, span, n_spans, n_slots;
    bool split;
};

// Workgroups of a pass that the card holds at once (registers and LDS: three to a CU up to D 64, two up
// to 128, one beyond).
int64_t resident(int D) { return D <= 64 ? 768 : D <= 128 ? 512 : 256; }

// Whether spans along the sequence pay where there are ``groups`` workgroups without them: the card holds
// ``more`` = resident / groups times as many, each span is walked through twice (the states' own pass costs
// half of the outputs'), and the states are summed in a launch between.  Whole sequences against spans in us,
// forward, by D, heads (one sequence) and tokens:
//   bf16  D 64   16: 20, 23 (256)  28, 23 (384)     128: 37, 31 (512)    256: 71, 63 (1024)  512: 356, 461 (4096)
//         D 96  128: 67, 59 (512)  96, 72 (768)     256: 480, 438 (4096)
//         D 128   1: 29, 31 (256)  40, 32 (384)      64: 54, 53 (512)  75, 58 (768)
//               128: 76, 76 (768)  98, 86 (1024)    256: 197, 219 (2048)  380, 401 (4096)
//         D 192  32: 97, 73 (512)                    64: 185, 169 (1024)
//         D 256  32: 80, 75 (512)  113, 88 (768)     64: 149, 149 (1024)  283, 250 (2048)
//   fp32  D 64  256: 53, 53 (384)  69, 63 (512)
//         D 128  64: 58, 49 (256)  128: 83, 83 (384)  110, 92 (512)  256: 817, 889 (4096)
//         D 256  32: 93, 81 (256)   64: 174, 171 (512)  253, 229 (768)
// D 65 to 128 need three times as many, and longer sequences in bf16 (two workgroups already share a CU;
// D 96 alone would rather be cut earlier), the others twice as many.  Over 1536 such calls of D 32 to 256,
// forward and backward, the rule's choice takes 0.4% more than the better one in the mean, 41% at most, and
// nowhere 5% more than one rule for all, measured at D 128 (which takes 1.1%, 57% at most).
bool spans_pay(int64_t groups, int T, int D, bool bf16) {
    const bool two = D > 64 && D <= 128;
    const int64_t want = resident(D), tokens = bf16 ? (two ? 4096 : 2800) : 1280;
    return want >= (two ? 3 : 2) * groups && T >= (bf16 ? 384 : 256) && T * want >= groups * tokens;
}

// How a pass is cut into workgroups: one per sequence, state and column tile, or, where that pays, as many
// along the sequence as the card holds (spans of at least kMinSpan tokens).  How long packed sequences are
// is not known here: they are cut wherever the card holds more, from 512 tokens on, and half a span of each
// is lost on average.  The query heads of a group go one after another through one workgroup, which reads
// their keys once, where there is work enough for every CU without them.
Plan plan(int n_seqs, int T, int HO, int HS, int D, bool packed, bool bf16) {
    Plan p{(D + decay_cols(D) - 1) / decay_cols(D), 1, max(T, 1), 1, n_seqs, false};
    const int64_t tokens = packed ? T : static_cast<int64_t>(n_seqs) * T, want = resident(D);
    if (HO > HS && tokens * HS * p.n_tiles >= want * 256) p.n_dst = HO / HS;
    const int64_t groups = static_cast<int64_t>(HO / p.n_dst) * p.n_tiles;
    if (packed ? T > 512 && n_seqs * groups < want : spans_pay(n_seqs * groups, T, D, bf16)) {
        int64_t slots = (want + groups - 1) / groups;  // wanted
        if (packed) slots = std::max<int64_t>(want / groups - (n_seqs + 1) / 2, (slots + 1) / 2);
        const int64_t span = std::max<int64_t>((tokens + slots - 1) / slots, kMinSpan);
        const int64_t n = (T + span - 1) / span;
        p.span = static_cast<int>(((T + n - 1) / n + 63) / 64 * 64);
        p.n_spans = spans_of(T, p.span);
        p.n_slots = packed ? T / p.span + n_seqs : n_seqs * p.n_spans;
        p.split = p.n_spans > 1;
    }
    return p;
}

size_t up(size_t n) { return (n + 255) / 256 * 256; }

struct Layout {
    size_t bytes = 0;
    size_t take(size_t n) {
        const size_t at = bytes;
        bytes += up(n);
        return at;
    }
};
struct FwdWs {
    size_t gathered, span_state, span_log, table, first_slot, bytes;
};
// Whether several workgroups read a first state that another one of them may already have replaced.
bool shares_states(const Plan& p, int HO, int HS) { return !p.split && HO / p.n_dst > HS; }
FwdWs fwd_ws(const Plan& p, int n_seqs, int Hq, int H, int D, bool packed, bool in_place) {
    const size_t state = static_cast<size_t>(H) * D * D * 4;
    Layout l;
    FwdWs w{};
    w.gathered = l.take(in_place && shares_states(p, Hq, H) ? n_seqs * state : 0);
    w.span_state = l.take(p.split ? p.n_slots * state : 0);
    w.span_log = l.take(p.split ? static_cast<size_t>(p.n_slots) * H * 8 : 0);
    w.table = l.take(packed ? static_cast<size_t>(p.n_slots) * 8 : 0);
    w.first_slot = l.take(packed ? static_cast<size_t>(n_seqs) * 4 : 0);
    w.bytes = l.bytes;
    return w;
}

// The backward's passes: one cut for all three, which run as one launch.  Where the gates' gradient is
// wanted, spans of at most kDecayGateSpan tokens, also where they do not pay (B8 T4096 H16 bf16, D 128: 898 us
// against 811 for whole sequences, D 256: 3405 against 2509): its sums stay short.
struct BwdPlan {
    Plan q, k;  // gq's pass, and gk's and gv's
};
BwdPlan plan_bwd(int B, int T, int Hq, int H, int D, bool gates, bool bf16) {
    BwdPlan p;
    p.k = Plan{(D + decay_cols(D) - 1) / decay_cols(D), 1, max(T, 1), 1, B, false};
    const int64_t tokens = static_cast<int64_t>(B) * T, want = resident(D);
    int n_dst = 1;
    if (Hq > H && tokens * H * p.k.n_tiles >= want * 256) n_dst = Hq / H;
    const int64_t groups = static_cast<int64_t>(Hq / n_dst + 2 * H) * p.k.n_tiles;
    int64_t span = p.k.span;
    if (spans_pay(B * groups, T, D, bf16)) span = std::max<int64_t>((tokens * groups + want - 1) / want, kMinSpan);
    if (gates) span = std::min<int64_t>(span, kDecayGateSpan);
    if (span < T) {
        const int64_t n = (T + span - 1) / span;
        p.k.span = static_cast<int>(((T + n - 1) / n + 63) / 64 * 64);
        p.k.n_spans = spans_of(T, p.k.span);
        p.k.n_slots = B * p.k.n_spans;
        p.k.split = p.k.n_spans > 1;
    }
    p.q = p.k;
    p.q.n_dst = n_dst;
    return p;
}

struct BwdWs {
    size_t ahead, back, ahead_log, back_log, gs0, r_part, c_part, near, gg_part, bytes;
};
BwdWs bwd_ws(const Plan& p, int B, int T, int Hq, int H, int D, bool gates) {
    const size_t state = static_cast<size_t>(H) * D * D * 4, rows = static_cast<size_t>(B) * T;
    const size_t slots = p.split ? p.n_slots : 0, tiles = p.n_tiles;
    Layout l;
    BwdWs w{};
    w.ahead = l.take(slots * state);
    w.back = l.take(slots * state);
    w.ahead_log = l.take(slots * H * 8);
    w.back_log = l.take(slots * H * 8);
    if (gates) {
        w.gs0 = l.take(B * state);
        w.r_part = l.take(tiles * rows * Hq * 4);
        w.c_part = l.take(tiles * rows * H * 4);
        w.near = l.take(rows * Hq * 4);
        w.gg_part = l.take(static_cast<size_t>(p.n_slots) * H * 4);
    }
    w.bytes = l.bytes;
    return w;
}

template <typename T>
T* at(void* base, size_t off) {
    return reinterpret_cast<T*>(static_cast<char*>(base) + off);
}

hipError_t run_kind(const DecayPasses& a, bool bf16, int kind, hipStream_t st) {
    return bf16 ? decay_pass_bf16(a, kind, st) : decay_pass_f32(a, kind, st);
}

void apply(DecayPass& x, const Plan& p) {
    x.n_tiles = p.n_tiles, x.n_dst = p.n_dst, x.span = p.span, x.n_spans = p.n_spans, x.n_slots_grid = p.n_slots;
}

// K and V change places, and with them a state's rows and columns.
DecayPass turned(DecayPass x) {
    std::swap(x.k, x.v);
    std::swap(x.k_sb, x.v_sb), std::swap(x.k_st, x.v_st), std::swap(x.k_sh, x.v_sh);
    std::swap(x.s_row, x.s_col), std::swap(x.u_row, x.u_col);
    return x;
}

// The states before the spans of each pass, from each span's own share.
hipError_t span_states(DecayPasses x, bool bf16, const int* first_slot, hipStream_t st) {
    for (int i = 0; i < x.n; ++i)  // (the way round that stores a state's rows in 16-byte pieces)
        if (x.pass[i].u_row != 1) x.pass[i] = turned(x.pass[i]);
    if (hipError_t e = run_kind(x, bf16, 2, st); e != hipSuccess) return e;
    const DecayPass& a = x.pass[0];
    const int64_t pairs = static_cast<int64_t>(a.n_seqs) * a.HS;
    // (four elements a thread, where that leaves a workgroup for every CU: 64 heads' 8 spans of D 128 take
    // 12 us, and 36 element by element; 4 heads' 128 spans, bound by the loads in flight, 25.5 and 24)
    const int V = a.D % 2 == 0 && pairs * x.n * a.D * a.D >= 256 * 1024 ? 4 : 1;
    const dim3 grid(static_cast<unsigned>((a.D * a.D / V + 255) / 256), static_cast<unsigned>(std::min<int64_t>(pairs, 65535)),
                    static_cast<unsigned>((pairs + 65534) / 65535 * x.n));
    if (V == 4) hipLaunchKernelGGL(scan_spans<4>, grid, dim3(256), 0, st, x, first_slot);
    else hipLaunchKernelGGL(scan_spans<1>, grid, dim3(256), 0, st, x, first_slot);
    return hipGetLastError();
}

}  // namespace

size_t decay_attn_ws_bytes(int n_seqs, int T, int Hq, int H, int D, bool packed, bool in_place) {
    const Plan x = plan(n_seqs, T, Hq, H, D, packed, true), y = plan(n_seqs, T, Hq, H, D, packed, false);
    return std::max(fwd_ws(x, n_seqs, Hq, H, D, packed, in_place).bytes,
                    fwd_ws(y, n_seqs, Hq, H, D, packed, in_place).bytes);
}
size_t decay_attn_bwd_ws_bytes(int B, int T, int Hq, int H, int D, bool gates) {
    const Plan x = plan_bwd(B, T, Hq, H, D, gates, true).k, y = plan_bwd(B, T, Hq, H, D, gates, false).k;
    return std::max(bwd_ws(x, B, T, Hq, H, D, gates).bytes, bwd_ws(y, B, T, Hq, H, D, gates).bytes);
}
// (as launch_pass has them; in the backward's launch every pass may have a workgroup per query head)
int64_t pass_groups(const Plan& p, int Hq) {
    return (static_cast<int64_t>(p.n_slots) * (Hq / p.n_dst) + 7) / 8 * 8 * p.n_tiles;
}
int64_t decay_attn_groups(int n_seqs, int T, int Hq, int H, int D, bool packed) {
    return std::max(pass_groups(plan(n_seqs, T, Hq, H, D, packed, true), Hq),
                    pass_groups(plan(n_seqs, T, Hq, H, D, packed, false), Hq));
}
int64_t decay_attn_bwd_groups(int B, int T, int Hq, int H, int D) {
    int64_t most = 0;
    for (bool bf16 : {false, true})
        for (bool gates : {false, true}) most = std::max(most, 3 * pass_groups(plan_bwd(B, T, Hq, H, D, gates, bf16).k, Hq));
    return most;
}

hipError_t launch_decay_attn(const DecayAttnArgs& a, hipStream_t st) {
    const bool packed = a.cu != nullptr, in_place = a.s0 && a.s0 == a.s_out;
    const Plan p = plan(a.n_seqs, a.T, a.Hq, a.H, a.D, packed, a.bf16);
    const FwdWs w = fwd_ws(p, a.n_seqs, a.Hq, a.H, a.D, packed, in_place);
    DecayPass x{};
    x.q = a.q, x.k = a.k, x.v = a.v;
    x.q_sb = a.strides[0], x.q_st = a.strides[1], x.q_sh = a.strides[2];
    x.k_sb = a.strides[3], x.k_st = a.strides[4], x.k_sh = a.strides[5];
    x.v_sb = a.strides[6], x.v_st = a.strides[7], x.v_sh = a.strides[8];
    x.g = a.g, x.g_sb = a.g_sb, x.g_st = a.g_st;
    x.cu = a.cu;
    x.s0 = a.s0, x.s_out = a.s_out, x.s_row = x.u_row = a.D, x.s_col = x.u_col = 1;
    x.slots = a.slots, x.n_slots = a.n_slots, x.bad_slot = a.bad_slot;
    x.o = a.o, x.out_bf16 = a.out_bf16;
    x.n_seqs = a.n_seqs, x.T = a.T, x.HO = a.Hq, x.HK = x.HS = a.H, x.D = a.D;
    apply(x, p);
    x.a_scale = x.into_scale = a.scale, x.out_scale = 1.f;
    int* first_slot = nullptr;
    if (packed) {
        int2* table = at<int2>(a.workspace, w.table);
        first_slot = at<int>(a.workspace, w.first_slot);
        hipLaunchKernelGGL(assign_slots, dim3(1), dim3(1024), 0, st, a.cu, a.n_seqs, a.T, p.span, p.n_slots, table,
                           first_slot, a.cu_flag);
        if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
        x.slot_table = table;
    }
    if (in_place && shares_states(p, a.Hq, a.H)) {
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
    if (p.split) {
        x.span_state = at<float>(a.workspace, w.span_state);
        x.span_log = at<double>(a.workspace, w.span_log);
        if (hipError_t e = span_states({{x}, 1}, a.bf16, first_slot, st); e != hipSuccess) return e;
    }
    return run_kind({{x}, 1}, a.bf16, 0, st);
}

hipError_t launch_decay_attn_bwd(const DecayAttnBwdArgs& a, hipStream_t st) {
    const bool gates = a.gg != nullptr;
    const BwdPlan p = plan_bwd(a.B, a.T, a.Hq, a.H, a.D, gates, a.bf16);
    const BwdWs w = bwd_ws(p.k, a.B, a.T, a.Hq, a.H, a.D, gates);
    struct Role {
        const void* p;
        const int64_t* s;
    };
    const int64_t go_strides[3] = {static_cast<int64_t>(a.T) * a.Hq * a.D, static_cast<int64_t>(a.Hq) * a.D, a.D};
    const Role q{a.q, a.strides}, k{a.k, a.strides + 3}, v{a.v, a.strides + 6}, go{a.go, go_strides};
    auto pass = [&](Role Q, Role K, Role V, Role aux, int HO, int HK, const Plan& cut, bool reverse, bool transposed,
                    const float* s0, float* s_out, void* o, bool part) {
        DecayPass x{};
        x.q = Q.p, x.q_sb = Q.s[0], x.q_st = Q.s[1], x.q_sh = Q.s[2];
        x.k = K.p, x.k_sb = K.s[0], x.k_st = K.s[1], x.k_sh = K.s[2];
        x.v = V.p, x.v_sb = V.s[0], x.v_st = V.s[1], x.v_sh = V.s[2];
        x.aux = aux.p, x.x_sb = aux.s[0], x.x_st = aux.s[1], x.x_sh = aux.s[2];
        x.g = a.g, x.g_sb = a.g_sb, x.g_st = a.g_st;
        x.s0 = s0, x.s_out = s_out;
        x.s_row = x.u_row = transposed ? 1 : a.D, x.s_col = x.u_col = transposed ? a.D : 1;
        x.o = o, x.out_bf16 = a.bf16, x.reverse = reverse;
        x.n_seqs = a.B, x.T = a.T, x.HO = HO, x.HK = HK, x.HS = a.H, x.D = a.D;
        apply(x, cut);
        if (cut.split) {
            x.span_state = at<float>(a.workspace, reverse ? w.back : w.ahead);
            x.span_log = at<double>(a.workspace, reverse ? w.back_log : w.ahead_log);
        }
        x.a_scale = a.scale, x.into_scale = reverse ? 1.f : a.scale, x.out_scale = reverse ? a.scale : 1.f;
        if (gates && part) x.part = at<float>(a.workspace, reverse ? w.c_part : w.r_part);
        x.n_rows = static_cast<int64_t>(a.B) * a.T;
        return x;
    };
    float* gs0 = a.gs0 ? a.gs0 : gates && a.s0 ? at<float>(a.workspace, w.gs0) : nullptr;
    const DecayPass gq = pass(go, v, k, q, a.Hq, a.H, p.q, false, true, a.s0, nullptr, a.gq, true);
    const DecayPass gv = pass(k, q, go, k, a.H, a.Hq, p.k, true, false, a.gs, gs0, a.gv, false);
    const DecayPass gk = pass(v, go, q, k, a.H, a.Hq, p.k, true, true, a.gs, nullptr, a.gk, true);
    if (p.k.split)  // (gk's and gv's states are the same, one transposed)
        if (hipError_t e = span_states({{gq, gk}, 2}, a.bf16, nullptr, st); e != hipSuccess) return e;
    if (hipError_t e = run_kind({{gq, gv, gk}, 3}, a.bf16, gates ? 1 : 0, st); e != hipSuccess) return e;
    if (!gates) return hipSuccess;
    const bool constant = a.g_sb == 0 && a.g_st == 0;
    if (a.T > 0) {
        float* near = at<float>(a.workspace, w.near);
        DecayNear n{};
        n.q = q.p, n.q_sb = q.s[0], n.q_st = q.s[1], n.q_sh = q.s[2];
        n.k = k.p, n.k_sb = k.s[0], n.k_st = k.s[1], n.k_sh = k.s[2];
        n.v = v.p, n.v_sb = v.s[0], n.v_st = v.s[1], n.v_sh = v.s[2];
        n.go = go.p, n.go_sb = go.s[0], n.go_st = go.s[1], n.go_sh = go.s[2];
        n.g = a.g, n.g_sb = a.g_sb, n.g_st = a.g_st;
        n.near = near, n.n_rows = static_cast<int64_t>(a.B) * a.T;
        n.B = a.B, n.T = a.T, n.Hq = a.Hq, n.H = a.H, n.D = a.D, n.scale = a.scale;
        if (hipError_t e = a.bf16 ? decay_near_bf16(n, st) : decay_near_f32(n, st); e != hipSuccess) return e;
        DecayGateGrad x{};
        x.g = a.g, x.g_sb = a.g_sb, x.g_st = a.g_st;
        x.r_part = gq.part, x.c_part = gk.part, x.near = near;
        x.ahead = gq.span_state, x.back = gk.span_state, x.s0 = a.s0, x.gs0 = gs0;
        x.gg = constant ? nullptr : a.gg, x.gg_part = constant ? at<float>(a.workspace, w.gg_part) : nullptr;
        x.n_rows = static_cast<int64_t>(a.B) * a.T;
        x.B = a.B, x.T = a.T, x.Hq = a.Hq, x.H = a.H, x.D = a.D;
        x.n_tiles = p.k.n_tiles, x.span = p.k.span, x.n_spans = p.k.n_spans, x.chunk = a.bf16 ? 64 : 32;
        const int64_t groups = static_cast<int64_t>(a.B) * a.H * p.k.n_spans;
        hipLaunchKernelGGL(gate_grad, dim3(static_cast<unsigned>(groups)), dim3(256), 0, st, x);
        if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    if (constant) {
        hipLaunchKernelGGL(sum_gate_parts, dim3(static_cast<unsigned>(a.H)), dim3(256), 0, st,
                           at<float>(a.workspace, w.gg_part), a.gg, a.T > 0 ? static_cast<int64_t>(p.k.n_slots) : 0, a.H);
        return hipGetLastError();
    }
    return hipSuccess;
}

// ---- one token --------------------------------------------------------------------------------
//
// S = e^g S + k v^T in place, o = scale S^T q for the group's query heads: the state is read and
// written once, 16 bytes a lane (K3's mapping), and everything else is small beside it.  CG column
// groups of 4, 256 / CG row groups.  More than 4 query heads take the new state from the caches
// again, 4 at a time.  256 tokens of 32 query and 8 key heads, D 128: 274 MB in 58 us, 4.7 TB/s (71 us
// with loads and stores that stay in the caches; a copy of 2 GiB runs at 5.0 TB/s here).
namespace {

typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));  // at any address of a float

template <int CG, typename E>
__global__ __launch_bounds__(256, 4) void decay_step(DecayAttnStepArgs a, int b0) {
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
                if (left >= 4) x = __builtin_nontemporal_load(reinterpret_cast<const f32x4_any*>(p));
                else
                    for (int r = 0; r < left; ++r) x[r] = p[r];
                if (m0 == 0) {
                    x = e * x + sk[d] * vv;
                    if (left >= 4) __builtin_nontemporal_store(x, reinterpret_cast<f32x4_any*>(p));
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
