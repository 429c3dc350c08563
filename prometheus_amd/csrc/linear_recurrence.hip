// linear_recurrence.hip — K12: the elementwise gated linear recurrence, its gradients and its
// single-token step.
//
//   h_t = exp(g_t) h_{t-1} + x_t          for every channel on its own
//   d_t = gh_t + exp(g_{t+1}) d_{t+1},  gx_t = d_t,  gg_t = d_t exp(g_t) h_{t-1}
//
// One thread walks one channel of one sequence.

#include "pm_common.h"
#include "pm_internal.h"

namespace pm {

// Row of a sequence's state in s0 and s_out, or -1 (a slot outside the pool).
__device__ __forceinline__ int64_t state_row(const int32_t* slots, int n_slots, int seq) {
    if (!slots) return seq;
    const int r = slots[seq];
    return r >= 0 && r < n_slots ? r : -1;
}

template <typename X, typename G, typename H>
__global__ __launch_bounds__(256) void recurrence_kernel(RecurrenceArgs a) {
    const int c = static_cast<int>(blockIdx.x) * 256 + static_cast<int>(threadIdx.x);
    for (int seq = blockIdx.y; seq < a.n_seqs; seq += gridDim.y) {
        const int64_t row = state_row(a.slots, a.n_slots, seq);
        if (row < 0 && a.bad && c == 0) atomicOr(a.bad, 1);
        if (c >= a.C) continue;
        int t0 = 0, t1 = a.T;
        int64_t xb = seq * a.x_sb, gb = seq * a.g_sb, hb = static_cast<int64_t>(seq) * a.T * a.C;
        if (a.cu_seqlens) {
            t0 = min(max(a.cu_seqlens[seq], 0), a.T);
            t1 = min(max(a.cu_seqlens[seq + 1], t0), a.T);
            xb = gb = hb = 0;
        }
        float s = a.s0 && row >= 0 ? a.s0[row * a.C + c] : 0.f;
        for (int t = t0; t < t1; ++t) {
            if (a.kept && (t - t0) % kRecSpan == 0) {
                const int64_t spans = (a.T + kRecSpan - 1) / kRecSpan;
                a.kept[(seq * spans + t / kRecSpan) * a.C + c] = s;
            }
            const float x = to_f32(static_cast<const X*>(a.x)[xb + t * a.x_st + c]);
            const float g = to_f32(static_cast<const G*>(a.g)[gb + t * a.g_st + c]);
            s = fmaf(expf(g), s, x);
            static_cast<H*>(a.h)[hb + static_cast<int64_t>(t) * a.C + c] = from_f32<H>(s);
        }
        if (row >= 0) a.s_out[row * a.C + c] = s;
    }
}

template <typename X, typename G, typename H>
__global__ __launch_bounds__(256) void recurrence_bwd_kernel(RecurrenceBwdArgs a) {
    const int c = static_cast<int>(blockIdx.x) * 256 + static_cast<int>(threadIdx.x);
    if (c >= a.C) return;
    const int64_t spans = (a.T + kRecSpan - 1) / kRecSpan;
    for (int b = blockIdx.y; b < a.B; b += gridDim.y) {
        const X* x = static_cast<const X*>(a.x) + b * a.x_sb + c;
        const G* g = static_cast<const G*>(a.g) + b * a.g_sb + c;
        const int64_t out = static_cast<int64_t>(b) * a.T * a.C + c;
        float carry = a.gs ? a.gs[static_cast<int64_t>(b) * a.C + c] : 0.f;  // exp(g_{t+1}) d_{t+1}
        for (int64_t p = spans - 1; p >= 0; --p) {
            const int t0 = static_cast<int>(p) * kRecSpan, n = min(kRecSpan, a.T - t0);
            float before[kRecSpan];
            float s = a.kept[(b * spans + p) * a.C + c];
            for (int i = 0; i < n; ++i) {
                before[i] = s;
                s = fmaf(expf(to_f32(g[(t0 + i) * a.g_st])), s, to_f32(x[(t0 + i) * a.x_st]));
            }
            for (int i = n - 1; i >= 0; --i) {
                const int64_t o = out + static_cast<int64_t>(t0 + i) * a.C;
                const float d = (a.gh ? to_f32(static_cast<const H*>(a.gh)[o]) : 0.f) + carry;
                carry = expf(to_f32(g[(t0 + i) * a.g_st])) * d;
                static_cast<X*>(a.gx)[o] = from_f32<X>(d);
                static_cast<G*>(a.gg)[o] = from_f32<G>(carry * before[i]);
            }
        }
        a.gs0[static_cast<int64_t>(b) * a.C + c] = carry;
    }
}

template <typename X, typename G, typename H>
__global__ __launch_bounds__(256) void recurrence_step_kernel(RecurrenceStepArgs a) {
    const int c = static_cast<int>(blockIdx.x) * 256 + static_cast<int>(threadIdx.x);
    if (c >= a.C) return;
    for (int b = blockIdx.y; b < a.B; b += gridDim.y) {
        const int64_t row = state_row(a.slots, a.n_slots, b);
        float s = 0.f;
        if (row >= 0) {
            s = fmaf(expf(to_f32(static_cast<const G*>(a.g)[b * a.g_sb + c])), a.s[row * a.C + c],
                     to_f32(static_cast<const X*>(a.x)[b * a.x_sb + c]));
            a.s[row * a.C + c] = s;
        }
        static_cast<H*>(a.h)[static_cast<int64_t>(b) * a.C + c] = from_f32<H>(s);
    }
}

// f(x, g, h) with a null pointer of each tensor's element type
template <typename F>
static void by_types(bool x_bf16, bool g_bf16, bool h_bf16, F f) {
    const uint16_t* b = nullptr;
    const float* s = nullptr;
    if (x_bf16 && g_bf16) h_bf16 ? f(b, b, b) : f(b, b, s);
    else if (x_bf16) h_bf16 ? f(b, s, b) : f(b, s, s);
    else h_bf16 ? f(s, s, b) : f(s, s, s);
}

template <typename A, typename K>
static hipError_t launch_rows(K kernel, const A& a, int rows, int C, hipStream_t st) {
    const dim3 grid(static_cast<unsigned>((C + 255) / 256), static_cast<unsigned>(rows < 65535 ? rows : 65535));
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, a);
    return hipGetLastError();
}

#define PM_ELEM(p) std::remove_const_t<std::remove_pointer_t<decltype(p)>>

hipError_t launch_recurrence(const RecurrenceArgs& a, hipStream_t st) {
    hipError_t e = hipSuccess;
    by_types(a.x_bf16, a.g_bf16, a.h_bf16, [&](auto x, auto g, auto h) {
        e = launch_rows(recurrence_kernel<PM_ELEM(x), PM_ELEM(g), PM_ELEM(h)>, a, a.n_seqs, a.C, st);
    });
    return e;
}

hipError_t launch_recurrence_bwd(const RecurrenceBwdArgs& a, hipStream_t st) {
    hipError_t e = hipSuccess;
    by_types(a.x_bf16, a.g_bf16, a.h_bf16, [&](auto x, auto g, auto h) {
        e = launch_rows(recurrence_bwd_kernel<PM_ELEM(x), PM_ELEM(g), PM_ELEM(h)>, a, a.B, a.C, st);
    });
    return e;
}

hipError_t launch_recurrence_step(const RecurrenceStepArgs& a, hipStream_t st) {
    hipError_t e = hipSuccess;
    by_types(a.x_bf16, a.g_bf16, a.h_bf16, [&](auto x, auto g, auto h) {
        e = launch_rows(recurrence_step_kernel<PM_ELEM(x), PM_ELEM(g), PM_ELEM(h)>, a, a.B, a.C, st);
    });
    return e;
}

}  // namespace pm
