// gated_norm.hip — K15: the norm of a layer's output rows with its weight and gate.
//
//   act(z) = z s (silu) or s (sigmoid), s = 1 / (1 + e^-z)
//   y = r x w act(z),        r = 1 / sqrt(mean x^2 + eps)               (gate after the norm)
//   y = r u w, u = x act(z), r = 1 / sqrt(mean u^2 + eps)               (gate before the norm)
// With n = r u (u = x where the gate comes after) and p = gy w [act(z)] the gradients are
//   gu = r (p - n mean(p n)),  gw = sum gy n [act(z)],  gz = act'(z) times gy n w, or gu x.
// mean(p n) = r mean(p u): both sums over the row are taken together.
//
// Every tensor is read and written once, in 16-byte pieces, so HBM bounds it; a workgroup keeps its
// weights in registers and walks through rows.  262,144 rows of 128 in bf16: forward 38 us (201 MB,
// 5.3 TB/s), backward 65 us (336 MB, 5.2 TB/s) and 4 us for the sum of the weight's gradient; a copy of
// 2 GiB runs at 5.0 TB/s here.

#include "pm_internal.h"
#include "pm_rows.h"
#include "pm_cdna4.h"

namespace pm {
namespace {

struct Act {
    float a, slope;
};
// With e = e^-|z|: s = 1 / (1 + e) or e / (1 + e), and its slope s (1 - s) = e / (1 + e)^2, which keeps its
// digits where the gate is wide open (1 - s has lost them at z = 16).
__device__ __forceinline__ Act act_of(float z, bool silu) {
    const float e = exp2_hw(fabsf(z) * -1.44269504f), r = __builtin_amdgcn_rcpf(1.f + e);
    const float s = z < 0.f ? e * r : r, d = e * r * r;
    return silu ? Act{z * s, s + z * d} : Act{s, d};
}

__device__ __forceinline__ int64_t row_at(int64_t row, int inner, int64_t so, int64_t si) {
    if (inner == 1) return row * so;
    const int64_t o = row / inner;
    return o * so + (row - o * inner) * si;
}

template <int M, int L, int NV, bool BWD>
__global__ __launch_bounds__(threads_of(L)) void gated_norm_kernel(GatedNormArgs a) {
    constexpr int GROUPS = threads_of(L) / L;
    __shared__ float red[L >= 256 ? 2 : 1][2][16];
    __shared__ float lds[BWD && L < 256 ? GROUPS * 8 * L * NV : 1];
    const int lane = threadIdx.x % L, group = threadIdx.x / L, C = a.C;
    int turn = 0;
    RowRegs<kMixed, NV, L> w;
    if (a.w) w.load(a.w, a.w_bf16, 0, lane, C);
    else w.fill(1.f);
    float gw[NV][8] = {};
    const int64_t rows = a.rows, step = static_cast<int64_t>(gridDim.x) * GROUPS;
    const float inv = 1.f / static_cast<float>(C);
    for (int64_t row0 = static_cast<int64_t>(blockIdx.x) * GROUPS; row0 < rows; row0 += step) {
        const int64_t row = row0 + group;
        if (L < 256 && row >= rows) break;  // (no barrier inside the loop where a group is not the workgroup)
        RowRegs<M, NV, L> x, z, gy;
        x.load(a.x, a.x_bf16, row_at(row, a.inner, a.x_so, a.x_si), lane, C);
        z.load(a.z, a.z_bf16, row_at(row, a.inner, a.z_so, a.z_si), lane, C);
        if (BWD) gy.load(a.gy, a.y_bf16, row * C, lane, C);
        float sums[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float act = act_of(z.v[i][j], a.silu).a;
                const float u = a.first ? x.v[i][j] * act : x.v[i][j];
                sums[0] += u * u;
                if (BWD) sums[1] += gy.v[i][j] * (a.first ? w.v[i][j] : w.v[i][j] * act) * u;
            }
        group_sum<L, 2>(sums, red, turn);
        const float r = 1.f / sqrtf(sums[0] * inv + a.eps);
        const float mean = r * sums[1] * inv;
        RowRegs<M, NV, L> gz;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const Act act = act_of(z.v[i][j], a.silu);
                const float xv = x.v[i][j], n = r * (a.first ? xv * act.a : xv);
                if (!BWD) {
                    x.v[i][j] = a.first ? n * w.v[i][j] : n * w.v[i][j] * act.a;
                    continue;
                }
                const float g = a.first ? gy.v[i][j] : gy.v[i][j] * act.a;
                gw[i][j] += g * n;
                const float gu = r * (g * w.v[i][j] - n * mean);
                x.v[i][j] = a.first ? gu * act.a : gu;
                gz.v[i][j] = (a.first ? gu * xv : gy.v[i][j] * n * w.v[i][j]) * act.slope;
            }
        if (BWD) {
            x.store(a.gx, a.x_bf16, row * C, lane, C);
            gz.store(a.gz, a.z_bf16, row * C, lane, C);
        } else {
            x.store(a.y, a.y_bf16, row * C, lane, C);
        }
    }
    if (BWD && a.gw) store_part<NV, L>(gw, lds, a.part, C);
}

template <int M, bool BWD>
struct Launch {
    const GatedNormArgs& a;
    hipStream_t st;
    template <int L, int NV>
    hipError_t run() const {
        const int64_t n = row_groups(a.rows, a.C, BWD);
        hipLaunchKernelGGL((gated_norm_kernel<M, L, NV, BWD>), dim3(static_cast<unsigned>(n)), dim3(threads_of(L)), 0, st, a);
        return hipGetLastError();
    }
};

template <bool BWD>
hipError_t by_types(const GatedNormArgs& a, hipStream_t st) {
    if (a.x_bf16 && a.z_bf16 && a.y_bf16) return by_width(a.C, Launch<kAllBf16, BWD>{a, st});
    if (!a.x_bf16 && !a.z_bf16 && !a.y_bf16) return by_width(a.C, Launch<kAllF32, BWD>{a, st});
    return by_width(a.C, Launch<kMixed, BWD>{a, st});
}

}  // namespace

int64_t gated_norm_groups(int64_t rows, int C) { return row_groups(rows, C, true); }

hipError_t launch_gated_norm(const GatedNormArgs& a, hipStream_t st) { return by_types<false>(a, st); }

hipError_t launch_gated_norm_bwd(const GatedNormArgs& a, hipStream_t st) {
    if (hipError_t e = by_types<true>(a, st); e != hipSuccess || !a.gw) return e;
    return launch_row_parts(a.part, {{a.gw, nullptr}}, static_cast<int>(gated_norm_groups(a.rows, a.C)), a.C, st);
}

}  // namespace pm
