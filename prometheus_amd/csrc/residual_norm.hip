// residual_norm.hip — K16: the norm after a block, the sum with the residual and the norm before the next.
//
//   b = x, or with a weight for it  b = rp x wp,  rp = 1 / sqrt(mean x^2 + eps)
//   h = residual + scale b,         y = r h w,    r = 1 / sqrt(mean h^2 + eps)
// y comes from the unrounded h.  With n = r h, p = gy w, np = rp x, pp = scale dh wp the gradients are
//   dh = gh + r (p - n mean(p n)),  gw = sum gy n,
//   gx = scale dh, or rp (pp - np mean(pp np)),  gwp = sum scale dh np.
// The backward takes h from x and the residual again, so that nothing depends on how h was rounded.
//
// Every tensor is read and written once, in 16-byte pieces, so HBM bounds it.  16,384 rows of 4096 in bf16,
// both norms: forward 103 us (537 MB, 5.2 TB/s), backward 165 us (805 MB, 4.9 TB/s) and 8 us for the sums of
// the weights' gradients; a copy of 2 GiB runs at 5.0 TB/s here.

#include "pm_internal.h"
#include "pm_rows.h"

namespace pm {
namespace {

template <int M, int L, int NV, bool BWD, bool POST>
__global__ __launch_bounds__(threads_of(L)) void residual_norm_kernel(ResidualNormArgs a) {
    constexpr int GROUPS = threads_of(L) / L;
    __shared__ float red1[L >= 256 ? 2 : 1][1][16], red2[L >= 256 ? 2 : 1][2][16];
    __shared__ float lds[BWD && L < 256 ? GROUPS * 8 * L * NV : 1];
    const int lane = threadIdx.x % L, group = threadIdx.x / L, C = a.C;
    int turn1 = 0, turn2 = 0;
    RowRegs<kMixed, NV, L> w, wp;
    if (a.w) w.load(a.w, a.w_bf16, 0, lane, C);
    else w.fill(1.f);
    if (POST) wp.load(a.wp, a.wp_bf16, 0, lane, C);
    float gw[NV][8] = {}, gwp[POST ? NV : 1][8] = {};
    const int64_t rows = a.rows, step = static_cast<int64_t>(gridDim.x) * GROUPS;
    const float inv = 1.f / static_cast<float>(C);
    for (int64_t row0 = static_cast<int64_t>(blockIdx.x) * GROUPS; row0 < rows; row0 += step) {
        const int64_t row = row0 + group;
        if (L < 256 && row >= rows) break;
        RowRegs<M, NV, L> x, h, gy, gh;
        x.load(a.x, a.x_bf16, row * a.x_st, lane, C);
        h.load(a.res, a.r_bf16, row * a.r_st, lane, C);
        if (BWD) {
            if (a.gy) gy.load(a.gy, a.x_bf16, row * C, lane, C);
            else gy.fill(0.f);
            if (a.gh) gh.load(a.gh, a.r_bf16, row * C, lane, C);
            else gh.fill(0.f);
        }
        float rp = 1.f;
        if (POST) {
            float s[1] = {0.f};
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) s[0] += x.v[i][j] * x.v[i][j];
            group_sum<L, 1>(s, red1, turn1);
            rp = 1.f / sqrtf(s[0] * inv + a.eps);
        }
        float sums[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float b = POST ? rp * x.v[i][j] * wp.v[i][j] : x.v[i][j];
                h.v[i][j] += a.scale * b;
                sums[0] += h.v[i][j] * h.v[i][j];
                if (BWD) sums[1] += gy.v[i][j] * w.v[i][j] * h.v[i][j];
            }
        group_sum<L, 2>(sums, red2, turn2);
        const float r = 1.f / sqrtf(sums[0] * inv + a.eps);
        if (!BWD) {
            h.store(a.h, a.r_bf16, row * C, lane, C);
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) h.v[i][j] *= r * w.v[i][j];
            h.store(a.y, a.x_bf16, row * C, lane, C);
            continue;
        }
        const float mean = r * sums[1] * inv;
        float s[1] = {0.f};
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float n = r * h.v[i][j];
                gw[i][j] += gy.v[i][j] * n;
                const float dh = gh.v[i][j] + r * (gy.v[i][j] * w.v[i][j] - n * mean);
                h.v[i][j] = dh;
                if (POST) {
                    const float g = a.scale * dh, np = rp * x.v[i][j];
                    gwp[i][j] += g * np;
                    s[0] += g * wp.v[i][j] * np;
                }
            }
        h.store(a.gres, a.r_bf16, row * C, lane, C);
        if (POST) group_sum<L, 1>(s, red1, turn1);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float g = a.scale * h.v[i][j];
                x.v[i][j] = POST ? rp * (g * wp.v[i][j] - rp * x.v[i][j] * (s[0] * inv)) : g;
            }
        x.store(a.gx, a.x_bf16, row * C, lane, C);
    }
    if (BWD && a.gw) store_part<NV, L>(gw, lds, a.part, C);
    if constexpr (BWD && POST)
        if (a.gwp) store_part<NV, L>(gwp, lds, a.part + static_cast<int64_t>(gridDim.x) * C, C);
}

template <int M, bool BWD>
struct Launch {
    const ResidualNormArgs& a;
    hipStream_t st;
    template <int L, int NV>
    hipError_t run() const {
        const dim3 grid(static_cast<unsigned>(row_groups(a.rows, a.C, BWD)));
        if (a.wp) hipLaunchKernelGGL((residual_norm_kernel<M, L, NV, BWD, true>), grid, dim3(threads_of(L)), 0, st, a);
        else hipLaunchKernelGGL((residual_norm_kernel<M, L, NV, BWD, false>), grid, dim3(threads_of(L)), 0, st, a);
        return hipGetLastError();
    }
};

template <bool BWD>
hipError_t by_types(const ResidualNormArgs& a, hipStream_t st) {
    if (a.x_bf16 && a.r_bf16) return by_width(a.C, Launch<kAllBf16, BWD>{a, st});
    if (!a.x_bf16 && !a.r_bf16) return by_width(a.C, Launch<kAllF32, BWD>{a, st});
    return by_width(a.C, Launch<kMixed, BWD>{a, st});
}

}  // namespace

int64_t residual_norm_groups(int64_t rows, int C) { return row_groups(rows, C, true); }

hipError_t launch_residual_norm(const ResidualNormArgs& a, hipStream_t st) { return by_types<false>(a, st); }

hipError_t launch_residual_norm_bwd(const ResidualNormArgs& a, hipStream_t st) {
    if (hipError_t e = by_types<true>(a, st); e != hipSuccess || !(a.gw || a.gwp)) return e;
    return launch_row_parts(a.part, {{a.gw, a.gwp}}, static_cast<int>(residual_norm_groups(a.rows, a.C)), a.C, st);
}

}  // namespace pm
