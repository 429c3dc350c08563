// norm_rotate.hip — K13: the norms of q's and k's heads and the position rotation, in one pass,
// and their gradients.
//
// For one head of one token, x of D elements, u = r x with
//   l2:  r = 1 / max(||x||, eps)          rms:  r = 1 / sqrt(mean x^2 + eps)
// y = u w, and the first R elements are turned in pairs by the angles of the token's position:
//   z1 = y1 cos - y2 sin,  z2 = y2 cos + y1 sin.
// Backward: gy is gz turned back, gw sums gy u over all rows, gu = gy w, and
//   l2:  gx = r (gu - u <gu, u>)  (r gu where ||x|| <= eps)     rms:  gx = r (gu - u <gu, u> / D)
//
// One wave to a row; any D up to 256, any strides and alignment.

#include "pm_common.h"
#include "pm_internal.h"

namespace pm {

constexpr int kRowMax = 256;  // largest D
constexpr int kPer = kRowMax / 64;

__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) x += __shfl_xor(x, m);
    return x;
}

// A row's place: side (q or k), batch row, token and head, from its index among
// B * T * (Hq + Hk) rows, tokens outermost.
struct Row {
    int side, b, t, h;
    int64_t in, out;
};
__device__ __forceinline__ Row row_of(const NormRotateArgs& a, int64_t r) {
    const int heads = a.H[0] + a.H[1];
    const int64_t tok = r / heads;
    int h = static_cast<int>(r - tok * heads);
    Row w;
    w.side = h >= a.H[0];
    if (w.side) h -= a.H[0];
    w.h = h;
    w.b = static_cast<int>(tok / a.T);
    w.t = static_cast<int>(tok - static_cast<int64_t>(w.b) * a.T);
    w.in = w.b * a.sb[w.side] + w.t * a.st[w.side] + h * a.sh[w.side];
    w.out = (tok * a.H[w.side] + h) * a.D;
    return w;
}

// The table's row of a token, or -1 where its position is outside the table: such rows of the
// outputs (and gradients) are NaN, and nothing outside the table is read.
__device__ __forceinline__ int64_t table_row(const NormRotateArgs& a, int b, int t) {
    int64_t p = t;
    if (a.pos) {
        const int64_t i = b * a.pos_sb + t;
        p = a.pos64 ? static_cast<const int64_t*>(a.pos)[i] : static_cast<const int32_t*>(a.pos)[i];
    }
    return p >= 0 && p < a.P ? p : -1;
}

__device__ __forceinline__ float weight_at(const NormRotateArgs& a, int side, int e) {
    const void* w = a.weight[side];
    if (!w) return 1.f;
    return a.w_bf16 ? bf16_to_f32(static_cast<const uint16_t*>(w)[e]) : static_cast<const float*>(w)[e];
}

// r of a row from its sum of squares (NaN stays NaN; `clipped`: l2 at or below eps)
__device__ __forceinline__ float row_scale(const NormRotateArgs& a, float ss, bool& clipped) {
    clipped = false;
    if (a.rms) return 1.f / sqrtf(ss / static_cast<float>(a.D) + a.eps);
    const float n = sqrtf(ss);
    clipped = n <= a.eps;
    return 1.f / (clipped ? a.eps : n);
}

// A row held by a wave, element lane + 64 j in v[j], turned by its position's angles (dir 1) or
// back (dir -1).  `buf` is the wave's own LDS row.
__device__ __forceinline__ void turn(const NormRotateArgs& a, int64_t trow, float dir, float (&v)[kPer], float* buf) {
    const int lane = threadIdx.x & 63, half = a.R / 2;
    const float nan = __uint_as_float(0x7fc00000u);
#pragma unroll
    for (int j = 0; j < kPer; ++j) buf[lane + 64 * j] = v[j];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const int e = lane + 64 * j;
        if (e < a.R) {
            const int p = a.interleaved ? e >> 1 : (e < half ? e : e - half);
            const bool first = a.interleaved ? !(e & 1) : e < half;
            const float other = buf[a.interleaved ? e ^ 1 : (first ? e + half : e - half)];
            const float c = trow < 0 ? nan : a.table[trow * a.R + p];
            const float s = trow < 0 ? nan : a.table[trow * a.R + half + p] * dir;
            v[j] = first ? fmaf(v[j], c, -other * s) : fmaf(v[j], c, other * s);
        } else if (trow < 0) {
            v[j] = nan;
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

template <typename E>
__global__ __launch_bounds__(256) void norm_rotate_kernel(NormRotateArgs a, int64_t rows) {
    __shared__ float buf[4][kRowMax];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t stride = static_cast<int64_t>(gridDim.x) * 4;
    for (int64_t r = static_cast<int64_t>(blockIdx.x) * 4 + w; r < rows; r += stride) {
        const Row at = row_of(a, r);
        const E* x = static_cast<const E*>(a.x[at.side]) + at.in;
        float v[kPer], ss = 0.f;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const int e = lane + 64 * j;
            v[j] = e < a.D ? to_f32(x[e]) : 0.f;
            ss = fmaf(v[j], v[j], ss);
        }
        bool clipped;
        const float scale = row_scale(a, wave_sum(ss), clipped);
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const int e = lane + 64 * j;
            v[j] = e < a.D ? v[j] * scale * weight_at(a, at.side, e) : 0.f;
        }
        if (a.table) turn(a, table_row(a, at.b, at.t), 1.f, v, buf[w]);
        E* y = static_cast<E*>(a.y[at.side]) + at.out;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const int e = lane + 64 * j;
            if (e < a.D) y[e] = from_f32<E>(v[j]);
        }
    }
}

// Each workgroup sums its rows' shares of the weights' gradients (its waves in order) into
// part[block][side][D]; weight_grad_kernel adds the workgroups' in order, so that the sums
// do not depend on which finishes first.
template <typename E>
__global__ __launch_bounds__(256) void norm_rotate_bwd_kernel(NormRotateArgs a, int64_t rows, float* part) {
    __shared__ float buf[4][kRowMax];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t stride = static_cast<int64_t>(gridDim.x) * 4;
    float gw[2][kPer] = {};
    for (int64_t r = static_cast<int64_t>(blockIdx.x) * 4 + w; r < rows; r += stride) {
        const Row at = row_of(a, r);
        const E* x = static_cast<const E*>(a.x[at.side]) + at.in;
        const E* gz = static_cast<const E*>(a.gy[at.side]);
        float u[kPer], gy[kPer], ss = 0.f, dot = 0.f;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const int e = lane + 64 * j;
            u[j] = e < a.D ? to_f32(x[e]) : 0.f;
            gy[j] = e < a.D && gz ? to_f32(gz[at.out + e]) : 0.f;
            ss = fmaf(u[j], u[j], ss);
        }
        bool clipped;
        const float scale = row_scale(a, wave_sum(ss), clipped);
        if (a.table) turn(a, table_row(a, at.b, at.t), -1.f, gy, buf[w]);
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const int e = lane + 64 * j;
            u[j] = e < a.D ? u[j] * scale : 0.f;
            if (e >= a.D) gy[j] = 0.f;
            if (at.side) gw[1][j] = fmaf(gy[j], u[j], gw[1][j]);
            else gw[0][j] = fmaf(gy[j], u[j], gw[0][j]);
            if (e < a.D) gy[j] *= weight_at(a, at.side, e);
            dot = fmaf(gy[j], u[j], dot);
        }
        dot = wave_sum(dot);
        if (a.rms) dot /= static_cast<float>(a.D);
        E* gx = static_cast<E*>(a.gx[at.side]) + at.out;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const int e = lane + 64 * j;
            if (e < a.D) gx[e] = from_f32<E>((clipped ? gy[j] : fmaf(-u[j], dot, gy[j])) * scale);
        }
    }
    if (!part) return;
    for (int side = 0; side < 2; ++side) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kPer; ++j) buf[w][lane + 64 * j] = side ? gw[1][j] : gw[0][j];
        __syncthreads();
        const int e = threadIdx.x;
        if (e < a.D)
            part[(static_cast<int64_t>(blockIdx.x) * 2 + side) * a.D + e] =
                (buf[0][e] + buf[1][e]) + (buf[2][e] + buf[3][e]);
    }
}

__global__ __launch_bounds__(256) void weight_grad_kernel(const float* part, int blocks, int D, float* gq, float* gk) {
    const int side = blockIdx.x, e = threadIdx.x;
    float* out = side ? gk : gq;
    if (!out || e >= D) return;
    float s = 0.f;
    for (int i = 0; i < blocks; ++i) s += part[(static_cast<int64_t>(i) * 2 + side) * D + e];
    out[e] = s;
}

static int row_blocks(int64_t rows, int most) {
    const int64_t b = (rows + 3) / 4;
    return static_cast<int>(b < most ? b : most);
}
constexpr int kBwdBlocks = 1024;

hipError_t launch_norm_rotate(const NormRotateArgs& a, hipStream_t st) {
    const int64_t rows = static_cast<int64_t>(a.B) * a.T * (a.H[0] + a.H[1]);
    const dim3 grid(static_cast<unsigned>(row_blocks(rows, 1 << 20)));
    if (a.bf16) hipLaunchKernelGGL(norm_rotate_kernel<uint16_t>, grid, dim3(256), 0, st, a, rows);
    else hipLaunchKernelGGL(norm_rotate_kernel<float>, grid, dim3(256), 0, st, a, rows);
    return hipGetLastError();
}

size_t norm_rotate_bwd_ws_bytes(int B, int T, int Hq, int Hk, int D) {
    const int64_t rows = static_cast<int64_t>(B) * T * (static_cast<int64_t>(Hq) + Hk);
    return static_cast<size_t>(row_blocks(rows, kBwdBlocks)) * 2 * D * sizeof(float);
}

hipError_t launch_norm_rotate_bwd(const NormRotateArgs& a, hipStream_t st) {
    const int64_t rows = static_cast<int64_t>(a.B) * a.T * (a.H[0] + a.H[1]);
    const int blocks = row_blocks(rows, kBwdBlocks);
    float* part = a.gw[0] || a.gw[1] ? static_cast<float*>(a.workspace) : nullptr;
    const dim3 grid(static_cast<unsigned>(blocks));
    if (a.bf16) hipLaunchKernelGGL(norm_rotate_bwd_kernel<uint16_t>, grid, dim3(256), 0, st, a, rows, part);
    else hipLaunchKernelGGL(norm_rotate_bwd_kernel<float>, grid, dim3(256), 0, st, a, rows, part);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || !part) return e;
    hipLaunchKernelGGL(weight_grad_kernel, dim3(2), dim3(256), 0, st, part, blocks, a.D, a.gw[0], a.gw[1]);
    return hipGetLastError();
}

}  // namespace pm
