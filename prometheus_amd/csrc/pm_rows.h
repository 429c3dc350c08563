// pm_rows.h — rows of C elements spread over groups of lanes, for the norms of whole rows.
//
// A group of L lanes holds a row, 8 NV elements a lane: lane l the elements 8 (l + L i) + [0, 8),
// i < NV, so that a load or store instruction of the group covers contiguous memory.  L is a power of
// two: up to 64, several rows a wave in workgroups of 256; from 256 on, a workgroup per row.
#pragma once

#include "pm_common.h"
#include "pm_vec.h"

namespace pm {
namespace {

constexpr int threads_of(int L) { return L < 256 ? 256 : L; }

// Types of a launch: every tensor bf16, every one fp32, or each as its flag says.
enum { kAllBf16 = 0, kAllF32 = 1, kMixed = 2 };

template <int M, int NV, int L>
struct RowRegs {
    float v[NV][8];

    // the row at element `at` of p, zeros past its C elements
    __device__ __forceinline__ void load(const void* p, bool bf16, int64_t at, int lane, int C) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int col = 8 * (lane + L * i), n = C - col;
            if (M == kAllBf16 || (M == kMixed && bf16)) {
                Row<uint16_t, 8> r;
                if (n > 0) r.load(static_cast<const uint16_t*>(p) + at + col, n);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[i][j] = n > 0 ? r[j] : 0.f;
            } else {
                Row<float, 8> r;
                if (n > 0) r.load(static_cast<const float*>(p) + at + col, n);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[i][j] = n > 0 ? r[j] : 0.f;
            }
        }
    }
    __device__ __forceinline__ void fill(float x) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = x;
    }
    __device__ __forceinline__ void store(void* p, bool bf16, int64_t at, int lane, int C) const {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int col = 8 * (lane + L * i), n = C - col;
            if (n <= 0) continue;
            if (M == kAllBf16 || (M == kMixed && bf16)) store_row<uint16_t, 8>(static_cast<uint16_t*>(p) + at + col, v[i], n);
            else store_row<float, 8>(static_cast<float*>(p) + at + col, v[i], n);
        }
    }
};

// The sums of N values over a group, every lane of it with the same bits.  From L = 256 on
// through LDS, in the half `turn` of `red` (consecutive calls take turns, so that one barrier a call is
// enough).
template <int L, int N>
__device__ __forceinline__ void group_sum(float (&x)[N], float (*red)[N][16], int& turn) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
        x[n] = dpp_add_rows<0xB1, 0xF>(x[n]);
        x[n] = dpp_add_rows<0x4E, 0xF>(x[n]);
        if constexpr (L >= 8) x[n] = dpp_add_rows<0x141, 0xF>(x[n]);
        if constexpr (L >= 16) x[n] = dpp_add_rows<0x140, 0xF>(x[n]);
        if constexpr (L >= 32) x[n] += __shfl_xor(x[n], 16);
        if constexpr (L >= 64) x[n] += __shfl_xor(x[n], 32);
    }
    if constexpr (L >= 256) {
        const int w = threadIdx.x >> 6;
#pragma unroll
        for (int n = 0; n < N; ++n)
            if ((threadIdx.x & 63) == 0) red[turn][n][w] = x[n];
        __syncthreads();
#pragma unroll
        for (int n = 0; n < N; ++n) {
            x[n] = red[turn][n][0];
#pragma unroll
            for (int i = 1; i < L / 64; ++i) x[n] += red[turn][n][i];
        }
        turn ^= 1;
    }
}

// A weight's gradient: what each group of the workgroup summed over its rows, to row blockIdx.x of
// part (groups in order, so that the sum does not depend on timing).
template <int NV, int L>
__device__ __forceinline__ void store_part(const float (&g)[NV][8], float* lds, float* part, int C) {
    const int lane = threadIdx.x % L, group = threadIdx.x / L;
    float* out = part + static_cast<int64_t>(blockIdx.x) * C;
    if constexpr (L >= 256) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int col = 8 * (lane + L * i) + j;
                if (col < C) out[col] = g[i][j];
            }
    } else {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) lds[group * (8 * L * NV) + 8 * (lane + L * i) + j] = g[i][j];
        __syncthreads();
        for (int col = threadIdx.x; col < C; col += 256) {
            float s = 0.f;
            for (int x = 0; x < 256 / L; ++x) s += lds[x * (8 * L * NV) + col];
            out[col] = s;
        }
    }
}

// gw[c] = the sum over n parts, COLS columns to a workgroup and 1024 / COLS threads to each, in an order
// that does not change; row blockIdx.y is another weight's.
struct RowParts {
    float* gw[2];
};
template <int COLS>
__global__ __launch_bounds__(1024) void sum_row_parts(const float* part, RowParts to, int n, int C) {
    constexpr int ROWS = 1024 / COLS;
    __shared__ float s[ROWS][COLS + 1];
    const int c = threadIdx.x % COLS, col = blockIdx.x * COLS + c, first = threadIdx.x / COLS;
    float* gw = to.gw[blockIdx.y];
    if (!gw) return;
    const float* p = part + static_cast<int64_t>(blockIdx.y) * n * C;
    float x[8] = {};  // (eight loads in flight)
    if (col < C)
        for (int i = first; i < n; i += 8 * ROWS)
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (i + ROWS * j < n) x[j] += p[static_cast<int64_t>(i + ROWS * j) * C + col];
    s[first][c] = ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
    for (int m = ROWS / 2; m > 0; m /= 2) {
        __syncthreads();
        if (first < m) s[first][c] += s[first + m][c];
    }
    if (first == 0 && col < C) gw[col] = s[0][c];
}
// Few columns are spread over more workgroups (C 128 of 2048 parts: 12 us with 16 columns each).
inline hipError_t launch_row_parts(const float* part, RowParts to, int n, int C, hipStream_t st) {
    const unsigned weights = to.gw[1] ? 2 : 1;
    if (C < 1024) hipLaunchKernelGGL(sum_row_parts<4>, dim3((C + 3) / 4, weights), dim3(1024), 0, st, part, to, n, C);
    else hipLaunchKernelGGL(sum_row_parts<16>, dim3((C + 15) / 16, weights), dim3(1024), 0, st, part, to, n, C);
    return hipGetLastError();
}

// How wide rows are held: f.template operator()<L, NV>().
template <typename F>
hipError_t by_width(int C, F f) {
    if (C <= 32) return f.template run<4, 1>();
    if (C <= 64) return f.template run<8, 1>();
    if (C <= 128) return f.template run<16, 1>();
    if (C <= 256) return f.template run<32, 1>();
    if (C <= 512) return f.template run<64, 1>();
    if (C <= 1024) return f.template run<64, 2>();
    if (C <= 2048) return f.template run<256, 1>();
    if (C <= 4096) return f.template run<512, 1>();
    if (C <= 8192) return f.template run<1024, 1>();
    return f.template run<1024, 2>();  // (C up to kMaxRow)
}
// Workgroups that walk through `rows` rows: as many as stay on the card together (a backward has the
// weights' gradients in registers too, and every workgroup more is another part to sum).
inline int64_t row_groups(int64_t rows, int C, bool bwd) {
    const int L = C <= 32 ? 4 : C <= 64 ? 8 : C <= 128 ? 16 : C <= 256 ? 32 : C <= 1024 ? 64 : C <= 2048 ? 256 : C <= 4096 ? 512 : 1024;
    const int64_t per = threads_of(L) / L, n = (rows + per - 1) / per, most = (bwd ? 1024 : 2048) * 256 / threads_of(L);
    return n < most ? n : most;
}

}  // namespace
}  // namespace pm
