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
// Bound by memory: 16 bytes in and out of an element's pair against a few multiply-adds. A lane
// holds both members of its pairs: V elements (16 bytes) at i and V at i + R / 2 (neighbouring
// pairs: 2 V in a row), so that the turn needs no other lane; the elements behind R are halved
// the same way. L lanes, the next power of two, hold a head; sums over a head go through L lanes
// by DPP. A group of L lanes takes NH heads of one token, whose angles it reads once (and, in a
// backward with weights, as many tokens as 1024 workgroups leave it). Any D up to 256, any strides
// and alignment.
//
// Measured at D = 128, bf16, calls among others on a card that copies at 5.0 TB/s: 16384 tokens of
// 16 + 16 heads forward 46 us (5.8 TB/s; one wave to a head, element by element, 361), backward 72
// (5.6 TB/s, the weights' gradients among it).

#include <type_traits>

#include "pm_internal.h"
#include "pm_vec.h"

namespace pm {

constexpr int kRowMax = 256;  // largest D
constexpr int kBlock = 256;
constexpr int kHeads = 2;          // heads of a token to a group of lanes (few rows: 1)
constexpr int kBwdBlocks = 1024;   // workgroups of a backward that sums weights' gradients

// Sum over groups of L lanes, every lane of a group with the same bits.
template <int L>
__device__ __forceinline__ float group_sum(float x) {
    if constexpr (L >= 2) x = dpp_add_rows<0xB1, 0xF>(x);   // lanes 1 apart
    if constexpr (L >= 4) x = dpp_add_rows<0x4E, 0xF>(x);   // 2
    if constexpr (L >= 8) x = dpp_add_rows<0x141, 0xF>(x);  // the mirror image in 8
    if constexpr (L >= 16) x = dpp_add_rows<0x140, 0xF>(x); // and in 16
    if constexpr (L >= 32) x += __shfl_xor(x, 16);
    if constexpr (L >= 64) x += __shfl_xor(x, 32);
    return x;
}

__device__ __forceinline__ int clamp_to(int n, int most) { return n < 0 ? 0 : n < most ? n : most; }

// Lane c's elements of a head: [a, a + na) and [b, b + nb), and its pairs [c V, c V + np).
struct Part {
    int a, na, b, nb, p, np;
};
template <int V, bool CONTIG>
__device__ __forceinline__ Part part_of(const NormRotateArgs& g, int c) {
    const int half = g.R / 2;
    Part w;
    w.p = c * V;
    w.np = clamp_to(half - w.p, V);
    if (CONTIG) {
        w.a = 2 * V * c, w.na = clamp_to(g.D - w.a, V);
        w.b = w.a + V, w.nb = clamp_to(g.D - w.b, V);
        return w;
    }
    const int turned = (half + V - 1) / V;
    if (c < turned) {
        w.a = w.p, w.b = half + w.p, w.na = w.nb = w.np;
        return w;
    }
    const int rest = g.D - g.R, first = (rest + 1) / 2, at = (c - turned) * V;
    w.a = g.R + at, w.na = clamp_to(first - at, V);
    w.b = g.R + first + at, w.nb = clamp_to(rest - first - at, V);
    return w;
}

// The lanes that a head takes.
static int lanes_of(int D, int R, int V, bool contig) {
    const int n = contig ? (D + 2 * V - 1) / (2 * V) : (R / 2 + V - 1) / V + ((D - R + 1) / 2 + V - 1) / V;
    int l = 2;
    while (l < n) l *= 2;
    return l;
}

// Item i of a side: heads i % chunks + {0, chunks, 2 chunks, ..} of token i / chunks, so that
// neighbouring groups of lanes read neighbouring heads.
struct Item {
    int b, t, h;
};
__device__ __forceinline__ Item item_of(const NormRotateArgs& a, int64_t i, int64_t items, int chunks) {
    Item w;
    if (items < (int64_t(1) << 32)) {  // (uniform: 32-bit divisions are a few instructions)
        const uint32_t u = static_cast<uint32_t>(i), tok = u / static_cast<uint32_t>(chunks);
        w.h = static_cast<int>(u - tok * chunks);
        w.b = static_cast<int>(tok / static_cast<uint32_t>(a.T));
        w.t = static_cast<int>(tok - static_cast<uint32_t>(w.b) * a.T);
    } else {
        const int64_t tok = i / chunks;
        w.h = static_cast<int>(i - tok * chunks);
        w.b = static_cast<int>(tok / a.T);
        w.t = static_cast<int>(tok - static_cast<int64_t>(w.b) * a.T);
    }
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

template <int V>
__device__ __forceinline__ void load_weight(const NormRotateArgs& a, int side, int e, int n, float (&w)[V]) {
    if (a.w_bf16) {
        Row<uint16_t, V> r;
        r.load(static_cast<const uint16_t*>(a.weight[side]) + e, n);
#pragma unroll
        for (int i = 0; i < V; ++i) w[i] = r[i];
    } else {
        Row<float, V> r;
        r.load(static_cast<const float*>(a.weight[side]) + e, n);
#pragma unroll
        for (int i = 0; i < V; ++i) w[i] = r[i];
    }
}

// The cosines and sines of a lane's pairs (1 and 0 where its elements are not turned); returns
// whether the token's position is in the table.
template <int V>
__device__ __forceinline__ bool load_angles(const NormRotateArgs& a, const Part& w, int b, int t, float (&c)[V],
                                            float (&s)[V]) {
    const int64_t row = table_row(a, b, t);
    const float* p = a.table + row * a.R + w.p;
    const int n = row < 0 ? 0 : w.np;
    Row<float, V> rc, rs;
    rc.load(p, n);
    rs.load(p + a.R / 2, n);
#pragma unroll
    for (int i = 0; i < V; ++i) c[i] = i < n ? rc[i] : 1.f, s[i] = rs[i];
    return row >= 0;
}

// The lane's pairs turned by their angles (dir 1) or back (-1).
template <int V, bool CONTIG>
__device__ __forceinline__ void turn(const float (&c)[V], const float (&s)[V], float dir, float (&ya)[V],
                                     float (&yb)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
        float& y1 = !CONTIG ? ya[i] : i < V / 2 ? ya[2 * i % V] : yb[2 * i % V];
        float& y2 = !CONTIG ? yb[i] : i < V / 2 ? ya[(2 * i + 1) % V] : yb[(2 * i + 1) % V];
        const float si = dir * s[i], z1 = fmaf(y1, c[i], -(y2 * si));
        y2 = fmaf(y2, c[i], y1 * si);
        y1 = z1;
    }
}

// r of a head from its sum of squares (NaN stays NaN; `clipped`: l2 at or below eps)
__device__ __forceinline__ float row_scale(const NormRotateArgs& a, float ss, bool& clipped) {
    clipped = false;
    if (a.rms) return 1.f / sqrtf(ss / static_cast<float>(a.D) + a.eps);
    const float n = sqrtf(ss);
    clipped = n <= a.eps;
    return 1.f / (clipped ? a.eps : n);
}

template <typename E, int L, bool CONTIG, int NH>
__global__ __launch_bounds__(kBlock) void norm_rotate_kernel(NormRotateArgs a, int q_blocks) {
    constexpr int V = 16 / sizeof(E), GROUPS = kBlock / L;
    const float nan = __uint_as_float(0x7fc00000u);
    const bool k = static_cast<int>(blockIdx.x) >= q_blocks;
    const int H = a.H[k], chunks = (H + NH - 1) / NH;
    const int64_t far = static_cast<int64_t>(chunks) * a.D;  // from one of a group's heads to its next
    const int64_t items = static_cast<int64_t>(a.B) * a.T * chunks;
    const int64_t step = static_cast<int64_t>(k ? gridDim.x - q_blocks : q_blocks) * GROUPS;
    const Part w = part_of<V, CONTIG>(a, threadIdx.x % L);
    float wa[V], wb[V];
    if (a.weight[k]) load_weight<V>(a, k, w.a, w.na, wa), load_weight<V>(a, k, w.b, w.nb, wb);

    for (int64_t i = static_cast<int64_t>(blockIdx.x - (k ? q_blocks : 0)) * GROUPS + threadIdx.x / L; i < items;
         i += step) {
        const Item at = item_of(a, i, items, chunks);
        const E* x = static_cast<const E*>(a.x[k]) + at.b * a.sb[k] + at.t * a.st[k] + at.h * a.sh[k];
        Row<E, V> xa[NH], xb[NH];
#pragma unroll
        for (int j = 0; j < NH; ++j) {
            const bool there = at.h + j * chunks < H;
            xa[j].load(x + j * chunks * a.sh[k] + w.a, there ? w.na : 0);
            xb[j].load(x + j * chunks * a.sh[k] + w.b, there ? w.nb : 0);
        }
        float c[V], s[V];
        const bool known = !a.R || load_angles<V>(a, w, at.b, at.t, c, s);
        E* y = static_cast<E*>(a.y[k]) + ((static_cast<int64_t>(at.b) * a.T + at.t) * H + at.h) * a.D;
#pragma unroll
        for (int j = 0; j < NH; ++j) {
            float ss = 0.f, ya[V], yb[V];
#pragma unroll
            for (int e = 0; e < V; ++e) ss = fmaf(xa[j][e], xa[j][e], ss), ss = fmaf(xb[j][e], xb[j][e], ss);
            bool clipped;
            float scale = row_scale(a, group_sum<L>(ss), clipped);
            if (!known) scale = nan;
#pragma unroll
            for (int e = 0; e < V; ++e) ya[e] = xa[j][e] * scale, yb[e] = xb[j][e] * scale;
            if (a.weight[k]) {
#pragma unroll
                for (int e = 0; e < V; ++e) ya[e] *= wa[e], yb[e] *= wb[e];
            }
            if (a.R) turn<V, CONTIG>(c, s, 1.f, ya, yb);
            if (at.h + j * chunks < H) {
                store_row<E, V>(y + j * far + w.a, ya, w.na);
                store_row<E, V>(y + j * far + w.b, yb, w.nb);
            }
        }
    }
}

// Each workgroup sums its heads' shares of its side's weight gradient in a fixed order into
// part[block][D]; weight_grad_kernel adds the workgroups' in a fixed order, so that the sums do
// not depend on which finishes first.
template <typename E, int L, bool CONTIG, int NH>
__global__ __launch_bounds__(kBlock) void norm_rotate_bwd_kernel(NormRotateArgs a, int q_blocks, float* part) {
    constexpr int V = 16 / sizeof(E), GROUPS = kBlock / L;
    __shared__ float buf[kBlock / 64][kRowMax];
    const float nan = __uint_as_float(0x7fc00000u);
    const bool k = static_cast<int>(blockIdx.x) >= q_blocks;
    const int H = a.H[k], chunks = (H + NH - 1) / NH;
    const int64_t far = static_cast<int64_t>(chunks) * a.D;  // from one of a group's heads to its next
    const int64_t items = static_cast<int64_t>(a.B) * a.T * chunks;
    const int64_t step = static_cast<int64_t>(k ? gridDim.x - q_blocks : q_blocks) * GROUPS;
    const Part w = part_of<V, CONTIG>(a, threadIdx.x % L);
    float wa[V], wb[V], ga[V] = {}, gb[V] = {};
    if (a.weight[k]) load_weight<V>(a, k, w.a, w.na, wa), load_weight<V>(a, k, w.b, w.nb, wb);

    for (int64_t i = static_cast<int64_t>(blockIdx.x - (k ? q_blocks : 0)) * GROUPS + threadIdx.x / L; i < items;
         i += step) {
        const Item at = item_of(a, i, items, chunks);
        const E* x = static_cast<const E*>(a.x[k]) + at.b * a.sb[k] + at.t * a.st[k] + at.h * a.sh[k];
        const int64_t out = ((static_cast<int64_t>(at.b) * a.T + at.t) * H + at.h) * a.D;
        const E* gz = static_cast<const E*>(a.gy[k]) + out;
        Row<E, V> xa[NH], xb[NH], za[NH], zb[NH];
#pragma unroll
        for (int j = 0; j < NH; ++j) {
            const bool there = at.h + j * chunks < H, any = there && a.gy[k];
            xa[j].load(x + j * chunks * a.sh[k] + w.a, there ? w.na : 0);
            xb[j].load(x + j * chunks * a.sh[k] + w.b, there ? w.nb : 0);
            za[j].load(gz + j * far + w.a, any ? w.na : 0);
            zb[j].load(gz + j * far + w.b, any ? w.nb : 0);
        }
        float c[V], s[V];
        const bool known = !a.R || load_angles<V>(a, w, at.b, at.t, c, s);
        E* gx = static_cast<E*>(a.gx[k]) + out;
#pragma unroll
        for (int j = 0; j < NH; ++j) {
            float ya[V], yb[V], ss = 0.f, dot = 0.f;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                ss = fmaf(xa[j][e], xa[j][e], ss), ss = fmaf(xb[j][e], xb[j][e], ss);
                ya[e] = za[j][e], yb[e] = zb[j][e];
            }
            if (a.R) turn<V, CONTIG>(c, s, -1.f, ya, yb);
            bool clipped;
            float scale = row_scale(a, group_sum<L>(ss), clipped);
            if (!known) scale = nan;
            if (a.weight[k]) {
                if (at.h + j * chunks < H) {
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        ga[e] = fmaf(ya[e], xa[j][e] * scale, ga[e]);
                        gb[e] = fmaf(yb[e], xb[j][e] * scale, gb[e]);
                    }
                }
#pragma unroll
                for (int e = 0; e < V; ++e) ya[e] *= wa[e], yb[e] *= wb[e];
            }
#pragma unroll
            for (int e = 0; e < V; ++e)
                dot = fmaf(ya[e], xa[j][e] * scale, dot), dot = fmaf(yb[e], xb[j][e] * scale, dot);
            dot = group_sum<L>(dot);
            if (a.rms) dot /= static_cast<float>(a.D);
            if (clipped) dot = 0.f;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                ya[e] = fmaf(xa[j][e] * scale, -dot, ya[e]) * scale;
                yb[e] = fmaf(xb[j][e] * scale, -dot, yb[e]) * scale;
            }
            if (at.h + j * chunks < H) {
                store_row<E, V>(gx + j * far + w.a, ya, w.na);
                store_row<E, V>(gx + j * far + w.b, yb, w.nb);
            }
        }
    }
    if (!a.gw[k]) return;
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
#pragma unroll
    for (int e = 0; e < V; ++e) {
#pragma unroll
        for (int m = L; m < 64; m *= 2) ga[e] += __shfl_xor(ga[e], m), gb[e] += __shfl_xor(gb[e], m);
        if (lane < L && e < w.na) buf[wave][w.a + e] = ga[e];
        if (lane < L && e < w.nb) buf[wave][w.b + e] = gb[e];
    }
    __syncthreads();
    const int e = threadIdx.x;
    if (e < a.D)
        part[static_cast<int64_t>(blockIdx.x) * a.D + e] = (buf[0][e] + buf[1][e]) + (buf[2][e] + buf[3][e]);
}

// Workgroup (c, side): columns 32 c .. of the sums over that side's workgroups, 32 threads to a column.
__global__ __launch_bounds__(1024) void weight_grad_kernel(const float* part, int q_blocks, int blocks, int D,
                                                           float* gq, float* gk) {
    __shared__ float buf[32][33];
    const int side = blockIdx.y, col = threadIdx.x % 32, row = threadIdx.x / 32;
    const int e = blockIdx.x * 32 + col, from = side ? q_blocks : 0, to = side ? blocks : q_blocks;
    float* out = side ? gk : gq;
    if (!out) return;
    float s = 0.f;
    if (e < D) {
#pragma unroll 8
        for (int i = from + row; i < to; i += 32) s += part[static_cast<int64_t>(i) * D + e];
    }
    buf[row][col] = s;
    __syncthreads();
    if (row > 0 || e >= D) return;
#pragma unroll
    for (int i = 1; i < 32; ++i) s += buf[i][col];
    out[e] = s;
}

// f(null pointer of E, L, contig, NH) for a call
template <typename E, typename F>
static void by_shape(const NormRotateArgs& a, int nh, F f) {
    const bool contig = a.interleaved || !a.R;
    const int l = lanes_of(a.D, a.R, 16 / sizeof(E), contig);
    E* e = nullptr;
    auto with_lanes = [&](auto lanes) {
        auto with_layout = [&](auto layout) {
            if (nh == 1) f(e, lanes, layout, std::integral_constant<int, 1>{});
            else f(e, lanes, layout, std::integral_constant<int, kHeads>{});
        };
        if (contig) with_layout(std::true_type{});
        else with_layout(std::false_type{});
    };
    switch (l) {
        case 2: with_lanes(std::integral_constant<int, 2>{}); break;
        case 4: with_lanes(std::integral_constant<int, 4>{}); break;
        case 8: with_lanes(std::integral_constant<int, 8>{}); break;
        case 16: with_lanes(std::integral_constant<int, 16>{}); break;
        case 32: with_lanes(std::integral_constant<int, 32>{}); break;
        default: with_lanes(std::integral_constant<int, 64>{}); break;
    }
}

// Heads to a group of lanes. Two share a token's angles and keep two rows' loads under way, as long
// as there are groups enough to fill the card, the twos are mostly whole, and a head is not so
// small that it is one or two lanes. Measured one to two (us, bf16): 16384 tokens of 16 + 16 heads
// of 128 forward 57 to 49, backward without weights 85 to 73, with them 83 to 80; 512 tokens of 32
// + 32 backward 12.9 to 11.9; but 256 of 32 + 32 forward 4.5 to 4.9, 16384 of 3 + 3 backward 20.6
// to 22.2, of 16 + 16 of 32 forward 17.4 to 20.9. Four: 51.5 and 76 of the first.
static int heads_of(const NormRotateArgs& a, int lanes) {
    const int64_t tokens = static_cast<int64_t>(a.B) * a.T;
    const int twos = (a.H[0] + kHeads - 1) / kHeads + (a.H[1] + kHeads - 1) / kHeads;
    const bool fill = tokens * twos * lanes >= 256 * 512, whole = 5 * (a.H[0] + a.H[1]) >= 4 * kHeads * twos;
    return fill && whole && lanes > 2 ? kHeads : 1;
}

// Workgroups of a side, at most `most`.
static int side_blocks(const NormRotateArgs& a, int side, int lanes, int nh, int64_t most) {
    const int64_t items = static_cast<int64_t>(a.B) * a.T * ((a.H[side] + nh - 1) / nh);
    const int64_t groups = kBlock / lanes, n = (items + groups - 1) / groups;
    return static_cast<int>(n < most ? n : most);
}

template <typename E>
static hipError_t forward(const NormRotateArgs& a, hipStream_t st) {
    const int lanes = lanes_of(a.D, a.R, 16 / sizeof(E), a.interleaved || !a.R), nh = heads_of(a, lanes);
    const int q = side_blocks(a, 0, lanes, nh, 1 << 20), k = side_blocks(a, 1, lanes, nh, 1 << 20);
    by_shape<E>(a, nh, [&](auto e, auto l, auto contig, auto n) {
        hipLaunchKernelGGL((norm_rotate_kernel<std::remove_pointer_t<decltype(e)>, l(), contig(), n()>), dim3(q + k),
                           dim3(kBlock), 0, st, a, q);
    });
    return hipGetLastError();
}

hipError_t launch_norm_rotate(const NormRotateArgs& a, hipStream_t st) {
    return a.bf16 ? forward<uint16_t>(a, st) : forward<float>(a, st);
}

// Workgroups of a backward with weights' gradients: kBwdBlocks shared out by heads, one at least.
static int q_share(int Hq, int Hk) {
    const int64_t n = static_cast<int64_t>(kBwdBlocks) * Hq / (static_cast<int64_t>(Hq) + Hk);
    return static_cast<int>(n < 1 ? 1 : n > kBwdBlocks - 1 ? kBwdBlocks - 1 : n);
}
size_t norm_rotate_bwd_ws_bytes(int B, int T, int Hq, int Hk, int D) {
    const int64_t rows = static_cast<int64_t>(B) * T * (static_cast<int64_t>(Hq) + Hk);
    return static_cast<size_t>(rows < kBwdBlocks ? rows : kBwdBlocks) * D * sizeof(float);
}

template <typename E>
static hipError_t backward(const NormRotateArgs& a, hipStream_t st) {
    const bool sums = a.gw[0] || a.gw[1];
    const int lanes = lanes_of(a.D, a.R, 16 / sizeof(E), a.interleaved || !a.R), nh = heads_of(a, lanes);
    const int share = q_share(a.H[0], a.H[1]);
    const int q = side_blocks(a, 0, lanes, nh, sums ? share : 1 << 20);
    const int k = side_blocks(a, 1, lanes, nh, sums ? kBwdBlocks - share : 1 << 20);
    float* part = static_cast<float*>(a.workspace);
    by_shape<E>(a, nh, [&](auto e, auto l, auto contig, auto n) {
        hipLaunchKernelGGL((norm_rotate_bwd_kernel<std::remove_pointer_t<decltype(e)>, l(), contig(), n()>),
                           dim3(q + k), dim3(kBlock), 0, st, a, q, part);
    });
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || !sums) return e;
    hipLaunchKernelGGL(weight_grad_kernel, dim3((a.D + 31) / 32, 2), dim3(1024), 0, st, part, q, q + k, a.D, a.gw[0],
                       a.gw[1]);
    return hipGetLastError();
}

hipError_t launch_norm_rotate_bwd(const NormRotateArgs& a, hipStream_t st) {
    return a.bf16 ? backward<uint16_t>(a, st) : backward<float>(a, st);
}

}  // namespace pm
