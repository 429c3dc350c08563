// linear_recurrence.hip — K12: the elementwise gated linear recurrence, its gradients and its
// single-token step.
//
//   h_t = exp(g_t) h_{t-1} + x_t          for every channel on its own
//   d_t = gh_t + exp(g_{t+1}) d_{t+1},  gx_t = d_t,  gg_t = d_t exp(g_t) h_{t-1}
//
// Bound by memory: one exponential and a few multiply-adds an element against 6 bytes (bf16
// forward) or 10 (backward). So every element is read once and written once: a tile of 256 tokens
// by one 128-byte line of channels stays in registers from its loads to its stores, and what
// tokens need of each other goes as affine maps s -> A s + H of the spans between them.
//   1. each thread folds its own 4 tokens of 8 (fp32: 4) channels into one map;
//   2. through LDS the tile's maps fold in a fixed tree: per part of the tile, then the tile;
//   3. a tile that is not its sequence's first waits for the state before it (below);
//   4. the state walks down the tree again and through each thread's tokens.
// The backward is the same with the message c_t = exp(g_t) d_t, c_t = exp(g_t) (gh_t + c_{t+1}),
// from the last tile to the first, on top of a forward inside the tile from the kept state.
//
// Between tiles (T > 256), in one pass: a tile publishes its map as soon as it is folded; the
// state before tile j is the state at the start of j's group of 16 tiles, taken through the maps
// of the group's tiles before j in order; the group's last tile publishes the next group's state.
// The order of every product and sum is fixed by j, not by which tile is done first, so results
// are the same bits every time; and the chain that cannot run in parallel is one hop in 16 tiles.
// Words carry value and readiness together (relaxed 8-byte atomics of agent scope; the workspace
// starts as all ones, which no value is), so no fences. Tiles are handed out by a counter in the
// order in which they wait for each other: the tiles a tile waits for are held by workgroups that
// run already, so every wait ends.

#include "pm_internal.h"
#include "pm_vec.h"

namespace pm {

constexpr int kTok = 4;                       // tokens to a thread
constexpr int kTileT = kRecSpan;              // tokens to a tile
constexpr int kLanesC = 8;                    // threads across the channels of a tile
constexpr int kThreads = kTileT / kTok * kLanesC;
constexpr int kGroup = 16;                    // tiles to a group

// The tiles of a call and the words through which they pass states (all null where each
// sequence is one tile).
struct Tiles {
    int cgroups;     // channel groups
    int64_t cols;    // sequences x channel groups
    int64_t tiles;   // tiles along the tokens
    uint32_t* next;  // the counter that hands out tiles
    uint64_t* map;   // [col][tile][channel]: H below, A above
    uint64_t* state; // [col][group][channel]: the state before the group below, 0 above
};

__device__ __forceinline__ uint64_t word(uint32_t above, float below) {
    return static_cast<uint64_t>(above) << 32 | __float_as_uint(below);
}
__device__ __forceinline__ void publish(uint64_t* p, uint64_t v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint64_t wait_word(uint64_t* p) {
    for (;;) {
        const uint64_t v = __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (static_cast<uint32_t>(v >> 32) != 0xffffffffu) return v;
        __builtin_amdgcn_s_sleep(1);
    }
}
__device__ __forceinline__ float low(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v)); }
__device__ __forceinline__ float high(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v >> 32)); }

// s -> A s + H. A negative A (PACKED only) is a map that a sequence starts in: its H is the state
// whatever came before, infinities and NaN included.
template <bool PACKED>
struct Map {
    float A, H;
    __device__ __forceinline__ void then(const Map& m) {
        const bool anew = PACKED && m.A < 0.f;
        H = anew ? m.H : fmaf(m.A, H, m.H);
        A = anew ? m.A : (PACKED && A < 0.f ? A : A * m.A);
    }
    __device__ __forceinline__ float of(float s) const { return PACKED && A < 0.f ? H : fmaf(A, s, H); }
    __device__ __forceinline__ uint64_t word() const {
        const uint32_t a = __float_as_uint(A);
        return pm::word(a == 0xffffffffu ? 0x7fc00000u : a, H);  // (a NaN all of whose bits are set)
    }
    static __device__ __forceinline__ Map read(uint64_t v) { return {high(v), low(v)}; }
};

__device__ __forceinline__ float gate(float g) { return __builtin_amdgcn_exp2f(g * 1.44269504088896341f); }

// Row of a sequence's state in s0 and s_out, or -1 (a slot outside the pool).
__device__ __forceinline__ int64_t state_row(const int32_t* slots, int n_slots, int seq) {
    if (!slots) return seq;
    const int r = slots[seq];
    return r >= 0 && r < n_slots ? r : -1;
}

// Where the thread (ch, part) of a tile's fold stands in a group's chain, and the state it takes
// from there. All threads of the workgroup call it; `lb` is LDS [PARTS][CW]. `j` counts tiles in
// the order in which they wait for each other, `first` is the state before tile 0.
template <bool PACKED, int CW, int PARTS>
__device__ __forceinline__ float state_before(const Tiles& p, int64_t col, int64_t j, int ch, int part, float first,
                                              Map<PACKED> (*lb)[CW]) {
    if (!p.next || j == 0) return first;
    constexpr int Q = (kGroup + PARTS - 1) / PARTS;  // tiles of the group to a part
    const int64_t g0 = j / kGroup * kGroup;
    const int n = static_cast<int>(j - g0);
    Map<PACKED> m{1.f, 0.f};
#pragma unroll
    for (int i = 0; i < Q; ++i) {
        const int q = part * Q + i;
        if (q < n) m.then(Map<PACKED>::read(wait_word(p.map + (col * p.tiles + g0 + q) * CW + ch)));
    }
    if (part == 0) {
        const int64_t groups = (p.tiles + kGroup - 1) / kGroup;
        const float s = g0 == 0 ? first : low(wait_word(p.state + (col * groups + j / kGroup) * CW + ch));
        m.H = m.of(s);
    }
    lb[part][ch] = m;
    __syncthreads();
    float s = lb[0][ch].H;
#pragma unroll
    for (int i = 1; i < PARTS; ++i)
        if (i * Q < n) s = lb[i][ch].of(s);
    return s;
}

template <int CW>
__device__ __forceinline__ void publish_state(const Tiles& p, int64_t col, int64_t j, int ch, float s) {
    if (!p.next || j % kGroup != kGroup - 1 || j + 1 >= p.tiles) return;
    const int64_t groups = (p.tiles + kGroup - 1) / kGroup;
    publish(p.state + (col * groups + j / kGroup + 1) * CW + ch, word(0, s));
}

// The next tile of a workgroup, or -1. `slot` is one LDS word.
__device__ __forceinline__ int64_t next_tile(const Tiles& p, int64_t last, uint32_t* slot) {
    const int64_t all = p.cols * p.tiles;
    int64_t id;
    if (p.next) {
        __syncthreads();  // the last tile's reads of LDS, this word's among them, are done
        if (threadIdx.x == 0) *slot = __hip_atomic_fetch_add(p.next, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        id = *slot;
    } else {
        if (last >= 0) __syncthreads();
        id = last < 0 ? blockIdx.x : last + gridDim.x;
    }
    return id < all ? id : -1;
}

template <typename X, typename G, typename H, int V, bool PACKED>
__global__ __launch_bounds__(kThreads, PACKED ? 2 : 4) void recurrence_kernel(RecurrenceArgs a, Tiles p) {
    constexpr int CW = kLanesC * V, TL = kTileT / kTok, PARTS = kThreads / CW, PER = TL / PARTS;
    __shared__ float sA[TL][CW], sH[TL][CW];
    __shared__ Map<PACKED> total[PARTS][CW], lb[PARTS][CW];
    __shared__ int start[PACKED ? kTileT : 1], stop[PACKED ? kTileT : 1];
    __shared__ float first[CW];
    __shared__ uint32_t slot;
    const int tid = threadIdx.x, lc = tid % kLanesC, tl = tid / kLanesC;
    const int ch = tid % CW, part = tid / CW;

    for (int64_t id = next_tile(p, -1, &slot); id >= 0; id = next_tile(p, id, &slot)) {
        const int64_t j = id / p.cols, col = id - j * p.cols;
        const int seq = PACKED ? 0 : static_cast<int>(col / p.cgroups);
        const int cbase = static_cast<int>(PACKED ? col : col % p.cgroups) * CW;
        const int c0 = cbase + lc * V, nc = a.C - c0;  // this thread's channels, and how many are there
        const int tile0 = static_cast<int>(j) * kTileT, t0 = tile0 + tl * kTok;
        const X* xp = static_cast<const X*>(a.x) + seq * a.x_sb + t0 * a.x_st + c0;
        const G* gp = static_cast<const G*>(a.g) + seq * a.g_sb + t0 * a.g_st + c0;
        Row<X, V> xr[kTok];
        Row<G, V> gr[kTok];
#pragma unroll
        for (int r = 0; r < kTok; ++r) {
            const int n = t0 + r < a.T ? nc : 0;
            xr[r].load(xp + r * a.x_st, n);
            gr[r].load(gp + r * a.g_st, n);
        }
        // the state before the sequence: read by its first tile only, before that tile's map is
        // out, as the last tile may write the same row of the pool soon after
        if (!PACKED && j == 0 && part == 0) {
            const int64_t row = state_row(a.slots, a.n_slots, seq);
            if (row < 0 && a.bad) atomicOr(a.bad, 1);
            first[ch] = a.s0 && row >= 0 && cbase + ch < a.C ? a.s0[row * a.C + cbase + ch] : 0.f;
        }
        unsigned starts = 0, stops = 0;  // bit r: a sequence starts (ends) with token t0 + r
        if constexpr (PACKED) {
            for (int i = tid; i < kTileT; i += kThreads) start[i] = stop[i] = -1;
            __syncthreads();
            for (int i = tid; i < a.n_seqs; i += kThreads) {
                const int b = min(max(a.cu_seqlens[i], 0), a.T), e = min(max(a.cu_seqlens[i + 1], b), a.T);
                if (b == e) continue;
                if (b >= tile0 && b < tile0 + kTileT) start[b - tile0] = i;
                if (e > tile0 && e <= tile0 + kTileT) stop[e - 1 - tile0] = i;
            }
            __syncthreads();
#pragma unroll
            for (int r = 0; r < kTok; ++r) {
                starts |= (start[tl * kTok + r] >= 0) << r;
                stops |= (stop[tl * kTok + r] >= 0) << r;
            }
        }
        float av[kTok][V], xv[kTok][V];
        Map<PACKED> m[V];
#pragma unroll
        for (int v = 0; v < V; ++v) m[v] = {1.f, 0.f};
#pragma unroll
        for (int r = 0; r < kTok; ++r) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                // (tokens past the end are zeros: gates of one and nothing added)
                av[r][v] = gate(gr[r][v]);
                xv[r][v] = xr[r][v];
            }
            if (PACKED && (starts >> r & 1)) {
                // the start's state goes into x here, where it is read once: the sequence's last
                // tile may write the same row of the pool as soon as this tile's map is out
                const int64_t row = state_row(a.slots, a.n_slots, start[tl * kTok + r]);
                if (row < 0 && a.bad) atomicOr(a.bad, 1);
                Row<float, V> s;
                s.load(a.s0 && row >= 0 ? a.s0 + row * a.C + c0 : nullptr, a.s0 && row >= 0 ? nc : 0);
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    xv[r][v] = fmaf(av[r][v], s[v], xv[r][v]);
                    m[v] = {-1.f, xv[r][v]};
                }
            } else {
#pragma unroll
                for (int v = 0; v < V; ++v) m[v].then({av[r][v], xv[r][v]});
            }
        }
#pragma unroll
        for (int v = 0; v < V; ++v) sA[tl][lc * V + v] = m[v].A, sH[tl][lc * V + v] = m[v].H;
        __syncthreads();

        Map<PACKED> mine[PER], sum{1.f, 0.f};
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            mine[i] = {sA[part * PER + i][ch], sH[part * PER + i][ch]};
            sum.then(mine[i]);
        }
        total[part][ch] = sum;
        __syncthreads();
        float s = !PACKED && j == 0 ? first[ch] : 0.f;
        if (p.next && part == 0) {
#pragma unroll
            for (int i = 1; i < PARTS; ++i) sum.then(total[i][ch]);
            if (!PACKED && j == 0) sum = {0.f, sum.of(s)};  // the first tile's map yields its state
            publish(p.map + (col * p.tiles + j) * CW + ch, sum.word());
        }
        s = state_before<PACKED, CW, PARTS>(p, col, j, ch, part, s, lb);
        if (a.kept && part == 0 && cbase + ch < a.C) a.kept[(seq * p.tiles + j) * a.C + cbase + ch] = s;
#pragma unroll
        for (int i = 0; i < PARTS; ++i)
            if (i < part) s = total[i][ch].of(s);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            sH[part * PER + i][ch] = s;
            s = mine[i].of(s);
        }
        if (part == PARTS - 1) publish_state<CW>(p, col, j, ch, s);
        __syncthreads();

        float h[V];
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = sH[tl][lc * V + v];
        H* hp = static_cast<H*>(a.h) + (static_cast<int64_t>(seq) * a.T + t0) * a.C + c0;
#pragma unroll
        for (int r = 0; r < kTok; ++r) {
            const int t = t0 + r;
#pragma unroll
            for (int v = 0; v < V; ++v)
                h[v] = PACKED && (starts >> r & 1) ? xv[r][v] : fmaf(av[r][v], h[v], xv[r][v]);
            if (t < a.T) store_row<H, V>(hp + static_cast<int64_t>(r) * a.C, h, nc);
            const int ends = PACKED ? (stops >> r & 1 ? stop[tl * kTok + r] : -1) : (t == a.T - 1 ? seq : -1);
            if (ends >= 0) {
                const int64_t row = state_row(a.slots, a.n_slots, ends);
                if (row >= 0) store_row<float, V>(a.s_out + row * a.C + c0, h, nc);
            }
        }
    }
}

// The gradients; tiles go from the last to the first, and c_t = exp(g_t) d_t is the state.
template <typename X, typename G, typename H, int V>
__global__ __launch_bounds__(kThreads, 4) void recurrence_bwd_kernel(RecurrenceBwdArgs a, Tiles p) {
    constexpr int CW = kLanesC * V, TL = kTileT / kTok, PARTS = kThreads / CW, PER = TL / PARTS;
    typedef Map<false> M;
    __shared__ float sA[TL][CW], sF[TL][CW], sB[TL][CW];
    __shared__ M fwd[PARTS][CW], bwd[PARTS][CW], lb[PARTS][CW];
    __shared__ uint32_t slot;
    const int tid = threadIdx.x, lc = tid % kLanesC, tl = tid / kLanesC;
    const int ch = tid % CW, part = tid / CW;

    for (int64_t id = next_tile(p, -1, &slot); id >= 0; id = next_tile(p, id, &slot)) {
        const int64_t j = id / p.cols, col = id - j * p.cols, tile = p.tiles - 1 - j;
        const int b = static_cast<int>(col / p.cgroups), cbase = static_cast<int>(col % p.cgroups) * CW;
        const int c0 = cbase + lc * V, nc = a.C - c0;
        const int t0 = static_cast<int>(tile) * kTileT + tl * kTok;
        const X* xp = static_cast<const X*>(a.x) + b * a.x_sb + t0 * a.x_st + c0;
        const G* gp = static_cast<const G*>(a.g) + b * a.g_sb + t0 * a.g_st + c0;
        const int64_t out = (static_cast<int64_t>(b) * a.T + t0) * a.C + c0;
        Row<X, V> xr[kTok];
        Row<G, V> gr[kTok];
        Row<H, V> hr[kTok];
#pragma unroll
        for (int r = 0; r < kTok; ++r) {
            const int n = t0 + r < a.T ? nc : 0;
            xr[r].load(xp + r * a.x_st, n);
            gr[r].load(gp + r * a.g_st, n);
            hr[r].load(static_cast<const H*>(a.gh) + out + static_cast<int64_t>(r) * a.C, a.gh ? n : 0);
        }
        float av[kTok][V];
        M f[V], w[V];  // the tokens' map of h, and of c
#pragma unroll
        for (int v = 0; v < V; ++v) f[v] = w[v] = {1.f, 0.f};
#pragma unroll
        for (int r = 0; r < kTok; ++r)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                av[r][v] = gate(gr[r][v]);
                f[v].then({av[r][v], xr[r][v]});
            }
#pragma unroll
        for (int r = kTok - 1; r >= 0; --r)
#pragma unroll
            for (int v = 0; v < V; ++v) w[v].H = av[r][v] * (w[v].H + hr[r][v]);
#pragma unroll
        for (int v = 0; v < V; ++v)
            sA[tl][lc * V + v] = f[v].A, sF[tl][lc * V + v] = f[v].H, sB[tl][lc * V + v] = w[v].H;
        __syncthreads();

        float A[PER], F[PER], B[PER];
        M up{1.f, 0.f}, down{1.f, 0.f};
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            A[i] = sA[part * PER + i][ch], F[i] = sF[part * PER + i][ch], B[i] = sB[part * PER + i][ch];
            up.then({A[i], F[i]});
        }
#pragma unroll
        for (int i = PER - 1; i >= 0; --i) down.then({A[i], B[i]});
        fwd[part][ch] = up;
        bwd[part][ch] = down;
        __syncthreads();
        if (p.next && part == PARTS - 1) {
#pragma unroll
            for (int i = PARTS - 2; i >= 0; --i) down.then(bwd[i][ch]);
            publish(p.map + (col * p.tiles + j) * CW + ch, down.word());
        }
        const bool there = cbase + ch < a.C;
        float c = a.gs && j < kGroup && there ? a.gs[static_cast<int64_t>(b) * a.C + cbase + ch] : 0.f;
        float h = there ? a.kept[(b * p.tiles + tile) * a.C + cbase + ch] : 0.f;
        c = state_before<false, CW, PARTS>(p, col, j, ch, part, c, lb);
#pragma unroll
        for (int i = 0; i < PARTS; ++i)
            if (i < part) h = fwd[i][ch].of(h);
#pragma unroll
        for (int i = PARTS - 1; i >= 0; --i)
            if (i > part) c = bwd[i][ch].of(c);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            sF[part * PER + i][ch] = h;
            h = fmaf(A[i], h, F[i]);
        }
#pragma unroll
        for (int i = PER - 1; i >= 0; --i) {
            sB[part * PER + i][ch] = c;
            c = fmaf(A[i], c, B[i]);
        }
        if (part == 0) {
            publish_state<CW>(p, col, j, ch, c);
            if (tile == 0 && there) a.gs0[static_cast<int64_t>(b) * a.C + cbase + ch] = c;
        }
        __syncthreads();

        float hb[kTok][V], cv[V];  // the state before each token; c behind it
#pragma unroll
        for (int v = 0; v < V; ++v) {
            hb[0][v] = sF[tl][lc * V + v], cv[v] = sB[tl][lc * V + v];
#pragma unroll
            for (int r = 1; r < kTok; ++r) hb[r][v] = fmaf(av[r - 1][v], hb[r - 1][v], xr[r - 1][v]);
        }
#pragma unroll
        for (int r = kTok - 1; r >= 0; --r) {
            float gx[V], gg[V];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                gx[v] = hr[r][v] + cv[v];
                cv[v] = av[r][v] * gx[v];
                gg[v] = cv[v] * hb[r][v];
            }
            if (t0 + r < a.T) {
                store_row<X, V>(static_cast<X*>(a.gx) + out + static_cast<int64_t>(r) * a.C, gx, nc);
                store_row<G, V>(static_cast<G*>(a.gg) + out + static_cast<int64_t>(r) * a.C, gg, nc);
            }
        }
    }
}

// Before a call: `n` words of the workspace to all ones and the counter to zero; and the states
// of sequences without tokens (all of them where T is 0), which pass through.
__global__ __launch_bounds__(256) void recurrence_begin_kernel(uint32_t* next, uint64_t* words, int64_t n,
                                                               RecurrenceArgs a) {
    const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, step = static_cast<int64_t>(gridDim.x) * 256;
    if (next && at == 0) *next = 0;
    for (int64_t i = at; i < n; i += step) words[i] = ~uint64_t(0);
    for (int seq = blockIdx.x; seq < a.n_seqs; seq += gridDim.x) {
        if (a.T > 0) {
            if (!a.cu_seqlens) break;
            const int b = min(max(a.cu_seqlens[seq], 0), a.T), e = min(max(a.cu_seqlens[seq + 1], b), a.T);
            if (b < e) continue;
        }
        const int64_t row = state_row(a.slots, a.n_slots, seq);
        if (row < 0) {
            if (a.bad && threadIdx.x == 0) atomicOr(a.bad, 1);
            continue;
        }
        for (int64_t c = threadIdx.x; c < a.C; c += 256)
            a.s_out[row * a.C + c] = a.s0 ? a.s0[row * a.C + c] : 0.f;
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
            s = fmaf(gate(to_f32(static_cast<const G*>(a.g)[b * a.g_sb + c])), a.s[row * a.C + c],
                     to_f32(static_cast<const X*>(a.x)[b * a.x_sb + c]));
            a.s[row * a.C + c] = s;
        }
        static_cast<H*>(a.h)[static_cast<int64_t>(b) * a.C + c] = from_f32<H>(s);
    }
}

// f(x, g, h) with a null pointer of each tensor's element type
template <typename F>
static void by_types(bool x_bf16, bool g_bf16, bool h_bf16, F f) {
    uint16_t* b = nullptr;
    float* s = nullptr;
    if (x_bf16 && g_bf16) h_bf16 ? f(b, b, b) : f(b, b, s);
    else if (x_bf16) h_bf16 ? f(b, s, b) : f(b, s, s);
    else h_bf16 ? f(s, s, b) : f(s, s, s);
}

#define PM_ELEM(p) std::remove_pointer_t<decltype(p)>

static int row_width(bool x_bf16) { return x_bf16 ? 8 : 4; }  // 16 bytes of x

// The tiles of n_seqs sequences (packed: one row of tokens), with the words in `workspace`.
static Tiles tiles_of(int n_seqs, int T, int C, bool packed, bool x_bf16, void* workspace) {
    const int cw = kLanesC * row_width(x_bf16);
    Tiles p{};
    p.cgroups = (C + cw - 1) / cw;
    p.cols = static_cast<int64_t>(packed ? 1 : n_seqs) * p.cgroups;
    p.tiles = (static_cast<int64_t>(T) + kTileT - 1) / kTileT;
    if (p.tiles > 1) {
        p.next = static_cast<uint32_t*>(workspace);
        p.map = static_cast<uint64_t*>(workspace) + 32;
        p.state = p.map + p.cols * p.tiles * cw;
    }
    return p;
}
static int64_t words_of(const Tiles& p, bool x_bf16) {
    if (p.tiles <= 1) return 0;
    return p.cols * (p.tiles + (p.tiles + kGroup - 1) / kGroup) * kLanesC * row_width(x_bf16);
}

int64_t recurrence_tiles(int n_seqs, int T, int C, bool packed, bool x_bf16) {
    const Tiles p = tiles_of(n_seqs, T, C, packed, x_bf16, nullptr);
    return p.cols * p.tiles;
}
size_t recurrence_ws_bytes(int n_seqs, int T, int C, bool packed, bool x_bf16) {
    const int64_t n = words_of(tiles_of(n_seqs, T, C, packed, x_bf16, nullptr), x_bf16);
    return n ? static_cast<size_t>(n + 32) * 8 : 0;
}

// Workgroups of a launch: one to a tile, up to a bound from which each takes several in turn.
static unsigned blocks_of(int64_t n) { return static_cast<unsigned>(n < (1 << 20) ? n : 1 << 20); }

static hipError_t begin(const Tiles& p, int64_t words, const RecurrenceArgs& a, hipStream_t st) {
    int64_t blocks = (words + 2047) / 2048;  // eight words a thread
    if (a.T == 0 || a.cu_seqlens) blocks = blocks > a.n_seqs ? blocks : a.n_seqs;
    blocks = blocks < 1 ? 1 : blocks > 8192 ? 8192 : blocks;
    hipLaunchKernelGGL(recurrence_begin_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, st, p.next, p.map,
                       words, a);
    return hipGetLastError();
}

hipError_t launch_recurrence(const RecurrenceArgs& a, hipStream_t st) {
    const bool packed = a.cu_seqlens != nullptr;
    const Tiles p = tiles_of(a.n_seqs, a.T, a.C, packed, a.x_bf16, a.workspace);
    hipError_t e = hipSuccess;
    if (p.next || packed || a.T == 0) e = begin(p, words_of(p, a.x_bf16), a, st);
    if (e != hipSuccess || a.T == 0) return e;
    by_types(a.x_bf16, a.g_bf16, a.h_bf16, [&](auto x, auto g, auto h) {
        typedef PM_ELEM(x) X;
        typedef PM_ELEM(g) G;
        typedef PM_ELEM(h) H;
        constexpr int V = sizeof(X) == 2 ? 8 : 4;
        const dim3 grid(blocks_of(p.cols * p.tiles));
        if (packed) hipLaunchKernelGGL((recurrence_kernel<X, G, H, V, true>), grid, dim3(kThreads), 0, st, a, p);
        else hipLaunchKernelGGL((recurrence_kernel<X, G, H, V, false>), grid, dim3(kThreads), 0, st, a, p);
        e = hipGetLastError();
    });
    return e;
}

hipError_t launch_recurrence_bwd(const RecurrenceBwdArgs& a, hipStream_t st) {
    const Tiles p = tiles_of(a.B, a.T, a.C, false, a.x_bf16, a.workspace);
    hipError_t e = hipSuccess;
    if (p.next || a.T == 0) {
        RecurrenceArgs none{};  // T 0: gs passes through to gs0
        none.n_seqs = a.T == 0 ? a.B : 0, none.C = a.C, none.s0 = a.gs, none.s_out = a.gs0;
        e = begin(p, words_of(p, a.x_bf16), none, st);
    }
    if (e != hipSuccess || a.T == 0) return e;
    by_types(a.x_bf16, a.g_bf16, a.h_bf16, [&](auto x, auto g, auto h) {
        typedef PM_ELEM(x) X;
        typedef PM_ELEM(g) G;
        typedef PM_ELEM(h) H;
        constexpr int V = sizeof(X) == 2 ? 8 : 4;
        hipLaunchKernelGGL((recurrence_bwd_kernel<X, G, H, V>), dim3(blocks_of(p.cols * p.tiles)), dim3(kThreads), 0, st,
                           a, p);
        e = hipGetLastError();
    });
    return e;
}

hipError_t launch_recurrence_step(const RecurrenceStepArgs& a, hipStream_t st) {
    hipError_t e = hipSuccess;
    const dim3 grid(static_cast<unsigned>((a.C + 255) / 256), static_cast<unsigned>(a.B < 65535 ? a.B : 65535));
    by_types(a.x_bf16, a.g_bf16, a.h_bf16, [&](auto x, auto g, auto h) {
        hipLaunchKernelGGL((recurrence_step_kernel<PM_ELEM(x), PM_ELEM(g), PM_ELEM(h)>), grid, dim3(256), 0, st, a);
        e = hipGetLastError();
    });
    return e;
}

}  // namespace pm
