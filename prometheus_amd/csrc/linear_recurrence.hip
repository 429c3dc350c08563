// linear_recurrence.hip — K12: the elementwise gated linear recurrence, its gradients and its
// single-token step.
//
//   h_t = exp(g_t) h_{t-1} + x_t          for every channel on its own
//   d_t = gh_t + exp(g_{t+1}) d_{t+1},  gx_t = d_t,  gg_t = d_t exp(g_t) h_{t-1}
//
// Bound by memory: one exponential and a few multiply-adds an element against 6 bytes (bf16
// forward) or 10 (backward). So every element is read once and written once: a tile of 512 tokens
// by one 128-byte line of channels stays in registers from its loads to its stores, and what
// tokens need of each other goes as affine maps s -> A s + H of the spans between them.
//   1. each thread folds its own 8 tokens of 8 (fp32: 4) channels into one map;
//   2. through LDS the tile's maps fold in a fixed tree: per part of the tile, then the tile;
//   3. a tile that is not its sequence's first waits for the state before it (below);
//   4. the state walks down the tree again and through each thread's tokens.
// The backward is the same with the message c_t = exp(g_t) d_t, c_t = exp(g_t) (gh_t + c_{t+1}),
// from the last tile to the first, on top of a forward inside the tile from the kept state.
//
// Between tiles, in one pass: a tile publishes its map as soon as it is folded; the state before
// tile j is the state at the start of j's group of 16 tiles, taken through the maps of the group's
// tiles before j in order; the group's last tile publishes the next group's state. The order of
// every product and sum is fixed by j, not by which tile is done first, so results are the same
// bits every time; and the chain that cannot run in parallel is one hop in 16 tiles. Words carry
// value and readiness together (relaxed 8-byte atomics of agent scope; the workspace starts as all
// ones, which no value is), so no fences. Tiles are handed out by a counter in the order in which
// they wait for each other, and a workgroup finishes its tile before it folds its next: the first
// tile that is not done is always somebody's to do, and waits for nothing, so every wait ends.
//
// Workgroups stay: while one walks and stores, its next tile's loads are under way (forward; the
// backward's registers hold one tile). A tile is 196 kB of traffic to a compute unit, whose 512
// threads hold x and gh as they are in memory, and make what they need of them again after the
// wait; the gates, of which an exponential is a quarter of a tile's arithmetic, are kept.
//
// Measured (calls among others, their begin kernels with them, on a card that copies at 5.0 TB/s):
// forward 4 x 4096 tokens of 4096 bf16 channels 71 us (5.6 TB/s), backward 134 (5.0 TB/s), 65521
// tokens of 2048 channels 144 (5.6 TB/s). On the way, when this form took 79, 131 and 146: 256-token
// tiles, a workgroup to each and every value held 121, 226 and 239; as here but gates made twice 88,
// 140 and 163; a branch at every row and words asked for after the tile's loads 82, 135 and 151. An
// elementwise pass over the same lines takes 84, over rows of 512 bytes 69; but wide tiles are short,
// and four times the hops and words cost more than the rows gain (256 bytes, two workgroups to a
// compute unit: 151 for the long one; 512 bytes: 183). Columns dealt to XCDs in runs of neighbours
// were slower (96 of 88), stores that stay out of the caches 2% faster.

#include "pm_internal.h"
#include "pm_vec.h"

namespace pm {

constexpr int kLanesC = 8;  // threads across the channels of a tile: a 128-byte line of x
constexpr int kGroup = 16;  // tiles to a group

// The shape of a tile: `tok` tokens to a thread, `threads` to a workgroup. Long tiles fill a
// compute unit with one workgroup and pass states on; of the others, which hold the whole of a
// short sequence, two or four fit.
template <int TOK, int THREADS, int BLOCKS, bool CHAINED>
struct Shape {
    static constexpr int tok = TOK, threads = THREADS, span = THREADS / kLanesC * TOK;
    static constexpr int blocks = BLOCKS;                       // workgroups that the card holds at a time
    static constexpr int waves = THREADS * BLOCKS / 256 / 256;  // to a SIMD
    static constexpr bool chained = CHAINED;
};
typedef Shape<8, 512, 256, true> Long;
typedef Shape<4, 512, 512, false> Middle;
typedef Shape<4, 256, 1024, false> Short;
static_assert(Long::span % kRecSpan == 0 && Middle::span % kRecSpan == 0 && Short::span == kRecSpan,
              "kept states start every tile");

// The tiles of a call and the words through which they pass states (all null where each
// sequence is one tile).
struct Tiles {
    int cgroups;     // channel groups
    int64_t cols;    // sequences x channel groups
    int64_t tiles;   // tiles along the tokens
    int span;        // tokens to a tile: which Shape
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
__device__ __forceinline__ uint64_t load_word(uint64_t* p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ bool missing(uint64_t v) { return static_cast<uint32_t>(v >> 32) == 0xffffffffu; }
__device__ __forceinline__ float low(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v)); }
__device__ __forceinline__ float high(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v >> 32)); }

// a b of factors of maps, which rounds to zero only where one of them is zero (a gate that is closed):
// an infinite state stays one through however many gates, as it does token by token, and 0 x inf comes
// of closed gates alone. (As bits: a factor is at least +0, but for a start's, of which the sign alone
// counts. To a finite state's share this adds at most 2^-149 of the state.)
__device__ __forceinline__ float product(float a, float b) {
    return __uint_as_float(max(__float_as_uint(a * b), min(min(__float_as_uint(a), __float_as_uint(b)), 1u)));
}

// s -> A s + H. An A whose sign bit is set (PACKED only) is a map that a sequence starts in: its H
// is the state whatever came before, infinities and NaN included.
template <bool PACKED>
struct Map {
    float A, H;
    __device__ __forceinline__ bool anew() const { return PACKED && static_cast<int>(__float_as_uint(A)) < 0; }
    // a token's gate (which has no sign) and input; the sign of A stays
    __device__ __forceinline__ void token(float a, float x) { H = fmaf(a, H, x), A *= a; }
    __device__ __forceinline__ void then(const Map& m) {
        H = m.of(H);
        A = m.anew() ? m.A : product(A, m.A);
    }
    __device__ __forceinline__ float of(float s) const { return anew() ? H : fmaf(A, s, H); }
    __device__ __forceinline__ uint64_t word() const {
        const uint32_t a = __float_as_uint(A);
        return pm::word(a == 0xffffffffu ? 0x7fc00000u : a, H);  // (a NaN all of whose bits are set)
    }
    static __device__ __forceinline__ Map read(uint64_t v) { return {high(v), low(v)}; }
};

// A thread's factors m[v].A, as they are in p, after its K tokens with the gates gate(r, v): where plain
// products have rounded to zero, which they hardly ever do, p gets what `product` says.
template <int K, int V, bool PACKED, typename F>
__device__ __forceinline__ void keep_open(float* p, const Map<PACKED> (&m)[V], F gate) {
    uint32_t least = ~0u;
#pragma unroll
    for (int v = 0; v < V; ++v) least = min(least, __float_as_uint(m[v].A));
    if (!__any(least == 0)) return;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        bool open = __float_as_uint(p[v]) == 0;  // (not a start's -0)
#pragma unroll
        for (int r = 0; r < K; ++r) open = open && gate(r, v) != 0.f;
        if (open) p[v] = product(0x1p-100f, 0x1p-100f);
    }
}

// (the hardware's exponential has no values below 2^-126: such a gate is zero)
__device__ __forceinline__ float gate(float g) { return __builtin_amdgcn_exp2f(g * 1.44269504088896341f); }

__host__ __device__ inline int64_t spans_of(int T) { return (static_cast<int64_t>(T) + kRecSpan - 1) / kRecSpan; }

// Row of a sequence's state in s0 and s_out, or -1 (a slot outside the pool).
__device__ __forceinline__ int64_t state_row(const int32_t* slots, int n_slots, int seq) {
    if (!slots) return seq;
    const int r = slots[seq];
    return r >= 0 && r < n_slots ? r : -1;
}

// Waits for all of the wave's loads. Where a branch may have left some under way, the compiler
// holds up the next use of their registers until every load before is back, the tile's own too.
__device__ __forceinline__ void loads_done() { __builtin_amdgcn_s_waitcnt(0x0f70); }  // vmcnt(0)

// What the thread (ch, part) of a tile's fold takes from the tiles before: some of the group's maps
// and, in part 0, the state at the group's start. `j` counts tiles in the order in which they wait
// for each other. All threads of a workgroup call all three.
template <bool CHAINED, bool PACKED, int CW, int PARTS>
struct Before {
    static constexpr int Q = (kGroup + PARTS - 1) / PARTS;  // tiles of the group to a part
    uint64_t* maps;
    uint64_t* from;
    uint64_t w[Q], s;
    int n;      // maps to read
    bool deep;  // whether to read the state

    // Asks for every word.
    __device__ __forceinline__ void look(const Tiles& p, int64_t col, int64_t j, int ch, int part) {
        if (!CHAINED || !p.next) return;
        const int64_t g0 = j / kGroup * kGroup, groups = (p.tiles + kGroup - 1) / kGroup;
        n = static_cast<int>(j - g0) - part * Q;
        deep = part == 0 && g0 > 0;
        maps = p.map + (col * p.tiles + g0 + part * Q) * CW + ch;
        from = p.state + (col * groups + j / kGroup) * CW + ch;
        if (deep) s = load_word(from);
#pragma unroll
        for (int i = 0; i < Q; ++i)
            if (i < n) w[i] = load_word(maps + static_cast<int64_t>(i) * CW);
    }
    // Waits for them. Loads come back in the order they were asked for, so this is done before the
    // next tile's are, which would have to come back first.
    __device__ __forceinline__ void wait(const Tiles& p) {
        if (!CHAINED || !p.next) return;
        for (;;) {  // (again for all that are missing at a time)
            const bool s_missing = deep && missing(s);
            bool any = s_missing, w_missing[Q];
#pragma unroll
            for (int i = 0; i < Q; ++i) w_missing[i] = i < n && missing(w[i]), any |= w_missing[i];
            if (!any) break;
            __builtin_amdgcn_s_sleep(1);
            if (s_missing) s = load_word(from);
#pragma unroll
            for (int i = 0; i < Q; ++i)
                if (w_missing[i]) w[i] = load_word(maps + static_cast<int64_t>(i) * CW);
        }
        loads_done();
    }
    // The state before tile j; `first` is that before tile 0, `lb` is LDS [PARTS][CW].
    __device__ __forceinline__ float state(const Tiles& p, int64_t j, int ch, int part, float first,
                                           Map<PACKED> (*lb)[CW]) {
        if (!CHAINED || !p.next || j == 0) return first;
        Map<PACKED> m{1.f, 0.f};
#pragma unroll
        for (int i = 0; i < Q; ++i)
            if (i < n) m.then(Map<PACKED>::read(w[i]));
        if (part == 0) m.H = m.of(deep ? low(s) : first);
        lb[part][ch] = m;
        __syncthreads();
        float before = lb[0][ch].H;
        const int all = static_cast<int>(j % kGroup);
#pragma unroll
        for (int i = 1; i < PARTS; ++i)
            if (i * Q < all) before = lb[i][ch].of(before);
        return before;
    }
};

template <int CW>
__device__ __forceinline__ void publish_state(const Tiles& p, int64_t col, int64_t j, int ch, float s) {
    if (!p.next || j % kGroup != kGroup - 1 || j + 1 >= p.tiles) return;
    const int64_t groups = (p.tiles + kGroup - 1) / kGroup;
    publish(p.state + (col * groups + j / kGroup + 1) * CW + ch, word(0, s));
}

// A workgroup's tiles: thread 0 asks for the next one early (ask), all threads have it after the
// barrier that follows tell.
struct Turns {
    const Tiles& p;
    uint32_t* slot;  // LDS
    uint32_t got;
    int64_t id;
    __device__ __forceinline__ Turns(const Tiles& tiles, uint32_t* lds) : p(tiles), slot(lds), got(0), id(blockIdx.x) {
        if (!p.next) return;
        ask();
        tell();
        __syncthreads();
        take();
        __syncthreads();
    }
    __device__ __forceinline__ bool done() const { return id >= p.cols * p.tiles; }
    __device__ __forceinline__ void ask() {
        if (p.next && threadIdx.x == 0)
            got = __hip_atomic_fetch_add(p.next, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __device__ __forceinline__ void tell() {
        if (p.next && threadIdx.x == 0) *slot = got;
    }
    __device__ __forceinline__ void take() { id = p.next ? *slot : id + gridDim.x; }
};

template <bool PACKED, int CW>
struct Place {
    int64_t j, col;
    int seq, cbase;
    __device__ __forceinline__ Place(const Tiles& p, int64_t id) {
        // (32 bits: the number of tiles is at most 2^31)
        const uint32_t u = static_cast<uint32_t>(id), cols = static_cast<uint32_t>(p.cols);
        const uint32_t q = u / cols, c = u - q * cols;
        j = q, col = c;
        const uint32_t b = PACKED ? 0 : c / static_cast<uint32_t>(p.cgroups);
        seq = static_cast<int>(b);
        cbase = static_cast<int>(c - b * p.cgroups) * CW;
    }
};

// A thread's rows of a tensor: token r at p + r st; those of `tokens` and `nc` channels that there
// are, zeros for the others.
template <typename E, int V, int K>
__device__ __forceinline__ void load_rows(Row<E, V> (&rows)[K], const E* p, int64_t st) {
#pragma unroll
    for (int r = 0; r < K; ++r) rows[r].load(p + r * st);
}
template <typename E, int V, int K>
__device__ __forceinline__ void load_rows(Row<E, V> (&rows)[K], const E* p, int64_t st, int tokens, int nc) {
#pragma unroll
    for (int r = 0; r < K; ++r) rows[r].load(p + r * st, r < tokens ? nc : 0);
}
// Whether every token and channel of the tile is there.
template <typename S, int CW>
__device__ __forceinline__ bool tile_full(int T, int C, int64_t tile, int cbase) {
    return (tile + 1) * S::span <= T && cbase + CW <= C;
}

// Keeps the compiler from carrying values made from a row across this point in registers: they
// are made again from the row, which costs less than the waves that the registers would.
template <typename E, int V>
__device__ __forceinline__ void forget(Row<E, V>& r) {
#pragma unroll
    for (uint32_t& w : r.raw) asm volatile("" : "+v"(w));
}

template <typename X, typename G, typename H, int V, typename S, bool PACKED>
__global__ __launch_bounds__(S::threads, S::waves) void recurrence_kernel(RecurrenceArgs a, Tiles p) {
    constexpr int K = S::tok, CW = kLanesC * V, TL = S::span / K, PARTS = S::threads / CW, PER = TL / PARTS;
    typedef Map<PACKED> M;
    __shared__ float sA[TL][CW], sH[TL][CW];
    __shared__ M total[PARTS][CW], lb[PARTS][CW];
    // where a packed sequence starts or ends in the tile: which one, by token, and the tokens, a
    // bit each, by thread (starts below, ends from bit K on)
    __shared__ int start[PACKED ? S::span : 1], stop[PACKED ? S::span : 1];
    __shared__ unsigned marks[PACKED ? TL : 1];
    __shared__ float first[CW];
    __shared__ uint32_t slot;
    const int tid = threadIdx.x, lc = tid % kLanesC, tl = tid / kLanesC;
    const int ch = tid % CW, part = tid / CW;

    // a sequence's offsets, clamped; the first S::threads sequences' stay in registers
    auto offset = [&](int i) { return min(max(a.cu_seqlens[i], 0), a.T); };
    int b0 = 0, e0 = 0;
    if constexpr (PACKED) {
        if (tid < a.n_seqs) b0 = offset(tid), e0 = offset(tid + 1);
        if (tid < TL) marks[tid] = 0;
        __syncthreads();
    }

    Before<S::chained, PACKED, CW, PARTS> before;
    Turns turns(p, &slot);
    Row<X, V> xn[K];
    Row<G, V> gn[K];
    auto load_next = [&] {
        if (turns.done()) return;
        const Place<PACKED, CW> at(p, turns.id);
        const int t0 = static_cast<int>(at.j) * S::span + tl * K, c0 = at.cbase + lc * V;
        const bool full = tile_full<S, CW>(a.T, a.C, at.j, at.cbase);
        const X* xp = static_cast<const X*>(a.x) + at.seq * a.x_sb + t0 * a.x_st + c0;
        const G* gp = static_cast<const G*>(a.g) + at.seq * a.g_sb + t0 * a.g_st + c0;
        if (full) {
            load_rows(xn, xp, a.x_st);
            load_rows(gn, gp, a.g_st);
        } else {
            load_rows(xn, xp, a.x_st, a.T - t0, a.C - c0);
            load_rows(gn, gp, a.g_st, a.T - t0, a.C - c0);
            loads_done();
        }
    };
    // (short tiles have other workgroups of their compute unit to read meanwhile, and spilled)
    if constexpr (S::chained) load_next();
    while (!turns.done()) {
        if constexpr (!S::chained) load_next();
        const Place<PACKED, CW> at(p, turns.id);
        const int64_t j = at.j, col = at.col;
        const int seq = at.seq, cbase = at.cbase;
        const int c0 = cbase + lc * V, nc = a.C - c0;  // this thread's channels, and how many are there
        const int tile0 = static_cast<int>(j) * S::span, t0 = tile0 + tl * K;
        const bool full = tile_full<S, CW>(a.T, a.C, j, cbase);
        Row<X, V> xr[K];
        Row<G, V> gr[K];
#pragma unroll
        for (int r = 0; r < K; ++r) xr[r] = xn[r], gr[r] = gn[r];
        turns.ask();
        before.look(p, col, j, ch, part);
        // the state before the sequence: read by its first tile only, before that tile's map is
        // out, as the last tile may write the same row of the pool soon after
        if (!PACKED && j == 0 && part == 0) {
            const int64_t row = state_row(a.slots, a.n_slots, seq);
            if (row < 0 && a.bad) atomicOr(a.bad, 1);
            first[ch] = a.s0 && row >= 0 && cbase + ch < a.C ? a.s0[row * a.C + cbase + ch] : 0.f;
        }
        H* hp = static_cast<H*>(a.h) + (static_cast<int64_t>(seq) * a.T + t0) * a.C + c0;
        auto finish = [&](int r, const float(&h)[V], int ends) {
            if (t0 + r < a.T) store_row<H, V>(hp + static_cast<int64_t>(r) * a.C, h, nc);
            if (ends >= 0) {
                const int64_t row = state_row(a.slots, a.n_slots, ends);
                if (row >= 0) store_row<float, V>(a.s_out + row * a.C + c0, h, nc);
            }
        };
        unsigned mark = 0;
        auto boundaries = [&](int b, int e, int i) {  // of sequence i, as far as they are in this tile
            const int u = b - tile0, w = e - 1 - tile0;
            if (b < e && u >= 0 && u < S::span) start[u] = i, atomicOr(marks + u / K, 1u << u % K);
            if (b < e && w >= 0 && w < S::span) stop[w] = i, atomicOr(marks + w / K, 1u << (K + w % K));
        };
        if constexpr (PACKED) {
            boundaries(b0, e0, tid);
            for (int i = tid + S::threads; i < a.n_seqs; i += S::threads) boundaries(offset(i), offset(i + 1), i);
            __syncthreads();
            mark = marks[tl];
        }
        int known = K;  // tokens from here on follow a sequence's start in this thread
        float av[K][V];
#pragma unroll
        for (int r = 0; r < K; ++r)
#pragma unroll
            for (int v = 0; v < V; ++v) av[r][v] = gate(gr[r][v]);
        M m[V];
#pragma unroll
        for (int v = 0; v < V; ++v) m[v] = {1.f, 0.f};
        // (tokens past the end are zeros: gates of one and nothing added)
        if (!PACKED || !__any(mark != 0)) {
#pragma unroll
            for (int r = 0; r < K; ++r)
#pragma unroll
                for (int v = 0; v < V; ++v) m[v].token(av[r][v], xr[r][v]);
        } else {
#pragma unroll
            for (int r = 0; r < K; ++r) {
                if (mark >> r & 1) {
                    // the start's state is read here, once: the sequence's last tile may write the
                    // same row of the pool as soon as this tile's map is out
                    const int64_t row = state_row(a.slots, a.n_slots, start[tl * K + r]);
                    if (row < 0 && a.bad) atomicOr(a.bad, 1);
                    Row<float, V> s;
                    s.load(a.s0 && row >= 0 ? a.s0 + row * a.C + c0 : nullptr, a.s0 && row >= 0 ? nc : 0);
#pragma unroll
                    for (int v = 0; v < V; ++v) m[v] = {-1.f, s[v]};
                    known = min(known, r);
                }
#pragma unroll
                for (int v = 0; v < V; ++v) m[v].token(av[r][v], xr[r][v]);
                if (known <= r) {
                    // nothing before this thread's tokens matters any more: h is there
                    float h[V];
#pragma unroll
                    for (int v = 0; v < V; ++v) h[v] = m[v].H;
                    finish(r, h, mark >> (K + r) & 1 ? stop[tl * K + r] : -1);
                }
            }
        }
#pragma unroll
        for (int v = 0; v < V; ++v) sA[tl][lc * V + v] = m[v].A, sH[tl][lc * V + v] = m[v].H;
        keep_open<K>(&sA[tl][lc * V], m, [&](int r, int v) { return av[r][v]; });
        __syncthreads();

        if (PACKED && tid < TL) marks[tid] = 0;  // (read above; the next tile's come after a barrier)
        M mine[PER], sum{1.f, 0.f};
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            mine[i] = {sA[part * PER + i][ch], sH[part * PER + i][ch]};
            sum.then(mine[i]);
        }
        total[part][ch] = sum;
        turns.tell();
        __syncthreads();
        turns.take();
        float s = !PACKED && j == 0 ? first[ch] : 0.f;
        if (S::chained && p.next && part == 0) {
#pragma unroll
            for (int i = 1; i < PARTS; ++i) sum.then(total[i][ch]);
            if (!PACKED && j == 0) sum = {0.f, sum.of(s)};  // the first tile's map yields its state
            publish(p.map + (col * p.tiles + j) * CW + ch, sum.word());
        }
        before.wait(p);
        if constexpr (S::chained) load_next();
        s = before.state(p, j, ch, part, s, lb);
#pragma unroll
        for (int i = 0; i < PARTS; ++i)
            if (i < part) s = total[i][ch].of(s);
        const int from = tile0 + part * PER * K;  // this part's first token
        if (!PACKED && a.kept && from % kRecSpan == 0 && from < a.T && cbase + ch < a.C)
            a.kept[(seq * spans_of(a.T) + from / kRecSpan) * a.C + cbase + ch] = s;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            sH[part * PER + i][ch] = s;
            s = mine[i].of(s);
        }
        if (S::chained && part == PARTS - 1) publish_state<CW>(p, col, j, ch, s);
        __syncthreads();

        float h[V];
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = sH[tl][lc * V + v];
        __syncthreads();  // (the next tile's maps go where these states were)
#pragma unroll
        for (int r = 0; r < K; ++r) forget(xr[r]);
        auto walk = [&](int r) {
#pragma unroll
            for (int v = 0; v < V; ++v) h[v] = fmaf(av[r][v], h[v], xr[r][v]);
        };
        if (full && (!PACKED || !__any(mark != 0))) {
#pragma unroll
            for (int r = 0; r < K; ++r) {
                walk(r);
                Row<H, V> out;
#pragma unroll
                for (int v = 0; v < V; ++v) out.set(v, h[v]);
                out.store(hp + static_cast<int64_t>(r) * a.C);
            }
            if (!PACKED && t0 + K == a.T) finish(K, h, seq);  // (token K is none of the tile's: the state alone)
        } else if (!PACKED) {
#pragma unroll
            for (int r = 0; r < K; ++r) {
                walk(r);
                finish(r, h, t0 + r == a.T - 1 ? seq : -1);
            }
        } else {
#pragma unroll
            for (int r = 0; r < K; ++r) {
                if (known <= r) break;
                walk(r);
                finish(r, h, mark >> (K + r) & 1 ? stop[tl * K + r] : -1);
            }
        }
        if constexpr (PACKED) __syncthreads();  // (and its boundaries where these are)
    }
}

// The gradients; tiles go from the last to the first, and c_t = exp(g_t) d_t is the state.
template <typename X, typename G, typename H, int V, typename S>
__global__ __launch_bounds__(S::threads, S::waves) void recurrence_bwd_kernel(RecurrenceBwdArgs a, Tiles p) {
    constexpr int K = S::tok, CW = kLanesC * V, TL = S::span / K, PARTS = S::threads / CW, PER = TL / PARTS;
    typedef Map<false> M;
    __shared__ float sA[TL][CW], sF[TL][CW], sB[TL][CW];
    __shared__ M fwd[PARTS][CW], bwd[PARTS][CW], lb[PARTS][CW];
    __shared__ uint32_t slot;
    const int tid = threadIdx.x, lc = tid % kLanesC, tl = tid / kLanesC;
    const int ch = tid % CW, part = tid / CW;

    Before<S::chained, false, CW, PARTS> before;
    Turns turns(p, &slot);
    while (!turns.done()) {
        const Place<false, CW> at(p, turns.id);
        const int64_t j = at.j, col = at.col, tile = p.tiles - 1 - j;
        const int b = at.seq, cbase = at.cbase;
        const int c0 = cbase + lc * V, nc = a.C - c0;
        const int t0 = static_cast<int>(tile) * S::span + tl * K;
        const int64_t out = (static_cast<int64_t>(b) * a.T + t0) * a.C + c0;
        const bool full = tile_full<S, CW>(a.T, a.C, tile, cbase);
        Row<X, V> xr[K];
        Row<G, V> gr[K];
        Row<H, V> hr[K];
        const X* xp = static_cast<const X*>(a.x) + b * a.x_sb + t0 * a.x_st + c0;
        const G* gp = static_cast<const G*>(a.g) + b * a.g_sb + t0 * a.g_st + c0;
        const H* hp = static_cast<const H*>(a.gh) + out;
        if (full && a.gh) {
            load_rows(xr, xp, a.x_st);
            load_rows(gr, gp, a.g_st);
            load_rows(hr, hp, a.C);
        } else {
            load_rows(xr, xp, a.x_st, a.T - t0, nc);
            load_rows(gr, gp, a.g_st, a.T - t0, nc);
            load_rows(hr, hp, a.C, a.gh ? a.T - t0 : 0, nc);
            loads_done();
        }
        turns.ask();
        before.look(p, col, j, ch, part);
        const bool there = cbase + ch < a.C;
        float h = there ? a.kept[(b * spans_of(a.T) + tile * (S::span / kRecSpan)) * a.C + cbase + ch] : 0.f;
        // (bf16 rows leave registers for the gates; beside fp32 rows they are made again: 132 us at 4 x
        // 4096 tokens of 2048 channels, kept 146)
        constexpr bool KEEP = sizeof(X) == 2;
        float av[KEEP ? K : 1][KEEP ? V : 1];
        if constexpr (KEEP) {
#pragma unroll
            for (int r = 0; r < K; ++r)
#pragma unroll
                for (int v = 0; v < V; ++v) av[r][v] = gate(gr[r][v]);
        }
        auto gate_at = [&](int r, int v) {
            if constexpr (KEEP) return av[r][v];
            else return gate(gr[r][v]);
        };
        M maps[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            M f{1.f, 0.f};  // the tokens' map of h
            float w = 0.f;  // and of c, whose factor is the same
#pragma unroll
            for (int r = 0; r < K; ++r) f.token(gate_at(r, v), xr[r][v]);
#pragma unroll
            for (int r = K - 1; r >= 0; --r) w = gate_at(r, v) * (w + hr[r][v]);
            sA[tl][lc * V + v] = f.A, sF[tl][lc * V + v] = f.H, sB[tl][lc * V + v] = w;
            maps[v].A = f.A;
        }
        keep_open<K>(&sA[tl][lc * V], maps, gate_at);
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
        turns.tell();
        __syncthreads();
        turns.take();
        if (S::chained && p.next && part == PARTS - 1) {
#pragma unroll
            for (int i = PARTS - 2; i >= 0; --i) down.then(bwd[i][ch]);
            publish(p.map + (col * p.tiles + j) * CW + ch, down.word());
        }
        float c = a.gs && j < kGroup && there ? a.gs[static_cast<int64_t>(b) * a.C + cbase + ch] : 0.f;
        before.wait(p);
        c = before.state(p, j, ch, part, c, lb);
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
            if (S::chained) publish_state<CW>(p, col, j, ch, c);
            if (tile == 0 && there) a.gs0[static_cast<int64_t>(b) * a.C + cbase + ch] = c;
        }
        __syncthreads();

        Row<X, V> gx[K];
        Row<G, V> gg[K];
#pragma unroll
        for (int r = 0; r < K; ++r) {
            forget(xr[r]), forget(hr[r]);
            if constexpr (!KEEP) forget(gr[r]);
        }
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float hb[K];  // the state before each token
            hb[0] = sF[tl][lc * V + v];
#pragma unroll
            for (int r = 1; r < K; ++r) hb[r] = fmaf(gate_at(r - 1, v), hb[r - 1], xr[r - 1][v]);
            float cv = sB[tl][lc * V + v];
#pragma unroll
            for (int r = K - 1; r >= 0; --r) {
                const float d = hr[r][v] + cv;
                cv = gate_at(r, v) * d;
                gx[r].set(v, d);
                gg[r].set(v, cv * hb[r]);
            }
        }
        __syncthreads();  // (the next tile's maps go where these states were)
        X* gxp = static_cast<X*>(a.gx) + out;
        G* ggp = static_cast<G*>(a.gg) + out;
        if (full) {
#pragma unroll
            for (int r = 0; r < K; ++r) {
                gx[r].store(gxp + static_cast<int64_t>(r) * a.C);
                gg[r].store(ggp + static_cast<int64_t>(r) * a.C);
            }
        } else {
#pragma unroll
            for (int r = 0; r < K; ++r)
                if (t0 + r < a.T) {
                    gx[r].store(gxp + static_cast<int64_t>(r) * a.C, nc);
                    gg[r].store(ggp + static_cast<int64_t>(r) * a.C, nc);
                }
        }
    }
}

// Before a call: `n` words of the workspace to all ones and the counter to zero; the check of a
// packed call's offsets; and the states of sequences without tokens (all of them where T is 0),
// which pass through.
__global__ __launch_bounds__(256) void recurrence_begin_kernel(uint32_t* next, uint64_t* words, int64_t n,
                                                               RecurrenceArgs a) {
    const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    const int64_t step = static_cast<int64_t>(gridDim.x) * 256;
    if (next && at == 0) *next = 0;
    for (int64_t i = at; i < n; i += step) words[i] = ~uint64_t(0);
    for (int seq = blockIdx.x; seq < a.n_seqs; seq += gridDim.x) {
        if (a.cu_seqlens && a.cu_flag && threadIdx.x == 0) {
            const int b = a.cu_seqlens[seq], e = a.cu_seqlens[seq + 1];
            const bool last = seq == a.n_seqs - 1;
            const int bits = (seq == 0 && b != 0 ? 1 : 0) | (last && e != a.T ? 2 : 0) | (e < b ? 4 : 0) |
                             (b < 0 || b > a.T || (last && (e < 0 || e > a.T)) ? 8 : 0);
            if (bits) atomicOr(a.cu_flag, bits);
        }
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
    // sequences that a short tile holds take it: as many bytes under way with fewer idle threads
    // (64 x 128 tokens of 2048 channels forward 18 us, in long tiles 67; 16 x 256 of 4096 middle
    // 17.5, long 34); longer ones never do (4 x 4096 of 4096: short 124, long 89)
    p.span = T <= Short::span ? Short::span : T <= Middle::span ? Middle::span : Long::span;
    p.tiles = (static_cast<int64_t>(T) + p.span - 1) / p.span;
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

// f(Shape, grid) of a call
template <typename F>
static void by_shape(const Tiles& p, F f) {
    const int64_t n = p.cols * p.tiles;
    auto go = [&](auto shape) {
        f(shape, dim3(static_cast<unsigned>(n < decltype(shape)::blocks ? n : decltype(shape)::blocks)));
    };
    if (p.span == Short::span) go(Short{});
    else if (p.span == Middle::span) go(Middle{});
    else go(Long{});
}

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
        by_shape(p, [&](auto shape, dim3 grid) {
            typedef decltype(shape) S;
            const dim3 block(S::threads);
            if (packed) hipLaunchKernelGGL((recurrence_kernel<X, G, H, V, S, true>), grid, block, 0, st, a, p);
            else hipLaunchKernelGGL((recurrence_kernel<X, G, H, V, S, false>), grid, block, 0, st, a, p);
        });
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
        by_shape(p, [&](auto shape, dim3 grid) {
            typedef decltype(shape) S;
            hipLaunchKernelGGL((recurrence_bwd_kernel<X, G, H, V, S>), grid, dim3(S::threads), 0, st, a, p);
        });
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
