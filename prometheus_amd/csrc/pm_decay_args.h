// pm_decay_args.h — what the kernels of K14 (pm_decay.h) take, for them and their callers.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace pm {

constexpr int kDecayGateSpan = 512;  // the longest span where the gates' gradient is wanted

// Columns of the state that a workgroup keeps (pm_decay.h: DecayTile).
constexpr int decay_cols(int D) { return D <= 64 ? 64 : 128; }

// Spans of a sequence, one at least.  (No sum with the span's length: both may be near 2^31.)
__host__ __device__ inline int spans_of(int len, int span) { return len > 0 ? 1 + (len - 1) / span : 1; }
// The last token of the span that begins at `begin` < len, plus one.
__host__ __device__ inline int span_end(int begin, int span, int len) {
    return span < len - begin ? begin + span : len;
}

// One pass over n_seqs sequences (roles as in pm_decay.h).  Strides are in elements; the elements of
// a head are contiguous.  HO heads of Q and O, HK of K and V, HS = min(HO, HK) states.
struct DecayPass {
    const void* q;
    const void* k;
    const void* v;
    int64_t q_sb, q_st, q_sh, k_sb, k_st, k_sh, v_sb, v_st, v_sh;
    const float* g;  // [b][t][HS], heads contiguous; both strides 0: one constant a head
    int64_t g_sb, g_st;
    const int32_t* cu;  // nullable: packed (T tokens, n_seqs + 1 offsets, clamped into [0, T])
    const float* s0;    // nullable: zeros; not read where span_state is given
    float* s_out;       // nullable
    int64_t s_row, s_col;  // strides of a state's rows (K's dimension) and columns (V's)
    const int32_t* slots;  // nullable: sequence i's state is row slots[i] of the pool s0, s_out
    int n_slots;
    int32_t* bad_slot;  // nullable
    bool s0_gathered;   // s0 holds the sequences' states in order, whatever the slots
    void* o;            // contiguous (.., HO, D)
    bool out_bf16, reverse;
    int n_seqs, T, HO, HK, HS, D;
    int n_dst;          // output heads a workgroup takes, one after another (1 where HK > HO)
    int n_tiles;        // column tiles of decay_cols(D)
    // Spans: workgroups along a sequence.  Slot i is span i % n_spans of sequence i / n_spans, or
    // (packed) slot_table[i] = (sequence, span), sequence -1: none; a sequence's slots are in a row.
    int span, n_spans, n_slots_grid;
    const int2* slot_table;
    float* span_state;  // nullable: [slot][HS] states before the spans, (D, D) with strides u_row, u_col
    int64_t u_row, u_col;
    double* span_log;   // [slot][HS] the log-decay of the span before, in units of log 2
    float a_scale, into_scale, out_scale;  // of A, of the state's part of O, of what enters the state
    // for the gates' gradient
    const void* aux;    // q (gq's pass), k (gk's)
    int64_t x_sb, x_st, x_sh;
    float* part;        // nullable; [tile][HO][row]: each token's product of aux with the state's part of O
    int64_t n_rows;
};

// Up to three passes that run as one launch.
struct DecayPasses {
    DecayPass pass[3];
    int n;
};

// The pairs inside chunks.
struct DecayNear {
    const void* q;
    const void* k;
    const void* v;
    const void* go;
    int64_t q_sb, q_st, q_sh, k_sb, k_st, k_sh, v_sb, v_st, v_sh, go_sb, go_st, go_sh;
    const float* g;
    int64_t g_sb, g_st;
    float* near;  // [Hq][row]
    int64_t n_rows;
    int B, T, Hq, H, D;
    float scale;
};

// The gates' gradient from what the passes left.
struct DecayGateGrad {
    const float* g;
    int64_t g_sb, g_st;
    const float* r_part;  // [tile][Hq][row]
    const float* c_part;  // [tile][H][row]
    const float* near;    // [Hq][row]
    const float* ahead;   // nullable: the states before the spans, [slot][H] (slots in order of time)
    const float* back;    // nullable: their gradients behind the spans, [slot][H], the last span's first
    const float* s0;      // nullable: the first state
    const float* gs0;     // its gradient, where s0 is given
    float* gg;            // nullable: (B, T, H)
    float* gg_part;       // nullable: (B, n_spans, H)
    int64_t n_rows;
    int B, T, Hq, H, D, n_tiles, span, n_spans, chunk;
};

// kind: 0 outputs and states, 1 the same and `part`s, 2 each span's own share of the state (from zeros) but
// the last one's, to the next slot of span_state.
hipError_t decay_pass_bf16(const DecayPasses& a, int kind, hipStream_t st);
hipError_t decay_pass_f32(const DecayPasses& a, int kind, hipStream_t st);
hipError_t decay_near_bf16(const DecayNear& a, hipStream_t st);
hipError_t decay_near_f32(const DecayNear& a, hipStream_t st);

}  // namespace pm
