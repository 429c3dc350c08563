// pm_layer_abi.hip — the extern "C" entry points of the operators beside the delta rule:
// K12 (linear_recurrence.hip) and K13 (norm_rotate.hip).
//
// As in pm_delta_abi.hip every argument is checked before anything is launched; errors are
// negative PM_E_* codes with a message in pm_last_error().

#include "pm_common.h"
#include "pm_internal.h"
#include "../../include/pm_delta.h"

static_assert(PM_RECURRENCE_SPAN == pm::kRecSpan, "the header's span is the kernels'");

namespace {

using pm::fail;

bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

int hip_fail(hipError_t e, const char* what) {
    return fail(static_cast<int>(e), "%s: HIP error %d (%s)", what, static_cast<int>(e), hipGetErrorString(e));
}

bool known(int dtype) { return dtype == PM_DTYPE_F32 || dtype == PM_DTYPE_BF16; }
size_t size_of(int dtype) { return dtype == PM_DTYPE_BF16 ? 2 : 4; }

constexpr int64_t kMaxElems = int64_t(1) << 40;
constexpr int64_t kMaxStride = int64_t(1) << 40;

// The types of x, g and h: bf16 gates go with bf16 x.
int check_types(int x, int g, int h) {
    if (!known(x) || !known(g) || !known(h))
        return fail(PM_E_DTYPE, "types %d, %d, %d: each must be PM_DTYPE_F32 or PM_DTYPE_BF16", x, g, h);
    if (x == PM_DTYPE_F32 && g == PM_DTYPE_BF16)
        return fail(PM_E_DTYPE, "bf16 log-gates need bf16 x");
    return 0;
}

int check_stride(const char* name, int64_t s) {
    if (s < 0 || s > kMaxStride) return fail(PM_E_SHAPE, "%s %lld out of range", name, static_cast<long long>(s));
    return 0;
}

bool sizes_fit(int n_seqs, int T, int C, bool packed, int x_dtype) {
    if (static_cast<int64_t>(n_seqs) * C > kMaxElems || T > INT32_MAX - 1024) return false;
    const int64_t rows = packed ? C : static_cast<int64_t>(n_seqs) * C;
    if (T > 0 && rows > kMaxElems / T) return false;
    // (the counter that hands out tiles has 32 bits)
    return pm::recurrence_tiles(n_seqs, T, C, packed, x_dtype == PM_DTYPE_BF16) <= (int64_t(1) << 31);
}

int check_sizes(int n_seqs, int T, int C, bool packed, int x_dtype) {
    if (n_seqs < 0 || T < 0 || C < 0) return fail(PM_E_SHAPE, "sizes must be >= 0 (got %d, %d, %d)", n_seqs, T, C);
    return sizes_fit(n_seqs, T, C, packed, x_dtype) ? 0 : fail(PM_E_SHAPE, "problem too large");
}

}  // namespace

extern "C" {

size_t pm_linear_recurrence_workspace_bytes(int n_seqs, int T, int C, int packed, int x_dtype) {
    if (!known(x_dtype) || n_seqs <= 0 || T <= 0 || C <= 0 || !sizes_fit(n_seqs, T, C, packed != 0, x_dtype)) return 0;
    return pm::recurrence_ws_bytes(n_seqs, T, C, packed != 0, x_dtype == PM_DTYPE_BF16);
}

int pm_linear_recurrence_varlen(const void* x, const void* g, const int32_t* cu_seqlens, const float* s0,
                                const int32_t* slots, int n_slots, int32_t* bad_slot, int32_t* cu_flag, void* h,
                                float* s_out, float* kept, int n_seqs, int T, int C, int64_t x_sb, int64_t x_st,
                                int64_t g_sb, int64_t g_st, int x_dtype, int g_dtype, int h_dtype, void* workspace,
                                size_t ws_bytes, void* stream) {
    pm::clear_error();
    if (int rc = check_types(x_dtype, g_dtype, h_dtype)) return rc;
    if (int rc = check_sizes(n_seqs, T, C, cu_seqlens != nullptr, x_dtype)) return rc;
    if (int rc = check_stride("x_sb", x_sb)) return rc;
    if (int rc = check_stride("x_st", x_st)) return rc;
    if (int rc = check_stride("g_sb", g_sb)) return rc;
    if (int rc = check_stride("g_st", g_st)) return rc;
    if (n_seqs == 0 || C == 0) return 0;
    if (slots && n_slots < 0) return fail(PM_E_SHAPE, "n_slots must be >= 0 (got %d)", n_slots);
    if (!s_out) return fail(PM_E_NULL, "s_out is NULL");
    if (slots && s0 != s_out) return fail(PM_E_SHAPE, "with slots, s0 and s_out are the same pool");
    if (T > 0 && (!x || !g || !h)) return fail(PM_E_NULL, "x, g and h must be non-NULL");
    if (kept && cu_seqlens) return fail(PM_E_UNSUPPORTED, "states are kept for fixed-length batches only");
    if (!aligned(x, size_of(x_dtype)) || !aligned(g, size_of(g_dtype)) || !aligned(h, size_of(h_dtype)) ||
        !aligned(s0, 4) || !aligned(s_out, 4) || !aligned(kept, 4) || !aligned(cu_seqlens, 4) || !aligned(slots, 4) ||
        !aligned(bad_slot, 4) || !aligned(cu_flag, 4))
        return fail(PM_E_ALIGN, "every buffer must be aligned to its element size");
    const size_t need = pm_linear_recurrence_workspace_bytes(n_seqs, T, C, cu_seqlens != nullptr, x_dtype);
    if (need && (!workspace || ws_bytes < need || !aligned(workspace, 16)))
        return fail(PM_E_WORKSPACE, "a 16-byte aligned workspace of %zu bytes is needed (got %zu)", need,
                    workspace ? ws_bytes : static_cast<size_t>(0));
    pm::RecurrenceArgs a{x, g, cu_seqlens, s0, slots, n_slots, bad_slot, h, s_out, kept, n_seqs, T, C, x_sb, x_st,
                         g_sb, g_st, x_dtype == PM_DTYPE_BF16, g_dtype == PM_DTYPE_BF16, h_dtype == PM_DTYPE_BF16,
                         workspace, cu_flag};
    hipError_t e = pm::launch_recurrence(a, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? 0 : hip_fail(e, "linear recurrence launch");
}

int pm_linear_recurrence(const void* x, const void* g, const int32_t* cu_seqlens, const float* s0,
                         const int32_t* slots, int n_slots, int32_t* bad_slot, void* h, float* s_out, float* kept,
                         int n_seqs, int T, int C, int64_t x_sb, int64_t x_st, int64_t g_sb, int64_t g_st,
                         int x_dtype, int g_dtype, int h_dtype, void* workspace, size_t ws_bytes, void* stream) {
    return pm_linear_recurrence_varlen(x, g, cu_seqlens, s0, slots, n_slots, bad_slot, nullptr, h, s_out, kept, n_seqs,
                                       T, C, x_sb, x_st, g_sb, g_st, x_dtype, g_dtype, h_dtype, workspace, ws_bytes,
                                       stream);
}

int pm_linear_recurrence_bwd(const void* x, const void* g, const float* kept, const void* gh, const float* gs,
                             void* gx, void* gg, float* gs0, int B, int T, int C, int64_t x_sb, int64_t x_st,
                             int64_t g_sb, int64_t g_st, int x_dtype, int g_dtype, int h_dtype, void* workspace,
                             size_t ws_bytes, void* stream) {
    pm::clear_error();
    if (int rc = check_types(x_dtype, g_dtype, h_dtype)) return rc;
    if (int rc = check_sizes(B, T, C, false, x_dtype)) return rc;
    if (int rc = check_stride("x_sb", x_sb)) return rc;
    if (int rc = check_stride("x_st", x_st)) return rc;
    if (int rc = check_stride("g_sb", g_sb)) return rc;
    if (int rc = check_stride("g_st", g_st)) return rc;
    if (B == 0 || C == 0) return 0;
    if (!gs0) return fail(PM_E_NULL, "gs0 is NULL");
    if (T > 0 && (!x || !g || !kept || !gx || !gg))
        return fail(PM_E_NULL, "x, g, kept, gx and gg must be non-NULL");
    if (!aligned(x, size_of(x_dtype)) || !aligned(g, size_of(g_dtype)) || !aligned(gh, size_of(h_dtype)) ||
        !aligned(gx, size_of(x_dtype)) || !aligned(gg, size_of(g_dtype)) || !aligned(kept, 4) || !aligned(gs, 4) ||
        !aligned(gs0, 4))
        return fail(PM_E_ALIGN, "every buffer must be aligned to its element size");
    const size_t need = pm_linear_recurrence_workspace_bytes(B, T, C, 0, x_dtype);
    if (need && (!workspace || ws_bytes < need || !aligned(workspace, 16)))
        return fail(PM_E_WORKSPACE, "a 16-byte aligned workspace of %zu bytes is needed (got %zu)", need,
                    workspace ? ws_bytes : static_cast<size_t>(0));
    pm::RecurrenceBwdArgs a{x, g, kept, gh, gs, gx, gg, gs0, B, T, C, x_sb, x_st, g_sb, g_st,
                            x_dtype == PM_DTYPE_BF16, g_dtype == PM_DTYPE_BF16, h_dtype == PM_DTYPE_BF16, workspace};
    hipError_t e = pm::launch_recurrence_bwd(a, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? 0 : hip_fail(e, "linear recurrence backward launch");
}

int pm_linear_recurrence_step(float* s_inout, const int32_t* slots, int n_slots, const void* x, const void* g, void* h,
                              int B, int C, int64_t x_sb, int64_t g_sb, int x_dtype, int g_dtype, int h_dtype,
                              void* stream) {
    pm::clear_error();
    if (int rc = check_types(x_dtype, g_dtype, h_dtype)) return rc;
    if (int rc = check_sizes(B, 1, C, false, x_dtype)) return rc;
    if (int rc = check_stride("x_sb", x_sb)) return rc;
    if (int rc = check_stride("g_sb", g_sb)) return rc;
    if (B == 0 || C == 0) return 0;
    if (slots && n_slots < 0) return fail(PM_E_SHAPE, "n_slots must be >= 0 (got %d)", n_slots);
    if (!s_inout || !x || !g || !h) return fail(PM_E_NULL, "s_inout, x, g and h must be non-NULL");
    if (!aligned(x, size_of(x_dtype)) || !aligned(g, size_of(g_dtype)) || !aligned(h, size_of(h_dtype)) ||
        !aligned(s_inout, 4) || !aligned(slots, 4))
        return fail(PM_E_ALIGN, "every buffer must be aligned to its element size");
    pm::RecurrenceStepArgs a{s_inout, slots, n_slots, x, g, h, B, C, x_sb, g_sb, x_dtype == PM_DTYPE_BF16,
                             g_dtype == PM_DTYPE_BF16, h_dtype == PM_DTYPE_BF16};
    hipError_t e = pm::launch_recurrence_step(a, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? 0 : hip_fail(e, "linear recurrence step launch");
}

}  // extern "C"

namespace {

// What the forward and the backward of norm_rotate check alike; fills `a`.
int norm_rotate_args(pm::NormRotateArgs& a, const void* q, const void* k, const float* table, const void* positions,
                     const void* q_weight, const void* k_weight, int B, int T, int Hq, int Hk, int D, int R, int P,
                     const int64_t* strides, int64_t pos_sb, int pos_is_int64, int norm, float eps, int interleaved,
                     int dtype, int w_dtype) {
    if (!known(dtype) || !known(w_dtype))
        return fail(PM_E_DTYPE, "types %d, %d: each must be PM_DTYPE_F32 or PM_DTYPE_BF16", dtype, w_dtype);
    if (norm != PM_NORM_L2 && norm != PM_NORM_RMS) return fail(PM_E_SHAPE, "norm %d is not PM_NORM_L2 or PM_NORM_RMS", norm);
    if (B < 0 || T < 0 || Hq < 0 || Hk < 0)
        return fail(PM_E_SHAPE, "B, T, Hq, Hk must be >= 0 (got %d, %d, %d, %d)", B, T, Hq, Hk);
    if (D < 1 || D > PM_DELTA_MAX_D) return fail(PM_E_SHAPE, "D must be in [1, %d] (got %d)", PM_DELTA_MAX_D, D);
    if (R < 0 || R > D || R % 2) return fail(PM_E_SHAPE, "R must be even and in [0, D] (got %d)", R);
    if (!(eps >= 0.f)) return fail(PM_E_SHAPE, "eps must be >= 0");
    const int64_t heads = static_cast<int64_t>(Hq) + Hk;
    if (heads > (1 << 24) || static_cast<int64_t>(B) * T > kMaxElems || static_cast<int64_t>(B) * T * heads > kMaxElems)
        return fail(PM_E_SHAPE, "problem too large");
    if (R && P > 0 && !table) return fail(PM_E_NULL, "table is NULL");  // (without rows there is nothing to read)
    if (R && P < 0) return fail(PM_E_SHAPE, "P must be >= 0 (got %d)", P);
    if (!strides) return fail(PM_E_NULL, "strides is NULL");
    for (int i = 0; i < 6; ++i)
        if (int rc = check_stride("a stride", strides[i])) return rc;
    if (int rc = check_stride("pos_sb", pos_sb)) return rc;
    const size_t es = size_of(dtype);
    const bool some = B > 0 && T > 0;
    if (some && ((Hq && !q) || (Hk && !k))) return fail(PM_E_NULL, "q and k must be non-NULL");
    if (!aligned(q, es) || !aligned(k, es) || !aligned(q_weight, size_of(w_dtype)) ||
        !aligned(k_weight, size_of(w_dtype)) || !aligned(table, 4) || !aligned(positions, pos_is_int64 ? 8 : 4))
        return fail(PM_E_ALIGN, "every buffer must be aligned to its element size");
    a = pm::NormRotateArgs{};
    a.x[0] = q, a.x[1] = k;
    a.weight[0] = q_weight, a.weight[1] = k_weight;
    a.H[0] = Hq, a.H[1] = Hk;
    for (int s = 0; s < 2; ++s) a.sb[s] = strides[3 * s], a.st[s] = strides[3 * s + 1], a.sh[s] = strides[3 * s + 2];
    a.table = R ? table : nullptr;
    a.pos = positions;
    a.pos_sb = pos_sb;
    a.B = B, a.T = T, a.D = D, a.R = R, a.P = P;
    a.pos64 = pos_is_int64 != 0;
    a.bf16 = dtype == PM_DTYPE_BF16;
    a.w_bf16 = w_dtype == PM_DTYPE_BF16;
    a.rms = norm == PM_NORM_RMS;
    a.interleaved = interleaved != 0;
    a.eps = eps;
    return 0;
}

}  // namespace

extern "C" {

int pm_norm_rotate(const void* q, const void* k, const float* table, const void* positions, const void* q_weight,
                   const void* k_weight, void* q_out, void* k_out, int B, int T, int Hq, int Hk, int D, int R, int P,
                   const int64_t* strides, int64_t pos_sb, int pos_is_int64, int norm, float eps, int interleaved,
                   int dtype, int w_dtype, void* stream) {
    pm::clear_error();
    pm::NormRotateArgs a;
    if (int rc = norm_rotate_args(a, q, k, table, positions, q_weight, k_weight, B, T, Hq, Hk, D, R, P, strides,
                                  pos_sb, pos_is_int64, norm, eps, interleaved, dtype, w_dtype))
        return rc;
    if (static_cast<int64_t>(B) * T * (static_cast<int64_t>(Hq) + Hk) == 0) return 0;
    if ((Hq && !q_out) || (Hk && !k_out)) return fail(PM_E_NULL, "q_out and k_out must be non-NULL");
    if (!aligned(q_out, size_of(dtype)) || !aligned(k_out, size_of(dtype)))
        return fail(PM_E_ALIGN, "every buffer must be aligned to its element size");
    a.y[0] = q_out, a.y[1] = k_out;
    hipError_t e = pm::launch_norm_rotate(a, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? 0 : hip_fail(e, "norm and rotation launch");
}

size_t pm_norm_rotate_bwd_workspace_bytes(int B, int T, int Hq, int Hk, int D) {
    if (B < 0 || T < 0 || Hq < 0 || Hk < 0 || D < 1 || D > PM_DELTA_MAX_D) return 0;
    return pm::norm_rotate_bwd_ws_bytes(B, T, Hq, Hk, D);
}

int pm_norm_rotate_bwd(const void* q, const void* k, const float* table, const void* positions, const void* q_weight,
                       const void* k_weight, const void* gq_out, const void* gk_out, void* gq, void* gk,
                       float* gq_weight, float* gk_weight, int B, int T, int Hq, int Hk, int D, int R, int P,
                       const int64_t* strides, int64_t pos_sb, int pos_is_int64, int norm, float eps, int interleaved,
                       int dtype, int w_dtype, void* workspace, size_t ws_bytes, void* stream) {
    pm::clear_error();
    pm::NormRotateArgs a;
    if (int rc = norm_rotate_args(a, q, k, table, positions, q_weight, k_weight, B, T, Hq, Hk, D, R, P, strides,
                                  pos_sb, pos_is_int64, norm, eps, interleaved, dtype, w_dtype))
        return rc;
    if (!aligned(gq_weight, 4) || !aligned(gk_weight, 4))
        return fail(PM_E_ALIGN, "every buffer must be aligned to its element size");
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (static_cast<int64_t>(B) * T * (static_cast<int64_t>(Hq) + Hk) == 0) {  // sums over nothing
        for (float* gw : {gq_weight, gk_weight})
            if (gw)
                if (hipError_t e = pm::launch_fill_zero(gw, static_cast<size_t>(D), st); e != hipSuccess)
                    return hip_fail(e, "weight gradient fill");
        return 0;
    }
    if ((Hq && !gq) || (Hk && !gk)) return fail(PM_E_NULL, "gq and gk must be non-NULL");
    const size_t es = size_of(dtype);
    if (!aligned(gq_out, es) || !aligned(gk_out, es) || !aligned(gq, es) || !aligned(gk, es))
        return fail(PM_E_ALIGN, "every buffer must be aligned to its element size");
    const size_t need = pm::norm_rotate_bwd_ws_bytes(B, T, Hq, Hk, D);
    if ((gq_weight || gk_weight) && (!workspace || ws_bytes < need || !aligned(workspace, 16)))
        return fail(PM_E_WORKSPACE, "the weights' gradients need a 16-byte aligned workspace of %zu bytes (got %zu)",
                    need, workspace ? ws_bytes : static_cast<size_t>(0));
    if ((gq_weight && !q_weight) || (gk_weight && !k_weight))
        return fail(PM_E_NULL, "a weight's gradient needs the weight");
    a.gy[0] = gq_out, a.gy[1] = gk_out;
    a.gx[0] = gq, a.gx[1] = gk;
    a.gw[0] = gq_weight, a.gw[1] = gk_weight;
    a.workspace = workspace;
    hipError_t e = pm::launch_norm_rotate_bwd(a, st);
    return e == hipSuccess ? 0 : hip_fail(e, "norm and rotation backward launch");
}

}  // extern "C"
