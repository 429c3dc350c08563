// pm_decay_abi.hip — the extern "C" entry points of K14 (decay_attention.hip) and of the norms around
// such a layer, K15 (gated_norm.hip) and K16 (residual_norm.hip).
//
// As in pm_delta_abi.hip every argument is checked before anything is launched; errors are
// negative PM_E_* codes with a message in pm_last_error().

#include <algorithm>
#include <cmath>

#include "pm_common.h"
#include "pm_internal.h"
#include "../../include/pm_delta.h"

static_assert(PM_NORM_MAX_ROW == pm::kMaxRow, "the header's widest row is the kernels'");

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

constexpr int64_t kMaxGroups = (int64_t(1) << 24) - 1;  // workgroups of 256 that one launch can have
constexpr int64_t kMaxTokenStride = int64_t(1) << 23;  // (64 tokens are reached with 32-bit offsets)

int check_stride(const char* name, int64_t s) {
    if (s < 0 || s > kMaxStride) return fail(PM_E_SHAPE, "%s %lld out of range", name, static_cast<long long>(s));
    return 0;
}

// What a call of K14 launches.
enum class Decay { kForward, kPacked, kBackward, kStep };

bool decay_sizes_fit(Decay call, int n, int T, int Hq, int H, int D) {
    if (n < 0 || T < 0 || Hq < 1 || H < 1 || Hq % H || D < 1 || D > PM_DELTA_MAX_D) return false;
    const int64_t width = static_cast<int64_t>(Hq) * D;
    if (T > INT32_MAX - 1024 || width > kMaxTokenStride) return false;
    const int64_t rows = (call == Decay::kPacked ? 1 : static_cast<int64_t>(n)) * std::max(T, 1);
    if (rows > kMaxElems / width || static_cast<int64_t>(n) * H > kMaxElems / (static_cast<int64_t>(D) * D)) return false;
    switch (call) {
        case Decay::kStep: return true;
        case Decay::kBackward:  // (the pairs inside chunks: a workgroup to 128 tokens at least)
            return static_cast<int64_t>(n) * Hq * (T / 128 + 1) <= kMaxGroups &&
                   pm::decay_attn_bwd_groups(n, T, Hq, H, D) <= kMaxGroups;
        default: return pm::decay_attn_groups(n, T, Hq, H, D, call == Decay::kPacked) <= kMaxGroups;
    }
}

// Sizes, types and strides that the calls of K14 share.
int check_decay(Decay call, int n, int T, int Hq, int H, int D, int dtype, int out_dtype, const int64_t* strides,
                int n_strides, int64_t g_sb, int64_t g_st, float scale) {
    if (!known(dtype) || !known(out_dtype))
        return fail(PM_E_DTYPE, "types %d, %d: each must be PM_DTYPE_F32 or PM_DTYPE_BF16", dtype, out_dtype);
    if (n < 0 || T < 0) return fail(PM_E_SHAPE, "sizes must be >= 0 (got %d, %d)", n, T);
    if (Hq < 1 || H < 1 || Hq % H) return fail(PM_E_SHAPE, "Hq must be a multiple of H >= 1 (got %d, %d)", Hq, H);
    if (D < 1 || D > PM_DELTA_MAX_D) return fail(PM_E_SHAPE, "D must be in [1, %d] (got %d)", PM_DELTA_MAX_D, D);
    if (!decay_sizes_fit(call, n, T, Hq, H, D)) return fail(PM_E_SHAPE, "problem too large");
    if (!strides) return fail(PM_E_NULL, "strides is NULL");
    for (int i = 0; i < n_strides; ++i)
        if (int rc = check_stride("a stride", strides[i])) return rc;
    if (n_strides == 9)
        for (int i = 1; i < 9; i += 3)
            if (T > 1 && strides[i] > kMaxTokenStride)
                return fail(PM_E_SHAPE, "token strides of at most %lld elements (got %lld)",
                            static_cast<long long>(kMaxTokenStride), static_cast<long long>(strides[i]));
    if (int rc = check_stride("g_sb", g_sb)) return rc;
    if (int rc = check_stride("g_st", g_st)) return rc;
    if (!std::isfinite(scale)) return fail(PM_E_SHAPE, "scale must be finite");
    return 0;
}

int check_ws(size_t need, const void* workspace, size_t ws_bytes) {
    if (need && (!workspace || ws_bytes < need || !aligned(workspace, 16)))
        return fail(PM_E_WORKSPACE, "a 16-byte aligned workspace of %zu bytes is needed (got %zu)", need,
                    workspace ? ws_bytes : static_cast<size_t>(0));
    return 0;
}

const char* const kAlign = "every buffer must be aligned to its element size";

}  // namespace

extern "C" {

size_t pm_decay_attention_workspace_bytes(int n_seqs, int T, int Hq, int H, int D, int packed,
                                          int in_place) {
    if (!decay_sizes_fit(packed ? Decay::kPacked : Decay::kForward, n_seqs, T, Hq, H, D)) return 0;
    return pm::decay_attn_ws_bytes(n_seqs, T, Hq, H, D, packed != 0, in_place != 0);
}

int pm_decay_attention(const void* q, const void* k, const void* v, const float* g, const int32_t* cu_seqlens,
                       const float* s0, const int32_t* slots, int n_slots, int32_t* bad_slot, int32_t* cu_flag, void* o,
                       float* s_out, int n_seqs, int T, int Hq, int H, int D, const int64_t* strides, int64_t g_sb,
                       int64_t g_st, int dtype, int out_dtype, float scale, void* workspace, size_t ws_bytes,
                       void* stream) {
    pm::clear_error();
    if (int rc = check_decay(cu_seqlens ? Decay::kPacked : Decay::kForward, n_seqs, T, Hq, H, D, dtype, out_dtype,
                             strides, 9, g_sb, g_st, scale)) return rc;
    if (n_seqs == 0) return 0;
    if (slots && n_slots < 0) return fail(PM_E_SHAPE, "n_slots must be >= 0 (got %d)", n_slots);
    if (!s_out) return fail(PM_E_NULL, "s_out is NULL");
    if (slots && s0 != s_out) return fail(PM_E_SHAPE, "with slots, s0 and s_out are the same pool");
    if (T > 0 && (!q || !k || !v || !g || !o)) return fail(PM_E_NULL, "q, k, v, g and o must be non-NULL");
    const size_t es = size_of(dtype);
    if (!aligned(q, es) || !aligned(k, es) || !aligned(v, es) || !aligned(o, size_of(out_dtype)) || !aligned(g, 4) ||
        !aligned(s0, 4) || !aligned(s_out, 4) || !aligned(cu_seqlens, 4) || !aligned(slots, 4) || !aligned(bad_slot, 4) ||
        !aligned(cu_flag, 4))
        return fail(PM_E_ALIGN, "%s", kAlign);
    if (int rc = check_ws(pm::decay_attn_ws_bytes(n_seqs, T, Hq, H, D, cu_seqlens != nullptr, s0 && s0 == s_out),
                          workspace, ws_bytes))
        return rc;
    pm::DecayAttnArgs a{q, k, v, strides, g, g_sb, g_st, cu_seqlens, cu_flag, s0, s_out, slots, n_slots, bad_slot, o,
                        n_seqs, T, Hq, H, D, dtype == PM_DTYPE_BF16, out_dtype == PM_DTYPE_BF16, scale, workspace};
    hipError_t e = pm::launch_decay_attn(a, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? 0 : hip_fail(e, "decay attention launch");
}

size_t pm_decay_attention_bwd_workspace_bytes(int B, int T, int Hq, int H, int D, int gates) {
    if (!decay_sizes_fit(Decay::kBackward, B, T, Hq, H, D)) return 0;
    return pm::decay_attn_bwd_ws_bytes(B, T, Hq, H, D, gates != 0);
}

int pm_decay_attention_bwd(const void* q, const void* k, const void* v, const float* g, const float* s0, const void* go,
                           const float* gs, void* gq, void* gk, void* gv, float* gg, float* gs0, int B, int T, int Hq,
                           int H, int D, const int64_t* strides, int64_t g_sb, int64_t g_st, int dtype, float scale,
                           void* workspace, size_t ws_bytes, void* stream) {
    pm::clear_error();
    if (int rc = check_decay(Decay::kBackward, B, T, Hq, H, D, dtype, dtype, strides, 9, g_sb, g_st, scale)) return rc;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (B == 0) {
        if (gg && g_sb == 0 && g_st == 0)
            if (hipError_t e = pm::launch_fill_zero(gg, static_cast<size_t>(H), st); e != hipSuccess)
                return hip_fail(e, "gate gradient fill");
        return 0;
    }
    if (T > 0 && (!q || !k || !v || !g || !go || !gq || !gk || !gv))
        return fail(PM_E_NULL, "q, k, v, g, go, gq, gk and gv must be non-NULL");
    const size_t es = size_of(dtype);
    if (!aligned(q, es) || !aligned(k, es) || !aligned(v, es) || !aligned(go, es) || !aligned(gq, es) ||
        !aligned(gk, es) || !aligned(gv, es) || !aligned(g, 4) || !aligned(s0, 4) || !aligned(gs, 4) || !aligned(gg, 4) ||
        !aligned(gs0, 4))
        return fail(PM_E_ALIGN, "%s", kAlign);
    if (int rc = check_ws(pm::decay_attn_bwd_ws_bytes(B, T, Hq, H, D, gg != nullptr), workspace, ws_bytes)) return rc;
    pm::DecayAttnBwdArgs a{q, k, v, strides, g, g_sb, g_st, s0, go, gs, gq, gk, gv, gg, gs0, B, T, Hq, H, D,
                           dtype == PM_DTYPE_BF16, scale, workspace};
    hipError_t e = pm::launch_decay_attn_bwd(a, st);
    return e == hipSuccess ? 0 : hip_fail(e, "decay attention backward launch");
}

int pm_decay_attention_step(float* s_inout, const int32_t* slots, int n_slots, const void* q, const void* k,
                            const void* v, const float* g, void* o, int B, int Hq, int H, int D, const int64_t* strides,
                            int64_t g_sb, int dtype, int out_dtype, float scale, void* stream) {
    pm::clear_error();
    if (int rc = check_decay(Decay::kStep, B, 1, Hq, H, D, dtype, out_dtype, strides, 6, g_sb, 0, scale)) return rc;
    if (B == 0) return 0;
    if (slots && n_slots < 0) return fail(PM_E_SHAPE, "n_slots must be >= 0 (got %d)", n_slots);
    if (!s_inout || !q || !k || !v || !g || !o) return fail(PM_E_NULL, "s_inout, q, k, v, g and o must be non-NULL");
    const size_t es = size_of(dtype);
    if (!aligned(q, es) || !aligned(k, es) || !aligned(v, es) || !aligned(o, size_of(out_dtype)) || !aligned(g, 4) ||
        !aligned(s_inout, 4) || !aligned(slots, 4))
        return fail(PM_E_ALIGN, "%s", kAlign);
    pm::DecayAttnStepArgs a{s_inout, slots, n_slots, q, k, v, {}, g, g_sb, o, B, Hq, H, D, dtype == PM_DTYPE_BF16,
                            out_dtype == PM_DTYPE_BF16, scale};
    for (int i = 0; i < 6; ++i) a.strides[i] = strides[i];
    hipError_t e = pm::launch_decay_attn_step(a, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? 0 : hip_fail(e, "decay attention step launch");
}

}  // extern "C"

namespace {

int check_rows(int64_t rows, int C, float eps) {
    if (rows < 0) return fail(PM_E_SHAPE, "rows must be >= 0 (got %lld)", static_cast<long long>(rows));
    if (C < 1 || C > PM_NORM_MAX_ROW) return fail(PM_E_SHAPE, "C must be in [1, %d] (got %d)", PM_NORM_MAX_ROW, C);
    if (rows > kMaxElems / C) return fail(PM_E_SHAPE, "problem too large");
    if (!(eps >= 0.f)) return fail(PM_E_SHAPE, "eps must be >= 0");
    return 0;
}

int gated_args(pm::GatedNormArgs& a, const void* x, const void* z, const void* w, int64_t rows, int inner, int C,
               const int64_t* strides, int activation, int gate_first, float eps, int x_dtype, int z_dtype, int y_dtype,
               int w_dtype) {
    if (!known(x_dtype) || !known(z_dtype) || !known(y_dtype) || !known(w_dtype))
        return fail(PM_E_DTYPE, "types %d, %d, %d, %d: each must be PM_DTYPE_F32 or PM_DTYPE_BF16", x_dtype, z_dtype,
                    y_dtype, w_dtype);
    if (int rc = check_rows(rows, C, eps)) return rc;
    if (activation != PM_ACT_SILU && activation != PM_ACT_SIGMOID)
        return fail(PM_E_SHAPE, "activation %d is not PM_ACT_SILU or PM_ACT_SIGMOID", activation);
    if (inner < 1) return fail(PM_E_SHAPE, "inner must be >= 1 (got %d)", inner);
    if (!strides) return fail(PM_E_NULL, "strides is NULL");
    for (int i = 0; i < 4; ++i)
        if (int rc = check_stride("a stride", strides[i])) return rc;
    if (rows > 0 && (!x || !z)) return fail(PM_E_NULL, "x and the gate must be non-NULL");
    if (!aligned(x, size_of(x_dtype)) || !aligned(z, size_of(z_dtype)) || !aligned(w, size_of(w_dtype)))
        return fail(PM_E_ALIGN, "%s", kAlign);
    a = pm::GatedNormArgs{};
    a.x = x, a.z = z, a.w = w;
    a.rows = rows, a.inner = inner, a.C = C;
    a.x_so = strides[0], a.x_si = strides[1], a.z_so = strides[2], a.z_si = strides[3];
    a.x_bf16 = x_dtype == PM_DTYPE_BF16, a.z_bf16 = z_dtype == PM_DTYPE_BF16, a.y_bf16 = y_dtype == PM_DTYPE_BF16;
    a.w_bf16 = w_dtype == PM_DTYPE_BF16;
    a.silu = activation == PM_ACT_SILU, a.first = gate_first != 0, a.eps = eps;
    return 0;
}

int residual_args(pm::ResidualNormArgs& a, const void* x, const void* residual, const void* w, const void* wp,
                  int64_t rows, int C, int64_t x_st, int64_t r_st, float scale, float eps, int dtype, int r_dtype,
                  int w_dtype, int wp_dtype) {
    if (!known(dtype) || !known(r_dtype) || !known(w_dtype) || !known(wp_dtype))
        return fail(PM_E_DTYPE, "types %d, %d, %d, %d: each must be PM_DTYPE_F32 or PM_DTYPE_BF16", dtype, r_dtype,
                    w_dtype, wp_dtype);
    if (int rc = check_rows(rows, C, eps)) return rc;
    if (!std::isfinite(scale)) return fail(PM_E_SHAPE, "scale must be finite");
    if (int rc = check_stride("x_st", x_st)) return rc;
    if (int rc = check_stride("r_st", r_st)) return rc;
    if (rows > 0 && (!x || !residual)) return fail(PM_E_NULL, "x and residual must be non-NULL");
    if (!aligned(x, size_of(dtype)) || !aligned(residual, size_of(r_dtype)) || !aligned(w, size_of(w_dtype)) ||
        !aligned(wp, size_of(wp_dtype)))
        return fail(PM_E_ALIGN, "%s", kAlign);
    a = pm::ResidualNormArgs{};
    a.x = x, a.res = residual, a.w = w, a.wp = wp;
    a.rows = rows, a.C = C, a.x_st = x_st, a.r_st = r_st;
    a.x_bf16 = dtype == PM_DTYPE_BF16, a.r_bf16 = r_dtype == PM_DTYPE_BF16;
    a.w_bf16 = w_dtype == PM_DTYPE_BF16, a.wp_bf16 = wp_dtype == PM_DTYPE_BF16;
    a.eps = eps, a.scale = scale;
    return 0;
}

// The gradients of weights over no rows.
int zero_weights(float* const* gws, int n, int C, hipStream_t st) {
    for (int i = 0; i < n; ++i)
        if (gws[i])
            if (hipError_t e = pm::launch_fill_zero(gws[i], static_cast<size_t>(C), st); e != hipSuccess)
                return hip_fail(e, "weight gradient fill");
    return 0;
}

}  // namespace

extern "C" {

int pm_gated_norm(const void* x, const void* gate, const void* weight, void* y, int64_t rows, int inner, int C,
                  const int64_t* strides, int activation, int gate_first, float eps, int x_dtype, int gate_dtype,
                  int y_dtype, int w_dtype, void* stream) {
    pm::clear_error();
    pm::GatedNormArgs a;
    if (int rc = gated_args(a, x, gate, weight, rows, inner, C, strides, activation, gate_first, eps, x_dtype, gate_dtype,
                            y_dtype, w_dtype))
        return rc;
    if (rows == 0) return 0;
    if (!y) return fail(PM_E_NULL, "y is NULL");
    if (!aligned(y, size_of(y_dtype))) return fail(PM_E_ALIGN, "%s", kAlign);
    a.y = y;
    hipError_t e = pm::launch_gated_norm(a, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? 0 : hip_fail(e, "gated norm launch");
}

size_t pm_gated_norm_bwd_workspace_bytes(int64_t rows, int C) {
    if (rows <= 0 || C < 1 || C > PM_NORM_MAX_ROW) return 0;
    return static_cast<size_t>(pm::gated_norm_groups(rows, C)) * C * 4;
}

int pm_gated_norm_bwd(const void* x, const void* gate, const void* weight, const void* gy, void* gx, void* g_gate,
                      float* g_weight, int64_t rows, int inner, int C, const int64_t* strides, int activation,
                      int gate_first, float eps, int x_dtype, int gate_dtype, int y_dtype, int w_dtype, void* workspace,
                      size_t ws_bytes, void* stream) {
    pm::clear_error();
    pm::GatedNormArgs a;
    if (int rc = gated_args(a, x, gate, weight, rows, inner, C, strides, activation, gate_first, eps, x_dtype, gate_dtype,
                            y_dtype, w_dtype))
        return rc;
    if (!aligned(g_weight, 4)) return fail(PM_E_ALIGN, "%s", kAlign);
    if (g_weight && !weight) return fail(PM_E_NULL, "a weight's gradient needs the weight");
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (rows == 0) return zero_weights(&g_weight, 1, C, st);
    if (!gy || !gx || !g_gate) return fail(PM_E_NULL, "gy, gx and g_gate must be non-NULL");
    if (!aligned(gy, size_of(y_dtype)) || !aligned(gx, size_of(x_dtype)) || !aligned(g_gate, size_of(gate_dtype)))
        return fail(PM_E_ALIGN, "%s", kAlign);
    if (g_weight)
        if (int rc = check_ws(pm_gated_norm_bwd_workspace_bytes(rows, C), workspace, ws_bytes)) return rc;
    a.gy = gy, a.gx = gx, a.gz = g_gate, a.gw = g_weight, a.part = static_cast<float*>(workspace);
    hipError_t e = pm::launch_gated_norm_bwd(a, st);
    return e == hipSuccess ? 0 : hip_fail(e, "gated norm backward launch");
}

int pm_residual_norm(const void* x, const void* residual, const void* weight, const void* post_weight, void* y, void* h,
                     int64_t rows, int C, int64_t x_st, int64_t r_st, float scale, float eps, int dtype, int r_dtype,
                     int w_dtype, int post_w_dtype, void* stream) {
    pm::clear_error();
    pm::ResidualNormArgs a;
    if (int rc = residual_args(a, x, residual, weight, post_weight, rows, C, x_st, r_st, scale, eps, dtype, r_dtype,
                               w_dtype, post_w_dtype))
        return rc;
    if (rows == 0) return 0;
    if (!y || !h) return fail(PM_E_NULL, "y and h must be non-NULL");
    if (!aligned(y, size_of(dtype)) || !aligned(h, size_of(r_dtype))) return fail(PM_E_ALIGN, "%s", kAlign);
    a.y = y, a.h = h;
    hipError_t e = pm::launch_residual_norm(a, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? 0 : hip_fail(e, "residual norm launch");
}

size_t pm_residual_norm_bwd_workspace_bytes(int64_t rows, int C) {
    if (rows <= 0 || C < 1 || C > PM_NORM_MAX_ROW) return 0;
    return 2 * static_cast<size_t>(pm::residual_norm_groups(rows, C)) * C * 4;
}

int pm_residual_norm_bwd(const void* x, const void* residual, const void* weight, const void* post_weight,
                         const void* gy, const void* gh, void* gx, void* g_residual, float* g_weight,
                         float* g_post_weight, int64_t rows, int C, int64_t x_st, int64_t r_st, float scale, float eps,
                         int dtype, int r_dtype, int w_dtype, int post_w_dtype, void* workspace, size_t ws_bytes,
                         void* stream) {
    pm::clear_error();
    pm::ResidualNormArgs a;
    if (int rc = residual_args(a, x, residual, weight, post_weight, rows, C, x_st, r_st, scale, eps, dtype, r_dtype,
                               w_dtype, post_w_dtype))
        return rc;
    if (!aligned(g_weight, 4) || !aligned(g_post_weight, 4)) return fail(PM_E_ALIGN, "%s", kAlign);
    if ((g_weight && !weight) || (g_post_weight && !post_weight))
        return fail(PM_E_NULL, "a weight's gradient needs the weight");
    hipStream_t st = static_cast<hipStream_t>(stream);
    float* const gws[2] = {g_weight, g_post_weight};
    if (rows == 0) return zero_weights(gws, 2, C, st);
    if (!gx || !g_residual) return fail(PM_E_NULL, "gx and g_residual must be non-NULL");
    if (!aligned(gy, size_of(dtype)) || !aligned(gh, size_of(r_dtype)) || !aligned(gx, size_of(dtype)) ||
        !aligned(g_residual, size_of(r_dtype)))
        return fail(PM_E_ALIGN, "%s", kAlign);
    if (g_weight || g_post_weight)
        if (int rc = check_ws(pm_residual_norm_bwd_workspace_bytes(rows, C), workspace, ws_bytes)) return rc;
    a.gy = gy, a.gh = gh, a.gx = gx, a.gres = g_residual, a.gw = g_weight, a.gwp = g_post_weight;
    a.part = static_cast<float*>(workspace);
    hipError_t e = pm::launch_residual_norm_bwd(a, st);
    return e == hipSuccess ? 0 : hip_fail(e, "residual norm backward launch");
}

}  // extern "C"
