// The C entries of the training operators (include/wc_b200.h): argument
// checks, then the launch.
#include <atomic>
#include <cmath>
#include <exception>
#include <initializer_list>
#include <string>

#include "../../include/wc_b200.h"
#include "cuda/train_ops.h"
#include "runtime.h"

namespace {

int bad(const char* what, const char* why) {
    wc::set_error(std::string(what) + ": " + why);
    return WC_E_ARG;
}

// Runs the launch and turns a CUDA error (the launch's own, or one pending
// from before) into a status.
template <class F>
int launched(const char* what, F&& f) {
    try {
        f();
    } catch (const std::exception& e) {
        wc::set_error(std::string(what) + ": " + e.what());
        return WC_E_CUDA;
    }
    const cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) return WC_OK;
    wc::set_error(std::string(what) + ": " + cudaGetErrorString(e));
    return WC_E_CUDA;
}

std::atomic<uint64_t> g_wait_ns{wc::DEFAULT_WAIT_NS};

bool type_ok(int t) { return t == WC_F32 || t == WC_F16 || t == WC_BF16; }
bool size_ok(int64_t rows, int64_t width) { return rows >= 0 && width >= 0 && rows <= (1ll << 31) && width <= (1ll << 31); }
bool off(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; }

// elements at addresses that are no multiple of their size
bool loose(int type, std::initializer_list<const void*> ps) {
    for (const void* p : ps)
        if (off(p, type == WC_F32 ? 4 : 2)) return true;
    return false;
}

}  // namespace

uint64_t wctrain::wait_limit() { return g_wait_ns; }

extern "C" {

int wc_debug_set_train_wait_limit(uint64_t ns) {
    g_wait_ns = ns ? ns : wc::DEFAULT_WAIT_NS;
    return WC_OK;
}

uint64_t wc_policy_loss_workspace(int64_t rows, int64_t width) {
    return size_ok(rows, width) ? wctrain::policy_loss_workspace(rows, width) : 0;
}

int wc_policy_loss(const wc_policy_loss_args* a, void* stream) {
    const char* me = "policy_loss";
    if (!a) return bad(me, "null arguments");
    if (!type_ok(a->type)) return bad(me, "unknown element type");
    if (a->action_bytes != 4 && a->action_bytes != 8) return bad(me, "action_bytes is 4 or 8");
    if (!size_ok(a->rows, a->width)) return bad(me, "sizes out of range");
    if (!a->loss) return bad(me, "null device pointer");
    if (!a->workspace || off(a->workspace, 16)) return bad(me, "no 16-byte aligned workspace");
    if (a->rows) {
        if (!a->actions || !a->old_logp || !a->advantages || !a->row_out) return bad(me, "null device pointer");
        if (a->width) {
            if (!a->logits) return bad(me, "null device pointer");
            if (a->ld_logits < a->width || (a->legal && a->ld_legal < a->width) || (a->dlogits && a->ld_dlogits < a->width))
                return bad(me, "row stride below the width");
        }
    }
    if (loose(a->type, {a->logits, a->dlogits}) || off(a->actions, a->action_bytes) ||
        loose(WC_F32, {a->old_logp, a->advantages, a->weights, a->ref_logp, a->upstream, a->loss, a->row_out}))
        return bad(me, "an address is not aligned to its elements");
    if (!(a->clip_low >= 0) || !(a->clip_high >= 0)) return bad(me, "a clip range below 0");
    if (!std::isfinite(a->kl_coef) || !std::isfinite(a->entropy_coef)) return bad(me, "a coefficient is not finite");
    return launched(me, [&] { wctrain::launch_policy_loss(*a, static_cast<cudaStream_t>(stream)); });
}

static int check_norm(const char* me, const wc_block_norm_args* a) {
    if (!a) return bad(me, "null arguments");
    if (!type_ok(a->type)) return bad(me, "unknown element type");
    if (a->kind != WC_NORM_LAYER && a->kind != WC_NORM_RMS) return bad(me, "unknown kind of norm");
    if (!size_ok(a->rows, a->width) || a->width > 16384) return bad(me, "sizes out of range (widths up to 16384)");
    if (a->gate && a->rows_per_gate < 1) return bad(me, "rows_per_gate below 1");
    if (a->kind == WC_NORM_RMS && (a->post_bias || a->pre_bias)) return bad(me, "RMSNorm has no bias");
    if ((a->post_bias && !a->post_weight) || (a->pre_bias && !a->pre_weight)) return bad(me, "a bias without its weight");
    if (!(a->eps >= 0) || !std::isfinite(a->eps)) return bad(me, "eps is not a finite number of at least 0");
    if (!std::isfinite(a->residual_scale)) return bad(me, "residual_scale is not finite");
    if (a->rows && a->width) {
        if (!a->x || !a->h || !a->stats) return bad(me, "null device pointer");
        if (a->ld_x < a->width || a->ld_h < a->width) return bad(me, "row stride below the width");
        if (off(a->stats, 16)) return bad(me, "stats is not 16-byte aligned");
        if (loose(a->type, {a->x, a->h, a->gate, a->y, a->n}) || loose(WC_F32, {a->post_weight, a->post_bias, a->pre_weight, a->pre_bias}))
            return bad(me, "an address is not aligned to its elements");
    }
    return WC_OK;
}

int wc_block_norm(const wc_block_norm_args* a, void* stream) {
    const char* me = "block_norm";
    if (const int rc = check_norm(me, a)) return rc;
    if ((a->n || a->n_q) && !a->pre_weight) return bad(me, "n needs a pre norm");
    if (!a->n_q != !a->n_scale) return bad(me, "n_q and n_scale come together");
    if (!a->rows || !a->width) return WC_OK;
    if (!a->y) return bad(me, "null device pointer");
    if (a->ld_y < a->width || (a->n && a->ld_n < a->width)) return bad(me, "row stride below the width");
    if (off(a->n_q, 16)) return bad(me, "n_q is not 16-byte aligned");
    return launched(me, [&] { wctrain::launch_block_norm(*a, static_cast<cudaStream_t>(stream)); });
}

uint64_t wc_block_norm_workspace(const wc_block_norm_args* a) {
    return check_norm("block_norm_workspace", a) == WC_OK && a->width ? wctrain::block_norm_workspace(*a) : 0;
}

int wc_block_norm_backward(const wc_block_norm_args* a, const wc_block_norm_grads* g, void* stream) {
    const char* me = "block_norm_backward";
    if (const int rc = check_norm(me, a)) return rc;
    if (!g) return bad(me, "null arguments");
    if (g->dn && !a->pre_weight) return bad(me, "dn needs a pre norm");
    if (a->rows && !g->dy && !g->dn) return bad(me, "neither dy nor dn");
    if (g->dgate && !a->gate) return bad(me, "dgate without a gate");
    if ((g->dpost_weight && !a->post_weight) || (g->dpost_bias && !a->post_bias) || (g->dpre_weight && !a->pre_weight) ||
        (g->dpre_bias && !a->pre_bias))
        return bad(me, "the gradient of a weight that is not there");
    if (!a->width) return WC_OK;
    if (!g->workspace || off(g->workspace, 16)) return bad(me, "no 16-byte aligned workspace");
    if (a->rows && ((g->dy && g->ld_dy < a->width) || (g->dn && g->ld_dn < a->width) || (g->dx && g->ld_dx < a->width) ||
                    (g->dh && g->ld_dh < a->width)))
        return bad(me, "row stride below the width");
    if (loose(a->type, {g->dy, g->dn, g->dx, g->dh, g->dgate}) ||
        loose(WC_F32, {g->dpost_weight, g->dpost_bias, g->dpre_weight, g->dpre_bias}))
        return bad(me, "an address is not aligned to its elements");
    return launched(me, [&] { wctrain::launch_block_norm_backward(*a, *g, static_cast<cudaStream_t>(stream)); });
}

static int check_act8(const char* me, const wc_act8_args* a, bool x, bool out) {
    if (!a) return bad(me, "null arguments");
    if (!type_ok(a->type)) return bad(me, "unknown element type");
    if (!size_ok(a->rows, a->width)) return bad(me, "sizes out of range");
    if (!a->rows || !a->width) return WC_OK;
    if (!a->q || !a->scale || (x && !a->x) || (out && !a->out)) return bad(me, "null device pointer");
    if ((x && a->ld_x < a->width) || (out && a->ld_out < a->width)) return bad(me, "row stride below the width");
    if (off(a->q, 16)) return bad(me, "q is not 16-byte aligned");
    if (loose(a->type, {x ? a->x : nullptr, out ? a->out : nullptr}) || loose(WC_F32, {a->bias, a->dbias}))
        return bad(me, "an address is not aligned to its elements");
    return WC_OK;
}

int wc_act8_pack(const wc_act8_args* a, void* stream) {
    if (const int rc = check_act8("act8_pack", a, true, false)) return rc;
    if (!a->rows || !a->width) return WC_OK;
    return launched("act8_pack", [&] { wctrain::launch_act8_pack(*a, static_cast<cudaStream_t>(stream)); });
}

int wc_act8_unpack(const wc_act8_args* a, void* stream) {
    if (const int rc = check_act8("act8_unpack", a, false, true)) return rc;
    if (!a->rows || !a->width) return WC_OK;
    return launched("act8_unpack", [&] { wctrain::launch_act8_unpack(*a, static_cast<cudaStream_t>(stream)); });
}

int wc_gelu8(const wc_act8_args* a, void* stream) {
    if (const int rc = check_act8("gelu8", a, true, true)) return rc;
    if (!a->rows || !a->width) return WC_OK;
    return launched("gelu8", [&] { wctrain::launch_gelu8(*a, static_cast<cudaStream_t>(stream)); });
}

uint64_t wc_gelu8_workspace(int64_t rows, int64_t width) {
    return size_ok(rows, width) ? wctrain::gelu8_workspace(rows, width) : 0;
}

int wc_gelu8_backward(const wc_act8_args* a, void* stream) {
    const char* me = "gelu8_backward";
    if (const int rc = check_act8(me, a, true, true)) return rc;
    if (!a->width) return WC_OK;
    if (a->dbias && (!a->workspace || off(a->workspace, 16))) return bad(me, "no 16-byte aligned workspace");
    if (!a->rows && !a->dbias) return WC_OK;
    return launched(me, [&] { wctrain::launch_gelu8_backward(*a, static_cast<cudaStream_t>(stream)); });
}

static int check_wgrad(const char* me, const wc_act8_wgrad_args* a) {
    if (!a) return bad(me, "null arguments");
    if (!type_ok(a->type) || !type_ok(a->out_type)) return bad(me, "unknown element type");
    if (!size_ok(a->rows, a->k) || !size_ok(a->rows, a->n) || a->k > (1 << 20) || a->n > (1 << 20))
        return bad(me, "sizes out of range (k and n up to 2^20)");
    if (a->k < 1) return bad(me, "k below 1");
    if ((a->rows / 64 + 1) * (a->k / 128 + 1) * (a->n / 64 + 1) >= 1ll << 31) return bad(me, "sizes out of range");
    return WC_OK;
}

uint64_t wc_act8_wgrad_workspace(const wc_act8_wgrad_args* a) {
    return check_wgrad("act8_wgrad_workspace", a) == WC_OK ? wctrain::wgrad8_workspace(*a) : 0;
}

int wc_act8_wgrad(const wc_act8_wgrad_args* a, void* stream) {
    const char* me = "act8_wgrad";
    if (const int rc = check_wgrad(me, a)) return rc;
    if (!a->n) return WC_OK;
    if (!a->dw) return bad(me, "null device pointer");
    if (!a->workspace || off(a->workspace, 16)) return bad(me, "no 16-byte aligned workspace");
    if (a->rows) {
        if (!a->dy || !a->q || !a->scale) return bad(me, "null device pointer");
        if (a->ld_dy < a->n) return bad(me, "row stride below the width");
        if (off(a->q, 16)) return bad(me, "q is not 16-byte aligned");
    }
    if (loose(a->type, {a->dy}) || loose(a->out_type, {a->dw}) || loose(WC_F32, {a->db}))
        return bad(me, "an address is not aligned to its elements");
    return launched(me, [&] { wctrain::launch_wgrad8(*a, static_cast<cudaStream_t>(stream)); });
}

}  // extern "C"
